"""Attention over selected pages, plainly and in 64 bits on the CPU: the cache write with page
bounds, the choice of pages and the attention over them, from their definitions (snowllm_amd/
sparse.py). Pools in the page layouts of tests/kvcache.py; row t of request b is row b * T + t."""
import torch

PAGE = 16


def block_of(table, b, page, blocks):
    """The block of a request's page, or -1."""
    if not 0 <= page < table.shape[1]:
        return -1
    e = int(table[b, page])
    return e if 0 <= e < blocks else -1


def norm_rotate(x, gamma, cos, sin, eps):
    """x [rows, heads, d] -> (values, magnitude of the terms that each value sums) in 64 bits."""
    x = x.double()
    if gamma is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * gamma.double()
    half = cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    y = torch.cat([a * c - b * s, a * s + b * c, rest], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs(), rest.abs()], -1)
    return y, size


def slots(table, starts, counts, T, blocks):
    """(row, block, offset) of every row that is written."""
    found = []
    for b in range(table.shape[0]):
        start, count = int(starts[b]), min(int(counts[b]), T)
        if start < 0:
            continue
        for t in range(count):
            blk = block_of(table, b, (start + t) // PAGE, blocks)
            if blk >= 0:
                found.append((b * T + t, blk, (start + t) % PAGE))
    return found


def key(k_pool, blk, off):
    """The cached key [Hkv, d] of a slot."""
    return k_pool[blk, :, :, off].reshape(k_pool.shape[1], -1)


def value(v_pool, blk, off):
    return v_pool[blk, :, off // 4, :, off % 4]


def page_limits(k_pool, bounds, table, starts, counts, T):
    """bounds with the touched pages' minima and maxima over their live keys."""
    out = bounds.clone()
    blocks = k_pool.shape[0]
    for b in range(table.shape[0]):
        start, count = int(starts[b]), min(int(counts[b]), T)
        if start < 0 or count <= 0:
            continue
        for page in range(start // PAGE, (start + count - 1) // PAGE + 1):
            blk = block_of(table, b, page, blocks)
            if blk < 0:
                continue
            live = min(PAGE, start + count - page * PAGE)
            keys = k_pool[blk, :, :, :live].permute(2, 0, 1, 3).flatten(2).float()
            nan = keys.isnan().any(0)
            out[blk, :, 0] = keys.amin(0).masked_fill(nan, float("nan")).to(out.dtype)
            out[blk, :, 1] = keys.amax(0).masked_fill(nan, float("nan")).to(out.dtype)
    return out


def scores(q, bounds, table, b, head, hkv):
    """[pages] of request b for one row's q [Hq, d] and one kv head; no page: NaN."""
    G, d = q.shape[0] // hkv, q.shape[1]
    entry = table[b].long()
    ok = (entry >= 0) & (entry < bounds.shape[0])
    box = bounds[entry.clamp(0, bounds.shape[0] - 1), head].double()      # [pages, 2, d]
    group = q[head * G:(head + 1) * G].double()
    up, down = group.clamp(min=0).sum(0), group.clamp(max=0).sum(0)
    s = (up * box[:, 1]).sum(-1) + (down * box[:, 0]).sum(-1)
    # the same only for finite values (0 . inf): otherwise as it is defined, NaN where a term is
    odd = ~box.isfinite().all(-1).all(-1) | ~group.isfinite().all()
    if odd.any():
        terms = group[:, None, None] * box[odd]                           # [G, pages, 2, d]
        s[odd] = torch.maximum(terms[:, :, 0], terms[:, :, 1]).sum((0, 2))
    return s.masked_fill(~ok, float("nan"))


def select(q, bounds, table, positions, budget, sink, recent):
    M, hkv = q.shape[0], bounds.shape[1]
    T = M // table.shape[0]
    out = torch.full((M, hkv, budget), -1, dtype=torch.int32)
    for m in range(M):
        pos = int(positions[m])
        n = min(pos // PAGE + 1, table.shape[1]) if pos >= 0 else 0
        for h in range(hkv):
            if n <= budget:
                chosen = list(range(n))
            else:
                s = scores(q[m], bounds, table, m // T, h, hkv).tolist()
                rank = {p: -s[p] if s[p] == s[p] else float("inf") for p in range(sink, n - recent)}
                best = sorted(rank, key=lambda p: (rank[p], p))[:budget - sink - recent]
                chosen = sorted([*range(sink), *best, *range(n - recent, n)])
            out[m, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out


def attend(q, k_pool, v_pool, table, positions, pages, scale):
    """-> (out [M, Hq, d], sum of weights times |v|, largest sum of |q k| times scale) in 64 bits."""
    M, Hq, d = q.shape
    blocks, hkv = k_pool.shape[:2]
    T, G = M // table.shape[0], Hq // hkv
    out = torch.zeros(M, Hq, d, dtype=torch.float64)
    size, reach = torch.zeros_like(out), torch.zeros(M, Hq, 1, dtype=torch.float64)
    for m in range(M):
        pos = int(positions[m])
        for h in range(hkv):
            ks, vs = [], []
            for p in pages[m, h].tolist():
                blk = block_of(table, m // T, p, blocks)
                live = min(PAGE, pos + 1 - p * PAGE)
                if blk < 0 or pos < 0 or live <= 0:
                    continue
                ks.append(k_pool[blk, h, :, :live].permute(1, 0, 2).reshape(live, d))
                vs.append(v_pool[blk, h].permute(0, 2, 1).reshape(PAGE, d)[:live])
            if not ks:
                continue
            k, v = torch.cat(ks).double(), torch.cat(vs).double()
            x = q[m, h * G:(h + 1) * G].double()
            w = (x @ k.t() * scale).softmax(-1)
            out[m, h * G:(h + 1) * G] = w @ v
            size[m, h * G:(h + 1) * G] = w @ v.abs()
            reach[m, h * G:(h + 1) * G] = (x.abs() @ k.abs().t()).amax(-1, keepdim=True) * scale
    return out, size, reach
