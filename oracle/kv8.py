"""The paged cache in 8 bits, plainly and in 64 bits on the CPU: angles of several axes, quantised
write, read back and attention, from their definitions (snowllm_amd/kv8.py). A cache is (k_pool,
v_pool, k_scale, v_scale); row t of request b is row b * T + t."""
import torch

from .sparse import PAGE, block_of

LEAST = 2.0 ** -100
GROUP = 64   # keys whose weights share a factor, or twice as many, in whole groups


def largest_near(wv, group, groups):
    """[groups] the largest of wv in a group or the one before or behind it."""
    most = torch.zeros(groups + 2, dtype=torch.float64).scatter_reduce(0, group + 1, wv, "amax")
    return torch.maximum(torch.maximum(most[:-2], most[1:-1]), most[2:])


def axis_of(i, sections, interleaved):
    """The axis of rotated pair i."""
    n = len(sections)
    if interleaved:
        return i % n if i // n < sections[i % n] else 0
    a = 0
    while i >= sections[a]:
        i -= sections[a]
        a += 1
    return a


def angles(positions, inv_freq, sections, interleaved):
    """[M, half] angles."""
    return torch.stack([positions[axis_of(i, sections, interleaved)].double() * float(f)
                        for i, f in enumerate(inv_freq)], 1)


def quantise(y):
    """(y / scale before its rounding, scale) of rows y [.., d] in 64 bits; NaN scales where a row is
    not finite."""
    fine = y.isfinite().all(-1)
    scale = y.abs().amax(-1).clamp(min=LEAST) / 127.0
    scale = torch.where(fine, scale, torch.full_like(scale, float("nan")))
    return torch.where(fine[..., None], y / scale[..., None], torch.zeros_like(y)), scale


def code_of(cache, blk, off):
    """Codes k, v [Hkv, d] and scales [Hkv] of a slot."""
    k, v, ks, vs = cache
    return (k[blk, :, off // 4, :, off % 4].reshape(k.shape[1], -1), v[blk, :, :, off], ks[blk, :, off],
            vs[blk, :, off])


def rows_of(cache, table, b, n):
    """Codes and scales of request b's first n positions: k, v [n, Hkv, d] int8, ks, vs [n, Hkv] f32,
    and [n] whether the position is in the cache."""
    k, v, ks, vs = cache
    blk = torch.tensor([block_of(table, b, p, k.shape[0]) for p in range((n + PAGE - 1) // PAGE)],
                       dtype=torch.int64)
    at = blk.clamp(min=0)
    hkv, d = v.shape[1], v.shape[2]
    kr = k[at].permute(0, 2, 4, 1, 3, 5).reshape(-1, hkv, d)[:n]
    vr = v[at].permute(0, 3, 1, 2).reshape(-1, hkv, d)[:n]
    return (kr, vr, ks[at].permute(0, 2, 1).reshape(-1, hkv)[:n], vs[at].permute(0, 2, 1).reshape(-1, hkv)[:n],
            (blk >= 0).repeat_interleave(PAGE)[:n])


def seen(start, count, t, n, tree):
    """[n] whether row t of a request sees its positions 0 .. n - 1."""
    p = torch.arange(n)
    if tree is None:
        return p <= start + t
    mask = int(tree)
    own = torch.tensor([0 <= int(x) - start < count and mask >> (int(x) - start) & 1 == 1 for x in p])
    return (p < start) | own


def attention(q, cache, table, starts, counts, scale, T, tree=None):
    """(out, error, live) of every row: out [M, Hq, d] in 64 bits, error [M, Hq, d] how far a kernel
    may be from it before its last rounding (see below), live [M] the rows that are written.

    error counts, with u = 2^-24 and W = sum_k w_k |v_k| of the normalised weights w:
      scores: q as 16-bit integers is off by half of max(max|q|, LEAST) / 32512 an element; the integer products are
        exact, their conversion, the two factors, the maximum's subtraction and the exponential are 8 u
        of the largest score plus 8 u; twice, for the weights and for their sum              -> 2 e W
      weights times v's scale as 16-bit integers of the largest of one or two GROUPs of keys (which two
        follows from where the keys are split): half a unit each, which is at least 2^-127 (2^-126 is the
        least unit) beside a sum of weights of at least 2^-4
      sums of the keys' groups and of splits, in any order: (n / GROUP + 64) u W."""
    u = 2.0 ** -24
    M, Hq, d = q.shape
    hkv = cache[1].shape[1]
    G = Hq // hkv
    out = torch.zeros(M, Hq, d, dtype=torch.float64)
    error = torch.zeros_like(out)
    live = torch.zeros(M, dtype=torch.bool)
    width = table.shape[1]
    for b in range(table.shape[0]):
        start, count = int(starts[b]), min(int(counts[b]), T)
        if start < 0 or count <= 0:
            continue
        n = min(start + count, width * PAGE)
        k, v, ks, vs, there = rows_of(cache, table, b, n)
        for t in range(count):
            m = b * T + t
            live[m] = True
            vis = seen(start, count, t, n, None if tree is None else tree[m]) & there
            if not vis.any():
                continue
            for h in range(hkv):
                kv = k[vis, h].double()
                key = kv * ks[vis, h].double()[:, None]
                val = v[vis, h].double() * vs[vis, h].double()[:, None]
                group = torch.arange(n)[vis] // GROUP
                for e in range(G):
                    x = q[m, h * G + e].double()
                    s = key @ x * scale
                    w = s.softmax(0)
                    o = w @ val
                    off = abs(scale) * x.abs().max().clamp(min=LEAST) / 65024 * key.abs().sum(1).max()
                    off = off + 8 * u * (s.abs().max() + 1)
                    big = w @ val.abs()
                    wv = w * vs[vis, h].double()
                    most = largest_near(wv, group, n // GROUP + 1)
                    out[m, h * G + e] = o
                    unit = most[group] / 65024 + 2.0 ** -123
                    error[m, h * G + e] = (2 * off * big + unit @ v[vis, h].double().abs()
                                           + (n / GROUP + 64) * u * big)
    return out, error, live
