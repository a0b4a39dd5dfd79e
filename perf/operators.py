"""The operators of attention over selected pages of a paged cache, as they are measured: the cache
write that keeps each page's bounds, the bounds of pages that another writer filled, the choice of
pages by their bounds, and the attention over the chosen pages.

A case is a dict of plain values with an "op":

  append   ops.kv_append         K/V rows rotated (and normalised) into the cache, bounds updated
  bounds   ops.page_bounds       element-wise minimum and maximum of a page's keys, from the pool
  select   ops.page_select       the pages each row reads, by an upper bound of its scores
  attend   ops.sparse_attention  softmax attention over the listed pages

`own` false: plain torch; true: the framework's operators. Shapes are those of the dense 8B and the
MoE 35B-A3B configurations of snowllm_amd/verify.py (geometry "dense" and "moe") and a 64-wide head.
"""
import math

import torch

own = False

PAGE = 16
EPS = 1e-6
# heads, kv heads, head size, rotated pairs, RoPE base, QK norm
GEOMETRY = {
    "dense": (32, 8, 128, 64, 1e6, False),
    "moe": (16, 2, 256, 32, 1e7, True),
    "small": (8, 2, 64, 32, 1e4, False),
}
SINK, RECENT = 1, 2   # pages at the start and at the end of the context that every row keeps


def listed():
    return [
        # one user's next token joins the cache of a dense model: the latency of a single launch
        dict(name="append_decode", op="append", geometry="dense", batch=1, tokens=1, context=8191,
             ragged=False),
        # four prompts of about 2048 tokens, normalised and rotated behind a cached prefix of odd
        # length
        dict(name="append_prompt", op="append", geometry="moe", batch=4, tokens=2048, context=1001,
             ragged=True),
        # the pages that sixteen blocks of nine rows touched through the attention's own writer
        dict(name="bounds_verify", op="bounds", geometry="dense", batch=16, tokens=9, context=8190,
             ragged=True),
        # a whole 220K cache that was filled without bounds
        dict(name="bounds_context", op="bounds", geometry="moe", batch=1, tokens=220011, context=0,
             ragged=False),
        # one user's next token at 8K
        dict(name="select_decode", op="select", geometry="moe", batch=1, tokens=1, context=8191,
             ragged=False, budget=64),
        # a verify block of eleven rows at 220K
        dict(name="select_verify", op="select", geometry="moe", batch=1, tokens=11, context=220000,
             ragged=False, budget=128),
        # a serving batch on the dense model, contexts from 16K to 32K
        dict(name="select_batch", op="select", geometry="dense", batch=32, tokens=1, context=32767,
             ragged=True, budget=64),
        # a chunk of a long prompt: every row chooses for itself
        dict(name="select_prompt", op="select", geometry="moe", batch=1, tokens=1024, context=64000,
             ragged=False, budget=64),
        # the attention that reads what the four choices above give
        dict(name="attend_decode", op="attend", geometry="moe", batch=1, tokens=1, context=8191,
             ragged=False, budget=64),
        dict(name="attend_verify", op="attend", geometry="moe", batch=1, tokens=11, context=220000,
             ragged=False, budget=128),
        dict(name="attend_batch", op="attend", geometry="dense", batch=64, tokens=1, context=8191,
             ragged=True, budget=64),
        dict(name="attend_prompt", op="attend", geometry="moe", batch=1, tokens=1024, context=64000,
             ragged=False, budget=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 1e15


def draw(rng):
    op = rng.choice(("append", "bounds", "select", "select", "attend", "attend"))
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        case = dict(op=op, geometry=rng.choice(("dense", "moe", "small")), batch=_log_int(rng, 1, 64),
                    tokens=_log_int(rng, 1, 2048), context=_log_int(rng, 1, 220000) - 1,
                    ragged=rng.random() < 0.5)
        if op == "bounds":
            case["tokens"] = _log_int(rng, 1, 220000)
            case["context"] = _log_int(rng, 1, 8192) - 1
        if op in ("select", "attend"):
            # blocks of a verify step more often than prompts
            if rng.random() < 0.6:
                case["tokens"] = rng.randint(1, 16)
            case["budget"] = _log_int(rng, 4, 256)
        heads, kv_heads, dim = GEOMETRY[case["geometry"]][:3]
        cells = case["batch"] * (case["context"] + case["tokens"])
        gathered = case["batch"] * case["tokens"] * kv_heads * case.get("budget", 0) * dim
        scored = case["batch"] * case["tokens"] * kv_heads * (case["context"] + case["tokens"]) // 16
        if (_cost(case) <= most and cells <= 1100000 and scored <= 20000000
                and (op != "attend" or gathered <= 40000000)):
            return case


# ------------------------------------------------------------------------------------------
# seeded inputs
# ------------------------------------------------------------------------------------------
def _lengths(case):
    """(tokens in the cache before the call, rows of the call) of every request."""
    B, T, ctx = case["batch"], case["tokens"], case["context"]
    if not case["ragged"]:
        return [(ctx, T)] * B
    return [(ctx - ctx * b // (2 * B), max(1, T - T * b // (3 * B))) for b in range(B)]


def _width(case):
    return (case["context"] + case["tokens"] + PAGE - 1) // PAGE


def _gen(seed, part):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1009 + part)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _keys(g, blocks, hkv, dim):
    """A K pool: the tokens of a page vary about a direction that the page has in common."""
    pool = torch.empty(blocks, hkv, dim // 16, PAGE, 16, dtype=torch.bfloat16, device="cuda")
    pool.normal_(0.0, 0.7, generator=g)
    return pool.add_(0.7 * _randn(g, blocks, hkv, dim // 16, 1, 16))


def prepare(case, seed):
    heads, hkv, dim, half, theta, norm = GEOMETRY[case["geometry"]]
    op, B, T, W = case["op"], case["batch"], case["tokens"], _width(case)
    g = _gen(seed, 1)
    lengths = _lengths(case)
    blocks = B * W + 8
    s = dict(op=op, heads=heads, kv_heads=hkv, dim=dim, batch=B, tokens=T)
    s["table"] = torch.randperm(blocks, device="cuda", generator=g)[:B * W].int().view(B, W)
    if op in ("append", "bounds"):
        s["starts"] = _ints([c for c, _ in lengths])
        s["counts"] = _ints([n for _, n in lengths])
        s["k_pool"] = _keys(g, blocks, hkv, dim)
        s["bounds"] = torch.zeros(blocks, hkv, 2, dim, dtype=torch.bfloat16, device="cuda")
        # the pages that get a token, and how many of a page's tokens are live then
        table = s["table"].cpu()
        pages = [(b, p, min(PAGE, c + n - p * PAGE)) for b, (c, n) in enumerate(lengths)
                 for p in range(c // PAGE, (c + n - 1) // PAGE + 1)]
        at = torch.tensor(pages)
        s["page_blocks"] = table[at[:, 0], at[:, 1]].long().cuda()
        s["page_live"] = at[:, 2].cuda()
    if op == "append":
        M = B * T
        proj = _randn(g, M, (heads + 2 * hkv) * dim).bfloat16()   # rows of a fused projection
        s["q"] = proj[:, :heads * dim].unflatten(1, (heads, dim))
        s["k"] = proj[:, heads * dim:(heads + hkv) * dim].unflatten(1, (hkv, dim))
        s["v"] = proj[:, (heads + hkv) * dim:].unflatten(1, (hkv, dim))
        s["v_pool"] = torch.empty(blocks, hkv, PAGE // 4, dim, 4, dtype=torch.bfloat16,
                                  device="cuda").normal_(generator=g)
        s["q_out"] = torch.zeros(M, heads, dim, dtype=torch.bfloat16, device="cuda")
        pos = torch.tensor([c for c, _ in lengths]).view(B, 1) + torch.arange(T).view(1, T)
        freq = theta ** (-torch.arange(half, dtype=torch.float64) / half)
        angle = (pos.view(M, 1).double() * freq).cuda()
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_gamma"] = (1.0 + 0.1 * _randn(g, dim)).bfloat16() if norm else None
        s["k_gamma"] = (1.0 + 0.1 * _randn(g, dim)).bfloat16() if norm else None
        # the live rows and their cache slots
        live = (torch.arange(T).view(1, T) < s["counts"].cpu().view(B, 1)).view(M)
        slots = (table.long().gather(1, (pos // PAGE).clamp(max=W - 1)) * PAGE + pos % PAGE).view(M)
        s["rows"] = live.nonzero().view(-1).cuda()
        s["slots"] = slots[live].cuda()
    if op in ("select", "attend"):
        pos = torch.tensor([[c + t if t < n else -1 for t in range(T)] for c, n in lengths])
        s["positions"] = pos.int().view(-1).cuda()
        s["q"] = (_randn(g, B * T, heads, dim) * (0.5 + _randn(g, dim).abs())).bfloat16()
        s["budget"] = case["budget"]
    if op == "select":
        centre = 0.8 * _randn(g, blocks, hkv, 1, dim)
        reach = 1.2 + 0.3 * _randn(g, blocks, hkv, 2, dim).abs()
        reach[:, :, 0].neg_()
        s["bounds"] = (centre + reach).bfloat16()
        s["pages"] = torch.empty(B * T, hkv, case["budget"], dtype=torch.int32, device="cuda")
    if op == "attend":
        s["scale"] = dim ** -0.5
        s["k_pool"] = _keys(g, blocks, hkv, dim)
        s["v_pool"] = torch.empty(blocks, hkv, PAGE // 4, dim, 4, dtype=torch.bfloat16,
                                  device="cuda").normal_(generator=g)
        s["pages"] = _lists(g, s["positions"].view(B, T), hkv, W, case["budget"])
        s["out"] = torch.empty(B * T, heads, dim, dtype=torch.bfloat16, device="cuda")
    return s


def _lists(g, positions, hkv, width, budget):
    """Page lists as the choice of pages gives them: the first page and the last two, and others of
    which the sixteen rows of a tile have most in common (about 1.5 budgets in all)."""
    B, T = positions.shape
    tiles = (T + 15) // 16
    common = torch.rand(B, tiles, 1, hkv, width, device="cuda", generator=g)
    single = torch.rand(B, T, hkv, width, device="cuda", generator=g)
    key = single * min(1.0, budget / width)
    key += common.expand(-1, -1, 16, -1, -1).reshape(B, tiles * 16, hkv, width)[:, :T]
    page = torch.arange(width, device="cuda")
    n = (positions.long() // PAGE + 1).view(B, T, 1, 1)        # 0 for a padding row
    key = key.masked_fill((page < SINK) | (page >= n - RECENT), 10.0).masked_fill(page >= n, -1.0)
    top, ids = key.topk(min(budget, width), dim=-1)
    ids = ids.masked_fill(top < 0.0, width).sort(dim=-1).values
    ids = ids.masked_fill(ids == width, -1)
    ids = torch.nn.functional.pad(ids, (0, max(0, budget - width)), value=-1)
    return ids.int().view(B * T, hkv, budget).contiguous()


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "bounds": _bounds, "select": _select, "attend": _attend}[state["op"]](state)


def _run_own(s):
    from snowllm_amd import ops

    if s["op"] == "append":
        ops.kv_append(s["k"], s["v"], s["cos"], s["sin"], s["k_pool"], s["v_pool"], s["table"],
                      s["starts"], s["counts"], bounds=s["bounds"], q=s["q"], q_out=s["q_out"],
                      q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS)
        return s["k_pool"], s["v_pool"], s["bounds"], s["q_out"]
    if s["op"] == "bounds":
        ops.page_bounds(s["k_pool"], s["bounds"], s["table"], s["starts"], s["counts"], s["tokens"])
        return s["bounds"]
    if s["op"] == "select":
        if "scratch" not in s:   # a program keeps its workspace
            s["scratch"] = ops.empty_bytes(ops.page_select_scratch_bytes(
                s["batch"], s["tokens"], s["heads"], s["kv_heads"], s["dim"], s["table"].shape[1]))
        ops.page_select(s["q"], s["bounds"], s["table"], s["positions"], s["pages"], s["scratch"],
                        sink=SINK, recent=RECENT)
        return s["pages"]
    if "scratch" not in s:
        s["scratch"] = ops.empty_bytes(ops.sparse_attention_scratch_bytes(
            s["batch"], s["tokens"], s["heads"], s["kv_heads"], s["dim"], s["budget"]))
    ops.sparse_attention(s["q"], s["k_pool"], s["v_pool"], s["out"], s["table"], s["positions"],
                         s["pages"], s["scale"], s["scratch"])
    return s["out"]


def _norm_rotate(x, gamma, cos, sin):
    """x [n, heads, dim] normalised per head (gamma given), its first 2 half elements rotated in
    the pairs (i, i + half), rounded once."""
    x = x.float()
    if gamma is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma.float()
    half = cos.shape[1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    c, d = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * d, b * c + a * d, rest], -1).bfloat16()


def _page_minmax(s):
    """The bounds of the touched pages, over their live tokens, into s["bounds"]."""
    keys = s["k_pool"][s["page_blocks"]].float()               # [pages, hkv, dim/16, 16 tokens, 16]
    dead = (torch.arange(PAGE, device="cuda") >= s["page_live"][:, None]).view(-1, 1, 1, PAGE, 1)
    low = keys.masked_fill(dead, float("inf")).amin(3).flatten(2)
    high = keys.masked_fill(dead, float("-inf")).amax(3).flatten(2)
    s["bounds"][s["page_blocks"]] = torch.stack([low, high], 2).bfloat16()


def _append(s):
    rows, slots = s["rows"], s["slots"]
    cos, sin = s["cos"][rows], s["sin"][rows]
    k = _norm_rotate(s["k"][rows], s["k_gamma"], cos, sin)
    block, off = slots // PAGE, slots % PAGE
    s["k_pool"][block, :, :, off] = k.unflatten(2, (-1, 16))
    s["v_pool"][block, :, off // 4, :, off % 4] = s["v"][rows]
    s["q_out"][rows] = _norm_rotate(s["q"][rows], s["q_gamma"], cos, sin)
    _page_minmax(s)
    return s["k_pool"], s["v_pool"], s["bounds"], s["q_out"]


def _bounds(s):
    _page_minmax(s)
    return s["bounds"]


def _select(s):
    """score = sum over the group's heads and the dims of max(q low, q high), in 64 bits: the choice
    turns on differences between nearly equal scores. Lowest page first among equals."""
    B, T, hkv, D = s["batch"], s["tokens"], s["kv_heads"], s["dim"]
    W = s["table"].shape[1]
    q = s["q"].double().view(B, T, hkv, -1, D)
    up = q.clamp(min=0).sum(3).transpose(1, 2).contiguous()            # [B, hkv, T, D]
    down = q.clamp(max=0).sum(3).transpose(1, 2).contiguous()
    bd = s["bounds"][s["table"].long()].double()                       # [B, W, hkv, 2, D]
    low = bd[:, :, :, 0].permute(0, 2, 3, 1).contiguous()              # [B, hkv, D, W]
    high = bd[:, :, :, 1].permute(0, 2, 3, 1).contiguous()
    score = torch.matmul(up, high) + torch.matmul(down, low)           # [B, hkv, T, W]
    score = score.transpose(1, 2)
    page = torch.arange(W, device="cuda")
    n = torch.div(s["positions"].long(), PAGE, rounding_mode="floor").view(B, T, 1, 1) + 1
    score = score.masked_fill((page < SINK) | (page >= n - RECENT), float("inf"))
    score = score.masked_fill(page >= n, float("-inf"))
    ids = score.sort(dim=-1, descending=True, stable=True).indices[..., :s["budget"]]
    ids = ids.masked_fill(ids >= n, W).sort(dim=-1).values
    ids = torch.nn.functional.pad(ids.masked_fill(ids == W, -1), (0, s["budget"] - ids.shape[-1]),
                                  value=-1)
    s["pages"].copy_(ids.view(B * T, hkv, -1))
    return s["pages"]


def _attend(s):
    B, T, hkv, D, heads = s["batch"], s["tokens"], s["kv_heads"], s["dim"], s["heads"]
    M, G = B * T, heads // hkv
    pages = s["pages"].long()                                          # [M, hkv, K]
    request = torch.arange(B, device="cuda").repeat_interleave(T).view(M, 1, 1)
    block = s["table"][request, pages.clamp(min=0)].long()
    head = torch.arange(hkv, device="cuda").view(1, hkv, 1)
    k = s["k_pool"][block, head]                                       # [M, hkv, K, D/16, 16, 16]
    k = k.transpose(3, 4).reshape(M, hkv, -1, D).float()               # [M, hkv, K * 16, D]
    v = s["v_pool"][block, head].transpose(4, 5).reshape(M, hkv, -1, D).float()
    q = s["q"].float().view(M, hkv, G, D)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    token = pages[..., None] * PAGE + torch.arange(PAGE, device="cuda")
    seen = (pages[..., None] >= 0) & (token <= s["positions"].long().view(M, 1, 1, 1))
    seen = seen.view(M, hkv, 1, -1)
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / total.clamp(min=torch.finfo(torch.float32).tiny)
    s["out"].copy_(out.view(M, heads, D))
    return s["out"]


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    heads, hkv, D, half, _, norm = GEOMETRY[case["geometry"]]
    lengths = _lengths(case)
    rows = sum(n for _, n in lengths)
    touched = sum((c + n - 1) // PAGE - c // PAGE + 1 for c, n in lengths)
    if case["op"] == "append":
        old = sum(c % PAGE for c, _ in lengths)                        # keys read for their bounds
        moved = 2 * rows * (heads + 2 * hkv) * D * 2 + rows * half * 8
        return {"bytes": moved + old * hkv * D * 2 + touched * hkv * 4 * D,
                "flops": rows * (heads + hkv) * (6 * half + (4 * D if norm else 0)) + rows * hkv * 2 * D}
    if case["op"] == "bounds":
        keys = sum(c + n - c // PAGE * PAGE for c, n in lengths)
        return {"bytes": keys * hkv * D * 2 + touched * hkv * 4 * D, "flops": keys * hkv * D * 2}
    last = [(c + n - 1) // PAGE + 1 for c, n in lengths]               # pages a request's rows see
    if case["op"] == "select":
        scores = sum(n * p for (_, n), p in zip(lengths, last)) * hkv
        return {"bytes": sum(last) * hkv * 4 * D + rows * heads * D * 2 + rows * hkv * case["budget"] * 4,
                "flops": scores * 4 * D}
    K = case["budget"]
    union = sum(min(p, K if n == 1 else (n + 15) // 16 * (3 * K // 2)) for (_, n), p in zip(lengths, last))
    pairs = sum(n * min(K, p) for (_, n), p in zip(lengths, last)) * PAGE * heads
    return {"bytes": union * hkv * 64 * D + rows * heads * D * 4 + rows * hkv * K * 4,
            "flops": pairs * 4 * D}


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    rows = case["batch"] * case["tokens"] * GEOMETRY[case["geometry"]][1]
    if case["op"] in ("select", "attend") and rows > 30000:
        return None                                                    # a loop over the rows
    s = prepare(case, seed)
    return {"append": _exact_append, "bounds": _exact_bounds, "select": _exact_select,
            "attend": _exact_attend}[case["op"]](s, _lengths(case))


def _exact_turn(x, gamma, cos, sin):
    x = x.double()
    if gamma is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * gamma.double()
    half = cos.shape[-1]
    z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous())
    z = z * torch.complex(cos.double(), sin.double())[:, None]
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)


def _exact_limits(s, k_pool, lengths):
    bounds = s["bounds"].double().clone()
    for b, (start, count) in enumerate(lengths):
        first = start // PAGE
        blocks = s["table"][b, first:(start + count - 1) // PAGE + 1].long()
        keys = k_pool[blocks].permute(0, 3, 1, 2, 4).flatten(3)        # [pages, 16, hkv, dim]
        live = start + count - first * PAGE
        whole = live // PAGE
        if whole:
            bounds[blocks[:whole], :, 0] = keys[:whole].amin(1)
            bounds[blocks[:whole], :, 1] = keys[:whole].amax(1)
        if live % PAGE:
            bounds[blocks[whole], :, 0] = keys[whole, :live % PAGE].amin(0)
            bounds[blocks[whole], :, 1] = keys[whole, :live % PAGE].amax(0)
    return bounds


def _exact_append(s, lengths):
    T, hkv, D = s["tokens"], s["kv_heads"], s["dim"]
    k_pool, v_pool, q_out = s["k_pool"].double(), s["v_pool"].double(), s["q_out"].double()
    for b, (start, count) in enumerate(lengths):
        rows = slice(b * T, b * T + count)
        cos, sin = s["cos"][rows], s["sin"][rows]
        q_out[rows] = _exact_turn(s["q"][rows], s["q_gamma"], cos, sin)
        pos = torch.arange(start, start + count, device="cuda")
        blk, off = s["table"][b].long()[pos // PAGE], pos % PAGE
        k = _exact_turn(s["k"][rows], s["k_gamma"], cos, sin)
        k_pool[blk, :, :, off] = k.view(count, hkv, D // 16, 16)
        v_pool[blk, :, off // 4, :, off % 4] = s["v"][rows].double()
    return k_pool, v_pool, _exact_limits(s, k_pool, lengths), q_out


def _exact_bounds(s, lengths):
    return _exact_limits(s, s["k_pool"].double(), lengths)


def _exact_select(s, lengths):
    T, hkv, D, K = s["tokens"], s["kv_heads"], s["dim"], s["budget"]
    pages = torch.full_like(s["pages"], -1)
    for b, (start, count) in enumerate(lengths):
        seen = (start + count - 1) // PAGE + 1
        for h in range(hkv):
            box = s["bounds"][s["table"][b, :seen].long(), h].double()  # [seen, 2, dim]
            for t in range(count):
                n = (start + t) // PAGE + 1
                if n <= K:
                    pages[b * T + t, h, :n] = torch.arange(n, device="cuda", dtype=torch.int32)
                    continue
                q = s["q"][b * T + t].view(hkv, -1, 1, D)[h].double()   # [group, 1, dim]
                middle = box[SINK:n - RECENT]
                score = torch.maximum(q * middle[:, 0], q * middle[:, 1]).sum((0, 2))
                best = (-score).argsort(stable=True)[:K - SINK - RECENT] + SINK
                keep = torch.cat([torch.arange(SINK, device="cuda"), best.sort().values,
                                  torch.arange(n - RECENT, n, device="cuda")])
                pages[b * T + t, h] = keep.int()
    return pages


def _exact_attend(s, lengths):
    T, hkv, D, heads = s["tokens"], s["kv_heads"], s["dim"], s["heads"]
    out = torch.zeros(s["batch"] * T, heads, D, dtype=torch.float64, device="cuda")
    at = torch.arange(PAGE, device="cuda")
    for b, (start, count) in enumerate(lengths):
        for h in range(hkv):
            for t in range(count):
                m = b * T + t
                ids = s["pages"][m, h].long()
                blk = s["table"][b].long()[ids.clamp(min=0)]
                keys = s["k_pool"][blk, h].double().permute(0, 2, 1, 3).reshape(-1, D)
                vals = s["v_pool"][blk, h].double().permute(0, 1, 3, 2).reshape(-1, D)
                token = (ids[:, None] * PAGE + at).view(-1)
                hidden = (token < 0) | (token > start + t)
                q = s["q"][m].view(hkv, -1, D)[h].double()
                weight = (q @ keys.t() * s["scale"]).masked_fill(hidden, float("-inf")).softmax(-1)
                out[m].view(hkv, -1, D)[h] = weight @ vals
    return out
