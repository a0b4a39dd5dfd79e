"""The operators of a paged KV cache in 8 bits, as they are measured: the angles of tokens with several
position axes, the cache write that quantises, the cache read back, and the attention of verify
blocks, single tokens and prompts over it.

A case is a dict of plain values with an "op":

  angles   ops.rope_axes       cos and sin of positions with three axes (time, height, width)
  append   ops.kv8_append      K/V rows normalised, rotated and quantised into the cache, and read
                               back with ops.kv8_read (what is held in 8 bits as the values it is)
  read     ops.kv8_read        cached rows back in bf16
  attend   ops.kv8_attention   softmax attention of new rows over the cache, causal or a tree

`own` false: plain torch; true: the framework's operators. Shapes are those of the dense 8B and the
MoE 35B-A3B configurations of snowllm_amd/verify.py (geometry "dense" and "moe") and a 64-wide head.

The cache: codes int8, one float32 scale per (token, kv head), K [blocks, Hkv, 4, d/16, 4, 16] (token
t of a page is group t / 4, place t % 4), V [blocks, Hkv, d, 16], scales [blocks, Hkv, 16]. A value
is code * scale, scale = max(largest magnitude of the head's row, 2^-100) / 127.
"""
import math
import random

import torch

own = False

PAGE = 16
EPS = 1e-6
LEAST = 2.0 ** -100
# heads, kv heads, head size, rotated pairs, RoPE base, QK norm
GEOMETRY = {
    "dense": (32, 8, 128, 64, 1e6, False),
    "moe": (16, 2, 256, 32, 1e7, True),
    "small": (8, 2, 64, 32, 1e4, False),
}


def listed():
    return [
        # the rows of one verify block behind a 220K context: a launch's latency
        dict(name="angles_verify", op="angles", geometry="moe", batch=1, tokens=11, context=220000,
             interleaved=True),
        # prompts of images and text, 32 of about 8192 tokens
        dict(name="angles_prompt", op="angles", geometry="moe", batch=32, tokens=8192, context=0,
             interleaved=False),
        # a serving batch's next tokens join the cache of a dense model
        dict(name="append_decode", op="append", geometry="dense", batch=64, tokens=1, context=8191,
             ragged=True),
        # four prompts of about 2048 tokens behind a cached prefix of odd length
        dict(name="append_prompt", op="append", geometry="moe", batch=4, tokens=2048, context=1001,
             ragged=True),
        # the odd end of a prefix that moves to another cache
        dict(name="read_prefix", op="read", geometry="dense", batch=1, tokens=333, context=777,
             ragged=False),
        # a whole long context, for an attention that takes bf16
        dict(name="read_context", op="read", geometry="moe", batch=1, tokens=131071, context=0,
             ragged=False),
        # one user's next token at 8K: latency
        dict(name="attend_decode", op="attend", geometry="moe", batch=1, tokens=1, context=8191,
             ragged=False, tree=False),
        # a verify block of nine rows on the dense model at 8K
        dict(name="attend_verify", op="attend", geometry="dense", batch=1, tokens=9, context=8192,
             ragged=False, tree=False),
        # a tree of eleven drafted rows behind 220K tokens
        dict(name="attend_tree", op="attend", geometry="moe", batch=1, tokens=11, context=220000,
             ragged=False, tree=True),
        # a serving batch of single tokens, contexts from 4K to 8K
        dict(name="attend_batch", op="attend", geometry="dense", batch=64, tokens=1, context=8191,
             ragged=True, tree=False),
        # verify blocks of sixteen requests of odd lengths
        dict(name="attend_blocks", op="attend", geometry="moe", batch=16, tokens=9, context=8187,
             ragged=True, tree=False),
        # a chunk of a long prompt: matrix work
        dict(name="attend_prompt", op="attend", geometry="moe", batch=1, tokens=1024, context=16001,
             ragged=False, tree=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 1e15


def draw(rng):
    op = rng.choice(("angles", "append", "read", "attend", "attend", "attend"))
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        case = dict(op=op, geometry=rng.choice(("dense", "moe", "small")), batch=_log_int(rng, 1, 64),
                    tokens=_log_int(rng, 1, 8192), context=_log_int(rng, 1, 220000) - 1)
        if op == "angles":
            case["interleaved"] = rng.random() < 0.5
        else:
            case["ragged"] = rng.random() < 0.5
        if op == "attend":
            # blocks of a verify step more often than prompts
            case["tokens"] = rng.randint(1, 16) if rng.random() < 0.6 else _log_int(rng, 1, 2048)
            case["tree"] = case["tokens"] <= 64 and rng.random() < 0.3
        heads, kv_heads, dim = GEOMETRY[case["geometry"]][:3]
        cells = case["batch"] * (case["context"] + case["tokens"]) * kv_heads * dim
        scores = case["batch"] * heads * case["tokens"] * (case["context"] + case["tokens"])
        if (_cost(case) <= most and (op == "angles" or cells <= 560000000)
                and (op != "attend" or scores <= 400000000)):
            return case


# ------------------------------------------------------------------------------------------
# seeded inputs
# ------------------------------------------------------------------------------------------
def _lengths(case):
    """(tokens in the cache before the call's rows, rows of the call) of every request."""
    B, T, ctx = case["batch"], case["tokens"], case["context"]
    if not case.get("ragged"):
        return [(ctx, T)] * B
    return [(ctx - ctx * b // (2 * B), max(1, T - T * b // (3 * B))) for b in range(B)]


def _width(case):
    return (case["context"] + case["tokens"] + PAGE - 1) // PAGE


def _sections(half):
    """Rotated pairs of the three axes: about 3 : 4 : 4, as 24, 20 and 20 of 64 or 12, 10, 10 of 32."""
    side = half * 10 // 32
    return half - 2 * side, side, side


def _gen(seed, part):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1009 + part)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _codes(g, *shape):
    """Codes of quantised rows: about normal, the largest near 127."""
    x = torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, 42.0, generator=g)
    return x.round_().clamp_(-127, 127).to(torch.int8)


def _cache(g, blocks, hkv, dim):
    k = _codes(g, blocks, hkv, 4, dim // 16, 4, 16)
    v = _codes(g, blocks, hkv, dim, PAGE)
    k_scale = (0.35 * _randn(g, blocks, hkv, PAGE)).exp_().mul_(0.024)
    v_scale = (0.5 * _randn(g, blocks, hkv, PAGE)).exp_().mul_(0.020)
    return k, v, k_scale, v_scale


def _tree(tokens, seed):
    """Ancestor masks of a random tree of drafted rows, as int64 bit patterns."""
    rng = random.Random(seed)
    masks = []
    for t in range(tokens):
        masks.append(1 << t | (masks[rng.randrange(max(0, t - 6), t)] if t else 0))
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def prepare(case, seed):
    heads, hkv, dim, half, theta, norm = GEOMETRY[case["geometry"]]
    op, B, T, W = case["op"], case["batch"], case["tokens"], _width(case)
    g = _gen(seed, 1)
    M = B * T
    freq = theta ** (-torch.arange(half, dtype=torch.float64) / half)
    s = dict(op=op, heads=heads, kv_heads=hkv, dim=dim, batch=B, tokens=T)
    if op == "angles":
        # a run of text, then pictures: time stands still over one while height and width run
        text = torch.arange(M, device="cuda") + case["context"]
        side = torch.randint(4, 64, (1,), device="cuda", generator=g)
        grid = torch.arange(M, device="cuda")
        picture = _randn(g, M // 256 + 1).repeat_interleave(256)[:M] > 0
        start = text - grid % 256
        s["positions"] = torch.stack([
            torch.where(picture, start, text),
            torch.where(picture, start + grid % 256 // side, text),
            torch.where(picture, start + grid % 256 % side, text)]).contiguous()
        s["inv_freq"] = freq.float().cuda()
        s["sections"], s["interleaved"] = _sections(half), case["interleaved"]
        s["cos"] = torch.empty(M, half, device="cuda")
        s["sin"] = torch.empty(M, half, device="cuda")
        return s
    lengths = _lengths(case)
    blocks = B * W + 8
    table = torch.randperm(blocks, device="cuda", generator=g)[:B * W].int().view(B, W)
    s["table"] = table
    s["cache"] = _cache(g, blocks, hkv, dim)
    s["starts"], s["counts"] = _ints([c for c, _ in lengths]), _ints([n for _, n in lengths])
    pos = s["starts"].long().view(B, 1) + torch.arange(T, device="cuda").view(1, T)
    live = torch.arange(T, device="cuda").view(1, T) < s["counts"].view(B, 1)
    if op in ("append", "read"):
        # the live rows and their cache slots
        slots = table.long().gather(1, (pos // PAGE).clamp(max=W - 1)) * PAGE + pos % PAGE
        s["rows"], s["slots"] = live.view(M).nonzero().view(-1), slots[live]
        s["k_out"] = torch.zeros(M, hkv, dim, dtype=torch.bfloat16, device="cuda")
        s["v_out"] = torch.zeros(M, hkv, dim, dtype=torch.bfloat16, device="cuda")
    if op == "append":
        proj = _randn(g, M, (heads + 2 * hkv) * dim)
        proj = (proj * (0.3 * _randn(g, M, 1)).exp_()).bfloat16()     # rows of a fused projection
        s["q"] = proj[:, :heads * dim].unflatten(1, (heads, dim))
        s["k"] = proj[:, heads * dim:(heads + hkv) * dim].unflatten(1, (hkv, dim))
        s["v"] = proj[:, (heads + hkv) * dim:].unflatten(1, (hkv, dim))
        angle = pos.view(M, 1).double() * freq.cuda()
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_out"] = torch.zeros(M, heads, dim, dtype=torch.bfloat16, device="cuda")
        s["q_gamma"] = (1.0 + 0.1 * _randn(g, dim)).bfloat16() if norm else None
        s["k_gamma"] = (1.0 + 0.1 * _randn(g, dim)).bfloat16() if norm else None
    if op == "attend":
        s["q"] = (_randn(g, M, heads, dim) * (0.5 + _randn(g, dim).abs())).bfloat16()
        s["scale"] = dim ** -0.5
        s["out"] = torch.zeros(M, heads, dim, dtype=torch.bfloat16, device="cuda")
        s["tree"] = _ints(_tree(T, seed) * B, torch.int64) if case["tree"] else None
    return s


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    return {"angles": _angles, "append": _append, "read": _read, "attend": _attend}[state["op"]](state)


def _run_own(s):
    from snowllm_amd import ops

    if s["op"] == "angles":
        ops.rope_axes(s["positions"], s["inv_freq"], s["cos"], s["sin"], s["sections"],
                      interleaved=s["interleaved"])
        return s["cos"], s["sin"]
    if s["op"] == "append":
        ops.kv8_append(s["k"], s["v"], s["cos"], s["sin"], s["cache"], s["table"], s["starts"],
                       s["counts"], q=s["q"], q_out=s["q_out"], q_gamma=s["q_gamma"],
                       k_gamma=s["k_gamma"], eps=EPS)
    if s["op"] in ("append", "read"):
        ops.kv8_read(s["cache"], s["table"], s["starts"], s["counts"], s["k_out"], s["v_out"])
        if s["op"] == "read":
            return s["k_out"], s["v_out"]
        return s["k_out"], s["v_out"], s["cache"][2], s["cache"][3], s["q_out"]
    if "scratch" not in s:   # a program keeps its workspace
        s["scratch"] = ops.empty_bytes(ops.kv8_attention_scratch_bytes(
            s["batch"], s["tokens"], s["heads"], s["kv_heads"], s["dim"], s["table"].shape[1]))
    ops.kv8_attention(s["q"], s["cache"], s["out"], s["table"], s["starts"], s["counts"], s["scale"],
                      s["scratch"], tree=s["tree"])
    return s["out"]


def _axis_of(half, sections, interleaved):
    """The axis of every rotated pair: sections one behind the other, or the pairs in turn (pair i
    belongs to axis i % axes as long as that axis has pairs left, to the first axis else)."""
    n = len(sections)
    if not interleaved:
        return [a for a in range(n) for _ in range(sections[a])]
    return [i % n if i < n * sections[i % n] else 0 for i in range(half)]


def _angles(s):
    axis = torch.tensor(_axis_of(s["inv_freq"].numel(), s["sections"], s["interleaved"]), device="cuda")
    angle = s["positions"].double()[axis].t() * s["inv_freq"].double()       # far positions: 64 bits
    s["cos"].copy_(angle.cos())
    s["sin"].copy_(angle.sin())
    return s["cos"], s["sin"]


def _norm_rotate(x, gamma, cos, sin):
    """x [n, heads, dim] normalised per head (gamma given), its first 2 half elements rotated in
    the pairs (i, i + half), in 32 bits."""
    x = x.float()
    if gamma is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma.float()
    half = cos.shape[1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    c, d = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * d, b * c + a * d, rest], -1)


def _quantise(x):
    scale = x.abs().amax(-1).clamp(min=LEAST) / 127.0
    return (x / scale[..., None]).round().to(torch.int8), scale


def _append(s):
    rows, block, off = s["rows"], s["slots"] // PAGE, s["slots"] % PAGE
    k_pool, v_pool, k_scale, v_scale = s["cache"]
    cos, sin = s["cos"][rows], s["sin"][rows]
    code, scale = _quantise(_norm_rotate(s["k"][rows], s["k_gamma"], cos, sin))
    k_pool[block, :, off // 4, :, off % 4] = code.unflatten(2, (-1, 16))
    k_scale[block, :, off] = scale
    code, scale = _quantise(s["v"][rows].float())
    v_pool[block, :, :, off] = code
    v_scale[block, :, off] = scale
    s["q_out"][rows] = _norm_rotate(s["q"][rows], s["q_gamma"], cos, sin).bfloat16()
    return (*_read(s), k_scale, v_scale, s["q_out"])


def _read(s):
    rows, block, off = s["rows"], s["slots"] // PAGE, s["slots"] % PAGE
    k_pool, v_pool, k_scale, v_scale = s["cache"]
    k = k_pool[block, :, off // 4, :, off % 4].flatten(2).float() * k_scale[block, :, off][..., None]
    v = v_pool[block, :, :, off].float() * v_scale[block, :, off][..., None]
    s["k_out"][rows] = k.bfloat16()
    s["v_out"][rows] = v.bfloat16()
    return s["k_out"], s["v_out"]


def _attend(s):
    B, T, hkv, D, heads = s["batch"], s["tokens"], s["kv_heads"], s["dim"], s["heads"]
    k_pool, v_pool, k_scale, v_scale = s["cache"]
    table = s["table"].long()
    L = table.shape[1] * PAGE
    k = k_pool[table].permute(0, 2, 4, 6, 1, 3, 5).reshape(B, hkv, -1, 16, L)   # [.., d/16, 16, tokens]
    k = k.flatten(2, 3).float() * k_scale[table].transpose(1, 2).reshape(B, hkv, 1, L)
    q = s["q"].float().view(B, T, hkv, -1, D).transpose(1, 2).reshape(B, hkv, -1, D)
    score = (torch.matmul(q, k) * s["scale"]).view(B, hkv, T, -1, L)
    del k
    token = torch.arange(L, device="cuda")
    start = s["starts"].long().view(B, 1, 1)
    row = torch.arange(T, device="cuda").view(1, T, 1)
    if s["tree"] is None:
        seen = token <= start + row
    else:
        place = token - start                                                   # within the block
        mask = s["tree"].view(B, T, 1) >> place.clamp(0, 63) & 1
        seen = (place < 0) | (mask.bool() & (place < T))
    score = score.masked_fill(~seen.view(B, 1, T, 1, L), float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    del score
    total = p.sum(-1, keepdim=True)
    v = v_pool[table].permute(0, 2, 1, 4, 3).reshape(B, hkv, L, D).float()
    v = v * v_scale[table].transpose(1, 2).reshape(B, hkv, L, 1)
    out = torch.matmul(p.view(B, hkv, -1, L), v).view(B, hkv, T, -1, D)
    out = out / total.clamp(min=torch.finfo(torch.float32).tiny)
    out = out.transpose(1, 2).reshape(B, T, heads, D)
    live = (row < s["counts"].view(B, 1, 1)).view(B, T, 1, 1)
    s["out"].copy_(torch.where(live, out, s["out"].view(B, T, heads, D)).view(B * T, heads, D))
    return s["out"]


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    heads, hkv, D, half, _, norm = GEOMETRY[case["geometry"]]
    if case["op"] == "angles":
        M = case["batch"] * case["tokens"]
        return {"bytes": M * 24 + half * 4 + M * half * 8, "flops": M * half * 20}
    lengths = _lengths(case)
    rows = sum(n for _, n in lengths)
    code = hkv * (2 * D + 8)                                     # a token's codes and scales
    if case["op"] == "read":
        return {"bytes": rows * (code + hkv * D * 4), "flops": rows * hkv * D * 2}
    if case["op"] == "append":
        moved = rows * ((2 * heads + 2 * hkv) * D * 2 + half * 8)
        return {"bytes": moved + rows * (2 * code + hkv * D * 4),
                "flops": rows * (heads + hkv) * (6 * half + (4 * D if norm else 0)) + rows * hkv * D * 8}
    keys = sum(c + n for c, n in lengths)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in lengths) * heads
    return {"bytes": keys * code + rows * heads * D * 4, "flops": pairs * 4 * D}


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "angles":
        return _exact_angles(s)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[case["op"]](
        s, _lengths(case))


def _exact_angles(s):
    pos, freq = s["positions"].cpu().double(), s["inv_freq"].cpu().double()
    half, n = freq.numel(), len(s["sections"])
    last = [sum(s["sections"][:a + 1]) for a in range(n)]
    turn = torch.empty(pos.shape[1], half, dtype=torch.float64)
    for i in range(half):
        if s["interleaved"]:
            axis = i % n if i // n < s["sections"][i % n] else 0
        else:
            axis = next(a for a in range(n) if i < last[a])
        turn[:, i] = pos[axis] * freq[i]
    return turn.cos(), turn.sin()


def _exact_turn(x, gamma, cos, sin):
    x = x.double()
    if gamma is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * gamma.double()
    half = cos.shape[-1]
    z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous())
    z = z * torch.complex(cos.double(), sin.double())[:, None]
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)


def _exact_code(x):
    scale = torch.maximum(x.abs().amax(-1), torch.tensor(LEAST, dtype=torch.float64, device="cuda")) / 127
    return torch.round(x / scale[..., None]) * scale[..., None], scale


def _exact_append(s, lengths):
    T, hkv, D = s["tokens"], s["kv_heads"], s["dim"]
    k_out, v_out, q_out = s["k_out"].double(), s["v_out"].double(), s["q_out"].double()
    k_scale, v_scale = s["cache"][2].double(), s["cache"][3].double()
    for b, (start, count) in enumerate(lengths):
        rows = slice(b * T, b * T + count)
        cos, sin = s["cos"][rows], s["sin"][rows]
        q_out[rows] = _exact_turn(s["q"][rows], s["q_gamma"], cos, sin)
        pos = torch.arange(start, start + count, device="cuda")
        blk, off = s["table"][b].long()[pos // PAGE], pos % PAGE
        k_out[rows], k_scale[blk, :, off] = _exact_code(_exact_turn(s["k"][rows], s["k_gamma"], cos, sin))
        v_out[rows], v_scale[blk, :, off] = _exact_code(s["v"][rows].double())
    return k_out, v_out, k_scale, v_scale, q_out


def _exact_rows(s, b, first, count):
    """K and V [count, hkv, dim] of a request's cached tokens, in 64 bits."""
    hkv, D = s["kv_heads"], s["dim"]
    k_pool, v_pool, k_scale, v_scale = s["cache"]
    p0, p1 = first // PAGE, (first + count - 1) // PAGE + 1
    blk = s["table"][b, p0:p1].long()
    at = slice(first - p0 * PAGE, first - p0 * PAGE + count)
    k = k_pool[blk].permute(0, 2, 4, 1, 3, 5).reshape(-1, hkv, D)[at].double()
    v = v_pool[blk].permute(0, 3, 1, 2).reshape(-1, hkv, D)[at].double()
    ks = k_scale[blk].permute(0, 2, 1).reshape(-1, hkv)[at].double()
    vs = v_scale[blk].permute(0, 2, 1).reshape(-1, hkv)[at].double()
    return k * ks[..., None], v * vs[..., None]


def _exact_read(s, lengths):
    T = s["tokens"]
    k_out, v_out = s["k_out"].double(), s["v_out"].double()
    for b, (start, count) in enumerate(lengths):
        k_out[b * T:b * T + count], v_out[b * T:b * T + count] = _exact_rows(s, b, start, count)
    return k_out, v_out


def _exact_attend(s, lengths):
    T, hkv, D, heads = s["tokens"], s["kv_heads"], s["dim"], s["heads"]
    out = s["out"].double()
    tree = None if s["tree"] is None else s["tree"].view(-1, T).tolist()
    for b, (start, count) in enumerate(lengths):
        k, v = _exact_rows(s, b, 0, start + count)
        block = torch.ones(count, count).tril()
        if tree is not None:
            block = torch.tensor([[tree[b][t] >> j & 1 for j in range(count)] for t in range(count)])
        hidden = torch.cat([torch.zeros(count, start), 1.0 - block], 1).bool().cuda()
        for h in range(hkv):
            q = s["q"][b * T:b * T + count].view(count, hkv, -1, D)[:, h].double()
            for e in range(heads // hkv):
                score = (q[:, e] @ k[:, h].t() * s["scale"]).masked_fill(hidden, float("-inf"))
                out[b * T:b * T + count].view(count, hkv, -1, D)[:, h, e] = score.softmax(-1) @ v[:, h]
    return out
