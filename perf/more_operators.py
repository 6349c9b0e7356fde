"""Normalized and rotated heads, a paged key/value cache in 4 bits and the attention that reads it: the workloads by
which their speed is followed.

Each case is one pass of one operator, as a program that uses the library calls it (device tensors in, device tensors
out, no host synchronisation):

  heads      x [T, heads, width] of queries (and of keys beside them): y = rotation(weight * x / rms(x)), the norm over
             the first `norm` values of a head and the rotation of `dims` values by the token's position
  heads_bwd  the gradients of that: of x, and of the weights that all heads and tokens share
  append     the new tokens' keys (normalized and rotated on the way) and values, rounded to E2M1 codes with one E8M0
             scale per 32 values, into their slots of a paged cache; returned as the BF16 values that they stand for
  attend     softmax(scale q K^T) V of each sequence's new tokens over its pages, causal, with a window and with sinks
             where the case has them, and the logarithm of each row's sum

With own = False the same results come from elementary torch operations in 32 bits (in 64 the mean square of a norm,
whose rounding decides codes).
"""

import ctypes as C
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# heads: query heads, key heads beside them in the same call, width, norm, weights, rotated dims (the last ones), pairing
HEADS = {
    "wq_b": (64, 0, 512, 512, False, 64, "pairs"),     # the 64 x 512 queries of the block-32 projections
    "q_b": (128, 0, 192, 0, False, 64, "pairs"),       # the 128 x (128 + 64) queries of the block-128 projections
    "gqa": (32, 8, 128, 128, True, 128, "halves"),     # grouped queries with their keys, norms of each
    "gqa64": (14, 2, 64, 64, True, 32, "halves"),
}
# caches: query heads, key heads, key width, value width, values apart from the keys, norm of a key, rotated dims,
# pairing, scale of the logits, and the columns [first, of) of the projection's output that the keys are
CACHES = {
    "wkv": (64, 1, 512, 512, False, 512, 64, "pairs", 512 ** -0.5, (0, 512)),
    "kv_a": (128, 1, 576, 512, False, 512, 64, "pairs", 192 ** -0.5, (1536, 2112)),   # stacked behind q_a
    "kv_a16": (16, 1, 576, 512, False, 512, 64, "pairs", 192 ** -0.5, (0, 576)),      # one of eight devices' heads
    "gqa": (32, 8, 128, 128, True, 128, 128, "halves", 128 ** -0.5, (0, 1024)),
    "gqa64": (14, 2, 64, 64, True, 0, 64, "halves", 0.125, (0, 128)),
}
EPS = 1e-6


def listed():
    return [
        # the next token of one session: its 64 query heads
        {"name": "heads-1", "kind": "heads", "heads": "wq_b", "tokens": 1, "type": "bf16"},
        # a prompt's queries and keys, norms with weights
        {"name": "heads-4096", "kind": "heads", "heads": "gqa", "tokens": 4096, "type": "bf16"},
        # a short sequence in training, FP32 activations
        {"name": "heads-bwd-333", "kind": "heads_bwd", "heads": "gqa64", "tokens": 333, "type": "f32"},
        # a training batch
        {"name": "heads-bwd-4096", "kind": "heads_bwd", "heads": "gqa", "tokens": 4096, "type": "bf16"},
        # a decode batch's latents
        {"name": "append-16", "kind": "append", "cache": "wkv", "tokens": 16, "page": 64, "type": "bf16"},
        # a long prompt's latents, a column range of a stacked projection output
        {"name": "append-4096", "kind": "append", "cache": "kv_a", "tokens": 4096, "page": 64, "type": "bf16"},
        # the next token of one session over a few thousand
        {"name": "attend-1", "kind": "attend", "cache": "wkv", "batch": 1, "new": 1, "shortest": 4099,
         "longest": 4099, "page": 64, "window": 0, "sinks": True},
        # a decode batch of sessions of all lengths over shared latents
        {"name": "attend-48", "kind": "attend", "cache": "wkv", "batch": 48, "new": 1, "shortest": 200,
         "longest": 30000, "page": 64, "window": 0, "sinks": True},
        # four drafted tokens a session, 128 heads
        {"name": "attend-drafts-12", "kind": "attend", "cache": "kv_a", "batch": 12, "new": 4, "shortest": 1000,
         "longest": 9001, "page": 32, "window": 0, "sinks": False},
        # a decode batch of grouped queries
        {"name": "attend-gqa-64", "kind": "attend", "cache": "gqa", "batch": 64, "new": 1, "shortest": 500,
         "longest": 16000, "page": 16, "window": 0, "sinks": False},
        # two prompts' last pieces behind what the cache holds of them
        {"name": "attend-prompt-gqa", "kind": "attend", "cache": "gqa", "batch": 2, "new": 2048, "shortest": 4500,
         "longest": 8192, "page": 64, "window": 0, "sinks": False},
        # prompts in a layer whose attention sees the last 128 tokens
        {"name": "attend-window", "kind": "attend", "cache": "wkv", "batch": 3, "new": 700, "shortest": 900,
         "longest": 5000, "page": 128, "window": 128, "sinks": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["heads", "heads_bwd", "append", "attend", "attend", "attend"])
    if kind in ("heads", "heads_bwd"):
        return {"kind": kind, "heads": rng.choice(sorted(HEADS)), "tokens": _log_int(rng, 1, 4096 if kind == "heads" else 2048),
                "type": rng.choice(["bf16", "f32"])}
    cache, page = rng.choice(sorted(CACHES)), rng.choice([16, 32, 64, 128, 256])
    if kind == "append":
        return {"kind": kind, "cache": cache, "tokens": _log_int(rng, 1, 4096), "page": page,
                "type": rng.choice(["bf16", "f32"])}
    heads, _, keys, values = CACHES[cache][:4]
    form = rng.choice(["token", "token", "drafts", "prompt"])
    new = 1 if form == "token" else rng.randint(2, 8) if form == "drafts" else _log_int(rng, 9, 1500)
    window = rng.choice([0, 0, 0, 128, 1000])
    batch = _log_int(rng, 1, 4 if form == "prompt" else 96)
    # at most half the work of the listed prompts, and plain scores of at most 2 GB
    most = min(16000, int(7e10 / (batch * new * heads * (keys + values))), int(5e8 / (batch * new * heads)))
    longest = _log_int(rng, 1, max(most, 1))
    return {"kind": kind, "cache": cache, "batch": batch, "new": new, "shortest": rng.randint(1, longest),
            "longest": longest, "page": page, "window": window, "sinks": rng.random() < 0.5}


# -- seeded inputs -------------------------------------------------------------------------------------

def _gen(seed, *tag):
    g = torch.Generator(device=DEVICE)
    value = seed & 0xFFFFFFFF
    for t in tag:
        value = (value * 1000003 + t + 1) & 0x7FFFFFFFFFFF
    g.manual_seed(value)
    return g


def _normal(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)


def _table(positions, dims):
    """FP32 [positions, dims]: the cosines of a position's dims / 2 angles, then their sines."""
    angle = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * torch.exp(
        torch.arange(0, dims, 2, dtype=torch.float64, device=DEVICE) * (-math.log(10000.0) / dims))
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def _lengths(case):
    """Lengths from the shortest to the longest, evenly in their logarithm, in a shuffled order."""
    b, lo, hi = case["batch"], case["shortest"], case["longest"]
    n = [int(round(lo * (hi / lo) ** (i / (b - 1)))) for i in range(b)] if b > 1 else [hi]
    return np.array(n, np.int64)[np.random.RandomState(b).permutation(b)]


def _news(case):
    """New tokens of each sequence: `new` for single tokens and drafts, ragged for prompts, no more than its length."""
    b, new = case["batch"], case["new"]
    n = np.full(b, new, np.int64)
    if new > 8:
        n -= np.arange(b, dtype=np.int64)[::-1] * (new // (3 * b))
        n = np.minimum(n, _lengths(case))
    return n


def _spans(case):
    """(sum of the cached tokens that some query sees, sum over queries of the tokens that each sees)."""
    span = pairs = 0
    for length, n in zip(_lengths(case).tolist(), _news(case).tolist()):
        w = case["window"] or length + n
        seen = np.clip(length - n + 1 + np.arange(n), 0, None)
        pairs += int(np.minimum(seen, w).sum())
        span += min(length, w + n - 1)
    return span, pairs


def _heads_inputs(s, case, seed):
    s.kind, s.t, s.type = case["kind"], case["tokens"], TYPES[case["type"]]
    hq, hk, s.width, s.norm, weights, s.dims, s.style = HEADS[case["heads"]]
    s.first = s.width - s.dims
    s.heads = [hq, hk] if hk else [hq]
    # queries and keys are column ranges of one projection output
    total = sum(s.heads) * s.width
    s.rows = _normal(_gen(seed, 1), s.t, total, dtype=s.type)
    s.positions = torch.randint(0, 8192, (s.t,), generator=_gen(seed, 2), device=DEVICE, dtype=torch.int32)
    s.table = _table(8192, s.dims)
    s.weights = [torch.rand(s.norm, generator=_gen(seed, 3, i), device=DEVICE) + 0.5 if weights else None
                 for i in range(len(s.heads))]
    if s.kind == "heads_bwd":
        s.dy = [_normal(_gen(seed, 4, i), s.t, h, s.width, dtype=s.type) for i, h in enumerate(s.heads)]


def _append_inputs(s, case, seed):
    s.kind, s.t, s.type, s.page = "append", case["tokens"], TYPES[case["type"]], case["page"]
    _, s.heads, s.width, s.vwidth, s.apart, s.norm, s.dims, s.style, _, (s.column, s.stride) = CACHES[case["cache"]]
    s.first = s.width - s.dims
    s.rows = _normal(_gen(seed, 1), s.t, s.stride, dtype=s.type, scale=2.0)
    s.values = _normal(_gen(seed, 5), s.t, s.heads, s.vwidth, dtype=s.type) if s.apart else None
    s.positions = torch.randint(0, 8192, (s.t,), generator=_gen(seed, 2), device=DEVICE, dtype=torch.int32)
    s.table = _table(8192, s.dims)
    s.weight = torch.rand(s.norm, generator=_gen(seed, 3), device=DEVICE) + 0.5 if s.norm else None
    # the tokens' slots: whole pages in any order for a prompt, slots of pages of their own for a decode batch
    s.pages = -(-s.t // s.page) + s.t // 8 + 1 if s.t > 64 else s.t + 1
    order = torch.randperm(s.pages, generator=_gen(seed, 6), device=DEVICE)
    i = torch.arange(s.t, device=DEVICE)
    s.slots = (order[i // s.page] * s.page + i % s.page if s.t > 64 else order[i] * s.page + (i * 7) % s.page).contiguous()


def _attend_inputs(s, case, seed):
    s.kind, s.page, s.window, s.b = "attend", case["page"], case["window"], case["batch"]
    s.hq, s.heads, s.width, s.vwidth, s.apart, _, _, _, s.scale, _ = CACHES[case["cache"]]
    lengths, news = _lengths(case), _news(case)
    s.t, s.most_new, s.most = int(news.sum()), int(news.max()), int(lengths.max())
    s.lengths = torch.from_numpy(lengths.astype(np.int32)).to(DEVICE)
    s.q_first = torch.from_numpy(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)).to(DEVICE)
    s.uniform = bool((news == news[0]).all())
    s.q = _normal(_gen(seed, 1), s.t, s.hq, s.width, scale=2.0 if s.width <= 128 else 1.5)
    held = -(-lengths // s.page)
    s.pages, s.columns = int(held.sum()) + 3, int(held.max())
    order = np.random.RandomState(seed & 0x7FFFFFFF).permutation(s.pages).astype(np.int32)
    table = np.full((s.b, s.columns), -1, np.int32)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    s.block_table = torch.from_numpy(table).to(DEVICE)
    s.sinks = torch.randn(s.hq, generator=_gen(seed, 7), device=DEVICE) + 1.0 if case["sinks"] else None

    def pool(tag, width):
        g = _gen(seed, tag)
        codes = torch.empty((s.pages, s.heads, s.page, width // 2), dtype=torch.uint8, device=DEVICE)
        scales = torch.zeros((s.pages, s.heads, s.page, -(-width // 128) * 4), dtype=torch.uint8, device=DEVICE)
        # what rounding normal values leaves: the codes of a block whose largest magnitude is 4 or 6
        step = max(1, (1 << 27) // (s.heads * s.page * width))
        for p in range(0, s.pages, step):
            x = torch.randn((min(step, s.pages - p), s.heads, s.page, width), generator=g, device=DEVICE).bfloat16().float()
            packed, e = _encode(x)
            codes[p:p + step] = packed
            scales[p:p + step, ..., :width // 32] = e
        return codes, scales
    s.k_codes, s.k_scales = pool(8, s.width)
    s.v_codes, s.v_scales = pool(9, s.vwidth) if s.apart else (None, None)


# -- E2M1 codes with E8M0 scales per 32 ------------------------------------------------------------------

def _encode(x):
    """FP32 [..., width] -> packed codes [..., width / 2] (the even value in the low nibble) and scale bytes
    [..., width / 32]: the smallest power of two that keeps the block's largest magnitude (at least 1e-4) within 6, and
    the nearest code, ties to the even one."""
    blocks = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(blocks.abs().amax(-1).clamp_min(1e-4))    # m in [0.5, 1)
    e = torch.where(m > 0.75, e - 2, e - 3).clamp_max(125)
    y = torch.ldexp(blocks, -e[..., None])
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
            + 8 * torch.signbit(y)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (e + 127).to(torch.uint8)


def _decode(packed, scales, width):
    """FP32 [..., width] of packed codes and scale bytes."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=DEVICE)
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).int()
    scale = torch.exp2(scales[..., :width // 32].float() - 127)
    return (grid[code].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


# -- states --------------------------------------------------------------------------------------------

_context = None


def _ctx():
    """The program's one device context."""
    global _context
    if _context is None:
        from vesper_amd import _lib
        _context = _lib.Context(0)
    return _context


class _State:
    pass


def _empty(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device=DEVICE)


def prepare(case, seed):
    s = _State()
    if case["kind"] in ("heads", "heads_bwd"):
        _heads_inputs(s, case, seed)
        s.y = [_empty(s.t, h, s.width, dtype=s.type) for h in s.heads]
        if s.kind == "heads_bwd":
            s.dx = _empty(s.t, sum(s.heads) * s.width, dtype=s.type)
            s.dweights = [None if w is None else _empty(s.norm, dtype=torch.float32) for w in s.weights]
        if own:
            _own_heads(s)
    elif case["kind"] == "append":
        _append_inputs(s, case, seed)
        s.k_codes = _empty(s.pages, s.heads, s.page, s.width // 2, dtype=torch.uint8)
        s.k_scales = _empty(s.pages, s.heads, s.page, -(-s.width // 128) * 4, dtype=torch.uint8)
        s.v_codes = s.v_scales = s.v = None
        s.k = _empty(s.t, s.heads, s.width)
        if s.apart:
            s.v_codes = _empty(s.pages, s.heads, s.page, s.vwidth // 2, dtype=torch.uint8)
            s.v_scales = _empty(s.pages, s.heads, s.page, -(-s.vwidth // 128) * 4, dtype=torch.uint8)
            s.v = _empty(s.t, s.heads, s.vwidth)
        if own:
            _own_cache(s)
            _own_append(s)
    else:
        _attend_inputs(s, case, seed)
        s.out = _empty(s.t, s.hq, s.vwidth)
        s.lse = _empty(s.t, s.hq, dtype=torch.float32)
        if own:
            _own_cache(s)
            _own_attend(s)
    return s


# -- plain forms ---------------------------------------------------------------------------------------

def _angles(s):
    """cos, sin [T, 1, dims / 2] of the tokens' positions."""
    row = s.table[s.positions.long()][:, None]
    return row.chunk(2, -1)


def _turn(x, cos, sin, style):
    """The rotation of x [T, heads, dims]; with -sin its inverse."""
    a, b = x.chunk(2, -1) if style == "halves" else (x[..., 0::2], x[..., 1::2])
    p, q = a * cos - b * sin, b * cos + a * sin
    return torch.cat([p, q], -1) if style == "halves" else torch.stack([p, q], -1).flatten(-2)


def _rms(x, norm):
    """1 / rms of the first `norm` values, computed in 64 bits and rounded to 32."""
    return torch.rsqrt(x[..., :norm].double().square().mean(-1, keepdim=True) + EPS).float()


def _normalized(x, s, weight):
    """FP32 x with its first s.norm values normalized and weighted, and its dims rotated."""
    if s.norm:
        y = x[..., :s.norm] * _rms(x, s.norm)
        x = torch.cat([y if weight is None else y * weight, x[..., s.norm:]], -1)
    cos, sin = _angles(s)
    return torch.cat([x[..., :s.first], _turn(x[..., s.first:], cos, sin, s.style)], -1)


def _columns(s):
    """The queries (and keys) [T, heads, width] of the projection's output."""
    return [c.unflatten(-1, (-1, s.width)) for c in s.rows.split([h * s.width for h in s.heads], -1)]


def _plain_heads(s):
    return [_normalized(x.float(), s, w).to(s.type) for x, w in zip(_columns(s), s.weights)]


def _plain_heads_bwd(s):
    cos, sin = _angles(s)

    def one(x, dy, weight):
        x, g = x.float(), dy.float()
        g = torch.cat([g[..., :s.first], _turn(g[..., s.first:], cos, -sin, s.style)], -1)
        if not s.norm:
            return g.to(s.type), None
        r = _rms(x, s.norm)
        unit, gn = x[..., :s.norm] * r, g[..., :s.norm]
        # a sum of up to 2^18 products in 32 bits would lose what the kernels keep
        dweight = None if weight is None else (gn.double() * unit.double()).sum((0, 1)).float()
        gw = gn if weight is None else gn * weight
        dn = r * (gw - unit * (gw * unit).mean(-1, keepdim=True))
        return torch.cat([dn, g[..., s.norm:]], -1).to(s.type), dweight
    both = [one(x, dy, w) for x, dy, w in zip(_columns(s), s.dy, s.weights)]
    return {"dx": torch.cat([d.flatten(1) for d, _ in both], 1), "dweights": [w for _, w in both]}


def _store(x, s, codes, scales):
    """Codes and scales of FP32 rows [T, heads, width] into their slots; the BF16 values that they stand for."""
    packed, e = _encode(x)
    page, at = s.slots // s.page, s.slots % s.page
    codes[page, :, at] = packed
    scales[page, :, at, :e.shape[-1]] = e
    return _decode(packed, e, x.shape[-1]).bfloat16()


def _plain_append(s):
    keys = s.rows[:, s.column:].unflatten(-1, (s.heads, s.width)).float()
    out = {"k": _store(_normalized(keys, s, s.weight).bfloat16().float(), s, s.k_codes, s.k_scales)}
    if s.apart:
        out["v"] = _store(s.values.bfloat16().float(), s, s.v_codes, s.v_scales)
    return out


def _gathered(s, codes, scales, width):
    """FP32 [B heads, longest, width] of every sequence's tokens."""
    table = s.block_table.clamp_min(0).long()
    x = _decode(codes[table].transpose(1, 2).contiguous(), scales[table].transpose(1, 2).contiguous(), width)
    return x.flatten(2, 3)[:, :, :s.most].reshape(s.b * s.heads, s.most, width)


def _plain_attend(s):
    """The sequences' new tokens padded to the most there are, two batched products, and back."""
    group, n = s.hq // s.heads, s.most_new
    news = s.q_first[1:] - s.q_first[:-1]
    i = torch.arange(n, device=DEVICE)
    at = (s.q_first[:-1, None] + i).clamp_max(s.t - 1).long()
    q = s.q[at].float().view(s.b, n, s.heads, group, s.width).permute(0, 2, 1, 3, 4).reshape(s.b * s.heads, n * group, s.width)
    keys = _gathered(s, s.k_codes, s.k_scales, s.width)
    score = torch.bmm(q, keys.transpose(1, 2).contiguous()).view(s.b, s.heads, n, group, s.most) * s.scale
    position = (s.lengths - news)[:, None] + i                     # of each query
    token = torch.arange(s.most, device=DEVICE)
    seen = token <= position[..., None]
    if s.window:
        seen &= token > position[..., None] - s.window
    score = score.masked_fill(~seen[:, None, :, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    lse = torch.log(total) + top
    if s.sinks is not None:
        total = total + torch.exp(s.sinks.view(1, s.heads, 1, group, 1) - top)
    values = _gathered(s, s.v_codes, s.v_scales, s.vwidth) if s.apart else keys[..., :s.vwidth].contiguous()
    out = torch.bmm(p.view(s.b * s.heads, n * group, s.most), values).view(s.b, s.heads, n, group, s.vwidth)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).to(torch.bfloat16)
    # the sequences' tokens one behind the other
    t = torch.arange(s.t, device=DEVICE)
    b = torch.searchsorted(s.q_first[1:].contiguous(), t, right=True)
    place = t - s.q_first[b]
    return {"out": out.permute(0, 2, 1, 3, 4)[b, place].reshape(s.t, s.hq, s.vwidth),
            "lse": lse.permute(0, 2, 1, 3, 4)[b, place].reshape(s.t, s.hq)}


PLAIN = {"heads": _plain_heads, "heads_bwd": _plain_heads_bwd, "append": _plain_append, "attend": _plain_attend}


# -- the library's calls -------------------------------------------------------------------------------

def _p(t):
    return None if t is None else t.data_ptr()


def _rotation(s):
    from vesper_amd import _lib
    return _lib.MxRotation(table=_p(s.table), table_positions=s.table.shape[0], positions=_p(s.positions), width=s.width,
                           norm=s.norm, first=s.first, dims=s.dims, style=_lib.MX_ROTATE[s.style], inverse=0, eps=EPS)


def _own_heads(s):
    """The structures that a program fills once for its buffers."""
    from vesper_amd import _lib
    s.rotation, size, column = _rotation(s), s.rows.element_size(), 0
    s.sets = (_lib.MxHeads * len(s.heads))()
    s.grads = (_lib.MxHeadsGrad * len(s.heads))()
    total = s.rows.shape[1]
    for i, h in enumerate(s.heads):
        x = s.rows.data_ptr() + column * size
        if s.kind == "heads":
            s.sets[i] = _lib.MxHeads(x, total, h, _p(s.weights[i]), _p(s.y[i]), h * s.width)
        else:
            s.grads[i] = _lib.MxHeadsGrad(x, total, h, _p(s.weights[i]), _p(s.dy[i]), h * s.width,
                                          s.dx.data_ptr() + column * size, total, _p(s.dweights[i]))
        column += h * s.width
    if s.kind == "heads_bwd":
        need = _ctx().lib.cdll.mx_rotate_heads_workspace_bytes(s.norm)
        s.workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=DEVICE)


def _own_cache(s):
    from vesper_amd import _lib
    s.cache = _lib.MxKv4(_p(s.k_codes), _p(s.k_scales), _p(s.v_codes), _p(s.v_scales), s.pages, s.page, s.heads, s.width,
                         s.vwidth)


def _own_append(s):
    from vesper_amd import _lib
    s.rotation = _rotation(s)
    s.call = _lib.MxKv4Append(s.rows.data_ptr() + s.column * s.rows.element_size(), s.stride, _p(s.values),
                              s.heads * s.vwidth, _lib.MX_ROWS["bf16" if s.type == torch.bfloat16 else "f32"], s.t,
                              _p(s.slots), _p(s.weight), _p(s.k), _p(s.v))


def _own_attend(s):
    from vesper_amd import _lib
    s.call = _lib.MxKv4Attend(_p(s.q), s.hq * s.width, s.hq, s.t, s.b, None if s.uniform else _p(s.q_first),
                              _p(s.block_table), s.columns, _p(s.lengths), s.scale, s.window, _p(s.sinks), _p(s.out),
                              s.hq * s.vwidth, _p(s.lse))
    need = _ctx().lib.cdll.mx_kv4_workspace_bytes(_ctx()._h(), C.byref(s.cache), s.hq, s.t, s.b)
    s.workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=DEVICE)


def _own(s):
    lib, h = _ctx().lib, _ctx()._h()
    if s.kind == "heads":
        code = 0 if s.type == torch.bfloat16 else 1   # MX_ROWS_*
        lib.rotate_heads(h, s.sets, len(s.heads), s.t, C.byref(s.rotation), code, code, None)
        return s.y
    if s.kind == "heads_bwd":
        lib.rotate_heads_backward(h, s.grads, len(s.heads), s.t, C.byref(s.rotation),
                                  0 if s.type == torch.bfloat16 else 1, s.workspace.data_ptr(), s.workspace.numel(), None)
        return {"dx": s.dx, "dweights": s.dweights}
    if s.kind == "append":
        lib.kv4_append(h, C.byref(s.cache), C.byref(s.call), C.byref(s.rotation), None)
        return {"k": s.k, "v": s.v} if s.apart else {"k": s.k}
    lib.kv4_attend(h, C.byref(s.cache), C.byref(s.call), s.workspace.data_ptr(), s.workspace.numel(), None)
    return {"out": s.out, "lse": s.lse}


def run(s):
    return _own(s) if own else PLAIN[s.kind](s)


# -- work ----------------------------------------------------------------------------------------------

def work(case):
    if case["kind"] in ("heads", "heads_bwd"):
        hq, hk, width, norm, weights, dims, _ = HEADS[case["heads"]]
        values, t = case["tokens"] * (hq + hk) * width, case["tokens"]
        size = 2 if case["type"] == "bf16" else 4
        tables = t * (4 + 4 * dims) + (8 * norm if weights else 0)
        # x is read for its norm; without one its gradient does not need it
        moved = 2 if case["kind"] == "heads" or not norm else 3
        return {"bytes": moved * size * values + tables, "flops": (8 if case["kind"] == "heads" else 16) * values}
    hq, heads, width, vwidth, apart, _, dims, _, _, _ = CACHES[case["cache"]]
    row = width / 2 + width / 32 + (vwidth / 2 + vwidth / 32 if apart else 0)
    if case["kind"] == "append":
        values, t = case["tokens"] * heads * (width + (vwidth if apart else 0)), case["tokens"]
        size = 2 if case["type"] == "bf16" else 4
        return {"bytes": (size + 2) * values + t * heads * row + t * (12 + 4 * dims), "flops": 12 * values}
    span, pairs = _spans(case)
    t = int(_news(case).sum())
    return {"bytes": span * heads * row + t * hq * (2 * width + 2 * vwidth + 4), "flops": 2 * pairs * hq * (width + vwidth)}


# -- the same results in 64 bits -----------------------------------------------------------------------

def _exact_matrices(s, inverse=False):
    """[T, dims, dims] rotations of the tokens."""
    half = s.dims // 2
    row = s.table.double()[s.positions.long()]
    c, n = row[:, :half], row[:, half:] * (-1 if inverse else 1)
    i = torch.arange(half, device=DEVICE)
    a, b = (i, i + half) if s.style == "halves" else (2 * i, 2 * i + 1)
    m = torch.zeros((s.t, s.dims, s.dims), dtype=torch.float64, device=DEVICE)
    m[:, a, a], m[:, a, b], m[:, b, a], m[:, b, b] = c, -n, n, c
    return m


def _exact_normalized(s, x, weight):
    x = x.double().clone()
    if s.norm:
        root = torch.sqrt((x[..., :s.norm] ** 2).sum(-1, keepdim=True) / s.norm + EPS)
        x[..., :s.norm] /= root
        if weight is not None:
            x[..., :s.norm] *= weight.double()
    for t0 in range(0, s.t, 512):
        m = _exact_matrices_of(s, t0, t0 + 512)
        x[t0:t0 + 512, :, s.first:] = torch.matmul(x[t0:t0 + 512, :, s.first:].contiguous(), m.transpose(1, 2).contiguous())
    return x


def _exact_matrices_of(s, t0, t1):
    part = _State()
    part.dims, part.style, part.table, part.positions = s.dims, s.style, s.table, s.positions[t0:t1]
    part.t = part.positions.numel()
    return _exact_matrices(part)


def _exact_rounded(x):
    """The values of FP32-representable x [..., width] rounded to E2M1 under E8M0 scales, by a search of the grid."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=DEVICE)
    blocks = x.unflatten(-1, (-1, 32))
    scale = torch.exp2(torch.ceil(torch.log2(blocks.abs().amax(-1, keepdim=True).clamp_min(1e-4) / 6.0)))
    y = blocks / scale
    high = torch.searchsorted(grid, y.abs().contiguous()).clamp(1, 7)
    low = high - 1
    to_low, to_high = y.abs() - grid[low], grid[high] - y.abs()
    pick = torch.where((to_high < to_low) | ((to_high == to_low) & (high % 2 == 0)), high, low)
    return (torch.sign(y) * grid[pick] * scale).flatten(-2)


def _exact_attend(s):
    group = s.hq // s.heads
    out = torch.zeros((s.t, s.hq, s.vwidth), dtype=torch.float64, device=DEVICE)
    lse = torch.zeros((s.t, s.hq), dtype=torch.float64, device=DEVICE)
    first, lengths = s.q_first.tolist(), s.lengths.tolist()

    def tokens(codes, scales, pages, head, length, width):
        rows = codes[pages, head].reshape(-1, width // 2)[:length]
        e = scales[pages, head].reshape(-1, scales.shape[-1])[:length, :width // 32].double() - 127
        low, high = (rows & 15).long(), (rows >> 4).long()
        code = torch.stack([low, high], -1).reshape(length, width)
        mag = torch.where(code % 8 < 2, (code % 8) * 0.5, (1 + (code % 2) * 0.5) * torch.exp2(((code % 8) // 2 - 1).double()))
        return (mag.double() * torch.where(code >= 8, -1.0, 1.0)).view(length, -1, 32).mul(torch.exp2(e)[..., None]).view(length, width)
    for b in range(s.b):
        n, length = first[b + 1] - first[b], lengths[b]
        pages = s.block_table[b, :-(-length // s.page)].long()
        for h in range(s.heads):
            k = tokens(s.k_codes, s.k_scales, pages, h, length, s.width)
            v = tokens(s.v_codes, s.v_scales, pages, h, length, s.vwidth) if s.apart else k[:, :s.vwidth]
            for i0 in range(0, n, 256):   # pieces, so that the scores stay small
                i1 = min(n, i0 + 256)
                q = s.q[first[b] + i0:first[b] + i1, h * group:(h + 1) * group].double()
                score = (q.reshape(-1, s.width) @ k.T).view(i1 - i0, group, length) * s.scale
                where = length - n + torch.arange(i0, i1, device=DEVICE)[:, None]
                t = torch.arange(length, device=DEVICE)[None, :]
                hidden = (t > where) | (t <= where - s.window if s.window else torch.zeros_like(t > where))
                score = score.masked_fill(hidden[:, None], -math.inf)
                total = torch.logsumexp(score, -1)
                with_sink = total if s.sinks is None else torch.logaddexp(
                    total, s.sinks[h * group:(h + 1) * group].double().expand_as(total))
                p = torch.exp(score - with_sink[..., None].clamp_min(-1e300))
                out[first[b] + i0:first[b] + i1, h * group:(h + 1) * group] = (p.view(-1, length) @ v).view(i1 - i0, group, -1)
                lse[first[b] + i0:first[b] + i1, h * group:(h + 1) * group] = total
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = _State()
    if case["kind"] == "heads":
        _heads_inputs(s, case, seed)
        return [_exact_normalized(s, x, w) for x, w in zip(_columns(s), s.weights)]
    if case["kind"] == "heads_bwd":
        _heads_inputs(s, case, seed)
        dx, dweights = [], []
        for x, dy, w in zip(_columns(s), s.dy, s.weights):   # by the product rule, from y = M (w x / root)
            x, g = x.double(), dy.double().clone()
            for t0 in range(0, s.t, 512):
                g[t0:t0 + 512, :, s.first:] = torch.matmul(g[t0:t0 + 512, :, s.first:].contiguous(),
                                                           _exact_matrices_of(s, t0, t0 + 512))
            if s.norm:
                xn, gn = x[..., :s.norm], g[..., :s.norm]
                square = (xn ** 2).sum(-1, keepdim=True) / s.norm + EPS
                dweights.append(None if w is None else (gn * xn / torch.sqrt(square)).sum((0, 1)))
                gw = gn if w is None else gn * w.double()
                g[..., :s.norm] = gw / torch.sqrt(square) - xn * (gw * xn).sum(-1, keepdim=True) / (s.norm * square ** 1.5)
            else:
                dweights.append(None)
            dx.append(g.flatten(1))
        return {"dx": torch.cat(dx, 1), "dweights": dweights}
    if case["kind"] == "append":
        _append_inputs(s, case, seed)
        keys = s.rows[:, s.column:].unflatten(-1, (s.heads, s.width))
        # the definition rounds to BF16 before the codes
        out = {"k": _exact_rounded(_exact_normalized(s, keys, s.weight).bfloat16().double())}
        if s.apart:
            out["v"] = _exact_rounded(s.values.bfloat16().double())
        return out
    _attend_inputs(s, case, seed)
    return _exact_attend(s)
