"""Tokens sorted by expert and back, and low-rank adapters of many requests: the workloads by which their speed
is followed.

Each case is one pass of one operator, as a program that uses the library calls it (device tensors in, device
tensors out, no host synchronisation):

  dispatch      routing ids [T, k] -> the plan (first row of each expert, row of each pair, pair of each row) and
                the tokens' rows in expert order, with the route weights in the same order. "mx8" rows are E4M3
                codes with their E8M0 block scales, moved by one plan
  combine       expert outputs in expert order -> one row per token: the (weighted) sum of its experts' rows in
                ascending expert order, the shared expert's row last
  combine_bwd   the gradients of the weighted sum: of every expert row, and of every route weight
  dispatch_bwd  the gradients of the copy: the sum of a token's rows, and of its weights
  adapters      y = base + scale * up (down x) with the low-rank pair of each token's request, beside a projection

With own = False the same results come from elementary torch operations in 32 bits.
"""

import ctypes as C
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
# hidden, experts, experts per token, route scale of vesper_amd.config.BASELINE and REFERENCE
MODELS = {"base": (7168, 256, 8, 2.5), "ref": (5120, 384, 6, 1.5)}
# rows x width of the FP8 projections the adapters stand beside (vesper_amd.projections)
PROJECTIONS = {"q_a": (1536, 7168), "q_b": (24576, 1536), "kv_a": (576, 7168), "o": (7168, 16384),
               "wq_a": (1280, 5120), "wkv": (512, 5120), "wo_b": (5120, 8192)}
STACKED = {"q_a": (0, 2112), "kv_a": (1536, 2112)}   # column and width of the stacked output these two share
ZIPF = 1.1
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # the next token of one session: its row to eight experts
        {"name": "dispatch-1", "kind": "dispatch", "model": "base", "tokens": 1, "rows": "bf16", "skew": False,
         "held": 256},
        # a prompt of the 384-expert model whose activations are quantized already: codes and scales move together
        {"name": "dispatch-codes-1000", "kind": "dispatch", "model": "ref", "tokens": 1000, "rows": "mx8",
         "skew": False, "held": 384},
        # a long prompt with skewed routing
        {"name": "dispatch-4096", "kind": "dispatch", "model": "base", "tokens": 4096, "rows": "bf16", "skew": True,
         "held": 256},
        # a decode batch whose experts applied the route weights before their last product: a plain ordered sum
        {"name": "combine-16", "kind": "combine", "model": "base", "tokens": 16, "rows": "bf16", "skew": False,
         "held": 256, "weighted": False, "shared": True},
        # a long prompt, weights applied here, the shared expert's rows last
        {"name": "combine-4096", "kind": "combine", "model": "base", "tokens": 4096, "rows": "bf16", "skew": True,
         "held": 256, "weighted": True, "shared": True},
        # one of eight expert-parallel ranks in training: the pairs of 48 of 384 experts are here, FP32 rows
        {"name": "combine-bwd-held-1500", "kind": "combine_bwd", "model": "ref", "tokens": 1500, "rows": "f32",
         "skew": False, "held": 48},
        # a training batch on one device
        {"name": "combine-bwd-4096", "kind": "combine_bwd", "model": "base", "tokens": 4096, "rows": "bf16",
         "skew": True, "held": 256},
        # a short sequence in training
        {"name": "dispatch-bwd-333", "kind": "dispatch_bwd", "model": "ref", "tokens": 333, "rows": "f32",
         "skew": False, "held": 384},
        # a training batch on one device
        {"name": "dispatch-bwd-4096", "kind": "dispatch_bwd", "model": "base", "tokens": 4096, "rows": "bf16",
         "skew": True, "held": 256},
        # one session with an adapter on q_b, added to the projection's FP32 sums
        {"name": "adapters-1", "kind": "adapters", "proj": "q_b", "tokens": 1, "adapters": 4, "rank": 16,
         "base": "f32"},
        # a decode batch of sessions with adapters of their own beside the output projection
        {"name": "adapters-24", "kind": "adapters", "proj": "o", "tokens": 24, "adapters": 16, "rank": 64,
         "base": "bf16"},
        # prompts of several requests in one batch
        {"name": "adapters-4096", "kind": "adapters", "proj": "o", "tokens": 4096, "adapters": 8, "rank": 64,
         "base": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["dispatch", "combine", "combine_bwd", "dispatch_bwd", "adapters", "adapters"])
    if kind == "adapters":
        return {"kind": kind, "proj": rng.choice(sorted(PROJECTIONS)), "tokens": _log_int(rng, 1, 4096),
                "adapters": _log_int(rng, 1, 32), "rank": rng.choice([8, 12, 16, 32, 64, 128]),
                "base": rng.choice(["bf16", "f32"])}
    model = rng.choice(["base", "ref"])
    experts = MODELS[model][1]
    case = {"kind": kind, "model": model, "rows": rng.choice(["bf16", "bf16", "f32"]), "skew": rng.random() < 0.5,
            "held": rng.choice([experts, experts, experts // 8])}
    if kind == "dispatch":
        case["rows"] = rng.choice(["bf16", "f32", "mx8"])
    if kind == "combine":
        case["weighted"], case["shared"] = rng.random() < 0.7, rng.random() < 0.5
    case["tokens"] = _log_int(rng, 1, 2048 if case["rows"] == "f32" else 4096)
    return case


# -- seeded inputs -------------------------------------------------------------------------------------

def _gen(seed, *tag):
    g = torch.Generator(device=DEVICE)
    value = seed & 0xFFFFFFFF
    for t in tag:
        value = (value * 1000003 + t + 1) & 0x7FFFFFFFFFFF
    g.manual_seed(value)
    return g


def _normal(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device=DEVICE).to(dtype)


def _routing(case, seed):
    """Distinct experts per token (the largest of log p + Gumbel noise; p uniform, or falling as 1 / rank^ZIPF over
    a random order) as ids relative to the first expert held here, and positive weights normalized to the route
    scale. Ids outside [0, held) are experts of other devices."""
    _, experts, k, scale = MODELS[case["model"]]
    g, t = _gen(seed, 4), case["tokens"]
    rank = torch.randperm(experts, generator=g, device=DEVICE).double() + 1
    noise = -torch.log(-torch.log(torch.rand((t, experts), generator=g, device=DEVICE,
                                             dtype=torch.float64).clamp(1e-300, 1 - 1e-16)))
    score = noise - ZIPF * torch.log(rank) if case["skew"] else noise
    ids = torch.topk(score, k, dim=1).indices
    ids = (ids - (experts - case["held"]) // 2).to(torch.int32).contiguous()
    raw = torch.rand((t, k), generator=g, device=DEVICE) * 0.95 + 0.05
    return ids, (raw / raw.sum(1, keepdim=True) * scale).contiguous()


def _mx8(x):
    """E4M3 codes and E8M0 scales of BF16 rows, per 32 values: the smallest power of two that keeps the block in
    range."""
    v = x.float().view(x.shape[0], -1, 32)
    amax = v.abs().amax(-1).clamp_min(1e-4)
    e = torch.ceil(torch.log2(amax.double() / 448.0))
    q = (v / torch.exp2(e).float()[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).view(x.shape[0], -1), (e + 127).to(torch.uint8).contiguous()


def _requests(case, seed):
    """Adapter of each token, -1 for none, on the host. A batch of few tokens is a decode batch (one token per
    request, in any order); a larger one is the concatenation of the requests' prompts."""
    r, t, n = np.random.RandomState(seed & 0x7FFFFFFF), case["tokens"], case["adapters"]
    if t <= 64:
        return r.randint(-1 if t > 1 else 0, n, t).astype(np.int32)
    parts = min(t, 2 * n + 1)
    cuts = np.sort(r.choice(np.arange(1, t), parts - 1, replace=False)) if parts > 1 else np.zeros(0, np.int64)
    lengths = np.diff(np.concatenate([[0], cuts, [t]]))
    return np.repeat(r.randint(-1, n, parts), lengths).astype(np.int32)


def _adapter_weights(case, seed):
    """down [S, rank, K], up [S, N, rank] BF16 and FP32 scales."""
    n, k = PROJECTIONS[case["proj"]]
    s, r = case["adapters"], case["rank"]
    g = _gen(seed, 6)
    down = _normal(g, s, r, k)
    up = torch.empty((s, n, r), dtype=torch.bfloat16, device=DEVICE)
    up.copy_(torch.randn((s, n, r), generator=g, device=DEVICE) * (1.0 / math.sqrt(k * r)))
    return down, up, (torch.rand(s, generator=g, device=DEVICE) * 1.5 + 0.5)


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
    """What the program keeps; the adapters' device memory goes back when it is dropped."""

    bank = None

    def __del__(self):
        if self.bank is not None:
            self.bank.close()


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _plan_outputs(s, pairs):
    s.first = torch.zeros(s.held + 1, dtype=torch.int32, device=DEVICE)
    s.pair_row = torch.zeros((s.tokens, s.k), dtype=torch.int32, device=DEVICE)
    s.row_pair = torch.zeros(pairs, dtype=torch.int32, device=DEVICE)


def _inputs(s, case, seed):
    """The routed kinds' inputs: everything drawn from the seed, by exact() too."""
    s.kind, s.tokens, s.held = case["kind"], case["tokens"], case["held"]
    s.hidden, _, s.k, _ = MODELS[case["model"]]
    s.rows_type = case["rows"]
    t, k, h = s.tokens, s.k, s.hidden
    s.ids, s.weights = _routing(case, seed)
    if s.kind == "dispatch":
        x = _normal(_gen(seed, 5), t, h, dtype=TYPES.get(s.rows_type, torch.bfloat16))
        s.x = list(_mx8(x)) if s.rows_type == "mx8" else [x]
        return
    dtype = TYPES[s.rows_type]
    s.rows = _normal(_gen(seed, 7), t * k, h, dtype=dtype)
    if s.kind == "combine":
        s.shared = _normal(_gen(seed, 8), t, h, dtype=dtype) if case["shared"] else None
        if not case["weighted"]:
            s.weights = None
    elif s.kind == "combine_bwd":
        s.dy = _normal(_gen(seed, 8), t, h, dtype=dtype)
    else:
        s.drow_weights = _normal(_gen(seed, 9), t * k, dtype=torch.float32)


def _adapter_inputs(s, case, seed):
    s.kind, s.tokens = "adapters", case["tokens"]
    s.n, s.width = PROJECTIONS[case["proj"]]
    s.column, s.stride = STACKED.get(case["proj"], (0, s.n))
    s.host_ids = _requests(case, seed)
    s.ids = torch.from_numpy(s.host_ids).to(DEVICE)
    s.x = _normal(_gen(seed, 5), s.tokens, s.width)
    # the projection's outputs: FP32 sums [T, N], or BF16 rows of the (stacked) output
    s.base = (_normal(_gen(seed, 8), s.tokens, s.n, dtype=torch.float32) if case["base"] == "f32" else
              _normal(_gen(seed, 8), s.tokens, s.stride)[:, s.column:s.column + s.n])
    s.down, s.up, s.scale = _adapter_weights(case, seed)


def prepare(case, seed):
    s = _State()
    if case["kind"] == "adapters":
        _adapter_inputs(s, case, seed)
        s.longest = int(np.bincount(s.host_ids + 1, minlength=1).max())   # tokens of the busiest adapter, or of none
        s.y = torch.zeros((s.tokens, s.stride), dtype=torch.bfloat16, device=DEVICE)[:, s.column:s.column + s.n]
        if own:
            from vesper_amd.adapters import AdapterBank
            s.bank = AdapterBank(_ctx(), s.n, s.width, slots=case["adapters"], max_rank=case["rank"],
                                 max_tokens=s.tokens)
            scales = s.scale.cpu().tolist()
            for slot in range(case["adapters"]):
                s.bank.load_device(slot, s.down[slot].data_ptr(), s.up[slot].data_ptr(), case["rank"], scales[slot])
        return s
    _inputs(s, case, seed)
    t, k, h = s.tokens, s.k, s.hidden
    _plan_outputs(s, t * k)
    if own:
        from vesper_amd import _lib
        s.plan = _lib.MxRowPlan(s.first.data_ptr(), s.pair_row.data_ptr(), s.row_pair.data_ptr())
    if s.kind == "dispatch":
        s.out = [torch.zeros((t * k, x.shape[1]), dtype=x.dtype, device=DEVICE) for x in s.x]
        s.row_weights = torch.zeros(t * k, device=DEVICE)
        return s
    first, pair_row, row_pair = _plan(s.ids, s.held)   # what the forward pass left
    s.first.copy_(first), s.pair_row.copy_(pair_row), s.row_pair.copy_(row_pair)
    dtype = s.rows.dtype
    if s.kind == "combine":
        s.y = torch.zeros((t, h), dtype=dtype, device=DEVICE)
    elif s.kind == "combine_bwd":
        s.drows = torch.zeros((t * k, h), dtype=dtype, device=DEVICE)
        s.dweights = torch.zeros((t, k), device=DEVICE)
    else:
        s.dx = torch.zeros((t, h), dtype=dtype, device=DEVICE)
        s.dweights = torch.zeros((t, k), device=DEVICE)
    return s


# -- plain forms ---------------------------------------------------------------------------------------

def _plan(ids, held):
    """first [held + 1], pair_row [T, k] (-1: not held), row_pair [T k]: pairs in the order of their expert, then of
    their index, the ones not held last."""
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < held), flat, torch.full_like(flat, held))
    row_pair = torch.argsort(key, stable=True)
    row = torch.empty_like(row_pair)
    row[row_pair] = torch.arange(flat.numel(), device=DEVICE)
    pair_row = torch.where(key < held, row, torch.full_like(row, -1)).view(ids.shape)
    first = (key[None, :] < torch.arange(held + 1, device=DEVICE)[:, None]).sum(1)
    return first.to(torch.int32), pair_row.to(torch.int32), row_pair.to(torch.int32)


def _plain_dispatch(s):
    first, pair_row, row_pair = _plan(s.ids, s.held)
    kept = torch.arange(row_pair.numel(), device=DEVICE) < first[-1]
    token = (row_pair // s.k).long()
    rows = [torch.where(kept[:, None], x[token], torch.zeros((), dtype=x.dtype, device=DEVICE)) for x in s.x]
    row_weights = torch.where(kept, s.weights.reshape(-1)[row_pair.long()], torch.zeros((), device=DEVICE))
    return {"rows": rows, "row_weights": row_weights, "first": first, "pair_row": pair_row, "row_pair": row_pair}


def _gathered(rows, pair_row):
    """FP32 [T, k, H]: the row of each pair, zero where there is none."""
    picked = rows[pair_row.clamp_min(0).long()].float()
    return torch.where((pair_row >= 0)[..., None], picked, torch.zeros((), device=DEVICE))


def _plain_combine(s):
    picked = _gathered(s.rows, s.pair_row)
    if s.weights is not None:
        picked = picked * s.weights[..., None]
    y = picked.sum(1)
    if s.shared is not None:
        y = y + s.shared.float()
    return y.to(s.rows.dtype)


def _plain_combine_bwd(s):
    kept = torch.arange(s.row_pair.numel(), device=DEVICE) < s.first[-1]
    pair = s.row_pair.long()
    drows = s.weights.reshape(-1)[pair][:, None] * s.dy[pair // s.k].float()
    drows = torch.where(kept[:, None], drows, torch.zeros((), device=DEVICE)).to(s.rows.dtype)
    return {"drows": drows, "dweights": (_gathered(s.rows, s.pair_row) * s.dy.float()[:, None, :]).sum(-1)}


def _plain_dispatch_bwd(s):
    picked = s.drow_weights[s.pair_row.clamp_min(0).long()]
    return {"dx": _gathered(s.rows, s.pair_row).sum(1).to(s.rows.dtype),
            "dweights": torch.where(s.pair_row >= 0, picked, torch.zeros((), device=DEVICE))}


def _plain_adapters(s):
    """The tokens of each adapter padded to the busiest one's count, two batched products, and back; the tokens
    without an adapter are one more group, with a pair of zeros."""
    groups, rank, width = s.down.shape
    group = torch.where(s.ids >= 0, s.ids, torch.full_like(s.ids, groups)).long()
    order = torch.argsort(group, stable=True)
    start = (group[None, :] < torch.arange(groups + 1, device=DEVICE)[:, None]).sum(1)
    place = torch.empty_like(order)
    place[order] = torch.arange(s.tokens, device=DEVICE) - start[group[order]]
    x = torch.zeros((groups + 1, s.longest, width), device=DEVICE)
    x[group, place] = s.x.float()
    zero = lambda w: torch.zeros((1, *w.shape[1:]), device=DEVICE)  # noqa: E731
    down = torch.cat([s.down.float(), zero(s.down)]).transpose(1, 2).contiguous()
    up = torch.cat([s.up.float(), zero(s.up)]).transpose(1, 2).contiguous()
    scale = torch.cat([s.scale, torch.zeros(1, device=DEVICE)])
    delta = torch.bmm(torch.bmm(x, down) * scale[:, None, None], up)
    return (s.base.float() + delta[group, place]).to(torch.bfloat16)


PLAIN = {"dispatch": _plain_dispatch, "combine": _plain_combine, "combine_bwd": _plain_combine_bwd,
         "dispatch_bwd": _plain_dispatch_bwd, "adapters": _plain_adapters}


# -- the library's calls -------------------------------------------------------------------------------

DTYPE = {"bf16": 0, "f32": 1, "mx8": 2}   # MX_ROWS_*


def _own(s):
    if s.kind == "adapters":
        s.bank.apply_device(s.x.data_ptr(), s.ids.data_ptr(), s.tokens, s.base.data_ptr(), s.y.data_ptr(),
                            base_dtype="f32" if s.base.dtype == torch.float32 else "bf16",
                            base_stride=s.base.stride(0), y_stride=s.stride)
        return s.y
    lib, h, dtype, t, k = _ctx().lib, _ctx()._h(), DTYPE[s.rows_type], s.tokens, s.k
    if s.kind == "dispatch":
        lib.dispatch(h, _p(s.ids), t, k, s.held, C.byref(s.plan), _p(s.x[0]), dtype, s.x[0].shape[1], _p(s.weights),
                     _p(s.out[0]), _p(s.row_weights), None)
        if s.rows_type == "mx8":   # the block scales, by the plan that the codes' call made
            lib.dispatch(h, None, t, k, s.held, C.byref(s.plan), _p(s.x[1]), dtype, s.x[1].shape[1], None,
                         _p(s.out[1]), None, None)
        return {"rows": s.out, "row_weights": s.row_weights, "first": s.first, "pair_row": s.pair_row,
                "row_pair": s.row_pair}
    if s.kind == "combine":
        lib.combine(h, _p(s.rows), dtype, _p(s.pair_row), _p(s.weights), _p(s.shared), t, k, s.hidden, _p(s.y), None)
        return s.y
    if s.kind == "combine_bwd":
        lib.combine_backward(h, _p(s.dy), _p(s.rows), dtype, _p(s.pair_row), _p(s.weights), t, k, s.hidden,
                             _p(s.drows), _p(s.dweights), None)
        return {"drows": s.drows, "dweights": s.dweights}
    lib.dispatch_backward(h, _p(s.rows), dtype, _p(s.pair_row), _p(s.drow_weights), t, k, s.hidden, _p(s.dx),
                          _p(s.dweights), None)
    return {"dx": s.dx, "dweights": s.dweights}


def run(s):
    return _own(s) if own else PLAIN[s.kind](s)


# -- work ----------------------------------------------------------------------------------------------

def work(case):
    t = case["tokens"]
    if case["kind"] == "adapters":
        n, k = PROJECTIONS[case["proj"]]
        r, s = case["rank"], case["adapters"]
        here = s * (1 - (1 - 1 / (s + 1)) ** (t if t <= 64 else min(t, 2 * s + 1)))   # distinct adapters named
        base = 4 if case["base"] == "f32" else 2
        return {"bytes": here * 2 * r * (n + k) + t * (2 * k + (base + 2) * n + 4), "flops": 2 * t * r * (n + k)}
    h, experts, k, _ = MODELS[case["model"]]
    pairs = t * k * case["held"] / experts          # pairs of experts held here, on average
    size = {"bf16": 2, "f32": 4, "mx8": 33 / 32}[case["rows"]]
    row = size * h
    if case["kind"] == "dispatch":
        return {"bytes": (t + pairs) * row + 8 * t * k + 4 * pairs + 8 * t * k + 4 * case["held"], "flops": 0}
    if case["kind"] == "combine":
        extra = (4 * t * k if case["weighted"] else 0) + (t * row if case["shared"] else 0)
        return {"bytes": (t + pairs) * row + 4 * t * k + extra, "flops": 2 * pairs * h}
    if case["kind"] == "combine_bwd":
        return {"bytes": (t + 2 * pairs) * row + 12 * t * k, "flops": 3 * pairs * h}
    return {"bytes": (t + pairs) * row + 12 * t * k, "flops": pairs * h}


# -- the same results in 64 bits -----------------------------------------------------------------------

def _e4m3_values(codes):
    return codes.view(torch.float8_e4m3fn).double()


def _exact_rows(s):
    """(pairs in expert order, their tokens, their rows, number held) from a search of every expert in turn."""
    flat = s.ids.reshape(-1)
    pairs = torch.cat([torch.nonzero(flat == e).reshape(-1) for e in range(s.held)])
    return pairs, pairs // s.k, torch.arange(pairs.numel(), device=DEVICE)


def exact(case, seed):
    s = _State()
    if case["kind"] == "adapters":
        _adapter_inputs(s, case, seed)
        y = s.base.double()
        for a in range(case["adapters"]):
            own_rows = torch.nonzero(s.ids == a).reshape(-1)
            if own_rows.numel():
                low = s.x[own_rows].double() @ s.down[a].double().T
                y = y.index_add(0, own_rows, s.scale[a].double() * (low @ s.up[a].double().T))
        return y
    _inputs(s, case, seed)
    pairs, tokens, rows = _exact_rows(s)
    t, k, h = s.tokens, s.k, s.hidden
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=DEVICE)  # noqa: E731
    if s.kind == "dispatch":
        row_weights = zeros(t * k)
        row_weights[rows] = s.weights.reshape(-1)[pairs].double()
        if s.rows_type == "mx8":
            moved = [None, None]   # whole numbers
        else:
            moved = [zeros(t * k, h)]
            moved[0][rows] = s.x[0][tokens].double()
        return {"rows": moved, "row_weights": row_weights, "first": None, "pair_row": None, "row_pair": None}
    weights = None if s.weights is None else s.weights.reshape(-1)[pairs].double()
    picked = s.rows[:pairs.numel()].double()   # expert order
    if s.kind == "combine":
        y = zeros(t, h) if s.shared is None else s.shared.double()
        return y.index_add(0, tokens, picked if weights is None else picked * weights[:, None])
    if s.kind == "combine_bwd":
        dy = s.dy.double()[tokens]
        drows, dweights = zeros(t * k, h), zeros(t * k)
        drows[rows] = dy * weights[:, None]
        dweights[pairs] = (picked * dy).sum(1)
        return {"drows": drows, "dweights": dweights.view(t, k)}
    dweights = zeros(t * k)
    dweights[pairs] = s.drow_weights[rows].double()
    return {"dx": zeros(t, h).index_add(0, tokens, picked), "dweights": dweights.view(t, k)}
