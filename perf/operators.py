"""What is measured of the operators of a mixture-of-experts layer on quantised weights: the router with the plan of the ragged products, the
products grouped by expert, the weighted sum of the experts' answers.

listed()   the cases that are timed by name
draw(rng)  one more case of the same ranges
prepare / run / work / exact   of one case

A case's "kind" says which operator a pass is:
  route     logits [tokens, experts] -> the experts that each token picks, their weights, and the pairs (token, pick) sorted by expert
  experts   C[r] = A[row of r] x dequant(B[expert of r])^T over the sorted pairs: the first product of a layer takes the tokens' rows through
            the plan ("gather"), the second one the first one's rows as they lie; "gated": rows 2i / 2i+1 of B are the gate and the up projection
            of channel i, C = silu(gate) * up
  combine   out[t] = sum of weight * the expert's answer over the picks of token t, plus the residual
Weights: int8 or int4 [experts, n, k], k contiguous, plain or in the pre-packed word order, scales per channel (fp32) or per group (bf16),
zero-points where a case says so.
"""
import math

import torch

own = False

_MOST_WORK = 2 * 8192 * 22016 * 4096   # flops of the largest listed case
_MOST_WEIGHTS = 8 * 22016 * 4096       # weights of all experts of the largest listed case


def _route(tokens, experts, top_k, f32=False, renormalize=True, padded=0):
    return dict(kind="route", tokens=tokens, experts=experts, top_k=top_k, f32=f32, renormalize=renormalize, padded=padded)


def _experts(tokens, experts, top_k, n, k, bits, group=0, zero=False, offset=False, packed=False, gated=False, gather=True):
    return dict(kind="experts", tokens=tokens, experts=experts, top_k=top_k, n=n, k=k, bits=bits, group=group, zero=zero, offset=offset,
                packed=packed, gated=gated, gather=gather)


def _combine(tokens, top_k, n, residual=True, padded=0):
    return dict(kind="combine", tokens=tokens, top_k=top_k, n=n, residual=residual, padded=padded)


def listed():
    cases = [
        # one token picks 8 of 64 experts: the decode loop of a single user, latency only
        ("route-t1", _route(1, 64, 8)),
        # a prompt of odd length in a batch padded to it: the last tokens are masked and pick nothing; fp32 logits
        ("route-t4099", _route(4099, 128, 8, f32=True, padded=300)),
        # one token through the gate and up projections of its 8 experts, int4 in groups of 128
        ("gateup-t1-int4", _experts(1, 64, 8, 2048, 4096, 4, 128, packed=True, gated=True)),
        # five drafted tokens being verified, down projection, zero-points, int4 weights as they were stored (not pre-packed)
        ("down-t5-int4-zero", _experts(5, 32, 4, 4096, 2816, 4, 128, zero=True, gather=False)),
        # sixteen users on 8 wide experts, int8 per channel: 32 rows on 8 experts
        ("gateup-t16-int8", _experts(16, 8, 2, 22016, 4096, 8, gated=True)),
        # a batch of 128 users: 16 rows per expert in the mean, some with several times as many, some with none
        ("gateup-t128-int4", _experts(128, 64, 8, 2048, 4096, 4, 128, packed=True, gated=True)),
        # a prompt of odd length, odd number of channels, groups of 64: 250 rows per expert in the mean
        ("down-t1001-int4", _experts(1001, 16, 4, 4104, 1408, 4, 64, gather=False)),
        # a prompt of 2048 tokens on many narrow experts, int4
        ("gateup-t2048-int4", _experts(2048, 64, 8, 2048, 4096, 4, 128, packed=True, gated=True)),
        # the largest: a prompt of 4096 tokens on 8 wide experts, int8 stored with offset 128 as the dense products take it
        ("gateup-t4096-int8", _experts(4096, 8, 2, 22016, 4096, 8, offset=True, gated=True)),
        # the weighted sum for five tokens, and for a prompt with padded tokens
        ("combine-t5", _combine(5, 4, 4096)),
        ("combine-t4099", _combine(4099, 8, 4096, padded=300)),
    ]
    return [dict(c, name=name) for name, c in cases]


def _log_uniform(rng, lo, hi, multiple=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / multiple)) * multiple))


def draw(rng):
    kind = rng.choice(["route", "experts", "experts", "experts", "experts", "combine"])
    tokens, experts = _log_uniform(rng, 1, 4096), _log_uniform(rng, 8, 128)
    top_k = rng.randint(1, 8)
    padded = rng.randint(0, tokens // 8)
    if kind == "route":
        return _route(tokens, experts, top_k, f32=rng.random() < 0.5, renormalize=rng.random() < 0.5, padded=padded)
    if kind == "combine":
        return _combine(tokens, top_k, _log_uniform(rng, 1024, 8192, 8), residual=rng.random() < 0.5, padded=padded)
    gated = rng.random() < 0.5
    k = _log_uniform(rng, 1024, 8192, 128)
    n = _log_uniform(rng, 1024, 11008, 16)
    experts = max(8, min(experts, _MOST_WEIGHTS // (n * k)))
    n = max(1024, min(n, _MOST_WEIGHTS // (experts * k) // 16 * 16))
    tokens = max(1, min(tokens, _MOST_WORK // (2 * top_k * n * k)))
    bits = rng.choice([8, 4, 4])
    group = rng.choice([128, 128, 64, 0]) if bits == 4 else rng.choice([0, 0, 128])
    return _experts(tokens, experts, top_k, n, k, bits, group, zero=bits == 4 and group > 0 and rng.random() < 0.4, offset=rng.random() < 0.3,
                    packed=rng.random() < 0.5, gated=gated, gather=rng.random() < 0.6)


class _Maker:
    """Inputs from a seed: activations ~ N(0, 1), integers uniform over their range, positive scales, zero-points near the middle, logits of
    a router that likes some experts better than others."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, device="cuda", generator=self.gen, dtype=torch.float32)

    def activations(self, rows, cols):
        return self.normal(rows, cols).to(torch.bfloat16)

    def logits(self, tokens, experts):
        return self.normal(tokens, experts) * 1.5 + self.normal(experts)

    def weights(self, case):
        rows = case["experts"] * case["n"]
        if case["bits"] == 4:   # two per byte along k; every byte is a legal pair
            q = torch.randint(0, 256, (rows, case["k"] // 2), device="cuda", generator=self.gen, dtype=torch.uint8)
        else:
            q = torch.randint(-127, 128, (rows, case["k"]), device="cuda", generator=self.gen, dtype=torch.int8)
            q = q ^ -128 if case["offset"] else q
        return q.reshape(case["experts"], case["n"], -1)

    def scales(self, case):
        e, n, k, group = case["experts"], case["n"], case["k"], case["group"]
        if group:
            per = 0.005 if case["bits"] == 4 else 0.0005
            return (torch.rand((e, n, k // group), device="cuda", generator=self.gen) * 9 * per + per).to(torch.bfloat16)
        return torch.rand((e, n), device="cuda", generator=self.gen) * 0.009 + 0.001

    def zeros(self, case):
        if not case["zero"]:
            return None
        z = torch.randint(-3, 4, (case["experts"], case["n"], case["k"] // case["group"]), device="cuda", generator=self.gen, dtype=torch.int16)
        return ((z + 8 if case["offset"] else z) & 15).to(torch.uint8)


def _picks(logits, top_k):
    """The k largest of every row in order, ties to the lowest index."""
    return torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top_k]


def _plan(ids, experts):
    """offsets, row_pair, pair_row of ids [tokens, top_k] (-1: no expert)."""
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(experts + 1, device=key.device)).sum(0)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=key.device)
    offsets[1:] = counts.cumsum(0)
    total = offsets[experts]
    place = torch.arange(flat.numel(), device=key.device)
    row_pair = torch.where(place < total, order, -1)
    pair_row = torch.empty_like(order)
    pair_row[order] = place
    pair_row = torch.where(flat < 0, -1, pair_row)
    return offsets.int(), row_pair.int(), pair_row.int().reshape(ids.shape)


def prepare(case, seed):
    make = _Maker(seed)
    tokens, top_k = case["tokens"], case["top_k"]
    pairs = tokens * top_k
    state = dict(case=case, stream=torch.cuda.current_stream().cuda_stream)

    def ints(*shape):
        return torch.empty(shape, device="cuda", dtype=torch.int32)

    if case["kind"] == "route":
        logits = make.logits(tokens, case["experts"])
        if case["padded"]:
            logits[tokens - case["padded"]:] = -math.inf
        state.update(logits=logits if case["f32"] else logits.to(torch.bfloat16), ids=ints(tokens, top_k), offsets=ints(case["experts"] + 1),
                     row_pair=ints(pairs), pair_row=ints(tokens, top_k), weights=torch.empty((tokens, top_k), device="cuda"))
    elif case["kind"] == "experts":
        ids = _picks(make.logits(tokens, case["experts"]), top_k)
        offsets, row_pair, _ = _plan(ids, case["experts"])
        out = case["n"] // 2 if case["gated"] else case["n"]
        state.update(a=make.activations(tokens if case["gather"] else pairs, case["k"]), b=make.weights(case), scale=make.scales(case),
                     zero=make.zeros(case), offsets=offsets, row_pair=row_pair, c=torch.empty((pairs, out), device="cuda", dtype=torch.bfloat16))
    else:
        ids = _picks(make.logits(tokens, 64), top_k)
        if case["padded"]:
            ids[tokens - case["padded"]:] = -1
        weights = torch.softmax(make.normal(tokens, top_k), 1)
        weights[ids < 0] = 0
        state.update(y=make.activations(pairs, case["n"]), weights=weights, pair_row=_plan(ids, 64)[2],
                     residual=make.activations(tokens, case["n"]) if case["residual"] else None,
                     out=torch.empty((tokens, case["n"]), device="cuda", dtype=torch.bfloat16))
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------

def _plain_route(state):
    case, logits = state["case"], state["logits"].float()
    ids = _picks(logits, case["top_k"])
    top = logits.gather(1, ids)
    there = top > -math.inf
    largest = logits.amax(1, keepdim=True)
    largest = torch.where(largest > -math.inf, largest, 0.0)
    every = torch.exp(top - largest) if case["renormalize"] else torch.exp(logits - largest)
    weights = torch.where(there, torch.exp(top - largest) / every.sum(1, keepdim=True), 0.0)
    ids = torch.where(there, ids, -1).int()
    offsets, row_pair, pair_row = _plan(ids, case["experts"])
    return dict(ids=ids, weights=weights, offsets=offsets, row_pair=row_pair, pair_row=pair_row)


def _integers(case, q):
    """Stored integers [..., bytes] -> fp32 values [..., k] in the order of k."""
    if case["bits"] == 8:
        v = (q.view(torch.uint8).float() - 128) if case["offset"] else q.float()
        order = [0, 2, 1, 3]    # place of weight i inside its 32-bit word when pre-packed
    else:
        nib = torch.stack([q & 15, q >> 4], -1).flatten(-2)
        v = nib.float() - 8 if case["offset"] else ((nib ^ 8).float() - 8)
        order = [0, 4, 1, 5, 2, 6, 3, 7]
    if case["packed"]:
        v = v.unflatten(-1, (-1, len(order)))[..., order].flatten(-2)
    return v


def _dequantised(case, b, scale, zero):
    v = _integers(case, b)
    if not case["group"]:
        return v * scale[..., None]
    v = v.unflatten(-1, (-1, case["group"]))
    if zero is not None:
        z = zero.float() - 8 if case["offset"] else (((zero & 15) ^ 8).float() - 8)
        v = v - z[..., None]
    return (v * scale.float()[..., None]).flatten(-2)


def _plain_experts(state):
    case, offsets = state["case"], state["offsets"].long()
    rows = state["row_pair"].numel()
    a = state["a"].float()
    if case["gather"]:
        a = a[state["row_pair"].long() // case["top_k"]]
    place = torch.arange(rows, device=a.device)
    expert = (place[:, None] >= offsets[1:]).sum(1)
    if rows <= case["experts"]:   # no more rows than experts: the weights of every row's expert
        pick = (lambda x: None if x is None else x[expert])
        w = _dequantised(case, pick(state["b"]), pick(state["scale"]), pick(state["zero"]))
        v = torch.bmm(w, a[:, :, None])[:, :, 0]
    else:                         # as many places per expert as the fullest one needs
        most = int((offsets[1:] - offsets[:-1]).max())
        inside = place - offsets[expert]
        padded = torch.zeros((case["experts"], most, case["k"]), device=a.device)
        padded[expert, inside] = a
        w = _dequantised(case, state["b"], state["scale"], state["zero"])
        v = torch.bmm(padded, w.transpose(1, 2))[expert, inside]
    if case["gated"]:
        gate, up = v[:, 0::2], v[:, 1::2]
        v = gate / (1 + torch.exp(-gate)) * up
    return v.to(torch.bfloat16)


def _plain_combine(state):
    row = state["pair_row"].long()
    there = (row >= 0)[..., None]
    terms = torch.where(there, state["y"].float()[row.clamp(min=0)] * state["weights"][..., None], 0.0)
    out = terms.sum(1)
    if state["residual"] is not None:
        out = out + state["residual"].float()
    return out.to(torch.bfloat16)


# ---- the framework's -----------------------------------------------------------------------------------------------------------------------

def _call(state):
    """The library's argument block of this state, as a program that owns its buffers keeps it."""
    import awesome_fusion_b200 as afb
    lib, case = afb.load(), state["case"]
    lib.init(torch.cuda.current_device())
    if case["kind"] == "route":
        scratch = torch.empty(max(1, lib.moe_route_workspace(case["tokens"], case["experts"])), device="cuda", dtype=torch.uint8)
        args = lib.make_moe_route_args(state["logits"], state["ids"], state["weights"], state["offsets"], state["row_pair"], state["pair_row"],
                                       tokens=case["tokens"], experts=case["experts"], top_k=case["top_k"], logits_f32=case["f32"],
                                       renormalize=case["renormalize"], workspace=scratch, workspace_bytes=scratch.numel())
        return lib.moe_route_launch, args, scratch
    if case["kind"] == "experts":
        gemm = lib.make_args(state["c"], state["a"], state["b"], state["scale"], state["c"].shape[0], case["n"], case["k"], ldc=state["c"].shape[1],
                             bits=case["bits"], group=case["group"], zero=state["zero"],
                             layout=afb.LAYOUT_COL_PACKED if case["packed"] else afb.LAYOUT_COL,
                             encoding=afb.ENC_OFFSET if case["offset"] else afb.ENC_TWOS,
                             scale_dtype=afb.SCALE_BF16 if case["group"] else afb.SCALE_F32)
        args = lib.make_expert_gemm_args(gemm, state["offsets"], experts=case["experts"], row_pair=state["row_pair"] if case["gather"] else None,
                                         top_k=case["top_k"] if case["gather"] else 1, a_rows=state["a"].shape[0], gated=case["gated"],
                                         activation=afb.ACT_SILU if case["gated"] else afb.ACT_NONE)
        return lib.expert_gemm_launch, args, None
    args = lib.make_moe_combine_args(state["out"], state["y"], state["weights"], state["pair_row"], tokens=case["tokens"], top_k=case["top_k"],
                                     rows=state["y"].shape[0], n=case["n"], residual=state["residual"])
    return lib.moe_combine_launch, args, None


def run(state):
    kind = state["case"]["kind"]
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        launch, args, _ = state["call"]
        launch(args, state["stream"])
        if kind == "route":
            return {name: state[name] for name in ("ids", "weights", "offsets", "row_pair", "pair_row")}
        return state["c"] if kind == "experts" else state["out"]
    return {"route": _plain_route, "experts": _plain_experts, "combine": _plain_combine}[kind](state)


def work(case):
    tokens, top_k = case["tokens"], case["top_k"]
    pairs = tokens * top_k
    if case["kind"] == "route":
        return {"bytes": tokens * case["experts"] * (4 if case["f32"] else 2) + 16 * pairs + 4 * (case["experts"] + 1), "flops": 0}
    if case["kind"] == "combine":
        # picks of padded tokens are neither read nor added
        real = (tokens - case["padded"]) * top_k
        return {"bytes": real * case["n"] * 2 + pairs * 8 + tokens * case["n"] * (4 if case["residual"] else 2), "flops": 2 * real * case["n"]}
    # how many experts have a row: those that `pairs` picks reach, at most
    active = min(case["experts"], pairs)
    n, k = case["n"], case["k"]
    scales = n * (k // case["group"]) * (3 if case["zero"] else 2) if case["group"] else 4 * n
    return {"bytes": active * (n * k * case["bits"] // 8 + scales) + 2 * k * (tokens if case["gather"] else pairs) +
            2 * pairs * (n // 2 if case["gated"] else n) + 4 * (case["experts"] + 1) + (4 * pairs if case["gather"] else 0),
            "flops": 2 * pairs * n * k}


# ---- in 64 bits, from the definitions --------------------------------------------------------------------------------------------------------

def _exact_experts(state):
    case = state["case"]
    bounds = state["offsets"].tolist()
    token = state["row_pair"].long() // case["top_k"] if case["gather"] else None
    out = torch.empty(state["c"].shape, device="cuda", dtype=torch.float64)
    for e in range(case["experts"]):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        byte = state["b"][e].view(torch.uint8).to(torch.int64)
        # stored integers in the order of the bytes, then weight i from its place
        if case["bits"] == 8:
            stored, word = byte, (lambda i: (i & ~3) | ((i & 3) >> 1) | ((i & 1) << 1))
            low, span = -128, 256
        else:
            stored, word = torch.stack([byte % 16, byte // 16], 2).reshape(byte.shape[0], -1), (lambda i: (i & ~7) | ((i & 7) >> 1) | ((i & 1) << 2))
            low, span = -8, 16

        def value(s):
            return s + low if case["offset"] else torch.where(s >= span // 2, s - span, s)

        if case["packed"]:
            stored = stored[:, word(torch.arange(case["k"], device="cuda"))]
        w = value(stored).double()
        if case["zero"]:
            w -= value(state["zero"][e].to(torch.int64)).double().repeat_interleave(case["group"], 1)
        scale = state["scale"][e].double()
        w *= scale.repeat_interleave(case["group"], 1) if case["group"] else scale[:, None]
        rows = state["a"][token[lo:hi]] if case["gather"] else state["a"][lo:hi]
        v = rows.double() @ w.T
        out[lo:hi] = v[:, 0::2] * torch.sigmoid(v[:, 0::2]) * v[:, 1::2] if case["gated"] else v
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "experts":
        return _exact_experts(state)
    if case["kind"] == "route":
        logits = state["logits"].double()
        picked = torch.topk(logits, case["top_k"], dim=1).values   # weights follow from the values; the picks themselves are whole numbers
        over = picked if case["renormalize"] else logits
        weights = torch.exp(picked - torch.logsumexp(over, 1, keepdim=True)).nan_to_num(0.0)
        return dict(ids=None, weights=weights, offsets=None, row_pair=None, pair_row=None)
    y = torch.cat([state["y"].double(), torch.zeros((1, case["n"]), device="cuda", dtype=torch.float64)])   # the last row stands for -1
    out = torch.einsum("tk,tkn->tn", state["weights"].double(), y[state["pair_row"].long()])
    return out + state["residual"].double() if state["residual"] is not None else out
