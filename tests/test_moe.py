"""Operators of a mixture-of-experts layer on quantised weights against plain 64-bit forms: the router and its plan, the products grouped by
expert (both forms), the weighted sum, and the layer made of them.

Tolerances.  A bf16 result is rounded once: off by at most 2^-8 / 2 of its value where it is a sum in fp32 (bf16 has 8 significant bits, so half a
step is 2^-9 of the next power of two above, at most 2^-8 relative).  In front of that the fp32 sum over k is off by less than 2^-15 of the sum of the
products' absolute values: they are exact (8 x 8 significant bits), a chunk of 64 to 1024 of them is added by the tensor cores, which keep at
least 2^-23 of the largest term each, and a few hundred sums in fp32 follow.  So |got - want| <= 2^-8 |want| + 2^-15 sum |a w|.
The form for many rows multiplies weight and group scale in fp16, whose rounding is off by at most 2^-11: none where the product fits (int4 without zero-points,
three significant bits times the eight of a bf16 scale), once otherwise, and once more for an fp32 scale that is rounded to fp16 itself: 2^-11 sum |a w| each.
"""
import ctypes
import math

import numpy as np
import pytest

import awesome_fusion_b200 as pkg

torch = pytest.importorskip("torch")

E_BAD, E_UNSUPPORTED, E_LARGE = -1, -2, -6
PTR = 0x10000


# ---- refusals, on the CPU ------------------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def lib():
    return pkg.load()


def _route(lib, **changes):
    args = lib.make_moe_route_args(PTR, PTR, PTR, PTR, PTR, PTR, tokens=100, experts=64, top_k=8, workspace=PTR, workspace_bytes=1 << 20)
    for name, value in changes.items():
        setattr(args, name, value)
    return lib.moe_route_launch_status(args)


def test_abi_sizes(lib):
    sizes = (ctypes.c_uint32 * 3)()
    assert lib.lib.afb_moe_abi_sizes(sizes) == 0
    assert list(sizes) == [ctypes.sizeof(t) for t in (pkg.MoeRouteArgs, pkg.ExpertGemmArgs, pkg.MoeCombineArgs)]
    assert lib.lib.afb_moe_abi_sizes(None) == E_BAD


@pytest.mark.parametrize("changes", [dict(ptr_logits=0), dict(ptr_ids=0), dict(ptr_weights=0), dict(ptr_offsets=0), dict(ptr_row_pair=0), dict(ptr_pair_row=0),
                                     dict(ptr_workspace=0), dict(workspace_bytes=8), dict(ptr_workspace=PTR + 2), dict(ptr_ids=PTR + 1), dict(ptr_logits=PTR + 1),
                                     dict(logits_f32=1, ptr_logits=PTR + 2), dict(experts=0), dict(experts=1025, ld_logits=1025), dict(top_k=0), dict(top_k=33),
                                     dict(experts=4, top_k=5), dict(ld_logits=63), dict(logits_f32=2), dict(renormalize=2), dict(reserved=1)])
def test_route_refuses(lib, changes):
    assert _route(lib, **changes) == E_BAD


def test_route_sizes(lib):
    assert _route(lib, tokens=1 << 30) == E_LARGE
    assert lib.moe_route_workspace(1, 64) == 0 and lib.moe_route_workspace(0, 64) == 0
    assert lib.moe_route_workspace(4096, 128) == 128 * 128 * 4
    assert lib.lib.afb_moe_route_workspace(1, 0, ctypes.byref(ctypes.c_uint64())) == E_BAD
    assert lib.lib.afb_moe_route_workspace(1, 1025, ctypes.byref(ctypes.c_uint64())) == E_BAD
    assert lib.lib.afb_moe_route_workspace(1, 8, None) == E_BAD


def _expert(lib, gemm=None, **changes):
    g = lib.make_args(PTR, PTR, PTR, PTR, 16, 256, 512)
    for name, value in (gemm or {}).items():
        setattr(g, name, value)
    args = lib.make_expert_gemm_args(g, PTR, experts=8, row_pair=PTR, top_k=2, a_rows=8)
    for name, value in changes.items():
        setattr(args, name, value)
    return lib.expert_gemm_launch_status(args)


@pytest.mark.parametrize("gemm, changes", [
    (dict(ptr_c=0), {}), (dict(ptr_a=0), {}), (dict(ptr_b=0), {}), (dict(ptr_scale=0), {}), (dict(n=0), {}), (dict(k=0), {}), (dict(lda=504), {}),
    (dict(ldb=256), {}), (dict(ldc=255), {}), (dict(b_bits=3), {}), (dict(b_encoding=2), {}), (dict(b_layout=3), {}), (dict(scale_dtype=2), {}),
    (dict(variant=4), {}), (dict(reserved=1), {}), (dict(reserved2=1), {}), (dict(group_size=96), {}), (dict(ptr_scale=PTR + 2), {}),
    (dict(ptr_c=PTR + 1), {}), (dict(ptr_a=PTR + 1), {}), ({}, dict(ptr_offsets=0)), ({}, dict(ptr_offsets=PTR + 2)), ({}, dict(ptr_row_pair=PTR + 1)),
    ({}, dict(experts=0)), ({}, dict(experts=1025)), ({}, dict(top_k=0)), ({}, dict(ptr_row_pair=0)), ({}, dict(gated=2)), ({}, dict(activation=2)),
    ({}, dict(reserved=1)), (dict(n=255, ldc=255), dict(gated=1)), ({}, dict(ptr_row_pair=0, top_k=1, a_rows=15)), ({}, dict(a_rows=0))])
def test_expert_gemm_refuses(lib, gemm, changes):
    assert _expert(lib, gemm, **changes) == E_BAD


@pytest.mark.parametrize("gemm", [dict(b_layout=pkg.LAYOUT_ROW), dict(variant=pkg.VARIANT_NAIVE), dict(flags=pkg.FLAG_C_F32), dict(flags=pkg.FLAG_PDL),
                                  dict(k=480, lda=512, ldb=512), dict(b_bits=4, k=448, lda=512, ldb=512), dict(lda=516), dict(ldb=520), dict(ptr_a=PTR + 8),
                                  dict(ptr_b=PTR + 4), dict(group_size=32), dict(k=576, lda=576, ldb=576, group_size=192)])
def test_expert_gemm_does_not_cover(lib, gemm):
    assert _expert(lib, gemm) == E_UNSUPPORTED


def test_expert_gemm_sizes(lib):
    assert _expert(lib, dict(m=1 << 31)) == E_LARGE
    assert _expert(lib, {}, a_rows=1 << 31) == E_LARGE
    assert _expert(lib, dict(n=1 << 28, ldc=1 << 28)) == E_LARGE
    assert _expert(lib, dict(k=1 << 24, lda=1 << 24, ldb=1 << 24)) == E_LARGE


def _combine(lib, **changes):
    args = lib.make_moe_combine_args(PTR, 2 * PTR, PTR, PTR, tokens=10, top_k=2, rows=20, n=64, residual=3 * PTR)
    for name, value in changes.items():
        setattr(args, name, value)
    return lib.moe_combine_launch_status(args)


@pytest.mark.parametrize("changes", [dict(ptr_out=0), dict(ptr_y=0), dict(ptr_weights=0), dict(ptr_pair_row=0), dict(ptr_out=PTR + 1), dict(ptr_y=PTR + 1),
                                     dict(ptr_residual=PTR + 1), dict(ptr_weights=PTR + 2), dict(ptr_pair_row=PTR + 2), dict(top_k=0), dict(n=0), dict(ld_out=63),
                                     dict(ld_y=63), dict(ld_residual=63), dict(reserved=1), dict(ptr_y=PTR), dict(ptr_residual=PTR, ld_residual=72)])
def test_combine_refuses(lib, changes):
    assert _combine(lib, **changes) == E_BAD


def test_torch_operators_infer_shapes_and_have_no_cpu_path():
    import awesome_fusion_b200.torch_op  # noqa: F401
    ops, meta = torch.ops.afb, dict(device="meta")
    weights, ids, offsets, row_pair, pair_row = ops.moe_route(torch.empty((5, 16), **meta), 3, True)
    assert [t.shape for t in (weights, ids, offsets, row_pair, pair_row)] == [(5, 3), (5, 3), (17,), (15,), (5, 3)]
    assert weights.dtype == torch.float32 and {t.dtype for t in (ids, offsets, row_pair, pair_row)} == {torch.int32}
    a, b, scale = torch.empty((5, 256), dtype=torch.bfloat16, **meta), torch.empty((16, 64, 128), dtype=torch.uint8, **meta), torch.empty((16, 64, 2), dtype=torch.bfloat16, **meta)
    assert ops.expert_gemm(a, b, scale, None, offsets, row_pair, 3, 4, 128, False, False, True).shape == (15, 32)
    assert ops.expert_gemm(a, b, scale, None, offsets, None, 1, 4, 128, False).shape == (5, 64)
    assert ops.moe_combine(torch.empty((15, 64), dtype=torch.bfloat16, **meta), weights, pair_row).shape == (5, 64)
    for bad in ((a, b, scale[:, :, :1], None, offsets, None, 1, 4, 128, False), (a, b, scale, None, offsets, None, 2, 4, 128, False), (a, b, scale, None, offsets[:5], None, 1, 4, 128, False)):
        with pytest.raises(Exception):
            ops.expert_gemm(*bad)
    for bad in ((torch.empty((5, 16), **meta), 17, True), (torch.empty((5, 16), **meta), 0, True), (torch.empty((5, 1025), **meta), 2, True)):
        with pytest.raises(Exception):
            ops.moe_route(*bad)
    with pytest.raises(Exception):
        ops.moe_route(torch.zeros((2, 4)), 1, True)
    with pytest.raises(Exception):
        ops.moe_combine(torch.zeros((2, 8), dtype=torch.bfloat16), torch.zeros((1, 2)), torch.zeros((1, 2), dtype=torch.int32))


# ---- plain forms in 64 bits -------------------------------------------------------------------------------------------------------------------

def plain_route(logits, top_k, renormalize):
    """numpy, token by token."""
    logits = np.asarray(logits, dtype=np.float64)
    tokens, experts = logits.shape
    ids, weights = np.full((tokens, top_k), -1, np.int64), np.zeros((tokens, top_k))
    for t in range(tokens):
        x = np.where(np.isnan(logits[t]), -np.inf, logits[t])
        order = [e for e in np.argsort(-x, kind="stable") if x[e] > -np.inf]
        if not order:
            continue
        terms = np.array([1.0 if x[e] == x[order[0]] else math.exp(x[e] - x[order[0]]) for e in order])
        picked = order[:top_k]
        ids[t, : len(picked)] = picked
        weights[t, : len(picked)] = terms[: len(picked)] / (terms[: len(picked)] if renormalize else terms).sum()
    flat = ids.reshape(-1)
    rows = [p for e in range(experts) for p in np.nonzero(flat == e)[0]]
    offsets = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(experts)])])
    row_pair, pair_row = np.full(flat.size, -1), np.full(flat.size, -1)
    row_pair[: len(rows)] = rows
    pair_row[rows] = np.arange(len(rows))
    return ids, weights, offsets, row_pair, pair_row.reshape(ids.shape)


def pack_words(q, bits):
    """[.., k] stored integers in the pre-packed order of every 32-bit word."""
    per = 32 // bits
    order = [0, 2, 1, 3] if bits == 8 else [0, 2, 4, 6, 1, 3, 5, 7]
    return q.reshape(*q.shape[:-1], -1, per)[..., order].reshape(q.shape)


class Experts:
    """Weights of `experts` matrices on the GPU with their values in 64 bits."""

    def __init__(self, experts, n, k, bits, group=0, zero=False, offset=False, packed=False, scale_f32=None, seed=0):
        rng = np.random.default_rng(seed)
        span, half = (256, 128) if bits == 8 else (16, 8)
        stored = rng.integers(0, span, (experts, n, k))
        value = (lambda s: s - half if offset else np.where(s >= half, s - span, s))
        w = value(stored).astype(np.float64)
        shape = (experts, n, k // group) if group else (experts, n)
        scale = rng.uniform(0.002, 0.02, shape).astype(np.float32)
        f32 = (not group) if scale_f32 is None else scale_f32
        self.scale = torch.tensor(scale) if f32 else torch.tensor(scale).bfloat16()
        self.zero = None
        spread = (lambda x: np.repeat(x, group, 2) if group else x[..., None])
        if zero:
            z = rng.integers(0, span, shape)
            w -= spread(value(z).astype(np.float64))
            self.zero = torch.tensor(z.astype(np.uint8)).cuda()
        self.w = torch.tensor(w * spread(self.scale.double().numpy())).cuda()
        if packed:
            stored = pack_words(stored, bits)
        q = stored.astype(np.uint8)
        if bits == 4:
            q = q[..., 0::2] | (q[..., 1::2] << 4)
        self.b, self.scale = torch.tensor(q).cuda(), self.scale.cuda()
        self.experts, self.n, self.k, self.bits, self.group, self.offset, self.packed = experts, n, k, bits, group, offset, packed

    def plain(self, a, offsets, row_pair=None, top_k=1, gated=False, variant=pkg.VARIANT_AUTO):
        """(result, bound of the error) in 64 bits; rows behind the last one: zero and zero."""
        f32 = self.scale.dtype == torch.float32
        roundings = 0 if not self.group or variant == pkg.VARIANT_DECODE else int(self.bits == 8 or self.zero is not None or f32) + int(f32)
        rows = a.shape[0] if row_pair is None else row_pair.numel()
        out = torch.zeros((rows, self.n // 2 if gated else self.n), dtype=torch.float64, device="cuda")
        off = torch.zeros_like(out)
        bounds = offsets.tolist()
        for e in range(self.experts):
            lo, hi = bounds[e], bounds[e + 1]
            if hi <= lo:
                continue
            x = (a[lo:hi] if row_pair is None else a[row_pair[lo:hi].long() // top_k]).double()
            v, s = x @ self.w[e].T, (x.abs() @ self.w[e].abs().T) * (2.0 ** -15 + roundings * 2.0 ** -11)
            if gated:
                # d(silu) <= 1.1 d(gate); the exponential and the division are off by a few 2^-22 of silu(gate)
                g, u = v[:, 0::2], v[:, 1::2]
                act = g * torch.sigmoid(g)
                v, s = act * u, 1.1 * s[:, 0::2] * (u.abs() + s[:, 1::2]) + (act.abs() + 1.1 * s[:, 0::2]) * s[:, 1::2] + 2.0 ** -18 * (act * u).abs()
            out[lo:hi], off[lo:hi] = v, s + 2.0 ** -8 * (v.abs() + s)
        return out, off

    def run(self, afb, a, offsets, row_pair=None, top_k=1, gated=False, variant=pkg.VARIANT_AUTO, rows=None, ldc=None, out=None, silu=None, stream=None):
        rows = rows or (a.shape[0] if row_pair is None else row_pair.numel())
        n_out = self.n // 2 if gated else self.n
        if out is None:
            out = torch.full((rows, ldc or n_out), 777.0, dtype=torch.bfloat16, device="cuda")
        gemm = afb.make_args(out, a, self.b, self.scale, rows, self.n, self.k, lda=a.stride(0), ldc=out.stride(0), bits=self.bits, group=self.group, zero=self.zero,
                             layout=pkg.LAYOUT_COL_PACKED if self.packed else pkg.LAYOUT_COL, encoding=pkg.ENC_OFFSET if self.offset else pkg.ENC_TWOS,
                             scale_dtype=pkg.SCALE_BF16 if self.scale.dtype == torch.bfloat16 else pkg.SCALE_F32, variant=variant)
        silu = gated if silu is None else silu
        afb.expert_gemm_launch(afb.make_expert_gemm_args(gemm, offsets, experts=self.experts, row_pair=row_pair, top_k=top_k, a_rows=a.shape[0], gated=gated,
                                                         activation=pkg.ACT_SILU if silu else pkg.ACT_NONE), stream)
        return out


def check(got, want, off):
    rounded = want.to(got.dtype)
    over = rounded.isinf()   # above the largest bf16: infinity is the result
    bad = torch.where(over, got != rounded, (got.double() - want).abs() > off)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} too far off, first at {bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]} +- {off[bad][0]}"


def offsets_of(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")


def activations(rows, k, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((rows, k), generator=gen).bfloat16().cuda()


# ---- the router -------------------------------------------------------------------------------------------------------------------------------

def run_route(afb, logits, top_k, renormalize, ld=None):
    tokens, experts = logits.shape
    i32 = dict(dtype=torch.int32, device="cuda")
    ids, offsets, row_pair, pair_row = (torch.full(s, 99, **i32) for s in ((tokens, top_k), (experts + 1,), (tokens * top_k,), (tokens, top_k)))
    weights = torch.full((tokens, top_k), 99.0, device="cuda")
    work = torch.empty(afb.moe_route_workspace(tokens, experts), dtype=torch.uint8, device="cuda")
    afb.moe_route_launch(afb.make_moe_route_args(logits, ids, weights, offsets, row_pair, pair_row, tokens=tokens, experts=experts, top_k=top_k, ld_logits=ld,
                                                 logits_f32=logits.dtype == torch.float32, renormalize=renormalize, workspace=work, workspace_bytes=work.numel()))
    torch.cuda.synchronize()
    return ids, weights, offsets, row_pair, pair_row


@pytest.mark.gpu
@pytest.mark.parametrize("tokens, experts, top_k", [(1, 1, 1), (1, 8, 8), (1, 64, 8), (3, 33, 5), (64, 8, 8), (65, 8, 8), (16, 128, 32), (17, 1024, 32), (200, 7, 3),
                                                    (1000, 257, 4), (4097, 64, 2), (5000, 512, 8)])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_route(afb, tokens, experts, top_k, kind):
    gen = torch.Generator().manual_seed(tokens + experts)
    logits = torch.randn((tokens, experts), generator=gen) * 2 + torch.randn(experts, generator=gen)
    # bf16 and the coarse grid make ties; masked logits; tokens of padding; infinities
    logits = logits.bfloat16() if kind == "bf16" else (logits * 4).round() / 4
    if experts > 2:
        logits[::3, 1] = -math.inf
        logits[1::5, experts - 1] = math.nan
        logits[2::7, 2] = math.inf
        logits[3::11, :2] = math.inf
        logits[4::13] = -0.0
        logits[4::13, 2] = 0.0
        logits[6::9, 1:] = -math.inf
    if tokens > 2:
        logits[tokens // 2: tokens // 2 + 2] = -math.inf
    for renormalize in (True, False):
        got = run_route(afb, logits.cuda(), top_k, renormalize)
        want = plain_route(logits.double().numpy(), top_k, renormalize)
        for i, name in ((0, "ids"), (2, "offsets"), (3, "row_pair"), (4, "pair_row")):
            assert np.array_equal(got[i].cpu().numpy(), want[i]), name
        # exp: 2 steps of 2^-24 and the difference in its argument (up to 30 here): 30 * 2^-24; a sum of up to 1024 terms, a division
        assert np.allclose(got[1].cpu().numpy(), want[1], rtol=2.0 ** -17, atol=1e-30)


@pytest.mark.gpu
def test_route_strides_and_empty(afb):
    wide = torch.randn((50, 96), device="cuda")
    part = wide[:, 16:80]
    got, want = run_route(afb, part, 4, True, ld=96), run_route(afb, part.contiguous(), 4, True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    offsets = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    afb.moe_route_launch(afb.make_moe_route_args(None, None, None, offsets, None, None, tokens=0, experts=8, top_k=2))
    assert offsets.tolist() == [0] * 9


# ---- the products -----------------------------------------------------------------------------------------------------------------------------

FORMS = [pkg.VARIANT_DECODE, pkg.VARIANT_PREFILL]
FORMATS = [dict(bits=8), dict(bits=8, offset=True, packed=True), dict(bits=8, zero=True), dict(bits=8, group=64), dict(bits=8, group=128, zero=True, packed=True),
           dict(bits=4), dict(bits=4, group=128, packed=True), dict(bits=4, group=64, zero=True, offset=True), dict(bits=4, group=256, scale_f32=True),
           dict(bits=4, group=64, packed=True), dict(bits=4, zero=True, offset=True), dict(bits=8, group=512, scale_f32=True, zero=True, offset=True)]


@pytest.mark.gpu
@pytest.mark.parametrize("variant", FORMS)
@pytest.mark.parametrize("fmt", FORMATS, ids=lambda f: "-".join(f"{k}{v}" for k, v in f.items()))
@pytest.mark.parametrize("gated", [False, True])
def test_expert_gemm_formats(afb, variant, fmt, gated):
    x = Experts(5, 200, 512, seed=3, **fmt)
    counts = [3, 0, 37, 1, 150]
    pairs = sum(counts)
    row_pair = torch.randperm(pairs, generator=torch.Generator().manual_seed(2)).int().cuda()
    a = activations((pairs + 2) // 3, 512)
    offsets = offsets_of(counts)
    got = x.run(afb, a, offsets, row_pair, 3, gated, variant)
    check(got, *x.plain(a, offsets, row_pair, 3, gated, variant))
    assert afb.read_status()[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("variant", FORMS)
@pytest.mark.parametrize("counts", [[1], [0, 0, 1, 0], [8, 9, 16, 17], [31, 32, 33, 0, 1], [300, 0, 0, 1, 127, 128, 129], [0, 0, 0, 0], [1] * 40, [700, 2]],
                         ids=lambda c: "x".join(map(str, c[:7])))
def test_expert_gemm_ragged(afb, variant, counts):
    """Ragged sizes with rows behind the last one, which stay as they are; every 128-channel edge."""
    for n, k, fmt in ((130, 1024, dict(bits=4, group=128)), (72, 192, dict(bits=8))):
        x = Experts(len(counts), n, k, seed=5, **fmt)
        rows = sum(counts) + 5
        a, offsets = activations(rows, k), offsets_of(counts)
        got = x.run(afb, a, offsets, variant=variant, ldc=n + 3)
        want, off = x.plain(a, offsets, variant=variant)
        check(got[: rows - 5, :n], want[: rows - 5], off[: rows - 5])
        assert (got[rows - 5:] == 777).all() and (got[:, n:] == 777).all()
    assert afb.read_status()[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("variant", FORMS)
@pytest.mark.parametrize("n, k, bits, group", [(1, 64, 8, 0), (7, 128, 4, 128), (128, 128, 4, 64), (129, 4160, 8, 64), (256, 14336, 4, 128), (3000, 192, 8, 0), (130, 8192, 8, 0), (40, 16512, 8, 64),
                                              (200, 320, 8, 64), (200, 128, 8, 0), (64, 16640, 4, 64)])
def test_expert_gemm_sizes_on_gpu(afb, variant, n, k, bits, group):
    x = Experts(3, n, k, bits, group, seed=7)
    counts = [20, 5, 61]
    a, offsets = activations(sum(counts), k), offsets_of(counts)
    check(x.run(afb, a, offsets, variant=variant), *x.plain(a, offsets, variant=variant))
    assert afb.read_status()[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("variant", FORMS)
def test_expert_gemm_strides_and_values(afb, variant):
    """Pitches of A and C, odd alignment of C, activation without gate, fp32 scales of groups, infinities and NaN in other rows."""
    x = Experts(4, 136, 256, 4, 128, seed=9)
    counts = [2, 40, 0, 9]
    offsets, rows = offsets_of(counts), 51
    wide = activations(rows, 512)
    a = wide[:, 128:384]
    want, off = x.plain(a, offsets)
    buf = torch.full((rows * 141 + 1,), 777.0, dtype=torch.bfloat16, device="cuda")
    out = buf[1:].view(rows, 141)
    check(x.run(afb, a, offsets, variant=variant, out=out)[:, :136], want, off)
    got = x.run(afb, a, offsets, variant=variant, silu=True)
    s = want * torch.sigmoid(want)
    check(got, s, 1.1 * off + 2.0 ** -8 * s.abs())
    # rows 5 and 50 are NaN and infinite: the others do not change
    plain = x.run(afb, a, offsets, variant=variant)
    a[5], a[50] = math.nan, math.inf
    got = x.run(afb, a, offsets, variant=variant)
    keep = [r for r in range(rows) if r not in (5, 50)]
    assert torch.equal(got[keep], plain[keep]) and got[5].isnan().all() and not got[50].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("variant", FORMS)
@pytest.mark.parametrize("fmt", [dict(bits=8), dict(bits=4, group=64, packed=True)], ids=lambda f: f"int{f['bits']}")
def test_expert_gemm_pitch_of_weights_and_odd_gates(afb, variant, fmt):
    """Rows of B with a pitch, an odd number of gated channels (no 4- or 8-byte store fits), a first row that is not row 0."""
    x = Experts(3, 130, 384, seed=23, **fmt)
    offsets = torch.tensor([4, 24, 24, 90], dtype=torch.int32, device="cuda")
    a = activations(90, 384)
    for gated in (False, True):
        want = x.run(afb, a, offsets, gated=gated, variant=variant)
        plain, off = x.plain(a, offsets, gated=gated, variant=variant)
        check(want[4:], plain[4:], off[4:])
        assert (want[:4] == 777).all()
        wide = torch.randint(0, 255, (3, 130, x.b.shape[2] + 64), device="cuda").to(torch.uint8)
        wide[:, :, : x.b.shape[2]] = x.b
        out = torch.full_like(want, 777.0)
        gemm = afb.make_args(out, a, wide, x.scale, 90, 130, 384, ldb=wide.shape[2] * 8 // x.bits, ldc=out.shape[1], bits=x.bits, group=x.group,
                             layout=pkg.LAYOUT_COL_PACKED if x.packed else pkg.LAYOUT_COL, variant=variant,
                             scale_dtype=pkg.SCALE_BF16 if x.group else pkg.SCALE_F32)
        afb.expert_gemm_launch(afb.make_expert_gemm_args(gemm, offsets, experts=3, gated=gated, activation=pkg.ACT_SILU if gated else pkg.ACT_NONE))
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", FORMS)
def test_expert_gemm_takes_bad_plans(afb, variant):
    """Rows of A that do not exist read as zeros, offsets outside 0 .. m as the nearer end: nothing is read or written out of bounds."""
    x = Experts(3, 64, 256, 8, seed=11)
    a = activations(4, 256)
    row_pair = torch.tensor([0, -1, 3, 4, 2 ** 31 - 1, 1, 2, 3], dtype=torch.int32, device="cuda")
    got = x.run(afb, a, offsets_of([3, 3, 2]), row_pair, 1, variant=variant)
    assert (got[[1, 3, 4]] == 0).all()
    keep = [0, 2, 5, 6, 7]
    want, off = x.plain(a, offsets_of([3, 3, 2]), row_pair.clamp(0, 3))
    check(got[keep], want[keep], off[keep])
    guard = torch.full((20, 64), 777.0, dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([-5, 3, 6, 1000], dtype=torch.int32, device="cuda")
    x.run(afb, a, offsets, row_pair, 1, variant=variant, rows=8, out=guard[6:14])
    assert torch.equal(guard[6:14], got) and (guard[:6] == 777).all() and (guard[14:] == 777).all()
    assert afb.read_status()[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("variant", FORMS)
@pytest.mark.parametrize("fmt", [dict(bits=4, group=128), dict(bits=8, group=64, zero=True), dict(bits=8), dict(bits=4, zero=True, group=64, packed=True)],
                         ids=lambda f: "-".join(f"{k}{v}" for k, v in f.items()))
def test_expert_gemm_ranges(afb, variant, fmt):
    """Rows of A from 2^-90 to 2^90, with one value far above the others, of zeros; channels whose scales differ by powers of two, are negative or zero."""
    x = Experts(3, 140, 512, seed=15, **fmt)
    counts = [40, 3, 50]
    offsets, a = offsets_of(counts), activations(sum(counts), 512)
    a = (a.float() * 2.0 ** torch.linspace(-90, 90, a.shape[0], device="cuda").round()[:, None]).bfloat16()
    a[4] = 0
    a[7, 100] = a[7, 100].abs().clamp(min=2.0 ** -80) * 2.0 ** 20
    a[60, 3] = 2.0 ** 120
    factor = 2.0 ** torch.randint(-7, 8, x.scale.shape, generator=torch.Generator().manual_seed(1)).cuda().float()
    factor[:, ::9] *= -1
    factor[:, 5] = 0
    x.scale = (x.scale.float() * factor).to(x.scale.dtype)
    x.w = x.w * (factor.double().repeat_interleave(x.group, 2) if x.group else factor.double()[..., None])
    want, off = x.plain(a, offsets, variant=variant)
    # what fp16 loses at the ends of its range: 2^-40 of the row's largest value, times the weights; a scale keeps all its bits (2^14 between them)
    for e in range(3):
        lo, hi = sum(counts[:e]), sum(counts[: e + 1])
        off[lo:hi] += 2.0 ** -40 * a[lo:hi].double().abs().amax(1, keepdim=True) * x.w[e].abs().sum(1)
    check(x.run(afb, a, offsets, variant=variant), want, off)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", FORMS)
@pytest.mark.parametrize("bits, group", [(4, 128), (8, 0), (8, 64)])
def test_expert_gemm_of_many_experts(afb, variant, bits, group):
    """The table of 1000 experts, most of them without a row."""
    x = Experts(1000, 24, 256, bits, group, seed=17)
    rng = np.random.default_rng(3)
    counts = np.where(rng.random(1000) < 0.1, rng.integers(1, 20, 1000), 0)
    counts[[0, 999]] = 1, 300
    offsets, a = offsets_of(counts), activations(int(counts.sum()), 256)
    check(x.run(afb, a, offsets, variant=variant), *x.plain(a, offsets, variant=variant))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", FORMS)
@pytest.mark.parametrize("fmt", [dict(bits=8), dict(bits=8, group=64), dict(bits=4, group=128, packed=True)], ids=lambda f: "-".join(f"{k}{v}" for k, v in f.items()))
def test_expert_gemm_after_a_call_full_of_nan(afb, variant, fmt):
    """Where a strip has places for more rows than the expert has, shared memory holds what an earlier launch left there: rows of NaN here."""
    x = Experts(8, 2304, 1024, seed=23, **fmt)
    full, counts = [32] * 8, [1, 5, 17, 0, 31, 2, 3, 9]
    offsets, a = offsets_of(counts), activations(sum(counts), 1024)
    want = x.plain(a, offsets, variant=variant)
    assert x.run(afb, torch.full((sum(full), 1024), math.nan, device="cuda", dtype=torch.bfloat16), offsets_of(full), variant=variant).isnan().all()
    check(x.run(afb, a, offsets, variant=variant), *want)
    assert afb.read_status()[0] == 0


@pytest.mark.gpu
def test_expert_gemm_without_workspace(afb):
    """cudaStreamPerThread names no stream to keep a workspace for: the form for few rows takes what would need one."""
    x = Experts(2, 72, 256, 4, 128, seed=19)
    offsets, a = offsets_of([90, 30]), activations(120, 256)
    got = x.run(afb, a, offsets, variant=pkg.VARIANT_PREFILL, stream=2)
    torch.cuda.synchronize()
    assert torch.equal(got, x.run(afb, a, offsets, variant=pkg.VARIANT_DECODE))


@pytest.mark.gpu
def test_expert_gemm_in_two_graphs_at_once(afb):
    """Two captured graphs, and the stream that they were captured on, at the same time: each has a workspace of its own."""
    x = Experts(8, 264, 1024, 4, 128, seed=21)
    counts = [100, 3, 260, 0, 40, 77, 1, 90]
    offsets, rows = offsets_of(counts), sum(counts)
    inputs = [activations(rows, 1024, seed=s) for s in range(3)]
    want = [x.run(afb, a, offsets, variant=pkg.VARIANT_PREFILL) for a in inputs]
    outs, graphs, stream = [torch.zeros_like(w) for w in want], [], torch.cuda.Stream()
    for a, out in list(zip(inputs, outs))[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            x.run(afb, a, offsets, variant=pkg.VARIANT_PREFILL, out=out, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                graph.replay()
        x.run(afb, inputs[2], offsets, variant=pkg.VARIANT_PREFILL, out=outs[2], stream=stream.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(w, o) for w, o in zip(want, outs))


@pytest.mark.gpu
def test_expert_gemm_same_bits_twice_and_side_by_side(afb):
    """Two streams at once, the same plan: the same bits as one after the other."""
    x = Experts(16, 520, 1024, 4, 128, seed=13)
    counts = [5, 40, 0, 1, 77, 130, 2, 2, 9, 33, 17, 0, 64, 3, 8, 100]
    offsets, a = offsets_of(counts), activations(sum(counts), 1024)
    for variant in FORMS:
        once = x.run(afb, a, offsets, variant=variant)
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = [torch.empty_like(once) for _ in range(8)]
        torch.cuda.synchronize()
        for i, out in enumerate(outs):
            x.run(afb, a, offsets, variant=variant, out=out, stream=streams[i % 2].cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(once, out) for out in outs)


# ---- the weighted sum ---------------------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("tokens, top_k, n", [(1, 1, 1), (1, 8, 4096), (5, 3, 1001), (300, 9, 264), (70000, 2, 8), (7, 32, 1032)])
@pytest.mark.parametrize("residual", [False, True])
def test_combine(afb, tokens, top_k, n, residual):
    gen = torch.Generator().manual_seed(n)
    rows = tokens * top_k
    y = torch.randn((rows, n), generator=gen).bfloat16().cuda()
    weights = torch.rand((tokens, top_k), generator=gen).cuda()
    pair_row = torch.randperm(rows, generator=gen).int().reshape(tokens, top_k).cuda()
    pair_row[::3, 0] = -1
    pair_row[tokens // 2] = -1
    pair_row[0, top_k - 1] = rows + 3
    weights[::3, 0] = math.nan      # of a pair without a row
    extra = torch.randn((tokens, n), generator=gen).bfloat16().cuda() if residual else None
    out = torch.full((tokens, n), 777.0, dtype=torch.bfloat16, device="cuda")
    afb.moe_combine_launch(afb.make_moe_combine_args(out, y, weights, pair_row, tokens=tokens, top_k=top_k, rows=rows, n=n, residual=extra))
    there = ((pair_row >= 0) & (pair_row < rows))[..., None]
    terms = torch.where(there, y.double()[pair_row.long().clamp(0, rows - 1)] * weights.double()[..., None], 0.0)
    want, size = terms.sum(1), terms.abs().sum(1)
    if residual:
        want, size = want + extra.double(), size + extra.double().abs()
    check(out, want, 2.0 ** -8 * want.abs() + (top_k + 2) * 2.0 ** -23 * size)
    if residual:   # in place
        afb.moe_combine_launch(afb.make_moe_combine_args(extra, y, weights, pair_row, tokens=tokens, top_k=top_k, rows=rows, n=n, residual=extra))
        assert torch.equal(extra, out)


@pytest.mark.gpu
def test_combine_strides_and_empty(afb):
    y, out, extra = (torch.randn((6, 80), device="cuda").bfloat16() for _ in range(3))
    weights, pair_row = torch.rand((3, 2), device="cuda"), torch.tensor([[0, 5], [2, -1], [4, 1]], dtype=torch.int32, device="cuda")
    plain = torch.empty((3, 60), dtype=torch.bfloat16, device="cuda")
    afb.moe_combine_launch(afb.make_moe_combine_args(plain, y[:, 10:70].contiguous(), weights, pair_row, tokens=3, top_k=2, rows=6, n=60,
                                                     residual=extra[:3, 10:70].contiguous()))
    before = out.clone()
    afb.moe_combine_launch(afb.make_moe_combine_args(out[:, 3:], y[:, 10:], weights, pair_row, tokens=3, top_k=2, rows=6, n=60, ld_out=80, ld_y=80,
                                                     residual=extra[:, 10:], ld_residual=80))
    assert torch.equal(out[:3, 3:63], plain)
    out[:3, 3:63] = before[:3, 3:63]
    assert torch.equal(out, before)
    afb.moe_combine_launch(afb.make_moe_combine_args(None, None, None, None, tokens=0, top_k=2, rows=0, n=60))
    x = Experts(2, 16, 64, 8)
    afb.expert_gemm_launch(afb.make_expert_gemm_args(afb.make_args(None, None, x.b, x.scale, 0, 16, 64), offsets_of([0, 0]), experts=2))


# ---- the layer ------------------------------------------------------------------------------------------------------------------------------------

def plain_layer(x, logits, first, second, top_k, renormalize, residual):
    """64 bits, with h and y rounded to bf16 where the layer keeps them so; the bound of the rounding that may fall either way."""
    ids, weights, offsets, row_pair, pair_row = plain_route(logits.double().cpu().numpy(), top_k, renormalize)
    offsets, row_pair = torch.tensor(offsets).int().cuda(), torch.tensor(row_pair).cuda()
    rows = int(offsets[-1])
    h, h_off = first.plain(x, offsets, row_pair, top_k, True)
    hq = h.bfloat16().double()
    y, y_off = second.plain(hq.bfloat16(), offsets)
    for e in range(second.experts):   # h may be a step off where its sum lies next to the middle of two bf16
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        y_off[lo:hi] += (h_off[lo:hi] + (hq - h)[lo:hi].abs()) @ second.w[e].abs().T
    out, off = torch.zeros(x.shape[0], second.n, dtype=torch.float64, device="cuda"), None
    off = torch.zeros_like(out)
    w = torch.tensor(weights).cuda()
    for j in range(top_k):
        row = torch.tensor(pair_row[:, j]).cuda()
        there = (row >= 0)[:, None]
        out += torch.where(there, y[row.clamp(min=0)] * w[:, j, None], 0.0)
        off += torch.where(there, (y_off[row.clamp(min=0)] + 2.0 ** -8 * y[row.clamp(min=0)].abs()) * w[:, j, None], 0.0)
    if residual is not None:
        out += residual.double()
    assert rows <= row_pair.numel()
    return out, off + 2.0 ** -8 * (out.abs() + off)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens, fmt", [(1, dict(bits=4, group=128, packed=True)), (7, dict(bits=8)), (150, dict(bits=4, group=64, zero=True)), (600, dict(bits=8, group=128))])
def test_layer(afb, tokens, fmt):
    from awesome_fusion_b200 import torch_op
    experts, k, f, top_k = 12, 512, 384, 3
    first, second = Experts(experts, 2 * f, k, seed=1, **fmt), Experts(experts, k, f, seed=2, **fmt)
    x, residual = activations(tokens, k), activations(tokens, k, seed=4)
    logits = activations(tokens, experts, seed=5)
    if tokens > 5:
        logits[tokens - 3:] = -math.inf   # padding
        logits[:, 4] = -math.inf          # an expert that is switched off
    kw = dict(bits=fmt["bits"], group_size=fmt.get("group", 0), packed=fmt.get("packed", False), zero1=first.zero, zero2=second.zero, residual=residual)
    call = (lambda: torch_op.moe_mlp(x, logits, first.b, first.scale, second.b, second.scale, top_k, **kw))
    got = call()
    want, off = plain_layer(x, logits, first, second, top_k, True, residual)
    check(got, want, off)
    if tokens > 5:
        assert torch.equal(got[tokens - 3:], residual[tokens - 3:])
    # captured, replayed on other tokens, next to an eager call on another stream
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    x.copy_(activations(tokens, k, seed=6))
    logits.copy_(activations(tokens, experts, seed=7))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = call()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, eager)
    check(captured, *plain_layer(x, logits, first, second, top_k, True, residual))
    assert afb.read_status()[0] == 0


@pytest.mark.gpu
def test_layer_of_no_tokens(afb):
    from awesome_fusion_b200 import torch_op
    first, second = Experts(4, 128, 128, 8), Experts(4, 128, 64, 8)
    x, logits = activations(0, 128), activations(0, 4)
    assert torch_op.moe_mlp(x, logits, first.b, first.scale, second.b, second.scale, 2).shape == (0, 128)


@pytest.mark.gpu
def test_torch_operators_refuse(afb):
    import awesome_fusion_b200.torch_op  # noqa: F401
    ops = torch.ops.afb
    x = Experts(4, 64, 128, 8)
    a, offsets = activations(6, 128), offsets_of([1, 2, 3, 0])
    good = (a, x.b, x.scale, None, offsets, None, 1, 8, 0, False)
    assert ops.expert_gemm(*good).shape == (6, 64)
    for i, bad in ((0, a.float()), (0, a[:, :64]), (1, x.b[0]), (2, x.scale[:2]), (2, x.scale.half()), (3, x.scale), (4, offsets[:4]), (4, offsets.long()), (5, offsets.long()),
                   (6, 2), (6, 0), (7, 5), (8, 48), (4, offsets.cpu())):
        args = list(good)
        args[i] = bad
        with pytest.raises((ValueError, RuntimeError)):
            ops.expert_gemm(*args)
    with pytest.raises(ValueError):
        ops.expert_gemm(activations(128, 6).t(), *good[1:])   # not contiguous
    for logits, k in ((a, 0), (a, 129), (a.half(), 1), (a[0], 1), (a.t(), 1)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.moe_route(logits, k)
    w, rows = torch.rand((3, 2), device="cuda"), torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    for args in ((a.float(), w, rows), (a, w[:2], rows), (a, w, rows.long()), (a, w, rows, a), (a, w.double(), rows), (a, w, rows.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            ops.moe_combine(*args)
