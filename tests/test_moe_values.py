"""Single values through the products grouped by expert: weights of 1 and 0 and scales of 1 pass a chosen number of A to the activation unchanged."""
import pytest

import awesome_fusion_b200 as pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FORMS = [pkg.VARIANT_DECODE, pkg.VARIANT_PREFILL]


def passed_through(afb, values, variant, group, gated, k=64):
    """silu(values) by the kernel, as a gate over an up projection of 1 or alone.  Channel 0 has a weight of 1 at k = 0, channel 1 one at k = 1, where A is 1."""
    rows = values.numel()
    a = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    a[:, 0], a[:, 1] = values, 1
    b = torch.zeros((1, 2, k), dtype=torch.int8, device="cuda")
    b[0, 0, 0] = b[0, 1, 1] = 1
    scale = torch.ones((1, 2, k // group) if group else (1, 2), device="cuda")
    out = torch.full((rows, 1 if gated else 2), 777.0, dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    gemm = afb.make_args(out, a, b, scale, rows, 2, k, ldc=out.shape[1], group=group, variant=variant)
    afb.expert_gemm_launch(afb.make_expert_gemm_args(gemm, offsets, experts=1, gated=gated, activation=pkg.ACT_SILU))
    torch.cuda.synchronize()
    return out[:, 0]


@pytest.mark.parametrize("variant", FORMS)
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("gated", [False, True])
def test_silu(afb, variant, group, gated):
    """Over the whole range of the activation: down to where the result leaves bf16 (-97), not only to where 1 + exp(-v) leaves fp32.  One rounding to bf16 is
    off by 2^-8 of the value or half of the smallest bf16, 2^-134; the kernel's own error is 2^-16 of the value (2^-10 in the range below 2^-126, where a bf16 has
    fewer than 8 bits itself)."""
    v = torch.cat([torch.linspace(-110, 110, 4001), -torch.logspace(-20, 2, 500, base=2.0), torch.linspace(-98, -80, 1000), torch.tensor([0.0, 2.0 ** -60, -2.0 ** -60])])
    if not group:
        v = torch.cat([v, torch.tensor([3e38, -3e38, 2.0 ** 100, -2.0 ** 100])])
    v = v.bfloat16().cuda()
    got, x = passed_through(afb, v, variant, group, gated).double(), v.double()
    want = x / (1 + torch.exp(-x))
    # Group scales, form for many rows: A goes through fp16 with its row's largest value between 2^14 and 2^15, in steps of 2^-24 at the low end: half of one is
    # 2^-25 / 2^14 = 2^-39 of that value.  The slope of silu is below 1.1.
    lost = 1.1 * 2.0 ** -39 * x.abs().clamp(min=1) if group and variant == pkg.VARIANT_PREFILL else 0.0
    own = torch.where(want.abs() < 2.0 ** -126, 2.0 ** -10, 2.0 ** -16) * want.abs()
    off = (got - want).abs()
    ok = off <= 2.0 ** -8 * (want.abs() + own) + 2.0 ** -134 + own + lost
    assert ok.all(), [(x[i].item(), got[i].item(), want[i].item()) for i in (~ok).nonzero()[:5, 0].tolist()]
    assert afb.read_status()[0] == 0


@pytest.mark.parametrize("variant", FORMS)
@pytest.mark.parametrize("fmt", [dict(bits=4, group=128), dict(bits=8, group=64, scale_f32=True), dict(bits=4, group=64, zero=True, packed=True)],
                         ids=lambda f: "-".join(f"{k}{v}" for k, v in f.items()))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("scales, rows", [(100, -70), (124, -104), (-90, 100), (-60, 20)])
def test_ends_of_the_range_of_group_scales(afb, variant, fmt, gated, scales, rows):
    """Scales of up to 2^118 on rows of 2^-104: the results are ordinary numbers, and no intermediate value may leave fp32 (sums of 2^29 in the kernel's units times
    2^104 does).  Bounds: as of the ordinary range, and what A loses in fp16, 2^-39 of the row's largest value for each weight."""
    from test_moe import Experts, activations, offsets_of
    from test_moe_finite import check
    x = Experts(2, 72, 512, seed=41, **fmt)
    a, offsets = (activations(70, 512).float() * 2.0 ** rows).bfloat16(), offsets_of([3, 67])
    x.scale = (x.scale.float() * 2.0 ** scales).to(x.scale.dtype)
    x.w = x.w * 2.0 ** scales
    want, off = x.plain(a, offsets, gated=gated, variant=variant)
    if variant == pkg.VARIANT_PREFILL:
        lost = torch.cat([2.0 ** -39 * a[lo:hi].double().abs().amax(1, keepdim=True) * x.w[e].abs().sum(1) for e, (lo, hi) in enumerate([(0, 3), (3, 70)])])
        if gated:   # silu(gate) * up: the slope of silu is below 1.1
            v = torch.cat([a[lo:hi].double() @ x.w[e].T for e, (lo, hi) in enumerate([(0, 3), (3, 70)])])
            g, u = v[:, 0::2], v[:, 1::2]
            lost = 1.1 * lost[:, 0::2] * (u.abs() + lost[:, 1::2]) + (g.abs() + 1.1 * lost[:, 0::2]) * lost[:, 1::2]
        off = off + 1.01 * lost
    check(x.run(afb, a, offsets, gated=gated, variant=variant), want, off)
    assert afb.read_status()[0] == 0
