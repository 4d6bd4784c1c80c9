"""Host threads whose first use of the GPU is a call of the library: nothing else has given them a context."""
import threading

import pytest

import awesome_fusion_b200 as pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def in_a_new_thread(call):
    out = []

    def work():
        try:
            call()
            out.append(None)
        except Exception as e:   # noqa: BLE001
            out.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    if out[0] is not None:
        raise out[0]


@pytest.mark.parametrize("m", [1, 16, 40, 128, 300])
@pytest.mark.parametrize("flags", [0, pkg.FLAG_PREFILL_SMEM_B, pkg.FLAG_PREFILL_TMEM_A])
def test_dense(afb, m, flags):
    a, b = torch.randn((m, 1024), device="cuda").bfloat16(), torch.randint(-127, 128, (512, 1024), device="cuda", dtype=torch.int8)
    scale, outs = torch.rand((512,), device="cuda"), [torch.zeros((m, 512), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    blocks = [afb.make_args(out, a, b, scale, m, 512, 1024, flags=flags if m > 16 else 0) for out in outs]
    afb.gemm_launch(blocks[0])
    torch.cuda.synchronize()
    in_a_new_thread(lambda: afb.gemm_launch(blocks[1]))
    assert torch.equal(*outs) and outs[0].any()


def test_fused(afb):
    a, b = torch.randn((200, 1024), device="cuda").bfloat16(), torch.randint(-127, 128, (512, 1024), device="cuda", dtype=torch.int8)
    scale, outs = torch.rand((512,), device="cuda"), [torch.zeros((200, 512), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    blocks = [afb.make_fused_args(afb.make_args(out, a, b, scale, 200, 512, 1024), activation=pkg.ACT_SILU) for out in outs]
    afb.gemm_fused_launch(blocks[0])
    torch.cuda.synchronize()
    in_a_new_thread(lambda: afb.gemm_fused_launch(blocks[1]))
    assert torch.equal(*outs) and outs[0].any()


@pytest.mark.parametrize("variant", [pkg.VARIANT_DECODE, pkg.VARIANT_PREFILL])
@pytest.mark.parametrize("fmt", [dict(bits=8), dict(bits=4, group=128)], ids=["int8", "int4-group128"])
def test_products_grouped_by_expert(afb, variant, fmt):
    from test_moe import Experts, activations, offsets_of
    x, offsets, a = Experts(3, 136, 512, seed=3, **fmt), offsets_of([4, 0, 50]), activations(54, 512)
    want = x.run(afb, a, offsets, variant=variant)
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    in_a_new_thread(lambda: x.run(afb, a, offsets, variant=variant, out=out, stream=torch.cuda.default_stream().cuda_stream))
    assert torch.equal(out, want)


def test_router_and_weighted_sum(afb):
    from test_moe import run_route
    logits = torch.randn((70, 16), device="cuda")
    want, got = run_route(afb, logits, 3, True), []
    in_a_new_thread(lambda: got.extend(run_route(afb, logits, 3, True)))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
