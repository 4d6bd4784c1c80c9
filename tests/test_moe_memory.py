"""Memory that a product grouped by expert hands its rows through from its first kernel to its second (group scales, form for many rows): whose it is, when it
goes back, what is left for others."""
import threading

import pytest

import awesome_fusion_b200 as pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_moe import Experts, activations, check, offsets_of  # noqa: E402
from test_workspaces import STREAMING, Gemm  # noqa: E402

MANY = dict(variant=pkg.VARIANT_PREFILL)


@pytest.mark.parametrize("on", ["the default stream", "a stream"])
def test_two_threads_on_one_stream(afb, on):
    """Each call is two kernels, and another thread's call, or its dense product, may come between them: the rows of one must not be the other's.
    Threads with other weights, numbers of rows and K, each result against the one computed alone; ctypes lets go of the interpreter in every call."""
    stream = torch.cuda.current_stream() if on == "the default stream" else torch.cuda.Stream()
    jobs = []
    for i, (counts, n, k, fmt) in enumerate([([100, 3, 260, 0, 40, 77, 1, 90], 264, 1024, dict(bits=4, group=128)), ([5, 90, 0, 140], 136, 512, dict(bits=8, group=64)),
                                             ([33] * 6, 256, 2048, dict(bits=4, group=64, zero=True, packed=True))]):
        x, offsets, a = Experts(len(counts), n, k, seed=31 + i, **fmt), offsets_of(counts), activations(sum(counts), k, seed=i)
        want = x.run(afb, a, offsets, **MANY)
        check(want, *x.plain(a, offsets, **MANY))
        outs = [torch.full_like(want, 777.0) for _ in range(60)]
        jobs.append((outs, want, lambda out, x=x, a=a, offsets=offsets: x.run(afb, a, offsets, out=out, stream=stream.cuda_stream, **MANY)))
    dense = Gemm(afb, *STREAMING, seed=21)
    outs = [torch.full_like(dense.want, 777.0) for _ in range(60)]
    blocks = [afb.make_args(out, dense.a, dense.b, dense.s, *STREAMING) for out in outs]
    jobs.append((outs, dense.want, lambda out: afb.gemm_launch(next(turns), stream.cuda_stream)))
    turns = iter(blocks)
    torch.cuda.synchronize()
    before, failed, gate = afb.expert_many_launch_count(), [], threading.Barrier(len(jobs))

    def work(outs, call):
        try:
            gate.wait(30)
            for out in outs:
                call(out)
        except Exception as e:   # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(outs, call)) for outs, _, call in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed and afb.expert_many_launch_count() - before == 3 * 60
    for outs, want, _ in jobs:
        assert all(torch.equal(out, want) for out in outs)
    assert afb.read_status()[0] == 0
