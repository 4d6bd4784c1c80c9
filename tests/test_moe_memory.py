"""Memory that a product grouped by expert hands its rows through from its first kernel to its second (group scales, form for many rows): whose it is, when it
goes back, what is left for others."""
import gc
import threading

import pytest

import awesome_fusion_b200 as pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_moe import Experts, activations, check, offsets_of  # noqa: E402
from test_workspaces import STREAMING, Gemm, _new_streams  # noqa: E402

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


class Prompt:
    """A product whose converted rows take rows * 8 KB."""

    def __init__(self, afb, rows, seed=5):
        self.afb, self.x = afb, Experts(4, 64, 4096, 4, 128, seed=seed)
        self.a, self.offsets = torch.randn((rows, 4096), device="cuda").bfloat16(), offsets_of([rows // 4] * 3 + [rows - rows // 4 * 3])
        self.want = self.run()
        some = torch.cat([torch.arange(300), torch.arange(rows - 300, rows)]).cuda() if rows > 600 else torch.arange(rows).cuda()
        ends = torch.tensor([0] + [int((some < o).sum()) for o in self.offsets[1:]], dtype=torch.int32, device="cuda")
        check(self.want[some], *self.x.plain(self.a[some], ends, **MANY))

    def run(self, out=None, stream=None):
        before = self.afb.expert_many_launch_count()
        out = self.x.run(self.afb, self.a, self.offsets, out=out, stream=torch.cuda.current_stream().cuda_stream if stream is None else stream, **MANY)
        assert self.afb.expert_many_launch_count() == before + 1, "the form for few rows took the call"
        return out

    def captured(self, stream=None):
        out, graph = torch.zeros_like(self.want), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            self.run(out)
        return graph, out


def held_since(start):
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    return start - torch.cuda.mem_get_info()[0]


def streaming_on_new_streams(afb, dense, count):
    before = afb.stream_launch_count()
    for s in _new_streams(afb, count):
        dense.launch(s)
        dense.check("dense product on a new stream")
    return afb.stream_launch_count() - before == count


def test_growing_prompts_on_many_streams_leave_the_dense_products_theirs(afb):
    """Rows of 75 MB to 0.6 GB, one call on each of twelve streams: every call in the form for many rows; nothing of it stays beyond the 1 GB that the pool keeps, and
    the streaming form still finds its workspaces."""
    dense = Gemm(afb, *STREAMING, seed=22)
    start = held_since(0) * -1
    for rows in (9216, 18500, 37000, 74000):
        p = Prompt(afb, rows)
        for s in _new_streams(afb, 3):
            out = torch.zeros_like(p.want)
            torch.cuda.synchronize()
            p.run(out, s)
            torch.cuda.synchronize()
            assert torch.equal(out, p.want)
        del p, out
    assert held_since(start) <= (1024 + 64) << 20
    assert streaming_on_new_streams(afb, dense, 8)


def test_a_call_above_a_gigabyte(afb):
    rows = 131072 + 900
    Prompt(afb, rows)   # asserts that the form for many rows took it, and compares its first and last rows


def test_captured_graphs_give_their_memory_back(afb):
    """24 graphs of 151 MB each, alive at the same time: the form for many rows in all of them, workspaces left for the dense products.  Destroyed, they leave no more than
    the pool keeps; graphs captured after them, in the memory that they had, do not disturb one that lives."""
    dense, p, first = Gemm(afb, *STREAMING, seed=23), Prompt(afb, 18500), Prompt(afb, 700, seed=8)
    start = held_since(0) * -1
    stays = first.captured()
    graphs = [p.captured() for _ in range(24)]
    assert held_since(start) > 24 * 144 - 1024 << 20   # 18500 rows of 8 KB are 144.5 MiB; up to 1 GiB of them were the pool's before
    assert streaming_on_new_streams(afb, dense, 8)
    for graph, out in graphs[::5] + [stays]:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, p.want) for _, out in graphs[::5]) and torch.equal(stays[1], first.want)
    del graphs, graph, out
    gc.collect()
    torch.cuda.synchronize()
    p.run()   # the library looks for memory of graphs that are gone
    assert held_since(start) <= (1024 + 128) << 20
    graph, out = p.captured()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            graph.replay()
        stays[1].zero_()
        stays[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(out, p.want) and torch.equal(stays[1], first.want)
        out.zero_()
    assert afb.read_status()[0] == 0


def test_a_layer_captured_with_sizes_that_grow_and_shrink(afb):
    """The calls of one capture share the memory of the largest so far."""
    prompts = [Prompt(afb, rows, seed=rows) for rows in (300, 5000, 40, 2000, 9000)]
    outs, graph = [torch.zeros_like(p.want) for p in prompts], torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for p, out in zip(prompts, outs):
            p.run(out)
    for _ in range(2):
        for out in outs:
            out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, p.want) for p, out in zip(prompts, outs))


def test_calls_next_to_a_capture_elsewhere(afb):
    """While one thread captures in global mode, another one's calls take and give back memory on streams that are new to the library."""
    p = Prompt(afb, 3000, seed=9)
    streams, outs, failed, x, graph = _new_streams(afb, 4), [torch.zeros_like(p.want) for _ in range(4)], [], torch.zeros(8, device="cuda"), torch.cuda.CUDAGraph()

    def calls():
        try:
            for s, out in zip(streams, outs):
                p.run(out, s)
        except Exception as e:   # noqa: BLE001
            failed.append(e)

    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x += 1
        t = threading.Thread(target=calls)
        t.start()
        t.join()
        x += 1
    torch.cuda.synchronize()
    assert not failed and all(torch.equal(out, p.want) for out in outs)
    graph.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [2.0] * 8


def test_finalize_with_a_captured_graph_alive(afb):
    """The graph's half of what it holds outlives the library's; after a new afb_init calls and captures work as before."""
    p = Prompt(afb, 900, seed=10)
    graph, out = p.captured()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, p.want)
    afb.finalize()
    del graph
    gc.collect()
    torch.cuda.synchronize()
    afb.init(0)
    assert torch.equal(p.run(), p.want)
    graph, out = p.captured()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, p.want)


def test_a_full_device_takes_the_form_without(afb):
    """Where the rows' memory is not to be had, eager or inside a capture, the form for few rows answers, and nothing of the refusal stays behind."""
    p = Prompt(afb, 74000, seed=12)   # 0.6 GB
    few = p.x.run(afb, p.a, p.offsets, variant=pkg.VARIANT_DECODE)
    out, captured, graph = torch.zeros_like(few), torch.zeros_like(few), torch.cuda.CUDAGraph()
    some = torch.ones(1, device="cuda")
    torch.cuda.synchronize()
    afb.finalize()   # the pool keeps nothing
    afb.init(0)
    torch.cuda.empty_cache()
    full = torch.empty(torch.cuda.mem_get_info()[0] - (400 << 20), dtype=torch.uint8, device="cuda")
    before = afb.expert_many_launch_count()
    p.x.run(afb, p.a, p.offsets, out=out, **MANY)
    with torch.cuda.graph(graph):
        p.x.run(afb, p.a, p.offsets, out=captured, stream=torch.cuda.current_stream().cuda_stream, **MANY)
    graph.replay()
    torch.cuda.synchronize()
    assert afb.expert_many_launch_count() == before
    assert torch.equal(out, few) and torch.equal(captured, few)
    some += 1   # no error was left for the next launch
    torch.cuda.synchronize()
    del full
    torch.cuda.empty_cache()
    assert torch.equal(p.run(), p.want)
    assert afb.read_status()[0] == 0 and some.item() == 2


def test_a_graph_destroyed_while_it_runs(afb):
    """Its memory goes to nobody else before its last launch has ended: calls on other streams look for memory meanwhile."""
    p, q = Prompt(afb, 18500, seed=13), Prompt(afb, 18500, seed=14)
    side, running = torch.cuda.Stream(), 0
    for _ in range(5):
        outs, graph = [torch.zeros_like(p.want) for _ in range(40)], torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for out in outs:
                p.run(out)
        other, end = [torch.zeros_like(q.want) for _ in range(8)], torch.cuda.Event()
        torch.cuda.synchronize()
        graph.replay()
        end.record()
        del graph
        for out in other:
            q.run(out, side.cuda_stream)
        running += not end.query()
        torch.cuda.synchronize()
        assert all(torch.equal(out, p.want) for out in outs) and all(torch.equal(out, q.want) for out in other)
    assert running, "the graph had always ended before the other calls were launched"


def test_two_branches_of_one_graph(afb):
    """A capture that forks: products on both streams run at the same time in the graph, each stream's in memory of its own."""
    p, q, graph, side = Prompt(afb, 6000, seed=15), Prompt(afb, 6000, seed=16), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    outs, others = ([torch.zeros_like(x.want) for _ in range(10)] for x in (p, q))
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        for out, other in zip(outs, others):
            p.run(out, main.cuda_stream)
            q.run(other, side.cuda_stream)
        main.wait_stream(side)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, p.want) for out in outs) and all(torch.equal(out, q.want) for out in others)
        for out in outs + others:
            out.zero_()
