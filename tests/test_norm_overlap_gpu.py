"""Gradient norms that run at once: on two streams, from two captured graphs, from a graph
beside plain calls.  Every one gives what it gives alone, to the last bit."""
import ctypes as C

import pytest
import torch

from test_adamw_gpu import comm  # noqa: F401

pytestmark = pytest.mark.gpu

import coconet_b200 as coco  # noqa: E402

# lists whose kernels leave room for another's; the second takes two launches
LISTS = ([300007, 17, 50001], [1 + (k * 37) % 900 for k in range(1100)], [5], [200001] * 3)


def _lists():
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    return [coco.TensorList([torch.randn(c, device="cuda", generator=gen) * (k + 1) for c in counts], None)
            for k, counts in enumerate(LISTS)]


def _alone(comm, lists):  # noqa: F811
    outs = []
    for lst in lists:
        outs.append(torch.zeros(2, device="cuda"))
        comm.grad_norm_scattered(lst, outs[-1], max_norm=0.5)
        torch.cuda.synchronize()
    assert len({float(o[0]) for o in outs}) == len(outs)
    return outs


def test_norms_on_two_streams_at_once(comm):  # noqa: F811
    lists = _lists()
    expect = _alone(comm, lists)
    rounds = 50
    outs = torch.zeros(rounds, len(lists), 2, device="cuda")
    streams = [torch.cuda.Stream() for _ in lists]
    torch.cuda.synchronize()
    for k in range(rounds):
        for lst, out, s in zip(lists, outs[k], streams):
            comm.grad_norm_scattered(lst, out, max_norm=0.5, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[k], torch.stack(expect)) for k in range(rounds))


def test_norms_from_graphs_and_streams_at_once(comm):  # noqa: F811
    lists = _lists()
    expect = _alone(comm, lists)
    outs = [torch.zeros(2, device="cuda") for _ in lists]
    plain = torch.zeros(40, 2, device="cuda")
    graphs = []
    for lst, out in zip(lists, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(3):   # several calls of one graph, too
                comm.grad_norm_scattered(lst, out, max_norm=0.5)
    streams = [torch.cuda.Stream() for _ in range(len(lists) + 1)]
    for _ in range(20):
        for o in outs:
            o.zero_()
        plain.zero_()
        torch.cuda.synchronize()
        for k in range(len(plain)):
            if k % 10 == 0:
                for g, s in zip(graphs, streams):
                    with torch.cuda.stream(s):
                        g.replay()
            comm.grad_norm_scattered(lists[0], plain[k], max_norm=0.5, stream=streams[-1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, expect))
        assert all(torch.equal(p, expect[0]) for p in plain)


def test_two_branches_of_one_graph(comm):  # noqa: F811
    lists = _lists()
    expect = _alone(comm, lists)
    outs = [torch.zeros(2, device="cuda") for _ in lists]
    side = [torch.cuda.Stream() for _ in lists]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        for lst, out, s in zip(lists, outs, side):
            s.wait_stream(main)
            comm.grad_norm_scattered(lst, out, max_norm=0.5, stream=s)
        for s in side:
            main.wait_stream(s)
    for _ in range(20):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, expect))


def test_a_norm_beside_a_fused_lamb_step(comm):  # noqa: F811
    """The fused LAMB step has partial norms, too; a norm on another stream leaves them alone."""
    lists = _lists()
    expect = _alone(comm, lists)
    n = 100003
    torch.manual_seed(1)
    g, w0 = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")

    def lamb(w, m, v):
        comm.fused_lamb(g, w, m, v, 1e-3, 0.9, 0.999, 1e-6, 0.01, 2)
    ref = [w0.clone(), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")]
    lamb(*ref)
    s = torch.cuda.Stream()
    for _ in range(20):
        mine = [w0.clone(), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")]
        outs = [torch.zeros(2, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        for k, o in enumerate(outs):
            comm.grad_norm_scattered(lists[0], o, max_norm=0.5, stream=s)
            if k == 3:
                lamb(*mine)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(mine, ref))
        assert all(torch.equal(o, expect[0]) for o in outs)


def test_graphs_give_their_memory_back(comm):  # noqa: F811
    """Partial sums of captured calls live as long as their graph: 3000 captures one after the other need no more
    device memory than a few (kept for good they would be 3000 times some KB)."""
    lst = _lists()[2]
    out = torch.zeros(2, device="cuda")

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            comm.grad_norm_scattered(lst, out, max_norm=0.5)
        graph.replay()
        graph.reset()
    for _ in range(50):
        capture()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(3000):
        capture()
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info()[0] <= 4 << 20
    comm.grad_norm_scattered(lst, out, max_norm=0.5)
    assert float(out[0]) > 0


def test_graphs_that_go_while_they_run(comm):  # noqa: F811
    """A graph is thrown away while its launch still waits its turn; what comes meanwhile does not get its memory."""
    lists = _lists()
    expect = _alone(comm, lists)
    a = torch.ones(4096, 4096, device="cuda")
    b = torch.empty_like(a)
    torch.matmul(a, a, out=b)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        outs = torch.zeros(2 * len(lists), 2, device="cuda")
        torch.cuda.synchronize()
        for k, lst in enumerate(lists):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                comm.grad_norm_scattered(lst, outs[2 * k], max_norm=0.5)
            with torch.cuda.stream(side):
                for _ in range(5):
                    torch.matmul(a, a, out=b)
                graph.replay()
            graph.reset()
            again = torch.cuda.CUDAGraph()
            with torch.cuda.graph(again):
                comm.grad_norm_scattered(lst, outs[2 * k + 1], max_norm=0.5)
            with torch.cuda.stream(other):
                again.replay()
            again.reset()
        torch.cuda.synchronize()
        for k, e in enumerate(expect):
            assert torch.equal(outs[2 * k], e) and torch.equal(outs[2 * k + 1], e)


def test_more_live_graphs_than_a_first_chunk_holds(comm):  # noqa: F811
    lst = _lists()[2]
    outs = [torch.zeros(2, device="cuda") for _ in range(200)]
    graphs = []
    for o in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            comm.grad_norm_scattered(lst, o, max_norm=0.5)
    expect = _alone(comm, [lst])[0]
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, expect) for o in outs)


def test_many_streams_that_come_and_go(comm):  # noqa: F811
    lst = _lists()[2]
    expect = _alone(comm, [lst])[0]
    rt = torch.cuda.cudart()
    outs = [torch.zeros(2, device="cuda") for _ in range(700)]
    torch.cuda.synchronize()
    for o in outs:
        h = C.c_void_p()
        assert int(rt.cudaStreamCreate(C.addressof(h))) == 0
        comm.grad_norm_scattered(lst, o, max_norm=0.5, stream=torch.cuda.ExternalStream(h.value))
        assert int(rt.cudaStreamDestroy(h.value)) == 0   # (frees it when its work is done)
    torch.cuda.synchronize()
    assert all(torch.equal(o, expect) for o in outs)
