"""Attention launches that may overlap on the GPU: on several streams, and in captured
graphs beside them. Each hands out its work items from a counter that no other
launch in flight may draw from; a shared one leaves rows unwritten."""

import ctypes

import pytest
import torch

from rig_b200 import kernels, ops


def _call(dev, b, h, kv, t, seed, classic=False):
    """A forward and backward over several items per block, and their outputs."""

    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randn(b, h, t, 64, generator=g, device=dev).bfloat16()
    k, v = (torch.randn(b, kv, t, 64, generator=g, device=dev).bfloat16() for _ in range(2))
    do = torch.randn(b, h, t, 64, generator=g, device=dev).bfloat16()
    out = [torch.empty_like(x) for x in (q, k, v, q)]  # dq, dk, dv, o
    lse = torch.empty(b, h, t, device=dev)
    if classic:
        fwd, bwd, size = ops.attention_fwd, ops.attention_bwd, None
        work, how = ops.attention_workspace(b, h, t, dev), dict(scale=0.125)
    else:
        fwd, bwd, size = ops.score_attention_fwd, ops.score_attention_bwd, ops.score_attention_workspace_size
        work = torch.empty(size(b, h, t), dtype=torch.uint8, device=dev)
        how = dict(scale=0.125, softcap=30.0, slopes=kernels.distance_slopes(h, dev))

    def run():
        fwd(q, k, v, out[3], lse, **how)
        bwd(q, k, v, out[3], do, lse, *out[:3], workspace=work, **how)

    return run, out + [lse]


@pytest.mark.gpu
@pytest.mark.parametrize("classic", [False, True])
def test_graph_beside_eager_launches_on_other_streams(cuda, classic):
    """A graph keeps its launches' counters for good; more eager launches than any
    rotation of counters would hold run beside its replays. dq is added up in any
    order, the rest has to be the same bits as when each call runs alone."""

    calls = [_call(cuda, 4, 12, 12 if classic else 4, 1000 + 9 * i, i, classic) for i in range(4)]
    want = []
    for run, out in calls:
        run()
        torch.cuda.synchronize()
        want.append([x.clone() for x in out])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for run, _ in calls[:2]:
            run()
    for _, out in calls:
        for x in out:
            x.fill_(float("nan"))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for i in range(50):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        for s, (run, _) in zip(streams[1:], calls[2:]):
            with torch.cuda.stream(s):
                run()
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    for (_, out), first in zip(calls, want):
        for x, y in zip(out[1:], first[1:]):
            assert torch.equal(x, y)
        assert (out[0].float() - first[0].float()).norm() <= 1e-3 * first[0].float().norm()
    graph.reset()


@pytest.mark.gpu
def test_counters_of_graphs_come_back(cuda):
    """More captured launches, in graphs that are dropped, than there are counters."""

    run, out = _call(cuda, 1, 1, 1, 200, 0)
    run()
    torch.cuda.synchronize()
    want = [x.clone() for x in out]
    for _ in range(140):  # 140 x 500 launches of forward and backward
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(250):
                run()
        graph.reset()
    run()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(out[1:], want[1:]))
    assert ops.device_error() == 0


@pytest.mark.gpu
def test_more_streams_than_counters(cuda):
    """A launch on each of more streams than there are counters, none of them used before."""

    q = torch.randn(2, 2, 300, 64, device=cuda).bfloat16()
    want, o, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(2, 2, 300, device=cuda)
    ops.score_attention_fwd(q, q, q, want, lse, scale=0.125, softcap=30.0)
    cudart, raw = torch.cuda.cudart(), ctypes.c_void_p()
    for i in range(66000):
        assert int(cudart.cudaStreamCreate(ctypes.addressof(raw))) == 0
        look = i % 3000 == 2999
        if look:
            torch.cuda.synchronize()
            o.zero_()
            torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.ExternalStream(raw.value)):
            ops.score_attention_fwd(q, q, q, o, lse, scale=0.125, softcap=30.0)
        assert int(cudart.cudaStreamDestroy(raw.value)) == 0
        if look:
            torch.cuda.synchronize()
            assert torch.equal(o, want)
    assert ops.device_error() == 0
