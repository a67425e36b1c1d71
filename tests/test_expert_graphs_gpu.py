"""The expert-layer operators captured in a CUDA graph and replayed on other
values, and on several streams at once.  Needs a B200."""

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"


def inputs(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(200, 264, generator=g, device=DEV).bfloat16()
    cuts = torch.randint(0, 201, (4,), generator=g, device=DEV).sort().values
    return {
        "x": x, "w": torch.randn(3, 264, 320, generator=g, device=DEV).bfloat16(),
        "odd": torch.randn(3, 264, 321, generator=g, device=DEV).bfloat16(),
        "dy": torch.randn(200, 320, generator=g, device=DEV).bfloat16(), "offsets": cuts,
        "packed": torch.randint(0, 256, (3, 500, 160), generator=g, device=DEV, dtype=torch.uint8),
        "scales": torch.rand(3, 500, 10, generator=g, device=DEV).bfloat16(),
        "zeros": torch.randint(0, 256, (3, 500, 10), generator=g, device=DEV, dtype=torch.uint8),
    }


def everything(v):
    y = oz.grouped_matmul(v["x"], v["w"], v["offsets"])
    dx, dw = oz.grouped_matmul_backward(v["dy"], v["x"], v["w"], v["offsets"], dw_dtype=torch.float32)
    return [y, dx, dw, oz.grouped_matmul(v["x"], v["odd"], v["offsets"]),
            oz.matmul_w4(y, v["packed"], v["scales"], v["zeros"], offsets=v["offsets"]),
            oz.orthogonalize(dw), oz.orthogonalize(dw[:, :60]), oz.orthogonalize(v["w"], num_splits=1)]


def test_graphs_follow_their_inputs():
    held = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        found = everything(held)
    for seed in (1, 2, 3):
        fresh = inputs(seed)
        want = everything(fresh)
        for name, t in held.items():
            t.copy_(fresh[name])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(found, want))
    assert oz.device_status() == 0


def test_streams_side_by_side():
    sets = [inputs(seed) for seed in range(4)]
    want = [everything(v) for v in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    found = [[] for _ in sets]
    for _ in range(8):
        for v, stream, out in zip(sets, streams, found):
            with torch.cuda.stream(stream):
                out.append(everything(v))
    torch.cuda.synchronize()
    for runs, expected in zip(found, want):
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(run, expected))
    assert oz.device_status() == 0
