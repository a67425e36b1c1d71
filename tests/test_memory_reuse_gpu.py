"""Calls one right after another on memory that each of them writes anew: a kernel may
start while those before it run, and must see what they wrote.  Needs a B200."""

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"


def repeated(turn, n=8, times=20):
    """turn(i) for every i, each alone, then back to back: the same results."""
    want = []
    for i in range(n):
        want.append([t.clone() for t in turn(i)])
        torch.cuda.synchronize()
    for _ in range(times):
        found = [turn(i) for i in range(n)]
        for a, b in zip(found, want):
            assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert oz.device_status() == 0


@pytest.mark.parametrize("zeros", [False, True], ids=["8", "zeros"])
@pytest.mark.parametrize("group", [32, 128])
def test_scales_of_4_bit_weights_written_just_before(group, zeros):
    # the clipped results are the scales that the product reads, in the same memory every turn
    g = torch.Generator(device=DEV).manual_seed(group)
    n, k = 1000, 512
    packed = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    given = [torch.randn(n, k // group, generator=g, device=DEV) * (i + 1) for i in range(8)]
    scales = torch.empty_like(given[0])
    z = torch.randint(0, 16, scales.shape, generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    x = torch.randn(4, k, generator=g, device=DEV, dtype=torch.bfloat16)

    def turn(i):
        norm = oz.clip_gradients([given[i]], 10.0 * (i + 1), out=[scales])
        return norm, oz.matmul_w4(x, packed, scales, z, out_dtype=torch.float32)

    repeated(turn)


def test_clipped_results_written_again():
    g = torch.Generator(device=DEV).manual_seed(1)
    grads = [[(torch.randn(m, generator=g, device=DEV) * (i + 1)).bfloat16() for m in (5000, 77, 40001)] for i in range(8)]
    spare = [torch.empty_like(t, dtype=torch.float32) for t in grads[0]]
    kept = [[torch.empty_like(t) for t in spare] for _ in range(8)]

    def turn(i):
        norm = oz.clip_gradients(grads[i], 1.0, out=spare)
        again = oz.clip_gradients(spare, 0.5, out=kept[i])          # reads what was just written
        return norm, again, *kept[i]

    repeated(turn)
