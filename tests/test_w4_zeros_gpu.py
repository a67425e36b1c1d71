"""4-bit products with every zero point a byte can hold, against (q - z) s in 64
bits.  Needs a B200.

Small whole numbers and power-of-two scales, whose products and sums are exact in
fp32: the fp32 result has to equal the definition.
"""

import itertools

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"

# rows, k, n, group: one and more warps a tile, each tile shape and each number of
# scales a chunk
SHAPES = [(1, 256, 64, 32), (3, 4256, 517, 32), (8, 1024, 129, 128), (1, 8192, 1000, 64), (4, 1024, 20000, 64),
          (4, 1024, 20000, 128), (2, 1024, 20011, 32), (9, 2048, 256, 128), (12, 320, 2000, 64), (16, 96, 700, 96),
          (17, 96, 1000, 96), (40, 384, 33, 192), (20, 256, 9000, 128)]


@pytest.mark.parametrize("zero", [0, 15, 16, 127, 128, 255, None], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_every_zero_point(dtype, zero):
    for t, k, n, group in SHAPES:
        g = torch.Generator(device=DEV).manual_seed(t + k + n)
        packed = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
        scales = 2.0 ** torch.randint(-2, 3, (n, k // group), generator=g, device=DEV)
        if zero is None:                                    # all of them, side by side
            z = torch.randint(0, 256, scales.shape, generator=g, device=DEV, dtype=torch.uint8)
        else:
            z = torch.full(scales.shape, zero, dtype=torch.uint8, device=DEV)
        x = torch.randint(-2, 3, (t, k), generator=g, device=DEV).to(dtype)
        q = torch.stack([packed % 16, packed // 16], -1).flatten(-2).double()
        w = (q - z.double().repeat_interleave(group, -1)) * scales.double().repeat_interleave(group, -1)
        y = oz.matmul_w4(x, packed, scales, z, out_dtype=torch.float32)
        assert torch.equal(y.double(), x.double() @ w.t()), (t, k, n, group)
    assert oz.device_status() == 0


def test_zero_points_of_experts():
    g = torch.Generator(device=DEV).manual_seed(3)
    e, k, n, group = 4, 512, 200, 64
    packed = torch.randint(0, 256, (e, n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.ones(e, n, k // group, device=DEV)
    z = torch.randint(0, 256, scales.shape, generator=g, device=DEV, dtype=torch.uint8)
    z[1] %= 128                                             # one expert without large ones
    offsets = torch.tensor([0, 3, 10, 10, 25], device=DEV)
    q = torch.stack([packed % 16, packed // 16], -1).flatten(-2).double()
    w = q - z.double().repeat_interleave(group, -1)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randint(-2, 3, (25, k), generator=g, device=DEV).to(dtype)
        y = oz.matmul_w4(x, packed, scales, z, offsets=offsets, out_dtype=torch.float32)
        for i, (a, b) in enumerate(itertools.pairwise(offsets.tolist())):
            assert torch.equal(y[a:b].double(), x[a:b].double() @ w[i].t())
