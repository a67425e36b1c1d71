"""Calls from threads that have no CUDA context yet.  Needs a B200.

A thread gets its context with its first runtime call that needs one; an operator
whose result comes from the allocator's cache may be that first call (as it may
be on a worker of the autograd engine).
"""

import threading

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"


def operands(dtype=torch.float16):
    g = torch.Generator(device=DEV).manual_seed(1)
    whole = lambda *shape: torch.randint(-2, 3, shape, generator=g, device=DEV).to(dtype)   # noqa: E731
    return whole(40, 64), whole(2, 64, 72), whole(40, 72), torch.tensor([0, 13, 40], device=DEV)


def four_bits():
    g = torch.Generator(device=DEV).manual_seed(2)
    return (torch.randint(0, 256, (72, 32), generator=g, device=DEV, dtype=torch.uint8),
            torch.ones(72, 2, dtype=torch.float16, device=DEV))


def floats(*shape):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)


def calls():
    x, w, dy, offsets = operands()
    packed, scales = four_bits()
    g, small = floats(300, 400), floats(40, 60)
    a, b = floats(256, 192).double(), floats(192, 320).double()
    slices = [oz.split_matrix(t, 2, 6, torch.int8) for t in (a[None], b.t()[None])]
    torch.cuda.synchronize()
    return {
        "grouped product": lambda: oz.grouped_matmul(x, w, offsets),
        "its gradients": lambda: oz.grouped_matmul_backward(dy, x, w, offsets)[1],
        "4 bits": lambda: oz.matmul_w4(x, packed, scales),
        "orthogonalize": lambda: oz.orthogonalize(g),
        "orthogonalize, small": lambda: oz.orthogonalize(small),
        "ozaki": lambda: oz.ozaki_matmul(a, b, num_splits=2),
        "split": lambda: oz.split_matrix(a.t()[None], 2, 6, torch.int8)[0],
        "cross GEMM": lambda: oz.cross_gemm(slices[0][0], slices[1][0].transpose(2, 3), slices[0][1], slices[1][1],
                                            2, torch.float64),
    }


NAMES = ["grouped product", "its gradients", "4 bits", "orthogonalize", "orthogonalize, small", "ozaki", "split",
         "cross GEMM"]


@pytest.mark.parametrize("name", NAMES)
def test_first_call_of_a_thread(name):
    call = calls()[name]
    want = call()
    found = []

    def body():
        try:
            found.append(call())
        except Exception as e:       # noqa: BLE001 - handed to the test's thread
            found.append(e)

    thread = threading.Thread(target=body)
    thread.start()
    thread.join()
    assert not isinstance(found[0], Exception), found[0]
    torch.cuda.synchronize()
    assert torch.equal(found[0], want)


def test_first_operator_of_a_backward_pass():
    x, w, dy, offsets = operands()
    x.requires_grad_()
    w.requires_grad_()
    want = oz.grouped_matmul_backward(dy, x.detach(), w.detach(), offsets)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(oz.grouped_matmul(x, w, offsets), (x, w), dy), want))
