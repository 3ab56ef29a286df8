"""The dense-layer and gradient operators together, as a program that trains a layer stack uses them: forward through two
layers, backward through both, the global norm and clip over every gradient, one Adam step on the flat parameter vector."""
import math

import numpy as np
import pytest

from linear_util import act64, backward, dact64, forward, grad_norm, ptr
from nerf_b200 import abi
from nerf_b200.abi import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,widths,act", [(1000, (63, 128, 16), "relu"), (513, (32, 64, 24), "silu")])
def test_training_step_of_a_stack(cuda, n, widths, act):
    """One flat vector holds the weights and biases of both layers, as nerf_b200_adam takes it: fp32 masters, the fp16
    mirror that the layers read, fp32 gradients that they write.  The gradients are compared with the 64-bit chain of
    the same rounded activations; dz and the passed dx are rounded to fp16 (2^-11 each), hence 4 * 2^-11 of the norms."""
    torch = cuda
    lib = abi.load()
    gen = torch.Generator(device="cuda").manual_seed(n)
    k, h, m = widths
    shapes = [(h, k), (1, h), (m, h), (1, m)]
    at, size = [], 0
    for a, b in shapes:
        at.append(size)
        size += (a * b + 7) // 8 * 8
    master = torch.zeros(size, device="cuda")
    for (a, b), o in zip(shapes, at):
        master[o: o + a * b] = torch.randn(a * b, generator=gen, device="cuda") / math.sqrt(b if a > 1 else 100.0)
    p16, grad = master.half(), torch.zeros(size, device="cuda")
    m1, m2 = torch.zeros(size, device="cuda"), torch.zeros(size, device="cuda")

    def part(v, i):
        a, b = shapes[i]
        t = v[at[i]: at[i] + a * b].view(a, b)
        return t if a > 1 else t[0]
    x = torch.randn(n, k, generator=gen, device="cuda").half()
    target = torch.randn(n, m, generator=gen, device="cuda")
    y1, z1, dy1 = (torch.empty(n, h, dtype=torch.float16, device="cuda") for _ in range(3))
    y2 = torch.empty(n, m, dtype=torch.float16, device="cuda")
    errs = [forward(torch, x, part(p16, 0), part(p16, 1), None, y1, z1, "f16", act),
            forward(torch, y1, part(p16, 2), part(p16, 3), None, y2, None, "f16", "none")]
    loss_scale = 128.0
    dy2 = ((y2.float() - target) * (2.0 * loss_scale / n)).half()
    errs.append(backward(torch, y1, part(p16, 2), None, dy2, None, dy1, part(grad, 2), part(grad, 3), "f16", "none", "f32")[0])
    errs.append(backward(torch, x, part(p16, 0), z1, dy1, None, None, part(grad, 0), part(grad, 1), "f16", act, "f32")[0])
    assert all(int(e) == 0 for e in errs)

    # the 64-bit chain
    X, W1, W2 = x.double(), part(p16, 0).double(), part(p16, 2).double()
    Z1 = X @ W1.T + part(p16, 1).double()
    Y1 = act64(torch, act, Z1)
    D2 = dy2.double()
    D1 = (D2 @ W2) * dact64(torch, act, Z1)
    want = {0: D1.T @ X, 1: D1.sum(0), 2: D2.T @ Y1, 3: D2.sum(0)}
    for i, g in want.items():
        got = part(grad, i).double()
        assert float((got - g).norm()) <= 4 * 2.0 ** -11 * float(g.norm()) * (1.0 if i >= 2 else 2.0), i
        if i == 3:
            assert float((got - g).abs().max()) <= (n + 2) * 2.0 ** -23 * float(D2.abs().sum(0).max())

    # the clip leaves the loss scale in the gradients, Adam takes it out
    before = grad.clone()
    norm = float(before.double().norm()) / loss_scale
    info = grad_norm(torch, [(grad, grad)], loss_scale, max_norm=norm / 4)
    assert abs(float(info[0]) - norm) <= 2.0 ** -19 * norm
    assert float((grad.double() - before.double() / 4).norm()) <= 2.0 ** -18 * float(before.double().norm())
    scal = np.array([1e-2, 1.0, 1.0 / (1.0 - 0.9), 1.0 / (1.0 - 0.99), 1.0 / loss_scale], np.float32)
    start = master.clone()
    check("adam", lib.nerf_b200_adam(ptr(master), ptr(p16), None, ptr(grad), ptr(m1), ptr(m2), 0, size, scal.ctypes.data, 0, 0.9, 0.99,
                                     1e-15, None))
    g = grad.double() / loss_scale
    moved = torch.where(g != 0, -1e-2 * g.sign(), torch.zeros_like(g))  # the first step of Adam: the rate, against the sign
    assert float((master.double() - start.double() - moved).abs().max()) <= 1e-6
    assert torch.equal(p16, master.half())


def test_a_single_row_through_the_stack(cuda):
    """The serving form: one row, then eight, through the same layers; a row's result does not depend on its company."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(2)
    k, h, m = 96, 256, 40
    w1, w2 = (torch.randn(s, generator=gen, device="cuda").mul(0.1).bfloat16() for s in ((h, k), (m, h)))
    b1 = torch.randn(h, generator=gen, device="cuda").bfloat16()
    x = torch.randn(8, k, generator=gen, device="cuda").bfloat16()

    def run(rows):
        a, y = torch.empty(len(rows), h, dtype=torch.bfloat16, device="cuda"), torch.empty(len(rows), m, dtype=torch.bfloat16, device="cuda")
        forward(torch, rows, w1, b1, None, a, None, "bf16", "gelu")
        forward(torch, a, w2, None, None, y, None, "bf16", "none")
        return y
    whole = run(x)
    A = act64(torch, "gelu", x.double() @ w1.double().T + b1.double()).bfloat16().double()
    want = A @ w2.double().T
    # the hidden row may round to a neighbour: one step of bf16 a term, and half a step for the result
    tol = 2.0 ** -7 * (A.abs() @ w2.double().abs().T) + 2.0 ** -8 * want.abs()
    assert bool(((whole.double() - want).abs() <= tol).all())
    for i in range(8):
        one = run(x[i: i + 1])
        assert bool(((one[0].double() - want[i]).abs() <= tol[i]).all())
