"""GPU tests of the gradient norm and clipping against 64-bit sums.

The squares are added in fp32 for at most 32 values, then in fp64; the norm is rounded to fp32 at its end: relative error
below 32 * 2^-24 / 2 (half of the squares' error) + 2^-24 < 2^-19.  The scale is a quotient in fp64, rounded: 2^-19 as
well; a clipped value adds a product and the rounding to its type."""
import math

import pytest

from linear_util import dtype_of, grad_norm, half_step

pytestmark = pytest.mark.gpu
REL = 2.0 ** -19


def _values(torch, gen, n, name, scale=1.0):
    return (torch.randn(n, generator=gen, device="cuda") * scale).to(dtype_of(torch, name))


def _norm64(torch, grads):
    return math.sqrt(sum(float(g.double()[torch.isfinite(g)].square().sum()) for g in grads))


def _nonfinite(info):
    return int(info.view(dtype=__import__("torch").int32)[2])


def _shifted(torch, v, shift):
    """The same values, `shift` values after a 256-byte boundary."""
    buf = torch.empty(v.numel() + shift + 8, dtype=v.dtype, device="cuda")
    out = buf[shift: shift + v.numel()]
    out.copy_(v)
    return out


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sizes", [[1], [7, 0, 8], [8191, 8192, 8193], [2048, 1024, 2048, 4096, 1024], [1000003]])
def test_norm(cuda, name, sizes):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(sum(sizes))
    for shift in (0, 1, 3):
        grads = [_shifted(torch, _values(torch, gen, n, name), shift) for n in sizes]
        info = grad_norm(torch, [(g, None) for g in grads], loss_scale=128.0)
        want = _norm64(torch, grads) / 128.0
        assert abs(float(info[0]) - want) <= REL * want and float(info[1]) == 1.0 and _nonfinite(info) == 0


def test_norm_of_many_mixed_tensors(cuda):
    """More tensors than one launch's table holds, of all types, some empty."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(1)
    names = ["f32", "f16", "bf16"]
    grads = [_values(torch, gen, (k * 37) % 1500, names[k % 3], 1.0 + k % 5) for k in range(1300)]
    info = grad_norm(torch, [(g, None) for g in grads], 2.0)
    want = _norm64(torch, grads) / 2.0
    assert abs(float(info[0]) - want) <= REL * want
    again = grad_norm(torch, [(g, None) for g in grads], 2.0)
    assert torch.equal(info, again)


def test_norm_of_nothing(cuda):
    torch = cuda
    empty = torch.empty(0, device="cuda")
    for items in ([], [(empty, None)], [(torch.zeros(5000, device="cuda"), None)]):
        info = grad_norm(torch, items)
        assert float(info[0]) == 0.0 and _nonfinite(info) == 0
    info = grad_norm(torch, [], max_norm=1.0)
    assert float(info[0]) == 0.0 and float(info[1]) == 1.0


@pytest.mark.parametrize("name,scale", [("f32", 1e30), ("f32", 1e-30), ("bf16", 1e30), ("bf16", 1e-30), ("f32", 1e-42), ("f16", 3e4), ("f16", 1e-7)])
def test_norm_at_the_ends_of_the_range(cuda, name, scale):
    """Squares that fp32 cannot hold."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(2)
    g = _values(torch, gen, 20000, name).sign().to(dtype_of(torch, name)) * scale
    g[::3] = 0
    info = grad_norm(torch, [(g, None)])
    want = _norm64(torch, [g])
    assert want > 0 and abs(float(info[0]) - want) <= REL * want + 2.0 ** -150
    mixed = torch.cat([g.float(), torch.full((100,), 1e-3, device="cuda")])
    info = grad_norm(torch, [(mixed, None)])
    want = _norm64(torch, [mixed])
    assert abs(float(info[0]) - want) <= REL * want


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_nonfinite_values_are_left_out_and_reported(cuda, name, bad):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(3)
    for at in (0, 8191, 9998):
        g, other = _values(torch, gen, 9999, name), _values(torch, gen, 100, "f32")
        g[at] = bad
        keep = g.clone()
        info = grad_norm(torch, [(g, g), (other, other)], 1.0, max_norm=1e-3)
        want = _norm64(torch, [g, other])
        assert _nonfinite(info) == 1 and float(info[1]) == 1.0 and abs(float(info[0]) - want) <= REL * want
        assert torch.equal(torch.nan_to_num(g.float(), 7.0), torch.nan_to_num(keep.float(), 7.0))  # left as it was
        out = torch.zeros(9999, device="cuda")
        grad_norm(torch, [(g, out)], 1.0, max_norm=1e-3)
        assert torch.equal(torch.nan_to_num(out, 7.0), torch.nan_to_num(keep.float(), 7.0))


@pytest.mark.parametrize("name,out", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("shift,out_shift", [(0, 0), (3, 3), (0, 1), (5, 0)])
def test_clip(cuda, name, out, shift, out_shift):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(4)
    sizes = [1, 100, 8192, 0, 100001, 17]
    grads = [_shifted(torch, _values(torch, gen, n, name), shift) for n in sizes]
    outs = [torch.full((n + out_shift + 8,), 9.0, dtype=dtype_of(torch, out), device="cuda") for n in sizes]
    parts = [o[out_shift: out_shift + n] for o, n in zip(outs, sizes)]
    norm = _norm64(torch, grads) / 4.0
    hs = half_step(torch, dtype_of(torch, out))
    for most in (0.3 * norm, 0.0, 10 * norm, float("inf")):
        keep = [g.clone() for g in grads]
        info = grad_norm(torch, list(zip(grads, parts)), 4.0, max_norm=most)
        scale = min(1.0, most / norm)
        assert abs(float(info[0]) - norm) <= REL * norm and abs(float(info[1]) - scale) <= REL * scale
        for g, k, p, o, n in zip(grads, keep, parts, outs, sizes):
            want = k.double() * scale
            tol = want.abs() * (REL + 2.0 ** -24 + hs) + (2.0 ** -25 if out == "f16" else 0.0)
            assert bool(((p.double() - want).abs() <= tol).all()) and torch.equal(g, k)
            assert bool((o[:out_shift] == 9.0).all()) and bool((o[out_shift + n:] == 9.0).all())
        if scale == 1.0:
            assert all(torch.equal(p.double(), g.double()) for p, g in zip(parts, grads))


def test_clip_in_place_twice(cuda):
    """In place the second clip to the same norm finds next to nothing to do, and a list of 700 tensors takes two tables."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(5)
    grads = [_values(torch, gen, 50 + k, "f32") for k in range(700)]
    keep = [g.clone() for g in grads]
    norm = _norm64(torch, grads)
    grad_norm(torch, [(g, g) for g in grads], 1.0, max_norm=norm / 2)
    for g, k in zip(grads, keep):
        assert bool(((g.double() - k.double() / 2).abs() <= k.double().abs() * (REL + 2.0 ** -23)).all())
    info = grad_norm(torch, [(g, g) for g in grads], 1.0, max_norm=norm / 2)
    assert abs(float(info[0]) - norm / 2) <= 2 * REL * norm and abs(float(info[1]) - 1.0) <= 4 * REL


def test_clip_in_a_graph_on_a_stream(cuda):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(6)
    grads = [_values(torch, gen, n, "f16") for n in (5000, 333)]
    outs = [torch.zeros(g.numel(), device="cuda") for g in grads]
    items = list(zip(grads, outs))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        info = grad_norm(torch, items, 1.0, max_norm=1.0, stream=torch.cuda.current_stream().cuda_stream)
    for seed in range(3):
        for t in grads:
            t.copy_(torch.randn(t.numel(), generator=gen, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        norm = _norm64(torch, grads)
        assert abs(float(info[0]) - norm) <= REL * norm
        for a, b in items:
            assert bool(((b.double() - a.double() / norm).abs() <= a.double().abs() / norm * (REL + 2.0 ** -23)).all())


def test_host_memory_is_refused(cuda):
    torch = cuda
    from linear_util import ptr, tensors
    from nerf_b200 import abi
    lib = abi.load()
    g, out = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    info, ws = torch.zeros(4, device="cuda"), torch.zeros(lib.nerf_b200_grad_workspace_bytes(1), dtype=torch.uint8, device="cuda")
    host = torch.zeros(65536, dtype=torch.uint8)
    at = (host.data_ptr() + 255) // 256 * 256
    for bad in ("grad", "out", "info", "ws"):
        t = tensors([(g, out)])
        if bad in ("grad", "out"):
            setattr(t[0], bad, at)
        pi, pw = at if bad == "info" else ptr(info), at if bad == "ws" else ptr(ws)
        assert lib.nerf_b200_grad_clip(t, 1, 1.0, 1.0, pi, pw, ws.numel(), None) == abi.NERF_STATUS_INVALID_USAGE, bad
    torch.cuda.synchronize()
    assert not out.any()
