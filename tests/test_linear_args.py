"""Refusals of the dense-layer and gradient-norm entry points: every one is found before any device work, so no GPU is
needed (the pointers are never dereferenced)."""
import ctypes as C

import pytest

from nerf_b200 import abi

INVALID = abi.NERF_STATUS_INVALID_USAGE
OK = 0x10000


def _desc(**kw):
    base = dict(n_rows=4, n_in=8, n_out=8, dtype=abi.NERF_B200_F16, activation=abi.NERF_B200_ACT_RELU, grad_dtype=abi.NERF_B200_F32)
    return abi.NerfB200Linear(**{**base, **kw})


def _forward(d, x=OK, w=OK, b=OK, r=None, y=OK, z=None, e=OK):
    return abi.load().nerf_b200_linear_forward(C.byref(d) if d is not None else None, x, w, b, r, y, z, e, None)


def _backward(d, x=OK, w=OK, z=OK, dy=OK, r=None, dx=OK, dw=OK, db=OK, ws=OK, size=1 << 30, e=OK):
    return abi.load().nerf_b200_linear_backward(C.byref(d) if d is not None else None, x, w, z, dy, r, dx, dw, db, ws, size, e, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=abi.NERF_B200_F32), dict(dtype=3), dict(activation=5), dict(n_in=0), dict(n_out=0), dict(n_in=(1 << 20) + 1),
    dict(n_rows=1 << 31), dict(ld_x=7), dict(ld_weight=7), dict(ld_y=7), dict(ld_pre=7), dict(ld_dy=7), dict(ld_dx=7),
    dict(ld_x=1 << 40), dict(grad_dtype=abi.NERF_B200_BF16), dict(accumulate=2), dict(reserved=1)])
def test_bad_descriptors(bad):
    d = _desc(**bad)
    assert _forward(d) == INVALID and _backward(d) == INVALID
    assert abi.load().nerf_b200_linear_backward_workspace_bytes(C.byref(d)) == 0


def test_missing_and_misaligned_arguments():
    d = _desc()
    assert _forward(None) == INVALID and _backward(None) == INVALID
    for k in ("x", "w", "y", "e"):
        assert _forward(d, **{k: None}) == INVALID, k
    for k in ("x", "w", "b", "r", "y", "z", "e"):
        assert _forward(d, **{k: OK + 1}) == INVALID, k
    assert _forward(_desc(ld_residual=7), r=OK) == INVALID
    for k in ("x", "w", "z", "dy", "ws", "e"):
        assert _backward(d, **{k: None}) == INVALID, k
    for k in ("x", "w", "z", "dy", "r", "dx", "dw", "db", "ws", "e"):
        assert _backward(d, **{k: OK + 1}) == INVALID, k
    assert _backward(d, dw=OK + 2) == INVALID and _backward(d, db=OK + 2) == INVALID  # fp32 gradients
    assert _backward(d, ws=OK + 16) == INVALID
    assert _backward(_desc(ld_residual=7), r=OK) == INVALID
    size = abi.load().nerf_b200_linear_backward_workspace_bytes(C.byref(d))
    assert size > 0 and _backward(d, size=size - 1) == INVALID


def test_outputs_over_operands_are_refused():
    d, at = _desc(), [OK + 0x1000 * i for i in range(12)]
    good = dict(x=at[0], w=at[1], b=at[2], r=at[3], y=at[4], z=at[5], e=at[6])
    for change in (dict(y=at[0]), dict(y=at[1]), dict(y=at[5]), dict(z=at[0]), dict(z=at[3])):
        assert _forward(d, **{**good, **change}) == INVALID, change
    assert _forward(_desc(ld_residual=16), **{**good, "r": at[4]}) == INVALID  # in place with another distance between rows
    good = dict(x=at[0], w=at[1], z=at[2], dy=at[3], r=None, dx=at[4], dw=at[5], db=at[6], ws=at[7], e=at[8])
    for change in (dict(dx=at[0]), dict(dx=at[1]), dict(dx=at[2]), dict(dx=at[3])):
        assert _backward(d, **{**good, **change}) == INVALID, change
    assert _backward(_desc(ld_residual=16), **{**good, "r": at[4]}) == INVALID


def test_nothing_to_do_needs_no_device():
    d = _desc(n_rows=0)
    assert _forward(d, x=None, w=None, y=None, e=None) == abi.NERF_STATUS_OK
    assert _backward(_desc(), dx=None, dw=None, db=None) == abi.NERF_STATUS_OK


def test_workspace_covers_its_parts():
    """dz (padded to whole 16-byte rows), one row of column sums a row range, and a partial tile a split."""
    lib = abi.load()
    for n, k, m in [(1, 8, 8), (1000, 64, 63), (100003, 63, 255), (65536, 256, 256), (7, 6000, 5000)]:
        d = _desc(n_rows=n, n_in=k, n_out=m)
        size = lib.nerf_b200_linear_backward_workspace_bytes(C.byref(d))
        assert size >= 2 * n * ((m + 7) // 8 * 8) + 4 * m
        none = _desc(n_rows=n, n_in=k, n_out=m, activation=abi.NERF_B200_ACT_NONE)
        assert lib.nerf_b200_linear_backward_workspace_bytes(C.byref(none)) < size


def _tensor(**kw):
    base = dict(grad=OK, out=OK, count=16, dtype=abi.NERF_B200_F32, out_dtype=abi.NERF_B200_F32)
    return abi.NerfB200GradTensor(**{**base, **kw})


def _clip(ts, n=None, scale=1.0, most=1.0, info=OK, ws=OK, size=1 << 30, clip=True):
    arr = (abi.NerfB200GradTensor * max(1, len(ts)))(*ts) if ts is not None else None
    n = len(ts) if n is None else n
    lib = abi.load()
    if clip:
        return lib.nerf_b200_grad_clip(arr, n, scale, most, info, ws, size, None)
    return lib.nerf_b200_grad_norm(arr, n, scale, info, ws, size, None)


def test_gradient_refusals():
    good = [_tensor()]
    for clip in (False, True):
        assert _clip(None, n=1, clip=clip) == INVALID
        for kw in (dict(info=None), dict(ws=None), dict(info=OK + 1), dict(ws=OK + 8), dict(size=16), dict(scale=0.0),
                   dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
            assert _clip(good, clip=clip, **kw) == INVALID, kw
        for kw in (dict(grad=None), dict(grad=OK + 2, out=OK + 2), dict(dtype=3), dict(count=1 << 41)):
            assert _clip([_tensor(**kw)], clip=clip) == INVALID, kw
        assert _clip(good, n=(1 << 24) + 1, clip=clip) == INVALID
    assert abi.load().nerf_b200_grad_workspace_bytes((1 << 24) + 1) == 0
    for most in (-1.0, float("nan")):
        assert _clip(good, most=most) == INVALID
    for kw in (dict(out=None), dict(out=OK + 2), dict(dtype=abi.NERF_B200_F32, out_dtype=abi.NERF_B200_F16),
               dict(dtype=abi.NERF_B200_F16, out_dtype=abi.NERF_B200_BF16)):
        assert _clip([_tensor(**kw)]) == INVALID, kw


def test_overlapping_outputs_are_refused():
    a, far = _tensor(), 0x40000
    assert _clip([a, a]) == INVALID                                                       # listed twice
    assert _clip([a, _tensor(grad=far, out=OK + 32)]) == INVALID                          # outputs overlap
    assert _clip([_tensor(grad=far, out=OK + 32), a]) == INVALID                          # in either order
    assert _clip([_tensor(out=far), _tensor(grad=far + 4, out=0x80000)]) == INVALID       # an output over another's gradient
    assert _clip([_tensor(out=OK + 4)]) == INVALID                                        # over its own, not in place
    assert _clip([_tensor(dtype=abi.NERF_B200_F16)]) == INVALID                           # in place into a wider type
