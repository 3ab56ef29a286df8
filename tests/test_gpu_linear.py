"""GPU tests of the dense layer (forward and backward) against its definition in 64 bits.

Small whole numbers make every fp32 sum exact, so layout, masking, tails and
strides are compared bit for bit after the one rounding of the result; real
numbers are compared within bounds counted from the roundings:
  z   K products summed in fp32, each addition off by at most one step: (K + 2) 2^-23 (|x| |w| + |b|)
  act 2^-23 (8 + 1.2 |z|) max(|z|, 1): the exponential is good to 2 + 1.2 |z| steps, a division and products follow;
      slopes are at most 1.13, so an error of z grows by no more than that
  out half a step of the result's type, and at least half of the type's smallest positive number
"""
import pytest

from linear_util import (ACTS, SENTINEL, act64, backward, dact64, dtype_of, forward, half_step, ints, matrix, untouched)

pytestmark = pytest.mark.gpu

# rows, in, out: one value, tile edges of 64 / 128 / 256, odd widths, several tiles each way, a long K; the last three
# have enough 256 x 256 tiles for pairs of CTAs in the forward, the input gradient and the weight gradient
SHAPES = [(1, 1, 1), (1, 64, 64), (2, 17, 9), (5, 64, 48), (63, 63, 65), (64, 128, 128), (127, 200, 256), (128, 64, 257), (129, 65, 64),
          (300, 320, 511), (1000, 63, 255), (257, 1024, 96), (19, 2048, 520), (4097, 32, 64), (20000, 64, 64), (2500, 520, 2056), (2500, 2049, 520), (700, 2328, 2312)]
# rows of one to seven values, fewer rows than a group of eight and just behind one, steps of K that end in a group
THIN = [(1000, 1, 3), (77, 3, 5), (7, 9, 129), (8, 65, 7), (9, 71, 130), (257, 5, 260), (135, 193, 15)]
# one long axis beside short ones: enough 256 x 256 tiles for pairs of CTAs, but most of each empty
LONG = [(600, 64, 19200), (600, 128, 19200), (520, 130, 19200), (600, 19200, 64), (520, 19200, 130), (40, 576, 19200), (70, 576, 19200),
        (19200, 576, 64), (19200, 520, 72)]


def _floor(torch, t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 if t == torch.float16 else 0.0


def _gen(torch, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("n,k,m", SHAPES + THIN + LONG)
@pytest.mark.parametrize("dtype,pad,shift", [("f16", 0, 0), ("bf16", 8, 8), ("f16", 1, 3), ("bf16", 2, 2)])
def test_forward_whole_numbers(cuda, n, k, m, dtype, pad, shift):
    torch = cuda
    t = dtype_of(torch, dtype)
    gen = _gen(torch, n * 7 + k * 3 + m)
    X, W, B, R = (ints(torch, gen, a, b) for a, b in ((n, k), (m, k), (1, m), (n, m)))
    (x, _), (w, _), (b, _), (r, _) = (matrix(torch, v, t, pad, shift) for v in (X, W, B, R))
    for act, with_b, with_r, with_z in (("none", False, False, False), ("relu", True, True, True), ("relu", True, False, True),
                                        ("none", False, True, False)):
        y, ybuf = matrix(torch, torch.zeros(n, m, device="cuda"), t, pad, shift)
        z, zbuf = matrix(torch, torch.zeros(n, m, device="cuda"), t, pad, shift)
        err = forward(torch, x, w, b if with_b else None, r if with_r else None, y, z if with_z else None, dtype, act)
        Z = X @ W.T + (B if with_b else 0)
        Y = act64(torch, act, Z) + (R if with_r else 0)
        assert int(err) == 0
        assert torch.equal(y, Y.to(t)), (act, with_b, with_r)
        assert untouched(torch, y, ybuf, pad, shift)
        if with_z:
            assert torch.equal(z, Z.to(t)) and untouched(torch, z, zbuf, pad, shift)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,k,m", [(1, 2048, 256), (33, 96, 100), (700, 513, 300), (20, 4096, 1000)])
def test_forward_bounds(cuda, n, k, m, dtype, act):
    torch = cuda
    t = dtype_of(torch, dtype)
    gen = _gen(torch, k + m)
    x, w, b, r = (torch.randn(s, generator=gen, device="cuda").mul(c).to(t) for s, c in
                  (((n, k), 1.0), ((m, k), 3.0 / k ** 0.5), ((m,), 1.0), ((n, m), 1.0)))
    y, z = torch.empty(n, m, dtype=t, device="cuda"), torch.empty(n, m, dtype=t, device="cuda")
    assert int(forward(torch, x, w, b, r, y, z, dtype, act)) == 0
    Z = x.double() @ w.double().T + b.double()
    ez = (k + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T + b.double().abs())
    hs, fl = half_step(torch, t), _floor(torch, t)
    assert bool(((z.double() - Z).abs() <= ez + hs * (Z.abs() + ez) + fl).all())
    Y = act64(torch, act, Z) + r.double()
    ey = 1.13 * ez + 2.0 ** -23 * (8 + 1.2 * Z.abs()) * Z.abs().clamp(min=1) + 2.0 ** -24 * Y.abs()
    assert bool(((y.double() - Y).abs() <= ey + hs * (Y.abs() + ey) + fl).all())


def test_forward_extreme_values(cuda):
    """Far ends of the activations, infinities and NaN: they stay in their rows, and the 16-bit overflow is infinity."""
    torch = cuda
    zs = torch.tensor([-6e4, -200.0, -88.0, -20.0, -0.0, 0.0, 20.0, 88.0, 200.0, 6e4, float("inf"), float("-inf"), float("nan")], device="cuda")
    x = torch.ones(3, 16, dtype=torch.bfloat16, device="cuda")
    x[1, 3] = float("nan")
    w = torch.zeros(zs.numel(), 16, dtype=torch.bfloat16, device="cuda")
    for act in ACTS:
        y, z = (torch.empty(3, zs.numel(), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        assert int(forward(torch, x, w, zs.bfloat16(), None, y, z, "bf16", act)) == 0
        want = act64(torch, act, zs.bfloat16().double())
        for row in (0, 2):
            fine = torch.isfinite(want)
            assert torch.allclose(y[row].double()[fine], want[fine], rtol=2.0 ** -8, atol=1e-30), act
            assert torch.equal(torch.isnan(z[row]), torch.isnan(zs)), act
            assert y[row, 10] == (1.0 if act == "sigmoid" else float("inf"))
        assert bool(torch.isnan(z[1]).all())
    x16, w16 = torch.full((1, 64), 60.0, dtype=torch.float16, device="cuda"), torch.full((8, 64), 60.0, dtype=torch.float16, device="cuda")
    y = torch.empty(1, 8, dtype=torch.float16, device="cuda")
    assert int(forward(torch, x16, w16, None, None, y, None, "f16", "none")) == 0
    assert bool(torch.isinf(y).all())


def test_residual_in_place_and_zero_rows(cuda):
    torch = cuda
    gen = _gen(torch, 3)
    X, W, R = ints(torch, gen, 200, 48), ints(torch, gen, 72, 48), ints(torch, gen, 200, 72)
    x, w, y = X.half(), W.half(), R.half()
    assert int(forward(torch, x, w, None, y, y, None, "f16", "relu")) == 0
    assert torch.equal(y, (act64(torch, "relu", X @ W.T) + R).half())
    keep = y.clone()
    forward(torch, x[:0], w, None, None, y[:0], None, "f16", "relu")
    for acc in (0, 1):
        dw, db = torch.ones(72, 48, device="cuda"), torch.ones(72, device="cuda")
        backward(torch, x[:0], w, y[:0], y[:0], None, x[:0], dw, db, "f16", "relu", "f32", acc)
        assert bool((dw == acc).all()) and bool((db == acc).all())
    assert torch.equal(y, keep)


@pytest.mark.parametrize("n,k,m", SHAPES + THIN + LONG)
@pytest.mark.parametrize("dtype,grad,pad,shift", [("f16", "f32", 0, 0), ("bf16", "bf16", 8, 8), ("f16", "f16", 1, 3), ("bf16", "f32", 2, 2)])
def test_backward_whole_numbers(cuda, n, k, m, dtype, grad, pad, shift):
    torch = cuda
    t, g = dtype_of(torch, dtype), dtype_of(torch, grad)
    gen = _gen(torch, n * 5 + k + m)
    X, W, Z, DY, R = (ints(torch, gen, a, b) for a, b in ((n, k), (m, k), (n, m), (n, m), (n, k)))
    (x, _), (w, _), (z, _), (dy, _), (r, _) = (matrix(torch, v, t, pad, shift) for v in (X, W, Z, DY, R))
    for act, with_r, acc in (("relu", True, 0), ("none", False, 1), ("relu", False, 1)):
        DZ = DY * dact64(torch, act, Z)
        dx, dxbuf = matrix(torch, torch.zeros(n, k, device="cuda"), t, pad, shift)
        dw0, db0 = ints(torch, gen, m, k).to(g), ints(torch, gen, 1, m)[0].to(g)
        dw, db = dw0.clone(), db0.clone()
        err, _ = backward(torch, x, w, z if act != "none" else None, dy, r if with_r else None, dx, dw, db, dtype, act, grad, acc)
        assert int(err) == 0
        assert torch.equal(dx, (DZ @ W + (R if with_r else 0)).to(t)) and untouched(torch, dx, dxbuf, pad, shift)
        assert torch.equal(dw, (DZ.T @ X + acc * dw0.double()).to(g)), (act, acc)
        assert torch.equal(db, (DZ.sum(0) + acc * db0.double()).to(g)), (act, acc)


@pytest.mark.parametrize("which", ["dx", "dw", "db", "dx dw", "dw db"])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_backward_parts(cuda, which, act):
    """Each gradient alone equals the one of the whole call, and nothing that a part does not need is asked for.  dx and
    dw come of the same dz by the same products.  The column sums may be added in another order (with dx they are made
    on its way): each order is off the exact sum by at most (n + 2) 2^-23 sum |dz|, so two by twice that."""
    torch = cuda
    gen = _gen(torch, 11)
    n, k, m = 333, 96, 160
    x, w, z, dy = (torch.randn(s, generator=gen, device="cuda").half() for s in ((n, k), (m, k), (n, m), (n, m)))
    z = z if act != "none" else None

    def call(parts):
        dx = torch.zeros(n, k, dtype=torch.float16, device="cuda") if "dx" in parts else None
        dw = torch.zeros(m, k, device="cuda") if "dw" in parts else None
        db = torch.zeros(m, device="cuda") if "db" in parts else None
        only_x, only_w = (x if "dw" in parts else None), (w if "dx" in parts else None)
        if only_x is None and only_w is None:
            only_w = w
        err, _ = backward(torch, only_x, only_w, z, dy, None, dx, dw, db, "f16", act, "f32")
        assert int(err) == 0
        return {"dx": dx, "dw": dw, "db": db}
    full, part = call("dx dw db"), call(which)
    for key in which.split():
        if key == "db":
            dz = dy.double().abs() * (dact64(torch, act, z.double()).abs() if z is not None else 1.0)
            assert bool(((full[key] - part[key]).double().abs() <= 2 * (n + 2) * 2.0 ** -23 * dz.sum(0)).all())
        else:
            assert torch.equal(full[key], part[key]), key


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,k,m", [(1, 300, 200), (40, 96, 100), (3000, 257, 130)])
def test_backward_bounds(cuda, n, k, m, dtype, act):
    """dz itself is off by the activation's bound and, where the activation is smooth, half a step of its type."""
    torch = cuda
    t = dtype_of(torch, dtype)
    gen = _gen(torch, n + m)
    x, w, z, dy, r = (torch.randn(s, generator=gen, device="cuda").mul(c).to(t) for s, c in
                      (((n, k), 1.0), ((m, k), k ** -0.5), ((n, m), 2.0), ((n, m), 1.0), ((n, k), 1.0)))
    dx, dw, db = torch.empty(n, k, dtype=t, device="cuda"), torch.empty(m, k, device="cuda"), torch.empty(m, device="cuda")
    err, _ = backward(torch, x, w, z if act != "none" else None, dy, r, dx, dw, db, dtype, act, "f32")
    assert int(err) == 0
    X, W, Z, DY = x.double(), w.double(), z.double(), dy.double()
    DZ = DY * dact64(torch, act, Z)
    smooth = act not in ("none", "relu")
    hs, fl = half_step(torch, t), _floor(torch, t)
    ef = DY.abs() * 2.0 ** -23 * (8 + 1.2 * Z.abs()) * Z.abs().clamp(min=1) if smooth else torch.zeros_like(DZ)  # before rounding
    ez = ef + (hs * (DZ.abs() + ef) + fl if smooth else 0.0)
    a = DZ.abs() + ez
    DX = DZ @ W + r.double()
    e = ez @ W.abs() + (m + 2) * 2.0 ** -23 * (a @ W.abs() + r.double().abs())
    assert bool(((dx.double() - DX).abs() <= e + hs * (DX.abs() + e) + fl).all())
    DW = DZ.T @ X
    e = ez.T @ X.abs() + (n + 2) * 2.0 ** -23 * (a.T @ X.abs())
    assert bool(((dw.double() - DW).abs() <= e).all())
    assert bool(((db.double() - DZ.sum(0)).abs() <= ef.sum(0) + (n + 2) * 2.0 ** -23 * (DZ.abs() + ef).sum(0)).all())


def test_backward_relu_ignores_closed_units(cuda):
    """Where pre <= 0 (and where it is NaN) nothing passes, whatever dy holds there."""
    torch = cuda
    gen = _gen(torch, 4)
    n, k, m = 200, 64, 96
    x, w, z, dy = (ints(torch, gen, a, b).half() for a, b in ((n, k), (m, k), (n, m), (n, m)))
    z[5] = -1.0
    closed = ~(z > 0)
    z[7, :] = float("nan")
    closed[7, :] = True
    clean = torch.where(closed, torch.zeros_like(dy), dy)
    dy = torch.where(closed, torch.full_like(dy, float("nan")), dy)
    dx, dw, db = torch.empty_like(x), torch.empty(m, k, device="cuda"), torch.empty(m, device="cuda")
    backward(torch, x, w, z, dy, None, dx, dw, db, "f16", "relu", "f32")
    D = clean.double()
    assert torch.equal(dx, (D @ w.double()).half()) and torch.equal(dw.double(), D.T @ x.double())
    assert torch.equal(db.double(), D.sum(0)) and not dx[5].any() and not dx[7].any()


def test_gradients_against_differences(cuda):
    """Directional differences of the 64-bit layer's scalar loss, at the kernel's own kept z: the kernel's gradients
    along random directions agree to the 16-bit roundings (2^-11 a term for dz, as much for dx) over many terms."""
    torch = cuda
    gen = _gen(torch, 8)
    n, k, m = 64, 48, 80
    for act in ACTS:
        x, w, b, dy = (torch.randn(s, generator=gen, device="cuda").mul(c).half() for s, c in
                       (((n, k), 1.0), ((m, k), 0.2), ((m,), 0.1), ((n, m), 1.0)))
        y, z = torch.empty(n, m, dtype=torch.float16, device="cuda"), torch.empty(n, m, dtype=torch.float16, device="cuda")
        forward(torch, x, w, b, None, y, z, "f16", act)
        dx, dw, db = torch.empty_like(x), torch.empty(m, k, device="cuda"), torch.empty(m, device="cuda")
        backward(torch, x, w, z, dy, None, dx, dw, db, "f16", act, "f32")
        base = z.double() - (x.double() @ w.double().T + b.double())  # differences are taken at the rounded z

        def loss(px, pw, pb):
            return (act64(torch, act, base + (x.double() + px) @ (w.double() + pw).T + b.double() + pb) * dy.double()).sum()
        h = 1e-7
        for px, pw, pb, got in ((1, 0, 0, dx), (0, 1, 0, dw), (0, 0, 1, db)):
            d = torch.randn(got.shape, generator=gen, device="cuda", dtype=torch.float64)
            zero = 0.0
            up = [d * h if p else zero for p in (px, pw, pb)]
            dn = [-d * h if p else zero for p in (px, pw, pb)]
            num = float((loss(*up) - loss(*dn)) / (2 * h))
            terms = float((got.double() * d).norm())
            assert abs(float((got.double() * d).sum()) - num) <= 8 * 2.0 ** -11 * terms + 1e-6 * abs(num) + 1e-4, act


def test_far_rows(cuda):
    """Rows whose offsets pass 32 bits."""
    torch = cuda
    gen = _gen(torch, 6)
    n, k, m, far = 70000, 64, 64, 65536
    X, W, B = ints(torch, gen, n, k), ints(torch, gen, m, k), ints(torch, gen, 1, m)[0]
    big = torch.empty(n * far, dtype=torch.float16, device="cuda")
    x, y, z = (big.view(n, far)[:, c: c + k] for c in (0, 64, 128))
    x.copy_(X)
    w, b = W.half(), B.half()
    assert int(forward(torch, x, w, b, None, y, z, "f16", "relu")) == 0
    Z = X @ W.T + B
    assert torch.equal(y, act64(torch, "relu", Z).half()) and torch.equal(z, Z.half())
    dx = big.view(n, far)[:, 192: 192 + k]
    dw, db = torch.empty(m, k, device="cuda"), torch.empty(m, device="cuda")
    DY = ints(torch, gen, n, m, 1)
    y.copy_(DY)
    err, _ = backward(torch, x, w, z, y, None, dx, dw, db, "f16", "relu", "f32")
    DZ = DY * (Z > 0)
    assert int(err) == 0
    assert torch.equal(dx, (DZ @ W).half()) and torch.equal(dw.double(), DZ.T @ X) and torch.equal(db.double(), DZ.sum(0))


def test_same_inputs_same_bits(cuda):
    torch = cuda
    gen = _gen(torch, 15)
    n, k, m = 30011, 200, 136
    x, w, z, dy = (torch.randn(s, generator=gen, device="cuda").bfloat16() for s in ((n, k), (m, k), (n, m), (n, m)))
    outs = []
    for _ in range(3):
        dx, dw, db = torch.empty_like(x), torch.empty(m, k, device="cuda"), torch.empty(m, device="cuda")
        backward(torch, x, w, z, dy, None, dx, dw, db, "bf16", "gelu", "f32")
        outs.append((dx, dw, db))
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))


def test_streams_and_graphs(cuda):
    """Two layers on two streams at once, each with its own workspace, captured and replayed on new contents."""
    torch = cuda
    gen = _gen(torch, 21)
    jobs = []
    for n, k, m in ((5000, 64, 64), (333, 129, 300)):
        t = {key: ints(torch, gen, a, b).half() for key, a, b in (("x", n, k), ("w", m, k), ("dy", n, m), ("z", n, m))}
        t.update(y=torch.empty(n, m, dtype=torch.float16, device="cuda"), dx=torch.empty(n, k, dtype=torch.float16, device="cuda"),
                 dw=torch.empty(m, k, device="cuda"), db=torch.empty(m, device="cuda"), s=torch.cuda.Stream())
        _, t["ws"] = backward(torch, t["x"], t["w"], t["z"], t["dy"], None, t["dx"], t["dw"], t["db"], "f16", "relu", "f32")
        jobs.append(t)
    torch.cuda.synchronize()
    graphs = []
    for t in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=t["s"]):
            raw = torch.cuda.current_stream().cuda_stream
            forward(torch, t["x"], t["w"], None, None, t["y"], t["z"], "f16", "relu", raw)
            backward(torch, t["x"], t["w"], t["z"], t["dy"], None, t["dx"], t["dw"], t["db"], "f16", "relu", "f32", 0, raw, t["ws"])
        graphs.append(g)
    for t in jobs:
        t["x"].copy_(ints(torch, gen, *t["x"].shape))
        t["dy"].copy_(ints(torch, gen, *t["dy"].shape))
    torch.cuda.synchronize()
    for _ in range(3):
        for g, t in zip(graphs, jobs):
            with torch.cuda.stream(t["s"]):
                g.replay()
    torch.cuda.synchronize()
    for t in jobs:
        Z = t["x"].double() @ t["w"].double().T
        DZ = t["dy"].double() * (Z > 0)
        assert torch.equal(t["y"], act64(torch, "relu", Z).half()) and torch.equal(t["dx"], (DZ @ t["w"].double()).half())
        assert torch.equal(t["dw"].double(), DZ.T @ t["x"].double()) and torch.equal(t["db"].double(), DZ.sum(0))


def test_host_memory_is_refused(cuda):
    import ctypes as C
    from linear_util import desc, ptr
    from nerf_b200 import abi
    torch = cuda
    n, k, m = 4, 16, 16
    dev = {key: torch.zeros(16, 16, dtype=torch.float16, device="cuda") for key in "xwbryz"}
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = desc(dev["x"], dev["w"], n, k, m, "f16", "relu")
    lib = abi.load()
    for bad in "xwbryz":
        p = {key: ptr(v) for key, v in dev.items()}
        p[bad] = torch.zeros(16, 16, dtype=torch.float16).data_ptr()
        assert lib.nerf_b200_linear_forward(C.byref(d), *(p[c] for c in "xwbryz"), ptr(err), None) == abi.NERF_STATUS_INVALID_USAGE, bad
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    for bad in ("x", "w", "z", "dy", "dx", "dw", "db", "ws"):
        p = dict(x=ptr(dev["x"]), w=ptr(dev["w"]), z=ptr(dev["z"]), dy=ptr(dev["y"]), r=None, dx=ptr(dev["r"]), dw=ptr(ws), db=ptr(ws) + 4096, ws=ptr(ws) + 65536)
        host = torch.zeros(1 << 20, dtype=torch.uint8)
        p[bad] = (host.data_ptr() + 255) // 256 * 256
        assert lib.nerf_b200_linear_backward(C.byref(d), p["x"], p["w"], p["z"], p["dy"], p["r"], p["dx"], p["dw"], p["db"], p["ws"],
                                             1 << 19, ptr(err), None) == abi.NERF_STATUS_INVALID_USAGE, bad
    torch.cuda.synchronize()
    assert SENTINEL == 77.0 and not ws.any() and not any(bool(v.any()) for v in dev.values())
