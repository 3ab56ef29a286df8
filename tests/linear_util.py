"""Buffers, 64-bit definitions and calls of the dense-layer and gradient-norm entry points (torch is used for memory,
streams and the 64-bit arithmetic of the definitions)."""
import ctypes as C
import math

from nerf_b200 import abi
from nerf_b200.abi import check

ACTS = ("none", "relu", "silu", "gelu", "sigmoid")
CODES = {"f32": abi.NERF_B200_F32, "f16": abi.NERF_B200_F16, "bf16": abi.NERF_B200_BF16}
SENTINEL = 77.0


def dtype_of(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def half_step(torch, t):
    return torch.finfo(t).eps / 2


def matrix(torch, values, t, pad=0, shift=0):
    """A device matrix holding `values`, rows `pad` values further apart than tight, first value `shift` values after a
    256-byte boundary; everything around it holds SENTINEL.  Returns (view, whole buffer)."""
    rows, cols = values.shape
    ld = cols + pad
    buf = torch.full((rows * ld + shift + 64,), SENTINEL, dtype=t, device="cuda")
    view = buf[shift: shift + rows * ld].view(rows, ld)[:, :cols]
    view.copy_(values)
    return view, buf


def untouched(torch, view, buf, pad, shift):
    """Whether nothing of buf outside the view's rows and columns was written."""
    keep = torch.ones_like(buf, dtype=torch.bool)
    rows, cols = view.shape
    keep[shift: shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] = False
    return bool((buf[keep] == SENTINEL).all())


def ptr(t):
    return None if t is None else t.data_ptr()


def ld(t):
    return 0 if t is None else t.stride(0)


def desc(x=None, w=None, n=0, n_in=0, n_out=0, dtype="f16", act="none", grad="f32", accumulate=0, **strides):
    return abi.NerfB200Linear(n_rows=n, n_in=n_in, n_out=n_out, dtype=CODES[dtype], activation=ACTS.index(act),
                              grad_dtype=CODES[grad], accumulate=accumulate, ld_x=ld(x), ld_weight=ld(w), **strides)


def forward(torch, x, w, b, r, y, z, dtype, act, stream=None):
    d = desc(x, w, x.shape[0], x.shape[1], w.shape[0], dtype, act, ld_y=ld(y), ld_pre=ld(z), ld_residual=ld(r))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    check("linear_forward", abi.load().nerf_b200_linear_forward(C.byref(d), ptr(x), ptr(w), ptr(b), ptr(r), ptr(y), ptr(z),
                                                                ptr(err), stream))
    return err


def backward(torch, x, w, z, dy, r, dx, dw, db, dtype, act, grad, accumulate=0, stream=None, workspace=None):
    n, n_out = dy.shape
    n_in = (x if x is not None else w).shape[1]
    d = desc(x, w, n, n_in, n_out, dtype, act, grad, accumulate, ld_pre=ld(z), ld_dy=ld(dy), ld_dx=ld(dx), ld_residual=ld(r))
    lib = abi.load()
    size = lib.nerf_b200_linear_backward_workspace_bytes(C.byref(d))
    assert size > 0
    if workspace is None:
        workspace = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN patterns: contents do not matter
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    check("linear_backward", lib.nerf_b200_linear_backward(C.byref(d), ptr(x), ptr(w), ptr(z), ptr(dy), ptr(r), ptr(dx), ptr(dw),
                                                           ptr(db), ptr(workspace), workspace.numel(), ptr(err), stream))
    return err, workspace


def act64(torch, name, z):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2.0)))
    return torch.sigmoid(z) if name == "sigmoid" else z


def dact64(torch, name, z):
    if name == "relu":
        return (z > 0).double()
    s = torch.sigmoid(z)
    if name == "silu":
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2.0))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return s * (1 - s) if name == "sigmoid" else torch.ones_like(z)


def ints(torch, gen, rows, cols, most=2):
    """Small whole numbers: their products and sums are exact in fp32, so results can be compared bit for bit."""
    return torch.randint(-most, most + 1, (rows, cols), generator=gen, device="cuda").double()


def tensors(items):
    """[(grad, out or None)] -> ctypes array of NerfB200GradTensor."""
    code = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}
    t = (abi.NerfB200GradTensor * max(1, len(items)))()
    for k, (g, o) in enumerate(items):
        t[k] = abi.NerfB200GradTensor(ptr(g), ptr(o), g.numel(), code[str(g.dtype)], code[str((o if o is not None else g).dtype)])
    return t


def grad_norm(torch, items, loss_scale=1.0, max_norm=None, stream=None):
    """The norm over [(grad, out or None)], or the clip where max_norm is given; returns the info tensor (4 words)."""
    lib = abi.load()
    info = torch.full((4,), -1.0, dtype=torch.float32, device="cuda")
    size = lib.nerf_b200_grad_workspace_bytes(len(items))
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    t = tensors(items)
    if max_norm is None:
        check("grad_norm", lib.nerf_b200_grad_norm(t, len(items), loss_scale, ptr(info), ptr(ws), size, stream))
    else:
        check("grad_clip", lib.nerf_b200_grad_clip(t, len(items), loss_scale, max_norm, ptr(info), ptr(ws), size, stream))
    return info
