"""Performance cases of the dense-layer and gradient-norm operators.

Four operators, used together they are one training step of a stack of dense layers:
  linear_forward   z = x W^T + b, y = act(z) + r
  linear_backward  dz = dy act'(z), dx = dz W + r, dW (+)= dz^T x, db (+)= sum of dz over the rows
  grad_norm        global norm of the finite values of many loss-scaled gradient tensors, and whether any is not finite
  grad_clip        the same, then every gradient times min(1, max_norm / norm) into its output

`own` selects the library's kernels; otherwise the same is computed with elementary torch operations in 32 bits.
"""
import ctypes
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # NERF_B200_F32, _F16, _BF16
ACTS = ("none", "relu", "silu", "gelu", "sigmoid")               # NERF_B200_ACT_*, in order
LOSS_SCALE = 128.0


# ------------------------------------------------------------------ the cases
def _linear(op, name, n, n_in, n_out, dtype, act, bias=True, residual=False, keep=False, pad=0, grad="f32", accumulate=False):
    return {"name": name, "op": op, "n": n, "n_in": n_in, "n_out": n_out, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "keep": keep, "pad": pad, "grad": grad, "accumulate": accumulate}


def _grads(op, name, tensors, total, dtype, out, layout):
    return {"name": name, "op": op, "tensors": tensors, "total": total, "dtype": dtype, "out": out, "layout": layout}


def listed():
    f, b, g, c = "linear_forward", "linear_backward", "grad_norm", "grad_clip"
    return [
        # one row through a square layer: a single query, where the weights' read and the call's latency are all there is
        _linear(f, "forward_one_row", 1, 2048, 2048, "bf16", "silu", residual=True),
        # a handful of rows through a wide layer: small-batch serving, bound by the weights' read
        _linear(f, "forward_few_rows", 19, 4096, 4096, "f16", "gelu"),
        # a hidden layer at the field's own width over a training step's samples, keeping z for the backward
        _linear(f, "forward_field", 262144, 64, 64, "f16", "relu", keep=True),
        # a frequency-encoded position (3 + 3 * 2 * 10 values, rows tight, so no row starts on a 16-byte boundary) into an odd width
        _linear(f, "forward_odd", 100003, 63, 255, "f16", "relu"),
        # a wide residual layer in training: bound by the matrix product
        _linear(f, "forward_wide", 16384, 4096, 4096, "bf16", "gelu", residual=True, keep=True),
        # the backward of the field's hidden layer: fp32 gradients for the optimiser
        _linear(b, "backward_field", 262144, 64, 64, "f16", "relu"),
        # a 256-wide layer over an odd number of rows, gradients added to those of an earlier micro-batch, skip gradient joined
        _linear(b, "backward_256", 65521, 256, 256, "f16", "relu", residual=True, accumulate=True),
        # the wide layer's backward, all gradients in bf16
        _linear(b, "backward_wide", 8192, 4096, 4096, "bf16", "silu", grad="same"),
        # the field MLPs' weights alone: latency
        _grads(g, "norm_small", 5, 10240, "f32", "f32", 1),
        # a hash table of 16 levels of up to 2^19 entries and the MLPs, as they stand after a training step's backward
        _grads(g, "norm_table", 6, 24500000, "table", "f32", 2),
        # the parameters of a stack of layers, fp16 gradients into the fp32 vector that Adam reads
        _grads(c, "clip_stack", 291, 30000001, "f16", "f32", 3),
        # a large model's shard: far more than the L2 cache holds
        _grads(c, "clip_large", 37, 200000000, "bf16", "same", 4),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear_forward", "linear_forward", "linear_backward", "linear_backward", "grad_norm", "grad_clip"])
    if op.startswith("linear"):
        most = 2.5e11 if op == "linear_forward" else 1.25e11  # n * n_in * n_out, of the largest listed cases
        while True:
            n, n_in, n_out = _spread(rng, 1, 400000), _spread(rng, 16, 6000), _spread(rng, 8, 6000)
            if rng.random() < 0.4:  # round widths, as most layers have
                n_in, n_out = -(-n_in // 32) * 32, -(-n_out // 32) * 32
            if n * n_in * n_out <= most and n * (n_in + n_out) <= 1.3e8:
                break
        act = rng.choice(ACTS)
        grad = rng.choice(["f32", "same"]) if act in ("none", "relu") else "same"
        c = _linear(op, "", n, n_in, n_out, rng.choice(["f16", "bf16"]), act, bias=rng.random() < 0.8, residual=rng.random() < 0.5,
                    keep=op == "linear_forward" and rng.random() < 0.5, pad=rng.choice([0, 0, 1, 8]), grad=grad,
                    accumulate=op == "linear_backward" and rng.random() < 0.3)
    else:
        tensors = _spread(rng, 1, 700)
        c = _grads(op, "", tensors, max(tensors, _spread(rng, 1000, 150000000)), rng.choice(["f16", "bf16", "f32", "mixed"]),
                   rng.choice(["same", "f32"]) if op == "grad_clip" else "f32", rng.randrange(1 << 20))
    del c["name"]
    return c


def _tensors(case):
    """[(count, dtype)] of a gradient case: the field's own shapes, or sizes spread over about three decades."""
    mlp = [2048, 1024, 2048, 4096, 1024]
    if case["dtype"] == "table":
        return [(case["total"] - sum(mlp), torch.float16)] + [(m, torch.float32) for m in mlp]
    if case["tensors"] == 5 and case["total"] == sum(mlp):
        return [(m, DTYPES[case["dtype"]]) for m in mlp]
    rng, k, total = random.Random(case["layout"]), case["tensors"], case["total"]
    share = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(k)]
    counts = [max(1, int(total * s / sum(share))) for s in share]
    counts[0] = max(1, counts[0] + total - sum(counts))
    kinds = [rng.choice(["f16", "bf16", "f32"]) if case["dtype"] == "mixed" else case["dtype"] for _ in range(k)]
    return [(n, DTYPES[d]) for n, d in zip(counts, kinds)]


def _part(n):
    return -(-n // 8) * 8


def _out_dtype(case, dtype):
    return torch.float32 if case["out"] == "f32" else dtype


# ------------------------------------------------------------------ the inputs
def _matrix(rows, cols, pad, dtype, gen, scale):
    """A rows x cols matrix whose rows are cols + pad values apart."""
    m = torch.empty((rows, cols + pad), dtype=dtype, device="cuda")
    return m.normal_(0.0, scale, generator=gen)[:, :cols] if gen is not None else m[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if not case["op"].startswith("linear"):
        kinds = _tensors(case)
        grads = [torch.randn(n, device="cuda", generator=gen).to(t) for n, t in kinds]
        norm = math.sqrt(sum(n for n, _ in kinds)) / LOSS_SCALE
        s = {"case": case, "grads": grads, "max_norm": 0.3 * norm}
        if case["op"] == "grad_clip":  # one flat vector for each type of gradient, every tensor's part a multiple of 8 values
            s["flat"] = {str(t): torch.zeros(sum(_part(n) for n, u in kinds if u == t), dtype=_out_dtype(case, t), device="cuda")
                         for t in dict.fromkeys(t for _, t in kinds)}
            parts = {t: iter(f.split([_part(n) for n, u in kinds if str(u) == t])) for t, f in s["flat"].items()}
            s["out"] = [next(parts[str(t)])[:n] for n, t in kinds]
            s["gaps"] = [g.new_zeros(_part(g.numel()) - g.numel()) for g in s["grads"]]
        s["info"] = torch.zeros(4, dtype=torch.float32, device="cuda")
        s["norm"], s["scale"], s["nonfinite"] = s["info"][0:1], s["info"][1:2], s["info"][2:3].view(torch.int32)
        return s
    n, k, m, t, pad = case["n"], case["n_in"], case["n_out"], DTYPES[case["dtype"]], case["pad"]
    s = {"case": case}
    s["x"] = _matrix(n, k, pad, t, gen, 1.0)
    s["w"] = _matrix(m, k, pad, t, gen, 1.0 / math.sqrt(k))
    s["b"] = torch.empty(m, dtype=t, device="cuda").normal_(0.0, 0.1, generator=gen) if case["bias"] else None
    if case["op"] == "linear_forward":
        s["r"] = _matrix(n, m, pad, t, gen, 1.0) if case["residual"] else None
        s["y"] = _matrix(n, m, pad, t, None, 0.0)
        s["z"] = _matrix(n, m, pad, t, None, 0.0) if case["keep"] else None
        return s
    g = torch.float32 if case["grad"] == "f32" else t
    s["z"] = _matrix(n, m, pad, t, gen, 1.0) if case["act"] != "none" else None
    s["dy"] = _matrix(n, m, pad, t, gen, 0.25)
    s["r"] = _matrix(n, k, pad, t, gen, 0.25) if case["residual"] else None
    s["dx"] = _matrix(n, k, pad, t, None, 0.0)
    s["dw"] = torch.empty((m, k), device="cuda").normal_(0.0, 1.0, generator=gen).to(g)
    s["db"] = torch.empty(m, device="cuda").normal_(0.0, 1.0, generator=gen).to(g) if case["bias"] else None
    return s


# ------------------------------------------------------------------ the plain forms
def _act(name, z):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _act_grad(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 - s)


def _plain_forward(s):
    case, t = s["case"], s["x"].dtype
    z = s["x"].float() @ s["w"].float().T
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(case["act"], z)
    if s["r"] is not None:
        y = y + s["r"].float()
    return {"y": y.to(t), "z": z.to(t)} if case["keep"] else {"y": y.to(t)}


def _plain_backward(s):
    case, t, g = s["case"], s["x"].dtype, s["dw"].dtype
    dz = s["dy"].float()
    if case["act"] != "none":
        dz = dz * _act_grad(case["act"], s["z"].float())
    dx = dz @ s["w"].float()
    if s["r"] is not None:
        dx = dx + s["r"].float()
    # sums over many rows lose digits in 32 bits where the result is kept in them
    wide = torch.float64 if g == torch.float32 and case["n"] > 4096 else torch.float32
    dw = (dz.to(wide).T @ s["x"].to(wide)).float()
    out = {"dx": dx.to(t), "dw": s["dw"].copy_(s["dw"].float() + dw if case["accumulate"] else dw)}
    if s["db"] is not None:
        db = dz.to(wide).sum(0).float()
        out["db"] = s["db"].copy_(s["db"].float() + db if case["accumulate"] else db)
    return out


def _plain_grads(s):
    clip = s["case"]["op"] == "grad_clip"
    kinds = dict.fromkeys(g.dtype for g in s["grads"])
    pairs = zip(s["grads"], s["gaps"]) if clip else zip(s["grads"])
    pairs = [(p[0].dtype, p) for p in pairs]
    flat = {t: torch.cat([v for u, p in pairs if u == t for v in p]).float() for t in kinds}
    fine = {t: torch.isfinite(f) for t, f in flat.items()}
    squares = [torch.where(fine[t], f, torch.zeros_like(f)).square().sum() for t, f in flat.items()]
    norm = torch.stack(squares).sum().sqrt() / LOSS_SCALE
    bad = 1 - torch.stack([f.all() for f in fine.values()]).all().int()
    if not clip:
        return {"norm": norm.reshape(1), "nonfinite": bad.reshape(1)}
    scale = torch.where((norm > s["max_norm"]) & (bad == 0), s["max_norm"] / norm, torch.ones_like(norm))
    return {"out": {str(t): (f * scale).to(s["flat"][str(t)].dtype) for t, f in flat.items()}, "norm": norm.reshape(1),
            "scale": scale.reshape(1), "nonfinite": bad.reshape(1)}


# ------------------------------------------------------------------ the library's calls
def _ptr(t):
    return None if t is None else t.data_ptr()


def _bind(s):
    """The call of a state: the library's descriptor, workspace and pointers, as a program makes them once for its buffers."""
    from nerf_b200 import abi
    lib, case = abi.load(), s["case"]
    if not case["op"].startswith("linear"):
        clip = case["op"] == "grad_clip"
        table = (abi.NerfB200GradTensor * len(s["grads"]))()
        for k, g in enumerate(s["grads"]):
            o = s["out"][k] if clip else None
            table[k] = abi.NerfB200GradTensor(g.data_ptr(), _ptr(o), g.numel(), CODES[g.dtype], CODES[o.dtype] if clip else 0)
        size = lib.nerf_b200_grad_workspace_bytes(len(table))
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        tail = (s["info"].data_ptr(), s["workspace"].data_ptr(), size, None)
        if clip:
            s["args"] = (table, len(table), LOSS_SCALE, s["max_norm"]) + tail
            return "nerf_b200_grad_clip", lib.nerf_b200_grad_clip, abi.check
        s["args"] = (table, len(table), LOSS_SCALE) + tail
        return "nerf_b200_grad_norm", lib.nerf_b200_grad_norm, abi.check
    d = abi.NerfB200Linear(n_rows=case["n"], n_in=case["n_in"], n_out=case["n_out"], dtype=CODES[s["x"].dtype],
                           activation=ACTS.index(case["act"]), ld_x=s["x"].stride(0), ld_weight=s["w"].stride(0))
    s["error"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if case["op"] == "linear_forward":
        d.ld_y = s["y"].stride(0)
        d.ld_residual = s["r"].stride(0) if s["r"] is not None else 0
        d.ld_pre = s["z"].stride(0) if s["z"] is not None else 0
        s["args"] = (ctypes.byref(d), _ptr(s["x"]), _ptr(s["w"]), _ptr(s["b"]), _ptr(s["r"]), _ptr(s["y"]), _ptr(s["z"]),
                     _ptr(s["error"]), None)
        return "nerf_b200_linear_forward", lib.nerf_b200_linear_forward, abi.check
    d.grad_dtype, d.accumulate = CODES[s["dw"].dtype], int(case["accumulate"])
    d.ld_dy, d.ld_dx = s["dy"].stride(0), s["dx"].stride(0)
    d.ld_pre = s["z"].stride(0) if s["z"] is not None else 0
    d.ld_residual = s["r"].stride(0) if s["r"] is not None else 0
    size = lib.nerf_b200_linear_backward_workspace_bytes(ctypes.byref(d))
    s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    s["args"] = (ctypes.byref(d), _ptr(s["x"]), _ptr(s["w"]), _ptr(s["z"]), _ptr(s["dy"]), _ptr(s["r"]), _ptr(s["dx"]),
                 _ptr(s["dw"]), _ptr(s["db"]), _ptr(s["workspace"]), size, _ptr(s["error"]), None)
    return "nerf_b200_linear_backward", lib.nerf_b200_linear_backward, abi.check


def _own(s):
    if "call" not in s:
        s["call"] = _bind(s)
    name, call, check = s["call"]
    check(name, call(*s["args"]))
    case = s["case"]
    if case["op"] == "linear_forward":
        return {"y": s["y"], "z": s["z"]} if case["keep"] else {"y": s["y"]}
    if case["op"] == "linear_backward":
        return {k: s[k] for k in ("dx", "dw", "db") if s[k] is not None}
    if case["op"] == "grad_norm":
        return {"norm": s["norm"], "nonfinite": s["nonfinite"]}
    return {"out": s["flat"], "norm": s["norm"], "scale": s["scale"], "nonfinite": s["nonfinite"]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "linear_forward":
        return _plain_forward(state)
    return _plain_backward(state) if op == "linear_backward" else _plain_grads(state)


# ------------------------------------------------------------------ the work, and the exact values
def work(case):
    if not case["op"].startswith("linear"):
        kinds = _tensors(case)
        size = lambda t: 4 if t == torch.float32 else 2  # noqa: E731
        read, total = sum(n * size(t) for n, t in kinds), sum(n for n, _ in kinds)
        if case["op"] == "grad_norm":
            return {"bytes": read, "flops": 2 * total}
        return {"bytes": read + sum(n * size(_out_dtype(case, t)) for n, t in kinds), "flops": 3 * total}
    n, k, m = case["n"], case["n_in"], case["n_out"]
    if case["op"] == "linear_forward":
        rows = n * k + n * m * (1 + case["residual"] + case["keep"])
        return {"bytes": 2 * (rows + m * k + m * case["bias"]), "flops": 2 * n * k * m}
    rows = n * m * (1 + (case["act"] != "none")) + n * k * (2 + case["residual"])
    grads = (m * k + m * case["bias"]) * (4 if case["grad"] == "f32" else 2) * (1 + case["accumulate"])
    return {"bytes": 2 * (rows + m * k) + grads, "flops": 4 * n * k * m}


def exact(case, seed):
    s = prepare(case, seed)
    if not case["op"].startswith("linear"):
        squares = [torch.dot(g.double(), g.double()) for g in s["grads"]]  # the inputs hold finite values alone
        norm = torch.stack(squares).sum().sqrt() / LOSS_SCALE
        if case["op"] == "grad_norm":
            return {"norm": norm.reshape(1), "nonfinite": None}
        scale = torch.clamp(s["max_norm"] / norm, max=1.0)
        out = {t: torch.zeros_like(f, dtype=torch.float64) for t, f in s["flat"].items()}
        at = dict.fromkeys(out, 0)
        for g in s["grads"]:
            t, n = str(g.dtype), g.numel()
            out[t][at[t]:at[t] + n] = g.double() * scale
            at[t] += _part(n)
        return {"out": out, "norm": norm.reshape(1), "scale": scale.reshape(1), "nonfinite": None}
    x, w = s["x"].double(), s["w"].double()
    bias = s["b"].double() if s["b"] is not None else torch.zeros(case["n_out"], dtype=torch.float64, device="cuda")
    nl = {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
          "gelu": lambda v: v * torch.special.ndtr(v), "sigmoid": torch.sigmoid}[case["act"]]
    if case["op"] == "linear_forward":
        z = torch.addmm(bias, x, w.t())
        y = nl(z) if s["r"] is None else nl(z) + s["r"].double()
        return {"y": y, "z": z} if case["keep"] else {"y": y}
    dz = s["dy"].double()
    if case["act"] != "none":  # the derivative of the activation at z, by the chain rule itself
        z = s["z"].double().requires_grad_(True)
        dz, = torch.autograd.grad(nl(z), z, dz)
    dx, dw, db = torch.mm(dz, w), torch.einsum("no,ni->oi", dz, x), torch.einsum("no->o", dz)
    if s["r"] is not None:
        dx += s["r"].double()
    if case["accumulate"]:
        dw = dw + s["dw"].double()
        db = db + s["db"].double() if s["db"] is not None else db
    return {"dx": dx, "dw": dw, "db": db} if s["db"] is not None else {"dx": dx, "dw": dw}
