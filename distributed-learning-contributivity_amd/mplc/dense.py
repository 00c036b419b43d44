"""Dense layer batched over models, with its epilogue and its gradients (host side of csrc/dense.hip).

    y[g] = act(x[g] @ w[g] + bias[g]) + residual[g]

for g over the models of a lockstep batch, beside the trainers' own dense layers (which are fixed to their two models):
kernels are [in][out] as Keras keeps them and may be views into the models' parameter rows, e.g.
``params[:, off:off + k * n].view(G, k, n)``.  Types: float32, bfloat16, float16; sums are fp32.  Rows may have any
stride; the elements of a row are contiguous.  Work goes to torch's current stream of the tensors' device.
"""
import ctypes

from . import _native

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
DTYPES = {"torch.float32": 0, "torch.bfloat16": 1, "torch.float16": 2}
MAX_SIZE = (1 << 31) - 1024


class DenseT(ctypes.Structure):
    _fields_ = [("n_models", ctypes.c_int32), ("rows", ctypes.c_int32), ("in_", ctypes.c_int32),
                ("out", ctypes.c_int32), ("dtype", ctypes.c_int32), ("activation", ctypes.c_int32),
                ("x_shared", ctypes.c_int32), ("pad0", ctypes.c_int32), ("counts", ctypes.c_void_p),
                ("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("x_ld", ctypes.c_int64),
                ("w", ctypes.c_void_p), ("w_stride", ctypes.c_int64), ("w_ld", ctypes.c_int64),
                ("bias", ctypes.c_void_p), ("bias_stride", ctypes.c_int64),
                ("residual", ctypes.c_void_p), ("residual_stride", ctypes.c_int64), ("residual_ld", ctypes.c_int64),
                ("y", ctypes.c_void_p), ("y_stride", ctypes.c_int64), ("y_ld", ctypes.c_int64),
                ("z", ctypes.c_void_p), ("z_stride", ctypes.c_int64), ("z_ld", ctypes.c_int64),
                ("dy", ctypes.c_void_p), ("dy_stride", ctypes.c_int64), ("dy_ld", ctypes.c_int64),
                ("dx", ctypes.c_void_p), ("dx_stride", ctypes.c_int64), ("dx_ld", ctypes.c_int64),
                ("dw", ctypes.c_void_p), ("dw_stride", ctypes.c_int64), ("dw_ld", ctypes.c_int64),
                ("db", ctypes.c_void_p), ("db_stride", ctypes.c_int64),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


_LIB = None


def _lib():
    global _LIB
    if _LIB is None:
        p = ctypes.POINTER(DenseT)
        lib = _native.lib()
        for name in ("mplc_dense_forward_workspace_bytes", "mplc_dense_backward_workspace_bytes"):
            _native.register(name, ctypes.c_size_t, [p])
        for name in ("mplc_dense_forward", "mplc_dense_backward"):
            _native.register(name, ctypes.c_int, [p, ctypes.c_void_p])
        _native.check_layout(lib.mplc_ops_layout, {"DENSE_T_BYTES": (0, ctypes.sizeof(DenseT))}, "dense layer")
        _LIB = lib
    return _LIB


def _tensor(t, name, dtype, device, shape):
    """A strided [models][rows][columns] (or [models][columns]) view the kernels can address; `shape` entries of None
    are free."""
    import torch
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if t.dim() != len(shape) or any(s is not None and s != d for s, d in zip(shape, t.shape)):
        raise ValueError(f"{name} must have the shape {list(shape)}, not {list(t.shape)}")
    if any(d > MAX_SIZE for d in t.shape):
        raise ValueError(f"{name} is too large: {list(t.shape)}")
    if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"the elements of a row of {name} must be contiguous (strides {t.stride()})")
    if t.dim() == 3 and t.numel() and t.shape[1] > 1 and t.stride(1) < t.shape[2]:
        raise ValueError(f"the rows of {name} overlap (strides {t.stride()})")


def _writable(t, name):
    """An output's models may not overlap one another either."""
    if t.numel() and t.shape[0] > 1:
        last = (t.shape[1] - 1) * t.stride(1) + t.shape[2] if t.dim() == 3 else t.shape[1]
        inside = t.stride(0) >= last
        # models side by side inside the rows of one matrix
        beside = t.dim() == 3 and t.stride(0) >= t.shape[2] and (
            t.shape[1] == 1 or t.stride(1) >= (t.shape[0] - 1) * t.stride(0) + t.shape[2])
        if not (inside or beside):
            raise ValueError(f"the models of {name} overlap (strides {t.stride()})")


def _no_overlap(outs, ins):
    """Outputs may share no memory with an input or with one another (checked on the spans the tensors cover)."""
    def span(t):
        n = 1 + sum((d - 1) * s for d, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + n * t.element_size()
    outs = [(n, t) for n, t in outs if t is not None and t.numel()]
    ins = [(n, t) for n, t in ins if t is not None and t.numel()]
    for i, (n, t) in enumerate(outs):
        a, b = span(t)
        for m, u in outs[i + 1:] + ins:
            c, d = span(u)
            if a < d and c < b and not _interleaved(t, u):
                raise ValueError(f"{n} and {m} share memory")


def _interleaved(t, u):
    """Views of the same parameter rows at different places of a row: the spans cross, the elements do not."""
    if t.dim() < 2 or u.dim() < 2 or t.element_size() != u.element_size():
        return False
    s = t.stride(0)
    if s <= 0 or s != u.stride(0) or t.shape[0] < 2 or u.shape[0] < 2:
        return False
    size = t.element_size()
    base = min(t.data_ptr(), u.data_ptr())
    places = []
    for v in (t, u):
        start = (v.data_ptr() - base) // size % s
        n = 1 + sum((d - 1) * k for d, k in zip(v.shape[1:], v.stride()[1:]))
        places.append((start, start + n))
    (a, b), (c, d) = places
    return b <= s and d <= s and (b <= c or d <= a)


def _ld(t):
    return max(t.stride(1), t.shape[2]) if t.shape[1] > 1 else t.shape[2]


def _setup(x, w, activation, counts):
    """The struct's sizes, and the shapes: (t, G, B, K, N, x as [1 or G, B, K])."""
    import torch
    if not isinstance(x, torch.Tensor) or not isinstance(w, torch.Tensor):
        raise TypeError("x and w must be tensors")
    if not w.is_cuda:
        raise ValueError("w must be a CUDA tensor")
    if str(w.dtype) not in DTYPES:
        raise ValueError(f"w must be float32, bfloat16 or float16, not {w.dtype}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation '{activation}' is not one of {', '.join(ACTIVATIONS)}")
    if w.dim() != 3:
        raise ValueError(f"w must be [models, in, out], not {list(w.shape)}")
    G, K, N = w.shape
    if K < 1 or N < 1:
        raise ValueError(f"w must have at least one input and one output: {list(w.shape)}")
    if G > 65535:
        raise ValueError("at most 65535 models per call")
    _tensor(w, "w", w.dtype, w.device, (G, K, N))
    if x.dim() not in (2, 3):
        raise ValueError(f"x must be [models, rows, in], or [1, rows, in] or [rows, in] shared by all models, "
                         f"not {list(x.shape)}")
    shared = x.dim() == 2 or (x.shape[0] == 1 and G != 1)
    x3 = x.unsqueeze(0) if x.dim() == 2 else x
    B = x3.shape[1]
    _tensor(x3, "x", w.dtype, w.device, (1 if shared else G, B, K))
    if counts is not None:
        _tensor(counts, "counts", torch.int32, w.device, (G,))
    t = DenseT()
    t.n_models, t.rows, t.in_, t.out = G, B, K, N
    t.dtype, t.activation, t.x_shared = DTYPES[str(w.dtype)], ACTIVATIONS[activation], int(shared)
    t.counts = None if counts is None else counts.data_ptr()
    t.x, t.x_stride, t.x_ld = x3.data_ptr(), (0 if shared else x3.stride(0)), _ld(x3)
    t.w, t.w_stride, t.w_ld = w.data_ptr(), w.stride(0), _ld(w)
    return t, G, B, K, N, x3


def _place(t, field, tensor):
    setattr(t, field, tensor.data_ptr())
    setattr(t, field + "_stride", tensor.stride(0))
    if tensor.dim() == 3:
        setattr(t, field + "_ld", _ld(tensor))


def _run(lib, name, t, device):
    import torch
    n = getattr(lib, name + "_workspace_bytes")(ctypes.byref(t))
    ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    t.workspace, t.workspace_bytes = (ws.data_ptr() if n else None), n
    with torch.cuda.device(device):
        _native.check(getattr(lib, name)(ctypes.byref(t), _native.stream_handle(device)), name)


def dense_forward(x, w, bias=None, residual=None, activation="none", counts=None, preact=None, out=None):
    """act(x @ w + bias) + residual for every model of the batch.

    x [G, B, K], or [1, B, K] / [B, K] shared by all models; w [G, K, N]; bias [G, N]; residual [G, B, N]; all of one
    type.  activation: "none", "relu", "gelu" (exact) or "silu".  counts (int32 [G], on the device): rows of each model's
    batch (clamped to [0, B]); rows behind a model's count are not read, and those of `out` and `preact` stay as they
    are.  preact (float32 [G, B, N]): receives x @ w + bias, which dense_backward needs for an activation.
    Returns out [G, B, N] (allocated where not given; then rows behind a count are 0)."""
    import torch
    t, G, B, K, N, x3 = _setup(x, w, activation, counts)
    dev, dt = w.device, w.dtype
    if bias is not None:
        _tensor(bias, "bias", dt, dev, (G, N))
        t.bias, t.bias_stride = bias.data_ptr(), bias.stride(0)
    if residual is not None:
        _tensor(residual, "residual", dt, dev, (G, B, N))
        _place(t, "residual", residual)
    if out is None:
        out = (torch.empty if counts is None else torch.zeros)((G, B, N), dtype=dt, device=dev)
    _tensor(out, "out", dt, dev, (G, B, N))
    _writable(out, "out")
    _place(t, "y", out)
    if preact is not None:
        _tensor(preact, "preact", torch.float32, dev, (G, B, N))
        _writable(preact, "preact")
        _place(t, "z", preact)
    _no_overlap([("out", out), ("preact", preact)],
                [("x", x3), ("w", w), ("bias", bias), ("residual", residual), ("counts", counts)])
    if G and B:
        _run(_lib(), "mplc_dense_forward", t, dev)
    return out


def dense_backward(dout, x, w, preact=None, activation="none", counts=None, need=("dx", "dw", "db"), dx=None, dw=None,
                   db=None):
    """Gradients of dense_forward's inputs from that of its output: (dx, dw, db); the residual's is dout itself.

    preact: what dense_forward wrote there (required for an activation).  dx has x's shape: a shared x gets the sum over
    the models.  need: which of the three are computed (the others are None).  dx, dw, db may be given; where dx is
    allocated here, rows behind a model's count are 0, and a given dx keeps them (a shared x has no such rows: a row that
    no model reaches gets 0)."""
    import torch
    t, G, B, K, N, x3 = _setup(x, w, activation, counts)
    dev, dt = w.device, w.dtype
    need = tuple(need)
    if any(n not in ("dx", "dw", "db") for n in need):
        raise ValueError(f"need holds 'dx', 'dw' and 'db' only, not {need}")
    _tensor(dout, "dout", dt, dev, (G, B, N))
    _place(t, "dy", dout)
    if activation != "none":
        if preact is None:
            raise ValueError(f"the gradient of '{activation}' needs preact (dense_forward(..., preact=))")
        _tensor(preact, "preact", torch.float32, dev, (G, B, N))
        _place(t, "z", preact)
    if "dx" in need:
        if dx is None:
            dx = (torch.empty if counts is None and G else torch.zeros)(x.shape, dtype=dt, device=dev)
        if dx.dim() != x.dim():
            raise ValueError(f"dx must have the shape {list(x.shape)}, not {list(dx.shape)}")
        dx3 = dx.unsqueeze(0) if dx.dim() == 2 else dx
        _tensor(dx3, "dx", dt, dev, tuple(x3.shape))
        _writable(dx3, "dx")
        _place(t, "dx", dx3)
    else:
        dx = dx3 = None
    if "dw" in need:
        dw = torch.empty((G, K, N), dtype=dt, device=dev) if dw is None else dw
        _tensor(dw, "dw", dt, dev, (G, K, N))
        _writable(dw, "dw")
        _place(t, "dw", dw)
    else:
        dw = None
    if "db" in need:
        db = torch.empty((G, N), dtype=dt, device=dev) if db is None else db
        _tensor(db, "db", dt, dev, (G, N))
        _writable(db, "db")
        t.db, t.db_stride = db.data_ptr(), db.stride(0)
    else:
        db = None
    _no_overlap([("dx", dx3), ("dw", dw), ("db", db)],
                [("x", x3), ("w", w), ("dout", dout), ("preact", preact if activation != "none" else None),
                 ("counts", counts)])
    if G and need:
        _run(_lib(), "mplc_dense_backward", t, dev)
    return dx, dw, db
