"""Dense layer batched over models, with its epilogue and its gradients (host side of csrc/dense.hip).

    y[g] = act(x[g] @ w[g] + bias[g]) + residual[g]

for g over the models of a lockstep batch, beside the trainers' own dense layers (which are fixed to their two models):
kernels are [in][out] as Keras keeps them and may be views into the models' parameter rows, e.g.
``params[:, off:off + k * n].view(G, k, n)``.  Types: float32, bfloat16, float16; sums are fp32.  Rows may have any
stride; the elements of a row are contiguous.  Work goes to torch's current stream of the tensors' device.  No autograd graph
is recorded: in grad mode, tensors that require grad are refused.
"""
import ctypes

import torch

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
_PLANS = {}  # what a call's shapes, strides, types and flags were found to need (_Plan); never an address or a value
MAX_PLANS = 4096


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


def _sig(t):
    """Everything about a tensor that its checks look at."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


class _Plan:
    """A checked call of given shapes: its struct without addresses, the workspace's size, and the bytes each tensor
    spans (for the overlap check, which needs the addresses)."""

    def __init__(self, lib, name, struct, device, fields, tensors):
        self.name, self.device = name, device
        self.fn = getattr(lib, name)
        self.index = device.index
        self.fields = fields  # (struct field, position among the call's tensors, is an output)
        self.struct = type(struct)
        self.workspace = int(getattr(lib, name + "_workspace_bytes")(ctypes.byref(struct)))
        struct.workspace_bytes = self.workspace
        self.bytes = bytes(struct)
        self.spans = [_span(t) for t in tensors]
        self.outs = [i for _, i, out in fields if out and self.spans[i]]
        self.ins = [i for _, i, out in fields if not out and self.spans[i]]
        self.models = struct.n_models

    def run(self, tensors, names, same=(), values=()):
        """Launch on torch's current stream.  same: pairs of positions that may be one and the same tensor; values:
        further fields of the struct."""
        if torch.is_grad_enabled():
            for t in tensors:
                if t is not None and t.requires_grad:
                    raise ValueError(f"{names[[u is t for u in tensors].index(True)]} requires grad, and the batched operators record no graph for it: call them under "
                                     "torch.no_grad() or with detached tensors")
        p = [0 if t is None else t.data_ptr() for t in tensors]
        _no_overlap(tensors, names, p, self.spans, self.outs, self.ins, same)
        st = self.struct.from_buffer_copy(self.bytes)
        for f, i, _ in self.fields:
            if p[i]:
                setattr(st, f, p[i])
        for f, v in values:
            setattr(st, f, v)
        if self.workspace:
            ws = torch.empty(self.workspace, dtype=torch.uint8, device=self.device)
            st.workspace = ws.data_ptr()
        if torch.cuda.current_device() == self.index:
            status = self.fn(ctypes.byref(st), _raw_stream(self.index))
        else:
            with torch.cuda.device(self.index):
                status = self.fn(ctypes.byref(st), _raw_stream(self.index))
        if status:
            _native.check(status, self.name)
        for i in self.outs:  # written behind torch's back
            torch._C._increment_version((tensors[i],))


def _raw_stream(index):
    return torch._C._cuda_getCurrentRawStream(index)


def _remember(key, plan):
    if len(_PLANS) >= MAX_PLANS:
        _PLANS.clear()
    _PLANS[key] = plan
    return plan


def _tensor(t, name, dtype, device, shape):
    """A strided [models][rows][columns] (or [models][columns]) view the kernels can address."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if tuple(t.shape) != tuple(shape):
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


def _span(t):
    """Bytes from a tensor's first element to behind its last."""
    return 0 if t is None or not t.numel() else \
        (1 + sum((d - 1) * s for d, s in zip(t.shape, t.stride()))) * t.element_size()


def _no_overlap(tensors, names, ptrs, spans, outs, ins, same=()):
    """Outputs (positions `outs`) may share no memory with an input or with one another."""
    for k, i in enumerate(outs):
        a, b = ptrs[i], ptrs[i] + spans[i]
        for j in outs[k + 1:] + ins:
            if a < ptrs[j] + spans[j] and ptrs[j] < b and not _interleaved(tensors[i], tensors[j]):
                if not ((i, j) in same and a == ptrs[j] and tensors[i].stride() == tensors[j].stride()):
                    raise ValueError(f"{names[i]} and {names[j]} share memory")


def _interleaved(t, u):
    """Views whose spans cross but whose elements do not: of the same parameter rows at different places of a row, or of the
    same matrix rows at different columns."""
    if t.element_size() != u.element_size():
        return False
    size = t.element_size()
    base = min(t.data_ptr(), u.data_ptr())
    if (t.data_ptr() - base) % size or (u.data_ptr() - base) % size:
        return False
    steps = [[(d, s) for d, s in zip(v.shape, v.stride()) if d > 1] for v in (t, u)]
    for period in {s for dims in steps for _, s in dims if s > 1}:
        # both lie in the same places of every `period` elements
        places = []
        for v, dims in zip((t, u), steps):
            if any(s >= period and s % period for _, s in dims):
                break
            start = (v.data_ptr() - base) // size % period
            places.append((start, start + 1 + sum((d - 1) * s for d, s in dims if s < period)))
        else:
            (a, b), (c, d) = places
            if b <= period and d <= period and (b <= c or d <= a):
                return True
    return False


def _ld(t):
    return max(t.stride(1), t.shape[2]) if t.shape[1] > 1 else t.shape[2]


def _three(t):
    return t if t is None or t.dim() != 2 else t.unsqueeze(0)


def _setup(x, w, activation, counts):
    """The struct's sizes and the shapes (t, G, B, K, N)."""
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
    x3 = _three(x)
    B = x3.shape[1]
    _tensor(x3, "x", w.dtype, w.device, (1 if shared else G, B, K))
    if counts is not None:
        _tensor(counts, "counts", torch.int32, w.device, (G,))
    t = DenseT()
    t.n_models, t.rows, t.in_, t.out = G, B, K, N
    t.dtype, t.activation, t.x_shared = DTYPES[str(w.dtype)], ACTIVATIONS[activation], int(shared)
    t.x_stride, t.x_ld = (0 if shared else x3.stride(0)), _ld(x3)
    t.w_stride, t.w_ld = w.stride(0), _ld(w)
    return t, G, B, K, N


def _place(t, field, tensor):
    setattr(t, field + "_stride", tensor.stride(0))
    if tensor.dim() == 3:
        setattr(t, field + "_ld", _ld(tensor))


_FORWARD = ("out", "preact", "x", "w", "bias", "residual", "counts")
_FORWARD_FIELDS = (("y", 0, True), ("z", 1, True), ("x", 2, False), ("w", 3, False), ("bias", 4, False),
                   ("residual", 5, False), ("counts", 6, False))


def _plan_forward(key, out, preact, x, w, bias, residual, counts, activation):
    t, G, B, K, N = _setup(x, w, activation, counts)
    dev, dt = w.device, w.dtype
    if bias is not None:
        _tensor(bias, "bias", dt, dev, (G, N))
        t.bias_stride = bias.stride(0)
    if residual is not None:
        _tensor(residual, "residual", dt, dev, (G, B, N))
        _place(t, "residual", residual)
    if out is not None:
        _tensor(out, "out", dt, dev, (G, B, N))
        _writable(out, "out")
    if preact is not None:
        _tensor(preact, "preact", torch.float32, dev, (G, B, N))
        _writable(preact, "preact")
        _place(t, "z", preact)
    if out is None:
        out = torch.empty((G, B, N), dtype=dt, device=dev)
    _place(t, "y", out)
    return _remember(key, _Plan(_lib(), "mplc_dense_forward", t, dev, _FORWARD_FIELDS,
                                (out, preact, _three(x), w, bias, residual, counts)))


def dense_forward(x, w, bias=None, residual=None, activation="none", counts=None, preact=None, out=None):
    """act(x @ w + bias) + residual for every model of the batch.

    x [G, B, K], or [1, B, K] / [B, K] shared by all models; w [G, K, N]; bias [G, N]; residual [G, B, N]; all of one
    type.  activation: "none", "relu", "gelu" (of the error function) or "silu".  counts (int32 [G], on the device): rows of each model's
    batch (clamped to [0, B]); rows behind a model's count are not read, and those of `out` and `preact` stay as they
    are.  preact (float32 [G, B, N]): receives x @ w + bias, which dense_backward needs for an activation.
    Returns out [G, B, N] (allocated where not given; then rows behind a count are 0)."""
    try:
        key = (0, activation, _sig(x), _sig(w), _sig(bias), _sig(residual), _sig(counts), _sig(preact), _sig(out))
        plan = _PLANS.get(key)
    except (AttributeError, TypeError):  # not tensors: the checks say so
        key = plan = None
    if plan is None:
        plan = _plan_forward(key, out, preact, x, w, bias, residual, counts, activation)
    if out is None:
        out = (torch.empty if counts is None else torch.zeros)((w.shape[0], x.shape[-2], w.shape[2]), dtype=w.dtype,
                                                               device=w.device)
    plan.run((out, preact, x, w, bias, residual, counts), _FORWARD)
    return out


_BACKWARD = ("dx", "dw", "db", "x", "w", "dout", "preact", "counts")
_BACKWARD_FIELDS = (("dx", 0, True), ("dw", 1, True), ("db", 2, True), ("x", 3, False), ("w", 4, False),
                    ("dy", 5, False), ("z", 6, False), ("counts", 7, False))


def _plan_backward(key, dx, dw, db, x, w, dout, preact, counts, activation, need):
    t, G, B, K, N = _setup(x, w, activation, counts)
    dev, dt = w.device, w.dtype
    if any(n not in ("dx", "dw", "db") for n in need):
        raise ValueError(f"need holds 'dx', 'dw' and 'db' only, not {need}")
    _tensor(dout, "dout", dt, dev, (G, B, N))
    _place(t, "dy", dout)
    if activation != "none":
        if preact is None:
            raise ValueError(f"the gradient of '{activation}' needs preact (dense_forward(..., preact=))")
        _tensor(preact, "preact", torch.float32, dev, (G, B, N))
        _place(t, "z", preact)
    x3 = _three(x)
    if "dx" in need:
        if dx is not None:
            if not isinstance(dx, torch.Tensor):
                raise TypeError("dx must be a tensor")
            if dx.dim() != x.dim():
                raise ValueError(f"dx must have the shape {list(x.shape)}, not {list(dx.shape)}")
            _tensor(_three(dx), "dx", dt, dev, tuple(x3.shape))
            _writable(_three(dx), "dx")
        else:
            dx = torch.empty(x.shape, dtype=dt, device=dev)
        _place(t, "dx", _three(dx))
        t.dx = 16  # wanted: the workspace query looks at that alone
    else:
        dx = None
    for name, field, v, shape in (("dw", "dw", dw, (G, K, N)), ("db", "db", db, (G, N))):
        if name in need:
            if v is not None:
                _tensor(v, name, dt, dev, shape)
                _writable(v, name)
            else:
                v = torch.empty(shape, dtype=dt, device=dev)
            _place(t, field, v)
            setattr(t, field, 16)
            if name == "dw":
                dw = v
            else:
                db = v
    plan = _Plan(_lib(), "mplc_dense_backward", t, dev, _BACKWARD_FIELDS,
                 (_three(dx), dw, db, x3, w, dout, preact if activation != "none" else None, counts))
    return _remember(key, plan)


def dense_backward(dout, x, w, preact=None, activation="none", counts=None, need=("dx", "dw", "db"), dx=None, dw=None,
                   db=None):
    """Gradients of dense_forward's inputs from that of its output: (dx, dw, db); the residual's is dout itself.

    preact: what dense_forward wrote there (required for an activation).  dx has x's shape: a shared x gets the sum over
    the models.  need: which of the three are computed (the others are None).  dx, dw, db may be given; where dx is
    allocated here, rows behind a model's count are 0, and a given dx keeps them (a shared x has no such rows: a row that
    no model reaches gets 0)."""
    need = tuple(need)
    dx, dw, db = (v if n in need else None for n, v in (("dx", dx), ("dw", dw), ("db", db)))
    if activation == "none":
        preact = None
    try:
        key = (1, activation, need, _sig(dout), _sig(x), _sig(w), _sig(preact), _sig(counts), _sig(dx), _sig(dw), _sig(db))
        plan = _PLANS.get(key)
    except (AttributeError, TypeError):
        key = plan = None
    if plan is None:
        plan = _plan_backward(key, dx, dw, db, x, w, dout, preact, counts, activation, need)
    G = w.shape[0]
    if dx is None and "dx" in need:
        dx = (torch.empty if counts is None and G else torch.zeros)(x.shape, dtype=w.dtype, device=w.device)
    if dw is None and "dw" in need:
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device)
    if db is None and "db" in need:
        db = torch.empty((G, w.shape[2]), dtype=w.dtype, device=w.device)
    if G and need:
        plan.run((dx, dw, db, x, w, dout, preact, counts), _BACKWARD)
    elif dx is not None:
        dx.zero_()  # the sum over no models
    return dx, dw, db
