"""Orthogonalised updates of weight matrices, batched over models (host side of csrc/muon.hip).

``orthogonalize`` brings the singular values of every matrix of a batch near one by Newton-Schulz products;
``muon_step`` is the Muon update of weights kept as [in][out] matrices, for instance views into the models' parameter rows
(``glob[:, off:off + k * n].view(C, k, n)``).  Beside mplc.fedavg: the engine uses it as the server's optimizer after a
round's average (``CoalitionEngine(server_optimizer=...)``).  Work goes to torch's current stream of the device.
"""
import ctypes
import math

from . import _native
from .dense import DTYPES, _ld, _no_overlap, _place, _run, _tensor, _writable

# a s + b s^3 + c s^5 per step: takes singular values of 0.01 .. 1 to about 0.7 .. 1.2 in five steps
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5


class MuonT(ctypes.Structure):
    _fields_ = [("n_models", ctypes.c_int32), ("rows", ctypes.c_int32), ("cols", ctypes.c_int32),
                ("dtype", ctypes.c_int32), ("steps", ctypes.c_int32), ("nesterov", ctypes.c_int32),
                ("a", ctypes.c_float), ("b", ctypes.c_float), ("c", ctypes.c_float), ("lr", ctypes.c_float),
                ("beta", ctypes.c_float), ("weight_decay", ctypes.c_float), ("scale", ctypes.c_float),
                ("pad0", ctypes.c_float),
                ("g", ctypes.c_void_p), ("g_stride", ctypes.c_int64), ("g_ld", ctypes.c_int64),
                ("out", ctypes.c_void_p), ("out_stride", ctypes.c_int64), ("out_ld", ctypes.c_int64),
                ("m", ctypes.c_void_p), ("m_stride", ctypes.c_int64), ("m_ld", ctypes.c_int64),
                ("w", ctypes.c_void_p), ("w_stride", ctypes.c_int64), ("w_ld", ctypes.c_int64),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


_LIB = None


class _Lib:
    """The two calls under the names _run uses, with their one workspace query."""

    def __init__(self, lib):
        self.mplc_orthogonalize, self.mplc_muon_step = lib.mplc_orthogonalize, lib.mplc_muon_step
        self.mplc_orthogonalize_workspace_bytes = self.mplc_muon_step_workspace_bytes = lib.mplc_muon_workspace_bytes


def _lib():
    global _LIB
    if _LIB is None:
        p = ctypes.POINTER(MuonT)
        lib = _native.lib()
        _native.register("mplc_muon_workspace_bytes", ctypes.c_size_t, [p])
        for name in ("mplc_orthogonalize", "mplc_muon_step"):
            _native.register(name, ctypes.c_int, [p, ctypes.c_void_p])
        _native.check_layout(lib.mplc_ops_layout, {"MUON_T_BYTES": (1, ctypes.sizeof(MuonT))}, "orthogonalised update")
        _LIB = _Lib(lib)
    return _LIB


def singular_range(steps, coefficients):
    """The largest singular value that `steps` steps can reach at any time from [0, 1]."""
    a, b, c = coefficients
    r = most = 1.0
    for _ in range(steps):
        roots = [r]
        if c == 0.0:
            q = [-a / (3 * b)] if b != 0.0 else []
        else:
            d = 9 * b * b - 20 * a * c
            q = [(-3 * b + s * math.sqrt(d)) / (10 * c) for s in (1, -1)] if d >= 0 else []
        roots += [math.sqrt(v) for v in q if 0 < v < r * r]
        r = max(abs(s * (a + s * s * (b + s * s * c))) for s in roots)
        most = max(most, r)
    return most


def _setup(g, name, steps, coefficients):
    import torch
    if not isinstance(g, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not g.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if str(g.dtype) not in DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {g.dtype}")
    if g.dim() not in (2, 3):
        raise ValueError(f"{name} must be [models, rows, cols] or [rows, cols], not {list(g.shape)}")
    g3 = g if g.dim() == 3 else g.unsqueeze(0)
    G, m, n = g3.shape
    if m < 1 or n < 1:
        raise ValueError(f"{name} has no elements: {list(g.shape)}")
    if G > 65535:
        raise ValueError("at most 65535 models per call")
    _tensor(g3, name, g.dtype, g.device, (G, m, n))
    if not 1 <= int(steps) <= 16:
        raise ValueError(f"steps must be 1 to 16, not {steps}")
    coefficients = tuple(float(v) for v in coefficients)
    if len(coefficients) != 3 or not all(abs(v) < 1e3 for v in coefficients):
        raise ValueError(f"coefficients must be three finite numbers (a, b, c), not {coefficients}")
    if singular_range(int(steps), coefficients) > 2.0:
        raise ValueError(f"coefficients {coefficients} let singular values grow past 2")
    t = MuonT()
    t.n_models, t.rows, t.cols, t.dtype, t.steps = G, m, n, DTYPES[str(g.dtype)], int(steps)
    t.a, t.b, t.c = coefficients
    t.g, t.g_stride, t.g_ld = g3.data_ptr(), g3.stride(0), _ld(g3)
    return t, g3


def orthogonalize(g, steps=STEPS, coefficients=COEFFICIENTS, out=None):
    """Each matrix of g ([G, m, n] or [m, n]) divided by its Frobenius norm, then `steps` times
    X <- a X + b (X X^T) X + c (X X^T)^2 X.  A zero matrix stays zero; one with an infinity or a NaN becomes NaN.
    Sums and intermediate matrices keep fp32's accuracy whatever g's type; the result is rounded to it once."""
    import torch
    t, g3 = _setup(g, "g", steps, coefficients)
    if out is None:
        out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    if out.dim() != g.dim():
        raise ValueError(f"out must have the shape {list(g.shape)}, not {list(out.shape)}")
    o3 = out if out.dim() == 3 else out.unsqueeze(0)
    _tensor(o3, "out", g.dtype, g.device, tuple(g3.shape))
    _writable(o3, "out")
    _place(t, "out", o3)
    if not (out.data_ptr() == g.data_ptr() and out.stride() == g.stride()):  # in place is fine: g is read first
        _no_overlap([("out", o3)], [("g", g3)])
    if t.n_models:
        _run(_lib(), "mplc_orthogonalize", t, g.device)
    return out


def update_scale(rows, cols):
    """sqrt(max(1, out / in)) of an [in][out] matrix: a step's size per output does not depend on the shape."""
    return math.sqrt(max(1.0, cols / rows))


def muon_step(w, grad, momentum, lr, beta=0.95, nesterov=True, weight_decay=0.0, steps=STEPS,
              coefficients=COEFFICIENTS, scale=None):
    """One Muon step on each matrix w [G, in, out] (or [in, out]), in place:

        momentum <- beta momentum + grad;   u = grad + beta momentum (nesterov) or momentum
        w <- (1 - lr weight_decay) w - lr scale orthogonalize(u)

    w and momentum are float32, grad any supported type; scale None: update_scale(in, out).  Returns w."""
    import torch
    t, g3 = _setup(grad, "grad", steps, coefficients)
    for name, v in (("w", w), ("momentum", momentum)):
        if not isinstance(v, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if v.shape != grad.shape:
            raise ValueError(f"{name} must have the shape {list(grad.shape)}, not {list(v.shape)}")
    w3, m3 = (w, momentum) if w.dim() == 3 else (w.unsqueeze(0), momentum.unsqueeze(0))
    for name, field, v in (("w", "w", w3), ("momentum", "m", m3)):
        _tensor(v, name, torch.float32, grad.device, tuple(g3.shape))
        _writable(v, name)
        _place(t, field, v)
    _no_overlap([("w", w3), ("momentum", m3)], [("grad", g3)])
    scale = update_scale(t.rows, t.cols) if scale is None else float(scale)
    values = {"lr": float(lr), "beta": float(beta), "weight_decay": float(weight_decay), "scale": scale}
    if not all(math.isfinite(v) for v in values.values()):
        raise ValueError(f"lr, beta, weight_decay and scale must be finite: {values}")
    t.nesterov = int(bool(nesterov))
    t.lr, t.beta, t.weight_decay, t.scale = float(lr), float(beta), float(weight_decay), scale
    if t.n_models:
        _run(_lib(), "mplc_muon_step", t, grad.device)
    return w
