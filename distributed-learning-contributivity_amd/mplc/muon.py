"""Orthogonalised updates of weight matrices, batched over models (host side of csrc/muon.hip).

``orthogonalize`` brings the singular values of every matrix of a batch near one by Newton-Schulz products;
``muon_step`` is the Muon update of weights kept as [in][out] matrices, for instance views into the models' parameter rows
(``glob[:, off:off + k * n].view(C, k, n)``).  Beside mplc.fedavg: the engine uses it as the server's optimizer after a
round's average (``CoalitionEngine(server_optimizer=...)``).  Work goes to torch's current stream of the device.  No autograd
graph is recorded: in grad mode, tensors that require grad are refused.
"""
import ctypes
import math
import operator

import torch

from . import _native
from .dense import _PLANS, DTYPES, _Plan, _ld, _place, _remember, _sig, _tensor, _three, _writable

# a s + b s^3 + c s^5 per step: takes singular values of 0.01 .. 1 to about 0.7 .. 1.2 in five steps
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
MAX_FLOAT = 3.4e38


class MuonT(ctypes.Structure):
    _fields_ = [("n_models", ctypes.c_int32), ("rows", ctypes.c_int32), ("cols", ctypes.c_int32),
                ("dtype", ctypes.c_int32), ("steps", ctypes.c_int32), ("nesterov", ctypes.c_int32),
                ("invariant", ctypes.c_int32), ("a", ctypes.c_float), ("b", ctypes.c_float), ("c", ctypes.c_float), ("lr", ctypes.c_float),
                ("beta", ctypes.c_float), ("weight_decay", ctypes.c_float), ("scale", ctypes.c_float),
                ("g", ctypes.c_void_p), ("g_stride", ctypes.c_int64), ("g_ld", ctypes.c_int64),
                ("out", ctypes.c_void_p), ("out_stride", ctypes.c_int64), ("out_ld", ctypes.c_int64),
                ("m", ctypes.c_void_p), ("m_stride", ctypes.c_int64), ("m_ld", ctypes.c_int64),
                ("w", ctypes.c_void_p), ("w_stride", ctypes.c_int64), ("w_ld", ctypes.c_int64),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


_LIB = None


class _Lib:
    """The two calls under the names a plan uses, with their one workspace query."""

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


def _setup(g, name, steps, coefficients, invariant):
    if not isinstance(g, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not g.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if str(g.dtype) not in DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {g.dtype}")
    if g.dim() not in (2, 3):
        raise ValueError(f"{name} must be [models, rows, cols] or [rows, cols], not {list(g.shape)}")
    g3 = _three(g)
    G, m, n = g3.shape
    if m < 1 or n < 1:
        raise ValueError(f"{name} has no elements: {list(g.shape)}")
    if G > 65535:
        raise ValueError("at most 65535 models per call")
    _tensor(g3, name, g.dtype, g.device, (G, m, n))
    if not 1 <= operator.index(steps) <= 16:
        raise ValueError(f"steps must be 1 to 16, not {steps}")
    coefficients = tuple(float(v) for v in coefficients)
    if len(coefficients) != 3 or not all(abs(v) < 1e3 for v in coefficients):
        raise ValueError(f"coefficients must be three finite numbers (a, b, c), not {coefficients}")
    if singular_range(operator.index(steps), coefficients) > 2.0:
        raise ValueError(f"coefficients {coefficients} let singular values grow past 2")
    t = MuonT()
    t.n_models, t.rows, t.cols, t.dtype, t.steps = G, m, n, DTYPES[str(g.dtype)], operator.index(steps)
    t.a, t.b, t.c = coefficients
    t.invariant = int(bool(invariant))
    _place(t, "g", g3)
    return t, g3


def _key(kind, steps, coefficients, invariant, tensors):
    try:  # numbers, not what holds them: a key is compared by value
        return (kind, operator.index(steps), tuple(float(v) for v in coefficients), bool(invariant)) + tuple(_sig(t) for t in tensors)
    except (AttributeError, TypeError, ValueError):  # not tensors, not numbers: the checks say so
        return None


def _plan_orthogonalize(key, out, g, steps, coefficients, invariant):
    t, g3 = _setup(g, "g", steps, coefficients, invariant)
    if out is None:
        out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    if not isinstance(out, torch.Tensor):
        raise TypeError("out must be a tensor")
    if out.dim() != g.dim():
        raise ValueError(f"out must have the shape {list(g.shape)}, not {list(out.shape)}")
    _tensor(_three(out), "out", g.dtype, g.device, tuple(g3.shape))
    _writable(_three(out), "out")
    _place(t, "out", _three(out))
    return _remember(key, _Plan(_lib(), "mplc_orthogonalize", t, g.device, (("out", 0, True), ("g", 1, False)),
                                (_three(out), g3)))


def orthogonalize(g, steps=STEPS, coefficients=COEFFICIENTS, out=None, batch_invariant=False):
    """Each matrix of g ([G, m, n] or [m, n]) divided by its Frobenius norm, then `steps` times
    X <- a X + b (X X^T) X + c (X X^T)^2 X.  A zero matrix stays zero; one with an infinity or a NaN becomes NaN.
    Sums and intermediate matrices keep fp32's accuracy whatever g's type; the result is rounded to it once.
    out may be g itself.  batch_invariant: a matrix's result has the same bits whichever matrices share the call (its
    sums are then split in one way, not in the best one for the batch)."""
    key = _key(2, steps, coefficients, batch_invariant, (g, out))
    plan = _PLANS.get(key) if key is not None else None
    if plan is None:
        plan = _plan_orthogonalize(key, out, g, steps, coefficients, batch_invariant)
    if out is None:
        out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    if plan.models:
        plan.run((out, g), ("out", "g"), same=((0, 1),))  # in place: g is read before anything is written
    return out


def update_scale(rows, cols):
    """sqrt(max(1, out / in)) of an [in][out] matrix: a step's size per output does not depend on the shape."""
    return math.sqrt(max(1.0, cols / rows))


def _plan_step(key, w, grad, momentum, steps, coefficients, invariant):
    t, g3 = _setup(grad, "grad", steps, coefficients, invariant)
    for name, field, v in (("w", "w", w), ("momentum", "m", momentum)):
        if not isinstance(v, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if v.shape != grad.shape:
            raise ValueError(f"{name} must have the shape {list(grad.shape)}, not {list(v.shape)}")
        _tensor(_three(v), name, torch.float32, grad.device, tuple(g3.shape))
        _writable(_three(v), name)
        _place(t, field, _three(v))
    return _remember(key, _Plan(_lib(), "mplc_muon_step", t, grad.device, (("w", 0, True), ("m", 1, True), ("g", 2, False)),
                                (_three(w), _three(momentum), g3)))


def muon_step(w, grad, momentum, lr, beta=0.95, nesterov=True, weight_decay=0.0, steps=STEPS,
              coefficients=COEFFICIENTS, scale=None, batch_invariant=False):
    """One Muon step on each matrix w [G, in, out] (or [in, out]), in place:

        momentum <- beta momentum + grad;   u = grad + beta momentum (nesterov) or momentum
        w <- (1 - lr weight_decay) w - lr scale orthogonalize(u)

    w and momentum are float32, grad any supported type; scale None: update_scale(in, out).  batch_invariant: as for
    orthogonalize.  Returns w."""
    key = _key(3, steps, coefficients, batch_invariant, (w, grad, momentum))
    plan = _PLANS.get(key) if key is not None else None
    if plan is None:
        plan = _plan_step(key, w, grad, momentum, steps, coefficients, batch_invariant)
    rows, cols = grad.shape[-2:]
    scale = update_scale(rows, cols) if scale is None else float(scale)
    lr, beta, weight_decay = float(lr), float(beta), float(weight_decay)
    if not all(abs(v) < MAX_FLOAT for v in (lr, lr * scale, beta, weight_decay, lr * weight_decay, scale)):  # as fp32, and not NaN
        raise ValueError(f"lr, beta, weight_decay and scale must be finite: {lr}, {beta}, {weight_decay}, {scale}")
    if plan.models:
        plan.run((w, momentum, grad), ("w", "momentum", "grad"), values=(
            ("lr", lr), ("beta", beta), ("weight_decay", weight_decay), ("scale", scale), ("nesterov", int(bool(nesterov)))))
    return w


class ServerMuon:
    """The server's optimizer of federated averaging: after a round's average, the matrices of a coalition's model move
    from where they stood before the round by a Muon step along (before - average) instead of taking the average; the
    other layers (biases) take it.  Convolution kernels [kh][kw][cin][cout] are [kh * kw * cin][cout] matrices.

    spec: {"name": "muon", "lr": .., and optionally "beta", "nesterov", "weight_decay", "steps"}, or "muon" for the defaults.
    Every coalition's result is independent of the coalitions it shares a batch with."""
    DEFAULTS = {"lr": 0.02, "beta": 0.9, "nesterov": True, "weight_decay": 0.0, "steps": STEPS}
    GROUP = 64  # coalitions per call: bounds the workspace

    def __init__(self, spec):
        if isinstance(spec, str):
            spec = {"name": spec}
        spec = dict(spec)
        name = spec.pop("name", None)
        if name != "muon":
            raise ValueError(f"server optimizer '{name}' is not a valid one: 'muon'")
        unknown = sorted(set(spec) - set(self.DEFAULTS))
        if unknown:
            raise ValueError(f"server optimizer 'muon' has no parameter {', '.join(unknown)}")
        self.params = {**self.DEFAULTS, **spec}
        p = self.params
        numbers = [float(p[k]) for k in ("lr", "beta", "weight_decay")]
        if not all(math.isfinite(v) for v in numbers) or not 0.0 <= numbers[1] < 1.0 or numbers[0] <= 0.0:
            raise ValueError(f"server optimizer 'muon': lr must be positive and beta in [0, 1): {p}")
        if int(p["steps"]) != p["steps"] or not 1 <= p["steps"] <= 16:
            raise ValueError(f"server optimizer 'muon': steps must be 1 to 16, not {p['steps']}")

    def describe(self):
        """A plain value that tells runs with different settings apart (the fingerprint of persisted values)."""
        return {"name": "muon", **self.params}

    @staticmethod
    def matrices(layers):
        """(offset, rows, cols) of the matrices among a model row's layers (offset, shape)."""
        return [(off, math.prod(shape[:-1]), shape[-1]) for off, shape in layers if len(shape) > 1]

    def step_bytes(self, layers, stride):
        """Device memory that apply() takes for each of a group's models: their differences and the steps' workspaces (those of
        different sizes side by side, as the allocator keeps a freed block for its size)."""
        total = 4 * stride
        for _, rows, cols in self.matrices(layers):
            t = MuonT()
            t.n_models, t.rows, t.cols, t.steps, t.invariant = self.GROUP, rows, cols, int(self.params["steps"]), 1
            total += -(-_lib().mplc_muon_step_workspace_bytes(ctypes.byref(t)) // self.GROUP)
        return total

    def apply(self, glob, before, momentum, layers):
        """glob, before, momentum [C, stride]: glob holds the round's averages and receives the new models; before, the
        models at the round's start, is used up."""
        for c in range(0, glob.shape[0], self.GROUP):
            g, b, m = glob[c:c + self.GROUP], before[c:c + self.GROUP], momentum[c:c + self.GROUP]
            grad = b - g
            for off, rows, cols in self.matrices(layers):
                w, d, mm = (t[:, off:off + rows * cols].view(t.shape[0], rows, cols) for t in (b, grad, m))
                muon_step(w, d, mm, lr=self.params["lr"], beta=self.params["beta"], nesterov=self.params["nesterov"],
                          weight_decay=self.params["weight_decay"], steps=int(self.params["steps"]),
                          batch_invariant=True)
                g[:, off:off + rows * cols].copy_(b[:, off:off + rows * cols])
