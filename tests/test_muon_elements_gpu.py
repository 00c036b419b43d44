"""GPU: the orthogonalised update element by element.  A norm over the matrix hides one wrong element at a cut row or column,
and bounds that allow for the growth of small singular values hide a lost half of the split operands."""
import pytest
import torch

from mplc import muon
from test_dense_gpu import half, tiny
from test_muon_gpu import SIZES, TYPES, rand
from test_operator_edges_gpu import LONG

pytestmark = pytest.mark.gpu
ALL = sorted(set(SIZES + LONG + [(300, 200), (200, 300), (150, 1000), (513, 257)]))
COEF = (1.0, -0.2, 0.1)  # P = a + b q + c q^2 stays in [0.9, 1]: a step hardly amplifies an error


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", ALL, ids=lambda s: "x".join(map(str, s)))
def test_16_bit_results_are_the_fp32_ones_rounded_once(size, dtype):
    """A 16-bit update is read exactly and summed as its fp32 copy is; only the result's rounding differs."""
    g = rand((2,) + size, TYPES[dtype], seed=sum(size))
    assert torch.equal(muon.orthogonalize(g), muon.orthogonalize(g.float()).to(g.dtype))
    w, m = rand((2,) + size, seed=1), rand((2,) + size, seed=2)
    w2, m2 = w.clone(), m.clone()
    muon.muon_step(w, g, m, lr=0.1, weight_decay=0.1)
    muon.muon_step(w2, g.float(), m2, lr=0.1, weight_decay=0.1)
    assert torch.equal(w, w2) and torch.equal(m, m2)


def scalar_bound(q, terms):
    """Relative error of an element whose column has the squared singular value q, for whichever phases the form takes.

    rho: a value in split fp16, and each product's and sum's rounding, 2^-22 at most.  A Gram element sums `terms` products of
    one sign and exact zeros, three matrix instructions each: (3 terms + 4) 2^-24 and its operands' 3 rho; |U| half of that.
    Then the scalar recurrence with every error at its worst: P's from q's, A <- P A P, Q <- P Q, X <- X Q."""
    rho, most = 2.0 ** -22, None
    gram = 3 * rho + (3 * terms + 4) * 2.0 ** -24
    a, b, c = COEF
    for phases in ([3, 2], [2, 2, 1], [1] * 5):
        rx, x2 = rho + gram / 2, q.clone()
        for n in phases:
            d, qq, rq = 2 * rx + gram, x2.clone(), torch.zeros_like(q)
            for _ in range(n):
                p = a + b * qq + c * qq * qq
                rp = (abs(b) * qq * (d + rho) + abs(c) * qq * qq * (2 * d + 3 * rho)) / p + 2 * rho
                rq = rq + rp + 2 * rho
                d = d + 2 * rp + 4 * rho
                qq, x2 = p * p * qq, p * p * x2
            rx = rx + rq + 2 * rho
        most = rx if most is None else torch.maximum(most, rx)
    return most


@pytest.mark.parametrize("size", ALL, ids=lambda s: "x".join(map(str, s)))
def test_elements_of_matrices_with_orthogonal_columns(size):
    """One element per row of the long side: the columns are orthogonal, every sum has terms of one sign and zeros, and each
    element of O(u) is its u times a number of its column.  The elements between are 0 exactly.  X is held at a scale of
    2^14, where fp16's last place is 2^-24: 2^-39 of |u|, once for each phase and the start, at most 6."""
    k, L = min(size), max(size)
    v = rand((3, L), seed=L + k).cpu()
    col = torch.arange(L) % k
    v = v * 0.5 ** col.clamp(max=6)  # singular values of every size below 1
    u = torch.zeros(3, L, k)
    u[:, torch.arange(L), col] = v
    g = (u if size[0] >= size[1] else u.transpose(1, 2).contiguous()).cuda()
    out = muon.orthogonalize(g, coefficients=COEF).cpu()
    out = out if size[0] >= size[1] else out.transpose(1, 2)
    off = torch.ones(L, k, dtype=torch.bool)
    off[torch.arange(L), col] = False
    assert (out[:, off] == 0).all()
    for i in range(3):
        x = v[i].double() / v[i].double().norm()
        q = torch.zeros(k, dtype=torch.float64).index_add_(0, col, x * x)
        s, f = q.clone(), torch.ones(k, dtype=torch.float64)
        for _ in range(5):
            p = COEF[0] + COEF[1] * s + COEF[2] * s * s
            s, f = s * p * p, f * p
        want = x * f[col]
        err = want.abs() * scalar_bound(q, -(-L // k))[col] + 6 * 2.0 ** -39
        got = out[i, torch.arange(L), col].double()
        assert ((got - want).abs() <= err + half(torch.float32) * (want.abs() + err) + tiny(torch.float32)).all(), i
