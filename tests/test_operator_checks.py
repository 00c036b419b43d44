"""CPU: the batched operators' memory checks against the elements themselves."""
import itertools

import pytest
import torch

from mplc import dense


def shares(t, u):
    """Whether two views have an element in common, by their addresses."""
    def places(v):
        idx = torch.zeros((), dtype=torch.int64)
        for d, s in zip(v.shape, v.stride()):
            idx = idx.unsqueeze(-1) + torch.arange(d) * s
        first = v.data_ptr() + idx.flatten() * v.element_size()
        return set((first[:, None] + torch.arange(v.element_size())).flatten().tolist())
    return bool(places(t) & places(u))


def refused(out, other):
    ts = (out, other)
    try:
        dense._no_overlap(ts, ("out", "other"), [t.data_ptr() for t in ts], [dense._span(t) for t in ts], [0], [1])
    except ValueError:
        return True
    return False


def views():
    buf = torch.zeros(4 * 96 + 8)
    for G in (1, 3):
        for off, rows, cols, ld, step in itertools.product((0, 5, 12, 16, 40), (1, 3), (1, 4, 8), (8, 16, 24), (24, 48, 96)):
            if cols <= ld and off + (G - 1) * step + (rows - 1) * ld + cols <= buf.numel():
                yield buf.as_strided((G, rows, cols), (step, ld, 1), off)
                if rows == 1:
                    yield buf.as_strided((G, cols), (step, 1), off)


def test_no_shared_element_passes_and_disjoint_ones_are_found():
    vs = list(views())
    wrong = sum(1 for t in vs for u in vs[::7] if shares(t, u) and not refused(t, u))
    assert wrong == 0


@pytest.mark.parametrize("G", [1, 2, 5])
def test_parts_of_the_same_rows_are_disjoint(G):
    both = torch.zeros(G, 6, 20)
    left, right = both[:, :, :12], both[:, :, 12:]
    assert not refused(left, right) and not refused(right, left) and refused(left, both[:, :, 11:])
    rows = torch.zeros(G, 200)  # one model's layers, a column of a matrix beside the others
    w, b = rows[:, :60].view(G, 6, 10), rows[:, 60:70]
    assert not refused(w, b) and not refused(w[:, :, :4], w[:, :, 4:]) and refused(w, rows[:, 59:63])
    top, bottom = both[:, :3], both[:, 3:]
    assert not refused(top, bottom) and refused(top, both[:, 2:])
    half = torch.zeros(G, 6, 20, dtype=torch.bfloat16)
    assert not refused(half[:, :, :10], half[:, :, 10:])


def test_few_rows_of_16_bit_weights_take_the_tiles_whether_cut_or_not():
    """The split of a sum is the tiles' one, which does not know where rows end; fp32's large cut weights have one of their own."""
    import ctypes
    lib = dense._lib()

    def split(dtype, G, B, K, N):
        t = dense.DenseT()
        t.n_models, t.rows, t.in_, t.out, t.dtype = G, B, K, N, dtype
        return lib.mplc_dense_forward_workspace_bytes(ctypes.byref(t)) // (4 * G * B * N)
    for B in (1, 2, 8):
        for G, K, N in ((3, 9216, 397), (81, 3256, 653), (1, 4096, 1021)):
            for dtype in (1, 2):
                assert split(dtype, G, B, K, N) == split(dtype, G, B, K, N + 3), (dtype, G, B, K, N)
        assert split(0, 3, B, 9216, 397) != split(0, 3, B, 9216, 400)
        assert split(0, 1, B, 300, 129) == split(0, 1, B, 300, 132)
