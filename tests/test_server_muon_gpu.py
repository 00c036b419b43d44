"""GPU: the server's Muon optimizer as a lockstep batch carries it on - its rounds enqueue without waiting for the device."""
import pytest

from test_server_muon import engine

pytestmark = pytest.mark.gpu


def test_a_round_does_not_wait_for_the_device():
    """Two lockstep batches on two streams are enqueued by one thread: an upload from pageable memory in one's round would
    hold back the other's."""
    import torch
    eng = engine(server_optimizer="muon")
    st = eng.trainer.prepare([(0, 1), (2,), (1, 2, 3)], 1)
    st.aggregate()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        st.aggregate()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    torch.cuda.synchronize()
    for ci, rows in ((0, (0, 1)), (2, (3, 4, 5))):
        for r in rows:
            assert torch.equal(st.params[r], st.glob[ci])
