"""What stands around the experts of a block where numbers or calls are out of the ordinary, without a GPU."""
import pytest

from deepep_efa_b200 import _ext


# ---- a copy that does not come --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("stages", [2, 3])
@pytest.mark.parametrize("boxes", [0, 1, 2, 3, 4, 7, 12])
def test_ring_of_a_warp_whose_wait_runs_out(stages, boxes):
    """The kernels' loop over a warp's boxes with the wait for each of them, or for none, running out: the copies that are still on their way are waited for, each in its
    slot with the parity of its use, once; nothing is started after that."""
    for fails_at in range(boxes + 1):
        ring, todo, flying, uses = _ext.load().FewTokensRing(stages), list(range(boxes)), [], [0] * stages

        def start():
            if todo:
                assert all(slot != ring.fill for slot, _ in flying)  # (a slot is filled when its box has been read)
                flying.append((ring.fill, uses[ring.fill] & 1))
                uses[ring.fill] += 1
                todo.pop(0)
                ring.started()
        for _ in range(stages):
            start()
        waits = []
        for box in range(boxes):
            if box >= fails_at:  # (the CTA's flag ends every wait from then on)
                ring.give_up(lambda slot, parity: waits.append((slot, parity)))
                assert not ring.alive and waits == flying and len(waits) == min(stages, boxes - fails_at)
            else:
                assert (ring.slot, ring.parity) == flying.pop(0)
            assert 0 <= ring.slot < stages
            ring.taken()
            if ring.alive:
                start()
                assert ring.flying == len(flying)
        assert ring.alive == (fails_at == boxes) and (not ring.alive or not flying) and ring.flying <= 0
