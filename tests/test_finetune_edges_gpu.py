"""Calls of the fine-tuning operators at the edges of what their documentation
allows, on the GPU."""
import pytest
import torch

from test_finetune_gpu import Preference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairs", [1, 40, 700])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_log_probabilities_over_the_reference_of_one_row_sequences(cuda_dev, pairs, dt):
    """Sequences of one row: logps and ref_logps have one size, so the one may take the other's place, and every warp of
    the pair has to have read the reference before it is written."""
    q = Preference(pairs, 1, 1001, 1008, dt, cuda_dev, seed=41, masked=0.0)
    q.call()
    q.check()
    want = [t.clone() for t in (q.losses, q.rewards, q.logps, q.dx)]
    ref = q.ref.clone()
    for _ in range(20):
        q.ref.copy_(ref)
        q.call(logps=q.ref)
        assert all(torch.equal(a, b) for a, b in zip(want, (q.losses, q.rewards, q.ref, q.dx)))
        w = q.w.clone()  # the rewards in the weights' place at the same time
        q.ref.copy_(ref)
        q.call(logps=q.ref, weights=w, rewards=w)
        assert all(torch.equal(a, b) for a, b in zip(want, (q.losses, w, q.ref, q.dx)))
