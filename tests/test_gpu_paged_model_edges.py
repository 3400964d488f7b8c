"""GPU tests of the model's paged cache at the edges of what its calls allow."""
import pytest

from test_gpu_forward import CFG, build

pytestmark = pytest.mark.gpu


def test_a_cache_that_does_not_fit_is_refused_and_the_next_one_made(sm, ref, dev):
    """The allocation's error is reported once: the calls after it succeed."""
    import torch
    model, _ = build(sm, ref, dev, "q8_0", sm.X_F32)
    with pytest.raises(sm.SparkmvError, match="paged cache"):
        model.paged(1 << 30, 1, 1)      # 2^30 pages of some kilobytes
    model.paged(2, 1, 1)
    model.set_pages(0, [1])
    logits = torch.full((1, CFG["vocab"]), float("nan"), device=dev)
    model.paged_step([[3]], [0], [0], logits)
    assert bool(torch.isfinite(logits).all())
