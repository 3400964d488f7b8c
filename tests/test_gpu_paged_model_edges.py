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


def test_new_tokens_need_pages_of_their_own(sm, ref, dev):
    """A token whose page is missing would be lost without a word, one that enters
    another slot's page would race with that slot's."""
    import torch
    model, _ = build(sm, ref, dev, "q8_0", sm.X_F32)
    model.paged(4, 3, 2)
    logits = torch.full((2, CFG["vocab"]), float("nan"), device=dev)
    with pytest.raises(sm.SparkmvError, match="slot 0 has no page for position 0"):
        model.paged_step([[3]], [0], [0], None)
    model.set_pages(0, [2])
    model.set_pages(1, [2, 3])      # shares slot 0's page, enters its own
    model.set_pages(2, [0, 0])
    for args, text in ((([[3] * 70], [0], [0]), "slot 0 has no page for position 64"), (([[3]], [0], [64]), "no page for position 64"),
                       (([[3], [4]], [0, 1], [5, 9]), "page 2 would take tokens of two places"),
                       (([[3] * 66], [2], [0]), "page 0 would take tokens of two places")):
        with pytest.raises(sm.SparkmvError, match=text):
            model.paged_step(*args, None)
    model.paged_step([[3] * 20], [0], [0], None)
    model.paged_step([[3], [4]], [0, 1], [20, 64], logits)
    assert bool(torch.isfinite(logits).all())
    model.set_pages(0, [])
    with pytest.raises(sm.SparkmvError, match="no page"):
        model.paged_step([[3]], [0], [21], None)
