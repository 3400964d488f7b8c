"""GPU tests of the model's step over the paged cache (sparkmv_model_paged_step)
against the oracle (oracle/paged.py model_step).

The GPU's keys and values differ from the oracle's in their last bits, so a
code next to a border may come out one step apart. Codes are held to that, and
the oracle then goes on from the GPU's codes and scales: what is left is the
forward's own arithmetic, with the bars of test_gpu_forward.py (1e-5 with f32
activations; with bf16, where a value next to a rounding border flips, 5e-3)."""
import ctypes

import numpy as np
import pytest

import paged
from test_gpu_forward import BF16_RUN_BAR, CFG, build, rel_l2

pytestmark = pytest.mark.gpu


class Mirror:
    """The oracle's caches of a model's paged one."""

    def __init__(self, sm, model, cfg, npages, nslots, max_pages):
        import torch
        self.sm, self.model, self.cfg = sm, model, cfg
        kvh, hd = cfg["kv_heads"], cfg["head_dim"]
        self.table = np.full((nslots, max_pages), -1, np.int32)
        self.caches = [{"k": np.zeros((npages, kvh, 64 * hd), np.int8), "v": np.zeros((npages, kvh, 64 * hd), np.int8),
                        "k_scale": np.zeros((npages, kvh), np.float32), "v_scale": np.zeros((npages, kvh), np.float32),
                        "pages": self.table} for _ in range(cfg["layers"])]
        self.tables = [sm.rope_table(max_pages * 64, int(np.float32(hd) * np.float32(cfg[p])), cfg[t]).cpu().numpy()
                       for p, t in (("rope_full_partial", "rope_full_theta"), ("rope_slide_partial", "rope_slide_theta"))]

    def pages(self, slot, pages):
        self.table[slot] = -1
        self.table[slot, :len(pages)] = pages
        self.model.set_pages(slot, pages)

    def device(self, li):
        import torch
        c = self.sm.KvCache()
        self.sm.check(self.sm.lib().sparkmv_model_paged_cache(self.model.h, li, ctypes.byref(c)), "cache")
        out = {}
        for name, ptr, dt in (("k", c.k, torch.int8), ("v", c.v, torch.int8), ("k_scale", c.k_scale, torch.float32),
                              ("v_scale", c.v_scale, torch.float32)):
            t = torch.empty(self.caches[li][name].shape, dtype=dt, device="cuda")
            self.sm._hip_copy(t.data_ptr(), ptr, t.numel() * t.element_size())
            out[name] = t.cpu().numpy()
        return out

    def check(self, li):
        """The GPU's codes and scales beside the oracle's, at the positions that
        are held (self.lens, after the step); the oracle then takes them over.

        Rows that differ by a relative L2 of r (self.r: 1e-3 where the prefill GEMM
        may run, 5e-3 with bf16 activations, the bars of the forward's own tests)
        are r * 40 steps apart in the mean square, a page's codes being of that
        size (127 at 3 to 4 times their root mean square): a share of
        sqrt(2 / pi) * 40 r of them rounds to a neighbour, and none to the next
        but one up to r = 1e-3, where five times the mean is a fifth of a step
        (5e-3: one step). The largest, five times the mean off at most, is off by
        5 r / 3.5 of itself."""
        got, mine, off = self.device(li), self.caches[li], paged.offsets(self.cfg["head_dim"])
        for s, n in self.lens.items():
            for j in range((n + 63) // 64):
                page, rows = self.table[s, j], min(64, n - 64 * j)
                for which, name in enumerate("kv"):
                    a, b = got[name + "_scale"][page], mine[name + "_scale"][page]
                    assert np.all(np.abs(a - b) <= 5 * self.r / 3.5 * np.abs(b)), (li, s, j, name)
                    at = off[which][:rows]
                    apart = np.abs(got[name][page][:, at].astype(int) - mine[name][page][:, at])
                    assert apart.max() <= (1 if self.r <= 1e-3 else 2) and (apart > 0).mean() <= 32 * self.r, (li, s, j, name, apart.max(), (apart > 0).mean())
                    mine[name][page][:, at] = got[name][page][:, at]
                    mine[name + "_scale"][page] = a


@pytest.mark.parametrize("xd", ["f32", "bf16"])
@pytest.mark.parametrize("head_kind", ["q8_0", "vq"])
def test_steps_of_several_sequences(sm, ref, dev, head_kind, xd):
    """Prompts, decode steps, a verified block and a cut back, with sequences
    coming and going; one of them crosses a page."""
    import torch
    cfg = dict(CFG, sliding_window=40)
    model, oracle = build(sm, ref, dev, head_kind, sm.X_F32 if xd == "f32" else sm.X_BF16, cfg)
    model.paged(9, 4, 3)
    mirror = Mirror(sm, model, cfg, 9, 4, 3)
    mirror.r = 1e-3 if xd == "f32" else 5e-3
    rng = np.random.default_rng(4)
    mirror.pages(2, [5, 1])
    mirror.pages(0, [7])
    mirror.pages(3, [0, 8, 2])
    lens = {2: 0, 0: 0, 3: 0}
    steps = [({2: 60, 0: 3}, False), ({2: 1, 0: 1}, False), ({3: 9, 0: 1, 2: 6}, True), ({3: 1, 2: 1, 0: 1}, False), ({2: -4}, None),
             ({2: 3}, True), ({3: 130}, False), ({3: 1, 2: 1}, False)]
    bar = 1e-5 if xd == "f32" else BF16_RUN_BAR
    for what, every in steps:
        if every is None:
            for s, d in what.items():
                lens[s] += d
            continue
        slots = list(what)
        toks = [[int(t) for t in rng.integers(0, cfg["vocab"], what[s])] for s in slots]
        flat, pos = [t for x in toks for t in x], [lens[s] for s in slots]
        qstart = np.concatenate([[0], np.cumsum([len(t) for t in toks])])
        logits = torch.full((len(flat) if every else len(slots), cfg["vocab"]), float("nan"), device=dev)
        model.paged_step(toks, slots, pos, logits, every=every)
        torch.cuda.synchronize()
        mirror.lens = {s: lens[s] + what.get(s, 0) for s in lens}
        want = paged.model_step(oracle, mirror.caches, mirror.tables, flat, slots, pos, qstart, mirror.check)
        want = want if every else want[qstart[1:] - 1]
        # more than 16 tokens enter the prefill GEMM as f16 (2^-11): 1e-3 relative L2 a
        # matrix. With bf16 outputs, attention of several tokens of a sequence holds
        # weights to 2^-15 of a page's largest, 2^-9 of the output over 64 of them: in
        # each of the three layers half a bf16 step more than the bar's own flips
        b = bar if len(flat) <= 16 else 2e-2
        if xd == "bf16" and max(len(t) for t in toks) > 1:
            b = max(b, BF16_RUN_BAR + 3 * 2.0 ** -9)
        err = max(rel_l2(g, w) for g, w in zip(logits.cpu().numpy(), want))
        print(f"head {head_kind} x {xd} {what}: logits relL2 {err:.2e}")
        assert err <= b
        for s in slots:
            lens[s] += what[s]
    # reading back, and the step without logits
    k = torch.empty(1, 5, cfg["kv_heads"], cfg["head_dim"], device=dev)
    v = torch.empty_like(k)
    one = lambda x: torch.tensor([x], dtype=torch.int32, device=dev)  # noqa: E731
    model.paged_read(1, one(60), k, v, slot=one(2))
    for j in range(5):
        wk, wv = paged.read(mirror.caches[1], 2, 60 + j, cfg["head_dim"])
        assert np.array_equal(k[0, j].cpu().numpy(), wk.astype(np.float32))
        assert np.array_equal(v[0, j].cpu().numpy(), wv.astype(np.float32))
    model.paged_step([[3]], [0], [lens[0]], None)
    torch.cuda.synchronize()


def test_paged_steps_stay_near_the_f32_cache(sm, ref, dev):
    """The same tokens through the f32 cache and the paged one: the logits differ
    by the codes' rounding (1/127 of a page's largest at most, an eighth of that
    in the mean), and the f32 cache is not touched by paged steps."""
    import torch
    model, _ = build(sm, ref, dev, "q8_0", sm.X_F32)
    model.paged(2, 1, 1)
    model.set_pages(0, [1])
    a = torch.empty(CFG["vocab"], device=dev)
    b = torch.empty(1, CFG["vocab"], device=dev)
    toks = [5, 17, 3, 250, 42, 7]
    for p, t in enumerate(toks):
        model.forward(t, p, a)
        model.paged_step([[t]], [0], [p], b)
        torch.cuda.synchronize()
        err = rel_l2(b[0].cpu().numpy(), a.cpu().numpy())
        print(f"position {p}: {err:.2e}")
        assert err <= 5e-2
    assert len(model) == len(toks)


def test_answers_of_a_step(sm, ref, dev):
    """A step's logits into log probabilities: the first alternative is argmax's,
    and its log probability is what the logits say."""
    import torch
    model, _ = build(sm, ref, dev, "q8_0", sm.X_F32)
    model.paged(3, 2, 1)
    model.set_pages(0, [0])
    model.set_pages(1, [2])
    logits = torch.empty(2, CFG["vocab"], device=dev)
    model.paged_step([[1, 2, 3], [9]], [0, 1], [0, 0], logits)
    given = torch.tensor([4, 5], dtype=torch.int32, device=dev)
    lp, ent, ids, tops = sm.logprobs(logits, given, 4)
    x = logits.double()
    want = torch.log_softmax(x, 1)
    for r in range(2):
        assert int(ids[r, 0]) == int(sm.argmax(logits[r].contiguous())[0])
        # the bounds of test_gpu_logprobs.py at logits of this size
        assert abs(float(lp[r]) - float(want[r, given[r]])) <= 1e-4
        assert abs(float(tops[r, 0]) - float(want[r].max())) <= 1e-4
        assert abs(float(ent[r]) + float((want[r].exp() * want[r]).sum())) <= 1e-3


def test_refusals(sm, ref, dev):
    import torch
    model, _ = build(sm, ref, dev, "q8_0", sm.X_F32)
    lg = torch.zeros(1, CFG["vocab"], device=dev)
    for call, text in (
            (lambda: model.paged_step([[1]], [0], [0], lg), "no paged cache"), (lambda: model.set_pages(0, [0]), "no paged cache"),
            (lambda: model.paged(0, 1, 1), "0 pages"), (lambda: model.paged(1, 1, 2049), "above 131072")):
        with pytest.raises(sm.SparkmvError, match=text):
            call()
    model.paged(4, 2, 2)
    model.set_pages(0, [0, 1])
    for call, text in (
            (lambda: model.paged(4, 2, 2), "already"), (lambda: model.set_pages(2, [0]), "slot 2"),
            (lambda: model.set_pages(0, [4]), "page 4"), (lambda: model.set_pages(0, [0, 1, 2]), "3 pages"),
            (lambda: model.paged_step([[1], [2]], [0, 0], [0, 0], None), "twice"),
            (lambda: model.paged_step([[1]], [2], [0], lg), "slot 2"), (lambda: model.paged_step([[]], [0], [0], lg), "one at least"),
            (lambda: model.paged_step([[1]], [0], [-1], lg), "positions -1"),
            (lambda: model.paged_step([[1, 1]], [0], [127], None), "exceed"),
            (lambda: model.paged_step([[CFG["vocab"]]], [0], [0], lg), "vocabulary"),
            (lambda: model.paged_step([[1] * 17], [0], [0], torch.zeros(17, CFG["vocab"], device=dev), every=True), "1..16 tokens"),
            (lambda: model.paged_step([[1]] * 17, list(range(17)), [0] * 17, None), "1..16 sequences"),
            (lambda: model.paged_step([[1] * 120, [1] * 100, [1] * 100], [0, 1, 2], [0, 0, 0], None), "slot 2"),
            (lambda: model.paged_step([[1]], [0], [0], lg.double()), "type"),
            (lambda: model.paged_step([[1]], [0, 1], [0], None), "token lists")):
        with pytest.raises(sm.SparkmvError, match=text):
            call()
