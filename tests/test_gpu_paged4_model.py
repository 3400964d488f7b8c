"""GPU tests of the model's step over the paged 4-bit cache (sparkmv_model_paged4)
against the oracle (oracle/paged.py model_step with oracle/paged4.py).

The GPU's keys and values differ from the oracle's in their last bits, so a code
next to a border may come out one apart, and a scale next to 7 times a power of two
twice as large. Codes are held to that, and the oracle then goes on from the GPU's:
what is left is the forward's own arithmetic. With f32 activations that is 1e-5, the
bar of test_gpu_forward.py.

With bf16 activations a value next to a rounding border rounds the other way on one
side, which moves later values across theirs: at most, every rounding falls
independently on both sides. A step of bf16 is 2^-8 to 2^-7 of the value, 0.72 * 2^-7
in the root mean square over a binade, and a rounding is off by step / sqrt(12) in the
root mean square: 1.62e-3 of the value, sqrt(2) times that between two sides. A token
passes 13 of them (normed input, attention's output, normed input and activation in
each of three layers, the final norm), which add up as squares: 8.3e-3 of a row, and
rows of 256 values scatter about that by 1 / sqrt(2 * 256), four times which is 18 %:
9.8e-3. Most steps meet far less, as few values lie next to a border."""
import ctypes

import numpy as np
import pytest

import paged
import paged4
from test_gpu_forward import CFG, build, rel_l2

pytestmark = pytest.mark.gpu


class Mirror:
    """The oracle's caches of a model's paged one."""

    def __init__(self, sm, model, cfg, npages, nslots, max_pages):
        self.sm, self.model, self.cfg = sm, model, cfg
        kvh, hd = cfg["kv_heads"], cfg["head_dim"]
        self.table = np.full((nslots, max_pages), -1, np.int32)
        self.caches = [{"data": np.zeros((npages, kvh, 68 * hd), np.uint8), "pages": self.table} for _ in range(cfg["layers"])]
        self.tables = [sm.rope_table(max_pages * 64, int(np.float32(hd) * np.float32(cfg[p])), cfg[t]).cpu().numpy()
                       for p, t in (("rope_full_partial", "rope_full_theta"), ("rope_slide_partial", "rope_slide_theta"))]

    def pages(self, slot, pages):
        self.table[slot] = -1
        self.table[slot, :len(pages)] = pages
        self.model.set_pages(slot, pages)

    def device(self, li):
        import torch
        c = self.sm.Kv4Cache()
        self.sm.check(self.sm.lib().sparkmv_model_paged4_cache(self.model.h, li, ctypes.byref(c)), "cache")
        t = torch.empty(self.caches[li]["data"].shape, dtype=torch.uint8, device="cuda")
        self.sm._hip_copy(t.data_ptr(), c.data, t.numel())
        return t.cpu().numpy()

    def check(self, li):
        """The GPU's cache beside the oracle's, at the positions that are held
        (self.lens, after the step); the oracle then takes it over.

        Both are off by at most one scale from what they were given. Rows that differ
        by a relative L2 of r (self.r, as in test_gpu_paged_model.py) are 1.7 r scales
        apart in the root mean square, the codes' steps half a scale where most are:
        a share of sqrt(2 / pi) * 3.4 r of them rounds to a neighbour; a largest
        element, twice the root mean square off at most, crosses its border with a
        chance of 3 r or so and takes half of its 32 codes along: 5 r in all, and
        twice that as a bar."""
        hd = self.cfg["head_dim"]
        got, mine, off = {"data": self.device(li)}, self.caches[li], paged4.offsets(hd)
        for s, n in self.lens.items():
            for j in range((n + 63) // 64):
                page, rows = self.table[s, j], min(64, n - 64 * j)
                for w, (a, b) in enumerate(zip(paged4.values(got, [page], hd), paged4.values(mine, [page], hd))):
                    at = off[2 * w + 1][:rows]
                    scale = sum(np.exp2(x["data"][page][:, at].astype(np.float64) - 127.0) for x in (got, mine))
                    apart = np.abs(a - b)[0][:, :rows]
                    assert np.all(apart <= 1.05 * scale) and (apart > 0).mean() <= 10 * self.r, (li, s, j, w, (apart > 0).mean())
        mine["data"][:] = got["data"]


@pytest.mark.parametrize("xd", ["f32", "bf16"])
@pytest.mark.parametrize("head_kind", ["q8_0", "vq"])
def test_steps_of_several_sequences(sm, ref, dev, head_kind, xd):
    """Prompts, decode steps, a verified block and a cut back, with sequences
    coming and going; one of them crosses a page."""
    import torch
    cfg = dict(CFG, sliding_window=40)
    model, oracle = build(sm, ref, dev, head_kind, sm.X_F32 if xd == "f32" else sm.X_BF16, cfg)
    model.paged(9, 4, 3, bits=4)
    mirror = Mirror(sm, model, cfg, 9, 4, 3)
    mirror.r = 1e-3 if xd == "f32" else 5e-3
    rng = np.random.default_rng(4)
    mirror.pages(2, [5, 1])
    mirror.pages(0, [7])
    mirror.pages(3, [0, 8, 2])
    lens = {2: 0, 0: 0, 3: 0}
    steps = [({2: 60, 0: 3}, False), ({2: 1, 0: 1}, False), ({3: 9, 0: 1, 2: 6}, True), ({3: 1, 2: 1, 0: 1}, False), ({2: -4}, None),
             ({2: 3}, True), ({3: 130}, False), ({3: 1, 2: 1}, False)]
    bar = 1e-5 if xd == "f32" else 9.8e-3
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
        want = paged.model_step(oracle, mirror.caches, mirror.tables, flat, slots, pos, qstart, mirror.check, paged4)
        want = want if every else want[qstart[1:] - 1]
        # more than 16 tokens enter the prefill GEMM as f16 (2^-11): 1e-3 relative L2 a matrix
        b = bar if len(flat) <= 16 else 2e-2
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
        wk, wv = paged4.read(mirror.caches[1], 2, 60 + j, cfg["head_dim"])
        assert np.array_equal(k[0, j].cpu().numpy(), wk.astype(np.float32))
        assert np.array_equal(v[0, j].cpu().numpy(), wv.astype(np.float32))
    model.paged_step([[3]], [0], [lens[0]], None)
    torch.cuda.synchronize()


def test_refusals(sm, ref, dev):
    """A model has one paged cache, of 8 or 4 bits, and each is read as what it is."""
    model, _ = build(sm, ref, dev, "q8_0", sm.X_F32)
    for call, text in ((lambda: model.paged(1, 1, 1, bits=5), "5 bits"), (lambda: model.paged(0, 1, 1, bits=4), "0 pages"),
                       (lambda: model.paged(1, 1, 2049, bits=4), "above 131072")):
        with pytest.raises(sm.SparkmvError, match=text):
            call()
    c8, c4 = sm.KvCache(), sm.Kv4Cache()
    L = sm.lib()
    assert L.sparkmv_model_paged4_cache(model.h, 0, ctypes.byref(c4)) == -1 and "no paged cache" in sm.last_error()
    model.paged(4, 2, 2, bits=4)
    for bits in (8, 4):
        with pytest.raises(sm.SparkmvError, match="already"):
            model.paged(4, 2, 2, bits=bits)
    assert L.sparkmv_model_paged_cache(model.h, 0, ctypes.byref(c8)) == -1 and "of 4 bits" in sm.last_error()
    assert L.sparkmv_model_paged4_cache(model.h, 99, ctypes.byref(c4)) == -1 and "layer 99" in sm.last_error()
    assert L.sparkmv_model_paged4_cache(model.h, 0, ctypes.byref(c4)) == 0 and c4.npages == 4
    other, _ = build(sm, ref, dev, "q8_0", sm.X_F32)
    other.paged(4, 2, 2)
    assert L.sparkmv_model_paged4_cache(other.h, 0, ctypes.byref(c4)) == -1 and "of 8 bits" in sm.last_error()
