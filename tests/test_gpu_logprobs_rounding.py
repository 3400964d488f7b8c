"""GPU test of what a log probability is rounded to (sparkmv_logprobs): once.

Rows of 2^18 equal logits and one far below them: the sum of exponentials is
2^18 (1 + e^-d / 2^18), whose f32 loses 2^-24 of it at most where e^-d < 2^-6,
and log z is then off by the logarithm of 1 .. 2, 2^-24 or so, and that. A result
between 16 and 32 has steps of 2^-19: half a step, and 2^-4 of one; between 8 and
16 of 2^-20: half, and 2^-3 of one."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_one_rounding(sm, dev, x):
    import torch
    rng = np.random.default_rng(7)
    rows, n = 64, 1 << 18
    dt = torch.float32 if x == "f32" else torch.bfloat16
    t = torch.from_numpy(rng.uniform(2, 4, (rows, 1)).astype(np.float32)).to(dev).to(dt).expand(rows, n).contiguous()
    tok = torch.from_numpy(rng.integers(0, n, rows).astype(np.int32)).to(dev)
    low = torch.from_numpy(rng.uniform(-9, -3, rows).astype(np.float32)).to(dev).to(dt)
    t[torch.arange(rows), tok.long()] = low
    lp, ent, ids, tops = sm.logprobs(t, tok, 3)
    big, v = t.double().max(1)[0].cpu().numpy(), low.double().cpu().numpy()
    lse = np.log((n - 1) + np.exp(v - big))
    want = v - big - lse
    assert np.all((want < -16) & (want > -32))
    err = np.abs(lp.double().cpu().numpy() - want) / 2.0 ** -19
    top = np.abs(tops.double().cpu().numpy() + lse[:, None]) / 2.0 ** -20      # 8 .. 16
    p = np.exp(want)
    e = np.abs(ent.double().cpu().numpy() - (lse + p * (big - v))) / 2.0 ** -20
    print(f"{x}: largest error in steps: given {err.max():.3f}, tops {top.max():.3f}, entropy {e.max():.3f}")
    assert err.max() <= 0.5 + 2.0 ** -4
    assert max(top.max(), e.max()) <= 0.5 + 2.0 ** -3
