"""GPU tests of head norms whose weights are far from 1, for bf16 rows: what
tests/test_gpu_rope.py says of their bound."""
import numpy as np
import pytest

import paged4
from test_gpu_kv import rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("x_size,w_size", [(1e17, 1e30), (1e-12, 1e-30), (1e-13, 1e36), (1.0, 1e36), (1e17, 1e-30)])
def test_weights_of_any_size(sm, dev, x_size, w_size, inter):
    """No product on the way leaves f32 where the result does not."""
    import torch
    rng = np.random.default_rng(11)
    hd, n = 128, 40
    x, f = rows(dev, rng.standard_normal((n, 4, hd)) * x_size, torch.bfloat16)
    w, wf = rows(dev, (1 + 0.3 * rng.standard_normal(hd)) * w_size, torch.float32)
    table, out = sm.rope_table(n, hd, 1e4, dev), torch.empty_like(x)
    eps = float(np.float32(1e-38))
    sm.qk_rope(torch.arange(n, dtype=torch.int32, device=dev), x, out, rope=table, interleaved=inter, q_norm=w, eps=eps)
    want = np.stack([paged4.turn(f[t], table.cpu().numpy()[t], inter, wf, eps) for t in range(n)])
    size = np.stack([np.abs(paged4.turn(f[t], None, inter, wf, eps)).max(-1, keepdims=True) for t in range(n)])
    assert np.isfinite(want).all() and np.abs(want).max() < 3e38
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want) * (1 + 1e-6) + 2.0 ** -20 * size)
