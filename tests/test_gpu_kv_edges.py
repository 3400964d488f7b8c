"""GPU tests of calls over the paged cache at the edges of what their arguments
allow: row starts that fall or wrap, bounds far above the call's rows, the
largest window, workspaces on other streams."""
import numpy as np
import pytest

from test_gpu_kv import Case, check_attention, rows, types
import paged

pytestmark = pytest.mark.gpu

LOW = -(1 << 31)


@pytest.mark.parametrize("group,max_q", [(1, 4), (4, None), (4, 2)])
def test_row_starts_that_fall(sm, dev, group, max_q):
    """A sequence whose rows end before they begin is left out, however far
    before: its rows and pages stay as they were, the others are served."""
    import torch
    kvh, hd, ntok = 2, 64, 14
    qstart = [0, 4, LOW, 4, 10, LOW + 3, 10, 12, 5]
    pos = [60, 5, 6, 100, 7, 8, 62, 9]
    c = Case(sm, dev, kvh, hd, len(pos), 2, 91)
    q, qf = rows(dev, c.rng.standard_normal((ntok, kvh * group, hd)), torch.float32)
    k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.float32)
    b = c.batch(pos, ntok, qstart, max_q=max_q)
    turned, out = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    table = sm.rope_table(128, 64, 1e4, dev)
    c.kv.append(b, q, k, k, table, turned)
    most = 1 << 30 if max_q is None else max_q
    want = paged.append(c.host, qf, kf, kf, table.cpu().numpy(), pos, qstart, None, most)
    c.same()
    got = turned.double().cpu().numpy()
    assert np.array_equal(got, np.where(np.isnan(want), 7.0, want).astype(np.float32).astype(np.float64))
    c.kv.attend(b, q, out)
    check_attention(c, q, qf, out, 0.125, 0, None, pos, qstart, None, most, f"group {group} max_q {max_q}")


@pytest.mark.parametrize("max_q", [5, 512, 20000, 1 << 30, (1 << 31) - 1])
@pytest.mark.parametrize("counts,group", [([1], 4), ([2], 2), ([1, 2, 1], 1), ([0, 1], 4), ([5, 9], 4)])
def test_max_q_far_above_the_rows(sm, dev, counts, group, max_q):
    """max_q only bounds: a context long enough to be split among workgroups
    and joined, with bounds that no launch could take for a size."""
    import torch
    kvh, hd = 2, 64
    n = len(counts)
    c = Case(sm, dev, kvh, hd, n, 50, 97)
    qstart = np.concatenate([[0], np.cumsum(counts)])
    ntok = int(qstart[-1])
    pos = [3000, 40, 2900][:n]
    q, qf = rows(dev, c.rng.standard_normal((ntok, kvh * group, hd)), torch.float32)
    k, kf = rows(dev, c.rng.standard_normal((ntok, kvh, hd)), torch.float32)
    b = c.batch(pos, ntok, qstart, max_q=max_q, max_len=3100)
    c.kv.append(b, None, k, k)
    paged.append(c.host, None, kf, kf, None, pos, qstart, None, max_q)
    c.same()
    out = torch.full_like(q, 7.0)
    c.kv.attend(b, q, out)
    check_attention(c, q, qf, out, 0.125, 0, None, pos, qstart, None, max_q, f"{counts} group {group} max_q {max_q}")
