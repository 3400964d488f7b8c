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


class Busy:
    """A block of memory that work queued on the current stream reads late, and
    that was handed back before: whoever gets it has to come after that work."""

    def __init__(self, dev, nbytes):
        import torch
        a = torch.ones(4096, 4096, device=dev)
        block = torch.full((nbytes,), 5, dtype=torch.uint8, device=dev)
        a @ a
        torch.cuda.synchronize()
        for _ in range(20):     # some milliseconds
            a = a @ a * 1e-4
        self.read = block.clone()

    def check(self):
        import torch
        torch.cuda.synchronize()
        assert torch.all(self.read == 5)


def operators(sm, dev):
    """(name, workspace bytes, one-shot call, its op, check) of the calls that make a workspace."""
    import torch
    c = Case(sm, dev, 2, 128, 2, 40, 101)
    pos, heads = [2500, 2400], 8
    q, qf = rows(dev, c.rng.standard_normal((2, heads, 128)), torch.float32)
    out = torch.full((2, heads, 128), 7.0, device=dev)
    b = c.batch(pos, max_len=2501)
    x = torch.from_numpy(c.rng.standard_normal((64, 20000)).astype(np.float32)).to(dev)
    want = torch.log_softmax(x.double().cpu(), 1)
    tok = torch.zeros(64, dtype=torch.int32, device=dev)
    lp, ent = torch.zeros(64, device=dev), torch.zeros(64, device=dev)
    ids, tops = torch.zeros(64, 5, dtype=torch.int32, device=dev), torch.zeros(64, 5, device=dev)

    def attended():
        check_attention(c, q, qf, out, 128 ** -0.5, 0, None, pos, None, None, note="attention")
        out.fill_(7.0)

    def answered(got):
        assert float((got[0].double().cpu() - want[:, 0]).abs().max()) <= 1e-4     # as tests/test_gpu_paged_model.py
        assert torch.equal(got[2][:, 0].cpu().long(), want.argmax(1))

    need = sm.lib().sparkmv_kv_attend_work(sm.ctypes.addressof(c.kv.c), sm.ctypes.addressof(b.c), heads)
    yield ("attend", need, lambda s: c.kv.attend(b, q, out, stream=s), lambda: c.kv.attend_op(b, q, out), lambda got: attended())
    yield ("logprobs", sm.lib().sparkmv_logprobs_work(64, 20000, 5), lambda s: sm.logprobs(x, tok, 5, stream=s),
           lambda: sm.logprobs_op(x, tok, lp, ent, ids, tops), lambda got: answered(got or (lp, ent, ids, tops)))


def test_calls_on_another_stream_make_their_memory_there(sm, dev):
    """A call on a given stream takes no memory that the current stream's earlier
    work is still reading; what it returns may be read on the current stream."""
    import torch
    s = torch.cuda.Stream(device=dev)
    for name, need, call, _, check in operators(sm, dev):
        s.wait_stream(torch.cuda.current_stream())
        call(s)     # loaded and warm
        torch.cuda.synchronize()
        busy = Busy(dev, need)
        got = call(s)
        torch.cuda.current_stream().wait_stream(s)
        busy.check()
        check(got)
    busy = Busy(dev, 1 << 20)
    table = sm.rope_table(4096, 64, 1e4, dev, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    busy.check()
    assert torch.equal(table, sm.rope_table(4096, 64, 1e4, dev))


@pytest.mark.parametrize("how", ["given", "current"])
def test_an_op_used_on_another_stream_than_it_was_made_on(sm, dev, how):
    """The workspace waits for the work that had its memory before, and is not
    handed out again while a stream that the call ran on is not done with it."""
    import torch
    s = torch.cuda.Stream(device=dev)

    def use(op):
        if how == "given":
            op(s)
        else:
            with torch.cuda.stream(s):
                op()

    for name, need, _, make, check in operators(sm, dev):
        s.wait_stream(torch.cuda.current_stream())
        use(make())
        torch.cuda.synchronize()
        busy = Busy(dev, need)
        op = make()
        use(op)
        torch.cuda.current_stream().wait_stream(s)
        busy.check()
        check(None)
        # dropped while its stream still runs it: the memory's next owner keeps its values
        op = make()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            Busy(dev, 1024)
        use(op)
        del op
        after = torch.full((need,), 9, dtype=torch.uint8, device=dev)
        torch.cuda.synchronize()
        assert torch.all(after == 9), name
        check(None)


def test_ops_in_graphs_and_on_streams_by_turns(sm, dev):
    """An op recorded on one stream, replayed, called on another and on the
    current one: the same outputs each time."""
    import torch
    for name, need, _, make, check in operators(sm, dev):
        s = torch.cuda.Stream(device=dev)
        op = make()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            op()
        for turn in range(3):
            graph.replay()
            torch.cuda.synchronize()
            check(None)
            op(s)
            torch.cuda.synchronize()
            check(None)
            op()
            torch.cuda.synchronize()
            check(None)


def test_the_largest_window(sm, dev):
    """A window that no position leaves is no window: the same launches, the same bits."""
    import torch
    c = Case(sm, dev, 2, 64, 2, 100, 103)
    q = torch.randn(2, 8, 64, device=dev)
    b = c.batch([6000, 5000], max_len=6001)
    out = [torch.full_like(q, 7.0) for _ in range(4)]
    for o, w in zip(out, (0, (1 << 31) - 1, (1 << 31) - 64, 1 << 30)):
        c.kv.attend(b, q, o, window=w)
    assert all(torch.equal(out[0], o) for o in out[1:])
