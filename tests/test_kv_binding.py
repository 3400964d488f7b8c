"""CPU tests of what the Python calls over the paged cache refuse before the
library is reached: tensors are stand-ins that have a device but no memory."""
import ctypes

import pytest
import torch


class Fake:
    """What the binding asks of a tensor."""

    def __init__(self, shape, dtype, device="cuda:0"):
        self.shape, self.dtype, self.device, self.is_cuda = tuple(shape), dtype, torch.device(device), True

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 20


@pytest.fixture
def model(sm, monkeypatch):
    """A Model with a paged cache of 2 heads of 64, whose library reads nothing."""
    class Lib:
        def sparkmv_model_paged_cache(self, h, layer, ref):
            c = ref._obj
            c.kv_heads, c.head_dim = 2, 64
            return 0

        def __getattr__(self, name):
            raise AssertionError(name + " was reached")

    monkeypatch.setattr(sm, "lib", lambda: Lib())
    m = sm.Model.__new__(sm.Model)
    m._L, m.h, m.cfg, m.paged_device = None, None, {"vocab": 10}, torch.device("cuda:0")
    return m


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.float16, torch.float64, torch.int32, torch.float8_e4m3fn])
def test_paged_read_takes_f32_and_bf16_only(sm, model, dtype):
    start = Fake((3,), torch.int32)
    for bad in (0, 1):
        outs = [Fake((3, 5, 2, 64), dtype if i == bad else torch.float32) for i in range(2)]
        with pytest.raises(sm.SparkmvError, match="type"):
            model.paged_read(0, start, *outs)
    with pytest.raises(sm.SparkmvError, match="type"):
        model.paged_read(0, start, *(Fake((3, 5, 2, 64), dtype) for _ in range(2)))


def test_paged_read_of_other_shapes_types_and_devices(sm, model):
    start, ok = Fake((3,), torch.int32), Fake((3, 5, 2, 64), torch.float32)
    for args, text in (
            ((start, ok, Fake((3, 5, 2, 64), torch.bfloat16)), "two types"), ((start, None, None), "nothing"),
            ((start, ok, Fake((3, 4, 2, 64), torch.float32)), "shape"), ((start, Fake((3, 5, 128), torch.float32), None), "shape"),
            ((Fake((3,), torch.int64), ok, ok), "type"), ((start, Fake((2, 5, 2, 64), torch.float32), None), "shape"),
            ((Fake((3,), torch.int32, "cuda:1"), ok, ok), "on cuda:1"),
            ((start, Fake((3, 5, 2, 64), torch.float32, "cuda:1"), ok), "on cuda:1"),
            ((start, ok, ok, Fake((3,), torch.int32, "cuda:1")), "on cuda:1"), ((start, ok, ok, Fake((2,), torch.int32)), "shape")):
        with pytest.raises(sm.SparkmvError, match=text):
            model.paged_read(0, *args)
    with pytest.raises(sm.SparkmvError, match="on cuda:1"):
        model.paged_step([[1]], [0], [0], Fake((1, 10), torch.float32, "cuda:1"))


def test_row_starts_need_their_number_of_rows(sm):
    pos, starts = Fake((2,), torch.int32), Fake((3,), torch.int32)
    with pytest.raises(sm.SparkmvError, match="without the number of rows"):
        sm.KVBatch(pos, qstart=starts)
    assert sm.KVBatch(pos, 9, starts).c.max_q == 9 and sm.KVBatch(pos).c.ntok == 2
