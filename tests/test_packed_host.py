"""What the packed-batch bindings refuse before the library is called (no GPU needed): a stand-in context names the
device, so every call here has to end in the bindings' own checks."""
import pytest
import torch

import ltx_b200 as L


class NoContext:
    device, h = 0, None

    def check(self, rc, what):
        raise AssertionError("the library was called")


CTX = NoContext()
BF16 = torch.bfloat16


def kind_of(fn, *args, **kw):
    with pytest.raises(L.LtxError) as e:
        fn(CTX, *args, **kw)
    return e.value.kind


class Fake:
    """A tensor that says it lies on a GPU (nothing reads its storage)."""

    def __init__(self, t, device=torch.device("cuda", 0)):
        self.t, self.device, self.is_cuda = t, device, device.type == "cuda"

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.device.index if self.is_cuda else -1

    def data_ptr(self):
        return 0


def fake(*shape, dtype=BF16, device=0):
    return Fake(torch.zeros(*shape, dtype=dtype), torch.device("cuda", device))


def test_host_tensors_and_other_devices_are_refused():
    t = torch.zeros(4, 8)
    assert kind_of(L.rope_table, None, t, t) == "INVALID_ARG"
    assert kind_of(L.rope_table, None, fake(4, 8, dtype=torch.float32, device=1), t) == "INVALID_ARG"
    q = fake(4, 128)
    o = fake(2, dtype=torch.int32)
    assert kind_of(L.attention_packed, q, fake(4, 128, device=1), q, q, o, o, 1, 1, 1.0) == "INVALID_ARG"
    assert kind_of(L.qk_norm_rope, torch.zeros(4, 128), None, q, None, 1, 0, None, None) == "INVALID_ARG"


def test_wrong_types_are_refused():
    q, o = fake(4, 128), fake(2, dtype=torch.int32)
    assert kind_of(L.attention_packed, q, q, q, q, fake(2, dtype=torch.int64), o, 1, 1, 1.0) == "DTYPE"
    assert kind_of(L.attention_packed, q, q, fake(4, 128, dtype=torch.float32), q, o, o, 1, 1, 1.0) == "DTYPE"
    assert kind_of(L.attention_packed, fake(4, 128, dtype=torch.float16), q, q, q, o, o, 1, 1, 1.0) == "DTYPE"
    assert kind_of(L.qk_norm_rope, q, None, fake(4, 128, dtype=torch.float16), None, 1, 0, None, None) == "DTYPE"
    x, w, a, b = fake(4, 64), fake(8, 64), fake(2, 16, 64), fake(2, 8, 16)
    i, c = fake(4, dtype=torch.int32), fake(2, dtype=torch.float32)
    assert kind_of(L.gemm_adapters, x, w, fake(4, 8), fake(4, dtype=torch.int64), a, b, c) == "DTYPE"
    assert kind_of(L.gemm_adapters, x, w, fake(4, 8), i, a, b, c, epilogue=L.EPI_F32) == "DTYPE"


def test_wrong_shapes_are_refused():
    q, o = fake(4, 128), fake(2, dtype=torch.int32)
    assert kind_of(L.attention_packed, q, q, q, q, o, fake(3, dtype=torch.int32), 1, 1, 1.0) == "SHAPE"
    assert kind_of(L.attention_packed, q, fake(5, 128), q, q, o, o, 1, 1, 1.0) == "SHAPE"
    assert kind_of(L.attention_packed, q, q, q, q, fake(0, dtype=torch.int32), o, 1, 1, 1.0) == "SHAPE"
    assert kind_of(L.attention_packed, q, q, q, q, o, o, 1, 1, 1.0, causal=True, prefix=fake(2, dtype=torch.int32)) == "SHAPE"
    turned = Fake(torch.zeros(128, 4, dtype=BF16).t())
    assert kind_of(L.attention_packed, turned, q, q, q, o, o, 1, 1, 1.0) == "SHAPE"
    repeated = Fake(torch.zeros(1, 128, dtype=BF16).expand(4, 128))
    assert kind_of(L.attention_packed, q, q, q, repeated, o, o, 1, 1, 1.0) == "SHAPE"
    x, w, a, b = fake(4, 64), fake(8, 64), fake(2, 16, 64), fake(2, 8, 16)
    i, c = fake(4, dtype=torch.int32), fake(2, dtype=torch.float32)
    assert kind_of(L.gemm_adapters, x, w, fake(4, 9), i, a, b, c) == "SHAPE"
    assert kind_of(L.gemm_adapters, x, w, fake(4, 8), i, a, fake(2, 9, 16), c) == "SHAPE"
    assert kind_of(L.gemm_adapters, x, w, fake(4, 8), i, a, fake(3, 8, 16), c) == "SHAPE"
    assert kind_of(L.gemm_adapters, x, w, fake(4, 8), fake(5, dtype=torch.int32), a, b, c) == "SHAPE"
    assert kind_of(L.qk_norm_rope, q, None, fake(4, 64), None, 1, 0, None, None) == "SHAPE"
    t = fake(4, 8, dtype=torch.float32)
    assert kind_of(L.qk_norm_rope, q, None, q, None, 1, 0, t, None) == "INVALID_ARG"
    assert kind_of(L.rope_table, fake(3, dtype=torch.int32), t, t) == "SHAPE"


def test_rows_of_one_value_keep_their_stride():
    """A column of a larger matrix, whatever its inner stride, is read at its rows' distance."""
    column = Fake(torch.zeros(5, 6, dtype=BF16)[:, ::3][:, 1:])
    assert column.stride() == (6, 3) and tuple(column.shape) == (5, 1)
    assert L._rows(CTX, "t", "x", column, (BF16,), 5, 1)[1] == 6
    assert L._rows(CTX, "t", "x", Fake(torch.zeros(5, 1, dtype=BF16)), (BF16,), 5, 1)[1] == 1
    assert L._rows(CTX, "t", "x", Fake(torch.zeros(5, 8, dtype=BF16)[:1, :6]), (BF16,), 1, 6)[1] >= 6
    with pytest.raises(L.LtxError) as e:
        L._rows(CTX, "t", "x", Fake(torch.zeros(1, 1, dtype=BF16).expand(5, 1)), (BF16,), 5, 1)
    assert e.value.kind == "SHAPE"


def test_a_single_rows_stride_does_not_count():
    """One row of a matrix whose rows are not 16-byte aligned is as good as any other that is."""
    row = Fake(torch.zeros(3, 68, dtype=BF16)[2:, :64])
    assert row.stride() == (68, 1)
    assert L._rows(CTX, "t", "x", row, (BF16,), 1, 64)[1] == 64
    assert L._rows(CTX, "t", "x", Fake(torch.zeros(3, 68, dtype=BF16)[:, :64]), (BF16,), 3, 64)[1] == 68


def test_key_heads_without_keys_are_refused():
    q = fake(4, 128)
    assert kind_of(L.qk_norm_rope, q, None, q, None, 1, 1, None, None) == "INVALID_ARG"
    assert kind_of(L.qk_norm_rope, q, q, q, None, 1, 1, None, None) == "INVALID_ARG"
