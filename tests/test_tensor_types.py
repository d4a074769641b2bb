"""Tensors of other types than f32 without a GPU: what takes f32 refuses them
before it allocates or launches anything."""
import numpy as np
import pytest

import smith_amd as S
from smith_amd import device, quantize


@pytest.fixture
def no_device(monkeypatch):
    """Whatever gets as far as the device fails as what it is."""
    def reached(*a, **k):
        raise AssertionError("the device was reached")
    monkeypatch.setattr(device, "ctx", reached)
    monkeypatch.setattr(device, "ops_ctx", reached)
    monkeypatch.setattr(device, "alloc", reached)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i32", "u8"])
@pytest.mark.parametrize("what", ["matmulQ4", "matmulQ8", "matmul_q4", "matmul_q8", "quantizeQ4", "quantizeQ8"])
def test_f32_is_asked_for(no_device, what, dtype):
    wq = S.QuantizedWeight(buffer=None, K=64, N=8, groups=2, totalBytes=2 * 8 * 34)
    a = S.Tensor([3, 64], dtype, buffer=1)  # never read
    with pytest.raises(ValueError, match="f32 wanted, got %s" % dtype):
        if what.startswith("matmul_"):
            quantize.matmul_reference_dispatch(what, a, wq)
        elif what.startswith("matmul"):
            getattr(S, what)(a, wq)
        else:
            getattr(S, what)(a)


@pytest.mark.parametrize("cos,sin", [("f16", "f16"), ("f32", "bf16"), ("u8", "f32"), ("f32", "i32")])
def test_rotary_tables_are_f32(no_device, cos, sin):
    pool = S.Tensor([8, 2, 16, 32], "f16", buffer=1)
    with pytest.raises(ValueError, match="cos and sin, f32 of one size"):
        S.pagedAppend(S.Tensor([5, 256], buffer=1), S.Tensor([5], "i32", buffer=1), S.Tensor([5], "i32", buffer=1), 4, pool,
                      pool, S.ROPE_HEAD, S.Tensor([800], cos, buffer=1), S.Tensor([800], sin, buffer=1))


@pytest.fixture
def host_memory(monkeypatch):
    """Tensors in host memory: what is uploaded is kept and downloaded."""
    held = {}
    monkeypatch.setattr(device, "alloc", lambda nbytes, mode=0: held.setdefault(len(held) + 1, None) or len(held))
    monkeypatch.setattr(device, "upload", lambda buf, a, offset=0: held.__setitem__(buf, a.tobytes()))
    monkeypatch.setattr(device, "download", lambda buf, nbytes, dtype, offset=0: np.frombuffer(held[buf][:nbytes], dtype))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "i32", "u8"])
def test_scalars_have_no_dimension(host_memory, dtype):
    one = 0x3F80 if dtype == "bf16" else 1
    for t, want in ((S.tensor(1.0, dtype=dtype), one), (S.zeros([], dtype), 0), (S.ones([], dtype), one),
                    (S.tensor(1.0, dtype=dtype).set_data(0.0), 0)):
        assert t.shape == [] and t.data.shape == () and S.toArray(t) == want
    assert S.tensor([[2.0, 4.0]], dtype=dtype).shape == [1, 2]
    assert S.toArray(S.tensor(np.arange(6.0).reshape(2, 3).T, dtype="f32")) == [[0, 3], [1, 4], [2, 5]]


def test_whole_numbers_in_bf16(host_memory):
    """Numbers are rounded whatever type they come in; an array of uint16, as
    .data gives it, is a bf16 tensor's own bits."""
    want = [0x3F80, 0xC000, 0x4380, 0x4380, 0x4382, 0]  # 1, -2, 256, 257 (a tie, to even), 259 (a tie), 0
    numbers = [1, -2, 256, 257, 259, 0]
    for values in (numbers, np.array(numbers, np.int32), np.array(numbers, np.float32), [float(x) for x in numbers]):
        assert S.tensor(values, dtype="bf16").data.tolist() == want
        assert S.create([6], "bf16").set_data(values).data.tolist() == want
    assert S.tensor(np.array([True, False]), dtype="bf16").data.tolist() == [0x3F80, 0]
    t = S.tensor(numbers, dtype="bf16")
    assert t.data.dtype == np.uint16
    assert S.tensor(t.data, dtype="bf16").data.tolist() == want
    assert S.create([6], "bf16").set_data(t.data).data.tolist() == want
