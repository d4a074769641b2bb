"""Tensors of other types than f32 without a GPU: what takes f32 refuses them
before it allocates or launches anything."""
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
