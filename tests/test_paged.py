"""The paged cache without a GPU: the code object holds the kernels the bridge
names, and the Python entry points refuse what does not fit."""
import re
import subprocess

import numpy as np
import pytest

import smith_amd as S
from smith_amd import device


def test_code_object_has_kernels():
    out = subprocess.run(["/opt/rocm/llvm/bin/llvm-readelf", "--syms", device.PAGED_CODE_OBJECT_PATH],
                         capture_output=True, text=True, check=True).stdout
    need = ["smith_paged_plan"]
    need += ["smith_paged_append_%s" % t for t in ("f32", "f16", "bf16")]
    need += ["smith_paged_attention_%s_d%d%s" % (t, d, e) for t in ("f32", "f16", "bf16", "rows_f32", "rows_f16", "rows_bf16")
             for d in (64, 96, 128) for e in ("", "_s") if not (e and t.startswith("rows"))]
    for k in need:
        assert re.search(r"\b%s\.kd\b" % k, out), k


def test_bf16_of_floats_rounds():
    from smith_amd.tensor import _host
    one = np.float32(1.0).view(np.uint32)
    bits = np.array([one, one + 0x7FFF, one + 0x8000, one + 0x8001, one + 0x18000, 0x7F7FFFFF, 0x7F800000, 0x7F800001,
                     0xFFFFFFFF, 0x80000001], np.uint32)
    want = [0x3F80, 0x3F80, 0x3F80, 0x3F81, 0x3F82, 0x7F80, 0x7F80, 0x7FC0, 0xFFFF, 0x8000]
    assert _host(bits.view(np.float32), "bf16").tolist() == want
    assert _host(np.array([1.0, -2.5]), "bf16").tolist() == [0x3F80, 0xC020]
    assert _host([0x3F80, 7], "bf16").tolist() == [0x3F80, 7]  # whole numbers are the bits


@pytest.mark.parametrize("dim", [4, 12, 136])
def test_cache_of_heads_that_no_kernel_takes(dim):
    with pytest.raises(ValueError, match="heads of %d dims" % dim):
        S.createPagedCache(dict(maxSeqLen=64, numKVHeads=2, headDim=dim, numLayers=1), 1, 4)


class Fake:
    """A tensor's shape and type without memory."""
    buffer = None

    def __init__(self, shape, dtype="f32"):
        self.shape, self.dtype, self.size = list(shape), dtype, int(np.prod(shape))


POOL = Fake([8, 2, 16, 32], "f16")


@pytest.mark.parametrize("change,message", [
    ({"cached": Fake([3])}, "pagedPlan: cached: i32"), ({"added": Fake([2], "i32")}, "pagedPlan: added: i32 \\[3\\]"),
    ({"freeCount": Fake([2], "i32")}, "freeCount"), ({"freePages": Fake([2, 2], "i32")}, "freePages"),
    ({"tables": Fake([2, 4], "i32")}, "tables: i32 \\[3, 4\\]"), ({"tables": Fake([3, 4])}, "tables")])
def test_plan_refusals(change, message):
    a = dict(cached=Fake([3], "i32"), added=Fake([3], "i32"), freePages=Fake([9], "i32"), freeCount=Fake([1], "i32"),
             tables=Fake([3, 4], "i32"), nPages=8, pageSize=16, maxRows=4)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        S.pagedPlan(**a)


@pytest.mark.parametrize("change,message", [
    ({"qkv": Fake([5, 255])}, "qkv: f32 \\[5, 256\\]"), ({"qkv": Fake([5, 256], "f16")}, "qkv"),
    ({"slots": Fake([4], "i32")}, "slots"), ({"positions": Fake([5])}, "positions"),
    ({"kPages": Fake([8, 2, 16, 32], "u8")}, "pages are"), ({"kPages": Fake([8, 16, 32], "f16")}, "pages are"),
    ({"vPages": Fake([8, 2, 16, 32])}, "vPages: f16"), ({"vPages": Fake([7, 2, 16, 32], "f16")}, "vPages"),
    ({"rope": S.ROPE_HEAD}, "need tables"), ({"rope": S.ROPE_ROW, "cos": Fake([64]), "sin": Fake([32])}, "of one size")])
def test_append_refusals(change, message):
    a = dict(qkv=Fake([5, 256]), slots=Fake([5], "i32"), positions=Fake([5], "i32"), numHeads=4, kPages=POOL, vPages=POOL)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        S.pagedAppend(**a)


@pytest.mark.parametrize("change,message", [
    ({"q": Fake([3, 100])}, "heads \\* 32"), ({"q": Fake([3, 128], "f16")}, "q is f32"),
    ({"lens": Fake([3])}, "lens"), ({"tables": Fake([2, 4], "i32")}, "tables"),
    ({"rowStart": Fake([3], "i32")}, "rowStart: i32 \\[4\\]"), ({"out": Fake([3, 64])}, "out"),
    ({"vPages": Fake([8, 2, 16, 32])}, "vPages")])
def test_attention_refusals(change, message):
    a = dict(q=Fake([3, 128]), lens=Fake([3], "i32"), tables=Fake([3, 4], "i32"), kPages=POOL, vPages=POOL)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        S.pagedAttention(**a)
