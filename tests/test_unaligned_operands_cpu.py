"""Dense operands that start anywhere in memory: what the host makes of them before a launch."""
import pytest
import torch

from flex_shard_b200.ops import _lib
from flex_shard_b200.ops.gemm import _rowmajor


@pytest.mark.parametrize("offset", [0, 1, 4, 7, 8])
def test_rows_for_the_copy_engine_start_on_a_boundary(offset):
    base = torch.randn(offset + 16 * 24).bfloat16()
    x = base[offset:].view(16, 24)
    y = _rowmajor(x)
    assert y.data_ptr() % 16 == 0 and y.stride() == (24, 1) and torch.equal(x, y)
    assert (y.data_ptr() == x.data_ptr()) == (x.data_ptr() % 16 == 0)      # copied only where it has to be


def test_a_single_row_of_any_stride():
    x = torch.randn(64).bfloat16().as_strided((1, 24), (7, 1))              # counts as contiguous
    y = _rowmajor(x)
    assert y.stride(0) % 8 == 0 and torch.equal(x, y)


@pytest.mark.skipif(not _lib.lib_path().exists(), reason="the native library is not built")
@pytest.mark.parametrize("codes,ld", [(4096 + 1, 128), (4096 + 2, 128), (4096, 130)])
def test_codes_off_a_word_are_refused(codes, ld):
    """The entry's own check, before anything is launched (the addresses are never used)."""
    from flex_shard_b200.ops import mxfp8

    mxfp8._ensure()
    assert _lib.load().fsb_mx_quant_act(8192, codes, 16384, 1, 128, 128, ld, None) == 1


@pytest.mark.skipif(not _lib.lib_path().exists(), reason="the native library is not built")
@pytest.mark.parametrize("codes,ld", [(4096 + 1, 128), (4096 + 2, 128), (4096, 130)])
def test_fp8_codes_off_a_word_are_refused(codes, ld):
    from flex_shard_b200.ops import fp8

    fp8._ensure()
    assert _lib.load().fsb_fp8_quant_act(8192, codes, 16384, 1, 128, 128, ld, None) == 1


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_dense(offset):
    base = torch.randn(offset + 64)
    x = base[offset:].view(4, 16)
    y = _lib.dense(x)
    assert y.data_ptr() % 16 == 0 and torch.equal(x, y) and (y is x) == (x.data_ptr() % 16 == 0)
    assert _lib.dense(x.t()).is_contiguous() and torch.equal(_lib.dense(x.t()), x.t())
