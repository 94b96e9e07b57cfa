"""The native entries of the 4-bit linear refuse scratch memory that is too short, before anything is launched (the addresses here
are never used: without a GPU a launch would give another error)."""
import pytest

from flex_shard_b200.ops import _lib
from flex_shard_b200.ops import mxfp4 as m4
from flex_shard_b200.ops.mxfp8 import blocked_scale_numel

pytestmark = pytest.mark.skipif(not _lib.lib_path().exists(), reason="the native library is not built")
BAD = 1
P = 1 << 20     # a 16-byte boundary


def linear(size, T=40, N=256, K=288, scratch=P):
    return _lib.load().fsb_mxfp4_linear(P, K, P, K // 2, P, P, N, scratch, size, T, N, K, P, None)


def input_gradient(size, T=40, N=256, K=384, scratch=P):
    return _lib.load().fsb_mxfp4_linear_dx(P, N, P, K // 2, P, P, scratch, size, T, N, K, P, None)


def weight_gradient(size, T=256, N=256, K=384, scratch=P):
    return _lib.load().fsb_mxfp4_linear_dw(P, N, P, K, P, 0, scratch, size, T, N, K, P, None)


@pytest.mark.parametrize("entry,size", [(linear, 40 * 144 + blocked_scale_numel(40, 288)),
                                        (input_gradient, 40 * 256 + 256 * 384 + blocked_scale_numel(40, 256)),
                                        (weight_gradient, (256 + 8) * 640)])
def test_short_scratch(entry, size):
    m4._ensure()
    for kw in (dict(size=size - 1), dict(size=0), dict(size=size, scratch=P + 8), dict(size=size, scratch=None)):
        assert entry(**kw) == BAD


def test_sizes_past_32_bits():
    m4._ensure()
    T, N, K = 1 << 20, 1 << 14, 1 << 14
    assert input_gradient((T * N + N * K) % 2 ** 32, T, N, K) == BAD
    assert weight_gradient((T + T // 32) * (N + K) % 2 ** 32, T, N, K) == BAD


def test_which_sizes_take_one_launch():
    m4._ensure()
    assert m4._one_launch(1, 6144, 4096) and m4._one_launch(16, 6144, 4096) and not m4._one_launch(16, 28672, 4096)
    assert not m4._one_launch(17, 128, 256) and m4._one_launch(1, 1, 32)
