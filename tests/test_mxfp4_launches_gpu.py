"""The launches that the 4-bit linear counts are those that it makes."""
import pytest
import torch

from flex_shard_b200.ops import _lib
from flex_shard_b200.ops import mxfp4 as m4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,N,K,launches", [(1, 6144, 4096, 1), (4, 28672, 4096, 1), (5, 6144, 4096, 1), (16, 6144, 4096, 1), (16, 256, 512, 1),
                                            (5, 28672, 4096, 2), (16, 28672, 4096, 2), (17, 256, 512, 2)])
def test_counted_launches(T, N, K, launches):
    x = torch.randn(T, K, device="cuda").bfloat16()
    wq, _, fwd, _ = m4.mx4_quantize_weight_operands(torch.randn(N, K, device="cuda").bfloat16())
    m4.mxfp4_linear(x, None, wq, fwd, None)
    before = _lib.launch_count()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        m4.mxfp4_linear(x, None, wq, fwd, None)
        torch.cuda.synchronize()
    kernels = sum(e.count for e in prof.key_averages() if "mxf4" in e.key or "mxfp4" in e.key or "mx4_" in e.key)
    assert _lib.launch_count() - before == launches
    assert kernels in (launches, 0)         # 0: a machine whose profiler records no kernels
