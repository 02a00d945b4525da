"""Host side of the cache calls on the GPU: the share-out's size, which kernel took a call."""
import ctypes as C
import math

import pytest

import cache_ref as ref
from test_cache import attend_args
from test_gpu_cache import DT, Problem, check_attend, eviction

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 100, 124, 125, 128, 200, 256])
def test_the_work_on_the_cuda_cores_is_shared_out_over_ctas_that_run_at_once(pkg, cuda, D):
    """The workspace holds two slots a CTA, from which their number follows; that many fit the SMs' shared memory (16 rows of Q, 64 of K and of V, 64 x 20 weights)."""
    import torch
    sm = torch.cuda.get_device_properties(0)
    need = pkg.lib().b200attn_cache_attend_workspace(bytes(attend_args(pkg, head_d=D, dtype=pkg.F32, num_heads=1, num_kv_heads=1, batch_sz=1, Kd=0, Vd=0, mask=0)))
    slot = (16 * (D + 2) + 3) // 4 * 4
    ctas = (need - 32) // (2 * slot * 4)    # (and one entry of 8 words)
    assert ctas % sm.multi_processor_count == 0 and ctas > 0
    pitch = ((D + 3) // 4 | 1) * 4
    smem = ((16 + 128) * pitch + 64 * 20) * 4
    assert ctas // sm.multi_processor_count * (smem + 1024) <= sm.shared_memory_per_multiprocessor - 1024
