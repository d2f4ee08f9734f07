"""Launches past what a device counts are refused before any of a call's kernels is launched, on the CPU: a plan's own numbers, pointers
that nothing follows."""
import ctypes

import pytest
import torch

from transformer_amd import _lib
from transformer_amd.paged_attention import PagedSequences


def _call(n, q_len, length, H, KV, longest):
    pages = [range(-(-length // 16))] * n
    s = PagedSequences([q_len] * n, [length] * n, pages, H, KV, longest=longest, device="cpu")
    a = _lib.MsdPaged()
    a.d_head, a.scale, a.q_rows, a.positions, a.plan, a.plan_host = 64, 0.125, n * q_len, 1024, 16, s.host.data_ptr()
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = (64 * H, 64), (65536, 64), (65536, 64)
    return s, a


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are none of a device's")
@pytest.mark.parametrize("n,q_len,H,KV,longest,ok", [
    (520, 5, 64, 8, 131072, False),      # 4,259,840 workgroups of 1024 threads: past 2^32
    (512, 5, 64, 8, 131072, False),      # 4,194,304: 2^32
    (512, 5, 64, 8, 130944, True),       # 4,190,208
    (1, 40, 4, 4, 2 ** 27, False),       # 2^22 of a single sequence
    (1, 40, 4, 4, 2 ** 27 - 128, True),
])
def test_the_weights_of_chunks(n, q_len, H, KV, longest, ok):
    keep, a = _call(n, q_len, 40, H, KV, longest)
    L, p = _lib.lib(), ctypes.byref(a)
    rc = L.msd_paged_attn(p, 256, 256, 256, 256, None, 0, 256, 256, None)
    assert (rc == _lib.MSD_E_CONFIG) != ok and rc != _lib.MSD_OK   # (there is no device: what is not refused fails to be launched)
    assert L.msd_paged_attn(p, 256, 256, 256, 256, None, 0, None, 256, None) not in (_lib.MSD_E_CONFIG, _lib.MSD_OK)
