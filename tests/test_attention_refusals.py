"""What attention refuses, on the CPU: wrong shapes, types and sequences raise before anything reaches a device, and the
C entry points return error codes."""
import ctypes

import pytest
import torch

from transformer_amd import _lib
from transformer_amd.attention import Sequences, attention


def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("q,k,v,match", [
    (_x(4, 64), _x(4, 64), _x(4, 64), "expected"),
    (_x(1, 4, 2, 64), _x(4, 2, 64), _x(4, 2, 64), "expected"),
    (_x(4, 2, 64), _x(4, 2, 64), _x(5, 2, 64), "expected"),
    (_x(4, 2, 64, dtype=torch.float32), _x(4, 2, 64), _x(4, 2, 64), "bfloat16"),
    (_x(4, 2, 64, dtype=torch.float16), _x(4, 2, 64, dtype=torch.float16), _x(4, 2, 64, dtype=torch.float16), "bfloat16"),
    (_x(4, 2, 64), _x(4, 2, 64), _x(4, 2, 64), "GPU"),
])
def test_operands(q, k, v, match):
    with pytest.raises(ValueError, match=match):
        attention(q, k, v)


@pytest.mark.parametrize("args,match", [
    (([3, -1],), "negative"),
    (([3], [3, 4]), "key sequences"),
    (([3, 4], None, [0]), "starts"),
    (([3, 4], None, [0, 2]), "overlap"),
    (([3, 4], None, [-1, 5]), "overlap|outside"),
    (([2 ** 31],), "outside"),
    (([1], [1], [0], [2 ** 31]), "outside"),
])
def test_sequences(args, match):
    with pytest.raises(ValueError, match=match):
        Sequences(*args, device="cpu")


def test_sequence_tables():
    s = Sequences([3, 0, 5], device="cpu")
    assert s.table.tolist() == [[3, 5, 3, 5], [0, 3, 0, 3], [3, 0, 3, 0]] and s.table.dtype == torch.int32
    assert (s.n, s.q_longest, s.k_longest, s.q_end, s.k_end, s.q_count, s.k_count) == (3, 5, 5, 8, 8, 8, 8)
    s = Sequences([2, 1], q_starts=range(0, 10, 5), device="cpu")   # a padded batch: the keys lie where the queries do
    assert s.table.tolist() == [[0, 2, 0, 2], [5, 1, 5, 1]] and (s.q_end, s.q_count) == (6, 3)
    s = Sequences([2, 1], [4, 0], device="cpu")
    assert s.table.tolist() == [[0, 2, 0, 4], [2, 1, 4, 0]]
    assert Sequences([], device="cpu").table.shape == (0, 4)


HOST = (ctypes.c_int32 * 8)(0, 10, 0, 20, 10, 9, 20, 20)


def _args(**kw):
    a = _lib.MsdAttn()
    if kw.get("seqs"):
        kw = {"seqs_host": ctypes.addressof(HOST), **kw}
    base = dict(n_seqs=2, q_len=10, k_len=20, n_heads=4, n_kv_heads=2, d_head=64, causal=1, scale=0.125, q_rows=20, k_rows=40)
    base.update({k: v for k, v in kw.items() if "stride" not in k})
    for k, v in base.items():
        setattr(a, k, v)
    a.q_stride[:], a.dout_stride[:] = (2560, 256, 64), (2560, 256, 64)
    a.k_stride[:], a.v_stride[:] = (2560, 128, 64), (2560, 128, 64)
    for k in ("q_stride", "k_stride", "v_stride", "dout_stride"):
        if k in kw:
            getattr(a, k)[:] = kw[k]
    return a


BAD = [dict(n_seqs=-1), dict(q_len=-1), dict(k_len=-1), dict(n_heads=0), dict(n_kv_heads=0), dict(n_heads=3), dict(d_head=0),
       dict(d_head=136), dict(d_head=60), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
       dict(scale=float("inf")), dict(q_rows=21), dict(k_rows=39), dict(q_stride=(2560, 256, 60)),
       dict(k_stride=(2560, -128, 64)), dict(v_stride=(2560, 1 << 25, 64)), dict(q_rows=1 << 31, seqs=16),
       dict(q_rows=5, seqs=16), dict(n_seqs=70000, q_rows=700000, k_rows=1400000),
       dict(q_rows=1 << 30, k_rows=40, seqs=16), dict(q_rows=18, seqs=16), dict(k_rows=39, seqs=16), dict(q_len=9, seqs=16),
       dict(k_len=19, seqs=16), dict(q_len=1 << 29, q_rows=1 << 29, n_seqs=1)]


@pytest.mark.parametrize("kw", BAD)
def test_c_refuses_shapes(kw):
    L, a = _lib.lib(), _args(**kw)
    p = ctypes.c_void_p(4096)
    assert L.msd_attn_workspace_bytes(ctypes.byref(a), 0) == _lib.MSD_E_CONFIG
    assert L.msd_attn_forward(ctypes.byref(a), p, p, p, p, p, p, p, None) == _lib.MSD_E_CONFIG
    assert L.msd_attn_backward(ctypes.byref(a), p, p, p, p, p, p, p, p, p, p, p, None) == _lib.MSD_E_CONFIG


def test_c_refuses_pointers():
    L, p = _lib.lib(), ctypes.c_void_p(4096)
    assert L.msd_attn_workspace_bytes(None, 0) == _lib.MSD_E_ARG
    assert L.msd_attn_forward(None, p, p, p, p, p, p, p, None) == _lib.MSD_E_ARG
    a = _args()
    for bad in (None, ctypes.c_void_p(4104)):
        for i in (0, 1, 2, 3):
            args = [p] * 7
            args[i] = bad
            assert L.msd_attn_forward(ctypes.byref(a), *args, None) == _lib.MSD_E_ARG
        for i in [i for i in range(11) if i != 4]:   # (out_low may be missing)
            args = [p] * 11
            args[i] = bad
            assert L.msd_attn_backward(ctypes.byref(a), *args, None) == _lib.MSD_E_ARG
    for kw in (dict(seqs=4100), dict(seqs=16, seqs_host=None), dict(seqs=16, seqs_host=4098)):
        a = _args(**kw)
        assert L.msd_attn_workspace_bytes(ctypes.byref(a), 0) == _lib.MSD_E_ARG
    assert L.msd_attn_workspace_bytes(ctypes.byref(_args(seqs=16)), 0) >= 0
    assert L.msd_attn_forward(ctypes.byref(a), p, p, p, p, p, p, p, None) == _lib.MSD_E_ARG
    a = _args(dout_stride=(1, 1, 1))
    assert L.msd_attn_backward(ctypes.byref(a), *[p] * 11, None) == _lib.MSD_E_CONFIG


def test_workspaces():
    L = _lib.lib()
    assert L.msd_attn_workspace_bytes(ctypes.byref(_args()), 0) >= 0
    assert L.msd_attn_workspace_bytes(ctypes.byref(_args()), 1) >= 8 * 20 * 4
    many = _args(n_seqs=64, q_len=2048, k_len=2048, q_rows=64 * 2048, k_rows=64 * 2048)   # enough workgroups: no parts
    assert L.msd_attn_workspace_bytes(ctypes.byref(many), 0) == 0
    assert L.msd_attn_workspace_bytes(ctypes.byref(many), 1) == 8 * 64 * 2048 * 4


@pytest.mark.parametrize("lens", [
    [(2 ** 25, 2 ** 25)],                         # 2^18 x 2^20 tiles of one sequence: counts beyond 32 bits
    [(100000, 1), (1, 10000)],                    # the parts of one sequence's rows, the keys of another
    [(2 ** 20, 0), (1, 2 ** 20)],
    [(0, 2 ** 25), (0, 0)],
])
@pytest.mark.parametrize("causal", [0, 1])
def test_workspace_of_uneven_sequences(lens, causal):
    """The plan's counts hold for the longest sequences, and its parts stay worth their memory."""
    rows, q, k = [], 0, 0
    for n, m in lens:
        rows += [q, n, k, m]
        q, k = q + n, k + m
    host = (ctypes.c_int32 * len(rows))(*rows)
    a = _args(n_seqs=len(lens), q_len=max(n for n, _ in lens), k_len=max(m for _, m in lens), n_heads=32, n_kv_heads=8, d_head=128,
              causal=causal, q_rows=q, k_rows=k, seqs=16, seqs_host=ctypes.addressof(host),
              q_stride=(0, 4096, 128), dout_stride=(0, 4096, 128), k_stride=(0, 1024, 128), v_stride=(0, 1024, 128))
    n = _lib.lib().msd_attn_workspace_bytes(ctypes.byref(a), 1)
    assert 8 * q * 32 <= n <= 8 * q * 32 + 256 + max(2 ** 31, 16 * k * 8 * 128 * (k > 2 ** 20), 4 * 5 * q * 32 * 128 * (k > 256))
