"""Workspaces of attention over sequences that leave rows out, on the CPU: they follow the sequences' rows, not the tensors'."""
import ctypes
import random

import pytest

from transformer_amd import _lib


def workspace(q_lens, k_lens=None, gap=0, H=32, KV=8, D=128, causal=1):
    """(forward's, backward's) bytes of sequences in rows of `gap` each (0: packed), and the bytes of the statistics of all rows."""
    k_lens, rows, q, k = k_lens or q_lens, [], 0, 0
    for n, m in zip(q_lens, k_lens):
        rows += [q, n, k, m]
        q, k = q + (gap or n), k + (gap or m)
    host, a = (ctypes.c_int32 * len(rows))(*rows), _lib.MsdAttn()
    a.n_seqs, a.q_len, a.k_len, a.q_rows, a.k_rows = len(q_lens), max(q_lens), max(k_lens), q, k
    a.n_heads, a.n_kv_heads, a.d_head, a.causal, a.scale = H, KV, D, causal, D ** -0.5
    a.q_stride[:], a.dout_stride[:] = [(0, H * D, D)] * 2
    a.k_stride[:], a.v_stride[:] = [(0, KV * D, D)] * 2
    a.seqs, a.seqs_host = 16, ctypes.addressof(host)
    n = [_lib.check(_lib.lib().msd_attn_workspace_bytes(ctypes.byref(a), i), "workspace") for i in (0, 1)]
    return *n, (8 * q * H + 255) // 256 * 256


@pytest.mark.parametrize("q_lens,k_lens,gap", [
    ([1] * 16, [4096] * 16, 4096),       # a new row of each sequence of a padded batch
    ([4] * 64, [2048] * 64, 2048),
    ([300] * 2, None, 4096),
    ([1], [100000], 131072),
    ([1], [1], 131072),
    ([700, 20, 3], None, 50000),
    ([3000, 1], [1, 3000], 60000),
    ([1] * 256, [129] * 256, 4096),
])
@pytest.mark.parametrize("H,KV,D", [(32, 8, 128), (16, 1, 64), (4, 4, 8)])
@pytest.mark.parametrize("causal", [0, 1])
def test_padding_takes_no_workspace(q_lens, k_lens, gap, H, KV, D, causal):
    packed, padded = (workspace(q_lens, k_lens, g, H, KV, D, causal) for g in (0, gap))
    assert padded[0] == packed[0] and padded[1] - padded[2] == packed[1] - packed[2]
    # splits times workgroups of 128 rows: below 2 x 512; two tensors of 8192 parts of 128 keys
    assert padded[0] <= 1024 * 128 * 4 * (D + 1) and padded[1] - padded[2] <= 2 ** 30


def test_sizes_of_one_new_row_each():
    forward, backward, stats = workspace([1] * 16, [4096] * 16, 4096)
    assert forward == 4 * 4 * (16 * 8) * 4 * (128 + 1)   # floats, splits, workgroups, rows of a workgroup, values of a row
    assert backward == stats + forward // (128 + 1) * 128


@pytest.mark.parametrize("lens", [[32768] + [64] * 2299, [65536] + [64] * 1099, [64] * 300 + [32768] + [64] * 2000,
                                  [4096] * 257 + [1] * 40000, [1] * 65535], ids=len)
def test_many_sequences_and_a_long_one(lens):
    """Launches of as many workgroups as the sequences have, not of the longest's for each: 2300 times 1024 of 8 K/V heads each
    would be more than a launch can hold."""
    forward, backward, stats = workspace(lens, H=32, KV=8, D=128)
    assert forward <= 1024 * 128 * 4 * 129 and backward - stats <= 2 ** 30


@pytest.mark.parametrize("seed", range(300))
def test_sizes_stay_bounded(seed):
    """Any lengths, packed: uneven and even ones, empty ones, rows without keys, few heads and many."""
    rng = random.Random(seed)
    n, longest = int(2 ** rng.uniform(0, 11)), 2 ** rng.uniform(1, 14)

    def lens(longest):
        power = rng.choice([1, 1, 0.1])   # (mostly short, or mostly long)
        return [int(longest * rng.random() ** (1 / power) if power < 1 else longest ** rng.random()) * (rng.random() < 0.9) for _ in range(n)]

    q_lens, k_lens = lens(longest), None if rng.random() < 0.5 else lens(2 ** rng.uniform(1, 15))
    KV = rng.choice([1, 2, 4, 8, 32])
    H, D = KV * rng.choice([1, 2, 4, 7, 16]), rng.choice([8, 64, 72, 128])
    if not sum(q_lens) * H < 2 ** 31:
        pytest.skip("more rows than the library counts")
    forward, backward, stats = workspace(q_lens, k_lens, 0, H, KV, D, rng.randint(0, 1))
    assert forward <= 1024 * 128 * 4 * (D + 1) and backward - stats <= 2 ** 30 + 256


@pytest.mark.parametrize("q,k,H,KV,D", [(100000, 1000, 4096, 1, 128), (100000, 128, 512, 1, 128), (120, 120, 56, 8, 128), (1, 1, 4096, 1, 128),
                                        (5000, 1, 4096, 4, 128), (30000, 30000, 64, 1, 128)])
@pytest.mark.parametrize("B", [1, 3])
@pytest.mark.parametrize("causal", [0, 1])
def test_sizes_of_dense_batches(q, k, H, KV, D, B, causal):
    a = _lib.MsdAttn()
    a.n_seqs, a.q_len, a.k_len, a.q_rows, a.k_rows = B, q, k, B * q, B * k
    a.n_heads, a.n_kv_heads, a.d_head, a.causal, a.scale = H, KV, D, causal, 0.1
    a.q_stride[:], a.dout_stride[:] = [(q * H * D, H * D, D)] * 2
    a.k_stride[:], a.v_stride[:] = [(k * KV * D, KV * D, D)] * 2
    n = [_lib.check(_lib.lib().msd_attn_workspace_bytes(ctypes.byref(a), i), "workspace") for i in (0, 1)]
    assert n[0] <= 1024 * 128 * 4 * (D + 1) and n[1] <= 8 * B * q * H + 2 ** 30 + 512
