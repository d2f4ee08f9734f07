"""What few rows (up to 32 of a K/V head's group) keep of their probabilities as operands of the product with the values: two bf16, the
second being what the first's rounding has taken off.  Of a P in [2^n, 2^(n + 1)) that is at most 2^(n - 8), which is rounded by half a
step of its own, at most 2^(n - 17): both together are P to 2^-17.

Tolerance, element by element, with u = 2^-8 and e = 2^-12 as in test_paged_attention_gpu.py: (2^-17 + e) sum P |v| + u |out|.  Where the
output is small against sum P |v| that is less than what one bf16 of P leaves, and the test says first that it tells the two apart."""
import math

import pytest
import torch

from test_paged_attention_gpu import E, U, near, rand, reference, rows_of, tables_of
from transformer_amd.paged_attention import PagedSequences, paged_attention

pytestmark = pytest.mark.gpu


def with_one_bf16(q, k_pages, v_pages, q_len, length, table, scale):
    """The output of a sequence if the probabilities, as powers of two below their row's largest, were rounded to bf16 once."""
    H, g = q.shape[1], q.shape[1] // k_pages.shape[0]
    k, v = rows_of(k_pages, table, length).double(), rows_of(v_pages, table, length).double()
    see = torch.arange(length, device=q.device)[None] <= torch.arange(length - q_len, length, device=q.device)[:, None]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for h in range(H):
        s = (q[:, h].double() @ k[h // g].T * scale).masked_fill(~see, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        out[:, h] = p.to(torch.bfloat16).double() @ v[h // g] / p.sum(-1, keepdim=True)
    return out


@pytest.mark.parametrize("H,KV,D", [(16, 4, 64), (8, 2, 128), (6, 2, 96), (4, 4, 32)])
@pytest.mark.parametrize("name,more", [("one launch", []), ("pieces", [(1, 3000)]), ("beside chunks", [(60, 700)])])
def test_two_terms(name, more, H, KV, D):
    few = [(1, 3), (1, 7), (2, 9), (1, 40), (3, 100), (1, 500)]
    q_lens, lengths = ([x[i] for x in few + more] for i in (0, 1))
    starts = [sum(q_lens[:s]) for s in range(len(q_lens))]
    tables, n = tables_of(lengths, 1)
    q, k, v = rand((sum(q_lens), H, D), 2, 1.5), rand((KV, 16 * n, D), 3), rand((KV, 16 * n, D), 4)
    old = torch.zeros(len(q_lens), KV, 0, device="cuda")
    (ref, _), (tol, _) = reference(q, k, v, q_lens, lengths, tables, starts, D ** -0.5, None, max(lengths))
    total = (tol - U * ref.abs()) / (U + E)   # sum P |v|
    rows = sum(n for n, _ in few)
    ref, tol = ref[:rows], ((2.0 ** -17 + E) * total + U * ref.abs())[:rows]
    for s, (m, length) in enumerate(few[:3]):
        i = slice(starts[s], starts[s] + m)
        one = with_one_bf16(q[i], k, v, m, length, tables[s], D ** -0.5)
        assert ((one.to(torch.bfloat16).double() - ref[i]).abs() > tol[i]).any()
    sequences = PagedSequences(q_lens, lengths, tables, H, KV)
    near(paged_attention(q, k, v, sequences)[:rows], ref, tol, "out")
    near(paged_attention(q, k, v, sequences, weights=old)[0][:rows], ref, tol, "out, with weights")
