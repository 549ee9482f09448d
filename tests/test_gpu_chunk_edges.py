"""Calls of the streaming operators at the edges of what their documentation allows, on the GPU. Tolerances
as in test_gpu_chunk.py."""
import pytest
import torch

import ab_attention_b200 as ab
from tests.test_gpu_chunk import Batch, clean_status, gen, hold, normal, reported  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- sequences with more tokens than the call covers ---------------------------------------------------------


@pytest.mark.parametrize("sizes,longest,heads,kv", [
    ([(2, 9000)], 1, 2, 1),                                     # few rows, equal parts: joined, a block a row
    ([(1, 9000), (2, 8000), (1, 700)], 1, 2, 1),                # few rows, equal spans
    ([(30, 9000)] + [(31, 700 + 50 * i) for i in range(5)], 30, 8, 8),  # ... joined by eight lanes a row
    ([(500, 9000)], 400, 4, 1),                                 # many rows, equal parts
    ([(300, 6000), (500, 6000), (20, 6000)], 300, 1, 1),        # many rows, equal spans
    ([(1, 40), (3, 50)], 1, 2, 1),                              # no join
])
def test_rows_of_dropped_sequences_stay(sizes, longest, heads, kv):
    """A sequence with more tokens than `longest` is reported, and its rows are left as they were."""
    b = Batch(31, sizes, heads, kv, 16, torch.bfloat16, behind=2)
    out = torch.full_like(b.q, 7)
    lse = torch.full(b.q.shape[:2], 7.0, device="cuda")
    junk = torch.full((1 << 26,), float("nan"), device="cuda")  # what a workspace may find
    del junk
    torch.ops.ab_attention.chunk_attention_out(b.q, *b.cache, *b.plan, longest, 0, 0, 1, out, lse)
    assert reported() == 1
    at = 0
    for s, (m, _) in enumerate(sizes):
        rows = slice(at, at + m)
        if m > longest:
            assert (out[rows] == 7).all() and (lse[rows] == 7).all()
        else:
            hold(out[rows], lse[rows], b.q[rows], b.k[s], b.v[s])
        at += m
    assert (out[at:] == 7).all() and (lse[at:] == 7).all()
