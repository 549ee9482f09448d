"""Calls of the streaming operators at the edges of what their documentation allows, on the GPU. Tolerances
as in test_gpu_chunk.py."""
import math

import pytest
import torch

import ab_attention_b200 as ab
from oracle import stream
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


# ---- a stream whose first call is captured --------------------------------------------------------------------


@pytest.mark.parametrize("batch,window,sinks,frames", [(1, None, 0, 4), (2, 2, 1, 9)])
def test_stream_attention_captured_first(batch, window, sinks, frames):
    """A stream's first call of every layer may be in a capture once its caches are there; the replays give what
    eager calls give. Without the caches the capture is refused."""
    def stream():
        return ab.StreamAttention(2, 5, 9, max_frames=frames, window_frames=window, sink_frames=sinks, batch=batch, page_size=16)

    def inputs(f):
        g = gen(f)
        return [normal(g, batch, 2, 45, 128) for _ in range(3)]

    eager, want = stream(), []
    for f in range(frames):
        q, k, v = inputs(f)
        want.append([eager(layer, q, k + layer, v).clone() for layer in range(2)])
        if f + 1 < frames:
            eager.advance()
    s, held = stream(), inputs(0)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="allocate"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        s(0, *held)
    s.allocate(range(2))
    caches = dict(s.caches)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [s(layer, held[0], held[1] + layer, held[2]) for layer in range(2)]
    for turn in range(2):
        for f in range(frames):
            for x, y in zip(held, inputs(f)):
                x.copy_(y)
            graph.replay()
            for x, y in zip(outs, want[f]):
                assert torch.equal(x, y)
            if f + 1 < frames:
                s.advance()
        s.reset()
    assert s.caches.keys() == caches.keys() and all(s.caches[x] is caches[x] for x in caches)


# ---- windows and blocks past 2^30 ---------------------------------------------------------------------------------


@pytest.mark.parametrize("window,block", [
    (2 ** 40 - 5, 2 ** 40),      # the window of the only block ends five keys after the first
    (2 ** 40 - 299, 2 ** 40),    # ... and after all but one
    (2 ** 35, 2 ** 40),          # ... and past the last: only the sinks are seen
    (2 ** 40, 2 ** 40), (2 ** 62, 2 ** 61), (2 ** 62, 2 ** 63 - 1), (2 ** 63 - 1, 1), (2 ** 30, 7), (2 ** 31, 2 ** 30 - 1),
    (2 ** 30 + 3, 2 ** 30 + 5), (10, 2 ** 30), (None, 2 ** 63 - 1),
])
@pytest.mark.parametrize("tokens", [2, 300])
def test_windows_and_blocks_of_any_size(window, block, tokens):
    g, keys = gen(tokens), 300
    q, k, v = normal(g, 1, 2, tokens, 128), normal(g, 1, 1, keys, 128), normal(g, 1, 1, keys, 128)
    # the definition's own sizes stay within 64 bits: a block past all positions ends where it says
    for sinks in (0, 3):
        o, lse = ab.window_attention(q, k, v, window=window, sinks=sinks, block=block, return_lse=True)
        hold(o[0].transpose(0, 1), lse[0].T, *(x[0].transpose(0, 1) for x in (q, k, v)), window=window, sinks=sinks, block=block)


def test_block_that_ends_past_2_to_30():
    """The second block of 805 million positions ends past 2^30, and without a window its tokens see all keys (of
    one page, in every place of the table): equal scores of 0, so the base-2 log-sum-exp is that of their count."""
    block, page = 0x30000000, 16384
    keys = torch.zeros(1, 1, page, 128, dtype=torch.bfloat16, device="cuda")
    values = torch.ones_like(keys)
    width = block // page + 1
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([width * page], dtype=torch.int32, device="cuda")
    q = torch.ones(1, 1, 128, dtype=torch.bfloat16, device="cuda")
    o, lse = ab.chunk_attention(q, ab.KVCache(keys, values), table, starts, lengths, block=block, return_lse=True)
    assert (o == 1).all()
    assert abs(lse.item() - math.log2(width * page)) < 5e-4


# ---- rows that repeat -----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim", [0, 1, 2])
@pytest.mark.parametrize("heads,kv", [(4, 2), (6, 2)])
def test_queries_that_repeat(heads, kv, dim):
    """Batches, heads or tokens of many rows that repeat by a stride of 0: as contiguous queries."""
    g = gen(dim)
    q, k, v = normal(g, 2, heads, 900, 128), normal(g, 2, kv, 1500, 128), normal(g, 2, kv, 1500, 128)
    one = q.narrow(dim, 0, 1).expand(2, heads, 900, 128)
    for x, y in zip(ab.window_attention(one, k, v, window=700, return_lse=True),
                    ab.window_attention(one.contiguous(), k, v, window=700, return_lse=True)):
        assert torch.equal(x, y)
    b = Batch(dim, [(700, 900), (300, 2000)], heads, kv, 32, torch.bfloat16)
    if dim > 0:
        one = b.q.narrow(2 - dim, 0, 1).expand(1000, heads, 128)
        for x, y in zip(ab.chunk_attention(one, b.cache, *b.plan, longest=700, return_lse=True),
                        ab.chunk_attention(one.contiguous(), b.cache, *b.plan, longest=700, return_lse=True)):
            assert torch.equal(x, y)


# ---- another device -------------------------------------------------------------------------------------------------


def test_stream_attention_keeps_its_device(monkeypatch):
    """The caches of a stream are made on the device that it was made on, whichever is current at a layer's first call."""
    made, kv_cache = [], ab.video.kv_cache
    monkeypatch.setattr(ab.video, "kv_cache", lambda *, device, **more: made.append(device) or kv_cache(device=device, **more))
    s = ab.StreamAttention(2, 5, 9, max_frames=2)
    s.allocate("ab")
    assert made == [s.page_table.device] * 2 and made[0].index is not None
    assert all(x.device == s.page_table.device for cache in s.caches.values() for x in cache)


# ---- fp16 over long rows ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens,keys,window,scale", [
    (1, 60000, None, 1), (300, 20000, None, 1), (300, 9000, None, 4), (32, 40000, None, 4), (260, 30000, 8000, 1),
])
def test_fp16_keeps_small_weights(tokens, keys, window, scale):
    """fp16 weights are lifted by 2^7 and the row's largest is at least its reference, so it is held as 2^7 or more.
    A weight below fp16's normal range is off by 2^-25 at most, 2^-32 of the largest: keys * 2^-32 * max |v| in
    all, beside what bf16 is held to with fp16's half step. Scores four times as large are off by four times as much."""
    g, half = gen(keys), torch.float16
    q = normal(g, 1, 4, tokens, 128, dtype=half) * scale
    k, v = normal(g, 1, 2, keys, 128, dtype=half), normal(g, 1, 2, keys, 128, dtype=half)
    o, lse = ab.window_attention(q, k, v, window=window, return_lse=True)
    ref, ref_lse, a = stream.attend(*(x[0].transpose(0, 1) for x in (q, k, v)), window=window)
    u = torch.finfo(half).eps / 2 * 1.01
    tol = (u + 4e-4 * scale) * a + u * ref.abs() + 2 ** -25 + keys * 2 ** -32 * v.double().abs().max()
    assert ((o[0].transpose(0, 1).double() - ref).abs() <= tol).all()
    assert ((lse[0].T.double() - ref_lse).abs() <= 5e-4 * scale).all()


# ---- the few-row kernel's ring of tiles under other traffic ---------------------------------------------------------


@pytest.mark.parametrize("page", [16, 128])
def test_tiles_stay_until_they_are_read(page):
    """Every CTA reports the sequences that are too long, which keeps the SMs' memory paths busy with atomics while
    the others' tiles are read: no tile may be written over before that. Equal calls give equal rows."""
    sizes = [(2, 357), (8, 74), (8, 407), (7, 1817), (8, 303), (1, 1979), (1, 1314), (1, 1456), (4, 1297), (1, 2307)] * 2
    sizes += [(8, 1591 - 40 * i) for i in range(14)] + [(1, 1528), (3, 1661), (1, 2172), (1, 2023), (2, 395), (1, 971)]
    b = Batch(page, sizes, 8, 8, page, torch.bfloat16)
    rows, at = [], 0
    for m, _ in sizes:
        rows += range(at, at + m) if m <= 3 else []
        at += m
    first = None
    for turn in range(60):
        o, lse = ab.chunk_attention(b.q, b.cache, *b.plan, longest=3, return_lse=True)
        o, lse = o[rows], lse[rows]
        if first is None:
            first, at = (o, lse), 0
            for s, (m, n) in enumerate(sizes):
                if m <= 3:
                    q = b.q[sum(x for x, _ in sizes[:s]):][:m]
                    hold(o[at:at + m], lse[at:at + m], q, b.k[s], b.v[s])
                    at += m
        assert torch.equal(o, first[0]) and torch.equal(lse, first[1])
    assert reported() == 1
