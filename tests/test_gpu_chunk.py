"""Streaming operators on the GPU against their float64 restatement (oracle/stream.py).

Tolerances, element by element, with u = eps / 2 of the element type (half a rounding step):

* A turn: y = a cos - b sin is rounded once (u |y|; half a step of the smallest number, 2^-25, below
  fp16's normal range). Before that it is float32: the angle is reduced in 64 bits and rounded to 32
  (|angle| <= pi: 2^-23 absolute), sine and cosine are good to 2 units (2^-23), two products and a sum
  round by 2^-24 each: |a| + |b| times less than 2^-21.
* Attention: each weight is rounded to the element type for its product with V (u * A, A the same
  weights over |V|), the row's sum is not, and the result is rounded once (u |o|, 2^-25 below fp16's
  normal range; a weight below it loses 2^-25 of the largest weight, at most 2^8 below one:
  fp16 adds 2^-25 * sum |v| / l with l >= 2^-8, taken as 2^-17 * max |v| * keys... see `hold`).
  float32 parts: a score is a sum of 128 products, off by 128 * 2^-24 * sum |q_d k_d| * 128^-0.5,
  about 6e-5 for normal inputs, and moves a weight by that much relative; its exponential, the sums and the
  joins add some 2^-20. 4e-4 * A covers these with room for rows whose products are larger.
* LSE: score error 6e-5 * log2(e), plus 2^-22 of the largest |score|, the sums and one log2: 5e-4.
"""
import math

import pytest
import torch

import ab_attention_b200 as ab
from ab_attention_b200 import _lib
from oracle import stream

pytestmark = pytest.mark.gpu

BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32
AXES = {
    "video": ab.RotaryAxes(),
    "wide": ab.RotaryAxes((16, 56, 56), 256.0),
    "text": ab.RotaryAxes((32, 48, 48), 1e6, paired=False, shared=True),
    "line": ab.RotaryAxes((128,), 5e5, paired=False, shared=True),
    "four": ab.RotaryAxes((2, 0, 60, 66), 1e4, paired=False),
}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=BF):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(autouse=True)
def clean_status():
    assert _lib.device_status(clear=True) == 0
    yield
    assert _lib.device_status(clear=True) == 0


def reported():
    """The device error word, cleared."""
    return _lib.device_status(clear=True)


# ---- rotary ------------------------------------------------------------------------------------------


def hold_turn(y, x, positions, axes, inverse=False):
    ref = stream.turn(x, positions, axes.sections, axes.theta, axes.paired, axes.shared, inverse)
    a = x.double().abs()
    both = a[..., 0::2] + a[..., 1::2] if axes.paired else a[..., :64] + a[..., 64:]
    both = both.repeat_interleave(2, -1) if axes.paired else torch.cat((both, both), -1)
    tol = half_step(y.dtype) * ref.abs() * (1 + 2 ** -10) + both * 2 ** -21 + (2 ** -25 if y.dtype == HALF else 0)
    over = ((y.double() - ref).abs() - tol).max().item()
    assert over <= 0, f"off by {over} more than the rounding allows"


@pytest.mark.parametrize("axes", AXES)
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("batch,heads,kv,tokens,far,inverse", [
    (1, 1, 1, 1, 0, False), (2, 40, 8, 1, 1000003, False), (1, 3, 3, 33, 5, True), (2, 5, 1, 1000, 70000, False),
    (3, 12, 4, 129, 1 << 27, True),
])
def test_rotary(axes, dtype, batch, heads, kv, tokens, far, inverse):
    g = gen(heads * tokens)
    axes = AXES[axes]
    q, k = normal(g, batch, heads, tokens, 128, dtype=dtype), normal(g, batch, kv, tokens, 128, dtype=dtype)
    p = torch.randint(0, 500, (tokens, len(axes.sections)), generator=g, device="cuda", dtype=torch.int32) + far
    a, b = ab.apply_rotary(q, k, p, axes, inverse=inverse)
    assert a.is_contiguous() and b.is_contiguous() and a.dtype == dtype
    hold_turn(a, q, p, axes, inverse)
    hold_turn(b, k, p, axes, inverse)


def test_rotary_layouts_and_positions_per_batch():
    """Projections as they come ([B, N, H, 128]), heads cut from a joint projection, a broadcast
    batch, and rows that are not aligned all give what contiguous rows give."""
    g, axes = gen(3), AXES["video"]
    joint = normal(g, 2, 50, 3 * 6, 128)
    q, k = joint[:, :, :6].transpose(1, 2), joint[:, :, 6:12].transpose(1, 2)
    p = torch.randint(-30, 90, (2, 50, 3), generator=g, device="cuda", dtype=torch.int32)
    a, b = ab.apply_rotary(q, k, p, axes)
    for i in range(2):
        hold_turn(a[i], q[i], p[i], axes)
        hold_turn(b[i], k[i], p[i], axes)
    same, none = ab.apply_rotary(q.contiguous(), None, p, axes)
    assert none is None and torch.equal(same, a)
    odd = torch.empty(2 * 6 * 50 * 128 + 1, dtype=BF, device="cuda")[1:].view(2, 6, 50, 128).copy_(q)
    assert torch.equal(ab.apply_rotary(odd, None, p, axes)[0], a)
    wide = torch.empty(2, 6, 50, 129, dtype=BF, device="cuda")[..., :128].copy_(q)
    assert torch.equal(ab.apply_rotary(wide, None, p, axes)[0], a)
    one = q[:1, :1].expand(2, 6, 50, 128)
    assert torch.equal(ab.apply_rotary(one, None, p, axes)[0], ab.apply_rotary(one.contiguous(), None, p, axes)[0])


def test_rotary_of_nothing():
    p = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    q, k = ab.apply_rotary(torch.empty(2, 3, 0, 128, dtype=BF, device="cuda"), torch.empty(2, 1, 0, 128, dtype=BF, device="cuda"), p)
    assert q.shape == (2, 3, 0, 128) and k.shape == (2, 1, 0, 128)


def test_rotary_gradient_by_differences():
    """d(y . w)/dx by the turn back of w, against the formula and central differences (the turn is linear:
    float32 differences of step 1 are off by the rounding of y alone, 256 * 2^-22 * |y . w|'s terms)."""
    g, axes = gen(9), AXES["text"]
    x, w = normal(g, 1, 2, 3, 128, dtype=F32), normal(g, 1, 2, 3, 128, dtype=F32)
    p = torch.randint(0, 100, (3, 3), generator=g, device="cuda", dtype=torch.int32)
    grad = ab.apply_rotary(w, None, p, axes, inverse=True)[0]
    hold_turn(grad, w, p, axes, inverse=True)
    for h, n, d in ((0, 0, 0), (1, 2, 5), (0, 1, 64), (1, 0, 127)):
        step = torch.zeros_like(x)
        step[0, h, n, d] = 1
        up, down = (ab.apply_rotary(x + s * step, None, p, axes)[0].double() for s in (1, -1))
        assert abs((((up - down) / 2) * w.double()).sum().item() - grad[0, h, n, d].item()) < 1e-4


# ---- attention ---------------------------------------------------------------------------------------------


def hold(o, lse, q, k, v, **rule):
    """o [N, H, 128], lse [N, H] against the definition for q [N, H, 128], k and v [K, Hk, 128]."""
    if o.numel() == 0:
        return
    ref, ref_lse, a = stream.attend(q, k, v, **rule)
    u = half_step(o.dtype)
    tol = (u * 1.01 + 4e-4) * a + u * 1.01 * ref.abs()
    if o.dtype == HALF:
        # weights below 2^-14 of the row's largest keep 2^-25 of it: at most keys * 2^-25 * max|v| in all
        tol = tol + 2 ** -25 + k.shape[0] * 2 ** -25 * (v.double().abs().max() if v.numel() else 0)
    assert torch.isfinite(o).all()
    over = ((o.double() - ref).abs() - tol).max().item()
    assert over <= 0, f"off by {over} more than the roundings allow"
    if lse is not None:
        empty = ref_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        assert (o[empty] == 0).all()
        assert ((lse.double() - ref_lse)[~empty].abs() <= 5e-4).all()


WINDOWS = [
    # batch, heads, kv, tokens, keys, window, sinks, block
    (1, 1, 1, 1, 1, None, 0, 1), (2, 4, 2, 1, 63, None, 0, 1), (1, 8, 1, 1, 5000, None, 0, 1), (3, 12, 12, 1, 1000, 100, 4, 1),
    (1, 40, 8, 1, 8191, 4096, 4, 1), (2, 6, 3, 3, 129, None, 0, 1), (1, 5, 1, 5, 300, 64, 0, 1), (2, 4, 4, 7, 7, None, 0, 1),
    (1, 2, 1, 33, 500, 40, 130, 1), (1, 3, 3, 128, 128, None, 0, 1), (1, 4, 1, 257, 257, 64, 3, 1), (2, 2, 2, 300, 1111, None, 0, 1),
    (1, 8, 2, 511, 511, 1, 0, 1), (1, 8, 2, 511, 2000, 100, 1, 1), (1, 2, 2, 1000, 1000, 200, 17, 96), (1, 3, 1, 640, 640, None, 0, 128),
    (2, 1, 1, 700, 900, 5, 0, 64), (1, 2, 2, 50, 20, None, 0, 1), (1, 2, 1, 300, 100, 10, 2, 1), (1, 2, 2, 900, 650, 40, 2, 32),
    (1, 7, 1, 200, 3000, 700, 140, 1), (1, 1, 1, 4100, 4100, 333, 7, 1), (1, 16, 2, 1000, 1000, 10000, 5000, 1),
    (1, 2, 2, 260, 1500, 260, 0, 10 ** 9), (1, 2, 2, 2, 600, 10 ** 12, 10 ** 12, 1),
]


@pytest.mark.parametrize("batch,heads,kv,tokens,keys,window,sinks,block", WINDOWS)
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_window_attention(batch, heads, kv, tokens, keys, window, sinks, block, dtype):
    g = gen(tokens + keys)
    q = normal(g, batch, heads, tokens, 128, dtype=dtype)
    k, v = normal(g, batch, kv, keys, 128, dtype=dtype), normal(g, batch, kv, keys, 128, dtype=dtype)
    o, lse = ab.window_attention(q, k, v, window=window, sinks=sinks, block=block, return_lse=True)
    for b in range(batch):
        hold(o[b].transpose(0, 1), lse[b].T, *(x[b].transpose(0, 1) for x in (q, k, v)), window=window, sinks=sinks, block=block)
    assert torch.equal(o, ab.window_attention(q, k, v, window=window, sinks=sinks, block=block))


@pytest.mark.parametrize("tokens,keys", [(1, 700), (200, 700), (600, 700)])
def test_window_attention_layouts(tokens, keys):
    """Projection layouts, broadcast and unaligned keys give what contiguous tensors give."""
    g = gen(tokens)
    q, k, v = (normal(g, 2, n, h, 128).transpose(1, 2) for n, h in ((tokens, 4), (keys, 2), (keys, 2)))
    want = ab.window_attention(*(x.contiguous() for x in (q, k, v)), window=300, sinks=3)
    assert torch.equal(ab.window_attention(q, k, v, window=300, sinks=3), want)
    odd = torch.empty(k.numel() + 1, dtype=BF, device="cuda")[1:].view(k.shape).copy_(k)
    assert torch.equal(ab.window_attention(q, odd, v, window=300, sinks=3), want)
    shared = k[:, :1].expand(-1, 2, -1, -1)
    assert torch.equal(ab.window_attention(q, shared, v), ab.window_attention(q, shared.contiguous(), v))


@pytest.mark.parametrize("tokens", [1, 70, 400])
def test_large_and_extreme_scores(tokens):
    """Scores of hundreds (a row is one key), one type's lowest value in K, and equal scores."""
    g = gen(tokens)
    q, k, v = normal(g, 1, 2, tokens, 128), normal(g, 1, 2, 500, 128), normal(g, 1, 2, 500, 128)
    for scale in (0.0, 30.0):
        o, lse = ab.window_attention(q * scale, k, v, return_lse=True)
        ref, ref_lse, a = stream.attend((q * scale)[0].transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1))
        # a score of s is off by 2^-17 |s| at most (128 roundings of 2^-24): 30 * 60 * 2^-17 = 0.014 of the weights
        tol = (2 ** -8 * 1.01 + (4e-4 if scale == 0 else 0.03)) * a + 2 ** -8 * 1.01 * ref.abs()
        assert ((o[0].transpose(0, 1).double() - ref).abs() <= tol).all()
        assert ((lse[0].T.double() - ref_lse).abs() <= 5e-4 + 2e-5 * ref_lse.abs()).all()
    k = k.clone()
    k[:, :, 7] = torch.finfo(BF).min / 256  # finite scores of +-1e36
    o = ab.window_attention(q, k, v)
    assert torch.isfinite(o).all()
    top = (q.double() @ k[:, :, 7, :, None].double())[..., 0] > 0
    seen = top[0] & (500 - tokens + torch.arange(tokens, device="cuda") >= 7)
    assert torch.equal(o[0][seen], v[0][:, None, 7].expand(-1, tokens, -1)[seen])


@pytest.mark.parametrize("tokens,keys", [(1, 40), (1, 20000), (3, 9000), (40, 700), (300, 3000)])
def test_nan_in_a_query_stays_in_its_row(tokens, keys):
    g = gen(keys)
    q, k, v = normal(g, 1, 4, tokens, 128), normal(g, 1, 2, keys, 128), normal(g, 1, 2, keys, 128)
    want, want_lse = ab.window_attention(q, k, v, return_lse=True)
    bad = q.clone()
    bad[0, 1, tokens // 2, 5] = math.nan
    o, lse = ab.window_attention(bad, k, v, return_lse=True)
    assert o[0, 1, tokens // 2].isnan().all() and lse[0, 1, tokens // 2].isnan()
    o[0, 1, tokens // 2], lse[0, 1, tokens // 2] = want[0, 1, tokens // 2], want_lse[0, 1, tokens // 2]
    assert torch.equal(o, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("batch,heads,kv,tokens,keys,rule", [
    (1, 12, 12, 1000, 1000, {"block": 1000}),           # fewer row tiles than half the SMs
    (2, 12, 4, 1045, 1300, {"window": 700, "sinks": 5}),  # 3 heads a key head: queries loaded one by one
    (1, 16, 4, 1032, 1032, {}),                         # 16.1 row tiles a key head: the last half has no rows
    (1, 38, 38, 1025, 1025, {"window": 400}),           # 190 row tiles, 42 of them in the last wave
    (3, 20, 20, 700, 700, {"block": 70}),               # 180 row tiles of three sequences
])
def test_row_tiles_in_halves(batch, heads, kv, tokens, keys, rule):
    """The row tiles of a last wave are taken in halves."""
    g = gen(tokens + heads)
    q = normal(g, batch, heads, tokens, 128)
    k, v = (normal(g, batch, kv, keys, 128) for _ in range(2))
    rule = {"window": None, "sinks": 0, "block": 1} | rule
    o, lse = ab.window_attention(q, k, v, return_lse=True, **rule)
    for b in range(batch):
        hold(o[b].transpose(0, 1), lse[b].T, *(x[b].transpose(0, 1) for x in (q, k, v)), **rule)


@pytest.mark.parametrize("heads,kv,tokens,keys,window,sinks,block", [
    (36, 36, 1500, 1500, 100, 3, 1), (40, 8, 1100, 1400, None, 0, 1), (24, 2, 777, 777, 33, 130, 64), (70, 14, 900, 300, None, 0, 1),
])
def test_many_tiles_of_rows(heads, kv, tokens, keys, window, sinks, block):
    """More row tiles than the GPU holds at a time, so that each CTA works on several, one after the other."""
    g = gen(heads)
    q, k, v = normal(g, 2, heads, tokens, 128), normal(g, 2, kv, keys, 128), normal(g, 2, kv, keys, 128)
    o, lse = ab.window_attention(q, k, v, window=window, sinks=sinks, block=block, return_lse=True)
    for b in range(2):
        hold(o[b].transpose(0, 1), lse[b].T, *(x[b].transpose(0, 1) for x in (q, k, v)), window=window, sinks=sinks, block=block)
    for _ in range(3):
        again = ab.window_attention(q, k, v, window=window, sinks=sinks, block=block, return_lse=True)
        assert torch.equal(again[0], o) and torch.equal(again[1], lse)


@pytest.mark.parametrize("heads,kv,page", [(16, 16, 16), (20, 4, 64)])
def test_many_ragged_chunks(heads, kv, page):
    """The same for ragged chunks: tiles of one group of rows and of two, sequences without keys or tokens among them."""
    sizes = [((37 * i) % 150, (211 * i) % 700) for i in range(90)] + [(0, 50), (130, 0), (300, 900), (128, 128), (129, 4)]
    b = Batch(page, sizes, heads, kv, page, BF)
    rule = {"window": None, "sinks": 0, "block": 1}
    first = ab.chunk_attention(b.q, b.cache, *b.plan, longest=300, return_lse=True, **rule)
    b.check(*first, **rule)
    for _ in range(3):
        again = ab.chunk_attention(b.q, b.cache, *b.plan, longest=300, return_lse=True, **rule)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.parametrize("tokens", [1, 300])
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_many_small_weights(tokens, dtype):
    """One key outweighs each of 60,000 others 2^22.6 times, and they make up the result. fp16 ends at 2^-24:
    weights are lifted by 2^7, so each is off by at most 2^-25 / 2^7 of the largest (bf16 keeps its 2^-8 of each)."""
    keys = 60000
    q, k = torch.ones(1, 1, tokens, 128, dtype=dtype, device="cuda"), torch.zeros(1, 1, keys, 128, dtype=dtype, device="cuda")
    v = torch.ones_like(k)
    k[:, :, 0], v[:, :, 0] = 1.384765625, 0
    o, lse = ab.window_attention(q, k, v, return_lse=True)
    ref, ref_lse, a = stream.attend(q[0].transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1))
    u = half_step(dtype)
    tol = (2.02 * u + 4e-4) * a + (keys * 2 ** -32 if dtype == HALF else 0)
    assert ((o[0].transpose(0, 1).double() - ref).abs() <= tol).all()
    assert ((lse[0].T.double() - ref_lse).abs() <= 5e-4).all()


def test_window_attention_of_nothing():
    empty = torch.empty(2, 4, 0, 128, dtype=BF, device="cuda")
    q = torch.randn(2, 4, 3, 128, device="cuda").to(BF)
    o, lse = ab.window_attention(q, empty, empty, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    o, lse = ab.window_attention(empty, q, q, return_lse=True)
    assert o.shape == (2, 4, 0, 128) and lse.shape == (2, 4, 0)


class Batch:
    """A cache with random pages, NaN in every row that no sequence owns, and packed new tokens."""

    def __init__(self, seed, sizes, heads, kv, page, dtype, behind=0, spare=2, token_major=False):
        g = gen(seed)
        self.sizes, self.heads, self.kv = sizes, heads, kv
        width = max(1, max((-(-n // page) for _, n in sizes), default=1)) + 1
        used = [-(-n // page) for _, n in sizes]
        pages = sum(used) + spare
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        # entries behind a sequence's pages name no page: never read
        self.table = torch.full((len(sizes), width), 10 ** 6, dtype=torch.int32, device="cuda")
        if token_major:
            self.keys, self.values = (torch.full((pages, page, kv, 128), math.nan, dtype=dtype, device="cuda").transpose(1, 2)
                                      for _ in range(2))
        else:
            self.keys, self.values = (torch.full((pages, kv, page, 128), math.nan, dtype=dtype, device="cuda") for _ in range(2))
        self.values[::2] = math.inf
        self.k, self.v, at = [], [], 0
        for s, (_, n) in enumerate(sizes):
            self.table[s, :used[s]] = order[at:at + used[s]]
            self.k.append(normal(g, n, kv, 128, dtype=dtype))
            self.v.append(normal(g, n, kv, 128, dtype=dtype))
            for x, rows in ((self.keys, self.k[s]), (self.values, self.v[s])):
                for i in range(used[s]):
                    part = rows[i * page:(i + 1) * page]
                    x[order[at + i].item(), :, :part.shape[0]] = part.transpose(0, 1)
            at += used[s]
        starts = [0]
        for m, _ in sizes:
            starts.append(starts[-1] + m)
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.lengths = torch.tensor([n for _, n in sizes], dtype=torch.int32, device="cuda")
        self.q = normal(g, starts[-1] + behind, heads, 128, dtype=dtype)
        self.cache = ab.KVCache(self.keys, self.values)

    @property
    def plan(self):
        return self.table, self.starts, self.lengths

    def check(self, o, lse, **rule):
        at = 0
        for s, (m, n) in enumerate(self.sizes):
            hold(o[at:at + m], None if lse is None else lse[at:at + m], self.q[at:at + m], self.k[s], self.v[s], **rule)
            at += m


CHUNKS = [
    # [(new, keys)], heads, kv, page, window, sinks, block
    ([(1, 1)], 1, 1, 16, None, 0, 1),
    ([(1, 17), (1, 1), (1, 100), (1, 333)], 8, 2, 16, None, 0, 1),
    ([(1, 2049), (0, 70), (1, 64), (0, 0), (1, 65)], 12, 12, 64, None, 0, 1),
    ([(1, 9000), (1, 5), (1, 4097)], 32, 4, 128, None, 0, 1),
    ([(1, 9000), (1, 5), (1, 4097)], 16, 1, 32, 1000, 7, 1),
    ([(3, 40), (2, 700), (1, 1), (4, 4)], 8, 1, 16, None, 0, 1),
    ([(5, 300), (2, 700)], 10, 2, 256, 129, 70, 1),
    ([(130, 130), (1, 900), (300, 1000), (0, 55), (64, 64)], 4, 2, 16, None, 0, 1),
    ([(257, 700), (128, 128)], 5, 5, 32, 150, 3, 1),
    ([(40, 1000), (700, 700)], 8, 8, 64, 64, 130, 16),
    ([(900, 2500)], 3, 1, 128, None, 0, 300),
    ([(600, 5000)], 12, 4, 384, 1500, 10, 1),
    ([(10, 4), (1, 0), (200, 150)], 4, 1, 16, None, 0, 1),  # more new tokens than keys: rows before the first key
    ([(1, 30)] * 70, 2, 2, 16, None, 0, 1),
    ([(2, 70)] * 40 + [(150, 180)] * 3, 6, 2, 16, 33, 2, 7),
]


@pytest.mark.parametrize("sizes,heads,kv,page,window,sinks,block", CHUNKS)
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_chunk_attention(sizes, heads, kv, page, window, sinks, block, dtype):
    b = Batch(len(sizes) + page, sizes, heads, kv, page, dtype, behind=3)
    rule = {"window": window, "sinks": sinks, "block": block}
    longest = max(m for m, _ in sizes)
    out = torch.full_like(b.q, 7)
    o, lse = ab.chunk_attention(b.q, b.cache, *b.plan, longest=longest, return_lse=True, out=out, **rule)
    assert o is out
    b.check(o, lse, **rule)
    assert (out[sum(m for m, _ in sizes):] == 7).all()  # rows behind the last sequence
    # without the hint, and with token-major pages
    o = ab.chunk_attention(b.q, b.cache, *b.plan, **rule)
    b.check(o, None, **rule)
    b = Batch(len(sizes) + page, sizes, heads, kv, page, dtype, token_major=True)
    b.check(*ab.chunk_attention(b.q, b.cache, *b.plan, longest=longest, return_lse=True, **rule), **rule)


@pytest.mark.parametrize("new,heads", [(1, 4), (90, 2)])
def test_pages_behind_the_window_may_be_gone(new, heads):
    """Pages that no new token sees may be given back: their table entries are not read."""
    page, n, window, sinks = 16, 1000, 100, 20
    b = Batch(5, [(new, n)], heads, 2, page, BF)
    rule = {"window": window, "sinks": sinks, "block": 1}
    want = ab.chunk_attention(b.q, b.cache, *b.plan, longest=new, **rule)
    first = (n - new + 1 - window) // page  # the first page that the first new token still sees
    b.table[0, -(-sinks // page):first] = -1
    assert torch.equal(ab.chunk_attention(b.q, b.cache, *b.plan, longest=new, **rule), want)
    b.check(want, None, **rule)


@pytest.mark.parametrize("count,most,keys,heads,kv", [(2, 400, 900, 4, 4), (31, 90, 700, 8, 2), (40, 70, 300, 8, 4), (75, 45, 200, 12, 12)])
def test_ragged_sequences_in_order_of_length(count, most, keys, heads, kv):
    """Sequences of many lengths, some equal, some without tokens or keys: every 32 are taken longest first."""
    sizes = []
    for s in range(count):
        new = s * 37 % (most + 1) if s % 5 else 0
        sizes.append((new, 0 if s % 10 == 0 else max(new, s * 101 % (keys + 1) // 50 * 50)))
    sizes[count // 2] = (most, keys)
    b = Batch(count, sizes, heads, kv, 16, BF, behind=2)
    for rule in ({"window": None, "sinks": 0, "block": 1}, {"window": 77, "sinks": 3, "block": 10}):
        o, lse = ab.chunk_attention(b.q, b.cache, *b.plan, longest=most, return_lse=True, **rule)
        b.check(o, lse, **rule)


@pytest.mark.parametrize("page", [16, 64, 128, 256, None])
@pytest.mark.parametrize("sinks,window", [(1, 1000), (64, 190), (65, 64), (130, 333), (190, 1)])
@pytest.mark.parametrize("new", [7, 290])
def test_sinks_beside_a_window(new, sinks, window, page):
    """The sinks' keys and the window's lie in one tile, and what lies between, which no token sees, is NaN."""
    n, heads, kv = 1733, 8, 2
    b = Batch(new + sinks, [(new, n)], heads, kv, page or 16, BF)
    rule = {"window": window, "sinks": sinks, "block": 1}
    hidden = range(sinks, n - new + 1 - window)
    if page:
        for j in hidden:
            at = b.table[0, j // page].item()
            b.keys[at, :, j % page] = b.values[at, :, j % page] = math.nan
        b.check(*ab.chunk_attention(b.q, b.cache, *b.plan, longest=new, return_lse=True, **rule), **rule)
        return
    q, k, v = (x.transpose(0, 1)[None].contiguous() for x in (b.q, b.k[0], b.v[0]))
    k[:, :, hidden.start:hidden.stop] = v[:, :, hidden.start:hidden.stop] = math.nan
    o, lse = ab.window_attention(q, k, v, return_lse=True, **rule)
    b.check(o[0].transpose(0, 1), lse[0].T, **rule)


@pytest.mark.parametrize("new", [1, 50])
def test_bad_pages_lengths_and_chunks_are_reported(new):
    """What the device finds wrong is reported in the device error word, and nothing is read or
    written out of range: a page that is needed and does not exist, a length past the table, starts past
    the tokens, and a sequence longer than `longest`."""
    b = Batch(6, [(new, 200), (new, 60)], 2, 1, 16, BF)
    good = ab.chunk_attention(b.q, b.cache, *b.plan, longest=new)
    assert reported() == 0
    for entry in (-1, b.keys.shape[0], 2 ** 31 - 1):
        table = b.table.clone()
        table[0, 5] = entry
        o = ab.chunk_attention(b.q, b.cache, table, b.starts, b.lengths, longest=new)
        assert reported() == 1 and torch.equal(o[new:], good[new:])
    lengths = b.lengths.clone()
    lengths[1] = 10 ** 6
    table = b.table.clone().fill_(0)
    table[0] = b.table[0]
    table[0, -(-200 // 16):] = 0
    o = ab.chunk_attention(b.q, b.cache, table, b.starts, lengths, longest=new)
    assert reported() == 1 and torch.equal(o[:new], good[:new])
    starts = b.starts.clone()
    starts[2] = 10 ** 6
    starts[0] = -3
    ab.chunk_attention(b.q, b.cache, *((b.table, starts, b.lengths)), longest=2 * new)
    assert reported() == 1
    if new > 1:
        out = torch.full_like(b.q, 7)
        ab.chunk_attention(b.q, b.cache, *b.plan, longest=new - 1, out=out)
        assert reported() == 1
        assert torch.equal(ab.chunk_attention(b.q, b.cache, *b.plan, longest=new), good)


@pytest.mark.parametrize("new", [1, 90])
def test_joint_buffers_and_strided_outputs(new):
    """Keys and values in one buffer, outputs head by head, queries whose heads repeat: as contiguous tensors."""
    b = Batch(14, [(new, 700), (new, 90)], 4, 2, 32, BF)
    want, want_lse = ab.chunk_attention(b.q, b.cache, *b.plan, longest=new, return_lse=True)
    joint = torch.stack((b.keys, b.values), 1)
    out = torch.empty(4, 2 * new, 128, dtype=BF, device="cuda").transpose(0, 1)
    got, lse = ab.chunk_attention(b.q, ab.KVCache(joint[:, 0], joint[:, 1]), *b.plan, longest=new, return_lse=True, out=out)
    assert got is out and torch.equal(got, want) and torch.equal(lse, want_lse)
    one = b.q[:, :1].expand(-1, 4, -1)
    assert torch.equal(ab.chunk_attention(one, b.cache, *b.plan, longest=new),
                       ab.chunk_attention(one.contiguous(), b.cache, *b.plan, longest=new))


@pytest.mark.parametrize("heads,kv,tokens,keys", [(256, 1, 3, 300), (96, 1, 9, 200), (34, 2, 40, 333), (130, 1, 1, 50)])
def test_wide_groups(heads, kv, tokens, keys):
    """Many query heads on one key head, in groups that do and do not divide a tile of rows."""
    g = gen(heads)
    q, k, v = normal(g, 1, heads, tokens, 128), normal(g, 1, kv, keys, 128), normal(g, 1, kv, keys, 128)
    o, lse = ab.window_attention(q, k, v, window=100, sinks=2, return_lse=True)
    hold(o[0].transpose(0, 1), lse[0].T, *(x[0].transpose(0, 1) for x in (q, k, v)), window=100, sinks=2)


def test_many_sequences():
    """More sequences than a grid's second and third dim hold."""
    g, n = gen(15), 70001
    q, k, v = normal(g, n, 1, 1, 128), normal(g, n, 1, 3, 128), normal(g, n, 1, 3, 128)
    o = ab.window_attention(q, k, v)
    s = (q.float() @ k.float().transpose(-1, -2) * 128 ** -0.5).softmax(-1)
    ref, a = s @ v.float(), s @ v.float().abs()
    assert ((o.float() - ref).abs() <= (2 ** -8 * 1.01 + 5e-4) * a + 2 ** -8 * 1.01 * ref.abs()).all()


def test_cache_past_32_bits():
    """Pages whose elements lie past 2^31: stored and read where they belong."""
    pages, kv, page, n = 132000, 1, 128, 300
    keys = torch.empty(pages, kv, page, 128, dtype=BF, device="cuda")
    values = torch.empty_like(keys)
    assert keys.numel() > 2 ** 31
    g = gen(16)
    table = torch.tensor([[pages - 1, 5, pages - 3]], dtype=torch.int32, device="cuda")
    starts, lengths = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, n], [n]))
    k, v, q = normal(g, n, kv, 128), normal(g, n, kv, 128), normal(g, n, 2, 128)
    cache = ab.KVCache(keys, values)
    ab.append_kv(cache, k, v, table, starts, lengths)
    assert torch.equal(keys[pages - 1, 0], k[:128, 0]) and torch.equal(values[pages - 3, 0, :44], v[256:, 0])
    o, lse = ab.chunk_attention(q, cache, table, starts, lengths, return_lse=True)
    hold(o, lse, q, k, v)
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    o, lse = ab.chunk_attention(q[-1:], cache, table, one, lengths, longest=1, return_lse=True)
    hold(o, lse, q[-1:], k, v)


def test_two_streams_at_once():
    """Calls that overlap on the GPU have workspaces of their own."""
    batches = [Batch(20 + i, [(1, 6000), (1, 900), (200, 700)], 4, 2, 16, BF) for i in range(2)]
    want = [ab.chunk_attention(b.q, b.cache, *b.plan) for b in batches]
    few = [ab.chunk_attention(b.q[:2], b.cache, b.table[:2], b.starts[:3], b.lengths[:2], longest=1) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (b, stream) in enumerate(zip(batches, streams)):
            with torch.cuda.stream(stream):
                got[i].append((ab.chunk_attention(b.q, b.cache, *b.plan),
                               ab.chunk_attention(b.q[:2], b.cache, b.table[:2], b.starts[:3], b.lengths[:2], longest=1)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) and torch.equal(y, few[i]) for x, y in got[i])


def test_first_call_of_a_process_in_a_capture():
    """A process whose first calls are captured (nothing warmed up) replays them."""
    import subprocess
    import sys

    code = """
import torch, ab_attention_b200 as ab
x = torch.randn(1, 2, 300, 128, device="cuda").bfloat16(); y = x[:, :, :1].contiguous(); p = torch.zeros(300, 3, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    outs = ab.window_attention(x, x, x), ab.window_attention(y, x, x), ab.apply_rotary(x, x, p)[0]
x.normal_(); y.copy_(x[:, :, -1:]); p.fill_(7)
g.replay()
want = ab.window_attention(x, x, x), ab.window_attention(y, x, x), ab.apply_rotary(x, x, p)[0]
assert all(torch.equal(a, b) for a, b in zip(outs, want))
print("replayed")
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert "replayed" in run.stdout, run.stderr[-2000:]


def test_inference_mode():
    b = Batch(17, [(2, 50)], 2, 2, 16, BF)
    want = ab.chunk_attention(b.q, b.cache, *b.plan)
    with torch.inference_mode():
        cache = ab.KVCache(b.keys.clone(), b.values.clone())
        assert torch.equal(ab.chunk_attention(b.q.clone(), cache, *b.plan), want)
        assert ab.append_kv(cache, b.k[0][:2], b.v[0][:2], *b.plan) is None


def test_chunk_attention_of_nothing():
    b = Batch(7, [(0, 30), (0, 0)], 4, 2, 16, BF)
    assert ab.chunk_attention(b.q, b.cache, *b.plan).shape == (0, 4, 128)
    b = Batch(7, [(0, 30), (0, 0)], 4, 2, 16, BF, behind=5)
    out = torch.full_like(b.q, 3)
    ab.chunk_attention(b.q, b.cache, *b.plan, longest=1, out=out)
    assert (out == 3).all()


# ---- append ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("sizes,heads,kv,page,axes", [
    ([(1, 1)], 2, 1, 16, "video"), ([(1, 40), (1, 1), (0, 9), (1, 64)], 8, 2, 32, "line"), ([(700, 900), (3, 3), (0, 0)], 6, 6, 64, "wide"),
    ([(130, 1000)], 5, 5, 384, "text"), ([(1, 30)] * 70, 4, 4, 16, "four"),
])
@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("turned", [True, False])
def test_append(sizes, heads, kv, page, axes, dtype, turned):
    axes = AXES[axes]
    b = Batch(page, sizes, heads, kv, page, dtype, behind=2, token_major=turned)
    g, tokens = gen(4), b.q.shape[0]
    # keys and values are parts of one joint projection: strided rows
    joint = normal(g, tokens, 2 * kv, 128, dtype=dtype)
    k, v = joint[:, :kv], joint[:, kv:]
    p = torch.randint(0, 5000, (tokens, len(axes.sections)), generator=g, device="cuda", dtype=torch.int32)
    before = b.keys.clone(), b.values.clone()
    q = ab.append_kv(b.cache, k, v, *b.plan, positions=p if turned else None, axes=axes, q=b.q if turned else None)
    if turned:
        hold_turn(q.transpose(0, 1), b.q.transpose(0, 1), p, axes)
    else:
        assert q is None
    at = 0
    for s, (m, n) in enumerate(sizes):
        for i in range(m):
            where, row = b.table[s, (n - m + i) // page].item(), (n - m + i) % page
            if turned:
                hold_turn(b.keys[where, :, row], k[at + i], p[at + i], axes)
            else:
                assert torch.equal(b.keys[where, :, row], k[at + i])
            assert torch.equal(b.values[where, :, row], v[at + i])
            before[0][where, :, row], before[1][where, :, row] = b.keys[where, :, row], b.values[where, :, row]
        at += m
    for got, want in zip((b.keys, b.values), before):  # nothing else is touched, NaN included
        assert torch.equal(got.contiguous().view(torch.int16), want.contiguous().view(torch.int16))


def test_append_reports_tokens_without_a_place():
    b = Batch(8, [(4, 20), (3, 3)], 2, 2, 16, BF)
    g = gen(1)
    k, v = normal(g, 7, 2, 128), normal(g, 7, 2, 128)
    spoiled = []
    for entry, lengths in ((-1, b.lengths), (b.keys.shape[0], b.lengths), (None, b.lengths + 1000), (None, b.lengths * 0)):
        table = b.table.clone()
        if entry is not None:
            table[0, 1] = entry
        before = b.keys.clone()
        ab.append_kv(b.cache, k, v, table, b.starts, lengths)
        spoiled.append(reported())
        if entry is None:
            assert torch.equal(before.view(torch.int16), b.keys.view(torch.int16))
        else:  # the other sequence's tokens are stored
            assert torch.equal(b.keys[b.table[1, 0].item(), :, :3].transpose(0, 1), k[4:])
    assert spoiled == [1, 1, 1, 1]


def test_no_gradients():
    """As everywhere in the package: results do not require grad, whatever the inputs do."""
    g = gen(12)
    q = normal(g, 1, 2, 5, 128).requires_grad_()
    p = torch.zeros(5, 3, dtype=torch.int32, device="cuda")
    assert not ab.apply_rotary(q, q, p)[0].requires_grad
    assert not ab.window_attention(q, q, q).requires_grad
    b = Batch(13, [(3, 20)], 2, 2, 16, BF)
    k = normal(g, 3, 2, 128).requires_grad_()
    turned = ab.append_kv(b.cache, k, k, *b.plan, positions=p[:3], q=b.q.requires_grad_())
    assert not turned.requires_grad and not b.keys.requires_grad
    assert not ab.chunk_attention(b.q, b.cache, *b.plan).requires_grad


# ---- streams, graphs, and a run of them together ---------------------------------------------------------------


def test_side_stream():
    b = Batch(9, [(1, 3000), (1, 50)], 8, 2, 16, BF)
    want = ab.chunk_attention(b.q, b.cache, *b.plan, longest=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        b.q.mul_(0.5)
        half = ab.chunk_attention(b.q, b.cache, *b.plan, longest=1)
    torch.cuda.current_stream().wait_stream(side)
    b.q.mul_(2)
    assert not torch.equal(half, want)
    assert torch.equal(ab.chunk_attention(b.q, b.cache, *b.plan, longest=1), want)


@pytest.mark.parametrize("new", [1, 150])
def test_graphs_replay_with_new_contents(new):
    """Two captured graphs (each with its own workspace) replayed in turn, with lengths and tables that
    change between replays, give what eager calls give."""
    b = Batch(10, [(new, 2500), (new, 600)], 4, 2, 16, BF)
    g = gen(2)
    k, v = normal(g, 2 * new, 2, 128), normal(g, 2 * new, 2, 128)
    p = torch.arange(2 * new, dtype=torch.int32, device="cuda")[:, None].contiguous()
    axes = AXES["line"]

    def step(window):
        q = ab.append_kv(b.cache, k, v, *b.plan, positions=p, axes=axes, q=b.q)
        return ab.chunk_attention(q, b.cache, *b.plan, longest=new, window=window, sinks=3, return_lse=True)

    step(None), step(70)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for window in (None, 70):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(window))
    for turn in range(3):
        b.q.normal_(generator=g)
        k.normal_(generator=g)
        b.lengths.sub_(turn)
        for graph in graphs:
            graph.replay()
        got = [tuple(x.clone() for x in out) for out in outs]
        for window, out in zip((None, 70), got):
            for x, y in zip(out, step(window)):
                assert torch.equal(x, y)


def test_frames_of_a_stream_equal_one_pass():
    """Frames appended and attended chunk by chunk give what one block-causal pass over all of them
    gives: the same weights in another order of sums, so both are within the definition's tolerance."""
    g, axes = gen(11), AXES["video"]
    frames, h, w, heads, kv, page = 4, 9, 15, 4, 2, 64
    block, n = h * w, 4 * h * w
    q, k, v = normal(g, n, heads, 128), normal(g, n, kv, 128), normal(g, n, kv, 128)
    cache = ab.kv_cache(20, kv, page_size=page)
    table = torch.randperm(20, generator=g, device="cuda")[None, :16].to(torch.int32).contiguous()
    starts = torch.tensor([0, block], dtype=torch.int32, device="cuda")
    outs = []
    for f in range(frames):
        rows = slice(f * block, (f + 1) * block)
        lengths = torch.tensor([(f + 1) * block], dtype=torch.int32, device="cuda")
        p = ab.grid_positions(1, h, w, first_frame=f, device="cuda")
        turned = ab.append_kv(cache, k[rows], v[rows], table, starts, lengths, positions=p, axes=axes, q=q[rows])
        outs.append(ab.chunk_attention(turned, cache, table, starts, lengths, longest=block, window=2 * block, sinks=10, block=block))
    p = ab.grid_positions(frames, h, w, device="cuda")
    tq, tk = ab.apply_rotary(q.transpose(0, 1)[None], k.transpose(0, 1)[None], p, axes)
    whole, lse = ab.window_attention(tq, tk, v.transpose(0, 1)[None], window=2 * block, sinks=10, block=block, return_lse=True)
    rows = [x[0].transpose(0, 1) for x in (tq, tk)]
    hold(whole[0].transpose(0, 1), lse[0].T, *rows, v, window=2 * block, sinks=10, block=block)
    hold(torch.cat(outs), None, *rows, v, window=2 * block, sinks=10, block=block)
    assert torch.equal(stream.rows_of(cache.keys, table[0], n), rows[1])


@pytest.mark.parametrize("batch,heads,kv,chunk,window,sinks,page,frames", [
    (1, 4, 4, 1, None, 0, 16, 5), (2, 6, 2, 2, 4, 1, 32, 12), (1, 2, 1, 1, 2, 2, 64, 9), (1, 3, 3, 3, 3, 0, 128, 9),
])
def test_stream_attention(batch, heads, kv, chunk, window, sinks, page, frames):
    """Chunk after chunk, two layers, two denoising steps each, pages used again behind the window: the last
    step's outputs are those of one pass over the whole video."""
    h, w, layers = 6, 11, 2
    frame, g = h * w, gen(frames)
    s = ab.StreamAttention(heads, h, w, kv_heads=kv, chunk_frames=chunk, window_frames=window, sink_frames=sinks, batch=batch,
                           max_frames=frames, page_size=page)
    q, k, v = (normal(g, layers, batch, x, frames * frame, 128) for x in (heads, kv, kv))
    with pytest.raises(ValueError, match="q must be"):
        s(0, q[0], k[0], v[0])
    for turn in range(2):  # a second video after reset()
        outs = [[] for _ in range(layers)]
        for f in range(0, frames, chunk):
            rows = slice(f * frame, (f + chunk) * frame)
            for layer in range(layers):
                s(layer, q[layer, :, :, rows] * 0.5, k[layer, :, :, rows] * 2, v[layer, :, :, rows] - 1)  # a noisier step
                outs[layer].append(s(layer, *(x[layer, :, :, rows] for x in (q, k, v))))
            if f + chunk < frames:
                s.advance()
        with pytest.raises(ValueError, match="holds"):
            s.advance()
        s.reset()
        p = ab.grid_positions(frames, h, w, device="cuda")
        for layer in range(layers):
            tq, tk = ab.apply_rotary(q[layer], k[layer], p)
            got = torch.cat(outs[layer], 2)
            for b in range(batch):
                hold(got[b].transpose(0, 1), None, tq[b].transpose(0, 1), tk[b].transpose(0, 1), v[layer, b].transpose(0, 1),
                     window=None if window is None else window * frame, sinks=sinks * frame, block=chunk * frame)
    if window is not None:
        assert s.caches[0].keys.shape[0] <= batch * (-(-(window + chunk + sinks) * frame // page) + 3)


def test_stream_attention_in_a_graph():
    """A captured step serves chunk after chunk: advance() moves its counters on."""
    g = gen(3)
    s = ab.StreamAttention(2, 5, 9, max_frames=6, window_frames=3)
    q, k, v = (normal(g, 1, 2, 45, 128) for _ in range(3))
    want = []
    for f in range(6):
        q.copy_(normal(gen(f), 1, 2, 45, 128)), k.copy_(normal(gen(f + 50), 1, 2, 45, 128))
        want.append(s(0, q, k, v).clone())
        if f < 5:
            s.advance()
    s.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s(0, q, k, v)
    for f in range(6):
        q.copy_(normal(gen(f), 1, 2, 45, 128)), k.copy_(normal(gen(f + 50), 1, 2, 45, 128))
        graph.replay()
        assert torch.equal(out, want[f])
        if f < 5:
            s.advance()
