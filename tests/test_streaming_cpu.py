"""Streaming operators without a GPU: shapes and refusals (Meta kernels run the CUDA kernels'
argument checks), the C ABI's validation, and known answers of the float64 restatement."""
import ctypes

import pytest
import torch

import ab_attention_b200 as ab
from ab_attention_b200 import _lib
from oracle import stream

BF = torch.bfloat16


def meta(*shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="meta")


def ints(*shape):
    return meta(*shape, dtype=torch.int32)


def batch(seqs=3, width=5):
    return ints(seqs, width), ints(seqs + 1), ints(seqs)


def test_shapes_and_types_of_results():
    q, k = ab.apply_rotary(meta(2, 6, 10, 128), meta(2, 3, 10, 128), ints(10, 3))
    assert q.shape == (2, 6, 10, 128) and k.shape == (2, 3, 10, 128) and q.dtype == BF
    q, k = ab.apply_rotary(meta(2, 10, 6, 128, dtype=torch.float32).transpose(1, 2), None, ints(2, 10, 1),
                           ab.RotaryAxes((128,)))
    assert q.shape == (2, 6, 10, 128) and q.is_contiguous() and k is None
    out, lse = ab.window_attention(meta(2, 6, 7, 128), meta(2, 2, 90, 128), meta(2, 2, 90, 128), window=5, return_lse=True)
    assert out.shape == (2, 6, 7, 128) and lse.shape == (2, 6, 7) and lse.dtype == torch.float32
    cache = ab.KVCache(meta(9, 2, 16, 128), meta(9, 2, 16, 128))
    out, lse = ab.chunk_attention(meta(11, 4, 128), cache, *batch(), return_lse=True)
    assert out.shape == (11, 4, 128) and lse.shape == (11, 4)
    assert ab.append_kv(cache, meta(11, 2, 128), meta(11, 2, 128), *batch()) is None
    q = ab.append_kv(cache, meta(11, 2, 128), meta(11, 2, 128), *batch(), positions=ints(11, 3), q=meta(11, 4, 128))
    assert q.shape == (11, 4, 128)


def test_grid_positions_are_row_major():
    p = ab.grid_positions(2, 3, 4, first_frame=5)
    assert p.shape == (24, 3) and p.dtype == torch.int32
    assert p[0].tolist() == [5, 0, 0] and p[1].tolist() == [5, 0, 1] and p[4].tolist() == [5, 1, 0] and p[-1].tolist() == [6, 2, 3]


@pytest.mark.parametrize("message,call", [
    ("q must be \\[B,H,N,128\\]", lambda: ab.apply_rotary(meta(2, 6, 10, 64), None, ints(10, 3))),
    ("q must be bfloat16, float16 or float32", lambda: ab.apply_rotary(meta(2, 6, 10, 128, dtype=torch.float64), None, ints(10, 3))),
    ("k must be \\[B,Hk,N,128\\]", lambda: ab.apply_rotary(meta(2, 6, 10, 128), meta(2, 6, 9, 128), ints(10, 3))),
    ("k must be BFloat16", lambda: ab.apply_rotary(meta(2, 6, 10, 128), meta(2, 6, 10, 128, dtype=torch.half), ints(10, 3))),
    ("positions must be int32", lambda: ab.apply_rotary(meta(2, 6, 10, 128), None, ints(9, 3))),
    ("positions must be int32", lambda: ab.apply_rotary(meta(2, 6, 10, 128), None, ints(10, 2))),
    ("positions must be Int", lambda: ab.apply_rotary(meta(2, 6, 10, 128), None, meta(10, 3, dtype=torch.int64))),
    ("sum to 128", lambda: ab.apply_rotary(meta(2, 6, 10, 128), None, ints(10, 2), ab.RotaryAxes((64, 32)))),
    ("even", lambda: ab.apply_rotary(meta(2, 6, 10, 128), None, ints(10, 2), ab.RotaryAxes((63, 65)))),
    ("1 to 4 axes", lambda: ab.apply_rotary(meta(2, 6, 10, 128), None, ints(10, 5), ab.RotaryAxes((28, 28, 28, 28, 16)))),
    ("theta", lambda: ab.apply_rotary(meta(2, 6, 10, 128), None, ints(10, 1), ab.RotaryAxes((128,), theta=0.0))),
    ("q must be bfloat16 or float16", lambda: ab.window_attention(*[meta(1, 2, 8, 128, dtype=torch.float32)] * 3)),
    ("Hk dividing", lambda: ab.window_attention(meta(1, 5, 8, 128), meta(1, 2, 8, 128), meta(1, 2, 8, 128))),
    ("v must have k's shape", lambda: ab.window_attention(meta(1, 4, 8, 128), meta(1, 2, 8, 128), meta(1, 2, 9, 128))),
    ("window must be positive", lambda: ab.window_attention(*[meta(1, 2, 8, 128)] * 3, window=0)),
    ("sinks must not be negative", lambda: ab.window_attention(*[meta(1, 2, 8, 128)] * 3, window=3, sinks=-1)),
    ("block must be positive", lambda: ab.window_attention(*[meta(1, 2, 8, 128)] * 3, block=0)),
])
def test_refusals(message, call):
    with pytest.raises(ValueError, match=message):
        call()


@pytest.mark.parametrize("message,change", [
    ("page size must be", {"cache": (9, 2, 24)}),
    ("page size must be", {"cache": (9, 2, 8)}),
    ("page size must be", {"cache": (9, 2, 192)}),
    ("must have pages", {"cache": (0, 2, 16)}),
    ("heads a multiple of 2", {"q": meta(11, 5, 128)}),
    ("q must be BFloat16", {"q": meta(11, 4, 128, dtype=torch.half)}),
    ("page_table must be contiguous int32", {"page_table": ints(15)}),
    ("page_table must be Int", {"page_table": meta(3, 5, dtype=torch.int64)}),
    ("starts must be int32 \\[4\\]", {"starts": ints(3)}),
    ("lengths must be int32 \\[3\\]", {"lengths": ints(4)}),
    ("longest must be positive", {"longest": 0}),
    ("window must be positive", {"window": -2}),
    ("block must be positive", {"block": 0}),
    ("out must have q's shape", {"out": meta(11, 2, 128)}),
    ("out must have contiguous 16-byte aligned rows", {"out": meta(11, 128, 4).transpose(1, 2)}),
])
def test_chunk_refusals(message, change):
    args = dict(zip(("page_table", "starts", "lengths"), batch()), q=meta(11, 4, 128), cache=(9, 2, 16))
    args.update(change)
    shape = args.pop("cache")
    cache = ab.KVCache(meta(*shape, 128), meta(*shape, 128))
    with pytest.raises(ValueError, match=message):
        ab.chunk_attention(args.pop("q"), cache, args.pop("page_table"), args.pop("starts"), args.pop("lengths"), **args)


@pytest.mark.parametrize("message,change", [
    ("k must be \\[tokens, 2, 128\\]", {"k": meta(11, 3, 128)}),
    ("v must be \\[tokens, 2, 128\\]", {"v": meta(10, 2, 128)}),
    ("v must be BFloat16", {"v": meta(11, 2, 128, dtype=torch.half)}),
    ("give both", {"q": meta(11, 4, 128)}),
    ("positions must be int32", {"positions": ints(10, 3)}),
    ("q must be \\[tokens, heads, 128\\]", {"q": meta(12, 4, 128), "positions": ints(11, 3)}),
    ("cache values must have", {"values": meta(9, 2, 32, 128)}),
    ("cache keys must be bfloat16 or float16", {"keys": meta(9, 2, 16, 128, dtype=torch.float32)}),
])
def test_append_refusals(message, change):
    args = dict(k=meta(11, 2, 128), v=meta(11, 2, 128), keys=meta(9, 2, 16, 128), values=meta(9, 2, 16, 128))
    args.update(change)
    cache = ab.KVCache(args.pop("keys"), args.pop("values"))
    with pytest.raises(ValueError, match=message):
        ab.append_kv(cache, args.pop("k"), args.pop("v"), *batch(), **args)


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 8, 128, dtype=BF)
    t = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    cache = ab.kv_cache(2, 2, page_size=16, device="cpu")
    for call in (lambda: ab.window_attention(x, x, x), lambda: ab.apply_rotary(x, None, torch.zeros(8, 3, dtype=torch.int32)),
                 lambda: ab.chunk_attention(x[0], cache, *t), lambda: ab.append_kv(cache, x[0], x[0], *t)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


class RotaryArgs(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("axes", ctypes.c_int32), ("sections", ctypes.c_int32 * 4), ("theta", ctypes.c_double),
                ("shared", ctypes.c_int32), ("halves", ctypes.c_int32), ("inverse", ctypes.c_int32), ("positions", ctypes.c_void_p),
                ("positions_batch", ctypes.c_int64), ("batch", ctypes.c_int64), ("tokens", ctypes.c_int64),
                *[(n, ctypes.c_void_p) for n in ("q", "k", "v", "q_out", "k_out", "v_out")],
                ("heads", ctypes.c_int64), ("kv_heads", ctypes.c_int64),
                *[(n, ctypes.c_int64 * 3) for n in ("q_stride", "k_stride", "v_stride", "q_out_stride", "k_out_stride", "v_out_stride")],
                *[(n, ctypes.c_void_p) for n in ("starts", "lengths", "page_table")],
                *[(n, ctypes.c_int64) for n in ("sequences", "table_width", "page_size", "pages")]]


class ChunkArgs(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), *[(n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "lse")],
                *[(n, ctypes.c_int64 * 3) for n in ("q_stride", "k_stride", "v_stride", "o_stride", "lse_stride")],
                *[(n, ctypes.c_int64) for n in ("sequences", "tokens", "longest", "keys", "heads", "kv_heads")],
                *[(n, ctypes.c_void_p) for n in ("starts", "lengths", "page_table")],
                *[(n, ctypes.c_int64) for n in ("table_width", "page_size", "pages", "window", "sinks", "block")]]


def rotary_args(**change):
    rows = (ctypes.c_int64 * 3)(128 * 8 * 2, 128 * 8, 128)
    a = RotaryArgs(dtype=0, axes=3, sections=(44, 42, 42, 0), theta=1e4, positions=64, batch=1, tokens=8, q=64, q_out=64, heads=2,
                   q_stride=rows, q_out_stride=rows)
    for name, value in change.items():
        setattr(a, name, value)
    return a


def chunk_args(**change):
    rows = (ctypes.c_int64 * 3)(128 * 8 * 2, 128 * 8, 128)
    a = ChunkArgs(dtype=0, q=64, k=64, v=64, o=64, q_stride=rows, k_stride=rows, v_stride=rows, o_stride=rows, sequences=1, tokens=8,
                  longest=8, keys=8, heads=2, kv_heads=2, block=1)
    for name, value in change.items():
        setattr(a, name, value)
    return a


odd = (ctypes.c_int64 * 3)(128 * 8 * 2, 128 * 8, 132)
paged = dict(page_table=64, starts=64, lengths=64, table_width=2, page_size=16, pages=4)


@pytest.mark.parametrize("change", [
    {"dtype": 3}, {"tokens": 0}, {"q": 66}, {"q_out": None}, {"q_stride": odd}, {"axes": 0}, {"axes": 5}, {"theta": -1.0},
    {"sections": (44, 42, 40, 0)}, {"sections": (45, 41, 42, 0)}, {"positions": None}, {"heads": 0}, {"q": None},
    {"page_table": 64}, {**paged, "k": 64, "v": 64, "k_out": 64, "v_out": 64, "kv_heads": 2, "page_size": 20},
    {**paged, "k": 64, "v": 64, "k_out": 64, "v_out": 64, "kv_heads": 2, "starts": None},
    {**paged, "k": 64, "v": 64, "k_out": 64, "v_out": 64, "kv_heads": 2, "batch": 2},
    {**paged, "k": 64, "v": None, "k_out": 64, "v_out": 64, "kv_heads": 2},
])
def test_rotary_entry_validates_before_launch(change):
    lib = _lib.load()
    assert lib.abx_rotary(ctypes.byref(rotary_args(**change)), None) == 1
    assert lib.abx_last_error()


@pytest.mark.parametrize("change,status", [
    ({"dtype": 2}, 1), ({"tokens": 0}, 1), ({"heads": 3}, 1), ({"kv_heads": 0}, 1), ({"longest": 9}, 1), ({"longest": 4}, 1),
    ({"window": -1}, 1), ({"sinks": -1}, 1), ({"block": 0}, 1), ({"q": 66}, 1), ({"o": None}, 1), ({"k_stride": odd}, 1),
    ({"keys": 0}, 1), ({"keys": 1 << 31}, 2), ({"tokens": 1 << 30, "longest": 1 << 30}, 2),
    ({**paged, "page_size": 48}, 1), ({**paged, "starts": None}, 1), ({**paged, "pages": 0}, 1), ({**paged, "table_width": 1 << 29}, 2),
])
def test_chunk_entry_validates_before_launch(change, status):
    lib = _lib.load()
    size = ctypes.c_size_t(7)
    assert lib.abx_chunk_workspace_size(ctypes.byref(chunk_args(**change)), ctypes.byref(size)) == status
    assert lib.abx_chunk_attention(ctypes.byref(chunk_args(**change)), None, 0, None) == status
    assert lib.abx_last_error()


def test_chunk_workspace():
    """Few rows against many keys are split over CTAs and need a workspace; a short call needs none, and
    a missing or short workspace is refused."""
    lib = _lib.load()
    size = ctypes.c_size_t(7)
    assert lib.abx_chunk_workspace_size(ctypes.byref(chunk_args()), ctypes.byref(size)) == 0 and size.value == 0
    long = chunk_args(tokens=1, longest=1, keys=100000)
    assert lib.abx_chunk_workspace_size(ctypes.byref(long), ctypes.byref(size)) == 0 and size.value > 0
    assert lib.abx_chunk_attention(ctypes.byref(long), None, 0, None) == 3
    assert lib.abx_chunk_attention(ctypes.byref(long), ctypes.c_void_p(256), size.value - 1, None) == 3
    assert lib.abx_chunk_attention(ctypes.byref(long), ctypes.c_void_p(264), size.value, None) == 3
    assert lib.abx_chunk_workspace_size(None, ctypes.byref(size)) == 1
    assert lib.abx_chunk_workspace_size(ctypes.byref(long), None) == 1


# ---- the float64 restatement against known answers ------------------------------------------------------


def test_restated_rule():
    causal = stream.sees(0, 5, 5, None, 0, 1)
    assert torch.equal(causal, torch.ones(5, 5).tril().bool())
    framed = stream.sees(0, 6, 6, None, 0, 3)
    assert framed.sum(1).tolist() == [3, 3, 3, 6, 6, 6]
    rolled = stream.sees(4, 4, 8, 2, 1, 1)
    assert rolled[0].nonzero()[:, 0].tolist() == [0, 3, 4] and rolled[3].nonzero()[:, 0].tolist() == [0, 6, 7]
    assert not stream.sees(-2, 2, 8, None, 0, 4).any()  # positions before the first key see nothing


def test_restated_turn():
    x = torch.randn(4, 128, dtype=torch.float64)
    p = torch.tensor([[0, 0, 0], [1, 2, 3], [100, 7, 9], [5, 5, 5]])
    for paired in (True, False):
        y = stream.turn(x, p, (44, 42, 42), 1e4, paired)
        assert torch.allclose(y[0], x[0]) and torch.allclose(y.norm(dim=-1), x.norm(dim=-1))
        assert torch.allclose(stream.turn(y, p, (44, 42, 42), 1e4, paired, inverse=True), x)
    # only relative positions matter to a product of two turned rows
    a, b = x[:1], x[1:2]
    dot = [(stream.turn(a, torch.tensor([[s + 3]]), (128,), 1e4) * stream.turn(b, torch.tensor([[s]]), (128,), 1e4)).sum()
           for s in (0, 50)]
    assert torch.allclose(dot[0], dot[1])


def test_restated_turn_back_is_the_gradient():
    x = torch.randn(3, 128, dtype=torch.float64, requires_grad=True)
    p = torch.tensor([[4, 2], [9, 1], [0, 77]])
    g = torch.randn(3, 128, dtype=torch.float64)

    def f(y):
        c = stream.turn(torch.eye(128, dtype=torch.float64), p[:1], (64, 64), 50.0)
        return y[0] @ c
    grad = torch.autograd.grad((f(x) * g[0]).sum(), x)[0][0]
    back = stream.turn(g[:1], p[:1], (64, 64), 50.0, inverse=True)[0]
    assert torch.allclose(grad, back)


def test_stream_attention_places():
    """Logical pages of a stream take distinct places while any of them is in the window."""
    s = ab.StreamAttention(2, 6, 11, kv_heads=1, chunk_frames=2, window_frames=4, sink_frames=1, batch=2, max_frames=40,
                           page_size=16, device="cpu")
    frame, table = 66, s.page_table
    assert table.shape == (2, -(-40 * 66 // 16)) and not set(table[0].tolist()) & set(table[1].tolist())
    for f in range(0, 40, 2):
        end = (f + 2) * frame
        keys = list(range(frame)) + list(range(max(0, end - 4 * frame), end))
        pages = sorted({x // 16 for x in keys})
        assert len({table[0, x].item() for x in pages}) == len(pages)
    for bad in (dict(window_frames=1), dict(sink_frames=-1), dict(max_frames=1), dict(batch=0)):
        with pytest.raises(ValueError):
            ab.StreamAttention(2, 6, 11, **{**dict(chunk_frames=2, max_frames=8, device="cpu"), **bad})
