"""Denoising schedule with per-layer sample-plan reuse (ab_attention/video.py:53-87).

The paper schedule keeps the first 10 steps and layer 0 dense; every other layer
builds a fresh plan on steps 11, 15, ..., 47 (an "anchor" every 4 steps) and
reuses it on the steps in between. `VideoAttention` keeps the reference's API
(`reset`, `step_end` as Diffusers' `callback_on_step_end`, `is_sparse`,
`attend`), anchors and seeds, so its plans are bit-identical to the reference's.
A B200 holds the plans in device memory (the reference parks them in pinned
host RAM to fit a single 80 GB GPU): a Wan2.1-14B layer's plan is 0.39 GB.
"""
from __future__ import annotations

import torch

from .attention import SamplePlan, apply_plan, build_plan, dense_attention, dense_cross_attention
from .cache import append_kv, chunk_attention, kv_cache
from .rotary import VIDEO_AXES, grid_positions


def plan_seed(layer: int, anchor: int) -> int:
    """Seed of the plan a layer builds at an anchor step (ab_attention/video.py:79)."""
    return 42 + layer * 1_000_003 + anchor * 97


def anchor_step(step: int) -> int:
    """The refresh step a sparse step reuses the plan of (ab_attention/video.py:77)."""
    return 11 + (step - 11) // 4 * 4


class VideoAttention:
    """One pipeline's denoising schedule and per-layer sample plans.

    Call ``reset()`` before each video and pass ``step_end`` as Diffusers'
    ``callback_on_step_end``. Wan's two sequential CFG calls share one plan.
    ``host_plans=True`` keeps stored plans in pinned host memory as the
    reference does (for callers short of device memory).
    """

    def __init__(self, sample_pages, *, dense=False, host_plans=False):
        self.sample_pages = sample_pages
        self.dense = dense
        self.host_plans = host_plans
        self.reset()

    def reset(self):
        self.step = 1
        self.plans = {}

    def step_end(self, pipe, index, timestep, callback_kwargs):
        self.step = index + 2  # Diffusers indices are zero-based.
        return callback_kwargs

    def is_sparse(self, layer):
        return not self.dense and self.step > 10 and layer > 0

    def _store(self, plan: SamplePlan, previous: SamplePlan | None) -> SamplePlan:
        if not self.host_plans:
            return plan
        if previous is None:
            previous = SamplePlan(*(torch.empty(t.shape, dtype=t.dtype, pin_memory=True) for t in plan))
        for storage, tensor in zip(previous, plan):
            storage.copy_(tensor)
        return previous

    def attend(self, layer, q, k, v, *, return_lse=False, text_kv=None):
        """Sparse attention of one layer at the current step, building the plan
        on an anchor step and reusing it otherwise."""
        anchor = anchor_step(self.step)
        stored_anchor, stored = self.plans.get(layer, (None, None))
        if stored_anchor != anchor:
            plan = build_plan(q, k, sample_pages=self.sample_pages, seed=plan_seed(layer, anchor))
            self.plans[layer] = (anchor, self._store(plan, stored))
        else:
            plan = SamplePlan(*(t.to(q.device, non_blocking=True) for t in stored))
        return apply_plan(q, k, v, plan, return_lse=return_lse, text_kv=text_kv)

    def __call__(self, layer, q, k, v, *, return_lse=False, text_kv=None):
        """Dense on the steps and layer the schedule keeps dense, else `attend`."""
        if self.is_sparse(layer):
            return self.attend(layer, q, k, v, return_lse=return_lse, text_kv=text_kv)
        if text_kv is not None:
            raise ValueError("text keys are only supported on sparse steps")
        return dense_attention(q, k, v, return_lse=return_lse)


def hunyuan_attention(schedule, layer, q, k, v, video_tokens, prompt_tokens):
    """One HunyuanVideo attention layer over [video | prompt | padding] tokens
    (ab_attention/video.py:129-151).

    On sparse steps the video queries attend to the layer's sampled video keys
    plus every prompt key with weight pi = 1 (the reference merges a sparse
    video state with an exact video->text state by LSE; that is the same
    softmax over the union, here one kernel), and the prompt queries attend
    exactly to every video and prompt key. On dense steps the video and prompt
    tokens attend exactly to each other. Padding tokens always form their own
    exact partition. q, k, v: [B, H, N, 128] bf16.
    """
    prompt_end = video_tokens + prompt_tokens
    sl = lambda x, a, b: x[:, :, a:b].contiguous()  # noqa: E731
    text_kv = (sl(k, video_tokens, prompt_end), sl(v, video_tokens, prompt_end)) if prompt_tokens else None
    video_k, video_v = sl(k, 0, video_tokens), sl(v, 0, video_tokens)
    if schedule.is_sparse(layer):
        outputs = [schedule.attend(layer, sl(q, 0, video_tokens), video_k, video_v, text_kv=text_kv)]
        if prompt_tokens:
            outputs.append(dense_cross_attention(sl(q, video_tokens, prompt_end), video_k, video_v,
                                                 extra_kv=text_kv))
    else:
        outputs = [dense_cross_attention(sl(q, 0, prompt_end), video_k, video_v, extra_kv=text_kv)]
    if prompt_end < q.shape[2]:
        outputs.append(dense_cross_attention(sl(q, prompt_end, q.shape[2]), None, None,
                                             extra_kv=(sl(k, prompt_end, q.shape[2]), sl(v, prompt_end, q.shape[2]))))
    return torch.cat(outputs, dim=2)


class StreamAttention:
    """Attention of a video that is generated chunk by chunk (no counterpart in the reference).

    A chunk is ``chunk_frames`` latent frames of ``height`` x ``width`` tokens. Its queries attend to
    the chunk itself in both directions and to the frames before it: to all of them, or to the last
    ``window_frames`` (the chunk's own counted) and the first ``sink_frames``. Keys and values
    live in a paged cache per layer, turned by their (frame, row, column) positions; with a
    window, pages behind it are used again, so the cache does not grow with the video.

    Call the object once per layer and denoising step of a chunk (each call replaces the chunk's keys and
    values), then ``advance()`` once the chunk is final. Nothing synchronises: ``advance`` updates device
    counters in place, so a captured step replays for chunk after chunk. Before a capture that has a layer's
    first call, ``allocate(layers)`` makes the caches.
    """

    def __init__(self, heads, height, width, *, max_frames, kv_heads=None, chunk_frames=1, window_frames=None, sink_frames=0,
                 batch=1, axes=VIDEO_AXES, page_size=128, dtype=torch.bfloat16, device="cuda"):
        if min(heads, height, width, chunk_frames, batch) < 1 or max_frames < chunk_frames:
            raise ValueError("heads, height, width, chunk_frames and batch must be positive, max_frames at least chunk_frames")
        if window_frames is not None and window_frames < chunk_frames:
            raise ValueError("window_frames must be at least chunk_frames: a chunk attends to itself")
        if sink_frames < 0:
            raise ValueError("sink_frames must not be negative")
        frame = height * width
        self.heads, self.kv_heads, self.batch, self.axes = heads, kv_heads or heads, batch, axes
        self.max_frames, self.chunk_frames, self.tokens = max_frames, chunk_frames, chunk_frames * frame
        self.window = None if window_frames is None else window_frames * frame
        self.sinks = sink_frames * frame
        # Logical pages of a sequence, and the places they take: the sinks' own, then a ring that holds the window,
        # the chunk and the pages cut by their ends.
        logical = -(-max_frames * frame // page_size)
        places = logical
        if self.window is not None:
            kept = -(-self.sinks // page_size)
            places = min(logical, kept + -(-(self.window + self.tokens) // page_size) + 2)
        page = torch.arange(logical, dtype=torch.int32)
        if places < logical:
            page = torch.where(page < kept, page, kept + (page - kept) % (places - kept))
        table = page + places * torch.arange(batch, dtype=torch.int32)[:, None]
        self.page_table = table.to(torch.int32).contiguous().to(device)
        self.starts = torch.arange(batch + 1, dtype=torch.int32, device=device) * self.tokens
        self.lengths = torch.empty(batch, dtype=torch.int32, device=device)
        self.positions = torch.empty(batch * self.tokens, 3, dtype=torch.int32, device=device)
        self._first = grid_positions(chunk_frames, height, width, device=device).repeat(batch, 1)
        self._cache = dict(pages=places * batch, kv_heads=self.kv_heads, page_size=page_size, dtype=dtype,
                           device=self.page_table.device)  # with its index: the caches are made later
        self.caches = {}
        self.reset()

    def reset(self):
        """The next chunk is the first."""
        self.frames = 0
        self.lengths.fill_(self.tokens)
        self.positions.copy_(self._first)

    def advance(self):
        """The current chunk is final; the next one follows it."""
        if self.frames + 2 * self.chunk_frames > self.max_frames:
            raise ValueError(f"the stream holds {self.max_frames} frames")
        self.frames += self.chunk_frames
        self.lengths.add_(self.tokens)
        self.positions[:, 0].add_(self.chunk_frames)

    def allocate(self, layers):
        """Creates the caches of these layers, where they have none. A layer's first call does it too, but not inside a
        CUDA graph capture: memory and fill would be the graph's own, and every replay would clear the chunks before."""
        missing = [layer for layer in layers if layer not in self.caches]
        if missing and self.page_table.is_cuda:
            with torch.cuda.device(self.page_table.device):
                if torch.cuda.is_current_stream_capturing():
                    raise ValueError(f"layer {missing[0]!r} has no cache yet: call allocate(layers) before the capture")
        for layer in missing:
            self.caches[layer] = kv_cache(**self._cache)

    @torch.no_grad()
    def __call__(self, layer, q, k, v):
        """q [B,H,N,128], k and v [B,Hk,N,128] of the chunk's N tokens (before rotation), any strides with
        contiguous rows; returns [B,H,N,128], a view of token-major [B,N,H,128] memory. A batch of more than one is
        copied first unless q, k and v are such views too (projections as they come, transposed)."""
        if q.shape != (self.batch, self.heads, self.tokens, 128):
            raise ValueError(f"q must be {[self.batch, self.heads, self.tokens, 128]} (got {list(q.shape)})")
        if k.shape != (self.batch, self.kv_heads, self.tokens, 128) or v.shape != k.shape:
            raise ValueError(f"k and v must be {[self.batch, self.kv_heads, self.tokens, 128]}")
        self.allocate((layer,))
        cache, where = self.caches[layer], (self.page_table, self.starts, self.lengths)
        q, k, v = (x.transpose(1, 2).flatten(0, 1) for x in (q, k, v))  # packed; a view for one batch, or of token-major memory
        q = append_kv(cache, k, v, *where, positions=self.positions, axes=self.axes, q=q)
        out = chunk_attention(q, cache, *where, longest=self.tokens, window=self.window, sinks=self.sinks, block=self.tokens)
        return out.unflatten(0, (self.batch, self.tokens)).transpose(1, 2)
