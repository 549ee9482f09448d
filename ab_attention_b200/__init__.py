"""B200-native AB-Attention sparse-attention hot path (IBCS + SIP + HT-weighted sparse prefill)."""
from .attention import (SamplePlan, ab_attention, apply_plan, build_plan, dense_attention,
                        dense_cross_attention, paged_attention, window_attention)
from .cache import KVCache, append_kv, chunk_attention, kv_cache
from .layout import cube_layout
from .rotary import RotaryAxes, apply_rotary, grid_positions

__all__ = ["SamplePlan", "ab_attention", "apply_plan", "build_plan", "dense_attention", "dense_cross_attention",
           "paged_attention", "cube_layout", "VideoAttention", "hunyuan_attention", "StreamAttention", "ab_attention_host",
           "window_attention", "KVCache", "kv_cache", "append_kv", "chunk_attention", "RotaryAxes", "apply_rotary",
           "grid_positions"]
from .video import StreamAttention, VideoAttention, hunyuan_attention  # noqa: E402
from .pipeline import ab_attention_host  # noqa: E402
