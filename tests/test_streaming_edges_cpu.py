"""Edges of the streaming operators' C ABI without a GPU: what the call refuses before a launch."""
import ctypes

import pytest

from ab_attention_b200 import _lib
from tests.test_streaming_cpu import chunk_args, paged


def strides(*of):
    return (ctypes.c_int64 * 3)(*of)


@pytest.mark.parametrize("name", ["k_stride", "v_stride"])
@pytest.mark.parametrize("change", [
    {"sequences": 2, "stride": (0, 1024, 128)}, {"stride": (2048, 0, 128)}, {"stride": (2048, 1024, 0)},
    {**paged, "stride": (0, 2048, 128)}, {**paged, "stride": (4096, 0, 128)}, {**paged, "stride": (4096, 2048, 0)},
])
def test_repeated_keys_are_refused(name, change):
    """Tensor maps describe k and v, and what a copy does at a stride of 0 is not documented."""
    lib, size, change = _lib.load(), ctypes.c_size_t(7), dict(change)
    args = chunk_args(**{name: strides(*change.pop("stride"))}, **change)
    assert lib.abx_chunk_workspace_size(ctypes.byref(args), ctypes.byref(size)) == 1
    assert lib.abx_chunk_attention(ctypes.byref(args), None, 0, None) == 1
    assert b"repeat" in lib.abx_last_error()


def test_strides_of_single_elements_do_not_count():
    lib, size = _lib.load(), ctypes.c_size_t(7)
    args = chunk_args(k_stride=strides(0, 1024, 128), v_stride=strides(0, 1024, 128), q_stride=strides(0, 0, 0))
    assert lib.abx_chunk_workspace_size(ctypes.byref(args), ctypes.byref(size)) == 0
