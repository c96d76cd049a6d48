"""Which tiles a chunk attention call takes, seen from the host: a call without
a workspace says how much it needs, and the needs of tiles of 128 and of 256
rows differ.  No call here reaches a GPU."""
import inspect
import re

import pytest

from vramancer_amd import _lib
from vramancer_amd.paged_chunk import paged_attention_chunk

BF, KV = _lib.VRM_SRC_BF16, _lib.VRM_KV_BF16


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _need(lib, N, B, H, KH, D, PS, max_pp, window=0, expected=None, q=BF, kv=KV, L=1, P=4):
    """Workspace bytes that the call asks for."""
    sc = 1 << 40 if kv == _lib.VRM_KV_I8 else None
    args = (16, q, H * D, D, 16, sc, 16, 16, 16, 16, None, None, 0, N, B, H, KH, D, PS, L, P, max_pp, 0, 0.1, 1, window)
    if expected is None:
        rc = lib.vrm_paged_chunk_attention(*args, kv, None)
    else:
        rc = lib.vrm_paged_chunk_attention_expecting(*args, expected, kv, None)
    assert rc == -3, lib.vrm_last_error()
    return int(re.search(rb"workspace of (\d+) bytes", lib.vrm_last_error())[1])


SHAPE = (64 * 32, 64, 32, 8, 128, 16)  # 64 sequences of 32 tokens: 128 rows a kv-head each


def test_window_in_a_wide_table(lib):
    """A window bounds what a tile sees, whatever the table holds."""
    small, large = _need(lib, *SHAPE, 16), _need(lib, *SHAPE, 3125)
    assert small < large
    assert _need(lib, *SHAPE, 3125, window=100) == small
    assert _need(lib, *SHAPE, 3125, window=800) == small
    assert _need(lib, *SHAPE, 3125, window=1000) == large
    assert _need(lib, *SHAPE, 3125, window=2 ** 31 - 1) == large
    assert _need(lib, *SHAPE, 16, window=4000) == small


def test_short_contexts_in_a_wide_table(lib):
    small, large = _need(lib, *SHAPE, 16), _need(lib, *SHAPE, 3125)
    assert _need(lib, *SHAPE, 3125, expected=200) == small
    assert _need(lib, *SHAPE, 3125, expected=0) == large
    assert _need(lib, *SHAPE, 3125, expected=1 << 30) == large
    assert _need(lib, *SHAPE, 16, expected=1 << 30) == small
    args = (16, BF, 4096, 128, 16, None, 16, 16, 16, 16, None, None, 0, *SHAPE, 1, 4, 64, 0, 0.1, 1, 0)
    assert lib.vrm_paged_chunk_attention_expecting(*args, -1, KV, None) == -1 and b"expected" in lib.vrm_last_error()
    assert "expected_context" in inspect.signature(paged_attention_chunk).parameters


@pytest.mark.parametrize("kv", [KV, _lib.VRM_KV_I8, _lib.VRM_KV_F32])
@pytest.mark.parametrize("N,B", [(1, 1), (17, 1), (300, 2), (1023, 1), (2048, 64), (4095, 3), (5000, 700)])
def test_the_workspace_is_enough_for_any_tiles(lib, N, B, kv):
    """vrm_paged_chunk_workspace_bytes knows neither window nor contexts."""
    seen = 0
    for H, KH, D in ((32, 8, 128), (28, 4, 64), (12, 12, 96), (7, 1, 256)):
        if N * (H // KH) // 128 * KH >= 900:
            continue  # tiles enough without shares: such calls need no workspace and would be launched
        for max_pp in (20, 64, 65, 1000, 20000):
            have = lib.vrm_paged_chunk_workspace_bytes(N, B, H, KH, D, 16, max_pp, BF, kv)
            for window, expected in ((0, 0), (1, 0), (1000, 0), (0, 1), (0, 1024), (5000, 2000)):
                assert 0 < _need(lib, N, B, H, KH, D, 16, max_pp, window, expected, kv=kv) <= have
                seen += 1
    assert seen


def test_calls_past_a_grids_threads(lib):
    """Batches of so many sequences that a launch would wrap are refused."""
    args = (16, BF, 128, 128, 16, None, 16, 16, 16, 16, None, 16, 1 << 62)
    for B, KH in ((1 << 20, 32), (1 << 24, 1), (1 << 30, 64)):
        rc = lib.vrm_paged_chunk_attention(*args, 4, B, KH, KH, 128, 16, 1, 4, 2, 0, 0.1, 1, 0, KV, None)
        assert rc == -2 and b"too many" in lib.vrm_last_error()
        assert lib.vrm_paged_chunk_workspace_bytes(4, B, KH, KH, 128, 16, 2, BF, KV) == 0


@pytest.mark.parametrize("scale", [3e38, -2.4e38, float("inf"), float("nan")])
def test_scales_past_float32(lib, scale):
    args = (16, BF, 1024, 128, 16, None, 16, 16, 16, 16, None, None, 0, 2048, 64, 8, 2, 128, 16, 1, 4, 64, 0)
    assert lib.vrm_paged_chunk_attention(*args, scale, 1, 0, KV, None) == -1 and b"scale" in lib.vrm_last_error()
    assert lib.vrm_paged_chunk_attention(*args, 2.3e38, 1, 0, KV, None) == -3  # (as far as the workspace)
