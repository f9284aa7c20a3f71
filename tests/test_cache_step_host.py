"""The cache operators' host side without a GPU, where it can go wrong."""

import pytest


@pytest.fixture(scope="module")
def lib():
    from wpt_b200 import _lib, build
    build.build()
    return _lib


@pytest.mark.parametrize("B, T, H, N", [(8, 4096, 16, 4096), (1, 131072, 32, 131072), (8, 32768, 32, 32768),
                                        (1, 1 << 20, 64, 1 << 20), (2, 1 << 20, 32, 700), (64, 8192, 32, 8192),
                                        (1000, 300, 8, 9000)])
def test_attn_weights_scratch_is_linear(lib, B, T, H, N):
    """13 bytes a (query, head) column, padded to whole tiles of 128, and up to 256 a key or 10 MB in all."""
    columns = -(-T * H // 128) * 128
    size = lib.lib().wpt_attn_weights_scratch_bytes(B, T, H, N)
    assert 0 < size <= 13 * B * columns + max(256 * B * N, 10 << 20)
