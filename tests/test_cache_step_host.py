"""The cache operators' host side without a GPU, where it can go wrong."""

import os
import random
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


def test_the_package_imports_without_cuda_bindings():
    """A torch built without CUDA has none of torch._C's CUDA functions: the import works, the first call refuses."""
    code = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda")]:
    delattr(torch._C, name)
import wpt_b200
try:
    wpt_b200.cache_evict(torch.zeros(1, 4, 8), torch.zeros(1, 4), torch.zeros(1, dtype=torch.int64), 2)
except ValueError as e:
    print(e)
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "CUDA device only" in run.stdout, run.stderr[-2000:]


def test_overlapping_places_are_found():
    """A table's strides, and two tables' of the same strides, against every byte of their places."""
    from wpt_b200.ops import _places_overlap, _tables_overlap
    rng = random.Random(0)

    def places(at, rows, sb, sn, size, N):
        each = [set(range(at + b * sb + n * sn, at + b * sb + n * sn + size)) for b in range(rows) for n in range(N)]
        every = set().union(*each)
        return every, len(every) < sum(map(len, each))

    found = 0
    for _ in range(4000):
        rows, N, N2 = rng.randint(1, 4), rng.randint(1, 5), rng.randint(1, 5)
        sb, sn, at = rng.choice([0, *range(40)]), rng.randint(0, 12), rng.randint(0, 60)
        size, size2 = rng.randint(1, 6), rng.randint(1, 6)
        one, shared = places(0, rows, sb, sn, size, N)
        other, shared2 = places(at, rows, sb, sn, size2, N2)
        assert _places_overlap(rows, sb, sn, size, N) == shared
        assert _places_overlap(rows, sb, sn, size, N, at, size2, N2) == bool(one & other)
        if not shared and not shared2:
            assert _tables_overlap(rows, [at, sb, sn, size2, N2, 0, sb, sn, size, N]) == bool(one & other)
            found += bool(one & other)
    assert found > 100
