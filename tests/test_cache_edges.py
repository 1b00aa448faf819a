"""Refusals of the cache operators at the edges of what they take (no GPU needed: arguments are looked at before the device;
where one is there and the library bound, calls that are not refused have no sequences and launch nothing)."""
import numpy as np
import pytest

from .test_cache_abi import LIMIT, SHAPE, lanes, lib, parts, sequences        # noqa: F401 (lib: a fixture)
from qiyas_b200 import blocks as B


def overlaps(row, head, rows, heads, dim):
    starts = np.sort((np.arange(rows)[:, None] * row + np.arange(heads) * head).ravel())
    return bool((np.diff(starts) < dim).any())


@pytest.mark.parametrize("rows,heads,row,head", [(9, 2, 64, 64), (9, 2, 128, 128), (9, 2, 128, 1151), (9, 2, 100, 150), (9, 2, 128, 64), (9, 2, 64, 576), (9, 2, 64, 575),
                                                 (9, 8, 64, 128), (9, 8, 130, 65), (9, 8, 128, 1024 + 64), (9, 8, 192, 64 + 9 * 192), (3, 2, 640, 320), (9, 8, 512, 64),
                                                 (2, 8, 64, 128), (2, 8, 65, 130), (9, 4, 256, 320), (9, 4, 300, 100), (1, 8, 0, 64), (9, 2, 576, 64)])
def test_written_rows_have_to_lie_apart(lib, rows, heads, row, head):      # noqa: F811
    """Rows of 64 values: strides that bring a head of one row onto another row's are refused, all others are not."""
    from qiyas_b200 import _lib
    cache, seq, at = parts(heads=heads), sequences(rows=rows, count=0), lanes(256, row, head)
    bad = overlaps(row, head, rows, heads, 64)
    rc = lib.qb200_cache_read(cache, seq, B.F16, at, None, None)
    assert (rc == SHAPE) == bad, rc
    rc = lib.qb200_cache_read(cache, seq, B.F16, None, at, None)
    assert (rc == SHAPE) == bad, rc
    cache = parts(heads=1)
    args = _lib.ATTENTION(256, 64 * heads, 64, 256, row, head, 0, 4096, 1 << 40, heads, 0, 0, 0.125, 1, 0)
    rc = lib.qb200_cache_attention(cache, seq, B.F16, args, None)
    assert (rc == SHAPE) == bad, rc
    assert lib.qb200_cache_write(parts(heads=heads), seq, B.F16, at, at, None) != SHAPE      # what is read may overlap


def test_strides_of_all_kinds(lib):                                         # noqa: F811
    rng = np.random.default_rng(7)
    refused = 0
    for _ in range(3000):
        rows, heads = int(rng.integers(1, 12)), int(rng.integers(1, 12))
        row, head = (int(rng.choice([64, 65, 80, 96, 100, 128, 130, 192, 256, 512, 640, 700, 777])) for _ in range(2))
        rc = lib.qb200_cache_read(parts(heads=heads), sequences(rows=rows, count=0), B.F16, lanes(256, row, head), None, None)
        assert (rc == SHAPE) == overlaps(row, head, rows, heads, 64), (rows, heads, row, head)
        refused += rc == SHAPE
    assert 500 < refused < 2500


@pytest.mark.parametrize("window,rows,refused", [(2 ** 31 - 2000, 100, False), (2 ** 31 - 3000, 3001, True), (2 ** 31 - 1, 2 ** 30, False), (2 ** 30, 2 ** 30, True), (2 ** 30, 2 ** 30 - 1, False)])
def test_windows_and_rows_that_leave_32_bits_together(lib, window, rows, refused):      # noqa: F811
    """Differences of a row's place and the window are taken in 32 bits; a window of all a sequence can have is none."""
    from qiyas_b200 import _lib
    cache, seq = parts(pages=2 ** 27 - 1, heads=1), sequences(rows=rows, count=0, width=2 ** 27 - 70)
    args = _lib.ATTENTION(256, 64, 64, 256, 64, 64, 0, 4096, 1 << 40, 1, 0, 0, 0.125, 1, window)
    rc = lib.qb200_cache_attention(cache, seq, B.F16, args, None)
    assert (rc == LIMIT) == refused, (rc, lib.qb200_last_error())


@pytest.mark.parametrize("change", [dict(max_queries=2 ** 31), dict(max_length=2 ** 40), dict(max_length=-2 ** 31 - 1), dict(window=2 ** 31), dict(max_queries=1.5),
                                    dict(window="16"), dict(workspace_bytes=-1), dict(scale="large")])
def test_numbers_the_library_cannot_hold_are_argument_errors(change):
    """As every other argument error of the mirror: ValueError, before the library is called."""
    import torch
    from qiyas_b200 import BlockCache
    from qiyas_b200.ops import GpuOps

    class Host:                     # the checks alone: tensors and "device" of the host, and no library
        device = -1
    ops = GpuOps.__new__(GpuOps)
    ops.gpu, ops.lib, ops._scratch = Host(), None, {}
    codes, scales = torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2)
    cache = BlockCache(codes, codes.clone(), scales, scales.clone())
    q, table, lengths = torch.zeros(3, 4, 64), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.CacheAttention(cache, q, torch.zeros_like(q), table, lengths, workspace=4096, stream=0, **change)
    bounds = {k: v for k, v in change.items() if k.startswith("max")}
    if bounds:
        with pytest.raises(ValueError):
            ops.attention_workspace_bytes(cache, q, table, lengths, **bounds)
