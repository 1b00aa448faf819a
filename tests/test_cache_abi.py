"""What the cache operators refuse, through the C ABI and the host mirror (no GPU needed: arguments are looked at before the device)."""
import ctypes as C

import pytest

from qiyas_b200 import blocks as B

FORMAT, SHAPE, POINTER, WORKSPACE, DEVICE, LIMIT = -1, -2, -3, -4, -5, -6


@pytest.fixture(scope="module")
def lib():
    from qiyas_b200 import _lib, build
    build.build()
    return _lib.load()


def parts(**change):
    from qiyas_b200 import _lib
    want = dict(k_codes=256, v_codes=512, k_scales=1024, v_scales=2048, pages=4, heads=2, page=16, dim=64)
    want.update(change)
    return _lib.CACHE(*want.values())


def sequences(**change):
    from qiyas_b200 import _lib
    want = dict(table=256, lengths=512, offsets=1024, count=3, width=2, rows=9)
    want.update(change)
    return _lib.SEQUENCES(*want.values())


def lanes(base=256, row=128, head=64):
    from qiyas_b200 import _lib
    return _lib.LANES(base, row, head)


def write(lib, cache=None, seq=None, kind=B.F16, k=256, row=128, head=64, v=256):
    return lib.qb200_cache_write(cache or parts(), seq or sequences(), kind, lanes(k, row, head), lanes(v, row, head), None)


def attention(lib, cache=None, seq=None, kind=B.F16, q=256, row=512, head=64, out=256, lse=0, heads=8, max_queries=0, max_length=0, scale=0.125, causal=1,
              window=0, workspace=4096, size=1 << 40):
    from qiyas_b200 import _lib
    args = _lib.ATTENTION(q, row, head, out, row, head, lse, workspace, size, heads, max_queries, max_length, scale, causal, window)
    return lib.qb200_cache_attention(cache or parts(), seq or sequences(), kind, args, None)


CACHES = [(dict(page=8), SHAPE), (dict(page=48), SHAPE), (dict(dim=24), SHAPE), (dict(dim=272), SHAPE), (dict(dim=0), SHAPE), (dict(pages=0), SHAPE),
          (dict(heads=-1), SHAPE), (dict(heads=70000), LIMIT), (dict(pages=2 ** 30), LIMIT), (dict(k_codes=0), POINTER), (dict(v_scales=0), POINTER),
          (dict(k_codes=264), POINTER), (dict(v_scales=1026), POINTER)]
SEQUENCES = [(dict(count=-1), SHAPE), (dict(width=-1), SHAPE), (dict(rows=-1), SHAPE), (dict(width=2 ** 28), LIMIT), (dict(count=2 ** 25, rows=2 ** 26), LIMIT),
             (dict(offsets=0, rows=2), SHAPE), (dict(lengths=0), POINTER), (dict(table=0), POINTER), (dict(table=258), POINTER), (dict(offsets=1025), POINTER)]


@pytest.mark.parametrize("change,code", CACHES)
def test_caches_that_are_refused(lib, change, code):
    assert write(lib, cache=parts(**change)) == code
    assert attention(lib, cache=parts(**change), heads=max(1, change.get("heads", 2)) * 2) == code
    assert lib.qb200_last_error()


@pytest.mark.parametrize("change,code", SEQUENCES)
def test_sequences_that_are_refused(lib, change, code):
    assert write(lib, seq=sequences(**change)) == code
    assert attention(lib, seq=sequences(**change)) == code
    assert lib.qb200_cache_read(parts(), sequences(**change), B.F16, lanes(), lanes(), None) == code


def test_rows_that_are_refused(lib):
    assert write(lib, kind=B.Q8_0) == FORMAT
    assert write(lib, k=0) == POINTER
    assert write(lib, v=257) == POINTER
    assert write(lib, kind=B.F32, k=258) == POINTER
    assert write(lib, row=-1) == SHAPE
    assert write(lib, head=1 << 60) == SHAPE
    assert lib.qb200_cache_read(parts(), sequences(), B.F16, None, None, None) == POINTER
    assert lib.qb200_cache_write(None, sequences(), B.F16, lanes(), lanes(), None) == POINTER
    assert lib.qb200_cache_write(parts(), None, B.F16, lanes(), lanes(), None) == POINTER
    assert lib.qb200_cache_write(parts(), sequences(), B.F16, lanes(), None, None) == POINTER
    assert lib.qb200_cache_attention(parts(), sequences(), B.F16, None, None) == POINTER


def test_attention_refuses(lib):
    assert attention(lib, heads=7) == SHAPE
    assert attention(lib, heads=0) == SHAPE
    assert attention(lib, window=-1) == SHAPE
    assert attention(lib, window=4, causal=0) == SHAPE
    assert attention(lib, scale=float("nan")) == SHAPE
    assert attention(lib, scale=float("inf")) == SHAPE
    assert attention(lib, max_queries=-1) == SHAPE
    assert attention(lib, max_length=-1) == SHAPE
    assert attention(lib, lse=1026) == POINTER
    assert attention(lib, q=0) == POINTER
    assert attention(lib, kind=B.BF16, out=257) == POINTER
    assert attention(lib, kind=100 + 7) == FORMAT
    assert attention(lib, seq=sequences(rows=2 ** 30), heads=8) == LIMIT
    assert attention(lib, workspace=4104) == WORKSPACE


@pytest.mark.parametrize("row,head", [(0, 64), (63, 64), (512, 0), (512, 48)])
def test_written_rows_that_overlap_are_refused(lib, row, head):
    from qiyas_b200 import _lib
    bad, good = lanes(256, row, head), lanes(256, 512, 64)
    assert lib.qb200_cache_read(parts(), sequences(), B.F16, bad, good, None) == SHAPE
    assert lib.qb200_cache_read(parts(), sequences(), B.F16, None, bad, None) == SHAPE
    args = _lib.ATTENTION(256, 512, 64, 256, row, head, 0, 4096, 1 << 40, 8, 0, 0, 0.125, 1, 0)
    assert lib.qb200_cache_attention(parts(), sequences(), B.F16, args, None) == SHAPE


def test_a_good_call_needs_a_device(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    assert write(lib) == DEVICE
    assert lib.qb200_cache_read(parts(), sequences(), B.F32, lanes(), None, None) == DEVICE
    assert attention(lib) == DEVICE


def test_the_mirror_refuses_what_the_abi_cannot_be_told():
    import torch
    from qiyas_b200 import BlockCache
    from qiyas_b200.ops import GpuOps
    codes, scales = torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2)
    cache = BlockCache(codes, codes.clone(), scales, scales.clone())
    assert cache.nbytes == 2 * (4 * 2 * 16 * 64 + 4 * 2 * 4)
    for bad in ((codes[:, :, :8], codes[:, :, :8], scales, scales), (codes, codes[:3], scales, scales), (codes, codes, scales[:3], scales),
                (codes.float(), codes, scales, scales), (codes, codes, scales.double(), scales), (codes.transpose(0, 1).contiguous().transpose(0, 1), codes, scales, scales),
                (codes[0], codes[0], scales, scales)):
        with pytest.raises((ValueError, NotImplementedError)):
            BlockCache(*bad)

    class Unbound:                  # the checks alone: a library that is bound to device 0
        device = 0
    ops = GpuOps.__new__(GpuOps)
    ops.gpu, ops.lib, ops._scratch = Unbound(), None, {}
    rows = torch.zeros(3, 2, 64)
    table, lengths = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for k, v in ((rows.double(), rows.double()), (rows[:, :1], rows), (rows[..., :48], rows), (rows, rows[:2]), (rows, rows.half()), (rows, rows),
                 (torch.zeros(3, 2, 128)[..., ::2], rows)):
        with pytest.raises((ValueError, NotImplementedError)):       # the last but one: rows that are not on the library's device
            ops.CacheWrite(cache, k, v, table, lengths)
    with pytest.raises(ValueError):
        ops.CacheRead(cache, None, None, table, lengths)
    for t, n, off in ((table[:2], lengths, None), (table.long(), lengths, None), (table, lengths.float(), None), (table, lengths, torch.zeros(3, dtype=torch.int32)),
                      (table.t(), lengths, None), (table, lengths[None], None), (torch.zeros(3, 4, dtype=torch.int32)[:, ::2], lengths, None)):
        with pytest.raises(ValueError):
            ops._sequences(cache, t, n, off, 3)


def test_packed_structures_have_the_headers_sizes():
    """The header compiled as C: sizes and offsets are those the mirror packs."""
    import os
    import subprocess
    import sys
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = """#include <stdio.h>
#include <stddef.h>
#include "qiyas_b200.h"
int main(void) { printf("%zu %zu %zu %zu %zu %zu %zu", sizeof(qb200_cache_t), sizeof(qb200_sequences_t), sizeof(qb200_lanes_t), sizeof(qb200_attention_t),
 offsetof(qb200_sequences_t, count), offsetof(qb200_attention_t, q_heads), offsetof(qb200_attention_t, scale)); return 0; }"""
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "a.c"), "w") as f:
            f.write(text)
        subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), "-o", os.path.join(d, "a"), os.path.join(d, "a.c")])
        got = [int(x) for x in subprocess.check_output([os.path.join(d, "a")]).split()]
    assert sys.maxsize > 2 ** 32
    assert got == [len(parts()), len(sequences()), len(lanes()), 96, 24, 72, 84]
