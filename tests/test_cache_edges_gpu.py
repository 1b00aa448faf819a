"""The cache operators at the edges of what they are documented to take: empty batches, scales of every kind, odd offsets, streams."""
import numpy as np
import pytest

from . import helpers as H
from .test_cache_gpu import Setup, gpu, ints, kind_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 16, 300])
@pytest.mark.parametrize("with_offsets", [True, False])
def test_a_batch_of_no_sequences_with_padded_rows(rows, with_offsets):
    """The row buffers of a captured step stay as they are when nobody is being served: rows, and no sequences."""
    import torch
    s = Setup(41, 1, 32, 2, 16, 32)
    o, cache = H.ops(), s.on_gpu()
    table, lengths = torch.empty(0, 2, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    offsets = ints([0]) if with_offsets else None
    k, q = torch.full((rows, 2, 32), 3.0, device="cuda"), torch.full((rows, 4, 32), 2.0, device="cuda")
    out_k, out_q = torch.full_like(k, 9.0), torch.full_like(q, 9.0)
    o.CacheWrite(cache, k, k, table, lengths, offsets=offsets)
    o.CacheRead(cache, out_k, None, table, lengths, offsets=offsets)
    o.CacheAttention(cache, q, out_q, table, lengths, offsets=offsets)
    assert o.gpu.status() == 0
    assert (out_k == 9).all() and (out_q == 9).all()
    assert np.array_equal(cache.k_codes.cpu().numpy(), s.k.codes) and np.array_equal(cache.k_scales.cpu().numpy(), s.k.scales)


def written(codes, scale, at, x):
    """The definition of a write of rows x [n, dim] behind `at` tokens of a block, codes [page, dim], whatever the block's scale."""
    codes, f32 = codes.copy(), np.float32
    finite = np.isfinite(x)
    need = f32(np.abs(np.where(finite, x, 0)).max() * f32(1 / 127))
    had = f32(scale) if at else f32(0)
    new = had if need <= abs(had) else max(need, f32(abs(had) * f32(1.25)))
    if at and new != had:
        codes[:at] = np.rint(codes[:at].astype(np.float64) * float(had) / float(new))
    if new == 0:
        codes[at:at + len(x)] = 0
    else:
        rounded = np.rint(np.where(finite, x, 0).astype(np.float64) / float(new))
        codes[at:at + len(x)] = np.where(finite, rounded, 127 * np.where(np.isnan(x), 0, np.sign(x)) * np.sign(float(new)))
    return codes, new


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,dim", [(16, 16), (16, 128), (64, 64), (64, 128), (128, 112), (128, 256)])
def test_writes_behind_blocks_of_any_scale(kind, page, dim):
    """A caller's blocks may have scales of zero and below, with codes other than zero: the earlier codes become the integers
    nearest c * s / scale where the scale changes (0 for s = 0), and stay where it stays."""
    scales = [0.0, -0.0, 0.0, -1e-3, -1.0, -0.02, 0.02, 0.0, -0.5]
    factor = [1.0, 1e-2, 0.0, 1.0, 1.0, 2.0, 2.0, np.inf, np.inf]                # of the rows written: below, above, zeros, an infinity
    s = Setup(42, len(scales), page, 2, page, dim)
    o = H.ops()
    at, n = page // 2 + 1, page // 4
    rng = s.rng
    x = rng.standard_normal((len(scales), n, 2, dim)).astype(np.float32)
    for b, f in enumerate(factor):
        if np.isinf(f):
            x[b, 0, :, 3], x[b, 1, :, 4] = np.inf, -np.inf
        else:
            x[b] *= np.float32(f)
        s.k.scales[s.table[b, 0]] = s.v.scales[s.table[b, 0]] = scales[b]
    t = gpu(x.reshape(-1, 2, dim), kind_of(kind))
    x = t.float().cpu().numpy().reshape(x.shape)
    cache = s.on_gpu()
    o.CacheWrite(cache, t, -t, gpu(s.table), ints([at] * len(scales)), offsets=ints(np.arange(len(scales) + 1) * n))
    assert o.gpu.status() == 32
    for b in range(len(scales)):
        for c, codes, held, sign in ((s.k, cache.k_codes, cache.k_scales, 1), (s.v, cache.v_codes, cache.v_scales, -1)):
            for h in range(2):
                p = int(s.table[b, 0])
                want, scale = written(c.codes[p, h], c.scales[p, h], at, sign * x[b, :, h])
                assert held[p, h].item() == scale, b
                assert np.array_equal(codes[p, h].cpu().numpy(), want), b
    out = H.empty(len(scales) * at * 2 * dim, t.dtype).view(-1, 2, dim)
    o.CacheRead(cache, out, None, gpu(s.table), ints([0] * len(scales)), offsets=ints(np.arange(len(scales) + 1) * at))
    assert (out[:at] == 0).all() and o.gpu.status() == 0                         # what a scale of zero held is zero still
