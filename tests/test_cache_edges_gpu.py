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
