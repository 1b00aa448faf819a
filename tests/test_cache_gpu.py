"""The cache operators on the GPU against their definitions in 64 bits."""
import numpy as np
import pytest

from . import helpers as H
from .cache_oracle import Cache, attend

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16"]


def kind_of(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def gpu(x, kind=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if kind is None else t.to(kind)


def ints(values):
    return gpu(np.asarray(values, np.int32))


class Setup:
    """A cache with random contents, pages in random order, for sequences that may grow to `most` tokens; what no sequence
    has written yet holds codes and scales that must not matter."""

    def __init__(self, seed, sequences, most, heads, page, dim, spare=3):
        self.rng = np.random.default_rng(seed)
        self.width = max(1, (most + page - 1) // page)
        self.pages = sequences * self.width + spare
        self.page, self.heads, self.dim = page, heads, dim
        self.table = self.rng.permutation(self.pages)[:sequences * self.width].reshape(sequences, self.width).astype(np.int32)
        shape = (self.pages, heads, page, dim)
        self.k, self.v = (Cache(self.rng.integers(-127, 128, shape).astype(np.int8),
                                (self.rng.uniform(0.2, 1, (self.pages, heads)) * s).astype(np.float32)) for s in (0.02, 0.01))

    def on_gpu(self):
        from qiyas_b200 import BlockCache
        return BlockCache(gpu(self.k.codes), gpu(self.v.codes), gpu(self.k.scales), gpu(self.v.scales))

    def rows(self, count, heads, kind, scale=1.0):
        """Values of the lane type, as a tensor and as the numbers it holds."""
        x = (self.rng.standard_normal((count, heads, self.dim)) * scale).astype(np.float32)
        t = gpu(x, kind_of(kind))
        return t, t.float().cpu().numpy()


def offsets_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


# ------------------------------------------------------------------------------------------------ write and read back

WRITES = [
    # heads, page, dim, tokens before, tokens written
    (1, 16, 16, [0], [1]),
    (2, 16, 128, [0, 5, 15, 16, 31], [1, 1, 1, 1, 1]),
    (3, 32, 80, [0, 1, 31, 32, 40], [1, 33, 2, 0, 100]),
    (2, 64, 64, [0, 63, 10], [200, 3, 0]),
    (1, 128, 256, [0, 127, 130], [129, 1, 260]),
    (5, 128, 96, [3, 0], [300, 128]),
    (2, 64, 112, [7, 0], [1, 64]),
    (1, 16, 256, [0, 9], [40, 7]),
    (2, 32, 192, [30, 2], [70, 29]),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,page,dim,before,new", WRITES)
def test_write_and_read_back(kind, heads, page, dim, before, new):
    import torch
    most = max(b + n for b, n in zip(before, new))
    s = Setup(dim + page, len(before), most, heads, page, dim)
    cache, o = s.on_gpu(), H.ops()
    offsets = offsets_of(new)
    rows = int(offsets[-1]) + 2                       # two rows behind the last sequence
    k, kn = s.rows(rows, heads, kind, 1.3)
    v, vn = s.rows(rows, heads, kind, 0.7)
    o.CacheWrite(cache, k, v, gpu(s.table), ints(before), offsets=ints(offsets))
    for b, (f, n) in enumerate(zip(before, new)):
        s.k.write(s.table[b], f, kn[offsets[b]:offsets[b] + n])
        s.v.write(s.table[b], f, vn[offsets[b]:offsets[b] + n])
    assert o.gpu.status() == 0
    assert np.array_equal(cache.k_codes.cpu().numpy(), s.k.codes)
    assert np.array_equal(cache.v_codes.cpu().numpy(), s.v.codes)
    assert np.array_equal(cache.k_scales.cpu().numpy(), s.k.scales)
    assert np.array_equal(cache.v_scales.cpu().numpy(), s.v.scales)

    # everything of every sequence, and what lies behind the last row stays
    counts = [b + n for b, n in zip(before, new)]
    offsets = offsets_of(counts)
    total = int(offsets[-1])
    ko = torch.full((total + 1, heads, dim), 7.0, dtype=kind_of(kind), device="cuda")
    vo = ko.clone()
    o.CacheRead(cache, ko, vo, gpu(s.table), ints([0] * len(before)), offsets=ints(offsets))
    assert o.gpu.status() == 0
    for got, c in ((ko, s.k), (vo, s.v)):
        want = np.concatenate([c.values(s.table[b], 0, n) for b, n in enumerate(counts)]).astype(np.float32)   # the f32 product, rounded
        assert torch.equal(got[:total], gpu(want).to(kind_of(kind)))
        assert (got[total:] == 7).all()


def test_tokens_one_by_one_stay_within_two_and_a_half_steps():
    import torch
    s = Setup(3, 1, 64, 2, 64, 32)
    cache, o = s.on_gpu(), H.ops()
    x = (s.rng.standard_normal((64, 2, 32)) * np.exp(np.arange(64) / 9)[:, None, None]).astype(np.float32)     # every token larger
    for i in range(64):
        t = gpu(x[i:i + 1])
        o.CacheWrite(cache, t, t, gpu(s.table), ints([i]))
        s.k.write(s.table[0], i, x[i:i + 1])
    assert np.array_equal(cache.k_codes.cpu().numpy(), s.k.codes)
    assert np.array_equal(cache.k_scales.cpu().numpy(), s.k.scales)
    step = s.k.scales[s.table[0, 0]]
    assert np.all(np.abs(s.k.values(s.table[0], 0, 64) - x) <= 2.5 * step[None, :, None] * (1 + 1e-6))
    # the same as one write, but for the rounding: half a step
    ko = torch.empty(64, 2, 32, device="cuda")
    o.CacheWrite(cache, gpu(x), gpu(x), gpu(s.table), ints([0]), offsets=ints([0, 64]))
    o.CacheRead(cache, ko, None, gpu(s.table), ints([0]), offsets=ints([0, 64]))
    step = cache.k_scales.cpu().numpy()[s.table[0, 0]]
    assert np.all(np.abs(ko.cpu().numpy() - x) <= 0.5 * step[None, :, None] * (1 + 1e-6))


@pytest.mark.parametrize("kind", KINDS)
def test_write_of_zeros_tiny_values_nan_and_infinities(kind):
    tiny = {"f32": 1e-44, "f16": 6e-8, "bf16": 1e-39}[kind]
    s = Setup(11, 6, 16, 1, 16, 16)
    cache, o = s.on_gpu(), H.ops()
    x = s.rng.standard_normal((6, 8, 1, 16)).astype(np.float32)
    x[0] = 0
    x[1] *= tiny
    x[2, 3, 0, 5] = np.nan
    x[3, 1, 0, 0], x[3, 2, 0, 1] = np.inf, -np.inf
    x[4] = 0
    x[4, 0, 0, 0] = np.inf
    x[5] = {"f32": 3e38, "f16": 65504, "bf16": 3e38}[kind] * np.sign(x[5])
    t = gpu(x.reshape(48, 1, 16), kind_of(kind))
    x = t.float().cpu().numpy().reshape(x.shape)
    o.CacheWrite(cache, t, t, gpu(s.table), ints([0] * 6), offsets=ints(np.arange(7) * 8))
    assert o.gpu.status() == 32
    for b in range(6):
        s.k.write(s.table[b], 0, x[b])
    assert np.array_equal(cache.k_scales.cpu().numpy(), s.k.scales)
    assert np.array_equal(cache.k_codes.cpu().numpy(), s.k.codes)


def test_ties_round_to_even_from_the_exact_quotient():
    s = Setup(12, 1, 16, 1, 16, 256)
    cache, o = s.on_gpu(), H.ops()
    for scale in (1.0, 0.375, 3.0, 0.1):
        half = (np.arange(256) - 127.5).astype(np.float32) * np.float32(scale)           # halves, and next to halves
        x = np.stack([half, np.nextafter(half, np.float32(0)), np.nextafter(half, np.float32(1e9) * np.sign(half)), half])
        x[3, 0] = np.float32(127) * np.float32(scale)
        x = np.clip(x, -127 * np.float32(scale), 127 * np.float32(scale)).astype(np.float32).reshape(4, 1, 256)
        o.CacheWrite(cache, gpu(x), gpu(-x), gpu(s.table), ints([0]), offsets=ints([0, 4]))
        s.k.write(s.table[0], 0, x)
        s.v.write(s.table[0], 0, -x)
        assert np.array_equal(cache.k_codes.cpu().numpy(), s.k.codes)
        assert np.array_equal(cache.v_codes.cpu().numpy(), s.v.codes)


@pytest.mark.parametrize("kind", KINDS)
def test_strides_and_alignment(kind):
    """Rows of a wider projection, a head order of their own, and a base that is not 16-byte aligned."""
    import torch
    s = Setup(21, 2, 40, 3, 16, 48)
    o = H.ops()
    wide, _ = s.rows(40, 9, kind)                                   # q, k and v of a row side by side
    flat = torch.cat([torch.zeros(1, dtype=wide.dtype, device="cuda"), wide.reshape(-1)])
    odd = flat[1:].view(40, 9, 48)
    swapped = wide.transpose(0, 1).contiguous().transpose(0, 1)     # heads outside rows
    for src in (wide, odd, swapped):
        cache = s.on_gpu()
        o.CacheWrite(cache, src[:, 3:6], src[:, 6:9], gpu(s.table), ints([3, 0]), offsets=ints([0, 17, 40]))
        want = Cache(s.k.codes.copy(), s.k.scales.copy())
        n = wide.float().cpu().numpy()
        want.write(s.table[0], 3, n[:17, 3:6])
        want.write(s.table[1], 0, n[17:, 3:6])
        assert np.array_equal(cache.k_codes.cpu().numpy(), want.codes)
        back = torch.zeros_like(src)
        o.CacheRead(cache, back[:, 3:6], None, gpu(s.table), ints([3, 0]), offsets=ints([0, 17, 40]))
        vals = np.concatenate([want.values(s.table[0], 3, 17), want.values(s.table[1], 0, 23)]).astype(np.float32)
        assert torch.equal(back[:, 3:6], gpu(vals).to(kind_of(kind)))
        assert (back[:, :3] == 0).all() and (back[:, 6:] == 0).all()


def test_pages_lengths_and_rows_outside_are_left_out():
    """A bad page, a length behind the table and offsets past the rows: nothing else is touched, and the status says so."""
    import torch
    s = Setup(31, 4, 32, 2, 16, 32)
    table = s.table.copy()
    table[0, 1], table[1, 0] = s.pages, -5
    cache, o = s.on_gpu(), H.ops()
    k, kn = s.rows(40, 2, "f32")
    new = [20, 10, 4, 6]
    before = [4, 0, 30, 40]                            # the third reaches past its two pages, the fourth begins behind them
    offsets = offsets_of(new)
    o.CacheWrite(cache, k, k, gpu(table), ints(before), offsets=ints(offsets))
    assert o.gpu.status() == 16
    s.k.write(s.table[0], 4, kn[0:12])                 # the part on the good page
    s.k.write(s.table[2], 30, kn[30:32])
    assert np.array_equal(cache.k_codes.cpu().numpy(), s.k.codes)
    assert np.array_equal(cache.k_scales.cpu().numpy(), s.k.scales)
    out = torch.full((40, 2, 32), 9.0, device="cuda")
    o.CacheRead(cache, out, None, gpu(table), ints(before), offsets=ints(offsets))
    assert o.gpu.status() == 16
    got = out.cpu().numpy()
    assert np.array_equal(got[:12], s.k.values(s.table[0], 4, 12).astype(np.float32))
    assert np.array_equal(got[30:32], s.k.values(s.table[2], 30, 2).astype(np.float32))
    assert (got[12:30] == 9).all() and (got[32:] == 9).all()
    # offsets that leave the rows
    o.CacheRead(cache, out, None, gpu(s.table), ints([0, 0, 0, 0]), offsets=ints([0, 5, 50, 20, 60]))
    assert o.gpu.status() == 16


# ------------------------------------------------------------------------------------------------ attention

def check_attention(s, kind, lens, counts, heads, group, causal=True, window=0, max_queries=0, max_length=0, q_scale=1.0, scale=None, with_offsets=True,
                    stream=None):
    """CacheAttention on a setup against the definition.  The tolerance, for a row with weights p: the scores are sums of dim
    products in f32 (an error of (dim + 8) * 2^-24 of scale * sum |q||k| each, 2^-20 for the cut of q, the exponentials and
    V's scales), the weights are cut to f16 (half a step, 2^-11; f32 lanes: two f16, 2^-21), and the sums over tokens run in
    f32 over tokens / 128 + 64 steps.  All of that is relative to sum p |v|; the output is rounded once more to its type.  Below
    f16's normal numbers a weight is off by half of 2^-24 whatever its size: the largest weight is 2^10 at least, so that is
    2^-35 of the largest of p * (V's scale), each time a code of V, 127 at most."""
    import torch
    o = H.ops()
    cache = s.on_gpu()
    rows = int(sum(counts))
    q, qn = s.rows(rows + 1, heads, kind, q_scale)
    out = torch.full((rows + 1, heads, s.dim), 5.0, dtype=kind_of(kind), device="cuda")
    lse = torch.full((rows + 1, heads), 5.0, device="cuda")
    offsets = offsets_of(counts)
    if scale is None:
        scale = s.dim ** -0.5
    o.CacheAttention(cache, q, out, gpu(s.table), ints(lens), offsets=ints(offsets) if with_offsets else None, max_queries=max_queries, max_length=max_length,
                     scale=scale, causal=causal, window=window, lse=lse, stream=stream)
    assert o.gpu.status() == 0
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert (got[rows:] == 5).all() and (got_lse[rows:] == 5).all()
    eps = torch.finfo(kind_of(kind)).eps / 2
    cut = 2.0 ** -21 if kind == "f32" else 2.0 ** -11
    for b, (length, n) in enumerate(zip(lens, counts)):
        if n == 0:
            continue
        at = slice(offsets[b], offsets[b] + n)
        k, v = s.k.values(s.table[b], 0, length), s.v.values(s.table[b], 0, length)
        want, want_lse, weight, size = attend(qn[at].astype(np.float64), k, v, scale, causal, window)
        score = (s.dim + 8) * 2.0 ** -24 * size + 2.0 ** -20 * (1 + np.abs(size))
        sums = (length / 128 + 64) * 2.0 ** -24
        # (p <= 1, so the largest V scale of the sequence bounds p * scale)
        floor = 2.0 ** -35 * length * 127 * max([s.v.scales[x].max() for x in s.table[b][:(length + s.page - 1) // s.page]], default=0)
        bound = weight * (2 * score[..., None] + cut + sums) + np.abs(want) * eps + floor + 1e-30
        if kind != "f32":
            bound = bound + (2.0 ** -25 if kind == "f16" else 0)            # f16 output below its normal numbers
        err = np.abs(got[at] - want)
        if kind == "f16":                                                   # from 65520 on (65504 and half a step) f16 rounds to infinity
            over = np.isinf(got[at]) & (np.sign(got[at]) == np.sign(want)) & (np.abs(want) + bound >= 65520)
            err = np.where(over, 0, err)
        assert np.all(err <= bound), (b, float(np.max(err / bound)))
        nothing = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(got_lse[at]), nothing)
        assert np.all(got[at][nothing] == 0)
        d = np.abs(np.where(nothing, 0, got_lse[at]) - np.where(nothing, 0, want_lse))
        assert np.all(d <= score + sums + 2.0 ** -21 * (1 + np.abs(np.where(nothing, 0, want_lse)))), b


LENGTHS = [0, 1, 15, 16, 17, 31, 32, 33, 64, 100, 129, 300]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,group,page,dim", [(2, 1, 16, 64), (1, 4, 16, 128), (2, 8, 32, 128), (1, 3, 64, 80), (2, 5, 128, 96), (1, 7, 16, 16),
                                                  (1, 8, 64, 256), (2, 9, 32, 128), (1, 16, 16, 64), (1, 12, 128, 192), (3, 2, 32, 112), (1, 33, 16, 48)])
def test_attention_of_single_tokens(kind, heads, group, page, dim):
    s = Setup(dim * 3 + group, len(LENGTHS), 300, heads, page, dim)
    check_attention(s, kind, LENGTHS, [1] * len(LENGTHS), heads * group, group, with_offsets=group % 2 == 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,group,page,dim,window,causal", [(2, 4, 16, 128, 0, True), (1, 2, 32, 64, 50, True), (1, 1, 64, 128, 1, True), (2, 3, 16, 256, 0, False),
                                                                (1, 8, 128, 96, 33, True), (3, 1, 16, 80, 17, True), (1, 5, 32, 192, 0, False)])
def test_attention_of_several_rows(kind, heads, group, page, dim, window, causal):
    lens = [5, 40, 0, 3, 64, 200, 129, 33]
    counts = [5, 7, 2, 9, 0, 50, 1, 33]                # the third and fourth have rows that see nothing
    s = Setup(dim + group, len(lens), 200, heads, page, dim)
    check_attention(s, kind, lens, counts, heads * group, group, causal, window)
    check_attention(s, kind, lens, counts, heads * group, group, causal, window, max_queries=1)        # the kernel for few rows


@pytest.mark.parametrize("kind", KINDS)
def test_attention_cut_over_many_blocks(kind):
    s = Setup(77, 3, 5000, 2, 16, 128)
    check_attention(s, kind, [5000, 1, 2777], [1, 1, 1], 16, 8)
    check_attention(s, kind, [5000, 1, 2777], [2, 0, 3], 8, 4, window=1500)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,group,page,dim,window", [(2, 4, 64, 128, 0), (1, 3, 16, 256, 0), (1, 8, 32, 64, 700), (2, 2, 128, 112, 100)])
def test_attention_of_pieces_of_prompts(kind, heads, group, page, dim, window):
    """Row tiles of 128 and 256, whole and not, over contexts that several blocks share."""
    lens, counts = [900, 1300, 70, 333], [40, 130, 70, 1]
    s = Setup(dim * 2 + group, len(lens), 1300, heads, page, dim)
    check_attention(s, kind, lens, counts, heads * group, group, True, window)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_many_sequences(kind):
    """More sequences than a warp has lanes, some without rows, some without tokens, their work cut into equal shares."""
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(0, 200, 75)]
    lens[3], lens[40], lens[74] = 3000, 2500, 0
    counts = [int(x) for x in rng.integers(0, 3, 75)]
    s = Setup(85, 75, 3000, 1, 16, 64)
    check_attention(s, kind, lens, counts, 2, 2, max_queries=2)
    check_attention(s, kind, lens, counts, 2, 2)
    counts = [1] * 75
    check_attention(s, kind, lens, counts, 2, 2, with_offsets=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,rising", [(128, 1.0), (128, 8.0), (192, 8.0)])
def test_long_parts_of_prompts(kind, dim, rising):
    """Parts of a thousand tokens and more in one block, of keys that stay as large or grow, so that the largest score comes
    late.  The definition in 64 bits, with torch; the tolerance of check_attention."""
    import torch
    o = H.ops()
    heads, group, lens, counts = 8, 4, [3000, 1300, 2100], [300, 257, 40]
    s = Setup(37, 3, 3000, heads, 64, dim)
    for row in s.table:
        s.k.scales[row] *= np.linspace(1 / rising, rising, s.width)[:, None].astype(np.float32)
    q, qn = s.rows(sum(counts), heads * group, kind)
    out, lse = torch.zeros_like(q), torch.zeros(sum(counts), heads * group, device="cuda")
    offsets = offsets_of(counts)
    scale = dim ** -0.5
    o.CacheAttention(s.on_gpu(), q, out, gpu(s.table), ints(lens), offsets=ints(offsets), lse=lse)
    assert o.gpu.status() == 0
    cut = 2.0 ** -21 if kind == "f32" else 2.0 ** -11
    for b, (length, n) in enumerate(zip(lens, counts)):
        at = slice(offsets[b], offsets[b] + n)
        k, v = (gpu(x.values(s.table[b], 0, length)).double().transpose(0, 1).repeat_interleave(group, 0) for x in (s.k, s.v))
        x = q[at].double().transpose(0, 1)
        scores = torch.matmul(x, k.transpose(1, 2)) * scale
        unseen = torch.arange(length, device="cuda") > length - n + torch.arange(n, device="cuda")[:, None]
        size = (torch.matmul(x.abs(), k.abs().transpose(1, 2)) * scale).masked_fill_(unseen, 0).amax(-1)
        scores.masked_fill_(unseen, -float("inf"))
        want_lse = torch.logsumexp(scores, -1)
        p = torch.exp(scores - want_lse[..., None])
        want, weight = torch.matmul(p, v), torch.matmul(p, v.abs())
        score = (dim + 8) * 2.0 ** -24 * size + 2.0 ** -20 * (1 + size)
        sums = (length / 128 + 64) * 2.0 ** -24
        floor = 2.0 ** -35 * length * 127 * float(s.v.scales[s.table[b]].max())
        bound = weight * (2 * score[..., None] + cut + sums) + want.abs() * torch.finfo(kind_of(kind)).eps / 2 + floor + 2.0 ** -25
        assert bool(((out[at].double().transpose(0, 1) - want).abs() <= bound).all()), b
        assert bool(((lse[at].double().transpose(0, 1) - want_lse).abs() <= score + sums + 2.0 ** -21 * (1 + want_lse.abs())).all()), b


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 100, 320, 319])
@pytest.mark.parametrize("max_queries", [0, 1])
def test_windows_of_all_there_is_and_more_rows_than_tokens(window, max_queries):
    s = Setup(35, 4, 320, 1, 64, 128)
    check_attention(s, "bf16", [320, 5, 0, 300], [9, 40, 30, 70], 2, 2, window=window, max_queries=max_queries)


def test_repeated_rows_of_q_and_of_what_is_written():
    """Rows read with a stride of 0: the same row for every token."""
    import torch
    o = H.ops()
    s = Setup(36, 2, 96, 2, 16, 64)
    cache = s.on_gpu()
    q = torch.randn(1, 4, 64, device="cuda").to(torch.bfloat16)
    out, wide = (torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    o.CacheAttention(cache, q.expand(2, 4, 64), out, gpu(s.table), ints([40, 90]))
    o.CacheAttention(cache, q.repeat(2, 1, 1), wide, gpu(s.table), ints([40, 90]))
    assert torch.equal(out, wide)
    k, back, v_back = torch.randn(1, 1, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    o.CacheWrite(cache, k.expand(2, 2, 64), k.expand(2, 2, 64), gpu(s.table), ints([0, 0]))
    o.CacheRead(cache, back, v_back, gpu(s.table), ints([0, 0]))
    assert torch.equal(back, v_back) and torch.equal(back[0, 0], back[1, 1])
    assert (back[0, 0] - k[0, 0]).abs().max() <= 0.5001 * k.abs().max() / 127
    assert o.gpu.status() == 0


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_attention_with_other_scales(scale):
    s = Setup(86, 2, 300, 1, 32, 128)
    check_attention(s, "f32", [300, 41], [3, 30], 4, 4, scale=scale)
    check_attention(s, "bf16", [300, 41], [3, 30], 4, 4, scale=scale, max_queries=1)


def test_bounds_that_are_too_small_change_nothing():
    s = Setup(78, 3, 400, 1, 32, 64)
    check_attention(s, "f16", [400, 30, 77], [20, 3, 40], 4, 4, max_queries=1, max_length=16)
    check_attention(s, "f16", [400, 30, 77], [20, 3, 40], 4, 4, max_queries=1)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_with_scales_far_apart(kind):
    """V's scales over many orders of ten, pages of zeros among them, first and last; sharp weights."""
    s = Setup(79, 3, 400, 2, 16, 64)
    s.v.scales *= np.exp(s.rng.uniform(-20, 20, s.v.scales.shape)).astype(np.float32)
    for b, slots in enumerate(([0, 5, 6, 24], [0, 1, 2], [])):
        for i in slots:
            s.v.scales[s.table[b, i]], s.v.codes[s.table[b, i]] = 0, 0
            s.k.scales[s.table[b, i]] *= 0 if i == 5 else 1
    check_attention(s, kind, [400, 40, 399], [1, 1, 1], 8, 4, q_scale=3.0)
    check_attention(s, kind, [400, 40, 399], [3, 2, 1], 8, 4, q_scale=1e-3)


def test_attention_over_a_dominant_token():
    """One token takes nearly all the weight and its value is zero: what is left is the small weights' sum."""
    s = Setup(80, 1, 2048, 1, 16, 64)
    s.v.scales[:] = 0.01
    p = s.table[0, 0]
    s.v.codes[p, 0, 0] = 0
    s.k.codes[p, 0, 0], s.k.scales[p, 0] = 127, 0.05
    import torch
    o, cache = H.ops(), s.on_gpu()
    q = torch.full((1, 1, 64), 0.3, device="cuda")
    out = torch.empty_like(q)
    o.CacheAttention(cache, q, out, gpu(s.table), ints([2048]))
    want, _, weight, _ = attend(q.double().cpu().numpy(), s.k.values(s.table[0], 0, 2048), s.v.values(s.table[0], 0, 2048), 0.125)
    assert weight.max() < 1e-3                          # the small weights: 5e-4 together, of values up to 1.27
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= weight * 2.0 ** -14)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_with_strides(kind):
    import torch
    s = Setup(81, 2, 90, 2, 16, 48)
    o, cache = H.ops(), s.on_gpu()
    lens, offsets = ints([90, 33]), ints([0, 3, 5])
    x, _ = s.rows(5, 10, kind)
    flat = torch.cat([torch.zeros(1, dtype=x.dtype, device="cuda"), x.reshape(-1)])
    want = torch.empty(5, 6, 48, dtype=x.dtype, device="cuda")
    o.CacheAttention(cache, x[:, 2:8].contiguous(), want, gpu(s.table), lens, offsets=offsets)
    for q in (x[:, 2:8], flat[1:].view(5, 10, 48)[:, 2:8], x.transpose(0, 1).contiguous().transpose(0, 1)[:, 2:8]):
        room = torch.zeros(5 * 10 * 48 + 1, dtype=x.dtype, device="cuda")
        for out in (room[1:].view(5, 10, 48)[:, 1:7], room[:-1].view(10, 5, 48).transpose(0, 1)[:, 1:7]):
            room.zero_()
            o.CacheAttention(cache, q, out, gpu(s.table), lens, offsets=offsets)
            assert torch.equal(out, want)
            assert int((room != 0).sum()) == int((want != 0).sum())


def test_attention_leaves_bad_pages_out():
    import torch
    s = Setup(82, 2, 64, 1, 16, 64)
    table = s.table.copy()
    table[0, 1], table[1, 3] = -1, s.pages + 7
    o, cache = H.ops(), s.on_gpu()
    q, qn = s.rows(2, 2, "f32")
    out = torch.empty_like(q)
    o.CacheAttention(cache, q, out, gpu(table), ints([64, 10 ** 6]))
    assert o.gpu.status() == 16
    for b, keep in enumerate(([*range(16), *range(32, 64)], range(48))):
        k, v = s.k.values(s.table[b], 0, 64)[list(keep)], s.v.values(s.table[b], 0, 64)[list(keep)]
        want = attend(qn[b:b + 1].astype(np.float64), k, v, 0.125)[0]
        assert np.allclose(out[b:b + 1].double().cpu().numpy(), want, rtol=0, atol=1e-5 * np.abs(v).max())


def test_nan_in_q_stays_in_its_row_and_unwritten_places_do_not_matter():
    import torch
    s = Setup(83, 2, 64, 1, 16, 64)
    o, cache = H.ops(), s.on_gpu()
    q, _ = s.rows(2, 4, "f16")
    want, out = torch.empty_like(q), torch.empty_like(q)
    lens = ints([35, 35])
    o.CacheAttention(cache, q, want, gpu(s.table), lens)
    # pages that no token of the sequences lies in, and the rest of the last one
    for c in (cache.k_scales, cache.v_scales):
        used = s.table[:, :3].reshape(-1)
        rest = np.setdiff1d(np.arange(s.pages), used)
        c[torch.from_numpy(rest).cuda()] = float("nan")
    for c in (cache.k_codes, cache.v_codes):
        c[torch.from_numpy(s.table[:, 2]).cuda().long(), :, 3:] = -128
    o.CacheAttention(cache, q, out, gpu(s.table), lens)
    assert torch.equal(out, want)
    q[0, 1, 3] = float("nan")
    o.CacheAttention(cache, q, out, gpu(s.table), lens)
    assert out[0, 1].isnan().all()
    out[0, 1] = want[0, 1]
    assert torch.equal(out, want)


def test_same_bits_every_time_and_on_another_stream_and_as_a_graph():
    import torch
    s = Setup(84, 3, 3000, 2, 16, 128)
    o, cache = H.ops(), s.on_gpu()
    q, _ = s.rows(3, 16, "bf16")
    lens, table = ints([3000, 17, 2049]), gpu(s.table)
    want, out = torch.empty_like(q), torch.empty_like(q)
    o.CacheAttention(cache, q, want, table, lens)
    for _ in range(20):
        out.fill_(float("nan"))
        o.CacheAttention(cache, q, out, table, lens)
        assert torch.equal(out, want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.default_stream())
    out.fill_(float("nan"))
    stream.wait_stream(torch.cuda.default_stream())
    o.CacheAttention(cache, q, out, table, lens, stream=stream)
    stream.synchronize()
    assert torch.equal(out, want)
    # two graphs with workspaces of their own, replayed side by side
    outs, graphs = [torch.empty_like(q) for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for g, t in zip(graphs, outs):
        with torch.cuda.graph(g):
            o.CacheAttention(cache, q, t, table, lens, stream=torch.cuda.current_stream())
    for _ in range(10):
        for g, t, st in zip(graphs, outs, streams):
            st.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(st):
                t.fill_(float("nan"))
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_calls_at_once_on_two_streams():
    """Both kernels and products of blocks beside each other: each call gives the bits it gives alone."""
    import torch
    from qiyas_b200 import blocks as B
    o = H.ops()
    s = Setup(38, 4, 2000, 2, 32, 128)
    cache, table, lens = s.on_gpu(), gpu(s.table), ints([2000, 700, 1999, 3])
    calls = []
    for n, kind in ((1, "bf16"), (100, "f32"), (60, "f16")):
        q = s.rows(4 * n, 8, kind)[0]
        calls.append((q, ints([0, n, 2 * n, 3 * n, 4 * n]), torch.empty_like(q)))
    rows, cols = 515, 4096
    a, x = gpu(B.make_weights(B.Q4_0, rows, cols, 5)), gpu(B.make_activations(cols, 6))
    y = torch.empty(rows, device="cuda")
    for q, at, out in calls:
        o.CacheAttention(cache, q, out, table, lens, offsets=at)
    o.GemvBlocks(B.Q4_0, a, x, y, rows, cols, fmt_x=B.F32)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(out) for _ in range(2)] for _, _, out in calls]
    ys = [torch.empty_like(y) for _ in range(2)]
    torch.cuda.synchronize()
    for turn in range(10):
        for i, stream in enumerate(streams):
            for k in range(3):
                q, at, _ = calls[(k + i) % 3]
                o.CacheAttention(cache, q, got[(k + i) % 3][i], table, lens, offsets=at, stream=stream)
            o.GemvBlocks(B.Q4_0, a, x, ys[i], rows, cols, fmt_x=B.F32, stream=stream)
    torch.cuda.synchronize()
    assert o.gpu.status() == 0
    for (_, _, out), pair in zip(calls, got):
        assert torch.equal(out, pair[0]) and torch.equal(out, pair[1])
    assert torch.equal(y, ys[0]) and torch.equal(y, ys[1])


def test_a_captured_step_writes_and_attends_with_new_lengths():
    """Write and attention in one graph, replayed as the sequences grow: lengths and rows are read on the device."""
    import torch
    s = Setup(87, 3, 100, 2, 16, 64)
    o, cache = H.ops(), s.on_gpu()
    table, before, after = gpu(s.table), ints([0, 15, 40]), ints([1, 16, 41])
    k, v, q = (torch.zeros(3, h, 64, device="cuda") for h in (2, 2, 6))
    out = torch.empty_like(q)
    o.CacheWrite(cache, k, v, table, ints([0, 0, 0]))          # once outside the capture; the page is written again below
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream()
        o.CacheWrite(cache, k, v, table, before, stream=st)
        o.CacheAttention(cache, q, out, table, after, stream=st)
    cache.k_codes.copy_(gpu(s.k.codes)), cache.v_codes.copy_(gpu(s.v.codes))
    cache.k_scales.copy_(gpu(s.k.scales)), cache.v_scales.copy_(gpu(s.v.scales))
    for step in range(20):
        lens = [step, 15 + step, 40 + step]
        rows = [s.rows(3, h, "f32")[1] for h in (2, 2, 6)]
        for t, x in zip((k, v, q), rows):
            t.copy_(gpu(x))
        before.copy_(ints(lens)), after.copy_(ints([n + 1 for n in lens]))
        graph.replay()
        for b, n in enumerate(lens):
            s.k.write(s.table[b], n, rows[0][b:b + 1])
            s.v.write(s.table[b], n, rows[1][b:b + 1])
            kk, vv = s.k.values(s.table[b], 0, n + 1), s.v.values(s.table[b], 0, n + 1)
            want = attend(rows[2][b:b + 1].astype(np.float64), kk, vv, 0.125)[0]
            assert np.abs(out[b:b + 1].double().cpu().numpy() - want).max() <= 2e-5 * np.abs(vv).max()
    assert np.array_equal(cache.k_codes.cpu().numpy(), s.k.codes)
    assert o.gpu.status() == 0


def test_empty_calls_do_nothing():
    import torch
    s = Setup(88, 2, 32, 1, 16, 32)
    o, cache = H.ops(), s.on_gpu()
    none = torch.empty(0, 1, 32, device="cuda")
    o.CacheWrite(cache, none, none, gpu(s.table), ints([0, 0]), offsets=ints([0, 0, 0]))
    o.CacheRead(cache, none, none, gpu(s.table), ints([0, 0]), offsets=ints([0, 0, 0]))
    o.CacheAttention(cache, none, none, gpu(s.table), ints([5, 5]), offsets=ints([0, 0, 0]))
    empty = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    o.CacheAttention(cache, none, none, empty, ints([]))
    rows = torch.full((4, 1, 32), 3.0, device="cuda")                   # rows, but of no sequence
    o.CacheWrite(cache, rows, rows, gpu(s.table), ints([0, 0]), offsets=ints([0, 0, 0]))
    out = torch.full_like(rows, 9.0)
    o.CacheAttention(cache, rows, out, gpu(s.table), ints([5, 5]), offsets=ints([0, 0, 0]))
    assert (out == 9).all() and o.gpu.status() == 0
    assert np.array_equal(cache.k_codes.cpu().numpy(), s.k.codes)


def test_a_layer_as_it_is_used():
    """Projection by gemv, the token's key and value into the cache, attention, projection of the result, over some steps."""
    import torch
    from qiyas_b200 import BlockCache
    from qiyas_b200 import blocks as B
    o = H.ops()
    heads, group, dim, page, width = 2, 4, 64, 16, 512
    rows = (heads * group + 2 * heads) * dim
    w_in, w_out = (gpu(B.make_weights(B.Q8_0, r, c, seed)) for r, c, seed in ((rows, width, 1), (width, heads * group * dim, 2)))
    cache = BlockCache.empty(8, heads, page, dim)
    table = ints(np.random.default_rng(4).permutation(8).reshape(1, 8))
    x = torch.randn(width, device="cuda") * 0.05
    ks, vs = [], []
    for step in range(40):
        y = torch.empty(rows, device="cuda")
        o.GemvBlocks(B.Q8_0, w_in, x, y, rows, width, fmt_x=B.F32)
        qkv = y.view(1, -1, dim)
        q, k, v = qkv[:, :heads * group], qkv[:, heads * group:heads * group + heads], qkv[:, heads * group + heads:]
        o.CacheWrite(cache, k, v, table, ints([step]))
        out = torch.empty(1, heads * group, dim, device="cuda")
        o.CacheAttention(cache, q, out, table, ints([step + 1]))
        z = torch.empty(width, device="cuda")
        o.GemvBlocks(B.Q8_0, w_out, out, z, width, heads * group * dim, fmt_x=B.F32)
        ks.append(k.double().cpu().numpy())
        vs.append(v.double().cpu().numpy())
        # 2.5 steps of a scale that is at most 1.25 * max / 127
        kk, vv = np.concatenate(ks), np.concatenate(vs)
        stored = Cache(cache.k_codes.cpu().numpy(), cache.k_scales.cpu().numpy()).values(table[0].cpu().numpy(), 0, step + 1)
        assert np.abs(stored - kk).max() <= 2.5 * 1.25 * np.abs(kk).max() / 127
        held = Cache(cache.v_codes.cpu().numpy(), cache.v_scales.cpu().numpy()).values(table[0].cpu().numpy(), 0, step + 1)
        want = attend(q.double().cpu().numpy(), stored, held, dim ** -0.5)[0]
        assert np.abs(out.double().cpu().numpy() - want).max() <= 2e-5 * np.abs(vv).max()
        x = z / z.norm()
    assert o.gpu.status() == 0
