"""The cache operators at the edges of what they are documented to take: empty batches, scales of every kind, odd offsets, streams."""
import numpy as np
import pytest

from . import helpers as H
from .test_cache_gpu import Setup, gpu, ints, kind_of, offsets_of

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


# query heads of a head of the cache, rows of each sequence: the kernel for few rows (one token, and a few), and the tile
# kernel (more than 64 rows a head, 48 above 128 dims), one and two row tiles a unit
ROWS = [(1, [1, 1, 1, 1]), (5, [3, 1, 2, 0]), (4, [1, 40, 17, 3]), (2, [130, 3, 200, 70])]
KINDS = ["f32", "f16", "bf16"]


def check(s, kind, lens, counts, group, causal=True, window=0, absent=(), status=0, q=None, out=None, table=None, far=False, **more):
    """CacheAttention against the definition in 64 bits, for scales of any sign and size.  absent: (sequence, slot) pairs whose
    pages `table` does not name.  The tolerance, for a row with weights p: the scores are sums of dim products in f32 ((dim + 8) *
    2^-24 of scale * sum |q||k|), 2^-20 for the cut of q and the exponentials; the logarithm r of a ratio of V's scales has two ulps,
    and four sums with it round by half an ulp each: r * 2^-21, r the logarithm of the sequence's largest scale to its smallest, 85 at
    most.  The weights are cut to f16 (half a step, 2^-11; f32 lanes: two f16, 2^-21), the sums over tokens run in f32 over tokens / 128 + 64 steps: all relative
    to sum p |v|.  The output is rounded once to its type.  Below f16's normal numbers a weight is off by 2^-35 of the largest of
    p * |V's scale| that the row sees, each time a code of V, 128 at most; far: scales more than 2^85 apart may count as 0, so the
    largest of the sequence, seen or not, takes that place."""
    import torch
    o, heads, rows = H.ops(), s.heads * group, int(sum(counts))
    if q is None:
        q = s.rows(rows, heads, kind)[0]
    if out is None:
        out = torch.full_like(q, 5.0)
    lse = torch.full((rows, heads), 5.0, device="cuda")
    offsets, scale = offsets_of(counts), s.dim ** -0.5
    o.CacheAttention(s.on_gpu(), q, out, gpu(s.table if table is None else table), ints(lens), offsets=ints(offsets), causal=causal, window=window,
                     lse=lse, **more)
    assert o.gpu.status() == status
    eps, cut = torch.finfo(q.dtype).eps / 2, 2.0 ** -21 if kind == "f32" else 2.0 ** -11
    for b, (length, n) in enumerate(zip(lens, counts)):
        if n == 0:
            continue
        length = min(length, s.width * s.page)
        at = slice(int(offsets[b]), int(offsets[b]) + n)
        token = np.arange(length)
        place = (length - n + np.arange(n))[:, None]
        seen = token <= place if causal else np.ones((n, length), bool)
        if window:
            seen &= token > place - window
        for x, slot in absent:
            if x == b:
                seen &= token // s.page != slot
        k, v = (gpu(c.values(s.table[b], 0, length)).permute(1, 0, 2).repeat_interleave(group, 0) for c in (s.k, s.v))
        x, seen = q[at].double().transpose(0, 1), gpu(seen)
        scores = (x @ k.transpose(1, 2) * scale).masked_fill(~seen, -float("inf"))
        size = (x.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~seen, 0).amax(-1) if length else torch.zeros(heads, n, device="cuda")
        want_lse = torch.logsumexp(scores, -1)
        p = torch.exp(scores - want_lse.masked_fill(want_lse.isneginf(), 0)[..., None])
        want, weight = p @ v, p @ v.abs()
        held = np.abs(s.v.scales[s.table[b][:(length + s.page - 1) // s.page]]).astype(np.float64)
        held = held[(held > 0) & np.isfinite(held)]
        ratio = min(85.0, np.log2(held.max() / held.min())) if held.size else 0.0
        score = (s.dim + 8) * 2.0 ** -24 * size + 2.0 ** -20 * (1 + size) + 2.0 ** -21 * ratio
        sums = (length / 128 + 64) * 2.0 ** -24
        most = gpu(np.where(np.isfinite(s.v.scales), np.abs(s.v.scales), 0)[s.table[b][token // s.page]].astype(np.float64))     # [tokens, heads]
        most = most.t().repeat_interleave(group, 0)[:, None].expand(heads, n, length)
        most = (most if far else most.masked_fill(~seen, 0)).amax(-1, keepdim=True) if length else 0
        floor = 2.0 ** -35 * length * 128 * most
        bound = weight * (2 * score[..., None] + cut + sums) + want.abs() * eps + floor + (2.0 ** -25 if kind == "f16" else 1e-30)
        err = (out[at].double().transpose(0, 1) - want).abs()
        if kind == "f16":                                # from 65520 on (65504 and half a step) f16 rounds to infinity
            got = out[at].double().transpose(0, 1)
            err = err.masked_fill(got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound >= 65520), 0)
        assert bool((err <= bound).all()), (b, float((err / bound).max()))
        nothing = want_lse.isneginf()
        got = lse[at].double().transpose(0, 1)
        assert torch.equal(got.isneginf(), nothing) and bool((out[at].transpose(0, 1)[nothing] == 0).all())
        off = (got - want_lse).masked_fill(nothing, 0).abs()
        assert bool((off <= score + sums + 2.0 ** -21 * (1 + want_lse.masked_fill(nothing, 0).abs())).all()), b
    return out, lse


def odd_scales(s, rng, both=True):
    """Scales of zero (and -0) and below zero among the others, under codes that are not zero; the first page, the last and a
    whole sequence of zeros among them."""
    for c in (s.k, s.v) if both else (s.v,):
        pick = rng.integers(0, 10, c.scales.shape)
        c.scales[pick < 3] *= -1
        c.scales[pick == 3], c.scales[pick == 4] = 0.0, -0.0
    s.v.scales[s.table[0, 0]] = 0
    s.v.scales[s.table[0, -1]] = 0
    s.v.scales[s.table[1]] = 0
    s.v.scales[s.table[2, 0]] = -np.abs(s.v.scales[s.table[2, 0]])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group,counts", ROWS)
@pytest.mark.parametrize("page,dim", [(16, 64), (32, 128), (16, 192), (128, 96), (64, 256)])
def test_attention_over_scales_of_zero_and_below(kind, group, counts, page, dim):
    s = Setup(43 + dim, 4, 400, 2, page, dim)
    odd_scales(s, s.rng)
    for c in (s.k, s.v):
        c.scales[s.table[:, 1]] = np.abs(c.scales).max()
    check(s, kind, [400, 131, 399, 50], counts, group)
    check(s, kind, [400, 131, 399, 50], counts, group, window=70, max_length=400)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("counts", [[1, 2], [100, 40]])
def test_attention_over_nothing_but_scales_of_zero(kind, counts):
    """Codes other than zero under scales of zero are zeros: they count in the denominator and add nothing."""
    import torch
    s = Setup(44, 2, 1500, 1, 16, 128)
    s.v.scales[s.table[0]] = 0
    s.v.scales[s.table[1, :40]], s.v.scales[s.table[1, 80:]] = 0, -0.0
    check(s, kind, [1500, 1500], counts, 4)
    o, cache, n = H.ops(), s.on_gpu(), sum(counts)
    q, _ = s.rows(n, 4, kind)
    out = torch.full_like(q, 3.0)
    o.CacheAttention(cache, q, out, gpu(s.table), ints([1500, 1500]), offsets=ints([0, counts[0], n]))
    assert (out[:counts[0]] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("counts", [[3, 2], [90, 40]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_scales_that_are_not_finite_reach_the_rows_that_see_them_only(kind, counts, bad):
    import torch
    s = Setup(45, 2, 200, 1, 16, 64)
    o, n = H.ops(), sum(counts)
    q, _ = s.rows(n, 4, kind)
    window, lens = 20, [200, 150]
    want, out = torch.empty_like(q), torch.empty_like(q)
    args = (gpu(s.table), ints(lens))
    o.CacheAttention(s.on_gpu(), q, want, *args, offsets=ints([0, counts[0], n]), window=window)
    slot = (lens[0] - 1) // 16                           # of the first sequence, seen by its last rows
    s.v.scales[s.table[0, slot]] = bad
    o.CacheAttention(s.on_gpu(), q, out, *args, offsets=ints([0, counts[0], n]), window=window)
    place = np.arange(lens[0] - counts[0], lens[0])
    sees = np.zeros(n, bool)
    sees[:counts[0]] = place >= slot * 16
    sees = torch.from_numpy(sees).cuda()
    assert sees.any() and out[sees].isnan().all()
    assert torch.equal(out[~sees], want[~sees]) and o.gpu.status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group,counts", ROWS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("order", ["up", "down", "any"])
def test_attention_over_scales_of_very_different_sizes(kind, group, counts, dim, order):
    """V's scales up to 2^84 apart: a row's result is right against what it sees, whatever else its neighbours see."""
    s = Setup(46 + dim, 4, 1300, 1, 16, dim)
    size = s.rng.uniform(-74, 10, (4, s.width, 1))
    if order != "any":
        size = np.sort(size, 1)[:, ::1 if order == "up" else -1]
    s.v.scales[s.table] = np.exp2(size).astype(np.float32)
    s.v.scales[s.table[3, 2]] *= -1
    s.v.scales[s.table[2, 5:7]] = 0
    check(s, kind, [1300, 131, 399, 50], counts, group)
    check(s, kind, [1300, 131, 399, 50], counts, group, window=9)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group,counts", ROWS)
@pytest.mark.parametrize("page,dim", [(16, 64), (16, 128), (32, 192)])
@pytest.mark.parametrize("small", [2.0 ** -30, 2.0 ** -70])
def test_small_scales_beside_scales_of_zero(kind, group, counts, page, dim, small):
    """Rows that see tokens of small scales and of scales of zero, and whose neighbours see large ones: the zeros weigh in the
    denominator alone, and what the small ones give is not lost beside them."""
    s = Setup(64 + dim, 4, 1300, 2, page, dim)
    for b in range(4):
        pattern = np.array([small, 0, small, -small, 0, 0, small, 1, small, 0, 0, -1, 0, small], np.float32)
        s.v.scales[s.table[b]] = np.resize(np.roll(pattern, b), s.width)[:, None]
    for window in (9, page + 3, 0):
        check(s, kind, [1300, 131, 399, 50], counts, group, window=window)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group,counts", ROWS)
@pytest.mark.parametrize("order", ["up", "down", "any"])
def test_attention_over_scales_that_the_type_hardly_holds(kind, group, counts, order):
    """V's scales from f32's least numbers (what a write of subnormal values leaves) to 2^112, and with them values next to the largest."""
    most = 112 if kind != "f16" else 0
    s = Setup(47, 4, 1300, 2, 16, 128)
    size = s.rng.uniform(-149, most, (4, s.width, 2))
    size[:, ::5] = s.rng.uniform(-149, -140, size[:, ::5].shape)
    if order != "any":
        size = np.sort(size, 1)[:, ::1 if order == "up" else -1]
    s.v.scales[s.table] = np.exp2(size).astype(np.float32)
    check(s, kind, [1300, 131, 399, 50], counts, group, far=True)
    check(s, kind, [1300, 131, 399, 50], counts, group, far=True, window=40)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("group,counts", ROWS)
@pytest.mark.parametrize("page,dim", [(32, 256), (16, 128)])
def test_scales_that_rise_behind_what_a_row_sees(kind, group, counts, page, dim):
    """Rows that see tokens close below a scale which only their neighbours see, far above those before."""
    s = Setup(49, 4, 1300, 2, page, dim)
    steps = np.linspace(-140, 112, s.width)              # rising evenly, and by jumps
    s.v.scales[s.table, 0] = np.exp2(steps)
    s.v.scales[s.table, 1] = np.exp2(np.floor(steps / 40) * 40 + s.rng.uniform(0, 17, s.width))
    for window in (70, 0):
        out, _ = check(s, kind, [1300, 131, 399, 50], counts, group, far=True, window=window)
        assert bool(out.isfinite().all())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1, 2], [100, 40]])
def test_attention_over_values_next_to_the_largest(kind, counts):
    s = Setup(48, 2, 3000, 2, 32, 64)
    s.v.scales[:] = np.float32(3.3e38 / 128)
    s.v.codes[:] = np.abs(s.v.codes.astype(np.int32)).clip(0, 127)
    out, _ = check(s, kind, [3000, 70], counts, 4)
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [128, 256])
def test_one_and_two_row_tiles_in_turn(kind, dim):
    """Many short units one after the other in a block, with one row tile and with two: the second issuing thread sits out runs
    of them and has to be back in step with the others."""
    import torch
    rng = np.random.default_rng(6)
    counts = [int(x) for x in rng.choice([1, 30, 127, 128, 129, 200, 256], 60)]
    counts[20:40] = [1] * 20
    lens = [n + int(x) for n, x in zip(counts, rng.integers(0, 70, 60))]
    s = Setup(50, 60, 330, 8, 16, dim)
    q = s.rows(sum(counts), 8, kind)[0]
    want, lse = check(s, kind, lens, counts, 1, q=q)
    o, cache, args = H.ops(), s.on_gpu(), (gpu(s.table), ints(lens), ints(offsets_of(counts)))
    for _ in range(20):
        out, out_lse = torch.full_like(q, 5.0), torch.empty_like(lse)
        o.CacheAttention(cache, q, out, *args, lse=out_lse)
        assert torch.equal(out, want) and torch.equal(out_lse, lse)
    assert o.gpu.status() == 0


def test_calls_without_a_stream_run_on_torchs_current_one():
    """Inside a side stream's context, and while a graph is captured: behind the torch operations that made their arguments."""
    import torch
    s = Setup(51, 3, 500, 2, 16, 64)
    o, cache, table = H.ops(), s.on_gpu(), gpu(s.table)
    before, after, offsets = ints([0, 100, 250]), ints([200, 250, 500]), ints([0, 200, 350, 600])
    x = [s.rows(600, h, "f32")[0] for h in (2, 2, 4)]
    k, v, q = (torch.zeros_like(t) for t in x)
    want_k, want_out = torch.empty_like(k), torch.empty_like(q)
    o.CacheWrite(cache, x[0], x[1], table, before, offsets=offsets)
    o.CacheRead(cache, want_k, None, table, before, offsets=offsets)
    o.CacheAttention(cache, x[2], want_out, table, after, offsets=offsets)
    slow = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        cache = s.on_gpu()
        got_k, got_out = torch.zeros_like(k), torch.zeros_like(q)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(10):
                slow = slow @ slow                           # milliseconds before the rows are there
            for t, made in zip((k, v, q), x):
                t.copy_(made)
            o.CacheWrite(cache, k, v, table, before, offsets=offsets)
            o.CacheRead(cache, got_k, None, table, before, offsets=offsets)
            o.CacheAttention(cache, q, got_out, table, after, offsets=offsets)
            sums = got_k.clone(), got_out.clone()
            for t in (k, v, q):
                t.zero_()
        side.synchronize()
        assert torch.equal(sums[0], want_k) and torch.equal(sums[1], want_out)
    cache = s.on_gpu()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o.CacheWrite(cache, x[0], x[1], table, before, offsets=offsets)
        o.CacheRead(cache, got_k, None, table, before, offsets=offsets)
        o.CacheAttention(cache, x[2], got_out, table, after, offsets=offsets)
    for t in (got_k, got_out):
        t.fill_(float("nan"))
    graph.replay()
    assert torch.equal(got_k, want_k) and torch.equal(got_out, want_out) and o.gpu.status() == 0


@pytest.mark.parametrize("what", ["write", "read", "attention", "encode", "decode"])
def test_a_call_with_nothing_to_do_orders_nothing(what):
    """Gemvs of a burst run side by side; a call between them that launches nothing says nothing about when they end, so a gemv
    that reads what an earlier one writes still waits for that one."""
    import torch
    from qiyas_b200 import blocks as B
    o = H.ops()
    s = Setup(52, 1, 16, 1, 16, 32)
    cache, table, lengths = s.on_gpu(), gpu(s.table), ints([0])
    none, offsets = torch.empty(0, 1, 32, device="cuda"), ints([0, 0])
    rows, cols = 8192, 8192
    big, small, last = (gpu(B.make_weights(B.Q8_0, r, c, i)) for i, (r, c) in enumerate([(rows, cols), (64, 256), (96, rows)]))
    xs = [torch.randn(cols, device="cuda") for _ in range(12)]
    x = torch.randn(256, device="cuda")
    y, z, out = torch.empty(rows, device="cuda"), torch.empty(64, device="cuda"), torch.empty(96, device="cuda")
    nothing = {"write": lambda: o.CacheWrite(cache, none, none, table, lengths, offsets=offsets, stream=0),
               "read": lambda: o.CacheRead(cache, none, none, table, lengths, offsets=offsets, stream=0),
               "attention": lambda: o.CacheAttention(cache, none, none, table, lengths, offsets=offsets, stream=0),
               "encode": lambda: o.Back(B.Q8_0, x, small, 0), "decode": lambda: o.Lanes(B.Q8_0, small, x, 0)}[what]
    want = []
    for v in xs:
        o.GemvBlocks(B.Q8_0, big, v, y, rows, cols, fmt_x=B.F32)
        torch.cuda.synchronize()
        o.GemvBlocks(B.Q8_0, last, y, out, 96, rows, fmt_x=B.F32)
        want.append(out.clone())
    got = [torch.empty_like(out) for _ in xs]
    torch.cuda.synchronize()
    for v, g in zip(xs, got):
        o.GemvBlocks(B.Q8_0, big, v, y, rows, cols, fmt_x=B.F32)
        o.GemvBlocks(B.Q8_0, small, x, z, 64, 256, fmt_x=B.F32)
        nothing()
        o.GemvBlocks(B.Q8_0, last, y, g, 96, rows, fmt_x=B.F32)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert torch.equal(w, g)


def test_a_tile_kernel_that_was_built_otherwise_is_left_aside(tmp_path):
    """A library whose tile kernel says at set-up that it cannot run (another number of registers than its warps share out): the
    products are as they were, and attention's other kernel takes prompts."""
    import os
    import shutil
    import subprocess
    import sys
    from qiyas_b200 import build
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    objects = [build._object(src) for src in build.SOURCES if src != "attend_tiles.cu"]
    if not shutil.which(nvcc) or not all(os.path.exists(f) for f in objects):
        pytest.skip("no compiler, or the package was not built here")
    stub = tmp_path / "stub.cu"
    stub.write_text("""#include "attend_device.cuh"
namespace qb {
cudaError_t attend_tiles_init() { return cudaErrorInvalidConfiguration; }
int attend_tiles(const AttendArgs &, int, cudaStream_t) { return (int)cudaErrorInvalidConfiguration; }
}
""")
    library = tmp_path / "libother.so"
    subprocess.check_call([nvcc, *build.FLAGS[:2], "-std=c++17", "-Xcompiler", "-fPIC", "-I", build.CSRC, "-shared", "-o", str(library), str(stub)] + objects)
    program = """
import sys
from qiyas_b200 import _lib, blocks as B
_lib.LIBRARY = sys.argv[1]
import numpy as np
from tests import helpers as H
from tests.test_cache_edges_gpu import Setup, check, gpu
import torch
y = torch.empty(64, device="cuda")
H.ops().GemvBlocks(B.Q8_0, gpu(B.make_weights(B.Q8_0, 64, 256, 1)), torch.ones(256, device="cuda"), y, 64, 256, fmt_x=B.F32)
assert y.isfinite().all() and (y != 0).any()
for kind in ("f32", "f16", "bf16"):
    for dim in (64, 128, 256):
        check(Setup(53, 3, 400, 2, 16, dim), kind, [400, 131, 399], [130, 3, 200], 4)
print("as it should be")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    ran = subprocess.run([sys.executable, "-c", program, str(library)], cwd=root, capture_output=True, text=True, timeout=300)
    assert "as it should be" in ran.stdout, ran.stderr[-2000:]


def bad_cases():
    """(lengths, offsets) of 70 sequences that do not fit 100 rows or 64 tokens: one of them only, in every place."""
    for b in (0, 1, 31, 32, 33, 69):
        for what in ("offset past the rows", "offsets that fall", "length", "negative length"):
            yield b, what


@pytest.mark.parametrize("max_queries", [0, 1])
@pytest.mark.parametrize("most", [64, 4096])
@pytest.mark.parametrize("b,what", list(bad_cases()))
def test_attention_reports_what_does_not_fit(b, what, most, max_queries):
    """Whichever sequence it is, cut into shares or not: bit 4, and the others have their results."""
    import torch
    s = Setup(54, 70, 64, 1, 16, 32)
    o, cache = H.ops(), s.on_gpu()
    q = s.rows(100, 2, "f32")[0]
    lens, offsets = np.full(70, 50, np.int32), np.arange(71, dtype=np.int32)
    want, out = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    o.CacheAttention(cache, q, want, gpu(s.table), ints(lens), offsets=ints(offsets), max_queries=max_queries, max_length=most)
    assert o.gpu.status() == 0
    bad_lens, bad_offsets = lens.copy(), offsets.copy()
    if what == "length":
        bad_lens[b] = 65
    elif what == "negative length":
        bad_lens[b] = -1
    elif what == "offset past the rows":
        bad_offsets[b + 1:] = 101 + np.arange(70 - b)
    else:
        bad_offsets[b + 1] = b - 1
    o.CacheAttention(cache, q, out, gpu(s.table), ints(bad_lens), offsets=ints(bad_offsets), max_queries=max_queries, max_length=most)
    assert o.gpu.status() == 16
    assert torch.equal(out[:max(0, b - 1)], want[:max(0, b - 1)])
    if "length" in what:
        assert torch.equal(out[b + 1:70], want[b + 1:70])
    assert (out[70:] == 7).all() or what == "offset past the rows"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("counts,dim", [([1, 1, 1], 128), ([1, 1, 1], 256), ([100, 3, 140], 64), ([60, 3, 40], 192)])
def test_a_workspace_of_the_callers_own(kind, counts, dim):
    """The size asked for is enough, nothing behind it is touched, less is refused, and one serves calls (and replays) in turn."""
    import torch
    s = Setup(55, 3, 3000, 2, 16, dim)
    o, cache, lens = H.ops(), s.on_gpu(), ints([3000, 1, 2049])
    q = s.rows(sum(counts), 8, kind)[0]
    args, bounds = (gpu(s.table), lens), dict(offsets=ints(offsets_of(counts)), max_queries=max(counts), max_length=3000)
    want, out = torch.empty_like(q), torch.full_like(q, 5.0)
    o.CacheAttention(cache, q, want, *args, **bounds)
    need = o.attention_workspace_bytes(cache, q, *args, **bounds)
    assert need > 0
    room = torch.full((need + 4096,), 0xa5, dtype=torch.uint8, device="cuda")
    for extra in (dict(workspace=room[:need]), dict(workspace=room.data_ptr(), workspace_bytes=need)):
        for _ in range(2):
            out.fill_(5.0)
            o.CacheAttention(cache, q, out, *args, **bounds, **extra)
            assert torch.equal(out, want)
    assert (room[need:] == 0xa5).all()
    for bad in (dict(workspace=room[:need - 1]), dict(workspace=room[8:]), dict(workspace=room, workspace_bytes=need - 1), dict(workspace=room.cpu()),
                dict(workspace=room[::2])):
        with pytest.raises(ValueError):
            o.CacheAttention(cache, q, out, *args, **bounds, **bad)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], [torch.empty_like(q) for _ in range(2)]
    for g, t in zip(graphs, outs):
        with torch.cuda.graph(g):
            o.CacheAttention(cache, q, t, *args, **bounds, workspace=room[:need])
    for _ in range(5):
        for g, t in zip(graphs, outs):
            t.fill_(5.0)
            g.replay()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    short = o.attention_workspace_bytes(cache, q[:1], args[0][:1], lens[:1], max_length=40)
    assert short == 0 and o.gpu.status() == 0            # short sequences are not cut


# ------------------------------------------------------------------------------------------------ the tile kernel's own paths

TILES = [(2, [90, 40], [400, 70]), (1, [260, 129], [700, 129]), (4, [70, 1], [1300, 1100])]        # query heads a head, rows, tokens


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group,counts,lens", TILES)
@pytest.mark.parametrize("dim", [48, 128, 192])
def test_tiles_with_strides(kind, group, counts, lens, dim):
    """q and out as slices of wider rows, with a head order of their own, and from bases that are not 16-byte aligned; what lies
    between the rows of out stays."""
    import torch
    s = Setup(56, 2, max(lens), 2, 32, dim)
    rows, heads = sum(counts), 2 * group
    x = s.rows(rows, heads + 2, kind, 2.0)[0]
    flat = torch.cat([torch.zeros(1, dtype=x.dtype, device="cuda"), x.reshape(-1)])
    qs = (x[:, 1:heads + 1], flat[1:].view(rows, heads + 2, dim)[:, 1:heads + 1], x.transpose(0, 1).contiguous().transpose(0, 1)[:, 1:heads + 1])
    for i, q in enumerate(qs):
        room = torch.full((rows * (heads + 2) * dim + 1,), 9.0, dtype=x.dtype, device="cuda")
        whole = (room[1:].view(rows, heads + 2, dim), room[:-1].view(rows, heads + 2, dim), room[:-1].view(heads + 2, rows, dim).transpose(0, 1))[i]
        out = whole[:, 1:heads + 1]
        check(s, kind, lens, counts, group, q=q, out=out, window=0 if i else 90)
        assert (whole[:, 0] == 9).all() and (whole[:, heads + 1] == 9).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group,counts,lens", TILES)
@pytest.mark.parametrize("page,dim", [(16, 64), (16, 128), (32, 256), (128, 192)])
def test_tiles_with_pages_that_are_not_there(kind, group, counts, lens, page, dim):
    """Pages the table does not name, inside tiles, whole tiles and the first and last: left out, and reported."""
    s = Setup(57, 2, max(lens), 2, page, dim)
    table, absent = s.table.copy(), []
    for b, length in enumerate(lens):
        last = (length - 1) // page
        for slot in {0, 3, 4, 5, 6, 7, 11, last} if b == 0 else {last // 2}:
            if slot <= last:
                table[b, slot] = -1 if slot % 2 else s.pages + slot
                absent.append((b, slot))
    check(s, kind, lens, counts, group, table=table, absent=absent, status=16)
    check(s, kind, lens, counts, group, table=table, absent=absent, status=16, window=page)      # some rows see nothing else


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group,counts,lens", TILES)
@pytest.mark.parametrize("dim", [64, 192])
def test_tiles_with_pages_missing_and_scales_of_all_kinds(kind, group, counts, lens, dim):
    s = Setup(58, 4, max(lens), 2, 16, dim)
    odd_scales(s, s.rng)
    table, absent = s.table.copy(), [(0, 2), (0, 17), (1, 1), (2, 0), (2, 40)]
    lens, counts = [*lens, *lens[::-1]], [*counts, 30, 2]
    for b, slot in absent:
        if slot < s.width:
            table[b, slot] = -7
    absent = [(b, slot) for b, slot in absent if slot < s.width]
    check(s, kind, lens, counts, group, table=table, absent=absent, status=16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group,counts,lens", TILES)
@pytest.mark.parametrize("dim", [128, 256])
def test_tiles_with_nan_rows_and_unwritten_places(kind, group, counts, lens, dim):
    """NaN and infinities in rows of q stay in their rows; codes and scales that no row sees do not matter."""
    import torch
    s = Setup(59, 2, max(lens) + 40, 2, 16, dim)
    o, cache, heads, rows = H.ops(), s.on_gpu(), 2 * group, sum(counts)
    q = s.rows(rows, heads, kind)[0]
    args = gpu(s.table), ints(lens), ints(offsets_of(counts))
    want, out = torch.empty_like(q), torch.empty_like(q)
    lse, want_lse = (torch.empty(rows, heads, device="cuda") for _ in range(2))
    o.CacheAttention(cache, q, want, *args, lse=want_lse)
    used = np.concatenate([s.table[b, :(n + 15) // 16] for b, n in enumerate(lens)])
    rest = torch.from_numpy(np.setdiff1d(np.arange(s.pages), used)).cuda()
    for c in (cache.k_scales, cache.v_scales):
        c[rest] = float("nan")
    for c in (cache.k_codes, cache.v_codes):
        c[rest] = 127
        for b, n in enumerate(lens):
            if n % 16:
                c[int(s.table[b, n // 16]), :, n % 16:] = -128
    o.CacheAttention(cache, q, out, *args, lse=lse)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    marks = [(0, 0, float("nan")), (rows - 1, heads - 1, float("inf")), (rows // 2, 1, -float("inf")), (3, heads - 1, float("nan"))]
    for r, h, x in marks:
        q[r, h, 5] = x
    o.CacheAttention(cache, q, out, *args, lse=lse)
    for r, h, _ in marks:
        assert out[r, h].isnan().all() and lse[r, h].isnan()
        out[r, h], lse[r, h] = want[r, h], want_lse[r, h]
    assert torch.equal(out, want) and torch.equal(lse, want_lse) and o.gpu.status() == 0


@pytest.mark.parametrize("dim", [64, 256])
def test_tiles_over_a_dominant_token(dim):
    """One token takes nearly all the weight and its value is zero: the small weights' sum is left, in every row.  The tolerance is
    `check`'s: scores of up to 15.3, two f16 a weight, and 2^-35 of the largest weight for each token."""
    s = Setup(60, 1, 2048, 1, 16, dim)
    s.v.scales[:] = 0.01
    p = s.table[0, 0]
    s.v.codes[p, 0, 0] = 0
    s.k.codes[p, 0, 0], s.k.scales[p, 0] = 127, 0.05
    import torch
    o, n = H.ops(), 150
    q = torch.full((n, 1, dim), 0.3 * 8 / dim ** 0.5, device="cuda")
    out = torch.empty_like(q)
    o.CacheAttention(s.on_gpu(), q, out, gpu(s.table), ints([2048]), offsets=ints([0, n]))
    k, v = (gpu(c.values(s.table[0], 0, 2048))[:, 0] for c in (s.k, s.v))
    scores = (q[:, 0].double() @ k.t() * dim ** -0.5).masked_fill(torch.arange(2048, device="cuda") > 2048 - n + torch.arange(n, device="cuda")[:, None], -float("inf"))
    weights = torch.softmax(scores, -1)
    assert weights[:, 0].min() > 0.99
    score = ((dim + 8) * 2.0 ** -24 + 2.0 ** -20) * 16.3
    bound = weights @ v.abs() * (2 * score + 2.0 ** -21 + (2048 / 128 + 64) * 2.0 ** -24) + 2.0 ** -35 * 2048 * 128 * 0.01
    assert bool(((out[:, 0].double() - weights @ v).abs() <= bound).all())


@pytest.mark.parametrize("page,dim", [(16, 16), (16, 128), (32, 64)])
def test_scales_that_grow_with_every_token(page, dim):
    """Blocks that a single warp writes, whose scale is read by all lanes and replaced by one, again and again: bit for bit."""
    s = Setup(61, 200, page, 3, page, dim)
    o, cache, table = H.ops(), s.on_gpu(), gpu(s.table)
    rng = s.rng
    for at in range(page):
        x = (rng.standard_normal((200, 3, dim)) * np.exp(at * rng.uniform(0, 0.5, (200, 3, 1)))).astype(np.float32)
        t = gpu(x)
        o.CacheWrite(cache, t, -t, table, ints([at] * 200))
        for b in range(200):
            p = s.table[b, 0]
            for h in range(3):
                s.k.codes[p, h], s.k.scales[p, h] = written(s.k.codes[p, h], s.k.scales[p, h], at, x[b:b + 1, h])
    pages = s.table[:, 0]
    assert np.array_equal(cache.k_codes.cpu().numpy()[pages], s.k.codes[pages]) and np.array_equal(cache.k_scales.cpu().numpy()[pages], s.k.scales[pages])
    assert np.array_equal(cache.v_scales.cpu().numpy()[pages], s.k.scales[pages]) and o.gpu.status() == 0


def test_codes_of_subnormal_scales_are_held_to_127():
    """Where the scale is f32's least number its rounding can leave quotients above 127."""
    s = Setup(62, 1, 16, 1, 16, 16)
    o, cache = H.ops(), s.on_gpu()
    least = np.float32(2.0 ** -149)
    x = (np.array([150, -150, 190, -190, 127, 100, -3, 0] * 2, np.float32) * least).reshape(1, 1, 16)
    o.CacheWrite(cache, gpu(x), gpu(x), gpu(s.table), ints([0]))
    p = int(s.table[0, 0])
    assert cache.k_scales[p, 0].item() == least and o.gpu.status() == 0
    assert cache.k_codes[p, 0, 0].tolist() == [127, -127, 127, -127, 127, 100, -3, 0] * 2


@pytest.mark.parametrize("op", ["write", "read", "rows", "tiles"])
@pytest.mark.parametrize("least", [-2 ** 31, -2 ** 31 + 1, -2 ** 31 + 39, -1, 2 ** 31 - 1])
def test_offsets_of_any_32_bits(op, least):
    """Offsets at both ends of their type: no rows for the sequences they are of, nothing touched outside the rows given."""
    import torch
    from qiyas_b200 import BlockCache
    s = Setup(63, 3, 200, 2, 16, 64)
    o, heads, rows, guard = H.ops(), 2 if op in ("write", "read") else 4, 90, 1 << 16
    room = torch.full((rows * heads * 64 + 2 * guard,), 7.0, device="cuda")
    x, table = room[guard:-guard].view(rows, heads, 64), gpu(s.table)
    x.copy_(torch.randn(rows, heads, 64, device="cuda"))
    codes = torch.full((s.k.codes.size + 2 * guard,), 7, dtype=torch.int8, device="cuda")
    scales = torch.full((s.k.scales.size + 2 * guard,), 7.0, device="cuda")
    codes[guard:-guard], scales[guard:-guard] = gpu(s.k.codes).reshape(-1), gpu(s.k.scales).reshape(-1)
    cache = BlockCache(codes[guard:-guard].view(s.k.codes.shape), gpu(s.v.codes), scales[guard:-guard].view(s.k.scales.shape), gpu(s.v.scales))
    for offsets in ([0, 40, least, 90], [0, least, least, 90], [least, 40, 60, least], [40, least, 50, 90]):
        if op == "write":
            o.CacheWrite(cache, x, x, table, ints([0, 10, 20]), offsets=ints(offsets))
        elif op == "read":
            o.CacheRead(cache, x, None, table, ints([0, 10, 20]), offsets=ints(offsets))
        else:
            q = torch.randn(rows, heads, 64, device="cuda")
            o.CacheAttention(cache, q, x, table, ints([200, 150, 100]), offsets=ints(offsets), max_queries=1 if op == "rows" else 0)
        assert o.gpu.status() == 16
        assert (room[:guard] == 7).all() and (room[-guard:] == 7).all()
        assert (codes[:guard] == 7).all() and (codes[-guard:] == 7).all() and (scales[:guard] == 7).all() and (scales[-guard:] == 7).all()
