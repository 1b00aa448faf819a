"""What is measured of the cache operators: keys and values quantised as they are written into a paged cache of int8 codes
with one f32 scale for each block of tokens and head, the same read back, and attention over that cache.

A cache is four tensors: codes of K and of V, int8 [pages, heads, page, dim], and scales of K and of V, f32 [pages, heads];
a stored value is code * scale.  `table[b, i]` is the page that holds tokens i * page .. of sequence b.  Rows of all
sequences lie behind one another, sequence b's at offsets[b] .. offsets[b + 1].

The definition of a write.  Let a be the largest magnitude that a call writes into a block (one page, one head), and s the
block's scale if it holds earlier tokens of the sequence, else 0.  With f32 arithmetic n = a / 127; where n <= s the scale
stays s, else it becomes max(n, 1.25 * s), and the earlier tokens' codes c become the integer nearest c * s / scale.  New
values x become the integer nearest x / scale (ties to even, both quotients exact).  A block of zeros has scale 0.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ops = None


def _case(name, op, kind, sequences, heads, group, dim, page, lo, hi, new_lo, new_hi, window=0, causal=True):
    """lo..hi: tokens of a sequence that are in the cache before the call's own; new_lo..new_hi: rows of a sequence in the call."""
    return dict(name=name, op=op, type=kind, sequences=sequences, heads=heads, group=group, dim=dim, page=page, lo=lo, hi=hi,
                new_lo=new_lo, new_hi=new_hi, window=window, causal=causal)


def listed():
    return [
        # one user's next token: its key and value go into a page that is partly full
        _case("write-one", "write", "bf16", 1, 8, 1, 128, 16, 1000, 1000, 1, 1),
        # a serving step: one token of each of 64 sequences of very different lengths
        _case("write-step", "write", "bf16", 64, 8, 1, 128, 16, 100, 8000, 1, 1),
        # prompts of four users, one after the other in one batch, the cache still empty
        _case("write-prompt", "write", "f16", 4, 8, 1, 128, 64, 0, 0, 500, 8192),
        # pieces of prompts behind what is there already, f32 lanes, sizes that fit nothing
        _case("write-odd", "write", "f32", 7, 5, 1, 80, 32, 3, 777, 1, 333),
        # kept prefixes read back, to be moved to another machine or another format
        _case("read-prefix", "read", "bf16", 16, 8, 1, 128, 16, 0, 300, 1000, 4096),
        # a window of a few sequences read back in f32
        _case("read-odd", "read", "f32", 5, 3, 1, 96, 128, 1, 900, 7, 1501),
        # the first tokens of an answer: a short prompt behind it, latency is what counts
        _case("attend-short", "attend", "bf16", 1, 8, 4, 128, 16, 128, 128, 1, 1),
        # a serving step over 32 sequences
        _case("attend-step", "attend", "bf16", 32, 8, 4, 128, 16, 500, 8000, 1, 1),
        # one user with a very long document
        _case("attend-long", "attend", "f16", 1, 8, 8, 128, 64, 131071, 131071, 1, 1),
        # a step of a model with as many key heads as query heads, f32 lanes, a sliding window
        _case("attend-window", "attend", "f32", 16, 32, 1, 64, 32, 20, 4095, 1, 1, window=1024),
        # five guessed tokens of each sequence looked at in one go
        _case("attend-guess", "attend", "f16", 8, 4, 8, 256, 32, 1500, 6000, 5, 5),
        # pieces of two prompts, each attending to what was cached before it and to itself
        _case("attend-prompt", "attend", "bf16", 2, 8, 4, 128, 64, 1000, 4096, 3000, 4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        op = rng.choice(["write", "write", "read", "attend", "attend", "attend", "attend"])
        kind = rng.choice(["f32", "f16", "bf16", "bf16"])
        heads, dim, page = _log(rng, 1, 32), rng.choice([64, 80, 96, 112, 128, 128, 128, 192, 256]), rng.choice([16, 32, 64, 128])
        sequences = _log(rng, 1, 100)
        hi = _log(rng, 1, 60000) if rng.random() < 0.9 else 0
        lo = rng.randint(0, hi)
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 16]) if op == "attend" else 1
        new_hi = _log(rng, 1, 6000) if op != "attend" or rng.random() < 0.5 else _log(rng, 1, 12)
        if op != "read" and rng.random() < 0.35:
            new_hi = 1
        new_lo = rng.randint(0, new_hi) if rng.random() < 0.5 else new_hi
        causal = op != "attend" or rng.random() < 0.85
        window = _log(rng, 1, 5000) if op == "attend" and causal and rng.random() < 0.25 else 0
        case = _case("", op, kind, sequences, heads, group, dim, page, lo, hi, new_lo, new_hi, window, causal)
        del case["name"]
        need = work(case)
        # the plain form holds the whole of its padded scores; the padding is bounded here, not what a case computes
        padded = sequences * heads * group * new_hi * (hi + new_hi) * 4 if op == "attend" else 0
        cached = sequences * heads * dim * (hi + new_hi) * 8
        rows = sum(_sizes(case)[1])
        if rows and need["bytes"] <= most[0] and need["flops"] <= most[1] and padded <= 5e9 and cached <= 9e9:
            return case


def _spread(lo, hi, count, salt):
    """`count` numbers over lo..hi, the last one hi."""
    return [hi if i == count - 1 else lo + int((hi - lo) * ((0.6180339887 * (i + 1) + salt) % 1.0) + 0.5) for i in range(count)]


def _sizes(case):
    """Tokens of each sequence in the cache before the call's rows, and rows of each sequence."""
    return _spread(case["lo"], case["hi"], case["sequences"], 0.37), _spread(case["new_lo"], case["new_hi"], case["sequences"], 0.11)


def _first_of_page(case):
    """Where each sequence's first page that a write touches begins."""
    before, new = _sizes(case)
    return [b // case["page"] * case["page"] if n else b for b, n in zip(before, new)]


def work(case):
    before, new = _sizes(case)
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    page, dim, heads, group = case["page"], case["dim"], case["heads"], case["group"]
    row = heads * dim
    if case["op"] == "read":
        pages = sum((b % page + n + page - 1) // page for b, n in zip(before, new))
        return {"bytes": 2 * (sum(new) * row * (1 + size) + pages * heads * 4), "flops": 2 * sum(new) * row}
    if case["op"] == "write":      # and what it touched read back
        pages = sum((b % page + n + page - 1) // page for b, n in zip(before, new))
        back = sum(b + n - f for b, n, f in zip(before, new, _first_of_page(case)))
        return {"bytes": 2 * (sum(new) * row * (size + 1) + back * row * (1 + size) + 2 * pages * heads * 4), "flops": 2 * (4 * sum(new) + back) * row}
    read = pairs = 0
    for b, n in zip(before, new):
        if not n:
            continue
        if not case["causal"]:
            read, pairs = read + b + n, pairs + n * (b + n)
        elif not case["window"]:
            read, pairs = read + b + n, pairs + n * b + n * (n + 1) // 2
        else:
            w = case["window"]
            read += min(b + n, w + n - 1)
            short = max(0, min(n, w - b))          # rows that see fewer tokens than the window holds
            pairs += short * b + short * (short + 1) // 2 + (n - short) * w
    pages = 2 * heads * 4 * (read // page + 1)
    return {"bytes": 2 * read * row + pages + sum(new) * heads * group * (2 * dim * size + 4), "flops": 4 * pairs * heads * group * dim}


def _made(case, seed):
    """Cache, table and rows of a case: values as layers produce them, a few channels much larger than the others."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    heads, dim, page = case["heads"], case["dim"], case["page"]
    before, new = _sizes(case)
    held = [b + n for b, n in zip(before, new)]
    width = max(b // page for b in held) + 2
    count = case["sequences"] * width
    cache = {}
    step = max(1, (64 << 20) // (heads * page * dim))
    for name, spread in (("k", 1.0), ("v", 0.6)):
        codes = torch.empty(count, heads, page, dim, dtype=torch.int8, device="cuda")
        scales = torch.empty(count, heads, dtype=torch.float32, device="cuda")
        gain = spread * (1 + 3 * (torch.rand(heads, 1, dim, generator=g, device="cuda") > 0.97))
        for at in range(0, count, step):
            x = torch.randn(min(step, count - at), heads, page, dim, generator=g, device="cuda") * gain
            s = x.abs().amax((2, 3)) / 127
            codes[at:at + step] = torch.round(x / s[:, :, None, None]).clamp_(-127, 127).to(torch.int8)
            scales[at:at + step] = s
        cache[name + "_codes"], cache[name + "_scales"] = codes, scales
    table = torch.randperm(count, generator=g, device="cuda").to(torch.int32).view(case["sequences"], width)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    rows = offsets[-1]
    s = dict(cache, case=case, table=table, rows=rows, page=page, most_new=max(new), most_held=max(held),
             before=torch.tensor(before, dtype=torch.int32, device="cuda"), held=torch.tensor(held, dtype=torch.int32, device="cuda"),
             offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    kind = TYPES[case["type"]]
    if case["op"] == "write":
        for name, spread in (("k", 1.0), ("v", 0.6)):
            s[name] = (torch.randn(rows, heads, dim, generator=g, device="cuda") * spread * 1.1).to(kind)
        first = _first_of_page(case)
        back = [0]
        for f, h in zip(first, held):
            back.append(back[-1] + h - f)
        s["first"], s["back_rows"] = torch.tensor(first, dtype=torch.int32, device="cuda"), back[-1]
        s["back"] = torch.tensor(back, dtype=torch.int32, device="cuda")
    elif case["op"] == "attend":
        s["q"] = (torch.randn(rows, heads * case["group"], dim, generator=g, device="cuda") * 1.5).to(kind)
        s["scale"] = 1 / math.sqrt(dim)
    return s


def prepare(case, seed):
    s = _made(case, seed)
    kind = TYPES[case["type"]]
    # the buffers that a user's program keeps for its results
    if case["op"] == "attend":
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["rows"], s["q"].shape[1], dtype=torch.float32, device="cuda")
    else:
        rows = s["back_rows"] if case["op"] == "write" else s["rows"]
        s["k_out"] = torch.empty(rows, case["heads"], case["dim"], dtype=kind, device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    return s


# ------------------------------------------------------------------------------------------------ the plain forms

def _plain_write(s, name):
    """Every page that a sequence touches at once: [sequences, touched pages, page, heads, dim]."""
    codes, scales, page, new = s[name + "_codes"], s[name + "_scales"], s["page"], s[name]
    before, held = s["before"].long(), s["held"].long()
    touched = (s["most_new"] + 2 * page - 2) // page
    first = before // page
    slot = first[:, None] + torch.arange(touched, device="cuda")
    inside = slot < s["table"].shape[1]
    ids = s["table"].gather(1, slot.clamp(max=s["table"].shape[1] - 1)).long()
    at = slot[:, :, None] * page + torch.arange(page, device="cuda")
    is_old, is_new = at < before[:, None, None], (at >= before[:, None, None]) & (at < held[:, None, None])
    row = (s["offsets"][:-1].long()[:, None, None] + at - before[:, None, None]).clamp(0, s["rows"] - 1)
    x = new[row].float() * is_new[..., None, None]
    old_codes, old = codes[ids], scales[ids]                                     # [b, t, heads, page, dim], [b, t, heads]
    old_scale = torch.where(is_old.any(2)[..., None], old, torch.zeros_like(old))
    need = x.abs().amax((2, 4)) / 127
    scale = torch.where(need <= old_scale, old_scale, torch.maximum(need, old_scale * 1.25))
    wide = torch.where(scale > 0, scale, torch.ones_like(scale)).double()[..., None, None]
    x = torch.round(x.transpose(2, 3).double() / wide)
    kept = torch.round(old_codes.double() * old_scale.double()[..., None, None] / wide)
    is_new, is_old = is_new[:, :, None, :, None], is_old[:, :, None, :, None]
    result = torch.where(is_new, x, torch.where(is_old, kept, old_codes.double())).to(torch.int8)
    writes = is_new.any(3).any(3) & inside[:, :, None]                           # [b, t, 1]: others keep what they have
    result = torch.where(writes[..., None, None], result, old_codes)
    scale = torch.where(writes, scale, old)
    # a slot past the table's end repeats its last page: it takes that page's own result
    last = (s["table"].shape[1] - 1 - first).clamp(0, touched - 1)
    pick = torch.minimum(torch.arange(touched, device="cuda")[None], last[:, None])
    result = result.gather(1, pick[:, :, None, None, None].expand_as(result))
    scale = scale.gather(1, pick[:, :, None].expand_as(scale))
    codes[ids.view(-1)] = result.flatten(0, 1)
    scales[ids.view(-1)] = scale.flatten(0, 1)


def _plain_read(s, name, first, offsets, rows, kind):
    counts = (offsets[1:] - offsets[:-1]).long()
    b = torch.repeat_interleave(torch.arange(counts.numel(), device="cuda"), counts, output_size=rows)
    at = torch.arange(rows, device="cuda") - offsets[:-1].long()[b] + first.long()[b]
    ids = s["table"][b, at // s["page"]].long()
    return (s[name + "_codes"][ids, :, at % s["page"]].float() * s[name + "_scales"][ids][..., None]).to(kind)


def _plain_attend(s):
    case, q, page = s["case"], s["q"], s["page"]
    heads, group, dim = case["heads"], case["group"], case["dim"]
    pages = (s["most_held"] + page - 1) // page
    ids = s["table"][:, :pages].long()
    length = pages * page

    def whole(name):                                                             # [sequences, heads, tokens, dim]
        x = s[name + "_codes"][ids].float() * s[name + "_scales"][ids][..., None, None]
        return x.transpose(1, 2).reshape(ids.shape[0], heads, length, dim)

    held = s["held"].long()
    new = (s["offsets"][1:] - s["offsets"][:-1]).long()
    i = torch.arange(s["most_new"], device="cuda")
    row = (s["offsets"][:-1].long()[:, None] + i).clamp(max=s["rows"] - 1)       # [sequences, queries]
    x = q[row].float().view(ids.shape[0], s["most_new"], heads, group, dim).permute(0, 2, 3, 1, 4)
    x = x.reshape(ids.shape[0], heads, group * s["most_new"], dim)
    scores = torch.matmul(x, whole("k").transpose(2, 3)).mul_(s["scale"]).view(ids.shape[0], heads, group, s["most_new"], length)
    at, token = held[:, None] - new[:, None] + i, torch.arange(length, device="cuda")
    seen = (token < held[:, None, None]).expand(-1, s["most_new"], -1)
    if case["causal"]:
        seen = seen & (token <= at[..., None])
    if case["window"]:
        seen = seen & (token > at[..., None] - case["window"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    lse = (total.log() + top).squeeze(-1)
    out = torch.matmul(weights.view(ids.shape[0], heads, group * s["most_new"], length), whole("v"))
    out = out.view(ids.shape[0], heads, group, s["most_new"], dim) / torch.where(total > 0, total, torch.ones_like(total))
    # back to rows behind one another
    b = torch.repeat_interleave(torch.arange(new.numel(), device="cuda"), new, output_size=s["rows"])
    i = torch.arange(s["rows"], device="cuda") - s["offsets"][:-1].long()[b]
    return out.permute(0, 3, 1, 2, 4)[b, i].reshape(q.shape).to(q.dtype), lse.permute(0, 3, 1, 2)[b, i].reshape(s["rows"], -1)


def run(s):
    case = s["case"]
    if own:
        return _run_own(s)
    kind = TYPES[case["type"]]
    if case["op"] == "attend":
        out, lse = _plain_attend(s)
        return {"out": out, "lse": lse}
    if case["op"] == "read":
        return {n: _plain_read(s, n, s["before"], s["offsets"], s["rows"], kind) for n in ("k", "v")}
    _plain_write(s, "k")
    _plain_write(s, "v")
    return {n: _plain_read(s, n, s["first"], s["back"], s["back_rows"], kind) for n in ("k", "v")}


def _run_own(s):
    """The calls that a user's program makes."""
    global _ops
    from qiyas_b200 import BlockCache, GpuOps
    if _ops is None:
        _ops = GpuOps(device=0)
    case = s["case"]
    cache = BlockCache(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
    if case["op"] == "attend":
        _ops.CacheAttention(cache, s["q"], s["out"], s["table"], s["held"], offsets=s["offsets"], max_queries=s["most_new"],
                            max_length=s["most_held"], scale=s["scale"], causal=case["causal"], window=case["window"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if case["op"] == "write":
        _ops.CacheWrite(cache, s["k"], s["v"], s["table"], s["before"], offsets=s["offsets"])
        _ops.CacheRead(cache, s["k_out"], s["v_out"], s["table"], s["first"], offsets=s["back"])
    else:
        _ops.CacheRead(cache, s["k_out"], s["v_out"], s["table"], s["before"], offsets=s["offsets"])
    return {"k": s["k_out"], "v": s["v_out"]}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    """A sequence at a time, in f64."""
    s = _made(case, seed)
    before, new = _sizes(case)
    page, table = case["page"], s["table"].cpu().tolist()

    def stored(name, b, first, last):
        """Tokens first..last of sequence b, [heads, tokens, dim]."""
        if first >= last:
            return torch.zeros(case["heads"], 0, case["dim"], dtype=torch.float64, device="cuda")
        lo, hi = first // page, (last + page - 1) // page
        ids = torch.tensor(table[b][lo:hi], device="cuda")
        x = s[name + "_codes"][ids].double().mul_(s[name + "_scales"][ids].double()[..., None, None])
        return x.permute(1, 0, 2, 3).flatten(1, 2)[:, first - lo * page:last - lo * page]

    if case["op"] == "attend":
        outs, lses, at = [], [], 0
        for b, (old, n) in enumerate(zip(before, new)):
            if not n:
                continue
            k, v = stored("k", b, 0, old + n), stored("v", b, 0, old + n)
            token = torch.arange(old + n, device="cuda")
            block = max(1, (256 << 20) // (case["heads"] * case["group"] * (old + n)))
            for i in range(0, n, block):
                m = min(block, n - i)
                q = s["q"][at + i:at + i + m].double().view(m, case["heads"], case["group"], -1).permute(1, 2, 0, 3).flatten(1, 2)
                e = (q @ k.transpose(1, 2) * s["scale"]).view(case["heads"], case["group"], m, old + n)
                place = (torch.arange(m, device="cuda") + old + i)[:, None]
                hidden = torch.zeros(m, old + n, dtype=torch.bool, device="cuda")
                if case["causal"]:
                    hidden |= token > place
                if case["window"]:
                    hidden |= token <= place - case["window"]
                e.masked_fill_(hidden, -math.inf)
                z = torch.logsumexp(e, -1, keepdim=True)
                o = (e - z).exp_().flatten(1, 2) @ v
                outs.append(o.view(case["heads"], case["group"], m, -1).permute(2, 0, 1, 3).flatten(1, 2))
                lses.append(z.squeeze(-1).permute(2, 0, 1).flatten(1, 2))
            at += n
        return {"out": torch.cat(outs), "lse": torch.cat(lses)}

    if case["op"] == "read":
        return {n: torch.cat([stored(n, b, f, f + r).transpose(0, 1) for b, (f, r) in enumerate(zip(before, new))]) for n in ("k", "v")}

    result = {}
    for name in ("k", "v"):
        parts, at = [], 0
        for b, (old, n) in enumerate(zip(before, new)):
            done = 0
            while done < n:
                start = old + done
                p, inside = start // page, start % page
                m = min(page - inside, n - done)
                x = s[name][at + done:at + done + m].double().transpose(0, 1)                # [heads, m, dim]
                need = (x.abs().amax((1, 2)).float() / 127)
                had = s[name + "_scales"][table[b][p]] if inside else torch.zeros_like(need)
                scale = torch.where(need <= had, had, torch.maximum(need, had * 1.25)).double()[:, None, None]
                safe = torch.where(scale > 0, scale, torch.ones_like(scale))
                c = s[name + "_codes"][table[b][p]][:, :inside].double()
                codes = torch.cat([torch.round(c * had.double()[:, None, None] / safe), torch.round(x / safe)], 1)
                parts.append((codes * scale).transpose(0, 1))
                done += m
            at += n
        result[name] = torch.cat(parts)
    return result
