// What the attention kernels share: how a call's work is cut into shares, the rows' limits, and the products' operands.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "cache.h"
#include "cache_device.cuh"

namespace qb {

constexpr float NOTHING = -1e30f;              // a maximum over nothing (finite: differences of two of them are 0)
constexpr int LEAST_TOKENS = 256;              // tokens a share has at least
// What a unit costs a block besides its tiles, in tiles of TT tokens: its rows of q, the join of its sums.  Measured: 3000
// cycles at 350 a tile in attend_rows.cu (32 tokens a tile), 25000 at 7000 in attend_tiles.cu.  The line of work below
// counts it, or a block that gets many short sequences ends long after the others.
__host__ __device__ constexpr int unit_pad(int tt) { return tt == 32 ? 8 : 10; }

struct AttendArgs {
    qb200_sequences_t seq;
    qb200_lanes_t q, out;
    float *lse;
    const int8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    int pages, heads, dim, log_page, group, q_heads, causal, window;
    float scale;
    int q_wide, out_wide;
    int whole;                                 // units are not cut: block c takes units c, c + grid, ...
    int chunks;                                // units a sequence and head, by the caller's bound
    int grid;
    uint32_t group_magic;                      // n / group = n * magic >> shift for 0 <= n < 2^31
    int group_shift;
    void *workspace;
    int *status;
};

__device__ __forceinline__ int by_group(const AttendArgs &p, int n) { return (int)(((uint64_t)(uint32_t)n * p.group_magic) >> p.group_shift); }

cudaError_t attend_rows_init();
int attend_rows(const AttendArgs &args, int type, int r, const CUtensorMap &kmap, const CUtensorMap &vmap, cudaStream_t stream);
cudaError_t attend_tiles_init();
int attend_tiles(const AttendArgs &args, int type, cudaStream_t stream);

// R rows of one head (R, and TT tokens a tile: the kernel's) of one sequence: rows r0 .. r1 - 1 of its queries x group, and the tokens they see together.
struct Unit {
    int b, h, rc;
    int row, n, len;                           // the sequence: first row, rows, tokens
    int r0, r1;
    int lo, hi;                                // tokens that any of the rows sees
    int t0, nt;                                // tiles: at least one, so that rows that see nothing are written too
};

__host__ __device__ constexpr size_t part_floats(int r, int dim) { return (size_t)r * (dim + 2); }

struct Sequence { int row, n, len; };          // first row, rows, tokens: held to what there is

__device__ __forceinline__ Sequence sequence_at(const AttendArgs &p, int b)
{
    Sequence s;
    bool bad;
    seq_rows(p.seq, b, s.row, s.n, bad);
    s.len = p.seq.lengths[b];
    const int most = p.seq.width << p.log_page;
    bad |= s.len < 0 || s.len > most;
    s.len = max(0, min(s.len, most));
    if (bad) atomicOr(p.status, STATUS_CACHE_RANGE);           // (by any lane: where a share is found each looks at another sequence)
    return s;
}

template <int R, int TT>
__device__ __forceinline__ Unit unit_of(const AttendArgs &p, const Sequence &s, int b, int h, int rc)
{
    Unit u;
    u.b = b;
    u.h = h;
    u.rc = rc;
    u.row = s.row;
    u.n = s.n;
    u.len = s.len;
    u.r0 = rc * R;
    u.r1 = min(u.r0 + R, u.n * p.group);
    const int first = by_group(p, u.r0), last = by_group(p, max(u.r1, 1) - 1);
    u.hi = p.causal ? max(0, min(u.len, u.len - u.n + last + 1)) : u.len;
    u.lo = p.window ? max(0, u.len - u.n + first + 1 - p.window) : 0;
    u.t0 = u.hi > u.lo ? u.lo / TT : 0;
    u.nt = u.hi > u.lo ? (u.hi + TT - 1) / TT - u.t0 : 1;
    return u;
}
// The tokens row `at` of a unit's sequence sees.
__device__ __forceinline__ void row_limits(const AttendArgs &p, const Unit &u, int at, int &lo, int &hi)
{
    const int place = u.len - u.n + by_group(p, at);
    hi = p.causal ? max(0, min(u.len, place + 1)) : u.len;
    lo = p.window ? max(0, place + 1 - p.window) : 0;
}

// ---------------------------------------------------------------------------------- shares
// a / b for 0 <= a < 2^52, b > 0.  Lines longer than 2^31 are rare: a double's quotient, put right.
static __device__ __noinline__ int64_t long_quotient(int64_t a, int64_t b)
{
    int64_t q = (int64_t)((double)a / (double)b);
    if (q * b > a) q--;
    if ((q + 1) * b <= a) q++;
    return q;
}
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b)
{
    return (a | b) >> 31 ? long_quotient(a, b) : (int64_t)((uint32_t)a / (uint32_t)b);
}

struct Start {
    int b, h, rc, at;                          // where a share begins: a unit, and a place in it
    int64_t left;                              // how long it is
};

// The line of work: sequence after sequence, head after head, unit after unit, a unit taking unit_pad places for itself and
// then one a tile.  It is cut into shares, one a block, but none of less than LEAST_TOKENS tokens unless every unit has one;
// shares are equally long, but for one place.
struct Line {
    Start start;                               // of the share asked for
    int64_t each;                              // places a share,
    int more, shares;                          // and one more in the first `more` of them
    __device__ __forceinline__ int64_t at(int block) const { return each * block + min(block, more); }
};

// Called by a whole warp, a lane a sequence (32 at a time).  This is the first thing a block does, and its instructions have
// to be fetched before they run: it is written for little code, not for few steps.
template <int R, int TT>
__device__ __noinline__ Line line_of(const AttendArgs &p, int block)
{
    const int lane = threadIdx.x & 31;
    Line line = {{p.seq.count, 0, 0, 0, 0}, 0, 0, 1};
    int64_t total = 0, x = -1, tiles = 0;      // x: the place looked for, from the first of the sequences at hand; -1: none yet
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
#pragma unroll 1
        for (int base = 0; base < p.seq.count; base += 32) {
            // the length of one head of this lane's sequence
            int64_t mine = 0;
            if (base + lane < p.seq.count) {
                const Sequence s = sequence_at(p, base + lane);
                const int chunks = (s.n * p.group + R - 1) / R;
#pragma unroll 1
                for (int rc = 0; rc < chunks; rc++) mine += unit_of<R, TT>(p, s, 0, 0, rc).nt + unit_pad(TT);
            }
            int64_t upto = mine * p.heads;     // and of those before it, all heads
#pragma unroll 1
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t other = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += other;
            }
            const int64_t all = __shfl_sync(0xffffffffu, upto, 31);
            if (pass == 0) {
                total += all;
                continue;
            }
            const unsigned after = __ballot_sync(0xffffffffu, upto > x);
            if (after) {
                const int k = __ffs(after) - 1;
                line.start.b = base + k;
                tiles = __shfl_sync(0xffffffffu, mine, k);
                x -= __shfl_sync(0xffffffffu, upto, k) - tiles * p.heads;
                break;
            }
            x -= all;
        }
        if (pass == 0) {
            const int64_t units = (int64_t)p.seq.count * p.heads * p.chunks;
            line.shares = (int)max((int64_t)1, min(min((int64_t)p.grid, total), max(units, total / (LEAST_TOKENS / TT))));
            if (block >= line.shares || total == 0) return line;
            line.each = quotient(total, line.shares);
            line.more = (int)(total - line.each * line.shares);
            x = line.at(block);
            line.start.left = line.at(block + 1) - x;
        }
    }
    if (line.start.b == p.seq.count || tiles == 0) {
        line.start.left = 0;
        return line;
    }
    line.start.h = (int)quotient(x, tiles);
    x -= line.start.h * tiles;
    const Sequence s = sequence_at(p, line.start.b);
    for (;;) {
        const int length = unit_of<R, TT>(p, s, 0, 0, line.start.rc).nt + unit_pad(TT);
        if (x < length) break;
        x -= length;
        line.start.rc++;
    }
    line.start.at = (int)x;
    return line;
}

// What a block leaves at the head of the workspace for the kernel that joins the parts: where its share begins.
struct Mark {
    Line line;
    int nt;                                    // tiles of the unit
};
__host__ __device__ constexpr size_t marks_bytes(int grid) { return ((size_t)grid * sizeof(Mark) + 255) / 256 * 256; }
__device__ __forceinline__ float *parts_of(const AttendArgs &p) { return (float *)((uint8_t *)p.workspace + marks_bytes(p.grid)); }

// attend_tiles.cu, f32 lanes: a block's sums so far, behind the parts.
__device__ __forceinline__ float *kept_of(const AttendArgs &p, int r) { return parts_of(p) + (size_t)p.grid * 2 * part_floats(r, p.dim); }

template <int R, int TT>
__device__ __forceinline__ Start share_of(const AttendArgs &p, int block)        // by a whole warp
{
    const Line line = line_of<R, TT>(p, block);
    if ((threadIdx.x & 31) == 0) {
        Mark m;
        m.line = line;
        m.nt = line.start.left > 0 ? unit_of<R, TT>(p, sequence_at(p, line.start.b), line.start.b, line.start.h, line.start.rc).nt : 0;
        ((Mark *)p.workspace)[block] = m;
    }
    return line.start;
}

struct Piece {                                 // tiles first .. first + count - 1 of a unit
    Unit unit;
    int first, count;
};

// The pieces of a block's share, one after the other.  WHOLE: the call's units may be uncut (args.whole).
template <int R, int TT, bool WHOLE>
struct Walk {
    const AttendArgs &p;
    Sequence seq;
    int b, h, rc, chunks, at;
    int64_t left;                              // of the share; whole: the next unit's number

    __device__ __forceinline__ Walk(const AttendArgs &args, const Start &s) : p(args), b(s.b), h(s.h), rc(s.rc), chunks(0), at(s.at), left(s.left)
    {
        if (WHOLE && p.whole) {
            left = blockIdx.x;
            rc = 0;
        } else if (b >= p.seq.count) left = 0;
        else if (left > 0) look();
    }
    __device__ __forceinline__ void look()
    {
        seq = sequence_at(p, b);
        chunks = (seq.n * p.group + R - 1) / R;
    }
    __device__ __forceinline__ bool next(Piece &piece)
    {
        if (WHOLE && p.whole) {
            rc += p.chunks;                                    // more rows than the caller's bound said
#pragma unroll 1
            while (rc >= chunks) {
                if (left >= (int64_t)p.seq.count * p.heads * p.chunks) return false;
                const int unit = (int)left;                    // fewer than 2^31: seen to on the host
                const int bh = unit / p.chunks;
                rc = unit - bh * p.chunks;
                b = bh / p.heads;
                h = bh - b * p.heads;
                left += gridDim.x;
                look();
            }
            piece.unit = unit_of<R, TT>(p, seq, b, h, rc);
            piece.first = 0;
            piece.count = piece.unit.nt;
            return true;
        }
#pragma unroll 1
        while (left > 0) {
#pragma unroll 1
            while (rc >= chunks) {
                rc = 0;
                if (++h == p.heads) {
                    h = 0;
                    if (++b >= p.seq.count) return false;
                    look();
                }
            }
            piece.unit = unit_of<R, TT>(p, seq, b, h, rc);
            const int to = (int)min((int64_t)(piece.unit.nt + unit_pad(TT)), at + left);
            if (to <= at) return false;
            piece.first = max(0, at - unit_pad(TT));
            piece.count = max(0, to - unit_pad(TT)) - piece.first;
            left -= to - at;
            at = 0;
            rc++;
            if (piece.count > 0) return true;
        }
        return false;
    }
};

// ---------------------------------------------------------------------------------- arithmetic
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The exponent that weights are taken against where the largest of them is 2^top against 0: that one becomes 2^at, where f16 holds it
// exactly (it is most of what a sharp row sums), and the exponent is a multiple of 2^-14, so that sums with the powers of two of
// `part_scale` are exact too.  f16 lanes, relative errors against 64 bits: 40 rows at dim 256 2.9e-4 with whole exponents, 2.5e-4 so;
// prompts 2.9e-4 and 2.7e-4.  at: 11 in attend_rows.cu (10: 2.6e-4, no quicker); 10 in attend_tiles.cu, where going back over O costs more and is
// seldomer then (prompts 1226 us at 11, 1136 at 10, whole exponents 1188; 2.65e-4 at 11).
__device__ __forceinline__ float exponent_for(float top, float at) { return rintf((top - at) * 16384.f) * (1.f / 16384.f); }
// A part of a row's sums, o * v0 and sum with weights against 2^m, is handed on with the sum brought to 2^-16 .. 2^-15 by a power of
// two (less where v0 times that would leave f32): parts then join whatever reference each had, and values next to f32's
// largest do not leave it.  Gives what o is to be multiplied by.
__device__ __forceinline__ float part_scale(float &m, float &sum, float v0)
{
    const int e = sum == 0.f ? 0 : max(min((int)(__float_as_uint(sum) >> 23) - 127 + 16, 126), (__float_as_int(v0) >> 23) - 253);
    const float up = __uint_as_float((uint32_t)(127 - e) << 23);
    sum *= up;
    m += (float)e;
    return v0 * up;
}
// A power of two that brings `top` to 2^13 .. 2^14, and its reciprocal; 1 for zero, infinities and NaN.
__device__ __forceinline__ void power_scale(float top, float &up, float &down)
{
    int e = (__float_as_uint(top) >> 23) & 255;
    if (top == 0.f || e == 255) e = 140;
    e = max(e, 14);
    up = __uint_as_float((uint32_t)(267 - e) << 23);
    down = __uint_as_float((uint32_t)(e - 13) << 23);
}
// Two values as f16 pairs: the nearest, and what is left.
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(a - f.x, b - f.y);
    hi = *(const uint32_t *)&h;
    lo = *(const uint32_t *)&r;
}
__device__ __forceinline__ uint32_t minus1152(uint32_t x)
{
    uint32_t y;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
    return y;
}
// Bytes 0, 1 (2, 3) of a word, codes + 128, as f16 codes.
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) { return minus1152(__byte_perm(w, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) { return minus1152(__byte_perm(w, 0x64646464u, 0x4342)); }
// A page number from the table.  It is fetched ahead, and looked at only where it is used, so that nothing waits for the
// table where the next pages are asked for.
struct Page {
    int id;
    bool wanted;                               // tokens that a row sees lie in it
};
__device__ __forceinline__ Page page_at(const AttendArgs &p, int b, int token, int tokens, int lo, int hi, bool there)
{
    Page g;
    g.wanted = there && token < hi && token + tokens > lo;
    g.id = -1;
    if (g.wanted) g.id = __ldg(p.seq.table + (int64_t)b * p.seq.width + (token >> p.log_page));
    return g;
}
__device__ __forceinline__ int page_number(const AttendArgs &p, const Page &g, bool report)        // -1: none
{
    if (g.id >= 0 && g.id < p.pages) return g.id;
    if (g.wanted && report) atomicOr(p.status, STATUS_CACHE_RANGE);
    return -1;
}
__device__ __forceinline__ float2 scales_at(const AttendArgs &p, int page, int h)      // of K and of V
{
    if (page < 0) return make_float2(0.f, 0.f);
    const int64_t i = (int64_t)page * p.heads + h;
    return make_float2(__ldg(p.k_scales + i), __ldg(p.v_scales + i));
}
// V's scales enter the weights against a reference v0, a power of two: the largest scale of those first met, rounded down.  A
// scale more than 2^ABOVE above v0 sets a new reference, one more than 2^BELOW below counts as 0.  So whatever the scales are, f32
// holds a weight (2^11 at its largest) beside one that is 2^(ABOVE + BELOW) larger by their scales and 2^30 by their scores, and the
// denominator of a part (2^17 tokens of 2^15 * 2^BELOW at most).
constexpr int ABOVE = 10, BELOW = 85;
__device__ __forceinline__ int exponent_of(float x) { return (__float_as_int(x) >> 23) & 255; }
// The bits of what V's scale asks of the reference: its size, or 0 where there is nothing to measure.
__device__ __forceinline__ uint32_t reference_of(bool there, float sv) { return there && fabsf(sv) <= 3.402823466e38f ? __float_as_uint(fabsf(sv)) : 0u; }
__device__ __forceinline__ void raise(float &v0, uint32_t largest)       // largest: of what several scales ask
{
    const float to = __uint_as_float(min(max(largest & 0x7f800000u, 1u << 23), 253u << 23));      // its inverse is a normal number too
    if (largest && (v0 == 0.f || exponent_of(to) > exponent_of(v0) + ABOVE)) v0 = to;
}
// Where the reference rises by 2^step, a row's exponent m falls by as much, so that its weights stay what they are, and so does O; the
// denominator rises, and where that would leave f32 (e: its exponent_of) m falls by less and O goes down for the rest.
__device__ __forceinline__ int fall_of(int step, int e) { return min(step, 127 + 100 - e); }
// How the tokens of a page are weighted.
struct Weighted {
    float log_ratio, inverse;                  // log2(|sv| / v0), added to the scores; v0 / |sv|, a weight's part of the denominator
    uint32_t mark;                             // what else V's scale asks for
};
constexpr uint32_t MARK_ZERO = 1, MARK_MINUS = 2;      // of a scale of 0 (in the denominator, nothing to the sums), and below 0
__device__ __forceinline__ Weighted weighted(bool there, float sv, float v0)
{
    Weighted w = {0.f, 1.f, 0};
    const float ratio = fabsf(sv) * __uint_as_float((uint32_t)(254 - exponent_of(v0)) << 23);
    if (!there) {
        w.log_ratio = -INFINITY;
        w.inverse = 0.f;
    } else if (!(fabsf(sv) <= 3.402823466e38f)) w.log_ratio = __int_as_float(0x7fffffff);     // rows that see it get NaN, others nothing of it
    else if (exponent_of(ratio) < 127 - BELOW) {       // as if it were the least that counts, so that it sets no row's exponent
        w.mark = MARK_ZERO;
        w.log_ratio = -BELOW;
        w.inverse = __uint_as_float((uint32_t)(127 + BELOW) << 23);
    } else {
        w.log_ratio = __log2f(ratio);
        w.inverse = __fdividef(1.f, ratio);
        w.mark = sv < 0.f ? MARK_MINUS : 0;
    }
    return w;
}
// Pairs of weights as the product with V takes them.
__device__ __forceinline__ uint32_t marked(uint32_t pair, bool zero, bool minus) { return zero ? 0u : pair ^ (minus ? 0x80008000u : 0u); }
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Byte offset of 16-byte chunk `chunk` of row `row` in a tile of 32 rows: rows of 128 bytes (64), chunks exchanged so that a column of rows lies in different banks.
template <int DT>
__device__ __forceinline__ uint32_t swizzled(int sub, int row, int chunk)
{
    if (DT == 64) return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    return sub * (32 * 128) + row * 128 + ((chunk ^ (row & 7)) << 4);
}
// Where row `at` of a unit's sequence goes, and its logarithm of the sum.
template <typename T>
__device__ __forceinline__ T *out_row(const AttendArgs &p, const Unit &u, int at)
{
    const int token = by_group(p, at);
    return (T *)p.out.base + (int64_t)(u.row + token) * p.out.row_stride + (int64_t)(u.h * p.group + at - token * p.group) * p.out.head_stride;
}
template <typename T>
__device__ __forceinline__ const T *q_row(const AttendArgs &p, const Unit &u, int at)
{
    const int token = by_group(p, at);
    return (const T *)p.q.base + (int64_t)(u.row + token) * p.q.row_stride + (int64_t)(u.h * p.group + at - token * p.group) * p.q.head_stride;
}
__device__ __forceinline__ void store_lse(const AttendArgs &p, const Unit &u, int at, float m, float sum)
{
    if (!p.lse) return;
    const int token = by_group(p, at);
    p.lse[(int64_t)(u.row + token) * p.q_heads + u.h * p.group + at - token * p.group] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
}
// What the sums are divided by; rows that see nothing get zeros.
__device__ __forceinline__ float inverse_of(float sum) { return sum > 0.f || sum != sum ? __fdiv_rn(1.f, sum) : 0.f; }

// Four dims of a row.
template <typename T>
__device__ __forceinline__ void store4(T *dst, const float4 &v, bool wide)
{
    if (sizeof(T) == 4) {
        if (wide) *(float4 *)dst = v;
        else {
            ((float *)dst)[0] = v.x;
            ((float *)dst)[1] = v.y;
            ((float *)dst)[2] = v.z;
            ((float *)dst)[3] = v.w;
        }
    } else {
        const uint32_t a = bits_of(v.x, dst), b = bits_of(v.y, dst), c = bits_of(v.z, dst), e = bits_of(v.w, dst);
        if (wide) *(uint2 *)dst = make_uint2(a | b << 16, c | e << 16);
        else {
            ((uint16_t *)dst)[0] = (uint16_t)a;
            ((uint16_t *)dst)[1] = (uint16_t)b;
            ((uint16_t *)dst)[2] = (uint16_t)c;
            ((uint16_t *)dst)[3] = (uint16_t)e;
        }
    }
}
template <typename T>
__device__ __forceinline__ void finish_row(const AttendArgs &p, const Unit &u, int at, int d, const float4 &acc, float m, float sum)
{
    const float inv = inverse_of(sum);
    store4<T>(out_row<T>(p, u, at) + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv), p.out_wide);
    if (d == 0) store_lse(p, u, at, m, sum);
}

// ---------------------------------------------------------------------------------- waits
// Bounded as mbar_wait is, with little code at each place (the warps of a block run different code and share the caches of
// instructions): a poll takes 20 cycles or more, so 2^26 of them are about a second at least.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
static __device__ __noinline__ bool gives_up(uint32_t polls, volatile int *abort, int *status, int status_bit)
{
    if (*abort) return true;
    if (polls < 1u << 26) return false;
    *abort = 1;
    atomicOr(status, status_bit);
    return true;
}
__device__ __forceinline__ bool mbar_wait_soon(uint32_t bar, uint32_t parity, volatile int *abort, int *status, int status_bit)
{
#pragma unroll 1
    for (uint32_t polls = 1; !mbar_test(bar, parity); polls++)
        if ((polls & 1023) == 0 && gives_up(polls, abort, status, status_bit)) return false;
    return true;
}
// The same for the lanes of a warp, which leave together.
__device__ __forceinline__ bool mbar_wait_soon_lanes(uint32_t bar, uint32_t parity, volatile int *abort, int *status, int status_bit)
{
    return __all_sync(0xffffffffu, mbar_wait_soon(bar, parity, abort, status, status_bit));
}

}  // namespace qb
