// Attention over the 8-bit cache for few rows: the query heads that share a head of the cache, for one token or a few.
//
// out = softmax(scale * q K^T) V with K = sk * ck, V = sv * cv (int8 codes, one f32 scale for each page and head).  What
// bounds it is the cache's bytes: at 8 rows 32 operations a byte.  So every byte of the cache is read once for all rows
// that share it, and the kernel is built to keep copies in flight:
//  * The work of a call is a line of tiles, 32 tokens of one head of one sequence each.  Block c of the grid takes the
//    c-th equal share of the line, whatever sequences lie in it: sequences of any lengths load all multiprocessors alike.
//    Where a share ends inside a sequence, its part goes to the workspace and a second, small kernel joins the parts.
//  * Four producer warps take the tiles in turn: table entries and scales 32 at a time, a lane each, and a tile's codes by TMA
//    tile copies with the 128-byte swizzle (the reads below then touch all banks) into a ring of stages.  A tile costs its
//    producer 700 to 1000 cycles, where the memory's pace is 350 for 8 KB: with one producer the kernel ran at 2 TB/s.
//    Asynchronous 16-byte copies by the lanes instead reached 3.6 TB/s, tile copies 4.6.  Eight consumer warps take the tiles
//    in turn, each with a softmax of its own, joined at the end of a share's part.
//  * A warp takes S^T = K q^T and O^T = V^T P^T with mma.sync m16n8k16 (f16, f32 sums): the tokens, then V's dims, are the
//    16 rows, the query rows the 8 columns, so 8 rows fill the instruction (tcgen05's 128 rows would be 15/16 padding).
//    The codes become f16 exactly (byte permute under an exponent of 1024, subtract 1152).  An order of dims or tokens
//    inside a product is free, so both operands are read as whole 16-byte chunks: lane (g, t) holds K's chunks 2t, 2t+1 of
//    token g, and V's chunk g of tokens 2t, 2t+1, 2t+8, 2t+9.
//  * sk goes into the score's factor.  sv goes into the exponent: with a reference v0 for a piece (a power of two, the
//    largest of its first pages' scales; `raise`), the weights are w = 2^(s + log2(sv / v0) - m), the sum of them with v0 / sv as
//    factor is the denominator, and O = v0 * sum w cv.  The producers take logarithms and quotients, a lane a page.
//    (|sv| is meant: where sv is below 0 the weights change sign, where it is 0 they are zeros in the second product, and a page
//    that is not there has weights of 0 in the denominator too.)
//    m is chosen so that w lies at 2^11 at its largest when it is set (`exponent_for`) and is kept while w stays below 2^15: f16
//    then holds weights down to 2^-24 of the largest with all its bits and errs by 2^-35 of it below, and the accumulators are
//    seldom rescaled.
//  * q is scaled by a power of two to a row's maximum of 2^13 and cut to f16; with f32 lanes q and w enter as the sum of
//    two f16 (SPL 2), which loses 2^-22.  With 16-bit lanes w is one f16, half a step of 2^-11 each, independent of one
//    another, and out = sum w v / sum w (the denominator has all 24 bits) is off by less than 2^-11 of sum p |v|, by a third of
//    that or less in the mean.  The output's own rounding is as large (f16) or 8 times as large (bf16).  Measured, f16, relative: prompts
//    2.7e-4 where f32 weights give 2.1e-4, 40 rows at dim 256 2.5e-4 and 2.1e-4, 131072 tokens 2.4e-4 and 2.1e-4; bf16 1.67e-3 and
//    1.66e-3.  Two f16 a weight bring it to what f32 weights give and cost f16 prompts 20 % (1164 -> 1391 us), dim 256 7 %,
//    steps 3 %, long documents 1 %: not taken, since a caller who needs more than f16's own rounding has f32 lanes.
//
// Measured (bf16, 8 heads of the cache, 128 dims): 32 sequences of 500 to 8000 tokens, 4 query heads a head 64 us = 4.6 TB/s of
// codes, 71 % of the copy peak; one of 131072 tokens, 8 a head 58 us, 71 %; a window of 1024 in f32, one row a head, 37 us, 25 %;
// 129 tokens 7 us on the device.  Of the 64 us, 45
// are the memory's; the partition at the start takes 3, the join's launch 4, and a piece's beginning and end 1.5 each.
#include <cuda.h>
#include "common.cuh"
#include "attend_device.cuh"
#include "attend_join.cuh"

namespace qb {

constexpr int RW = 8;                          // consumer warps
constexpr int RP = 4;                          // producer warps
constexpr int RTHREADS = 32 * (RW + RP);
constexpr uint32_t ROWS_HEADER = 2048;

template <int DT, int NB, int SPL>
struct RowsCfg {
    static constexpr int R = 8 * NB;           // rows a unit
    static constexpr int KS = DT / 16;         // k-steps of a score
    static constexpr int SUB = DT == 256 ? 2 : 1;               // tile copies of at most 128 bytes of dims
    static constexpr int SW = DT == 64 ? 64 : 128;              // bytes a row of a copy
    static constexpr uint32_t HALF = 32 * DT, STAGE = 2 * HALF;  // K, then V
    static constexpr int S = DT == 64 ? 24 : DT == 128 ? 16 : 8;
    static constexpr uint32_t MROW = DT + 4;                    // floats a row of the joining buffer
    static constexpr uint32_t O_RING = 0, O_Q = S * STAGE, O_MERGE = O_Q + KS * NB * SPL * 256, O_ML = O_MERGE + RW * R * MROW * 4;
    static constexpr uint32_t O_HEAD = O_ML + RW * R * 16, SMEM = O_HEAD + ROWS_HEADER + 1024;
    static_assert(S % RW == 0 && S % RP == 0, "a stage has one consumer warp and one producer");
    static_assert(SMEM <= 232448, "227 KB of shared memory");
};

struct RowsHead {                              // at O_HEAD
    uint64_t full[24], empty[24];
    float4 scales[24][2];                      // of a stage's page, or two of 16 tokens: sk, log2(|sv| / v0), v0 / |sv|, v0
    float factor[16];                          // rows: scale * log2 e / (what q was scaled by)
    int lo[16], hi[16];                        // rows: tokens they see
    Start start;
    int abort;
};
static_assert(sizeof(RowsHead) <= ROWS_HEADER, "the header fits");

struct Batch { int b, h, lo, hi, tile, count; bool starts; };      // tiles of one piece; starts: its first

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void *map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}

// c += A.b.  The tensor cores cut their sums off, where f32 additions round: with f32 lanes (b = b[0] + b[1]) the products of 16
// are summed by themselves, what the cut left first, and added with a rounding.
template <int SPL>
__device__ __forceinline__ void add_products(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint2 (&b)[SPL])
{
    if (SPL == 1) {
        mma16816(c, a0, a1, a2, a3, b[0].x, b[0].y);
        return;
    }
    float d[4] = {0.f, 0.f, 0.f, 0.f};
    mma16816(d, a0, a1, a2, a3, b[SPL - 1].x, b[SPL - 1].y);
    mma16816(d, a0, a1, a2, a3, b[0].x, b[0].y);
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] += d[i];
}

template <int DT, int NB, int SPL, typename T>
__global__ void __launch_bounds__(RTHREADS, 1)
attend_rows_kernel(const __grid_constant__ AttendArgs p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap)
{
    using C = RowsCfg<DT, NB, SPL>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    RowsHead *head = (RowsHead *)(smem + C::O_HEAD);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = smem_u32(smem), full0 = smem_u32(head->full), empty0 = smem_u32(head->empty);

    if (threadIdx.x == 0) {
        head->abort = 0;
        for (int i = 0; i < C::S; i++) {
            mbar_init(full0 + 8 * i, 1);
            mbar_init(empty0 + 8 * i, 1);
        }
        mbar_fence_init();
    }
    if (warp == 0) {
        const Start s = p.whole ? Start{} : share_of<C::R, 32>(p, blockIdx.x);
        if (lane == 0) head->start = s;
    }
    __syncthreads();
    if (!p.whole) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the joining kernel waits beside this one
    Walk<C::R, 32, true> walk(p, head->start);
    volatile int *abort = &head->abort;
    uint32_t seq = 0;                          // tiles of this block so far

    if (warp >= RW) {
        // ------------------------------------------------------------------ producers: every RP-th tile each
        // A batch: as many tiles of a piece as 32 pages hold, a lane a page.  Its page numbers are fetched two batches
        // ahead, its scales one ahead.
        const int per = p.log_page == 4 ? 2 : 1, most = 32 / per, mine = warp - RW;      // pages a tile, tiles a batch
        Piece piece;
        int at = 0;
        bool more = walk.next(piece);
        auto next_batch = [&]() {
            Batch t;
            if (more && at >= piece.count) {
                at = 0;
                more = walk.next(piece);
            }
            t.b = piece.unit.b;
            t.h = piece.unit.h;
            t.lo = piece.unit.lo;
            t.hi = piece.unit.hi;
            t.tile = piece.unit.t0 + piece.first + at;
            t.starts = at == 0;
            t.count = more ? min(most, piece.count - at) : 0;
            at += t.count;
            return t;
        };
        auto page_of = [&](const Batch &t) {
            const int token = (t.tile + lane / per) * 32 + (per == 2 ? (lane & 1) * 16 : 0);
            return page_at(p, t.b, token, 32 / per, t.lo, t.hi, lane / per < t.count);
        };
        // a copy: the tokens of one page in the tile, up to 128 bytes of each; a lane a copy
        const int rows = 32 / per, which = lane & 1, sub = (lane >> 1) % C::SUB, second = lane / (2 * C::SUB);
        const uint32_t bytes = rows * C::SW, offset = which * C::HALF + sub * (32 * 128) + second * 16 * C::SW;
        uint32_t issued = 0;                   // this warp's tiles so far: stages mine, mine + RP, ... in turn
        Batch now = next_batch();
        int id = page_number(p, page_of(now), mine == 0);
        float2 sc = scales_at(p, id, now.h);
        Batch next = next_batch();
        Page id_next = page_of(next);
        float vref = 0.f;                      // what V's scales of the piece are taken against
        while (now.count) {
            const Batch after = next_batch();
            const int id_then = page_number(p, id_next, mine == 0);
            const float2 sc_then = scales_at(p, id_then, next.h);
            id_next = page_of(after);
            float4 own;                        // this lane's page, for the consumers
            bool made = false;
            auto make = [&]() {                // by every producer for every batch: they all have the same reference
                made = true;
                if (now.starts) vref = 0.f;
                raise(vref, __reduce_max_sync(0xffffffffu, reference_of(id >= 0, sc.y)));
                // what is seldom needed lies in the signs: V's scale is below 0; it counts as 0
                const Weighted v = weighted(id >= 0, sc.y, vref);
                own = make_float4(sc.x, v.log_ratio, v.mark == MARK_MINUS ? -v.inverse : v.inverse, v.mark == MARK_ZERO ? -vref : vref);
            };
            for (int k = (mine - seq) & (RP - 1); k < now.count; k += RP) {
                const uint32_t tile = seq + k;
                const int stage = tile % C::S;
                if (tile >= C::S && !mbar_wait_soon_lanes(empty0 + 8 * stage, (tile / C::S - 1) & 1, abort, p.status, STATUS_ATTEND_WAIT)) goto done;
                const int base = (now.tile + k) * 32, l0 = k * per, l1 = l0 + per - 1;
                const int id0 = __shfl_sync(0xffffffffu, id, l0), id1 = __shfl_sync(0xffffffffu, id, l1);
                const int live = (id0 >= 0 ? 1 : 0) + (per == 2 && id1 >= 0 ? 1 : 0);
                if (lane == 0 && live) mbar_expect_tx(full0 + 8 * stage, live * 2 * C::SUB * bytes);
                issued++;
                __syncwarp();
                const int page = second ? id1 : id0;
                if (lane < 2 * C::SUB * per && page >= 0) {
                    const int row = ((page * p.heads + now.h) << p.log_page) + ((base + second * 16) & ((1 << p.log_page) - 1));
                    tma_load_2d(ring + stage * C::STAGE + offset, which ? &vmap : &kmap, sub * 128, row, full0 + 8 * stage);
                }
                if (!made) make();             // beside the first copy
                if (lane == l0 || lane == l1) head->scales[stage][lane - l0] = own;
                __syncwarp();
                if (lane == 0) mbar_arrive(full0 + 8 * stage);
            }
            if (!made) make();
            seq += now.count;
            now = next;
            id = id_then;
            sc = sc_then;
            next = after;
        }
    done:
        // no copy may be under way when the block ends, whoever gave up
        for (int i = 0; i < C::S; i++)
            if (i % RP == mine && issued > i / RP) {
                // the newest of this warp's tiles in stage i
                const uint32_t uses = (issued - 1 - i / RP) / (C::S / RP);
                const long long from = clock64();
                while (!mbar_try_wait(full0 + 8 * i, uses & 1) && clock64() - from < WAIT_CYCLES) { }
            }
        return;
    }

    // ---------------------------------------------------------------------- consumers
    const int g = lane >> 2, t = lane & 3, pages16 = p.log_page == 4;
    uint2 *qs = (uint2 *)(smem + C::O_Q);
    float *merge = (float *)(smem + C::O_MERGE);
    float4 *ml = (float4 *)(smem + C::O_ML);       // of a warp's part of a row: exponent, sum, what its O is to be multiplied by
    // this warp's rows of q for a piece: asked for while the piece before it runs
    auto rows_of = [&](const Unit &u, Vec8<T> (&q)[NB]) {
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const int at = u.r0 + warp + i * RW;
            q[i] = at < u.r1 && lane < p.dim / 8 ? load8<T>(q_row<T>(p, u, at) + lane * 8, p.q_wide) : zero8<T>();
        }
    };
    Piece piece, coming;
    Vec8<T> q[NB];
    bool gone = false, more = walk.next(coming);
    if (more) rows_of(coming.unit, q);
    while (more) {
        piece = coming;
        const Unit &u = piece.unit;
        // the rows of q, scaled and cut, in the order of the products' operands
        named_bar_sync(1, 32 * RW);            // the last piece's buffers are free
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const int r = warp + i * RW, at = u.r0 + r;
            float x[8];
            unpack8(q[i], x);
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(x[k]));
#pragma unroll
            for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            float up, down;
            power_scale(top, up, down);
            if (lane * 8 < DT) {
                const int sub = lane / 16, chunk = DT == 64 ? lane / 2 : (lane % 16) / 2;
                const int tt = DT == 64 ? chunk : chunk >> 1, ii = DT == 64 ? 0 : chunk & 1;
#pragma unroll
                for (int j = 0; j < 2; j++) {  // four dims each
                    const int ks = (sub * 2 + ii) * 4 + (lane & 1) * 2 + j;
                    uint32_t hi0, lo0, hi1, lo1;
                    split2(x[4 * j] * up, x[4 * j + 1] * up, hi0, lo0);
                    split2(x[4 * j + 2] * up, x[4 * j + 3] * up, hi1, lo1);
                    uint2 *dst = qs + ((ks * NB + r / 8) * SPL) * 32 + (r & 7) * 4 + tt;
                    dst[0] = make_uint2(hi0, hi1);
                    if (SPL == 2) dst[32] = make_uint2(lo0, lo1);
                }
            }
            if (lane == 0) {
                head->factor[r] = p.scale * 1.4426950408889634f * down;
                int lo, hi;
                row_limits(p, u, at < u.r1 ? at : u.r1 - 1, lo, hi);
                head->lo[r] = lo;
                head->hi[r] = hi;
            }
        }
        more = walk.next(coming);
        if (more) rows_of(coming.unit, q);
        named_bar_sync(1, 32 * RW);
        float factor[NB][2];
        int lo[NB][2], hi[NB][2];
        int lo_most = 0, hi_least = 0x7fffffff;
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int r = nb * 8 + 2 * t + c;
                factor[nb][c] = head->factor[r];
                lo[nb][c] = head->lo[r];
                hi[nb][c] = head->hi[r];
            }
        for (int r = 0; r < C::R; r++) {
            lo_most = max(lo_most, head->lo[r]);
            hi_least = min(hi_least, head->hi[r]);
        }

        float o[C::SUB * (DT == 64 ? 2 : 4)][2][NB][4];          // [16-byte chunk's word][pair of dims]
#pragma unroll
        for (int i = 0; i < C::SUB * (DT == 64 ? 2 : 4); i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[i][j][nb][c] = 0.f;
        float mm[NB][2], l[NB][2];             // the exponent that weights are taken against; their sum, this lane's tokens
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int c = 0; c < 2; c++) { mm[nb][c] = NOTHING; l[nb][c] = 0.f; }
        float vref = 0.f;

        const int mine = (int)((warp - seq) & (RW - 1));          // this warp's first tile of the piece
        for (int j = mine; j < piece.count && !gone; j += RW) {
            const uint32_t at = seq + j;
            const int stage = at % C::S;
            if (!mbar_wait_soon_lanes(full0 + 8 * stage, (at / C::S) & 1, abort, p.status, STATUS_ATTEND_WAIT)) { gone = true; break; }
            const uint8_t *kt = smem + stage * C::STAGE, *vt = kt + C::HALF;
            const int base = (u.t0 + piece.first + j) * 32;

            // ---- scores
            float s[2][NB][4];
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int c = 0; c < 4; c++) s[mt][nb][c] = 0.f;
#pragma unroll
            for (int sub = 0; sub < C::SUB; sub++)
#pragma unroll
                for (int i = 0; i < (DT == 64 ? 1 : 2); i++) {
                    uint4 a[2][2];             // [tile of 16 tokens][token g, g + 8]
#pragma unroll
                    for (int mt = 0; mt < 2; mt++)
#pragma unroll
                        for (int e = 0; e < 2; e++) a[mt][e] = *(const uint4 *)(kt + swizzled<DT>(sub, mt * 16 + e * 8 + g, DT == 64 ? t : 2 * t + i));
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        uint2 b[NB][SPL];
#pragma unroll
                        for (int nb = 0; nb < NB; nb++)
#pragma unroll
                            for (int x = 0; x < SPL; x++) b[nb][x] = qs[((((sub * 2 + i) * 4 + q) * NB + nb) * SPL + x) * 32 + lane];
#pragma unroll
                        for (int mt = 0; mt < 2; mt++) {
                            const uint32_t w0 = word(a[mt][0], q) ^ 0x80808080u, w1 = word(a[mt][1], q) ^ 0x80808080u;
                            const uint32_t a0 = codes_lo(w0), a1 = codes_lo(w1), a2 = codes_hi(w0), a3 = codes_hi(w1);
#pragma unroll
                            for (int nb = 0; nb < NB; nb++) add_products<SPL>(s[mt][nb], a0, a1, a2, a3, b[nb]);
                        }
                    }
                }

            // ---- weights
            const float4 *sc[2] = { &head->scales[stage][0], &head->scales[stage][pages16] };
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int c = 0; c < 4; c++) s[mt][nb][c] = __fmaf_rn(s[mt][nb][c], factor[nb][c & 1] * sc[mt]->x, sc[mt]->y);
            if (base < lo_most || base + 32 > hi_least) {
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const int token = base + mt * 16 + g + (c >> 1) * 8;
                            if (token < lo[nb][c & 1] || token >= hi[nb][c & 1]) s[mt][nb][c] = -INFINITY;
                        }
            }
            if (fabsf(sc[1]->w) != vref) {     // what V's scales are taken against: the first, seldom another
                const int step = vref == 0.f ? 0 : exponent_of(sc[1]->w) - exponent_of(vref);
                vref = fabsf(sc[1]->w);
                if (step) {
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            int e = exponent_of(l[nb][c]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) e = max(e, __shfl_xor_sync(0xffffffffu, e, d));
                            const float fall = (float)fall_of(step, e), less = exp2_fast(fall - (float)step);
                            mm[nb][c] -= fall;
                            l[nb][c] *= exp2_fast(fall);
#pragma unroll
                            for (int i = 0; i < C::SUB * (DT == 64 ? 2 : 4); i++)
#pragma unroll
                                for (int k = 0; k < 2; k++) {
                                    o[i][k][nb][c] *= less;
                                    o[i][k][nb][c + 2] *= less;
                                }
                        }
                }
            }
            bool above = false;
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int c = 0; c < 4; c++) above |= s[mt][nb][c] > mm[nb][c & 1] + 15.f;
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float top = fmaxf(fmaxf(s[0][nb][c], s[0][nb][c + 2]), fmaxf(s[1][nb][c], s[1][nb][c + 2]));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        const float next = fmaxf(mm[nb][c], exponent_for(top, 11.f)), less = exp2_fast(mm[nb][c] - next);
                        mm[nb][c] = next;
                        l[nb][c] *= less;
#pragma unroll
                        for (int i = 0; i < C::SUB * (DT == 64 ? 2 : 4); i++)
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                o[i][k][nb][c] *= less;
                                o[i][k][nb][c + 2] *= less;
                            }
                    }
            }
            uint2 w[2][NB][SPL];
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    uint32_t half[SPL][2];
                    float e[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        e[c] = exp2_fast(s[mt][nb][c] - mm[nb][c & 1]);
                        l[nb][c & 1] = __fmaf_rn(e[c], fabsf(sc[mt]->z), l[nb][c & 1]);
                    }
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        uint32_t a, b;
                        split2(e[2 * k], e[2 * k + 1], a, b);
                        half[0][k] = transposed8(a);
                        if (SPL == 2) half[SPL - 1][k] = transposed8(b);
                    }
#pragma unroll
                    for (int z = 0; z < SPL; z++) w[mt][nb][z] = make_uint2(half[z][0], half[z][1]);
                }
            if (__float_as_int(sc[0]->z) < 0 || __float_as_int(sc[0]->w) < 0 || __float_as_int(sc[1]->z) < 0 || __float_as_int(sc[1]->w) < 0) {   // seldom: scales of V of 0 or below
#pragma unroll
                for (int mt = 0; mt < 2; mt++) {
                    const bool minus = __float_as_int(sc[mt]->z) < 0, zero = __float_as_int(sc[mt]->w) < 0;
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
#pragma unroll
                        for (int z = 0; z < SPL; z++) {
                            w[mt][nb][z].x = marked(w[mt][nb][z].x, zero, minus);
                            w[mt][nb][z].y = marked(w[mt][nb][z].y, zero, minus);
                        }
                }
            }

            // ---- O^T += V^T P^T
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int sub = 0; sub < C::SUB; sub++) {
                    uint4 r[4];                // this lane's dims of tokens 2t, 2t+1, 2t+8, 2t+9
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int token = mt * 16 + 2 * t + (e & 1) + (e >> 1) * 8;
                        if (DT == 64) {
                            const uint2 h = *(const uint2 *)(vt + swizzled<DT>(0, token, g >> 1) + (g & 1) * 8);
                            r[e] = make_uint4(h.x, h.y, 0, 0);
                        } else r[e] = *(const uint4 *)(vt + swizzled<DT>(sub, token, g));
                    }
#pragma unroll
                    for (int q = 0; q < (DT == 64 ? 2 : 4); q++) {
                        const uint32_t w0 = word(r[0], q) ^ 0x80808080u, w1 = word(r[1], q) ^ 0x80808080u;
                        const uint32_t w2 = word(r[2], q) ^ 0x80808080u, w3 = word(r[3], q) ^ 0x80808080u;
                        const uint32_t x0 = __byte_perm(w0, w1, 0x5140), x1 = __byte_perm(w0, w1, 0x7362);
                        const uint32_t y0 = __byte_perm(w2, w3, 0x5140), y1 = __byte_perm(w2, w3, 0x7362);
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const uint32_t x = k ? x1 : x0, y = k ? y1 : y0;
                            const uint32_t a0 = codes_lo(x), a1 = codes_hi(x), a2 = codes_lo(y), a3 = codes_hi(y);
#pragma unroll
                            for (int nb = 0; nb < NB; nb++) add_products<SPL>(o[sub * 4 + q][k][nb], a0, a1, a2, a3, w[mt][nb]);
                        }
                    }
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * stage);
        }
        seq += piece.count;

        // ---- the warps' parts of this piece
        const float v0 = vref > 0.f ? vref : 1.f;
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float sum = l[nb][c];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                const int r = nb * 8 + 2 * t + c;
                // O's factor is taken below, where the parts are joined (f32 window: 38.0 us, taken here 38.6); at dim 256 that spills (60.5 us, here 58.6)
                const float scale = part_scale(mm[nb][c], sum, v0), times = DT == 256 ? scale : 1.f;
                if (g == 0) ml[warp * C::R + r] = make_float4(mm[nb][c], sum, DT == 256 ? 1.f : scale, 0.f);
                float *row = merge + (warp * C::R + r) * C::MROW;
#pragma unroll
                for (int i = 0; i < C::SUB * (DT == 64 ? 2 : 4); i++) {
                    const int dim = DT == 64 ? 8 * g + 4 * i : (i / 4) * 128 + 16 * g + 4 * (i % 4);
                    *(float4 *)(row + dim) = make_float4(o[i][0][nb][c] * times, o[i][0][nb][c + 2] * times, o[i][1][nb][c] * times, o[i][1][nb][c + 2] * times);
                }
            }
        named_bar_sync(1, 32 * RW);
        const int rows = u.r1 - u.r0, quads = p.dim / 4;
        const bool complete = piece.first == 0 && piece.count == u.nt;
        for (int i = threadIdx.x; i < rows * quads; i += 32 * RW) {
            const int r = i / quads, d = (i - r * quads) * 4;
            float m = NOTHING;
#pragma unroll
            for (int k = 0; k < RW; k++) m = fmaxf(m, ml[k * C::R + r].x);
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < RW; k++) {
                const float4 part = ml[k * C::R + r];
                const float f = exp2_fast(part.x - m), fo = DT == 256 ? f : f * part.z;
                const float4 x = *(const float4 *)(merge + (k * C::R + r) * C::MROW + d);
                sum = __fmaf_rn(part.y, f, sum);
                acc.x = __fmaf_rn(x.x, fo, acc.x);
                acc.y = __fmaf_rn(x.y, fo, acc.y);
                acc.z = __fmaf_rn(x.z, fo, acc.z);
                acc.w = __fmaf_rn(x.w, fo, acc.w);
            }
            if (complete) finish_row<T>(p, u, u.r0 + r, d, acc, m, sum);
            else {
                float *slot = parts_of(p) + (size_t)(blockIdx.x * 2 + (piece.first ? 0 : 1)) * part_floats(C::R, p.dim);
                *(float4 *)(slot + C::R * 2 + r * p.dim + d) = acc;
                if (d == 0) *(float2 *)(slot + r * 2) = make_float2(m, sum);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- host

template <int DT, int NB, int SPL, typename T>
static cudaError_t set_rows_attr()
{
    return cudaFuncSetAttribute(attend_rows_kernel<DT, NB, SPL, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)RowsCfg<DT, NB, SPL>::SMEM);
}
template <int DT, int NB>
static cudaError_t set_rows_attrs()
{
    cudaError_t e;
    if ((e = set_rows_attr<DT, NB, 2, float>()) || (e = set_rows_attr<DT, NB, 1, __half>())) return e;
    return set_rows_attr<DT, NB, 1, __nv_bfloat16>();
}

cudaError_t attend_rows_init()
{
    cudaError_t e;
    if ((e = set_rows_attrs<64, 1>()) || (e = set_rows_attrs<64, 2>()) || (e = set_rows_attrs<128, 1>()) || (e = set_rows_attrs<128, 2>())) return e;
    return set_rows_attrs<256, 1>();
}

template <int DT, int NB, int SPL, typename T>
static int launch_rows(const AttendArgs &args, const CUtensorMap &kmap, const CUtensorMap &vmap, cudaStream_t stream)
{
    attend_rows_kernel<DT, NB, SPL, T><<<args.grid, RTHREADS, RowsCfg<DT, NB, SPL>::SMEM, stream>>>(args, kmap, vmap);
    const cudaError_t e = cudaGetLastError();
    return e || args.whole ? (int)e : launch_join<8 * NB, 32, T>(args, stream);
}

template <int SPL, typename T>
static int launch_rows_dim(const AttendArgs &args, int r, const CUtensorMap &kmap, const CUtensorMap &vmap, cudaStream_t stream)
{
    if (args.dim <= 64) return r == 16 ? launch_rows<64, 2, SPL, T>(args, kmap, vmap, stream) : launch_rows<64, 1, SPL, T>(args, kmap, vmap, stream);
    if (args.dim <= 128) return r == 16 ? launch_rows<128, 2, SPL, T>(args, kmap, vmap, stream) : launch_rows<128, 1, SPL, T>(args, kmap, vmap, stream);
    return launch_rows<256, 1, SPL, T>(args, kmap, vmap, stream);
}

int attend_rows(const AttendArgs &args, int type, int r, const CUtensorMap &kmap, const CUtensorMap &vmap, cudaStream_t stream)
{
    if (type == QB200_F32) return launch_rows_dim<2, float>(args, r, kmap, vmap, stream);
    if (type == QB200_F16) return launch_rows_dim<1, __half>(args, r, kmap, vmap, stream);
    return launch_rows_dim<1, __nv_bfloat16>(args, r, kmap, vmap, stream);
}

}  // namespace qb
