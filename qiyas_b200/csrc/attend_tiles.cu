// Attention over the 8-bit cache for many rows (prompts, large groups) on the fifth-generation tensor cores.
//
// out = softmax(scale * q K^T) V as in attend_rows.cu, with 128 rows (tokens x the query heads of a group) a row tile, up to
// two row tiles a block, and tiles of 64 tokens of the cache.  Here the operations bound it: two row tiles, 64 tokens and 128
// dims are 1280 cycles of the tensor pipe and 1024 of the exponential unit.  So:
//  * S = q K^T and O += P V are tcgen05.mma kind::f16 (codes are exact in f16), a thread a row tile issuing them, S, P and O
//    in tensor memory: P replaces S in place as f16 and is read from there as the second product's A operand.
//  * Four converter warps (eight for dims over 128) fetch the codes, 16 bytes a load, a tile ahead in registers, and store
//    them as f16: K as core matrices of 8 tokens x 8 dims, V as rows of 64 dims with the 128-byte swizzle, which the second
//    product reads across (a row a dim: MN-major; from unswizzled core matrices it took half as long again).  Every byte of
//    the cache is converted once for the 256 rows of a block.  One warp fetches the tiles' scales.
//  * Four softmax warps a row tile, a thread a row, with two buffers of S: the tensor pipe is a tile of tokens ahead.
//  * A thread reads its row of S once and takes the weights against the exponent it has: only where one would pass 2^15 does
//    it raise the exponent and go back over what the row has of O.
//  * The registers are shared out between the warps' kinds (setmaxnreg): up to 128 dims 16-bit lanes spill nothing, f32 lanes 12 bytes,
//    over 128 dims all 72.
// Scales, exponents and the cut of q and w (what it costs, and why) are those of attend_rows.cu; so are the shares of the
// grid's blocks.  One warp takes the logarithms of V's scales; where a tile has scales of 0 or below, the stored weights are put right
// after the fact, out of the way of the others (in their loop it took prompts from 1.18 to 1.21 ms).
//
// Measured: 7894 queries of 32 heads (8 of the cache) over up to 8192 tokens, causal, 128 dims, bf16: 1.13 to 1.15 ms, 680 TFLOP/s, 40 %
// of the library's bf16 product; 3900 of them over up to 4000 tokens: f32 603 us, at 256 dims in bf16 947 us.  Three chains are
// near one another there (measured at 1.18 ms, with the work of one left out in a copy): the
// converters 1.01 ms, the softmax 1.00 ms, the products with their barriers 0.82 ms; what they wait for is mostly
// instructions (16 warps of four kinds, 90 KB of code).  Tried and dropped: tiles of 128 tokens with one buffer of S a row tile
// (1.3 ms: the chain from a product through softmax to the next is not hidden), a maximum pass over S before the weights
// (1.7 ms), one issuing thread (1.3 ms), issue by a whole warp (1.56 ms), a quarter or half of the exponentials as
// polynomials on the fma pipe (4 and 18 % slower: the exponential unit is not the bound), five commits a tile
// instead of two (3 %).
#include <type_traits>
#include "common.cuh"
#include "attend_device.cuh"
#include "attend_join.cuh"
#include "tcgen05.cuh"

namespace qb {

template <int DC, int SPL>
struct TilesCfg {
    static constexpr int TT = 64;                               // tokens a tile
    static constexpr int NQ = DC == 128 ? 2 : 1;                // row tiles a block
    static constexpr int R = 128 * NQ;
    static constexpr int SLOTS = (SPL == 1 ? 2 : 1) * (DC == 128 ? 2 : 1);      // of K and of V
    static constexpr int NG = TT / 16;
    static constexpr int CW = DC == 128 ? 4 : 8, KW = CW / 2;   // converter warps: half of them for K, half for V
    static constexpr int WARPS = 4 * NQ + CW + 4, THREADS = 32 * WARPS;       // the last four: two issue the products, one fetches scales
    // registers a thread: of the launch, and of the softmax, converter and last warps (checked against the build when the
    // library is bound, and the kernel left aside where it differs: a share above the launch's would wait for good)
    static constexpr int REGS = 128, SOFT_REGS = NQ == 2 ? 152 : 176, CONV_REGS = NQ == 2 ? 128 : 104, REST_REGS = NQ == 2 ? 80 : 128;
    static_assert(NQ * SOFT_REGS + CW / 4 * CONV_REGS + REST_REGS <= WARPS / 4 * REGS, "the shares of the registers fit the launch's");
    static constexpr uint32_t QTILE = 128 * DC * 2, SLOT = TT * DC * 2;
    static constexpr uint32_t O_Q = 0, O_K = NQ * SPL * QTILE, O_V = O_K + SLOTS * SLOT, O_HEAD = O_V + SLOTS * SLOT, SMEM = O_HEAD + 2048 + 1024;
    static_assert(SMEM <= 232448, "227 KB of shared memory");
    // f32 lanes: tiles whose products O takes before it is added, with a rounding, to what is kept in the workspace.  The tensor
    // cores cut their sums off, and the cuts of a long sum add up.  4 heads x 4, 4 x 1000 queries over 9000 tokens: 636 us
    // without, 695, 770 and 895 with 16, 8 and 4 tiles; 200 queries over 20000 tokens, against 64 bits: off by 4.7e-6 without,
    // 2.3e-6, 1.4e-6 and 0.9e-6 (dim 256, 3000 tokens: 4.2e-6, 2.5e-6, 1.6e-6, 1.1e-6; with f32 products throughout 1.6e-6).
    static constexpr int KEEP = 8;
    __host__ __device__ static constexpr uint32_t s_col(int t, int b) { return (2 * t + b) * TT; }
    __host__ __device__ static constexpr uint32_t o_col(int t) { return 256 + t * 128; }
};

struct TilesHead {
    uint64_t qfull, ofull, drain;
    uint64_t kfull[4], kempty[4], vfull[4], vempty[4];
    uint64_t sfull[4], pfull[4], odone[2];     // of the S buffers, two a row tile; of O before a piece's last tile
    float4 scales[4][4];                       // beside K's slots, of a tile's groups of 16 tokens: sk, log2(|sv| / v0), v0 / |sv|, and v0
                                               // (the first group's: a bit a group, V's scale counts as 0, and from bit 16 on, it is below 0;
                                               // the second's: by how many powers of two v0 rose with this tile)
    Start start;
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(TilesHead) <= 2048, "the header fits");

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
                   "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] . B, A's row of 16 f16 in eight columns.
__device__ __forceinline__ void mma_issue_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// The tiles of a block's share in order, for the converters.
template <int R, int TT>
struct KvTile {
    int b, h, base, lo, hi;
    bool there, starts;                        // starts: the first of a piece
};
template <int R, int TT>
struct KvWalk {
    Walk<R, TT, false> walk;
    Piece piece;
    int at;
    bool more;
    __device__ __forceinline__ KvWalk(const AttendArgs &p, const Start &s) : walk(p, s), at(0) { more = walk.next(piece); }
    __device__ __forceinline__ KvTile<R, TT> next()
    {
        KvTile<R, TT> t;
        if (more && at == piece.count) {
            at = 0;
            more = walk.next(piece);
        }
        t.there = more;
        t.starts = at == 0;
        if (more) {
            t.b = piece.unit.b;
            t.h = piece.unit.h;
            t.base = (piece.unit.t0 + piece.first + at) * TT;
            t.lo = piece.unit.lo;
            t.hi = piece.unit.hi;
            at++;
        }
        return t;
    }
};

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 16 bytes of global memory into shared memory.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Pairs of f32 in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <int DC, int SPL, typename T>
__global__ void __launch_bounds__((TilesCfg<DC, SPL>::THREADS), 1) attend_tiles_kernel(const __grid_constant__ AttendArgs p)
{
    using C = TilesCfg<DC, SPL>;
    constexpr int TT = C::TT, NQ = C::NQ, R = C::R, SLOTS = C::SLOTS, NG = C::NG, CW = C::CW, KW = C::KW;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    TilesHead *head = (TilesHead *)(smem + C::O_HEAD);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base_u32 = smem_u32(smem);
    const uint32_t qfull = smem_u32(&head->qfull), ofull = smem_u32(&head->ofull), drain = smem_u32(&head->drain);
    const uint32_t kfull = smem_u32(head->kfull), kempty = smem_u32(head->kempty), vfull = smem_u32(head->vfull), vempty = smem_u32(head->vempty);
    const uint32_t sfull = smem_u32(head->sfull), pfull = smem_u32(head->pfull), odone = smem_u32(head->odone);

    if (threadIdx.x == 0) {
        head->abort = 0;
        mbar_init(qfull, 4 * NQ);
        mbar_init(ofull, 2);
        mbar_init(drain, 2);
        for (int i = 0; i < 2; i++) mbar_init(odone + 8 * i, 1);
        for (int i = 0; i < 4; i++) {
            mbar_init(kfull + 8 * i, KW + 1);           // the converters', and the tile's scales

            mbar_init(kempty + 8 * i, 8);          // the softmax warps' (with one row tile they arrive twice)
            mbar_init(vfull + 8 * i, KW);
            mbar_init(vempty + 8 * i, 2);          // the products' ends, of both row tiles (or twice of one)
            mbar_init(sfull + 8 * i, 1);
            mbar_init(pfull + 8 * i, 4);
        }
        mbar_fence_init();
    }
    if (warp == 0) {
        const Start s = share_of<R, TT>(p, blockIdx.x);
        if (lane == 0) head->start = s;
    }
    if (warp == 4 * NQ + CW) tmem_alloc(smem_u32(&head->tmem), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");           // the joining kernel waits beside this one
    const uint32_t tmem = head->tmem;
    volatile int *abort = &head->abort;
    int *status = p.status;

    if (warp < 4 * NQ) {
        // ------------------------------------------------------------------ softmax: a thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFT_REGS));
        const int t = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        Walk<R, TT, false> walk(p, head->start);
        Piece piece;
        uint32_t pieces = 0, seq = 0, tiles = 0, ends = 0;       // so far: pieces, tiles of the block, of this row tile; phases of odone
        while (walk.next(piece)) {
            const Unit &u = piece.unit;
            const int nq = NQ == 2 && u.r1 - u.r0 > 128 ? 2 : 1;
            const bool active = t < nq;
            const int n = piece.count;
            const int at = u.r0 + t * 128 + quarter * 32 + lane;
            float factor = p.scale * 1.4426950408889634f;
            if (active) {
                // q: its rows are copied as they are to where their core matrices will be (8 f16 dims, or 4 of f32: 16 bytes), all
                // copies under way at once; then each thread scales and cuts its own row in place (f16 lanes stay as they are)
                uint8_t *tile = smem + C::O_Q + t * SPL * C::QTILE;
                const T *mine = q_row<T>(p, u, min(at, u.r1 - 1));
                const int groups = p.dim / 8, rows = min(32, u.r1 - (at - lane));
                if (p.q_wide) {
                    constexpr int PER = DC == 128 ? 2 : 1, WIDTH = 32 / PER;
                    const int col = lane % WIDTH;
#pragma unroll 1
                    for (int i = lane / WIDTH; i - lane / WIDTH < rows; i += PER) {
                        const T *src = (const T *)__shfl_sync(0xffffffffu, (unsigned long long)mine, i & 31) + col * 8;
                        const int r = quarter * 32 + i;
                        const uint32_t dst = smem_u32(tile) + col * 2048 + (r >> 3) * 128 + (r & 7) * 16;
                        if (col < groups && i < rows) {
                            copy16(dst, src);
                            if (SPL == 2) copy16(dst + C::QTILE, src + 4);
                        }
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    __syncwarp();
                }
                uint8_t *row = tile + ((at - u.r0 - t * 128) >> 3) * 128 + (lane & 7) * 16;
                const bool valid = lane < rows;
                if (!p.q_wide || !valid || !std::is_same<T, __half>::value) {
                    float top = 0.f, up = 1.f, down = 1.f;
#pragma unroll 1
                    for (int pass = 0; pass < 2; pass++) {
#pragma unroll 2
                        for (int g = 0; g < groups; g++) {
                            Vec8<T> raw = zero8<T>();
                            if (valid && p.q_wide) {
                                const uint4 a = *(const uint4 *)(row + g * 2048);
                                raw.w[0] = a.x; raw.w[1] = a.y; raw.w[2] = a.z; raw.w[3] = a.w;
                                if (SPL == 2) {
                                    const uint4 b = *(const uint4 *)(row + g * 2048 + C::QTILE);
                                    raw.w[sizeof(T) * 2 - 4] = b.x; raw.w[sizeof(T) * 2 - 3] = b.y; raw.w[sizeof(T) * 2 - 2] = b.z; raw.w[sizeof(T) * 2 - 1] = b.w;
                                }
                            } else if (valid) raw = load8<T>(mine + g * 8, false);
                            float x[8];
                            unpack8(raw, x);
                            if (pass == 0) {
#pragma unroll
                                for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(x[k]));
                                continue;
                            }
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) split2(x[2 * k] * up, x[2 * k + 1] * up, hi[k], lo[k]);
                            *(uint4 *)(row + g * 2048) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            if (SPL == 2) *(uint4 *)(row + g * 2048 + C::QTILE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        }
                        if (pass == 0) power_scale(top, up, down);
                    }
                    factor *= down;
                }
                fence_proxy_async();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(qfull);

            float l = 0.f, mm = 0.f, vref = 0.f;
            // f32 lanes: O so far, [dim][row], and the exponent it was taken against
            float *kept = SPL == 2 ? kept_of(p, R) + (size_t)blockIdx.x * R * p.dim + (size_t)t * 128 * p.dim + quarter * 32 + lane : nullptr;
            float kept_mm = -INFINITY;
            bool fresh = true;                                   // nothing seen yet: mm says nothing
            bool ok = true;
            if (active) {
                int lo, hi;
                row_limits(p, u, min(at, u.r1 - 1), lo, hi);
                const int lo_most = __reduce_max_sync(0xffffffffu, lo), hi_least = __reduce_min_sync(0xffffffffu, hi);
                const int first = (u.t0 + piece.first) * TT;
                for (int j = 0; j < n; j++) {
                    const int base = first + j * TT;
                    const int buf = (tiles + j) & 1;
                    const uint32_t sbar = sfull + 8 * (2 * t + buf), use = (tiles + j) >> 1;
                    const bool whole = base >= lo_most && base + TT <= hi_least;
                    const uint32_t s_at = tmem + lanes + C::s_col(t, buf), o_at = tmem + lanes + C::o_col(t);
                    if (!mbar_wait_soon_lanes(sbar, use & 1, abort, status, STATUS_ATTEND_WAIT)) { ok = false; break; }
                    tc_fence_after();

                    uint32_t v[2][32];
                    tmem_ld32(s_at, v[0]);
                    tmem_ld32(s_at + 32, v[1]);
                    float4 sc[NG];
#pragma unroll
                    for (int e = 0; e < NG; e++) sc[e] = head->scales[(seq + j) % SLOTS][e];
                    vref = sc[NG - 1].w;
                    const uint32_t marks = __float_as_uint(sc[0].w);
                    const float step = sc[1].w;
                    tmem_ld_landed32(v[0]);
                    tmem_ld_landed32(v[1]);
                    __syncwarp();
                    if (lane < 3 - nq) mbar_arrive(kempty + 8 * ((seq + j) % SLOTS));        // K and the scales have been read
                    float x[64];                                 // scores, in powers of two against mm
#pragma unroll
                    for (int i = 0; i < 64; i += 2) {
                        const float f = factor * sc[i / 16].x, a = sc[i / 16].y - mm;
                        unpair(pair_fma(pair(__uint_as_float(v[i / 32][i % 32]), __uint_as_float(v[i / 32][i % 32 + 1])), pair(f, f), pair(a, a)), x[i], x[i + 1]);
                    }
                    if (!whole) {
                        const int from = lo - base, to = hi - base;
#pragma unroll
                        for (int i = 0; i < 64; i++) x[i] = i >= from && i < to ? x[i] : -INFINITY;
                    }
                    float tops[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        tops[q] = max3(x[16 * q], x[16 * q + 1], x[16 * q + 2]);
#pragma unroll
                        for (int i = 3; i < 15; i += 2) tops[q] = max3(tops[q], x[16 * q + i], x[16 * q + i + 1]);
                        tops[q] = fmaxf(tops[q], x[16 * q + 15]);
                    }
                    const float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
                    // seldom: the exponent the weights are taken against goes up
                    const bool above = fresh ? top > -INFINITY : top > 15.f;
                    const bool keep = SPL == 2 && j > 0 && j % C::KEEP == 0;
                    if (keep || step > 0.f || __any_sync(0xffffffffu, above)) {
                        // (or what V's scales are taken against does, seldom: the sums keep their values)
                        float up = 0.f, less = 1.f, o_less = 1.f;
                        if (fresh) {
                            if (top > -INFINITY) up = exponent_for(top, 10.f);
                            fresh = top == -INFINITY;
                        } else {
                            const float down = step > 0.f ? (float)fall_of((int)step, exponent_of(l)) : 0.f;
                            up = top + down > 15.f ? exponent_for(top, 10.f) : -down;
                            less = exp2_fast(-up);
                            o_less = exp2_fast(-up - step);
                        }
                        mm += up;
                        l *= less;
                        kept_mm -= step;
#pragma unroll
                        for (int i = 0; i < 64; i++) x[i] -= up;
                        if (j > 0) {                             // O so far, once the product before has ended
                            // S of the next tile is issued behind that product, so its end is the product's too; the last tile has
                            // no next one, and a barrier of its own
                            const bool last = j + 1 == n;
                            if (!mbar_wait_soon_lanes(last ? odone + 8 * t : sfull + 8 * (2 * t + (buf ^ 1)), (last ? ends : (tiles + j + 1) >> 1) & 1, abort, status,
                                                      STATUS_ATTEND_WAIT)) { ok = false; break; }
                            tc_fence_after();
                            const float kept_less = exp2_fast(kept_mm - mm);
#pragma unroll 1
                            for (int d = 0; d < p.dim; d += 16) {
                                uint32_t w[16];
                                tmem_ld16(o_at + d, w);
                                tmem_ld_landed16(w);
#pragma unroll
                                for (int i = 0; i < 16; i++) w[i] = __float_as_uint(__uint_as_float(w[i]) * o_less);
                                if (keep) {
                                    if (j != C::KEEP) {
#pragma unroll
                                        for (int i = 0; i < 16; i++) w[i] = __float_as_uint(__fmaf_rn(kept[(d + i) * 128], kept_less, __uint_as_float(w[i])));
                                    }
#pragma unroll
                                    for (int i = 0; i < 16; i++) {
                                        kept[(d + i) * 128] = __uint_as_float(w[i]);
                                        w[i] = 0;
                                    }
                                }
                                tmem_st16(o_at + d, w);
                            }
                            if (keep) kept_mm = fresh ? -INFINITY : mm;
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 2; c++) {                // 32 tokens: 16 columns of weights (32: the two f16)
                        uint32_t w[16], w2[16];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                const float *y = x + 32 * c + 16 * e + i;
                                const float e0 = exp2_fast(y[0]), e1 = exp2_fast(y[1]), e2 = exp2_fast(y[2]), e3 = exp2_fast(y[3]);
                                sum0 = pair_add(sum0, pair(e0, e1));
                                sum1 = pair_add(sum1, pair(e2, e3));
                                split2(e0, e1, w[8 * e + i / 2], w2[8 * e + i / 2]);
                                split2(e2, e3, w[8 * e + i / 2 + 1], w2[8 * e + i / 2 + 1]);
                            }
                            float s0, s1;
                            unpair(pair_add(sum0, sum1), s0, s1);
                            l = __fmaf_rn(s0 + s1, sc[2 * c + e].z, l);
                        }
                        tmem_st16(s_at + (SPL == 2 ? 32 : 16) * c, w);
                        if (SPL == 2) tmem_st16(s_at + 32 * c + 16, w2);
                    }
                    tmem_st_wait();
                    if (marks) {                                 // seldom: scales of 0 or below; what was stored is put right
#pragma unroll 1
                        for (int c = 0; c < 2 * SPL; c++) {
                            uint32_t w[16];
                            tmem_ld16(s_at + 16 * c, w);
                            tmem_ld_landed16(w);
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const int e = 2 * (c / SPL) + i / 8;
                                w[i] = marked(w[i], marks >> e & 1, marks >> (16 + e) & 1);
                            }
                            tmem_st16(s_at + 16 * c, w);
                        }
                        tmem_st_wait();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(pfull + 8 * (2 * t + buf));
                }
            }
            seq += n;
            if (active) {
                tiles += n;
                ends += n > 1;
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok || !mbar_wait_lanes(ofull, pieces & 1, abort, status, STATUS_ATTEND_WAIT)) break;
            pieces++;
            if (!active) continue;
            tc_fence_after();
            const bool complete = piece.first == 0 && n == u.nt;
            const int r = at - u.r0;
            float *slot = parts_of(p) + (size_t)(blockIdx.x * 2 + (piece.first ? 0 : 1)) * part_floats(R, p.dim);
            float *part = slot + R * 2 + (size_t)r * p.dim;
            T *dst = out_row<T>(p, u, min(at, u.r1 - 1));
            const float kept_less = exp2_fast(kept_mm - mm);
            const float v0 = vref > 0.f ? vref : 1.f;
            float f = v0 * inverse_of(l);                        // (l is 1/2 at least where a row has seen something)
            if (!complete) {
                if (fresh) mm = NOTHING;
                f = part_scale(mm, l, v0);
            }
#pragma unroll 1
            for (int d = 0; d < p.dim; d += 16) {
                uint32_t v[16];
                tmem_ld16(tmem + lanes + C::o_col(t) + d, v);
                tmem_ld_landed16(v);
                if (SPL == 2 && n > C::KEEP) {
#pragma unroll
                    for (int i = 0; i < 16; i++) v[i] = __float_as_uint(__fmaf_rn(kept[(d + i) * 128], kept_less, __uint_as_float(v[i])));
                }
                if (at < u.r1) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 x = make_float4(__uint_as_float(v[i]) * f, __uint_as_float(v[i + 1]) * f, __uint_as_float(v[i + 2]) * f, __uint_as_float(v[i + 3]) * f);
                        if (complete) store4<T>(dst + d + i, x, p.out_wide);
                        else *(float4 *)(part + d + i) = x;
                    }
                }
            }
            if (at < u.r1) {
                if (complete) store_lse(p, u, at, mm, l);
                else *(float2 *)(slot + r * 2) = make_float2(mm, l);
            }
        }
    } else if (warp < 4 * NQ + CW) {
        // ------------------------------------------------------------------ converters
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::CONV_REGS));
        const int kv = (warp - 4 * NQ) / KW, w = (warp - 4 * NQ) % KW;
        const int8_t *codes = kv ? p.v_codes : p.k_codes;
        const uint32_t full = kv ? vfull : kfull, empty = kv ? vempty : kempty;
        uint8_t *slots = smem + (kv ? C::O_V : C::O_K);
        constexpr int GROUPS = TT / 8 / KW, HALVES = DC / 64;        // groups of 8 tokens a warp; a lane: a token and every fourth chunk of 16 dims
        constexpr int LOADS = GROUPS * HALVES;
        const int r8 = lane & 7, c4 = lane >> 3, chunks = p.dim >> 4;
        // where a chunk's two halves of 8 dims go.  K: core matrices, [8 dims][8 tokens]; V: rows of 64 dims, 128 bytes, with
        // the chunks of a row exchanged by its number (the 128-byte swizzle)
        const int at0 = kv ? w * 1024 + r8 * 128 + ((2 * c4 ^ r8) << 4) : 2 * c4 * (TT * 16) + w * 128 + r8 * 16;
        const int at1 = kv ? w * 1024 + r8 * 128 + (((2 * c4 + 1) ^ r8) << 4) : at0 + TT * 16;
        KvWalk<R, TT> tiles(p, head->start);
        auto page_of = [&](const KvTile<R, TT> &t) {             // lane i: the page of this warp's i-th group
            return page_at(p, t.b, t.base + (lane * KW + w) * 8, 8, t.lo, t.hi, t.there && lane < GROUPS);
        };
        auto load = [&](const KvTile<R, TT> &t, int id, uint4 (&raw)[LOADS]) {
#pragma unroll
            for (int i = 0; i < GROUPS; i++) {
                const int page = __shfl_sync(0xffffffffu, id, i);
                const int token = t.base + (i * KW + w) * 8 + r8;
                const int8_t *row = codes + ((((int64_t)page * p.heads + t.h) << p.log_page) + (token & ((1 << p.log_page) - 1))) * p.dim;
#pragma unroll
                for (int k = 0; k < HALVES; k++)
                    raw[i * HALVES + k] = page >= 0 && c4 + 4 * k < chunks ? __ldg((const uint4 *)row + c4 + 4 * k) : make_uint4(0, 0, 0, 0);
            }
        };
        // three tiles at a time: one is converted, the next one's loads are under way, the page of the one after is asked for
        KvTile<R, TT> now, next;
        now.there = next.there = false;
        Page page = {-1, false};
        uint4 raw[LOADS], coming[LOADS];
        uint32_t seq = 0;
#pragma unroll 1
        do {
            if (next.there) load(next, page_number(p, page, false), coming);
            const KvTile<R, TT> after = tiles.next();
            page = page_of(after);
            if (now.there) {
                const uint32_t slot = seq % SLOTS, use = seq / SLOTS;
                if (use > 0 && !mbar_wait_soon_lanes(empty + 8 * slot, (use - 1) & 1, abort, status, STATUS_ATTEND_WAIT)) break;
                uint8_t *dst = slots + slot * C::SLOT;
#pragma unroll
                for (int i = 0; i < GROUPS; i++)
#pragma unroll
                    for (int k = 0; k < HALVES; k++) {
                        if (c4 + 4 * k < chunks) {
                            uint32_t h[8];
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                const uint32_t x = word(raw[i * HALVES + k], q) ^ 0x80808080u;
                                h[2 * q] = codes_lo(x);
                                h[2 * q + 1] = codes_hi(x);
                            }
                            uint8_t *at = dst + i * (KW * (kv ? 1024 : 128)) + k * (TT * 128);
                            *(uint4 *)(at + at0) = make_uint4(h[0], h[1], h[2], h[3]);
                            *(uint4 *)(at + at1) = make_uint4(h[4], h[5], h[6], h[7]);
                        }
                    }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(full + 8 * slot);
                seq++;
            }
            now = next;
            next = after;
#pragma unroll
            for (int i = 0; i < LOADS; i++) raw[i] = coming[i];
        } while (now.there || next.there);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REST_REGS));
        const int issuer = warp - 4 * NQ - CW;
        if (issuer == 2) {
            // -------------------------------------------------------------- a warp fetches the tiles' scales
            // a lane a group of 16 tokens; pages are asked for two tiles ahead, scales one
            KvWalk<R, TT> walk(p, head->start);
            auto page_of = [&](const KvTile<R, TT> &t) { return page_at(p, t.b, t.base + lane * 16, 16, t.lo, t.hi, t.there && lane < NG); };
            KvTile<R, TT> now, next;
            now.there = next.there = false;
            Page page = {-1, false};
            float2 sc = make_float2(0.f, 0.f);
            bool there = false;
            float vref = 0.f;
            uint32_t seq = 0;
#pragma unroll 1
            do {
                float2 sc_next = make_float2(0.f, 0.f);
                bool there_next = false;
                if (next.there) {
                    const int id = page_number(p, page, true);
                    sc_next = scales_at(p, id, next.h);
                    there_next = id >= 0;
                }
                const KvTile<R, TT> after = walk.next();
                page = page_of(after);
                if (now.there) {
                if (now.starts) vref = 0.f;
                const float before = vref;
                raise(vref, __reduce_max_sync(0xffffffffu, reference_of(there, sc.y)));
                const Weighted v = weighted(there, sc.y, vref);
                const uint32_t marks = __ballot_sync(0xffffffffu, v.mark == MARK_ZERO) | __ballot_sync(0xffffffffu, v.mark == MARK_MINUS) << 16;
                if (seq >= SLOTS && !mbar_wait_soon_lanes(kempty + 8 * (seq % SLOTS), (seq / SLOTS - 1) & 1, abort, status, STATUS_ATTEND_WAIT)) break;
                if (lane < NG) head->scales[seq % SLOTS][lane] = make_float4(sc.x, v.log_ratio, v.inverse, lane == 0 ? __uint_as_float(marks) : lane == 1 && before > 0.f ? (float)(exponent_of(vref) - exponent_of(before)) : lane == 1 ? 0.f : vref);
                __syncwarp();
                if (lane == 0) mbar_arrive(kfull + 8 * (seq % SLOTS));
                seq++;
                }
                now = next;
                sc = sc_next;
                there = there_next;
                next = after;
            } while (now.there || next.there);
        }
        if (issuer < 2 && lane == 0) {
        // ------------------------------------------------------------------ a thread a row tile issues its products
        Walk<R, TT, false> walk(p, head->start);
        Piece piece;
        const uint32_t s_desc = idesc_of(1, 128, TT), o_desc = idesc_of(1, 128, p.dim) | 1u << 16;      // B of the second: a row a dim
        const int t = issuer;
        uint32_t seq = 0, tiles = 0, pieces = 0;               // tiles of the block, of this row tile; pieces
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) { ok = ok && mbar_wait_soon(bar, parity & 1, abort, status, STATUS_ATTEND_WAIT); return ok; };
        // descriptors count addresses in 16 bytes: a step of 16 dims (tokens) is an addition
        const uint64_t q_desc = smem_desc(base_u32 + C::O_Q, 2048, 128), k_desc = smem_desc(base_u32 + C::O_K, TT * 16, 128);
        const uint64_t v_desc = smem_desc(base_u32 + C::O_V, TT * 128, 1024) | (uint64_t)2 << 61;      // 128-byte swizzle
        const int steps = p.dim / 16;
        // V's slots are released by two arrivals: with one row tile both come from its thread
        auto release = [&](uint32_t bar, int nq) {
            mma_commit(bar);
            if (nq == 1) mma_commit(bar);
        };
        auto scores = [&](int j) {
            const uint32_t slot = (seq + j) % SLOTS;
            const int buf = (tiles + j) & 1;
            if (!wait(kfull + 8 * slot, (seq + j) / SLOTS)) return;
            tc_fence_after();
            uint32_t accumulate = 0;
#pragma unroll
            for (int x = SPL - 1; x >= 0; x--) {               // what the cut of q left first: sums are cut off at their size
                uint64_t qd = q_desc + (t * SPL + x) * (C::QTILE >> 4), kd = k_desc + slot * (C::SLOT >> 4);
#pragma unroll 1
                for (int d = 0; d < steps; d++) {
                    mma_issue<1>(tmem + C::s_col(t, buf), qd, kd, s_desc, accumulate);
                    accumulate = 1;
                    qd += 4096 >> 4;
                    kd += TT * 32 >> 4;
                }
            }
            mma_commit(sfull + 8 * (2 * t + buf));
        };
        auto sums = [&](int j, int nq, bool last) {          // last: of those that another tile's weights follow
            const uint32_t slot = (seq + j) % SLOTS;
            const int buf = (tiles + j) & 1;
            if (!wait(vfull + 8 * slot, (seq + j) / SLOTS) || !wait(pfull + 8 * (2 * t + buf), (tiles + j) >> 1)) return;
            tc_fence_after();
            uint64_t vd = v_desc + slot * (C::SLOT >> 4);
            uint32_t col = tmem + C::s_col(t, buf), accumulate = j;
            const uint32_t o_at = tmem + C::o_col(t);
#pragma unroll 1
            for (int s = 0; s < TT / 32; s++) {                // 32 tokens: their weights lie in 16 columns (32: the two f16)
                mma_issue_ts(o_at, col, vd, o_desc, accumulate);
                if (SPL == 2) mma_issue_ts(o_at, col + 16, vd, o_desc, 1);
                vd += 2048 >> 4;
                mma_issue_ts(o_at, col + 8, vd, o_desc, 1);
                if (SPL == 2) mma_issue_ts(o_at, col + 24, vd, o_desc, 1);
                vd += 2048 >> 4;
                col += SPL == 2 ? 32 : 16;
                accumulate = 1;
            }
            if (last) mma_commit(odone + 8 * t);
            release(vempty + 8 * slot, nq);
        };
        while (ok && walk.next(piece)) {
            const int n = piece.count, nq = NQ == 2 && piece.unit.r1 - piece.unit.r0 > 128 ? 2 : 1;
            if (!wait(qfull, pieces)) break;
            tc_fence_after();
            if (t < nq) {
                // S of a tile takes the place of the weights two tiles back: behind their product, in this thread's order
                scores(0);
                for (int j = 0; j < n && ok; j++) {
                    if (j + 1 < n) scores(j + 1);
                    if (ok) sums(j, nq, j + 2 == n);
                }
                if (!ok) break;
                mma_commit(ofull);
                tiles += n;
            } else mbar_arrive(ofull);                         // it has looked at qfull, which may go on to its next phase
            seq += n;
            pieces++;
        }
        // nothing may run on the tensor cores when the block gives its memory back
        mma_commit(drain);
        const long long from = clock64();
        while (!mbar_try_wait(drain, 0) && clock64() - from < WAIT_CYCLES) { }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 4 * NQ + CW) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------------------------- host

template <int DC, int SPL, typename T>
static cudaError_t set_tiles_attr()
{
    cudaFuncAttributes is;
    cudaError_t e = cudaFuncGetAttributes(&is, attend_tiles_kernel<DC, SPL, T>);
    if (e) return e;
    if (is.numRegs != TilesCfg<DC, SPL>::REGS) return cudaErrorInvalidConfiguration;      // its warps share out just these
    return cudaFuncSetAttribute(attend_tiles_kernel<DC, SPL, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)TilesCfg<DC, SPL>::SMEM);
}

cudaError_t attend_tiles_init()
{
    cudaError_t e;
    if ((e = set_tiles_attr<128, 2, float>()) || (e = set_tiles_attr<128, 1, __half>()) || (e = set_tiles_attr<128, 1, __nv_bfloat16>())) return e;
    if ((e = set_tiles_attr<256, 2, float>()) || (e = set_tiles_attr<256, 1, __half>())) return e;
    return set_tiles_attr<256, 1, __nv_bfloat16>();
}

template <int DC, int SPL, typename T>
static int launch_tiles(const AttendArgs &args, cudaStream_t stream)
{
    using C = TilesCfg<DC, SPL>;
    attend_tiles_kernel<DC, SPL, T><<<args.grid, C::THREADS, C::SMEM, stream>>>(args);
    const cudaError_t e = cudaGetLastError();
    return e ? (int)e : launch_join<C::R, C::TT, T>(args, stream);
}

int attend_tiles(const AttendArgs &args, int type, cudaStream_t stream)
{
    if (type == QB200_F32) return args.dim <= 128 ? launch_tiles<128, 2, float>(args, stream) : launch_tiles<256, 2, float>(args, stream);
    if (type == QB200_F16) return args.dim <= 128 ? launch_tiles<128, 1, __half>(args, stream) : launch_tiles<256, 1, __half>(args, stream);
    return args.dim <= 128 ? launch_tiles<128, 1, __nv_bfloat16>(args, stream) : launch_tiles<256, 1, __nv_bfloat16>(args, stream);
}

}  // namespace qb
