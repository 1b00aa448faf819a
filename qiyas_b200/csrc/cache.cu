// A cache of keys and values in 8 bits: what is written is quantised on the way in, and read back.
//
// A block is `page` tokens of one sequence in one head: int8 codes [page][dim], contiguous, and one f32 scale.  The
// arithmetic (also in the header): n = max|x| * (1/127); the scale s of a block that holds earlier tokens stays where n <= |s|,
// else it becomes max(n, 1.25 |s|) and the earlier codes c are rounded again to rn(c * s / scale); new codes are
// rn(x / scale).  Growth by a quarter at least bounds what repeated rounding costs: the errors of the earlier roundings
// shrink by 4/5 with each later one, half a step * 1 / (1 - 4/5) = 2.5 steps, whatever the number of tokens.
//
// One group of threads (a warp, or a whole block of several) owns one (sequence, page, head, K or V), so a scale has one
// writer and nothing is atomic.  A group holds everything it writes in registers: each value is read once.  Which sequence
// and page a group has follows from the rows' offsets alone: sequence b gets rows/page + 2 places, as many as it can touch.
//
// The memory bounds long prompts: 25 370 tokens of 8 heads x 128 in f16, pages of 64, are written in 42 us and read back in 27,
// 4.5 TB/s together (69 % of the copy peak); 43 288 tokens in bf16, pages of 16, are read back at 5.4 TB/s (83 %).  A write is
// 10 instructions a value, and three quarters of the issue slots are taken: the largest magnitude as bits, two values at a time (it was 5 a value in floats, 65 us), and the check of the
// rounding eight values at a time.  One token a sequence is a launch's latency, 3 to 5 us
// (64 sequences, 8 heads x 128, pages of 16, replayed: 3.2 us); where a block's scale grows the serial loop over its earlier codes
// shows: 12 us if a tenth of the blocks grow, 13 if all do (pages of 64: 5.7, 18.6, 24.8).
#include "common.cuh"
#include "cache.h"
#include "cache_device.cuh"

namespace qb {

static int *g_cache_status = nullptr;

struct CacheArgs {
    qb200_lanes_t lanes[2];
    int8_t *codes[2];
    float *scales[2];
    qb200_sequences_t seq;
    int pages, heads, page, dim;
    int log_page;
    int items;                 // places: (sequence, page) pairs
    int wide;                  // bit i: lanes[i] may be read and written 16 bytes at a time
    int *status;
};

struct Item {                  // tokens [first, first + count) of page `page` of a sequence, rows from `row`
    int page;                  // -1: nothing to do
    int first, count;          // inside the page
    int row;
};

// Which sequence place `item` belongs to: the last b with floor(offsets[b] / page) + 2 b <= item, by a search in which
// every lane of the warp looks at another sequence.
__device__ __forceinline__ int sequence_of(const CacheArgs &p, int item)
{
    if (!p.seq.offsets) return item;
    const int lane = threadIdx.x & 31;
    int lo = 0, n = p.seq.count;                     // the answer is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int b = lo + lane * step;
        bool at = false;
        if (lane * step < n) at = (p.seq.offsets[b] >> p.log_page) + 2 * b <= item;
        const unsigned mask = __ballot_sync(0xffffffffu, at);
        const int k = mask ? 31 - __clz(mask) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

__device__ __forceinline__ Item item_of(const CacheArgs &p, int item)
{
    Item it;
    it.page = -1;
    it.first = it.count = it.row = 0;
    if (item >= p.items) return it;
    const int b = sequence_of(p, item);
    int row, n;
    bool bad;
    seq_rows(p.seq, b, row, n, bad);
    const int start = p.seq.lengths[b];
    const int capacity = p.seq.width << p.log_page;   // below 2^31: checked on the host
    const int slot = p.seq.offsets ? item - ((p.seq.offsets[b] >> p.log_page) + 2 * b) : 0;
    if (start < 0 || start > capacity || n > capacity - start) {
        bad = true;
        if (start < 0 || start > capacity) n = 0;
        else n = capacity - start;
    }
    const int page0 = start >> p.log_page;
    const int lo = max(start, (page0 + slot) << p.log_page);
    const int hi = min(start + n, (page0 + slot + 1) << p.log_page);
    if (slot >= 0 && page0 + slot < p.seq.width && hi > lo) {
        const int page = p.seq.table[(int64_t)b * p.seq.width + page0 + slot];
        if (page >= 0 && page < p.pages) {
            it.page = page;
            it.first = lo & (p.page - 1);
            it.count = hi - lo;
            it.row = row + lo - start;
        } else bad = true;
    }
    if (bad && (threadIdx.x & 31) == 0) atomicOr(p.status, STATUS_CACHE_RANGE);
    return it;
}

// Eight x / scale to the nearest integers, ties to even, from the exact quotients.  Adding 1.5 * 2^23 to the product with
// the reciprocal rounds it; the sum's low byte is the code.  The product is off by less than 2^-16, so only a quotient next to
// a half can go to the wrong side, and the remainder x - q * scale, which an fma gives exactly here, says so.  That is looked
// at for the eight together: seldom is there one.
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float scale, float inverse, float half)
{
    constexpr float MAGIC = 12582912.f;
    float m[8], most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        m[i] = __fmaf_rn(x[i], inverse, MAGIC);
        most = fmaxf(most, fabsf(__fmaf_rn(-__fsub_rn(m[i], MAGIC), scale, x[i])));
    }
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; i++) c[i] = __float_as_uint(m[i]);
    if (most >= half) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float r = __fmaf_rn(-__fsub_rn(m[i], MAGIC), scale, x[i]);
            if (fabsf(r) > half || (fabsf(r) == half && (c[i] & 1u))) c[i] += r > 0.f ? 1u : 0xffffffffu;
        }
    }
    uint2 w;
    w.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    w.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
    return w;
}

// The same for scales whose reciprocal leaves the type's range or whose half is not exact, for a caller's scales below zero, and
// for NaN and infinities.
__device__ __noinline__ uint32_t code_of_any(float x, float scale)
{
    if (scale == 0.f || x != x) return 0;
    if (fabsf(x) > 3.402823466e38f) return (uint32_t)((x > 0.f) == (scale > 0.f) ? 127 : -127) & 0xffu;
    const double q = rint((double)x / (double)scale);
    return (uint32_t)(int)fmin(fmax(q, -127.), 127.) & 0xffu;
}

constexpr int NV = 8;          // vectors of eight values a thread holds
// threads a block: four items of a warp each, or one item
__host__ __device__ constexpr int item_threads(int lanes) { return lanes == 32 ? 128 : lanes; }

// LANES threads own one item (32: several items a block; more: the block has one).
template <typename T, int LANES>
__global__ void __launch_bounds__(item_threads(LANES)) cache_write_kernel(const __grid_constant__ CacheArgs p)
{
    constexpr int THREADS = item_threads(LANES);
    constexpr int PER = THREADS / LANES;
    __shared__ uint32_t s_max[32];
    const int group = threadIdx.x / LANES, tid = threadIdx.x % LANES;
    const Item it = item_of(p, blockIdx.x * PER + group);
    if (it.page < 0) return;                       // uniform over the group; with one group a block, over the block
    const int head = blockIdx.y, kv = blockIdx.z;
    const int vecs = p.dim >> 3, total = it.count * vecs;
    const T *src = (const T *)p.lanes[kv].base + (int64_t)it.row * p.lanes[kv].row_stride + (int64_t)head * p.lanes[kv].head_stride;
    const int64_t stride = p.lanes[kv].row_stride;
    const bool wide = (p.wide >> kv) & 1;
    const int64_t block = (int64_t)it.page * p.heads + head;
    int8_t *codes = p.codes[kv] + (block << p.log_page) * p.dim;
    float *scale_at = p.scales[kv] + block;
    const float had = it.first ? *scale_at : 0.f;

    // one pass over the new rows: into registers, with their largest magnitude
    Vec8<T> x[NV];
    {
        int row = tid / vecs, col = tid % vecs;
        const int drow = LANES / vecs, dcol = LANES % vecs;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            x[j] = tid + j * LANES < total ? load8<T>(src + row * stride + col * 8, wide) : zero8<T>();
            row += drow;
            col += dcol;
            if (col >= vecs) { col -= vecs; row++; }
        }
    }
    // magnitudes compare as their bits do, and infinities and NaN lie above all others
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < NV; j++) bits = largest8(x[j], bits);
    bits = largest_of(bits, (const T *)nullptr);
    bits = __reduce_max_sync(0xffffffffu, bits);
    if (LANES > 32) {
        if ((tid & 31) == 0) s_max[tid >> 5] = bits;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < LANES / 32; w++) bits = max(bits, s_max[w]);
    }
    float top = magnitude(bits, (const T *)nullptr);
    const bool odd = !(top <= 3.402823466e38f);
    if (odd) {                                     // seldom: the largest of the finite ones
        top = 0.f;
#pragma unroll 1
        for (int j = 0; j < NV; j++) {
            float v[8];
            unpack8(x[0], v);
#pragma unroll
            for (int k = 1; k < NV; k++)
                if (k == j) unpack8(x[k], v);
#pragma unroll
            for (int i = 0; i < 8; i++) top = fabsf(v[i]) <= 3.402823466e38f ? fmaxf(top, fabsf(v[i])) : top;
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (LANES > 32) {
            __syncthreads();
            if ((tid & 31) == 0) s_max[tid >> 5] = __float_as_uint(top);
            __syncthreads();
#pragma unroll
            for (int w = 0; w < LANES / 32; w++) top = fmaxf(top, __uint_as_float(s_max[w]));
        }
    }
    if (odd && tid == 0) atomicOr(p.status, STATUS_CACHE_VALUE);

    const float need = __fmul_rn(top, 1.f / 127.f);
    const float scale = need <= fabsf(had) ? had : fmaxf(need, __fmul_rn(fabsf(had), 1.25f));
    if (scale != had && it.first) {
        // the earlier tokens' codes in the new scale (exact products, correctly rounded quotients): zeros where it was 0
        const int words = it.first * p.dim >> 2;
        uint32_t *old = (uint32_t *)codes;
        const double s0 = had, s1 = scale;
        for (int i = tid; i < words; i += LANES) {
            const uint32_t w = old[i];
            uint32_t n = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) n |= ((uint32_t)(int)rint((double)(int8_t)(w >> 8 * k) * s0 / s1) & 0xffu) << 8 * k;
            old[i] = n;
        }
    }
    if (LANES == 32) __syncwarp();                 // every lane has read the scale (a block of several warps met above)
    if (tid == 0 && (scale != had || !it.first)) *scale_at = scale;

    uint2 *dst = (uint2 *)(codes + it.first * p.dim);
    // the quick form needs a reciprocal and a half inside the normal numbers
    const bool plain = !odd && scale > 1e-30f && scale < 1e30f;
    const float inverse = plain ? __fdiv_rn(1.f, scale) : 0.f, half = 0.5f * scale;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (tid + j * LANES >= total) break;
        float v[8];
        unpack8(x[j], v);
        uint2 w;
        if (plain) w = codes_of(v, scale, inverse, half);
        else {
            uint32_t c[8];
#pragma unroll
            for (int i = 0; i < 8; i++) c[i] = code_of_any(v[i], scale);
            w.x = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
            w.y = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
        }
        dst[tid + j * LANES] = w;
    }
}

// Byte i of a word of codes as a float: under the exponent of 2^23 the code + 128 is the last byte.  (Conversions from integers
// run on the unit of the exponentials, a quarter as wide: it was 81 % busy, and reading took 31 us where it takes 27.)
__device__ __forceinline__ float code_at(uint32_t w, int i)
{
    return __fsub_rn(__uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7440 + i)), 8388736.f);
}

template <typename T, int LANES>
__global__ void __launch_bounds__(item_threads(LANES)) cache_read_kernel(const __grid_constant__ CacheArgs p)
{
    constexpr int THREADS = item_threads(LANES);
    constexpr int PER = THREADS / LANES;
    const int group = threadIdx.x / LANES, tid = threadIdx.x % LANES;
    const int kv = blockIdx.z;
    if (!p.lanes[kv].base) return;
    const Item it = item_of(p, blockIdx.x * PER + group);
    if (it.page < 0) return;
    const int head = blockIdx.y;
    const int vecs = p.dim >> 3, total = it.count * vecs;
    const int64_t block = (int64_t)it.page * p.heads + head;
    const uint2 *src = (const uint2 *)(p.codes[kv] + (block << p.log_page) * p.dim + it.first * p.dim);
    const float scale = p.scales[kv][block];
    T *dst = (T *)p.lanes[kv].base + (int64_t)it.row * p.lanes[kv].row_stride + (int64_t)head * p.lanes[kv].head_stride;
    const int64_t stride = p.lanes[kv].row_stride;
    const bool wide = (p.wide >> kv) & 1;
    uint2 c[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) c[j] = tid + j * LANES < total ? src[tid + j * LANES] : make_uint2(0, 0);
    int row = tid / vecs, col = tid % vecs;
    const int drow = LANES / vecs, dcol = LANES % vecs;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (tid + j * LANES >= total) break;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __fmul_rn(code_at(i < 4 ? c[j].x : c[j].y, i & 3), scale);
        store8<T>(dst + row * stride + col * 8, v, wide);
        row += drow;
        col += dcol;
        if (col >= vecs) { col -= vecs; row++; }
    }
}

cudaError_t cache_init(int *status)
{
    g_cache_status = status;
    return cudaSuccess;
}

static CacheArgs args_of(const qb200_cache_t &c, const qb200_sequences_t &s, int size, const qb200_lanes_t &k, const qb200_lanes_t &v)
{
    CacheArgs p;
    p.lanes[0] = k;
    p.lanes[1] = v;
    p.codes[0] = (int8_t *)c.k_codes;
    p.codes[1] = (int8_t *)c.v_codes;
    p.scales[0] = c.k_scales;
    p.scales[1] = c.v_scales;
    p.seq = s;
    p.pages = c.pages;
    p.heads = c.heads;
    p.page = c.page;
    p.dim = c.dim;
    p.log_page = c.page == 16 ? 4 : c.page == 32 ? 5 : c.page == 64 ? 6 : 7;
    p.items = s.offsets ? s.rows / c.page + 2 * s.count : s.count;
    p.wide = 0;
    for (int i = 0; i < 2; i++)
        if (((uintptr_t)p.lanes[i].base & 15) == 0 && p.lanes[i].row_stride * size % 16 == 0 && p.lanes[i].head_stride * size % 16 == 0) p.wide |= 1 << i;
    p.status = g_cache_status;
    return p;
}

template <typename T, int LANES>
static void launch(bool write, const CacheArgs &p, cudaStream_t stream)
{
    constexpr int THREADS = item_threads(LANES), PER = THREADS / LANES;
    const dim3 grid((p.items + PER - 1) / PER, p.heads, 2);
    if (write) cache_write_kernel<T, LANES><<<grid, THREADS, 0, stream>>>(p);
    else cache_read_kernel<T, LANES><<<grid, THREADS, 0, stream>>>(p);
}

template <typename T>
static int run(bool write, const CacheArgs &p, cudaStream_t stream)
{
    const int values = p.page * p.dim;        // a group of LANES threads holds LANES * 64 values
    if (values <= 2048) launch<T, 32>(write, p, stream);
    else if (values <= 4096) launch<T, 64>(write, p, stream);
    else if (values <= 8192) launch<T, 128>(write, p, stream);
    else if (values <= 16384) launch<T, 256>(write, p, stream);
    else launch<T, 512>(write, p, stream);
    return (int)cudaGetLastError();
}

static int dispatch(bool write, int type, const CacheArgs &p, cudaStream_t stream)
{
    if (type == QB200_F32) return run<float>(write, p, stream);
    if (type == QB200_F16) return run<__half>(write, p, stream);
    return run<__nv_bfloat16>(write, p, stream);
}

int cache_write(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const qb200_lanes_t &k, const qb200_lanes_t &v, cudaStream_t stream)
{
    return dispatch(true, type, args_of(c, s, type == QB200_F32 ? 4 : 2, k, v), stream);
}

int cache_read(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const qb200_lanes_t &k, const qb200_lanes_t &v, cudaStream_t stream)
{
    return dispatch(false, type, args_of(c, s, type == QB200_F32 ? 4 : 2, k, v), stream);
}

}  // namespace qb
