// Attention over the 8-bit cache: which kernel takes a call, and how its work is cut.
//
//  * attend_rows.cu: few rows (query heads x tokens that share a head of the cache): the cache's bytes bound it.
//  * attend_tiles.cu: more rows: the tensor cores (tcgen05) take 128 rows of queries at a time.
#include <cuda.h>
#include "common.cuh"
#include "attend_device.cuh"

namespace qb {

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled g_attend_encode = nullptr;
static int *g_attend_status = nullptr;
static int g_attend_sms = 0;
static bool g_attend_tiles = false;        // the tile kernel can run as it is built

// Attention's kernels ask for more of the device and the build than the products do; what they miss is theirs alone.  Without
// the tile kernel the other takes every call; without that, calls are refused.
cudaError_t attend_init(int sm_count, int max_smem, int *status)
{
    g_attend_status = status;
    g_attend_sms = sm_count;
    g_attend_tiles = false;
    if (max_smem < 232448) return cudaErrorInvalidValue;
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found);
    if (e) return e;
    if (found != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
    g_attend_encode = (EncodeTiled)fn;
    if ((e = attend_rows_init())) return e;
    g_attend_tiles = attend_tiles_init() == cudaSuccess;
    return cudaSuccess;
}

// What a call is cut into: rows a unit, by the kernel that takes it.
struct Plan {
    bool tiles;                // attend_tiles.cu
    int r;
    bool whole;                // no unit is cut: units are short, and cutting them would cost a second launch
};

static Plan plan_of(const qb200_cache_t &c, const qb200_sequences_t &s, const qb200_attention_t &a)
{
    const int64_t rows = (int64_t)(a.q_heads / c.heads) * a.max_queries;
    Plan plan;
    // Few rows: attend_rows.cu, which reads the cache (from the L2 after the first time) once for every 16 rows of a head, 8
    // where dim is over 128.  Measured at 8 sequences of 6000 tokens, 4 heads, bf16, us (rows, then tiles): dim 128: 16 rows
    // 26 and 51, 32 rows 36 and 52, 64 rows 47 and 53, 96 rows 74 and 55; dim 256: 16 rows 44 and 86, 40 rows 81 and 88, 64
    // rows 121 and 92; dim 64: 64 rows 32 and 39, 96 rows 49 and 41.
    plan.tiles = g_attend_tiles && rows > (c.dim <= 128 ? 64 : 48);
    plan.r = plan.tiles ? (c.dim <= 128 ? 256 : 128) : c.dim <= 128 && rows > 8 ? 16 : 8;
    // Units cut (equal shares, a second kernel) or each to a block of its own.  In tokens of 128 dims a block takes (about 11
    // cycles each): a unit costs 256 besides its tokens where the blocks stay, 556 where each has its own, the cut ones' partition
    // and second kernel 1500 once.  Measured, 8 heads, bf16, us (whole, cut): 1 sequence of 500 tokens 6.9 and 10.1, of 1000
    // 9.4 and 10.7, of 2000 14.6 and 11.6; 16 sequences of 2000 18 and 23; 64 of 1000 42 and 38.
    const int64_t units = (int64_t)s.count * c.heads * ((rows + plan.r - 1) / plan.r);
    const int64_t length = (int64_t)a.max_length * c.dim / 128, waves = (units + g_attend_sms - 1) / (g_attend_sms > 0 ? g_attend_sms : 1);
    plan.whole = !plan.tiles && units < 1 << 30 && waves * (length + 556) <= units * (length + 256) / (g_attend_sms > 0 ? g_attend_sms : 1) + 1500;
    return plan;
}

size_t attend_workspace_bytes(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const qb200_attention_t &a)
{
    const Plan plan = plan_of(c, s, a);
    if (plan.whole) return 0;
    const size_t kept = plan.tiles && type == QB200_F32 ? (size_t)plan.r * c.dim : 0;
    return marks_bytes(g_attend_sms) + (size_t)g_attend_sms * (2 * part_floats(plan.r, c.dim) + kept) * 4;
}

// The codes as rows of dim bytes, fetched box_rows tokens and box_dim dims at a time (zeros past dim).
static bool codes_map(CUtensorMap &map, const void *codes, const qb200_cache_t &c, int box_dim, int box_rows)
{
    const cuuint64_t dims[2] = { (cuuint64_t)c.dim, (cuuint64_t)c.pages * c.heads * c.page }, strides[1] = { (cuuint64_t)c.dim };
    const cuuint32_t box[2] = { (cuuint32_t)box_dim, (cuuint32_t)box_rows }, estr[2] = { 1, 1 };
    return g_attend_encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           box_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int attend(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const qb200_attention_t &call, cudaStream_t stream)
{
    const int size = type == QB200_F32 ? 4 : 2;
    AttendArgs a;
    a.seq = s;
    a.q = call.q;
    a.out = call.out;
    a.lse = call.lse;
    a.k_codes = (const int8_t *)c.k_codes;
    a.v_codes = (const int8_t *)c.v_codes;
    a.k_scales = c.k_scales;
    a.v_scales = c.v_scales;
    a.pages = c.pages;
    a.heads = c.heads;
    a.dim = c.dim;
    a.log_page = c.page == 16 ? 4 : c.page == 32 ? 5 : c.page == 64 ? 6 : 7;
    a.group = call.q_heads / c.heads;
    a.q_heads = call.q_heads;
    int log_group = 0;
    while (((int64_t)1 << log_group) < a.group) log_group++;
    a.group_shift = 31 + log_group;
    a.group_magic = (uint32_t)((((uint64_t)1 << a.group_shift) + a.group - 1) / a.group);
    a.causal = call.causal != 0;
    a.window = call.window;
    a.scale = call.scale;
    a.q_wide = ((uintptr_t)call.q.base & 15) == 0 && call.q.row_stride * size % 16 == 0 && call.q.head_stride * size % 16 == 0;
    a.out_wide = ((uintptr_t)call.out.base & (4 * size - 1)) == 0 && call.out.row_stride % 4 == 0 && call.out.head_stride % 4 == 0;
    a.workspace = call.workspace;
    a.status = g_attend_status;
    const Plan plan = plan_of(c, s, call);
    a.chunks = (int)(((int64_t)a.group * call.max_queries + plan.r - 1) / plan.r);
    a.whole = plan.whole;
    const int64_t units = (int64_t)s.count * c.heads * a.chunks;
    a.grid = plan.whole ? (int)(units < 1 << 20 ? units : 1 << 20) : g_attend_sms;
    if (plan.tiles) return attend_tiles(a, type, stream);
    CUtensorMap kmap, vmap;
    const int box = c.dim <= 64 ? 64 : 128, rows = c.page < 32 ? c.page : 32;
    if (!codes_map(kmap, c.k_codes, c, box, rows) || !codes_map(vmap, c.v_codes, c, box, rows)) return (int)cudaErrorInvalidValue;
    return attend_rows(a, type, plan.r, kmap, vmap, stream);
}

}  // namespace qb
