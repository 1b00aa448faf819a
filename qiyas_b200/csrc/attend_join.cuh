// The second kernel of an attention call whose work was cut inside sequences.
#pragma once

#include "attend_device.cuh"

namespace qb {

// Joins the parts of the units that a share's end cuts: block c looks after the unit that the c-th boundary cuts first.
template <int R, int TT, typename T>
__global__ void __launch_bounds__(256) attend_join_kernel(const __grid_constant__ AttendArgs p)
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int block = blockIdx.x + 1;
    const Mark mark = ((const Mark *)p.workspace)[block];
    const Line &line = mark.line;
    const Start &cut = line.start;
    const int64_t place = line.at(block);
    // not inside a unit's tiles, or not the first boundary inside them
    if (block >= line.shares || cut.left == 0 || cut.at <= unit_pad(TT) || cut.at - unit_pad(TT) > place - line.at(block - 1)) return;
    const int64_t end = place - cut.at + unit_pad(TT) + mark.nt;
    int parts = 1;
#pragma unroll 1
    for (int k = block; k < line.shares && line.at(k) < end; k++) parts++;
    const Unit u = unit_of<R, TT>(p, sequence_at(p, cut.b), cut.b, cut.h, cut.rc);
    const int rows = u.r1 - u.r0, quads = p.dim / 4;
    const size_t size = part_floats(R, p.dim);
    const float *first = parts_of(p) + (size_t)((block - 1) * 2 + 1) * size;      // the part that begins the unit
    for (int i = blockIdx.y * 256 + threadIdx.x; i < rows * quads; i += 256 * gridDim.y) {
        const int r = i / quads, d = (i - r * quads) * 4;
        float m = NOTHING, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int k0 = 0; k0 < parts; k0 += 8) {            // eight parts' loads at a time, in the order of the tokens
            float2 s[8];
            float4 x[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                s[k] = make_float2(NOTHING, 0.f);
                x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k0 + k < parts) {
                    const float *part = first + (k0 + k ? (size_t)(2 * (k0 + k) - 1) * size : 0);
                    s[k] = *(const float2 *)(part + r * 2);
                    x[k] = *(const float4 *)(part + R * 2 + r * p.dim + d);
                }
            }
            float top = m;
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, s[k].x);
            const float less = exp2_fast(m - top);
            m = top;
            sum *= less;
            acc = make_float4(acc.x * less, acc.y * less, acc.z * less, acc.w * less);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float f = exp2_fast(s[k].x - m);
                sum = __fmaf_rn(s[k].y, f, sum);
                acc.x = __fmaf_rn(x[k].x, f, acc.x);
                acc.y = __fmaf_rn(x[k].y, f, acc.y);
                acc.z = __fmaf_rn(x[k].z, f, acc.z);
                acc.w = __fmaf_rn(x[k].w, f, acc.w);
            }
        }
        finish_row<T>(p, u, u.r0 + r, d, acc, m, sum);
    }
}

// Launched beside the kernel whose parts it joins (a programmatic dependent: it waits for that kernel's end itself).
template <int R, int TT, typename T>
static int launch_join(const AttendArgs &args, cudaStream_t stream)
{
    if (args.grid < 2) return 0;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(args.grid - 1, R > 16 ? R / 32 : 1);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, attend_join_kernel<R, TT, T>, args);
}

}  // namespace qb
