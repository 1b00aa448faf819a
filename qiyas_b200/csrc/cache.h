// Launch interface of the cache operators (cache.cu, attend_rows.cu) and what their kernels share.  As in launch.h, every
// function returns 0, a negative QB200_E_* code or a positive cudaError_t; arguments have been validated by the caller.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/qiyas_b200.h"

namespace qb {

// status bits of the cache operators (the word of qb200_device_status)
constexpr int STATUS_ATTEND_WAIT = 8;
constexpr int STATUS_CACHE_RANGE = 16;
constexpr int STATUS_CACHE_VALUE = 32;

struct Lanes {                  // element (row, head, i) at base + row * row + head * head + i
    void *base;
    int64_t row, head;
};

cudaError_t cache_init(int *status);
int cache_write(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const Lanes &k, const Lanes &v, cudaStream_t stream);
int cache_read(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const Lanes &k, const Lanes &v, cudaStream_t stream);

struct AttendCall {
    qb200_cache_t cache;
    qb200_sequences_t seq;
    Lanes q, out;
    float *lse;
    int type, q_heads, max_queries, max_length, causal, window;
    float scale;
    void *workspace;
};
cudaError_t attend_init(int sm_count, int max_smem, int *status);
size_t attend_workspace_bytes(int dim, int heads, int type, int count, int rows, int q_heads, int max_queries, int max_length);
int attend(const AttendCall &call, cudaStream_t stream);

}  // namespace qb
