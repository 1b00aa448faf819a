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

// Of the calls below each launches something: there are sequences, and there are rows (rows of no sequence would have no
// lengths and offsets to look at).
cudaError_t cache_init(int *status);
int cache_write(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const qb200_lanes_t &k, const qb200_lanes_t &v, cudaStream_t stream);
// either of k and v may have no base
int cache_read(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const qb200_lanes_t &k, const qb200_lanes_t &v, cudaStream_t stream);

// max_queries and max_length have been given values
cudaError_t attend_init(int sm_count, int max_smem, int *status);
size_t attend_workspace_bytes(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const qb200_attention_t &a);
int attend(const qb200_cache_t &c, const qb200_sequences_t &s, int type, const qb200_attention_t &a, cudaStream_t stream);

}  // namespace qb
