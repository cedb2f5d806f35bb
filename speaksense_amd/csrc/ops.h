// Operators on a caller's device buffers (include/speaksense.h, "decoder operators"): launch wrappers of kernels_kv.hip and kernels_sample.hip.
// The caller's structs arrive checked (capi.cpp); every launch goes to the caller's stream on the current device and returns without waiting.
#pragma once
#include "../../include/speaksense.h"
#include "common.h"

namespace ss {

void launch_kv_append(const ss_kv_cache& c, const ss_kv_batch& b, const ss_kv_rows& k, const ss_kv_rows& v, hipStream_t st);
void launch_kv_read(const ss_kv_cache& c, const ss_kv_batch& b, const ss_kv_rows& k, const ss_kv_rows& v, hipStream_t st);

// How one attention call is cut: a pure function of the host-known sizes, so that the workspace query and the launch agree.
struct KvPlan {
    bool tile;                 // the tile kernel; else that of at most 16 query rows per key head
    int qc;                    // tile kernel: 16-row column tiles per wave
    int splits, split_keys;    // key ranges per sequence and their length
    int64_t workspace;         // bytes of partial results
};
KvPlan kv_attention_plan(const ss_kv_cache& c, const ss_kv_batch& b, int n_heads);
void launch_kv_attention(const ss_kv_cache& c, const ss_kv_batch& b, const ss_kv_rows& q, int n_heads, float scale, bool causal, const ss_kv_rows& out,
                         float* lse, void* workspace, hipStream_t st);

void launch_sample_rows(const ss_sample_rows_args& a, hipStream_t st);

}  // namespace ss
