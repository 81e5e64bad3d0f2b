// stream_ops.h — streaming time-axis attention: per-head norms with rotary
// positions, a rolling key/value cache, attention over a sliding window with
// visible first tokens (prompt form and few-token form).  Arguments as in
// include/mbr_b200.h; every function throws mbr::Error on a bad argument,
// enqueues on `st` and returns.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/mbr_b200.h"

namespace mbr {
namespace streamops {

void qk_norm_rope(const mbr_view& q, const mbr_view& k, const mbr_view& qo, const mbr_view& ko, int64_t seqs,
                  int64_t tokens, int Hq, int Hkv, int D, const float* gamma_q, const float* gamma_k, float eps,
                  const float* cs, const float* sn, int64_t table_rows, const int32_t* pos, int axes,
                  const int* pairs, int dtype, cudaStream_t st);

void cache_append(const mbr_kv_cache& c, const mbr_view& k, const mbr_view& v, const int32_t* pos,
                  const int32_t* count, int64_t tokens, cudaStream_t st);
void cache_read(const mbr_kv_cache& c, const int32_t* pos, const int32_t* count, int64_t tokens, const mbr_view& k,
                const mbr_view& v, cudaStream_t st);

void window_attention(const mbr_view& q, const mbr_view& k, const mbr_view& v, const mbr_view& out, int64_t seqs,
                      int64_t Nq, int64_t Nk, int Hq, int Hkv, int D, const int32_t* q_len, const int32_t* kv_len,
                      int left, int right, int sinks, float scale, const float* gates, int dtype, void* workspace,
                      int64_t workspace_bytes, cudaStream_t st);
int64_t window_attention_workspace(int64_t seqs, int64_t Nq, int64_t Nk, int Hq, int Hkv, int D, int left, int right,
                                   int sinks, int dtype);
void cache_attention(const mbr_view& q, const mbr_kv_cache& c, const mbr_view& out, const int32_t* length,
                     int64_t tokens, int Hq, int left, int right, float scale, const float* gates, void* workspace,
                     int64_t workspace_bytes, cudaStream_t st);
int64_t cache_attention_workspace(const mbr_kv_cache& c, int64_t tokens, int Hq, int left, int right);

// Current device (checked against the per-device tables below).
constexpr int kMaxStreamDevices = 64;
int stream_device();
// Error word that the bounded waits of this stream's attention kernels set
// (KERR_* of sm100.cuh), host-mapped, never freed.
int* stream_error_word(cudaStream_t st);
// Throws if the stream's word is set, and clears it: an earlier call ran out of a wait.
void raise_stream_error(cudaStream_t st);
// The same after what the stream holds has run.
void stream_check(cudaStream_t st);

// Checks a cache's sizes and type; check_cache its buffers too (true when its rows are 4-bit codes).
void check_cache_fields(const mbr_kv_cache& c);
bool check_cache(const mbr_kv_cache& c);
// True if every row of the view starts on a 16-byte boundary (es: element size).
inline bool rows_aligned16(const mbr_view& v, int es) {
    return (((uintptr_t)v.data | (uintptr_t)(v.seq * es) | (uintptr_t)(v.token * es) | (uintptr_t)(v.head * es)) &
            15) == 0;
}

}  // namespace streamops
}  // namespace mbr
