// stream_attn_step.h — attention of a few queries over many keys (fp16/bf16).
#pragma once

#include "stream_attn.cuh"

namespace mbr {
namespace streamops {

// How a call is divided.  Items are (sequence, key head, row tile); `outer` CTAs
// share an item's keys, and in each of them a group of `inner` warps (a power of
// two).
struct StepPlan {
    int64_t items, tiles;
    int inner, outer, rows;  // rows: of a tile
    bool half;               // at most 8 rows
    int64_t bytes;           // workspace: the results of `outer` CTAs, which a second kernel joins (0: none)
};
// keys: the most keys any tile can see.
StepPlan step_plan(int64_t seqs, int64_t tokens, int Hq, int Hkv, int D, bool q4, int64_t keys);
// Warps of a CTA (one CTA an SM) for a head size of up to dp.  16-bit rows need
// bytes in flight more than warps (heads of 64: 29.5 us with 8 warps against 32
// with 16 for a frame over 1000 keys); codes need issue slots filled (334 us with 8
// against 263 with 16 for 960 sequences).
constexpr int step_warps(int dp, bool q4) { return q4 && dp < 128 ? 16 : 8; }

struct StepArgs {
    AttnArgs a;
    // byte strides of key, value and (4 bits) step/offset rows
    int64_t k_seq, k_head, k_tok, v_seq, v_head, v_tok, s_seq, s_head;
    float scale_log2;  // scale * log2(e)
    unsigned items;
    int tiles, inner_log2, outer, rows, half;
    FastDiv by_tiles, by_outer;
    int q_vec;        // query rows are 16-byte aligned
    float* part_o;    // [items * outer][rows][DP]
    float2* part_ml;  // [items * outer][rows] (offset, sum)
    int* err;         // error word of bounded waits
};

bool step_supported(const AttnArgs& a, int dtype, bool cached);
void attend_step(const AttnArgs& a, int dtype, bool cached, bool q4, const StepPlan& plan, void* workspace,
                 cudaStream_t st);

}  // namespace streamops
}  // namespace mbr
