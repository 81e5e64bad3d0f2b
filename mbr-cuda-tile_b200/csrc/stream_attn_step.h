// stream_attn_step.h — attention of a few queries over many keys (fp16/bf16).
#pragma once

#include "stream_attn.cuh"

namespace mbr {
namespace streamops {

// How a call is divided: items are (sequence, key head, row tile), each walked
// in `parts` parts whose results lie in the workspace.
struct StepPlan {
    int64_t items, tiles;
    int parts, rows;  // rows: of a tile
    bool half;        // at most 8 rows
    int64_t bytes;    // workspace
};
// keys: the most keys any tile can see.
StepPlan step_plan(int64_t seqs, int64_t tokens, int Hq, int Hkv, int D, int64_t keys);

struct StepArgs {
    AttnArgs a;
    // byte strides of key, value and (4 bits) step/offset rows
    int64_t k_seq, k_head, k_tok, v_seq, v_head, v_tok, s_seq, s_head;
    float scale_log2;  // scale * log2(e)
    int64_t items, tiles;
    int parts, rows, half;
    int q_vec;        // query rows are 16-byte aligned
    int packed;       // a token's row follows the one before it
    float* part_o;    // [items * parts][rows][DP]
    float2* part_ml;  // [items * parts][rows] (offset, sum)
    int* err;         // error word of bounded waits
};

bool step_supported(const AttnArgs& a, int dtype, bool cached);
void attend_step(const AttnArgs& a, int dtype, bool cached, bool q4, const StepPlan& plan, void* workspace,
                 cudaStream_t st);

}  // namespace streamops
}  // namespace mbr
