// stream_attn_tc.h — windowed attention of many queries on the tensor cores (fp16/bf16).
#pragma once

#include "stream_attn.cuh"

namespace mbr {
namespace streamops {

// Layouts its TMA maps take: 16-byte rows in q, k, v and out.
bool tile_supported(const AttnArgs& a, int dtype);
void attend_tiles(const AttnArgs& a, int dtype, cudaStream_t st);

}  // namespace streamops
}  // namespace mbr
