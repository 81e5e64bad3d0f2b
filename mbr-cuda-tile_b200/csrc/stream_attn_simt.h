// stream_attn_simt.h — windowed attention of many queries on the CUDA cores (any type and layout).
#pragma once

#include "stream_attn.cuh"

namespace mbr {
namespace streamops {

void attend_simt(const AttnArgs& a, int dtype, cudaStream_t st);

}  // namespace streamops
}  // namespace mbr
