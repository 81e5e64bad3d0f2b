// stream_error.cu — the error words that the streaming attention kernels' bounded
// waits set, one for each stream: host memory that the device writes, so the
// host sees it without a copy.
#include <map>
#include <mutex>
#include <string>
#include <utility>

#include "common.h"
#include "sm100.cuh"
#include "stream_ops.h"

namespace mbr {
namespace streamops {

namespace {

// Words are dealt from blocks that are never freed: a kernel or a graph may hold
// a word's address for as long as the process runs.  A handle that the runtime
// gives out again after its stream was destroyed gets the same word.
struct Words {
    static constexpr int kBlock = 1024;
    std::mutex mu;
    std::map<std::pair<int, cudaStream_t>, int*> of;
    int* block = nullptr;
    int used = kBlock;
};
Words& words() {
    static Words* const w = new Words;  // outlives every static destructor
    return *w;
}

// The word of a stream, or null if it has none and `make` is false.  A handle says which stream it is on any
// device, but for the names of each device's default streams.
int* word_of(cudaStream_t st, bool make) {
    if (st == cudaStreamLegacy) st = nullptr;  // two names of one stream
    const int dev = st == nullptr || st == cudaStreamPerThread ? stream_device() : -1;
    Words& w = words();
    const std::lock_guard<std::mutex> lock(w.mu);
    const auto at = w.of.find({dev, st});
    if (at != w.of.end()) return at->second;
    if (!make) return nullptr;
    if (w.used == Words::kBlock) {  // visible to every device
        int* p = nullptr;
        MBR_CUDA(cudaHostAlloc((void**)&p, Words::kBlock * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable));
        for (int i = 0; i < Words::kBlock; ++i) p[i] = sm100::KERR_NONE;
        w.block = p, w.used = 0;
    }
    return w.of[{dev, st}] = w.block + w.used++;  // unified addressing: the device uses the same address
}

}  // namespace

int* stream_error_word(cudaStream_t st) { return word_of(st, true); }

void raise_stream_error(cudaStream_t st) {
    int* const w = word_of(st, false);
    if (!w) return;
    const int e = __atomic_exchange_n(w, sm100::KERR_NONE, __ATOMIC_ACQ_REL);
    if (e == sm100::KERR_NONE) return;
    if (e == sm100::KERR_SMEM_ALIGN)
        throw Error(ERR_CUDA, "an earlier streaming attention kernel of this stream found its shared memory misaligned");
    throw Error(ERR_TIMEOUT, "a kernel-side wait of an earlier streaming attention call on this stream ran out (error " +
                                 std::to_string(e) + "): what it and the calls behind it wrote is void");
}

void stream_check(cudaStream_t st) {
    MBR_CUDA(cudaStreamSynchronize(st));
    raise_stream_error(st);
}

}  // namespace streamops
}  // namespace mbr
