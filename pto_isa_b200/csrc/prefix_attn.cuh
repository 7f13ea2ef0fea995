// Declarations shared by the two kernels of the attention over a shared prefix.
#pragma once
#include "internal.h"
#include "mx_format.cuh"

namespace pto_b200 {

struct AttnArgs {
    const uint8_t *k, *v, *ks, *vs;
    const uint16_t *q;
    int64_t q_batch, q_token, q_head; // strides in elements
    const int32_t *prefix_pages;
    const int32_t *table;
    const int32_t *lens;
    int64_t table_stride;
    int64_t num_pages;
    float *part_o;   // [slot][16][d]
    float2 *part_ml; // [slot][16]: m (log2 units), l
    uint16_t *o;
    float *lse;
    float scale_log2;
    int page_shift;
    int batch, tokens, heads, kv_heads, group;
    int prefix_len, own_max;
    // prefix_splits pieces of prefix_chunk keys, each for prefix_tiles tiles of 16 rows; in the wide kernel a block makes
    // prefix_pieces / prefix_splits pieces of its chunk
    int prefix_tiles, prefix_splits, prefix_pieces, prefix_chunk, prefix_wide;
    int own_tiles, own_splits, own_min;
};

constexpr int kPieceRows = 16; // rows of a slot of partial results

// The kernels of one call overlap: a kernel lets the next one start as soon as its own blocks are all running, and the next
// one waits before it touches what the earlier ones write.  Only kernels of the same call are launched that way: the
// first one starts when everything before it on the stream is complete.
__device__ __forceinline__ void programmatic_trigger()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void programmatic_wait()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... Params, typename... Args>
int launch_overlapped(void (*kernel)(Params...), unsigned blocks, int threads, int smem, cudaStream_t stream, bool after_own, Args... args)
{
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.dynamicSmemBytes = static_cast<size_t>(smem);
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = after_own ? 1 : 0;
    return check_cuda(cudaLaunchKernelEx(&config, kernel, args...), "kernel launch");
}

// keys by the tensor memory of one block per SM: 128-row tiles of the prefix's rows against 128 keys at a time
int launch_prefix_wide(const AttnArgs &a, int fmt, int d, bool bf16, DeviceStatus *status, cudaStream_t stream);

} // namespace pto_b200
