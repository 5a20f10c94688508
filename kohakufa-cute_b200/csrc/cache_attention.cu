// Attention of a few query rows to the 4-bit key/value cache: decode_rows.cuh on quantized_cache.cuh's format.
#include "decode_rows.cuh"
#include "launchers.h"

namespace kfa {

bool cache_attention_countable(const CacheAttentionCall& c) {
    return c.D == 128 ? rows::countable<128, true>(c) : rows::countable<64, true>(c);
}

size_t cache_attention_workspace_bytes(const CacheAttentionCall& c) {
    return c.D == 128 ? rows::workspace_bytes<128, true>(c) : rows::workspace_bytes<64, true>(c);
}

cudaError_t launch_cache_attention(const CacheAttentionCall& c, bool bf16, void* workspace, int* launches, cudaStream_t st) {
    RowsCall p = {};
    p.c = c;
    const cudaError_t e =
        bf16 ? rows::dispatch<__nv_bfloat16, true>(p, workspace, st) : rows::dispatch<__half, true>(p, workspace, st);
    *launches = p.cluster ? 1 : 2;
    return e;
}

}  // namespace kfa
