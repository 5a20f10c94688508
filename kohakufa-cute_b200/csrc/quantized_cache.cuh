// Format of the 4-bit key/value cache, shared by the kernels that write it, read it back and attend to it.
//
// Each token's row of D channels is held in groups of 64 channels.  A group has a scale and a zero in the model's
// 16-bit type and 64 codes of 4 bits; byte i of a row holds channels 2i (low half) and 2i + 1 (high half):
//     low = min x, scale = round16((max x - low) / 15), zero = low, code = round_half_even((x - low) / scale), 0..15
//     value = zero + scale * code          (read back in 16 bits it saturates at the type's largest value; attention
//                                           takes it as it is, in FP32)
// 36 bytes per group instead of 128.  A group whose values are all equal (or whose scale underflows to zero) has
// codes 0 and is read back as `low`; a group with a value that is not finite, or whose max - low is beyond FP32 (BF16 only),
// has a NaN scale and reads back as NaN.
#pragma once
#include "kfa_common.cuh"

namespace kfa {

constexpr int kCacheGroup = 64;

struct CacheView {  // one of the two halves (keys or values) of a cache
    uint8_t* codes;   // [B, H, capacity, D / 2] bytes
    uint16_t* params; // [B, H, capacity, D / 64, 2]: (scale, zero)
    int64_t cs[3];    // strides of codes: batch, head, token (bytes)
    int64_t ps[3];    // strides of params: batch, head, token (16-bit elements)
};

struct CacheCall {
    CacheView half[2];       // keys, values
    const void* in[2];       // write: new rows [B, H, n, D]
    void* out[2];            // read: rows [B, H, n, D]
    int64_t rs[2][3];        // strides of those rows: batch, head, token (elements)
    const int32_t* starts;   // position of row 0 per batch, or null: `start`
    const int32_t* lengths;  // write: rows per batch, or null: all n
    int64_t start;
    int B, H, n, D, capacity;
};

struct CacheAttentionCall {
    CacheView half[2];      // keys, values
    const void* q;          // [B, Hq, Sq, D]
    void* out;              // like q
    int64_t qs[3], os[3];   // batch, head, row (elements); unit channel stride
    const int32_t* starts;  // position of query row 0 per batch, or null: `start`
    int64_t start, window;  // window: longer than every position when the call has none
    int sinks;
    int B, Hq, Hkv, Sq, Sk, D, group;  // Sk = rows of the cache
    float scale;
    int* status;      // as in AttnParams
    int* abort_flag;
};

}  // namespace kfa
