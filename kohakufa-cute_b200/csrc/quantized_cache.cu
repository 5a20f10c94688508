// Writing and reading the 4-bit key/value cache (format: quantized_cache.cuh).
//
// Both are one pass over the data: eight threads own a group of 64 channels of one token, eight channels each, so a
// thread loads (or stores) 16 bytes of the 16-bit row and stores (or loads) one word of eight codes; the group's
// minimum and maximum are joined over the eight lanes by three shuffles each.  The bound is HBM: 128 bytes of 16-bit
// values against 36 of the cache per group.  Keys and values go in one launch.
#include "kfa_common.cuh"
#include "launchers.h"
#include "quantized_cache.cuh"

#include <type_traits>

namespace kfa {
namespace {

constexpr int kThreads = 256;

// The place of thread `id` of a call: half, batch, head, row and the first of its eight channels.
struct Place {
    int which, b, h, r, d;
};
__device__ __forceinline__ bool place_of(const CacheCall& p, int64_t id, Place& t) {
    const int pieces = p.D / 8;
    const int64_t rows = (int64_t)p.B * p.H * p.n;
    int64_t row = id / pieces;
    t.d = (int)(id - row * pieces) * 8;
    if (row >= 2 * rows) return false;
    t.which = row >= rows ? 1 : 0;
    split_row(row - t.which * rows, p.n, p.H, t.r, t.h, t.b);
    return true;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) cache_write(CacheCall p) {
    Place t;
    const bool live = place_of(p, (int64_t)blockIdx.x * kThreads + threadIdx.x, t);
    int64_t at = -1;
    if (live) {
        const int length = p.lengths ? min(p.lengths[t.b], p.n) : p.n;
        if (t.r < length) at = (p.starts ? (int64_t)p.starts[t.b] : p.start) + t.r;
    }
    const bool kept = at >= 0 && at < p.capacity;  // (the eight lanes of a group agree)
    float x[8] = {};
    if (kept) {
        const T* row = reinterpret_cast<const T*>(p.in[t.which]) + t.b * p.rs[t.which][0] + t.h * p.rs[t.which][1] +
                       t.r * p.rs[t.which][2] + t.d;
        const uint4 raw = *reinterpret_cast<const uint4*>(row);
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
    }
    // fminf / fmaxf skip NaN: the sum of |x| * 0 carries it (and infinities) to the scale
    float low = x[0], high = x[0], bad = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        low = fminf(low, x[i]);
        high = fmaxf(high, x[i]);
        bad = fmaf(x[i], 0.f, bad);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        bad += __shfl_xor_sync(0xffffffffu, bad, o);
    }
    const T scale16 = from_float<T>(__fdiv_rn(high - low, 15.f) + bad);
    const float scale = to_float<T>(scale16);
    if (!kept) return;
    uint32_t word = 0;
    if (scale > 0.f && scale < INFINITY) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float code = fminf(rintf(__fdiv_rn(x[i] - low, scale)), 15.f);
            word |= static_cast<uint32_t>(code) << (4 * i);
        }
    }
    const CacheView& c = p.half[t.which];
    *reinterpret_cast<uint32_t*>(c.codes + t.b * c.cs[0] + t.h * c.cs[1] + at * c.cs[2] + t.d / 2) = word;
    if (t.d % kCacheGroup == 0) {
        T pair[2] = {scale < INFINITY ? scale16 : from_float<T>(NAN), from_float<T>(low)};
        *reinterpret_cast<uint32_t*>(c.params + t.b * c.ps[0] + t.h * c.ps[1] + at * c.ps[2] + t.d / kCacheGroup * 2) =
            *reinterpret_cast<const uint32_t*>(pair);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) cache_read(CacheCall p) {
    Place t;
    if (!place_of(p, (int64_t)blockIdx.x * kThreads + threadIdx.x, t)) return;
    const int64_t at = (p.starts ? (int64_t)p.starts[t.b] : p.start) + t.r;
    T v[8];
    if (at >= 0 && at < p.capacity) {
        const CacheView& c = p.half[t.which];
        const uint32_t word =
            *reinterpret_cast<const uint32_t*>(c.codes + t.b * c.cs[0] + t.h * c.cs[1] + at * c.cs[2] + t.d / 2);
        const uint32_t pair = *reinterpret_cast<const uint32_t*>(c.params + t.b * c.ps[0] + t.h * c.ps[1] +
                                                                at * c.ps[2] + t.d / kCacheGroup * 2);
        const T* e = reinterpret_cast<const T*>(&pair);
        const float scale = to_float<T>(e[0]), zero = to_float<T>(e[1]);
        // the rounded scale may carry the top of a group past the type's largest value: it saturates (a NaN does not)
        constexpr float kMost = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = fmaf(scale, (float)((word >> (4 * i)) & 15u), zero);
            v[i] = from_float<T>(x > kMost ? kMost : x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = from_float<T>(0.f);
    }
    T* row = reinterpret_cast<T*>(p.out[t.which]) + t.b * p.rs[t.which][0] + t.h * p.rs[t.which][1] +
             t.r * p.rs[t.which][2] + t.d;
    *reinterpret_cast<uint4*>(row) = *reinterpret_cast<const uint4*>(v);
}

}  // namespace

cudaError_t launch_cache_write(const CacheCall& p, bool bf16, cudaStream_t st) {
    const int64_t threads = 2 * (int64_t)p.B * p.H * p.n * (p.D / 8);
    const unsigned grid = (unsigned)((threads + kThreads - 1) / kThreads);
    if (bf16) cache_write<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
    else cache_write<__half><<<grid, kThreads, 0, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_cache_read(const CacheCall& p, bool bf16, cudaStream_t st) {
    const int64_t threads = 2 * (int64_t)p.B * p.H * p.n * (p.D / 8);
    const unsigned grid = (unsigned)((threads + kThreads - 1) / kThreads);
    if (bf16) cache_read<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
    else cache_read<__half><<<grid, kThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace kfa
