// Writing and reading the 4-bit key/value cache (format: quantized_cache.cuh).
//
// Both are one pass over the data: eight threads own a group of 64 channels of one token, eight channels each, so a
// thread loads (or stores) 16 bytes of the 16-bit row and stores (or loads) one word of eight codes; the group's
// minimum and maximum are joined over the eight lanes by three shuffles each.  The bound is HBM: 128 bytes of 16-bit
// values against 36 of the cache per group.  Keys and values go in one launch.  A CTA owns a piece of one (batch, head)
// plane, and a thread kRows of its rows, whose loads are in flight together.
#include "kfa_common.cuh"
#include "launchers.h"
#include "quantized_cache.cuh"
#include "sm100_ptx.cuh"

#include <type_traits>

namespace kfa {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 4;  // rows per thread

// The CTA's plane and the thread's first row and channel; the thread's rows are `step` apart.
struct Place {
    int which, b, h, r, step, d;
    bool live;
};
__device__ __forceinline__ Place place_of(const CacheCall& p) {
    const uint32_t pieces = p.D / 8, step = kThreads / pieces, per_cta = step * kRows;
    const uint32_t tiles = ((uint32_t)p.n + per_cta - 1) / per_cta, plane = blockIdx.x / tiles;
    Place t;
    t.h = (int)(plane % (uint32_t)p.H);
    const uint32_t rest = plane / (uint32_t)p.H;
    t.b = (int)(rest % (uint32_t)p.B);
    t.which = (int)(rest / (uint32_t)p.B);
    const uint32_t sub = threadIdx.x / pieces;
    t.d = (int)(threadIdx.x - sub * pieces) * 8;
    t.step = (int)step;
    t.r = (int)((blockIdx.x - plane * tiles) * per_cta + sub);
    t.live = sub < step;  // (a row of 3, 5, 6 or 7 groups does not divide the CTA's threads)
    return t;
}

// Pairs of 16-bit floats: a * b + c rounded once, the smaller and the larger of two (a NaN stays one).
template <bool BF16>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) cache_write(CacheCall p) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    const Place t = place_of(p);
    const int length = p.lengths ? min(p.lengths[t.b], p.n) : p.n;
    const int64_t start = p.starts ? (int64_t)p.starts[t.b] : p.start;
    const T* rows = reinterpret_cast<const T*>(p.in[t.which]) + t.b * p.rs[t.which][0] + t.h * p.rs[t.which][1] + t.d;
    const CacheView& c = p.half[t.which];
    uint8_t* codes = c.codes + t.b * c.cs[0] + t.h * c.cs[1] + t.d / 2;
    uint16_t* params = c.params + t.b * c.ps[0] + t.h * c.ps[1] + t.d / kCacheGroup * 2;
    uint4 raw[kRows];
    bool kept[kRows];  // (the eight lanes of a group agree)
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        const int r = t.r + j * t.step;
        kept[j] = t.live && r < length && start + r >= 0 && start + r < p.capacity;
        raw[j] = kept[j] ? *reinterpret_cast<const uint4*>(rows + r * p.rs[t.which][2]) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        float x[8];
        const float2 e0 = unpack2<BF16>(raw[j].x), e1 = unpack2<BF16>(raw[j].y), e2 = unpack2<BF16>(raw[j].z),
                     e3 = unpack2<BF16>(raw[j].w);
        x[0] = e0.x, x[1] = e0.y, x[2] = e1.x, x[3] = e1.y, x[4] = e2.x, x[5] = e2.y, x[6] = e3.x, x[7] = e3.y;
        // minimum and maximum of packed pairs, which keep a NaN; an infinity makes the difference infinite or NaN
        uint32_t least = min2<BF16>(min2<BF16>(raw[j].x, raw[j].y), min2<BF16>(raw[j].z, raw[j].w));
        uint32_t most = max2<BF16>(max2<BF16>(raw[j].x, raw[j].y), max2<BF16>(raw[j].z, raw[j].w));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            least = min2<BF16>(least, __shfl_xor_sync(0xffffffffu, least, o));
            most = max2<BF16>(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        least = min2<BF16>(least, __byte_perm(least, 0, 0x1032));
        most = max2<BF16>(most, __byte_perm(most, 0, 0x1032));
        const float low = unpack2<BF16>(least).x, high = unpack2<BF16>(most).x;
        const T scale16 = from_float<T>(__fdiv_rn(high - low, 15.f));
        const float scale = to_float<T>(scale16);
        uint32_t word = 0;
        if (scale > 0x1p-90f && scale < 0x1p90f) {
            // (x - low) / scale correctly rounded from one reciprocal: a quotient, its exact remainder, one correction
            // (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990; the
            // 16-bit scale has no mantissa of ones, and nothing over- or underflows in this range).  The sum with
            // 1.5 * 2^23 rounds it to an integer, half to even, into the low bits.
            const float inverse = __frcp_rn(scale);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = x[i] - low, q = a * inverse;
                const float code = fminf(fmaf(fmaf(-q, scale, a), inverse, q), 15.f);
                word |= (__float_as_uint(code + 12582912.f) & 15u) << (4 * i);
            }
        } else if (scale > 0.f && scale < INFINITY) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                word |= static_cast<uint32_t>(fminf(rintf(__fdiv_rn(x[i] - low, scale)), 15.f)) << (4 * i);
        }
        if (!kept[j]) continue;
        const int64_t at = start + t.r + j * t.step;
        *reinterpret_cast<uint32_t*>(codes + at * c.cs[2]) = word;
        if (t.d % kCacheGroup == 0) {
            T pair[2] = {scale < INFINITY ? scale16 : from_float<T>(NAN), from_float<T>(low)};
            *reinterpret_cast<uint32_t*>(params + at * c.ps[2]) = *reinterpret_cast<const uint32_t*>(pair);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) cache_read(CacheCall p) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    const Place t = place_of(p);
    if (!t.live) return;
    const int64_t start = p.starts ? (int64_t)p.starts[t.b] : p.start;
    T* rows = reinterpret_cast<T*>(p.out[t.which]) + t.b * p.rs[t.which][0] + t.h * p.rs[t.which][1] + t.d;
    const CacheView& c = p.half[t.which];
    const uint8_t* codes = c.codes + t.b * c.cs[0] + t.h * c.cs[1] + t.d / 2;
    const uint16_t* params = c.params + t.b * c.ps[0] + t.h * c.ps[1] + t.d / kCacheGroup * 2;
    uint32_t word[kRows], pair[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        const int64_t at = start + t.r + j * t.step;
        const bool inside = t.r + j * t.step < p.n && at >= 0 && at < p.capacity;
        word[j] = inside ? *reinterpret_cast<const uint32_t*>(codes + at * c.cs[2]) : 0u;
        pair[j] = inside ? *reinterpret_cast<const uint32_t*>(params + at * c.ps[2]) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        const int r = t.r + j * t.step;
        if (r >= p.n) break;
        const uint32_t scale = __byte_perm(pair[j], 0, 0x1010), zero = __byte_perm(pair[j], 0, 0x3232);
        // Codes n and n + 4 as a pair of floats: masked into the mantissa of 16.0, less 16.  The value saturates (the
        // rounded scale may carry the top of a group past the type's largest value).
        constexpr uint32_t mask = BF16 ? 0x00780078u : 0x03c003c0u, sixteen = BF16 ? 0x41804180u : 0x4c004c00u;
        constexpr uint32_t less = BF16 ? 0xc180c180u : 0xcc00cc00u, one = BF16 ? 0x3f803f80u : 0x3c003c00u;
        const uint32_t w = word[j];
        uint32_t v[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int to = (BF16 ? 3 : 6) - 4 * n;
            const uint32_t x = ((to >= 0 ? w << (to >= 0 ? to : 0) : w >> (to < 0 ? -to : 0)) & mask) | sixteen;
            v[n] = min2<BF16>(fma2<BF16>(fma2<BF16>(x, one, less), scale, zero), BF16 ? 0x7f7f7f7fu : 0x7bff7bffu);
        }
        *reinterpret_cast<uint4*>(rows + r * p.rs[t.which][2]) =
            make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                       __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632));
    }
}

unsigned grid_of(const CacheCall& p) {
    const int64_t per_cta = kThreads / (p.D / 8) * kRows, tiles = (p.n + per_cta - 1) / per_cta;
    return (unsigned)(2 * (int64_t)p.B * p.H * tiles);
}

}  // namespace

cudaError_t launch_cache_write(const CacheCall& p, bool bf16, cudaStream_t st) {
    const unsigned grid = grid_of(p);
    if (bf16) cache_write<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
    else cache_write<__half><<<grid, kThreads, 0, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_cache_read(const CacheCall& p, bool bf16, cudaStream_t st) {
    const unsigned grid = grid_of(p);
    if (bf16) cache_read<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
    else cache_read<__half><<<grid, kThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace kfa
