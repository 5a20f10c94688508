// Writing and reading the 4-bit key/value cache (format: quantized_cache.cuh).
//
// Both are one pass over the data: a thread owns kSpan channels of a group of 64 of one token (sixteen when it writes,
// eight when it reads).  A writer joins the group's minimum and maximum over four lanes by two shuffles each; what a
// group costs, and not its bytes, bounds the writer, so that more channels per thread pay.  The other bound is HBM: 128
// bytes of 16-bit values against 36 of the cache per group.  Keys and values go in one launch.  A CTA owns a piece of
// one (batch, head) plane, and a thread kRows of its rows, whose loads are in flight together.
#include "kfa_common.cuh"
#include "launchers.h"
#include "quantized_cache.cuh"
#include "sm100_ptx.cuh"

#include <type_traits>

namespace kfa {
namespace {

constexpr int kThreads = 256;
constexpr int kWriteSpan = 16, kReadSpan = 8;  // channels per thread

// Rows per thread: four loads of 16 bytes in flight.
template <int SPAN>
__host__ __device__ constexpr int rows_of() { return 32 / SPAN; }

// The CTA's plane and the thread's first row and channel; the thread's rows are `step` apart.
struct Place {
    int which, b, h, r, step, d;
    bool live;
};
template <int SPAN>
__device__ __forceinline__ Place place_of(const CacheCall& p) {
    const uint32_t pieces = p.D / SPAN, step = kThreads / pieces, per_cta = step * rows_of<SPAN>();
    const uint32_t tiles = ((uint32_t)p.n + per_cta - 1) / per_cta, plane = blockIdx.x / tiles;
    Place t;
    t.h = (int)(plane % (uint32_t)p.H);
    const uint32_t rest = plane / (uint32_t)p.H;
    t.b = (int)(rest % (uint32_t)p.B);
    t.which = (int)(rest / (uint32_t)p.B);
    const uint32_t sub = threadIdx.x / pieces;
    t.d = (int)(threadIdx.x - sub * pieces) * SPAN;
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
    constexpr int kRows = rows_of<kWriteSpan>();
    const Place t = place_of<kWriteSpan>(p);
    const int length = p.lengths ? min(p.lengths[t.b], p.n) : p.n;
    const int64_t start = p.starts ? (int64_t)p.starts[t.b] : p.start;
    const T* rows = reinterpret_cast<const T*>(p.in[t.which]) + t.b * p.rs[t.which][0] + t.h * p.rs[t.which][1] + t.d;
    const CacheView& c = p.half[t.which];
    uint8_t* codes = c.codes + t.b * c.cs[0] + t.h * c.cs[1] + t.d / 2;
    uint16_t* params = c.params + t.b * c.ps[0] + t.h * c.ps[1] + t.d / kCacheGroup * 2;
    uint32_t raw[kRows][kWriteSpan / 2];
    bool kept[kRows];  // (the four lanes of a group agree)
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        const int r = t.r + j * t.step;
        kept[j] = t.live && r < length && start + r >= 0 && start + r < p.capacity;
#pragma unroll
        for (int x = 0; x < kWriteSpan / 8; ++x) {
            const uint4 v = kept[j] ? *reinterpret_cast<const uint4*>(rows + r * p.rs[t.which][2] + 8 * x) : make_uint4(0, 0, 0, 0);
            raw[j][4 * x] = v.x, raw[j][4 * x + 1] = v.y, raw[j][4 * x + 2] = v.z, raw[j][4 * x + 3] = v.w;
        }
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        if (!__any_sync(0xffffffffu, kept[j])) continue;
        // minimum and maximum of packed pairs, which keep a NaN; an infinity makes the difference infinite or NaN
        uint32_t least = raw[j][0], most = raw[j][0];
#pragma unroll
        for (int x = 1; x < kWriteSpan / 2; ++x) {
            least = min2<BF16>(least, raw[j][x]);
            most = max2<BF16>(most, raw[j][x]);
        }
#pragma unroll
        for (int o = 1; o < kCacheGroup / kWriteSpan; o <<= 1) {
            least = min2<BF16>(least, __shfl_xor_sync(0xffffffffu, least, o));
            most = max2<BF16>(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        least = min2<BF16>(least, __byte_perm(least, 0, 0x1032));
        most = max2<BF16>(most, __byte_perm(most, 0, 0x1032));
        const float low = unpack2<BF16>(least).x, range = unpack2<BF16>(most).x - low;
        // Quotients correctly rounded from a reciprocal: a quotient, its exact remainder, one correction (Markstein,
        // "Computation of elementary functions on the IBM RISC System/6000 processor", 1990; neither 15 nor a 16-bit
        // scale has a mantissa of ones).  It needs a range in which nothing over- or underflows: the smallest and the
        // largest groups are divided as they are.
        float scale;
        uint32_t word[kWriteSpan / 8] = {};
        T scale16;
        constexpr float kLeast = BF16 ? 0x1p-80f : 0x1p-10f;  // (FP16: the scale is a normal number)
        if (range > kLeast && range < 0x1p80f) {
            constexpr float kFifteenth = 1.f / 15.f;
            const float q = range * kFifteenth;
            scale16 = from_float<T>(fmaf(fmaf(-15.f, q, range), kFifteenth, q));
            scale = to_float<T>(scale16);
            const float inverse = __frcp_rn(scale);
            // The sum with 1.5 * 2^23 rounds a quotient to an integer, half to even, in its low bits; what the other bits
            // of the eight sums add up to, shifted by their codes' places, is taken off again.
            constexpr uint32_t kBits = 0x4b400000u, kAll = kBits * 0x11111111u;
#pragma unroll
            for (int x = 0; x < kWriteSpan / 2; ++x) {
                const float2 v = unpack2<BF16>(raw[j][x]);
                const float a = v.x - low, b = v.y - low, qa = a * inverse, qb = b * inverse;
                const float ca = fmaf(fmaf(-qa, scale, a), inverse, qa) + 12582912.f;
                const float cb = fmaf(fmaf(-qb, scale, b), inverse, qb) + 12582912.f;
                word[x / 4] += (__float_as_uint(ca) << (8 * (x % 4))) + (__float_as_uint(cb) << (8 * (x % 4) + 4));
            }
#pragma unroll
            for (int x = 0; x < kWriteSpan / 8; ++x) word[x] -= kAll;
        } else {
            scale16 = from_float<T>(__fdiv_rn(range, 15.f));
            scale = to_float<T>(scale16);
            if (scale > 0.f && scale < INFINITY) {
#pragma unroll
                for (int x = 0; x < kWriteSpan / 2; ++x) {
                    const float2 v = unpack2<BF16>(raw[j][x]);
                    const float ca = fminf(rintf(__fdiv_rn(v.x - low, scale)), 15.f);
                    const float cb = fminf(rintf(__fdiv_rn(v.y - low, scale)), 15.f);
                    word[x / 4] |= (static_cast<uint32_t>(ca) | static_cast<uint32_t>(cb) << 4) << (8 * (x % 4));
                }
            }
        }
        if (!kept[j]) continue;
        const int64_t at = start + t.r + j * t.step;
        *reinterpret_cast<uint2*>(codes + at * c.cs[2]) = make_uint2(word[0], word[1]);
        if (t.d % kCacheGroup == 0) {
            T pair[2] = {scale < INFINITY ? scale16 : from_float<T>(NAN), from_float<T>(low)};
            *reinterpret_cast<uint32_t*>(params + at * c.ps[2]) = *reinterpret_cast<const uint32_t*>(pair);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) cache_read(CacheCall p) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr int kRows = rows_of<kReadSpan>();
    const Place t = place_of<kReadSpan>(p);
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

template <int SPAN>
unsigned grid_of(const CacheCall& p) {
    const int64_t per_cta = kThreads / (p.D / SPAN) * rows_of<SPAN>(), tiles = (p.n + per_cta - 1) / per_cta;
    return (unsigned)(2 * (int64_t)p.B * p.H * tiles);
}

}  // namespace

cudaError_t launch_cache_write(const CacheCall& p, bool bf16, cudaStream_t st) {
    const unsigned grid = grid_of<kWriteSpan>(p);
    if (bf16) cache_write<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
    else cache_write<__half><<<grid, kThreads, 0, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_cache_read(const CacheCall& p, bool bf16, cudaStream_t st) {
    const unsigned grid = grid_of<kReadSpan>(p);
    if (bf16) cache_read<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
    else cache_read<__half><<<grid, kThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace kfa
