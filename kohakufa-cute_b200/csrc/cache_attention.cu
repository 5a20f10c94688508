// Attention of a few query rows to the 4-bit key/value cache (format: quantized_cache.cuh), with the sliding window
// and sinks of window.cuh where the call has them.
//
// One CTA owns one query row.  Per block of 128 keys a thread forms one score (its key's codes, dequantised in FP32),
// the block joins maximum and sum, and then each thread owns channels and adds the block's values up.
#include "kfa_common.cuh"
#include "launchers.h"
#include "quantized_cache.cuh"
#include "window.cuh"

namespace kfa {
namespace {

constexpr int kKeys = 128;

template <typename T>
__global__ void __launch_bounds__(kKeys) cache_attention(CacheAttentionCall p) {
    __shared__ float q[512], w[kKeys], part[4];
    const int64_t row_id = blockIdx.x;
    int r, h, b;
    split_row(row_id, p.Sq, p.Hq, r, h, b);
    const int kvh = h / p.group;
    const T* qrow = reinterpret_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + r * p.qs[2];
    for (int d = threadIdx.x; d < p.D; d += kKeys) q[d] = to_float<T>(qrow[d]);
    __syncthreads();
    const int64_t start = p.starts ? (int64_t)p.starts[b] : p.start;
    const WindowSpan span = window_span(start, r, p.window, p.Sk);
    const float sign = p.scale < 0.f ? -1.f : 1.f, c2 = fabsf(p.scale) * kLog2e;
    const CacheView &kc = p.half[0], &vc = p.half[1];
    float m = -INFINITY, l = 0.f, acc[4] = {};
    const int warp = threadIdx.x >> 5;
    for (int k0 = 0; k0 < span.hi; k0 += kKeys) {
        if (k0 >= p.sinks && k0 + kKeys <= span.lo) continue;
        const int key = k0 + threadIdx.x;
        float s = -INFINITY;
        if (window_sees(span, p.sinks, key)) {
            const uint32_t* codes = reinterpret_cast<const uint32_t*>(kc.codes + b * kc.cs[0] + kvh * kc.cs[1] + key * kc.cs[2]);
            const T* params = reinterpret_cast<const T*>(kc.params + b * kc.ps[0] + kvh * kc.ps[1] + key * kc.ps[2]);
            s = 0.f;
            for (int g = 0; g < p.D / kCacheGroup; ++g) {
                const float scale = to_float<T>(params[2 * g]), zero = to_float<T>(params[2 * g + 1]);
                for (int i = 0; i < kCacheGroup / 8; ++i) {
                    const uint32_t word = codes[g * (kCacheGroup / 8) + i];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        s = fmaf(q[g * kCacheGroup + i * 8 + e], fmaf(scale, (float)((word >> (4 * e)) & 15u), zero), s);
                }
            }
            s *= sign;
        }
        float mx = warp_max(s);
        if ((threadIdx.x & 31) == 0) part[warp] = mx;
        __syncthreads();
        const float m_new = fmaxf(m, fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
        const float alpha = m == -INFINITY ? 0.f : fast_ex2((m - m_new) * c2);
        const float pr = s == -INFINITY ? 0.f : fast_ex2((s - m_new) * c2);
        w[threadIdx.x] = pr;
        __syncthreads();
        m = m_new;
        float sum = 0.f;
        for (int j = 0; j < kKeys; ++j) sum += w[j];
        l = l * alpha + sum;
        for (int x = 0; x < 4; ++x) {
            const int d = threadIdx.x + x * kKeys;
            if (d >= p.D) break;
            float a = acc[x] * alpha;
            for (int j = 0; j < kKeys; ++j) {
                if (w[j] == 0.f) continue;
                const int64_t at = k0 + j;
                const uint8_t byte = vc.codes[b * vc.cs[0] + kvh * vc.cs[1] + at * vc.cs[2] + d / 2];
                const T* params = reinterpret_cast<const T*>(vc.params + b * vc.ps[0] + kvh * vc.ps[1] + at * vc.ps[2]) +
                                  d / kCacheGroup * 2;
                const float code = (float)((d & 1) ? byte >> 4 : byte & 15);
                a = fmaf(w[j], fmaf(to_float<T>(params[0]), code, to_float<T>(params[1])), a);
            }
            acc[x] = a;
        }
        __syncthreads();
    }
    T* out = reinterpret_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + r * p.os[2];
    for (int x = 0; x < 4; ++x) {
        const int d = threadIdx.x + x * kKeys;
        if (d < p.D) out[d] = from_float<T>(l > 0.f ? acc[x] / l : 0.f);
    }
}

}  // namespace

size_t cache_attention_workspace_bytes(const CacheAttentionCall& p) {
    (void)p;
    return 0;
}

cudaError_t launch_cache_attention(const CacheAttentionCall& p, bool bf16, void* workspace, cudaStream_t st) {
    (void)workspace;
    const unsigned grid = (unsigned)((int64_t)p.B * p.Hq * p.Sq);
    if (bf16) cache_attention<__nv_bfloat16><<<grid, kKeys, 0, st>>>(p);
    else cache_attention<__half><<<grid, kKeys, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace kfa
