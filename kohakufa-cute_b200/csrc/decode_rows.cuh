// Attention of a few query rows per K/V head to a long key/value cache, held in 16 bits or in 4 (quantized_cache.cuh),
// with positions per sequence and the sliding window and sinks of window.cuh.
//
// Such a call is bound by the HBM time of the keys and values that some row sees.  To keep the arithmetic below that,
// the two products run on the tensor cores' register path (mma m16n8k16), where a fragment of eight query rows costs
// nothing extra and the cache goes from shared memory to registers once:
//   S^T = K q^T     A = 16 tokens x 16 channels, B = 16 channels x 8 query rows
//   O^T = V^T P^T   A = 16 channels x 16 tokens, B = 16 tokens x 8 query rows (P^T by two 8x8 register transposes)
// The probabilities enter the second product in 16 bits, as they do in the other forward kernels (one rounding each, relative
// to the row's reference; their sum is of the unrounded ones); everything between is FP32.
// (tcgen05 wants 128 rows of operand A in shared memory: the 4-bit cache would have to be widened into it, 4 x the
// bytes, and its rows are tokens only in one of the two products.)
//
// 4-bit caches are never widened to values.  Codes become 16-bit floats in two instructions per pair (shift, and one
// logic operation that masks the code into the mantissa of a base, 16 to 1024), and scale and zero of a token's group of
// 64 channels are applied to sums, in FP32:
//   s    = sum_g  scale_g * (sum_d q_d (base_d + code_d) - sum_d q_d base_d)  +  zero_g * (sum_d q_d)
//   o_d  = sum_t  round16(p_t scale_g) * (code_d - 8)  +  sum_t p_t (zero_g + 8 scale_g)
// The codes less 8 are centred, so the one rounding, of p * scale, weighs like the rounding of p against 16-bit values.
// (In FP16 a product p * scale below 2^-14 is rounded in steps of 2^-24; values that small lead to outputs which FP16
// holds in steps of that size themselves.)
//
// Work is cut evenly however ragged the batch is: the blocks of tokens that the units (sequence, K/V head, chunk of
// query rows) have to read are numbered through, and each CTA takes an equal piece of that line; where a unit spans
// several CTAs their partial (maximum, sum, accumulator) are merged by a second, dependent launch.  The lengths come
// from device memory, so a captured call follows new positions.  Short calls (few units of few blocks) skip the second
// launch: a cluster of up to eight CTAs owns a unit and merges over distributed shared memory.  Within a CTA the warps
// take blocks in turn, each with its own ring of asynchronous copies.  (A piece per warp, without the merge within the
// CTA, was no faster: 114 against 113 us at 16 x 32768 tokens, 44 against 42 at 16 x 8192, and slower for one sequence.)
// More than 16 rows per K/V head widen the codes once per 16.  (Once per 32, into shared memory for four warps of eight
// rows each, was slower, 58 against 44 us at 32 rows: every warp then reads the whole tile from there.)
//
// Measured: 16-bit cache, 48 sequences with windows of 4096 tokens, 8 K/V heads of 128: 126 us, 6.4 TB/s, the HBM copy
// rate.  4-bit cache, 16 x 24 600 tokens on average: 113 us, 4.1 TB/s (64 %): issue slots 58 % and the integer pipe 57 %
// busy, about 730 instructions per 32 tokens and warp, of which 240 shift and mask codes and 64 centre them.  What it
// took: 154 us with a lane's own address per copy; 149 with contiguous copies; 134 with mask and base in one instruction;
// 113 with 64 tokens per block (more independent chains per warp; three CTAs of 168 registers instead of four of 128).
#pragma once
#include "kfa_common.cuh"
#include "quantized_cache.cuh"
#include "sm100_ptx.cuh"
#include "window.cuh"

#include <atomic>
#include <type_traits>

namespace kfa {

struct RowsCall {
    CacheAttentionCall c;
    const void* kv[2];    // 16-bit cache: keys, values
    int64_t kvs[2][3];    // batch, head, token strides (elements)
    int rows, chunks;     // query rows per K/V head, pieces of 8 * NT of them
    int ctas;
    int cluster;          // != 0: a thread-block cluster of that many CTAs serves a unit, and there is no second launch
    uint32_t lowest, others;  // see Bases
    float* part_o;        // [ctas][2][8 NT][D]: a CTA's first and last piece of a unit
    float* part_ml;       // [ctas][2][8 NT][2]: maximum, sum
};

namespace rows {

constexpr int kWarps = 4;
constexpr int kCluster = 8;  // CTAs of a cluster at most

// CTAs per SM that registers and shared memory allow (the launch bounds hold the compiler to it).
template <int D, bool Q4, int NT>
constexpr int resident() {
    return Q4 ? (D == 64 ? (NT == 1 ? 4 : 3) : (NT == 1 ? 3 : 2)) : (D == 64 ? 3 : 2);
}

template <int D, bool Q4, int NT>
struct Cfg {
    static constexpr int kGroups = D / kCacheGroup;
    static constexpr int kBlock = Q4 ? (NT == 1 ? 64 : 32) : 16;  // tokens per block
    static constexpr int kRow = Q4 ? D / 2 : D * 2;            // bytes of a token's codes or channels
    static constexpr int kParam = Q4 ? 4 * kGroups : 0;        // bytes of a token's scales and zeros
    static constexpr int kHalf = kBlock * (kRow + kParam);     // one block of keys or of values
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kStages = Q4 ? (D == 128 && NT == 1 ? 2 : 3) : (D == 64 ? 4 : 3);
    static constexpr int kRing = kWarps * kStages * kStage;
};

// ------------------------------------------------------------------ the line of blocks
struct Blocks {
    int sinks, first, count;  // blocks [0, sinks), then `count - sinks` blocks from `first` on
    __device__ __forceinline__ int block(int i) const { return i + (i < sinks ? 0 : first - sinks); }
};

__device__ __forceinline__ Blocks blocks_of(const CacheAttentionCall& c, int64_t start, int size) {
    const WindowSpan a = window_span(start, 0, c.window, c.Sk), z = window_span(start, c.Sq - 1, c.window, c.Sk);
    Blocks n;
    n.sinks = (min(c.sinks, z.hi) + size - 1) / size;
    n.first = max(a.lo / size, n.sinks);
    n.count = n.sinks + (a.lo < z.hi ? max((z.hi + size - 1) / size - n.first, 0) : 0);
    return n;
}

__device__ __forceinline__ int64_t start_of(const CacheAttentionCall& c, int b) {
    return c.starts ? (int64_t)c.starts[b] : c.start;
}

// The blocks of the sequences, a lane of the (converged) warp per sequence: those of a batch of up to 32 are formed once.
struct Line {
    const CacheAttentionCall& c;
    uint32_t units;
    int size, lane;
    uint32_t mine;  // blocks of sequence `lane` in all its units
    __device__ __forceinline__ uint32_t of(int b) const {
        return b < c.B ? blocks_of(c, start_of(c, b), size).count * units : 0u;
    }
    __device__ __forceinline__ Line(const CacheAttentionCall& call, uint32_t units_, int size_)
        : c(call), units(units_), size(size_), lane(threadIdx.x & 31), mine(of(threadIdx.x & 31)) {}
    // Blocks of the sequences before `end` (fewer than 2^31 in all: the host sees to that).
    __device__ __forceinline__ uint32_t before(int end) const {
        uint32_t sum = lane < end ? mine : 0u;
        for (int b = lane + 32; b < end; b += 32) sum += of(b);
        return __reduce_add_sync(0xffffffffu, sum);
    }
    // The sequence that position `at` of the line falls into and the position of its first block.
    __device__ __forceinline__ int sequence_at(uint32_t at, uint32_t& base) const {
        uint32_t done = 0;
        for (int b0 = 0; b0 < c.B; b0 += 32) {
            const uint32_t here = b0 == 0 ? mine : of(b0 + lane);
            uint32_t sum = here;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, at < done + sum);
            if (hit) {
                const int src = __ffs(hit) - 1;
                base = done + __shfl_sync(0xffffffffu, sum - here, src);
                return b0 + src;
            }
            done += __shfl_sync(0xffffffffu, sum, 31);
        }
        base = done;
        return c.B;  // behind the line
    }
};

// The line cut into equal pieces: `ctas` of them get blocks (every one at least one), the first `longer` one block more.
struct Cut {
    uint32_t ctas, each, longer;
    __device__ __forceinline__ Cut(uint32_t total, uint32_t most) {
        ctas = min(total, most);
        each = ctas ? total / ctas : 0;
        longer = total - each * ctas;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t i) const { return i * each + min(i, longer); }
    __device__ __forceinline__ uint32_t owner(uint32_t at) const {
        const uint32_t split = longer * (each + 1);
        return at < split ? at / (each + 1) : longer + (at - split) / each;
    }
};

// ------------------------------------------------------------------ instructions
// d = A B + (c0, c1, c0, c1)
template <bool BF16>
__device__ __forceinline__ void mma_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, float c0, float c1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Asynchronous copy of N bytes (zeros when `live` is false: nothing is read then).
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool live) {
    const int bytes = live ? N : 0;
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(bytes) : "memory");
}
// One contiguous copy, counted in bytes on `bar`.
__device__ __forceinline__ void copy_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Code t (0..3) of both halves of a word as a pair of 16-bit floats base<t> + code: the four bits land in the mantissa of
// the base (in BF16 the lowest code is in place already: 128 + code; in FP16 the second: 64 + code).  The integer pipe,
// which has the masks and the shifts, bounds the kernel; shifting by multiplications on the FMA pipe was slower (169
// against 154 us).
template <bool BF16, int t>
__host__ __device__ constexpr float base_of() { return BF16 ? (t == 0 ? 128.f : 16.f) : 64.f; }
struct Bases {
    uint32_t lowest, others;  // the bases' bits in both halves, from the launch: values the compiler does not know stay in
                              // registers, and mask and base go into one three-input logic instruction
};
template <uint32_t mask>
__device__ __forceinline__ uint32_t masked_or(uint32_t x, uint32_t base) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "n"(mask), "r"(base));
    return y;
}
template <bool BF16, int t>
__device__ __forceinline__ uint32_t widen(uint32_t w, const Bases& base) {
    constexpr int to = BF16 ? (t == 0 ? 0 : 3) : 4, shift = to - 4 * t;  // where the four bits go in the mantissa
    const uint32_t x = shift >= 0 ? w << (shift >= 0 ? shift : 0) : w >> (shift < 0 ? -shift : 0);
    return masked_or<(0x000f000fu << to)>(x, BF16 && t == 0 ? base.lowest : base.others);
}
// The same less the base and 8: code - 8, exactly.  In FP16, where the base goes at once, the codes of a byte stay where
// they are (1024 + code, 64 + code), and one shift serves both of the upper byte.  (Taking the bases off by one more
// product, with a constant operand, was slower: 122 against 112 us at 16 x 32768 tokens.)
template <bool BF16, int t>
__device__ __forceinline__ uint32_t centred(uint32_t w, const Bases& base) {
    uint32_t y;
    if constexpr (BF16) {
        const uint32_t x = widen<BF16, t>(w, base);
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(t == 0 ? 0x43084308u : 0x41c041c0u));
    } else {
        const uint32_t at = t < 2 ? w : w >> 8;
        const uint32_t x = t % 2 == 0 ? masked_or<0x000f000fu>(at, base.lowest) : masked_or<0x00f000f0u>(at, base.others);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(t % 2 == 0 ? 0x64086408u : 0x54805480u));
    }
    return y;
}

// What probabilities relative to the maximum m weigh relative to the maximum `top`.  They are formed as 2^(s c2 - round(m
// c2)), so that the weight takes the same rounded products: the references then cancel exactly, however large an offset all
// scores share (with (m - top) c2 the parts of warps, CTAs and re-basings were off by up to ln 2 half steps of m c2 against
// one another: 2 % at scores of 2^19).
__device__ __forceinline__ float reference_weight(float m, float top, float c2) {
    return m == -INFINITY ? 0.f : ex2(__fsub_rn(__fmul_rn(m, c2), __fmul_rn(top, c2)));
}

// ------------------------------------------------------------------ one unit's piece, one warp
// Running state of a warp over its blocks: thread (g, i) = (lane / 4, lane % 4) holds the maximum of query rows 2i and
// 2i + 1, its own part of their sums, and the accumulator of those rows at its channels (channel_of).
template <int D, bool Q4, int NT>
struct State {
    static constexpr int kTiles = D / 16;
    float m[NT][2], l[NT][2], z[NT][2][Q4 ? D / kCacheGroup : 1];
    float o[kTiles][NT][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[n][e] = -INFINITY;
                l[n][e] = 0.f;
#pragma unroll
                for (int g = 0; g < (Q4 ? D / kCacheGroup : 1); ++g) z[n][e][g] = 0.f;
            }
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t][n][e] = 0.f;
    }
};

// Channel of accumulator row `upper` * 8 + g of tile t.
template <bool Q4>
__device__ __forceinline__ int channel_of(int t, int g, int upper) {
    return Q4 ? (t >> 2) * kCacheGroup + 8 * g + (t & 3) + 4 * upper : 16 * t + g + 8 * upper;
}

// Scores of a block in S[mt][n][e] (token mt * 16 + g + 8 * (e >> 1), query row 2i + (e & 1) of row tile n).
template <typename T, int D, int NT>
__device__ __forceinline__ void scores_q4(float (&s)[Cfg<D, true, NT>::kBlock / 16][NT][4], const uint8_t* codes, const uint8_t* params,
                                          const uint32_t (&qf)[NT][D / 16][2], const float (&qsum)[NT][2][D / 64],
                                          const float (&qbase)[NT][2][D / 64], const Bases& base, int g, int i) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    using C = Cfg<D, true, NT>;
#pragma unroll
    for (int mt = 0; mt < C::kBlock / 16; ++mt) {
        const int t0 = mt * 16 + g;
#pragma unroll
        for (int grp = 0; grp < C::kGroups; ++grp) {
            uint32_t w[2][2], pr[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint2 pair = *reinterpret_cast<const uint2*>(codes + (t0 + 8 * u) * C::kRow + grp * 32 + i * 8);
                w[u][0] = pair.x;
                w[u][1] = pair.y;
                pr[u] = *reinterpret_cast<const uint32_t*>(params + (t0 + 8 * u) * C::kParam + grp * 4);
            }
            float acc[NT][4];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t a = w[0][x], b = w[1][x];
                const uint32_t a0 = widen<BF16, 0>(a, base), a1 = widen<BF16, 1>(a, base), a2 = widen<BF16, 2>(a, base), a3 = widen<BF16, 3>(a, base);
                const uint32_t b0 = widen<BF16, 0>(b, base), b1 = widen<BF16, 1>(b, base), b2 = widen<BF16, 2>(b, base), b3 = widen<BF16, 3>(b, base);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (x == 0)
                        mma_from<BF16>(acc[n], a0, b0, a1, b1, qf[n][grp * 4][0], qf[n][grp * 4][1], qbase[n][0][grp], qbase[n][1][grp]);
                    else
                        mma<BF16>(acc[n], a0, b0, a1, b1, qf[n][grp * 4 + 2][0], qf[n][grp * 4 + 2][1]);
                    mma<BF16>(acc[n], a2, b2, a3, b3, qf[n][grp * 4 + x * 2 + 1][0], qf[n][grp * 4 + x * 2 + 1][1]);
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float2 sz = unpack2<BF16>(pr[u]);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        s[mt][n][2 * u + e] =
                            fmaf(sz.x, acc[n][2 * u + e],
                                 grp == 0 ? sz.y * qsum[n][e][0] : fmaf(sz.y, qsum[n][e][grp], s[mt][n][2 * u + e]));
            }
        }
    }
}

template <typename T, int D, int NT>
__device__ __forceinline__ void scores_16(float (&s)[1][NT][4], uint32_t tile, const uint32_t (&qf)[NT][D / 16][2], int lane) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][n][e] = 0.f;
    const int row = (lane & 7) + (lane & 8);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t a[4];
        const int chunk = 2 * ks + (lane >> 4);
        ldmatrix4<false>(a, tile + row * (D * 2) + ((chunk ^ (row & 7)) << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma<BF16>(s[0][n], a[0], a[1], a[2], a[3], qf[n][ks][0], qf[n][ks][1]);
    }
}

// One block: softmax and both products.  CLEAN: every row sees every token of it.
template <typename T, int D, bool Q4, int NT, bool CLEAN>
__device__ __forceinline__ void block_step(State<D, Q4, NT>& st, const uint8_t* stage, const uint32_t (&qf)[NT][D / 16][2],
                                           const float (&qsum)[NT][2][D / 64], const float (&qbase)[NT][2][D / 64],
                                           const CacheAttentionCall& c, const Bases& base, int64_t start,
                                           int key0, int row0, float c2, int lane) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    using C = Cfg<D, Q4, NT>;
    constexpr int MT = C::kBlock / 16;
    const int g = lane >> 2, i = lane & 3;
    float s[MT][NT][4];
    if constexpr (Q4) scores_q4<T, D, NT>(s, stage, stage + C::kBlock * C::kRow, qf, qsum, qbase, base, g, i);
    else scores_16<T, D, NT>(s, smem_u32(stage), qf, lane);

    // The reference of the probabilities is re-based only when a score beats it by more than 2^kSlack in probability
    // terms (which keeps p * scale inside FP16): one vote per block instead of a maximum over the lanes.
    constexpr float kSlack = BF16 ? 8.f : 2.f;
    bool grown = false;
    float mn[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (!CLEAN) {
                const WindowSpan span = window_span(start, (row0 + n * 8 + 2 * i + e) % c.Sq, c.window, c.Sk);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        if (!window_sees(span, c.sinks, key0 + mt * 16 + g + 8 * u)) s[mt][n][2 * u + e] = -INFINITY;
            }
            float mx = st.m[n][e];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mx = max3(mx, s[mt][n][e], s[mt][n][2 + e]);
            mn[n][e] = mx;
            grown = grown || (mx > st.m[n][e] && !((mx - st.m[n][e]) * c2 <= kSlack));  // (also a first score)
        }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) mn[n][e] = fmaxf(mn[n][e], __shfl_xor_sync(0xffffffffu, mn[n][e], o));
                const float alpha = reference_weight(st.m[n][e], mn[n][e], c2);
                st.m[n][e] = mn[n][e];
                st.l[n][e] *= alpha;
                if (Q4) {
#pragma unroll
                    for (int grp = 0; grp < C::kGroups; ++grp) st.z[n][e][Q4 ? grp : 0] *= alpha;
                }
#pragma unroll
                for (int t = 0; t < D / 16; ++t) {
                    st.o[t][n][e] *= alpha;
                    st.o[t][n][2 + e] *= alpha;
                }
            }
    }
    // probabilities, in place of the scores
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            // (the rounding of m c2 is a factor that alpha and the merges' weights share: reference_weight)
            const float mc = !CLEAN && st.m[n][e] == -INFINITY ? 0.f : -__fmul_rn(st.m[n][e], c2);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float& x = s[mt][n][2 * u + e];
                    const float p = ex2(fmaf(x, c2, mc));
                    x = !CLEAN && x == -INFINITY ? 0.f : p;
                    st.l[n][e] += x;
                }
        }

    const uint8_t* values = stage + C::kHalf;
    if constexpr (Q4) {
        const uint8_t* params = values + C::kBlock * C::kRow;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int grp = 0; grp < C::kGroups; ++grp) {
                uint32_t bf[NT][2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float2 sz = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(params + (mt * 16 + g + 8 * u) * C::kParam + grp * 4));
                    const float off = fmaf(sz.x, 8.f, sz.y);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float p0 = s[mt][n][2 * u], p1 = s[mt][n][2 * u + 1];
                        float w0 = p0 * sz.x, w1 = p1 * sz.x;
                        if (CLEAN) {
                            st.z[n][0][grp] = fmaf(p0, off, st.z[n][0][grp]);
                            st.z[n][1][grp] = fmaf(p1, off, st.z[n][1][grp]);
                        } else {  // a token this row does not see may hold anything
                            w0 = p0 == 0.f ? 0.f : w0;
                            w1 = p1 == 0.f ? 0.f : w1;
                            st.z[n][0][grp] += p0 == 0.f ? 0.f : p0 * off;
                            st.z[n][1][grp] += p1 == 0.f ? 0.f : p1 * off;
                        }
                        bf[n][u] = transpose8(pack2<BF16>(w0, w1));
                    }
                }
                uint32_t w[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int token = mt * 16 + 2 * i + (x & 1) + (x >> 1) * 8;
                    w[x] = *reinterpret_cast<const uint32_t*>(values + token * C::kRow + grp * 32 + g * 4);
                }
                const uint32_t lo0 = __byte_perm(w[0], w[1], 0x5410), hi0 = __byte_perm(w[0], w[1], 0x7632);
                const uint32_t lo1 = __byte_perm(w[2], w[3], 0x5410), hi1 = __byte_perm(w[2], w[3], 0x7632);
                auto tile = [&](auto t_) {
                    constexpr int t = decltype(t_)::value;
                    const uint32_t a0 = centred<BF16, t>(lo0, base), a1 = centred<BF16, t>(hi0, base);
                    const uint32_t a2 = centred<BF16, t>(lo1, base), a3 = centred<BF16, t>(hi1, base);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma<BF16>(st.o[grp * 4 + t][n], a0, a1, a2, a3, bf[n][0], bf[n][1]);
                };
                tile(std::integral_constant<int, 0>{});
                tile(std::integral_constant<int, 1>{});
                tile(std::integral_constant<int, 2>{});
                tile(std::integral_constant<int, 3>{});
            }
        }
    } else {
        uint32_t bf[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) bf[n][u] = transpose8(pack2<BF16>(s[0][n][2 * u], s[0][n][2 * u + 1]));
        const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            uint32_t a[4];
            const int chunk = 2 * t + ((lane >> 3) & 1);
            ldmatrix4<true>(a, smem_u32(values) + row * (D * 2) + ((chunk ^ (row & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma<BF16>(st.o[t][n], a[0], a[1], a[2], a[3], bf[n][0], bf[n][1]);
        }
    }
}

// ------------------------------------------------------------------ kernels
template <typename T, int D, bool Q4, int NT>
__global__ void __launch_bounds__(kWarps * 32, resident<D, Q4, NT>()) decode_rows(const RowsCall p) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    using C = Cfg<D, Q4, NT>;
    constexpr int R = 8 * NT;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float sm_m[kWarps][R], sm_l[kWarps][R];
    __shared__ uint64_t arrived[kWarps][C::kStages];  // 4-bit caches with dense rows: the stage's codes are there
    __shared__ int abort_word;
    const CacheAttentionCall& c = p.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge may be scheduled; it waits for this grid
    const uint32_t units = c.Hkv * p.chunks;
    // This CTA's piece of the line; in a cluster its share of one unit, counted from that unit's first block.
    const Line line(c, units, C::kBlock);
    const uint32_t my_unit = p.cluster ? blockIdx.x / p.cluster : 0, my_rank = p.cluster ? blockIdx.x % p.cluster : 0;
    uint32_t begin, end;
    if (p.cluster) {
        const uint32_t n = blocks_of(c, start_of(c, (int)(my_unit / units)), C::kBlock).count;
        begin = n * my_rank / p.cluster;
        end = n * (my_rank + 1) / p.cluster;
    } else {
        const Cut cut(line.before(c.B), p.ctas);
        if (blockIdx.x >= cut.ctas) return;
        begin = cut.begin(blockIdx.x);
        end = cut.begin(blockIdx.x + 1);
    }
    uint8_t* my_ring = ring + warp * C::kStages * C::kStage;
    const float c2 = fabsf(c.scale) * kLog2e;
    const Bases bases{p.lowest, p.others};
    State<D, Q4, NT> st;
    // Dense rows of codes come as two contiguous copies per block (one of keys, one of values), which cost one thread
    // a few instructions instead of eight address computations per lane.
    const bool packed = Q4 && c.half[0].ps[2] == 2 * C::kGroups && c.half[1].ps[2] == 2 * C::kGroups;
    const bool dense = Q4 && c.half[0].cs[2] == C::kRow && c.half[1].cs[2] == C::kRow;
    int at_stage = 0, into = 0;   // the stage that is read next, and the one that is filled next
    uint32_t parity = 0;          // of the arrival at the stage that is read next
    if (threadIdx.x == 0) abort_word = *reinterpret_cast<volatile int*>(c.abort_flag) != 0 ? 90 : 0;
    if (lane == 0) {
        for (int n = 0; n < C::kStages; ++n) mbar_init(&arrived[warp][n], 1);
        mbar_fence_init();
    }
    __syncthreads();
    bool ok = abort_word == 0;
    if (!ok) {
        if (!p.cluster) return;
        end = begin;  // (a cluster's CTAs stay to its barriers: the others read this one's part)
    }
    float* sm_o = reinterpret_cast<float*>(ring);              // [warp][R][D], where the ring is idle
    float* cta_o = sm_o + kWarps * R * D;                       // a cluster's CTA: its part, [R][D]
    float2* cta_ml = reinterpret_cast<float2*>(cta_o + R * D);  // and its (maximum, sum), [R]

    for (uint32_t at = begin; at < end;) {
        uint32_t base = 0;
        const int b = p.cluster ? (int)(my_unit / units) : line.sequence_at(at, base);
        const int64_t start = start_of(c, b);
        const Blocks blocks = blocks_of(c, start, C::kBlock);
        const int unit = p.cluster ? (int)(my_unit % units) : (int)((at - base) / (uint32_t)blocks.count);
        const int from = p.cluster ? (int)at : (int)(at - base) - unit * blocks.count;
        const int count = min((int)(end - at), blocks.count - from);
        const int kvh = unit / p.chunks, row0 = unit % p.chunks * R;
        const WindowSpan low = window_span(start, 0, c.window, c.Sk), high = window_span(start, c.Sq - 1, c.window, c.Sk);

        // the copies of this warp's block `n` (blocks warp, warp + kWarps, ... of the piece) into its ring
        const int mine = count > warp ? (count - warp + kWarps - 1) / kWarps : 0;
        const uint8_t* plane[2];
        const uint8_t* param_plane[2] = {};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if constexpr (Q4) {
                const CacheView& v = c.half[half];
                plane[half] = v.codes + b * v.cs[0] + kvh * v.cs[1];
                param_plane[half] = reinterpret_cast<const uint8_t*>(v.params + b * v.ps[0] + kvh * v.ps[1]);
            } else {
                plane[half] = static_cast<const uint8_t*>(p.kv[half]) + 2 * (b * p.kvs[half][0] + kvh * p.kvs[half][1]);
            }
        }
        const bool bulk_params = packed && dense && ((reinterpret_cast<uintptr_t>(param_plane[0]) |
                                                      reinterpret_cast<uintptr_t>(param_plane[1])) & 15) == 0;
        auto request = [&](int n) {
            if (n < mine) {
                const int key0 = blocks.block(from + warp + n * kWarps) * C::kBlock;
                const uint32_t dst = smem_u32(my_ring + into * C::kStage);
                if constexpr (Q4) {
                    // scales and zeros come contiguously too where they can (a whole block, 16-byte aligned)
                    const bool with_params = bulk_params && key0 + C::kBlock <= c.Sk;
                    if (!with_params) {
#pragma unroll
                        for (int token = lane; token < C::kBlock; token += 32) {
                            const int key = key0 + token;
                            const bool live = key < high.hi && (key >= low.lo || key < c.sinks);
#pragma unroll
                            for (int half = 0; half < 2; ++half)
                                copy_async<C::kParam>(dst + half * C::kHalf + C::kBlock * C::kRow + token * C::kParam,
                                                      param_plane[half] + (live ? key * c.half[half].ps[2] * 2 : 0), live);
                        }
                    }
                    if (dense) {
                        // (tokens that no row sees come along; rows behind the cache's end do not, and leave what was
                        // there before: a code is a finite number whatever it is)
                        if (lane == 0) {
                            const uint32_t bytes = min(C::kBlock, c.Sk - key0) * C::kRow;
                            uint64_t* bar = &arrived[warp][into];
                            mbar_expect_tx(bar, 2 * bytes + (with_params ? 2 * C::kBlock * C::kParam : 0));
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                copy_bulk(dst + half * C::kHalf, plane[half] + (int64_t)key0 * C::kRow, bytes, bar);
                                if (with_params)
                                    copy_bulk(dst + half * C::kHalf + C::kBlock * C::kRow,
                                              param_plane[half] + (int64_t)key0 * C::kParam, C::kBlock * C::kParam, bar);
                            }
                        }
                        copy_commit();
                        into = into + 1 == C::kStages ? 0 : into + 1;
                        return;
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    constexpr int kChunks = C::kRow / 16;
                    const uint8_t* src = plane[half];
                    const int64_t step = Q4 ? c.half[half].cs[2] : 2 * p.kvs[half][2];
#pragma unroll
                    for (int x = 0; x < C::kBlock * kChunks / 32; ++x) {
                        const int idx = x * 32 + lane, token = idx / kChunks, chunk = idx % kChunks, key = key0 + token;
                        const bool live = key < high.hi && (key >= low.lo || key < c.sinks);
                        const int to = Q4 ? chunk : chunk ^ (token & 7);
                        copy_async<16>(dst + half * C::kHalf + token * C::kRow + to * 16, src + (live ? key * step : 0) + chunk * 16, live);
                    }
                }
                into = into + 1 == C::kStages ? 0 : into + 1;
            }
            copy_commit();
        };
#pragma unroll
        for (int n = 0; n < C::kStages - 1; ++n) request(n);

        // the query rows as operand B, and their sums over the groups
        uint32_t qf[NT][D / 16][2];
        float qsum[NT][2][D / 64], qbase[NT][2][D / 64];  // sum_d q_d and -sum_d q_d base_d of query rows 2i, 2i + 1
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = row0 + n * 8 + g;
            const bool live = r < p.rows;
            const int head = kvh * c.group + r / c.Sq, sq = r % c.Sq;
            const T* qrow = static_cast<const T*>(c.q) + (live ? b * c.qs[0] + head * c.qs[1] + sq * c.qs[2] : 0);
            const uint32_t flip = c.scale < 0.f ? 0x80008000u : 0u;
            if constexpr (Q4) {
#pragma unroll
                for (int grp = 0; grp < C::kGroups; ++grp) {
                    float sum = 0.f, based = 0.f;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        uint4 raw = live ? *reinterpret_cast<const uint4*>(qrow + grp * 64 + i * 16 + x * 8) : make_uint4(0, 0, 0, 0);
                        raw.x ^= flip, raw.y ^= flip, raw.z ^= flip, raw.w ^= flip;
                        // channels 0..7 in raw.x .. raw.w; a pair is (channel j, channel j + 4)
                        qf[n][grp * 4 + x * 2][0] = __byte_perm(raw.x, raw.z, 0x5410);
                        qf[n][grp * 4 + x * 2][1] = __byte_perm(raw.x, raw.z, 0x7632);
                        qf[n][grp * 4 + x * 2 + 1][0] = __byte_perm(raw.y, raw.w, 0x5410);
                        qf[n][grp * 4 + x * 2 + 1][1] = __byte_perm(raw.y, raw.w, 0x7632);
                        const float2 e0 = unpack2<BF16>(raw.x), e1 = unpack2<BF16>(raw.y), e2 = unpack2<BF16>(raw.z),
                                     e3 = unpack2<BF16>(raw.w);
                        const float first = e0.x + e2.x, rest = ((e0.y + e2.y) + (e1.x + e3.x)) + (e1.y + e3.y);
                        sum += first + rest;
                        based -= base_of<BF16, 0>() * first + base_of<BF16, 1>() * rest;
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);  // row g
                    based += __shfl_xor_sync(0xffffffffu, based, 1);
                    based += __shfl_xor_sync(0xffffffffu, based, 2);
                    qsum[n][0][grp] = __shfl_sync(0xffffffffu, sum, 8 * i);
                    qsum[n][1][grp] = __shfl_sync(0xffffffffu, sum, 8 * i + 4);
                    qbase[n][0][grp] = __shfl_sync(0xffffffffu, based, 8 * i);
                    qbase[n][1][grp] = __shfl_sync(0xffffffffu, based, 8 * i + 4);
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        qf[n][ks][x] = live ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + x * 8 + 2 * i) ^ flip : 0u;
            }
        }

        st.clear();
        for (int n = 0; n < mine; ++n) {
            copy_wait<C::kStages - 2>();
            if (dense) {
                ok = mbar_wait(&arrived[warp][at_stage], parity, &abort_word, 1);
                if (__any_sync(0xffffffffu, !ok)) {
                    // gave up: a last, short wait for the copies still under way, then to the tear-down
                    for (int m = n; m < mine && m < n + C::kStages - 1; ++m) {
                        for (int tries = 0; tries < 4096 && !mbar_try_wait(&arrived[warp][at_stage], parity); ++tries) {}
                        at_stage = at_stage + 1 == C::kStages ? 0 : at_stage + 1;
                        parity ^= at_stage == 0 ? 1u : 0u;
                    }
                    break;
                }
            }
            __syncwarp();
            request(n + C::kStages - 1);  // into the stage that the previous block has left
            const int key0 = blocks.block(from + warp + n * kWarps) * C::kBlock;
            const uint8_t* stage = my_ring + at_stage * C::kStage;
            at_stage = at_stage + 1 == C::kStages ? 0 : at_stage + 1;
            parity ^= at_stage == 0 ? 1u : 0u;
            const bool clean = key0 + C::kBlock <= low.hi && (key0 >= high.lo || key0 + C::kBlock <= c.sinks);
            if (clean) block_step<T, D, Q4, NT, true>(st, stage, qf, qsum, qbase, c, bases, start, key0, row0, c2, lane);
            else block_step<T, D, Q4, NT, false>(st, stage, qf, qsum, qbase, c, bases, start, key0, row0, c2, lane);
            __syncwarp();
        }
        copy_wait<0>();

        // the warps of the CTA, merged in a fixed order through the (now idle) ring
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = st.l[n][e];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                const int r = n * 8 + 2 * i + e;
                if (g == 0) {
                    sm_m[warp][r] = st.m[n][e];
                    sm_l[warp][r] = l;
                }
                float z[Q4 ? D / 64 : 1] = {};
                if (Q4) {
#pragma unroll
                    for (int grp = 0; grp < D / 64; ++grp) {
                        float x = st.z[n][e][Q4 ? grp : 0];
                        x += __shfl_xor_sync(0xffffffffu, x, 4);
                        x += __shfl_xor_sync(0xffffffffu, x, 8);
                        x += __shfl_xor_sync(0xffffffffu, x, 16);
                        z[Q4 ? grp : 0] = x;
                    }
                }
#pragma unroll
                for (int t = 0; t < D / 16; ++t)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        sm_o[(warp * R + r) * D + channel_of<Q4>(t, g, u)] = st.o[t][n][2 * u + e] + z[Q4 ? t >> 2 : 0];
            }
        __syncthreads();
        const bool whole = count == blocks.count;
        const int slot = at == begin ? 0 : 1;
        for (int idx = threadIdx.x; idx < R * (D / 4); idx += kWarps * 32) {
            const int r = idx / (D / 4), d = idx % (D / 4) * 4;
            float mx = sm_m[0][r];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, sm_m[w][r]);
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float weight = reference_weight(sm_m[w][r], mx, c2);
                const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * R + r) * D + d);
                sum += sm_l[w][r] * weight;
                acc.x = fmaf(x.x, weight, acc.x), acc.y = fmaf(x.y, weight, acc.y);
                acc.z = fmaf(x.z, weight, acc.z), acc.w = fmaf(x.w, weight, acc.w);
            }
            if (p.cluster) {
                *reinterpret_cast<float4*>(cta_o + r * D + d) = acc;
                if (d == 0) cta_ml[r] = make_float2(mx, sum);
            } else if (whole) {
                const int row = row0 + r;
                if (row < p.rows) {
                    const float inv = sum > 0.f ? 1.f / sum : 0.f;
                    T* out = static_cast<T*>(c.out) + b * c.os[0] + (kvh * c.group + row / c.Sq) * c.os[1] + row % c.Sq * c.os[2] + d;
                    *reinterpret_cast<uint2*>(out) =
                        make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
                }
            } else {
                const int64_t piece = ((int64_t)blockIdx.x * 2 + slot) * R + r;
                *reinterpret_cast<float4*>(p.part_o + piece * D + d) = acc;
                if (d == 0) *reinterpret_cast<float2*>(p.part_ml + piece * 2) = make_float2(mx, sum);
            }
        }
        fence_async_smem();  // the next piece's contiguous copies come in behind what was written here
        __syncthreads();
        at += count;
        if (abort_word != 0) break;
    }
    if (p.cluster) {
        if (begin == end) {  // no block for this CTA
            for (int r = threadIdx.x; r < R; r += kWarps * 32) cta_ml[r] = make_float2(-INFINITY, 0.f);
            for (int x = threadIdx.x; x < R * D / 4; x += kWarps * 32) reinterpret_cast<float4*>(cta_o)[x] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        cluster_barrier();
        const int b = (int)(my_unit / units), unit = (int)(my_unit % units), kvh = unit / p.chunks, row0 = unit % p.chunks * R;
        for (int idx = threadIdx.x * p.cluster + my_rank; idx < R * (D / 4); idx += kWarps * 32 * p.cluster) {
            const int r = idx / (D / 4), d = idx % (D / 4) * 4, row = row0 + r;
            if (row >= p.rows) break;
            float2 ml[kCluster];
            float4 x[kCluster];
            float mx = -INFINITY, sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kCluster; ++w) {
                if (w < p.cluster) {
                    ml[w] = cluster_load2(cluster_address(cta_ml + r, w));
                    x[w] = cluster_load4(cluster_address(cta_o + r * D + d, w));
                } else {
                    ml[w] = make_float2(-INFINITY, 0.f);
                    x[w] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
                mx = fmaxf(mx, ml[w].x);
            }
#pragma unroll
            for (int w = 0; w < kCluster; ++w) {
                const float weight = reference_weight(ml[w].x, mx, c2);
                sum += ml[w].y * weight;
                acc.x = fmaf(x[w].x, weight, acc.x), acc.y = fmaf(x[w].y, weight, acc.y);
                acc.z = fmaf(x[w].z, weight, acc.z), acc.w = fmaf(x[w].w, weight, acc.w);
            }
            const float inv = sum > 0.f ? 1.f / sum : 0.f;
            T* out = static_cast<T*>(c.out) + b * c.os[0] + (kvh * c.group + row / c.Sq) * c.os[1] + row % c.Sq * c.os[2] + d;
            *reinterpret_cast<uint2*>(out) = make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
        }
        cluster_barrier();  // nobody leaves while its part is read
    }
    if (threadIdx.x == 0 && abort_word != 0) {
        *c.status = 5000 + abort_word;
        *reinterpret_cast<volatile int*>(c.abort_flag) = 1;  // later tensor-memory and decoding launches skip their work
    }
}

// One CTA per unit: units that one CTA served whole are done; the others' pieces are merged, in an order that the cut
// alone decides; a sequence without a visible key gets its zeros here.
template <typename T, int D, bool Q4, int NT>
__global__ void __launch_bounds__(1024) merge_rows(const RowsCall p) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    using C = Cfg<D, Q4, NT>;
    constexpr int R = 8 * NT;
    constexpr int kLanes = D / 4, kParts = 1024 / kLanes / R;  // four channels per thread; a row's pieces kParts at a time
    const CacheAttentionCall& c = p.c;
    const uint32_t units = c.Hkv * p.chunks;
    const int b = (int)(blockIdx.x / units), unit = (int)(blockIdx.x % units);
    const int kvh = unit / p.chunks, row0 = unit % p.chunks * R;
    const Line line(c, units, C::kBlock);
    const Cut cut(line.before(c.B), p.ctas);
    const int count = blocks_of(c, start_of(c, b), C::kBlock).count;
    int first = 0, last = -1;
    uint32_t u0 = 0;
    if (count > 0) {
        u0 = line.before(b) + (uint32_t)unit * count;
        first = (int)cut.owner(u0);
        last = (int)cut.owner(u0 + count - 1);
    }
    // (also where there is nothing to merge: this grid's end has to mean the end of the other one)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (count > 0 && first == last) return;
    const float c2 = fabsf(c.scale) * kLog2e;
    const int slot0 = count > 0 && u0 == cut.begin(first) ? 0 : 1;
    const int lane = threadIdx.x % kLanes, part = threadIdx.x / kLanes % kParts, r = threadIdx.x / kLanes / kParts, d = lane * 4;
    if (row0 + r >= p.rows) last = -1;  // (first > last: nothing to do, and nothing written below)
    float mx = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // this thread's pieces (part, part + kParts, ...): their loads do not depend on one another
#pragma unroll 8
    for (int i = first + part; i <= last; i += kParts) {
        const int64_t piece = ((int64_t)i * 2 + (i == first ? slot0 : 0)) * R + r;
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + piece * 2);
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + piece * D + d);
        const float m = fmaxf(mx, ml.x);
        const float keep = reference_weight(mx, m, c2), weight = reference_weight(ml.x, m, c2);
        mx = m;
        sum = sum * keep + ml.y * weight;
        acc.x = fmaf(x.x, weight, acc.x * keep), acc.y = fmaf(x.y, weight, acc.y * keep);
        acc.z = fmaf(x.z, weight, acc.z * keep), acc.w = fmaf(x.w, weight, acc.w * keep);
    }
    if constexpr (kParts > 1) {
        __shared__ float sm_m[R][kParts], sm_l[R][kParts];
        __shared__ float4 sm_o[R][kParts][kLanes];
        sm_o[r][part][lane] = acc;
        if (lane == 0) {
            sm_m[r][part] = mx;
            sm_l[r][part] = sum;
        }
        __syncthreads();
        if (part != 0) return;
        for (int w = 1; w < kParts; ++w) mx = fmaxf(mx, sm_m[r][w]);
        sum = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kParts; ++w) {
            const float weight = reference_weight(sm_m[r][w], mx, c2);
            const float4 x = sm_o[r][w][lane];
            sum += sm_l[r][w] * weight;
            acc.x = fmaf(x.x, weight, acc.x), acc.y = fmaf(x.y, weight, acc.y);
            acc.z = fmaf(x.z, weight, acc.z), acc.w = fmaf(x.w, weight, acc.w);
        }
    }
    if (row0 + r >= p.rows) return;
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const int row = row0 + r;
    T* out = static_cast<T*>(c.out) + b * c.os[0] + (kvh * c.group + row / c.Sq) * c.os[1] + row % c.Sq * c.os[2] + d;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
}

// ------------------------------------------------------------------ host
template <int D, bool Q4, int NT>
int64_t most_blocks(const CacheAttentionCall& c) {  // of one unit
    constexpr int size = Cfg<D, Q4, NT>::kBlock;
    const int64_t keys = c.window < c.Sk ? c.window + c.Sq - 1 : c.Sk;
    const int64_t all = (c.Sk + size - 1) / size, some = (keys + size - 1) / size + 1 + (c.sinks + size - 1) / size;
    return some < all ? some : all;
}

// Whether the line of blocks can be counted in 31 bits.
template <int D, bool Q4>
bool countable(const CacheAttentionCall& c) {
    const int64_t chunks = ((int64_t)c.group * c.Sq + 7) / 8;
    return (int64_t)c.B * c.Hkv * chunks * 8 <= INT32_MAX && (int64_t)c.B * c.Hkv * chunks * most_blocks<D, Q4, 2>(c) <= INT32_MAX;
}

inline int row_tiles(const CacheAttentionCall& c) { return (int64_t)c.group * c.Sq <= 8 ? 1 : 2; }

template <int D, bool Q4, int NT>
int plan_ctas(const CacheAttentionCall& c, int chunks) {
    // As many CTAs as are resident at once, but no fewer blocks for a CTA than it has warps.
    const int64_t line = (int64_t)c.B * c.Hkv * chunks * most_blocks<D, Q4, NT>(c);
    const int64_t most = 148 * resident<D, Q4, NT>();
    const int64_t want = (line + kWarps - 1) / kWarps;
    return (int)(want < 1 ? 1 : (want > most ? most : want));
}

// The CTAs of a cluster per unit, or 0 for the line of blocks cut over all CTAs and a second launch that merges.
// Clusters of at most eight, nine tenths of what is resident (at 48 units of six, 97 % of the places, some did not find
// theirs in a first wave: 14.1 us, five each 8.5, the line 11.0), where a warp gets at most two rounds of blocks more
// than in the line, which costs a second launch and a second start at every cut; four for 16-bit rows, whose blocks
// are a quarter as long.  D128, 32 query heads on 8, GPU time of a step in a graph, line -> clusters:
//   4-bit: B1 1024 tokens 7.9 -> 8.0 us, 4096 10.0 -> 10.0, 8192 (3 rounds more, kept in the line) 12.4 -> 13.4;
//     B6 4096 19.1 -> 15.0; B12 8192 38.5 -> 35.3; B16 8192 46.4 -> 45.0, 16384 (3 more) 76.8 -> 80.9;
//     64 heads, 4 rows, B8 4096 41.0 -> 38.0.
//   16-bit: B1 window 256 9.4 -> 6.3, 1024 10.7 -> 8.0, 2048 13.0 -> 9.9, 4000 (7 more) 12.3 -> 12.5;
//     B8 window 1024 13.9 -> 11.3; B12 window 1000 15.5 -> 14.6; B32 window 1024 29.0 -> 25.5.
// Outside graphs a call saves 2.5 us of host time besides.
template <int D, bool Q4, int NT>
int cluster_size(const CacheAttentionCall& c, int chunks) {
    const int64_t units = (int64_t)c.B * c.Hkv * chunks, blocks = most_blocks<D, Q4, NT>(c);
    const int64_t fit = 133 * resident<D, Q4, NT>() / units, size = fit < kCluster ? fit : kCluster;
    if (size == 0) return 0;
    const int64_t line = (int64_t)plan_ctas<D, Q4, NT>(c, chunks) * kWarps;
    const int64_t rounds = (blocks + size * kWarps - 1) / (size * kWarps), spread = (units * blocks + line - 1) / line;
    return rounds <= spread + (Q4 ? 2 : 4) ? (int)size : 0;
}

template <int D, bool Q4>
size_t workspace_bytes(const CacheAttentionCall& c) {
    const int NT = row_tiles(c), R = 8 * NT, chunks = (c.group * c.Sq + R - 1) / R;
    // (a call that clusters serve keeps nothing; 16 bytes keep the size positive)
    if (NT == 1 ? cluster_size<D, Q4, 1>(c, chunks) : cluster_size<D, Q4, 2>(c, chunks)) return 16;
    const int ctas = NT == 1 ? plan_ctas<D, Q4, 1>(c, chunks) : plan_ctas<D, Q4, 2>(c, chunks);
    return (size_t)ctas * 2 * R * (D + 2) * sizeof(float);
}

template <typename T, int D, bool Q4, int NT>
cudaError_t launch(RowsCall& p, void* workspace, cudaStream_t st) {
    using C = Cfg<D, Q4, NT>;
    constexpr int R = 8 * NT;
    constexpr int kMerge = kWarps * R * D * 4;
    constexpr int kSmem = C::kRing > kMerge ? C::kRing : kMerge;
    p.rows = p.c.group * p.c.Sq;
    p.chunks = (p.rows + R - 1) / R;
    p.cluster = cluster_size<D, Q4, NT>(p.c, p.chunks);
    p.ctas = p.cluster ? p.c.B * p.c.Hkv * p.chunks * p.cluster : plan_ctas<D, Q4, NT>(p.c, p.chunks);
    p.lowest = std::is_same<T, __nv_bfloat16>::value ? 0x43004300u : 0x64006400u;  // 128 or 1024
    p.others = std::is_same<T, __nv_bfloat16>::value ? 0x41804180u : 0x54005400u;  // 16 or 64
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + (size_t)p.ctas * 2 * R * D;
    // the shared-memory opt-in holds per device; a decoding step is short enough for the call to show, so it is made once
    static std::atomic<uint64_t> opted{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (!(opted.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(decode_rows<T, D, Q4, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return e;
        opted.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t config = {};
    if (p.cluster) {
        static_assert(C::kRing >= (kWarps + 1) * R * D * 4 + R * 8, "the warps' and the CTA's rows go through the ring");
        config.gridDim = dim3((unsigned)p.ctas);
        config.blockDim = dim3(kWarps * 32);
        config.dynamicSmemBytes = kSmem;
        config.stream = st;
        cudaLaunchAttribute together[1];
        together[0].id = cudaLaunchAttributeClusterDimension;
        together[0].val.clusterDim.x = (unsigned)p.cluster;
        together[0].val.clusterDim.y = together[0].val.clusterDim.z = 1;
        config.attrs = together;
        config.numAttrs = 1;
        return cudaLaunchKernelEx(&config, decode_rows<T, D, Q4, NT>, (const RowsCall)p);
    }
    decode_rows<T, D, Q4, NT><<<p.ctas, kWarps * 32, kSmem, st>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    config.gridDim = dim3((unsigned)((int64_t)p.c.B * p.c.Hkv * p.chunks));
    config.blockDim = dim3(1024);
    config.stream = st;
    cudaLaunchAttribute dependent[1];
    dependent[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    dependent[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = dependent;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, merge_rows<T, D, Q4, NT>, (const RowsCall)p);
}

template <typename T, bool Q4>
cudaError_t dispatch(RowsCall& p, void* workspace, cudaStream_t st) {
    const bool one = row_tiles(p.c) == 1;
    if (p.c.D == 128)
        return one ? launch<T, 128, Q4, 1>(p, workspace, st) : launch<T, 128, Q4, 2>(p, workspace, st);
    return one ? launch<T, 64, Q4, 1>(p, workspace, st) : launch<T, 64, Q4, 2>(p, workspace, st);
}

}  // namespace rows
}  // namespace kfa
