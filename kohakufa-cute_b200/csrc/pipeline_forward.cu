// Attention forward on the Blackwell tensor-memory pipeline (tcgen05 + TMEM + TMA),
// head dims that are multiples of 8 up to 128 (run as 64 or 128 channels: the tiled loads fill the channels
// beyond the head with zeros, which add nothing to either product, and the tiled store drops them again),
// FP16/BF16, causal and/or boolean masks, grouped-query heads.
//
// One CTA owns 256 query rows of one (batch, query head) as two 128-row tiles and walks the 128-key tiles they can see.
// Warp roles (384 threads):
//   warps 0-3  softmax of query tile 0   (thread i <-> TMEM lane i <-> query row i)
//   warps 4-7  softmax of query tile 1
//   warp  8    issues every tcgen05.mma (one elected lane), owns the TMEM allocation
//   warp  9    TMA loader (one elected lane); warps 10-11 idle (they complete the warpgroup so
//              that registers can be moved from it to the softmax warpgroups)
// Tensor memory (512 columns): S0 | S1 | O0 | O1, 128 columns each.  Windowed calls: one tile of 128 rows, 256 threads
// (warps 0-3 softmax, 4 products, 5 loader, 6-7 idle), S | O in 256 columns, and two such CTAs per SM.
// The 16-bit probabilities overwrite the first 64 columns of their score tile and feed the second
// product straight from tensor memory; they are handed over in two halves of 64 keys, so
// the first half of P*V runs while the second half of the exponentials is formed.  While
// one tile's softmax runs, the tensor core works on the other tile (of the other CTA in windowed calls), and K/V tiles
// are shared by both tiles of a CTA.  Block-wise callers (one block of a longer key sequence per call) get
// the tile folded into a running FP32 state instead of a normalised output.
//
// Arithmetic (reference behaviour: src/kohakufa_cute/blackwell_pipeline.py:141-209,
// 423-439 and kernels.py:1286-1333 of the reference project): scores are used unscaled,
// the row maximum is subtracted before the multiplication by |scale|*log2e, the
// normaliser sums unrounded probabilities while the product uses probabilities rounded
// once to the input type, and the saved statistics are the exact unscaled row maximum
// and log2 of the normaliser relative to it.  The accumulator is re-based only when
// the running maximum has grown by more than 2^8 in probability terms; the statistics
// are corrected for the difference at the end, so they do not depend on that choice.
#include "kfa_common.cuh"
#include "launchers.h"
#include "sm100_ptx.cuh"
#include "tensor_map.h"
#include "window.cuh"

#include <atomic>
#include <type_traits>

namespace kfa {
namespace {


constexpr int kTileQ = 128;
constexpr int kTileK = 128;
// Query tiles per CTA: two that share their K/V tiles, in one CTA per SM; in windowed calls one, in two CTAs per SM.  A
// window gives a CTA only a few key tiles (ten at a window of 1024), so that start-up and drain, which a CTA alone on its
// SM leaves idle, were a third of its time.
__host__ __device__ constexpr int threads_of(int tiles) { return 128 * tiles + 128; }  // softmax warpgroups; (MMA, loader, 2 idle warps)
// The accumulator is re-based when the row maximum has grown by more than 2^kRebase in probability terms.  Until then
// probabilities are formed against the stale maximum and may reach 2^kRebase: 2^14 stays inside FP16, and BF16 has
// FP32's range (row sums stay below 2^32 * keys, far inside FP32).  Re-basing costs a round trip of the output
// accumulator through registers on the softmax's critical path, so it should be rare also for large logits.
template <bool BF16>
__host__ __device__ constexpr float rebase_limit() { return BF16 ? 32.0f : 14.0f; }
constexpr int kMaxKeyTiles = 4096;  // masked calls keep one state byte per key tile in shared memory

template <int D, int TILES>
struct FwdCfg {
    static constexpr int kChunks = D / 64;                 // 64-channel TMA boxes per tile
    static constexpr int kTileBytes = kTileK * D * 2;      // one Q, K or V tile
    static constexpr int kStages = TILES == 2 ? (D == 128 ? 4 : 6) : (D == 128 ? 2 : 4);  // K/V ring slots
    static constexpr int kSmemBytes =
        TILES * kTileBytes + kStages * kTileBytes + 1024 /*align*/ + 256 /*barriers*/ + kMaxKeyTiles;
};

struct FwdMaps {
    CUtensorMap q, k, v, o;
};

struct Shared {
    uint64_t q_full;
    uint64_t kv_full[6];
    uint64_t kv_empty[6];
    uint64_t s_ready[2];
    uint64_t p_half[2][2];  // [tile][half of the keys]: those probabilities of the tile are in tensor memory
    uint64_t o_staged[2];  // every softmax thread of the tile has put its output row into shared memory
    uint32_t tmem_base;
    int abort_word;
    uint8_t tile_state[kMaxKeyTiles];  // per key tile of this CTA: 0 hidden, 1 mixed, 2 visible (masked calls)
};

// Combined state of key tile j (128 keys) for the CTA's query rows [q0, q0 + 256), from the 64x64
// table entries: 0 hidden, 2 visible, 1 mixed.  Masks broadcast over queries have one row of entries.
__device__ __forceinline__ int key_tile_state(const AttnParams& p, int b, int h, int q0, int j) {
    if (!p.has_mask) return 2;
    const int nk64 = (p.Sk + 63) >> 6;
    const int32_t* base = p.blocks + (int64_t)b * p.bs[0] + (int64_t)h * p.bs[1];
    int r0 = 0, r1 = 0;
    if (p.bs[2] != 0) {
        r0 = q0 >> 6;
        r1 = (min(q0 + 2 * kTileQ, p.Sq) - 1) >> 6;
    }
    const int c1 = min(2 * j + 1, nk64 - 1);
    bool any = false, all = true;
    for (int r = r0; r <= r1; ++r)
        for (int c = 2 * j; c <= c1; ++c) {
            const int s = base[(int64_t)r * p.bs[2] + (int64_t)c * p.bs[3]];
            any = any || s != 0;
            all = all && s == 2;
        }
    return all ? 2 : (any ? 1 : 0);
}

// MASKED = false is the instantiation for calls without a mask (the flag is cleared at compile time).
// WINDOW is the instantiation for sliding-window calls (window.cuh; neither a mask nor `causal` then): the query tile
// walks the key tiles of the sinks and of its window, and positions come from device memory where the call gives one per
// sequence.  With `key_splits` a cluster of CTAs shares a tile's keys.
template <int D, bool BF16, bool MASKED, bool WINDOW>
__global__ void __launch_bounds__(threads_of(WINDOW ? 1 : 2), WINDOW ? 2 : 1)
    pipeline_forward(const __grid_constant__ FwdMaps maps, AttnParams p) {
    if (!MASKED) p.has_mask = 0;
    constexpr int kTiles = WINDOW ? 1 : 2, kThreads = threads_of(kTiles), kRoleWarp = 4 * kTiles;
    constexpr uint32_t kColO = 128 * kTiles, kTmemCols = 256 * kTiles;  // accumulators behind the score tiles
    using Cfg = FwdCfg<D, kTiles>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;                              // the query tiles
    uint8_t* sKV = smem + kTiles * Cfg::kTileBytes;  // ring of K/V tiles
    Shared& sh = *reinterpret_cast<Shared*>(sKV + Cfg::kStages * Cfg::kTileBytes);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // A windowed call of few query tiles: a cluster of CTAs per tile, each with a piece of its key tiles.
    const int splits = WINDOW && p.key_splits > 1 ? p.key_splits : 1;
    const unsigned block = blockIdx.x / splits;
    const int piece = blockIdx.x % splits;
    const int nblk = (p.Sq + kTiles * kTileQ - 1) / (kTiles * kTileQ);
    // Heavy (late) causal blocks first.  Large grids go head by head (a head's CTAs share K/V in L2 and the
    // last wave is made of light blocks); grids of a few waves go block-row by block-row over all heads, so
    // that no head's heavy blocks start in the last wave.
    const int64_t nbh = (int64_t)p.B * p.Hq;
    // (row by row also when all K/V of the call fit in half of L2: measured 4.6 % faster on 2048 CTAs)
    const bool by_row = (int64_t)(gridDim.x / splits) < KFA_ROW_MAJOR_LIMIT ||
                        (int64_t)p.B * p.Hkv * p.Sk * D * 4 <= (int64_t(64) << 20);
    const int qblk = nblk - 1 - (int)(by_row ? block / nbh : block % nblk);
    const int64_t bh = by_row ? block % nbh : block / nblk;
    const int h = (int)(bh % p.Hq), b = (int)(bh / p.Hq);
    const int kvh = h / p.group;
    const int q0 = qblk * kTiles * kTileQ;

    // key tiles each query tile may see: those below n_t[t]; in a windowed call the ones that `seen` names (n_t[0] is
    // the end of them)
    int n_t[2];
    const int64_t start = WINDOW ? window_start(p, b) : 0;
    WindowTiles seen = {0, 0, 0};
    int seen_lo = 0, seen_hi = 0;  // keys some row of the tile sees, apart from sinks below seen_lo
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int row_lo = q0 + t * kTileQ;
        if (row_lo >= p.Sq || t >= kTiles) {
            n_t[t] = 0;
        } else if (WINDOW) {
            const int row_hi = min(p.Sq, row_lo + kTileQ);
            seen = window_key_tiles(start, row_lo, row_hi, p.window, p.sinks, p.Sk);
            if (splits > 1) seen = window_piece(seen, piece, splits);
            seen_lo = window_span(start, row_lo, p.window, p.Sk).lo;
            seen_hi = window_span(start, row_hi - 1, p.window, p.Sk).hi;
            n_t[t] = seen.end;
        } else {
            const int row_hi = min(p.Sq, row_lo + kTileQ);
            const int k_hi = p.causal ? min(p.Sk, row_hi) : p.Sk;
            n_t[t] = (k_hi + kTileK - 1) / kTileK;
        }
    }
    const int n_max = max(n_t[0], n_t[1]);

    if (threadIdx.x == 0) {
        sh.abort_word = *reinterpret_cast<volatile int*>(p.abort_flag) != 0 ? 90 : 0;  // 90: an earlier CTA gave up
        mbar_init(&sh.q_full, 1);
        for (int i = 0; i < Cfg::kStages; ++i) {
            mbar_init(&sh.kv_full[i], 1);
            mbar_init(&sh.kv_empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sh.s_ready[t], 1);
            mbar_init(&sh.p_half[t][0], kTileQ);
            mbar_init(&sh.p_half[t][1], kTileQ);
            mbar_init(&sh.o_staged[t], kTileQ);
        }
        mbar_fence_init();
    }
    if (warp == kRoleWarp) {
        tmem_alloc(&sh.tmem_base, kTmemCols);
        tmem_relinquish();
    }
    if (p.has_mask)
        for (int j = threadIdx.x; j < n_max; j += kThreads) sh.tile_state[j] = (uint8_t)key_tile_state(p, b, h, q0, j);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_base;
    const uint8_t* states = sh.tile_state;
    const bool masked_call = p.has_mask != 0;
    auto state_of = [&](int j) -> int { return masked_call ? states[j] : 2; };
    // the CTA's walk over its key tiles; query tile t sees those below n_t[t]
    auto first_tile = [&]() -> int {
        if (WINDOW) return seen.begin();
        int j = 0;
        while (j < n_max && state_of(j) == 0) ++j;
        return j;
    };
    auto next_tile = [&](int j) -> int {
        if (WINDOW) return seen.next(j);
        ++j;
        while (j < n_max && state_of(j) == 0) ++j;
        return j;
    };
    volatile int* abort_word = &sh.abort_word;

    const bool dead = sh.abort_word != 0;  // set before the barrier above: skip straight to the tear-down
    if (dead) {
        if (WINDOW && splits > 1) {  // (a cluster's CTAs stay to its barriers: the others read this one's part)
            cluster_barrier();
            cluster_barrier();
        }
    } else if (warp >= kRoleWarp) {
      // registers move to the softmax warpgroups: (2 x 208 + 88) x 128 of 168 x 384, or (200 + 56) x 128 of 128 x 256
      if (kTiles == 2) reg_dealloc<88>();
      else reg_dealloc<56>();
      if (warp == kRoleWarp + 1) {
        // ------------------------------------------------------------ loader
        if (elect_one()) {
            tma_prefetch_desc(&maps.q);
            tma_prefetch_desc(&maps.k);
            tma_prefetch_desc(&maps.v);
            const int active = (n_t[0] > 0 ? 1 : 0) + (n_t[1] > 0 ? 1 : 0);
            mbar_expect_tx(&sh.q_full, active * Cfg::kTileBytes);
            for (int t = 0; t < kTiles; ++t)
                if (n_t[t] > 0)
                    for (int c = 0; c < Cfg::kChunks; ++c)
                        tma_load_4d(sQ + t * Cfg::kTileBytes + c * (kTileQ * 128), &maps.q, &sh.q_full, c * 64,
                                    q0 + t * kTileQ, h, b);
            int slot_use = 0;
            bool ok = true;
            for (int j = first_tile(); j < n_max && ok; j = next_tile(j)) {
                for (int which = 0; which < 2 && ok; ++which) {  // K tile, then V tile
                    const int slot = slot_use % Cfg::kStages, round = slot_use / Cfg::kStages;
                    if (round > 0) ok = mbar_wait(&sh.kv_empty[slot], (round - 1) & 1, abort_word, 10);
                    if (!ok) break;
                    mbar_expect_tx(&sh.kv_full[slot], Cfg::kTileBytes);
                    const CUtensorMap* map = which == 0 ? &maps.k : &maps.v;
                    for (int c = 0; c < Cfg::kChunks; ++c)
                        tma_load_4d(sKV + slot * Cfg::kTileBytes + c * (kTileK * 128), map, &sh.kv_full[slot], c * 64,
                                    j * kTileK, kvh, b);
                    ++slot_use;
                }
            }
        }
      } else if (warp == kRoleWarp) {
        // ------------------------------------------------------- MMA issuer
        if (elect_one()) {
            // a negative scale takes the maximum over -S: negate the A operand of the score product
            const uint32_t idesc_s =
                umma_idesc(kTileQ, kTileK, BF16 ? 1 : 0, false, false) | (p.scale < 0.f ? kUmmaNegateA : 0u);
            constexpr uint32_t idesc_o = umma_idesc(kTileQ, D, BF16 ? 1 : 0, false, true);
            const uint32_t q_addr = smem_u32(sQ), kv_addr = smem_u32(sKV);
            // Descriptors are built once; per instruction only the start-address field advances.
            const uint64_t q_desc = umma_desc_sw128(q_addr, 16, 1024), k_desc = umma_desc_sw128(kv_addr, 16, 1024);
            const uint64_t v_desc = umma_desc_sw128(kv_addr, kTileK * 128, 1024);
            auto issue_s = [&](int t, int slot) {
                const uint32_t a0 = t * Cfg::kTileBytes, b0 = slot * Cfg::kTileBytes;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = (kk / 4) * (kTileQ * 128) + (kk % 4) * 32;
                    umma_ss(tmem + t * 128, umma_desc_advance(q_desc, a0 + off), umma_desc_advance(k_desc, b0 + off),
                            idesc_s, kk > 0);
                }
            };
            // P*V over one half of the tile's keys (the half whose probabilities have been handed over: the first
            // half of the product runs while the softmax still forms the second half of the probabilities)
            auto issue_o = [&](int t, int slot, int half, bool accumulate) {
                const uint32_t b0 = slot * Cfg::kTileBytes;
#pragma unroll
                for (int kk = half * (kTileK / 32); kk < (half + 1) * (kTileK / 32); ++kk)
                    umma_ts(tmem + kColO + t * 128, tmem + t * 128 + kk * 8, umma_desc_advance(v_desc, b0 + kk * 2048),
                            idesc_o, accumulate || kk > 0);
            };
            // The same in a windowed call (of its one tile): steps of 16 keys that no row sees are left out.
            bool begun = false;  // the accumulator holds something
            auto issue_o_window = [&](int slot, int half, int j) {
                const uint32_t b0 = slot * Cfg::kTileBytes;
#pragma unroll
                for (int kk = half * (kTileK / 32); kk < (half + 1) * (kTileK / 32); ++kk) {
                    const int key = j * kTileK + kk * 16;
                    if (key >= seen_hi || (key + 16 <= seen_lo && key >= p.sinks)) continue;
                    umma_ts(tmem + kColO, tmem + kk * 8, umma_desc_advance(v_desc, b0 + kk * 2048), idesc_o, begun);
                    begun = true;
                }
            };
            // Values behind the last key that the CTA's rows see may never have been written (the free end of a
            // cache): their probabilities are zero, but zero times a NaN is not.  The rest of the 16-key step the
            // last key falls into is overwritten with zeros (at most 15 rows; rows beyond Sk arrive as zeros).
            auto clear_unseen = [&](int slot, int j) {
                const int r0 = seen_hi - j * kTileK;
                if (r0 <= 0 || r0 >= kTileK || seen_hi >= p.Sk || r0 % 16 == 0) return;
                uint8_t* tile = sKV + slot * Cfg::kTileBytes;
                for (int r = r0; r % 16 != 0; ++r)
                    for (int c = 0; c < Cfg::kChunks; ++c)
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            *reinterpret_cast<uint4*>(tile + c * (kTileK * 128) + r * 128 + x * 16) = make_uint4(0, 0, 0, 0);
                fence_async_smem();
            };
            bool ok = mbar_wait(&sh.q_full, 0, abort_word, 20);
            int slot_use = 0, iter[2] = {0, 0};
            PH_DECL;
            // first visible key tile
            int j = first_tile();
            if (ok && j < n_max) {
                const int slot = slot_use % Cfg::kStages;
                ok = mbar_wait(&sh.kv_full[slot], (slot_use / Cfg::kStages) & 1, abort_word, 21);
                if (ok) {
                    tc_fence_after();
                    for (int t = 0; t < kTiles; ++t)
                        if (j < n_t[t]) {
                            issue_s(t, slot);
                            umma_commit(&sh.s_ready[t]);
                        }
                    umma_commit(&sh.kv_empty[slot]);
                    ++slot_use;
                }
            }
            while (ok && j < n_max) {
                const int jn = next_tile(j);
                const int v_slot = slot_use % Cfg::kStages, v_par = (slot_use / Cfg::kStages) & 1;
                ++slot_use;
                int k_slot = -1, k_par = 0;
                if (jn < n_max) {
                    k_slot = slot_use % Cfg::kStages;
                    k_par = (slot_use / Cfg::kStages) & 1;
                    ++slot_use;
                }
                PH(5);
                ok = mbar_wait(&sh.kv_full[v_slot], v_par, abort_word, 22);
                PH(0);
                bool k_waited = false;
                if (WINDOW && ok) clear_unseen(v_slot, j);
                for (int t = 0; t < kTiles && ok; ++t) {
                    if (j >= n_t[t]) continue;
                    ok = mbar_wait(&sh.p_half[t][0], iter[t] & 1, abort_word, 23 + t);
                    if (!ok) break;
                    PH(1);
                    tc_fence_after();
                    if (WINDOW) issue_o_window(v_slot, 0, j);
                    else issue_o(t, v_slot, 0, iter[t] > 0);
                    PH(2);
                    ok = mbar_wait(&sh.p_half[t][1], iter[t] & 1, abort_word, 26 + t);
                    if (!ok) break;
                    PH(1);
                    tc_fence_after();
                    if (WINDOW) issue_o_window(v_slot, 1, j);
                    else issue_o(t, v_slot, 1, true);
                    PH(2);
                    ++iter[t];
                    if (jn < n_t[t]) {
                        if (!k_waited) {
                            ok = mbar_wait(&sh.kv_full[k_slot], k_par, abort_word, 25);
                            if (!ok) break;
                            tc_fence_after();
                            k_waited = true;
                        }
                        PH(3);
                        issue_s(t, k_slot);
                    }
                    umma_commit(&sh.s_ready[t]);  // one per score tile, and one behind the last product
                    PH(4);
                }
                if (!ok) break;
                umma_commit(&sh.kv_empty[v_slot]);
                if (k_slot >= 0) umma_commit(&sh.kv_empty[k_slot]);
                j = jn;
            }
            PH_FLUSH(2);
        }
      }
      if (WINDOW && splits > 1) {
          __syncwarp();
          cluster_barrier();
          cluster_barrier();
      }
    } else {
        if (kTiles == 2) reg_alloc<208>();
        else reg_alloc<200>();
        // ---------------------------------------------------------- softmax
        const int t = kTiles == 1 ? 0 : warp >> 2;
        const int row_in_tile = (warp & 3) * 32 + lane;
        const int row = q0 + t * kTileQ + row_in_tile;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t s_addr = lane_base + t * 128, o_addr = lane_base + kColO + t * 128;
        const float c2 = fabsf(p.scale) * kLog2e;
        const uint64_t c2_pair = f2_pack(c2, c2);
        // this row's line of the mask (every row shares one line when the mask is broadcast over queries)
        const uint8_t* kmask = p.has_mask ? p.mask + (int64_t)b * p.ms[0] + (int64_t)h * p.ms[1] +
                                                (int64_t)min(row, p.Sq - 1) * p.ms[2]
                                          : nullptr;
        float m_used = -INFINITY, m_true = -INFINITY, l = 0.f;
        int iter = 0;
        bool ok = true;
        PH_DECL;
        // a windowed call: this row's window
        const WindowSpan span = WINDOW ? window_span(start, min(row, p.Sq - 1), p.window, p.Sk) : WindowSpan{0, 0};
        const int n_mine = t == 0 ? n_t[0] : n_t[1];
        for (int j = WINDOW ? seen.begin() : 0; j < n_mine && ok; j = WINDOW ? seen.next(j) : j + 1) {
            const int state = state_of(j);
            if (state == 0) continue;
            PH(5);
            ok = mbar_wait(&sh.s_ready[t], iter & 1, abort_word, 30 + t);
            if (!ok) break;
            PH(0);
            tc_fence_after();
            // scores arrive already multiplied by sign(scale) (negated A operand for negative scales)
            float s[kTileK];
#pragma unroll
            for (int c = 0; c < kTileK; c += 32) {
                uint32_t r[32];
                tmem_ld32(s_addr + c, r);
#pragma unroll
                for (int i = 0; i < 32; ++i) s[c + i] = __uint_as_float(r[i]);
            }
            tmem_wait_ld();
            tmem_loaded(s);
            PH(1);
            const int key0 = j * kTileK;
            // leading columns of this tile that pass the sequence-end and causal bounds for this row
            int lim = p.Sk - key0;
            if (WINDOW) lim = span.hi - key0;
            else if (p.causal) lim = min(lim, row - key0 + 1);
            if (lim < kTileK) {
#pragma unroll
                for (int c = 0; c < kTileK; ++c) s[c] = c < lim ? s[c] : -INFINITY;
            }
            if (WINDOW) {  // columns before the window, apart from the sinks
                const int lo = span.lo - key0, sink = p.sinks - key0;
                if (lo > 0 && lo > sink) {
#pragma unroll
                    for (int c = 0; c < kTileK; ++c) s[c] = c < lo && c >= sink ? -INFINITY : s[c];
                }
            }
            if (state == 1) {
#pragma unroll
                for (int c = 0; c < kTileK; ++c) {
                    const int key = min(key0 + c, p.Sk - 1);
                    s[c] = kmask[(int64_t)key * p.ms[3]] != 0 ? s[c] : -INFINITY;
                }
            }
            // four independent chains of three-input maxima
            float mx0 = max3(s[0], s[1], s[2]), mx1 = max3(s[3], s[4], s[5]);
            float mx2 = max3(s[6], s[7], s[8]), mx3 = max3(s[9], s[10], s[11]);
#pragma unroll
            for (int c = 12; c < kTileK - 4; c += 8) {
                mx0 = max3(mx0, s[c], s[c + 1]);
                mx1 = max3(mx1, s[c + 2], s[c + 3]);
                mx2 = max3(mx2, s[c + 4], s[c + 5]);
                mx3 = max3(mx3, s[c + 6], s[c + 7]);
            }
            mx0 = max3(mx0, s[kTileK - 4], s[kTileK - 3]);
            mx1 = max3(mx1, s[kTileK - 2], s[kTileK - 1]);
            const float mx = fmaxf(max3(mx0, mx1, mx2), mx3);
            m_true = fmaxf(m_true, mx);
            const bool rebase = mx > m_used && (m_used == -INFINITY || (mx - m_used) * c2 > rebase_limit<BF16>());
            float alpha = 1.f;
            if (rebase) {
                alpha = (m_used == -INFINITY) ? 0.f : ex2((m_used - mx) * c2);
                l *= alpha;
                m_used = mx;
            }
            if (iter > 0 && __any_sync(0xffffffffu, rebase)) {
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t r[32];
                    tmem_ld32(o_addr + c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                    tmem_st32(o_addr + c, r);
                }
            }
            PH(2);
            const float m_safe = (m_used == -INFINITY) ? 0.f : m_used;
            const uint64_t m_pair = f2_pack(m_safe, m_safe);
            uint64_t sum_a = f2_pack(0.f, 0.f), sum_b = sum_a;
#pragma unroll
            for (int c = 0; c < kTileK; c += 32) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    // (s - m) first, then the multiplication by |scale|*log2e, two lanes per instruction
                    float pa, pb, pc, pd;
                    f2_unpack(f2_mul(f2_sub(f2_pack(s[c + 2 * i], s[c + 2 * i + 1]), m_pair), c2_pair), pa, pb);
                    f2_unpack(f2_mul(f2_sub(f2_pack(s[c + 2 * i + 2], s[c + 2 * i + 3]), m_pair), c2_pair), pc, pd);
                    pa = ex2(pa);
                    pb = ex2(pb);
                    pc = ex2(pc);
                    pd = ex2(pd);
                    sum_a = f2_add(sum_a, f2_pack(pa, pb));
                    sum_b = f2_add(sum_b, f2_pack(pc, pd));
                    w[i] = pack2<BF16>(pa, pb);
                    w[i + 1] = pack2<BF16>(pc, pd);
                }
                tmem_st16(s_addr + c / 2, w);
                if (c == kTileK / 2 - 32) {  // the first half of the keys is done: hand it over
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&sh.p_half[t][0]);
                }
            }
            {
                float x0, x1, x2, x3;
                f2_unpack(sum_a, x0, x1);
                f2_unpack(sum_b, x2, x3);
                l += (x0 + x1) + (x2 + x3);
            }
            PH(3);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&sh.p_half[t][1]);
            PH(4);
            ++iter;
        }
        if ((threadIdx.x & 127) == 0) PH_FLUSH(t);
        // epilogue: wait for the last product, normalise, store
        if (WINDOW && splits > 1) {
            // The pieces' accumulators and (reference, sum, maximum), in place of the ring and the query tile, are merged
            // in their order over distributed shared memory; each CTA writes its share of the rows.
            float4* part_o = reinterpret_cast<float4*>(sKV);  // [128 rows][D / 4], chunks exchanged by the row
            float4* part_ml = reinterpret_cast<float4*>(sQ);
            static_assert(!WINDOW || kTileQ * D * 4 <= Cfg::kStages * Cfg::kTileBytes, "a tile's accumulator fits the ring");
            constexpr int kChunks4 = D / 4;
            if (iter > 0 && ok) ok = mbar_wait(&sh.s_ready[t], iter & 1, abort_word, 32 + t);
            if (!ok) iter = 0;
            if (__any_sync(0xffffffffu, iter > 0)) {  // (a piece's tiles are the same for all rows)
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t r[32];
                    tmem_ld32(o_addr + c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        part_o[row_in_tile * kChunks4 + (((c + i) / 4) ^ (row_in_tile & (kChunks4 - 1)))] =
                            make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]), __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
                }
            }
            part_ml[row_in_tile] = make_float4(iter > 0 ? m_used : -INFINITY, iter > 0 ? l : 0.f, iter > 0 ? m_true : -INFINITY, 0.f);
            cluster_barrier();
            auto merge = [&](auto pieces_) {
                constexpr int S = decltype(pieces_)::value, kRows = kTileQ / S, kWarpRows = kRows / 4, kAtOnce = 32 / kChunks4;
                using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
                for (int r4 = 0; r4 < kWarpRows; r4 += 4) {
                    const int r0 = piece * kRows + (warp & 3) * kWarpRows + r4;
                    // the weights of four rows' pieces: lane 8 row + piece
                    const int from = lane & 7, r = r0 + (lane >> 3);
                    float4 ml = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
                    if (from < S) ml = cluster_load4(cluster_address(part_ml + r, from));
                    float m = ml.x, top = ml.z;
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) {
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    }
                    // (a piece without a visible key has no accumulator either: weight zero, and nothing is loaded)
                    float weight = ml.x == -INFINITY ? 0.f : ex2((ml.x - m) * c2), sum = ml.y * weight;
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    // (a sum that is not a number stays one: every weight of the row becomes NaN, and so does its output, as
                    // where one CTA has all the keys)
                    weight *= sum == 0.f ? 0.f : 1.f / sum;
                    if (from == 0 && q0 + r < p.Sq && p.maximum) {
                        const int64_t si = ((int64_t)b * p.Hq + h) * p.Sq + q0 + r;
                        p.maximum[si] = top;
                        p.logsum[si] = sum > 0.f ? log2f(sum) + (m - top) * c2 : 0.f;
                    }
                    const int c = lane & (kChunks4 - 1);
#pragma unroll(8 / S > 4 / kAtOnce ? 4 / kAtOnce : 8 / S)
                    for (int i = 0; i < 4; i += kAtOnce) {
                        const int mine = i + lane / kChunks4, row_at = r0 + mine;
                        float4 x[S], acc = make_float4(0.f, 0.f, 0.f, 0.f);
                        float w[S];
#pragma unroll
                        for (int n = 0; n < S; ++n) {
                            w[n] = __shfl_sync(0xffffffffu, weight, 8 * mine + n);
                            x[n] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (w[n] != 0.f)
                                x[n] = cluster_load4(cluster_address(part_o + row_at * kChunks4 + (c ^ (row_at & (kChunks4 - 1))), n));
                        }
#pragma unroll
                        for (int n = 0; n < S; ++n) {
                            acc.x = fmaf(x[n].x, w[n], acc.x), acc.y = fmaf(x[n].y, w[n], acc.y);
                            acc.z = fmaf(x[n].z, w[n], acc.z), acc.w = fmaf(x[n].w, w[n], acc.w);
                        }
                        if (q0 + row_at < p.Sq && c * 4 < p.D) {
                            T* to = reinterpret_cast<T*>(p.out) + (int64_t)b * p.os[0] + (int64_t)h * p.os[1] +
                                    (int64_t)(q0 + row_at) * p.os[2] + c * 4;
                            *reinterpret_cast<uint2*>(to) = make_uint2(pack2<BF16>(acc.x, acc.y), pack2<BF16>(acc.z, acc.w));
                        }
                    }
                }
            };
            if (splits == 2) merge(std::integral_constant<int, 2>{});
            else if (splits == 4) merge(std::integral_constant<int, 4>{});
            else merge(std::integral_constant<int, 8>{});
            cluster_barrier();  // nobody leaves while its part is read
            iter = -1;          // (nothing is left to write)
        }
        if (ok && iter == 0 && row < p.Sq && (WINDOW || n_t[t] > 0) && !p.running) {
            // every key tile of this row is hidden: zero output, empty statistics
            using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
            T* orow = reinterpret_cast<T*>(p.out) + (int64_t)b * p.os[0] + (int64_t)h * p.os[1] + (int64_t)row * p.os[2];
            const int64_t si = ((int64_t)b * p.Hq + h) * p.Sq + row;
            for (int d = 0; d < p.D; d += 8) *reinterpret_cast<uint4*>(orow + d) = make_uint4(0, 0, 0, 0);
            if (p.maximum) {  // no statistics are kept for a forward pass without gradients
                p.maximum[si] = -INFINITY;
                p.logsum[si] = 0.f;
            }
        }
        if (iter > 0 && p.running) {
            // Block of a longer key sequence: fold (accumulator, maximum, sum) into the caller's running FP32 state
            // with the (maximum, sum) merge of the reference's split forward (split_forward.py:219-245); nothing is
            // rounded to the 16-bit type and nothing is divided here.
            if (ok) ok = mbar_wait(&sh.s_ready[t], iter & 1, abort_word, 32 + t);
            if (ok) {
                // (every lane runs the tensor-memory loads, which are warp-wide; rows beyond the sequence end
                // only skip the global accesses)
                tc_fence_after();
                const bool live = row < p.Sq;
                const int64_t si = (int64_t)b * p.ss[0] + (int64_t)h * p.ss[1] + (live ? row : 0);
                const float m_old = live ? p.maximum[si] : -INFINITY, l_old = live ? p.run_sum[si] : 0.f;
                const float m_new = fmaxf(m_old, m_true);
                const float w_old = m_old == -INFINITY ? 0.f : ex2((m_old - m_new) * c2);
                const float w_blk = m_used == -INFINITY ? 0.f : ex2((m_used - m_new) * c2);
                float* arow = reinterpret_cast<float*>(p.out) + (int64_t)b * p.os[0] + (int64_t)h * p.os[1] +
                              (int64_t)row * p.os[2];
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t r[32];
                    tmem_ld32(o_addr + c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        if (live && c + i < p.D) {
                            float4 a = *reinterpret_cast<float4*>(arow + c + i);
                            a.x = a.x * w_old + __uint_as_float(r[i]) * w_blk;
                            a.y = a.y * w_old + __uint_as_float(r[i + 1]) * w_blk;
                            a.z = a.z * w_old + __uint_as_float(r[i + 2]) * w_blk;
                            a.w = a.w * w_old + __uint_as_float(r[i + 3]) * w_blk;
                            *reinterpret_cast<float4*>(arow + c + i) = a;
                        }
                    }
                }
                if (live) {
                    p.maximum[si] = m_new;
                    p.run_sum[si] = l_old * w_old + l * w_blk;
                }
            }
        } else if (iter > 0) {
            if (ok) ok = mbar_wait(&sh.s_ready[t], iter & 1, abort_word, 32 + t);
            if (ok) {
                tc_fence_after();
                const float den = l > 0.f ? l : 1.f;
                const float inv_den = 1.f / den;  // one division per row; the elements are multiplied
                // The normalised tile goes through this tile's (now dead) Q buffer in the swizzled box layout and
                // leaves as tiled stores: whole 128-byte lines instead of 16 bytes per row and instruction.
                uint8_t* stage = sQ + t * Cfg::kTileBytes;
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t r[32];
                    tmem_ld32(o_addr + c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint4 w;
                        w.x = pack2<BF16>(__uint_as_float(r[i]) * inv_den, __uint_as_float(r[i + 1]) * inv_den);
                        w.y = pack2<BF16>(__uint_as_float(r[i + 2]) * inv_den, __uint_as_float(r[i + 3]) * inv_den);
                        w.z = pack2<BF16>(__uint_as_float(r[i + 4]) * inv_den, __uint_as_float(r[i + 5]) * inv_den);
                        w.w = pack2<BF16>(__uint_as_float(r[i + 6]) * inv_den, __uint_as_float(r[i + 7]) * inv_den);
                        const int chunk = (c + i) >> 3;  // 16-byte chunk of the row: box chunk / 8, position chunk % 8
                        *reinterpret_cast<uint4*>(stage + (chunk >> 3) * (kTileQ * 128) + sw128_chunk(row_in_tile, chunk & 7)) = w;
                    }
                }
                fence_async_smem();
                mbar_arrive(&sh.o_staged[t]);
                if (row_in_tile == 0 && mbar_wait(&sh.o_staged[t], 0, abort_word, 34 + t)) {
                    for (int c = 0; c < Cfg::kChunks; ++c)
                        tma_store_4d(&maps.o, stage + c * (kTileQ * 128), c * 64, q0 + t * kTileQ, h, b);
                    tma_store_commit();
                    tma_store_wait_read();
                }
                if (row < p.Sq && p.maximum) {
                    const int64_t si = ((int64_t)b * p.Hq + h) * p.Sq + row;
                    p.maximum[si] = m_true;
                    p.logsum[si] = l > 0.f ? log2f(l) + (m_used - m_true) * c2 : 0.f;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sh.abort_word != 0 && sh.abort_word != 90) {  // 90 = skipped: already reported
        *p.status = 1000 + sh.abort_word;
        *reinterpret_cast<volatile int*>(p.abort_flag) = 1;  // the remaining CTAs of this and later launches skip their work
    }
    if (warp == kRoleWarp) tmem_dealloc(tmem, kTmemCols);
}

std::atomic<int> g_configured{0};

template <int D, bool BF16>
cudaError_t launch_t(const AttnParams& p, cudaStream_t st) {
    const int tiles = p.window > 0 ? 1 : 2;
    const int smem_bytes = tiles == 1 ? FwdCfg<D, 1>::kSmemBytes : FwdCfg<D, 2>::kSmemBytes;
    // The shared-memory opt-in is per device; it is cheap, so it is simply repeated per call.
    auto kernel = p.window > 0 ? pipeline_forward<D, BF16, false, true>
                  : p.has_mask ? pipeline_forward<D, BF16, true, false>
                               : pipeline_forward<D, BF16, false, false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
    if (e != cudaSuccess) return e;
    constexpr int variant = (D == 128 ? 0 : 2) + (BF16 ? 0 : 1);  // D = channels the kernel runs with (p.D rounded up)
    const int bit = 1 << variant;
    if (!(g_configured.load() & bit)) g_configured |= bit;
    FwdMaps maps;
    const CUtensorMapDataType dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (!encode_bhsd_map(&maps.q, p.q, dt, p.D, p.Sq, p.Hq, p.B, p.qs, 64, kTileQ)) return cudaErrorInvalidValue;
    if (!encode_bhsd_map(&maps.k, p.k, dt, p.D, p.Sk, p.Hkv, p.B, p.ks, 64, kTileK)) return cudaErrorInvalidValue;
    if (!encode_bhsd_map(&maps.v, p.v, dt, p.D, p.Sk, p.Hkv, p.B, p.vs, 64, kTileK)) return cudaErrorInvalidValue;
    if (p.running)
        maps.o = maps.q;  // not used: the running state is written with plain stores
    else if (!encode_bhsd_map(&maps.o, p.out, dt, p.D, p.Sq, p.Hq, p.B, p.os, 64, kTileQ))
        return cudaErrorInvalidValue;
    const int64_t grid = (int64_t)((p.Sq + tiles * kTileQ - 1) / (tiles * kTileQ)) * p.B * p.Hq;
    const int splits = p.window > 0 ? window_key_splits(p) : 1;
    if (splits > 1) {
        AttnParams split = p;
        split.key_splits = splits;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)(grid * splits));
        config.blockDim = dim3(threads_of(tiles));
        config.dynamicSmemBytes = smem_bytes;
        config.stream = st;
        cudaLaunchAttribute together[1];
        together[0].id = cudaLaunchAttributeClusterDimension;
        together[0].val.clusterDim.x = (unsigned)splits;
        together[0].val.clusterDim.y = together[0].val.clusterDim.z = 1;
        config.attrs = together;
        config.numAttrs = 1;
        return cudaLaunchKernelEx(&config, kernel, maps, split);
    }
    kernel<<<(unsigned)grid, threads_of(tiles), smem_bytes, st>>>(maps, p);
    return cudaGetLastError();
}

}  // namespace

bool pipeline_forward_supported(const AttnParams& p, bool bf16) {
    (void)bf16;
    if (p.D < 8 || p.D > 128 || p.D % 8 != 0) return false;  // rows of whole 16-byte pieces
    if (p.nd != 0) return false;
    if (p.scale == 0.f || p.Sk < 2) return false;  // hidden scores are -inf; -inf * 0 is not representable in the fast path
    if (p.has_mask && (p.Sk + kTileK - 1) / kTileK > kMaxKeyTiles) return false;
    if (!tma_compatible(p.q, p.qs, p.B, p.Hq, p.Sq) || !tma_compatible(p.k, p.ks, p.B, p.Hkv, p.Sk) ||
        !tma_compatible(p.v, p.vs, p.B, p.Hkv, p.Sk))
        return false;
    if (p.running) {  // FP32 rows read and written as 16-byte vectors
        if (p.os[3] != 1 || reinterpret_cast<uintptr_t>(p.out) % 16 != 0 || p.os[0] % 4 || p.os[1] % 4 || p.os[2] % 4)
            return false;
    } else if (!tma_compatible(p.out, p.os, p.B, p.Hq, p.Sq)) {
        return false;  // 16-byte vector stores per row
    }
    return true;
}

cudaError_t launch_pipeline_forward(const AttnParams& p, bool bf16, cudaStream_t st) {
    if (p.D > 64) return bf16 ? launch_t<128, true>(p, st) : launch_t<128, false>(p, st);
    return bf16 ? launch_t<64, true>(p, st) : launch_t<64, false>(p, st);
}

KFA_PHASE_EXPORT(kfa_debug_phases_fwd)

int pipeline_forward_variants() { return __builtin_popcount(g_configured.load()); }
void pipeline_forward_forget() { g_configured = 0; }

}  // namespace kfa
