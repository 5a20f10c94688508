// Sliding-window attention of a few query rows to a 16-bit key/value cache: decode_rows.cuh on 16-bit rows.
#include "decode_rows.cuh"
#include "launchers.h"

namespace kfa {
namespace {

CacheAttentionCall call_of(const AttnParams& p) {
    CacheAttentionCall c = {};
    c.q = p.q;
    c.out = p.out;
    for (int i = 0; i < 3; ++i) {
        c.qs[i] = p.qs[i];
        c.os[i] = p.os[i];
    }
    c.starts = p.starts;
    c.start = p.start;
    c.window = p.window;
    c.sinks = p.sinks;
    c.B = p.B;
    c.Hq = p.Hq;
    c.Hkv = p.Hkv;
    c.Sq = p.Sq;
    c.Sk = p.Sk;
    c.D = p.D;
    c.group = p.group;
    c.scale = p.scale;
    c.status = p.status;
    c.abort_flag = p.abort_flag;
    return c;
}

}  // namespace

// Up to 16 query rows per K/V head, a unit reads its keys once and nothing beats that.  More rows come in pieces of 16,
// each of which reads the window of all rows; the tensor-memory forward has a CTA per head and 128 rows, which reads that
// of its own.  About 155 units (D 128; 220 at D 64) cost what a wave of 296 such CTAs does for the same keys, also where
// the wave is not full, since units spread over idle SMs and a CTA does not; about 65 (95) where clusters share a tile's
// keys there.  Times in a graph, tensor-memory forward -> this, D 128, by batch, query / K/V heads, rows, window:
// 16 64/8 4 4096: 299 -> 83 us; 48 64/8 8 1024: 282 -> 165; 8 16/8 16 2048: 36 -> 29; 1 8/1 33 1024: 15 -> 12; kept
// there: 1 64/8 33 4096: 32 -> 50; 16 32/8 16 1000: 52 -> 59.  D 64: 16 64/8 4 1024: 88 -> 23.
bool window_decode_shape(const AttnParams& p) {
    if (p.D != 64 && p.D != 128) return false;
    const int64_t rows = (int64_t)p.Sq * p.group;
    if (rows > 16) {
        const int64_t seen = p.window < p.Sk ? p.window : p.Sk;
        const double units = (double)p.B * p.Hkv * (double)((rows + 15) / 16);
        const double waves = (double)(((int64_t)p.B * p.Hq * ((p.Sq + 127) / 128) + 295) / 296);
        const double wave = window_key_splits(p) > 1 ? (p.D == 128 ? 65. : 95.) : (p.D == 128 ? 155. : 220.);
        if (units * (double)(seen + p.Sq) > wave * waves * (double)(seen + (p.Sq < 128 ? p.Sq : 128))) return false;
    }
    const CacheAttentionCall c = call_of(p);
    return p.D == 128 ? rows::countable<128, false>(c) : rows::countable<64, false>(c);
}

size_t window_decode_workspace_bytes(const AttnParams& p) {
    const CacheAttentionCall c = call_of(p);
    return p.D == 128 ? rows::workspace_bytes<128, false>(c) : rows::workspace_bytes<64, false>(c);
}

cudaError_t launch_window_decode(const AttnParams& p, bool bf16, void* workspace, int* launches, cudaStream_t st) {
    RowsCall r = {};
    r.c = call_of(p);
    r.kv[0] = p.k;
    r.kv[1] = p.v;
    for (int i = 0; i < 3; ++i) {
        r.kvs[0][i] = p.ks[i];
        r.kvs[1][i] = p.vs[i];
    }
    const cudaError_t e =
        bf16 ? rows::dispatch<__nv_bfloat16, false>(r, workspace, st) : rows::dispatch<__half, false>(r, workspace, st);
    *launches = r.cluster ? 1 : 2;
    return e;
}

}  // namespace kfa
