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

bool window_decode_shape(const AttnParams& p) {
    if ((p.D != 64 && p.D != 128) || (int64_t)p.Sq * p.group > 16) return false;
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
