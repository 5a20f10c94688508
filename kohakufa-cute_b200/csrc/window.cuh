// Visibility of the sliding window with sinks, shared by every kernel that serves it.
//
// Query row r of batch b stands at key position pos = start_b + r and sees key c iff
//     0 <= c < Sk,  c <= pos,  and  (c > pos - window  or  c < sinks),
// i.e. the keys [lo, hi) of its window and the first `sinks` keys below hi.  Positions are formed in 64 bits (a start
// may be any 32-bit value, a window as long as the caller likes); the bounds then fit 32 bits because they are clipped
// to [0, Sk].  A row before the first key (pos < 0), or far behind the last one without sinks, sees nothing.
#pragma once
#include "kfa_common.cuh"

namespace kfa {

__device__ __forceinline__ int64_t window_start(const AttnParams& p, int b) {
    return p.starts ? (int64_t)p.starts[b] : p.start;
}

struct WindowSpan {
    int lo, hi;  // keys of the row's window: [lo, hi), lo <= hi
};

__host__ __device__ __forceinline__ WindowSpan window_span(int64_t start, int row, int64_t window, int Sk) {
    const int64_t end = start + row + 1, begin = end - window;
    WindowSpan s;
    s.hi = (int)(end < 0 ? 0 : (end > Sk ? Sk : end));
    s.lo = (int)(begin < 0 ? 0 : (begin > s.hi ? s.hi : begin));
    return s;
}

__host__ __device__ __forceinline__ bool window_sees(const WindowSpan& s, int sinks, int key) {
    return key < s.hi && (key >= s.lo || key < sinks);
}

// The 128-key tiles that the rows [row0, row1) of one sequence can see: [0, sink_end) and [first, end),
// sink_end <= first <= end (nothing visible: all three zero).
struct WindowTiles {
    int sink_end, first, end;
    __host__ __device__ __forceinline__ int begin() const { return sink_end > 0 ? 0 : first; }
    __host__ __device__ __forceinline__ int next(int j) const {
        ++j;
        return j >= sink_end && j < first ? first : j;
    }
    __host__ __device__ __forceinline__ bool has(int j) const { return j < sink_end || (j >= first && j < end); }
};

__host__ __device__ __forceinline__ WindowTiles window_key_tiles(int64_t start, int row0, int row1, int64_t window,
                                                                 int sinks, int Sk) {
    const int lo = window_span(start, row0, window, Sk).lo, hi = window_span(start, row1 - 1, window, Sk).hi;
    const int seen_sinks = sinks < hi ? sinks : hi;
    WindowTiles t;
    t.sink_end = (seen_sinks + 127) >> 7;
    t.first = t.end = t.sink_end;
    if (lo < hi) {
        if ((lo >> 7) > t.first) t.first = lo >> 7;
        if (((hi + 127) >> 7) > t.first) t.end = (hi + 127) >> 7;
        else t.end = t.first;
    }
    return t;
}

// Piece `piece` of `pieces` of these tiles, in equal parts; the sinks' tiles all belong to the first.
__host__ __device__ __forceinline__ WindowTiles window_piece(const WindowTiles& all, int piece, int pieces) {
    const int window = all.end - all.first, total = all.sink_end + window;
    auto before = [&](int i) {  // window tiles of the pieces before i
        const int n = (int)((int64_t)total * i / pieces) - all.sink_end;
        return i == 0 || n < 0 ? 0 : n;
    };
    WindowTiles t;
    t.sink_end = piece == 0 ? all.sink_end : 0;
    t.first = all.first + before(piece);
    t.end = all.first + before(piece + 1);
    if (t.first == t.end) t.first = t.end = t.sink_end;
    return t;
}

// The 128-row query tiles [first, end) that hold a row which sees one of the keys [key0, key1), key1 <= Sk.  A tile in
// between may hold no such row when the range of keys has sinks at its head; its scores are hidden one by one then.
struct WindowRange {
    int first, end;
};

__host__ __device__ __forceinline__ WindowRange window_query_tiles(int64_t start, int key0, int key1, int64_t window,
                                                                   int sinks, int Sq) {
    int64_t r0 = key0 - start, r1 = key0 < sinks ? Sq : key1 - 1 + window - start;
    r0 = r0 < 0 ? 0 : r0;
    r1 = r1 > Sq ? Sq : r1;
    if (r0 >= r1) return WindowRange{0, 0};
    return WindowRange{(int)(r0 >> 7), (int)((r1 + 127) >> 7)};
}

// CTAs per query tile of the tensor-memory forward (1: no cluster).  Where the tiles leave most SMs empty, a cluster of
// two, four or eight shares a tile's keys: at most one CTA per SM, or two (nine tenths of the places, which clusters
// have to find) where that makes four and more.  Times in a graph, D 128, by batch, heads, rows, window, one CTA -> a
// cluster: 1 8 512 1024: 22.9 -> 14.6 us (four); 8 8 40 2048: 36.4 -> 23.4 (four); 1 64 64 4096: 62.7 -> 31.6 (four);
// left alone: 16 8 33 1000: 24.2 -> 25.7 (two, two per SM); 2 8 1000 300, four key tiles: 17.7 -> 21.1 (two).
inline int window_key_splits(const AttnParams& p) {
    const int64_t tiles = (int64_t)p.B * p.Hq * ((p.Sq + 127) / 128);
    const int64_t keys = (p.window < p.Sk ? p.window : p.Sk) / 128 + 1 + (p.sinks + 127) / 128;
    int splits = 1;
    for (int more = 2; more <= 8; more *= 2)
        if (keys >= (more == 8 ? 20 : more + 6) && (tiles * more <= 148 || (more >= 4 && tiles * more <= 266))) splits = more;
    return splits;
}

}  // namespace kfa
