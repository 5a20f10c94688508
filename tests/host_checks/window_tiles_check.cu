// Host check of the sliding-window geometry: the tile ranges the tensor-memory kernels walk hold every visible
// (query, key) pair, hold no tile that nobody needs (query side: between the sinks and the window), and the spans of a
// row equal the definition.  Prints the number of pairs compared; exits non-zero on the first difference.
#include "../../kohakufa-cute_b200/csrc/window.cuh"

#include <cstdio>
#include <vector>

static bool defined(int64_t start, int row, int key, int64_t window, int sinks, int Sk) {
    const int64_t pos = start + row;
    return key >= 0 && key < Sk && key <= pos && (key > pos - window || key < sinks);
}

int main() {
    const int sizes[] = {1, 2, 100, 128, 129, 300, 513, 1000};
    const int64_t starts[] = {-2147483648LL, -700, -129, -1, 0, 1, 127, 128, 400, 900, 1500, 2147483647LL};
    const int64_t windows[] = {1, 2, 100, 128, 129, 333, 2000, 2147483647LL, int64_t(1) << 40};
    const int sink_counts[] = {0, 1, 4, 127, 128, 130, 600};
    long long pairs = 0;
    for (int Sq : sizes)
        for (int Sk : sizes)
            for (int64_t start : starts)
                for (int64_t window : windows)
                    for (int asked : sink_counts) {
                        const int sinks = asked < Sk ? asked : Sk;
                        std::vector<kfa::WindowTiles> keys;
                        for (int r0 = 0; r0 < Sq; r0 += 128)
                            keys.push_back(kfa::window_key_tiles(start, r0, r0 + 128 < Sq ? r0 + 128 : Sq, window, sinks, Sk));
                        std::vector<kfa::WindowRange> queries;
                        for (int k0 = 0; k0 < Sk; k0 += 128)
                            queries.push_back(kfa::window_query_tiles(start, k0, k0 + 128 < Sk ? k0 + 128 : Sk, window, sinks, Sq));
                        const int nq = (int)keys.size(), nk = (int)queries.size();
                        std::vector<char> needed(nq * nk, 0);
                        for (int r = 0; r < Sq; ++r) {
                            const kfa::WindowSpan span = kfa::window_span(start, r, window, Sk);
                            for (int c = 0; c < Sk; ++c) {
                                const bool seen = defined(start, r, c, window, sinks, Sk);
                                if (seen != kfa::window_sees(span, sinks, c)) {
                                    std::printf("span: Sq %d Sk %d start %lld window %lld sinks %d row %d key %d\n", Sq, Sk,
                                                (long long)start, (long long)window, sinks, r, c);
                                    return 1;
                                }
                                if (seen) needed[(r >> 7) * nk + (c >> 7)] = 1;
                                ++pairs;
                            }
                        }
                        for (int tq = 0; tq < nq; ++tq) {
                            // the walk visits the tiles that has() names, in ascending order
                            std::vector<char> walked(nk + 1, 0);
                            int last = -1;
                            for (int j = keys[tq].begin(); j < keys[tq].end; j = keys[tq].next(j)) {
                                if (j <= last || j >= nk) return 2;
                                walked[j] = 1;
                                last = j;
                            }
                            for (int pieces : {2, 4, 8}) {  // one after the other, they walk the same tiles
                                int j = keys[tq].begin();
                                for (int piece = 0; piece < pieces; ++piece) {
                                    const kfa::WindowTiles part = kfa::window_piece(keys[tq], piece, pieces);
                                    for (int i = part.begin(); i < part.end; i = part.next(i)) {
                                        if (i != j || !part.has(i)) return 7;
                                        j = keys[tq].next(j);
                                    }
                                }
                                if (j < keys[tq].end) return 8;
                            }
                            for (int tk = 0; tk < nk; ++tk) {
                                if (walked[tk] != keys[tq].has(tk) || walked[tk] < needed[tq * nk + tk]) {
                                    std::printf("key tiles: Sq %d Sk %d start %lld window %lld sinks %d tile %d %d\n", Sq, Sk,
                                                (long long)start, (long long)window, sinks, tq, tk);
                                    return 3;
                                }
                                if (walked[tk] && !needed[tq * nk + tk]) return 4;
                                if (needed[tq * nk + tk] && (tq < queries[tk].first || tq >= queries[tk].end)) {
                                    std::printf("query tiles: Sq %d Sk %d start %lld window %lld sinks %d tile %d %d\n", Sq, Sk,
                                                (long long)start, (long long)window, sinks, tq, tk);
                                    return 5;
                                }
                            }
                        }
                        for (int tk = 0; tk < nk; ++tk)
                            if (queries[tk].first < 0 || queries[tk].end > nq) return 6;
                    }
    std::printf("ok %lld\n", pairs);
    return 0;
}
