// Index arithmetic of the attention masks (csrc/attention_mask.hpp) against the definition, key by key, and at the limits of its range.
#include <climits>
#include <cstdio>
#include <vector>

#include "attention_mask.hpp"

using namespace sddmm;

static bool seen(Window w, const Sequence &s, int i, int j)
{
    const long long pos = (long long)s.nk - s.nq + i;
    return j < s.prefix || ((w.left < 0 || j >= pos - w.left) && (w.right < 0 || j <= pos + w.right));
}

template <int T, int BQ>
static long check(Window w, const Sequence &s)
{
    long bad = 0;
    for (int i0 = 0; i0 < s.nq; i0 += BQ) {
        const int i1 = min_of(s.nq, i0 + BQ);
        const Reach r = reach_of(w, s, i0, i1);
        const KeyTiles t = key_tiles<T>(r);
        std::vector<int> visits((s.nk + T - 1) / T, 0);
        for (int n = 0; n < t.n; ++n) {
            if (t.tile(n) < 0 || t.tile(n) >= (int)visits.size()) { ++bad; continue; }
            ++visits[t.tile(n)];
            if (n > 0 && t.tile(n) <= t.tile(n - 1)) ++bad;
        }
        for (int k = 0; k < (int)visits.size(); ++k) {
            for (int i = i0; i < i1; ++i) {  // as bits: the places that a query sees
                const int pos = s.nk - s.nq + i;
                const int lo = w.left < 0 ? 0 : max_of(0, pos - w.left), hi = w.right < 0 ? s.nk - 1 : min_of(s.nk - 1, pos + w.right);
                const unsigned bits = seen_bits(lo, hi, s.prefix, k * T);
                for (int j = 0; j < 32; ++j)
                    if ((bits >> j & 1u) != (unsigned)(k * T + j < s.nk && seen(w, s, i, k * T + j))) ++bad;
            }
            bool any = false, all = true;
            for (int i = i0; i < i1; ++i)
                for (int j = k * T; j < k * T + T; ++j) {
                    const bool x = j < s.nk && seen(w, s, i, j);
                    if (x != key_seen(w, s, s.nk - s.nq + i, j)) ++bad;
                    any = any || x;
                    all = all && x;
                }
            if (visits[k] > 1 || (any && !visits[k])) ++bad;
            if (tile_is_open<T>(w, s, r, k * T) && !all) ++bad;  // (a tile half prefix, half window may count as not open)
        }
    }
    for (int k0 = 0; k0 < s.nk; k0 += T) {
        int a, b;
        queries_of(w, s, k0, min_of(s.nk, k0 + T), a, b);
        if (a < 0 || b > s.nq || a > b) ++bad;
        for (int i = 0; i < s.nq; ++i)
            for (int j = k0; j < min_of(s.nk, k0 + T); ++j)
                if (seen(w, s, i, j) && (i < a || i >= b)) ++bad;
    }
    return bad;
}

int main()
{
    int failures = 0;
    long cases = 0, bad = 0;
    const int lengths[] = {0, 1, 3, 7, 8, 9, 20, 33};
    for (int nq : lengths)
        for (int nk : lengths)
            for (int left : {-1, 0, 1, 5, 40})
                for (int right : {-1, 0, 2, 11})
                    for (int prefix : {0, 1, 8, 13, 33}) {
                        const Sequence s{0, nq, 0, nk, min_of(prefix, nk)};
                        bad += check<8, 8>(Window{left, right}, s) + check<4, 16>(Window{left, right}, s);
                        ++cases;
                    }
    printf("%s: %ld masks, %ld wrong\n", bad == 0 ? "ok" : "FAILED", cases, bad);
    failures += bad != 0;
    // the largest arrays and windows: nothing wraps
    bad = 0;
    const int most = 1 << 29, wide = (1 << 30) - 1;
    for (int nq : {1, most})
        for (int nk : {1, most})
            for (int left : {-1, 0, wide})
                for (int right : {-1, 0, wide}) {
                    const Window w{left, right};
                    const Sequence s{0, nq, 0, nk, 0};
                    for (int i : {0, nq - 1})
                        for (int j : {0, nk - 1}) {
                            bad += key_seen(w, s, nk - nq + i, j) != seen(w, s, i, j);
                            int a, b;
                            queries_of(w, s, j, j + 1, a, b);
                            bad += seen(w, s, i, j) && (i < a || i >= b);
                            const KeyTiles t = key_tiles<128>(reach_of(w, s, i, i + 1));
                            bool there = false;
                            if (t.n > 0) there = t.tile(0) <= j / 128 && j / 128 <= t.tile(t.n - 1);
                            bad += seen(w, s, i, j) && !there;
                        }
                }
    printf("%s: limits, %ld wrong\n", bad == 0 ? "ok" : "FAILED", bad);
    failures += bad != 0;
    bad = most_blocks(0, 0, 0, 64) != 0 || most_blocks(10, 3, 5, 64) != 3 || most_blocks(6400, 2, 6400, 64) != 102;
    printf("%s: blocks\n", bad == 0 ? "ok" : "FAILED");
    return failures + (bad != 0);
}
