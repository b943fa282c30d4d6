// The mask of attention as index arithmetic: which keys a block of queries may see, and the other way round.  Host and device.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define MASK_FN __host__ __device__ __forceinline__
#else
#define MASK_FN inline
#endif

namespace sddmm {

MASK_FN int min_of(int a, int b) { return a < b ? a : b; }
MASK_FN int max_of(int a, int b) { return a > b ? a : b; }

// One sequence of the batch.
struct Sequence {
    int q0, nq, k0, nk, prefix;  // prefix <= nk
};
// Key j is seen from position pos: j < prefix, or pos - left <= j <= pos + right; -1: no limit; at most 2^30 - 1, and all rows at most 2^29.
struct Window {
    int left, right;
};

// The keys that queries [i0, i1) of a sequence may see: [0, prefix) and [lo, hi].
struct Reach {
    int prefix, lo, hi;  // lo > hi: none beside the prefix
    int first_pos, last_pos;
};
MASK_FN Reach reach_of(Window w, const Sequence &s, int i0, int i1)
{
    Reach r;
    r.prefix = s.prefix;
    r.first_pos = s.nk - s.nq + i0;
    r.last_pos = s.nk - s.nq + i1 - 1;
    r.lo = w.left < 0 ? 0 : max_of(0, r.first_pos - w.left);
    r.hi = w.right < 0 ? s.nk - 1 : min_of(s.nk - 1, r.last_pos + w.right);
    return r;
}
// Tiles of T keys that a block of queries goes through: the first n_prefix, then from band0 on, n in all.
struct KeyTiles {
    int n_prefix, band0, n;
    MASK_FN int tile(int i) const { return i < n_prefix ? i : band0 + (i - n_prefix); }
};
template <int T>
MASK_FN KeyTiles key_tiles(const Reach &r)
{
    KeyTiles t;
    t.n_prefix = (r.prefix + T - 1) / T;
    t.band0 = max_of(t.n_prefix, r.lo / T);
    const int end = r.lo <= r.hi ? r.hi / T + 1 : 0;
    t.n = t.n_prefix + max_of(0, end - t.band0);
    return t;
}
// Whether every query of the block sees all of keys [k0, k0 + T).
template <int T>
MASK_FN bool tile_is_open(Window w, const Sequence &s, const Reach &r, int k0)
{
    if (k0 + T > s.nk) return false;
    if (k0 + T <= r.prefix) return true;
    return (w.left < 0 || k0 >= r.last_pos - w.left) && (w.right < 0 || k0 + T - 1 <= r.first_pos + w.right);
}
MASK_FN bool key_seen(Window w, const Sequence &s, int pos, int j)
{
    return j < s.nk && (j < s.prefix || ((w.left < 0 || j >= pos - w.left) && (w.right < 0 || j <= pos + w.right)));
}
// Bits of 32 places from `at` on: those in [lo, hi], and those below pre.
MASK_FN unsigned seen_bits(int lo, int hi, int pre, int at)
{
    const int a = lo - at, b = hi - at, c = pre - at;
    const unsigned up = a <= 0 ? 0xffffffffu : a > 31 ? 0u : 0xffffffffu << a;
    const unsigned down = b >= 31 ? 0xffffffffu : b < 0 ? 0u : 0xffffffffu >> (31 - b);
    const unsigned first = c >= 32 ? 0xffffffffu : c <= 0 ? 0u : 0xffffffffu >> (32 - c);
    return (up & down) | first;
}
// The queries [i0, i1) of a sequence that may see a key of [k0, k1): all where the prefix reaches in.
MASK_FN void queries_of(Window w, const Sequence &s, int k0, int k1, int &i0, int &i1)
{
    const int off = s.nk - s.nq;  // pos = off + i
    i0 = 0;
    i1 = s.nq;
    if (k0 < s.prefix) return;
    if (w.right >= 0) i0 = max_of(0, k0 - w.right - off);
    if (w.left >= 0) i1 = min_of(s.nq, k1 + w.left - off);
    if (i1 < i0) i1 = i0;
}
// Blocks that find_block() can be asked for, at most.
inline int64_t most_blocks(int64_t rows, int n_seqs, int most, int T)
{
    const int64_t a = rows / T + n_seqs, b = (int64_t)n_seqs * ((most + T - 1) / T);
    return a < b ? a : b;
}


}  // namespace sddmm
