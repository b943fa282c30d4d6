// Attention, forward and backward, for every type, stride and head width up to 128: products in fp32 FMAs.
//
// One pass over the keys with the running maximum and sum of the softmax.  A block of 256 threads has 64 queries (or, for the gradients
// of K and V, 64 keys) and goes through tiles of 64 of the other side; a thread holds 4 x 4 scores and 4 rows x DP/16 columns of its
// accumulators in registers, operands lie in shared memory as fp32 rows with four floats of padding (128-bit loads of
// eight neighbouring rows then meet all banks).  The gradients are two kernels, each with the scores anew: dQ (which also leaves
// delta_i = dO_i.O_i for the other) and dK, dV, which sums over the query heads of its group.  No atomics: results do not
// depend on scheduling.
// The forward kernel in fp32 cuts the keys into parts where its blocks leave multiprocessors idle; attention_join_kernel adds them up.
// A tile's copies are asked for as soon as the last one in its place has been used, and come in under the product in between.
//
// What bounds it: the FMA pipe and the shared-memory loads that feed it (two 128-bit loads per 16 FMAs).  fp32, 1,900 + 1,333 tokens that
// see their past and a prefix of 500, 8 heads of 64: 244 us, 24.7 TFLOP/s; gradient of 701 + 950 tokens, 4 / 2 heads of 80: 190 us, 12.4.
#include <climits>
#include <cmath>
#include <type_traits>

#include "attention_strict.cuh"
#include "device_utils.cuh"

namespace sddmm {

namespace {

constexpr int B = GENERAL_ROWS, THREADS = 256, PS = B + 4;

// Rows [row0, row0 + n) of one head into shared memory, zeros behind row n; a row of D columns has `stride` = D + 4 floats.  fp32 rows with
// 16-byte alignment come by asynchronous copies, which the caller waits for (arrived()); others have been stored when this returns.
template <class T>
__device__ __forceinline__ void load_rows(float *dst, const HeadArray &a, int64_t row0, int n, int head, int D, int stride)
{
    const T *src = static_cast<const T *>(a.data) + row0 * a.row + head * a.head;
    const bool vec = sizeof(T) == 4 && (((uintptr_t)src | (uintptr_t)(a.row * 4)) & 15) == 0;
    const int quads = D / 4, step = THREADS / quads;  // a thread keeps its columns: `step` rows at once
    const int c = threadIdx.x % quads * 4;
    if ((int)threadIdx.x < step * quads)
        for (int r = threadIdx.x / quads; r < B; r += step) {
            const T *x = src + (r < n ? r : 0) * a.row + c;
            float *to = dst + r * stride + c;
            if (vec) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dev::smem_u32(to)), "l"(x), "r"(r < n ? 16 : 0) : "memory");
            } else {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < n) v = make_float4(to_f(x[0]), to_f(x[1]), to_f(x[2]), to_f(x[3]));
                *reinterpret_cast<float4 *>(to) = v;
            }
        }
    asm volatile("cp.async.commit_group;" ::: "memory");
}
// All of this thread's copies but the last `N` load_rows() have landed.
template <int N> __device__ __forceinline__ void arrived() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float4 at4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
using F2 = unsigned long long;  // two fp32 values: one FMA instruction for both
using dev::ffma2;
using dev::fold2;
__device__ __forceinline__ F2 twice(float x)
{
    F2 r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ ulonglong2 pairs(const float *p) { return *reinterpret_cast<const ulonglong2 *>(p); }
// acc[r][c] = row ty + 16 r of x times row tx + 16 c of y, D columns
__device__ __forceinline__ void rows_times_rows(float (&acc)[4][4], const float *x, const float *y, int ty, int tx, int D)
{
    F2 sum[4][4] = {};
    const int stride = D + 4;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
        ulonglong2 a[4], b[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) a[r] = pairs(x + (ty + 16 * r) * stride + d);
#pragma unroll
        for (int c = 0; c < 4; ++c) b[c] = pairs(y + (tx + 16 * c) * stride + d);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[r][c] = ffma2(a[r].y, b[c].y, ffma2(a[r].x, b[c].x, sum[r][c]));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = fold2(sum[r][c]);
}
// Four columns of a row.
struct Quad {
    F2 a, b;
};
__device__ __forceinline__ float4 open(Quad q)
{
    float4 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(q.a));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.z), "=f"(v.w) : "l"(q.b));
    return v;
}
__device__ __forceinline__ void add_times(Quad &acc, float w, ulonglong2 v)
{
    const F2 ww = twice(w);
    acc.a = ffma2(ww, v.x, acc.a);
    acc.b = ffma2(ww, v.y, acc.b);
}
// acc[r][c] += sum_j w[row ty + 16 r][j] * x[j][4 tx + 64 c ..]; columns from the head's width on are anything
template <int DP>
__device__ __forceinline__ void weights_times_rows(Quad (&acc)[4][DP / 64], const float *w, const float *x, int ty, int tx, int stride)
{
#pragma unroll 4
    for (int j = 0; j < B; j += 4) {
        float4 p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = at4(w + (ty + 16 * r) * PS + j);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                const ulonglong2 v = pairs(x + (j + u) * stride + 4 * tx + 64 * c);
#pragma unroll
                for (int r = 0; r < 4; ++r) add_times(acc[r][c], u == 0 ? p[r].x : u == 1 ? p[r].y : u == 2 ? p[r].z : p[r].w, v);
            }
    }
}
// acc[r][c] += sum_i w[i][4 ty + r] * x[i][4 tx + 64 c ..]
template <int DP>
__device__ __forceinline__ void weights_t_times_rows(Quad (&acc)[4][DP / 64], const float *w, const float *x, int ty, int tx, int stride)
{
#pragma unroll 4
    for (int i = 0; i < B; ++i) {
        const float4 p = at4(w + i * PS + 4 * ty);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const ulonglong2 v = pairs(x + i * stride + 4 * tx + 64 * c);
            add_times(acc[0][c], p.x, v);
            add_times(acc[1][c], p.y, v);
            add_times(acc[2][c], p.z, v);
            add_times(acc[3][c], p.w, v);
        }
    }
}
template <class T>
__device__ __forceinline__ void store4(const HeadArray &a, int64_t row, int head, int col, int D, float4 v)
{
    if (col >= D) return;
    T *dst = static_cast<T *>(a.data) + row * a.row + head * a.head + col;
    dst[0] = from_f<T>(v.x);
    dst[1] = from_f<T>(v.y);
    dst[2] = from_f<T>(v.z);
    dst[3] = from_f<T>(v.w);
}
__device__ __forceinline__ float over16(float x, bool sum)
{
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
        const float y = __shfl_xor_sync(0xffffffffu, x, o);
        x = sum ? x + y : fmaxf(x, y);
    }
    return x;
}
// Bits of the block's rows that are not finite, for whole warps to walk through; every thread calls it, with a barrier on both sides.
__device__ __forceinline__ void collect(unsigned long long *bits, bool bad, int row)
{
    if (bad) atomicOr(bits, 1ull << row);
}

// PARTS: the keys of a block may be cut (a form of its own: what it has to remember costs the other 4 %).
template <class T, int DP, bool PARTS>
__global__ void __launch_bounds__(THREADS, 2) attention_forward_general_kernel(const AttentionParams p)
{
    extern __shared__ float sm[];
    __shared__ unsigned long long bad;
    __shared__ float bad_lse[B];
    if (threadIdx.x == 0) bad = 0;
    const int stride = p.head_dim + 4;
    float *sq = sm, *sk = sq + B * stride, *sv = sk + B * stride, *sp = sv + B * stride;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, head = blockIdx.x % p.q_heads, kv = head / p.group;
    const unsigned splits = PARTS ? p.n_splits : 1, behind = (gridDim.x - 1 - blockIdx.x) / p.q_heads, part = PARTS ? behind % splits : 0;
    if (PARTS) next_kernel_may_come();
    Sequence s;
    int seq, block;
    // the last blocks of a causal sequence have the most keys: they go first
    if (!find_block<B>(p, behind / splits, false, s, seq, block)) return;
    const int i0 = block * B, n = min(B, s.nq - i0);
    const Reach reach = reach_of(p.window, s, i0, i0 + n);
    const KeyTiles tiles = key_tiles<B>(reach);
    const Part mine = PARTS ? part_of(p, tiles.n, part) : Part{0, tiles.n, true};
    if (PARTS && mine.end < 0) return;
    const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
    load_rows<T>(sq, p.q, (int64_t)s.q0 + i0, n, head, p.head_dim, stride);
    Quad o[4][DP / 64] = {};
    float top[4], sum[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) top[r] = -INFINITY, sum[r] = 0.f;
    auto fetch = [&](float *to, const HeadArray &a, int t) {
        const int j0 = tiles.tile(t) * B;
        load_rows<T>(to, a, (int64_t)s.k0 + j0, min(B, s.nk - j0), kv, p.head_dim, stride);
    };
    if (tiles.n > 0) fetch(sk, p.k, mine.first), fetch(sv, p.v, mine.first);
    for (int t = mine.first; t < mine.end; ++t) {
        const int j0 = tiles.tile(t) * B;
        arrived<1>();  // K, and Q
        __syncthreads();
        const bool all = tile_is_open<B>(p.window, s, reach, j0);  // nothing is hidden here
        float x[4][4];
        rows_times_rows(x, sq, sk, ty, tx, p.head_dim);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int pos = reach.first_pos + ty + 16 * r;
            float most = -INFINITY, unused;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = j0 + tx + 16 * c;
                const float v = score(p, slope, x[r][c], pos, j, unused);
                x[r][c] = all || key_seen(p.window, s, pos, j) ? v : -INFINITY;
                most = fmaxf(most, x[r][c]);
            }
            const float now = fmaxf(top[r], over16(most, false));
            const float base = now == -INFINITY ? 0.f : now;  // a row that has seen nothing yet
            const float shrink = exp2f((top[r] - base) * LOG2E);
            float add = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float e = exp2f((x[r][c] - base) * LOG2E);
                add += e;
                sp[(ty + 16 * r) * PS + tx + 16 * c] = e;
            }
            sum[r] = sum[r] * shrink + add;  // (of this thread's columns)
            top[r] = now;
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                const F2 by = twice(shrink);
                o[r][c].a = ffma2(o[r][c].a, by, 0ull);
                o[r][c].b = ffma2(o[r][c].b, by, 0ull);
            }
        }
        arrived<0>();  // V
        __syncthreads();
        const bool more = t + 1 < mine.end;
        if (more) fetch(sk, p.k, t + 1);  // under the product with V
        weights_times_rows<DP>(o, sp, sv, ty, tx, stride);
        __syncthreads();
        if (more) fetch(sv, p.v, t + 1);  // under the next scores
    }
    arrived<0>();  // (a block without tiles: its rows' copies)
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[r] = over16(sum[r], true);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = ty + 16 * r;
        if (i >= n) continue;
        const float inv = sum[r] > 0.f ? 1.f / sum[r] : sum[r] == 0.f ? 0.f : NAN;
        const int64_t row = (int64_t)s.q0 + i0 + i;
        if (PARTS && !mine.alone) {  // for attention_join_kernel, which also looks after what is not finite
            const int64_t at = (part * p.q_rows + row) * p.q_heads + head;
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                const float4 v = open(o[r][c]);
                if (4 * tx + 64 * c < p.head_dim)
                    *reinterpret_cast<float4 *>(p.part_o + at * p.head_dim + 4 * tx + 64 * c) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            }
            if (tx == 0) p.part_lse[at] = sum[r] == 0.f ? -INFINITY : top[r] * LOG2E + log2f(sum[r]);
            continue;
        }
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float4 v = open(o[r][c]);
            collect(&bad, not_finite(v) && 4 * tx + 64 * c < p.head_dim, i);
            store4<T>(p.o, row, head, 4 * tx + 64 * c, p.head_dim, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        }
        if (tx == 0) {
            bad_lse[i] = sum[r] == 0.f ? -INFINITY : top[r] + logf(sum[r]);
            if (p.lse) p.lse[(int64_t)head * p.q_rows + row] = bad_lse[i];
        }
    }
    __syncthreads();
    int turn = 0;
    for (unsigned long long left = bad; left; left &= left - 1, ++turn) {
        const int i = __ffsll((long long)left) - 1;
        if (turn % (THREADS / 32) == (int)threadIdx.x / 32) strict::output_row<T>(p, s, head, i0 + i, bad_lse[i]);
    }
}

// dQ of 64 queries; leaves delta for attention_dkv_general_kernel.
template <class T, int DP>
__global__ void __launch_bounds__(THREADS, 2) attention_dq_general_kernel(const AttentionParams p)
{
    extern __shared__ float sm[];
    __shared__ unsigned long long bad;
    __shared__ float bad_lse[B], bad_delta[B];
    if (threadIdx.x == 0) bad = 0;
    const int stride = p.head_dim + 4;
    float *sq = sm, *sdo = sq + B * stride, *sk = sdo + B * stride, *sv = sk + B * stride, *sds = sv + B * stride;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const unsigned block_of = blockIdx.x / p.n_splits, part = blockIdx.x % p.n_splits, blocks = gridDim.x / p.n_splits;
    const int head = block_of % p.q_heads, kv = head / p.group;
    Sequence s;
    int seq, block;
    next_kernel_may_come();
    if (!find_block<B>(p, (blocks - 1 - block_of) / p.q_heads, false, s, seq, block)) return;
    const int i0 = block * B, n = min(B, s.nq - i0);
    const Reach reach = reach_of(p.window, s, i0, i0 + n);
    const KeyTiles tiles = key_tiles<B>(reach);
    const Part mine = part_of(p, tiles.n, part);
    if (mine.end < 0) return;
    const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
    load_rows<T>(sq, p.q, (int64_t)s.q0 + i0, n, head, p.head_dim, stride);
    load_rows<T>(sdo, p.d_o, (int64_t)s.q0 + i0, n, head, p.head_dim, stride);
    load_rows<T>(sk, p.o, (int64_t)s.q0 + i0, n, head, p.head_dim, stride);
    arrived<0>();
    __syncthreads();
    float delta[4], lse[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = ty + 16 * r;
        float d = 0.f;
        for (int c = tx; c < p.head_dim; c += 16) d = fmaf(sdo[i * stride + c], sk[i * stride + c], d);
        delta[r] = over16(d, true);
        const int64_t at = (int64_t)head * p.q_rows + s.q0 + i0 + i;
        lse[r] = i < n ? __ldg(p.lse + at) : -INFINITY;
        if (tx == 0) {
            bad_lse[i] = lse[r];
            bad_delta[i] = delta[r];
            if (i < n && part == 0) p.delta[at] = delta[r];
        }
    }
    Quad dq[4][DP / 64] = {};
    auto fetch = [&](float *to, const HeadArray &a, int t) {
        const int j0 = tiles.tile(t) * B;
        load_rows<T>(to, a, (int64_t)s.k0 + j0, min(B, s.nk - j0), kv, p.head_dim, stride);
    };
    __syncthreads();  // (O lay where K is to lie)
    if (mine.first < mine.end) fetch(sv, p.v, mine.first), fetch(sk, p.k, mine.first);
    for (int t = mine.first; t < mine.end; ++t) {
        const int j0 = tiles.tile(t) * B;
        const bool all = tile_is_open<B>(p.window, s, reach, j0);
        float x[4][4], dp[4][4];
        arrived<1>();
        __syncthreads();
        rows_times_rows(dp, sdo, sv, ty, tx, p.head_dim);
        arrived<0>();
        __syncthreads();
        rows_times_rows(x, sq, sk, ty, tx, p.head_dim);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int pos = reach.first_pos + ty + 16 * r;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = j0 + tx + 16 * c;
                float dcap;
                const float v = score(p, slope, x[r][c], pos, j, dcap);
                float ds = 0.f;
                if (lse[r] != -INFINITY && (all || key_seen(p.window, s, pos, j))) ds = exp2f((v - lse[r]) * LOG2E) * (dp[r][c] - delta[r]) * dcap * p.scale;
                sds[(ty + 16 * r) * PS + tx + 16 * c] = ds;
            }
        }
        __syncthreads();
        const bool more = t + 1 < mine.end;
        if (more) fetch(sv, p.v, t + 1);  // under the product with K
        weights_times_rows<DP>(dq, sds, sk, ty, tx, stride);
        __syncthreads();
        if (more) fetch(sk, p.k, t + 1);  // under the next dP
    }
    arrived<0>();  // (a block without tiles: its rows' copies)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = ty + 16 * r;
        if (i >= n) continue;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float4 v = open(dq[r][c]);
            if (mine.alone) {
                collect(&bad, not_finite(v) && 4 * tx + 64 * c < p.head_dim, i);
                store4<T>(p.dq, (int64_t)s.q0 + i0 + i, head, 4 * tx + 64 * c, p.head_dim, v);
            } else if (4 * tx + 64 * c < p.head_dim) {
                *reinterpret_cast<float4 *>(p.part_o + ((part * p.q_rows + s.q0 + i0 + i) * p.q_heads + head) * p.head_dim + 4 * tx + 64 * c) = v;
            }
        }
    }
    __syncthreads();
    int turn = 0;
    for (unsigned long long left = bad; left; left &= left - 1, ++turn) {
        const int i = __ffsll((long long)left) - 1;
        if (turn % (THREADS / 32) == (int)threadIdx.x / 32) strict::dq_row<T>(p, s, head, i0 + i, bad_lse[i], bad_delta[i]);
    }
}

// dK and dV of 64 keys, over all queries of all heads of the group.
// (Two blocks on a multiprocessor for heads of 64, which shared memory allows: 1,000 tokens of 8 heads 173 -> 159 us with dQ.)
template <class T, int DP>
__global__ void __launch_bounds__(THREADS, DP == 64 ? 2 : 1) attention_dkv_general_kernel(const AttentionParams p)
{
    extern __shared__ float sm[];
    __shared__ unsigned long long bad;
    if (threadIdx.x == 0) bad = 0;
    const int stride = p.head_dim + 4;
    float *sk = sm, *sv = sk + B * stride, *sq = sv + B * stride, *sdo = sq + B * stride, *sp = sdo + B * stride, *sds = sp + B * PS;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const unsigned block_of = blockIdx.x / p.n_splits, part = blockIdx.x % p.n_splits;
    const int kv = block_of % p.kv_heads;
    Sequence s;
    int seq, block;
    // the first keys of a causal sequence are seen by the most queries: they go first
    const bool found = find_block<B>(p, block_of / p.kv_heads, true, s, seq, block);
    next_kernel_may_come();
    behind_last_kernel();
    if (!found) return;
    const int j0 = block * B, m = min(B, s.nk - j0);
    int from, per_head;
    query_tiles<B>(p, s, j0, m, from, per_head);
    const Part mine = part_of(p, per_head * p.group, part);
    if (mine.end < 0) return;
    load_rows<T>(sk, p.k, (int64_t)s.k0 + j0, m, kv, p.head_dim, stride);
    load_rows<T>(sv, p.v, (int64_t)s.k0 + j0, m, kv, p.head_dim, stride);
    Quad dk[4][DP / 64] = {}, dv[4][DP / 64] = {};
    auto fetch = [&](float *to, const HeadArray &a, int t) {
        const int i0 = (from + t % per_head) * B;
        load_rows<T>(to, a, (int64_t)s.q0 + i0, min(B, s.nq - i0), kv * p.group + t / per_head, p.head_dim, stride);
    };
    if (mine.first < mine.end) fetch(sdo, p.d_o, mine.first), fetch(sq, p.q, mine.first);
    for (int t = mine.first; t < mine.end; ++t) {
        const int head = kv * p.group + t / per_head, i0 = (from + t % per_head) * B, n = min(B, s.nq - i0);
        const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
        float x[4][4], dp[4][4], lse[4], delta[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {  // (on their way under the products)
            const int i = ty + 16 * r;
            const int64_t at = (int64_t)head * p.q_rows + s.q0 + i0 + i;
            lse[r] = i < n ? __ldg(p.lse + at) : -INFINITY;
            delta[r] = i < n ? p.delta[at] : 0.f;
        }
        const bool all = n == B && tile_is_open<B>(p.window, s, reach_of(p.window, s, i0, i0 + n), j0);
        arrived<1>();
        __syncthreads();
        rows_times_rows(dp, sdo, sv, ty, tx, p.head_dim);
        arrived<0>();
        __syncthreads();
        rows_times_rows(x, sq, sk, ty, tx, p.head_dim);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = ty + 16 * r, pos = s.nk - s.nq + i0 + i;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = j0 + tx + 16 * c;
                float dcap;
                const float v = score(p, slope, x[r][c], pos, j, dcap);
                float e = 0.f, ds = 0.f;
                if (lse[r] != -INFINITY && (all || key_seen(p.window, s, pos, j))) {
                    e = exp2f((v - lse[r]) * LOG2E);
                    ds = e * (dp[r][c] - delta[r]) * dcap * p.scale;
                }
                sp[i * PS + tx + 16 * c] = e;
                sds[i * PS + tx + 16 * c] = ds;
            }
        }
        __syncthreads();
        const bool more = t + 1 < mine.end;
        weights_t_times_rows<DP>(dv, sp, sdo, ty, tx, stride);
        __syncthreads();
        if (more) fetch(sdo, p.d_o, t + 1);  // under the product with Q
        weights_t_times_rows<DP>(dk, sds, sq, ty, tx, stride);
        __syncthreads();
        if (more) fetch(sq, p.q, t + 1);  // under the next dP
    }
    arrived<0>();  // (a block without tiles: its rows' copies)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (4 * ty + r >= m) continue;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const int64_t row = (int64_t)s.k0 + j0 + 4 * ty + r;
            const float4 a = open(dk[r][c]), b = open(dv[r][c]);
            if (mine.alone) {
                collect(&bad, (not_finite(a) || not_finite(b)) && 4 * tx + 64 * c < p.head_dim, 4 * ty + r);
                store4<T>(p.dk, row, kv, 4 * tx + 64 * c, p.head_dim, a);
                store4<T>(p.dv, row, kv, 4 * tx + 64 * c, p.head_dim, b);
            } else if (4 * tx + 64 * c < p.head_dim) {
                float *to = p.part_o + (((2 * part) * p.k_rows + row) * p.kv_heads + kv) * p.head_dim + 4 * tx + 64 * c;
                *reinterpret_cast<float4 *>(to) = a;
                *reinterpret_cast<float4 *>(to + p.k_rows * p.kv_heads * p.head_dim) = b;
            }
        }
    }
    __syncthreads();
    int turn = 0;
    for (unsigned long long left = bad; left; left &= left - 1, ++turn)
        if (turn % (THREADS / 32) == (int)threadIdx.x / 32) strict::dkv_row<T>(p, s, kv, j0 + __ffsll((long long)left) - 1);
}

// The parts' sums of 16 rows added in order; KV: dK and dV, else dQ.  TILE: rows of the blocks that left them.
constexpr int SUM_ROWS = 16;
template <class T, bool KV, int TILE>
__global__ void __launch_bounds__(THREADS) attention_sum_parts_kernel(const AttentionParams p)
{
    __shared__ unsigned bad;
    if (threadIdx.x == 0) bad = 0;
    const unsigned slice = blockIdx.x % (TILE / SUM_ROWS), block_of = blockIdx.x / (TILE / SUM_ROWS);
    const int heads = KV ? p.kv_heads : p.q_heads, head = block_of % heads;
    Sequence s;
    int seq, block;
    const bool found = find_block<TILE>(p, block_of / heads, KV, s, seq, block);
    next_kernel_may_come();
    behind_last_kernel();
    if (!found) return;
    const int t0 = block * TILE, in_tile = min(TILE, (KV ? s.nk : s.nq) - t0), r0 = t0 + slice * SUM_ROWS, rows = min(SUM_ROWS, t0 + in_tile - r0);
    if (rows <= 0) return;
    int tiles;
    if (KV) {
        int from, per_head;
        query_tiles<TILE>(p, s, t0, in_tile, from, per_head);
        tiles = per_head * p.group;
    } else {
        tiles = key_tiles<TILE>(reach_of(p.window, s, t0, t0 + in_tile)).n;
    }
    const int parts = (tiles + p.chunk_tiles - 1) / p.chunk_tiles;
    if (parts <= 1) return;
    __syncthreads();
    const int quads = p.head_dim / 4;
    const int64_t array = (KV ? p.k_rows : p.q_rows) * heads * p.head_dim;
    for (int i = threadIdx.x; i < rows * quads; i += THREADS) {
        const int r = i / quads, c = i % quads * 4;
        const int64_t row = (int64_t)(KV ? s.k0 : s.q0) + r0 + r;
#pragma unroll
        for (int x = 0; x < (KV ? 2 : 1); ++x) {
            const float *from = p.part_o + x * array + (row * heads + head) * p.head_dim + c;
            float4 sum = at4(from);
#pragma unroll 4
            for (int k = 1; k < parts; ++k) {
                const float4 v = at4(from + k * array * (KV ? 2 : 1));
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
            if (not_finite(sum)) atomicOr(&bad, 1u << r);
            store4<T>(KV ? (x ? p.dv : p.dk) : p.dq, row, head, c, p.head_dim, sum);
        }
    }
    __syncthreads();
    int turn = 0;
    for (unsigned left = bad; left; left &= left - 1, ++turn) {
        const int r = __ffs(left) - 1;
        if (turn % (THREADS / 32) != (int)threadIdx.x / 32) continue;
        const int64_t at = (int64_t)head * p.q_rows + s.q0 + r0 + r;
        if (KV) strict::dkv_row<T>(p, s, head, r0 + r);
        else strict::dq_row<T>(p, s, head, r0 + r, __ldg(p.lse + at), p.delta[at]);
    }
}

template <class Kern>
cudaError_t launch(Kern kern, SmemOptinCache &optin, unsigned grid, size_t smem, const AttentionParams &p, cudaStream_t s, bool behind = false)
{
    const cudaError_t e = optin_dynamic_smem(kern, smem, optin);
    if (e != cudaSuccess) return e;
    if (grid == 0) return cudaSuccess;
    if (behind) return launch_behind(kern, grid, THREADS, smem, s, p);
    kern<<<grid, THREADS, smem, s>>>(p);
    return cudaGetLastError();
}
size_t smem_of(int head_dim, int tiles, int weights) { return ((size_t)tiles * B * (head_dim + 4) + (size_t)weights * B * PS) * sizeof(float); }

template <class T, int DP>
cudaError_t forward_of(const AttentionParams &p, cudaStream_t s)
{
    static SmemOptinCache optin;
    const unsigned grid = (unsigned)(p.max_q > 0 ? p.q_heads * most_blocks(p.q_rows, p.n_seqs, p.max_q, B) : 1);
    if constexpr (std::is_same<T, float>::value) {
        static SmemOptinCache optin_parts;
        if (p.n_splits > 1) return launch(attention_forward_general_kernel<T, DP, true>, optin_parts, grid * p.n_splits, smem_of(p.head_dim, 3, 1), p, s);
    }
    return launch(attention_forward_general_kernel<T, DP, false>, optin, grid, smem_of(p.head_dim, 3, 1), p, s);
}
template <class T, int DP>
cudaError_t backward_of(const AttentionParams &p0, const Parts &parts, cudaStream_t s)
{
    static SmemOptinCache optin_q, optin_kv;
    const unsigned grid_q = (unsigned)(p0.max_q > 0 || p0.max_k > 0 ? p0.q_heads * most_blocks(p0.q_rows, p0.n_seqs, p0.max_q, B) : 1);
    const unsigned grid_kv = (unsigned)(p0.kv_heads * most_blocks(p0.k_rows, p0.n_seqs, p0.max_k, B));
    AttentionParams p = p0;
    p.n_splits = parts.n_q;
    p.chunk_tiles = parts.tiles_q;
    cudaError_t e = launch(attention_dq_general_kernel<T, DP>, optin_q, grid_q * parts.n_q, smem_of(p.head_dim, 4, 1), p, s);
    if (e == cudaSuccess && parts.n_q > 1) e = launch_attention_sum_parts(p, false, B, s);
    if (e != cudaSuccess) return e;
    p.n_splits = parts.n_kv;
    p.chunk_tiles = parts.tiles_kv;
    e = launch(attention_dkv_general_kernel<T, DP>, optin_kv, grid_kv * parts.n_kv, smem_of(p.head_dim, 4, 2), p, s, grid_q > 0);
    if (e == cudaSuccess && parts.n_kv > 1) e = launch_attention_sum_parts(p, true, B, s);
    return e;
}

// parts null: forward
template <class T>
cudaError_t by_width(const Parts *parts, const AttentionParams &p, cudaStream_t s)
{
    if (p.head_dim <= 64) return parts ? backward_of<T, 64>(p, *parts, s) : forward_of<T, 64>(p, s);
    return parts ? backward_of<T, 128>(p, *parts, s) : forward_of<T, 128>(p, s);
}
cudaError_t by_type(const Parts *parts, const AttentionParams &p, cudaStream_t s)
{
    switch (p.dtype) {
    case 0: return by_width<float>(parts, p, s);
    case 1: return by_width<__half>(parts, p, s);
    default: return by_width<__nv_bfloat16>(parts, p, s);
    }
}

}  // namespace

Parts plan_attention_parts(const AttentionParams &p, int tile, int per_sm, int sm_count)
{
    // Parts until there are `per_sm` blocks for a multiprocessor (a causal mask leaves some with little to do), of two tiles at least, and at
    // most 256 MB of sums.
    auto cut = [&](int64_t blocks, int64_t tiles, int64_t bytes_of_one, int &n, int &each) {
        n = 1;
        each = (int)(tiles > 0 ? tiles : 1);
        if (blocks <= 0 || tiles <= 2) return;
        int64_t want = ((int64_t)per_sm * sm_count + blocks - 1) / blocks;
        if (want > (256ll << 20) / (bytes_of_one > 0 ? bytes_of_one : 1)) want = (256ll << 20) / (bytes_of_one > 0 ? bytes_of_one : 1);
        if (want > (tiles + 1) / 2) want = (tiles + 1) / 2;
        if (want <= 1) return;
        each = (int)((tiles + want - 1) / want);
        n = (int)((tiles + each - 1) / each);
    };
    Parts g{};
    const int64_t bytes_q = 4 * p.q_rows * p.q_heads * p.head_dim, bytes_kv = 8 * p.k_rows * p.kv_heads * p.head_dim;
    cut(p.q_heads * most_blocks(p.q_rows, p.n_seqs, p.max_q, tile), (p.max_k + tile - 1) / tile, bytes_q, g.n_q, g.tiles_q);
    cut(p.kv_heads * most_blocks(p.k_rows, p.n_seqs, p.max_k, tile), (int64_t)((p.max_q + tile - 1) / tile) * p.group, bytes_kv, g.n_kv, g.tiles_kv);
    const int64_t q = g.n_q > 1 ? g.n_q * bytes_q : 0, kv = g.n_kv > 1 ? g.n_kv * bytes_kv : 0;
    g.bytes = q > kv ? q : kv;  // one behind the other
    return g;
}

cudaError_t launch_attention_sum_parts(const AttentionParams &p, bool kv, int tile, cudaStream_t s)
{
    const unsigned grid = (unsigned)(kv ? p.kv_heads * most_blocks(p.k_rows, p.n_seqs, p.max_k, tile) : p.q_heads * most_blocks(p.q_rows, p.n_seqs, p.max_q, tile)) * (tile / SUM_ROWS);
    if (grid == 0) return cudaSuccess;
    auto run = [&](auto of_kv, auto of_q) { return launch_behind(kv ? of_kv : of_q, grid, THREADS, 0, s, p); };
    if (p.dtype == 0) return run(attention_sum_parts_kernel<float, true, 64>, attention_sum_parts_kernel<float, false, 64>);
    if (p.dtype == 1) return run(attention_sum_parts_kernel<__half, true, 128>, attention_sum_parts_kernel<__half, false, 128>);
    return run(attention_sum_parts_kernel<__nv_bfloat16, true, 128>, attention_sum_parts_kernel<__nv_bfloat16, false, 128>);
}

ForwardPlan plan_attention_forward_general(const AttentionParams &p, int sm_count)
{
    // fp32 alone: 16-bit types come here for strides and alignment, which a plan does not know
    const int64_t tiles = p.max_k > 0 ? (p.max_k + B - 1) / B : 1, blocks = p.q_heads * most_blocks(p.q_rows, p.n_seqs, p.max_q, B);
    const int64_t bytes = p.q_rows * p.q_heads * (int64_t)(p.head_dim + 1) * 4, rows = p.q_rows * p.q_heads;
    const bool narrow = p.head_dim <= 64;
    const int resident = narrow ? 2 : 1;  // blocks on a multiprocessor, by shared memory
    ForwardPlan best{1, 1 << 30, 0, INFINITY};
    for (int64_t n = 1; n <= 128 && (n == 1 || (n <= tiles / 2 && n * bytes <= 256ll << 20)); ++n) {
        const int64_t each = (tiles + n - 1) / n;
        if (n > 1 && (p.dtype != 0 || (tiles + each - 1) / each != n || (int64_t)p.n_seqs * p.max_q * p.q_heads > INT32_MAX)) continue;
        // A tile of 64 keys takes 6.5 us of a block alone and 7.7 of two together, of 128 columns 10; the join takes 6 and 1 for 800 rows.  One part / parts:
        // 64 queries on 2,000 keys, 8 heads of 64, 209 / 23 us; 1,000 on 1,000 107 / 78, of 128 165 / 107; where blocks fill the GPU anyway, 1,900 + 1,333
        // tokens, 268 / 342 (measured before tiles without masks were told apart).
        // Waves: whole ones where all blocks have as much to do; else the short ones fill the last.
        const double full = (double)(blocks * n) / (resident * sm_count), fill = p.window.right >= 0 && p.max_k < 2ll * p.max_q ? full : ceil(full);
        const double tile = !narrow ? 10. : blocks * n > sm_count ? 7.7 : 6.5;
        const double us = 5. + (n > 1 ? 6. + rows / 800. : 0.) + (fill > 1. ? fill : 1.) * (double)each * tile;
        if (us < best.us) best = ForwardPlan{(int)n, n == 1 ? 1 << 30 : (int)each, n == 1 ? 0 : n * bytes, us};
    }
    return best;
}

cudaError_t launch_attention_forward_general(const AttentionParams &p0, const ForwardPlan &f, void *workspace, cudaStream_t s)
{
    AttentionParams p = p0;
    p.n_splits = f.n_splits;
    p.chunk_tiles = f.chunk_tiles;
    p.part_o = static_cast<float *>(workspace);
    p.part_lse = p.part_o + (f.n_splits == 1 ? 0 : (int64_t)f.n_splits * p.q_rows * p.q_heads * p.head_dim);
    const cudaError_t e = by_type(nullptr, p, s);
    return e == cudaSuccess && p.n_splits > 1 ? launch_attention_join(p, JOIN_GENERAL, s) : e;
}
cudaError_t launch_attention_backward_general(const AttentionParams &p, const Parts &parts, cudaStream_t s) { return by_type(&parts, p, s); }

}  // namespace sddmm
