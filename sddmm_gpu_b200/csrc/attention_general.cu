// Attention, forward and backward, for every type, stride and head width up to 128: products in fp32 FMAs.
//
// One pass over the keys with the running maximum and sum of the softmax.  A block of 256 threads has 64 queries (or, for the gradients
// of K and V, 64 keys) and goes through tiles of 64 of the other side; a thread holds 4 x 4 scores and 4 rows x DP/16 columns of its
// accumulators in registers, operands lie in shared memory as fp32 rows with four floats of padding (128-bit loads of
// eight neighbouring rows then meet all banks).  The gradients are two kernels, each with the scores anew: dQ (which also leaves
// delta_i = dO_i.O_i for the other) and dK, dV, which sums over the query heads of its group.  No atomics: results do not
// depend on scheduling.
//
// What bounds it: the FMA pipe and the shared-memory loads that feed it (two 128-bit loads per 16 FMAs).
#include "attention_strict.cuh"

namespace sddmm {

namespace {

constexpr int B = 64, THREADS = 256, PS = B + 4;

// Rows [row0, row0 + n) of one head into shared memory, zeros behind row n and column D.
template <class T, int DP>
__device__ __forceinline__ void load_rows(float *dst, const HeadArray &a, int64_t row0, int n, int head, int D)
{
    const T *src = static_cast<const T *>(a.data) + row0 * a.row + head * a.head;
    const bool vec = sizeof(T) == 4 && (((uintptr_t)src | (uintptr_t)(a.row * 4)) & 15) == 0;
    for (int i = threadIdx.x; i < B * DP / 4; i += THREADS) {
        const int r = i / (DP / 4), c = i % (DP / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n && c < D) {
            const T *x = src + r * a.row + c;
            if (vec) v = __ldg(reinterpret_cast<const float4 *>(x));
            else v = make_float4(to_f(x[0]), to_f(x[1]), to_f(x[2]), to_f(x[3]));
        }
        *reinterpret_cast<float4 *>(dst + r * (DP + 4) + c) = v;
    }
}
__device__ __forceinline__ float4 at4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ void fma4(float4 &a, float x, float4 v)
{
    a.x = fmaf(x, v.x, a.x);
    a.y = fmaf(x, v.y, a.y);
    a.z = fmaf(x, v.z, a.z);
    a.w = fmaf(x, v.w, a.w);
}
// acc[r][c] = row ty + 16 r of x times row tx + 16 c of y
template <int DP>
__device__ __forceinline__ void rows_times_rows(float (&acc)[4][4], const float *x, const float *y, int ty, int tx)
{
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
        float4 a[4], b[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) a[r] = at4(x + (ty + 16 * r) * (DP + 4) + d);
#pragma unroll
        for (int c = 0; c < 4; ++c) b[c] = at4(y + (tx + 16 * c) * (DP + 4) + d);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                acc[r][c] = fmaf(a[r].w, b[c].w, fmaf(a[r].z, b[c].z, fmaf(a[r].y, b[c].y, fmaf(a[r].x, b[c].x, acc[r][c]))));
    }
}
// acc[r][c] += sum_j w[row ty + 16 r][j] * x[j][4 tx + 64 c ..]
template <int DP>
__device__ __forceinline__ void weights_times_rows(float4 (&acc)[4][DP / 64], const float *w, const float *x, int ty, int tx)
{
#pragma unroll 2
    for (int j = 0; j < B; j += 4) {
        float4 p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = at4(w + (ty + 16 * r) * PS + j);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                const float4 v = at4(x + (j + u) * (DP + 4) + 4 * tx + 64 * c);
#pragma unroll
                for (int r = 0; r < 4; ++r) fma4(acc[r][c], u == 0 ? p[r].x : u == 1 ? p[r].y : u == 2 ? p[r].z : p[r].w, v);
            }
    }
}
// acc[r][c] += sum_i w[i][4 ty + r] * x[i][4 tx + 64 c ..]
template <int DP>
__device__ __forceinline__ void weights_t_times_rows(float4 (&acc)[4][DP / 64], const float *w, const float *x, int ty, int tx)
{
#pragma unroll 4
    for (int i = 0; i < B; ++i) {
        const float4 p = at4(w + i * PS + 4 * ty);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float4 v = at4(x + i * (DP + 4) + 4 * tx + 64 * c);
            fma4(acc[0][c], p.x, v);
            fma4(acc[1][c], p.y, v);
            fma4(acc[2][c], p.z, v);
            fma4(acc[3][c], p.w, v);
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

template <class T, int DP>
__global__ void __launch_bounds__(THREADS) attention_forward_general_kernel(const AttentionParams p)
{
    extern __shared__ float sm[];
    __shared__ unsigned long long bad;
    __shared__ float bad_lse[B];
    if (threadIdx.x == 0) bad = 0;
    float *sq = sm, *sk = sq + B * (DP + 4), *sv = sk + B * (DP + 4), *sp = sv + B * (DP + 4);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, head = blockIdx.x % p.q_heads, kv = head / p.group;
    Sequence s;
    int seq, block;
    // the last blocks of a causal sequence have the most keys: they go first
    if (!find_block<B>(p, (gridDim.x - 1 - blockIdx.x) / p.q_heads, false, s, seq, block)) return;
    const int i0 = block * B, n = min(B, s.nq - i0);
    const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
    load_rows<T, DP>(sq, p.q, (int64_t)s.q0 + i0, n, head, p.head_dim);
    const Reach reach = reach_of(p.window, s, i0, i0 + n);
    const KeyTiles tiles = key_tiles<B>(reach);
    float4 o[4][DP / 64] = {};
    float top[4], sum[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) top[r] = -INFINITY, sum[r] = 0.f;
    for (int t = 0; t < tiles.n; ++t) {
        const int j0 = tiles.tile(t) * B, m = min(B, s.nk - j0);
        __syncthreads();
        load_rows<T, DP>(sk, p.k, (int64_t)s.k0 + j0, m, kv, p.head_dim);
        load_rows<T, DP>(sv, p.v, (int64_t)s.k0 + j0, m, kv, p.head_dim);
        __syncthreads();
        float x[4][4];
        rows_times_rows<DP>(x, sq, sk, ty, tx);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int pos = reach.first_pos + ty + 16 * r;
            float most = -INFINITY, unused;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = j0 + tx + 16 * c;
                const float v = score(p, slope, x[r][c], pos, j, unused);
                x[r][c] = key_seen(p.window, s, pos, j) ? v : -INFINITY;
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
            sum[r] = sum[r] * shrink + over16(add, true);
            top[r] = now;
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                o[r][c].x *= shrink;
                o[r][c].y *= shrink;
                o[r][c].z *= shrink;
                o[r][c].w *= shrink;
            }
        }
        __syncthreads();
        weights_times_rows<DP>(o, sp, sv, ty, tx);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = ty + 16 * r;
        if (i >= n) continue;
        const float inv = sum[r] > 0.f ? 1.f / sum[r] : sum[r] == 0.f ? 0.f : NAN;
        const int64_t row = (int64_t)s.q0 + i0 + i;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float4 v = o[r][c];
            collect(&bad, not_finite(v), i);
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
__global__ void __launch_bounds__(THREADS) attention_dq_general_kernel(const AttentionParams p)
{
    extern __shared__ float sm[];
    __shared__ unsigned long long bad;
    __shared__ float bad_lse[B], bad_delta[B];
    if (threadIdx.x == 0) bad = 0;
    float *sq = sm, *sdo = sq + B * (DP + 4), *sk = sdo + B * (DP + 4), *sv = sk + B * (DP + 4), *sds = sv + B * (DP + 4);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, head = blockIdx.x % p.q_heads, kv = head / p.group;
    Sequence s;
    int seq, block;
    if (!find_block<B>(p, (gridDim.x - 1 - blockIdx.x) / p.q_heads, false, s, seq, block)) return;
    const int i0 = block * B, n = min(B, s.nq - i0);
    const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
    load_rows<T, DP>(sq, p.q, (int64_t)s.q0 + i0, n, head, p.head_dim);
    load_rows<T, DP>(sdo, p.d_o, (int64_t)s.q0 + i0, n, head, p.head_dim);
    load_rows<T, DP>(sk, p.o, (int64_t)s.q0 + i0, n, head, p.head_dim);
    __syncthreads();
    float delta[4], lse[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = ty + 16 * r;
        float d = 0.f;
        for (int c = tx; c < p.head_dim; c += 16) d = fmaf(sdo[i * (DP + 4) + c], sk[i * (DP + 4) + c], d);
        delta[r] = over16(d, true);
        const int64_t at = (int64_t)head * p.q_rows + s.q0 + i0 + i;
        lse[r] = i < n ? __ldg(p.lse + at) : -INFINITY;
        if (tx == 0) {
            bad_lse[i] = lse[r];
            bad_delta[i] = delta[r];
            if (i < n) p.delta[at] = delta[r];
        }
    }
    const Reach reach = reach_of(p.window, s, i0, i0 + n);
    const KeyTiles tiles = key_tiles<B>(reach);
    float4 dq[4][DP / 64] = {};
    for (int t = 0; t < tiles.n; ++t) {
        const int j0 = tiles.tile(t) * B, m = min(B, s.nk - j0);
        __syncthreads();
        load_rows<T, DP>(sk, p.k, (int64_t)s.k0 + j0, m, kv, p.head_dim);
        load_rows<T, DP>(sv, p.v, (int64_t)s.k0 + j0, m, kv, p.head_dim);
        __syncthreads();
        float x[4][4], dp[4][4];
        rows_times_rows<DP>(x, sq, sk, ty, tx);
        rows_times_rows<DP>(dp, sdo, sv, ty, tx);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int pos = reach.first_pos + ty + 16 * r;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = j0 + tx + 16 * c;
                float dcap;
                const float v = score(p, slope, x[r][c], pos, j, dcap);
                float ds = 0.f;
                if (lse[r] != -INFINITY && key_seen(p.window, s, pos, j)) ds = exp2f((v - lse[r]) * LOG2E) * (dp[r][c] - delta[r]) * dcap * p.scale;
                sds[(ty + 16 * r) * PS + tx + 16 * c] = ds;
            }
        }
        __syncthreads();
        weights_times_rows<DP>(dq, sds, sk, ty, tx);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (ty + 16 * r >= n) continue;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            collect(&bad, not_finite(dq[r][c]), ty + 16 * r);
            store4<T>(p.dq, (int64_t)s.q0 + i0 + ty + 16 * r, head, 4 * tx + 64 * c, p.head_dim, dq[r][c]);
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
template <class T, int DP>
__global__ void __launch_bounds__(THREADS) attention_dkv_general_kernel(const AttentionParams p)
{
    extern __shared__ float sm[];
    __shared__ unsigned long long bad;
    if (threadIdx.x == 0) bad = 0;
    float *sk = sm, *sv = sk + B * (DP + 4), *sq = sv + B * (DP + 4), *sdo = sq + B * (DP + 4), *sp = sdo + B * (DP + 4), *sds = sp + B * PS;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, kv = blockIdx.x % p.kv_heads;
    Sequence s;
    int seq, block;
    // the first keys of a causal sequence are seen by the most queries: they go first
    if (!find_block<B>(p, blockIdx.x / p.kv_heads, true, s, seq, block)) return;
    const int j0 = block * B, m = min(B, s.nk - j0);
    load_rows<T, DP>(sk, p.k, (int64_t)s.k0 + j0, m, kv, p.head_dim);
    load_rows<T, DP>(sv, p.v, (int64_t)s.k0 + j0, m, kv, p.head_dim);
    int from, to;
    queries_of(p.window, s, j0, j0 + m, from, to);
    float4 dk[4][DP / 64] = {}, dv[4][DP / 64] = {};
    for (int head = kv * p.group; head < (kv + 1) * p.group; ++head) {
        const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
        for (int i0 = from / B * B; i0 < to; i0 += B) {
            const int n = min(B, s.nq - i0);
            __syncthreads();
            load_rows<T, DP>(sq, p.q, (int64_t)s.q0 + i0, n, head, p.head_dim);
            load_rows<T, DP>(sdo, p.d_o, (int64_t)s.q0 + i0, n, head, p.head_dim);
            __syncthreads();
            float x[4][4], dp[4][4];
            rows_times_rows<DP>(x, sq, sk, ty, tx);
            rows_times_rows<DP>(dp, sdo, sv, ty, tx);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = ty + 16 * r, pos = s.nk - s.nq + i0 + i;
                const int64_t at = (int64_t)head * p.q_rows + s.q0 + i0 + i;
                const float lse = i < n ? __ldg(p.lse + at) : -INFINITY, delta = i < n ? p.delta[at] : 0.f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int j = j0 + tx + 16 * c;
                    float dcap;
                    const float v = score(p, slope, x[r][c], pos, j, dcap);
                    float e = 0.f, ds = 0.f;
                    if (lse != -INFINITY && key_seen(p.window, s, pos, j)) {
                        e = exp2f((v - lse) * LOG2E);
                        ds = e * (dp[r][c] - delta) * dcap * p.scale;
                    }
                    sp[i * PS + tx + 16 * c] = e;
                    sds[i * PS + tx + 16 * c] = ds;
                }
            }
            __syncthreads();
            weights_t_times_rows<DP>(dv, sp, sdo, ty, tx);
            weights_t_times_rows<DP>(dk, sds, sq, ty, tx);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (4 * ty + r >= m) continue;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const int64_t row = (int64_t)s.k0 + j0 + 4 * ty + r;
            collect(&bad, not_finite(dk[r][c]) || not_finite(dv[r][c]), 4 * ty + r);
            store4<T>(p.dk, row, kv, 4 * tx + 64 * c, p.head_dim, dk[r][c]);
            store4<T>(p.dv, row, kv, 4 * tx + 64 * c, p.head_dim, dv[r][c]);
        }
    }
    __syncthreads();
    int turn = 0;
    for (unsigned long long left = bad; left; left &= left - 1, ++turn)
        if (turn % (THREADS / 32) == (int)threadIdx.x / 32) strict::dkv_row<T>(p, s, kv, j0 + __ffsll((long long)left) - 1);
}

template <class Kern>
cudaError_t launch(Kern kern, SmemOptinCache &optin, unsigned grid, size_t smem, const AttentionParams &p, cudaStream_t s)
{
    const cudaError_t e = optin_dynamic_smem(kern, smem, optin);
    if (e != cudaSuccess) return e;
    if (grid == 0) return cudaSuccess;
    kern<<<grid, THREADS, smem, s>>>(p);
    return cudaGetLastError();
}
constexpr size_t smem_of(int DP, int tiles, int weights) { return ((size_t)tiles * B * (DP + 4) + (size_t)weights * B * PS) * sizeof(float); }

template <class T, int DP>
cudaError_t forward_of(const AttentionParams &p, cudaStream_t s)
{
    static SmemOptinCache optin;
    const unsigned grid = (unsigned)(p.q_heads * most_blocks(p.q_rows, p.n_seqs, p.max_q, B));
    return launch(attention_forward_general_kernel<T, DP>, optin, grid, smem_of(DP, 3, 1), p, s);
}
template <class T, int DP>
cudaError_t backward_of(const AttentionParams &p, cudaStream_t s)
{
    static SmemOptinCache optin_q, optin_kv;
    const unsigned grid_q = (unsigned)(p.q_heads * most_blocks(p.q_rows, p.n_seqs, p.max_q, B));
    const unsigned grid_kv = (unsigned)(p.kv_heads * most_blocks(p.k_rows, p.n_seqs, p.max_k, B));
    const cudaError_t e = launch(attention_dq_general_kernel<T, DP>, optin_q, grid_q, smem_of(DP, 4, 1), p, s);
    return e != cudaSuccess ? e : launch(attention_dkv_general_kernel<T, DP>, optin_kv, grid_kv, smem_of(DP, 4, 2), p, s);
}

template <class T>
cudaError_t by_width(bool backward, const AttentionParams &p, cudaStream_t s)
{
    if (p.head_dim <= 64) return backward ? backward_of<T, 64>(p, s) : forward_of<T, 64>(p, s);
    return backward ? backward_of<T, 128>(p, s) : forward_of<T, 128>(p, s);
}
cudaError_t by_type(bool backward, const AttentionParams &p, cudaStream_t s)
{
    switch (p.dtype) {
    case 0: return by_width<float>(backward, p, s);
    case 1: return by_width<__half>(backward, p, s);
    default: return by_width<__nv_bfloat16>(backward, p, s);
    }
}

}  // namespace

cudaError_t launch_attention_forward_general(const AttentionParams &p, cudaStream_t s) { return by_type(false, p, s); }
cudaError_t launch_attention_backward_general(const AttentionParams &p, cudaStream_t s) { return by_type(true, p, s); }

}  // namespace sddmm
