// Rows of results, one at a time, from the definition: nothing of what a row does not see is touched.
//
// The tiled kernels multiply hidden places by zero weights, and 0 x NaN is NaN: a row whose tile held a NaN or an infinity in a hidden place
// comes out not finite, although the definition gives numbers.  A block looks for such rows when it is done and a warp computes each of
// them again here.  Where what is seen is itself not finite the walk ends as soon as no number is left, so that a training run that has
// diverged does not crawl.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention.cuh"

namespace sddmm {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Score of query position pos and key j from their product, and (slope of the cap) 1 - tanh^2.
__device__ __forceinline__ float score(const AttentionParams &p, float slope, float qk, int pos, int j, float &dcap)
{
    float x = qk * p.scale;
    dcap = 1.f;
    if (p.cap > 0.f) {
        const float t = tanhf(x / p.cap);
        x = p.cap * t;
        dcap = 1.f - t * t;
    }
    return x - slope * (float)abs(pos - j);
}

namespace strict {

constexpr int PER_LANE = 4;  // columns of a lane: lane, lane + 32, ...

template <class T>
__device__ __forceinline__ void load(float (&x)[PER_LANE], const HeadArray &a, int64_t row, int head, int D)
{
    const T *src = static_cast<const T *>(a.data) + row * a.row + head * a.head;
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c) {
        const int at = (threadIdx.x & 31) + 32 * c;
        x[c] = at < D ? to_f(src[at]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store(const float (&x)[PER_LANE], const HeadArray &a, int64_t row, int head, int D)
{
    T *dst = static_cast<T *>(a.data) + row * a.row + head * a.head;
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c) {
        const int at = (threadIdx.x & 31) + 32 * c;
        if (at < D) dst[at] = from_f<T>(x[c]);
    }
}
__device__ __forceinline__ float dot(const float (&x)[PER_LANE], const float (&y)[PER_LANE])
{
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c) s = fmaf(x[c], y[c], s);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}
__device__ __forceinline__ void axpy(float (&y)[PER_LANE], float a, const float (&x)[PER_LANE])
{
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c) y[c] = fmaf(a, x[c], y[c]);
}
__device__ __forceinline__ bool no_number_left(const float (&x)[PER_LANE], int D)
{
    bool nan = true;
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c)
        if ((int)(threadIdx.x & 31) + 32 * c < D) nan = nan && isnan(x[c]);
    return __all_sync(0xffffffffu, nan);
}

// One warp: O of query i from its lse.
template <class T>
__device__ __forceinline__ void output_row(const AttentionParams &p, const Sequence &s, int head, int i, float lse)
{
    if (isnan(lse)) return;
    const int kv = head / p.group, pos = s.nk - s.nq + i;
    const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
    float q[PER_LANE], k[PER_LANE], v[PER_LANE], o[PER_LANE] = {}, unused;
    load<T>(q, p.q, (int64_t)s.q0 + i, head, p.head_dim);
    const KeyTiles tiles = key_tiles<1>(reach_of(p.window, s, i, i + 1));
    if (lse != -INFINITY)
        for (int t = 0; t < tiles.n && ((t & 15) || !no_number_left(o, p.head_dim)); ++t) {
            const int j = tiles.tile(t);
            load<T>(k, p.k, (int64_t)s.k0 + j, kv, p.head_dim);
            load<T>(v, p.v, (int64_t)s.k0 + j, kv, p.head_dim);
            axpy(o, exp2f((score(p, slope, dot(q, k), pos, j, unused) - lse) * LOG2E), v);
        }
    store<T>(o, p.o, (int64_t)s.q0 + i, head, p.head_dim);
}

// One warp: dQ of query i.
template <class T>
__device__ __forceinline__ void dq_row(const AttentionParams &p, const Sequence &s, int head, int i, float lse, float delta)
{
    if (isnan(lse) || isnan(delta)) return;
    const int kv = head / p.group, pos = s.nk - s.nq + i;
    const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
    float q[PER_LANE], d_o[PER_LANE], k[PER_LANE], v[PER_LANE], dq[PER_LANE] = {}, dcap;
    load<T>(q, p.q, (int64_t)s.q0 + i, head, p.head_dim);
    load<T>(d_o, p.d_o, (int64_t)s.q0 + i, head, p.head_dim);
    const KeyTiles tiles = key_tiles<1>(reach_of(p.window, s, i, i + 1));
    if (lse != -INFINITY)
        for (int t = 0; t < tiles.n && ((t & 15) || !no_number_left(dq, p.head_dim)); ++t) {
            const int j = tiles.tile(t);
            load<T>(k, p.k, (int64_t)s.k0 + j, kv, p.head_dim);
            load<T>(v, p.v, (int64_t)s.k0 + j, kv, p.head_dim);
            const float e = exp2f((score(p, slope, dot(q, k), pos, j, dcap) - lse) * LOG2E);
            axpy(dq, e * (dot(d_o, v) - delta) * dcap * p.scale, k);
        }
    store<T>(dq, p.dq, (int64_t)s.q0 + i, head, p.head_dim);
}

// One warp: dK and dV of key j.
template <class T>
__device__ __forceinline__ void dkv_row(const AttentionParams &p, const Sequence &s, int kv, int j)
{
    float k[PER_LANE], v[PER_LANE], q[PER_LANE], d_o[PER_LANE], dk[PER_LANE] = {}, dv[PER_LANE] = {}, dcap;
    load<T>(k, p.k, (int64_t)s.k0 + j, kv, p.head_dim);
    load<T>(v, p.v, (int64_t)s.k0 + j, kv, p.head_dim);
    int from, to;
    queries_of(p.window, s, j, j + 1, from, to);
    for (int head = kv * p.group; head < (kv + 1) * p.group; ++head) {
        const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
        for (int i = from; i < to; ++i) {
            const int64_t at = (int64_t)head * p.q_rows + s.q0 + i;
            const float lse = __ldg(p.lse + at);
            if (lse == -INFINITY) continue;
            load<T>(q, p.q, (int64_t)s.q0 + i, head, p.head_dim);
            load<T>(d_o, p.d_o, (int64_t)s.q0 + i, head, p.head_dim);
            const float e = exp2f((score(p, slope, dot(q, k), s.nk - s.nq + i, j, dcap) - lse) * LOG2E);
            axpy(dv, e, d_o);
            axpy(dk, e * (dot(d_o, v) - p.delta[at]) * dcap * p.scale, q);
            if ((i & 15) == 15 && no_number_left(dk, p.head_dim) && no_number_left(dv, p.head_dim)) {
                head = p.q_heads;
                break;
            }
        }
    }
    store<T>(dk, p.dk, (int64_t)s.k0 + j, kv, p.head_dim);
    store<T>(dv, p.dv, (int64_t)s.k0 + j, kv, p.head_dim);
}

}  // namespace strict

__device__ __forceinline__ bool not_finite(float4 v) { return !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w)); }

}  // namespace sddmm
