// Rows of results, one at a time, from the definition: nothing of what a row does not see is touched.
//
// The tiled kernels multiply hidden places by zero weights, and 0 x NaN is NaN: a row whose tile held a NaN or an infinity in a hidden place
// comes out not finite, although the definition gives numbers.  A block looks for such rows when it is done and a warp computes each of
// them again here: the columns that are not finite, since a number that came out is right.  A NaN may have come from a hidden place and goes
// on until the walk meets one that is seen; an infinity cannot have (0 x infinity is NaN), but may be a sum that ran over, and is settled once
// the walk has one too.  So where what is seen is itself not finite the walk ends there.
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
// The columns that were not finite.
template <class T>
__device__ __forceinline__ void store(const float (&x)[PER_LANE], unsigned was, const HeadArray &a, int64_t row, int head, int D)
{
    T *dst = static_cast<T *>(a.data) + row * a.row + head * a.head;
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c) {
        const int at = (threadIdx.x & 31) + 32 * c;
        if (at < D && !(was & 1u << c)) dst[at] = from_f<T>(x[c]);
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
// What the kernel stored in this thread's columns: bit c, a number (or no column of the head); bit 8 + c, an infinity.
template <class T>
__device__ __forceinline__ unsigned stored(const HeadArray &a, int64_t row, int head, int D)
{
    float x[PER_LANE];
    load<T>(x, a, row, head, D);
    unsigned kinds = 0;
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c) kinds |= isfinite(x[c]) ? 1u << c : isinf(x[c]) ? 256u << c : 0u;
    return kinds;
}
// Whether no column is left that the walk might still change.
__device__ __forceinline__ bool settled(const float (&x)[PER_LANE], unsigned was)
{
    bool yes = true;
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c) yes = yes && ((was & 1u << c) || isnan(x[c]) || ((was & 256u << c) && isinf(x[c])));
    return __all_sync(0xffffffffu, yes);
}

// One warp: O of query i from its lse.
template <class T>
__device__ __forceinline__ void output_row(const AttentionParams &p, const Sequence &s, int head, int i, float lse)
{
    if (isnan(lse)) return;
    const int kv = head / p.group, pos = s.nk - s.nq + i;
    const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
    float q[PER_LANE], k[PER_LANE], v[PER_LANE], o[PER_LANE] = {}, unused;
    const unsigned was = stored<T>(p.o, (int64_t)s.q0 + i, head, p.head_dim);
    load<T>(q, p.q, (int64_t)s.q0 + i, head, p.head_dim);
    const KeyTiles tiles = key_tiles<1>(reach_of(p.window, s, i, i + 1));
    if (lse != -INFINITY)
        for (int t = 0; t < tiles.n && ((t & 15) || !settled(o, was)); ++t) {
            const int j = tiles.tile(t);
            load<T>(k, p.k, (int64_t)s.k0 + j, kv, p.head_dim);
            load<T>(v, p.v, (int64_t)s.k0 + j, kv, p.head_dim);
            axpy(o, exp2f((score(p, slope, dot(q, k), pos, j, unused) - lse) * LOG2E), v);
        }
    store<T>(o, was, p.o, (int64_t)s.q0 + i, head, p.head_dim);
}

// One warp: dQ of query i.
template <class T>
__device__ __forceinline__ void dq_row(const AttentionParams &p, const Sequence &s, int head, int i, float lse, float delta)
{
    if (isnan(lse) || (isnan(delta) && lse != -INFINITY)) return;  // (a row that sees nothing has no gradient, whatever dO holds)
    const int kv = head / p.group, pos = s.nk - s.nq + i;
    const float slope = p.slopes ? __ldg(p.slopes + head) : 0.f;
    float q[PER_LANE], d_o[PER_LANE], k[PER_LANE], v[PER_LANE], dq[PER_LANE] = {}, dcap;
    const unsigned was = stored<T>(p.dq, (int64_t)s.q0 + i, head, p.head_dim);
    load<T>(q, p.q, (int64_t)s.q0 + i, head, p.head_dim);
    load<T>(d_o, p.d_o, (int64_t)s.q0 + i, head, p.head_dim);
    const KeyTiles tiles = key_tiles<1>(reach_of(p.window, s, i, i + 1));
    if (lse != -INFINITY)
        for (int t = 0; t < tiles.n && ((t & 15) || !settled(dq, was)); ++t) {
            const int j = tiles.tile(t);
            load<T>(k, p.k, (int64_t)s.k0 + j, kv, p.head_dim);
            load<T>(v, p.v, (int64_t)s.k0 + j, kv, p.head_dim);
            const float e = exp2f((score(p, slope, dot(q, k), pos, j, dcap) - lse) * LOG2E);
            axpy(dq, e * (dot(d_o, v) - delta) * dcap * p.scale, k);
        }
    store<T>(dq, was, p.dq, (int64_t)s.q0 + i, head, p.head_dim);
}

// One warp: dK and dV of key j.
template <class T>
__device__ __forceinline__ void dkv_row(const AttentionParams &p, const Sequence &s, int kv, int j)
{
    float k[PER_LANE], v[PER_LANE], q[PER_LANE], d_o[PER_LANE], dk[PER_LANE] = {}, dv[PER_LANE] = {}, dcap;
    const unsigned dk_was = stored<T>(p.dk, (int64_t)s.k0 + j, kv, p.head_dim), dv_was = stored<T>(p.dv, (int64_t)s.k0 + j, kv, p.head_dim);
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
            if ((i & 15) == 15 && settled(dk, dk_was) && settled(dv, dv_was)) {
                head = p.q_heads;
                break;
            }
        }
    }
    store<T>(dk, dk_was, p.dk, (int64_t)s.k0 + j, kv, p.head_dim);
    store<T>(dv, dv_was, p.dv, (int64_t)s.k0 + j, kv, p.head_dim);
}

}  // namespace strict

__device__ __forceinline__ bool not_finite(float4 v) { return !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w)); }

}  // namespace sddmm
