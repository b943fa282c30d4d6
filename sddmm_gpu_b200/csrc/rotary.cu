// Rotary positions: pairs (a, b) of a head turned by angle = position * frequency,
//
//   (a, b) -> m (a cos - b sin, b cos + a sin),
//
// for up to four arrays of the same rows in one launch (Q, K and, only copied, V), each to an array of its own, in place, or to listed rows
// (of a cache).  A frequency comes as turns a position, whole turns left out, cut to 64 bits behind the point, so that position * frequency modulo
// one turn is an integer product that wraps, near or far; its upper 32 bits become the argument of sincospi.  The angle is thus off by
// |position| 2^-64 turns, from the cut, and 2^-25 of half a turn, from the argument: the first is the lesser up to positions of 2^38.  The inverse
// turns the other way: also the gradient of the rotation.
//
// What bounds it: DRAM, and next to it the sines (56 % of the issue slots at 25 % occupancy).  A thread keeps the sines of V pairs (16 bytes
// of each half) of one row and takes up to HEADS heads, whose loads are all asked for before the first is used.  32,768 rows of
// 32 + 8 heads of 128, bfloat16 (671 MB): 124 us (5.4 TB/s) with four heads and three blocks of 256 threads a multiprocessor;
// two blocks 134, four (spilling) 155; two heads 147 to 161, eight 147.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <string>

#include "attention.cuh"
#include "device_guard.hpp"
#include "engine_internal.hpp"
#include "sddmm_b200.h"

namespace {

constexpr int MAX_PAIRS = 256, MAX_PARTS = 4, THREADS = 256, HEADS = 4;

struct RotaryPart {
    const void *src;
    void *dst;
    int64_t src_row, src_head, dst_row, dst_head;  // strides in elements
    const int64_t *dst_rows;
    int64_t n_dst_rows;
    int heads, chunks;       // heads in chunks of HEADS (or fewer)
    int turn, copy;          // units of V pairs that are turned, units of V elements that are copied, in a head
    int copy_from;           // first element that is copied
    int64_t items;
};
struct RotaryParams {
    RotaryPart part[MAX_PARTS];
    const int64_t *positions;
    int64_t position0, n_rows;
    float magnitude;
    int half;         // rot_dim / 2
    int interleaved;
    int per;          // heads a thread takes
    int *status;
    uint64_t turns[MAX_PAIRS];  // a position
};

template <class T, int V> struct alignas(sizeof(T) * V) Vec { T x[V]; };
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void narrow(float x, float &y) { y = x; }
__device__ __forceinline__ void narrow(float x, __half &y) { y = __float2half_rn(x); }
__device__ __forceinline__ void narrow(float x, __nv_bfloat16 &y) { y = __float2bfloat16_rn(x); }

template <class T, int V>
__global__ void __launch_bounds__(THREADS, 3) rotary_kernel(const __grid_constant__ RotaryParams p)
{
    const RotaryPart &part = p.part[blockIdx.y];
    const int64_t item = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    if (item >= part.items) return;
    const unsigned units = part.turn + part.copy;
    int u, chunk;
    int64_t row;
    if (part.items <= UINT32_MAX) {  // 32-bit divisions, nearly always
        const unsigned rest = (unsigned)item / units;
        u = (int)((unsigned)item - rest * units);
        row = rest / (unsigned)part.chunks;
        chunk = (int)(rest - (unsigned)row * part.chunks);
    } else {
        const int64_t rest = item / units;
        u = (int)(item % units);
        chunk = (int)(rest % part.chunks);
        row = rest / part.chunks;
    }
    int64_t to = row;
    if (part.dst_rows) {
        to = part.dst_rows[row];
        if (to < 0) return;  // not wanted
        if (to >= part.n_dst_rows) {
            sddmm::report_bad_index(p.status);
            return;
        }
    }
    const int h0 = chunk * p.per, n = min(p.per, part.heads - h0);
    const T *src = static_cast<const T *>(part.src) + row * part.src_row + h0 * part.src_head;
    T *dst = static_cast<T *>(part.dst) + to * part.dst_row + h0 * part.dst_head;
    using W = Vec<T, V>;
    if (u >= part.turn) {
        const int c = part.copy_from + (u - part.turn) * V;
        W v[HEADS];
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
            if (h < n) v[h] = *reinterpret_cast<const W *>(src + h * part.src_head + c);
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
            if (h < n) *reinterpret_cast<W *>(dst + h * part.dst_head + c) = v[h];
        return;
    }
    const int i0 = u * V;                                              // first pair
    const int ca = p.interleaved ? 2 * i0 : i0, cb = p.interleaved ? 2 * i0 + V : p.half + i0;  // the two vectors that hold the pairs
    W a[HEADS], b[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
        if (h < n) {
            a[h] = *reinterpret_cast<const W *>(src + h * part.src_head + ca);
            b[h] = *reinterpret_cast<const W *>(src + h * part.src_head + cb);
        }
    const uint64_t pos = (uint64_t)(p.positions ? p.positions[row] : p.position0 + row);
    float cs[V], sn[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int hi = (int)((pos * p.turns[i0 + i]) >> 32);  // turns times 2^32, from -1/2 to 1/2
        sincospif((float)hi * 4.656612873077393e-10f, &sn[i], &cs[i]);  // 2^-31: in half turns
        cs[i] *= p.magnitude;
        sn[i] *= p.magnitude;
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
        if (h < n) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                // pair i: interleaved, elements 2i and 2i + 1 of the two vectors behind one another
                T &xa = p.interleaved ? (2 * i < V ? a[h].x[2 * i % V] : b[h].x[2 * i % V]) : a[h].x[i];
                T &xb = p.interleaved ? (2 * i + 1 < V ? a[h].x[(2 * i + 1) % V] : b[h].x[(2 * i + 1) % V]) : b[h].x[i];
                const float x = widen(xa), y = widen(xb);
                narrow(x * cs[i] - y * sn[i], xa);
                narrow(y * cs[i] + x * sn[i], xb);
            }
            *reinterpret_cast<W *>(dst + h * part.dst_head + ca) = a[h];
            *reinterpret_cast<W *>(dst + h * part.dst_head + cb) = b[h];
        }
}

template <class T, int V>
cudaError_t launch(const RotaryParams &p, int n_parts, cudaStream_t s)
{
    int64_t most = 0;
    for (int i = 0; i < n_parts; ++i) most = p.part[i].items > most ? p.part[i].items : most;
    if (most == 0) return cudaSuccess;
    const dim3 grid((unsigned)((most + THREADS - 1) / THREADS), n_parts);
    rotary_kernel<T, V><<<grid, THREADS, 0, s>>>(p);
    return cudaGetLastError();
}
template <class T>
cudaError_t by_vector(int V, const RotaryParams &p, int n_parts, cudaStream_t s)
{
    switch (V) {
    case 8: if constexpr (sizeof(T) == 2) return launch<T, 8>(p, n_parts, s); [[fallthrough]];
    case 4: return launch<T, 4>(p, n_parts, s);
    case 2: return launch<T, 2>(p, n_parts, s);
    default: return launch<T, 1>(p, n_parts, s);
    }
}

constexpr double MOST_FREQUENCY = 18446744073709551616.0;  // 2^64 radians a position
// f radians (|f| < 2^64) as turns, whole ones left out, cut to 64 bits behind the point: f = m 2^e times 1 / (2 pi), in whole numbers.
uint64_t turns_of(double f)
{
    // 256 bits of 1 / (2 pi), the last ones first (by Machin's formula for pi): off by 2^-192 turns for the largest f
    static constexpr uint64_t PER_RADIAN[4] = {0x7f9458eaf7aef158u, 0x36d8a5664f10e410u, 0x7f09d5f47d4d3770u, 0x28be60db9391054au};
    if (f == 0) return 0;
    int e;
    const uint64_t m = (uint64_t)std::ldexp(std::frexp(std::fabs(f), &e), 53);
    uint64_t product[5], carry = 0;
    for (int i = 0; i < 4; ++i) {
        const unsigned __int128 x = (unsigned __int128)m * PER_RADIAN[i] + carry;
        product[i] = (uint64_t)x;
        carry = (uint64_t)(x >> 64);
    }
    product[4] = carry;
    // |f| = m 2^(e - 53); product 2^(e - 53 - 256) turns, of which the bits from 2^-64 to 2^-1 are wanted
    const int shift = 192 + 53 - e, word = shift / 64, bit = shift % 64;
    uint64_t t = 0;
    if (word < 5) t = product[word] >> bit;
    if (bit && word + 1 < 5) t |= product[word + 1] << (64 - bit);
    return f < 0 ? 0 - t : t;
}

int bad(sddmm_handle_s *h, const std::string &why)
{
    h->last_error = why;
    return SDDMM_INVALID_ARG;
}

}  // namespace

int sddmm_rotary_frequencies(int rot_dim, double base, double factor, double original_len, double low_turns, double high_turns,
                             double *frequencies)
{
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > 2 * MAX_PAIRS || !frequencies || !(base > 0) || !std::isfinite(base) || !(factor > 0) ||
        !std::isfinite(factor) || !(original_len >= 0) || !std::isfinite(original_len))
        return SDDMM_INVALID_ARG;
    if (original_len > 0 && !(low_turns >= 0 && high_turns > low_turns && std::isfinite(high_turns))) return SDDMM_INVALID_ARG;
    for (int i = 0; i < rot_dim / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / rot_dim);
        double kept = 0;
        if (original_len > 0) {
            const double turns = original_len * f / (2 * M_PI);
            kept = (turns - low_turns) / (high_turns - low_turns);
            kept = kept < 0 ? 0 : kept > 1 ? 1 : kept;
        }
        frequencies[i] = f * (kept + (1 - kept) / factor);
    }
    return SDDMM_OK;
}

int sddmm_rotary(sddmm_handle_t h, const sddmm_rotary_desc *d, const sddmm_rotary_part *parts, int n_parts, uint32_t flags)
{
    using namespace sddmm;
    if (!h) return SDDMM_INVALID_ARG;
    if (!d || !parts || n_parts < 1 || n_parts > MAX_PARTS) return bad(h, "a description and one to four parts");
    if (flags & ~(uint32_t)SDDMM_FLAG_ASYNC) return bad(h, "unknown flag");
    if (d->dtype != SDDMM_F32 && d->dtype != SDDMM_F16 && d->dtype != SDDMM_BF16) return bad(h, "unknown dtype");
    if (d->layout != SDDMM_ROTARY_HALF && d->layout != SDDMM_ROTARY_INTERLEAVED) return bad(h, "unknown layout");
    if (d->head_dim < 1 || d->rot_dim < 0 || d->rot_dim % 2 || d->rot_dim > d->head_dim || d->rot_dim > 2 * MAX_PAIRS)
        return bad(h, "rot_dim must be even, at most head_dim and at most 512");
    if (d->n_rows < 0 || d->n_rows > INT32_MAX) return bad(h, "n_rows goes from 0 to 2^31 - 1");
    if (d->rot_dim > 0 && !d->frequencies) return bad(h, "no frequencies");
    if (!std::isfinite(d->magnitude)) return bad(h, "magnitude must be finite");
    DeviceGuard guard(h->device);
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (!(flags & SDDMM_FLAG_ASYNC) && cudaStreamIsCapturing(h->stream, &capture) == cudaSuccess && capture != cudaStreamCaptureStatusNone)
        return bad(h, "a captured call must be asynchronous");
    if (d->n_rows > 0 && d->positions && (!on_device(d->positions, h->device) || (uintptr_t)d->positions % 8))
        return bad(h, "positions must be int64 in device memory of the handle's GPU");
    const size_t size = d->dtype == SDDMM_F32 ? 4 : 2;
    RotaryParams p{};
    p.positions = d->positions;
    p.position0 = d->position0;
    p.n_rows = d->n_rows;
    p.magnitude = d->magnitude;
    p.half = d->rot_dim / 2;
    p.interleaved = d->layout == SDDMM_ROTARY_INTERLEAVED;
    p.status = h->d_status;
    for (int i = 0; i < p.half; ++i) {
        if (!(std::fabs(d->frequencies[i]) < MOST_FREQUENCY)) return bad(h, "a frequency is not finite, or of 2^64 radians or more");
        p.turns[i] = turns_of(d->inverse ? -d->frequencies[i] : d->frequencies[i]);
    }
    // Elements of an access: 16 bytes, or as many as all pieces, addresses and strides are multiples of
    int V = (int)(16 / size);
    auto fit = [&](uint64_t elements) { while (V > 1 && elements % V) V /= 2; };
    auto fit_bytes = [&](const void *q) { while (V > 1 && (uintptr_t)q % (V * size)) V /= 2; };
    bool any = false;
    for (int i = 0; i < n_parts; ++i) {
        const sddmm_rotary_part &a = parts[i];
        const std::string name = "part " + std::to_string(i);
        if (a.heads < 1) return bad(h, name + ": no heads");
        if (d->n_rows == 0) continue;
        if (!on_device(a.src, h->device) || !on_device(a.dst, h->device) || (uintptr_t)a.src % size || (uintptr_t)a.dst % size)
            return bad(h, name + " must be device memory of the handle's GPU, aligned to its elements");
        if (a.dst_rows && (!on_device(a.dst_rows, h->device) || (uintptr_t)a.dst_rows % 8 || a.n_dst_rows < 0))
            return bad(h, name + ": dst_rows must be int64 in device memory of the handle's GPU");
        if (a.src_row_stride < 0 || a.src_head_stride < 0 || a.dst_row_stride < 0 || a.dst_head_stride < 0)
            return bad(h, name + " has a negative stride");
        if (!strides_apart(a.dst_head_stride, a.heads, a.dst_row_stride, a.dst_rows ? a.n_dst_rows : d->n_rows, d->head_dim))
            return bad(h, name + " is written, and its strides let entries overlap");
        const bool in_place = a.src == a.dst && a.src_row_stride == a.dst_row_stride && a.src_head_stride == a.dst_head_stride && !a.dst_rows;
        RotaryPart &q = p.part[i];
        q = RotaryPart{a.src, a.dst, a.src_row_stride, a.src_head_stride, a.dst_row_stride, a.dst_head_stride, a.dst_rows, a.n_dst_rows,
                       a.heads, 0, 0, 0, 0, 0};
        q.turn = a.rotate ? p.half : 0;       // in pairs, for now
        q.copy_from = 2 * q.turn;
        q.copy = in_place ? 0 : d->head_dim - q.copy_from;  // in elements, for now
        fit(q.turn);
        fit(q.copy);
        fit(q.copy_from);
        for (int64_t st : {a.src_row_stride, a.src_head_stride, a.dst_row_stride, a.dst_head_stride}) fit((uint64_t)st);
        fit_bytes(a.src);
        fit_bytes(a.dst);
        any = true;
    }
    if (!any) return SDDMM_OK;
    // What is written is read by no other thread and written by no other: in place, thread by thread; or rows of a cache by different lists
    for (int i = 0; i < n_parts; ++i) {
        if (p.part[i].turn + p.part[i].copy == 0) continue;
        for (int j = 0; j < n_parts; ++j) {
            const bool in_place = i == j && parts[i].src_row_stride == parts[i].dst_row_stride && parts[i].src_head_stride == parts[i].dst_head_stride && !parts[i].dst_rows;
            const bool lists = parts[i].dst_rows && parts[j].dst_rows && parts[i].dst_rows != parts[j].dst_rows;
            if ((parts[i].dst == parts[j].src && !in_place) || (i != j && parts[i].dst == parts[j].dst && !lists))
                return bad(h, "part " + std::to_string(i) + " writes what part " + std::to_string(j) + " reads or writes");
        }
    }
    // Heads a thread takes: its sines serve all of them; fewer where that leaves the GPU without enough threads
    int64_t threads = 0;
    for (int i = 0; i < n_parts; ++i) threads += (int64_t)(p.part[i].turn + p.part[i].copy) / V * p.part[i].heads * d->n_rows;
    p.per = HEADS;
    while (p.per > 1 && threads / p.per < (int64_t)h->sm_count * 1024) p.per /= 2;
    for (int i = 0; i < n_parts; ++i) {
        RotaryPart &q = p.part[i];
        q.turn /= V;
        q.copy /= V;
        q.chunks = (q.heads + p.per - 1) / p.per;
        q.items = (int64_t)(q.turn + q.copy) * q.chunks * d->n_rows;
        if (q.items / THREADS >= INT_MAX) return bad(h, "too many heads and rows for one launch");
    }
    cudaError_t e = d->dtype == SDDMM_F32 ? by_vector<float>(V, p, n_parts, h->stream)
                    : d->dtype == SDDMM_F16 ? by_vector<__half>(V, p, n_parts, h->stream)
                                            : by_vector<__nv_bfloat16>(V, p, n_parts, h->stream);
    if (e == cudaSuccess) {
        ++h->n_launches;
        if (flags & SDDMM_FLAG_ASYNC) return SDDMM_OK;
        e = cudaStreamSynchronize(h->stream);
        if (e == cudaSuccess) return device_status(h);
    }
    h->last_error = std::string("rotary: ") + cudaGetErrorString(e);
    (void)cudaGetLastError();
    return SDDMM_CUDA_ERROR;
}
