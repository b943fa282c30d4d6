// Attention, forward, for few queries of many keys in fp32 (single tokens over a cache): the cut into chunks, the parts and their join are
// those of attention_few_tc.cu; products are fp32 FMAs.
//
// A block has ROWS rows, (query, head) pairs of one KV head, and a chunk of the keys; each of its twelve warps takes every twelfth tile of 16
// keys through a tile of K and one of V of its own in shared memory: the next K is on its way while the weights and the output are computed,
// the next V while the scores are.  Scores: a lane has a key and half of its columns, all rows at once, so that a 128-bit load of K feeds
// 4 ROWS FMAs (Q comes as broadcasts); output: a lane has four columns, and a 128-bit load of V feeds 4 ROWS FMAs.  ROWS is the least power of two that has the rows,
// up to 8: single tokens with heads of their own would spend eight times the FMAs on one row.
//
// What bounds it: memory for a row or two (32 tokens of 8 heads of 128 over 4,000 keys each: 161 us, 6.5 TB/s); FMAs and shared memory for 8
// (200 queries, 8 heads of 128 on one, 8,000 keys: 419 us, where the general kernel in parts takes 264); beginning, ending and the join for short caches (a token of 32 / 8 heads, 8,000
// keys: 27 us, of which 10 are memory).  Twelve warps with one tile each of K and V instead of four with two: 710 -> 161, 1,109 -> 419, 51 -> 33.
#include <cmath>

#include "attention_strict.cuh"
#include "device_utils.cuh"

namespace sddmm {

namespace {

constexpr int KEYS = FEW_F32_KEYS, WARPS = 12;
// Blocks on a multiprocessor: by registers and by shared memory.
constexpr int by_registers(int rows) { return rows <= 4 ? 2 : 1; }

template <int ROWS>
__global__ void __launch_bounds__(WARPS * 32, by_registers(ROWS)) attention_few_f32_kernel(const AttentionParams p, int row_tiles)
{
    extern __shared__ __align__(16) float sm[];
    __shared__ __align__(16) float w_p[WARPS][KEYS][ROWS];
    __shared__ float w_most[WARPS][ROWS], w_sum[WARPS][ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.head_dim, stride = D + 4;
    const unsigned heads_and_rows = gridDim.x / p.n_splits, b = blockIdx.x % heads_and_rows, chunk = blockIdx.x / heads_and_rows;
    const int tile = b % row_tiles, kv = b / row_tiles % p.kv_heads, seq = b / row_tiles / p.kv_heads;
    if (p.n_splits > 1) next_kernel_may_come();
    const Sequence s = sequence_of(p, seq);
    const int rows = s.nq * p.group, r0 = tile * ROWS;
    if (r0 >= rows) return;
    const Chunks<KEYS> ch = chunks_of<KEYS>(p, s, tile, ROWS);
    if ((int)chunk >= ch.n) return;
    const int first = chunk * p.chunk_tiles, end = min(ch.keys.n, first + p.chunk_tiles);
    float *const sq = sm, *const sk = sm + ROWS * D + warp * 2 * KEYS * stride, *const sv = sk + KEYS * stride;
    const int mine = max(0, (end - first - warp + WARPS - 1) / WARPS);
    const float *K = static_cast<const float *>(p.k.data) + (int64_t)s.k0 * p.k.row + kv * p.k.head;
    const float *V = static_cast<const float *>(p.v.data) + (int64_t)s.k0 * p.v.row + kv * p.v.head;
    // Lanes of a row: the power of two that has its 16-byte pieces.
    const int quads = D / 4, lanes = quads <= 2 ? 2 : quads <= 4 ? 4 : quads <= 8 ? 8 : quads <= 16 ? 16 : 32;
    const int first_row = lane / lanes, piece = lane % lanes * 4, rows_at_once = 32 / lanes;
    auto fetch = [&](int n, const float *from, int64_t row_stride, float *to) {
        if (n < mine && piece < D) {
            const int j0 = ch.keys.tile(first + warp + n * WARPS) * KEYS;
            for (int r = first_row; r < KEYS; r += rows_at_once) {
                const int j = j0 + r;
                const int bytes = j < s.nk ? 16 : 0;  // zeros behind the sequence's end
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dev::smem_u32(to + r * stride + piece)),
                             "l"(from + (j < s.nk ? j : 0) * row_stride + piece), "r"(bytes)
                             : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(0, K, p.k.row, sk);
    fetch(0, V, p.v.row, sv);
    for (int f = threadIdx.x; f < ROWS * D; f += WARPS * 32) {
        const int r = min(r0 + f / D, rows - 1);
        sq[f] = static_cast<const float *>(p.q.data)[((int64_t)s.q0 + r / p.group) * p.q.row + (kv * p.group + r % p.group) * p.q.head + f % D];
    }
    __syncthreads();
    const int key = lane & 15, half = lane >> 4, column = 4 * lane;
    float most[ROWS], sum[ROWS], slope[ROWS];
    int pos[ROWS];
    float4 o[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int row = min(r0 + r, rows - 1);
        pos[r] = s.nk - s.nq + row / p.group;
        slope[r] = p.slopes ? __ldg(p.slopes + kv * p.group + row % p.group) : 0.f;
        most[r] = -INFINITY, sum[r] = 0.f, o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int n = 0; n < mine; ++n) {
        const int j = ch.keys.tile(first + warp + n * WARPS) * KEYS + key;
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        float x[ROWS] = {};
#pragma unroll 2
        for (int d = half * (D / 2); d < (half + 1) * (D / 2); d += 4) {
            const float4 a = *reinterpret_cast<const float4 *>(sk + key * stride + d);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) x[r] = dev::dot4(*reinterpret_cast<const float4 *>(sq + r * D + d), a, x[r]);
        }
        __syncwarp();
        fetch(n + 1, K, p.k.row, sk);
        float now[ROWS];
        bool more = false;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            x[r] += __shfl_xor_sync(0xffffffffu, x[r], 16);
            float unused;
            const float z = score(p, slope[r], x[r], pos[r], j, unused);
            x[r] = key_seen(p.window, s, pos[r], j) ? z : -INFINITY;
            now[r] = x[r];
        }
#pragma unroll
        for (int q = 8; q >= 1; q >>= 1)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) now[r] = fmaxf(now[r], __shfl_xor_sync(0xffffffffu, now[r], q));
#pragma unroll
        for (int r = 0; r < ROWS; ++r) more = more || now[r] > most[r];
        if (more) {  // (the same in all lanes)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                now[r] = fmaxf(now[r], most[r]);
                const float shrink = now[r] == most[r] ? 1.f : exp2f((most[r] - now[r]) * LOG2E);
                sum[r] *= shrink;
                o[r].x *= shrink, o[r].y *= shrink, o[r].z *= shrink, o[r].w *= shrink;
                most[r] = now[r];
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            x[r] = exp2f((x[r] - (most[r] == -INFINITY ? 0.f : most[r])) * LOG2E);
            sum[r] += x[r];
            if (half == 0) w_p[warp][key][r] = x[r];
        }
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        if (column < D) {
#pragma unroll 4
            for (int u = 0; u < KEYS; ++u) {
                const float4 y = *reinterpret_cast<const float4 *>(sv + u * stride + column);
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    const float w = w_p[warp][u][r];
                    o[r].x = fmaf(w, y.x, o[r].x), o[r].y = fmaf(w, y.y, o[r].y), o[r].z = fmaf(w, y.z, o[r].z), o[r].w = fmaf(w, y.w, o[r].w);
                }
            }
        }
        __syncwarp();
        fetch(n + 1, V, p.v.row, sv);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // the warps' parts, in order
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
#pragma unroll
        for (int q = 8; q >= 1; q >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], q);
        if (lane == 0) w_most[warp][r] = most[r], w_sum[warp][r] = sum[r];
    }
    __syncthreads();  // (all rings are done with, too)
    float *const parts = sm;  // WARPS x ROWS x D
    if (column < D)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int v = 0; v < WARPS; ++v) top = fmaxf(top, w_most[v][r]);
            const float by = most[r] == -INFINITY ? 0.f : exp2f((most[r] - top) * LOG2E);
            *reinterpret_cast<float4 *>(parts + (warp * ROWS + r) * D + column) = make_float4(o[r].x * by, o[r].y * by, o[r].z * by, o[r].w * by);
        }
    __syncthreads();
    const bool last = ch.n == 1;
    if (const int r = warp; r < ROWS && r0 + r < rows) {
        const int i = (r0 + r) / p.group, head = kv * p.group + (r0 + r) % p.group;
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) top = fmaxf(top, w_most[v][r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) total += w_sum[v][r] * exp2f((w_most[v][r] - base) * LOG2E);
        const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : NAN;
        const float lse2 = total == 0.f ? -INFINITY : base * LOG2E + log2f(total), lse = total == 0.f ? -INFINITY : base + logf(total);
        const int64_t at = ((int64_t)s.q0 + i) * p.q_heads + head;
        bool wrong = false;
        for (int d = lane; d < D; d += 32) {
            float y = 0.f;
#pragma unroll
            for (int v = 0; v < WARPS; ++v) y += parts[(v * ROWS + r) * D + d];
            y *= inv;
            if (last) {
                wrong = wrong || !isfinite(y);
                static_cast<float *>(p.o.data)[((int64_t)s.q0 + i) * p.o.row + head * p.o.head + d] = y;
            } else {
                p.part_o[(chunk * (int64_t)p.q_rows * p.q_heads + at) * D + d] = y;
            }
        }
        if (lane == 0) {
            if (!last) p.part_lse[chunk * (int64_t)p.q_rows * p.q_heads + at] = lse2;
            else if (p.lse) p.lse[(int64_t)head * p.q_rows + s.q0 + i] = lse;
        }
        if (__any_sync(0xffffffffu, wrong)) {
            __syncwarp();
            strict::output_row<float>(p, s, head, i, lse);
        }
    }
}

size_t smem_of(int rows, int D)
{
    const size_t tiles = (size_t)rows * D + (size_t)WARPS * 2 * KEYS * (D + 4), parts = (size_t)WARPS * rows * D;
    return (tiles > parts ? tiles : parts) * sizeof(float);
}
bool wide(const HeadArray &a) { return (uintptr_t)a.data % 16 == 0 && a.row % 4 == 0 && a.head % 4 == 0; }

template <int ROWS>
cudaError_t launch(const AttentionParams &p, cudaStream_t s)
{
    static SmemOptinCache optin;
    const cudaError_t e = optin_dynamic_smem(attention_few_f32_kernel<ROWS>, smem_of(ROWS, 128), optin);
    if (e != cudaSuccess) return e;
    const int row_tiles = (int)(((int64_t)p.max_q * p.group + ROWS - 1) / ROWS);
    const unsigned grid = (unsigned)((int64_t)p.n_seqs * p.kv_heads * row_tiles * p.n_splits);
    attention_few_f32_kernel<ROWS><<<grid, WARPS * 32, smem_of(ROWS, p.head_dim), s>>>(p, row_tiles);
    return cudaGetLastError();
}

}  // namespace

ForwardPlan plan_attention_few_f32(const AttentionParams &p, int sm_count)
{
    if (p.dtype != 0) return ForwardPlan{0, 1, 0, INFINITY};
    const int rows = few_rows_f32(p), resident = rows <= 4 && p.head_dim <= 64 ? 2 : 1;
    // (Two tiles a warp at least; four: a token of 32 / 8 heads over 8,000 keys 27 -> 33 us)
    ForwardPlan f = plan_few(p, rows, KEYS, WARPS, 2 * WARPS, resident, sm_count);
    if (f.n_splits == 0) return f;
    // A block begins and ends in 5 us; its warps' 16 keys of 64 columns take 1.2, and 0.33 a row.  A join takes 6.
    const double tiles = (double)((p.max_k + KEYS - 1) / KEYS + 1), blocks = f.us / tiles * f.n_splits;
    const double steps = ceil((tiles < f.chunk_tiles ? tiles : f.chunk_tiles) / WARPS);
    f.us = 3. + ceil(blocks / (resident * sm_count)) * (5. + steps * (1.2 + 0.33 * rows) * (p.head_dim <= 64 ? 1. : 1.7)) + (f.n_splits > 1 ? 6. : 0.);
    return f;
}

cudaError_t launch_attention_few_f32(const AttentionParams &p0, const ForwardPlan &f, void *workspace, bool *taken, cudaStream_t s)
{
    *taken = f.n_splits > 0 && wide(p0.k) && wide(p0.v);
    if (!*taken) return cudaSuccess;
    AttentionParams p = p0;
    p.n_splits = f.n_splits;
    p.chunk_tiles = f.chunk_tiles;
    p.part_o = static_cast<float *>(workspace);
    p.part_lse = p.part_o + (f.n_splits == 1 ? 0 : (int64_t)f.n_splits * p.q_rows * p.q_heads * p.head_dim);
    const int rows = few_rows_f32(p);
    const cudaError_t e = rows == 1 ? launch<1>(p, s) : rows == 2 ? launch<2>(p, s) : rows == 4 ? launch<4>(p, s) : launch<8>(p, s);
    return e == cudaSuccess && p.n_splits > 1 ? launch_attention_join(p, JOIN_FEW_F32, s) : e;
}

}  // namespace sddmm
