// Attention, forward, for few queries of many keys (single tokens over a cache), fp16 and bfloat16.
//
// The query heads of a group read the same keys and values, so a row here is a (query, head) pair of one KV head, query by query, and 16
// rows are one tile of the matrix instruction (mma.sync m16n8k16: 16 rows would leave seven eighths of a tcgen05 tile empty, and the
// memory, not the tensor core, is what bounds this).  The keys that the rows see are cut into chunks, a block each: many blocks however
// few the sequences.  A block is four warps; a warp takes every fourth tile of 16 keys of the chunk, copies K and V rows into a ring of
// its own in shared memory (16-byte asynchronous copies, zeros behind the sequence's end, three stages), keeps maximum, sum and
// output in registers, and waits for no other warp before the end.  The warps' parts are added in order; where a sequence has several
// chunks the parts go to the workspace and a second kernel, a block for each row, adds them in order.  Nothing depends on scheduling.
//
// What bounds it: memory in the middle, beginning, end and join around it (10 us).  One token on 32,801 keys, 32 / 8 heads of 128, bfloat16: 30.7 us,
// 4.4 TB/s; 32 tokens on 4,000 each, 8 heads: 95 us, 5.5 TB/s.
#include <cmath>
#include <type_traits>

#include "attention_strict.cuh"
#include "device_utils.cuh"
#include "tc_utils.cuh"

namespace sddmm {

namespace {

constexpr int KEYS = FEW_KEYS, WARPS = 4, STAGES = 3, ROWS = FEW_ROWS;
constexpr float RAISE = 8.f;
constexpr int MOST_TILES = 16;  // of a warp, in one chunk
constexpr int resident_blocks(int head_dim) { return head_dim <= 64 ? 4 : 2; }  // of a multiprocessor, by registers

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <class E>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<E, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class E> __device__ __forceinline__ float2 unpack(uint32_t x)
{
    return std::is_same<E, __half>::value ? __half22float2(reinterpret_cast<const __half2 &>(x)) : __bfloat1622float2(reinterpret_cast<const __nv_bfloat162 &>(x));
}

template <class E, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(WARPS * 32, resident_blocks(DP)) attention_few_kernel(const AttentionParams p, int row_tiles)
{
    constexpr int ROW_BYTES = DP * 2, PIECES = DP / 8, TILE_BYTES = KEYS * ROW_BYTES, STAGE_BYTES = 2 * TILE_BYTES;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ float w_most[WARPS][ROWS], w_sum[WARPS][ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // first chunks first: those that a short sequence does not have come last
    const unsigned heads_and_rows = gridDim.x / p.n_splits, b = blockIdx.x % heads_and_rows, chunk = blockIdx.x / heads_and_rows;
    const int tile = b % row_tiles, kv = b / row_tiles % p.kv_heads, seq = b / row_tiles / p.kv_heads;
    const Sequence s = sequence_of(p, seq);
    const int rows = s.nq * p.group, r0 = tile * ROWS;
    if (r0 >= rows) return;
    const Chunks<KEYS> ch = chunks_of<KEYS>(p, s, tile, ROWS);
    if ((int)chunk >= ch.n) return;
    const int first = chunk * p.chunk_tiles, end = min(ch.keys.n, first + p.chunk_tiles);
    const int D = p.head_dim;
    if (p.n_splits > 1) next_kernel_may_come();

    // ---- the ring: this warp's tiles first + warp, + 4, ... ----
    const int mine = max(0, (end - first - warp + WARPS - 1) / WARPS);
    const uint32_t ring = dev::smem_u32(smem) + warp * STAGES * STAGE_BYTES;
    const E *K = static_cast<const E *>(p.k.data) + (int64_t)s.k0 * p.k.row + kv * p.k.head;
    const E *V = static_cast<const E *>(p.v.data) + (int64_t)s.k0 * p.v.row + kv * p.v.head;
    auto fetch = [&](int n) {
        if (n < mine) {
            const int j0 = ch.keys.tile(first + warp + n * WARPS) * KEYS;
            const uint32_t at = ring + n % STAGES * STAGE_BYTES;
#pragma unroll
            for (int i = 0; i < KEYS * PIECES / 32; ++i) {
                const int f = i * 32 + lane, r = f / PIECES, c = f % PIECES, j = j0 + r;
                const int bytes = j < s.nk && c * 8 < D ? 16 : 0;
                const uint32_t to = at + r * ROW_BYTES + (c ^ (r & 7)) * 16;
                const int64_t row = bytes ? j : 0;
                const int col = bytes ? c * 8 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(K + row * p.k.row + col), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + TILE_BYTES), "l"(V + row * p.v.row + col), "r"(bytes) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int n = 0; n < STAGES - 1; ++n) fetch(n);

    // ---- Q: this thread's two rows, lane / 4 and 8 further ----
    uint32_t q[DP / 16][4];
    int lo[2], hi[2], pos[2];
    float slope[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int r = min(r0 + lane / 4 + 8 * x, rows - 1), i = r / p.group, head = kv * p.group + r % p.group;
        const E *src = static_cast<const E *>(p.q.data) + ((int64_t)s.q0 + i) * p.q.row + head * p.q.head;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int d = 16 * k + 8 * y + lane % 4 * 2;
                q[k][x + 2 * y] = d < D ? *reinterpret_cast<const uint32_t *>(src + d) : 0u;
            }
        pos[x] = s.nk - s.nq + i;
        lo[x] = p.window.left < 0 ? 0 : max(0, pos[x] - p.window.left);
        hi[x] = p.window.right < 0 ? s.nk - 1 : min(s.nk - 1, pos[x] + p.window.right);
        slope[x] = BIAS ? __ldg(p.slopes + head) * LOG2E : 0.f;
    }
    const float c = !CAP ? p.scale * LOG2E : p.of_cap, top_of = p.cap * LOG2E;
    const tc::Tanh tanh_c = tc::tanh_polynomial(c, top_of);
    float o[DP / 8][4];
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
    float most[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

    for (int n = 0; n < mine; ++n) {
        fetch(n + STAGES - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        const int j0 = ch.keys.tile(first + warp + n * WARPS) * KEYS;
        const uint32_t at = ring + n % STAGES * STAGE_BYTES;
        float x[2][4] = {};
        {
            const int r = lane / 16 * 8 + lane % 8, h = lane / 8 & 1;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                uint32_t m[4];
                ldmatrix4(m, at + r * ROW_BYTES + ((2 * k + h) ^ (r & 7)) * 16);
                mma<E>(x[0], q[k], m[0], m[1]);
                mma<E>(x[1], q[k], m[2], m[3]);
            }
        }
        const bool open = tile_is_open<KEYS>(p.window, s, ch.reach, j0);
        if (CAP) {
            float size = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) size = tc::max3_abs(size, x[0][e], x[1][e]);
            if (p.pre == 1.f && __all_sync(0xffffffffu, size <= tanh_c.range)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) tc::split(tc::tanh2(tc::two(x[0][e], x[1][e]), tanh_c), x[0][e], x[1][e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) tc::split(tc::tanh_any(tc::two(x[0][e] * p.pre, x[1][e] * p.pre), tanh_c, c, top_of, 0.f), x[0][e], x[1][e]);
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int w = e >> 1, j = j0 + 8 * t + lane % 4 * 2 + (e & 1);
                float z = x[t][e];
                if (!CAP) z *= c;
                if (BIAS) z = fmaf(-slope[w], fabsf((float)(pos[w] - j)), z);
                if (!open && !(j < s.prefix || (j >= lo[w] && j <= hi[w]))) z = -INFINITY;
                x[t][e] = z;
            }
        uint32_t pw[4], rest[4];  // weights, rounded, and what the rounding left: a second product, at hardly a cost beside memory
                                  // (24 tokens 34.0 -> 36.6 us, four 30.7 -> 30.7; the results' error 1.15 -> 1.00 times their own rounding)
        float now[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            now[w] = fmaxf(fmaxf(x[0][2 * w], x[0][2 * w + 1]), fmaxf(x[1][2 * w], x[1][2 * w + 1]));
            now[w] = fmaxf(now[w], __shfl_xor_sync(0xffffffffu, now[w], 1));
            now[w] = fmaxf(now[w], __shfl_xor_sync(0xffffffffu, now[w], 2));
        }
        if (__any_sync(0xffffffffu, now[0] > most[0] + RAISE || now[1] > most[1] + RAISE)) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const bool raise = now[w] > most[w] + RAISE;
                const float shrink = raise ? tc::ex2(most[w] - now[w]) : 1.f;
                if (raise) most[w] = now[w];
                sum[w] *= shrink;
#pragma unroll
                for (int d = 0; d < DP / 8; ++d) o[d][2 * w] *= shrink, o[d][2 * w + 1] *= shrink;
            }
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const float less = most[w] == -INFINITY ? 0.f : most[w];
            float e[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) e[u] = tc::ex2(x[u >> 1][2 * w + (u & 1)] - less);
            sum[w] += (e[0] + e[1]) + (e[2] + e[3]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                pw[w + 2 * u] = tc::pack<E>(e[2 * u], e[2 * u + 1]);
                const float2 y = unpack<E>(pw[w + 2 * u]);
                rest[w + 2 * u] = tc::pack<E>(e[2 * u] - y.x, e[2 * u + 1] - y.y);
            }
        }
        {
            const int r = lane & 15, h = lane >> 4;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t m[4];
                ldmatrix4_t(m, at + TILE_BYTES + r * ROW_BYTES + ((2 * d + h) ^ (r & 7)) * 16);
                mma<E>(o[2 * d], pw, m[0], m[1]);
                mma<E>(o[2 * d + 1], pw, m[2], m[3]);
                mma<E>(o[2 * d], rest, m[0], m[1]);
                mma<E>(o[2 * d + 1], rest, m[2], m[3]);
            }
        }
        __syncwarp();  // the stage may be filled again
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the four warps' parts ----
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 1);
        sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 2);
        if (lane % 4 == 0) w_most[warp][lane / 4 + 8 * w] = most[w], w_sum[warp][lane / 4 + 8 * w] = sum[w];
    }
    __syncthreads();  // (all rings are done with, too)
    float *const parts = reinterpret_cast<float *>(smem);  // WARPS x ROWS x (DP + 4)
    constexpr int PITCH = DP + 4;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const int r = lane / 4 + 8 * w;
        float top = -INFINITY;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) top = fmaxf(top, w_most[v][r]);
        const float by = most[w] == -INFINITY ? 0.f : tc::ex2(most[w] - top);
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
            *reinterpret_cast<float2 *>(parts + (warp * ROWS + r) * PITCH + 8 * d + lane % 4 * 2) = make_float2(o[d][2 * w] * by, o[d][2 * w + 1] * by);
    }
    __syncthreads();
    const bool last = ch.n == 1;
#pragma unroll
    for (int x = 0; x < ROWS / WARPS; ++x) {
        const int r = warp + x * WARPS;
        if (r0 + r >= rows) break;
        const int i = (r0 + r) / p.group, head = kv * p.group + (r0 + r) % p.group;
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) top = fmaxf(top, w_most[v][r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) total += w_sum[v][r] * tc::ex2(w_most[v][r] - base);
        const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : NAN;
        const float lse2 = total == 0.f ? -INFINITY : base + log2f(total);
        const int64_t at = ((int64_t)s.q0 + i) * p.q_heads + head;
        bool wrong = false;
        for (int d = 2 * lane; d < D; d += 64) {
            float2 y = make_float2(0.f, 0.f);
#pragma unroll
            for (int v = 0; v < WARPS; ++v) {
                const float2 z = *reinterpret_cast<const float2 *>(parts + (v * ROWS + r) * PITCH + d);
                y.x += z.x, y.y += z.y;
            }
            y.x *= inv, y.y *= inv;
            if (last) {
                wrong = wrong || !isfinite(y.x) || !isfinite(y.y);
                *reinterpret_cast<uint32_t *>(static_cast<E *>(p.o.data) + ((int64_t)s.q0 + i) * p.o.row + head * p.o.head + d) = tc::pack<E>(y.x, y.y);
            } else {
                *reinterpret_cast<float2 *>(p.part_o + (chunk * (int64_t)p.q_rows * p.q_heads + at) * D + d) = y;
            }
        }
        if (lane == 0) {
            if (!last) p.part_lse[chunk * (int64_t)p.q_rows * p.q_heads + at] = lse2;
            else if (p.lse) p.lse[(int64_t)head * p.q_rows + s.q0 + i] = lse2 * LN2;
        }
        if (__any_sync(0xffffffffu, wrong)) {
            __syncwarp();
            strict::output_row<E>(p, s, head, i, lse2 * LN2);
        }
    }
}

// The parts of one row added up, a block for a row: warps take chunks in turn, eight at once, so that all of a row's parts are asked for
// before the first is used.
template <class E, JoinOf OF>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttentionParams p)
{
    constexpr int JOIN_WARPS = 8, AT_ONCE = 8;
    __shared__ float part[JOIN_WARPS][128], w_most[JOIN_WARPS], w_sum[JOIN_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.head_dim;
    const int head = blockIdx.x % p.q_heads, i = blockIdx.x / p.q_heads % p.max_q, seq = blockIdx.x / p.q_heads / p.max_q;
    const Sequence s = sequence_of(p, seq);
    int n = 0;
    if (i >= s.nq) {
    } else if (OF == JOIN_PROMPT || OF == JOIN_GENERAL) {
        constexpr int ROWS_OF = OF == JOIN_PROMPT ? PROMPT_QUERIES : GENERAL_ROWS, KEYS_OF = OF == JOIN_PROMPT ? PROMPT_KEYS : GENERAL_ROWS;
        const int i0 = i / ROWS_OF * ROWS_OF;
        n = (key_tiles<KEYS_OF>(reach_of(p.window, s, i0, min(s.nq, i0 + ROWS_OF))).n + p.chunk_tiles - 1) / p.chunk_tiles;
    } else {
        const int rows = OF == JOIN_FEW ? FEW_ROWS : few_rows_f32(p);
        n = chunks_of<OF == JOIN_FEW ? FEW_KEYS : FEW_F32_KEYS>(p, s, (i * p.group + head % p.group) / rows, rows).n;
    }
    behind_last_kernel();
    if (n <= 1) return;
    const int64_t stride = (int64_t)p.q_rows * p.q_heads, at = ((int64_t)s.q0 + i) * p.q_heads + head;
    float y[4] = {}, top = -INFINITY, total = 0.f;
    for (int c0 = warp; c0 < n; c0 += JOIN_WARPS * AT_ONCE) {
        float l[AT_ONCE];
        float4 v[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int c = c0 + k * JOIN_WARPS;
            l[k] = c < n ? p.part_lse[c * stride + at] : -INFINITY;
            v[k] = c < n && 4 * lane < D ? *reinterpret_cast<const float4 *>(p.part_o + (c * stride + at) * D + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float now = top;
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) now = fmaxf(now, l[k]);
        const float base = now == -INFINITY ? 0.f : now, shrink = tc::ex2(top - base);
        top = now;
        total *= shrink;
#pragma unroll
        for (int x = 0; x < 4; ++x) y[x] *= shrink;
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const float w = tc::ex2(l[k] - base);
            total += w;
            y[0] = fmaf(w, v[k].x, y[0]), y[1] = fmaf(w, v[k].y, y[1]), y[2] = fmaf(w, v[k].z, y[2]), y[3] = fmaf(w, v[k].w, y[3]);
        }
    }
    *reinterpret_cast<float4 *>(&part[warp][4 * lane]) = make_float4(y[0], y[1], y[2], y[3]);
    if (lane == 0) w_most[warp] = top, w_sum[warp] = total;
    __syncthreads();
    if (warp != 0) return;
    top = -INFINITY;
#pragma unroll
    for (int v = 0; v < JOIN_WARPS; ++v) top = fmaxf(top, w_most[v]);
    const float base = top == -INFINITY ? 0.f : top;
    float by[JOIN_WARPS];
    total = 0.f;
#pragma unroll
    for (int v = 0; v < JOIN_WARPS; ++v) {
        by[v] = tc::ex2(w_most[v] - base);
        total += by[v] * w_sum[v];
    }
    const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : NAN;
    const float lse = total == 0.f ? -INFINITY : (base + log2f(total)) * LN2;
    bool wrong = false;
    for (int d = lane; d < D; d += 32) {
        float x = 0.f;
#pragma unroll
        for (int v = 0; v < JOIN_WARPS; ++v) x = fmaf(by[v], part[v][d], x);
        x *= inv;
        wrong = wrong || !isfinite(x);
        static_cast<E *>(p.o.data)[((int64_t)s.q0 + i) * p.o.row + head * p.o.head + d] = from_f<E>(x);
    }
    if (p.lse && lane == 0) p.lse[(int64_t)head * p.q_rows + s.q0 + i] = lse;
    if (__any_sync(0xffffffffu, wrong)) {
        __syncwarp();
        strict::output_row<E>(p, s, head, i, lse);
    }
}

template <class E, JoinOf OF>
cudaError_t launch_join(const AttentionParams &p, cudaStream_t s)
{
    // (24 tokens: 37 us as an ordinary launch, 33 so)
    return launch_behind(attention_join_kernel<E, OF>, (unsigned)((int64_t)p.n_seqs * p.max_q * p.q_heads), 256, 0, s, p);
}

template <class E, int DP, bool CAP, bool BIAS>
cudaError_t launch(const AttentionParams &p, cudaStream_t s)
{
    constexpr size_t ring = (size_t)WARPS * STAGES * 2 * KEYS * DP * 2, parts = (size_t)WARPS * ROWS * (DP + 4) * 4;
    constexpr size_t smem = ring > parts ? ring : parts;
    static SmemOptinCache optin;
    cudaError_t e = optin_dynamic_smem(attention_few_kernel<E, DP, CAP, BIAS>, smem, optin);
    if (e != cudaSuccess) return e;
    const int row_tiles = (int)(((int64_t)p.max_q * p.group + ROWS - 1) / ROWS);
    const unsigned grid = (unsigned)((int64_t)p.n_seqs * p.kv_heads * row_tiles * p.n_splits);
    attention_few_kernel<E, DP, CAP, BIAS><<<grid, WARPS * 32, smem, s>>>(p, row_tiles);
    e = cudaGetLastError();
    if (e != cudaSuccess || p.n_splits == 1) return e;
    return launch_join<E, JOIN_FEW>(p, s);
}
template <class E, int DP>
cudaError_t by_score(const AttentionParams &p, cudaStream_t s)
{
    if (p.cap > 0.f) return p.slopes ? launch<E, DP, true, true>(p, s) : launch<E, DP, true, false>(p, s);
    return p.slopes ? launch<E, DP, false, true>(p, s) : launch<E, DP, false, false>(p, s);
}

bool wide(const HeadArray &a) { return (uintptr_t)a.data % 16 == 0 && a.row % 8 == 0 && a.head % 8 == 0; }

}  // namespace

ForwardPlan plan_few(const AttentionParams &p, int rows, int keys, int warps, int least, int resident_of_one, int sm_count)
{
    ForwardPlan f{0, 1, 0, INFINITY};
    if (p.max_q == 0 || p.n_seqs == 0 || (int64_t)p.max_q * p.group > INT32_MAX) return f;
    const int64_t row_tiles = ((int64_t)p.max_q * p.group + rows - 1) / rows, blocks = row_tiles * p.kv_heads * p.n_seqs;
    const int64_t tiles = (p.max_k + keys - 1) / keys + 1;  // (+ 1: prefix and window may begin inside tiles)
    auto bytes_of = [&](int64_t n) { return n == 1 ? 0 : n * p.q_rows * p.q_heads * (int64_t)(p.head_dim + 1) * 4; };
    auto n_of = [&](int64_t c) { return tiles <= c ? (int64_t)1 : (tiles + c - 1) / c; };
    // As many chunks as fill whole waves of resident blocks, of MOST_TILES key tiles a warp at most: longer ones leave the last block of ragged
    // sequences alone, shorter ones spend their time beginning and ending.
    const int64_t most = warps * MOST_TILES, resident = (int64_t)resident_of_one * sm_count, waves = (tiles * blocks + resident * most - 1) / (resident * most);
    const int64_t want = resident * waves / blocks > 1 ? resident * waves / blocks : 1;
    int64_t chunk = ((tiles + want - 1) / want + warps - 1) / warps * warps;
    if (chunk < least) chunk = least;
    while (n_of(chunk) > 1 && bytes_of(n_of(chunk)) > (1ll << 30)) chunk *= 2;
    const int64_t n = n_of(chunk);
    if (n * blocks > INT32_MAX || (int64_t)p.n_seqs * p.max_q * p.q_heads > INT32_MAX) return f;
    f.chunk_tiles = (int)chunk;
    f.n_splits = (int)n;
    f.bytes = bytes_of(n);
    // rows of the sequences, not of the longest
    const int64_t most_rows = p.n_seqs * row_tiles, all_rows = p.q_rows * p.group / rows + p.n_seqs;
    f.us = (double)(all_rows < most_rows ? all_rows : most_rows) * p.kv_heads * tiles;
    return f;
}

ForwardPlan plan_attention_few_tc(const AttentionParams &p, int sm_count)
{
    if (p.dtype == 0) return ForwardPlan{0, 1, 0, INFINITY};
    ForwardPlan f = plan_few(p, ROWS, KEYS, WARPS, 4 * WARPS, resident_blocks(p.head_dim), sm_count);
    // (8 us, and 0.19 for 16 rows x 16 keys on a multiprocessor, however many warps it has; 6 more with a join)
    f.us = 8. + 0.19 * f.us / sm_count + (f.n_splits > 1 ? 6. : 0.);
    return f;
}

cudaError_t launch_attention_join(const AttentionParams &p, JoinOf of, cudaStream_t s)
{
    if (p.dtype == 0) return of == JOIN_GENERAL ? launch_join<float, JOIN_GENERAL>(p, s) : launch_join<float, JOIN_FEW_F32>(p, s);
    if (of == JOIN_PROMPT) return p.dtype == 1 ? launch_join<__half, JOIN_PROMPT>(p, s) : launch_join<__nv_bfloat16, JOIN_PROMPT>(p, s);
    return p.dtype == 1 ? launch_join<__half, JOIN_FEW>(p, s) : launch_join<__nv_bfloat16, JOIN_FEW>(p, s);
}

cudaError_t launch_attention_few_tc(const AttentionParams &p0, const ForwardPlan &f, void *workspace, bool *taken, cudaStream_t s)
{
    *taken = f.n_splits > 0 && wide(p0.q) && wide(p0.k) && wide(p0.v) && wide(p0.o);
    if (!*taken) return cudaSuccess;
    AttentionParams p = p0;
    p.n_splits = f.n_splits;
    p.chunk_tiles = f.chunk_tiles;
    p.part_o = static_cast<float *>(workspace);
    p.part_lse = p.part_o + (f.n_splits == 1 ? 0 : (int64_t)f.n_splits * p.q_rows * p.q_heads * p.head_dim);
    if (p.dtype == 1) return p.head_dim <= 64 ? by_score<__half, 64>(p, s) : by_score<__half, 128>(p, s);
    return p.head_dim <= 64 ? by_score<__nv_bfloat16, 64>(p, s) : by_score<__nv_bfloat16, 128>(p, s);
}

}  // namespace sddmm
