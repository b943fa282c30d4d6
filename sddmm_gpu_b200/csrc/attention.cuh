// Attention over a mask that is described, not listed: what its kernels share.
//
//   s_ij   = cap tanh(scale q_i.k_j / cap) - slope_h |pos_i - j|,   pos_i = n_k - n_q + i
//   seen   : j < prefix, or pos_i - left <= j <= pos_i + right
//   lse_i  = log sum_j exp s_ij,   O_i = sum_j exp(s_ij - lse_i) V_j;   nothing seen: O_i = 0, lse_i = -inf
//
// for the queries i and keys j of one sequence of a batch.  Sequences lie one behind the other in Q, and packed or in slots in K and
// V; offsets and lengths are read on the device, and a sequence whose numbers leave the arrays or the plan's limits is
// left out and reported.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "attention_mask.hpp"
#include "common.cuh"

namespace sddmm {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct HeadArray {  // rows x heads x head_dim, the last dimension contiguous
    void *data;
    int64_t row, head;  // strides in elements
};

struct AttentionParams {
    int n_seqs, q_heads, kv_heads, group, head_dim, dtype;
    int max_q, max_k;
    int64_t q_rows, k_rows;
    float scale, cap;  // cap 0: none
    Window window;
    const int32_t *q_offsets, *k_offsets, *k_len, *prefix;
    const float *slopes;
    HeadArray q, k, v, o, d_o, dq, dk, dv;
    float *lse;    // q_heads x q_rows
    float *delta;  // q_heads x q_rows, workspace of the backward pass
    float *d_o_most;  // the same, fp16: the largest |dO| of every tile of queries of a head (tile_index())
    float *part_o, *part_lse;  // parts of a split long axis (workspace)
    int n_splits, chunk_tiles;  // chunks of the keys, at most; key tiles of one
    int *status;
    float of_cap, pre;  // tensor-core kernels: scale / cap, and 1; where it is out of tanh_polynomial()'s reach 1, and that, as a first factor of the products
};

__device__ __forceinline__ void report_bad_index(int *dev_status)
{
    reinterpret_cast<volatile int *>(dev_status)[BAD_INDEX_WORD] = (int)DEV_BAD_INDEX;
    __threadfence_system();
}

// Sequence b; one whose numbers are not good (negative, outside the arrays, above the plan's limits) counts as empty.
__device__ __forceinline__ Sequence sequence_of(const AttentionParams &p, int b)
{
    Sequence s;
    s.q0 = __ldg(p.q_offsets + b);
    s.nq = __ldg(p.q_offsets + b + 1) - s.q0;
    const int32_t *ko = p.k_offsets ? p.k_offsets : p.q_offsets;
    s.k0 = __ldg(ko + b);
    const int room = __ldg(ko + b + 1) - s.k0;
    s.nk = p.k_len ? __ldg(p.k_len + b) : room;
    s.prefix = p.prefix ? max(0, min(__ldg(p.prefix + b), s.nk)) : 0;
    const bool good = s.q0 >= 0 && s.nq >= 0 && s.nq <= p.max_q && (int64_t)s.q0 + s.nq <= p.q_rows && s.k0 >= 0 && s.nk >= 0 &&
                      s.nk <= room && s.nk <= p.max_k && (int64_t)s.k0 + s.nk <= p.k_rows;
    if (!good) {
        report_bad_index(p.status);
        s.q0 = s.nq = s.k0 = s.nk = s.prefix = 0;
    }
    return s;
}

// Block `index` of ceil(n / T) blocks per sequence, over all sequences: its sequence and its number there.  Returns false behind
// the last one.  keys: blocks of keys, else of queries.  All threads of a warp call it together.
template <int T>
__device__ __forceinline__ bool find_block(const AttentionParams &p, int index, bool keys, Sequence &s, int &seq, int &number)
{
    const int lane = threadIdx.x & 31;
    int before = 0;
    auto among = [&](const Sequence &mine, int b0) {  // the 32 sequences from b0 on, one a lane
        const int blocks = ((keys ? mine.nk : mine.nq) + T - 1) / T;
        int sum = blocks;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, index < before + sum);
        if (!hit) {
            before += __shfl_sync(0xffffffffu, sum, 31);
            return false;
        }
        const int l = __ffs(hit) - 1;
        number = index - before - __shfl_sync(0xffffffffu, sum - blocks, l);
        seq = b0 + l;
        s.q0 = __shfl_sync(0xffffffffu, mine.q0, l);
        s.nq = __shfl_sync(0xffffffffu, mine.nq, l);
        s.k0 = __shfl_sync(0xffffffffu, mine.k0, l);
        s.nk = __shfl_sync(0xffffffffu, mine.nk, l);
        s.prefix = __shfl_sync(0xffffffffu, mine.prefix, l);
        return true;
    };
    if (p.n_seqs <= 32) {
        Sequence mine = {};
        if (lane < p.n_seqs) mine = sequence_of(p, lane);
        return among(mine, 0);
    }
    constexpr int AT_ONCE = 4;  // groups whose numbers are asked for together
    for (int b0 = 0; b0 < p.n_seqs; b0 += 32 * AT_ONCE) {
        Sequence of[AT_ONCE] = {};
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x)
            if (b0 + 32 * x + lane < p.n_seqs) of[x] = sequence_of(p, b0 + 32 * x + lane);
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x)
            if (among(of[x], b0 + 32 * x)) return true;
    }
    return false;
}
// How a forward kernel cuts the keys (n_splits 1: not, 0: it does not take the call), bytes of the parts, and about how long it takes.
struct ForwardPlan {
    int n_splits, chunk_tiles;
    int64_t bytes;
    double us;
};
ForwardPlan plan_attention_few_tc(const AttentionParams &p, int sm_count);
ForwardPlan plan_attention_forward_tc(const AttentionParams &p, int sm_count);
// *taken false, and nothing launched, where the call's type, strides or alignment do not allow the kernel.
cudaError_t launch_attention_few_tc(const AttentionParams &p, const ForwardPlan &f, void *workspace, bool *taken, cudaStream_t s);
cudaError_t launch_attention_forward_tc(const AttentionParams &p, const ForwardPlan &f, void *workspace, bool *taken, cudaStream_t s);
ForwardPlan plan_attention_few_f32(const AttentionParams &p, int sm_count);
cudaError_t launch_attention_few_f32(const AttentionParams &p, const ForwardPlan &f, void *workspace, bool *taken, cudaStream_t s);
// For the kernels of few rows: how the keys are cut for blocks of `rows` rows and `warps` warps, in tiles of `keys` keys, `least` of them or more, with
// `resident` blocks on a multiprocessor.  (us here: the units of rows x keys in all.)
ForwardPlan plan_few(const AttentionParams &p, int rows, int keys, int warps, int least, int resident, int sm_count);
constexpr int FEW_ROWS = 16, FEW_KEYS = 16, FEW_F32_KEYS = 16;
// Rows of a block in fp32.
__host__ __device__ inline int few_rows_f32(const AttentionParams &p)
{
    const int64_t rows = (int64_t)p.max_q * p.group;
    return rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
}
// The chunks that the keys of row tile `tile` of such a kernel are cut into.
template <int KEYS> struct Chunks {
    KeyTiles keys;
    Reach reach;
    int n;
};
template <int KEYS>
__device__ __forceinline__ Chunks<KEYS> chunks_of(const AttentionParams &p, const Sequence &s, int tile, int rows)
{
    const int r0 = tile * rows, r1 = min(r0 + rows, s.nq * p.group);
    Chunks<KEYS> c;
    c.reach = reach_of(p.window, s, r0 / p.group, (r1 - 1) / p.group + 1);
    c.keys = key_tiles<KEYS>(c.reach);
    c.n = max(1, (c.keys.n + p.chunk_tiles - 1) / p.chunk_tiles);
    return c;
}
// Adds up parts: of the kernels of few rows, of the prompt kernel, whose blocks have 256 queries and go through tiles
// of 128 keys, or of the general one, with 64 of both.
constexpr int PROMPT_QUERIES = 256, PROMPT_KEYS = 128, GENERAL_ROWS = 64;
enum JoinOf { JOIN_FEW, JOIN_PROMPT, JOIN_FEW_F32, JOIN_GENERAL };
cudaError_t launch_attention_join(const AttentionParams &p, JoinOf of, cudaStream_t s);

// Launches of one call behind one another: a kernel is set up while the one before it ends.  Every block of such a kernel calls
// behind_last_kernel() before it touches what that one wrote or reads, and before it ends, so that no grid ends before the one it stands
// behind; the kernel before it calls next_kernel_may_come().
__device__ __forceinline__ void behind_last_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void next_kernel_may_come() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <class... Args, class... Given>
inline cudaError_t launch_behind(void (*kernel)(Args...), unsigned grid, unsigned threads, size_t smem, cudaStream_t s, const Given &...args)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

ForwardPlan plan_attention_forward_general(const AttentionParams &p, int sm_count);
cudaError_t launch_attention_forward_general(const AttentionParams &p, const ForwardPlan &f, void *workspace, cudaStream_t s);
// Where the blocks of a backward kernel alone would leave multiprocessors idle, the tiles that a block goes through are cut into parts, a
// block each, which leave their sums in the workspace (parts x rows x heads x head_dim, dK and dV behind one another) for
// launch_attention_sum_parts().  Most parts of a block, tiles of a part, bytes of the sums (16-byte aligned, p.part_o).
struct Parts {
    int n_q, tiles_q, n_kv, tiles_kv;
    int64_t bytes;
};
constexpr Parts ONE_PART{1, 1 << 30, 1, 1 << 30, 0};
Parts plan_attention_parts(const AttentionParams &p, int tile, int per_sm, int sm_count);
// tile: rows of a block; 64 for fp32, 128 for 16-bit types
cudaError_t launch_attention_sum_parts(const AttentionParams &p, bool kv, int tile, cudaStream_t s);
struct Part {
    int first, end;  // tiles
    bool alone;      // no other part: the block stores its results itself
};
__device__ __forceinline__ Part part_of(const AttentionParams &p, int tiles, int part)
{
    const int each = p.chunk_tiles, n = max(1, (tiles + each - 1) / each);
    return Part{part * each, part < n ? min(tiles, (part + 1) * each) : -1, n == 1};  // (end -1: there is no such part)
}
// The tiles of T queries that see keys [j0, j0 + m): `per_head` from `from` on, for every head of the group.
template <int T>
__device__ __forceinline__ void query_tiles(const AttentionParams &p, const Sequence &s, int j0, int m, int &from, int &per_head)
{
    int to;
    queries_of(p.window, s, j0, j0 + m, from, to);
    from /= T;
    per_head = to > from * T ? (to + T - 1) / T - from : 0;
}
// A place for every tile of 128 queries: q_rows / 128 + n_seqs a head.  (A sequence's last tile is at most as far as the next one's first row, whose own
// tiles lie one further for their sequence's number.)
constexpr int DO_TILE = 128;
__host__ __device__ inline int64_t most_tiles(const AttentionParams &p) { return p.q_rows / DO_TILE + p.n_seqs; }
__device__ __forceinline__ int64_t tile_index(const AttentionParams &p, const Sequence &s, int seq, int head, int tile)
{
    return head * most_tiles(p) + s.q0 / DO_TILE + seq + tile;
}
cudaError_t launch_attention_backward_general(const AttentionParams &p, const Parts &parts, cudaStream_t s);
cudaError_t launch_attention_backward_tc(const AttentionParams &p, const Parts &parts, bool *taken, cudaStream_t s);

}  // namespace sddmm
