// Attention, forward, on the tensor cores (tcgen05), for fp16 and bfloat16.
//
// A block has 256 queries of one head, two tiles of 128, and goes once over the keys in tiles of 128:
//
//   warps 0-3, 4-7  softmax of a tile each, a row a thread: reads its scores from tensor memory, masks them where the tile is not open,
//                   keeps running maximum and sum in registers, writes the weights, rounded to the operands' type, back to tensor memory
//                   over the scores;
//   warp 8          one thread issues S = Q K^T (both operands in shared memory) and O += P V (P in tensor memory, V read as it
//                   lies, MN-major), alternating between the two tiles: one tile's products run under the other's softmax;
//   warp 9          one thread brings Q, K and V by tile copies into a ring of four stages.
//
// The maximum that weights are relative to is only raised when it has grown by more than 2^8: weights then reach 256 at most, which
// neither type minds, and the accumulator in tensor memory is rescaled by hardly any tile.  A tile's next scores come behind its last
// weights' product in the order of issue, so the accumulator is at rest whenever new scores are there.
//
// Rows of K and V behind a sequence's end are another sequence's, or of no sequence: scores of such keys are masked, and such rows of V are
// zeroed in shared memory, since 0 x NaN is NaN.  Hidden places inside the sequence: attention_strict.cuh.
#include "attention_strict.cuh"
#include "tc_utils.cuh"

#include <type_traits>

namespace sddmm {

namespace {

using tc::mbar_arrive;
using tc::mbar_fence_init;
using tc::mbar_init;

constexpr int T = 128;  // queries of a tile, keys of a tile
constexpr int STAGES = 4;
constexpr int SOFTMAX_WARPS = 8, MMA_WARP = 8, LOAD_WARP = 9, THREADS = 384;
constexpr uint32_t TMEM_COLUMNS = 512, O_COLUMN = 256;
constexpr float RAISE = 8.f;
// Registers of a thread: 168 at launch (384 threads), shared out anew: 2 x 216 + 72 = 3 x 168.
#define SOFTMAX_REGISTERS "216"
#define OTHER_REGISTERS "72"

struct alignas(64) Maps {
    CUtensorMap q, k, v;
};

template <class E, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(THREADS, 1) attention_forward_tc_kernel(const AttentionParams p, const __grid_constant__ Maps maps)
{
    constexpr int BOXES = DP / 64, TILE_BYTES = T * DP * 2, BOX_BYTES = T * 128;
    constexpr bool BF16 = sizeof(E) == 2 && !std::is_same<E, __half>::value;
    extern __shared__ __align__(1024) unsigned char smem[];  // Q tiles, then the ring
    __shared__ uint64_t q_full, full[STAGES], empty[STAGES], s_full[2], p_ready[2], o_full[2], tail;
    __shared__ uint32_t tmem_holder;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.x % p.q_heads, kv = head / p.group;
    Sequence s;
    int seq, block;
    // the last blocks of a causal sequence have the most keys: they go first
    if (!find_block<2 * T>(p, (gridDim.x - 1 - blockIdx.x) / p.q_heads, false, s, seq, block)) return;
    const int i0 = block * 2 * T;
    const KeyTiles all = key_tiles<T>(reach_of(p.window, s, i0, min(s.nq, i0 + 2 * T)));
    Reach reach[2];
    bool there[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        there[t] = i0 + t * T < s.nq;
        reach[t] = reach_of(p.window, s, i0 + t * T, min(s.nq, i0 + t * T + T));
    }
    // whether a tile of queries sees any of key tile k
    auto active = [&](int t, int k) {
        const int j0 = k * T;
        return there[t] && (j0 < reach[t].prefix || (j0 <= reach[t].hi && j0 + T > reach[t].lo && reach[t].lo <= reach[t].hi));
    };

    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        mbar_init(&tail, 1);
        for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int t = 0; t < 2; ++t) mbar_init(&s_full[t], 1), mbar_init(&p_ready[t], 4), mbar_init(&o_full[t], 1);
        mbar_fence_init();
    }
    if (warp == MMA_WARP) tc::tmem_alloc(&tmem_holder, TMEM_COLUMNS);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_holder, base = tc::smem_u32(smem), ring = base + 2 * TILE_BYTES;
    bool ok = true;

    if (warp >= SOFTMAX_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 " OTHER_REGISTERS ";");
        if (warp == LOAD_WARP) {
            if (all.n > 0) {
                if (lane == 0) {
                    tc::expect_bytes(&q_full, (there[1] ? 2 : 1) * TILE_BYTES);
                    for (int t = 0; t < (there[1] ? 2 : 1); ++t)
                        for (int b = 0; b < BOXES; ++b) tc::load_box(base + t * TILE_BYTES + b * BOX_BYTES, &maps.q, 64 * b, head, s.q0 + i0 + t * T, &q_full);
                }
                int issued = 0;
                for (int n = 0; n < 2 * all.n && ok; ++n) {  // K, V, K, V, ...
                    const int stage = n % STAGES, j0 = all.tile(n / 2) * T;
                    if (n >= STAGES) ok = tc::warp_wait(&empty[stage], (n / STAGES - 1) & 1);
                    if (!ok) break;
                    const bool v = n & 1, cut = v && j0 + T > s.nk;
                    const uint32_t at = ring + stage * TILE_BYTES;
                    uint64_t *bar = cut ? &tail : &full[stage];
                    if (lane == 0) {
                        tc::expect_bytes(bar, TILE_BYTES);
                        for (int b = 0; b < BOXES; ++b) tc::load_box(at + b * BOX_BYTES, v ? &maps.v : &maps.k, 64 * b, kv, s.k0 + j0, bar);
                    }
                    ++issued;
                    if (cut) {  // the last tile of a sequence, at most once
                        ok = tc::warp_wait(&tail, 0);
                        if (!ok) break;
                        const int first = s.nk - j0;
                        for (int i = lane; i < (T - first) * BOXES * 8; i += 32) {
                            const int b = i / ((T - first) * 8), r = first + i / 8 % (T - first);
                            *reinterpret_cast<uint4 *>(smem + 2 * TILE_BYTES + stage * TILE_BYTES + b * BOX_BYTES + r * 128 + i % 8 * 16) = make_uint4(0, 0, 0, 0);
                        }
                        tc::fence_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&full[stage]);
                    }
                }
                // copies of a role that gave up still land in this block's shared memory: wait for them
                if (!ok)
                    for (int n = issued > STAGES ? issued - STAGES : 0; n < issued; ++n) (void)tc::wait(&full[n % STAGES], (n / STAGES) & 1);
            }
        } else if (warp == MMA_WARP) {
            constexpr uint32_t ID_S = tc::instr_desc(BF16, T, T, false, false), ID_O = tc::instr_desc(BF16, T, DP, false, true);
            bool begun[2] = {false, false};
            unsigned n_p[2] = {0, 0};
            auto scores = [&](int t, int stage) {  // S of tile t
                if (tc::elected()) {
    #pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        const uint32_t o = k / 4 * BOX_BYTES + k % 4 * 32;
                        tc::mma_ss(tmem + t * T, tc::smem_desc(base + t * TILE_BYTES + o, 16), tc::smem_desc(ring + stage * TILE_BYTES + o, 16), ID_S, k > 0);
                    }
                    tc::commit(&s_full[t]);
                }
                __syncwarp();
            };
            if (all.n > 0) {
                ok = tc::warp_wait(&q_full, 0) && tc::warp_wait(&full[0], 0);
                if (ok) {
                    tc::fence_after();
                    for (int t = 0; t < 2; ++t)
                        if (active(t, all.tile(0))) scores(t, 0);
                    if (tc::elected()) tc::commit(&empty[0]);
                }
            }
            for (int u = 0; u < all.n && ok; ++u) {
                const int kt = all.tile(u), vs = (2 * u + 1) % STAGES, ks = (2 * u + 2) % STAGES;
                const bool more = u + 1 < all.n;
                ok = tc::warp_wait(&full[vs], ((2 * u + 1) / STAGES) & 1);
                for (int t = 0; t < 2 && ok; ++t) {
                    if (active(t, kt)) {
                        ok = tc::warp_wait(&p_ready[t], n_p[t]++ & 1);
                        if (!ok) break;
                        tc::fence_after();
                        if (tc::elected()) {
    #pragma unroll
                            for (int k = 0; k < T / 16; ++k)
                                tc::mma_ts(tmem + O_COLUMN + t * T, tmem + t * T + k * 8, tc::smem_desc(ring + vs * TILE_BYTES + k * 2048, BOX_BYTES), ID_O,
                                           begun[t] || k > 0);
                        }
                        __syncwarp();
                        begun[t] = true;
                    }
                    if (more) {
                        if (t == 0) ok = tc::warp_wait(&full[ks], ((2 * u + 2) / STAGES) & 1);
                        if (!ok) break;
                        tc::fence_after();
                        if (active(t, all.tile(u + 1))) scores(t, ks);
                    }
                }
                if (!ok) break;
                if (tc::elected()) {
                    tc::commit(&empty[vs]);
                    if (more) tc::commit(&empty[ks]);
                }
            }
            if (tc::elected()) {
                tc::commit(&o_full[0]);
                tc::commit(&o_full[1]);
            }
            __syncwarp();
            // nothing of this block is in flight when it ends, also where a role has given up
            ok = tc::warp_wait(&o_full[0], 0) && tc::warp_wait(&o_full[1], 0) && ok;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 " SOFTMAX_REGISTERS ";");
        const int t = warp >> 2, row = (warp & 3) * 32 + lane, i = i0 + t * T + row;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const float slope = BIAS ? __ldg(p.slopes + head) * LOG2E : 0.f;
        const float c = CAP ? 2.f * LOG2E * p.scale / p.cap : p.scale * LOG2E, top_of = p.cap * LOG2E;
        const int pos = s.nk - s.nq + i;
        const int lo = p.window.left < 0 ? 0 : max(0, pos - p.window.left), hi = p.window.right < 0 ? s.nk - 1 : min(s.nk - 1, pos + p.window.right);
        float most = -INFINITY, sum = 0.f;  // in units of log 2
        unsigned n_s = 0;
        for (int u = 0; u < all.n && ok; ++u) {
            const int j0 = all.tile(u) * T;
            if (!active(t, all.tile(u))) continue;
            ok = tc::warp_wait(&s_full[t], n_s & 1);
            if (!ok) break;
            tc::fence_after();
            float x[T];
#pragma unroll
            for (int b = 0; b < T / 32; ++b) tc::tmem_ld32(reinterpret_cast<uint32_t *>(x) + 32 * b, mine + t * T + 32 * b);
            tc::wait_ld();
            if (CAP) {
                // cap tanh(y) = cap - 2 cap / (1 + e^2y)
#pragma unroll
                for (int j = 0; j < T; ++j) x[j] = fmaf(-2.f * top_of, tc::rcp(1.f + tc::ex2(x[j] * c)), top_of);
            }
            if (BIAS) {
                const float at = (float)(pos - j0);
#pragma unroll
                for (int j = 0; j < T; ++j) x[j] = fmaf(-slope, fabsf(at - (float)j), CAP ? x[j] : x[j] * c);
            }
            if (!tile_is_open<T>(p.window, s, reach[t], j0)) {
                const int a = lo - j0, n = hi - lo, pre = s.prefix - j0;  // n < 0: nothing beside the prefix
#pragma unroll
                for (int j = 0; j < T; ++j)
                    if (!(j < pre || (n >= 0 && (unsigned)(j - a) <= (unsigned)n))) x[j] = -INFINITY;
            }
            float m4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int j = 4; j < T; j += 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) m4[k] = fmaxf(m4[k], x[j + k]);
            }
            float now = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            if (!CAP && !BIAS) now *= c;
            const bool raise = now > most + RAISE;  // (-inf + RAISE = -inf: any row's first)
            if (__any_sync(0xffffffffu, raise)) {
                const float to = raise ? now : most;
                const float shrink = raise ? tc::ex2(most - to) : 1.f;  // 0 for a row's first
                most = to;
                sum *= shrink;
                if (n_s > 0) {
#pragma unroll
                    for (int b = 0; b < DP / 32; ++b) {
                        uint32_t o[32];
                        tc::tmem_ld32(o, mine + O_COLUMN + t * T + 32 * b);
                        tc::wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
                        tc::tmem_st32(mine + O_COLUMN + t * T + 32 * b, o);
                    }
                }
            }
            const float less = most == -INFINITY ? 0.f : most;
            float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < T / 64; ++b) {
                uint32_t w[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const int at = 64 * b + 2 * j;
                    const float e0 = tc::ex2(CAP || BIAS ? x[at] - less : fmaf(x[at], c, -less));
                    const float e1 = tc::ex2(CAP || BIAS ? x[at + 1] - less : fmaf(x[at + 1], c, -less));
                    s4[j & 3] += e0 + e1;
                    w[j] = tc::pack<E>(e0, e1);
                }
                tc::tmem_st32(mine + t * T + 32 * b, w);
            }
            sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[t]);
            ++n_s;
        }
        if (ok && n_s > 0) ok = tc::warp_wait(&o_full[t], 0);
        if (ok && there[t]) {
            tc::fence_after();
            const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
            const float lse = sum == 0.f ? -INFINITY : (most + log2f(sum)) * LN2;
            bool bad = false;
            E *dst = static_cast<E *>(p.o.data) + ((int64_t)s.q0 + i) * p.o.row + head * p.o.head;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) {
                float o[32];
                if (n_s > 0) {
                    tc::tmem_ld32(reinterpret_cast<uint32_t *>(o), mine + O_COLUMN + t * T + 32 * b);
                    tc::wait_ld();
                }
                uint32_t w[16];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    o[j] = n_s > 0 ? o[j] * inv : 0.f;
                    bad = bad || (!isfinite(o[j]) && 32 * b + j < p.head_dim);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) w[j] = tc::pack<E>(o[2 * j], o[2 * j + 1]);
                if (i < s.nq) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (32 * b + 8 * j < p.head_dim)
                            *reinterpret_cast<uint4 *>(dst + 32 * b + 8 * j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                }
            }
            if (p.lse && i < s.nq) p.lse[(int64_t)head * p.q_rows + s.q0 + i] = lse;
            for (unsigned left = __ballot_sync(0xffffffffu, bad && i < s.nq); left; left &= left - 1) {
                const int l = __ffs(left) - 1;
                __syncwarp();
                strict::output_row<E>(p, s, head, i - lane + l, __shfl_sync(0xffffffffu, lse, l));
            }
        }
    }
    if (!ok && lane == 0) dev::report_timeout(p.status);
    tc::fence_before();
    __syncthreads();
    if (warp == MMA_WARP) tc::tmem_dealloc(tmem, TMEM_COLUMNS);
}

template <class E, int DP, bool CAP, bool BIAS>
cudaError_t launch(const AttentionParams &p, const Maps &maps, cudaStream_t s)
{
    constexpr size_t smem = (2 + STAGES) * T * DP * 2;
    static SmemOptinCache optin;
    const cudaError_t e = optin_dynamic_smem(attention_forward_tc_kernel<E, DP, CAP, BIAS>, smem, optin);
    if (e != cudaSuccess) return e;
    const unsigned grid = (unsigned)(p.q_heads * most_blocks(p.q_rows, p.n_seqs, p.max_q, 2 * T));
    if (grid == 0) return cudaSuccess;
    attention_forward_tc_kernel<E, DP, CAP, BIAS><<<grid, THREADS, smem, s>>>(p, maps);
    return cudaGetLastError();
}
template <class E, int DP>
cudaError_t by_score(const AttentionParams &p, const Maps &maps, cudaStream_t s)
{
    if (p.cap > 0.f) return p.slopes ? launch<E, DP, true, true>(p, maps, s) : launch<E, DP, true, false>(p, maps, s);
    return p.slopes ? launch<E, DP, false, true>(p, maps, s) : launch<E, DP, false, false>(p, maps, s);
}

}  // namespace

bool attention_forward_tc_takes(const AttentionParams &p)
{
    // 16-byte stores of O
    return p.dtype != 0 && (uintptr_t)p.o.data % 16 == 0 && p.o.row % 8 == 0 && p.o.head % 8 == 0 && p.k_rows > 0;
}

cudaError_t launch_attention_forward_tc(const AttentionParams &p, bool *taken, cudaStream_t s)
{
    Maps maps;
    *taken = attention_forward_tc_takes(p) && make_tensor_map(&maps.q, p.q, p.dtype, p.head_dim, p.q_heads, p.q_rows, T) &&
             make_tensor_map(&maps.k, p.k, p.dtype, p.head_dim, p.kv_heads, p.k_rows, T) &&
             make_tensor_map(&maps.v, p.v, p.dtype, p.head_dim, p.kv_heads, p.k_rows, T);
    if (!*taken) return cudaSuccess;
    if (p.dtype == 1) return p.head_dim <= 64 ? by_score<__half, 64>(p, maps, s) : by_score<__half, 128>(p, maps, s);
    return p.head_dim <= 64 ? by_score<__nv_bfloat16, 64>(p, maps, s) : by_score<__nv_bfloat16, 128>(p, maps, s);
}

}  // namespace sddmm
