// Attention, forward, on the tensor cores (tcgen05), for fp16 and bfloat16.
//
// A block has 256 queries of one head, two tiles of 128, and goes once over the keys in tiles of 128:
//
//   warps 0-7, 8-15  softmax of a tile each, half of a row a thread: reads its scores from tensor memory, masks them where the tile is not open,
//                    keeps the row's running maximum (with the thread that has the other half) and its sum in registers, writes the
//                    weights, rounded to the operands' type, back to tensor memory;
//   warp 16          one thread issues S = Q K^T (both operands in shared memory) and O += P V (P in tensor memory, V read as it
//                    lies, MN-major), for the two tiles of queries in turn;
//   warp 17          one thread brings Q, K and V by tile copies into rings.
//
// Tensor memory holds the scores and O of both tiles.  Heads of up to 64 leave room for the weights beside the scores, so the next
// tile's scores come as soon as the last ones have been read; wider ones do not, the weights lie over the scores, and the chain
// softmax, P V, next S of one tile of queries runs under that of the other.  That chain is what bounds the kernel: a product of
// 128 x 128 x 16 takes the tensor core 64 clocks and its issue 67, so S and P V of a tile are 1,056; with a whole row a thread the
// softmax of a tile took 2,000 more.  8,192 causal tokens, 16 heads of 128, bfloat16: 313 us, 878 TFLOP/s, 3,745 clocks a step of 256 queries
// by 128 keys of which the products' issue is 2,112; 16,384 tokens under a band of 256 and 80 global, 4 heads of 64: 41 us.
// With a cap: prompts of 1 to 2,111 tokens, 16 / 4 heads of 128, 112 us; where most scores are near the cap, tanh goes by exponentials
// beside the polynomial (4,096 tokens, 8 heads of 128: 97 us with small scores, 158 so).
//
// The maximum that weights are relative to is only raised when it has grown by more than 2^8: weights then reach 256 at most, which
// neither type minds, and the accumulator in tensor memory is rescaled by hardly any tile.
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
using tc::F2;

constexpr int T = 128;  // queries of a tile
constexpr int KT = 128;  // keys of a tile
constexpr int SOFTMAX_WARPS = 16, MMA_WARP = 16, LOAD_WARP = 17, THREADS = 640;
constexpr int COLUMNS = KT / 2;  // of a thread
static_assert(2 * T == PROMPT_QUERIES && KT == PROMPT_KEYS, "the join goes by these");
constexpr uint32_t TMEM_COLUMNS = 512, O_COLUMN = 256;  // S at 0 and 128
constexpr float RAISE = 8.f;
// Registers of a thread: 96 at launch (640 threads), shared out anew: 4 x 104 + 64 = 5 x 96.
#define SOFTMAX_REGISTERS "104"
#define OTHER_REGISTERS "64"

struct alignas(64) Maps {
    CUtensorMap q, k, v;
};

template <int DP> struct Shape {
    static constexpr int BOXES = DP / 64, Q_BYTES = T * DP * 2, TILE_BYTES = KT * DP * 2, Q_BOX = T * 128, BOX = KT * 128;
    static constexpr int STAGES = DP == 64 ? 4 : 2;  // of K and of V
    static constexpr int SMEM = 2 * Q_BYTES + 2 * STAGES * TILE_BYTES;
    // weights of tile t of the queries; the two halves of a row are P_APART columns apart
    static constexpr bool BESIDE = DP == 64;
    static constexpr uint32_t P_AT = BESIDE ? 384 : 0, P_TILE = BESIDE ? 64 : 128, P_APART = BESIDE ? 32 : 64;
    static constexpr uint32_t O_TILE = DP == 64 ? 64 : 128;
};

// barrier.cta.red.and over the 256 threads of a tile of queries (named barrier 1 + tile): one answer for all of them
__device__ __forceinline__ bool tile_all(int tile, bool mine)
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r)
                 : "r"((uint32_t)mine), "r"(1 + tile)
                 : "memory");
    return r != 0;
}

// PARTS: the keys of a block may be cut (a form of its own: what it has to remember cost the other 8 % in registers)
template <class E, int DP, bool CAP, bool BIAS, bool PARTS>
__global__ void __launch_bounds__(THREADS, 1) attention_forward_tc_kernel(const AttentionParams p, const __grid_constant__ Maps maps)
{
    using Sh = Shape<DP>;
    constexpr int BOXES = Sh::BOXES, Q_BYTES = Sh::Q_BYTES, TILE_BYTES = Sh::TILE_BYTES, Q_BOX = Sh::Q_BOX, BOX = Sh::BOX, STAGES = Sh::STAGES;
    constexpr bool BESIDE = Sh::BESIDE;
    // Every eighth exponential without the special function unit, where FMAs are to spare: band, heads of 64, 41.9 -> 41.0 us; long prompt,
    // heads of 128, 313 -> 317; with a cap, whose tanh takes the FMAs, heads of 128, 108 -> 115.
    constexpr bool POLY = DP == 64 && !CAP;
    constexpr bool BF16 = sizeof(E) == 2 && !std::is_same<E, __half>::value;
    extern __shared__ __align__(1024) unsigned char smem[];  // two tiles of Q, the rings of K and of V
    __shared__ uint64_t q_full, full[2][STAGES], empty[2][STAGES], s_full[2], s_read[2], p_ready[2], o_done[2], o_full, tail;  // [K, V], [tile of Q]
    __shared__ uint32_t tmem_holder, bad[8];
    __shared__ float row_most[2][2][2][T], row_sum[2][2][T], row_lse[2 * T];  // [step parity][tile][half]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (PARTS) next_kernel_may_come();
    const unsigned splits = PARTS ? p.n_splits : 1, blocks = gridDim.x / splits, block_of = blockIdx.x / splits, part = PARTS ? blockIdx.x % splits : 0;
    const int head = block_of % p.q_heads, kv = head / p.group;
    Sequence s;
    int seq, block;
    // the last blocks of a causal sequence have the most keys: they go first
    if (!find_block<2 * T>(p, (blocks - 1 - block_of) / p.q_heads, false, s, seq, block)) return;
    const int i0 = block * 2 * T;
    const KeyTiles of_block = key_tiles<KT>(reach_of(p.window, s, i0, min(s.nq, i0 + 2 * T)));
    // a part of them where the blocks alone would leave multiprocessors idle: parts are joined as those of few queries are
    const Part mine_of = PARTS ? part_of(p, of_block.n, part) : Part{0, of_block.n, true};
    if (mine_of.end < 0) return;
    struct {
        KeyTiles keys;
        int first, n;
        __device__ __forceinline__ int tile(int u) const { return keys.tile(PARTS ? first + u : u); }
    } const all{of_block, mine_of.first, mine_of.end - mine_of.first};
    Reach reach[2];
    bool there[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        there[t] = i0 + t * T < s.nq;
        reach[t] = reach_of(p.window, s, i0 + t * T, min(s.nq, i0 + t * T + T));
    }
    // whether a tile of queries sees any of key tile k
    auto active = [&](int t, int k) {
        const int j0 = k * KT;
        return there[t] && (j0 < reach[t].prefix || (j0 <= reach[t].hi && j0 + KT > reach[t].lo && reach[t].lo <= reach[t].hi));
    };

    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        mbar_init(&tail, 1);
        mbar_init(&o_full, 1);
        for (int x = 0; x < 2; ++x) {
            for (int i = 0; i < STAGES; ++i) mbar_init(&full[x][i], 1), mbar_init(&empty[x][i], 1);
            mbar_init(&s_full[x], 1);
            mbar_init(&s_read[x], 8);
            mbar_init(&p_ready[x], 8);
            mbar_init(&o_done[x], 1);
        }
        mbar_fence_init();
    }
    if (threadIdx.x < 8) bad[threadIdx.x] = 0;
    if (warp == MMA_WARP) tc::tmem_alloc(&tmem_holder, TMEM_COLUMNS);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_holder, base = tc::smem_u32(smem), rings = base + 2 * Q_BYTES;
    bool ok = true;

    if (warp >= SOFTMAX_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 " OTHER_REGISTERS ";");
        if (warp == LOAD_WARP && all.n > 0) {
            if (lane == 0) {
                tc::expect_bytes(&q_full, (there[1] ? 2 : 1) * Q_BYTES);
                for (int t = 0; t < (there[1] ? 2 : 1); ++t)
                    for (int b = 0; b < BOXES; ++b) tc::load_box(base + t * Q_BYTES + b * Q_BOX, &maps.q, 64 * b, head, s.q0 + i0 + t * T, &q_full);
            }
            int issued[2] = {0, 0};
            // in the order of use: K0, K1, V0, K2, V1, K3, ...
            for (int n = 0; n < 2 * all.n && ok; ++n) {
                const int v = n < 2 || n == 2 * all.n - 1 ? (all.n == 1 ? n : n >= 2) : 1 - (n & 1), u = issued[v];
                const int stage = u % STAGES, j0 = all.tile(u) * KT;
                if (u >= STAGES) ok = tc::warp_wait(&empty[v][stage], (u / STAGES - 1) & 1);
                if (!ok) break;
                const bool cut = v && j0 + KT > s.nk;
                const uint32_t slot = 2 * Q_BYTES + (v * STAGES + stage) * TILE_BYTES;
                uint64_t *bar = cut ? &tail : &full[v][stage];
                if (lane == 0) {
                    tc::expect_bytes(bar, TILE_BYTES);
                    for (int b = 0; b < BOXES; ++b) tc::load_box(base + slot + b * BOX, v ? &maps.v : &maps.k, 64 * b, kv, s.k0 + j0, bar);
                }
                ++issued[v];
                if (cut) {  // the last tile of a sequence, at most once
                    ok = tc::warp_wait(&tail, 0);
                    if (!ok) break;
                    tc::zero_rows<KT, BOXES>(smem + slot, s.nk - j0);
                    tc::fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[v][stage]);
                }
            }
            // copies of a role that gave up still land in this block's shared memory: wait for them
            if (!ok)
                for (int v = 0; v < 2; ++v)
                    for (int u = max(0, issued[v] - STAGES); u < issued[v]; ++u) (void)tc::wait(&full[v][u % STAGES], (u / STAGES) & 1);
        } else if (warp == MMA_WARP) {
            constexpr uint32_t ID_S = tc::instr_desc(BF16, T, KT, false, false), ID_O = tc::instr_desc(BF16, T, DP, false, true);
            const uint64_t q_desc = tc::smem_desc(base, 16), k_desc = tc::smem_desc(rings, 16), v_desc = tc::smem_desc(rings + STAGES * TILE_BYTES, BOX);
            unsigned n_s[2] = {0, 0}, n_p[2] = {0, 0};  // tiles of keys that a tile of queries has had
            // S of a tile of queries; the tile of keys has been waited for, and what lay in the place has been read
            auto scores = [&](int t, int u) {
                if (!active(t, all.tile(u))) return;
                const uint64_t q = q_desc + t * (Q_BYTES >> 4), k_at = k_desc + __shfl_sync(0xffffffffu, u % STAGES, 0) * (TILE_BYTES >> 4);
                ++n_s[t];
                if (tc::elected()) {
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        tc::mma_ss(tmem + t * T, q + ((k / 4 * Q_BOX + k % 4 * 32) >> 4), k_at + ((k / 4 * BOX + k % 4 * 32) >> 4), ID_S, k > 0);
                    tc::commit(&s_full[t]);
                }
                __syncwarp();
            };
            auto k_done = [&](int u) {
                if (tc::elected()) tc::commit(&empty[0][u % STAGES]);
                __syncwarp();
            };
            auto wait_tile = [&](int v, int u) {
                ok = ok && tc::warp_wait(&full[v][u % STAGES], (u / STAGES) & 1);
                tc::fence_after();
                return ok;
            };
            auto weights = [&](int t, int u) {
                if (!active(t, all.tile(u))) return;
                const unsigned n = n_p[t]++;
                ok = ok && tc::warp_wait(&p_ready[t], n & 1);
                if (!ok) return;
                tc::fence_after();
                const uint64_t v_at = v_desc + __shfl_sync(0xffffffffu, u % STAGES, 0) * (TILE_BYTES >> 4);
                if (tc::elected()) {
#pragma unroll
                    for (int k = 0; k < KT / 16; ++k)
                        tc::mma_ts(tmem + O_COLUMN + t * Sh::O_TILE, tmem + Sh::P_AT + t * Sh::P_TILE + k / 4 * Sh::P_APART + k % 4 * 8, v_at + k * (2048 >> 4), ID_O,
                                   n > 0 || k > 0);
                    tc::commit(&o_done[t]);
                }
                __syncwarp();
            };
            if (all.n > 0) {
                ok = tc::warp_wait(&q_full, 0);
                if (ok && wait_tile(0, 0)) {
                    scores(0, 0);
                    scores(1, 0);
                    k_done(0);
                }
            }
            for (int u = 0; u < all.n && ok; ++u) {
                const bool more = u + 1 < all.n;
                if (BESIDE) {
                    if (more) {
                        if (!wait_tile(0, u + 1)) break;
                        for (int t = 0; t < 2; ++t) {
                            if (n_s[t] > 0) ok = ok && tc::warp_wait(&s_read[t], (n_s[t] - 1) & 1);
                            if (!ok) break;
                            tc::fence_after();
                            scores(t, u + 1);
                        }
                        if (!ok) break;
                        k_done(u + 1);
                    }
                    if (!wait_tile(1, u)) break;
                    weights(0, u);
                    weights(1, u);
                } else {
                    if (!wait_tile(1, u)) break;
                    weights(0, u);
                    if (more && wait_tile(0, u + 1)) scores(0, u + 1);
                    weights(1, u);
                    if (more && ok) {
                        scores(1, u + 1);
                        k_done(u + 1);
                    }
                }
                if (tc::elected()) tc::commit(&empty[1][u % STAGES]);
                __syncwarp();
            }
            if (tc::elected()) tc::commit(&o_full);
            __syncwarp();
            // nothing of this block is in flight when it ends, also where a role has given up
            ok = tc::warp_wait(&o_full, 0) && ok;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 " SOFTMAX_REGISTERS ";");
        const int t = warp >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane, i = i0 + t * T + row;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t my_scores = mine + t * T + half * COLUMNS, my_weights = mine + Sh::P_AT + t * Sh::P_TILE + half * Sh::P_APART;
        const float slope = BIAS ? __ldg(p.slopes + head) * LOG2E : 0.f;
        const float c = !CAP ? p.scale * LOG2E : p.of_cap, top_of = p.cap * LOG2E;
        const tc::Tanh tanh_c = tc::tanh_polynomial(c, top_of);
        const int pos = s.nk - s.nq + i;
        const int lo = p.window.left < 0 ? 0 : max(0, pos - p.window.left), hi = p.window.right < 0 ? s.nk - 1 : min(s.nk - 1, pos + p.window.right);
        float most = -INFINITY, sum = 0.f;  // in units of log 2
        unsigned n_s = 0;
        for (int u = 0; u < all.n; ++u) {
            if (!active(t, all.tile(u))) continue;
            const int j0 = all.tile(u) * KT + half * COLUMNS;
            ok = ok && tc::warp_wait(&s_full[t], n_s & 1);
            tc::fence_after();
            F2 x[COLUMNS / 2];  // two keys each
#pragma unroll
            for (int b = 0; b < COLUMNS / 32; ++b) tc::tmem_ld32(reinterpret_cast<uint32_t *>(x) + 32 * b, my_scores + 32 * b);
            tc::wait_ld();
            if (BESIDE) {
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_read[t]);  // the next scores may come
            }
            // Without a bias the capped scores keep their order, so the row's maximum is found among the products, and tanh comes with the
            // exponentials: its FMAs (1,500 clocks a tile) run beside their special function unit (1,000).
            bool small = true;
            if (CAP) {
                float size = 0.f;
#pragma unroll
                for (int j = 0; j < COLUMNS / 2; ++j) {
                    float a, b;
                    tc::split(x[j], a, b);
                    size = tc::max3_abs(size, a, b);
                }
                small = p.pre == 1.f && __all_sync(0xffffffffu, size <= tanh_c.range);
                if (!small && p.pre != 1.f) {
#pragma unroll
                    for (int j = 0; j < COLUMNS / 2; ++j) x[j] = tc::mul2(x[j], tc::two(p.pre, p.pre));
                }
            }
            if (CAP && BIAS) {
                if (small) {
#pragma unroll
                    for (int j = 0; j < COLUMNS / 2; ++j) x[j] = tc::tanh2(x[j], tanh_c);
                } else {
#pragma unroll
                    for (int j = 0; j < COLUMNS / 2; ++j) x[j] = tc::tanh_any(x[j], tanh_c, c, top_of, 0.f);
                }
            }
            if (BIAS) {
                const float at = (float)(pos - j0);
                // all keys of the tile on one side of all rows of the warp: the distance is linear
                const int warp_pos = pos - lane;
                const float side = j0 + COLUMNS - 1 <= warp_pos ? slope : j0 >= warp_pos + 31 ? -slope : 0.f;
                if (j0 + COLUMNS - 1 <= warp_pos || j0 >= warp_pos + 31) {
#pragma unroll
                    for (int j = 0; j < COLUMNS / 2; ++j) {
                        const F2 less = tc::ffma2(tc::two(side, side), tc::two(2.f * j, 2.f * j + 1.f), tc::two(-side * at, -side * at));
                        x[j] = CAP ? tc::add2(x[j], less) : tc::ffma2(x[j], tc::two(c, c), less);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < COLUMNS / 2; ++j) {
                        float a, b;
                        tc::split(x[j], a, b);
                        x[j] = tc::two(fmaf(-slope, fabsf(at - 2.f * j), CAP ? a : a * c), fmaf(-slope, fabsf(at - (2.f * j + 1.f)), CAP ? b : b * c));
                    }
                }
            }
            const bool open = tile_is_open<COLUMNS>(p.window, s, reach[t], j0);
            unsigned seen_of[COLUMNS / 32];
            if (!open) {
#pragma unroll
                for (int b = 0; b < COLUMNS / 32; ++b) {
                    const unsigned seen = seen_of[b] = seen_bits(lo, hi, s.prefix, j0 + 32 * b);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float a0, a1;
                        tc::split(x[16 * b + j], a0, a1);
                        a0 = seen & 1u << 2 * j ? a0 : -INFINITY;
                        a1 = seen & 2u << 2 * j ? a1 : -INFINITY;
                        x[16 * b + j] = tc::two(a0, a1);
                    }
                }
            }
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < COLUMNS / 2; ++j) {
                float a, b;
                tc::split(x[j], a, b);
                m4[j & 3] = tc::max3(m4[j & 3], a, b);
            }
            float now = fmaxf(tc::max3(m4[0], m4[1], m4[2]), m4[3]);
            if (!CAP && !BIAS) now *= c;
            // with the other half of the row; a role's giving up is told to the whole tile here
            row_most[n_s & 1][t][half][row] = now;
            if (!tile_all(t, ok)) {
                ok = false;
                break;
            }
            now = fmaxf(now, row_most[n_s & 1][t][half ^ 1][row]);
            if (CAP && !BIAS && now > -INFINITY) now = fmaf(-2.f * top_of, tc::rcp(1.f + tc::ex2(now * (2.f * LOG2E * c))), top_of);
            const bool raise = now > most + RAISE;  // (-inf + RAISE = -inf: any row's first)
            if (__any_sync(0xffffffffu, raise)) {
                const float to = raise ? now : most;
                const float shrink = raise ? tc::ex2(most - to) : 1.f;  // 0 for a row's first
                most = to;
                sum *= shrink;
                if (n_s > 0) {
                    // the products so far, at most one of which is under way; each half of the row has half of O's columns
                    ok = tc::warp_wait(&o_done[t], (n_s - 1) & 1);
                    tc::fence_after();
#pragma unroll 1
                    for (int b = 0; b < DP / 32; ++b) {
                        uint32_t o[16];
                        const uint32_t at = mine + O_COLUMN + t * Sh::O_TILE + half * (DP / 2) + 16 * b;
                        tc::tmem_ld16(o, at);
                        tc::wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
                        tc::tmem_st16(at, o);
                    }
                }
            }
            const float less = most == -INFINITY ? 0.f : -most;
            F2 s2[2] = {0, 0};
            uint32_t w[COLUMNS / 2];
            auto weigh = [&](auto all_seen, auto is_small) {
#pragma unroll
                for (int j = 0; j < COLUMNS / 2; ++j) {
                    F2 e;
                    float e0, e1;
                    if (CAP && !BIAS) {
                        if (decltype(is_small)::value) e = tc::ffma2(x[j], tc::tanh_over_x(x[j], tanh_c), tc::two(less, less));
                        else e = tc::tanh_any(x[j], tanh_c, c, top_of, less);
                        if (!decltype(all_seen)::value) {
                            tc::split(e, e0, e1);
                            e = tc::two(seen_of[j / 16] & 1u << 2 * (j % 16) ? e0 : -INFINITY, seen_of[j / 16] & 2u << 2 * (j % 16) ? e1 : -INFINITY);
                        }
                    } else {
                        e = BIAS ? tc::add2(x[j], tc::two(less, less)) : tc::ffma2(x[j], tc::two(c, c), tc::two(less, less));
                    }
                    if (POLY && j % 8 == 0) {
                        tc::split(tc::ex2_poly(e), e0, e1);
                    } else {
                        tc::split(e, e0, e1);
                        e0 = tc::ex2(e0), e1 = tc::ex2(e1);
                    }
                    s2[j & 1] = tc::add2(s2[j & 1], tc::two(e0, e1));
                    w[j] = tc::pack<E>(e0, e1);
                }
            };
            if (!CAP || BIAS || (open && small)) weigh(std::true_type(), std::true_type());
            else if (small) weigh(std::false_type(), std::true_type());
            else {
                if (open) seen_of[0] = seen_of[1] = ~0u;
                weigh(std::false_type(), std::false_type());
            }
            if (BESIDE && n_s > 0) ok = ok && tc::warp_wait(&o_done[t], (n_s - 1) & 1);  // the last weights have been used
            tc::tmem_st32(my_weights, w);
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[t]);
            float e0, e1;
            tc::split(tc::add2(s2[0], s2[1]), e0, e1);
            sum += e0 + e1;
            ++n_s;
        }
        if (all.n > 0) ok = ok && tc::warp_wait(&q_full, 0) && tc::warp_wait(&o_full, 0);
        row_sum[t][half][row] = sum;
        ok = tile_all(t, ok);
        if (ok && there[t]) {
            tc::fence_after();
            sum = row_sum[t][0][row] + row_sum[t][1][row];
            const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
            const float lse = sum == 0.f ? -INFINITY : (most + log2f(sum)) * LN2;
            float zero = 0.f;  // NaN as soon as a result is not finite
            unsigned char *const stage = smem + warp * 32 * DP;  // of the tiles of Q, which are done with
#pragma unroll
            for (int b = 0; b < DP / 64; ++b) {
                float o[32];
                if (n_s > 0) {
                    tc::tmem_ld32(reinterpret_cast<uint32_t *>(o), mine + O_COLUMN + t * Sh::O_TILE + half * (DP / 2) + 32 * b);
                    tc::wait_ld();
                }
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    o[j] = n_s > 0 ? o[j] * inv : 0.f;
                    zero = fmaf(o[j], 0.f, zero);
                }
                if (!PARTS || mine_of.alone) {
                    tc::stage_32<E, DP / 2>(stage, 32 * b, o);
                } else if (i < s.nq) {
                    const int first = half * (DP / 2) + 32 * b;
                    float *to = p.part_o + ((part * p.q_rows + s.q0 + i) * p.q_heads + head) * p.head_dim + first;
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        if (first + j < p.head_dim) *reinterpret_cast<float4 *>(to + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                }
            }
            const int row0 = i - lane;
            if (!PARTS || mine_of.alone)
                tc::store_staged<E, DP / 2>(stage, static_cast<E *>(p.o.data) + ((int64_t)s.q0 + row0) * p.o.row + head * p.o.head + half * (DP / 2), p.o.row, s.nq - row0,
                                        p.head_dim - half * (DP / 2));
            if (half == 0 && i < s.nq) {
                if (PARTS && !mine_of.alone) p.part_lse[(part * p.q_rows + s.q0 + i) * p.q_heads + head] = sum == 0.f ? -INFINITY : most + log2f(sum);
                else if (p.lse) p.lse[(int64_t)head * p.q_rows + s.q0 + i] = lse;
            }
            if (half == 0) row_lse[t * T + row] = lse;
            const unsigned rows = __ballot_sync(0xffffffffu, zero != 0.f && i < s.nq && (!PARTS || mine_of.alone));
            if (lane == 0 && rows) atomicOr(&bad[t * 4 + (warp & 3)], rows);
        }
    }
    if (!ok && lane == 0) dev::report_timeout(p.status);
    tc::fence_before();
    __syncthreads();
    if (warp == MMA_WARP) tc::tmem_dealloc(tmem, TMEM_COLUMNS);
    if (warp < SOFTMAX_WARPS)
        for (int q = 0; q < 8; ++q)
            for (unsigned left = bad[q], turn = 0; left; left &= left - 1, ++turn)
                if (turn % SOFTMAX_WARPS == (unsigned)warp) {
                    const int r = 32 * q + __ffs(left) - 1;
                    strict::output_row<E>(p, s, head, i0 + r, row_lse[r]);
                }
}

template <class E, int DP, bool CAP, bool BIAS, bool PARTS>
cudaError_t launch(const AttentionParams &p, const Maps &maps, cudaStream_t s)
{
    constexpr size_t smem = Shape<DP>::SMEM;
    static SmemOptinCache optin;
    const cudaError_t e = optin_dynamic_smem(attention_forward_tc_kernel<E, DP, CAP, BIAS, PARTS>, smem, optin);
    if (e != cudaSuccess) return e;
    const unsigned grid = (unsigned)(p.q_heads * most_blocks(p.q_rows, p.n_seqs, p.max_q, 2 * T));
    if (grid == 0) return cudaSuccess;
    attention_forward_tc_kernel<E, DP, CAP, BIAS, PARTS><<<grid * p.n_splits, THREADS, smem, s>>>(p, maps);
    return cudaGetLastError();
}
template <class E, int DP, bool CAP, bool BIAS>
cudaError_t launch(const AttentionParams &p, const Maps &maps, cudaStream_t s)
{
    return p.n_splits > 1 ? launch<E, DP, CAP, BIAS, true>(p, maps, s) : launch<E, DP, CAP, BIAS, false>(p, maps, s);
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

ForwardPlan plan_attention_forward_tc(const AttentionParams &p, int sm_count)
{
    // Parts until there is a block for every multiprocessor, of two tiles of keys at least, and at most 256 MB of them.
    const int64_t blocks = p.q_heads * most_blocks(p.q_rows, p.n_seqs, p.max_q, 2 * T), tiles = (p.max_k + KT - 1) / KT;
    const int64_t bytes = p.q_rows * p.q_heads * (int64_t)(p.head_dim + 1) * 4;
    ForwardPlan f{1, (int)(tiles > 0 ? tiles : 1), 0, 0.};
    int64_t want = blocks > 0 ? sm_count / blocks : 1;
    if (want > tiles / 2) want = tiles / 2;
    if (bytes > 0 && want > (256ll << 20) / bytes) want = (256ll << 20) / bytes;
    if (want > 1 && (int64_t)p.n_seqs * p.max_q * p.q_heads <= INT32_MAX) {
        f.chunk_tiles = (int)((tiles + want - 1) / want);
        f.n_splits = (int)((tiles + f.chunk_tiles - 1) / f.chunk_tiles);
        f.bytes = f.n_splits > 1 ? f.n_splits * bytes : 0;
    }
    // (8 us and 2.0 a tile of 256 x 128 for every wave of blocks; 6 more with a join, most of it the second launch)
    const int64_t waves = (blocks * f.n_splits + sm_count - 1) / sm_count;
    f.us = 8. + 2.0 * (double)waves * f.chunk_tiles + (f.n_splits > 1 ? 6. : 0.);
    return f;
}

cudaError_t launch_attention_forward_tc(const AttentionParams &p0, const ForwardPlan &f, void *workspace, bool *taken, cudaStream_t s)
{
    Maps maps;
    AttentionParams p = p0;
    p.n_splits = f.n_splits;
    p.chunk_tiles = f.chunk_tiles;
    p.part_o = static_cast<float *>(workspace);
    p.part_lse = p.part_o + (f.n_splits == 1 ? 0 : (int64_t)f.n_splits * p.q_rows * p.q_heads * p.head_dim);
    *taken = attention_forward_tc_takes(p) && make_tensor_map(&maps.q, p.q, p.dtype, p.head_dim, p.q_heads, p.q_rows, T) &&
             make_tensor_map(&maps.k, p.k, p.dtype, p.head_dim, p.kv_heads, p.k_rows, KT) &&
             make_tensor_map(&maps.v, p.v, p.dtype, p.head_dim, p.kv_heads, p.k_rows, KT);
    if (!*taken) return cudaSuccess;
    cudaError_t e;
    if (p.dtype == 1) e = p.head_dim <= 64 ? by_score<__half, 64>(p, maps, s) : by_score<__half, 128>(p, maps, s);
    else e = p.head_dim <= 64 ? by_score<__nv_bfloat16, 64>(p, maps, s) : by_score<__nv_bfloat16, 128>(p, maps, s);
    return e == cudaSuccess && p.n_splits > 1 ? launch_attention_join(p, JOIN_PROMPT, s) : e;
}

}  // namespace sddmm
