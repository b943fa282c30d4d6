// Attention, backward, on the tensor cores (tcgen05), for fp16 and bfloat16: two kernels of one shape, without atomics.
//
//   dQ      a block has 128 queries of a head, Q and dO in shared memory, and goes over the keys in tiles of 128:
//             S = Q K^T, dP = dO V^T, dS = P (dP - delta), dQ += dS K
//   dK, dV  a block has 128 keys of a KV head, K and V in shared memory, and goes over the queries of all heads of the group:
//             S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//
// with P = exp(S - lse) and delta_i = dO_i.O_i, which the first kernel leaves for the second.  Scores are computed in both (7 products
// where one kernel would do with 5): a single kernel would have to add up dQ over blocks, by atomics in no fixed order, in a
// fp32 array of its own.  P and dS are rounded to the operands' type, as every operand of the tensor cores is.  fp16 has five bits of exponent,
// so there P (dP - delta) is multiplied by a power of two first that brings the largest |dO| to 4 .. 8, and the sums are divided by it again: a power for
// every row in the dQ kernel, one for all rows that a block goes through in the other, from what the first kernel leaves for each tile.  (It costs
// nothing: dP comes in by an FMA, and delta is multiplied once.)  Beyond 65,504 rows are computed anew (attention_strict.cuh).
//
//   warps 0-15  a row of the block in every thread, a quarter of the tile's columns in each group of four warps: scores from tensor
//               memory, weights and score gradients back to it;
//   warp 16     one thread issues the products; the second operand of the last ones is the streamed tile as it lies, MN-major;
//   warp 17     one thread brings the tiles by tile copies;
//   warp 18     (dK, dV) brings lse and delta of the tile's queries, negative, two tiles ahead.
//
// dQ: score gradients have a place of their own in tensor memory (two, in turn), so the next tile's scores are computed as soon as the
// last ones have been read.  dK, dV: tensor memory is full (S, dP, dV, dK); P and dS take the place of S and dP, and the
// products take turns: dV, S of the next tile, dK, dP of the next tile.
//
// What bounds them: the row warps' chain beside the products' issue: dQ 2,170 clocks a tile for 1,600 of issue, dK, dV 3,200 for 2,112.
// 8,192 causal tokens, 8 heads of 128, bfloat16: 468 us, 735 TFLOP/s of the five products that it cannot do without.
#include <type_traits>

#include "attention_strict.cuh"
#include "tc_utils.cuh"

namespace sddmm {

namespace {

using tc::mbar_arrive;
using tc::mbar_fence_init;
using tc::mbar_init;
using tc::F2;

constexpr int T = 128;
static_assert(T == DO_TILE, "the workspace has a place for every tile");
constexpr int ROW_WARPS = 16, MMA_WARP = 16, LOAD_WARP = 17, STATS_WARP = 18, THREADS = 640;
constexpr int MINE = 32;  // columns of a thread
constexpr uint32_t TMEM_COLUMNS = 512, S_AT = 0, DP_AT = 128;
// dQ: accumulator, then two places of 64 columns for score gradients.  dK, dV: the two accumulators.
constexpr uint32_t DQ_AT = 256, DS_AT = 384, DV_AT = 256, DK_AT = 384;
// Registers of a thread: 96 at launch (640 threads), shared out anew: 4 x 104 + 64 = 5 x 96.
#define ROW_REGISTERS "104"
#define OTHER_REGISTERS "64"

struct alignas(64) Maps {
    CUtensorMap q, k, v, d_o;
};

template <int DP, bool KV> struct Shape {
    static constexpr int BOXES = DP / 64, TILE_BYTES = T * DP * 2, BOX_BYTES = T * 128;
    // The streamed tiles: K or Q is used by S and again, an iteration later, by the last product; V or dO is done with earlier in
    // the dQ kernel.  With one ring of five for both, V waited for the slot of a K (3,270 clocks a tile of dQ; with two rings 2,600 then, 2,170 now).
    static constexpr int SLOTS0 = DP == 64 ? 4 : 3, SLOTS1 = DP == 64 ? 4 : 2;
    static constexpr int SMEM = (2 + SLOTS0 + SLOTS1) * TILE_BYTES;
};

// Power of two that brings `most` to 4 .. 8 (1 for zero), and its inverse; fp16 values and their maxima, not infinite.
__device__ __forceinline__ float power_for(float most) { return most > 0.f ? __uint_as_float((256u - (__float_as_uint(most) >> 23)) << 23) : 1.f; }
__device__ __forceinline__ float inverse_power(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }
// The largest finite magnitude of eight fp16 values, as fp16 bits
__device__ __forceinline__ unsigned most_finite(const uint4 &v)
{
    unsigned m = 0;
    for (unsigned w : {v.x, v.y, v.z, v.w}) {
        w &= 0x7fff7fffu;
        m = __vmaxu2(m, w & __vcmpltu2(w, 0x7c007c00u));
    }
    return max(m & 0xffffu, m >> 16);
}

__device__ __forceinline__ F2 pick(const ulonglong2 &v, int second) { return second ? v.y : v.x; }

template <class E, int DP, bool CAP, bool BIAS, bool KV>
__global__ void __launch_bounds__(THREADS, 1) attention_backward_tc_kernel(const AttentionParams p, const __grid_constant__ Maps maps)
{
    using Sh = Shape<DP, KV>;
    constexpr int BOXES = Sh::BOXES, TILE_BYTES = Sh::TILE_BYTES, BOX_BYTES = Sh::BOX_BYTES, SLOTS0 = Sh::SLOTS0, SLOTS1 = Sh::SLOTS1;
    constexpr bool BF16 = !std::is_same<E, __half>::value;
    constexpr bool POWER = !BF16;
    // dK, dV in fp16: P times 2^8 as an operand, since the weights of a long sequence are subnormal (one of 60,000 equal ones was off by 2^-9.5 of itself)
    constexpr float RAISED = POWER && KV ? 8.f : 0.f, RAISE_BY = POWER && KV ? 256.f : 1.f;
    extern __shared__ __align__(1024) unsigned char smem[];  // the block's two tiles, the two rings
    // dQ: s_full = scores and dP there, p_ready = they have been read.  ds_ready, of even and odd tiles: in the dQ kernel a warp may be done with
    // the next tile before another is done with this one, and its arrival must not count for this one.
    __shared__ uint64_t own_full, full[SLOTS0 + SLOTS1], empty[SLOTS0 + SLOTS1], s_full, dp_full, p_ready, ds_ready[2], acc_full, tail, stats_full[2];
    __shared__ uint32_t tmem_holder, bad[4];
    __shared__ __align__(16) float stats[KV ? 4 : 3][T];  // dQ: lse, delta and the largest |dO| of the rows; else lse and delta of the columns, of two tiles
    __shared__ unsigned warp_most[THREADS / 32];
    float *const row_lse = stats[0], *const row_delta = stats[1], *const row_most = stats[KV ? 0 : 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned blocks = gridDim.x / p.n_splits, block_of = blockIdx.x / p.n_splits, part = blockIdx.x % p.n_splits;
    const int heads = KV ? p.kv_heads : p.q_heads, head = block_of % heads, kv = KV ? head : head / p.group;
    Sequence s;
    int seq, block;
    next_kernel_may_come();
    // causal sequences: the last queries see the most keys, the first keys are seen by the most queries
    const bool found = find_block<T>(p, KV ? block_of / heads : (blocks - 1 - block_of) / heads, KV, s, seq, block);
    if (KV) behind_last_kernel();
    if (!found) return;
    const int r0 = block * T, n_rows = min(T, (KV ? s.nk : s.nq) - r0);
    // the tiles of the other side
    Reach reach = {};
    KeyTiles keys = {};
    int from = 0, per_head = 0, tiles;
    if (KV) {
        query_tiles<T>(p, s, r0, n_rows, from, per_head);
        tiles = per_head * p.group;
    } else {
        reach = reach_of(p.window, s, r0, r0 + n_rows);
        keys = key_tiles<T>(reach);
        tiles = keys.n;
    }
    const Part mine_of = part_of(p, tiles, part);
    if (mine_of.end < 0) return;
    const int begin = mine_of.first, count = mine_of.end - begin;
    // streamed tile n: even ones K or Q, odd ones V or dO; its slot, and the how manieth of that slot it is
    auto slot_of = [](int n) { return n & 1 ? SLOTS0 + n / 2 % SLOTS1 : n / 2 % SLOTS0; };
    auto turn_of = [](int n) { return n & 1 ? n / 2 / SLOTS1 : n / 2 / SLOTS0; };
    auto tile_at = [&](int j) { return (KV ? from + (begin + j) % per_head : keys.tile(begin + j)) * T; };
    auto head_at = [&](int j) { return KV ? kv * p.group + (begin + j) / per_head : head; };

    if (threadIdx.x == 0) {
        mbar_init(&own_full, 1);
        mbar_init(&tail, 1);
        for (int i = 0; i < SLOTS0 + SLOTS1; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        mbar_init(&s_full, 1);
        mbar_init(&dp_full, 1);
        mbar_init(&p_ready, ROW_WARPS);
        mbar_init(&ds_ready[0], ROW_WARPS);
        mbar_init(&ds_ready[1], ROW_WARPS);
        mbar_init(&acc_full, 1);
        mbar_init(&stats_full[0], 1);
        mbar_init(&stats_full[1], 1);
        mbar_fence_init();
    }
    if (threadIdx.x < 4) bad[threadIdx.x] = 0;
    if (POWER && KV) {
        unsigned most = 0;  // (as bits: none is negative)
        for (int j = threadIdx.x; j < count; j += THREADS) most = max(most, __float_as_uint(p.d_o_most[tile_index(p, s, seq, head_at(j), tile_at(j) / T)]));
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) warp_most[warp] = most;
    }
    if (warp == MMA_WARP) tc::tmem_alloc(&tmem_holder, TMEM_COLUMNS);
    const int group = warp >> 2, row = (warp & 3) * 32 + lane;  // of warps 0-15: columns MINE * group .. of that row
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_holder, base = tc::smem_u32(smem), ring = base + 2 * TILE_BYTES;
    bool ok = true;
    float power = 1.f;  // fp16: of the row (dQ) or of the block
    if (POWER && KV) {
        unsigned most = 0;
        for (int w = 0; w < THREADS / 32; ++w) most = max(most, warp_most[w]);
        power = power_for(__uint_as_float(most)) * (1.f / RAISE_BY);  // (for a product with raised weights)
    }

    if (warp >= ROW_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 " OTHER_REGISTERS ";");
        if (warp == LOAD_WARP && count > 0) {
            const CUtensorMap *own0 = KV ? &maps.k : &maps.q, *own1 = KV ? &maps.v : &maps.d_o;
            const CUtensorMap *other0 = KV ? &maps.q : &maps.k, *other1 = KV ? &maps.d_o : &maps.v;
            const int own_row = (KV ? s.k0 : s.q0) + r0, other_row = KV ? s.q0 : s.k0, there = KV ? s.nq : s.nk;
            if (lane == 0) {
                tc::expect_bytes(&own_full, 2 * TILE_BYTES);
                for (int b = 0; b < BOXES; ++b) tc::load_box(base + b * BOX_BYTES, own0, 64 * b, head, own_row, &own_full);
                for (int b = 0; b < BOXES; ++b) tc::load_box(base + TILE_BYTES + b * BOX_BYTES, own1, 64 * b, head, own_row, &own_full);
            }
            int issued = 0;
            unsigned tails = 0;
            for (int n = 0; n < 2 * count && ok; ++n) {
                const int slot = slot_of(n), turn = turn_of(n), t0 = tile_at(n / 2), of = KV ? head_at(n / 2) : kv;
                if (turn > 0) ok = tc::warp_wait(&empty[slot], (turn - 1) & 1);
                if (!ok) break;
                // rows behind the sequence's end, where they meet zero weights in a product: zeros (0 x NaN is NaN)
                const bool second = n & 1, cut = (KV || !second) && t0 + T > there;
                const uint32_t at = ring + slot * TILE_BYTES;
                uint64_t *bar = cut ? &tail : &full[slot];
                if (lane == 0) {
                    tc::expect_bytes(bar, TILE_BYTES);
                    for (int b = 0; b < BOXES; ++b) tc::load_box(at + b * BOX_BYTES, second ? other1 : other0, 64 * b, of, other_row + t0, bar);
                }
                ++issued;
                if (cut) {
                    ok = tc::warp_wait(&tail, tails++ & 1);
                    if (!ok) break;
                    tc::zero_rows<T, BOXES>(smem + (2 + slot) * TILE_BYTES, there - t0);
                    tc::fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[slot]);
                }
            }
            // copies of a role that gave up still land in this block's shared memory: wait for them
            if (!ok)
                for (int n = max(0, issued - 2 * max(SLOTS0, SLOTS1)); n < issued; ++n) (void)tc::wait(&full[slot_of(n)], turn_of(n) & 1);
        } else if (KV && warp == STATS_WARP) {
            int tile = count > 0 ? tile_at(0) : 0, of = count > 0 ? head_at(0) : 0;
            for (int j = 0; j < count && ok; ++j) {
                if (j >= 2) ok = tc::warp_wait(&ds_ready[j & 1], (j - 2) >> 1 & 1);  // of tile j - 2: the rows are done with its values
                if (!ok) break;
                const int64_t at = (int64_t)of * p.q_rows + s.q0;  // (delta: an ordinary load, the kernel before wrote it while this one may have been there)
#pragma unroll
                for (int x = 0; x < T / 32; ++x) {
                    const int i = tile + 32 * x + lane;
                    const float l = i < s.nq ? __ldg(p.lse + at + i) : -INFINITY, d = i < s.nq ? p.delta[at + i] : 0.f;
                    stats[(2 * j & 2)][32 * x + lane] = l == -INFINITY ? -INFINITY : fmaf(-l, LOG2E, RAISED);  // nothing seen: weights of zero
                    stats[(2 * j & 2) + 1][32 * x + lane] = POWER ? -d * power : -d;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&stats_full[j & 1]);
                tile += T;
                if (tile == (from + per_head) * T) tile = from * T, ++of;
            }
        } else if (warp == MMA_WARP) {
            constexpr uint32_t ID_S = tc::instr_desc(BF16, T, T, false, false), ID_ACC = tc::instr_desc(BF16, T, DP, false, true);
            const uint64_t own_desc = tc::smem_desc(base, 16), rows_desc = tc::smem_desc(ring, 16), tile_desc = tc::smem_desc(ring, BOX_BYTES);
            // own tile x (0 or 1) times the streamed tile of a slot, rows by rows
            auto rows_by_rows = [&](uint32_t to, int x, int slot) {
                const uint64_t a = own_desc + x * (TILE_BYTES >> 4), b = rows_desc + __shfl_sync(0xffffffffu, slot, 0) * (TILE_BYTES >> 4);
                if (tc::elected()) {
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        const int o = (k / 4 * BOX_BYTES + k % 4 * 32) >> 4;
                        tc::mma_ss(tmem + to, a + o, b + o, ID_S, k > 0);
                    }
                }
                __syncwarp();
            };
            // accumulator += weights (runs of 16 columns, `apart` columns from one to the next) times the streamed tile
            auto weights_by_tile = [&](uint32_t to, uint32_t weights, uint32_t apart, int slot, bool add) {
                const uint64_t b = tile_desc + __shfl_sync(0xffffffffu, slot, 0) * (TILE_BYTES >> 4);
                if (tc::elected()) {
#pragma unroll
                    for (int k = 0; k < T / 16; ++k)
                        tc::mma_ts(tmem + to, tmem + weights + k / 2 * apart + k % 2 * 8, b + k * (2048 >> 4), ID_ACC, add || k > 0);
                }
                __syncwarp();
            };
            auto done = [&](uint64_t *bar) {
                if (tc::elected()) tc::commit(bar);
            };
            auto wait_tile = [&](int n) {
                ok = ok && tc::warp_wait(&full[slot_of(n)], turn_of(n) & 1);
                tc::fence_after();
                return ok;
            };
            if (count > 0) {
                ok = tc::warp_wait(&own_full, 0);
                if (ok && wait_tile(0)) {
                    rows_by_rows(S_AT, 0, 0);
                    if (KV) done(&s_full);
                    if (wait_tile(1)) {
                        rows_by_rows(DP_AT, 1, slot_of(1));
                        done(KV ? &dp_full : &s_full);
                        if (!KV) done(&empty[slot_of(1)]);
                    }
                }
            }
            for (int j = 0; j < count && ok; ++j) {
                const int n = 2 * j;
                const bool more = j + 1 < count;
                if (KV) {
                    ok = tc::warp_wait(&p_ready, j & 1);
                    if (!ok) break;
                    tc::fence_after();
                    weights_by_tile(DV_AT, S_AT, MINE, slot_of(n + 1), j > 0);
                    done(&empty[slot_of(n + 1)]);
                    if (more) {
                        if (!wait_tile(n + 2)) break;
                        rows_by_rows(S_AT, 0, slot_of(n + 2));
                        done(&s_full);
                    }
                    ok = tc::warp_wait(&ds_ready[j & 1], j >> 1 & 1);
                    if (!ok) break;
                    tc::fence_after();
                    weights_by_tile(DK_AT, DP_AT, MINE, slot_of(n), j > 0);
                    done(&empty[slot_of(n)]);
                    if (more) {
                        if (!wait_tile(n + 3)) break;
                        rows_by_rows(DP_AT, 1, slot_of(n + 3));
                        done(&dp_full);
                    }
                } else {
                    if (more) {
                        if (!wait_tile(n + 2)) break;
                        ok = tc::warp_wait(&p_ready, j & 1);
                        if (!ok) break;
                        tc::fence_after();
                        rows_by_rows(S_AT, 0, slot_of(n + 2));
                        if (!wait_tile(n + 3)) break;
                        rows_by_rows(DP_AT, 1, slot_of(n + 3));
                        done(&s_full);
                        done(&empty[slot_of(n + 3)]);
                    }
                    ok = tc::warp_wait(&ds_ready[j & 1], j >> 1 & 1);
                    if (!ok) break;
                    tc::fence_after();
                    weights_by_tile(DQ_AT, DS_AT + 64 * (j & 1), MINE / 2, slot_of(n), j > 0);
                    done(&empty[slot_of(n)]);
                }
            }
            // nothing of this block is in flight when it ends, also where a role has given up
            done(&acc_full);
            __syncwarp();
            ok = tc::warp_wait(&acc_full, 0) && ok;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 " ROW_REGISTERS ";");
        if (!KV) {
            // delta: 16 bytes of O and dO in each lane, DP / 8 lanes a row, all rows of the warp asked for at once
            constexpr int LANES = DP / 8, AT_ONCE = 32 / LANES, TURNS = T / ROW_WARPS / AT_ONCE;
            uint4 o[TURNS], d_o[TURNS];
            float l[TURNS];
            const int c = lane % LANES * 8;
#pragma unroll
            for (int k = 0; k < TURNS; ++k) {
                const int r = warp * (T / ROW_WARPS) + k * AT_ONCE + lane / LANES;
                const int64_t at = (int64_t)s.q0 + r0 + r;
                o[k] = d_o[k] = make_uint4(0, 0, 0, 0);
                l[k] = r < n_rows ? __ldg(p.lse + (int64_t)head * p.q_rows + at) : -INFINITY;
                if (r < n_rows && c < p.head_dim) {
                    o[k] = *reinterpret_cast<const uint4 *>(static_cast<const E *>(p.o.data) + at * p.o.row + head * p.o.head + c);
                    d_o[k] = *reinterpret_cast<const uint4 *>(static_cast<const E *>(p.d_o.data) + at * p.d_o.row + head * p.d_o.head + c);
                }
            }
#pragma unroll
            for (int k = 0; k < TURNS; ++k) {
                const int r = warp * (T / ROW_WARPS) + k * AT_ONCE + lane / LANES;
                const E *a = reinterpret_cast<const E *>(&o[k]), *b = reinterpret_cast<const E *>(&d_o[k]);
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) d = fmaf(to_f(a[e]), to_f(b[e]), d);
#pragma unroll
                for (int x = LANES / 2; x >= 1; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
                if (POWER) {
                    unsigned most = most_finite(d_o[k]);
#pragma unroll
                    for (int x = LANES / 2; x >= 1; x >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, x));
                    if (lane % LANES == 0) row_most[r] = __half2float(__ushort_as_half((unsigned short)most));
                }
                if (lane % LANES == 0) {
                    const int64_t at = (int64_t)head * p.q_rows + s.q0 + r0 + r;
                    row_delta[r] = d;
                    row_lse[r] = l[k];
                    if (r < n_rows && part == 0) p.delta[at] = d;
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(ROW_WARPS * 32) : "memory");  // (all row warps come here, and nothing before can keep one)
            if (POWER && warp == 0 && part == 0) {
                unsigned most = 0;
                for (int r = lane; r < T; r += 32) most = max(most, __float_as_uint(row_most[r]));
                most = __reduce_max_sync(0xffffffffu, most);
                if (lane == 0) p.d_o_most[tile_index(p, s, seq, head, block)] = __uint_as_float(most);
            }
        }
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const float c = !CAP ? p.scale * LOG2E : p.of_cap, top_of = p.cap * LOG2E;
        const tc::Tanh tanh_c = tc::tanh_polynomial(c, 1.f);
        float slope = BIAS && !KV ? __ldg(p.slopes + head) * LOG2E : 0.f;
        const int off = s.nk - s.nq;
        // what a row sees: columns [lo, hi] of the other side, and the first `pre`
        int lo, hi, pre;
        float lse2 = 0.f, delta = 0.f;  // dQ: of the row, negative
        if (KV) {
            const int j = r0 + row;
            pre = j < s.prefix ? s.nq : 0;
            lo = p.window.right < 0 ? 0 : max(0, j - p.window.right - off);
            hi = p.window.left < 0 ? s.nq - 1 : min(s.nq - 1, j + p.window.left - off);
            if (row >= n_rows) pre = 0, lo = 0, hi = -1;
        } else {
            const int pos = off + r0 + row;
            pre = s.prefix;
            lo = p.window.left < 0 ? 0 : max(0, pos - p.window.left);
            hi = p.window.right < 0 ? s.nk - 1 : min(s.nk - 1, pos + p.window.right);
            if (POWER) power = power_for(row_most[row]);
            delta = POWER ? -row_delta[row] * power : -row_delta[row];
            lse2 = row_lse[row] == -INFINITY ? -INFINITY : -row_lse[row] * LOG2E;  // a row that has seen nothing: weights of zero
        }
        int next_tile = KV && count > 0 ? tile_at(0) : 0, next_head = KV && count > 0 ? head_at(0) : 0;  // dK, dV
        for (int j = 0; j < count && ok; ++j) {
            const int t0 = KV ? next_tile : tile_at(j), c0 = t0 + MINE * group;
            const float *const my_lse = stats[2 * j & 2] + MINE * group, *const my_delta = stats[(2 * j & 2) + 1] + MINE * group;
            if (KV) {
                if (BIAS) slope = __ldg(p.slopes + next_head) * LOG2E;
                next_tile += T;
                if (next_tile == (from + per_head) * T) next_tile = from * T, ++next_head;
            }
            bool open;
            if (KV) open = n_rows == T && t0 + T <= s.nq && tile_is_open<T>(p.window, s, reach_of(p.window, s, t0, t0 + T), r0);
            else open = tile_is_open<T>(p.window, s, reach, t0);
            const unsigned seen = open ? ~0u : seen_bits(lo, hi, pre, c0);
            if (KV) ok = tc::warp_wait(&stats_full[j & 1], j >> 1 & 1);
            ok = ok && tc::warp_wait(&s_full, j & 1);
            if (!ok) break;
            tc::fence_after();
            F2 x[MINE / 2], y[MINE / 2];  // two columns each
            tc::tmem_ld32(reinterpret_cast<uint32_t *>(x), mine + S_AT + MINE * group);
            if (!KV) tc::tmem_ld32(reinterpret_cast<uint32_t *>(y), mine + DP_AT + MINE * group);
            tc::wait_ld();
            if (!KV) {
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready);  // the next tile's scores may come
            }
            const float away = KV ? (float)(off + c0 - (r0 + row)) : (float)(c0 - (off + r0 + row));
            bool small = true;
            if (CAP) {
                float size = 0.f;
#pragma unroll
                for (int u = 0; u < MINE / 2; ++u) {
                    float a, b;
                    tc::split(x[u], a, b);
                    size = tc::max3_abs(size, a, b);
                }
                small = p.pre == 1.f && __all_sync(0xffffffffu, size <= tanh_c.range);
            }
            // weights into w; x leaves as weight, with a cap times 1 - tanh^2
            uint32_t w[MINE / 2];
            auto weigh = [&](auto all_seen, auto is_small) {
#pragma unroll
                for (int u = 0; u < MINE / 2; ++u) {
                    const F2 l2 = KV ? pick(reinterpret_cast<const ulonglong2 *>(my_lse)[u / 2], u & 1) : tc::two(lse2, lse2);
                    F2 z = x[u], dcap = 0;
                    if (CAP) {
                        const F2 th = decltype(is_small)::value ? tc::tanh2(z, tanh_c) : tc::tanh_any(tc::mul2(z, tc::two(p.pre, p.pre)), tanh_c, c, 1.f, 0.f);
                        dcap = tc::ffma2(tc::mul2(th, th), tc::two(-1.f, -1.f), tc::two(1.f, 1.f));
                        z = BIAS ? tc::mul2(th, tc::two(top_of, top_of)) : tc::ffma2(th, tc::two(top_of, top_of), l2);
                    }
                    if (BIAS) {
                        const F2 far = tc::two(-slope * fabsf(away + 2.f * u), -slope * fabsf(away + (2.f * u + 1.f)));
                        z = CAP ? tc::add2(z, far) : tc::ffma2(z, tc::two(c, c), far);
                    }
                    if (BIAS) z = tc::add2(z, l2);
                    else if (!CAP) z = tc::ffma2(z, tc::two(c, c), l2);
                    float e0, e1;
                    tc::split(z, e0, e1);
                    e0 = tc::ex2(e0), e1 = tc::ex2(e1);
                    if (!decltype(all_seen)::value) {
                        e0 = seen & 1u << 2 * u ? e0 : 0.f;
                        e1 = seen & 2u << 2 * u ? e1 : 0.f;
                    }
                    x[u] = tc::two(e0, e1);
                    if (KV) w[u] = tc::pack<E>(e0, e1);
                    if (CAP) {
                        x[u] = tc::mul2(x[u], dcap);
                        if (!decltype(all_seen)::value) {  // (the slope of a hidden score may be NaN)
                            tc::split(x[u], e0, e1);
                            x[u] = tc::two(seen & 1u << 2 * u ? e0 : 0.f, seen & 2u << 2 * u ? e1 : 0.f);
                        }
                    }
                }
            };
            if (open && small) weigh(std::true_type(), std::true_type());
            else if (small) weigh(std::false_type(), std::true_type());
            else weigh(std::false_type(), std::false_type());
            if (KV) {
                tc::tmem_st16(mine + S_AT + MINE * group, w);
                tc::wait_st();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready);
                ok = tc::warp_wait(&dp_full, j & 1);
                if (!ok) break;
                tc::fence_after();
                tc::tmem_ld32(reinterpret_cast<uint32_t *>(y), mine + DP_AT + MINE * group);
                tc::wait_ld();
            }
#pragma unroll
            for (int u = 0; u < MINE / 2; ++u) {
                const F2 d = KV ? pick(reinterpret_cast<const ulonglong2 *>(my_delta)[u / 2], u & 1) : tc::two(delta, delta);
                float g0, g1;
                tc::split(tc::mul2(x[u], POWER ? tc::ffma2(y[u], tc::two(power, power), d) : tc::add2(y[u], d)), g0, g1);
                w[u] = tc::pack<E>(g0, g1);
            }
            if (!open) {
                // hidden: zero whatever dP holds
#pragma unroll
                for (int u = 0; u < MINE / 2; ++u) w[u] &= (seen & 1u << 2 * u ? 0xffffu : 0u) | (seen & 2u << 2 * u ? 0xffff0000u : 0u);
            }
            tc::tmem_st16(mine + (KV ? DP_AT + MINE * group : DS_AT + 64 * (j & 1) + MINE / 2 * group), w);
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ds_ready[j & 1]);
        }
        if (ok) ok = tc::warp_wait(&acc_full, 0);
        if (ok) {
            tc::fence_after();
            // dQ: the columns shared out over the groups of warps; dK, dV: an array in two groups each
            constexpr int COLUMNS = KV ? DP / 2 : DP / 4 < 32 ? 32 : DP / 4;
            const HeadArray &to = KV ? (group < 2 ? p.dv : p.dk) : p.dq;
            const int first = COLUMNS * (KV ? group & 1 : group);
            const uint32_t from_column = (KV ? (group < 2 ? DV_AT : DK_AT) : DQ_AT) + first;
            const float by = (KV && group < 2 ? 1.f : POWER ? p.scale * inverse_power(power) : p.scale) * (1.f / RAISE_BY);
            float zero = 0.f;  // NaN as soon as a result is not finite
            if (first < DP) {
                unsigned char *const stage = smem + warp * 32 * COLUMNS * 2;  // the block's own tiles are done with
#pragma unroll
                for (int b = 0; b < COLUMNS / 32; ++b) {
                    float o[32];
                    if (count > 0) {
                        tc::tmem_ld32(reinterpret_cast<uint32_t *>(o), mine + from_column + 32 * b);
                        tc::wait_ld();
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        o[i] = count > 0 ? o[i] * by : 0.f;
                        zero = fmaf(o[i], 0.f, zero);
                    }
                    if (mine_of.alone) {
                        tc::stage_32<E, COLUMNS>(stage, 32 * b, o);
                    } else if (row < n_rows) {
                        const int64_t array = (KV ? p.k_rows : p.q_rows) * heads * p.head_dim;
                        float *sums = p.part_o + (KV ? 2 * part + (group < 2) : part) * array + (((KV ? s.k0 : s.q0) + (int64_t)r0 + row) * heads + head) * p.head_dim;
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (first + 32 * b + i < p.head_dim) *reinterpret_cast<float4 *>(sums + first + 32 * b + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
                const int row0 = (warp & 3) * 32;
                if (mine_of.alone)
                    tc::store_staged<E, COLUMNS>(stage, static_cast<E *>(to.data) + ((int64_t)(KV ? s.k0 : s.q0) + r0 + row0) * to.row + head * to.head + first,
                                             to.row, n_rows - row0, p.head_dim - first);
            }
            const unsigned rows = __ballot_sync(0xffffffffu, zero != 0.f && row < n_rows && mine_of.alone);
            if (lane == 0 && rows) atomicOr(&bad[warp & 3], rows);
        }
    }
    if (!ok && lane == 0) dev::report_timeout(p.status);
    tc::fence_before();
    __syncthreads();
    if (warp == MMA_WARP) tc::tmem_dealloc(tmem, TMEM_COLUMNS);
    if (warp < ROW_WARPS)
        for (int q = 0; q < 4; ++q)
            for (unsigned left = bad[q], turn = 0; left; left &= left - 1, ++turn)
                if (turn % ROW_WARPS == (unsigned)warp) {
                    const int r = 32 * q + __ffs(left) - 1;
                    if (KV) strict::dkv_row<E>(p, s, kv, r0 + r);
                    else strict::dq_row<E>(p, s, head, r0 + r, row_lse[r], row_delta[r]);
                }
}

template <class E, int DP, bool CAP, bool BIAS>
cudaError_t launch(const AttentionParams &p0, const Parts &parts, const Maps &maps, cudaStream_t s)
{
    static SmemOptinCache optin_q, optin_kv;
    constexpr size_t smem_q = Shape<DP, false>::SMEM, smem_kv = Shape<DP, true>::SMEM;
    cudaError_t e = optin_dynamic_smem(attention_backward_tc_kernel<E, DP, CAP, BIAS, false>, smem_q, optin_q);
    if (e == cudaSuccess) e = optin_dynamic_smem(attention_backward_tc_kernel<E, DP, CAP, BIAS, true>, smem_kv, optin_kv);
    if (e != cudaSuccess) return e;
    const unsigned grid_q = (unsigned)(p0.q_heads * most_blocks(p0.q_rows, p0.n_seqs, p0.max_q, T));
    const unsigned grid_kv = (unsigned)(p0.kv_heads * most_blocks(p0.k_rows, p0.n_seqs, p0.max_k, T));
    AttentionParams p = p0;
    p.n_splits = parts.n_q;
    p.chunk_tiles = parts.tiles_q;
    if (grid_q) attention_backward_tc_kernel<E, DP, CAP, BIAS, false><<<grid_q * parts.n_q, THREADS, smem_q, s>>>(p, maps);
    e = cudaGetLastError();
    if (e == cudaSuccess && parts.n_q > 1) e = launch_attention_sum_parts(p, false, T, s);
    if (e != cudaSuccess) return e;
    p.n_splits = parts.n_kv;
    p.chunk_tiles = parts.tiles_kv;
    if (grid_kv && grid_q) {
        e = launch_behind(attention_backward_tc_kernel<E, DP, CAP, BIAS, true>, grid_kv * parts.n_kv, THREADS, smem_kv, s, p, maps);
    } else if (grid_kv) {
        attention_backward_tc_kernel<E, DP, CAP, BIAS, true><<<grid_kv * parts.n_kv, THREADS, smem_kv, s>>>(p, maps);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess && parts.n_kv > 1) e = launch_attention_sum_parts(p, true, T, s);
    return e;
}
template <class E, int DP>
cudaError_t by_score(const AttentionParams &p, const Parts &parts, const Maps &maps, cudaStream_t s)
{
    if (p.cap > 0.f) return p.slopes ? launch<E, DP, true, true>(p, parts, maps, s) : launch<E, DP, true, false>(p, parts, maps, s);
    return p.slopes ? launch<E, DP, false, true>(p, parts, maps, s) : launch<E, DP, false, false>(p, parts, maps, s);
}

// 16-byte accesses to the rows of an array
bool wide(const HeadArray &a) { return (uintptr_t)a.data % 16 == 0 && a.row % 8 == 0 && a.head % 8 == 0; }

}  // namespace

cudaError_t launch_attention_backward_tc(const AttentionParams &p, const Parts &parts, bool *taken, cudaStream_t s)
{
    Maps maps;
    *taken = p.dtype != 0 && wide(p.o) && wide(p.d_o) && wide(p.dq) && wide(p.dk) && wide(p.dv) &&
             make_tensor_map(&maps.q, p.q, p.dtype, p.head_dim, p.q_heads, p.q_rows, T) &&
             make_tensor_map(&maps.k, p.k, p.dtype, p.head_dim, p.kv_heads, p.k_rows, T) &&
             make_tensor_map(&maps.v, p.v, p.dtype, p.head_dim, p.kv_heads, p.k_rows, T) &&
             make_tensor_map(&maps.d_o, p.d_o, p.dtype, p.head_dim, p.q_heads, p.q_rows, T);
    if (!*taken) return cudaSuccess;
    if (p.dtype == 1) return p.head_dim <= 64 ? by_score<__half, 64>(p, parts, maps, s) : by_score<__half, 128>(p, parts, maps, s);
    return p.head_dim <= 64 ? by_score<__nv_bfloat16, 64>(p, parts, maps, s) : by_score<__nv_bfloat16, 128>(p, parts, maps, s);
}

}  // namespace sddmm
