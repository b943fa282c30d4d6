// Tensor-core building blocks of the attention kernels: tile copies (TMA), shared-memory and instruction descriptors of tcgen05.mma with
// 16-bit operands, tensor memory, bounded waits.
//
// Operand tiles lie in shared memory as boxes of 64 elements (128 bytes) by some rows, with the 128-byte swizzle: the 16-byte piece c of
// row r sits at piece c ^ (r % 8) of the row's line; eight rows are 1,024 bytes.  Two ways to read such a box:
//   K-major  (the 64 elements are the product's K): 16 of them, a K step, are 32 bytes further in every line;
//   MN-major (the rows are the product's K): a K step is 16 rows, 2,048 bytes; boxes beside one another continue M or N.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "attention.cuh"
#include "device_utils.cuh"

namespace sddmm {
namespace tc {

using dev::mbar_arrive;
using dev::mbar_fence_init;
using dev::mbar_init;
using dev::mbar_try_wait;
using dev::smem_u32;

// Shared-memory matrix descriptor: start address, leading / stride byte offsets (all >> 4), version 1, 128-byte swizzle.
// K-major: stride = 1,024 (from eight rows to the next), leading unused.  MN-major: stride = 1,024 (from eight K rows to the
// next), leading = bytes from a box of 64 to the one that continues M or N.
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr, uint32_t lbo_bytes)
{
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)((lbo_bytes >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024u >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptor of kind::f16: D fp32, A and B both fp16 or both bfloat16, K-major or MN-major each.
__host__ __device__ constexpr uint32_t instr_desc(bool bf16, int M, int N, bool a_mn, bool b_mn)
{
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// D (tensor memory) = or += A B^T, one K step of 16; A from shared memory or (ts) from tensor memory, two elements a column.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}
// One thread of a converged warp, the same one every time.  The compiler keeps what such a region computes in uniform registers, which is where
// tcgen05.mma takes its descriptors from; behind a test of the lane number every MMA waits for its operands to be moved there.
__device__ __forceinline__ bool elected()
{
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}
// Arrives on the barrier when all MMAs that this thread has issued are complete.
__device__ __forceinline__ void commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tmem_alloc(uint32_t *holder, uint32_t columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t tmem, uint32_t columns)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// 32 columns of this warp's 32 lanes, a lane's row in a thread; loads are complete behind wait_ld().
#define TC_R8(m, v, i) m(v[i]), m(v[i + 1]), m(v[i + 2]), m(v[i + 3]), m(v[i + 4]), m(v[i + 5]), m(v[i + 6]), m(v[i + 7])
#define TC_OUT(x) "=r"(x)
#define TC_IN(x) "r"(x)
__device__ __forceinline__ void tmem_ld32(uint32_t *v, uint32_t taddr)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : TC_R8(TC_OUT, v, 0), TC_R8(TC_OUT, v, 8), TC_R8(TC_OUT, v, 16), TC_R8(TC_OUT, v, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *v)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::TC_R8(TC_IN, v, 0), TC_R8(TC_IN, v, 8), TC_R8(TC_IN, v, 16),
        TC_R8(TC_IN, v, 24), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t *v, uint32_t taddr)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : TC_R8(TC_OUT, v, 0), TC_R8(TC_OUT, v, 8)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *v)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::TC_R8(TC_IN, v, 0),
        TC_R8(TC_IN, v, 8), "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void expect_bytes(uint64_t *bar, uint32_t bytes)
{
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// Box of a rows x heads x head_dim array: elements from `x` on (a multiple of 64), one head, rows from `row` on.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, int x, int head, int row, uint64_t *bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
        "r"(x), "r"(head), "r"(row), "r"(smem_u32(bar))
        : "memory");
}

// Rows [first, ROWS) of a tile set to zero by a warp (whole rows, so the swizzle does not matter).
template <int ROWS, int BOXES>
__device__ __forceinline__ void zero_rows(unsigned char *tile, int first)
{
    const int lane = threadIdx.x & 31;
    for (int r = first + lane / 8; r < ROWS; r += 4)
#pragma unroll
        for (int b = 0; b < BOXES; ++b) *reinterpret_cast<uint4 *>(tile + b * ROWS * 128 + r * 128 + lane % 8 * 16) = make_uint4(0, 0, 0, 0);
}

// Bounded wait of a thread.  try_wait suspends the thread by itself, so there is no sleep between polls; the limit is wall-clock time, with
// a count behind it.
static __device__ __forceinline__ bool wait_long(uint64_t *bar, unsigned parity)
{
    dev::WaitClock clock;
#pragma unroll 1
    for (int it = 0; it < dev::MBAR_SPIN_LIMIT; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if (clock.expired(it)) return false;
    }
    return false;
}
__device__ __forceinline__ bool wait(uint64_t *bar, unsigned parity) { return mbar_try_wait(bar, parity) || wait_long(bar, parity); }

// The same for a whole warp: one answer for all of its threads.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, unsigned parity) { return __all_sync(0xffffffffu, wait(bar, parity)); }

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// ---- two fp32 values in 64 bits: one instruction for both ----
using F2 = unsigned long long;
using dev::ffma2;
__device__ __forceinline__ F2 two(float a, float b)
{
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split(F2 x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b)
{
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b)
{
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c)
{
    float r;
    asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x of both values without the special function unit, x <= 8: x = n + f, |f| <= 1/2, from adding and taking away 1.5 x 2^23; 2^f as a
// polynomial (Chebyshev interpolation of degree 5: off by 2.5e-7 of the value); 2^n by its exponent, which is 0 for n = -127: from -126.5 down to -inf the result is 0.  NaN stays NaN.
__device__ __forceinline__ F2 ex2_poly(F2 x)
{
    float a, b;
    split(x, a, b);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
    x = two(a, b);
    const float big = 12582912.f;
    const F2 r = add2(x, two(big, big)), f = add2(x, mul2(add2(r, two(-big, -big)), two(-1.f, -1.f)));
    F2 p = two(0.00134004327f, 0.00134004327f);
    p = ffma2(p, f, two(0.00967603736f, 0.00967603736f));
    p = ffma2(p, f, two(0.0555032715f, 0.0555032715f));
    p = ffma2(p, f, two(0.240221068f, 0.240221068f));
    p = ffma2(p, f, two(0.693147182f, 0.693147182f));
    p = ffma2(p, f, two(1.0f, 1.0f));
    split(r, a, b);
    return mul2(p, two(__uint_as_float((__float_as_uint(a) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(b) << 23) + 0x3f800000u)));
}
// tanh(c x) = x (a polynomial in x^2), where |c x| <= 0.6: Chebyshev interpolation of tanh(y) / y in y^2, off by 9e-8, its coefficients
// times by c^(2i + 1).  c^9 has to stay among the normal numbers, with room for `by`: c from TANH_LEAST to TANH_MOST.  Where scale / cap is
// not in there c is 1, and products are multiplied by it (AttentionParams::pre) first and go by tanh_any().
constexpr float TANH_LEAST = 2e-4f, TANH_MOST = 1e4f;
struct Tanh {
    F2 a[5];
    float range;  // of |x|
};
__device__ __forceinline__ Tanh tanh_polynomial(float c, float by)
{
    constexpr float C[5] = {0.99999994f, -0.33332324f, 0.133103579f, -0.0521096252f, 0.0154866902f};
    Tanh t;
    float power = c * by;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        t.a[i] = two(C[i] * power, C[i] * power);
        power *= c * c;
    }
    t.range = 0.6f / c;
    return t;
}
__device__ __forceinline__ F2 tanh_over_x(F2 x, const Tanh &t)
{
    const F2 u = mul2(x, x);
    F2 p = t.a[4];
#pragma unroll
    for (int i = 3; i >= 0; --i) p = ffma2(p, u, t.a[i]);
    return p;
}
__device__ __forceinline__ F2 tanh2(F2 x, const Tanh &t) { return mul2(tanh_over_x(x, t), x); }
// Both values, each from `near` where |x| <= range, else from `far`; as instructions, so that no lane branches.  (With conditional expressions, and
// the other way by single values: 4,096 causal tokens, 8 heads of 128, most scores near their cap, 255 us; so 158.)
__device__ __forceinline__ F2 by_size(F2 x, float range, F2 near, F2 far)
{
    float a, b, n0, n1, f0, f1;
    split(x, a, b), split(near, n0, n1), split(far, f0, f1);
    asm("{\n\t.reg .pred p;\n\tsetp.le.f32 p, %1, %2;\n\tselp.f32 %0, %0, %3, p;\n\t}" : "+f"(n0) : "f"(fabsf(a)), "f"(range), "f"(f0));
    asm("{\n\t.reg .pred p;\n\tsetp.le.f32 p, %1, %2;\n\tselp.f32 %0, %0, %3, p;\n\t}" : "+f"(n1) : "f"(fabsf(b)), "f"(range), "f"(f1));
    return two(n0, n1);
}
// by tanh(c x) + more of any size, for products a few of which leave the polynomial's range: each by its own size alone, so that what comes out
// of one does not depend on the others.  Within the range the bits are those of ffma2(x, tanh_over_x(x, t), more), `by` being in t's factors;
// beyond it by (1 - 2 / (1 + e^2cx)).
__device__ __forceinline__ F2 tanh_any(F2 x, const Tanh &t, float c, float by, float more)
{
    float a, b;
    const float c2 = 2.f * LOG2E * c;
    split(mul2(x, two(c2, c2)), a, b);
    split(add2(two(ex2(a), ex2(b)), two(1.f, 1.f)), a, b);
    const F2 far = ffma2(two(rcp(a), rcp(b)), two(-2.f * by, -2.f * by), two(by + more, by + more));
    return by_size(x, t.range, ffma2(x, tanh_over_x(x, t), two(more, more)), far);
}
// Two values in a word, the first in its lower half.
template <class T> __device__ __forceinline__ uint32_t pack(float a, float b);
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack<__half>(float a, float b)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// Results of a warp, a row a thread, to global memory: through a piece of shared memory (32 rows of COLUMNS 16-bit values) that the warp has to
// itself, so that a store instruction writes whole rows and not 16 bytes of each of 32 rows (which took 16,000 clocks a block).
template <int COLUMNS>
__device__ __forceinline__ uint4 *staged(unsigned char *stage, int row, int piece)  // 16-byte piece of a row, spread over the banks
{
    return reinterpret_cast<uint4 *>(stage + row * COLUMNS * 2 + (piece ^ (row & (COLUMNS / 8 < 8 ? COLUMNS / 8 - 1 : 7))) * 16);
}
template <class E, int COLUMNS>
__device__ __forceinline__ void stage_32(unsigned char *stage, int column, const float (&v)[32])
{
    const int row = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *staged<COLUMNS>(stage, row, column / 8 + i) = make_uint4(pack<E>(v[8 * i], v[8 * i + 1]), pack<E>(v[8 * i + 2], v[8 * i + 3]),
                                                                   pack<E>(v[8 * i + 4], v[8 * i + 5]), pack<E>(v[8 * i + 6], v[8 * i + 7]));
}
// dst: the warp's first row, at the first of COLUMNS columns; `rows` rows and `columns` columns (a multiple of 8) exist.
template <class E, int COLUMNS>
__device__ __forceinline__ void store_staged(const unsigned char *stage, E *dst, int64_t row_stride, int rows, int columns)
{
    __syncwarp();
    constexpr int PIECES = COLUMNS / 8, AT_ONCE = 32 / PIECES;
    const int lane = threadIdx.x & 31, piece = lane % PIECES;
    uint4 v[32 / AT_ONCE];
#pragma unroll
    for (int i = 0; i < 32 / AT_ONCE; ++i) v[i] = *staged<COLUMNS>(const_cast<unsigned char *>(stage), i * AT_ONCE + lane / PIECES, piece);
#pragma unroll
    for (int i = 0; i < 32 / AT_ONCE; ++i) {
        const int row = i * AT_ONCE + lane / PIECES;
        if (row < rows && piece * 8 < columns) *reinterpret_cast<uint4 *>(dst + row * row_stride + piece * 8) = v[i];
    }
    __syncwarp();
}

}  // namespace tc

// Tensor map of one array for boxes of 64 elements x `box_rows` rows; false where the array cannot have one (strides, alignment).
bool make_tensor_map(CUtensorMap *map, const HeadArray &a, int dtype, int head_dim, int heads, int64_t rows, int box_rows);

}  // namespace sddmm
