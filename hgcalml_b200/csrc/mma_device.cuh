// Tensor-core building blocks for kernels whose accumulators live in tensor memory: barriers, tile copies, matrix products.
//
// Tiles in shared memory are rows of 128 bytes, swizzled in groups of eight rows as the copy engine writes them (1024-byte
// aligned); wider rows are several such tiles behind each other.  The same tile serves a product that sums along its rows (K-major)
// and one that sums over them (MN-major).
#pragma once

#include "common.cuh"

namespace hgc {
namespace mma {

__device__ __forceinline__ unsigned smem_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }

// One thread of a warp, the same one every time; all of the warp's lanes call this together.  Copies, products and their commits
// are issued by the thread that it elects and by no other means: in a branch that is merely taken by one lane the assembler
// cannot know that one thread issues, and operands that have to be uniform are gathered lane by lane.
__device__ __forceinline__ bool elect()
{
    unsigned elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected) :: "memory");
    return elected != 0;
}

// ----------------------------------------------------------------------------------------------------------- barriers
__device__ __forceinline__ void barrier_init(unsigned bar, unsigned count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_init_done()
{
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void arrive(unsigned bar)
{
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_expect(unsigned bar, unsigned bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}

// Waits end: after kPatience, or when another wait of the block has given up, the block's flag is set, every later wait returns
// and no more copies or products are issued, so that the block runs to its end and frees its tensor memory.  The clock is looked at
// only after many tries: a try sleeps until the barrier's phase ends or some time has passed.
constexpr long long kPatience = 8000000000ll;  // cycles
__device__ __forceinline__ bool try_wait(unsigned bar, unsigned parity)
{
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ bool wait(unsigned bar, unsigned parity, volatile int *gave_up, unsigned *status)
{
    for (int i = 0; i < 16; i++)
        if (try_wait(bar, parity)) return true;
    const long long begin = clock64();
    do {
        for (int i = 0; i < 64; i++)
            if (try_wait(bar, parity)) return true;
        if (*gave_up) return false;
    } while (clock64() - begin < kPatience);
    *gave_up = 1;
    flag_status(status, HGC_STATUS_ITERATION_CAP);
    return false;
}
static __device__ __noinline__ bool wait_out_of_line(unsigned bar, unsigned parity, volatile int *gave_up, unsigned *status)
{
    return wait(bar, parity, gave_up, status);
}
// For a warp, whose lanes go on together.  LITTLE: with few instructions here, for code that the instruction caches hardly hold
// (forward pass 1.05 -> 0.91 ms at 16k x 16k rows, 8 heads of 64); without it the sums and scores are issued sooner (backward pass
// 2.07 -> 1.84).
template <bool LITTLE = false>
__device__ __forceinline__ bool wait_warp(unsigned bar, unsigned parity, volatile int *gave_up, unsigned *status)
{
    bool done;
    if (LITTLE) done = try_wait(bar, parity) || wait_out_of_line(bar, parity, gave_up, status);
    else done = wait(bar, parity, gave_up, status);
    return __all_sync(0xffffffffu, done);
}
// A wait for what is under way whatever happened before.
__device__ __forceinline__ void drain(unsigned bar, unsigned parity)
{
    const long long begin = clock64();
    while (!try_wait(bar, parity) && clock64() - begin < kPatience) {}
}

// -------------------------------------------------------------------------------------------------------- tile copies
// A box of a three-dimensional tensor (columns, heads, rows) to shared memory; what lies outside the tensor is filled with zeros.
__device__ __forceinline__ void copy_box(unsigned dst, const void *map, unsigned bar, int column, int head, int row)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 :: "r"(dst), "l"(map), "r"(bar), "r"(column), "r"(head), "r"(row) : "memory");
}
// Ordinary writes to shared memory before, products that read them after.
__device__ __forceinline__ void writes_before_products() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---------------------------------------------------------------------------------------------------------- products
template <typename T> struct Code;
template <> struct Code<__half> { static constexpr unsigned value = 0; };
template <> struct Code<__nv_bfloat16> { static constexpr unsigned value = 1; };

// 128 x n products of 16-bit operands with sums in float32; `over_rows`: the second operand is summed over its rows.
template <typename T> __device__ __forceinline__ unsigned shape(int n, bool over_rows)
{
    return (1u << 4) | (Code<T>::value << 7) | (Code<T>::value << 10) | ((over_rows ? 1u : 0u) << 16) | ((unsigned)(n >> 3) << 17) | (8u << 24);
}
// Operand in shared memory; `apart`: bytes between the tiles of 64 columns (used where columns are not summed over).
__device__ __forceinline__ unsigned long long operand(unsigned address, unsigned apart)
{
    return (unsigned long long)((address & 0x3ffff) >> 4) | (unsigned long long)(apart >> 4) << 16 | (unsigned long long)(1024 >> 4) << 32 |
           1ull << 46 | 2ull << 61;
}
// d (+)= a b, 16 summed elements; one thread issues
__device__ __forceinline__ void product(unsigned d, unsigned long long a, unsigned long long b, unsigned shape, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(shape), "r"((unsigned)add) : "memory");
}
// the same with the first operand in tensor memory
__device__ __forceinline__ void product_from_tmem(unsigned d, unsigned a, unsigned long long b, unsigned shape, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(shape), "r"((unsigned)add) : "memory");
}
// The barrier is arrived at when all products that this thread has issued are done.
__device__ __forceinline__ void arrive_when_done(unsigned bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// d[128 x n] = a[128 rows] . b[n rows], both K-major, over 16 `steps` columns; tiles of 64 columns lie A_APART and B_APART bytes
// behind each other.  The thread that issues is a chain of its own, so that all it does per product is to add constants to the
// operands.
template <int CHUNKS, unsigned A_APART, unsigned B_APART>
__device__ __forceinline__ void product_along(unsigned d, unsigned a, unsigned b, int steps, unsigned shape)
{
    const unsigned long long oa = operand(a, 16), ob = operand(b, 16);
#pragma unroll
    for (int k = 0; k < 4 * CHUNKS; k++)
        if (k < steps) product(d, oa + (k / 4 * A_APART + k % 4 * 32) / 16, ob + (k / 4 * B_APART + k % 4 * 32) / 16, shape, k > 0);
}
// d[128 x columns] (+)= a[128 x 16 STEPS] b[16 STEPS rows], tiles of 64 columns APART bytes behind each other.  a is in tensor
// memory, its halves where the 32-bit values were that they come from: the second one begins 8 STEPS columns behind the first.
template <int STEPS, unsigned APART>
__device__ __forceinline__ void product_over(unsigned d, unsigned a, unsigned b, unsigned shape, bool add)
{
    const unsigned long long ob = operand(b, APART);
#pragma unroll
    for (int k = 0; k < STEPS; k++) product_from_tmem(d, a + 8 * k + (2 * k >= STEPS ? 4 * STEPS : 0), ob + 2048 / 16 * k, shape, add || k > 0);
}

// ------------------------------------------------------------------------------------------------------ tensor memory
// One warp allocates and frees; the address is written to shared memory.
__device__ __forceinline__ void tmem_alloc(unsigned *to, unsigned columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_address(to)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(unsigned address, unsigned columns)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(address), "r"(columns) : "memory");
}
#define HGC_R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
#define HGC_R16(v, i) HGC_R4(v, i), HGC_R4(v, i + 4), HGC_R4(v, i + 8), HGC_R4(v, i + 12)
// the same where an input follows that must not share a register with what is written first
#define HGC_E4(v, i) "=&r"(v[i]), "=&r"(v[i + 1]), "=&r"(v[i + 2]), "=&r"(v[i + 3])
#define HGC_E16(v, i) HGC_E4(v, i), HGC_E4(v, i + 4), HGC_E4(v, i + 8), HGC_E4(v, i + 12)
#define HGC_S4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
#define HGC_S16(v, i) HGC_S4(v, i), HGC_S4(v, i + 4), HGC_S4(v, i + 8), HGC_S4(v, i + 12)
// A lane's row of 32 or 16 columns.  Warp w of a group of four reaches rows 32 w .. 32 w + 31.  A load and the wait for it are one
// statement: in between, its registers are written at any time, and the compiler, to which they are values that are there already,
// may have moved these values elsewhere and given the registers to something else.  (Loads and waits apart from each other faulted
// in some builds of the kernels for wide heads, at no fixed place.)
#define HGC_LD32 "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
__device__ __forceinline__ void tmem_load32(unsigned (&v)[32], unsigned address)
{
    asm volatile(HGC_LD32 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, "
                 "%25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : HGC_R16(v, 0), HGC_R16(v, 16) : "r"(address) : "memory");
}
__device__ __forceinline__ void tmem_load32(unsigned (&v)[32], unsigned address, unsigned (&w)[32], unsigned address2)
{
    asm volatile(HGC_LD32 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, "
                 "%25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
                 HGC_LD32 "{%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, "
                 "%55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\ttcgen05.wait::ld.sync.aligned;"
                 : HGC_E16(v, 0), HGC_E16(v, 16), HGC_E16(w, 0), HGC_E16(w, 16) : "r"(address), "r"(address2) : "memory");
}
__device__ __forceinline__ void tmem_load16(unsigned (&v)[16], unsigned address)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : HGC_R16(v, 0) : "r"(address) : "memory");
}
__device__ __forceinline__ void tmem_store16(unsigned address, const unsigned (&v)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 :: "r"(address), HGC_S16(v, 0) : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x)  // relative error 2^-22
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Pairs of floats: one instruction for both.
typedef unsigned long long pair;
__device__ __forceinline__ pair pair_of(float a, float b)
{
    pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 parts(pair a)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ pair fma2(pair a, pair b, pair c)
{
    pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ pair add2(pair a, pair b)
{
    pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ pair mul2(pair a, pair b)
{
    pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// What is no number stays it.
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max2(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 2^x of two floats of at most 127 without the special function unit: 2^n from the integer n next to x, put into the exponent,
// times a polynomial of degree three in x - n that is off by 1.0e-04 at most (root mean square 6.4e-05), less than a quarter of half
// precision's largest rounding.  Its coefficients give the least maximal relative error on [-1/2, 1/2] that goes with 2^0 = 1.
// Below 2^-126 it stays there.  What is no number gives a finite one or an infinity, so a row that may hold it has to tell by
// something else, as its maximum does.
__device__ __forceinline__ float2 exp2_arithmetic(float2 v)
{
    const pair x = pair_of(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
    const pair magic = pair_of(12582912.f, 12582912.f), unmagic = pair_of(-12582912.f, -12582912.f), minus = pair_of(-1.f, -1.f);
    const pair t = add2(x, magic);                        // n in the low bits
    const pair f = fma2(add2(t, unmagic), minus, x);
    pair y = fma2(f, pair_of(0.0550091006f, 0.0550091006f), pair_of(0.242210984f, 0.242210984f));
    y = fma2(y, f, pair_of(0.693282902f, 0.693282902f));
    y = fma2(y, f, pair_of(1.f, 1.f));
    const float2 p = parts(y), n = parts(t);
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(n.x) << 23)),
                       __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(n.y) << 23)));
}
// two floats rounded to 16 bits, the first in the lower half
template <typename T> __device__ __forceinline__ unsigned pack2(float a, float b);
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float a, float b)
{
    unsigned r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <> __device__ __forceinline__ unsigned pack2<__half>(float a, float b)
{
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <typename T> __device__ __forceinline__ float2 unpack2(unsigned v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(unsigned v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }

}  // namespace mma
}  // namespace hgc
