// tcgen05, TMEM and packed fp32 as the attention and the 4-bit kernels use them (sm_100a, one block's tensor core).
#pragma once

#include "lora_pipe.cuh"

namespace b200lora {

namespace {

constexpr int kTcRows = 128;                       // rows of a multiplication, and lanes of TMEM
constexpr int kTmemCols = 512;

__device__ __forceinline__ void tmem_alloc(unsigned smem_dst) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "n"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(unsigned taddr) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "n"(kTmemCols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Bounded wait that says whether the phase is complete; on expiry it records `code`, and others then give up early.  A thread that issues
// copies or multiplications issues no more once a wait of its has expired, and nobody whose wait has expired says that a place
// may be filled again: so no barrier is armed while a phase of it is open.  At the end of the block, whoever issued
// something waits for it (mbar_drain, with a limit too) before its place is used for anything else, freed, or left to the next block.
__device__ __forceinline__ bool mbar_reached(unsigned bar, unsigned parity, unsigned* err, unsigned code) {
    for (unsigned i = 0; i < kSpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 0x3ffu) == 0x3ffu && *reinterpret_cast<volatile unsigned*>(err) != 0u) return false;
    }
    atomicMax(err, code);
    return false;
}
__device__ __forceinline__ void mbar_drain(unsigned bar, unsigned parity) {
    for (unsigned i = 0; i < kSpinLimit && !mbar_try_wait(bar, parity); ++i) {}
}
// Shared-memory operands with 128-byte swizzle: panels of 64 elements, [rows][128 bytes], 16-byte piece c of row r at
// c ^ (r % 8); 1024 bytes from one eight rows to the next.  Their descriptors as two words, of which only the low one
// changes: address in units of 16 bytes, and above it for an operand whose rows are the contraction the distance of two panels.
constexpr unsigned kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr unsigned kPanel = kTcRows * 128;                // bytes of a panel of 128 rows
constexpr unsigned kRowsAreRows = 1u << 16, kRowsAreDepth = (kPanel >> 4) << 16;
__device__ __forceinline__ unsigned desc_low(unsigned saddr, unsigned kind) { return ((saddr >> 4) & 0x3fffu) | kind; }
// D (+)= A B^T, A and B from shared memory
template <bool ACC>
__device__ __forceinline__ void mma_ss(unsigned d, unsigned a, unsigned b, unsigned idesc) {
    asm volatile("{ .reg .pred p; .reg .b64 x, y; mov.b64 x, {%1, %3}; mov.b64 y, {%2, %3}; setp.ne.b32 p, %5, 0;"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p; }"
                 ::"r"(d), "r"(a), "r"(b), "r"(kDescHigh), "r"(idesc), "n"(ACC) : "memory");
}
// D (+)= A B, A from TMEM
__device__ __forceinline__ void mma_ts(unsigned d, unsigned a, unsigned b, unsigned idesc, unsigned accumulate) {
    asm volatile("{ .reg .pred p; .reg .b64 y; mov.b64 y, {%2, %3}; setp.ne.b32 p, %5, 0;"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p; }"
                 ::"r"(d), "r"(a), "r"(b), "r"(kDescHigh), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_ld32(unsigned taddr, unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
          "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_st32(unsigned taddr, const unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
          "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
          "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_st16(unsigned taddr, const unsigned (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tc_ld16(unsigned taddr, unsigned (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void lds16(unsigned addr, unsigned (&v)[4]) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void sts16(unsigned addr, unsigned a, unsigned b, unsigned c, unsigned d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// two fp32 numbers at a time
__device__ __forceinline__ unsigned long long pair(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(unsigned long long v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// kind::f16, fp32 sums, M = 128; b_mn: the second operand's rows are the contraction
__device__ __forceinline__ unsigned idesc_of(bool bf16, int n, bool b_mn) {
    const unsigned fmt = bf16 ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn ? 1u << 16 : 0u) | ((unsigned)(n >> 3) << 17) | ((unsigned)(kTcRows >> 4) << 24);
}
// byte address of 16-byte piece `piece` of row `row` in an operand of 128 rows
__device__ __forceinline__ unsigned swizzled(unsigned base, int row, int piece) {
    return base + (piece >> 3) * kPanel + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}

}  // namespace

}  // namespace b200lora
