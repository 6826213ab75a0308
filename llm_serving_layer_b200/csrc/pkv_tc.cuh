// pkv_tc.cuh — what the tcgen05 / TMEM attention kernels share: tile constants,
// descriptors, tensor-memory loads and stores, the softmax inner loop and the
// work-claim counters.
#pragma once

#include "pkv_common.cuh"

namespace pkv {

constexpr int TC_D = 64;                      // head_dim
constexpr int TC_P = 16;                      // tokens per page
constexpr int TC_ROWS = 128;                  // query rows per CTA (UMMA M)
constexpr int TC_KB = 64;                     // keys per block (UMMA N of S)
constexpr int TC_PPB = TC_KB / TC_P;          // pages per block
constexpr int TC_PAGE = TC_P * TC_D * 2;      // 2 KiB: one head's slice of a page
constexpr int TC_KTILE = TC_KB * TC_D * 2;    // 8 KiB
constexpr int TC_QTILE = TC_ROWS * TC_D * 2;  // 16 KiB
constexpr int TC_THREADS = 192;
constexpr float TC_RESCALE = 8.f;             // rescale O when the max grows by > 2^8

// ---------------------------------------------------------------- tcgen05 helpers
// Shared-memory matrix descriptor, 128B swizzle: start address, leading byte
// offset 16 B (unused by swizzled K-major; one 64-element atom in MN), stride
// byte offset 1024 B between 8-row groups, descriptor version 1.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
  return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor of kind::f16: fp32 accumulate, A/B element format
// (0 = f16, 1 = bf16, always equal), A K-major, B K- or MN-major, N, M = 128.
__host__ __device__ constexpr uint32_t idesc_f16(int fmt, int b_mn_major, int n) {
  return (1u << 4) | (uint32_t(fmt) << 7) | (uint32_t(fmt) << 10) | (uint32_t(b_mn_major) << 16) |
         (uint32_t(n >> 3) << 17) | (uint32_t(TC_ROWS >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// arrive on `bar` once every tcgen05 operation this thread issued so far completed
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

#define PKV_R8(i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define PKV_W8(i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])

// 32 consecutive 32-bit TMEM columns of this thread's lane; waits for the load
// inside the same asm statement, so the registers are valid when it returns.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : PKV_R8(0), PKV_R8(8), PKV_R8(16), PKV_R8(24)
      : "r"(taddr)
      : "memory");
}
// 64 consecutive 32-bit TMEM columns (two loads, one wait).
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : PKV_R8(0), PKV_R8(8), PKV_R8(16), PKV_R8(24), PKV_R8(32), PKV_R8(40), PKV_R8(48), PKV_R8(56)
      : "r"(taddr), "r"(taddr + 32)
      : "memory");
}
// 32 consecutive 32-bit TMEM columns of this thread's lane <- r; waits for the store.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n\t"
      "tcgen05.wait::st.sync.aligned;" ::"r"(taddr),
      PKV_W8(0), PKV_W8(8), PKV_W8(16), PKV_W8(24)
      : "memory");
}
#undef PKV_R8
#undef PKV_W8

// Packed fp32 pairs (sm_100's two-wide FMA / add) and a three-input max: the
// softmax threads are bound by instruction issue, so each pair of scores
// takes one FMA and one add instead of two each.
__device__ __forceinline__ unsigned long long f32x2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f32x2_split(unsigned long long v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma_f32x2(unsigned long long a, unsigned long long b,
                                                        unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long add_f32x2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                                           int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n\t"
      "tcgen05.wait::st.sync.aligned;" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// O row *= alpha (the lazy rescale; rare): out of line, so that the registers
// it needs are saved on its own path and not reserved in the block loop.
static __device__ __noinline__ void tl_rescale_o(uint32_t tO, float alpha) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t o[16];
    tmem_ld16(tO + q * 16, o);
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
    tmem_st16(tO + q * 16, o);
  }
}

// exp2(s * sc - mu) of a row's 64 scores, packed to pairs of the pool dtype
// and stored as the row of P in shared memory (16-byte chunk c of row r at
// r * 128 + ((c ^ (r & 7)) << 4): the 128B swizzle of a K-major operand); the
// sum of the exponentials, as they were before that rounding, is added to `l`.
// The rounding is the tensor cores' operand type: relative 2^-11 (fp16) or 2^-8
// (bf16) of weights that sum to 1 moves an output by that part of max |v| at most,
// as its own rounding does; a 32-bit P would be a tf32 product at half the rate.
template <typename T>
__device__ __forceinline__ void tl_exp64_smem(const uint32_t (&s)[64], unsigned long long sc2,
                                              unsigned long long nmu2, float& l, unsigned char* prow, int r) {
  unsigned long long lt2[2] = {0ull, 0ull};
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t pk[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = c * 8 + 2 * i;
      float x0, x1;
      f32x2_split(fma_f32x2(f32x2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), sc2, nmu2), x0, x1);
      const float p0 = ex2(x0), p1 = ex2(x1);
      lt2[i & 1] = add_f32x2(lt2[i & 1], f32x2(p0, p1));
      pk[i] = MmaOp<T>::pack(p0, p1);
    }
    *reinterpret_cast<uint4*>(prow + ((c ^ (r & 7)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
  }
  float a0, a1, b0, b1;
  f32x2_split(lt2[0], a0, a1);
  f32x2_split(lt2[1], b0, b1);
  l += (a0 + a1) + (b0 + b1);
}

// A CTA of the lean kernel is done with the claim counter: the last one of
// the launch zeroes both counters for the next launch with the same plan
// (which claims only after its griddepcontrol.wait, i.e. after this launch
// completed).
__device__ __forceinline__ void tl_count_exit(int32_t* claim) {
  __threadfence();
  if (atomicAdd(claim + 1, 1) == int(gridDim.x) - 1) {
    claim[0] = 0;
    claim[1] = 0;
    __threadfence();
  }
}

// Tensor map of the step's query rows (pkv_prefill_tc.cu).
int q_tmap(int32_t dtype, const void* q, int n_tokens, int n_heads, int groups, CUtensorMap* out);

}  // namespace pkv
