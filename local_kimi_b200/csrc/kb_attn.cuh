// kb_attn.cuh - pieces shared by the attention kernels: the error path of
// bounded waits, 16-bit element types, warp-level matrix steps and the host's
// argument checks and tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "kb_math.cuh"

namespace kb {
namespace attn {

constexpr uint32_t ERR_WAIT = 2u;               // bounded wait ran out (device error bit 1)
constexpr long long WAIT_NS = 2000000000LL;
constexpr long long DRAIN_NS = 200000000LL;
constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ long long now_ns() {
  long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// A try that lets the hardware put the thread to sleep for up to `ns`.
__device__ __forceinline__ bool mbar_try_wait_for(uint64_t* bar, uint32_t parity, uint32_t ns) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity), "r"(ns)
      : "memory");
  return ok != 0;
}

// Bounded wait on a barrier phase; false on abort or after 2 s (recorded, and
// the CTA's other roles are told through the abort flag).
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* abort_f,
                                           uint32_t* err) {
  // A few plain tries (waking up takes longer), then asleep: many polling warps
  // would take issue slots from the working ones.
  for (int i = 0; i < 2; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = now_ns();
  while (true) {
    if (mbar_try_wait_for(bar, parity, 200000u)) return true;
    if (*abort_f) return false;
    if (now_ns() - t0 > WAIT_NS) {
      *abort_f = 1;
      atomicOr(err, ERR_WAIT);
      return false;
    }
  }
}

// The same for a whole warp in step: all of its lanes go on or none.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_f,
                                          uint32_t* err) {
  return __all_sync(0xffffffffu, wait_phase(bar, parity, abort_f, err)) != 0;
}

// Wait on the error path for copies in flight: short limit, nothing recorded.
__device__ __forceinline__ void drain_phase(uint64_t* bar, uint32_t parity) {
  const long long t0 = now_ns();
  while (!mbar_try_wait(bar, parity))
    if (now_ns() - t0 > DRAIN_NS) return;
}

// Two fp32 values rounded to a pair of 16-bit elements, `lo` in the low half.
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t d;
  if (F16) {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  }
  return d;
}

template <bool F16>
__device__ __forceinline__ float element(uint16_t bits) {
  return F16 ? __half2float(__ushort_as_half(bits)) : bf16_bits_to_float(bits);
}

// Whether a 16-bit element is an infinity or not-a-number (exponent all ones).
template <bool F16>
__device__ __forceinline__ bool odd_element(uint16_t bits) {
  const uint16_t m = F16 ? 0x7c00 : 0x7f80;
  return (bits & m) == m;
}

// Whether any of eight elements is no number.  Adding one exponent step to the
// exponent bits carries into the sign bit's place only where they are all ones.
template <bool F16>
__device__ __forceinline__ bool has_odd(const uint4& v) {
  constexpr uint32_t M = F16 ? 0x7c007c00u : 0x7f807f80u, ONE = F16 ? 0x04000400u : 0x00800080u;
  const uint32_t t = ((v.x & M) + ONE) | ((v.y & M) + ONE) | ((v.z & M) + ONE) | ((v.w & M) + ONE);
  return (t & 0x80008000u) != 0;
}

// Zeroes the elements of eight that are no numbers.
template <bool F16>
__device__ __forceinline__ void clear_odd(uint4& v) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (odd_element<F16>((uint16_t)w[i])) w[i] &= 0xffff0000u;
    if (odd_element<F16>((uint16_t)(w[i] >> 16))) w[i] &= 0x0000ffffu;
  }
}

// D[16x8] += A[16x16] * B[16x8], fp32 accumulate.
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if (F16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    mma_bf16_16816(d, a[0], a[1], a[2], a[3], b0, b1);
  }
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z,
                                            int w, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%2, %3, %4, %5}], [%6], %7;"
      ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z),
        "r"(w), "r"(smem_addr(bar)), "l"(policy)
      : "memory");
}

// A value that all lanes have, or lane `from`'s, as one the compiler knows to be the
// same for the warp.
__device__ __forceinline__ int uniform(int x) { return __reduce_min_sync(0xffffffffu, x); }
__device__ __forceinline__ int uniform_of(int x, int from) {
  return __reduce_max_sync(0xffffffffu, (int)(threadIdx.x & 31) == from ? x : (int)0x80000000);
}

// The same for a whole warp in step, of which one lane (`one`) issues it: with no
// branch around it, and the operands made uniform for the compiler, they stay in
// the uniform registers that the instruction reads.
__device__ __forceinline__ void tma_load_4d_one(uint32_t one, void* dst, const CUtensorMap* map,
                                                int x, int y, int z, int w, uint64_t* bar,
                                                uint64_t policy) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %8, 0;\n"
      " @q cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%2, %3, %4, %5}], [%6], %7;\n}"
      ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z),
        "r"(w), "r"(smem_addr(bar)), "l"(policy), "r"(one)
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void fence_proxy_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src)
               : "memory");
}

// Arrives on `bar` once every cp.async of this thread so far has landed.
__device__ __forceinline__ void cp_async_arrive_noinc(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}

// Rows [first, end) of request b, cut to the rows there are.
__device__ __forceinline__ void request_rows(const int* cu, int b, int64_t total, int64_t& first,
                                             int64_t& end) {
  first = min(max((int64_t)cu[b], (int64_t)0), total);
  end = min(max((int64_t)cu[b + 1], first), total);
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------
int check_heads(int64_t Hq, int64_t Hkv, int64_t Dk, int64_t Dv, int dtype);

// Tensor map over 16-bit elements [dims[3]][dims[2]][dims[1]][dims[0]], element
// strides of the outer three, boxes of 64 x rows x box2 x 1 elements written in
// the 128-byte swizzle; what lies outside the tensor reads as zero.
int make_map_4d(CUtensorMap* map, const void* base, int f16, const int64_t (&dims)[4],
                const int64_t (&strides)[3], int rows, int box2);

// Dynamic shared-memory limit of a kernel, set once per device.
int allow_smem(const void* kernel, int bytes, bool (&done)[64], std::mutex& mu);

}  // namespace attn
}  // namespace kb
