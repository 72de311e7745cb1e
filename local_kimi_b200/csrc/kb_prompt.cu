// kb_prompt.cu - causal attention over packed prompts.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / l_i,  s_ij = scale * q_i . k_j over the visible j,
//   m_i = max_j s_ij, l_i = sum_j exp(s_ij - m_i), lse_i = m_i + log(l_i)
// visible: j <= i + (Lk - Lq).  A row that sees no key gives 0 and lse -infinity.
//
// One warp per (row, head); the lanes hold the head's dimensions, and keys are
// visited one at a time with a running maximum and sum.
#include "kb_attn.cuh"

namespace kb {
namespace attn {

constexpr int THREADS = 256;
constexpr int MAX_DIM = 256;
constexpr int PER = MAX_DIM / 32;

struct Args {
  const uint16_t *q, *k, *v;
  int64_t q_tok, q_head, k_row, k_head, v_row, v_head;
  uint16_t* out;            // [total, Hq, Dv] contiguous
  float* lse;               // [total, Hq] or NULL
  const int *cu_q, *cu_k;
  int64_t total_q, total_k;
  int B, Hq, Hkv, Dk, Dv, f16;
  float scale;
};

__device__ __forceinline__ float value(uint16_t bits, int f16) {
  return f16 ? __half2float(__ushort_as_half(bits)) : bf16_bits_to_float(bits);
}

__global__ void __launch_bounds__(THREADS) rows_kernel(const Args A) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  if (item >= A.total_q * A.Hq) return;
  const int64_t row = item / A.Hq;
  const int h = (int)(item - row * A.Hq), hk = h / (A.Hq / A.Hkv);
  int lo = 0, hi = A.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (A.cu_q[mid] <= row) lo = mid; else hi = mid - 1;
  }
  const int b = lo;
  const int64_t first = A.cu_q[b], end = min((int64_t)A.cu_q[b + 1], A.total_q);
  float acc[PER] = {};
  float m = -INFINITY, l = 0.f;
  if (row >= first && row < end) {
    const int i = (int)(row - first), n = (int)(end - first);
    const int64_t base = min(max((int64_t)A.cu_k[b], (int64_t)0), A.total_k);
    const int64_t lk = min(max((int64_t)A.cu_k[b + 1], base), A.total_k) - base;
    const int64_t keys = i + 1 + lk - n;
    float qv[PER];
    const uint16_t* q = A.q + row * A.q_tok + h * A.q_head;
#pragma unroll
    for (int c = 0; c < PER; ++c)
      qv[c] = lane + 32 * c < A.Dk ? value(q[lane + 32 * c], A.f16) * A.scale : 0.f;
    for (int64_t j = 0; j < keys; ++j) {
      const uint16_t* k = A.k + (base + j) * A.k_row + hk * A.k_head;
      const uint16_t* v = A.v + (base + j) * A.v_row + hk * A.v_head;
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < PER; ++c)
        if (lane + 32 * c < A.Dk) s += qv[c] * value(k[lane + 32 * c], A.f16);
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (s == -INFINITY) continue;
      const float top = fmaxf(m, s);
      const float fix = expf(m - top), w = expf(s - top);
      m = top;
      l = l * fix + w;
#pragma unroll
      for (int c = 0; c < PER; ++c)
        if (lane + 32 * c < A.Dv) acc[c] = acc[c] * fix + w * value(v[lane + 32 * c], A.f16);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const int d = lane + 32 * c;
    if (d >= A.Dv) continue;
    const float o = l == 0.f ? 0.f : acc[c] * inv;
    A.out[item * A.Dv + d] = A.f16 ? __half_as_ushort(__float2half_rn(o)) : float_to_bf16_bits(o);
  }
  if (A.lse && lane == 0) A.lse[item] = l == 0.f ? -INFINITY : m + logf(l);
}

static int launch_rows(Args& A, void* stream) {
  const int64_t items = A.total_q * A.Hq;
  const int64_t grid = (items + THREADS / 32 - 1) / (THREADS / 32);
  KB_REQUIRE(grid < ((int64_t)1 << 31), KB_ERR_UNSUPPORTED, "attention: too many rows");
  return launch(rows_kernel, dim3((unsigned)grid), dim3(THREADS), 0, stream, A);
}

}  // namespace attn
}  // namespace kb

extern "C" int kb_prompt_attention(const uint16_t* q, int64_t q_token_stride,
                                   int64_t q_head_stride, const uint16_t* k,
                                   int64_t k_token_stride, int64_t k_head_stride,
                                   const uint16_t* v, int64_t v_token_stride,
                                   int64_t v_head_stride, int dtype, const int32_t* cu_q,
                                   const int32_t* cu_k, int64_t B, int64_t total_q,
                                   int64_t total_k, int64_t max_q, int64_t Hq, int64_t Hkv,
                                   int64_t Dk, int64_t Dv, float scale, uint16_t* out, float* lse,
                                   void* stream) {
  kb::clear_error();
  KB_REQUIRE(B >= 0 && total_q >= 0 && total_k >= 0 && max_q >= 0, KB_ERR_BAD_SHAPE,
             "prompt attention: bad shape");
  const int st = kb::attn::check_heads(Hq, Hkv, Dk, Dv, dtype);
  if (st != KB_OK) return st;
  if (B == 0 || total_q == 0) return KB_OK;
  KB_REQUIRE(q && cu_q && cu_k && out && (total_k == 0 || (k && v)), KB_ERR_NULL_POINTER,
             "prompt attention: NULL pointer");
  KB_REQUIRE(B < ((int64_t)1 << 30) && total_q < ((int64_t)1 << 31) && total_k < ((int64_t)1 << 31),
             KB_ERR_UNSUPPORTED, "prompt attention: too many tokens");
  kb::attn::Args A = {};
  A.q = q;
  A.k = k;
  A.v = v;
  A.q_tok = q_token_stride;
  A.q_head = q_head_stride;
  A.k_row = k_token_stride;
  A.k_head = k_head_stride;
  A.v_row = v_token_stride;
  A.v_head = v_head_stride;
  A.out = out;
  A.lse = lse;
  A.cu_q = cu_q;
  A.cu_k = cu_k;
  A.total_q = total_q;
  A.total_k = total_k;
  A.B = (int)B;
  A.Hq = (int)Hq;
  A.Hkv = (int)Hkv;
  A.Dk = (int)Dk;
  A.Dv = (int)Dv;
  A.f16 = dtype;
  A.scale = scale;
  return kb::attn::launch_rows(A, stream);
}
