// kb_attn.cu - causal attention over packed prompts and attention of drafted
// tokens over a paged cache.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / l_i,  s_ij = scale * q_i . k_j over the visible j,
//   m_i = max_j s_ij, l_i = sum_j exp(s_ij - m_i), lse_i = m_i + log(l_i)
// Prompts: j <= i + (Lk - Lq).  Paged: j < context, or tree bit j - context of
// the token's mask (without masks: j <= context + i).  A row that sees no key
// gives 0 and lse -infinity.
//
// One warp per (row, head); the lanes hold the head's dimensions, and keys are
// visited one at a time with a running maximum and sum.
#include <cuda_fp16.h>

#include "kb_common.cuh"

namespace kb {
namespace attn {

constexpr int THREADS = 256;
constexpr int MAX_DIM = 256;
constexpr int PER = MAX_DIM / 32;

struct Args {
  const uint16_t *q, *k, *v;
  int64_t q_tok, q_head, k_page, k_row, k_head, v_page, v_row, v_head;
  uint16_t* out;            // [total, Hq, Dv] contiguous
  float* lse;               // [total, Hq] or NULL
  const int *cu_q, *cu_k;   // cu_k: packed prompts
  const int* table;         // paged
  int64_t table_stride;
  const int* context;
  const int64_t* mask;
  int64_t n_pages;
  int64_t total_q, total_k;
  int B, width, ps, Hq, Hkv, Dk, Dv, f16, paged;
  float scale;
  uint32_t* err;
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
    int64_t keys, base = 0, ctx = 0;
    uint64_t word = ~0ull;
    if (A.paged) {
      ctx = max(0, A.context[b]);
      keys = A.mask ? ctx + n : ctx + i + 1;
      if (A.mask) word = (uint64_t)A.mask[row];
    } else {
      base = min(max((int64_t)A.cu_k[b], (int64_t)0), A.total_k);
      const int64_t lk = min(max((int64_t)A.cu_k[b + 1], base), A.total_k) - base;
      keys = i + 1 + lk - n;
      keys = keys < 0 ? 0 : keys;
    }
    float qv[PER];
    const uint16_t* q = A.q + row * A.q_tok + h * A.q_head;
#pragma unroll
    for (int c = 0; c < PER; ++c)
      qv[c] = lane + 32 * c < A.Dk ? value(q[lane + 32 * c], A.f16) * A.scale : 0.f;
    for (int64_t j = 0; j < keys; ++j) {
      if (A.paged && A.mask && j >= ctx && (j - ctx >= 64 || !((word >> (j - ctx)) & 1))) continue;
      int64_t page = 0, r = base + j;
      if (A.paged) {
        const int64_t col = j / A.ps;
        page = col < A.width ? A.table[(int64_t)b * A.table_stride + col] : -1;
        if (page < 0 || page >= A.n_pages) {
          if (lane == 0) atomicOr(A.err, ERR_PAGE);
          continue;
        }
        r = j - col * A.ps;
      }
      const uint16_t* k = A.k + page * A.k_page + r * A.k_row + hk * A.k_head;
      const uint16_t* v = A.v + page * A.v_page + r * A.v_row + hk * A.v_head;
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

static int check_heads(int64_t Hq, int64_t Hkv, int64_t Dk, int64_t Dv, int dtype) {
  KB_REQUIRE(Hq > 0 && Hkv > 0 && Hq % Hkv == 0, KB_ERR_BAD_SHAPE,
             "attention: query heads must be a multiple of key/value heads");
  KB_REQUIRE(Dk > 0 && Dk <= 192 && Dk % 8 == 0 && Dv > 0 && Dv <= 128 && Dv % 8 == 0,
             KB_ERR_UNSUPPORTED,
             "attention: head widths must be multiples of 8, keys up to 192 and values up to 128");
  KB_REQUIRE(dtype == 0 || dtype == 1, KB_ERR_UNSUPPORTED, "attention: unknown element type");
  return KB_OK;
}

static int launch_rows(Args& A, void* stream) {
  const int dev = bind_stream_device(stream);
  A.err = device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
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

extern "C" size_t kb_tree_attention_workspace_size(int64_t Hkv, int64_t group, int64_t max_tokens,
                                                   int64_t Dv) {
  (void)Hkv;
  (void)group;
  (void)max_tokens;
  (void)Dv;
  return 0;
}

extern "C" int kb_tree_attention(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride,
                                 const uint16_t* k_cache, const int64_t* k_strides,
                                 const uint16_t* v_cache, const int64_t* v_strides, int dtype,
                                 int64_t n_pages, int64_t page_size, const int32_t* block_table,
                                 int64_t table_stride, int64_t table_width,
                                 const int32_t* context_lens, const int32_t* cu_tokens,
                                 const int64_t* tree_mask, int64_t B, int64_t total,
                                 int64_t max_tokens, int64_t Hq, int64_t Hkv, int64_t Dk,
                                 int64_t Dv, float scale, uint16_t* out, float* lse,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  kb::clear_error();
  (void)workspace;
  (void)workspace_bytes;
  KB_REQUIRE(B >= 0 && total >= 0 && max_tokens >= 0 && n_pages >= 0 && table_width >= 0,
             KB_ERR_BAD_SHAPE, "tree attention: bad shape");
  const int st = kb::attn::check_heads(Hq, Hkv, Dk, Dv, dtype);
  if (st != KB_OK) return st;
  KB_REQUIRE(page_size >= 8 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
             KB_ERR_UNSUPPORTED, "tree attention: the page size must be a power of two from 8");
  if (B == 0 || total == 0) return KB_OK;
  KB_REQUIRE(q && k_strides && v_strides && cu_tokens && context_lens && out &&
                 (n_pages == 0 || (k_cache && v_cache)) && (table_width == 0 || block_table),
             KB_ERR_NULL_POINTER, "tree attention: NULL pointer");
  KB_REQUIRE(!tree_mask || max_tokens <= 64, KB_ERR_UNSUPPORTED,
             "tree attention: a masked tree has at most 64 tokens");
  kb::attn::Args A = {};
  A.paged = 1;
  A.q = q;
  A.k = k_cache;
  A.v = v_cache;
  A.q_tok = q_token_stride;
  A.q_head = q_head_stride;
  A.k_page = k_strides[0];
  A.k_row = k_strides[1];
  A.k_head = k_strides[2];
  A.v_page = v_strides[0];
  A.v_row = v_strides[1];
  A.v_head = v_strides[2];
  A.out = out;
  A.lse = lse;
  A.cu_q = cu_tokens;
  A.table = block_table;
  A.table_stride = table_stride;
  A.context = context_lens;
  A.mask = tree_mask;
  A.n_pages = n_pages;
  A.total_q = total;
  A.B = (int)B;
  A.width = (int)table_width;
  A.ps = (int)page_size;
  A.Hq = (int)Hq;
  A.Hkv = (int)Hkv;
  A.Dk = (int)Dk;
  A.Dv = (int)Dv;
  A.f16 = dtype;
  A.scale = scale;
  return kb::attn::launch_rows(A, stream);
}
