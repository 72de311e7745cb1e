// kb_logits.cu - logits as a request wants them: penalties for tokens that its history holds,
// biases, and the mask of a grammar.
//
// For a row of request b and a token t, with c = how often t is in the request's answer (its
// history behind the prompt, and for a row of drafted tokens the tokens from the root to it),
// all in fp32, one after the other, and rounded once to the logits' type:
//   x = x > 0 ? x / repetition_b : x * repetition_b      if t is in the prompt or c > 0
//   x = x - frequency_b * c;  x = x - presence_b         if c > 0
//   x = x + the request's biases of t, summed in their order
//   x = -infinity                                        if the row's mask does not have t
//
// Bound: HBM, the logits read and written once.  A CTA takes a slice of the vocabulary and a
// request, counts the history's tokens of its slice in shared memory (a 32-bit word a token:
// bit 0 the prompt, from bit 1 up the count; integers, so the order of the atomics does not
// show) and then streams its part of each of the request's rows, eight tokens a thread and
// step.  A bit a token says whether there is anything to do: eight bits, read beside eight
// bits of the mask, let most pieces pass with a copy, and pieces that the mask empties are
// written without being read.  The history is read again by every slice, from L2.
#include "kb_common.cuh"

#include <cuda_fp16.h>

namespace kb {
namespace logits {

constexpr int THREADS = 256;
constexpr int MOST_BIASES = 4096;

struct Args {
  const uint8_t* x;
  uint8_t* y;
  int64_t x_row, y_row;                      // elements
  int64_t rows;
  int V, slice;
  const int64_t* history;                    // [B, ...]
  int64_t history_row;
  const int *lens, *prompts;                 // prompts may be NULL: all of it is answer
  int longest;                               // columns of history
  const float *repetition, *presence, *frequency;       // each may be NULL
  const int64_t* bias_ids;
  const float* bias_values;
  int64_t ids_row, values_row;
  int biases;
  const uint32_t* allowed;                   // [rows, words]
  int64_t allowed_row;
  const int* cu;                             // NULL: row b is request b's
  const int64_t* tokens;                     // drafted tokens, with cu
  const int64_t* mask;                       // NULL: chains
  int B;
  uint32_t* err;
};

template <int TYPE>                          // 0 bf16, 1 f16, 2 f32
struct Element;
template <>
struct Element<0> {
  using T = uint16_t;
  static __device__ __forceinline__ float load(T v) { return bf16_bits_to_float(v); }
  static __device__ __forceinline__ T store(float v) { return float_to_bf16_bits(v); }
  static constexpr T NONE = 0xff80u;         // -infinity
};
template <>
struct Element<1> {
  using T = uint16_t;
  static __device__ __forceinline__ float load(T v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ T store(float v) {
    return __half_as_ushort(__float2half_rn(v));
  }
  static constexpr T NONE = 0xfc00u;
};
template <>
struct Element<2> {
  using T = uint32_t;
  static __device__ __forceinline__ float load(T v) { return __uint_as_float(v); }
  static __device__ __forceinline__ T store(float v) { return __float_as_uint(v); }
  static constexpr T NONE = 0xff800000u;
};

// Eight bits from bit t on of a row of `words` words.
__device__ __forceinline__ uint32_t eight(const uint32_t* row, int t, int words) {
  const int w = t >> 5, s = t & 31;
  const uint32_t lo = row[w], hi = s > 24 && w + 1 < words ? row[w + 1] : 0u;
  return __funnelshift_r(lo, hi, s) & 0xffu;
}

struct Slice {
  const uint32_t* count;                     // words of the slice's tokens
  const uint32_t* flag;                      // bits: something to do
  const int* bias_at;                        // biases of the slice in their order
  const float* bias;
  int biases;
  float repetition, presence, frequency;
};
constexpr uint32_t BIASED = 0x80000000u;

__device__ __forceinline__ float adjust(float x, uint32_t word, int t, const Slice& S) {
  const uint32_t c = (word & ~BIASED) >> 1;
  if (word & ~BIASED) x = x > 0.f ? x / S.repetition : x * S.repetition;
  if (c) {
    x = __fsub_rn(x, __fmul_rn(S.frequency, (float)c));
    x = __fsub_rn(x, S.presence);
  }
  if (word & BIASED) {
    float sum = 0.f;
    for (int i = 0; i < S.biases; ++i)
      if (S.bias_at[i] == t) sum += S.bias[i];
    x += sum;
  }
  return x;
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS) adjust_kernel(const Args A) {
  using E = Element<TYPE>;
  using T = typename E::T;
  constexpr int VECS = sizeof(T) / 2;        // 16-byte pieces of eight tokens
  extern __shared__ uint32_t smem[];
  uint32_t* count = smem;                                 // [slice]
  uint32_t* flag = count + A.slice;                       // [slice / 32]
  int* bias_at = reinterpret_cast<int*>(flag + A.slice / 32);   // [biases]
  float* bias = reinterpret_cast<float*>(bias_at + A.biases);
  __shared__ int s_biases, s_warp[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.y, v0 = blockIdx.x * A.slice, v1 = min(A.V, v0 + A.slice);
  for (int i = tid; i < A.slice + A.slice / 32; i += THREADS) smem[i] = 0;
  if (tid == 0) s_biases = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  // The request's rows; the last block of rows takes those outside every request.
  int64_t r0 = b, r1 = b + 1, skip0 = 0, skip1 = 0;
  const bool spare = b == A.B;
  if (A.cu != nullptr) {
    const int64_t lo = min(max((int64_t)A.cu[spare ? 0 : b], (int64_t)0), A.rows);
    const int64_t hi = min(max((int64_t)A.cu[spare ? A.B : b + 1], lo), A.rows);
    r0 = spare ? 0 : lo;
    r1 = spare ? A.rows : hi;
    if (spare) {
      skip0 = lo;
      skip1 = hi;
    }
  } else if (spare) {
    r0 = A.B;
    r1 = A.rows;
  }
  if (r0 >= r1) return;
  Slice S = {count, flag, bias_at, bias, 0, 1.f, 0.f, 0.f};
  if (!spare) {
    if (A.repetition) S.repetition = A.repetition[b];
    if (A.presence) S.presence = A.presence[b];
    if (A.frequency) S.frequency = A.frequency[b];
  }
  const bool counts = S.repetition != 1.f || S.presence != 0.f || S.frequency != 0.f;
  if (counts && A.history != nullptr) {
    const int64_t* h = A.history + (int64_t)b * A.history_row;
    const int n = min(max(A.lens[b], 0), A.longest);
    const int p = A.prompts ? min(max(A.prompts[b], 0), n) : 0;
#pragma unroll 4
    for (int i = tid; i < n; i += THREADS) {
      const int64_t t = __ldg(h + i);
      if (t >= A.V) atomicOr(A.err, ERR_TREE);
      if (t < v0 || t >= v1) continue;
      const int at = (int)(t - v0);
      if (i < p)
        atomicOr(&count[at], 1u);
      else
        atomicAdd(&count[at], 2u);
      atomicOr(&flag[at >> 5], 1u << (at & 31));
    }
  }
  if (A.bias_ids != nullptr && !spare) {
    // The slice's biases, kept in their order.
    for (int i0 = 0; i0 < A.biases; i0 += THREADS) {
      const int i = i0 + tid;
      const int64_t t = i < A.biases ? __ldg(A.bias_ids + (int64_t)b * A.ids_row + i) : -1;
      if (t >= A.V) atomicOr(A.err, ERR_TREE);
      const bool here = t >= v0 && t < v1;
      const unsigned votes = __ballot_sync(0xffffffffu, here);
      if (lane == 0) s_warp[warp] = __popc(votes);
      __syncthreads();
      int at = s_biases + __popc(votes & ((1u << lane) - 1u)), all = 0;
      for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) at += s_warp[w];
        all += s_warp[w];
      }
      if (here) {
        bias_at[at] = (int)t;
        bias[at] = __ldg(A.bias_values + (int64_t)b * A.values_row + i);
        atomicOr(&count[t - v0], BIASED);
        atomicOr(&flag[(t - v0) >> 5], 1u << ((t - v0) & 31));
      }
      __syncthreads();
      if (tid == 0) s_biases += all;
      __syncthreads();
    }
    S.biases = s_biases;
  }
  __syncthreads();

  const bool same = A.x == A.y;              // in place: what does not change stays
  for (int64_t r = r0; r < r1; ++r) {
    if (r >= skip0 && r < skip1) continue;
    // The drafted tokens above the row's prediction.
    auto drafted = [&](bool on) {
      const int64_t j = r - r0;
      const uint64_t word = A.mask ? (uint64_t)A.mask[r] : 0;
      for (int64_t i = tid; i <= (A.mask ? (int64_t)63 : j); i += THREADS) {
        if (r0 + i >= r1 || (A.mask && !((word >> i) & 1))) continue;
        const int64_t t = A.tokens[r0 + i];
        if (t >= A.V) atomicOr(A.err, ERR_TREE);
        if (t < v0 || t >= v1) continue;
        const int at = (int)(t - v0);
        if (on) {
          atomicAdd(&count[at], 2u);
          atomicOr(&flag[at >> 5], 1u << (at & 31));
        } else {
          atomicSub(&count[at], 2u);         // (its flag may stay: it only means looking)
        }
      }
    };
    const bool draft = counts && A.tokens != nullptr && !spare;
    if (draft) {
      drafted(true);
      __syncthreads();
    }
    const T* x = reinterpret_cast<const T*>(A.x) + r * A.x_row;
    T* y = reinterpret_cast<T*>(A.y) + r * A.y_row;
    const uint32_t* allowed = A.allowed && !spare ? A.allowed + r * A.allowed_row : nullptr;
    const int words = (A.V + 31) / 32;
    // 16-byte pieces where input and output lie alike, single tokens at the ends.
    const uint32_t lead = (uint32_t)(reinterpret_cast<uintptr_t>(x + v0) & 15);
    const bool alike = lead == (uint32_t)(reinterpret_cast<uintptr_t>(y + v0) & 15);
    int a = min(v1, v0 + (int)(((16u - lead) & 15u) / sizeof(T)));
    int z = a + (v1 - a) / 8 * 8;
    if (!alike) a = z = v1;
    for (int k = tid; k < (a - v0) + (v1 - z); k += THREADS) {
      const int t = k < a - v0 ? v0 + k : z + k - (a - v0);
      const bool out = allowed && !((__ldg(allowed + (t >> 5)) >> (t & 31)) & 1);
      const uint32_t word = count[t - v0];
      if (out)
        y[t] = E::NONE;
      else if (word)
        y[t] = E::store(adjust(E::load(x[t]), word, t, S));
      else if (!same)
        y[t] = x[t];
    }
    constexpr int UNDERWAY = 4 / VECS;
    for (int t0 = a + tid * 8; t0 < z; t0 += THREADS * 8 * UNDERWAY) {
      uint32_t todo[UNDERWAY], in[UNDERWAY];
      uint4 v[UNDERWAY][VECS];
#pragma unroll
      for (int u = 0; u < UNDERWAY; ++u) {
        const int t = t0 + u * THREADS * 8;
        in[u] = 0xffu;
        if (allowed && t < z) in[u] = eight(allowed, t, words);
      }
#pragma unroll
      for (int u = 0; u < UNDERWAY; ++u) {
        const int t = t0 + u * THREADS * 8;
        todo[u] = t < z ? eight(flag, t - v0, A.slice / 32) & in[u] : 0;
        if (t < z && in[u] != 0 && !(same && todo[u] == 0 && in[u] == 0xffu))
#pragma unroll
          for (int k = 0; k < VECS; ++k)
            v[u][k] = *(reinterpret_cast<const uint4*>(x + t) + k);
      }
#pragma unroll
      for (int u = 0; u < UNDERWAY; ++u) {
        const int t = t0 + u * THREADS * 8;
        if (t >= z || (same && todo[u] == 0 && in[u] == 0xffu)) continue;
        union {
          uint4 q[VECS];
          T e[8];
        } w;
#pragma unroll
        for (int k = 0; k < VECS; ++k) w.q[k] = in[u] ? v[u][k] : make_uint4(0, 0, 0, 0);
        if (in[u] != 0xffu)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!((in[u] >> i) & 1)) w.e[i] = E::NONE;
        if (todo[u])
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if ((todo[u] >> i) & 1) {
              const uint32_t word = count[t + i - v0];
              if (word) w.e[i] = E::store(adjust(E::load(w.e[i]), word, t + i, S));
            }
#pragma unroll
        for (int k = 0; k < VECS; ++k) *(reinterpret_cast<uint4*>(y + t) + k) = w.q[k];
      }
    }
    if (draft) {
      __syncthreads();
      drafted(false);
      __syncthreads();
    }
  }
}

template <int TYPE>
static int launch_adjust(const Args& A, dim3 grid, size_t smem, void* stream) {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        adjust_kernel<TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
    KB_REQUIRE(e == cudaSuccess, KB_ERR_DEVICE, "adjust logits: shared-memory limit: %s",
               cudaGetErrorString(e));
  }
  return launch(adjust_kernel<TYPE>, grid, dim3(THREADS), smem, stream, A);
}

}  // namespace logits
}  // namespace kb

extern "C" int kb_adjust_logits(const void* logits, int64_t row_stride, int64_t rows, int64_t V,
                                int dtype, void* out, int64_t out_stride, int64_t B,
                                const int64_t* history, int64_t history_stride, int64_t longest,
                                const int32_t* history_lens, const int32_t* prompt_lens,
                                const float* repetition, const float* presence,
                                const float* frequency, const int64_t* bias_ids,
                                int64_t ids_stride, const float* bias_values,
                                int64_t values_stride, int64_t n_biases, const int32_t* allowed,
                                int64_t allowed_stride, const int32_t* cu_tokens,
                                const int64_t* tokens, const int64_t* tree_mask, void* stream) {
  namespace lg = kb::logits;
  kb::clear_error();
  KB_REQUIRE(rows >= 0 && V > 0 && B >= 0 && longest >= 0 && n_biases >= 0 && row_stride >= V &&
                 out_stride >= V && (!allowed || allowed_stride >= (V + 31) / 32),
             KB_ERR_BAD_SHAPE, "adjust logits: bad shape");
  KB_REQUIRE(dtype >= 0 && dtype <= 2, KB_ERR_UNSUPPORTED, "adjust logits: unknown element type");
  KB_REQUIRE(V < ((int64_t)1 << 30) && B < 65535 && longest < ((int64_t)1 << 30),
             KB_ERR_UNSUPPORTED, "adjust logits: more than 65534 requests or 2^30 tokens");
  KB_REQUIRE(n_biases <= lg::MOST_BIASES, KB_ERR_UNSUPPORTED,
             "adjust logits: more than %d biases a request", lg::MOST_BIASES);
  if (rows == 0) return KB_OK;
  KB_REQUIRE(logits && out && (!history || history_lens || B == 0) &&
                 (!bias_ids || bias_values) && (!tokens || cu_tokens) && (!tree_mask || tokens) &&
                 (cu_tokens || B <= rows),
             KB_ERR_NULL_POINTER, "adjust logits: NULL pointer");
  const size_t size = dtype == 2 ? 4 : 2;
  KB_REQUIRE((((uintptr_t)logits | (uintptr_t)out) & (size - 1)) == 0, KB_ERR_ALIGNMENT,
             "adjust logits: unaligned pointer");
  const int dev = kb::bind_stream_device(stream);
  lg::Args A = {};
  A.x = static_cast<const uint8_t*>(logits);
  A.y = static_cast<uint8_t*>(out);
  A.x_row = row_stride;
  A.y_row = out_stride;
  A.rows = rows;
  A.V = (int)V;
  A.history = longest > 0 ? history : nullptr;
  A.history_row = history_stride;
  A.lens = history_lens;
  A.prompts = prompt_lens;
  A.longest = (int)longest;
  A.repetition = repetition;
  A.presence = presence;
  A.frequency = frequency;
  A.bias_ids = n_biases > 0 ? bias_ids : nullptr;
  A.bias_values = bias_values;
  A.ids_row = ids_stride;
  A.values_row = values_stride;
  A.biases = A.bias_ids ? (int)n_biases : 0;
  A.allowed = reinterpret_cast<const uint32_t*>(allowed);
  A.allowed_row = allowed_stride;
  A.cu = cu_tokens;
  A.tokens = tokens;
  A.mask = tree_mask;
  A.B = (int)B;
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  // Slices as wide as leaves four CTAs an SM: each reads the whole history.
  const int64_t want = (int64_t)kb::num_sms(dev) * 4;
  int slice = 1024;
  while (slice < 16384 && (V + slice - 1) / slice * (B > 0 ? B : 1) > want) slice *= 2;
  A.slice = slice;
  const size_t smem = (size_t)slice * 4 + slice / 8 + (size_t)A.biases * 8;
  const dim3 grid((unsigned)((V + slice - 1) / slice), (unsigned)(B + 1));
  if (dtype == 0) return lg::launch_adjust<0>(A, grid, smem, stream);
  if (dtype == 1) return lg::launch_adjust<1>(A, grid, smem, stream);
  return lg::launch_adjust<2>(A, grid, smem, stream);
}
