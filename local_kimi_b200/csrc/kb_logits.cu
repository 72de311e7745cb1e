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
// Bound: HBM, the logits read and written once; with long histories the latencies of a CTA's
// steps.  A CTA has a slice of the vocabulary and a few rows.  It asks for its part of a row (eight
// tokens a thread and piece, all of them under way; pieces that the mask empties are not read),
// counts the request's history in shared memory while they arrive, and writes the part, masked.
// Then it lists the tokens that the history, the drafts or the biases name (a bit a token says
// which) and adjusts those over what it has just written, dealt out evenly to its threads: few
// tokens change, and frequent ones lie together, so adjusting them where they lie in the pieces
// left most lanes of most warps idle.  Counts: a word a token, bit 0 the prompt, from bit 1 up how
// often (integers, so the order of the atomics does not show); 16 bits where no history can have
// 2^15 tokens, else 32.  Every slice reads the whole history again, from L2, by asynchronous
// copies to places that the copying thread alone reads: 2048 tokens on their way.
//
// Measured, 163840 tokens in bf16, replayed: 256 rows 60.5 us (176 MB less what masks leave out,
// 2.9 TB/s), with histories of 10 tokens 39, without any 31 (5.4 TB/s); one request of nine
// drafted rows 10.6.  Slices of 16384 tokens and 512 threads: 61.0 (histories of 8000 tokens 78
// instead of 92, none 35 instead of 31).
#include <algorithm>

#include "kb_common.cuh"

#include <cuda_fp16.h>

namespace kb {
namespace logits {

constexpr int THREADS = 256;
constexpr int RING = 2048;                  // tokens of the history on their way to a CTA
constexpr int MOST_BIASES = 4096;

struct Args {
  const uint8_t* x;
  uint8_t* y;
  int64_t x_row, y_row;                      // elements
  int64_t rows;
  int V, rows_each;
  const int64_t* history;                    // [B, ...]
  int64_t history_row;
  const int *lens, *prompts;                 // prompts may be NULL: all of it is answer
  int longest;                               // columns of history
  const float *repetition, *presence, *frequency;       // each may be NULL
  const int64_t* bias_ids;
  const float* bias_values;
  int64_t ids_row, values_row;
  int biases;
  const uint32_t* allowed;                   // [rows, words], of any stride: rows may share them
  int64_t allowed_row;
  const int* cu;                             // NULL: row b is request b's
  const int64_t* tokens;                     // drafted tokens, with cu
  const int64_t* mask;                       // NULL: chains
  int B;
  uint32_t* err;
};

// Eight bytes to shared memory on the way; waits for all but the last N groups of them.
__device__ __forceinline__ void cp_async8(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(to)),
               "l"(from)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mask_pairs(uint4& q, uint32_t bits, uint32_t none) {
  // Bytes of w, or of `none` where the bit is not set.
  auto pair = [&](uint32_t w, int at) {
    const uint32_t off = ~bits >> at;
    return prmt(w, none, 0x3210u + (off & 1) * 0x44u + (off & 2) * 0x2200u);
  };
  q = make_uint4(pair(q.x, 0), pair(q.y, 2), pair(q.z, 4), pair(q.w, 6));
}

template <int TYPE>                          // 0 bf16, 1 f16, 2 f32
struct Element;
template <>
struct Element<0> {
  using T = uint16_t;
  static __device__ __forceinline__ float load(T v) { return bf16_bits_to_float(v); }
  static __device__ __forceinline__ T store(float v) { return float_to_bf16_bits(v); }
  static constexpr T NONE = 0xff80u;         // -infinity
  // Elements of a 16-byte piece whose bit is not set: -infinity.
  static __device__ __forceinline__ void mask(uint4& q, uint32_t bits) {
    mask_pairs(q, bits, 0xff80ff80u);
  }
};
template <>
struct Element<1> {
  using T = uint16_t;
  static __device__ __forceinline__ float load(T v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ T store(float v) {
    return __half_as_ushort(__float2half_rn(v));
  }
  static constexpr T NONE = 0xfc00u;
  static __device__ __forceinline__ void mask(uint4& q, uint32_t bits) {
    mask_pairs(q, bits, 0xfc00fc00u);
  }
};
template <>
struct Element<2> {
  using T = uint32_t;
  static __device__ __forceinline__ float load(T v) { return __uint_as_float(v); }
  static __device__ __forceinline__ T store(float v) { return __float_as_uint(v); }
  static constexpr T NONE = 0xff800000u;
  static __device__ __forceinline__ void mask(uint4& q, uint32_t bits) {
    if (!(bits & 1)) q.x = NONE;
    if (!(bits & 2)) q.y = NONE;
    if (!(bits & 4)) q.z = NONE;
    if (!(bits & 8)) q.w = NONE;
  }
};

// Eight bits from bit t on of a row of `words` words; a byte where rows start at one.
__device__ __forceinline__ uint32_t eight(const uint32_t* row, int t, int words, bool bytes) {
  if (bytes) return reinterpret_cast<const uint8_t*>(row)[t >> 3];
  const int w = t >> 5, s = t & 31;
  const uint32_t lo = row[w], hi = s > 24 && w + 1 < words ? row[w + 1] : 0u;
  return __funnelshift_r(lo, hi, s) & 0xffu;
}

// Words of counts: bit 0: in the prompt, from bit 1 up: how often in the answer.
template <bool WIDE>
struct Counts {
  uint32_t* words;
  static constexpr int BYTES = WIDE ? 4 : 2;
  __device__ __forceinline__ uint32_t get(int at) const {
    return WIDE ? words[at] : reinterpret_cast<const uint16_t*>(words)[at];
  }
  __device__ __forceinline__ void add(int at, uint32_t v) const {
    if (WIDE)
      atomicAdd(words + at, v);
    else
      atomicAdd(words + (at >> 1), v << (16 * (at & 1)));
  }
  __device__ __forceinline__ void sub(int at, uint32_t v) const {
    if (WIDE)
      atomicSub(words + at, v);
    else
      atomicSub(words + (at >> 1), v << (16 * (at & 1)));
  }
  __device__ __forceinline__ void prompt(int at) const {
    if (WIDE)
      atomicOr(words + at, 1u);
    else
      atomicOr(words + (at >> 1), 1u << (16 * (at & 1)));
  }
};

struct Request {
  float repetition, presence, frequency;
  int biases;                                // of the slice
};

template <int TYPE, bool WIDE, int PIECES>   // pieces of eight tokens a thread
__global__ void __launch_bounds__(THREADS, PIECES == 1 ? 5 : TYPE == 2 ? 3 : 4)
    adjust_kernel(const Args A) {
  using E = Element<TYPE>;
  using T = typename E::T;
  constexpr int VECS = sizeof(T) / 2;        // 16-byte loads of a piece
  constexpr int SLICE = THREADS * 8 * PIECES;
  extern __shared__ __align__(16) uint32_t smem[];
  uint32_t* flag = smem;                                  // [SLICE / 32] something to do
  uint32_t* biased = flag + SLICE / 32;                   // [SLICE / 32]
  const Counts<WIDE> count = {biased + SLICE / 32};       // [SLICE]
  // Tokens of the history on their way, [RING / THREADS][THREADS]; then a list of tokens, [SLICE].
  constexpr int PART = RING / THREADS / 2;
  int64_t* ring = reinterpret_cast<int64_t*>(smem + SLICE / 16 + SLICE * Counts<WIDE>::BYTES / 4);
  uint16_t* list = reinterpret_cast<uint16_t*>(ring);
  int* bias_at = reinterpret_cast<int*>(ring + RING);
  float* bias = reinterpret_cast<float*>(bias_at + A.biases);
  __shared__ int s_biases, s_found[2], s_warp[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int v0 = blockIdx.x * SLICE, v1 = min(A.V, v0 + SLICE);
  const int words = (A.V + 31) / 32;
  const bool same = A.x == A.y;              // in place: what does not change stays
  if (tid < 2) s_found[tid] = 0;
  pdl_wait();
  pdl_launch_dependents();

  int current = -1;                          // the request whose counts these are
  Request R = {1.f, 0.f, 0.f, 0};
  bool counts = false;
  const int64_t last = min(A.rows, ((int64_t)blockIdx.y + 1) * A.rows_each);
  for (int64_t r = (int64_t)blockIdx.y * A.rows_each; r < last; ++r) {
    // The row's request: the last that starts at or before it.  -1: outside all.
    int b = (int)min(r, (int64_t)A.B);
    int64_t first = r;
    if (A.cu != nullptr) {
      b = -1;
      for (int i0 = 0; i0 <= A.B; i0 += THREADS)
        b += __syncthreads_count(i0 + tid <= A.B && (int64_t)__ldg(A.cu + i0 + tid) <= r);
      if (b >= 0) first = max((int64_t)A.cu[b], (int64_t)0);
    }
    if (b >= A.B) b = -1;

    // The row's part: 16-byte pieces where input and output lie alike, single tokens at the ends.
    const T* x = reinterpret_cast<const T*>(A.x) + r * A.x_row;
    T* y = reinterpret_cast<T*>(A.y) + r * A.y_row;
    const uint32_t* allowed = A.allowed && b >= 0 ? A.allowed + r * A.allowed_row : nullptr;
    const uint32_t lead = (uint32_t)(reinterpret_cast<uintptr_t>(x + v0) & 15);
    const bool alike = lead == (uint32_t)(reinterpret_cast<uintptr_t>(y + v0) & 15);
    int a = min(v1, v0 + (int)(((16u - lead) & 15u) / sizeof(T)));
    int z = a + (v1 - a) / 8 * 8;
    if (!alike) a = z = v1;
    const bool bytes = (a & 7) == 0;
    // What a new request needs, and the row's mask: one wait for all of them.
    const bool fresh = b != current;
    const bool told = fresh && b >= 0 && A.history != nullptr;
    int n = 0, p = 0;
    if (fresh) {
      R = {1.f, 0.f, 0.f, 0};
      if (b >= 0) {
        if (A.repetition) R.repetition = A.repetition[b];
        if (A.presence) R.presence = A.presence[b];
        if (A.frequency) R.frequency = A.frequency[b];
      }
      if (told) {
        n = A.lens[b];
        p = A.prompts ? A.prompts[b] : 0;
      }
    }
    uint32_t open = ~0u;                     // the mask of the thread's word of flags
    if (allowed && tid < SLICE / 32 && v0 / 32 + tid < words) open = __ldg(allowed + v0 / 32 + tid);
    uint32_t in[PIECES];
    uint4 v[PIECES][VECS];
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int t = a + (tid + u * THREADS) * 8;
      in[u] = t < z ? allowed ? eight(allowed, t, words, bytes) : 0xffu : 0u;
    }
    if (fresh) {
      __syncthreads();
      for (int i = tid; i < (SLICE / 16 + SLICE * Counts<WIDE>::BYTES / 4) / 4; i += THREADS)
        reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
      if (tid == 0) s_biases = 0;
    }
    // (In place a part that nothing changes is not read; that is not known yet.)
    if (!same)
#pragma unroll
      for (int u = 0; u < PIECES; ++u)
        if (in[u])
#pragma unroll
          for (int k = 0; k < VECS; ++k)
            v[u][k] = ldg_stream_v4(reinterpret_cast<const uint4*>(
                                        x + a + (tid + u * THREADS) * 8) + k);

    if (fresh) {
      // The counts of the request's history.
      current = b;
      counts = R.repetition != 1.f || R.presence != 0.f || R.frequency != 0.f;
      __syncthreads();
      if (counts && told) {
        n = min(max(n, 0), A.longest);
        p = min(max(p, 0), n);
        const uint64_t width = (uint64_t)(v1 - v0);
        const bool end = v1 == A.V;          // tells of tokens behind the vocabulary
        auto seen = [&](int64_t t, int i) {
          const uint64_t off = (uint64_t)(t - v0);
          if (off < width) {
            const int at = (int)off;
            if (i < p)
              count.prompt(at);
            else
              count.add(at, 2u);
            atomicOr(&flag[at >> 5], 1u << (at & 31));
          } else if (end && t >= v1) {
            atomicOr(A.err, ERR_TREE);
          }
        };
        const int64_t* history = A.history + (int64_t)b * A.history_row;
        auto ask = [&](int k) {
#pragma unroll
          for (int u = 0; u < PART; ++u) {
            const int i = (k * PART + u) * THREADS + tid;
            if (i < n) cp_async8(&ring[((k & 1) * PART + u) * THREADS + tid], history + i);
          }
          cp_async_commit();
        };
        ask(0);
        ask(1);
#pragma unroll 1
        for (int k = 0; k * PART * THREADS < n; ++k) {
          cp_async_wait<1>();
#pragma unroll
          for (int u = 0; u < PART; ++u) {
            const int i = (k * PART + u) * THREADS + tid;
            if (i < n) seen(ring[((k & 1) * PART + u) * THREADS + tid], i);
          }
          ask(k + 2);
        }
        cp_async_wait<0>();
      }
      if (A.biases && b >= 0) {
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
            atomicOr(&biased[(t - v0) >> 5], 1u << ((t - v0) & 31));
            atomicOr(&flag[(t - v0) >> 5], 1u << ((t - v0) & 31));
          }
          __syncthreads();
          if (tid == 0) s_biases += all;
          __syncthreads();
        }
        R.biases = s_biases;
      }
      __syncthreads();
    }
    // The drafted tokens above the row's prediction.
    const bool draft = counts && A.tokens != nullptr && b >= 0;
    auto drafted = [&](bool on) {
      const uint64_t word = A.mask ? (uint64_t)A.mask[r] : 0;
      const int64_t end = min(A.rows, (int64_t)A.cu[b + 1]);
      for (int64_t i = tid; i <= (A.mask ? (int64_t)63 : r - first); i += THREADS) {
        if (first + i >= end || (A.mask && !((word >> i) & 1))) continue;
        const int64_t t = A.tokens[first + i];
        if (t >= A.V) atomicOr(A.err, ERR_TREE);
        if (t < v0 || t >= v1) continue;
        const int at = (int)(t - v0);
        if (on) {
          count.add(at, 2u);
          atomicOr(&flag[at >> 5], 1u << (at & 31));
        } else {
          count.sub(at, 2u);                 // (its flag may stay: it only means looking)
        }
      }
    };
    if (draft) {
      drafted(true);
      __syncthreads();
    }
    auto adjust = [&](float f, int t) {
      const int at = t - v0;
      const uint32_t word = count.get(at), c = word >> 1;
      if (word) f = f > 0.f ? f / R.repetition : f * R.repetition;
      if (c) {
        f = __fsub_rn(f, __fmul_rn(R.frequency, (float)c));
        f = __fsub_rn(f, R.presence);
      }
      if ((biased[at >> 5] >> (at & 31)) & 1) {
        float sum = 0.f;
        for (int i = 0; i < R.biases; ++i)
          if (bias_at[i] == t) sum += bias[i];
        f += sum;
      }
      return f;
    };
#pragma unroll 1
    for (int k = tid; k < (a - v0) + (v1 - z); k += THREADS) {
      const int t = k < a - v0 ? v0 + k : z + k - (a - v0);
      if (allowed && !((__ldg(allowed + (t >> 5)) >> (t & 31)) & 1))
        y[t] = E::NONE;
      else if (!same)
        y[t] = x[t];
    }
    if (tid == 0) s_found[(r + 1) & 1] = 0;  // (between two rows that count is a barrier)
    // The pieces: copied, or masked.
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int t = a + (tid + u * THREADS) * 8;
      if (t >= z || (same && in[u] == 0xffu)) continue;
#pragma unroll
      for (int k = 0; k < VECS; ++k) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (in[u]) q = same ? *(reinterpret_cast<const uint4*>(x + t) + k) : v[u][k];
        if (in[u] != 0xffu) E::mask(q, in[u] >> (8 / VECS * k));
        *(reinterpret_cast<uint4*>(y + t) + k) = q;
      }
    }
    if (!counts && !R.biases) continue;
    // The tokens that change, listed in any order and dealt out to all threads, over what has
    // just been written.
    static_assert(SLICE / 32 <= THREADS, "a word of flags a thread");
    uint32_t bits = tid < SLICE / 32 ? flag[tid] & open : 0u;
    int found = __popc(bits), at = -found;
    for (int o = 1; o < 32; o <<= 1) {
      const int before = __shfl_up_sync(0xffffffffu, found, o);
      if (lane >= o) found += before;
    }
    at += found;
    const int start = lane == 31 ? atomicAdd(&s_found[r & 1], found) : 0;
    at += __shfl_sync(0xffffffffu, start, 31);
    for (; bits != 0; bits &= bits - 1) list[at++] = (uint16_t)(tid * 32 + __ffs(bits) - 1);
    __syncthreads();
    found = s_found[r & 1];
    constexpr int AT_ONCE = 4;
#pragma unroll 1
    for (int i0 = tid; i0 < found; i0 += THREADS * AT_ONCE) {
      T f[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
        if (i0 + THREADS * u < found) f[u] = x[v0 + list[i0 + THREADS * u]];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
        if (i0 + THREADS * u < found) {
          const int t = v0 + list[i0 + THREADS * u];
          y[t] = E::store(adjust(E::load(f[u]), t));
        }
    }
    if (draft && r + 1 < last) {
      __syncthreads();
      drafted(false);
      __syncthreads();
    }
  }
}

template <int TYPE, bool WIDE, int PIECES>
static int launch_slices(Args A, int sms, void* stream) {
  constexpr int SLICE = THREADS * 8 * PIECES;
  constexpr size_t FIXED = (size_t)SLICE / 4 + (size_t)SLICE * Counts<WIDE>::BYTES + RING * 8;
  static_assert(SLICE * 2 <= RING * 8, "the list in the ring's place");
  const size_t smem = FIXED + (size_t)A.biases * 8;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(adjust_kernel<TYPE, WIDE, PIECES>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(FIXED + MOST_BIASES * 8));
    KB_REQUIRE(e == cudaSuccess, KB_ERR_DEVICE, "adjust logits: shared-memory limit: %s",
               cudaGetErrorString(e));
  }
  const int64_t slices = (A.V + SLICE - 1) / SLICE;
  // Several rows of drafts a CTA, whose requests' histories are counted once, where that
  // leaves eight CTAs an SM.  (128 requests of nine rows: 297 us, 343 with a row a CTA; 32
  // requests: 82 and 92.)
  A.rows_each = 1;
  if (A.cu != nullptr)
    A.rows_each = (int)std::min<int64_t>(64, std::max<int64_t>(1, slices * A.rows / (8 * sms)));
  const int64_t y = (A.rows + A.rows_each - 1) / A.rows_each;
  KB_REQUIRE(y <= 65535, KB_ERR_UNSUPPORTED, "adjust logits: more than 65535 rows");
  return launch(adjust_kernel<TYPE, WIDE, PIECES>, dim3((unsigned)slices, (unsigned)y),
                dim3(THREADS), smem, stream, A);
}

template <int TYPE, bool WIDE>
static int launch_wide(const Args& A, int sms, void* stream) {
  // Slices of 8192 tokens, or, where those are fewer than the SMs, of 2048.  With 20 wide slices
  // a row and histories of 3500 tokens: 1 row 7.5 us wide, 6.2 narrow; 4 rows 7.6 and 7.0; 8 rows
  // 7.9 and 10.3; 32 rows 14.5 and 26.2.
  if ((A.V + 8191) / 8192 * A.rows >= sms) return launch_slices<TYPE, WIDE, 4>(A, sms, stream);
  return launch_slices<TYPE, WIDE, 1>(A, sms, stream);
}

template <int TYPE>
static int launch_adjust(const Args& A, int sms, void* stream) {
  // 15 bits count a history of fewer tokens, drafted ones included.
  const int64_t most = (A.history ? A.longest : 0) + (A.mask ? 64 : A.tokens ? A.rows : 0);
  return most < 32768 ? launch_wide<TYPE, false>(A, sms, stream)
                      : launch_wide<TYPE, true>(A, sms, stream);
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
                 out_stride >= V && (!allowed || allowed_stride >= 0),
             KB_ERR_BAD_SHAPE, "adjust logits: bad shape");
  KB_REQUIRE(dtype >= 0 && dtype <= 2, KB_ERR_UNSUPPORTED, "adjust logits: unknown element type");
  KB_REQUIRE(V < ((int64_t)1 << 30) && B < 65535 && longest < ((int64_t)1 << 30) &&
                 rows < ((int64_t)1 << 30),
             KB_ERR_UNSUPPORTED, "adjust logits: more than 65534 requests or 2^30 tokens");
  KB_REQUIRE(n_biases <= lg::MOST_BIASES, KB_ERR_UNSUPPORTED,
             "adjust logits: more than %d biases a request", lg::MOST_BIASES);
  if (rows == 0) return KB_OK;
  KB_REQUIRE(logits && out && (!history || history_lens || B == 0) &&
                 (!bias_ids || bias_values) && (!tokens || cu_tokens) && (!tree_mask || tokens) &&
                 (cu_tokens || B <= rows),
             KB_ERR_NULL_POINTER, "adjust logits: NULL pointer");
  KB_REQUIRE(logits != out || rows == 1 || row_stride == out_stride, KB_ERR_BAD_SHAPE,
             "adjust logits: in place, the rows have one stride");
  const size_t size = dtype == 2 ? 4 : 2;
  KB_REQUIRE((((uintptr_t)logits | (uintptr_t)out) & (size - 1)) == 0 &&
                 (((uintptr_t)history | (uintptr_t)bias_ids | (uintptr_t)tokens |
                   (uintptr_t)tree_mask) & 7) == 0 &&
                 (((uintptr_t)history_lens | (uintptr_t)prompt_lens | (uintptr_t)repetition |
                   (uintptr_t)presence | (uintptr_t)frequency | (uintptr_t)bias_values |
                   (uintptr_t)allowed | (uintptr_t)cu_tokens) & 3) == 0,
             KB_ERR_ALIGNMENT, "adjust logits: unaligned pointer");
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
  const int sms = kb::num_sms(dev);
  if (dtype == 0) return lg::launch_adjust<0>(A, sms, stream);
  if (dtype == 1) return lg::launch_adjust<1>(A, sms, stream);
  return lg::launch_adjust<2>(A, sms, stream);
}
