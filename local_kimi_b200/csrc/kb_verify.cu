// kb_verify.cu - verification of drafted tokens against the target's logits.
//
// A request has n tree tokens (token 0 the root, already decided); row t of
// its logits is the target's prediction after token t.  With p = softmax(row
// / temperature) the walk starts at the root and tries the children of the
// current node in index order:
//   no draft probabilities: child x is taken if u * rem < p(x), rem starting
//     at 1; a refused child leaves the distribution: rem -= p(x), p(x) = 0;
//   draft probabilities q (chains): taken if u * q(x) < p(x); a refused child
//     leaves p = max(p - q, 0).
// At the last node the next token is argmax_i p_i / e_i (lowest index on
// ties), e the given exponential noise: token i wins with probability
// p_i / sum(p), and no sum over the vocabulary enters the choice.  If nothing
// is left of p by rounding, the row's own p is used.  Temperature 0 takes
// the child that is the row's argmax (lowest index) and ends with the argmax.
//
// Two launches.  row_kernel reads every logit once, 16 bytes a load, with a
// running maximum and sum of exponentials per thread (or the argmax) of each
// row segment, fp32.  pick_kernel joins the segments, walks the tree from
// shared memory, and scans the last node's row with the noise (and q): its
// CTAs split the vocabulary, each joins its best (value, index) key with a
// 64-bit atomicMax, and the request's last CTA writes the token.  What the second launch
// takes from the first is in the call's own workspace, so calls from several threads
// may meet on a stream in any order.  Bound by the
// bytes: the logits once, and of one row a request logits, noise and q again.
// Measured: 256 requests of up to 5 tokens, 163840 wide, with q: 122 us, 54 for the
// rows (4.7 TB/s; special function unit 63 % busy) and 70 for the picks (4.3
// TB/s; 41 % of the warps there, which wait for loads: 8.5 of them stalled for each
// that issues); one request of 9 tokens: 18.4 us with a cold cache, 12.5 replayed at once.
//
// Rows start anywhere (an odd vocabulary): the loads begin at the row's first
// 16-byte boundary, what lies before and after goes one by one.  The fast
// loops assume finite sums; a segment whose sum is not finite or zero is
// read again with not-a-number as absent and infinity as the largest number.
#include <cuda_fp16.h>

#include <float.h>

#include "kb_math.cuh"

namespace kb {
namespace verify {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 64;
constexpr int MAX_SEGMENTS = 32;

enum Type : int { BF16 = 0, F16 = 1, F32 = 2 };

struct Stat {
  float top;      // max logit (greedy: the largest logit)
  float sum;      // sum of exp((x - top) / T)
  int arg;        // greedy: its index
  int pad;
};

struct Race {               // of a request's CTAs for its next token
  unsigned long long best;
  int arrived;
  int pad;
};

struct Args {
  const void* logits;
  int64_t row_stride;
  int64_t skew;             // elements from `logits`, moved down to a 16-byte boundary, to row 0
  int64_t rows;
  int V;
  const int64_t* tokens;
  const int* parents;       // NULL: a chain
  const int* cu;
  int B, most;              // most: tree tokens of a request at most
  const float* coin;
  const float* noise;
  int64_t noise_stride;
  const float* temps;
  const float* probs;       // NULL: drafted tokens without probabilities
  int64_t probs_stride;
  int64_t* out;             // [B, most]
  int* path;                // [B, most]
  int* accepted;            // [B]
  Stat* stats;              // [rows][segments]
  Race* race;               // [B], zeroed by row_kernel
  int segments;             // of a row in row_kernel
  int parts;                // CTAs of a request in pick_kernel
  uint32_t* err;
};

template <int TYPE>
__device__ __forceinline__ float logit(const void* base, int64_t i) {
  if (TYPE == F32) return __ldg(static_cast<const float*>(base) + i);
  const uint16_t bits = __ldg(static_cast<const uint16_t*>(base) + i);
  return TYPE == BF16 ? bf16_bits_to_float(bits) : __half2float(__ushort_as_half(bits));
}

// Not-a-number counts as absent, +infinity as the largest finite value.
__device__ __forceinline__ float tidy(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }

__device__ __forceinline__ float weight(float x, float top, float inv_t) {
  return top == -INFINITY ? 0.f : expf((x - top) * inv_t);
}

// 1 / T, kept where its products stay numbers: a T next to zero leaves the largest logits
// alone, one without bound gives every finite logit the same weight.
__device__ __forceinline__ float inverse(float t) {
  return t > 0.f ? fminf(fmaxf(1.0f / t, FLT_MIN), FLT_MAX / 2) : 1.0f;
}

// Tokens [first, first + n) of request b, cut to the rows there are.
__device__ __forceinline__ void request(const Args& A, int b, int64_t& first, int& n) {
  const int64_t s = min(max((int64_t)A.cu[b], (int64_t)0), A.rows);
  const int64_t e = min(max((int64_t)A.cu[b + 1], s), A.rows);
  first = s;
  n = (int)min(e - s, (int64_t)A.most);
}

constexpr float LOWEST = -1e30f;       // start of a running maximum

// Elements of a 16-byte load.
template <int TYPE>
constexpr int PIECE = TYPE == F32 ? 4 : 8;

template <int TYPE>
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[PIECE<TYPE>]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (TYPE == F32) {
      x[i] = __uint_as_float(w[i]);
    } else if (TYPE == BF16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// The 16-byte pieces within elements [lo, hi) of a row that starts at element
// `base` of a 16-byte aligned array: first element of the first whole piece
// (relative to the row) and their number.
template <int TYPE>
__device__ __forceinline__ void whole_pieces(int64_t base, int lo, int hi, int& first,
                                             int& count) {
  constexpr int P = PIECE<TYPE>;
  const int skew = (int)((base + lo) & (P - 1));
  first = min(hi, skew ? lo + P - skew : lo);
  count = (hi - first) / P;
}

template <int TYPE>
__device__ __forceinline__ uint4 piece(const void* p, int64_t element) {
  return ldg_stream_v4(static_cast<const uint8_t*>(p) + element * (TYPE == F32 ? 4 : 2));
}

// Running (maximum, sum) of a thread over its share of [lo, hi).
template <int TYPE>
__device__ __forceinline__ void sum_segment(const Args& A, int64_t base, int lo, int hi, float c2,
                                            float& top, float& sum) {
  constexpr int P = PIECE<TYPE>, BATCH = 4;
  int first, count;
  whole_pieces<TYPE>(base, lo, hi, first, count);
  const int tid = threadIdx.x;
  top = LOWEST;
  sum = 0.f;
  auto take = [&](float x) {
    if (x > top) {
      sum *= exp2_fast((top - x) * c2);
      top = x;
    }
    sum += exp2_fast((x - top) * c2);
  };
  for (int i = tid; i < count; i += THREADS * BATCH) {
    float x[BATCH * P];
    uint4 v[BATCH];
    const bool all = i + (BATCH - 1) * THREADS < count;
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      v[u] = piece<TYPE>(A.logits, base + first + (int64_t)min(i + u * THREADS, count - 1) * P);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      unpack<TYPE>(v[u], *reinterpret_cast<float(*)[P]>(&x[u * P]));
      if (!all && i + u * THREADS >= count)
#pragma unroll
        for (int j = 0; j < P; ++j) x[u * P + j] = -INFINITY;
    }
    float m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int j = 4; j < BATCH * P; j += 4) {
      m[(j >> 1) & 2] = max3(m[(j >> 1) & 2], x[j], x[j + 1]);
      m[((j >> 1) & 2) + 1] = max3(m[((j >> 1) & 2) + 1], x[j + 2], x[j + 3]);
    }
    const float most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    if (most > top) {
      sum *= exp2_fast((top - most) * c2);
      top = most;
    }
    // (x - top) first: the difference is exact where it matters, x * c2 is not.
    const float2 off = make_float2(-top, -top), mul = make_float2(c2, c2);
    float2 part[2] = {};
#pragma unroll
    for (int j = 0; j < BATCH * P; j += 2) {
      float2 y = fmul2(fadd2(make_float2(x[j], x[j + 1]), off), mul);
      y.x = exp2_fast(y.x);
      y.y = exp2_fast(y.y);
      part[(j >> 1) & 1] = fadd2(part[(j >> 1) & 1], y);
    }
    part[0] = fadd2(part[0], part[1]);
    sum += part[0].x + part[0].y;
  }
  // Before the first whole piece and after the last.
  for (int i = lo + tid; i < first; i += THREADS) take(logit<TYPE>(A.logits, base + i));
  for (int i = first + count * P + tid; i < hi; i += THREADS)
    take(logit<TYPE>(A.logits, base + i));
}

// Largest logit of a thread's share and its index (lowest among equals).
template <int TYPE>
__device__ __forceinline__ void best_segment(const Args& A, int64_t base, int lo, int hi,
                                             float& top, int& arg) {
  constexpr int P = PIECE<TYPE>;
  int first, count;
  whole_pieces<TYPE>(base, lo, hi, first, count);
  const int tid = threadIdx.x;
  top = -INFINITY;
  arg = INT_MAX;
  auto take = [&](float x, int i) {
    if (x > top || arg == INT_MAX) {
      top = fmaxf(x, -INFINITY);       // not-a-number: absent
      arg = i;
    }
  };
  for (int i = lo + tid; i < first; i += THREADS) take(logit<TYPE>(A.logits, base + i), i);
#pragma unroll 4
  for (int i = tid; i < count; i += THREADS) {
    float x[P];
    const int at = first + i * P;
    unpack<TYPE>(piece<TYPE>(A.logits, base + at), x);
#pragma unroll
    for (int j = 0; j < P; ++j) take(x[j], at + j);
  }
  for (int i = first + count * P + tid; i < hi; i += THREADS)
    take(logit<TYPE>(A.logits, base + i), i);
}

__device__ __forceinline__ float block_max(float v, float* red) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < THREADS / 32; ++w) v = fmaxf(v, red[w]);
  __syncthreads();
  return v;
}

__device__ __forceinline__ float block_sum(float v, float* red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < THREADS / 32; ++w) v += red[w];
  __syncthreads();
  return v;
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS) row_kernel(const Args A) {
  __shared__ float red[THREADS / 32];
  __shared__ float s_top[THREADS / 32];
  __shared__ int s_arg[THREADS / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x / A.segments, seg = blockIdx.x - t * A.segments;
  if (blockIdx.x == 0 && threadIdx.x == 0) A.race[blockIdx.y] = Race{0, 0, 0};
  int64_t first;
  int n;
  request(A, blockIdx.y, first, n);
  if (t >= n) return;
  const int64_t row = first + t;
  const float temp = A.temps[blockIdx.y];
  const int lo = (int)((int64_t)A.V * seg / A.segments);
  const int hi = (int)((int64_t)A.V * (seg + 1) / A.segments);
  const int64_t base = row * A.row_stride + A.skew;
  float top, sum = 0.f;
  int arg = 0;
  if (temp > 0.f) {
    const float inv_t = inverse(temp), c2 = inv_t * LOG2E;
    float mine, part;
    sum_segment<TYPE>(A, base, lo, hi, c2, mine, part);
    top = block_max(mine, red);
    sum = block_sum(part * exp2_fast((mine - top) * c2), red);
    if (!(sum > 0.f && sum < INFINITY)) {
      // Something that is no number, or nothing above the start of the maximum.
      float m = -INFINITY;
      for (int i = lo + threadIdx.x; i < hi; i += THREADS)
        m = fmaxf(m, tidy(logit<TYPE>(A.logits, base + i)));
      top = block_max(m, red);
      float p = 0.f;
      for (int i = lo + threadIdx.x; i < hi; i += THREADS)
        p += weight(tidy(logit<TYPE>(A.logits, base + i)), top, inv_t);
      sum = block_sum(p, red);
    }
  } else {
    best_segment<TYPE>(A, base, lo, hi, top, arg);
    for (int o = 16; o > 0; o >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, top, o);
      const int j = __shfl_xor_sync(0xffffffffu, arg, o);
      if (y > top || (y == top && j < arg)) {
        top = y;
        arg = j;
      }
    }
    if ((threadIdx.x & 31) == 0) {
      s_top[threadIdx.x >> 5] = top;
      s_arg[threadIdx.x >> 5] = arg;
    }
    __syncthreads();
    top = s_top[0];
    arg = s_arg[0];
    for (int w = 1; w < THREADS / 32; ++w)
      if (s_top[w] > top || (s_top[w] == top && s_arg[w] < arg)) {
        top = s_top[w];
        arg = s_arg[w];
      }
  }
  if (threadIdx.x == 0) A.stats[row * A.segments + seg] = Stat{top, sum, arg, 0};
}

// A key of the race: the value, then the lowest index.
__device__ __forceinline__ unsigned long long race_key(float v, int i) {
  return ((unsigned long long)__float_as_uint(v) << 32) |
         (unsigned long long)(0xffffffffu - (uint32_t)i);
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS, 4) pick_kernel(const Args A) {
  __shared__ float s_top[MAX_TOKENS], s_sum[MAX_TOKENS], s_px[MAX_TOKENS], s_qx[MAX_TOKENS];
  __shared__ float s_coin[MAX_TOKENS];
  __shared__ int s_arg[MAX_TOKENS], s_par[MAX_TOKENS], s_lost[MAX_TOKENS], s_path[MAX_TOKENS];
  __shared__ int64_t s_tok[MAX_TOKENS];
  __shared__ int s_cur, s_count, s_nlost, s_refused;
  __shared__ unsigned long long s_best[THREADS / 32], s_won;
  __shared__ bool s_last;
  const int b = blockIdx.y, part = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();
  int64_t first;
  int n;
  request(A, b, first, n);
  int64_t* out = A.out + (int64_t)b * A.most;
  int* path = A.path + (int64_t)b * A.most;
  if (n == 0) {
    if (part == 0) {
      for (int i = tid; i < A.most; i += THREADS) {
        out[i] = -1;
        path[i] = -1;
      }
      if (tid == 0) A.accepted[b] = 0;
    }
    return;
  }
  const float temp = A.temps[b];
  const float inv_t = inverse(temp);
  const bool greedy = !(temp > 0.f);
  // A warp joins the segments of a row, a lane each.
  static_assert(MAX_SEGMENTS <= 32, "a lane for each segment");
  for (int t = warp; t < n; t += THREADS / 32) {
    Stat st = {-INFINITY, 0.f, INT_MAX, 0};
    if (lane < A.segments) st = A.stats[(first + t) * A.segments + lane];
    float top = st.top;
    int arg = st.arg;
    for (int o = 16; o > 0; o >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, top, o);
      const int j = __shfl_xor_sync(0xffffffffu, arg, o);
      if (y > top || (y == top && j < arg)) {
        top = y;
        arg = j;
      }
    }
    float sum = st.sum * weight(st.top, top, inv_t);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      s_top[t] = top;
      s_sum[t] = sum;
      s_arg[t] = arg;
    }
  }
  for (int t = tid; t < n; t += THREADS) {
    int up = t == 0 ? -1 : (A.parents ? A.parents[first + t] : t - 1);
    const int64_t x = A.tokens[first + t];
    if (t > 0 && (up < 0 || up >= t || x < 0 || x >= A.V)) {
      atomicOr(A.err, ERR_TREE);   // a bad parent or token: the drafted token is never taken
      up = -2;
    }
    s_par[t] = up;
    s_tok[t] = x;
    s_coin[t] = A.coin[first + t];
    s_qx[t] = A.probs && up >= 0 ? A.probs[(first + t) * A.probs_stride + x] : 1.f;
  }
  __syncthreads();
  for (int t = tid; t < n; t += THREADS) {
    const int up = s_par[t];
    float p = 0.f;
    if (up >= 0 && !greedy)
      p = weight(tidy(logit<TYPE>(A.logits, (first + up) * A.row_stride + A.skew +
                                                    s_tok[t])), s_top[up],
                 inv_t) / s_sum[up];
    s_px[t] = p;
  }
  __syncthreads();
  if (tid == 0) {
    int cur = 0, count = 0, nlost = 0, refused = -1;
    float rem = 1.f;
    s_path[0] = 0;
    for (int i = 1; i < n; ++i) {
      if (s_par[i] != cur) continue;
      bool take;
      float p = s_px[i];
      if (greedy) {
        take = s_tok[i] == s_arg[cur];
      } else {
        for (int j = 0; j < nlost; ++j)
          if (s_lost[j] == (int)s_tok[i]) p = 0.f;
        take = s_coin[i] * (A.probs ? s_qx[i] : rem) < p;
      }
      if (take) {
        cur = i;
        s_path[++count] = i;
        nlost = 0;
        refused = -1;
        rem = 1.f;
      } else {
        s_lost[nlost++] = (int)s_tok[i];
        refused = i;
        rem = fmaxf(rem - p, 0.f);
      }
    }
    s_cur = cur;
    s_count = count;
    s_nlost = nlost;
    s_refused = refused;
  }
  __syncthreads();
  const int cur = s_cur, taken = s_count, nlost = s_nlost;
  if (part == 0) {
    for (int i = tid; i < A.most; i += THREADS) {
      path[i] = i <= taken ? s_path[i] : -1;
      if (i != taken) out[i] = i < taken ? s_tok[s_path[i + 1]] : -1;
    }
    if (tid == 0) {
      A.accepted[b] = taken;
      if (greedy) out[taken] = s_arg[cur];
    }
  }
  if (greedy) return;
  const float* q = A.probs && s_refused >= 0 ? A.probs + (first + s_refused) * A.probs_stride
                                             : nullptr;
  const float* noise = A.noise + (int64_t)b * A.noise_stride;
  const int64_t base = (first + cur) * A.row_stride + A.skew;
  const float top = s_top[cur], c2 = inv_t * LOG2E;
  const float share = q ? 1.0f / s_sum[cur] : 1.0f;
  const int lo = (int)((int64_t)A.V * part / A.parts);
  const int hi = (int)((int64_t)A.V * (part + 1) / A.parts);
  float best = 0.f;
  int arg = -1;
  // Strictly larger wins, so equal values go to the lower index.  Without draft
  // probabilities the sum of the weights does not matter; the refused tokens are
  // looked up for a new best only.
  auto take = [&](float x, float e, float qi, int i) {
    // Not-a-number loses every comparison, as does a row of nothing but -infinity.
    const float v = __fdividef(exp2_fast((x - top) * c2) * share - qi, e);
    if (v > best) {
      bool lost = false;
      if (!A.probs)
        for (int j = 0; j < nlost; ++j) lost = lost || s_lost[j] == i;
      if (!lost) {
        best = v;
        arg = i;
      }
    }
  };
  constexpr int P = PIECE<TYPE>;
  int start, count;
  whole_pieces<TYPE>(base, lo, hi, start, count);
  // A row with an infinite logit goes one by one, with infinity as the largest number.
  if (top == FLT_MAX) {
    start = hi;
    count = 0;
  }
  for (int i = lo + tid; i < start; i += THREADS)
    take(tidy(logit<TYPE>(A.logits, base + i)), noise[i], q ? q[i] : 0.f, i);
  const bool wide =
      ((uintptr_t)(noise + start) & 15) == 0 && (!q || ((uintptr_t)(q + start) & 15) == 0);
  constexpr int BATCH = 2;
  for (int i0 = tid; i0 < count; i0 += THREADS * BATCH) {
    uint4 v[BATCH];
    float e[BATCH][P], qv[BATCH][P];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = min(i0 + u * THREADS, count - 1);
      const int at = start + i * P;
      v[u] = piece<TYPE>(A.logits, base + at);
#pragma unroll
      for (int j = 0; j < P; j += 4) {
        if (wide) {
          *reinterpret_cast<uint4*>(&e[u][j]) = ldg_stream_v4(noise + at + j);
          if (q) *reinterpret_cast<uint4*>(&qv[u][j]) = ldg_stream_v4(q + at + j);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            e[u][j + k] = noise[at + j + k];
            if (q) qv[u][j + k] = q[at + j + k];
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = i0 + u * THREADS;
      if (i >= count) break;
      float x[P];
      unpack<TYPE>(v[u], x);
#pragma unroll
      for (int j = 0; j < P; ++j) take(x[j], e[u][j], q ? qv[u][j] : 0.f, start + i * P + j);
    }
  }
  for (int i = start + count * P + tid; i < hi; i += THREADS)
    take(logit<TYPE>(A.logits, base + i), noise[i], q ? q[i] : 0.f, i);
  unsigned long long key = arg < 0 ? 0 : race_key(best, arg);
  auto join = [&]() {
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      if (other > key) key = other;
    }
    if (lane == 0) s_best[warp] = key;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w)
      if (s_best[w] > key) key = s_best[w];
  };
  join();
  if (tid == 0) {
    atomicMax(&A.race[b].best, key);
    __threadfence();
    s_last = atomicAdd(&A.race[b].arrived, 1) == A.parts - 1;
    if (s_last) s_won = atomicMax(&A.race[b].best, 0ull);
  }
  __syncthreads();
  if (!s_last) return;
  key = s_won;
  if (key == 0) {
    // Nothing is left by rounding: the row's own p, from the first token on.
    float v = -1.f;
    int at = INT_MAX;
    for (int i = tid; i < A.V; i += THREADS) {
      const float w = weight(tidy(logit<TYPE>(A.logits, base + i)), top, inv_t) / noise[i];
      if (w > v) {
        v = w;
        at = i;
      }
    }
    key = at == INT_MAX ? 0 : race_key(v, at);
    join();
    if (key == 0) key = race_key(0.f, 0);      // noise that compares with nothing: token 0
  }
  if (tid == 0) out[taken] = (int64_t)(0xffffffffu - (uint32_t)key);
}

// Segments of a row: enough CTAs (48 an SM, of at least 4096 elements) that the
// last ones to run do not leave most SMs idle.  CTAs of a request in the second
// kernel: about the four an SM that run at once, since each walks the tree first
// (ten a request instead of two: 126 instead of 70 us for 256 requests), of at
// least 2048 elements: for one request 163840 wide, 80 CTAs take both kernels to
// 18.4 us, 32 CTAs 24.6, 40 CTAs 20.5, 160 CTAs 18.7 to 20.4; 16 requests and more
// are the same with each.
static void split(int64_t B, int64_t most, int64_t V, int sms, int* segments, int* parts) {
  auto pick = [&](int64_t units, int64_t per_sm, int64_t least, int64_t limit) {
    int64_t s = per_sm * sms / units;
    const int64_t by_size = (V + least - 1) / least;
    if (s > by_size) s = by_size;
    if (s > limit) s = limit;
    return (int)(s < 1 ? 1 : s);
  };
  *segments = pick(B * most, 48, 4096, MAX_SEGMENTS);
  *parts = pick(B, 4, 2048, 65535);
}

static size_t power_of_two(int64_t n) {
  size_t p = 16;
  while ((int64_t)p < n) p *= 2;
  return p;
}

static size_t race_bytes(int64_t B) { return power_of_two(B) * sizeof(Race); }

}  // namespace verify
}  // namespace kb

extern "C" size_t kb_verify_drafts_workspace_size(int64_t B, int64_t rows) {
  if (B <= 0 || rows < 0) return 0;
  return kb::verify::race_bytes(B) +
         kb::verify::power_of_two(rows) * kb::verify::MAX_SEGMENTS * sizeof(kb::verify::Stat);
}

extern "C" int kb_verify_drafts(const void* logits, int64_t row_stride, int64_t rows, int64_t V,
                                int dtype, const int64_t* tokens, const int32_t* parents,
                                const int32_t* cu_tokens, int64_t B, int64_t max_tokens,
                                const float* accept_u, const float* noise, int64_t noise_stride,
                                const float* temperature, const float* draft_probs,
                                int64_t probs_stride, int64_t* out_tokens, int32_t* path,
                                int32_t* accepted, void* workspace, size_t workspace_bytes,
                                void* stream) {
  namespace v = kb::verify;
  kb::clear_error();
  KB_REQUIRE(B >= 0 && rows >= 0 && V > 0 && max_tokens > 0, KB_ERR_BAD_SHAPE,
             "verify: bad shape");
  if (B == 0) return KB_OK;
  KB_REQUIRE(dtype >= 0 && dtype <= 2, KB_ERR_UNSUPPORTED, "verify: unknown logits type");
  KB_REQUIRE(max_tokens <= v::MAX_TOKENS && B <= 65535 && V < ((int64_t)1 << 30),
             KB_ERR_UNSUPPORTED, "verify: at most %d tokens a request and 65535 requests",
             v::MAX_TOKENS);
  KB_REQUIRE(row_stride >= V && noise_stride >= V && (!draft_probs || probs_stride >= V),
             KB_ERR_BAD_SHAPE, "verify: row strides too small");
  KB_REQUIRE(!(parents && draft_probs), KB_ERR_UNSUPPORTED,
             "verify: draft probabilities go with chains, not trees");
  KB_REQUIRE((rows == 0 || (logits && tokens)) && cu_tokens && accept_u && noise && temperature &&
                 out_tokens && path && accepted && workspace,
             KB_ERR_NULL_POINTER, "verify: NULL pointer");
  const size_t need = kb_verify_drafts_workspace_size(B, rows);
  KB_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, KB_ERR_WORKSPACE,
             "verify: workspace of %zu bytes (256-byte aligned) required, %zu given",
             need, workspace_bytes);
  const int dev = kb::bind_stream_device(stream);
  v::Args A = {};
  const int size = dtype == v::F32 ? 4 : 2;
  KB_REQUIRE(rows == 0 || (uintptr_t)logits % size == 0, KB_ERR_ALIGNMENT,
             "verify: logits must be aligned to their elements");
  A.skew = (int64_t)((uintptr_t)logits & 15) / size;
  A.logits = static_cast<const uint8_t*>(logits) - A.skew * size;
  A.row_stride = row_stride;
  A.rows = rows;
  A.V = (int)V;
  A.tokens = tokens;
  A.parents = parents;
  A.cu = cu_tokens;
  A.B = (int)B;
  A.most = (int)max_tokens;
  A.coin = accept_u;
  A.noise = noise;
  A.noise_stride = noise_stride;
  A.temps = temperature;
  A.probs = draft_probs;
  A.probs_stride = probs_stride;
  A.out = out_tokens;
  A.path = path;
  A.accepted = accepted;
  A.race = static_cast<v::Race*>(workspace);
  A.stats = reinterpret_cast<v::Stat*>(static_cast<uint8_t*>(workspace) + v::race_bytes(B));
  v::split(B, max_tokens, V, kb::num_sms(dev), &A.segments, &A.parts);
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  const dim3 g1((unsigned)(max_tokens * A.segments), (unsigned)B);
  const dim3 g2((unsigned)A.parts, (unsigned)B);
  auto run = [&](auto rowk, auto pickk) {
    int st = kb::launch(rowk, g1, dim3(v::THREADS), 0, stream, A);
    return st != KB_OK ? st : kb::launch(pickk, g2, dim3(v::THREADS), 0, stream, A);
  };
  if (dtype == v::BF16) return run(v::row_kernel<v::BF16>, v::pick_kernel<v::BF16>);
  if (dtype == v::F16) return run(v::row_kernel<v::F16>, v::pick_kernel<v::F16>);
  return run(v::row_kernel<v::F32>, v::pick_kernel<v::F32>);
}
