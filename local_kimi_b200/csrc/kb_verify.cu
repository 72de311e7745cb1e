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
// Two launches.  row_kernel reads every logit once: (max, sum of exp) or the
// argmax of each row segment, fp32.  pick_kernel joins the segments, walks
// the tree from shared memory, and scans the last node's row with the noise
// (and q): its CTAs split the vocabulary, each joins its best (value, index)
// key with a 64-bit atomicMax, and the request's last CTA writes the token.
// Bound by the bytes of the logits.
#include <cuda_fp16.h>

#include <float.h>

#include "kb_common.cuh"

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
  Race* race;               // [B], zero between calls
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

__device__ __forceinline__ float inverse(float t) { return t > 0.f ? 1.0f / t : 1.0f; }

// Tokens [first, first + n) of request b, cut to the rows there are.
__device__ __forceinline__ void request(const Args& A, int b, int64_t& first, int& n) {
  const int64_t s = min(max((int64_t)A.cu[b], (int64_t)0), A.rows);
  const int64_t e = min(max((int64_t)A.cu[b + 1], s), A.rows);
  first = s;
  n = (int)min(e - s, (int64_t)A.most);
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS) row_kernel(const Args A) {
  __shared__ float s_a[THREADS / 32], s_b[THREADS / 32];
  __shared__ int s_i[THREADS / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x / A.segments, seg = blockIdx.x - t * A.segments;
  int64_t first;
  int n;
  request(A, blockIdx.y, first, n);
  if (t >= n) return;
  const int64_t row = first + t;
  const float temp = A.temps[blockIdx.y];
  const float inv_t = inverse(temp);
  const int lo = (int)((int64_t)A.V * seg / A.segments);
  const int hi = (int)((int64_t)A.V * (seg + 1) / A.segments);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t base = row * A.row_stride;
  float top = -INFINITY;
  int arg = INT_MAX;
  for (int i = lo + tid; i < hi; i += THREADS) {
    const float x = tidy(logit<TYPE>(A.logits, base + i));
    if (x > top || arg == INT_MAX) {
      top = x;
      arg = i;
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float y = __shfl_xor_sync(0xffffffffu, top, o);
    const int j = __shfl_xor_sync(0xffffffffu, arg, o);
    if (y > top || (y == top && j < arg)) {
      top = y;
      arg = j;
    }
  }
  if (lane == 0) {
    s_a[warp] = top;
    s_i[warp] = arg;
  }
  __syncthreads();
  top = s_a[0];
  arg = s_i[0];
  for (int w = 1; w < THREADS / 32; ++w)
    if (s_a[w] > top || (s_a[w] == top && s_i[w] < arg)) {
      top = s_a[w];
      arg = s_i[w];
    }
  float sum = 0.f;
  if (temp > 0.f)
    for (int i = lo + tid; i < hi; i += THREADS)
      sum += weight(tidy(logit<TYPE>(A.logits, base + i)), top, inv_t);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_b[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    float s = 0.f;
    for (int w = 0; w < THREADS / 32; ++w) s += s_b[w];
    A.stats[row * A.segments + seg] = Stat{top, s, arg, 0};
  }
}

// Joins two keys of the race: (class, value, lowest index).  Class 1: a
// weight is left; class 0: nothing is left and the row's own p stands in.
__device__ __forceinline__ unsigned long long race_key(float left, float p, float e, int i) {
  const bool some = left > 0.f;
  const float v = (some ? left : p) / e;
  const uint32_t bits = __float_as_uint(fmaxf(v, 0.f));
  return ((unsigned long long)some << 63) | ((unsigned long long)bits << 32) |
         (unsigned long long)(0xffffffffu - (uint32_t)i);
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS) pick_kernel(const Args A) {
  __shared__ float s_top[MAX_TOKENS], s_sum[MAX_TOKENS], s_px[MAX_TOKENS], s_qx[MAX_TOKENS];
  __shared__ float s_coin[MAX_TOKENS];
  __shared__ int s_arg[MAX_TOKENS], s_par[MAX_TOKENS], s_lost[MAX_TOKENS], s_path[MAX_TOKENS];
  __shared__ int64_t s_tok[MAX_TOKENS];
  __shared__ int s_cur, s_count, s_nlost, s_refused;
  __shared__ unsigned long long s_best[THREADS / 32];
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
  for (int t = tid; t < n; t += THREADS) {
    const Stat* st = A.stats + (first + t) * A.segments;
    float top = st[0].top;
    int arg = st[0].arg;
    for (int s = 1; s < A.segments; ++s)
      if (st[s].top > top) {
        top = st[s].top;
        arg = st[s].arg;
      }
    float sum = 0.f;
    for (int s = 0; s < A.segments; ++s) sum += st[s].sum * weight(st[s].top, top, inv_t);
    s_top[t] = top;
    s_sum[t] = sum;
    s_arg[t] = arg;
    int up = t == 0 ? -1 : (A.parents ? A.parents[first + t] : t - 1);
    const int64_t x = A.tokens[first + t];
    if (t > 0 && (up < 0 || up >= t || x < 0 || x >= A.V)) {
      atomicOr(A.err, ERR_TREE);   // a bad parent or token: the drafted token is never taken
      up = -2;
    }
    s_par[t] = up;
    s_tok[t] = x;
    s_coin[t] = A.coin ? A.coin[first + t] : 0.f;
    s_qx[t] = A.probs && up >= 0 ? A.probs[(first + t) * A.probs_stride + x] : 1.f;
  }
  __syncthreads();
  for (int t = tid; t < n; t += THREADS) {
    const int up = s_par[t];
    float p = 0.f;
    if (up >= 0 && !greedy)
      p = weight(tidy(logit<TYPE>(A.logits, (first + up) * A.row_stride + s_tok[t])), s_top[up],
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
  const int cur = s_cur, count = s_count, nlost = s_nlost;
  if (part == 0) {
    for (int i = tid; i < A.most; i += THREADS) {
      path[i] = i <= count ? s_path[i] : -1;
      if (i != count) out[i] = i < count ? s_tok[s_path[i + 1]] : -1;
    }
    if (tid == 0) {
      A.accepted[b] = count;
      if (greedy) out[count] = s_arg[cur];
    }
  }
  if (greedy) return;
  const float* q = A.probs && s_refused >= 0 ? A.probs + (first + s_refused) * A.probs_stride
                                             : nullptr;
  const float* noise = A.noise + (int64_t)b * A.noise_stride;
  const int64_t base = (first + cur) * A.row_stride;
  const float top = s_top[cur], sum = s_sum[cur];
  const int lo = (int)((int64_t)A.V * part / A.parts);
  const int hi = (int)((int64_t)A.V * (part + 1) / A.parts);
  unsigned long long best = 0;
  for (int i = lo + tid; i < hi; i += THREADS) {
    const float p = weight(tidy(logit<TYPE>(A.logits, base + i)), top, inv_t) / sum;
    float left = q ? fmaxf(p - q[i], 0.f) : p;
    if (!A.probs)
      for (int j = 0; j < nlost; ++j)
        if (s_lost[j] == i) left = 0.f;
    const unsigned long long key = race_key(left, p, noise[i], i);
    if (key > best) best = key;
  }
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
    if (other > best) best = other;
  }
  if (lane == 0) s_best[warp] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < THREADS / 32; ++w)
      if (s_best[w] > best) best = s_best[w];
    atomicMax(&A.race[b].best, best);
    __threadfence();
    if (atomicAdd(&A.race[b].arrived, 1) == A.parts - 1) {
      const unsigned long long won = atomicExch(&A.race[b].best, 0ull);
      A.race[b].arrived = 0;
      out[count] = (int64_t)(0xffffffffu - (uint32_t)won);
    }
  }
}

// Segments of a row and CTAs of a request: enough CTAs to fill the GPU.
static void split(int64_t B, int64_t most, int64_t V, int sms, int* segments, int* parts) {
  auto pick = [&](int64_t units) {
    int64_t s = (2 * (int64_t)sms + units - 1) / units;
    const int64_t by_size = (V + 4095) / 4096;
    if (s > by_size) s = by_size;
    if (s > MAX_SEGMENTS) s = MAX_SEGMENTS;
    return (int)(s < 1 ? 1 : s);
  };
  *segments = pick(B * most);
  *parts = pick(B);
}

static size_t power_of_two(int64_t n) {
  size_t p = 16;
  while ((int64_t)p < n) p *= 2;
  return p;
}

// The counters of up to MAX_REQUESTS requests come first, at the same place
// for every call, so that whatever call used the buffer before left them zero.
constexpr int MAX_REQUESTS = 65536;
constexpr size_t COUNTER_BYTES = MAX_REQUESTS * sizeof(Race);

}  // namespace verify
}  // namespace kb

extern "C" size_t kb_verify_drafts_workspace_size(int64_t B, int64_t rows) {
  if (B <= 0 || rows < 0) return 0;
  return kb::verify::COUNTER_BYTES +
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
             "verify: workspace of %zu bytes (256-byte aligned, zeroed once) required, %zu given",
             need, workspace_bytes);
  const int dev = kb::bind_stream_device(stream);
  v::Args A = {};
  A.logits = logits;
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
  A.stats = reinterpret_cast<v::Stat*>(static_cast<uint8_t*>(workspace) + v::COUNTER_BYTES);
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
