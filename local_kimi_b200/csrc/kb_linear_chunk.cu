// kb_linear_chunk.cu - linear attention with a decay for each head over prompts, in chunks of
// 128 tokens on the 5th-generation tensor cores (bf16).
//
// With b_i the running sum of the decays' logarithms in a chunk, for its rows i and j <= i:
//   P_ij = (q_i . k_j) exp(b_i - b_j)
//   o_i  = scale * (exp(b_i) q_i S + sum_j P_ij v_j)
//   S'   = exp(b_C) S + sum_j k_j (exp(b_C - b_j) v_j)^T
// Every exponent is at most 0.  Rows and keys in groups of 32: within one, exp(b_i - b_j) is
// computed; across groups it is exp(b_e - b_j) exp(b_i - b_e), e the last row of j's group, so
// that a row needs one exponential a group.  The sums are made in 64 bits and kept for each group
// from its start on, b_i - b_e from there and the sums of the groups between.  A decay that is 0 in fp32 (below e^-104, -infinity
// too) counts as e^-104 in the sums, whose exponentials then are 0.
//
// One persistent CTA per SM; a unit is one head of one request (or of a segment of it), its
// chunks one after the other.  Q, K and V tiles (128 rows, 64-element blocks in the 128-byte
// swizzle) arrive by tensor copies in two or three stages.  A kernel before makes the decays of all
// chunks and orders the requests.
//
//   warp 26: the units and the copies.
//   warp 24: issues S = Q K^T, O = Q S (the state), O += P V.
//   warp 25: issues S^T += V'^T K, V' = the values with their decay to the chunk's end.
//   warps 0-7: the state, in their registers in fp32 (a value column a thread, half of the key
//     rows each); its bf16 copy is what Q S reads.
//   warps 8-15: P from the scores, a row per thread and half the columns each; the part of the
//     state scaled by exp(b_i) in tensor memory before P V is added to it; the outputs, which
//     leave by tensor copies from the place of the chunk's queries.
//   warps 16-23: V', 32 rows at a time in two buffers, transposed on the way from shared to
//     tensor memory (eight by eight pieces, ldmatrix and 16-lane stores).
//
// Few heads: a request is cut into segments, and a first pass over all but the last makes each
// one's gain and decay alone (warps 0-7 hold it, 8-23 make V' in four buffers, nothing else
// runs); the second starts each segment from the gains before it.
//
// Bound: not the memory (8192 tokens of 32 heads of 128 x 128 move 269 MB, 41 us) nor the tensor
// cores (51 GFLOP a pass, three of six products the parts of V'; active 38 % of the second pass),
// but a chunk's way from the scores over P and P V to the outputs: 6000 clocks of latencies in
// one CTA an SM, since the state and two stages take the shared memory.  Roles on warps of their
// own let the state, V' and the copies of other chunks run beside it.  The first pass takes 2200
// clocks a chunk.  Measured, replayed: 104 us; 24 prompts of 1 to 2047 tokens with 24 heads
// 128 x 64 on 4 of queries and keys 67 us (108 MB at least: 16.4).  Token by token: 10700 and
// 2630.  What does not fill the chain either: with values up to 64 wide half of the gain's 128
// rows are empty, and each value head walks its chunks alone, also where it shares q and k with
// others (their copies and Q K^T again for each).
//
// The code is in short loops, not unrolled: all roles together have to fit the instruction cache
// (126 -> 111 us).  Slower: outputs by warps apart from the weights' (114 to 135 us, one barrier
// and one exchange more in the chunk's way), prefetching stages into L2 (111).
//
// Roundings.  P and the copy of the state are rounded once to bf16 before they meet the values
// and the queries: the outputs have 8 bits themselves, and end 1.4 times as far from the exact
// ones as fp32 products rounded once (0.0023 of their norm, 0.0017).  P's exponents are off by
// at most 2^-11 (two fp32 values below 4802 of a group), their exponentials, the approximate
// instruction's, by 2^-22 of themselves: together a tenth of P's rounding.  The state must not
// lose bits: V' (fp32 products) enters the tensor cores as the sum of three bf16 values, 24 bits
// in all.
//
// 512 columns of tensor memory, allocated in full: scores and P 128 (P takes 64 of them), O 128,
// the state's gain 128, V' 2 x 48, 64 apart (in the first pass 4 x 48 in the place of scores and
// O).
//
// A row past the request's end belongs to a neighbour: its keys and values are zeroed in shared
// memory.  A value that is no number is zeroed too, since it would meet zero weights; the rows
// from its token on are set to not-a-number at the end, and the state gets it from V'.
#include <algorithm>

#include "kb_linear.cuh"
#include "kb_tcgen05.cuh"

namespace kb {
namespace linear {

constexpr int CHUNK = 128;
constexpr int BLOCK = CHUNK * 128;           // bytes of 128 rows x 64 elements
constexpr int THREADS = 896;
constexpr int MOST_STAGES = 3;
constexpr int STATE_WARPS = 8, OUT_WARPS = 8, VALUE_WARPS = 8;
constexpr int VALUE_FIRST = STATE_WARPS + OUT_WARPS;
constexpr int MMA_WARP = 24, GAIN_WARP = 25, COPY_WARP = 26;
constexpr float RESET = -104.f;
constexpr int GROUP = 32;                    // rows of V' that are made at a time
constexpr uint32_t S_AT = 0, O_AT = 128, GAIN_AT = 256, PARTS_STEP = 64;

// The decays of a chunk and head.
struct Decays {
  float at[CHUNK];                           // b_i from the row's group's start on, base 2
  float left[CHUNK];                         // exp(b_e - b_j), e the last row of j's group
  float on[CHUNK / GROUP];                   // exp(b_C - b_e) of each group
  float keep;                                // exp(b_C)
  float whole[CHUNK / GROUP - 1];            // the sums of whole groups, base 2
};
static_assert(sizeof(Decays) % 16 == 0, "bulk copies");

struct ChunkArgs {
  Args a;
  Decays* decays;                            // [chunks][H], place_of() chunks
  int* order;                                // requests, longest first; NULL: units by number
  int* taken;                                // with it: units taken beyond each CTA's first
  int segments, segment;                     // of a request at most; tokens of one
  float* sums;                               // [B][segments][H][DKP][DVP]: a segment's gain
  float* keeps;                              // [B][segments][H]: its decay
  // In the place of a request's last segment's gain, which nobody starts from: the state that a
  // request of several segments starts from.  (Its last segment may be done, and its state
  // written, before another one begins.)
  __device__ __forceinline__ float* kept(int b, int h, int unit) const {
    return sums + (((int64_t)b * segments + segments - 1) * a.H + h) * unit;
  }
};

struct Item {
  int64_t first;                             // the chunk's first token
  int n;                                     // its tokens, -1: the end
  int64_t place;                             // of its decays
  int b, h, seg;
  int starts;                                // the unit's first chunk; 2: of several segments
  int ends;                                  // the unit's last chunk; 2: the request's
  int odd;                                   // values that are no numbers
};

template <int DKP, int DVP, bool STATES>
struct ChunkShape {
  static constexpr int KC = DKP / 64, VC = DVP / 64;
  static constexpr int K_AT = STATES ? 0 : KC * BLOCK;   // of a stage: Q, K, V
  static constexpr int V_AT = K_AT + KC * BLOCK;
  static constexpr int STAGE = V_AT + VC * BLOCK;
  static constexpr int STATE = STATES ? 0 : KC * DVP * 128;   // bytes of the bf16 copy
  // Groups of V' at a time: without scores and outputs their warps and columns serve it too.
  // Outputs leave through the place of Q where that is as wide.
  static constexpr bool STAGED = DKP >= DVP;
  static constexpr int BUFFERS = STATES ? 4 : 2;
  static constexpr uint32_t PARTS_AT = STATES ? 0 : 384;
  static constexpr int FIT = (224 * 1024 - STATE) / STAGE;
  static_assert(FIT >= 2, "stages");
  static constexpr int STAGES = FIT < MOST_STAGES ? FIT : MOST_STAGES;
  // (Three stages leave room for their arrays.)
  static constexpr int FIXED = STAGES > 2 ? 4608 : 3 * 1024;
  static constexpr int SMEM = STAGES * STAGE + STATE + FIXED;
};

template <int N>                             // stages
struct ChunkShared {
  alignas(16) Decays decays[N];
  uint8_t odd_from[2][CHUNK];                // of each value column, of every other group
  Item item[N], out[N];                      // out: whose outputs are to be sent
  uint64_t full[N], q_full[N], info[N], empty[N], staged[N];
  uint64_t clean[N];                         // (the values may run ahead of the outputs)
  uint64_t v_full[4], v_free[4];             // of the groups of V'
  uint64_t s_full, q_done, p_full, o_full, o_free, state_ready, gain_done, gain_free, drain;
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(ChunkShared<2>) <= 3 * 1024 && sizeof(ChunkShared<3>) <= 4608, "shared memory");

__device__ __forceinline__ void store_tile(const CUtensorMap* map, const void* from, int x, int y,
                                           int z) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];"
      ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(0),
        "r"(smem_addr(from))
      : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

__device__ __forceinline__ void stored_from_shared() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
               : "memory");
}

// 16 lanes of tensor memory x 4 columns from 8 x 8 pieces as ldmatrix transposes them: thread t
// has column t % 4 of row t / 4 (v0) and of row 8 + t / 4 (v1).
__device__ __forceinline__ void tmem_st_pieces(uint32_t taddr, uint32_t v0, uint32_t v1) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x1.b32 [%0], {%1,%2};"
               ::"r"(taddr), "r"(v0), "r"(v1)
               : "memory");
}

// (Beside a store to global memory, plain code makes one store of both whose space is unknown.)
__device__ __forceinline__ void store_shared(uint32_t to, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};"
               ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) {
  return __uint_as_float(w & 0xffff0000u);
}

// Where a request's chunks' decays start: places enough for all before, without a sum over them.
__device__ __forceinline__ int64_t place_of(int64_t first, int b) { return first / CHUNK + b; }

// The units of this CTA and their chunks, in order.
//
// With more units than CTAs a CTA takes its next from a counter, one ahead, requests longest
// first.
struct Items {
  const ChunkArgs& C;
  int64_t unit, units;
  int64_t at, first, end, last;              // tokens: the unit's left; the request's
  Item next;
  bool states;
  int ahead;
  __device__ __forceinline__ Items(const ChunkArgs& c, bool s)
      : C(c), at(0), first(0), end(0), last(0), states(s), ahead(blockIdx.x) {
    unit = (int64_t)blockIdx.x - gridDim.x;
    units = (int64_t)C.a.B * C.segments * C.a.H;
    advance();
  }
  __device__ __forceinline__ void advance() {
    const Args& A = C.a;
    next.starts = 0;
    while (at >= end) {
      if (C.order == nullptr) {
        unit += gridDim.x;
      } else {
        unit = __shfl_sync(0xffffffffu, ahead, 0);
        if ((threadIdx.x & 31) == 0 && unit < units)
          ahead = (int)gridDim.x + atomicAdd(C.taken, 1);
      }
      if (unit >= units) {
        next.n = -1;
        return;
      }
      const int64_t bs = unit / A.H;
      next.h = (int)(unit - bs * A.H);
      next.b = (int)(bs / C.segments);
      next.seg = (int)(bs - (int64_t)next.b * C.segments);
      if (C.order != nullptr) next.b = __ldg(C.order + next.b);
      const int n = request_tokens(A, next.b, first);
      at = first + (int64_t)next.seg * C.segment;
      last = first + n;
      end = min(last, at + C.segment);
      // The last segment's gain is nobody's start.
      if (states && end >= last) end = at;
      next.starts = n > C.segment ? 2 : 1;
    }
    next.first = at;
    next.n = (int)min(end - at, (int64_t)CHUNK);
    next.place = (place_of(first, next.b) + (at - first) / CHUNK) * A.H + next.h;
    at += CHUNK;
    next.ends = at < end ? 0 : end < last ? 1 : 2;
  }
};

// ---------------------------------------------------------------------------
// The decays of every chunk, a warp a chunk and head (which clears rows past a request's longest
// too); the last CTA orders the requests, or the last ones copy states.
// (A warp of the chunks' kernel that made them beside its other work took 5000 to 8000 clocks a
// chunk, more than the chunk: 8192 tokens x 32 heads 122 us.)
// ---------------------------------------------------------------------------

constexpr int PREPARE_THREADS = 256;

// A row a lane, four groups side by side.  All sums are in 64 bits and rounded once, when they are
// stored.  Nothing is summed across groups but what a weight needs: a sum over the chunk may reach
// 19000 (base 2) beside differences next to nothing, where fp32's step is half of a bf16 weight's.
// In a group it stays below 4802, and a difference within 2^-11.
__device__ __forceinline__ void chunk_decays(const Args& A, int64_t first, int n, int h,
                                             Decays* D) {
  constexpr int GROUPS = CHUNK / GROUP;
  const int lane = threadIdx.x & 31;
  float log[GROUPS];
  double up[GROUPS], behind[GROUPS];
  unsigned marks[GROUPS];
  int none = CHUNK;                          // the first logarithm that is no number
#pragma unroll
  for (int p = 0; p < GROUPS; ++p) {
    const int j = p * GROUP + lane;
    log[p] = j < n ? __ldg(A.decay + (first + j) * A.decay_tok + h) : 0.f;
  }
#pragma unroll
  for (int p = 0; p < GROUPS; ++p) {
    const float x = decay_of(log[p]);
    marks[p] = __ballot_sync(0xffffffffu, x <= RESET);
    const unsigned odd = __ballot_sync(0xffffffffu, x != x);
    if (odd) none = min(none, p * GROUP + __ffs(odd) - 1);
    up[p] = x != x ? 0.0 : fmaxf(x, RESET) * 1.4426950408889634;
    behind[p] = __shfl_down_sync(0xffffffffu, up[p], 1);
    if (lane == 31) behind[p] = 0.0;
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int p = 0; p < GROUPS; ++p) {
      const double z = __shfl_down_sync(0xffffffffu, behind[p], o);
      if (lane + o < 32) behind[p] += z;
    }
  double whole[GROUPS], after = 0.0;
  float at[GROUPS], left[GROUPS], on[GROUPS];
  int later = 0;
#pragma unroll
  for (int p = 0; p < GROUPS; ++p) {
    whole[p] = __shfl_sync(0xffffffffu, up[p] + behind[p], 0);
    at[p] = (float)(whole[p] - behind[p]);
  }
#pragma unroll
  for (int p = GROUPS - 1; p >= 0; --p) {
    on[p] = later ? 0.f : exp2f((float)after);
    after += whole[p];
    later |= marks[p] != 0;
    // A reset behind the row, in its group.
    const unsigned rest = lane < 31 ? marks[p] >> (lane + 1) : 0u;
    left[p] = p * GROUP + lane >= n || rest ? 0.f : exp2f((float)behind[p]);
  }
  float keep = later ? 0.f : exp2f((float)after);
  if (none < CHUNK) {                        // all sums over it are none either
    keep = NAN;
#pragma unroll
    for (int p = 0; p < GROUPS; ++p) {
      if (p * GROUP + lane >= none) at[p] = NAN;
      if (p == none / GROUP && p * GROUP + lane < none) left[p] = NAN;
      on[p] = NAN;
    }
  }
#pragma unroll
  for (int p = 0; p < GROUPS; ++p) {
    const int j = p * GROUP + lane;
    D->at[j] = at[p];
    D->left[j] = left[p];
  }
  if (lane == 0) {
    *reinterpret_cast<float4*>(D->on) = make_float4(on[0], on[1], on[2], on[3]);
    *reinterpret_cast<float4*>(&D->keep) =
        make_float4(keep, (float)whole[0], (float)whole[1], (float)whole[2]);
  }
}

template <bool SEGMENTS>                     // (their copies' registers cost the others 2 us)
__global__ void __launch_bounds__(PREPARE_THREADS)
    prepare_kernel(const ChunkArgs C, int64_t places, int unit) {
  const Args& A = C.a;
  constexpr int BUCKETS = 4 * PREPARE_THREADS;
  __shared__ int starts[BUCKETS];
  __shared__ int sums[PREPARE_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t rest = (int64_t)blockIdx.x - (places * A.H + PREPARE_THREADS / 32 - 1) /
                                                 (PREPARE_THREADS / 32);
  if (SEGMENTS && rest >= 0) {
    // A CTA a head: the states that segments start from.
    const int b = (int)(rest / A.H), h = (int)(rest - (int64_t)b * A.H);
    int64_t first;
    const float* from = request_state(A, b, h);
    if (from == nullptr || request_tokens(A, b, first) <= C.segment) return;
    float* to = C.kept(b, h, unit);
    constexpr int AT_ONCE = 16;
    static_assert(AT_ONCE * PREPARE_THREADS * 4 >= 128 * 128, "a state");
    float4 x[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = (tid + u * PREPARE_THREADS) * 4;
      if (i < A.Dk * A.Dv) x[u] = __ldcg(reinterpret_cast<const float4*>(from + i));
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = (tid + u * PREPARE_THREADS) * 4;
      if (i < A.Dk * A.Dv) *reinterpret_cast<float4*>(to + i) = x[u];
    }
    return;
  }
  if (rest < 0) {
    const int64_t at = (int64_t)blockIdx.x * (PREPARE_THREADS / 32) + warp;
    if (at >= places * A.H) return;
    const int64_t place = at / A.H;
    const int h = (int)(at - place * A.H);
    // The request: the last whose chunks start at or before the place.
    int lo = 0, hi = A.B - 1;
    auto start = [&](int b) {
      return place_of(min(max((int64_t)__ldg(A.cu + b), (int64_t)0), A.total), b);
    };
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start(mid) <= place) lo = mid; else hi = mid - 1;
    }
    int64_t first, end;
    const int n = request_tokens(A, lo, first, end);
    const int64_t skip = (place - place_of(first, lo)) * CHUNK;
    if (skip < 0 || first + skip >= end) return;
    // Rows of a request past its longest: zero.
    const int64_t after = min(end, first + skip + CHUNK);
    for (int64_t row = first + max(skip, (int64_t)n); row < after; ++row)
      if (lane * 8 < A.Dv)
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(A.out) + (row * A.H + h) * A.Dv)[lane] =
            make_uint4(0, 0, 0, 0);
    if (skip >= n) return;
    chunk_decays(A, first + skip, (int)min(n - skip, (int64_t)CHUNK), h, C.decays + at);
    return;
  }
  // Requests by number of chunks, most first; the longest ones together.
  auto bucket = [&](int b) {
    int64_t first;
    const int n = request_tokens(A, b, first);
    return BUCKETS - 1 - min((n + CHUNK - 1) / CHUNK, BUCKETS - 1);
  };
  if (tid == 0) *C.taken = 0;
  for (int i = tid; i < BUCKETS; i += PREPARE_THREADS) starts[i] = 0;
  __syncthreads();
  for (int b = tid; b < A.B; b += PREPARE_THREADS) atomicAdd(&starts[bucket(b)], 1);
  __syncthreads();
  int mine[4], in = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) in += mine[i] = starts[tid * 4 + i];
  const int own = in;
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += u;
  }
  if (lane == 31) sums[warp] = in;
  __syncthreads();
  for (int w = 0; w < warp; ++w) in += sums[w];
  in -= own;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    starts[tid * 4 + i] = in;
    in += mine[i];
  }
  __syncthreads();
  for (int b = tid; b < A.B; b += PREPARE_THREADS) C.order[atomicAdd(&starts[bucket(b)], 1)] = b;
}

template <int DKP, int DVP, bool STATES>
__global__ void __launch_bounds__(THREADS, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                 const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to,
                 const ChunkArgs C) {
  using Sh = ChunkShape<DKP, DVP, STATES>;
  constexpr int KC = Sh::KC, VC = Sh::VC, STAGES = Sh::STAGES;
  constexpr int HALF = DKP / 2;              // key rows of a thread's part of the state
  const Args& A = C.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* copy_of_state = smem + STAGES * Sh::STAGE;
  auto* B = reinterpret_cast<ChunkShared<STAGES>*>(copy_of_state + Sh::STATE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_f = &B->abort_flag;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&B->full[i], 1);
      mbar_init(&B->q_full[i], 1);
      mbar_init(&B->clean[i], VALUE_WARPS);
      mbar_init(&B->info[i], 1);
      mbar_init(&B->empty[i], STATES ? 1 + 4 * Sh::BUFFERS + STATE_WARPS
                                     : 2 + VALUE_WARPS + STATE_WARPS + OUT_WARPS);
      mbar_init(&B->staged[i], OUT_WARPS);
    }
    for (int i = 0; i < Sh::BUFFERS; ++i) {
      mbar_init(&B->v_full[i], 4);
      mbar_init(&B->v_free[i], 1);
    }
    mbar_init(&B->s_full, 1);
    mbar_init(&B->q_done, 1);
    mbar_init(&B->p_full, OUT_WARPS);
    mbar_init(&B->o_full, 1);
    mbar_init(&B->o_free, OUT_WARPS);
    mbar_init(&B->state_ready, STATE_WARPS);
    mbar_init(&B->gain_done, 1);
    mbar_init(&B->gain_free, STATE_WARPS);
    mbar_init(&B->drain, STATES ? 1 : 2);
    B->abort_flag = 0;
    mbar_fence_init();
    if (!STATES) attn::prefetch_map(&tq);
    attn::prefetch_map(&tk);
    attn::prefetch_map(&tv);
    if (!STATES) attn::prefetch_map(&to);
  }
  if (warp == COPY_WARP) tc::tmem_alloc_all(&B->tmem);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = B->tmem;
  pdl_wait();
  pdl_launch_dependents();

  // Rows outside every request: zero.
  if (!STATES) {
    const int64_t lead = min(max((int64_t)A.cu[0], (int64_t)0), A.total);
    const int64_t tail = min(max((int64_t)A.cu[A.B], lead), A.total);
    const int64_t width = (int64_t)A.H * A.Dv / 8, spare = (lead + A.total - tail) * width;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < spare;
         i += (int64_t)gridDim.x * THREADS)
      static_cast<uint4*>(A.out)[i < lead * width ? i : i - lead * width + tail * width] =
          make_uint4(0, 0, 0, 0);
  }

  // Bounded waits of a warp in step; one arrival a warp.
  bool ok = true;
  auto need = [&](uint64_t* bar, uint32_t parity) {
    ok = attn::warp_wait(bar, parity, abort_f, A.err);
    return ok;
  };
  auto arrive = [&](uint64_t* bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  int st = 0;
  uint32_t ph = 0, one_phase = 0;            // of the stages; of the barriers met once a chunk
  auto turn = [&]() {
    one_phase ^= 1u;
    if (++st == STAGES) {
      st = 0;
      ph ^= 1u;
    }
  };

  if (warp < STATE_WARPS) {
    // ------------------------------------------------------------------ the state
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int part = warp >> 2;              // key rows part * HALF ..
    const int dv = (warp & 3) * 32 + lane;
    const uint32_t gain_at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + GAIN_AT + part * HALF;
    const bool active = (warp & 3) * 32 < DVP;
    const int rows = dv < A.Dv ? min(max(A.Dk - part * HALF, 0), HALF) : 0;   // that there are
    float s[HALF];
    float all = 1.f;                         // the unit's decay so far
    // Segments' gains lie [DKP][DVP], zero where the head is narrower.
    const int64_t gain_mine = part * HALF * DVP + dv;
    // The bf16 copy, a value column's key rows side by side: what Q S reads.
    auto copy_state = [&]() {
      if (active) {
        uint8_t* row = copy_of_state + dv * 128;
#pragma unroll
        for (int c = 0; c < HALF / 8; ++c) {
          uint4 w;
          w.x = attn::pack2<false>(s[8 * c], s[8 * c + 1]);
          w.y = attn::pack2<false>(s[8 * c + 2], s[8 * c + 3]);
          w.z = attn::pack2<false>(s[8 * c + 4], s[8 * c + 5]);
          w.w = attn::pack2<false>(s[8 * c + 6], s[8 * c + 7]);
          const int piece = DKP == 64 ? part * 4 + c : c;
          uint8_t* block = row + (DKP == 64 ? 0 : part * DVP * 128);
          *reinterpret_cast<uint4*>(block + ((piece ^ (dv & 7)) << 4)) = w;
        }
      }
      attn::fence_proxy_async();
      arrive(&B->state_ready);
    };
    while (true) {
      if (!need(&B->info[st], ph)) break;
      const int n = B->item[st].n, b = B->item[st].b, h = B->item[st].h, seg = B->item[st].seg;
      const int starts = B->item[st].starts, ends = B->item[st].ends;
      if (n < 0) break;
      if (starts) {
        // What the unit starts from: the request's state, and the gains of the segments before.
#pragma unroll
        for (int i = 0; i < HALF; ++i) s[i] = 0.f;
        if (!STATES) {
          const float* from = request_state(A, b, h);
          if (from != nullptr && rows > 0) {
            if (starts == 2) from = C.kept(b, h, DKP * DVP);
            from += (int64_t)part * HALF * A.Dv + dv;
#pragma unroll
            for (int c = 0; c < HALF; c += 8, from += 8 * A.Dv) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (c < rows) s[c + i] = __ldcg(from + i * A.Dv);      // (rows: eights)
              asm volatile("" : "+l"(from));
            }
          }
          for (int g = 0; g < seg; ++g) {
            const int64_t u = ((int64_t)b * C.segments + g) * A.H + h;
            const float all_of_it = __ldcg(C.keeps + u);
            const float* gain = C.sums + u * (DKP * DVP) + gain_mine;
            if (active)
#pragma unroll
              for (int c = 0; c < HALF; c += 32) {
                float x[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = __ldcg(gain + (c + i) * DVP);
#pragma unroll
                for (int i = 0; i < 32; ++i) s[c + i] = fmaf(s[c + i], all_of_it, x[i]);
              }
          }
        }
      }
      if (!STATES) copy_state();
      if (!need(&B->full[st], ph)) break;
      const float keep = B->decays[st].keep;
      arrive(&B->empty[st]);
      if (!need(&B->gain_done, one_phase)) break;
      tc::tc_fence_after();
      if (active)
#pragma unroll
        for (int c = 0; c < HALF; c += 16) {
          uint32_t gain[16];
          tc::tmem_ld16(gain_at + c, gain);
          tc::tmem_ld_wait();
          tc::hold_regs(gain);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[c + i] = fmaf(s[c + i], keep, __uint_as_float(gain[i]));
        }
      tc::tc_fence_before();
      arrive(&B->gain_free);
      if (!STATES && !need(&B->q_done, one_phase)) break;
      if (ends) {
        const int64_t u = ((int64_t)b * C.segments + seg) * A.H + h;
        if (STATES) {
          if (threadIdx.x == 0) C.keeps[u] = all * keep;
          float* to = C.sums + u * (DKP * DVP) + gain_mine;
          if (active)
#pragma unroll
            for (int i = 0; i < HALF; ++i) to[i * DVP] = s[i];
        } else if (ends == 2) {
          float* to = request_state(A, b, h);
          if (to != nullptr && rows > 0) {
            to += (int64_t)part * HALF * A.Dv + dv;
#pragma unroll
            for (int c = 0; c < HALF; c += 8, to += 8 * A.Dv) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (c < rows) to[i * A.Dv] = s[c + i];
              asm volatile("" : "+l"(to));
            }
          }
        }
      }
      all = ends ? 1.f : all * keep;
      turn();
    }
  } else if (!STATES && warp < VALUE_FIRST) {
    // ---------------------------------------------------------------- the outputs
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    const int part = (warp >> 2) & 1;        // columns part * 64 .. of the scores
    const int warp_group = warp & 3, q0 = warp_group * GROUP, row = q0 + lane;
    const uint32_t lanes = tmem + ((uint32_t)q0 << 16);
    constexpr int COLS = DVP / 2;            // of the outputs a thread has
    while (true) {
      if (!need(&B->info[st], ph)) break;
      const Item I = B->item[st];
      if (I.n < 0) break;
      if (!need(&B->full[st], ph)) break;
      const Decays& D = B->decays[st];
      const float mine = D.at[row];
      if (!need(&B->s_full, one_phase)) break;
      tc::tc_fence_after();
      // (Loops that stay loops, here and below: each scheduler runs warps of every role, whose
      // code does not fit its instruction cache together.)
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        const int j0 = part * 64 + c * 16;   // columns of the scores
        uint32_t p[8];
        if (j0 >= q0 + GROUP) {              // all behind the rows
#pragma unroll
          for (int i = 0; i < 8; ++i) p[i] = 0;
        } else {
          uint32_t x[16];
          tc::tmem_ld16(lanes + S_AT + j0, x);
          tc::tmem_ld_wait();
          tc::hold_regs(x);
          auto scores = [&](int i) {
            return make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
          };
          if (j0 < q0) {
            // All before the rows: the decay to the group's end, and on to the row.
            const int group = j0 / GROUP;
            float b = mine;
            if (warp_group - group > 1) b += D.whole[group + 1];
            if (warp_group - group > 2) b += D.whole[2];
            const float on = exp2_fast(b);
            const float2 on2 = make_float2(on, on);
            const float* left = &D.left[j0];
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 d = *reinterpret_cast<const float4*>(left + i);
              const float2 a = fmul2(fmul2(scores(i), make_float2(d.x, d.y)), on2);
              const float2 b = fmul2(fmul2(scores(i + 2), make_float2(d.z, d.w)), on2);
              p[i / 2] = attn::pack2<false>(a.x, a.y);
              p[i / 2 + 1] = attn::pack2<false>(b.x, b.y);
            }
          } else {
            const float2 here = make_float2(mine, mine), minus = make_float2(-1.f, -1.f);
            const float* at = &D.at[j0];
            // Columns up to the row.
            const uint32_t seen = (0xffffffffu >> (31 - lane)) >> (j0 - q0);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 b = *reinterpret_cast<const float4*>(at + i);
              float2 e = ffma2(make_float2(b.x, b.y), minus, here);
              float2 f = ffma2(make_float2(b.z, b.w), minus, here);
              e = fmul2(scores(i), make_float2(exp2_fast(e.x), exp2_fast(e.y)));
              f = fmul2(scores(i + 2), make_float2(exp2_fast(f.x), exp2_fast(f.y)));
              if (!((seen >> i) & 1)) e.x = 0.f;
              if (!((seen >> (i + 1)) & 1)) e.y = 0.f;
              if (!((seen >> (i + 2)) & 1)) f.x = 0.f;
              if (!((seen >> (i + 3)) & 1)) f.y = 0.f;
              p[i / 2] = attn::pack2<false>(e.x, e.y);
              p[i / 2 + 1] = attn::pack2<false>(f.x, f.y);
            }
          }
        }
        // (In place of scores that this thread has read.)
        tmem_st8(lanes + S_AT + part * 64 + c * 8, p);
      }
      if (!need(&B->q_done, one_phase)) break;
      tc::tc_fence_after();
      float b = mine;
      for (int g = 0; g < warp_group; ++g) b += D.whole[g];
      const float gain = exp2_fast(b);
#pragma unroll 1
      for (int c = 0; c < COLS / 16; ++c) {
        uint32_t o[16];
        tc::tmem_ld16(lanes + O_AT + part * COLS + c * 16, o);
        tc::tmem_ld_wait();
        tc::hold_regs(o);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * gain);
        tc::tmem_st16(lanes + O_AT + part * COLS + c * 16, o);
      }
      tc::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B->p_full);
      if (!need(&B->o_full, one_phase)) break;
      tc::tc_fence_after();
      const int odd = *const_cast<volatile int*>(&B->item[st].odd);
      // The warp's 32 rows and COLS columns go through the place of the queries, which nobody
      // reads any more; the rows at a request's end go out by themselves.
      uint16_t* out = static_cast<uint16_t*>(A.out) +
                      ((I.first + row) * A.H + I.h) * A.Dv + part * COLS;
      uint8_t* tile = smem + st * Sh::STAGE + (part * CHUNK + q0) * COLS * 2;
      const bool whole = Sh::STAGED && q0 + 32 <= I.n && odd == 0;
      if (odd == 0) arrive(&B->empty[st]);
      const float2 scale2 = make_float2(A.scale, A.scale);
#pragma unroll 1
      for (int c = 0; c < COLS / 16; ++c) {
        uint32_t o[16];
        tc::tmem_ld16(lanes + O_AT + part * COLS + c * 16, o);
        tc::tmem_ld_wait();
        tc::hold_regs(o);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 x = fmul2(make_float2(__uint_as_float(o[8 * i + 2 * k]),
                                               __uint_as_float(o[8 * i + 2 * k + 1])), scale2);
            w[k] = attn::pack2<false>(x.x, x.y);
          }
          const uint4 piece = make_uint4(w[0], w[1], w[2], w[3]);
          const int at = (c * 2 + i) ^ (COLS == 64 ? lane & 7 : (lane >> 1) & 3);
          if (whole)
            store_shared(smem_addr(tile) + lane * COLS * 2 + at * 16, piece);
          else if (row < I.n && part * COLS + c * 16 + i * 8 < A.Dv)
            *reinterpret_cast<uint4*>(out + c * 16 + i * 8) = piece;
        }
      }
      if (odd && row < I.n)
        for (int d = part * COLS; d < min(A.Dv, (part + 1) * COLS); ++d)
          for (int buffer = 0; buffer < 2; ++buffer)
            if (((odd >> (buffer * 4 + (d >> 5))) & 1) && row >= B->odd_from[buffer][d])
              out[d - part * COLS] = 0x7fff;
      tc::tc_fence_before();
      if (whole) attn::fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&B->o_free);
        mbar_arrive(&B->staged[st]);
        if (odd) mbar_arrive(&B->empty[st]);
      }
      turn();
    }
  } else if (warp < MMA_WARP) {
    // ------------------------------------------- the values with their decay, V'
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // A strip of 32 columns; the groups of rows of one of the buffers.
    constexpr int FIRST = STATES ? STATE_WARPS : VALUE_FIRST;
    const int strip = warp & 3, buffer = (warp - FIRST) >> 2;
    const uint32_t to =
        tmem + ((uint32_t)(strip * 32) << 16) + Sh::PARTS_AT + buffer * PARTS_STEP;
    const bool active = strip * 32 < DVP;
    uint32_t free_phase = 1;
    bool any = false;                        // a chunk before this one
    while (ok) {
      if (!need(&B->info[st], ph)) break;
      const int n = B->item[st].n;
      if (n < 0) break;
      if (!need(&B->full[st], ph)) break;
      uint8_t* k_tile = smem + st * Sh::STAGE + Sh::K_AT;
      uint8_t* v_tile = smem + st * Sh::STAGE + Sh::V_AT + (active ? (strip >> 1) * BLOCK : 0);
      if (n < CHUNK) {
        // Rows of a neighbour: zero.  (Of this buffer's groups, since a group's product waits for
        // its buffer's warps alone; of the values, those that this warp reads.)
        for (int j = n + strip * 4 + (lane >> 3); j < CHUNK; j += 16)
          if ((j / GROUP) % Sh::BUFFERS == buffer)
            for (int c = 0; c < KC; ++c)
              *reinterpret_cast<uint4*>(k_tile + c * BLOCK + j * 128 + (lane & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
        if (active)
          for (int j = n + (lane >> 2); j < CHUNK; j += 8)
            if ((j / GROUP) % Sh::BUFFERS == buffer)
              *reinterpret_cast<uint4*>(v_tile + j * 128 +
                                        ((((strip & 1) * 4 + (lane & 3)) ^ (j & 7)) << 4)) =
                  make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      float2 odd = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int g = buffer; g < CHUNK / GROUP; g += Sh::BUFFERS) {
        const float on = B->decays[st].on[g];
        const float2 on2 = make_float2(on, on);
        if (!need(&B->v_free[buffer], free_phase)) break;
        free_phase ^= 1u;
        tc::tc_fence_after();
        // Eight rows a piece: pairs of rows of column 8 c + lane / 4, rows 2 (lane % 4) and on.
        const uint32_t from = smem_addr(v_tile) + (g * GROUP + (lane & 7)) * 128 +
                              ((((strip & 1) * 4 + (lane >> 3)) ^ (lane & 7)) << 4);
        const float* left = &B->decays[st].left[g * GROUP + (lane & 3) * 2];
#pragma unroll 1
        for (int r = 0; r < 4; ++r) {
          uint32_t w[4], part[3][4];         // low, middle, high
          attn::ldmatrix_x4_trans(w, from + r * 8 * 128);
          const float2 d = fmul2(*reinterpret_cast<const float2*>(left + r * 8), on2);
          const float2 minus = make_float2(-1.f, -1.f);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float2 x = make_float2(low_half(w[c]), high_half(w[c]));
            odd = ffma2(x, make_float2(0.f, 0.f), odd);
            x = fmul2(x, d);
            const uint32_t hi = attn::pack2<false>(x.x, x.y);
            x = ffma2(make_float2(low_half(hi), high_half(hi)), minus, x);
            const uint32_t mid = attn::pack2<false>(x.x, x.y);
            x = ffma2(make_float2(low_half(mid), high_half(mid)), minus, x);
            part[0][c] = attn::pack2<false>(x.x, x.y);
            part[1][c] = mid;
            part[2][c] = hi;
          }
          if (active)
#pragma unroll
            for (int t = 0; t < 3; ++t) {
              tmem_st_pieces(to + t * 16 + r * 4, part[t][0], part[t][1]);
              tmem_st_pieces(to + (16u << 16) + t * 16 + r * 4, part[t][2], part[t][3]);
            }
        }
        tc::tmem_st_wait();
        attn::fence_proxy_async();           // the zeroed keys
        tc::tc_fence_before();
        arrive(&B->v_full[buffer]);
      }
      if (!ok) break;
      // (The test is true of not-a-number.)
      const bool first_one = !any;
      any = true;
      if (!STATES && active && __any_sync(0xffffffffu, odd.x + odd.y != 0.f)) {
        const int dv = strip * 32 + lane, piece = (dv & 63) >> 3;
        int first = 255;
        for (int j = 0; j < n; ++j) {
          if ((j / GROUP) % Sh::BUFFERS != buffer) continue;
          uint16_t* e = reinterpret_cast<uint16_t*>(v_tile + j * 128 + (dv & 7) * 2 +
                                                    ((piece ^ (j & 7)) << 4));
          if (attn::odd_element<false>(*e)) {
            first = min(first, j);
            *e = 0;
          }
        }
        // (The outputs of the chunk before may still be reading theirs.)
        if (!first_one && !need(&B->staged[st == 0 ? STAGES - 1 : st - 1],
                                st == 0 ? ph ^ 1u : ph))
          break;
        B->odd_from[buffer][dv] = (uint8_t)first;
        __syncwarp();
        if (lane == 0) atomicOr(&B->item[st].odd, 1 << (buffer * 4 + strip));
        attn::fence_proxy_async();
      }
      __syncwarp();
      if (lane == 0) {
        if (!STATES) mbar_arrive(&B->clean[st]);
        mbar_arrive(&B->empty[st]);
      }
      turn();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // A and B bf16, sums fp32, 128 rows.
    constexpr uint32_t COMMON = (1u << 4) | (1u << 7) | (1u << 10) | ((CHUNK >> 4) << 24);
    constexpr uint32_t MN = 1u << 16;        // B as it lies: rows along the products' axis
    const uint32_t one = tc::elect_one();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t base = smem_addr(smem);
    if (warp == MMA_WARP && !STATES) {
      // -------------------------------------------------------- scores and outputs
      constexpr uint32_t ID_S = COMMON | ((CHUNK >> 3) << 17);
      constexpr uint32_t ID_Q = COMMON | ((DVP >> 3) << 17);
      constexpr uint32_t ID_P = COMMON | MN | ((DVP >> 3) << 17);
      const uint32_t state_at = smem_addr(copy_of_state);
      while (true) {
        if (!need(&B->info[st], ph)) break;
        if (B->item[st].n < 0) break;
        if (!need(&B->full[st], ph) || !need(&B->q_full[st], ph)) break;
        tc::tc_fence_after();
        const uint32_t q_at = base + st * Sh::STAGE, k_at = q_at + Sh::K_AT;
        const uint32_t v_at = q_at + Sh::V_AT;
#pragma unroll 1
        for (int c = 0; c < KC; ++c) {
          const uint64_t a = tc::sw128_desc(q_at + c * BLOCK);
          const uint64_t b = tc::sw128_desc(k_at + c * BLOCK);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc::umma_one(one, tm + S_AT, a + k * 2, b + k * 2, ID_S, c + k > 0);
        }
        tc::umma_commit_one(one, &B->s_full);
        if (!need(&B->state_ready, one_phase) || !need(&B->o_free, one_phase ^ 1u)) break;
        tc::tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < KC; ++c) {
          const uint64_t a = tc::sw128_desc(q_at + c * BLOCK);
          const uint64_t b = tc::sw128_desc(state_at + c * DVP * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc::umma_one(one, tm + O_AT, a + k * 2, b + k * 2, ID_Q, c + k > 0);
        }
        tc::umma_commit_one(one, &B->q_done);
        if (!need(&B->clean[st], ph) || !need(&B->p_full, one_phase)) break;
        tc::tc_fence_after();
        const uint64_t b = tc::sw128_desc_mn(v_at, BLOCK);
#pragma unroll 2
        for (int k = 0; k < CHUNK / 16; ++k)
          tc::umma_ts_one(one, tm + O_AT, tm + S_AT + (k >> 2) * 64 + (k & 3) * 8,
                          b + k * (2048 >> 4), ID_P, 1);
        tc::umma_commit_one(one, &B->o_full);
        tc::umma_commit_one(one, &B->empty[st]);
        turn();
      }
      tc::umma_commit_one(one, &B->drain);
      attn::drain_phase(&B->drain, 0);
    } else if (warp == GAIN_WARP) {
      // --------------------------------------------------------- the state's gain
      constexpr uint32_t ID_V = COMMON | MN | ((DKP >> 3) << 17);
      uint32_t full_phase = 0;
      while (ok) {
        if (!need(&B->info[st], ph)) break;
        if (B->item[st].n < 0) break;
        if (!need(&B->full[st], ph) || !need(&B->gain_free, one_phase ^ 1u)) break;
        const uint64_t b = tc::sw128_desc_mn(base + st * Sh::STAGE + Sh::K_AT, BLOCK);
#pragma unroll 1
        for (int g = 0; g < CHUNK / GROUP; ++g) {
          const int buffer = g % Sh::BUFFERS;
          if (!need(&B->v_full[buffer], full_phase)) break;
          tc::tc_fence_after();
#pragma unroll 1
          for (int t = 0; t < 3; ++t)
#pragma unroll
            for (int k = 0; k < GROUP / 16; ++k)
              tc::umma_ts_one(one, tm + GAIN_AT,
                              tm + Sh::PARTS_AT + buffer * PARTS_STEP + t * 16 + k * 8,
                              b + (g * (GROUP / 16) + k) * (2048 >> 4), ID_V,
                              (uint32_t)(g + t + k > 0));
          tc::umma_commit_one(one, &B->v_free[buffer]);
          full_phase ^= (uint32_t)(buffer == Sh::BUFFERS - 1);
        }
        if (!ok) break;
        tc::umma_commit_one(one, &B->gain_done);
        tc::umma_commit_one(one, &B->empty[st]);
        turn();
      }
      tc::umma_commit_one(one, &B->drain);
      attn::drain_phase(&B->drain, 0);
    } else if (warp == COPY_WARP) {
      // -------------------------------------------------------------------- copies
      const uint64_t keep_in_l2 = l2_evict_last_policy(), once = l2_evict_first_policy();
      const uint64_t k_policy = STATES || A.k_group > 1 ? keep_in_l2 : once;
      const uint64_t q_policy = A.q_group > 1 ? keep_in_l2 : once;
      const uint64_t v_policy = STATES ? keep_in_l2 : once;
      // A stage's outputs leave before its next queries.  Lanes 0 to 7: 32 rows and COLS columns
      // each.
      auto send = [&](int st, uint32_t parity) {
        if (!need(&B->staged[st], parity)) return;
        const Item& I = B->out[st];
        const int part = lane >> 2, q0 = (lane & 3) * 32;
        if (Sh::STAGED && lane < 8 && q0 + 32 <= I.n && I.odd == 0 && part * (DVP / 2) < A.Dv) {
          store_tile(&to, smem + st * Sh::STAGE + (part * CHUNK + q0) * DVP, part * (DVP / 2), I.h,
                     (int)I.first + q0);
          stored_from_shared();
        }
        __syncwarp();
      };
      Items items(C, STATES);
      int sent = 0;
      while (true) {
        if (!need(&B->empty[st], ph ^ 1u)) break;
        const bool more = items.next.n >= 0;
        const int token = (int)items.next.first, h = items.next.h;
        uint8_t* to_stage = smem + st * Sh::STAGE;
        if (lane == 0) {
          if (!STATES && sent >= STAGES) B->out[st] = B->item[st];
          Item I = items.next;
          I.odd = 0;
          B->item[st] = I;
          mbar_arrive(&B->info[st]);
          if (more) {
            mbar_arrive_expect_tx(&B->full[st],
                                  (uint32_t)((KC + VC) * BLOCK + sizeof(Decays)));
            bulk_g2s(&B->decays[st], C.decays + items.next.place, sizeof(Decays), &B->full[st],
                     once);
            for (int c = 0; c < KC; ++c)
              attn::tma_load_4d(to_stage + Sh::K_AT + c * BLOCK, &tk, c * 64, h / A.k_group, token,
                                0, &B->full[st], k_policy);
            for (int c = 0; c < VC; ++c)
              attn::tma_load_4d(to_stage + Sh::V_AT + c * BLOCK, &tv, c * 64, h, token, 0,
                                &B->full[st], v_policy);
          }
        }
        __syncwarp();
        if (!more) break;
        if (!STATES) {
          if (sent >= STAGES) send(st, ph ^ 1u);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&B->q_full[st], (uint32_t)(KC * BLOCK));
            for (int c = 0; c < KC; ++c)
              attn::tma_load_4d(to_stage + c * BLOCK, &tq, c * 64, h / A.q_group, token, 0,
                                &B->q_full[st], q_policy);
          }
          __syncwarp();
        }
        ++sent;
        items.advance();
        turn();
      }
      // The last outputs: `st` is the oldest stage, if all are in use, its item set aside.
      if (!STATES && ok)
        for (int i = max(0, STAGES - sent); i < STAGES && ok; ++i) {
          const int at = (st + i) % STAGES;
          const uint32_t parity = (uint32_t)((sent - STAGES + i) / STAGES) & 1u;
          if (i > 0) {
            if (!need(&B->staged[at], parity)) break;
            if (lane == 0) B->out[at] = B->item[at];
            __syncwarp();
          }
          send(at, parity);
        }
      // On the error path, copies in flight land before the CTA may exit.
      if (*abort_f)
        for (int i = 0; i < STAGES; ++i)
          for (uint32_t parity = 0; parity < 2; ++parity) {
            attn::drain_phase(&B->full[i], parity);
            if (!STATES) attn::drain_phase(&B->q_full[i], parity);
          }
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == COPY_WARP) {
    tc::tc_fence_after();
    tc::tmem_free_all(tmem);
  }
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------

template <int DKP, int DVP, bool STATES>
static int launch_chunk(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                        const CUtensorMap& mo, const ChunkArgs& C, int grid, void* stream) {
  using Sh = ChunkShape<DKP, DVP, STATES>;
  static_assert(Sh::SMEM <= 227 * 1024, "shared memory");
  static std::mutex mu;
  static bool done[64] = {};
  const void* fn = reinterpret_cast<const void*>(&chunk_kernel<DKP, DVP, STATES>);
  const int st = attn::allow_smem(fn, Sh::SMEM, done, mu);
  if (st != KB_OK) return st;
  return launch(chunk_kernel<DKP, DVP, STATES>, dim3((unsigned)grid), dim3(THREADS),
                (size_t)Sh::SMEM, stream, mq, mk, mv, mo, C);
}

static int64_t padded(int64_t width) { return width <= 64 ? 64 : 128; }

// Segments of a request: as many as make the longest way of a CTA shortest, in chunks.  A unit
// costs START beside its chunks, each segment's gain that it starts from GAIN; a segment but
// the last is read twice, for its gain (half a chunk's cost) and its outputs.  (One request of 32
// heads, in the segments chosen and whole: 512 tokens 21 us both, 1024 30 and 33, 2048 41 and 56,
// 8192 104 and 198; 8 heads, 8192 tokens: 50 and 195.)  One length for all requests, as if
// each were as long as the longest: a long request beside short ones is cut less or not at all (32 heads, 8192 tokens beside 300 175 us, beside four requests of
// 100 to 500 208).
static void segments_of(int64_t heads, int64_t longest, int sms, int& segments, int& segment) {
  constexpr double START = 2.0, GAIN = 0.4;
  const int64_t chunks = (longest + CHUNK - 1) / CHUNK;
  double best = 0.0;
  segments = 1;
  segment = (int)(chunks * CHUNK);
  for (int64_t n = 1; n <= chunks && n <= 64 && (n == 1 || heads * n <= 2 * sms); ++n) {
    const int64_t each = (chunks + n - 1) / n, parts = (chunks + each - 1) / each;
    const int64_t turns = (heads * parts + sms - 1) / sms;
    double cost = turns * (each + START) + GAIN * (parts - 1);
    if (parts > 1) cost += ((heads * (parts - 1) + sms - 1) / sms) * (0.5 * each + START);
    if (n > 1 && cost >= best) continue;
    best = cost;
    segments = (int)parts;
    segment = (int)(each * CHUNK);
  }
}

// Requests of several lengths on fewer CTAs than units.  (24 prompts of 1 to 2047 tokens, 24
// heads: 80 us with the units dealt out by number, 66 from a counter in this order.)
static bool by_order(int64_t B, int64_t H, int segments, int sms) {
  return segments == 1 && B > 1 && B * H > sms && B * H < ((int64_t)1 << 30);
}

// The workspace: decays, then segments' gains and decays, or the order and its counter.
struct Layout {
  int segments, segment;
  bool order;
  int64_t places;
  size_t sums, keeps, taken, bytes;
  Layout(int64_t B, int64_t H, int64_t Dk, int64_t Dv, int64_t total, int64_t longest, int sms) {
    segments_of(B * H, longest, sms, segments, segment);
    order = by_order(B, H, segments, sms);
    places = total / CHUNK + B + 1;
    sums = (size_t)(places * H) * sizeof(Decays);
    const size_t units = segments > 1 ? (size_t)(B * segments * H) : 0;
    keeps = sums + units * padded(Dk) * padded(Dv) * sizeof(float);
    taken = keeps + units * sizeof(float);
    bytes = taken + (order ? (size_t)(B + 1) * sizeof(int) : 0);
  }
};

size_t chunk_workspace(int64_t B, int64_t H, int64_t Dk, int64_t Dv, int64_t total,
                       int64_t longest, int sms) {
  return Layout(B, H, Dk, Dv, total, longest, sms).bytes;
}

int launch_chunks(const Args& A, int64_t Hq, int64_t Hk, int sms, void* workspace,
                  size_t workspace_bytes, void* stream) {
  const Layout L(A.B, A.H, A.Dk, A.Dv, A.total, A.longest, sms);
  KB_REQUIRE(workspace_bytes >= L.bytes && workspace, KB_ERR_WORKSPACE,
             "linear attention: workspace of %zu bytes, %zu needed", workspace_bytes, L.bytes);
  KB_REQUIRE(((uintptr_t)workspace & 15) == 0, KB_ERR_ALIGNMENT,
             "linear attention: the workspace must be 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  ChunkArgs C = {};
  C.a = A;
  C.segments = L.segments;
  C.segment = L.segment;
  C.decays = reinterpret_cast<Decays*>(ws);
  C.sums = reinterpret_cast<float*>(ws + L.sums);
  C.keeps = reinterpret_cast<float*>(ws + L.keeps);
  if (L.order) {
    C.taken = reinterpret_cast<int*>(ws + L.taken);
    C.order = C.taken + 1;
  }
  const int64_t warps = PREPARE_THREADS / 32, ctas = (L.places * A.H + warps - 1) / warps;
  KB_REQUIRE(ctas < ((int64_t)1 << 31) - 1, KB_ERR_UNSUPPORTED,
             "linear attention: too many tokens and heads");
  CUtensorMap mq, mk, mv, mo;
  int st = attn::make_map_4d(&mq, A.q, 0, {A.Dk, Hq, A.total, 1}, {A.q_head, A.q_tok, 8}, 1,
                             CHUNK);
  if (st == KB_OK)
    st = attn::make_map_4d(&mk, A.k, 0, {A.Dk, Hk, A.total, 1}, {A.k_head, A.k_tok, 8}, 1, CHUNK);
  if (st == KB_OK)
    st = attn::make_map_4d(&mv, A.v, 0, {A.Dv, A.H, A.total, 1}, {A.v_head, A.v_tok, 8}, 1,
                           CHUNK);
  // The outputs in boxes of 32 rows and the columns of a warp.
  if (st == KB_OK)
    st = attn::make_map_4d(&mo, A.out, 0, {A.Dv, A.H, A.total, 1},
                           {A.Dv, (int64_t)A.H * A.Dv, 8}, 1, 32, A.Dv <= 64 ? 32 : 64);
  if (st != KB_OK) return st;
  // Beside the decays: the order, or the states that segments start from.
  const int64_t more = L.order ? 1 : L.segments > 1 && A.state ? (int64_t)A.B * A.H : 0;
  st = launch(L.segments > 1 ? prepare_kernel<true> : prepare_kernel<false>,
              dim3((unsigned)(ctas + more)), dim3(PREPARE_THREADS), 0, stream, C, L.places,
              (int)(padded(A.Dk) * padded(A.Dv)));
  const int grid = (int)std::min<int64_t>((int64_t)A.B * C.segments * A.H, sms);
  for (int pass = C.segments > 1 ? 0 : 1; pass < 2 && st == KB_OK; ++pass) {
    const bool states = pass == 0;
    if (A.Dk <= 64 && A.Dv <= 64)
      st = states ? launch_chunk<64, 64, true>(mq, mk, mv, mo, C, grid, stream)
                  : launch_chunk<64, 64, false>(mq, mk, mv, mo, C, grid, stream);
    else if (A.Dk <= 64)
      st = states ? launch_chunk<64, 128, true>(mq, mk, mv, mo, C, grid, stream)
                  : launch_chunk<64, 128, false>(mq, mk, mv, mo, C, grid, stream);
    else if (A.Dv <= 64)
      st = states ? launch_chunk<128, 64, true>(mq, mk, mv, mo, C, grid, stream)
                  : launch_chunk<128, 64, false>(mq, mk, mv, mo, C, grid, stream);
    else
      st = states ? launch_chunk<128, 128, true>(mq, mk, mv, mo, C, grid, stream)
                  : launch_chunk<128, 128, false>(mq, mk, mv, mo, C, grid, stream);
  }
  return st;
}

}  // namespace linear
}  // namespace kb
