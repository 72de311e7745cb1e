// kb_prompt.cu - causal attention over packed prompts, and attention of many
// rows (drafted trees, grouped heads) over the paged cache, on the
// 5th-generation tensor cores.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / l_i,  s_ij = scale * q_i . k_j over the visible j,
//   m_i = max_j s_ij, l_i = sum_j exp(s_ij - m_i), lse_i = m_i + log(l_i)
// visible: j <= i + (Lk - Lq), or the token's tree word (kb_tree.cu).  A row that
// sees no key gives 0 and lse -infinity.
//
// One persistent CTA per SM.  A unit is 256 rows of one request, two tiles A
// and B of 128, against all the keys they see, 64 a step.  The heads of a
// group that share keys lie side by side in the rows (row = token * pack +
// head, pack the largest power of two in the group), so short prompts fill
// tiles and keys are read once for them.  Units go out heaviest (latest rows)
// first, there and back over the CTAs.
//
//   warp 10: the list of units, and copies.  It counts, 32 requests at a time,
//     which have rows that late, tells the other warps this CTA's units through
//     a ring of four, and brings in Q tiles and a ring of stages (8 KB blocks
//     of 64 rows x 64 elements), by tensor copies in the 128-byte swizzle.  A
//     stage holds the keys of step h + 2 and the values of step h: what the
//     MMAs read one after the other, under one barrier pair.
//   warps 8 and 9: issue the MMAs of tiles A and B (one warp for both spent as
//     long in its waits and commits as the tensor core in the products).
//     S = Q K^T (both from shared memory) into tensor memory, O += P V with P
//     from tensor memory (it replaces the S it came from) and V from shared
//     memory, rows of V as they lie (MN-major).  Each tile has two S buffers,
//     so S of step h + 2 is issued behind P V of step h, and the softmax finds
//     its next scores waiting.  P V of a step is issued before the S that
//     overwrites its P, by the same thread, and MMAs run in order.
//   warps 0-3 and 4-7: softmax of tiles A and B, a row per thread: maximum,
//     exponentials in base 2, row sum in fp32, and P rounded once to the
//     inputs' type.  The running maximum only moves, and O is only rescaled,
//     when a row's maximum rose by more than 2^8: weights stay within fp32
//     and the 16-bit types, and the final division makes up for the rest.
//
// 512 columns of tensor memory: two S of 64 for A and for B, O A, O B.  The
// registers of the softmax are full (200 of them): holding all of O at the end
// spills and costs a quarter more time (8192 tokens: 545 -> 696 us).
//
// Bound.  MMAs: 51 clocks each for S (128 x 64 x 16, both operands from shared
// memory: reading A sets the rate; 64 clocks at 128 x 128 x 16) and 64 for P V,
// which is 1322 clocks for a step of A and B at 128-wide heads, 1726 at 192 + 128.
// The softmax of both tiles takes 1630 to 1700 a step whatever the width: its exponentials
// (16 a clock and SM) are 768 of that by count, three in four of 16384; the rest is
// its chain of wait, load, maximum and vote.  One pair of exponentials in POLY_EVERY is computed on
// the FMA pipes (2 to 4 % at 192 + 128; every second or third pair is no better).  Taking
// the weights relative to the last step's maximum, beside the new one, is slower
// (1830).  With steps of 128 keys and one S a tile, each tile's MMAs waited for its
// softmax in turn: 3600 clocks for 128 keys at 128 wide, 4430 at 192 + 128.
// Measured: 8192 tokens x 32 heads, 192 + 128: 545 us alone (1260 TFLOP/s), 656 back
// to back under the power cap (1047; cuBLAS 1403); 24 prompts of 1 to 2047 tokens,
// 32/8 heads of 128: 139 us (736 TFLOP/s; units of few steps, 5500 clocks of start and
// end each); 5 prompts of 37 tokens over up to 2048 keys, 8/2 heads of 64: 5.9 us and
// 0.83 a step (replayed).
//
// Paged cache (PAGED).  A unit is up to 256 rows (token * group + head) of one
// request and key/value head, against the cache in 64-key steps; with few rows
// tile B is idle and the bytes of the cache bound the work.  All units' steps
// form one line cut into equal runs, one per CTA, as in kb_tree.cu; a unit that
// falls to several CTAs is joined from fp32 partial sums by the CTA that finishes
// last.  16 trees of up to 24 tokens, 4 heads a group, up to 4095 cached: 43 us; a step
// of one tile takes 1.1 us, a CTA's first scores are there after 6, and partial sums
// take 3 us, counting them 1, joining them 5.  Keys and values come page by page; q too
// by tensor copies where one tile holds a request's rows, else by gathered 16-byte copies
// into the same layout.
//
// In the last tiles of a unit some rows do not see some keys, or the tile
// reaches past the request's end into its neighbour.  A value there that is
// infinite or not a number must not meet a zero weight: warp 11 zeroes such
// elements in those tiles before the MMA reads them, and at the end the rows
// that do see them take them from memory.
#include <algorithm>
#include <type_traits>

#include "kb_runs.cuh"
#include "kb_tcgen05.cuh"

namespace kb {
namespace attn {

constexpr int TILE = 128;                  // rows of a tile
constexpr int STEP = 64;                   // keys of a step
constexpr int BLOCK = STEP * 128;          // bytes of 64 rows x 64 elements
constexpr int PROMPT_THREADS = 384;
constexpr int MMA_WARP = 8, COPY_WARP = 10, CLEAN_WARP = 11;   // MMA: and 9
constexpr int UNITS = 4;                   // units told ahead
constexpr int MAX_STAGES = 8;
constexpr int ROWS_COST = 4;               // paged: a unit's start and end, in steps
constexpr int POLY_EVERY = 4;              // one in so many pairs of exponentials on the FMA pipes
constexpr float RESCALE = 8.0f;            // log2 of the growth that moves the maximum

struct PromptArgs {
  const uint16_t *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  uint16_t* out;            // [total, Hq, Dv] contiguous
  float* lse;               // [total, Hq] or NULL
  const int *cu_q, *cu_k;
  int64_t total_q, total_k;
  int B, Hq, g, Dk, Dv;
  int pack_shift;           // log2 of the heads that share a tile's rows
  int blocks;               // 256-row units of the longest request
  float scale2;             // scale * log2(e)
  uint32_t* err;
  // Paged: k and v are the caches, k_tok and v_tok the strides of a page's rows.
  const int* table;
  int64_t table_stride;
  const int* context;
  const int64_t* mask;      // NULL: causal
  int64_t n_pages, v_page;
  int width, ps, Hkv;
  int places;               // of a table's row
  int most;                 // tokens of a request at most
  int* counters;            // [2 * CTAs], zero between calls
  int part_rows;            // rows of a unit: 128 or 256
  float* part_ml;           // [2 * CTAs][part_rows][2]: m (log2), l
  float* part_o;            // [2 * CTAs][DVP / 4][part_rows][4]
};

template <int DKP, int DVP>
struct PromptShape {
  static constexpr int KC = DKP / 64;                    // blocks of a step's keys
  static constexpr int VC = DVP / 64;                    // ... and values
  static constexpr int Q_TILE = 2 * KC * BLOCK;          // bytes of a Q tile (128 rows)
  static constexpr int STAGE = (KC + VC) * BLOCK;
  static constexpr int FIXED = 1024 + 1536;              // alignment, barriers
  static constexpr int FIT = (227 * 1024 - FIXED - 2 * Q_TILE) / STAGE;
  static constexpr int STAGES = FIT > MAX_STAGES ? MAX_STAGES : FIT;
  static constexpr int SMEM = FIXED + 2 * Q_TILE + STAGES * STAGE;
  static_assert(STAGES >= 3, "keys two steps ahead of the values");
};

// A unit as warp 10 tells it to the others.
struct Unit {
  int q0, k0;               // first query and key of the request
  int n, m;                 // its queries and keys
  int head0;                // first head
  int t0;                   // first token of tile A (paged: first row)
  int steps[2];             // steps of keys that tiles A and B see
  int whole;                // of them, those that every row of A sees whole
  int count;                // number of the unit in this CTA, -1: the end
  // Paged: the request, the run's first step of the unit, the steps this CTA had
  // before; whether the run has all steps, or the first; the CTAs that share it.
  int b, j0, base, all, starts, c0, parts;
};
constexpr int SEEN = 16;                   // steps whose key words are kept

struct PromptBars {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t clean[MAX_STAGES];   // full, and the values without odd elements
  uint64_t unit_full[UNITS], unit_empty[UNITS];
  uint64_t q_full[2], q_empty[2];
  uint64_t s_full[2][2], p_full[2][2];   // of a tile's two buffers
  uint64_t o_near[2], o_full[2];         // P V of the unit's last step but one, last step
  uint64_t drain;
  Unit unit[UNITS];
  int odd[16];              // units that had odd elements, by their number's last four bits
  uint64_t valid[SEEN];     // paged: which keys of a step exist, by the CTA's count of steps
  uint64_t meet[2];         // paged: a tile's softmax warps together
  int joined[2];
  RunStart start;
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(PromptBars) <= 1536, "barrier block");

// A warp's way through the CTA's units.
struct Walk {
  PromptBars* B;
  uint32_t* err;
  int slot;
  uint32_t phase;
  __device__ __forceinline__ Walk(PromptBars* b, uint32_t* e) : B(b), err(e), slot(0), phase(0) {}
  // The next unit; false at the end or on abort.
  __device__ __forceinline__ bool next(Unit& U) {
    if (!warp_wait(&B->unit_full[slot], phase, &B->abort_flag, err)) return false;
    U = B->unit[slot];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&B->unit_empty[slot]);
    if (++slot == UNITS) {
      slot = 0;
      phase ^= 1u;
    }
    return U.count >= 0;
  }
};
constexpr int WALKERS = 8 + 3;               // softmax warps, two of MMAs, cleaning

// 2^x for a pair of x <= 64 on the FMA pipes: x = n + f with n the nearest
// whole number (left in the low bits of x + 1.5 * 2^23) and |f| <= 1/2, 2^f by a
// polynomial of degree 4 fitted here to least relative error (2.7e-6, and
// 4e-8 on average, far below the rounding of the weights), n added to the exponent.  Below
// 2^-126, at -infinity and for what is no number the result is 2^-126.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  const float2 big = make_float2(12582912.f, 12582912.f);
  const float2 nbig = make_float2(-12582912.f, -12582912.f);
  x.x = fmaxf(x.x, -126.f);
  x.y = fmaxf(x.y, -126.f);
  const float2 t = fadd2(x, big);
  const float2 n = fadd2(t, nbig);
  const float2 f = ffma2(n, make_float2(-1.f, -1.f), x);
  float2 p = make_float2(0.00957010221f, 0.00957010221f);
  p = ffma2(p, f, make_float2(0.0559178591f, 0.0559178591f));
  p = ffma2(p, f, make_float2(0.240247443f, 0.240247443f));
  p = ffma2(p, f, make_float2(0.693121791f, 0.693121791f));
  p = ffma2(p, f, make_float2(0.999999285f, 0.999999285f));
  return make_float2(__int_as_float((__float_as_int(t.x) << 23) + __float_as_int(p.x)),
                     __int_as_float((__float_as_int(t.y) << 23) + __float_as_int(p.y)));
}

// Adds to a row's outputs d0..d0+31 the values that are no numbers of the keys
// [first, last]: they were kept out of the tile products.
template <bool F16>
__device__ __forceinline__ void add_odd(const PromptArgs& A, const uint16_t* v, int d0,
                                        float (&o)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint16_t u = d0 + i < A.Dv ? v[d0 + i] : 0;
    if (odd_element<F16>(u)) o[i] += element<F16>(u);
  }
}

// Which of 64 keys from `key` on a row sees: those up to `limit`, or (word) the
// context and the tree's bits.
__device__ __forceinline__ uint64_t low_bits(int n) {
  return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull;
}
__device__ __forceinline__ uint64_t tree_bits(uint64_t word, int ctx, int key) {
  const int d = ctx - key;
  return d >= 64 ? ~0ull : d >= 0 ? low_bits(d) | (word << d) : d > -64 ? word >> -d : 0ull;
}

// Half of a transposition: lanes `step` apart keep one piece and swap the other.
__device__ __forceinline__ void swap_pieces(uint4& a, uint4& b, int upper, int step) {
  uint4 give = upper ? a : b;
  give.x = __shfl_xor_sync(0xffffffffu, give.x, step);
  give.y = __shfl_xor_sync(0xffffffffu, give.y, step);
  give.z = __shfl_xor_sync(0xffffffffu, give.z, step);
  give.w = __shfl_xor_sync(0xffffffffu, give.w, step);
  if (upper) a = give; else b = give;
}

// A row whose keys several CTAs had: their sums joined, 64 columns at a time.
template <int DVP, bool F16>
__device__ __forceinline__ void join_parts(const PromptArgs& A, const Unit& U, int row,
                                           int64_t at) {
  auto slot = [&](int c) { return (int64_t)(U.c0 + c) * 2 + (c == 0); };
  float top = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int c = 0; c < U.parts; ++c) {
    const float2 ml =
        __ldcg(reinterpret_cast<const float2*>(A.part_ml + (slot(c) * A.part_rows + row) * 2));
    const float t = fmaxf(top, ml.x);
    sum = sum * part_factor(top, t) + ml.y * part_factor(ml.x, t);
    top = t;
  }
  const bool none = sum == 0.f;
  const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
  for (int d = 0; d < DVP; d += 64) {
    float o[64] = {};
    for (int c = 0; c < U.parts && !none; ++c) {
      const float m = __ldcg(A.part_ml + (slot(c) * A.part_rows + row) * 2);
      float4 v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k)
        v[k] = __ldcg(reinterpret_cast<const float4*>(
            A.part_o + ((slot(c) * (DVP / 4) + d / 4 + k) * A.part_rows + row) * 4));
      // A part that counts nothing still hands on values that are no numbers, as a
      // weight of zero does in a tile.
      const float f = part_factor(m, top) * inv;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        o[4 * k] += v[k].x * f;
        o[4 * k + 1] += v[k].y * f;
        o[4 * k + 2] += v[k].z * f;
        o[4 * k + 3] += v[k].w * f;
      }
    }
#pragma unroll
    for (int k = 0; k < 64; k += 8)
      if (d + k < A.Dv) {
        uint4 w;
        w.x = pack2<F16>(o[k], o[k + 1]);
        w.y = pack2<F16>(o[k + 2], o[k + 3]);
        w.z = pack2<F16>(o[k + 4], o[k + 5]);
        w.w = pack2<F16>(o[k + 6], o[k + 7]);
        *reinterpret_cast<uint4*>(A.out + at * A.Dv + d + k) = w;
      }
  }
  if (A.lse) A.lse[at] = none ? -INFINITY : (top + log2f(sum)) * LN2;
}

// The copies of a CTA whose tile B is idle: four of its warps bring in 16 rows of every
// step each, in boxes of 16 rows (8 in pages of 8) x 64 elements.  A copy takes the
// warp that issues it 100 to 190 clocks whatever its size, so one warp needs 1600
// to 3150 a step where the softmax takes 1500; 16-byte copies by these four warps
// get in the way of the softmax (2300 a step).
template <int KC, int VC, int STAGES>
__device__ __forceinline__ void copy_quarter(const CUtensorMap& tk, const CUtensorMap& tv,
                                             const PromptArgs& A, PromptBars* B, uint8_t* ring,
                                             int quarter) {
  constexpr int STAGE = (KC + VC) * BLOCK;
  const uint64_t once = l2_evict_first_policy();
  const uint32_t one = tc::elect_one();
  const int lane = threadIdx.x & 31, shift = 31 - __clz(A.ps);
  const int box = min(A.ps, 16), boxes = 16 / box;
  const int r0 = uniform(quarter) * 16;
  int st = 0;
  uint32_t ph = 1;
  bool ok = true;
  Unit U;
  for (Walk walk(B, A.err); ok && walk.next(U);) {
    const int steps = uniform(U.steps[0]), hk = uniform(U.head0 / A.g), j0 = uniform(U.j0);
    // Page of the step's rows r0 (lane 0) and r0 + 8 (lane 1); -1: none.
    auto page_of = [&](int step) {
      const int key = (j0 + step) * STEP + r0 + (lane & 1) * 8, e = key >> shift;
      if (step >= steps || key >= U.m || e >= A.width) return -1;
      const int id = __ldg(A.table + (int64_t)U.b * A.table_stride + e);
      return id < A.n_pages ? id : -1;
    };
    int ids[4] = {-1, -1, page_of(0), -1};     // steps j, j + 1, j + 2, j + 3
    for (int j = -2; j < steps; ++j) {
      ids[3] = page_of(j + 3);                 // in time for the next round
      ok = warp_wait(&B->empty[st], ph, &B->abort_flag, A.err);
      if (!ok) break;
      uint8_t* at = ring + st * STAGE + r0 * 128;
      const int k_row = (j0 + j + 2) * STEP + r0, v_row = (j0 + j) * STEP + r0;
      int k_page[2], v_page[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        k_page[i] = i < boxes ? uniform_of(ids[2], i) : -1;
        v_page[i] = i < boxes ? uniform_of(ids[0], i) : -1;
      }
      const int copies = KC * ((k_page[0] >= 0) + (k_page[1] >= 0)) +
                         VC * ((v_page[0] >= 0) + (v_page[1] >= 0));
      if (lane == 0) mbar_arrive_expect_tx(&B->full[st], (uint32_t)(copies * box * 128));
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i >= boxes) break;
        const uint32_t k_one = k_page[i] >= 0 ? one : 0, v_one = v_page[i] >= 0 ? one : 0;
#pragma unroll
        for (int c = 0; c < KC; ++c)
          tma_load_4d_one(k_one, at + c * BLOCK + i * 1024, &tk, c * 64,
                          (k_row + i * 8) & (A.ps - 1), hk, k_page[i], &B->full[st], once);
#pragma unroll
        for (int c = 0; c < VC; ++c)
          tma_load_4d_one(v_one, at + (KC + c) * BLOCK + i * 1024, &tv, c * 64,
                          (v_row + i * 8) & (A.ps - 1), hk, v_page[i], &B->full[st], once);
      }
      ids[0] = ids[1];
      ids[1] = ids[2];
      ids[2] = ids[3];
      if (++st == STAGES) {
        st = 0;
        ph ^= 1u;
      }
    }
  }
}

// Largest score of a row's step; not a number where a score is none.
__device__ __forceinline__ float row_max(const float (&s)[2][32]) {
  float m[4] = {s[0][0], s[0][1], s[1][0], s[1][1]};
#pragma unroll
  for (int i = 2; i < 30; i += 4)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      m[c] = max3_nan(m[c], s[c >> 1][i + (c & 1) * 2], s[c >> 1][i + (c & 1) * 2 + 1]);
  m[0] = max3_nan(m[0], s[0][30], s[0][31]);
  m[2] = max3_nan(m[2], s[1][30], s[1][31]);
  return max_nan(max3_nan(m[0], m[1], m[2]), m[3]);
}

template <int DKP, int DVP, bool F16, bool PAGED>
__global__ void __launch_bounds__(PROMPT_THREADS, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                  const __grid_constant__ CUtensorMap tv, const PromptArgs A) {
  using S = PromptShape<DKP, DVP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      smem_raw + ((1024u - (static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw)) & 1023u)) &
                  1023u);
  uint8_t* qs = smem;                           // [2] tiles
  uint8_t* ring = qs + 2 * S::Q_TILE;           // [STAGES] keys, values
  PromptBars* B = reinterpret_cast<PromptBars*>(ring + S::STAGES * S::STAGE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_f = &B->abort_flag;
  // No request has rows for tile B: its warps bring in keys and values.
  const bool solo = PAGED && A.part_rows == TILE;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&B->full[i], solo ? 5 : 1);
      mbar_init(&B->empty[i], 2);
      mbar_init(&B->clean[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B->q_full[i], PAGED && !solo ? 32 : 1);
      mbar_init(&B->meet[i], 4);
      mbar_init(&B->q_empty[i], 1);
      mbar_init(&B->o_near[i], 1);
      mbar_init(&B->o_full[i], 1);
      for (int j = 0; j < 2; ++j) {
        mbar_init(&B->s_full[i][j], 1);
        mbar_init(&B->p_full[i][j], 4);
      }
    }
    for (int i = 0; i < UNITS; ++i) {
      mbar_init(&B->unit_full[i], 1);
      mbar_init(&B->unit_empty[i], WALKERS);
    }
    for (int i = 0; i < 16; ++i) B->odd[i] = -1;
    mbar_init(&B->drain, 2);
    B->abort_flag = 0;
    mbar_fence_init();
    if (!PAGED || solo) prefetch_map(&tq);
    prefetch_map(&tk);
    prefetch_map(&tv);
  }
  if (warp == CLEAN_WARP) tc::tmem_alloc_all(&B->tmem);
  // Columns of q past the head's width stay zero (gathered rows do not write them).
  if (PAGED && !solo && A.Dk < DKP) {
    for (int i = threadIdx.x; i < 2 * S::Q_TILE / 16; i += PROMPT_THREADS)
      reinterpret_cast<uint4*>(qs)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = B->tmem;
  pdl_wait();
  pdl_launch_dependents();
  const Lengths L = {A.cu_q, A.context, A.total_q, A.places, A.g,
                     A.Hkv, 2 * TILE, A.most, ROWS_COST};
  Run run = {};
  if (PAGED) run = find_run<PROMPT_THREADS>(L, A.B, &B->start, A.err);

  // Rows outside every request: zero.
  {
    const int64_t lead = min(max((int64_t)A.cu_q[0], (int64_t)0), A.total_q);
    const int64_t tail = min(max((int64_t)A.cu_q[A.B], lead), A.total_q);
    const int64_t spare = (lead + A.total_q - tail) * A.Hq;
    for (int64_t i = (int64_t)blockIdx.x * PROMPT_THREADS + threadIdx.x; i < spare;
         i += (int64_t)gridDim.x * PROMPT_THREADS) {
      const int64_t r = i < lead * A.Hq ? i : i - lead * A.Hq + tail * A.Hq;
      for (int d = 0; d < A.Dv; d += 8)
        *reinterpret_cast<uint4*>(A.out + r * A.Dv + d) = make_uint4(0, 0, 0, 0);
      if (A.lse) A.lse[r] = -INFINITY;
    }
  }

  if (warp < 8) {
    // ------------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int tile = warp >> 2;
    const int row = threadIdx.x & (TILE - 1);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + tile * 2 * STEP;
    const uint32_t o_at = tmem + lanes + 256 + tile * TILE;
    const float scale2 = A.scale2;
    const int span = TILE >> A.pack_shift;
    int buf = 0;                          // the next step's S buffer
    uint32_t s_phase = 0, near_phase = 0, end_phase = 0, meet_phase = 0;
    Unit U;
    const bool copies = solo && tile == 1;
    if (copies) copy_quarter<S::KC, S::VC, S::STAGES>(tk, tv, A, B, ring, warp & 3);
    for (Walk walk(B, A.err); !copies && walk.next(U);) {
      // The row's token and head; keys are limited by `limit`, or in a tree by `word`.
      const int at_row = U.t0 + tile * TILE + row;          // paged
      const int first = PAGED ? (U.t0 + tile * TILE) / A.g : U.t0 + tile * span;
      if (first >= U.n) continue;
      const int tok = PAGED ? at_row / A.g : first + (row >> A.pack_shift);
      const int head = U.head0 + (PAGED ? at_row - tok * A.g
                                        : (row & ((1 << A.pack_shift) - 1)));
      const bool real = tok < U.n;
      const int limit = min(tok, U.n - 1) + U.m - U.n;      // last key the row sees
      const bool tree = PAGED && A.mask != nullptr;
      const uint64_t word = tree ? (uint64_t)A.mask[U.q0 + min(tok, U.n - 1)] : 0;
      // Steps up to this key are seen whole by every row of the tile.
      const int clear = tree ? U.m - U.n - 1 : first + U.m - U.n;
      const int j0 = PAGED ? U.j0 : 0;
      float top = -INFINITY, sum = 0.f;                     // in log2 units
      bool ok = true;
      const int steps = U.steps[tile];
      for (int j = 0; j < steps; ++j) {
        if (!warp_wait(&B->s_full[tile][buf], s_phase, abort_f, A.err)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const uint32_t here = s_at + buf * STEP;
        float s[2][32];
        tc::tmem_ld32(here, s[0]);
        tc::tmem_ld32(here + 32, s[1]);
        tc::tmem_ld_wait();
        tc::hold_regs(s[0]);
        tc::hold_regs(s[1]);
        const int key = (j0 + j) * STEP;
        uint64_t there = ~0ull;                            // keys that exist
        if (PAGED) there = *const_cast<volatile uint64_t*>(&B->valid[(U.base + j) & (SEEN - 1)]);
        const bool edge = key + STEP - 1 > clear || there != ~0ull;   // not seen by all rows
        if (edge) {
          const uint64_t seen =
              there & (tree ? tree_bits(word, U.m - U.n, key) : low_bits(limit - key + 1));
          const uint32_t half[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((half[c] >> i) & 1)) s[c][i] = -INFINITY;
        }
        const float mine = row_max(s) * scale2;
        // A score that is no number or infinite (also only once scaled) makes the row no
        // number, whatever the polynomial makes of its weight.
        if (!(mine < INFINITY)) sum = NAN;
        if (j == 0) {
          top = mine;
        } else if (__any_sync(0xffffffffu, mine > top + RESCALE)) {
          // O may be touched once P V of the last step is done: the next step's
          // S was issued behind it.
          if (!(j + 1 < steps ? warp_wait(&B->s_full[tile][buf ^ 1], s_phase ^ (uint32_t)buf,
                                          abort_f, A.err)
                              : warp_wait(&B->o_near[tile], near_phase, abort_f, A.err))) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const float now = mine > top + RESCALE ? mine : top;
          const float fix = now == top ? 1.f : exp2_fast(top - now);
          sum *= fix;
          top = now;
          // 16 columns at a time: the scores stay in registers beside them.
#pragma unroll 1
          for (int c = 0; c < DVP / 16; ++c) {
            uint32_t o[16];
            tc::tmem_ld16(o_at + c * 16, o);
            tc::tmem_ld_wait();
            tc::hold_regs(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
            tc::tmem_st16(o_at + c * 16, o);
          }
          tc::tmem_st_wait();
        }
        const float at = top == -INFINITY ? 0.f : top;
        const float2 mul = make_float2(scale2, scale2), off = make_float2(-at, -at);
        float2 part[4] = {};
        // A masked key's weight has to be zero, which the polynomial's is not.
        auto weights = [&](auto every) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float2 x = make_float2(s[c][2 * i], s[c][2 * i + 1]);
              x = ffma2(x, mul, off);
              if (i % decltype(every)::value + 1 == decltype(every)::value) {
                x = exp2_poly(x);
              } else {
                x.x = exp2_fast(x.x);
                x.y = exp2_fast(x.y);
              }
              part[i & 3] = fadd2(part[i & 3], x);
              p[i] = pack2<F16>(x.x, x.y);
            }
            tc::tmem_st16(here + c * 16, p);
          }
        };
        if (edge)
          weights(std::integral_constant<int, 64>{});   // none
        else
          weights(std::integral_constant<int, POLY_EVERY>{});
        tc::tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->p_full[tile][buf]);
        part[0] = fadd2(fadd2(part[0], part[1]), fadd2(part[2], part[3]));
        sum += part[0].x + part[0].y;
        if (buf) s_phase ^= 1u;
        buf ^= 1;
      }
      if (!ok) break;
      const int64_t at = (int64_t)(U.q0 + tok) * A.Hq + head;
      // The four rows whose pieces this lane stores: four lanes side by side
      // exchange 16-byte pieces, so a store covers 64 bytes of eight rows and not
      // 16 bytes of 32.
      const bool whole = !PAGED || U.all;
      uint16_t* out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (row & ~3) + i, paged_row = U.t0 + tile * TILE + r;
        const int t = PAGED ? paged_row / A.g : first + (r >> A.pack_shift);
        const int h = U.head0 + (PAGED ? paged_row - t * A.g : (r & ((1 << A.pack_shift) - 1)));
        out[i] = t < U.n ? A.out + ((int64_t)(U.q0 + t) * A.Hq + h) * A.Dv + (lane & 3) * 8
                         : nullptr;
      }
      const int64_t part_slot = (int64_t)blockIdx.x * 2 + U.starts;
      if (steps > 1) near_phase ^= 1u;
      bool odd = false;
      if (steps > 0) {
        if (!warp_wait(&B->o_full[tile], end_phase, abort_f, A.err)) break;
        end_phase ^= 1u;
        tc::tc_fence_after();
        odd = *const_cast<volatile int*>(&B->odd[U.count & 15]) == U.count;
      }
      // A row that saw no key (or only keys of score -infinity, to which the polynomial
      // gives its least weight) is zero.
      if (top == -INFINITY && sum == sum) sum = 0.f;
      const bool none = sum == 0.f || (!PAGED && limit < 0);
      const float inv = !whole ? 1.f : none ? 0.f : 1.f / sum;
#pragma unroll
      for (int c = 0; c < DVP / 32; ++c) {
        float o[32];
        if (steps > 0) {
          tc::tmem_ld32(o_at + c * 32, o);
          tc::tmem_ld_wait();
          tc::hold_regs(o);
          if (odd) {
            if (PAGED) {
              for (int key = j0 * STEP; key < min((j0 + steps) * STEP, U.m); ++key) {
                const int e = key / A.ps;
                const int id = e < A.width ? A.table[(int64_t)U.b * A.table_stride + e] : -1;
                const bool sees = tree ? (tree_bits(word, U.m - U.n, key) & 1) != 0 : key <= limit;
                if (id >= 0 && id < A.n_pages && sees)
                  add_odd<F16>(A, A.v + id * A.v_page + (key - e * A.ps) * A.v_tok +
                                      U.head0 / A.g * A.v_head, c * 32, o);
              }
            } else {
              for (int key = U.whole * STEP; key <= limit; ++key)
                add_odd<F16>(A, A.v + (U.k0 + (int64_t)key) * A.v_tok + head / A.g * A.v_head,
                             c * 32, o);
            }
          }
        }
        if (!whole) {
          // This CTA's share of the sums, columns by fours: a warp stores 512 bytes.
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            if (real)
              *reinterpret_cast<float4*>(A.part_o + ((part_slot * (DVP / 4) + c * 8 + i / 4) *
                                                     A.part_rows + tile * TILE + row) * 4) =
                  make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          continue;
        }
        uint4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i].x = pack2<F16>(o[8 * i] * inv, o[8 * i + 1] * inv);
          w[i].y = pack2<F16>(o[8 * i + 2] * inv, o[8 * i + 3] * inv);
          w[i].z = pack2<F16>(o[8 * i + 4] * inv, o[8 * i + 5] * inv);
          w[i].w = pack2<F16>(o[8 * i + 6] * inv, o[8 * i + 7] * inv);
          if (none) w[i] = make_uint4(0, 0, 0, 0);
        }
        swap_pieces(w[0], w[1], lane & 1, 1);
        swap_pieces(w[2], w[3], lane & 1, 1);
        swap_pieces(w[0], w[2], lane & 2, 2);
        swap_pieces(w[1], w[3], lane & 2, 2);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (out[i] && c * 32 + (lane & 3) * 8 < A.Dv)
            *reinterpret_cast<uint4*>(out[i] + c * 32) = w[i];
      }
      tc::tc_fence_before();
      if (whole) {
        if (real && A.lse) A.lse[at] = none ? -INFINITY : (top + log2f(sum)) * LN2;
        __syncwarp();
        continue;
      }
      if (real)
        *reinterpret_cast<float2*>(A.part_ml + (part_slot * A.part_rows + tile * TILE + row) * 2) =
            make_float2(top, sum);
      // The last of the unit's CTAs joins the tile's sums, in CTA order.
      auto meet = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->meet[tile]);
        ok = warp_wait(&B->meet[tile], meet_phase, abort_f, A.err);
        meet_phase ^= 1u;
        return ok;
      };
      __threadfence();
      if (!meet()) break;
      if (row == 0) {
        int* counter = A.counters + U.c0 * 2 + tile;
        const int old = atomicAdd(counter, 1);
        B->joined[tile] = old == U.parts - 1;
        if (old == U.parts - 1) *counter = 0;
      }
      if (!meet()) break;
      if (*const_cast<volatile int*>(&B->joined[tile])) {
        __threadfence();
        if (real) join_parts<DVP, F16>(A, U, tile * TILE + row, at);
      }
      if (!meet()) break;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp < COPY_WARP) {
      // --------------------------------------------------------------- MMA issue
      constexpr uint32_t TYPE = F16 ? 0u : 1u;
      constexpr uint32_t COMMON = (1u << 4) | (TYPE << 7) | (TYPE << 10) | ((TILE >> 4) << 24);
      constexpr uint32_t ID_S = COMMON | ((STEP >> 3) << 17);
      constexpr uint32_t ID_O = COMMON | (1u << 16) | ((DVP >> 3) << 17);    // V: MN-major
      // The warp goes through this in step (what it reads from memory is made
      // uniform for the compiler), one lane issues.
      const uint32_t one = tc::elect_one();
      const int tile = __shfl_sync(0xffffffffu, warp - MMA_WARP, 0);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t q_at = smem_addr(qs) + tile * S::Q_TILE, r_at = smem_addr(ring);
      const uint32_t s_to = tm + tile * 2 * STEP, o_to = tm + 256 + tile * TILE;
      int st = 0;                         // stage of the next keys and values
      uint32_t ph = 0, q_phase = 0, p_phase = 0;
      int s_buf = 0, p_buf = 0;           // S buffers of the next scores and weights
      bool ok = true;
      auto need = [&](uint64_t* bar, uint32_t ph) {
        ok = warp_wait(bar, ph, abort_f, A.err);
        return ok;
      };
      // S of the tile's next step, from the keys of the stage.
      auto score = [&]() {
        const uint32_t d = s_to + s_buf * STEP;
        uint32_t acc = 0;
#pragma unroll
        for (int c = 0; c < S::KC; ++c) {
          const uint64_t a = tc::sw128_desc(q_at + c * 2 * BLOCK);
          const uint64_t b = tc::sw128_desc(r_at + st * S::STAGE + c * BLOCK);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            tc::umma_one(one, d, a + k * 2, b + k * 2, ID_S, acc);
            acc = 1;
          }
        }
        tc::umma_commit_one(one, &B->s_full[tile][s_buf]);
        s_buf ^= 1;
      };
      // O += P V of its next step, with the values of the stage.
      auto product = [&](bool first) {
        const uint32_t p = s_to + p_buf * STEP;
        const uint64_t b = tc::sw128_desc_mn(r_at + st * S::STAGE + S::KC * BLOCK, BLOCK);
        uint32_t acc = first ? 0 : 1;
#pragma unroll
        for (int k = 0; k < STEP / 16; ++k) {
          tc::umma_ts_one(one, o_to, p + k * 8, b + k * (2048 >> 4), ID_O, acc);
          acc = 1;
        }
      };
      Unit U;
      for (Walk walk(B, A.err); ok && walk.next(U);) {
        const int mine = __shfl_sync(0xffffffffu, U.steps[tile], 0);
        const int all = __shfl_sync(0xffffffffu, max(U.steps[0], U.steps[1]), 0);
        // Products of step j and scores of step j + 2.  A stage that only the other
        // tile uses is waited for too and passed on: both warps stay within one round
        // of the ring.
        for (int j = -2; j < all && all > 0; ++j) {
          if (!need(&B->clean[st], ph)) break;
          if (j >= 0 && j < mine) {
            if (!need(&B->p_full[tile][p_buf], p_phase)) break;
            tc::tc_fence_after();
            product(j == 0);
            p_phase ^= (uint32_t)p_buf;
            p_buf ^= 1;
            if (j + 2 == mine) tc::umma_commit_one(one, &B->o_near[tile]);
            if (j + 1 == mine) tc::umma_commit_one(one, &B->o_full[tile]);
          }
          if (j + 2 < mine) {
            if (j == -2) {
              if (!need(&B->q_full[tile], q_phase)) break;
              q_phase ^= 1u;
              if (PAGED && !solo) fence_proxy_async();      // q came by ordinary copies
            }
            tc::tc_fence_after();
            score();
            if (j + 3 == mine) tc::umma_commit_one(one, &B->q_empty[tile]);
          }
          tc::umma_commit_one(one, &B->empty[st]);
          if (++st == S::STAGES) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
      // Every product issued is done before the tensor memory goes.
      tc::umma_commit_one(one, &B->drain);
      drain_phase(&B->drain, 0);
    } else if (warp == COPY_WARP) {
      // -------------------------------------------------- list of units, and copies
      const uint64_t keep = l2_evict_last_policy(), once = l2_evict_first_policy();
      const int groups = A.Hq >> A.pack_shift, span = TILE >> A.pack_shift;
      int slot = 0, round = 0, count = 0, held = -1;
      uint32_t told = 1;
      int want = blockIdx.x, before = 0;     // this CTA's next unit on the list; units before here
      int64_t first = 0, end = 0;
      int st = 0;                            // stage of the next step
      uint32_t ph = 1, q_phase[2] = {1, 1};
      bool ok = true;
      auto need = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && warp_wait(bar, parity, abort_f, A.err);
        return ok;
      };
      auto tell = [&](const Unit& U) {
        if (!need(&B->unit_empty[slot], told)) return;
        if (lane == 0) {
          B->unit[slot] = U;
          mbar_arrive(&B->unit_full[slot]);
        }
        if (++slot == UNITS) {
          slot = 0;
          told ^= 1u;
        }
      };
      // Copies are issued by the warp in step, one lane doing it.
      const uint32_t one = tc::elect_one();
      const int box = min(A.ps, STEP), pages = STEP / max(box, 1);      // paged
      int ids = -1, have = -1, id_k = -1, id_w = -1, id_v = -1;
      auto copy = [&](const Unit& U) {
        const int steps = uniform(max(U.steps[0], U.steps[1]));
        const int hk = uniform(U.head0 / A.g), key0 = uniform(U.k0), j0 = uniform(U.j0);
        have = -1;
        auto queries = [&](int i) {
          if (U.steps[i] == 0 || !need(&B->q_empty[i], q_phase[i])) return;
          q_phase[i] ^= 1u;
          if (PAGED && !solo) {
            const int pieces = A.Dk / 8, rows = min(TILE, U.n * A.g - U.t0 - i * TILE);
            for (int x = lane; x < rows * pieces; x += 32) {
              const int r = x / pieces, c = x - r * pieces, at = U.t0 + i * TILE + r;
              const int t = at / A.g;
              cp_async16(qs + i * S::Q_TILE + (c >> 3) * 2 * BLOCK + r * 128 +
                             (((c ^ r) & 7) << 4),
                         A.q + (U.q0 + (int64_t)t) * A.q_tok +
                             (U.head0 + (int64_t)(at - t * A.g)) * A.q_head + c * 8);
            }
            cp_async_arrive_noinc(&B->q_full[i]);
            return;
          }
          if (lane != 0) return;
          // Paged: the group's heads of as many tokens as a tile has room for.
          const int rows = PAGED ? TILE / A.g * A.g : TILE;
          mbar_arrive_expect_tx(&B->q_full[i], (uint32_t)(S::KC * 128 * rows));
          for (int c = 0; c < S::KC; ++c)
            tma_load_4d(qs + i * S::Q_TILE + c * 2 * BLOCK, &tq, c * 64, U.head0,
                        PAGED ? U.q0 : U.q0 + U.t0 + i * span, 0, &B->q_full[i], once);
        };
        for (int j = -2; j < steps && steps > 0; ++j) {
          if (j == -2) queries(0);
          if (!need(&B->empty[st], ph)) break;
          const bool keys = j + 2 < steps, values = j >= 0;
          uint8_t* at = ring + st * S::STAGE;
          if (PAGED) {
            // Pages of the keys; those of the values are the keys' of two steps ago.
            id_v = id_w;
            id_w = id_k;
            id_k = -1;
            const int k_row = (j0 + j + 2) * STEP, v_row = (j0 + j) * STEP;
            if (keys) {
              id_k = page_ids(A, U.b, U.m, k_row, ids, have);
              uint64_t there = low_bits(U.m - k_row);
              const unsigned live = __ballot_sync(0xffffffffu, lane < pages && id_k >= 0);
              if (live != (1u << pages) - 1u) {
                uint64_t got = 0;
                for (int i = 0; i < pages; ++i)
                  if ((live >> i) & 1) got |= low_bits(box) << (i * box);
                if (lane == 0 && (there & ~got)) atomicOr(A.err, ERR_PAGE);
                there &= got;
              }
              if (lane == 0) B->valid[(U.base + j + 2) & (SEEN - 1)] = there;
            }
            if (solo) {
              // Warps 4-7 bring the rows in; this adds the word.
              __syncwarp();
              if (lane == 0) mbar_arrive(&B->full[st]);
            } else {
              const unsigned in = __ballot_sync(0xffffffffu, lane < pages && id_k >= 0);
              const unsigned out = __ballot_sync(0xffffffffu, values && lane < pages && id_v >= 0);
              if (lane == 0)
                mbar_arrive_expect_tx(&B->full[st], (uint32_t)((__popc(in) * S::KC +
                                                                __popc(out) * S::VC) * box * 128));
              __syncwarp();
              // A copy per page and 64-element column block, a lane each.
              for (int x0 = 0; x0 < pages * (S::KC + S::VC); x0 += 32) {
                const int x = x0 + lane;
                const int i = min(x / (S::KC + S::VC), pages - 1), c = x - i * (S::KC + S::VC);
                const int k_page = __shfl_sync(0xffffffffu, id_k, i);
                const int v_page = __shfl_sync(0xffffffffu, id_v, i);
                if (x >= pages * (S::KC + S::VC)) continue;
                const int row = i * box;
                if (c < S::KC) {
                  if ((in >> i) & 1)
                    tma_load_4d(at + c * BLOCK + row * 128, &tk, c * 64,
                                (k_row + row) & (A.ps - 1), hk, k_page, &B->full[st], once);
                } else if ((out >> i) & 1) {
                  tma_load_4d(at + c * BLOCK + row * 128, &tv, (c - S::KC) * 64,
                              (v_row + row) & (A.ps - 1), hk, v_page, &B->full[st], once);
                }
              }
              __syncwarp();
            }
          } else {
            if (lane == 0)
              mbar_arrive_expect_tx(&B->full[st], (uint32_t)(((keys ? S::KC : 0) +
                                                              (values ? S::VC : 0)) * BLOCK));
            __syncwarp();
            const uint32_t k_one = keys ? one : 0, v_one = values ? one : 0;
#pragma unroll
            for (int c = 0; c < S::KC; ++c)
              tma_load_4d_one(k_one, at + c * BLOCK, &tk, c * 64, hk, key0 + (j + 2) * STEP, 0,
                              &B->full[st], keep);
#pragma unroll
            for (int d = 0; d < S::VC; ++d)
              tma_load_4d_one(v_one, at + (S::KC + d) * BLOCK, &tv, d * 64, hk, key0 + j * STEP, 0,
                              &B->full[st], keep);
          }
          if (++st == S::STAGES) {
            st = 0;
            ph ^= 1u;
          }
          if (j == -2) queries(1);
        }
      };
      if (PAGED && run.lo < run.hi) {
        // This CTA's run of the line of steps.
        int64_t pos = run.lo, line = B->start.base;
        Request R = B->start.r;
        int b = B->start.b, base = 0;
        while (pos < run.hi && ok) {
          const int64_t w = L.length(R);
          if (pos >= line + w) {
            line += w;
            R = L.look(++b);
            continue;
          }
          const RunPart P = run_part(R, pos, line, run, ROWS_COST);
          pos = P.until;
          if (P.t1 <= P.t0) continue;          // the run ends in the unit's start
          Unit U = {};
          U.q0 = (int)R.first;
          U.n = R.n;
          U.m = (int)(R.ctx + R.n);
          U.head0 = P.hk * A.g;
          U.t0 = P.block * 2 * TILE;
          const int rows = R.n * A.g - U.t0;
          U.steps[0] = (int)(P.t1 - P.t0);
          U.steps[1] = rows > TILE ? U.steps[0] : 0;
          U.whole = max((int)(R.ctx / STEP - P.t0), 0);
          U.count = count++;
          U.b = b;
          U.j0 = (int)P.t0;
          U.base = base;
          U.all = P.t0 == 0 && P.t1 == R.tiles;
          U.starts = P.t0 == 0;
          U.c0 = P.c0;
          U.parts = P.parts;
          base += U.steps[0];
          tell(U);
          if (ok) copy(U);
        }
      }
      for (int block = A.blocks - 1; !PAGED && block >= 0 && ok; --block) {
        const int t0 = (block * 2 * TILE) >> A.pack_shift;
        for (int b0 = 0; b0 < A.B && ok; b0 += 32) {
          if (held != b0) {
            held = b0;
            first = end = 0;
            if (b0 + lane < A.B) request_rows(A.cu_q, b0 + lane, A.total_q, first, end);
          }
          const unsigned late = __ballot_sync(0xffffffffu, end - first > t0);
          const int limit = before + __popc(late) * groups;
          while (ok && want < limit) {
            const int at = (want - before) / groups;
            const int from = __fns(late, 0, at + 1);
            Unit U;
            U.q0 = __shfl_sync(0xffffffffu, (int)first, from);
            U.n = __shfl_sync(0xffffffffu, (int)(end - first), from);
            int64_t k0, k1;
            request_rows(A.cu_k, b0 + from, A.total_k, k0, k1);
            U.k0 = (int)k0;
            U.m = (int)(k1 - k0);
            U.head0 = (want - before - at * groups) << A.pack_shift;
            U.t0 = t0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int top = t0 + i * span, last = min(U.n, top + span) - 1;
              const int keys = top < U.n ? min(max(last + U.m - U.n + 1, 0), U.m) : 0;
              U.steps[i] = (keys + STEP - 1) / STEP;
            }
            U.whole = max(t0 + U.m - U.n + 1, 0) / STEP;
            U.count = count++;
            tell(U);
            if (ok) copy(U);
            ++round;
            want = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
          }
          before = limit;
        }
      }
      Unit last = {};
      last.count = -1;
      if (ok) tell(last);
      // On the error path, copies in flight land before the CTA may exit.
      if (*abort_f) {
        for (int i = 0; i < S::STAGES; ++i)
          for (uint32_t parity = 0; parity < 2; ++parity) {
            drain_phase(&B->full[i], parity);
          }
        for (int i = 0; i < 2; ++i) {
          drain_phase(&B->q_full[i], 0);
          drain_phase(&B->q_full[i], 1);
        }
      }
    }
    if (warp == CLEAN_WARP) {
      // ------------------------------------------------------------ odd elements
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      Unit U;
      for (Walk walk(B, A.err); ok && walk.next(U);) {
        const int steps = max(U.steps[0], U.steps[1]);
        for (int j = -2; j < steps && steps > 0; ++j) {
          // Every stage is waited for, so that this warp stays within one round
          // of the ring of the others.
          ok = warp_wait(&B->full[st], ph, abort_f, A.err);
          if (!ok) break;
          // (Paged: a page outside the cache was not copied, the place holds anything.)
          if (j >= 0 && (j >= U.whole || (PAGED && *const_cast<volatile uint64_t*>(
                                              &B->valid[(U.base + j) & (SEEN - 1)]) != ~0ull))) {
            // A quick look first: the largest magnitude of each half, as bits.
            uint4* at = reinterpret_cast<uint4*>(ring + st * S::STAGE + S::KC * BLOCK) + lane;
            uint32_t most[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < S::VC * BLOCK / 512; ++i) {
              const uint4 x = at[i * 32];
              most[0] = __vmaxu2(most[0], x.x & 0x7fff7fffu);
              most[1] = __vmaxu2(most[1], x.y & 0x7fff7fffu);
              most[2] = __vmaxu2(most[2], x.z & 0x7fff7fffu);
              most[3] = __vmaxu2(most[3], x.w & 0x7fff7fffu);
            }
            const uint32_t top = __vmaxu2(__vmaxu2(most[0], most[1]), __vmaxu2(most[2], most[3]));
            const bool odd =
                odd_element<F16>((uint16_t)top) || odd_element<F16>((uint16_t)(top >> 16));
            if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
              for (int i = 0; i < S::VC * BLOCK / 512; ++i) {
                uint4 x = at[i * 32];
                clear_odd<F16>(x);
                at[i * 32] = x;
              }
              B->odd[U.count & 15] = U.count;
              fence_proxy_async();
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&B->clean[st]);
          if (++st == S::STAGES) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == CLEAN_WARP) {
    tc::tc_fence_after();
    tc::tmem_free_all(tmem);
  }
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------

template <int DKP, int DVP, bool F16, bool PAGED>
static int launch_prompt(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                         const PromptArgs& A, int grid, void* stream) {
  using S = PromptShape<DKP, DVP>;
  static std::mutex mu;
  static bool done[64] = {};
  const void* fn = reinterpret_cast<const void*>(&prompt_kernel<DKP, DVP, F16, PAGED>);
  const int st = allow_smem(fn, S::SMEM, done, mu);
  if (st != KB_OK) return st;
  return launch(prompt_kernel<DKP, DVP, F16, PAGED>, dim3(grid), dim3(PROMPT_THREADS),
                (size_t)S::SMEM, stream, mq, mk, mv, A);
}

template <bool PAGED>
static int launch_widths(int64_t Dk, int64_t Dv, int f16, const CUtensorMap& mq,
                         const CUtensorMap& mk, const CUtensorMap& mv, const PromptArgs& A,
                         int grid, void* stream) {
  if (Dk <= 64 && Dv <= 64)
    return f16 ? launch_prompt<64, 64, true, PAGED>(mq, mk, mv, A, grid, stream)
               : launch_prompt<64, 64, false, PAGED>(mq, mk, mv, A, grid, stream);
  if (Dk <= 128)
    return f16 ? launch_prompt<128, 128, true, PAGED>(mq, mk, mv, A, grid, stream)
               : launch_prompt<128, 128, false, PAGED>(mq, mk, mv, A, grid, stream);
  return f16 ? launch_prompt<192, 128, true, PAGED>(mq, mk, mv, A, grid, stream)
             : launch_prompt<192, 128, false, PAGED>(mq, mk, mv, A, grid, stream);
}

constexpr int ROW_CTAS = 160;                // CTAs the workspace of the paged form is made for
constexpr size_t ROW_COUNTERS = 2 * ROW_CTAS * sizeof(int);
static_assert(ROW_COUNTERS <= ZEROED, "counters where callers zero");

// Counters, then two partial sums a CTA: maximum and sum, 128 values, of the 128 or
// 256 rows of a unit.
static int part_rows(int64_t rows) { return rows > TILE ? 2 * TILE : TILE; }

size_t rows_workspace(int64_t rows) {
  return ROW_COUNTERS + (size_t)2 * ROW_CTAS * part_rows(rows) * (2 + 128) * sizeof(float);
}

int launch_rows(const TreeCall& T, int64_t rows, int sms, void* workspace, void* stream) {
  PromptArgs A = {};
  A.q = T.q;
  A.v = T.v;
  A.q_tok = T.q_tok;
  A.q_head = T.q_head;
  A.v_page = T.v_page;
  A.v_tok = T.v_row;
  A.v_head = T.v_head;
  A.out = T.out;
  A.lse = T.lse;
  A.cu_q = T.cu;
  A.total_q = T.total;
  A.B = T.B;
  A.Hq = T.Hq;
  A.Hkv = T.Hkv;
  A.g = T.Hq / T.Hkv;
  A.Dk = T.Dk;
  A.Dv = T.Dv;
  A.scale2 = T.scale2;
  A.err = T.err;
  A.table = T.table;
  A.table_stride = T.table_stride;
  A.context = T.context;
  A.mask = T.mask;
  A.n_pages = T.n_pages;
  A.width = T.width;
  A.ps = T.ps;
  A.places = T.places;
  A.most = T.most;
  A.counters = static_cast<int*>(workspace);
  A.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ROW_COUNTERS);
  A.part_rows = part_rows(rows);
  A.part_o = A.part_ml + (size_t)2 * ROW_CTAS * A.part_rows * 2;
  // One tile of rows: q by tensor copies, keys and values in boxes of 16 rows.
  const bool solo = A.part_rows == TILE;
  const int box = std::min(T.ps, solo ? 16 : STEP);
  CUtensorMap mq = {}, mk, mv;
  int st = KB_OK;
  if (solo) st = make_map_4d(&mq, T.q, T.f16, {T.Dk, T.Hq, T.total, 1}, {T.q_head, T.q_tok, 8},
                             A.g, TILE / A.g);
  if (st == KB_OK) st = make_map_4d(&mk, T.k, T.f16, {T.Dk, T.ps, T.Hkv, T.n_pages},
                                    {T.k_row, T.k_head, T.k_page}, box, 1);
  if (st == KB_OK) st = make_map_4d(&mv, T.v, T.f16, {T.Dv, T.ps, T.Hkv, T.n_pages},
                                    {T.v_row, T.v_head, T.v_page}, box, 1);
  if (st != KB_OK) return st;
  return launch_widths<true>(T.Dk, T.Dv, T.f16, mq, mk, mv, A, std::min(sms, ROW_CTAS), stream);
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
  namespace at = kb::attn;
  kb::clear_error();
  KB_REQUIRE(B >= 0 && total_q >= 0 && total_k >= 0 && max_q >= 0, KB_ERR_BAD_SHAPE,
             "prompt attention: bad shape");
  int st = at::check_heads(Hq, Hkv, Dk, Dv, dtype);
  if (st != KB_OK) return st;
  if (B == 0 || total_q == 0) return KB_OK;
  KB_REQUIRE(scale > 0.f, KB_ERR_BAD_SHAPE, "attention: the scale must be positive");
  KB_REQUIRE(max_q > 0, KB_ERR_BAD_SHAPE, "prompt attention: tokens but max_q 0");
  KB_REQUIRE(q && cu_q && cu_k && out && (total_k == 0 || (k && v)), KB_ERR_NULL_POINTER,
             "prompt attention: NULL pointer");
  constexpr int64_t kMax = (int64_t)1 << 30;
  KB_REQUIRE(B <= 65535 && total_q <= kMax && total_k <= kMax && Hq <= 65535, KB_ERR_UNSUPPORTED,
             "prompt attention: more than 2^30 tokens or 65535 requests or heads");
  const bool ok =
      (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0 &&
      ((q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride |
        v_head_stride) & 7) == 0;
  KB_REQUIRE(ok, KB_ERR_ALIGNMENT,
             "prompt attention: pointers must be 16-byte aligned and strides multiples of 8");
  const int dev = kb::bind_stream_device(stream);
  at::PromptArgs A = {};
  A.q = q;
  A.k = k;
  A.v = v;
  A.q_tok = q_token_stride;
  A.q_head = q_head_stride;
  A.k_tok = k_token_stride;
  A.k_head = k_head_stride;
  A.v_tok = v_token_stride;
  A.v_head = v_head_stride;
  A.out = out;
  A.lse = lse;
  A.cu_q = cu_q;
  A.cu_k = cu_k;
  A.total_q = total_q;
  A.total_k = total_k;
  A.B = (int)B;
  A.Hq = (int)Hq;
  A.g = (int)(Hq / Hkv);
  A.Dk = (int)Dk;
  A.Dv = (int)Dv;
  while (A.pack_shift < 7 && A.g % (2 << A.pack_shift) == 0) ++A.pack_shift;
  A.scale2 = scale * kb::LOG2E;
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  const int pack = 1 << A.pack_shift;
  const int64_t longest = std::min(max_q, total_q);
  const int64_t blocks = (longest * pack + 2 * at::TILE - 1) / (2 * at::TILE);
  const int64_t units = blocks * B * (Hq / pack);
  KB_REQUIRE(units <= kMax, KB_ERR_UNSUPPORTED, "prompt attention: too many units of rows");
  A.blocks = (int)blocks;
  CUtensorMap mq, mk, mv;
  st = at::make_map_4d(&mq, q, dtype, {Dk, Hq, total_q, 1}, {q_head_stride, q_token_stride, 8},
                       pack, at::TILE / pack);
  if (st != KB_OK) return st;
  // Without keys no tile is ever copied: any valid map will do.
  const int64_t keys = std::max<int64_t>(total_k, 1);
  st = at::make_map_4d(&mk, total_k ? k : q, dtype, {Dk, Hkv, keys, 1},
                       {k_head_stride, k_token_stride, 8}, 1, at::STEP);
  if (st != KB_OK) return st;
  st = at::make_map_4d(&mv, total_k ? v : q, dtype, {Dv, Hkv, keys, 1},
                       {v_head_stride, v_token_stride, 8}, 1, at::STEP);
  if (st != KB_OK) return st;
  const int grid = (int)std::min<int64_t>(kb::num_sms(dev), units);
  return at::launch_widths<false>(Dk, Dv, dtype, mq, mk, mv, A, grid, stream);
}
