// kb_prompt.cu - causal attention over packed prompts on the 5th-generation
// tensor cores.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / l_i,  s_ij = scale * q_i . k_j over the visible j,
//   m_i = max_j s_ij, l_i = sum_j exp(s_ij - m_i), lse_i = m_i + log(l_i)
// visible: j <= i + (Lk - Lq).  A row that sees no key gives 0 and lse -infinity.
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
// 512 columns of tensor memory: two S of 64 for A and for B, O A, O B.  Bound:
// MMAs, 51 clocks each for S (128 x 64 x 16, both operands from shared
// memory: the copies of A set the rate; 64 clocks at 128 x 128 x 16) and 64
// for P V, which is 2644 clocks for 128 keys of A and B at 128-wide heads,
// 3452 at 192 + 128.  With steps of 128 keys and one S a tile the MMAs are 2048
// and 2560 clocks, but each waits for the softmax of its own tile in turn:
// 3600 and 4430 measured.  The exponentials (16 a clock and SM) would take
// 2048; one pair in POLY_EVERY goes to the FMA pipes.
//
// In the last tiles of a unit some rows do not see some keys, or the tile
// reaches past the request's end into its neighbour.  A value there that is
// infinite or not a number must not meet a zero weight: warp 11 zeroes such
// elements in those tiles before the MMA reads them, and at the end the rows
// that do see them take them from memory.
#include <algorithm>
#include <type_traits>

#include "kb_attn.cuh"
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
};

template <int DKP, int DVP>
struct PromptShape {
  static constexpr int KC = DKP / 64;                    // blocks of a step's keys
  static constexpr int VC = DVP / 64;                    // ... and values
  static constexpr int Q_TILE = 2 * KC * BLOCK;          // bytes of a Q tile (128 rows)
  static constexpr int STAGE = (KC + VC) * BLOCK;
  static constexpr int FIXED = 1024 + 1024;              // alignment, barriers
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
  int t0;                   // first token of tile A
  int steps[2];             // steps of keys that tiles A and B see
  int whole;                // of them, those that every row of A sees whole
  int count;                // number of the unit in this CTA, -1: the end
};

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
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(PromptBars) <= 1024, "barrier block");

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
// 2^-126 the result stays there.
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
__device__ __forceinline__ void add_odd(const PromptArgs& A, const uint16_t* v, int first,
                                        int last, int d0, float (&o)[32]) {
  for (int64_t j = first; j <= last; ++j) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint16_t u = d0 + i < A.Dv ? v[j * A.v_tok + d0 + i] : 0;
      if (odd_element<F16>(u)) o[i] += element<F16>(u);
    }
  }
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

template <int DKP, int DVP, bool F16>
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

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&B->full[i], 1);
      mbar_init(&B->empty[i], 2);
      mbar_init(&B->clean[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B->q_full[i], 1);
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
    prefetch_map(&tq);
    prefetch_map(&tk);
    prefetch_map(&tv);
  }
  if (warp == CLEAN_WARP) tc::tmem_alloc_all(&B->tmem);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = B->tmem;
  pdl_wait();
  pdl_launch_dependents();

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
    uint32_t s_phase = 0, near_phase = 0, end_phase = 0;
    Unit U;
    for (Walk walk(B, A.err); walk.next(U);) {
      const int first = U.t0 + tile * span;
      if (first >= U.n) continue;
      const int tok = first + (row >> A.pack_shift);
      const int head = U.head0 + (row & ((1 << A.pack_shift) - 1));
      const bool real = tok < U.n;
      const int limit = min(tok, U.n - 1) + U.m - U.n;      // last key the row sees
      const int clear = first + U.m - U.n;                  // ... and the tile's first row
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
        const bool edge = j * STEP + STEP - 1 > clear;     // keys that some rows do not see
        if (edge) {
          const int last = limit - j * STEP;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i > last) s[c][i] = -INFINITY;
        }
        float mx[4] = {s[0][0], s[0][1], s[1][0], s[1][1]};
#pragma unroll
        for (int i = 2; i < 30; i += 4)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            mx[c] = max3(mx[c], s[c >> 1][i + (c & 1) * 2], s[c >> 1][i + (c & 1) * 2 + 1]);
        mx[0] = max3(mx[0], s[0][30], s[0][31]);
        mx[2] = max3(mx[2], s[1][30], s[1][31]);
        const float mine = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * scale2;
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
      uint16_t* out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (row & ~3) + i, t = first + (r >> A.pack_shift);
        const int h = U.head0 + (r & ((1 << A.pack_shift) - 1));
        out[i] = t < U.n ? A.out + ((int64_t)(U.q0 + t) * A.Hq + h) * A.Dv + (lane & 3) * 8
                         : nullptr;
      }
      if (steps > 1) near_phase ^= 1u;
      bool odd = false;
      if (steps > 0) {
        if (!warp_wait(&B->o_full[tile], end_phase, abort_f, A.err)) break;
        end_phase ^= 1u;
        tc::tc_fence_after();
        odd = *const_cast<volatile int*>(&B->odd[U.count & 15]) == U.count;
      }
      // A row that saw no key (or only keys of score -infinity) is zero.
      const bool none = sum == 0.f || limit < 0;
      const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
      for (int c = 0; c < DVP / 32; ++c) {
        float o[32];
        if (steps > 0) {
          tc::tmem_ld32(o_at + c * 32, o);
          tc::tmem_ld_wait();
          tc::hold_regs(o);
          if (odd)
            add_odd<F16>(A, A.v + U.k0 * A.v_tok + head / A.g * A.v_head, U.whole * STEP, limit,
                         c * 32, o);
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
      if (real && A.lse) A.lse[at] = none ? -INFINITY : (top + log2f(sum)) * LN2;
      __syncwarp();
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
      auto copy = [&](const Unit& U) {
        const int steps = max(U.steps[0], U.steps[1]);
        const int hk = U.head0 / A.g;
        auto queries = [&](int i) {
          if (U.steps[i] == 0 || !need(&B->q_empty[i], q_phase[i])) return;
          q_phase[i] ^= 1u;
          if (lane != 0) return;
          mbar_arrive_expect_tx(&B->q_full[i], (uint32_t)S::Q_TILE);
          for (int c = 0; c < S::KC; ++c)
            tma_load_4d(qs + i * S::Q_TILE + c * 2 * BLOCK, &tq, c * 64, U.head0,
                        U.q0 + U.t0 + i * span, 0, &B->q_full[i], once);
        };
        for (int j = -2; j < steps && steps > 0; ++j) {
          if (j == -2) queries(0);
          if (!need(&B->empty[st], ph)) break;
          const bool keys = j + 2 < steps, values = j >= 0;
          if (lane == 0) {
            uint8_t* at = ring + st * S::STAGE;
            mbar_arrive_expect_tx(&B->full[st], (uint32_t)(((keys ? S::KC : 0) +
                                                            (values ? S::VC : 0)) * BLOCK));
            if (keys)
              for (int c = 0; c < S::KC; ++c)
                tma_load_4d(at + c * BLOCK, &tk, c * 64, hk, U.k0 + (j + 2) * STEP, 0,
                            &B->full[st], keep);
            if (values)
              for (int d = 0; d < S::VC; ++d)
                tma_load_4d(at + (S::KC + d) * BLOCK, &tv, d * 64, hk, U.k0 + j * STEP, 0,
                            &B->full[st], keep);
          }
          if (++st == S::STAGES) {
            st = 0;
            ph ^= 1u;
          }
          if (j == -2) queries(1);
        }
      };
      for (int block = A.blocks - 1; block >= 0 && ok; --block) {
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
          if (j >= 0 && j >= U.whole) {
            bool any = false;
            uint4* at = reinterpret_cast<uint4*>(ring + st * S::STAGE + S::KC * BLOCK) + lane;
#pragma unroll 8
            for (int i = 0; i < S::VC * BLOCK / 512; ++i) {
              uint4 x = at[i * 32];
              if (has_odd<F16>(x)) {
                clear_odd<F16>(x);
                at[i * 32] = x;
                any = true;
              }
            }
            if (any) {
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

template <int DKP, int DVP, bool F16>
static int launch_prompt(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                         const PromptArgs& A, int grid, void* stream) {
  using S = PromptShape<DKP, DVP>;
  static std::mutex mu;
  static bool done[64] = {};
  const void* fn = reinterpret_cast<const void*>(&prompt_kernel<DKP, DVP, F16>);
  const int st = allow_smem(fn, S::SMEM, done, mu);
  if (st != KB_OK) return st;
  return launch(prompt_kernel<DKP, DVP, F16>, dim3(grid), dim3(PROMPT_THREADS), (size_t)S::SMEM,
                stream, mq, mk, mv, A);
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
  if (Dk <= 64 && Dv <= 64)
    return dtype ? at::launch_prompt<64, 64, true>(mq, mk, mv, A, grid, stream)
                 : at::launch_prompt<64, 64, false>(mq, mk, mv, A, grid, stream);
  if (Dk <= 128)
    return dtype ? at::launch_prompt<128, 128, true>(mq, mk, mv, A, grid, stream)
                 : at::launch_prompt<128, 128, false>(mq, mk, mv, A, grid, stream);
  return dtype ? at::launch_prompt<192, 128, true>(mq, mk, mv, A, grid, stream)
               : at::launch_prompt<192, 128, false>(mq, mk, mv, A, grid, stream);
}
