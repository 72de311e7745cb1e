// kb_linear_chunk.cu - linear attention with a decay for each head over prompts, in chunks of
// 128 tokens on the 5th-generation tensor cores (bf16).
//
// With b_i the running sum of the decays' logarithms in a chunk, for its rows i and j <= i:
//   P_ij = (q_i . k_j) exp(b_i - b_j)
//   o_i  = scale * (exp(b_i) q_i S + sum_j P_ij v_j)
//   S'   = exp(b_C) S + sum_j k_j (exp(b_C - b_j) v_j)^T
// Every exponent is at most 0.  The sums of logarithms are made in 64 bits; a decay that is 0
// in fp32 (below e^-104, -infinity too) is a reset: what lies before it does not count.
//
// One persistent CTA per SM; a unit is one head of one request (or of a segment of it), its
// chunks one after the other.  Q, K and V tiles (128 rows, 64-element blocks in the 128-byte
// swizzle) arrive by tensor copies in two stages.
//
//   warp 18: the units, the copies and the decays of each chunk.
//   warp 16: issues S = Q K^T, O = Q S (the state), O += P V.
//   warp 17: issues S^T += V'^T K, V' = the values with their decay to the chunk's end.
//   warps 8-15: P from the scores, a row per thread and half the columns each; the part of the
//     state scaled by exp(b_i) in tensor memory before P V is added to it; the outputs.
//   warps 0-7: V' and the state.  The state lives in these warps' registers in fp32 (a value
//     column a thread, half of the key rows each); its bf16 copy is what Q S reads.
//
// Roundings.  P and the copy of the state are rounded once to bf16 before they meet the values
// and the queries: the outputs have 8 bits themselves.  The state must not lose bits: V' (fp32
// products) enters the tensor cores as the sum of three bf16 values, 24 bits in all.
//
// 512 columns of tensor memory: scores and P 128, O 128, the state's gain 128, and two of the
// three parts of V' (the third replaces the first once that is used).
//
// A row past the request's end belongs to a neighbour: its keys and values are zeroed in shared
// memory.  A value that is no number is zeroed too, since it would meet zero weights; the rows
// from its token on are set to not-a-number at the end, and the state gets it from V'.
#include <algorithm>

#include "kb_linear.cuh"
#include "kb_tcgen05.cuh"

namespace kb {
namespace linear {

using attn::wait_phase;
using attn::warp_wait;

constexpr int CHUNK = 128;
constexpr int BLOCK = CHUNK * 128;           // bytes of 128 rows x 64 elements
constexpr int THREADS = 640;
constexpr int STAGES = 2;
constexpr int PREPARE_WARPS = 8;             // and as many of outputs
constexpr int MMA_WARP = 16, GAIN_WARP = 17, COPY_WARP = 18;
constexpr float RESET = -104.f;
constexpr uint32_t S_AT = 0, O_AT = 128, GAIN_AT = 256, V1_AT = 384, V2_AT = 448;

struct ChunkArgs {
  Args a;
  int segments, segment;                     // of a request at most; tokens of one
  float* sums;                               // [B][segments][H][Dk][Dv]: a segment's gain
  float* keeps;                              // [B][segments][H]: its decay
};

struct Item {
  int64_t first;                             // the chunk's first token
  int n;                                     // its tokens, -1: the end
  int b, h, seg;
  int starts, ends;                          // the unit's first, last chunk; 2: the request's
  int odd;                                   // values that are no numbers
  int resets;
  float keep;                                // exp(b_C)
};

template <int DKP, int DVP>
struct ChunkShape {
  static constexpr int KC = DKP / 64, VC = DVP / 64;
  static constexpr int STAGE = (2 * KC + VC) * BLOCK;
  static constexpr int STATE = KC * DVP * 128;           // bytes of the bf16 copy
  static constexpr int FIXED = 3072;
  static constexpr int SMEM = STAGES * STAGE + STATE + FIXED;
};

struct ChunkShared {
  float at[STAGES][CHUNK];                   // b_i, base 2
  float left[STAGES][CHUNK];                 // exp(b_C - b_j)
  uint8_t since[STAGES][CHUNK];              // the last reset up to the row, plus 1; 0: none
  uint8_t odd_from[2][CHUNK];                // of each value column, of a chunk's halves
  Item item[STAGES];
  uint64_t full[STAGES], info[STAGES], empty[STAGES];
  uint64_t s_full, q_done, p_full, o_full, o_free, state_ready, clean, v_two, v_half, v_three,
      gain_done, drain;
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(ChunkShared) <= 3072, "fixed shared memory");

// Half of a transposition: lanes `step` apart keep one piece and swap the other.
__device__ __forceinline__ void swap_pieces(uint4& a, uint4& b, int upper, int step) {
  uint4 give = upper ? a : b;
  give.x = __shfl_xor_sync(0xffffffffu, give.x, step);
  give.y = __shfl_xor_sync(0xffffffffu, give.y, step);
  give.z = __shfl_xor_sync(0xffffffffu, give.z, step);
  give.w = __shfl_xor_sync(0xffffffffu, give.w, step);
  if (upper) a = give; else b = give;
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) {
  return __uint_as_float(w & 0xffff0000u);
}

// The units of this CTA and their chunks, in order.
struct Items {
  const ChunkArgs& C;
  int64_t unit, units;
  int64_t at, end, last;                     // tokens of the unit left; the request's end
  Item next;
  bool states;
  __device__ __forceinline__ Items(const ChunkArgs& c, bool s) : C(c), at(0), end(0), last(0), states(s) {
    unit = (int64_t)blockIdx.x - gridDim.x;
    units = (int64_t)C.a.B * C.segments * C.a.H;
    advance();
  }
  __device__ __forceinline__ void advance() {
    const Args& A = C.a;
    next.starts = 0;
    while (at >= end) {
      unit += gridDim.x;
      if (unit >= units) {
        next.n = -1;
        return;
      }
      const int64_t bs = unit / A.H;
      next.h = (int)(unit - bs * A.H);
      next.b = (int)(bs / C.segments);
      next.seg = (int)(bs - (int64_t)next.b * C.segments);
      int64_t first;
      const int n = request_tokens(A, next.b, first);
      at = first + (int64_t)next.seg * C.segment;
      last = first + n;
      end = min(last, at + C.segment);
      // The last segment's gain is nobody's start.
      if (states && end >= last) end = at;
      next.starts = 1;
    }
    next.first = at;
    next.n = (int)min(end - at, (int64_t)CHUNK);
    at += CHUNK;
    next.ends = at < end ? 0 : end < last ? 1 : 2;
  }
};

template <int DKP, int DVP, bool STATES>
__global__ void __launch_bounds__(THREADS, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                 const __grid_constant__ CUtensorMap tv, const ChunkArgs C) {
  using Sh = ChunkShape<DKP, DVP>;
  constexpr int KC = Sh::KC, VC = Sh::VC;
  constexpr int HALF = DKP / 2;              // key rows of a thread's part of the state
  const Args& A = C.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* copy_of_state = smem + STAGES * Sh::STAGE;
  ChunkShared* B = reinterpret_cast<ChunkShared*>(copy_of_state + Sh::STATE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_f = &B->abort_flag;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&B->full[i], 1);
      mbar_init(&B->info[i], 1);
      mbar_init(&B->empty[i], STATES ? 1 + PREPARE_WARPS : 2 + 2 * PREPARE_WARPS);
    }
    mbar_init(&B->s_full, 1);
    mbar_init(&B->q_done, 1);
    mbar_init(&B->p_full, PREPARE_WARPS);
    mbar_init(&B->o_full, 1);
    mbar_init(&B->o_free, PREPARE_WARPS);
    mbar_init(&B->state_ready, PREPARE_WARPS);
    mbar_init(&B->clean, PREPARE_WARPS);
    mbar_init(&B->v_two, PREPARE_WARPS);
    mbar_init(&B->v_half, 1);
    mbar_init(&B->v_three, PREPARE_WARPS);
    mbar_init(&B->gain_done, 1);
    mbar_init(&B->drain, STATES ? 1 : 2);
    B->abort_flag = 0;
    mbar_fence_init();
    if (!STATES) attn::prefetch_map(&tq);
    attn::prefetch_map(&tk);
    attn::prefetch_map(&tv);
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

  if (warp < PREPARE_WARPS) {
    // ------------------------------------------------------------------ the state
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    const int part = warp >> 2;              // key rows part * HALF .., chunk rows part * 64 ..
    const int dv = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool active = (warp & 3) * 32 < DVP;
    float s[HALF];
    float all = 1.f;                         // the unit's decay so far
    int st = 0;
    uint32_t ph = 0, one_phase = 0;          // of the stages; of the barriers met once a chunk
    bool ok = true;
    auto need = [&](uint64_t* bar, uint32_t parity) {
      ok = warp_wait(bar, parity, abort_f, A.err);
      return ok;
    };
    auto arrive = [&](uint64_t* bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
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
      const Item I = B->item[st];
      if (I.n < 0) break;
      if (I.starts) {
        // What the unit starts from: the request's state, and the gains of the segments before.
        const float* from = STATES ? nullptr : request_state(A, I.b, I.h);
        const bool mine = active && dv < A.Dv;
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
          const int dk = part * HALF + i;
          s[i] = from != nullptr && mine && dk < A.Dk ? __ldcg(from + (int64_t)dk * A.Dv + dv) : 0.f;
        }
        if (!STATES) {
          for (int g = 0; g < I.seg; ++g) {
            const int64_t u = ((int64_t)I.b * C.segments + g) * A.H + I.h;
            const float keep = __ldcg(C.keeps + u);
            const float* gain = C.sums + u * A.Dk * A.Dv;
#pragma unroll
            for (int i = 0; i < HALF; ++i) {
              const int dk = part * HALF + i;
              const float x = mine && dk < A.Dk ? __ldcg(gain + (int64_t)dk * A.Dv + dv) : 0.f;
              s[i] = fmaf(s[i], keep, x);
            }
          }
          copy_state();
        }
      }
      if (!need(&B->full[st], ph)) break;
      uint8_t* k_tile = smem + st * Sh::STAGE + KC * BLOCK;
      uint8_t* v_tile = k_tile + KC * BLOCK;
      if (I.n < CHUNK) {
        // Rows of a neighbour: zero.  (Of the values, those that this warp reads.)
        for (int x = threadIdx.x; x < (CHUNK - I.n) * 8 * KC; x += PREPARE_WARPS * 32) {
          const int r = x >> 3, c = r / (CHUNK - I.n);
          *reinterpret_cast<uint4*>(k_tile + c * BLOCK + (I.n + r - c * (CHUNK - I.n)) * 128 +
                                    (x & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        if (active)
          for (int j = max(I.n, part * 64) + (lane >> 2); j < part * 64 + 64; j += 8) {
            const int piece = (((warp & 1) * 4 + (lane & 3)) ^ (j & 7)) << 4;
            *reinterpret_cast<uint4*>(v_tile + ((warp & 3) >> 1) * BLOCK + j * 128 + piece) =
                make_uint4(0, 0, 0, 0);
          }
        __syncwarp();
      }
      uint32_t last[32];                     // the third part of V', pairs of chunk rows
      if (active) {
        const uint8_t* column = v_tile + (dv >> 6) * BLOCK + (dv & 7) * 2;
        const int piece = (dv & 63) >> 3;
        const float* left = &B->left[st][part * 64];
        float odd = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {        // 16 rows a round
          uint32_t lo[8], mid[8];
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float4 d = *reinterpret_cast<const float4*>(left + c * 16 + i * 2);
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int j = part * 64 + c * 16 + i * 2 + u;
              x[u] = bf16_bits_to_float(*reinterpret_cast<const uint16_t*>(
                  column + j * 128 + ((piece ^ (j & 7)) << 4)));
              odd = fmaf(x[u], 0.f, odd);
            }
            x[0] *= d.x;
            x[1] *= d.y;
            x[2] *= d.z;
            x[3] *= d.w;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t h = attn::pack2<false>(x[2 * u], x[2 * u + 1]);
              const float r0 = x[2 * u] - low_half(h), r1 = x[2 * u + 1] - high_half(h);
              const uint32_t m = attn::pack2<false>(r0, r1);
              lo[i + u] = attn::pack2<false>(r0 - low_half(m), r1 - high_half(m));
              mid[i + u] = m;
              last[c * 8 + i + u] = h;
            }
          }
          tmem_st8(lanes + V1_AT + part * 32 + c * 8, lo);
          tmem_st8(lanes + V2_AT + part * 32 + c * 8, mid);
        }
        if (__any_sync(0xffffffffu, odd != 0.f)) {     // true of not-a-number
          int from = 255;
          for (int j = part * 64; j < part * 64 + 64; ++j) {
            uint16_t* e = reinterpret_cast<uint16_t*>(v_tile + (dv >> 6) * BLOCK + (dv & 7) * 2 +
                                                      j * 128 + ((piece ^ (j & 7)) << 4));
            if (attn::odd_element<false>(*e)) {
              from = min(from, j);
              *e = 0;
            }
          }
          B->odd_from[part][dv] = (uint8_t)from;
          __syncwarp();
          if (lane == 0) atomicOr(&B->item[st].odd, 1 << warp);
        }
        tc::tmem_st_wait();
      }
      attn::fence_proxy_async();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (!STATES) mbar_arrive(&B->clean);
        mbar_arrive(&B->v_two);
      }
      if (!need(&B->v_half, one_phase)) break;
      tc::tc_fence_after();
      if (active) {
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_st8(lanes + V1_AT + part * 32 + c * 8, last + c * 8);
        tc::tmem_st_wait();
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&B->v_three);
        mbar_arrive(&B->empty[st]);
      }
      if (!need(&B->gain_done, one_phase)) break;
      tc::tc_fence_after();
      if (active)
#pragma unroll
        for (int c = 0; c < HALF / 32; ++c) {
          float gain[32];
          tc::tmem_ld32(lanes + GAIN_AT + part * HALF + c * 32, gain);
          tc::tmem_ld_wait();
          tc::hold_regs(gain);
#pragma unroll
          for (int i = 0; i < 32; ++i) s[c * 32 + i] = fmaf(s[c * 32 + i], I.keep, gain[i]);
        }
      tc::tc_fence_before();
      if (!STATES && !need(&B->q_done, one_phase)) break;
      if (I.ends) {
        const int64_t u = ((int64_t)I.b * C.segments + I.seg) * A.H + I.h;
        float* to = STATES ? C.sums + u * A.Dk * A.Dv
                           : I.ends == 2 ? request_state(A, I.b, I.h) : nullptr;
        if (STATES && threadIdx.x == 0) C.keeps[u] = all * I.keep;
        if (to != nullptr && active && dv < A.Dv)
#pragma unroll
          for (int i = 0; i < HALF; ++i) {
            const int dk = part * HALF + i;
            if (dk < A.Dk) to[(int64_t)dk * A.Dv + dv] = s[i];
          }
      } else if (!STATES) {
        copy_state();
      }
      all = I.ends ? 1.f : all * I.keep;
      one_phase ^= 1u;
      if (++st == STAGES) {
        st = 0;
        ph ^= 1u;
      }
    }
  } else if (warp < 2 * PREPARE_WARPS) {
    // ---------------------------------------------------------------- the outputs
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int part = (warp >> 2) & 1;        // columns part * 64 .. of the scores
    const int q0 = (warp & 3) * 32, row = q0 + lane;
    const uint32_t lanes = tmem + ((uint32_t)q0 << 16);
    constexpr int COLS = DVP / 2;            // of the outputs a thread has
    int st = 0;
    uint32_t ph = 0, one_phase = 0;
    bool ok = true;
    auto need = [&](uint64_t* bar, uint32_t parity) {
      ok = warp_wait(bar, parity, abort_f, A.err);
      return ok;
    };
    while (!STATES) {
      if (!need(&B->info[st], ph)) break;
      const Item I = B->item[st];
      if (I.n < 0) break;
      const float mine = B->at[st][row];
      const int since = B->since[st][row];
      if (!need(&B->s_full, one_phase)) break;
      tc::tc_fence_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int j0 = part * 64 + c * 32;
        uint32_t p[16];
        if (j0 > q0) {                       // all behind the rows
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = 0;
        } else {
          float x[32];
          tc::tmem_ld32(lanes + S_AT + j0, x);
          tc::tmem_ld_wait();
          tc::hold_regs(x);
          const float* at = &B->at[st][j0];
          const float2 here = make_float2(mine, mine), minus = make_float2(-1.f, -1.f);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 b = *reinterpret_cast<const float4*>(at + i);
            float2 e = ffma2(make_float2(b.x, b.y), minus, here);
            float2 f = ffma2(make_float2(b.z, b.w), minus, here);
            e = make_float2(exp2_fast(e.x), exp2_fast(e.y));
            f = make_float2(exp2_fast(f.x), exp2_fast(f.y));
            e = fmul2(make_float2(x[i], x[i + 1]), e);
            f = fmul2(make_float2(x[i + 2], x[i + 3]), f);
            x[i] = e.x;
            x[i + 1] = e.y;
            x[i + 2] = f.x;
            x[i + 3] = f.y;
          }
          if (j0 == q0 || I.resets) {
            const int lo = since - 1 - j0, hi = row - j0;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i > hi || i < lo) x[i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = attn::pack2<false>(x[2 * i], x[2 * i + 1]);
        }
        // (In place of scores that this thread has read.)
        tc::tmem_st16(lanes + S_AT + part * 64 + c * 16, p);
      }
      if (!need(&B->q_done, one_phase)) break;
      tc::tc_fence_after();
      const float gain = since ? 0.f : exp2_fast(mine);
#pragma unroll
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
      // Four lanes side by side exchange 16-byte pieces, so that a store covers 64 bytes of
      // eight rows and not 16 of 32.
      uint16_t* out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (row & ~3) + i;
        out[i] = r < I.n ? static_cast<uint16_t*>(A.out) + ((I.first + r) * A.H + I.h) * A.Dv +
                               part * COLS + (lane & 3) * 8
                         : nullptr;
      }
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) {
        const int d0 = part * COLS + c * 32;
        float o[32];
        tc::tmem_ld32(lanes + O_AT + d0, o);
        tc::tmem_ld_wait();
        tc::hold_regs(o);
        if (odd)
          for (int half = 0; half < 2; ++half)
            if ((odd >> (half * 4 + (d0 >> 5))) & 1)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (row >= B->odd_from[half][d0 + i]) o[i] = NAN;
        uint4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i].x = attn::pack2<false>(o[8 * i] * A.scale, o[8 * i + 1] * A.scale);
          w[i].y = attn::pack2<false>(o[8 * i + 2] * A.scale, o[8 * i + 3] * A.scale);
          w[i].z = attn::pack2<false>(o[8 * i + 4] * A.scale, o[8 * i + 5] * A.scale);
          w[i].w = attn::pack2<false>(o[8 * i + 6] * A.scale, o[8 * i + 7] * A.scale);
        }
        swap_pieces(w[0], w[1], lane & 1, 1);
        swap_pieces(w[2], w[3], lane & 1, 1);
        swap_pieces(w[0], w[2], lane & 2, 2);
        swap_pieces(w[1], w[3], lane & 2, 2);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (out[i] && d0 + (lane & 3) * 8 < A.Dv)
            *reinterpret_cast<uint4*>(out[i] + c * 32) = w[i];
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&B->o_free);
        mbar_arrive(&B->empty[st]);
      }
      one_phase ^= 1u;
      if (++st == STAGES) {
        st = 0;
        ph ^= 1u;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    int st = 0;
    uint32_t ph = 0, one_phase = 0;
    bool ok = true;
    auto need = [&](uint64_t* bar, uint32_t parity) {
      ok = warp_wait(bar, parity, abort_f, A.err);
      return ok;
    };
    auto turn = [&]() {
      one_phase ^= 1u;
      if (++st == STAGES) {
        st = 0;
        ph ^= 1u;
      }
    };
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
        if (!need(&B->full[st], ph)) break;
        tc::tc_fence_after();
        const uint32_t q_at = base + st * Sh::STAGE, k_at = q_at + KC * BLOCK;
        const uint32_t v_at = k_at + KC * BLOCK;
#pragma unroll
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
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const uint64_t a = tc::sw128_desc(q_at + c * BLOCK);
          const uint64_t b = tc::sw128_desc(state_at + c * DVP * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc::umma_one(one, tm + O_AT, a + k * 2, b + k * 2, ID_Q, c + k > 0);
        }
        tc::umma_commit_one(one, &B->q_done);
        if (!need(&B->clean, one_phase) || !need(&B->p_full, one_phase)) break;
        tc::tc_fence_after();
        const uint64_t b = tc::sw128_desc_mn(v_at, BLOCK);
#pragma unroll
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
      while (true) {
        if (!need(&B->info[st], ph)) break;
        if (B->item[st].n < 0) break;
        if (!need(&B->full[st], ph) || !need(&B->v_two, one_phase)) break;
        tc::tc_fence_after();
        const uint64_t b = tc::sw128_desc_mn(base + st * Sh::STAGE + KC * BLOCK, BLOCK);
        auto product = [&](uint32_t from, uint32_t more) {
#pragma unroll
          for (int k = 0; k < CHUNK / 16; ++k)
            tc::umma_ts_one(one, tm + GAIN_AT, tm + from + k * 8, b + k * (2048 >> 4), ID_V,
                            more | (uint32_t)(k > 0));
        };
        product(V1_AT, 0);
        tc::umma_commit_one(one, &B->v_half);
        product(V2_AT, 1);
        if (!need(&B->v_three, one_phase)) break;
        tc::tc_fence_after();
        product(V1_AT, 1);
        tc::umma_commit_one(one, &B->gain_done);
        tc::umma_commit_one(one, &B->empty[st]);
        turn();
      }
      tc::umma_commit_one(one, &B->drain);
      attn::drain_phase(&B->drain, 0);
    } else if (warp == COPY_WARP) {
      // --------------------------------------------------------- units and copies
      const uint64_t keep_in_l2 = l2_evict_last_policy(), once = l2_evict_first_policy();
      const uint64_t k_policy = STATES || A.k_group > 1 ? keep_in_l2 : once;
      const uint64_t q_policy = A.q_group > 1 ? keep_in_l2 : once;
      const uint64_t v_policy = STATES ? keep_in_l2 : once;
      Items items(C, STATES);
      float g[4], ahead[4];
      auto fetch = [&](float (&x)[4]) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = lane * 4 + u;
          x[u] = j < items.next.n ? __ldg(A.decay + (items.next.first + j) * A.decay_tok +
                                          items.next.h)
                                  : 0.f;
        }
      };
      fetch(ahead);
      int sent = 0;
      while (true) {
        Item I = items.next;
#pragma unroll
        for (int u = 0; u < 4; ++u) g[u] = ahead[u];
        if (!need(&B->empty[st], ph ^ 1u)) break;
        if (I.n < 0) {
          if (lane == 0) {
            B->item[st].n = -1;
            mbar_arrive(&B->info[st]);
          }
          break;
        }
        if (lane == 0) {
          uint8_t* to = smem + st * Sh::STAGE;
          const int token = (int)I.first;
          mbar_arrive_expect_tx(&B->full[st],
                                (uint32_t)((STATES ? KC + VC : 2 * KC + VC) * BLOCK));
          for (int c = 0; c < KC; ++c) {
            if (!STATES)
              attn::tma_load_4d(to + c * BLOCK, &tq, c * 64, I.h / A.q_group, token, 0,
                                &B->full[st], q_policy);
            attn::tma_load_4d(to + (KC + c) * BLOCK, &tk, c * 64, I.h / A.k_group, token, 0,
                              &B->full[st], k_policy);
          }
          for (int c = 0; c < VC; ++c)
            attn::tma_load_4d(to + (2 * KC + c) * BLOCK, &tv, c * 64, I.h, token, 0,
                              &B->full[st], v_policy);
        }
        __syncwarp();
        ++sent;
        items.advance();
        fetch(ahead);
        // The chunk's decays: sums in 64 bits, and the last reset up to each row.
        double sum[4];
        int since[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float x = decay_of(g[u]);
          const bool reset = x <= RESET;
          sum[u] = (u ? sum[u - 1] : 0.0) + (reset ? 0.0 : (double)x);
          since[u] = reset ? lane * 4 + u + 1 : u ? since[u - 1] : 0;
        }
        double run = sum[3];
        int last = since[3];
        for (int o = 1; o < 32; o <<= 1) {
          const double r = __shfl_up_sync(0xffffffffu, run, o);
          const int l = __shfl_up_sync(0xffffffffu, last, o);
          if (lane >= o) {
            run += r;
            last = max(last, l);
          }
        }
        const double all = __shfl_sync(0xffffffffu, run, 31);
        const int resets = __shfl_sync(0xffffffffu, last, 31);
        double before = __shfl_up_sync(0xffffffffu, run, 1);
        int earlier = __shfl_up_sync(0xffffffffu, last, 1);
        if (lane == 0) {
          before = 0.0;
          earlier = 0;
        }
        constexpr double TO_2 = 1.4426950408889634;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = lane * 4 + u;
          const double b = before + sum[u];
          B->at[st][j] = (float)(b * TO_2);
          B->left[st][j] =
              j < I.n && j + 1 >= resets ? exp2f((float)((all - b) * TO_2)) : 0.f;
          B->since[st][j] = (uint8_t)max(since[u], earlier);
        }
        I.odd = 0;
        I.resets = resets;
        I.keep = resets ? 0.f : exp2f((float)(all * TO_2));
        if (lane == 0) B->item[st] = I;
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->info[st]);
        turn();
      }
      // On the error path, copies in flight land before the CTA may exit.
      if (*abort_f)
        for (int i = 0; i < STAGES; ++i)
          for (uint32_t parity = 0; parity < 2; ++parity) attn::drain_phase(&B->full[i], parity);
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
                        const ChunkArgs& C, int grid, void* stream) {
  using Sh = ChunkShape<DKP, DVP>;
  static std::mutex mu;
  static bool done[64] = {};
  const void* fn = reinterpret_cast<const void*>(&chunk_kernel<DKP, DVP, STATES>);
  const int st = attn::allow_smem(fn, Sh::SMEM, done, mu);
  if (st != KB_OK) return st;
  return launch(chunk_kernel<DKP, DVP, STATES>, dim3((unsigned)grid), dim3(THREADS),
                (size_t)Sh::SMEM, stream, mq, mk, mv, C);
}

// Segments of a request: where there are fewer heads of requests than SMs, about two units an
// SM, of 4 chunks at least (a segment but the last is read twice, for its gain and its outputs).
static void segments_of(int64_t heads, int64_t longest, int sms, int& segments, int& segment) {
  const int64_t want = heads < sms ? (2 * sms + heads - 1) / heads : 1;
  int64_t each = ((longest + want - 1) / want + CHUNK - 1) / CHUNK * CHUNK;
  if (each < 4 * CHUNK) each = 4 * CHUNK;
  segments = (int)((longest + each - 1) / each);
  segment = (int)each;
}

size_t chunk_workspace(int64_t B, int64_t H, int64_t Dk, int64_t Dv, int64_t longest, int sms) {
  int segments, segment;
  segments_of(B * H, longest, sms, segments, segment);
  return segments > 1 ? (size_t)(B * segments * H) * (Dk * Dv + 1) * sizeof(float) : 0;
}

int launch_chunks(const Args& A, int64_t Hq, int64_t Hk, int sms, void* workspace,
                  size_t workspace_bytes, void* stream) {
  ChunkArgs C = {};
  C.a = A;
  segments_of((int64_t)A.B * A.H, A.longest, sms, C.segments, C.segment);
  const size_t need = chunk_workspace(A.B, A.H, A.Dk, A.Dv, A.longest, sms);
  KB_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), KB_ERR_WORKSPACE,
             "linear attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  C.sums = static_cast<float*>(workspace);
  C.keeps = C.sums + (size_t)A.B * C.segments * A.H * A.Dk * A.Dv;
  CUtensorMap mq, mk, mv;
  int st = attn::make_map_4d(&mq, A.q, 0, {A.Dk, Hq, A.total, 1}, {A.q_head, A.q_tok, 8}, 1,
                             CHUNK);
  if (st == KB_OK)
    st = attn::make_map_4d(&mk, A.k, 0, {A.Dk, Hk, A.total, 1}, {A.k_head, A.k_tok, 8}, 1, CHUNK);
  if (st == KB_OK)
    st = attn::make_map_4d(&mv, A.v, 0, {A.Dv, A.H, A.total, 1}, {A.v_head, A.v_tok, 8}, 1,
                           CHUNK);
  if (st != KB_OK) return st;
  const int grid = (int)std::min<int64_t>((int64_t)A.B * C.segments * A.H, sms);
  for (int pass = C.segments > 1 ? 0 : 1; pass < 2 && st == KB_OK; ++pass) {
    const bool states = pass == 0;
    if (A.Dk <= 64 && A.Dv <= 64)
      st = states ? launch_chunk<64, 64, true>(mq, mk, mv, C, grid, stream)
                  : launch_chunk<64, 64, false>(mq, mk, mv, C, grid, stream);
    else if (A.Dk <= 64)
      st = states ? launch_chunk<64, 128, true>(mq, mk, mv, C, grid, stream)
                  : launch_chunk<64, 128, false>(mq, mk, mv, C, grid, stream);
    else if (A.Dv <= 64)
      st = states ? launch_chunk<128, 64, true>(mq, mk, mv, C, grid, stream)
                  : launch_chunk<128, 64, false>(mq, mk, mv, C, grid, stream);
    else
      st = states ? launch_chunk<128, 128, true>(mq, mk, mv, C, grid, stream)
                  : launch_chunk<128, 128, false>(mq, mk, mv, C, grid, stream);
  }
  return st;
}

}  // namespace linear
}  // namespace kb
