// kb_tree.cu - attention of this step's tokens (one each, or drafted trees)
// over the paged cache.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / l_i,  s_ij = scale * q_i . k_j over the visible j,
//   m_i = max_j s_ij, l_i = sum_j exp(s_ij - m_i), lse_i = m_i + log(l_i)
// visible: j < context, or bit j - context of the token's tree word (without
// words: j <= context + i).  A row that sees no key gives 0 and lse -infinity.
//
// Every cached key and value is read once and meets few rows (tokens x heads
// of a group), so the bytes of the cache bound the work.  The rows of one
// (request, key/value head), at most 16 here, are one A operand of the warp-level
// matrix instruction, whose results the softmax has in registers; the 5th-generation
// tensor core would spend 7/8 of its 128-row tile on padding.
//
// Work split.  All (request, head, row block, 64-key tile) units form one line
// of tiles, cut into equal runs, one per CTA: any mix of lengths keeps every SM
// reading to the end.  A (request, head, block) whose tiles fall to several
// CTAs is joined from their fp32 partial sums by the CTA that finishes last
// (in CTA order, so results do not change from run to run).
//
// Measured: 32 requests of 512 to 8192 tokens, 32 heads of 192 + 128: 315 us, 6.56
// TB/s (the measured copy bandwidth); one request of 4096: 23 us, of which its bytes
// are 12.8; the rest is a start of dependent loads and the joining of 9 parts a head.
//
// A CTA: one producer warp walks the run, looks pages up (32 table entries at a
// time) and brings each tile in by tensor copies in the 128-byte swizzle (box:
// one page's rows, 64 elements), several tiles ahead; the rows of q come the
// same way, one row a copy.  Four consumer warps: each takes 16 of the tile's keys
// with its own running maximum and sum in registers, so no barrier among them is
// needed until the unit's or the run's end.
//
// Rows of a page past the request's end were never written and may hold
// anything: they are masked as keys and zeroed as values.  A value that is
// infinite or not a number in a hidden drafted token must not meet a zero
// weight: such elements are zeroed in the tile, and at the end the rows that
// see them take them from the cache.
#include <algorithm>

#include "kb_runs.cuh"

namespace kb {
namespace attn {

constexpr int CHUNK = KT * 128;            // bytes of 64 keys x 64 elements
constexpr int UNIT_COST = 2;               // a unit's start and end, in tiles
constexpr int MAX_CTAS = 320;              // counters in the workspace

struct TreeArgs {
  const uint16_t* q;
  int64_t q_tok, q_head;
  uint16_t* out;            // [total, Hq, Dv] contiguous
  float* lse;               // [total, Hq] or NULL
  const uint16_t* v;        // the value cache, for values that are no numbers
  int64_t v_page, v_row, v_head;
  const int* cu;
  const int* table;
  int64_t table_stride;
  const int* context;
  const int64_t* mask;
  int64_t n_pages, total;
  int B, width, ps, Hq, Hkv, g, Dk, Dv;
  int places;               // of a table's row, up to MAX_PLACES
  int most;                 // tokens of a request at most
  float scale2;             // scale * log2(e)
  int* counters;            // [MAX_CTAS], zero between calls
  float* part_ml;           // [2 * CTAs][rows][2]: m (log2), l
  float* part_o;            // [2 * CTAs][rows][DVP]
  uint32_t* err;
};

// What the consumers need to know about the run's part of one unit.
struct Segment {
  int64_t first;            // first row (token) of the request
  int64_t ctx;              // cached tokens before this step's
  int64_t t0, t1;           // tiles of the unit
  int b, n;                 // request; this step's tokens
  int hk, row0, rows;       // head, first row of the block (token * g + head), rows in it
  int whole;                // the run holds all of the unit's tiles
  int starts;               // ... its first tile
  int end;                  // no segment: the run is over
  int c0, parts;            // the CTAs that share the unit: first, number
};

template <int DKP, int DVP>
struct TreeShape {
  static constexpr int RB = 16;                            // rows of a unit
  static constexpr int NW = 4;                             // consumer warps, sharing a tile's keys
  static constexpr int KPW = KT / NW;                      // keys of a warp
  static constexpr int THREADS = (NW + 1) * 32;
  static constexpr int KC = DKP / 64, VC = DVP / 64;
  static constexpr int STAGE = (KC + VC) * CHUNK;
  static constexpr int QP = DKP * 2 + 16;                  // row pitch of q: no bank conflicts
  static constexpr int Q_BYTES = RB * QP;
  static constexpr int X_BYTES = NW / 2 * 32 * (DVP / 2 + 4) * 4;
  static constexpr int CTAS_PER_SM = 2;
  static constexpr int BUDGET = 113 * 1024;
  static constexpr int FIXED = 2 * Q_BYTES + X_BYTES + 1024 + 2048;   // alignment, barriers
  static constexpr int FIT = (BUDGET - FIXED) / STAGE;
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int SMEM = FIXED + STAGES * STAGE;
  static_assert(STAGES >= 2, "two tiles in flight at least");
};

template <int STAGES>
struct TreeBars {
  uint64_t full[STAGES], empty[STAGES];
  uint64_t q_full[2], q_empty[2];
  uint64_t all;               // consumer warps together
  uint64_t valid[STAGES];     // which keys of the tile exist
  int64_t key0[STAGES];       // first key of the tile
  int last[STAGES];           // last tile of its segment
  Segment seg[2];
  int odd[2];                 // a value of the segment's step is no number
  RunStart start;
  int abort_flag, joined;
};

template <int DKP, int DVP, bool F16>
__global__ void __launch_bounds__(TreeShape<DKP, DVP>::THREADS,
                                  TreeShape<DKP, DVP>::CTAS_PER_SM)
    tree_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                const TreeArgs A) {
  using S = TreeShape<DKP, DVP>;
  using Bars = TreeBars<S::STAGES>;
  static_assert(sizeof(Bars) <= 2048, "barrier block");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      smem_raw + ((1024u - (static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw)) & 1023u)) &
                  1023u);
  uint8_t* ring = smem;                                       // [STAGES][K chunks, V chunks]
  uint8_t* qbuf = ring + S::STAGES * S::STAGE;                // [2][RB][QP]
  float* xbuf = reinterpret_cast<float*>(qbuf + 2 * S::Q_BYTES);
  Bars* B = reinterpret_cast<Bars*>(qbuf + 2 * S::Q_BYTES + S::X_BYTES);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_f = &B->abort_flag;

  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&B->full[i], 1);
      mbar_init(&B->empty[i], S::NW);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B->q_full[i], 1);
      mbar_init(&B->q_empty[i], S::NW);
    }
    mbar_init(&B->all, S::NW);
    B->abort_flag = 0;
    B->odd[0] = B->odd[1] = 0;
    mbar_fence_init();
    prefetch_map(&tk);
    prefetch_map(&tv);
  }
  // Columns of q past the head's width stay zero (the copies do not write them).
  if (A.Dk < DKP) {
    for (int i = tid; i < 2 * S::Q_BYTES / 16; i += S::THREADS)
      reinterpret_cast<uint4*>(qbuf)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async();
  }
  pdl_wait();
  pdl_launch_dependents();

  const Lengths L = {A.cu, A.context, A.total, A.places, A.g,
                     A.Hkv, S::RB, A.most, UNIT_COST};
  const Run run = find_run<S::THREADS>(L, A.B, &B->start, A.err);
  // Rows outside every request: zero.
  {
    const int64_t lead = min(max((int64_t)A.cu[0], (int64_t)0), A.total);
    const int64_t tail = min(max((int64_t)A.cu[A.B], lead), A.total);
    const int64_t spare = (lead + A.total - tail) * A.Hq;
    for (int64_t i = (int64_t)blockIdx.x * S::THREADS + tid; i < spare;
         i += (int64_t)gridDim.x * S::THREADS) {
      const int64_t r = i < lead * A.Hq ? i : i - lead * A.Hq + tail * A.Hq;
      for (int d = 0; d < A.Dv; d += 8)
        *reinterpret_cast<uint4*>(A.out + r * A.Dv + d) = make_uint4(0, 0, 0, 0);
      if (A.lse) A.lse[r] = -INFINITY;
    }
  }
  const int cta = blockIdx.x;
  if (run.lo >= run.hi) return;

  if (warp == S::NW) {
    // ---------------------------------------------------------------- producer
    const uint64_t pol = l2_evict_first_policy();
    const int ps = A.ps, box = min(ps, KT), ppt = KT / box;
    int64_t pos = run.lo, base = B->start.base;
    Request R = B->start.r;
    int b = B->start.b, seg = 0, stage = 0;
    uint32_t phase = 0;
    bool ok = true, again = false;
    while (pos < run.hi && ok) {
      const int64_t w = L.length(R);
      if (pos >= base + w) {
        base += w;
        R = L.look(++b);
        continue;
      }
      const RunPart P = run_part(R, pos, base, run, UNIT_COST);
      const int64_t t0 = P.t0, t1 = P.t1;
      const int hk = P.hk;
      pos = P.until;
      if (t1 <= t0) continue;                           // the run ends in the unit's start
      const int sb = seg & 1;
      if (seg >= 2 && !warp_wait(&B->q_empty[sb], ((seg >> 1) - 1) & 1, abort_f, A.err)) break;
      const int row0 = P.block * S::RB;
      const int rows = (int)min((int64_t)S::RB, (int64_t)R.n * A.g - row0);
      if (lane == 0) {
        Segment& G = B->seg[sb];
        G.first = R.first;
        G.ctx = R.ctx;
        G.b = b;
        G.n = R.n;
        G.t0 = t0;
        G.t1 = t1;
        G.hk = hk;
        G.row0 = row0;
        G.rows = rows;
        G.whole = t0 == 0 && t1 == R.tiles;
        G.starts = t0 == 0;
        G.c0 = P.c0;
        G.parts = P.parts;
        G.end = 0;
        mbar_arrive_expect_tx(&B->q_full[sb], (uint32_t)(rows * A.Dk * 2));
      }
      __syncwarp();
      for (int r = lane; r < rows; r += 32) {
        const int tok = (row0 + r) / A.g, h = row0 + r - tok * A.g;
        bulk_g2s(qbuf + sb * S::Q_BYTES + r * S::QP,
                 A.q + (R.first + tok) * A.q_tok + (int64_t)(hk * A.g + h) * A.q_head,
                 (uint32_t)(A.Dk * 2), &B->q_full[sb], pol);
      }
      const int64_t end = R.ctx + R.n;
      int have = -1, ids = -1;   // table entries held by the lanes
      for (int64_t tile = t0; tile < t1; ++tile) {
        if (again && !warp_wait(&B->empty[stage], phase ^ 1u, abort_f, A.err)) {
          ok = false;
          break;
        }
        const int64_t key0 = tile * KT;
        const int mine_id = page_ids(A, b, end, key0, ids, have);
        const unsigned live = __ballot_sync(0xffffffffu, lane < ppt && mine_id >= 0);
        const int64_t left = end - key0;
        uint64_t valid = left >= KT ? ~0ull : (1ull << left) - 1ull;
        if (live != (ppt == 32 ? 0xffffffffu : (1u << ppt) - 1u)) {
          uint64_t got = 0;
          for (int i = 0; i < ppt; ++i)
            if ((live >> i) & 1)
              got |= (box == 64 ? ~0ull : ((1ull << box) - 1ull)) << (i * box);
          if (lane == 0 && (valid & ~got)) atomicOr(A.err, ERR_PAGE);
          valid &= got;
        }
        if (lane == 0) {
          B->valid[stage] = valid;
          B->key0[stage] = key0;
          B->last[stage] = tile + 1 == t1;
          mbar_arrive_expect_tx(&B->full[stage],
                                (uint32_t)(__popc(live) * box * 128 * (S::KC + S::VC)));
        }
        __syncwarp();
        // One copy per page and 64-element column block.
        uint8_t* dst = ring + stage * S::STAGE;
        const int row = ppt > 1 ? 0 : (int)(key0 & (ps - 1));
        for (int i0 = 0; i0 < ppt * (S::KC + S::VC); i0 += 32) {
          const int i = i0 + lane;
          const int p = min(i / (S::KC + S::VC), ppt - 1), c = i - p * (S::KC + S::VC);
          const int id = __shfl_sync(0xffffffffu, mine_id, p);
          if (i >= ppt * (S::KC + S::VC) || !((live >> p) & 1)) continue;
          if (c < S::KC)
            tma_load_4d(dst + c * CHUNK + p * box * 128, &tk, c * 64, row, hk, id,
                        &B->full[stage], pol);
          else
            tma_load_4d(dst + c * CHUNK + p * box * 128, &tv, (c - S::KC) * 64, row, hk, id,
                        &B->full[stage], pol);
        }
        __syncwarp();
        if (++stage == S::STAGES) {
          stage = 0;
          phase ^= 1u;
          again = true;
        }
      }
      ++seg;
    }
    if (seg < 2 || warp_wait(&B->q_empty[seg & 1], ((seg >> 1) - 1) & 1, abort_f, A.err)) {
      if (lane == 0) {
        B->seg[seg & 1].end = 1;
        mbar_arrive(&B->q_full[seg & 1]);
      }
    }
    // On the error path, copies in flight land before the CTA may exit.
    if (*abort_f) {
      for (int i = 0; i < S::STAGES; ++i) {
        drain_phase(&B->full[i], 0);
        drain_phase(&B->full[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        drain_phase(&B->q_full[i], 0);
        drain_phase(&B->q_full[i], 1);
      }
    }
    return;
  }

  // ------------------------------------------------------------------ consumers
  int stage = 0, seg = 0;
  uint32_t phase = 0;
  const int frow = lane >> 2, fcol = (lane & 3) * 2;     // accumulator row and column
  // Barriers among consumer warps, bounded like every wait.
  uint32_t all_phase = 0;
  auto meet = [&](uint64_t* bar, uint32_t& ph) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
    const bool ok = warp_wait(bar, ph, abort_f, A.err);
    ph ^= 1u;
    return ok;
  };
  for (;; ++seg) {
    const int sb = seg & 1;
    if (!warp_wait(&B->q_full[sb], (seg >> 1) & 1, abort_f, A.err)) return;
    const Segment& G = B->seg[sb];     // the producer waits for q_empty to reuse it
    if (G.end) return;
    const int64_t ctx = G.ctx;
    uint32_t qf[DKP / 16][4];
    {
      const uint32_t base = smem_addr(qbuf + sb * S::Q_BYTES) +
                            (uint32_t)(((lane & 15)) * S::QP + (lane >> 4) * 16);
#pragma unroll
      for (int k = 0; k < DKP / 16; ++k) ldmatrix_x4(qf[k], base + k * 32);
    }
    // The tree words of this thread's two rows.
    int tok[2];
    uint64_t word[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = frow + i * 8;
      tok[i] = (G.row0 + min(r, G.rows - 1)) / A.g;
      word[i] = A.mask ? (uint64_t)A.mask[G.first + tok[i]] : 0;
    }
    auto sees = [&](int i, int64_t key) {
      const int64_t j = key - ctx;
      if (j < 0) return true;
      return A.mask ? (j < 64 && ((word[i] >> j) & 1)) : j <= tok[i];
    };
    float o[DVP / 8][4];
#pragma unroll
    for (int i = 0; i < DVP / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (bool last = false; !last;) {
      if (!warp_wait(&B->full[stage], phase, abort_f, A.err)) return;
      last = B->last[stage] != 0;
      const uint64_t valid = B->valid[stage];
      const int64_t key0 = B->key0[stage];
      const bool step_keys = key0 + KT > ctx;
      uint8_t* kt = ring + stage * S::STAGE;
      uint8_t* vt = kt + S::KC * CHUNK;
      float s[S::KPW / 8][4];
#pragma unroll
      for (int i = 0; i < S::KPW / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll
      for (int k = 0; k < DKP / 16; ++k) {
#pragma unroll
        for (int n = 0; n < S::KPW / 16; ++n) {
          const int row = warp * S::KPW + n * 16 + (lane & 7) + ((lane >> 4) & 1) * 8;
          const int piece = (k & 3) * 2 + ((lane >> 3) & 1);
          uint32_t b[4];
          ldmatrix_x4(b, smem_addr(kt) + (uint32_t)((k >> 2) * CHUNK + row * 128 +
                                                    ((piece ^ (row & 7)) << 4)));
          mma_16816<F16>(s[2 * n], qf[k], b[0], b[1]);
          mma_16816<F16>(s[2 * n + 1], qf[k], b[2], b[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < S::KPW / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] *= A.scale2;
      if (step_keys || valid != ~0ull) {
#pragma unroll
        for (int i = 0; i < S::KPW / 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = warp * S::KPW + i * 8 + fcol + (j & 1);
            if (!((valid >> c) & 1) || !sees(j >> 1, key0 + c)) s[i][j] = -INFINITY;
          }
        // Values of keys that do not exist become zero, and so do elements of
        // this step's values that are no numbers (noted for the end).  Each warp
        // does so for its own 16 keys, which no other reads.
        const bool scan = step_keys && (G.n > 1 || A.mask);
        const uint32_t there = (uint32_t)(valid >> (warp * S::KPW));
        bool wrote = false;
        if (scan || valid != ~0ull)
#pragma unroll 4
          for (int x = lane; x < S::KPW * (DVP / 8); x += 32) {
            const int r = x / (DVP / 8), c = warp * S::KPW + r, piece = x - r * (DVP / 8);
            uint4* at = reinterpret_cast<uint4*>(vt + (piece >> 3) * CHUNK + c * 128 +
                                                 (((piece & 7) ^ (c & 7)) << 4));
            if (!((there >> r) & 1)) {
              *at = make_uint4(0, 0, 0, 0);
              wrote = true;
            } else if (scan && key0 + c >= ctx) {
              uint4 v = *at;
              if (has_odd<F16>(v)) {
                clear_odd<F16>(v);
                B->odd[sb] = 1;
                *at = v;
                wrote = true;
              }
            }
          }
        if (__any_sync(0xffffffffu, wrote)) fence_proxy_async();   // before the next copy
        __syncwarp();
      }
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int i = 0; i < S::KPW / 8; ++i) {
        top[0] = fmaxf(top[0], fmaxf(s[i][0], s[i][1]));
        top[1] = fmaxf(top[1], fmaxf(s[i][2], s[i][3]));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      }
      if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
        float fix[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          fix[i] = top[i] == -INFINITY ? 1.f : exp2_fast(m[i] - top[i]);
          l[i] *= fix[i];
          m[i] = top[i];
        }
#pragma unroll
        for (int i = 0; i < DVP / 8; ++i) {
          o[i][0] *= fix[0];
          o[i][1] *= fix[0];
          o[i][2] *= fix[1];
          o[i][3] *= fix[1];
        }
      }
      const float at0 = m[0] == -INFINITY ? 0.f : m[0], at1 = m[1] == -INFINITY ? 0.f : m[1];
      uint32_t p[S::KPW / 16][4];
#pragma unroll
      for (int i = 0; i < S::KPW / 8; ++i) {
        const float e0 = exp2_fast(s[i][0] - at0), e1 = exp2_fast(s[i][1] - at0);
        const float e2 = exp2_fast(s[i][2] - at1), e3 = exp2_fast(s[i][3] - at1);
        l[0] += e0 + e1;
        l[1] += e2 + e3;
        // One rounding of the weights, to the type the tensor core multiplies.
        p[i >> 1][(i & 1) * 2] = pack2<F16>(e0, e1);
        p[i >> 1][(i & 1) * 2 + 1] = pack2<F16>(e2, e3);
      }
#pragma unroll
      for (int n = 0; n < S::KPW / 16; ++n) {
        const int row = warp * S::KPW + n * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int i = 0; i < DVP / 16; ++i) {
          const int piece = (i & 3) * 2 + (lane >> 4);
          uint32_t b[4];
          ldmatrix_x4_trans(b, smem_addr(vt) + (uint32_t)((i >> 2) * CHUNK + row * 128 +
                                                          ((piece ^ (row & 7)) << 4)));
          mma_16816<F16>(o[2 * i], p[n], b[0], b[1]);
          mma_16816<F16>(o[2 * i + 1], p[n], b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&B->empty[stage]);
      if (++stage == S::STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }

    // Join the warps that shared the keys: half of them hand over, then half
    // of the rest.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    constexpr int XF = DVP / 2 + 4;
    const bool upper = G.rows > 8;      // rows in the second half of the 16
#pragma unroll
    for (int half = S::NW / 2; half >= 1; half >>= 1) {
      float* x = xbuf + (size_t)(warp & (half - 1)) * 32 * XF + lane;
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int i = 0; i < DVP / 8; ++i) {
          x[(i * 4) * 32] = o[i][0];
          x[(i * 4 + 1) * 32] = o[i][1];
        }
        if (upper)
#pragma unroll
          for (int i = 0; i < DVP / 8; ++i) {
            x[(i * 4 + 2) * 32] = o[i][2];
            x[(i * 4 + 3) * 32] = o[i][3];
          }
        x[(XF - 4) * 32] = m[0];
        x[(XF - 3) * 32] = m[1];
        x[(XF - 2) * 32] = l[0];
        x[(XF - 1) * 32] = l[1];
      }
      if (!meet(&B->all, all_phase)) return;
      if (warp < half) {
        float f0[2], f1[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float om = x[(XF - 4 + i) * 32], ol = x[(XF - 2 + i) * 32];
          const float t = fmaxf(m[i], om);
          f0[i] = part_factor(m[i], t);
          f1[i] = part_factor(om, t);
          m[i] = t;
          l[i] = l[i] * f0[i] + ol * f1[i];
        }
#pragma unroll
        for (int i = 0; i < DVP / 8; ++i) {
          o[i][0] = o[i][0] * f0[0] + x[(i * 4) * 32] * f1[0];
          o[i][1] = o[i][1] * f0[0] + x[(i * 4 + 1) * 32] * f1[0];
        }
        if (upper)
#pragma unroll
          for (int i = 0; i < DVP / 8; ++i) {
            o[i][2] = o[i][2] * f0[1] + x[(i * 4 + 2) * 32] * f1[1];
            o[i][3] = o[i][3] * f0[1] + x[(i * 4 + 3) * 32] * f1[1];
          }
      }
      if (!meet(&B->all, all_phase)) return;
    }

    if (warp == 0) {
      if (B->odd[sb]) {
        // Values that are no numbers, from the cache, to the rows that see them.
        for (int64_t key = max(ctx, G.t0 * KT); key < min(ctx + G.n, G.t1 * KT); ++key) {
          const int64_t e = key / A.ps;
          const int id = e < A.width ? A.table[(int64_t)G.b * A.table_stride + e] : -1;
          if (id < 0 || id >= A.n_pages) continue;
          const uint16_t* v = A.v + id * A.v_page + (key - e * A.ps) * A.v_row + G.hk * A.v_head;
          const bool s0 = sees(0, key), s1 = sees(1, key);
#pragma unroll
          for (int i = 0; i < DVP / 8; ++i)
            for (int j = 0; j < 2 && i * 8 < A.Dv; ++j) {
              const uint16_t u = v[i * 8 + fcol + j];
              if (!odd_element<F16>(u)) continue;
              if (s0) o[i][j] += element<F16>(u);
              if (s1) o[i][2 + j] += element<F16>(u);
            }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = frow + h * 8;
        if (r >= G.rows) continue;
        if (G.whole) {
          const int t = (G.row0 + r) / A.g;
          const int64_t at = (G.first + t) * A.Hq + G.hk * A.g + (G.row0 + r - t * A.g);
          const float inv = l[h] > 0.f ? 1.f / l[h] : l[h] == 0.f ? 0.f : l[h];
          uint16_t* out = A.out + at * A.Dv;
#pragma unroll
          for (int i = 0; i < DVP / 8; ++i)
            if (i * 8 < A.Dv)
              *reinterpret_cast<uint32_t*>(out + i * 8 + fcol) =
                  pack2<F16>(o[i][2 * h] * inv, o[i][2 * h + 1] * inv);
          if (A.lse && (lane & 3) == 0)
            A.lse[at] = l[h] == 0.f ? -INFINITY : (m[h] + log2f(l[h])) * LN2;
        } else {
          const int64_t slot = ((int64_t)cta * 2 + G.starts) * S::RB + r;
          float* po = A.part_o + slot * DVP;
#pragma unroll
          for (int i = 0; i < DVP / 8; ++i)
            *reinterpret_cast<float2*>(po + i * 8 + fcol) =
                make_float2(o[i][2 * h], o[i][2 * h + 1]);
          if ((lane & 3) == 0)
            *reinterpret_cast<float2*>(A.part_ml + slot * 2) = make_float2(m[h], l[h]);
        }
      }
    }
    if (!G.whole) {
      // The last of the unit's CTAs joins their sums, in CTA order.
      __threadfence();
      if (!meet(&B->all, all_phase)) return;
      if (tid == 0) {
        const int old = atomicAdd(&A.counters[G.c0], 1);
        B->joined = old == G.parts - 1;
        if (B->joined) A.counters[G.c0] = 0;
      }
      if (!meet(&B->all, all_phase)) return;
      if (B->joined) {
        __threadfence();
        // Few items: several threads share an item's partial sums.
        constexpr int T = S::NW * 32;
        const int quads = A.Dv / 4, items = G.rows * quads;
        int share = 1;
        while (share < 32 && share * 2 * items <= T) share *= 2;
        for (int base = 0; base < items; base += T / share) {
          const int it = base + tid % (T / share), sh = tid / (T / share);
          const int r = min(it, items - 1) / quads, d = (min(it, items - 1) - r * quads) * 4;
          float tm = -INFINITY, tl = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
          for (int c = sh; c < G.parts; c += 4 * share) {
            float2 ml[4];
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int cc = c + u * share;
              ml[u] = make_float2(-INFINITY, 0.f);
              v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (cc < G.parts) {
                const int64_t slot = ((int64_t)(G.c0 + cc) * 2 + (cc == 0)) * S::RB + r;
                ml[u] = __ldcg(reinterpret_cast<const float2*>(A.part_ml + slot * 2));
                v[u] = __ldcg(reinterpret_cast<const float4*>(A.part_o + slot * DVP + d));
              }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const float t = fmaxf(tm, ml[u].x);
              const float f0 = part_factor(tm, t), f1 = part_factor(ml[u].x, t);
              tm = t;
              tl = tl * f0 + ml[u].y * f1;
              acc[0] = acc[0] * f0 + v[u].x * f1;
              acc[1] = acc[1] * f0 + v[u].y * f1;
              acc[2] = acc[2] * f0 + v[u].z * f1;
              acc[3] = acc[3] * f0 + v[u].w * f1;
            }
          }
          if (share > 1) {
            // Through shared memory, in order.
            float* x = xbuf + tid * 6;
            x[0] = tm;
            x[1] = tl;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[2 + j] = acc[j];
            if (!meet(&B->all, all_phase)) return;
            if (sh == 0)
              for (int u = 1; u < share; ++u) {
                const float* y = xbuf + (tid + u * (T / share)) * 6;
                const float t = fmaxf(tm, y[0]);
                const float f0 = part_factor(tm, t), f1 = part_factor(y[0], t);
                tm = t;
                tl = tl * f0 + y[1] * f1;
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = acc[j] * f0 + y[2 + j] * f1;
              }
            if (!meet(&B->all, all_phase)) return;
          }
          if (sh == 0 && it < items) {
            const int t = (G.row0 + r) / A.g;
            const int64_t at = (G.first + t) * A.Hq + G.hk * A.g + (G.row0 + r - t * A.g);
            const float inv = tl > 0.f ? 1.f / tl : tl == 0.f ? 0.f : tl;
            uint2 w;
            w.x = pack2<F16>(acc[0] * inv, acc[1] * inv);
            w.y = pack2<F16>(acc[2] * inv, acc[3] * inv);
            *reinterpret_cast<uint2*>(A.out + at * A.Dv + d) = w;
            if (A.lse && d == 0) A.lse[at] = tl == 0.f ? -INFINITY : (tm + log2f(tl)) * LN2;
          }
        }
      }
    }
    // Everyone is done with the segment and the exchange buffer.
    if (B->odd[sb]) {
      if (!meet(&B->all, all_phase)) return;
      if (tid == 0) B->odd[sb] = 0;
    }
    if (!meet(&B->all, all_phase)) return;
    if (lane == 0) mbar_arrive(&B->q_empty[sb]);
  }
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------

// Rows (tokens x heads of a group) up to which the warp-level matrix steps are
// used; more rows go to the 5th-generation tensor cores (kb_prompt.cu), which pad
// to 128.  Measured (replayed, us, here / there):
//   16 rows: 16 requests of 2048, 8 key/value heads of 128: 35 / 47, of 64: 23 / 44;
//     64 requests of 1024: 57 / 98; 16 of 2048, 32 heads of 192 + 128: 112 / 141;
//     4 of 16000, 2 heads of 128: 49 / 53;
//   32 rows (two blocks here, which read the keys twice): 53 / 48, 34 / 44, 99 / 98,
//     213 / 161, 45 / 48.
constexpr int64_t MMA_ROWS = 16;

template <int DKP, int DVP, bool F16>
static int launch_tree(const CUtensorMap& mk, const CUtensorMap& mv, TreeArgs& A, int sms,
                       void* stream) {
  using S = TreeShape<DKP, DVP>;
  static std::mutex mu;
  static bool done[64] = {};
  const void* fn = reinterpret_cast<const void*>(&tree_kernel<DKP, DVP, F16>);
  const int st = allow_smem(fn, S::SMEM, done, mu);
  if (st != KB_OK) return st;
  const int grid = std::min(sms * S::CTAS_PER_SM, MAX_CTAS);
  return launch(tree_kernel<DKP, DVP, F16>, dim3(grid), dim3(S::THREADS), (size_t)S::SMEM,
                stream, mk, mv, A);
}

template <int DKP, int DVP>
static int launch_mma(int f16, const CUtensorMap& mk, const CUtensorMap& mv, TreeArgs& A, int sms,
                      void* stream) {
  return f16 ? launch_tree<DKP, DVP, true>(mk, mv, A, sms, stream)
             : launch_tree<DKP, DVP, false>(mk, mv, A, sms, stream);
}

constexpr size_t COUNTER_BYTES = MAX_CTAS * sizeof(int);
static_assert(COUNTER_BYTES <= ZEROED, "counters where callers zero");

// Counters, then two partial sums a CTA (the end of one unit and the start of
// another): maximum and sum of a row, and up to 128 values of it.
static size_t tree_workspace(int64_t rows) {
  if (rows > MMA_ROWS) return rows_workspace(rows);
  return COUNTER_BYTES + (size_t)2 * MAX_CTAS * MMA_ROWS * (2 + 128) * sizeof(float);
}

}  // namespace attn
}  // namespace kb

extern "C" size_t kb_tree_attention_workspace_size(int64_t group, int64_t max_tokens) {
  if (group <= 0 || max_tokens <= 0) return 0;
  return kb::attn::tree_workspace(group * max_tokens);
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
  namespace at = kb::attn;
  kb::clear_error();
  KB_REQUIRE(B >= 0 && total >= 0 && max_tokens >= 0 && n_pages >= 0 && table_width >= 0,
             KB_ERR_BAD_SHAPE, "tree attention: bad shape");
  int st = at::check_heads(Hq, Hkv, Dk, Dv, dtype);
  if (st != KB_OK) return st;
  KB_REQUIRE(page_size >= 8 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
             KB_ERR_UNSUPPORTED, "tree attention: the page size must be a power of two from 8");
  if (B == 0 || total == 0) return KB_OK;
  KB_REQUIRE(scale > 0.f, KB_ERR_BAD_SHAPE, "attention: the scale must be positive");
  KB_REQUIRE(max_tokens > 0 && n_pages > 0, KB_ERR_BAD_SHAPE,
             "tree attention: tokens but max_tokens 0, or a cache without pages");
  KB_REQUIRE(q && k_strides && v_strides && cu_tokens && context_lens && out && k_cache &&
                 v_cache && (table_width == 0 || block_table),
             KB_ERR_NULL_POINTER, "tree attention: NULL pointer");
  KB_REQUIRE(!tree_mask || max_tokens <= 64, KB_ERR_UNSUPPORTED,
             "tree attention: a masked tree has at most 64 tokens");
  constexpr int64_t kMax = (int64_t)1 << 30;
  KB_REQUIRE(B <= kMax && total <= kMax && n_pages <= kMax && table_width <= kMax &&
                 max_tokens * (Hq / Hkv) <= kMax && Hq <= 65535,
             KB_ERR_UNSUPPORTED, "tree attention: more than 2^30 tokens, pages or requests");
  bool ok = (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) == 0 &&
            ((q_token_stride | q_head_stride) & 7) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && ((k_strides[i] | v_strides[i]) & 7) == 0;
  KB_REQUIRE(ok, KB_ERR_ALIGNMENT,
             "tree attention: pointers must be 16-byte aligned and strides multiples of 8");
  const size_t need = kb_tree_attention_workspace_size(Hq / Hkv, max_tokens);
  KB_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0,
             KB_ERR_WORKSPACE,
             "tree attention: workspace of %zu bytes (256-byte aligned, zeroed once) required, "
             "%zu given",
             need, workspace_bytes);
  const int dev = kb::bind_stream_device(stream);
  uint32_t* err = kb::device_error_word(dev);
  KB_REQUIRE(err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  const int sms = kb::num_sms(dev);
  const int64_t block_rows = max_tokens * (Hq / Hkv);
  if (block_rows > at::MMA_ROWS) {
    at::TreeCall T = {};
    T.q = q;
    T.k = k_cache;
    T.v = v_cache;
    T.k_page = k_strides[0];
    T.k_row = k_strides[1];
    T.k_head = k_strides[2];
    T.q_tok = q_token_stride;
    T.q_head = q_head_stride;
    T.v_page = v_strides[0];
    T.v_row = v_strides[1];
    T.v_head = v_strides[2];
    T.out = out;
    T.lse = lse;
    T.cu = cu_tokens;
    T.table = block_table;
    T.context = context_lens;
    T.mask = tree_mask;
    T.table_stride = table_stride;
    T.n_pages = n_pages;
    T.total = total;
    T.B = (int)B;
    T.width = (int)table_width;
    T.ps = (int)page_size;
    T.places = (int)std::min<int64_t>(table_width * page_size, at::MAX_PLACES);
    T.Hq = (int)Hq;
    T.Hkv = (int)Hkv;
    T.Dk = (int)Dk;
    T.Dv = (int)Dv;
    T.f16 = dtype;
    T.scale2 = scale * kb::LOG2E;
    T.most = (int)max_tokens;
    T.err = err;
    return at::launch_rows(T, block_rows, sms, workspace, stream);
  }
  const int rows = (int)std::min<int64_t>(page_size, at::KT);
  CUtensorMap mk, mv;
  st = at::make_map_4d(&mk, k_cache, dtype, {Dk, page_size, Hkv, n_pages},
                       {k_strides[1], k_strides[2], k_strides[0]}, rows, 1);
  if (st != KB_OK) return st;
  st = at::make_map_4d(&mv, v_cache, dtype, {Dv, page_size, Hkv, n_pages},
                       {v_strides[1], v_strides[2], v_strides[0]}, rows, 1);
  if (st != KB_OK) return st;
  at::TreeArgs A = {};
  A.q = q;
  A.q_tok = q_token_stride;
  A.q_head = q_head_stride;
  A.v = v_cache;
  A.v_page = v_strides[0];
  A.v_row = v_strides[1];
  A.v_head = v_strides[2];
  A.out = out;
  A.lse = lse;
  A.cu = cu_tokens;
  A.table = block_table;
  A.table_stride = table_stride;
  A.context = context_lens;
  A.mask = tree_mask;
  A.n_pages = n_pages;
  A.total = total;
  A.B = (int)B;
  A.width = (int)table_width;
  A.ps = (int)page_size;
  A.places = (int)std::min<int64_t>(table_width * page_size, at::MAX_PLACES);
  A.Hq = (int)Hq;
  A.Hkv = (int)Hkv;
  A.g = (int)(Hq / Hkv);
  A.Dk = (int)Dk;
  A.Dv = (int)Dv;
  A.scale2 = scale * kb::LOG2E;
  A.counters = static_cast<int*>(workspace);
  A.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + at::COUNTER_BYTES);
  A.part_o = A.part_ml + (size_t)2 * at::MAX_CTAS * at::MMA_ROWS * 2;
  A.most = (int)max_tokens;
  A.err = err;
  if (Dk <= 64 && Dv <= 64) return at::launch_mma<64, 64>(dtype, mk, mv, A, sms, stream);
  if (Dk <= 128) return at::launch_mma<128, 128>(dtype, mk, mv, A, sms, stream);
  return at::launch_mma<192, 128>(dtype, mk, mv, A, sms, stream);
}
