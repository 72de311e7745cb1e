// kb_runs.cuh - how attention over the paged cache is split: all (request, head,
// block of rows, 64-key tile) units lie on one line, cut into equal runs, one per
// CTA, so that any mix of lengths keeps every SM reading to the end.
#pragma once

#include "kb_attn.cuh"

namespace kb {
namespace attn {

constexpr int KT = 64;                     // keys of a tile
constexpr size_t ZEROED = 4096;            // bytes at a workspace's start that callers zero
constexpr int MIN_TILES = 2;               // tiles that make another CTA worth its partial sums

// A request: its rows, context, tiles of KT keys and blocks of rows.
struct Request {
  int64_t first, ctx, tiles;
  int n, blocks;
};

// The request a run starts in, and where its tiles start on the line.
struct RunStart {
  Request r;
  int64_t base;
  int b;
  int64_t scan[16];         // of find_run
};

// Lengths on the line.  A unit counts `cost` tiles more than it has, for its start
// and its end.  Places past the table have no keys and no tiles, so a length that is
// wrong costs no more than the table's; contexts count up to MAX_CONTEXT (places and
// their tiles stay within 32 bits).
constexpr int MAX_CONTEXT = (1 << 30) - 2 * KT, MAX_PLACES = 0x7fffffff - KT;
struct Lengths {
  const int *cu, *context;
  int64_t total;
  int places;               // of a table's row
  int g, heads, rows, most; // query heads of a key/value head; rows of a block; tokens at most
  int cost;
  __device__ __forceinline__ Request look(int b) const {
    Request R;
    int64_t end;
    const int ctx = min(max(context[b], 0), MAX_CONTEXT);
    request_rows(cu, b, total, R.first, end);
    R.n = (int)min(end - R.first, (int64_t)most);
    R.ctx = ctx;
    R.tiles = R.n ? max((min(ctx + R.n, places) + KT - 1) / KT, 1) : 0;
    R.blocks = (int)(((int64_t)R.n * g + rows - 1) / rows);
    return R;
  }
  __device__ __forceinline__ int64_t length(const Request& R) const {
    return R.n ? (R.tiles + cost) * R.blocks * heads : (int64_t)0;
  }
};

// Quotient of non-negative numbers; the 64-bit division takes most of a
// microsecond of a producer's start.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// Places [lo, hi) of a line of `total` are this CTA's, one of `ctas`.
struct Run {
  int64_t lo, hi, total;
  int ctas;
  __device__ __forceinline__ int of(int64_t place) const {      // the CTA that has a place
    return (int)quotient((place + 1) * ctas - 1, total);
  }
};

// The part of a unit that a run has from `pos` on: head, block of rows, tiles
// [t0, t1) (none if the run ends in the unit's start), the CTAs that share it.
struct RunPart {
  int64_t t0, t1, until;
  int hk, block, c0, parts;
};

__device__ __forceinline__ RunPart run_part(const Request& R, int64_t pos, int64_t base,
                                            const Run& run, int cost) {
  RunPart P;
  const int64_t len = R.tiles + cost;
  const int unit = (int)quotient(pos - base, len);
  P.hk = unit / R.blocks;
  P.block = unit - P.hk * R.blocks;
  const int64_t u0 = base + unit * len + cost;     // where the unit's first tile is
  P.until = min(run.hi, u0 + R.tiles);
  P.t0 = max(pos - u0, (int64_t)0);
  P.t1 = P.until - u0;
  P.c0 = run.of(u0);
  P.parts = run.of(u0 + R.tiles - 1) - P.c0 + 1;
  return P;
}

// All threads of the CTA: the line's length, this CTA's run, and in `start` (shared
// memory, valid on return) the request it starts in.  Tokens past the table are recorded.
template <int THREADS>
__device__ __forceinline__ Run find_run(const Lengths& L, int B, RunStart* start, uint32_t* err) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int WARPS = THREADS / 32;
  static_assert(WARPS <= 16, "a sum for each warp");
  const int per = (B + THREADS - 1) / THREADS;
  const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
  int64_t mine = 0;
  Request R0 = {};
  for (int b = b0; b < b1; ++b) {
    const Request R = L.look(b);
    if (b == b0) R0 = R;
    mine += L.length(R);
    if (blockIdx.x == 0 && R.n && (int)R.ctx + R.n > L.places) atomicOr(err, ERR_PAGE);
  }
  int64_t incl = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) start->scan[warp] = incl;
  __syncthreads();
  int64_t excl = incl - mine;
  Run run = {0, 0, 0, 1};
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) excl += start->scan[w];
    run.total += start->scan[w];
  }
  run.ctas = (int)min((int64_t)gridDim.x,
                      max((run.total + MIN_TILES - 1) / MIN_TILES, (int64_t)1));
  if ((int)blockIdx.x < run.ctas && run.total > 0) {
    run.lo = quotient(run.total * blockIdx.x, run.ctas);
    run.hi = quotient(run.total * (blockIdx.x + 1), run.ctas);
    if (mine > 0 && excl <= run.lo && run.lo < excl + mine) {
      int64_t at = excl;
      for (int b = b0; b < b1; ++b) {
        if (b > b0) R0 = L.look(b);
        const int64_t w = L.length(R0);
        if (run.lo < at + w) {
          start->r = R0;
          start->base = at;
          start->b = b;
          break;
        }
        at += w;
      }
    }
  }
  __syncthreads();
  return run;
}

// Page ids of a tile's pages in lanes 0.. (-1: none in the cache), for keys from
// `key` of request b, which has `end`; 32 table entries from `have` on (-1: none
// yet) are held at a time, for keys that only grow.
template <class Args>
__device__ __forceinline__ int page_ids(const Args& A, int b, int64_t end, int64_t key, int& ids,
                                        int& have) {
  const int lane = threadIdx.x & 31;
  const int shift = 31 - __clz(A.ps), pages = max(1, KT >> shift);
  const int entry = (int)(key >> shift);
  if (have < 0 || entry + pages > have + 32) {
    have = entry;
    const int e = have + lane;
    ids = e < A.width && (int64_t)e * A.ps < end ? A.table[(int64_t)b * A.table_stride + e] : -1;
    if (ids >= A.n_pages) ids = -1;
  }
  return __shfl_sync(0xffffffffu, ids, entry - have + min(lane, pages - 1));
}

// What the sums of a part with the maximum m (log2) count in sums relative to t, at least
// m.  Where neither saw a score above -infinity both count as they are: their sums are
// zero, or not a number where their scores were, and that has to stay.
__device__ __forceinline__ float part_factor(float m, float t) {
  return t == -INFINITY ? 1.f : exp2_fast(m - t);
}

// What the tensor-core form for many rows needs of a tree attention call.
struct TreeCall {
  const uint16_t *q, *k, *v;
  int64_t q_tok, q_head, k_page, k_row, k_head, v_page, v_row, v_head;
  uint16_t* out;
  float* lse;
  const int *cu, *table, *context;
  const int64_t* mask;
  int64_t table_stride, n_pages, total;
  int B, width, ps, places, Hq, Hkv, Dk, Dv, f16, most;
  float scale2;
  uint32_t* err;
};
// `rows`: tokens x heads of a group, of the request with most.
size_t rows_workspace(int64_t rows);
int launch_rows(const TreeCall& T, int64_t rows, int sms, void* workspace, void* stream);

}  // namespace attn
}  // namespace kb
