// kb_pages.cu - the pages of a cache as requests come and go: rows of the block table that
// share another row's full pages (fork), pages that no row holds any more (free), used pages
// moved to the lowest places of the pool (compact), and copies of pages.
//
// A page that several rows of the table name is shared; nothing counts its owners.  A page
// is held while a row that keeps it names it, so free and compact read the table (of row b
// the first ceil(reserved_b / ps) entries) and mark pages in bitmaps:
//   free:     gone = given up by some row, and kept by none;
//             free[head - |gone| : head] = the gone pages in ascending order
//   compact:  M = used | free, low = the |used| lowest pages of M;
//             the i-th of used \ low moves to the i-th of free & low
// Both are whole-pool sums, so they run as one cluster of up to 8 CTAs: each marks its share
// of the rows in bitmaps of its own shared memory, then takes its share of the pool and joins
// all CTAs' words of it through distributed shared memory.  Nothing is kept between calls and
// no order of atomics shows: the bitmaps are sets.
//   fork of row s to row t, L = context_s, f = L / ps, r = L % ps:
//   table[t, :f] = table[s, :f]; if r > 0: table[t, f] = the next page of the free list, and
//   the caller copies the first r rows of page table[s, f] there (the copy list).
#include <cooperative_groups.h>

#include "kb_common.cuh"

namespace kb {
namespace pages {

namespace cg = cooperative_groups;

constexpr int THREADS = 256;                 // fork, copy
constexpr int WIDE = 1024;                   // free, compact
constexpr int CLUSTER = 8;
constexpr int MAX_REQUESTS = 12288;
constexpr int MAX_PAGES = 1 << 19;           // two bitmaps and a share: 144 KB at most
constexpr int LONGEST = (1 << 30) - 1;
// One CTA marks as many table entries in the time that a cluster takes to meet.  (Pages given
// back, entries and pages together 4096: 6.3 us alone, 7.3 by eight CTAs; 8192: 7.7 and 7.3;
// 16384: 10.9 and 7.3; 65536: 31 and 9.  Compaction: 8.4 and 11.6, 10 and 11.8, 13.4 and 12, 28
// and 13.4.)
constexpr int64_t ALONE = 8192;

__device__ __forceinline__ int length_of(const int* lens, int b) {
  return min(max(__ldg(lens + b), 0), LONGEST);
}

__device__ __forceinline__ int pages_of(int tokens, int ps) {
  return (int)(((uint32_t)tokens + (uint32_t)ps - 1) / (uint32_t)ps);
}

__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// ---------------------------------------------------------------------------
// Fork.  A CTA takes a pair at a time; each finds for itself which pairs may be made (their
// rows' first namers, in shared memory) and sums the pages of the pairs before its own.
// ---------------------------------------------------------------------------

struct ForkArgs {
  int *context, *reserved;                   // reserved may be NULL
  int* table;
  int64_t table_stride;
  const int *sources, *targets;
  const int *free_pages, *free_head;
  int B, width, n, nfree, ps;
  int *copy_from, *copy_to, *copy_rows, *head_out, *missing;
  uint32_t* err;
};

__global__ void __launch_bounds__(THREADS) fork_kernel(const ForkArgs A) {
  extern __shared__ int first[];             // [B] the first pair that names the row as target
  uint32_t* is_source = reinterpret_cast<uint32_t*>(first + A.B);
  __shared__ int part[3][THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();
  for (int b = tid; b < A.B; b += THREADS) first[b] = A.n;
  for (int b = tid; b < (A.B + 31) / 32; b += THREADS) is_source[b] = 0;
  __syncthreads();
  for (int i = tid; i < A.n; i += THREADS) {
    const int s = __ldg(A.sources + i), t = __ldg(A.targets + i);
    if (s >= A.B || t >= A.B) atomicOr(A.err, ERR_PAGE);
    if (s < 0 || t < 0 || s >= A.B || t >= A.B) continue;
    atomicMin(&first[t], i);
    atomicOr(&is_source[s >> 5], 1u << (s & 31));
  }
  __syncthreads();
  // What pair i asks for: 0 nothing, 1 a page, -1 more places than a row has, -2: skipped.
  // (A target's context is never read: no target is a source.)
  auto wants = [&](int i, int& s, int& t, int& len) {
    s = __ldg(A.sources + i);
    t = __ldg(A.targets + i);
    len = 0;
    if (s < 0 || t < 0 || s >= A.B || t >= A.B) return -2;
    if (first[t] != i || ((is_source[t >> 5] >> (t & 31)) & 1)) {
      atomicOr(A.err, ERR_PAGE);
      return -2;
    }
    len = length_of(A.context, s);
    if (pages_of(len, A.ps) > A.width) return -1;
    return len % A.ps != 0 ? 1 : 0;
  };
  const int head = max(0, *A.free_head), avail = max(0, A.nfree - head);
  for (int p = blockIdx.x; p < A.n; p += gridDim.x) {
    int before = 0, all = 0, wide = 0, s, t, len;
    for (int i = tid; i < A.n; i += THREADS) {
      const int w = wants(i, s, t, len);
      before += i < p && w == 1;
      all += w == 1;
      wide += w == -1;
    }
    before = warp_sum(before);
    all = warp_sum(all);
    wide = warp_sum(wide);
    if (lane == 0) {
      part[0][warp] = before;
      part[1][warp] = all;
      part[2][warp] = wide;
    }
    __syncthreads();
    before = all = wide = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      before += part[0][w];
      all += part[1][w];
      wide += part[2][w];
    }
    __syncthreads();
    if (p == 0 && tid == 0) {
      *A.head_out = head + min(all, avail);
      *A.missing = max(0, all - avail) + wide;
    }
    const int w = wants(p, s, t, len);
    const bool given = w == 1 && before < avail, made = w == 0 || given;
    const int full = made ? len / A.ps : 0;
    const int fresh = given ? __ldg(A.free_pages + head + before) : -1;
    int* row = A.table + (int64_t)t * A.table_stride;
    const int* from = A.table + (int64_t)s * A.table_stride;
    for (int c = tid; w != -2 && c < A.width; c += THREADS)
      row[c] = c < full ? from[c] : c == full ? fresh : -1;
    if (tid == 0) {
      A.copy_from[p] = given ? from[full] : -1;
      A.copy_to[p] = fresh;
      A.copy_rows[p] = given ? len - full * A.ps : 0;
      if (w != -2) {
        A.context[t] = made ? len : 0;
        if (A.reserved) A.reserved[t] = made ? len : 0;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Free and compact.
// ---------------------------------------------------------------------------

struct PoolArgs {
  const int* table;
  int64_t table_stride;
  const int *reserved, *keep;                // keep: free only
  const int* free_in;                        // compact
  int* free_pages;                           // free: updated in place; compact: the new list
  const int* free_head;
  int B, width, nfree, ps, P;
  int* head_out;
  // Compact.
  int* table_out;                            // [B, width]
  int *copy_from, *copy_to;                  // [P / 2]
  int* map;                                  // [P] scratch: where a moved page goes
  uint32_t* err;
};

struct PoolShared {
  int part[4][WIDE / 32];
  int count[4];                              // of this CTA, read by the others
};

// Sums of up to four numbers a thread over the CTA: each thread's sums of those before it,
// and the whole in S.count.
template <int N>
__device__ __forceinline__ void block_scan(const int (&v)[N], int (&before)[N], PoolShared& S) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int in[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    in[k] = v[k];
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, in[k], o);
      if (lane >= o) in[k] += u;
    }
    if (lane == 31) S.part[k][warp] = in[k];
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      int p = S.part[k][lane];
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, p, o);
        if (lane >= o) p += u;
      }
      if (lane == 31) S.count[k] = p;
      S.part[k][lane] = p - S.part[k][lane];
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) before[k] = S.part[k][warp] + in[k] - v[k];
}

// Sums of the CTAs before this one, and of all.
template <int N>
__device__ __forceinline__ void cluster_scan(int (&before)[N], int (&all)[N], PoolShared& S,
                                             cg::cluster_group& cluster) {
  cluster.sync();
  const int rank = (int)cluster.block_rank(), n = (int)cluster.num_blocks();
#pragma unroll
  for (int k = 0; k < N; ++k) before[k] = all[k] = 0;
  for (int c = 0; c < n; ++c) {
    const int* count = cluster.map_shared_rank(S.count, c);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int v = count[k];
      if (c < rank) before[k] += v;
      all[k] += v;
    }
  }
}

// A bit for each page that the rows name: `second` for columns from keep_b on (free), else
// all in `first`.
template <bool FREE>
__device__ __forceinline__ void mark_rows(const PoolArgs& A, uint32_t* first, uint32_t* second,
                                          int rank, int ctas) {
  // A warp a row; the lengths of its next 32 rows at once, eight loads of a row under way.
  // (2048 rows of up to 250 pages: 12.4 us; with lengths and loads one by one 15.3.)
  constexpr int AT_ONCE = 8;
  const int lane = threadIdx.x & 31, warps = ctas * (WIDE / 32);
  for (int b0 = rank * (WIDE / 32) + (threadIdx.x >> 5); b0 < A.B; b0 += warps * 32) {
    const int mine = b0 + lane * warps;
    int have = 0, keep = 0;
    if (mine < A.B) {
      const int len = length_of(A.reserved, mine);
      have = min(pages_of(len, A.ps), A.width);
      keep = FREE ? pages_of(min(length_of(A.keep, mine), len), A.ps) : have;
    }
    for (int j = 0; j < 32 && b0 + j * warps < A.B; ++j) {
      const int have_j = __shfl_sync(0xffffffffu, have, j);
      const int keep_j = __shfl_sync(0xffffffffu, keep, j);
      const int* row = A.table + (int64_t)(b0 + j * warps) * A.table_stride;
      for (int c0 = lane; c0 < have_j + lane; c0 += 32 * AT_ONCE) {
        int id[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
          id[u] = c0 + 32 * u < have_j ? __ldg(row + c0 + 32 * u) : -1;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
          if (id[u] < 0) continue;
          if (id[u] >= A.P)
            atomicOr(A.err, ERR_PAGE);
          else
            atomicOr((FREE && c0 + 32 * u >= keep_j ? second : first) + (id[u] >> 5),
                     1u << (id[u] & 31));
        }
      }
    }
  }
}

__global__ void __launch_bounds__(WIDE) free_kernel(const PoolArgs A) {
  extern __shared__ uint32_t words[];
  __shared__ PoolShared S;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int W = (A.P + 31) / 32, per = (W + ctas - 1) / ctas;
  uint32_t *kept = words, *gone = words + W, *mine = words + 2 * W;
  for (int i = threadIdx.x; i < 2 * W; i += WIDE) words[i] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  mark_rows<true>(A, kept, gone, rank, ctas);
  cluster.sync();
  // This CTA's share of the pool; each thread a run of its words.
  const int w0 = min(W, rank * per), words_here = min(W, w0 + per) - w0;
  for (int i = threadIdx.x; i < words_here; i += WIDE) {
    uint32_t k = 0, g = 0;
    for (int c = 0; c < ctas; ++c) {
      k |= cluster.map_shared_rank(kept, c)[w0 + i];
      g |= cluster.map_shared_rank(gone, c)[w0 + i];
    }
    mine[i] = g & ~k;
  }
  __syncthreads();
  const int run = (words_here + WIDE - 1) / WIDE;
  const int i0 = min(words_here, (int)threadIdx.x * run), i1 = min(words_here, i0 + run);
  int count[1] = {0}, at[1], ahead[1], all[1];
  for (int i = i0; i < i1; ++i) count[0] += __popc(mine[i]);
  block_scan(count, at, S);
  cluster_scan(ahead, all, S, cluster);
  const int head = min(max(0, *A.free_head), A.nfree);
  if (rank == 0 && threadIdx.x == 0) {
    *A.head_out = max(0, head - all[0]);
    if (all[0] > head) atomicOr(A.err, ERR_PAGE);   // no room in front of the list
  }
  int place = head - all[0] + ahead[0] + at[0];
  for (int i = i0; i < i1; ++i)
    for (uint32_t w = mine[i]; w != 0; w &= w - 1, ++place)
      if (place >= 0) A.free_pages[place] = (w0 + i) * 32 + __ffs(w) - 1;
  cluster.sync();                            // no CTA leaves while its words are read
}

// The lowest n set bits of a word.
__device__ __forceinline__ uint32_t lowest(uint32_t w, int n) {
  if (n <= 0) return 0;
  if (n >= __popc(w)) return w;
  return w & ((1u << __fns(w, 0, n + 1)) - 1u);
}

__global__ void __launch_bounds__(WIDE) compact_kernel(const PoolArgs A) {
  extern __shared__ uint32_t words[];
  __shared__ PoolShared S;
  __shared__ int s_first;                    // the lowest page above the low ones, of this CTA
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int W = (A.P + 31) / 32, per = (W + ctas - 1) / ctas, half = A.P / 2;
  uint32_t *used = words, *spare = words + W, *mine = words + 2 * W;   // mine: [2][per]
  for (int i = threadIdx.x; i < 2 * W; i += WIDE) words[i] = 0;
  if (threadIdx.x == 0) s_first = A.P;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int at0 = rank * WIDE + threadIdx.x, step = ctas * WIDE;
  const int head = min(max(0, *A.free_head), A.nfree);
  mark_rows<false>(A, used, used, rank, ctas);
  for (int i = head + at0; i < A.nfree; i += step) {
    const int id = __ldg(A.free_in + i);
    if (id >= 0 && id < A.P)
      atomicOr(spare + (id >> 5), 1u << (id & 31));
    else if (id >= A.P)
      atomicOr(A.err, ERR_PAGE);
  }
  cluster.sync();
  const int w0 = min(W, rank * per), words_here = min(W, w0 + per) - w0;
  uint32_t *u_mine = mine, *s_mine = mine + per;
  for (int i = threadIdx.x; i < words_here; i += WIDE) {
    uint32_t u = 0, f = 0;
    for (int c = 0; c < ctas; ++c) {
      u |= cluster.map_shared_rank(used, c)[w0 + i];
      f |= cluster.map_shared_rank(spare, c)[w0 + i];
    }
    u_mine[i] = u;
    s_mine[i] = f & ~u;
  }
  __syncthreads();
  const int run = (words_here + WIDE - 1) / WIDE;
  const int i0 = min(words_here, (int)threadIdx.x * run), i1 = min(words_here, i0 + run);
  // How many pages of M, and used ones, lie below each thread's words.
  int count[2] = {0, 0}, at[2], ahead[2], all[2];
  for (int i = i0; i < i1; ++i) {
    count[0] += __popc(u_mine[i] | s_mine[i]);
    count[1] += __popc(u_mine[i]);
  }
  block_scan(count, at, S);
  cluster_scan(ahead, all, S, cluster);
  cluster.sync();                            // S.count is written again
  const int kept = all[1], rest = all[0] - all[1];
  int below = ahead[0] + at[0];
  int moves[3] = {0, 0, 0}, to[3], lead[3], sum[3];
  {
    int b = below;
    for (int i = i0; i < i1; ++i) {
      const uint32_t m = u_mine[i] | s_mine[i], low = lowest(m, kept - b);
      b += __popc(m);
      moves[0] += __popc(u_mine[i] & ~low);
      moves[1] += __popc(s_mine[i] & low);
      moves[2] += __popc(m & ~low);
      if (m & ~low) atomicMin(&s_first, (w0 + i) * 32 + __ffs(m & ~low) - 1);
    }
  }
  block_scan(moves, to, S);
  cluster_scan(lead, sum, S, cluster);
  int first = A.P;
  for (int c = 0; c < ctas; ++c) first = min(first, *cluster.map_shared_rank(&s_first, c));
  int a = lead[0] + to[0], z = lead[1] + to[1], f = A.nfree - rest + lead[2] + to[2];
  for (int i = i0; i < i1; ++i) {
    const uint32_t m = u_mine[i] | s_mine[i], low = lowest(m, kept - below);
    below += __popc(m);
    const int base = (w0 + i) * 32 - 1;
    for (uint32_t w = u_mine[i] & ~low; w != 0; w &= w - 1) A.copy_from[a++] = base + __ffs(w);
    for (uint32_t w = s_mine[i] & low; w != 0; w &= w - 1) A.copy_to[z++] = base + __ffs(w);
    for (uint32_t w = m & ~low; w != 0; w &= w - 1) A.free_pages[f++] = base + __ffs(w);
  }
  const int moved = sum[0];
  for (int i = moved + at0; i < half; i += step) A.copy_from[i] = A.copy_to[i] = -1;
  for (int i = at0; i < A.nfree - rest; i += step) A.free_pages[i] = __ldg(A.free_in + i);
  if (at0 == 0) *A.head_out = A.nfree - rest;
  __threadfence();
  cluster.sync();
  for (int i = at0; i < moved; i += step) A.map[__ldcg(A.copy_from + i)] = __ldcg(A.copy_to + i);
  __threadfence();
  cluster.sync();
  // The rows with their pages' new places; a warp a row.
  const int lane = threadIdx.x & 31, warps = ctas * (WIDE / 32);
  for (int b = rank * (WIDE / 32) + (threadIdx.x >> 5); b < A.B; b += warps) {
    const int have = min(pages_of(length_of(A.reserved, b), A.ps), A.width);
    const int* row = A.table + (int64_t)b * A.table_stride;
    int* out = A.table_out + (int64_t)b * A.width;
#pragma unroll 4
    for (int c = lane; c < A.width; c += 32) {
      int id = c < have ? __ldg(row + c) : -1;
      if (id >= A.P || id < 0) id = -1;
      out[c] = id >= first ? __ldcg(A.map + id) : id;
    }
  }
}

// ---------------------------------------------------------------------------
// Copies.  An item is one head of one page (keys, then values); the items of a CTA that name
// pages are listed first, so that lists that are mostly padding cost no waiting.
// ---------------------------------------------------------------------------

struct CopyArgs {
  uint16_t *kc, *vc;
  int64_t k_page, k_row, k_head, v_page, v_row, v_head;
  const int *from, *to, *rows;               // rows may be NULL: whole pages
  int64_t pages;
  int n, H, ps, ck, cv;                      // ck, cv: 16-byte pieces of a row
  uint32_t* err;
};

// One head's first `rows` rows; a thread has four pieces under way.
__device__ __forceinline__ void copy_rows(uint16_t* to, const uint16_t* from, int64_t row_stride,
                                          int rows, int pieces) {
  const int total = rows * pieces, dr = THREADS / pieces, dc = THREADS - dr * pieces;
  int r = threadIdx.x / pieces, c = threadIdx.x - r * pieces;
  for (int x = threadIdx.x; x < total; x += 4 * THREADS) {
    uint4 v[4];
    int64_t at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      at[u] = r * row_stride + c * 8;
      if (x + u * THREADS < total) v[u] = ldg_stream_v4(from + at[u]);
      r += dr;
      c += dc;
      if (c >= pieces) {
        c -= pieces;
        ++r;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (x + u * THREADS < total) *reinterpret_cast<uint4*>(to + at[u]) = v[u];
  }
}

__global__ void __launch_bounds__(THREADS) copy_kernel(const CopyArgs A) {
  __shared__ int list[THREADS];
  __shared__ int found;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t items = (int64_t)A.n * A.H, step = gridDim.x;
  for (int64_t base = blockIdx.x; base < items; base += step * THREADS) {
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    const int64_t w = base + threadIdx.x * step;
    if (w < items) {
      const int i = (int)(w / A.H), a = __ldg(A.from + i), z = __ldg(A.to + i);
      const bool real = a >= 0 && z >= 0 && a < A.pages && z < A.pages;
      if (a >= A.pages || z >= A.pages) atomicOr(A.err, ERR_PAGE);
      if (real && a != z && (A.rows == nullptr || __ldg(A.rows + i) > 0))
        list[atomicAdd(&found, 1)] = (int)threadIdx.x;
    }
    __syncthreads();
    for (int j = 0; j < found; ++j) {
      const int64_t w = base + list[j] * step;
      const int i = (int)(w / A.H), h = (int)(w - (int64_t)i * A.H);
      const int64_t a = __ldg(A.from + i), z = __ldg(A.to + i);
      const int rows = A.rows ? min(__ldg(A.rows + i), A.ps) : A.ps;
      copy_rows(A.kc + z * A.k_page + h * A.k_head, A.kc + a * A.k_page + h * A.k_head, A.k_row,
                rows, A.ck);
      copy_rows(A.vc + z * A.v_page + h * A.v_head, A.vc + a * A.v_page + h * A.v_head, A.v_row,
                rows, A.cv);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------

static int launch_cluster(void (*kernel)(PoolArgs), size_t smem, int ctas, void* stream,
                          const PoolArgs& A) {
  bind_stream_device(stream);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       200 * 1024);
  KB_REQUIRE(e == cudaSuccess, KB_ERR_DEVICE, "pages: shared-memory limit: %s",
             cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(WIDE);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kernel, A);
  KB_REQUIRE(e == cudaSuccess, KB_ERR_LAUNCH, "kernel launch failed: %s", cudaGetErrorString(e));
  return KB_OK;
}

static int check_pool(int64_t B, int64_t table_stride, int64_t width, int64_t n_free,
                      int64_t page_size, int64_t n_pages) {
  constexpr int64_t kMax = (int64_t)1 << 30;
  KB_REQUIRE(B > 0 && width > 0 && table_stride >= width && n_free >= 0 && page_size > 0 &&
                 n_pages > 0,
             KB_ERR_BAD_SHAPE, "pages: bad shape");
  KB_REQUIRE(B <= MAX_REQUESTS && width <= kMax && n_free <= kMax && page_size <= kMax &&
                 n_pages <= MAX_PAGES,
             KB_ERR_UNSUPPORTED, "pages: more than %d requests or %d pages", MAX_REQUESTS,
             MAX_PAGES);
  return KB_OK;
}

static int pool_ctas(int64_t B, int64_t width, int64_t n_pages) {
  return B * width + n_pages <= ALONE ? 1 : CLUSTER;
}

}  // namespace pages
}  // namespace kb

extern "C" int kb_paged_fork(int32_t* context_lens, int32_t* reserved_lens, int64_t B,
                             int32_t* block_table, int64_t table_stride, int64_t table_width,
                             const int32_t* sources, const int32_t* targets, int64_t n,
                             const int32_t* free_pages, int64_t n_free, const int32_t* free_head,
                             int64_t page_size, int32_t* copy_from, int32_t* copy_to,
                             int32_t* copy_rows, int32_t* free_head_out, int32_t* missing,
                             void* stream) {
  namespace pg = kb::pages;
  kb::clear_error();
  int st = pg::check_pool(B, table_stride, table_width, n_free, page_size, 1);
  if (st != KB_OK) return st;
  KB_REQUIRE(n > 0, KB_ERR_BAD_SHAPE, "paged fork: no pairs");
  KB_REQUIRE(n <= pg::MAX_REQUESTS, KB_ERR_UNSUPPORTED, "paged fork: more than %d pairs",
             pg::MAX_REQUESTS);
  KB_REQUIRE(context_lens && block_table && sources && targets && (free_pages || n_free == 0) &&
                 free_head && copy_from && copy_to && copy_rows && free_head_out && missing,
             KB_ERR_NULL_POINTER, "paged fork: NULL pointer");
  const int dev = kb::bind_stream_device(stream);
  pg::ForkArgs A = {};
  A.context = context_lens;
  A.reserved = reserved_lens;
  A.table = block_table;
  A.table_stride = table_stride;
  A.sources = sources;
  A.targets = targets;
  A.free_pages = free_pages;
  A.free_head = free_head;
  A.B = (int)B;
  A.width = (int)table_width;
  A.n = (int)n;
  A.nfree = (int)n_free;
  A.ps = (int)page_size;
  A.copy_from = copy_from;
  A.copy_to = copy_to;
  A.copy_rows = copy_rows;
  A.head_out = free_head_out;
  A.missing = missing;
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  const size_t smem = (size_t)(B + (B + 31) / 32) * sizeof(int);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        pg::fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
    KB_REQUIRE(e == cudaSuccess, KB_ERR_DEVICE, "paged fork: shared-memory limit: %s",
               cudaGetErrorString(e));
  }
  const int64_t sms = kb::num_sms(dev);
  return kb::launch(pg::fork_kernel, dim3((unsigned)(n < 2 * sms ? n : 2 * sms)),
                    dim3(pg::THREADS), smem, stream, A);
}

extern "C" int kb_paged_free(const int32_t* reserved_lens, const int32_t* keep_lens, int64_t B,
                             const int32_t* block_table, int64_t table_stride,
                             int64_t table_width, int32_t* free_pages, int64_t n_free,
                             const int32_t* free_head, int64_t page_size, int64_t n_pages,
                             int32_t* free_head_out, void* stream) {
  namespace pg = kb::pages;
  kb::clear_error();
  int st = pg::check_pool(B, table_stride, table_width, n_free, page_size, n_pages);
  if (st != KB_OK) return st;
  KB_REQUIRE(reserved_lens && keep_lens && block_table && (free_pages || n_free == 0) &&
                 free_head && free_head_out,
             KB_ERR_NULL_POINTER, "paged free: NULL pointer");
  const int dev = kb::bind_stream_device(stream);
  pg::PoolArgs A = {};
  A.table = block_table;
  A.table_stride = table_stride;
  A.reserved = reserved_lens;
  A.keep = keep_lens;
  A.free_pages = free_pages;
  A.free_head = free_head;
  A.B = (int)B;
  A.width = (int)table_width;
  A.nfree = (int)n_free;
  A.ps = (int)page_size;
  A.P = (int)n_pages;
  A.head_out = free_head_out;
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  const int ctas = pg::pool_ctas(B, table_width, n_pages);
  const size_t W = (size_t)(n_pages + 31) / 32, per = (W + ctas - 1) / ctas;
  return pg::launch_cluster(pg::free_kernel, (2 * W + per) * 4, ctas, stream, A);
}

extern "C" int kb_paged_compact(const int32_t* reserved_lens, int64_t B,
                                const int32_t* block_table, int64_t table_stride,
                                int64_t table_width, const int32_t* free_pages, int64_t n_free,
                                const int32_t* free_head, int64_t page_size, int64_t n_pages,
                                int32_t* table_out, int32_t* free_out, int32_t* copy_from,
                                int32_t* copy_to, int32_t* free_head_out, int32_t* scratch,
                                void* stream) {
  namespace pg = kb::pages;
  kb::clear_error();
  int st = pg::check_pool(B, table_stride, table_width, n_free, page_size, n_pages);
  if (st != KB_OK) return st;
  KB_REQUIRE(reserved_lens && block_table && (n_free == 0 || (free_pages && free_out)) &&
                 free_head && table_out && (n_pages < 2 || (copy_from && copy_to)) &&
                 free_head_out && scratch,
             KB_ERR_NULL_POINTER, "paged compact: NULL pointer");
  const int dev = kb::bind_stream_device(stream);
  pg::PoolArgs A = {};
  A.table = block_table;
  A.table_stride = table_stride;
  A.reserved = reserved_lens;
  A.free_in = free_pages;
  A.free_pages = free_out;
  A.free_head = free_head;
  A.B = (int)B;
  A.width = (int)table_width;
  A.nfree = (int)n_free;
  A.ps = (int)page_size;
  A.P = (int)n_pages;
  A.head_out = free_head_out;
  A.table_out = table_out;
  A.copy_from = copy_from;
  A.copy_to = copy_to;
  A.map = scratch;
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  const int ctas = pg::pool_ctas(B, table_width, n_pages);
  const size_t W = (size_t)(n_pages + 31) / 32, per = (W + ctas - 1) / ctas;
  return pg::launch_cluster(pg::compact_kernel, (2 * W + 2 * per) * 4, ctas, stream, A);
}

extern "C" int kb_paged_copy(uint16_t* k_cache, const int64_t* k_strides, uint16_t* v_cache,
                             const int64_t* v_strides, int64_t n_pages, int64_t page_size,
                             int64_t H, int64_t Dk, int64_t Dv, const int32_t* copy_from,
                             const int32_t* copy_to, const int32_t* copy_rows, int64_t n,
                             void* stream) {
  namespace pg = kb::pages;
  kb::clear_error();
  KB_REQUIRE(n >= 0 && H > 0 && Dk > 0 && Dv > 0 && n_pages >= 0 && page_size > 0,
             KB_ERR_BAD_SHAPE, "paged copy: bad shape");
  if (n == 0 || n_pages == 0) return KB_OK;
  KB_REQUIRE(k_cache && v_cache && k_strides && v_strides && copy_from && copy_to,
             KB_ERR_NULL_POINTER, "paged copy: NULL pointer");
  KB_REQUIRE(Dk % 8 == 0 && Dv % 8 == 0 && Dk <= 2048 && Dv <= 2048 && H <= 65535 &&
                 page_size <= (1 << 20) && n < ((int64_t)1 << 30),
             KB_ERR_UNSUPPORTED, "paged copy: head widths must be multiples of 8 up to 2048");
  bool ok = (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && ((k_strides[i] | v_strides[i]) & 7) == 0;
  KB_REQUIRE(ok, KB_ERR_ALIGNMENT,
             "paged copy: pointers must be 16-byte aligned and strides multiples of 8");
  const int64_t extents[3] = {n_pages, page_size, H};
  for (int i = 0; i < 3; ++i)
    KB_REQUIRE(extents[i] <= 1 || (k_strides[i] > 0 && v_strides[i] > 0), KB_ERR_BAD_SHAPE,
               "paged copy: strides of the caches must be positive");
  const int dev = kb::bind_stream_device(stream);
  pg::CopyArgs A = {};
  A.kc = k_cache;
  A.vc = v_cache;
  A.k_page = k_strides[0];
  A.k_row = k_strides[1];
  A.k_head = k_strides[2];
  A.v_page = v_strides[0];
  A.v_row = v_strides[1];
  A.v_head = v_strides[2];
  A.from = copy_from;
  A.to = copy_to;
  A.rows = copy_rows;
  A.pages = n_pages;
  A.n = (int)n;
  A.H = (int)H;
  A.ps = (int)page_size;
  A.ck = (int)(Dk / 8);
  A.cv = (int)(Dv / 8);
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  const int64_t items = n * H, most = (int64_t)kb::num_sms(dev) * 8;
  return kb::launch(pg::copy_kernel, dim3((unsigned)(items < most ? items : most)),
                    dim3(pg::THREADS), 0, stream, A);
}
