// kb_paged.cu - block tables, slot maps and tree masks from request lengths,
// and storing new keys and values by slot.
//
// Request b has c_b cached tokens and n_b new ones; a page holds ps token rows, and
// the request's pages reach r_b >= c_b tokens (drafted tokens that were refused leave
// their pages to it).
//   need_b  = max(0, ceil((c_b + n_b) / ps) - ceil(r_b / ps))  pages to take
//   first_b = head + sum_{a < b} need_a                        in the free list
//   table[b, ceil(r_b / ps) + i] = free[first_b + i]
//   token t of b: place p = c_b + t, slot = table[b, p / ps] * ps + p % ps
//   with a tree: mask_t = bit t | mask_parent(t), position = c_b + depth(t)
//
// One launch, no dependence between CTAs: every CTA sums the requests' needs
// itself (two ints a request, from L2), keeps the running sums in shared
// memory and then takes its share of the fresh pages and of the new tokens,
// each found by a binary search in the sums.  A token in a fresh page reads
// the free list, not the table entry another CTA may be writing.  A few
// kilobytes of traffic.  A few requests cost launch and dependent-load latency, many the
// sums that every CTA makes (replayed, with few tokens: 32 requests 3.2 us, 256 3.6,
// 1024 4.5, 2048 6.5, 8192 46; 2048 with 200 thousand tokens 10.9).
#include "kb_common.cuh"

namespace kb {
namespace paged {

constexpr int THREADS = 256;
constexpr int MAX_REQUESTS = 12288;          // four int arrays of shared memory

struct PlanArgs {
  const int* context;
  const int* reserved;     // NULL: context
  const int* fresh;        // new tokens of each request
  int* table;
  int64_t table_stride;
  const int* free_pages;
  const int* free_head;
  const int* parents;      // NULL: no tree
  int B, width, nfree, ps, N;
  int* cu;
  int64_t* slots;
  int* positions;
  int64_t* mask;
  int* head_out;
  int* missing;
  uint32_t* err;
};

// Lengths count up to 2^30 - 1, so that two and their pages stay within 31 bits (a page's
// rows up to 2^30).
constexpr int LONGEST = (1 << 30) - 1;
__device__ __forceinline__ uint32_t length_of(const int* lens, int b) {
  return (uint32_t)min(max(__ldg(lens + b), 0), LONGEST);
}

__device__ __forceinline__ int pages_of(uint32_t tokens, uint32_t ps) {
  return (int)((tokens + ps - 1) / ps);
}

// Largest i in [0, n) with sums[i] <= v (sums ascending, sums[0] = 0).
__device__ __forceinline__ int find(const int* sums, int n, int v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= v) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Sums stop above the 2^30 that any output holds: lengths that nobody meant must not
// wrap around to places before it.
__device__ __forceinline__ int add(int a, int b) {
  return (int)min((uint32_t)a + (uint32_t)b, (1u << 30) + 1u);
}

// Running sums over a warp, and those of the lanes before.
__device__ __forceinline__ int warp_scan(int v, int lane, int& before) {
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = add(v, u);
  }
  before = __shfl_up_sync(0xffffffffu, v, 1);
  if (lane == 0) before = 0;
  return v;
}

__global__ void __launch_bounds__(THREADS) plan_kernel(const PlanArgs A) {
  extern __shared__ int sums[];
  int* s_tok = sums;                 // [B + 1] first token of each request
  int* s_page = sums + A.B + 1;      // [B + 1] first fresh page of each request
  int* s_ctx = s_page + A.B + 1;     // [B] cached tokens
  int* s_have = s_ctx + A.B;         // [B] pages
  __shared__ int s_part[THREADS / 32][3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ps = (uint32_t)A.ps;
  pdl_wait();
  // Each thread takes a run of consecutive requests.
  const int per = (A.B + THREADS - 1) / THREADS;
  const int b0 = min(A.B, tid * per), b1 = min(A.B, b0 + per);
  int tok = 0, page = 0, lost = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    const uint32_t c = length_of(A.context, b), n = length_of(A.fresh, b);
    const int have = pages_of(A.reserved ? max(c, length_of(A.reserved, b)) : c, ps);
    const int want = pages_of(c + n, ps), need = max(0, min(want, A.width) - have);
    s_tok[b] = tok;
    s_page[b] = page;
    s_ctx[b] = (int)c;
    s_have[b] = have;
    tok = add(tok, (int)n);
    page = add(page, need);
    lost = add(lost, max(0, want - have) - need);
  }
  int tok0, page0, lost0;
  const int tok_in = warp_scan(tok, lane, tok0), page_in = warp_scan(page, lane, page0);
  const int lost_in = warp_scan(lost, lane, lost0);
  if (lane == 31) {
    s_part[warp][0] = tok_in;
    s_part[warp][1] = page_in;
    s_part[warp][2] = lost_in;
  }
  __syncthreads();
  int tokens = 0, pages = 0, beyond = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) {
      tok0 = add(tok0, s_part[w][0]);
      page0 = add(page0, s_part[w][1]);
    }
    tokens = add(tokens, s_part[w][0]);
    pages = add(pages, s_part[w][1]);
    beyond = add(beyond, s_part[w][2]);
  }
  for (int b = b0; b < b1; ++b) {
    s_tok[b] = add(s_tok[b], tok0);
    s_page[b] = add(s_page[b], page0);
  }
  if (tid == 0) {
    s_tok[A.B] = tokens;
    s_page[A.B] = pages;
  }
  const int head = max(0, *A.free_head);
  const int avail = max(0, A.nfree - head);
  __syncthreads();
  pdl_launch_dependents();

  const int at = blockIdx.x * THREADS + tid, step = gridDim.x * THREADS;
  for (int b = at; b <= A.B; b += step) A.cu[b] = min(s_tok[b], A.N);
  if (at == 0) {
    *A.head_out = head + min(pages, avail);
    *A.missing = add(beyond, max(0, pages - avail));
    if (tokens > A.N) atomicOr(A.err, ERR_PAGE);
  }
  for (int i = at; i < pages; i += step) {
    const int b = find(s_page, A.B, i);
    const int col = s_have[b] + i - s_page[b];
    A.table[(int64_t)b * A.table_stride + col] = i < avail ? __ldg(A.free_pages + head + i) : -1;
  }
  // The page of a token: a fresh one, or an entry that no CTA writes.
  auto place_of = [&](int i, uint32_t& place, int& b) {
    b = find(s_tok, A.B, i);
    const uint32_t c = (uint32_t)s_ctx[b];
    place = c + (uint32_t)(i - s_tok[b]);
    const int col = (int)(place / ps), have = s_have[b];
    if (col >= A.width) return -1;
    if (col < have) return __ldg(A.table + (int64_t)b * A.table_stride + col);
    const int f = s_page[b] + col - have;
    return f < avail ? __ldg(A.free_pages + head + f) : -1;
  };
  constexpr int BATCH = 4;
  for (int i0 = at; i0 < A.N; i0 += BATCH * step) {
    int id[BATCH], b[BATCH];
    uint32_t place[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = i0 + u * step;
      id[u] = -1;
      place[u] = 0;
      b[u] = 0;
      if (i < min(tokens, A.N)) id[u] = place_of(i, place[u], b[u]);
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = i0 + u * step;
      if (i >= A.N) break;
      int64_t word = 0;
      int position = (int)place[u];
      if (A.parents != nullptr && i < tokens) {
        // Up the tree: parents come before their children, so this ends.
        const int t = i - s_tok[b[u]];
        int node = t, depth = 0;
        if (t < 64) {
          word = (int64_t)1 << t;
          while (node > 0) {
            const int up = __ldg(A.parents + s_tok[b[u]] + node);
            if (up < 0 || up >= node) {
              atomicOr(A.err, ERR_TREE);
              break;
            }
            word |= (int64_t)1 << up;
            node = up;
            ++depth;
          }
        } else {
          atomicOr(A.err, ERR_TREE);
        }
        position = s_ctx[b[u]] + depth;
      }
      A.slots[i] = id[u] >= 0 ? (int64_t)id[u] * A.ps + place[u] % ps : -1;
      A.positions[i] = position;
      if (A.mask != nullptr) A.mask[i] = word;
    }
  }
}

// ---------------------------------------------------------------------------
// What the pages reach once a plan has given what it could.  A request's fresh table
// entries are pages and then, where the pool was empty, -1: the first -1 is found by
// halving, 9 dependent loads for a prompt of 512 pages.
// ---------------------------------------------------------------------------

struct ReserveArgs {
  const int *context, *fresh, *table;
  int64_t table_stride;
  int B, width, ps;
  int* reserved;
};

__global__ void __launch_bounds__(THREADS) reserve_kernel(const ReserveArgs A) {
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x * THREADS + threadIdx.x;
  if (b >= A.B) return;
  const uint32_t ps = (uint32_t)A.ps, c = length_of(A.context, b), n = length_of(A.fresh, b);
  const uint32_t before = max(c, (uint32_t)min(max(A.reserved[b], 0), LONGEST));
  int pages = pages_of(before, ps), end = max(pages, min(pages_of(c + n, ps), A.width));
  while (pages < end) {
    const int mid = pages + ((end - pages) >> 1);
    if (A.table[(int64_t)b * A.table_stride + mid] >= 0) pages = mid + 1; else end = mid;
  }
  const uint32_t reach = max(before, min(c + n, (uint32_t)pages * ps));
  A.reserved[b] = (int)min(reach, (uint32_t)LONGEST);
}

// ---------------------------------------------------------------------------
// Keys and values into their slots.
// ---------------------------------------------------------------------------

struct AppendArgs {
  const uint16_t *k, *v;
  int64_t k_tok, k_head, v_tok, v_head;            // element strides
  uint16_t *kc, *vc;
  int64_t kc_page, kc_row, kc_head, vc_page, vc_row, vc_head;
  const int64_t* slots;
  int64_t nslots;
  int N, H, ps, ck, cv;                            // ck, cv: 16-byte pieces of a row
  uint32_t* err;
};

// Four 16-byte pieces per thread, loaded before any is stored; a token's pieces
// are its heads' key rows and then its heads' value rows, so neighbouring threads
// move neighbouring bytes.  8192 tokens of 8 heads of 128 + 128: 15.3 us replayed (4.4
// TB/s), bound by instructions: 168 a piece, most of them the divisions that find its
// head, page and row, at 66 % of the issue slots.  The order of the slots is of no
// account (in order 15.2 us, single rows at random 15.3).
constexpr int PIECES = 4;

__global__ void __launch_bounds__(THREADS) append_kernel(const AppendArgs A) {
  pdl_wait();
  pdl_launch_dependents();
  const int keys = A.H * A.ck, pieces = keys + A.H * A.cv;      // of a token
  const int64_t base = (int64_t)blockIdx.x * (THREADS * PIECES);
  const int64_t t0 = base / pieces;
  const int r0 = (int)(base - t0 * pieces) + threadIdx.x;
  uint4 x[PIECES];
  uint16_t* to[PIECES];
#pragma unroll
  for (int u = 0; u < PIECES; ++u) {
    const int over = (r0 + u * THREADS) / pieces;
    int r = r0 + u * THREADS - over * pieces;
    const int64_t t = t0 + over;
    to[u] = nullptr;
    if (t >= A.N) continue;
    const int64_t slot = __ldg(A.slots + t);
    if (slot < 0) continue;
    if (slot >= A.nslots) {
      atomicOr(A.err, ERR_PAGE);
      continue;
    }
    const int64_t page = slot / A.ps, row = slot - page * A.ps;
    if (r < keys) {
      const int h = r / A.ck, c = r - h * A.ck;
      x[u] = ldg_stream_v4(A.k + t * A.k_tok + h * A.k_head + c * 8);
      to[u] = A.kc + page * A.kc_page + row * A.kc_row + h * A.kc_head + c * 8;
    } else {
      r -= keys;
      const int h = r / A.cv, c = r - h * A.cv;
      x[u] = ldg_stream_v4(A.v + t * A.v_tok + h * A.v_head + c * 8);
      to[u] = A.vc + page * A.vc_page + row * A.vc_row + h * A.vc_head + c * 8;
    }
  }
#pragma unroll
  for (int u = 0; u < PIECES; ++u)
    if (to[u] != nullptr) *reinterpret_cast<uint4*>(to[u]) = x[u];
}

}  // namespace paged
}  // namespace kb

extern "C" int kb_paged_plan(const int32_t* context_lens, const int32_t* reserved_lens,
                             const int32_t* new_lens, int64_t B,
                             int32_t* block_table, int64_t table_stride, int64_t table_width,
                             const int32_t* free_pages, int64_t n_free, const int32_t* free_head,
                             int64_t page_size, int64_t n_tokens, const int32_t* parents,
                             int32_t* cu_tokens, int64_t* slots, int32_t* positions,
                             int64_t* tree_mask, int32_t* free_head_out, int32_t* missing,
                             void* stream) {
  kb::clear_error();
  constexpr int64_t kMax = (int64_t)1 << 30;
  KB_REQUIRE(B > 0 && table_width > 0 && table_stride >= table_width && n_free >= 0 &&
                 n_tokens >= 0 && page_size > 0,
             KB_ERR_BAD_SHAPE, "paged plan: bad shape");
  KB_REQUIRE(B <= kb::paged::MAX_REQUESTS && n_tokens <= kMax && n_free <= kMax &&
                 table_width <= kMax && page_size <= kMax,
             KB_ERR_UNSUPPORTED, "paged plan: more than %d requests or 2^30 tokens or pages",
             kb::paged::MAX_REQUESTS);
  KB_REQUIRE(context_lens && new_lens && block_table && (free_pages || n_free == 0) &&
                 free_head && cu_tokens && (n_tokens == 0 || (slots && positions)) &&
                 free_head_out && missing && (!parents || tree_mask || n_tokens == 0),
             KB_ERR_NULL_POINTER, "paged plan: NULL pointer");
  const int dev = kb::bind_stream_device(stream);
  kb::paged::PlanArgs A = {};
  A.context = context_lens;
  A.reserved = reserved_lens;
  A.fresh = new_lens;
  A.table = block_table;
  A.table_stride = table_stride;
  A.free_pages = free_pages;
  A.free_head = free_head;
  A.parents = parents;
  A.B = (int)B;
  A.width = (int)table_width;
  A.nfree = (int)n_free;
  A.ps = (int)page_size;
  A.N = (int)n_tokens;
  A.cu = cu_tokens;
  A.slots = slots;
  A.positions = positions;
  A.mask = parents ? tree_mask : nullptr;
  A.head_out = free_head_out;
  A.missing = missing;
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  const size_t smem = (size_t)(4 * B + 2) * sizeof(int);
  static_assert((4 * kb::paged::MAX_REQUESTS + 2) * sizeof(int) <= 200 * 1024, "shared memory");
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kb::paged::plan_kernel,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    KB_REQUIRE(e == cudaSuccess, KB_ERR_DEVICE, "paged plan: shared-memory limit: %s",
               cudaGetErrorString(e));
  }
  const int64_t items = n_tokens > B ? n_tokens : B;
  int64_t grid = (items + kb::paged::THREADS - 1) / kb::paged::THREADS;
  const int sms = kb::num_sms(dev);
  if (grid > sms) grid = sms;
  return kb::launch(kb::paged::plan_kernel, dim3((unsigned)grid), dim3(kb::paged::THREADS), smem,
                    stream, A);
}

extern "C" int kb_paged_reserve(const int32_t* context_lens, const int32_t* new_lens, int64_t B,
                                const int32_t* block_table, int64_t table_stride,
                                int64_t table_width, int64_t page_size, int32_t* reserved_lens,
                                void* stream) {
  kb::clear_error();
  constexpr int64_t kMax = (int64_t)1 << 30;
  KB_REQUIRE(B > 0 && table_width > 0 && table_stride >= table_width && page_size > 0,
             KB_ERR_BAD_SHAPE, "paged reserve: bad shape");
  KB_REQUIRE(B <= kb::paged::MAX_REQUESTS && table_width <= kMax && page_size <= kMax,
             KB_ERR_UNSUPPORTED, "paged reserve: more than %d requests or 2^30 tokens or pages",
             kb::paged::MAX_REQUESTS);
  KB_REQUIRE(context_lens && new_lens && block_table && reserved_lens, KB_ERR_NULL_POINTER,
             "paged reserve: NULL pointer");
  kb::paged::ReserveArgs A = {};
  A.context = context_lens;
  A.fresh = new_lens;
  A.table = block_table;
  A.table_stride = table_stride;
  A.B = (int)B;
  A.width = (int)table_width;
  A.ps = (int)page_size;
  A.reserved = reserved_lens;
  const int64_t grid = (B + kb::paged::THREADS - 1) / kb::paged::THREADS;
  return kb::launch(kb::paged::reserve_kernel, dim3((unsigned)grid), dim3(kb::paged::THREADS), 0,
                    stream, A);
}

extern "C" int kb_paged_append(const uint16_t* k, int64_t k_token_stride, int64_t k_head_stride,
                               const uint16_t* v, int64_t v_token_stride, int64_t v_head_stride,
                               int64_t N, int64_t H, int64_t Dk, int64_t Dv, uint16_t* k_cache,
                               const int64_t* k_strides, uint16_t* v_cache,
                               const int64_t* v_strides, int64_t n_pages, int64_t page_size,
                               const int64_t* slots, void* stream) {
  kb::clear_error();
  KB_REQUIRE(N >= 0 && H > 0 && Dk > 0 && Dv > 0 && n_pages >= 0 && page_size > 0,
             KB_ERR_BAD_SHAPE, "paged append: bad shape");
  if (N == 0) return KB_OK;
  KB_REQUIRE(k && v && slots && k_strides && v_strides &&
                 (n_pages == 0 || (k_cache && v_cache)),
             KB_ERR_NULL_POINTER, "paged append: NULL pointer");
  KB_REQUIRE(Dk % 8 == 0 && Dv % 8 == 0 && N < ((int64_t)1 << 31) &&
                 H * (Dk + Dv) < ((int64_t)1 << 31),
             KB_ERR_UNSUPPORTED, "paged append: head widths must be multiples of 8");
  bool ok = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0 &&
            ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && ((k_strides[i] | v_strides[i]) & 7) == 0;
  KB_REQUIRE(ok, KB_ERR_ALIGNMENT,
             "paged append: pointers must be 16-byte aligned and strides multiples of 8");
  const int64_t extents[3] = {n_pages, page_size, H};
  for (int i = 0; i < 3; ++i)
    KB_REQUIRE(extents[i] <= 1 || (k_strides[i] > 0 && v_strides[i] > 0), KB_ERR_BAD_SHAPE,
               "paged append: strides of the caches must be positive");
  const int dev = kb::bind_stream_device(stream);
  kb::paged::AppendArgs A = {};
  A.k = k;
  A.v = v;
  A.k_tok = k_token_stride;
  A.k_head = k_head_stride;
  A.v_tok = v_token_stride;
  A.v_head = v_head_stride;
  A.kc = k_cache;
  A.vc = v_cache;
  A.kc_page = k_strides[0];
  A.kc_row = k_strides[1];
  A.kc_head = k_strides[2];
  A.vc_page = v_strides[0];
  A.vc_row = v_strides[1];
  A.vc_head = v_strides[2];
  A.slots = slots;
  A.nslots = n_pages * page_size;
  A.N = (int)N;
  A.H = (int)H;
  A.ps = (int)page_size;
  A.ck = (int)(Dk / 8);
  A.cv = (int)(Dv / 8);
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  constexpr int64_t kBlock = kb::paged::THREADS * kb::paged::PIECES;
  const int64_t grid = (N * H * (A.ck + A.cv) + kBlock - 1) / kBlock;
  KB_REQUIRE(grid < ((int64_t)1 << 31), KB_ERR_UNSUPPORTED, "paged append: too many tokens");
  return kb::launch(kb::paged::append_kernel, dim3((unsigned)grid), dim3(kb::paged::THREADS), 0,
                    stream, A);
}
