// kb_linear.cu - linear attention with a decay for each head in fp32: token by token, and in
// blocks of 32 tokens.
//
// For head h of a request, with the state S [Dk, Dv] in fp32:
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale * q_t S_t
// One token a request (decoding), or a few: the state is read once, updated in registers
// and written once.  A CTA has a head's state, or, where there are few heads, 32 of its
// columns (they are independent): 256 threads, four columns and Dk / 8 (Dk / 32) rows each.
// The sums over the rows meet in shared memory, one barrier a token.  Longer prompts go in
// blocks (below), bf16 ones in chunks on the tensor cores (kb_linear_chunk.cu).
//
// Bound: HBM, the states read and written: 256 requests of 32 heads of 128 x 128 move 1.08 GB in
// 175 us, 6.2 TB/s.  One request, 2.8 us (4 MB): a launch and one trip to memory.  Each further
// token of 256 requests takes about 44 us more, its barrier and its sums across threads one after
// the other beside the states in registers (4 tokens 306 us, 170 at the copy's rate).
// The state, the sums and the products are fp32; an output is rounded once, when it is stored.
#include "kb_linear.cuh"

namespace kb {
namespace linear {

constexpr int THREADS = 256;
constexpr int WIDEST = 128;                  // Dk, Dv

template <int TYPE>                          // 0 bf16, 1 f16, 2 f32
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if (TYPE == 2) return __ldg(static_cast<const float*>(p) + i);
  return attn::element<TYPE == 1>(__ldg(static_cast<const uint16_t*>(p) + i));
}

template <int TYPE>
__device__ __forceinline__ float4 load4(const void* p, int64_t i) {
  if (TYPE == 2) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i));
  constexpr bool F16 = TYPE == 1;
  return make_float4(attn::element<F16>((uint16_t)w.x), attn::element<F16>((uint16_t)(w.x >> 16)),
                     attn::element<F16>((uint16_t)w.y), attn::element<F16>((uint16_t)(w.y >> 16)));
}

template <int TYPE>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if (TYPE == 2)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<uint16_t*>(p)[i] = (uint16_t)attn::pack2<TYPE == 1>(v, 0.f);
}

// Rows outside every request: zero.
template <int TYPE>
__device__ __forceinline__ void clear_outside(const Args& A) {
  const int64_t lead = min(max((int64_t)A.cu[0], (int64_t)0), A.total);
  const int64_t tail = min(max((int64_t)A.cu[A.B], lead), A.total);
  const int64_t width = (int64_t)A.H * A.Dv, spare = (lead + A.total - tail) * width;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < spare;
       i += (int64_t)gridDim.x * THREADS)
    store1<TYPE>(A.out, i < lead * width ? i : i - lead * width + tail * width, 0.f);
}

// Rows [row, end) of a request past its longest: zero in a CTA's columns [col, col + width).
template <int TYPE>
__device__ __forceinline__ void clear_past(const Args& A, int h, int64_t row, int64_t end, int col,
                                           int width) {
  width = min(width, A.Dv - col);
  for (int64_t i = threadIdx.x; i < (end - row) * width; i += THREADS)
    store1<TYPE>(A.out, ((row + i / width) * A.H + h) * A.Dv + col + i % width, 0.f);
}

// COLS: columns of a CTA, 128 or 32.
template <int TYPE, int COLS>
__global__ void __launch_bounds__(THREADS) token_kernel(const Args A) {
  constexpr int CG = COLS / 4, RG = THREADS / CG, ROWS = WIDEST / RG;
  __shared__ float kq[2][2][WIDEST];
  __shared__ float4 red[2][THREADS / 32][CG];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int parts = (A.Dv + COLS - 1) / COLS;
  const int part = blockIdx.x % parts, bh = blockIdx.x / parts;
  const int b = bh / A.H, h = bh - b * A.H;
  const int cg = tid % CG, rg = tid / CG;
  const int col = part * COLS + cg * 4;
  const bool live = col < A.Dv;
  pdl_wait();
  pdl_launch_dependents();

  if (A.cu != nullptr) clear_outside<TYPE>(A);
  int64_t first, end;
  const int n = request_tokens(A, b, first, end);
  if (n <= 0) return;
  clear_past<TYPE>(A, h, first + n, end, part * COLS, COLS);
  float* state = request_state(A, b, h);
  float4 s[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int i = rg + RG * j;
    s[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (state != nullptr && live && i < A.Dk)
      s[j] = *reinterpret_cast<const float4*>(state + (int64_t)i * A.Dv + col);
  }
  const int64_t kh = (int64_t)(h / A.k_group) * A.k_head, qh = (int64_t)(h / A.q_group) * A.q_head;
  const int64_t vh = (int64_t)h * A.v_head + col;
  const int at = tid & (WIDEST - 1);
  // Threads 0-127 bring in k, the others q.
  auto fetch = [&](int t) {
    if (at >= A.Dk) return 0.f;
    return tid < WIDEST ? load1<TYPE>(A.k, (first + t) * A.k_tok + kh + at)
                        : load1<TYPE>(A.q, (first + t) * A.q_tok + qh + at) * A.scale;
  };
  auto values = [&](int t) {
    return live ? load4<TYPE>(A.v, (first + t) * A.v_tok + vh) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  auto decay = [&](int t) { return __ldg(A.decay + (first + t) * A.decay_tok + h); };
  auto finish = [&](int t) {                 // the sums of token t
    if (tid >= COLS || part * COLS + tid >= A.Dv) return;
    const float* sums = reinterpret_cast<const float*>(&red[t & 1][0][0]);
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) o += sums[w * COLS + tid];
    store1<TYPE>(A.out, ((first + t) * A.H + h) * A.Dv + part * COLS + tid, o);
  };
  kq[0][tid / WIDEST][at] = fetch(0);
  float4 v = values(0);
  float g = decay(0);
  for (int t = 0; t < n; ++t) {
    const float keep = expf(decay_of(g));
    const float4 now = v;
    float next = 0.f;
    if (t + 1 < n) {
      next = fetch(t + 1);
      v = values(t + 1);
      g = decay(t + 1);
    }
    __syncthreads();
    if (t > 0) finish(t - 1);
    const float* k = kq[t & 1][0];
    const float* q = kq[t & 1][1];
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const float kk = k[rg + RG * j], qq = q[rg + RG * j];
      s[j].x = fmaf(kk, now.x, s[j].x * keep);
      s[j].y = fmaf(kk, now.y, s[j].y * keep);
      s[j].z = fmaf(kk, now.z, s[j].z * keep);
      s[j].w = fmaf(kk, now.w, s[j].w * keep);
      o.x = fmaf(qq, s[j].x, o.x);
      o.y = fmaf(qq, s[j].y, o.y);
      o.z = fmaf(qq, s[j].z, o.z);
      o.w = fmaf(qq, s[j].w, o.w);
    }
#pragma unroll
    for (int d = CG; d < 32; d *= 2) {
      o.x += __shfl_xor_sync(0xffffffffu, o.x, d);
      o.y += __shfl_xor_sync(0xffffffffu, o.y, d);
      o.z += __shfl_xor_sync(0xffffffffu, o.z, d);
      o.w += __shfl_xor_sync(0xffffffffu, o.w, d);
    }
    if (lane < CG) red[t & 1][warp][lane] = o;
    if (t + 1 < n) kq[(t + 1) & 1][tid / WIDEST][at] = next;
  }
  __syncthreads();
  finish(n - 1);
  if (state != nullptr && live)
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int i = rg + RG * j;
      if (i < A.Dk) *reinterpret_cast<float4*>(state + (int64_t)i * A.Dv + col) = s[j];
    }
}

// ---------------------------------------------------------------------------
// f16 and f32 prompts, 32 tokens at a time in fp32.
//
// With b_i the running sum of the decays' logarithms in a block, for its rows i and j <= i:
//   P_ij = (q_i . k_j) exp(b_i - b_j),  o_i = exp(b_i) q_i S + sum_j P_ij v_j
//   S'   = exp(b_31) S + sum_j k_j exp(b_31 - b_j) v_j
// The sums are in 64 bits: their differences decide small exponents next to large ones.  A CTA
// has 32 columns of a head's state, in registers (16 rows of a column a thread) and, for q S, in
// shared memory.  Bound: shared-memory loads, 12 for 32 products a warp while scores and q S are
// made (the scores again for each 32 columns), and with one CTA an SM their latencies; no tensor
// cores, whose products would need these types in bf16 parts.  Measured, 32 heads of 128 x 128:
// one f16 prompt of 8192 tokens 1.77 ms, 6.9 us a block (token by token 10.7), f32 1.61 (6.1); 16
// prompts of 512 tokens 1.12 ms, 5 us a block and SM.
// ---------------------------------------------------------------------------

constexpr int BLOCK = 32;
constexpr int K_ROW = WIDEST + 4;            // (k by rows: 16-byte loads without conflicts)

struct BlockShared {
  float q[BLOCK][WIDEST], k[BLOCK][K_ROW], s[WIDEST][BLOCK], v[BLOCK][BLOCK], p[BLOCK][BLOCK];
  double b[BLOCK];                           // the running sums
  float start[BLOCK], rest[BLOCK];           // exp(b_i); exp(b_31 - b_j)
  int since[BLOCK];                          // the last reset up to the row, plus 1; 0: none
  int none;                                  // the first logarithm that is no number
};

// exp of a difference in 64 bits, to expf's accuracy.
__device__ __forceinline__ float exp_of(double d) {
  const float high = (float)d, e = expf(high);
  return high > -104.f ? fmaf(e, (float)(d - (double)high), e) : e;
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS, 2) block_kernel(const Args A) {
  extern __shared__ __align__(16) uint8_t smem[];
  BlockShared& B = *reinterpret_cast<BlockShared*>(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int parts = (A.Dv + BLOCK - 1) / BLOCK;
  const int part = blockIdx.x % parts, bh = blockIdx.x / parts;
  const int b = bh / A.H, h = bh - b * A.H;
  const int col = part * BLOCK + lane;       // of the state and of the outputs
  const bool live = col < A.Dv;
  constexpr int ROWS = WIDEST / (THREADS / 32);          // of the state, a warp
  pdl_wait();
  pdl_launch_dependents();
  clear_outside<TYPE>(A);
  int64_t first, end;
  const int n = request_tokens(A, b, first, end);
  if (n <= 0) return;
  clear_past<TYPE>(A, h, first + n, end, part * BLOCK, BLOCK);
  float* state = request_state(A, b, h);
  float s[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int d = warp * ROWS + r;
    s[r] = state != nullptr && live && d < A.Dk ? state[(int64_t)d * A.Dv + col] : 0.f;
    B.s[d][lane] = s[r];
  }
  const int64_t kh = (int64_t)(h / A.k_group) * A.k_head, qh = (int64_t)(h / A.q_group) * A.q_head;
  // The next block's rows, four of q and of k a warp; a piece of v a thread.
  float4 q[4], k[4], v;
  float g = 0.f;
  const int v_row = tid / (BLOCK / 4), v_col = tid % (BLOCK / 4) * 4;
  auto fetch = [&](int t0) {
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t t = first + t0 + warp + 8 * u;
      const bool real = t0 + warp + 8 * u < n && lane * 4 < A.Dk;
      q[u] = real ? load4<TYPE>(A.q, t * A.q_tok + qh + lane * 4) : zero;
      k[u] = real ? load4<TYPE>(A.k, t * A.k_tok + kh + lane * 4) : zero;
    }
    v = t0 + v_row < n && part * BLOCK + v_col < A.Dv
            ? load4<TYPE>(A.v, (first + t0 + v_row) * A.v_tok + (int64_t)h * A.v_head +
                                   part * BLOCK + v_col)
            : zero;
    if (warp == 0)
      g = t0 + lane < n ? __ldg(A.decay + (first + t0 + lane) * A.decay_tok + h) : 0.f;
  };
  fetch(0);
#pragma unroll 1
  for (int t0 = 0; t0 < n; t0 += BLOCK) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float4 x = make_float4(q[u].x * A.scale, q[u].y * A.scale, q[u].z * A.scale,
                                   q[u].w * A.scale);
      *reinterpret_cast<float4*>(&B.q[warp + 8 * u][lane * 4]) = x;
      *reinterpret_cast<float4*>(&B.k[warp + 8 * u][lane * 4]) = k[u];
    }
    *reinterpret_cast<float4*>(&B.v[v_row][v_col]) = v;
    if (warp == 0) {
      // A decay that is 0 in fp32 is a reset; it counts as such, not in the sums.
      const float x = decay_of(g);
      const unsigned resets = __ballot_sync(0xffffffffu, x <= -104.f);
      const unsigned odd = __ballot_sync(0xffffffffu, x != x);
      double sum = x <= -104.f ? 0.0 : (double)x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double before = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += before;
      }
      const unsigned up = resets & (0xffffffffu >> (31 - lane));
      const int since = up ? 32 - __clz(up) : 0, last = resets ? 32 - __clz(resets) : 0;
      const double all = __shfl_sync(0xffffffffu, sum, 31);
      const int none = odd ? __ffs(odd) - 1 : BLOCK;
      B.b[lane] = sum;
      B.since[lane] = since;
      B.start[lane] = lane >= none ? NAN : since ? 0.f : exp_of(sum);
      B.rest[lane] = none < BLOCK ? NAN : lane + 1 < last ? 0.f : exp_of(all - sum);
      if (lane == 0) B.none = none;
    }
    __syncthreads();
    if (t0 + BLOCK < n) fetch(t0 + BLOCK);
    // A warp's four rows: scores with key `lane`, and q S in column `lane`.
    const int i0 = warp * 4;
    float score[4] = {}, o[4] = {};
#pragma unroll 4
    for (int d = 0; d < A.Dk; d += 4) {
      const float4 kk = *reinterpret_cast<const float4*>(&B.k[lane][d]);
      const float s0 = B.s[d][lane], s1 = B.s[d + 1][lane], s2 = B.s[d + 2][lane],
                  s3 = B.s[d + 3][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float4 qq = *reinterpret_cast<const float4*>(&B.q[i0 + r][d]);
        score[r] = fmaf(qq.w, kk.w, fmaf(qq.z, kk.z, fmaf(qq.y, kk.y, fmaf(qq.x, kk.x, score[r]))));
        o[r] = fmaf(qq.w, s3, fmaf(qq.z, s2, fmaf(qq.y, s1, fmaf(qq.x, s0, o[r]))));
      }
    }
    const int none = B.none;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = i0 + r;
      float w = 0.f;
      if (lane <= i) w = i >= none ? NAN : lane + 1 < B.since[i] ? 0.f : exp_of(B.b[i] - B.b[lane]);
      B.p[i][lane] = lane <= i ? score[r] * w : 0.f;
      o[r] *= B.start[i];
    }
    __syncwarp();
#pragma unroll 4
    for (int j = 0; j < i0; ++j) {
      const float x = B.v[j][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = fmaf(B.p[i0 + r][j], x, o[r]);
    }
    // (Values behind a row do not meet its zero weights: they may be no numbers.)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = B.v[i0 + j][lane];
#pragma unroll
      for (int r = j; r < 4; ++r) o[r] = fmaf(B.p[i0 + r][i0 + j], x, o[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (live && t0 + i0 + r < n)
        store1<TYPE>(A.out, ((first + t0 + i0 + r) * A.H + h) * A.Dv + col, o[r]);
    const float keep = B.start[BLOCK - 1];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) s[r] *= keep;
    const int real = min(n - t0, BLOCK);
#pragma unroll 2
    for (int j = 0; j < real; ++j) {
      const float x = B.v[j][lane] * B.rest[j];
#pragma unroll
      for (int r = 0; r < ROWS; r += 4) {
        const float4 kk = *reinterpret_cast<const float4*>(&B.k[j][warp * ROWS + r]);
        s[r] = fmaf(kk.x, x, s[r]);
        s[r + 1] = fmaf(kk.y, x, s[r + 1]);
        s[r + 2] = fmaf(kk.z, x, s[r + 2]);
        s[r + 3] = fmaf(kk.w, x, s[r + 3]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; ++r) B.s[warp * ROWS + r][lane] = s[r];
  }
  if (state != nullptr && live)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int d = warp * ROWS + r;
      if (d < A.Dk) state[(int64_t)d * A.Dv + col] = s[r];
    }
}

template <int TYPE>
static int launch_blocks(const Args& A, void* stream) {
  const cudaError_t e =
      cudaFuncSetAttribute(block_kernel<TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)sizeof(BlockShared));
  KB_REQUIRE(e == cudaSuccess, KB_ERR_DEVICE, "linear attention: shared-memory limit: %s",
             cudaGetErrorString(e));
  const int64_t ctas = (int64_t)A.B * A.H * ((A.Dv + BLOCK - 1) / BLOCK);
  return launch(block_kernel<TYPE>, dim3((unsigned)ctas), dim3(THREADS), sizeof(BlockShared),
                stream, A);
}

template <int TYPE>
static int launch_tokens(const Args& A, int sms, void* stream) {
  const int64_t heads = (int64_t)A.B * A.H;
  // Few heads: their columns on several CTAs each.  (32 heads of 128 x 128, one token: 1 request
  // 3.3 us split and 5.0 whole, 2 requests 3.2 and 4.5, 4 requests 5.5 and 5.1, 9 requests 8.1
  // and 7.2; eight tokens: 8.7 and 10.4 for 1 request, 15.5 and 10.7 for 4.  The rule is the
  // widest heads'.  Narrower ones leave threads of a whole CTA idle and would gain from more
  // splitting: 256 requests, one token, 128 x 64 114 split and 126 whole, 64 x 64 79 and 103,
  // 16 x 16 77 both.)
  if (heads * 2 < sms && A.Dv > 32)
    return launch(token_kernel<TYPE, 32>, dim3((unsigned)(heads * ((A.Dv + 31) / 32))),
                  dim3(THREADS), 0, stream, A);
  return launch(token_kernel<TYPE, 128>, dim3((unsigned)heads), dim3(THREADS), 0, stream, A);
}

static int check(const Args& A, int dtype, int64_t B, int64_t H, int64_t Hq, int64_t Hk,
                 int64_t Dk, int64_t Dv, int64_t total) {
  KB_REQUIRE(H > 0 && Hq > 0 && Hk > 0 && H % Hq == 0 && H % Hk == 0, KB_ERR_BAD_SHAPE,
             "linear attention: heads must be a multiple of the queries' and keys' heads");
  KB_REQUIRE(Dk > 0 && Dk <= WIDEST && Dk % 8 == 0 && Dv > 0 && Dv <= WIDEST && Dv % 8 == 0,
             KB_ERR_UNSUPPORTED, "linear attention: widths must be multiples of 8 up to %d",
             WIDEST);
  KB_REQUIRE(dtype >= 0 && dtype <= 2, KB_ERR_UNSUPPORTED,
             "linear attention: unknown element type");
  KB_REQUIRE(B >= 0 && total >= 0, KB_ERR_BAD_SHAPE, "linear attention: bad shape");
  KB_REQUIRE(B <= ((int64_t)1 << 20) && H <= 65535 && B * H <= ((int64_t)1 << 28) &&
                 total <= ((int64_t)1 << 30),
             KB_ERR_UNSUPPORTED, "linear attention: more than 2^30 tokens or 2^28 heads");
  KB_REQUIRE(A.scale > 0.f, KB_ERR_BAD_SHAPE, "linear attention: the scale must be positive");
  if (A.state != nullptr) {
    // A block of its own for every slot and head: the slots' apart from all heads of one, or the
    // heads' from all slots.
    const int64_t block = Dk * Dv, heads = H - 1, slots = A.slots - 1;
    const bool apart = (heads == 0 || A.state_head >= block) &&
                       (slots == 0 || A.state_slot >= block) &&
                       (heads == 0 || slots == 0 || (A.state_slot - block) / heads >= A.state_head ||
                        (A.state_head - block) / slots >= A.state_slot);
    KB_REQUIRE(apart, KB_ERR_BAD_SHAPE, "linear attention: the states overlap");
  }
  if (B == 0 || total == 0) return KB_OK;
  KB_REQUIRE(A.q && A.k && A.v && A.decay && A.out, KB_ERR_NULL_POINTER,
             "linear attention: NULL pointer");
  const int64_t unit = dtype == 2 ? 3 : 7;   // 16 bytes
  KB_REQUIRE((((uintptr_t)A.q | (uintptr_t)A.k | (uintptr_t)A.v | (uintptr_t)A.out |
               (uintptr_t)A.state) & 15) == 0 &&
                 ((A.q_tok | A.q_head | A.k_tok | A.k_head | A.v_tok | A.v_head) & unit) == 0 &&
                 ((A.state_slot | A.state_head) & 3) == 0,
             KB_ERR_ALIGNMENT, "linear attention: rows must be 16-byte aligned");
  return KB_OK;
}

static Args arguments(const void* q, int64_t q_tok, int64_t q_head, int64_t Hq, const void* k,
                      int64_t k_tok, int64_t k_head, int64_t Hk, const void* v, int64_t v_tok,
                      int64_t v_head, int64_t H, int64_t Dk, int64_t Dv, const float* log_decay,
                      int per_token, float* state, int64_t state_slot, int64_t state_head,
                      int64_t slots, const int32_t* index, float scale, void* out) {
  Args A = {};
  A.q = q;
  A.k = k;
  A.v = v;
  A.q_tok = q_tok;
  A.q_head = q_head;
  A.k_tok = k_tok;
  A.k_head = k_head;
  A.v_tok = v_tok;
  A.v_head = v_head;
  A.decay = log_decay;
  A.decay_tok = per_token ? H : 0;
  A.state = slots > 0 ? state : nullptr;
  A.state_slot = state_slot;
  A.state_head = state_head;
  A.slots = (int)(slots < ((int64_t)1 << 30) ? slots : ((int64_t)1 << 30));
  A.index = index;
  A.H = (int)H;
  A.q_group = Hq > 0 ? (int)(H / Hq) : 1;
  A.k_group = Hk > 0 ? (int)(H / Hk) : 1;
  A.Dk = (int)Dk;
  A.Dv = (int)Dv;
  A.scale = scale;
  A.out = out;
  return A;
}

// On the tensor cores: bf16 prompts of more than a few tokens.
// (32 heads of 128 x 128, token by token and in chunks: 1 request of 8 tokens 8.6 and 11.4 us, of
// 16 14.5 and 11.4; 16 requests of 8 tokens 25 and 30, of 9 27 and 30, of 16 42 and 31; 256
// requests of 4 tokens 306 and 373, of 8 463 and 373.  Other widths cross where these do: 16
// requests of 8 and of 12 tokens, 128 x 64 24 and 28, 32 and 29; 64 x 64 22 and 25, 31 and 25;
// 16 x 16 22 and 24, 30 and 24; 256 requests of 8 heads, of 8 tokens 128 x 64 88 and 75, 16 x 16
// 74 and 62.)
static bool in_chunks(int dtype, int64_t heads, int64_t longest, int sms) {
  return dtype == 0 && longest > (heads > 16 * sms ? 5 : 8);
}

static int run_tokens(const Args& A, int dtype, int sms, void* stream) {
  // Blocks of 32 tokens: from 13 on where each SM has a CTA at most, else from 41.  (32 heads of
  // 128 x 128, token by token and in blocks: 1 request of 12 tokens f16 11.5 and 8.1 us, f32 8.4
  // and 8.1; of 32 26 and 9, 17 and 9; 16 requests of 32 tokens f16 74 and 81, f32 69 and 82; 256
  // requests of 32 f16 1396 and 1260, f32 1082 and 1300.  The rule is the widest heads': with
  // fewer value columns to make the scores again for, blocks win sooner.  16 requests of 32 heads,
  // f16, of 12 and of 40 tokens: 128 x 64 32 and 37, 90 and 71; 64 x 64 31 and 28, 88 and 54;
  // 16 x 16 31 and 13, 88 and 24.)
  const bool few = (int64_t)A.B * A.H * ((A.Dv + BLOCK - 1) / BLOCK) <= sms;
  if (A.cu != nullptr && A.longest > (few ? 12 : 40)) {
    if (dtype == 1) return launch_blocks<1>(A, stream);
    if (dtype == 2) return launch_blocks<2>(A, stream);
  }
  if (dtype == 0) return launch_tokens<0>(A, sms, stream);
  if (dtype == 1) return launch_tokens<1>(A, sms, stream);
  return launch_tokens<2>(A, sms, stream);
}

}  // namespace linear
}  // namespace kb

extern "C" int kb_linear_attention_step(const void* q, int64_t q_token_stride,
                                        int64_t q_head_stride, int64_t Hq, const void* k,
                                        int64_t k_token_stride, int64_t k_head_stride,
                                        int64_t Hk, const void* v, int64_t v_token_stride,
                                        int64_t v_head_stride, int64_t H, int64_t Dk, int64_t Dv,
                                        int dtype, const float* log_decay, int per_token,
                                        float* state, int64_t state_slot_stride,
                                        int64_t state_head_stride, int64_t slots,
                                        const int32_t* state_index, int64_t B, float scale,
                                        void* out, void* stream) {
  namespace ln = kb::linear;
  kb::clear_error();
  ln::Args A = ln::arguments(q, q_token_stride, q_head_stride, Hq, k, k_token_stride,
                             k_head_stride, Hk, v, v_token_stride, v_head_stride, H, Dk, Dv,
                             log_decay, per_token, state, state_slot_stride, state_head_stride,
                             slots, state_index, scale, out);
  const int st = ln::check(A, dtype, B, H, Hq, Hk, Dk, Dv, B);
  if (st != KB_OK || B == 0) return st;
  A.total = B;
  A.B = (int)B;
  A.longest = 1;
  const int dev = kb::bind_stream_device(stream);
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  return ln::run_tokens(A, dtype, kb::num_sms(dev), stream);
}

extern "C" int kb_linear_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                   int64_t Hq, const void* k, int64_t k_token_stride,
                                   int64_t k_head_stride, int64_t Hk, const void* v,
                                   int64_t v_token_stride, int64_t v_head_stride, int64_t H,
                                   int64_t Dk, int64_t Dv, int dtype, const float* log_decay,
                                   int per_token, float* state, int64_t state_slot_stride,
                                   int64_t state_head_stride, int64_t slots,
                                   const int32_t* state_index, const int32_t* cu_tokens,
                                   int64_t B, int64_t total, int64_t max_tokens, float scale,
                                   void* out, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  namespace ln = kb::linear;
  kb::clear_error();
  ln::Args A = ln::arguments(q, q_token_stride, q_head_stride, Hq, k, k_token_stride,
                             k_head_stride, Hk, v, v_token_stride, v_head_stride, H, Dk, Dv,
                             log_decay, per_token, state, state_slot_stride, state_head_stride,
                             slots, state_index, scale, out);
  const int st = ln::check(A, dtype, B, H, Hq, Hk, Dk, Dv, total);
  if (st != KB_OK || B == 0 || total == 0) return st;
  KB_REQUIRE(cu_tokens, KB_ERR_NULL_POINTER, "linear attention: NULL pointer");
  KB_REQUIRE(max_tokens > 0, KB_ERR_BAD_SHAPE, "linear attention: tokens but max_tokens 0");
  A.cu = cu_tokens;
  A.total = total;
  A.B = (int)B;
  A.longest = (int)(max_tokens < total ? max_tokens : total);
  const int dev = kb::bind_stream_device(stream);
  A.err = kb::device_error_word(dev);
  KB_REQUIRE(A.err != nullptr, KB_ERR_LAUNCH, "device error word unavailable");
  const int sms = kb::num_sms(dev);
  if (ln::in_chunks(dtype, B * H, A.longest, sms))
    return ln::launch_chunks(A, Hq, Hk, sms, workspace, workspace_bytes, stream);
  return ln::run_tokens(A, dtype, sms, stream);
}

extern "C" size_t kb_linear_attention_workspace_size(int64_t B, int64_t H, int64_t Dk, int64_t Dv,
                                                     int dtype, int64_t total,
                                                     int64_t max_tokens) {
  namespace ln = kb::linear;
  const int64_t longest = max_tokens < total ? max_tokens : total;
  if (B <= 0 || H <= 0 || Dk <= 0 || Dv <= 0) return 0;
  const int sms = kb::num_sms(kb::bind_stream_device(nullptr));
  if (!ln::in_chunks(dtype, B * H, longest, sms)) return 0;
  return ln::chunk_workspace(B, H, Dk, Dv, total, longest, sms);
}
