// kb_linear.cu - linear attention with a decay for each head, token by token.
//
// For head h of a request, with the state S [Dk, Dv] in fp32:
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale * q_t S_t
// One token a request (decoding), or a few: the state is read once, updated in registers
// and written once.  A CTA has a head's state, or, where there are few heads, 32 of its
// columns (they are independent): 256 threads, four columns and Dk / 8 (Dk / 32) rows each.
// The sums over the rows meet in shared memory, one barrier a token.  Longer bf16 prompts go in
// chunks (kb_linear_chunk.cu).
//
// Bound: HBM, the states read and written: 256 requests of 32 heads of 128 x 128 move 1.08 GB in
// 177 us, 6.07 TB/s.  One request, 2.8 us (4 MB): a launch and one trip to memory.
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

  // Rows outside every request: zero.
  if (A.cu != nullptr) {
    const int64_t lead = min(max((int64_t)A.cu[0], (int64_t)0), A.total);
    const int64_t tail = min(max((int64_t)A.cu[A.B], lead), A.total);
    const int64_t width = (int64_t)A.H * A.Dv, spare = (lead + A.total - tail) * width;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + tid; i < spare;
         i += (int64_t)gridDim.x * THREADS)
      store1<TYPE>(A.out, i < lead * width ? i : i - lead * width + tail * width, 0.f);
  }
  int64_t first;
  const int n = request_tokens(A, b, first);
  if (n <= 0) return;
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

template <int TYPE>
static int launch_tokens(const Args& A, int sms, void* stream) {
  const int64_t heads = (int64_t)A.B * A.H;
  // Few heads: their columns on several CTAs each.  (32 heads of 128 x 128, one token: 1 request
  // 3.3 us split and 5.0 whole, 2 requests 3.2 and 4.5, 4 requests 5.5 and 5.1, 9 requests 8.1
  // and 7.2; eight tokens: 8.7 and 10.4 for 1 request, 15.5 and 10.7 for 4.)
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

// Token by token for a few tokens, and for types that the tensor cores' form does not take.
// (32 heads, token by token and in chunks: 1 request of 8 tokens 8.5 and 11.2 us, of 16 14.5 and
// 11.2; 16 requests of 8 tokens 25 and 32, of 16 42 and 32; 256 requests of 4 tokens 308 and 376,
// of 8 463 and 381.)
static bool in_chunks(int dtype, int64_t heads, int64_t longest, int sms) {
  return dtype == 0 && longest > (heads > 16 * sms ? 5 : 8);
}

static int run_tokens(const Args& A, int dtype, int sms, void* stream) {
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
