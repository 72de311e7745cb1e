// kb_linear.cuh - what the two forms of linear attention share.
#pragma once

#include "kb_attn.cuh"

namespace kb {
namespace linear {

struct Args {
  const void *q, *k, *v;                     // [tokens, heads, width], unit inner stride
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  const float* decay;                        // [tokens, H], or [H] with decay_tok 0
  int64_t decay_tok;
  float* state;                              // [slots][H][Dk][Dv] or NULL: from zero, not kept
  int64_t state_slot, state_head;
  const int* index;                          // slot of each request, NULL: its number
  int slots;
  const int* cu;                             // NULL: one token a request
  void* out;                                 // [tokens, H, Dv] contiguous
  int64_t total;
  int B, H, q_group, k_group, Dk, Dv;        // groups: heads that share q, k
  int longest;                               // tokens of a request at most
  float scale;
  uint32_t* err;
};

// A request's tokens [first, first + n), and where its rows end: past first + n where it has more
// tokens than it may.
__device__ __forceinline__ int request_tokens(const Args& A, int b, int64_t& first, int64_t& end) {
  if (A.cu == nullptr) {
    first = b;
    end = b + 1;
    return 1;
  }
  attn::request_rows(A.cu, b, A.total, first, end);
  return (int)min(end - first, (int64_t)A.longest);
}

__device__ __forceinline__ int request_tokens(const Args& A, int b, int64_t& first) {
  int64_t end;
  return request_tokens(A, b, first, end);
}

// Where a request's state lies; NULL: it starts from zero and is not kept.
__device__ __forceinline__ float* request_state(const Args& A, int b, int h) {
  if (A.state == nullptr) return nullptr;
  const int slot = A.index ? __ldg(A.index + b) : b;
  if (slot < 0) return nullptr;
  if (slot >= A.slots) {
    atomicOr(A.err, ERR_PAGE);
    return nullptr;
  }
  return A.state + slot * A.state_slot + h * A.state_head;
}

// A decay's logarithm as it counts: above 0 it is no decay, and counts as 0.
__device__ __forceinline__ float decay_of(float g) { return g > 0.f ? 0.f : g; }

// Prompts in chunks on the tensor cores (kb_linear_chunk.cu), bf16.
size_t chunk_workspace(int64_t B, int64_t H, int64_t Dk, int64_t Dv, int64_t total,
                       int64_t longest, int sms);
int launch_chunks(const Args& A, int64_t Hq, int64_t Hk, int sms, void* workspace,
                  size_t workspace_bytes, void* stream);

}  // namespace linear
}  // namespace kb
