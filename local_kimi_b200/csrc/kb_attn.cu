// kb_attn.cu - host helpers shared by the attention kernels.
#include "kb_attn.cuh"

namespace kb {
namespace attn {

int check_heads(int64_t Hq, int64_t Hkv, int64_t Dk, int64_t Dv, int dtype) {
  KB_REQUIRE(Hq > 0 && Hkv > 0 && Hq % Hkv == 0, KB_ERR_BAD_SHAPE,
             "attention: query heads must be a multiple of key/value heads");
  KB_REQUIRE(Dk > 0 && Dk <= 192 && Dk % 8 == 0 && Dv > 0 && Dv <= 128 && Dv % 8 == 0,
             KB_ERR_UNSUPPORTED,
             "attention: head widths must be multiples of 8, keys up to 192 and values up to 128");
  KB_REQUIRE(dtype == 0 || dtype == 1, KB_ERR_UNSUPPORTED, "attention: unknown element type");
  return KB_OK;
}

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

int make_map_4d(CUtensorMap* map, const void* base, int f16, const int64_t (&dims)[4],
                const int64_t (&strides)[3], int rows, int box2) {
  auto enc = encode_fn();
  KB_REQUIRE(enc != nullptr, KB_ERR_DEVICE, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t d[4], s[3];
  for (int i = 0; i < 4; ++i) d[i] = (cuuint64_t)dims[i];
  for (int i = 0; i < 3; ++i) {
    // The stride of an extent of one is never used; keep it a legal one.
    KB_REQUIRE(dims[i + 1] == 1 || strides[i] > 0, KB_ERR_BAD_SHAPE,
               "attention: strides must be positive");
    s[i] = (cuuint64_t)(dims[i + 1] == 1 ? 16 : strides[i] * 2);
  }
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, (cuuint32_t)box2, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(
      map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
      const_cast<void*>(base), d, s, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  KB_REQUIRE(r == CUDA_SUCCESS, KB_ERR_DEVICE, "attention: tensor map encoding failed (%d)",
             (int)r);
  return KB_OK;
}

int allow_smem(const void* kernel, int bytes, bool (&done)[64], std::mutex& mu) {
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  KB_REQUIRE(e == cudaSuccess && dev >= 0 && dev < 64, KB_ERR_DEVICE,
             "attention: no usable current device (%s)", cudaGetErrorString(e));
  std::lock_guard<std::mutex> lock(mu);
  if (done[dev]) return KB_OK;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  KB_REQUIRE(e == cudaSuccess, KB_ERR_DEVICE,
             "attention: setting the shared-memory limit failed: %s", cudaGetErrorString(e));
  done[dev] = true;
  return KB_OK;
}

}  // namespace attn
}  // namespace kb
