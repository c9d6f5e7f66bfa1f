// Dots of a few rows with 4-bit weights and a scale for each group along k.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string>

#include "kernels.h"

namespace b200sd {
namespace {

struct W4Args {
  const void* x;
  const uint8_t* w;
  const void* scale;
  const uint8_t* zero;
  const void* bias;
  void* d;
  int32_t m, n, k, group;
  int32_t x_dtype, scale_dtype, bias_dtype, d_dtype, is_signed;
};

__device__ __forceinline__ float LoadAs(const void* p, int64_t i, int32_t dtype) {
  if (dtype == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == kF16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

// One warp per weight row and four rows of x.
__global__ void __launch_bounds__(128) w4_dot_kernel(const W4Args a) {
  const int row = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32, m0 = blockIdx.y * 4;
  if (row >= a.n) return;
  const int groups = a.k / a.group;
  float acc[4] = {};
  for (int k0 = lane * 8; k0 < a.k; k0 += 256) {
    const uint32_t word = *reinterpret_cast<const uint32_t*>(a.w + static_cast<int64_t>(row) * (a.k / 2) + k0 / 2);
    const int64_t g = static_cast<int64_t>(row) * groups + k0 / a.group;
    const float s = LoadAs(a.scale, g, a.scale_dtype);
    const int z = a.is_signed ? 8 : a.zero[g] & 15;
    for (int i = 0; i < 8; ++i) {
      int q = word >> (4 * i) & 15;
      if (a.is_signed) q ^= 8;
      const float w = static_cast<float>(q - z) * s;
      for (int r = 0; r < 4; ++r)
        if (m0 + r < a.m) acc[r] += w * LoadAs(a.x, static_cast<int64_t>(m0 + r) * a.k + k0 + i, a.x_dtype);
    }
  }
  for (int r = 0; r < 4; ++r) {
    for (int o = 16; o > 0; o /= 2) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
    if (lane == 0 && m0 + r < a.m) {
      const float y = acc[r] + (a.bias != nullptr ? LoadAs(a.bias, row, a.bias_dtype) : 0.0f);
      const int64_t at = static_cast<int64_t>(m0 + r) * a.n + row;
      if (a.d_dtype == kBF16) static_cast<__nv_bfloat16*>(a.d)[at] = __float2bfloat16_rn(y);
      else if (a.d_dtype == kF16) static_cast<__half*>(a.d)[at] = __float2half_rn(y);
      else static_cast<float*>(a.d)[at] = y;
    }
  }
}

}  // namespace

Status ValidateDotW4(const B200SD_DotW4& a, bool check_pointers) {
  auto bad = [](const std::string& m) { return Status::Error(kInvalidArgument, m); };
  auto is_float = [](int32_t t) { return t == kBF16 || t == kF16 || t == kF32; };
  if (a.struct_size < sizeof(a)) return bad("B200SD_DotW4.struct_size is smaller than this library's struct");
  if (!(a.x_dtype == kBF16 || a.x_dtype == kF16)) return bad("x must be BF16 or F16");
  if (!(a.weight_type == kS4 || a.weight_type == kU4)) return bad("weight_type must be S4 or U4");
  if (!is_float(a.scale_dtype)) return bad("scales must be BF16, F16 or F32");
  if (a.d_dtype != a.x_dtype && a.d_dtype != kF32) return bad("the result must have x's type or F32");
  if (a.epilogue != B200SD_EPILOGUE_DEFAULT && a.epilogue != B200SD_EPILOGUE_BIAS) return Status::Error(kUnimplemented, "the 4-bit dot knows the epilogues DEFAULT and BIAS only");
  const bool has_bias = a.epilogue == B200SD_EPILOGUE_BIAS;
  if (has_bias && !is_float(a.bias_dtype)) return bad("bias must be BF16, F16 or F32");
  if (a.m < 0 || a.n <= 0 || a.k <= 0) return bad("n and k must be positive and m not negative");
  if (a.n > (1 << 24) || a.k > (1 << 24)) return bad("dimension too large");
  if (!(a.group == 32 || a.group == 64 || (a.group > 0 && a.group % 128 == 0)) || a.k % a.group) return bad("group must be 32, 64 or a multiple of 128, and divide k");
  if (a.m > 64) return Status::Error(kUnimplemented, "the 4-bit dot is for few rows: m must be at most 64");
  if (!check_pointers || a.m == 0) return Status::Ok();
  if (a.x == nullptr || a.w == nullptr || a.scale == nullptr || a.d == nullptr) return bad("x, w, scale and d must not be null");
  if (a.weight_type == kU4 && a.zero == nullptr) return bad("U4 weights need zero points");
  if (has_bias && a.bias == nullptr) return bad("epilogue adds a vector bias but bias is null");
  if ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w)) % 16) return bad("x and w must be 16-byte aligned");
  const auto aligned = [](const void* p, int32_t t) { return reinterpret_cast<uintptr_t>(p) % (t == kF32 ? 4 : 2) == 0; };
  if (!aligned(a.scale, a.scale_dtype) || !aligned(a.d, a.d_dtype) || (has_bias && !aligned(a.bias, a.bias_dtype))) return bad("scale, bias and d must be aligned to their elements");
  return Status::Ok();
}

Status LaunchDotW4(const B200SD_DotW4& a, cudaStream_t stream, LaunchStats* stats) {
  if (a.m == 0) return Status::Ok();
  const W4Args args{a.x, static_cast<const uint8_t*>(a.w), a.scale, static_cast<const uint8_t*>(a.zero), a.epilogue == B200SD_EPILOGUE_BIAS ? a.bias : nullptr, a.d,
                    static_cast<int32_t>(a.m), static_cast<int32_t>(a.n), static_cast<int32_t>(a.k), static_cast<int32_t>(a.group),
                    a.x_dtype, a.scale_dtype, a.bias_dtype, a.d_dtype, a.weight_type == kS4};
  const dim3 grid(static_cast<unsigned>((a.n + 3) / 4), static_cast<unsigned>((a.m + 3) / 4));
  w4_dot_kernel<<<grid, 128, 0, stream>>>(args);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return Status::Error(kInternal, std::string("w4_dot_kernel launch: ") + cudaGetErrorString(e));
  stats->launches = 1;
  return Status::Ok();
}

}  // namespace b200sd
