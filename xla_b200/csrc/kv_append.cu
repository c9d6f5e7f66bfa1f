// Appending keys and values to the paged 8-bit cache.
//
// One block per (page that new tokens reach, head, sequence, keys or values).  It takes the largest magnitude of the
// page's new tokens, raises the page's scale to the power of two at which that fits, re-rounds the page's earlier
// codes where the scale grew, and stores the new ones.  A scale that is a power of two costs an 8-bit float no
// precision -- it only moves the range -- and makes the re-rounding of earlier codes a shift of their exponents, which
// is exact down to the subnormals; a scale of amax / max would round every earlier code of the page again each time a
// token raises it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv_cache.cuh"

namespace b200sd {
namespace {

constexpr int kThreads = 128;

struct AppendArgs {
  const void* fresh[2];          // keys, values
  uint8_t* pages[2];
  float* scale[2];
  const int32_t* page_table;
  const int32_t* seq_lens;
  const int32_t* new_lens;
  int32_t new_tokens, kv_heads, head_dim, page_tokens;
  int64_t num_pages, table_width;
  uint32_t* status;
};

template <typename T> __device__ __forceinline__ float ToFloat(T x);
template <> __device__ __forceinline__ float ToFloat(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float ToFloat(__nv_bfloat16 x) { return __bfloat162float(x); }

// Two values to two codes, the first in the low byte: nearest, ties to even, saturating.
template <int kCode>
__device__ __forceinline__ uint32_t Encode2(float lo, float hi) {
  if constexpr (kCode == kS8) {
    auto one = [](float x) { return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x == x ? x : 0.0f, -127.0f), 127.0f))) & 255u; };
    return one(lo) | one(hi) << 8;
  } else {
    uint16_t r;
    if constexpr (kCode == kF8E4M3FN) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
  }
}
// Two codes to the f32 values they are, exactly.
template <int kCode>
__device__ __forceinline__ float2 Decode2(uint32_t codes) {
  if constexpr (kCode == kS8) {
    return make_float2(static_cast<float>(static_cast<int8_t>(codes)), static_cast<float>(static_cast<int8_t>(codes >> 8)));
  } else {
    uint32_t h;
    const uint16_t c = static_cast<uint16_t>(codes);
    if constexpr (kCode == kF8E4M3FN) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
    else asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(c));
    return __half22float2(*reinterpret_cast<__half2*>(&h));
  }
}

// Eight values divided by the scale (one division each, as the definition has it) and encoded.  `inverse` is not 0
// where the scale is a power of two: the product with it is the same quotient, rounded once.
template <int kCode>
__device__ __forceinline__ uint2 EncodeScaled(const float (&x)[8], float scale, float inverse) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = inverse != 0.0f ? x[i] * inverse : __fdiv_rn(x[i], scale);
  return make_uint2(Encode2<kCode>(y[0], y[1]) | Encode2<kCode>(y[2], y[3]) << 16, Encode2<kCode>(y[4], y[5]) | Encode2<kCode>(y[6], y[7]) << 16);
}

template <int kCode, typename T>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendArgs a) {
  __shared__ uint32_t warp_max[kThreads / 32];
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, head = blockIdx.y;
  const int32_t length = a.seq_lens[b];
  const int64_t len = length > 0 ? length : 0;
  const int64_t count = a.new_lens != nullptr ? min(max(a.new_lens[b], 0), a.new_tokens) : a.new_tokens;
  const int64_t start = len - count;                       // position of the first new token; below 0 where the first ones are padding
  const int64_t first = start > 0 ? start : 0;
  const int64_t index = first / a.page_tokens + blockIdx.x;
  const int64_t base = index * a.page_tokens;              // position of the page's first slot
  const int64_t lo = first > base ? first : base;
  const int64_t hi = len < base + a.page_tokens ? len : base + a.page_tokens;
  if (length < 0 && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.status, kStatusBadPage);
  if (lo >= hi) return;
  const int64_t page = index < a.table_width ? a.page_table[b * a.table_width + index] : -1;
  if (page < 0 || page >= a.num_pages) {
    if (threadIdx.x == 0) atomicOr(a.status, kStatusBadPage);
    return;
  }
  float* scale_at = a.scale[which] + page * a.kv_heads + head;
  uint8_t* codes = a.pages[which] + (page * a.kv_heads + head) * a.page_tokens * a.head_dim;
  const int chunks = a.head_dim / 8;                       // of eight values
  const int held = static_cast<int>(lo - base), total = static_cast<int>(hi - lo) * chunks;
  const float before = held > 0 ? *scale_at : 0.0f;
  // Row `t` of the page's new tokens: token lo + t - start of the call.
  const T* rows = static_cast<const T*>(a.fresh[which]) + ((static_cast<int64_t>(b) * a.new_tokens + (lo - start)) * a.kv_heads + head) * a.head_dim;
  const int64_t row_stride = static_cast<int64_t>(a.kv_heads) * a.head_dim;
  auto load = [&](int c, float (&x)[8]) {
    const int t = c / chunks, d = (c - t * chunks) * 8;
    const uint4 raw = *reinterpret_cast<const uint4*>(rows + t * row_stride + d);
    const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ToFloat(v[i]);
  };
  uint32_t top = 0;                                        // bit pattern of the largest finite magnitude
  for (int c = threadIdx.x; c < total; c += kThreads) {
    float x[8];
    load(c, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = __float_as_uint(x[i]) & 0x7fffffffu;
      if (bits < 0x7f800000u) top = max(top, bits);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) top = max(top, warp_max[i]);
  // top = f * 2^e with f in [0.5, 1); the type's largest is F * 2^E: the scale is 2^(e - E), one more where f > F.
  constexpr uint32_t kLimit = static_cast<uint32_t>((CodeTraits<kCode>::kFraction * 2 - 1) * 8388608.0f);
  int power = static_cast<int>(top >> 23) - 126 - CodeTraits<kCode>::kExponent + ((top & 0x7fffffu) > kLimit ? 1 : 0);
  power = max(power, -126);
  const float scale = fmaxf(before, __uint_as_float(static_cast<uint32_t>(power + 127) << 23));
  const float inverse = (__float_as_uint(scale) & 0x7fffffu) == 0 ? 1.0f / scale : 0.0f;
  if (threadIdx.x == 0) *scale_at = scale;
  if (held > 0 && scale != before) {
    for (int c = threadIdx.x; c < held * chunks; c += kThreads) {
      uint2* at = reinterpret_cast<uint2*>(codes) + c;
      const uint2 old = *at;
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = Decode2<kCode>((i < 2 ? old.x : old.y) >> (i % 2 * 16));
        x[2 * i] = v.x * before;
        x[2 * i + 1] = v.y * before;
      }
      *at = EncodeScaled<kCode>(x, scale, inverse);
    }
  }
  for (int c = threadIdx.x; c < total; c += kThreads) {
    float x[8];
    load(c, x);
    *(reinterpret_cast<uint2*>(codes) + held * chunks + c) = EncodeScaled<kCode>(x, scale, inverse);
  }
}

template <int kCode>
void Launch(const B200SD_KvCacheAppend& a, const AppendArgs& args, dim3 grid, cudaStream_t stream) {
  if (a.new_dtype == kBF16) kv_append_kernel<kCode, __nv_bfloat16><<<grid, kThreads, 0, stream>>>(args);
  else kv_append_kernel<kCode, __half><<<grid, kThreads, 0, stream>>>(args);
}

}  // namespace

Status ValidateKvCacheAppend(const B200SD_KvCacheAppend& a, bool check_pointers) {
  if (a.struct_size < sizeof(a)) return Status::Error(kInvalidArgument, "B200SD_KvCacheAppend.struct_size is smaller than this library's struct");
  Status st = ValidateCache(a, a.new_dtype, check_pointers);
  if (!st.ok()) return st;
  if (a.new_tokens > (int64_t{1} << 30)) return Status::Error(kInvalidArgument, "too many new tokens");
  if (!check_pointers || a.batch == 0 || a.new_tokens == 0) return Status::Ok();
  if (a.k_new == nullptr || a.v_new == nullptr) return Status::Error(kInvalidArgument, "k_new and v_new must not be null");
  if ((reinterpret_cast<uintptr_t>(a.k_new) | reinterpret_cast<uintptr_t>(a.v_new)) % 16) return Status::Error(kInvalidArgument, "k_new and v_new must be 16-byte aligned");
  return Status::Ok();
}

Status LaunchKvCacheAppend(const B200SD_KvCacheAppend& a, cudaStream_t stream, LaunchStats* stats) {
  if (a.batch == 0 || a.new_tokens == 0) return Status::Ok();
  AppendArgs args{{a.k_new, a.v_new}, {static_cast<uint8_t*>(a.k_pages), static_cast<uint8_t*>(a.v_pages)}, {a.k_scale, a.v_scale},
                  a.page_table, a.seq_lens, a.new_lens,
                  static_cast<int32_t>(a.new_tokens), static_cast<int32_t>(a.kv_heads), static_cast<int32_t>(a.head_dim), static_cast<int32_t>(a.page_tokens),
                  a.num_pages, a.table_width, StatusWordPtr()};
  // n tokens in a row reach at most (n - 1 + page - 1) / page + 1 pages.
  const dim3 grid(static_cast<unsigned>((a.new_tokens + a.page_tokens - 2) / a.page_tokens + 1), static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(2 * a.batch));
  switch (a.cache_dtype) {
    case kF8E4M3FN: Launch<kF8E4M3FN>(a, args, grid, stream); break;
    case kF8E5M2: Launch<kF8E5M2>(a, args, grid, stream); break;
    default: Launch<kS8>(a, args, grid, stream); break;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return Status::Error(kInternal, std::string("kv_append_kernel launch: ") + cudaGetErrorString(e));
  stats->launches = 1;
  return Status::Ok();
}

}  // namespace b200sd
