// Appending keys and values to the paged 8-bit cache.
//
// One warp for 16 slots of a page that new tokens reach, for each head, of the keys or the values; the warps of a page, and
// of as many pages as make 128 slots, form a block.  They take the largest magnitude of the page's new tokens, raise the
// page's scale to the power of two at which that fits, re-round the page's earlier codes where the scale grew, and store the
// new ones.  A scale that is a power of two costs an 8-bit float no precision -- it only moves the range -- and makes the
// re-rounding of earlier codes a shift of their exponents, which is exact down to the subnormals; a scale of amax / max
// would round every earlier code of the page again each time a token raises it.  An 8-bit integer pays for it: up to one of its
// seven bits goes unused, and earlier codes lose the bits by which the scale grows.
//
// 4096 tokens for each of 8 sequences, 8 heads of 128, bf16 to e4m3, take 26.5 us (123 MB, 4.6 TB/s; the bytes alone 18.8).
// A block's loads are all under way at once, behind its length and its page, and their rounding follows; only other blocks
// fill its pauses: four to an SM, at 64 registers and a few of them spilled, where three took 29.4 us, and warps of 8 slots
// in blocks of 512 threads 40.  With a warp for a whole page of 64 slots, which looks at its values in one pass and reads
// them again to round them, it was 52 us.  One token for each sequence of a batch takes 7.7 us, the host's part of the call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.cuh"

namespace b200sd {
namespace {

constexpr int kMostWarps = 8;                    // of a block
constexpr int kKept = 8;                         // pieces of eight values that a lane keeps from the first look to the rounding

struct AppendArgs {
  const void* fresh[2];          // keys, values
  uint8_t* pages[2];
  float* scale[2];
  const int32_t* page_table;
  const int32_t* seq_lens;
  const int32_t* new_lens;
  int32_t new_tokens, kv_heads, head_dim, page_tokens;
  uint32_t chunk_inverse;         // 2^32 / (head_dim / 8), rounded up
  int64_t num_pages, table_width;
  uint32_t* status;
};

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

// Eight values divided by the scale (one division each, as the definition has it) and encoded.
template <int kCode, bool kByPower>
__device__ __forceinline__ uint2 EncodeScaled(const float (&x)[8], float scale, float inverse) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = kByPower ? x[i] * inverse : __fdiv_rn(x[i], scale);
  return make_uint2(Encode2<kCode>(y[0], y[1]) | Encode2<kCode>(y[2], y[3]) << 16, Encode2<kCode>(y[4], y[5]) | Encode2<kCode>(y[6], y[7]) << 16);
}

template <typename T>
__device__ __forceinline__ void Unpack(const uint4& raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 v;
    if constexpr (sizeof(T) == 2 && std::is_same_v<T, __nv_bfloat16>) v = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    else v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = v.x, x[2 * i + 1] = v.y;
  }
}

// The new tokens of a page's slots and where their codes go.
template <int kCode, typename T>
struct PageWork {
  const T* rows;                                // token t of them at rows + t * row_stride, less than 2^26 values on
  int32_t row_stride;
  uint8_t* codes;
  int chunks, held, total;                      // chunks of eight of a token; earlier tokens of the page; chunks of the new ones
  uint32_t inverse_chunks;

  __device__ __forceinline__ uint4 Load(int c) const {
    const int t = static_cast<int>(__umulhi(c, inverse_chunks)), d = (c - t * chunks) * 8;      // c below 2^13, two chunks at least
    return *reinterpret_cast<const uint4*>(rows + t * row_stride + d);
  }
  // The rounding of everything, by lanes `lane` of `lanes`; `kept` are the first chunks of this lane.
  template <bool kByPower>
  __device__ __forceinline__ void Store(const uint4 (&kept)[kKept], int lane, int lanes, float before, float scale, float inverse) const {
    if (held > 0 && scale != before) {
#pragma unroll 1
      for (int c = lane; c < held * chunks; c += lanes) {
        uint2* at = reinterpret_cast<uint2*>(codes) + c;
        const uint2 old = *at;
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = Decode2<kCode>((i < 2 ? old.x : old.y) >> (i % 2 * 16));
          x[2 * i] = v.x * before;
          x[2 * i + 1] = v.y * before;
        }
        *at = EncodeScaled<kCode, kByPower>(x, scale, inverse);
      }
    }
    auto store = [&](const uint4& raw, int c) {
      float x[8];
      Unpack<T>(raw, x);
      *(reinterpret_cast<uint2*>(codes) + held * chunks + c) = EncodeScaled<kCode, kByPower>(x, scale, inverse);
    };
    if (kKept * lanes <= total) {
#pragma unroll
      for (int j = 0; j < kKept; ++j) store(kept[j], lane + j * lanes);
    } else {
#pragma unroll
      for (int j = 0; j < kKept; ++j)
        if (lane + j * lanes < total) store(kept[j], lane + j * lanes);
    }
#pragma unroll 1
    for (int c = lane + kKept * lanes; c < total; c += lanes) store(Load(c), c);
  }
};

template <int kCode, typename T>
__global__ void __launch_bounds__(32 * kMostWarps, 4) kv_append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ uint32_t warp_max[kMostWarps];
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, head = blockIdx.y, warp = threadIdx.x / 32;
  const int page_warps = a.page_tokens / 16, lanes = 32 * page_warps, lane = threadIdx.x % lanes;
  griddep_wait();
  if (threadIdx.x == 0) griddep_launch_dependents();
  const int32_t length = a.seq_lens[b];
  const int64_t len = length > 0 ? length : 0;
  const int64_t count = a.new_lens != nullptr ? min(max(a.new_lens[b], 0), a.new_tokens) : a.new_tokens;
  const int64_t start = len - count;                       // position of the first new token; below 0 where the first ones are padding
  const int64_t first = start > 0 ? start : 0;
  const int64_t block_index = first / a.page_tokens + blockIdx.x * (blockDim.x / lanes);
  if (length < 0 && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.status, kStatusBadPage);
  if (first >= len || block_index * a.page_tokens >= len) return;         // nothing for the whole block
  const int64_t index = block_index + threadIdx.x / lanes;
  const int64_t base = index * a.page_tokens;              // position of the page's first slot
  const int64_t lo = first > base ? first : base;
  const int64_t hi = len < base + a.page_tokens ? len : base + a.page_tokens;
  int64_t page = lo < hi && index < a.table_width ? a.page_table[b * a.table_width + index] : -1;
  if (page < 0 || page >= a.num_pages) {
    if (lo < hi && lane == 0) atomicOr(a.status, kStatusBadPage);
    page = -1;
  }
  PageWork<kCode, T> work;
  work.chunks = a.head_dim / 8;
  work.held = static_cast<int>(lo - base);
  work.total = page >= 0 ? static_cast<int>(hi - lo) * work.chunks : 0;
  work.inverse_chunks = a.chunk_inverse;
  // Row `t` of the page's new tokens: token lo + t - start of the call.
  work.rows = static_cast<const T*>(a.fresh[which]) + ((static_cast<int64_t>(b) * a.new_tokens + (lo - start)) * a.kv_heads + head) * a.head_dim;
  work.row_stride = a.kv_heads * a.head_dim;
  work.codes = a.pages[which] + (page * a.kv_heads + head) * a.page_tokens * a.head_dim;
  float* scale_at = a.scale[which] + page * a.kv_heads + head;
  const float before = page >= 0 && work.held > 0 ? *scale_at : 0.0f;

  // A lane's chunks are kept, all their loads under way at once (16 slots of 128 columns are 8 for each lane; of wider heads
  // the rest is read twice).  From one to the next, `lanes` chunks on, it is some tokens and `rest` chunks, or a token more
  // where that passes the token's end; a page full of new tokens needs no other test.
  uint4 kept[kKept];
  const int tokens_on = static_cast<int>(__umulhi(lanes, work.inverse_chunks)), rest = lanes - tokens_on * work.chunks;
  const int first_token = static_cast<int>(__umulhi(lane, work.inverse_chunks));
  int place = lane - first_token * work.chunks;             // of the chunk in its token
  int offset = first_token * work.row_stride + place * 8;
  const int on = tokens_on * work.row_stride + rest * 8, over = work.row_stride - work.chunks * 8;
  auto next = [&] {
    place += rest;
    offset += on;
    if (place >= work.chunks) place -= work.chunks, offset += over;
  };
  if (kKept * lanes <= work.total) {
#pragma unroll
    for (int j = 0; j < kKept; ++j, next()) kept[j] = *reinterpret_cast<const uint4*>(work.rows + offset);
  } else {
#pragma unroll
    for (int j = 0; j < kKept; ++j, next()) {
      kept[j] = make_uint4(0, 0, 0, 0);
      if (lane + j * lanes < work.total) kept[j] = *reinterpret_cast<const uint4*>(work.rows + offset);
    }
  }
  constexpr uint32_t kInfinity = std::is_same_v<T, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
  auto most_of = [](const uint4& v, uint32_t so_far) {     // the larger magnitudes, as the type's bits, in both halves
    return __vmaxu2(__vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)), so_far);
  };
  auto finite_of = [](uint4 v) {                           // infinities and NaN taken out
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((w[i] & kInfinity) == kInfinity) w[i] &= 0xffff0000u;
      if ((w[i] >> 16 & kInfinity) == kInfinity) w[i] &= 0x0000ffffu;
    }
    return v;
  };
  uint32_t both = 0;
#pragma unroll
  for (int j = 0; j < kKept; ++j) both = most_of(kept[j], both);
#pragma unroll 1
  for (int c = lane + kKept * lanes; c < work.total; c += lanes) both = most_of(work.Load(c), both);
  if (max(both & 0xffffu, both >> 16) >= kInfinity) {      // rare: look again, at the finite ones
    both = 0;
#pragma unroll
    for (int j = 0; j < kKept; ++j) both = most_of(finite_of(kept[j]), both);
#pragma unroll 1
    for (int c = lane + kKept * lanes; c < work.total; c += lanes) both = most_of(finite_of(work.Load(c)), both);
  }
  const uint32_t bits16 = __reduce_max_sync(0xffffffffu, max(both & 0xffffu, both >> 16));
  uint32_t top = std::is_same_v<T, __nv_bfloat16> ? bits16 << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(bits16))));
  if (page_warps > 1) {
    if (threadIdx.x % 32 == 0) warp_max[warp] = top;
    __syncthreads();
    for (int i = 0; i < page_warps; ++i) top = max(top, warp_max[warp / page_warps * page_warps + i]);
  }
  if (page < 0) return;
  // top = f * 2^e with f in [0.5, 1); the type's largest is F * 2^E: the scale is 2^(e - E), one more where f > F.
  constexpr uint32_t kLimit = static_cast<uint32_t>((CodeTraits<kCode>::kFraction * 2 - 1) * 8388608.0f);
  int power = static_cast<int>(top >> 23) - 126 - CodeTraits<kCode>::kExponent + ((top & 0x7fffffu) > kLimit ? 1 : 0);
  power = max(power, -126);
  const float scale = fmaxf(before, __uint_as_float(static_cast<uint32_t>(power + 127) << 23));
  if (lane == 0) *scale_at = scale;
  // By a power of two the product with its inverse is the quotient, rounded once.
  if ((__float_as_uint(scale) & 0x7fffffu) == 0) work.template Store<true>(kept, lane, lanes, before, scale, 1.0f / scale);
  else work.template Store<false>(kept, lane, lanes, before, scale, 0.0f);
}

template <int kCode>
cudaError_t Launch(const B200SD_KvCacheAppend& a, const AppendArgs& args, dim3 grid, dim3 block, cudaStream_t stream) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;     // see griddep_wait() in the kernel
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, a.new_dtype == kBF16 ? kv_append_kernel<kCode, __nv_bfloat16> : kv_append_kernel<kCode, __half>, args);
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
                  0xffffffffu / static_cast<uint32_t>(a.head_dim / 8) + 1, a.num_pages, a.table_width, StatusWordPtr()};
  // n tokens in a row reach at most (n - 1 + page - 1) / page + 1 pages; a block takes several where they are small and many.
  const int64_t reach = (a.new_tokens + a.page_tokens - 2) / a.page_tokens + 1, page_warps = a.page_tokens / 16;
  const int64_t together = std::min<int64_t>(kMostWarps / page_warps, reach);
  const dim3 grid(static_cast<unsigned>((reach + together - 1) / together), static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(2 * a.batch));
  const dim3 block(static_cast<unsigned>(32 * page_warps * together));
  const cudaError_t e = a.cache_dtype == kF8E4M3FN ? Launch<kF8E4M3FN>(a, args, grid, block, stream)
                        : a.cache_dtype == kF8E5M2 ? Launch<kF8E5M2>(a, args, grid, block, stream)
                                                   : Launch<kS8>(a, args, grid, block, stream);
  if (e != cudaSuccess) return Status::Error(kInternal, std::string("kv_append_kernel launch: ") + cudaGetErrorString(e));
  stats->launches = 1;
  return Status::Ok();
}

}  // namespace b200sd
