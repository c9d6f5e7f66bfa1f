// Attention of each sequence's last tokens over the paged 8-bit cache.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv_cache.cuh"

namespace b200sd {
namespace {

struct AttentionArgs {
  const void* q;
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const float* k_scale;
  const float* v_scale;
  const int32_t* page_table;
  const int32_t* seq_lens;
  const int32_t* new_lens;
  void* out;
  float* lse;
  int32_t batch, new_tokens, heads, kv_heads, head_dim, page_tokens;
  int64_t num_pages, table_width, window;
  float softmax_scale;
  int32_t is_bf16, cache_dtype;
  uint32_t* status;
};

__device__ __forceinline__ float Decode(uint8_t code, int32_t type) {
  if (type == kS8) return static_cast<float>(static_cast<int8_t>(code));
  uint32_t h;
  const uint16_t c = code;
  if (type == kF8E4M3FN) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  else asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(c));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
}

// One warp per row: running maximum, sum and weighted values, token by token.
__global__ void __launch_bounds__(32) kv_attention_kernel(const AttentionArgs a) {
  const int lane = threadIdx.x, h = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
  const int64_t row = (static_cast<int64_t>(b) * a.new_tokens + i) * a.heads + h;
  const int64_t len = a.seq_lens[b];
  const int64_t count = a.new_lens != nullptr ? min(max(a.new_lens[b], 0), a.new_tokens) : a.new_tokens;
  int64_t end = i < count ? len - count + i + 1 : 0;             // one behind the last position that the row sees
  const int64_t first = a.window > 0 && end > a.window ? end - a.window : 0;
  const int64_t capacity = a.table_width * a.page_tokens;
  if (end > capacity) {
    if (lane == 0) atomicOr(a.status, kStatusBadPage);
    end = capacity;
  }
  float q[8], o[8] = {};
  for (int j = 0; j < 8; ++j) {
    const int d = j * 32 + lane;
    q[j] = d >= a.head_dim ? 0.0f
           : a.is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[row * a.head_dim + d])
                       : __half2float(static_cast<const __half*>(a.q)[row * a.head_dim + d]);
  }
  float top = -INFINITY, sum = 0.0f;
  const int kv = h / (a.heads / a.kv_heads);
  for (int64_t t = first; t < end; ++t) {
    const int64_t page = a.page_table[b * a.table_width + t / a.page_tokens];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) atomicOr(a.status, kStatusBadPage);
      continue;
    }
    const int64_t at = ((page * a.kv_heads + kv) * a.page_tokens + t % a.page_tokens) * a.head_dim;
    float s = 0.0f;
    for (int j = 0; j < 8; ++j)
      if (j * 32 + lane < a.head_dim) s += q[j] * Decode(a.k_pages[at + j * 32 + lane], a.cache_dtype);
    for (int w = 16; w > 0; w /= 2) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= a.softmax_scale * a.k_scale[page * a.kv_heads + kv];
    if (s == -INFINITY) continue;
    const float next = fmaxf(top, s), fade = expf(top - next), p = expf(s - next), vs = a.v_scale[page * a.kv_heads + kv];
    sum = sum * fade + p;
    for (int j = 0; j < 8; ++j)
      if (j * 32 + lane < a.head_dim) o[j] = o[j] * fade + p * (vs * Decode(a.v_pages[at + j * 32 + lane], a.cache_dtype));
    top = next;
  }
  for (int j = 0; j < 8; ++j) {
    const int d = j * 32 + lane;
    if (d >= a.head_dim) continue;
    const float y = sum == 0.0f ? 0.0f : o[j] / sum;
    if (a.is_bf16) static_cast<__nv_bfloat16*>(a.out)[row * a.head_dim + d] = __float2bfloat16_rn(y);
    else static_cast<__half*>(a.out)[row * a.head_dim + d] = __float2half_rn(y);
  }
  if (a.lse != nullptr && lane == 0) a.lse[row] = top + logf(sum);
}

}  // namespace

Status ValidatePagedAttention(const B200SD_PagedAttention& a, bool check_pointers) {
  auto bad = [](const std::string& m) { return Status::Error(kInvalidArgument, m); };
  if (a.struct_size < sizeof(a)) return bad("B200SD_PagedAttention.struct_size is smaller than this library's struct");
  Status st = ValidateCache(a, a.q_dtype, check_pointers);
  if (!st.ok()) return st;
  if (a.heads < 1 || a.heads > 4096 || a.heads % a.kv_heads) return bad("heads must be a multiple of kv_heads, at most 4096");
  if (a.new_tokens > 64) return Status::Error(kUnimplemented, "more than 64 new tokens for a sequence");
  if (a.window < 0) return bad("window must not be negative");
  if (!(a.softmax_scale - a.softmax_scale == 0.0f)) return bad("softmax_scale must be finite");
  if (!check_pointers || a.batch == 0 || a.new_tokens == 0) return Status::Ok();
  if (a.q == nullptr || a.out == nullptr) return bad("q and out must not be null");
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) % 16) return bad("q and out must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(a.lse) % 4) return bad("lse must be 4-byte aligned");
  const size_t need = PagedAttentionWorkspaceBytes(a.batch, a.new_tokens, a.heads, a.kv_heads, a.head_dim);
  if (a.workspace_bytes < need || (need > 0 && a.workspace == nullptr)) return bad("the call needs a workspace of " + std::to_string(need) + " bytes");
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16) return bad("the workspace must be 16-byte aligned");
  return Status::Ok();
}

size_t PagedAttentionWorkspaceBytes(int64_t batch, int64_t new_tokens, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  if (batch < 1 || new_tokens < 1 || kv_heads < 1 || heads < kv_heads || head_dim < 16) return 0;
  return 16;
}

Status LaunchPagedAttention(const B200SD_PagedAttention& a, cudaStream_t stream, LaunchStats* stats) {
  if (a.batch == 0 || a.new_tokens == 0) return Status::Ok();
  const AttentionArgs args{a.q, static_cast<const uint8_t*>(a.k_pages), static_cast<const uint8_t*>(a.v_pages), a.k_scale, a.v_scale,
                           a.page_table, a.seq_lens, a.new_lens, a.out, a.lse,
                           static_cast<int32_t>(a.batch), static_cast<int32_t>(a.new_tokens), static_cast<int32_t>(a.heads), static_cast<int32_t>(a.kv_heads),
                           static_cast<int32_t>(a.head_dim), static_cast<int32_t>(a.page_tokens),
                           a.num_pages, a.table_width, a.window, a.softmax_scale, a.q_dtype == kBF16, a.cache_dtype, StatusWordPtr()};
  kv_attention_kernel<<<dim3(static_cast<unsigned>(a.heads), static_cast<unsigned>(a.new_tokens), static_cast<unsigned>(a.batch)), 32, 0, stream>>>(args);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return Status::Error(kInternal, std::string("kv_attention_kernel launch: ") + cudaGetErrorString(e));
  stats->launches = 1;
  return Status::Ok();
}

}  // namespace b200sd
