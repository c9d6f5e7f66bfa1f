// What the append and the attention share: the addressing of the paged 8-bit cache and its checks.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "kernels.h"
#include "ptx.cuh"

namespace b200sd {

// The largest magnitude of a cache type as fraction * 2^exponent, the fraction in [0.5, 1).
template <int kCode> struct CodeTraits;
template <> struct CodeTraits<kF8E4M3FN> { static constexpr float kMax = 448.0f, kFraction = 0.875f; static constexpr int kExponent = 9; };
template <> struct CodeTraits<kF8E5M2> { static constexpr float kMax = 57344.0f, kFraction = 0.875f; static constexpr int kExponent = 16; };
template <> struct CodeTraits<kS8> { static constexpr float kMax = 127.0f, kFraction = 0.9921875f; static constexpr int kExponent = 7; };

// The checks that both calls make of the cache and of the tensors that index it.
template <typename Args>
Status ValidateCache(const Args& a, int32_t value_dtype, bool check_pointers) {
  auto bad = [](const std::string& m) { return Status::Error(kInvalidArgument, m); };
  if (!(a.cache_dtype == kF8E4M3FN || a.cache_dtype == kF8E5M2 || a.cache_dtype == kS8)) return bad("the cache must be F8E4M3FN, F8E5M2 or S8");
  if (!(value_dtype == kBF16 || value_dtype == kF16)) return bad("queries, keys and values must be BF16 or F16");
  if (a.batch < 0 || a.new_tokens < 0 || a.num_pages < 0 || a.table_width < 0) return bad("dimensions must not be negative");
  if (a.kv_heads < 1 || a.kv_heads > 1024) return bad("kv_heads must be between 1 and 1024");
  if (a.head_dim < 16 || a.head_dim > 256 || a.head_dim % 16) return bad("head_dim must be a multiple of 16 between 16 and 256");
  if (!(a.page_tokens == 16 || a.page_tokens == 32 || a.page_tokens == 64 || a.page_tokens == 128)) return bad("a page must hold 16, 32, 64 or 128 tokens");
  if (a.batch > 4096) return Status::Error(kUnimplemented, "more than 4096 sequences");
  if (a.num_pages > INT32_MAX / a.kv_heads) return bad("too many pages for 32-bit numbers of (page, head)");
  if (a.table_width > (int64_t{1} << 30) / a.page_tokens) return bad("page_table is too wide: a sequence has at most 2^30 tokens");
  if (!check_pointers || a.batch == 0 || a.new_tokens == 0) return Status::Ok();
  if (a.seq_lens == nullptr) return bad("seq_lens must not be null");
  if (a.num_pages > 0 && a.table_width > 0 &&
      (a.k_pages == nullptr || a.v_pages == nullptr || a.k_scale == nullptr || a.v_scale == nullptr || a.page_table == nullptr))
    return bad("the cache, its scales and its page table must not be null");
  if ((reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages)) % 16) return bad("k_pages and v_pages must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(a.k_scale) | reinterpret_cast<uintptr_t>(a.v_scale) | reinterpret_cast<uintptr_t>(a.page_table) |
       reinterpret_cast<uintptr_t>(a.seq_lens) | reinterpret_cast<uintptr_t>(a.new_lens)) % 4)
    return bad("scales, page table and lengths must be 4-byte aligned");
  return Status::Ok();
}

}  // namespace b200sd
