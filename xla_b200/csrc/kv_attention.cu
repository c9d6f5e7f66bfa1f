// Attention of each sequence's last tokens over the paged 8-bit cache.
//
// For one key head the queries of a sequence -- the heads that share the key head, times the new tokens -- are the rows of
// one product, so the cache is read once for all of them: 8 or 16 rows per pass.  A step is bound by reading the codes:
// one byte of keys or values is used for 2 * rows operations.
//
// Work.  An item is (sequence, key head, block of rows); its units are one for every 128 tokens (64 of wide heads) behind a
// few that stand for what an item costs besides its tokens.  The units of all items, in one line, are dealt out to the CTAs
// in equal consecutive shares, whatever the lengths are; an item that a share's end cuts leaves its pieces (maximum, sum,
// weighted values) in the workspace, and a second kernel joins them in order, so that the result does not depend on timing.
//
// A CTA is four warps, and each warp works on its own tokens, two tiles of 16 of every 128: they come through a ring in
// shared memory that only this warp fills (TMA, one box per tile of keys or values) and reads, so no barrier stands
// between loading and computing until an item ends.  TMA's swizzle puts the 16-byte pieces of a row at piece ^ (row & 7),
// which leaves both kinds of reads below without bank conflicts.
//
// Arithmetic, on mma.m16n8k16 with f16 operands and f32 sums; codes of all three cache types are f16 numbers, exactly.
// Queries are f16 too: bf16 rows are multiplied by a power of two that brings their largest value to 2^13, so nothing is
// rounded but what lies 2^27 below it.
//   scores^T [16 tokens, 8 rows] = keys [16, d] queries^T [d, 8]: the order of the products along d is free, so a
//     lane takes 16 consecutive bytes of a key and feeds them to four products.
//   values^T [d, 16 tokens] weights^T [16, 8]: a lane takes 16 bytes at the same place of four tokens, pairs the bytes of
//     two tokens with prmt and decodes the pairs; the weights turn from score layout to operand layout with movmatrix.
// Token m of the 16 is row m ^ ((m & 1) << 2) of the tile in both products.
//
// Measured with cold caches: two sequences of 100003 to 131072 tokens, 8 key heads of 128, 86 us (5.5 TB/s of codes); 32 of 0
// to 4096 tokens 35 us (3.9 TB/s: 9 us pass before the tiles flow and 3 to 4 in joining the pieces); 16 of 5 to 8191 with 5
// new tokens, 40 rows for each of 4 key heads, 59 us (bound by issue: the codes are decoded for each 16 rows); one of 37
// tokens 7.8 us, the host's part of the call.
//
// Softmax.  A page has one scale for its values, so the weight of a token that enters the product is
// exp2(score + log2(value scale) - M) with one running M per row: the largest weight stays the same even if the scales of
// pages lie far apart, and the 11 bits of f16 (chosen over bf16's 8, at the same speed) are relative to what matters.  That is
// enough for results in bf16, which are rounded to 8 bits afterwards.  For results in f16 a weight is two f16 numbers, 22
// bits, both multiplied with the decoded values: 33.6 us instead of 32.6 for the batch above, 63 instead of 58 for the new tokens.
// M lies 9 below the largest score when it is set, so that weights keep all their bits down to 2^-23 of the largest.  The
// sum takes the weight times the inverse scale, in f32.  M moves only when a new score passes the one that set it by
// more than 6, so most tiles rescale nothing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>
#include <mutex>

#include "kv_cache.cuh"

namespace b200sd {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 16;                       // tokens of a warp's step
constexpr int kMaxCtas = 148 * 5;               // of one launch; bounds the workspace
constexpr int64_t kMostItems = 1 << 26;         // of a launch: an item is at least one unit and less than 17
constexpr float kLift = 9.0f;                   // binary digits that a row's largest weight is lifted by ...
constexpr float kSlack = 6.0f;                  // ... and that a later one may pass it by: together below f16's 2^15.99

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
  float* work;                                  // the pieces of cut items, two places for each CTA ...
  int4* cut;                                    // ... and for each CTA the item that the end of its share cuts first: b, item, pieces (0: none), new tokens
  int32_t batch, new_tokens, heads, kv_heads, head_dim, page_shift;
  int32_t rows, blocks;                         // rows of a (sequence, key head), and blocks of them
  int32_t num_pages, table_width, window;       // window: 0 none
  int32_t unit_shift, extra;                    // log2 of the tokens of a unit, a multiple of the CTA's step; units without tokens in front of an item
  int32_t min_units;                            // a CTA's share is not smaller
  float scale;                                  // softmax_scale * log2(e)
  int32_t is_bf16;
  int32_t lose;                                 // LoseCopy()
  uint32_t* status;
};

// The positions of one sequence that some row sees, from a multiple of kTile on.
struct Span {
  int32_t base;                                 // position of the first new token
  int32_t count;                                // new tokens
  int32_t lo, hi;                               // hi is at most 2^30
  int32_t units;
};

__device__ __forceinline__ Span SpanOf(const AttentionArgs& a, int b) {
  Span s;
  const int32_t len = a.seq_lens[b];
  s.count = a.new_lens != nullptr ? min(max(a.new_lens[b], 0), a.new_tokens) : a.new_tokens;
  s.base = max(len, 0) - s.count;               // below 0 for a length that does not hold the new tokens
  const int32_t capacity = a.table_width << a.page_shift;
  s.hi = s.count > 0 ? min(max(len, 0), capacity) : 0;
  // The window of a length far outside of the table begins behind it; positions a CTA's step beyond `lo` stay 32-bit numbers.
  s.lo = a.window > 0 ? min(max(0, s.base + 1 - a.window) & ~(kTile - 1), s.hi) : 0;
  s.units = max(1, a.extra + (s.hi > s.lo ? ((s.hi - s.lo - 1) >> a.unit_shift) + 1 : 0));      // an item without tokens still has rows to write
  return s;
}

// The share of one CTA: `left` units from `begin` on, and where a unit lies: unit `offset` of item `item` of sequence `b`.
struct Share {
  int32_t b, item, offset;
  int32_t left, begin;
};

// The line of `total` units, dealt out to `ctas`: `per` to each, and one more to the first `more` of them.
struct Deal {
  int32_t total, ctas, per, more;
  __device__ int32_t Begin(int32_t cta) const { return cta * per + min(cta, more); }
  __device__ int32_t CtaOf(int32_t u) const {
    const int32_t large = more * (per + 1);
    return u < large ? u / (per + 1) : more + (u - large) / per;
  }
};

// The share of CTA `cta`, with b, item and offset of its first unit.  Every warp finds out for itself, its
// lanes taking consecutive sequences.  The launch chooses units large enough that the line has less than 2^31.
__device__ Share Locate(const AttentionArgs& a, int cta, Deal* deal) {
  const int lane = threadIdx.x % 32;
  const int each = (a.batch + 31) / 32, first = min(lane * each, a.batch), end = min(first + each, a.batch);
  const int32_t items = a.kv_heads * a.blocks;
  int32_t mine = 0, most = 1;
#pragma unroll 1
  for (int b = first; b < end; ++b) {
    const int32_t units = SpanOf(a, b).units;
    mine += units * items;
    most = max(most, units);
  }
  int32_t before = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int32_t v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  const int32_t total = __shfl_sync(0xffffffffu, before, 31);
  before -= mine;
  deal->total = total;
  // The second kernel walks through an item's pieces, so shares are large enough that the largest item has about 128, and no
  // item more than 162.  (One sequence of 131072 tokens beside 15 idle ones, one key head: 28.2 us, and 42.8 without this.)
  const int32_t least = max(a.min_units, (__reduce_max_sync(0xffffffffu, most) + 64) / 128);
  deal->ctas = max(1, min(static_cast<int32_t>(gridDim.x), total / least));
  deal->per = total / deal->ctas;
  deal->more = total - deal->per * deal->ctas;
  if (cta >= deal->ctas) return {0, 0, 0, 0, 0};
  auto place = [&](int32_t u) -> Share {
    const bool here = u >= before && u < before + mine;
    int32_t b = first, at = u - before, units = 1;
    if (here) {
      units = SpanOf(a, b).units;
      while (at >= units * items) {
        at -= units * items;
        units = SpanOf(a, ++b).units;
      }
    }
    const int32_t item = at / units, from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    return {__shfl_sync(0xffffffffu, b, from), __shfl_sync(0xffffffffu, item, from), __shfl_sync(0xffffffffu, at - item * units, from), 0, u};
  };
  // A share does not end with units without tokens; the next one takes them.
  int32_t u0 = deal->Begin(cta), u1 = deal->Begin(cta + 1);
  Share at_begin = place(u0);
  if (at_begin.offset <= a.extra) u0 -= at_begin.offset, at_begin.offset = 0;
  if (u1 < total) {
    const int32_t into = place(u1).offset;
    if (into <= a.extra) u1 -= into;
  }
  if (u0 >= u1) return {0, 0, 0, 0, 0};
  at_begin.begin = u0;
  at_begin.left = u1 - u0;
  return at_begin;
}

// Steps through the pieces of items that make up a share.
struct Walk {
  int32_t b, item, offset, left;
  Span span;

  __device__ Walk(const AttentionArgs& a, const Share& s) : b(s.b), item(s.item), offset(s.offset), left(s.left) {
    if (left > 0) span = SpanOf(a, b);
  }
  __device__ int32_t Units() const { return min(left, span.units - offset); }
  __device__ int32_t Begin(const AttentionArgs& a) const { return span.lo + (max(0, offset - a.extra) << a.unit_shift); }
  __device__ int32_t End(const AttentionArgs& a) const {
    return static_cast<int32_t>(min(static_cast<int64_t>(span.hi), span.lo + (static_cast<int64_t>(max(0, offset + Units() - a.extra)) << a.unit_shift)));
  }
  __device__ void Next(const AttentionArgs& a) {
    const int32_t n = Units();
    left -= n;
    offset += n;
    if (offset == span.units) {
      offset = 0;
      if (++item == a.kv_heads * a.blocks) {
        item = 0;
        ++b;
        if (left > 0) span = SpanOf(a, b);
      }
    }
  }
};

// Four codes, two by two, to f16 pairs.
template <int kCode>
__device__ __forceinline__ void Decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kCode == kF8E4M3FN) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else if constexpr (kCode == kF8E5M2) {      // the upper half of an f16
    lo = __byte_perm(w, 0, 0x1404);
    hi = __byte_perm(w, 0, 0x3424);
  } else {                                      // 1024 + (code + 128) has the code's bits, offset, in its low byte
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
    uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 lv = __hsub2(*reinterpret_cast<__half2*>(&l), bias), hv = __hsub2(*reinterpret_cast<__half2*>(&h), bias);
    lo = *reinterpret_cast<const uint32_t*>(&lv);
    hi = *reinterpret_cast<const uint32_t*>(&hv);
  }
}
template <int kCode>
__device__ __forceinline__ float Decode1(uint32_t code) {
  uint32_t lo, hi;
  Decode4<kCode>(code & 255u, lo, hi);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(lo)));
}
// Whether one of four codes is NaN or infinite.
template <int kCode>
__device__ __forceinline__ bool NotFinite4(uint32_t w) {
  if constexpr (kCode == kS8) return false;
  const uint32_t bits = kCode == kF8E4M3FN ? 0x7f7f7f7fu : 0x7c7c7c7cu;
  const uint32_t left = (w & bits) ^ bits;                                  // a zero byte is such a code
  return ((left - 0x01010101u) & ~left & 0x80808080u) != 0;
}

__device__ __forceinline__ void Mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t Transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Rings, exchange buffers and per-tile numbers of one instantiation.
template <int kDim, int kRowTiles>
struct Layout {
  static constexpr int kPair = kDim == 256 ? 1 : 2;                         // tiles of a stage
  static constexpr int kStages = kDim == 64 ? 3 : 2;
  static constexpr int kStep = kTile * kPair * kWarps;                      // tokens of a CTA's step
  static constexpr int kTileBytes = kTile * kDim;                           // of keys, and again of values
  static constexpr int kRows = 8 * kRowTiles;
  static constexpr int kRing = kWarps * kStages * kPair * 2 * kTileBytes;
  static constexpr int kPart = 32 * kRowTiles * (kDim / 16 + 1);            // float4s of a warp's part of an item: values, then maxima and sums
  static constexpr int kNumbers = kWarps * kStages * kPair;                 // float4s
  static constexpr int kBytes = 1024 + kRing + 2 * kPart * 16 + kNumbers * 16 + kWarps * kStages * 8 + 16;
  static constexpr int kSlot = kRows * (kDim + 2);                          // floats of a piece in the workspace
};

// Byte of 16-byte piece `c` of row `r` in a tile: TMA's swizzles by 64 and by 128 bytes; 256 columns are two boxes.
template <int kDim>
__device__ __forceinline__ int PieceAt(int r, int c) {
  if constexpr (kDim == 64) return r * 64 + (c ^ ((r >> 1) & 3)) * 16;
  return (c >> 3) * (kTile * 128) + r * 128 + ((c & 7) ^ (r & 7)) * 16;
}
// Column of the values' product that m-tile `mt` of lane group `g` holds (its row g; row g + 8 is the next column).
template <int kDim>
__device__ __forceinline__ int Column(int g, int mt) {
  if constexpr (kDim == 64) return 8 * g + 2 * mt;
  return (mt / 8) * 128 + 16 * g + 2 * (mt % 8);
}

// Part of a row of the result from its weighted values `o` (kCount columns at `d`), its sum and its running maximum.
template <int kCount>
__device__ __forceinline__ void StoreRow(const AttentionArgs& a, int b, int head, int row, int count, int d, const float (&o)[kCount], float m, float sum) {
  const int share = a.heads / a.kv_heads, i = row / share;
  const int64_t at = (static_cast<int64_t>(b) * a.new_tokens + i) * a.heads + head * share + row % share;
  const bool empty = i >= count || (m == -INFINITY && sum == 0.0f);
  if (a.lse != nullptr && d == 0) a.lse[at] = empty ? -INFINITY : 0.69314718055994531f * (m + log2f(sum));
  if (d >= a.head_dim) return;
  const float inv = empty ? 0.0f : 1.0f / sum;
  uint32_t packed[kCount / 2];
#pragma unroll
  for (int j = 0; j < kCount / 2; ++j) {
    const float x = empty ? 0.0f : o[2 * j] * inv, y = empty ? 0.0f : o[2 * j + 1] * inv;
    if (a.is_bf16) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
      packed[j] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __half2 v = __floats2half2_rn(x, y);
      packed[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  uint16_t* to = static_cast<uint16_t*>(a.out) + at * a.head_dim + d;
  if constexpr (kCount == 4) {
    *reinterpret_cast<uint2*>(to) = make_uint2(packed[0], packed[1]);
  } else {
#pragma unroll
    for (int j = 0; j < kCount / 8; ++j) *reinterpret_cast<uint4*>(to + 8 * j) = make_uint4(packed[4 * j], packed[4 * j + 1], packed[4 * j + 2], packed[4 * j + 3]);
  }
}

// kF16: queries and results are f16, not bf16.
template <int kCode, int kDim, int kRowTiles, bool kF16>
__global__ void __launch_bounds__(kThreads) kv_attention_kernel(const __grid_constant__ AttentionArgs a, const __grid_constant__ CUtensorMap key_map,
                                                                const __grid_constant__ CUtensorMap value_map) {
  using L = Layout<kDim, kRowTiles>;
  constexpr int kPair = L::kPair, kStages = L::kStages, kStep = L::kStep, kStageBytes = kPair * 2 * L::kTileBytes;
  constexpr int kBoxes = kDim == 256 ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (1024 - (smem_u32(smem_raw) & 1023)) % 1024;       // the swizzle goes by the address
  __shared__ int abort_flag;
  __shared__ Deal shared_deal;                             // for the end of the share
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  uint8_t* ring = smem + warp * kStages * kStageBytes;
  float4* exchange = reinterpret_cast<float4*>(smem + L::kRing);
  float4* numbers = exchange + 2 * L::kPart + warp * kStages * kPair;
  uint64_t* full = reinterpret_cast<uint64_t*>(exchange + 2 * L::kPart + L::kNumbers) + warp * kStages;
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  __syncthreads();
  griddep_wait();
  if (threadIdx.x == 0) griddep_launch_dependents();
  Deal deal;
  const Share share = Locate(a, blockIdx.x, &deal);
  if (threadIdx.x == 0) {
    shared_deal = deal;
    a.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  if (share.left == 0) return;

  // This lane's part of an item's queries, as they are.  The first item's are sent for before the tiles, which they would
  // otherwise queue behind.
  const int group = a.heads / a.kv_heads;
  uint32_t q[kRowTiles][kDim / 64][4][2];
  auto load_queries = [&](int b, int item) {
    const int head = item / a.blocks, row0 = (item - head * a.blocks) * L::kRows;
#pragma unroll
    for (int n = 0; n < kRowTiles; ++n) {
      const int row = row0 + n * 8 + g;
      const uint16_t* from = static_cast<const uint16_t*>(a.q) +
          ((static_cast<int64_t>(b) * a.new_tokens + row / group) * a.heads + head * group + row % group) * a.head_dim;
#pragma unroll
      for (int hf = 0; hf < kDim / 64; ++hf) {
        uint4 v[2] = {};
        if (row < a.rows && 64 * hf + 16 * t < a.head_dim) {
          v[0] = *reinterpret_cast<const uint4*>(from + 64 * hf + 16 * t);
          v[1] = *reinterpret_cast<const uint4*>(from + 64 * hf + 16 * t + 8);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q[n][hf][j][0] = j < 2 ? (j == 0 ? v[0].x : v[0].z) : (j == 2 ? v[1].x : v[1].z);
          q[n][hf][j][1] = j < 2 ? (j == 0 ? v[0].y : v[0].w) : (j == 2 ? v[1].y : v[1].w);
        }
      }
    }
  };
  load_queries(share.b, share.item);

  // ---- loading: this warp's tiles of the whole share, one after the other -----------------------
  // Pages and scales come for 32 tiles at a time, one per lane.  A tile is sent for as soon as its page is known; what the
  // scales become is written beside the stage (`flush`) when it is about to be used.
  Walk ahead(a, share);
  int32_t load_pos = ahead.Begin(a) + warp * (kTile * kPair), load_end = ahead.End(a), batch_at = 32;      // batch_at: tile of the batch that comes next
  int32_t page_of = -1, load_stage = 0, pending = 0;       // lane j: page of tile j of the batch; stages whose numbers are not written
  bool raw = false;
  float4 of_tile = {};                                     // key scale, log2 of the value scale, its inverse, its sign; -infinity marks a tile that is not there
  auto flush = [&] {
    if (pending == 0) return;
    if (raw) {
      const float size = fminf(fmaxf(fabsf(of_tile.w), 0x1p-100f), 0x1p100f);
      // x + (x - x): an infinite scale makes infinities of both signs of a key, whose product is no number.
      of_tile = page_of >= 0 ? make_float4(of_tile.x + (of_tile.x - of_tile.x), log2f(size), 1.0f / size, of_tile.w / size) : make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
      raw = false;
    }
    const int at = lane - (batch_at - pending * kPair);    // this lane's tile among the pending ones
    if (at >= 0 && at < pending * kPair) {
      int stage = load_stage - pending + at / kPair;
      if (stage < 0) stage += kStages;
      numbers[stage * kPair + at % kPair] = of_tile;
    }
    pending = 0;
  };
  auto issue = [&] {
    while (ahead.left > 0 && load_pos >= load_end) {
      ahead.Next(a);
      flush();
      batch_at = 32;
      if (ahead.left == 0) break;
      load_pos = ahead.Begin(a) + warp * (kTile * kPair);
      load_end = ahead.End(a);
    }
    if (ahead.left == 0) return;
    const int head = ahead.item / a.blocks;
    if (batch_at == 32) {
      flush();
      const int64_t pos = static_cast<int64_t>(load_pos) + lane / kPair * kStep + lane % kPair * kTile;
      page_of = -1;
      if (pos < load_end) {
        page_of = a.page_table[static_cast<int64_t>(ahead.b) * a.table_width + (pos >> a.page_shift)];
        if (page_of < 0 || page_of >= a.num_pages) {
          page_of = -1;
          atomicOr(a.status, kStatusBadPage);              // its tokens count as not seen
        }
      }
      const int64_t at = static_cast<int64_t>(max(page_of, 0)) * a.kv_heads + head;
      if (page_of >= 0) of_tile.x = a.k_scale[at], of_tile.w = a.v_scale[at];
      raw = true;
      batch_at = 0;
    }
    int32_t pages[kPair];
#pragma unroll
    for (int i = 0; i < kPair; ++i) pages[i] = __shfl_sync(0xffffffffu, page_of, batch_at + i);
    const bool lost = kTiming && a.lose && share.begin == 0 && warp == 0 && load_pos == ahead.Begin(a) && ahead.left == share.left;
    if (lane == 0 && !lost) {
      int tiles = 0;
#pragma unroll
      for (int i = 0; i < kPair; ++i) tiles += pages[i] >= 0 ? 1 : 0;
      mbar_arrive_expect_tx(&full[load_stage], tiles * 2 * L::kTileBytes);
#pragma unroll
      for (int i = 0; i < kPair; ++i) {
        if (pages[i] < 0) continue;
        const int slot = (load_pos + i * kTile) & ((1 << a.page_shift) - 1), matrix = pages[i] * a.kv_heads + head;
        uint8_t* dst = ring + load_stage * kStageBytes + i * 2 * L::kTileBytes;
#pragma unroll
        for (int box = 0; box < kBoxes; ++box) {
          tma_load_3d(dst + box * (kTile * 128), &key_map, &full[load_stage], box * 128, slot, matrix);
          tma_load_3d(dst + L::kTileBytes + box * (kTile * 128), &value_map, &full[load_stage], box * 128, slot, matrix);
        }
      }
    }
    batch_at += kPair;
    load_pos += kStep;
    ++pending;
    if (++load_stage == kStages) load_stage = 0;
  };
#pragma unroll 1
  for (int s = 0; s < kStages; ++s) issue();

  // ---- computing, piece by piece ---------------------------------------------------------------
  int stage = 0;
  uint32_t parity = 0;
  for (Walk walk(a, share); walk.left > 0; walk.Next(a)) {
    const int head = walk.item / a.blocks, row0 = (walk.item % a.blocks) * L::kRows;
    const Span& span = walk.span;
    const int32_t begin = walk.Begin(a), end = walk.End(a);
    if (threadIdx.x == 0 && span.count > 0) {
      const int32_t len = a.seq_lens[walk.b];
      if (len < 0 || len > static_cast<int64_t>(a.table_width) << a.page_shift) atomicOr(a.status, kStatusBadPage);
    }

    // Queries as the products want them, and what turns a product into a score, for the rows 2t and 2t + 1 of each 8.
    float factor[kRowTiles][2];
    int32_t row_end[kRowTiles][2], row_begin[kRowTiles][2];
#pragma unroll
    for (int n = 0; n < kRowTiles; ++n) {
      float mine = 1.0f;
      if constexpr (!kF16) {
        uint32_t top = 0;                                  // exponent of the row's largest value
#pragma unroll
        for (int hf = 0; hf < kDim / 64; ++hf)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t w = q[n][hf][j / 2][j % 2];
            top = max(top, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
          }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int power = top >= 0x7f80u || top == 0 ? 0 : min(126, 13 - (static_cast<int>(top >> 7) - 127));
        const float up = __uint_as_float(static_cast<uint32_t>(127 + power) << 23);
        mine = 1.0f / up;
#pragma unroll
        for (int hf = 0; hf < kDim / 64; ++hf)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t& w = q[n][hf][j / 2][j % 2];
            const __half2 h = __floats2half2_rn(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
            w = *reinterpret_cast<const uint32_t*>(&h);
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        factor[n][e] = a.scale * __shfl_sync(0xffffffffu, mine, (2 * t + e) * 4);
        const int r = row0 + n * 8 + 2 * t + e, i = r / group;
        row_end[n][e] = r < a.rows && i < span.count ? span.base + i + 1 : INT32_MIN;
        row_begin[n][e] = a.window > 0 ? row_end[n][e] - (row_end[n][e] == INT32_MIN ? 0 : a.window) : 0;
      }
    }
    // Tiles inside [all_begin, all_end) are seen by every row of the block that sees anything, tiles outside of
    // [any_begin, any_end) by none.
    const int first_i = min(row0 / group, span.count - 1), last_i = min((min(row0 + L::kRows, a.rows) - 1) / group, span.count - 1);
    const int32_t all_end = span.base + first_i + 1, any_end = span.base + last_i + 1;
    const int32_t all_begin = a.window > 0 ? any_end - a.window : 0, any_begin = a.window > 0 ? all_end - a.window : 0;

    float o[kRowTiles][kDim / 16][4] = {};
    float top[kRowTiles][2], sum[kRowTiles][2];
#pragma unroll
    for (int n = 0; n < kRowTiles; ++n) top[n][0] = top[n][1] = -INFINITY, sum[n][0] = sum[n][1] = 0.0f;

    const int kr = g ^ ((g & 1) << 2);
#pragma unroll 1
    for (int32_t pos = begin + warp * (kTile * kPair); pos < end; pos += kStep) {
      flush();
      const uint8_t* tiles = ring + stage * kStageBytes;
      const uint64_t limit = kTiming && a.lose ? kLostCopyNs : kWaitLimitNs;
      if (!mbar_wait_warp(&full[stage], parity, &abort_flag, a.status, kStatusTileTimeout, limit)) {      // this warp leaves, and what the CTA writes is not the result
        const int ahead_by = load_stage - stage;
        await_copies(full, kStages, stage, parity, ahead_by > 0 ? ahead_by : ahead_by + kStages, a.status, kStatusTileTimeout, limit);
        return;
      }
      __syncwarp();
      float4 num[kPair];
#pragma unroll
      for (int i = 0; i < kPair; ++i) num[i] = numbers[stage * kPair + i];
      if (++stage == kStages) stage = 0, parity ^= 1;

      float s[kPair][kRowTiles][4] = {};
#pragma unroll
      for (int hf = 0; hf < kDim / 64; ++hf)
#pragma unroll
        for (int i = 0; i < kPair; ++i) {
          const uint8_t* keys = tiles + i * 2 * L::kTileBytes;
          const uint4 ka = *reinterpret_cast<const uint4*>(keys + PieceAt<kDim>(kr, 4 * hf + t));
          const uint4 kb = *reinterpret_cast<const uint4*>(keys + PieceAt<kDim>(kr + 8, 4 * hf + t));
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a0, a1, a2, a3;
            Decode4<kCode>(wa[j], a0, a2);
            Decode4<kCode>(wb[j], a1, a3);
#pragma unroll
            for (int n = 0; n < kRowTiles; ++n) Mma(s[i][n], a0, a1, a2, a3, q[n][hf][j][0], q[n][hf][j][1]);
          }
        }
      bool whole = pos >= all_begin && pos + kTile * kPair <= all_end;
#pragma unroll
      for (int i = 0; i < kPair; ++i) whole = whole && num[i].y != -INFINITY;
      bool move = false;
      float high[kRowTiles][2];
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
        for (int i = 0; i < kPair; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][n][e] = fmaf(s[i][n][e], factor[n][e % 2] * num[i].x, num[i].y);
        if (!whole) {
#pragma unroll
          for (int i = 0; i < kPair; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int32_t at = pos + i * kTile + kr + (e / 2) * 8;
              if (num[i].y == -INFINITY || at >= row_end[n][e % 2] || at < row_begin[n][e % 2]) s[i][n][e] = -INFINITY;
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float h = fmaxf(s[0][n][e], s[0][n][e + 2]);
          if (kPair == 2) h = fmaxf(h, fmaxf(s[kPair - 1][n][e], s[kPair - 1][n][e + 2]));
          h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, 4));
          h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, 8));
          h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, 16));
          high[n][e] = h;
          move |= h > top[n][e] + (kLift + kSlack);
        }
      }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int n = 0; n < kRowTiles; ++n) {
          float fade[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float next = fmaxf(top[n][e], high[n][e] - kLift);
            fade[e] = next == -INFINITY ? 1.0f : Exp2(top[n][e] - next);
            top[n][e] = next;
            sum[n][e] *= fade[e];
          }
#pragma unroll
          for (int mt = 0; mt < kDim / 16; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][mt][e] *= fade[e % 2];
        }
      }
      uint32_t p[kPair][kRowTiles][2];
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
        const float from[2] = {top[n][0] == -INFINITY ? 0.0f : top[n][0], top[n][1] == -INFINITY ? 0.0f : top[n][1]};
#pragma unroll
        for (int i = 0; i < kPair; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[i][n][e] = Exp2(s[i][n][e] - from[e % 2]);
            sum[n][e % 2] = fmaf(s[i][n][e], num[i].z, sum[n][e % 2]);
          }
        }
      }
      bool odd = num[0].w != 1.0f;                         // a negative scale, or one that is no number: not for rows that do not see the token
      if (kPair == 2) odd = odd || num[kPair - 1].w != 1.0f;
      if (odd) {
#pragma unroll
        for (int i = 0; i < kPair; ++i)
#pragma unroll
          for (int n = 0; n < kRowTiles; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int32_t at = pos + i * kTile + kr + (e / 2) * 8;
              s[i][n][e] = at < row_end[n][e % 2] && at >= row_begin[n][e % 2] ? s[i][n][e] * num[i].w : 0.0f;
            }
      }
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
        for (int i = 0; i < kPair; ++i) {
          const __half2 l = __floats2half2_rn(s[i][n][0], s[i][n][1]), h = __floats2half2_rn(s[i][n][2], s[i][n][3]);
          p[i][n][0] = Transpose8x8(*reinterpret_cast<const uint32_t*>(&l));
          p[i][n][1] = Transpose8x8(*reinterpret_cast<const uint32_t*>(&h));
        }
      }
      // Values: the pieces at this lane's columns of tokens 2t, 2t + 1, 2t + 8 and 2t + 9.
      const int r0 = 2 * t, r1 = (2 * t + 1) ^ 4;
#pragma unroll
      for (int i = 0; i < kPair; ++i) {
        if (num[i].y == -INFINITY) continue;               // not loaded
        const uint8_t* values = tiles + i * 2 * L::kTileBytes + L::kTileBytes;
        uint32_t fine[kRowTiles][2];                       // what the f16 weights are short of
        if constexpr (kF16) {
#pragma unroll
          for (int n = 0; n < kRowTiles; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 held = __half22float2(__floats2half2_rn(s[i][n][2 * h], s[i][n][2 * h + 1]));
              const __half2 rest = __floats2half2_rn(s[i][n][2 * h] - held.x, s[i][n][2 * h + 1] - held.y);
              fine[n][h] = Transpose8x8(*reinterpret_cast<const uint32_t*>(&rest));
            }
        }
#pragma unroll
        for (int part = 0; part < (kDim == 256 ? 2 : 1); ++part) {
          constexpr int kWords = kDim == 64 ? 2 : 4;
          uint32_t w[4][kWords];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = (r & 1 ? r1 : r0) + (r & 2 ? 8 : 0);
            if constexpr (kDim == 64) {
              const uint2 v = *reinterpret_cast<const uint2*>(values + PieceAt<kDim>(row, g >> 1) + (g & 1) * 8);
              w[r][0] = v.x, w[r][1] = v.y;
            } else {
              const uint4 v = *reinterpret_cast<const uint4*>(values + PieceAt<kDim>(row, part * 8 + g));
              w[r][0] = v.x, w[r][1] = v.y, w[r][2] = v.z, w[r][3] = v.w;
            }
          }
          if (!whole) {
            // Weight 0 does not silence a NaN: codes that no row sees are taken out, and where some rows see one that
            // is not finite, the products of the tile are formed one by one.
            bool scalar = false;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int32_t at = pos + i * kTile + (r & 1 ? r1 : r0) + (r & 2 ? 8 : 0);
              const bool unseen = at >= any_end || at < any_begin;
#pragma unroll
              for (int j = 0; j < kWords; ++j) {
                if (unseen) w[r][j] = 0;
                scalar |= NotFinite4<kCode>(w[r][j]);
              }
            }
            if (kCode != kS8 && all_end != any_end && __any_sync(0xffffffffu, scalar)) {
#pragma unroll 1
              for (int token = 0; token < kTile; ++token) {
                const int row = token ^ ((token & 1) << 2), at = pos + i * kTile + row;
#pragma unroll
                for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const float low = __shfl_sync(0xffffffffu, s[i][n][e], (token & 7) * 4 + t), upper = __shfl_sync(0xffffffffu, s[i][n][e + 2], (token & 7) * 4 + t);
                    const float weight = token < 8 ? low : upper;
                    if (at < row_end[n][e] && at >= row_begin[n][e]) {
#pragma unroll
                      for (int m = 0; m < 2 * kWords; ++m) {
                        const int column = Column<kDim>(g, part * 8 + m);
                        const uint8_t* codes = values + PieceAt<kDim>(row, column / 16) + column % 16;
                        o[n][part * 8 + m][e] += weight * Decode1<kCode>(codes[0]);
                        o[n][part * 8 + m][e + 2] += weight * Decode1<kCode>(codes[1]);
                      }
                    }
                  }
                }
              }
              continue;
            }
          }
#pragma unroll
          for (int j = 0; j < kWords; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t a0, a1, a2, a3;
              Decode4<kCode>(__byte_perm(w[0][j], w[1][j], h == 0 ? 0x5140 : 0x7362), a0, a1);
              Decode4<kCode>(__byte_perm(w[2][j], w[3][j], h == 0 ? 0x5140 : 0x7362), a2, a3);
#pragma unroll
              for (int n = 0; n < kRowTiles; ++n) {
                Mma(o[n][part * 8 + 2 * j + h], a0, a1, a2, a3, p[i][n][0], p[i][n][1]);
                if constexpr (kF16) Mma(o[n][part * 8 + 2 * j + h], a0, a1, a2, a3, fine[n][0], fine[n][1]);
              }
            }
          }
        }
      }
      __syncwarp();                                        // all lanes have read the stage
      issue();
    }

    if (walk.left > walk.Units()) {                        // the next item's queries, on their way while this one is put together
      const bool same = walk.item + 1 < a.kv_heads * a.blocks;
      load_queries(same ? walk.b : walk.b + 1, same ? walk.item + 1 : 0);
    }

    // ---- the piece's end: warps 2 and 3 hand their parts to 0 and 1, then 1 to 0; a lane's part is one of the same places ----
#pragma unroll
    for (int n = 0; n < kRowTiles; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], 4);
        sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], 8);
        sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], 16);
      }
    __syncthreads();                                       // the buffers of the piece before have been read
#pragma unroll 1
    for (int from = 2; from > 0; from /= 2) {
      if (warp >= from && warp < 2 * from) {
        float4* to = exchange + (warp & 1) * L::kPart + lane;
#pragma unroll
        for (int n = 0; n < kRowTiles; ++n) {
#pragma unroll
          for (int mt = 0; mt < kDim / 16; ++mt) to[(n * (kDim / 16) + mt) * 32] = make_float4(o[n][mt][0], o[n][mt][1], o[n][mt][2], o[n][mt][3]);
          to[(kRowTiles * (kDim / 16) + n) * 32] = make_float4(top[n][0], top[n][1], sum[n][0], sum[n][1]);
        }
      }
      __syncthreads();
      if (warp < from) {
        const float4* with = exchange + (from == 2 ? warp : 1) * L::kPart + lane;
#pragma unroll
        for (int n = 0; n < kRowTiles; ++n) {
          const float4 other = with[(kRowTiles * (kDim / 16) + n) * 32];
          const float their_top[2] = {other.x, other.y}, their_sum[2] = {other.z, other.w};
          float mine[2], theirs[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float m = fmaxf(top[n][e], their_top[e]);
            mine[e] = top[n][e] == -INFINITY ? 0.0f : Exp2(top[n][e] - m);
            theirs[e] = their_top[e] == -INFINITY ? 0.0f : Exp2(their_top[e] - m);
            sum[n][e] = sum[n][e] * mine[e] + their_sum[e] * theirs[e];
            top[n][e] = m;
          }
#pragma unroll
          for (int mt = 0; mt < kDim / 16; ++mt) {
            const float4 v = with[(n * (kDim / 16) + mt) * 32];
            o[n][mt][0] = o[n][mt][0] * mine[0] + v.x * theirs[0], o[n][mt][1] = o[n][mt][1] * mine[1] + v.y * theirs[1];
            o[n][mt][2] = o[n][mt][2] * mine[0] + v.z * theirs[0], o[n][mt][3] = o[n][mt][3] * mine[1] + v.w * theirs[1];
          }
        }
      }
    }
    if (warp == 0) {
      const bool complete = walk.offset == 0 && walk.Units() == span.units;
      if (lane == 0 && walk.offset == 0 && !complete) {
        const int32_t first = share.begin + (share.left - walk.left);    // the item's first unit
        a.cut[blockIdx.x] = make_int4(walk.b, walk.item, shared_deal.CtaOf(first + span.units - 1) - static_cast<int32_t>(blockIdx.x) + 1, span.count);
      }
      float* slot = a.work + (static_cast<int64_t>(blockIdx.x) * 2 + (walk.offset == 0 ? 1 : 0)) * L::kSlot;
      constexpr int kRun = kDim == 64 ? 8 : 16;              // columns in a row that a lane holds
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = n * 8 + 2 * t + e;
#pragma unroll
          for (int part = 0; part < kDim / 8 / kRun; ++part) {
            float run[kRun];
#pragma unroll
            for (int j = 0; j < kRun; ++j) run[j] = o[n][part * 8 + j / 2][e + j % 2 * 2];
            const int d = part * 128 + g * kRun;
            if (complete) {
              if (row0 + row < a.rows) StoreRow(a, walk.b, head, row0 + row, span.count, d, run, top[n][e], sum[n][e]);
            } else {
#pragma unroll
              for (int j = 0; j < kRun / 4; ++j) *reinterpret_cast<float4*>(slot + row * kDim + d + 4 * j) = make_float4(run[4 * j], run[4 * j + 1], run[4 * j + 2], run[4 * j + 3]);
              if (d == 0) {
                slot[L::kRows * kDim + row] = top[n][e];
                slot[L::kRows * kDim + L::kRows + row] = sum[n][e];
              }
            }
          }
        }
    }
  }
}

// Joins the pieces of the item that the end of CTA blockIdx.x's share cuts first: maximum over the pieces, then the
// pieces' sums and values times exp2(their maximum - it), in the order of the pieces.  A warp has a row, and sends for 8
// pieces at once, or 4 where a block has 16 rows.  (Blocks of 8 rows come in as soon as one block of the first kernel has left; 32
// sequences of 0 to 4096 tokens 33.7 us, with 4 pieces at once 34.4, and with two warps for a row and 4 pieces each 34.1.)
template <int kRowTiles>
constexpr int kJoinThreads = 256 * kRowTiles;

template <int kDim, int kRowTiles>
__global__ void __launch_bounds__(kJoinThreads<kRowTiles>) kv_attention_join_kernel(const AttentionArgs a) {
  using L = Layout<kDim, kRowTiles>;
  static_assert(kJoinThreads<kRowTiles> == 32 * L::kRows);
  constexpr int kVectors = kDim == 256 ? 2 : 1;             // of four columns, per lane
  const int c = blockIdx.x, row = threadIdx.x / 32, lane = threadIdx.x % 32;
  griddep_wait();
  if (threadIdx.x == 0) griddep_launch_dependents();
  const int4 cut = a.cut[c];
  const int pieces = cut.z, item_row = (cut.y % a.blocks) * L::kRows + row;
  if (pieces == 0 || item_row >= a.rows) return;
  auto slot_of = [&](int p) { return a.work + (static_cast<int64_t>(c + p) * 2 + (p == 0 ? 1 : 0)) * L::kSlot; };
  // A few pieces are sent for at once; their maximum is known when they come.
  constexpr int kAtOnce = kRowTiles == 1 ? 8 : 4;
  const bool mine = lane * 4 < kDim;
  float first_max[kAtOnce], first_sum[kAtOnce];
  float4 first_values[kAtOnce][kVectors];
#pragma unroll
  for (int p = 0; p < kAtOnce; ++p) {
    first_max[p] = -INFINITY, first_sum[p] = 0.0f;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) first_values[p][i] = make_float4(0, 0, 0, 0);
    if (p < pieces) {
      const float* slot = slot_of(p);
      first_max[p] = slot[L::kRows * kDim + row], first_sum[p] = slot[L::kRows * kDim + L::kRows + row];
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
        if (mine) first_values[p][i] = *reinterpret_cast<const float4*>(slot + row * kDim + i * 128 + lane * 4);
    }
  }
  float m = -INFINITY;
  for (int p = lane; p < pieces; p += 32) m = fmaxf(m, slot_of(p)[L::kRows * kDim + row]);
#pragma unroll
  for (int o = 16; o > 0; o /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float total = 0.0f;
  float4 y[kVectors] = {};
  auto add = [&](float piece_max, float piece_sum, const float4 (&v)[kVectors]) {
    const float fade = piece_max == -INFINITY ? 0.0f : Exp2(piece_max - m);
    total = fmaf(piece_sum, fade, total);
#pragma unroll
    for (int i = 0; i < kVectors; ++i) y[i].x = fmaf(v[i].x, fade, y[i].x), y[i].y = fmaf(v[i].y, fade, y[i].y), y[i].z = fmaf(v[i].z, fade, y[i].z), y[i].w = fmaf(v[i].w, fade, y[i].w);
  };
#pragma unroll
  for (int p = 0; p < kAtOnce; ++p) add(first_max[p], first_sum[p], first_values[p]);
#pragma unroll 8
  for (int p = kAtOnce; p < pieces; ++p) {
    const float* slot = slot_of(p);
    const float piece_max = slot[L::kRows * kDim + row], piece_sum = slot[L::kRows * kDim + L::kRows + row];
    float4 v[kVectors] = {};
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      if (mine) v[i] = *reinterpret_cast<const float4*>(slot + row * kDim + i * 128 + lane * 4);
    add(piece_max, piece_sum, v);
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i)
    if (mine) {
      const float run[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
      StoreRow(a, cut.x, cut.y / a.blocks, item_row, cut.w, i * 128 + lane * 4, run, m, total);
    }
}

struct Variant {
  void (*main[2])(AttentionArgs, CUtensorMap, CUtensorMap);       // of bf16, of f16
  void (*join)(AttentionArgs);
  int dim, row_tiles, bytes, slot, step;
};
template <int kCode, int kDim, int kRowTiles>
constexpr Variant MakeVariant() {
  using L = Layout<kDim, kRowTiles>;
  return {{kv_attention_kernel<kCode, kDim, kRowTiles, false>, kv_attention_kernel<kCode, kDim, kRowTiles, true>}, kv_attention_join_kernel<kDim, kRowTiles>, kDim, kRowTiles, L::kBytes, L::kSlot, L::kStep};
}
// Per cache type: heads up to 64, 128 and 256 wide, 8 or 16 rows at a time.  16 rows of 256 columns do not fit the registers.
constexpr int kShapes = 5;
#define B200SD_ATTENTION_VARIANTS(code) MakeVariant<code, 64, 1>(), MakeVariant<code, 64, 2>(), MakeVariant<code, 128, 1>(), MakeVariant<code, 128, 2>(), MakeVariant<code, 256, 1>()
const Variant kVariants[3][kShapes] = {{B200SD_ATTENTION_VARIANTS(kF8E4M3FN)}, {B200SD_ATTENTION_VARIANTS(kF8E5M2)}, {B200SD_ATTENTION_VARIANTS(kS8)}};
#undef B200SD_ATTENTION_VARIANTS
int g_ctas_per_sm[3][kShapes][2];               // the same on every B200; written once, by the first InitAttentionKernels

int ShapeIndex(int64_t head_dim, int64_t rows) {
  if (head_dim > 128) return 4;
  return (head_dim > 64 ? 2 : 0) + (rows > 8 ? 1 : 0);
}

}  // namespace

Status InitAttentionKernels() {
  int ctas[3][kShapes][2];
  for (int c = 0; c < 3; ++c)
    for (int s = 0; s < kShapes; ++s)
      for (int f = 0; f < 2; ++f) {
        const Variant& v = kVariants[c][s];
        cudaError_t e = cudaFuncSetAttribute(v.main[f], cudaFuncAttributeMaxDynamicSharedMemorySize, v.bytes);
        int n = 0;
        // The two kernels alternate on an SM; with the same split of its memory it needs not be empty in between.
        if (e == cudaSuccess) e = cudaFuncSetAttribute(v.main[f], cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(v.join, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, v.main[f], kThreads, v.bytes);
        if (e != cudaSuccess) return Status::Error(kInternal, std::string("kv_attention_kernel set-up: ") + cudaGetErrorString(e));
        ctas[c][s][f] = n > 0 ? n : 1;
      }
  static std::once_flag once;                   // another device may be launching already
  std::call_once(once, [&] { std::memcpy(g_ctas_per_sm, ctas, sizeof(ctas)); });
  return Status::Ok();
}

Status ValidatePagedAttention(const B200SD_PagedAttention& a, bool check_pointers) {
  auto bad = [](const std::string& m) { return Status::Error(kInvalidArgument, m); };
  if (a.struct_size < sizeof(a)) return bad("B200SD_PagedAttention.struct_size is smaller than this library's struct");
  Status st = ValidateCache(a, a.q_dtype, check_pointers);
  if (!st.ok()) return st;
  if (a.heads < 1 || a.heads > 4096 || a.heads % a.kv_heads) return bad("heads must be a multiple of kv_heads, at most 4096");
  if (a.new_tokens > 64) return Status::Error(kUnimplemented, "more than 64 new tokens for a sequence");
  if (a.window < 0) return bad("window must not be negative");
  if (!(a.softmax_scale - a.softmax_scale == 0.0f)) return bad("softmax_scale must be finite");
  const int64_t rows = a.new_tokens * (a.heads / a.kv_heads), block = 8 * kVariants[0][ShapeIndex(a.head_dim, rows)].row_tiles;
  if (a.batch * a.kv_heads * ((rows + block - 1) / block) > kMostItems) return Status::Error(kUnimplemented, "too many queries for one call");
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
  B200SD_PagedAttention a{};
  a.struct_size = sizeof(a);
  a.batch = batch, a.new_tokens = new_tokens, a.heads = heads, a.kv_heads = kv_heads, a.head_dim = head_dim;
  a.page_tokens = 16, a.q_dtype = kBF16, a.cache_dtype = kS8;
  if (batch == 0 || new_tokens == 0 || !ValidatePagedAttention(a, /*check_pointers=*/false).ok()) return 0;
  const Variant& v = kVariants[0][ShapeIndex(head_dim, new_tokens * (heads / kv_heads))];
  return kMaxCtas * (2 * v.slot * sizeof(float) + sizeof(int4));
}

Status LaunchPagedAttention(const B200SD_PagedAttention& a, cudaStream_t stream, LaunchStats* stats) {
  if (a.batch == 0 || a.new_tokens == 0) return Status::Ok();
  const int code = a.cache_dtype == kF8E4M3FN ? 0 : a.cache_dtype == kF8E5M2 ? 1 : 2;
  const int64_t rows = a.new_tokens * (a.heads / a.kv_heads);
  const int shape = ShapeIndex(a.head_dim, rows);
  const Variant& v = kVariants[code][shape];
  const int of_type = a.q_dtype == kF16 ? 1 : 0, ctas_per_sm = g_ctas_per_sm[code][shape][of_type];
  const int64_t block = 8 * v.row_tiles, blocks = (rows + block - 1) / block;
  int shift = 4;
  while ((1 << shift) < a.page_tokens) ++shift;
  // The most positions that a sequence's rows see.  Where their keys are few bytes it is not cut: the second kernel would
  // cost more than it saves.  (Cut and not, in us: 4 sequences, 8 heads of 128, up to 250 tokens 10.5 and 8.8, 500 10.9 and
  // 11.4, 1000 11.3 and 16.5; heads of 64, 500 tokens 10.7 and 10.3, 1000 13.4 and 14.8; of 256, 250 tokens 11.8 and 12.2; 64
  // sequences, heads of 128, 250 tokens 17.8 and 16.7, 500 24.4 and 25.2.)
  const int64_t window = std::min(a.window, int64_t{1} << 30);          // as good as none: no sequence is longer
  const int64_t capacity = a.table_width * a.page_tokens, seen = window > 0 ? std::min(capacity, window + a.new_tokens + kTile) : capacity;
  const bool cut = seen * v.dim > (48 << 10);
  int unit_shift = 30;
  if (cut)
    for (unit_shift = 6; (1 << unit_shift) < v.step; ++unit_shift) {}
  const auto units = [&] { return (seen + (int64_t{1} << unit_shift) - 1) >> unit_shift; };
  while (a.batch * a.kv_heads * blocks * (units() + 16) >= INT32_MAX) ++unit_shift;       // the line's positions are 32-bit numbers
  // An item costs a CTA about 4 us besides its tokens, as much as it needs for 192 KiB of them shared by the CTAs of an SM.
  // (When it was added, sequences of 0 to 4096 tokens, in us without and with: 41 and 37; 40 rows per key head: 107 and 60.)
  const int extra = cut ? std::max(1, static_cast<int>((192 << 10) / (ctas_per_sm * v.step * v.dim * 2))) : 0;
  AttentionArgs args{a.q, static_cast<const uint8_t*>(a.k_pages), static_cast<const uint8_t*>(a.v_pages), a.k_scale, a.v_scale,
                     a.page_table, a.seq_lens, a.new_lens, a.out, a.lse, static_cast<float*>(a.workspace),
                     reinterpret_cast<int4*>(static_cast<float*>(a.workspace) + int64_t{kMaxCtas} * 2 * v.slot),
                     static_cast<int32_t>(a.batch), static_cast<int32_t>(a.new_tokens), static_cast<int32_t>(a.heads), static_cast<int32_t>(a.kv_heads),
                     static_cast<int32_t>(a.head_dim), shift, static_cast<int32_t>(rows), static_cast<int32_t>(blocks),
                     static_cast<int32_t>(a.num_pages), static_cast<int32_t>(a.table_width), static_cast<int32_t>(window),
                     unit_shift, extra, cut ? 2 : 1, a.softmax_scale * 1.4426950408889634f, a.q_dtype == kBF16, LoseCopy(), StatusWordPtr()};
  CUtensorMap key_map, value_map;
  const bool none = a.num_pages == 0;                                 // then no page is valid, and no tile is loaded
  const int64_t matrices = none ? 1 : a.num_pages * a.kv_heads;
  Status st = MakeTileMap(&key_map, none ? a.q : a.k_pages, matrices, none ? 16 : a.page_tokens, none ? 16 : a.head_dim, v.dim == 64 ? 64 : 128);
  if (st.ok()) st = MakeTileMap(&value_map, none ? a.q : a.v_pages, matrices, none ? 16 : a.page_tokens, none ? 16 : a.head_dim, v.dim == 64 ? 64 : 128);
  if (!st.ok()) return st;
  const int64_t most = a.batch * a.kv_heads * blocks * (cut ? units() + extra : 1);
  int64_t grid = static_cast<int64_t>(DeviceSmCount()) * ctas_per_sm;
  grid = grid < kMaxCtas ? grid : kMaxCtas;
  // No more CTAs than take part where all items are as large as the largest (see Locate).
  const int64_t items = a.batch * a.kv_heads * blocks;
  grid = grid < items * 128 ? grid : items * 128;
  grid = grid < most ? grid : most;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;     // see griddep_wait() in the kernels
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = v.bytes;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, v.main[of_type], args, key_map, value_map);
  stats->launches = 1;
  if (e == cudaSuccess && cut) {
    cfg.blockDim = dim3(v.row_tiles == 1 ? kJoinThreads<1> : kJoinThreads<2>);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, v.join, args);
    stats->launches = 2;
  }
  if (e != cudaSuccess) return Status::Error(kInternal, std::string("kv_attention_kernel launch: ") + cudaGetErrorString(e));
  return Status::Ok();
}

}  // namespace b200sd
