// Dots of a few rows with 4-bit weights and a scale for each group along k.
//
// Bound by reading the weights once (n * k / 2 bytes); at the copy rate an SM has about 44 clocks for a KiB of them, 176
// instruction slots for 2048 weights, so the other half of the work is decoding cheaply.
//
// Products run on mma.m16n8k16 with 16 weight rows on the large side and 8 rows of x on the other: A is the weights as
// they lie in memory, B is x.  The order along k inside a product is free, so a lane feeds two products from one
// 32-bit word of 8 weights, in the pairs (0, 4), (1, 5), (2, 6), (3, 7) of its nibbles, and x is paired the same way.  A
// lane's word, half or whole 16-byte piece is chosen so that one product never mixes two groups; a group's f32 sum is
// multiplied by its scale in f32 and added up.
//
// A CTA owns n / CTAs consecutive rows, whole rows of bytes with none read twice or by two CTAs whatever n is.  A block of
// 32 of its rows and 128 of k are a unit, which a warp brings in through its own cp.async ring.
//
// A masked nibble plus an offset is an f16 or bf16 number (1024 + n, 128 + n), and one subtraction leaves w - z, exactly: 9
// instructions for 8 weights in f16, 11 in bf16.  The wide kernel takes x as it is, in phases that the warps of a CTA share.
// The other one, for one or two rows, first puts all of x into shared memory, paired, as f16 whatever its type: f16 as it is, a
// bf16 row multiplied by the power of two that brings its largest finite value to 2^15 (what lies 2^32 below that is rounded,
// to 2^-40 of it).
// (Cheaper operands were tried and lost bits.  The nibbles as they stand under a mask, 16-bit subnormals, are 5 instructions, but
// the zero points then come off a group's sum as z times the sum of x: at an outlier of x whose weight is z, the sum before is
// many times the one after.  And products of subnormals are lined up for the sum by the exponent that they would have if they
// were normal, so that 10 of the 24 bits of an f32 sum are zeros.)
//
// Measured with cold caches: 28672 x 8192 in groups of 128 for one row 34 us (3.6 TB/s; the bytes alone take 18.5), 8192 x
// 28672 with zero points for 16 rows 59.4 us, 5003 x 4416 in groups of 32 for 5 rows 10.8 us, 1024 x 2048 for one row 7.6
// us, the host's part of a call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <string>
#include <type_traits>

#include "kernels.h"
#include "ptx.cuh"

namespace b200sd {
namespace {

struct W4Args {
  const void* x;
  const uint8_t* w;
  const void* scale;
  const uint8_t* zero;
  const void* bias;
  void* d;
  int32_t m, n, k, groups;
  int32_t group_shift;                          // log2 of the 128-blocks of k in a group (groups of 128 and more) ...
  int32_t blocks_per_group;                     // ... or their number where it is no power of two
  int32_t rows, rows_left;                      // of a CTA: `rows`, and one more for the first `rows_left`
  int32_t steps, per_round;                     // 128-blocks of k; blocks of rows whose sums fit shared memory, or steps of a phase
  uint32_t* status;
  uint32_t piece_inverse;                       // 2^32 / (16 * steps), rounded up
  int32_t x_is_bf16, scale_dtype, bias_dtype, d_dtype, is_signed;
  int32_t lose;                                 // LoseCopy()
};

// Scales and bias: their bits, loaded ahead, and what they stand for.  kType 0 takes the type from the arguments.
template <int kType>
__device__ __forceinline__ uint32_t LoadBits(const void* p, int64_t i, int32_t dtype) {
  if (kType == kF32 || (kType == 0 && dtype == kF32)) return static_cast<const uint32_t*>(p)[i];
  return static_cast<const uint16_t*>(p)[i];
}
template <int kType>
__device__ __forceinline__ float ValueOf(uint32_t bits, int32_t dtype) {
  if (kType == kF32 || (kType == 0 && dtype == kF32)) return __uint_as_float(bits);
  if (kType == kBF16 || (kType == 0 && dtype == kBF16)) return __uint_as_float(bits << 16);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}
__device__ __forceinline__ void CopyAsync16If(bool wanted, uint32_t dst, const void* src) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p cp.async.cg.shared.global [%0], [%1], 16;\n\t}" ::"r"(dst), "l"(src), "r"(static_cast<int>(wanted)) : "memory");
}
// Loads that stay whole (a compiler short of registers takes a vector apart), from addresses that stay in registers.
__device__ __forceinline__ uint4 LoadShared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void StoreShared16(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint2 LoadShared8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t LoadShared4(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t Kept(uint32_t x) {
  asm volatile("" : "+r"(x));
  return x;
}
__device__ __forceinline__ void CopyAsync16OrZero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// (w & mask) ^ magic in one instruction; written out because the compiler splits it where a part of `magic` is not constant.
__device__ __forceinline__ uint32_t MaskXor(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(v) : "r"(w), "r"(mask), "r"(magic));
  return v;
}

// How a word's nibbles become operands, w - z, exactly; `flip` (8 for two's complement) turns -8 .. 7 into 0 .. 15 with zero point 8.
// The offsets -(1024 + z), -(64 + z) and -(128 + z) of one weight row and group have z in their low bits,
// so they are put together, not converted.
template <typename T> struct Offset;
template <> struct Offset<__half> {
  uint32_t low, high;
  __device__ void Set(uint32_t z) { low = 0xe400e400u | z * 0x00010001u, high = 0xd400d400u | z * 0x00100010u; }
  __device__ __forceinline__ void Decode8(uint32_t w, uint32_t flip, uint32_t (&v)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t a = MaskXor(w >> (8 * i), 0x000f000fu, 0x64006400u ^ flip);                  // 1024 + n
      const uint32_t b = MaskXor(w >> (8 * i), 0x00f000f0u, 0x64006400u ^ flip << 4);             // 1024 + 16 n
      asm("add.f16x2 %0, %1, %2;" : "=r"(v[2 * i]) : "r"(a), "r"(low));
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v[2 * i + 1]) : "r"(b), "r"(0x2c002c00u), "r"(high));   // times 1 / 16
    }
  }
};
template <> struct Offset<__nv_bfloat16> {
  uint32_t low;
  __device__ void Set(uint32_t z) { low = 0xc300c300u | z * 0x00010001u; }
  __device__ __forceinline__ void Decode8(uint32_t w, uint32_t flip, uint32_t (&v)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = MaskXor(w >> (4 * i), 0x000f000fu, 0x43004300u ^ flip);                  // 128 + n
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v[i]) : "r"(a), "r"(0x3f803f80u), "r"(low));     // times 1
    }
  }
};

template <typename T>
__device__ __forceinline__ void Mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Either kernel's unit is 32 weight rows, in two tiles of the products, by 128 of k.
constexpr int kTiles = 2, kRows = 16 * kTiles, kStageBytes = kTiles * 1024;
using One = std::integral_constant<int, 1>;      // tiles of a unit that have rows of weights
using Two = std::integral_constant<int, 2>;
constexpr int kSumStride = kRows + 4;           // floats between two rows of x in the sums
constexpr int kStages = 3;                      // of a warp's ring

// Where 16-byte piece `c` of weight row `r` (64 bytes of a unit) and piece `c` of row `r` of x (256 bytes) lie: so that the
// reads below have no bank conflicts.
__device__ __forceinline__ int WeightPiece(int r, int c) { return r * 64 + (c ^ ((r & 2) | ((r >> 2) & 1))) * 16; }
template <int kGroup>
__device__ __forceinline__ int InputPiece(int r, int c) {
  const int at = kGroup == 128 ? (c % 4) * 4 + c / 4 : kGroup == 64 ? (c & 8) + (c % 2) * 4 + c % 8 / 2 : c;
  return r * 256 + (at ^ ((r & 1) << 2)) * 16;
}

// Eight values of x in the order of the weights' pairs.
__device__ __forceinline__ uint4 Paired(uint4 v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
}

// The two values of a word of x, in f32.
__device__ __forceinline__ float2 Unpack(uint32_t w, bool is_bf16) {
  if (is_bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// All of x to shared memory, `inputs`: paired, as f16, scaled if it was bf16; `factors` [row] what brings a row's sums
// back.  The copies are under way before the weights', so that they do not
// queue behind them; a thread works on the pieces that it has copied itself, in place.  The loops are not unrolled: this
// code runs once, and its instructions are fetched cold.
template <int kGroup, int kThreads>
struct Staging {
  const W4Args& a;
  int all, total;                               // pieces of 16 bytes of a row, with its padding to whole steps, and of all rows
  uint32_t inverse, inputs;
  __device__ Staging(const W4Args& args, uint32_t to) : a(args), all(args.steps * 16), total(all * args.m), inverse(args.piece_inverse), inputs(to) {}
  __device__ __forceinline__ void Place(int i, int& r, int& c, uint32_t& at) const {
    r = all == total ? 0 : static_cast<int>(__umulhi(i, inverse));       // i / all, for i < total and total * all < 2^32
    c = i - r * all;
    at = inputs + (c / 16 * a.m) * 256 + InputPiece<kGroup>(r, c % 16);
  }
  __device__ __forceinline__ void Copy() const {
    int r, c;
    uint32_t at;
#pragma unroll 1
    for (int i = threadIdx.x; i < total; i += kThreads) {
      Place(i, r, c, at);
      const bool there = c < a.k / 8;
      CopyAsync16OrZero(at, there ? static_cast<const uint16_t*>(a.x) + (r * a.k + c * 8) : a.x, there);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // `top` [row] holds zeros on entry.
  __device__ __forceinline__ void Convert(float* factors, uint32_t* top) const {
    int r, c;
    uint32_t at;
    if (a.x_is_bf16) {
      const uint32_t lanes = threadIdx.x % 32 < 16 ? 0x0000ffffu : 0xffff0000u;     // 16 lanes in a row share r
      auto finite = [](uint32_t w) {
        w &= 0x7fff7fffu;
        if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
        if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
        return w;
      };
#pragma unroll 1
      for (int i = threadIdx.x; i < total; i += kThreads) {
        Place(i, r, c, at);
        const uint4 v = LoadShared16(at);
        const uint32_t both = __vmaxu2(__vmaxu2(finite(v.x), finite(v.y)), __vmaxu2(finite(v.z), finite(v.w)));
        const uint32_t most = __reduce_max_sync(lanes, max(both & 0xffffu, both >> 16));
        if (threadIdx.x % 16 == 0 && most > 0) atomicMax(top + r, most << 16);
      }
      __syncthreads();
    }
#pragma unroll 1
    for (int i = threadIdx.x; i < total; i += kThreads) {
      Place(i, r, c, at);
      uint4 v = LoadShared16(at);
      const int power = top[r] == 0 ? 0 : min(126, 15 - (static_cast<int>(top[r] >> 23) - 127));
      if (a.x_is_bf16) {
        const float up = __uint_as_float(static_cast<uint32_t>(127 + power) << 23);
        auto scaled = [&](uint32_t w) {
          const float2 x = Unpack(w, true);
          const __half2 h = __floats2half2_rn(x.x * up, x.y * up);
          return *reinterpret_cast<const uint32_t*>(&h);
        };
        v = make_uint4(scaled(v.x), scaled(v.y), scaled(v.z), scaled(v.w));
      }
      StoreShared16(at, Paired(v));
      if (c == 0) factors[r] = __uint_as_float(static_cast<uint32_t>(127 - power) << 23);
    }
    __syncthreads();
  }
};

struct Resident {
  static constexpr int kWarps = 24, kMost = 2;              // kMost: rows of x
  static constexpr int kBlocks = 8;                         // whose sums have room, for one row of x
  static constexpr int kSums = kBlocks * kWarps * kSumStride;
  // Each row's factor, its largest value, and what is behind them up to whole lines of banks.
  static constexpr int kHead = (kSums * 4 + 2 * kMost * 4 + 127) / 128 * 128, kRing = kWarps * kStages * kStageBytes;
  static int64_t PerRound(int64_t m, int64_t) { return kBlocks / m; }
  static int64_t Bytes(int64_t m, int64_t steps) { return kHead + kRing + steps * m * 256; }
};

// One or two rows of x, all of it in shared memory.  The warps take the units of the CTA in turn and leave their sums of
// each block in shared memory, where they are added in the order of the warps, as many blocks at a time as have room.  Bound
// by issue, about 380 instructions of a warp for a unit of 2 KiB with all that surrounds it, and by 8 us in front and
// behind: x, the first units, the sums.  (With the nibbles as operands 24 warps took 33.4 us for 28672 x 8192 and one row, and
// 16 took 36.4.)  kGroup: 32, 64 or 128
// (which stands for its multiples too).  kScale: the scales' type, kSigned: two's complement, no zero points.
template <int kGroup, int kScale, bool kSigned>
__global__ void __launch_bounds__(Resident::kWarps * 32) w4_dot_kernel(const __grid_constant__ W4Args a) {
  using S = Resident;
  constexpr int kPerStep = 128 / kGroup;                    // groups of a step
  constexpr int kWords = kGroup / 32;                       // words of a lane in a group
  constexpr int kWarps = S::kWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  if (threadIdx.x == 0) griddep_launch_dependents();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int cta = blockIdx.x, first = cta * a.rows + min(cta, a.rows_left), last = first + a.rows + (cta < a.rows_left ? 1 : 0);
  const int steps = a.steps, row_bytes = a.k / 2, blocks = (last - first + kRows - 1) / kRows, per_round = a.per_round;
  float* sums = reinterpret_cast<float*>(smem);
  float* factors = sums + S::kSums;
  uint8_t* ring = smem + S::kHead + warp * kStages * kStageBytes;
  uint8_t* resident = smem + S::kHead + S::kRing;
  constexpr uint32_t flip = kSigned ? 0x00080008u : 0u;
  // A CTA's rows of the weights and of the scales span less than 4 GiB, so 32-bit offsets from its first row do.
  const uint8_t* w_base = a.w + static_cast<int64_t>(first) * row_bytes;
  const uint8_t* scale_base = static_cast<const uint8_t*>(a.scale) + static_cast<int64_t>(first) * a.groups * (kScale == kF32 ? 4 : 2);
  const uint8_t* zero_base = a.zero + static_cast<int64_t>(first) * a.groups;

  // A warp's units of a round of blocks are the warp-th, the (warp + warps)-th ... of the line (block, step): within a block
  // every kWarps-th step, and what is left over carries into the next block.
  //
  // Loading: each lane brings piece `t` of rows g, g + 8, ... of a unit.  What lies behind the last row or the end of k is
  // not loaded: old bytes there are finite weights too, of rows that are not stored or against a 0 of x.
  const uint32_t eight_rows = 8 * row_bytes, next_block = kRows * row_bytes - steps * 64;
  int load_step = warp, load_block = 0, load_round = per_round, load_rows = last - first - g;
  uint32_t load_from = static_cast<uint32_t>(g) * row_bytes + warp * 64 + t * 16, load_to = Kept(smem_u32(ring) + WeightPiece(g, t));
  auto to_next_block = [&] {
    while (load_step >= steps && load_block < blocks) {
      ++load_block;
      load_rows -= kRows;
      load_step -= steps;
      load_from += next_block;
      if (load_block == load_round) {                       // every round starts with the warp-th unit
        load_round += per_round;
        load_from += (warp - load_step) * 64;
        load_step = warp;
      }
    }
  };
  if (load_step >= steps) to_next_block();
  auto load = [&](uint32_t stage) {                         // `stage`: its place in the ring, in bytes
    if (load_block < blocks) {
      const uint32_t dst = load_to + stage;
      const int rows = load_step * 64 + t * 16 < row_bytes ? load_rows : 0;
#pragma unroll
      for (int i = 0; i < 2 * kTiles; ++i)
        CopyAsync16If(8 * i < rows, dst + i * 512, w_base + (load_from + i * eight_rows));
      load_step += kWarps;
      load_from += kWarps * 64;
      if (load_step >= steps) to_next_block();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // Scales and zero points of a unit for this lane's rows; with several groups in a step the four lanes of a row hold one
  // each.  Rows behind the last take its numbers, groups behind the end of k a scale of 0.  They are loaded a unit ahead,
  // into the registers that the unit before has just used; in front of a block, its first unit's.
  uint32_t scale[kTiles][2], zero[kTiles][2], row_at[kTiles][2];
  auto load_numbers = [&](int step, auto tiles_of_unit) {
    const uint32_t group = kGroup == 128 ? (a.group_shift >= 0 ? step >> a.group_shift : step / a.blocks_per_group) : step * kPerStep + t % kPerStep;
    const bool there = kGroup == 128 || group < a.groups;
#pragma unroll
    for (int r = 0; r < decltype(tiles_of_unit)::value; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = row_at[r][h] + (there ? group : 0);
        scale[r][h] = LoadBits<kScale>(scale_base, at, a.scale_dtype);
        if (!there) scale[r][h] = 0;
        if (!kSigned) zero[r][h] = zero_base[at] & 15u;
      }
  };
  auto set_rows = [&](int block) {
    const int row = min(block, blocks - 1) * kRows + g, most = last - first - 1;
#pragma unroll
    for (int r = 0; r < kTiles; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) row_at[r][h] = static_cast<uint32_t>(min(row + r * 16 + h * 8, most)) * a.groups;
  };

  uint32_t* top = reinterpret_cast<uint32_t*>(factors + S::kMost);
  if (threadIdx.x < S::kMost) top[threadIdx.x] = 0;
  __syncthreads();
  griddep_wait();
  const Staging<kGroup, kWarps * 32> staging(a, smem_u32(resident));
  staging.Copy();
#pragma unroll 1
  for (int s = 0; s < kStages - 1; ++s) load(s * kStageBytes);
  set_rows(0);
  load_numbers(min(warp, steps - 1), Two());
  asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");         // this thread's part of x has come
  staging.Convert(factors, top);

  // Places of this lane's words and of its pieces of x; behind the last row of x any will do, its column is not stored.
  uint32_t weight_at[kPerStep], input_at[4];
#pragma unroll
  for (int i = 0; i < kPerStep; ++i)
    weight_at[i] = Kept(smem_u32(ring) + (kGroup == 128 ? WeightPiece(g, t) : kGroup == 64 ? WeightPiece(g, i * 2 + t / 2) + t % 2 * 8 : WeightPiece(g, i) + t * 4));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int piece = kGroup == 128 ? t * 4 + i : kGroup == 64 ? i / 2 * 8 + t * 2 + i % 2 : i * 4 + t;
    input_at[i] = Kept(smem_u32(resident) + InputPiece<kGroup>(min(g, a.m - 1), piece));
  }

  const bool half = (last - first - 1) % kRows < 16;        // of the last block only one tile has rows
  uint32_t stage = 0, load_stage = (kStages - 1) * kStageBytes;
  for (int round = 0; round < blocks; round += per_round) {
    const int round_end = min(round + per_round, blocks);
    int step = warp;
    for (int block = round; block < round_end; ++block) {
      float acc[kTiles][4] = {};
      auto run = [&](auto tiles_of_unit) {
        constexpr int kOfUnit = decltype(tiles_of_unit)::value;
        for (; step < steps; step += kWarps) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
          __syncwarp();
          load(load_stage);
          load_stage = stage;
          const uint32_t inputs = step * (a.m * 256);
#pragma unroll
          for (int group = 0; group < kPerStep; ++group) {
            const int holder = (lane & ~3) | group;           // the lane with this group's numbers
            float part[kTiles][4] = {};
            Offset<__half> decoder[kTiles][2];
#pragma unroll
            for (int r = 0; r < kOfUnit; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h) decoder[r][h].Set(kSigned ? 8u : kGroup == 128 ? zero[r][h] : __shfl_sync(0xffffffffu, zero[r][h], holder));
            // The words of this group, of rows g and g + 8 of each tile.
            uint32_t w[kTiles][2][kWords];
#pragma unroll
            for (int r = 0; r < kOfUnit; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t at = weight_at[group] + stage + (r * 16 + h * 8) * 64;
                if constexpr (kGroup == 128) {
                  const uint4 v = LoadShared16(at);
                  w[r][h][0] = v.x, w[r][h][1] = v.y, w[r][h][2] = v.z, w[r][h][3] = v.w;
                } else if constexpr (kGroup == 64) {
                  const uint2 v = LoadShared8(at);
                  w[r][h][0] = v.x, w[r][h][1] = v.y;
                } else {
                  w[r][h][0] = LoadShared4(at);
                }
              }
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
              const uint4 b = LoadShared16(input_at[group * kWords + i] + inputs);
#pragma unroll
              for (int r = 0; r < kOfUnit; ++r) {
                uint32_t low[4], high[4];
                decoder[r][0].Decode8(w[r][0][i], flip, low);
                decoder[r][1].Decode8(w[r][1][i], flip, high);
                Mma<__half>(part[r], low[0], high[0], low[1], high[1], b.x, b.y);
                Mma<__half>(part[r], low[2], high[2], low[3], high[3], b.z, b.w);
              }
            }
#pragma unroll
            for (int r = 0; r < kOfUnit; ++r) {
              float s0 = ValueOf<kScale>(scale[r][0], kScale), s1 = ValueOf<kScale>(scale[r][1], kScale);
              if (kGroup < 128) s0 = __shfl_sync(0xffffffffu, s0, holder), s1 = __shfl_sync(0xffffffffu, s1, holder);
              acc[r][0] = fmaf(part[r][0], s0, acc[r][0]), acc[r][1] = fmaf(part[r][1], s0, acc[r][1]);
              acc[r][2] = fmaf(part[r][2], s1, acc[r][2]), acc[r][3] = fmaf(part[r][3], s1, acc[r][3]);
            }
          }
          stage = stage == (kStages - 1) * kStageBytes ? 0 : stage + kStageBytes;
          if (step + kWarps < steps) load_numbers(step + kWarps, tiles_of_unit);
        }
      };
      if (half && block == blocks - 1) run(One());
      else run(Two());
      step -= steps;
      if (block + 1 == round_end) step = warp;
      set_rows(block + 1);
      if (step < steps) load_numbers(step, Two());
      // This warp's sums of the block, zeros where it had no unit of it.
      float* mine = sums + ((block - round) * kWarps + warp) * a.m * kSumStride;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (2 * t + e < a.m) {
#pragma unroll
          for (int r = 0; r < kTiles; ++r) {
            mine[(2 * t + e) * kSumStride + r * 16 + g] = acc[r][e];
            mine[(2 * t + e) * kSumStride + r * 16 + 8 + g] = acc[r][e + 2];
          }
        }
    }
    __syncthreads();
    const int rows = min(round_end * kRows, last - first) - round * kRows;
#pragma unroll 1
    for (int i = threadIdx.x; i < rows; i += kWarps * 32) {
      const int at = first + round * kRows + i;
      const float bias = a.bias != nullptr ? ValueOf<0>(LoadBits<0>(a.bias, at, a.bias_dtype), a.bias_dtype) : 0.0f;
#pragma unroll 1
      for (int x_row = 0; x_row < a.m; ++x_row) {
        const float* part = sums + (i / kRows * kWarps * a.m + x_row) * kSumStride + i % kRows;
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) y += part[w * a.m * kSumStride];
        y = y * factors[x_row] + bias;
        const int64_t place = static_cast<int64_t>(x_row) * a.n + at;
        if (a.d_dtype == kBF16) static_cast<__nv_bfloat16*>(a.d)[place] = __float2bfloat16_rn(y);
        else if (a.d_dtype == kF16) static_cast<__half*>(a.d)[place] = __float2half_rn(y);
        else static_cast<float*>(a.d)[place] = y;
      }
    }
    __syncthreads();                                        // the sums have been read
  }
}

// Up to 32 rows of x, as they are.  All warps of a CTA share a phase of x, some steps of k for all rows, as it is stored (one
// bulk copy per row); the next one is on its way meanwhile.  A warp keeps its block of 32 weight rows from the first phase
// to the last, alone or with others that take every so manieth step of it, and its sums in registers, so x is read once per
// CTA (per 512 of its rows).  Bound by issue and the matrix pipe: 463 instructions of a warp for a unit and 16 rows.
// (x through each warp's ring beside the weights, once for every block of 32 rows, took 292 us instead of 149 for 33 rows
// against 28672 x 8192, 15.0 instead of 11.7 for 5 rows against 5003 x 4416.)  16 warps leave 128 registers to a thread;
// 20 and 24 were slower, by 3 % and 7 % at 8 rows and, short of registers, by half and more at 16.  Four columns of products, for
// 17 to 32 rows, spill up to 140 bytes of a thread: 28672 x 8192 takes 51 us for 16 rows, 89 for 17 and 96 for 32.
template <typename T_, int kCols_>
struct WideShape {
  using T = T_;
  static constexpr int kCols = kCols_, kWarps = 16;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  // Steps of a phase: as many as fit, twice, for every phase costs a barrier.
  static int64_t Phase(int64_t m, int64_t steps) { return std::min<int64_t>(steps, ((227 * 1024 - kRing - 64) / (2 * m) - 16) / 256); }
  static int64_t Bytes(int64_t m, int64_t steps) { return kRing + 64 + m * std::max<int64_t>(2 * (Phase(m, steps) * 256 + 16), kWarps * kSumStride * 4); }
};

template <int kGroup, typename S>
__global__ void __launch_bounds__(S::kWarps * 32) w4_dot_wide_kernel(const __grid_constant__ W4Args a) {
  using T = typename S::T;
  constexpr int kPerStep = 128 / kGroup, kWords = kGroup / 32, kCols = S::kCols, kWarps = S::kWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  if (threadIdx.x == 0) griddep_launch_dependents();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const bool is_signed = a.is_signed != 0;
  const uint32_t flip = is_signed ? 0x00080008u : 0u;
  const int cta = blockIdx.x, first = cta * a.rows + min(cta, a.rows_left), last = first + a.rows + (cta < a.rows_left ? 1 : 0);
  const int steps = a.steps, row_bytes = a.k / 2, phase_steps = a.per_round, phases = (steps + phase_steps - 1) / phase_steps;
  uint8_t* ring = smem + warp * kStages * 2048;
  uint64_t* arrived = reinterpret_cast<uint64_t*>(smem + S::kRing);          // of the two halves of the buffer of x
  volatile int* abort_flag = reinterpret_cast<int*>(arrived + 2);
  uint8_t* x_buffer = smem + S::kRing + 64;
  float* sums = reinterpret_cast<float*>(x_buffer);                          // at the end
  const int x_pitch = phase_steps * 256 + 16;               // bytes between two rows of x in a phase: neighbours not in the same banks
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_init(&arrived[0], 1);
    mbar_init(&arrived[1], 1);
    fence_mbar_init();
  }
  __syncthreads();
  griddep_wait();

  uint32_t x_parity = 0;                                    // bit h: parity of the next wait for half h
  const uint64_t limit = kTiming && a.lose ? kLostCopyNs : kWaitLimitNs;
  // After an expired wait, in front of phase `next`'s: the copies of the phase before it and of its own are waited for, once.
  auto land = [&](int next) {
    const int late = (next - 1) & 1;
    await_copies(arrived, 2, late, (x_parity >> late & 1) ^ 1, 1, a.status, kStatusTileTimeout, limit);
    if (next < phases) await_copies(arrived, 2, next & 1, x_parity >> (next & 1) & 1, 1, a.status, kStatusTileTimeout, limit);
    *abort_flag = 2;
  };
  auto load_x = [&](int phase) {                            // one copy per row, by the first warp; and zeros behind the end of k
    if (phase >= phases) return;
    if (warp == 0 && *abort_flag) {                         // nothing is sent for any more, the last barrier may never complete
      if (lane == 0 && *abort_flag == 1) land(phase - 1);
      return;
    }
    uint8_t* to = x_buffer + (phase & 1) * (a.m * x_pitch);
    const int begin = phase * phase_steps * 128, end = min(a.k, begin + phase_steps * 128), bytes = (end - begin) * 2;
    if (warp == 0 && !(kTiming && a.lose && blockIdx.x == 0 && phase == 0)) {
      if (lane == 0) mbar_arrive_expect_tx(&arrived[phase & 1], a.m * bytes);
      __syncwarp();
      if (lane < a.m)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to + lane * x_pitch)),
                     "l"(static_cast<const uint16_t*>(a.x) + (lane * static_cast<int64_t>(a.k) + begin)), "r"(bytes), "r"(smem_u32(&arrived[phase & 1])) : "memory");
    }
    const int missing = ((end + 127) / 128 * 128 - end) * 2 / 16;        // pieces of 16 bytes; the next barrier comes before their use
    for (int i = threadIdx.x; i < a.m * missing; i += kWarps * 32)
      *reinterpret_cast<uint4*>(to + i / missing * x_pitch + bytes + i % missing * 16) = make_uint4(0, 0, 0, 0);
  };
  uint32_t row_offset[kCols];                               // of this lane's rows of x; behind the last one any will do
#pragma unroll
  for (int c = 0; c < kCols; ++c) row_offset[c] = min(c * 8 + g, a.m - 1) * x_pitch;

  for (int chunk = first; chunk < last; chunk += kWarps * kRows) {
    // Blocks of two tiles, and one of one where the last 16 rows or fewer are left: it costs half, and gets the warps that
    // the others leave.  A warp without a share only helps with x.
    const int rows = min(last - chunk, kWarps * kRows), tiles = (rows + 15) / 16, whole = tiles / 2;
    const int whole_shares = 2 * kWarps / tiles, half_shares = tiles % 2 ? max(1, min(whole_shares, kWarps - whole * whole_shares)) : 0;
    const bool half = warp >= whole * whole_shares;
    const int shares = half ? half_shares : whole_shares, block = half ? whole : warp % whole;
    const int share = half ? warp - whole * whole_shares : warp / whole, row = chunk + block * kRows;
    const bool works = share < shares;

    const uint8_t* w_base = a.w + static_cast<int64_t>(row + g) * row_bytes + t * 16;
    const int left = chunk + rows - row - g;
    const uint32_t to = Kept(smem_u32(ring) + WeightPiece(g, t));
    int load_step = works ? share : steps, load_stage = 0;
    auto load = [&] {
      if (load_step < steps) {
        const bool there = load_step * 64 + t * 16 < row_bytes;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          CopyAsync16If(there && 8 * i < left, to + load_stage * 2048 + i * 512, w_base + (static_cast<int64_t>(8 * i) * row_bytes + load_step * 64));
        load_step += shares;
        load_stage = load_stage + 1 == kStages ? 0 : load_stage + 1;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint32_t scale[2][2], zero[2][2], row_at[2][2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) row_at[r][h] = static_cast<uint32_t>(min(block * kRows + r * 16 + h * 8 + g, rows - 1)) * a.groups;
    const uint8_t* scale_base = static_cast<const uint8_t*>(a.scale) + static_cast<int64_t>(chunk) * a.groups * (a.scale_dtype == kF32 ? 4 : 2);
    const uint8_t* zero_base = a.zero + static_cast<int64_t>(chunk) * a.groups;
    auto load_numbers = [&](int step, auto tiles_of_unit) {
      const uint32_t group = kGroup == 128 ? (a.group_shift >= 0 ? step >> a.group_shift : step / a.blocks_per_group) : step * kPerStep + t % kPerStep;
      const bool there = kGroup == 128 || group < a.groups;
#pragma unroll
      for (int r = 0; r < decltype(tiles_of_unit)::value; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t at = row_at[r][h] + (there ? group : 0);
          scale[r][h] = LoadBits<0>(scale_base, at, a.scale_dtype);
          if (!there) scale[r][h] = 0;
          zero[r][h] = 8;
          if (!is_signed) zero[r][h] = zero_base[at] & 15u;
        }
    };
    fence_proxy_async_smem();                               // what this thread wrote where x goes: zeros, sums
    __syncthreads();                                        // the sums of the chunk before have been read
    load_x(0);
    for (int s = 0; s < kStages - 1; ++s) load();
    int step = share, stage = 0;
    if (works && step < steps) load_numbers(step, Two());
    float acc[2][kCols][4] = {};

#pragma unroll 1
    for (int phase = 0; phase < phases; ++phase) {
      __syncthreads();                                      // the phase before has been read by all warps
      load_x(phase + 1);
      (void)mbar_wait(&arrived[phase & 1], (x_parity >> (phase & 1)) & 1, abort_flag, a.status, kStatusTileTimeout, limit);
      x_parity ^= 1u << (phase & 1);
      const uint32_t x_at = smem_u32(x_buffer) + (phase & 1) * (a.m * x_pitch) + t * (kGroup == 128 ? 64 : kGroup == 64 ? 32 : 16);
      const int end = min(steps, (phase + 1) * phase_steps);
      auto run = [&](auto tiles_of_unit) {
        constexpr int kOfUnit = decltype(tiles_of_unit)::value;
#pragma unroll 1
        for (; step < end; step += shares) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
          __syncwarp();
          load();
          const uint32_t weights = smem_u32(ring) + stage * 2048, inputs = x_at + (step - phase * phase_steps) * 256;
          stage = stage + 1 == kStages ? 0 : stage + 1;
#pragma unroll
          for (int group = 0; group < kPerStep; ++group) {
            const int holder = (lane & ~3) | group;
            Offset<T> decoder[2][2];
#pragma unroll
            for (int r = 0; r < kOfUnit; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h) decoder[r][h].Set(kGroup == 128 || is_signed ? zero[r][h] : __shfl_sync(0xffffffffu, zero[r][h], holder));
            float part[2][kCols][4] = {};
            uint32_t w[2][2][kWords];
#pragma unroll
            for (int r = 0; r < kOfUnit; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int at = r * 16 + h * 8 + g;
                if constexpr (kGroup == 128) {
                  const uint4 v = LoadShared16(weights + WeightPiece(at, t));
                  w[r][h][0] = v.x, w[r][h][1] = v.y, w[r][h][2] = v.z, w[r][h][3] = v.w;
                } else if constexpr (kGroup == 64) {
                  const uint2 v = LoadShared8(weights + WeightPiece(at, group * 2 + t / 2) + t % 2 * 8);
                  w[r][h][0] = v.x, w[r][h][1] = v.y;
                } else {
                  w[r][h][0] = LoadShared4(weights + WeightPiece(at, group) + t * 4);
                }
              }
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
              uint32_t low[2][4], high[2][4];
#pragma unroll
              for (int r = 0; r < kOfUnit; ++r) {
                decoder[r][0].Decode8(w[r][0][i], flip, low[r]);
                decoder[r][1].Decode8(w[r][1][i], flip, high[r]);
              }
#pragma unroll
              for (int c = 0; c < kCols; ++c) {
                const uint4 b = Paired(LoadShared16(inputs + row_offset[c] + (group * (kGroup / 8) + i) * 16));
#pragma unroll
                for (int r = 0; r < kOfUnit; ++r) {
                  Mma<T>(part[r][c], low[r][0], high[r][0], low[r][1], high[r][1], b.x, b.y);
                  Mma<T>(part[r][c], low[r][2], high[r][2], low[r][3], high[r][3], b.z, b.w);
                }
              }
            }
#pragma unroll
            for (int r = 0; r < kOfUnit; ++r) {
              float s0 = ValueOf<0>(scale[r][0], a.scale_dtype), s1 = ValueOf<0>(scale[r][1], a.scale_dtype);
              if (kGroup < 128) s0 = __shfl_sync(0xffffffffu, s0, holder), s1 = __shfl_sync(0xffffffffu, s1, holder);
#pragma unroll
              for (int c = 0; c < kCols; ++c) {
                acc[r][c][0] = fmaf(part[r][c][0], s0, acc[r][c][0]), acc[r][c][1] = fmaf(part[r][c][1], s0, acc[r][c][1]);
                acc[r][c][2] = fmaf(part[r][c][2], s1, acc[r][c][2]), acc[r][c][3] = fmaf(part[r][c][3], s1, acc[r][c][3]);
              }
            }
          }
          if (step + shares < steps) load_numbers(step + shares, tiles_of_unit);
        }
      };
      if (works && half) run(One());
      else if (works) run(Two());
    }
    __syncthreads();                                        // x has been read: its place takes the sums
    if (*abort_flag) {                                      // a wait expired: no result
      if (threadIdx.x == 0 && *abort_flag == 1) land(phases);
      asm volatile("cp.async.wait_all;" ::: "memory");
      return;
    }
    if (works) {
      float* mine = sums + warp * a.m * kSumStride;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (c * 8 + 2 * t + e < a.m) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              mine[(c * 8 + 2 * t + e) * kSumStride + r * 16 + g] = acc[r][c][e];
              mine[(c * 8 + 2 * t + e) * kSumStride + r * 16 + 8 + g] = acc[r][c][e + 2];
            }
          }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < rows * a.m; i += kWarps * 32) {
      const int x_row = i / rows, in_chunk = i - x_row * rows, at = chunk + in_chunk;
      const int of_block = in_chunk / kRows;
      const bool in_whole = of_block < whole;
      const float* part = sums + ((in_whole ? of_block : whole * whole_shares) * a.m + x_row) * kSumStride + in_chunk % kRows;
      const int parts = in_whole ? whole_shares : half_shares, apart = (in_whole ? whole : 1) * a.m * kSumStride;
      float y = 0.0f;
#pragma unroll 1
      for (int w = 0; w < parts; ++w) y += part[w * apart];
      if (a.bias != nullptr) y += ValueOf<0>(LoadBits<0>(a.bias, at, a.bias_dtype), a.bias_dtype);
      const int64_t place = static_cast<int64_t>(x_row) * a.n + at;
      if (a.d_dtype == kBF16) static_cast<__nv_bfloat16*>(a.d)[place] = __float2bfloat16_rn(y);
      else if (a.d_dtype == kF16) static_cast<__half*>(a.d)[place] = __float2half_rn(y);
      else static_cast<float*>(a.d)[place] = y;
    }
  }
}

struct Variant {
  void (*kernel)(W4Args);
  int64_t (*bytes)(int64_t m, int64_t steps);
  int64_t (*per_round)(int64_t m, int64_t steps);
  int warps, registers;
};
constexpr int64_t kSmemPerSm = 228 * 1024, kSmemPerCta = 227 * 1024, kSmemReserved = 1024;
template <int kGroup, typename S>
Variant MakeWide() {
  return {w4_dot_wide_kernel<kGroup, S>, S::Bytes, S::Phase, S::kWarps, 0};
}
struct Variants {
  Variant resident[3][3][2];                     // group, type of the scales, two's complement
  Variant wide[2][3][3];                         // type of x, group, for 8, 16 and 32 rows of x
  template <int kGroup, int kScale, bool kSigned>
  void Fill(Variant& to) {
    to = {w4_dot_kernel<kGroup, kScale, kSigned>, Resident::Bytes, Resident::PerRound, Resident::kWarps, 0};
  }
  template <int kGroup, typename T>
  void FillWide(Variant* to) {
    to[0] = MakeWide<kGroup, WideShape<T, 1>>();
    to[1] = MakeWide<kGroup, WideShape<T, 2>>();
    to[2] = MakeWide<kGroup, WideShape<T, 4>>();
  }
  template <int kGroup>
  void FillGroup(int at) {
    Fill<kGroup, kF16, false>(resident[at][0][0]);
    Fill<kGroup, kF16, true>(resident[at][0][1]);
    Fill<kGroup, kBF16, false>(resident[at][1][0]);
    Fill<kGroup, kBF16, true>(resident[at][1][1]);
    Fill<kGroup, kF32, false>(resident[at][2][0]);
    Fill<kGroup, kF32, true>(resident[at][2][1]);
    FillWide<kGroup, __half>(wide[0][at]);
    FillWide<kGroup, __nv_bfloat16>(wide[1][at]);
  }
  Variants() {
    FillGroup<32>(0);
    FillGroup<64>(1);
    FillGroup<128>(2);
  }
};
Variants& TheVariants() {
  static Variants v;
  return v;
}

}  // namespace

Status InitW4Kernels() {
  static_assert(std::is_standard_layout_v<Variants>);
  Variant* v = reinterpret_cast<Variant*>(&TheVariants());
  constexpr size_t kCount = sizeof(Variants) / sizeof(Variant);
  int registers[kCount];
  for (size_t i = 0; i < kCount; ++i) {
    cudaFuncAttributes attr{};
    cudaError_t e = cudaFuncSetAttribute(v[i].kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerCta);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, v[i].kernel);
    if (e != cudaSuccess) return Status::Error(kInternal, std::string("w4_dot_kernel set-up: ") + cudaGetErrorString(e));
    registers[i] = attr.numRegs;
  }
  static std::once_flag once;                               // the same on every device; another one may be launching already
  std::call_once(once, [&] {
    for (size_t i = 0; i < kCount; ++i) v[i].registers = registers[i];
  });
  return Status::Ok();
}

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
  if (a.m > 32) {                                           // half of the rows at a time: the sums of 64 do not fit the registers
    B200SD_DotW4 half = a;
    LaunchStats first, second;
    half.m = a.m / 2;
    Status st = LaunchDotW4(half, stream, &first);
    if (!st.ok()) return st;
    half.x = static_cast<const uint16_t*>(a.x) + half.m * a.k;
    half.d = static_cast<uint8_t*>(a.d) + half.m * a.n * (a.d_dtype == kF32 ? 4 : 2);
    half.m = a.m - half.m;
    st = LaunchDotW4(half, stream, &second);
    stats->launches = first.launches + second.launches;
    return st;
  }
  const int64_t steps = (a.k + 127) / 128;
  const int group_at = a.group == 32 ? 0 : a.group == 64 ? 1 : 2, scale_at = a.scale_dtype == kF16 ? 0 : a.scale_dtype == kBF16 ? 1 : 2;
  const Variant& resident = TheVariants().resident[group_at][scale_at][a.weight_type == kS4];
  // With x resident every CTA pairs all of it first, and has fewer instructions for the weights afterwards.  Which of the two
  // is faster, resident against wide in us, calls one after the other in a graph:
  //   groups of 32: m 1, 256 x 512 2.9 and 3.2, 4096 x 4096 6.9 and 8.4, 28672 x 8192 39.3 and 55.0; m 2 the same 3.0 and
  //     3.2, 7.7 and 8.4, 41.9 and 55.0, but 65536 x 1024 20.8 and 18.3, 16384 x 1024 7.3 and 7.2: a short k does not pay for
  //     the second row.
  //   longer groups, two's complement (groups of 128): m 1, 8192 x 8192 15.6 and 13.5, 16384 x 8192 22.0 and 22.0, 36864 x 4608
  //     25.5 and 25.1, 24576 x 8192 29.9 and 35.0, 28672 x 8192 33.5 and 38.6, 57344 x 8192 57.8 and 73.5; m 2, 16384 x 8192 24.4
  //     and 22.0, 24576 x 8192 33.0 and 35.0, 57344 x 8192 61.7 and 73.5, 131072 x 2048 45.5 and 41.7.
  //   zero points, which cost this kernel more: m 1, 28672 x 6144 31.2 and 31.2, 24576 x 8192 35.7 and 37.0, 57344 x 8192 70.0 and
  //     76.5; m 2, 24576 x 8192 38.8 and 37.1, 131072 x 4096 80.8 and 74.2.
  // So groups of 32 have it unless k is short for two rows, and of the others many weights, about 200 million, with k long
  // enough for the warps of a CTA, two rows with zero points never.
  const bool pays = a.group == 32 ? a.m == 1 || a.k >= 2048
                                  : a.n * a.k >= 200'000'000 && a.k >= 4096 && (a.m == 1 || a.weight_type == kS4);
  const bool is_resident = a.m <= Resident::kMost && pays && resident.bytes(a.m, steps) <= kSmemPerCta;
  const Variant& v = is_resident ? resident : TheVariants().wide[a.x_dtype == kBF16][group_at][a.m <= 8 ? 0 : a.m <= 16 ? 1 : 2];
  const int bytes = static_cast<int>(v.bytes(a.m, steps)), threads = v.warps * 32;
  const int by_registers = 65536 / (threads * ((v.registers + 7) / 8 * 8)), by_smem = static_cast<int>(kSmemPerSm / (bytes + kSmemReserved));
  const int per_sm = std::max(1, std::min({by_registers, by_smem, 2048 / threads}));
  // One CTA per resident slot, each with its even share of the rows, but no more CTAs than tiles of 8 rows.
  const int64_t ctas = std::min<int64_t>(static_cast<int64_t>(DeviceSmCount()) * per_sm, (a.n + 7) / 8);
  const int64_t blocks_per_group = a.group >= 128 ? a.group / 128 : 1;
  int group_shift = 0;
  while ((int64_t{1} << group_shift) < blocks_per_group) ++group_shift;
  if ((int64_t{1} << group_shift) != blocks_per_group) group_shift = -1;
  const W4Args args{a.x, static_cast<const uint8_t*>(a.w), a.scale, static_cast<const uint8_t*>(a.zero), a.epilogue == B200SD_EPILOGUE_BIAS ? a.bias : nullptr, a.d,
                    static_cast<int32_t>(a.m), static_cast<int32_t>(a.n), static_cast<int32_t>(a.k), static_cast<int32_t>(a.k / a.group),
                    group_shift, static_cast<int32_t>(blocks_per_group),
                    static_cast<int32_t>(a.n / ctas), static_cast<int32_t>(a.n % ctas), static_cast<int32_t>(steps), static_cast<int32_t>(v.per_round(a.m, steps)), StatusWordPtr(),
                    0xffffffffu / static_cast<uint32_t>(steps * 16) + 1, a.x_dtype == kBF16, a.scale_dtype, a.bias_dtype, a.d_dtype, a.weight_type == kS4, LoseCopy()};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;     // see griddep_wait() in the kernel
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, v.kernel, args);
  if (e != cudaSuccess) return Status::Error(kInternal, std::string("w4_dot_kernel launch: ") + cudaGetErrorString(e));
  stats->launches = 1;
  return Status::Ok();
}

}  // namespace b200sd
