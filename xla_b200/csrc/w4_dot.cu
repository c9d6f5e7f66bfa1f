// Dots of a few rows with 4-bit weights and a scale for each group along k.
//
// Bound by reading the weights once (n * k / 2 bytes); at the copy rate an SM has about 44 clocks for a KiB of them, 176
// instruction slots for 2048 weights, so the other half of the work is decoding cheaply.
//
// Products run on mma.m16n8k16 with 16 weight rows on the large side and 8 rows of x on the other: A is the weights as
// they lie in memory, B is x.  The order along k inside a product is free, so a lane feeds two products from one
// 32-bit word of 8 weights: the pairs (i, i + 4) of its nibbles are one mask away from being f16 or bf16 numbers with a
// constant offset (1024 + w, 128 + w), and one subtraction takes the offset and the zero point away -- exactly, the
// operands are the integers w - z.  x is paired the same way.  A lane's word, half or whole 16-byte piece is chosen so
// that one product never mixes two groups; a group's f32 sum is multiplied by its scale in f32 and added up.
//
// A CTA owns n / CTAs consecutive rows, whole rows of bytes with none read twice or by two CTAs whatever n is; its warps
// split k among them in steps of 128 (and, where k is short, also the rows), each with its own cp.async ring for its
// weights and the matching part of x, and add their sums through shared memory once per block of rows, in a fixed order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
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
  int32_t k_warps;                              // warps that share a block of rows
  int32_t scale_dtype, bias_dtype, d_dtype, is_signed;
};

__device__ __forceinline__ float ScaleValue(uint32_t raw, int32_t dtype) {
  if (dtype == kBF16) return __uint_as_float(raw << 16);
  if (dtype == kF16) return __half2float(__ushort_as_half(static_cast<unsigned short>(raw)));
  return __uint_as_float(raw);
}
__device__ __forceinline__ uint32_t LoadRaw(const void* p, int64_t i, int32_t dtype) {
  if (dtype == kF32) return __ldg(static_cast<const uint32_t*>(p) + i);
  return __ldg(static_cast<const unsigned short*>(p) + i);
}
__device__ __forceinline__ void CopyAsync16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// What turns masked nibbles into operands: offset + zero point of one weight row and group, for both halves.
template <typename T> struct Offsets;
template <> struct Offsets<__half> {
  __half2 low, high;
  __device__ explicit Offsets(int z) {
    low = __half2half2(__int2half_rn(-1024 - z));
    high = __half2half2(__int2half_rn(-64 - z));
  }
};
template <> struct Offsets<__nv_bfloat16> {
  __nv_bfloat162 low;
  __device__ explicit Offsets(int z) { low = __bfloat162bfloat162(__int2bfloat16_rn(-128 - z)); }
};

// The pairs (0, 4), (1, 5), (2, 6), (3, 7) of a word's nibbles, w - z each; `flip` is 8 for two's complement.
__device__ __forceinline__ void Decode8(uint32_t w, uint32_t flip, const Offsets<__half>& o, uint32_t (&v)[4]) {
  const __half2 sixteenth = __half2half2(__ushort_as_half(0x2c00));
  const uint32_t low = 0x64006400u | flip, high = 0x64006400u | flip << 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t shifted = w >> (8 * i);
    const uint32_t a = (shifted & 0x000f000fu) ^ low, b = (shifted & 0x00f000f0u) ^ high;       // 1024 + n, 1024 + 16 n
    const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&a), o.low);
    const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&b), sixteenth, o.high);
    v[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
    v[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
  }
}
__device__ __forceinline__ void Decode8(uint32_t w, uint32_t flip, const Offsets<__nv_bfloat16>& o, uint32_t (&v)[4]) {
  const uint32_t low = 0x43004300u | flip;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = ((w >> (4 * i)) & 0x000f000fu) ^ low;                                    // 128 + n
    const __nv_bfloat162 x = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&a), o.low);
    v[i] = *reinterpret_cast<const uint32_t*>(&x);
  }
}

template <typename T>
__device__ __forceinline__ void Mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// kGroup: 32, 64 or 128 (which stands for its multiples too); kTiles: weight row tiles of 16 of a warp; kCols: tiles of 8
// rows of x.
template <int kTiles_, int kCols_, int kWarps_, int kStages_>
struct Shape {
  static constexpr int kTiles = kTiles_, kCols = kCols_, kWarps = kWarps_, kStages = kStages_;
  static constexpr int kRows = 16 * kTiles;                 // weight rows of a warp's block
  static constexpr int kStride = kRows + 4;                 // floats between two rows of x in the sums
  static constexpr int kSums = kWarps * 8 * kCols * kStride * 4;
  static int Bytes(int m) { return kSums + kWarps * kStages * (kTiles * 1024 + m * 256); }
};

// Where 16-byte piece `c` of weight row `r` (64 bytes of a step) and piece `c` of row `r` of x (256 bytes) lie: so that the
// reads below have no bank conflicts.
__device__ __forceinline__ int WeightPiece(int r, int c) { return r * 64 + (c ^ ((r & 2) | ((r >> 2) & 1))) * 16; }
template <int kGroup>
__device__ __forceinline__ int InputPiece(int r, int c) {
  const int at = kGroup == 128 ? (c % 4) * 4 + c / 4 : kGroup == 64 ? (c & 8) + (c % 2) * 4 + c % 8 / 2 : c;
  return r * 256 + (at ^ ((r & 1) << 2)) * 16;
}

template <typename T, int kGroup, typename S>
__global__ void __launch_bounds__(S::kWarps * 32) w4_dot_kernel(const W4Args a) {
  constexpr int kPerStep = 128 / kGroup;                    // groups of a step
  constexpr int kWords = kGroup / 32;                       // words of a lane in a group
  extern __shared__ __align__(128) uint8_t smem[];
  if (threadIdx.x == 0) griddep_launch_dependents();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int wk = warp % a.k_warps, wn = warp / a.k_warps, row_step = S::kRows * (S::kWarps / a.k_warps);
  const int first = static_cast<int>(static_cast<int64_t>(blockIdx.x) * a.n / gridDim.x);
  const int last = static_cast<int>(static_cast<int64_t>(blockIdx.x + 1) * a.n / gridDim.x);
  const int steps = (a.k + 127) / 128, row_bytes = a.k / 2;
  const int stage_bytes = S::kTiles * 1024 + a.m * 256;
  float* sums = reinterpret_cast<float*>(smem);
  uint8_t* ring = smem + S::kSums + warp * S::kStages * stage_bytes;
  const uint32_t flip = a.is_signed ? 0x00080008u : 0u;

  int load_row = first + wn * S::kRows, load_step = wk;
  auto load = [&](int stage) {
    if (load_row < last && load_step < steps) {
      const uint32_t dst = smem_u32(ring + stage * stage_bytes);
#pragma unroll
      for (int i = 0; i < 2 * S::kTiles; ++i) {
        const int piece = i * 32 + lane, r = piece / 4, c = piece % 4, at = load_step * 64 + c * 16;
        const bool in = load_row + r < last && at < row_bytes;
        CopyAsync16(dst + WeightPiece(r, c), in ? a.w + static_cast<int64_t>(load_row + r) * row_bytes + at : a.w, in ? 16 : 0);
      }
      for (int piece = lane; piece < a.m * 16; piece += 32) {
        const int r = piece / 16, c = piece % 16, at = load_step * 128 + c * 8;
        const bool in = at < a.k;
        CopyAsync16(dst + S::kTiles * 1024 + InputPiece<kGroup>(r, c), in ? static_cast<const T*>(a.x) + static_cast<int64_t>(r) * a.k + at : a.x, in ? 16 : 0);
      }
      load_step += a.k_warps;
      if (load_step >= steps) {
        load_step = wk;
        load_row += row_step;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // Scales (as they are stored) and zero points of a step for this lane's rows; with several groups in a step the four lanes
  // of a row hold one each.
  auto load_scales = [&](int row, int step, uint32_t (&scale)[S::kTiles][2], int (&zero)[S::kTiles][2]) {
    const int group = kGroup == 128 ? (a.group_shift >= 0 ? step >> a.group_shift : step / a.blocks_per_group) : step * kPerStep + t;
#pragma unroll
    for (int r = 0; r < S::kTiles; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = row + r * 16 + h * 8 + g;
        scale[r][h] = 0;
        zero[r][h] = 8;
        if (at < last && step < steps && group < a.groups && (kGroup == 128 || t < kPerStep)) {
          const int64_t i = static_cast<int64_t>(at) * a.groups + group;
          scale[r][h] = LoadRaw(a.scale, i, a.scale_dtype);
          if (!a.is_signed) zero[r][h] = __ldg(a.zero + i) & 15;
        }
      }
  };

  griddep_wait();
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) load(s);
  uint32_t next_scale[S::kTiles][2];
  int next_zero[S::kTiles][2];
  load_scales(first + wn * S::kRows, wk, next_scale, next_zero);

  int stage = 0;
  for (int block = first; block < last; block += row_step) {
    const int row = block + wn * S::kRows;
    float acc[S::kTiles][S::kCols][4] = {};
    if (row < last) {
      for (int step = wk; step < steps; step += a.k_warps) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
        __syncwarp();
        load(stage == 0 ? S::kStages - 1 : stage - 1);
        const uint8_t* weights = ring + stage * stage_bytes;
        const uint8_t* inputs = weights + S::kTiles * 1024;
        stage = stage + 1 == S::kStages ? 0 : stage + 1;
        uint32_t scale[S::kTiles][2];
        int zero[S::kTiles][2];
#pragma unroll
        for (int r = 0; r < S::kTiles; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) scale[r][h] = next_scale[r][h], zero[r][h] = next_zero[r][h];
        const bool more = step + a.k_warps < steps;
        load_scales(more ? row : row + row_step, more ? step + a.k_warps : wk, next_scale, next_zero);

#pragma unroll
        for (int group = 0; group < kPerStep; ++group) {
          // The words of this group, of rows g and g + 8 of each tile.
          uint32_t w[S::kTiles][2][kWords];
#pragma unroll
          for (int r = 0; r < S::kTiles; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int at = r * 16 + h * 8 + g;
              if constexpr (kGroup == 128) {
                const uint4 v = *reinterpret_cast<const uint4*>(weights + WeightPiece(at, t));
                w[r][h][0] = v.x, w[r][h][1] = v.y, w[r][h][2] = v.z, w[r][h][3] = v.w;
              } else if constexpr (kGroup == 64) {
                const uint2 v = *reinterpret_cast<const uint2*>(weights + WeightPiece(at, group * 2 + t / 2) + t % 2 * 8);
                w[r][h][0] = v.x, w[r][h][1] = v.y;
              } else {
                w[r][h][0] = *reinterpret_cast<const uint32_t*>(weights + WeightPiece(at, group) + t * 4);
              }
            }
          float part[S::kTiles][S::kCols][4] = {};
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            uint32_t b[S::kCols][4];
#pragma unroll
            for (int c = 0; c < S::kCols; ++c) {
              const int piece = kGroup == 128 ? t * 4 + i : kGroup == 64 ? group * 8 + t * 2 + i : group * 4 + t;
              uint4 v = {};
              if (c * 8 + g < a.m) v = *reinterpret_cast<const uint4*>(inputs + InputPiece<kGroup>(c * 8 + g, piece));
              b[c][0] = __byte_perm(v.x, v.z, 0x5410), b[c][1] = __byte_perm(v.x, v.z, 0x7632);
              b[c][2] = __byte_perm(v.y, v.w, 0x5410), b[c][3] = __byte_perm(v.y, v.w, 0x7632);
            }
#pragma unroll
            for (int r = 0; r < S::kTiles; ++r) {
              uint32_t low[4], high[4];
              const int from = kGroup == 128 ? lane : (lane & ~3) | group;
              const int z0 = kGroup == 128 ? zero[r][0] : __shfl_sync(0xffffffffu, zero[r][0], from);
              const int z1 = kGroup == 128 ? zero[r][1] : __shfl_sync(0xffffffffu, zero[r][1], from);
              Decode8(w[r][0][i], flip, Offsets<T>(z0), low);
              Decode8(w[r][1][i], flip, Offsets<T>(z1), high);
#pragma unroll
              for (int c = 0; c < S::kCols; ++c) {
                Mma<T>(part[r][c], low[0], high[0], low[1], high[1], b[c][0], b[c][1]);
                Mma<T>(part[r][c], low[2], high[2], low[3], high[3], b[c][2], b[c][3]);
              }
            }
          }
#pragma unroll
          for (int r = 0; r < S::kTiles; ++r) {
            const int from = (lane & ~3) | group;
            const float s0 = ScaleValue(kGroup == 128 ? scale[r][0] : __shfl_sync(0xffffffffu, scale[r][0], from), a.scale_dtype);
            const float s1 = ScaleValue(kGroup == 128 ? scale[r][1] : __shfl_sync(0xffffffffu, scale[r][1], from), a.scale_dtype);
#pragma unroll
            for (int c = 0; c < S::kCols; ++c) {
              acc[r][c][0] = fmaf(part[r][c][0], s0, acc[r][c][0]);
              acc[r][c][1] = fmaf(part[r][c][1], s0, acc[r][c][1]);
              acc[r][c][2] = fmaf(part[r][c][2], s1, acc[r][c][2]);
              acc[r][c][3] = fmaf(part[r][c][3], s1, acc[r][c][3]);
            }
          }
        }
      }
    }
    // The warps' sums of this block of rows, added in the order of the warps.
    __syncthreads();                                        // those of the block before have been read
    float* mine = sums + warp * 8 * S::kCols * S::kStride;
#pragma unroll
    for (int r = 0; r < S::kTiles; ++r)
#pragma unroll
      for (int c = 0; c < S::kCols; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[(c * 8 + 2 * t + e % 2) * S::kStride + r * 16 + e / 2 * 8 + g] = acc[r][c][e];
    __syncthreads();
    for (int i = threadIdx.x; i < a.m * row_step; i += S::kWarps * 32) {
      const int x_row = i / row_step, in_block = i % row_step, at = block + in_block;
      if (at >= last) continue;
      const float* from = sums + (in_block / S::kRows * a.k_warps * 8 * S::kCols + x_row) * S::kStride + in_block % S::kRows;
      float y = 0.0f;
      for (int w = 0; w < a.k_warps; ++w) y += from[w * 8 * S::kCols * S::kStride];
      if (a.bias != nullptr) y += ScaleValue(LoadRaw(a.bias, at, a.bias_dtype), a.bias_dtype);
      const int64_t to = static_cast<int64_t>(x_row) * a.n + at;
      if (a.d_dtype == kBF16) static_cast<__nv_bfloat16*>(a.d)[to] = __float2bfloat16_rn(y);
      else if (a.d_dtype == kF16) static_cast<__half*>(a.d)[to] = __float2half_rn(y);
      else static_cast<float*>(a.d)[to] = y;
    }
  }
}

// Per tile count of x: how many weight rows share a piece of x, the warps, and the stages of a ring.  A CTA reads x once
// per block of rows, m / (4 * tiles) bytes of it for a byte of weights.
using Shape8 = Shape<2, 1, 8, 4>;
using Shape16 = Shape<4, 2, 4, 4>;
using Shape32 = Shape<4, 4, 4, 4>;
using Shape64 = Shape<2, 8, 4, 2>;

struct Variant {
  void (*kernel)(W4Args);
  int rows, warps, registers;
};
constexpr int kShapes = 4;
template <typename T, int kGroup>
void Fill(Variant* v) {
  v[0] = {w4_dot_kernel<T, kGroup, Shape8>, Shape8::kRows, Shape8::kWarps, 0};
  v[1] = {w4_dot_kernel<T, kGroup, Shape16>, Shape16::kRows, Shape16::kWarps, 0};
  v[2] = {w4_dot_kernel<T, kGroup, Shape32>, Shape32::kRows, Shape32::kWarps, 0};
  v[3] = {w4_dot_kernel<T, kGroup, Shape64>, Shape64::kRows, Shape64::kWarps, 0};
}
int SmemBytes(int shape, int m) {
  switch (shape) {
    case 0: return Shape8::Bytes(m);
    case 1: return Shape16::Bytes(m);
    case 2: return Shape32::Bytes(m);
    default: return Shape64::Bytes(m);
  }
}
struct Variants {
  Variant v[2][3][kShapes];
  Variants() {
    Fill<__half, 32>(v[0][0]);
    Fill<__half, 64>(v[0][1]);
    Fill<__half, 128>(v[0][2]);
    Fill<__nv_bfloat16, 32>(v[1][0]);
    Fill<__nv_bfloat16, 64>(v[1][1]);
    Fill<__nv_bfloat16, 128>(v[1][2]);
  }
};
Variants& TheVariants() {
  static Variants v;
  return v;
}
constexpr int kSmemPerSm = 227 * 1024;

}  // namespace

Status InitW4Kernels() {
  for (auto& types : TheVariants().v)
    for (auto& groups : types)
      for (int s = 0; s < kShapes; ++s) {
        cudaFuncAttributes attr{};
        cudaError_t e = cudaFuncSetAttribute(groups[s].kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SmemBytes(s, 8 << s));
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, groups[s].kernel);
        if (e != cudaSuccess) return Status::Error(kInternal, std::string("w4_dot_kernel set-up: ") + cudaGetErrorString(e));
        groups[s].registers = attr.numRegs;
      }
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
  const int shape = a.m <= 8 ? 0 : a.m <= 16 ? 1 : a.m <= 32 ? 2 : 3;
  const Variant& v = TheVariants().v[a.x_dtype == kBF16][a.group == 32 ? 0 : a.group == 64 ? 1 : 2][shape];
  const int bytes = SmemBytes(shape, static_cast<int>(a.m)), threads = v.warps * 32;
  const int by_registers = 65536 / (threads * ((v.registers + 7) / 8 * 8)), by_smem = kSmemPerSm / (bytes + 1024);
  const int per_sm = std::max(1, std::min({by_registers, by_smem, 2048 / threads}));
  // One CTA per resident slot, each with its even share of the rows, but no more CTAs than tiles of 8 rows.
  const int64_t ctas = std::min<int64_t>(static_cast<int64_t>(DeviceSmCount()) * per_sm, (a.n + 7) / 8);
  // All warps split k where that leaves each at least 8 steps of it; otherwise some take other rows, if the CTA has them.
  const int64_t steps = (a.k + 127) / 128, rows = (a.n + ctas - 1) / ctas;
  int k_warps = v.warps;
  while (k_warps > 1 && steps / k_warps < 8 && rows >= static_cast<int64_t>(v.rows) * (v.warps / k_warps) * 2) k_warps /= 2;
  const int64_t blocks_per_group = a.group >= 128 ? a.group / 128 : 1;
  int group_shift = 0;
  while ((int64_t{1} << group_shift) < blocks_per_group) ++group_shift;
  if ((int64_t{1} << group_shift) != blocks_per_group) group_shift = -1;
  const W4Args args{a.x, static_cast<const uint8_t*>(a.w), a.scale, static_cast<const uint8_t*>(a.zero), a.epilogue == B200SD_EPILOGUE_BIAS ? a.bias : nullptr, a.d,
                    static_cast<int32_t>(a.m), static_cast<int32_t>(a.n), static_cast<int32_t>(a.k), static_cast<int32_t>(a.k / a.group),
                    group_shift, static_cast<int32_t>(blocks_per_group), k_warps, a.scale_dtype, a.bias_dtype, a.d_dtype, a.weight_type == kS4};
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
