// 4-bit microscaled values: quantisation, dequantisation, and products on the block-scaled tensor cores of sm_100a.
//
// 32 neighbouring values of a row share a power of two, 2^e with e = floor(log2(largest magnitude)) - 2 (at least -127): the largest magnitude
// then lies in [4, 8) and becomes 4 or 6 of the element's values 0, 0.5, 1, 1.5, 2, 3, 4, 6. x 2^-e is exact in fp32, so the one rounding is to
// the nearest of those, ties to the even code, above 6 to 6. A block that holds an infinity or a NaN stands for NaNs.
//
// The product multiplies both operands as they are (kind::mxf4): the tensor core takes 64 of k at a time, scales the products of every 32
// by the two powers and adds in fp32.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "purlin/gemm.h"
#include "purlin/gemm_skinny.cuh"
#include "purlin/mx4.h"
#include "purlin/tc_sm100.cuh"
#include "purlin/telemetry.hpp"
#include "purlin/tensor_map.hpp"
#include "purlin/wait_limit.hpp"

using namespace purlin;

namespace {

constexpr int kBlock = 32;                      // values that share a scale
constexpr int kScaleRows = 128, kScaleCols = 128, kScaleBytes = 512;

// ------------------------------------------------------------------------------------------
// quantisation and the way back: bound by memory
// ------------------------------------------------------------------------------------------
// Four lanes have the 32 values of a block (8 each, 16 bytes of bf16 or fp16), a warp 256 columns, and a step of a warp is four of those side by
// side in one row. The scale needs the exponent of the largest magnitude only, a byte, so the four blocks of a lane travel through the
// shuffles in one word, and four more shuffles' worth of bytes become the words of the scales' layout in two. With one shuffle chain per block and
// 64-bit index arithmetic the instructions, not the memory, were the bound. One B200, 8192 x 8192 bf16: 27.3 us, 6.2 TB/s (0.95 of a copy);
// the way back 24.8 us; 14336 x 8192 fp32 78.5 us, 6.8 TB/s; with one chain per block 8192 x 8192 took 104 us there and back.
constexpr int kVec = 8, kWarpCols = 32 * kVec, kQuantThreads = 256, kUnroll = 4, kStepCols = kUnroll * kWarpCols;

// Not through the non-coherent path, and no pointer of these kernels promises it (const, restrict): that path is for memory that nobody writes during a
// kernel's whole life, and these kernels are set up while the one before them may still write what they will read.
PURLIN_D uint4 ldOnce(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <int TYPE> struct Raw { uint4 v[TYPE == PURLIN_MX4_FP32 ? 2 : 1]; };
template <int TYPE> PURLIN_D Raw<TYPE> loadRaw(const unsigned char* p) {
  Raw<TYPE> r;
  r.v[0] = ldOnce(p);
  if constexpr (TYPE == PURLIN_MX4_FP32) r.v[1] = ldOnce(p + 16);
  return r;
}
// The exponent field that the largest magnitude has in fp32: 255 for infinities and NaNs, 0 for zeros (and below 2^-126, which the scale does not tell
// apart). Magnitudes compare as their bit patterns.
template <int TYPE> PURLIN_D uint32_t peakExponent(const Raw<TYPE>& r) {
  if constexpr (TYPE == PURLIN_MX4_FP32) {
    uint32_t m = max(max(r.v[0].x & 0x7fffffffu, r.v[0].y & 0x7fffffffu), max(r.v[0].z & 0x7fffffffu, r.v[0].w & 0x7fffffffu));
    m = max(m, max(max(r.v[1].x & 0x7fffffffu, r.v[1].y & 0x7fffffffu), max(r.v[1].z & 0x7fffffffu, r.v[1].w & 0x7fffffffu)));
    return m >> 23;
  } else {
    const uint32_t m = __vmaxu2(__vmaxu2(r.v[0].x & 0x7fff7fffu, r.v[0].y & 0x7fff7fffu), __vmaxu2(r.v[0].z & 0x7fff7fffu, r.v[0].w & 0x7fff7fffu));
    const uint32_t top = max(m & 0xffffu, m >> 16);
    if constexpr (TYPE == PURLIN_MX4_BF16) return top >> 7;
    else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(top)))) >> 23;
  }
}
template <int TYPE> PURLIN_D void toFloats(const Raw<TYPE>& r, float (&f)[kVec]) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
  if constexpr (TYPE == PURLIN_MX4_FP32) {
    const uint32_t u[4] = {r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = __uint_as_float(w[i]); f[4 + i] = __uint_as_float(u[i]); }
  } else if constexpr (TYPE == PURLIN_MX4_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x; f[2 * i + 1] = v.y;
    }
  }
}

// eight values times a power of two, rounded to the nearest of the format (ties to the even code), the first in the lowest four bits
PURLIN_D uint32_t packCodes(const float (&f)[kVec], float inverse) {
  float2 v[kVec / 2];
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i) v[i] = __fmul2_rn(make_float2(f[2 * i], f[2 * i + 1]), make_float2(inverse, inverse));
  uint32_t codes;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(codes) : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
  return codes;
}

PURLIN_D size_t scaleOffset(int row, int col, int colBlocks) {       // of the scale of this row's block that begins at `col`
  return (size_t(row / kScaleRows) * size_t(colBlocks) + size_t(col / kScaleCols)) * kScaleBytes + size_t(row % 32) * 16 + size_t(row / 32 % 4) * 4 + size_t(col / kBlock % 4);
}

// Rows past the last one (up to the scales' 128) write their zeros.
template <int TYPE>
__global__ void __launch_bounds__(kQuantThreads) quantizeKernel(const unsigned char* x, unsigned char* data, unsigned char* scales, int rows, int cols, uint32_t steps, uint32_t total) {
  tc::gridDependencyWait();
  tc::gridLaunchDependents();
  constexpr int kSize = TYPE == PURLIN_MX4_FP32 ? 4 : 2;
  const int lane = threadIdx.x & 31;
  const uint32_t warps = gridDim.x * (kQuantThreads / 32);
  const int colBlocks = (cols + kScaleCols - 1) / kScaleCols;
  for (uint32_t i = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5); i < total; i += warps) {
    const int row = int(i / steps), col = int(i % steps) * kStepCols + lane * kVec;
    const size_t at = size_t(row) * size_t(cols) + size_t(col);
    Raw<TYPE> raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      raw[u].v[0] = make_uint4(0, 0, 0, 0);
      if constexpr (TYPE == PURLIN_MX4_FP32) raw[u].v[1] = make_uint4(0, 0, 0, 0);
      if (row < rows && col + u * kWarpCols < cols) raw[u] = loadRaw<TYPE>(x + (at + size_t(u * kWarpCols)) * kSize);
    }
    uint32_t peaks = 0;                                       // a byte for each of the four blocks
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) peaks |= peakExponent<TYPE>(raw[u]) << (8 * u);
    peaks = __vmaxu4(peaks, __shfl_xor_sync(0xffffffffu, peaks, 1));
    peaks = __vmaxu4(peaks, __shfl_xor_sync(0xffffffffu, peaks, 2));
    // a scale is the exponent less 2, at least 0, and stays 255
    const uint32_t bad = __vcmpeq4(peaks, 0xffffffffu), scale4 = __vsubus4(peaks, 0x02020202u) | bad;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t scale = scale4 >> (8 * u) & 255u;
      const float inverse = __uint_as_float((254u - scale) << 23);       // (of a scale of 255 not used)
      float f[kVec];
      toFloats<TYPE>(raw[u], f);
      uint32_t codes = packCodes(f, inverse);
      if (scale == 255u) codes = 0;
      if (row < rows && col + u * kWarpCols < cols) *reinterpret_cast<uint32_t*>(data + (at + size_t(u * kWarpCols)) / 2) = codes;
    }
    // Four blocks side by side (lanes 0, 4, 8, 12 of sixteen) make a word of the scales, and each lane has a byte for each of four such words:
    // a transposition of 4 x 4 bytes, after which the q-th four lanes hold the word of step q.
    const int q = lane / 4 % 4;
    const uint32_t other = __shfl_xor_sync(0xffffffffu, scale4, 4);
    const uint32_t pair = q & 1 ? __byte_perm(other, scale4, 0x7351) : __byte_perm(scale4, other, 0x6240);    // [word q%2: two blocks][word q%2 + 2: two blocks]
    const uint32_t far = __shfl_xor_sync(0xffffffffu, pair, 8);
    const uint32_t word = q & 2 ? __byte_perm(far, pair, 0x7632) : __byte_perm(pair, far, 0x5410);
    const int first = int(i % steps) * kStepCols + q * kWarpCols + lane / 16 * kScaleCols;
    if (lane % 4 == 0 && first < cols) *reinterpret_cast<uint32_t*>(scales + scaleOffset(row, first, colBlocks)) = word;
  }
}

PURLIN_D float powerOf(uint32_t scale) {      // 2^(scale - 127); 2^-127 is below the normal numbers, 255 is the NaN
  return __uint_as_float(scale == 255u ? 0x7fffffffu : scale ? scale << 23 : 0x00400000u);
}

template <int TYPE>
__global__ void __launch_bounds__(kQuantThreads) dequantizeKernel(const unsigned char* data, const unsigned char* scales, unsigned char* out, int rows, int cols, uint32_t steps, uint32_t total) {
  tc::gridDependencyWait();
  tc::gridLaunchDependents();
  const int lane = threadIdx.x & 31;
  const uint32_t warps = gridDim.x * (kQuantThreads / 32);
  const int colBlocks = (cols + kScaleCols - 1) / kScaleCols;
  for (uint32_t i = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5); i < total; i += warps) {
    const int row = int(i / steps), col = int(i % steps) * kStepCols + lane * kVec;
    const size_t at = size_t(row) * size_t(cols) + size_t(col);
    const unsigned char* scaleAt = scales + scaleOffset(row, col, colBlocks);          // (256 columns further on: two blocks of 512 bytes)
    uint32_t codes[kUnroll], scale[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      codes[u] = scale[u] = 0;
      if (col + u * kWarpCols < cols) {
        codes[u] = *reinterpret_cast<const uint32_t*>(data + (at + size_t(u * kWarpCols)) / 2);
        scale[u] = scaleAt[u * (kWarpCols / kScaleCols * kScaleBytes)];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (col + u * kWarpCols >= cols) continue;
      const float power = powerOf(scale[u]);
      float f[kVec];
#pragma unroll
      for (int e = 0; e < kVec; e += 2) {
        const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(__nv_fp4x2_storage_t(codes[u] >> (4 * e)), __NV_E2M1);
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
        f[e] = v.x * power;
        f[e + 1] = v.y * power;
      }
      if constexpr (TYPE == PURLIN_MX4_FP32) {
        float4* to = reinterpret_cast<float4*>(out + (at + size_t(u * kWarpCols)) * 4);
        __stcs(to, make_float4(f[0], f[1], f[2], f[3]));
        __stcs(to + 1, make_float4(f[4], f[5], f[6], f[7]));
      } else {
        __stcs(reinterpret_cast<uint4*>(out + (at + size_t(u * kWarpCols)) * 2),
               make_uint4(skinny::pack2(f[0], f[1]), skinny::pack2(f[2], f[3]), skinny::pack2(f[4], f[5]), skinny::pack2(f[6], f[7])));
      }
    }
  }
}

// ------------------------------------------------------------------------------------------
// the tensor core's side
// ------------------------------------------------------------------------------------------
constexpr int kBK = 256;                        // of k in a stage: 128 bytes of a row
constexpr int kBM = 128, kABytes = kBM * 128;
constexpr int kScaleStage = 1024;               // scales of 128 rows in a stage: two blocks
constexpr int kSmemLimit = 227 * 1024;

// e2m1 x e2m1 -> fp32, powers of two as scales, both operands K-major; M = 128 (one CTA) or 256 (a pair). `half`: which two of a word's
// four scales (64 of k) the instruction takes.
PURLIN_D uint32_t instrDescMx4(uint32_t n, uint32_t m, uint32_t half) {
  return (half << 5) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 7) << 27) | (half << 30);
}
// The producing and the issuing warp stay whole: all lanes wait and count, and the instructions below are predicated on one lane. In a branch of one
// lane the compiler has to move every operand into the uniform registers that these instructions read, which made a copy of scales
// take 45 cycles of the issuing thread instead of 8 and an MMA of few columns 48 instead of 32, with loops of run-time length around them about 90.
PURLIN_D uint32_t electOne() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e;
}
PURLIN_D bool waitAll(uint32_t bar, uint32_t parity, volatile int* abortWord, uint64_t timeoutNs) {
  return __all_sync(0xffffffffu, tc::mbarWait(bar, parity, abortWord, timeoutNs)) != 0;
}
template <int CTAS> PURLIN_D void mmaMx4(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scaleA, uint32_t scaleB, uint32_t accumulate) {
  if constexpr (CTAS == 2)
    asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 e, %7, 0;\n\t"
                 "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scaleA), "r"(scaleB), "r"(accumulate), "r"(elected) : "memory");
  else
    asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 e, %7, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scaleA), "r"(scaleB), "r"(accumulate), "r"(elected) : "memory");
}
// 512 bytes of scales (32 rows of 16 bytes) from shared memory into four columns of all four quarters of the TMEM lanes
PURLIN_D uint64_t scaleDesc(uint32_t smemByteAddr) {       // groups of 8 rows, 128 bytes apart, no swizzle
  const uint32_t lo = ((smemByteAddr >> 4) & 0x3FFFu) | (1u << 16), hi = (128u >> 4) | (1u << 14);
  return uint64_t(lo) | (uint64_t(hi) << 32);
}
template <int CTAS> PURLIN_D void scalesToTmem(uint32_t elected, uint32_t taddr, uint64_t desc) {
  if constexpr (CTAS == 2)
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(elected) : "memory");
  else
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(elected) : "memory");
}
template <int CTAS> PURLIN_D void commit(uint32_t elected, uint32_t bar) {      // on this barrier, of both CTAs of a pair
  if constexpr (CTAS == 2)
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t"
                 "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar), "h"(uint16_t(3)), "r"(elected) : "memory");
  else
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(elected) : "memory");
}

struct alignas(64) Maps { CUtensorMap a, b, sa, sb, c, bCut; };      // bCut: b in the boxes of a cut tile

// Scales as [row blocks][rows of 128 bytes, four to a block of 512]: eight of those, of one or two row blocks
PURLIN_D void loadScales(uint32_t smemDst, const CUtensorMap* map, int y, int rowBlock, uint32_t clusterBarAddress) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(smemDst), "l"(map), "r"(clusterBarAddress), "r"(0), "r"(y), "r"(rowBlock) : "memory");
}
PURLIN_D void loadScalesHere(uint32_t smemDst, const CUtensorMap* map, int y, int rowBlock, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(smemDst), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(rowBlock) : "memory");
}

// ---- many rows: 256 rows of A x up to 256 rows of W per CTA pair ----
// One accumulator of 256 columns; the scales of a stage take the columns behind it (two sets in turn). The epilogue gives the accumulator back
// as soon as its values are in registers; it activates, packs and stores them under the next main loop.
constexpr int kWideThreads = 32 * 10, kWideStages = 6, kMaxCols = 256;      // (4 stages were 5 % slower, 5 by 1 to 2 %)
constexpr int kWideStage = kABytes + kMaxCols / 2 * 128 + 3 * kScaleStage;      // [A][B half][scales A][scales B: two blocks of rows]
constexpr int kStageTileBytes = 32 * 64, kWideStaging = 8 * kStageTileBytes;      // 32 rows x 32 columns of the output per epilogue warp
constexpr int kBarrierBytes = 256;
constexpr int kScaleTmem = 256, kScaleSet = 32;                                   // columns: [A k-block 0, 1: 4 each][B k-block 0, 1: 8 each]
constexpr size_t kWideSmem = size_t(kWideStages) * kWideStage + kWideStaging + kBarrierBytes;
static_assert(kWideSmem <= size_t(kSmemLimit) && kWideStage % 1024 == 0, "the ring and the staging tiles fit one CTA per SM");

struct WideParams {
  int M, N, K, bn;                    // bn: columns of a tile, a multiple of 64, so they lie in two row blocks of W's scales
  int tilesM, tilesN, items, fullItems;
  int cut;                            // items [fullItems, items) are the tiles of a small last wave, cut into so many parts (1, 2 or 4) of 64 columns or more
  uint32_t* status;
  uint64_t timeoutNs;
};

struct WideItem { int row0, col0, cols; };     // first row of the pair's 256, first column and number of columns
constexpr int kBand = 8;
PURLIN_D WideItem wideItem(const WideParams& p, int it) {
  const bool whole = it < p.fullItems;
  const int tile = whole ? it : p.fullItems + (it - p.fullItems) / p.cut;
  const int perBand = kBand * p.tilesN, band = tile / perBand, within = tile - band * perBand, first = band * kBand;
  const int rows = min(p.tilesM - first, kBand);
  WideItem w{(first + within % rows) * 2 * kBM, within / rows * p.bn, p.bn};
  if (!whole) { w.cols = p.bn / p.cut; w.col0 += (it - p.fullItems) % p.cut * w.cols; }
  return w;
}

template <bool SWIGLU>
__global__ void __launch_bounds__(kWideThreads, 1) mx4WideKernel(const __grid_constant__ Maps maps, const __grid_constant__ WideParams p) {
  extern __shared__ __align__(1024) unsigned char smem[];     // swizzled tiles need 1024-byte alignment
  const uint32_t base = tc::smemAddr(smem);
  const uint32_t stagingAll = base + uint32_t(kWideStages) * kWideStage, barBase = stagingAll + kWideStaging;
  auto fullBar = [&](uint32_t s) { return barBase + 8u * s; };
  auto emptyBar = [&](uint32_t s) { return barBase + 8u * (uint32_t(kWideStages) + s); };
  const uint32_t tmemFull = barBase + 8u * (2 * kWideStages), tmemEmpty = tmemFull + 8u;
  uint32_t* words = reinterpret_cast<uint32_t*>(smem + size_t(kWideStages) * kWideStage + kWideStaging + 8 * (2 * kWideStages + 2));
  volatile uint32_t* tmemBaseWord = words;
  volatile int* abortWord = reinterpret_cast<volatile int*>(words + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ctaRank = tc::clusterCtaRank();
  const int pairIdx = int(blockIdx.x) / 2, numPairs = int(gridDim.x) / 2;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kWideStages; ++s) { tc::mbarInit(fullBar(s), 1); tc::mbarInit(emptyBar(s), 1); }
    tc::mbarInit(tmemFull, 1);
    tc::mbarInit(tmemEmpty, 16);                       // the epilogue warps of both CTAs
    *abortWord = 0;
    tc::mbarFenceInit();
    tc::tmaPrefetchDescriptor(&maps.a);
    tc::tmaPrefetchDescriptor(&maps.b);
  }
  if (warp == 1) { tc::tmemAllocPair(tc::smemAddr(words), 512); tc::tmemRelinquishPair(); }
  tc::fenceBeforeThreadSync();
  tc::clusterSync();
  tc::fenceAfterThreadSync();
  tc::gridDependencyWait();
  tc::gridLaunchDependents();
  const uint32_t tmemBase = *tmemBaseWord;
  const uint32_t leaderBars = tc::mapToCta(barBase, 0);
  const int kBlocks = (p.K + kBK - 1) / kBK;

  if (warp == 0) {
    const uint32_t elected = electOne();
    uint32_t st = 0, ph = 0;
    bool ok = true;
    for (int it = pairIdx; it < p.items && ok; it += numPairs) {
      const WideItem w = wideItem(p, it);
      const int half = w.cols / 2;
      const int aRow = w.row0 + int(ctaRank) * kBM, bRow = w.col0 + int(ctaRank) * half;
      // row blocks of the scales: this CTA's rows of A, all columns of the tile (two blocks; what lies past the last one reads as zero)
      const int sa = aRow / kScaleRows, sb = w.col0 / kScaleRows;
      const uint32_t bytes = uint32_t(2 * (kABytes + half * 128 + 3 * kScaleStage));
      for (int kb = 0; kb < kBlocks; ++kb) {
        ok = waitAll(emptyBar(st), ph ^ 1, abortWord, p.timeoutNs);
        if (!ok) { if (elected) skinny::recordTimeout(p.status, 1, it, kb); break; }
        const uint32_t sA = base + st * kWideStage, sB = sA + kABytes, sS = sB + kMaxCols / 2 * 128;
        const uint32_t full = leaderBars + 8u * st;
        if (elected) {
          if (ctaRank == 0) tc::mbarExpectTx(fullBar(st), bytes);
          tc::tmaLoad2dPair(sA, &maps.a, kb * 128, aRow, full);
          tc::tmaLoad2dPair(sB, it < p.fullItems ? &maps.b : &maps.bCut, kb * 128, bRow, full);
          loadScales(sS, &maps.sa, 8 * kb, sa, full);
          loadScales(sS + kScaleStage, &maps.sb, 8 * kb, sb, full);
        }
        __syncwarp();
        if (++st == kWideStages) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (ctaRank == 0) {
      const uint32_t elected = electOne();
      uint32_t st = 0, ph = 0, use = 0, set = 0;
      bool ok = true;
      const uint64_t descA0 = tc::smemDescSw128(base), descB0 = tc::smemDescSw128(base + kABytes), descS0 = scaleDesc(base + kABytes + kMaxCols / 2 * 128);
      for (int it = pairIdx; it < p.items && ok; it += numPairs, ++use) {
        const WideItem w = wideItem(p, it);
        const uint32_t shift = uint32_t(w.col0 % kScaleRows / 32);
        const bool twoBlocks = w.col0 % kScaleRows + w.cols > kScaleRows;
        const uint32_t idesc = instrDescMx4(uint32_t(w.cols), 2 * kBM, 0), idescHigh = instrDescMx4(uint32_t(w.cols), 2 * kBM, 1);
        ok = waitAll(tmemEmpty, (use & 1) ^ 1, abortWord, p.timeoutNs);
        if (!ok) { if (elected) skinny::recordTimeout(p.status, 2, it, 0); break; }
        for (int kb = 0; kb < kBlocks; ++kb, set ^= 1) {
          ok = waitAll(fullBar(st), ph, abortWord, p.timeoutNs);
          if (!ok) { if (elected) skinny::recordTimeout(p.status, 3, it, kb); break; }
          tc::fenceAfterThreadSync();
          const uint64_t off = uint64_t(st * (kWideStage >> 4)), da = descA0 + off, db = descB0 + off, ds = descS0 + off;
          const uint32_t scaleA = tmemBase + kScaleTmem + set * kScaleSet, scaleB = scaleA + 8;
          // In the stage: [scales of A: two blocks][of the first 128 columns: two blocks][of the next 128], 512 bytes each. The copies that a half of
          // the k-block needs come right before its MMAs, and columns that lie in one row block need no second copy: with few columns the
          // copies take as long as the MMAs (us, all copies first / so: 256 x 4096 x 14336 18.1 / 16.8, 256 x 8192 x 8192 13.0 / 12.1).
#pragma unroll
          for (uint32_t q = 0; q < 2; ++q) {
            scalesToTmem<2>(elected, scaleA + 4 * q, ds + 32 * q);
            scalesToTmem<2>(elected, scaleB + 8 * q, ds + 64 + 32 * q);
            if (twoBlocks) scalesToTmem<2>(elected, scaleB + 8 * q + 4, ds + 128 + 32 * q);
#pragma unroll
            for (uint32_t k = 2 * q; k < 2 * q + 2; ++k)      // (past K values and scales are zeros)
              mmaMx4<2>(elected, tmemBase, da + 2 * k, db + 2 * k, k & 1 ? idescHigh : idesc, scaleA + 4 * q, scaleB + 8 * q + shift, uint32_t(kb != 0 || k != 0));
          }
          commit<2>(elected, emptyBar(st));
          if (++st == kWideStages) { st = 0; ph ^= 1; }
        }
        if (ok) commit<2>(elected, tmemFull);
      }
    }
  } else {
    // ---- epilogue: two warps per quarter of the lanes, each up to two units of 64 accumulator columns ----
    constexpr int kOutWords = SWIGLU ? 8 : 16;         // packed outputs of 32 accumulator columns
    const int quarter = warp & 3, half = (warp - 2) / 4;
    const uint32_t buf = stagingAll + uint32_t(warp - 2) * kStageTileBytes;
    uint32_t use = 0;
    bool ok = true;
    for (int it = pairIdx; it < p.items && ok; it += numPairs, ++use) {
      const WideItem w = wideItem(p, it);
      const int units = w.cols / 64, first = half ? (units + 1) / 2 : 0, count = half ? units / 2 : (units + 1) / 2;
      const int row0 = w.row0 + int(ctaRank) * kBM + quarter * 32;
      ok = tc::mbarWait(tmemFull, use & 1, abortWord, p.timeoutNs);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) { if (lane == 0) skinny::recordTimeout(p.status, 5, it, 0); break; }
      tc::fenceAfterThreadSync();
      const uint32_t taddr = tmemBase + (uint32_t(quarter * 32) << 16) + uint32_t(first * 64);
      // all of this warp's values first: the accumulator goes back before any of them is activated, packed or stored
      uint32_t r[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c < 2 * count) tc::tmemLoad32(taddr + uint32_t(c * 32), r[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c < 2 * count) tc::tmemLoadWaitFor(r[c]);
      tc::fenceBeforeThreadSync();
      __syncwarp();
      if (lane == 0) tc::mbarArriveClusterTmem(leaderBars + 8u * (2 * kWideStages + 1));
      // Staging: 32 rows of 64 bytes (32 columns) with the 64-byte swizzle. Without the gate that is 32 accumulator columns, with it 64.
      constexpr int kChunks = SWIGLU ? 2 : 1;
#pragma unroll
      for (int u = 0; u < 4 / kChunks; ++u) {
        if (u * kChunks < 2 * count) {
          if (lane == 0) tc::bulkWaitGroupRead<0>();
          __syncwarp();
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const uint32_t (&v)[32] = r[kChunks * u + c];
            uint32_t o[kOutWords];
            if constexpr (SWIGLU) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                o[i] = skinny::pack2(skinny::siluOf(__uint_as_float(v[2 * i])) * __uint_as_float(v[16 + 2 * i]),
                                     skinny::siluOf(__uint_as_float(v[2 * i + 1])) * __uint_as_float(v[17 + 2 * i]));
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = skinny::pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
            }
#pragma unroll
            for (int j = 0; j < kOutWords / 4; ++j) {
              const uint32_t piece = uint32_t(c * (kOutWords / 4) + j);
              tc::stShared16(buf + uint32_t(lane) * 64u + (piece ^ uint32_t(lane >> 1 & 3)) * 16u, o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            }
          }
          tc::fenceProxyAsyncShared();
          __syncwarp();
          const int acc = w.col0 + first * 64 + u * kChunks * 32;
          if (lane == 0) { tc::tmaStore2d(&maps.c, SWIGLU ? acc / 2 : acc, row0, buf); tc::bulkCommitGroup(); }
        }
      }
    }
    if (lane == 0) tc::bulkWaitGroup<0>();
  }

  if (*abortWord) tc::landingPause();
  tc::fenceBeforeThreadSync();
  tc::clusterSync();
  if (warp == 1) tc::tmemDeallocPair(tmemBase, 512);
}

// ---- few rows: 128 rows of W are the rows of the MMA, the activations its columns, k split over a cluster ----
// As in gemm_skinny.cuh: what bounds it is the read of W, every byte of which passes one SM once; the fp32 partial tiles are added in distributed
// shared memory in ascending k order.
// DENSE: the activations come as bf16, and the four warps that wait for the sums quantise them in the meantime, every CTA its own k range of
// them, straight into the stages: one launch instead of two for a handful of tokens (one B200, us, two launches / one: 1 x 2048 x 2048 5.5 / 4.3, 1 x 7168 x 8192 8.9 / 7.6,
// 4 x 57344 x 8192 43.6 / 42.0; with two tokens to a warp 50.8, so up to four tokens).
constexpr int kFewThreads = skinny::kThreads, kWRows = 128, kMostFewRows = 80;
constexpr int kDenseTokens = 4, kDenseBytes = kDenseTokens * kBK * 2;      // a token to a warp; of bf16 activations in a stage

struct FewParams {
  int N, K, tokens, cols;              // cols: columns of the MMA, tokens rounded up to 16
  int stages, tmemCols, ahead;
  __nv_bfloat16* C;
  int ldc;
  uint32_t* status;
  uint64_t timeoutNs;
};
PURLIN_HD int fewStageBytes(int cols, bool dense) { return kABytes + cols * 128 + 2 * kScaleStage + (dense ? kDenseBytes : 0); }     // [W][X][scales W][scales X][bf16 X]

// Token w, 256 columns to a stage: from the bf16 values that TMA has brought into the stage to codes in the swizzled tile and scales in their blocks.
// (Tokens that there are not are zeros.) Plain loads, however early, would be waited for by every fence to the tensor core's proxy.
PURLIN_D bool quantiseStages(const FewParams& p, uint32_t base, uint32_t stageBytes, uint32_t fullBars, uint32_t denseBars, int w, int lane, int count, volatile int* abortWord) {
  uint32_t st = 0, ph = 0;
  for (int i = 0; i < count; ++i) {
    if (!waitAll(denseBars + 8u * st, ph, abortWord, p.timeoutNs)) { if (lane == 0) skinny::recordTimeout(p.status, 7, w, i); return false; }
    const uint32_t sX = base + st * stageBytes + kABytes, sS = sX + uint32_t(p.cols * 128) + kScaleStage, sD = sS + kScaleStage;
    Raw<PURLIN_MX4_BF16> raw;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(raw.v[0].x), "=r"(raw.v[0].y), "=r"(raw.v[0].z), "=r"(raw.v[0].w) : "r"(sD + uint32_t(w) * (kBK * 2) + uint32_t(lane) * 16u) : "memory");
    uint32_t peak = peakExponent<PURLIN_MX4_BF16>(raw);
    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
    const uint32_t scale = peak == 255u ? 255u : peak > 2u ? peak - 2u : 0u;
    float f[kVec];
    toFloats<PURLIN_MX4_BF16>(raw, f);
    const uint32_t codes = scale == 255u ? 0u : packCodes(f, __uint_as_float((254u - scale) << 23));
    uint32_t word = scale << (8 * (lane / 4 % 4));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(sX + uint32_t(w) * 128u + (uint32_t(lane / 4) ^ uint32_t(w & 7)) * 16u + uint32_t(lane % 4) * 4u), "r"(codes) : "memory");
    if (lane % 16 == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(sS + uint32_t(lane / 16) * kScaleBytes + uint32_t(w) * 16u), "r"(word) : "memory");
    tc::fenceProxyAsyncShared();
    __syncwarp();
    if (lane == 0) tc::mbarArrive(fullBars + 8u * st);
    if (++st == uint32_t(p.stages)) { st = 0; ph ^= 1; }
  }
  return true;
}

template <bool SWIGLU, bool DENSE>
__global__ void __launch_bounds__(kFewThreads, 2) mx4FewKernel(const __grid_constant__ Maps maps, const __grid_constant__ FewParams p) {
  extern __shared__ unsigned char smemRaw[];
  const uint32_t rawAddr = tc::smemAddr(smemRaw);
  const uint32_t base = (rawAddr + 1023u) & ~1023u;
  unsigned char* smem = smemRaw + (base - rawAddr);
  const uint32_t stageBytes = uint32_t(fewStageBytes(p.cols, DENSE));
  const uint32_t barBase = base + uint32_t(p.stages) * stageBytes;
  auto fullBar = [&](uint32_t s) { return barBase + 8u * s; };
  auto emptyBar = [&](uint32_t s) { return barBase + 8u * (uint32_t(p.stages) + s); };
  const uint32_t accFull = barBase + 8u * (2u * uint32_t(p.stages)), mmasDone = accFull + 8u, denseBars = mmasDone + 8u;      // denseBars: bf16 activations of a stage
  uint32_t* words = reinterpret_cast<uint32_t*>(smem + size_t(p.stages) * stageBytes + 8 * (3 * p.stages + 2));
  volatile uint32_t* tmemBaseWord = words;
  volatile int* abortWord = reinterpret_cast<volatile int*>(words + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t split;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(split));
  const uint32_t part = tc::clusterCtaRank();
  const int tile = int(blockIdx.x / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { tc::mbarInit(fullBar(s), DENSE ? 5 : 1); tc::mbarInit(emptyBar(s), 1); tc::mbarInit(denseBars + 8u * uint32_t(s), 1); }      // (the four quantising warps arrive too)
    tc::mbarInit(accFull, 1);
    tc::mbarInit(mmasDone, 1);
    *abortWord = 0;
    tc::mbarFenceInit();
    tc::tmaPrefetchDescriptor(&maps.a);
    tc::tmaPrefetchDescriptor(&maps.b);
  }
  const int kBlocks = (p.K + kBK - 1) / kBK;
  const int kBegin = int(int64_t(kBlocks) * part / split), kEnd = int(int64_t(kBlocks) * (part + 1) / split);
  // The first lap of the ring is asked into L2 while the kernel before this one (the quantisation of the activations) drains.
  if (warp == 0 && lane == 0)
    for (int kb = kBegin; kb < min(kEnd, kBegin + p.ahead); ++kb) tc::tmaPrefetchL2(&maps.a, kb * 128, tile * kWRows);
  if (warp == 1) { tc::tmemAlloc(tc::smemAddr(words), uint32_t(p.tmemCols)); tc::tmemRelinquish(); }
  tc::gridDependencyWait();
  tc::fenceBeforeThreadSync();
  __syncthreads();
  tc::fenceAfterThreadSync();
  const uint32_t tmemBase = *tmemBaseWord;
  uint32_t peer[skinny::kMaxSplit];
#pragma unroll
  for (int q = 0; q < skinny::kMaxSplit; ++q) peer[q] = uint32_t(q) < split ? tc::mapToCta(base, uint32_t(q)) : 0u;

  bool ok = true;
  uint32_t st = 0, ph = 0;
  if (warp == 0) {
    const uint32_t elected = electOne();
    for (int kb = kBegin; kb < kEnd && ok; ++kb) {
      ok = waitAll(emptyBar(st), ph ^ 1, abortWord, p.timeoutNs);
      if (!ok) { if (elected) skinny::recordTimeout(p.status, 1, tile, kb); break; }
      const uint32_t sW = base + st * stageBytes, sX = sW + kABytes, sS = sX + uint32_t(p.cols * 128);
      if (elected) {
        tc::mbarExpectTx(fullBar(st), DENSE ? uint32_t(kABytes + kScaleStage) : stageBytes);
        tc::tmaLoad2d(sW, &maps.a, kb * 128, tile * kWRows, fullBar(st));
        loadScalesHere(sS, &maps.sa, 8 * kb, tile, fullBar(st));
        if constexpr (DENSE) {
          tc::mbarExpectTx(denseBars + 8u * st, kDenseBytes);
          tc::tmaLoad2d(sS + 2 * kScaleStage, &maps.b, kb * kBK, 0, denseBars + 8u * st);
        } else {
          tc::tmaLoad2d(sX, &maps.b, kb * 128, 0, fullBar(st));
          loadScalesHere(sS + kScaleStage, &maps.sb, 8 * kb, 0, fullBar(st));
        }
      }
      __syncwarp();
      if (++st == uint32_t(p.stages)) { st = 0; ph ^= 1; }
    }
  } else if (warp == 1) {
    const uint32_t elected = electOne();
    const uint32_t idesc = instrDescMx4(uint32_t(p.cols), kWRows, 0), idescHigh = instrDescMx4(uint32_t(p.cols), kWRows, 1);
    const uint64_t descW = tc::smemDescSw128(base), descX = tc::smemDescSw128(base + kABytes), descS = scaleDesc(base + kABytes + uint32_t(p.cols * 128));
    const uint32_t scales = tmemBase + uint32_t((p.cols + 31) / 32 * 32);
    uint32_t set = 0;
    for (int kb = kBegin; kb < kEnd && ok; ++kb, set ^= 1) {
      ok = waitAll(fullBar(st), ph, abortWord, p.timeoutNs);
      if (!ok) { if (elected) skinny::recordTimeout(p.status, 3, tile, kb); break; }
      tc::fenceAfterThreadSync();
      const uint64_t off = uint64_t(st * (stageBytes >> 4));
      const uint32_t scaleW = scales + set * 16, scaleX = scaleW + 8;
#pragma unroll
      for (uint32_t q = 0; q < 2; ++q) {
        scalesToTmem<1>(elected, scaleW + 4 * q, descS + off + 32 * q);
        scalesToTmem<1>(elected, scaleX + 4 * q, descS + off + 64 + 32 * q);
      }
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k)          // (past K values and scales are zeros)
        mmaMx4<1>(elected, tmemBase, descW + off + 2 * k, descX + off + 2 * k, k & 1 ? idescHigh : idesc, scaleW + 4 * (k / 2), scaleX + 4 * (k / 2),
                  uint32_t(kb != kBegin || k != 0));
      commit<1>(elected, emptyBar(st));
      if (++st == uint32_t(p.stages)) { st = 0; ph ^= 1; }
    }
    if (ok) commit<1>(elected, accFull);
  } else {
    // ---- this CTA's partial tile: TMEM (lane = row of W, column = token) -> shared memory [token][row of W] ----
    const int quarter = warp & 3;
    if constexpr (DENSE) ok = quantiseStages(p, base, stageBytes, barBase, denseBars, warp - 2, lane, kEnd - kBegin, abortWord);
    if (ok) ok = waitAll(accFull, 0, abortWord, p.timeoutNs);
    if (!ok && lane == 0) skinny::recordTimeout(p.status, 5, tile, 0);
    if (ok) {
      // every load has landed and every MMA has read its stage, so the stages' memory is free
      tc::fenceAfterThreadSync();
      const uint32_t taddr = tmemBase + (uint32_t(quarter * 32) << 16);
      float* mine = reinterpret_cast<float*>(smem) + quarter * 32 + lane;
      for (int c = 0; c < p.tokens; c += 32) {
        uint32_t r[32];
        tc::tmemLoad32(taddr + uint32_t(c), r);
        tc::tmemLoadWaitFor(r);
#pragma unroll
        for (int i = 0; i < 32; ++i) if (c + i < p.tokens) mine[size_t(c + i) * kWRows] = __uint_as_float(r[i]);
      }
      tc::fenceBeforeThreadSync();
    }
  }
  if (!ok) {                            // the partial tile of this CTA is not what its peers would add: they learn of it through their abort words
    const uint32_t word = tc::smemAddr(words + 1);
    for (uint32_t q = 0; q < split; ++q) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::mapToCta(word, q)), "r"(1) : "memory");
  }
  __syncwarp();
  tc::clusterSync();                    // every partial tile of the cluster is in shared memory
  tc::gridLaunchDependents();
  if (*abortWord == 0) {
    constexpr int kOut = SWIGLU ? kWRows / 2 : kWRows, kPieces = kOut / 8;
    const int outCols = SWIGLU ? p.N / 2 : p.N, n0 = tile * kOut;
    const int begin = int(int64_t(p.tokens) * kPieces * part / split), end = int(int64_t(p.tokens) * kPieces * (part + 1) / split);
    for (int i = begin + int(threadIdx.x); i < end; i += kFewThreads) {
      const int t = i / kPieces, piece = i % kPieces;
      if (n0 + piece * 8 + 8 > outCols) continue;
      float v[8];
      if constexpr (SWIGLU) {
        const uint32_t at = uint32_t(t * kWRows + (piece >> 1) * 32 + (piece & 1) * 8) * 4u;
        float u[8];
        skinny::sumPartials(peer, int(split), at, v);
        skinny::sumPartials(peer, int(split), at + 64u, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = skinny::siluOf(v[e]) * u[e];
      } else {
        skinny::sumPartials(peer, int(split), uint32_t(t * kWRows + piece * 8) * 4u, v);
      }
      st16(p.C + size_t(t) * p.ldc + n0 + piece * 8, Vec16{{skinny::pack2(v[0], v[1]), skinny::pack2(v[2], v[3]), skinny::pack2(v[4], v[5]), skinny::pack2(v[6], v[7])}});
    }
  }
  tc::clusterSync();                    // nobody leaves behind a partial tile that a peer still reads
  if (*abortWord) {
    if (DENSE) tc::landingPause();      // (a stage that was not quantised never completes)
    else if (warp == 0 && lane == 0) for (uint32_t s = 0; s < uint32_t(p.stages); ++s) tc::mbarDrain(fullBar(s), s < st ? ph : ph ^ 1);
    if (warp == 1) {                    // (a commit counts what its own thread has issued)
      const uint32_t elected = electOne();
      commit<1>(elected, mmasDone);
      if (elected) tc::mbarDrain(mmasDone, 0);
    }
    __syncwarp();
  }
  tc::fenceBeforeThreadSync();
  __syncthreads();
  if (warp == 1) tc::tmemDealloc(tmemBase, uint32_t(p.tmemCols));
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
struct Device { int sms = 0, index = -1; };
bool currentDevice(Device& d) {
  static std::mutex mu;
  static int sms[64] = {};
  if (cudaGetDevice(&d.index) != cudaSuccess || d.index < 0 || d.index >= 64) { setError("mx4 launch: no current device"); return false; }
  std::lock_guard<std::mutex> lock(mu);
  if (!sms[d.index]) cudaDeviceGetAttribute(&sms[d.index], cudaDevAttrMultiProcessorCount, d.index);
  d.sms = sms[d.index];
  return d.sms > 0;
}

bool launched(cudaError_t e) {
  if (e != cudaSuccess) setError(std::string("mx4 launch: ") + cudaGetErrorString(e));
  return e == cudaSuccess;
}

bool sizesFit(int rows, int cols) {
  if (rows <= 0 || cols <= 0) { setError("mx4: dimensions must be positive"); return false; }
  if (cols % kBlock) { setError("mx4: the columns must be a multiple of 32"); return false; }
  if (rows > INT32_MAX - kScaleRows || cols > INT32_MAX - kStepCols) { setError("mx4: dimensions too large"); return false; }
  return true;
}

// steps of a row and of all rows, their number rounded up to a multiple of `unit`
bool stepsOf(int rows, int cols, int unit, uint32_t& steps, uint32_t& total) {
  steps = uint32_t((cols + kStepCols - 1) / kStepCols);
  const uint64_t all = uint64_t((rows + unit - 1) / unit) * uint64_t(unit) * steps;
  if (all > uint64_t(INT32_MAX)) { setError("mx4: the tensor is too large"); return false; }      // the walk counts in 32 bits
  total = uint32_t(all);
  return true;
}

template <typename... A>
int launchRows(void (*kernel)(A...), uint32_t total, const Device& dev, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
  constexpr int kWarps = kQuantThreads / 32;
  cfg.gridDim = dim3(std::min((total + kWarps - 1) / kWarps, uint32_t(dev.sms) * 32u));      // (8 per SM, all resident at once: 5 to 20 % slower)
  cfg.blockDim = dim3(kQuantThreads); cfg.stream = stream; cfg.attrs = attr; cfg.numAttrs = 1;
  return launched(cudaLaunchKernelEx(&cfg, kernel, args...)) ? 0 : 1;
}

// the scales of 128 rows x 256 columns, of `rowBlocks` row blocks, to a box; past the edges zeros
bool scaleMap(CUtensorMap* map, const void* ptr, int rows, int cols, int rowBlocks) {
  const TensorMapEncodeFn fn = tensorMapEncodeFn();
  if (!fn) { setError("cuTensorMapEncodeTiled is not available from this driver"); return false; }
  if (reinterpret_cast<uintptr_t>(ptr) % 16) { setError("TMA operands need 16-byte aligned base and row pitch"); return false; }
  const uint64_t blocks = uint64_t(cols + kScaleCols - 1) / kScaleCols;
  const cuuint64_t dims[3] = {128, blocks * 4, uint64_t(rows + kScaleRows - 1) / kScaleRows}, strides[2] = {128, blocks * kScaleBytes};
  const cuuint32_t box[3] = {128, kScaleStage / 128, uint32_t(rowBlocks)}, elem[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { setError("cuTensorMapEncodeTiled failed with code " + std::to_string(int(r))); return false; }
  return true;
}
// the output, in boxes of 32 rows x 64 bytes (32 columns)
bool outputMap(CUtensorMap* map, void* ptr, uint64_t rows, uint64_t cols) {
  const TensorMapEncodeFn fn = tensorMapEncodeFn();
  if (reinterpret_cast<uintptr_t>(ptr) % 16 || cols * 2 % 16) { setError("TMA operands need 16-byte aligned base and row pitch"); return false; }
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {cols * 2};
  const cuuint32_t box[2] = {32, 32}, elem[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { setError("cuTensorMapEncodeTiled failed with code " + std::to_string(int(r))); return false; }
  return true;
}

// bf16 activations, a few rows x 256 columns to a box, as they lie
bool denseMap(CUtensorMap* map, const void* ptr, int rows, int cols) {
  const TensorMapEncodeFn fn = tensorMapEncodeFn();
  if (!fn) { setError("cuTensorMapEncodeTiled is not available from this driver"); return false; }
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)}, strides[1] = {cuuint64_t(cols) * 2};
  const cuuint32_t box[2] = {kBK, kDenseTokens}, elem[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { setError("cuTensorMapEncodeTiled failed with code " + std::to_string(int(r))); return false; }
  return true;
}

size_t scaleBytes(int rows, int cols) { return size_t((rows + kScaleRows - 1) / kScaleRows) * size_t((cols + kScaleCols - 1) / kScaleCols) * kScaleBytes; }

bool optIn(const void* kernel, bool& done) {
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if (!done && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit) != cudaSuccess) { setError("cannot opt in to 227 KiB of shared memory"); return false; }
  done = true;
  return true;
}

int launchFew(const void* x, const void* aData, const void* aScales, const void* wData, const void* wScales, void* C, int M, int N, int K, bool swiglu, uint32_t* status, const Device& dev,
              cudaStream_t stream) {
  const int outCols = swiglu ? N / 2 : N;
  if (reinterpret_cast<uintptr_t>(C) % 16) { setError("TMA operands need 16-byte aligned base and row pitch"); return 1; }
  FewParams p{};
  p.N = N; p.K = K; p.tokens = M; p.cols = (M + 15) / 16 * 16;
  p.C = static_cast<__nv_bfloat16*>(C); p.ldc = outCols; p.status = status; p.timeoutNs = waitLimitNs((int64_t(K) + kBK - 1) / kBK);
  const int tiles = (N + kWRows - 1) / kWRows, kBlocks = (K + kBK - 1) / kBK;
  // k is cut while that brings more CTAs to work (two to an SM) and leaves each at least four k-blocks
  int split = 1;
  while (split < skinny::kMaxSplit && int64_t(tiles) * split * 2 <= 2 * int64_t(dev.sms) && kBlocks >= 8 * split) split *= 2;
  p.tmemCols = p.cols <= 32 ? 64 : 128;      // the accumulator's columns in 32s, and 32 for scales: kMostFewRows take 96 and 32
  // the partial tile [tokens][128] in fp32 takes the place of the stages
  const int room = 113 * 1024 - 1024 - 256, stage = fewStageBytes(p.cols, x != nullptr);
  p.stages = std::max(std::min({room / stage, 8, std::max((kBlocks + split - 1) / split, 2)}), (M * kWRows * 4 + stage - 1) / stage);
  p.ahead = std::min(p.stages, 4);
  Maps maps{};
  if (!makeTensorMap(&maps.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, wData, uint64_t(N), uint64_t(K) / 2, uint64_t(K) / 2, kWRows) || !scaleMap(&maps.sa, wScales, N, K, 1)) return 1;
  if (x ? !denseMap(&maps.b, x, M, K)
        : !makeTensorMap(&maps.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, aData, uint64_t(M), uint64_t(K) / 2, uint64_t(K) / 2, uint32_t(p.cols)) || !scaleMap(&maps.sb, aScales, M, K, 1)) return 1;
  auto kernel = x ? (swiglu ? mx4FewKernel<true, true> : mx4FewKernel<false, true>) : swiglu ? mx4FewKernel<true, false> : mx4FewKernel<false, false>;
  static bool done[64][4] = {};
  if (!optIn(reinterpret_cast<const void*>(kernel), done[dev.index][(x ? 2 : 0) + swiglu])) return 1;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = unsigned(split); attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(unsigned(tiles) * unsigned(split)); cfg.blockDim = dim3(kFewThreads); cfg.stream = stream;
  cfg.dynamicSmemBytes = size_t(p.stages) * size_t(stage) + kBarrierBytes + 1024; cfg.attrs = attr; cfg.numAttrs = 2;
  return launched(cudaLaunchKernelEx(&cfg, kernel, maps, p)) ? 0 : 1;
}

bool productFits(int M, int N, int K, int epilogue) {
  if (!sizesFit(M, K) || !sizesFit(N, K)) return false;
  if (epilogue != PURLIN_EPI_STORE && epilogue != PURLIN_EPI_SWIGLU) { setError("unknown epilogue"); return false; }
  const bool swiglu = epilogue == PURLIN_EPI_SWIGLU;
  if (N % (swiglu ? 32 : 8)) { setError(swiglu ? "the SwiGLU epilogue needs N to be a multiple of 32" : "mx4: N must be a multiple of 8"); return false; }
  if (int64_t(M) * N / 4096 > INT32_MAX / 4 || scaleBytes(std::max(M, N), K) / 128 > size_t(INT32_MAX)) { setError("mx4: the product is too large"); return false; }   // tile numbers, TMA coordinates
  return true;
}
bool overlap(const void* a, size_t aBytes, const void* b, size_t bBytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + bBytes && y < x + aBytes;
}
size_t productBytes(int M, int N, int epilogue) { return size_t(M) * size_t(epilogue == PURLIN_EPI_SWIGLU ? N / 2 : N) * 2; }
// Tiles of C are stored while others still read their operands.
bool apartFromOutput(const void* data, const void* scales, int rows, int cols, const void* C, size_t bytes) {
  if (!overlap(data, size_t(rows) * size_t(cols) / 2, C, bytes) && !overlap(scales, scaleBytes(rows, cols), C, bytes)) return true;
  setError("mx4: C overlaps a quantised operand");
  return false;
}
// whether the product quantises its activations itself
bool quantisedInside(int dtype, int M) { return dtype == PURLIN_MX4_BF16 && M <= kDenseTokens; }

// Rows of A up to which the kernel for few rows is taken. The other one does not care how many of 256 there are; us, few rows 64 /
// few rows 96 / the other: N, K 1024, 7168 6.3 / 7.3 / 9.1; 2048, 2048 5.1 / 5.6 / 5.1; 4096, 14336 13.3 / 17.1 / 15.2; 8192, 8192 few rows 64 11.3,
// the other 10.9; 14336, 2048 7.4 and 7.5; 28672, 4096 11.2 and 14.4.
int fewRows(int N) { return N < 8192 ? kMostFewRows : 64; }

int launchWide(const void* aData, const void* aScales, const void* wData, const void* wScales, void* C, int M, int N, int K, bool swiglu, uint32_t* status, const Device& dev,
               cudaStream_t stream) {
  auto kernel = swiglu ? mx4WideKernel<true> : mx4WideKernel<false>;
  static bool done[64][2] = {};
  if (!optIn(reinterpret_cast<const void*>(kernel), done[dev.index][swiglu])) return 1;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kWideThreads); cfg.stream = stream; cfg.dynamicSmemBytes = kWideSmem; cfg.attrs = attr;
  static std::mutex mu;
  static int known[64][2] = {};
  int pairs;
  {
    std::lock_guard<std::mutex> lock(mu);
    int& n = known[dev.index][swiglu];
    if (!n) {                           // pairs must sit on SMs of one GPC: ask how many the device can hold at once
      n = dev.sms / 2;
      cfg.gridDim = dim3(unsigned(dev.sms / 2 * 2)); cfg.numAttrs = 1;
      int m = 0;
      if (cudaOccupancyMaxActiveClusters(&m, kernel, &cfg) == cudaSuccess && m > 0) n = std::min(n, m);
    }
    pairs = n;
  }
  WideParams p{};
  p.M = M; p.N = N; p.K = K; p.status = status; p.timeoutNs = waitLimitNs(2 * ((int64_t(K) + kBK - 1) / kBK));
  p.tilesM = (M + 2 * kBM - 1) / (2 * kBM);
  // The width that is expected to take least: a tile costs its columns and about 48 columns' worth besides (fill, drain, the loads of A). Tiles of a
  // last wave that leaves pairs idle are cut where every part finds a pair (us, uncut / in halves / in quarters:
  // 1000 x 14336 x 8192 gated 50.9 / 46.0 / 45.7, 4096 x 4864 x 2048 20.7 / 19.3 / 19.0).
  double least = 1e30;
  for (int bn : {256, 192, 128}) {
    const int tilesN = (N + bn - 1) / bn, tiles = p.tilesM * tilesN, rest = tiles % pairs;
    const int cut = tiles <= pairs || !rest ? 1 : bn == 256 && 4 * rest <= pairs ? 4 : bn != 192 && 2 * rest <= pairs ? 2 : 1;
    const double cost = double(tiles / pairs) * (bn + 48) + (rest ? bn / cut + 48 : 0);
    if (cost < least) {
      least = cost;
      p.bn = bn; p.tilesN = tilesN; p.cut = cut;
      p.fullItems = cut > 1 ? tiles - rest : tiles;
      p.items = p.fullItems + (tiles - p.fullItems) * cut;
    }
  }
  const int outCols = swiglu ? N / 2 : N;
  Maps maps{};
  if (!makeTensorMap(&maps.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, aData, uint64_t(M), uint64_t(K) / 2, uint64_t(K) / 2, kBM) ||
      !makeTensorMap(&maps.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, wData, uint64_t(N), uint64_t(K) / 2, uint64_t(K) / 2, uint32_t(p.bn / 2)) ||
      !(p.cut == 1 || makeTensorMap(&maps.bCut, CU_TENSOR_MAP_DATA_TYPE_UINT8, wData, uint64_t(N), uint64_t(K) / 2, uint64_t(K) / 2, uint32_t(p.bn / 2 / p.cut))) ||
      !scaleMap(&maps.sa, aScales, M, K, 1) || !scaleMap(&maps.sb, wScales, N, K, 2) ||
      !outputMap(&maps.c, C, uint64_t(M), uint64_t(outCols))) return 1;
  cfg.gridDim = dim3(unsigned(2 * std::min(pairs, p.items))); cfg.numAttrs = 2;
  return launched(cudaLaunchKernelEx(&cfg, kernel, maps, p)) ? 0 : 1;
}

}  // namespace

extern "C" {

size_t purlin_mx4_scale_bytes(int rows, int cols) { return rows > 0 && cols > 0 ? scaleBytes(rows, cols) : 0; }

int purlin_mx4_quantize(const void* x, int dtype, void* data, void* scales, int rows, int cols, void* stream) {
  NvtxRange range("mx4Quantize", size_t(rows) * size_t(cols) / 2);
  if (!sizesFit(rows, cols)) return 1;
  if (!x || !data || !scales) { setError("mx4: an operand is missing"); return 1; }
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(scales)) % 16) { setError("mx4: tensors must start on a 16-byte boundary"); return 1; }
  Device dev;
  if (!currentDevice(dev)) return 1;
  uint32_t steps, total;
  if (!stepsOf(rows, cols, kScaleRows, steps, total)) return 1;
  auto kernel = dtype == PURLIN_MX4_BF16 ? quantizeKernel<PURLIN_MX4_BF16> : dtype == PURLIN_MX4_FP16 ? quantizeKernel<PURLIN_MX4_FP16>
              : dtype == PURLIN_MX4_FP32 ? quantizeKernel<PURLIN_MX4_FP32> : nullptr;
  if (!kernel) { setError("mx4: unknown type"); return 1; }
  return launchRows(kernel, total, dev, static_cast<cudaStream_t>(stream), static_cast<const unsigned char*>(x), static_cast<unsigned char*>(data),
                    static_cast<unsigned char*>(scales), rows, cols, steps, total);
}

int purlin_mx4_dequantize(const void* data, const void* scales, void* out, int dtype, int rows, int cols, void* stream) {
  NvtxRange range("mx4Dequantize", size_t(rows) * size_t(cols) / 2);
  if (!sizesFit(rows, cols)) return 1;
  if (!data || !scales || !out) { setError("mx4: an operand is missing"); return 1; }
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(scales)) % 16) { setError("mx4: tensors must start on a 16-byte boundary"); return 1; }
  Device dev;
  if (!currentDevice(dev)) return 1;
  uint32_t steps, total;
  if (!stepsOf(rows, cols, 1, steps, total)) return 1;
  auto kernel = dtype == PURLIN_MX4_BF16 ? dequantizeKernel<PURLIN_MX4_BF16> : dtype == PURLIN_MX4_FP32 ? dequantizeKernel<PURLIN_MX4_FP32> : nullptr;
  if (!kernel) { setError("mx4: values come back in bf16 or fp32"); return 1; }
  return launchRows(kernel, total, dev, static_cast<cudaStream_t>(stream), static_cast<const unsigned char*>(data), static_cast<const unsigned char*>(scales),
                    static_cast<unsigned char*>(out), rows, cols, steps, total);
}

int purlin_mx4_gemm(const void* aData, const void* aScales, const void* wData, const void* wScales, void* C, int M, int N, int K, int epilogue, uint32_t* status, void* stream) {
  const bool swiglu = epilogue == PURLIN_EPI_SWIGLU;
  NvtxRange range(swiglu ? "mx4GemmSwiglu" : "mx4Gemm", size_t(M) * size_t(N) * 2);
  Device dev;
  if (!productFits(M, N, K, epilogue)) return 1;
  if (!aData || !aScales || !wData || !wScales || !C) { setError("mx4: an operand is missing"); return 1; }
  const size_t bytes = productBytes(M, N, epilogue);
  if (!apartFromOutput(aData, aScales, M, K, C, bytes) || !apartFromOutput(wData, wScales, N, K, C, bytes)) return 1;
  if (!currentDevice(dev)) return 1;
  return M <= fewRows(N) ? launchFew(nullptr, aData, aScales, wData, wScales, C, M, N, K, swiglu, status, dev, static_cast<cudaStream_t>(stream))
                         : launchWide(aData, aScales, wData, wScales, C, M, N, K, swiglu, status, dev, static_cast<cudaStream_t>(stream));
}

size_t purlin_mx4_workspace_bytes(int dtype, int M, int K) {
  return M <= 0 || K <= 0 || quantisedInside(dtype, M) ? 0 : size_t(M) * size_t(K) / 2 + scaleBytes(M, K);
}

int purlin_mx4_linear(const void* x, int dtype, void* workspace, const void* wData, const void* wScales, void* C, int M, int N, int K, int epilogue, uint32_t* status, void* stream) {
  if (!productFits(M, N, K, epilogue)) return 1;
  // Where C overlaps x, x is quantised by a launch of its own first: inside the product CTAs that are done would write over what others still read.
  const size_t bytes = productBytes(M, N, epilogue);
  const bool overX = overlap(x, size_t(M) * size_t(K) * (dtype == PURLIN_MX4_FP32 ? 4 : 2), C, bytes);
  if (quantisedInside(dtype, M) && !overX) {
    const bool swiglu = epilogue == PURLIN_EPI_SWIGLU;
    NvtxRange range(swiglu ? "mx4LinearSwiglu" : "mx4Linear", size_t(M) * size_t(N) * 2);
    Device dev;
    if (!x || !wData || !wScales || !C) { setError("mx4: an operand is missing"); return 1; }
    if (reinterpret_cast<uintptr_t>(x) % 16) { setError("mx4: tensors must start on a 16-byte boundary"); return 1; }
    if (!apartFromOutput(wData, wScales, N, K, C, bytes)) return 1;
    if (!currentDevice(dev)) return 1;
    return launchFew(x, nullptr, nullptr, wData, wScales, C, M, N, K, swiglu, status, dev, static_cast<cudaStream_t>(stream));
  }
  unsigned char* data = static_cast<unsigned char*>(workspace);
  if (!data) { setError(overX ? "mx4: C overlaps x, which takes a workspace" : "mx4: an operand is missing"); return 1; }
  unsigned char* scales = data + size_t(M) * size_t(K) / 2;       // (a row is a multiple of 16 bytes)
  const int rc = purlin_mx4_quantize(x, dtype, data, scales, M, K, stream);
  return rc ? rc : purlin_mx4_gemm(data, scales, wData, wScales, C, M, N, K, epilogue, status, stream);
}

}  // extern "C"
