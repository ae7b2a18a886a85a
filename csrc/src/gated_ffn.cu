// The gated feed-forward block for training, on the tensor cores of sm_100a.
//
//   forward    Z = X Wgu^T (16 columns of gate, 16 of up in turn), h = act(G) * U, y = h Wd^T
//   backward   dh = dY Wd;  dU = dh act(G);  dG = dh U act'(G);  dX = dZ Wgu;  dWgu = dZ^T X;  dWd = dY^T h
//
// Every product here is D[m, n] = sum_k A(m, k) B(n, k) of one kernel whose operands may lie in memory with k contiguous (a row of X, of a
// weight in the forward) or with m or n contiguous (a weight in dX = dZ Wgu, both operands of a weight's gradient, where k counts tokens).
// The tensor core reads either order from shared memory, so nothing is ever transposed in memory. TMA fills zeros past every edge, so
// any number of tokens is summed over without a remainder path.
//
// Both projections, the activation and the product are one launch (epilogue kGate); dh is never written: the epilogue of dY Wd turns the
// accumulator and the saved pre-activations into dZ (kGateGrad).
//
// The pre-activations are saved in 24 bits (fp32 without its last mantissa byte), in the order in which the threads of both epilogues hold
// them: a warp's 32 rows x 32 columns are 3 KiB in a row, six 16-byte pieces per lane, so that neither side passes them through shared
// memory. In bf16 their rounding would be the largest error of dZ (dX against 64 bits: 2.9e-3 instead of 2.35e-3, of which 1.66e-3 each are
// the roundings of dZ and of dX); with h they take the 8 bytes per element of h that separate bf16 tensors of gate, up, act(gate) and h would.
// h and dZ are rounded to bf16 because they are operands of tensor-core products; all sums are fp32 in tensor memory.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "purlin/gated_ffn.h"
#include "purlin/gemm.h"
#include "purlin/gemm_skinny.cuh"
#include "purlin/tc_sm100.cuh"
#include "purlin/telemetry.hpp"
#include "purlin/tensor_map.hpp"

using namespace purlin;

namespace {

constexpr int kBM = 128, kBK = 64;
constexpr int kABytes = kBM * kBK * 2;          // 16 KiB
constexpr int kBoxBytes = 64 * 128;             // a box of 64 x 64 of an operand whose rows or columns are contiguous
constexpr int kAccStride = 256, kTmemCols = 512;
constexpr int kEpiWarps = 8, kThreads = 32 * (2 + kEpiWarps);
constexpr int kStageTileBytes = 32 * 128;       // 32 rows x 64 bf16 columns, 128-byte swizzle
constexpr int kStageTiles = 2;                  // of every epilogue warp
constexpr int kStagingBytes = kEpiWarps * kStageTiles * kStageTileBytes;
constexpr int kBarrierBytes = 256, kMaxStages = 12;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kSavedVectors = 6;                // 16-byte pieces of 32 values in 24 bits
constexpr size_t kSavedBlock = size_t(kSavedVectors) * 32 * 16;   // 32 rows x 32 columns
static_assert(8 * (2 * kMaxStages + 4) + 8 <= kBarrierBytes, "the barriers, the TMEM base and the abort word fit their block");

enum { kStore = 0, kGate = 1, kGateGrad = 2 };

struct Params {
  int M, N, K, bn, stages, aBytes;       // aBytes: of one block of A in a stage (fewer than 128 rows where there are fewer)
  int tilesM, tilesN;
  int items, fullItems;                  // tiles [0, fullItems) whole, then the remaining ones as halves of one accumulator
  __nv_bfloat16* C;                      // output, or dZ
  int ldc;
  uint4* saved;                          // pre-activations: written by kGate (unless null), read by kGateGrad
  int savedCols;                         // its 32-column blocks per row block
  int activation;
  uint32_t* status;
  uint64_t timeoutNs;
};
struct alignas(64) Maps { CUtensorMap a, b, c; };

PURLIN_D float sigmoidOf(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
// act(g) = g sigmoid(s(g)): s = g (silu), s = 2 sqrt(2 / pi) (g + 0.044715 g^3) (gelu with the tanh). Past |g| = 16 the sigmoid is 0 or 1
// in fp32, so the cube is taken of the clamped value and cannot overflow.
constexpr float kGeluScale = 1.5957691216057308f, kGeluCube = 0.044715f;
PURLIN_D void activate(int activation, float g, float& act, float& grad) {
  float s = g, ds = 1.f;
  if (activation == PURLIN_ACT_GELU) {
    const float c = fminf(fmaxf(g, -16.f), 16.f), c2 = c * c;
    s = kGeluScale * c * fmaf(kGeluCube, c2, 1.f);
    ds = kGeluScale * fmaf(3.f * kGeluCube, c2, 1.f);
  }
  const float sig = sigmoidOf(s);
  act = g * sig;
  grad = fmaf(act * (1.f - sig), ds, sig);
}

// 32 fp32 values without their last byte <-> 24 words. (Cut, not rounded: a NaN stays one.)
PURLIN_D void pack24(const uint32_t (&v)[32], uint32_t (&w)[24]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[3 * i] = __byte_perm(v[4 * i], v[4 * i + 1], 0x5321);
    w[3 * i + 1] = __byte_perm(v[4 * i + 1], v[4 * i + 2], 0x6532);
    w[3 * i + 2] = __byte_perm(v[4 * i + 2], v[4 * i + 3], 0x7653);
  }
}
template <int I> PURLIN_D float unpack24(const uint32_t (&w)[24]) {
  constexpr int q = I / 4, r = I % 4;
  if constexpr (r == 0) return __uint_as_float(w[3 * q] << 8);
  else if constexpr (r == 1) return __uint_as_float(__byte_perm(w[3 * q], w[3 * q + 1], 0x5430) & 0xffffff00u);
  else if constexpr (r == 2) return __uint_as_float(__byte_perm(w[3 * q + 1], w[3 * q + 2], 0x4320) & 0xffffff00u);
  else return __uint_as_float(w[3 * q + 2] & 0xffffff00u);
}
PURLIN_D uint4 ldStream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
PURLIN_D void loadSaved(const uint4* block, int lane, uint32_t (&w)[24]) {
#pragma unroll
  for (int i = 0; i < kSavedVectors; ++i) {
    const uint4 v = ldStream(block + i * 32 + lane);
    w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
  }
}

// dG (o[0..7]) and dU (o[8..15]) of 16 columns, packed to bf16, from dh (columns C0 ... of the 32 in r) and the saved block
template <int C0, int J = 0>
PURLIN_D void gateGrad(int activation, const uint32_t (&r)[32], const uint32_t (&w)[24], uint32_t (&o)[16]) {
  if constexpr (J < 16) {
    float a0, d0, a1, d1;
    activate(activation, unpack24<J>(w), a0, d0);
    activate(activation, unpack24<J + 1>(w), a1, d1);
    const float h0 = __uint_as_float(r[C0 + J]), h1 = __uint_as_float(r[C0 + J + 1]);
    o[J / 2] = skinny::pack2(h0 * unpack24<16 + J>(w) * d0, h1 * unpack24<17 + J>(w) * d1);
    o[8 + J / 2] = skinny::pack2(h0 * a0, h1 * a1);
    gateGrad<C0, J + 2>(activation, r, w, o);
  }
}

// Tile t -> (row block, column block), rows fastest inside bands of row blocks: the tiles in flight share operands in L2
constexpr int kBand = 8;
PURLIN_D void tileCoord(const Params& p, int t, int& mIdx, int& nIdx) {
  const int perBand = kBand * p.tilesN, band = t / perBand, within = t - band * perBand, first = band * kBand;
  const int rows = min(p.tilesM - first, kBand);
  mIdx = first + within % rows;
  nIdx = within / rows;
}
struct Item { int tile, first, count; };     // accumulators [first, first + count) of a tile
template <int ACCS> PURLIN_D Item itemOf(const Params& p, int i) {
  if (ACCS == 1 || i < p.fullItems) return Item{i, 0, ACCS};
  const int j = i - p.fullItems;
  return Item{p.fullItems + (j >> 1), j & 1, 1};
}

// CTAS = 2: a cluster of two CTAs owns a tile: each loads its 128 rows of A per accumulator and its half of B's columns, CTA 0 issues one
// 256-row MMA for the pair. ACCS = 2: a tile is two accumulators tall; they share B, and their MMAs alternate (an MMA waits for the one before
// into the same columns). ACCS = 1: tiles alternate between the two accumulators, the epilogue of one runs under the MMAs of the next.
template <bool A_MN, bool B_MN, int EPI, int CTAS, int ACCS>
__global__ void __launch_bounds__(kThreads, 1) ffnKernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  extern __shared__ unsigned char smemRaw[];
  const uint32_t rawAddr = tc::smemAddr(smemRaw);
  const uint32_t base = (rawAddr + 1023u) & ~1023u;
  unsigned char* smem = smemRaw + (base - rawAddr);
  const int bnLocal = p.bn / CTAS;
  const int bBytes = bnLocal * kBK * 2;
  const uint32_t stageBytes = uint32_t(ACCS * p.aBytes + bBytes);      // [A block 0][A block 1][B], a multiple of 1 KiB
  const uint32_t stagingAll = base + uint32_t(p.stages) * stageBytes;
  const uint32_t barBase = stagingAll + kStagingBytes;
  auto fullBar = [&](uint32_t s) { return barBase + 8u * s; };
  auto emptyBar = [&](uint32_t s) { return barBase + 8u * (uint32_t(kMaxStages) + s); };
  auto tmemFullBar = [&](int a) { return barBase + 8u * uint32_t(2 * kMaxStages + a); };
  auto tmemEmptyBar = [&](int a) { return barBase + 8u * uint32_t(2 * kMaxStages + 2 + a); };
  uint32_t* words = reinterpret_cast<uint32_t*>(smem + size_t(p.stages) * stageBytes + kStagingBytes + 8 * (2 * kMaxStages + 4));
  volatile uint32_t* tmemBaseWord = words;
  volatile int* abortWord = reinterpret_cast<volatile int*>(words + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ctaRank = CTAS == 2 ? tc::clusterCtaRank() : 0u;
  const int pairIdx = int(blockIdx.x) / CTAS, numPairs = int(gridDim.x) / CTAS;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) { tc::mbarInit(fullBar(s), 1); tc::mbarInit(emptyBar(s), 1); }
    for (int a = 0; a < 2; ++a) { tc::mbarInit(tmemFullBar(a), 1); tc::mbarInit(tmemEmptyBar(a), kEpiWarps / 2 * CTAS); }
    *abortWord = 0;
    tc::mbarFenceInit();
    tc::tmaPrefetchDescriptor(&maps.a);
    tc::tmaPrefetchDescriptor(&maps.b);
  }
  if (warp == 1) {
    if constexpr (CTAS == 2) { tc::tmemAllocPair(tc::smemAddr(words), kTmemCols); tc::tmemRelinquishPair(); }
    else { tc::tmemAlloc(tc::smemAddr(words), kTmemCols); tc::tmemRelinquish(); }
  }
  tc::fenceBeforeThreadSync();
  if constexpr (CTAS == 2) tc::clusterSync(); else __syncthreads();    // the pair's barriers exist before any remote arrival
  tc::fenceAfterThreadSync();
  tc::gridDependencyWait();                                             // from here on memory that earlier kernels write may be read
  tc::gridLaunchDependents();
  const uint32_t tmemBase = *tmemBaseWord;
  const uint32_t leaderBars = CTAS == 2 ? tc::mapToCta(barBase, 0) : barBase;
  const int kBlocks = (p.K + kBK - 1) / kBK;

  if (warp == 0) {
    // ---- TMA producer ----
    if (lane == 0) {
      uint32_t st = 0, ph = 0;
      bool ok = true;
      for (int it = pairIdx; it < p.items && ok; it += numPairs) {
        const Item item = itemOf<ACCS>(p, it);
        int mIdx, nIdx;
        tileCoord(p, item.tile, mIdx, nIdx);
        const int aRow = ((mIdx * ACCS + item.first) * CTAS + int(ctaRank)) * kBM, bRow = nIdx * p.bn + int(ctaRank) * bnLocal;
        for (int kb = 0; kb < kBlocks; ++kb) {
          ok = tc::mbarWait(emptyBar(st), ph ^ 1, abortWord, p.timeoutNs);
          if (!ok) { skinny::recordTimeout(p.status, 1, item.tile, kb); break; }
          const uint32_t sA = base + st * stageBytes, sB = sA + uint32_t(ACCS * p.aBytes);
          const uint32_t full = leaderBars + 8u * st;                   // both CTAs' bytes are credited to CTA 0's barrier
          if (CTAS == 1 || ctaRank == 0) tc::mbarExpectTx(fullBar(st), uint32_t(CTAS * (item.count * p.aBytes + bBytes)));
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if constexpr (CTAS == 2) tc::tmaLoad2dPair(dst, map, x, y, full);
            else tc::tmaLoad2d(dst, map, x, y, fullBar(st));
          };
#pragma unroll
          for (int a = 0; a < ACCS; ++a) {
            if (a >= item.count) break;
            const int row = aRow + a * CTAS * kBM;
            if constexpr (A_MN) {
              load(sA + uint32_t(a * kABytes), &maps.a, row, kb * kBK);
              load(sA + uint32_t(a * kABytes + kBoxBytes), &maps.a, row + 64, kb * kBK);
            } else {
              load(sA + uint32_t(a * p.aBytes), &maps.a, kb * kBK, row);
            }
          }
          if constexpr (B_MN) {
            for (int j = 0; j < bnLocal / 64; ++j) load(sB + uint32_t(j * kBoxBytes), &maps.b, bRow + 64 * j, kb * kBK);
          } else {
            load(sB, &maps.b, kb * kBK, bRow);
          }
          if (++st == uint32_t(p.stages)) { st = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issuer (CTA 0 of a pair) ----
    if (lane == 0 && ctaRank == 0) {
      const uint32_t idesc = tc::instrDescBf16(uint32_t(p.bn), uint32_t(kBM * CTAS)) | (A_MN ? tc::kInstrDescAMnMajor : 0u) | (B_MN ? tc::kInstrDescBMnMajor : 0u);
      const uint64_t descA0 = A_MN ? tc::smemDescSw128MnMajor(base) : tc::smemDescSw128(base);
      const uint32_t bBase = base + uint32_t(ACCS * p.aBytes);
      const uint64_t descB0 = B_MN ? tc::smemDescSw128MnMajor(bBase) : tc::smemDescSw128(bBase);
      constexpr uint32_t kStepA = A_MN ? 128 : 2, kStepB = B_MN ? 128 : 2;        // 16 of k, in units of 16 bytes
      const uint32_t stageStep = stageBytes >> 4, accStep = uint32_t(p.aBytes) >> 4;
      uint32_t st = 0, ph = 0, accIt = 0, use0 = 0, use1 = 0;
      bool ok = true;
      auto commit = [&](uint32_t bar) {                                 // on this barrier of every CTA of the tile
        if constexpr (CTAS == 2) tc::mmaCommitPairs(bar, 3u);
        else tc::mmaCommit(bar);
      };
      for (int it = pairIdx; it < p.items && ok; it += numPairs, ++accIt) {
        const Item item = itemOf<ACCS>(p, it);
        const int a0 = ACCS == 1 ? int(accIt & 1) : 0;
        const bool two = ACCS == 2 && item.count == 2;
        ok = tc::mbarWait(tmemEmptyBar(a0), ((a0 ? use1 : use0) & 1) ^ 1, abortWord, p.timeoutNs);
        if (ok && two) ok = tc::mbarWait(tmemEmptyBar(1), (use1 & 1) ^ 1, abortWord, p.timeoutNs);
        if (!ok) { skinny::recordTimeout(p.status, 2, item.tile, 0); break; }
        const uint32_t d0 = tmemBase + uint32_t(a0) * kAccStride, d1 = tmemBase + kAccStride;
        for (int kb = 0; kb < kBlocks; ++kb) {
          ok = tc::mbarWait(fullBar(st), ph, abortWord, p.timeoutNs);
          if (!ok) { skinny::recordTimeout(p.status, 3, item.tile, kb); break; }
          tc::fenceAfterThreadSync();
          const uint64_t da = descA0 + uint64_t(st * stageStep), db = descB0 + uint64_t(st * stageStep);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            const uint32_t accumulate = uint32_t((kb | k) != 0);
            if constexpr (CTAS == 2) {
              tc::mmaPair(d0, da + kStepA * k, db + kStepB * k, idesc, accumulate);
              if constexpr (ACCS == 2) { if (two) tc::mmaPair(d1, da + accStep + kStepA * k, db + kStepB * k, idesc, accumulate); }
            } else {
              tc::mma(d0, da + kStepA * k, db + kStepB * k, idesc, accumulate);
            }
          }
          commit(emptyBar(st));
          if (++st == uint32_t(p.stages)) { st = 0; ph ^= 1; }
        }
        if (ok) {
          commit(tmemFullBar(a0));
          if (a0) ++use1; else ++use0;
          if (two) { commit(tmemFullBar(1)); ++use1; }
        }
      }
    }
  } else {
    // ---- epilogue: four warps for each accumulator ----
    const int quarter = warp & 3, group = (warp - 2) / 4;               // a warp may only touch TMEM lanes [32 * (warp % 4), +32)
    const uint32_t stagingWarp = stagingAll + uint32_t(warp - 2) * uint32_t(kStageTiles * kStageTileBytes);
    const uint32_t rowAddr = uint32_t(lane) * 128u, swz = uint32_t(lane & 7);
    uint32_t accIt = 0, uses = 0, tileCount = 0;
    bool ok = true;
    for (int it = pairIdx; it < p.items && ok; it += numPairs, ++accIt) {
      const Item item = itemOf<ACCS>(p, it);
      if (ACCS == 1 ? int(accIt & 1) != group : group >= item.count) continue;
      int mIdx, nIdx;
      tileCoord(p, item.tile, mIdx, nIdx);
      const int row0 = ((mIdx * ACCS + item.first + (ACCS == 2 ? group : 0)) * CTAS + int(ctaRank)) * kBM + quarter * 32;
      const int n0 = nIdx * p.bn, rowsValid = min(p.M - row0, 32);
      // chunks of 32 accumulator columns that hold output
      const int nChunks = rowsValid <= 0 ? 0 : (min(p.bn, p.N - n0) + 31) / 32;
      uint4* saved = nullptr;                                           // of this warp's rows and the tile's first columns
      uint32_t z[24];
      if constexpr (EPI == kGate) { if (p.saved) saved = p.saved + (size_t(row0 / 32) * size_t(p.savedCols) + size_t(n0 / 32)) * (kSavedBlock / 16); }
      if constexpr (EPI == kGateGrad) {
        saved = p.saved + (size_t(row0 / 32) * size_t(p.savedCols) + size_t(n0 / 16)) * (kSavedBlock / 16);
        if (nChunks > 0) loadSaved(saved, lane, z);                     // on the way while the tile's last MMAs run
      }
      ok = tc::mbarWait(tmemFullBar(group), uses & 1, abortWord, p.timeoutNs);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) { if (lane == 0) skinny::recordTimeout(p.status, 5, item.tile, group); break; }
      ++uses;
      tc::fenceAfterThreadSync();
      const uint32_t taddr = tmemBase + (uint32_t(quarter * 32) << 16) + uint32_t(group) * kAccStride;
      auto stagingTile = [&]() {                                        // a tile whose last TMA store has read it
        const uint32_t buf = stagingWarp + (tileCount++ % uint32_t(kStageTiles)) * kStageTileBytes;
        if (lane == 0) tc::bulkWaitGroupRead<kStageTiles - 1>();
        __syncwarp();
        return buf;
      };
      auto put = [&](uint32_t buf, int piece, const uint32_t* o) {      // 8 columns of this lane's row
        tc::stShared16(buf + rowAddr + (uint32_t(piece) ^ swz) * 16u, o[0], o[1], o[2], o[3]);
      };
      auto drain = [&](uint32_t buf, int col) {                         // columns and rows past the output are clipped
        tc::fenceProxyAsyncShared();
        __syncwarp();
        if (lane == 0) { tc::tmaStore2d(&maps.c, col, row0, buf); tc::bulkCommitGroup(); }
      };
      if constexpr (EPI == kGateGrad) {
        // 32 columns of dh are 64 of dZ: [16 dG][16 dU][16 dG][16 dU], one staging tile
        const int blocks = min(p.bn, p.N - n0) / 16;                    // saved blocks of this tile (N is a multiple of 16)
#pragma unroll 1
        for (int c = 0; c < nChunks; ++c) {
          uint32_t r[32], o[16];
          tc::tmemLoad32(taddr + uint32_t(c * 32), r);
          const uint32_t buf = stagingTile();
          tc::tmemLoadWaitFor(r);
          gateGrad<0>(p.activation, r, z, o);
          if (2 * c + 1 < blocks) loadSaved(saved + size_t(2 * c + 1) * (kSavedBlock / 16), lane, z);
#pragma unroll
          for (int j = 0; j < 4; ++j) put(buf, j, o + 4 * j);
          if (2 * c + 1 < blocks) gateGrad<16>(p.activation, r, z, o);  // (else these columns are past the output)
          if (2 * c + 2 < blocks) loadSaved(saved + size_t(2 * c + 2) * (kSavedBlock / 16), lane, z);
#pragma unroll
          for (int j = 0; j < 4; ++j) put(buf, 4 + j, o + 4 * j);
          drain(buf, 2 * n0 + c * 64);
        }
      } else {
        constexpr int kOut = EPI == kGate ? 16 : 32, kPerTile = 64 / kOut;      // output columns of a chunk, chunks of a staging tile
        uint32_t ra[32], rb[32];
        if (nChunks > 0) tc::tmemLoad32(taddr, ra);
#pragma unroll 1
        for (int c0 = 0; c0 < nChunks; c0 += kPerTile) {
          const uint32_t buf = stagingTile();
          auto stage = [&](const uint32_t (&r)[32], int c, int slot) {
            uint32_t o[kOut / 2];
            if constexpr (EPI == kGate) {
              if (saved) {
                uint32_t w[24];
                pack24(r, w);
                uint4* to = saved + size_t(c) * (kSavedBlock / 16) + lane;
#pragma unroll
                for (int i = 0; i < kSavedVectors; ++i) __stcs(to + i * 32, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float a0, a1, unused;
                activate(p.activation, __uint_as_float(r[2 * i]), a0, unused);
                activate(p.activation, __uint_as_float(r[2 * i + 1]), a1, unused);
                o[i] = skinny::pack2(a0 * __uint_as_float(r[16 + 2 * i]), a1 * __uint_as_float(r[17 + 2 * i]));
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = skinny::pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
            }
#pragma unroll
            for (int j = 0; j < kOut / 8; ++j) put(buf, slot * (kOut / 8) + j, o + 4 * j);
          };
#pragma unroll
          for (int sl = 0; sl < kPerTile; ++sl) {
            const int c = c0 + sl;
            if (c < nChunks) {
              if (sl % 2 == 0) {
                tc::tmemLoadWaitFor(ra);
                if (c + 1 < nChunks) tc::tmemLoad32(taddr + uint32_t((c + 1) * 32), rb);
                stage(ra, c, sl);
              } else {
                tc::tmemLoadWaitFor(rb);
                if (c + 1 < nChunks) tc::tmemLoad32(taddr + uint32_t((c + 1) * 32), ra);
                stage(rb, c, sl);
              }
            }
          }
          drain(buf, (EPI == kGate ? n0 / 2 : n0) + c0 / kPerTile * 64);
        }
      }
      // hand the accumulator back to the MMA warp (of CTA 0)
      tc::fenceBeforeThreadSync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CTAS == 2) tc::mbarArriveClusterTmem(leaderBars + 8u * uint32_t(2 * kMaxStages + 2 + group));
        else tc::mbarArrive(tmemEmptyBar(group));
      }
    }
    if (lane == 0) tc::bulkWaitGroup<0>();
  }

  if (*abortWord) tc::landingPause();   // copies already in flight land before shared memory and TMEM go away
  tc::fenceBeforeThreadSync();
  if constexpr (CTAS == 2) tc::clusterSync(); else __syncthreads();     // neither CTA frees TMEM the pair's MMA still writes
  if (warp == 1) {
    if constexpr (CTAS == 2) tc::tmemDeallocPair(tmemBase, kTmemCols);
    else tc::tmemDealloc(tmemBase, kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
struct Operand { const void* ptr; int rows, cols; };    // as it lies in memory, row-major bf16

struct Shape { int ctas, accs, bn; };

struct Device { int sms = 0, index = -1; };
bool currentDevice(Device& d) {
  static std::mutex mu;
  static int sms[64] = {};
  if (cudaGetDevice(&d.index) != cudaSuccess || d.index < 0 || d.index >= 64) { setError("feed-forward launch: no current device"); return false; }
  std::lock_guard<std::mutex> lock(mu);
  if (!sms[d.index]) cudaDeviceGetAttribute(&sms[d.index], cudaDevAttrMultiProcessorCount, d.index);
  d.sms = sms[d.index];
  return d.sms > 0;
}

// The tile that is expected to take least. A k-block (64 of k) of a tile takes the longest of its MMAs (bn / 2 cycles per 16 of k and accumulator,
// more where they all go into one accumulator) and its loads from L2 (about 56 bytes a cycle and SM); a tile adds its fill and its epilogue.
Shape chooseShape(int M, int N, int K, int sms, int epi) {
  Shape best{2, 2, 256};
  double least = 1e30;
  const double kBlocks = (K + kBK - 1) / kBK;
  auto consider = [&](Shape s) {
    const int tileRows = kBM * s.ctas * s.accs, units = sms / s.ctas;
    const int64_t tiles = int64_t((M + tileRows - 1) / tileRows) * ((N + s.bn - 1) / s.bn);
    double waves = double((tiles + units - 1) / units);
    const int64_t rest = tiles % units;
    if (s.accs == 2 && tiles > units && rest > 0 && 2 * rest <= units) waves -= 0.5;
    const double rowsOfA = std::min(M, kBM);
    const double mma = 4.0 * s.accs * s.bn / 2 * (s.accs == 2 ? 1.0 : 1.36);
    const double load = (s.accs * rowsOfA + s.bn / s.ctas) * 128.0 / 56;
    const double epilogue = s.bn * (s.accs == 2 ? 16.0 : 8.0) * (epi == kStore ? 1.0 : 2.0);
    const double block = std::max(mma, load);
    // with one accumulator per tile the epilogue hides under the next tile's main loop, but for the last one
    const double cycles = s.accs == 2 ? waves * (kBlocks * block + 1500 + epilogue)
                                      : waves * std::max(kBlocks * block + 500, epilogue) + 1500 + epilogue;
    if (cycles < least) { least = cycles; best = s; }
  };
  consider({2, 2, 256});
  consider({2, 2, 128});
  consider({1, 1, 256});
  consider({1, 1, 128});
  if (epi != kGate) consider({1, 1, 64});     // (64 columns of Z are 32 of h: half a staging tile)
  return best;
}

template <bool A_MN, bool B_MN, int EPI, int CTAS, int ACCS>
int launchAs(const Maps& maps, Params p, const Device& dev, cudaStream_t stream) {
  auto kernel = ffnKernel<A_MN, B_MN, EPI, CTAS, ACCS>;
  // shared-memory opt-in and cluster occupancy belong to the device's copy of the kernel: resolved once per device
  static std::mutex mu;
  static int known[64] = {};
  int units;
  {
    std::lock_guard<std::mutex> lock(mu);
    int& n = known[dev.index];
    if (!n) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit) != cudaSuccess) { setError("cannot opt in to 227 KiB of shared memory"); return 1; }
      n = dev.sms / CTAS;
      if (CTAS == 2) {                  // pairs must sit on SMs of one GPC: ask how many the device can hold at once
        cudaLaunchConfig_t q{};
        cudaLaunchAttribute qa[1];
        qa[0].id = cudaLaunchAttributeClusterDimension; qa[0].val.clusterDim.x = 2; qa[0].val.clusterDim.y = 1; qa[0].val.clusterDim.z = 1;
        q.gridDim = dim3(unsigned(dev.sms / 2 * 2)); q.blockDim = dim3(kThreads); q.dynamicSmemBytes = kSmemLimit; q.attrs = qa; q.numAttrs = 1;
        int m = 0;
        if (cudaOccupancyMaxActiveClusters(&m, kernel, &q) == cudaSuccess && m > 0) n = std::min(n, m);
      }
    }
    units = n;
  }
  const int tiles = p.tilesM * p.tilesN;
  units = std::min(units, tiles);
  p.items = p.fullItems = tiles;
  if (ACCS == 2) {
    // a last wave that fills at most half of the pairs is issued as halves of tiles
    const int rest = tiles % units;
    if (tiles > units && rest > 0 && 2 * rest <= units) { p.fullItems = tiles - rest; p.items = p.fullItems + 2 * rest; }
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = CTAS; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(unsigned(units * CTAS)); cfg.blockDim = dim3(kThreads); cfg.stream = stream;
  cfg.dynamicSmemBytes = size_t(p.stages) * size_t(ACCS * p.aBytes + p.bn / CTAS * kBK * 2) + kStagingBytes + kBarrierBytes + 1024;
  cfg.attrs = attr; cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps, p);
  if (e != cudaSuccess) { setError(std::string("feed-forward launch: ") + cudaGetErrorString(e)); return 1; }
  return 0;
}

// C[M, N] (or the gated forms) = sum over k; an operand is [rows of D, K] row-major, or [K, rows of D] where its _MN is set
template <bool A_MN, bool B_MN, int EPI>
int product(const void* A, const void* B, void* C, int M, int N, int K, void* saved, int activation, uint32_t* status, cudaStream_t stream) {
  Device dev;
  if (!currentDevice(dev)) return 1;
  const Shape s = chooseShape(M, N, K, dev.sms, EPI);
  Params p{};
  p.M = M; p.N = N; p.K = K; p.bn = s.bn;
  const int tileRows = kBM * s.ctas * s.accs;
  p.tilesM = (M + tileRows - 1) / tileRows; p.tilesN = (N + s.bn - 1) / s.bn;
  // Few rows of A (as many as one tile has at most) take only their own room in a stage: the MMA's other rows read what lies behind, and
  // rows of the accumulator that are no rows of D are never stored.
  const int boxRows = A_MN || s.ctas == 2 ? kBM : std::min(kBM, (M + 7) / 8 * 8);
  p.aBytes = boxRows * kBK * 2;
  const int stageBytes = s.accs * p.aBytes + s.bn / s.ctas * kBK * 2;
  p.stages = std::min((kSmemLimit - kBarrierBytes - 1024 - kStagingBytes) / stageBytes, kMaxStages);
  const int outCols = EPI == kGate ? N / 2 : EPI == kGateGrad ? 2 * N : N;
  p.C = static_cast<__nv_bfloat16*>(C); p.ldc = outCols;
  p.saved = static_cast<uint4*>(saved); p.savedCols = EPI == kGate ? N / 32 : N / 16;
  p.activation = activation; p.status = status; p.timeoutNs = 2ull * 1000 * 1000 * 1000;
  Maps maps{};
  auto bf16Map = [](CUtensorMap& m, const void* ptr, int rows, int cols, int boxRows) {
    return makeTensorMap(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, ptr, uint64_t(rows), uint64_t(cols) * 2, uint64_t(cols) * 2, uint32_t(boxRows));
  };
  if (!(A_MN ? bf16Map(maps.a, A, K, M, kBK) : bf16Map(maps.a, A, M, K, boxRows)) ||
      !(B_MN ? bf16Map(maps.b, B, K, N, kBK) : bf16Map(maps.b, B, N, K, s.bn / s.ctas)) || !bf16Map(maps.c, C, M, outCols, 32)) return 1;
  return s.ctas == 2 ? launchAs<A_MN, B_MN, EPI, 2, 2>(maps, p, dev, stream) : launchAs<A_MN, B_MN, EPI, 1, 1>(maps, p, dev, stream);
}

bool sizesFit(int tokens, int hidden, int intermediate, int activation) {
  if (tokens <= 0 || hidden <= 0 || intermediate <= 0) { setError("feed-forward: dimensions must be positive"); return false; }
  if (hidden % 8 || intermediate % 16) { setError("feed-forward: hidden must be a multiple of 8 and intermediate of 16"); return false; }
  if (intermediate > INT32_MAX / 4 || hidden > INT32_MAX / 4 || tokens > INT32_MAX / 4) { setError("feed-forward: dimensions above 2^29"); return false; }
  if (activation != PURLIN_ACT_SILU && activation != PURLIN_ACT_GELU) { setError("feed-forward: unknown activation"); return false; }
  return true;
}

}  // namespace

extern "C" {

size_t purlin_ffn_saved_bytes(int tokens, int intermediate) {
  if (tokens <= 0 || intermediate <= 0) return 0;
  return size_t((tokens + 31) / 32) * size_t(intermediate / 16) * kSavedBlock;
}

int purlin_ffn_forward(const void* x, const void* wGateUp, const void* wDown, void* hOut, void* saved, void* y, int tokens, int hidden,
                       int intermediate, int activation, uint32_t* status, void* stream) {
  NvtxRange range("ffnForward", size_t(tokens) * size_t(hidden) * 2);
  if (!sizesFit(tokens, hidden, intermediate, activation)) return 1;
  if (reinterpret_cast<uintptr_t>(saved) % 16) { setError("feed-forward: the saved pre-activations need 16-byte alignment"); return 1; }
  const int rc = !saved && activation == PURLIN_ACT_SILU
      ? purlin_gemm_bf16(x, wGateUp, hOut, tokens, 2 * intermediate, hidden, PURLIN_EPI_SWIGLU, 0, status, stream)
      : product<false, false, kGate>(x, wGateUp, hOut, tokens, 2 * intermediate, hidden, saved, activation, status, static_cast<cudaStream_t>(stream));
  if (rc || !y) return rc;
  return purlin_gemm_bf16(hOut, wDown, y, tokens, hidden, intermediate, PURLIN_EPI_STORE, 0, status, stream);
}

int purlin_ffn_backward(const void* x, const void* wGateUp, const void* wDown, const void* h, const void* saved, const void* dy, void* dz,
                        void* dx, void* dGateUp, void* dDown, int tokens, int hidden, int intermediate, int activation, uint32_t* status, void* stream) {
  NvtxRange range("ffnBackward", size_t(tokens) * size_t(hidden) * 2);
  if (!sizesFit(tokens, hidden, intermediate, activation)) return 1;
  if (reinterpret_cast<uintptr_t>(saved) % 16) { setError("feed-forward: the saved pre-activations need 16-byte alignment"); return 1; }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc = 0;
  if (dx || dGateUp)
    rc = product<false, true, kGateGrad>(dy, wDown, dz, tokens, intermediate, hidden, const_cast<void*>(saved), activation, status, s);
  if (!rc && dx) rc = product<false, true, kStore>(dz, wGateUp, dx, tokens, hidden, 2 * intermediate, nullptr, activation, status, s);
  if (!rc && dGateUp) rc = product<true, true, kStore>(dz, x, dGateUp, 2 * intermediate, hidden, tokens, nullptr, activation, status, s);
  if (!rc && dDown) rc = product<true, true, kStore>(dy, h, dDown, hidden, intermediate, tokens, nullptr, activation, status, s);
  return rc;
}

}  // extern "C"
