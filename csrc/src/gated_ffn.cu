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
// memory. In bf16 their rounding would be as large an error of dZ as its own (dX against 64 bits by adding roundings as independent: 2.9e-3, and 2.35e-3, as measured,
// without it: 1.66e-3 each for dZ and dX); with h they take the 8 bytes per element of h that separate bf16 tensors of gate, up, act(gate) and h would.
// h and dZ are rounded to bf16 because they are operands of tensor-core products; all sums are fp32 in tensor memory.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>
#include <type_traits>

#include "purlin/ffn_schedule.hpp"
#include "purlin/gated_ffn.h"
#include "purlin/gemm.h"
#include "purlin/gemm_skinny.cuh"
#include "purlin/tc_sm100.cuh"
#include "purlin/telemetry.hpp"
#include "purlin/tensor_map.hpp"
#include "purlin/wait_limit.hpp"

using namespace purlin;
using namespace purlin::ffn;

namespace {

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

// One product. A launch has one, or the three gradients, which need one another as little as their tiles do.
struct alignas(64) Group {
  CUtensorMap a, b, c;
  Tiles t;                               // (with t.split above 1 the sums go to `partial` and finishKernel adds them up)
  int aMn;                               // m is contiguous in A (k otherwise)
  int aBytes;                            // that one block of A brings into a stage: fewer than 128 rows of it where there are fewer
};

struct alignas(64) Params {
  Group g[kMaxGroups];
  Schedule schedule;
  int bn, stages, aBytes;                // aBytes: room of one block of A in a stage
  uint4* saved;                          // pre-activations: written by kGate (unless null), read by kGateGrad
  int savedCols;                         // its 32-column blocks per row block
  int activation;
  float4* partial;                       // of the first group, where its k is split: [part][tile][accumulator, CTA, quarter][32 columns][8][32 lanes]
  uint32_t* status;
  uint64_t timeoutNs;
};

PURLIN_D float sigmoidOf(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
// act(g) = g sigmoid(s(g)): s = g (silu), s = 2 sqrt(2 / pi) (g + 0.044715 g^3) (gelu with the tanh). Past |g| = 16 the sigmoid is 0 or 1
// in fp32, so the cube is taken of the clamped value and cannot overflow.
constexpr float kGeluScale = 1.5957691216057308f, kGeluCube = 0.044715f;
template <int ACT> PURLIN_D void activate(float g, float& act, float& grad) {
  float s = g, ds = 1.f;
  if constexpr (ACT == PURLIN_ACT_GELU) {
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

template <int ACT> PURLIN_D void gate(const uint32_t (&r)[32], uint32_t (&o)[8]) {      // act(gate) * up of 32 columns (16 of each), packed to bf16
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a0, a1, unused;
    activate<ACT>(__uint_as_float(r[2 * i]), a0, unused);
    activate<ACT>(__uint_as_float(r[2 * i + 1]), a1, unused);
    o[i] = skinny::pack2(a0 * __uint_as_float(r[16 + 2 * i]), a1 * __uint_as_float(r[17 + 2 * i]));
  }
}
// dG (o[0..7]) and dU (o[8..15]) of 16 columns, packed to bf16, from dh (columns C0 ... of the 32 in r) and the saved block
template <int ACT, int C0, int J = 0>
PURLIN_D void gateGrad(const uint32_t (&r)[32], const uint32_t (&w)[24], uint32_t (&o)[16]) {
  if constexpr (J < 16) {
    float a0, d0, a1, d1;
    activate<ACT>(unpack24<J>(w), a0, d0);
    activate<ACT>(unpack24<J + 1>(w), a1, d1);
    const float h0 = __uint_as_float(r[C0 + J]), h1 = __uint_as_float(r[C0 + J + 1]);
    o[J / 2] = skinny::pack2(h0 * unpack24<16 + J>(w) * d0, h1 * unpack24<17 + J>(w) * d1);
    o[8 + J / 2] = skinny::pack2(h0 * a0, h1 * a1);
    gateGrad<ACT, C0, J + 2>(r, w, o);
  }
}

// The producing and the issuing warp stay whole, their instructions are predicated on one lane: in a branch of one lane every operand of an
// MMA would have to be moved into uniform registers first.
PURLIN_D uint32_t electOne() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e;
}
PURLIN_D bool waitAll(uint32_t bar, uint32_t parity, volatile int* abortWord, uint64_t timeoutNs) {
  return __all_sync(0xffffffffu, tc::mbarWait(bar, parity, abortWord, timeoutNs)) != 0;
}
template <int CTAS> PURLIN_D void mma(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 2)
    asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
  else
    asm volatile("{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
template <int CTAS> PURLIN_D void commit(uint32_t elected, uint32_t bar) {      // on this barrier of every CTA of the tile
  if constexpr (CTAS == 2)
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t"
                 "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar), "h"(uint16_t(3)), "r"(elected) : "memory");
  else
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(elected) : "memory");
}

constexpr int kPartialBlock = 8 * 32;    // 32 rows x 32 columns of partial sums in 16-byte pieces: eight for every lane (a row), 512 bytes side by side
// CTAS = 2: a cluster of two CTAs owns a tile: each loads its 128 rows of A per accumulator and its half of B's columns, CTA 0 issues one
// 256-row MMA for the pair. ACCS = 2: a tile is two accumulators tall; they share B, and their MMAs alternate (an MMA waits for the one before
// into the same columns). ACCS = 1: tiles alternate between the two accumulators, the epilogue of one runs under the MMAs of the next.
template <bool B_MN, int EPI, int CTAS, int ACCS>
__global__ void __launch_bounds__(kThreads, 1) ffnKernel(const __grid_constant__ Params p) {
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
    tc::tmaPrefetchDescriptor(&p.g[0].a);
    tc::tmaPrefetchDescriptor(&p.g[0].b);
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
  auto groupOf = [&](int i) -> const Tiles& { return p.g[i].t; };
  constexpr bool kAnyA = EPI == kStore;       // A's order goes by the product (k is contiguous in the others)

  if (warp == 0) {
    // ---- TMA producer ----
    const uint32_t elected = electOne();
    uint32_t st = 0, ph = 0;
    forItems<CTAS, ACCS>(p.schedule, p.bn, pairIdx, numPairs, groupOf, [&](const Item& m) {
      const Group& g = p.g[m.group];
      const int aRow = m.row + int(ctaRank) * kBM, bRow = m.col + int(ctaRank) * bnLocal;
      const KRange k = kRangeOf(g.t, m.part);
      const bool aMn = kAnyA && g.aMn;
      const uint32_t bytes = uint32_t(CTAS * (m.count * g.aBytes + bBytes));
      for (int kb = k.begin; kb < k.end; ++kb) {
        const bool ok = waitAll(emptyBar(st), ph ^ 1, abortWord, p.timeoutNs);
        if (!ok) { if (elected) skinny::recordTimeout(p.status, 1, m.tile, kb); return false; }
        if (elected) {
          const uint32_t sA = base + st * stageBytes, sB = sA + uint32_t(ACCS * p.aBytes);
          const uint32_t full = leaderBars + 8u * st;                   // both CTAs' bytes are credited to CTA 0's barrier
          if (CTAS == 1 || ctaRank == 0) tc::mbarExpectTx(fullBar(st), bytes);
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if constexpr (CTAS == 2) tc::tmaLoad2dPair(dst, map, x, y, full);
            else tc::tmaLoad2d(dst, map, x, y, fullBar(st));
          };
#pragma unroll
          for (int a = 0; a < ACCS; ++a) {
            if (a >= m.count) break;
            const int row = aRow + a * CTAS * kBM;
            const uint32_t dst = sA + uint32_t(a * p.aBytes);
            if (aMn) {
              load(dst, &g.a, row, kb * kBK);
              load(dst + kBoxBytes, &g.a, row + 64, kb * kBK);
            } else {
              load(dst, &g.a, kb * kBK, row);
            }
          }
          if constexpr (B_MN) {
            for (int j = 0; j < bnLocal / 64; ++j) load(sB + uint32_t(j * kBoxBytes), &g.b, bRow + 64 * j, kb * kBK);
          } else {
            load(sB, &g.b, kb * kBK, bRow);
          }
        }
        __syncwarp();
        if (++st == uint32_t(p.stages)) { st = 0; ph ^= 1; }
      }
      return true;
    });
  } else if (warp == 1) {
    // ---- MMA issuer (CTA 0 of a pair) ----
    if (ctaRank == 0) {
      const uint32_t elected = electOne();
      const uint32_t bBase = base + uint32_t(ACCS * p.aBytes);
      const uint64_t descB0 = B_MN ? tc::smemDescSw128MnMajor(bBase) : tc::smemDescSw128(bBase);
      constexpr uint32_t kStepK = 2, kStepMn = 128;                     // 16 of k, in units of 16 bytes
      constexpr uint32_t kStepB = B_MN ? kStepMn : kStepK;
      const uint32_t stageStep = stageBytes >> 4, accStep = uint32_t(p.aBytes) >> 4;
      uint32_t st = 0, ph = 0, accIt = 0, use0 = 0, use1 = 0;
      forItems<CTAS, ACCS>(p.schedule, p.bn, pairIdx, numPairs, groupOf, [&](const Item& m) {
        const Group& g = p.g[m.group];
        const KRange range = kRangeOf(g.t, m.part);
        const int a0 = ACCS == 1 ? int(accIt & 1) : 0;
        const bool two = ACCS == 2 && m.count == 2;
        bool ok = waitAll(tmemEmptyBar(a0), ((a0 ? use1 : use0) & 1) ^ 1, abortWord, p.timeoutNs);
        if (ok && two) ok = waitAll(tmemEmptyBar(1), (use1 & 1) ^ 1, abortWord, p.timeoutNs);
        if (!ok) { if (elected) skinny::recordTimeout(p.status, 2, m.tile, 0); return false; }
        const uint32_t d0 = tmemBase + uint32_t(a0) * kAccStride, d1 = tmemBase + kAccStride;
        auto mainLoop = [&](auto both, auto order) {
          constexpr bool aMn = decltype(order)::value;
          constexpr uint32_t kStepA = aMn ? kStepMn : kStepK;
          const uint32_t idesc = tc::instrDescBf16(uint32_t(p.bn), uint32_t(kBM * CTAS)) | (aMn ? tc::kInstrDescAMnMajor : 0u) | (B_MN ? tc::kInstrDescBMnMajor : 0u);
          const uint64_t descA0 = aMn ? tc::smemDescSw128MnMajor(base) : tc::smemDescSw128(base);
          for (int kb = range.begin; kb < range.end; ++kb) {
            ok = waitAll(fullBar(st), ph, abortWord, p.timeoutNs);
            if (!ok) { if (elected) skinny::recordTimeout(p.status, 3, m.tile, kb); return; }
            tc::fenceAfterThreadSync();
            const uint64_t off = uint64_t(st * stageStep), da = descA0 + off, db = descB0 + off;
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              const uint32_t accumulate = uint32_t(kb != range.begin || k != 0);
              mma<CTAS>(elected, d0, da + kStepA * k, db + kStepB * k, idesc, accumulate);
              if constexpr (decltype(both)::value) mma<CTAS>(elected, d1, da + accStep + kStepA * k, db + kStepB * k, idesc, accumulate);
            }
            commit<CTAS>(elected, emptyBar(st));
            if (++st == uint32_t(p.stages)) { st = 0; ph ^= 1; }
          }
        };
        auto inOrder = [&](auto both) {
          if constexpr (kAnyA) { if (g.aMn) mainLoop(both, std::true_type{}); else mainLoop(both, std::false_type{}); }
          else mainLoop(both, std::false_type{});
        };
        if constexpr (ACCS == 2) { if (two) inOrder(std::true_type{}); else inOrder(std::false_type{}); }
        else inOrder(std::false_type{});
        if (!ok) return false;
        commit<CTAS>(elected, tmemFullBar(a0));
        if (a0) ++use1; else ++use0;
        if (two) { commit<CTAS>(elected, tmemFullBar(1)); ++use1; }
        ++accIt;
        return true;
      });
    }
  } else {
    // ---- epilogue: four warps for each accumulator ----
    const int quarter = warp & 3, group = (warp - 2) / 4;               // a warp may only touch TMEM lanes [32 * (warp % 4), +32)
    const uint32_t stagingWarp = stagingAll + uint32_t(warp - 2) * uint32_t(kStageTiles * kStageTileBytes);
    const uint32_t rowAddr = uint32_t(lane) * 128u, swz = uint32_t(lane & 7);
    uint32_t accIt = 0, uses = 0, tileCount = 0;
    forItems<CTAS, ACCS>(p.schedule, p.bn, pairIdx, numPairs, groupOf, [&](const Item& m) {
      const uint32_t number = accIt++;
      if (ACCS == 1 ? int(number & 1) != group : group >= m.count) return true;
      const Group& g = p.g[m.group];
      const int row0 = m.row + ((ACCS == 2 ? group : 0) * CTAS + int(ctaRank)) * kBM + quarter * 32;
      const int n0 = m.col, rowsValid = min(g.t.M - row0, 32);
      // chunks of 32 accumulator columns that hold output
      const int nChunks = rowsValid <= 0 ? 0 : (min(p.bn, g.t.N - n0) + 31) / 32;
      uint4* saved = nullptr;                                           // of this warp's rows and the tile's first columns
      uint32_t z[24], z1[24] = {};
      const int blocks = min(p.bn, g.t.N - n0) / 16;                      // kGateGrad: saved blocks of this tile (N is a multiple of 16)
      if constexpr (EPI == kGate) { if (p.saved) saved = p.saved + (size_t(row0 / 32) * size_t(p.savedCols) + size_t(n0 / 32)) * (kSavedBlock / 16); }
      if constexpr (EPI == kGateGrad) {
        saved = p.saved + (size_t(row0 / 32) * size_t(p.savedCols) + size_t(n0 / 16)) * (kSavedBlock / 16);
        if (nChunks > 0) {                                              // (a warp without rows has no saved blocks)
          loadSaved(saved, lane, z);                                    // on the way while the tile's last MMAs run
          if (blocks > 1) loadSaved(saved + kSavedBlock / 16, lane, z1);
        }
      }
      if (!waitAll(tmemFullBar(group), uses & 1, abortWord, p.timeoutNs)) { if (lane == 0) skinny::recordTimeout(p.status, 5, m.tile, group); return false; }
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
        if (lane == 0) { tc::tmaStore2d(&g.c, col, row0, buf); tc::bulkCommitGroup(); }
      };
      if (EPI == kStore && g.t.split > 1) {
        const size_t block = ((size_t(m.part) * size_t(g.t.tilesM * g.t.tilesN) + size_t(m.tile)) * (ACCS * CTAS) + size_t((m.row / (CTAS * kBM) % ACCS + (ACCS == 2 && m.count == 2 ? group : 0)) * CTAS + int(ctaRank))) * 4 + size_t(quarter);
        float4* to = p.partial + block * size_t(p.bn / 32) * kPartialBlock + lane;
#pragma unroll 1
        for (int c = 0; c < nChunks; ++c) {
          uint32_t r[32];
          tc::tmemLoad32(taddr + uint32_t(c * 32), r);
          tc::tmemLoadWaitFor(r);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            to[size_t(c) * kPartialBlock + i * 32] = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]), __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
        }
      } else if constexpr (EPI == kGateGrad) {
        // 32 columns of dh are 64 of dZ: [16 dG][16 dU][16 dG][16 dU], one staging tile. The saved blocks of the next 32 are on the way meanwhile.
        uint32_t r[32];
        if (nChunks > 0) tc::tmemLoad32(taddr, r);
#pragma unroll 1
        for (int c = 0; c < nChunks; ++c) {
          uint32_t o[32];
          const uint32_t buf = stagingTile();
          tc::tmemLoadWaitFor(r);
          uint32_t (&o0)[16] = *reinterpret_cast<uint32_t (*)[16]>(o), (&o1)[16] = *reinterpret_cast<uint32_t (*)[16]>(o + 16);
          if (p.activation == PURLIN_ACT_GELU) { gateGrad<PURLIN_ACT_GELU, 0>(r, z, o0); gateGrad<PURLIN_ACT_GELU, 16>(r, z1, o1); }
          else { gateGrad<PURLIN_ACT_SILU, 0>(r, z, o0); gateGrad<PURLIN_ACT_SILU, 16>(r, z1, o1); }
          if (c + 1 < nChunks) {
            tc::tmemLoad32(taddr + uint32_t((c + 1) * 32), r);
            loadSaved(saved + size_t(2 * c + 2) * (kSavedBlock / 16), lane, z);
            if (2 * c + 3 < blocks) loadSaved(saved + size_t(2 * c + 3) * (kSavedBlock / 16), lane, z1);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) put(buf, j, o + 4 * j);
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
              if (p.activation == PURLIN_ACT_GELU) gate<PURLIN_ACT_GELU>(r, o); else gate<PURLIN_ACT_SILU>(r, o);
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
      return true;
    });
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

// The parts of a product whose k was split, added in ascending order of k: a warp per 32 rows x 32 columns, a row to a lane, as the epilogue
// laid them down. (A second launch and not the last part's epilogue: one warp adding up sixteen parts takes far longer than all.)
constexpr int kFinishThreads = 256;
__global__ void __launch_bounds__(kFinishThreads) finishKernel(const float4* partial, __nv_bfloat16* out, int M, int N, int split, int tiles, int tilesM, int tilesN,
                                                                int blocksM, int bn, int64_t warps) {
  tc::gridDependencyWait();
  tc::gridLaunchDependents();
  const int lane = threadIdx.x & 31;
  const int64_t w = int64_t(blockIdx.x) * (kFinishThreads / 32) + (threadIdx.x >> 5);
  if (w >= warps) return;
  const int chunks = bn / 32, c = int(w % chunks);
  const int64_t block = w / chunks;                            // tile, then accumulator, CTA and quarter: blocksM blocks of 32 rows
  const int tile = int(block / blocksM), rowBlock = int(block % blocksM);
  Tiles g{};
  g.tilesM = tilesM; g.tilesN = tilesN;
  int mIdx, nIdx;
  tileCoord(g, tile, mIdx, nIdx);
  const int row = (mIdx * blocksM + rowBlock) * 32 + lane, col = nIdx * bn + c * 32;
  if (row - lane >= M || col >= N) return;
  const size_t stride = size_t(tiles) * size_t(blocksM) * size_t(chunks) * kPartialBlock;
  const float4* from = partial + (size_t(block) * size_t(chunks) + size_t(c)) * kPartialBlock + lane;
  float4 sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = __ldcs(from + i * 32);
#pragma unroll 2
  for (int s = 1; s < split; ++s) {
    from += stride;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 v = __ldcs(from + i * 32);
      sum[i].x += v.x; sum[i].y += v.y; sum[i].z += v.z; sum[i].w += v.w;
    }
  }
  if (row >= M) return;
  __nv_bfloat16* to = out + size_t(row) * size_t(N) + col;
#pragma unroll
  for (int i = 0; i < 4; ++i)                                   // (N is a multiple of 8)
    if (col + 8 * i < N)
      *reinterpret_cast<uint4*>(to + 8 * i) = make_uint4(skinny::pack2(sum[2 * i].x, sum[2 * i].y), skinny::pack2(sum[2 * i].z, sum[2 * i].w),
                                                         skinny::pack2(sum[2 * i + 1].x, sum[2 * i + 1].y), skinny::pack2(sum[2 * i + 1].z, sum[2 * i + 1].w));
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
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

template <bool B_MN, int EPI, int CTAS, int ACCS>
int launchAs(Params& p, int groups, const Shape& s, const Device& dev, cudaStream_t stream) {
  auto kernel = ffnKernel<B_MN, EPI, CTAS, ACCS>;
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
  int64_t tiles = 0, kBlocks = 0, longest = 0;
  for (int i = 0; i < groups; ++i) {
    const Sizes z{p.g[i].t.M, p.g[i].t.N, p.g[i].t.K};
    const int tileRows = kBM * CTAS * ACCS;
    p.g[i].t.tilesM = (z.M + tileRows - 1) / tileRows; p.g[i].t.tilesN = (z.N + s.bn - 1) / s.bn;
    if (tilesOf(z, s) * p.g[i].t.split > INT32_MAX / 4) { setError("feed-forward: the product is too large"); return 1; }
    tiles += tilesOf(z, s) * p.g[i].t.split;
    const int64_t each = (int64_t(z.K) + kBK - 1) / kBK;
    kBlocks += tilesOf(z, s) * each;
    longest = std::max(longest, each);
  }
  units = int(std::min<int64_t>(units, tiles));
  p.timeoutNs = waitLimitNs(kBlocks / units + 2 * longest);
  Tiles work[kMaxGroups];
  for (int i = 0; i < groups; ++i) work[i] = p.g[i].t;
  shareOut(p.schedule, work, groups, s, units, EPI);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = CTAS; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(unsigned(units * CTAS)); cfg.blockDim = dim3(kThreads); cfg.stream = stream;
  cfg.dynamicSmemBytes = size_t(p.stages) * size_t(ACCS * p.aBytes + p.bn / CTAS * kBK * 2) + kStagingBytes + kBarrierBytes + 1024;
  cfg.attrs = attr; cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) { setError(std::string("feed-forward launch: ") + cudaGetErrorString(e)); return 1; }
  return 0;
}

// C[M, N] (or the gated forms) = sum over k of A(m, k) B(n, k). A is [M, K] row-major, or [K, M] with aMn; B is [N, K], or [K, N] with B_MN.
struct Product { const void *A, *B; void* C; int M, N, K; bool aMn; };
// A function of the sizes (and of the number of SMs): each thread keeps those of its recent sizes, some microseconds of host time.
Shape shapeOf(const Product* products, int n, const Device& dev, int epi, bool mayCut) {
  struct Known { Sizes z[kMaxGroups]; int n, sms, epi; bool mayCut; Shape s; };
  static thread_local Known recent[64] = {};
  Sizes z[kMaxGroups] = {};
  uint32_t hash = uint32_t(n * 8 + epi * 2 + int(mayCut)) * 2654435761u;
  for (int i = 0; i < n; ++i) {
    z[i] = Sizes{products[i].M, products[i].N, products[i].K};
    hash = (hash ^ uint32_t(z[i].M)) * 2246822519u + uint32_t(z[i].N) * 3266489917u + uint32_t(z[i].K);
  }
  Known& k = recent[hash >> 26];
  bool same = k.n == n && k.sms == dev.sms && k.epi == epi && k.mayCut == mayCut;
  for (int i = 0; i < n; ++i) same = same && k.z[i].M == z[i].M && k.z[i].N == z[i].N && k.z[i].K == z[i].K;
  if (!same) {
    k.s = chooseShape(z, n, dev.sms, epi, mayCut);
    for (int i = 0; i < n; ++i) k.z[i] = z[i];
    k.n = n; k.sms = dev.sms; k.epi = epi; k.mayCut = mayCut;
  }
  return k.s;
}
// `partial`: room for the parts of the first product's k, or null where it is not to be cut
template <bool B_MN, int EPI>
int run(const Product* products, int n, void* saved, void* partial, int activation, uint32_t* status, cudaStream_t stream) {
  Device dev;
  if (!currentDevice(dev)) return 1;
  Params p{};
  const Shape s = shapeOf(products, n, dev, EPI, partial != nullptr);
  p.bn = s.bn;
  p.partial = static_cast<float4*>(partial);
  p.saved = static_cast<uint4*>(saved); p.savedCols = EPI == kGate ? products[0].N / 32 : products[0].N / 16;
  p.activation = activation; p.status = status;
  auto bf16Map = [](CUtensorMap& m, const void* ptr, int rows, int cols, int boxRows) {
    return makeTensorMap(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, ptr, uint64_t(rows), uint64_t(cols) * 2, uint64_t(cols) * 2, uint32_t(boxRows));
  };
  for (int i = 0; i < n; ++i) {
    const Product& q = products[i];
    Group& g = p.g[i];
    g.t.M = q.M; g.t.N = q.N; g.t.K = q.K; g.aMn = q.aMn; g.t.split = i ? 1 : s.split;
    // Few rows of A take only their own room in a stage: the MMA's other rows read what lies behind, and rows of the accumulator that are no
    // rows of the result are never stored.
    const int boxRows = q.aMn || s.ctas == 2 ? kBM : std::min(kBM, (q.M + 7) / 8 * 8);
    g.aBytes = boxRows * kBK * 2;
    p.aBytes = std::max(p.aBytes, g.aBytes);
    const int outCols = EPI == kGate ? q.N / 2 : EPI == kGateGrad ? 2 * q.N : q.N;
    if (!(q.aMn ? bf16Map(g.a, q.A, q.K, q.M, kBK) : bf16Map(g.a, q.A, q.M, q.K, boxRows)) ||
        !(B_MN ? bf16Map(g.b, q.B, q.K, q.N, kBK) : bf16Map(g.b, q.B, q.N, q.K, s.bn / s.ctas)) || !bf16Map(g.c, q.C, q.M, outCols, 32)) return 1;
  }
  const int stageBytes = s.accs * p.aBytes + s.bn / s.ctas * kBK * 2;
  p.stages = std::min((kSmemLimit - kBarrierBytes - 1024 - kStagingBytes) / stageBytes, kMaxStages);
  const int rc = s.accs == 2 ? launchAs<B_MN, EPI, 2, 2>(p, n, s, dev, stream)
               : s.ctas == 2 ? launchAs<B_MN, EPI, 2, 1>(p, n, s, dev, stream) : launchAs<B_MN, EPI, 1, 1>(p, n, s, dev, stream);
  if (rc || s.split == 1) return rc;
  const Group& g = p.g[0];
  const int blocksM = s.ctas * s.accs * 4, tiles = g.t.tilesM * g.t.tilesN;
  const int64_t warps = int64_t(tiles) * blocksM * (s.bn / 32);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(unsigned((warps + kFinishThreads / 32 - 1) / (kFinishThreads / 32))); cfg.blockDim = dim3(kFinishThreads); cfg.stream = stream; cfg.attrs = attr; cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, finishKernel, static_cast<const float4*>(p.partial), static_cast<__nv_bfloat16*>(products[0].C), g.t.M, g.t.N, g.t.split, tiles, g.t.tilesM, g.t.tilesN,
                                           blocksM, s.bn, warps);
  if (e != cudaSuccess) { setError(std::string("feed-forward launch: ") + cudaGetErrorString(e)); return 1; }
  return 0;
}

// the gradients that are wanted, dx first
int gradients(Product (&g)[kMaxGroups], const void* x, const void* wGateUp, const void* h, const void* dy, const void* dz, void* dx, void* dGateUp, void* dDown, int tokens, int hidden,
              int intermediate) {
  int n = 0;
  if (dx) g[n++] = Product{dz, wGateUp, dx, tokens, hidden, 2 * intermediate, false};
  if (dGateUp) g[n++] = Product{dz, x, dGateUp, 2 * intermediate, hidden, tokens, true};
  if (dDown) g[n++] = Product{dy, h, dDown, hidden, intermediate, tokens, true};
  return n;
}

bool sizesFit(int tokens, int hidden, int intermediate, int activation) {
  if (tokens <= 0 || hidden <= 0 || intermediate <= 0) { setError("feed-forward: dimensions must be positive"); return false; }
  if (hidden % 8 || intermediate % 16) { setError("feed-forward: hidden must be a multiple of 8 and intermediate of 16"); return false; }
  if (intermediate > INT32_MAX / 4 || hidden > INT32_MAX / 4 || tokens > INT32_MAX / 4) { setError("feed-forward: dimensions must be below 2^29"); return false; }
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
  if (!x || !wGateUp || !hOut || (y && !wDown)) { setError("feed-forward: an operand is missing"); return 1; }
  const Product up{x, wGateUp, hOut, tokens, 2 * intermediate, hidden, false};
  const int rc = !saved && activation == PURLIN_ACT_SILU
      ? purlin_gemm_bf16(x, wGateUp, hOut, tokens, 2 * intermediate, hidden, PURLIN_EPI_SWIGLU, 0, status, stream)
      : run<false, kGate>(&up, 1, saved, nullptr, activation, status, static_cast<cudaStream_t>(stream));
  if (rc || !y) return rc;
  return purlin_gemm_bf16(hOut, wDown, y, tokens, hidden, intermediate, PURLIN_EPI_STORE, 0, status, stream);
}

int purlin_ffn_backward(const void* x, const void* wGateUp, const void* wDown, const void* h, const void* saved, const void* dy, void* dz,
                        void* dx, void* dGateUp, void* dDown, void* workspace, size_t workspaceBytes, int tokens, int hidden, int intermediate, int activation, uint32_t* status,
                        void* stream) {
  NvtxRange range("ffnBackward", size_t(tokens) * size_t(hidden) * 2);
  if (!sizesFit(tokens, hidden, intermediate, activation)) return 1;
  if ((reinterpret_cast<uintptr_t>(saved) | reinterpret_cast<uintptr_t>(workspace)) % 16) { setError("feed-forward: the saved pre-activations and the workspace need 16-byte alignment"); return 1; }
  if (!dy || ((dx || dGateUp) && (!wDown || !saved || !dz)) || (dx && !wGateUp) || (dGateUp && !x) || (dDown && !h)) { setError("feed-forward: an operand of a gradient is missing"); return 1; }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dx || dGateUp) {
    const Product gradZ{dy, wDown, dz, tokens, intermediate, hidden, false};
    if (run<true, kGateGrad>(&gradZ, 1, const_cast<void*>(saved), nullptr, activation, status, s)) return 1;
  }
  Product grads[kMaxGroups];
  const int n = gradients(grads, x, wGateUp, h, dy, dz, dx, dGateUp, dDown, tokens, hidden, intermediate);
  if (!n) return 0;
  const size_t parts = purlin_ffn_workspace_bytes(tokens, hidden, intermediate, dx != nullptr, dGateUp != nullptr, dDown != nullptr);
  return run<true, kStore>(grads, n, nullptr, parts && workspaceBytes >= parts ? workspace : nullptr, activation, status, s);
}

size_t purlin_ffn_workspace_bytes(int tokens, int hidden, int intermediate, int wantDx, int wantGateUp, int wantDown) {
  Device dev;
  if (!wantDx || tokens <= 0 || hidden <= 0 || intermediate <= 0 || !currentDevice(dev)) return 0;
  Product grads[kMaxGroups];
  void* some = grads;                   // (sizes only)
  const int n = gradients(grads, some, some, some, some, some, some, wantGateUp ? some : nullptr, wantDown ? some : nullptr, tokens, hidden, intermediate);
  return partialBytes(Sizes{grads[0].M, grads[0].N, grads[0].K}, shapeOf(grads, n, dev, kStore, true));
}

}  // extern "C"
