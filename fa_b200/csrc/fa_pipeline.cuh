// fa_pipeline.cuh -- what the dense attention kernels (fa_kernel.cuh, where the
// pipeline is described) and the paged chunk kernel (paged_chunk.cu) share:
// tile sizes, roles, register split, tensor and shared memory, barriers,
// descriptors, and the softmax's row helpers.
#pragma once
#include <cstdint>
#include "ptx.cuh"

namespace b200fa {

constexpr int kBlockM = 128;    // query rows per unit (per CTA)
constexpr int kBlockN = 128;    // keys per KV block
constexpr int kHeadDim = 128;   // head dimension (fixed)
constexpr int kPairKeys = kBlockN / 2;    // K rows of a block held by each CTA
constexpr int kPairDims = kHeadDim / 2;   // V head-dim columns held by each CTA
constexpr int kItemUnits = 2;   // query units per work item (one per CTA)
constexpr int kRing = 5;        // entries of the K ring and of the V ring (one stage each)
constexpr int kQTileBytes = kBlockM * kHeadDim * 2;   // 32 KiB
constexpr int kQHalfBytes = kQTileBytes / 2;          // TMA box: 64 cols x 128 rows
constexpr int kKBoxRows = kPairKeys;                  // K rows of a block held by each CTA
constexpr int kKBoxBytes = kKBoxRows * 128;           // TMA box: 64 cols x 64 rows
constexpr int kStageBytes = 2 * kKBoxBytes;           // 16 KiB
static_assert(kBlockN * kPairDims * 2 == kStageBytes, "K and V stages must have the same size");
constexpr int kThreads = 384;      // 3 warpgroups
constexpr int kSIssuerWarp = 8;    // rank 0: issues every S product
constexpr int kLoadWarp = 9;
constexpr int kPVIssuerWarp = 10;  // rank 0: issues every PV product
constexpr int kForwardWarp = 11;   // rank 1
// Register split (setmaxnreg): launch 384 x 168 = 64512; softmax warpgroups
// 256 x 208 + warpgroup 2 128 x 88 = 64512.  ptxas holds each region to its
// share (both build flavours compile spill-free at this split).
#ifndef B200FA_SOFTMAX_REGS
#define B200FA_SOFTMAX_REGS 208
#endif
constexpr uint32_t kLaunchRegs = 168;
constexpr uint32_t kSoftmaxRegs = B200FA_SOFTMAX_REGS;
constexpr uint32_t kControlRegs = (kThreads * kLaunchRegs - 256 * kSoftmaxRegs) / 128 / 8 * 8;
static_assert(256 * kSoftmaxRegs + 128 * kControlRegs <= kThreads * kLaunchRegs, "register split exceeds the launch budget");
constexpr float kRescaleLog2 = 8.0f;  // lazy-rescale threshold (factor 256)

// Tensor memory columns.
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 0;       // O, 128 columns
constexpr uint32_t kTmemP = 128;     // + 64 b: P buffer b (FP16 pairs, 64 columns)
constexpr uint32_t kTmemS = 256;     // + 128 b: S buffer b (FP32, 128 columns)
static_assert(kTmemS + 2 * 128 <= kTmemCols, "TMEM budget");

// Barrier slots.  "rank 0" barriers are only waited on in rank 0.
constexpr int kBarQFull = 0;     // [2] Q tile landed (rank 0: own TMA + rank 1's forward; rank 1: own TMA)
constexpr int kBarQEmpty = 2;    // [2] Q tile free (the epilogue's store read it)                local
constexpr int kBarSFull = 4;     // [2] S buffer b computed                    (S issuer commit to both CTAs)
constexpr int kBarSFree = 6;     // [2] rank 0: S buffer b read by one group's 4 warps in each CTA
constexpr int kBarPFull = 8;     // [2] rank 0: P buffer b written by one group's 4 warps in each CTA
constexpr int kBarPVDone = 10;   // [2] PV of P buffer b done; O holds every block so far (PV issuer commit)
constexpr int kBarRef = 12;      // [2] reference maximum of block g published (g % 2; 4 warps)  local
constexpr int kBarXchg = 14;     // [1] epilogue row-sum exchange (8 warps)                        local
constexpr int kBarOStaged = 15;  // [1] O tile staged in smem (8 warps)                            local
constexpr int kBarDrain = 16;    // [2] rank 0: MMA drain of the S / PV issuer at exit
constexpr int kBarKFull = 18;    // [kRing] K stage landed (rank 0: own TMA + rank 1's forward)
constexpr int kBarKEmpty = kBarKFull + kRing;   // [kRing] S of its block done (S issuer commit to both CTAs)
constexpr int kBarVFull = kBarKEmpty + kRing;   // [kRing] V stage landed (rank 0: own TMA + rank 1's forward)
constexpr int kBarVEmpty = kBarVFull + kRing;   // [kRing] PV of its block done (PV issuer commit to both CTAs)
constexpr int kNumBars = kBarVEmpty + kRing;
constexpr uint32_t kGroupWarps = 8;  // one group's warps in the pair (arrivals on "S free" / "P full")

constexpr int kSmemQ = 0;
constexpr int kSmemK = 2 * kQTileBytes;
constexpr int kSmemV = kSmemK + kRing * kStageBytes;
constexpr int kSmemBar = kSmemV + kRing * kStageBytes;
constexpr int kSmemXchg = kSmemBar + kNumBars * 8;        // float [2][128] reference / row-sum exchange
constexpr int kSmemMisc = kSmemXchg + 2 * kBlockM * 4;    // TMEM base, abort flag, 6 block counters
constexpr int kSmemUsed = kSmemMisc + 8 + 4 * 6 + 8;  // + start time (trace)
constexpr int kSmemBytes = kSmemUsed + 1024;  // + slack for 1024-B alignment
static_assert(kSmemBytes <= 232448, "shared memory budget exceeded");
static_assert(kSmemBar % 8 == 0, "mbarrier alignment");
static_assert(kKBoxBytes % 1024 == 0 && kStageBytes % 1024 == 0, "128-byte swizzle atoms must stay 1024-B aligned");

// tcgen05 instruction descriptors, kind::f16 (PTX ISA "Instruction
// descriptor"): bits 4-5 D format (1 = F32), 7-9 A format (0 = F16),
// 10-12 B format (0 = F16), 15 A major (0 = K), 16 B major (1 = MN),
// 17-22 N>>3, 24-28 M>>4.  M = 256: the pair's rows; N = 128 for both
// products (S: the block's keys, 64 per CTA; PV: the head dims, 64 per CTA).
constexpr uint32_t kIdescQK = (1u << 4) | (uint32_t(kBlockN >> 3) << 17) | (uint32_t(256 >> 4) << 24);
constexpr uint32_t kIdescPV = (1u << 4) | (1u << 16) | (uint32_t(kHeadDim >> 3) << 17) | (uint32_t(256 >> 4) << 24);
static_assert(kBlockN % 16 == 0 && kBlockN <= 256, "M=256 needs N a multiple of 16");

// Shared-memory matrix descriptors (PTX ISA "Matrix Descriptor"), 128-byte
// swizzle, sm_100 version bit.  Low word: start address >> 4 (bits 0-13),
// leading byte offset >> 4 (bits 16-29).  High word: stride byte offset >> 4
// (bits 0-13), version 1 (bit 14), layout SWIZZLE_128B = 2 (bits 29-31).
// Rows of 128 B, 8-row groups 1024 B apart (SBO) for Q, K (K-major) and V
// (MN-major: rows are keys, 64 head-dim columns per row).  The leading
// offset is unused: swizzled K-major layouts ignore it and each CTA's V
// half is a single 64-column block; it is set to 16 B.  Offsets added to a
// descriptor's start address never carry out of bits 0-13: shared addresses
// are below 256 KiB.
constexpr uint32_t kDescHi = uint32_t(1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr) {
  return (uint64_t(kDescHi) << 32) | uint64_t(((saddr & 0x3FFFFu) >> 4) | (1u << 16));
}

constexpr uint32_t kDevTimeout = 1u;

// The CTA counts its key blocks over all its items: block g has its K in K
// ring entry g % kRing, its V in V ring entry g % kRing (the (g / kRing)-th
// use of each), its scores in S buffer g % 2 and its P in P buffer g % 2.
__device__ __forceinline__ uint32_t ring_entry(uint32_t g) { return g % kRing; }
__device__ __forceinline__ uint32_t ring_parity(uint32_t g) { return (g / kRing) & 1u; }
__device__ __forceinline__ uint32_t buf(uint32_t g) { return g & 1u; }
__device__ __forceinline__ uint32_t buf_parity(uint32_t g) { return (g >> 1) & 1u; }

// Row maximum of 64 scores: 3-input max, four independent chains.
__device__ __forceinline__ float row_max64(const uint32_t* r) {
  float mc0 = -INFINITY, mc1 = -INFINITY, mc2 = -INFINITY, mc3 = -INFINITY;
#pragma unroll
  for (int i = 0; i < 64; i += 8) {
    mc0 = max3(mc0, __uint_as_float(r[i + 0]), __uint_as_float(r[i + 1]));
    mc1 = max3(mc1, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
    mc2 = max3(mc2, __uint_as_float(r[i + 4]), __uint_as_float(r[i + 5]));
    mc3 = max3(mc3, __uint_as_float(r[i + 6]), __uint_as_float(r[i + 7]));
  }
  return fmaxf(fmaxf(mc0, mc1), fmaxf(mc2, mc3));
}

// Bits 0 .. x-1 of a word (none for x <= 0, all for x >= 32).
__device__ __forceinline__ uint32_t bits_below(int x) {
  return x <= 0 ? 0u : x >= 32 ? 0xffffffffu : (1u << x) - 1u;
}

// O row of this thread (128 FP32 columns in TMEM) times `f`, in place.
__device__ __forceinline__ void scale_o_row(uint32_t tO, float f) {
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t o[32];
    tmem_ld32(tO + 32u * uint32_t(c), o);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
    tmem_st32(tO + 32u * uint32_t(c), o);
  }
  tmem_wait_st();
}

}  // namespace b200fa
