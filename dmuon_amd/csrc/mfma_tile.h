// Pieces of the gfx950 MFMA product kernels that every family of them uses: 16-bit element types,
// the matrix instruction, LDS tile layouts and their swizzles, waits and barriers, and the order in
// which an XCD's blocks take tiles.
#pragma once

#include "dmuon_amd_internal.h"

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

namespace dmuon {

__device__ __forceinline__ uint16_t f2bf(float f) {
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}
__device__ __forceinline__ float bf2f(uint16_t h) {
  return __uint_as_float(static_cast<uint32_t>(h) << 16);
}

// Operand / intermediate element type of one kernel instance: E = ELT_BF16 or ELT_F16. The
// product operands, the addend C and the outputs D / D^T are 16-bit words of that type; the
// accumulators are fp32 either way (round to nearest even on the way out).
template <int E>
__device__ __forceinline__ uint16_t to_elt(float f) {
  if constexpr (E == ELT_F16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  else return f2bf(f);
}
template <int E>
__device__ __forceinline__ float from_elt(uint16_t h) {
  if constexpr (E == ELT_F16) return static_cast<float>(__builtin_bit_cast(_Float16, h));
  else return bf2f(h);
}
// Two values rounded (nearest even) to E and packed, low half first: one packed convert
// instruction on gfx950 instead of two converts and a pack.
template <int E>
__device__ __forceinline__ unsigned pack2_elt(float lo, float hi) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  if constexpr (E == ELT_F16) {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2_t{lo, hi}, f16x2_t));
  } else {
    typedef __bf16 b16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2_t{lo, hi}, b16x2_t));
  }
}
// v_mfma_f32_16x16x32: a lane holds row (l % 16) of both operands at k-chunk l / 16, and four
// consecutive output columns of one row. It gives the same bits as the 32x32x16 form (measured:
// the products accumulate in the same order and round identically), and on MI355X it sustains
// a higher clock under the board's power limit at equal MFMA work (sustained MFMA-only loops:
// 1.90 vs 1.65-1.69 PFLOP/s; with 0.5 KB of fragment reads per 32 KFLOP: 1.70 vs 1.53).
template <int E>
__device__ __forceinline__ f32x4_t mfma_16x16x32(bf16x8_t b, bf16x8_t a, f32x4_t c) {
  if constexpr (E == ELT_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, b),
                                                  __builtin_bit_cast(f16x8_t, a), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0);
}

// k-major operand (stored [K][N], N contiguous): a slice of BK k-rows sits in LDS row by row,
// 16-byte chunk c of row r at slot c ^ kswz(r). ds_read_b64_tr_b16 gives lane i of each 16-lane
// group element i % 4 of the 8 bytes addressed by lane 4j + i / 4 of that group (j = 0..3), so
// when the 16 lanes of group g address rows 8g + s / 4 (s = lane % 16) at values 4 (s % 4) ..
// of a 16-value block, lane i receives the 4 consecutive k of value i -- half of the 16x16x32
// operand; a second read 4 rows further gives the other half. The swizzle spreads the 16 rows
// of one read over all 64 banks (two passes for its 512 bytes).
typedef short s16x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ int kswz(int r) { return 2 * ((r & 3) | (((r >> 3) & 1) << 2)); }
__device__ __forceinline__ bf16x8_t read_kmajor(const char* p, int row_bytes) {
  typedef __attribute__((address_space(3))) s16x4_t* lds_s4_t;
  const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)(p));
  const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)(p + 4 * row_bytes));
  return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// The ping-pong kernel keeps a k-major B tile as four column blocks of 64 values, BK rows of
// 128 bytes each; rows r and r + 1 share a 256-byte bank line, so the swizzle of a read's 16
// rows (two passes) comes from row bits 1 and 3.
__device__ __forceinline__ int kswz64(int r) { return 2 * (((r >> 1) & 1) | (((r >> 3) & 1) << 1)); }
__device__ __forceinline__ int kmajor64_lane_off(int lane, int n0) {
  const int s16 = lane & 15, g = lane >> 4;
  const int h = 2 * (((s16 >> 3) & 1) | ((g & 1) << 1));   // kswz64 of every row this lane reads
  const int chunk = ((n0 / 8) ^ h) | ((s16 & 3) >> 1);
  return (8 * g + (s16 >> 2)) * 128 + chunk * 16 + (s16 & 1) * 8;
}
// byte offset, within a k-major slice of `row_bytes`-wide rows, of what lane (s = lane % 16,
// g = lane / 16) addresses for the 16-value block starting at value n0 (a multiple of 16)
__device__ __forceinline__ int kmajor_lane_off(int lane, int n0, int row_bytes) {
  const int s16 = lane & 15, g = lane >> 4;
  const int h = 2 * ((s16 >> 2) | ((g & 1) << 2));          // kswz of every row this lane reads
  const int chunk = ((n0 / 8) ^ h) | ((s16 & 3) >> 1);
  return (8 * g + (s16 >> 2)) * row_bytes + chunk * 16 + (s16 & 1) * 8;
}

// A wave's accumulators as the epilogue walks them: per 32-row slab x of the wave tile, NQ groups
// of four values -- group q of a lane holds slab row row(q), columns col(q) .. col(q) + 3. Indices
// are compile-time after unrolling, so the registers are addressed statically.
template <int BI, int BJ>            // BI x BJ blocks of 16x16 (v_mfma_f32_16x16x32)
struct Acc16 {
  static constexpr int SLABS = BI / 2, NQ = 2 * BJ;
  f32x4_t (&acc)[BI][BJ];
  int lane;
  __device__ __forceinline__ int row(int q) const { return 16 * (q / BJ) + (lane & 15); }
  __device__ __forceinline__ int col(int q) const { return 16 * (q % BJ) + 4 * (lane >> 4); }
  __device__ __forceinline__ float val(int x, int q, int e) const { return acc[2 * x + q / BJ][q % BJ][e]; }
};

// Maps the hardware block id (blocks are dealt round-robin over the 8 XCDs) to a logical tile.
// The logical tiles go in windows of 8 x kXcdWindow, one run of kXcdWindow consecutive tiles
// per XCD: with a window of one tile per CU (gfx950: 8 XCDs x 32 CUs), the blocks resident at
// any time cover one contiguous stretch of the tile order, so all XCDs work on the same few
// matrices and the operand panels one XCD's L2 misses bring into the shared Infinity Cache serve
// the others (c5 step 299.0 -> 291.9 ms, NT 50.0 -> 51.3% of peak, same box), while each XCD's
// own run keeps the neighbouring tiles that share panels in its L2. (Whole contiguous ranges per
// XCD, every XCD on its own matrices, and windows of 8, 16, 24, 48 or 64 tiles per XCD were
// slower.) The last partial window falls back to contiguous ranges of its remainder.
__host__ __device__ __forceinline__ int xcd_remap_contig(int b, int nb) {
  const int q = nb >> 3, r = nb & 7;
  const int x = b & 7, idx = b >> 3;
  const int base = (x < r) ? x * (q + 1) : r * (q + 1) + (x - r) * q;
  return base + idx;
}
constexpr int kXcdWindow = 32;
__host__ __device__ __forceinline__ int xcd_remap(int b, int nb) {
  constexpr int W = kXcdWindow, WW = 8 * kXcdWindow;
  const int x = b & 7, idx = b >> 3;
  const int full = nb / WW;
  if (idx < full * W) return (idx / W) * WW + x * W + idx % W;
  return full * WW + xcd_remap_contig(b - full * WW, nb - full * WW);
}

template <int BM_, int BN_, int BK_, int S_, int WM_, int WN_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, BK = BK_, S = S_, WM = WM_, WN = WN_;
  static constexpr int NW = WM * WN;              // waves per block
  static constexpr int NT = 64 * NW;              // threads per block
  static constexpr int WTM = BM / WM, WTN = BN / WN;  // wave sub-tile
  static constexpr int TI = WTM / 32;             // MFMA blocks along i per wave
  static constexpr int TJ = WTN / 32;             // MFMA blocks along j per wave
  static constexpr int ROWB = BK * 2;             // bytes of one tile row in LDS
  static constexpr int CPR = BK / 8;              // 16-byte chunks per row
  static constexpr int RPI = 1024 / ROWB;         // rows filled by one DMA wave instruction
  static constexpr int A_INST = BM / RPI / NW;    // DMA instructions per wave per slice
  static constexpr int B_INST = BN / RPI / NW;
  static constexpr int LPT = A_INST + B_INST;     // outstanding loads a slice adds per wave
  static constexpr int RPL = 256 / ROWB;          // rows per 256-byte LDS bank line (64 banks)
  static constexpr int A_BYTES = BM * ROWB;
  static constexpr int STAGE = (BM + BN) * ROWB;
  // epilogue staging per wave: one 32-row slab row-major at pitch EPN (WTN values + 16 B: rows
  // stay 16-byte aligned for the 16-byte reads of the stores), two slabs transposed at pitch EPT
  // (64 values + 16 B: the four lane groups of a scatter hit different banks), and the fp32 slab
  // of the final step (32 rows of WTN + 4 floats)
  static constexpr int EPN = WTN * 2 + 16;
  static constexpr int EPT = 64 * 2 + 16;
  static constexpr int EPF = 32 * (WTN + 4) * 4;
  static constexpr int EPI_MAX2 = 32 * EPN + WTN * EPT;
  static constexpr int EPI_REGION_RAW = (EPI_MAX2 > EPF ? EPI_MAX2 : EPF);
  static constexpr int EPI_REGION = (EPI_REGION_RAW + 15) / 16 * 16;
  static constexpr int LDS_BYTES = (S * STAGE > NW * EPI_REGION ? S * STAGE : NW * EPI_REGION);
  static_assert(BM % (NW * RPI) == 0 && BN % (NW * RPI) == 0, "tile rows vs DMA rows");
  static_assert(S * LPT <= 63 && S <= 10, "vmcnt range (the prologue has S slices in flight)");
  // LDS slot of 16-byte chunk kc of row r. A ds_read_b128 serves 16 lanes (256 B, all 64
  // banks) per pass; a fragment read has those 16 lanes on 16 consecutive rows at one chunk,
  // so rows sharing a bank line (r % RPL) must take distinct slots along r / RPL.
  static __device__ __forceinline__ int slot(int kc, int r) { return kc ^ ((r / RPL) & (CPR - 1)); }
};

// s_waitcnt vmcnt(N) with expcnt/lgkmcnt left alone (gfx9 encoding: vmcnt[3:0] + vmcnt[5:4] at
// bits 15:14, expcnt bits 6:4 = 7, lgkmcnt bits 11:8 = 15).
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N <= 63, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
}

// Workgroup barrier without the memory fence of __syncthreads (which would also wait for every
// in-flight LDS DMA); the empty asm statements keep the compiler from moving LDS accesses
// across it.
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A barrier that is also a scheduling fence: the compiler treats s_barrier as ordering memory
// accesses only, and would otherwise move arithmetic (the MFMAs of a ping-pong phase) across it.
__device__ __forceinline__ void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <class T>
__device__ __forceinline__ void wait_slices() {
  // wait until slice 0 of the ring has landed: at most S - 1 newer slices (T::LPT loads each)
  // still in flight
  wait_vmcnt<(T::S - 1) * T::LPT>();
}

// End-of-slice meeting point: wait until at most N loads of this wave are in flight (its share
// of the next slice has landed) and all of its LDS reads have returned (its fragments of the
// current slot are in registers), then s_barrier. gfx9 s_waitcnt encoding: vmcnt[3:0] +
// vmcnt[5:4] at bits 15:14, expcnt bits 6:4 = 7 (untouched), lgkmcnt bits 11:8 = 0.
template <int N>
__device__ __forceinline__ void slice_barrier() {
  static_assert(N >= 0 && N <= 63, "vmcnt range");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace dmuon
