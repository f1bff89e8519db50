// Products of the vocabulary losses on gfx950:
//   logits          Z  = H W^T      (tokens x vocabulary; both operands row by row)
//   hidden gradient dH = G W        (W k-major)
//   weight gradient dW = G^T H      (both operands k-major)
// with the softmax statistics of the logits' columns taken in the first one's epilogue.
//
// 256 x 256 tiles, 8 waves of 128 x 64 in two groups that run one phase apart: while one wave of a
// SIMD issues the MFMAs of a 64-wide K slice from registers, its partner reads its next fragments
// from LDS and moves operands (buffer loads straight into a two-slot LDS ring), so the matrix pipe
// waits for neither. Both operands may be stored row by row (K contiguous) or k-major; a k-major
// slice lies in LDS as four blocks of 64 values by 64 k-rows and is read through transposing LDS
// reads. Sizes need no padding: loads past an operand's rows give 0 by the buffer range, loads past
// K by an offset outside it (row form) or by the range of the slice (k-major), and a wave whose
// whole sub-tile lies outside the result does no MFMA work.
//
// Bound by the matrix pipe under the board's power limit. 8192 tokens x 128256 x 4096 in bf16: logits
// with their statistics and exponentials 6.35 ms (1.36 PFLOP/s), hidden gradient 5.61 (1.53), weight
// gradient 6.54 (1.32); a library's plain products of that size take 6.05, 6.23 and 7.26. Where K is
// short, a tile's first loads and results (5 to 6 us) show: 2047 x 32001 x 2048 0.22 ms (1.21) for the
// logits. Up to 256 tokens it is reading the weight: 5.7 TB/s for one token of 128256 x 4096.
#include "dmuon_amd_internal.h"
#include "head_loss.h"
#include "mfma_tile.h"

#include <type_traits>

namespace dmuon {
namespace {

constexpr int kTile = 256, kSlice = 64, kCus = 256;
constexpr float kInf = __builtin_inff();
// rows of any pitch and bases of any element alignment
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));
typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));

using T = Tile<256, 256, 64, 2, 2, 4>;

// How an operand of R rows by K lies in memory.
//   ROWS      [R][ld], K contiguous
//   KMAJOR    [K][ld], R contiguous
//   G_ROWS    rows of the logit gradient (R tokens, K classes): blocks of 64 classes, [K / 64][ld][64]
//   G_KMAJOR  its columns (R classes, K tokens) in the same blocks, [R / 64][ld][64]
enum Form { ROWS, KMAJOR, G_ROWS, G_KMAJOR };

// One operand's part of the LDS ring: what each wave v of a group moves of a slice, in instructions
// of 8 rows (k-major: k-rows) of 128 bytes. A lane's place in instruction q + 2 is 16 rows further,
// and the swizzle moves its chunk of 8 values by an xor of 4 chunks between even and odd q, so one
// byte offset and one chunk a lane describe them all.
template <Form F>
struct Mover {
  static constexpr bool kKMajor = F == KMAJOR || F == G_KMAJOR;
  const uint16_t* base;                   // what the wave moves of slice 0 starts here, or before it
  long long ld;
  int rows, K, width;                     // rows of the tile inside the operand; KMAJOR: values
  unsigned off;                           // byte offset of this lane's row in instruction 0
  int chunk;                              // first value of its chunk
  char* lds;

  // k-major: this wave's block of 64 values; in row form B's block of 64 rows, or A's rows v * 32 and
  // 128 + v * 32
  __device__ __forceinline__ void init(const uint16_t* X, long long ld_, int r0, int n, int k,
                                       int v, int rows_of_wave, int lane, char* lds_) {
    ld = ld_;
    K = k;
    rows = min(kTile, n - r0);
    width = (n + 7) / 8 * 8 - r0;         // whole chunks: the rows are padded to them
    static_assert(T::CPR == 8 && T::RPI == 8 && T::RPL == 2, "8 rows of 8 chunks an instruction");
    if constexpr (kKMajor) {
      lds = lds_ + v * kSlice * 128;
      chunk = 8 * ((lane & 7) ^ kswz64(lane >> 3));
      if constexpr (F == KMAJOR) {
        base = X + r0;
        off = (unsigned)((lane >> 3) * ld + v * 64) * 2u;
      } else {
        // a block of classes past the last one holds nothing to move
        rows = r0 + 64 * v < n ? 1 : 0;
        base = X + (long long)(r0 / 64 + v) * ld * 64;
        off = (unsigned)(lane >> 3) * 128u;
      }
    } else {
      lds = lds_ + v * rows_of_wave * T::ROWB;
      chunk = 8 * T::slot(lane & 7, lane >> 3);
      const int r = v * rows_of_wave + (lane >> 3);
      if constexpr (F == ROWS) {
        base = X + (long long)r0 * ld;
        off = (unsigned)(r * ld) * 2u;
      } else {
        base = X + (long long)r0 * 64;
        off = (unsigned)r * 128u;
      }
    }
  }
  // N instructions of slice `s` into ring slot `slot`, starting `hi` rows further
  template <int N>
  __device__ __forceinline__ void issue(int s, int slot, int hi) const {
    typedef __attribute__((address_space(3))) void* lds_ptr_t;
    const int k0 = s * kSlice;
    const uint16_t* p = base;
    int bytes;
    unsigned step = 1024u;                // 8 rows of a block of 64
    if constexpr (F == KMAJOR) {
      p += (long long)k0 * ld;
      bytes = (int)(((long long)(min(kSlice, K - k0) - 1) * ld + width) * 2);
      step = 8u * (unsigned)ld * 2u;
    } else if constexpr (F == G_KMAJOR) {
      p += (long long)k0 * 64;
      bytes = rows * min(kSlice, K - k0) * 128;
    } else if constexpr (F == G_ROWS) {
      p += (long long)s * ld * 64;
      bytes = rows * 128;
    } else {
      bytes = (int)(((long long)(rows - 1) * ld + (K + 7) / 8 * 8) * 2);
      step = 8u * (unsigned)ld * 2u;
    }
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(p), (short)0, bytes, 0x00020000);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int c = chunk ^ (32 * (q & 1));
      unsigned o = off + (unsigned)c * 2u + (unsigned)(hi / 8) * step + (unsigned)q * step;
      // a chunk past K in the last slice: an offset outside any range reads 0
      if constexpr (F == ROWS) o = c + k0 >= K ? 0x80000000u : o + (unsigned)k0 * 2u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (lds_ptr_t)(lds + slot * T::STAGE + hi * T::ROWB + q * 1024), 16, o, 0, 0, 0);
    }
  }
};

// 16 x 64 logits of a wave: statistics, and the exponentials (through LDS, so that a store writes
// whole rows of their block of 64 columns) or the logits themselves. acc[y]: columns 16 y ..
template <int MODE>
__device__ __forceinline__ void logits_epilogue(const HeadGemm& a, const f32x4_t (&acc)[4], int i0,
                                                int jw, int lane, char* slab) {
  const int jl = 4 * (lane >> 4), i = i0 + (lane & 15);
  const bool inside = jw + 64 <= a.N;
  const long long block = (long long)(jw / 64) * a.M;    // first row of these columns' block
  const float k = a.scale * kLog2e;       // positive: the largest sum is the largest logit
  f32x4_t z[4];
  float top = -kInf;
#pragma unroll
  for (int y = 0; y < 4; ++y) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // columns past the vocabulary: no maximum, no share of the sum
      z[y][e] = inside || jw + jl + 16 * y + e < a.N ? acc[y][e] : -kInf;
      top = fmaxf(top, z[y][e]);
    }
    if (MODE == HG_LOGITS && i < a.M)
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.Z) + (block + i) * 64 + jl + 16 * y) = z[y] * k;
  }
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  // 2^kExpShift exp(z - m) as one multiply-add and v_exp_f32; a row of -inf throughout sums to 0
  const float m = top * k, from = (top == -kInf ? 0.f : m) - (float)kExpShift;
  float s = 0.f;
#pragma unroll
  for (int y = 0; y < 4; ++y) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      z[y][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[y][e], k, -from));
      s += z[y][e];
    }
    if constexpr (MODE == HG_EXP) {
      const u32x2_t o = {pack2_elt<ELT_F16>(z[y][0], z[y][1]), pack2_elt<ELT_F16>(z[y][2], z[y][3])};
      *reinterpret_cast<u32x2_t*>(slab + (lane & 15) * T::EPN + (jl + 16 * y) * 2) = o;
    }
  }
  s += __shfl_xor(s, 16);
  s += __shfl_xor(s, 32);
  if (lane < 16 && i < a.M)
    a.stats[block + i] = make_float2(m, s * (1.f / (float)(1 << kExpShift)));
  if constexpr (MODE == HG_EXP) {
    const int cr = lane >> 3, cc = lane & 7;
    u32x4_t d[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      d[k] = *reinterpret_cast<const u32x4_t*>(slab + (8 * k + cr) * T::EPN + 16 * cc);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = i0 + 8 * k + cr;
      if (r < a.M)
        __builtin_nontemporal_store(
            d[k], reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.Z) + (block + r) * 64 + 8 * cc));
    }
  }
}

// A wave's 16 XB x 64 values of a gradient: fp32 sums, or the scaled result. 16-bit results pass
// through LDS slab by slab, so that the stores are whole 128-byte row segments.
template <int E, int XB>
__device__ __forceinline__ void grad_epilogue(const HeadGemm& a, f32x4_t (&acc)[XB][4], int iw,
                                              int jw, int lane, char* slab, int split) {
  const int jl = 4 * (lane >> 4);
  const bool whole = a.out && a.splits == 1;
  const float alpha = whole ? a.alpha[0] : 1.f;
  // parts and gathered sums hold the gradient's own scale, whatever shift its values were stored with
  const float up = E == ELT_F16 && a.peak
      ? __uint_as_float((unsigned)(127 + peak_shift(*a.peak)) << 23) : 1.f;
  const bool f32 = !whole || a.out_dtype == DT_F32;
  float* part = a.part + (a.splits > 1 ? (long long)split * a.M * a.ldp : 0);
  float* dst = whole ? static_cast<float*>(a.out) : part;
  // Past the caches where a row's segments are whole lines; parts of lines have to meet in L2 first
  // (48935 x 2088 over 22 tokens: 93 us past it, 43 through it; 128256 x 4096: 205 and 234).
  const bool lines = a.ldo % 64 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 127) == 0;
  const long long ldd = whole ? a.ldo : a.ldp;
#pragma unroll
  for (int x = 0; x < XB; ++x) {
    const int i = iw + 16 * x + (lane & 15);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int j = jw + jl + 16 * y;
      f32x4_t v = acc[x][y];
      if constexpr (E == ELT_F16) v *= up;
      if (a.add_part && i < a.M && j < a.N) {
        const float* p = part + (long long)i * a.ldp + j;
        if (j + 3 < a.N) v += *reinterpret_cast<const f32x4_any_t*>(p);
        else
          for (int e = 0; e < 4; ++e)
            if (j + e < a.N) v[e] += p[e];
      }
      v *= alpha;
      if (f32) {
        if (i >= a.M || j >= a.N) continue;
        float* p = dst + (long long)i * ldd + j;
        if (j + 3 < a.N) *reinterpret_cast<f32x4_any_t*>(p) = v;
        else
          for (int e = 0; e < 4; ++e)
            if (j + e < a.N) p[e] = v[e];
      } else {
        const u32x2_t o = {pack2_elt<E>(v[0], v[1]), pack2_elt<E>(v[2], v[3])};
        *reinterpret_cast<u32x2_t*>(slab + (16 * (x & 1) + (lane & 15)) * T::EPN +
                                    (jl + 16 * y) * 2) = o;
      }
    }
    if (!f32 && (x & 1)) {
      const int cr = lane >> 3, cc = lane & 7;
      u32x4_t d[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        d[k] = *reinterpret_cast<const u32x4_t*>(slab + (8 * k + cr) * T::EPN + 16 * cc);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = iw + 16 * (x - 1) + 8 * k + cr, c = jw + 8 * cc;
        if (r >= a.M || c >= a.N) continue;
        uint16_t* p = static_cast<uint16_t*>(a.out) + (long long)r * a.ldo + c;
        if (c + 7 < a.N) {
          if (lines) __builtin_nontemporal_store(d[k], reinterpret_cast<u32x4_any_t*>(p));
          else *reinterpret_cast<u32x4_any_t*>(p) = d[k];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < a.N) p[e] = (uint16_t)(d[k][e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  }
}

// One tile. Group 0 (waves 0-3) owns tile rows 0-127, group 1 rows 128-255:
//   group 0:  |0 M0 |1 C0 |2 M1 |3 C1 |4 ...         |2KT-1 C(KT-1) |2KT epilogue
//   group 1:  |0    |1 M0 |2 C0 |3 M1 |4 ... M(KT-1) |2KT C(KT-1), epilogue
// M(k): fragments of slice k into registers; C(k): its MFMAs. The refill DMA is issued in memory
// phases: group 0's M(k) starts A of slice k + 1 (its slot's last readers ended at the barrier that
// opened the phase) and waits for it at the end of C(k); group 1's M(k) refills each wave's own B
// block with slice k + 2 after its own reads of it (group 0 read it in the phase before) and waits
// for slice k + 1's B. LIVE false: the wave's sub-tile lies outside the result; it moves operands
// and passes the barriers only.
template <int E, int MODE, Form FA, Form FB, bool LIVE>
__device__ __forceinline__ void head_tile(const HeadGemm& a, char* smem, int bi, int bj, int split) {
  constexpr int KS = kSlice / 32;
  constexpr bool AKM = Mover<FA>::kKMajor, BKM = Mover<FB>::kKMajor;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int grp = wave >> 2, v = wave & 3;
  const int wj = grp == 0 ? 3 - v : v;    // group 1's wave v reads the B block it moves
  const int i0 = bi * kTile, j0 = bj * kTile;

  Mover<FA> ma;
  Mover<FB> mb;
  ma.init(a.A, a.lda, i0, a.M, a.K, v, 32, lane, smem);
  mb.init(a.B, a.ldb, j0, a.N, a.K, v, 64, lane, smem + T::A_BYTES);
  auto issue_a = [&](int s, int slot) {
    if constexpr (AKM) {
      ma.template issue<8>(s, slot, 0);
    } else {
      ma.template issue<4>(s, slot, 0);
      ma.template issue<4>(s, slot, 128);
    }
  };

  f32x4_t acc[8][4];
#pragma unroll
  for (int x = 0; x < 8; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) acc[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  const int arow0 = grp * 128 + (lane & 15), brow0 = wj * 64 + (lane & 15), kq = lane >> 4;
  int kaoff[4], kboff[4];
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    kaoff[y] = AKM ? grp * 2 * kSlice * 128 + kmajor64_lane_off(lane, 16 * y) : 0;
    kboff[y] = BKM ? wj * kSlice * 128 + kmajor64_lane_off(lane, 16 * y) : 0;
  }
  bf16x8_t af[KS][8], bfr[KS][4];
  auto mem_phase = [&](int slot) {
    if constexpr (!LIVE) return;
    const char* sa = smem + slot * T::STAGE;
    const char* sb = sa + T::A_BYTES;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int kc = ks * 4 + kq;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int row = arow0 + x * 16;
        if constexpr (AKM)
          af[ks][x] = read_kmajor(sa + kaoff[x & 3] + (x >> 2) * kSlice * 128 + ks * 32 * 128, 128);
        else
          af[ks][x] = *reinterpret_cast<const bf16x8_t*>(sa + row * T::ROWB + (T::slot(kc, row) << 4));
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int row = brow0 + y * 16;
        if constexpr (BKM)
          bfr[ks][y] = read_kmajor(sb + kboff[y] + ks * 32 * 128, 128);
        else
          bfr[ks][y] = *reinterpret_cast<const bf16x8_t*>(sb + row * T::ROWB + (T::slot(kc, row) << 4));
      }
    }
  };
  auto compute_phase = [&]() {
    if constexpr (!LIVE) return;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int x = 0; x < 8; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = mfma_16x16x32<E>(bfr[ks][y], af[ks][x], acc[x][y]);
  };

  // slices of this split
  const int all = (a.K + kSlice - 1) / kSlice, per = (all + a.splits - 1) / a.splits;
  const int s0 = split * per, KT = min(per, all - s0);
  // Few rows: every tile has rows of B to itself, and starts elsewhere in K. (Rows of a power of two
  // bytes begin on the same memory channel; together the tiles would ask a few channels at a time: 64
  // rows against 128256 columns of 4096 take 185 us, 234 with every tile from 0 on.)
  const int first = a.few && KT > 0 ? (int)(blockIdx.x >> 3) * 5 % KT : 0;
  auto slice = [&](int k) { return s0 + k + first - (k + first >= KT ? KT : 0); };
  if (KT > 0) {
    if (grp == 1) {
      // slices 0 and 1 (past the end: the last slice again, into a slot never read)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        issue_a(slice(min(s, KT - 1)), s);
        mb.template issue<8>(slice(min(s, KT - 1)), s, 0);
      }
      wait_vmcnt<16>();                   // slice 0 has landed
    }
    phase_barrier();
    if (grp == 1) phase_barrier();        // group 1 starts one phase behind
    auto iteration = [&](int kt, auto ra_c, auto rb_c, auto last_c) {
      constexpr bool RA = decltype(ra_c)::value, RB = decltype(rb_c)::value;
      constexpr bool LAST = decltype(last_c)::value;
      mem_phase(kt & 1);
      if (RA && grp == 0) issue_a(slice(kt + 1), (kt + 1) & 1);
      __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): this wave's fragments are in registers
      if (grp == 1) {
        if (RB) {
          mb.template issue<8>(slice(kt + 2), kt & 1, 0);
          wait_vmcnt<8>();                // all of slice kt + 1 has landed
        } else {
          wait_vmcnt<0>();
        }
      }
      phase_barrier();
      compute_phase();
      if (RA && grp == 0) wait_vmcnt<0>();  // slice kt + 1's A has landed
      // the last slice: group 1 stops at the barrier before its MFMAs, which is also the one after
      // group 0's; no wave reads the ring after it
      if (!(LAST && grp == 1)) phase_barrier();
    };
    const std::false_type no{};
    const std::true_type yes{};
    if (KT >= 3) {
      iteration(0, no, yes, no);
      int kt = 1;
      for (; kt + 2 < KT; ++kt) iteration(kt, yes, yes, no);
      iteration(kt, yes, no, no);
      iteration(kt + 1, no, no, yes);
    } else {
      for (int kt = 0; kt + 1 < KT; ++kt) iteration(kt, no, no, no);
      iteration(KT - 1, no, no, yes);
    }
    wait_vmcnt<0>();
  }
  if constexpr (LIVE) {
    const int iw = i0 + grp * 128, jw = j0 + wj * 64;
    char* slab = smem + wave * T::EPI_REGION;
    if constexpr (MODE == HG_GRAD) grad_epilogue<E, 8>(a, acc, iw, jw, lane, slab, split);
    else
#pragma unroll
      for (int x = 0; x < 8; ++x) logits_epilogue<MODE>(a, acc[x], iw + 16 * x, jw, lane, slab);
  }
}

template <int E, int MODE, Form FA, Form FB>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void head_gemm_kernel(const HeadGemm a) {
  __shared__ __attribute__((aligned(16))) char smem[T::LDS_BYTES];
  // groups of 8 tile rows walked column by column, so that the tiles an XCD holds share panels
  const int mt = (a.M + kTile - 1) / kTile, nt = (a.N + kTile - 1) / kTile;
  int t = xcd_remap(blockIdx.x, gridDim.x);
  const int split = t / (mt * nt);
  t -= split * mt * nt;
  const int g = t / (8 * nt), rows = min(mt - 8 * g, 8), r = t - g * 8 * nt;
  const int bi = __builtin_amdgcn_readfirstlane(8 * g + r % rows);
  const int bj = __builtin_amdgcn_readfirstlane(r / rows);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int grp = wave >> 2, v = wave & 3;
  const bool live = bi * kTile + 128 * grp < a.M && bj * kTile + 64 * (grp == 0 ? 3 - v : v) < a.N;
  const int sp = __builtin_amdgcn_readfirstlane(split);
  if (live) head_tile<E, MODE, FA, FB, true>(a, smem, bi, bj, sp);
  else head_tile<E, MODE, FA, FB, false>(a, smem, bi, bj, sp);
}

// out = alpha * sum over the splits, by block `block` of `blocks`. Memory bound: two parts of 2047 x
// 2048 values (42 MB with the result, largely from the caches) 17 us.
__device__ __forceinline__ void join_splits(const HeadGemm& a, int block, int blocks) {
  const long long n = (long long)a.M * a.N;
  const float alpha = a.alpha[0];
  for (long long k = block * 256LL + threadIdx.x; k < n; k += 256LL * blocks) {
    const long long i = k / a.N, j = k - i * a.N, at = i * a.ldo + j;
    float s = 0.f;
#pragma unroll 8
    for (int p = 0; p < a.splits; ++p) s += a.part[((long long)p * a.M + i) * a.ldp + j];
    s *= alpha;
    if (a.out_dtype == DT_F32) static_cast<float*>(a.out)[at] = s;
    else static_cast<uint16_t*>(a.out)[at] = a.out_dtype == DT_F16 ? to_elt<ELT_F16>(s)
                                                                   : to_elt<ELT_BF16>(s);
  }
}

// A weight gradient over few tokens: bound by writing it. 128 x 128 tiles, four waves of 64 x 64, one
// K slice in LDS at a time; three blocks a CU (148 registers) hide each other's waits, where a 256-tile of a slice or
// two waits alone for its first loads and its stores (see weight_is_short). 64 tokens x 128256 x
// 4096: 226 us, 4.7 TB/s. The first `joins` blocks (whole eights, so that the others stay on their
// XCDs) join the hidden gradient's parts, `h`.
template <int E>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3, 4)))
void head_short_kernel(const HeadGemm a, const HeadGemm h, int joins) {
  if ((int)blockIdx.x < joins) return join_splits(h, blockIdx.x, joins);
  constexpr int kSide = 128, kBlock = kSlice * 128;    // LDS bytes of 64 values of a slice
  constexpr int kSlab = 32 * T::EPN;
  static_assert(4 * kSlab <= 4 * kBlock, "results pass through the slices' place");
  __shared__ __attribute__((aligned(16))) char smem[4 * kBlock];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int mt = (a.M + kSide - 1) / kSide, nt = (a.N + kSide - 1) / kSide;
  const int t = xcd_remap(blockIdx.x - joins, gridDim.x - joins);
  const int g = t / (8 * nt), rows = min(mt - 8 * g, 8), r = t - g * 8 * nt;
  const int i0 = __builtin_amdgcn_readfirstlane((8 * g + r % rows) * kSide);
  const int j0 = __builtin_amdgcn_readfirstlane(r / rows * kSide);
  // waves 0 and 1 move the slice's 64-value blocks of A, 2 and 3 those of B
  Mover<G_KMAJOR> ma;
  Mover<KMAJOR> mb;
  ma.init(a.A, a.lda, i0, a.M, a.K, wave & 1, 64, lane, smem);
  mb.init(a.B, a.ldb, j0, a.N, a.K, wave & 1, 64, lane, smem + 2 * kBlock);
  const int wi = wave >> 1, wj = wave & 1;
  f32x4_t acc[4][4];
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) acc[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int KT = (a.K + kSlice - 1) / kSlice;
  for (int s = 0; s < KT; ++s) {
    if (s > 0) __syncthreads();           // the slice before has been read
    if (wave < 2) ma.issue<8>(s, 0, 0);
    else mb.issue<8>(s, 0, 0);
    wait_vmcnt<0>();
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      bf16x8_t af[4], bfr[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int off = kmajor64_lane_off(lane, 16 * x) + ks * 32 * 128;
        af[x] = read_kmajor(smem + wi * kBlock + off, 128);
        bfr[x] = read_kmajor(smem + (2 + wj) * kBlock + off, 128);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = mfma_16x16x32<E>(bfr[y], af[x], acc[x][y]);
    }
  }
  __syncthreads();
  const int iw = i0 + wi * 64, jw = j0 + wj * 64;
  if (iw < a.M && jw < a.N) grad_epilogue<E, 4>(a, acc, iw, jw, lane, smem + wave * kSlab, 0);
}

// Logits of a small call, whose 256-tiles would leave most CUs idle and wait alone on theirs. A block
// takes 16 MB rows by 64 columns, its four waves every fourth 64-wide K step each, straight from
// memory into MFMA operands (a lane's 16 bytes are its operand); the partial sums join through LDS,
// and wave x finishes rows 16 x .. (see head_logits_small). Bound by the latency of its loads and the
// launch: 64 tokens x 8192 x 512 8.4 us, 77 x 1003 x 300 6.8.
template <int E, int MODE, int MB>
__global__ __launch_bounds__(256) void head_small_kernel(const HeadGemm a) {
  __shared__ __attribute__((aligned(16))) f32x4_t part[4][MB * 4][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int i0 = blockIdx.y * 16 * MB, jw = blockIdx.x * 64;
  const int kl = 8 * (lane >> 4);
  // rows past the operands repeat the last one: their results are not used
  const uint16_t *hp[MB], *wp[4];
  f32x4_t acc[MB][4];
#pragma unroll
  for (int x = 0; x < MB; ++x)
    hp[x] = a.A + (long long)min(i0 + 16 * x + (lane & 15), a.M - 1) * a.lda + kl;
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    wp[y] = a.B + (long long)min(jw + 16 * y + (lane & 15), a.N - 1) * a.ldb + kl;
#pragma unroll
    for (int x = 0; x < MB; ++x) acc[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  struct Step {
    bf16x8_t h[2][MB], w[2][4];
  };
  auto load = [&](Step& s, int k0) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int k = k0 + 32 * p;
      const bool in = k + kl < a.K;
#pragma unroll
      for (int y = 0; y < 4; ++y)
        s.w[p][y] = in ? *reinterpret_cast<const bf16x8_t*>(wp[y] + k) : bf16x8_t{};
#pragma unroll
      for (int x = 0; x < MB; ++x)
        s.h[p][x] = in ? *reinterpret_cast<const bf16x8_t*>(hp[x] + k) : bf16x8_t{};
    }
  };
  auto multiply = [&](const Step& s) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int x = 0; x < MB; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = mfma_16x16x32<E>(s.w[p][y], s.h[p][x], acc[x][y]);
  };
  // the blocks start at different steps: see head_tile
  const int n = (a.K + 4 * kSlice - 1) / (4 * kSlice), first = n > 0 ? (int)(blockIdx.x >> 3) % n : 0;
  auto step = [&](int i) {
    const int q = i + first - (i + first >= n ? n : 0);
    return i < n ? (4 * q + wave) * kSlice : a.K;
  };
  Step s[2];
  load(s[0], step(0));
  for (int i = 0; i < n; i += 2) {
    load(s[1], step(i + 1));
    multiply(s[0]);
    load(s[0], step(i + 2));
    multiply(s[1]);
  }
#pragma unroll
  for (int x = 0; x < MB; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) part[wave][4 * x + y][lane] = acc[x][y];
  __syncthreads();
  f32x4_t sum[4];
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    sum[y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (wave < MB)
#pragma unroll
      for (int w = 0; w < 4; ++w) sum[y] += part[w][4 * wave + y][lane];
  }
  __syncthreads();                        // the exponentials' way out lies over the sums
  if (wave < MB && i0 + 16 * wave < a.M)
    logits_epilogue<MODE>(a, sum, i0 + 16 * wave, jw, lane,
                          reinterpret_cast<char*>(part) + wave * 16 * T::EPN);
}

__global__ __launch_bounds__(256) void join_splits_kernel(const HeadGemm a) {
  join_splits(a, blockIdx.x, gridDim.x);
}

long long tiles_of(int M, int N) {
  return ((long long)M + kTile - 1) / kTile * ((N + kTile - 1) / kTile);
}

// Whether a weight gradient [M][N] over K tokens takes the 128-tiles. Measured against the 256-tiles:
// 128256 x 4096 over 64 tokens 226 against 261 us, over 192 316 against 326, over 256 376 against
// 372; 32000 x 2048 (1000 256-tiles) 29 against 38, over 512 73 against 76; 8192 x 512 (64) 5.1
// against 9, over 512 9.7 against 17.
bool weight_is_short(int M, int N, int K) {
  return K <= 192 || (K <= 512 && tiles_of(M, N) <= 4 * kCus);
}

unsigned join_blocks(const HeadGemm& a) {
  const long long n = ((long long)a.M * a.N + 255) / 256;
  return n < 4096 ? (unsigned)((n + 7) / 8 * 8) : 4096u;
}

}  // namespace

bool head_joins_later(const HeadGemm& h, int vocab) {
  return h.splits > 1 && weight_is_short(vocab, h.N, h.M);
}

// Measured against the 256-tiles, in us (K 1024 / 4096): 16 rows 7.5 / 22 against 20 / 63 (4096
// columns), 14 / 56 against 21 / 71 (32768), 213 against 184 (128256 x 4096); 64 rows 10.9 / 32 against
// 20 / 64 (4096), 12 / 42 against 21 / 70 (16384), 21 / 79 against 21 / 72 (32768).
int head_logits_small(int tokens, int vocab) {
  const long long cols = (vocab + 63) / 64;
  if (tokens <= 16) return cols < 4 * kCus ? 1 : 0;
  return (tokens + 63) / 64 * cols <= kCus * 3 / 2 ? 2 : 0;
}

// The least of: waves of tiles on 256 CUs times the slices of a tile, and the join of the parts. In
// units of one slice's time (1.5 us): a tile costs 4 more for its first loads and its results, the
// join 3 for its launch, 0.05 a part and 8 bytes a value and part at 4 TB/s. Within 5% of the best of
// 1 .. 64 parts for 1 .. 2047 tokens of 1000 x 256 .. 128256 x 4096 but for a few of 20 us.
int head_gemm_splits(int M, int N, int K, bool weight) {
  if (weight && weight_is_short(M, N, K)) return 1;
  constexpr int kMost = 64, kLeast = 2;
  const long long tiles = tiles_of(M, N);
  const int slices = (K + kSlice - 1) / kSlice;
  int best = 1;
  double least = 0.;
  for (int s = 1; s <= kMost && s * kLeast <= slices + kLeast - 1; ++s) {
    const int per = (slices + s - 1) / s;
    if (s > 1 && (slices + per - 1) / per != s) continue;      // an empty part
    const double waves = (double)((tiles * s + kCus - 1) / kCus);
    const double cost = waves * (per + 4) + (s > 1 ? 3 + 0.05 * s + 1.3e-6 * s * M * N : 0.);
    if (s == 1 || cost < least) best = s, least = cost;
  }
  return best;
}

hipError_t launch_head_gemm(const HeadGemm& a, hipStream_t stream) {
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  const long long nb = tiles_of(a.M, a.N) * a.splits;
  // 32-bit offsets inside a tile's 256 rows (or a slice's 64), whole 16-byte chunks
  const auto fits = [](const void* p, long long ld, long long width) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && ld >= width && ld < (1 << 22);
  };
  const bool grad = a.mode == HG_GRAD;
  if (a.splits < 1 || nb > 0x7fffffffLL || a.K < 0 ||
      (a.K > 0 && !fits(a.B, a.ldb, a.b_kmajor ? a.N : a.K)) ||
      (a.K > 0 && !grad && !fits(a.A, a.lda, a.K)) ||
      (a.K > 0 && grad && ((reinterpret_cast<uintptr_t>(a.A) & 15) || a.lda < (a.a_kmajor ? a.K : a.M))))
    return hipErrorInvalidValue;
  if (a.splits > 1 && (a.mode != HG_GRAD || !a.out || !a.part || a.add_part))
    return hipErrorInvalidValue;
  if (a.mode == HG_GRAD ? !a.b_kmajor
                        : a.a_kmajor || a.b_kmajor || !a.stats || (a.mode != HG_STATS && !a.Z))
    return hipErrorInvalidValue;
  if (a.small && !grad) {
    const int mb = a.small == 1 ? 16 : 64;
    const dim3 sg((unsigned)((a.N + 63) / 64), (unsigned)((a.M + mb - 1) / mb));
#define DMUON_SMALL(E, MODE)                                                                     \
  do {                                                                                           \
    if (mb == 16) hipLaunchKernelGGL((head_small_kernel<E, MODE, 1>), sg, dim3(256), 0, stream, a); \
    else hipLaunchKernelGGL((head_small_kernel<E, MODE, 4>), sg, dim3(256), 0, stream, a);       \
  } while (0)
    if (a.elt == ELT_F16 && a.mode == HG_STATS) DMUON_SMALL(ELT_F16, HG_STATS);
    else if (a.elt == ELT_F16 && a.mode == HG_LOGITS) DMUON_SMALL(ELT_F16, HG_LOGITS);
    else if (a.elt == ELT_BF16 && a.mode == HG_STATS) DMUON_SMALL(ELT_BF16, HG_STATS);
    else if (a.elt == ELT_BF16 && a.mode == HG_EXP) DMUON_SMALL(ELT_BF16, HG_EXP);
    else return hipErrorInvalidValue;
#undef DMUON_SMALL
    return hipGetLastError();
  }
  if (a.mode == HG_GRAD && a.a_kmajor && a.splits == 1 && weight_is_short(a.M, a.N, a.K)) {
    const long long tiles = ((long long)a.M + 127) / 128 * ((a.N + 127) / 128);
    const unsigned joins = a.join ? join_blocks(*a.join) : 0;
    if (tiles > 0x7fffffffLL - joins) return hipErrorInvalidValue;
    const HeadGemm& h = a.join ? *a.join : a;
    const dim3 tg((unsigned)tiles + joins);
    if (a.elt == ELT_F16)
      hipLaunchKernelGGL(head_short_kernel<ELT_F16>, tg, dim3(256), 0, stream, a, h, (int)joins);
    else
      hipLaunchKernelGGL(head_short_kernel<ELT_BF16>, tg, dim3(256), 0, stream, a, h, (int)joins);
    return hipGetLastError();
  }
  if (a.join) return hipErrorInvalidValue;
  const dim3 grid((unsigned)nb);
#define DMUON_HG(E, MODE, FA, FB) \
  hipLaunchKernelGGL((head_gemm_kernel<E, MODE, FA, FB>), grid, dim3(512), 0, stream, a)
#define DMUON_HG_E(E)                                                     \
  do {                                                                    \
    if (a.mode == HG_STATS) DMUON_HG(E, HG_STATS, ROWS, ROWS);          \
    else if (a.mode == (E == ELT_F16 ? HG_LOGITS : HG_EXP))               \
      DMUON_HG(E, (E == ELT_F16 ? HG_LOGITS : HG_EXP), ROWS, ROWS);       \
    else if (a.mode != HG_GRAD) return hipErrorInvalidValue;              \
    else if (a.a_kmajor) DMUON_HG(E, HG_GRAD, G_KMAJOR, KMAJOR);          \
    else DMUON_HG(E, HG_GRAD, G_ROWS, KMAJOR);                            \
  } while (0)
  if (a.elt == ELT_F16) DMUON_HG_E(ELT_F16);
  else DMUON_HG_E(ELT_BF16);
#undef DMUON_HG_E
#undef DMUON_HG
  if (a.splits > 1 && !a.join_later)
    hipLaunchKernelGGL(join_splits_kernel, dim3(join_blocks(a)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace dmuon
