// Internal declarations of attention over heads. Not part of the public C ABI.
//
// A key head's queries are worked on together: row r of a (sequence, key head) is query r / group of
// query head kvh * group + r % group, so that a tile of rows reads its keys and values once for all the
// query heads that share them, and their gradients sum over those heads in one accumulator.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mfma_tile.h"

namespace dmuon {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// One sequence of a packed call: tokens q0 .. q0 + qn - 1 and k0 .. k0 + kn - 1
struct Sequence {
  int q0, qn, k0, kn;
};

struct Attention {
  const uint16_t* q; const uint16_t* k; const uint16_t* v; const uint16_t* dout;
  uint16_t* out; uint16_t* dq; uint16_t* dk; uint16_t* dv;   // dense [tokens][heads][dim]
  uint16_t* rest;                         // what out's rounding left, rounded itself, or NULL
  float* lse;                             // [tokens][heads], log2 of the row's sum; +inf: sees nothing
  float* delta;                           // [tokens][heads], minus the sum of dout out
  // strides in elements
  long long q_batch, q_token, q_head, k_batch, k_token, k_head, v_batch, v_token, v_head;
  long long do_batch, do_token, do_head;
  const int64_t* kv_lengths;              // [batch] or NULL
  const Sequence* seqs;                   // packed: [batch + 4], the last four the tokens in no sequence
  const int2* q_tiles; const int2* k_tiles;   // packed: (sequence, tile) of each tile
  const int* counts;                      // packed: tiles in q_tiles and in k_tiles
  int batch, heads, kv_heads, group, dim;
  int q_len, kv_len;                      // of a sequence; packed: of all
  int tiles;                              // tiles of one (sequence, key head); packed: of one key head
  int window;                             // 0: none
  int causal, dtype;
  float scale, c;                         // c = scale log2(e)
  int splits;                             // parts of the key axis, joined by a second kernel
  int few;                                // tiles of kFewRows rows, each wave alone
  float* part; float2* part_stats;        // [splits][tokens][heads][dim] sums, [..][2] (reference, sum)
  // gradients: tiles of keys of one (sequence, key head) (packed: of one key head), parts of their rows and
  // [key_splits][key tokens][kv_heads][2][dim] dk and dv of each
  int key_tiles, key_splits;
};

// Where a block works: its sequence's tokens, pointers' offsets and the tile's number
struct Place {
  long long q_off, k_off, v_off, do_off;  // of token 0 of the sequence and the key head's first head
  long long q_row, k_row;                 // tokens before the sequence in dense results
  int qn, kn, kvh, tile, split;
  bool live;
};

// Blocks of one (sequence, key head) follow each other, on one XCD as far as there are several of them:
// its L2 then serves the keys and values. BACK: the tiles of late queries come first, which see most.
template <bool KEYS>
__device__ __forceinline__ Place place_of(const Attention& a, int id, int blocks, bool back) {
  Place p;
  const int splits = KEYS ? a.key_splits : a.splits, tiles = KEYS ? a.key_tiles : a.tiles;
  id = xcd_remap_contig(id, blocks);
  p.split = id % splits;
  id /= splits;
  int t = id % tiles;
  const int unit = id / tiles;
  p.kvh = unit % a.kv_heads;
  const int b = unit / a.kv_heads;
  if (a.seqs) {
    const int n = a.counts[KEYS ? 1 : 0];
    p.live = t < n;
    if (!p.live) return p;
    if (back) t = n - 1 - t;
    const int2 at = (KEYS ? a.k_tiles : a.q_tiles)[t];
    const Sequence s = a.seqs[at.x];
    p.tile = at.y;
    p.qn = s.qn;
    p.kn = s.kn;
    p.q_row = s.q0;
    p.k_row = s.k0;
    p.q_off = s.q0 * a.q_token;
    p.k_off = s.k0 * a.k_token;
    p.v_off = s.k0 * a.v_token;
    p.do_off = s.q0 * a.do_token;
  } else {
    p.live = true;
    p.tile = back ? tiles - 1 - t : t;
    p.qn = a.q_len;
    p.kn = a.kv_len;
    if (a.kv_lengths) {
      const int64_t n = a.kv_lengths[b];
      p.kn = n < 0 ? 0 : n < a.kv_len ? (int)n : a.kv_len;
    }
    p.q_row = (long long)b * a.q_len;
    p.k_row = (long long)b * a.kv_len;
    p.q_off = b * a.q_batch;
    p.k_off = b * a.k_batch;
    p.v_off = b * a.v_batch;
    p.do_off = b * a.do_batch;
  }
  const long long h = (long long)p.kvh * a.group;
  p.q_off += h * a.q_head;
  p.do_off += h * a.do_head;
  p.k_off += p.kvh * a.k_head;
  p.v_off += p.kvh * a.v_head;
  return p;
}

template <int E>
__device__ __forceinline__ f32x16_t mfma_32x32x16(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  if constexpr (E == ELT_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// A tile of rows of D 16-bit values in LDS, row after row; 16-byte chunk c of row r stands at slot
// c ^ slot_mask(r). Two kinds of reads go over it without a bank conflict: the row form of an operand
// (16 consecutive rows at one chunk) and the transposing form (4 consecutive rows, 64 bytes of each).
template <int D>
__device__ __forceinline__ int slot_mask(int r) {
  if constexpr (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);     // two rows share a line of all banks
}

// v_mfma_f32_32x32x16, lane l with h = l / 32: operands hold row (column) l % 32 and the k values
// 8 h .. 8 h + 7 of a step of 16; the result holds column l % 32, and register i row
// 8 (i / 4) + 4 h + i % 4. Registers 8 t .. 8 t + 7 of a result are the k values of step t of an operand
// whose k order is 16 t + 4 h + (0..3), then 8 further: a product's result goes into the next product
// without leaving its lane, where the other operand is read in that order.
__device__ __forceinline__ int result_row(int i, int h) { return 8 * (i / 4) + 4 * h + i % 4; }

// Byte offset of the row form: row l % 32, k step s at offset ^ 32 s
template <int D>
__device__ __forceinline__ int row_form(int lane) {
  const int r = lane & 31;
  return r * D * 2 + (((lane >> 5) ^ slot_mask<D>(r)) << 4);
}
// Byte offset of the transposing form: values 32 b .. 32 b + 31 of the rows in the order above at
// offset ^ 64 b, and their second four (offset ^ 32) + 8 rows
template <int D>
__device__ __forceinline__ int turned_form(int lane) {
  const int s = lane & 15, g = lane >> 4, r = 4 * (g >> 1) + (s >> 2);
  return r * D * 2 + (((2 * (g & 1) + ((s & 3) >> 1)) ^ slot_mask<D>(r)) << 4) + (s & 1) * 8;
}
template <int D>
__device__ __forceinline__ bf16x8_t read_turned(const char* lds, int at) {
  typedef __attribute__((address_space(3))) s16x4_t* lds_s4_t;
  const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)(lds + at));
  const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t)(lds + (at ^ 32) + 16 * D));
  return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A result's 32 rows (keys, or queries' rows) from `at` on, of which those under `end` or from `begin` on stay and
// the others become `off`: a comparison with a constant and a selection a value.
__device__ __forceinline__ void cut_end(f32x16_t& s, int at, int end, int h, float off) {
  const int stay = end - at - 4 * h;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = result_row(i, 0) < stay ? s[i] : off;
}
__device__ __forceinline__ void cut_begin(f32x16_t& s, int at, int begin, int h, float off) {
  const int stay = begin - at - 4 * h;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = result_row(i, 0) >= stay ? s[i] : off;
}

// Registers from .. from + 7 of a result, rounded: one k step of the next product's operand
template <int E>
__device__ __forceinline__ bf16x8_t pack8(const f32x16_t& v, int from) {
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2_elt<E>(v[from + 2 * i], v[from + 2 * i + 1]);
  return __builtin_bit_cast(bf16x8_t, w);
}

constexpr unsigned kNowhere = 0x80000000u;     // outside any buffer range: reads 0

// Loads of a wave that works alone are of use to no other: not temporal (the loads' second policy bit).
// 48 x 1 token over up to 8192 keys: 181 -> 165 us.
constexpr int kPastCaches = 2;

// Moves ROWS rows of one pitch from memory into LDS, WAVES waves together. The swizzle repeats after four
// instructions of a wave, so four offsets describe them all.
template <int D, int ROWS, int WAVES>
struct TileMover {
  static constexpr int CPR = D / 8, RPI = 64 / CPR, N = ROWS / RPI / WAVES, PART = N < 4 ? N : 4;
  static_assert(N * RPI * WAVES == ROWS && (N <= 4 || (WAVES == 1 && N % 4 == 0)), "whole instructions");
  unsigned off[4];                        // [PART] makes clang drop the host stubs of the kernels
  int wave;
  __device__ __forceinline__ void init(long long pitch, int dim, int wave_, int lane) {
    wave = wave_;
#pragma unroll
    for (int i = 0; i < PART; ++i) {
      const int r = (wave * N + i) * RPI + lane / CPR;
      const int chunk = (lane % CPR) ^ slot_mask<D>(r);
      off[i] = chunk * 8 < dim ? (unsigned)(r * (int)pitch * 2 + chunk * 16) : kNowhere;
    }
  }
  // rows p .. of which `rows` > 0 are there: the rest reads 0
  __device__ __forceinline__ void issue(const uint16_t* p, long long pitch, int dim, int rows,
                                        char* lds) const {
    typedef __attribute__((address_space(3))) void* lds_ptr_t;
    constexpr int STEP = N > 4 ? 4 * RPI : ROWS;          // rows of a resource
#pragma unroll
    for (int part = 0; part < N / PART; ++part) {
      const int left = rows - part * STEP;
      const int bytes = left > 0 ? (((left < STEP ? left : STEP) - 1) * (int)pitch + dim) * 2 : 0;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint16_t*>(p + part * STEP * pitch), (short)0, bytes, 0x00020000);
#pragma unroll
      for (int i = 0; i < PART; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(lds + (wave * N + part * 4 + i) * 1024), 16,
                                                 off[i], 0, 0, WAVES == 1 ? kPastCaches : 0);
    }
  }
};

// The value of the other half of the wave's lanes (lane ^ 32) joined to this lane's
__device__ __forceinline__ float half_max(float x) {
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// What a query sees of the keys: lo .. hi - 1
struct Sight {
  int lo, hi;
};
__device__ __forceinline__ Sight sight_of(const Attention& a, const Place& p, int query) {
  Sight s = {0, p.kn};
  if (a.causal) {
    const int last = query + p.kn - p.qn;
    s.hi = last + 1 < p.kn ? last + 1 : p.kn;
    if (a.window && last - a.window + 1 > 0) s.lo = last - a.window + 1;
  }
  return s;
}

// What any of the 32 rows from `first` on sees: a wave passes over the other tiles of its block.
__device__ __forceinline__ Sight wave_sight(const Attention& a, const Place& p, int first, int rows) {
  if (first >= rows) return Sight{0, 0};
  const int last = first + 31 < rows ? first + 31 : rows - 1;
  return Sight{sight_of(a, p, first / a.group).lo, sight_of(a, p, last / a.group).hi};
}

constexpr float kLog2e = 1.44269504088896340736f;

// rows and keys of a block's tile; rows of one wave that works alone
constexpr int kQueryRows = 128, kKeyRows = 128, kFewRows = 32;
// the tables of a packed call; tiles of `rows` rows
hipError_t launch_attention_tables(const Attention& a, const int64_t* q_starts, const int64_t* kv_starts,
                                   int q_rows, int k_rows, Sequence* seqs, int2* q_tiles, int2* k_tiles,
                                   int* counts, hipStream_t stream);
hipError_t launch_attention(const Attention& a, hipStream_t stream);
hipError_t launch_attention_grad(const Attention& a, hipStream_t stream);

}  // namespace dmuon
