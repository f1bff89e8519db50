// The gradients of attention over heads on gfx950. With S = c q k^T, P = exp2(S log2(e) - lse) formed
// anew and delta = sum of do o over a row:
//   dv = P^T do,  dP = do v^T,  dS = P (dP - delta),  dq = scale dS k,  dk = scale dS^T q
// Blocks over keys (dk, dv) and blocks over queries (dq), in one launch, each with its sums in registers:
// seven products where one pass would do with five, but no sums over blocks, so no atomics and one order.
// Where the keys' blocks are few their rows are split, and a second kernel joins the parts in their order.
//
// Bound like the forward pass, by two pipes that hardly overlap: 2 x 8192 causal tokens, 32/8 heads of 128, bf16
// 3.6 ms (1.07 PFLOP/s of the seven products, 0.76 of five; matrix pipe busy 54% of the cycles, vector pipe 39,
// both at once 15); 16384 packed tokens in 23 documents 0.62 ms; 8191 tokens of 16 heads of 64 in a window of
// 1024 in fp16 172 us (33%, 58, 15). The key blocks' sums (dk and dv of 32 keys a wave) and operands take 192 of
// 256 registers; a third of what they read from LDS is turned on the way (transposing reads).
//
// P and dS are rounded to the operands' type between the products. In fp16 they are held times powers of
// two: P times 2^10 (a long row's probabilities are under the type's normal range) and dS by one that follows
// the largest dS so far of a row (blocks over queries) or of a key (blocks over keys), so that it neither over-
// nor underflows with a loss scale, a row's length or what other rows and sequences hold.
#include "attention.h"

namespace dmuon {
namespace {

constexpr int kTile = 64;                 // rows or keys of a tile in LDS
constexpr float kInf = __builtin_inff();

template <int E>
constexpr float kShift = E == ELT_F16 ? 10.f : 0.f;

// fp16's dS is held times 2^60 until its largest magnitude reaches 2^15; then, and whenever it does so again,
// times the power that brings it to 2^13 .. 2^14. That costs one maximum of the values at hand, and the sums
// are multiplied (exactly) where the power falls. 2^-38 of the largest is then the least error that is not
// relative; dS under 2^-47 in all of a row is lost to fp16's results anyway. In fp32 dS 2^70 < 2^112. One power
// for the whole call took no maximum (2 x 4096 tokens of 32/8 heads with gradients 894 us at dim 64 and 1418 at
// 128, this 933 and 1435), but lost the rows that are 2^20 under the call's largest.
constexpr float kFull = 32768.f;
constexpr int kFirstPower = 60;
// A lane's 16 of a row's (key's) 32 values: the largest, and what the power changes by for both lanes'
__device__ __forceinline__ float largest(const f32x16_t& v) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) most = fmaxf(fmaxf(fabsf(v[i]), fabsf(v[i + 1])), most);
  return most;
}
__device__ __forceinline__ int power_step(float most) {
  most = half_max(most);
  // most < 2^frexp; infinities stay what they are
  return most >= kFull && most < kInf ? 14 - __builtin_amdgcn_frexp_expf(most) : 0;
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }

// A row's share of a transposed result: values result_row(i, h) of each 32
template <int E, int DB>
__device__ __forceinline__ void store_turned(uint16_t* out, const f32x16_t* v, float f, int h, int dim) {
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * b + result_row(i, h);
      if (d < dim)
        *reinterpret_cast<u32x2_t*>(out + d) = u32x2_t{pack2_elt<E>(v[b][i] * f, v[b][i + 1] * f),
                                                       pack2_elt<E>(v[b][i + 2] * f, v[b][i + 3] * f)};
    }
}

// Moves a tile's rows of queries (row r is query r / group of head r % group) into LDS, 4 waves together. A
// tile holds the rows of whole queries, up to 64 of them (more heads a key head: any 64 rows), and zeros.
__device__ __forceinline__ int tile_rows(int group) { return group <= kTile ? kTile / group * group : kTile; }
template <int D>
struct RowMover {
  static constexpr int CPR = D / 8, RPI = 64 / CPR, N = kTile / RPI / 4;
  int wave, row, chunk;
  __device__ __forceinline__ void init(int wave_, int lane) {
    wave = wave_;
    row = wave * N * RPI + lane / CPR;    // of instruction 0
    chunk = lane % CPR;
  }
  // offset of instruction i's row from the first one's, `rem` rows into a query
  __device__ __forceinline__ unsigned offset(int i, int rem, long long token, long long head, int group,
                                             int dim) const {
    const int r = row + i * RPI, q = (rem + r) / group;
    const int c = chunk ^ slot_mask<D>(r);
    return c * 8 < dim ? (unsigned)(q * (int)token + (rem + r - q * group) * (int)head) * 2u + (unsigned)c * 16u
                       : kNowhere;
  }
  // the rows behind p, of which `left` are there, by the offsets that `at` gives
  template <class F>
  __device__ __forceinline__ void issue(const uint16_t* p, int left, char* lds, F at) const {
    typedef __attribute__((address_space(3))) void* lds_ptr_t;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(p), (short)0, 0x7fffffff, 0x00020000);
#pragma unroll
    for (int i = 0; i < N; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(lds + (wave * N + i) * 1024), 16,
                                               row + i * RPI < left ? at(i) : kNowhere, 0, 0, 0);
  }
};

// What the products need besides: -delta of every row (of out and what its rounding left: all of a row's dS
// share delta's error, which took dq's from 1.4 to 1.5 to 1.6 times its own rounding). L lanes a row, 8 values
// each. Reading do, out and rest at 6.3 TB/s: 64 us for 2 x 8192 tokens of 32 heads of 128, 9 for 8191 of 16 of 64.
template <int E, int L>
__global__ __launch_bounds__(256) void attention_delta_kernel(const Attention a) {
  const int at = 8 * (threadIdx.x % L);
  const long long rows = (long long)a.q_len * a.heads * (a.seqs ? 1 : a.batch);
  const long long row = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= rows) return;
  float s = 0.f;
  if (at < a.dim) {
    const long long token = row / a.heads, b = a.seqs ? 0 : token / a.q_len;
    const int head = (int)(row - token * a.heads);
    const uint16_t* d = a.dout + b * a.do_batch + (token - b * a.q_len) * a.do_token + head * a.do_head + at;
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(d);
    const u32x4_t y = *reinterpret_cast<const u32x4_t*>(a.out + row * a.dim + at);
    u32x4_t z = {};
    if (a.rest) z = *reinterpret_cast<const u32x4_t*>(a.rest + row * a.dim + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      auto value = [&](const u32x4_t& w) { return from_elt<E>((uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2])); };
      s += value(x) * (value(y) + value(z));
    }
  }
  for (int o = 1; o < L; o <<= 1) s += __shfl_xor(s, o);
  if (threadIdx.x % L == 0) a.delta[row] = -s;
}

// dk and dv of 128 keys, 32 a wave and one a lane: S = Q K^T and dP = dO V^T leave a lane 16 rows of every
// 32 for its key, which go as they are into dV^T = dO^T P and dK^T = Q^T dS.
template <int D>
struct KeysLds {
  static constexpr int TILE = kTile * D * 2, SLOT = 2 * TILE + 2 * kTile * 4;
  static constexpr int OFFSETS = 2 * SLOT, BYTES = OFFSETS + 256 * 32 + kTile * 4;
};
template <int E, int D>
__device__ __forceinline__ void keys_block(const Attention& a, int id, int blocks, char* lds) {
  constexpr int KS = D / 16, DB = D / 32, TILE = KeysLds<D>::TILE, SLOT = KeysLds<D>::SLOT;
  const Place p = place_of<true>(a, id, blocks, false);
  if (!p.live) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int j0 = p.tile * kKeyRows, j = j0 + wave * 32 + (lane & 31);
  const int rows = p.qn * a.group, before = p.kn - p.qn;

  bf16x8_t kf[KS], vf[KS];
  const bool key_live = j < p.kn;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int at = 16 * s + 8 * h;
    kf[s] = vf[s] = bf16x8_t{};
    if (key_live && at < a.dim) {
      kf[s] = *reinterpret_cast<const bf16x8_t*>(a.k + p.k_off + j * a.k_token + at);
      vf[s] = *reinterpret_cast<const bf16x8_t*>(a.v + p.v_off + j * a.v_token + at);
    }
  }
  // rows that see a key: its own, and those of all keys of the block
  auto rows_of = [&](int key, int* lo, int* hi) {
    *lo = 0;
    *hi = p.qn;
    if (a.causal) {
      if (key - before > 0) *lo = key - before;
      if (a.window && key - before + a.window < p.qn) *hi = key - before + a.window;
    }
  };
  const int last_key = j0 + kKeyRows < p.kn ? j0 + kKeyRows - 1 : p.kn - 1;
  int lo, hi, first_lo, first_hi, last_lo, last_hi;
  rows_of(j, &lo, &hi);
  if (!key_live) hi = 0;
  lo *= a.group;
  hi = hi > 0 ? hi * a.group : 0;
  rows_of(j0, &first_lo, &first_hi);
  rows_of(last_key, &last_lo, &last_hi);
  const int r_lo = first_lo * a.group, r_hi = last_hi > 0 ? last_hi * a.group : 0;
  // rows that see every key of the block need no mask
  const int full_lo = last_lo * a.group;
  const int full_hi = last_key == j0 + kKeyRows - 1 ? first_hi * a.group : 0;
  // rows that see any of this wave's keys: it passes over the other tiles
  const int j_first = j0 + wave * 32, j_last = j_first + 31 < p.kn ? j_first + 31 : p.kn - 1;
  int mine_lo = 0, mine_hi = 0;
  if (j_first < p.kn) {
    int unused;
    rows_of(j_first, &mine_lo, &unused);
    rows_of(j_last, &unused, &mine_hi);
    mine_lo *= a.group;
    mine_hi = mine_hi > 0 ? mine_hi * a.group : 0;
  }
  // tiles of whole queries; a part of them where the rows are split
  const int tr = tile_rows(a.group);
  int n = r_hi > r_lo && j0 < p.kn ? (r_hi - r_lo + tr - 1) / tr : 0, end = n;
  if (a.key_splits > 1) {
    const int each = (n + a.key_splits - 1) / a.key_splits;
    end = n - p.split * each;
    n = end < 0 ? 0 : end < each ? end : each;
  }
  // (rows that see nothing stand before r_lo, in no tile: no key's sums meet what they hold.)
  // From the last rows back: under a causal mask all blocks of a key head begin with the same rows then,
  // and find them in their XCD's L2
  auto first_row = [&](int t) { return r_lo + (end - 1 - t) * tr; };

  RowMover<D> mover;
  mover.init(wave, lane);
  // a lane's offsets of q and dout and of a row's statistics, kept in LDS: the sums need the registers
  unsigned* offsets = reinterpret_cast<unsigned*>(lds + KeysLds<D>::OFFSETS) + threadIdx.x * 8;
  unsigned* stat_at = reinterpret_cast<unsigned*>(lds + KeysLds<D>::OFFSETS + 256 * 32) + lane;
  if (a.group <= kTile) {
#pragma unroll
    for (int i = 0; i < RowMover<D>::N; ++i) {
      offsets[i] = mover.offset(i, 0, a.q_token, a.q_head, a.group, a.dim);
      offsets[4 + i] = mover.offset(i, 0, a.do_token, a.do_head, a.group, a.dim);
    }
    const int q = lane / a.group;
    if (wave == 0) *stat_at = (unsigned)(q * a.heads + lane - q * a.group) * 4u;
  }
  __syncthreads();
  const long long row0 = p.q_row * a.heads + (long long)p.kvh * a.group;
  auto fetch = [&](int t, char* to) __attribute__((always_inline)) {
    typedef __attribute__((address_space(3))) void* lds_ptr_t;
    const int r0 = first_row(t), q0 = r0 / a.group;
    const int left = rows - r0 < tr ? rows - r0 : tr;
    const uint16_t *q = a.q + p.q_off + q0 * a.q_token, *d = a.dout + p.do_off + q0 * a.do_token;
    const float* stats = (wave == 0 ? a.lse : a.delta) + row0 + (long long)q0 * a.heads;
    unsigned stat_off;
    if (a.group <= kTile) {
      const u32x4_t qo = *reinterpret_cast<const u32x4_t*>(offsets);
      const u32x4_t dof = *reinterpret_cast<const u32x4_t*>(offsets + 4);
      stat_off = *stat_at;
      mover.issue(q, left, to, [&](int i) { return qo[i]; });
      mover.issue(d, left, to + TILE, [&](int i) { return dof[i]; });
    } else {
      const int rem = r0 - q0 * a.group;
      mover.issue(q, left, to, [&](int i) { return mover.offset(i, rem, a.q_token, a.q_head, a.group, a.dim); });
      mover.issue(d, left, to + TILE,
                  [&](int i) { return mover.offset(i, rem, a.do_token, a.do_head, a.group, a.dim); });
      const int over = (rem + lane) / a.group;
      stat_off = (unsigned)(over * a.heads + rem + lane - over * a.group) * 4u;
    }
    if (wave < 2) {
      // lse (wave 0) and -delta (wave 1) of the rows
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<float*>(stats), (short)0, 0x7fffffff, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(to + 2 * TILE + wave * kTile * 4), 4,
                                               lane < left ? stat_off : kNowhere, 0, 0, 0);
    }
  };
  const int row_at = row_form<D>(lane), turn_at = turned_form<D>(lane);
  float sigma = E == ELT_F16 ? power(kFirstPower) : 1.f;
  f32x16_t dk[DB], dv[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) dk[b] = dv[b] = f32x16_t{};

  auto step = [&](int t, const char* __restrict__ qt, char* __restrict__ next) __attribute__((always_inline)) {
    const char* dt = qt + TILE;
    const float* stats = reinterpret_cast<const float*>(qt + 2 * TILE);
    if (t + 1 < n) fetch(t + 1, next);
    const int r0 = first_row(t);
    if (r0 >= mine_hi || r0 + kTile <= mine_lo) return;
    const bool early = r0 < full_lo, late = r0 + kTile > full_hi;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      // the reads' addresses are formed anew each time: held over the loop they would take the registers
      // that the sums need
      int ra = row_at, ta = turn_at;
      asm volatile("" : "+v"(ra), "+v"(ta));
      f32x16_t s = {}, dp;
#pragma unroll
      for (int k = 0; k < KS; ++k)
        s = mfma_32x32x16<E>(*reinterpret_cast<const bf16x8_t*>(qt + y * 64 * D + (ra ^ (32 * k))), kf[k], s);
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4_t lse = *reinterpret_cast<const f32x4_t*>(stats + 32 * y + result_row(i, h));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[i + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + e], a.c, kShift<E> - lse[e]));
      }
      if (early) cut_begin(s, r0 + 32 * y, lo, h, 0.f);
      if (late) cut_end(s, r0 + 32 * y, hi, h, 0.f);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8_t pf = pack8<E>(s, 8 * u);
#pragma unroll
        for (int b = 0; b < DB; ++b)
          dv[b] = mfma_32x32x16<E>(read_turned<D>(dt + (2 * y + u) * 32 * D, ta ^ (64 * b)), pf, dv[b]);
      }
      asm volatile("" : "+v"(ra), "+v"(ta));
      // dP - delta: the product begins at -delta. Rows that are not there are zeros throughout.
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4_t delta = *reinterpret_cast<const f32x4_t*>(stats + kTile + 32 * y + result_row(i, h));
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[i + e] = delta[e];
      }
#pragma unroll
      for (int k = 0; k < KS; ++k)
        dp = mfma_32x32x16<E>(*reinterpret_cast<const bf16x8_t*>(dt + y * 64 * D + (ra ^ (32 * k))), vf[k], dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = s[i] * (E == ELT_F16 ? dp[i] * sigma : dp[i]);
      // rows that do not see the key have no share, whatever their dout holds
      if (early) cut_begin(dp, r0 + 32 * y, lo, h, 0.f);
      if (late) cut_end(dp, r0 + 32 * y, hi, h, 0.f);
      if constexpr (E == ELT_F16) {
        const float most = largest(dp);
        if (__ballot(most >= kFull)) {
          const float f = power(power_step(most));
          sigma *= f;
          dp *= f;
#pragma unroll
          for (int b = 0; b < DB; ++b) dk[b] *= f;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8_t sf = pack8<E>(dp, 8 * u);
#pragma unroll
        for (int b = 0; b < DB; ++b)
          dk[b] = mfma_32x32x16<E>(read_turned<D>(qt + (2 * y + u) * 32 * D, ta ^ (64 * b)), sf, dk[b]);
      }
    }
  };
  if (n > 0) fetch(0, lds);
  for (int t = 0; t < n; ++t) {
    slice_barrier<0>();                   // this tile has landed, the slot filled next has been read
    step(t, lds + (t & 1) * SLOT, lds + ((t & 1) ^ 1) * SLOT);
  }
  // keys past a sequence's own, up to the tensor's, have no gradient
  const int most = a.seqs ? p.kn : a.kv_len;
  if (j >= most) return;
  const long long key = (p.k_row + j) * a.kv_heads + p.kvh;
  constexpr float down = E == ELT_F16 ? 1.f / 1024.f : 1.f;
  const float fk = a.scale * down / sigma;
  if (a.key_splits > 1) {
    const long long keys = (long long)a.kv_len * a.kv_heads * (a.seqs ? 1 : a.batch);
    float* part = a.part + (p.split * keys + key) * 2 * a.dim;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * b + result_row(i, h);
        if (d >= a.dim) continue;
        *reinterpret_cast<f32x4_t*>(part + d) =
            f32x4_t{dk[b][i] * fk, dk[b][i + 1] * fk, dk[b][i + 2] * fk, dk[b][i + 3] * fk};
        *reinterpret_cast<f32x4_t*>(part + a.dim + d) =
            f32x4_t{dv[b][i] * down, dv[b][i + 1] * down, dv[b][i + 2] * down, dv[b][i + 3] * down};
      }
    return;
  }
  if (a.dk) store_turned<E, DB>(a.dk + key * a.dim, dk, fk, h, a.dim);
  if (a.dv) store_turned<E, DB>(a.dv + key * a.dim, dv, down, h, a.dim);
}

// Joins the parts of the keys' gradients in their order: 16 lanes a key, 8 values of dk and dv each.
template <int E>
__global__ __launch_bounds__(256) void attention_keys_join_kernel(const Attention a) {
  const long long keys = (long long)a.kv_len * a.kv_heads * (a.seqs ? 1 : a.batch);
  const long long key = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int at = 8 * (threadIdx.x & 15);
  if (key >= keys || at >= a.dim) return;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    uint16_t* out = z ? a.dv : a.dk;
    if (!out) continue;
    f32x4_t lo = {}, hi = {};
#pragma unroll 4
    for (int s = 0; s < a.key_splits; ++s) {
      const float* part = a.part + ((s * keys + key) * 2 + z) * a.dim + at;
      lo += *reinterpret_cast<const f32x4_t*>(part);
      hi += *reinterpret_cast<const f32x4_t*>(part + 4);
    }
    *reinterpret_cast<u32x4_t*>(out + key * a.dim + at) =
        u32x4_t{pack2_elt<E>(lo[0], lo[1]), pack2_elt<E>(lo[2], lo[3]), pack2_elt<E>(hi[0], hi[1]),
                pack2_elt<E>(hi[2], hi[3])};
  }
}

// dq of 128 rows, 32 a wave and one a lane: S^T = K Q^T and dP^T = V dO^T, dQ^T = K^T dS^T.
template <int E, int D>
__device__ __forceinline__ void queries_block(const Attention& a, int id, int blocks, char* lds) {
  constexpr int KS = D / 16, DB = D / 32, TILE = kTile * D * 2;
  const Place p = place_of<false>(a, id, blocks, a.causal);
  if (!p.live) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int r0 = p.tile * kQueryRows, rows = p.qn * a.group;
  const int r = r0 + wave * 32 + (lane & 31);
  const bool live = r < rows;
  const int query = r / a.group, head = r - query * a.group;
  const long long row = (p.q_row + query) * a.heads + (long long)p.kvh * a.group + head;
  bf16x8_t qf[KS], df[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int at = 16 * s + 8 * h;
    qf[s] = df[s] = bf16x8_t{};
    if (live && at < a.dim) {
      qf[s] = *reinterpret_cast<const bf16x8_t*>(a.q + p.q_off + query * a.q_token + head * a.q_head + at);
      df[s] = *reinterpret_cast<const bf16x8_t*>(a.dout + p.do_off + query * a.do_token + head * a.do_head + at);
    }
  }
  const float lse = live ? a.lse[row] : kInf, minus_delta = live ? a.delta[row] : 0.f;
  const Sight see = live ? sight_of(a, p, query) : Sight{0, 0};
  const int last_row = r0 + kQueryRows < rows ? r0 + kQueryRows - 1 : rows - 1;
  const Sight first = sight_of(a, p, r0 / a.group), last = sight_of(a, p, last_row / a.group);
  const int t0 = first.lo / kTile, t1 = (last.hi + kTile - 1) / kTile;
  const int full_lo = last.lo, full_hi = last_row == r0 + kQueryRows - 1 ? first.hi : 0;
  const Sight mine = wave_sight(a, p, r0 + wave * 32, rows);

  TileMover<D, kTile, 4> mk, mv;
  mk.init(a.k_token, a.dim, wave, lane);
  mv.init(a.v_token, a.dim, wave, lane);
  auto fetch = [&](int t, char* to) __attribute__((always_inline)) {
    const int j0 = t * kTile;
    mk.issue(a.k + p.k_off + j0 * a.k_token, a.k_token, a.dim, p.kn - j0, to);
    mv.issue(a.v + p.v_off + j0 * a.v_token, a.v_token, a.dim, p.kn - j0, to + TILE);
  };
  const int row_at = row_form<D>(lane), turn_at = turned_form<D>(lane);
  // the exponent takes in dS's power of two
  int up = E == ELT_F16 ? kFirstPower : 0;
  float from = lse - (float)up;
  f32x16_t dq[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) dq[b] = f32x16_t{};
  auto step = [&](int t, const char* __restrict__ kt, char* __restrict__ next) __attribute__((always_inline)) {
    const char* vt = kt + TILE;
    if (t + 1 < t1) fetch(t + 1, next);
    const int j0 = t * kTile;
    if (j0 >= mine.hi || j0 + kTile <= mine.lo) return;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      f32x16_t s = {}, dp = {};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int at = y * 64 * D + (row_at ^ (32 * k));
        s = mfma_32x32x16<E>(*reinterpret_cast<const bf16x8_t*>(kt + at), qf[k], s);
        dp = mfma_32x32x16<E>(*reinterpret_cast<const bf16x8_t*>(vt + at), df[k], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        dp[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.c, -from)) * (dp[i] + minus_delta);
      if (j0 + kTile > full_hi) cut_end(dp, j0 + 32 * y, see.hi, h, 0.f);
      if (j0 < full_lo) cut_begin(dp, j0 + 32 * y, see.lo, h, 0.f);
      if constexpr (E == ELT_F16) {
        const float most = largest(dp);
        if (__ballot(most >= kFull)) {
          const int by = power_step(most);
          const float f = power(by);
          up += by;
          from = lse - (float)up;
          dp *= f;
#pragma unroll
          for (int b = 0; b < DB; ++b) dq[b] *= f;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8_t sf = pack8<E>(dp, 8 * u);
#pragma unroll
        for (int b = 0; b < DB; ++b)
          dq[b] = mfma_32x32x16<E>(read_turned<D>(kt + (2 * y + u) * 32 * D, turn_at ^ (64 * b)), sf, dq[b]);
      }
    }
  };
  if (t0 < t1) fetch(t0, lds);
  for (int t = t0; t < t1; ++t) {
    slice_barrier<0>();                   // this tile has landed, the slot filled next has been read
    const int slot = (t - t0) & 1;
    step(t, lds + slot * 2 * TILE, lds + (slot ^ 1) * 2 * TILE);
  }
  if (live) store_turned<E, DB>(a.dq + row * a.dim, dq, a.scale * power(-up), h, a.dim);
}

// The keys' blocks come first: they take longer. Waves of a SIMD: two of dim 128 by their registers, three of
// dim 64 (190 -> 170 us at 8191 x 16 heads in a window of 1024).
template <int E, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2, D == 64 ? 3 : 2)))
void attention_grad_kernel(const Attention a, int key_blocks, int query_blocks) {
  __shared__ __attribute__((aligned(1024))) char lds[KeysLds<D>::BYTES];
  // a multiple of 8 blocks keeps each XCD's blocks on it
  const int from = (key_blocks + 7) / 8 * 8, id = blockIdx.x;
  if (id < key_blocks) keys_block<E, D>(a, id, key_blocks, lds);
  else if (id >= from) queries_block<E, D>(a, id - from, query_blocks, lds);
}

template <int E, int D>
void launch_main(const Attention& a, long long key_blocks, long long query_blocks, hipStream_t stream) {
  const long long blocks = (key_blocks + 7) / 8 * 8 + query_blocks;
  if (blocks > 0)
    hipLaunchKernelGGL((attention_grad_kernel<E, D>), dim3((unsigned)blocks), dim3(256), 0, stream, a,
                       (int)key_blocks, (int)query_blocks);
}

}  // namespace

hipError_t launch_attention_grad(const Attention& a, hipStream_t stream) {
  const long long batch = a.seqs ? 1 : a.batch;
  const long long rows = (long long)a.q_len * a.heads * batch, keys = (long long)a.kv_len * a.kv_heads * batch;
  const long long units = (long long)a.kv_heads * batch;
  const long long key_blocks = a.dk || a.dv ? units * a.key_tiles * a.key_splits : 0;
  const long long query_blocks = a.dq ? units * a.tiles : 0;
  if (rows / 16 > 0x7ffffff0LL || keys / 16 > 0x7ffffff0LL || key_blocks + query_blocks > 0x7ffffff0LL)
    return hipErrorInvalidValue;
  const bool f16 = a.dtype == DT_F16, wide = a.dim > 64;
  const unsigned blocks = (unsigned)(wide ? (rows + 15) / 16 : (rows + 31) / 32);
#define DMUON_DELTA(E, L) \
  hipLaunchKernelGGL((attention_delta_kernel<E, L>), dim3(blocks), dim3(256), 0, stream, a)
  if (blocks > 0) {
    if (f16 && wide) DMUON_DELTA(ELT_F16, 16);
    else if (f16) DMUON_DELTA(ELT_F16, 8);
    else if (wide) DMUON_DELTA(ELT_BF16, 16);
    else DMUON_DELTA(ELT_BF16, 8);
  }
#undef DMUON_DELTA
  if (f16) {
    if (wide) launch_main<ELT_F16, 128>(a, key_blocks, query_blocks, stream);
    else launch_main<ELT_F16, 64>(a, key_blocks, query_blocks, stream);
  } else {
    if (wide) launch_main<ELT_BF16, 128>(a, key_blocks, query_blocks, stream);
    else launch_main<ELT_BF16, 64>(a, key_blocks, query_blocks, stream);
  }
  if (key_blocks > 0 && a.key_splits > 1) {
    const dim3 grid((unsigned)((keys + 15) / 16));
    if (f16) hipLaunchKernelGGL((attention_keys_join_kernel<ELT_F16>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attention_keys_join_kernel<ELT_BF16>), grid, dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace dmuon
