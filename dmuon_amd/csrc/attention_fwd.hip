// Attention over heads on gfx950: o = softmax(c q k^T) v in one pass over the keys with the running
// maximum and sum of each row.
//
//   s = c q k^T - m,  p = 2^s,  l = sum p,  o = sum p v / l,  m any reference near the row's maximum
// Scores, sums and statistics are fp32. p is rounded to the operands' type before it meets v, as the matrix
// instruction takes it (2^-9 of each term on average, against the result's own rounding of as much).
//
// 4 dim operations a pair of a query and a key on the matrix pipe, some five on the vector one. A wave has all
// of a tile's scores before their softmax and that before P v, so that only the SIMD's other waves can overlap
// the two pipes, and they hardly do. Dim 128: 2 x 8192 causal tokens, 32/8 heads, bf16 1.07 ms (1.03 PFLOP/s, at
// 1.8 of 2.4 GHz under the board's power limit), of whose cycles the matrix pipe is busy 54%, the vector pipe 49
// and both at once 20; 2047 tokens over 32768 keys 1.01 ms (1.05). Dim 64: 8191 tokens of 16 heads in a window
// of 1024 in fp16 57 us (0.57), matrix pipe 25%, vector pipe 46, both 13. Single tokens are bound by
// reading the cache: 48 x 1 over up to 8192 keys 155 us (6.6 TB/s). A tile of 64 keys lies in LDS twice, one
// copy read while the other is loaded; keys go through LDS since all waves read them, queries stay in
// registers. 64 rows a wave (half the reads, one wave a SIMD) took 1.44 ms where 32 took 1.04. Heads are padded
// with zeros to 64 or 128 values, which the products do not leave out: 2 x 4096 tokens of 32/8 heads in bf16
// take 181 us at dim 64, 237 at 80, 244 at 96, 264 at 128, and as long at 32 as at 64.
#include "attention.h"

namespace dmuon {
namespace {

constexpr float kInf = __builtin_inff();
// A row's reference where all it sees has the score -infinity; only a row that sees nothing keeps -infinity itself
constexpr float kLeast = -3.402823466e38f;
constexpr int kKeys = 64;                 // keys of a tile

// What is left of two values behind their rounding
template <int E>
__device__ __forceinline__ unsigned rest2(unsigned w, float lo, float hi) {
  return pack2_elt<E>(lo - from_elt<E>((uint16_t)w), hi - from_elt<E>((uint16_t)(w >> 16)));
}

// A lane's half of a row: the result and its statistics, or, of one part of the keys, the unfinished sums.
template <int E, int DB>
__device__ __forceinline__ void store_row(const Attention& a, const Place& p, bool live, int query, int head,
                                          const f32x16_t* o, float ref, float total, int h) {
  if (!live) return;
  const long long row = (p.q_row + query) * a.heads + (long long)p.kvh * a.group + head;
  if (a.splits > 1) {
    const long long at = (long long)p.split * a.q_len * a.heads * (a.seqs ? 1 : a.batch) + row;
    float* part = a.part + at * a.dim;
    if (h == 0) a.part_stats[at] = make_float2(ref, total);
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * b + result_row(i, h);
        if (d < a.dim)
          *reinterpret_cast<f32x4_t*>(part + d) = f32x4_t{o[b][i], o[b][i + 1], o[b][i + 2], o[b][i + 3]};
      }
    return;
  }
  // a row that sees nothing is 0; one that sees scores of -infinity alone is 0 / 0
  const float f = ref == -kInf ? 0.f : 1.f / total;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * b + result_row(i, h);
      if (d >= a.dim) continue;
      const u32x2_t w = {pack2_elt<E>(o[b][i] * f, o[b][i + 1] * f),
                         pack2_elt<E>(o[b][i + 2] * f, o[b][i + 3] * f)};
      *reinterpret_cast<u32x2_t*>(a.out + row * a.dim + d) = w;
      if (a.rest)
        *reinterpret_cast<u32x2_t*>(a.rest + row * a.dim + d) =
            u32x2_t{rest2<E>(w[0], o[b][i] * f, o[b][i + 1] * f),
                    rest2<E>(w[1], o[b][i + 2] * f, o[b][i + 3] * f)};
    }
  if (a.lse && h == 0) a.lse[row] = ref == -kInf ? kInf : ref + __log2f(total);
}

// A block has 128 rows of queries, 32 a wave and one a lane (l % 32): S^T = K Q^T leaves each lane 16 keys of
// every 32 for its own row, the other half of the wave's lanes the rest, and goes as it is into
// O^T = V^T P^T.
// Waves of a SIMD: two of dim 128 by their registers, four of dim 64 (68 -> 63 us at 8191 x 16 heads in a
// window of 1024).
template <int E, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : 2, D == 64 ? 4 : 2)))
void attention_kernel(const Attention a) {
  constexpr int KS = D / 16, DB = D / 32, TILE = kKeys * D * 2;
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];
  const Place p = place_of<false>(a, blockIdx.x, gridDim.x, a.causal);
  if (!p.live) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int r0 = p.tile * kQueryRows, rows = p.qn * a.group;

  // this lane's row; rows past the last one see nothing
  const int r = r0 + wave * 32 + (lane & 31), query = r / a.group, head = r - query * a.group;
  const bool live = r < rows;
  bf16x8_t qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int at = 16 * s + 8 * h;
    qf[s] = bf16x8_t{};
    if (live && at < a.dim)
      qf[s] = *reinterpret_cast<const bf16x8_t*>(a.q + p.q_off + query * a.q_token + head * a.q_head + at);
  }
  const Sight see = live ? sight_of(a, p, query) : Sight{0, 0};
  // the block's tiles: what its first and last row see
  const int last_row = r0 + kQueryRows < rows ? r0 + kQueryRows - 1 : rows - 1;
  const Sight first = sight_of(a, p, r0 / a.group), last = sight_of(a, p, last_row / a.group);
  int t0 = first.lo / kKeys, t1 = (last.hi + kKeys - 1) / kKeys;
  if (t1 < t0) t1 = t0;
  if (a.splits > 1) {
    const int each = (t1 - t0 + a.splits - 1) / a.splits;
    t0 = t0 + p.split * each < t1 ? t0 + p.split * each : t1;
    t1 = t0 + each < t1 ? t0 + each : t1;
  }
  const Sight mine = wave_sight(a, p, r0 + wave * 32, rows);
  // keys that every row sees need no mask
  const int full_lo = last.lo, full_hi = last_row == r0 + kQueryRows - 1 ? first.hi : 0;

  TileMover<D, kKeys, 4> mk, mv;
  mk.init(a.k_token, a.dim, wave, lane);
  mv.init(a.v_token, a.dim, wave, lane);
  auto fetch = [&](int t, char* to) __attribute__((always_inline)) {
    const int j0 = t * kKeys;
    mk.issue(a.k + p.k_off + j0 * a.k_token, a.k_token, a.dim, p.kn - j0, to);
    mv.issue(a.v + p.v_off + j0 * a.v_token, a.v_token, a.dim, p.kn - j0, to + TILE);
  };
  const int row_at = row_form<D>(lane), turn_at = turned_form<D>(lane);

  f32x16_t o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) o[b] = f32x16_t{};
  float ref = -kInf, sum = 0.f;
  // the slots' pointers are restrict: the compiler need not wait for loads into `next` before reads of `kt`
  auto step = [&](int t, const char* __restrict__ kt, char* __restrict__ next) __attribute__((always_inline)) {
    const char* vt = kt + TILE;
    if (t + 1 < t1) fetch(t + 1, next);
    const int j0 = t * kKeys;
    if (j0 >= mine.hi || j0 + kKeys <= mine.lo) return;
    f32x16_t s[2] = {};
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        s[b] = mfma_32x32x16<E>(*reinterpret_cast<const bf16x8_t*>(kt + b * 64 * D + (row_at ^ (32 * k))), qf[k],
                                s[b]);
    // six reads ahead of the products (read and used in pairs, 2 x 8192 tokens took 1070 us where these
    // take 1040)
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int i = 0; i < KS - 3; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, 6, 0);
    if (j0 + kKeys > full_hi) {
      cut_end(s[0], j0, see.hi, h, -kInf);
      cut_end(s[1], j0 + 32, see.hi, h, -kInf);
    }
    if (j0 < full_lo) {
      cut_begin(s[0], j0, see.lo, h, -kInf);
      cut_begin(s[1], j0 + 32, see.lo, h, -kInf);
    }
    float top = -kInf;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = half_max(top) * a.c;
    // the reference follows the maximum only when that has grown by 2^8: any reference gives the same
    // quotient, and sums and 16-bit probabilities have room for 256
    if (__ballot(top > ref + 8.f)) {
      const float now = fmaxf(ref, top), from = now == -kInf ? 0.f : now;
      const float f = __builtin_amdgcn_exp2f(ref - from);
      ref = now;
      sum *= f;
#pragma unroll
      for (int b = 0; b < DB; ++b) o[b] *= f;
    }
    const float from = ref == -kInf ? 0.f : ref;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], a.c, -from));
        sum += s[b][i];
      }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bf16x8_t pf = pack8<E>(s[u / 2], 8 * (u & 1));
#pragma unroll
      for (int b = 0; b < DB; ++b)
        o[b] = mfma_32x32x16<E>(read_turned<D>(vt + u * 32 * D, turn_at ^ (64 * b)), pf, o[b]);
    }
  };
  if (t0 < t1) fetch(t0, lds);
  for (int t = t0; t < t1; ++t) {
    slice_barrier<0>();                   // this tile has landed, the slot filled next has been read
    const int slot = (t - t0) & 1;
    step(t, lds + slot * 2 * TILE, lds + (slot ^ 1) * 2 * TILE);
  }
  if (see.hi > see.lo) ref = fmaxf(ref, kLeast);
  store_row<E, DB>(a, p, live, query, head, o, ref, half_sum(sum), h);
}

// Few rows over many keys (single tokens over a cache): a wave for itself takes 32 rows and a part of the
// keys, 32 at a time. Bound by reading k and v: no wave waits for another, and the next two tiles of both
// are in flight while one is worked on (24 to 32 KB a wave, five waves a CU).
template <int E, int D>
__global__ __launch_bounds__(64) void attention_few_kernel(const Attention a) {
  constexpr int KS = D / 16, DB = D / 32, KEYS = 32, TILE = KEYS * D * 2, LOADS = TILE / 1024;
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];
  const Place p = place_of<false>(a, blockIdx.x, gridDim.x, false);
  if (!p.live) return;
  const int lane = threadIdx.x, h = lane >> 5;
  const int r0 = p.tile * kFewRows, rows = p.qn * a.group;
  const int r = r0 + (lane & 31), query = r / a.group, head = r - query * a.group;
  const bool live = r < rows;
  const int last_row = r0 + kFewRows < rows ? r0 + kFewRows - 1 : rows - 1;
  const Sight first = sight_of(a, p, r0 / a.group), last = sight_of(a, p, last_row / a.group);
  const Sight see = live ? sight_of(a, p, query) : Sight{0, 0};
  int t0 = first.lo / KEYS, t1 = (last.hi + KEYS - 1) / KEYS;
  if (t1 < t0) t1 = t0;
  const int each = (t1 - t0 + a.splits - 1) / a.splits;
  t0 = t0 + p.split * each < t1 ? t0 + p.split * each : t1;
  t1 = t0 + each < t1 ? t0 + each : t1;
  // keys that every row sees; rows past the last one are not stored, and need no mask
  const int full_lo = last.lo, full_hi = first.hi;

  TileMover<D, KEYS, 1> mk, mv;
  mk.init(a.k_token, a.dim, 0, lane);
  mv.init(a.v_token, a.dim, 0, lane);
  auto fetch_k = [&](int t, char* to) __attribute__((always_inline)) {
    const int j0 = t * KEYS;
    mk.issue(a.k + p.k_off + j0 * a.k_token, a.k_token, a.dim, p.kn - j0, to);
  };
  auto fetch_v = [&](int t, char* to) __attribute__((always_inline)) {
    const int j0 = t * KEYS;
    mv.issue(a.v + p.v_off + j0 * a.v_token, a.v_token, a.dim, p.kn - j0, to);
  };
  bf16x8_t qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int at = 16 * s + 8 * h;
    qf[s] = bf16x8_t{};
    if (live && at < a.dim)
      qf[s] = *reinterpret_cast<const bf16x8_t*>(a.q + p.q_off + query * a.q_token + head * a.q_head + at);
  }
  const int row_at = row_form<D>(lane), turn_at = turned_form<D>(lane);
  f32x16_t o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) o[b] = f32x16_t{};
  float ref = -kInf, sum = 0.f;
  // A slot is filled again as soon as it has been read: the waits count the loads of the three tiles behind
  // (none are missing before the last two). The slots are restrict so that the compiler adds no waits of its
  // own, each read and filled through its one pointer; the empty asm statements keep reads and loads of one slot
  // in their order.
  auto step = [&](int t, char* __restrict__ kt, char* __restrict__ vt) __attribute__((always_inline)) {
    const bool more = t + 2 < t1;
    if (more) wait_vmcnt<3 * LOADS>();
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    f32x16_t s = {};
#pragma unroll
    for (int k = 0; k < KS; ++k)
      s = mfma_32x32x16<E>(*reinterpret_cast<const bf16x8_t*>(kt + (row_at ^ (32 * k))), qf[k], s);
    asm volatile("" : "+v"(s) : : "memory");
    if (more) fetch_k(t + 2, kt);
    const int j0 = t * KEYS;
    if (j0 + KEYS > full_hi) cut_end(s, j0, see.hi, h, -kInf);
    if (j0 < full_lo) cut_begin(s, j0, see.lo, h, -kInf);
    float top = -kInf;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
    top = half_max(top) * a.c;
    if (__ballot(top > ref + 8.f)) {
      const float now = fmaxf(ref, top), from = now == -kInf ? 0.f : now;
      const float f = __builtin_amdgcn_exp2f(ref - from);
      ref = now;
      sum *= f;
#pragma unroll
      for (int b = 0; b < DB; ++b) o[b] *= f;
    }
    const float from = ref == -kInf ? 0.f : ref;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.c, -from));
      sum += s[i];
    }
    if (more) wait_vmcnt<3 * LOADS>();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bf16x8_t pf = pack8<E>(s, 8 * u);
#pragma unroll
      for (int b = 0; b < DB; ++b)
        o[b] = mfma_32x32x16<E>(read_turned<D>(vt + u * 32 * D, turn_at ^ (64 * b)), pf, o[b]);
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): every read of the slot has returned
    asm volatile("" ::: "memory");
    if (more) fetch_v(t + 2, vt);
  };
  for (int t = t0; t < t1 && t < t0 + 2; ++t) {
    fetch_k(t, lds + (t - t0) * 2 * TILE);
    fetch_v(t, lds + (t - t0) * 2 * TILE + TILE);
  }
  for (int t = t0; t < t1; ++t) {
    char* slot = lds + ((t - t0) & 1) * 2 * TILE;
    step(t, slot, slot + TILE);
  }
  if (see.hi > see.lo) ref = fmaxf(ref, kLeast);
  store_row<E, DB>(a, p, live, query, head, o, ref, half_sum(sum), h);
}

// Joins the parts of the key axis (64 at most): one wave a row, two values a lane.
template <int E>
__global__ __launch_bounds__(256) void attention_join_kernel(const Attention a) {
  const long long rows = (long long)a.q_len * a.heads * (a.seqs ? 1 : a.batch);
  const long long row = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= rows) return;
  // part l's statistics in lane l
  float2 st = make_float2(-kInf, 0.f);
  if (lane < a.splits) st = a.part_stats[lane * rows + row];
  float top = st.x;
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float from = top == -kInf ? 0.f : top;
  const float f = __builtin_amdgcn_exp2f(st.x - from);
  float total = f * st.y;
  for (int o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o);
  float o0 = 0.f, o1 = 0.f;
  const int d = 2 * lane < a.dim ? 2 * lane : 0;
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    float2 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int s = s0 + k < a.splits ? s0 + k : a.splits - 1;
      v[k] = *reinterpret_cast<const float2*>(a.part + (s * rows + row) * a.dim + d);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float g = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), (s0 + k) & 63));
      o0 += s0 + k < a.splits ? g * v[k].x : 0.f;
      o1 += s0 + k < a.splits ? g * v[k].y : 0.f;
    }
  }
  const float g = top == -kInf ? 0.f : 1.f / total;
  if (2 * lane < a.dim) {
    const unsigned w = pack2_elt<E>(o0 * g, o1 * g);
    *reinterpret_cast<unsigned*>(a.out + row * a.dim + d) = w;
    if (a.rest) *reinterpret_cast<unsigned*>(a.rest + row * a.dim + d) = rest2<E>(w, o0 * g, o1 * g);
  }
  if (a.lse && lane == 0) a.lse[row] = top == -kInf ? kInf : top + __log2f(total);
}

// Sequences and tiles of a packed call. Starts that fall are taken as the largest before them, and all
// lie within the tokens that are there. Four further sequences hold the tokens before the first and behind
// the last start: queries that see nothing, and keys that nothing sees. One block; a sequence's tiles are written
// by one thread (23 documents of 16384 tokens: 8 us).
__global__ __launch_bounds__(1024) void attention_tables_kernel(
    const int64_t* q_starts, const int64_t* k_starts, int n, int group, int q_tokens, int k_tokens,
    int q_rows, int k_rows, Sequence* seqs, int2* q_tiles, int2* k_tiles, int* counts) {
  __shared__ int lds[2][16], carry[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // inclusive scan over the block of a pair, by maximum or by sum
  auto scan = [&](int& x, int& y, bool sum) {
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(x, d), v = __shfl_up(y, d);
      if (lane >= d) {
        x = sum ? x + u : (x > u ? x : u);
        y = sum ? y + v : (y > v ? y : v);
      }
    }
    __syncthreads();
    if (lane == 63) lds[0][wave] = x, lds[1][wave] = y;
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      const int u = lds[0][w], v = lds[1][w];
      x = sum ? x + u : (x > u ? x : u);
      y = sum ? y + v : (y > v ? y : v);
    }
  };
  auto held = [](int64_t s, int most) { return s < 0 ? 0 : s < most ? (int)s : most; };
  if (tid < 4) carry[tid] = 0;
  // the starts, made to rise
  for (int base = 0; base <= n; base += 1024) {
    const int i = base + tid;
    int q = i <= n ? held(q_starts[i], q_tokens) : 0, k = i <= n ? held(k_starts[i], k_tokens) : 0;
    __syncthreads();
    q = q > carry[0] ? q : carry[0];
    k = k > carry[1] ? k : carry[1];
    scan(q, k, false);
    __syncthreads();
    if (tid == 1023) carry[0] = q, carry[1] = k;
    if (i <= n) {
      seqs[i].q0 = q;                     // [n] is overwritten below, once read
      seqs[i].k0 = k;
    }
  }
  __syncthreads();
  __threadfence_block();
  const int q_first = seqs[0].q0, k_first = seqs[0].k0, q_end = seqs[n].q0, k_end = seqs[n].k0;
  __syncthreads();
  for (int i = tid; i < n; i += 1024) {
    const int q1 = seqs[i + 1].q0, k1 = seqs[i + 1].k0;
    seqs[i].qn = q1 - seqs[i].q0;
    seqs[i].kn = k1 - seqs[i].k0;
  }
  __syncthreads();
  if (tid == 0) {
    seqs[n] = Sequence{0, q_first, 0, 0};
    seqs[n + 1] = Sequence{q_end, q_tokens - q_end, 0, 0};
    seqs[n + 2] = Sequence{0, 0, 0, k_first};
    seqs[n + 3] = Sequence{0, 0, k_end, k_tokens - k_end};
  }
  __syncthreads();
  __threadfence_block();
  for (int base = 0; base < n + 4; base += 1024) {
    const int i = base + tid;
    int q = 0, k = 0;
    if (i < n + 4) {
      q = (int)(((long long)seqs[i].qn * group + q_rows - 1) / q_rows);
      k = (seqs[i].kn + k_rows - 1) / k_rows;
    }
    int qe = q, ke = k;
    scan(qe, ke, true);
    const int qb = carry[2] + qe - q, kb = carry[3] + ke - k;
    for (int t = 0; t < q; ++t) q_tiles[qb + t] = make_int2(i, t);
    for (int t = 0; t < k; ++t) k_tiles[kb + t] = make_int2(i, t);
    __syncthreads();
    if (tid == 1023) carry[2] += qe, carry[3] += ke;
    __syncthreads();
  }
  if (tid < 2) counts[tid] = carry[2 + tid];
}

template <int E, int D>
void launch(const Attention& a, unsigned blocks, hipStream_t stream) {
  if (a.few) hipLaunchKernelGGL((attention_few_kernel<E, D>), dim3(blocks), dim3(64), 0, stream, a);
  else hipLaunchKernelGGL((attention_kernel<E, D>), dim3(blocks), dim3(256), 0, stream, a);
}

}  // namespace

hipError_t launch_attention_tables(const Attention& a, const int64_t* q_starts, const int64_t* kv_starts,
                                   int q_rows, int k_rows, Sequence* seqs, int2* q_tiles, int2* k_tiles,
                                   int* counts, hipStream_t stream) {
  hipLaunchKernelGGL(attention_tables_kernel, dim3(1), dim3(1024), 0, stream, q_starts, kv_starts, a.batch,
                     a.group, a.q_len, a.kv_len, q_rows, k_rows, seqs, q_tiles, k_tiles, counts);
  return hipGetLastError();
}

hipError_t launch_attention(const Attention& a, hipStream_t stream) {
  const long long units = (long long)a.kv_heads * (a.seqs ? 1 : a.batch);
  const long long blocks = units * a.tiles * a.splits;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  if (blocks > 0) {
    const bool wide = a.dim > 64;
    if (a.dtype == DT_F16) {
      if (wide) launch<ELT_F16, 128>(a, (unsigned)blocks, stream);
      else launch<ELT_F16, 64>(a, (unsigned)blocks, stream);
    } else {
      if (wide) launch<ELT_BF16, 128>(a, (unsigned)blocks, stream);
      else launch<ELT_BF16, 64>(a, (unsigned)blocks, stream);
    }
    if (a.splits > 1) {
      const long long rows = (long long)a.q_len * a.heads * (a.seqs ? 1 : a.batch);
      if ((rows + 3) / 4 > 0x7fffffffLL) return hipErrorInvalidValue;
      const dim3 grid((unsigned)((rows + 3) / 4));
      if (a.dtype == DT_F16)
        hipLaunchKernelGGL((attention_join_kernel<ELT_F16>), grid, dim3(256), 0, stream, a);
      else
        hipLaunchKernelGGL((attention_join_kernel<ELT_BF16>), grid, dim3(256), 0, stream, a);
    }
  }
  return hipGetLastError();
}

}  // namespace dmuon
