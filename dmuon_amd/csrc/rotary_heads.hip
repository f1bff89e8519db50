// Norms of queries and keys for each head with the position rotation on gfx950, and their gradients.
//
//   xhat = x rsqrt(mean x^2 + eps), z = xhat w  (no weight: z = x),  y = R(position) z
// R turns the pair (a, b) by the angle t = position inv_freq: (a cos t - b sin t, b cos t + a sin t).
// Backward, g = R^T dy:  dw = sum g xhat,  dx = r (g w - xhat mean(g w xhat)).
//
// Memory bound: forward reads x and writes y; backward reads x and dy and writes dx (the root mean
// square is formed anew). A lane has the same 8 pairs of every head (4, or 1, where a head has no more), so
// that pairs half a rotation apart need no exchange, and one exchange of sums joins the lanes of a head.
// The lanes of a group keep a token's cosines and sines in registers and walk its heads, the next one's
// loads in flight: angles are formed once a token and part of the heads, in turns, as sums of two fp64 values
// reduced to an eighth of a turn around a multiple of a quarter: all 64-bit positions are as exact as near ones.
//
// 16384 tokens of 32 + 8 heads of 128 in bf16, read from rows of 48 heads: forward 73 us (4.6 TB/s), backward
// 94 (5.3) and 4 of joining the weights' gradients; 1777 x 6 heads of 72 in fp32, pairs side by side 7 and 11.
// One token 6.9, of which the angles' chain of fp64 instructions is one. In fp32, 16384 tokens of 40 heads of 128 as
// dense rows 192 (3.5 TB/s) and 196 (5.1). Rotated widths or heads that are no multiple of 8 go value by value:
// heads of 80 in bf16 with 80 rotated 60 and 70 us, with 20 rotated 92 and 366.
#include "../../include/dmuon_amd.h"
#include "dmuon_amd_internal.h"
#include "mfma_tile.h"

#pragma clang fp contract(fast)

namespace dmuon {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 512;

struct Heads {
  const void* x[2]; void* y[2]; const void* dy[2]; void* dx[2];   // queries, keys
  const void* w[2];                       // [dim] or NULL
  void* dw[2]; float* part[2];            // [parts * blocks][dim]
  long long token[2], head[2], dtoken[2], dhead[2];               // strides in elements
  const int64_t* positions; const void* inv_freq;
  long long tokens, period;
  int heads[2], dim, rotary, dtype, w_dtype[2], freq_double, interleaved;
  int pairs, lanes;                       // of a lane; of a head: a power of two
  int per_part, parts[2];                 // heads that one group walks; parts of the queries', keys' heads
  int blocks;                             // of one part
  float eps;
};

__device__ __forceinline__ float element(const void* p, int t, long long at) {
  if (t == DT_F32) return static_cast<const float*>(p)[at];
  const uint16_t u = static_cast<const uint16_t*>(p)[at];
  return t == DT_F16 ? from_elt<ELT_F16>(u) : from_elt<ELT_BF16>(u);
}
__device__ __forceinline__ void set_element(void* p, int t, long long at, float v) {
  if (t == DT_F32) static_cast<float*>(p)[at] = v;
  else static_cast<uint16_t*>(p)[at] = t == DT_F16 ? to_elt<ELT_F16>(v) : to_elt<ELT_BF16>(v);
}

// N (4 or 8) values of type T as they lie in memory, at any element alignment
template <int T, int N>
struct Run {
  static constexpr int W = T == DT_F32 ? N : N / 2;      // 32-bit words
  unsigned w[W];
  __device__ __forceinline__ void load(const void* p, long long at) {
    typedef unsigned words_t __attribute__((ext_vector_type(W < 4 ? 2 : 4)));
    typedef words_t any_t __attribute__((aligned(T == DT_F32 ? 4 : 2)));
    constexpr int V = W < 4 ? 2 : 4;
    const char* src = static_cast<const char*>(p) + at * (T == DT_F32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < W; i += V) {
      const words_t x = *reinterpret_cast<const any_t*>(src + 4 * i);
#pragma unroll
      for (int k = 0; k < V; ++k) w[i + k] = x[k];
    }
  }
  __device__ __forceinline__ void store(void* p, long long at) const {
    typedef unsigned words_t __attribute__((ext_vector_type(W < 4 ? 2 : 4)));
    typedef words_t any_t __attribute__((aligned(T == DT_F32 ? 4 : 2)));
    constexpr int V = W < 4 ? 2 : 4;
    char* dst = static_cast<char*>(p) + at * (T == DT_F32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < W; i += V) {
      words_t x;
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] = w[i + k];
      __builtin_nontemporal_store(x, reinterpret_cast<any_t*>(dst + 4 * i));
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (T == DT_F32) return __uint_as_float(w[i]);
    const uint16_t u = (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2]);
    return T == DT_F16 ? from_elt<ELT_F16>(u) : from_elt<ELT_BF16>(u);
  }
  __device__ __forceinline__ void set2(int i, float a, float b) {    // values i and i + 1
    if constexpr (T == DT_F32) {
      w[i] = __float_as_uint(a);
      w[i + 1] = __float_as_uint(b);
    } else {
      w[i / 2] = pack2_elt<T == DT_F16 ? ELT_F16 : ELT_BF16>(a, b);
    }
  }
};

// Where pair p of a head lies: a rotated pair for p < rotary / 2, two neighbours behind them.
__device__ __forceinline__ void pair_at(const Heads& a, int p, int* i, int* j) {
  const int half = a.rotary / 2;
  if (p < half && !a.interleaved) {
    *i = p;
    *j = p + half;
  } else {
    *i = 2 * p;
    *j = 2 * p + 1;
  }
}

// A lane's P pairs of a head, from pair `p` on: P = 8 (rotary and dim multiples of 16) or 4 (of 8) are two
// runs of P values, the pairs' first and second ones or, SIDE by side, one run behind the other. (Values that
// are not rotated may pair as they lie.)
template <int T, int P, bool SIDE>
struct Pairs {
  Run<T, P> r[2];
  __device__ __forceinline__ void load(const void* src, long long at, int i, int j) {
    r[0].load(src, at + i);
    r[1].load(src, at + j);
  }
  // where value k of both runs stands among the pairs' first ones, then their second ones
  static __device__ __forceinline__ constexpr int place(int run, int k) {
    return SIDE ? ((run * P + k) & 1) * P + (run * P + k) / 2 : run * P + k;
  }
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int k = 0; k < P; ++k) v[place(0, k)] = r[0].get(k), v[place(1, k)] = r[1].get(k);
  }
  __device__ __forceinline__ void set(const float* v) {
#pragma unroll
    for (int k = 0; k < P; k += 2) {
      r[0].set2(k, v[place(0, k)], v[place(0, k + 1)]);
      r[1].set2(k, v[place(1, k)], v[place(1, k + 1)]);
    }
  }
  __device__ __forceinline__ void store(void* dst, long long at, int i, int j) const {
    r[0].store(dst, at + i);
    r[1].store(dst, at + j);
  }
};
template <int T, bool SIDE>
struct Pairs<T, 1, SIDE> {
  float a, b;
  __device__ __forceinline__ void load(const void* src, long long at, int i, int j) {
    a = element(src, T, at + i);
    b = element(src, T, at + j);
  }
  __device__ __forceinline__ void get(float* v) const { v[0] = a, v[1] = b; }
  __device__ __forceinline__ void set(const float* v) { a = v[0], b = v[1]; }
  __device__ __forceinline__ void store(void* dst, long long at, int i, int j) const {
    set_element(dst, T, at + i, a);
    set_element(dst, T, at + j, b);
  }
};

// The place in its head of a lane's value k (the pairs' first values, then their second), whose runs begin
// at i and j
template <int P, bool SIDE>
__device__ __forceinline__ int value_at(int i, int j, int k) {
  if (P > 1 && SIDE) return i + 2 * (k % P) + k / P;
  return k < P ? i + k : j + k - P;
}

// The position in two parts that fp64 holds: position = hi + lo, hi a multiple of 2^32
struct Position {
  double hi, lo;
};
__device__ __forceinline__ Position position_of(int64_t p) {
  return {(double)(p >> 32) * 4294967296., (double)(unsigned)p};
}

// cos and sin of position * inv_freq. In quarters of a turn the angle is position f 2 / pi, formed as sums of
// two: f 2 / pi = fh + fl to 2^-105 of it, and the products of both parts of the position with fh as their
// rounded values, of which whole turns are dropped without an error, and the rest of those. What is rounded is
// under 2^12 quarters then: angles of 64-bit positions and frequencies up to 1 (products up to 2^63) are
// within 2^-40, ones under 2^31 within 2^-50. Within an eighth of a turn the Taylor polynomials are off by less
// than 2^-29. No contraction: a product that is rounded in one place must be the same in the other.
__device__ __forceinline__ float2 turn_of(const Heads& a, const Position& position, int pair) {
#pragma clang fp contract(off)
  constexpr double kTwoByPi = 0x1.45f306dc9c883p-1, kTwoByPiRest = -0x1.6b01ec5417056p-55;
  const double f = a.freq_double ? static_cast<const double*>(a.inv_freq)[pair]
                                 : (double)static_cast<const float*>(a.inv_freq)[pair];
  const double fh = f * kTwoByPi;
  const double fl = __builtin_fma(f, kTwoByPiRest, __builtin_fma(f, kTwoByPi, -fh));
  const double p = position.hi * fh, q = position.lo * fh;
  const double rest = __builtin_fma(position.hi, fh, -p) + __builtin_fma(position.lo, fh, -q) +
                      (position.hi + position.lo) * fl;
  const double near = (p - 4. * rint(p * 0.25)) + (q - 4. * rint(q * 0.25));
  const double whole = rint(near + rest);
  const float t = (float)((near - whole) + rest) * 1.57079632679489661923f, z = t * t;
  const float s = t + t * z * (-1.f / 6.f + z * (1.f / 120.f + z * (-1.f / 5040.f + z * (1.f / 362880.f))));
  const float c = 1.f + z * (-0.5f + z * (1.f / 24.f + z * (-1.f / 720.f + z * (1.f / 40320.f -
                                                                              z * (1.f / 3628800.f)))));
  const int k = (int)(whole - 4. * floor(whole * 0.25));
  const float cc = k & 1 ? s : c, ss = k & 1 ? c : s;
  return make_float2(k == 1 || k == 2 ? -cc : cc, k >= 2 ? -ss : ss);
}

// GRAD: x and dy to dx and the weights' partial sums; otherwise x to y. SLOTS: of P pairs a lane.
// blockIdx.y is the part of the heads: the queries' parts, then the keys'.
// SIDE: rotated pairs are neighbours (of P = 1: either, by their places).
template <int T, int P, int SLOTS, bool SIDE, bool GRAD>
__global__ __launch_bounds__(kThreads) void rotary_heads_kernel(const Heads a) {
  // heads whose loads are in flight: forward 79 us of one, 75 of two (16384 tokens of 32 + 8 heads of 128)
  constexpr int AHEAD = GRAD ? 1 : 2;
  __shared__ float sums[GRAD ? kThreads : 1][2 * P + 1];
  const int sub = threadIdx.x % a.lanes, group = threadIdx.x / a.lanes, groups = kThreads / a.lanes;
  const int half = a.rotary / 2;
  const int z = (int)blockIdx.y >= a.parts[0], part = (int)blockIdx.y - (z ? a.parts[0] : 0);
  const int h0 = part * a.per_part, h1 = min(h0 + a.per_part, a.heads[z]);
  const bool norm = a.w[z] != nullptr;
  const float inv = 1.f / (float)a.dim;
  const void* x = a.x[z];
  const void* dy = a.dy[z];
  void* to = GRAD ? a.dx[z] : a.y[z];
  int pair[SLOTS], vi[SLOTS], vj[SLOTS];
  bool live[SLOTS];
  float w[SLOTS][2 * P], dw[SLOTS][2 * P];
#pragma unroll
  for (int u = 0; u < SLOTS; ++u) {
    pair[u] = (u * a.lanes + sub) * P;
    live[u] = pair[u] < a.dim / 2;
    if (!live[u]) pair[u] = 0;
    pair_at(a, pair[u], &vi[u], &vj[u]);
    if (P > 1 && vj[u] == vi[u] + 1) vj[u] = vi[u] + P;
#pragma unroll
    for (int i = 0; i < 2 * P; ++i) {
      w[u][i] = norm && live[u] ? element(a.w[z], a.w_dtype[z], value_at<P, SIDE>(vi[u], vj[u], i)) : 1.f;
      dw[u][i] = 0.f;
    }
  }
  for (long long token = (long long)blockIdx.x * groups + group; token < a.tokens;
       token += (long long)gridDim.x * groups) {
    long long at = token * a.token[z] + h0 * a.head[z], dat = token * a.dtoken[z] + h0 * a.dhead[z];
    long long out = (token * a.heads[z] + h0) * a.dim;
    // AHEAD heads' loads are in flight
    Pairs<T, P, SIDE> xr[AHEAD][SLOTS], gr[AHEAD][SLOTS];
    auto fetch = [&](int ring) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < SLOTS; ++u) {
        if (!GRAD || norm) xr[ring][u].load(x, at, vi[u], vj[u]);
        if (GRAD && dy) gr[ring][u].load(dy, dat, vi[u], vj[u]);
      }
      at += a.head[z];
      dat += a.dhead[z];
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (h0 + k < h1) fetch(k);
    float2 cs[SLOTS][P];
    {
      const long long slot = a.period == a.tokens ? token : token % a.period;
      const Position position = position_of(a.positions[slot]);
#pragma unroll
      for (int u = 0; u < SLOTS; ++u)
#pragma unroll
        for (int k = 0; k < P; ++k)
          cs[u][k] = pair[u] + k < half ? turn_of(a, position, pair[u] + k) : make_float2(1.f, 0.f);
    }
    for (int first = h0; first < h1; first += AHEAD)
#pragma unroll
    for (int ring = 0; ring < AHEAD; ++ring) {
      const int h = first + ring;
      if (h >= h1) break;
      float v[SLOTS][2 * P], g[SLOTS][2 * P];
#pragma unroll
      for (int u = 0; u < SLOTS; ++u) {
        if (!GRAD || norm) xr[ring][u].get(v[u]);
#pragma unroll
        for (int k = 0; k < 2 * P; ++k) g[u][k] = 0.f;
        if (GRAD && dy) gr[ring][u].get(g[u]);
      }
      if (h + AHEAD < h1) fetch(ring);
      // turns the pairs; back: by the opposite angle
      auto rotate = [&](float (&p)[SLOTS][2 * P], float sign) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < SLOTS; ++u)
#pragma unroll
          for (int k = 0; k < P; ++k) {
            const float i = p[u][k], j = p[u][P + k], s = sign * cs[u][k].y;
            p[u][k] = i * cs[u][k].x - j * s;
            p[u][P + k] = j * cs[u][k].x + i * s;
          }
      };
      float sq = 0.f, dot = 0.f;
      if constexpr (GRAD) rotate(g, -1.f);
      if (norm) {
#pragma unroll
        for (int u = 0; u < SLOTS; ++u)
#pragma unroll
          for (int k = 0; k < 2 * P; ++k) {
            const float e = live[u] ? v[u][k] : 0.f;
            sq += e * e;
            if constexpr (GRAD) dot += g[u][k] * w[u][k] * e;
          }
        for (int o = 1; o < a.lanes; o <<= 1) {
          sq += __shfl_xor(sq, o);
          if constexpr (GRAD) dot += __shfl_xor(dot, o);
        }
        const float r = __builtin_amdgcn_rsqf(sq * inv + a.eps);
        const float m = dot * r * inv;
#pragma unroll
        for (int u = 0; u < SLOTS; ++u)
#pragma unroll
          for (int k = 0; k < 2 * P; ++k) {
            v[u][k] *= r;
            if constexpr (GRAD) {
              dw[u][k] += g[u][k] * v[u][k];
              g[u][k] = r * (g[u][k] * w[u][k] - v[u][k] * m);
            } else {
              v[u][k] *= w[u][k];
            }
          }
      }
      if constexpr (!GRAD) rotate(v, 1.f);
      if (to)
#pragma unroll
        for (int u = 0; u < SLOTS; ++u)
          if (live[u]) {
            Pairs<T, P, SIDE> y;
            y.set(GRAD ? g[u] : v[u]);
            y.store(to, out, vi[u], vj[u]);
          }
      out += a.dim;
    }
  }
  if constexpr (GRAD) {
    if (!a.dw[z]) return;
    // the groups' shares in their order, through LDS
    float* dst = a.part[z] + ((long long)part * gridDim.x + blockIdx.x) * a.dim;
#pragma unroll
    for (int u = 0; u < SLOTS; ++u) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 2 * P; ++k) sums[threadIdx.x][k] = dw[u][k];
      __syncthreads();
      // a thread sums one value: sub's value k
      for (int i = threadIdx.x; i < a.lanes * 2 * P; i += kThreads) {
        const int l = i / (2 * P), k = i % (2 * P), p = (u * a.lanes + l) * P;
        if (p >= a.dim / 2) continue;
        float total = 0.f;
        for (int g = 0; g < groups; ++g) total += sums[g * a.lanes + l][k];
        int vi0, vj0;
        pair_at(a, p, &vi0, &vj0);
        if (P > 1 && vj0 == vi0 + 1) vj0 = vi0 + P;
        dst[value_at<P, SIDE>(vi0, vj0, k)] = total;
      }
    }
  }
}

// Column sums of the blocks' partial rows in a fixed order: 32 columns by 32 strands a block.
__global__ __launch_bounds__(1024) void rotary_heads_sum_kernel(const Heads a) {
  __shared__ float lds[32][33];
  const int z = blockIdx.y, lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, rows = a.parts[z] * a.blocks;
  if (!a.dw[z]) return;
  float s = 0.f;
  if (c < a.dim) {
#pragma unroll 4
    for (int k = strand; k < rows; k += 32) s += a.part[z][(long long)k * a.dim + c];
  }
  lds[strand][lane] = s;
  __syncthreads();
  const int cc = threadIdx.x >> 5;
  s = lds[lane][cc];
  for (int o = 16; o; o >>= 1) s += __shfl_xor(s, o);
  const int oc = blockIdx.x * 32 + cc;
  if (lane == 0 && oc < a.dim) set_element(a.dw[z], a.w_dtype[z], oc, s);
}

constexpr long long kCus = 256;

// Lanes, parts and blocks of a call
void shape(Heads* a, bool grad) {
  a->pairs = a->rotary % 16 == 0 && a->dim % 16 == 0 ? 8 : a->rotary % 8 == 0 && a->dim % 8 == 0 ? 4 : 1;
  const int slots = a->dim / 2 / a->pairs;
  a->lanes = 1;
  while (a->lanes < slots && a->lanes < 64) a->lanes *= 2;
  const int groups = kThreads / a->lanes;
  const long long all = (a->tokens + groups - 1) / groups;
  // few tokens: a group walks few heads. More than 16 a group leave too few groups, fewer form the angles too
  // often: forward and backward over 16384 tokens of 32 + 8 heads of 128 in bf16 72 and 94 us at 16, 74 and
  // 106 at 8, 84 and 114 at 4
  a->per_part = 16;
  auto blocks_at = [&](int per) {
    return all * ((a->heads[0] + per - 1) / per + (a->heads[1] + per - 1) / per);
  };
  while (a->per_part > 1 && blocks_at(a->per_part) < kCus * 4) a->per_part /= 2;
  while ((a->heads[0] + a->heads[1]) / a->per_part > 32768) a->per_part *= 2;    // a grid's second extent
  for (int z = 0; z < 2; ++z) a->parts[z] = (a->heads[z] + a->per_part - 1) / a->per_part;
  // the gradient's partial rows: as many blocks as their registers let run at once (of 512 it took 113 us,
  // of 1024 98, of 768 94)
  const long long most = grad ? (kCus * 3 + a->parts[0] + a->parts[1] - 1) / (a->parts[0] + a->parts[1])
                              : 0x7fffffffLL;
  a->blocks = (int)(all < most ? all : most);
}

template <int T, bool GRAD>
void launch(const Heads& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.blocks, (unsigned)(a.parts[0] + a.parts[1]));
#define DMUON_RH(P, SLOTS, SIDE) \
  hipLaunchKernelGGL((rotary_heads_kernel<T, P, SLOTS, SIDE, GRAD>), grid, dim3(kThreads), 0, stream, a)
  if (a.pairs == 8 && a.interleaved) DMUON_RH(8, 1, true);
  else if (a.pairs == 8) DMUON_RH(8, 1, false);
  else if (a.pairs == 4 && a.interleaved) DMUON_RH(4, 1, true);
  else if (a.pairs == 4) DMUON_RH(4, 1, false);
  else if (a.dim <= 128) DMUON_RH(1, 1, false);
  else DMUON_RH(1, 4, false);
#undef DMUON_RH
}

template <bool GRAD>
hipError_t launch_heads(const Heads& a, hipStream_t stream) {
  if (a.blocks > 0) {
    if (a.dtype == DT_F32) launch<DT_F32, GRAD>(a, stream);
    else if (a.dtype == DT_F16) launch<DT_F16, GRAD>(a, stream);
    else launch<DT_BF16, GRAD>(a, stream);
  }
  if (GRAD && (a.dw[0] || a.dw[1]))
    hipLaunchKernelGGL(rotary_heads_sum_kernel, dim3((unsigned)((a.dim + 31) / 32), 2), dim3(1024), 0, stream,
                       a);
  return hipGetLastError();
}

// Partial rows of the weights' gradients, in bytes
int64_t partials(Heads* h, void* ws) {
  int64_t at = 0;
  for (int z = 0; z < 2; ++z) {
    if (!h->dw[z]) continue;
    h->part[z] = ws ? static_cast<float*>(ws) + at : nullptr;
    at += (int64_t)h->parts[z] * h->blocks * h->dim;
  }
  return at * 4;
}

bool float_code(int c) {
  return c == DMUON_DTYPE_F32 || c == DMUON_DTYPE_BF16 || c == DMUON_DTYPE_F16;
}

int check(const char* who, const dmuon_rotary_heads_args* a) {
  if (!a) return fail("%s: NULL arguments", who);
  if (!float_code(a->dtype) || (a->q_weight && !float_code(a->q_weight_dtype)) ||
      (a->k_weight && !float_code(a->k_weight_dtype)))
    return fail("%s: unknown dtype code", who);
  if (a->tokens < 0 || a->tokens > (1LL << 31) || a->heads < 1 || a->kv_heads < 1 || a->heads > 65536 ||
      a->kv_heads > 65536)
    return fail("%s: tokens must be 0 .. 2^31 and heads 1 .. 65536", who);
  if (a->dim < 2 || a->dim > kMaxDim || a->dim % 2)
    return fail("%s: dim must be even and 2 .. %d, got %lld", who, kMaxDim, (long long)a->dim);
  if (a->rotary_dim < 2 || a->rotary_dim > a->dim || a->rotary_dim % 2)
    return fail("%s: rotary_dim must be even and 2 .. dim, got %lld", who, (long long)a->rotary_dim);
  if (a->tokens > 0 && (a->period < 1 || a->period > a->tokens || a->tokens % a->period))
    return fail("%s: the %lld positions must divide the %lld tokens", who, (long long)a->period,
                (long long)a->tokens);
  if (!a->inv_freq || (a->tokens > 0 && (!a->q || !a->k || !a->positions)))
    return fail("%s: q, k, positions or inv_freq is NULL", who);
  return 0;
}

Heads describe(const dmuon_rotary_heads_args& a, bool grad) {
  Heads h{};
  h.x[0] = a.q; h.x[1] = a.k;
  h.w[0] = a.q_weight; h.w[1] = a.k_weight;
  h.w_dtype[0] = a.q_weight_dtype; h.w_dtype[1] = a.k_weight_dtype;
  h.token[0] = a.q_token; h.head[0] = a.q_head;
  h.token[1] = a.k_token; h.head[1] = a.k_head;
  h.dtoken[0] = a.dq_out_token; h.dhead[0] = a.dq_out_head;
  h.dtoken[1] = a.dk_out_token; h.dhead[1] = a.dk_out_head;
  h.y[0] = a.q_out; h.y[1] = a.k_out;
  h.dy[0] = a.dq_out; h.dy[1] = a.dk_out;
  h.dx[0] = a.dq; h.dx[1] = a.dk;
  h.dw[0] = a.d_q_weight; h.dw[1] = a.d_k_weight;
  h.positions = a.positions;
  h.inv_freq = a.inv_freq;
  h.freq_double = a.inv_freq_double;
  h.tokens = a.tokens;
  h.period = a.period;
  h.heads[0] = (int)a.heads; h.heads[1] = (int)a.kv_heads;
  h.dim = (int)a.dim;
  h.rotary = (int)a.rotary_dim;
  h.interleaved = a.interleaved;
  h.dtype = a.dtype;
  h.eps = a.eps;
  shape(&h, grad);
  return h;
}

}  // namespace
}  // namespace dmuon

using namespace dmuon;

extern "C" {

int dmuon_rotary_heads(const dmuon_rotary_heads_args* args, void* stream) {
  const char* who = "dmuon_rotary_heads";
  if (check(who, args)) return 1;
  if (args->tokens > 0 && (!args->q_out || !args->k_out)) return fail("%s: a result is NULL", who);
  return check_launch(launch_heads<false>(describe(*args, false), static_cast<hipStream_t>(stream)), who);
}

int dmuon_rotary_heads_grad_workspace_size(const dmuon_rotary_heads_args* args, int64_t* workspace_bytes) {
  const char* who = "dmuon_rotary_heads_grad_workspace_size";
  if (!workspace_bytes) return fail("%s: NULL output", who);
  if (check(who, args)) return 1;
  Heads h = describe(*args, true);
  *workspace_bytes = partials(&h, nullptr);
  return 0;
}

int dmuon_rotary_heads_grad(const dmuon_rotary_heads_args* args, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const char* who = "dmuon_rotary_heads_grad";
  if (check(who, args)) return 1;
  if ((args->d_q_weight && !args->q_weight) || (args->d_k_weight && !args->k_weight))
    return fail("%s: a gradient of an operand that is not there", who);
  Heads h = describe(*args, true);
  const int64_t need = partials(&h, workspace);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail("%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", who, (long long)need,
                (long long)workspace_bytes);
  return check_launch(launch_heads<true>(h, static_cast<hipStream_t>(stream)), who);
}

}  // extern "C"
