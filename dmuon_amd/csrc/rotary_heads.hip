// Norms of queries and keys for each head with the position rotation on gfx950, and their gradients.
//
//   xhat = x rsqrt(mean x^2 + eps), z = xhat w  (no weight: z = x),  y = R(position) z
// R turns the pair (a, b) by the angle t = position inv_freq: (a cos t - b sin t, b cos t + a sin t).
// Backward, g = R^T dy:  dw = sum g xhat,  dx = r (g w - xhat mean(g w xhat)).
//
// Memory bound: forward reads x and writes y; backward reads x and dy and writes dx (the root mean
// square is formed anew). A head's values are spread over 4 pairs a lane: pairs half a rotation apart need
// no exchange between lanes, and one exchange of sums joins the lanes of a head. A block works on a few
// tokens, whose cosines and sines it forms once for all heads: in turns, reduced in 64 bits to an eighth
// of a turn around a multiple of a quarter, so that positions of any size keep 32 bits of accuracy.
#include "../../include/dmuon_amd.h"
#include "dmuon_amd_internal.h"
#include "mfma_tile.h"

#pragma clang fp contract(fast)

namespace dmuon {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 512, kMaxAngles = 1024;   // angles a block holds

struct Heads {
  const void* x[2]; void* y[2]; const void* dy[2]; void* dx[2];   // queries, keys
  const void* w[2];                       // [dim] or NULL
  void* dw[2]; float* part;               // [2][blocks][dim]
  long long token[2], head[2], dtoken[2], dhead[2];               // strides in elements
  const int64_t* positions; const void* inv_freq;
  long long tokens, period, tokens_per_block;
  int heads[2], dim, rotary, dtype, w_dtype[2], freq_double, interleaved;
  int lanes;                              // of a head: a power of two
  int at_once;                            // tokens whose angles a block holds
  int blocks;
  float eps;
};

typedef u32x4_t v16_t __attribute__((aligned(2)));
typedef u32x2_t v8_t __attribute__((aligned(2)));

__device__ __forceinline__ float element(const void* p, int t, long long at) {
  if (t == DT_F32) return static_cast<const float*>(p)[at];
  const uint16_t u = static_cast<const uint16_t*>(p)[at];
  return t == DT_F16 ? from_elt<ELT_F16>(u) : from_elt<ELT_BF16>(u);
}
__device__ __forceinline__ void set_element(void* p, int t, long long at, float v) {
  if (t == DT_F32) static_cast<float*>(p)[at] = v;
  else static_cast<uint16_t*>(p)[at] = t == DT_F16 ? to_elt<ELT_F16>(v) : to_elt<ELT_BF16>(v);
}

// Four values of type T from `p`, at any element alignment
template <int T>
__device__ __forceinline__ void load4(const void* p, long long at, float* v) {
  if constexpr (T == DT_F32) {
    typedef f32x4_t f4_t __attribute__((aligned(4)));
    const f32x4_t x = *reinterpret_cast<const f4_t*>(static_cast<const float*>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x[i];
  } else {
    const u32x2_t x = *reinterpret_cast<const v8_t*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t u = (uint16_t)(i & 1 ? x[i / 2] >> 16 : x[i / 2]);
      v[i] = T == DT_F16 ? from_elt<ELT_F16>(u) : from_elt<ELT_BF16>(u);
    }
  }
}
template <int T>
__device__ __forceinline__ void store4(void* p, long long at, const float* v) {
  if constexpr (T == DT_F32) {
    typedef f32x4_t f4_t __attribute__((aligned(4)));
    *reinterpret_cast<f4_t*>(static_cast<float*>(p) + at) = f32x4_t{v[0], v[1], v[2], v[3]};
  } else {
    constexpr int E = T == DT_F16 ? ELT_F16 : ELT_BF16;
    *reinterpret_cast<v8_t*>(static_cast<uint16_t*>(p) + at) =
        u32x2_t{pack2_elt<E>(v[0], v[1]), pack2_elt<E>(v[2], v[3])};
  }
}

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

// P pairs from pair `p` on (P = 4: rotary and dim are multiples of 8): v[0 .. P) are the pairs' first
// values, v[P .. 2P) their second
template <int T, int P>
__device__ __forceinline__ void load_pairs(const Heads& a, const void* src, long long at, int p, float* v) {
  int i, j;
  pair_at(a, p, &i, &j);
  if constexpr (P == 1) {
    v[0] = element(src, T, at + i);
    v[1] = element(src, T, at + j);
  } else {
    const bool apart = j - i > 1;
    float lo[4], hi[4];
    load4<T>(src, at + i, lo);
    load4<T>(src, at + (apart ? j : i + 4), hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float side = k < 2 ? lo[2 * k] : hi[2 * k - 4], next = k < 2 ? lo[2 * k + 1] : hi[2 * k - 3];
      v[k] = apart ? lo[k] : side;
      v[4 + k] = apart ? hi[k] : next;
    }
  }
}
template <int T, int P>
__device__ __forceinline__ void store_pairs(const Heads& a, void* dst, long long at, int p, const float* v) {
  int i, j;
  pair_at(a, p, &i, &j);
  if constexpr (P == 1) {
    set_element(dst, T, at + i, v[0]);
    set_element(dst, T, at + j, v[1]);
  } else {
    const bool apart = j - i > 1;
    float lo[4], hi[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      lo[k] = apart ? v[k] : v[(k & 1) * 4 + k / 2];
      hi[k] = apart ? v[4 + k] : v[(k & 1) * 4 + 2 + k / 2];
    }
    store4<T>(dst, at + i, lo);
    store4<T>(dst, at + (apart ? j : i + 4), hi);
  }
}

// cos and sin of position * inv_freq
__device__ __forceinline__ float2 turn_of(const Heads& a, long long position, int pair) {
  const double f = a.freq_double ? static_cast<const double*>(a.inv_freq)[pair]
                                 : (double)static_cast<const float*>(a.inv_freq)[pair];
  const double turns = (double)position * f * 0.15915494309189533577;
  const double quarters = rint(turns * 4.);
  const float rest = (float)(turns - quarters * 0.25) * 2.f;     // in half turns, at most a quarter
  const int k = (int)(quarters - 4. * floor(quarters * 0.25));
  const float c = cospif(rest), s = sinpif(rest);
  return k == 0 ? make_float2(c, s) : k == 1 ? make_float2(-s, c)
       : k == 2 ? make_float2(-c, -s) : make_float2(s, -c);
}

// GRAD: x and dy to dx and the weights' partial sums; otherwise x to y. SLOTS: of P pairs a lane.
template <int T, int P, int SLOTS, bool GRAD>
__global__ __launch_bounds__(kThreads) void rotary_heads_kernel(const Heads a) {
  __shared__ float2 turn[kMaxAngles];
  __shared__ float sums[GRAD ? kThreads : 1][2 * P + 1];
  const int sub = threadIdx.x % a.lanes, group = threadIdx.x / a.lanes, groups = kThreads / a.lanes;
  const int half = a.rotary / 2, pairs = a.dim / 2, all = a.heads[0] + a.heads[1];
  const float inv = 1.f / (float)a.dim;
  int pair[SLOTS];
  bool live[SLOTS];
  float w[2][SLOTS][2 * P], dw[2][SLOTS][2 * P];
#pragma unroll
  for (int u = 0; u < SLOTS; ++u) {
    pair[u] = (u * a.lanes + sub) * P;
    live[u] = pair[u] < pairs;
    if (!live[u]) pair[u] = 0;
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int i = 0; i < 2 * P; ++i) {
        int at[2];
        pair_at(a, pair[u] + i % P, &at[0], &at[1]);
        w[z][u][i] = a.w[z] && live[u] ? element(a.w[z], a.w_dtype[z], at[i / P]) : 1.f;
        dw[z][u][i] = 0.f;
      }
  }
  const long long begin = (long long)blockIdx.x * a.tokens_per_block;
  const long long end = begin + a.tokens_per_block < a.tokens ? begin + a.tokens_per_block : a.tokens;
  for (long long t0 = begin; t0 < end; t0 += a.at_once) {
    const int n = end - t0 < a.at_once ? (int)(end - t0) : a.at_once;
    __syncthreads();
    for (int i = threadIdx.x; i < n * half; i += kThreads)
      turn[i] = turn_of(a, a.positions[a.period == a.tokens ? t0 + i / half : (t0 + i / half) % a.period],
                        i % half);
    __syncthreads();
    for (int i = group; i < (n * all + groups - 1) / groups * groups; i += groups) {
      // groups past the last head repeat it without a share of the sums
      const bool mine = i < n * all;
      const int it = mine ? i : n * all - 1;
      const int t = it / all, hd = it - t * all, z = hd >= a.heads[0];
      const int hz = z ? hd - a.heads[0] : hd;
      const bool norm = z ? a.w[1] != nullptr : a.w[0] != nullptr;
      const long long token = t0 + t;
      const long long at = token * (z ? a.token[1] : a.token[0]) + hz * (z ? a.head[1] : a.head[0]);
      const long long out = (token * (z ? a.heads[1] : a.heads[0]) + hz) * a.dim;
      const void* src = z ? a.x[1] : a.x[0];
      float x[SLOTS][2 * P], g[SLOTS][2 * P];
      if constexpr (GRAD) {
        const void* dsrc = z ? a.dy[1] : a.dy[0];
        const long long dat = token * (z ? a.dtoken[1] : a.dtoken[0]) + hz * (z ? a.dhead[1] : a.dhead[0]);
#pragma unroll
        for (int u = 0; u < SLOTS; ++u) {
          if (dsrc) load_pairs<T, P>(a, dsrc, dat, pair[u], g[u]);
          else
#pragma unroll
            for (int k = 0; k < 2 * P; ++k) g[u][k] = 0.f;
        }
      }
      if (!GRAD || norm)
#pragma unroll
        for (int u = 0; u < SLOTS; ++u) load_pairs<T, P>(a, src, at, pair[u], x[u]);
      // turns the pairs of v; back: by the opposite angle
      auto rotate = [&](float (&v)[SLOTS][2 * P], float sign) {
#pragma unroll
        for (int u = 0; u < SLOTS; ++u)
#pragma unroll
          for (int k = 0; k < P; ++k)
            if (pair[u] + k < half) {
              const float2 cs = turn[t * half + pair[u] + k];
              const float p = v[u][k], q = v[u][P + k], s = sign * cs.y;
              v[u][k] = p * cs.x - q * s;
              v[u][P + k] = q * cs.x + p * s;
            }
      };
      float sq = 0.f, dot = 0.f;
      if constexpr (GRAD) {
        rotate(g, -1.f);
        if (norm) {
#pragma unroll
          for (int u = 0; u < SLOTS; ++u)
#pragma unroll
            for (int k = 0; k < 2 * P; ++k)
              if (live[u]) {
                sq += x[u][k] * x[u][k];
                dot += g[u][k] * (z ? w[1][u][k] : w[0][u][k]) * x[u][k];
              }
          for (int o = 1; o < a.lanes; o <<= 1) sq += __shfl_xor(sq, o), dot += __shfl_xor(dot, o);
          const float r = 1.f / sqrtf(sq * inv + a.eps);
          const float m = dot * r * inv;
#pragma unroll
          for (int u = 0; u < SLOTS; ++u)
#pragma unroll
            for (int k = 0; k < 2 * P; ++k) {
              const float xh = x[u][k] * r;
              const float share = mine ? g[u][k] * xh : 0.f;
              dw[0][u][k] += z ? 0.f : share;
              dw[1][u][k] += z ? share : 0.f;
              g[u][k] = r * (g[u][k] * (z ? w[1][u][k] : w[0][u][k]) - xh * m);
            }
        }
        void* dst = z ? a.dx[1] : a.dx[0];
        if (dst && mine)
#pragma unroll
          for (int u = 0; u < SLOTS; ++u)
            if (live[u]) store_pairs<T, P>(a, dst, out, pair[u], g[u]);
      } else {
        if (norm) {
#pragma unroll
          for (int u = 0; u < SLOTS; ++u)
#pragma unroll
            for (int k = 0; k < 2 * P; ++k)
              if (live[u]) sq += x[u][k] * x[u][k];
          for (int o = 1; o < a.lanes; o <<= 1) sq += __shfl_xor(sq, o);
          const float r = 1.f / sqrtf(sq * inv + a.eps);
#pragma unroll
          for (int u = 0; u < SLOTS; ++u)
#pragma unroll
            for (int k = 0; k < 2 * P; ++k) x[u][k] = x[u][k] * r * (z ? w[1][u][k] : w[0][u][k]);
        }
        rotate(x, 1.f);
        void* dst = z ? a.y[1] : a.y[0];
        if (mine)
#pragma unroll
          for (int u = 0; u < SLOTS; ++u)
            if (live[u]) store_pairs<T, P>(a, dst, out, pair[u], x[u]);
      }
    }
  }
  if constexpr (GRAD) {
    // the groups' shares in their order, through LDS
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      if (!a.dw[z]) continue;
      float* dst = a.part + ((long long)z * a.blocks + blockIdx.x) * a.dim;
#pragma unroll
      for (int u = 0; u < SLOTS; ++u) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2 * P; ++k) sums[threadIdx.x][k] = dw[z][u][k];
        __syncthreads();
        if (group || !live[u]) continue;
#pragma unroll
        for (int k = 0; k < 2 * P; ++k) {
          float total = 0.f;
          for (int g = 0; g < groups; ++g) total += sums[g * a.lanes + sub][k];
          int at[2];
          pair_at(a, pair[u] + k % P, &at[0], &at[1]);
          dst[at[k / P]] = total;
        }
      }
    }
  }
}

// Column sums of the blocks' partial rows in a fixed order: 32 columns by 32 strands a block.
__global__ __launch_bounds__(1024) void rotary_heads_sum_kernel(const Heads a) {
  __shared__ float lds[32][33];
  const int z = blockIdx.y, lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  if (!a.dw[z]) return;
  float s = 0.f;
  if (c < a.dim)
    for (int k = strand; k < a.blocks; k += 32) s += a.part[((long long)z * a.blocks + k) * a.dim + c];
  lds[strand][lane] = s;
  __syncthreads();
  const int cc = threadIdx.x >> 5;
  s = lds[lane][cc];
  for (int o = 16; o; o >>= 1) s += __shfl_xor(s, o);
  const int oc = blockIdx.x * 32 + cc;
  if (lane == 0 && oc < a.dim) set_element(a.dw[z], a.w_dtype[z], oc, s);
}

constexpr int64_t kCus = 256;

// Lanes, tokens and blocks of a call
void shape(Heads* a, bool grad) {
  const bool four = a->rotary % 8 == 0 && a->dim % 8 == 0;
  const int slots = four ? a->dim / 8 : a->dim / 2;
  a->lanes = 4;
  while (a->lanes < slots && a->lanes < 64) a->lanes *= 2;
  const int half = a->rotary / 2;
  a->at_once = half ? kThreads / half : 8;
  if (a->at_once < 1) a->at_once = 1;
  if (a->at_once > 16) a->at_once = 16;
  const long long want = grad ? kCus * 4 : 0x7fffffffLL;
  a->tokens_per_block = (a->tokens + want - 1) / want;
  a->tokens_per_block = (a->tokens_per_block + a->at_once - 1) / a->at_once * a->at_once;
  if (a->tokens_per_block < 1) a->tokens_per_block = 1;
  a->blocks = (int)((a->tokens + a->tokens_per_block - 1) / a->tokens_per_block);
}

template <int T, bool GRAD>
void launch(const Heads& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.blocks);
  const bool four = a.rotary % 8 == 0 && a.dim % 8 == 0;
  if (four)
    hipLaunchKernelGGL((rotary_heads_kernel<T, 4, 1, GRAD>), grid, dim3(kThreads), 0, stream, a);
  else if (a.dim <= 128)
    hipLaunchKernelGGL((rotary_heads_kernel<T, 1, 1, GRAD>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((rotary_heads_kernel<T, 1, 4, GRAD>), grid, dim3(kThreads), 0, stream, a);
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
  *workspace_bytes = args->d_q_weight || args->d_k_weight
                         ? 8LL * describe(*args, true).blocks * args->dim : 0;
  return 0;
}

int dmuon_rotary_heads_grad(const dmuon_rotary_heads_args* args, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const char* who = "dmuon_rotary_heads_grad";
  if (check(who, args)) return 1;
  if ((args->d_q_weight && !args->q_weight) || (args->d_k_weight && !args->k_weight))
    return fail("%s: a gradient of an operand that is not there", who);
  Heads h = describe(*args, true);
  const int64_t need = h.dw[0] || h.dw[1] ? 8LL * h.blocks * h.dim : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail("%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", who, (long long)need,
                (long long)workspace_bytes);
  h.part = static_cast<float*>(workspace);
  return check_launch(launch_heads<true>(h, static_cast<hipStream_t>(stream)), who);
}

}  // extern "C"
