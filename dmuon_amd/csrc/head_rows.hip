// Row kernels of the vocabulary losses on gfx950: targets and their logits, log-sum-exp, loss and
// logit gradient between the products, and the reductions. Sums and exponentials are fp32.
#include "../../include/dmuon_amd.h"
#include "dmuon_amd_internal.h"
#include "head_loss.h"
#include "mfma_tile.h"

namespace dmuon {
namespace {

typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));

constexpr float kInf = __builtin_inff();

__device__ __forceinline__ float wave_sum(float v) {
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
  for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
// Sum (or maximum) over a block of up to 16 waves, in every thread.
template <bool MAX>
__device__ __forceinline__ float block_join(float v, float* lds) {
  v = MAX ? wave_max(v) : wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  const int waves = blockDim.x >> 6;
  float r = lds[0];
  for (int w = 1; w < waves; ++w) r = MAX ? fmaxf(r, lds[w]) : r + lds[w];
  return r;
}

// h . w[k] over `dim` values from element-aligned rows, in every lane, for N rows at once.
template <int E, int N>
__device__ __forceinline__ void wave_dots(const uint16_t* h, const uint16_t* const (&w)[N], int dim,
                                          int lane, float (&s)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = 0.f;
#pragma unroll 2
  for (int c = lane * 8; c + 8 <= dim; c += 512) {
    const u32x4_t x = *reinterpret_cast<const u32x4_any_t*>(h + c);
    u32x4_t y[N];
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] = *reinterpret_cast<const u32x4_any_t*>(w[k] + c);
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[k] = __builtin_fmaf(from_elt<E>(x[e] & 0xffff), from_elt<E>(y[k][e] & 0xffff), s[k]);
        s[k] = __builtin_fmaf(from_elt<E>(x[e] >> 16), from_elt<E>(y[k][e] >> 16), s[k]);
      }
  }
  const int c = dim / 8 * 8 + lane;
  if (c < dim)
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = __builtin_fmaf(from_elt<E>(h[c]), from_elt<E>(w[k][c]), s[k]);
  for (int o = 1; o < 64; o <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] += __shfl_xor(s[k], o);
}

// The entries of a row and their logits. Hard targets: one, with probability 1. A teacher's list:
// softmax of the live logits over the temperature (of their differences from the largest, which the
// temperature cannot overflow), or their exponentials under the teacher's own log-sum-exp. A class outside the vocabulary that is neither the ignored index nor padding makes
// the row's mass NaN, so its loss and gradients show it. The entries' logits are formed here, in
// fp32 from the rows themselves: the products' epilogue would have to search every row's list in
// each of its tiles. Hard targets take one wave a row, lists four.
// Memory bound by the gathered rows of W: 4096 rows of 64 entries x 4096 columns (2.1 GB, classes of
// several rows from the caches) 258 us.
template <int E>
__global__ __launch_bounds__(256) void head_targets_kernel(HeadRows r, const uint16_t* H,
                                                           long long ldh, const uint16_t* W,
                                                           long long ldw, int dim) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float it = 1.f / r.temperature;
  if (r.targets) {
    const int row = blockIdx.x * 4 + wave;
    if (row >= r.n) return;
    const long long t = r.targets[row];
    const bool counted = t != r.ignore_index, inside = t >= 0 && t < r.vocab;
    const bool live = counted && inside;
    float z[1] = {0.f};
    if (live) {
      const uint16_t* const w[1] = {W + t * ldw};
      wave_dots<E, 1>(H + row * ldh, w, dim, lane, z);
    }
    if (lane) return;
    r.ids[row] = live ? (int)t : -1;
    r.probs[row] = live ? 1.f : 0.f;
    r.logits[row] = z[0];
    r.mass[row] = !counted ? -1.f : inside ? 1.f : __builtin_nanf("");
    if (row == 0 && r.peak) *r.peak = 0u;
    return;
  }
  const int row = blockIdx.x;
  const long long base = (long long)row * r.k_list;
  float top = -kInf;
  int live = 0, outside = 0;
  for (int k = lane; k < r.k_list; k += 64) {
    const long long id = r.teacher_ids[base + k];
    if (id < 0) continue;
    live = 1;
    outside |= id >= r.vocab;
    top = fmaxf(top, r.teacher_logits[base + k]);
  }
  live = __any(live);
  outside = __any(outside);
  top = wave_max(top);
  const float from = r.teacher_lse ? 0.f : top, under = r.teacher_lse ? r.teacher_lse[row] : 0.f;
  auto share = [&](float v) { return expf((v - from) * it - under); };
  float sum = 0.f;
  for (int k = lane; k < r.k_list; k += 64)
    if (r.teacher_ids[base + k] >= 0) {
      const float v = r.teacher_logits[base + k];
      sum += v == -kInf ? 0.f : share(v);
    }
  sum = wave_sum(sum);
  const float norm = r.teacher_lse ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  if (wave == 0 && lane == 0) {
    r.mass[row] = !live ? -1.f : outside ? __builtin_nanf("") : r.teacher_lse ? sum : sum * norm;
    if (row == 0 && r.peak) *r.peak = 0u;
  }
  // four entries a wave at a time: their loads and sums overlap
  for (int k0 = 4 * wave; k0 < r.k_list; k0 += 16) {
    const uint16_t* w[4];
    float q[4], z[4];
    int cls[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + e < r.k_list ? k0 + e : k0;
      const long long id = r.teacher_ids[base + k];
      const float v = r.teacher_logits[base + k];          // padding's too: four loads at a time
      q[e] = id < 0 || v == -kInf ? 0.f : share(v) * norm;
      cls[e] = id >= 0 && id < r.vocab && q[e] != 0.f ? (int)id : -1;
      w[e] = W + (cls[e] < 0 ? 0 : cls[e]) * ldw;         // an entry without a class: any row
    }
    wave_dots<E, 4>(H + row * ldh, w, dim, lane, z);
    if (lane) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (k0 + e >= r.k_list) continue;
      r.ids[base + k0 + e] = cls[e];
      r.probs[base + k0 + e] = q[e];
      r.logits[base + k0 + e] = z[e] * it;
    }
  }
}

// What a row's stored logit gradient is multiplied with: 2^kGradShift, 0 for a row that is not
// counted; with gradients of the rows' losses, times the row's share of the largest.
constexpr float kUnit = (float)(1 << kGradShift);
__device__ __forceinline__ float row_weight(const HeadRows& r, long long n) {
  return r.mass[n] < 0.f ? 0.f : r.row_grad ? r.row_weight[n] : kUnit;
}

// Row weights and alpha from the rows' gradients: the gradient of row n is alpha * row_weight[n] *
// (...). The weights are relative to the largest, so that a 16-bit logit gradient neither over- nor
// underflows with the size of the batch or a loss scale. The largest finite one: an infinite gradient
// is its own row's. One block.
__global__ __launch_bounds__(1024) void head_weights_kernel(HeadRows r) {
  __shared__ float lds[16];
  float top = 0.f;
  for (int n = threadIdx.x; n < r.n; n += 1024)
    if (!(r.mass[n] < 0.f) && fabsf(r.row_grad[n]) < kInf) top = fmaxf(top, fabsf(r.row_grad[n]));
  top = block_join<true>(top, lds);
  if (top == 0.f) top = 1.f;
  for (int n = threadIdx.x; n < r.n; n += 1024)
    r.row_weight[n] = r.row_grad[n] == 0.f ? 0.f : kUnit * (r.row_grad[n] / top);
  if (threadIdx.x == 0) r.alpha[0] = top * r.temperature / kUnit;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// (maximum, sum of exponentials) of two sets of logits as one, in units of log 2
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  if (top == -kInf) s += s2;              // empty sets, or a NaN to keep
  else s = s * exp2_fast(m - top) + s2 * exp2_fast(m2 - top);
  m = top;
}

// log-sum-exp, loss, row weight and factor of `side` rows a block (a power of two, at most 16): 1024
// threads, thread t for row t % side, every 1024 / side-th statistic and entry. 8192 rows of 2004 statistics
// (131 MB) 30 us, 4.4 TB/s; a few rows cost their chain of dependent steps, 5 to 9 us.
__global__ __launch_bounds__(1024) void head_lse_kernel(HeadRows r, int first, int rows,
                                                        const float2* __restrict__ stats, int side,
                                                        bool grads) {
  __shared__ float lds[3][16][16];
  const int rl = threadIdx.x & (side - 1), strand = threadIdx.x / side, strands = 1024 / side;
  const int row = blockIdx.x * side + rl, wave = threadIdx.x >> 6;
  const bool in = row < rows;
  const long long n = first + (in ? row : 0);
  const int tiles = (r.vocab + kStatCols - 1) / kStatCols;
  float m = -kInf, s = 0.f;
  if (in) {
#pragma unroll 4
    for (int t = strand; t < tiles; t += strands) {
      const float2 o = stats[(long long)t * rows + row];
      join(m, s, o.x, o.y);
    }
  }
  for (int o = side; o < 64; o <<= 1) {
    const float m2 = __shfl_xor(m, o), s2 = __shfl_xor(s, o);
    join(m, s, m2, s2);
  }
  if ((threadIdx.x & 63) < side) lds[0][wave][rl] = m, lds[1][wave][rl] = s;
  __syncthreads();
  m = lds[0][0][rl], s = lds[1][0][rl];
  for (int w = 1; w < 16; ++w) join(m, s, lds[0][w][rl], lds[1][w][rl]);
  const float lse = (log2f(s) + m) * kLn2;
  const float mass = r.mass[n];
  const bool counted = !(mass < 0.f);
  float loss = 0.f;
  if (in && counted)
    for (int k = strand; k < r.k_list; k += strands) {
      const long long at = n * r.k_list + k;
      if (r.ids[at] < 0) continue;
      const float q = r.probs[at], z = r.logits[at];
      loss += r.targets ? lse - z : q * (logf(q) - (z - lse));
    }
  for (int o = side; o < 64; o <<= 1) loss += __shfl_xor(loss, o);
  if ((threadIdx.x & 63) < side) lds[2][wave][rl] = loss;
  __syncthreads();
  if (!in || strand) return;
  loss = 0.f;
  for (int w = 0; w < 16; ++w) loss += lds[2][w][rl];
  if (counted) {
    loss = loss * r.temperature * r.temperature + r.z_loss * lse * lse;
    if (mass != mass) loss = mass;
  }
  r.top[n] = m;
  r.loss[n] = loss;
  if (grads) {
    const float w = row_weight(r, n);
    r.row_weight[n] = w;
    const float c = mass + 2.f * r.z_loss * lse, top_value = fabsf(w) * (fabsf(c) + mass);
    r.factor[n] = w == 0.f ? 0.f : w * c / s;
    // the largest of the rows: an order of atomics does not show; infinities and NaN stay their row's
    if (r.peak && top_value >= (float)(1 << kPeakBits) && top_value < kInf)
      atomicMax(r.peak, __float_as_uint(top_value));
  }
}

// The reduced loss and alpha of its gradient, by a block of 256 threads: four strands of rows each,
// so that their loads are in flight together.
__device__ __forceinline__ void reduce_losses(const HeadRows& r, float* lds) {
  float sum[4] = {}, count[4] = {};       // the count is exact: at most 2^24 rows
  for (int n = threadIdx.x; n < r.n; n += 1024)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = n + 256 * k < r.n;
      const int m = in ? n + 256 * k : n;
      const float loss = r.loss[m], mass = r.mass[m];
      sum[k] += in ? loss : 0.f;
      count[k] += in && !(mass < 0.f) ? 1.f : 0.f;
    }
  const float total = block_join<false>((sum[0] + sum[1]) + (sum[2] + sum[3]), lds);
  const float rows = block_join<false>((count[0] + count[1]) + (count[2] + count[3]), lds);
  if (threadIdx.x == 0) {
    const float g = r.reduction == DMUON_LOSS_MEAN ? 1.f / fmaxf(rows, 1.f) : 1.f;
    r.mean[0] = r.reduction == DMUON_LOSS_MEAN ? total / fmaxf(rows, 1.f) : total;
    r.alpha[0] = g * r.temperature / kUnit;
  }
}

__device__ __forceinline__ float peak_down(const HeadRows& r) {
  return __uint_as_float((unsigned)(127 - peak_shift(*r.peak)) << 23);
}

// The logit gradient: factor * 2^(z - top) - row_weight * q, in place of the exponentials (whose share
// 2^(m - top) is one of a block's row) or from the logits (LOGITS). Crosses memory once, 2 + 2 bytes
// a logit or 4 + 2: 4 x 32 rows of one block of 64 classes a workgroup, 16 bytes a thread and step.
// A hard target's own class comes from its fp32 logit: softmax - 1 cancels where the student is
// sure. (So the row's maximum and 1 / sum go in apart: their log-sum-exp would lose what 1 - p is
// made of.) LOGITS is fp16: its values shrink by peak_shift.
// Blocks past the rows' are the reduction's, which the products after this kernel wait for and nothing
// in it: a launch of its own cost small calls 4 us.
// Memory bound: 8192 x 128256 in place (4.2 GB) 737 us, 5.7 TB/s.
template <int E, bool LOGITS>
__global__ __launch_bounds__(256) void head_grad_kernel(HeadRows r, int first, int rows,
                                                        const float2* __restrict__ stats,
                                                        const float* __restrict__ Z, uint16_t* G) {
  __shared__ float lds[16];
  const int tile = blockIdx.y, c = threadIdx.x & 7;
  if ((int)blockIdx.x * 128 >= rows) {
    if (tile == 0) reduce_losses(r, lds);
    return;
  }
  const int row0 = blockIdx.x * 128 + (threadIdx.x >> 3);
  const float down = LOGITS ? peak_down(r) : 1.f;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int row = row0 + 32 * p;
    if (row >= rows) return;
    const long long n = first + row, at = ((long long)tile * rows + row) * 64 + 8 * c;
    const float f = r.factor[n] * down, top = r.top[n];
    const int id = r.targets ? r.ids[n] : -1;
    float v[8];
    if (f == 0.f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    } else if constexpr (!LOGITS) {
      const u32x4_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(G + at));
      const float k = f * (1.f / (float)(1 << kExpShift)) *
                      exp2_fast(stats[(long long)tile * rows + row].x - top);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = k * from_elt<ELT_F16>(x[e] & 0xffff);
        v[2 * e + 1] = k * from_elt<ELT_F16>(x[e] >> 16);
      }
    } else {
      const f32x4_t* z = reinterpret_cast<const f32x4_t*>(Z + at);
      const f32x4_t lo = __builtin_nontemporal_load(z), hi = __builtin_nontemporal_load(z + 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = f * exp2_fast(lo[e] - top);
        v[4 + e] = f * exp2_fast(hi[e] - top);
      }
    }
    if (id >> 3 == 8 * tile + c) {
      const float g = f * exp2_fast(__builtin_fmaf(r.logits[n], kLog2e, -top)) - r.row_weight[n] * down;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (id & 7) == e ? g : v[e];
    }
    *reinterpret_cast<u32x4_t*>(G + at) = u32x4_t{pack2_elt<E>(v[0], v[1]), pack2_elt<E>(v[2], v[3]),
                                                  pack2_elt<E>(v[4], v[5]), pack2_elt<E>(v[6], v[7])};
  }
}

// The classes of the teachers' lists, from their fp32 logits: mass p - q cancels where the student
// is sure. Entries of one class in one row sum their probabilities and write the same value. One wave
// a row, 64 entries against 64 from lane to lane: 4096 rows of 64 entries 16 us.
template <int E>
__global__ __launch_bounds__(256) void head_entries_kernel(HeadRows r, int first, int rows,
                                                           uint16_t* G) {
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (row >= rows) return;
  const long long n = first + row;
  const float down = E == ELT_F16 ? peak_down(r) : 1.f;
  const float w = r.row_weight[n] * down, f = r.factor[n] * down, top = r.top[n];
  if (w == 0.f) return;
  const int* ids = r.ids + n * r.k_list;
  const float* probs = r.probs + n * r.k_list;
  for (int k0 = 0; k0 < r.k_list; k0 += 64) {
    const int id = k0 + lane < r.k_list ? ids[k0 + lane] : -1;
    float q = 0.f;
    for (int j0 = 0; j0 < r.k_list; j0 += 64) {
      const int jd = j0 + lane < r.k_list ? ids[j0 + lane] : -1;
      const float jq = j0 + lane < r.k_list ? probs[j0 + lane] : 0.f;
      const int m = min(64, r.k_list - j0);
      for (int j = 0; j < m; ++j) {
        const float p = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(jq), j));
        q += __builtin_amdgcn_readlane(jd, j) == id ? p : 0.f;
      }
    }
    if (id < 0) continue;
    const float p = f == 0.f ? 0.f
        : f * exp2_fast(__builtin_fmaf(r.logits[n * r.k_list + k0 + lane], kLog2e, -top));
    G[((long long)(id >> 6) * rows + row) * 64 + (id & 63)] = to_elt<E>(p - w * q);
  }
}

// The reduced loss alone, of calls without gradients.
__global__ __launch_bounds__(256) void head_reduce_kernel(HeadRows r) {
  __shared__ float lds[16];
  reduce_losses(r, lds);
}

// Eight values a thread, of operand blockIdx.y: one launch for both. Bound by its launch where it
// matters (1003 x 300 and 77 x 300: two launches 3.6 us each); memory bound for a large weight.
__global__ __launch_bounds__(256) void head_pad_kernel(HeadPad a) {
  const int k = blockIdx.y, chunks = a.pad / 8;
  const long long i = blockIdx.x * 256LL + threadIdx.x, row = i / chunks;
  if (row >= a.rows[k]) return;
  const int c = (int)(i - row * chunks) * 8;
  const uint16_t* s = a.src[k] + row * a.ld[k] + c;
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (c + 8 <= a.dim) v = *reinterpret_cast<const u32x4_any_t*>(s);
  else
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < a.dim) v[e >> 1] |= (uint32_t)s[e] << (16 * (e & 1));
  *reinterpret_cast<u32x4_t*>(a.dst[k] + row * a.pad + c) = v;
}

// dst = factor * src for two dense arrays, 8 values a thread and step. Memory bound: 50001 x 1528 and
// 1023 x 1528 values from fp32 to fp16 (468 MB) 98 us, 4.8 TB/s; in place at factor 1 2 to 5 us.
template <int S, int D>
__global__ __launch_bounds__(256) void scale_by_kernel(ScaleBy a) {
  typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));
  const float f = a.factor[0];
  if (S == D && f == 1.f && a.in_place) return;
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const long long n = a.n[k];
    for (long long i = (blockIdx.x * 256LL + threadIdx.x) * 8; i < n; i += 256LL * 8 * gridDim.x) {
      float v[8];
      const bool whole = i + 8 <= n;
      if constexpr (S == DT_F32) {
        const float* p = static_cast<const float*>(a.src[k]) + i;
        if (whole) {
          const f32x4_t x = *reinterpret_cast<const f32x4_any_t*>(p);
          const f32x4_t y = *reinterpret_cast<const f32x4_any_t*>(p + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = x[e], v[e + 4] = y[e];
        } else {
          for (int e = 0; e < 8; ++e) v[e] = i + e < n ? p[e] : 0.f;
        }
      } else {
        constexpr int E = S == DT_F16 ? ELT_F16 : ELT_BF16;
        const uint16_t* p = static_cast<const uint16_t*>(a.src[k]) + i;
        if (whole) {
          const u32x4_t x = *reinterpret_cast<const u32x4_any_t*>(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[2 * e] = from_elt<E>(x[e] & 0xffff);
            v[2 * e + 1] = from_elt<E>(x[e] >> 16);
          }
        } else {
          for (int e = 0; e < 8; ++e) v[e] = i + e < n ? from_elt<E>(p[e]) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= f;
      if constexpr (D == DT_F32) {
        float* p = static_cast<float*>(a.dst[k]) + i;
        if (whole) {
          *reinterpret_cast<f32x4_any_t*>(p) = f32x4_t{v[0], v[1], v[2], v[3]};
          *reinterpret_cast<f32x4_any_t*>(p + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
        } else {
          for (int e = 0; e < 8; ++e)
            if (i + e < n) p[e] = v[e];
        }
      } else {
        constexpr int E = D == DT_F16 ? ELT_F16 : ELT_BF16;
        uint16_t* p = static_cast<uint16_t*>(a.dst[k]) + i;
        if (whole) {
          *reinterpret_cast<u32x4_any_t*>(p) = u32x4_t{pack2_elt<E>(v[0], v[1]), pack2_elt<E>(v[2], v[3]),
                                                       pack2_elt<E>(v[4], v[5]), pack2_elt<E>(v[6], v[7])};
        } else {
          for (int e = 0; e < 8; ++e)
            if (i + e < n) p[e] = to_elt<E>(v[e]);
        }
      }
    }
  }
}

}  // namespace

hipError_t launch_head_targets(const HeadRows& r, const uint16_t* H, long long ldh,
                               const uint16_t* W, long long ldw, int dim, int elt, bool grads,
                               hipStream_t stream) {
  if (r.n > 0) {
    const dim3 grid((unsigned)(r.targets ? (r.n + 3) / 4 : r.n));
    if (elt == ELT_F16)
      hipLaunchKernelGGL(head_targets_kernel<ELT_F16>, grid, dim3(256), 0, stream, r, H, ldh, W, ldw, dim);
    else
      hipLaunchKernelGGL(head_targets_kernel<ELT_BF16>, grid, dim3(256), 0, stream, r, H, ldh, W, ldw, dim);
  }
  if (grads && r.reduction == DMUON_LOSS_ROWS)
    hipLaunchKernelGGL(head_weights_kernel, dim3(1), dim3(1024), 0, stream, r);
  return hipGetLastError();
}

static hipError_t reduce(const HeadRows& r, hipStream_t stream) {
  if (r.reduction != DMUON_LOSS_ROWS)
    hipLaunchKernelGGL(head_reduce_kernel, dim3(1), dim3(256), 0, stream, r);
  return hipGetLastError();
}

hipError_t launch_head_rows(const HeadRows& r, int first, int rows, const float2* stats,
                            const void* Z, uint16_t* G, int elt, hipStream_t stream) {
  if (rows <= 0) return reduce(r, stream);
  const int tiles = (r.vocab + kStatCols - 1) / kStatCols;
  // Neighbouring rows share the lines of a statistic; few rows take more threads each. Over 128256
  // classes, rows a block 1 / 4 / 16: 64 rows 7.6 / 8.7 / 14.8 us, 256 10.2 / 9.6 / 15.6, 1000 25.8 /
  // 14.2 / 15.9, 2048 42.6 / 25.8 / 16.1. By the call's rows, not the chunk's (256 of 8192 rows lose 6
  // us): it sets the order in which statistics and entries join, and so a loss's bits.
  const int side = r.n >= 1024 ? 16 : r.n >= 128 ? 4 : 1;
  hipLaunchKernelGGL(head_lse_kernel, dim3((unsigned)((rows + side - 1) / side)), dim3(1024), 0,
                     stream, r, first, rows, stats, side, G != nullptr);
  if (!G) return first + rows < r.n ? hipGetLastError() : reduce(r, stream);
  if (tiles > 65535 || (Z == G) != (elt == ELT_BF16) || (elt == ELT_F16) != (r.peak != nullptr))
    return hipErrorInvalidValue;
  const dim3 grid((unsigned)((rows + 127) / 128 + (r.reduction != DMUON_LOSS_ROWS)), (unsigned)tiles);
  const dim3 lists((unsigned)((rows + 3) / 4));
  const float* logits = static_cast<const float*>(Z);
  if (elt == ELT_F16) {
    hipLaunchKernelGGL((head_grad_kernel<ELT_F16, true>), grid, dim3(256), 0, stream, r, first, rows,
                       stats, logits, G);
    if (!r.targets)
      hipLaunchKernelGGL(head_entries_kernel<ELT_F16>, lists, dim3(256), 0, stream, r, first, rows, G);
  } else {
    hipLaunchKernelGGL((head_grad_kernel<ELT_BF16, false>), grid, dim3(256), 0, stream, r, first, rows,
                       stats, nullptr, G);
    if (!r.targets)
      hipLaunchKernelGGL(head_entries_kernel<ELT_BF16>, lists, dim3(256), 0, stream, r, first, rows, G);
  }
  return hipGetLastError();
}

hipError_t launch_head_pad(const HeadPad& a, hipStream_t stream) {
  long long most = 0;
  for (int k = 0; k < a.n; ++k) most = a.rows[k] > most ? a.rows[k] : most;
  if (most == 0) return hipSuccess;
  const long long blocks = (most * (a.pad / 8) + 255) / 256;
  if (a.pad < a.dim || a.pad % 8 != 0 || blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL(head_pad_kernel, dim3((unsigned)blocks, (unsigned)a.n), dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <int S>
static void scale_from(const ScaleBy& a, int dst_dtype, dim3 grid, hipStream_t stream) {
  if (dst_dtype == DT_F32) hipLaunchKernelGGL((scale_by_kernel<S, DT_F32>), grid, dim3(256), 0, stream, a);
  else if (dst_dtype == DT_F16) hipLaunchKernelGGL((scale_by_kernel<S, DT_F16>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((scale_by_kernel<S, DT_BF16>), grid, dim3(256), 0, stream, a);
}

hipError_t launch_scale_by(const ScaleBy& a, int src_dtype, int dst_dtype, hipStream_t stream) {
  const long long n = a.n[0] > a.n[1] ? a.n[0] : a.n[1], want = (n + 2047) / 2048;
  if (want <= 0) return hipSuccess;
  const dim3 grid((unsigned)(want < 2048 ? want : 2048));
  if (src_dtype == DT_F32) scale_from<DT_F32>(a, dst_dtype, grid, stream);
  else if (src_dtype == DT_F16) scale_from<DT_F16>(a, dst_dtype, grid, stream);
  else scale_from<DT_BF16>(a, dst_dtype, grid, stream);
  return hipGetLastError();
}

}  // namespace dmuon
