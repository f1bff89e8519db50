// Row kernels of the vocabulary losses on gfx950: targets, log-sum-exp and loss, the logit
// gradient between the products, and the reductions. All of them stream their rows once; sums and
// exponentials are fp32.
#include "../../include/dmuon_amd.h"
#include "dmuon_amd_internal.h"
#include "head_loss.h"

namespace dmuon {
namespace {

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

// The entries of a row. Hard targets: one, with probability 1. A teacher's list: softmax of the
// live logits over the temperature, or their exponentials under the teacher's own log-sum-exp. A
// class outside the vocabulary that is neither the ignored index nor padding makes the row's mass
// NaN, so its loss and gradients show it. One wave per row.
__global__ __launch_bounds__(256) void head_targets_kernel(HeadRows r) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= r.n) return;
  if (r.targets) {
    if (lane) return;
    const long long t = r.targets[row];
    const bool counted = t != r.ignore_index, inside = t >= 0 && t < r.vocab;
    r.ids[row] = counted && inside ? (int)t : -1;
    r.probs[row] = counted && inside ? 1.f : 0.f;
    r.mass[row] = !counted ? -1.f : inside ? 1.f : __builtin_nanf("");
    return;
  }
  const long long base = (long long)row * r.k_list;
  const float it = 1.f / r.temperature;
  float top = -kInf;
  int live = 0, outside = 0;
  for (int k = lane; k < r.k_list; k += 64) {
    const long long id = r.teacher_ids[base + k];
    if (id < 0) continue;
    live = 1;
    outside |= id >= r.vocab;
    top = fmaxf(top, r.teacher_logits[base + k] * it);
  }
  live = __any(live);
  outside = __any(outside);
  top = wave_max(top);
  const float shift = r.teacher_lse ? r.teacher_lse[row] : top;
  float sum = 0.f;
  for (int k = lane; k < r.k_list; k += 64)
    if (r.teacher_ids[base + k] >= 0) {
      const float v = r.teacher_logits[base + k] * it;
      sum += v == -kInf ? 0.f : expf(v - shift);
    }
  sum = wave_sum(sum);
  const float norm = r.teacher_lse ? 1.f : sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  float mass = 0.f;
  for (int k = lane; k < r.k_list; k += 64) {
    const long long id = r.teacher_ids[base + k];
    float q = 0.f;
    if (id >= 0) {
      const float v = r.teacher_logits[base + k] * it;
      q = v == -kInf ? 0.f : expf(v - shift) * norm;
    }
    r.ids[base + k] = id >= 0 && id < r.vocab ? (int)id : -1;
    r.probs[base + k] = q;
    mass += q;
  }
  mass = wave_sum(mass);
  if (lane == 0) r.mass[row] = !live ? -1.f : outside ? __builtin_nanf("") : mass;
}

// Row weights and alpha: the gradient of row n is alpha * row_weight[n] * (...). The weights are
// relative to the largest, so that a 16-bit logit gradient neither over- nor underflows with the
// size of the batch or a loss scale. One block.
__global__ __launch_bounds__(1024) void head_weights_kernel(HeadRows r) {
  __shared__ float lds[16];
  const float unit = (float)(1 << kGradShift);
  float count = 0.f, top = 0.f;
  for (int n = threadIdx.x; n < r.n; n += 1024)
    if (!(r.mass[n] < 0.f)) {
      count += 1.f;                       // exact: at most 2^24 rows
      if (r.row_grad) top = fmaxf(top, fabsf(r.row_grad[n]));
    }
  count = block_join<false>(count, lds);
  top = block_join<true>(top, lds);
  const float t = r.temperature;
  for (int n = threadIdx.x; n < r.n; n += 1024) {
    const bool counted = !(r.mass[n] < 0.f);
    float w = unit;
    if (r.row_grad) w = r.row_grad[n] == 0.f ? 0.f : unit * (r.row_grad[n] / top);
    r.row_weight[n] = counted ? w : 0.f;
  }
  if (threadIdx.x == 0) {
    const float g = r.row_grad ? top : r.reduction == DMUON_LOSS_MEAN ? 1.f / fmaxf(count, 1.f) : 1.f;
    r.alpha[0] = g * t / unit;
  }
}

// log-sum-exp and loss of 16 rows a block, 16 threads a row.
__global__ __launch_bounds__(256) void head_loss_kernel(HeadRows r, int first, int rows,
                                                        const float* __restrict__ Z, long long ldz,
                                                        const float2* __restrict__ stats) {
  __shared__ float2 part[16][17];
  const int rl = threadIdx.x & 15, strand = threadIdx.x >> 4;
  const int row = blockIdx.x * 16 + rl;
  const int tiles = (r.vocab + kStatCols - 1) / kStatCols;
  float m = -kInf, s = 0.f;
  auto join = [&](float2 o) {
    const float top = fmaxf(m, o.x);
    if (top == -kInf) { s += o.y; return; }
    s = s * expf(m - top) + o.y * expf(o.x - top);
    m = top;
  };
  if (row < rows)
    for (int t = strand; t < tiles; t += 16) join(stats[(long long)t * rows + row]);
  part[strand][rl] = make_float2(m, s);
  __syncthreads();
  if (row >= rows) return;
  m = -kInf;
  s = 0.f;
  for (int k = 0; k < 16; ++k) join(part[k][rl]);
  const float lse = logf(s) + m;
  const long long n = first + row;
  const float mass = r.mass[n];
  float loss = 0.f;
  if (!(mass < 0.f)) {
    for (int k = strand; k < r.k_list; k += 16) {
      const int id = r.ids[n * r.k_list + k];
      const float q = r.probs[n * r.k_list + k];
      if (id < 0 || q == 0.f) continue;
      const float z = Z[(long long)row * ldz + id];
      loss += r.targets ? lse - z : q * (logf(q) - (z - lse));
    }
  }
  __syncthreads();
  part[strand][rl].x = loss;
  __syncthreads();
  if (strand) return;
  loss = 0.f;
  for (int k = 0; k < 16; ++k) loss += part[k][rl].x;
  if (!(mass < 0.f)) {
    loss = loss * r.temperature * r.temperature + r.z_loss * lse * lse;
    if (mass != mass) loss = mass;
  }
  r.lse[n] = lse;
  r.loss[n] = loss;
}

template <int E>
__device__ __forceinline__ uint16_t to_elt(float f) {
  if constexpr (E == ELT_F16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  else return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}
template <int E>
__device__ __forceinline__ float from_elt(uint16_t h) {
  if constexpr (E == ELT_F16) return static_cast<float>(__builtin_bit_cast(_Float16, h));
  else return __uint_as_float(static_cast<uint32_t>(h) << 16);
}

// row weight times mass, with the z-loss term: d(z_loss lse^2) = 2 z_loss lse softmax
__device__ __forceinline__ float row_factor(const HeadRows& r, long long n) {
  return r.row_weight[n] * (r.mass[n] + (r.targets ? 2.f * r.z_loss * r.lse[n] : 0.f));
}

template <int E>
__global__ __launch_bounds__(256) void head_grad_kernel(HeadRows r, int first,
                                                        const float* __restrict__ Z, long long ldz,
                                                        uint16_t* __restrict__ G, long long ldg) {
  const long long n = first + blockIdx.y;
  const long long row = blockIdx.y;
  const int c0 = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (c0 >= ldg) return;
  const float w = r.row_weight[n], f = row_factor(r, n), lse = r.lse[n];
  for (int e = 0; e < 8; ++e) {
    const int c = c0 + e;
    float g = 0.f;
    if (c < r.vocab && w != 0.f) g = f * expf(Z[row * ldz + c] - lse);
    if (c < ldg) G[row * ldg + c] = to_elt<E>(g);
  }
}
// The entries' classes, from their fp32 logits: mass p - q cancels where the student is sure.
// Entries of one class in one row write the same value. One wave per row.
template <int E>
__global__ __launch_bounds__(256) void head_grad_entries_kernel(HeadRows r, int first, int rows,
                                                                const float* __restrict__ Z,
                                                                long long ldz,
                                                                uint16_t* __restrict__ G,
                                                                long long ldg) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  const long long n = first + row;
  const float w = r.row_weight[n], f = row_factor(r, n), lse = r.lse[n];
  if (w == 0.f) return;
  const int* ids = r.ids + n * r.k_list;
  const float* probs = r.probs + n * r.k_list;
  for (int k = lane; k < r.k_list; k += 64) {
    const int id = ids[k];
    if (id < 0) continue;
    float q = 0.f;
    for (int j = 0; j < r.k_list; ++j)
      if (ids[j] == id) q += probs[j];
    G[row * ldg + id] = to_elt<E>(f * expf(Z[(long long)row * ldz + id] - lse) - w * q);
  }
}

__global__ __launch_bounds__(1024) void head_reduce_kernel(HeadRows r) {
  __shared__ float lds[16];
  float sum = 0.f, count = 0.f;
  for (int n = threadIdx.x; n < r.n; n += 1024) {
    sum += r.loss[n];
    count += r.mass[n] < 0.f ? 0.f : 1.f;
  }
  sum = block_join<false>(sum, lds);
  count = block_join<false>(count, lds);
  if (threadIdx.x == 0)
    r.mean[0] = r.reduction == DMUON_LOSS_MEAN ? sum / fmaxf(count, 1.f) : sum;
}

template <int S, int D>
__global__ __launch_bounds__(256) void scale_by_kernel(const void* src, void* dst, long long n,
                                                       const float* factor) {
  const float f = factor[0];
  if (S == D && src == dst && f == 1.f) return;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += 256LL * gridDim.x) {
    float v;
    if constexpr (S == DT_F32) v = static_cast<const float*>(src)[i];
    else v = from_elt<S == DT_F16 ? ELT_F16 : ELT_BF16>(static_cast<const uint16_t*>(src)[i]);
    v *= f;
    if constexpr (D == DT_F32) static_cast<float*>(dst)[i] = v;
    else static_cast<uint16_t*>(dst)[i] = to_elt<D == DT_F16 ? ELT_F16 : ELT_BF16>(v);
  }
}

}  // namespace

hipError_t launch_head_targets(const HeadRows& r, bool grads, hipStream_t stream) {
  if (r.n > 0)
    hipLaunchKernelGGL(head_targets_kernel, dim3((unsigned)((r.n + 3) / 4)), dim3(256), 0, stream, r);
  if (grads) hipLaunchKernelGGL(head_weights_kernel, dim3(1), dim3(1024), 0, stream, r);
  return hipGetLastError();
}

hipError_t launch_head_loss(const HeadRows& r, int first, int rows, const float* Z, long long ldz,
                            const float2* stats, hipStream_t stream) {
  if (rows <= 0) return hipSuccess;
  hipLaunchKernelGGL(head_loss_kernel, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, stream, r,
                     first, rows, Z, ldz, stats);
  return hipGetLastError();
}

hipError_t launch_head_grad(const HeadRows& r, int first, int rows, const float* Z, long long ldz,
                            uint16_t* G, long long ldg, int elt, hipStream_t stream) {
  if (rows <= 0) return hipSuccess;
  const dim3 grid((unsigned)((ldg + 2047) / 2048), (unsigned)rows);
  const dim3 rgrid((unsigned)((rows + 3) / 4));
  if (elt == ELT_F16) {
    hipLaunchKernelGGL(head_grad_kernel<ELT_F16>, grid, dim3(256), 0, stream, r, first, Z, ldz, G, ldg);
    hipLaunchKernelGGL(head_grad_entries_kernel<ELT_F16>, rgrid, dim3(256), 0, stream, r, first,
                       rows, Z, ldz, G, ldg);
  } else {
    hipLaunchKernelGGL(head_grad_kernel<ELT_BF16>, grid, dim3(256), 0, stream, r, first, Z, ldz, G, ldg);
    hipLaunchKernelGGL(head_grad_entries_kernel<ELT_BF16>, rgrid, dim3(256), 0, stream, r, first,
                       rows, Z, ldz, G, ldg);
  }
  return hipGetLastError();
}

hipError_t launch_head_reduce(const HeadRows& r, hipStream_t stream) {
  hipLaunchKernelGGL(head_reduce_kernel, dim3(1), dim3(1024), 0, stream, r);
  return hipGetLastError();
}

template <int S>
static void scale_from(const void* src, void* dst, int dst_dtype, long long n, const float* factor,
                       dim3 grid, hipStream_t stream) {
  if (dst_dtype == DT_F32)
    hipLaunchKernelGGL((scale_by_kernel<S, DT_F32>), grid, dim3(256), 0, stream, src, dst, n, factor);
  else if (dst_dtype == DT_F16)
    hipLaunchKernelGGL((scale_by_kernel<S, DT_F16>), grid, dim3(256), 0, stream, src, dst, n, factor);
  else
    hipLaunchKernelGGL((scale_by_kernel<S, DT_BF16>), grid, dim3(256), 0, stream, src, dst, n, factor);
}

hipError_t launch_scale_by(const void* src, int src_dtype, void* dst, int dst_dtype, long long n,
                           const float* factor, hipStream_t stream) {
  if (n <= 0) return hipSuccess;
  const long long want = (n + 2047) / 2048;
  const dim3 grid((unsigned)(want < 8192 ? want : 8192));
  if (src_dtype == DT_F32) scale_from<DT_F32>(src, dst, dst_dtype, n, factor, grid, stream);
  else if (src_dtype == DT_F16) scale_from<DT_F16>(src, dst, dst_dtype, n, factor, grid, stream);
  else scale_from<DT_BF16>(src, dst, dst_dtype, n, factor, grid, stream);
  return hipGetLastError();
}

}  // namespace dmuon
