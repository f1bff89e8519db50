// The norms around a block with its gate and residual scale on gfx950, and their gradients.
//
//   r = rsqrt(mean y^2 + eps), u = y r w_post (u = y without w_post)
//   x' = a x + gate u,  s = rsqrt(mean x'^2 + eps),  h = x' s w_pre
//
// Memory bound: forward reads x and y and writes x' and h; backward reads x, y, dx', dh and writes
// dx and dy. The backward pass forms x' again from x and y in fp32 -- the same bytes as reading the
// rounded x', and its own rounding does not enter the weights' gradients. r and s of every row are
// kept (8 bytes a row), so that a row needs one joint reduction of three sums:
//   A = sum g xhat,  B1 = sum c yhat (e + s g),  B2 = sum c yhat xhat
// with g = w_pre dh, c = gate w_post, xhat = x' s, yhat = y r, e = dx'; then
//   d = e + s (g - xhat A / D),  sum c yhat d = B1 - s A / D B2
//   dx = a d,  dy = r (c d - yhat (sum c yhat d) / D)
// instead of a second reduction that waits for d.
//
// A block keeps its columns in registers -- NV chunks of 8 columns a thread -- and walks a
// contiguous range of rows, so the weights are read once a block (the gate once a group) and the
// gradients of the weights add up in registers; each block then writes one partial row, which a
// second kernel sums in a fixed order.
#include "../../include/dmuon_amd.h"
#include "dmuon_amd_internal.h"
#include "residual_norm.h"

namespace dmuon {
namespace {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
// rows of any pitch and bases of any element alignment: the vectors state the element's alignment
typedef u32x4_t v16_t __attribute__((aligned(2)));
typedef u32x4_t v32_t __attribute__((aligned(4)));

__device__ __forceinline__ float half_to_f(unsigned bits, int t) {
  if (t == DT_F16) return static_cast<float>(__builtin_bit_cast(_Float16, (uint16_t)bits));
  return __uint_as_float(bits << 16);
}
__device__ __forceinline__ unsigned f_to_half(float f, int t) {
  if (t == DT_F16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}

// n (at most 8) values from element `at` on; the rest are 0
__device__ __forceinline__ void load8(const void* p, int t, long long at, int n, float* v) {
  if (t == DT_F32) {
    const float* q = static_cast<const float*>(p) + at;
    if (n >= 8) {
      const u32x4_t a = *(const v32_t*)q, b = *(const v32_t*)(q + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[i + 4] = __uint_as_float(b[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? q[i] : 0.f;
    }
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + at;
    if (n >= 8) {
      const u32x4_t a = *(const v16_t*)q;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = half_to_f(a[i] & 0xffff, t);
        v[2 * i + 1] = half_to_f(a[i] >> 16, t);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? half_to_f(q[i], t) : 0.f;
    }
  }
}
__device__ __forceinline__ void store8(void* p, int t, long long at, int n, const float* v) {
  if (t == DT_F32) {
    float* q = static_cast<float*>(p) + at;
    if (n >= 8) {
      u32x4_t a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[i + 4]);
      *(v32_t*)q = a;
      *(v32_t*)(q + 4) = b;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = v[i];
    }
  } else {
    uint16_t* q = static_cast<uint16_t*>(p) + at;
    if (n >= 8) {
      u32x4_t a;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = f_to_half(v[2 * i], t) | (f_to_half(v[2 * i + 1], t) << 16);
      *(v16_t*)q = a;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = (uint16_t)f_to_half(v[i], t);
    }
  }
}

// Sums of `C` values over the threads of a row (blockDim.x of them): shuffles in a wave, then one
// LDS exchange where the row has several waves. `flip` alternates so that a row's values are not
// overwritten while the row before is still being read.
template <int C>
__device__ __forceinline__ void row_sums(float* v, float (*lds)[4][16][C], int flip) {
#pragma unroll
  for (int c = 0; c < C; ++c)
    for (int o = 1; o < 64; o <<= 1) v[c] += __shfl_xor(v[c], o);
  const int waves = blockDim.x >> 6;
  if (waves == 1) return;
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int c = 0; c < C; ++c) lds[flip][threadIdx.y][w][c] = v[c];
  __syncthreads();
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] = lds[flip][threadIdx.y][0][c];
  for (int k = 1; k < waves; ++k)
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] += lds[flip][threadIdx.y][k][c];
}

template <int T, int NV>
__global__ __launch_bounds__(NV == 1 ? 256 : NV == 2 ? 512 : 1024) void residual_norm_kernel(ResidualNorm a) {
  __shared__ float lds[2][4][16][1];
  const float inv = 1.f / (float)a.dim;
  const long long first = (long long)blockIdx.x * a.rows_per_block;
  const long long end = first + a.rows_per_block < a.rows ? first + a.rows_per_block : a.rows;
  int cnt[NV];
  float pre[NV][8], post[NV][8], gate[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * blockDim.x + threadIdx.x) * 8;
    cnt[v] = a.dim - c;
    if (cnt[v] <= 0) cnt[v] = 0;
    load8(a.w_pre, a.pre_dtype, c, cnt[v], pre[v]);
#pragma unroll
    for (int i = 0; i < 8; ++i) post[v][i] = gate[v][i] = 1.f;
    if (a.w_post) load8(a.w_post, a.post_dtype, c, cnt[v], post[v]);
  }
  long long group = -1;
  for (long long base = first; base < end; base += blockDim.y) {
    const long long row = base + threadIdx.y < end ? base + threadIdx.y : end - 1;
    float x[NV][8], y[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * blockDim.x + threadIdx.x) * 8;
      load8(a.x, T, row * a.ld_x + c, cnt[v], x[v]);
      if (a.y) load8(a.y, T, row * a.ld_y + c, cnt[v], y[v]);
    }
    if (a.gate) {
      const long long g = row / a.rows_per_group;
      if (g != group) {
        group = g;
#pragma unroll
        for (int v = 0; v < NV; ++v)
          load8(a.gate, a.gate_dtype, g * a.dim + (v * blockDim.x + threadIdx.x) * 8, cnt[v], gate[v]);
      }
    }
    float r = 1.f;
    if (a.y && a.w_post) {
      float sq[1] = {0.f};
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) sq[0] += y[v][i] * y[v][i];
      row_sums<1>(sq, lds, 0);
      r = 1.f / sqrtf(sq[0] * inv + a.eps);
    }
    float sq[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[v][i] *= a.scale;
        if (a.y) x[v][i] += gate[v][i] * (y[v][i] * r * post[v][i]);
        sq[0] += x[v][i] * x[v][i];
      }
    row_sums<1>(sq, lds, 1);
    const float s = 1.f / sqrtf(sq[0] * inv + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const long long at = row * a.dim + (v * blockDim.x + threadIdx.x) * 8;
      if (a.x_new) store8(a.x_new, T, at, cnt[v], x[v]);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[v][i] = x[v][i] * s * pre[v][i];
      store8(a.h, T, at, cnt[v], x[v]);
    }
    if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(r, s);
    // one more meeting before the first exchange's values are overwritten by the next row
    if (blockDim.x > 64 && !(a.y && a.w_post)) __syncthreads();
  }
}

template <int T, int NV>
__global__ __launch_bounds__(NV == 1 ? 256 : NV == 2 ? 512 : 1024) void residual_norm_grad_kernel(ResidualNorm a) {
  __shared__ float lds[2][4][16][3];
  const float inv = 1.f / (float)a.dim;
  // rows of this block: a part of one gate group, or several whole groups
  long long first, end;
  if (a.parts > 1) {
    const long long g = blockIdx.x / a.parts, p = blockIdx.x % a.parts;
    first = g * a.rows_per_group + p * a.rows_per_block;
    const long long stop = (g + 1) * a.rows_per_group;
    end = first + a.rows_per_block < stop ? first + a.rows_per_block : stop;
  } else {
    first = (long long)blockIdx.x * a.rows_per_block;
    end = first + a.rows_per_block < a.rows ? first + a.rows_per_block : a.rows;
  }
  int cnt[NV];
  float pre[NV][8], post[NV][8], gate[NV][8];
  float d_pre[NV][8], d_post[NV][8], d_gate[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * blockDim.x + threadIdx.x) * 8;
    cnt[v] = a.dim - c;
    if (cnt[v] <= 0) cnt[v] = 0;
    load8(a.w_pre, a.pre_dtype, c, cnt[v], pre[v]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      post[v][i] = gate[v][i] = 1.f;
      d_pre[v][i] = d_post[v][i] = d_gate[v][i] = 0.f;
    }
    if (a.w_post) load8(a.w_post, a.post_dtype, c, cnt[v], post[v]);
  }
  int flip = 0;
  long long group = -1;
  for (long long row = first; row < end; ++row) {
    float x[NV][8], y[NV][8], e[NV][8], g[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * blockDim.x + threadIdx.x) * 8;
      load8(a.x, T, row * a.ld_x + c, cnt[v], x[v]);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[v][i] = e[v][i] = g[v][i] = 0.f;
      if (a.y) load8(a.y, T, row * a.ld_y + c, cnt[v], y[v]);
      if (a.dx_new) load8(a.dx_new, T, row * a.ld_dx_new + c, cnt[v], e[v]);
      if (a.dh) load8(a.dh, T, row * a.ld_dh + c, cnt[v], g[v]);
    }
    if (a.gate) {
      const long long q = row / a.rows_per_group;
      if (q != group) {
        group = q;
#pragma unroll
        for (int v = 0; v < NV; ++v)
          load8(a.gate, a.gate_dtype, q * a.dim + (v * blockDim.x + threadIdx.x) * 8, cnt[v], gate[v]);
      }
    }
    const float2 rs = a.stats[row];
    const float r = rs.x, s = rs.y;
    float sums[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[v][i] *= r;                                   // yhat
        x[v][i] = a.scale * x[v][i];
        if (a.y) x[v][i] += gate[v][i] * (y[v][i] * post[v][i]);
        x[v][i] *= s;                                   // xhat
        d_pre[v][i] += g[v][i] * x[v][i];
        g[v][i] *= pre[v][i];
        const float cy = gate[v][i] * post[v][i] * y[v][i];
        e[v][i] += s * g[v][i];
        sums[0] += g[v][i] * x[v][i];
        sums[1] += cy * e[v][i];
        sums[2] += cy * x[v][i];
      }
    row_sums<3>(sums, lds, flip);
    flip ^= 1;
    const float ka = s * sums[0] * inv;
    const float kb = a.w_post ? (sums[1] - ka * sums[2]) * inv : 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const long long at = row * a.dim + (v * blockDim.x + threadIdx.x) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = e[v][i] - ka * x[v][i];
        const float du = gate[v][i] * d;
        d_gate[v][i] += d * (y[v][i] * post[v][i]);
        d_post[v][i] += du * y[v][i];
        x[v][i] = a.scale * d;
        y[v][i] = r * (post[v][i] * du - y[v][i] * kb);
      }
      if (a.dx) store8(a.dx, T, at, cnt[v], x[v]);
      if (a.dy) store8(a.dy, T, at, cnt[v], y[v]);
    }
    // the end of a gate group (parts == 1: its gradient is whole), or of this block's part
    if (a.d_gate && (row + 1 == end || (row + 1) % a.rows_per_group == 0)) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * blockDim.x + threadIdx.x) * 8;
        if (a.parts > 1)
          store8(a.gate_part, DT_F32, (long long)blockIdx.x * a.dim + c, cnt[v], d_gate[v]);
        else
          store8(a.d_gate, a.gate_dtype, row / a.rows_per_group * a.dim + c, cnt[v], d_gate[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) d_gate[v][i] = 0.f;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const long long at = (long long)blockIdx.x * a.dim + (v * blockDim.x + threadIdx.x) * 8;
    if (a.d_pre) store8(a.pre_part, DT_F32, at, cnt[v], d_pre[v]);
    if (a.d_post) store8(a.post_part, DT_F32, at, cnt[v], d_post[v]);
  }
}

// out[g][c] = sum of rows g * n .. g * n + n - 1 of part [..][dim], 64 columns a block, 16 strands.
__global__ __launch_bounds__(1024) void sum_rows_kernel(const float* __restrict__ part, long long n,
                                                        int dim, void* out, int dtype) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, strand = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  const long long g = blockIdx.y;
  float s = 0.f;
  if (c < dim)
    for (long long k = strand; k < n; k += 16) s += part[(g * n + k) * dim + c];
  lds[strand][lane] = s;
  __syncthreads();
  if (strand || c >= dim) return;
  for (int k = 1; k < 16; ++k) s += lds[k][lane];
  if (dtype == DT_F32) static_cast<float*>(out)[g * dim + c] = s;
  else static_cast<uint16_t*>(out)[g * dim + c] = (uint16_t)f_to_half(s, dtype);
}

// Threads of a row and chunks of 8 columns a thread: as few waves as hold the row with one chunk,
// then two (whose gradients fit the registers of 512 threads), then four.
bool row_shape(int dim, int* threads, int* nv) {
  const int chunks = (dim + 7) / 8;
  for (int t = 64; t <= 1024; t *= 2)
    for (int v = 1; v <= 4; v *= 2)
      if (t * v >= chunks && (v == 1 ? t <= 256 : v == 2 ? t <= 512 : t == 1024)) {
        *threads = t;
        *nv = v;
        return true;
      }
  return false;
}

constexpr long long kGradBlocks = 1024;

}  // namespace

void residual_norm_split(ResidualNorm* a) {
  const long long groups = a->gate ? a->rows / a->rows_per_group : 1;
  const long long per = a->gate ? a->rows_per_group : a->rows;
  if (!a->gate) a->rows_per_group = a->rows > 0 ? a->rows : 1;
  if (groups >= kGradBlocks || per <= 1) {
    const long long gpb = (groups + kGradBlocks - 1) / kGradBlocks;
    a->parts = 1;
    a->rows_per_block = gpb * (per > 0 ? per : 1);
    a->blocks = groups > 0 ? (groups + gpb - 1) / gpb : 0;
    if (a->rows == 0) a->blocks = 0;
    return;
  }
  long long parts = kGradBlocks / groups;
  if (parts > per) parts = per;
  a->rows_per_block = (per + parts - 1) / parts;
  a->parts = (int)((per + a->rows_per_block - 1) / a->rows_per_block);
  a->blocks = groups * a->parts;
}

hipError_t launch_residual_norm(ResidualNorm a, hipStream_t stream) {
  int threads, nv;
  if (!row_shape(a.dim, &threads, &nv)) return hipErrorInvalidValue;
  if (a.rows <= 0) return hipSuccess;
  const int ry = threads < 256 ? 256 / threads : 1;
  // a few rows a block once every CU has eight blocks
  a.rows_per_block = (a.rows + 2047) / 2048;
  a.rows_per_block = (a.rows_per_block + ry - 1) / ry * ry;
  const dim3 grid((unsigned)((a.rows + a.rows_per_block - 1) / a.rows_per_block));
#define DMUON_RN(T, NV) \
  hipLaunchKernelGGL((residual_norm_kernel<T, NV>), grid, dim3(threads, ry), 0, stream, a)
#define DMUON_RN_T(NV)                              \
  do {                                              \
    if (a.dtype == DT_F32) DMUON_RN(DT_F32, NV);    \
    else if (a.dtype == DT_F16) DMUON_RN(DT_F16, NV); \
    else DMUON_RN(DT_BF16, NV);                     \
  } while (0)
  if (nv == 1) DMUON_RN_T(1);
    else if (nv == 2) DMUON_RN_T(2);
    else DMUON_RN_T(4);
#undef DMUON_RN_T
#undef DMUON_RN
  return hipGetLastError();
}

hipError_t launch_residual_norm_grad(const ResidualNorm& a, hipStream_t stream) {
  int threads, nv;
  if (!row_shape(a.dim, &threads, &nv) || a.blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  if (a.blocks > 0) {
    const dim3 grid((unsigned)a.blocks);
#define DMUON_RN(T, NV) \
  hipLaunchKernelGGL((residual_norm_grad_kernel<T, NV>), grid, dim3(threads), 0, stream, a)
#define DMUON_RN_T(NV)                              \
  do {                                              \
    if (a.dtype == DT_F32) DMUON_RN(DT_F32, NV);    \
    else if (a.dtype == DT_F16) DMUON_RN(DT_F16, NV); \
    else DMUON_RN(DT_BF16, NV);                     \
  } while (0)
    if (nv == 1) DMUON_RN_T(1);
    else if (nv == 2) DMUON_RN_T(2);
    else DMUON_RN_T(4);
#undef DMUON_RN_T
#undef DMUON_RN
  }
  const unsigned cols = (unsigned)((a.dim + 63) / 64);
  auto sum = [&](const float* part, long long groups, long long n, void* out, int dtype) {
    hipLaunchKernelGGL(sum_rows_kernel, dim3(cols, (unsigned)groups), dim3(1024), 0, stream, part,
                       n, a.dim, out, dtype);
  };
  if (a.d_pre) sum(a.pre_part, 1, a.blocks, a.d_pre, a.pre_dtype);
  if (a.d_post) sum(a.post_part, 1, a.blocks, a.d_post, a.post_dtype);
  if (a.d_gate && a.parts > 1)
    sum(a.gate_part, a.rows / a.rows_per_group, a.parts, a.d_gate, a.gate_dtype);
  return hipGetLastError();
}

}  // namespace dmuon

using namespace dmuon;

namespace {

constexpr int64_t kMaxDim = 32768;

int check(const char* who, const dmuon_residual_norm_args* a) {
  if (!a) return fail("%s: NULL arguments", who);
  const int codes[4] = {a->dtype, a->pre_dtype, a->w_post ? a->post_dtype : a->dtype,
                        a->gate ? a->gate_dtype : a->dtype};
  for (int c : codes)
    if (c != DMUON_DTYPE_F32 && c != DMUON_DTYPE_BF16 && c != DMUON_DTYPE_F16)
      return fail("%s: unknown dtype code %d", who, c);
  if (a->rows < 0 || a->rows > (1LL << 31) || a->dim < 1 || a->dim > kMaxDim)
    return fail("%s: rows must be 0 .. 2^31 and dim 1 .. %lld, got %lld and %lld", who,
                (long long)kMaxDim, (long long)a->rows, (long long)a->dim);
  if (!a->w_pre) return fail("%s: w_pre is NULL", who);
  if (a->rows > 0 && !a->y && (a->w_post || a->gate))
    return fail("%s: w_post and gate need the block's output y", who);
  if (a->gate && (a->gates < 1 || a->rows % a->gates != 0))
    return fail("%s: the %lld gate rows must divide the %lld rows", who, (long long)a->gates,
                (long long)a->rows);
  if (a->rows > 0 && (!a->x || a->ld_x < a->dim || (a->y && a->ld_y < a->dim)))
    return fail("%s: x is NULL or a pitch is under dim", who);
  return 0;
}

ResidualNorm describe(const dmuon_residual_norm_args& a) {
  ResidualNorm r{};
  r.x = a.x; r.y = a.y; r.dtype = a.dtype;
  r.ld_x = a.ld_x; r.ld_y = a.ld_y;
  r.w_pre = a.w_pre; r.w_post = a.w_post; r.gate = a.gate;
  r.pre_dtype = a.pre_dtype; r.post_dtype = a.post_dtype; r.gate_dtype = a.gate_dtype;
  r.rows = a.rows; r.dim = (int)a.dim;
  r.rows_per_group = a.gate && a.rows > 0 ? a.rows / a.gates : 1;
  r.scale = a.scale; r.eps = a.eps;
  r.stats = reinterpret_cast<float2*>(a.stats);
  return r;
}

// Partial rows of the weights' gradients in the workspace, in floats.
int64_t partials(ResidualNorm* r, const dmuon_residual_norm_args& a, char* ws) {
  residual_norm_split(r);
  int64_t at = 0;
  auto take = [&](bool want, int64_t n) {
    float* p = want && ws ? reinterpret_cast<float*>(ws) + at : nullptr;
    if (want) at += n;
    return p;
  };
  r->pre_part = take(a.d_pre != nullptr, r->blocks * a.dim);
  r->post_part = take(a.d_post != nullptr, r->blocks * a.dim);
  r->gate_part = take(a.d_gate && r->parts > 1, r->blocks * a.dim);
  return at;
}

}  // namespace

extern "C" {

int dmuon_residual_norm(const dmuon_residual_norm_args* args, void* stream) {
  const char* who = "dmuon_residual_norm";
  if (check(who, args)) return 1;
  if (args->rows > 0 && !args->h) return fail("%s: h is NULL", who);
  ResidualNorm r = describe(*args);
  r.x_new = args->x_new;
  r.h = args->h;
  if (!r.gate) r.rows_per_group = args->rows > 0 ? args->rows : 1;
  return check_launch(launch_residual_norm(r, static_cast<hipStream_t>(stream)), who);
}

int dmuon_residual_norm_grad_workspace_size(const dmuon_residual_norm_args* args,
                                            int64_t* workspace_bytes) {
  const char* who = "dmuon_residual_norm_grad_workspace_size";
  if (!workspace_bytes) return fail("%s: NULL output", who);
  if (check(who, args)) return 1;
  ResidualNorm r = describe(*args);
  *workspace_bytes = partials(&r, *args, nullptr) * 4;
  return 0;
}

int dmuon_residual_norm_grad(const dmuon_residual_norm_args* args, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const char* who = "dmuon_residual_norm_grad";
  if (check(who, args)) return 1;
  const dmuon_residual_norm_args& a = *args;
  if (a.rows > 0 && !a.stats) return fail("%s: stats is NULL", who);
  if ((a.dx_new && a.ld_dx_new < a.dim) || (a.dh && a.ld_dh < a.dim))
    return fail("%s: a pitch is under dim", who);
  if ((a.d_post && !a.w_post) || (a.d_gate && !a.gate) || (a.rows > 0 && a.dy && !a.y))
    return fail("%s: a gradient of an operand that is not there", who);
  ResidualNorm r = describe(a);
  const int64_t need = partials(&r, a, static_cast<char*>(workspace)) * 4;
  if (need > 0 && (!workspace || workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail("%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", who,
                (long long)need, (long long)workspace_bytes);
  r.dx_new = a.dx_new; r.dh = a.dh;
  r.ld_dx_new = a.ld_dx_new; r.ld_dh = a.ld_dh;
  r.dx = a.dx; r.dy = a.dy;
  r.d_pre = a.d_pre; r.d_post = a.d_post; r.d_gate = a.d_gate;
  return check_launch(launch_residual_norm_grad(r, static_cast<hipStream_t>(stream)), who);
}

}  // extern "C"
