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
// A row is spread over blockDim.x threads, 8 columns each (16 past 2048 columns forward, past 8192
// backward), blockDim.y rows side by side. A block keeps its columns' weights in registers and walks
// a contiguous range of rows, the next row's loads in flight under the sums of this one; the weights'
// gradients add up in registers too, and each block writes one partial row, which a second kernel
// sums in a fixed order.
//
// With the weights' gradients, forward and backward in TB/s: bf16 16384 x 4096 100 and 174 us (5.4 and
// 4.6), 8192 x 8192 104 and 161 (5.2, 5.0), 32768 x 2048 5.2 and 4.4; fp32 16384 x 4096 228 and 446
// (4.7, 3.6). Widths whose blocks of 64 to 768 threads leave a part of a CU's waves empty are slower,
// whatever their rows' alignment: bf16 13328 x 6032 164 and 250 us (3.9, 3.9), x 6030 167 and 253,
// 40000 x 1008 4.2 and 4.0, x 1002 4.1 and 3.9; 12288 x 5120 4.2 and 4.8. A gate per token 5.4 and 3.9
// (16384 x 4096), without a block's output 5.4 and 5.0.
//
// Registers: 128 where a block may have 1024 threads. The forward kernel of two chunks spills 29 in
// fp32 and none in 16 bits; the backward kernel of one row a block 24 in fp32 (70 with several gate
// groups a block) and 5 (12) in 16 bits; of two chunks 385 to 597, which costs rows past 8192 columns
// three quarters of the rate: 2048 x 16384 297 us in bf16 (1.4 TB/s), 493 in fp32. Several rows a block
// spill none.
#include "../../include/dmuon_amd.h"
#include "dmuon_amd_internal.h"
#include "mfma_tile.h"
#include "residual_norm.h"

// a * b + c in one instruction: the backward pass has some twenty operations a value, which would
// otherwise cost as much as its memory traffic
#pragma clang fp contract(fast)

namespace dmuon {
namespace {

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

// 8 values as they lie in memory
template <int T>
struct Raw {
  u32x4_t v[T == DT_F32 ? 2 : 1];
};
// 8 values from element `at` on, or, of a row of less, n of them and zeros. (`whole` is the same for
// all threads: a vector load beside a per-element one in another lane would have to be waited for
// before the other may write its registers.) ONCE: past the caches
template <int T, bool ONCE = false>
__device__ __forceinline__ Raw<T> load_raw(const void* p, long long at, bool whole, int n) {
  Raw<T> r;
  if constexpr (T == DT_F32) {
    const float* q = static_cast<const float*>(p) + at;
    if (whole) {
      r.v[0] = ONCE ? __builtin_nontemporal_load((const v32_t*)q) : *(const v32_t*)q;
      r.v[1] = ONCE ? __builtin_nontemporal_load((const v32_t*)(q + 4)) : *(const v32_t*)(q + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i / 4][i % 4] = i < n ? __float_as_uint(q[i]) : 0u;
    }
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + at;
    if (whole) {
      r.v[0] = ONCE ? __builtin_nontemporal_load((const v16_t*)q) : *(const v16_t*)q;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        r.v[0][i] = (2 * i < n ? q[2 * i] : 0u) | ((2 * i + 1 < n ? q[2 * i + 1] : 0u) << 16);
    }
  }
  return r;
}
template <int T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float* v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (T == DT_F32) v[i] = __uint_as_float(r.v[i / 4][i % 4]);
    else v[i] = half_to_f((i & 1) ? r.v[0][i / 2] >> 16 : r.v[0][i / 2] & 0xffff, T);
  }
}

// A thread's chunk of 8 columns of a row. The last chunk of a row that is no multiple of 8 begins
// earlier, over columns of the one before, and threads past the row's end repeat it: every thread
// loads a whole vector. The first `lo` columns are not the thread's: they count as zeros and are not
// stored. Rows of less than 8: n columns, none past the first thread.
struct Cols {
  int at, lo, dim;
  __device__ __forceinline__ void init(int c, int dim_) {
    dim = dim_;
    at = dim >= 8 ? min(c, dim - 8) : c;
    lo = c - at;
  }
  __device__ __forceinline__ bool whole() const { return dim >= 8; }
  __device__ __forceinline__ int n() const { return whole() ? 8 : max(dim - at, 0); }
};
template <int T, bool ONCE = false>
__device__ __forceinline__ Raw<T> load_raw(const void* p, long long row, const Cols& c) {
  return load_raw<T, ONCE>(p, row + c.at, c.whole(), c.n());
}
__device__ __forceinline__ void load8(const void* p, int t, long long row, const Cols& c, float* v) {
  if (t == DT_F32) unpack<DT_F32>(load_raw<DT_F32>(p, row, c), v);
  else if (t == DT_F16) unpack<DT_F16>(load_raw<DT_F16>(p, row, c), v);
  else unpack<DT_BF16>(load_raw<DT_BF16>(p, row, c), v);
}
template <int T>
__device__ __forceinline__ void unpack(const Raw<T>& r, const Cols& c, float* v) {
  unpack<T>(r, v);
  if (c.lo > 0)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < c.lo ? 0.f : v[i];
}
__device__ __forceinline__ void store8(void* p, int t, long long row, const Cols& c, const float* v) {
  const long long at = row + c.at;
  const int n = c.n();
  const bool all = c.lo == 0 && c.whole();
  if (t == DT_F32) {
    float* q = static_cast<float*>(p) + at;
    if (all) {
      u32x4_t a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[i + 4]);
      __builtin_nontemporal_store(a, (v32_t*)q);
      __builtin_nontemporal_store(b, (v32_t*)(q + 4));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= c.lo && i < n) q[i] = v[i];
    }
  } else {
    uint16_t* q = static_cast<uint16_t*>(p) + at;
    if (all) {
      u32x4_t a;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        a[i] = t == DT_F16 ? pack2_elt<ELT_F16>(v[2 * i], v[2 * i + 1])
                           : pack2_elt<ELT_BF16>(v[2 * i], v[2 * i + 1]);
      __builtin_nontemporal_store(a, (v16_t*)q);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= c.lo && i < n) q[i] = (uint16_t)f_to_half(v[i], t);
    }
  }
}

// Sums of `C` values over the threads of a row (blockDim.x of them: a power of two, or whole waves):
// shuffles in a wave, then one LDS exchange where the row has several waves. The caller passes another
// area than in its call before, so that no area is written while it may still be read. The barrier
// leaves loads in flight.
template <int C>
__device__ __forceinline__ void row_sums(float* v, float (*lds)[16][C], int ty) {
  const int lanes = blockDim.x < 64 ? blockDim.x : 64;
  for (int o = 1; o < lanes; o <<= 1)
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] += __shfl_xor(v[c], o);
  const int waves = blockDim.x >> 6;
  if (waves <= 1) return;
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int c = 0; c < C; ++c) lds[ty][w][c] = v[c];
  __builtin_amdgcn_s_waitcnt(0xC07F);     // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] = lds[ty][0][c];
  for (int k = 1; k < waves; ++k)
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] += lds[ty][k][c];
}

// c = gate w_post of this thread's columns for gate row `group`
template <int NV>
__device__ __forceinline__ void load_factors(const ResidualNorm& a, long long group, const Cols* col,
                                             float (*c)[8]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[v][i] = g[i] = 1.f;
    if (a.w_post) load8(a.w_post, a.post_dtype, 0, col[v], c[v]);
    if (a.gate) load8(a.gate, a.gate_dtype, group * a.dim, col[v], g);
#pragma unroll
    for (int i = 0; i < 8; ++i) c[v][i] *= g[i];
  }
}

// NV chunks of 8 columns a thread. MANY: several rows side by side in 256 threads; otherwise the row is
// the same for the block and its addresses stay scalar.
template <int T, int NV, bool MANY>
__global__ __launch_bounds__(MANY ? 256 : 1024) void residual_norm_kernel(ResidualNorm a) {
  __shared__ float lds[4][4][16][1];
  const int ty = MANY ? threadIdx.y : 0, rows_at_once = MANY ? blockDim.y : 1;
  const float inv = 1.f / (float)a.dim;
  const long long first = (long long)blockIdx.x * a.rows_per_block;
  const long long end = first + a.rows_per_block < a.rows ? first + a.rows_per_block : a.rows;
  Cols col[NV];
  float pre[NV][8], c[NV][8];
  Raw<T> xr[NV], yr[NV];
  auto fetch = [&](long long row) {
    if (row >= end) row = end - 1;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      xr[v] = load_raw<T>(a.x, row * a.ld_x, col[v]);
      if (a.y) yr[v] = load_raw<T>(a.y, row * a.ld_y, col[v]);
    }
  };
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    col[v].init((v * blockDim.x + threadIdx.x) * 8, a.dim);
  }
  fetch(first + ty);
#pragma unroll
  for (int v = 0; v < NV; ++v) load8(a.w_pre, a.pre_dtype, 0, col[v], pre[v]);
  int flip = 0;
  long long group = -1;
  for (long long base = first; base < end; base += rows_at_once) {
    // threads past the last row repeat it: the barriers need every wave
    const long long row = base + ty < end ? base + ty : end - 1;
    float x[NV][8], y[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      unpack<T>(xr[v], col[v], x[v]);
      if (a.y) unpack<T>(yr[v], col[v], y[v]);
    }
    fetch(row + rows_at_once);
    const long long g = a.gate ? row / a.rows_per_group : 0;
    if (g != group) {
      group = g;
      load_factors<NV>(a, g, col, c);
    }
    float r = 1.f;
    if (a.w_post) {
      float sq[1] = {0.f};
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) sq[0] += y[v][i] * y[v][i];
      row_sums<1>(sq, lds[flip], ty);
      r = 1.f / sqrtf(sq[0] * inv + a.eps);
    }
    float sq[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[v][i] *= a.scale;
        if (a.y) x[v][i] += c[v][i] * (y[v][i] * r);
        sq[0] += x[v][i] * x[v][i];
      }
    row_sums<1>(sq, lds[2 + flip], ty);
    flip ^= 1;
    const float s = 1.f / sqrtf(sq[0] * inv + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const long long at = row * a.dim;
      if (a.x_new) store8(a.x_new, T, at, col[v], x[v]);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[v][i] = x[v][i] * s * pre[v][i];
      store8(a.h, T, at, col[v], x[v]);
    }
    if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(r, s);
  }
}

// The gradients of gate and w_post come from one sum a column and gate group, t = sum d yhat:
// d_gate = w_post t, d_post = sum over the groups of gate t. GROUPS: a block has several gate groups.
template <int T, int NV, bool MANY, bool GROUPS>
__global__ __launch_bounds__(MANY ? 256 : 1024) void residual_norm_grad_kernel(ResidualNorm a) {
  __shared__ float lds[2][4][16][3];
  __shared__ float acc[MANY ? 256 * 8 : 1];
  const int ty = MANY ? threadIdx.y : 0, rows_at_once = MANY ? blockDim.y : 1;
  const float inv = 1.f / (float)a.dim;
  // rows of this block: a part of one gate group, or several whole groups (then not MANY)
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
  Cols col[NV];
  float pre[NV][8], c[NV][8], d_pre[NV][8], d_post[NV][8], t[NV][8];
  Raw<T> xr[NV], yr[NV], er[NV], gr[NV];
  float2 rs;
  auto fetch = [&](long long row) {
    if (row >= end) row = end - 1;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      xr[v] = load_raw<T, true>(a.x, row * a.ld_x, col[v]);
      if (a.y) yr[v] = load_raw<T, true>(a.y, row * a.ld_y, col[v]);
      if (a.dx_new) er[v] = load_raw<T, true>(a.dx_new, row * a.ld_dx_new, col[v]);
      if (a.dh) gr[v] = load_raw<T, true>(a.dh, row * a.ld_dh, col[v]);
    }
    rs = a.stats[row];
  };
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    col[v].init((v * blockDim.x + threadIdx.x) * 8, a.dim);
#pragma unroll
    for (int i = 0; i < 8; ++i) d_pre[v][i] = d_post[v][i] = t[v][i] = 0.f;
  }
  fetch(first + ty);
#pragma unroll
  for (int v = 0; v < NV; ++v) load8(a.w_pre, a.pre_dtype, 0, col[v], pre[v]);
  // a gate group's end in this block: its shares of the gradients, into `out` row `at`
  auto flush = [&](long long group, void* out, int dtype, long long at) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 1.f;
      if (a.gate) load8(a.gate, a.gate_dtype, group * a.dim, col[v], w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        d_post[v][i] += w[i] * t[v][i];
        w[i] = 1.f;
      }
      if (out) {
        if (a.w_post) load8(a.w_post, a.post_dtype, 0, col[v], w);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] *= t[v][i];
        store8(out, dtype, at * a.dim, col[v], w);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) t[v][i] = 0.f;
    }
  };
  int flip = 0;
  long long group = -1;
  for (long long base = first; base < end; base += rows_at_once) {
    // threads past the last row repeat it without a share of the sums
    const bool live = base + ty < end;
    const long long row = live ? base + ty : end - 1;
    const long long q = a.gate ? row / a.rows_per_group : 0;
    if (q != group) {
      if (GROUPS && group >= 0) flush(group, a.d_gate, a.gate_dtype, group);
      group = q;
      load_factors<NV>(a, q, col, c);
    }
    float x[NV][8], y[NV][8], e[NV][8], g[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      unpack<T>(xr[v], col[v], x[v]);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[v][i] = e[v][i] = g[v][i] = 0.f;
      if (a.y) unpack<T>(yr[v], col[v], y[v]);
      if (a.dx_new) unpack<T>(er[v], col[v], e[v]);
      if (a.dh) unpack<T>(gr[v], col[v], g[v]);
    }
    const float r = rs.x, s = rs.y;
    fetch(row + rows_at_once);
    float sums[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[v][i] *= r;                                   // yhat
        const float cy = c[v][i] * y[v][i];
        x[v][i] = a.scale * x[v][i];
        if (a.y) x[v][i] += cy;
        x[v][i] *= s;                                   // xhat
        if (live) d_pre[v][i] += g[v][i] * x[v][i];
        g[v][i] *= pre[v][i];
        e[v][i] += s * g[v][i];
        sums[0] += g[v][i] * x[v][i];
        sums[1] += cy * e[v][i];
        sums[2] += cy * x[v][i];
      }
    row_sums<3>(sums, lds[flip], ty);
    flip ^= 1;
    const float ka = s * sums[0] * inv;
    const float kb = a.w_post ? (sums[1] - ka * sums[2]) * inv : 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const long long at = row * a.dim;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = e[v][i] - ka * x[v][i];
        if (live) t[v][i] += d * y[v][i];
        x[v][i] = a.scale * d;
        y[v][i] = r * (c[v][i] * d - y[v][i] * kb);
      }
      if (a.dx) store8(a.dx, T, at, col[v], x[v]);
      if (a.dy) store8(a.dy, T, at, col[v], y[v]);
    }
  }
  // rows side by side join through LDS in their order, into row 0's threads
  auto gather = [&](float (&d)[NV][8]) {
    if constexpr (MANY) {
      float* mine = acc + (ty * blockDim.x + threadIdx.x) * 8;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[i] = d[0][i];
      __syncthreads();
      if (ty == 0)
        for (int k = 1; k < rows_at_once; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) d[0][i] += mine[k * blockDim.x * 8 + i];
    }
  };
  gather(t);
  gather(d_pre);
  if (ty) return;
  if (a.parts > 1) flush(group, a.d_gate ? a.gate_part : nullptr, DT_F32, blockIdx.x);
  else flush(group, a.d_gate, a.gate_dtype, group);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const long long at = (long long)blockIdx.x * a.dim;
    if (a.d_pre) store8(a.pre_part, DT_F32, at, col[v], d_pre[v]);
    if (a.d_post) store8(a.post_part, DT_F32, at, col[v], d_post[v]);
  }
}

// Column sums of partial rows, 32 columns by 32 strands a block: blockIdx.y 0 and 1 are the two
// weights' rows, the rest the gate groups' (`parts` rows each). The rows are still in the caches: 8 us at 16384 x 4096.
__global__ __launch_bounds__(1024) void sum_partials_kernel(ResidualNorm a) {
  __shared__ float lds[32][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int job = blockIdx.y;
  const float* part = job == 0 ? a.pre_part : job == 1 ? a.post_part : a.gate_part;
  void* out = job == 0 ? a.d_pre : job == 1 ? a.d_post : a.d_gate;
  const int dtype = job == 0 ? a.pre_dtype : job == 1 ? a.post_dtype : a.gate_dtype;
  if (!out) return;
  const long long n = job < 2 ? a.blocks : a.parts, g = job < 2 ? 0 : job - 2;
  float s = 0.f;
  if (c < a.dim) {
#pragma unroll 4
    for (long long k = strand; k < n; k += 32) s += part[(g * n + k) * a.dim + c];
  }
  lds[strand][lane] = s;
  __syncthreads();
  // a wave sums two columns: strands pairwise, always in the same order
  const int cc = threadIdx.x >> 5;
  s = lds[lane][cc];
  for (int o = 16; o; o >>= 1) s += __shfl_xor(s, o);
  const int oc = blockIdx.x * 32 + cc;
  if (lane || oc >= a.dim) return;
  if (dtype == DT_F32) static_cast<float*>(out)[g * a.dim + oc] = s;
  else static_cast<uint16_t*>(out)[g * a.dim + oc] = (uint16_t)f_to_half(s, dtype);
}

// Threads of a row (a power of two up to 128, then whole waves up to 1024) and chunks of 8 columns a
// thread: two for rows longer than `one`.
bool row_shape(int dim, int one, int* threads, int* nv) {
  const int chunks = (dim + 7) / 8;
  if (chunks > 2048) return false;
  *nv = dim > one ? 2 : 1;
  *threads = 8;
  while (*threads * *nv < chunks && *threads < 128) *threads *= 2;
  if (*threads * *nv < chunks) *threads = ((chunks + *nv - 1) / *nv + 63) / 64 * 64;
  return true;
}

constexpr long long kCus = 256;
// Forward, two chunks a thread measured 98 against 106 us (16384 x 4096) and 105 against 129 (8192 x
// 8192); the backward pass has no registers for them in less than 1024 threads.
constexpr int kOneForward = 2048, kOneBackward = 8192;

}  // namespace

void residual_norm_split(ResidualNorm* a) {
  int threads = 64, nv = 1;
  row_shape(a->dim, kOneBackward, &threads, &nv);
  const long long groups = a->gate ? a->rows / a->rows_per_group : 1;
  if (!a->gate) a->rows_per_group = a->rows > 0 ? a->rows : 1;
  const long long per = a->rows_per_group;
  // as many blocks as their registers let run at once: 16 waves a CU, or three blocks of 256 threads
  // (four took 196 us where three take 176: 65536 x 1024)
  auto want = [&](int lanes) { return lanes > 1 ? kCus * 3 : kCus * (1024 / threads); };
  a->lanes = threads < 256 ? 256 / threads : 1;
  if (a->rows <= 0) {
    a->parts = 0;                         // the gate's gradient is a sum of none
    a->blocks = 0;
    a->rows_per_block = 1;
  } else if (groups > want(a->lanes) / 2 && groups > 1) {
    // whole groups: one row at a time, since a block's rows may lie in several of them
    a->lanes = 1;
    const long long each = (groups + want(1) - 1) / want(1);
    a->parts = 1;
    a->rows_per_block = each * per;
    a->blocks = (groups + each - 1) / each;
  } else {
    long long parts = want(a->lanes) / groups, most = (per + a->lanes - 1) / a->lanes;
    if (parts > most) parts = most;
    a->rows_per_block = (per + parts - 1) / parts;
    a->rows_per_block = (a->rows_per_block + a->lanes - 1) / a->lanes * a->lanes;
    a->parts = (int)((per + a->rows_per_block - 1) / a->rows_per_block);
    a->blocks = groups * a->parts;
    if (a->parts == 1) a->rows_per_block = per;
  }
}

hipError_t launch_residual_norm(ResidualNorm a, hipStream_t stream) {
  int threads, nv;
  if (!row_shape(a.dim, kOneForward, &threads, &nv)) return hipErrorInvalidValue;
  if (a.rows <= 0) return hipSuccess;
  const int lanes = threads < 256 ? 256 / threads : 1;
  // rows of two chunks a thread have 192 threads or more
  if (nv == 2 && lanes > 1) return hipErrorInvalidValue;
  const long long want = kCus * 4096 / (threads * lanes);
  a.rows_per_block = (a.rows + want - 1) / want;
  a.rows_per_block = (a.rows_per_block + lanes - 1) / lanes * lanes;
  const dim3 grid((unsigned)((a.rows + a.rows_per_block - 1) / a.rows_per_block));
  const dim3 block(threads, lanes);
#define DMUON_RN(T, NV, MANY) \
  hipLaunchKernelGGL((residual_norm_kernel<T, NV, MANY>), grid, block, 0, stream, a)
#define DMUON_RN_T(T)                                  \
  do {                                                 \
    if (lanes > 1) DMUON_RN(T, 1, true);               \
    else if (nv == 1) DMUON_RN(T, 1, false);           \
    else DMUON_RN(T, 2, false);                        \
  } while (0)
  if (a.dtype == DT_F32) DMUON_RN_T(DT_F32);
  else if (a.dtype == DT_F16) DMUON_RN_T(DT_F16);
  else DMUON_RN_T(DT_BF16);
#undef DMUON_RN_T
#undef DMUON_RN
  return hipGetLastError();
}

hipError_t launch_residual_norm_grad(const ResidualNorm& a, hipStream_t stream) {
  int threads, nv;
  if (!row_shape(a.dim, kOneBackward, &threads, &nv) || a.blocks > 0x7fffffffLL) return hipErrorInvalidValue;
  if (a.blocks > 0) {
    const dim3 grid((unsigned)a.blocks), block(threads, a.lanes);
#define DMUON_RN(T, NV, MANY, GROUPS) \
  hipLaunchKernelGGL((residual_norm_grad_kernel<T, NV, MANY, GROUPS>), grid, block, 0, stream, a)
#define DMUON_RN_T(T)                                  \
  do {                                                 \
    if (nv == 2) DMUON_RN(T, 2, false, true);          \
    else if (a.lanes > 1) DMUON_RN(T, 1, true, false); \
    else if (several) DMUON_RN(T, 1, false, true);     \
    else DMUON_RN(T, 1, false, false);                 \
  } while (0)
    const bool several = a.rows_per_block > a.rows_per_group;
    if (a.dtype == DT_F32) DMUON_RN_T(DT_F32);
    else if (a.dtype == DT_F16) DMUON_RN_T(DT_F16);
    else DMUON_RN_T(DT_BF16);
#undef DMUON_RN_T
#undef DMUON_RN
  }
  const bool gates = a.d_gate && a.parts != 1;
  if (a.d_pre || a.d_post || gates) {
    const dim3 grid((unsigned)((a.dim + 31) / 32),
                    (unsigned)(gates ? 2 + a.gates : a.d_post ? 2 : 1));
    hipLaunchKernelGGL(sum_partials_kernel, grid, dim3(1024), 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace dmuon

using namespace dmuon;

namespace {

constexpr int64_t kMaxDim = 16384;

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
  r.gates = a.gate ? a.gates : 0;
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
