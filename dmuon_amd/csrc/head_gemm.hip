// Products of the vocabulary losses on gfx950:
//   logits          Z  = H W^T      (tokens x vocabulary; both operands row by row)
//   hidden gradient dH = G W        (W k-major)
//   weight gradient dW = G^T H      (both operands k-major)
// with the softmax statistics of the logits' columns taken in the first one's epilogue.
#include "dmuon_amd_internal.h"
#include "head_loss.h"

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

namespace dmuon {
namespace {

template <int E>
__device__ __forceinline__ uint16_t to_elt(float f) {
  if constexpr (E == ELT_F16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  else return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}
template <int E>
__device__ __forceinline__ f32x4_t mfma_16x16x32(bf16x8_t b, bf16x8_t a, f32x4_t c) {
  if constexpr (E == ELT_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, b),
                                                  __builtin_bit_cast(f16x8_t, a), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0);
}

// 64 x 64 tile, four waves of 16 rows; operands pass through registers one value at a time, so
// any stride, alignment and size is right.
template <int E, int MODE>
__global__ __launch_bounds__(256) void head_gemm_kernel(HeadGemm a) {
  constexpr int T = 64, BK = 32, PITCH = BK + 8;
  __shared__ __attribute__((aligned(16))) uint16_t sa[T * PITCH], sb[T * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int j0 = blockIdx.x * T, i0 = blockIdx.y * T;
  f32x4_t acc[4] = {};
  auto fill = [&](uint16_t* s, const uint16_t* X, long long ld, int kmajor, int r0, int rows,
                  int k0) {
    for (int e = tid; e < T * BK; e += 256) {
      const int r = kmajor ? e % T : e / BK, k = kmajor ? e / T : e % BK;
      uint16_t v = 0;
      if (r0 + r < rows && k0 + k < a.K)
        v = kmajor ? X[(long long)(k0 + k) * ld + r0 + r] : X[(long long)(r0 + r) * ld + k0 + k];
      s[r * PITCH + k] = v;
    }
  };
  for (int k0 = 0; k0 < a.K; k0 += BK) {
    fill(sa, a.A, a.lda, a.a_kmajor, i0, a.M, k0);
    fill(sb, a.B, a.ldb, a.b_kmajor, j0, a.N, k0);
    __syncthreads();
    const int at = (lane & 15) * PITCH + 8 * (lane >> 4);
    const bf16x8_t af = *reinterpret_cast<const bf16x8_t*>(sa + wave * 16 * PITCH + at);
#pragma unroll
    for (int y = 0; y < 4; ++y)
      acc[y] = mfma_16x16x32<E>(*reinterpret_cast<const bf16x8_t*>(sb + y * 16 * PITCH + at), af,
                                acc[y]);
    __syncthreads();
  }
  // a lane holds row lane % 16, columns 16 y + 4 (lane / 16) .. + 3
  const int i = i0 + wave * 16 + (lane & 15), jl = j0 + 4 * (lane >> 4);
  if constexpr (MODE == HG_LOGITS) {
    float m = -__builtin_inff();
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = jl + 16 * y + e;
        const float z = acc[y][e] * a.scale;
        if (j < a.N) m = fmaxf(m, z);
        if (a.Z && i < a.M && j < a.N) a.Z[(long long)i * a.ldz + j] = z;
      }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    float s = 0.f;
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (jl + 16 * y + e < a.N) {
          const float z = acc[y][e] * a.scale;
          s += z == -__builtin_inff() ? 0.f : __expf(z - m);
        }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane < 16 && i < a.M) a.stats[(long long)blockIdx.x * a.M + i] = make_float2(m, s);
  } else {
    if (i >= a.M) return;
    const float alpha = a.out ? a.alpha[0] : 1.f;
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = jl + 16 * y + e;
        if (j >= a.N) continue;
        float v = acc[y][e];
        if (a.add_part) v += a.part[(long long)i * a.ldp + j];
        const long long o = (long long)i * a.ldo + j;
        if (!a.out) a.part[(long long)i * a.ldp + j] = v;
        else if (a.out_dtype == DT_F32) static_cast<float*>(a.out)[o] = alpha * v;
        else static_cast<uint16_t*>(a.out)[o] = to_elt<E>(alpha * v);
      }
  }
}

}  // namespace

hipError_t launch_head_gemm(const HeadGemm& a, hipStream_t stream) {
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  const long long nb = (a.N + 63) / 64, mb = (a.M + 63) / 64;
  if (mb > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)nb, (unsigned)mb);
#define DMUON_HG(E, MODE) hipLaunchKernelGGL((head_gemm_kernel<E, MODE>), grid, dim3(256), 0, stream, a)
  if (a.elt == ELT_F16) {
    if (a.mode == HG_LOGITS) DMUON_HG(ELT_F16, HG_LOGITS); else DMUON_HG(ELT_F16, HG_GRAD);
  } else {
    if (a.mode == HG_LOGITS) DMUON_HG(ELT_BF16, HG_LOGITS); else DMUON_HG(ELT_BF16, HG_GRAD);
  }
#undef DMUON_HG
  return hipGetLastError();
}

}  // namespace dmuon
