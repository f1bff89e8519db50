// Internal declarations of the vocabulary losses: the products of hidden states with a head's
// weight and the row kernels between them. Not part of the public C ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dmuon {

// Columns of one softmax statistic: every row keeps a (maximum, sum of exponentials) pair per
// kStatCols columns of the logits.
constexpr int kStatCols = 64;
// The logit gradient is stored as 2^kGradShift times its row's value over the largest row weight:
// fp16 then holds probabilities down to 2^-24 with all their bits and 2^-34 with some. A row's
// largest value is its factor mass + 2 z_loss lse and its mass at most. Where they reach 2^kPeakBits
// (an unusual z_loss or teacher), fp16 gradients shrink by the power of two that keeps them under it,
// and the products' sums grow by it again: peak_shift of the largest so far.
constexpr int kGradShift = 10, kPeakBits = 15;
__host__ __device__ __forceinline__ int peak_shift(unsigned peak) {
  const int shift = (int)(peak >> 23) - (127 + kPeakBits - 1);
  return shift > 0 ? shift : 0;
}

// What a product writes. Logits z = scale * acc and their statistics are in units of log 2.
//   HG_STATS   the softmax statistics of z
//   HG_EXP     those and Z = fp16(2^kExpShift 2^(z - m)), m the row's maximum in its statistic's
//              columns; 0 in the columns past N
//   HG_LOGITS  those and Z = z in fp32
//   HG_GRAD    out = alpha[0] * (acc + part) rounded to out_dtype, or part (+)= acc in fp32
enum HeadGemmMode : int { HG_STATS = 0, HG_EXP = 1, HG_LOGITS = 2, HG_GRAD = 3 };
// fp16 holds exponentials down to 2^-29 of their maximum with all its bits
constexpr int kExpShift = 15;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// Rows up to which the logits have one row of tiles, bound by reading the weight.
constexpr int kFewRows = 256;

// The logits and their gradient lie in blocks of kStatCols classes, [ceil(vocab / 64)][rows][64]: a
// tile of any of the three products reads and writes them in runs of 8 to 32 KiB, where rows of the
// whole vocabulary would be 128 bytes at a time (hidden gradient of 8192 x 128256 x 4096: 6.08 ms
// that way, 5.73 in blocks).
//
// acc[i][j] = sum_k A(i, k) * B(j, k). HG_GRAD: A is the logit gradient in its blocks, lda its rows
// (a_kmajor: i is the class, k the token). Otherwise A's element (i, k) is A[i * lda + k]. B's is
// B[j * ldb + k], or B[k * ldb + j] with b_kmajor.
struct HeadGemm {
  const uint16_t* A; long long lda; int a_kmajor;
  const uint16_t* B; long long ldb; int b_kmajor;
  int M, N, K;
  int mode, elt;
  float scale;
  void* Z;                                // HG_EXP, HG_LOGITS: [ceil(N / 64)][M][64]
  float2* stats;                          // [ceil(N / 64)][M]
  const float* alpha;
  const unsigned* peak;                   // HG_GRAD in fp16: see HeadRows; NULL: no shift
  void* out; long long ldo; int out_dtype;   // HG_GRAD: result (DT_F32 or the operands'), or NULL
  float* part; long long ldp;             // HG_GRAD: fp32 sums [M][ldp], or NULL
  int add_part;                           // part holds earlier sums to add to
  int few, small;                         // logits: of a call of at most kFewRows rows; its
                                          // head_logits_small
  int splits;                             // HG_GRAD: K in so many parts, part [splits][M][ldp]
  int join_later;                         // a hidden gradient whose parts a weight gradient's launch,
  const HeadGemm* join;                   // with it in `join`, makes the result (see head_joins_later)
};
// Whether the parts of hidden gradient h (its sizes and splits) join in the launch of the weight
// gradient of `vocab` classes: one of few tokens, whose kernel takes them beside its tiles. A launch of
// their own costs a small call's step 4 us more.
bool head_joins_later(const HeadGemm& h, int vocab);
// Whether a call's logits take the kernel for small ones (1: of at most 16 rows, 2: of more). By the
// call's sizes, not a chunk's: chunks do not change its bits.
int head_logits_small(int tokens, int vocab);
// K splits that fill the chip where a gradient has few tiles (1: none); weight: of the weight.
int head_gemm_splits(int M, int N, int K, bool weight);
// Operands at 16-byte alignment with pitches of whole 16-byte chunks. Rows that end inside a chunk
// are readable to its end, and hold zeros there in row form (past K).
hipError_t launch_head_gemm(const HeadGemm& a, hipStream_t stream);

// One call's rows as the kernels see them. Entry k of row n is the class ids[n * k_list + k] with
// the target probability probs[..] (0 for padding, whose id is -1).
struct HeadRows {
  int n;                                  // tokens of the call
  int vocab, k_list;
  const int64_t* targets;                 // hard targets [n] (k_list 1), or
  const int64_t* teacher_ids;             // [n][k_list]
  const float* teacher_logits;            // [n][k_list]
  const float* teacher_lse;               // [n] or NULL
  long long ignore_index;
  float z_loss, temperature;
  int reduction;                          // DMUON_LOSS_*
  const float* row_grad;                  // DMUON_LOSS_ROWS: dL / d loss[n], or NULL
  int* ids; float* probs;                 // [n][k_list]
  float* logits;                          // [n][k_list]: the entries' logits (over temperature)
  float* mass;                            // [n]: sum of the row's probs, < 0: not counted
  float* top;                             // [n]: the largest logit, in units of log 2
  float* loss;                            // [n]
  float* row_weight;                      // [n]: 2^kGradShift * row gradient / largest, 0: not counted
  float* factor;                          // [n]: of 2^(z - top) in the logit gradient
  float* alpha;                           // [1]: what turns a stored gradient into the real one
  unsigned* peak;                         // [1], fp16 gradients: bits of the largest row value so far
                                          // of 2^kPeakBits and more, or 0
  float* mean;                            // [1] or NULL: the reduced loss
};
// ids, probs, mass and logits of every row (H, W: the products' operands, any alignment); with
// `grads` of unreduced losses the row weights and alpha.
hipError_t launch_head_targets(const HeadRows& r, const uint16_t* H, long long ldh,
                               const uint16_t* W, long long ldw, int dim, int elt, bool grads,
                               hipStream_t stream);
// Top, loss, row weight and factor of rows first .. first + rows - 1 from their statistics, and with G
// their logit gradients row_weight (mass softmax - target probability), 0 past the vocabulary's end:
// in place of the exponentials (Z == G), or from the fp32 logits Z. Unless reduction is
// DMUON_LOSS_ROWS, mean[0] = sum of the losses, divided by the number of counted rows for
// DMUON_LOSS_MEAN, and alpha: with the last rows, with G after every chunk (mean is right after the
// last; alpha, which the gradient's products take, after each).
hipError_t launch_head_rows(const HeadRows& r, int first, int rows, const float2* stats,
                            const void* Z, uint16_t* G, int elt, hipStream_t stream);

// Copies of up to two operands with rows of `pad` values (a multiple of 8) at 16-byte alignment, zeros
// past `dim`: what the products read where an operand's own rows do not fit their loads.
struct HeadPad {
  const uint16_t* src[2]; long long ld[2];
  uint16_t* dst[2];
  int rows[2];
  int n, dim, pad;
  void add(const uint16_t* s, long long lds, int count, void* d) {
    src[n] = s;
    ld[n] = lds;
    rows[n] = count;
    dst[n++] = static_cast<uint16_t*>(d);
  }
};
hipError_t launch_head_pad(const HeadPad& a, hipStream_t stream);

// dst[k] = factor[0] * src[k] for n[k] values, k = 0 and 1; in_place: every dst is its src, and
// nothing moves where the factor is 1.
struct ScaleBy {
  const void* src[2]; void* dst[2];
  long long n[2];
  const float* factor;
  int in_place;
};
hipError_t launch_scale_by(const ScaleBy& a, int src_dtype, int dst_dtype, hipStream_t stream);

}  // namespace dmuon
