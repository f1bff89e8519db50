// dmuon_head_loss: argument checks, workspace layout and launch sequence of the vocabulary losses.
//
// The rows go through in chunks of tokens. Per chunk: the logits' product with the softmax statistics
// of every 64 columns, each row's log-sum-exp and loss, the logit gradient, and its two products
// with the weight and the hidden states. The weight's gradient sums over the chunks in fp32.
//
// Between the first product and the others a logit takes two bytes where the operands are bf16:
// exp(z - m) in fp16, m the maximum of the row's 64 columns, which the row kernel turns into the
// bf16 gradient in place. Its 2^-11 is small against the 2^-8 of the gradient's own rounding down to
// probabilities of 2^-29 of their block's largest; under that fp16 has fewer bits, and under 2^-40
// none: such a class's share of the gradient, less than 1e-12 of its neighbour's, is left out. For
// fp16 operands it is not: there the product writes fp32 logits and the gradient has its own place,
// six bytes a logit.
#include "../../include/dmuon_amd.h"
#include "dmuon_amd_internal.h"
#include "head_loss.h"

#include <cmath>

using namespace dmuon;

namespace {

int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Workspace of a chunk's logits, logit gradient and statistics; a call of more tokens takes several
// chunks. (In bf16 the weight gradient's fp32 sums over them then take the place of the hidden
// gradient's parts, whose K is not split: 8192 x 128256 x 4096 in one chunk 19.3 ms, in chunks of 4096
// 20.2, 2048 24.8, 1024 37.9, 256 118; fp16, whose sums are the result, 22.7, -, 24.6, 28.6, 57.)
constexpr int64_t kChunkBytes = int64_t(4) << 30;

// Blocks of 64 classes are a grid's second dimension.
constexpr int64_t kMaxVocab = int64_t(65535) * 64;

struct Layout {
  int64_t chunk, ld;                      // tokens of a chunk, classes in whole blocks
  int64_t ids, probs, logits, mass, top, loss, row_weight, factor, alpha, peak, Z, stats, G, part, H, W, bytes;
  int64_t pad;                            // pitch of the copies of hidden and weight
  bool copy_h, copy_w;
  bool gathers, split_h;                  // the weight gradient sums over chunks; the hidden one's K is
                                          // split: not where those sums have the parts' place
};

// The products read whole 16-byte chunks of aligned rows; anything else runs on zero-padded copies.
bool in_place(const void* p, int64_t ld, int64_t dim) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && dim % 8 == 0 && ld < (1 << 22);
}

int elt_of(int dtype, int* elt) {
  if (dtype == DMUON_DTYPE_BF16) *elt = ELT_BF16;
  else if (dtype == DMUON_DTYPE_F16) *elt = ELT_F16;
  else return 1;
  return 0;
}

int check(const char* who, const dmuon_head_loss_args* a) {
  int elt;
  if (!a) return fail("%s: NULL arguments", who);
  if (elt_of(a->dtype, &elt))
    return fail("%s: dtype code %d is not a 16-bit type (bf16 %d, fp16 %d)", who, a->dtype,
                DMUON_DTYPE_BF16, DMUON_DTYPE_F16);
  if (a->grad_dtype != a->dtype && a->grad_dtype != DMUON_DTYPE_F32)
    return fail("%s: gradients are fp32 or of the operands' dtype, got code %d", who,
                a->grad_dtype);
  if (a->tokens < 0 || a->tokens > (1 << 24))
    return fail("%s: tokens must be 0 .. 2^24, got %lld", who, (long long)a->tokens);
  if (a->vocab < 1 || a->vocab > kMaxVocab || a->dim < 1 || a->dim > (1 << 20))
    return fail("%s: vocab must be 1 .. %lld and dim 1 .. 2^20, got %lld and %lld", who,
                (long long)kMaxVocab, (long long)a->vocab, (long long)a->dim);
  if (a->ld_hidden < a->dim || a->ld_weight < a->dim)
    return fail("%s: the pitches of hidden and weight must be at least dim", who);
  if (a->chunk_tokens < 0) return fail("%s: chunk_tokens must not be negative", who);
  if (a->reduction != DMUON_LOSS_ROWS && a->reduction != DMUON_LOSS_MEAN &&
      a->reduction != DMUON_LOSS_SUM)
    return fail("%s: unknown reduction %d", who, a->reduction);
  if ((a->targets != nullptr) == (a->teacher_ids != nullptr) && a->tokens > 0)
    return fail("%s: needs either targets or a teacher's lists", who);
  if (a->teacher_ids) {
    if (a->k_list < 1 || a->k_list > 4096)
      return fail("%s: k_list must be 1 .. 4096, got %lld", who, (long long)a->k_list);
    if (!a->teacher_logits) return fail("%s: teacher_logits is NULL", who);
    if (!(a->temperature > 0.f) || !std::isfinite(a->temperature) || !std::isfinite(1.f / a->temperature))
      return fail("%s: temperature must be positive, and finite like its inverse", who);
    if (a->z_loss != 0.f) return fail("%s: z_loss goes with hard targets", who);
  }
  return 0;
}

Layout lay_out(const dmuon_head_loss_args& a) {
  const bool grads = a.d_hidden || a.d_weight;
  Layout l{};
  const int64_t k = a.teacher_ids ? a.k_list : 1, tiles = round_up(a.vocab, kStatCols) / kStatCols;
  const bool f16 = a.dtype == DMUON_DTYPE_F16;
  l.ld = round_up(a.vocab, 64);
  const int64_t row = (grads ? l.ld * (f16 ? 6 : 2) : 0) + tiles * 8;
  l.chunk = a.chunk_tokens > 0 ? a.chunk_tokens : kChunkBytes / row;
  if (l.chunk > 256) l.chunk = l.chunk / 256 * 256;
  if (l.chunk < 1) l.chunk = 1;
  if (l.chunk < a.tokens && a.chunk_tokens == 0) {
    // chunks of one size, in whole tiles
    const int64_t n = (a.tokens + l.chunk - 1) / l.chunk;
    l.chunk = round_up((a.tokens + n - 1) / n, l.chunk < 256 ? 1 : 256);
  }
  if (l.chunk > a.tokens) l.chunk = a.tokens;
  auto take = [&](int64_t bytes) {
    const int64_t at = l.bytes;
    l.bytes += round_up(bytes, 256);
    return at;
  };
  l.ids = take(a.tokens * k * 4);
  l.probs = take(a.tokens * k * 4);
  l.logits = take(a.tokens * k * 4);
  l.mass = take(a.tokens * 4);
  l.top = take(a.tokens * 4);
  l.loss = take(a.loss ? 0 : a.tokens * 4);
  l.row_weight = take(a.tokens * 4);
  l.factor = take(a.tokens * 4);
  l.alpha = take(4);
  l.peak = take(grads && f16 ? 4 : 0);
  l.stats = take(l.chunk * tiles * 8);
  l.G = take(grads ? l.chunk * l.ld * 2 : 0);
  l.Z = grads && f16 ? take(l.chunk * l.ld * 4) : l.G;
  // fp32 sums: the weight's gradient over several chunks, or of split products
  int64_t part = 0;
  l.gathers = a.d_weight && l.chunk < a.tokens;
  l.split_h = !l.gathers || a.grad_dtype == DMUON_DTYPE_F32;
  if (l.gathers) {
    if (!l.split_h) part = a.vocab * a.dim * 4;
  } else if (a.d_weight) {
    const int s = head_gemm_splits((int)a.vocab, (int)a.dim, (int)a.tokens, true);
    if (s > 1) part = s * a.vocab * a.dim * 4;
  }
  if (a.d_hidden && l.split_h)
    for (int64_t rows : {l.chunk, l.chunk > 0 ? a.tokens % l.chunk : 0}) {
      const int s = head_gemm_splits((int)rows, (int)a.dim, (int)a.vocab, false);
      if (s > 1 && s * rows * a.dim * 4 > part) part = s * rows * a.dim * 4;
    }
  l.part = take(part);
  l.pad = round_up(a.dim, 64);
  l.copy_h = !in_place(a.hidden, a.ld_hidden, a.dim);
  l.copy_w = !in_place(a.weight, a.ld_weight, a.dim);
  l.H = take(l.copy_h ? l.chunk * l.pad * 2 : 0);
  l.W = take(l.copy_w ? a.vocab * l.pad * 2 : 0);
  return l;
}

}  // namespace

extern "C" {

int dmuon_head_loss_workspace_size(const dmuon_head_loss_args* args, int64_t* workspace_bytes) {
  const char* who = "dmuon_head_loss_workspace_size";
  if (!workspace_bytes) return fail("%s: NULL output", who);
  if (check(who, args)) return 1;
  *workspace_bytes = lay_out(*args).bytes;
  return 0;
}

int dmuon_head_loss(const dmuon_head_loss_args* args, void* workspace, int64_t workspace_bytes,
                    void* stream_) {
  const char* who = "dmuon_head_loss";
  if (check(who, args)) return 1;
  const dmuon_head_loss_args& a = *args;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const bool grads = a.d_hidden || a.d_weight;
  if (!a.weight || (a.tokens > 0 && !a.hidden)) return fail("%s: NULL hidden or weight", who);
  if (a.reduction == DMUON_LOSS_ROWS && a.tokens > 0 && !a.loss) return fail("%s: loss is NULL", who);
  if (a.reduction != DMUON_LOSS_ROWS && !a.reduced) return fail("%s: reduced is NULL", who);
  if (a.reduction == DMUON_LOSS_ROWS && grads && a.tokens > 0 && !a.row_grad)
    return fail("%s: the gradients of unreduced losses need row_grad", who);
  const Layout l = lay_out(a);
  if (workspace_bytes < l.bytes || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail("%s: needs a 256-byte aligned workspace of %lld bytes, got %lld", who,
                (long long)l.bytes, (long long)workspace_bytes);
  int elt = 0;
  elt_of(a.dtype, &elt);
  const int64_t grad_size = a.grad_dtype == DMUON_DTYPE_F32 ? 4 : 2;
  char* ws = static_cast<char*>(workspace);
  auto floats = [&](int64_t at) { return reinterpret_cast<float*>(ws + at); };

  HeadRows r{};
  r.n = (int)a.tokens;
  r.vocab = (int)a.vocab;
  r.k_list = a.teacher_ids ? (int)a.k_list : 1;
  r.targets = a.targets;
  r.teacher_ids = a.teacher_ids;
  r.teacher_logits = a.teacher_logits;
  r.teacher_lse = a.teacher_lse;
  r.ignore_index = a.ignore_index;
  r.z_loss = a.teacher_ids ? 0.f : a.z_loss;
  r.temperature = a.teacher_ids ? a.temperature : 1.f;
  r.reduction = a.reduction;
  r.row_grad = a.reduction == DMUON_LOSS_ROWS ? a.row_grad : nullptr;
  r.ids = reinterpret_cast<int*>(ws + l.ids);
  r.probs = floats(l.probs);
  r.logits = floats(l.logits);
  r.mass = floats(l.mass);
  r.top = floats(l.top);
  r.loss = a.loss ? a.loss : floats(l.loss);
  r.row_weight = floats(l.row_weight);
  r.factor = floats(l.factor);
  r.alpha = floats(l.alpha);
  r.peak = grads && elt == ELT_F16 ? reinterpret_cast<unsigned*>(ws + l.peak) : nullptr;
  r.mean = a.reduced;
  void* Z = ws + l.Z;
  float2* stats = reinterpret_cast<float2*>(ws + l.stats);
  uint16_t* G = reinterpret_cast<uint16_t*>(ws + l.G);
  const uint16_t* H = static_cast<const uint16_t*>(a.hidden);
  const uint16_t* W = static_cast<const uint16_t*>(a.weight);

  int64_t ldw = a.ld_weight;
  if (l.copy_w) {
    W = reinterpret_cast<const uint16_t*>(ws + l.W);
    ldw = l.pad;
  }
  if (check_launch(launch_head_targets(r, H, a.ld_hidden, static_cast<const uint16_t*>(a.weight),
                                       a.ld_weight, (int)a.dim, elt, grads, stream), who)) return 1;
  for (int64_t first = 0; first < a.tokens || first == 0; first += l.chunk) {
    const int rows = (int)(a.tokens - first < l.chunk ? a.tokens - first : l.chunk);
    const uint16_t* Hc = H + first * a.ld_hidden;
    int64_t ldh = a.ld_hidden;
    HeadPad pad{};
    pad.dim = (int)a.dim;
    pad.pad = (int)l.pad;
    if (l.copy_w && first == 0)
      pad.add(static_cast<const uint16_t*>(a.weight), a.ld_weight, (int)a.vocab, ws + l.W);
    if (l.copy_h) {
      pad.add(Hc, ldh, rows, ws + l.H);
      Hc = reinterpret_cast<const uint16_t*>(ws + l.H);
      ldh = l.pad;
    }
    if (check_launch(launch_head_pad(pad, stream), who)) return 1;
    HeadGemm g{};
    g.elt = elt;
    g.mode = !grads ? HG_STATS : elt == ELT_F16 ? HG_LOGITS : HG_EXP;
    g.splits = 1;
    g.few = a.tokens <= kFewRows;
    g.small = head_logits_small((int)a.tokens, (int)a.vocab);
    g.A = Hc; g.lda = ldh;
    g.B = W; g.ldb = ldw;
    g.M = rows; g.N = (int)a.vocab; g.K = (int)a.dim;
    g.scale = 1.f / r.temperature;
    g.Z = Z;
    g.stats = stats;
    if (check_launch(launch_head_gemm(g, stream), who)) return 1;
    if (check_launch(launch_head_rows(r, (int)first, rows, stats, Z, grads ? G : nullptr, elt, stream),
                     who)) return 1;
    if (grads) {
      g = HeadGemm{};
      g.elt = elt;
      g.mode = HG_GRAD;
      g.alpha = r.alpha;
      g.peak = rows > 0 ? r.peak : nullptr;
      g.out_dtype = a.grad_dtype;
      if (a.d_hidden) {
        g.A = G; g.lda = rows;
        g.B = W; g.ldb = ldw; g.b_kmajor = 1;
        g.M = rows; g.N = (int)a.dim; g.K = (int)a.vocab;
        g.splits = l.split_h ? head_gemm_splits(rows, g.N, g.K, false) : 1;
        g.part = floats(l.part); g.ldp = a.dim;
        g.out = static_cast<char*>(a.d_hidden) + first * a.dim * grad_size; g.ldo = a.dim;
        g.join_later = a.d_weight && head_joins_later(g, (int)a.vocab);
        if (check_launch(launch_head_gemm(g, stream), who)) return 1;
      }
      if (a.d_weight) {
        const HeadGemm h = g;
        g.join_later = 0;
        g.join = h.join_later ? &h : nullptr;
        const bool last = first + rows >= a.tokens;
        g.A = G; g.lda = rows; g.a_kmajor = 1;
        g.B = Hc; g.ldb = ldh; g.b_kmajor = 1;
        g.M = (int)a.vocab; g.N = (int)a.dim; g.K = rows;
        g.splits = l.gathers ? 1 : head_gemm_splits(g.M, g.N, g.K, true);
        g.out = last ? a.d_weight : nullptr; g.ldo = a.dim;
        // fp32 results gather in place
        g.part = l.gathers && grad_size == 4 ? static_cast<float*>(a.d_weight) : floats(l.part);
        g.ldp = a.dim;
        g.add_part = first > 0;
        if (check_launch(launch_head_gemm(g, stream), who)) return 1;
      }
    }
    if (l.chunk <= 0) break;
  }
  return 0;
}

int dmuon_scale_by(const void* src, void* dst, int64_t n, const void* src2, void* dst2, int64_t n2,
                   int src_dtype, int dst_dtype, const float* factor, void* stream) {
  const char* who = "dmuon_scale_by";
  for (int t : {src_dtype, dst_dtype})
    if (t != DMUON_DTYPE_F32 && t != DMUON_DTYPE_BF16 && t != DMUON_DTYPE_F16)
      return fail("%s: unknown dtype code %d", who, t);
  if (n < 0 || n2 < 0) return fail("%s: negative size", who);
  if (n == 0 && n2 == 0) return 0;
  if ((n > 0 && (!src || !dst)) || (n2 > 0 && (!src2 || !dst2)) || !factor)
    return fail("%s: NULL argument", who);
  const bool in1 = n > 0 && src == dst, in2 = n2 > 0 && src2 == dst2;
  if (src_dtype != dst_dtype && (in1 || in2)) return fail("%s: in place needs one dtype", who);
  ScaleBy a{{src, src2}, {dst, dst2}, {n, n2}, factor, (in1 || n == 0) && (in2 || n2 == 0)};
  return check_launch(launch_scale_by(a, src_dtype, dst_dtype, static_cast<hipStream_t>(stream)), who);
}

}  // extern "C"
