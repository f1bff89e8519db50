// C entry points of attention over heads: argument checks, the plan, the workspace.
#include "../../include/dmuon_amd.h"
#include "attention.h"

namespace dmuon {
namespace {

constexpr int64_t kMost = 1LL << 30;

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check(const char* who, const dmuon_attention_args* a) {
  if (!a) return fail("%s: NULL arguments", who);
  if (a->dtype != DMUON_DTYPE_BF16 && a->dtype != DMUON_DTYPE_F16)
    return fail("%s: unknown dtype code %d", who, a->dtype);
  if (a->dim < 8 || a->dim > 128 || a->dim % 8)
    return fail("%s: dim must be a multiple of 8 and 8 .. 128, got %lld", who, (long long)a->dim);
  if (a->batch < 0 || a->batch > (1 << 20) || a->q_len < 0 || a->kv_len < 0 || a->q_len > kMost ||
      a->kv_len > kMost)
    return fail("%s: batch must be 0 .. 2^20, lengths 0 .. 2^30", who);
  if (a->kv_heads < 1 || a->heads < 1 || a->heads > 65536 || a->heads % a->kv_heads)
    return fail("%s: heads must be 1 .. 65536 and a multiple of kv_heads, got %lld and %lld", who,
                (long long)a->heads, (long long)a->kv_heads);
  if (a->q_len * (a->heads / a->kv_heads) > kMost)
    return fail("%s: q_len times the heads of a key head must be at most 2^30", who);
  // a normal fp32 number, and one times log2(e)
  if (!(a->scale >= 0x1p-126f && a->scale < 0x1p127f))
    return fail("%s: scale must be 2^-126 .. 2^127", who);
  if (a->window < 0 || (a->window > 0 && !a->causal))
    return fail("%s: a window must be positive, and needs causal", who);
  if ((a->q_starts == nullptr) != (a->kv_starts == nullptr))
    return fail("%s: q_starts and kv_starts come together", who);
  if (a->q_starts && a->kv_lengths) return fail("%s: kv_lengths are of sequences that are not packed", who);
  const int64_t units = a->q_starts ? 1 : a->batch;
  const bool rows = units > 0 && a->q_len > 0, keys = units > 0 && a->kv_len > 0;
  if ((rows && !a->q) || (keys && (!a->k || !a->v))) return fail("%s: q, k or v is NULL", who);
  if (!aligned(a->q) || !aligned(a->k) || !aligned(a->v))
    return fail("%s: q, k and v must be 16-byte aligned", who);
  const int64_t all[9] = {a->q_batch, a->q_token, a->q_head, a->k_batch, a->k_token,
                          a->k_head, a->v_batch, a->v_token, a->v_head};
  for (int64_t s : all)
    if (s < 0 || s % 8) return fail("%s: strides must be multiples of 8 values", who);
  if (a->k_token < a->dim || a->v_token < a->dim || a->k_token >= (1 << 24) || a->v_token >= (1 << 24))
    return fail("%s: tokens of k and v must be dim .. 2^24 values apart", who);
  if (65 * a->q_token + a->heads / a->kv_heads * a->q_head >= kMost)
    return fail("%s: a tile of q must span less than 2^30 values", who);
  return 0;
}

Attention describe(const dmuon_attention_args& a) {
  Attention r{};
  r.q = static_cast<const uint16_t*>(a.q);
  r.k = static_cast<const uint16_t*>(a.k);
  r.v = static_cast<const uint16_t*>(a.v);
  r.out = static_cast<uint16_t*>(a.out);
  r.lse = a.lse;
  r.rest = static_cast<uint16_t*>(a.rest);
  r.q_batch = a.q_batch; r.q_token = a.q_token; r.q_head = a.q_head;
  r.k_batch = a.k_batch; r.k_token = a.k_token; r.k_head = a.k_head;
  r.v_batch = a.v_batch; r.v_token = a.v_token; r.v_head = a.v_head;
  r.kv_lengths = a.kv_lengths;
  r.batch = (int)a.batch;
  r.heads = (int)a.heads;
  r.kv_heads = (int)a.kv_heads;
  r.group = (int)(a.heads / a.kv_heads);
  r.dim = (int)a.dim;
  r.q_len = (int)a.q_len;
  r.kv_len = (int)a.kv_len;
  // a window that reaches over all keys is none
  r.window = a.window < a.kv_len ? (int)a.window : 0;
  r.causal = a.causal != 0;
  r.dtype = a.dtype;
  r.scale = a.scale;
  r.c = a.scale * kLog2e;
  r.splits = 1;
  return r;
}

int64_t tiles_of(const Attention& a, bool packed, int64_t rows, int tile) {
  // packed: every sequence and gap may end inside a tile
  return packed ? rows / tile + a.batch + 4 : (rows + tile - 1) / tile;
}

struct Carver {
  char* base;
  int64_t at = 0;
  template <class T>
  T* take(int64_t n) {
    char* p = base ? base + at : nullptr;
    at += (n * (int64_t)sizeof(T) + 255) / 256 * 256;
    return reinterpret_cast<T*>(p);
  }
};

struct Tables {
  Sequence* seqs = nullptr;
  int2 *q = nullptr, *k = nullptr;
  int* counts = nullptr;
};
Tables tables(Attention* r, const dmuon_attention_args& a, Carver* c) {
  Tables t;
  r->tiles = (int)tiles_of(*r, a.q_starts != nullptr, (int64_t)r->q_len * r->group,
                           r->few ? kFewRows : kQueryRows);
  if (!a.q_starts) return t;
  t.seqs = c->take<Sequence>(r->batch + 4);
  t.q = c->take<int2>(r->tiles);
  t.k = c->take<int2>(tiles_of(*r, true, r->kv_len, kKeyRows));
  t.counts = c->take<int>(2);
  r->seqs = t.seqs;
  r->q_tiles = t.q;
  r->k_tiles = t.k;
  r->counts = t.counts;
  return t;
}

// Sequences of at most kFewRows rows a key head go to waves that work alone: 16 x 8 tokens over 8192 keys of
// 32/8 heads take 102 us there, 9 tokens 112 in blocks of 128 rows, 16 126 and 32 141. Packed: on average, one kernel
// for all of a call (a long sequence among many single tokens: 300 single ones over 1024 keys each and a piece of
// 2000 over 4000 take 551 us in one call, 216 and 135 in two).
bool few_rows(const Attention& a, bool packed) {
  const int64_t rows = (int64_t)a.q_len * a.group;
  return packed ? rows <= (int64_t)kFewRows * a.batch : rows <= kFewRows;
}

// Few rows over many keys do not fill the card: the keys are split. Waves that work alone take pieces of 1024
// keys (48 x 8 x 8192 keys: 157 us, of 512 165, of 256 173), or fewer where that leaves less than two waves a
// CU; blocks of 128 rows, where they are under 512, pieces of 256 or more, up to four blocks a CU. 64 parts at
// most, as the join holds one a lane: a single row tile of one or two key heads leaves CUs idle (1 token over 65536
// keys of 1, 2 and 8 key heads: 42, 43 and 52 us).
int splits_of(const Attention& a, bool packed) {
  const int64_t units = (int64_t)a.kv_heads * (packed ? 1 : a.batch);
  const int64_t blocks = units * a.tiles;
  const int64_t keys = packed && a.batch ? a.kv_len / a.batch : a.kv_len;
  if (blocks < 1) return 1;
  int64_t s;
  if (a.few) {
    s = (keys + 1023) / 1024;
    if (s * blocks < 512) s = (512 + blocks - 1) / blocks;
    if (s > (keys + 31) / 32) s = (keys + 31) / 32;
  } else {
    if (blocks >= 512) return 1;
    s = 1024 / blocks;
    if (s > keys / 256) s = keys / 256;
  }
  return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}

// Few keys' tiles: their rows are split, to a tile of 64 at the least
int key_splits_of(const Attention& a, bool packed) {
  const int64_t blocks = (int64_t)a.kv_heads * (packed ? 1 : a.batch) * a.key_tiles;
  const int64_t rows = (int64_t)a.q_len * a.group / (packed && a.batch ? a.batch : 1);
  if (blocks < 1 || blocks >= 512) return 1;
  const int64_t s = 512 / blocks, most = rows / 64;
  return most < 2 || s < 2 ? 1 : (int)(s < most ? (s < 16 ? s : 16) : (most < 16 ? most : 16));
}

struct Plan {
  Attention a;
  Tables t;
  int64_t bytes;
};
Plan plan_forward(const dmuon_attention_args& a, void* ws) {
  Plan p{describe(a), {}, 0};
  Carver c{static_cast<char*>(ws)};
  const bool packed = a.q_starts != nullptr;
  p.a.few = few_rows(p.a, packed);
  p.t = tables(&p.a, a, &c);
  p.a.splits = splits_of(p.a, packed);
  if (p.a.splits > 1) {
    const int64_t rows = p.a.splits * a.q_len * a.heads * (packed ? 1 : a.batch);
    p.a.part = c.take<float>(rows * a.dim);
    p.a.part_stats = c.take<float2>(rows);
  }
  p.bytes = c.at;
  return p;
}
Plan plan_grad(const dmuon_attention_args& a, void* ws) {
  Plan p{describe(a), {}, 0};
  Carver c{static_cast<char*>(ws)};
  const bool packed = a.q_starts != nullptr;
  p.t = tables(&p.a, a, &c);
  const int64_t batch = packed ? 1 : a.batch;
  p.a.delta = c.take<float>(a.q_len * a.heads * batch);
  p.a.key_tiles = (int)tiles_of(p.a, packed, p.a.kv_len, kKeyRows);
  p.a.key_splits = key_splits_of(p.a, packed);
  if (p.a.key_splits > 1) p.a.part = c.take<float>(p.a.key_splits * a.kv_len * a.kv_heads * batch * 2 * a.dim);
  p.bytes = c.at;
  return p;
}

int check_workspace(const char* who, int64_t need, const void* ws, int64_t bytes) {
  if (need > 0 && (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255)))
    return fail("%s: needs a 256-byte aligned workspace of %lld bytes, got %lld", who, (long long)need,
                (long long)bytes);
  return 0;
}

hipError_t fill_tables(const Plan& p, const dmuon_attention_args& a, hipStream_t s) {
  if (!a.q_starts) return hipSuccess;
  return launch_attention_tables(p.a, a.q_starts, a.kv_starts, p.a.few ? kFewRows : kQueryRows, kKeyRows, p.t.seqs, p.t.q, p.t.k,
                                 p.t.counts, s);
}

}  // namespace
}  // namespace dmuon

using namespace dmuon;

extern "C" {

int dmuon_attention_workspace_size(const dmuon_attention_args* args, int64_t* workspace_bytes) {
  const char* who = "dmuon_attention_workspace_size";
  if (!workspace_bytes) return fail("%s: NULL output", who);
  if (check(who, args)) return 1;
  *workspace_bytes = plan_forward(*args, nullptr).bytes;
  return 0;
}

int dmuon_attention(const dmuon_attention_args* args, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "dmuon_attention";
  if (check(who, args)) return 1;
  const Plan p = plan_forward(*args, workspace);
  if (check_workspace(who, p.bytes, workspace, workspace_bytes)) return 1;
  if (args->q_len == 0 || (!args->q_starts && args->batch == 0)) return 0;
  if (!args->out || !aligned(args->out) || !aligned(args->rest))
    return fail("%s: out is NULL, or out or rest not 16-byte aligned", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = check_launch(fill_tables(p, *args, s), who)) return rc;
  return check_launch(launch_attention(p.a, s), who);
}

int dmuon_attention_grad_workspace_size(const dmuon_attention_args* args, int64_t* workspace_bytes) {
  const char* who = "dmuon_attention_grad_workspace_size";
  if (!workspace_bytes) return fail("%s: NULL output", who);
  if (check(who, args)) return 1;
  *workspace_bytes = plan_grad(*args, nullptr).bytes;
  return 0;
}

int dmuon_attention_grad(const dmuon_attention_args* args, void* workspace, int64_t workspace_bytes,
                         void* stream) {
  const char* who = "dmuon_attention_grad";
  if (check(who, args)) return 1;
  const dmuon_attention_args& a = *args;
  const bool rows = a.q_len > 0 && (a.q_starts || a.batch > 0);
  if (rows && (!a.out || !a.lse || !a.dout)) return fail("%s: out, lse or dout is NULL", who);
  if (!aligned(a.out) || !aligned(a.rest) || !aligned(a.dout) || !aligned(a.dq) || !aligned(a.dk) || !aligned(a.dv))
    return fail("%s: out, rest, dout and the gradients must be 16-byte aligned", who);
  for (int64_t s : {a.do_batch, a.do_token, a.do_head})
    if (s < 0 || s % 8) return fail("%s: strides must be multiples of 8 values", who);
  if (65 * a.do_token + a.heads / a.kv_heads * a.do_head >= kMost)
    return fail("%s: a tile of dout must span less than 2^30 values", who);
  Plan p = plan_grad(a, workspace);
  if (check_workspace(who, p.bytes, workspace, workspace_bytes)) return 1;
  p.a.dout = static_cast<const uint16_t*>(a.dout);
  p.a.do_batch = a.do_batch; p.a.do_token = a.do_token; p.a.do_head = a.do_head;
  p.a.dq = static_cast<uint16_t*>(a.dq);
  p.a.dk = static_cast<uint16_t*>(a.dk);
  p.a.dv = static_cast<uint16_t*>(a.dv);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = check_launch(fill_tables(p, a, s), who)) return rc;
  return check_launch(launch_attention_grad(p.a, s), who);
}

}  // extern "C"
