// Token lookup with scaling on gfx950, and its gradient by sorted tokens.
//
//   y_t = s W[token_t],   dW[v] = s sum of dy_t over the t with token_t = v
//
// Memory bound: forward reads and writes a row a token; backward reads a row a token and writes every
// row of dW, most of them zeros. The gradient sorts the positions by token (stable, so that a class's rows
// add up in their order), walks the sorted positions in runs of 8 or 32, and joins the classes that cross
// from one run to the next in a second kernel: the sums of a class that makes up most of the text are
// spread like any other's, the join adds its runs one after the other (131072 tokens of 128256 x 4096 in bf16,
// lookup and gradient: 844 us, with half of them one class 967, all of them 1065). Sums are fp32, rounded once.
//
// 16384 tokens of 128256 x 4096 in bf16: lookup 32 us (8.4 TB/s, some of it from the caches), sort 21 (which
// clears 88 MB of the gradient meanwhile), sums 185 (6.2), joining 9. 1023 tokens of 5003 x 300 in fp16: 3, 8, 5
// and 3.5. One block sorting 16384 tokens under the clearing of dW took as long in all (radix of 9 bits 96 us, of
// 4 bits in LDS 38).
#include "../../include/dmuon_amd.h"
#include "dmuon_amd_internal.h"
#include "mfma_tile.h"

namespace dmuon {
namespace {

constexpr int kRun = 32;                  // sorted positions of a block, at most
constexpr int kAhead = 8;
constexpr int kDigit = 9, kBins = 1 << kDigit;
constexpr int kSortTile = 1024, kSortBlocks = 64, kSortAlone = 2048;
constexpr int kFillRows = 32;             // rows of dW that a block of the sums clears
constexpr long long kFillChunks = 4096;   // 16-byte chunks that a block of the sort clears
// what the launches of one pass of the sort clear: as much as they take time (3 and 5 us) at the rate of
// stores
constexpr long long kFillHist = 16LL << 20, kFillScatter = 28LL << 20;

struct Lookup {
  const int64_t* tokens; const void* weight; void* out;
  const void* dy; void* dw;
  long long n, vocab, ld, ld_dy, padding;
  int dim, dtype;
  float scale;
  // sorted: keys and positions, of the pass under way and of the next
  unsigned* key[2]; unsigned* at[2]; unsigned* hist;
  int passes, sort_blocks;
  long long sort_chunk, runs, fills;
  int run;                                // sorted positions of a block
  long long fill_at, fill_rows;           // rows of dW that a launch of the sort clears, behind its own work
  float* part;                            // [runs][2][dim]
};

typedef u32x4_t v16_t __attribute__((aligned(2)));
typedef f32x4_t f4_t __attribute__((aligned(4)));

// V values of type T (8, or 4 of fp32) at any element alignment
template <int T>
struct Vec {
  static constexpr int V = T == DT_F32 ? 4 : 8;
  float f[V];
  __device__ __forceinline__ void load(const void* p, long long at) {
    if constexpr (T == DT_F32) {
      const f32x4_t x = *reinterpret_cast<const f4_t*>(static_cast<const float*>(p) + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = x[i];
    } else {
      const u32x4_t x = *reinterpret_cast<const v16_t*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t u = (uint16_t)(i & 1 ? x[i / 2] >> 16 : x[i / 2]);
        f[i] = T == DT_F16 ? from_elt<ELT_F16>(u) : from_elt<ELT_BF16>(u);
      }
    }
  }
  // past the caches
  __device__ __forceinline__ void store(void* p, long long at) const {
    if constexpr (T == DT_F32) {
      const f32x4_t x = {f[0], f[1], f[2], f[3]};
      __builtin_nontemporal_store(x, reinterpret_cast<f4_t*>(static_cast<float*>(p) + at));
    } else {
      constexpr int E = T == DT_F16 ? ELT_F16 : ELT_BF16;
      const u32x4_t x = {pack2_elt<E>(f[0], f[1]), pack2_elt<E>(f[2], f[3]), pack2_elt<E>(f[4], f[5]),
                         pack2_elt<E>(f[6], f[7])};
      __builtin_nontemporal_store(x, reinterpret_cast<v16_t*>(static_cast<uint16_t*>(p) + at));
    }
  }
  // rows of less than V values: the first n
  __device__ __forceinline__ void load_n(const void* p, long long at, int n) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      f[i] = 0.f;
      if (i < n) {
        if constexpr (T == DT_F32) f[i] = static_cast<const float*>(p)[at + i];
        else {
          const uint16_t u = static_cast<const uint16_t*>(p)[at + i];
          f[i] = T == DT_F16 ? from_elt<ELT_F16>(u) : from_elt<ELT_BF16>(u);
        }
      }
    }
  }
  __device__ __forceinline__ void store_n(void* p, long long at, int n) const {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) {
        if constexpr (T == DT_F32) static_cast<float*>(p)[at + i] = f[i];
        else static_cast<uint16_t*>(p)[at + i] = T == DT_F16 ? to_elt<ELT_F16>(f[i]) : to_elt<ELT_BF16>(f[i]);
      }
  }
};

// Chunk c of a row: the last one of a row that is no multiple of V begins earlier, over values that the
// one before holds too, and gives them the same result. Rows of less than V values are SHORT: known to the
// compiler, since a branch at each load would have one wait for the other.
template <int T, bool SHORT>
__device__ __forceinline__ int chunk_at(int c, int dim) {
  constexpr int V = Vec<T>::V;
  return SHORT ? 0 : c * V + V <= dim ? c * V : dim - V;
}
template <int T, bool SHORT>
__device__ __forceinline__ void load_chunk(Vec<T>& v, const void* p, long long row, int at, int dim) {
  if constexpr (SHORT) v.load_n(p, row, dim);
  else v.load(p, row + at);
}
template <int T, bool SHORT>
__device__ __forceinline__ void store_chunk(const Vec<T>& v, void* p, long long row, int at, int dim) {
  if constexpr (SHORT) v.store_n(p, row, dim);
  else v.store(p, row + at);
}

// One chunk a thread, `lanes` threads a row
template <int T, bool SHORT>
__global__ __launch_bounds__(256) void embedding_kernel(const Lookup a, int chunks) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long t = id / chunks;
  if (t >= a.n) return;
  const int at = chunk_at<T, SHORT>((int)(id - t * chunks), a.dim);
  const long long v = a.tokens[t];
  Vec<T> x;
  if (v >= 0 && v < a.vocab) {
    load_chunk<T, SHORT>(x, a.weight, v * a.ld, at, a.dim);
#pragma unroll
    for (int i = 0; i < Vec<T>::V; ++i) x.f[i] *= a.scale;
  } else {
    // no class: no numbers
#pragma unroll
    for (int i = 0; i < Vec<T>::V; ++i) x.f[i] = __builtin_nanf("");
  }
  store_chunk<T, SHORT>(x, a.out, t * a.dim, at, a.dim);
}

// ---- the sort: least digit first, 9 bits a pass, every block a contiguous piece -----------------

// The sort leaves most of the card idle: further blocks clear rows of dW meanwhile, as 16-byte chunks of
// one range. What a token names among them is written again by the sums.
__device__ __forceinline__ void clear_rows(const Lookup& a, int block) {
  const long long size = a.dtype == DT_F32 ? 4 : 2;
  char* base = static_cast<char*>(a.dw) + a.fill_at * a.dim * size;
  const long long bytes = a.fill_rows * a.dim * size;
  // up to the first whole chunk, and behind the last one, in 2-byte steps
  const long long head = (16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15, lead = head < bytes ? head : bytes;
  const long long chunks = (bytes - lead) / 16, from = (long long)block * kFillChunks;
  if (block == 0) {
    for (long long i = threadIdx.x; i < lead / 2; i += blockDim.x) reinterpret_cast<uint16_t*>(base)[i] = 0;
    for (long long i = (lead + chunks * 16) / 2 + threadIdx.x; i < bytes / 2; i += blockDim.x)
      reinterpret_cast<uint16_t*>(base)[i] = 0;
  }
  const long long to = from + kFillChunks < chunks ? from + kFillChunks : chunks;
  for (long long i = from + threadIdx.x; i < to; i += blockDim.x)
    __builtin_nontemporal_store(u32x4_t{}, reinterpret_cast<u32x4_t*>(base + lead) + i);
}

// Pass 0 takes the tokens; those without a gradient come behind all others, as class `vocab`.
__device__ __forceinline__ unsigned key_of(const Lookup& a, int pass, long long i) {
  if (pass) return a.key[pass & 1][i];
  const int64_t v = a.tokens[i];
  return v >= 0 && v < a.vocab && v != a.padding ? (unsigned)v : (unsigned)a.vocab;
}

__global__ __launch_bounds__(1024) void embedding_hist_kernel(const Lookup a, int pass) {
  __shared__ unsigned bins[kBins];
  if ((int)blockIdx.x >= a.sort_blocks) return clear_rows(a, (int)blockIdx.x - a.sort_blocks);
  for (int i = threadIdx.x; i < kBins; i += 1024) bins[i] = 0;
  __syncthreads();
  const long long begin = blockIdx.x * a.sort_chunk;
  const long long end = begin + a.sort_chunk < a.n ? begin + a.sort_chunk : a.n;
  for (long long i = begin + threadIdx.x; i < end; i += 1024)
    atomicAdd(&bins[key_of(a, pass, i) >> (pass * kDigit) & (kBins - 1)], 1u);
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += 1024) a.hist[blockIdx.x * kBins + i] = bins[i];
}

__device__ __forceinline__ void scatter(const Lookup& a, int pass, bool alone) {
  __shared__ unsigned place[kBins];       // where the next of each digit goes
  __shared__ unsigned of_wave[16][kBins];
  __shared__ unsigned scan[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // places: digits before, then this digit in the blocks before
  unsigned before = 0, total = 0;
  if (alone) {
    // the only block counts its digits itself
    if (tid < kBins) place[tid] = 0;
    __syncthreads();
    for (long long i = tid; i < a.n; i += 1024)
      atomicAdd(&place[key_of(a, pass, i) >> (pass * kDigit) & (kBins - 1)], 1u);
    __syncthreads();
    if (tid < kBins) total = place[tid];
    __syncthreads();
  } else if (tid < kBins) {
    for (int b0 = 0; b0 < a.sort_blocks; b0 += 16) {
      unsigned h[16];                     // loaded side by side: one after the other they took 5 us of 8
#pragma unroll
      for (int k = 0; k < 16; ++k) h[k] = b0 + k < a.sort_blocks ? a.hist[(b0 + k) * kBins + tid] : 0u;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        before += b0 + k < (int)blockIdx.x ? h[k] : 0u;
        total += h[k];
      }
    }
  }
  unsigned sum = total;
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned u = __shfl_up(sum, d);
    if (lane >= d) sum += u;
  }
  if (tid < kBins && lane == 63) scan[wave] = sum;
  __syncthreads();
  if (tid < kBins) {
    for (int w = 0; w < wave; ++w) sum += scan[w];
    place[tid] = sum - total + before;
  }
  const long long begin = blockIdx.x * a.sort_chunk;
  const long long end = begin + a.sort_chunk < a.n ? begin + a.sort_chunk : a.n;
  for (long long i0 = begin; i0 < end; i0 += kSortTile) {
    const long long i = i0 + tid;
    const bool live = i < end;
    const unsigned key = live ? key_of(a, pass, i) : 0u;
    const unsigned at = live ? (pass ? a.at[pass & 1][i] : (unsigned)i) : 0u;
    const unsigned digit = key >> (pass * kDigit) & (kBins - 1);
    __syncthreads();
    for (int k = tid; k < 16 * kBins; k += 1024) (&of_wave[0][0])[k] = 0;
    __syncthreads();
    // lanes of the wave with the same digit
    unsigned long long same = __ballot(live);
#pragma unroll
    for (int b = 0; b < kDigit; ++b) {
      const unsigned long long set = __ballot(digit >> b & 1u);
      same &= digit >> b & 1u ? set : ~set;
    }
    const unsigned rank = __popcll(same & ((1ULL << lane) - 1));
    if (live && rank == 0) of_wave[wave][digit] = __popcll(same);
    __syncthreads();
    if (tid < kBins) {
      unsigned p = place[tid];
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        const unsigned c = of_wave[w][tid];
        of_wave[w][tid] = p;
        p += c;
      }
      place[tid] = p;
    }
    __syncthreads();
    if (live) {
      const unsigned to = of_wave[wave][digit] + rank;
      a.key[(pass + 1) & 1][to] = key;
      a.at[(pass + 1) & 1][to] = at;
    }
  }
}

__global__ __launch_bounds__(1024) void embedding_scatter_kernel(const Lookup a, int pass) {
  if ((int)blockIdx.x >= a.sort_blocks) return clear_rows(a, (int)blockIdx.x - a.sort_blocks);
  scatter(a, pass, false);
}

// All passes of a few tokens in one block (1023 tokens: 7 us for the four launches' 15)
__global__ __launch_bounds__(1024) void embedding_sort_kernel(const Lookup a) {
  if (blockIdx.x) return clear_rows(a, (int)blockIdx.x - 1);
  for (int pass = 0; pass < a.passes; ++pass) {
    scatter(a, pass, true);
    __threadfence_block();
    __syncthreads();
  }
}

// ---- sums over the sorted positions -------------------------------------------------------------

// A block: one run of sorted positions for 256 chunks of columns, or, behind the runs, the rows of dW
// that no token names.
template <int T, bool SHORT>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const Lookup a, int chunks) {
  __shared__ unsigned keys[kRun + 2], at[kRun];
  const unsigned* key = a.key[a.passes & 1];
  const int tid = threadIdx.x;
  if (blockIdx.x >= a.runs) {
    __shared__ unsigned present;
    const long long v0 = a.fill_at + (blockIdx.x - a.runs) * kFillRows;
    const int rows = a.vocab - v0 < kFillRows ? (int)(a.vocab - v0) : kFillRows;
    if (tid == 0) present = 0;
    __syncthreads();
    if (tid < rows) {
      // does any position hold class v0 + tid?
      const unsigned v = (unsigned)(v0 + tid);
      long long lo = 0, hi = a.n;
      while (lo < hi) {
        const long long mid = (lo + hi) / 2;
        if (key[mid] < v) lo = mid + 1;
        else hi = mid;
      }
      if (lo < a.n && key[lo] == v) atomicOr(&present, 1u << tid);
    }
    __syncthreads();
    const unsigned held = present;
    Vec<T> zero;
#pragma unroll
    for (int i = 0; i < Vec<T>::V; ++i) zero.f[i] = 0.f;
    for (int r = 0; r < rows; ++r) {
      if (held >> r & 1u) continue;
      for (int c = tid; c < chunks; c += 256)
        store_chunk<T, SHORT>(zero, a.dw, (v0 + r) * a.dim, chunk_at<T, SHORT>(c, a.dim), a.dim);
    }
    return;
  }
  const long long run = blockIdx.x, begin = run * a.run;
  const int n = a.n - begin < a.run ? (int)(a.n - begin) : a.run;
  // keys[0] and keys[n + 1]: the neighbours', or none
  if (tid < n + 2) {
    const long long i = begin + tid - 1;
    keys[tid] = i >= 0 && i < a.n ? key[i] : 0xffffffffu;
  }
  if (tid < n) at[tid] = a.at[a.passes & 1][begin + tid];
  __syncthreads();
  for (int c = blockIdx.y * 256 + tid; c < chunks; c += gridDim.y * 256) {
    const int col = chunk_at<T, SHORT>(c, a.dim);
    Vec<T> sum;
    bool whole = keys[0] != keys[1];      // the class begins in this run
    // kAhead rows' loads side by side (one after the other, 32 rows took 23 us)
    for (int i0 = 0; i0 < n && keys[i0 + 1] < (unsigned)a.vocab; i0 += kAhead) {
      Vec<T> x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        load_chunk<T, SHORT>(x[k], a.dy, at[i0 + k < n ? i0 + k : n - 1] * a.ld_dy, col, a.dim);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = i0 + k;
        const unsigned v = i < n ? keys[i + 1] : 0xffffffffu;
        if (v >= (unsigned)a.vocab) break;               // behind all classes
        if (i == 0 || keys[i] != v) sum = x[k];
        else
#pragma unroll
          for (int e = 0; e < Vec<T>::V; ++e) sum.f[e] += x[k].f[e];
        const bool more = keys[i + 2] == v;
        if (more && i + 1 < n) continue;
        if (whole && !more) {
#pragma unroll
          for (int e = 0; e < Vec<T>::V; ++e) sum.f[e] *= a.scale;
          store_chunk<T, SHORT>(sum, a.dw, (long long)v * a.dim, col, a.dim);
        } else {
          // part of a class that came from the run before, or that goes on in the next one
          float* part = a.part + (run * 2 + (whole ? 1 : 0)) * a.dim;
          if constexpr (SHORT) {
            for (int e = 0; e < a.dim; ++e) part[e] = sum.f[e];
          } else {
#pragma unroll
            for (int e = 0; e < Vec<T>::V; ++e) part[col + e] = sum.f[e];
          }
        }
        whole = true;
      }
    }
  }
}

// Classes that cross runs: the block of the run where one begins adds the later runs' parts in their order.
template <int T>
__global__ __launch_bounds__(256) void embedding_join_kernel(const Lookup a) {
  const unsigned* key = a.key[a.passes & 1];
  const long long run = blockIdx.x;
  const long long last = run * a.run + a.run - 1;            // there is a run behind
  const unsigned k = key[last];
  if (k >= (unsigned)a.vocab || key[last + 1] != k) return;
  if (key[run * a.run] == k && run > 0 && key[run * a.run - 1] == k) return;   // began before
  // the runs that the class goes on in: 64 at a time, a lane each
  const int lane = threadIdx.x & 63;
  long long stop = run + 1;
  for (;;) {
    const long long r = stop + lane, end = r * a.run + a.run;
    const bool on = r < a.runs && end < a.n && key[end - 1] == k && key[end] == k;
    const unsigned long long all = __ballot(on);
    if (~all) {
      stop += __ffsll(~all);              // the first one that it does not leave counts too
      break;
    }
    stop += 64;
  }
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= a.dim) return;
  float s = a.part[(run * 2 + 1) * a.dim + c];
  for (long long r0 = run + 1; r0 < stop; r0 += 8) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = r0 + i < stop ? a.part[(r0 + i) * 2 * a.dim + c] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i];
  }
  s *= a.scale;
  const long long to = (long long)k * a.dim + c;
  if constexpr (T == DT_F32) static_cast<float*>(a.dw)[to] = s;
  else static_cast<uint16_t*>(a.dw)[to] = T == DT_F16 ? to_elt<ELT_F16>(s) : to_elt<ELT_BF16>(s);
}

template <int T>
void launch_forward(const Lookup& a, hipStream_t stream) {
  const int chunks = (a.dim + Vec<T>::V - 1) / Vec<T>::V;
  const dim3 grid((unsigned)((a.n * chunks + 255) / 256));
  if (a.dim < Vec<T>::V)
    hipLaunchKernelGGL((embedding_kernel<T, true>), grid, dim3(256), 0, stream, a, chunks);
  else
    hipLaunchKernelGGL((embedding_kernel<T, false>), grid, dim3(256), 0, stream, a, chunks);
}

template <int T>
void launch_sums(const Lookup& a, hipStream_t stream) {
  const int chunks = (a.dim + Vec<T>::V - 1) / Vec<T>::V;
  const dim3 grid((unsigned)(a.runs + a.fills));
  if (a.runs + a.fills > 0 && a.dim < Vec<T>::V)
    hipLaunchKernelGGL((embedding_sum_kernel<T, true>), grid, dim3(256), 0, stream, a, chunks);
  else if (a.runs + a.fills > 0)
    hipLaunchKernelGGL((embedding_sum_kernel<T, false>), grid, dim3(256), 0, stream, a, chunks);
  if (a.runs > 1)
    hipLaunchKernelGGL((embedding_join_kernel<T>), dim3((unsigned)(a.runs - 1), (unsigned)((a.dim + 255) / 256)),
                       dim3(256), 0, stream, a);
}

int check(const char* who, const dmuon_embedding_args* a) {
  if (!a) return fail("%s: NULL arguments", who);
  if (a->dtype != DMUON_DTYPE_F32 && a->dtype != DMUON_DTYPE_BF16 && a->dtype != DMUON_DTYPE_F16)
    return fail("%s: unknown dtype code %d", who, a->dtype);
  if (a->tokens_n < 0 || a->tokens_n > (1LL << 30) || a->vocab < 1 || a->vocab > (1LL << 30) || a->dim < 1 ||
      a->dim > (1LL << 20))
    return fail("%s: tokens must be 0 .. 2^30, vocab 1 .. 2^30 and dim 1 .. 2^20", who);
  if (a->tokens_n > 0 && !a->tokens) return fail("%s: tokens is NULL", who);
  return 0;
}

// The sort's passes and pieces, and the workspace's parts; its bytes
int64_t plan(Lookup* l, const dmuon_embedding_args& a, char* ws) {
  l->tokens = a.tokens;
  l->n = a.tokens_n;
  l->vocab = a.vocab;
  l->dim = (int)a.dim;
  l->dtype = a.dtype;
  l->scale = a.scale;
  l->padding = a.padding_idx;
  l->passes = 1;
  while (l->passes * kDigit < 32 && (a.vocab >> (l->passes * kDigit))) ++l->passes;
  long long blocks = l->n <= kSortAlone ? (l->n > 0) : (l->n + kSortTile - 1) / kSortTile;
  if (blocks > kSortBlocks) blocks = kSortBlocks;
  l->sort_chunk = blocks ? ((l->n + blocks - 1) / blocks + kSortTile - 1) / kSortTile * kSortTile : kSortTile;
  l->sort_blocks = (int)((l->n + l->sort_chunk - 1) / l->sort_chunk);
  // a few tokens: short runs, whose rows are all loaded at once (1023 tokens of 300: 22 us in runs of 32)
  l->run = l->n <= 8192 ? kAhead : kRun;
  l->runs = (l->n + l->run - 1) / l->run;
  l->fills = (l->vocab + kFillRows - 1) / kFillRows;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = ws ? ws + at : nullptr;
    at += (bytes + 15) / 16 * 16;
    return p;
  };
  for (int i = 0; i < 2; ++i) {
    l->key[i] = reinterpret_cast<unsigned*>(take(4 * l->n));
    l->at[i] = reinterpret_cast<unsigned*>(take(4 * l->n));
  }
  l->hist = reinterpret_cast<unsigned*>(take(4LL * l->sort_blocks * kBins));
  l->part = reinterpret_cast<float*>(take(8 * l->runs * a.dim));
  return at;
}

}  // namespace
}  // namespace dmuon

using namespace dmuon;

extern "C" {

int dmuon_embedding(const dmuon_embedding_args* args, void* stream) {
  const char* who = "dmuon_embedding";
  if (check(who, args)) return 1;
  const dmuon_embedding_args& a = *args;
  if (a.tokens_n > 0 && (!a.weight || !a.out || a.ld_weight < a.dim))
    return fail("%s: weight or out is NULL, or the pitch is under dim", who);
  if (a.tokens_n == 0) return 0;
  Lookup l{};
  plan(&l, a, nullptr);
  l.weight = a.weight;
  l.out = a.out;
  l.ld = a.ld_weight;
  const long long v = a.dtype == DMUON_DTYPE_F32 ? 4 : 8;
  if ((a.tokens_n * ((a.dim + v - 1) / v) + 255) / 256 > 0x7fffffffLL)
    return fail("%s: too many values", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.dtype == DMUON_DTYPE_F32) launch_forward<DT_F32>(l, s);
  else if (a.dtype == DMUON_DTYPE_F16) launch_forward<DT_F16>(l, s);
  else launch_forward<DT_BF16>(l, s);
  return check_launch(hipGetLastError(), who);
}

int dmuon_embedding_grad_workspace_size(const dmuon_embedding_args* args, int64_t* workspace_bytes) {
  const char* who = "dmuon_embedding_grad_workspace_size";
  if (!workspace_bytes) return fail("%s: NULL output", who);
  if (check(who, args)) return 1;
  Lookup l{};
  *workspace_bytes = plan(&l, *args, nullptr);
  return 0;
}

int dmuon_embedding_grad(const dmuon_embedding_args* args, void* workspace, int64_t workspace_bytes,
                         void* stream) {
  const char* who = "dmuon_embedding_grad";
  if (check(who, args)) return 1;
  const dmuon_embedding_args& a = *args;
  if (!a.d_weight || (a.tokens_n > 0 && (!a.dy || a.ld_dy < a.dim)))
    return fail("%s: d_weight or dy is NULL, or the pitch is under dim", who);
  Lookup l{};
  const int64_t need = plan(&l, a, static_cast<char*>(workspace));
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail("%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", who, (long long)need,
                (long long)workspace_bytes);
  l.dy = a.dy;
  l.ld_dy = a.ld_dy;
  l.dw = a.d_weight;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t row = l.dim * (a.dtype == DMUON_DTYPE_F32 ? 4LL : 2LL);
  // rows that the next launch clears; its blocks
  auto share = [&](int64_t bytes) {
    l.fill_rows = bytes / row < l.vocab - l.fill_at ? bytes / row : l.vocab - l.fill_at;
    return (unsigned)(l.sort_blocks + ((l.fill_rows * row + 15) / 16 + kFillChunks - 1) / kFillChunks);
  };
  if (l.sort_blocks == 1) {
    const unsigned blocks = share(kFillHist + kFillScatter);
    hipLaunchKernelGGL(embedding_sort_kernel, dim3(blocks), dim3(1024), 0, s, l);
    l.fill_at += l.fill_rows;
  } else if (l.n > 0) {
    for (int p = 0; p < l.passes; ++p) {
      unsigned blocks = share(kFillHist);
      hipLaunchKernelGGL(embedding_hist_kernel, dim3(blocks), dim3(1024), 0, s, l, p);
      l.fill_at += l.fill_rows;
      blocks = share(kFillScatter);
      hipLaunchKernelGGL(embedding_scatter_kernel, dim3(blocks), dim3(1024), 0, s, l, p);
      l.fill_at += l.fill_rows;
    }
  }
  l.fills = (l.vocab - l.fill_at + kFillRows - 1) / kFillRows;
  if (a.dtype == DMUON_DTYPE_F32) launch_sums<DT_F32>(l, s);
  else if (a.dtype == DMUON_DTYPE_F16) launch_sums<DT_F16>(l, s);
  else launch_sums<DT_BF16>(l, s);
  return check_launch(hipGetLastError(), who);
}

}  // extern "C"
