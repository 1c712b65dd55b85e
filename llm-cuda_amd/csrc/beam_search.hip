// Beam search over the paged KV cache: the selection of the best continuations
// over beams and vocabulary, and the reordering of the caches that follows it.
#include <math.h>

#include "lc_common.h"

namespace {

// ---------------------------------------------------------------------------
// Selection. value(w, v) = s_w + x_wv - lse_w with lse_w = ln sum_u exp(x_wu);
// the K largest of a group's W x V values, ties to the lowest w V + v.
//
// Inside a beam the values are ordered as its logits, so the K best of a group
// are among the K best logits of every beam, and those among the K best of
// every chunk of a beam. One pass over the logits (they are read once, from HBM,
// into registers) gives each chunk's K best and its part of the softmax sum; a
// second, small launch joins the chunks: one workgroup per group.
//
// A chunk's K best without a sort: the K-th largest of a wave's 64 lane maxima
// (found bit by bit on ballots) bounds the chunk's K-th largest from below, so
// only elements that reach the best such bound of the four waves are gathered
// (about K to 2K of them); each one's rank is the number of gathered keys above
// it. Keys are (order-preserving bits of the logit, inverted index): all are
// different, and ties rank by index.
//
// The order of candidates of different beams hangs on their lse: the terms of
// its sum are fp32 (v_exp_f32 of exact or once-rounded differences), added in
// fp32 inside a wave (2048 terms at most) and in 64 bits from there on, and the
// values are formed and compared in 64 bits and rounded to fp32 on output.
// ---------------------------------------------------------------------------
constexpr int kBeamThreads = 256;
constexpr int kBeamWaves = kBeamThreads / 64;
constexpr int kMaxCount = 64;      // candidates per group: lanes of a wave
constexpr int kMaxWidth = 256;     // beams per group: threads of a workgroup
constexpr int kChunkCap = 1024;    // gathered keys of a chunk
constexpr int kMergeCap = 2048;    // gathered candidates of a group

// Order-preserving bits of a float (not NaN); -0 counts as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
// The same in 64 bits; NaN is above everything.
__device__ __forceinline__ uint64_t ordered64(double x) {
  if (x != x) return ~0ull;
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
  return u ^ ((u >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double from_ordered64(uint64_t k) {
  if (k == ~0ull) return NAN;
  return __builtin_bit_cast(double, k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull));
}

// The largest t that at least `count` of the wave's keys reach, bits `top` .. 0.
__device__ __forceinline__ uint32_t wave_kth_largest(uint32_t key, int count, int top) {
  uint32_t t = 0;
  for (int bit = top; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    if (__popcll(__ballot(key >= c)) >= count) t = c;
  }
  return t;
}

struct SelectArgs {
  const void* logits;
  int64_t s_group, s_beam;  // element strides of logits
  const float* scores;      // [N, W]
  const uint8_t* finished;  // [N, W] or null
  uint64_t* keys;           // [N*W, chunks, K]
  double* sums;             // [N*W, chunks]
  float* tops;              // [N*W, chunks]
  float* out_scores;        // [N, K]
  int64_t* out_tokens;
  int64_t* out_parents;
  uint8_t* out_finished;
  int W, V, K, chunks, eos;
};

// 16 bytes of T from an address that may be unaligned.
template <typename T>
__device__ __forceinline__ Vec16<T> load16_any(const T* p) {
  Vec16<T> v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

template <typename T, int ITEMS>
__global__ __launch_bounds__(kBeamThreads) void beam_chunk_kernel(SelectArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int CHUNK = kBeamThreads * ITEMS;
  static_assert(ITEMS % VEC == 0, "whole vectors per thread");
  __shared__ uint64_t list[kChunkCap];
  __shared__ uint64_t bound[kBeamWaves];
  __shared__ float w_top[kBeamWaves], w_sum[kBeamWaves];
  __shared__ int count;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x - static_cast<int>(row) * a.chunks;
  if (a.finished != nullptr && a.finished[row]) return;
  const int64_t n = row / a.W;
  const T* x = static_cast<const T*>(a.logits) + n * a.s_group + (row - n * a.W) * a.s_beam;
  const int c0 = chunk * CHUNK;

  // Element i of this thread: index c0 + (i / VEC) * 256 VEC + tid VEC + i % VEC,
  // whatever the row's alignment, so equal rows give equal sums.
  float v[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS / VEC; ++j) {
    const int at = c0 + (j * kBeamThreads + tid) * VEC;
    if (at + VEC <= a.V) {
      const Vec16<T> raw = load16_any(x + at);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j * VEC + e] = lc_to_f32(raw.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j * VEC + e] = at + e < a.V ? lc_to_f32(x[at + e]) : -INFINITY;
    }
  }
  if (tid == 0) count = 0;

  // This wave's part of the softmax sum. NaN and +inf make it NaN.
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) top = fmaxf(top, v[i]);
  const float w_max = lc_wave_max(top);
  const float ref = w_max == -INFINITY ? 0.f : w_max;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) sum += lc_exp2((v[i] - ref) * kLog2e);
  sum = lc_wave_sum(sum);

  // The wave's bound: the K-th largest (value, lowest index) of its lanes.
  const uint32_t key = ordered(top);
  const uint32_t t = wave_kth_largest(key, a.K, 31);
  uint32_t t_index = 0xffffffffu;  // of elements equal to t: those of at most this index
  if (__popcll(__ballot(key >= t)) > a.K) {
    // More lanes than needed at t: the lowest indices among them are enough.
    uint32_t low = 0;  // inverted lowest index of this lane's elements equal to t
    if (key == t) {
      const float tv = from_ordered(t);
#pragma unroll
      for (int i = ITEMS - 1; i >= 0; --i)
        if (v[i] == tv) low = ~static_cast<uint32_t>(((i / VEC) * kBeamThreads + tid) * VEC + i % VEC) & 0x1fffu;
    }
    const int more = a.K - __popcll(__ballot(key > t));
    static_assert(CHUNK <= 0x2000, "indices inside a chunk are 13 bits");
    const uint32_t kth = wave_kth_largest(key == t ? low + 1 : 0, more, 13);
    t_index = 0x1fffu - (kth - 1);
  }
  if (lane == 0) {
    w_top[wave] = w_max;
    w_sum[wave] = sum;
    bound[wave] = (static_cast<uint64_t>(t) << 32) | static_cast<uint32_t>(~t_index);
  }
  __syncthreads();
  uint64_t limit = bound[0];
#pragma unroll
  for (int w = 1; w < kBeamWaves; ++w) limit = max(limit, bound[w]);

  auto key_of = [&](int i) -> uint64_t {
    const uint32_t at = ((i / VEC) * kBeamThreads + tid) * VEC + i % VEC;
    const float f = v[i] == v[i] ? v[i] : -INFINITY;
    return (static_cast<uint64_t>(ordered(f)) << 32) | static_cast<uint32_t>(~at);
  };
  if (key >= static_cast<uint32_t>(limit >> 32)) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint64_t k = key_of(i);
      if (k >= limit) {
        const int pos = atomicAdd(&count, 1);
        if (pos < kChunkCap) list[pos] = k;
      }
    }
  }
  __syncthreads();
  const int m = count;
  uint64_t* out = a.keys + (row * a.chunks + chunk) * a.K;
  // (stored with the index in the row, not in the chunk)
  auto store = [&](int rank, uint64_t k) {
    out[rank] = (k & 0xffffffff00000000ull) |
                static_cast<uint32_t>(~(~static_cast<uint32_t>(k) + static_cast<uint32_t>(c0)));
  };
  if (m <= kChunkCap) {
    for (int i = tid; i < m; i += kBeamThreads) {
      const uint64_t k = list[i];
      int rank = 0;
      for (int j = 0; j < m; ++j) rank += list[j] > k;
      if (rank < a.K) store(rank, k);
    }
  } else {
    // Values laid out against the bound (few lanes hold most of the best): the
    // largest key below the last one, K times.
    uint64_t last = ~0ull;
    for (int r = 0; r < a.K; ++r) {
      uint64_t best = 0;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const uint64_t k = key_of(i);
        if (k < last && k > best) best = k;
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t other = __shfl_xor(static_cast<unsigned long long>(best), o, 64);
        best = max(best, other);
      }
      __syncthreads();
      if (lane == 0) bound[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kBeamWaves; ++w) best = max(best, bound[w]);
      if (tid == 0) store(r, best);
      last = best;
    }
  }
  if (tid == 0) {
    // The chunk's sum relative to its largest logit.
    float hi = w_top[0];
#pragma unroll
    for (int w = 1; w < kBeamWaves; ++w) hi = fmaxf(hi, w_top[w]);
    double s = 0;
#pragma unroll
    for (int w = 0; w < kBeamWaves; ++w)
      s += w_top[w] == -INFINITY ? static_cast<double>(w_sum[w])
                                 : w_sum[w] * exp(static_cast<double>(w_top[w]) - hi);
    a.sums[row * a.chunks + chunk] = s;
    a.tops[row * a.chunks + chunk] = hi;
  }
}

// One workgroup per group: the beams' lse, then the K best of their chunks' lists.
// Beams without ordinary values stand for themselves: finished (the eos token at
// their score, -inf elsewhere), empty (no finite logit, or a score of -inf: -inf
// everywhere) and undefined (NaN or +inf in the logits or the score: NaN).
enum : int { kBeamOrdinary = 0, kBeamFinished, kBeamEmpty, kBeamUndefined };

__global__ __launch_bounds__(kBeamThreads) void beam_merge_kernel(SelectArgs a) {
  __shared__ double base[kMaxWidth];  // score - ln of the sum relative to `peak`
  __shared__ float peak[kMaxWidth];   // the beam's largest logit
  __shared__ int kind[kMaxWidth];
  __shared__ uint64_t value[kMergeCap];
  __shared__ uint32_t flat[kMergeCap];  // inverted w V + v
  __shared__ uint32_t bound[kBeamWaves];
  __shared__ uint64_t best_v[kBeamWaves];
  __shared__ uint32_t best_f[kBeamWaves];
  __shared__ int count;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t n = blockIdx.x;
  const int K = a.K;
  if (tid == 0) count = 0;
  for (int w = wave; w < a.W; w += kBeamWaves) {
    const int64_t row = n * a.W + w;
    const float score = a.scores[row];
    if (a.finished != nullptr && a.finished[row]) {
      if (lane == 0) {
        kind[w] = kBeamFinished;
        base[w] = score;
      }
      continue;
    }
    float top = -INFINITY;
    for (int c = lane; c < a.chunks; c += 64) top = fmaxf(top, a.tops[row * a.chunks + c]);
    top = lc_wave_max(top);
    double sum = 0;
    for (int c = lane; c < a.chunks; c += 64) {
      const float t = a.tops[row * a.chunks + c];
      const double s = a.sums[row * a.chunks + c];
      sum += t == -INFINITY ? s : s * exp(static_cast<double>(t) - top);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) {
      const bool empty = sum == 0 || score == -INFINITY;
      kind[w] = sum != sum || !(score < INFINITY) ? kBeamUndefined
                : empty                           ? kBeamEmpty
                                                  : kBeamOrdinary;
      // (the largest logit is taken off the logits, not added to the score: beside a
      // row of a type's lowest value neither the score nor the log would count)
      base[w] = score - log(sum);
      peak[w] = top;
    }
  }
  __syncthreads();

  // Candidate k of list (w, c): its value and inverted flat index; a value of 0
  // (below every number): none.
  const int lists = a.W * a.chunks;
  auto candidate = [&](int w, int c, int k, uint64_t& v, uint32_t& f) {
    v = 0;
    f = 0;
    const int kd = kind[w];
    uint32_t token = static_cast<uint32_t>(k);
    if (kd == kBeamOrdinary) {
      const uint64_t e = a.keys[((n * a.W + w) * a.chunks + c) * K + k];
      token = ~static_cast<uint32_t>(e);
      if (token >= static_cast<uint32_t>(a.V)) return;
      const float x = from_ordered(static_cast<uint32_t>(e >> 32));
      v = ordered64(base[w] + (static_cast<double>(x) - peak[w]));
    } else {
      if (c != 0) return;
      if (kd == kBeamFinished) {
        // eos first, then the lowest tokens
        if (k == 0)
          token = static_cast<uint32_t>(a.eos);
        else
          token = static_cast<uint32_t>(k - 1 < a.eos ? k - 1 : k);
      }
      if (token >= static_cast<uint32_t>(a.V)) return;
      v = ordered64(kd == kBeamUndefined               ? static_cast<double>(NAN)
                    : kd == kBeamFinished && k == 0 ? base[w]
                                                    : -static_cast<double>(INFINITY));
    }
    f = ~(static_cast<uint32_t>(w) * static_cast<uint32_t>(a.V) + token);
  };

  // A lower bound of the K-th largest value (its upper 32 bits) from the lists'
  // first candidates, as in the chunks.
  uint64_t head = 0;
  for (int l = tid; l < lists; l += kBeamThreads) {
    uint64_t v;
    uint32_t f;
    candidate(l / a.chunks, l % a.chunks, 0, v, f);
    head = max(head, v);
  }
  const uint32_t t = wave_kth_largest(static_cast<uint32_t>(head >> 32), K, 31);
  if (lane == 0) bound[wave] = t;
  __syncthreads();
  uint32_t limit = bound[0];
#pragma unroll
  for (int w = 1; w < kBeamWaves; ++w) limit = max(limit, bound[w]);

  const int total = lists * K;
  for (int i = tid; i < total; i += kBeamThreads) {
    uint64_t v;
    uint32_t f;
    const int l = i / K;
    candidate(l / a.chunks, l % a.chunks, i - l * K, v, f);
    if (v != 0 && static_cast<uint32_t>(v >> 32) >= limit) {
      const int pos = atomicAdd(&count, 1);
      if (pos < kMergeCap) {
        value[pos] = v;
        flat[pos] = f;
      }
    }
  }
  __syncthreads();
  const int m = count;
  auto store = [&](int rank, uint64_t v, uint32_t f) {
    const uint32_t at = ~f;
    const int w = static_cast<int>(at / static_cast<uint32_t>(a.V));
    const int token = static_cast<int>(at - static_cast<uint32_t>(w) * static_cast<uint32_t>(a.V));
    const int64_t o = n * K + rank;
    a.out_scores[o] = static_cast<float>(from_ordered64(v));
    a.out_tokens[o] = token;
    a.out_parents[o] = w;
    if (a.out_finished != nullptr)
      a.out_finished[o] = token == a.eos || (a.finished != nullptr && a.finished[n * a.W + w]);
  };
  if (m <= kMergeCap) {
    for (int i = tid; i < m; i += kBeamThreads) {
      const uint64_t v = value[i];
      const uint32_t f = flat[i];
      int rank = 0;
      for (int j = 0; j < m; ++j) rank += value[j] > v || (value[j] == v && flat[j] > f);
      if (rank < K) store(rank, v, f);
    }
  } else {
    uint64_t last_v = ~0ull;
    uint32_t last_f = ~0u;
    for (int r = 0; r < K; ++r) {
      uint64_t bv = 0;
      uint32_t bf = 0;
      auto take = [&](uint64_t v, uint32_t f) {
        if (v > bv || (v == bv && f > bf)) {
          bv = v;
          bf = f;
        }
      };
      for (int i = tid; i < total; i += kBeamThreads) {
        uint64_t v;
        uint32_t f;
        const int l = i / K;
        candidate(l / a.chunks, l % a.chunks, i - l * K, v, f);
        if (r == 0 || v < last_v || (v == last_v && f < last_f)) take(v, f);
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t ov = __shfl_xor(static_cast<unsigned long long>(bv), o, 64);
        const uint32_t of = __shfl_xor(bf, o, 64);
        take(ov, of);
      }
      __syncthreads();
      if (lane == 0) {
        best_v[wave] = bv;
        best_f[wave] = bf;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kBeamWaves; ++w) take(best_v[w], best_f[w]);
      if (tid == 0) store(r, bv, bf);
      last_v = bv;
      last_f = bf;
    }
  }
}

// Elements of a row per chunk (workgroup).
int64_t beam_chunk(int64_t rows, int64_t V) {
  (void)rows;
  (void)V;
  return kBeamThreads * 32;
}

template <typename T>
int launch_select(SelectArgs a, int64_t groups, hipStream_t st) {
  const int64_t rows = groups * a.W;
  beam_chunk_kernel<T, 32><<<static_cast<unsigned>(rows * a.chunks), kBeamThreads, 0, st>>>(a);
  const int rc = lc_check_launch("lc_beam_select (chunks)");
  if (rc != LC_OK) return rc;
  beam_merge_kernel<<<static_cast<unsigned>(groups), kBeamThreads, 0, st>>>(a);
  return lc_check_launch("lc_beam_select (merge)");
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// ---------------------------------------------------------------------------
// Reordering. Sequence (n, w) continues what (n, parents[n, w]) holds. The
// sequences of a group hold the same number of tokens, t: column c = t / P of the
// table is the page being filled (t % P slots), the columns before it hold whole
// pages, which several sequences may share, and the pages from column c on are
// each one sequence's. A parent's first child keeps the parent's page c; its
// other children take the pages c of the sequences that nobody continues, in
// order, and copy the filled slots: no page that is read is written, so the
// copies need no order among themselves, and column c stays a permutation of
// the group's own pages.
//
// One launch: the new table goes to another buffer (its old entries are read by
// every workgroup), a workgroup per group writes it, and one workgroup per
// (sequence, layer, K or V) copies.
// ---------------------------------------------------------------------------
struct ReorderArgs {
  void* kp;
  void* vp;
  int64_t s_layer, s_page, s_head, s_tok;
  const int32_t* table;
  int64_t t_stride;
  int32_t* out;
  int64_t o_stride;
  const int32_t* lens;
  const int64_t* parents;  // [N, W]
  int W, B, groups, max_pages, num_pages, Hkv, P;
  int row_units;  // 16-byte (VEC) or single elements per token row
};

template <typename U>  // the unit of a copy: 16 bytes, or one element
__global__ __launch_bounds__(256) void kv_reorder_kernel(ReorderArgs a, int elem_per_unit) {
  __shared__ int parent[kMaxWidth], first[kMaxWidth], home[kMaxWidth], used[kMaxWidth];
  __shared__ int scan_x[4], scan_f[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool rewrites = static_cast<int>(blockIdx.x) < a.groups && blockIdx.y == 0;
  const int b = static_cast<int>(blockIdx.x) - a.groups;
  if (!rewrites && b < 0) return;
  const int n = rewrites ? blockIdx.x : b / a.W;
  const int W = a.W;

  const int cap = a.max_pages * a.P;
  int len = a.lens[(int64_t)n * W];
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int col = len / a.P, fill = len - col * a.P;
  if (!rewrites && fill == 0) return;

  // Thread w: beam w's parent, whether it is the parent's first child, and the
  // beam whose page c it takes (its parent's, or a childless one's).
  int p = 0;
  if (tid < W) {
    const int64_t given = a.parents[(int64_t)n * W + tid];
    p = given >= 0 && given < W ? static_cast<int>(given) : tid;
    parent[tid] = p;
    first[tid] = W;
  }
  __syncthreads();
  if (tid < W) atomicMin(&first[p], tid);
  __syncthreads();
  const bool extra = tid < W && first[p] != tid;
  const bool spare = tid < W && first[tid] == W;
  const unsigned long long mx = __ballot(extra), mf = __ballot(spare);
  if (lane == 0) {
    scan_x[wave] = __popcll(mx);
    scan_f[wave] = __popcll(mf);
  }
  __syncthreads();
  const unsigned long long below = (1ull << lane) - 1;
  int ix = __popcll(mx & below), is = __popcll(mf & below);
  for (int w = 0; w < wave; ++w) {
    ix += scan_x[w];
    is += scan_f[w];
  }
  if (spare) used[is] = tid;  // the i-th childless beam
  __syncthreads();
  if (tid < W) home[tid] = extra ? used[ix] : p;
  __syncthreads();

  if (rewrites) {
    const int total = W * a.max_pages;
    for (int i = tid; i < total; i += 256) {
      const int w = i / a.max_pages, c = i - w * a.max_pages;
      const int from = c < col ? parent[w] : c == col && fill > 0 ? home[w] : w;
      a.out[((int64_t)n * W + w) * a.o_stride + c] = a.table[((int64_t)n * W + from) * a.t_stride + c];
    }
    return;
  }
  const int w = b - n * W;
  if (home[w] == parent[w]) return;
  const int src = a.table[((int64_t)n * W + parent[w]) * a.t_stride + col];
  const int dst = a.table[((int64_t)n * W + home[w]) * a.t_stride + col];
  if (static_cast<unsigned>(src) >= static_cast<unsigned>(a.num_pages) ||
      static_cast<unsigned>(dst) >= static_cast<unsigned>(a.num_pages) || src == dst)
    return;
  const int layer = blockIdx.y >> 1;
  U* pool = static_cast<U*>((blockIdx.y & 1) ? a.vp : a.kp) + layer * (a.s_layer / elem_per_unit);
  const U* from = pool + src * (a.s_page / elem_per_unit);
  U* to = pool + dst * (a.s_page / elem_per_unit);
  const int64_t s_head = a.s_head / elem_per_unit, s_tok = a.s_tok / elem_per_unit;
  const int per_head = fill * a.row_units, total = per_head * a.Hkv;
  constexpr int kFlight = 4;
  for (int i0 = tid; i0 < total; i0 += 256 * kFlight) {
    U x[kFlight];
    int64_t at[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const int i = min(i0 + k * 256, total - 1);
      const int h = i / per_head, r = i - h * per_head;
      const int tok = r / a.row_units;
      at[k] = h * s_head + tok * s_tok + (r - tok * a.row_units);
      x[k] = from[at[k]];
    }
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      if (i0 + k * 256 < total) to[at[k]] = x[k];
  }
}

}  // namespace

extern "C" {

int64_t lc_beam_select_workspace_bytes(int64_t groups, int64_t width, int64_t vocab,
                                       int64_t count) {
  if (groups < 0 || width <= 0 || vocab <= 0 || count <= 0) return -1;
  const int64_t rows = groups * width, lists = rows * lc_cdiv(vocab, beam_chunk(rows, vocab));
  return align256(lists * count * 8) + align256(lists * 8) + lists * 4;
}

int lc_beam_select(const void* logits, int64_t group_stride, int64_t beam_stride,
                   const float* scores, const uint8_t* finished, int64_t eos, int64_t groups,
                   int64_t width, int64_t vocab, int64_t count, float* out_scores,
                   int64_t* out_tokens, int64_t* out_parents, uint8_t* out_finished,
                   void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  static const char* who = "lc_beam_select";
  LC_REQUIRE(groups >= 0 && groups < (1LL << 31), "%s: %lld groups", who, (long long)groups);
  LC_REQUIRE(width > 0 && width <= kMaxWidth, "%s: width %lld not in [1, %d]", who,
             (long long)width, kMaxWidth);
  LC_REQUIRE(vocab > 0 && vocab < (1LL << 31) / width, "%s: width x vocab %lld x %lld not below 2^31",
             who, (long long)width, (long long)vocab);
  LC_REQUIRE(count > 0 && count <= kMaxCount && count <= width * vocab,
             "%s: %lld candidates not in [1, %d] and [1, width x vocab]", who, (long long)count,
             kMaxCount);
  LC_REQUIRE(dtype == LC_DTYPE_F32 || dtype == LC_DTYPE_F16 || dtype == LC_DTYPE_BF16,
             "%s: unknown dtype %d", who, dtype);
  LC_REQUIRE(finished == nullptr || (eos >= 0 && eos < vocab),
             "%s: eos token %lld outside the vocabulary", who, (long long)eos);
  if (groups == 0) return LC_OK;
  LC_REQUIRE(logits && scores && out_scores && out_tokens && out_parents && workspace,
             "%s: null pointer", who);
  LC_REQUIRE(group_stride >= 0 && beam_stride >= 0, "%s: negative stride", who);
  const int64_t rows = groups * width, chunks = lc_cdiv(vocab, beam_chunk(rows, vocab));
  LC_REQUIRE(rows * chunks < (1LL << 24), "%s: too many rows (%lld)", who, (long long)rows);
  const int64_t need = lc_beam_select_workspace_bytes(groups, width, vocab, count);
  if (workspace_bytes < need)
    return lc_fail(LC_EWORKSPACE, "%s: workspace %lld < %lld bytes", who,
                   (long long)workspace_bytes, (long long)need);
  LC_REQUIRE(lc_aligned(workspace, 256), "%s: workspace not 256-byte aligned", who);

  SelectArgs a{};
  a.logits = logits;
  a.s_group = group_stride;
  a.s_beam = beam_stride;
  a.scores = scores;
  a.finished = finished;
  a.keys = static_cast<uint64_t*>(workspace);
  char* at = static_cast<char*>(workspace) + align256(rows * chunks * count * 8);
  a.sums = reinterpret_cast<double*>(at);
  a.tops = reinterpret_cast<float*>(at + align256(rows * chunks * 8));
  a.out_scores = out_scores;
  a.out_tokens = out_tokens;
  a.out_parents = out_parents;
  a.out_finished = out_finished;
  a.W = static_cast<int>(width);
  a.V = static_cast<int>(vocab);
  a.K = static_cast<int>(count);
  a.chunks = static_cast<int>(chunks);
  a.eos = static_cast<int>(eos);
  hipStream_t st = lc_stream(stream);
  switch (dtype) {
    case LC_DTYPE_F32:
      return launch_select<float>(a, groups, st);
    case LC_DTYPE_BF16:
      return launch_select<bf16_t>(a, groups, st);
    default:
      return launch_select<f16_t>(a, groups, st);
  }
}

int lc_paged_kv_reorder(void* key_pages, void* value_pages, int64_t kv_s_layer, int64_t kv_s_page,
                        int64_t kv_s_head, int64_t kv_s_tok, int64_t layers, int64_t num_pages,
                        const int32_t* block_table, int64_t bt_stride, int32_t* out_table,
                        int64_t out_stride, int64_t max_pages_per_seq, const int32_t* seq_lens,
                        const int64_t* parents, int64_t groups, int64_t width, int64_t Hkv,
                        int64_t D, int64_t page_size, int dtype, void* stream) {
  static const char* who = "lc_paged_kv_reorder";
  LC_REQUIRE(width > 0 && width <= kMaxWidth, "%s: width %lld not in [1, %d]", who,
             (long long)width, kMaxWidth);
  LC_REQUIRE(groups >= 0 && groups * width < (1LL << 20), "%s: %lld groups of %lld", who,
             (long long)groups, (long long)width);
  LC_REQUIRE(layers >= 0 && layers < 32768, "%s: %lld layers", who, (long long)layers);
  LC_REQUIRE(Hkv > 0 && D > 0 && page_size > 0 && max_pages_per_seq >= 0 && num_pages >= 0 &&
                 num_pages < (1LL << 31),
             "%s: bad sizes", who);
  LC_REQUIRE(max_pages_per_seq < (1LL << 30) / page_size, "%s: a table of 2^30 tokens or more", who);
  LC_REQUIRE(Hkv < (1LL << 28) / page_size && D < (1LL << 28) / (page_size * Hkv),
             "%s: pages of 2^28 elements or more", who);
  LC_REQUIRE(dtype == LC_DTYPE_F32 || dtype == LC_DTYPE_F16 || dtype == LC_DTYPE_BF16,
             "%s: unknown dtype %d", who, dtype);
  if (groups == 0 || max_pages_per_seq == 0) return LC_OK;
  LC_REQUIRE(block_table && out_table && seq_lens && parents &&
                 ((key_pages && value_pages) || layers == 0),
             "%s: null pointer", who);
  LC_REQUIRE(bt_stride >= max_pages_per_seq && out_stride >= max_pages_per_seq,
             "%s: table stride < row length", who);
  LC_REQUIRE(kv_s_layer >= 0 && kv_s_page >= 0 && kv_s_head >= 0 && kv_s_tok >= 0,
             "%s: negative stride", who);
  const int64_t rows = groups * width;
  const char* t0 = reinterpret_cast<const char*>(block_table);
  const char* o0 = reinterpret_cast<const char*>(out_table);
  LC_REQUIRE(o0 >= t0 + ((rows - 1) * bt_stride + max_pages_per_seq) * 4 ||
                 t0 >= o0 + ((rows - 1) * out_stride + max_pages_per_seq) * 4,
             "%s: the new table overlaps the old one", who);

  ReorderArgs a{};
  a.kp = key_pages;
  a.vp = value_pages;
  a.s_layer = kv_s_layer;
  a.s_page = kv_s_page;
  a.s_head = kv_s_head;
  a.s_tok = kv_s_tok;
  a.table = block_table;
  a.t_stride = bt_stride;
  a.out = out_table;
  a.o_stride = out_stride;
  a.lens = seq_lens;
  a.parents = parents;
  a.W = static_cast<int>(width);
  a.B = static_cast<int>(rows);
  a.groups = static_cast<int>(groups);
  a.max_pages = static_cast<int>(max_pages_per_seq);
  a.num_pages = static_cast<int>(num_pages);
  a.Hkv = static_cast<int>(Hkv);
  a.P = static_cast<int>(page_size);
  const int esz = lc_dtype_size(dtype);
  const int vec = 16 / esz;
  const dim3 grid(static_cast<unsigned>(groups + rows), static_cast<unsigned>(layers > 0 ? 2 * layers : 1));
  const bool wide = D % vec == 0 && kv_s_layer % vec == 0 && kv_s_page % vec == 0 &&
                    kv_s_head % vec == 0 && kv_s_tok % vec == 0 && lc_aligned(key_pages, 16) &&
                    lc_aligned(value_pages, 16);
  hipStream_t st = lc_stream(stream);
  a.row_units = static_cast<int>(wide ? D / vec : D);
  const bool copies = layers > 0 && num_pages > 0;
  if (!copies) a.num_pages = 0;
  if (wide)
    kv_reorder_kernel<u32x4_t><<<grid, 256, 0, st>>>(a, vec);
  else if (esz == 4)
    kv_reorder_kernel<uint32_t><<<grid, 256, 0, st>>>(a, 1);
  else
    kv_reorder_kernel<uint16_t><<<grid, 256, 0, st>>>(a, 1);
  return lc_check_launch("lc_paged_kv_reorder");
}

}  // extern "C"
