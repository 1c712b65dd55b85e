// Beam search over the paged KV cache: the selection of the best continuations
// over beams and vocabulary, and the reordering of the caches that follows it.
#include <math.h>

#include <type_traits>

#include "lc_common.h"

namespace {

// ---------------------------------------------------------------------------
// Selection. value(w, v) = s_w + x_wv - lse_w with lse_w = ln sum_u exp(x_wu);
// the K largest of a group's W x V values, ties to the lowest w V + v.
//
// Inside a beam the values are ordered as its logits, so the K best of a group
// are among the K best logits of every beam, and those among the K best of
// every chunk of a beam. One pass over the logits (they are read once, from HBM,
// into registers) gives each chunk's K best and its part of the softmax sum; one
// workgroup per group then joins the chunks, in a launch of its own or, for small
// calls, in the same one.
//
// A chunk's K best without a sort: the k-th largest of a wave's 64 lane maxima
// (found on ballots, two bits at a time) bounds the chunk's K-th largest from
// below, so only elements that reach the bound are gathered (little more than K);
// each one's rank is the number of gathered keys above it. Keys are
// (order-preserving bits of the logit, inverted index): all are different, and ties
// rank by index.
//
// Bound: for many rows the instructions beside the loads (256 rows of 128256 fp32, 131
// MB: chunks 27.7 us, 4.7 TB/s, where a read stream reaches 6.9; join 10.7), for few the
// latency of two dependent passes (4 rows of 32000: 5.2 + 6.3 us; what the host takes for
// the call, 15 us, is longer).
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
constexpr int kWaveCap = 256;      // gathered keys of a chunk's wave
constexpr int kTieSlack = 8;       // lanes at the K-th value before ties are cut by index
constexpr int kMergeCap = 4096;    // gathered candidates of a group
constexpr int kMergeThreads = 1024;
constexpr int kHeldCandidates = 2048;  // most that the merge holds before the sums are joined
constexpr int kJoinCounters = 4096;
constexpr int kJoinWidth = 32;  // most beams of a group that are joined in the same launch
constexpr int kReachCap = 1024;    // lists of a group whose candidates are looked through

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

// The largest t with the bits below LOW clear that at least `count` of the wave's
// keys reach, two bits at a time (the three compares of a step are independent).
// t: their bits above TOP.
template <int TOP, int LOW>
__device__ __forceinline__ uint32_t wave_kth_largest(uint32_t key, int count, uint32_t t = 0) {
  static_assert((TOP - LOW) % 2 == 1, "whole pairs of bits");
#pragma unroll
  for (int bit = TOP - 1; bit >= LOW; bit -= 2) {
    const uint32_t c1 = t | (1u << bit), c2 = t | (2u << bit), c3 = t | (3u << bit);
    const int n1 = __popcll(__ballot(key >= c1)), n2 = __popcll(__ballot(key >= c2)),
              n3 = __popcll(__ballot(key >= c3));
    t = n3 >= count ? c3 : n2 >= count ? c2 : n1 >= count ? c1 : t;
  }
  return t;
}

// The same of four keys a lane.
template <int TOP, int LOW>
__device__ __forceinline__ uint32_t wave_kth_of_4(const uint32_t (&key)[4], int count) {
  static_assert((TOP - LOW) % 2 == 1, "whole pairs of bits");
  uint32_t t = 0;
#pragma unroll
  for (int bit = TOP - 1; bit >= LOW; bit -= 2) {
    const uint32_t c1 = t | (1u << bit), c2 = t | (2u << bit), c3 = t | (3u << bit);
    int n1 = 0, n2 = 0, n3 = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      n1 += __popcll(__ballot(key[i] >= c1));
      n2 += __popcll(__ballot(key[i] >= c2));
      n3 += __popcll(__ballot(key[i] >= c3));
    }
    t = n3 >= count ? c3 : n2 >= count ? c2 : n1 >= count ? c1 : t;
  }
  return t;
}

// The lowest bit of ordered(x) that tells values of T apart; those below it are
// all clear (x >= 0) or all set.
template <typename T>
constexpr int ordered_low() { return 0; }
template <>
constexpr int ordered_low<bf16_t>() { return 16; }
template <>
constexpr int ordered_low<f16_t>() { return 12; }

// Wave reductions on DPP moves (shifts inside rows of 16 lanes, then the row totals
// broadcast to the rows after them); the result is in lane 63.
template <typename F>
__device__ __forceinline__ float wave_reduce(float x, float none, F op) {
  auto step = [&](auto ctrl, auto rows) {
    const int moved = __builtin_amdgcn_update_dpp(
        __float_as_int(none), __float_as_int(x), decltype(ctrl)::value, decltype(rows)::value, 0xf,
        false);
    x = op(x, __int_as_float(moved));
  };
  typedef std::integral_constant<int, 0xf> All;
  step(std::integral_constant<int, 0x111>(), All());  // row_shr:1
  step(std::integral_constant<int, 0x112>(), All());
  step(std::integral_constant<int, 0x114>(), All());
  step(std::integral_constant<int, 0x118>(), All());
  step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());  // row_bcast:15
  step(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());  // row_bcast:31
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ int wave_incl_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
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
  int* counters;  // [N] tickets (beam_select_kernel)
  int W, V, K, chunks, eos;
};

// 16 bytes of T from an address that may be unaligned.
template <typename T>
__device__ __forceinline__ Vec16<T> load16_any(const T* p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
  const u4 x = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
  Vec16<T> v;
  __builtin_memcpy(&v, &x, 16);
  return v;
}

// A chunk's part (key, sum or largest logit) for the join. Where a workgroup of the
// same launch reads it, it goes through to memory by relaxed accesses of device scope.
template <bool JOIN, typename P>
__device__ __forceinline__ P part(const P* from) {
  return JOIN ? __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *from;
}
template <bool JOIN, typename P, typename X>
__device__ __forceinline__ void put_part(P* to, X from) {
  const P x = from;
  if (JOIN)
    __hip_atomic_store(to, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else
    *to = x;
}

// One workgroup per group: the beams' lse, then the K best of their chunks' lists.
// Beams without ordinary values stand for themselves: finished (the eos token at
// their score, -inf elsewhere), empty (no finite logit, or a score of -inf, finished
// or not: -inf everywhere) and undefined (NaN or +inf in the logits or the score: NaN).
enum : int { kBeamOrdinary = 0, kBeamFinished, kBeamEmpty, kBeamUndefined };

// kMergeThreads threads, room for kMergeCap gathered candidates. JOIN: the chunks' parts
// were written by other workgroups of this launch, and there are few of them.
template <int kMergeThreads, int kMergeCap, bool JOIN>
__device__ __forceinline__ void beam_merge(const SelectArgs& a, int64_t n) {
  constexpr int kMergeWaves = kMergeThreads / 64;
  __shared__ double base[kMaxWidth];  // score - ln of the sum relative to `peak`
  __shared__ float peak[kMaxWidth];   // the beam's largest logit
  __shared__ int kind[kMaxWidth];
  __shared__ uint64_t value[kMergeCap];
  __shared__ uint32_t flat[kMergeCap];  // inverted w V + v
  __shared__ int reach[kReachCap];      // lists whose best candidate reaches the bound
  __shared__ uint64_t bound[kMergeWaves];
  __shared__ uint64_t best_v[kMergeWaves];
  __shared__ uint32_t best_f[kMergeWaves];
  __shared__ int above[kMergeWaves];
  __shared__ int count, reached;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int K = a.K, lists = a.W * a.chunks;
  if (tid == 0) count = reached = 0;
  // Few candidates: every thread's kHeld of them, the lists' first ones first, are
  // loaded before the sums are joined; else a list's first and last, and of the rest
  // only those of lists that turn out to matter.
  constexpr int kHeld = kHeldCandidates / kMergeThreads;
  const bool few = JOIN || lists * K <= kHeld * kMergeThreads;  // (launch_select's rule)
  uint64_t held[kHeld];
  int held_l[kHeld], held_k[kHeld];
  if (few) {
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const uint32_t i = tid + r * kMergeThreads;
      held_k[r] = static_cast<int>(i / static_cast<uint32_t>(lists));
      held_l[r] = static_cast<int>(i) - held_k[r] * lists;
      held[r] = part<JOIN>(a.keys + (n * lists + held_l[r]) * K + min(held_k[r], K - 1));
    }
  } else {
    const uint64_t* list = a.keys + (n * lists + min(tid, lists - 1)) * K;
    held[0] = part<JOIN>(list);
    held[1] = part<JOIN>(list + K - 1);
  }
  // A row's chunks on the fewest lanes (a power of two) that hold them, so that a wave
  // joins several rows in one round trip (64 beams of 4 chunks: the merge 19.4 us with
  // a wave per row, 12.5 so).
  int lanes = 64;
  while (lanes / 2 >= a.chunks) lanes /= 2;
  const int at_once = 64 / lanes, c0 = lane & (lanes - 1);
  for (int w0 = wave * at_once; w0 < a.W; w0 += kMergeWaves * at_once) {
    const int w = w0 + lane / lanes;
    const int64_t row = n * a.W + min(w, a.W - 1);
    const float score = a.scores[row];
    const bool done = a.finished != nullptr && a.finished[row];  // (its sums are not there)
    float t0 = -INFINITY;
    double s0 = 0;
    if (c0 < a.chunks) {
      t0 = part<JOIN>(a.tops + row * a.chunks + c0);
      s0 = part<JOIN>(a.sums + row * a.chunks + c0);
    }
    float top = t0;
    for (int c = c0 + 64; c < a.chunks; c += 64)
      top = fmaxf(top, part<JOIN>(a.tops + row * a.chunks + c));
    for (int o = lanes / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    auto weighed = [&](float t, double s) {
      return t == -INFINITY ? s : s * exp(static_cast<double>(t) - top);
    };
    double sum = weighed(t0, s0);
    for (int c = c0 + 64; c < a.chunks; c += 64)
      sum += weighed(part<JOIN>(a.tops + row * a.chunks + c),
                     part<JOIN>(a.sums + row * a.chunks + c));
    for (int o = lanes / 2; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (c0 == 0 && w < a.W) {
      // (a finished beam's score may be -inf: its eos is one of equal tokens then)
      const bool dead = score == -INFINITY;
      kind[w] = done                                ? (dead ? kBeamEmpty : kBeamFinished)
                : sum != sum || !(score < INFINITY) ? kBeamUndefined
                : sum == 0 || dead                  ? kBeamEmpty
                                                    : kBeamOrdinary;
      // (the largest logit is taken off the logits, not added to the score: beside a
      // row of a type's lowest value neither the score nor the log would count)
      base[w] = done ? score : score - log(sum);
      peak[w] = top;
    }
  }
  __syncthreads();

  // Candidate k of list l = w * chunks + c, whose key is e: its value and inverted
  // flat index; a value of 0 (below every number): none.
  auto candidate_of = [&](int l, int k, uint64_t e, uint64_t& v, uint32_t& f) {
    const int w = static_cast<int>(static_cast<uint32_t>(l) / static_cast<uint32_t>(a.chunks));
    v = 0;
    f = 0;
    const int kd = kind[w];
    uint32_t token = static_cast<uint32_t>(k);
    if (kd == kBeamOrdinary) {
      token = ~static_cast<uint32_t>(e);
      if (token >= static_cast<uint32_t>(a.V)) return;
      const float x = from_ordered(static_cast<uint32_t>(e >> 32));
      v = ordered64(base[w] + (static_cast<double>(x) - peak[w]));
    } else {
      if (l != w * a.chunks) return;
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

  auto candidate = [&](int l, int k, uint64_t& v, uint32_t& f) {
    candidate_of(l, k, part<JOIN>(a.keys + (n * lists + l) * K + k), v, f);
  };

  // Candidates below `limit` are out. A candidate's key is the upper half of its value
  // and, for -inf alone (where equal halves are equal values), its inverted index.
  const uint32_t none_hi = static_cast<uint32_t>(ordered64(-static_cast<double>(INFINITY)) >> 32);
  auto key_of = [&](uint64_t v, uint32_t f) -> uint64_t {
    const uint32_t hi = static_cast<uint32_t>(v >> 32);
    return (static_cast<uint64_t>(hi) << 32) | (hi == none_hi ? f : 0);
  };
  uint64_t limit = 1;
  auto add = [&](uint64_t v, uint32_t f) {  // (whole waves)
    const bool hit = v != 0 && key_of(v, f) >= limit;
    const unsigned long long hits = __ballot(hit);
    if (hits == 0) return;
    int first = 0;
    if (lane == 0) first = atomicAdd(&count, __popcll(hits));
    const int pos = __builtin_amdgcn_readfirstlane(first) + __popcll(hits & ((1ull << lane) - 1));
    if (hit && pos < kMergeCap) {
      value[pos] = v;
      flat[pos] = f;
    }
  };
  // Raises the limit to the least of the waves' q-th best gathered candidates, q = K /
  // kMergeWaves rounded up (so K reach it), and drops what is below.
  constexpr int kEach = kMergeCap / kMergeThreads;
  auto prune = [&](int m) {
    uint64_t v[kEach];
    uint32_t f[kEach];
    uint64_t best = 0;
#pragma unroll
    for (int r = 0; r < kEach; ++r) {
      const int i = r * kMergeThreads + lane * kMergeWaves + wave;
      v[r] = i < m ? value[i] : 0;
      f[r] = i < m ? flat[i] : 0;
      if (i < m) best = max(best, key_of(v[r], f[r]));
    }
    const int q = (K + kMergeWaves - 1) / kMergeWaves;
    const uint32_t hi = static_cast<uint32_t>(best >> 32), lo = static_cast<uint32_t>(best);
    const uint32_t t = wave_kth_largest<31, 0>(hi, q);
    uint32_t cut = 0;
    if (__builtin_expect(t == none_hi, 0)) {
      const int more = q - __popcll(__ballot(hi > t));
      cut = wave_kth_largest<31, 0>(hi == t ? lo : 0, more);
    }
    if (lane == 0) bound[wave] = (static_cast<uint64_t>(t) << 32) | cut;
    __syncthreads();
    uint64_t least = bound[0];
#pragma unroll
    for (int w = 1; w < kMergeWaves; ++w) least = min(least, bound[w]);
    limit = max(limit, least);
    if (tid == 0) count = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kEach; ++r) add(v[r], f[r]);
    __syncthreads();
  };
  // The K-th best of a wave's lanes, each with its best value, is a lower bound of the
  // K-th largest value (where there are many, of all lists' first ones); so is the lowest
  // above -inf where K are above it (one live beam: the others' -inf fill the waves).
  uint64_t head = 0, held_v[kHeld];
  uint32_t held_f[kHeld];
  int n_above = 0;
  if (few) {
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      held_v[r] = 0;
      held_f[r] = 0;
      if (held_k[r] < K) candidate_of(held_l[r], held_k[r], held[r], held_v[r], held_f[r]);
      head = max(head, held_v[r]);
      n_above += __popcll(__ballot(static_cast<uint32_t>(held_v[r] >> 32) > none_hi));
    }
  } else {
    for (int l = tid; l < lists; l += kMergeThreads) {
      uint64_t v;
      uint32_t f;
      candidate_of(l, 0, l == tid ? held[0] : part<JOIN>(a.keys + (n * lists + l) * K), v, f);
      head = max(head, v);
    }
  }
  uint32_t t = 0;
  if (few) {
    t = wave_kth_largest<31, 0>(static_cast<uint32_t>(head >> 32), K);
  } else {
    reach[tid] = static_cast<int>(head >> 32);
    __syncthreads();
    if (wave == 0) {  // the K-th best of 256 threads or groups of threads
      uint32_t best[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kMergeThreads; i += 64)
        best[(i >> 6) & 3] = max(best[(i >> 6) & 3], static_cast<uint32_t>(reach[i + lane]));
      t = wave_kth_of_4<31, 10>(best, K);
    }
    // (and a list's K-th is one as well, the highest where a beam stands out)
    uint64_t v = 0;
    uint32_t f;
    if (tid < lists) candidate_of(tid, K - 1, held[1], v, f);
    uint32_t last = static_cast<uint32_t>(v >> 32);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
      last = max(last, static_cast<uint32_t>(__shfl_xor(static_cast<int>(last), o, 64)));
    t = max(t, last);
  }
  if (lane == 0) {
    bound[wave] = static_cast<uint64_t>(t) << 32;
    above[wave] = n_above;
  }
  __syncthreads();
  n_above = 0;
#pragma unroll
  for (int w = 0; w < kMergeWaves; ++w) {
    limit = max(limit, bound[w]);
    n_above += above[w];
  }
  if (n_above >= K) limit = max(limit, (static_cast<uint64_t>(none_hi) + 1) << 32);
  bool fits = true;
  if (few) {
#pragma unroll
    for (int r = 0; r < kHeld; ++r) add(held_v[r], held_f[r]);
    __syncthreads();
  } else {
    for (int l = tid; l < lists; l += kMergeThreads) {
      uint64_t v = head;
      uint32_t f;
      if (lists > kMergeThreads) candidate(l, 0, v, f);
      if (v != 0 && static_cast<uint32_t>(v >> 32) >= static_cast<uint32_t>(limit >> 32)) {
        const int pos = atomicAdd(&reached, 1);
        if (pos < kReachCap) reach[pos] = l;
      }
    }
    __syncthreads();
    // A wave takes one of these lists (of all, where they are too many), a lane one of
    // its candidates; room for the next lists' is made after every two.
    const bool listed = reached <= kReachCap;
    const int n_lists = listed ? reached : lists;
    constexpr int kRounds = kMergeCap / 2 / (kMergeWaves * kMaxCount);
    for (int i0 = 0; i0 < n_lists; i0 += kRounds * kMergeWaves) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const int i = i0 + r * kMergeWaves + wave;
        uint64_t v = 0;
        uint32_t f = 0;
        if (i < n_lists && lane < K) candidate(listed ? reach[i] : i, lane, v, f);
        add(v, f);
      }
      __syncthreads();
      int m = count;
      __syncthreads();
      if (__builtin_expect(m > kMergeCap / 2, 0)) {
        prune(m);
        m = count;
        __syncthreads();
      }
      fits = fits && m <= kMergeCap / 2;
    }
    __syncthreads();
  }
  for (int i = 0; i < 2 && __builtin_expect(fits && count > 2 * K + 64, 0); ++i) prune(count);
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
  if (__builtin_expect(fits, 1)) {
    // Eight threads count the candidates above each one.
    const int eighth = tid & 7;
    for (int i = tid >> 3; i < (m + 7) / 8 * 8; i += kMergeThreads / 8) {
      const uint64_t v = i < m ? value[i] : 0;
      const uint32_t f = i < m ? flat[i] : 0;
      int rank = 0;
#pragma unroll 4
      for (int j = eighth; j < m; j += 8) rank += value[j] > v || (value[j] == v && flat[j] > f);
      rank += __shfl_xor(rank, 1, 64);
      rank += __shfl_xor(rank, 2, 64);
      rank += __shfl_xor(rank, 4, 64);
      if (eighth == 0 && i < m && rank < K) store(rank, v, f);
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
      for (int i = tid; i < lists * K; i += kMergeThreads) {
        uint64_t v;
        uint32_t f;
        const int l = i / K;
        candidate(l, i - l * K, v, f);
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
      for (int w = 0; w < kMergeWaves; ++w) take(best_v[w], best_f[w]);
      if (tid == 0) store(r, bv, bf);
      last_v = bv;
      last_f = bf;
    }
  }
}

__global__ __launch_bounds__(kMergeThreads) void beam_merge_kernel(SelectArgs a) {
  beam_merge<kMergeThreads, kMergeCap, false>(a, blockIdx.x);
}

template <typename T, int ITEMS, bool JOIN>
__device__ __forceinline__ void beam_chunk(const SelectArgs& a) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int CHUNK = kBeamThreads * ITEMS;
  static_assert(ITEMS % VEC == 0, "whole vectors per thread");
  static_assert(CHUNK < (1 << 14), "inverted indices inside a chunk are 14 bits");
  static_assert((CHUNK & (CHUNK - 1)) == 0, "a row's chunks end at 2^31 at most");
  __shared__ uint64_t list[kBeamWaves][kWaveCap];
  __shared__ uint64_t bound_k[kBeamWaves], bound_q[kBeamWaves];
  __shared__ float w_top[kBeamWaves], w_sum[kBeamWaves];
  __shared__ int found[kBeamWaves];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // (below 2^24 workgroups)
  const int row = static_cast<int>(blockIdx.x / static_cast<uint32_t>(a.chunks));
  const int chunk = static_cast<int>(blockIdx.x) - row * a.chunks;
  // (few rows: the flag arrives with the logits instead of before them)
  const bool done = a.finished != nullptr && a.finished[row] != 0;
  if (ITEMS > 8 && done) return;
  const int n = static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(a.W));
  const T* x = static_cast<const T*>(a.logits) + n * a.s_group + (row - n * a.W) * a.s_beam;
  const int c0 = chunk * CHUNK;

  // Element i of this thread, in the chunk; whatever the row's alignment, so equal
  // rows give equal sums.
  auto index_of = [&](int i) -> uint32_t {
    return ((i / VEC) * kBeamThreads + tid) * VEC + i % VEC;
  };
  float v[ITEMS];
  if (a.V >= VEC) {
    // Every load is issued before the first is used; a vector across the row's end
    // is read again element by element, one past it reads the row's last ones.
    Vec16<T> raw[ITEMS / VEC];
#pragma unroll
    for (int j = 0; j < ITEMS / VEC; ++j)
      raw[j] = load16_any(x + min(c0 + static_cast<int>(index_of(j * VEC)), a.V - VEC));
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) v[i] = lc_to_f32(raw[i / VEC].v[i % VEC]);
    if (ITEMS <= 8 && done) return;
    if (c0 > a.V - CHUNK) {  // (the chunk's end may be 2^31; its indices are below)
#pragma unroll
      for (int j = 0; j < ITEMS / VEC; ++j) {
        const int at = c0 + static_cast<int>(index_of(j * VEC));
        if (at > a.V - VEC) {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            v[j * VEC + e] = at + e < a.V ? lc_to_f32(x[at + e]) : -INFINITY;
        }
      }
    }
  } else {
    if (done) return;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int at = c0 + static_cast<int>(index_of(i));
      v[i] = at < a.V ? lc_to_f32(x[at]) : -INFINITY;
    }
  }

  // This wave's part of the softmax sum, relative to its largest logit, whose term is
  // exactly 1 (a beam with one logit left keeps its score). NaN and +inf make it NaN.
  float top = v[0];
#pragma unroll
  for (int i = 1; i < ITEMS; ++i) top = fmaxf(top, v[i]);
  if (!(top >= -INFINITY)) top = -INFINITY;  // (all NaN)
  const float w_max = wave_reduce(top, -INFINITY, [](float p, float q) { return fmaxf(p, q); });
  const float ref = w_max == -INFINITY ? 0.f : w_max;
  float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) part[i % 4] += lc_exp2((v[i] - ref) * kLog2e);
  const float sum = wave_reduce((part[0] + part[1]) + (part[2] + part[3]), 0.f,
                                [](float p, float q) { return p + q; });

  // Two lower bounds of the chunk's K-th largest from the lanes' largest values:
  // the K-th largest of one wave, and the least of the waves' q-th largest, q = K /
  // 4 rounded up. The first always holds enough; the second, where all waves are
  // alike, little more. Elements equal to a bound count up to an index.
  // Their upper 16 bits do, but where many lanes share the K-th's or it is -inf, whose
  // upper bits alone would be a NaN's.
  const uint32_t key = ordered(top);
  constexpr int LOW = ordered_low<T>();
  auto whole = [](uint32_t t) {  // (a negative value's bits below LOW are set)
    return t < 0x80000000u ? t | ((1u << LOW) - 1) : t;
  };
  uint32_t t = wave_kth_largest<31, 16>(key, a.K);
  if constexpr (LOW < 16) {
    if (__builtin_expect(
            t < ordered(-INFINITY) || __popcll(__ballot((key ^ t) < 0x10000u)) > kTieSlack, 0))
      t = whole(wave_kth_largest<15, LOW>(key, a.K, t));
  } else {
    t = whole(t);
  }
  const int q = (a.K + kBeamWaves - 1) / kBeamWaves;
  uint32_t tq = ordered(w_max);
  if (q != 1) {
    tq = wave_kth_largest<31, 16>(key, q);
    if (LOW == 16) tq = whole(tq);
  }
  uint32_t t_index = CHUNK - 1;
  if (__builtin_expect(t == ordered(-INFINITY) || __popcll(__ballot(key == t)) > kTieSlack, 0)) {
    // Many elements at t (all masked ones, say): the lowest indices among them do. A
    // lane's first vector, the wave's first VEC x 64 indices in order, mostly holds them.
    const float tv = from_ordered(t);
    const int more = a.K - __popcll(__ballot(key > t));
    int at_t = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) at_t += v[i] == tv;
    const unsigned long long full = __ballot(wave_incl_scan(at_t) >= more);
    if (full != 0) {
      t_index = (wave * 64 + __builtin_ctzll(full)) * VEC + VEC - 1;
    } else {
      uint32_t low = 0;  // one more than the inverted lowest index of this lane's at t
#pragma unroll
      for (int i = ITEMS - 1; i >= 0; --i)
        if (v[i] == tv) low = CHUNK - index_of(i);
      t_index = CHUNK - wave_kth_largest<13, 0>(key == t ? low : 0, more);
    }
  }
  if (lane == 0) {
    w_top[wave] = w_max;
    w_sum[wave] = sum;
    bound_k[wave] = (static_cast<uint64_t>(t) << 32) | (CHUNK - t_index);
    bound_q[wave] = (static_cast<uint64_t>(tq) << 32) | 1;
  }
  __syncthreads();
  uint64_t limit = bound_k[0], least = bound_q[0];
#pragma unroll
  for (int w = 1; w < kBeamWaves; ++w) {
    limit = max(limit, bound_k[w]);
    least = min(least, bound_q[w]);
  }
  limit = max(limit, least);
  const float lim = from_ordered(static_cast<uint32_t>(limit >> 32));
  const uint32_t lim_index = CHUNK - static_cast<uint32_t>(limit);

  // (NaN: below every number; its beam's list is not used)
  auto key_at = [](float f, uint32_t i) -> uint64_t {
    return (static_cast<uint64_t>(ordered(f == f ? f : -INFINITY)) << 32) | ~i;
  };
  // Gather what reaches the bound, each wave into its own part of the list.
  int n_found = 0;
  if (__ballot(top >= lim)) {
    auto gather = [&](int i, bool hit) {
      const unsigned long long hits = __ballot(hit);
      if (hits == 0) return;
      const int pos = n_found + __builtin_amdgcn_mbcnt_hi(
                                    static_cast<uint32_t>(hits >> 32),
                                    __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(hits), 0));
      if (hit && pos < kWaveCap) list[wave][pos] = key_at(v[i], index_of(i));
      n_found += __popcll(hits);
    };
    if (__builtin_expect(lim_index == CHUNK - 1, 1)) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) gather(i, v[i] >= lim);
    } else {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        gather(i, v[i] > lim || (v[i] == lim && index_of(i) <= lim_index));
    }
  }
  if (lane == 0) found[wave] = n_found;
  __syncthreads();
  int m = 0, most = 0, before[kBeamWaves];
#pragma unroll
  for (int w = 0; w < kBeamWaves; ++w) {
    before[w] = m;
    m += found[w];
    most = max(most, found[w]);
  }
  uint64_t* out = a.keys + (static_cast<int64_t>(row) * a.chunks + chunk) * a.K;
  // (stored with the index in the row, not in the chunk)
  auto store = [&](int rank, uint64_t k) {
    const uint32_t at = ~(~static_cast<uint32_t>(k) + static_cast<uint32_t>(c0));
    put_part<JOIN>(out + rank, (k & 0xffffffff00000000ull) | at);
  };
  if (__builtin_expect(most <= kWaveCap, 1)) {
    // Four threads count the keys above each one, a wave's part of the list each.
    static_assert(kBeamWaves == 4, "a thread per part");
    const int seg = tid & 3, n_seg = found[seg];
    for (int i = tid >> 2; i < (m + 15) / 16 * 16; i += kBeamThreads / 4) {
      int at = 0;
#pragma unroll
      for (int w = 1; w < kBeamWaves; ++w) at = i >= before[w] ? w : at;
      const uint64_t k = i < m ? list[at][i - before[at]] : ~0ull;
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n_seg; ++j) rank += list[seg][j] > k;
      rank += __shfl_xor(rank, 1, 64);
      rank += __shfl_xor(rank, 2, 64);
      if (seg == 0 && i < m && rank < a.K) store(rank, k);
    }
  } else {
    // Values laid out against the bounds (few lanes hold most of the best): the next
    // element after the last one, K times. (Floats, not keys: those the compiler would
    // make before the loop and keep, in registers that the kernel has not.)
    float last_f = INFINITY;
    uint32_t last_i = ~0u;
    for (int r = 0; r < a.K; ++r) {
      float f = -INFINITY;
      uint32_t at = ~0u;
#pragma unroll
      for (int i = ITEMS - 1; i >= 0; --i) {
        const uint32_t here = index_of(i);
        if ((v[i] < last_f || (v[i] == last_f && here > last_i)) && v[i] >= f) {
          f = v[i];
          at = here;
        }
      }
      uint64_t best = at == ~0u ? 0 : key_at(f, at);
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t other = __shfl_xor(static_cast<unsigned long long>(best), o, 64);
        best = max(best, other);
      }
      __syncthreads();
      if (lane == 0) bound_k[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kBeamWaves; ++w) best = max(best, bound_k[w]);
      if (tid == 0) store(r, best);
      last_f = from_ordered(static_cast<uint32_t>(best >> 32));  // (0, none left: NaN)
      last_i = ~static_cast<uint32_t>(best);
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
    put_part<JOIN>(a.sums + static_cast<int64_t>(row) * a.chunks + chunk, s);
    put_part<JOIN>(a.tops + static_cast<int64_t>(row) * a.chunks + chunk, hi);
  }
}

// (8 waves per SIMD: 256 rows of 128256 fp32, 131 MB, take 27.7 us, 4.7 TB/s; 31.3 with 5)
template <typename T, int ITEMS>
__global__ __launch_bounds__(kBeamThreads, 8) void beam_chunk_kernel(SelectArgs a) {
  beam_chunk<T, ITEMS, false>(a);
}

// Few beams and candidates: the workgroup of a group that finishes last (its ticket on
// counters[n], zero at entry and left zero) joins the chunks, in the same launch. The
// GPU takes about as long as in two (calls in a graph, us: 4 beams of 32000 10.7 / 11.2, 16
// of 1003 11.9 / 12.4, 32 of 2000 15.4 / 13.5, 8 groups of 4 x 32000 15.9 / 12.1), and the
// host, which such a call waits for, a launch less: 17.4 -> 15.4 us a call. Of 23 sizes
// of 1 to 60 groups, 1 to 32 beams and 1000 to 128256 tokens the joined call is 0.5 to 2.4
// us shorter at 22; with 32 beams and 64 candidates it is 0.5 us longer.
template <typename T>
__global__ __launch_bounds__(kBeamThreads) void beam_select_kernel(SelectArgs a) {
  __shared__ int last;
  beam_chunk<T, 8, true>(a);
  const int64_t n = blockIdx.x / (a.W * a.chunks);
  // (every wave's stores have reached memory before the ticket is taken)
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  lc_compiler_fence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int t =
        __hip_atomic_fetch_add(a.counters + n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = t == a.W * a.chunks - 1;
    if (last) __hip_atomic_store(a.counters + n, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  lc_compiler_fence();
  beam_merge<kBeamThreads, kHeldCandidates, true>(a, n);
}

// Logits of a row per workgroup: 8192 where that gives every CU a workgroup, else
// 2048, so that a few rows' latency is short (four times the lists to join: with 31
// beams of 55157 the join took 17 us, the chunks 11).
int beam_items(int64_t rows, int64_t V) {
  return rows * lc_cdiv(V, kBeamThreads * 32) >= lc_cu_count() ? 32 : 8;
}
int64_t beam_chunks(int64_t rows, int64_t V) {
  return lc_cdiv(V, kBeamThreads * beam_items(rows, V));
}

template <typename T>
int launch_select(SelectArgs a, int64_t groups, hipStream_t st) {
  const int64_t rows = groups * a.W;
  const unsigned blocks = static_cast<unsigned>(rows * a.chunks);
  // One launch where the join is small, since its workgroup has 256 threads.
  if (a.counters != nullptr && beam_items(rows, a.V) == 8 && groups <= kJoinCounters &&
      a.W <= kJoinWidth && (int64_t)a.W * a.chunks * a.K <= kHeldCandidates) {
    beam_select_kernel<T><<<blocks, kBeamThreads, 0, st>>>(a);
    return lc_check_launch("lc_beam_select");
  }
  if (beam_items(rows, a.V) == 32)
    beam_chunk_kernel<T, 32><<<blocks, kBeamThreads, 0, st>>>(a);
  else
    beam_chunk_kernel<T, 8><<<blocks, kBeamThreads, 0, st>>>(a);
  const int rc = lc_check_launch("lc_beam_select (chunks)");
  if (rc != LC_OK) return rc;
  beam_merge_kernel<<<static_cast<unsigned>(groups), kMergeThreads, 0, st>>>(a);
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
// Bound: HBM (4 groups of 8, 3 childless each, 32 layers of 8 x 44 x 128 bf16 slots: 138
// MB read and written in 38 us) or, for few copies, the launch and the chain parents ->
// table -> page (5.5 us).
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

int64_t lc_beam_select_counter_count(void) { return kJoinCounters; }

int64_t lc_beam_select_workspace_bytes(int64_t groups, int64_t width, int64_t vocab,
                                       int64_t count) {
  if (groups < 0 || width <= 0 || vocab <= 0 || count <= 0) return -1;
  const int64_t rows = groups * width, lists = rows * beam_chunks(rows, vocab);
  return align256(lists * count * 8) + align256(lists * 8) + lists * 4;
}

int lc_beam_select(const void* logits, int64_t group_stride, int64_t beam_stride,
                   const float* scores, const uint8_t* finished, int64_t eos, int64_t groups,
                   int64_t width, int64_t vocab, int64_t count, float* out_scores,
                   int64_t* out_tokens, int64_t* out_parents, uint8_t* out_finished,
                   void* workspace, int64_t workspace_bytes, int32_t* counters, int dtype,
                   void* stream) {
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
  const int64_t rows = groups * width, chunks = beam_chunks(rows, vocab);
  LC_REQUIRE(rows * chunks < (1LL << 24), "%s: too many rows (%lld)", who, (long long)rows);
  const int64_t need = lc_beam_select_workspace_bytes(groups, width, vocab, count);
  if (workspace_bytes < need)
    return lc_fail(LC_EWORKSPACE, "%s: workspace %lld < %lld bytes", who,
                   (long long)workspace_bytes, (long long)need);
  LC_REQUIRE(lc_aligned(workspace, 256), "%s: workspace not 256-byte aligned", who);
  LC_REQUIRE(lc_aligned(counters, 4), "%s: counters not 4-byte aligned", who);

  SelectArgs a{};
  a.counters = counters;
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
  LC_REQUIRE(width * max_pages_per_seq < (1LL << 31) - 256,
             "%s: a table of 2^31 entries a group or more", who);
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
