// Verification of drafted tokens against the target model's probabilities, from
// given random numbers.
//
// p_i = softmax(x[b, i] / temperature), q_i = softmax(y[b, i] / temperature) (or all
// mass on the drafted token). Draft i stands iff all before it do and u_i q_i(d_i) <
// p_i(d_i); with a of them standing, the next token is drawn by u_K from w = p_a, or
// from w = max(p_a - q_a, 0) where draft a was refused: the first v with
// sum_{j <= v} w_j > u_K sum_j w_j. So every token is distributed as the target's.
//
// A token's interval on the running sum may be any small part of it, and a border off by
// 1e-7 of the sum (what fp32 terms leave) gives another token in a hundredth of the
// draws from 128256 tokens. The sums that choose a token are therefore formed in 64
// bits from 64-bit exponentials; they concern one row of a sequence (two with a refused
// draft). Whether a draft stands is one comparison, for which sums of fp32 terms
// (added in 64 bits from a wave's on) do: a sum off by some 1e-7, at worst 2.2e-6 (see
// verify_stats_kernel), turns as large a part of the comparisons.
//
// Launches: statistics of every chunk of every row; decisions, a workgroup per sequence; the
// 64-bit sums of the chosen rows; the residual's, where drafts have logits; the token. 64
// sequences of up to 5 drafts, 128256 fp32 logits: 38 + 5 + 21 + 19 + 14 us; one of 4 drafts
// without logits, 32000 bf16: 3.5 + 3.8 + 3.7 + 7.2.
#include <math.h>

#include <type_traits>

#include "lc_common.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kItems = 8;                  // consecutive elements of a thread
constexpr int kBlock = kThreads * kItems;  // and of a workgroup
constexpr int kDecideThreads = 1024, kDecideWaves = kDecideThreads / 64;
constexpr int kMaxDrafts = 255;
// A residual max(p - q, 0) that sums to less is rounding: p and q agree.
constexpr double kAgree = 2.3283064365386963e-10;  // 2^-32

struct Stat {  // of a chunk of a row
  float top;   // its largest logit (NaN: it holds one)
  int arg;     // where it first is (only where all mass may be there)
  double sum;  // of exp((x - top) / temperature)
};

struct Verdict {      // of a sequence
  int accepted;       // drafts that stand
  int chosen;         // whether the new token is known
  int refused;        // whether a draft was refused
  int q_arg;          // all of the refused draft's q is here (-1: it is spread, or none)
  float p_top, q_top;
};

struct VerifyArgs {
  const void* x;  // [B, K + 1, V]
  int64_t x_sb, x_si;
  const void* y;  // [B, K, V] or null
  int64_t y_sb, y_si;
  const int64_t* drafts;  // [B, K]
  const float* u;         // [B, K + 1]
  const int32_t* lens;    // [B] or null
  const float* temps;     // [B] or null: temperature
  double temperature;
  int64_t* tokens;    // [B, K + 1]
  int32_t* accepted;  // [B]
  Stat* stats;        // [B, 2 K + 1, chunks]
  Verdict* verdicts;  // [B]
  double* sums;       // 3 of [B, chunks]: p's terms; q's, or p's without q_arg; the residual
  int B, K, V, chunks;
  int blocks;  // of kBlock elements of a chunk
};

__device__ __forceinline__ double temperature_of(const VerifyArgs& a, int b) {
  return a.temps != nullptr ? static_cast<double>(a.temps[b]) : a.temperature;
}
// A positive finite temperature; others stand for the first largest logit.
__device__ __forceinline__ bool spreads(double temp) { return temp > 0 && temp < INFINITY; }
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) {
  if (a.lens == nullptr) return a.K;
  const int n = a.lens[b];
  return n < 0 ? 0 : n > a.K ? a.K : n;
}

// (0 times it stays 0)
__device__ __forceinline__ double inverse(double temp) { return fmin(1.0 / temp, 1e300); }

template <typename T>
__device__ __forceinline__ const T* target_row(const VerifyArgs& a, int b, int i) {
  return static_cast<const T*>(a.x) + (int64_t)b * a.x_sb + (int64_t)i * a.x_si;
}
template <typename T>
__device__ __forceinline__ const T* draft_row(const VerifyArgs& a, int b, int i) {
  return static_cast<const T*>(a.y) + (int64_t)b * a.y_sb + (int64_t)i * a.y_si;
}

// This thread's kItems consecutive elements of a row from v0 on; past the end: -inf. (A
// row may begin anywhere.)
template <typename T>
__device__ __forceinline__ void load_items(const T* row, int64_t v0, int V, float (&v)[kItems]) {
  constexpr int VEC = 16 / sizeof(T);
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
  if (v0 + kItems <= V) {
#pragma unroll
    for (int j = 0; j < kItems / VEC; ++j) {
      const u4 raw = *reinterpret_cast<const u4*>(row + v0 + j * VEC);
      Vec16<T> x;
      __builtin_memcpy(&x, &raw, 16);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j * VEC + e] = lc_to_f32(x.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kItems; ++e) v[e] = v0 + e < V ? lc_to_f32(row[v0 + e]) : -INFINITY;
  }
}

// x of another lane of the wave, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ double lane_move(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
// Sum over the lanes up to this one, and over all (the last lane's).
__device__ __forceinline__ double wave_scan_f64(double x) {
  x += lane_move<0x111, 0xf>(x);  // row_shr:1
  x += lane_move<0x112, 0xf>(x);
  x += lane_move<0x114, 0xf>(x);
  x += lane_move<0x118, 0xf>(x);
  x += lane_move<0x142, 0xa>(x);  // row_bcast:15
  x += lane_move<0x143, 0xc>(x);  // row_bcast:31
  return x;
}
__device__ __forceinline__ double last_lane(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), 63);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), 63);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ double wave_sum_f64(double x) { return last_lane(wave_scan_f64(x)); }

// e^y for y <= 0, off by at most 2^-46.6 + |y| 2^-54.7 relatively (2^-44.8 at -700): y =
// k ln 2 + z with |z| <= ln 2 / 2, and the power series of e^z up to z^11. The next term
// is 2^-46.7 of e^z where z is -ln 2 / 2; one double for ln 2 is off by 2^-55.3, k times
// (a large |y| means a small term). k, found by adding 1.5 * 2^52, goes into the
// exponent's bits; below -700 the term is 0.
__device__ __forceinline__ double exp_f64(double y) {
  constexpr double kShift = 6755399441055744.0;
  const double t = fma(y, 1.4426950408889634, kShift);
  const double z = fma(kShift - t, 0.6931471805599453, y);
  double p = 1.0 / 39916800;
  p = fma(p, z, 1.0 / 3628800);
  p = fma(p, z, 1.0 / 362880);
  p = fma(p, z, 1.0 / 40320);
  p = fma(p, z, 1.0 / 5040);
  p = fma(p, z, 1.0 / 720);
  p = fma(p, z, 1.0 / 120);
  p = fma(p, z, 1.0 / 24);
  p = fma(p, z, 1.0 / 6);
  p = fma(p, z, 0.5);
  p = fma(p, z, 1.0);
  p = fma(p, z, 1.0);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  const uint32_t high = static_cast<uint32_t>(bits >> 32) +
                        (static_cast<uint32_t>(__builtin_bit_cast(uint64_t, t)) << 20);
  const double e = __builtin_bit_cast(double, (static_cast<uint64_t>(high) << 32) | static_cast<uint32_t>(bits));
  return y >= -700.0 ? e : 0.0;
}

// Chunk statistics: one workgroup per (chunk, row); rows are a sequence's K + 1 target
// rows, then its K draft rows. Rows past the sequence's drafts are not read. Bound by
// reading the logits once (64 sequences of up to 5 drafts, 128256 fp32 logits: 240 MB in 37
// us, 6.5 TB/s).
// How far a chunk's sum may be off: three roundings of a term's exponent (the difference, the
// scale, the product), 3 * 2^-24 times the terms' mean exponent, which is at most 6.2 (8191
// equal logits under one that is larger by 7.2 temperatures); the exponential, 2^-23; 16
// additions, 2^-24 each. Together 2.2e-6; the roundings of other rows mostly cancel.
template <typename T, int BLOCKS>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
  const int rows = 2 * a.K + 1;
  const int chunk = blockIdx.x % a.chunks, br = blockIdx.x / a.chunks;
  const int b = br / rows, r = br % rows;
  const int n = drafts_of(a, b);
  const bool target = r <= a.K;
  const int i = target ? r : r - (a.K + 1);
  if (target ? i > n : (a.y == nullptr || i >= n)) return;
  const T* row = target ? target_row<T>(a, b, i) : draft_row<T>(a, b, i);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t v0 = (int64_t)chunk * (BLOCKS * kBlock) + tid * kItems;
  float v[BLOCKS][kItems];
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) load_items(row, v0 + j * kBlock, a.V, v[j]);
  __shared__ float tops[kWaves], sums[kWaves];
  __shared__ int first;
  float top = -INFINITY;  // (fmaxf passes over NaN)
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
    for (int e = 0; e < kItems; ++e) top = fmaxf(top, v[j][e]);
  const float mine = top;
  top = lc_wave_max(top);
  if (lane == 0) tops[wave] = top;
  if (tid == 0) first = 0x7fffffff;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
  const double temp = temperature_of(a, b);
  // (kept finite and above 0: 0 and -inf stay what they are)
  const float c = static_cast<float>(fmin(fmax(1.4426950408889634 / temp, 1e-37), 1e37));
  const float ref = top == -INFINITY ? 0.f : top;
  float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
    for (int e = 0; e < kItems; ++e) part[e % 4] += lc_exp2((v[j][e] - ref) * c);
  const float s = lc_wave_sum((part[0] + part[1]) + (part[2] + part[3]));
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  double all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += sums[w];
  // NaN and +inf make the sum NaN. Then, and where the temperature puts all mass on the
  // largest logit, its first place is needed.
  bool nan = false;
  if (all != all) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
      for (int e = 0; e < kItems; ++e) any |= v[j][e] != v[j][e];
    nan = __syncthreads_or(any);
  }
  if (all != all || !spreads(temp)) {
    if (nan || mine == top) {
      int at = 0x7fffffff;
#pragma unroll
      for (int j = BLOCKS - 1; j >= 0; --j)
#pragma unroll
        for (int e = kItems - 1; e >= 0; --e) {
          const int64_t p = v0 + j * kBlock + e;
          if (p < a.V && (nan ? v[j][e] != v[j][e] : v[j][e] == top)) at = static_cast<int>(p);
        }
      if (at != 0x7fffffff) atomicMin(&first, at);
    }
    __syncthreads();
  }
  if (tid == 0)
    a.stats[((int64_t)b * rows + r) * a.chunks + chunk] = Stat{nan ? NAN : top, first, all};
}

// A row's largest logit, where it is, and its sum, from its chunks (one wave).
struct RowSum {
  double sum;
  float top;
  int arg;      // where all mass is; -1: it is spread
};
__device__ __forceinline__ RowSum row_sum(const VerifyArgs& a, int b, int r, double temp) {
  const Stat* s = a.stats + ((int64_t)b * (2 * a.K + 1) + r) * a.chunks;
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  int nan = 0x7fffffff;
  for (int c = lane; c < a.chunks; c += 64) {
    if (s[c].top != s[c].top)
      nan = min(nan, s[c].arg);
    else
      top = fmaxf(top, s[c].top);
  }
  top = lc_wave_max(top);
  const bool any_nan = __ballot(nan != 0x7fffffff) != 0;
  if (!any_nan && fabsf(top) < INFINITY && spreads(temp)) {
    double sum = 0;
    for (int c = lane; c < a.chunks; c += 64)
      sum += s[c].sum * exp_f64((static_cast<double>(s[c].top) - top) / temp);
    return RowSum{wave_sum_f64(sum), top, -1};
  }
  int arg = nan;
  if (!any_nan)
    for (int c = lane; c < a.chunks; c += 64)
      if (s[c].top == top) arg = min(arg, s[c].arg);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) arg = min(arg, __shfl_xor(arg, o, 64));
  // (a row of -inf alone has no sum that told its first place: it is 0)
  return RowSum{1, top, arg == 0x7fffffff ? 0 : arg};
}

template <typename T>
__device__ __forceinline__ double chance(const T* row, int64_t d, int V, const RowSum& s,
                                         double temp) {
  if (d < 0 || d >= V) return 0;
  if (s.arg >= 0) return d == s.arg ? 1 : 0;
  return exp_f64((static_cast<double>(lc_to_f32(row[d])) - s.top) / temp) / s.sum;
}

// One workgroup per sequence: its rows' sums, a wave each, then which drafts stand. Where
// all mass of the next row is in one place, that is the new token.
template <typename T>
__global__ __launch_bounds__(kDecideThreads) void verify_decide_kernel(VerifyArgs a) {
  __shared__ RowSum rs[2 * kMaxDrafts + 1];
  __shared__ int fell;
  const int b = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const int n = drafts_of(a, b);
  const double temp = temperature_of(a, b);
  if (tid == 0) fell = n;
  const int live = n + 1 + (a.y != nullptr ? n : 0);
  for (int i = wave; i < live; i += kDecideWaves) {
    const RowSum s = row_sum(a, b, i <= n ? i : a.K + i - n, temp);
    if ((tid & 63) == 0) rs[i] = s;
  }
  __syncthreads();
  if (tid < n) {
    const int64_t d = a.drafts[(int64_t)b * a.K + tid];
    const double p = chance(target_row<T>(a, b, tid), d, a.V, rs[tid], temp);
    const double q =
        a.y == nullptr ? 1 : chance(draft_row<T>(a, b, tid), d, a.V, rs[n + 1 + tid], temp);
    if (!(a.u[(int64_t)b * (a.K + 1) + tid] * q < p)) atomicMin(&fell, tid);
  }
  __syncthreads();
  const int accepted = fell;
  const RowSum p = rs[accepted];
  for (int i = tid; i <= a.K; i += kDecideThreads)
    a.tokens[(int64_t)b * (a.K + 1) + i] = i < accepted                  ? a.drafts[(int64_t)b * a.K + i]
                                           : i == accepted && p.arg >= 0 ? p.arg
                                                                         : -1;
  if (tid == 0) {
    Verdict v{accepted, p.arg >= 0, accepted < n, -1, p.top, 0.f};
    if (v.refused && a.y != nullptr) {
      v.q_top = rs[n + 1 + accepted].top;
      v.q_arg = rs[n + 1 + accepted].arg;
    } else if (v.refused) {
      const int64_t d = a.drafts[(int64_t)b * a.K + accepted];
      v.q_arg = d >= 0 && d < a.V ? static_cast<int>(d) : -1;
    }
    a.accepted[b] = accepted;
    a.verdicts[b] = v;
  }
}

// The row's terms of this thread's elements, not divided by their sum (past the end: 0).
__device__ __forceinline__ void terms(const float (&x)[kItems], float top, double inv_temp,
                                      double (&e)[kItems]) {
#pragma unroll
  for (int i = 0; i < kItems; ++i) e[i] = exp_f64((static_cast<double>(x[i]) - top) * inv_temp);
}

template <int WAVES>
__device__ __forceinline__ double block_sum(double x, double* sums) {
  x = wave_sum_f64(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
  __syncthreads();
  double all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) all += sums[w];
  return all;
}

// A refused draft's q is spread over the vocabulary: its terms are needed.
__device__ __forceinline__ bool reads_draft(const VerifyArgs& a, const Verdict& v) {
  return v.refused && v.q_arg < 0 && a.y != nullptr;
}
__device__ __forceinline__ double* plane(const VerifyArgs& a, int which, int b) {
  return a.sums + ((int64_t)which * a.B + b) * a.chunks;
}

// 64-bit sums of a chunk's terms. One round of workgroups, which load and then compute: of 21
// us (64 rows and the refused drafts', 128256 fp32 logits) the vector units issue for 14
// (7.3 million instructions in 4096 waves, mostly 64-bit exponentials).
template <typename T, int BLOCKS>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
  __shared__ double sums[kWaves];
  const int chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
  const Verdict v = a.verdicts[b];
  if (v.chosen) return;
  const bool both = reads_draft(a, v);
  const double inv = inverse(temperature_of(a, b));
  const int64_t v0 = (int64_t)chunk * (BLOCKS * kBlock) + threadIdx.x * kItems;
  float x[BLOCKS][kItems], y[BLOCKS][kItems];
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) load_items(target_row<T>(a, b, v.accepted), v0 + j * kBlock, a.V, x[j]);
  if (both)
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j)
      load_items(draft_row<T>(a, b, v.accepted), v0 + j * kBlock, a.V, y[j]);
  double sp = 0, sq = 0;
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) {
    double e[kItems];
    terms(x[j], v.p_top, inv, e);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      sp += e[i];
      if (v0 + j * kBlock + i != v.q_arg) sq += e[i];
    }
  }
  if (both) {
    sq = 0;
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      double e[kItems];
      terms(y[j], v.q_top, inv, e);
#pragma unroll
      for (int i = 0; i < kItems; ++i) sq += e[i];
    }
  }
  sp = block_sum<kWaves>(sp, sums);
  sq = block_sum<kWaves>(sq, sums);
  if (threadIdx.x == 0) {
    plane(a, 0, b)[chunk] = sp;
    plane(a, 1, b)[chunk] = sq;
  }
}

// Sum of a plane's chunks of sequence b, by all threads of the workgroup.
template <int WAVES>
__device__ __forceinline__ double row_total(const VerifyArgs& a, int which, int b, double* sums) {
  double s = 0;
  for (int c = threadIdx.x; c < a.chunks; c += WAVES * 64) s += plane(a, which, b)[c];
  return block_sum<WAVES>(s, sums);
}

// max(p - q, 0) of elements of both rows.
__device__ __forceinline__ void residual(const Verdict& v, const float (&x)[kItems],
                                         const float (&y)[kItems], double inv, double inv_zp,
                                         double inv_zq, double (&w)[kItems]) {
  double e[kItems];
  terms(x, v.p_top, inv, w);
  terms(y, v.q_top, inv, e);
#pragma unroll
  for (int i = 0; i < kItems; ++i) w[i] = fmax(w[i] * inv_zp - e[i] * inv_zq, 0.0);
}

// Sums of a chunk's residual.
template <typename T, int BLOCKS>
__global__ __launch_bounds__(kThreads) void verify_residual_kernel(VerifyArgs a) {
  __shared__ double sums[kWaves];
  const int chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
  const Verdict v = a.verdicts[b];
  if (v.chosen || !reads_draft(a, v)) return;
  const double inv = inverse(temperature_of(a, b));
  const int64_t v0 = (int64_t)chunk * (BLOCKS * kBlock) + threadIdx.x * kItems;
  float x[BLOCKS][kItems], y[BLOCKS][kItems];
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) {
    load_items(target_row<T>(a, b, v.accepted), v0 + j * kBlock, a.V, x[j]);
    load_items(draft_row<T>(a, b, v.accepted), v0 + j * kBlock, a.V, y[j]);
  }
  const double zp = 1.0 / row_total<kWaves>(a, 0, b, sums), zq = 1.0 / row_total<kWaves>(a, 1, b, sums);
  double s = 0;
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) {
    double w[kItems];
    residual(v, x[j], y[j], inv, zp, zq, w);
#pragma unroll
    for (int i = 0; i < kItems; ++i) s += w[i];
  }
  s = block_sum<kWaves>(s, sums);
  if (threadIdx.x == 0) plane(a, 2, b)[chunk] = s;
}

// Running sum over the workgroup's threads: of those before this one.
template <int WAVES>
__device__ __forceinline__ double scan_before(double x, double* sums, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double incl = wave_scan_f64(x);
  __syncthreads();
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  double base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) base += sums[w];
    total += sums[w];
  }
  return base + (incl - x);
}

// The token: the chunk in which the running sum passes u times the sum, then the
// element. A workgroup per sequence; its first wave finds the chunk.
template <typename T, int BLOCKS>
__global__ __launch_bounds__(kThreads * BLOCKS) void verify_token_kernel(VerifyArgs a) {
  __shared__ double sums[kWaves * BLOCKS];
  __shared__ int pick, last, chosen_chunk, chosen_plane;
  __shared__ double zs[2], chosen_before, chosen_target;
  const int b = blockIdx.x, tid = threadIdx.x;
  const Verdict v = a.verdicts[b];
  if (v.chosen) return;
  const bool both = reads_draft(a, v);
  const double inv = inverse(temperature_of(a, b));
  if (tid < 64) {
    double s0 = 0, s1 = 0, s2 = 0;
    for (int c = tid; c < a.chunks; c += 64) {
      s0 += plane(a, 0, b)[c];
      s1 += plane(a, 1, b)[c];
      if (both) s2 += plane(a, 2, b)[c];
    }
    const double u = a.u[(int64_t)b * (a.K + 1) + a.K];
    s0 = wave_sum_f64(s0);
    s1 = wave_sum_f64(s1);
    s2 = wave_sum_f64(s2);
    // The weights: p, p without q_arg, or the residual of both rows.
    int which = 0;
    if (v.refused && (both ? s2 : s1 / s0) >= kAgree) which = both ? 2 : 1;
    const double target = u * (which == 0 ? s0 : which == 1 ? s1 : s2);
    // The first chunk whose running sum is above the target, else the last that weighs
    // anything, and the sum before it.
    int found = -1, heavy = 0;
    double run = 0, before = 0, before_heavy = 0;
    for (int c0 = 0; c0 < a.chunks && found < 0; c0 += 64) {
      const double s = c0 + tid < a.chunks ? plane(a, which, b)[c0 + tid] : 0;
      const double incl = run + wave_scan_f64(s);
      const unsigned long long above = __ballot(s > 0 && incl > target), some = __ballot(s > 0);
      auto before_of = [&](int lane) {
        const uint64_t x = __builtin_bit_cast(uint64_t, incl - s);
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(x), lane);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane);
        return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
      };
      if (above != 0) {
        const int l = __builtin_ctzll(above);
        found = c0 + l;
        before = before_of(l);
      } else if (some != 0) {
        const int l = 63 - __builtin_clzll(some);
        heavy = c0 + l;
        before_heavy = before_of(l);
      }
      run = last_lane(incl);
    }
    if (tid == 0) {
      chosen_chunk = found >= 0 ? found : heavy;
      chosen_before = found >= 0 ? before : before_heavy;
      chosen_plane = which;
      chosen_target = target;
      zs[0] = s0;
      zs[1] = s1;
      pick = 0x7fffffff;
      last = 0;
    }
  }
  __syncthreads();
  const int which = chosen_plane;
  const double target = chosen_target;
  const int64_t v0 = (int64_t)chosen_chunk * (BLOCKS * kBlock) + tid * kItems;
  float x[kItems];
  double w[kItems];
  load_items(target_row<T>(a, b, v.accepted), v0, a.V, x);
  if (which == 2) {
    float y[kItems];
    load_items(draft_row<T>(a, b, v.accepted), v0, a.V, y);
    residual(v, x, y, inv, 1.0 / zs[0], 1.0 / zs[1], w);
  } else {
    terms(x, v.p_top, inv, w);
    if (which == 1)
#pragma unroll
      for (int i = 0; i < kItems; ++i)
        if (v0 + i == v.q_arg) w[i] = 0;
  }
  double s = 0, all;
#pragma unroll
  for (int i = 0; i < kItems; ++i) s += w[i];
  double at = chosen_before + scan_before<kWaves * BLOCKS>(s, sums, all);
  int mine = 0x7fffffff, end = 0;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    at += w[i];
    if (w[i] > 0) {
      end = static_cast<int>(v0 + i);
      if (at > target && mine == 0x7fffffff) mine = end;
    }
  }
  if (mine != 0x7fffffff) atomicMin(&pick, mine);
  if (end > 0) atomicMax(&last, end);
  __syncthreads();
  if (tid == 0)
    a.tokens[(int64_t)b * (a.K + 1) + v.accepted] = pick != 0x7fffffff ? pick : last;
}

// Elements of a row per workgroup: 8192 where that still gives every CU one in the first
// pass, else 2048, for the latency of a few rows. The workspace's size does not depend on
// which drafts have logits, so all 2 K + 1 rows of a sequence count, whether they are read
// or not.
int blocks_per_chunk(int64_t B, int64_t K, int64_t V) {
  return B * (2 * K + 1) * lc_cdiv(V, 4 * kBlock) >= lc_cu_count() ? 4 : 1;
}
int64_t chunks_of(int64_t B, int64_t K, int64_t V) {
  return lc_cdiv(V, kBlock * blocks_per_chunk(B, K, V));
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

template <typename T>
int launch_verify(const VerifyArgs& a, hipStream_t st) {
  static const char* who = "lc_verify_draft_tokens";
  const unsigned rows = static_cast<unsigned>(a.B * (2 * a.K + 1));
  if (a.blocks == 4)
    verify_stats_kernel<T, 4><<<rows * a.chunks, kThreads, 0, st>>>(a);
  else
    verify_stats_kernel<T, 1><<<rows * a.chunks, kThreads, 0, st>>>(a);
  int rc = lc_check_launch(who);
  if (rc != LC_OK) return rc;
  verify_decide_kernel<T><<<a.B, kDecideThreads, 0, st>>>(a);
  rc = lc_check_launch(who);
  if (rc != LC_OK) return rc;
  if (a.blocks == 4)
    verify_sums_kernel<T, 4><<<a.B * a.chunks, kThreads, 0, st>>>(a);
  else
    verify_sums_kernel<T, 1><<<a.B * a.chunks, kThreads, 0, st>>>(a);
  rc = lc_check_launch(who);
  if (rc != LC_OK) return rc;
  if (a.y != nullptr) {
    if (a.blocks == 4)
      verify_residual_kernel<T, 4><<<a.B * a.chunks, kThreads, 0, st>>>(a);
    else
      verify_residual_kernel<T, 1><<<a.B * a.chunks, kThreads, 0, st>>>(a);
    rc = lc_check_launch(who);
    if (rc != LC_OK) return rc;
  }
  if (a.blocks == 4)
    verify_token_kernel<T, 4><<<a.B, 4 * kThreads, 0, st>>>(a);
  else
    verify_token_kernel<T, 1><<<a.B, kThreads, 0, st>>>(a);
  return lc_check_launch(who);
}

}  // namespace

extern "C" {

int64_t lc_verify_draft_tokens_workspace_bytes(int64_t B, int64_t drafts, int64_t vocab) {
  if (B < 0 || drafts < 0 || vocab <= 0) return -1;
  const int64_t chunks = chunks_of(B, drafts, vocab);
  return align256(B * (2 * drafts + 1) * chunks * sizeof(Stat)) + align256(B * sizeof(Verdict)) +
         B * chunks * 3 * 8;
}

int lc_verify_draft_tokens(const void* logits, int64_t l_sb, int64_t l_si, const void* draft_logits,
                           int64_t d_sb, int64_t d_si, const int64_t* draft_tokens,
                           const float* uniforms, const int32_t* draft_lens,
                           const float* temperatures, double temperature, int64_t B, int64_t drafts,
                           int64_t vocab, int64_t* tokens, int32_t* accepted, void* workspace,
                           int64_t workspace_bytes, int dtype, void* stream) {
  static const char* who = "lc_verify_draft_tokens";
  LC_REQUIRE(B >= 0 && drafts >= 0 && drafts <= kMaxDrafts, "%s: %lld sequences of %lld drafts (below 256)",
             who, (long long)B, (long long)drafts);
  // (a launch has fewer than 2^32 threads)
  LC_REQUIRE(B < (1LL << 32) / kDecideThreads, "%s: %lld sequences (below 2^22)", who, (long long)B);
  LC_REQUIRE(vocab > 0 && vocab < (1LL << 31) - 4 * kBlock, "%s: vocabulary of %lld", who,
             (long long)vocab);
  LC_REQUIRE(dtype == LC_DTYPE_F32 || dtype == LC_DTYPE_F16 || dtype == LC_DTYPE_BF16,
             "%s: unknown dtype %d", who, dtype);
  if (B == 0) return LC_OK;
  LC_REQUIRE(logits && uniforms && tokens && accepted && workspace && (draft_tokens || drafts == 0),
             "%s: null pointer", who);
  LC_REQUIRE(l_sb >= 0 && l_si >= 0 && d_sb >= 0 && d_si >= 0, "%s: negative stride", who);
  const int64_t chunks = chunks_of(B, drafts, vocab);
  LC_REQUIRE(B < (1LL << 24) / ((2 * drafts + 1) * chunks), "%s: too many rows (%lld of %lld)", who,
             (long long)(B * (2 * drafts + 1)), (long long)vocab);
  const int64_t need = lc_verify_draft_tokens_workspace_bytes(B, drafts, vocab);
  if (workspace_bytes < need)
    return lc_fail(LC_EWORKSPACE, "%s: workspace %lld < %lld bytes", who,
                   (long long)workspace_bytes, (long long)need);
  LC_REQUIRE(lc_aligned(workspace, 256), "%s: workspace not 256-byte aligned", who);

  VerifyArgs a{};
  a.x = logits;
  a.x_sb = l_sb;
  a.x_si = l_si;
  a.y = drafts > 0 ? draft_logits : nullptr;
  a.y_sb = d_sb;
  a.y_si = d_si;
  a.drafts = draft_tokens;
  a.u = uniforms;
  a.lens = draft_lens;
  a.temps = temperatures;
  a.temperature = temperature;
  a.tokens = tokens;
  a.accepted = accepted;
  a.B = static_cast<int>(B);
  a.K = static_cast<int>(drafts);
  a.V = static_cast<int>(vocab);
  a.chunks = static_cast<int>(chunks);
  a.blocks = blocks_per_chunk(B, drafts, vocab);
  char* at = static_cast<char*>(workspace);
  a.stats = reinterpret_cast<Stat*>(at);
  at += align256(B * (2 * drafts + 1) * chunks * sizeof(Stat));
  a.verdicts = reinterpret_cast<Verdict*>(at);
  at += align256(B * sizeof(Verdict));
  a.sums = reinterpret_cast<double*>(at);
  hipStream_t st = lc_stream(stream);
  switch (dtype) {
    case LC_DTYPE_F32:
      return launch_verify<float>(a, st);
    case LC_DTYPE_BF16:
      return launch_verify<bf16_t>(a, st);
    default:
      return launch_verify<f16_t>(a, st);
  }
}

}  // extern "C"
