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
// (added in 64 bits from a wave's on) do: off by 1e-7, it falls otherwise in as
// many of ten million.
#include <math.h>

#include <type_traits>

#include "lc_common.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kItems = 8;                    // elements of a chunk per thread
constexpr int kChunk = kThreads * kItems;    // elements of a row per workgroup
// A residual max(p - q, 0) that sums to less is rounding: p and q agree.
constexpr double kAgree = 2.3283064365386963e-10;  // 2^-32

struct Stat {  // of a chunk of a row
  float top;   // its largest logit (NaN: it holds one)
  int arg;     // where it first is
  double sum;  // of exp((x - top) / temperature)
};

struct Verdict {      // of a sequence
  int accepted;       // drafts that stand
  int refused;        // whether one was refused
  int p_arg, q_arg;   // the row's mass is all here (-1: it is spread)
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
  double* sums;       // [B, chunks, 3]: of p's terms, q's, and the residual
  int B, K, V, chunks;
};

__device__ __forceinline__ double temperature_of(const VerifyArgs& a, int b) {
  return a.temps != nullptr ? static_cast<double>(a.temps[b]) : a.temperature;
}
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) {
  if (a.lens == nullptr) return a.K;
  const int n = a.lens[b];
  return n < 0 ? 0 : n > a.K ? a.K : n;
}

template <typename T>
__device__ __forceinline__ const T* target_row(const VerifyArgs& a, int b, int i) {
  return static_cast<const T*>(a.x) + (int64_t)b * a.x_sb + (int64_t)i * a.x_si;
}
template <typename T>
__device__ __forceinline__ const T* draft_row(const VerifyArgs& a, int b, int i) {
  return static_cast<const T*>(a.y) + (int64_t)b * a.y_sb + (int64_t)i * a.y_si;
}

// This thread's kItems consecutive elements of a row from v0 on; past the end: -inf.
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

__device__ __forceinline__ double wave_sum_f64(double x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// Largest value and first place of it; NaN is the largest.
struct Top {
  float top;
  int arg;
};
__device__ __forceinline__ bool before(float x, int i, float y, int j) {
  const bool nx = x != x, ny = y != y;
  if (nx != ny) return nx;
  if (!nx && x != y) return x > y;
  return i < j;
}
__device__ __forceinline__ Top first_of(Top a, Top b) {
  return before(b.top, b.arg, a.top, a.arg) ? b : a;
}

// Chunk statistics: one workgroup per (chunk, row); rows are a sequence's K + 1 target
// rows, then its K draft rows. Rows past the sequence's drafts are not read.
template <typename T>
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
  const int64_t v0 = (int64_t)chunk * kChunk + tid * kItems;
  float v[kItems];
  load_items(row, v0, a.V, v);
  Top t{-INFINITY, 0x7fffffff};
#pragma unroll
  for (int e = 0; e < kItems; ++e)
    if (v0 + e < a.V) t = first_of(t, Top{v[e], static_cast<int>(v0 + e)});
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1)
    t = first_of(t, Top{__shfl_xor(t.top, o, 64), __shfl_xor(t.arg, o, 64)});
  __shared__ Top tops[kWaves];
  __shared__ double sums[kWaves];
  if (lane == 0) tops[wave] = t;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) t = first_of(t, tops[w]);
  const double temp = temperature_of(a, b);
  // (kept finite and above 0: 0 and -inf stay what they are)
  const float c = static_cast<float>(fmin(fmax(1.4426950408889634 / temp, 1e-37), 1e37));
  float part = 0.f;
#pragma unroll
  for (int e = 0; e < kItems; ++e) part += lc_exp2((v[e] - t.top) * c);
  const double s = wave_sum_f64(part);
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  if (tid == 0) {
    double all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all += sums[w];
    a.stats[((int64_t)b * rows + r) * a.chunks + chunk] = Stat{t.top, t.arg, all};
  }
}

// A row's largest logit, where it is, and its sum, from its chunks (one wave).
struct RowSum {
  float top;
  int arg;
  double sum;
  bool peaked;  // all mass at arg
};
__device__ __forceinline__ RowSum row_sum(const VerifyArgs& a, int b, int r, double temp) {
  const Stat* s = a.stats + ((int64_t)b * (2 * a.K + 1) + r) * a.chunks;
  const int lane = threadIdx.x & 63;
  Top t{-INFINITY, 0x7fffffff};
  for (int c = lane; c < a.chunks; c += 64) t = first_of(t, Top{s[c].top, s[c].arg});
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1)
    t = first_of(t, Top{__shfl_xor(t.top, o, 64), __shfl_xor(t.arg, o, 64)});
  const bool peaked = !(temp > 0 && temp < INFINITY) || !(fabsf(t.top) < INFINITY);
  double sum = 0;
  if (!peaked)
    for (int c = lane; c < a.chunks; c += 64)
      if (s[c].top != -INFINITY) sum += s[c].sum * exp((static_cast<double>(s[c].top) - t.top) / temp);
  return RowSum{t.top, t.arg, wave_sum_f64(sum), peaked};
}

template <typename T>
__device__ __forceinline__ double chance(const T* row, int64_t d, int V, const RowSum& s,
                                         double temp) {
  if (d < 0 || d >= V) return 0;
  if (s.peaked) return d == s.arg ? 1 : 0;
  return exp((static_cast<double>(lc_to_f32(row[d])) - s.top) / temp) / s.sum;
}

// One wave per sequence: which drafts stand.
template <typename T>
__global__ __launch_bounds__(64) void verify_decide_kernel(VerifyArgs a) {
  const int b = blockIdx.x;
  const int n = drafts_of(a, b);
  const double temp = temperature_of(a, b);
  Verdict v{};
  v.q_arg = -1;
  RowSum p;
  for (int i = 0;; ++i) {
    p = row_sum(a, b, i, temp);
    v.accepted = i;
    if (i == n) break;
    const int64_t d = a.drafts[(int64_t)b * a.K + i];
    const double pd = chance(target_row<T>(a, b, i), d, a.V, p, temp);
    double qd = 1;
    RowSum q{0.f, -1, 1, true};
    if (a.y != nullptr) {
      q = row_sum(a, b, a.K + 1 + i, temp);
      qd = chance(draft_row<T>(a, b, i), d, a.V, q, temp);
    }
    if (!(a.u[(int64_t)b * (a.K + 1) + i] * qd < pd)) {
      v.refused = 1;
      v.q_top = q.top;
      v.q_arg = a.y == nullptr ? (d >= 0 && d < a.V ? static_cast<int>(d) : -1)
                               : q.peaked ? q.arg : -1;
      break;
    }
  }
  v.p_top = p.top;
  v.p_arg = p.peaked ? p.arg : -1;
  for (int i = threadIdx.x; i <= a.K; i += 64)
    a.tokens[(int64_t)b * (a.K + 1) + i] = i < v.accepted ? a.drafts[(int64_t)b * a.K + i] : -1;
  if (threadIdx.x == 0) {
    a.accepted[b] = v.accepted;
    a.verdicts[b] = v;
  }
}

// The row's terms of this thread's elements, not divided by their sum.
__device__ __forceinline__ void terms(const float (&x)[kItems], int64_t v0, int V, float top,
                                      int arg, double temp, double (&e)[kItems]) {
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int64_t v = v0 + i;
    e[i] = v >= V ? 0
           : arg >= 0 ? (v == arg ? 1 : 0)
                      : exp((static_cast<double>(x[i]) - top) / temp);
  }
}

__device__ __forceinline__ double block_sum(double x, double* sums) {
  x = wave_sum_f64(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
  __syncthreads();
  double all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += sums[w];
  return all;
}

// A refused draft's other row is spread over the vocabulary: its terms are needed.
__device__ __forceinline__ bool reads_draft(const VerifyArgs& a, const Verdict& v) {
  return v.refused && v.q_arg < 0 && a.y != nullptr;
}

// 64-bit sums of a chunk's terms.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
  __shared__ double sums[kWaves];
  const int chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
  const Verdict v = a.verdicts[b];
  const double temp = temperature_of(a, b);
  const int64_t v0 = (int64_t)chunk * kChunk + threadIdx.x * kItems;
  float x[kItems];
  double e[kItems], s = 0;
  load_items(target_row<T>(a, b, v.accepted), v0, a.V, x);
  terms(x, v0, a.V, v.p_top, v.p_arg, temp, e);
#pragma unroll
  for (int i = 0; i < kItems; ++i) s += e[i];
  const double sp = block_sum(s, sums);
  double sq = 0;
  if (reads_draft(a, v)) {
    load_items(draft_row<T>(a, b, v.accepted), v0, a.V, x);
    terms(x, v0, a.V, v.q_top, v.q_arg, temp, e);
    s = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) s += e[i];
    sq = block_sum(s, sums);
  }
  if (threadIdx.x == 0) {
    double* to = a.sums + ((int64_t)b * a.chunks + chunk) * 3;
    to[0] = sp;
    to[1] = sq;
  }
}

__device__ __forceinline__ double column_sum(const VerifyArgs& a, int b, int which, double* sums) {
  double s = 0;
  for (int c = threadIdx.x; c < a.chunks; c += kThreads)
    s += a.sums[((int64_t)b * a.chunks + c) * 3 + which];
  return block_sum(s, sums);
}

// What this thread's elements weigh after a refused draft.
template <typename T>
__device__ __forceinline__ void residual(const VerifyArgs& a, const Verdict& v, int b, int64_t v0,
                                         double temp, double zp, double zq, double (&w)[kItems]) {
  float x[kItems];
  load_items(target_row<T>(a, b, v.accepted), v0, a.V, x);
  terms(x, v0, a.V, v.p_top, v.p_arg, temp, w);
  double e[kItems];
  if (reads_draft(a, v)) {
    load_items(draft_row<T>(a, b, v.accepted), v0, a.V, x);
    terms(x, v0, a.V, v.q_top, v.q_arg, temp, e);
  } else {
#pragma unroll
    for (int i = 0; i < kItems; ++i) e[i] = v0 + i == v.q_arg ? 1 : 0;
    zq = 1;
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const double d = w[i] / zp - e[i] / zq;
    w[i] = d > 0 ? d : 0;
  }
}

// Sums of a chunk's residual.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_residual_kernel(VerifyArgs a) {
  __shared__ double sums[kWaves];
  const int chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
  const Verdict v = a.verdicts[b];
  if (!v.refused) return;
  const double zp = column_sum(a, b, 0, sums), zq = column_sum(a, b, 1, sums);
  double w[kItems], s = 0;
  residual<T>(a, v, b, (int64_t)chunk * kChunk + threadIdx.x * kItems, temperature_of(a, b), zp, zq, w);
#pragma unroll
  for (int i = 0; i < kItems; ++i) s += w[i];
  s = block_sum(s, sums);
  if (threadIdx.x == 0) a.sums[((int64_t)b * a.chunks + chunk) * 3 + 2] = s;
}

// Running sum over the workgroup's threads: of those before this one.
__device__ __forceinline__ double scan_before(double x, double* sums, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double incl = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  double base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) base += sums[w];
    total += sums[w];
  }
  return base + (incl - x);
}

// The token: the chunk in which the running sum passes u times the sum, then the
// element.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_token_kernel(VerifyArgs a) {
  __shared__ double sums[kWaves];
  __shared__ int pick, last;
  __shared__ double pick_base;
  const int b = blockIdx.x, tid = threadIdx.x;
  const Verdict v = a.verdicts[b];
  const double temp = temperature_of(a, b);
  const double u = a.u[(int64_t)b * (a.K + 1) + a.K];
  double zp = 0, zq = 0, total = 0;
  int which = 0;
  if (v.refused) {
    zp = column_sum(a, b, 0, sums);
    zq = column_sum(a, b, 1, sums);
    total = column_sum(a, b, 2, sums);
    if (total >= kAgree) which = 2;
  }
  if (which == 0) total = column_sum(a, b, 0, sums);
  const double target = u * total;
  // The first chunk whose running sum is above the target (else the last that weighs
  // anything).
  if (tid == 0) {
    pick = 0x7fffffff;
    last = 0;
  }
  __syncthreads();
  double run = 0;
  for (int c0 = 0; c0 < a.chunks; c0 += kThreads) {
    const int c = c0 + tid;
    const double s = c < a.chunks ? a.sums[((int64_t)b * a.chunks + c) * 3 + which] : 0;
    double all;
    const double base = run + scan_before(s, sums, all);
    if (s > 0) {
      atomicMax(&last, c);
      if (base + s > target) atomicMin(&pick, c);
    }
    run += all;
  }
  __syncthreads();
  const int chunk = pick < a.chunks ? pick : last;
  __syncthreads();
  // The sum before that chunk, in the same order.
  run = 0;
  for (int c0 = 0; c0 <= chunk; c0 += kThreads) {
    const int c = c0 + tid;
    const double s = c < a.chunks ? a.sums[((int64_t)b * a.chunks + c) * 3 + which] : 0;
    double all;
    const double base = run + scan_before(s, sums, all);
    if (c == chunk) pick_base = base;
    run += all;
  }
  if (tid == 0) {
    pick = 0x7fffffff;
    last = 0;
  }
  __syncthreads();
  const int64_t v0 = (int64_t)chunk * kChunk + tid * kItems;
  double w[kItems];
  if (which == 2) {
    residual<T>(a, v, b, v0, temp, zp, zq, w);
  } else {
    float x[kItems];
    load_items(target_row<T>(a, b, v.accepted), v0, a.V, x);
    terms(x, v0, a.V, v.p_top, v.p_arg, temp, w);
  }
  double s = 0, all;
#pragma unroll
  for (int i = 0; i < kItems; ++i) s += w[i];
  run = pick_base + scan_before(s, sums, all);
  int mine = 0x7fffffff, end = 0;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    run += w[i];
    if (w[i] > 0) {
      end = static_cast<int>(v0 + i);
      if (run > target && mine == 0x7fffffff) mine = end;
    }
  }
  if (mine != 0x7fffffff) atomicMin(&pick, mine);
  if (end > 0) atomicMax(&last, end);
  __syncthreads();
  if (tid == 0)
    a.tokens[(int64_t)b * (a.K + 1) + v.accepted] = pick != 0x7fffffff ? pick : last;
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

template <typename T>
int launch_verify(const VerifyArgs& a, hipStream_t st) {
  static const char* who = "lc_verify_draft_tokens";
  const unsigned rows = static_cast<unsigned>(a.B * (2 * a.K + 1));
  verify_stats_kernel<T><<<rows * a.chunks, kThreads, 0, st>>>(a);
  int rc = lc_check_launch(who);
  if (rc != LC_OK) return rc;
  verify_decide_kernel<T><<<a.B, 64, 0, st>>>(a);
  rc = lc_check_launch(who);
  if (rc != LC_OK) return rc;
  verify_sums_kernel<T><<<a.B * a.chunks, kThreads, 0, st>>>(a);
  rc = lc_check_launch(who);
  if (rc != LC_OK) return rc;
  verify_residual_kernel<T><<<a.B * a.chunks, kThreads, 0, st>>>(a);
  rc = lc_check_launch(who);
  if (rc != LC_OK) return rc;
  verify_token_kernel<T><<<a.B, kThreads, 0, st>>>(a);
  return lc_check_launch(who);
}

}  // namespace

extern "C" {

int64_t lc_verify_draft_tokens_workspace_bytes(int64_t B, int64_t drafts, int64_t vocab) {
  if (B < 0 || drafts < 0 || vocab <= 0) return -1;
  const int64_t chunks = lc_cdiv(vocab, kChunk);
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
  LC_REQUIRE(B >= 0 && drafts >= 0 && drafts < 256, "%s: %lld sequences of %lld drafts (below 256)",
             who, (long long)B, (long long)drafts);
  LC_REQUIRE(vocab > 0 && vocab < (1LL << 31) - kChunk, "%s: vocabulary of %lld", who,
             (long long)vocab);
  LC_REQUIRE(dtype == LC_DTYPE_F32 || dtype == LC_DTYPE_F16 || dtype == LC_DTYPE_BF16,
             "%s: unknown dtype %d", who, dtype);
  if (B == 0) return LC_OK;
  LC_REQUIRE(logits && uniforms && tokens && accepted && workspace && (draft_tokens || drafts == 0),
             "%s: null pointer", who);
  LC_REQUIRE(l_sb >= 0 && l_si >= 0 && d_sb >= 0 && d_si >= 0, "%s: negative stride", who);
  const int64_t chunks = lc_cdiv(vocab, kChunk);
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
