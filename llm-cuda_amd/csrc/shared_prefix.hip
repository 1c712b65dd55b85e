// One-token GQA attention of a batch whose groups of sequences share a prefix,
// over the paged KV cache.
//
// N groups of W sequences: sequence b = n W + w attends to the tokens of group
// n's prefix (pages prefix_table[n]) and then to its own (pages block_table[b]).
// Softmax over a union of disjoint token ranges is a weighted mean of the ranges'
// own softmaxes:
//   out = sum_i 2^(lse_i - M) o_i / sum_i 2^(lse_i - M),  M = max_i lse_i
// (lse in log2 units), so the prefix of a group is computed once for all of its
// rows, cut into prefix_splits ranges, beside own_splits ranges of every
// sequence's own tokens; each range leaves its normalised fp32 output and lse in
// the workspace, and a merge launch joins them (or, in small calls, the workgroup
// that finishes last).
//
// Bound: reading K and V once (4 groups of 8 x (4096 + 128) tokens, 8B heads: 84 MB in
// 19.8 us + merge 3.9; 64 x (8192 + 625): 200 MB in 48.8 + 5.9), until a prefix has some
// 130 rows per kv head, from where it is the matrix rate (256 x (8192 + 200): 77 to 80 +
// 8.2 us, 400 TFLOP/s of QK and one PV in all).
#include <math.h>

#include "lc_common.h"
#include "paged_tiles.h"

namespace {

using namespace lc_attn;

struct SharedArgs {
  const void* q;
  int64_t q_sb, q_sh;
  const void* kp;
  const void* vp;
  int64_t s_page, s_head, s_tok;
  const int32_t* ptab;  // [N, p_pages]
  int64_t ptab_stride;
  const int32_t* plens;  // [N]
  const int32_t* btab;   // [B, s_pages]
  int64_t btab_stride;
  const int32_t* slens;  // [B]
  float* part_o;         // [B*Hq, p_splits + s_splits, D]
  float* part_lse;       // [B*Hq, p_splits + s_splits], log2 units
  int B, W, Hq, Hkv, G, D, P, p_shift, num_pages, p_pages, s_pages, p_splits, s_splits;
  float scale_log2;
  // Not null: the last workgroup of a group and kv head to finish (its ticket on
  // counters[n * Hkv + kvh], zero at entry and left zero) writes their output.
  int* counters;
  int expected;  // workgroups of a group and kv head
  void* out;
  int64_t o_sb, o_sh;
  float* lse;
};

// Tokens of a range are a multiple of this.
constexpr int kSharedStep = 64;

// x as an fp32 value: a product that is converted to f16 next may otherwise be taken
// by one instruction that rounds once, here and not there.
__device__ __forceinline__ float rounded(float x) {
  __asm__("" : "+v"(x));
  return x;
}

__device__ __forceinline__ int clamp_len(int len, int pages, int P) {
  const int cap = pages * P;
  return len < 0 ? 0 : len > cap ? cap : len;
}

// Tokens per range of `len` tokens cut into at most `splits` equal ranges.
__device__ __forceinline__ int range_tokens(int len, int splits) {
  const int each = (len + splits - 1) / splits;
  return (each + kSharedStep - 1) / kSharedStep * kSharedStep;
}

__device__ __forceinline__ int range_count(int len, int splits) {
  if (len <= 0 || splits <= 0) return 0;
  const int each = range_tokens(len, splits);
  return (len + each - 1) / each;
}

// Element offset of token tok of a table row and kv head; -1 where its page entry
// is invalid. tok is within the row's capacity.
__device__ __forceinline__ int64_t token_offset(const SharedArgs& a, const int32_t* row, int kvh,
                                                int tok) {
  const int page = a.p_shift >= 0 ? tok >> a.p_shift : tok / a.P;
  const int slot = tok - page * a.P;
  const int phys = row[page];
  if (static_cast<unsigned>(phys) >= static_cast<unsigned>(a.num_pages)) return -1;
  return (int64_t)phys * a.s_page + (int64_t)kvh * a.s_head + (int64_t)slot * a.s_tok;
}

// Generic kernel: one wave per (sequence, query head, range), lanes across
// head_dim, one token at a time. Any dtype, head_dim <= 256 and strides.
template <typename T>
__global__ __launch_bounds__(64) void shared_generic_kernel(SharedArgs a) {
  const int lane = threadIdx.x;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const bool prefix = split < a.p_splits;
  const int n = b / a.W;
  const int len = prefix ? clamp_len(a.plens[n], a.p_pages, a.P)
                         : clamp_len(a.slens[b], a.s_pages, a.P);
  const int splits = prefix ? a.p_splits : a.s_splits;
  const int each = range_tokens(len, splits);
  const int t_begin = (prefix ? split : split - a.p_splits) * each;
  if (t_begin >= len) return;
  const int t_end = min(len, t_begin + each);
  const int32_t* row = prefix ? a.ptab + (int64_t)n * a.ptab_stride
                              : a.btab + (int64_t)b * a.btab_stride;
  const int kvh = h / a.G;
  const T* kp = static_cast<const T*>(a.kp);
  const T* vp = static_cast<const T*>(a.vp);
  const T* qh = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh;

  float qv[4], acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    qv[i] = d < a.D ? lc_to_f32(qh[d]) : 0.f;
    acc[i] = 0.f;
  }
  float m_run = -INFINITY, l_run = 0.f;
  for (int t = t_begin; t < t_end; ++t) {
    const int64_t off = token_offset(a, row, kvh, t);
    if (off < 0) continue;  // uniform across the wave
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < a.D) dot = fmaf(qv[i], lc_to_f32(kp[off + d]), dot);
    }
    const float s = lc_wave_sum(dot) * a.scale_log2;
    if (s == -INFINITY) continue;
    const float m_new = fmaxf(m_run, s);
    const float alpha = lc_exp2(m_run - m_new);
    const float p = lc_exp2(s - m_new);
    l_run = l_run * alpha + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      const float vv = d < a.D ? lc_to_f32(vp[off + d]) : 0.f;
      acc[i] = fmaf(p, vv, acc[i] * alpha);
    }
    m_run = m_new;
  }
  const int64_t pidx = ((int64_t)b * a.Hq + h) * (a.p_splits + a.s_splits) + split;
  const float inv_l = l_run > 0.f ? 1.0f / l_run : l_run;  // (NaN stays NaN)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < a.D) a.part_o[pidx * a.D + d] = acc[i] * inv_l;
  }
  if (lane == 0) a.part_lse[pidx] = l_run == 0.f ? -INFINITY : m_run + lc_log2(l_run);
}

// ---------------------------------------------------------------------------
// MFMA kernel (bf16/f16, head_dim a multiple of 8 up to 128, pages of a power of
// two from 8 up): one workgroup of 4 waves per (token range, 32 WR rows). A prefix's
// rows are the W G query heads of its sequences that share a kv head, row r = w G +
// g; a sequence's own rows are its G heads.
//   S^T[tok x 32 rows] = K Q^T, O^T[d x 32 rows] += V^T P^T   (32x32x16 MFMA)
// so a byte of K and V is read once for all rows of the workgroup. Up to 32 rows
// the waves take token steps of their own (paged_stream). With more, tiles
// of 64 tokens go through LDS (double-buffered, by DMA), which the waves share: with
// 128 rows each has 32 rows and all tokens, with 64 rows 32 tokens, and the token
// halves' softmax states are joined through LDS at the end.
// Tokens are named by a table, so every lane finds the address of its own 16-byte
// chunk of a DMA; lanes whose token is past the range, whose page entry is invalid
// or whose chunk is past head_dim read zeros instead, and their scores are masked.
// The matrix instructions take the weights P in the data type, so each goes there as
// two values of it, the weight cut off and what that left (to 2^-15 of a bf16 weight,
// 2^-21 of an f16 one, down to 2^-25); their sum stays in fp32. A rounded weight alone
// would leave an error as large as the output's own rounding, for values without a
// common mean average the output down as much as the errors (8448 bf16 tokens: 2.3e-3
// rms of the output, 1.66e-3 with both, which is the output's rounding). The second
// value is free where K and V are streamed (4 groups of 8 x 4224, a call in a graph:
// 22.2 -> 22.7 us); where a prefix has many rows, PV is twice the matrix work: 64 x
// (8192 + 625) 52 -> 56 us, 256 x (8192 + 200) 75 -> 86.
// ---------------------------------------------------------------------------

// A partial output or logsumexp. Where another workgroup of the same launch reads it
// (on another XCD, maybe), it is written through to memory by relaxed stores of
// device scope, and read by such loads: no cache has to be written back or
// invalidated (fences did that for every workgroup: 20 us a launch instead of 12.8).
__device__ __forceinline__ void put4(const SharedArgs& a, float* to, f32x4_t x) {
  if (a.counters != nullptr) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    uint64_t* p = reinterpret_cast<uint64_t*>(to);
    __hip_atomic_store(p, __builtin_bit_cast(uint64_t, f32x2{x[0], x[1]}), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(p + 1, __builtin_bit_cast(uint64_t, f32x2{x[2], x[3]}), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  } else {
    *reinterpret_cast<f32x4_t*>(to) = x;
  }
}
__device__ __forceinline__ void put(const SharedArgs& a, float* to, float x) {
  if (a.counters != nullptr)
    __hip_atomic_store(to, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else
    *to = x;
}
__device__ __forceinline__ float got(const float* from) {
  return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4_t got4(const float* from) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const uint64_t* p = reinterpret_cast<const uint64_t*>(from);
  const f32x2 lo = __builtin_bit_cast(
      f32x2, __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  const f32x2 hi = __builtin_bit_cast(
      f32x2, __hip_atomic_load(p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  return f32x4_t{lo[0], lo[1], hi[0], hi[1]};
}

struct RangeItem {
  static constexpr bool kCausal = false;
  const int32_t* table;  // the token range's table row
  int b0, row0, rows;    // row r is sequence b0 + r / G, head r % G of the kv head
  int kvh, t_begin, t_end, slot;

  template <typename T>
  __device__ __forceinline__ const T* query(const SharedArgs& a, int r) const {
    return static_cast<const T*>(a.q) + (int64_t)(b0 + r / a.G) * a.q_sb +
           (int64_t)(kvh * a.G + r % a.G) * a.q_sh;
  }
  // (the row's partial output and logsumexp)
  __device__ __forceinline__ int64_t row(const SharedArgs& a, int r) const {
    return ((int64_t)(b0 + r / a.G) * a.Hq + kvh * a.G + r % a.G) * (a.p_splits + a.s_splits) + slot;
  }
  __device__ __forceinline__ void store4(const SharedArgs& a, int64_t row, int d, f32x4_t x) const {
    put4(a, a.part_o + row * a.D + d, x);
  }
  __device__ __forceinline__ void store_lse(const SharedArgs& a, int64_t row, float x) const {
    put(a, a.part_lse + row, x);
  }
};

// The merge in the same launch, for few rows and ranges: every workgroup of group n
// and kv head kvh takes a ticket after its partials, and the one with the last joins
// all ranges of their rows, a thread per 4 columns. Which workgroup that is changes
// nothing in the sums, which equal shared_merge_kernel's bit for bit.
//
// The GPU takes longer so (4 beams of 1000 tokens: 13.1 us for 11.1 in two launches; 20
// with fences, which write the whole L2 back, in place of write-through partials), but
// the host, which such a call waits for, loses a launch. Eager calls, us, joined / in
// two launches (in brackets on the GPU):
//   8B heads, 4 x 4 beams, K and V 12 MB 15.1 / 17.1 (13.2 / 11.2), 21 MB 15.9 / 16.8,
//     29 MB 16.7 / 16.8, 37 MB 18.5 / 16.8, 70 MB 21.8 / 20.6
//   16/8 heads of 64, 8 x 4 beams, 6 to 53 MB 15.0 / 16.9
// The joining workgroup takes two rounds for 16 rows of 128 there; four rounds (8B, 4 x
// 8 beams) are no gain, 8 MB 16.7 / 17.1 and 17 MB 19.5 / 17.0, and eight (70B, 2 x 8
// beams) lose, 5.5 MB 20.9 / 17.0.
constexpr int kJoinRanges = 16;             // most ranges per row
constexpr int64_t kJoinBytes = 96 << 10;    // most partials of a group and kv head
constexpr int64_t kJoinRead = 16 << 20;     // most bytes of K and V, by the tables' widths
constexpr int64_t kJoinOutputs = 2048;      // most outputs of a group and kv head
constexpr int kJoinCounters = 4096;

template <typename T>
__device__ __forceinline__ void join_last(const SharedArgs& a, int n, int kvh) {
  __shared__ int last;
  // (every wave's stores have reached memory before the ticket is taken)
  __builtin_amdgcn_s_waitcnt(kWaitVm0Lgkm0);
  lc_compiler_fence();
  __syncthreads();
  if (threadIdx.x == 0) {
    int* c = a.counters + n * a.Hkv + kvh;
    const int t = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = t == a.expected - 1;
    if (last) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  lc_compiler_fence();
  const int chunks = a.D / 4, total = a.W * a.G * chunks, stride = a.p_splits + a.s_splits;
  const int n_p = range_count(clamp_len(a.plens[n], a.p_pages, a.P), a.p_splits);
  for (int i = threadIdx.x; i < total; i += 256) {
    const int r = i / chunks, d = (i - r * chunks) * 4;
    const int b = n * a.W + r / a.G, h = kvh * a.G + r % a.G;
    const int n_all = n_p + range_count(clamp_len(a.slens[b], a.s_pages, a.P), a.s_splits);
    const int64_t base = ((int64_t)b * a.Hq + h) * stride;
    float w[kJoinRanges], m = -INFINITY;
    f32x4_t o[kJoinRanges];
#pragma unroll
    for (int j = 0; j < kJoinRanges; ++j) {
      w[j] = -INFINITY;
      if (j < n_all) {
        const int64_t at = base + (j < n_p ? j : a.p_splits + (j - n_p));
        w[j] = got(a.part_lse + at);
        o[j] = got4(a.part_o + at * a.D + d);
      }
    }
#pragma unroll
    for (int j = 0; j < kJoinRanges; ++j) m = fmaxf(m, w[j]);
    const float m_use = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kJoinRanges; ++j) {
      if (j < n_all) {
        const float f = lc_exp2(w[j] - m_use);  // (NaN passes)
        sum += f;
        if (f != 0.f) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, o[j][e], acc[e]);
        }
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    T* to = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = lc_from_f32<T>(rounded(acc[e] * inv));
    if (a.lse != nullptr && d == 0)
      a.lse[(int64_t)b * a.Hq + h] = sum == 0.f ? -INFINITY : (m_use + lc_log2(sum)) * kLn2;
  }
}

// Work of block `id` below p_blocks: a range of a prefix and `tile_rows` of its
// group's rows. A range's row tiles read the same K and V: they get block ids 8
// apart, which run on one XCD, and find it in its L2. False: a block past the last
// range. The range may be empty.
__device__ __forceinline__ bool prefix_item(const SharedArgs& a, int id, int row_tiles,
                                            int tile_rows, RangeItem& it) {
  const int run = id / (8 * row_tiles), rest = id - run * 8 * row_tiles;
  const int pair = run * 8 + (rest & 7), tile = rest >> 3;
  const int units = (a.B / a.W) * a.Hkv;
  const int split = pair / units, u = pair - split * units;
  if (split >= a.p_splits) return false;
  const int n = u / a.Hkv;
  const int len = clamp_len(a.plens[n], a.p_pages, a.P);
  const int each = range_tokens(len, a.p_splits);
  it.t_begin = split * each;
  it.t_end = min(len, it.t_begin + each);
  it.table = a.ptab + (int64_t)n * a.ptab_stride;
  it.kvh = u - n * a.Hkv;
  it.b0 = n * a.W;
  it.rows = a.W * a.G;
  it.row0 = tile * tile_rows;
  it.slot = split;
  return true;
}

// Item i of the sequences' own ranges: all kv heads of a sequence follow one another
// (one table row, and neighbours in a page). An item without tokens is left empty.
__device__ __forceinline__ void own_item(const SharedArgs& a, int i, int head_groups,
                                         RangeItem& it) {
  const int units = a.B * a.Hkv * head_groups;
  const int split = i / units, u = i - split * units;
  const int hg = u % head_groups, bk = u / head_groups;
  const int b = bk / a.Hkv;
  const bool item = split < a.s_splits;
  const int len = item ? clamp_len(a.slens[b], a.s_pages, a.P) : 0;
  const int each = range_tokens(len, a.s_splits);
  it.t_begin = split * each;
  it.t_end = min(len, it.t_begin + each);
  it.table = a.btab + (int64_t)(item ? b : 0) * a.btab_stride;
  it.kvh = item ? bk - b * a.Hkv : 0;
  it.b0 = item ? b : 0;
  it.rows = a.G;
  it.row0 = hg * 32;
  it.slot = a.p_splits + split;
}

// Workgroups below p_blocks take the prefixes' ranges, the others the sequences'
// own, 4 / own_waves of them each.
template <typename T, int DPAD, int WR>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void
shared_mfma_kernel(SharedArgs a, int p_blocks, int row_tiles, int head_groups, int own_waves) {
  constexpr int TILE_B = kTile * DPAD * (int)sizeof(T);
  // (separate arrays: the compiler tracks a DMA by the array that it writes)
  __shared__ __align__(16) char lds_k0[TILE_B];
  __shared__ __align__(16) char lds_k1[TILE_B];
  __shared__ __align__(16) char lds_v0[TILE_B];
  __shared__ __align__(16) char lds_v1[TILE_B];
  __shared__ float lds_ml[4 * 128];
  LC_LDS char *k0 = (LC_LDS char*)lds_k0, *k1 = (LC_LDS char*)lds_k1;
  LC_LDS char *v0 = (LC_LDS char*)lds_v0, *v1 = (LC_LDS char*)lds_v1;
  RangeItem it;
  const int id = blockIdx.x;
  if (id < p_blocks) {
    if (!prefix_item(a, id, row_tiles, 32 * WR, it)) return;
    if (it.t_begin < it.t_end) {
      if constexpr (WR > 1)
        paged_range<T, DPAD, WR>(a, it, k0, k1, v0, v1);
      else
        paged_stream<T, DPAD>(a, it, 4, k0, k1, v0, v1, (LC_LDS float*)lds_ml);
    }
  } else {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    own_item(a, (id - p_blocks) * (4 / own_waves) + wave / own_waves, head_groups, it);
    if (own_waves < 4 || it.t_begin < it.t_end)
      paged_stream<T, DPAD>(a, it, own_waves, k0, k1, v0, v1, (LC_LDS float*)lds_ml);
  }
  if (a.counters != nullptr) join_last<T>(a, it.b0 / a.W, it.kvh);
}


template <int DPAD>
__global__ __launch_bounds__(256) __attribute__((
    amdgpu_waves_per_eu(DPAD <= 64 ? 2 : 1, DPAD <= 64 ? 2 : 1))) void
shared_f32_kernel(SharedArgs a, int p_blocks, int row_tiles, int head_groups) {
  RangeItem it;
  const int id = blockIdx.x;
  if (id < p_blocks) {
    if (!prefix_item(a, id, row_tiles, 32, it)) return;
  } else {
    own_item(a, id - p_blocks, head_groups, it);
  }
  if (it.t_begin < it.t_end) paged_f32_range<DPAD>(a, it);
  if (a.counters != nullptr) join_last<float>(a, it.b0 / a.W, it.kvh);
}

// Merge: one wave per (sequence, query head) joins the live ranges of its
// prefix and of its own tokens; each lane owns VPL consecutive floats of
// head_dim. A row without tokens gets out = 0, lse = -inf.
template <typename T, int VPL>
__global__ __launch_bounds__(64) void shared_merge_kernel(SharedArgs a, T* __restrict__ out,
                                                          int64_t o_sb, int64_t o_sh,
                                                          float* __restrict__ lse_out) {
  constexpr int kBatch = 8;  // rows loaded before the first is added; divides 64
  const int lane = threadIdx.x;
  const int h = blockIdx.x, b = blockIdx.y;
  const int n_p = range_count(clamp_len(a.plens[b / a.W], a.p_pages, a.P), a.p_splits);
  const int n_s = range_count(clamp_len(a.slens[b], a.s_pages, a.P), a.s_splits);
  const int n_all = n_p + n_s;
  const int64_t base = ((int64_t)b * a.Hq + h) * (a.p_splits + a.s_splits);
  auto slot = [&](int j) { return j < n_p ? j : a.p_splits + (j - n_p); };
  const int d0 = lane * VPL;
  const int dl = d0 < a.D ? d0 : 0;  // lanes past head_dim read (and drop) column 0
  const float* rows = a.part_o + base * a.D + dl;

  float mx = -INFINITY;
  bool nan = false;
  for (int j = lane; j < n_all; j += 64) {
    const float x = a.part_lse[base + slot(j)];
    nan |= x != x;
    mx = fmaxf(mx, x);
  }
  mx = lc_wave_max(mx);
  if (__ballot(nan)) mx = NAN;
  float acc[VPL];
#pragma unroll
  for (int e = 0; e < VPL; ++e) acc[e] = 0.f;
  float wsum = 0.f;
  if (mx != -INFINITY) {
    for (int s0 = 0; s0 < n_all; s0 += 64) {
      const int n = min(64, n_all - s0);
      const float w = lane < n ? lc_exp2(a.part_lse[base + slot(s0 + lane)] - mx) : 0.f;
      for (int j0 = 0; j0 < n; j0 += kBatch) {
        float v[kBatch][VPL];
#pragma unroll
        for (int jj = 0; jj < kBatch; ++jj) {
          const int64_t at = (int64_t)slot(min(s0 + j0 + jj, n_all - 1)) * a.D;
#pragma unroll
          for (int e = 0; e < VPL; ++e) v[jj][e] = rows[at + e];
        }
#pragma unroll
        for (int jj = 0; jj < kBatch; ++jj) {
          const float wj =
              __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), min(j0 + jj, 63)));
          if (j0 + jj < n && wj != 0.f) {  // (range after range, as join_last sums them)
            wsum += wj;
#pragma unroll
            for (int e = 0; e < VPL; ++e) acc[e] = fmaf(wj, v[jj][e], acc[e]);
          }
        }
      }
    }
  }
  const float inv = wsum == 0.f ? 0.f : 1.0f / wsum;
  T* oh = out + (int64_t)b * o_sb + (int64_t)h * o_sh;
#pragma unroll
  for (int e = 0; e < VPL; ++e)
    if (d0 + e < a.D) oh[d0 + e] = lc_from_f32<T>(rounded(acc[e] * inv));
  if (lse_out != nullptr && lane == 0)
    lse_out[(int64_t)b * a.Hq + h] = wsum == 0.f ? -INFINITY : (mx + lc_log2(wsum)) * kLn2;
}

struct SharedPlan {
  int wr;         // row tiles of 32 of a prefix's workgroups
  int own_waves;  // waves that share a range of a sequence's own tokens
  int p_splits, s_splits;
};

// Ranges per prefix and per sequence, such that a range is what one CU would do if
// all tokens were dealt out evenly: every further range costs its partial outputs
// (512 bytes a row, written and read back) and a start. A prefix token of a 128-row
// tile counts as six of a stream's (a QK and two PV products for four times the rows),
// of a 64-row tile as three (GPU time of a call, us, by ranges per prefix; 8B heads):
//   256 x (8192 + 200) tokens  2: 125  3: 97  4: 86  5: 93  6: 93  8: 101
//   64 x (8192 + 625)          8: 58  9: 57  10: 56  12: 56  16: 57  20: 72
//   4 groups x 8 x (4096 + 128)  4: 25.3  6: 23.1  8: 23.2  13: 29.6  16: 31.1
// No range is shorter than two tiles.
// A range of a sequence's own tokens is shared by 4, 2 or 1 waves: one wave has no
// join at the end and a longer run of steps, which pays with many short ranges
// (behind 1024 tokens, us with 4 / 2 / 1 waves: 8B heads, 256 x 40 tokens 47 / 37 / 35, 64
// x 200 27.5 / 27.9 / 24.5, 64 x 800 49 / 49 / 51, 64 x 1600 81 / 83 / 87; 16/8 heads of 64,
// 200 x 200 33 / 28 / 24, 64 x 1600 47 / 45 / 63); where the ranges are few, four finish
// sooner (8B, 16 x 100: 13.1 / 14.2 / 16.2). Of 43 such sizes the rule takes the fastest,
// within 5%, at 39; at the others it loses up to 13% (70B heads, 64 x 100: 28.9 for 25.6).
SharedPlan shared_plan(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t p_cap,
                       int64_t s_cap, int dtype) {
  if (B == 0) return SharedPlan{1, 4, 0, 0};
  const int64_t G = Hq / Hkv, W = B / N, cus = lc_cu_count();
  const int wr = dtype == LC_DTYPE_F32 || W * G <= 32 ? 1 : W * G <= 64 ? 2 : 4;
  const int64_t up = N * Hkv * lc_cdiv(W * G, 32 * wr), us = B * Hkv * lc_cdiv(G, 32);
  const int64_t weight = wr == 1 ? 1 : wr * 3 / 2;
  const int64_t each = lc_cdiv(up * p_cap * weight + us * s_cap, cus);
  auto splits = [&](int64_t cap, int64_t tokens) -> int {
    if (cap == 0) return 0;
    const int64_t s = lc_cdiv(cap, tokens < 2 * kSharedStep ? 2 * kSharedStep : tokens);
    return static_cast<int>(s < 64 ? s : 64);
  };
  SharedPlan p;
  p.wr = wr;
  p.p_splits = splits(p_cap, lc_cdiv(each, weight));
  p.s_splits = splits(s_cap, each);
  const int64_t ranges = us * p.s_splits;
  const int64_t steps = p.s_splits > 0 ? lc_cdiv(lc_cdiv(s_cap, p.s_splits), 32) : 0;
  p.own_waves = ranges < 2 * cus || steps > 40 ? 4 : steps > 12 ? 2 : 1;
  return p;
}

int64_t shared_bytes(int64_t rows, int64_t D, const SharedPlan& p) {
  const int64_t n = rows * (p.p_splits + p.s_splits);
  return (n * D * 4 + 255) / 256 * 256 + n * 4;
}

template <typename T>
int launch_merge(const SharedArgs& a, void* out, int64_t o_sb, int64_t o_sh, float* lse,
                 hipStream_t st) {
  dim3 grid(a.Hq, a.B);
  T* o = static_cast<T*>(out);
  if (a.D <= 64)
    shared_merge_kernel<T, 1><<<grid, 64, 0, st>>>(a, o, o_sb, o_sh, lse);
  else if (a.D <= 128)
    shared_merge_kernel<T, 2><<<grid, 64, 0, st>>>(a, o, o_sb, o_sh, lse);
  else
    shared_merge_kernel<T, 4><<<grid, 64, 0, st>>>(a, o, o_sb, o_sh, lse);
  return lc_check_launch("lc_shared_prefix_decode_fwd (merge)");
}

template <typename T, int DPAD>
int launch_mfma(const SharedArgs& a, int wr, int own_waves, hipStream_t st) {
  const int64_t row_tiles = lc_cdiv((int64_t)a.W * a.G, 32 * wr), head_groups = lc_cdiv(a.G, 32);
  const int64_t pairs = (int64_t)(a.B / a.W) * a.Hkv * a.p_splits;
  const int64_t p_blocks = lc_cdiv(pairs, 8) * 8 * row_tiles;
  const int64_t items = (int64_t)a.B * a.Hkv * head_groups * a.s_splits;
  const int64_t blocks = p_blocks + lc_cdiv(items, 4 / own_waves);
  LC_REQUIRE(blocks < (1LL << 24), "lc_shared_prefix_decode_fwd: %lld workgroups",
             (long long)blocks);
  const dim3 grid(static_cast<unsigned>(blocks));
  const int pb = static_cast<int>(p_blocks), rt = static_cast<int>(row_tiles),
            hg = static_cast<int>(head_groups);
  if (wr == 1)
    shared_mfma_kernel<T, DPAD, 1><<<grid, 256, 0, st>>>(a, pb, rt, hg, own_waves);
  else if (wr == 2)
    shared_mfma_kernel<T, DPAD, 2><<<grid, 256, 0, st>>>(a, pb, rt, hg, own_waves);
  else
    shared_mfma_kernel<T, DPAD, 4><<<grid, 256, 0, st>>>(a, pb, rt, hg, own_waves);
  return lc_check_launch("lc_shared_prefix_decode_fwd (mfma)");
}

int launch_f32(const SharedArgs& a, hipStream_t st) {
  const int64_t row_tiles = lc_cdiv((int64_t)a.W * a.G, 32), head_groups = lc_cdiv(a.G, 32);
  const int64_t pairs = (int64_t)(a.B / a.W) * a.Hkv * a.p_splits;
  const int64_t p_blocks = lc_cdiv(pairs, 8) * 8 * row_tiles;
  const int64_t blocks = p_blocks + (int64_t)a.B * a.Hkv * head_groups * a.s_splits;
  LC_REQUIRE(blocks < (1LL << 24), "lc_shared_prefix_decode_fwd: %lld workgroups",
             (long long)blocks);
  const dim3 grid(static_cast<unsigned>(blocks));
  const int pb = static_cast<int>(p_blocks), rt = static_cast<int>(row_tiles),
            hg = static_cast<int>(head_groups);
  if (a.D <= 32)
    shared_f32_kernel<32><<<grid, 256, 0, st>>>(a, pb, rt, hg);
  else if (a.D <= 64)
    shared_f32_kernel<64><<<grid, 256, 0, st>>>(a, pb, rt, hg);
  else
    shared_f32_kernel<128><<<grid, 256, 0, st>>>(a, pb, rt, hg);
  return lc_check_launch("lc_shared_prefix_decode_fwd (fp32 mfma)");
}

template <typename T>
int launch_shared(SharedArgs a, int wr, int own_waves, bool mfma, int32_t* counters, void* out,
                  int64_t o_sb, int64_t o_sh, float* lse, hipStream_t st) {
  const int splits = a.p_splits + a.s_splits;
  // One launch where the grid is one round of workgroups, which read little, and each
  // joins little.
  const int64_t rows = (int64_t)a.W * a.G, tiles = lc_cdiv(rows, 32 * wr);
  const int64_t expected = tiles * a.p_splits + (int64_t)a.W * lc_cdiv(a.G, 32) * a.s_splits;
  const int64_t units = (int64_t)(a.B / a.W) * a.Hkv;
  const bool join = counters != nullptr && mfma && own_waves == 4 && splits > 0 &&
                    splits <= kJoinRanges && rows * a.D <= kJoinOutputs &&
                    rows * splits * a.D * 4 <= kJoinBytes &&
                    units <= kJoinCounters && units * expected <= 2 * lc_cu_count() &&
                    units * ((int64_t)a.p_pages + (int64_t)a.W * a.s_pages) * a.P * a.D * 2 *
                            (int64_t)sizeof(T) <= kJoinRead;
  if (join) {
    a.counters = counters;
    a.expected = static_cast<int>(expected);
    a.out = out;
    a.o_sb = o_sb;
    a.o_sh = o_sh;
    a.lse = lse;
  }
  if (splits > 0 && mfma) {
    if constexpr (sizeof(T) == 2) {
      const int rc = a.D <= 64 ? launch_mfma<T, 64>(a, wr, own_waves, st)
                                 : launch_mfma<T, 128>(a, wr, own_waves, st);
      if (rc != LC_OK) return rc;
    } else {
      const int rc = launch_f32(a, st);
      if (rc != LC_OK) return rc;
    }
  } else if (splits > 0) {
    shared_generic_kernel<T><<<dim3(splits, a.Hq, a.B), 64, 0, st>>>(a);
    const int rc = lc_check_launch("lc_shared_prefix_decode_fwd (generic)");
    if (rc != LC_OK) return rc;
  }
  if (join) return LC_OK;
  return launch_merge<T>(a, out, o_sb, o_sh, lse, st);
}

}  // namespace

extern "C" {

int64_t lc_shared_prefix_decode_counter_count(void) { return kJoinCounters; }

int64_t lc_shared_prefix_decode_workspace_bytes(int64_t B, int64_t groups, int64_t Hq, int64_t Hkv,
                                                int64_t D, int64_t prefix_capacity,
                                                int64_t own_capacity, int dtype) {
  if (B < 0 || groups <= 0 || B % groups != 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || D <= 0 ||
      prefix_capacity < 0 || own_capacity < 0)
    return -1;
  return shared_bytes(B * Hq, D,
                      shared_plan(B, groups, Hq, Hkv, prefix_capacity, own_capacity, dtype));
}

int lc_shared_prefix_decode_fwd(const void* q, int64_t q_sb, int64_t q_sh, const void* key_pages,
                                const void* value_pages, int64_t kv_s_page, int64_t kv_s_head,
                                int64_t kv_s_tok, int64_t num_pages, const int32_t* prefix_table,
                                int64_t pt_stride, int64_t max_prefix_pages,
                                const int32_t* prefix_lens, const int32_t* block_table,
                                int64_t bt_stride, int64_t max_pages_per_seq,
                                const int32_t* seq_lens, void* out, int64_t o_sb, int64_t o_sh,
                                float* lse, void* workspace, int64_t workspace_bytes,
                                int32_t* counters, int64_t B, int64_t groups, int64_t Hq,
                                int64_t Hkv, int64_t D, int64_t page_size, float scale, int dtype, void* stream) {
  static const char* who = "lc_shared_prefix_decode_fwd";
  LC_REQUIRE(B >= 0 && B < 65536, "%s: batch %lld out of range", who, (long long)B);
  LC_REQUIRE(groups > 0 ? B % groups == 0 : B == 0,
             "%s: batch %lld is not a multiple of %lld groups", who, (long long)B,
             (long long)groups);
  LC_REQUIRE(Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq < 65536,
             "%s: n_heads (%lld) must be a multiple of n_kv_heads (%lld)", who, (long long)Hq,
             (long long)Hkv);
  LC_REQUIRE(D > 0 && D <= 256, "%s: head_dim %lld not in [1, 256]", who, (long long)D);
  LC_REQUIRE(dtype == LC_DTYPE_F32 || dtype == LC_DTYPE_F16 || dtype == LC_DTYPE_BF16,
             "%s: unknown dtype %d", who, dtype);
  if (B == 0) return LC_OK;
  LC_REQUIRE(q && key_pages && value_pages && prefix_lens && seq_lens && out && workspace,
             "%s: null pointer", who);
  LC_REQUIRE(page_size > 0 && num_pages > 0 && num_pages < (1LL << 31) && max_prefix_pages >= 0 &&
                 max_pages_per_seq >= 0,
             "%s: page_size and num_pages must be > 0, table widths >= 0", who);
  LC_REQUIRE((prefix_table || max_prefix_pages == 0) && (block_table || max_pages_per_seq == 0),
             "%s: null table", who);
  LC_REQUIRE(max_prefix_pages < (1LL << 30) / page_size &&
                 max_pages_per_seq < (1LL << 30) / page_size,
             "%s: a table of 2^30 tokens or more", who);
  LC_REQUIRE(pt_stride >= max_prefix_pages && bt_stride >= max_pages_per_seq,
             "%s: table stride < row length", who);
  LC_REQUIRE(q_sb >= 0 && q_sh >= 0 && o_sb >= 0 && o_sh >= 0 && kv_s_page >= 0 &&
                 kv_s_head >= 0 && kv_s_tok >= 0,
             "%s: negative stride", who);
  const SharedPlan plan = shared_plan(B, groups, Hq, Hkv, max_prefix_pages * page_size,
                                      max_pages_per_seq * page_size, dtype);
  const int64_t need = shared_bytes(B * Hq, D, plan);
  if (workspace_bytes < need)
    return lc_fail(LC_EWORKSPACE, "%s: workspace %lld < %lld bytes", who,
                   (long long)workspace_bytes, (long long)need);
  LC_REQUIRE(lc_aligned(workspace, 256), "%s: workspace not 256-byte aligned", who);
  LC_REQUIRE(lc_aligned(counters, 4), "%s: counters not 4-byte aligned", who);

  SharedArgs a{};
  a.q = q;
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.kp = key_pages;
  a.vp = value_pages;
  a.s_page = kv_s_page;
  a.s_head = kv_s_head;
  a.s_tok = kv_s_tok;
  a.ptab = prefix_table;
  a.ptab_stride = pt_stride;
  a.plens = prefix_lens;
  a.btab = block_table;
  a.btab_stride = bt_stride;
  a.slens = seq_lens;
  const int64_t n = B * Hq * (plan.p_splits + plan.s_splits);
  a.part_o = static_cast<float*>(workspace);
  a.part_lse =
      reinterpret_cast<float*>(static_cast<char*>(workspace) + (n * D * 4 + 255) / 256 * 256);
  a.B = static_cast<int>(B);
  a.W = static_cast<int>(B / groups);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.G = static_cast<int>(Hq / Hkv);
  a.D = static_cast<int>(D);
  a.P = static_cast<int>(page_size);
  a.p_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctzll(page_size) : -1;
  a.num_pages = static_cast<int>(num_pages);
  a.p_pages = static_cast<int>(max_prefix_pages);
  a.s_pages = static_cast<int>(max_pages_per_seq);
  a.p_splits = plan.p_splits;
  a.s_splits = plan.s_splits;
  a.scale_log2 = scale * kLog2e;
  // The matrix kernels take whole 16-byte vectors of rows, pages of a power of two
  // from 8 tokens up, and 32-bit strides (a page's rows within 2 GiB).
  const int64_t vec = 16 / lc_dtype_size(dtype);
  const bool mfma = D % vec == 0 && D <= 128 && q_sb % vec == 0 && q_sh % vec == 0 &&
                    kv_s_page % vec == 0 && kv_s_head % vec == 0 && kv_s_tok % vec == 0 &&
                    a.p_shift >= 3 && kv_s_tok < (1LL << 29) / page_size &&
                    kv_s_page < (1LL << 32) && scale > 0 && lc_aligned(q, 16) &&
                    lc_aligned(key_pages, 16) && lc_aligned(value_pages, 16);
  hipStream_t st = lc_stream(stream);
  switch (dtype) {
    case LC_DTYPE_F32:
      return launch_shared<float>(a, plan.wr, plan.own_waves, mfma, counters, out, o_sb, o_sh, lse,
                                 st);
    case LC_DTYPE_BF16:
      return launch_shared<bf16_t>(a, plan.wr, plan.own_waves, mfma, counters, out, o_sb, o_sh, lse,
                                  st);
    default:
      return launch_shared<f16_t>(a, plan.wr, plan.own_waves, mfma, counters, out, o_sb, o_sh, lse,
                                 st);
  }
}

}  // extern "C"
