// GQA attention of the newest tokens of every sequence over the paged KV cache.
//
// Sequence b holds L tokens, n of which (n <= T) are its queries: query i stands at
// position p = L - n + i and attends to tokens 0 .. p. A kv head's T G query rows (row
// r = i G + g) share K and V; a tile of them takes tokens 0 .. its last row's p, cut
// into `splits` equal ranges, whose normalised outputs and logsumexps a merge launch
// joins:
//   out = sum_i 2^(lse_i - M) o_i / sum_i 2^(lse_i - M),  M = max_i lse_i
// (lse in log2 units); one range writes the output itself.
//
// Bound: reading K and V once (32 sequences of 4096 tokens, 5 queries, 8B heads: 537 MB in
// 90 us, 5.9 TB/s; 8 of 32768, 70B: 1.07 GB in 194 us + merge 6.7), from some hundred rows a kv
// head on the matrix and softmax work of the tiles (3 x up to 160 queries behind up to 4000
// tokens, f16: 63 us + merge 12: the matrix units are busy a quarter of it, the vector units
// a third; two waves a SIMD, and a second round of 88 workgroups). fp32: see paged_f32_range.
#include <math.h>

#include "lc_common.h"
#include "paged_tiles.h"

namespace {

using namespace lc_attn;

struct ExtendArgs {
  const void* q;
  int64_t q_sb, q_sh, q_st;
  const void* kp;
  const void* vp;
  int64_t s_page, s_head, s_tok;
  const int32_t* table;  // [B, pages]
  int64_t t_stride;
  const int32_t* lens;   // [B]
  const int32_t* qlens;  // [B] or null: T
  void* out;
  int64_t o_sb, o_sh, o_st;
  float* lse;       // [B, Hq, T] or null
  float* part_o;    // [B, Hq, T, splits, D]
  float* part_lse;  // [B, Hq, T, splits], log2 units
  int B, T, Hq, Hkv, G, D, P, p_shift, num_pages, pages, splits, tile_rows;
  float scale_log2;
};

// Tokens of a range are a multiple of this.
constexpr int kStep = 64;

// Length and queries of a sequence.
struct Seq {
  int len, n;
};
__device__ __forceinline__ Seq sequence(const ExtendArgs& a, int b) {
  const int cap = a.pages * a.P, len = a.lens[b];
  const int n = a.qlens == nullptr ? a.T : a.qlens[b];
  return Seq{len < 0 ? 0 : len > cap ? cap : len, n < 0 ? 0 : n > a.T ? a.T : n};
}
// Tokens that query i sees.
__device__ __forceinline__ int visible(const Seq& s, int i) {
  return i < s.n ? max(0, s.len - s.n + i + 1) : 0;
}
// Tokens that a tile of rows from row0 on needs: those of its last live row.
__device__ __forceinline__ int tile_len(const ExtendArgs& a, const Seq& s, int row0) {
  const int last = min(min(row0 + a.tile_rows, a.T * a.G) - 1, s.n * a.G - 1);
  return last < row0 ? 0 : visible(s, last / a.G);
}
__device__ __forceinline__ int range_tokens(int len, int splits) {
  const int each = (len + splits - 1) / splits;
  return (each + kStep - 1) / kStep * kStep;
}
__device__ __forceinline__ int range_count(int len, int splits) {
  if (len <= 0) return 0;
  const int each = range_tokens(len, splits);
  return (len + each - 1) / each;
}

// Element offset of token tok of a table row and kv head; -1 where its page entry
// is invalid. tok is within the row's capacity.
__device__ __forceinline__ int64_t token_offset(const ExtendArgs& a, const int32_t* row, int kvh,
                                                int tok) {
  const int page = a.p_shift >= 0 ? tok >> a.p_shift : tok / a.P;
  const int slot = tok - page * a.P;
  const int phys = row[page];
  if (static_cast<unsigned>(phys) >= static_cast<unsigned>(a.num_pages)) return -1;
  return (int64_t)phys * a.s_page + (int64_t)kvh * a.s_head + (int64_t)slot * a.s_tok;
}

// Generic kernel: one wave per (row, range), lanes across head_dim, one token at a
// time. Any dtype, head_dim <= 256 and strides.
template <typename T>
__global__ __launch_bounds__(64) void extend_generic_kernel(ExtendArgs a) {
  const int lane = threadIdx.x;
  const int i = blockIdx.x % a.T, rest = blockIdx.x / a.T;
  const int split = rest % a.splits, bh = rest / a.splits;
  const int h = bh % a.Hq, b = bh / a.Hq;
  const int kvh = h / a.G, r = i * a.G + h % a.G;
  const Seq s = sequence(a, b);
  const int len = tile_len(a, s, r / a.tile_rows * a.tile_rows);
  const int each = range_tokens(len, a.splits);
  const int t_begin = split * each;
  if (t_begin >= len) return;
  const int t_end = min(min(len, t_begin + each), visible(s, i));
  const int32_t* row = a.table + (int64_t)b * a.t_stride;
  const T* kp = static_cast<const T*>(a.kp);
  const T* vp = static_cast<const T*>(a.vp);
  const T* qh = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh +
                (int64_t)i * a.q_st;

  float qv[4], acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = lane + 64 * j;
    qv[j] = d < a.D ? lc_to_f32(qh[d]) : 0.f;
    acc[j] = 0.f;
  }
  float m_run = -INFINITY, l_run = 0.f;
  for (int t = t_begin; t < t_end; ++t) {
    const int64_t off = token_offset(a, row, kvh, t);
    if (off < 0) continue;  // uniform across the wave
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = lane + 64 * j;
      if (d < a.D) dot = fmaf(qv[j], lc_to_f32(kp[off + d]), dot);
    }
    const float x = lc_wave_sum(dot) * a.scale_log2;
    if (x == -INFINITY) continue;
    const float m_new = fmaxf(m_run, x);
    const float alpha = lc_exp2(m_run - m_new);
    const float p = lc_exp2(x - m_new);
    l_run = l_run * alpha + p;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = lane + 64 * j;
      const float vv = d < a.D ? lc_to_f32(vp[off + d]) : 0.f;
      acc[j] = fmaf(p, vv, acc[j] * alpha);
    }
    m_run = m_new;
  }
  const int64_t pidx = (((int64_t)b * a.Hq + h) * a.T + i) * a.splits + split;
  const float inv_l = l_run > 0.f ? 1.0f / l_run : l_run;  // (NaN stays NaN)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = lane + 64 * j;
    if (d < a.D) a.part_o[pidx * a.D + d] = acc[j] * inv_l;
  }
  if (lane == 0) a.part_lse[pidx] = l_run == 0.f ? -INFINITY : m_run + lc_log2(l_run);
}

// A range of a sequence's tokens and a tile of a kv head's rows, row r = i G + g.
template <typename T>
struct ExtendItem {
  static constexpr bool kCausal = true;
  const int32_t* table;
  Seq seq;
  int b, kvh, row0, rows, t_begin, t_end, split, all_see;

  template <typename Q>
  __device__ __forceinline__ const Q* query(const ExtendArgs& a, int r) const {
    const int i = r / a.G;
    return static_cast<const Q*>(a.q) + (int64_t)b * a.q_sb + (int64_t)i * a.q_st +
           (int64_t)(kvh * a.G + (r - i * a.G)) * a.q_sh;
  }
  __device__ __forceinline__ int limit(const ExtendArgs& a, int r) const {
    return visible(seq, r / a.G);
  }
  // Where a row's results go: with one range they are the row's output.
  struct Row {
    T* out;
    float* part;
    int64_t lse;
  };
  __device__ __forceinline__ Row row(const ExtendArgs& a, int r) const {
    const int i = r / a.G, h = kvh * a.G + (r - i * a.G);
    const int64_t at = (((int64_t)b * a.Hq + h) * a.T + i) * a.splits + split;
    return Row{static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)i * a.o_st + (int64_t)h * a.o_sh,
               a.part_o + at * a.D, at};
  }
  __device__ __forceinline__ void store4(const ExtendArgs& a, const Row& row, int d, f32x4_t x) const {
    if (a.splits == 1) {
      typedef T t4 __attribute__((ext_vector_type(4)));
      t4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = lc_from_f32<T>(x[e]);
      *reinterpret_cast<t4*>(row.out + d) = y;
    } else {
      *reinterpret_cast<f32x4_t*>(row.part + d) = x;
    }
  }
  __device__ __forceinline__ void store_lse(const ExtendArgs& a, const Row& row, float x) const {
    if (a.splits > 1)
      a.part_lse[row.lse] = x;
    else if (a.lse != nullptr)
      a.lse[row.lse] = x * kLn2;
  }
};

// Work item `at` of the grid. A range's row tiles read the same K and V: they get items 8
// apart, which run on one XCD, and find it in its L2; the last tile, which sees the
// most tokens, first. False: an item past the last range. The range may be empty.
template <typename T>
__device__ __forceinline__ bool extend_item(const ExtendArgs& a, int at, int row_tiles,
                                            ExtendItem<T>& it) {
  const int run = at / (8 * row_tiles), rest = at - run * 8 * row_tiles;
  const int pair = run * 8 + (rest & 7), tile = row_tiles - 1 - (rest >> 3);
  const int units = a.B * a.Hkv;
  const int split = pair / units, u = pair - split * units;
  const bool live = split < a.splits;
  it.split = live ? split : 0;
  it.b = live ? u / a.Hkv : 0;
  it.kvh = live ? u - it.b * a.Hkv : 0;
  it.table = a.table + (int64_t)it.b * a.t_stride;
  it.seq = sequence(a, it.b);
  it.rows = a.T * a.G;
  it.row0 = tile * a.tile_rows;
  const int len = live ? tile_len(a, it.seq, it.row0) : 0;
  const int each = range_tokens(len, a.splits);
  it.t_begin = it.split * each;
  it.t_end = min(len, it.t_begin + each);
  it.all_see = max(1, visible(it.seq, it.row0 / a.G));
  return live;
}

// Outputs of a tile that sees no token, written by `threads` threads.
template <typename T>
__device__ __forceinline__ void clear_rows(const ExtendArgs& a, const ExtendItem<T>& it, int thread,
                                           int threads) {
  const int chunks = a.D / 4, end = min(it.rows, it.row0 + a.tile_rows);
  for (int e = thread; e < (end - it.row0) * chunks; e += threads) {
    const int r = it.row0 + e / chunks, d = e % chunks * 4;
    const auto row = it.row(a, r);
    it.store4(a, row, d, f32x4_t{0.f, 0.f, 0.f, 0.f});
    if (d == 0) it.store_lse(a, row, -INFINITY);
  }
}

// bf16/f16, head_dim a multiple of 8 up to 128, pages of a power of two from 8 up (see
// paged_tiles.h): a workgroup of 4 waves per range and tile of 32 WR rows; with one
// tile of 32 rows, `waves` of its waves per range.
template <typename T, int DPAD, int WR>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void
extend_mfma_kernel(ExtendArgs a, int row_tiles, int waves) {
  constexpr int TILE_B = kTile * DPAD * (int)sizeof(T);
  // (separate arrays: the compiler tracks a DMA by the array that it writes)
  __shared__ __align__(16) char lds_k0[TILE_B];
  __shared__ __align__(16) char lds_k1[TILE_B];
  __shared__ __align__(16) char lds_v0[TILE_B];
  __shared__ __align__(16) char lds_v1[TILE_B];
  __shared__ float lds_scratch[4 * 512];
  LC_LDS char *k0 = (LC_LDS char*)lds_k0, *k1 = (LC_LDS char*)lds_k1;
  LC_LDS char *v0 = (LC_LDS char*)lds_v0, *v1 = (LC_LDS char*)lds_v1;
  ExtendItem<T> it;
  if constexpr (WR > 1) {
    if (!extend_item(a, blockIdx.x, row_tiles, it)) return;
    if (it.t_begin < it.t_end)
      paged_range<T, DPAD, WR>(a, it, k0, k1, v0, v1, (LC_LDS float*)lds_scratch);
    else if (a.splits == 1)
      clear_rows(a, it, threadIdx.x, 256);
  } else {
    __shared__ float lds_ml[4 * 128];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool live = extend_item(a, blockIdx.x * (4 / waves) + wave / waves, row_tiles, it);
    if (waves < 4 || it.t_begin < it.t_end)
      paged_stream<T, DPAD>(a, it, waves, k0, k1, v0, v1, (LC_LDS float*)lds_ml,
                            (LC_LDS float*)lds_scratch);
    if (live && it.t_begin >= it.t_end && a.splits == 1)
      clear_rows(a, it, threadIdx.x % (64 * waves), 64 * waves);
  }
}

template <int DPAD>
__global__ __launch_bounds__(256) __attribute__((
    amdgpu_waves_per_eu(DPAD <= 64 ? 2 : 1, DPAD <= 64 ? 2 : 1))) void
extend_f32_kernel(ExtendArgs a, int row_tiles) {
  ExtendItem<float> it;
  if (!extend_item(a, blockIdx.x, row_tiles, it)) return;
  if (it.t_begin < it.t_end)
    paged_f32_range<DPAD>(a, it);
  else if (a.splits == 1)
    clear_rows(a, it, threadIdx.x, 256);
}

// Merge: one wave per row joins its tile's ranges; each lane owns VPL consecutive
// floats of head_dim. A row that sees no token gets out = 0, lse = -inf.
template <typename T, int VPL>
__global__ __launch_bounds__(256) void extend_merge_kernel(ExtendArgs a, int64_t rows) {
  constexpr int kBatch = 8;
  const int lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= rows) return;
  const int i = static_cast<int>(at % a.T);
  const int64_t bh = at / a.T;
  const int h = static_cast<int>(bh % a.Hq), b = static_cast<int>(bh / a.Hq);
  const Seq s = sequence(a, b);
  const int r = i * a.G + h % a.G;
  const int n_all = visible(s, i) == 0
                        ? 0
                        : range_count(tile_len(a, s, r / a.tile_rows * a.tile_rows), a.splits);
  const int d0 = lane * VPL, dl = d0 < a.D ? d0 : 0;
  const float* part = a.part_o + at * a.splits * a.D + dl;
  const float* plse = a.part_lse + at * a.splits;
  float w = lane < n_all ? plse[lane] : -INFINITY;  // (splits <= 64)
  float mx = lc_wave_max(w);
  if (__ballot(w != w)) mx = NAN;
  float acc[VPL], wsum = 0.f;
#pragma unroll
  for (int e = 0; e < VPL; ++e) acc[e] = 0.f;
  if (mx != -INFINITY) {
    w = lane < n_all ? lc_exp2(w - mx) : 0.f;
    for (int j0 = 0; j0 < n_all; j0 += kBatch) {
      float v[kBatch][VPL];
#pragma unroll
      for (int jj = 0; jj < kBatch; ++jj)
#pragma unroll
        for (int e = 0; e < VPL; ++e) v[jj][e] = part[(int64_t)min(j0 + jj, n_all - 1) * a.D + e];
#pragma unroll
      for (int jj = 0; jj < kBatch; ++jj) {
        const float wj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), min(j0 + jj, 63)));
        if (j0 + jj < n_all && wj != 0.f) {
          wsum += wj;
#pragma unroll
          for (int e = 0; e < VPL; ++e) acc[e] = fmaf(wj, v[jj][e], acc[e]);
        }
      }
    }
  }
  const float inv = wsum == 0.f ? 0.f : 1.0f / wsum;
  T* oh = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)i * a.o_st;
#pragma unroll
  for (int e = 0; e < VPL; ++e)
    if (d0 + e < a.D) oh[d0 + e] = lc_from_f32<T>(acc[e] * inv);
  if (a.lse != nullptr && lane == 0)
    a.lse[at] = wsum == 0.f ? -INFINITY : (mx + lc_log2(wsum)) * kLn2;
}

struct ExtendPlan {
  int wr;      // row tiles of 32 of a workgroup
  int splits;  // ranges of a tile's tokens
  int waves;   // waves that share a range where wr is 1
};

// Ranges of a full table: as many as give the CUs one round of workgroups, two of them each
// where tiles go through LDS, rounded up (us at 1 / 2 / 4 / 8 ranges: 32 sequences of 5
// queries behind up to 4096 tokens, 8B heads 67 / 73 / 77 / 85; 8 behind 32768, 70B 625 / 334
// / 198 / 199; one of 256 queries behind 4000, 8B 132 / 87 / 62 / 56). None is shorter than
// 128 tokens there: 5 queries behind 1000 take 14.1 us cut in 8, 21 in one piece. The rule
// goes by the table's width, which the host knows; a sequence that leaves most of its row
// unused is cut into as many, of 64 tokens or more (us in tables 1 / 8 / 64 times as wide as
// the longest sequence: one of 1000 tokens 14.2 / 15.0 / 14.9; 256 of 400, whose ranges then
// get two waves, 84 / 91 / 91; 32 of 4096, and chunks of 160 behind 4000, within 1%).
// Waves that share a range: four where the ranges are at most a round of workgroups (us
// with 4 / 2 / 1 waves: 64 sequences of 1000 tokens, 8B heads 49 / 51 / 61, 48 of up to 1500
// 41 / 49 / 79), two above (96 of up to 300 32 / 26 / 29, 128 of 2000 186 / 173 / 173), one
// for many short ones (256 of 400 101 / 90 / 82, of up to 800 119 / 114 / 117).
ExtendPlan extend_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t cap, int dtype) {
  const int64_t rows = T * (Hq / Hkv), cus = lc_cu_count();
  ExtendPlan p{1, 1, 4};
  if (dtype != LC_DTYPE_F32) p.wr = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  const int64_t units = B * Hkv * lc_cdiv(rows, 32 * p.wr);
  if (units == 0 || cap == 0) return p;
  int64_t s = lc_cdiv(p.wr == 1 ? cus : 2 * cus, units);
  const int64_t most = lc_cdiv(cap, 2 * kStep);
  s = s < most ? s : most;
  p.splits = static_cast<int>(s < 64 ? s : 64);
  const int64_t ranges = units * p.splits, steps = lc_cdiv(lc_cdiv(cap, p.splits), 32);
  p.waves = ranges <= 2 * cus ? 4 : ranges >= 6 * cus && steps <= 20 ? 1 : 2;
  return p;
}
int64_t extend_bytes(int64_t rows, int64_t D, const ExtendPlan& p) {
  const int64_t n = rows * p.splits;
  return (n * D * 4 + 255) / 256 * 256 + n * 4;
}

template <typename T, int DPAD>
int launch_mfma(const ExtendArgs& a, const ExtendPlan& p, hipStream_t st) {
  const int64_t row_tiles = lc_cdiv((int64_t)a.T * a.G, a.tile_rows);
  const int64_t items = lc_cdiv((int64_t)a.B * a.Hkv * a.splits, 8) * 8 * row_tiles;
  const int64_t blocks = p.wr == 1 ? lc_cdiv(items, 4 / p.waves) : items;
  LC_REQUIRE(blocks < (1LL << 24), "lc_paged_extend_fwd: %lld workgroups", (long long)blocks);
  const dim3 grid(static_cast<unsigned>(blocks));
  const int rt = static_cast<int>(row_tiles);
  if (p.wr == 1)
    extend_mfma_kernel<T, DPAD, 1><<<grid, 256, 0, st>>>(a, rt, p.waves);
  else if (p.wr == 2)
    extend_mfma_kernel<T, DPAD, 2><<<grid, 256, 0, st>>>(a, rt, p.waves);
  else
    extend_mfma_kernel<T, DPAD, 4><<<grid, 256, 0, st>>>(a, rt, p.waves);
  return lc_check_launch("lc_paged_extend_fwd (mfma)");
}

int launch_f32(const ExtendArgs& a, hipStream_t st) {
  const int64_t row_tiles = lc_cdiv((int64_t)a.T * a.G, a.tile_rows);
  const int64_t blocks = lc_cdiv((int64_t)a.B * a.Hkv * a.splits, 8) * 8 * row_tiles;
  LC_REQUIRE(blocks < (1LL << 24), "lc_paged_extend_fwd: %lld workgroups", (long long)blocks);
  const dim3 grid(static_cast<unsigned>(blocks));
  const int rt = static_cast<int>(row_tiles);
  if (a.D <= 32)
    extend_f32_kernel<32><<<grid, 256, 0, st>>>(a, rt);
  else if (a.D <= 64)
    extend_f32_kernel<64><<<grid, 256, 0, st>>>(a, rt);
  else
    extend_f32_kernel<128><<<grid, 256, 0, st>>>(a, rt);
  return lc_check_launch("lc_paged_extend_fwd (fp32 mfma)");
}

template <typename T>
int launch_extend(const ExtendArgs& a, const ExtendPlan& p, bool mfma, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Hq * a.T;
  int rc;
  if (!mfma) {
    extend_generic_kernel<T><<<static_cast<unsigned>(rows * a.splits), 64, 0, st>>>(a);
    rc = lc_check_launch("lc_paged_extend_fwd (generic)");
  } else if constexpr (sizeof(T) == 2) {
    rc = a.D <= 64 ? launch_mfma<T, 64>(a, p, st) : launch_mfma<T, 128>(a, p, st);
  } else {
    rc = launch_f32(a, st);
  }
  if (rc != LC_OK || (mfma && a.splits == 1)) return rc;
  const unsigned blocks = static_cast<unsigned>(lc_cdiv(rows, 4));
  if (a.D <= 64)
    extend_merge_kernel<T, 1><<<blocks, 256, 0, st>>>(a, rows);
  else if (a.D <= 128)
    extend_merge_kernel<T, 2><<<blocks, 256, 0, st>>>(a, rows);
  else
    extend_merge_kernel<T, 4><<<blocks, 256, 0, st>>>(a, rows);
  return lc_check_launch("lc_paged_extend_fwd (merge)");
}

}  // namespace

extern "C" {

int64_t lc_paged_extend_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                        int64_t capacity, int dtype) {
  if (B < 0 || T < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || D <= 0 || capacity < 0) return -1;
  return extend_bytes(B * Hq * T, D, extend_plan(B, T, Hq, Hkv, capacity, dtype));
}

int lc_paged_extend_fwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st,
                        const void* key_pages, const void* value_pages, int64_t kv_s_page,
                        int64_t kv_s_head, int64_t kv_s_tok, int64_t num_pages,
                        const int32_t* block_table, int64_t bt_stride, int64_t max_pages_per_seq,
                        const int32_t* seq_lens, const int32_t* query_lens, void* out,
                        int64_t o_sb, int64_t o_sh, int64_t o_st, float* lse, void* workspace,
                        int64_t workspace_bytes, int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                        int64_t D, int64_t page_size, float scale, int dtype, void* stream) {
  static const char* who = "lc_paged_extend_fwd";
  LC_REQUIRE(B >= 0 && B < 65536 && T >= 0 && T < (1LL << 20), "%s: batch %lld of %lld queries",
             who, (long long)B, (long long)T);
  LC_REQUIRE(Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq < 65536,
             "%s: n_heads (%lld) must be a multiple of n_kv_heads (%lld)", who, (long long)Hq,
             (long long)Hkv);
  LC_REQUIRE(D > 0 && D <= 256, "%s: head_dim %lld not in [1, 256]", who, (long long)D);
  LC_REQUIRE(dtype == LC_DTYPE_F32 || dtype == LC_DTYPE_F16 || dtype == LC_DTYPE_BF16,
             "%s: unknown dtype %d", who, dtype);
  if (B == 0 || T == 0) return LC_OK;
  LC_REQUIRE(q && key_pages && value_pages && seq_lens && out && workspace, "%s: null pointer", who);
  LC_REQUIRE(page_size > 0 && num_pages > 0 && num_pages < (1LL << 31) && max_pages_per_seq >= 0,
             "%s: page_size and num_pages must be > 0, the table's width >= 0", who);
  LC_REQUIRE(block_table || max_pages_per_seq == 0, "%s: null table", who);
  LC_REQUIRE(max_pages_per_seq < (1LL << 30) / page_size, "%s: a table of 2^30 tokens or more", who);
  LC_REQUIRE(bt_stride >= max_pages_per_seq, "%s: table stride < row length", who);
  LC_REQUIRE(q_sb >= 0 && q_sh >= 0 && q_st >= 0 && o_sb >= 0 && o_sh >= 0 && o_st >= 0 &&
                 kv_s_page >= 0 && kv_s_head >= 0 && kv_s_tok >= 0,
             "%s: negative stride", who);
  const ExtendPlan plan = extend_plan(B, T, Hq, Hkv, max_pages_per_seq * page_size, dtype);
  LC_REQUIRE(B * Hq * T < (1LL << 26) / plan.splits, "%s: %lld query rows", who,
             (long long)(B * Hq * T));
  const int64_t need = extend_bytes(B * Hq * T, D, plan);
  if (workspace_bytes < need)
    return lc_fail(LC_EWORKSPACE, "%s: workspace %lld < %lld bytes", who,
                   (long long)workspace_bytes, (long long)need);
  LC_REQUIRE(lc_aligned(workspace, 256), "%s: workspace not 256-byte aligned", who);

  ExtendArgs a{};
  a.q = q;
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.q_st = q_st;
  a.kp = key_pages;
  a.vp = value_pages;
  a.s_page = kv_s_page;
  a.s_head = kv_s_head;
  a.s_tok = kv_s_tok;
  a.table = block_table;
  a.t_stride = bt_stride;
  a.lens = seq_lens;
  a.qlens = query_lens;
  a.out = out;
  a.o_sb = o_sb;
  a.o_sh = o_sh;
  a.o_st = o_st;
  a.lse = lse;
  const int64_t n = B * Hq * T * plan.splits;
  a.part_o = static_cast<float*>(workspace);
  a.part_lse =
      reinterpret_cast<float*>(static_cast<char*>(workspace) + (n * D * 4 + 255) / 256 * 256);
  a.B = static_cast<int>(B);
  a.T = static_cast<int>(T);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.G = static_cast<int>(Hq / Hkv);
  a.D = static_cast<int>(D);
  a.P = static_cast<int>(page_size);
  a.p_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctzll(page_size) : -1;
  a.num_pages = static_cast<int>(num_pages);
  a.pages = static_cast<int>(max_pages_per_seq);
  a.splits = plan.splits;
  a.tile_rows = 32 * plan.wr;
  a.scale_log2 = scale * kLog2e;
  // The matrix kernels take whole 16-byte vectors of rows, pages of a power of two
  // from 8 tokens up, and 32-bit strides (a page's rows within 2 GiB).
  const int64_t vec = 16 / lc_dtype_size(dtype);
  const bool mfma = D % vec == 0 && D <= 128 && q_sb % vec == 0 && q_sh % vec == 0 &&
                    q_st % vec == 0 && kv_s_page % vec == 0 && kv_s_head % vec == 0 &&
                    kv_s_tok % vec == 0 && o_sb % 4 == 0 && o_sh % 4 == 0 && o_st % 4 == 0 &&
                    a.p_shift >= 3 && kv_s_tok < (1LL << 29) / page_size &&
                    kv_s_page < (1LL << 32) && scale > 0 && max_pages_per_seq > 0 &&
                    lc_aligned(q, 16) && lc_aligned(key_pages, 16) &&
                    lc_aligned(value_pages, 16) && lc_aligned(out, 16);
  hipStream_t st = lc_stream(stream);
  switch (dtype) {
    case LC_DTYPE_F32:
      return launch_extend<float>(a, plan, mfma, st);
    case LC_DTYPE_BF16:
      return launch_extend<bf16_t>(a, plan, mfma, st);
    default:
      return launch_extend<f16_t>(a, plan, mfma, st);
  }
}

}  // extern "C"
