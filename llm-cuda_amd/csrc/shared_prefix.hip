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

#include "attn_f32.h"
#include "attn_tiles.h"
#include "lc_common.h"

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
// the waves take token steps of their own (shared_stream below). With more, tiles
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
constexpr int kTile = 64;  // tokens per tile
constexpr float kSharedRescaleLog2 = 8.0f;

__device__ __attribute__((aligned(16))) const uint32_t shared_zeros[4] = {0, 0, 0, 0};

// Two weights, each as a value of the data type below it and what is left, rounded.
// Both parts of a weight above 0 are above 0, so that an infinite V stays infinite (a
// remainder of 0 or of the other sign would make it NaN).
template <typename V>
__device__ __forceinline__ void split_weights(float p0, float p1, V& whole, V& rest, int i) {
  typedef std::remove_reference_t<decltype(whole[0])> T;
  // (the next number below; 0 and a remainder of 0 for 0)
  const uint32_t u0 = __builtin_elementwise_sub_sat(__float_as_uint(p0), 1u),
                 u1 = __builtin_elementwise_sub_sat(__float_as_uint(p1), 1u);
  if constexpr (std::is_same_v<T, bf16_t>) {
    whole[i] = __builtin_bit_cast(T, static_cast<uint16_t>(u0 >> 16));
    whole[i + 1] = __builtin_bit_cast(T, static_cast<uint16_t>(u1 >> 16));
    rest[i] = static_cast<T>(p0 - __uint_as_float(u0 & 0xffff0000u));
    rest[i + 1] = static_cast<T>(p1 - __uint_as_float(u1 & 0xffff0000u));
  } else {
    const auto w = __builtin_amdgcn_cvt_pkrtz(__uint_as_float(u0), __uint_as_float(u1));
    whole[i] = static_cast<T>(w[0]);
    whole[i + 1] = static_cast<T>(w[1]);
    rest[i] = static_cast<T>(p0 - static_cast<float>(w[0]));
    rest[i + 1] = static_cast<T>(p1 - static_cast<float>(w[1]));
  }
}

struct RangeItem {
  const int32_t* table;  // the token range's table row
  int b0, row0, rows;    // row r is sequence b0 + r / G, head r % G of the kv head
  int kvh, t_begin, t_end, slot;
};

// Where the token of each lane lies: its byte offset in the pools, and the bytes of
// the RPI rows from it on that hold tokens of the range (0: none, or an invalid
// page). One lane's answer serves a whole DMA instruction, by v_readlane: computed
// by all lanes at once, it costs a few instructions per tile instead of a 64-bit
// scalar product and its branches per DMA instruction.
struct RowPlace {
  uint32_t lo, hi;
  int bytes;
};
template <int RPI>
__device__ __forceinline__ RowPlace row_place(const SharedArgs& a, int page, int tok, int t_end,
                                              int esz) {
  const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages) && tok < t_end;
  const uint32_t slot = static_cast<uint32_t>(tok & (a.P - 1)) * static_cast<uint32_t>(a.s_tok);
  const uint64_t at =
      (static_cast<uint64_t>(static_cast<uint32_t>(page)) * static_cast<uint32_t>(a.s_page) + slot) *
      static_cast<uint32_t>(esz);
  RowPlace p;
  p.lo = ok ? static_cast<uint32_t>(at) : 0;
  p.hi = ok ? static_cast<uint32_t>(at >> 32) : 0;
  p.bytes = ok ? ((min(RPI, t_end - tok) - 1) * static_cast<int>(a.s_tok) + a.D) * esz : 0;
  return p;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const void* base, const RowPlace& p,
                                                             int lane) {
  const uint64_t at =
      (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(p.hi), lane))) << 32) |
      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(p.lo), lane));
  return __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(base) + at), 0,
      __builtin_amdgcn_readlane(p.bytes, lane), 0x00020000);
}

// Operands of a lane's query row: step s takes the 8 elements of chunk hh CPR / 2 + s
// (zeros for a row that is none, or past head_dim).
template <typename T, int DPAD>
__device__ __forceinline__ void load_rows(const SharedArgs& a, int b, int h, bool row_ok, int hh,
                                          typename Mfma32<T>::v8 (&qop)[DPAD / 16]) {
  typedef typename Mfma32<T>::v8 v8;
  constexpr int CPR = DPAD / 8;
  const T* qh = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh;
#pragma unroll
  for (int s = 0; s < DPAD / 16; ++s) {
    const int d0 = (hh * (CPR / 2) + s) * 8;
    const bool ok = row_ok && d0 < a.D;
    const v8 x = *reinterpret_cast<const v8*>(qh + (ok ? d0 : 0));
    qop[s] = ok ? x : v8{};
  }
}

// LDS addresses of a tile's operands from token row0 on (rows of DPAD, chunks
// swizzled by pf_swz): K rows for S^T, V columns for O^T by transposed reads.
template <typename T, int DPAD>
__device__ __forceinline__ void operand_addresses(int lane, int row0, int (&kaddr)[DPAD / 16],
                                                  int (&vaddr)[2][DPAD / 32]) {
  constexpr int CPR = DPAD / 8, ROW_B = DPAD * (int)sizeof(T);
  const int l32 = lane & 31, hh = lane >> 5;
#pragma unroll
  for (int s = 0; s < DPAD / 16; ++s)
    kaddr[s] = (row0 + l32) * ROW_B + (((hh * (CPR / 2) + s) ^ pf_swz<CPR>(l32)) << 4);
  const int gq = lane >> 4, te = (lane & 15) >> 2, tc = lane & 3;
#pragma unroll
  for (int jj = 0; jj < 2; ++jj)
#pragma unroll
    for (int dt = 0; dt < DPAD / 32; ++dt) {
      const int kr = jj * 8 + hh * 4 + te;
      const int d = dt * 32 + (gq & 1) * 16 + 4 * tc;
      vaddr[jj][dt] = (row0 + kr) * ROW_B +
                      ((((d >> 3) ^ pf_swz<CPR>(kr)) << 4) | ((d & 7) * (int)sizeof(T)));
    }
}

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

// Writes columns dt * 32 .. of a row's partial output.
__device__ __forceinline__ void store_columns(const SharedArgs& a, int64_t pidx, int dt, int hh,
                                              const f32x16_t& o, float inv_l) {
  float* po = a.part_o + pidx * a.D;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d0 = dt * 32 + j * 8 + hh * 4;
    if (d0 < a.D) {  // (D % 8 == 0: whole groups of 4)
      f32x4_t w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = o[j * 4 + e] * inv_l;
      put4(a, po + d0, w);
    }
  }
}

template <typename T, int DPAD, int WR>
__device__ __forceinline__ void shared_range(const SharedArgs& a, const RangeItem& it,
                                             LC_LDS char* lds_k0, LC_LDS char* lds_k1,
                                             LC_LDS char* lds_v0, LC_LDS char* lds_v1) {
  typedef Mfma32<T> Ops;
  typedef typename Ops::v8 v8;
  constexpr int KS = DPAD / 16, DTL = DPAD / 32, CPR = DPAD / 8;
  constexpr int RPI = 64 / CPR;           // token rows per DMA instruction
  constexpr int NIW = kTile / (RPI * 4);  // DMA instructions per wave and tensor
  constexpr int ROW_B = DPAD * (int)sizeof(T);
  constexpr int NKT = WR == 4 ? 2 : 1;  // 32-token blocks per wave and tile
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);
  const int l32 = lane & 31, hh = lane >> 5;
  const int wr = WR == 4 ? wave : (wave & 1);
  const int wk = WR == 4 ? 0 : (wave >> 1);

  // This lane's query row (a wave whose rows are none computes on zeros: it shares
  // the others' steps anyway).
  const int r_abs = it.row0 + wr * 32 + l32;
  const bool row_ok = r_abs < it.rows;
  const int r_safe = row_ok ? r_abs : it.row0;
  const int b = it.b0 + r_safe / a.G;
  const int h = it.kvh * a.G + r_safe % a.G;
  v8 qop[KS];
  load_rows<T, DPAD>(a, b, h, row_ok, hh, qop);

  const T* kp = static_cast<const T*>(a.kp) + (int64_t)it.kvh * a.s_head;
  const T* vp = static_cast<const T*>(a.vp) + (int64_t)it.kvh * a.s_head;
  const int last_page = (it.t_end - 1) >> a.p_shift;
  // Page entry of the tile's token t0 + lane (past the range: one that is not used).
  auto fetch = [&](int t0) { return it.table[min((t0 + lane) >> a.p_shift, last_page)]; };
  // DMA of one tensor's tile: this lane's 16-byte chunk of its row.
  PfLoadOffsets<NIW> off;
#pragma unroll
  for (int u = 0; u < NIW; ++u) {
    const int row = (wave * NIW + u) * RPI + lane / CPR;
    const int ch = (lane % CPR) ^ pf_swz<CPR>(row);
    off.o[u] = ch * 8 < a.D ? static_cast<int>(((lane / CPR) * a.s_tok + ch * 8) * sizeof(T)) : -16;
  }
  auto place = [&](int t0, int pages) {
    return row_place<RPI>(a, pages, t0 + lane, it.t_end, sizeof(T));
  };
  auto issue = [&](const T* base, const RowPlace& at, LC_LDS char* dst) {
#pragma unroll
    for (int u = 0; u < NIW; ++u) {
      const int row0 = (wave_s * NIW + u) * RPI;
      const int vo = off.o[u];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(row_buffer(base, at, row0),
                                               (LC_LDS void*)(dst + row0 * ROW_B), 16, vo, 0, 0, 0);
    }
  };

  // LDS addresses of the operands (see the prefill kernel's).
  int kaddr[KS], vaddr[2][DTL];
  operand_addresses<T, DPAD>(lane, wk * 32, kaddr, vaddr);

  f32x16_t o[DTL];
#pragma unroll
  for (int i = 0; i < DTL; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  float m_ref = -INFINITY, l_lane = 0.f, l_tile = 0.f;
  f32x16_t x[NKT];  // raw scores of the next tile
  f32x16_t y[NKT];  // exponents of the current tile, relative to m_ref
  v8 pop[NKT][2], rem[NKT][2];

  auto qk = [&](LC_LDS const char* kt_lds) __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) x[kt][r] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
        x[kt] = Ops::mma(*reinterpret_cast<LC_LDS const v8*>(kt_lds + kaddr[s] + kt * 32 * ROW_B),
                         qop[s], x[kt]);
  };
  auto pv = [&](LC_LDS const char* vt_lds) __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int jp = 0; jp < 2; ++jp)
#pragma unroll
        for (int dt = 0; dt < DTL; ++dt) {
          const int rowoff = (kt * 32 + jp * 16) * ROW_B;
          const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (LC_LDS i16x4_t*)(vt_lds + vaddr[0][dt] + rowoff));
          const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (LC_LDS i16x4_t*)(vt_lds + vaddr[1][dt] + rowoff));
          const i16x8_t both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          o[dt] = Ops::mma(__builtin_bit_cast(v8, both), pop[kt][jp], o[dt]);
          o[dt] = Ops::mma(__builtin_bit_cast(v8, both), rem[kt][jp], o[dt]);
        }
  };
  // Scores of tokens that are none are masked; rows without a reference max (only
  // before the first live tile) take the tile's.
  constexpr uint64_t kAll = NKT == 2 ? ~0ull : 0xffffffffull;
  auto prepare = [&](uint64_t live) __attribute__((always_inline)) {
    const uint64_t mine = (live >> (wk * 32)) & kAll;
    if (mine != kAll) {
      const uint64_t bits = mine >> (hh * 4);
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!((bits >> (kt * 32 + (r >> 2) * 8 + (r & 3))) & 1)) x[kt][r] = -INFINITY;
    }
    if (__ballot(m_ref == -INFINITY)) {
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, x[kt][r]);
      mx = pf_half_max(mx) * a.scale_log2;
      if (m_ref == -INFINITY) m_ref = mx;
    }
  };
  auto shift = [&]() __attribute__((always_inline)) {
    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) y[kt][r] = fmaf(x[kt][r], a.scale_log2, -m_use);
  };
  auto weigh = [&]() __attribute__((always_inline)) {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = lc_exp2(y[kt][r]), p1 = lc_exp2(y[kt][r + 1]);
        s0 += p0;
        s1 += p1;
        split_weights(p0, p1, pop[kt][r >> 3], rem[kt][r >> 3], r & 7);
      }
    l_tile = s0 + s1;
  };
  // A weight past 2^8 (then its lane's sum is too): the rows whose max grew move
  // their reference there, with O and l, and the tile is weighed again.
  auto settle = [&]() __attribute__((always_inline)) {
    if (__builtin_expect(__ballot(l_tile > 256.f) != 0, 0)) {
      float up = 0.f;
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) up = fmaxf(up, y[kt][r]);
      up = pf_half_max(up);
      const float alpha = lc_exp2(-up);
      l_lane *= alpha;
#pragma unroll
      for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
      m_ref += up;  // (a row without a finite score so far, up 0, stays without a reference)
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) y[kt][r] -= up;
      weigh();
    }
    l_lane += l_tile;
  };

  // Step t computes S of tile t + 1 beside the softmax and PV of tile t: K runs a
  // tile ahead of V. Its DMA (K of tile t + 2, V of t + 1) goes into the buffers that
  // step t - 1 read; the page entries of tile t + 3 are on their way.
  const int tb = it.t_begin;
  const int n_tiles = (it.t_end - tb + kTile - 1) / kTile;
  int pg3;             // page entries
  RowPlace at1, at2;   // of tiles t + 1 and t + 2
  uint64_t live1;
  {
    const int pg0 = fetch(tb), pg1 = fetch(tb + kTile), pg2 = fetch(tb + 2 * kTile);
    pg3 = fetch(tb + 3 * kTile);
    const RowPlace at0 = place(tb, pg0);
    at1 = place(tb + kTile, pg1);
    at2 = place(tb + 2 * kTile, pg2);
    issue(kp, at0, lds_k0);
    issue(vp, at0, lds_v0);
    if (n_tiles > 1) issue(kp, at1, lds_k1);
    const uint64_t live0 = __ballot(at0.bytes != 0);
    live1 = __ballot(at1.bytes != 0);
    pf_barrier<true>();
    qk(lds_k0);
    prepare(live0);
    shift();
  }
  auto step = [&](int t, LC_LDS char* kc, LC_LDS char* vc, LC_LDS char* kn, LC_LDS char* vn)
      __attribute__((always_inline)) {
    // Tiles K t + 1 and V t are in LDS; the other buffers' reads are done.
    pf_barrier<true>();
    const int t0 = tb + t * kTile;
    if (t + 2 < n_tiles) issue(kp, at2, kc);
    issue(vp, at1, vn);
    const uint64_t live = live1;
    at1 = at2;
    live1 = __ballot(at1.bytes != 0);
    at2 = place(t0 + 3 * kTile, pg3);
    pg3 = fetch(t0 + 4 * kTile);
    // One matrix instruction, its operands' reads LA ahead, and vector work.
    constexpr int NQ = NKT * KS, NP = NKT * 2 * DTL, LA = 4;
    qk(kn);
    weigh();
    __builtin_amdgcn_sched_group_barrier(0x100, LA, 0);
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (j + LA < NQ) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
    }
    settle();
    prepare(live);
    pv(vc);
    shift();
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * LA, 0);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (j + LA < NP) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
    }
  };
  int t = 0;
  for (; t + 2 < n_tiles; t += 2) {
    step(t, lds_k0, lds_v0, lds_k1, lds_v1);
    step(t + 1, lds_k1, lds_v1, lds_k0, lds_v0);
  }
  if (t + 1 < n_tiles) step(t, lds_k0, lds_v0, lds_k1, lds_v1);
  // The last tile.
  weigh();
  settle();
  pf_barrier<true>();
  pv(n_tiles & 1 ? lds_v0 : lds_v1);

  float l_tot = l_lane;
  {
    const unsigned u = __float_as_uint(l_lane);
    const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    l_tot = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  if constexpr (WR != 4) {
    // The second token half's state goes to the first half's wave: O in the K
    // buffers, [row tile][register][lane], then m and l.
    __syncthreads();
    LC_LDS float* rec = (LC_LDS float*)(wr == 0 ? lds_k0 : lds_k1);
    LC_LDS float* ml = (LC_LDS float*)lds_v0 + wr * 128;
    if (wk == 1) {
#pragma unroll
      for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) rec[(dt * 16 + r) * 64 + lane] = o[dt][r];
      ml[lane] = m_ref;
      ml[64 + lane] = l_tot;
    }
    __syncthreads();
    if (wk != 0) return;
    const float m2 = ml[lane], l2 = ml[64 + lane];
    const float m = fmaxf(m_ref, m2);
    const float w1 = m_ref == -INFINITY ? (l_tot == 0.f ? 0.f : 1.f) : lc_exp2(m_ref - m);
    const float w2 = m2 == -INFINITY ? (l2 == 0.f ? 0.f : 1.f) : lc_exp2(m2 - m);
    l_tot = l_tot * w1 + l2 * w2;
#pragma unroll
    for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = o[dt][r] * w1 + rec[(dt * 16 + r) * 64 + lane] * w2;
    m_ref = m;
  }
  if (!row_ok) return;
  const int64_t pidx = ((int64_t)b * a.Hq + h) * (a.p_splits + a.s_splits) + it.slot;
  const float inv_l = l_tot == 0.f ? 0.f : 1.0f / l_tot;
#pragma unroll
  for (int dt = 0; dt < DTL; ++dt) store_columns(a, pidx, dt, hh, o[dt], inv_l);
  if (hh == 0) put(a, a.part_lse + pidx, l_tot == 0.f ? -INFINITY : m_ref + lc_log2(l_tot));
}

// Up to 32 rows: bound by reading K and V, so the waves stream on their own, without
// barriers: groups of gw waves (1, 2 or 4) share a range, wave i of a group taking
// every gw-th 32-token step. `it` may be empty. A step's K and V rows
// are loaded into registers (16 KB in flight per wave, 8 waves on a CU) while the
// previous step computes from the wave's LDS. An instruction loads RPI token rows,
// which share a page (pages of a power of two from RPI up): a scalar base and one
// lane offset address it.
template <typename T, int DPAD>
__device__ __forceinline__ void shared_stream(const SharedArgs& a, const RangeItem& it, int gw,
                                              LC_LDS char* b0, LC_LDS char* b1, LC_LDS char* b2,
                                              LC_LDS char* b3, LC_LDS float* ml) {
  typedef Mfma32<T> Ops;
  typedef typename Ops::v8 v8;
  constexpr int KS = DPAD / 16, DTL = DPAD / 32, CPR = DPAD / 8;
  constexpr int RPI = 64 / CPR, NI = 32 / RPI;
  constexpr int ROW_B = DPAD * (int)sizeof(T);
  constexpr int kStep = 32;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wg = wave & (gw - 1);  // this wave in its group
  const int l32 = lane & 31, hh = lane >> 5;
  auto buffer = [&](int w) { return w == 0 ? b0 : w == 1 ? b1 : w == 2 ? b2 : b3; };
  LC_LDS char* lds_k = buffer(wave);
  LC_LDS char* lds_v = lds_k + kStep * ROW_B;

  const int r_abs = it.row0 + l32;
  const bool row_ok = r_abs < it.rows;
  const int r_safe = row_ok ? r_abs : it.row0;
  const int b = it.b0 + r_safe / a.G;
  const int h = it.kvh * a.G + r_safe % a.G;
  v8 qop[KS];
  load_rows<T, DPAD>(a, b, h, row_ok, hh, qop);

  const T* kp = static_cast<const T*>(a.kp) + (int64_t)it.kvh * a.s_head;
  const T* vp = static_cast<const T*>(a.vp) + (int64_t)it.kvh * a.s_head;
  const int last_page = (it.t_end - 1) >> a.p_shift;
  const int srow = lane / CPR, chunk = lane % CPR;
  const int lane_off =
      chunk * 8 < a.D ? static_cast<int>((srow * a.s_tok + chunk * 8) * sizeof(T)) : -16;
  // Page entry of token t + l32 (past the range: an entry that is not used).
  auto fetch = [&](int t) { return it.table[min((t + l32) >> a.p_shift, last_page)]; };
  auto place = [&](int t, int page) {
    return row_place<RPI>(a, page, t + l32, it.t_end, sizeof(T));
  };
  // Rows past the range, of invalid pages or past head_dim lie outside the
  // instruction's buffer and read zeros (which also keeps 0 x NaN out of the second
  // product); no branch separates the loads.
  u32x4_t sk[NI], sv[NI];
  auto issue = [&](const RowPlace& at) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      sk[i] = __builtin_amdgcn_raw_buffer_load_b128(row_buffer(kp, at, i * RPI), lane_off, 0, 2);
      sv[i] = __builtin_amdgcn_raw_buffer_load_b128(row_buffer(vp, at, i * RPI), lane_off, 0, 2);
    }
  };  // (2: non-temporal)

  int kaddr[KS], vaddr[2][DTL];
  operand_addresses<T, DPAD>(lane, 0, kaddr, vaddr);

  f32x16_t o[DTL];
#pragma unroll
  for (int i = 0; i < DTL; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  float m_ref = -INFINITY, l_lane = 0.f;

  const int t0 = it.t_begin + wg * kStep;
  const int next = gw * kStep;
  // (the places of a step's rows are found a step ahead of its loads, and its page
  // entries a step before that)
  RowPlace at_next{};
  int page_next = 0;
  uint32_t live_next = 0;
  if (t0 < it.t_end) {
    const int page = fetch(t0), page1 = fetch(t0 + next);
    page_next = fetch(t0 + 2 * next);
    const RowPlace at = place(t0, page);
    issue(at);
    live_next = static_cast<uint32_t>(__ballot(at.bytes != 0));
    at_next = place(t0 + next, page1);
  }
  for (int t = t0; t < it.t_end; t += next) {
    const uint32_t live = live_next;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = i * RPI + srow;
      const int at = row * ROW_B + ((chunk ^ pf_swz<CPR>(row)) << 4);
      *reinterpret_cast<LC_LDS u32x4_t*>(lds_k + at) = sk[i];
      *reinterpret_cast<LC_LDS u32x4_t*>(lds_v + at) = sv[i];
    }
    if (t + next < it.t_end) {
      issue(at_next);
      live_next = static_cast<uint32_t>(__ballot(at_next.bytes != 0));
      at_next = place(t + 2 * next, page_next);
      page_next = fetch(t + 3 * next);
    }
    lc_compiler_fence();
    if (live == 0) continue;

    f32x16_t x;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      x = Ops::mma(*reinterpret_cast<LC_LDS const v8*>(lds_k + kaddr[s]), qop[s], x);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= a.scale_log2;
    if (live != 0xffffffffu) {
      const uint32_t mine = live >> (hh * 4);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!((mine >> ((r >> 2) * 8 + (r & 3))) & 1)) x[r] = -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, x[r]);
    mx = pf_half_max(mx);
    if (__ballot(mx > m_ref + kSharedRescaleLog2)) {
      const float m_new = fmaxf(m_ref, mx);
      const float alpha = m_new == -INFINITY ? 1.f : lc_exp2(m_ref - m_new);
      l_lane *= alpha;
#pragma unroll
      for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
      m_ref = m_new;
    }
    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
    v8 pop[2], rem[2];
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const float p0 = lc_exp2(x[r] - m_use), p1 = lc_exp2(x[r + 1] - m_use);
      l_lane += p0;
      l_lane += p1;
      split_weights(p0, p1, pop[r >> 3], rem[r >> 3], r & 7);
    }
#pragma unroll
    for (int jp = 0; jp < 2; ++jp)
#pragma unroll
      for (int dt = 0; dt < DTL; ++dt) {
        const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (LC_LDS i16x4_t*)(lds_v + vaddr[0][dt] + jp * 16 * ROW_B));
        const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (LC_LDS i16x4_t*)(lds_v + vaddr[1][dt] + jp * 16 * ROW_B));
        const i16x8_t both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        o[dt] = Ops::mma(__builtin_bit_cast(v8, both), pop[jp], o[dt]);
        o[dt] = Ops::mma(__builtin_bit_cast(v8, both), rem[jp], o[dt]);
      }
    lc_compiler_fence();
  }

  float l;
  {
    const unsigned u = __float_as_uint(l_lane);
    const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  const int64_t pidx = ((int64_t)b * a.Hq + h) * (a.p_splits + a.s_splits) + it.slot;
  if (gw == 1) {
    if (!row_ok || it.t_begin >= it.t_end) return;
    const float inv_l = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int dt = 0; dt < DTL; ++dt) store_columns(a, pidx, dt, hh, o[dt], inv_l);
    if (hh == 0) a.part_lse[pidx] = l == 0.f ? -INFINITY : m_ref + lc_log2(l);
    return;
  }
  // Join the group's waves: each leaves O in its own buffer, [register][lane], and
  // takes every gw-th block of 32 columns of all of them.
  LC_LDS float* rec = (LC_LDS float*)lds_k;
#pragma unroll
  for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) rec[(dt * 16 + r) * 64 + lane] = o[dt][r];
  ml[wave * 128 + lane] = m_ref;
  ml[wave * 128 + 64 + lane] = l;
  __syncthreads();
  if (it.t_begin >= it.t_end) return;
  const int w0 = wave - wg;
  float m = -INFINITY;
  for (int w = w0; w < w0 + gw; ++w) m = fmaxf(m, ml[w * 128 + lane]);
  // (a wave without tokens has m = -inf, l = 0 and O = 0; NaN passes)
  auto weight = [&](int w) {
    const float mw = ml[w * 128 + lane], lw = ml[w * 128 + 64 + lane];
    return lw == 0.f ? 0.f : mw == -INFINITY ? 1.f : lc_exp2(mw - m);
  };
  l = 0.f;
  for (int w = w0; w < w0 + gw; ++w) l += ml[w * 128 + 64 + lane] * weight(w);
  const float inv_l = l == 0.f ? 0.f : 1.0f / l;
  for (int dt = wg; dt < DTL; dt += gw) {
    f32x16_t sum;
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.f;
    for (int w = w0; w < w0 + gw; ++w) {
      const float f = weight(w);
      LC_LDS const float* from = (LC_LDS const float*)buffer(w) + dt * 16 * 64 + lane;
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[r] += from[r * 64] * f;
    }
    if (row_ok) store_columns(a, pidx, dt, hh, sum, inv_l);
  }
  if (row_ok && wg == 0 && hh == 0)
    put(a, a.part_lse + pidx, l == 0.f ? -INFINITY : m + lc_log2(l));
}

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
        shared_range<T, DPAD, WR>(a, it, k0, k1, v0, v1);
      else
        shared_stream<T, DPAD>(a, it, 4, k0, k1, v0, v1, (LC_LDS float*)lds_ml);
    }
  } else {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    own_item(a, (id - p_blocks) * (4 / own_waves) + wave / own_waves, head_groups, it);
    if (own_waves < 4 || it.t_begin < it.t_end)
      shared_stream<T, DPAD>(a, it, own_waves, k0, k1, v0, v1, (LC_LDS float*)lds_ml);
  }
  if (a.counters != nullptr) join_last<T>(a, it.b0 / a.W, it.kvh);
}

// ---------------------------------------------------------------------------
// fp32 on v_mfma_f32_32x32x2_f32 (head_dim a multiple of 4 up to 128, pages of a
// power of two from 8 up): 32 rows per workgroup, whose 4 waves take every fourth
// 32-token step of the range and are joined through LDS. Operands come straight
// from global memory into registers, in the forms of attn_f32.h: a K row per lane,
// at the lane's own address; V rows in groups of 8 tokens, which share a page.
// Bound by the fp32 matrix rate where rows fill the tile, else by the start and the
// latency of few steps.
// ---------------------------------------------------------------------------
template <int DPAD>
__device__ __forceinline__ void shared_f32_range(const SharedArgs& a, const RangeItem& it) {
  constexpr int DTL = DPAD / 32, LD = DPAD + 4, NC = DPAD / 8;
  __shared__ __align__(16) float slab[4][32 * LD];
  __shared__ float ms[4][32], ls[4][32];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const int r_abs = it.row0 + l32;
  const bool row_ok = r_abs < it.rows;
  F32Row<DPAD> q, k;
  {
    const int r = row_ok ? r_abs : it.row0;
    const float* qh = static_cast<const float*>(a.q) + (int64_t)(it.b0 + r / a.G) * a.q_sb +
                      (int64_t)(it.kvh * a.G + r % a.G) * a.q_sh;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int d = i * 8 + hh * 4;
      const bool ok = row_ok && d < a.D;
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(qh + (ok ? d : 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) q.c[i][e] = ok ? x[e] : 0.f;
    }
  }
  const float* kp = static_cast<const float*>(a.kp) + (int64_t)it.kvh * a.s_head;
  const float* vp = static_cast<const float*>(a.vp) + (int64_t)it.kvh * a.s_head;
  const int last_page = (it.t_end - 1) >> a.p_shift;
  auto fetch = [&](int t) { return it.table[min((t + l32) >> a.p_shift, last_page)]; };
  auto place = [&](int t, int page) { return row_place<8>(a, page, t + l32, it.t_end, 4); };
  auto load_k = [&](const RowPlace& at) {
    const char* row = reinterpret_cast<const char*>(kp) +
                      ((static_cast<uint64_t>(at.hi) << 32) | at.lo) + hh * 16;
    const char* none = reinterpret_cast<const char*>(shared_zeros);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const bool ok = at.bytes != 0 && i * 8 + hh * 4 < a.D;
      k.c[i] = *reinterpret_cast<const f32x4_t*>(ok ? row + i * 32 : none);
    }
  };
  const int row_b = static_cast<int>(a.s_tok * 4);
  const int v_off = l32 * DTL < a.D ? 4 * hh * row_b + l32 * DTL * 4 : kF32Oob;

  f32x16_t o[DTL];
#pragma unroll
  for (int dt = 0; dt < DTL; ++dt) f32_zero(o[dt]);
  float m = -INFINITY, l = 0.f;
  constexpr int kNext = 4 * 32;
  const int t0 = it.t_begin + wave * 32;
  RowPlace at{};
  int page_next = 0;
  if (t0 < it.t_end) {
    const int page = fetch(t0);
    page_next = fetch(t0 + kNext);
    at = place(t0, page);
    load_k(at);
  }
  for (int t = t0; t < it.t_end; t += kNext) {
    const uint32_t live = static_cast<uint32_t>(__ballot(at.bytes != 0));
    F32Cols<DTL> v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __amdgpu_buffer_rsrc_t rs = row_buffer(vp, at, j * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v.n[j * 4 + i] = f32_load_dims<DTL>(
            rs, static_cast<int>(static_cast<unsigned>(v_off) + static_cast<unsigned>(i * row_b)));
    }
    __builtin_amdgcn_sched_barrier(0);
    f32x16_t s;
    f32_zero(s);
    f32_dot<DPAD>(s, k, q);
    at = place(t + kNext, page_next);
    page_next = fetch(t + 2 * kNext);
    load_k(at);
    __builtin_amdgcn_sched_barrier(0);
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] *= a.scale_log2;
      if (live != 0xffffffffu && !((live >> (8 * (r >> 2) + 4 * hh + (r & 3))) & 1))
        s[r] = -INFINITY;
      mx = fmaxf(mx, s[r]);
    }
    const float m_new = fmaxf(m, pf_half_max(mx));
    if (__ballot(m_new > m) != 0) {
      const float alpha = m_new == -INFINITY ? 1.f : lc_exp2(m - m_new);
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
      m = m_new;
    }
    const float m_use = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = lc_exp2(s[r] - m_use);
      l += s[r];
    }
    f32_outer<DTL>(o, v, s);
  }

  l += __shfl_xor(l, 32, 64);
  f32_put<DPAD>(slab[wave], o, l32, hh);
  if (hh == 0) {
    ms[wave][l32] = m;
    ls[wave][l32] = l;
  }
  __syncthreads();
  constexpr int CPR = DPAD / 4;
#pragma unroll
  for (int e = tid; e < 32 * CPR; e += 256) {
    const int row = e / CPR, d = (e - row * CPR) * 4, r = it.row0 + row;
    if (r >= it.rows || d >= a.D) continue;
    float mt = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, ms[w][row]);
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // (a wave without tokens has m = -inf, l = 0 and O = 0; NaN passes)
      const float mw = ms[w][row], lw = ls[w][row];
      const float f = lw == 0.f ? 0.f : mw == -INFINITY ? 1.f : lc_exp2(mw - mt);
      lt = fmaf(lw, f, lt);
      const f32x4_t ow = *reinterpret_cast<const f32x4_t*>(&slab[w][row * LD + d]);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(ow[i], f, acc[i]);
    }
    const float inv = lt == 0.f ? 0.f : 1.0f / lt;
    const int b = it.b0 + r / a.G, h = it.kvh * a.G + r % a.G;
    const int64_t pidx = ((int64_t)b * a.Hq + h) * (a.p_splits + a.s_splits) + it.slot;
    f32x4_t out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = acc[i] * inv;
    put4(a, a.part_o + pidx * a.D + d, out);
    if (d == 0) put(a, a.part_lse + pidx, lt == 0.f ? -INFINITY : mt + lc_log2(lt));
  }
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
  if (it.t_begin < it.t_end) shared_f32_range<DPAD>(a, it);
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
