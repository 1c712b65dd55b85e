// Building blocks of attention from several query rows that share a kv head to tokens
// named by a table row: the rows of a group of sequences that share a prefix, or the
// newest tokens of one sequence.
//
// A is the kernel's arguments: kp, vp, s_page, s_head, s_tok, num_pages, P (a power of
// two), p_shift, D, scale_log2. Item is a range of tokens and a tile of rows:
//   table, kvh, t_begin, t_end   the tokens
//   row0, rows                   the rows row0 .. of `rows` in all
//   query<T>(a, r)               a row's query
//   row(a, r)                    the place of its results, to which
//   store4(a, row, d, x), store_lse(a, row, x)
//                                write 4 of its normalised outputs and its log2 logsumexp
//   kCausal                      whether the rows see unequal numbers of tokens: then
//   limit(a, r), all_see         row r sees those before limit(a, r), and every row that
//                                sees any sees those before all_see; `scratch` is 512 floats
//                                of LDS for each wave
#pragma once

#include <type_traits>

#include "attn_f32.h"
#include "attn_tiles.h"
#include "lc_common.h"

namespace lc_attn {

constexpr int kTile = 64;  // tokens per tile
constexpr float kPagedRescaleLog2 = 8.0f;

__device__ __attribute__((aligned(16))) const uint32_t paged_zeros[4] = {0, 0, 0, 0};

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

// Where the token of each lane lies: its byte offset in the pools, and the bytes of
// the RPI rows from it on that hold tokens of the range (0: none, or an invalid
// page). One lane's answer serves a whole DMA instruction, by v_readlane: computed
// by all lanes at once, it costs a few instructions per tile instead of a 64-bit
// scalar product and its branches per DMA instruction.
struct RowPlace {
  uint32_t lo, hi;
  int bytes;
};
template <int RPI, typename A>
__device__ __forceinline__ RowPlace row_place(const A& a, int page, int tok, int t_end,
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
__device__ __forceinline__ void load_query(const T* qh, int D, bool row_ok, int hh,
                                           typename Mfma32<T>::v8 (&qop)[DPAD / 16]) {
  typedef typename Mfma32<T>::v8 v8;
  constexpr int CPR = DPAD / 8;
#pragma unroll
  for (int s = 0; s < DPAD / 16; ++s) {
    const int d0 = (hh * (CPR / 2) + s) * 8;
    const bool ok = row_ok && d0 < D;
    const v8 x = *reinterpret_cast<const v8*>(qh + (ok ? d0 : 0));
    qop[s] = ok ? x : v8{};
  }
}

// LDS addresses of a tile's operands from token row0 (a multiple of 32) on (rows of
// DPAD, chunks swizzled by pf_swz): k(s), K rows of step s for S^T; v(jj, dt), V columns
// of block dt and tokens 8 jj on for O^T by transposed reads. They differ from the first
// ones in bits that the swizzle and the tokens' rows leave to themselves. kMade: made
// anew where they are used, since their registers would take the place of query operands,
// and one of those read back from scratch waits for all loads in flight (newest tokens,
// 32 sequences of 4096 at 8 kv heads: 109 us, 91 so; shared prefixes, whose kernel keeps
// its operands anyway, take 5-10% longer with many rows).
template <typename T, int DPAD, bool kMade>
struct Operands {
  static constexpr int CPR = DPAD / 8, ROW_B = DPAD * (int)sizeof(T);
  static constexpr int KS = DPAD / 16, DTL = DPAD / 32;
  int k_at[kMade ? 1 : KS], v_at[kMade ? 1 : 2 * DTL];

  __device__ __forceinline__ Operands(int lane, int row0) {
    const int l32 = lane & 31, hh = lane >> 5;
    const int k0 = (row0 + l32) * ROW_B + (((hh * (CPR / 2)) ^ pf_swz<CPR>(l32)) << 4);
    const int gq = lane >> 4, te = (lane & 15) >> 2, tc = lane & 3;
    const int kr = hh * 4 + te, d = (gq & 1) * 16 + 4 * tc;
    const int v0 =
        (row0 + kr) * ROW_B + ((((d >> 3) ^ pf_swz<CPR>(kr)) << 4) | ((d & 7) * (int)sizeof(T)));
#pragma unroll
    for (int s = 0; s < (kMade ? 1 : KS); ++s) k_at[s] = k0 ^ (s << 4);
#pragma unroll
    for (int i = 0; i < (kMade ? 1 : 2 * DTL); ++i) v_at[i] = v0 ^ v_bits(i / DTL, i % DTL);
  }
  static __device__ __forceinline__ int v_bits(int jj, int dt) {
    return dt << 6 | (jj ? 8 * ROW_B | 32 : 0);
  }
  // Before a use of k or v: not made earlier than here.
  __device__ __forceinline__ void fresh_k() {
    if constexpr (kMade) __asm__("" : "+v"(k_at[0]));
  }
  __device__ __forceinline__ void fresh_v() {
    if constexpr (kMade) __asm__("" : "+v"(v_at[0]));
  }
  __device__ __forceinline__ int k(int s) const { return kMade ? k_at[0] ^ (s << 4) : k_at[kMade ? 0 : s]; }
  __device__ __forceinline__ int v(int jj, int dt) const {
    return kMade ? v_at[0] ^ v_bits(jj, dt) : v_at[kMade ? 0 : jj * DTL + dt];
  }
};

// Writes columns dt * 32 .. of a row's output.
template <typename A, typename Item, typename Row>
__device__ __forceinline__ void store_columns(const A& a, const Item& it, const Row& row, int dt,
                                              int hh, const f32x16_t& o, float inv_l) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d0 = dt * 32 + j * 8 + hh * 4;
    if (d0 < a.D) {  // (D % 8 == 0: whole groups of 4)
      f32x4_t w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = o[j * 4 + e] * inv_l;
      it.store4(a, row, d0, w);
    }
  }
}

// The low n bits (0 to 64).
__device__ __forceinline__ uint64_t low_bits(int n) {
  return n >= 64 ? ~0ull : n <= 0 ? 0 : (1ull << n) - 1;
}

// Whether any value of `bytes` (a multiple of 1024) of this wave's part of a V tile is
// infinite or NaN.
template <typename T>
__device__ __forceinline__ bool tile_nonfinite(LC_LDS const char* v, int bytes, int lane) {
  constexpr uint32_t kExp = std::is_same_v<T, bf16_t> ? 0x7f807f80u : 0x7c007c00u;
  uint32_t bad = 0;
  for (int at = lane * 16; at < bytes; at += 1024) {
    const u32x4_t x = *reinterpret_cast<LC_LDS const u32x4_t*>(v + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t z = (x[e] & kExp) ^ kExp;  // a half of 0: exponent bits all set
      bad |= (z - 0x00010001u) & ~z;
    }
  }
  return __ballot((bad & 0x80008000u) != 0) != 0;
}

// O += P V of 16 tokens, token by token, so that a token has a part in the rows that
// see it alone (bit t of `seen`: the lane's row sees token t): a matrix product would
// make 0 times an infinite V of the others NaN. Rare, so a rolled loop: the weights, whole
// + rest, go through 512 floats of this wave's LDS.
template <typename T, int DPAD>
__device__ __forceinline__ void add_tokens(f32x16_t (&o)[DPAD / 32],
                                           const typename Mfma32<T>::v8& whole,
                                           const typename Mfma32<T>::v8& rest,
                                           LC_LDS const char* v, int row0, uint32_t seen, int lane,
                                           LC_LDS float* scratch) {
  constexpr int CPR = DPAD / 8, ROW_B = DPAD * (int)sizeof(T);
  const int hh = lane >> 5;
#pragma unroll
  for (int r = 0; r < 8; ++r)
    scratch[r * 64 + lane] = static_cast<float>(whole[r]) + static_cast<float>(rest[r]);
  lc_compiler_fence();
#pragma unroll 1
  for (int n = 0; n < 16; ++n) {
    // (register r of the wave's two halves: tokens 4 apart)
    const int half = n & 1, r = n >> 1, tok = (r >> 2) * 8 + half * 4 + (r & 3), row = row0 + tok;
    const float w = scratch[r * 64 + (lane & 31) + half * 32];
    const bool sees = (seen >> tok) & 1;
#pragma unroll
    for (int dt = 0; dt < DPAD / 32; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = dt * 32 + j * 8 + hh * 4;
        typedef T t4 __attribute__((ext_vector_type(4)));
        const t4 x = *reinterpret_cast<LC_LDS const t4*>(
            v + row * ROW_B + (((d >> 3) ^ pf_swz<CPR>(row)) << 4) + (d & 7) * (int)sizeof(T));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[dt][j * 4 + e] = sees ? fmaf(w, static_cast<float>(x[e]), o[dt][j * 4 + e]) : o[dt][j * 4 + e];
      }
  }
  lc_compiler_fence();
}

// A row that has seen nothing is 0, whatever the tokens that others see left in it.
template <int N>
__device__ __forceinline__ void clear_unseen(f32x16_t (&o)[N], float l) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = l == 0.f ? 0.f : o[i][r];
}

// More than 32 rows: tiles of 64 tokens go through LDS (double-buffered, by DMA), which
// the workgroup's 4 waves share: with 128 rows (WR 4) each has 32 rows and all tokens,
// with 64 rows 32 tokens, and the token halves' softmax states are joined through LDS at
// the end.
template <typename T, int DPAD, int WR, typename A, typename Item>
__device__ __forceinline__ void paged_range(const A& a, const Item& it, LC_LDS char* lds_k0,
                                            LC_LDS char* lds_k1, LC_LDS char* lds_v0,
                                            LC_LDS char* lds_v1, LC_LDS float* scratch = nullptr) {
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
  v8 qop[KS];
  load_query<T, DPAD>(it.template query<T>(a, r_safe), a.D, row_ok, hh, qop);
  // Tokens that this lane's row sees.
  int lim = 0, all_see = 0;
  if constexpr (Item::kCausal) {
    lim = row_ok ? it.limit(a, r_abs) : 0;
    all_see = it.all_see;
  }

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
  Operands<T, DPAD, Item::kCausal> at_lds(lane, wk * 32);

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
    at_lds.fresh_k();
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) x[kt][r] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
        x[kt] = Ops::mma(*reinterpret_cast<LC_LDS const v8*>(kt_lds + at_lds.k(s) + kt * 32 * ROW_B),
                         qop[s], x[kt]);
  };
  auto pv = [&](LC_LDS const char* vt_lds) __attribute__((always_inline)) {
    at_lds.fresh_v();
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int jp = 0; jp < 2; ++jp)
#pragma unroll
        for (int dt = 0; dt < DTL; ++dt) {
          const int rowoff = (kt * 32 + jp * 16) * ROW_B;
          const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (LC_LDS i16x4_t*)(vt_lds + at_lds.v(0, dt) + rowoff));
          const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (LC_LDS i16x4_t*)(vt_lds + at_lds.v(1, dt) + rowoff));
          const i16x8_t both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          o[dt] = Ops::mma(__builtin_bit_cast(v8, both), pop[kt][jp], o[dt]);
          o[dt] = Ops::mma(__builtin_bit_cast(v8, both), rem[kt][jp], o[dt]);
        }
  };
  // A tile that some rows see in part, with an infinite or NaN V.
  auto by_token = [&](int t0, LC_LDS const char* vt_lds, auto part) __attribute__((always_inline)) {
    if constexpr (part)
      return t0 + kTile > all_see &&
             tile_nonfinite<T>(vt_lds + wk * 32 * ROW_B, NKT * 32 * ROW_B, lane);
    else
      return false;
  };
  auto add_all = [&](int t0, LC_LDS const char* vt_lds) __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
      const int first = wk * 32 + kt * 32;
#pragma unroll
      for (int jp = 0; jp < 2; ++jp)
        add_tokens<T, DPAD>(o, pop[kt][jp], rem[kt][jp], vt_lds, first + jp * 16,
                            static_cast<uint32_t>(low_bits(lim - (t0 + first + jp * 16))), lane,
                            scratch + wave * 512);
    }
  };
  // Scores of tokens that are none are masked; rows without a reference max (only
  // before the first live tile) take the tile's.
  constexpr uint64_t kAll = NKT == 2 ? ~0ull : 0xffffffffull;
  auto prepare = [&](uint64_t live, int t0, auto part) __attribute__((always_inline)) {
    uint64_t mine = (live >> (wk * 32)) & kAll;
    const bool some = mine != kAll || part;
    if constexpr (part) mine &= low_bits(lim - (t0 + wk * 32));
    if (some) {
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
    prepare(live0, tb, std::bool_constant<Item::kCausal>());
    shift();
  }
  // `part`: not all rows that see any of tiles t and t + 1 may see all of them.
  auto step = [&](int t, LC_LDS char* kc, LC_LDS char* vc, LC_LDS char* kn, LC_LDS char* vn,
                  auto part) __attribute__((always_inline)) {
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
    prepare(live, t0 + kTile, part);
    if (__builtin_expect(by_token(t0, vc, part), 0)) {
      add_all(t0, vc);
      shift();
      return;
    }
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
  const std::bool_constant<Item::kCausal> some_part;
  int t = 0;
  if constexpr (Item::kCausal) {
    const int n_all = min(n_tiles, max(0, all_see - tb) / kTile);
    for (; t + 2 < n_all; t += 2) {
      step(t, lds_k0, lds_v0, lds_k1, lds_v1, std::false_type());
      step(t + 1, lds_k1, lds_v1, lds_k0, lds_v0, std::false_type());
    }
  }
  for (; __builtin_expect(t + 2 < n_tiles, !Item::kCausal); t += 2) {
    step(t, lds_k0, lds_v0, lds_k1, lds_v1, some_part);
    step(t + 1, lds_k1, lds_v1, lds_k0, lds_v0, some_part);
  }
  if (t + 1 < n_tiles) step(t, lds_k0, lds_v0, lds_k1, lds_v1, some_part);
  // The last tile.
  weigh();
  settle();
  pf_barrier<true>();
  {
    LC_LDS char* vt = n_tiles & 1 ? lds_v0 : lds_v1;
    const int t0 = tb + (n_tiles - 1) * kTile;
    if (__builtin_expect(by_token(t0, vt, some_part), 0))
      add_all(t0, vt);
    else
      pv(vt);
  }

  float l_tot = l_lane;
  {
    const unsigned u = __float_as_uint(l_lane);
    const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    l_tot = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  if constexpr (Item::kCausal)
    if (lim <= 0) l_tot = 0.f;
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
    // (by l first: a row that sees nothing has l = 0 and any reference, +inf among them; NaN
    // passes)
    const float w1 = l_tot == 0.f ? 0.f : m_ref == -INFINITY ? 1.f : lc_exp2(m_ref - m);
    const float w2 = l2 == 0.f ? 0.f : m2 == -INFINITY ? 1.f : lc_exp2(m2 - m);
    l_tot = l_tot * w1 + l2 * w2;
#pragma unroll
    for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = o[dt][r] * w1 + rec[(dt * 16 + r) * 64 + lane] * w2;
    m_ref = m;
  }
  if (!row_ok) return;
  const auto row = it.row(a, r_abs);
  const float inv_l = l_tot == 0.f ? 0.f : 1.0f / l_tot;
  if constexpr (Item::kCausal) clear_unseen(o, l_tot);
#pragma unroll
  for (int dt = 0; dt < DTL; ++dt) store_columns(a, it, row, dt, hh, o[dt], inv_l);
  if (hh == 0) it.store_lse(a, row, l_tot == 0.f ? -INFINITY : m_ref + lc_log2(l_tot));
}

// Up to 32 rows: bound by reading K and V, so the waves stream on their own, without
// barriers: groups of gw waves (1, 2 or 4) share a range, wave i of a group taking
// every gw-th 32-token step. `it` may be empty. A step's K and V rows
// are loaded into registers (16 KB in flight per wave, 8 waves on a CU) while the
// previous step computes from the wave's LDS. An instruction loads RPI token rows,
// which share a page (pages of a power of two from RPI up): a scalar base and one
// lane offset address it.
template <typename T, int DPAD, typename A, typename Item>
__device__ __forceinline__ void paged_stream(const A& a, const Item& it, int gw, LC_LDS char* b0,
                                             LC_LDS char* b1, LC_LDS char* b2, LC_LDS char* b3,
                                             LC_LDS float* ml, LC_LDS float* scratch = nullptr) {
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
  v8 qop[KS];
  load_query<T, DPAD>(it.template query<T>(a, r_safe), a.D, row_ok, hh, qop);
  // Tokens that this lane's row sees.
  int lim = 0;
  if constexpr (Item::kCausal) lim = row_ok ? it.limit(a, r_abs) : 0;

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

  Operands<T, DPAD, Item::kCausal> at_lds(lane, 0);

  f32x16_t o[DTL];
#pragma unroll
  for (int i = 0; i < DTL; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  float m_ref = -INFINITY, l_lane = 0.f;

  int t0 = it.t_begin + wg * kStep, t_end = it.t_end, next = gw * kStep;
  if constexpr (Item::kCausal) {
    // (a wave's tokens in one run)
    const int steps = max(0, it.t_end - it.t_begin + kStep - 1) / kStep;
    t0 = it.t_begin + wg * steps / gw * kStep;
    t_end = min(it.t_end, it.t_begin + (wg + 1) * steps / gw * kStep);
    next = kStep;
  }
  // (the places of a step's rows are found a step ahead of its loads, and its page
  // entries a step before that)
  RowPlace at_next{};
  int page_next = 0;
  uint32_t live_next = 0;
  if (t0 < t_end) {
    const int page = fetch(t0), page1 = fetch(t0 + next);
    page_next = fetch(t0 + 2 * next);
    const RowPlace at = place(t0, page);
    issue(at);
    live_next = static_cast<uint32_t>(__ballot(at.bytes != 0));
    at_next = place(t0 + next, page1);
  }
  // A step; `part`: not all rows that see any of its tokens may see all of them.
  auto step = [&](int t, auto part) __attribute__((always_inline)) {
    const uint32_t live = live_next;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = i * RPI + srow;
      const int at = row * ROW_B + ((chunk ^ pf_swz<CPR>(row)) << 4);
      *reinterpret_cast<LC_LDS u32x4_t*>(lds_k + at) = sk[i];
      *reinterpret_cast<LC_LDS u32x4_t*>(lds_v + at) = sv[i];
    }
    if (t + next < t_end) {
      issue(at_next);
      live_next = static_cast<uint32_t>(__ballot(at_next.bytes != 0));
      at_next = place(t + 2 * next, page_next);
      page_next = fetch(t + 3 * next);
    }
    lc_compiler_fence();
    if (live == 0) return;

    at_lds.fresh_k();
    at_lds.fresh_v();
    f32x16_t x;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      x = Ops::mma(*reinterpret_cast<LC_LDS const v8*>(lds_k + at_lds.k(s)), qop[s], x);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= a.scale_log2;
    uint32_t sees = live;
    if constexpr (part) sees &= static_cast<uint32_t>(low_bits(lim - t));
    if (part || live != 0xffffffffu) {
      const uint32_t mine = sees >> (hh * 4);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!((mine >> ((r >> 2) * 8 + (r & 3))) & 1)) x[r] = -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, x[r]);
    mx = pf_half_max(mx);
    if (__ballot(mx > m_ref + kPagedRescaleLog2)) {
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
    bool by_token = false;
    if constexpr (part) by_token = tile_nonfinite<T>(lds_v, kStep * ROW_B, lane);
    if (__builtin_expect(by_token, 0)) {
#pragma unroll
      for (int jp = 0; jp < 2; ++jp)
        add_tokens<T, DPAD>(o, pop[jp], rem[jp], lds_v, jp * 16, sees >> (jp * 16), lane,
                            scratch + wave * 512);
    } else {
#pragma unroll
      for (int jp = 0; jp < 2; ++jp)
#pragma unroll
        for (int dt = 0; dt < DTL; ++dt) {
          const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (LC_LDS i16x4_t*)(lds_v + at_lds.v(0, dt) + jp * 16 * ROW_B));
          const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (LC_LDS i16x4_t*)(lds_v + at_lds.v(1, dt) + jp * 16 * ROW_B));
          const i16x8_t both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          o[dt] = Ops::mma(__builtin_bit_cast(v8, both), pop[jp], o[dt]);
          o[dt] = Ops::mma(__builtin_bit_cast(v8, both), rem[jp], o[dt]);
        }
    }
    lc_compiler_fence();
  };
  int t = t0;
  int t_all = t_end;
  if constexpr (Item::kCausal) t_all = min(t_all, it.all_see - kStep + 1);
  for (; t < t_all; t += next) step(t, std::false_type());
  if constexpr (Item::kCausal)
    for (; __builtin_expect(t < t_end, 0); t += next) step(t, std::true_type());

  float l;
  {
    const unsigned u = __float_as_uint(l_lane);
    const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  if constexpr (Item::kCausal) {
    if (lim <= 0) l = 0.f;
    clear_unseen(o, l);
  }
  const auto row = it.row(a, r_safe);
  if (gw == 1) {
    if (!row_ok || it.t_begin >= it.t_end) return;
    const float inv_l = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int dt = 0; dt < DTL; ++dt) store_columns(a, it, row, dt, hh, o[dt], inv_l);
    if (hh == 0) it.store_lse(a, row, l == 0.f ? -INFINITY : m_ref + lc_log2(l));
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
    if (row_ok) store_columns(a, it, row, dt, hh, sum, inv_l);
  }
  if (row_ok && wg == 0 && hh == 0)
    it.store_lse(a, row, l == 0.f ? -INFINITY : m + lc_log2(l));
}

// ---------------------------------------------------------------------------
// fp32 on v_mfma_f32_32x32x2_f32 (head_dim a multiple of 4 up to 128, pages of a
// power of two from 8 up): 32 rows per workgroup, whose 4 waves take every fourth
// 32-token step of the range and are joined through LDS. Operands come straight
// from global memory into registers, in the forms of attn_f32.h: a K row per lane,
// at the lane's own address; V rows in groups of 8 tokens, which share a page.
// Bound by the fp32 matrix rate where rows fill the tile, else by the start and the
// latency of few steps. As the newest tokens' kernel, 16/8 heads of 64: 16 sequences of 4096
// tokens, 5 queries (10 of 32 rows used) 62 us, 4.3 TB/s; 2 of 4000, 128 queries 60 us, 69
// TFLOP/s of the 153 of a large product. In both the matrix units are busy half the time:
// one wave a SIMD, whose softmax has no other wave's matrix work beside it.
// ---------------------------------------------------------------------------
template <int DPAD, typename A, typename Item>
__device__ __forceinline__ void paged_f32_range(const A& a, const Item& it) {
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
    const float* qh = it.template query<float>(a, row_ok ? r_abs : it.row0);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int d = i * 8 + hh * 4;
      const bool ok = row_ok && d < a.D;
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(qh + (ok ? d : 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) q.c[i][e] = ok ? x[e] : 0.f;
    }
  }
  int lim = 0;
  if constexpr (Item::kCausal) lim = row_ok ? it.limit(a, r_abs) : 0;
  const float* kp = static_cast<const float*>(a.kp) + (int64_t)it.kvh * a.s_head;
  const float* vp = static_cast<const float*>(a.vp) + (int64_t)it.kvh * a.s_head;
  const int last_page = (it.t_end - 1) >> a.p_shift;
  auto fetch = [&](int t) { return it.table[min((t + l32) >> a.p_shift, last_page)]; };
  auto place = [&](int t, int page) { return row_place<8>(a, page, t + l32, it.t_end, 4); };
  auto load_k = [&](const RowPlace& at) {
    const char* row = reinterpret_cast<const char*>(kp) +
                      ((static_cast<uint64_t>(at.hi) << 32) | at.lo) + hh * 16;
    const char* none = reinterpret_cast<const char*>(paged_zeros);
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
    uint32_t live = static_cast<uint32_t>(__ballot(at.bytes != 0));
    const RowPlace here = at;
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
    bool ahead = false;  // some rows see the step's tokens in part
    if constexpr (Item::kCausal) {
      ahead = t + 32 > it.all_see;
      if (ahead) live &= static_cast<uint32_t>(low_bits(lim - t));
    }
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
    bool by_token = false;
    if constexpr (Item::kCausal) by_token = ahead && v.any_nonfinite();
    if (__builtin_expect(by_token, 0)) {
      // Token by token, as add_tokens.
      float* p = slab[wave];
#pragma unroll
      for (int r = 0; r < 16; ++r) p[(8 * (r >> 2) + 4 * hh + (r & 3)) * 33 + l32] = s[r];
      lc_compiler_fence();
#pragma unroll 1
      for (int n = 0; n < 32; ++n) {
        const float w = p[n * 33 + l32];
        const bool sees = (live >> n) & 1;
        const __amdgpu_buffer_rsrc_t rs = row_buffer(vp, here, n);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = (8 * (r >> 2) + 4 * hh + (r & 3)) * DTL;
          const F32Dims<DTL> x = f32_load_dims<DTL>(rs, d < a.D ? d * 4 : kF32Oob);
#pragma unroll
          for (int dt = 0; dt < DTL; ++dt) o[dt][r] = sees ? fmaf(x.v[dt], w, o[dt][r]) : o[dt][r];
        }
      }
      lc_compiler_fence();
    } else {
      f32_outer<DTL>(o, v, s);
    }
  }

  l += __shfl_xor(l, 32, 64);
  if constexpr (Item::kCausal) {
    if (lim <= 0) l = 0.f;
    clear_unseen(o, l);
  }
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
    f32x4_t out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = acc[i] * inv;
    const auto place = it.row(a, r);
    it.store4(a, place, d, out);
    if (d == 0) it.store_lse(a, place, lt == 0.f ? -INFINITY : mt + lc_log2(lt));
  }
}

}  // namespace lc_attn
