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
// the workspace, and a merge launch joins them.
#include <math.h>

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
};

// Tokens of a range are a multiple of this.
constexpr int kSharedStep = 64;

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
      wsum += w;
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
          if (j0 + jj < n && wj != 0.f) {
#pragma unroll
            for (int e = 0; e < VPL; ++e) acc[e] = fmaf(wj, v[jj][e], acc[e]);
          }
        }
      }
    }
  }
  wsum = lc_wave_sum(wsum);
  const float inv = wsum == 0.f ? 0.f : 1.0f / wsum;
  T* oh = out + (int64_t)b * o_sb + (int64_t)h * o_sh;
#pragma unroll
  for (int e = 0; e < VPL; ++e)
    if (d0 + e < a.D) oh[d0 + e] = lc_from_f32<T>(acc[e] * inv);
  if (lse_out != nullptr && lane == 0)
    lse_out[(int64_t)b * a.Hq + h] = wsum == 0.f ? -INFINITY : (mx + lc_log2(wsum)) * kLn2;
}

struct SharedPlan {
  int p_splits, s_splits;
};

// Ranges per prefix and per sequence: about one round of the CUs over all
// tokens, no range shorter than two steps.
SharedPlan shared_plan(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t p_cap,
                       int64_t s_cap) {
  const int64_t G = Hq / Hkv, W = B / N;
  const int64_t up = N * Hkv * lc_cdiv(W * G, 128), us = B * Hkv * lc_cdiv(G, 32);
  const int64_t total = up * p_cap + us * s_cap;
  int64_t each = lc_cdiv(total, lc_cu_count());
  if (each < 2 * kSharedStep) each = 2 * kSharedStep;
  auto splits = [&](int64_t cap) -> int {
    if (cap == 0) return 0;
    const int64_t s = lc_cdiv(cap, each);
    return static_cast<int>(s < 64 ? s : 64);
  };
  return SharedPlan{splits(p_cap), splits(s_cap)};
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

template <typename T>
int launch_shared(const SharedArgs& a, void* out, int64_t o_sb, int64_t o_sh, float* lse,
                  hipStream_t st) {
  const int splits = a.p_splits + a.s_splits;
  if (splits > 0) {
    shared_generic_kernel<T><<<dim3(splits, a.Hq, a.B), 64, 0, st>>>(a);
    const int rc = lc_check_launch("lc_shared_prefix_decode_fwd (generic)");
    if (rc != LC_OK) return rc;
  }
  return launch_merge<T>(a, out, o_sb, o_sh, lse, st);
}

}  // namespace

extern "C" {

int64_t lc_shared_prefix_decode_workspace_bytes(int64_t B, int64_t groups, int64_t Hq, int64_t Hkv,
                                                int64_t D, int64_t prefix_capacity,
                                                int64_t own_capacity) {
  if (B < 0 || groups <= 0 || B % groups != 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || D <= 0 ||
      prefix_capacity < 0 || own_capacity < 0)
    return -1;
  return shared_bytes(B * Hq, D, shared_plan(B, groups, Hq, Hkv, prefix_capacity, own_capacity));
}

int lc_shared_prefix_decode_fwd(const void* q, int64_t q_sb, int64_t q_sh, const void* key_pages,
                                const void* value_pages, int64_t kv_s_page, int64_t kv_s_head,
                                int64_t kv_s_tok, int64_t num_pages, const int32_t* prefix_table,
                                int64_t pt_stride, int64_t max_prefix_pages,
                                const int32_t* prefix_lens, const int32_t* block_table,
                                int64_t bt_stride, int64_t max_pages_per_seq,
                                const int32_t* seq_lens, void* out, int64_t o_sb, int64_t o_sh,
                                float* lse, void* workspace, int64_t workspace_bytes, int64_t B,
                                int64_t groups, int64_t Hq, int64_t Hkv, int64_t D,
                                int64_t page_size, float scale, int dtype, void* stream) {
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
                                      max_pages_per_seq * page_size);
  const int64_t need = shared_bytes(B * Hq, D, plan);
  if (workspace_bytes < need)
    return lc_fail(LC_EWORKSPACE, "%s: workspace %lld < %lld bytes", who,
                   (long long)workspace_bytes, (long long)need);
  LC_REQUIRE(lc_aligned(workspace, 256), "%s: workspace not 256-byte aligned", who);

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
  hipStream_t st = lc_stream(stream);
  switch (dtype) {
    case LC_DTYPE_F32:
      return launch_shared<float>(a, out, o_sb, o_sh, lse, st);
    case LC_DTYPE_BF16:
      return launch_shared<bf16_t>(a, out, o_sb, o_sh, lse, st);
    default:
      return launch_shared<f16_t>(a, out, o_sb, o_sh, lse, st);
  }
}

}  // extern "C"
