// Pages of a pool that sequences take, share and give back: resizing, forking and
// compaction of the paged KV cache.
//
// A pool is N pages, each in every layer's K and V; refs[p] counts the table entries
// that name page p, and a page with refs 0 is free. Nothing else is kept: the free
// pages are found by a pass over refs, lowest first, so results depend on the inputs
// alone. The tables and counts are read from one buffer and written to another, and a
// page that is copied goes to a page that was free when the call began: no order
// among the workgroups is needed, and a call whose result is not taken has changed
// nothing that is in use.
//
// Two launches each. The first (plan): one workgroup lists the pages that the call
// hands out or moves, the others copy refs. The second (apply): table entries and
// counts, a thread each, and the copies, dealt out to workgroups that read their
// number from the plan. Bound by the two launches (7 us for 256 rows of 76 entries over 21200
// pages, nothing copied) or the copies (see copy_slots).
#include <math.h>

#include "lc_common.h"

namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
// Pages of a thread in a pass over refs: 16, or 1 in pools that few passes of that cover
// (a thread's pages are one after another: 11.2 us for the plan of a compaction of 38 pages
// with 16, 7.0 with 1).
constexpr int kManyPages = 16;
constexpr int64_t kSmallPool = 4 * kPlanThreads;
constexpr int kApplyThreads = 256;
constexpr int kCopyBlocks = 2048;

struct CopyRec {
  int src, dst, slots, none;
};

struct PoolArgs {
  void* kp;
  void* vp;
  int64_t s_layer, s_page, s_head, s_tok;
  const int32_t* table;
  int64_t t_stride;
  int32_t* out;  // [rows, M], contiguous
  const int32_t* lens;
  const int32_t* new_lens;  // resize
  const int64_t* parents;   // fork, [R]
  int32_t* out_lens;        // fork, [R]
  const int32_t* refs;
  int32_t* out_refs;
  int32_t* map;      // compact, [N]
  int32_t* missing;  // [1]
  int32_t* head;     // workspace: pages found, copies
  int32_t* off;      // workspace, [rows]: rank of a row's first new page
  int32_t* list;     // workspace: the new pages in order (compact: the holes)
  int32_t* first;    // workspace, fork, [B]: a row's first child
  int32_t* kids;     // workspace, fork, [B]: its number of children
  CopyRec* copies;   // workspace
  int B, R, M, N, P, Hkv, D, layers;
  int table_blocks;
  bool refs_wide;  // refs is 16-byte aligned
};

__device__ __forceinline__ int held_len(const PoolArgs& a, int len) {
  const int cap = a.M * a.P;
  return len < 0 ? 0 : len > cap ? cap : len;
}
__device__ __forceinline__ bool valid(const PoolArgs& a, int page) {
  return static_cast<unsigned>(page) < static_cast<unsigned>(a.N);
}
__device__ __forceinline__ int pages_of(const PoolArgs& a, int len) { return (len + a.P - 1) / a.P; }

// Sum of x over the threads before this one; total: over all of them.
__device__ __forceinline__ int block_scan(int x, int& total, int* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    const int s = sums[w];
    before += w < wave ? s : 0;
    total += s;
  }
  __syncthreads();
  return before + incl - x;
}

// A thread's share of a pass over refs, from page p0 on; pages past the pool count as
// `none`.
template <int PAGES>
__device__ __forceinline__ void load_refs(const PoolArgs& a, int64_t p0, int none, int (&r)[PAGES]) {
  if (PAGES % 4 == 0 && a.refs_wide && p0 + PAGES <= a.N) {
#pragma unroll
    for (int i = 0; i + 4 <= PAGES; i += 4) {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(a.refs + p0 + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) r[i + e] = static_cast<int>(x[e]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < PAGES; ++i) r[i] = p0 + i < a.N ? a.refs[p0 + i] : none;
  }
}

// The `want` lowest free pages into list; returns how many there are of them.
template <int PAGES>
__device__ __forceinline__ int find_free(const PoolArgs& a, int want, int* sums) {
  int found = 0;
  for (int64_t p0 = 0; p0 < a.N && found < want; p0 += kPlanThreads * PAGES) {
    int r[PAGES], n = 0, total;
    const int64_t mine = p0 + threadIdx.x * PAGES;
    load_refs(a, mine, 1, r);
#pragma unroll
    for (int i = 0; i < PAGES; ++i) n += r[i] == 0;
    int rank = found + block_scan(n, total, sums);
#pragma unroll
    for (int i = 0; i < PAGES; ++i)
      if (r[i] == 0) {
        if (rank < want) a.list[rank] = static_cast<int>(mine + i);
        ++rank;
      }
    found += total;
  }
  return found < want ? found : want;
}

// The plan's other workgroups: refs to out_refs.
__device__ __forceinline__ void copy_refs(const PoolArgs& a) {
  const int64_t stride = (int64_t)(gridDim.x - 1) * kPlanThreads;
  for (int64_t p = (int64_t)(blockIdx.x - 1) * kPlanThreads + threadIdx.x; p < a.N; p += stride)
    a.out_refs[p] = a.refs[p];
}

// What becomes of row b in a resize.
struct Resized {
  int held, want, fill, shared;  // shared: the page that it copies its slots from, or -1
};
__device__ __forceinline__ Resized resized(const PoolArgs& a, int b) {
  const int len = held_len(a, a.lens[b]), now = held_len(a, a.new_lens[b]);
  Resized s{pages_of(a, len), pages_of(a, now), len % a.P, -1};
  if (now > len && s.fill > 0) {
    const int page = a.table[(int64_t)b * a.t_stride + len / a.P];
    if (valid(a, page) && a.refs[page] > 1) s.shared = page;
  }
  return s;
}

template <int PAGES>
__global__ __launch_bounds__(kPlanThreads) void resize_plan_kernel(PoolArgs a) {
  __shared__ int sums[kPlanWaves];
  if (blockIdx.x > 0) return copy_refs(a);
  int want = 0, n_copies = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    Resized s{0, 0, 0, -1};
    if (b < a.B) s = resized(a, b);
    const int copy = s.shared >= 0;
    int total;
    const int at = want + block_scan(max(0, s.want - s.held) + copy, total, sums);
    if (b < a.B) a.off[b] = at;
    want += total;
    const int c = n_copies + block_scan(copy, total, sums);
    if (copy) a.copies[c] = CopyRec{s.shared, at, s.fill, 0};  // (dst: the rank, for now)
    n_copies += total;
  }
  const int found = find_free<PAGES>(a, want, sums);
  __syncthreads();
  for (int c = threadIdx.x; c < n_copies; c += kPlanThreads) {
    const int rank = a.copies[c].dst;
    a.copies[c].dst = rank < found ? a.list[rank] : -1;
  }
  if (threadIdx.x == 0) {
    a.head[0] = found;
    a.head[1] = n_copies;
    a.missing[0] = want - found;
  }
}

// The plan's copies, dealt out to `blocks` workgroups of which this is number `block`:
// a page's K or V of one layer each, or, where these are few, a part of it.
// U: the unit of a copy, 16 bytes or one element. kStream: stores past the caches, for
// copies of whole pages that nobody reads soon (compaction of 445 MB: 107 -> 84 us, 5.3
// TB/s, the rate of a large copy; loads past them as well: 102). A fork's sources and
// copies are read next (33 us so, 28 through the caches).
template <typename U, bool kStream = false>
__device__ __forceinline__ void copy_slots(const PoolArgs& a, int elem_per_unit, int block,
                                           int blocks) {
  const int n = a.head[1];
  const int64_t items = (int64_t)n * a.layers * 2;
  if (items == 0) return;
  const int row_units = a.D / elem_per_unit;
  const int64_t s_head = a.s_head / elem_per_unit, s_tok = a.s_tok / elem_per_unit;
  const bool rows_join = s_tok == row_units, heads_join = rows_join && s_head == (int64_t)a.P * s_tok;
  const int most = max(1, a.Hkv * a.P * row_units / (kApplyThreads * 4));
  const int parts = static_cast<int>(max((int64_t)1, min((int64_t)most, blocks / items)));
  for (int64_t w = block; w < items * parts; w += blocks) {
    const int part = static_cast<int>(w % parts);
    const int64_t item = w / parts;
    const int kv = static_cast<int>(item & 1);
    const int64_t cl = item >> 1;
    const int layer = static_cast<int>(cl % a.layers);
    const CopyRec c = a.copies[cl / a.layers];
    if (!valid(a, c.src) || !valid(a, c.dst) || c.src == c.dst) continue;
    U* pool = static_cast<U*>(kv ? a.vp : a.kp) + layer * (a.s_layer / elem_per_unit);
    const U* from = pool + c.src * (a.s_page / elem_per_unit);
    U* to = pool + c.dst * (a.s_page / elem_per_unit);
    const int per_head = c.slots * row_units, total = per_head * a.Hkv;
    // A run of units that follow one another in memory.
    const int run = heads_join && c.slots == a.P ? total : rows_join ? per_head : row_units;
    const int each = ((total + parts - 1) / parts + kApplyThreads - 1) / kApplyThreads * kApplyThreads;
    const int begin = part * each, end = min(total, begin + each);
    constexpr int kFlight = kStream ? 8 : 4;
    for (int i0 = begin + static_cast<int>(threadIdx.x); i0 < end; i0 += kApplyThreads * kFlight) {
      U x[kFlight];
      int64_t at[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int i = min(i0 + k * kApplyThreads, end - 1);
        const int g = i / run, in = i - g * run;
        int64_t base = 0;
        if (run == per_head)
          base = g * s_head;
        else if (run == row_units)
          base = g / c.slots * s_head + g % c.slots * s_tok;
        at[k] = base + in;
        x[k] = from[at[k]];
      }
#pragma unroll
      for (int k = 0; k < kFlight; ++k)
        if (i0 + k * kApplyThreads < end) {
          if constexpr (kStream)
            __builtin_nontemporal_store(x[k], to + at[k]);
          else
            to[at[k]] = x[k];
        }
    }
  }
}

template <typename U>
__global__ __launch_bounds__(kApplyThreads) void resize_apply_kernel(PoolArgs a, int elem_per_unit) {
  if (static_cast<int>(blockIdx.x) >= a.table_blocks)
    return copy_slots<U>(a, elem_per_unit, blockIdx.x - a.table_blocks, gridDim.x - a.table_blocks);
  const int found = a.head[0], total = a.B * a.M;
  for (int i = blockIdx.x * kApplyThreads + threadIdx.x; i < total;
       i += a.table_blocks * kApplyThreads) {
    const int b = i / a.M, c = i - b * a.M;
    const Resized s = resized(a, b);
    const int copy = s.shared >= 0;
    const int old = c < s.held ? a.table[(int64_t)b * a.t_stride + c] : -1;
    int now = c < s.want ? old : -1, rank = -1;
    if (copy && c == s.held - 1)
      rank = a.off[b];
    else if (c >= s.held && c < s.want)
      rank = a.off[b] + copy + (c - s.held);
    if (rank >= 0) {
      now = rank < found ? a.list[rank] : -1;
      if (now >= 0) atomicAdd(a.out_refs + now, 1);
    }
    if (c < s.held && (c >= s.want || rank >= 0) && valid(a, old)) atomicAdd(a.out_refs + old, -1);
    a.out[i] = now;
  }
}

__device__ __forceinline__ int parent_of(const PoolArgs& a, int r) {
  const int64_t p = a.parents[r];
  return p >= 0 && p < a.B ? static_cast<int>(p) : -1;
}

// Values of another thread's atomics in this launch.
__device__ __forceinline__ int got(const int32_t* from) {
  return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int PAGES>
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(PoolArgs a) {
  __shared__ int sums[kPlanWaves];
  if (blockIdx.x > 0) return copy_refs(a);
  for (int b = threadIdx.x; b < a.B; b += kPlanThreads) {
    __hip_atomic_store(a.first + b, a.R, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(a.kids + b, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  for (int r = threadIdx.x; r < a.R; r += kPlanThreads) {
    const int p = parent_of(a, r);
    if (p >= 0) {
      atomicMin(a.first + p, r);
      atomicAdd(a.kids + p, 1);
    }
  }
  __syncthreads();
  int want = 0;
  for (int r0 = 0; r0 < a.R; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    const int p = r < a.R ? parent_of(a, r) : -1;
    int copy = 0, page = -1, fill = 0;
    if (p >= 0) {
      const int len = held_len(a, a.lens[p]);
      fill = len % a.P;
      if (fill > 0 && got(a.first + p) != r) {
        page = a.table[(int64_t)p * a.t_stride + len / a.P];
        copy = valid(a, page);
      }
    }
    int total;
    const int at = want + block_scan(copy, total, sums);
    if (r < a.R) a.off[r] = copy ? at : -1;
    if (copy) a.copies[at] = CopyRec{page, at, fill, 0};
    want += total;
  }
  const int found = find_free<PAGES>(a, want, sums);
  __syncthreads();
  for (int c = threadIdx.x; c < want; c += kPlanThreads)
    a.copies[c].dst = c < found ? a.list[c] : -1;
  if (threadIdx.x == 0) {
    a.head[0] = found;
    a.head[1] = want;
    a.missing[0] = want - found;
  }
}

template <typename U>
__global__ __launch_bounds__(kApplyThreads) void fork_apply_kernel(PoolArgs a, int elem_per_unit) {
  if (static_cast<int>(blockIdx.x) >= a.table_blocks)
    return copy_slots<U>(a, elem_per_unit, blockIdx.x - a.table_blocks, gridDim.x - a.table_blocks);
  const int found = a.head[0], id = blockIdx.x * kApplyThreads + threadIdx.x;
  const int stride = a.table_blocks * kApplyThreads;
  for (int i = id; i < a.R * a.M; i += stride) {
    const int r = i / a.M, c = i - r * a.M;
    const int p = parent_of(a, r);
    const int len = p >= 0 ? held_len(a, a.lens[p]) : 0;
    int now = c < pages_of(a, len) ? a.table[(int64_t)p * a.t_stride + c] : -1;
    if (c == len / a.P && a.off[r] >= 0) {
      now = a.off[r] < found ? a.list[a.off[r]] : -1;
      if (now >= 0) atomicAdd(a.out_refs + now, 1);
    }
    a.out[i] = now;
    if (c == 0) a.out_lens[r] = len;
  }
  // A whole page gains the row's children and loses the row; the page being filled
  // stays with the first child.
  for (int i = id; i < a.B * a.M; i += stride) {
    const int b = i / a.M, c = i - b * a.M;
    const int len = held_len(a, a.lens[b]);
    if (c >= pages_of(a, len)) continue;
    const int kids = a.kids[b], more = (c == len / a.P ? min(kids, 1) : kids) - 1;
    const int page = a.table[(int64_t)b * a.t_stride + c];
    if (more != 0 && valid(a, page)) atomicAdd(a.out_refs + page, more);
  }
}

// n pages are in use. Those with an index of n or more move, in order, into the free
// ones below n, in order: as many of one as of the other. The holes come before the
// pages that move there, so one pass finds both.
template <int PAGES>
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(PoolArgs a) {
  __shared__ int sums[kPlanWaves];
  __shared__ int live_total;
  if (threadIdx.x == 0) live_total = 0;
  __syncthreads();
  constexpr int kPass = kPlanThreads * PAGES;
  int r[PAGES], n = 0;
  for (int64_t p0 = 0; p0 < a.N; p0 += kPass) {
    load_refs(a, p0 + threadIdx.x * PAGES, 0, r);
#pragma unroll
    for (int i = 0; i < PAGES; ++i) n += r[i] != 0;
  }
  atomicAdd(&live_total, n);
  __syncthreads();
  n = live_total;
  int holes = 0, moves = 0;
  for (int64_t p0 = 0; p0 < a.N; p0 += kPass) {
    const int64_t mine = p0 + threadIdx.x * PAGES;
    load_refs(a, mine, 0, r);
    int h = 0, m = 0, total;
#pragma unroll
    for (int i = 0; i < PAGES; ++i) {
      h += r[i] == 0 && mine + i < n;
      m += r[i] != 0 && mine + i >= n;
    }
    int at_h = holes + block_scan(h, total, sums);
    holes += total;
#pragma unroll
    for (int i = 0; i < PAGES; ++i)
      if (r[i] == 0 && mine + i < n) a.list[at_h++] = static_cast<int>(mine + i);
    int at_m = moves + block_scan(m, total, sums);  // (its barriers: the holes are written)
    moves += total;
    // (all loads before the first store)
    int to[PAGES];
    int at = at_m;
#pragma unroll
    for (int i = 0; i < PAGES; ++i) {
      to[i] = r[i] == 0 ? -1 : static_cast<int>(mine + i);
      if (r[i] != 0 && mine + i >= n) to[i] = a.list[at++];
    }
#pragma unroll
    for (int i = 0; i < PAGES; ++i) {
      const int64_t p = mine + i;
      if (p < a.N) {
        if (r[i] != 0 && p >= n) {
          a.copies[at_m++] = CopyRec{static_cast<int>(p), to[i], a.P, 0};
          a.out_refs[to[i]] = r[i];
        }
        a.map[p] = to[i];
        if (p >= n)
          a.out_refs[p] = 0;
        else if (r[i] != 0)
          a.out_refs[p] = r[i];
      }
    }
  }
  if (threadIdx.x == 0) a.head[1] = moves;
}

template <typename U>
__global__ __launch_bounds__(kApplyThreads) void compact_apply_kernel(PoolArgs a, int elem_per_unit) {
  if (static_cast<int>(blockIdx.x) >= a.table_blocks)
    return copy_slots<U, true>(a, elem_per_unit, blockIdx.x - a.table_blocks, gridDim.x - a.table_blocks);
  for (int i = blockIdx.x * kApplyThreads + threadIdx.x; i < a.B * a.M;
       i += a.table_blocks * kApplyThreads) {
    const int b = i / a.M, c = i - b * a.M;
    int now = -1;
    if (c < pages_of(a, held_len(a, a.lens[b]))) {
      now = a.table[(int64_t)b * a.t_stride + c];
      if (valid(a, now)) now = a.map[now];
    }
    a.out[i] = now;
  }
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// Most pages that a call can hand out or move, and most copies.
struct PoolNeeds {
  int64_t list, copies;
};
enum PoolOp { kResize, kFork, kCompact };
PoolNeeds pool_needs(PoolOp op, int64_t B, int64_t R, int64_t M, int64_t N) {
  if (op == kCompact) return {N / 2 + 1, N / 2 + 1};
  const int64_t most = op == kFork ? R : B * M;
  return {most < N ? most : N, R};
}
int64_t pool_bytes(PoolOp op, int64_t B, int64_t R, int64_t M, int64_t N) {
  const PoolNeeds n = pool_needs(op, B, R, M, N);
  return 256 + align256(n.copies * sizeof(CopyRec)) + align256(R * 4) + align256(n.list * 4) +
         (op == kFork ? 2 * align256(B * 4) : 0);
}

int check_pool(const char* who, const PoolArgs& a, int64_t B, int64_t R, int64_t M, int64_t N,
               int64_t layers, int64_t Hkv, int64_t D, int64_t page_size, int64_t bt_stride,
               int dtype) {
  LC_REQUIRE(B >= 0 && R >= 0 && B < (1LL << 20) && R < (1LL << 20), "%s: %lld and %lld rows", who,
             (long long)B, (long long)R);
  LC_REQUIRE(layers >= 0 && layers < 32768, "%s: %lld layers", who, (long long)layers);
  LC_REQUIRE(Hkv > 0 && D > 0 && page_size > 0 && M >= 0 && N >= 0 && N < (1LL << 31) - (1 << 20),
             "%s: bad sizes", who);
  LC_REQUIRE(M < (1LL << 30) / page_size, "%s: a table of 2^30 tokens or more", who);
  LC_REQUIRE((B > R ? B : R) * M < (1LL << 30), "%s: a table of 2^30 entries or more", who);
  LC_REQUIRE(Hkv < (1LL << 28) / page_size && D < (1LL << 28) / (page_size * Hkv),
             "%s: pages of 2^28 elements or more", who);
  LC_REQUIRE(dtype == LC_DTYPE_F32 || dtype == LC_DTYPE_F16 || dtype == LC_DTYPE_BF16,
             "%s: unknown dtype %d", who, dtype);
  LC_REQUIRE(bt_stride >= M, "%s: table stride < row length", who);
  LC_REQUIRE(a.s_layer >= 0 && a.s_page >= 0 && a.s_head >= 0 && a.s_tok >= 0,
             "%s: negative stride", who);
  LC_REQUIRE((a.kp && a.vp) || layers == 0 || N == 0, "%s: null pool", who);
  LC_REQUIRE((a.refs && a.out_refs) || N == 0, "%s: null reference counts", who);
  LC_REQUIRE(a.refs != a.out_refs || N == 0, "%s: the new counts overlap the old ones", who);
  LC_REQUIRE(a.lens || B == 0, "%s: null lengths", who);
  LC_REQUIRE(a.table || B * M == 0, "%s: null table", who);
  LC_REQUIRE(a.out || R * M == 0, "%s: null table", who);
  LC_REQUIRE(a.out == nullptr || a.out != a.table, "%s: the new table overlaps the old one", who);
  return LC_OK;
}

int place_workspace(const char* who, PoolOp op, PoolArgs& a, int64_t B, int64_t R, int64_t M,
                    int64_t N, void* workspace, int64_t workspace_bytes) {
  LC_REQUIRE(workspace != nullptr, "%s: null pointer", who);
  const int64_t need = pool_bytes(op, B, R, M, N);
  if (workspace_bytes < need)
    return lc_fail(LC_EWORKSPACE, "%s: workspace %lld < %lld bytes", who,
                   (long long)workspace_bytes, (long long)need);
  LC_REQUIRE(lc_aligned(workspace, 256), "%s: workspace not 256-byte aligned", who);
  const PoolNeeds n = pool_needs(op, B, R, M, N);
  char* at = static_cast<char*>(workspace);
  a.head = reinterpret_cast<int32_t*>(at);
  at += 256;
  a.copies = reinterpret_cast<CopyRec*>(at);
  at += align256(n.copies * sizeof(CopyRec));
  a.off = reinterpret_cast<int32_t*>(at);
  at += align256(R * 4);
  a.list = reinterpret_cast<int32_t*>(at);
  at += align256(n.list * 4);
  if (op == kFork) {
    a.first = reinterpret_cast<int32_t*>(at);
    a.kids = reinterpret_cast<int32_t*>(at + align256(B * 4));
  }
  return LC_OK;
}

int launch_pool(const char* who, PoolOp op, PoolArgs a, int dtype, hipStream_t st) {
  const PoolNeeds needs = pool_needs(op, a.B, a.R, a.M, a.N);
  const int64_t refs_blocks = lc_cdiv(a.N, kPlanThreads);
  const unsigned plan = op == kCompact ? 1
                                       : 1 + static_cast<unsigned>(refs_blocks < 255 ? refs_blocks : 255);
  const bool small = a.N <= kSmallPool;
  if (op == kResize)
    small ? resize_plan_kernel<1><<<plan, kPlanThreads, 0, st>>>(a)
          : resize_plan_kernel<kManyPages><<<plan, kPlanThreads, 0, st>>>(a);
  else if (op == kFork)
    small ? fork_plan_kernel<1><<<plan, kPlanThreads, 0, st>>>(a)
          : fork_plan_kernel<kManyPages><<<plan, kPlanThreads, 0, st>>>(a);
  else
    small ? compact_plan_kernel<1><<<plan, kPlanThreads, 0, st>>>(a)
          : compact_plan_kernel<kManyPages><<<plan, kPlanThreads, 0, st>>>(a);
  const int rc = lc_check_launch(who);
  if (rc != LC_OK) return rc;
  const int64_t entries = (int64_t)(a.B > a.R ? a.B : a.R) * a.M;
  const int64_t tb = lc_cdiv(entries, kApplyThreads);
  a.table_blocks = static_cast<int>(tb < 1 ? 1 : tb > 1024 ? 1024 : tb);
  // (at most a workgroup to 16 KB of a page's K or V, the least part of copy_slots)
  const int64_t most = needs.copies * a.layers * 2 *
                       lc_cdiv((int64_t)a.Hkv * a.P * a.D * lc_dtype_size(dtype), 16384);
  const int64_t cb = a.N == 0 ? 0 : most < kCopyBlocks ? most : kCopyBlocks;
  const unsigned grid = static_cast<unsigned>(a.table_blocks + cb);
  const int esz = lc_dtype_size(dtype), vec = 16 / esz;
  const bool wide = a.D % vec == 0 && a.s_layer % vec == 0 && a.s_page % vec == 0 &&
                    a.s_head % vec == 0 && a.s_tok % vec == 0 && lc_aligned(a.kp, 16) &&
                    lc_aligned(a.vp, 16);
  auto apply = [&](auto unit, int elems) {
    typedef decltype(unit) U;
    if (op == kResize)
      resize_apply_kernel<U><<<grid, kApplyThreads, 0, st>>>(a, elems);
    else if (op == kFork)
      fork_apply_kernel<U><<<grid, kApplyThreads, 0, st>>>(a, elems);
    else
      compact_apply_kernel<U><<<grid, kApplyThreads, 0, st>>>(a, elems);
  };
  if (wide)
    apply(u32x4_t{}, vec);
  else if (esz == 4)
    apply(uint32_t{}, 1);
  else
    apply(uint16_t{}, 1);
  return lc_check_launch(who);
}

PoolArgs pool_args(void* kp, void* vp, int64_t s_layer, int64_t s_page, int64_t s_head,
                   int64_t s_tok, int64_t layers, int64_t N, const int32_t* table,
                   int64_t bt_stride, int64_t M, const int32_t* lens, const int32_t* refs,
                   int32_t* out_table, int32_t* out_refs, int64_t B, int64_t R, int64_t Hkv,
                   int64_t D, int64_t page_size) {
  PoolArgs a{};
  a.kp = kp;
  a.vp = vp;
  a.s_layer = s_layer;
  a.s_page = s_page;
  a.s_head = s_head;
  a.s_tok = s_tok;
  a.table = table;
  a.t_stride = bt_stride;
  a.out = out_table;
  a.lens = lens;
  a.refs = refs;
  a.refs_wide = lc_aligned(refs, 16);
  a.out_refs = out_refs;
  a.B = static_cast<int>(B);
  a.R = static_cast<int>(R);
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.P = static_cast<int>(page_size);
  a.Hkv = static_cast<int>(Hkv);
  a.D = static_cast<int>(D);
  a.layers = static_cast<int>(layers);
  return a;
}

}  // namespace

extern "C" {

int64_t lc_paged_kv_resize_workspace_bytes(int64_t B, int64_t max_pages_per_seq, int64_t num_pages) {
  if (B < 0 || max_pages_per_seq < 0 || num_pages < 0) return -1;
  return pool_bytes(kResize, B, B, max_pages_per_seq, num_pages);
}

int lc_paged_kv_resize(void* key_pages, void* value_pages, int64_t kv_s_layer, int64_t kv_s_page,
                       int64_t kv_s_head, int64_t kv_s_tok, int64_t layers, int64_t num_pages,
                       const int32_t* block_table, int64_t bt_stride, int64_t max_pages_per_seq,
                       const int32_t* seq_lens, const int32_t* new_lens, const int32_t* page_refs,
                       int32_t* out_table, int32_t* out_refs, int32_t* missing, void* workspace,
                       int64_t workspace_bytes, int64_t B, int64_t Hkv, int64_t D,
                       int64_t page_size, int dtype, void* stream) {
  static const char* who = "lc_paged_kv_resize";
  PoolArgs a = pool_args(key_pages, value_pages, kv_s_layer, kv_s_page, kv_s_head, kv_s_tok, layers,
                         num_pages, block_table, bt_stride, max_pages_per_seq, seq_lens, page_refs,
                         out_table, out_refs, B, B, Hkv, D, page_size);
  int rc = check_pool(who, a, B, B, max_pages_per_seq, num_pages, layers, Hkv, D, page_size,
                      bt_stride, dtype);
  if (rc != LC_OK) return rc;
  LC_REQUIRE((new_lens || B == 0) && missing, "%s: null pointer", who);
  a.new_lens = new_lens;
  a.missing = missing;
  rc = place_workspace(who, kResize, a, B, B, max_pages_per_seq, num_pages, workspace,
                       workspace_bytes);
  if (rc != LC_OK) return rc;
  return launch_pool(who, kResize, a, dtype, lc_stream(stream));
}

int64_t lc_paged_kv_fork_workspace_bytes(int64_t B, int64_t children, int64_t num_pages) {
  if (B < 0 || children < 0 || num_pages < 0) return -1;
  return pool_bytes(kFork, B, children, 0, num_pages);
}

int lc_paged_kv_fork(void* key_pages, void* value_pages, int64_t kv_s_layer, int64_t kv_s_page,
                     int64_t kv_s_head, int64_t kv_s_tok, int64_t layers, int64_t num_pages,
                     const int32_t* block_table, int64_t bt_stride, int64_t max_pages_per_seq,
                     const int32_t* seq_lens, const int64_t* parents, const int32_t* page_refs,
                     int32_t* out_table, int32_t* out_lens, int32_t* out_refs, int32_t* missing,
                     void* workspace, int64_t workspace_bytes, int64_t B, int64_t children,
                     int64_t Hkv, int64_t D, int64_t page_size, int dtype, void* stream) {
  static const char* who = "lc_paged_kv_fork";
  PoolArgs a = pool_args(key_pages, value_pages, kv_s_layer, kv_s_page, kv_s_head, kv_s_tok, layers,
                         num_pages, block_table, bt_stride, max_pages_per_seq, seq_lens, page_refs,
                         out_table, out_refs, B, children, Hkv, D, page_size);
  int rc = check_pool(who, a, B, children, max_pages_per_seq, num_pages, layers, Hkv, D, page_size,
                      bt_stride, dtype);
  if (rc != LC_OK) return rc;
  LC_REQUIRE(max_pages_per_seq > 0, "%s: a table without columns", who);
  LC_REQUIRE(((parents && out_lens) || children == 0) && missing, "%s: null pointer", who);
  a.parents = parents;
  a.out_lens = out_lens;
  a.missing = missing;
  rc = place_workspace(who, kFork, a, B, children, max_pages_per_seq, num_pages, workspace,
                       workspace_bytes);
  if (rc != LC_OK) return rc;
  return launch_pool(who, kFork, a, dtype, lc_stream(stream));
}

int64_t lc_paged_kv_compact_workspace_bytes(int64_t num_pages) {
  if (num_pages < 0) return -1;
  return pool_bytes(kCompact, 0, 0, 0, num_pages);
}

int lc_paged_kv_compact(void* key_pages, void* value_pages, int64_t kv_s_layer, int64_t kv_s_page,
                        int64_t kv_s_head, int64_t kv_s_tok, int64_t layers, int64_t num_pages,
                        const int32_t* block_table, int64_t bt_stride, int64_t max_pages_per_seq,
                        const int32_t* seq_lens, const int32_t* page_refs, int32_t* out_table,
                        int32_t* out_refs, int32_t* page_map, void* workspace,
                        int64_t workspace_bytes, int64_t B, int64_t Hkv, int64_t D,
                        int64_t page_size, int dtype, void* stream) {
  static const char* who = "lc_paged_kv_compact";
  PoolArgs a = pool_args(key_pages, value_pages, kv_s_layer, kv_s_page, kv_s_head, kv_s_tok, layers,
                         num_pages, block_table, bt_stride, max_pages_per_seq, seq_lens, page_refs,
                         out_table, out_refs, B, B, Hkv, D, page_size);
  int rc = check_pool(who, a, B, B, max_pages_per_seq, num_pages, layers, Hkv, D, page_size,
                      bt_stride, dtype);
  if (rc != LC_OK) return rc;
  LC_REQUIRE(page_map || num_pages == 0, "%s: null pointer", who);
  a.map = page_map;
  rc = place_workspace(who, kCompact, a, 0, 0, 0, num_pages, workspace, workspace_bytes);
  if (rc != LC_OK) return rc;
  return launch_pool(who, kCompact, a, dtype, lc_stream(stream));
}

}  // extern "C"
