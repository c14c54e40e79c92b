// Builds the plan of a ragged step (chunk_plan.cuh) in one launch of one
// workgroup: a step has one plan, read by every layer, and its work -- a few
// scans over the sequences and the wide tiles -- is bound by the launch and
// the round trips of its dependent loads, not by bytes or operations: 4.1 us for
// one sequence, 5.9 for 32, 7.7 for 64, 8.0 with 128 wide tiles. (With shuffles
// for the prefixes, a second search for each share's end and prefixes read through
// generic addresses: 7.8, 10, 12 and 14.)
#include "chunk_plan.h"

#include "chunk_plan.cuh"
#include "host_common.h"

namespace rlse {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

struct PlanParams {
  const int* cu;
  const int* lens;
  int num_seqs, total_tokens, max_tokens, G, Hkv, mbps, window, sinks, cus;
  int thin_rows, thin_groups;
  uint32_t stamp;
  ChunkPlanView v;
  int wide_cap;
};

// Inclusive prefix of x over the wave's lanes (row: over each 16 lanes), by data
// parallel primitives: a few cycles a step, where shuffles go through LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ int from_lane(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, ROWS == 0xf);
}
__device__ __forceinline__ int row_scan(int x) {
  x += from_lane<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x += from_lane<0x112, 0xf>(x);
  x += from_lane<0x114, 0xf>(x);
  return x + from_lane<0x118, 0xf>(x);
}
__device__ __forceinline__ int wave_scan(int x) {
  x = row_scan(x);
  x += from_lane<0x142, 0xa>(x);        // row_bcast 15 to rows 1 and 3,
  return x + from_lane<0x143, 0xc>(x);  // row_bcast 31 to rows 2 and 3
}

// Exclusive prefixes of the N values x over the workgroup, and their sums
// (s_w: kPlanWaves * N ints). (One pass for all: the round trips count here.)
template <int N>
__device__ __forceinline__ void block_scan(int (&x)[N], int (*s_w)[N], int (&sum)[N]) {
  static_assert(kPlanWaves == 16, "a row holds the waves' sums");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int inc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) inc[i] = wave_scan(x[i]);
  __syncthreads();
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < N; ++i) s_w[wave][i] = inc[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int all = row_scan(s_w[lane & 15][i]);
    sum[i] = __builtin_amdgcn_readlane(all, 15);
    x[i] = inc[i] - x[i] + (wave ? __builtin_amdgcn_readlane(all, wave - 1) : 0);
  }
}

// Last index i of a[0..n) with a[i] <= u (a[0] = 0). The first kHeld prefixes
// are held in LDS: a search through memory is a round trip per step.
constexpr int kHeld = 4096;
__device__ __forceinline__ int unit0_of(const int* held, const ChunkTile* a, int n, int i) {
  int u = held[min(i, kHeld - 1)];
  // (Else the two become one load from either address, slow for both.)
  asm volatile("" : "+v"(u));
  if (n > kHeld && i >= kHeld) u = a[i].unit0;
  return u;
}
__device__ __forceinline__ int tile_of(const int* held, const ChunkTile* a, int n, int u) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (unit0_of(held, a, n, mid) <= u) lo = mid; else hi = mid;
  }
  return lo;
}

// A list's shares: `units` units of each of Hkv heads over at most max_groups
// workgroups of at least min_units each, equal shares, but a boundary within
// snap units of a tile's moves there, and with `whole` (n * Hkv <= max_groups)
// each gets one tile. (A tile cut for the sake of a few units costs more than
// they do.) Worked out by kDealThreads threads, t among them; starts and
// firsts: max_groups + 1 numbers in LDS, where each share starts and in which
// tile. I: an integer type that holds units * Hkv * max_groups.
constexpr int kMaxShares = 1024;
constexpr int kDealThreads = kPlanThreads / 2;
struct DealList {
  const int* held;
  const ChunkTile* tiles;
  int n, units, max_groups, min_units, snap;
  bool whole, from_end;
  ChunkShare* out;
  __device__ int unit0(int i) const {
    const int u = unit0_of(held, tiles, n, min(i, n - 1));
    return i < n ? u : units;
  }
};
template <typename I>
__device__ int deal_groups(const DealList& d, int Hkv) {
  if (d.whole) return d.n * Hkv;
  const I want = ((I)d.units * Hkv + d.min_units - 1) / d.min_units;
  return (int)(want < (I)d.max_groups ? want : (I)d.max_groups);
}
template <typename I>
__device__ void deal_starts(const DealList& d, int Hkv, int t, I* starts, int* firsts) {
  const I total = (I)d.units * Hkv;
  if (total == 0) return;
  const int groups = deal_groups<I>(d, Hkv);
  const int snap = (int)min((I)d.snap, total / (4 * groups));
  for (int w = t; w <= groups; w += kDealThreads) {
    I x = total * w / groups;
    int i = 0;
    if (d.whole) {
      i = w % d.n;
      x = w < groups ? (I)(w / d.n) * d.units + d.unit0(i) : total;
    } else if (w > 0 && w < groups) {
      const int head = (int)(x / d.units), u = (int)(x - (I)head * d.units);
      i = tile_of(d.held, d.tiles, d.n, u);
      const int lo = d.unit0(i), hi = d.unit0(i + 1);
      if (u - lo <= snap) {
        x -= u - lo;
      } else if (hi - u <= snap) {
        x += hi - u;
        if (++i == d.n) i = 0;
      }
    }
    starts[w] = x;
    firsts[w] = i;
  }
}
template <typename I>
__device__ void deal_shares(const DealList& d, int Hkv, int t, const I* starts,
                            const int* firsts) {
  const I total = (I)d.units * Hkv;
  const int groups = total ? deal_groups<I>(d, Hkv) : 0;
  for (int b = t; b < d.max_groups; b += kDealThreads) {
    if (b >= groups) {
      d.out[b].count = 0;
      continue;
    }
    const int w = share_index(b, groups);
    const I from = starts[w], to = starts[w + 1];
    const int units = d.units;
    const int tile = firsts[w], after = firsts[w + 1];
    const int end_head = (int)((to - 1) / units);
    const I base = (I)end_head * units;
    // (The next share's tile, or the one before where that starts there.)
    const int to_u = (int)(to - base);
    const int end_tile = to_u == units ? d.n - 1 : after - (d.unit0(after) == to_u);
    // The tile's copy, on its way during the rest.
    const u32x4_t* at = reinterpret_cast<const u32x4_t*>(d.tiles + (d.from_end ? end_tile : tile));
    const u32x4_t at0 = at[0], at1 = at[1];
    auto holder = [&](I x) {  // the share that has unit x
      int i = d.whole ? w : (int)(x * groups / total);
      while (starts[i] > x) --i;
      while (starts[i + 1] <= x) ++i;
      return i;
    };
    const int head = (int)(from / units), lo = d.unit0(tile);
    const int u0 = (int)(from - (I)head * units) - lo;
    const int first = u0 ? holder(from - u0) : w;
    const I tile_end = from - u0 + (d.unit0(tile + 1) - lo);
    const int pieces = (tile_end > to ? holder(tile_end - 1) : w) - first + 1;
    const int end_lo = d.unit0(end_tile);
    const I end = base + d.unit0(end_tile + 1);
    const int last = end > to && base + end_lo >= from ? holder(end - 1) : w;
    u32x4_t* out = reinterpret_cast<u32x4_t*>(d.out + b);
    out[0] = u32x4_t{(uint32_t)w, (uint32_t)head, (uint32_t)u0, (uint32_t)(to - from)};
    out[1] = u32x4_t{(uint32_t)first, (uint32_t)pieces, (uint32_t)last, (uint32_t)tile};
    out[2] = at0;
    out[3] = at1;
    out[4] = u32x4_t{(uint32_t)end_tile, (uint32_t)end_head, (uint32_t)(to_u - end_lo), 0u};
  }
}

__global__ __launch_bounds__(kPlanThreads) void chunk_plan_kernel(PlanParams p) {
  __shared__ int s_wide[kMaxChunkSeqs + 1];  // wide tiles before each sequence
  __shared__ int s_w[kPlanWaves][5], s_w1[kPlanWaves][1];
  __shared__ int s_held[2][kHeld];  // unit0 of the thin and the wide tiles
  __shared__ unsigned long long s_starts[2][kMaxShares + 1];
  __shared__ int s_firsts[2][kMaxShares + 1];
  __shared__ unsigned s_flags;
  __shared__ int s_longest;  // pages of the longest thin tile
  const int tid = threadIdx.x;
  if (tid == 0) {
    s_flags = 0;
    s_longest = 0;
  }
  __syncthreads();

  int thin_tiles = 0, thin_units = 0, wide_tiles = 0, score_seqs = 0, score_units = 0;
  for (int b0 = 0; b0 < p.num_seqs; b0 += kPlanThreads) {
    const int b = b0 + tid;
    ChunkTile t{};
    int thin = 0, wide = 0, tiles = 0, blocks = 0;
    if (b < p.num_seqs) {
      const int c0 = p.cu[b], c1 = p.cu[b + 1], len = p.lens[b];
      const int n = c1 - c0;
      const bool bad = c0 < 0 || c1 < c0 || c1 > p.total_tokens || n > p.max_tokens ||
                       (n > 0 && (len < n || len > p.mbps * 16));
      if (bad) atomicOr(&s_flags, RLSE_WS_ERR_LENGTH);
      if (!bad && n > 0) {
        t.seq = b;
        t.tok0 = c0;
        t.n = n;
        t.off = len - n;
        tile_pages(t.off, 0, n - 1, p.window, p.sinks, &t.wp0, &t.pages);
        const long long rows = (long long)n * p.G;
        thin = rows <= p.thin_rows;
        wide = !thin;
        tiles = wide ? (int)((rows + kWideRows - 1) / kWideRows) : 0;
        blocks = wide ? (t.pages + kScorePages - 1) / kScorePages : 0;
      }
    }
    int x[5] = {thin, thin ? t.pages : 0, wide, blocks, tiles}, sum[5];
    block_scan(x, s_w, sum);
    if (thin) {
      const int at = x[0] + thin_tiles;
      t.unit0 = x[1] + thin_units;
      p.v.thin[at] = t;
      if (at < kHeld) s_held[0][at] = t.unit0;
      atomicMax(&s_longest, t.pages);
    }
    if (wide) {
      const int at = x[2] + score_seqs;
      t.unit0 = x[3] + score_units;
      p.v.score[at] = t;
      s_wide[at] = x[4] + wide_tiles;
    }
    thin_tiles += sum[0];
    thin_units += sum[1];
    score_seqs += sum[2];
    score_units += sum[3];
    wide_tiles += sum[4];
  }
  if (wide_tiles > p.wide_cap) {  // cu_tokens overlap
    wide_tiles = p.wide_cap;
    if (tid == 0) atomicOr(&s_flags, RLSE_WS_ERR_LENGTH);
  }
  __syncthreads();

  // The wide tiles, one thread each: its sequence is the last of the
  // wide ones (score order) with no more tiles before it.
  int wide_units = 0;
  for (int i0 = 0; i0 < wide_tiles; i0 += kPlanThreads) {
    const int i = i0 + tid;
    ChunkTile t{};
    int units = 0;
    if (i < wide_tiles) {
      int lo = 0, hi = score_seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_wide[mid] <= i) lo = mid; else hi = mid;
      }
      t = p.v.score[lo];
      t.row0 = (i - s_wide[lo]) * kWideRows;
      const int last = min(t.row0 + kWideRows, t.n * p.G) - 1;
      tile_pages(t.off, t.row0 / p.G, last / p.G, p.window, p.sinks, &t.wp0, &t.pages);
      units = (t.pages + kWidePages - 1) / kWidePages;
    }
    int x[1] = {units}, sum[1];
    block_scan(x, s_w1, sum);
    t.unit0 = x[0] + wide_units;
    wide_units += sum[0];
    if (i < wide_tiles) {
      p.v.wide[i] = t;
      if (i < kHeld) s_held[1][i] = t.unit0;
    }
  }
  __syncthreads();

  // The thin list's shares by the first half of the threads, the wide one's
  // by the second.
  const bool second = tid >= kDealThreads;
  DealList d;
  d.held = s_held[second];
  d.tiles = second ? p.v.wide : p.v.thin;
  d.n = second ? wide_tiles : thin_tiles;
  d.units = second ? wide_units : thin_units;
  d.max_groups = second ? p.cus : p.thin_groups;
  d.min_units = second ? kWideMinUnits : kThinMinUnits;
  d.snap = second ? kWideSnap : kThinSnap;
  d.whole = !second && (long long)thin_tiles * p.Hkv <= p.thin_groups && s_longest <= kThinWhole;
  d.from_end = second;
  d.out = second ? p.v.wide_share : p.v.thin_share;
  const int t = tid & (kDealThreads - 1);
  unsigned long long* starts = s_starts[second];
  int* firsts = s_firsts[second];
  // (64-bit divisions take a few microseconds here.)
  if ((unsigned long long)max(thin_units, wide_units) * p.Hkv * p.thin_groups < (1ull << 31)) {
    deal_starts(d, p.Hkv, t, reinterpret_cast<unsigned*>(starts), firsts);
    __syncthreads();
    deal_shares(d, p.Hkv, t, reinterpret_cast<const unsigned*>(starts), firsts);
  } else {
    deal_starts(d, p.Hkv, t, starts, firsts);
    __syncthreads();
    deal_shares(d, p.Hkv, t, static_cast<const unsigned long long*>(starts), firsts);
  }
  if (tid == 0) {
    ChunkHead h;
    h.flags = s_flags;
    h.stamp = p.stamp;
    h.thin_tiles = thin_tiles;
    h.thin_units = thin_units;
    h.wide_tiles = wide_tiles;
    h.wide_units = wide_units;
    h.score_seqs = score_seqs;
    h.score_units = score_units;
    *p.v.head = h;
  }
}

}  // namespace

int validate_chunk_shape(const char* what, int num_seqs, int total_tokens, int max_tokens, int Hq,
                         int Hkv, int mbps, int window, int sinks) {
  if (num_seqs <= 0 || num_seqs > kMaxChunkSeqs)
    return fail(RLSE_ERR_INVALID_VALUE, "%s: num_seqs %d outside 1..%d", what, num_seqs,
                kMaxChunkSeqs);
  if (total_tokens <= 0 || max_tokens <= 0 || max_tokens > total_tokens)
    return fail(RLSE_ERR_INVALID_VALUE, "%s: need 1 <= max_tokens (%d) <= total_tokens (%d)", what,
                max_tokens, total_tokens);
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0)
    return fail(RLSE_ERR_INVALID_VALUE, "%s: num_heads %d not a multiple of num_kv_heads %d", what,
                Hq, Hkv);
  if (Hq / Hkv > kMaxGroup)
    return fail(RLSE_ERR_INVALID_VALUE, "%s: group size %d above %d", what, Hq / Hkv, kMaxGroup);
  if ((long long)total_tokens * Hq > 0x7fffffffLL / 256)
    return fail(RLSE_ERR_INVALID_VALUE, "%s: total_tokens * num_heads too large", what);
  // (A list's units, at most 2^15 + num_seqs wide tiles of a quarter of the
  // pages each, are counted in 31 bits.)
  if (mbps <= 0 || mbps > (1 << 17))
    return fail(RLSE_ERR_INVALID_VALUE, "%s: max_blocks_per_seq %d outside 1..2^17", what, mbps);
  if ((long long)mbps * num_seqs > 0x7fffffffLL)
    return fail(RLSE_ERR_INVALID_VALUE, "%s: num_seqs * max_blocks_per_seq too large", what);
  if (window < 0 || sinks < 0 || sinks > (1 << 28))
    return fail(RLSE_ERR_INVALID_VALUE, "%s: window %d or sinks %d out of range", what, window,
                sinks);
  return RLSE_OK;
}

}  // namespace rlse

using namespace rlse;

extern "C" int rlse_chunk_plan_size(int num_seqs, int total_tokens, int num_heads,
                                    int num_kv_heads, size_t* bytes) {
  if (!bytes) return fail(RLSE_ERR_INVALID_VALUE, "chunk_plan_size: null output");
  int st = validate_chunk_shape("chunk_plan_size", num_seqs, total_tokens, 1, num_heads,
                                num_kv_heads, 1, 0, 0);
  if (st) return st;
  int cus = 0;
  st = device_cu_count(&cus);
  if (st) return st;
  *bytes = chunk_plan_bytes(num_seqs, total_tokens, num_heads / num_kv_heads, cus);
  return RLSE_OK;
}

extern "C" int rlse_chunk_plan(const int32_t* cu_tokens, const int32_t* seq_lens, int num_seqs,
                               int total_tokens, int max_tokens, int num_heads, int num_kv_heads,
                               int max_blocks_per_seq, int window, int sinks, void* plan,
                               size_t plan_bytes, rlse_stream_t stream) {
  int st = validate_chunk_shape("chunk_plan", num_seqs, total_tokens, max_tokens, num_heads,
                                num_kv_heads, max_blocks_per_seq, window, sinks);
  if (st) return st;
  if (!cu_tokens || !seq_lens || !plan)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_plan: null pointer argument");
  if (reinterpret_cast<uintptr_t>(plan) & 15)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_plan: plan is not 16-byte aligned");
  PlanParams p{};
  st = device_cu_count(&p.cus);
  if (st) return st;
  p.G = num_heads / num_kv_heads;
  const size_t need = chunk_plan_bytes(num_seqs, total_tokens, p.G, p.cus);
  if (plan_bytes < need)
    return fail(RLSE_ERR_BUFFER_TOO_SMALL, "chunk_plan: plan %zu bytes < %zu needed", plan_bytes,
                need);
  p.cu = cu_tokens;
  p.lens = seq_lens;
  p.num_seqs = num_seqs;
  p.total_tokens = total_tokens;
  p.max_tokens = max_tokens;
  p.Hkv = num_kv_heads;
  p.thin_rows = thin_row_limit(num_seqs, max_tokens * p.G);
  p.thin_groups = thin_groups(p.cus, thin_waves(num_seqs, num_kv_heads, p.cus));
  if (p.thin_groups > kMaxShares)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_plan: %d compute units", p.cus);
  p.mbps = max_blocks_per_seq;
  p.window = window;
  p.sinks = sinks;
  p.stamp = chunk_stamp({num_seqs, total_tokens, max_tokens, num_heads, num_kv_heads,
                         max_blocks_per_seq, window, sinks, p.cus});
  p.v = chunk_plan_view(plan, num_seqs, total_tokens, p.G, p.cus);
  p.wide_cap = (int)wide_tile_cap(total_tokens, p.G, num_seqs);
  hipLaunchKernelGGL(chunk_plan_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), p);
  return launch_status("chunk_plan_kernel");
}
