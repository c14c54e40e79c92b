// Builds the plan of a ragged step (chunk_plan.cuh) in one launch of one
// workgroup: a step has one plan, read by every layer, and its work -- a few
// scans over the sequences and the wide tiles -- is bound by the launch and
// the round trips of its dependent loads, not by bytes or operations.
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

// Exclusive prefix of x over the workgroup, and its sum (s_w: kPlanWaves ints).
__device__ __forceinline__ int block_scan(int x, int* s_w, int* sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(inc, o, 64);
    if (lane >= o) inc += y;
  }
  __syncthreads();
  if (lane == 63) s_w[wave] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kPlanWaves; ++i) {
    const int s = s_w[i];
    before += i < wave ? s : 0;
    all += s;
  }
  *sum = all;
  return before + inc - x;
}

// Last index i of a[0..n) with a[i] <= u (a[0] = 0). The first kHeld prefixes
// are held in LDS: a search through memory is a round trip per step.
constexpr int kHeld = 4096;
__device__ __forceinline__ int tile_of(const int* held, const ChunkTile* a, int n, int u) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((mid < kHeld ? held[mid] : a[mid].unit0) <= u) lo = mid; else hi = mid;
  }
  return lo;
}

// Shares of `units` units of each of Hkv heads over at most max_groups
// workgroups of at least min_units each: equal shares, but a boundary within
// snap units of a tile's moves there, and with `whole` (n * Hkv <= max_groups)
// each gets one tile. (A tile cut
// for the sake of a few units costs more than they do.) I: an integer type that holds units * Hkv *
// max_groups; starts: max_groups + 1 of them in LDS.
constexpr int kMaxShares = 1024;
template <typename I>
__device__ void deal(const int* held, const ChunkTile* tiles, int n, int units, int Hkv,
                     int max_groups, int min_units, int snap, bool whole, bool from_end,
                     I* starts, ChunkShare* out) {
  const I total = (I)units * Hkv;
  const I want = (total + min_units - 1) / min_units;
  const int groups = whole ? n * Hkv : (int)(want < (I)max_groups ? want : (I)max_groups);
  auto unit0 = [&](int i) { return i < n ? (i < kHeld ? held[i] : tiles[i].unit0) : units; };
  snap = min((I)snap, total / (4 * groups));
  for (int w = threadIdx.x; w <= groups; w += kPlanThreads) {
    I x = total * w / groups;
    if (whole) {
      x = w < groups ? (I)(w / n) * units + unit0(w % n) : total;
    } else if (w > 0 && w < groups) {
      const int head = (int)(x / units), u = (int)(x - (I)head * units);
      const int i = tile_of(held, tiles, n, u), lo = unit0(i), hi = unit0(i + 1);
      if (u - lo <= snap)
        x -= u - lo;
      else if (hi - u <= snap)
        x += hi - u;
    }
    starts[w] = x;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < max_groups; b += kPlanThreads) {
    if (b >= groups) {
      out[b].count = 0;
      continue;
    }
    ChunkShare s;
    s.w = share_index(b, groups);
    const I from = starts[s.w], to = starts[s.w + 1];
    auto holder = [&](I x) {  // the share that has unit x
      int w = (int)(x * groups / total);
      while (starts[w] > x) --w;
      while (starts[w + 1] <= x) ++w;
      return w;
    };
    s.head = (int)(from / units);
    const int u = (int)(from - (I)s.head * units);
    s.tile = tile_of(held, tiles, n, u);
    s.u0 = u - unit0(s.tile);
    s.count = (int)(to - from);
    s.first = s.u0 ? holder(from - s.u0) : s.w;
    const I tile_end = from - s.u0 + (unit0(s.tile + 1) - unit0(s.tile));
    s.pieces = (tile_end > to ? holder(tile_end - 1) : s.w) - s.first + 1;
    s.end_head = (int)((to - 1) / units);
    const I base = (I)s.end_head * units;
    s.end_tile = tile_of(held, tiles, n, (int)(to - 1 - base));
    const I end = base + unit0(s.end_tile + 1);
    s.last = end > to && base + unit0(s.end_tile) >= from ? holder(end - 1) : s.w;
    s.end_u = (int)(to - base - unit0(s.end_tile));
    s.at = tiles[from_end ? s.end_tile : s.tile];
    out[b] = s;
  }
  __syncthreads();
}
__device__ void deal_shares(const int* held, const ChunkTile* tiles, int n, int units, int Hkv,
                            int max_groups, int min_units, int snap, bool whole,
                            bool from_end, unsigned long long* starts, ChunkShare* out) {
  if (units == 0) {
    for (int b = threadIdx.x; b < max_groups; b += kPlanThreads) out[b].count = 0;
    return;
  }
  // (64-bit divisions take a few microseconds here.)
  if ((unsigned long long)units * Hkv * max_groups < (1ull << 31))
    deal<unsigned>(held, tiles, n, units, Hkv, max_groups, min_units, snap, whole, from_end,
                   reinterpret_cast<unsigned*>(starts), out);
  else
    deal<unsigned long long>(held, tiles, n, units, Hkv, max_groups, min_units, snap, whole,
                             from_end, starts, out);
}

__global__ __launch_bounds__(kPlanThreads) void chunk_plan_kernel(PlanParams p) {
  __shared__ int s_wide[kMaxChunkSeqs + 1];  // wide tiles before each sequence
  __shared__ int s_w[kPlanWaves];
  __shared__ int s_thin[kHeld], s_unit[kHeld];  // unit0 of the thin and the wide tiles
  __shared__ unsigned long long s_starts[kMaxShares + 1];
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
    int sum;
    int at = block_scan(thin, s_w, &sum) + thin_tiles;
    thin_tiles += sum;
    int u = block_scan(thin ? t.pages : 0, s_w, &sum) + thin_units;
    thin_units += sum;
    if (thin) {
      t.unit0 = u;
      p.v.thin[at] = t;
      if (at < kHeld) s_thin[at] = u;
      atomicMax(&s_longest, t.pages);
    }
    at = block_scan(wide, s_w, &sum) + score_seqs;
    score_seqs += sum;
    u = block_scan(blocks, s_w, &sum) + score_units;
    score_units += sum;
    if (wide) {
      t.unit0 = u;
      p.v.score[at] = t;
    }
    const int w0 = block_scan(tiles, s_w, &sum) + wide_tiles;
    wide_tiles += sum;
    if (wide) s_wide[at] = w0;
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
    int sum;
    t.unit0 = block_scan(units, s_w, &sum) + wide_units;
    wide_units += sum;
    if (i < wide_tiles) {
      p.v.wide[i] = t;
      if (i < kHeld) s_unit[i] = t.unit0;
    }
  }
  __syncthreads();

  deal_shares(s_thin, p.v.thin, thin_tiles, thin_units, p.Hkv, p.thin_groups, kThinMinUnits,
              kThinSnap, (long long)thin_tiles * p.Hkv <= p.thin_groups && s_longest <= kThinWhole,
              false, s_starts, p.v.thin_share);
  deal_shares(s_unit, p.v.wide, wide_tiles, wide_units, p.Hkv, p.cus, kWideMinUnits, kWideSnap,
              false, true, s_starts, p.v.wide_share);
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
  if (mbps <= 0 || mbps > (1 << 24))
    return fail(RLSE_ERR_INVALID_VALUE, "%s: max_blocks_per_seq %d outside 1..2^24", what, mbps);
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
