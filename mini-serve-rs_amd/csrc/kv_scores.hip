// The weight every cached key receives from a ragged step's queries (gfx950):
//   w[b][h][k] = (what k had before, for keys older than the chunk)
//              + sum over new tokens t and heads of KV head h that see k of
//                e^(scale q.k - lse[t][head])
// with the log-sum-exp that the step's attention left, so every query gives a
// weight of one in all. No counterpart in the reference. The rows, pages and
// shares are the plan's (chunk_plan.cuh).
//
// Both kernels hold keys still and pass the queries over them, so that a key's
// sum stays in one place and no partial sums are added by atomics: the same
// call gives the same bits. S = Q . K^T puts one key in each accumulator
// column, its rows in the lanes' accumulator elements, so the sum over rows is
// a sum in the lane and one or two exchanges at the end. Products accumulate,
// and weights sum, in f32.
//  - thin sequences (at most 32 rows): HBM bound on K. A wave takes a page at
//    a time, 16 keys of all rows on 16x16 MFMAs. 64 tokens after 1000-4000, 14/2
//    heads of 64 in bf16: 16 us, 2.7 TB/s (a launch's start and the chain of loads to
//    its first pages are most of it); 128 after 2000, 32/8 heads of 128: 113 us, 4.7 TB/s.
//  - wide ones: bound by the exponentials (16 a lane and 32x32 tile, at a
//    quarter of the VALU's rate) beside the MFMAs. A workgroup holds 128 keys
//    in registers and streams the rows through LDS, 64 (f32: 32) at a time;
//    three of them share a compute unit, to cover each other's loads. Two chunks of
//    2000 tokens under a window of 4096, 32/8 heads of 128 in bf16: 205 us, 660
//    TFLOP/s.
#include <math.h>

#include "chunk_plan.cuh"
#include "chunk_plan.h"
#include "host_common.h"

namespace rlse {
namespace {

constexpr float kLog2E = 1.4426950408889634f;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct ScoreParams {
  const void* q;       // [tokens][Hq][D]
  const void* k_pool;  // [num_blocks][Hkv][16][D]
  const int* tables;   // [num_seqs][mbps]
  const float* lse;    // [tokens][Hq]
  const float* prev;   // [num_seqs][Hkv][mbps*16], NULL, or scores itself
  float* scores;
  ChunkPlanView v;
  uint32_t stamp;
  int Hq, Hkv, G, mbps, num_blocks, window, sinks;
  float c;  // scale * log2(e)
  RowDiv div{1};
};

template <typename T>
__device__ __forceinline__ f32x4_t mma16(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (std::is_same<T, bf16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  } else if constexpr (std::is_same<T, f16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  } else {
    const float4 x = __builtin_bit_cast(float4, a), y = __builtin_bit_cast(float4, b);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, c, 0, 0, 0);
  }
}
template <typename T>
__device__ __forceinline__ f32x16_t mma32(uint4 a, uint4 b, f32x16_t c) {
  if constexpr (std::is_same<T, bf16>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  } else if constexpr (std::is_same<T, f16>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  } else {
    const float4 x = __builtin_bit_cast(float4, a), y = __builtin_bit_cast(float4, b);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, y.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, y.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, y.z, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, y.w, c, 0, 0, 0);
  }
}

// A row's log-sum-exp in log2 units; +inf (no weight) for a row that saw no
// key.
__device__ __forceinline__ float row_lse(float lse) {
  return lse == -INFINITY ? INFINITY : lse * kLog2E;
}
// Whether a row whose own key is at kmax sees key k.
__device__ __forceinline__ bool row_sees(int k, int kmax, int window, int sinks) {
  return (k <= kmax) & ((window <= 0) | (k > kmax - window) | (k < sinks));  // (no branches)
}

// Keys between the sinks' pages and the window's, which no row sees, keep
// what they had: unit u of `units` carries its share of them over.
__device__ __forceinline__ void carry_gap(const ScoreParams& p, size_t row, int wp0,
                                          int sink_pages, int u, int units, int thread,
                                          int threads) {
  if (wp0 == 0 || p.prev == p.scores) return;
  const long long lo = 16LL * sink_pages, gap = 16LL * wp0 - lo;
  const int a = (int)(lo + gap * u / units), b = (int)(lo + gap * (u + 1) / units);
  for (int k = a + thread; k < b; k += threads)
    p.scores[row + k] = p.prev ? p.prev[row + k] : 0.f;
}
// What key k (of a sequence with `off` older ones) had before.
__device__ __forceinline__ float had(const ScoreParams& p, size_t row, int k, int off) {
  return p.prev && k < off ? p.prev[row + k] : 0.f;
}

template <typename T, int D, int RT, int W, bool STREAM>
__global__ __launch_bounds__(64 * W) void score_thin_kernel(ScoreParams p) {
  constexpr int ES = (int)sizeof(T), N = D * ES / 64;
  // Pages in registers: one at work, the others in flight.
  constexpr int NBUF = 4;
  if (p.v.head->stamp != p.stamp) {
    if (blockIdx.x == 0 && threadIdx.x == 0) ws_raise(&p.v.head->flags, RLSE_WS_ERR_PLAN);
    return;
  }
  const int tiles = p.v.head->thin_tiles;
  const ChunkShare share = p.v.thin_share[blockIdx.x];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 15, quad = lane >> 4;
  const int Hq = p.Hq, Hkv = p.Hkv, G = p.G;
  const int sink_pages = (p.sinks + 15) >> 4;
  const T* __restrict__ qb = static_cast<const T*>(p.q);
  const T* __restrict__ kp = static_cast<const T*>(p.k_pool);

  int ti = __builtin_amdgcn_readfirstlane(share.tile);
  int h = __builtin_amdgcn_readfirstlane(share.head);
  int u0 = __builtin_amdgcn_readfirstlane(share.u0);
  int left = __builtin_amdgcn_readfirstlane(share.count);
  ChunkTile t = share.at;
  while (left > 0) {
    const int n = __builtin_amdgcn_readfirstlane(t.n), off = __builtin_amdgcn_readfirstlane(t.off);
    const int tok0 = __builtin_amdgcn_readfirstlane(t.tok0);
    const int wp0 = __builtin_amdgcn_readfirstlane(t.wp0);
    const int pages = __builtin_amdgcn_readfirstlane(t.pages);
    const int seq = __builtin_amdgcn_readfirstlane(t.seq);
    const int* __restrict__ table = p.tables + (size_t)seq * p.mbps;
    const size_t out = ((size_t)seq * Hkv + h) * p.mbps * 16;
    const int seg = min(left, pages - u0);
    const int rows = n * G, kend = off + n;
    const int np = (seg - wave + W - 1) / W;  // this wave's pages

    int ids = -1, pgs = 0, ids_at = 0;
    auto fetch_ids = [&](int from) __attribute__((always_inline)) {
      const int i = from + lane;
      ids = -1;
      pgs = 0;
      if (i < np) {
        pgs = real_page(u0 + wave + i * W, wp0, sink_pages);
        const int id = table[pgs];
        ids = (unsigned)id < (unsigned)p.num_blocks ? id : -1;
      }
      ids_at = from;
    };
    fetch_ids(0);

    // Queries in the A-operand layout (lane l: row l % 16; past the last row
    // that row again, for zeros times an infinite key are NaN), and the rows of
    // this lane's accumulator elements: row 4 (l / 16) + i, of no weight (lse
    // +inf) past the last.
    uint4 q[RT][N];
    float lse[RT][4];
    int kmax[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      {
        const int row = min(rt * 16 + col, rows - 1);
        const int tok = row / G, g = row - tok * G;
        const T* src = qb + ((size_t)(tok0 + tok) * Hq + h * G + g) * D + quad * (16 / ES);
#pragma unroll
        for (int r = 0; r < N; ++r)
          q[rt][r] = *reinterpret_cast<const uint4*>(src + r * (64 / ES));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = rt * 16 + quad * 4 + i;
        const bool real = row < rows;
        const int tok = real ? row / G : 0, g = real ? row - tok * G : 0;
        lse[rt][i] = real ? row_lse(p.lse[(size_t)(tok0 + tok) * Hq + h * G + g]) : INFINITY;
        kmax[rt][i] = off + tok;
      }
    }

    struct Page {
      uint4 k[N];
      float had;  // what its keys had before, one a lane
      int id, pos;
    };
    auto load = [&](Page& b, int i) __attribute__((always_inline)) {
      if (i >= ids_at + 64) fetch_ids(i);
      b.id = __builtin_amdgcn_readlane(ids, i - ids_at);
      b.pos = __builtin_amdgcn_readlane(pgs, i - ids_at) * 16;
      const size_t at = ((size_t)(b.id < 0 ? 0 : b.id) * Hkv + h) * 16 * D;
      const int rec = b.id < 0 ? 0 : min(kend - b.pos, 16) * D * ES;
      const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(kp + at), 0, rec,
                                                        kBufferWord3);
#pragma unroll
      for (int r = 0; r < N; ++r)
        b.k[r] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
                                               rk, col * D * ES + quad * 16 + r * 64, 0,
                                               STREAM ? kLoadNonTemporal : 0));
      b.had = i < np ? had(p, out, b.pos + col, off) : 0.f;
    };
    auto compute = [&](const Page& b, int i) __attribute__((always_inline)) {
      if (i >= np) return;  // (uniform)
      float w = 0.f;
      if (b.id >= 0) {
        f32x4_t x[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) x[rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < N; ++r)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) x[rt] = mma16<T>(q[rt][r], b.k[r], x[rt]);
        const bool whole = b.pos + 15 <= off && (p.window <= 0 || b.pos > kend - 1 - p.window ||
                                                 b.pos + 16 <= p.sinks);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = __builtin_amdgcn_exp2f(fmaf(x[rt][j], p.c, -lse[rt][j]));
            w += whole || (rt * 16 + quad * 4 + j < rows &&
                           row_sees(b.pos + col, kmax[rt][j], p.window, p.sinks))
                     ? e
                     : 0.f;
          }
        w += __shfl_xor(w, 16, 64);
        w += __shfl_xor(w, 32, 64);
      }
      if (lane < 16 && b.pos + col < kend) p.scores[out + b.pos + col] = w + b.had;
    };

    Page buf[NBUF];
#pragma unroll
    for (int i = 0; i < NBUF - 1; ++i) load(buf[i], i);
    for (int i = 0; i < np; i += NBUF) {
#pragma unroll
      for (int j = 0; j < NBUF; ++j) {
        load(buf[(j + NBUF - 1) % NBUF], i + j + NBUF - 1);
        compute(buf[j], i + j);
      }
    }
    for (int u = u0 + wave; u < u0 + seg; u += W)
      carry_gap(p, out, wp0, sink_pages, u, pages, lane, 64);
    left -= seg;
    u0 = 0;
    if (++ti == tiles) {
      ti = 0;
      ++h;
    }
    if (left > 0) t = p.v.thin[ti];
  }
}

constexpr int kWideWaves = 4;
constexpr int kWideThreads = 64 * kWideWaves;
constexpr int kScoreKeys = 16 * kScorePages;  // keys a workgroup holds
constexpr int kBlockRows = 128;  // a block's beginning and end cost about as many rows

template <typename T, int D>
__global__ __launch_bounds__(kWideThreads, 3) void score_wide_kernel(ScoreParams p) {
  constexpr int ES = (int)sizeof(T);
  constexpr int KB = D * ES / 32;          // 16-byte packets of a lane's key
  constexpr int KS = ES == 2 ? 2 : 1;      // 32-key blocks per wave
  constexpr int KG = kScoreKeys / (32 * KS), RG = kWideWaves / KG;  // key and row groups
  constexpr int ROWS = 32 * RG;            // rows per stage
  constexpr int PPR = D * ES / 16;
  constexpr int QPT = ROWS * PPR / kWideThreads;  // packets per thread and stage
  constexpr int PAD = ES == 2 ? 8 : 4;     // rows 4 banks apart
  static_assert(ROWS * PPR % kWideThreads == 0, "a stage splits evenly");
  __shared__ __align__(16) T s_q[2][ROWS][D + PAD];
  __shared__ __align__(16) float s_lse[2][ROWS];
  __shared__ __align__(16) int s_kmax[2][ROWS];
  __shared__ float s_sum[RG][kScoreKeys];
  __shared__ __align__(16) int s_rows[kWideThreads];
  __shared__ int s_order[kWideThreads];
  static_assert(kWideThreads == 256 && kMaxChunkSeqs < 1 << 23, "an order packs both");

  if (p.v.head->stamp != p.stamp) {
    if (blockIdx.x == 0 && threadIdx.x == 0) ws_raise(&p.v.head->flags, RLSE_WS_ERR_PLAN);
    return;
  }
  const int units = p.v.head->score_units, seqs = p.v.head->score_seqs;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int half = lane >> 5, col = lane & 31;
  const int kg = wave % KG, rg = wave / KG;
  const int Hq = p.Hq, Hkv = p.Hkv, G = p.G;
  const int sink_pages = (p.sinks + 15) >> 4;
  const RowDiv div = p.div;
  const T* __restrict__ qb = static_cast<const T*>(p.q);
  const T* __restrict__ kp = static_cast<const T*>(p.k_pool);

  // The sequence of a key block (of one head).
  auto tile_at = [&](int ub) __attribute__((always_inline)) {
    int lo = 0, hi = seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.v.score[mid].unit0 <= ub) lo = mid; else hi = mid;
    }
    return lo;
  };
  // Rows that see a key of block u: from the first key's own token to the last
  // one whose window reaches the last key (sinks: to the end).
  auto rows_of = [&](const ChunkTile& t, int u, int* r_lo, int* r_hi)
                     __attribute__((always_inline)) {
    const int vfirst = u * kScorePages, vlast = min(vfirst + kScorePages, t.pages) - 1;
    const int pos0 = real_page(vfirst, t.wp0, sink_pages) * 16;
    const int pos1 = real_page(vlast, t.wp0, sink_pages) * 16 + 15;
    int t_hi = t.n - 1;
    if (p.window > 0 && pos0 >= p.sinks)
      t_hi = (int)min((long long)t_hi, (long long)pos1 + p.window - 1 - t.off);
    *r_lo = max(0, pos0 - t.off) * G / ROWS * ROWS;
    *r_hi = (t_hi + 1) * G;
  };

  // The blocks of all KV heads, heads outermost, lie in eight contiguous runs,
  // one for each XCD (workgroup b runs on XCD b % 8). Every compute unit of it
  // holds three workgroups, at places c, c + its units, and so on; a run of up
  // to kWideThreads blocks is sorted by the rows they meet, and dealt to and
  // fro over the compute units, so that each gets about the same. (In order of
  // their keys, 2 chunks of 2000 tokens under a window of 4096 with sinks gave
  // some 382 stages of rows where the mean was 269: 254 us, 219 dealt so.)
  const long long total = (long long)units * p.Hkv;
  const long long run0 = total * (blockIdx.x & 7) >> 3;
  const int run = (int)((total * ((blockIdx.x & 7) + 1) >> 3) - run0);
  const int place = blockIdx.x >> 3, places = ((int)gridDim.x + 7 - (blockIdx.x & 7)) >> 3;
  const int columns = (places + 2) / 3;
  if (run == 0) return;
  // Block i of the run is block (rem0 + i) % units of head h0 + (rem0 + i) / units.
  const int h0 = (int)(run0 / units);
  const unsigned rem0 = (unsigned)(run0 - (long long)h0 * units);
  const bool sorted = run <= kWideThreads;
  if (sorted) {
    int rows = 0, lo = 0;
    if (tid < run) {
      const int ub = (int)((rem0 + tid) % (unsigned)units);
      lo = tile_at(ub);
      const ChunkTile t = p.v.score[lo];
      int r_lo, r_hi;
      rows_of(t, ub - t.unit0, &r_lo, &r_hi);
      rows = max(r_hi - r_lo, 0) + kBlockRows;
    }
    s_rows[tid] = rows;  // (0 past the run's end)
    __syncthreads();
    int rank = 0;
    for (int i = 0; i < run; i += 4) {
      const int4 r = *reinterpret_cast<const int4*>(s_rows + i);
      rank += (r.x > rows) | ((r.x == rows) & (i < tid));
      rank += (r.y > rows) | ((r.y == rows) & (i + 1 < tid));
      rank += (r.z > rows) | ((r.z == rows) & (i + 2 < tid));
      rank += (r.w > rows) | ((r.w == rows) & (i + 3 < tid));
    }
    if (tid < run) s_order[rank] = lo << 8 | tid;
    __syncthreads();
  }

  for (int round = place / columns;; round += 3) {
    if (round * columns >= run) break;
    int at = round * columns + (round & 1 ? columns - 1 - place % columns : place % columns);
    if (at >= run) continue;
    int lo = -1;
    if (sorted) {
      const int order = __builtin_amdgcn_readfirstlane(s_order[at]);
      lo = order >> 8;
      at = order & 255;
    }
    const int h = h0 + (int)((rem0 + at) / (unsigned)units);
    const int ub = (int)((rem0 + at) % (unsigned)units);
    if (lo < 0) lo = tile_at(ub);
    const ChunkTile t = p.v.score[lo];
    const int n = __builtin_amdgcn_readfirstlane(t.n), off = __builtin_amdgcn_readfirstlane(t.off);
    const int tok0 = __builtin_amdgcn_readfirstlane(t.tok0);
    const int wp0 = __builtin_amdgcn_readfirstlane(t.wp0);
    const int pages = __builtin_amdgcn_readfirstlane(t.pages);
    const int seq = __builtin_amdgcn_readfirstlane(t.seq);
    const int u = ub - __builtin_amdgcn_readfirstlane(t.unit0);
    const int* __restrict__ table = p.tables + (size_t)seq * p.mbps;
    const size_t out = ((size_t)seq * Hkv + h) * p.mbps * 16;
    const int rows = n * G, kend = off + n;

    // (Page ids, rows and keys are requested before any is waited for.)
    // Page of this lane's key in each of the wave's 32-key blocks.
    int id[KS], pg[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int vi = u * kScorePages + (kg * KS + i) * 2 + (col >> 4);
      pg[i] = real_page(min(vi, pages - 1), wp0, sink_pages);
      id[i] = table[pg[i]];
      if (vi >= pages || (unsigned)id[i] >= (unsigned)p.num_blocks) id[i] = -1;
    }
    const int vfirst = u * kScorePages, vlast = min(vfirst + kScorePages, pages) - 1;
    int r_lo, r_hi;
    rows_of(t, u, &r_lo, &r_hi);
    r_lo = __builtin_amdgcn_readfirstlane(r_lo);
    r_hi = __builtin_amdgcn_readfirstlane(r_hi);

    // What the key that this thread will write had before.
    float before = 0.f;
    if (tid < kScoreKeys && vfirst + (tid >> 4) <= vlast)
      before = had(p, out, real_page(vfirst + (tid >> 4), wp0, sink_pages) * 16 + (tid & 15), off);

    // Row r of this head's: token r / G, head r % G of the group.
    const auto rq = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T*>(qb + ((size_t)tok0 * Hq + h * G) * D), 0,
        (int)(((unsigned)(n - 1) * Hq + G) * (D * ES)), kBufferWord3);
    const float* __restrict__ lh = p.lse + (size_t)tok0 * Hq + h * G;
    auto row_at = [&](int row) __attribute__((always_inline)) {
      return row + div.token(row) * (Hq - G);
    };
    u32x4_t qst[QPT];
    float lst = 0.f;
    int kst = 0;
    auto load = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < QPT; ++j) {
        const int pk = tid + j * kWideThreads;
        // (Rows past the last lie past the descriptor's end: zeros.)
        qst[j] = __builtin_amdgcn_raw_buffer_load_b128(
            rq, (int)((unsigned)row_at(r0 + pk / PPR) * (D * ES) + pk % PPR * 16), 0, 0);
      }
      if (tid < ROWS) {
        // (Rows past the last read it again; they see no key.)
        const int row = min(r0 + tid, rows - 1);
        lst = lh[row_at(row)];
        kst = r0 + tid < rows ? off + div.token(row) : -1;
      }
    };
    auto store = [&](int bf) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < QPT; ++j) {
        const int pk = tid + j * kWideThreads;
        *reinterpret_cast<u32x4_t*>(&s_q[bf][pk / PPR][pk % PPR * (16 / ES)]) = qst[j];
      }
      if (tid < ROWS) {
        s_lse[bf][tid] = kst < 0 ? INFINITY : row_lse(lst);
        s_kmax[bf][tid] = kst;
      }
    };
    if (r_lo < r_hi) load(r_lo);

    int key[KS];
    unsigned reach[KS];  // rows see key when their own is at key .. key + reach
    uint4 k[KS][KB];
    bool valid = true;
    int first_key = 0x7fffffff, last_key = -1;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const uint64_t ok = __ballot(id[i] >= 0);
#pragma unroll
      for (int j = 0; j < 32; j += 16) {
        const int pos = __builtin_amdgcn_readlane(pg[i], j) * 16;
        if (ok >> j & 1) {
          first_key = min(first_key, pos);
          last_key = max(last_key, pos + 15);
        } else {
          valid = false;
        }
      }
      const int at = pg[i] * 16 + (col & 15);
      const bool here = id[i] >= 0 && at < kend;
      key[i] = here ? at : 0x7fffffff;
      reach[i] = !here ? 0u
                 : p.window > 0 && at >= p.sinks ? (unsigned)p.window - 1u
                                                 : 0x7fffffffu;
      const T* src = kp + (((size_t)max(id[i], 0) * Hkv + h) * 16 + (col & 15)) * D;
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        // 16-bit: elements 16 b + 8 half ..; f32: half * D/2 + 4 b ..
        const int e = ES == 2 ? b * 16 + half * 8 : half * (D / 2) + b * 4;
        k[i][b] = here ? *reinterpret_cast<const uint4*>(src + e) : make_uint4(0, 0, 0, 0);
      }
    }

    float sum[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) sum[i] = 0.f;
    __syncthreads();  // the stages of the unit before are read
    if (r_lo < r_hi) {
      store(0);
      __syncthreads();
      int bf = 0;
      for (int r0 = r_lo;; r0 += ROWS) {
        const bool more = r0 + ROWS < r_hi;
        if (more) load(r0 + ROWS);
        // This wave's rows, and what they see of its keys.
        const int ra = r0 + rg * 32, rb = min(ra + 31, rows - 1);
        const int kmax_lo = off + div.token(min(ra, rows - 1)), kmax_hi = off + div.token(rb);
        const bool none =
            ra >= rows || first_key > kmax_hi ||
            (p.window > 0 && last_key <= kmax_lo - p.window && first_key >= p.sinks);
        if (!none) {
          f32x16_t x[KS];
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[i][e] = 0.f;
          // Rows come from LDS four products ahead (as the compiler schedules the
          // reads: 3% slower).
          auto operand = [&](int b) __attribute__((always_inline)) {
            const int at = ES == 2 ? b * 16 + half * 8 : half * (D / 2) + b * 4;
            return *reinterpret_cast<const uint4*>(&s_q[bf][rg * 32 + col][at]);
          };
          constexpr int R = 4;
          uint4 ring[R];
#pragma unroll
          for (int b = 0; b < R; ++b) ring[b] = operand(b);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int b = 0; b < KB; ++b) {
            const uint4 a = ring[b % R];
#pragma unroll
            for (int i = 0; i < KS; ++i) x[i] = mma32<T>(a, k[i][b], x[i]);
            if (b + R < KB) ring[b % R] = operand(b + R);
            __builtin_amdgcn_sched_barrier(0);
          }
          const bool whole = valid && last_key <= kmax_lo && last_key < kend && rb == ra + 31 &&
                             (p.window <= 0 || first_key > kmax_hi - p.window ||
                              last_key < p.sinks);
          // Accumulator element e is row 8 (e/4) + 4 half + e%4 of the 32.
          const float* ls = &s_lse[bf][rg * 32 + half * 4];
          if (whole) {
#pragma unroll
            for (int e4 = 0; e4 < 16; e4 += 4) {
              const float4 l = *reinterpret_cast<const float4*>(ls + e4 * 2);
#pragma unroll
              for (int i = 0; i < KS; ++i) {
                sum[i] += __builtin_amdgcn_exp2f(fmaf(x[i][e4], p.c, -l.x));
                sum[i] += __builtin_amdgcn_exp2f(fmaf(x[i][e4 + 1], p.c, -l.y));
                sum[i] += __builtin_amdgcn_exp2f(fmaf(x[i][e4 + 2], p.c, -l.z));
                sum[i] += __builtin_amdgcn_exp2f(fmaf(x[i][e4 + 3], p.c, -l.w));
              }
            }
          } else {
            const int* ms = &s_kmax[bf][rg * 32 + half * 4];
#pragma unroll
            for (int e4 = 0; e4 < 16; e4 += 4) {
              const float4 l4 = *reinterpret_cast<const float4*>(ls + e4 * 2);
              const int4 m4 = *reinterpret_cast<const int4*>(ms + e4 * 2);
              const float l[4] = {l4.x, l4.y, l4.z, l4.w};
              const int own[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                  const float w = __builtin_amdgcn_exp2f(fmaf(x[i][e4 + j], p.c, -l[j]));
                  sum[i] += (unsigned)(own[j] - key[i]) <= reach[i] ? w : 0.f;
                }
            }
          }
        }
        if (!more) break;
        store(bf ^ 1);
        __syncthreads();
        bf ^= 1;
      }
    }
    // The row groups' and lane halves' sums, in that order.
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const float w = sum[i] + __shfl_xor(sum[i], 32, 64);
      if (half == 0) s_sum[rg][kg * 32 * KS + i * 32 + col] = w;
    }
    __syncthreads();
    if (tid < kScoreKeys) {
      const int vi = vfirst + (tid >> 4);
      if (vi <= vlast) {
        float w = s_sum[0][tid];
#pragma unroll
        for (int i = 1; i < RG; ++i) w += s_sum[i][tid];
        const int key = real_page(vi, wp0, sink_pages) * 16 + (tid & 15);
        if (key < kend) p.scores[out + key] = w + before;
      }
    }
    carry_gap(p, out, wp0, sink_pages, u, (pages + kScorePages - 1) / kScorePages, tid,
              kWideThreads);
  }
}

template <typename T, int D>
int launch_scores(const ScoreParams& p, int max_rows, int thin_rows, int waves, bool shared,
                  int cus, hipStream_t stream) {
  int st = RLSE_OK;
  if (thin_rows > 0) {
    auto run = [&](auto rt, auto w) {
      constexpr int RT = decltype(rt)::value, W = decltype(w)::value;
      const dim3 grid(thin_groups(cus, W)), block(64 * W);
      if (shared)
        hipLaunchKernelGGL((score_thin_kernel<T, D, RT, W, false>), grid, block, 0, stream, p);
      else
        hipLaunchKernelGGL((score_thin_kernel<T, D, RT, W, true>), grid, block, 0, stream, p);
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 8> eight;
    if (waves == 8)
      max_rows <= 16 ? run(one, eight) : run(two, eight);
    else
      max_rows <= 16 ? run(one, four) : run(two, four);
    st = launch_status("score_thin_kernel");
  }
  if (st || max_rows <= thin_rows) return st;
  hipLaunchKernelGGL((score_wide_kernel<T, D>), dim3(3 * cus), dim3(kWideThreads), 0, stream, p);
  return launch_status("score_wide_kernel");
}

}  // namespace
}  // namespace rlse

using namespace rlse;

extern "C" int rlse_kv_scores(const void* q, const void* k_pool, const int32_t* block_tables,
                              void* plan, const float* lse, const float* prev, float* scores,
                              int num_seqs, int total_tokens, int max_tokens, int num_heads,
                              int num_kv_heads, int head_dim, int max_blocks_per_seq,
                              int num_blocks, int window, int sinks, float scale, int dtype,
                              int flags, rlse_stream_t stream) {
  int st = validate_chunk_shape("kv_scores", num_seqs, total_tokens, max_tokens, num_heads,
                                num_kv_heads, max_blocks_per_seq, window, sinks);
  if (st) return st;
  if (head_dim != 64 && head_dim != 128)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_scores: head_dim %d not in {64, 128}", head_dim);
  if (dtype != RLSE_DTYPE_BF16 && dtype != RLSE_DTYPE_F16 && dtype != RLSE_DTYPE_F32)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_scores: bad dtype %d", dtype);
  if (num_blocks <= 0)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_scores: num_blocks %d", num_blocks);
  if (!(scale > 0.f) || !isfinite(scale))
    return fail(RLSE_ERR_INVALID_VALUE, "kv_scores: scale must be finite and positive");
  if (flags & ~RLSE_CHUNK_SHARED_PAGES)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_scores: unknown flags 0x%x", flags);
  if (!q || !k_pool || !block_tables || !plan || !lse || !scores)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_scores: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) |
       reinterpret_cast<uintptr_t>(plan)) & 15)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_scores: a buffer is not 16-byte aligned");
  const size_t floats = (size_t)num_seqs * num_kv_heads * max_blocks_per_seq * 16;
  if (prev && prev != scores && overlap(prev, floats * 4, scores, floats * 4))
    return fail(RLSE_ERR_INVALID_VALUE, "kv_scores: prev overlaps scores and is not scores");
  int cus = 0;
  st = device_cu_count(&cus);
  if (st) return st;
  ScoreParams p{};
  p.q = q;
  p.k_pool = k_pool;
  p.tables = block_tables;
  p.lse = lse;
  p.prev = prev;
  p.scores = scores;
  p.G = num_heads / num_kv_heads;
  p.v = chunk_plan_view(plan, num_seqs, total_tokens, p.G, cus);
  p.stamp = chunk_stamp({num_seqs, total_tokens, max_tokens, num_heads, num_kv_heads,
                         max_blocks_per_seq, window, sinks, cus});
  p.Hq = num_heads;
  p.Hkv = num_kv_heads;
  p.mbps = max_blocks_per_seq;
  p.num_blocks = num_blocks;
  p.window = window;
  p.sinks = sinks;
  p.c = scale * kLog2E;
  p.div = RowDiv(p.G);
  const int max_rows = max_tokens * p.G;
  const hipStream_t s = as_stream(stream);
  auto run = [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    return launch_scores<T, D>(p, max_rows, thin_row_limit(num_seqs, max_rows),
                               thin_waves(num_seqs, num_kv_heads, cus),
                               flags & RLSE_CHUNK_SHARED_PAGES, cus, s);
  };
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  if (dtype == RLSE_DTYPE_BF16) return head_dim == 128 ? run(bf16{}, d128) : run(bf16{}, d64);
  if (dtype == RLSE_DTYPE_F16) return head_dim == 128 ? run(f16{}, d128) : run(f16{}, d64);
  return head_dim == 128 ? run(float{}, d128) : run(float{}, d64);
}
