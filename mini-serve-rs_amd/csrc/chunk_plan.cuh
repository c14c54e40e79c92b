// The plan of a ragged step: which tiles of query rows its sequences make,
// which keys each tile reads, and which workgroup takes which of them. Built
// once per step on the device (chunk_plan_kernel) and read by every layer's
// attention and key-weight launches.
//
// Sequence b has n = cu_tokens[b+1] - cu_tokens[b] new tokens at positions
// off .. off+n-1, off = seq_lens[b] - n. For a KV head its n*G rows (row =
// t*G + g) are tiled: a thin sequence (n*G <= kThinRows) is one tile, of rows
// that fit one or two MFMA columns blocks and whose keys every wave reads once;
// a wide one takes tiles of kWideRows rows that share each key through LDS.
//
// A tile reads the pages that hold a key one of its rows sees. Under a window
// these are the sinks' pages and the pages from the first row's window start
// to the last row's own key: virtual page i is table entry i for i < the sink
// pages, else i - sink pages + wp0 (wp0 = 0: no gap, i itself).
//
// Work units (thin: a page; wide: four pages) of all (KV head, tile) pairs,
// heads outermost, are laid end to end and dealt to the workgroups in equal
// contiguous shares, so ragged lengths balance; a tile cut by a share's end
// leaves partial softmax states that a merge joins.
#pragma once

#include "common.cuh"

namespace rlse {

// Rows (tokens * group size) of a thin sequence at most. 8 sequences of 20 or 32
// rows after 4000 keys, 32/8 heads of 128, plan and layer: 42.5 and 44.3 us
// thin, 48.5 and 49.4 wide.
constexpr int kThinRows = 32;
constexpr int kWideRows = 256;      // rows per wide tile
constexpr int kWidePages = 4;       // pages per wide unit
constexpr int kScorePages = 8;     // pages per unit of the wide key-weight launch
constexpr int kMaxChunkSeqs = 4096; // prefix tables of the plan launch live in LDS
constexpr int kThinMinUnits = 8;    // smallest share of a workgroup: pages,
constexpr int kWideMinUnits = 4;    //   and wide units
// How far a share's boundary moves to a tile's rather than cut it: a cut costs
// a thin workgroup about what it streams in the time of 16 pages, a wide one
// about a unit.
constexpr int kThinSnap = 16;
// Pages of a thin tile that is not cut while there are workgroups for all: a
// cut takes 8 us (pieces stored, counted and joined; one token after 700,
// 16/8 heads of 128: 15.7 us cut, 11.4 whole), as long as 64 f32 pages or more
// than 100 of 16 bits.
constexpr int kThinWhole = 64;
constexpr int kWideSnap = 1;

// Rows of a thin sequence at most in a step of num_seqs sequences of up to
// max_rows rows. A single sequence that may be wide is taken as wide whatever
// it turns out to have: the step then has no thin launch.
__host__ __device__ inline int thin_row_limit(int num_seqs, int max_rows) {
  return num_seqs == 1 && max_rows > kThinRows ? 0 : kThinRows;
}

// Waves of a thin workgroup, and how many workgroups share the step: eight a
// compute unit either way. In one workgroup of 8 the waves of a tile meet in
// LDS; with many tiles two of 4 cover each other's joins. Plan and layer, 32/8
// heads of 128 in bf16, 8 waves then 4: 48 tokens after 2000 85 and 92 us, 8 after
// 4000 40 and 45; 128 after 2000 187 and 178, 128 after 100-4000 204 and 209.
__host__ __device__ inline int thin_waves(int num_seqs, int Hkv, int cus) {
  return (long long)num_seqs * Hkv <= 2LL * cus ? 8 : 4;
}
__host__ __device__ inline int thin_groups(int cus, int waves) { return cus * (8 / waves); }

struct ChunkTile {
  int unit0;     // units of this list's tiles before it (of one KV head)
  int seq;
  int tok0;      // cu_tokens[seq]
  int n;         // new tokens
  int off;       // keys before them
  int row0;      // first row of the tile
  int wp0;       // first page after the sinks' (0: the pages are 0, 1, ...)
  int pages;     // virtual pages
};

// A workgroup's share of a list, number w: units u0 .. of (head, tile) to unit
// end_u - 1 of (end_head, end_tile), count in all (0: none). The tile it works
// on first -- the thin kernels start at the share's start, the wide ones at its
// end -- is copied here (`at`), so that a workgroup's first loads all go out
// together. first: the share that holds the start tile's start, pieces: how
// many shares hold some of that tile. last: the share that holds the end
// tile's end; w itself, too, where that tile started before the share.
struct ChunkShare {
  int w, head, u0, count, first, pieces, last, tile;
  ChunkTile at;
  int end_tile, end_head, end_u, pad[13];
};
static_assert(sizeof(ChunkShare) == 128, "a share is a cache line");
static_assert(offsetof(ChunkShare, first) == 16 && offsetof(ChunkShare, at) == 32 &&
                  offsetof(ChunkShare, end_tile) == 64,
              "the plan stores shares as fours of words");

struct ChunkHead {
  uint32_t flags;  // RLSE_WS_ERR_* of this step
  uint32_t stamp;  // chunk_stamp of the call that built the plan
  int thin_tiles, thin_units;
  int wide_tiles, wide_units;
  int score_seqs, score_units;  // wide sequences, and their key blocks
};
constexpr int kChunkHeadBytes = 256;

// A row's token, row / G, by multiplication: exact for row * G < 2^32 (rows are
// below 2^23 and G at most kMaxGroup).
constexpr int kMaxGroup = 256;
struct RowDiv {
  unsigned mul;
  int G;
  __host__ __device__ explicit RowDiv(int g)
      : mul(g > 1 ? (unsigned)(0x100000000ull / (unsigned)g + 1) : 0u), G(g) {}
  __host__ __device__ int token(int row) const {
    return G == 1 ? row : (int)((unsigned long long)(unsigned)row * mul >> 32);
  }
};

// What the plan's users agree on, in one word (FNV-1a over the arguments).
struct ChunkShape {
  int num_seqs, total_tokens, max_tokens, Hq, Hkv, mbps, window, sinks, cus;
};
inline uint32_t chunk_stamp(const ChunkShape& s) {
  const int v[9] = {s.num_seqs, s.total_tokens, s.max_tokens, s.Hq, s.Hkv,
                    s.mbps, s.window, s.sinks, s.cus};
  uint32_t h = 2166136261u;
  for (int x : v)
    for (int i = 0; i < 4; ++i) h = (h ^ ((uint32_t)x >> (8 * i) & 255u)) * 16777619u;
  return h;
}

// Places of the plan's parts.
struct ChunkPlanView {
  ChunkHead* head;
  ChunkTile* thin;    // [num_seqs]
  ChunkTile* score;   // [num_seqs]: wide sequences, all their rows
  ChunkTile* wide;    // [wide_cap]
  ChunkShare* thin_share;  // [2 * cus], by workgroup
  ChunkShare* wide_share;  // [cus]
};
__host__ __device__ inline long long wide_tile_cap(long long total_tokens, int G, int num_seqs) {
  return total_tokens * G / kWideRows + num_seqs;
}
__host__ __device__ inline size_t chunk_plan_bytes(int num_seqs, int total_tokens, int G, int cus) {
  return kChunkHeadBytes +
         sizeof(ChunkShare) * (size_t)(3 * cus) +
         sizeof(ChunkTile) * (size_t)(2LL * num_seqs + wide_tile_cap(total_tokens, G, num_seqs));
}
__host__ __device__ inline ChunkPlanView chunk_plan_view(void* plan, int num_seqs,
                                                         int total_tokens, int G, int cus) {
  ChunkPlanView v;
  char* p = static_cast<char*>(plan);
  v.head = reinterpret_cast<ChunkHead*>(p);
  v.thin_share = reinterpret_cast<ChunkShare*>(p + kChunkHeadBytes);
  v.wide_share = v.thin_share + 2 * cus;
  v.thin = reinterpret_cast<ChunkTile*>(v.wide_share + cus);
  v.score = v.thin + num_seqs;
  v.wide = v.score + num_seqs;
  return v;
}

// Pages of a sequence's tile: tokens t0 .. t1 of off + n keys.
__device__ __forceinline__ void tile_pages(int off, int t0, int t1, int window, int sinks, int* wp0,
                                           int* pages) {
  const int end = (off + t1 + 16) >> 4;  // pages up to the last row's own key
  *wp0 = 0;
  *pages = end;
  if (window > 0) {
    const int lo = off + t0 - window + 1;
    const int sp = (sinks + 15) >> 4;
    if (lo > 0 && (lo >> 4) > sp) {
      *wp0 = lo >> 4;
      *pages = sp + end - *wp0;
    }
  }
}
// Table entry of virtual page i.
__device__ __forceinline__ int real_page(int i, int wp0, int sink_pages) {
  return wp0 == 0 || i < sink_pages ? i : i - sink_pages + wp0;
}

// Workgroup b of the `groups` at work: workgroup b runs on XCD b % 8, so each
// XCD gets a contiguous run of shares (neighbouring shares read one head's
// keys) and few shares still spread over all XCDs.
__device__ __forceinline__ int share_index(int b, int groups) {
  const int x = b & 7, q = groups >> 3, r = groups & 7;
  return x * q + min(x, r) + (b >> 3);
}

}  // namespace rlse
