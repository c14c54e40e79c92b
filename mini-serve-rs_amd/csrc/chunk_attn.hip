// Attention of a ragged step over the paged KV pool, with a sliding window
// and sinks, on MFMA tiles (gfx950).
//
// The reference attends one sequence at a time, causally and without a window
// (src/backends/qwen2.rs:177-203, 329-345, 476-503). Here a step holds any
// number of sequences with any number of new tokens each; the query at
// position p sees key k when k <= p and (no window, or p - k < window, or
// k < sinks), and
//   out = sum_k e^(s_k - max) v_k / sum_k e^(s_k - max),  s_k = scale q.k,
// with lse = max + log sum beside it. The rows, pages and shares are the
// plan's (chunk_plan.cuh).
//
// Two kernels, by the rows a sequence has per KV head (tokens * group size):
//  - thin (at most 32 rows: decode steps, drafts): HBM bound. A wave streams
//    its own pages, 16 keys at a time, and every key meets all rows at once
//    (S^T = K.Q^T on 16x16 MFMAs with K straight from memory in the operand
//    layout); the waves of a workgroup meet at the tile's end. 48 tokens after
//    4096-32768 keys, 32/8 heads of 128 in f16: 554 us, 6.5 TB/s; 32 tokens under a
//    window of 1024, 16/8 heads: 25 us, of which 20 are HBM's; one token after 700:
//    12 us, a chain of loads. Pages are read with non-temporal loads unless the
//    caller says that sequences share them: 32 tokens after 4000 keys 81 us, 91
//    cacheable; with one table for all, 44 and 42.
//  - wide: MFMA bound. Eight waves of 32 rows share 64 keys staged in LDS.
// Softmax statistics, sums and accumulators are f32; probabilities are
// rounded to the K/V type for the product with V (2^-9 relative in bf16, as
// large as the output's own rounding), while the sum takes them unrounded.
//
// Keys a row does not see get no weight whatever their K and V hold: scores
// are replaced, not added to, and where a page is not wholly visible an
// infinite or NaN value of V reaches only the rows that see its key (split_word).
#include <math.h>

#include <mutex>

#include "chunk_plan.cuh"
#include "chunk_plan.h"
#include "host_common.h"

namespace rlse {
namespace {

// The running max of a query's softmax moves only when a score exceeds it by
// more than this many powers of two (probabilities stay below 2^8).
constexpr float kLazyLog2 = 8.f;
constexpr float kLn2 = 0.69314718055994531f;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;
typedef __attribute__((address_space(3))) void lds_void_t;

// 16-bit tiles: 16x16x32 and 32x32x16 products of 16-byte operands, and
// 16x16x16 ones of 8-byte operands.
template <typename T>
struct Tile;
template <>
struct Tile<bf16> {
  static __device__ __forceinline__ f32x4_t mma16(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t mma16h(uint2 a, uint2 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4_t, a),
                                                     __builtin_bit_cast(i16x4_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_t mma32(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kInf = 0x7f80u, kOne = 0x3f80u;
};
template <>
struct Tile<f16> {
  static __device__ __forceinline__ f32x4_t mma16(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t mma16h(uint2 a, uint2 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a),
                                                 __builtin_bit_cast(f16x4_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_t mma32(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kInf = 0x7c00u, kOne = 0x3c00u;
};

struct ChunkParams {
  const void* q;       // [tokens][Hq][D]
  const void* k_pool;  // [num_blocks][Hkv][16][D]
  const void* v_pool;
  const int* tables;   // [num_seqs][mbps]
  void* out;           // [tokens][Hq][D]
  float* lse;          // [tokens][Hq] or NULL
  ChunkPlanView v;
  uint32_t stamp;
  float* thin_part;    // [2 * groups][kThinRows * (D + 2)]
  uint32_t* thin_done; // [groups]: pieces of the tile cut at a share's end
  float* wide_part;    // [2 * groups][wide_part_floats(D)]
  uint32_t* wide_done; // [groups]: pieces of two-piece tiles left so far
  int Hq, Hkv, G, mbps, num_blocks, window, sinks;
  float c;             // scale * log2(e)
};

// Two 16-bit values of one operand word, split: those that are not
// finite taken out of `w` and marked with a one in pos (+inf, NaN) and
// neg (-inf, NaN).
template <typename T>
__device__ __forceinline__ uint32_t split_word(uint32_t w, uint32_t* pos, uint32_t* neg) {
  constexpr uint32_t inf = Tile<T>::kInf, one = Tile<T>::kOne;
  uint32_t keep = 0;
  *pos = *neg = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = w >> (16 * i) & 0xffffu, mag = x & 0x7fffu;
    keep |= (mag >= inf ? 0u : x) << (16 * i);
    *pos |= (mag > inf || x == inf ? one : 0u) << (16 * i);
    *neg |= (mag > inf || (mag == inf && x != inf) ? one : 0u) << (16 * i);
  }
  return keep;
}
__device__ __forceinline__ float split_word(float w, float* pos, float* neg) {
  const float mag = fabsf(w);
  const bool nan = w != w, big = mag == INFINITY;
  *pos = nan || w == INFINITY ? 1.f : 0.f;
  *neg = nan || (big && w < 0.f) ? 1.f : 0.f;
  return nan || big ? 0.f : w;
}
// Ones for two keys that a row sees. (By position: a probability that the type
// rounds to zero is none.)
template <typename T>
__device__ __forceinline__ uint32_t seen_word(bool a, bool b) {
  return (a ? Tile<T>::kOne : 0u) | (b ? Tile<T>::kOne << 16 : 0u);
}
// What infinities and NaNs of V add to a row that sees them p or n times.
__device__ __forceinline__ float not_finite(float p, float n) {
  return (p > 0.f ? INFINITY : 0.f) + (n > 0.f ? -INFINITY : 0.f);
}

// Partial states handed between workgroups of one launch: pairs of floats
// stored and loaded at agent scope, coherent across the XCDs' caches.
__device__ __forceinline__ void st_pair(float* p, float a, float b) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p),
                     (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void ld_pair(const float* p, float* out) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  out[0] = __uint_as_float((uint32_t)v);
  out[1] = __uint_as_float((uint32_t)(v >> 32));
}

// Requests 16 bytes a lane through a buffer descriptor, to lds + 16 * lane (lds
// the same for the wave).
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, void* lds, int off) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)lds, 16, off, 0, 0, 0);
#endif
}
// Waits for the wave's LDS accesses.
__device__ __forceinline__ void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 3 << 14);
}

// The weight of a partial state of max m under the joint max M (both -inf:
// nothing was seen; its sums are 0, or NaN from a NaN score, and stay so).
__device__ __forceinline__ float state_weight(float m, float M) {
  return __builtin_amdgcn_exp2f(m - (M == -INFINITY ? 0.f : M));
}
__device__ __forceinline__ float inverse_sum(float L) { return L == 0.f ? 0.f : 1.f / L; }
__device__ __forceinline__ float state_lse(float M, float L) {
  return (M + __builtin_amdgcn_logf(L)) * kLn2;
}
// N consecutive values of a row, N 2 or a multiple of 4.
template <typename T, int N>
__device__ __forceinline__ void write_row(T* dst, const float* v, float inv) {
  if constexpr (N == 2) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint32_t*>(dst) = Packet<T>::pack2(v[0] * inv, v[1] * inv);
    else
      *reinterpret_cast<float2*>(dst) = make_float2(v[0] * inv, v[1] * inv);
    return;
  }
#pragma unroll
  for (int i = 0; i + 3 < N; i += 4) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(dst + i) =
          make_uint2(Packet<T>::pack2(v[i] * inv, v[i + 1] * inv),
                     Packet<T>::pack2(v[i + 2] * inv, v[i + 3] * inv));
    else
      *reinterpret_cast<float4*>(dst + i) =
          make_float4(v[i] * inv, v[i + 1] * inv, v[i + 2] * inv, v[i + 3] * inv);
  }
}

// One row's limits: it sees key k when k <= kmax and (k >= wlo or k < sinks).
struct RowSpan {
  int kmax, wlo;
  __device__ __forceinline__ bool sees(int k, int sinks) const {
    return (k <= kmax) & ((k >= wlo) | (k < sinks));  // (no branches)
  }
};
__device__ __forceinline__ RowSpan row_span(int off, int t, int window) {
  RowSpan s;
  s.kmax = off + t;
  s.wlo = window > 0 ? s.kmax - window + 1 : 0;
  return s;
}

// ---------------------------------------------------------------------------
// Thin sequences
// ---------------------------------------------------------------------------

// A page of K and V in registers. 16-bit: K in the A-operand layout of
// 16x16x32 products (lane l: key l % 16, elements 32 r + 8 (l / 16) .. +8 in
// load r), V as it lies (packet l + 64 r). f32: the same with 16-byte packets
// of four elements, K's being 16 r + 4 (l / 16) .. +4.
template <typename T, int D>
struct PageRegs {
  static constexpr int N = D * (int)sizeof(T) / 64;
  uint4 k[N], v[N];
  int pos;  // position of its first key, -1: no page
};

// V rows of a wave's page in LDS, padded: 16-bit rows by 16 elements (the
// four rows of a transposing read on banks of their own), f32 rows by 4.
template <typename T, int D, int W>
struct ThinLds {
  static constexpr int kPad = sizeof(T) == 2 ? 16 : 4;
  T v[W][16][D + kPad];
};

template <typename T, int D, int RT, int W, bool STREAM>
__global__ __launch_bounds__(64 * W, 8 / W) void chunk_thin_kernel(ChunkParams p) {
  constexpr int N = PageRegs<T, D>::N;
  constexpr int ES = (int)sizeof(T), PPR = D * ES / 16;  // packets per row
  constexpr int DT = D / 16;
  constexpr int POL = STREAM ? kLoadNonTemporal : 0;
  // Pages in registers: one at work, the others in flight (as many as fit).
  constexpr int NBUF = ES == 2 ? (RT == 1 ? 3 : 2) : D == 128 && RT == 2 ? 1 : 2;
  constexpr int kExRow = D + 4;
  __shared__ __align__(16) ThinLds<T, D, W> s;
  __shared__ __align__(16) float s_ex[W][16][kExRow];
  __shared__ float s_ml[W][16][2];
  __shared__ int s_last;

  if (p.v.head->stamp != p.stamp) {
    if (blockIdx.x == 0 && threadIdx.x == 0) ws_raise(&p.v.head->flags, RLSE_WS_ERR_PLAN);
    return;
  }
  const int tiles = p.v.head->thin_tiles;
  const ChunkShare share = p.v.thin_share[blockIdx.x];
  const int w = __builtin_amdgcn_readfirstlane(share.w);

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int col = lane & 15, quad = lane >> 4;
  const int Hq = p.Hq, Hkv = p.Hkv, G = p.G;
  const int sink_pages = (p.sinks + 15) >> 4;
  const T* __restrict__ qb = static_cast<const T*>(p.q);
  const T* __restrict__ kp = static_cast<const T*>(p.k_pool);
  const T* __restrict__ vp = static_cast<const T*>(p.v_pool);

  int ti = __builtin_amdgcn_readfirstlane(share.tile);
  int left = __builtin_amdgcn_readfirstlane(share.count);
  if (left == 0) return;
  bool head_piece = share.u0 > 0;

  // The piece at work: units u0 .. u0 + seg - 1 of tile t for KV head h. This
  // wave's pages are virtual pages u0 + wave, + W, ..., np of them;
  // ids and pgs hold 64 of their ids and table places, one a lane.
  int h, u0, n, off, tok0, wp0, pages, seg, np;
  const int* __restrict__ table;
  int ids, pgs, ids_at;
  uint4 q[RT][N];
  RowSpan span[RT];
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
  // Requests the page ids and queries of a piece.
  auto open = [&](const ChunkTile& t, int head, int first) __attribute__((always_inline)) {
    h = head;
    u0 = first;
    n = __builtin_amdgcn_readfirstlane(t.n);
    off = __builtin_amdgcn_readfirstlane(t.off);
    tok0 = __builtin_amdgcn_readfirstlane(t.tok0);
    wp0 = __builtin_amdgcn_readfirstlane(t.wp0);
    pages = __builtin_amdgcn_readfirstlane(t.pages);
    table = p.tables + (size_t)__builtin_amdgcn_readfirstlane(t.seq) * p.mbps;
    seg = min(left, pages - u0);
    np = (seg - wave + W - 1) / W;
    fetch_ids(0);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = rt * 16 + col;
      const bool real = row < n * G;
      const int tok = real ? row / G : 0, g = real ? row - tok * G : 0;
      span[rt] = row_span(off, tok, p.window);
      const T* src = qb + ((size_t)(tok0 + tok) * Hq + h * G + g) * D + quad * (16 / ES);
#pragma unroll
      for (int r = 0; r < N; ++r)
        q[rt][r] = real ? *reinterpret_cast<const uint4*>(src + r * (64 / ES))
                        : make_uint4(0, 0, 0, 0);
    }
  };
  open(share.at, __builtin_amdgcn_readfirstlane(share.head),
       __builtin_amdgcn_readfirstlane(share.u0));

  while (true) {
    const int kend = off + n;
    // The next tile's record, in flight during this one.
    const int tn = ti + 1 == tiles ? 0 : ti + 1;
    const ChunkTile tile_next = p.v.thin[tn];

    f32x4_t o[RT][DT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -INFINITY;
      l[rt] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[rt][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // Raw buffer loads through a descriptor of the (page, head) tile: no page
    // (past the wave's last, an id out of range) is a descriptor of no
    // records, and rows past the last key any row sees lie past its end;
    // both read as zeros without a memory access.
    auto load = [&](PageRegs<T, D>& b, int i) __attribute__((always_inline)) {
      if (i >= ids_at + 64) fetch_ids(i);
      const int id = __builtin_amdgcn_readlane(ids, i - ids_at);
      const int pos = __builtin_amdgcn_readlane(pgs, i - ids_at) * 16;
      const size_t at = ((size_t)(id < 0 ? 0 : id) * Hkv + h) * 16 * D;
      const int rec = id < 0 ? 0 : min(kend - pos, 16) * D * ES;
      const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(kp + at), 0, rec,
                                                        kBufferWord3);
      const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(vp + at), 0, rec,
                                                        kBufferWord3);
#pragma unroll
      for (int r = 0; r < N; ++r) {
        b.k[r] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
                                               rk, col * D * ES + quad * 16 + r * 64, 0, POL));
        b.v[r] = __builtin_bit_cast(
            uint4, __builtin_amdgcn_raw_buffer_load_b128(rv, (lane + 64 * r) * 16, 0, POL));
      }
      b.pos = id < 0 ? -1 : pos;
    };

    auto compute = [&](const PageRegs<T, D>& b) __attribute__((always_inline)) {
      if (b.pos < 0) return;  // (uniform)
      // V to this wave's LDS rows; the products below read it transposed.
#pragma unroll
      for (int r = 0; r < N; ++r) {
        const int pk = lane + 64 * r;
        *reinterpret_cast<uint4*>(&s.v[wave][pk / PPR][(pk % PPR) * (16 / ES)]) = b.v[r];
      }
      f32x4_t x[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) x[rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < N; ++r)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          if constexpr (ES == 2) {
            x[rt] = Tile<T>::mma16(b.k[r], q[rt][r], x[rt]);
          } else {
            const float* kf = reinterpret_cast<const float*>(&b.k[r]);
            const float* qf = reinterpret_cast<const float*>(&q[rt][r]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              x[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], qf[j], x[rt], 0, 0, 0);
          }
        }
      // Every row sees every key of the page: up to the first new token, and
      // from the last one's window on or among the sinks.
      const bool whole = b.pos + 15 <= off &&
                         (p.window <= 0 || b.pos > kend - 1 - p.window || b.pos + 16 <= p.sinks);
      auto seen = [&](int rt, int i) __attribute__((always_inline)) {
        return span[rt].sees(b.pos + quad * 4 + i, p.sinks);
      };
      uint2 pk[RT];
      float pf[RT][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!seen(rt, i)) x[rt][i] = -INFINITY;
        }
        // Lazy online softmax in log2 units, the state equal in the four
        // lanes of a row.
        const float mx = fmaxf(fmaxf(x[rt][0], x[rt][1]), fmaxf(x[rt][2], x[rt][3])) * p.c;
        if (__any(mx > m[rt] + kLazyLog2)) {
          float top = fmaxf(mx, __shfl_xor(mx, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float mn = fmaxf(m[rt], top);
          const float a = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[rt] - mn);
          l[rt] *= a;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[rt][d] *= a;
          m[rt] = mn;
        }
        const float nm = m[rt] == -INFINITY ? 0.f : -m[rt];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pf[rt][i] = __builtin_amdgcn_exp2f(fmaf(x[rt][i], p.c, nm));
          l[rt] += pf[rt][i];
        }
        if constexpr (ES == 2)
          pk[rt] = make_uint2(Packet<T>::pack2(pf[rt][0], pf[rt][1]),
                              Packet<T>::pack2(pf[rt][2], pf[rt][3]));
      }
      // O^T += V^T . P^T
      if constexpr (ES == 2) {
        const uint16_t* row =
            reinterpret_cast<const uint16_t*>(&s.v[wave][quad * 4 + (col >> 2)][(col & 3) * 4]);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const uint2 a = __builtin_bit_cast(
              uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(row + 16 * d)));
          if (whole) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt][d] = Tile<T>::mma16h(a, pk[rt], o[rt][d]);
          } else {
            // Values that are not finite reach only the rows that see their key.
            uint2 pos, neg;
            const uint2 fin = make_uint2(split_word<T>(a.x, &pos.x, &neg.x),
                                         split_word<T>(a.y, &pos.y, &neg.y));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const uint2 see = make_uint2(seen_word<T>(seen(rt, 0), seen(rt, 1)),
                                           seen_word<T>(seen(rt, 2), seen(rt, 3)));
              const f32x4_t zero{0.f, 0.f, 0.f, 0.f};
              const f32x4_t cp = Tile<T>::mma16h(pos, see, zero);
              const f32x4_t cn = Tile<T>::mma16h(neg, see, zero);
              o[rt][d] = Tile<T>::mma16h(fin, pk[rt], o[rt][d]);
#pragma unroll
              for (int i = 0; i < 4; ++i) o[rt][d][i] += not_finite(cp[i], cn[i]);
            }
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const float a = s.v[wave][quad * 4 + i][16 * d + col];
            if (whole) {
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
                o[rt][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, pf[rt][i], o[rt][d], 0, 0, 0);
            } else {
              float pos, neg;
              const float fin = split_word(a, &pos, &neg);
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) {
                const float see = seen(rt, i) ? 1.f : 0.f;
                const f32x4_t zero{0.f, 0.f, 0.f, 0.f};
                const f32x4_t cp = __builtin_amdgcn_mfma_f32_16x16x4f32(pos, see, zero, 0, 0, 0);
                const f32x4_t cn = __builtin_amdgcn_mfma_f32_16x16x4f32(neg, see, zero, 0, 0, 0);
                o[rt][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(fin, pf[rt][i], o[rt][d], 0, 0, 0);
#pragma unroll
                for (int k = 0; k < 4; ++k) o[rt][d][k] += not_finite(cp[k], cn[k]);
              }
            }
          }
      }
    };

    PageRegs<T, D> buf[NBUF];
#pragma unroll
    for (int i = 0; i < NBUF - 1; ++i) load(buf[i], i);
    for (int i = 0; i < np; i += NBUF) {
#pragma unroll
      for (int j = 0; j < NBUF; ++j) {
        load(buf[(j + NBUF - 1) % NBUF], i + j + NBUF - 1);
        compute(buf[j]);
      }
    }

    // The waves' states meet in LDS, 16 rows at a time, TPR threads a
    // row, DPT dimensions each.
    const bool cut = seg < pages;
    const int rows = n * G, tok_at = tok0, head = h;
    left -= seg;
    ti = tn;
    if (left > 0) open(tile_next, tn == 0 ? h + 1 : h, 0);  // on its way during the join
    float* part = nullptr;
    if (cut)
      part = p.thin_part + (size_t)(2 * w + (head_piece ? 0 : 1)) * kThinRows * (D + 2);
    constexpr int TPR = 4 * W, DPT = D / TPR;
    const int er = tid / TPR, ed = tid % TPR * DPT;
    auto finish = [&](int row, float M, float L, const float* acc)
                      __attribute__((always_inline)) {
      if (row >= rows) return;
      const int tok = row / G;
      const size_t at = (size_t)(tok_at + tok) * Hq + head * G + row - tok * G;
      write_row<T, DPT>(static_cast<T*>(p.out) + at * D + ed, acc, inverse_sum(L));
      if (p.lse && tid % TPR == 0) p.lse[at] = state_lse(M, L);
    };
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (rt * 16 >= rows) break;
      __syncthreads();
      float ls = l[rt] + __shfl_xor(l[rt], 16, 64);
      ls += __shfl_xor(ls, 32, 64);
      if (lane < 16) {
        s_ml[wave][col][0] = m[rt];
        s_ml[wave][col][1] = ls;
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
        *reinterpret_cast<f32x4_t*>(&s_ex[wave][col][16 * d + quad * 4]) = o[rt][d];
      __syncthreads();
      float M = -INFINITY, L = 0.f, acc[DPT];
#pragma unroll
      for (int i = 0; i < DPT; ++i) acc[i] = 0.f;
#pragma unroll
      for (int k = 0; k < W; ++k) M = fmaxf(M, s_ml[k][er][0]);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float a = state_weight(s_ml[k][er][0], M);
        L += s_ml[k][er][1] * a;
#pragma unroll
        for (int i = 0; i < DPT; ++i) acc[i] += s_ex[k][er][ed + i] * a;
      }
      const int row = rt * 16 + er;
      if (!cut) {
        finish(row, M, L, acc);
      } else {
        float* dst = part + row * (D + 2);
#pragma unroll
        for (int i = 0; i < DPT; i += 2) st_pair(dst + ed + i, acc[i], acc[i + 1]);
        if (tid % TPR == 0) st_pair(dst + D, M, L);
      }
    }

    if (cut) {
      // The tile's last piece to arrive joins them all, in their order (the
      // result does not depend on who does). Piece stores are agent scope and
      // waited for before the count rises, so no cache holds an older copy.
      const int first = head_piece ? share.first : w;
      const int npieces = head_piece ? share.pieces : share.last - w + 1;
      wait_vm_stores();
      __syncthreads();
      if (tid == 0)
        s_last = (int)__hip_atomic_fetch_add(p.thin_done + first, 1u, __ATOMIC_RELAXED,
                                             __HIP_MEMORY_SCOPE_AGENT) == npieces - 1;
      __syncthreads();
      if (s_last) {
        if (tid == 0) st_word(p.thin_done + first, 0u);
        for (int r0 = 0; r0 < rows; r0 += 16) {
          const int row = r0 + er;
          if (row >= rows) break;
          float M = -INFINITY, L = 0.f, acc[DPT];
#pragma unroll
          for (int i = 0; i < DPT; ++i) acc[i] = 0.f;
          // kJoin pieces' loads go out together; those past the last read it
          // again and are not joined.
          constexpr int kJoin = 4;
          for (int k0 = 0; k0 < npieces; k0 += kJoin) {
            float ml[kJoin][2], a[kJoin][DPT];
#pragma unroll
            for (int j = 0; j < kJoin; ++j) {
              const int k = min(k0 + j, npieces - 1);
              const float* src = p.thin_part + (size_t)(2 * (first + k) + (k == 0 ? 1 : 0)) *
                                                   kThinRows * (D + 2) + row * (D + 2);
              ld_pair(src + D, ml[j]);
#pragma unroll
              for (int i = 0; i < DPT; i += 2) ld_pair(src + ed + i, a[j] + i);
            }
#pragma unroll
            for (int j = 0; j < kJoin; ++j) {
              if (k0 + j >= npieces) break;
              const float mn = fmaxf(M, ml[j][0]);
              const float sa = state_weight(M, mn), sb = state_weight(ml[j][0], mn);
              L = L * sa + ml[j][1] * sb;
#pragma unroll
              for (int i = 0; i < DPT; ++i) acc[i] = acc[i] * sa + a[j][i] * sb;
              M = mn;
            }
          }
          finish(row, M, L, acc);
        }
      }
    }
    if (left == 0) break;
    head_piece = false;
  }
}

constexpr int kPartLanes = 2 * kWideRows;  // two lanes a row
// Floats of a wide tile's partial state: per lane 4 D/32 fours of its row, and
// (m, l).
constexpr int wide_part_floats(int D) { return (D / 8 + 1) * 4 * kPartLanes; }

// The units (of kWidePages pages, 64 keys) of a wide tile whose keys some rows
// all see: from lo to hi - 1, and the first `sunk` among the sinks. kmin: the
// first row's own key; wlo: where the last row's window starts. Worked out
// once per tile, so that a unit costs the loop three comparisons.
struct UnitSpan {
  int lo, hi, sunk;
  __device__ __forceinline__ bool has(int u) const {
    return ((u >= lo) & (u < hi)) | (u < sunk);
  }
};
__device__ __forceinline__ UnitSpan unit_span(int kmin, int wlo, int wp0, int sink_pages,
                                              int sinks) {
  constexpr int P = kWidePages;
  const int skip = wp0 > 0 ? sink_pages : 0;  // virtual pages before the window's
  UnitSpan s;
  s.lo = (skip + max(0, ((wlo + 15) >> 4) - wp0) + P - 1) / P;
  s.hi = max(0, ((kmin + 1) >> 4) - wp0 + skip) / P;
  s.sunk = min(sinks / (16 * P), wp0 > 0 ? sink_pages / P : s.hi);
  return s;
}

// What becomes of a wide workgroup's piece of a tile: units to be joined with
// others' before it (head) or after it (tail), or the whole tile. The lane
// holds O^T rows d = 32 db + 8 (i/4) + 4 half + i%4 of its row (at `at` in q
// and out), its max and its whole sum.
//
// A tile of two pieces is the end of one share and the start of the next. A
// workgroup takes its share from the end, so the first piece is done early and
// the second late: the second's workgroup finds the first waiting and joins it
// from its registers. Nobody waits: a piece that finds no other is left in
// memory and counted, and the one counted second joins. (The joined bits are
// the same either way.) Pieces of a tile cut more than once are left for
// chunk_merge_kernel, where several workgroups join each. Against a merge of
// every cut tile in a launch of its own: 24 ragged chunks of
// 1-301 tokens after 100-3000, 28/4 heads of 128: 186 -> 170 us.
template <typename T, int D>
__device__ __forceinline__ void wide_finish(const ChunkParams& p, const ChunkShare& share, int w,
                                            bool head, bool tail, bool live, bool real, size_t at,
                                            f32x16_t (&o)[D / 32], float m, float lsum) {
  constexpr int DB = D / 32;
  __shared__ int s_counted;
  const int tid = threadIdx.x, half = (tid & 63) >> 5;
  bool done = !head && !tail;
  if (!done) {
    const int first = head ? share.first : w;
    const int pieces = head ? share.pieces : share.last - w + 1;
    uint32_t* count = p.wide_done + first;
    auto slot = [&](int of, bool tail_piece) {
      return p.wide_part + (size_t)(2 * of + (tail_piece ? 1 : 0)) * wide_part_floats(D) + 4 * tid;
    };
    bool join = false;
    if (pieces == 2 && head) {
      if (tid == 0) s_counted = (int)ld_word(count);
      __syncthreads();
      join = s_counted == 1;
      __syncthreads();
    }
    if (!join) {
      // Slot k of thread tid: four floats, 1 KB of consecutive bytes a wave.
      float* part = slot(w, !head);
      if (live) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; i += 2)
            st_pair(part + (d * 4 + i / 4) * 4 * kPartLanes + i % 4, o[d][i], o[d][i + 1]);
        st_pair(part + 4 * DB * 4 * kPartLanes, m, lsum);
      }
      if (pieces == 2) {
        wait_vm_stores();
        __syncthreads();
        if (tid == 0)
          s_counted = (int)__hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        join = s_counted == 1;
      }
    }
    if (join) {
      if (tid == 0) st_word(count, 0u);
      if (live) {
        const float* part = head ? slot(first, true) : slot(w + 1, false);
        float ml[2];
        ld_pair(part + 4 * DB * 4 * kPartLanes, ml);
        const float M = fmaxf(m, ml[0]);
        // a: the first piece's weight, b: the second's.
        const float mine = state_weight(m, M), other = state_weight(ml[0], M);
        const float a = head ? other : mine, b = head ? mine : other;
        auto joined = [&](float own, float read) __attribute__((always_inline)) {
          return fmaf(head ? read : own, a, mul_rn(head ? own : read, b));
        };
        lsum = joined(lsum, ml[1]);
        m = M;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float x[2];
            ld_pair(part + (d * 4 + i / 4) * 4 * kPartLanes + i % 4, x);
            o[d][i] = joined(o[d][i], x[0]);
            o[d][i + 1] = joined(o[d][i + 1], x[1]);
          }
      }
      done = true;
    }
  }
  if (done && real) {
    T* dst = static_cast<T*>(p.out) + at * D;
    const float inv = inverse_sum(lsum);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const float v[4] = {o[d][i4 * 4], o[d][i4 * 4 + 1], o[d][i4 * 4 + 2], o[d][i4 * 4 + 3]};
        write_row<T, 4>(dst + d * 32 + i4 * 8 + half * 4, v, inv);
      }
    if (p.lse && half == 0) p.lse[at] = state_lse(m, lsum);
  }
}

// ---------------------------------------------------------------------------
// Wide sequences, 16-bit
// ---------------------------------------------------------------------------
// A workgroup of 8 waves, two a SIMD, takes a tile of 256 rows, each wave 32 of
// them, and streams its share of the tile's pages four (64 keys) at a time
// through LDS. Per wave (v_mfma_f32_32x32x16; lane l holds A[l%32][8*(l/32)+j],
// B[8*(l/32)+j][l%32] and accumulator element i at
// [8*(i/4) + 4*(l/32) + i%4][l%32]):
//   S^T (keys x rows) = K . Q^T, so each lane owns one row: max and sum are
//   over 16 values in the lane and lane l^32, and
//   O^T (d x rows) += V^T . P^T takes the probabilities from the accumulator
//   as they lie; V^T comes from row-major LDS through transposing reads.
// Both halves of a stage's work, 32 MFMAs and the softmax between them, take a
// wave more than a thousand cycles, on different pipes. So the two waves of a
// SIMD take turns: while waves 0-3 run the products of a stage (q.k, and p.v
// of the stage before), waves 4-7 run their softmax, and a barrier swaps them.
// Waves 4-7 are thus half a stage behind. A stage's keys and values go straight
// to LDS, each wave's part a turn or two before it is used, which three
// buffers allow (through registers, stored between the turns: 5% slower). A
// turn's operands are read from LDS six MFMAs ahead (as the compiler schedules
// the reads, a turn of products took 1.75 times as long).
// Two prompts of 4096 tokens after 0-6000, 32/8 heads of 128 in bf16: 740-780 us,
// 870-915 TFLOP/s of the 1194 that a large matrix product reaches here. A stage
// of 64 keys takes 4030 cycles (products 1850, softmax 1470, the rest loads,
// waits and barriers) at a clock that long launches bring down to 1.76 GHz
// (1.94 in one of 290 us): what they draw bounds them, so that a turn
// shortened by a tenth gains a few per cent.
constexpr int kWideWaves = 8;
constexpr int kWideThreads = 64 * kWideWaves;
constexpr int kWideKeys = 16 * kWidePages;
constexpr int kWideBufs = 3;

template <typename T, int D>
struct WideLds {
  T k[kWideBufs][kWideKeys][D];
  T v[kWideBufs][kWideKeys][D];
  // Packet (16 bytes) c of a row lies at place c ^ turn: rows that one read
  // takes together are on banks of their own (64 four-byte banks). K: 8
  // consecutive rows, one packet of each; V (transposing reads): 4 consecutive
  // rows, the same four packets of each.
  static __device__ __forceinline__ int turn_k(int row) { return row & (D / 8 - 1); }
  static __device__ __forceinline__ int turn_v(int row) {
    return D == 128 ? (row & 3) << 2 : (row & 2) << 1;
  }
};

template <typename T, int D>
__global__ __launch_bounds__(kWideThreads, 1) void chunk_wide_kernel(ChunkParams p) {
  constexpr int DB = D / 32;                           // 32-dimension blocks of O^T
  constexpr int KB = D / 16;                           // 16-dimension steps of q.k
  constexpr int PPR = D / 8;                           // packets per row
  constexpr int KPT = kWideKeys * PPR / kWideThreads;  // packets per thread and stage
  __shared__ __align__(16) WideLds<T, D> s;
  __shared__ uint32_t s_odd[kWideBufs][2];  // keys of a stage with V not finite

  if (p.v.head->stamp != p.stamp) {
    if (blockIdx.x == 0 && threadIdx.x == 0) ws_raise(&p.v.head->flags, RLSE_WS_ERR_PLAN);
    return;
  }
  const int tiles = p.v.head->wide_tiles;
  const ChunkShare share = p.v.wide_share[blockIdx.x];
  const int w = __builtin_amdgcn_readfirstlane(share.w);

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int half = lane >> 5, col = lane & 31;
  const int Hq = p.Hq, Hkv = p.Hkv, G = p.G;
  const int sink_pages = (p.sinks + 15) >> 4;
  const T* __restrict__ qb = static_cast<const T*>(p.q);
  const T* __restrict__ kp = static_cast<const T*>(p.k_pool);
  const T* __restrict__ vp = static_cast<const T*>(p.v_pool);

  // Place j of this thread in a stage: key kk0 + j * kWideThreads / PPR, place
  // dc of its row; its page is the same for the wave, whose places are 1 KB of
  // consecutive LDS.
  const int kk0 = tid / PPR, dc = tid % PPR;
  constexpr int kStep = kWideThreads / PPR;  // 32 or 64 keys
  const int koff = (kk0 & 15) * D * 2 + (dc ^ WideLds<T, D>::turn_k(kk0)) * 16;
  const int voff = (kk0 & 15) * D * 2 + (dc ^ WideLds<T, D>::turn_v(kk0)) * 16;
  const int pg0 = __builtin_amdgcn_readfirstlane(kk0 >> 4);

  // Transposing V reads: within a 16-lane group lane 4j + a points at key row
  // j, columns 4a ..; half h takes keys 4h .. and 8 + 4h ..
  const int tr_g = lane >> 4, tr_j = (lane & 15) >> 2, tr_a = lane & 3;
  const int tr_row = (tr_g >> 1) * 4 + tr_j, tr_col = (tr_g & 1) * 16 + tr_a * 4;

  // The share's tiles from its last to its first (see wide_finish).
  int ti = __builtin_amdgcn_readfirstlane(share.end_tile);
  int h = __builtin_amdgcn_readfirstlane(share.end_head);
  int u_end = __builtin_amdgcn_readfirstlane(share.end_u);
  int left = __builtin_amdgcn_readfirstlane(share.count);
  ChunkTile t = share.at;
  while (left > 0) {
    const int n = __builtin_amdgcn_readfirstlane(t.n), off = __builtin_amdgcn_readfirstlane(t.off);
    const int tok0 = __builtin_amdgcn_readfirstlane(t.tok0);
    const int row0 = __builtin_amdgcn_readfirstlane(t.row0);
    const int wp0 = __builtin_amdgcn_readfirstlane(t.wp0);
    const int pages = __builtin_amdgcn_readfirstlane(t.pages);
    const int* __restrict__ table =
        p.tables + (size_t)__builtin_amdgcn_readfirstlane(t.seq) * p.mbps;
    const int units = (pages + kWidePages - 1) / kWidePages;
    const int seg = min(left, u_end), u0 = u_end - seg;
    const int rows = n * G;
    const int last_row = min(rows, row0 + kWideRows) - 1;
    const int kend = off + last_row / G + 1;  // keys the tile's rows see end here

    const int wrow = row0 + wave * 32;
    const bool live = wrow < rows;  // the wave has rows (else it only stages)
    const int row = min(wrow + col, rows - 1), tok = row / G;
    const size_t at = (size_t)(tok0 + tok) * Hq + h * G + row - tok * G;
    const RowSpan span = row_span(off, tok, p.window);
    // The units that every row of the wave sees whole, and of the tile.
    const UnitSpan mine = unit_span(
        off + min(wrow, rows - 1) / G,
        p.window > 0 ? off + min(wrow + 31, rows - 1) / G - p.window + 1 : 0, wp0, sink_pages,
        p.sinks);
    const UnitSpan all = unit_span(off + row0 / G, p.window > 0 ? kend - p.window : 0, wp0,
                                   sink_pages, p.sinks);

    // Page ids of 16 units at a time, one a lane; the valid ones as a mask.
    int ids, ids_at;
    uint64_t ids_ok;
    auto fetch_ids = [&](int u) __attribute__((always_inline)) {
      ids_at = u * kWidePages;
      const int vi = ids_at + lane;
      ids = table[real_page(min(vi, pages - 1), wp0, sink_pages)];
      const bool ok = vi < pages && (unsigned)ids < (unsigned)p.num_blocks;
      if (!ok) ids = -1;
      ids_ok = __ballot(ok);
    };
    auto page_pos = [&](int vi) __attribute__((always_inline)) {
      return real_page(min(vi, pages - 1), wp0, sink_pages) * 16;
    };

    uint4 q[KB];
#pragma unroll
    for (int i = 0; i < KB; ++i)
      q[i] = *reinterpret_cast<const uint4*>(qb + at * D + i * 16 + half * 8);
    f32x16_t o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = -INFINITY, l = 0.f;

    // Raw buffer loads through descriptors of the (page, head) tiles: no valid
    // page is a descriptor of no records, and the keys of the last page that
    // no row sees lie past its end; both read as zeros.
    const T* __restrict__ kh = kp + (size_t)h * 16 * D;
    const T* __restrict__ vh = vp + (size_t)h * 16 * D;
    const unsigned page_elems = Hkv * 16 * D;
    const int last_rec = (((kend - 1) & 15) + 1) * D * 2;
    unsigned oks = 0;  // valid pages of the last 8 units loaded, a bit each
    auto load = [&](int u, int bf) __attribute__((always_inline)) {
      if (u * kWidePages >= ids_at + 64) fetch_ids(u);
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        const int vi = u * kWidePages + pg0 + j * (kStep / 16);
        const int id = __builtin_amdgcn_readlane(ids, vi - ids_at);
        const size_t base = (size_t)(unsigned)max(id, 0) * page_elems;
        const int rec = id < 0 ? 0 : vi + 1 < pages ? 16 * D * 2 : last_rec;
        const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(kh + base), 0, rec,
                                                          kBufferWord3);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(vh + base), 0, rec,
                                                          kBufferWord3);
        const int kk = wave * (64 / PPR) + j * kStep;
        load_lds(rk, &s.k[bf][kk][0], koff);
        load_lds(rv, &s.v[bf][kk][0], voff);
      }
      const int at4 = (u & 7) * 4;
      oks = (oks & ~(15u << at4)) |
            ((unsigned)(ids_ok >> (u * kWidePages - ids_at)) & 15u) << at4;
    };
    // Units with all four pages valid that every row (of the tile) sees whole.
    auto ok_of = [&](int u) __attribute__((always_inline)) { return oks >> (u & 7) * 4 & 15u; };
    auto whole_of = [&](int u) __attribute__((always_inline)) {
      return ok_of(u) == 15u && all.has(u);
    };
    // Waits for this thread's part of unit u; where not all of the unit is
    // seen, its values of V that are not finite become zeros and are noted.
    auto arrive = [&](int u, int bf) __attribute__((always_inline)) {
      wait_vm_stores();
      if (whole_of(u)) return;
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        const int kk = kk0 + j * kStep;
        u32x4_t* at = reinterpret_cast<u32x4_t*>(&s.v[bf][kk][dc * 8]);
        u32x4_t y = *at;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          constexpr uint32_t inf = Tile<T>::kInf;
          const uint32_t x = y[i];
          const bool lo = (x & inf) == inf, hi = (x & inf << 16) == inf << 16;
          odd = odd | lo | hi;
          y[i] = x & (lo ? 0xffff0000u : ~0u) & (hi ? 0xffffu : ~0u);
        }
        if (odd) {
          *at = y;
          atomicOr(&s_odd[bf][kk >> 5], 1u << (kk & 31));
        }
      }
    };

    // Buffer of unit u: (u - u0) % kWideBufs, kept as three rotating indices.
    int b_prev = 2, b_cur = 0, b_next = 1;
    f32x16_t x[2];
    uint4 pk[4];  // P^T operands of the four 16-key blocks
    // Operand i of a turn's products: the K operands of q.k, then the V^T ones
    // of p.v.
    constexpr int NK = 2 * KB, NV = 4 * DB;
    auto operand = [&](int i, int bk, int bv) __attribute__((always_inline)) {
      if (i < NK) {
        const int kb = i >> 1, sb = i & 1;
        return *reinterpret_cast<const uint4*>(
            &s.k[bk][sb * 32 + col][((kb * 2 + half) ^ WideLds<T, D>::turn_k(col)) * 8]);
      }
      const int kq = (i - NK) / DB, d = (i - NK) % DB;
      const uint16_t* v0 = reinterpret_cast<const uint16_t*>(
          &s.v[bv][kq * 16 + tr_row][((d * 32 + tr_col) ^ WideLds<T, D>::turn_v(tr_row) * 8)]);
      const uint2 lo = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)v0));
      const uint2 hi = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                     (lds_i16x4_t*)(v0 + 8 * D)));
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    };
    auto products = [&](auto qk, auto pv, int bk, int bv, int ul) __attribute__((always_inline)) {
      constexpr int from = decltype(qk)::value ? 0 : NK, to = decltype(pv)::value ? NK + NV : NK;
      constexpr int R = 6;  // operands in flight from LDS ahead of their MFMA
      __builtin_amdgcn_s_setprio(1);
      if constexpr (decltype(qk)::value) {
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[sb][i] = 0.f;
      }
      uint4 ring[R];
#pragma unroll
      for (int i = 0; i < R; ++i) ring[i] = operand(from + i, bk, bv);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = from; i < to; ++i) {
        const uint4 a = ring[(i - from) % R];
        if (i < NK)
          x[i & 1] = Tile<T>::mma32(a, q[i >> 1], x[i & 1]);
        else
          o[(i - NK) % DB] = Tile<T>::mma32(a, pk[(i - NK) / DB], o[(i - NK) % DB]);
        if (i + R < to) ring[(i - from) % R] = operand(i + R, bk, bv);
        if (i + R == to && ul < u_end) load(ul, b_next);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    };
    auto softmax = [&](int u) __attribute__((always_inline)) {
      const unsigned ok = ok_of(u);
      if (!(ok == 15u && mine.has(u))) {
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int kk = (i >> 2) * 8 + half * 4 + (i & 3), pg = sb * 2 + (i >> 3);
            const bool see = (ok >> pg & 1) &
                             span.sees(page_pos(u * kWidePages + pg) + (kk & 15), p.sinks);
            x[sb][i] = see ? x[sb][i] : -INFINITY;
          }
      }
      float mx = x[0][0];
#pragma unroll
      for (int sb = 0; sb < 2; ++sb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[sb][i]);
      if (__any(mx * p.c > m + kLazyLog2)) {
        const float mn = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)) * p.c);
        const float a = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= a;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[d][i] *= a;
        m = mn;
      }
      const float nm = m == -INFINITY ? 0.f : -m;
      float sum = 0.f;
#pragma unroll
      for (int sb = 0; sb < 2; ++sb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[sb][i] = __builtin_amdgcn_exp2f(fmaf(x[sb][i], p.c, nm));
          sum += x[sb][i];
        }
      l += sum;
#pragma unroll
      for (int kq = 0; kq < 4; ++kq) {
        const f32x16_t& y = x[kq >> 1];
        const int e = (kq & 1) * 8;
        pk[kq] = make_uint4(
            Packet<T>::pack2(y[e], y[e + 1]), Packet<T>::pack2(y[e + 2], y[e + 3]),
            Packet<T>::pack2(y[e + 4], y[e + 5]), Packet<T>::pack2(y[e + 6], y[e + 7]));
        // (Kept in this turn: the compiler would move it to its use.)
        asm volatile("" : "+v"(pk[kq].x), "+v"(pk[kq].y), "+v"(pk[kq].z), "+v"(pk[kq].w));
      }
    };
    // What a stage's values of V that are not finite add to the rows that see
    // their keys.
    auto add_odd = [&](int bf, int u) __attribute__((always_inline)) {
      for (int sb = 0; sb < 2; ++sb) {
        uint32_t odd = __builtin_amdgcn_readfirstlane(s_odd[bf][sb]);
        while (odd) {
          const int kk = sb * 32 + __builtin_ctz(odd);
          odd &= odd - 1;
          if (!(ok_of(u) >> (kk >> 4) & 1)) continue;
          const int pg = real_page(u * kWidePages + (kk >> 4), wp0, sink_pages);
          const T* src = vp + (((size_t)table[pg] * Hkv + h) * 16 + (kk & 15)) * D;
          const bool see = span.sees(pg * 16 + (kk & 15), p.sinks);
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
              const uint2 y = *reinterpret_cast<const uint2*>(src + d * 32 + i4 * 8 + half * 4);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                T e;
                const uint16_t bits = (uint16_t)((i < 2 ? y.x : y.y) >> (16 * (i & 1)));
                __builtin_memcpy(&e, &bits, 2);
                const float v = Elem<T>::to_f32(e);
                o[d][i4 * 4 + i] += (see & !(v - v == 0.f)) ? v : 0.f;
              }
              __builtin_amdgcn_sched_barrier(0);  // (else all loads' registers at once)
            }
        }
      }
    };
    auto turn = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      wait_lds();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };

    __syncthreads();  // the stages of the segment before are read
    if (tid < 2 * kWideBufs) s_odd[tid >> 1][tid & 1] = 0;
    __syncthreads();
    fetch_ids(u0);
    load(u0, 0);
    arrive(u0, 0);
    turn();
    const bool behind = wave >= kWideWaves / 2;
    if (behind) {
      if (seg > 1) load(u0 + 1, 1);
      turn();
      // (Waves 0-3 loaded theirs in this turn and wait for it in the next.)
    }
    for (int u = u0; u < u_end; ++u) {
      if (!live && !behind && u + 1 < u_end) load(u + 1, b_next);
      if (live) {
        if (u > u0)
          products(std::true_type{}, std::true_type{}, b_cur, b_prev, behind ? u_end : u + 1);
        else
          products(std::true_type{}, std::false_type{}, b_cur, b_prev, behind ? u_end : u + 1);
        if (u > u0 && !whole_of(u - 1)) add_odd(b_prev, u - 1);
      }
      if (behind && u + 1 < u_end) arrive(u + 1, b_next);
      turn();
      if (behind && u + 2 < u_end) load(u + 2, b_prev);
      if (live) softmax(u);
      if (!behind && u + 1 < u_end) arrive(u + 1, b_next);
      turn();
      const int b = b_prev;
      b_prev = b_cur;
      b_cur = b_next;
      b_next = b;
    }
    if (live) {
      products(std::false_type{}, std::true_type{}, 0, b_prev, u_end);
      if (!whole_of(u_end - 1)) add_odd(b_prev, u_end - 1);
    }
    if (!behind) turn();

    wide_finish<T, D>(p, share, w, u0 > 0, u_end < units, live, wrow + col < rows, at, o, m,
                      l + __shfl_xor(l, 32, 64));
    left -= seg;
    if (ti-- == 0) {
      ti = tiles - 1;
      --h;
    }
    if (left > 0) {
      t = p.v.wide[ti];
      u_end = (__builtin_amdgcn_readfirstlane(t.pages) + kWidePages - 1) / kWidePages;
    }
  }
}

// ---------------------------------------------------------------------------
// Wide sequences, f32
// ---------------------------------------------------------------------------
// 1024 tokens after 2048, 32/8 heads of 128: 345 us, 125 TFLOP/s of the 154 that a
// large f32 matrix product reaches here.
// The same products on v_mfma_f32_32x32x2_f32, whose rate bounds them: lane half
// h contracts dimension h*D/2 + j at step j of S^T = K . Q^T, and step j of
// O^T += V^T . P^T pairs the two keys that the lane halves hold in accumulator
// element j. Eight waves of 32 rows (a row's f32 state takes twice the
// registers), 64 keys staged in one of two LDS buffers while the next are
// loaded.
constexpr int kWide32Waves = 8;
constexpr int kWide32Threads = 64 * kWide32Waves;

template <int D>
struct Wide32Lds {
  // K rows 4 banks apart, the V rows of the lane halves (4 apart) 32.
  float k[2][kWideKeys][D + 4];
  float v[2][kWideKeys][D + 8];
};

template <int D>
__global__ __launch_bounds__(kWide32Threads, 1) void chunk_wide32_kernel(ChunkParams p) {
  constexpr int DB = D / 32;                           // 32-dimension blocks of O^T
  constexpr int KB = D / 8;                            // 16-byte packets of a lane's query
  constexpr int PPR = D / 4;                           // packets per row
  constexpr int KPT = kWideKeys * PPR / kWide32Threads;  // packets per thread and stage
  __shared__ __align__(16) Wide32Lds<D> s;
  __shared__ uint32_t s_odd[2][2];  // keys of a stage with V not finite

  if (p.v.head->stamp != p.stamp) {
    if (blockIdx.x == 0 && threadIdx.x == 0) ws_raise(&p.v.head->flags, RLSE_WS_ERR_PLAN);
    return;
  }
  const int tiles = p.v.head->wide_tiles;
  const ChunkShare share = p.v.wide_share[blockIdx.x];
  const int w = __builtin_amdgcn_readfirstlane(share.w);

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int half = lane >> 5, col = lane & 31;
  const int Hq = p.Hq, Hkv = p.Hkv, G = p.G;
  const int sink_pages = (p.sinks + 15) >> 4;
  const float* __restrict__ qb = static_cast<const float*>(p.q);
  const float* __restrict__ kp = static_cast<const float*>(p.k_pool);
  const float* __restrict__ vp = static_cast<const float*>(p.v_pool);

  // Packet j of this thread in a stage: key kk0 + j * kWide32Threads / PPR,
  // chunk dc of its row; its page is the same for the wave.
  const int kk0 = tid / PPR, dc = tid % PPR;
  constexpr int kStep = kWide32Threads / PPR;  // 16 or 32 keys
  const int voff = (kk0 & 15) * D * 4 + dc * 16;
  const int pg0 = __builtin_amdgcn_readfirstlane(kk0 >> 4);

  // The share's tiles from its last to its first (see wide_finish).
  int ti = __builtin_amdgcn_readfirstlane(share.end_tile);
  int h = __builtin_amdgcn_readfirstlane(share.end_head);
  int u_end = __builtin_amdgcn_readfirstlane(share.end_u);
  int left = __builtin_amdgcn_readfirstlane(share.count);
  ChunkTile t = share.at;
  while (left > 0) {
    const int n = __builtin_amdgcn_readfirstlane(t.n), off = __builtin_amdgcn_readfirstlane(t.off);
    const int tok0 = __builtin_amdgcn_readfirstlane(t.tok0);
    const int row0 = __builtin_amdgcn_readfirstlane(t.row0);
    const int wp0 = __builtin_amdgcn_readfirstlane(t.wp0);
    const int pages = __builtin_amdgcn_readfirstlane(t.pages);
    const int* __restrict__ table =
        p.tables + (size_t)__builtin_amdgcn_readfirstlane(t.seq) * p.mbps;
    const int units = (pages + kWidePages - 1) / kWidePages;
    const int seg = min(left, u_end), u0 = u_end - seg;
    const int rows = n * G;
    const int last_row = min(rows, row0 + kWideRows) - 1;
    const int kend = off + last_row / G + 1;  // keys the tile's rows see end here

    const int wrow = row0 + wave * 32;
    const bool live = wrow < rows;  // the wave has rows (else it only stages)
    const int row = min(wrow + col, rows - 1), tok = row / G;
    const size_t at = (size_t)(tok0 + tok) * Hq + h * G + row - tok * G;
    const RowSpan span = row_span(off, tok, p.window);
    // The units that every row of the wave sees whole, and of the tile.
    const UnitSpan mine = unit_span(
        off + min(wrow, rows - 1) / G,
        p.window > 0 ? off + min(wrow + 31, rows - 1) / G - p.window + 1 : 0, wp0, sink_pages,
        p.sinks);
    const UnitSpan all = unit_span(off + row0 / G, p.window > 0 ? kend - p.window : 0, wp0,
                                   sink_pages, p.sinks);

    // Page ids of 16 units at a time, one a lane; the valid ones as a mask.
    int ids, ids_at;
    uint64_t ids_ok;
    auto fetch_ids = [&](int u) __attribute__((always_inline)) {
      ids_at = u * kWidePages;
      const int vi = ids_at + lane;
      ids = table[real_page(min(vi, pages - 1), wp0, sink_pages)];
      const bool ok = vi < pages && (unsigned)ids < (unsigned)p.num_blocks;
      if (!ok) ids = -1;
      ids_ok = __ballot(ok);
    };
    auto page_pos = [&](int vi) __attribute__((always_inline)) {
      return real_page(min(vi, pages - 1), wp0, sink_pages) * 16;
    };

    float4 q[KB];  // dimensions half * D/2 + 4 i ..
#pragma unroll
    for (int i = 0; i < KB; ++i)
      q[i] = *reinterpret_cast<const float4*>(qb + at * D + half * (D / 2) + i * 4);
    f32x16_t o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = -INFINITY, l = 0.f;

    // Raw buffer loads through descriptors of the (page, head) tiles: no valid
    // page is a descriptor of no records, and the keys of the last page that
    // no row sees lie past its end; both read as zeros.
    const float* __restrict__ kh = kp + (size_t)h * 16 * D;
    const float* __restrict__ vh = vp + (size_t)h * 16 * D;
    const unsigned page_elems = Hkv * 16 * D;
    const int last_rec = (((kend - 1) & 15) + 1) * D * 4;
    u32x4_t kst[KPT], vst[KPT];
    auto load = [&](int u) __attribute__((always_inline)) {
      if (u * kWidePages >= ids_at + 64) fetch_ids(u);
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        const int vi = u * kWidePages + pg0 + j * (kStep / 16);
        const int id = __builtin_amdgcn_readlane(ids, vi - ids_at);
        const size_t base = (size_t)(unsigned)max(id, 0) * page_elems;
        const int rec = id < 0 ? 0 : vi + 1 < pages ? 16 * D * 4 : last_rec;
        const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(kh + base), 0, rec,
                                                          kBufferWord3);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(vh + base), 0, rec,
                                                          kBufferWord3);
        kst[j] = __builtin_amdgcn_raw_buffer_load_b128(rk, voff, 0, 0);
        vst[j] = __builtin_amdgcn_raw_buffer_load_b128(rv, voff, 0, 0);
      }
      return (unsigned)(ids_ok >> (u * kWidePages - ids_at)) & 15u;
    };
    auto store = [&](int bf, bool whole) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        const int kk = kk0 + j * kStep;
        if (!whole) {
          bool odd = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool x = (vst[j][i] & 0x7f800000u) == 0x7f800000u;
            odd = odd || x;
            vst[j][i] = x ? 0u : vst[j][i];
          }
          if (odd) atomicOr(&s_odd[bf][kk >> 5], 1u << (kk & 31));
        }
        *reinterpret_cast<u32x4_t*>(&s.k[bf][kk][dc * 4]) = kst[j];
        *reinterpret_cast<u32x4_t*>(&s.v[bf][kk][dc * 4]) = vst[j];
      }
    };

    __syncthreads();  // the stages of the segment before are read
    if (tid < 4) s_odd[tid >> 1][tid & 1] = 0;
    __syncthreads();
    fetch_ids(u0);
    unsigned ok = load(u0), ok_next = 0;
    bool whole_t = ok == 15u && all.has(u0);
    store(0, whole_t);
    __syncthreads();
    int bf = 0;
    for (int u = u0;; ++u) {
      const bool more = u + 1 < u_end;
      if (more) ok_next = load(u + 1);  // in flight during this stage's math
      if (live) {
        f32x16_t x[2];
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[sb][i] = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int sb = 0; sb < 2; ++sb) {
            const float4 a = *reinterpret_cast<const float4*>(
                &s.k[bf][sb * 32 + col][half * (D / 2) + kb * 4]);
            x[sb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, q[kb].x, x[sb], 0, 0, 0);
            x[sb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, q[kb].y, x[sb], 0, 0, 0);
            x[sb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, q[kb].z, x[sb], 0, 0, 0);
            x[sb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, q[kb].w, x[sb], 0, 0, 0);
          }
        if (!(ok == 15u && mine.has(u))) {
#pragma unroll
          for (int sb = 0; sb < 2; ++sb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int kk = (i >> 2) * 8 + half * 4 + (i & 3), pg = sb * 2 + (i >> 3);
              const bool see = (ok >> pg & 1) &
                               span.sees(page_pos(u * kWidePages + pg) + (kk & 15), p.sinks);
              x[sb][i] = see ? x[sb][i] : -INFINITY;
            }
        }
        float mx = x[0][0];
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[sb][i]);
        if (__any(mx * p.c > m + kLazyLog2)) {
          const float mn = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)) * p.c);
          const float a = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
          l *= a;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= a;
          m = mn;
        }
        const float nm = m == -INFINITY ? 0.f : -m;
        float sum = 0.f;
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            x[sb][i] = __builtin_amdgcn_exp2f(fmaf(x[sb][i], p.c, nm));
            sum += x[sb][i];
          }
        l += sum;
#pragma unroll
        for (int sb = 0; sb < 2; ++sb)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float* v = &s.v[bf][sb * 32 + (j >> 2) * 8 + half * 4 + (j & 3)][col];
#pragma unroll
            for (int d = 0; d < DB; ++d)
              o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[d * 32], x[sb][j], o[d], 0, 0, 0);
          }
        if (!whole_t) {
          // What values of V that are not finite add to rows that see their keys.
          for (int sb = 0; sb < 2; ++sb) {
            uint32_t odd = __builtin_amdgcn_readfirstlane(s_odd[bf][sb]);
            while (odd) {
              const int kk = sb * 32 + __builtin_ctz(odd);
              odd &= odd - 1;
              if (!(ok >> (kk >> 4) & 1)) continue;
              const int pg = real_page(u * kWidePages + (kk >> 4), wp0, sink_pages);
              const float* src = vp + (((size_t)table[pg] * Hkv + h) * 16 + (kk & 15)) * D;
              const bool see = span.sees(pg * 16 + (kk & 15), p.sinks);
#pragma unroll
              for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float v = src[d * 32 + (i >> 2) * 8 + half * 4 + (i & 3)];
                  o[d][i] += see && !(v - v == 0.f) ? v : 0.f;
                }
            }
          }
        }
      }
      if (!more) break;
      ok = ok_next;
      whole_t = ok == 15u && all.has(u + 1);
      store(bf ^ 1, whole_t);
      __syncthreads();
      bf ^= 1;
    }

    wide_finish<float, D>(p, share, w, u0 > 0, u_end < units, live, wrow + col < rows, at, o, m,
                          l + __shfl_xor(l, 32, 64));
    left -= seg;
    if (ti-- == 0) {
      ti = tiles - 1;
      --h;
    }
    if (left > 0) {
      t = p.v.wide[ti];
      u_end = (__builtin_amdgcn_readfirstlane(t.pages) + kWidePages - 1) / kWidePages;
    }
  }
}

// Joins the wide tiles that were cut into three pieces or more: workgroup (b, d)
// dimension block d of the tile that workgroup b's share ends in, if it starts
// there. The pieces combine online in their order.
template <typename T, int D>
__global__ __launch_bounds__(kPartLanes) void chunk_merge_kernel(ChunkParams p) {
  constexpr int DB = D / 32;
  if (p.v.head->stamp != p.stamp) return;
  const ChunkShare share = p.v.wide_share[blockIdx.x / DB];
  const int w = share.w, d = blockIdx.x % DB;
  if (share.count == 0 || share.last < w + 2) return;  // three pieces or more
  const ChunkTile t = p.v.wide[share.end_tile];
  const int h = share.end_head;
  const int tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int row = t.row0 + wave * 32 + col, rows = t.n * p.G;
  if (row >= rows) return;
  float M = -INFINITY, L = 0.f, acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int k = w; k <= share.last; ++k) {
    const size_t slot = 2 * k + (k == w ? 1 : 0);
    const float4* part =
        reinterpret_cast<const float4*>(p.wide_part + slot * wide_part_floats(D)) + tid;
    const float4 ml = part[4 * DB * kPartLanes];
    float4 a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = part[(d * 4 + i) * kPartLanes];
    const float mn = fmaxf(M, ml.x);
    const float sa = state_weight(M, mn), sb = state_weight(ml.x, mn);
    L = L * sa + ml.y * sb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[i * 4] = acc[i * 4] * sa + a[i].x * sb;
      acc[i * 4 + 1] = acc[i * 4 + 1] * sa + a[i].y * sb;
      acc[i * 4 + 2] = acc[i * 4 + 2] * sa + a[i].z * sb;
      acc[i * 4 + 3] = acc[i * 4 + 3] * sa + a[i].w * sb;
    }
    M = mn;
  }
  const int tok = row / p.G;
  const size_t at = (size_t)(t.tok0 + tok) * p.Hq + h * p.G + row - tok * p.G;
  T* dst = static_cast<T*>(p.out) + at * D + d * 32;
  const float inv = inverse_sum(L);
#pragma unroll
  for (int i4 = 0; i4 < 4; ++i4) write_row<T, 4>(dst + i4 * 8 + half * 4, acc + i4 * 4, inv);
  if (p.lse && d == 0 && half == 0) p.lse[at] = state_lse(M, L);
}

// Workspace: header (word 0 unused by these kernels' errors, which the plan
// holds), the tiles' piece counts, then the pieces.
struct ChunkWorkspace {
  size_t done, wide_done, thin, wide, bytes;
};
ChunkWorkspace chunk_workspace(int max_rows, int D, int cus) {
  ChunkWorkspace ws;
  ws.done = 256;
  ws.wide_done = ws.done + (size_t)2 * cus * sizeof(uint32_t);
  ws.thin = ws.done + ((size_t)3 * cus * sizeof(uint32_t) + 255) / 256 * 256;
  ws.wide = ws.thin + (size_t)4 * cus * kThinRows * (D + 2) * sizeof(float);
  ws.bytes = ws.wide;
  if (max_rows > kThinRows)
    ws.bytes += (size_t)2 * cus * wide_part_floats(D) * sizeof(float);
  return ws;
}

template <typename T, int D>
int launch_chunk(const ChunkParams& p, int max_rows, int thin_rows, int waves, bool shared,
                 int cus, hipStream_t stream) {
  int st = RLSE_OK;
  if (thin_rows > 0) {
    auto run = [&](auto rt, auto w) {
      constexpr int RT = decltype(rt)::value, W = decltype(w)::value;
      const dim3 grid(thin_groups(cus, W)), block(64 * W);
      if (shared)
        hipLaunchKernelGGL((chunk_thin_kernel<T, D, RT, W, false>), grid, block, 0, stream, p);
      else
        hipLaunchKernelGGL((chunk_thin_kernel<T, D, RT, W, true>), grid, block, 0, stream, p);
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 8> eight;
    if (waves == 8)
      max_rows <= 16 ? run(one, eight) : run(two, eight);
    else
      max_rows <= 16 ? run(one, four) : run(two, four);
    st = launch_status("chunk_thin_kernel");
  }
  if (st || max_rows <= thin_rows) return st;
  if constexpr (sizeof(T) == 4)
    hipLaunchKernelGGL((chunk_wide32_kernel<D>), dim3(cus), dim3(kWide32Threads), 0, stream, p);
  else
    hipLaunchKernelGGL((chunk_wide_kernel<T, D>), dim3(cus), dim3(kWideThreads), 0, stream, p);
  st = launch_status("chunk_wide_kernel");
  if (st) return st;
  hipLaunchKernelGGL((chunk_merge_kernel<T, D>), dim3(cus * (D / 32)), dim3(kPartLanes), 0,
                     stream, p);
  return launch_status("chunk_merge_kernel");
}

}  // namespace
}  // namespace rlse

using namespace rlse;

extern "C" int rlse_chunk_workspace_size(int num_seqs, int total_tokens, int max_tokens,
                                         int num_heads, int num_kv_heads, int head_dim,
                                         size_t* bytes) {
  if (!bytes) return fail(RLSE_ERR_INVALID_VALUE, "chunk_workspace_size: null output");
  int st = validate_chunk_shape("chunk_workspace_size", num_seqs, total_tokens, max_tokens,
                                num_heads, num_kv_heads, 1, 0, 0);
  if (st) return st;
  if (head_dim != 64 && head_dim != 128)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_workspace_size: head_dim %d not in {64, 128}",
                head_dim);
  int cus = 0;
  st = device_cu_count(&cus);
  if (st) return st;
  *bytes = chunk_workspace(max_tokens * (num_heads / num_kv_heads), head_dim, cus).bytes;
  return RLSE_OK;
}

extern "C" int rlse_chunk_attn(const void* q, const void* k_pool, const void* v_pool,
                               const int32_t* block_tables, void* plan, void* out, float* lse,
                               int num_seqs, int total_tokens, int max_tokens, int num_heads,
                               int num_kv_heads, int head_dim, int max_blocks_per_seq,
                               int num_blocks, int window, int sinks, float scale, int dtype,
                               void* workspace, size_t workspace_bytes, int flags,
                               rlse_stream_t stream) {
  int st = validate_chunk_shape("chunk_attn", num_seqs, total_tokens, max_tokens, num_heads,
                                num_kv_heads, max_blocks_per_seq, window, sinks);
  if (st) return st;
  if (head_dim != 64 && head_dim != 128)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_attn: head_dim %d not in {64, 128}", head_dim);
  if (dtype != RLSE_DTYPE_BF16 && dtype != RLSE_DTYPE_F16 && dtype != RLSE_DTYPE_F32)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_attn: bad dtype %d", dtype);
  if (num_blocks <= 0)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_attn: num_blocks %d", num_blocks);
  if (!(scale > 0.f) || !isfinite(scale))
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_attn: scale must be finite and positive");
  if (flags & ~RLSE_CHUNK_SHARED_PAGES)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_attn: unknown flags 0x%x", flags);
  if (!q || !k_pool || !v_pool || !block_tables || !plan || !out || !workspace)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_attn: null pointer argument");
  const uintptr_t align = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) |
                          reinterpret_cast<uintptr_t>(v_pool) | reinterpret_cast<uintptr_t>(plan) |
                          reinterpret_cast<uintptr_t>(out) |
                          reinterpret_cast<uintptr_t>(workspace);
  if (align & 15)
    return fail(RLSE_ERR_INVALID_VALUE, "chunk_attn: a buffer is not 16-byte aligned");
  int cus = 0;
  st = device_cu_count(&cus);
  if (st) return st;
  ChunkParams p{};
  p.G = num_heads / num_kv_heads;
  const int max_rows = max_tokens * p.G;
  const ChunkWorkspace ws = chunk_workspace(max_rows, head_dim, cus);
  if (workspace_bytes < ws.bytes)
    return fail(RLSE_ERR_BUFFER_TOO_SMALL, "chunk_attn: workspace %zu bytes < %zu needed",
                workspace_bytes, ws.bytes);
  char* base = static_cast<char*>(workspace);
  p.q = q;
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.tables = block_tables;
  p.out = out;
  p.lse = lse;
  p.v = chunk_plan_view(plan, num_seqs, total_tokens, p.G, cus);
  p.stamp = chunk_stamp({num_seqs, total_tokens, max_tokens, num_heads, num_kv_heads,
                         max_blocks_per_seq, window, sinks, cus});
  p.thin_done = reinterpret_cast<uint32_t*>(base + ws.done);
  p.thin_part = reinterpret_cast<float*>(base + ws.thin);
  p.wide_part = reinterpret_cast<float*>(base + ws.wide);
  p.wide_done = reinterpret_cast<uint32_t*>(base + ws.wide_done);
  p.Hq = num_heads;
  p.Hkv = num_kv_heads;
  p.mbps = max_blocks_per_seq;
  p.num_blocks = num_blocks;
  p.window = window;
  p.sinks = sinks;
  p.c = scale * 1.4426950408889634f;
  const hipStream_t s = as_stream(stream);
  auto run = [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    return launch_chunk<T, D>(p, max_rows, thin_row_limit(num_seqs, max_rows),
                              thin_waves(num_seqs, num_kv_heads, cus),
                              flags & RLSE_CHUNK_SHARED_PAGES, cus, s);
  };
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  if (dtype == RLSE_DTYPE_BF16) return head_dim == 128 ? run(bf16{}, d128) : run(bf16{}, d64);
  if (dtype == RLSE_DTYPE_F16) return head_dim == 128 ? run(f16{}, d128) : run(f16{}, d64);
  return head_dim == 128 ? run(float{}, d128) : run(float{}, d64);
}
