// Eviction from the paged cache by accumulated weight (gfx950). For every
// layer, sequence and KV head of more than `budget` keys, the first `sinks`,
// the last `recent` and the heaviest of those between stay, `budget` in all,
// in their order; their K and V rows and weights move to fresh pages. No
// counterpart in the reference, which drops nothing but whole requests. The
// old pages are only read, so pages shared with other sequences or with the
// prefix cache need no copy first, and no row waits for another.
//
//  - Selection: one workgroup per (layer, sequence, head). The m-th heaviest
//    weight is found by three histograms (11, 11 and 10 bits) of the weights'
//    order-preserving bit patterns, then the kept keys are numbered by ballots
//    in key order: weights above it, and of those equal to it the first ones.
//    No float arithmetic, and integer counts only: the answer is exact. Bound by
//    the barriers between its passes: 8 us for one head of 1500 keys, 58 us for
//    3584 heads of 1500-4096.
//  - Move: HBM bound, a copy of rows picked by index, with non-temporal loads
//    and stores, for nothing is read twice (Qwen3-0.6B, 28 layers of 16
//    sequences cut to 1024 keys, 3.8 GB: 682 us, 5.5 TB/s; 737 us cacheable,
//    as a copy of contiguous memory takes). A second launch: in one with the
//    selection, each workgroup moving its own head, too few loads are in
//    flight (780 us for the two at their best, 743 apart).
#include <math.h>

#include "common.cuh"
#include "host_common.h"

namespace rlse {
namespace {

struct EvictParams {
  const void* k_pool;
  const void* v_pool;
  const int* tables;       // [B][mbps]
  const int* lens;
  long long layer_packets;  // between layers' pools
  const float* scores;     // [L] x [B][Hkv][mbps*16]
  long long score_stride;
  const int* new_tables;   // [B][nbps]
  int* new_lens;
  float* new_scores;       // as scores
  int* keep;               // [L][B][Hkv][budget]
  int layers, B, Hkv, mbps, nbps, num_blocks, budget, sinks, recent;
};

__device__ __forceinline__ int evict_len(const EvictParams& p, int b) {
  const int len = p.lens[b];
  return len < 0 || len > p.mbps * 16 ? 0 : len;
}

constexpr int kSelectThreads = 512;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kBins = 2048;
constexpr int kCached = 4096;  // weights' patterns held in LDS (16 KB: four workgroups a CU)

// Larger weights have larger patterns; both zeros the same one; NaN the
// smallest of all, 0.
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Numbers the kept keys of the workgroup's head and moves their weights.
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictParams p) {
  __shared__ uint32_t s_key[kCached];
  __shared__ int s_bin[kBins];
  __shared__ int s_wave[kSelectWaves][2];
  __shared__ int s_pick[2];  // bin of the m-th heaviest, and its rank in the bin
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.x % p.Hkv;
  const int lb = blockIdx.x / p.Hkv;
  const int b = lb % p.B, layer = lb / p.B;
  const int len = evict_len(p, b);
  const int budget = p.budget;
  const size_t row = (size_t)layer * p.score_stride + ((size_t)b * p.Hkv + h) * p.mbps * 16;
  const float* __restrict__ w = p.scores + row;
  float* __restrict__ nw = p.new_scores + row;
  int* keep = p.keep + (size_t)blockIdx.x * budget;
  if (layer == 0 && h == 0 && tid == 0) p.new_lens[b] = min(len, budget);

  if (len <= budget) {
    for (int i = tid; i < budget; i += kSelectThreads) {
      keep[i] = i < len ? i : -1;
      if (i < len) nw[i] = w[i];
    }
    return;
  }
  // The ends stay; of the mid keys from `sinks` on, the `want` heaviest do.
  const int mid = len - p.sinks - p.recent, want = budget - p.sinks - p.recent;
  for (int i = tid; i < p.sinks; i += kSelectThreads) {
    keep[i] = i;
    nw[i] = w[i];
  }
  for (int i = tid; i < p.recent; i += kSelectThreads) {
    keep[budget - p.recent + i] = len - p.recent + i;
    nw[budget - p.recent + i] = w[len - p.recent + i];
  }
  if (want == 0) return;
  const float* __restrict__ mw = w + p.sinks;
  for (int i = tid; i < min(mid, kCached); i += kSelectThreads) s_key[i] = weight_order(mw[i]);
  auto key_of = [&](int i) __attribute__((always_inline)) {
    return i < kCached ? s_key[i] : weight_order(mw[i]);
  };

  // Digit by digit from the top: the bin that holds the m-th heaviest of the
  // keys that agree with the digits so far.
  uint32_t prefix = 0;
  int rank = want;  // of the key sought among those that agree, from 1
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const int bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kBins; i += kSelectThreads) s_bin[i] = 0;
    __syncthreads();
    for (int i = tid; i < mid; i += kSelectThreads) {
      const uint32_t k = key_of(i);
      if (pass == 0 || k >> (shift + bits) == prefix)
        atomicAdd(&s_bin[k >> shift & ((1u << bits) - 1)], 1);
    }
    __syncthreads();
    // Keys in the bins above each thread's own four, heaviest bins first.
    constexpr int PER = kBins / kSelectThreads;
    int mine[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      mine[i] = s_bin[kBins - 1 - (tid * PER + i)];
      sum += mine[i];
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(inc, o, 64);
      if (lane >= o) inc += y;
    }
    if (lane == 63) s_wave[wave][0] = inc;
    __syncthreads();
    int before = inc - sum;
    for (int i = 0; i < wave; ++i) before += s_wave[i][0];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (before < rank && rank <= before + mine[i]) {
        s_pick[0] = kBins - 1 - (tid * PER + i);
        s_pick[1] = rank - before;
      }
      before += mine[i];
    }
    __syncthreads();
    prefix = prefix << bits | (uint32_t)s_pick[0];
    rank = s_pick[1];
  }
  // Keys above `prefix` stay, and the first `rank` of those equal to it. Each
  // wave numbers a run of consecutive keys: count, then place.
  const int run = ((mid + kSelectWaves - 1) / kSelectWaves + 63) & ~63;
  const int begin = min(wave * run, mid), end = min(begin + run, mid);
  int gt = 0, eq = 0;
  for (int i0 = begin; i0 < end; i0 += 64) {
    const int i = i0 + lane;
    const uint32_t k = i < end ? key_of(i) : 0u;
    gt += __popcll(__ballot(i < end && k > prefix));
    eq += __popcll(__ballot(i < end && k == prefix));
  }
  if (lane == 0) {
    s_wave[wave][0] = gt;
    s_wave[wave][1] = eq;
  }
  __syncthreads();
  gt = eq = 0;
  for (int i = 0; i < wave; ++i) {
    gt += s_wave[i][0];
    eq += s_wave[i][1];
  }
  const unsigned long long below = (1ull << lane) - 1;
  for (int i0 = begin; i0 < end; i0 += 64) {
    const int i = i0 + lane;
    const uint32_t k = i < end ? key_of(i) : 0u;
    const unsigned long long mg = __ballot(i < end && k > prefix);
    const unsigned long long me = __ballot(i < end && k == prefix);
    const int g = gt + __popcll(mg & below), e = eq + __popcll(me & below);
    if (i < end && (k > prefix || (k == prefix && e < rank))) {
      keep[p.sinks + g + min(e, rank)] = p.sinks + i;
    }
    gt += __popcll(mg);
    eq += __popcll(me);
  }
  // Their weights, once keep is written (in the loop each would wait for its
  // own load).
  __syncthreads();
  for (int i = p.sinks + tid; i < p.sinks + want; i += kSelectThreads) nw[i] = w[keep[i]];
}

constexpr int kMoveThreads = 256;
constexpr int kMovePackets = 2;  // per thread, of K and of V

// PPR: 16-byte packets per row.
template <int PPR>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictParams p, int groups) {
  constexpr int kRows = kMovePackets * kMoveThreads / PPR;
  const int r = blockIdx.x / groups;  // (layer * B + b) * Hkv + h
  const int h = r % p.Hkv, lb = r / p.Hkv, b = lb % p.B, layer = lb / p.B;
  const int first = blockIdx.x % groups * kRows, end = min(evict_len(p, b), p.budget);
  const int* __restrict__ keep = p.keep + (size_t)r * p.budget;
  const int* __restrict__ table = p.tables + (size_t)b * p.mbps;
  const int* __restrict__ fresh = p.new_tables + (size_t)b * p.nbps;
  const u32x4_t* kp = static_cast<const u32x4_t*>(p.k_pool) + (size_t)layer * p.layer_packets;
  const u32x4_t* vp = static_cast<const u32x4_t*>(p.v_pool) + (size_t)layer * p.layer_packets;
  u32x4_t* ko = const_cast<u32x4_t*>(kp);
  u32x4_t* vo = const_cast<u32x4_t*>(vp);
  u32x4_t k[kMovePackets], v[kMovePackets];
  size_t to[kMovePackets];
  bool ok[kMovePackets];
#pragma unroll
  for (int i = 0; i < kMovePackets; ++i) {
    const int pk = threadIdx.x + i * kMoveThreads;
    const int j = first + pk / PPR, c = pk % PPR;
    ok[i] = false;
    if (j < end) {
      const int src = keep[j];
      const int from = table[src >> 4], dst = fresh[j >> 4];
      ok[i] = (unsigned)from < (unsigned)p.num_blocks && (unsigned)dst < (unsigned)p.num_blocks;
      const size_t at = (((size_t)(ok[i] ? from : 0) * p.Hkv + h) * 16 + (src & 15)) * PPR + c;
      to[i] = (((size_t)(ok[i] ? dst : 0) * p.Hkv + h) * 16 + (j & 15)) * PPR + c;
      if (ok[i]) {
        k[i] = __builtin_nontemporal_load(kp + at);
        v[i] = __builtin_nontemporal_load(vp + at);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kMovePackets; ++i)
    if (ok[i]) {
      __builtin_nontemporal_store(k[i], ko + to[i]);
      __builtin_nontemporal_store(v[i], vo + to[i]);
    }
}

// Whether a layer of a and one of b, `bytes` each and `stride` bytes apart, share
// a byte. (Two sets of weights may lie between each other, layer by layer.)
bool layers_overlap(const void* a, const void* b, int layers, long long stride, long long bytes) {
  const long long delta = (long long)(reinterpret_cast<uintptr_t>(b) -
                                      reinterpret_cast<uintptr_t>(a));
  if (layers == 1) return delta < bytes && delta > -bytes;
  // The whole strides next below and above their distance.
  long long k = delta / stride;
  if (delta < k * stride) --k;
  for (int i = 0; i < 2; ++i, ++k) {
    const long long off = delta - k * stride;
    if (k < layers && k > -layers && off < bytes && off > -bytes) return true;
  }
  return false;
}

template <int PPR>
int launch_evict(const EvictParams& p, int heads, hipStream_t stream) {
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)heads), dim3(kSelectThreads), 0, stream,
                     p);
  const int st = launch_status("evict_select_kernel");
  if (st) return st;
  constexpr int kRows = kMovePackets * kMoveThreads / PPR;
  const int groups = (p.budget + kRows - 1) / kRows;
  hipLaunchKernelGGL((evict_move_kernel<PPR>), dim3((unsigned)(heads * groups)),
                     dim3(kMoveThreads), 0, stream, p, groups);
  return launch_status("evict_move_kernel");
}

}  // namespace
}  // namespace rlse

using namespace rlse;

extern "C" int rlse_kv_evict(void* k_pool, void* v_pool, long long layer_stride_elems,
                             int num_layers, const int32_t* block_tables,
                             const int32_t* seq_lens, const float* scores,
                             long long score_layer_stride, const int32_t* new_tables,
                             int32_t* new_lens, float* new_scores, int32_t* keep, int num_seqs,
                             int num_kv_heads, int head_dim, int max_blocks_per_seq,
                             int new_blocks_per_seq, int num_blocks, int budget, int sinks,
                             int recent, int dtype, rlse_stream_t stream) {
  const size_t es = dtype_size(dtype);
  if (es == 0) return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: bad dtype %d", dtype);
  if (head_dim != 64 && head_dim != 128)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: head_dim %d not in {64, 128}", head_dim);
  if (num_layers <= 0 || num_seqs <= 0 || num_kv_heads <= 0 || num_blocks <= 0)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: bad shape (layers %d, seqs %d, heads %d)",
                num_layers, num_seqs, num_kv_heads);
  if (max_blocks_per_seq <= 0 || max_blocks_per_seq > (1 << 24) || new_blocks_per_seq <= 0)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: bad table widths %d, %d", max_blocks_per_seq,
                new_blocks_per_seq);
  if (budget <= 0 || budget > max_blocks_per_seq * 16 ||
      (long long)new_blocks_per_seq * 16 < budget)
    return fail(RLSE_ERR_INVALID_VALUE,
                "kv_evict: budget %d outside 1..%d or above the new tables' %lld keys", budget,
                max_blocks_per_seq * 16, new_blocks_per_seq * 16LL);
  if (sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: sinks %d + recent %d outside 0..budget %d",
                sinks, recent, budget);
  const long long row = (long long)num_seqs * num_kv_heads * max_blocks_per_seq * 16;
  const long long page = (long long)num_kv_heads * 16 * head_dim;
  if (num_layers > 1 && (score_layer_stride < row || layer_stride_elems < page * num_blocks ||
                         layer_stride_elems * (long long)es % 16 != 0))
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: layer strides %lld, %lld too small or odd",
                layer_stride_elems, score_layer_stride);
  const long long heads = (long long)num_layers * num_seqs * num_kv_heads;
  if (heads * ((long long)budget / 8 + 1) > 0x7fffffffLL)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: too many heads and keys for one call");
  if (!k_pool || !v_pool || !block_tables || !seq_lens || !scores || !new_tables || !new_lens ||
      !new_scores || !keep)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: null pointer argument");
  if (layers_overlap(scores, new_scores, num_layers, score_layer_stride * 4, row * 4))
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: new_scores overlaps scores");
  if (overlap(seq_lens, (size_t)num_seqs * 4, new_lens, (size_t)num_seqs * 4))
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: new_lens overlaps seq_lens");
  if ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15)
    return fail(RLSE_ERR_INVALID_VALUE, "kv_evict: a pool is not 16-byte aligned");
  EvictParams p{};
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.tables = block_tables;
  p.lens = seq_lens;
  p.scores = scores;
  p.score_stride = num_layers > 1 ? score_layer_stride : 0;
  p.new_tables = new_tables;
  p.new_lens = new_lens;
  p.new_scores = new_scores;
  p.keep = keep;
  p.layers = num_layers;
  p.B = num_seqs;
  p.Hkv = num_kv_heads;
  p.mbps = max_blocks_per_seq;
  p.nbps = new_blocks_per_seq;
  p.num_blocks = num_blocks;
  p.budget = budget;
  p.sinks = sinks;
  p.recent = recent;
  p.layer_packets = num_layers > 1 ? layer_stride_elems * (long long)es / 16 : 0;
  const hipStream_t s = as_stream(stream);
  switch (head_dim * es / 16) {
    case 8:
      return launch_evict<8>(p, (int)heads, s);
    case 16:
      return launch_evict<16>(p, (int)heads, s);
    default:
      return launch_evict<32>(p, (int)heads, s);
  }
}
