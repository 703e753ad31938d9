// Gradient of a token table by sorted tokens (no reference counterpart):
// grad[v] (+)= scale * sum over t with tokens[t] = v, t ascending, of drop(dy[t]).
//
//   1. a stable radix sort of (token, position) pairs; padding and
//      out-of-range tokens get the key `vocab` and sort behind the others.  Up
//      to 131,072 tokens one cluster of CTAs sorts in its shared memory;
//   2. sum_kernel: the sorted positions are cut into tiles of K; one thread
//      holds eight columns of a tile and adds its rows in order in FP32
//      registers, writing a row of grad at each end of a run.  The parts of a
//      run that crosses tiles are added through shared memory among the tiles
//      of a CTA, its block; a run that crosses blocks leaves FP32 partial rows
//      in the scratch.  More CTAs of the same grid zero the rows of an
//      overwritten grad that no token names;
//   3. join_kernel adds such a run's partial rows in a fixed order.
// Up to kSmallTokens, step 1 is left out: every CTA of the sums sorts the
// tokens for itself.
// No atomics on floats: the same inputs give the same bits.
//
// Bounds (B200).  65,539 bf16 rows of 4,096 into an FP32 table of 131,072 rows:
// 412 us for 2.63 GB, 0.98 of the copy bandwidth (sort 31, sums and zeros 367,
// joins 7).  32,768 rows of 2,048, dropout on, added to a table of 32,768 rows:
// 97 us (sort 14, sums 76, joins 8; the bytes take 44), the sums held by the
// masks' instructions (25 per element, 2.6 a cycle and SM); without dropout 78 us
// (sums 49).  There 1,024 CTAs of sums share 592 places, 1.7 waves.  262,144 bf16
// rows of 512 into an FP32 table of 50,000: 141 us where the bytes take 57 (sort
// 78, sums 59, joins 8).  Small calls are chains of launches and latencies: 14 us
// for 300 tokens.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "dfc_philox.cuh"

namespace dfc {
namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kNoKey = 0xFFFFFFFFu;

// Programmatic dependent launch: the next kernel's CTAs may become resident
// early; they wait here until the kernel before is complete.
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- rows without a token ---------------------------------------------------
// Zeros are zeros in every type: rows as bytes.
struct Fill {
  char* grad;
  int64_t pitch, bytes;  // of a row
  int64_t rows;
  int per_warp;          // rows of a warp, at most 32
  int unit;              // 16, 4 or 2: grad, pitch and bytes are multiples of it
};

constexpr int kZeroBytes = 16384;
constexpr int kBulkBytes = 512;  // shorter rows are written by ordinary stores

__device__ __forceinline__ void clear_zeros(void* zeros) {
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  for (int i = tid; i < kZeroBytes / 16; i += blockDim.x * blockDim.y)
    static_cast<uint4*>(zeros)[i] = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// One warp: zeros for the rows first + r whose bit r of `empty` is set.  Long
// rows are bulk copies from zeros in shared memory, one lane a row, so that the
// rate does not depend on how many threads an SM holds (16-byte stores: 554 us
// instead of 370 for 1.8 GB with 512 threads per SM).
__device__ __forceinline__ void fill_rows(const Fill& f, int64_t first, uint32_t empty, const void* zeros) {
  const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31;
  if (f.unit == 16 && f.bytes >= kBulkBytes) {
    if ((empty >> lane) & 1u) {
      char* row = f.grad + (first + lane) * f.pitch;
      const uint32_t from = static_cast<uint32_t>(__cvta_generic_to_shared(zeros));
      for (int64_t at = 0; at < f.bytes; at += kZeroBytes)
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(row + at), "r"(from),
                     "r"(static_cast<uint32_t>(min(f.bytes - at, static_cast<int64_t>(kZeroBytes))))
                     : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    return;
  }
  for (; empty; empty &= empty - 1) {
    char* row = f.grad + (first + __ffs(empty) - 1) * f.pitch;
    for (int64_t at = static_cast<int64_t>(lane) * f.unit; at < f.bytes; at += 32 * f.unit) {
      if (f.unit == 16)
        *reinterpret_cast<uint4*>(row + at) = make_uint4(0u, 0u, 0u, 0u);
      else if (f.unit == 4)
        *reinterpret_cast<uint32_t*>(row + at) = 0u;
      else
        *reinterpret_cast<uint16_t*>(row + at) = 0;
    }
  }
}

__device__ __forceinline__ void fill_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ---- 1. sort ------------------------------------------------------------------
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;

struct Tokens {
  const void* ids;
  int wide;
  int64_t vocab;
  int64_t padding_idx;
  int32_t* error_flag;
};

__device__ __forceinline__ uint32_t token_key(const Tokens& tk, int64_t t) {
  const int64_t v = tk.wide ? static_cast<const int64_t*>(tk.ids)[t]
                            : static_cast<int64_t>(static_cast<const int32_t*>(tk.ids)[t]);
  if (static_cast<uint64_t>(v) >= static_cast<uint64_t>(tk.vocab)) {
    if (tk.error_flag) *tk.error_flag = 1;
    return static_cast<uint32_t>(tk.vocab);
  }
  return v == tk.padding_idx ? static_cast<uint32_t>(tk.vocab) : static_cast<uint32_t>(v);
}

// Item `round` of a thread: warp w owns kSortItems * 32 consecutive items.
__device__ __forceinline__ int64_t sort_item(int round) {
  return static_cast<int64_t>(blockIdx.x) * kSortTile + (threadIdx.x >> 5) * (kSortItems * 32) +
         round * 32 + (threadIdx.x & 31);
}

// Counts of each digit in each tile: hist[digit * tiles + tile].  The first
// pass makes the keys from the tokens, the others read them.
__global__ void __launch_bounds__(kSortThreads)
    sort_count_kernel(Tokens tk, const uint32_t* keys, int64_t n, int shift, int bins, uint32_t* hist) {
  __shared__ uint32_t count[kMaxBins];
  for (int b = threadIdx.x; b < bins; b += kSortThreads) count[b] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = sort_item(r);
    if (i < n) {
      const uint32_t key = keys ? keys[i] : token_key(tk, i);
      atomicAdd(&count[(key >> shift) & (bins - 1)], 1u);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads)
    hist[static_cast<int64_t>(b) * gridDim.x + blockIdx.x] = count[b];
}

// The lanes of the warp whose digit is this lane's, among those with `on`:
// one ballot per digit bit.  (MATCH.ANY measured 22.2 us for the sort of
// 32,768 tokens.)
__device__ __forceinline__ uint32_t same_digit(uint32_t digit, bool on, int bits) {
  uint32_t same = __ballot_sync(0xFFFFFFFFu, on);
#pragma unroll
  for (int b = 0; b < kMaxDigitBits; ++b) {
    if (b < bits) {
      const bool one = (digit >> b) & 1u;
      const uint32_t ones = __ballot_sync(0xFFFFFFFFu, one);
      same &= one ? ones : ~ones;
    }
  }
  return same;
}

__device__ __forceinline__ uint32_t warp_inclusive(uint32_t x) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, d);
    if ((threadIdx.x & 31) >= d) x += y;
  }
  return x;
}

// Exclusive scan of `total` counts in place, one CTA of 1024 threads: 18 us for
// the 32,768 counts of a pass over 262,144 tokens, beside 8 for the count and 12
// to 14 for the scatter.
__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t* hist, int64_t total) {
  __shared__ uint32_t warp_sum[32];
  __shared__ uint32_t carry;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int64_t base = 0; base < total; base += 4096) {
    const int64_t i = base + 4 * threadIdx.x;
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < total ? hist[i + j] : 0u;
    const uint32_t mine = v[0] + v[1] + v[2] + v[3];
    const uint32_t inc = warp_inclusive(mine);
    if ((threadIdx.x & 31) == 31) warp_sum[threadIdx.x >> 5] = inc;
    __syncthreads();
    if (threadIdx.x < 32) warp_sum[threadIdx.x] = warp_inclusive(warp_sum[threadIdx.x]);
    __syncthreads();
    uint32_t run = carry + inc - mine + (threadIdx.x >= 32 ? warp_sum[(threadIdx.x >> 5) - 1] : 0u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i + j < total) hist[i + j] = run;
      run += v[j];
    }
    __syncthreads();
    if (threadIdx.x == 0) carry += warp_sum[31];
    __syncthreads();
  }
}

// Items to their places: the digit's base in this tile, plus the earlier
// warps' items of the digit, plus the warp's own earlier ones.
__global__ void __launch_bounds__(kSortThreads)
    sort_scatter_kernel(Tokens tk, const uint32_t* keys, const uint32_t* pos, int64_t n, int shift,
                        int bins, const uint32_t* hist, uint32_t* out_keys, uint32_t* out_pos) {
  __shared__ uint32_t count[kSortWarps][kMaxBins];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = threadIdx.x; b < kSortWarps * kMaxBins; b += kSortThreads) (&count[0][0])[b] = 0;
  __syncthreads();
  uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = sort_item(r);
    const bool on = i < n;
    key[r] = !on ? 0u : keys ? keys[i] : token_key(tk, i);
    const uint32_t d = (key[r] >> shift) & (bins - 1);
    const uint32_t same = same_digit(d, on, __ffs(bins) - 1);
    uint32_t before = 0;
    if (on) before = count[warp][d];
    rank[r] = before + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (on && (same >> lane) == 1u) count[warp][d] = rank[r] + 1;  // the last lane of the digit
    __syncwarp();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads) {
    uint32_t run = hist[static_cast<int64_t>(b) * gridDim.x + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = count[w][b];
      count[w][b] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int64_t i = sort_item(r);
    if (i < n) {
      const uint32_t at = count[warp][(key[r] >> shift) & (bins - 1)] + rank[r];
      out_keys[at] = key[r];
      out_pos[at] = keys ? pos[i] : static_cast<uint32_t>(i);
    }
  }
}

// The whole sort in one cluster: CTA q holds the items [q * chunk, (q + 1) *
// chunk) of the current order in registers, ITEMS a thread.  A pass counts the
// digits of each warp's items, turns the counts into places (prefix over the
// warps here, over the digits and CTAs through distributed shared memory),
// orders the CTA's items in shared memory, so that a warp then sends runs of
// neighbouring items, and sends each to the CTA that owns its place; the last
// pass writes to global memory.  (Items sent straight from their threads, one
// scattered 8-byte store each: 42 us for 65,536 tokens on 8 CTAs.)
constexpr int kClusterThreads = 1024;
constexpr int kClusterWarps = kClusterThreads / 32;
constexpr int kMaxClusterItems = 8;
template <int ITEMS>
constexpr size_t cluster_smem(int bins) {
  return static_cast<size_t>(bins) * (2 * kClusterWarps + 2 + 2 * 4) + 2 * 8 * kClusterThreads * ITEMS;
}

template <int ITEMS>
__global__ void __launch_bounds__(kClusterThreads, 1)
    sort_cluster_kernel(Tokens tk, uint32_t n, int passes, int digit_bits, uint32_t* out_keys,
                        uint32_t* out_pos) {
  constexpr uint32_t kChunk = kClusterThreads * ITEMS;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint32_t warp_own[kClusterWarps], warp_all[kClusterWarps];
  const uint32_t bins = 1u << digit_bits;
  uint2* ordered = reinterpret_cast<uint2*>(smem);
  uint2* arrived = ordered + kChunk;
  uint32_t* start = reinterpret_cast<uint32_t*>(arrived + kChunk);  // places of the digits in `ordered`
  uint32_t* move = start + bins;                                    // from there to the whole order
  uint16_t* total = reinterpret_cast<uint16_t*>(move + bins);       // this CTA's items per digit
  uint16_t* count = total + bins;                                   // [warp][digit]
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), ctas = cluster.num_blocks();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t item0 = warp * (ITEMS * 32) + lane;  // + 32 per round
  const uint32_t here = n > rank * kChunk ? min(n - rank * kChunk, kChunk) : 0u;  // items of this CTA
  uint32_t key[ITEMS], pos[ITEMS];
  let_next_start();
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    pos[r] = rank * kChunk + item0 + 32 * r;
    key[r] = item0 + 32 * r < here ? token_key(tk, pos[r]) : 0u;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * digit_bits;
    for (uint32_t i = threadIdx.x; i < bins * kClusterWarps / 2; i += kClusterThreads)
      reinterpret_cast<uint32_t*>(count)[i] = 0u;
    uint32_t place[ITEMS];  // among the equal digits of the round, bit 8: the last of them
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const bool on = item0 + 32 * r < here;
      const uint32_t same = same_digit((key[r] >> shift) & (bins - 1), on, digit_bits);
      place[r] = __popc(same & ((1u << lane) - 1)) | (on && (same >> lane) == 1u ? 256u : 0u);
    }
    __syncthreads();
    uint16_t* mine = count + warp * bins;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {  // then among the warp's equal digits
      const uint32_t d = (key[r] >> shift) & (bins - 1);
      const bool last = place[r] & 256u;
      place[r] = (place[r] & 255u) + mine[d];
      __syncwarp();
      if (last) mine[d] = static_cast<uint16_t>(place[r] + 1);
      __syncwarp();
    }
    __syncthreads();
    uint32_t own = 0, all = 0, earlier = 0;
    if (threadIdx.x < bins) {
#pragma unroll 16
      for (int w = 0; w < kClusterWarps; ++w) {
        const uint32_t c = count[w * bins + threadIdx.x];
        count[w * bins + threadIdx.x] = static_cast<uint16_t>(own);
        own += c;
      }
      total[threadIdx.x] = static_cast<uint16_t>(own);
    }
    cluster.sync();
    if (threadIdx.x < bins) {
#pragma unroll 8
      for (uint32_t q = 0; q < ctas; ++q) {
        const uint32_t c = cluster.map_shared_rank(total, q)[threadIdx.x];
        earlier += q < rank ? c : 0u;
        all += c;
      }
    }
    const bool last = p + 1 == passes;
    // nothing of this CTA's shared memory is read by others after this: they
    // meet again before the first one leaves
    if (last) cluster.barrier_arrive();
    const uint32_t own_inc = warp_inclusive(own), all_inc = warp_inclusive(all);
    if (lane == 31) {
      warp_own[warp] = own_inc;
      warp_all[warp] = all_inc;
    }
    __syncthreads();
    if (warp == 0) warp_own[lane] = warp_inclusive(warp_own[lane]);
    if (warp == 1) warp_all[lane] = warp_inclusive(warp_all[lane]);
    __syncthreads();
    if (threadIdx.x < bins) {
      const uint32_t first = own_inc - own + (warp > 0 ? warp_own[warp - 1] : 0u);
      start[threadIdx.x] = first;
      move[threadIdx.x] = earlier + all_inc - all + (warp > 0 ? warp_all[warp - 1] : 0u) - first;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      if (item0 + 32 * r < here) {
        const uint32_t d = (key[r] >> shift) & (bins - 1);
        ordered[start[d] + mine[d] + place[r]] = make_uint2(key[r], pos[r]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const uint32_t i = threadIdx.x + r * kClusterThreads;
      if (i < here) {
        const uint2 kp = ordered[i];
        const uint32_t at = i + move[(kp.x >> shift) & (bins - 1)];
        if (last) {
          out_keys[at] = kp.x;
          out_pos[at] = kp.y;
        } else {
          cluster.map_shared_rank(arrived, at / kChunk)[at % kChunk] = kp;
        }
      }
    }
    if (last) {
      cluster.barrier_wait();
    } else {
      cluster.sync();  // the items have arrived
#pragma unroll
      for (int r = 0; r < ITEMS; ++r) {
        if (item0 + 32 * r < here) {
          const uint2 kp = arrived[item0 + 32 * r];
          key[r] = kp.x;
          pos[r] = kp.y;
        }
      }
    }
  }
}

// ---- 2. sums of runs ------------------------------------------------------------
// Everything but addresses fits 32 bits: a row's place is one 32 x 32 -> 64-bit
// product.
struct SumArgs {
  const uint32_t* keys;  // sorted
  const uint32_t* pos;
  uint32_t n;
  uint32_t tile;         // K
  uint32_t block;        // positions of a CTA's tiles
  const void* dy;
  uint32_t dy_pitch;
  void* grad;
  uint32_t grad_pitch;
  uint32_t vocab, dim;
  float scale;
  int accumulate;
  int wide_grad;  // rows on 32-byte boundaries
  Tokens tokens;         // SMALL: sorted by every CTA; the first one writes `keys` out for the join
  uint32_t* keys_out;
  float* partial;        // 2 rows a block: a run from before it, a run that goes on behind it
  uint32_t partial_pitch;  // dim rounded up to 8
  DropArgs drop;
};

template <typename T>
__device__ __forceinline__ T* row_at(T* base, uint32_t row, uint32_t pitch) {
  return base + static_cast<uint64_t>(row) * pitch;
}

// The fates of the eight elements e[u] .. e[u] + 7 for two rows.  VEC: e is a
// multiple of eight, they are one group; otherwise they may reach into the next.
template <bool VEC>
struct Fates {
  uint4 w[2];

  __device__ __forceinline__ void set(const uint64_t (&e)[2], const DropArgs& a, const DropKey& k) {
    uint64_t g[2] = {e[0] >> 3, e[1] >> 3};
    drop_words<2>(g, a, k, w);
    if constexpr (!VEC) {  // w[u].x: one bit per element
      uint32_t bits[2] = {0u, 0u};
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) bits[u] |= kept(w[u], j, a.cmp) ? 1u << j : 0u;
      ++g[0];
      ++g[1];
      drop_words<2>(g, a, k, w);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) bits[u] |= kept(w[u], j, a.cmp) ? 256u << j : 0u;
        w[u].x = bits[u] >> (e[u] & 7);
      }
    }
  }

  // acc[j] += v[j] where kept (the scale is applied to the sum)
  __device__ __forceinline__ void add(int u, const DropArgs& a, const float (&v)[8], float (&acc)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (VEC ? kept(w[u], j, a.cmp) : (w[u].x >> j) & 1u) acc[j] = __fadd_rn(acc[j], v[j]);
  }
};

template <typename TG>
__device__ __forceinline__ void put_one(const SumArgs& s, uint32_t key, uint32_t c, float sum) {
  TG* at = row_at(static_cast<TG*>(s.grad), key, s.grad_pitch) + c;
  float v = __fmul_rn(sum, s.scale);
  if (s.accumulate) v = __fadd_rn(to_f32(*at), v);
  *at = from_f32<TG>(v);
}

__device__ __forceinline__ void store8_shared(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// Columns c .. c + 7 of a finished row.  Where rows are no whole 16-byte pieces
// and a warp has one tile (warp != NULL, 256 floats of shared memory), its
// lanes exchange columns, so that each store covers 32 neighbouring ones.
template <typename TG, bool VEC>
__device__ __forceinline__ void put_row8(const SumArgs& s, uint32_t key, uint32_t c, const float (&sum)[8],
                                         float* warp) {
  if constexpr (VEC) {
    TG* at = row_at(static_cast<TG*>(s.grad), key, s.grad_pitch) + c;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(sum[j], s.scale);
    if (s.accumulate) {
      float g[8];
      unpack8<TG>(load8(at, s.wide_grad), g);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __fadd_rn(g[j], v[j]);
    }
    store8(at, pack8<TG>(v), s.wide_grad);
  } else if (warp) {
    const int lane = threadIdx.x & 31;
    store8_shared(warp + 8 * lane, sum);
    __syncwarp();
    const int first = static_cast<int>(c) - 7 * lane, left = static_cast<int>(s.dim) - first;
    TG* at = row_at(static_cast<TG*>(s.grad), key, s.grad_pitch) + first;
    float g[8];  // all loads before the first store
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = s.accumulate && 32 * j < left ? to_f32(at[32 * j]) : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = __fmul_rn(warp[32 * j + lane], s.scale);
      if (32 * j < left) at[32 * j] = from_f32<TG>(s.accumulate ? __fadd_rn(g[j], v) : v);
    }
    __syncwarp();
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < s.dim) put_one<TG>(s, key, c + j, sum[j]);
  }
}

constexpr int kSumThreads = 256;
constexpr int kSumLanes = 64;  // threads of a tile's slab of 512 columns, at most
// Rows that a thread has on the way, in shared memory of its own: kStages groups
// of `rows` rows, `pieces` 16-byte pieces each (whole ones, or the blocks around
// eight elements that lie anywhere).
constexpr int kStages = 2;
template <typename TD, bool VEC>
struct Ring {
  static constexpr int pieces = VEC ? sizeof(TD) / 2 : Blocks<TD>::N;
  static constexpr int rows = VEC && sizeof(TD) == 2 ? 4 : 2;
  static constexpr int bytes = kStages * rows * pieces * 16 * kSumThreads;
};
constexpr int kPartBytes = 2 * 8 * 4 * kSumThreads;
static_assert(kPartBytes >= kZeroBytes, "the zeros that rows are filled from lie there");

// The first position at which the sorted keys reach `row` (lanes 0..15 of the
// warp) or `end` (lanes 16..31): each step, the half-warp's lanes look at the 16
// ends of equal parts of what is left.
__device__ __forceinline__ uint32_t half_warp_search(const SumArgs& s, uint32_t row) {
  const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31;
  uint32_t a = 0, b = s.n;  // keys before a are below row, keys from b on are not
  while (__any_sync(0xFFFFFFFFu, a < b)) {
    const uint32_t step = (b - a + 15) / 16, at = a + ((lane & 15) + 1) * step - 1;
    const bool below = a < b && at < b && s.keys[at] < row;  // one half may be done before the other
    const int parts = __popc((__ballot_sync(0xFFFFFFFFu, below) >> (lane & 16)) & 0xFFFFu);
    if (a < b) {
      const uint32_t next = a + parts * step;
      b = min(b, next + step - 1);
      a = min(next, b);
    }
  }
  return a;
}

// Zeros for those rows of CTA `cta`, f.per_warp a warp, that the sorted keys lack.
__device__ __forceinline__ void fill_searched(const SumArgs& s, const Fill& f, uint32_t cta, void* zeros) {
  clear_zeros(zeros);
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, lane = tid & 31;
  const uint32_t first = (cta * (kSumThreads / 32) + (tid >> 5)) * f.per_warp;  // rows < 2^30 + a CTA's
  const uint32_t found = half_warp_search(s, lane < 16 ? first : first + f.per_warp);
  uint32_t a = __shfl_sync(0xFFFFFFFFu, found, 0);
  const uint32_t end = __shfl_sync(0xFFFFFFFFu, found, 16);
  const uint32_t row = first + lane;
  bool empty = false;
  if (lane < f.per_warp && row < f.rows) {
    uint32_t b = end;  // the first key >= row lies in [a, end]
    while (a < b) {
      const uint32_t m = (a + b) / 2;
      if (s.keys[m] < row)
        a = m + 1;
      else
        b = m;
    }
    empty = a == end || s.keys[a] != row;
  }
  __syncthreads();  // the zeros
  fill_rows(f, first, __ballot_sync(0xFFFFFFFFu, empty), zeros);
  fill_done();
}

// N keys from position i on (kNoKey behind hi); i is a multiple of N and the
// arrays are allocated in whole tiles.
template <int N>
__device__ __forceinline__ void load_ids(const uint32_t* ids, uint32_t i, uint32_t (&v)[N]) {
  if constexpr (N == 4) {
    const uint4 q = *reinterpret_cast<const uint4*>(ids + i);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  } else {
    const uint2 q = *reinterpret_cast<const uint2*>(ids + i);
    v[0] = q.x, v[1] = q.y;
  }
}

// The rows of a tile, columns c .. c + 7, group by group.
template <typename TD, typename TG, bool VEC>
struct Rows {
  static constexpr int N = Ring<TD, VEC>::rows, P = Ring<TD, VEC>::pieces;
  const SumArgs& s;
  const uint32_t *keys, *ids;  // sorted, with their positions
  const TD* dy;                // column c of row 0
  uint32_t c, hi;
  uint32_t ring;               // this thread's slot of the first piece

  __device__ __forceinline__ uint32_t slot(int stage, int u, int p) const {
    return ring + ((stage * N + u) * P + p) * (16 * kSumThreads);
  }

  // Whole pieces, or blocks that lie within dy.
  __device__ __forceinline__ bool by_pieces(const TD* from) const {
    if (VEC) return true;
    const TD* whole = static_cast<const TD*>(s.dy);
    return Blocks<TD>::within(from, whole, row_at(whole, s.n - 1, s.dy_pitch) + s.dim);
  }

  // Rows of the group at i go on their way into stage `stage`.  Rows of an
  // accumulated grad that the ends of its runs will read are brought into L2.
  __device__ __forceinline__ void request(uint32_t i, int stage) const {
    if (i < hi && c < s.dim) {
      uint32_t key[N], pos[N];
      load_ids<N>(keys, i, key);
      load_ids<N>(ids, i, pos);
#pragma unroll
      for (int u = 0; u < N; ++u) {
        if (i + u < hi && key[u] < s.vocab) {
          const TD* from = row_at(dy, pos[u], s.dy_pitch);
          if (by_pieces(from)) {
            const char* piece = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(from) & ~uintptr_t{15});
#pragma unroll
            for (int p = 0; p < P; ++p)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot(stage, u, p)), "l"(piece + 16 * p)
                           : "memory");
          }
          if (s.accumulate && (u == 0 || key[u] != key[u - 1]))
            asm volatile("prefetch.global.L2 [%0];" ::"l"(row_at(static_cast<const TG*>(s.grad), key[u], s.grad_pitch) + c));
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  __device__ __forceinline__ void arrived() const {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
  }

  // Row u of the group; what lies behind the last column is undefined.
  __device__ __forceinline__ Raw8<TD> get(int stage, int u, uint32_t pos) const {
    if constexpr (VEC) {
      Raw8<TD> r;
#pragma unroll
      for (int p = 0; p < P; ++p) shared16(slot(stage, u, p), r.q[p]);
      return r;
    } else {
      const TD* from = row_at(dy, pos, s.dy_pitch);
      if (!by_pieces(from)) return load8_single(from, static_cast<int>(min(s.dim - c, 8u)));
      Blocks<TD> b;
#pragma unroll
      for (int p = 0; p < P; ++p) shared16(slot(stage, u, p), b.q[p]);
      return b.at(from);
    }
  }

  __device__ __forceinline__ static void shared16(uint32_t at, uint4& q) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                 : "r"(at)
                 : "memory");
  }
};

// What a tile leaves for the sums across tiles: the row its first run adds to
// (it began before the tile), whether that run goes on behind the tile too, and
// the row of a last run that begins in the tile and goes on behind it.
struct Ends {
  uint32_t head, tail;  // kNoKey: none
  int through;
};
constexpr int kEndsBytes = static_cast<int>(sizeof(Ends)) * kSumThreads;
constexpr int kExchangeBytes = 8 * 4 * kSumThreads;  // put_row8()
// Shared memory: part | ends | exchange (rows of any width) | sorted tokens (SMALL) | ring
template <typename TD, bool VEC, bool SMALL>
struct SumSmem {
  static constexpr int exchange = kPartBytes + kEndsBytes;
  static constexpr int tokens = exchange + (VEC ? 0 : kExchangeBytes);
  static constexpr int ring = tokens + (SMALL ? 8 * 2 * kSumThreads : 0);
  static constexpr int bytes = ring + Ring<TD, VEC>::bytes;
};
constexpr int kSumCtas = 3;  // per SM; 4 (64 registers) measured the same within 2%

// ---- up to kSmallTokens tokens: one CTA sorts them alone -----------------------
constexpr int kSmallTokens = 2 * kSumThreads;
constexpr int kSmallBits = 9;  // of a position
constexpr int64_t kSmallVocab = int64_t{1} << (32 - kSmallBits);

// Bitonic sort of kSumThreads * E words key << kSmallBits | position, E (one or
// two) consecutive ones a thread: distances within a thread in registers, within a warp by
// shuffles, the others through `words` in shared memory.  All words differ
// (padding aside), so the order is by key, then position.
template <int E>
__device__ __noinline__ void small_sort(uint32_t (&x)[2], uint32_t* words, int tid) {
#pragma unroll 1
  for (int k = 2; k <= kSumThreads * E; k <<= 1) {
#pragma unroll 1
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j < E) {  // E = 2
        const uint32_t lo = min(x[0], x[1]), hi = max(x[0], x[1]);
        const bool up = (tid * E & k) == 0;
        x[0] = up ? lo : hi;
        x[1] = up ? hi : lo;
        continue;
      }
      if (j >= 32 * E) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) words[tid * E + e] = x[e];
        __syncthreads();
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = tid * E + e;
        const uint32_t y = j >= 32 * E ? words[i ^ j] : __shfl_xor_sync(0xFFFFFFFFu, x[e], j / E);
        x[e] = ((i & j) == 0) == ((i & k) == 0) ? min(x[e], y) : max(x[e], y);
      }
    }
  }
}

// keys[i], pos[i] of the n tokens in sorted order, in shared memory (whole groups
// of four: read, not used, behind n).
__device__ __forceinline__ void small_sort_tokens(const Tokens& tk, int n, uint32_t* keys, uint32_t* pos) {
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  const int e = n <= kSumThreads ? 1 : 2;  // items a thread
  uint32_t x[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int t = tid * e + j;
    x[j] = j < e && t < n ? token_key(tk, t) << kSmallBits | t : 0xFFFFFFFFu;
  }
  if (e == 1)
    small_sort<1>(x, keys, tid);
  else
    small_sort<2>(x, keys, tid);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (j < e) {
      keys[tid * e + j] = x[j] >> kSmallBits;
      pos[tid * e + j] = x[j] & ((1u << kSmallBits) - 1);
    }
  }
  __syncthreads();
}

// fill_searched() without sorted keys: the CTA looks at all tokens.
__device__ __forceinline__ void fill_marked(const Tokens& tk, int n, const Fill& f, uint32_t cta, void* zeros,
                                            uint32_t* named) {
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, warp = tid >> 5;
  const int64_t first = static_cast<int64_t>(cta) * (kSumThreads / 32) * f.per_warp;
  clear_zeros(zeros);
  if (tid < kSumThreads / 32) named[tid] = 0u;  // one word a warp, a bit per row
  __syncthreads();
  for (int t = tid; t < n; t += kSumThreads) {
    const uint32_t row = token_key(tk, t) - static_cast<uint32_t>(first);
    const uint32_t owner = row / f.per_warp;
    if (owner < kSumThreads / 32) atomicOr(&named[owner], 1u << (row % f.per_warp));
  }
  __syncthreads();
  const int64_t mine = first + static_cast<int64_t>(warp) * f.per_warp, left = f.rows - mine;
  uint32_t empty = ~named[warp];
  const int64_t rows = min(left, static_cast<int64_t>(f.per_warp));
  if (rows < 32) empty &= rows > 0 ? (1u << rows) - 1 : 0u;
  fill_rows(f, mine, empty, zeros);
  fill_done();
}

// A CTA sums blockDim.y tiles, one after the other, of a slab of 8 * blockDim.x
// columns; those behind sum_ctas zero rows (in the order of their addresses:
// spread evenly among the others they took 460 us instead of 420 in all).
template <typename TD, typename TG, bool DROP, bool VEC, bool SMALL>
__global__ void __launch_bounds__(kSumThreads, kSumCtas)
    sum_kernel(SumArgs s, uint32_t slabs, uint32_t sum_ctas, Fill f) {
  using Smem = SumSmem<TD, VEC, SMALL>;
  extern __shared__ __align__(128) unsigned char smem[];  // Smem::bytes
  float* part = reinterpret_cast<float*>(smem);            // [head, tail][tile][column]
  Ends* ends = reinterpret_cast<Ends*>(smem + kPartBytes);
  let_next_start();
  wait_for_previous();
  uint32_t* small = reinterpret_cast<uint32_t*>(smem + Smem::tokens);  // SMALL: 2 * kSmallTokens words
  if (blockIdx.x >= sum_ctas) {
    if (SMALL)
      fill_marked(s.tokens, static_cast<int>(s.n), f, blockIdx.x - sum_ctas, smem, small);
    else
      fill_searched(s, f, blockIdx.x - sum_ctas, smem);
    return;
  }
  const uint32_t* keys = SMALL ? small : s.keys;
  const uint32_t* ids = SMALL ? small + kSmallTokens : s.pos;
  if (SMALL) {
    small_sort_tokens(s.tokens, static_cast<int>(s.n), small, small + kSmallTokens);
    if (blockIdx.x == 0)
      for (uint32_t i = threadIdx.y * blockDim.x + threadIdx.x; i < s.n; i += kSumThreads) s.keys_out[i] = keys[i];
  }
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  const uint32_t block = blockIdx.x / slabs;
  const uint32_t c0 = 8 * (blockIdx.x % slabs) * blockDim.x;
  const uint32_t c = c0 + 8 * threadIdx.x;
  const uint32_t lo = block * s.block + threadIdx.y * s.tile;
  const uint32_t hi = min(lo + s.tile, s.n);
  Ends mine{kNoKey, kNoKey, 0};
  // (lanes behind the last column stay for the exchange of columns)
  float* warp = nullptr;
  if (!VEC && blockDim.x >= 32) warp = reinterpret_cast<float*>(smem + Smem::exchange) + 8 * (tid & ~31);
  if (lo < hi && (c < s.dim || warp)) {
    constexpr int N = Ring<TD, VEC>::rows;
    DropKey k{};
    if (DROP) k = drop_key(s.drop);
    const Rows<TD, TG, VEC> rows{s, keys, ids, static_cast<const TD*>(s.dy) + c, c, hi,
                                 static_cast<uint32_t>(__cvta_generic_to_shared(smem + Smem::ring)) + 16 * tid};
    const uint32_t before = lo > 0 ? keys[lo - 1] : kNoKey;
    const uint32_t behind = hi < s.n ? keys[hi] : kNoKey;
    float acc[8];
    uint32_t run = kNoKey;
    bool first = true;  // no run of the tile has ended yet
#pragma unroll
    for (int g = 0; g < kStages; ++g) rows.request(lo + g * N, g);
    int stage = 0;
    for (uint32_t i = lo; i < hi; i += N) {
      rows.arrived();
      uint32_t key[N], pos[N];
      load_ids<N>(keys, i, key);
      if (DROP || !VEC) load_ids<N>(ids, i, pos);
#pragma unroll
      for (int u = 0; u < N; u += 2) {
        Fates<VEC> fates;
        if (DROP)
          fates.set({static_cast<uint64_t>(pos[u]) * s.dim + c, static_cast<uint64_t>(pos[u + 1]) * s.dim + c}, s.drop, k);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t id = key[u + h];
          if (i + u + h >= hi || id >= s.vocab) continue;
          float v[8] = {};
          if (VEC || c < s.dim) unpack8<TD>(rows.get(stage, u + h, pos[u + h]), v);
          if (id != run) {
            if (run != kNoKey) {
              if (first && run == before) {
                store8_shared(part + 8 * tid, acc);
                mine.head = run;
              } else {
                put_row8<TG, VEC>(s, run, c, acc, warp);
              }
              first = false;
            }
            run = id;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
          }
          if (DROP) {
            fates.add(h, s.drop, v, acc);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = __fadd_rn(acc[j], v[j]);
          }
        }
      }
      rows.request(i + kStages * N, stage);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    if (run != kNoKey) {
      if (first && run == before) {
        store8_shared(part + 8 * tid, acc);
        mine.head = run;
        mine.through = run == behind;
      } else if (run == behind) {
        store8_shared(part + 8 * (kSumThreads + tid), acc);
        mine.tail = run;
      } else {
        put_row8<TG, VEC>(s, run, c, acc, warp);
      }
    }
  }
  if (threadIdx.x == 0) ends[threadIdx.y] = mine;
  __syncthreads();
  // Runs across tiles: one thread per column goes through the tiles in order.
  const int columns = 8 * blockDim.x;
  for (int col = threadIdx.y * blockDim.x + threadIdx.x; col < columns; col += kSumThreads) {
    if (c0 + col >= s.dim) break;
    float acc = 0.0f;
    bool from_before = false, open = false;
    for (int t = 0; t < blockDim.y; ++t) {
      const Ends e = ends[t];
      if (e.head != kNoKey) {
        const float x = part[t * columns + col];
        if (t == 0) {
          acc = x;
          from_before = open = true;
        } else {
          acc = __fadd_rn(acc, x);
        }
        if (!e.through) {
          if (from_before)
            row_at(s.partial, 2 * block, s.partial_pitch)[c0 + col] = acc;
          else
            put_one<TG>(s, e.head, c0 + col, acc);
          open = from_before = false;
        }
      }
      if (e.tail != kNoKey) {
        acc = part[8 * kSumThreads + t * columns + col];
        open = true;
      }
    }
    if (open) row_at(s.partial, 2 * block + (from_before ? 0 : 1), s.partial_pitch)[c0 + col] = acc;
  }
}

// ---- 3. runs that cross blocks ----------------------------------------------------
constexpr int kJoinLanes = 64;
constexpr int kJoinParts = 4;
constexpr int kJoinThreads = kJoinLanes * kJoinParts;

__device__ __forceinline__ void add4(float4& a, const float4& b) {
  a.x = __fadd_rn(a.x, b.x);
  a.y = __fadd_rn(a.y, b.y);
  a.z = __fadd_rn(a.z, b.z);
  a.w = __fadd_rn(a.w, b.w);
}

// Block blockIdx.x, if a run begins in it and goes on behind it; 4 columns per
// lane.  Part q adds the run's partial rows q, q + 4, ...; part 0 the four sums.
template <typename TG>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(SumArgs s) {
  __shared__ float4 sums[kJoinParts][kJoinLanes];
  let_next_start();
  wait_for_previous();
  const uint32_t block = blockIdx.x;
  const uint32_t lo = block * s.block, hi = lo + s.block;
  if (hi >= s.n) return;
  const uint32_t key = s.keys[hi - 1], behind = s.keys[hi];
  const uint32_t before = lo > 0 ? s.keys[lo - 1] : kNoKey;
  if (key >= s.vocab || behind != key || before == key) return;
  // the blocks behind this one whose first item has the key are consecutive
  const int tid = threadIdx.y * kJoinLanes + threadIdx.x;
  int more = 0;
  for (int found = kJoinThreads; found == kJoinThreads; more += found) {
    const uint64_t i = static_cast<uint64_t>(block + 1 + more + tid) * s.block;
    found = __syncthreads_count(i < s.n && s.keys[i] == key);
  }
  const uint32_t c = 4 * (blockIdx.y * kJoinLanes + threadIdx.x);
  const bool on = c < s.dim;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (on) {
    constexpr int kAhead = 8;  // loads under way
    for (int j0 = threadIdx.y; j0 <= more; j0 += kAhead * kJoinParts) {
      float4 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int j = j0 + u * kJoinParts;
        const uint32_t row = j == 0 ? 2 * block + 1 : 2 * (block + j);
        if (j <= more) v[u] = *reinterpret_cast<const float4*>(row_at(s.partial, row, s.partial_pitch) + c);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (j0 + u * kJoinParts <= more) add4(acc, v[u]);
    }
  }
  sums[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.y != 0 || !on) return;
#pragma unroll
  for (int q = 1; q < kJoinParts; ++q) add4(acc, sums[q][threadIdx.x]);
  const float f[4] = {acc.x, acc.y, acc.z, acc.w};
  TG* at = row_at(static_cast<TG*>(s.grad), key, s.grad_pitch) + c;
  const int left = static_cast<int>(s.dim - c);
  float g[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) g[j] = s.accumulate && j < left ? to_f32(at[j]) : 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float v = __fmul_rn(f[j], s.scale);
    if (j < left) at[j] = from_f32<TG>(s.accumulate ? __fadd_rn(g[j], v) : v);
  }
}

// ---- host -------------------------------------------------------------------------
// Threads of a slab, slabs of a row, tiles of a CTA.
struct Shape {
  int lanes;
  int64_t slabs;
  int tiles;
};

Shape shape(int64_t dim) {
  const int64_t need = (dim + 7) / 8;
  int lanes = 1;
  while (lanes < need && lanes < kSumLanes) lanes *= 2;
  return {lanes, (need + lanes - 1) / lanes, kSumThreads / lanes};
}

// K: enough threads for every SM, no more ends of tiles than that takes.  Chosen
// from two shapes, whatever the registers of the instantiation.
// Measured with 77,000 / 153,600 / 307,000 / 614,000 threads wanted: 32,768 rows
// of 2,048 with dropout 134 / 119 / 105 / 109 us, 32,768 rows of 1,536 of which
// half are one token 85 / 73 / 75 / 81 us.
constexpr int kMinTile = 8, kMaxTile = 256;
constexpr int64_t kThreadsWanted = 300000;

int tile_tokens(int64_t n, int64_t dim) {
  const Shape sh = shape(dim);
  int tile = kMinTile;
  while (tile < kMaxTile && tile * kThreadsWanted < n * sh.slabs * sh.lanes) tile *= 2;
  return tile;
}

struct Layout {
  int64_t sort_tiles;
  int passes, digit_bits, tile;
  int64_t block, partial_pitch;
  size_t keys[2], pos[2], hist, partial, bytes;
};

Layout layout(int64_t n, int64_t vocab, int64_t dim) {
  Layout l{};
  int bits = 1;
  while ((vocab >> bits) != 0) ++bits;  // keys 0 .. vocab
  l.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  l.digit_bits = (bits + l.passes - 1) / l.passes;
  l.sort_tiles = (n + kSortTile - 1) / kSortTile;
  l.tile = tile_tokens(n, dim);
  l.block = int64_t{l.tile} * shape(dim).tiles;
  l.partial_pitch = (dim + 7) / 8 * 8;
  size_t at = 0;
  auto take = [&at](int64_t bytes) {
    const size_t here = at;
    at += static_cast<size_t>(bytes + 255) / 256 * 256;
    return here;
  };
  const int64_t whole = (n + kMaxTile - 1) / kMaxTile * kMaxTile;
  // a device with clusters of eight CTAs sorts more than their share by the other kernels
  const bool cluster = n <= int64_t{8} * kMaxClusterItems * kClusterThreads;
  for (int i = 0; i < (cluster ? 1 : 2); ++i) {
    l.keys[i] = take(4 * whole);
    l.pos[i] = take(4 * whole);
  }
  if (!cluster) l.hist = take(l.sort_tiles * (int64_t{4} << l.digit_bits));
  l.partial = take(8 * ((n + l.block - 1) / l.block) * l.partial_pitch);
  l.bytes = at;
  return l;
}

template <int ITEMS>
cudaLaunchConfig_t cluster_config(int ctas, size_t smem, cudaStream_t st, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = ctas;
  attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// The kernel's limits on the current device: shared memory, and clusters of
// more than eight CTAs, which a device may not offer.
template <int ITEMS>
cudaError_t allow_cluster() {
  cudaError_t e = cudaFuncSetAttribute(sort_cluster_kernel<ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(cluster_smem<ITEMS>(kMaxBins)));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(sort_cluster_kernel<ITEMS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

template <int ITEMS>
cudaError_t sort_cluster(const Tokens& tk, int64_t n, int ctas, const Layout& l, uint32_t* keys,
                         uint32_t* pos, cudaStream_t st) {
  const cudaError_t e = allow_cluster<ITEMS>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = cluster_config<ITEMS>(ctas, cluster_smem<ITEMS>(1 << l.digit_bits), st, &attr);
  return cudaLaunchKernelEx(&cfg, sort_cluster_kernel<ITEMS>, tk, static_cast<uint32_t>(n), l.passes,
                            l.digit_bits, keys, pos);
}

// CTAs of the largest cluster on the current device (read once per device).
int max_cluster() {
  constexpr int kDevices = 256;
  static std::atomic<int> known[kDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) {
    cudaGetLastError();
    return 8;
  }
  int ctas = known[dev].load(std::memory_order_relaxed);
  if (ctas == 0) {
    ctas = 8;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg =
        cluster_config<kMaxClusterItems>(16, cluster_smem<kMaxClusterItems>(kMaxBins), nullptr, &attr);
    int clusters = 0;
    if (allow_cluster<kMaxClusterItems>() == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&clusters, sort_cluster_kernel<kMaxClusterItems>, &cfg) == cudaSuccess &&
        clusters > 0)
      ctas = 16;
    cudaGetLastError();
    known[dev].store(ctas, std::memory_order_relaxed);
  }
  return ctas;
}

template <typename Kernel, typename... Args>
cudaError_t launch_next(Kernel kernel, dim3 grid, dim3 block, int smem, cudaStream_t st,
                        const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int failed(cudaError_t e) {
  cudaGetLastError();
  set_cuda_error(e);
  return DFC_ERR_CUDA;
}

// Sorted keys and positions of the tokens: DFC_OK or an error.
int sort_tokens(const Tokens& tk, int64_t n, const Layout& l, char* scratch, const uint32_t** keys_out,
                const uint32_t** pos_out, cudaStream_t st) {
  uint32_t *keys[2], *pos[2];
  for (int i = 0; i < 2; ++i) {
    keys[i] = reinterpret_cast<uint32_t*>(scratch + l.keys[i]);
    pos[i] = reinterpret_cast<uint32_t*>(scratch + l.pos[i]);
  }
  *keys_out = keys[0];
  *pos_out = pos[0];
  const int64_t threads = (n + kClusterThreads - 1) / kClusterThreads;  // full CTAs at one item a thread
  const int most = max_cluster();
  if (threads <= int64_t{most} * kMaxClusterItems) {
    int ctas = 1, items = 1;
    while (ctas < threads && ctas < most) ctas *= 2;
    while (int64_t{ctas} * items < threads) items *= 2;
    const auto sort = items == 1   ? sort_cluster<1>
                      : items == 2 ? sort_cluster<2>
                      : items == 4 ? sort_cluster<4>
                                   : sort_cluster<kMaxClusterItems>;
    const cudaError_t e = sort(tk, n, ctas, l, keys[0], pos[0], st);
    return e == cudaSuccess ? DFC_OK : failed(e);
  }
  uint32_t* hist = reinterpret_cast<uint32_t*>(scratch + l.hist);
  const unsigned tiles = static_cast<unsigned>(l.sort_tiles);
  const int bins = 1 << l.digit_bits;
  int from = 0;
  for (int p = 0; p < l.passes; ++p) {
    const uint32_t* k_in = p ? keys[from] : nullptr;
    const int to = p ? 1 - from : 0;
    sort_count_kernel<<<tiles, kSortThreads, 0, st>>>(tk, k_in, n, p * l.digit_bits, bins, hist);
    sort_scan_kernel<<<1, 1024, 0, st>>>(hist, l.sort_tiles * bins);
    sort_scatter_kernel<<<tiles, kSortThreads, 0, st>>>(tk, k_in, pos[from], n, p * l.digit_bits, bins,
                                                        hist, keys[to], pos[to]);
    from = to;
  }
  *keys_out = keys[from];
  *pos_out = pos[from];
  return launch_status();
}

bool sizes_ok(int64_t n, int64_t vocab, int64_t dim) {
  return n >= 0 && n <= DFC_MAX_TOKENS && vocab >= 0 && vocab <= DFC_MAX_VOCAB && dim >= 0 &&
         dim <= DFC_MAX_DIM && n * dim <= (int64_t{1} << 39);
}

template <typename TD, typename TG, bool DROP, bool VEC, bool SMALL>
int launch_sums(const SumArgs& s, const Fill& f, cudaStream_t st) {
  const Shape sh = shape(s.dim);
  const int64_t blocks = (int64_t{s.n} + s.block - 1) / s.block;
  const int64_t sum_ctas = blocks * sh.slabs;
  const int64_t cta_rows = int64_t{f.per_warp} * kSumThreads / 32;
  const int64_t fill_ctas = f.rows > 0 ? (f.rows + cta_rows - 1) / cta_rows : 0;
  if (sum_ctas + fill_ctas == 0) return DFC_OK;
  const auto kernel = sum_kernel<TD, TG, DROP, VEC, SMALL>;
  constexpr int smem = SumSmem<TD, VEC, SMALL>::bytes;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return failed(e);
  e = launch_next(kernel, dim3(static_cast<unsigned>(sum_ctas + fill_ctas)), dim3(sh.lanes, sh.tiles), smem, st,
                  s, static_cast<uint32_t>(sh.slabs), static_cast<uint32_t>(sum_ctas), f);
  if (e == cudaSuccess && blocks > 1)
    e = launch_next(join_kernel<TG>,
                    dim3(static_cast<unsigned>(blocks - 1),
                         static_cast<unsigned>((s.dim + 4 * kJoinLanes - 1) / (4 * kJoinLanes))),
                    dim3(kJoinLanes, kJoinParts), 0, st, s);
  return e == cudaSuccess ? launch_status() : failed(e);
}

// Every CTA sorts the tokens itself, one launch less: 16.7 -> 13.8 us for 300
// tokens of 384 FP32 columns, 18.7 -> 14.8 for 400 of 4,096 bf16 ones.  Up to
// 1,024 tokens it cost more where rows are wide (24.6 instead of 20.7 us for 600
// of 4,096) and gained at most 2 us elsewhere.
bool small(int64_t n, int64_t vocab) { return n <= kSmallTokens && vocab < kSmallVocab; }

template <typename TD, typename TG, bool DROP, bool VEC>
int run_sums(const SumArgs& s, const Fill& f, cudaStream_t st) {
  return small(s.n, s.vocab) ? launch_sums<TD, TG, DROP, VEC, true>(s, f, st)
                             : launch_sums<TD, TG, DROP, VEC, false>(s, f, st);
}

template <typename TD, typename TG>
int by_path(const SumArgs& s, const Fill& f, bool drop, cudaStream_t st) {
  const bool vec = s.dim % 8 == 0 && aligned(s.dy, 16) && aligned(s.grad, 16) &&
                   s.dy_pitch % (16 / sizeof(TD)) == 0 &&
                   s.grad_pitch % (16 / sizeof(TG)) == 0;
  if (vec) return drop ? run_sums<TD, TG, true, true>(s, f, st) : run_sums<TD, TG, false, true>(s, f, st);
  return drop ? run_sums<TD, TG, true, false>(s, f, st) : run_sums<TD, TG, false, false>(s, f, st);
}

template <typename TD>
int by_grad(const SumArgs& s, const Fill& f, int32_t grad_dtype, bool drop, cudaStream_t st) {
  if (grad_dtype == DFC_DTYPE_F32) return by_path<TD, float>(s, f, drop, st);
  if (grad_dtype == DFC_DTYPE_BF16) return by_path<TD, bf16>(s, f, drop, st);
  return by_path<TD, f16>(s, f, drop, st);
}

}  // namespace
}  // namespace dfc

extern "C" size_t dfc_embedding_grad_scratch_bytes(int64_t n_tokens, int64_t vocab, int64_t dim) {
  using namespace dfc;
  if (!sizes_ok(n_tokens, vocab, dim)) return 0;
  return layout(n_tokens, vocab, dim).bytes;
}

extern "C" int dfc_embedding_grad(const void* tokens, int32_t token_bytes, int64_t n_tokens,
                                  const void* dy, int32_t dy_dtype, int64_t dy_pitch, void* grad,
                                  int32_t grad_dtype, int64_t grad_pitch, int64_t vocab,
                                  int64_t dim, float scale, int64_t padding_idx, int32_t accumulate,
                                  const DfcDropout* dropout, int32_t* error_flag, void* scratch,
                                  size_t scratch_bytes, void* stream) {
  using namespace dfc;
  if (!sizes_ok(n_tokens, vocab, dim) || dy_pitch < 0 || dy_pitch > DFC_MAX_PITCH || grad_pitch < dim ||
      grad_pitch > DFC_MAX_PITCH)
    return DFC_ERR_SIZE;
  if ((token_bytes != 4 && token_bytes != 8) || !known_dtype(dy_dtype) || !known_dtype(grad_dtype))
    return DFC_ERR_DTYPE;
  SumArgs s{};
  bool drop;
  const int rc = make_drop_args(dropout, &s.drop, &drop);
  if (rc != DFC_OK) return rc;
  if (dim == 0) return DFC_OK;
  if ((!grad && vocab > 0) || (n_tokens > 0 && (!tokens || !dy || !scratch))) return DFC_ERR_NULL;
  if (!aligned(tokens, token_bytes) || !aligned(dy, dtype_size(dy_dtype)) ||
      !aligned(grad, dtype_size(grad_dtype)) || !aligned(error_flag, 4) || !aligned(scratch, 16))
    return DFC_ERR_ALIGN;
  const Layout l = layout(n_tokens, vocab, dim);
  if (scratch_bytes < l.bytes) return DFC_ERR_SCRATCH;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* base = static_cast<char*>(scratch);
  Fill f{};
  if (!accumulate) {
    const int64_t size = static_cast<int64_t>(dtype_size(grad_dtype));
    const uintptr_t all = reinterpret_cast<uintptr_t>(grad) | static_cast<uintptr_t>(grad_pitch * size) |
                          static_cast<uintptr_t>(dim * size);
    // about 16 KB a warp
    const int per_warp = static_cast<int>(std::min<int64_t>(32, std::max<int64_t>(1, 16384 / (dim * size))));
    f = Fill{static_cast<char*>(grad), grad_pitch * size, dim * size, vocab, per_warp,
             all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2};
  }
  s.tokens = Tokens{tokens, token_bytes == 8, vocab, padding_idx, error_flag};
  s.keys_out = reinterpret_cast<uint32_t*>(base + l.keys[0]);
  s.keys = s.keys_out;
  if (n_tokens > 0 && !small(n_tokens, vocab)) {
    const int rc = sort_tokens(s.tokens, n_tokens, l, base, &s.keys, &s.pos, st);
    if (rc != DFC_OK) return rc;
  }
  s.n = static_cast<uint32_t>(n_tokens);
  s.tile = l.tile;
  s.block = static_cast<uint32_t>(l.block);
  s.dy = dy;
  s.dy_pitch = static_cast<uint32_t>(dy_pitch);
  s.grad = grad;
  s.grad_pitch = static_cast<uint32_t>(grad_pitch);
  s.vocab = static_cast<uint32_t>(vocab);
  s.dim = static_cast<uint32_t>(dim);
  // dropout's scale belongs to every term of the sum: applied once, to the sum
  s.scale = drop ? static_cast<float>(static_cast<double>(scale) * (dropout->p < 1.0 ? 1.0 / (1.0 - dropout->p) : 0.0))
                 : scale;
  s.accumulate = accumulate != 0;
  s.wide_grad = aligned(grad, 32) && grad_pitch % 8 == 0;
  s.partial = reinterpret_cast<float*>(base + l.partial);
  s.partial_pitch = static_cast<uint32_t>(l.partial_pitch);
  if (dy_dtype == DFC_DTYPE_F32) return by_grad<float>(s, f, grad_dtype, drop, st);
  if (dy_dtype == DFC_DTYPE_BF16) return by_grad<bf16>(s, f, grad_dtype, drop, st);
  return by_grad<f16>(s, f, grad_dtype, drop, st);
}
