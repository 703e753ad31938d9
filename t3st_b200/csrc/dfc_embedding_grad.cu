// Gradient of a token table by sorted tokens (no reference counterpart):
// grad[v] (+)= scale * sum over t with tokens[t] = v, t ascending, of drop(dy[t]).
//
//   1. a stable radix sort of (token, position) pairs; padding and
//      out-of-range tokens get the key `vocab` and sort behind the others;
//   2. sum_kernel: the sorted positions are cut into tiles of K; one thread
//      holds eight columns of a tile and adds its rows in order in FP32
//      registers, writing a row of grad at each end of a run.  A run that
//      crosses tile borders leaves FP32 partial rows in the scratch instead;
//   3. join_kernel adds such a run's partial rows in a fixed order;
//   4. fill_kernel zeroes the rows of an overwritten grad that no token names.
// No atomics on floats: the same inputs give the same bits.
#include <algorithm>

#include "dfc_philox.cuh"

namespace dfc {
namespace {

constexpr uint32_t kNoKey = 0xFFFFFFFFu;

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

__device__ __forceinline__ uint32_t warp_inclusive(uint32_t x) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, d);
    if ((threadIdx.x & 31) >= d) x += y;
  }
  return x;
}

// Exclusive scan of `total` counts in place, one CTA of 1024 threads.
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
    const uint32_t d = on ? (key[r] >> shift) & (bins - 1) : kNoKey;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, d);
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

// ---- 2. sums of runs ------------------------------------------------------------
struct SumArgs {
  const uint32_t* keys;  // sorted
  const uint32_t* pos;
  int64_t n;
  int tile;              // K
  const void* dy;
  int64_t dy_pitch;
  void* grad;
  int64_t grad_pitch;
  int64_t vocab, dim;
  float scale;
  int accumulate;
  float* partial;        // 2 rows a tile: a run from before it, a run that goes on behind it
  int64_t partial_pitch; // dim rounded up to 8
  DropArgs drop;
};

// Columns c .. c + 7 (those below dim) of a row in FP32.
template <typename T, bool VEC>
__device__ __forceinline__ void row8(const T* row, int64_t c, int64_t dim, float (&v)[8]) {
  if constexpr (VEC) {
    unpack8<T>(load8(row + c), v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < dim ? to_f32(row[c + j]) : 0.0f;
  }
}

// v[j] = element e + j kept ? v[j] : 0 (the scale is applied to the sum).
template <bool VEC>
__device__ __forceinline__ void mask8(float (&v)[8], int64_t e, const DropArgs& a, const DropKey& k) {
  const uint4 w = drop_words(e >> 3, a, k);
  if (VEC || (e & 7) == 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = kept(w, j, a.cmp) ? v[j] : 0.0f;
  } else {
    const uint4 x = drop_words((e >> 3) + 1, a, k);
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      bits |= (kept(w, j, a.cmp) ? 1u << j : 0u) | (kept(x, j, a.cmp) ? 256u << j : 0u);
    bits >>= e & 7;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (bits >> j) & 1u ? v[j] : 0.0f;
  }
}

template <typename TG, bool VEC>
__device__ __forceinline__ void put_row8(const SumArgs& s, uint32_t key, int64_t c, float (&v)[8]) {
  TG* row = static_cast<TG*>(s.grad) + key * s.grad_pitch;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], s.scale);
  if (s.accumulate) {
    float g[8];
    row8<TG, VEC>(row, c, s.dim, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fadd_rn(g[j], v[j]);
  }
  if constexpr (VEC) {
    store8(row + c, pack8<TG>(v));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < s.dim) row[c + j] = from_f32<TG>(v[j]);
  }
}

constexpr int kSumThreads = 128;
constexpr int kBatch = 4;

template <typename TD, typename TG, bool DROP, bool VEC>
__global__ void __launch_bounds__(kSumThreads) sum_kernel(SumArgs s) {
  const int64_t c = 8 * (static_cast<int64_t>(blockIdx.y) * blockDim.x + threadIdx.x);
  const int64_t tile = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t lo = tile * s.tile;
  if (c >= s.dim || lo >= s.n) return;
  const int64_t hi = min(lo + s.tile, s.n);
  DropKey k{};
  if (DROP) k = drop_key(s.drop);
  const TD* dy = static_cast<const TD*>(s.dy);
  const uint32_t before = lo > 0 ? s.keys[lo - 1] : kNoKey;
  const uint32_t behind = hi < s.n ? s.keys[hi] : kNoKey;
  float acc[8];
  uint32_t run = kNoKey;
  bool first = true;  // no row of the tile has ended a run yet
  for (int64_t i = lo; i < hi; i += kBatch) {
    uint32_t key[kBatch];
    float v[kBatch][8];
    int64_t p[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const bool on = i + u < hi;
      key[u] = on ? s.keys[i + u] : kNoKey;
      p[u] = on ? s.pos[i + u] : 0;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (key[u] < s.vocab) row8<TD, VEC>(dy + p[u] * s.dy_pitch, c, s.dim, v[u]);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (key[u] >= s.vocab) continue;
      if (DROP) mask8<VEC>(v[u], p[u] * s.dim + c, s.drop, k);
      if (key[u] == run) {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = __fadd_rn(acc[j], v[u][j]);
      } else {
        if (run != kNoKey) {
          if (first && run == before)
            store8(s.partial + 2 * tile * s.partial_pitch + c, pack8<float>(acc));
          else
            put_row8<TG, VEC>(s, run, c, acc);
          first = false;
        }
        run = key[u];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = v[u][j];
      }
    }
  }
  if (run == kNoKey) return;
  if (first && run == before)
    store8(s.partial + 2 * tile * s.partial_pitch + c, pack8<float>(acc));
  else if (run == behind)
    store8(s.partial + (2 * tile + 1) * s.partial_pitch + c, pack8<float>(acc));
  else
    put_row8<TG, VEC>(s, run, c, acc);
}

// ---- 3. runs that cross tile borders --------------------------------------------
constexpr int kJoinWarps = 8;

// Tile blockIdx.x, if a run begins in it and goes on behind it; columns 4 per
// lane.  Warp w adds partial rows w, w + 8, ... of the run, warp 0 the eight sums.
template <typename TG>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(SumArgs s) {
  __shared__ float4 sums[kJoinWarps][32];
  const int64_t tile = blockIdx.x;
  const int64_t lo = tile * s.tile, hi = lo + s.tile;
  if (hi >= s.n) return;
  const uint32_t key = s.keys[hi - 1];
  if (key >= s.vocab || s.keys[hi] != key) return;
  if (lo > 0 && s.keys[lo - 1] == key) return;  // it began earlier
  // the last tile whose first item still has the key
  int64_t last = tile + 1, end = (s.n - 1) / s.tile;
  while (last < end) {
    const int64_t mid = (last + end + 1) / 2;
    if (s.keys[mid * s.tile] == key)
      last = mid;
    else
      end = mid - 1;
  }
  const int64_t c = 4 * (static_cast<int64_t>(blockIdx.y) * 32 + threadIdx.x);
  const bool on = c < s.dim;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (on) {
    for (int64_t j = threadIdx.y; j <= last - tile; j += kJoinWarps) {
      const int64_t row = j == 0 ? 2 * tile + 1 : 2 * (tile + j);
      const float4 v = *reinterpret_cast<const float4*>(s.partial + row * s.partial_pitch + c);
      acc.x = __fadd_rn(acc.x, v.x);
      acc.y = __fadd_rn(acc.y, v.y);
      acc.z = __fadd_rn(acc.z, v.z);
      acc.w = __fadd_rn(acc.w, v.w);
    }
  }
  sums[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.y != 0 || !on) return;
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) {
    const float4 v = sums[w][threadIdx.x];
    acc.x = __fadd_rn(acc.x, v.x);
    acc.y = __fadd_rn(acc.y, v.y);
    acc.z = __fadd_rn(acc.z, v.z);
    acc.w = __fadd_rn(acc.w, v.w);
  }
  const float f[4] = {acc.x, acc.y, acc.z, acc.w};
  TG* row = static_cast<TG*>(s.grad) + key * s.grad_pitch;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (c + j < s.dim) {
      float v = __fmul_rn(f[j], s.scale);
      if (s.accumulate) v = __fadd_rn(to_f32(row[c + j]), v);
      row[c + j] = from_f32<TG>(v);
    }
  }
}

// ---- 4. rows without a token -----------------------------------------------------
constexpr int kFillThreads = 256;
constexpr int kFillRows = 32;

template <typename TG, bool VEC>
__global__ void __launch_bounds__(kFillThreads) fill_kernel(SumArgs s, int rows) {
  __shared__ int empty[kFillRows];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * rows;
  if (threadIdx.x < rows) {
    const int64_t v = first + threadIdx.x;
    int64_t a = 0, b = s.n;  // the first sorted key >= v
    while (a < b) {
      const int64_t m = (a + b) / 2;
      if (s.keys[m] < v)
        a = m + 1;
      else
        b = m;
    }
    empty[threadIdx.x] = v < s.vocab && !(a < s.n && s.keys[a] == v);
  }
  __syncthreads();
  for (int r = 0; r < rows; ++r) {
    if (!empty[r]) continue;
    TG* row = static_cast<TG*>(s.grad) + (first + r) * s.grad_pitch;
    if constexpr (VEC) {
      const float z[8] = {};
      for (int64_t c = 8ll * threadIdx.x; c < s.dim; c += 8 * kFillThreads) store8(row + c, pack8<TG>(z));
    } else {
      for (int64_t c = threadIdx.x; c < s.dim; c += kFillThreads) row[c] = from_f32<TG>(0.0f);
    }
  }
}

// ---- host -------------------------------------------------------------------------
int tile_tokens(int64_t, int64_t) { return 32; }

struct Layout {
  int64_t sort_tiles;
  int passes, digit_bits, tile;
  int64_t tiles, partial_pitch;
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
  l.tiles = (n + l.tile - 1) / l.tile;
  l.partial_pitch = (dim + 7) / 8 * 8;
  size_t at = 0;
  auto take = [&at](int64_t bytes) {
    const size_t here = at;
    at += static_cast<size_t>(bytes + 255) / 256 * 256;
    return here;
  };
  for (int i = 0; i < 2; ++i) {
    l.keys[i] = take(4 * n);
    l.pos[i] = take(4 * n);
  }
  l.hist = take(l.sort_tiles * (int64_t{4} << l.digit_bits));
  l.partial = take(8 * l.tiles * l.partial_pitch);
  l.bytes = at;
  return l;
}

bool sizes_ok(int64_t n, int64_t vocab, int64_t dim) {
  return n >= 0 && n <= DFC_MAX_TOKENS && vocab >= 0 && vocab <= DFC_MAX_VOCAB && dim >= 0 &&
         dim <= DFC_MAX_DIM && n * dim <= (int64_t{1} << 39);
}

template <typename TD, typename TG, bool DROP, bool VEC>
int run_sums(const SumArgs& s, cudaStream_t st) {
  const int64_t tiles = (s.n + s.tile - 1) / s.tile;
  const int64_t lanes_needed = (s.dim + 7) / 8;
  int lanes = 1;
  while (lanes < lanes_needed && lanes < kSumThreads) lanes *= 2;
  const int subs = kSumThreads / lanes;
  if (tiles > 0) {
    const dim3 grid(static_cast<unsigned>((tiles + subs - 1) / subs),
                    static_cast<unsigned>((lanes_needed + lanes - 1) / lanes));
    sum_kernel<TD, TG, DROP, VEC><<<grid, dim3(lanes, subs), 0, st>>>(s);
    if (tiles > 1) {
      const dim3 jgrid(static_cast<unsigned>(tiles - 1), static_cast<unsigned>((s.dim + 127) / 128));
      join_kernel<TG><<<jgrid, dim3(32, kJoinWarps), 0, st>>>(s);
    }
  }
  if (!s.accumulate && s.vocab > 0) {
    const int64_t row_bytes = s.dim * static_cast<int64_t>(sizeof(TG));
    const int rows = static_cast<int>(std::min<int64_t>(kFillRows, std::max<int64_t>(1, 65536 / row_bytes)));
    fill_kernel<TG, VEC><<<static_cast<unsigned>((s.vocab + rows - 1) / rows), kFillThreads, 0, st>>>(s, rows);
  }
  return launch_status();
}

template <typename TD, typename TG>
int by_path(const SumArgs& s, bool drop, cudaStream_t st) {
  const bool vec = s.dim % 8 == 0 && aligned(s.dy, 16) && aligned(s.grad, 16) &&
                   s.dy_pitch * static_cast<int64_t>(sizeof(TD)) % 16 == 0 &&
                   s.grad_pitch * static_cast<int64_t>(sizeof(TG)) % 16 == 0;
  if (vec) return drop ? run_sums<TD, TG, true, true>(s, st) : run_sums<TD, TG, false, true>(s, st);
  return drop ? run_sums<TD, TG, true, false>(s, st) : run_sums<TD, TG, false, false>(s, st);
}

template <typename TD>
int by_grad(const SumArgs& s, int32_t grad_dtype, bool drop, cudaStream_t st) {
  if (grad_dtype == DFC_DTYPE_F32) return by_path<TD, float>(s, drop, st);
  if (grad_dtype == DFC_DTYPE_BF16) return by_path<TD, bf16>(s, drop, st);
  return by_path<TD, f16>(s, drop, st);
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
  if (!sizes_ok(n_tokens, vocab, dim) || dy_pitch < 0 || grad_pitch < dim) return DFC_ERR_SIZE;
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
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(base + l.keys[0]), reinterpret_cast<uint32_t*>(base + l.keys[1])};
  uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(base + l.pos[0]), reinterpret_cast<uint32_t*>(base + l.pos[1])};
  uint32_t* hist = reinterpret_cast<uint32_t*>(base + l.hist);
  const Tokens tk{tokens, token_bytes == 8, vocab, padding_idx, error_flag};
  int from = 0;
  if (n_tokens > 0) {
    const unsigned tiles = static_cast<unsigned>(l.sort_tiles);
    const int bins = 1 << l.digit_bits;
    for (int p = 0; p < l.passes; ++p) {
      const uint32_t* k_in = p ? keys[from] : nullptr;
      const int to = p ? 1 - from : 0;
      sort_count_kernel<<<tiles, kSortThreads, 0, st>>>(tk, k_in, n_tokens, p * l.digit_bits, bins, hist);
      sort_scan_kernel<<<1, 1024, 0, st>>>(hist, l.sort_tiles * bins);
      sort_scatter_kernel<<<tiles, kSortThreads, 0, st>>>(tk, k_in, pos[from], n_tokens,
                                                          p * l.digit_bits, bins, hist, keys[to], pos[to]);
      from = to;
    }
  }
  s.keys = keys[from];
  s.pos = pos[from];
  s.n = n_tokens;
  s.tile = l.tile;
  s.dy = dy;
  s.dy_pitch = dy_pitch;
  s.grad = grad;
  s.grad_pitch = grad_pitch;
  s.vocab = vocab;
  s.dim = dim;
  // dropout's scale belongs to every term of the sum: applied once, to the sum
  s.scale = drop ? static_cast<float>(static_cast<double>(scale) * (dropout->p < 1.0 ? 1.0 / (1.0 - dropout->p) : 0.0))
                 : scale;
  s.accumulate = accumulate != 0;
  s.partial = reinterpret_cast<float*>(base + l.partial);
  s.partial_pitch = l.partial_pitch;
  if (dy_dtype == DFC_DTYPE_F32) return by_grad<float>(s, grad_dtype, drop, st);
  if (dy_dtype == DFC_DTYPE_BF16) return by_grad<bf16>(s, grad_dtype, drop, st);
  return by_grad<f16>(s, grad_dtype, drop, st);
}
