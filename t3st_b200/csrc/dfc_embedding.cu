// Rows of a token table, scaled, with dropout in the same pass (no reference
// counterpart): out[t] = drop(scale * table[tokens[t]]), FP32 arithmetic, one
// rounding to the output type.  A token outside [0, vocab) reads nothing: its
// row becomes NaN and *error_flag is set.
//
// One thread per eight output elements (one dropout group: out is contiguous,
// so group g is elements 8g..8g+7 of it).  When a row is a whole number of
// 16-byte pieces the table is read in such pieces; otherwise from the 16-byte
// blocks around the elements, shifted into place, and element by element where
// a group spans rows.
//
// Bounds (B200, 16,384 tokens of 4,096 columns, FP32 table of 131,072 rows to
// bf16, frequencies falling as one over the rank; 39 us at the measured copy
// bandwidth, each named row counted once): without dropout 49 us; with it 72 us
// (69 without the launch), held by the issue of instructions, not by HBM: 27 per
// element, 3.0 a cycle and SM.  Of the 219 per group of eight, dropout_vec_kernel
// needs 166 for the same masks; three integer divisions a thread (token and
// column of each group) are part of the rest.
#include "dfc_philox.cuh"

namespace dfc {
namespace {

constexpr int kThreads = 256;
// Groups per thread, with registers for 6 CTAs per SM.  The case above with
// dropout: 73.7 us (launch included; 1 group 88.0, 4 groups 77.8 at 4 CTAs).
constexpr int kGroups = 2;

__device__ __forceinline__ int64_t token_at(const void* tokens, int wide, int64_t t) {
  return wide ? static_cast<const int64_t*>(tokens)[t]
              : static_cast<int64_t>(static_cast<const int32_t*>(tokens)[t]);
}

template <typename TT, typename TO, bool DROP>
__global__ void __launch_bounds__(kThreads, 6)
    embed_vec_kernel(const void* tokens, int wide, const TT* table, uint32_t pitch, int64_t vocab,
                     uint32_t row_groups, int64_t groups, float scale, TO* out, int wide_table,
                     int wide_out, int32_t* error_flag, DropArgs a) {
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (kThreads * kGroups);
  const int64_t t0 = base / row_groups;
  const uint32_t c0 = static_cast<uint32_t>(base - t0 * row_groups);
  Raw8<TT> X[kGroups];
  bool bad[kGroups];
#pragma unroll
  for (int u = 0; u < kGroups; ++u) {
    const uint32_t local = u * kThreads + threadIdx.x;
    if (base + local < groups) {
      const uint32_t q = c0 + local;
      const uint32_t dt = q / row_groups;
      const int64_t v = token_at(tokens, wide, t0 + dt);
      bad[u] = static_cast<uint64_t>(v) >= static_cast<uint64_t>(vocab);
      if (!bad[u]) X[u] = load8(table + static_cast<uint64_t>(static_cast<uint32_t>(v)) * pitch + 8ll * (q - dt * row_groups), wide_table);
    }
  }
  uint4 w[kGroups];
  if (DROP) {
    uint64_t g[kGroups];
#pragma unroll
    for (int u = 0; u < kGroups; ++u) g[u] = base + u * kThreads + threadIdx.x;
    drop_words<kGroups>(g, a, drop_key(a), w);
  }
#pragma unroll
  for (int u = 0; u < kGroups; ++u) {
    const int64_t g = base + u * kThreads + threadIdx.x;
    if (g < groups) {
      float v[8];
      if (bad[u]) {
        if (error_flag) *error_flag = 1;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = u2f(0x7FC00000u);
      } else {
        unpack8<TT>(X[u], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], scale);
      }
      if (DROP) drop8(v, w[u], a);
      store8(out + 8 * g, pack8<TO>(v), wide_out);
    }
  }
}

// i / d for i * d < 2^64, with per_d = ceil(2^64 / d) (0 for d = 1).
__device__ __forceinline__ int64_t row_of(int64_t i, uint64_t per_d) {
  return per_d ? static_cast<int64_t>(__umul64hi(static_cast<uint64_t>(i), per_d)) : i;
}

// Rows of any width, one group a thread (two a thread, their blocks asked for
// together: 20.5 instead of 16.4 us for 8,192 FP32 rows of 1,001 to bf16).
// 5,003 fp16 rows of 1,001 with dropout take 12.3 us where the bytes take 2.3:
// 45 instructions an element, a mask that is begun only when the row's blocks
// have arrived, and 2,446 CTAs on 1,184 places, so that a third wave is almost
// empty.
template <typename TT, typename TO, bool DROP>
__global__ void __launch_bounds__(kThreads)
    embed_any_kernel(const void* tokens, int wide, const TT* table, int64_t pitch, int64_t vocab,
                     int64_t dim, uint64_t per_dim, int64_t n, float scale, TO* out, int out_aligned,
                     int32_t* error_flag, DropArgs a) {
  const int64_t g = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (8 * g >= n) return;
  int64_t t = row_of(8 * g, per_dim);
  int64_t d = 8 * g - t * dim;
  int64_t v = token_at(tokens, wide, t);
  float x[8];
  const bool one_row = d + 8 <= dim && static_cast<uint64_t>(v) < static_cast<uint64_t>(vocab);
  if (one_row) {
    unpack8<TT>(load8_any(table + v * pitch + d, table, table + (vocab - 1) * pitch + dim), x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(x[j], scale);
  }
#pragma unroll
  for (int j = 0; !one_row && j < 8; ++j) {
    x[j] = 0.0f;
    if (8 * g + j < n) {
      if (d == dim) {
        d = 0;
        v = token_at(tokens, wide, ++t);
      }
      if (static_cast<uint64_t>(v) < static_cast<uint64_t>(vocab)) {
        x[j] = __fmul_rn(to_f32(table[v * pitch + d]), scale);
      } else {
        x[j] = u2f(0x7FC00000u);
        if (error_flag) *error_flag = 1;
      }
      ++d;
    }
  }
  if (DROP) {
    uint4 w[1];
    drop_words<1>({static_cast<uint64_t>(g)}, a, drop_key(a), w);
    drop8(x, w[0], a);
  }
  if (out_aligned && 8 * g + 8 <= n) {
    store8(out + 8 * g, pack8<TO>(x), 0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (8 * g + j < n) out[8 * g + j] = from_f32<TO>(x[j]);
  }
}

struct EmbedCall {
  const void* tokens;
  int wide;
  int64_t n_tokens;
  const void* table;
  int64_t pitch, vocab, dim;
  float scale;
  void* out;
  int32_t* error_flag;
  DropArgs drop;
  cudaStream_t st;
};

template <typename TT, typename TO, bool DROP>
int launch(const EmbedCall& c) {
  const TT* table = static_cast<const TT*>(c.table);
  TO* out = static_cast<TO*>(c.out);
  const int64_t n = c.n_tokens * c.dim;
  const bool vec = c.dim % 8 == 0 && aligned(table, 16) && aligned(out, 16) &&
                   c.pitch * static_cast<int64_t>(sizeof(TT)) % 16 == 0;
  if (vec) {
    const int64_t groups = n / 8, tile = kThreads * kGroups;
    embed_vec_kernel<TT, TO, DROP><<<static_cast<unsigned>((groups + tile - 1) / tile), kThreads, 0, c.st>>>(
        c.tokens, c.wide, table, static_cast<uint32_t>(c.pitch), c.vocab, static_cast<uint32_t>(c.dim / 8), groups, c.scale,
        out, aligned(table, 32) && c.pitch % 8 == 0, aligned(out, 32), c.error_flag, c.drop);
  } else {
    const int64_t groups = (n + 7) / 8;
    embed_any_kernel<TT, TO, DROP>
        <<<static_cast<unsigned>((groups + kThreads - 1) / kThreads), kThreads, 0, c.st>>>(
            c.tokens, c.wide, table, c.pitch, c.vocab, c.dim, c.dim > 1 ? ~0ull / c.dim + 1 : 0ull, n, c.scale, out,
            aligned(out, 16) ? 1 : 0, c.error_flag, c.drop);
  }
  return launch_status();
}

template <typename TT>
int by_out(const EmbedCall& c, int32_t out_dtype, bool drop) {
  if (out_dtype == DFC_DTYPE_F32) return drop ? launch<TT, float, true>(c) : launch<TT, float, false>(c);
  if (out_dtype == DFC_DTYPE_BF16) return drop ? launch<TT, bf16, true>(c) : launch<TT, bf16, false>(c);
  return drop ? launch<TT, f16, true>(c) : launch<TT, f16, false>(c);
}

}  // namespace
}  // namespace dfc

extern "C" int dfc_embedding(const void* tokens, int32_t token_bytes, int64_t n_tokens,
                             const void* table, int32_t table_dtype, int64_t table_pitch,
                             int64_t vocab, int64_t dim, float scale, void* out, int32_t out_dtype,
                             const DfcDropout* dropout, int32_t* error_flag, void* stream) {
  using namespace dfc;
  if (n_tokens < 0 || n_tokens > DFC_MAX_TOKENS || vocab < 0 || vocab > DFC_MAX_VOCAB || dim < 0 ||
      dim > DFC_MAX_DIM || table_pitch < 0 || table_pitch > DFC_MAX_PITCH || n_tokens * dim > (int64_t{1} << 39))
    return DFC_ERR_SIZE;
  if ((token_bytes != 4 && token_bytes != 8) || !known_dtype(table_dtype) || !known_dtype(out_dtype))
    return DFC_ERR_DTYPE;
  EmbedCall c{};
  bool drop;
  const int rc = make_drop_args(dropout, &c.drop, &drop);
  if (rc != DFC_OK) return rc;
  if (n_tokens == 0 || dim == 0) return DFC_OK;
  if (!tokens || !out || (!table && vocab > 0)) return DFC_ERR_NULL;
  if (!aligned(tokens, token_bytes) || !aligned(table, dtype_size(table_dtype)) ||
      !aligned(out, dtype_size(out_dtype)) || !aligned(error_flag, 4))
    return DFC_ERR_ALIGN;
  c.tokens = tokens;
  c.wide = token_bytes == 8;
  c.n_tokens = n_tokens;
  c.table = table;
  c.pitch = table_pitch;
  c.vocab = vocab;
  c.dim = dim;
  c.scale = scale;
  c.out = out;
  c.error_flag = error_flag;
  c.st = static_cast<cudaStream_t>(stream);
  if (table_dtype == DFC_DTYPE_F32) return by_out<float>(c, out_dtype, drop);
  if (table_dtype == DFC_DTYPE_BF16) return by_out<bf16>(c, out_dtype, drop);
  return by_out<f16>(c, out_dtype, drop);
}
