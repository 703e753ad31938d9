// Dropout with a mask computed from a counter (dfc_philox.cuh), optionally
// added to a residual: y = r + (keep ? x * s : 0), in FP32, rounded once to
// the element type.  The same call on dy with the same counter is the
// gradient.  Dropped elements are zero whatever x holds (Inf and NaN too).
//
// One thread takes kGroups groups of eight elements: one Philox call and one
// 16-byte access per 16-bit operand and group.  One CTA per tile of consecutive
// groups, in address order (the shape dfc_compress_ef measured best), all
// loads issued before the first is used.
//
// Bounds (B200, 2^26 elements, p = 0.1, launch included; floors at the measured
// copy bandwidth): FP32 with residual 123 us (floor 123), without 84 (82); bf16
// with residual 65.5 (61.5; 24 instructions an element, 3.1 a cycle and SM),
// without 57 (41; 21 instructions, 2.9 a cycle and SM).  The last is bound by the
// issue of instructions: of the four a cycle that an SM can start three are
// used, the ALU pipe (comparisons, selections, xors) is at 62% of its peak and
// the pipe of the rounds' wide products at 44%.
#include "dfc_philox.cuh"

namespace dfc {
namespace {

constexpr int kThreads = 256;
// Groups per thread: two for 16-bit types, one for FP32 (32 bytes of each
// operand in flight per thread either way), and registers for 6 CTAs per SM (40;
// the 16-bit forms with residual and dropout spill 24 bytes a thread there).
// Of 1, 2 and 4 groups at 3 to 6 CTAs, 2^26 elements with residual, launch
// included: bf16 65.5 us (1 group 73.7; 4 groups 65.5 at 3 CTAs, but 8.2 us
// instead of 6.2 for 2^16 elements), FP32 122.9 us (2 groups 124.9, 4 groups 132).
template <typename T>
constexpr int kGroups = sizeof(T) == 2 ? 2 : 1;

// Element accesses of group g, for any alignment and for a last group of
// fewer than eight elements.
template <typename T, bool RES, bool DROP>
__device__ __forceinline__ void drop_group(const T* x, const T* res, T* y, int64_t g, int64_t n,
                                           const DropArgs& a, const DropKey& k) {
  uint4 w[1] = {};
  if (DROP) drop_words<1>({static_cast<uint64_t>(g)}, a, k, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t i = 8 * g + j;
    if (i < n) {
      float v = to_f32(x[i]);
      if (DROP) v = kept(w[0], j, a.cmp) ? __fmul_rn(v, a.scale) : 0.0f;
      if (RES) v = __fadd_rn(to_f32(res[i]), v);
      y[i] = from_f32<T>(v);
    }
  }
}

// x, res and y on 16-byte boundaries.
template <typename T, bool RES, bool DROP>
__global__ void __launch_bounds__(kThreads, 6)
    dropout_vec_kernel(const T* x, const T* res, T* y, int64_t n, int wide, DropArgs a) {
  constexpr int G = kGroups<T>;
  const int64_t groups = n / 8;
  const int64_t g0 = static_cast<int64_t>(blockIdx.x) * (kThreads * G) + threadIdx.x;
  Raw8<T> X[G], R[G];
#pragma unroll
  for (int u = 0; u < G; ++u) {
    const int64_t g = g0 + u * kThreads;
    if (g < groups) {
      X[u] = load8(x + 8 * g, wide);
      if (RES) R[u] = load8(res + 8 * g, wide);
    }
  }
  DropKey k{};
  uint4 w[G];
  if (DROP) {
    k = drop_key(a);
    uint64_t g[G];
#pragma unroll
    for (int u = 0; u < G; ++u) g[u] = g0 + u * kThreads;
    drop_words<G>(g, a, k, w);
  }
#pragma unroll
  for (int u = 0; u < G; ++u) {
    const int64_t g = g0 + u * kThreads;
    if (g < groups) {
      float v[8];
      unpack8<T>(X[u], v);
      if (DROP) drop8(v, w[u], a);
      if (RES) {
        float f[8];
        unpack8<T>(R[u], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fadd_rn(f[j], v[j]);
      }
      store8(y + 8 * g, pack8<T>(v), wide);
    } else if (g == groups && 8 * g < n) {
      drop_group<T, RES, DROP>(x, res, y, g, n, a, k);
    }
  }
}

// Any alignment: element accesses, 16 or 32 bytes apart between lanes.  2^26
// elements off 16-byte boundaries: bf16 174 us, with residual 180, FP32 283 and
// 297; loads in flight bound it (1.4 instructions a cycle and SM).
template <typename T, bool RES, bool DROP>
__global__ void __launch_bounds__(kThreads)
    dropout_any_kernel(const T* x, const T* res, T* y, int64_t n, DropArgs a) {
  DropKey k{};
  if (DROP) k = drop_key(a);
  drop_group<T, RES, DROP>(x, res, y, static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, n, a, k);
}

template <typename T, bool RES, bool DROP>
int launch(const void* x, const void* res, void* y, int64_t n, const DropArgs& a, cudaStream_t st) {
  const T* px = static_cast<const T*>(x);
  const T* pr = static_cast<const T*>(res);
  T* py = static_cast<T*>(y);
  const int64_t groups = (n + 7) / 8;
  const bool vec = aligned(x, 16) && aligned(res, 16) && aligned(y, 16);
  const int64_t tile = vec ? kThreads * kGroups<T> : kThreads;
  const unsigned grid = static_cast<unsigned>((groups + tile - 1) / tile);
  if (vec)
    dropout_vec_kernel<T, RES, DROP><<<grid, kThreads, 0, st>>>(
        px, pr, py, n, aligned(x, 32) && aligned(res, 32) && aligned(y, 32), a);
  else
    dropout_any_kernel<T, RES, DROP><<<grid, kThreads, 0, st>>>(px, pr, py, n, a);
  return launch_status();
}

template <typename T>
int dispatch(const void* x, const void* res, void* y, int64_t n, const DropArgs& a, bool drop,
             cudaStream_t st) {
  if (res) return drop ? launch<T, true, true>(x, res, y, n, a, st) : launch<T, true, false>(x, res, y, n, a, st);
  return drop ? launch<T, false, true>(x, res, y, n, a, st) : launch<T, false, false>(x, res, y, n, a, st);
}

}  // namespace
}  // namespace dfc

extern "C" int dfc_dropout(const void* x, const void* residual, void* y, int64_t n, int32_t dtype,
                           const DfcDropout* dropout, void* stream) {
  using namespace dfc;
  if (n < 0 || n > (int64_t{1} << 39)) return DFC_ERR_SIZE;
  if (!known_dtype(dtype)) return DFC_ERR_DTYPE;
  DropArgs a;
  bool drop;
  const int rc = make_drop_args(dropout, &a, &drop);
  if (rc != DFC_OK) return rc;
  if (n == 0) return DFC_OK;
  if (!x || !y) return DFC_ERR_NULL;
  const uintptr_t size = dtype_size(dtype);
  if (!aligned(x, size) || !aligned(residual, size) || !aligned(y, size)) return DFC_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DFC_DTYPE_F32) return dispatch<float>(x, residual, y, n, a, drop, st);
  if (dtype == DFC_DTYPE_BF16) return dispatch<bf16>(x, residual, y, n, a, drop, st);
  return dispatch<f16>(x, residual, y, n, a, drop, st);
}
