// Dropout with a mask computed from a counter (dfc_philox.cuh), optionally
// added to a residual: y = r + (keep ? x * s : 0), in FP32, rounded once to
// the element type.  The same call on dy with the same counter is the
// gradient.  Dropped elements are zero whatever x holds (Inf and NaN too).
//
// One thread per group of eight elements: one Philox call and one 16-byte
// access per 16-bit operand.  One CTA per tile of 2 x kThreads groups, in
// address order (the shape dfc_compress_ef measured best), both groups' loads
// issued before either is used.
#include "dfc_philox.cuh"

namespace dfc {
namespace {

constexpr int kThreads = 256;
constexpr int kGroups = 2;  // groups per thread

template <typename T, bool RES, bool DROP>
__device__ __forceinline__ void finish8(float (&v)[8], const Raw8<T>& r, uint64_t g,
                                        const DropArgs& a, const DropKey& k) {
  if (DROP) drop8(v, g, a, k);
  if (RES) {
    float f[8];
    unpack8<T>(r, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fadd_rn(f[j], v[j]);
  }
}

// Groups of eight that lie on 16-byte boundaries.
template <typename T, bool RES, bool DROP>
__global__ void __launch_bounds__(kThreads)
    dropout_vec_kernel(const T* x, const T* res, T* y, int64_t groups, DropArgs a) {
  DropKey k{};
  if (DROP) k = drop_key(a);
  const int64_t g0 = static_cast<int64_t>(blockIdx.x) * (kThreads * kGroups) + threadIdx.x;
  Raw8<T> X[kGroups], R[kGroups];
#pragma unroll
  for (int u = 0; u < kGroups; ++u) {
    const int64_t g = g0 + u * kThreads;
    if (g < groups) {
      X[u] = load8(x + 8 * g);
      if (RES) R[u] = load8(res + 8 * g);
    }
  }
#pragma unroll
  for (int u = 0; u < kGroups; ++u) {
    const int64_t g = g0 + u * kThreads;
    if (g < groups) {
      float v[8];
      unpack8<T>(X[u], v);
      finish8<T, RES, DROP>(v, R[u], g, a, k);
      store8(y + 8 * g, pack8<T>(v));
    }
  }
}

// Any alignment, and the last group when n is no multiple of eight: element
// accesses, groups from first_group on.
template <typename T, bool RES, bool DROP>
__global__ void __launch_bounds__(kThreads)
    dropout_any_kernel(const T* x, const T* res, T* y, int64_t first_group, int64_t n, DropArgs a) {
  DropKey k{};
  if (DROP) k = drop_key(a);
  const int64_t g = first_group + static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (8 * g >= n) return;
  uint4 w{};
  if (DROP) w = drop_words(g, a, k);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t i = 8 * g + j;
    if (i < n) {
      float v = to_f32(x[i]);
      if (DROP) v = kept(w, j, a.cmp) ? __fmul_rn(v, a.scale) : 0.0f;
      if (RES) v = __fadd_rn(to_f32(res[i]), v);
      y[i] = from_f32<T>(v);
    }
  }
}

template <typename T, bool RES, bool DROP>
int launch(const void* x, const void* res, void* y, int64_t n, const DropArgs& a, cudaStream_t st) {
  const T* px = static_cast<const T*>(x);
  const T* pr = static_cast<const T*>(res);
  T* py = static_cast<T*>(y);
  int64_t done = 0;
  if (aligned(x, 16) && aligned(res, 16) && aligned(y, 16)) {
    done = n / 8;
    const int64_t tile = kThreads * kGroups;
    if (done > 0)
      dropout_vec_kernel<T, RES, DROP>
          <<<static_cast<unsigned>((done + tile - 1) / tile), kThreads, 0, st>>>(px, pr, py, done, a);
  }
  const int64_t rest = (n + 7) / 8 - done;
  if (rest > 0)
    dropout_any_kernel<T, RES, DROP>
        <<<static_cast<unsigned>((rest + kThreads - 1) / kThreads), kThreads, 0, st>>>(px, pr, py,
                                                                                     done, n, a);
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
