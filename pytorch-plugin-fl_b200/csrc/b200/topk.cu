// The k largest elements of each row with their indices, and the gradient.
//
// Order: descending by value; equal values (and -0 and +0) by ascending
// index; NaN counts as larger than everything, as in argmax.  Every element
// therefore has a distinct 64-bit key, (ordered value bits, ~index), and the
// result is the k largest keys in descending order: one right answer.
#include "vocab_rows.cuh"

namespace flb200 {
namespace {

constexpr int kMaxTop = 1024;
constexpr int kBlock = 512;

// Monotone 32-bit image of a value: unsigned order is float order, NaN on top.
__device__ __forceinline__ uint32_t value_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);  // -0 -> +0
  if (f != f) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t element_key(float f, uint32_t index) {
  return ((uint64_t)value_key(f) << 32) | (uint32_t)~index;
}

// Descending bitonic sort of n (a power of two) keys in shared memory by the
// whole CTA.
__device__ __forceinline__ void sort_desc(uint64_t* s, int n) {
  for (int size = 2; size <= n; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kBlock) {
        const int lo = 2 * i - (i & (stride - 1));
        const uint64_t a = s[lo], b = s[lo + stride];
        const bool desc = (lo & size) == 0;
        if ((a < b) == desc) {
          s[lo] = b;
          s[lo + stride] = a;
        }
      }
    }
  }
  __syncthreads();
}

// The k largest keys of a row by radix selection: eight passes at most over
// the row, each a histogram of the next 8 bits of the keys that match the
// prefix found so far, until the keys at or above the prefix are exactly k.
template <typename T>
__global__ void __launch_bounds__(kBlock)
topk_kernel(const T* __restrict__ x, int64_t ld, int cols, int k, int kpow2, T* __restrict__ values,
            int64_t* __restrict__ indices) {
  __shared__ uint64_t best[kMaxTop];
  __shared__ int hist[256];
  __shared__ int pick, above, filled;
  pdl_prologue();
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ld;
  const int tid = threadIdx.x;
  uint64_t prefix = 0;
  int need = k, shift = 64;
  while (shift > 0) {
    shift -= 8;
    for (int i = tid; i < 256; i += kBlock) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < cols; i += kBlock) {
      const uint64_t key = element_key(Elem<T>::to_f(xr[i]), (uint32_t)i);
      if (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int sum = 0, d = 255;
      while (sum + hist[d] < need) sum += hist[d--];
      pick = d;
      above = sum;
    }
    __syncthreads();
    prefix |= (uint64_t)pick << shift;
    need -= above;
    const bool done = hist[pick] == need;
    __syncthreads();
    if (done) break;
  }
  if (tid == 0) filled = 0;
  for (int i = tid; i < kpow2; i += kBlock) best[i] = 0;
  __syncthreads();
  for (int i = tid; i < cols; i += kBlock) {
    const uint64_t key = element_key(Elem<T>::to_f(xr[i]), (uint32_t)i);
    if (key >= prefix) best[atomicAdd(&filled, 1)] = key;
  }
  sort_desc(best, kpow2);
  for (int i = tid; i < k; i += kBlock) {
    const uint32_t at = ~(uint32_t)best[i];
    indices[row * k + i] = at;
    values[row * k + i] = xr[at];
  }
}

// Gradient: zeros, and dvalues at the indices (distinct in a row).
template <typename T>
__global__ void __launch_bounds__(kBlock)
topk_bwd_kernel(const T* __restrict__ dv, const int64_t* __restrict__ indices, int cols, int k,
                T* __restrict__ dx) {
  pdl_prologue();
  const int64_t row = blockIdx.x;
  T* dr = dx + row * (int64_t)cols;
  const RowSplit sp = split_row(dr, cols);
  uint4* body = reinterpret_cast<uint4*>(dr + sp.head);
  const int e = single_of(sp, threadIdx.x, Elem<T>::kVec);
  if (e >= 0) dr[e] = Elem<T>::from_f(0.f);
  for (int p = threadIdx.x; p < sp.nvec; p += kBlock) st_stream(body + p, make_uint4(0, 0, 0, 0));
  __syncthreads();
  for (int i = threadIdx.x; i < k; i += kBlock) {
    const int64_t at = indices[row * k + i];
    if (at >= 0 && at < cols) dr[at] = dv[row * k + i];
  }
}

}  // namespace
}  // namespace flb200

extern "C" {

FL_B200_API int fl_b200_topk_lastdim(const void* x, int64_t ld, int64_t rows, int64_t cols,
                                     int64_t k, void* values, int64_t* indices, int dtype,
                                     fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(rows >= 0 && k >= 0 && k <= cols);
  if (!is_float_dtype(dtype)) return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (k > kMaxTop || rows > 0x7fffffffLL || cols > 0x7fffff00LL) return FL_B200_ERR_TOO_LARGE;
  if (rows == 0 || k == 0) return FL_B200_OK;
  FLB_CHECK_ARG(x && values && indices && (rows == 1 || ld >= cols));
  int kpow2 = 1;
  while (kpow2 < k) kpow2 *= 2;
  return dispatch_float(dtype, [&](auto t) {
    using T = decltype(t);
    launch_k(topk_kernel<T>, dim3((unsigned)rows), dim3(kBlock), 0, (cudaStream_t)stream,
             reinterpret_cast<const T*>(x), ld, (int)cols, (int)k, kpow2,
             reinterpret_cast<T*>(values), indices);
    return launch_status();
  });
}

FL_B200_API int fl_b200_topk_bwd(const void* dvalues, const int64_t* indices, void* dx, int64_t rows,
                                 int64_t cols, int64_t k, int dtype, fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(rows >= 0 && k >= 0 && k <= cols);
  if (!is_float_dtype(dtype)) return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (k > kMaxTop || rows > 0x7fffffffLL || cols > 0x7fffff00LL) return FL_B200_ERR_TOO_LARGE;
  if (rows == 0 || cols == 0) return FL_B200_OK;
  FLB_CHECK_ARG(dx && (k == 0 || (dvalues && indices)));
  return dispatch_float(dtype, [&](auto t) {
    using T = decltype(t);
    launch_k(topk_bwd_kernel<T>, dim3((unsigned)rows), dim3(kBlock), 0, (cudaStream_t)stream,
             reinterpret_cast<const T*>(dvalues), indices, (int)cols, (int)k,
             reinterpret_cast<T*>(dx));
    return launch_status();
  });
}

}  // extern "C"
