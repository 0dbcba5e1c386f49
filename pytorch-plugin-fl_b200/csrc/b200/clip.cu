// The norm of a list of tensors taken as one vector, and the tensors clipped
// to a bound on it.
//
//   norm = sqrt(sum x^2) or max |x|;  out = x * min(1, max_norm / (norm + 1e-6))
//
// Two launches over all tensors, whatever their number, sizes and types: the
// table of tensors is a kernel parameter, so nothing is copied to the device
// and a captured graph holds its own.  (Lists longer than one table take a
// launch of each kind for every table.)  Work is dealt in chunks of 32 KB; a
// resident CTA walks every gridDim-th chunk and looks its tensor up in the
// table.  The first launch leaves one fp64 partial sum a CTA; every CTA of the
// second adds them all in one order (a few hundred loads from L2), so there
// are no atomics, nothing to set to zero and the norm has one order of
// addition for a given list and GPU.
//
// Bound by memory: the tensors are read, and read and written again (961 M
// bf16 elements: 920 us, 6.3 TB/s over the three; the norm is not known before
// all has been read).  The second launch walks the chunks backwards: what the
// first read last is still in L2 (33 MB lie there whole: 128 tensors in
// 10.6 us).  Where the factor is 1 and a tensor is its own output, it writes
// nothing.
//
// Squares are added in fp32 over a thread's share of a chunk (64 elements of
// 16 bits), then in fp64; a share whose fp32 sum is not well inside the range
// is added again in fp64 from registers, so the norm of tiny or huge
// gradients is right where fp32 squares would be 0 or inf.
#include <vector>

#include "common.cuh"

namespace flb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kPacks = 8;                       // 16-byte packs a thread and chunk
constexpr int kChunkBytes = kThreads * kPacks * 16;

// MAXT tensors a launch.  Chunk c of the launch belongs to the tensor t with
// first[t] <= c < first[t + 1].
template <int MAXT>
struct Table {
  int count;
  uint32_t chunks;
  const void* in[MAXT];
  void* out[MAXT];
  int64_t numel[MAXT];
  uint32_t first[MAXT + 1];
  uint8_t dtype[MAXT];
};

// The tensor of chunk c: a few steps where a walk from one end took as many as
// there are tensors (2 us of the launch for 128).
template <int MAXT>
__device__ __forceinline__ int tensor_of(const Table<MAXT>& tab, uint32_t c, int last) {
  if (tab.first[last] <= c && c < tab.first[last + 1]) return last;  // as the chunk before
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (tab.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The packs of a tensor: elements from the first 16-byte boundary at or
// before its first one.
struct Span {
  int64_t first, last;  // in elements from that boundary
};
template <typename T>
__device__ __forceinline__ Span span_of(const void* p, int64_t numel) {
  const int64_t shift = (int64_t)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
  return {shift, shift + numel};
}

// |x| as an integer that orders as it does, NaN above everything.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <typename T, bool MAX>
__device__ __forceinline__ void add_chunk(const void* p, int64_t numel, int64_t chunk, double& sum, uint32_t& top) {
  constexpr int VW = Elem<T>::kVec;
  const Span s = span_of<T>(p, numel);
  const T* base = static_cast<const T*>(p) - s.first;
  const int64_t e0 = chunk * (kChunkBytes / (int64_t)sizeof(T)) + (int64_t)threadIdx.x * VW;
  uint4 v[kPacks];
  if (e0 - threadIdx.x * VW >= s.first && e0 - threadIdx.x * VW + kChunkBytes / (int64_t)sizeof(T) <= s.last) {
#pragma unroll
    for (int i = 0; i < kPacks; ++i) v[i] = ld_plain(base + e0 + (int64_t)i * kThreads * VW);
  } else {
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      const int64_t e = e0 + (int64_t)i * kThreads * VW;
      v[i] = make_uint4(0, 0, 0, 0);
      if (e >= s.first && e + VW <= s.last) {
        v[i] = ld_plain(base + e);
      } else if (e + VW > s.first && e < s.last) {
        float f[VW];
#pragma unroll
        for (int k = 0; k < VW; ++k)
          f[k] = e + k >= s.first && e + k < s.last ? Elem<T>::to_f(base[e + k]) : 0.f;
        v[i] = pack<T>(f);
      }
    }
  }
  float acc = 0.f;
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    float f[VW];
    unpack<T>(v[i], f);
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      if constexpr (MAX) top = max(top, magnitude(f[k]));
      else acc = fmaf(f[k], f[k], acc);
    }
  }
  if constexpr (!MAX) {
    if (acc > 1e-20f && acc < 1e38f) {
      sum += (double)acc;
    } else {
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        float f[VW];
        unpack<T>(v[i], f);
#pragma unroll
        for (int k = 0; k < VW; ++k) sum = fma((double)f[k], (double)f[k], sum);
      }
    }
  }
}

// One partial a CTA: the sum of squares, or the largest magnitude's bits.
template <int MAXT, bool MAX>
__global__ void __launch_bounds__(kThreads)
norm_kernel(const __grid_constant__ Table<MAXT> tab, double* partial) {
  pdl_prologue();
  __shared__ double warp_sum[kThreads / 32];
  double sum = 0.0;
  uint32_t top = 0;
  int t = 0;
  for (uint32_t c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
    t = tensor_of(tab, c, t);
    const int64_t chunk = c - tab.first[t];
    switch (tab.dtype[t]) {
      case FL_B200_F32: add_chunk<float, MAX>(tab.in[t], tab.numel[t], chunk, sum, top); break;
      case FL_B200_BF16: add_chunk<__nv_bfloat16, MAX>(tab.in[t], tab.numel[t], chunk, sum, top); break;
      default: add_chunk<__half, MAX>(tab.in[t], tab.numel[t], chunk, sum, top); break;
    }
  }
  if constexpr (MAX) sum = (double)top;  // exact: 31 bits
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const double o = __shfl_xor_sync(0xffffffffu, sum, off);
    sum = MAX ? fmax(sum, o) : sum + o;
  }
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) sum = MAX ? fmax(sum, warp_sum[w]) : sum + warp_sum[w];
    partial[blockIdx.x] = sum;
  }
}

// The norm from n partials, in every thread of the CTA.
__device__ __forceinline__ double norm_of(const double* partial, int n, bool max_norm) {
  __shared__ double warp_sum[kThreads / 32];
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) sum = max_norm ? fmax(sum, partial[i]) : sum + partial[i];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const double o = __shfl_xor_sync(0xffffffffu, sum, off);
    sum = max_norm ? fmax(sum, o) : sum + o;
  }
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = warp_sum[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) sum = max_norm ? fmax(sum, warp_sum[w]) : sum + warp_sum[w];
  return max_norm ? (double)__uint_as_float((uint32_t)sum) : sqrt(sum);
}

__global__ void __launch_bounds__(kThreads)
norm_result_kernel(const double* partial, int n, int max_norm, float* norm) {
  pdl_prologue();
  const double r = norm_of(partial, n, max_norm != 0);
  if (threadIdx.x == 0) *norm = (float)r;
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const void* p, void* q, int64_t numel, int64_t chunk, float factor) {
  constexpr int VW = Elem<T>::kVec;
  const Span s = span_of<T>(p, numel);
  const T* base = static_cast<const T*>(p) - s.first;
  T* out = static_cast<T*>(q) - s.first;
  const int64_t c0 = chunk * (kChunkBytes / (int64_t)sizeof(T));
  // both on the same place of a 16-byte pack, or element by element
  if (((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15u) == 0) {
    uint4 v[kPacks];
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      const int64_t e = c0 + (int64_t)(i * kThreads + threadIdx.x) * VW;
      if (e >= s.first && e + VW <= s.last) v[i] = ld_plain(base + e);
    }
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      const int64_t e = c0 + (int64_t)(i * kThreads + threadIdx.x) * VW;
      if (e >= s.first && e + VW <= s.last) {
        float f[VW];
        unpack<T>(v[i], f);
#pragma unroll
        for (int k = 0; k < VW; ++k) f[k] *= factor;
        st_stream(out + e, pack<T>(f));
      } else if (e + VW > s.first && e < s.last) {
        for (int k = 0; k < VW; ++k)
          if (e + k >= s.first && e + k < s.last) out[e + k] = Elem<T>::from_f(Elem<T>::to_f(base[e + k]) * factor);
      }
    }
  } else {
    const int64_t c1 = min(s.last, c0 + kChunkBytes / (int64_t)sizeof(T));
#pragma unroll 8
    for (int64_t e = max(c0, s.first) + threadIdx.x; e < c1; e += kThreads)
      out[e] = Elem<T>::from_f(Elem<T>::to_f(base[e]) * factor);
  }
}

template <int MAXT>
__global__ void __launch_bounds__(kThreads)
scale_kernel(const __grid_constant__ Table<MAXT> tab, const double* partial, int n, int max_kind, float bound,
             float* norm) {
  pdl_prologue();
  const double r = norm_of(partial, n, max_kind != 0);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)r;
  // NaN stays NaN: a comparison with it is false
  const double ratio = (double)bound / (r + 1e-6);
  const float factor = ratio >= 1.0 ? 1.f : (float)ratio;
  int t = 0;
  for (uint32_t i = blockIdx.x; i < tab.chunks; i += gridDim.x) {
    const uint32_t c = tab.chunks - 1 - i;
    t = tensor_of(tab, c, t);
    if (factor == 1.f && tab.in[t] == tab.out[t]) continue;
    const int64_t chunk = c - tab.first[t];
    switch (tab.dtype[t]) {
      case FL_B200_F32: scale_chunk<float>(tab.in[t], tab.out[t], tab.numel[t], chunk, factor); break;
      case FL_B200_BF16: scale_chunk<__nv_bfloat16>(tab.in[t], tab.out[t], tab.numel[t], chunk, factor); break;
      default: scale_chunk<__half>(tab.in[t], tab.out[t], tab.numel[t], chunk, factor); break;
    }
  }
}

struct List {
  const void* const* in;
  void* const* out;  // NULL: the norm alone
  const int64_t* numel;
  const int* dtype;
  int64_t count;
};

int grid_of(uint32_t chunks, const DeviceInfo& dev) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(chunks, 4ll * dev.sm_count));
}

// Fills one table from tensor `from` on; returns the tensor after its last.
template <int MAXT>
int64_t fill(const List& l, int64_t from, Table<MAXT>& tab) {
  tab.count = 0;
  tab.chunks = 0;
  int64_t i = from;
  for (; i < l.count && tab.count < MAXT; ++i) {
    const int64_t n = l.numel[i];
    if (n == 0) continue;
    const int64_t size = dtype_size(l.dtype[i]);
    const int64_t shift = (int64_t)(reinterpret_cast<uintptr_t>(l.in[i]) & 15u);
    const int64_t chunks = ceil_div(shift + n * size, kChunkBytes);
    if (tab.chunks + chunks > 0x7fffffff) {
      if (tab.count == 0) return -1;
      break;
    }
    const int t = tab.count++;
    tab.in[t] = l.in[i];
    tab.out[t] = l.out ? l.out[i] : nullptr;
    tab.numel[t] = n;
    tab.dtype[t] = (uint8_t)l.dtype[i];
    tab.first[t] = tab.chunks;
    tab.chunks += (uint32_t)chunks;
    tab.first[t + 1] = tab.chunks;
  }
  return i;
}

template <int MAXT>
int run(const List& l, int max_kind, float bound, float* norm, double* partial, const DeviceInfo& dev,
        cudaStream_t stream) {
  static thread_local Table<MAXT> tab;  // kilobytes: not on the caller's stack
  int n = 0;
  const int room = (int)(ceil_div(l.count, MAXT) * 4 * dev.sm_count);
  for (int64_t i = 0; i < l.count;) {
    i = fill(l, i, tab);
    if (i < 0) return FL_B200_ERR_TOO_LARGE;
    if (tab.count == 0) break;
    const int grid = grid_of(tab.chunks, dev);
    if (n + grid > room) return FL_B200_ERR_WORKSPACE;
    if (max_kind) launch_k((norm_kernel<MAXT, true>), grid, kThreads, 0, stream, tab, partial + n);
    else launch_k((norm_kernel<MAXT, false>), grid, kThreads, 0, stream, tab, partial + n);
    n += grid;
  }
  if (l.out == nullptr || n == 0) {
    launch_k(norm_result_kernel, 1, kThreads, 0, stream, (const double*)partial, n, max_kind, norm);
    return launch_status();
  }
  for (int64_t i = 0; i < l.count;) {
    i = fill(l, i, tab);
    if (tab.count == 0) break;
    launch_k(scale_kernel<MAXT>, grid_of(tab.chunks, dev), kThreads, 0, stream, tab, (const double*)partial, n,
             max_kind, bound, norm);
    norm = nullptr;
  }
  return launch_status();
}

// Whether every output lies apart from all other outputs and from all tensors
// but its own: CTAs scale them in no order, so one written under another's
// hands would come out scaled once, twice or in parts.
bool outputs_apart(const List& l) {
  struct Range {
    uintptr_t lo, hi;
  };
  static thread_local std::vector<Range> outs;
  outs.clear();
  outs.reserve((size_t)l.count);
  auto range = [&](const void* p, int64_t i) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    return Range{lo, lo + (uintptr_t)(l.numel[i] * dtype_size(l.dtype[i]))};
  };
  for (int64_t i = 0; i < l.count; ++i)
    if (l.numel[i]) outs.push_back(range(l.out[i], i));
  const auto before = [](const Range& a, const Range& b) { return a.lo < b.lo; };
  std::sort(outs.begin(), outs.end(), before);
  for (size_t i = 1; i < outs.size(); ++i)
    if (outs[i - 1].hi > outs[i].lo) return false;
  for (int64_t i = 0; i < l.count; ++i) {
    if (l.numel[i] == 0 || l.in[i] == l.out[i]) continue;
    const Range r = range(l.in[i], i);
    auto next = std::lower_bound(outs.begin(), outs.end(), r, before);
    if (next != outs.end() && next->lo < r.hi) return false;
    if (next != outs.begin() && (next - 1)->hi > r.lo) return false;
  }
  return true;
}

// A table's size is that of the launch's parameters: 20 KB for 512 tensors.
int any(const List& l, int max_kind, float bound, float* norm, void* workspace, size_t bytes,
        cudaStream_t stream) {
  FLB_CHECK_ARG(l.count >= 0 && norm && (max_kind == 0 || max_kind == 1));
  FLB_CHECK_ARG(l.count == 0 || (l.in && l.numel && l.dtype));
  if (!aligned_to(4, {norm})) return FL_B200_ERR_MISALIGNED;
  int64_t tensors = 0;
  for (int64_t i = 0; i < l.count; ++i) {
    if (!is_float_dtype(l.dtype[i])) return FL_B200_ERR_UNSUPPORTED_DTYPE;
    FLB_CHECK_ARG(l.numel[i] >= 0 && (l.numel[i] == 0 || (l.in[i] && (!l.out || l.out[i]))));
    const int size = dtype_size(l.dtype[i]);
    const uintptr_t p = reinterpret_cast<uintptr_t>(l.in[i]), q = l.out ? reinterpret_cast<uintptr_t>(l.out[i]) : p;
    if (l.numel[i] && ((p | q) % size) != 0) return FL_B200_ERR_MISALIGNED;
    tensors += l.numel[i] > 0;
  }
  if (l.out) {
    try {
      FLB_CHECK_ARG(outputs_apart(l));
    } catch (...) {  // no memory for the list
      return FL_B200_ERR_TOO_LARGE;
    }
  }
  DeviceInfo dev;
  const int st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  if (workspace == nullptr || bytes < fl_b200_grad_norm_workspace_size(l.count)) return FL_B200_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FL_B200_ERR_MISALIGNED;
  auto* partial = static_cast<double*>(workspace);
  if (tensors <= 32) return run<32>(l, max_kind, bound, norm, partial, dev, stream);
  if (tensors <= 128) return run<128>(l, max_kind, bound, norm, partial, dev, stream);
  return run<512>(l, max_kind, bound, norm, partial, dev, stream);
}

}  // namespace
}  // namespace flb200

extern "C" {

FL_B200_API size_t fl_b200_grad_norm_workspace_size(int64_t count) {
  using namespace flb200;
  DeviceInfo dev;
  if (count < 0 || current_device_info(&dev) != FL_B200_OK) return 0;
  return (size_t)std::max<int64_t>(1, ceil_div(count, 32)) * 4 * dev.sm_count * sizeof(double);
}

FL_B200_API int fl_b200_grad_norm(const void* const* tensors, const int64_t* numels, const int* dtypes,
                                  int64_t count, int max_kind, float* norm, void* workspace,
                                  size_t workspace_bytes, fl_b200_stream_t stream) {
  return flb200::any({tensors, nullptr, numels, dtypes, count}, max_kind, 0.f, norm, workspace, workspace_bytes,
                     static_cast<cudaStream_t>(stream));
}

FL_B200_API int fl_b200_clip_grads(const void* const* tensors, void* const* outs, const int64_t* numels,
                                   const int* dtypes, int64_t count, float max_norm, int max_kind, float* norm,
                                   void* workspace, size_t workspace_bytes, fl_b200_stream_t stream) {
  FLB_CHECK_ARG(max_norm >= 0.f && (count <= 0 || outs));
  return flb200::any({tensors, outs, numels, dtypes, count}, max_kind, max_norm, norm, workspace, workspace_bytes,
                     static_cast<cudaStream_t>(stream));
}

}  // extern "C"
