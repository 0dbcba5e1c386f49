// The k largest elements of each row with their indices, and the gradient.
//
// Order: descending by value; equal values (and -0 and +0) by ascending
// index; NaN counts as larger than everything, as in argmax.  Every element
// therefore has a distinct 64-bit key, (ordered value bits, ~index), and the
// result is the k largest keys in descending order: one right answer.
#include "vocab_rows.cuh"

namespace flb200 {
namespace {

constexpr int kMaxTop = FL_B200_TOPK_MAX;
constexpr int kBlock = 512;
constexpr int kWarps = kBlock / 32;
constexpr int kPacks = 8;      // 16-byte packs a thread holds: a chunk of the row is kBlock * kPacks
constexpr int kCap = 3072;     // candidates kept
constexpr int kTighten = 1536; // above this many the threshold is raised over the candidates
constexpr int kQueue = 512;    // packs of a chunk that hold candidates
constexpr int kSort = 2048;    // keys sorted at the end: at most 1.25 * kMaxTop

// Monotone 32-bit image of a value: unsigned order is float order, NaN on
// top; never 0.
__device__ __forceinline__ uint32_t value_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);  // -0 -> +0
  if (f != f) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t element_key(float f, uint32_t index) {
  return ((uint64_t)value_key(f) << 32) | (uint32_t)~index;
}

// NaN-propagating maximum of a pack.
template <typename T>
__device__ __forceinline__ float pack_top(const uint4& u) {
  float r;
  if constexpr (std::is_same<T, float>::value) {
    float a, b;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(__uint_as_float(u.x)), "f"(__uint_as_float(u.y)));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(__uint_as_float(u.z)), "f"(__uint_as_float(u.w)));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  } else {
    uint32_t a, b, c;
    if constexpr (std::is_same<T, __half>::value) {
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(a) : "r"(u.x), "r"(u.y));
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(b) : "r"(u.z), "r"(u.w));
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    } else {
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(u.x), "r"(u.y));
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(u.z), "r"(u.w));
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    }
    const uint64_t p = pair_from_bits<T>(c);
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(f2_lo(p)), "f"(f2_hi(p)));
  }
  return r;
}

struct Shared {
  uint64_t cand[kCap];       // candidates, in no order
  union {
    struct {
      uint4 pack[kQueue];
      int at[kQueue];
    } q;
    uint64_t sort[kSort];
  };
  int sums[2][kWarps];
  int hist[256];
  int filled, queued[2], pick, above;
  uint4 stage[kPacks][kBlock];  // the next chunk, each thread's own packs
};

// Sum of v over the CTA, in every thread.  `parity` alternates between the
// two halves of the scratch, so that one barrier a call is enough.
__device__ __forceinline__ int block_sum(Shared& s, int v, int& parity) {
  const int lane = threadIdx.x & 31;
  v = __reduce_add_sync(0xffffffffu, v);
  if (lane == 0) s.sums[parity][threadIdx.x >> 5] = v;
  __syncthreads();
  v = __reduce_add_sync(0xffffffffu, lane < kWarps ? s.sums[parity][lane] : 0);
  parity ^= 1;
  return v;
}

// A key K that at least k of the counted keys reach, and at most `enough`
// where that is possible: found bit by bit below the bits that `lo` and `hi`
// share, all counted keys lying between these two.  count(K) is the thread's
// own number of keys >= K.
template <typename K, typename F>
__device__ __forceinline__ K bisect(Shared& s, K lo, K hi, int k, int enough, int& parity, F count) {
  K at = lo;
  int bit = (int)sizeof(K) * 8 - 1;
  while (bit >= 0 && (((lo ^ hi) >> bit) & 1) == 0) --bit;
  at = bit < 0 ? lo : (lo >> bit >> 1) << bit << 1;
  for (; bit >= 0; --bit) {
    const K tried = at | ((K)1 << bit);
    const int n = block_sum(s, count(tried), parity);
    if (n >= k) {
      at = tried;
      if (n <= enough) break;
    }
  }
  return at;
}

__device__ __forceinline__ void append(Shared& s, uint64_t key) {
  const int slot = atomicAdd(&s.filled, 1);
  if (slot < kCap) s.cand[slot] = key;
}

// Keeps the candidates at or above a 64-bit key.
__device__ __forceinline__ void keep_above(Shared& s, int n, uint64_t floor) {
  uint64_t mine[kCap / kBlock];
#pragma unroll
  for (int i = 0; i < kCap / kBlock; ++i) {
    const int j = threadIdx.x + i * kBlock;
    mine[i] = j < n ? s.cand[j] : 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) s.filled = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kCap / kBlock; ++i)
    if (mine[i] >= floor && mine[i] != 0) append(s, mine[i]);
  __syncthreads();
}

// Descending bitonic sort of s.sort[0..n), n a power of two.
__device__ __forceinline__ void sort_desc(Shared& s, int n) {
  for (int size = 2; size <= n; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kBlock) {
        const int lo = 2 * i - (i & (stride - 1));
        const uint64_t a = s.sort[lo], b = s.sort[lo + stride];
        if ((a < b) == ((lo & size) == 0)) {
          s.sort[lo] = b;
          s.sort[lo + stride] = a;
        }
      }
    }
  }
  __syncthreads();
}

// The k largest keys of elements [lo, hi) by radix selection: eight passes
// at most, each a histogram of the next 8 bits of the keys that match the
// prefix found so far, until exactly k keys reach it.  For slices whose
// candidates overflow; right for any values.
template <typename T>
__device__ __noinline__ void radix_select(Shared& s, const T* xr, int lo, int hi, int k) {
  const int tid = threadIdx.x;
  uint64_t prefix = 0;
  int need = k, shift = 64;
  while (shift > 0) {
    shift -= 8;
    for (int i = tid; i < 256; i += kBlock) s.hist[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kBlock) {
      const uint64_t key = element_key(Elem<T>::to_f(xr[i]), (uint32_t)i);
      if (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&s.hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int sum = 0, d = 255;
      while (d > 0 && sum + s.hist[d] < need) sum += s.hist[d--];
      s.pick = d;
      s.above = sum;
    }
    __syncthreads();
    prefix |= (uint64_t)s.pick << shift;
    need -= s.above;
    const bool done = s.hist[s.pick] == need;
    __syncthreads();
    if (done) break;
  }
  if (tid == 0) s.filled = 0;
  __syncthreads();
  for (int i = lo + tid; i < hi; i += kBlock) {
    const uint64_t key = element_key(Elem<T>::to_f(xr[i]), (uint32_t)i);
    if (key >= prefix) append(s, key);
  }
  __syncthreads();
}

// Descending bitonic sort across the lanes of a warp.
__device__ __forceinline__ uint32_t warp_sort_desc(uint32_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      const uint32_t w = __shfl_xor_sync(0xffffffffu, v, stride);
      const bool larger = ((lane & stride) == 0) == ((lane & size) == 0);
      v = larger ? max(v, w) : min(v, w);
    }
  }
  return v;
}

// The 16-byte packs of one slice.
struct Packs {
  const uint4* body;
  int nvec;
};
// Copies chunk `base` of the slice into the thread's own stage slots.
__device__ __forceinline__ void issue(Shared& s, const Packs& src, int base) {
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    const int p = base + i * kBlock + threadIdx.x;
    if (p < src.nvec) cp_async16(&s.stage[i][threadIdx.x], src.body + p);
  }
  cp_async_commit();
}

// Candidates of elements [lo, hi) of a row, which hold its k largest keys
// (k <= hi - lo); returns their number, in every thread, more than kCap when
// they did not fit.  The slice's first chunk has been issued; the first chunk
// of `next` is when this returns.
//
// The slice is read once, a chunk at a time, against a threshold below which
// nothing can be among the k largest.  The first threshold comes from the
// first chunk: each of its W warps sorts its threads' maxima, and the least
// of the warps' ceil(k / W)-th is reached by k elements (a little over twice
// k reach it when the row is in no order).  After that a pack matters only if
// its maximum exceeds the threshold, which few do: they go to a queue whose
// elements the whole CTA then tests.  An element of a later chunk that only
// equals the threshold loses to the k before it, so the test is strict there
// and ties resolve by index.
template <typename T>
__device__ __forceinline__ int collect(Shared& s, const T* xr, int lo, int hi, int k, const Packs& next,
                                       int& parity) {
  constexpr int VW = Elem<T>::kVec;
  const int tid = threadIdx.x, lane = tid & 31;
  const RowSplit sp = split_row(xr + lo, hi - lo);
  const Packs src = {reinterpret_cast<const uint4*>(xr + lo + sp.head), sp.nvec};
  if (tid == 0) s.filled = s.queued[0] = s.queued[1] = 0;
  __syncthreads();
  if (tid < sp.head) append(s, element_key(Elem<T>::to_f(xr[lo + tid]), (uint32_t)(lo + tid)));
  if (sp.nvec == 0) issue(s, next, 0);
  uint32_t reached = 0;  // a key that k elements seen so far reach (0: none known)
  int turn = 0;
  bool fits = true;
  for (int base = 0; base < sp.nvec; base += kBlock * kPacks, turn ^= 1) {
    uint4 u[kPacks];
    uint32_t top[kPacks];
    cp_async_wait_all();
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      const int p = base + i * kBlock + tid;
      u[i] = s.stage[i][tid];
      top[i] = p < sp.nvec ? value_key(pack_top<T>(u[i])) : 0;
    }
    if (base + kBlock * kPacks < sp.nvec) {
      issue(s, src, base + kBlock * kPacks);
    } else {
      issue(s, next, 0);
    }
    if (!fits || reached == 0xffffffffu) continue;  // (k NaN are kept)
    uint32_t least = reached + 1;  // what an element of this chunk must reach to matter
    const int warps = min(kWarps, (sp.nvec - base) / 32);  // with a pack in every thread
    if (reached == 0 && warps * 32 >= k) {
      uint32_t most = top[0];
#pragma unroll
      for (int i = 1; i < kPacks; ++i) most = max(most, top[i]);
      most = __shfl_sync(0xffffffffu, warp_sort_desc(most), (k + warps - 1) / warps - 1);
      if (lane == 0) s.sums[parity][tid >> 5] = (int)most;
      __syncthreads();
      least = reached =
          __reduce_min_sync(0xffffffffu, lane < warps ? (uint32_t)s.sums[parity][lane] : 0xffffffffu);
      parity ^= 1;
    }
    const auto packs_over = [&](uint32_t c) {
      int m = 0;
#pragma unroll
      for (int i = 0; i < kPacks; ++i) m += top[i] >= c;
      return m;
    };
    int hits = block_sum(s, packs_over(least), parity);
    const int n = s.filled;  // (appends follow the next barrier)
    if (tid == 0) s.queued[turn ^ 1] = 0;
    fits = n <= kCap;
    if (!fits) continue;
    if (n > kTighten || hits > max(4 * k, kQueue)) {
      if (hits >= k) {  // rising rows: the k-th largest maximum of this chunk's packs
        const uint32_t t = bisect<uint32_t>(s, 0u, ~0u, k, k + k / 8, parity, packs_over);
        if (t > least) least = reached = t;
      }
      if (n > kTighten) {  // the k-th largest of the candidates
        const uint32_t t = bisect<uint32_t>(s, 0u, ~0u, k, k + k / 8, parity, [&](uint32_t c) {
          int m = 0;
          for (int j = tid; j < n; j += kBlock) m += (uint32_t)(s.cand[j] >> 32) >= c;
          return m;
        });
        keep_above(s, n, (uint64_t)t << 32);
        reached = max(reached, t);
        if (t == 0xffffffffu) continue;
        least = max(least, t + 1);
      }
      hits = block_sum(s, packs_over(least), parity);
    }
    if (hits == 0) continue;
    if (hits <= kQueue) {
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        if (top[i] < least) continue;
        const int slot = atomicAdd(&s.queued[turn], 1);
        s.q.pack[slot] = u[i];
        s.q.at[slot] = base + i * kBlock + tid;
      }
      __syncthreads();
      const int queued = s.queued[turn];
      const T* q = reinterpret_cast<const T*>(s.q.pack);
      for (int j = tid; j < queued * VW; j += kBlock) {
        const int e = lo + sp.head + s.q.at[j / VW] * VW + j % VW;
        const uint64_t key = element_key(Elem<T>::to_f(q[j]), (uint32_t)e);
        if ((uint32_t)(key >> 32) >= least) append(s, key);
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        if (top[i] < least) continue;
        float f[VW];
        unpack<T>(u[i], f);
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          const int e = lo + sp.head + (base + i * kBlock + tid) * VW + j;
          if (value_key(f[j]) >= least) append(s, element_key(f[j], (uint32_t)e));
        }
      }
    }
  }
  __syncthreads();
  if (tid < sp.tail) {
    const int e = hi - sp.tail + tid;
    append(s, element_key(Elem<T>::to_f(xr[e]), (uint32_t)e));
  }
  __syncthreads();
  return fits ? s.filled : kCap + 1;
}

// One CTA a row, walking rows, or a cluster with a slice of the row in each
// CTA when there are few: every CTA finds its slice's k largest, CTA 0 takes
// them all and orders the k largest of the row.
template <typename T>
__global__ void __launch_bounds__(kBlock, 2)
topk_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int cols, int k, T* __restrict__ values,
            int64_t* __restrict__ indices) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  pdl_prologue();
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int tid = threadIdx.x;
  int parity = 0;
  // slices of whole groups of 64 elements
  const int per = (int)(ceil_div(ceil_div(cols, C), 64) * 64);
  const int lo = min(cols, rank * per), hi = min(cols, lo + per);
  const int want = min(k, hi - lo);
  const auto packs_of = [&](int64_t row) {
    if (row >= rows) return Packs{nullptr, 0};
    const T* at = x + row * ld + lo;
    const RowSplit sp = split_row(at, hi - lo);
    return Packs{reinterpret_cast<const uint4*>(at + sp.head), sp.nvec};
  };
  const int64_t step = cluster_count();
  issue(s, packs_of(cluster_id()), 0);
  for (int64_t row = cluster_id(); row < rows; row += step) {
    const T* xr = x + row * ld;
    int n = collect(s, xr, lo, hi, want, packs_of(row + step), parity);
    if (n > kCap) {
      radix_select(s, xr, lo, hi, want);
      n = want;
    }
    // to a few more than k at most, without their order
    const auto shrink = [&](int most) {
      const uint64_t f = bisect<uint64_t>(s, 0ull, ~0ull, min(k, n), most, parity, [&](uint64_t c) {
        int m = 0;
        for (int j = tid; j < n; j += kBlock) m += s.cand[j] >= c;
        return m;
      });
      keep_above(s, n, f);
      n = s.filled;
    };
    // few keys: each one's place is the number of keys above it
    const auto place_all = [&](auto put) {
      int per_key = 32;
      while (per_key * n > kBlock) per_key >>= 1;
      const int i = tid / per_key;
      const uint64_t key = i < n ? s.cand[i] : 0;
      int place = 0;
      for (int j = tid % per_key; j < n; j += per_key) place += s.cand[j] > key;
      for (int o = per_key >> 1; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
      if (i < n && tid % per_key == 0 && place < k) put(place, key);
    };
    const int most = max(k + k / 4, 128);
    if (n > most) shrink(most);
    if (C > 1) {
      // this slice's k largest, 0 past the last
      if (n <= kBlock / 2) {
        for (int i = tid; i < k; i += kBlock) s.sort[i] = 0;
        __syncthreads();
        place_all([&](int place, uint64_t key) { s.sort[place] = key; });
      } else {
        if (n > k) shrink(k);
        for (int i = tid; i < k; i += kBlock) s.sort[i] = i < n ? s.cand[i] : 0;
      }
      cluster_sync_all();
      if (rank == 0) {
        for (int i = tid; i < C * k; i += kBlock)
          s.cand[i] = (uint64_t)ld_remote_s64(remote_smem(&s.sort[i % k], i / k));
        n = C * k;
        __syncthreads();
      }
      cluster_sync_all();  // the others' lists are read
      if (rank == 0 && n > most) shrink(most);
    }
    if (rank == 0) {
      const auto put = [&](int place, uint64_t key) {
        const uint32_t at = ~(uint32_t)key;
        indices[row * k + place] = at;
        values[row * k + place] = xr[at];
      };
      if (n <= kBlock / 2) {
        place_all(put);
      } else {
        int size = 1;
        while (size < n) size <<= 1;
        for (int i = tid; i < size; i += kBlock) s.sort[i] = i < n ? s.cand[i] : 0;
        sort_desc(s, size);
        for (int i = tid; i < k; i += kBlock) put(i, s.sort[i]);
      }
    }
    __syncthreads();  // the next row's candidates take these ones' place
  }
  cp_async_wait_all();
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
  DeviceInfo dev;
  const int st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  return dispatch_float(dtype, [&](auto t) {
    using T = decltype(t);
    // few rows: up to 8 CTAs a row, with a pack a thread at least, whose
    // lists fit CTA 0
    int cluster = 1;
    while (cluster < 8 && rows * cluster < dev.sm_count && cluster * 2 * k <= kCap &&
           cols / (cluster * 2) >= kBlock * Elem<T>::kVec)
      cluster *= 2;
    // (per launch: the attribute is held per device)
    if (cudaFuncSetAttribute(topk_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)sizeof(Shared)) != cudaSuccess)
      return launch_status();
    const int64_t ctas = std::min<int64_t>(rows, 2 * dev.sm_count) * cluster;
    return launch_cluster(topk_kernel<T>, cluster > 1 ? rows * cluster : ctas, cluster, kBlock,
                          sizeof(Shared), (cudaStream_t)stream, reinterpret_cast<const T*>(x), ld,
                          rows, (int)cols, (int)k, reinterpret_cast<T*>(values), indices);
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
