// Helpers of the vocabulary-row kernels (distill.cu, topk.cu, verify.cu):
// rows of any length and alignment split into 16-byte packs, thread-block
// clusters that share one row, and small typed loads.
#pragma once

#include <atomic>

#include "common.cuh"

namespace flb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Rows and indices in them are ints; the kernels add up to 2^17 to one.
constexpr int64_t kMaxCols = 0x7ff00000;
constexpr float kLowest = -3.402823466e+38f;  // running maxima start here, not at -inf:
                                              // x - m stays defined for x = -inf

// 2^x, relative error about 2^-22; results below 2^-126 flush to 0.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A row as `head` single elements, `nvec` 16-byte packs on 16-byte
// boundaries, and `tail` single elements (head, tail < elements per pack).
struct RowSplit {
  int head, nvec, tail;
};
template <typename T>
__device__ __forceinline__ RowSplit split_row(const T* x, int cols) {
  constexpr int VW = Elem<T>::kVec;
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  RowSplit s;
  s.head = min((VW - off) % VW, cols);
  s.nvec = (cols - s.head) / VW;
  s.tail = cols - s.head - s.nvec * VW;
  return s;
}
// The single element of thread `t` (a CTA has at least 16 threads): threads
// 0..7 take the head, 8..15 the tail; -1 where there is none.
__device__ __forceinline__ int single_of(const RowSplit& s, int t, int vw) {
  if (t < s.head) return t;
  if (t >= 8 && t < 8 + s.tail) return s.head + s.nvec * vw + (t - 8);
  return -1;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_id() {
  uint32_t r;
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_count() {
  uint32_t r;
  asm("mov.u32 %0, %%nclusterid.x;" : "=r"(r));
  return r;
}
// Barrier of every thread of the cluster (release / acquire at cluster scope).
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of this CTA's shared object `p` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t remote_smem(const void* p, uint32_t rank) {
  const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 ld_remote_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ int ld_remote_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_remote_s32(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ long long ld_remote_s64(uint32_t addr) {
  long long v;
  asm volatile("ld.shared::cluster.s64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// ---- transaction barriers in shared memory: a CTA's exchange slots ---------
__device__ __forceinline__ void bar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(bar)),
               "r"(count)
               : "memory");
}
// Makes initialised barriers visible to the cluster (followed by a cluster
// barrier).
__device__ __forceinline__ void bar_init_fence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
// One arrival that announces `bytes` to come in this phase.
__device__ __forceinline__ void bar_expect(uint64_t* bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(bar)),
               "r"(bytes)
               : "memory");
}
// Stores (a, b) to `slot` of a CTA of the cluster and counts its 8 bytes on
// that CTA's barrier (both addresses from remote_smem).
__device__ __forceinline__ void send_f2(uint32_t slot, float a, float b, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(
                   slot),
               "f"(a), "f"(b), "r"(bar)
               : "memory");
}
// Counts `bytes` on this CTA's barrier as if they had come.
__device__ __forceinline__ void bar_give(uint64_t* bar, int bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cta.b64 [%0], %1;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Whether the phase of this parity is over: at once, and after a while that
// the hardware sets if it is not.
__device__ __forceinline__ bool bar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{ .reg .pred p; mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; "
      "selp.u32 %0, 1, 0, p; }"
      : "=r"(done)
      : "r"((uint32_t)__cvta_generic_to_shared(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; "
      "selp.u32 %0, 1, 0, p; }"
      : "=r"(done)
      : "r"((uint32_t)__cvta_generic_to_shared(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
// Waits for the phase of this parity, `limit` nanoseconds at most (0: not at
// all) and no longer once *lost is set; a wait takes microseconds.  Whether the
// phase is over.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, const volatile int* lost,
                                         uint32_t limit) {
  if (bar_test(bar, parity)) return true;
  if (limit == 0) return false;
  if (bar_try(bar, parity)) return true;  // (before the clock is read, which takes longer)
  const uint64_t start = nanoseconds();
  while (!*lost && nanoseconds() - start < limit)
    if (bar_try(bar, parity)) return true;
  return false;
}
// Asynchronous bulk copies of 16-byte multiples between 16-byte boundaries:
// global to this CTA's shared memory, counted on its barrier, and back, in
// this thread's bulk groups.
__device__ __forceinline__ void bulk_load(void* smem, const void* gmem, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          (uint32_t)__cvta_generic_to_shared(smem)),
      "l"(gmem), "r"(bytes), "r"((uint32_t)__cvta_generic_to_shared(bar))
      : "memory");
}
__device__ __forceinline__ void bulk_store(void* gmem, const void* smem, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(gmem),
               "r"((uint32_t)__cvta_generic_to_shared(smem)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// Returns once the committed stores have read shared memory / are done.
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// Orders this thread's shared memory accesses before later bulk copies (of
// threads that a barrier puts after it).
__device__ __forceinline__ void bulk_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Named barriers: all `threads` threads meet (sync), or are counted without
// waiting (arrive).
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void named_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Element i of an array whose type is known at run time.
__device__ __forceinline__ float load_float(const void* p, int dtype, int64_t i) {
  if (dtype == FL_B200_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == FL_B200_BF16)
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_float(void* p, int dtype, int64_t i, float v) {
  if (dtype == FL_B200_F32) {
    reinterpret_cast<float*>(p)[i] = v;
  } else if (dtype == FL_B200_BF16) {
    reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  } else {
    reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  }
}
__device__ __forceinline__ int64_t load_index(const void* p, int dtype, int64_t i) {
  return dtype == FL_B200_I64 ? reinterpret_cast<const int64_t*>(p)[i]
                              : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ float warp_sum(float v) { return group_reduce_warp<SumOp, 32>(v); }

// Lets `kern` use `smem` bytes of dynamic shared memory, and clusters of more
// than 8 CTAs where `wide`; asked for once a kernel and device (`done`, a
// static of the caller's).
template <typename K>
inline bool allow_smem(K kern, size_t smem, bool wide, std::atomic<int> (&done)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  const int want = wide ? 2 : 1;
  if (done[dev].load(std::memory_order_acquire) >= want) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
      (wide && cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)) {
    set_last_cuda_error(cudaGetLastError());
    return false;
  }
  done[dev].store(want, std::memory_order_release);
  return true;
}

// Launches `kern` with `ctas` CTAs in clusters of `cluster`.
template <typename... KArgs, typename... Args>
inline int launch_cluster(void (*kern)(KArgs...), int64_t ctas, int cluster, int block, size_t smem,
                          cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  (void)cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
  return launch_status();
}

}  // namespace
}  // namespace flb200
