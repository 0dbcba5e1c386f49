// Distillation from a teacher's top logits: the loss, its gradients, and both
// in one call.
//
// A row holds the student's logits z[0..V), the teacher's list of k logits t
// and their token ids; entries whose id lies outside [0, V) are absent.  With
// temperature tau,
//   p_j  = softmax over the list's present entries of t / tau,
//   q    = softmax(z / tau) over the whole row,
//   loss = tau^2 * KL = tau^2 * sum_j p_j (log p_j - log q[id_j]),
//   dz_v = w tau (q_v - sum over id_j = v of p_j),
//   dt_j = w tau p_j (log p_j - log q[id_j] - KL)
// for a row weight w.  A row whose list is empty has loss 0 and zero
// gradients whatever its logits hold.  An id may repeat: its entries add.
//
// All sums and statistics are fp32, over differences from the row's maximum:
// exp((x - m) log2e / tau) is 2^((x - m) c), so a row at the type's lowest
// value comes out uniform and -inf entries have q = 0.  The forward stores
// (m, S = sum 2^((z - m) c)) a row, S = 0 for a row without a list; the
// backward multiplies by 1 / S what it exponentiates against the same m, so
// the two agree to the rounding of the exponential itself.
#include "vocab_rows.cuh"

namespace flb200 {
namespace {

constexpr int kMaxList = 1024;      // teacher entries a row
constexpr int kStream = 512;        // threads that walk the row
constexpr int kBlock = kStream + 32;  // and one warp for the teacher's list
constexpr int kUnroll = 4;

struct Taught {
  const void* t;
  int64_t ld_t;
  const void* ids;
  int64_t ld_ids;
  int t_dtype, ids_dtype;
  int k;
  float c;    // log2(e) / tau
  float tau;
};

// The teacher's list of one row in shared memory.
struct List {
  int id[kMaxList];     // -1: absent
  float t2[kMaxList];   // (t - max t) c; p_j = 2^t2 / total
  float z[kMaxList];    // the student's logit at id
  float total;          // sum 2^t2, 0 when the list is empty
};

// Read by the 32 lanes of one warp.  NaN among the teacher's logits makes
// every p NaN; a list of -inf alone counts as empty.
template <typename T>
__device__ __forceinline__ void load_list(List& s, const Taught& a, const T* x, int64_t row, int cols,
                                          bool want_z) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
  for (int j = lane; j < a.k; j += 32) {
    const int64_t id = load_index(a.ids, a.ids_dtype, row * a.ld_ids + j);
    const bool in = id >= 0 && id < cols;
    const float t = in ? load_float(a.t, a.t_dtype, row * a.ld_t + j) : -INFINITY;
    s.id[j] = in ? (int)id : -1;
    s.t2[j] = t;
    if (want_z) s.z[j] = in ? Elem<T>::to_f(x[id]) : 0.f;
    top = MaxOp::combine(top, t);
  }
  top = group_reduce_warp<MaxOp, 32>(top);
  float total = 0.f;
  if (top != -INFINITY) {
    for (int j = lane; j < a.k; j += 32) {
      const float t2 = (s.t2[j] - top) * a.c;
      s.t2[j] = t2;
      if (s.id[j] >= 0) total += exp2f(t2);
    }
  }
  total = warp_sum(total);
  if (lane == 0) s.total = total;
  __syncwarp();
}

// KL of the row in nats, in every lane of the warp that loaded the list.
__device__ __forceinline__ float list_kl(const List& s, const Taught& a, float m, float sum) {
  const int lane = threadIdx.x & 31;
  float d = 0.f;
  for (int j = lane; j < a.k; j += 32) {
    if (s.id[j] < 0) continue;
    const float e = exp2f(s.t2[j]);
    if (e != 0.f) d += e * (s.t2[j] - (s.z[j] - m) * a.c);
  }
  d = warp_sum(d);
  return kLn2 * (d / s.total) + (logf(sum) - logf(s.total));
}

// Running maximum and sum of 2^((x - m) c).
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * ex2((a.m - m) * c) + b.s * ex2((b.m - m) * c)};
}
__device__ __forceinline__ MaxSum warp_merge(MaxSum v, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const MaxSum w = {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o)};
    v = merge(v, w, c);
  }
  return v;
}

// Folds N values into v.
template <int N>
__device__ __forceinline__ void fold(MaxSum& v, const float (&f)[N], float c) {
  float top = f[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, f[i]);
  if (top > v.m) {
    v.s *= ex2((v.m - top) * c);
    v.m = top;
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s += ex2((f[i] - v.m) * c);
  v.s += s;
}

// A row's statistics are final once S is not 0: a row of -inf alone, whose
// softmax is undefined, has S = NaN so that it is not taken for a row
// without a list.
__device__ __forceinline__ float final_sum(float s) { return s == 0.f ? NAN : s; }

// Loss and statistics.  One CTA a row, or a cluster of CTAs with a slice of
// packs each when there are few rows.
template <typename T>
__global__ void __launch_bounds__(kBlock, 2)
distill_fwd_kernel(const T* __restrict__ x, int64_t ld, Taught a, int cols,
                   float* __restrict__ loss, float2* __restrict__ stats) {
  constexpr int VW = Elem<T>::kVec;
  __shared__ List list;
  __shared__ float2 part[kStream / 32];
  __shared__ float2 mine;
  pdl_prologue();
  const uint32_t rank = cluster_rank(), C = cluster_size();
  const int64_t row = cluster_id();
  const T* xr = x + row * ld;
  const int tid = threadIdx.x;
  if (tid >= kStream) {
    if (rank == 0) load_list(list, a, xr, row, cols, true);
  } else {
    const RowSplit sp = split_row(xr, cols);
    const uint4* body = reinterpret_cast<const uint4*>(xr + sp.head);
    const int per = (sp.nvec + (int)C - 1) / (int)C;
    const int end = min(sp.nvec, (int)(rank + 1) * per);
    MaxSum v = {kLowest, 0.f};
    if (rank == 0) {
      const int e = single_of(sp, tid, VW);
      if (e >= 0) {
        const float f[1] = {Elem<T>::to_f(xr[e])};
        fold<1>(v, f, a.c);
      }
    }
    int p = (int)rank * per + tid;
    for (; p + (kUnroll - 1) * kStream < end; p += kUnroll * kStream) {
      uint4 u[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) u[i] = ld_stream(body + p + i * kStream);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        float f[VW];
        unpack<T>(u[i], f);
        fold<VW>(v, f, a.c);
      }
    }
    for (; p < end; p += kStream) {
      float f[VW];
      unpack<T>(ld_stream(body + p), f);
      fold<VW>(v, f, a.c);
    }
    v = warp_merge(v, a.c);
    if ((tid & 31) == 0) part[tid >> 5] = make_float2(v.m, v.s);
  }
  __syncthreads();
  if (tid >= kStream) {
    const int lane = tid & 31;
    const float2 q = lane < kStream / 32 ? part[lane] : make_float2(kLowest, 0.f);
    MaxSum v = warp_merge({q.x, q.y}, a.c);
    if (lane == 0) mine = make_float2(v.m, v.s);
  }
  if (C > 1) cluster_sync_all();
  if (tid >= kStream && rank == 0) {
    const int lane = tid & 31;
    __syncwarp();
    float2 q = make_float2(kLowest, 0.f);
    if (lane < (int)C) q = C > 1 ? ld_remote_f2(remote_smem(&mine, lane)) : mine;
    const MaxSum v = warp_merge({q.x, q.y}, a.c);
    const bool live = list.total != 0.f;
    const float sum = final_sum(v.s);
    const float kl = live ? list_kl(list, a, v.m, sum) : 0.f;
    if (lane == 0) {
      loss[row] = a.tau * a.tau * kl;
      stats[row] = live ? make_float2(v.m, sum) : make_float2(0.f, 0.f);
    }
  }
  if (C > 1) cluster_sync_all();  // no CTA leaves while rank 0 may read its pair
}

// sum of p over the entries of the list that name entry j's token, and
// whether j is the first of them (which writes the token's gradient).
__device__ __forceinline__ bool token_mass(const List& s, int k, int j, float& mass) {
  const int id = s.id[j];
  float m = 0.f;
  for (int i = 0; i < k; ++i) {
    if (s.id[i] != id) continue;
    if (i < j) return false;
    m += exp2f(s.t2[i]);
  }
  mass = m / s.total;
  return true;
}

// Gradients of both operands from the forward's statistics: q w tau streamed
// over a chunk of the row, then the tokens of the teacher's list that lie in
// it written again, whole, from fp32.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kBlock, 2)
distill_bwd_kernel(const float* __restrict__ dloss, int64_t dloss_stride, const T* __restrict__ x,
                   int64_t ld, const float2* __restrict__ stats, Taught a, int cols, int chunk,
                   int chunks, T* __restrict__ dx, int64_t ld_dx, void* __restrict__ dt) {
  constexpr int VW = Elem<T>::kVec;
  __shared__ List list;
  pdl_prologue();
  const int64_t row = blockIdx.x / (unsigned)chunks;
  const int part = (int)(blockIdx.x % (unsigned)chunks);
  const T* xr = x + row * ld;
  const int tid = threadIdx.x;
  const float2 st = stats[row];
  const bool live = st.y != 0.f;
  const float gt = (dloss != nullptr ? dloss[row * dloss_stride] : 1.f) * a.tau;
  const float f = gt / st.y;
  const int from = part * chunk, to = min(cols, from + chunk);  // elements
  if (tid >= kStream) {
    if (live) {
      const bool want = dt != nullptr && part == 0;
      load_list(list, a, xr, row, cols, want);
      if (want) {
        const float kl = list_kl(list, a, st.x, st.y);
        const float lse = logf(st.y), lt = logf(list.total);
        for (int j = tid & 31; j < a.k; j += 32) {
          float g = 0.f;
          if (list.id[j] >= 0) {
            const float e = exp2f(list.t2[j]);
            if (e != 0.f) {
              const float gap = kLn2 * (list.t2[j] - (list.z[j] - st.x) * a.c) + (lse - lt);
              g = gt * (e / list.total) * (gap - kl);
            }
          }
          store_float(dt, a.t_dtype, row * a.k + j, g);
        }
      }
    } else if (dt != nullptr && part == 0) {
      for (int j = tid & 31; j < a.k; j += 32) store_float(dt, a.t_dtype, row * a.k + j, 0.f);
    }
  } else if (dx != nullptr) {
    T* dr = dx + row * ld_dx;
    const auto grad = [&](float z) { return live ? ex2((z - st.x) * a.c) * f : 0.f; };
    if constexpr (VEC) {
      const RowSplit sp = split_row(xr, cols);
      const uint4* body = reinterpret_cast<const uint4*>(xr + sp.head);
      uint4* out = reinterpret_cast<uint4*>(dr + sp.head);
      // pack p belongs to the chunk that holds element p * VW
      const int p1 = part == chunks - 1 ? sp.nvec : min(sp.nvec, to / VW);
      if (part == 0) {
        const int e = single_of(sp, tid, VW);
        if (e >= 0) dr[e] = Elem<T>::from_f(live ? grad(Elem<T>::to_f(xr[e])) : 0.f);
      }
      for (int p = from / VW + tid; p < p1; p += kUnroll * kStream) {
        uint4 u[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
          if (live && p + i * kStream < p1) u[i] = ld_stream(body + p + i * kStream);
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
          if (p + i * kStream >= p1) break;
          float v[VW];
          if (live) unpack<T>(u[i], v);
#pragma unroll
          for (int j = 0; j < VW; ++j) v[j] = grad(v[j]);
          st_stream(out + p + i * kStream, pack<T>(v));
        }
      }
    } else {
      for (int e = from + tid; e < to; e += kStream)
        dr[e] = Elem<T>::from_f(live ? grad(Elem<T>::to_f(xr[e])) : 0.f);
    }
  }
  if (!live || dx == nullptr) return;  // (the whole CTA)
  __syncthreads();
  // chunk 0 writes the row's single elements, the others only whole packs;
  // here every chunk takes the tokens whose element it wrote
  int first = from, last = to;
  int single_lo = 0, single_hi = 0;  // [0, single_lo) and [single_hi, cols) belong to chunk 0
  if constexpr (VEC) {
    const RowSplit sp = split_row(xr, cols);
    const int p1 = part == chunks - 1 ? sp.nvec : min(sp.nvec, to / VW);
    first = sp.head + from / VW * VW;
    last = sp.head + p1 * VW;
    single_lo = sp.head;
    single_hi = sp.head + sp.nvec * VW;
  }
  T* dr = dx + row * ld_dx;
  for (int j = tid; j < a.k; j += kBlock) {
    const int id = list.id[j];
    if (id < 0) continue;
    bool here = id >= first && id < last;
    if constexpr (VEC) here = (id < single_lo || id >= single_hi) ? part == 0 : here;
    float mass;
    if (!here || !token_mass(list, a.k, j, mass)) continue;
    const float q = ex2((Elem<T>::to_f(xr[id]) - st.x) * a.c) / st.y;
    dr[id] = Elem<T>::from_f(gt * (q - mass));
  }
}

// ------------------------------------------------------------------ host ---

bool list_dtypes_ok(int t_dtype, int ids_dtype) {
  return is_float_dtype(t_dtype) && (ids_dtype == FL_B200_I32 || ids_dtype == FL_B200_I64);
}

int check_shapes(int64_t rows, int64_t cols, int64_t k, float temperature) {
  FLB_CHECK_ARG(rows >= 0 && cols >= 0 && k >= 0);
  FLB_CHECK_ARG(temperature > 0.f && temperature <= 3.0e38f);
  if (k > kMaxList || cols > 0x7fffff00LL || rows > 0x7fffffffLL) return FL_B200_ERR_TOO_LARGE;
  FLB_CHECK_ARG(rows == 0 || cols > 0);
  return FL_B200_OK;
}

Taught taught(const void* t, int64_t ld_t, int t_dtype, const void* ids, int64_t ld_ids,
              int ids_dtype, int64_t k, float temperature) {
  return {t, ld_t, ids, ld_ids, t_dtype, ids_dtype, (int)k, kLog2e / temperature, temperature};
}

template <typename T>
int run_fwd(const void* x, int64_t ld, const Taught& a, int64_t rows, int64_t cols, float* loss,
            float* stats, cudaStream_t stream) {
  DeviceInfo dev;
  const int st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  int cluster = 1;
  while (cluster < 8 && rows * cluster < 2 * dev.sm_count &&
         cols / (cluster * 2) >= kStream * Elem<T>::kVec)
    cluster *= 2;
  return launch_cluster(distill_fwd_kernel<T>, rows * cluster, cluster, kBlock, 0, stream,
                        reinterpret_cast<const T*>(x), ld, a, (int)cols, loss,
                        reinterpret_cast<float2*>(stats));
}

template <typename T>
int run_bwd(const float* dloss, int64_t dloss_stride, const void* x, int64_t ld, const float* stats,
            const Taught& a, int64_t rows, int64_t cols, void* dx, int64_t ld_dx, void* dt,
            cudaStream_t stream) {
  // a vector store needs the gradient's rows on the logits' 16-byte phase
  const auto phase = [](const void* p) { return reinterpret_cast<uintptr_t>(p) & 15u; };
  const bool vec = dx == nullptr || (phase(x) == phase(dx) && ((ld - ld_dx) * (int64_t)sizeof(T)) % 16 == 0);
  int chunks = 1;
  int64_t chunk = cols;
  if (dx != nullptr) {
    chunk = (int64_t)kStream * kUnroll * Elem<T>::kVec;
    chunks = (int)ceil_div(cols, chunk);
  }
  if (rows * chunks > 0x7fffffffLL) return FL_B200_ERR_TOO_LARGE;
  const auto go = [&](auto kern) {
    launch_k(kern, dim3((unsigned)(rows * chunks)), dim3(kBlock), 0, stream, dloss, dloss_stride,
             reinterpret_cast<const T*>(x), ld, reinterpret_cast<const float2*>(stats), a, (int)cols,
             (int)chunk, chunks, reinterpret_cast<T*>(dx), ld_dx, dt);
    return launch_status();
  };
  return vec ? go(distill_bwd_kernel<T, true>) : go(distill_bwd_kernel<T, false>);
}

}  // namespace
}  // namespace flb200

extern "C" {

FL_B200_API int fl_b200_distill_topk_fwd(const void* logits, int64_t ld, const void* teacher,
                                         int64_t ld_t, int t_dtype, const void* ids, int64_t ld_ids,
                                         int ids_dtype, int64_t rows, int64_t cols, int64_t k,
                                         float temperature, float* loss, float* stats, int dtype,
                                         fl_b200_stream_t stream) {
  using namespace flb200;
  const int st = check_shapes(rows, cols, k, temperature);
  if (st != FL_B200_OK) return st;
  if (!is_float_dtype(dtype) || !list_dtypes_ok(t_dtype, ids_dtype))
    return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (rows == 0) return FL_B200_OK;
  FLB_CHECK_ARG(logits && loss && stats && (k == 0 || (teacher && ids)));
  FLB_CHECK_ARG((rows == 1 || ld >= cols) && ld_t >= 0 && ld_ids >= 0);
  if (reinterpret_cast<uintptr_t>(stats) % 8) return FL_B200_ERR_MISALIGNED;
  const Taught a = taught(teacher, ld_t, t_dtype, ids, ld_ids, ids_dtype, k, temperature);
  return dispatch_float(dtype, [&](auto t) {
    return run_fwd<decltype(t)>(logits, ld, a, rows, cols, loss, stats, (cudaStream_t)stream);
  });
}

FL_B200_API int fl_b200_distill_topk_bwd(const float* dloss, int64_t dloss_stride,
                                         const void* logits, int64_t ld, const float* stats,
                                         const void* teacher, int64_t ld_t, int t_dtype,
                                         const void* ids, int64_t ld_ids, int ids_dtype,
                                         void* dlogits, int64_t ld_dlogits, void* dteacher,
                                         int64_t rows, int64_t cols, int64_t k, float temperature,
                                         int dtype, fl_b200_stream_t stream) {
  using namespace flb200;
  const int st = check_shapes(rows, cols, k, temperature);
  if (st != FL_B200_OK) return st;
  if (!is_float_dtype(dtype) || !list_dtypes_ok(t_dtype, ids_dtype))
    return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (rows == 0 || (dlogits == nullptr && dteacher == nullptr)) return FL_B200_OK;
  FLB_CHECK_ARG(dloss_stride >= 0 && logits && stats && (k == 0 || (teacher && ids)));
  FLB_CHECK_ARG((rows == 1 || ld >= cols) && ld_t >= 0 && ld_ids >= 0);
  FLB_CHECK_ARG(dlogits == nullptr || rows == 1 || ld_dlogits >= cols);
  if (reinterpret_cast<uintptr_t>(stats) % 8) return FL_B200_ERR_MISALIGNED;
  const Taught a = taught(teacher, ld_t, t_dtype, ids, ld_ids, ids_dtype, k, temperature);
  return dispatch_float(dtype, [&](auto t) {
    return run_bwd<decltype(t)>(dloss, dloss_stride, logits, ld, stats, a, rows, cols, dlogits,
                                ld_dlogits, dteacher, (cudaStream_t)stream);
  });
}

FL_B200_API int fl_b200_distill_topk_grad(const void* logits, int64_t ld, const void* teacher,
                                          int64_t ld_t, int t_dtype, const void* ids,
                                          int64_t ld_ids, int ids_dtype, const float* row_weight,
                                          int64_t weight_stride, int64_t rows, int64_t cols,
                                          int64_t k, float temperature, float* loss, float* stats,
                                          void* dlogits, int64_t ld_dlogits, int dtype,
                                          fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(rows <= 0 || (dlogits && (rows == 1 || ld_dlogits >= cols)));
  FLB_CHECK_ARG(weight_stride >= 0);
  const int st = fl_b200_distill_topk_fwd(logits, ld, teacher, ld_t, t_dtype, ids, ld_ids, ids_dtype,
                                          rows, cols, k, temperature, loss, stats, dtype, stream);
  if (st != FL_B200_OK) return st;
  return fl_b200_distill_topk_bwd(row_weight, weight_stride, logits, ld, stats, teacher, ld_t,
                                  t_dtype, ids, ld_ids, ids_dtype, dlogits, ld_dlogits, nullptr,
                                  rows, cols, k, temperature, dtype, stream);
}

}  // extern "C"
