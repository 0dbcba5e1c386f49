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
#include <atomic>

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

// ---------------------------------------------- loss and gradient at once ---
//
// One read of the logits and one write of the gradient: a cluster holds a row
// on chip, 32 elements a thread, as exponentials 2^((z - m_w) c) against the
// warp's own maximum.  Every warp sends its (m_w, sum) to every CTA of the
// cluster (st.async on a transaction barrier: no fence, no second hop through
// a CTA total); each warp then folds all pairs to (M, S) and stores
// w tau e 2^((m_w - M) c) / S.  While a row is exchanged and stored, the next
// ones travel to shared memory through a ring of cp.async copies, each thread
// its own.  A further warp reads the teacher's lists one row ahead, writes the
// tokens of its CTA's slice again once the row is stored, and in CTA 0 the
// loss.
constexpr int kGradList = 256;       // teacher entries a row that this kernel takes
constexpr int kHold = 32;            // elements a thread holds
constexpr int kQuads = 3;            // ring slots of four packs
constexpr int kMaxCluster = 16;
constexpr int kMarkBits = 32768;     // marks of the tokens named so far, by id modulo this

struct GradList {
  int id[kGradList];      // -1: absent
  float t2[kGradList];    // (t - max t) c
  float z[kGradList];     // the logit at id (CTA 0: every entry; else those of its slice)
  float mass[kGradList];  // sum of p over the entries with this id; -1 but at the first of them
};

template <int NT>
struct GradShared {
  uint4 ring[kQuads][4][NT];
  float2 pair[2][kMaxCluster * (NT / 32)];
  GradList list[2];
  uint32_t marks[kMarkBits / 32];
  float2 stat[2];   // (M, S) of the row, for the list's warp
  float by[2];      // w tau
  float total[2];   // of the list's 2^t2; 0: nothing taught
  uint64_t bar[2];
  int lost;
};

// Reads a row's list; one warp.
template <typename T, int NT>
__device__ __forceinline__ void read_list(GradShared<NT>& s, int par, const Taught& a, const T* x,
                                          int64_t row, int cols, int lo, int hi, float by) {
  constexpr int U = 4;  // entries a lane whose loads are in flight together
  GradList& l = s.list[par];
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
  for (int j0 = lane; j0 < a.k; j0 += 32 * U) {
    int64_t id[U];
    float t[U], z[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int j = j0 + 32 * i;
      id[i] = j < a.k ? load_index(a.ids, a.ids_dtype, row * a.ld_ids + j) : -1;
      t[i] = j < a.k ? load_float(a.t, a.t_dtype, row * a.ld_t + j) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) z[i] = id[i] >= lo && id[i] < hi ? Elem<T>::to_f(x[id[i]]) : 0.f;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int j = j0 + 32 * i;
      if (j >= a.k) break;
      const bool in = id[i] >= 0 && id[i] < cols;
      l.id[j] = in ? (int)id[i] : -1;
      l.t2[j] = in ? t[i] : -INFINITY;
      l.z[j] = z[i];
      top = MaxOp::combine(top, l.t2[j]);
    }
  }
  top = group_reduce_warp<MaxOp, 32>(top);
  float total = 0.f;
  if (top != -INFINITY) {
    for (int j = lane; j < a.k; j += 32) {
      l.t2[j] = (l.t2[j] - top) * a.c;
      if (l.id[j] >= 0) total += exp2f(l.t2[j]);
    }
  }
  total = warp_sum(total);
  // masses: an id whose mark was set already may be a repeated one
  __syncwarp();
  for (int j0 = 0; j0 < a.k; j0 += 32) {
    const int j = j0 + lane;
    const int id = j < a.k ? l.id[j] : -1;
    bool again = false;
    if (id >= 0) {
      const uint32_t h = (uint32_t)id % kMarkBits;
      again = (atomicOr(&s.marks[h / 32], 1u << (h % 32)) >> (h % 32)) & 1;
      l.mass[j] = exp2f(l.t2[j]) / total;
    } else if (j < a.k) {
      l.mass[j] = -1.f;
    }
    __syncwarp();
    uint32_t votes = __ballot_sync(0xffffffffu, again);
    while (votes != 0) {
      // the warp goes over the list so far for one such id: its first entry
      // takes the sum of all
      const int same = l.id[j0 + __ffs(votes) - 1];
      votes &= votes - 1;
      const int end = min(a.k, j0 + 32);
      int first = end;
      float mass = 0.f;
      for (int i = lane; i < end; i += 32) {
        if (l.id[i] != same) continue;
        first = min(first, i);
        if (l.mass[i] != -1.f) mass += l.mass[i];
      }
      __syncwarp();
      first = __reduce_min_sync(0xffffffffu, first);
      mass = warp_sum(mass);
      for (int i = lane; i < end; i += 32)
        if (l.id[i] == same) l.mass[i] = i == first ? mass : -1.f;
      __syncwarp();
    }
  }
  for (int j = lane; j < a.k; j += 32)
    if (l.id[j] >= 0) s.marks[(uint32_t)l.id[j] % kMarkBits / 32] = 0;
  if (lane == 0) {
    s.total[par] = total;
    s.by[par] = by;
  }
  __syncwarp();
}

// Warp-wide maximum; NaN only if every lane has one.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

template <typename T, int NT, int MINB>
__global__ void __launch_bounds__(NT + 32, MINB)
distill_grad_kernel(const T* __restrict__ x, int64_t ld, Taught a, const float* __restrict__ weight,
                    int64_t weight_stride, int64_t rows, int cols, float* __restrict__ loss,
                    float2* __restrict__ stats, T* __restrict__ dx, int64_t ld_dx) {
  constexpr int VW = Elem<T>::kVec;
  constexpr int P = kHold / VW;  // packs a thread: 4 of a 16-bit type, 8 of fp32
  constexpr int Q = P / 4;       // ring slots a row
  constexpr int W = NT / 32;
  constexpr int kListed = 1, kStored = 3;  // named barriers, two of each
  extern __shared__ __align__(16) unsigned char smem[];
  GradShared<NT>& s = *reinterpret_cast<GradShared<NT>*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int64_t first = cluster_id(), step = cluster_count();
  for (int i = tid; i < kMarkBits / 32; i += NT + 32) s.marks[i] = 0;
  if (tid == 0) {
    bar_init(&s.bar[0], 1);
    bar_init(&s.bar[1], 1);
    s.lost = 0;
    bar_init_fence();
  }
  pdl_prologue();
  cluster_sync_all();
  // this CTA's packs [from, to) of a row's split
  const auto slice = [&](const RowSplit& sp, int& from, int& to) {
    const int per = (sp.nvec + C - 1) / C;
    from = min(sp.nvec, rank * per);
    to = min(sp.nvec, from + per);
  };
  if (warp == W) {
    // the teacher's lists
    const auto read = [&](int64_t row, int par) {
      if (row >= rows) return;
      const T* xr = x + row * ld;
      const RowSplit sp = split_row(xr, cols);
      int from, to;
      slice(sp, from, to);
      const float w = weight != nullptr ? weight[row * weight_stride] : 1.f;
      read_list<T, NT>(s, par, a, xr, row, cols, rank == 0 ? 0 : sp.head + from * VW,
                       rank == 0 ? cols : sp.head + to * VW, w * a.tau);
      named_arrive(kListed + par, NT + 32);
    };
    read(first, 0);
    int par = 0;
    for (int64_t row = first; row < rows; row += step, par ^= 1) {
      read(row + step, par ^ 1);
      named_sync(kStored + par, NT + 32);
      const GradList& l = s.list[par];
      const float total = s.total[par], by = s.by[par];
      const float2 st = s.stat[par];
      const bool live = total != 0.f;
      if (live) {
        const RowSplit sp = split_row(x + row * ld, cols);
        int from, to;
        slice(sp, from, to);
        const int lo = sp.head + from * VW, hi = sp.head + to * VW;
        T* dr = dx + row * ld_dx;
        for (int j = lane; j < a.k; j += 32) {
          const int id = l.id[j];
          const bool single = id < sp.head || id >= sp.head + sp.nvec * VW;  // CTA 0's
          if (id < 0 || l.mass[j] == -1.f) continue;
          if (single ? rank != 0 : (id < lo || id >= hi)) continue;
          dr[id] = Elem<T>::from_f(by * (ex2((l.z[j] - st.x) * a.c) / st.y - l.mass[j]));
        }
      }
      if (rank == 0) {
        float d = 0.f;
        if (live) {
          for (int j = lane; j < a.k; j += 32) {
            if (l.id[j] < 0) continue;
            const float e = exp2f(l.t2[j]);
            if (e != 0.f) d += e * (l.t2[j] - (l.z[j] - st.x) * a.c);
          }
        }
        d = warp_sum(d);
        if (lane == 0) {
          const float kl = live ? kLn2 * (d / total) + (logf(st.y) - logf(total)) : 0.f;
          loss[row] = a.tau * a.tau * kl;
          stats[row] = live ? st : make_float2(0.f, 0.f);
        }
      }
      __syncwarp();  // the list has been read
    }
  } else {
    const auto issue = [&](int64_t row, int quad, int slot) {
      if (row < rows) {
        const T* xr = x + row * ld;
        const RowSplit sp = split_row(xr, cols);
        int from, to;
        slice(sp, from, to);
        from += quad * 4 * NT + tid;
        const uint4* at = reinterpret_cast<const uint4*>(xr + sp.head) + from;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (from + i * NT < to) cp_async16(&s.ring[slot][i][tid], at + i * NT);
      }
      cp_async_commit();
    };
    int64_t ahead = first;  // the next quad to issue
    int ahead_quad = 0;
    const auto issue_next = [&](int slot) {
      issue(ahead, ahead_quad, slot);
      if (++ahead_quad == Q) {
        ahead_quad = 0;
        ahead += step;
      }
    };
#pragma unroll
    for (int i = 0; i < kQuads; ++i) issue_next(i);
    // where this warp's pairs go: lane r's copy to CTA r
    const uint32_t to_pair = remote_smem(&s.pair[0][rank * W + warp], lane < C ? lane : 0);
    const uint32_t to_bar = remote_smem(&s.bar[0], lane < C ? lane : 0);
    int par = 0, slot = 0;
    uint32_t phase = 0;
    for (int64_t row = first; row < rows; row += step) {
      const T* xr = x + row * ld;
      const RowSplit sp = split_row(xr, cols);
      int from, to;
      slice(sp, from, to);
      const int left = to - from - tid;  // the thread's packs end here
      const bool edge = rank == 0 && warp == 0;  // has the row's single elements
      const int single = edge ? single_of(sp, lane, VW) : -1;
      float xs = single >= 0 ? Elem<T>::to_f(xr[single]) : -INFINITY;
      if (tid == 0) bar_expect(&s.bar[par], C * W * 8);
      float e[P][VW];
      float m = fmaxf(kLowest, xs);
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        cp_async_wait_pending<kQuads - 1>();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 u = s.ring[slot][i][tid];
          unpack<T>(u, e[4 * k + i]);
          if ((4 * k + i) * NT >= left) {
#pragma unroll
            for (int j = 0; j < VW; ++j) e[4 * k + i][j] = -INFINITY;
          }
#pragma unroll
          for (int j = 0; j < VW; j += 2) m = fmax3(m, e[4 * k + i][j], e[4 * k + i][j + 1]);
        }
        issue_next(slot);
        slot = slot + 1 == kQuads ? 0 : slot + 1;
      }
      m = warp_max(m);
      float sum = ex2((xs - m) * a.c);
      xs = sum;
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          e[i][j] = ex2((e[i][j] - m) * a.c);
          sum += e[i][j];
        }
      sum = warp_sum(sum);
      if (lane < C) send_f2(to_pair + par * (uint32_t)sizeof(s.pair[0]), m, sum, to_bar + par * 8);
      named_sync(kListed + par, NT + 32);
      const float by = s.by[par];
      const bool live = s.total[par] != 0.f;
      bar_wait(&s.bar[par], phase, &s.lost);
      float M = kLowest, S = 0.f;
      for (int i = lane; i < C * W; i += 32) M = fmaxf(M, s.pair[par][i].x);
      M = warp_max(M);
      for (int i = lane; i < C * W; i += 32) {
        const float2 q = s.pair[par][i];
        S += q.y * ex2((q.x - M) * a.c);
      }
      S = final_sum(warp_sum(S));
      if (s.lost) S = NAN;
      if (tid == 0) s.stat[par] = make_float2(M, S);
      const float f = live ? ex2((m - M) * a.c) * (by / S) : 0.f;
      T* dr = dx + row * ld_dx;
      uint4* out = reinterpret_cast<uint4*>(dr + sp.head) + from + tid;
      if (single >= 0) dr[single] = Elem<T>::from_f(live ? xs * f : 0.f);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (i * NT < left) {
#pragma unroll
          for (int j = 0; j < VW; ++j) e[i][j] = live ? e[i][j] * f : 0.f;
          st_stream(out + i * NT, pack<T>(e[i]));
        }
      }
      named_arrive(kStored + par, NT + 32);
      phase ^= par;
      par ^= 1;
    }
    cp_async_wait_all();
  }
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while pairs may still be sent to it
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

// Whether two matrices' rows all begin at the same offset from a 16-byte
// boundary, which storing whole packs of one for the other's needs.
bool same_phase(const void* x, int64_t ld, const void* y, int64_t ld_y, int64_t size) {
  return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15u) == 0 &&
         (ld - ld_y) * size % 16 == 0;
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
  const bool vec = dx == nullptr || same_phase(x, ld, dx, ld_dx, sizeof(T));
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

// Clusters of `cluster` CTAs of a kernel that are resident at once, asked for
// once a device; 0 when the kernel cannot run so.
template <typename T, int NT>
int grad_clusters(int cluster, cudaLaunchConfig_t cfg) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][kMaxCluster + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return 0;
  int n = known[dev][cluster].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveClusters(&n, distill_grad_kernel<T, NT, NT == 512 ? 2 : NT == 256 ? 3 : 5>,
                                       &cfg) != cudaSuccess)
      n = 0;
    (void)cudaGetLastError();
    known[dev][cluster].store(n > 0 ? n : -1, std::memory_order_relaxed);
  }
  return n > 0 ? n : 0;
}

// The one-pass kernel; returns -1 where it does not apply.
template <typename T, int NT>
int run_grad(const void* x, int64_t ld, const Taught& a, const float* weight, int64_t weight_stride,
             int64_t rows, int64_t cols, float* loss, float* stats, void* dx, int64_t ld_dx,
             cudaStream_t stream) {
  const auto kern = distill_grad_kernel<T, NT, NT == 512 ? 2 : NT == 256 ? 3 : 5>;
  const int64_t cluster = ceil_div(cols, (int64_t)NT * kHold);
  if (cluster > kMaxCluster || a.k > kGradList) return -1;
  const size_t smem = sizeof(GradShared<NT>);
  // (per launch: the attributes are held per device)
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
      (cluster > 8 &&
       cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)) {
    (void)cudaGetLastError();
    return -1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.blockDim = dim3(NT + 32);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int clusters = grad_clusters<T, NT>((int)cluster, cfg);
  if (clusters == 0) return -1;
  return launch_cluster(kern, std::min<int64_t>(rows, clusters) * cluster, (int)cluster, NT + 32, smem,
                        stream, reinterpret_cast<const T*>(x), ld, a, weight, weight_stride, rows,
                        (int)cols, loss, reinterpret_cast<float2*>(stats), reinterpret_cast<T*>(dx),
                        ld_dx);
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
  int st = check_shapes(rows, cols, k, temperature);
  if (st != FL_B200_OK) return st;
  if (!is_float_dtype(dtype) || !list_dtypes_ok(t_dtype, ids_dtype))
    return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (rows == 0) return FL_B200_OK;
  FLB_CHECK_ARG(logits && loss && stats && (k == 0 || (teacher && ids)));
  FLB_CHECK_ARG((rows == 1 || ld >= cols) && ld_t >= 0 && ld_ids >= 0);
  if (reinterpret_cast<uintptr_t>(stats) % 8) return FL_B200_ERR_MISALIGNED;
  if (same_phase(logits, ld, dlogits, ld_dlogits, dtype_size(dtype))) {
    const Taught a = taught(teacher, ld_t, t_dtype, ids, ld_ids, ids_dtype, k, temperature);
    st = dispatch_float(dtype, [&](auto t) {
      using T = decltype(t);
      const auto go = [&](auto threads) {
        return run_grad<T, decltype(threads)::value>(logits, ld, a, row_weight, weight_stride, rows, cols,
                                                     loss, stats, dlogits, ld_dlogits,
                                                     (cudaStream_t)stream);
      };
      if (cols <= 128 * kHold) return go(std::integral_constant<int, 128>{});
      if (cols <= 256 * kHold) return go(std::integral_constant<int, 256>{});
      return go(std::integral_constant<int, 512>{});
    });
    if (st != -1) return st;
  }
  // rows that no cluster holds, long lists, gradients off the logits' phase
  st = fl_b200_distill_topk_fwd(logits, ld, teacher, ld_t, t_dtype, ids, ld_ids, ids_dtype,
                                          rows, cols, k, temperature, loss, stats, dtype, stream);
  if (st != FL_B200_OK) return st;
  return fl_b200_distill_topk_bwd(row_weight, weight_stride, logits, ld, stats, teacher, ld_t,
                                  t_dtype, ids, ld_ids, ids_dtype, dlogits, ld_dlogits, nullptr,
                                  rows, cols, k, temperature, dtype, stream);
}

}  // extern "C"
