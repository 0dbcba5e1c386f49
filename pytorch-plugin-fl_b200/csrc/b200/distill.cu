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
constexpr int kUnroll = 4;          // packs a thread loads before it uses one

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
  constexpr int U = 4;  // entries a lane whose loads are in flight together
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
  for (int j0 = lane; j0 < a.k; j0 += 32 * U) {
    int64_t id[U];
    float t[U];
    T z[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int j = min(j0 + 32 * i, a.k - 1);
      id[i] = load_index(a.ids, a.ids_dtype, row * a.ld_ids + j);
      t[i] = load_float(a.t, a.t_dtype, row * a.ld_t + j);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (id[i] < 0 || id[i] >= cols) id[i] = -1;
      z[i] = x[want_z && id[i] >= 0 ? id[i] : 0];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int j = j0 + 32 * i;
      if (j >= a.k) break;
      s.id[j] = (int)id[i];
      s.t2[j] = id[i] >= 0 ? t[i] : -INFINITY;
      s.z[j] = Elem<T>::to_f(z[i]);
      top = MaxOp::combine(top, s.t2[j]);
    }
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

// Folds one value into v.
__device__ __forceinline__ void fold(MaxSum& v, float f, float c) {
  const float m = fmaxf(v.m, f);
  v = {m, v.s * ex2((v.m - m) * c) + ex2((f - m) * c)};
}

// A row's statistics are final once S is not 0: a row of -inf alone, whose
// softmax is undefined, has S = NaN so that it is not taken for a row
// without a list.
__device__ __forceinline__ float final_sum(float s) { return s == 0.f ? NAN : s; }

constexpr int kGradList = 128;  // the longest list that a warp holds in registers
constexpr int kMarkBits = 16384;  // marks of the tokens named so far, by id modulo this

// Warp-wide maximum; NaN only if every lane has one.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The same, NaN if any lane has one.
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// An element's bits in a register of their own (a 16-bit register that a load
// fills is copied at once, which waits for the load).
template <typename T>
__device__ __forceinline__ uint32_t load_bits(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return __float_as_uint(*p);
  } else {
    return *reinterpret_cast<const unsigned short*>(p);
  }
}
template <typename T>
__device__ __forceinline__ float bits_value(uint32_t b) {
  if constexpr (std::is_same<T, float>::value) {
    return __uint_as_float(b);
  } else if constexpr (std::is_same<T, __half>::value) {
    return __half2float(__ushort_as_half((unsigned short)b));
  } else {
    return __uint_as_float(b << 16);
  }
}

// A row's list on its way, E entries a lane, as loaded: a value
// that is not touched until the next row's turn does not hold the warp up.
// (For the same reason the loads are not conditional: lanes past the list
// load its last entry.)
template <int E>
struct ListAhead {
  static constexpr int kEach = E;
  long long id[kEach];
  uint32_t t[kEach];
  float w;

  __device__ __forceinline__ void load(const Taught& a, const float* weight, int64_t weight_stride,
                                       int64_t row) {
    const int lane = threadIdx.x & 31;
    w = 1.f;
    if (weight != nullptr) w = weight[row * weight_stride];
    const int64_t at = row * a.ld_ids, at_t = row * a.ld_t;
    const auto each = [&](auto take) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (32 * i >= a.k) break;
        take(i, min(lane + 32 * i, a.k - 1));
      }
    };
    if (a.ids_dtype == FL_B200_I64) {
      const long long* p = reinterpret_cast<const long long*>(a.ids) + at;
      each([&](int i, int j) { id[i] = p[j]; });
    } else {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(a.ids) + at;
      each([&](int i, int j) { id[i] = p[j]; });  // (zero-extended: negative ones end up past V)
    }
    if (a.t_dtype == FL_B200_F32) {
      const float* p = reinterpret_cast<const float*>(a.t) + at_t;
      each([&](int i, int j) { t[i] = load_bits(p + j); });
    } else {
      const __half* p = reinterpret_cast<const __half*>(a.t) + at_t;
      each([&](int i, int j) { t[i] = load_bits(p + j); });
    }
  }
  __device__ __forceinline__ int token(int i, int k, int cols) const {  // -1: absent
    const bool in = (int)(threadIdx.x & 31) + 32 * i < k && (unsigned long long)id[i] < (unsigned)cols;
    return in ? (int)id[i] : -1;
  }
  __device__ __forceinline__ float logit(int i, int dtype) const {
    if (dtype == FL_B200_F32) return bits_value<float>(t[i]);
    return dtype == FL_B200_BF16 ? bits_value<__nv_bfloat16>(t[i]) : bits_value<__half>(t[i]);
  }
};

// 1 / x within an ulp (x a sum of exponentials: normal, or NaN).
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A row's list in hand, spread over a warp as ListAhead is.  (Registers and
// unrolled loops: what this warp does between a row's sums and its scale holds
// up all the others, and a loop over shared memory took ten times as long.)
template <typename T, int E>
struct ListHeld {
  static constexpr int kEach = E;
  int id[kEach];      // -1: absent
  uint32_t z[kEach];  // the logit's bits, of entries in [lo, hi)
  float t2[kEach];    // (t - max t) c
  float e[kEach];     // 2^t2, 0 where absent
  float mass[kEach];  // sum of p over the entries with this id; -1 but at the first of them
  float total;        // of e; 0 when nothing is taught
  float by;           // w tau

  // Everything but the masses.
  __device__ __forceinline__ void set(const Taught& a, const ListAhead<E>& in, const T* x, int cols, int lo,
                                      int hi) {
    by = in.w * a.tau;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (32 * i >= a.k) break;
      id[i] = in.token(i, a.k, cols);
      z[i] = load_bits(x + (id[i] >= lo && id[i] < hi ? id[i] : 0));  // (used once the row is summed)
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (32 * i >= a.k) break;
      t2[i] = id[i] >= 0 ? in.logit(i, a.t_dtype) : -INFINITY;
      top = MaxOp::combine(top, t2[i]);
    }
    top = warp_max_nan(top);
    total = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (32 * i >= a.k) break;
      t2[i] = (t2[i] - top) * a.c;
      e[i] = id[i] >= 0 && top != -INFINITY ? ex2(t2[i]) : 0.f;
      total += e[i];
    }
    total = warp_sum(total);
  }

  __device__ __forceinline__ void set_masses(const Taught& a, uint32_t* marks) {
    const int lane = threadIdx.x & 31;
    const float inverse = reciprocal(total);
    // an id whose mark was set already may be a repeated one
    uint32_t again = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (32 * i >= a.k) break;
      mass[i] = id[i] >= 0 ? e[i] * inverse : -1.f;
      if (id[i] >= 0) {
        const uint32_t h = (uint32_t)id[i] % kMarkBits;
        again |= ((atomicOr(&marks[h / 32], 1u << (h % 32)) >> (h % 32)) & 1) << i;
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (32 * i >= a.k) break;
      if (id[i] >= 0) marks[(uint32_t)id[i] % kMarkBits / 32] = 0;
    }
    // each id under suspicion against the whole list: its first entry takes
    // the sum of all
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (32 * i >= a.k) break;
      uint32_t votes = __ballot_sync(0xffffffffu, (again >> i) & 1);
      while (votes != 0) {
        const int same = __shfl_sync(0xffffffffu, id[i], __ffs(votes) - 1);
        votes &= votes - 1;
        int first = kGradList, count = 0;
        float sum = 0.f;
#pragma unroll
        for (int n = kEach - 1; n >= 0; --n) {
          if (32 * n >= a.k || id[n] != same) continue;
          first = lane + 32 * n;
          ++count;
          if (mass[n] != -1.f) sum += mass[n];
        }
        if (__reduce_add_sync(0xffffffffu, count) == 1) continue;  // another id with its mark
        first = __reduce_min_sync(0xffffffffu, first);
        sum = warp_sum(sum);
#pragma unroll
        for (int n = 0; n < kEach; ++n)
          if (32 * n < a.k && id[n] == same) mass[n] = lane + 32 * n == first ? sum : -1.f;
      }
    }
    __syncwarp();
  }
};

// Maximum of a pack's elements (NaN ignored unless all are).
template <typename T>
__device__ __forceinline__ float pack_max(const uint4& u) {
  if constexpr (std::is_same<T, float>::value) {
    return fmaxf(fmax3(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z)),
                 __uint_as_float(u.w));
  } else {
    uint32_t a, b, c;
    if constexpr (std::is_same<T, __half>::value) {
      asm("max.f16x2 %0, %1, %2;" : "=r"(a) : "r"(u.x), "r"(u.y));
      asm("max.f16x2 %0, %1, %2;" : "=r"(b) : "r"(u.z), "r"(u.w));
      asm("max.f16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    } else {
      asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(u.x), "r"(u.y));
      asm("max.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(u.z), "r"(u.w));
      asm("max.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    }
    const uint64_t p = pair_from_bits<T>(c);
    return fmaxf(f2_lo(p), f2_hi(p));
  }
}
// A word of -infinities.
template <typename T>
__device__ __forceinline__ constexpr uint32_t lowest_word() {
  return std::is_same<T, float>::value ? 0xff800000u
         : std::is_same<T, __half>::value ? 0xfc00fc00u
                                          : 0xff80ff80u;
}
// A pack as fp32 pairs, and pairs times f rounded to a pack.
template <typename T>
__device__ __forceinline__ void to_pairs(const uint4& u, uint64_t (&e)[Elem<T>::kVec / 2]) {
  if constexpr (std::is_same<T, float>::value) {
    e[0] = f2_make(__uint_as_float(u.x), __uint_as_float(u.y));
    e[1] = f2_make(__uint_as_float(u.z), __uint_as_float(u.w));
  } else {
    e[0] = pair_from_bits<T>(u.x);
    e[1] = pair_from_bits<T>(u.y);
    e[2] = pair_from_bits<T>(u.z);
    e[3] = pair_from_bits<T>(u.w);
  }
}
template <typename T>
__device__ __forceinline__ uint4 from_pairs(const uint64_t (&e)[Elem<T>::kVec / 2], uint64_t f) {
  if constexpr (std::is_same<T, float>::value) {
    const uint64_t a = f2_mul(e[0], f), b = f2_mul(e[1], f);
    return make_uint4(__float_as_uint(f2_lo(a)), __float_as_uint(f2_hi(a)), __float_as_uint(f2_lo(b)),
                      __float_as_uint(f2_hi(b)));
  } else {
    return make_uint4(pair_to_bits<T>(f2_mul(e[0], f)), pair_to_bits<T>(f2_mul(e[1], f)),
                      pair_to_bits<T>(f2_mul(e[2], f)), pair_to_bits<T>(f2_mul(e[3], f)));
  }
}

// Folds N packs into v, the exponentials in fp32 pairs.
template <typename T, int N>
__device__ __forceinline__ void fold_packs(MaxSum& v, const uint4 (&u)[N], float c) {
  constexpr int VW = Elem<T>::kVec;
  float top = pack_max<T>(u[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, pack_max<T>(u[i]));
  if (top > v.m) {
    v.s *= ex2((v.m - top) * c);
    v.m = top;
  }
  const uint64_t minus = f2_make(-v.m, -v.m), c2 = f2_make(c, c);
  uint64_t sum = 0;  // (two zeros)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint64_t e[VW / 2];
    to_pairs<T>(u[i], e);
#pragma unroll
    for (int j = 0; j < VW / 2; ++j) {
      const uint64_t d = f2_mul(f2_add(e[j], minus), c2);
      sum = f2_add(sum, f2_make(ex2(f2_lo(d)), ex2(f2_hi(d))));
    }
  }
  v.s += f2_lo(sum) + f2_hi(sum);
}

// A row's list as the two-kernel path uses it: held by the last warp of the
// CTA, E entries a lane, or in shared memory (E = 0: any length up to
// kMaxList).
template <typename T, int E>
struct ListOf {
  struct Shared {
    uint32_t marks[kMarkBits / 32];
  };
  ListHeld<T, E> held;
  float total;

  __device__ __forceinline__ void load(Shared& s, const Taught& a, const float*, int64_t, const T* x,
                                       int64_t row, int cols, int lo, int hi, bool masses) {
    ListAhead<E> in;
    in.load(a, nullptr, 0, row);
    if (!masses) {
      held.set(a, in, x, cols, lo, hi);
      total = held.total;
      return;
    }
    for (int i = threadIdx.x & 31; i < kMarkBits / 32; i += 32) s.marks[i] = 0;
    __syncwarp();
    held.set(a, in, x, cols, lo, hi);
    held.set_masses(a, s.marks);
    total = held.total;
  }
  // sum of p_j ((t_j - max t) - (z_j - m)) / tau, by the warp
  __device__ __forceinline__ float kl(Shared&, const Taught& a, float m, float sum) const {
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (32 * i >= a.k) break;
      if (held.id[i] >= 0 && held.e[i] != 0.f)
        d += held.e[i] * (held.t2[i] - (bits_value<T>(held.z[i]) - m) * a.c);
    }
    d = warp_sum(d);
    return kLn2 * (d / total) + (logf(sum) - logf(total));
  }
  __device__ __forceinline__ void teacher(Shared& s, const Taught& a, float m, float sum, float gt,
                                          void* dt, int64_t row) const {
    const float all = kl(s, a, m, sum), logs = logf(sum) - logf(total);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (int)(threadIdx.x & 31) + 32 * i;
      if (j >= a.k) break;
      float g = 0.f;
      if (held.id[i] >= 0 && held.e[i] != 0.f) {
        const float gap = kLn2 * (held.t2[i] - (bits_value<T>(held.z[i]) - m) * a.c) + logs;
        g = gt * (held.e[i] / total) * (gap - all);
      }
      store_float(dt, a.t_dtype, row * a.k + j, g);
    }
  }
  // Calls put(id, z, mass) once for every token of the list, by the warp.
  template <typename F>
  __device__ __forceinline__ void tokens(Shared&, const Taught& a, const T*, int warp_from, F put) const {
    if ((int)threadIdx.x < warp_from) return;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (32 * i >= a.k) break;
      if (held.id[i] >= 0 && held.mass[i] != -1.f)
        put(held.id[i], bits_value<T>(held.z[i]), held.mass[i]);
    }
  }
};

template <typename T>
struct ListOf<T, 0> {
  static constexpr int kMarks = 65536;
  struct Shared : List {
    float mass[kMaxList];  // sum of p over the entries with this id; -1 but at the first of them
    uint32_t marks[kMarks / 32];
    short suspect[kMaxList];
    int suspects;
  };
  float total;

  __device__ __forceinline__ void load(Shared& s, const Taught& a, const float*, int64_t, const T* x,
                                       int64_t row, int cols, int, int, bool) {
    load_list(s, a, x, row, cols, true);
    total = s.total;
  }
  __device__ __forceinline__ float kl(Shared& s, const Taught& a, float m, float sum) const {
    return list_kl(s, a, m, sum);
  }
  __device__ __forceinline__ void teacher(Shared& s, const Taught& a, float m, float sum, float gt,
                                          void* dt, int64_t row) const {
    const float all = list_kl(s, a, m, sum), logs = logf(sum) - logf(total);
    for (int j = threadIdx.x & 31; j < a.k; j += 32) {
      float g = 0.f;
      const float e = s.id[j] >= 0 ? exp2f(s.t2[j]) : 0.f;
      if (e != 0.f) {
        const float gap = kLn2 * (s.t2[j] - (s.z[j] - m) * a.c) + logs;
        g = gt * (e / total) * (gap - all);
      }
      store_float(dt, a.t_dtype, row * a.k + j, g);
    }
  }
  // By the whole CTA (several barriers).  An entry whose id's mark was set
  // already may be a repeated one: a warp looks through the list for it.
  template <typename F>
  __device__ __forceinline__ void tokens(Shared& s, const Taught& a, const T*, int, F put) const {
    const int lane = threadIdx.x & 31;
    const float inverse = reciprocal(s.total);
    for (int i = threadIdx.x; i < kMarks / 32; i += blockDim.x) s.marks[i] = 0;
    if (threadIdx.x == 0) s.suspects = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < a.k; j += blockDim.x) {
      const int id = s.id[j];
      s.mass[j] = id >= 0 ? exp2f(s.t2[j]) * inverse : -1.f;
      const uint32_t h = (uint32_t)id % kMarks;
      if (id >= 0 && (atomicOr(&s.marks[h / 32], 1u << (h % 32)) >> (h % 32)) & 1)
        s.suspect[atomicAdd(&s.suspects, 1)] = (short)j;
    }
    __syncthreads();
    for (int n = threadIdx.x >> 5; n < s.suspects; n += blockDim.x >> 5) {
      const int same = s.id[s.suspect[n]];
      int first = kMaxList, count = 0;
      float sum = 0.f;
      for (int j = lane; j < a.k; j += 32) {
        if (s.id[j] != same) continue;
        first = min(first, j);
        ++count;
        sum += exp2f(s.t2[j]) * inverse;
      }
      __syncwarp();
      if (__reduce_add_sync(0xffffffffu, count) == 1) continue;
      first = __reduce_min_sync(0xffffffffu, first);
      sum = warp_sum(sum);
      // (two warps at one id write the same values)
      for (int j = lane; j < a.k; j += 32)
        if (s.id[j] == same) s.mass[j] = j == first ? sum : -1.f;
    }
    __syncthreads();
    for (int j = threadIdx.x; j < a.k; j += blockDim.x)
      if (s.id[j] >= 0 && s.mass[j] != -1.f) put(s.id[j], s.z[j], s.mass[j]);
  }
};

// Loss and statistics: one read of the logits, with the running maximum and
// sum of a softmax in each thread.  One CTA a row, or a cluster of CTAs with a
// slice of packs each when there are few rows; a further warp reads the list
// meanwhile.  Bound by HBM: 8192 x 128256 bf16 in 302 us replayed from a graph
// (7.0 TB/s, above the 6.5 TB/s that a copy reaches, as nothing is written) and
// 330 to 360 us called again and again (5.8 to 6.4 TB/s); 32 x 32000 fp32 takes
// 3.5 to 4.3 us, its launch and three trips to memory.
template <typename T, int NS, int E>
__global__ void __launch_bounds__(NS + 32, 1024 / NS)
distill_fwd_kernel(const T* __restrict__ x, int64_t ld, Taught a, int cols,
                   float* __restrict__ loss, float2* __restrict__ stats) {
  constexpr int VW = Elem<T>::kVec;
  __shared__ typename ListOf<T, E>::Shared shared;
  ListOf<T, E> list;
  __shared__ float2 part[NS / 32];
  __shared__ float2 mine;
  pdl_prologue();
  const uint32_t rank = cluster_rank(), C = cluster_size();
  const int64_t row = cluster_id();
  const T* xr = x + row * ld;
  const int tid = threadIdx.x;
  if (tid >= NS) {
    if (rank == 0) list.load(shared, a, nullptr, 0, xr, row, cols, 0, cols, false);
  } else {
    const RowSplit sp = split_row(xr, cols);
    const uint4* body = reinterpret_cast<const uint4*>(xr + sp.head);
    const int per = (sp.nvec + (int)C - 1) / (int)C;
    const int end = min(sp.nvec, (int)(rank + 1) * per);
    MaxSum v = {kLowest, 0.f};
    if (rank == 0) {
      const int e = single_of(sp, tid, VW);
      if (e >= 0) fold(v, Elem<T>::to_f(xr[e]), a.c);
    }
    int p = (int)rank * per + tid;
    for (; p + 7 * NS < end; p += 8 * NS) {
      uint4 u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = ld_stream(body + p + i * NS);
      fold_packs<T, 8>(v, u, a.c);
    }
    constexpr uint32_t none = lowest_word<T>();
    for (; p < end; p += kUnroll * NS) {
      uint4 u[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        u[i] = p + i * NS < end ? ld_stream(body + p + i * NS) : make_uint4(none, none, none, none);
      fold_packs<T, kUnroll>(v, u, a.c);
    }
    v = warp_merge(v, a.c);
    if ((tid & 31) == 0) part[tid >> 5] = make_float2(v.m, v.s);
  }
  __syncthreads();
  if (tid >= NS) {
    const int lane = tid & 31;
    const float2 q = lane < NS / 32 ? part[lane] : make_float2(kLowest, 0.f);
    MaxSum v = warp_merge({q.x, q.y}, a.c);
    if (lane == 0) mine = make_float2(v.m, v.s);
  }
  if (C > 1) cluster_sync_all();
  if (tid >= NS && rank == 0) {
    const int lane = tid & 31;
    __syncwarp();
    float2 q = make_float2(kLowest, 0.f);
    if (lane < (int)C) q = C > 1 ? ld_remote_f2(remote_smem(&mine, lane)) : mine;
    const MaxSum v = warp_merge({q.x, q.y}, a.c);
    const bool live = list.total != 0.f;
    const float sum = final_sum(v.s);
    const float kl = live ? list.kl(shared, a, v.m, sum) : 0.f;
    if (lane == 0) {
      loss[row] = a.tau * a.tau * kl;
      stats[row] = live ? make_float2(v.m, sum) : make_float2(0.f, 0.f);
    }
  }
  if (C > 1) cluster_sync_all();  // no CTA leaves while rank 0 may read its pair
}

// Gradients of both operands from the forward's statistics: q w tau streamed
// over a chunk of the row, then the tokens of the teacher's list that lie in
// it written again, whole, from fp32 (so that each element is rounded once).
// Bound by HBM: 2048 x 128256 bf16 in 165 to 169 us (6.2 to 6.4 TB/s, 95 to
// 97% of the measured copy rate), 203 to 211 us with 256 teacher logits.
template <typename T, bool VEC, int NS, int E>
__global__ void __launch_bounds__(NS + 32, 1024 / NS)
distill_bwd_kernel(const float* __restrict__ dloss, int64_t dloss_stride, const T* __restrict__ x,
                   int64_t ld, const float2* __restrict__ stats, Taught a, int cols, int chunk,
                   int chunks, T* __restrict__ dx, int64_t ld_dx, void* __restrict__ dt) {
  constexpr int VW = Elem<T>::kVec;
  __shared__ typename ListOf<T, E>::Shared shared;
  ListOf<T, E> list;
  pdl_prologue();
  const int64_t row = blockIdx.x / (unsigned)chunks;
  const int part = (int)(blockIdx.x % (unsigned)chunks);
  const T* xr = x + row * ld;
  T* dr = dx + row * ld_dx;
  const int tid = threadIdx.x;
  const float2 st = stats[row];
  const bool live = st.y != 0.f;
  const float gt = (dloss != nullptr ? dloss[row * dloss_stride] : 1.f) * a.tau;
  const float f = gt / st.y;
  // elements [from, to); whole packs where VEC: pack p belongs to the chunk
  // that holds element p * VW, and the row's single elements to chunk 0
  const int from = part * chunk, to = min(cols, from + chunk);
  const RowSplit sp = split_row(xr, cols);
  const int p0 = min(sp.nvec, from / VW), p1 = part == chunks - 1 ? sp.nvec : min(sp.nvec, to / VW);
  const int lo = VEC ? sp.head + p0 * VW : from, hi = VEC ? sp.head + p1 * VW : to;
  const bool want_dt = dt != nullptr && part == 0;
  if (tid >= NS) {
    if (live)
      list.load(shared, a, nullptr, 0, xr, row, cols, part == 0 ? 0 : lo, part == 0 ? cols : hi, dx != nullptr);
    if (want_dt) {
      if (live) {
        list.teacher(shared, a, st.x, st.y, gt, dt, row);
      } else {
        for (int j = tid - NS; j < a.k; j += 32) store_float(dt, a.t_dtype, row * a.k + j, 0.f);
      }
    }
  } else if (dx != nullptr) {
    const auto grad = [&](float z) { return live ? ex2((z - st.x) * a.c) * f : 0.f; };
    if constexpr (VEC) {
      const uint4* body = reinterpret_cast<const uint4*>(xr + sp.head);
      uint4* out = reinterpret_cast<uint4*>(dr + sp.head);
      if (part == 0) {
        const int e = single_of(sp, tid, VW);
        if (e >= 0) dr[e] = Elem<T>::from_f(live ? grad(Elem<T>::to_f(xr[e])) : 0.f);
      }
      if (live) {
        const uint64_t minus = f2_make(-st.x, -st.x), c2 = f2_make(a.c, a.c), f2 = f2_make(f, f);
        for (int p = p0 + tid; p < p1; p += kUnroll * NS) {
          uint4 u[kUnroll];
#pragma unroll
          for (int i = 0; i < kUnroll; ++i)
            if (p + i * NS < p1) u[i] = ld_stream(body + p + i * NS);
#pragma unroll
          for (int i = 0; i < kUnroll; ++i) {
            if (p + i * NS >= p1) break;
            uint64_t e[VW / 2];
            to_pairs<T>(u[i], e);
#pragma unroll
            for (int j = 0; j < VW / 2; ++j) {
              const uint64_t d = f2_mul(f2_add(e[j], minus), c2);
              e[j] = f2_make(ex2(f2_lo(d)), ex2(f2_hi(d)));
            }
            st_stream(out + p + i * NS, from_pairs<T>(e, f2));
          }
        }
      } else {
        for (int p = p0 + tid; p < p1; p += NS) st_stream(out + p, make_uint4(0, 0, 0, 0));
      }
    } else {
      for (int e = from + tid; e < to; e += NS)
        dr[e] = Elem<T>::from_f(live ? grad(Elem<T>::to_f(xr[e])) : 0.f);
    }
  }
  if (!live || dx == nullptr) return;  // (the whole CTA)
  __syncthreads();                     // the chunk is stored
  const auto put = [&](int id, float z, float mass) {
    const bool single = VEC && (id < sp.head || id >= sp.head + sp.nvec * VW);
    if (single ? part == 0 : (id >= lo && id < hi))
      dr[id] = Elem<T>::from_f(gt * (ex2((z - st.x) * a.c) * reciprocal(st.y) - mass));
  };
  list.tokens(shared, a, xr, NS, put);
}

// Many short rows, a warp each: loss and statistics (LOSS), gradients (GRAD)
// from given statistics, or both, the row's second read from L2.  In the
// kernels above a row's chain (the list, its logits, the sums' meeting) holds a
// whole CTA; here it holds a warp, of which 32 an SM are under way.
constexpr int kRowWarps = 4;

template <typename T, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(kRowWarps * 32, GRAD ? 6 : 8)
distill_rows_kernel(const T* __restrict__ x, int64_t ld, Taught a, const float* __restrict__ weight,
                    int64_t weight_stride, int64_t rows, int cols, float* __restrict__ loss,
                    float2* __restrict__ stats, T* __restrict__ dx, int64_t ld_dx, void* __restrict__ dt) {
  constexpr int VW = Elem<T>::kVec, U = kUnroll;
  __shared__ typename ListOf<T, 2>::Shared shared[GRAD ? kRowWarps : 1];
  ListOf<T, 2> list;
  pdl_prologue();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + warp;
  if (row >= rows) return;
  const T* xr = x + row * ld;
  const RowSplit sp = split_row(xr, cols);
  const uint4* body = reinterpret_cast<const uint4*>(xr + sp.head);
  const int e = single_of(sp, lane, VW);
  ListAhead<2> in;
  in.load(a, weight, weight_stride, row);
  float2 st = LOSS ? make_float2(0.f, 0.f) : stats[row];
  const float alone = e >= 0 ? Elem<T>::to_f(xr[e]) : kLowest;
  uint4 u[U];
  constexpr uint32_t none = lowest_word<T>();
  const auto load = [&](uint4 (&u)[U], int p) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      u[i] = p + 32 * i < sp.nvec ? (GRAD ? ld_cached(body + p + 32 * i) : ld_stream(body + p + 32 * i))
                                  : make_uint4(none, none, none, none);
  };
  load(u, lane);
  uint32_t* marks = shared[GRAD ? warp : 0].marks;
  if constexpr (GRAD) {
    for (int i = lane; i < kMarkBits / 32; i += 32) marks[i] = 0;
    __syncwarp();
  }
  list.held.set(a, in, xr, cols, 0, cols);
  list.total = list.held.total;
  bool live = st.y != 0.f;
  if constexpr (LOSS) {
    MaxSum v = {kLowest, 0.f};
    if (e >= 0) fold(v, alone, a.c);
    for (int p = 32 * U; p < sp.nvec; p += 32 * U) {
      uint4 next[U];
      load(next, p + lane);
      fold_packs<T, U>(v, u, a.c);
#pragma unroll
      for (int i = 0; i < U; ++i) u[i] = next[i];
    }
    fold_packs<T, U>(v, u, a.c);
    v = warp_merge(v, a.c);
    live = list.total != 0.f;
    const float sum = final_sum(v.s);
    const float kl = live ? list.kl(shared[0], a, v.m, sum) : 0.f;
    st = live ? make_float2(v.m, sum) : make_float2(0.f, 0.f);
    if (lane == 0) {
      loss[row] = a.tau * a.tau * kl;
      stats[row] = st;
    }
    if (GRAD) load(u, lane);
  }
  if constexpr (GRAD) {
    T* dr = dx + row * ld_dx;
    uint4* out = reinterpret_cast<uint4*>(dr + sp.head);
    const float gt = list.held.by, f = gt / st.y;
    if (dt != nullptr) {
      if (live) {
        list.teacher(shared[0], a, st.x, st.y, gt, dt, row);
      } else {
        for (int j = lane; j < a.k; j += 32) store_float(dt, a.t_dtype, row * a.k + j, 0.f);
      }
    }
    if (!live) {
      if (e >= 0) dr[e] = Elem<T>::from_f(0.f);
      for (int p = lane; p < sp.nvec; p += 32) st_stream(out + p, make_uint4(0, 0, 0, 0));
      return;
    }
    list.held.set_masses(a, marks);
    if (e >= 0) dr[e] = Elem<T>::from_f(ex2((alone - st.x) * a.c) * f);
    const uint64_t minus = f2_make(-st.x, -st.x), c2 = f2_make(a.c, a.c), f2 = f2_make(f, f);
    const auto write = [&](int p) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (p + 32 * i >= sp.nvec) break;
        uint64_t g[VW / 2];
        to_pairs<T>(u[i], g);
#pragma unroll
        for (int j = 0; j < VW / 2; ++j) {
          const uint64_t d = f2_mul(f2_add(g[j], minus), c2);
          g[j] = f2_make(ex2(f2_lo(d)), ex2(f2_hi(d)));
        }
        st_stream(out + p + 32 * i, from_pairs<T>(g, f2));
      }
    };
    int p = lane;
    for (; p - lane + 32 * U < sp.nvec; p += 32 * U) {
      uint4 next[U];
      load(next, p + 32 * U);
      write(p);
#pragma unroll
      for (int i = 0; i < U; ++i) u[i] = next[i];
    }
    write(p);
    __syncwarp();  // the row is stored
    list.tokens(shared[0], a, xr, 0, [&](int id, float z, float mass) {
      dr[id] = Elem<T>::from_f(gt * (ex2((z - st.x) * a.c) * reciprocal(st.y) - mass));
    });
  }
}

// ---------------------------------------------- loss and gradient at once ---
//
// One read of the logits and one write of the gradient: a cluster holds a row
// on chip, 128 bytes of logits a thread, as exponentials 2^((z - m_w) c)
// against the warp's own maximum.  Every warp sends its (m_w, sum) to every
// CTA of the cluster (st.async on a transaction barrier: no fence, no second
// hop through a CTA total), where one warp folds all pairs to (M, S); the
// others then write w tau e 2^((m_w - M) c) / S over the logits in shared
// memory.  Three
// stages of a row's slice take turns: one arriving, one in hand, one leaving,
// each by one bulk copy, so that neither memory direction holds up the warps
// (stores from registers did: a third of a row's time was theirs).
//
// That warp is one of two more, a row each in turn, which read the teacher's
// lists ahead, put the gradients of the tokens they name in place, issue the
// copies and in CTA 0 write the loss (a single one took longer over 64 entries
// than the holders over a row).
//
// Measured (of the 6.5 TB/s that a copy reaches): 2048 x 128256 bf16 with 64
// teacher logits 182 us (89%), 1024 x 128256 fp32 178 us (91%), 32768 x 8192
// bf16 172 us (96%).  (1 to 2% of the first two are the checks of given-up
// waits.)  What is left for 16-bit types at long rows is the chain
// of a row: wait, exponentials, exchange, scale, with two CTAs an SM to overlap.
constexpr int kPacks = 8;            // 16-byte packs a thread holds
constexpr int kStages = 3;
constexpr int kMaxCluster = 16;

// No wait lasts longer than a limit.  A thread that gives up tells every CTA of
// the cluster; from then on its CTAs only step through their rows: nothing more
// is expected of a barrier, sent or copied.  What had been under way is counted
// at the end and waited for, so that nothing arrives in the shared memory of a
// CTA that has left, and every row of the cluster is reported as NaN.
template <int NT>
struct GradShared {
  uint4 stage[kStages][kPacks][NT];
  float2 pair[2][kMaxCluster * (NT / 32)];
  uint32_t marks[2][kMarkBits / 32];
  float2 scale[2];  // the row's M, and w tau / S
  int state[2];     // kLive: something is taught; kDead: a wait has been given up
  uint64_t bar[2];          // the row's pairs have come
  uint64_t full[kStages];   // the stage's logits have come
  int lost;                 // a CTA of the cluster has given up a wait
  int expected[2], loaded[kStages];  // phases begun, of bar and full
  int sent[NT / 32];                 // rows whose pairs this warp has sent
};
constexpr int kLive = 1, kDead = 2;

// Clusters that gave up a wait, on this device.
__device__ unsigned long long lost_clusters;
constexpr uint32_t kDrainLimit = 2000000000u;  // nanoseconds

// Waits for what is still on its way to this CTA's shared memory, once no CTA
// of the cluster sends or copies any more.  By one warp.  (All pairs that were
// sent arrive: sent and expected bytes tell what each barrier is short of, or
// has had beyond its last phase.)
template <int NT>
__device__ __noinline__ void drain(GradShared<NT>& s, int C) {
  constexpr int W = NT / 32;
  const int lane = threadIdx.x & 31;
  const int zero = 0;
  int pairs[2] = {0, 0};
  if (lane < C) {
    for (int w = 0; w < W; ++w) {
      const int n = ld_remote_s32(remote_smem(&s.sent[w], lane));
      pairs[0] += (n + 1) / 2;  // rows alternate between the barriers
      pairs[1] += n / 2;
    }
  }
  for (int par = 0; par < 2; ++par) {
    const int n = __reduce_add_sync(0xffffffffu, pairs[par]);
    if (lane != 0) continue;
    const int begun = s.expected[par], over = n - begun * C * W;
    if (over < 0) bar_give(&s.bar[par], -over * 8);
    const bool settled = begun == 0 || bar_wait(&s.bar[par], (begun - 1) & 1, &zero, kDrainLimit);
    if (over > 0 && settled) {
      bar_expect(&s.bar[par], over * 8);
      (void)bar_wait(&s.bar[par], begun & 1, &zero, kDrainLimit);
    }
  }
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i)
      if (s.loaded[i] > 0) (void)bar_wait(&s.full[i], (s.loaded[i] - 1) & 1, &zero, kDrainLimit);
  }
}

constexpr int kHelpers = 64;  // threads besides the NT that hold the row
// Named barriers, two of each for alternate rows: a barrier's next use follows,
// through the other kind, every wait on this one.
constexpr int kScaled = 1;  // the row's scale is known: the holders wait for the list's warp
constexpr int kHeld = 3;    // the gradient is in place: the list's warp waits for the holders

// Reports every row of this cluster as NaN.
template <typename T, int NT>
__device__ __noinline__ void report_lost(const T* x, int64_t ld, int64_t rows, int cols, float* loss,
                                         float2* stats, T* dx, int64_t ld_dx) {
  constexpr int VW = Elem<T>::kVec;
  const int tid = threadIdx.x;
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const float none = NAN;
  const uint32_t word = std::is_same<T, float>::value    ? __float_as_uint(none)
                        : std::is_same<T, __half>::value ? 0x7e007e00u
                                                         : 0x7fc07fc0u;
  for (int64_t row = cluster_id(); row < rows; row += cluster_count()) {
    const RowSplit sp = split_row(x + row * ld, cols);
    T* dr = dx + row * ld_dx;
    uint4* out = reinterpret_cast<uint4*>(dr + sp.head);
    for (int p = rank * (NT + kHelpers) + tid; p < sp.nvec; p += C * (NT + kHelpers))
      out[p] = make_uint4(word, word, word, word);
    if (rank != 0) continue;
    const int e = single_of(sp, tid, VW);
    if (e >= 0) dr[e] = Elem<T>::from_f(none);
    if (tid == 0) {
      loss[row] = none;
      stats[row] = make_float2(none, none);
    }
  }
  if (rank == 0 && tid == 0) atomicAdd(&lost_clusters, 1ull);
}

// E entries of a list a lane.
template <typename T, int NT, int E>
__global__ void __launch_bounds__(NT + kHelpers, NT == 256 ? 2 : NT == 128 ? 3 : 5)
distill_grad_kernel(const T* __restrict__ x, int64_t ld, Taught a, const float* __restrict__ weight,
                    int64_t weight_stride, int64_t rows, int cols, float* __restrict__ loss,
                    float2* __restrict__ stats, T* __restrict__ dx, int64_t ld_dx, uint32_t limit) {
  constexpr int VW = Elem<T>::kVec;
  constexpr int P = kPacks;
  constexpr int W = NT / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  GradShared<NT>& s = *reinterpret_cast<GradShared<NT>*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int64_t first = cluster_id(), step = cluster_count();
  for (int i = tid; i < 2 * (kMarkBits / 32); i += NT + kHelpers) s.marks[0][i] = 0;
  if (tid == 0) {
    bar_init(&s.bar[0], 1);
    bar_init(&s.bar[1], 1);
    for (int i = 0; i < kStages; ++i) bar_init(&s.full[i], 1);
    s.lost = 0;
    s.expected[0] = s.expected[1] = 0;
    for (int i = 0; i < kStages; ++i) s.loaded[i] = 0;
    bar_init_fence();
  }
  pdl_prologue();
  cluster_sync_all();
  // this CTA's packs [from, to) of a row's split (a row has cols / VW packs or
  // one fewer, by its alignment: no division a row)
  const int most = cols / VW, per_most = (most + C - 1) / C, per_less = (most + C - 2) / C;
  const auto slice = [&](const RowSplit& sp, int& from, int& to) {
    const int per = sp.nvec == most ? per_most : per_less;
    from = min(sp.nvec, rank * per);
    to = min(sp.nvec, from + per);
  };
  const auto give_up = [&] {
    for (int r = 0; r < (int)cluster_size(); ++r) st_remote_s32(remote_smem(&s.lost, r), 1);
  };
  if (warp >= W) {
    // every other row's list, and its copies
    const int par = warp - W;
    bool ok = true;  // no wait has been given up, as far as this warp knows
    ListAhead<E> next;
    ListHeld<T, E> list;
    const auto set = [&](int64_t row) {
      const T* xr = x + row * ld;
      const RowSplit sp = split_row(xr, cols);
      int from, to;
      slice(sp, from, to);
      if (lane == 0 && ok) {
        bar_expect(&s.bar[par], C * W * 8);
        ++s.expected[par];
      }
      list.set(a, next, xr, cols, rank == 0 ? 0 : sp.head + from * VW,
               rank == 0 ? cols : sp.head + to * VW);
      if (row + 2 * step < rows) next.load(a, weight, weight_stride, row + 2 * step);
    };
    const auto load = [&](int64_t row, int stage) {
      if (row >= rows || lane != 0 || !ok) return;
      const T* xr = x + row * ld;
      const RowSplit sp = split_row(xr, cols);
      int from, to;
      slice(sp, from, to);
      bar_expect(&s.full[stage], (to - from) * 16);
      ++s.loaded[stage];
      if (to > from)
        bulk_load(s.stage[stage], reinterpret_cast<const uint4*>(xr + sp.head) + from, (to - from) * 16,
                  &s.full[stage]);
    };
    for (int i = par; i < kStages; i += 2) load(first + i * step, i);
    if (first + par * step < rows) {
      next.load(a, weight, weight_stride, first + par * step);
      set(first + par * step);
    }
    int stage = par;
    uint32_t phase = 0;
    for (int64_t row = first + par * step; row < rows; row += 2 * step, phase ^= 1) {
      if (ok && !bar_wait(&s.bar[par], phase, &s.lost, limit)) {
        give_up();
        ok = false;
      }
      const int lost = *(volatile int*)&s.lost;
      constexpr int kPairs = kMaxCluster * W / 32;  // a lane's, at most
      float2 q[kPairs];
      float M = kLowest, S = 0.f;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        q[i] = lane + 32 * i < C * W ? s.pair[par][lane + 32 * i] : make_float2(kLowest, 0.f);
        M = fmaxf(M, q[i].x);
      }
      M = warp_max(M);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) S += q[i].y * ex2((q[i].x - M) * a.c);
      S = final_sum(warp_sum(S));
      const float inverse = reciprocal(S);
      const bool live = list.total != 0.f;
      if (lane == 0) {
        s.scale[par] = make_float2(M, list.by * inverse);
        s.state[par] = (live ? kLive : 0) | (ok && lost == 0 ? 0 : kDead);
      }
      __syncwarp();
      named_arrive(kScaled + par, NT + 32);
      list.set_masses(a, s.marks[par]);  // (while the holders write the row)
      const RowSplit sp = split_row(x + row * ld, cols);
      int from, to;
      slice(sp, from, to);
      T* dr = dx + row * ld_dx;
      named_sync(kHeld + par, NT + 32);
      ok = __all_sync(0xffffffffu, ok && *(volatile int*)&s.lost == 0);  // (so every holder had the row)
      if (live) {
        const int lo = sp.head + from * VW, hi = sp.head + to * VW;
        T* held = reinterpret_cast<T*>(s.stage[stage]);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          if (32 * i >= a.k) break;
          const int id = list.id[i];
          const float q = ex2((bits_value<T>(list.z[i]) - M) * a.c) * inverse;
          const T g = Elem<T>::from_f(list.by * (q - list.mass[i]));
          const bool mine = id >= 0 && list.mass[i] != -1.f;
          if (mine && id >= lo && id < hi) held[id - lo] = g;
          // the row's single elements are CTA 0's
          if (mine && rank == 0 && (id < sp.head || id >= sp.head + sp.nvec * VW)) dr[id] = g;
        }
        bulk_fence();
        __syncwarp();
      }
      if (lane == 0) {
        if (to > from && ok)
          bulk_store(reinterpret_cast<uint4*>(dr + sp.head) + from, s.stage[stage], (to - from) * 16);
        bulk_commit();
      }
      if (rank == 0) {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          if (32 * i >= a.k) break;
          if (live && list.id[i] >= 0 && list.e[i] != 0.f)
            d += list.e[i] * (list.t2[i] - (bits_value<T>(list.z[i]) - M) * a.c);
        }
        d = warp_sum(d);
        if (lane == 0) {
          const float kl = live ? kLn2 * (d / list.total) + (logf(S) - logf(list.total)) : 0.f;
          loss[row] = a.tau * a.tau * kl;
          stats[row] = live ? make_float2(M, S) : make_float2(0.f, 0.f);
        }
      }
      // (the store reads its stage meanwhile)
      if (row + 2 * step < rows) set(row + 2 * step);
      if (lane == 0) bulk_wait_read();
      __syncwarp();
      load(row + kStages * step, stage);
      stage = (stage + 2) % kStages;
    }
    if (lane == 0) bulk_wait();
  } else {
    // where this warp's pairs go: lane r's copy to CTA r
    const uint32_t to_pair = remote_smem(&s.pair[0][rank * W + warp], lane < C ? lane : 0);
    const uint32_t to_bar = remote_smem(&s.bar[0], lane < C ? lane : 0);
    const uint64_t c2 = f2_make(a.c, a.c);
    const bool edge = rank == 0 && warp == 0;  // has the rows' single elements
    const auto single_at = [&](const T* xr) {
      return edge ? single_of(split_row(xr, cols), lane, VW) : -1;
    };
    int single = single_at(x + first * ld);
    float xs = single >= 0 ? Elem<T>::to_f((x + first * ld)[single]) : -INFINITY;
    int par = 0, stage = 0;
    uint32_t stage_phase = 0;
    bool ok = true;
    if (lane == 0) s.sent[warp] = 0;
    // (32 bits hold a row and one step more)
    for (uint32_t row = (uint32_t)first; row < (uint32_t)rows; row += (uint32_t)step) {
      const RowSplit sp = split_row(x + row * ld, cols);
      int from, to;
      slice(sp, from, to);
      const int left = to - from - tid;  // the thread's packs end here
      const bool whole = __all_sync(0xffffffffu, left > (P - 1) * NT);
      uint4* held = &s.stage[stage][0][tid];
      // values, then exponentials, in pairs
      uint64_t e[P][VW / 2];
      float m = fmaxf(kLowest, xs);
      if (ok && !bar_wait(&s.full[stage], stage_phase, &s.lost, limit)) give_up();
#pragma unroll
      for (int i = 0; i < P; ++i) {
        uint4 u = held[i * NT];
        if (!whole && i * NT >= left) {
          const uint32_t none = lowest_word<T>();
          u = make_uint4(none, none, none, none);
        }
        m = fmaxf(m, pack_max<T>(u));
        to_pairs<T>(u, e[i]);
      }
      m = warp_max(m);
      xs = ex2((xs - m) * a.c);
      const uint64_t minus = f2_make(-m, -m);
      uint64_t sum2 = f2_make(xs, 0.f);
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int j = 0; j < VW / 2; ++j) {
          const uint64_t d = f2_mul(f2_add(e[i][j], minus), c2);
          e[i][j] = f2_make(ex2(f2_lo(d)), ex2(f2_hi(d)));
          sum2 = f2_add(sum2, e[i][j]);
        }
      const float sum = warp_sum(f2_lo(sum2) + f2_hi(sum2));
      if (ok) {
        if (lane < C) send_f2(to_pair + par * (uint32_t)sizeof(s.pair[0]), m, sum, to_bar + par * 8);
        if (lane == 0) ++s.sent[warp];
      }
      // the next row's single element travels while this row is exchanged
      const float es = xs;
      const int at_single = single;
      const T* following = x + (row + (uint32_t)step) * ld;
      single = row + (uint32_t)step < (uint32_t)rows ? single_at(following) : -1;
      xs = single >= 0 ? Elem<T>::to_f(following[single]) : -INFINITY;
      named_sync(kScaled + par, NT + 32);
      const int state = s.state[par];
      ok = ok && (state & kDead) == 0;
      if (state & kLive) {
        const float2 sc = s.scale[par];
        const float f = ex2((m - sc.x) * a.c) * sc.y;
        const uint64_t f2 = f2_make(f, f);
        if (at_single >= 0) dx[row * ld_dx + at_single] = Elem<T>::from_f(es * f);
#pragma unroll
        for (int i = 0; i < P; ++i) held[i * NT] = from_pairs<T>(e[i], f2);
      } else {
        if (at_single >= 0) dx[row * ld_dx + at_single] = Elem<T>::from_f(0.f);
#pragma unroll
        for (int i = 0; i < P; ++i) held[i * NT] = make_uint4(0, 0, 0, 0);
      }
      bulk_fence();
      named_arrive(kHeld + par, NT + 32);
      par ^= 1;
      if (++stage == kStages) {
        stage = 0;
        stage_phase ^= 1;
      }
    }
  }
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while pairs may still be sent to it
  if (*(volatile int*)&s.lost == 0) return;  // (the same in every CTA of the cluster)
  if (threadIdx.x < 32) drain(s, (int)cluster_size());
  __syncwarp();
  cluster_sync_all();  // the counts are read, and nothing of the cluster's is under way
  report_lost<T, NT>(x, ld, rows, cols, loss, stats, dx, ld_dx);
}

// ------------------------------------------------------------------ host ---

std::atomic<uint32_t> g_wait_limit{2000000000u};  // nanoseconds; fl_b200_set_wait_limit

bool list_dtypes_ok(int t_dtype, int ids_dtype) {
  return is_float_dtype(t_dtype) && (ids_dtype == FL_B200_I32 || ids_dtype == FL_B200_I64);
}

int check_shapes(int64_t rows, int64_t cols, int64_t k, float temperature) {
  FLB_CHECK_ARG(rows >= 0 && cols >= 0 && k >= 0);
  // (and log2(e) / temperature finite)
  FLB_CHECK_ARG(temperature > 1e-37f && temperature <= 3.0e38f);
  if (k > kMaxList || cols > kMaxCols || rows > 0x7fffffffLL) return FL_B200_ERR_TOO_LARGE;
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

// The rows of a matrix in memory, and whether a row of one meets a row of
// another.  (Rows may lie between each other's.)
struct Region {
  const void* p;
  int64_t ld, cols, rows;  // elements
  int64_t size;
};
bool meet(const Region& a, const Region& b) {
  if (a.p == nullptr || b.p == nullptr || a.cols == 0 || b.cols == 0) return false;
  const uintptr_t la = a.ld * a.size, lb = b.ld * b.size, na = a.cols * a.size, nb = b.cols * b.size;
  uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  if (x + (a.rows - 1) * la + na <= y || y + (b.rows - 1) * lb + nb <= x) return false;
  for (int64_t i = 0, j = 0; i < a.rows && j < b.rows;) {
    if (x + na <= y) {
      x += la;
      ++i;
    } else if (y + nb <= x) {
      y += lb;
      ++j;
    } else {
      return true;
    }
  }
  return false;
}

// Calls go(NS, E): the threads that stream a row (and one warp more for its
// list) and the list's entries a lane.  Rows of up to 64 KB go to CTAs of 128
// threads, of which more are resident to hide the lists' latency (forward,
// 8192 x 16384 bf16: 52 us, 62 us with 256, 93 us with 512); from there on 256
// do as well.
template <typename T, typename F>
int with_geometry(int64_t cols, int64_t k, F&& go) {
  using Small = std::integral_constant<int, 128>;
  using Large = std::integral_constant<int, 256>;
  using Held = std::integral_constant<int, 2>;
  using Any = std::integral_constant<int, 0>;
  if (cols * (int64_t)sizeof(T) <= 65536) return k <= 64 && k > 0 ? go(Small{}, Held{}) : go(Small{}, Any{});
  return k <= 64 && k > 0 ? go(Large{}, Held{}) : go(Large{}, Any{});
}

// Whether a warp a row is the form to take, by the bytes of a row.  The loss
// alone gains up to 16 KB (16000 rows of 1024 bf16, 32 entries: 11.2 us, 40.0
// with a CTA a row; of 8000: 43, 71; 700 of 8000: 5.5, 6.7), the two at once up
// to 6 KB, where the row is still in L1 when it is read again (16000 x 1024: 19
// us, 45; 16000 x 2048: 32, 46; 16000 x 4096: 53, 52).  The gradient alone has one read to hide its list
// behind: up to 2 KB, or to 8 KB where rows are many (16000 x 4096: 45 us, 55;
// 700 x 4096: 6.2, 4.0).
enum class Rows { kLoss, kGrad, kBoth };
bool short_rows(Rows what, const DeviceInfo& dev, int64_t rows, int64_t bytes, int64_t k) {
  int64_t most = rows > 16 * dev.sm_count ? 8192 : 2048;
  if (what == Rows::kLoss) most = 16384;
  if (what == Rows::kBoth) most = 6144;
  return k > 0 && k <= 64 && rows > 4 * dev.sm_count && bytes <= most;
}
template <typename T, bool LOSS, bool GRAD>
int run_rows(const void* x, int64_t ld, const Taught& a, const float* weight, int64_t weight_stride,
             int64_t rows, int64_t cols, float* loss, float* stats, void* dx, int64_t ld_dx, void* dt,
             cudaStream_t stream) {
  launch_k(distill_rows_kernel<T, LOSS, GRAD>, dim3((unsigned)ceil_div(rows, kRowWarps)), dim3(kRowWarps * 32),
           0, stream, reinterpret_cast<const T*>(x), ld, a, weight, weight_stride, rows, (int)cols, loss,
           reinterpret_cast<float2*>(stats), reinterpret_cast<T*>(dx), ld_dx, dt);
  return launch_status();
}

template <typename T>
int run_fwd(const void* x, int64_t ld, const Taught& a, int64_t rows, int64_t cols, float* loss,
            float* stats, cudaStream_t stream) {
  DeviceInfo dev;
  const int st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  if (short_rows(Rows::kLoss, dev, rows, cols * sizeof(T), a.k))
    return run_rows<T, true, false>(x, ld, a, nullptr, 0, rows, cols, loss, stats, nullptr, 0, nullptr, stream);
  return with_geometry<T>(cols, a.k, [&](auto ns, auto e) {
    constexpr int NS = decltype(ns)::value;
    int cluster = 1;
    while (cluster < 8 && rows * cluster < 2 * dev.sm_count && cols / (cluster * 2) >= NS * Elem<T>::kVec)
      cluster *= 2;
    return launch_cluster(distill_fwd_kernel<T, NS, decltype(e)::value>, rows * cluster, cluster, NS + 32,
                          0, stream, reinterpret_cast<const T*>(x), ld, a, (int)cols, loss,
                          reinterpret_cast<float2*>(stats));
  });
}

template <typename T>
int run_bwd(const float* dloss, int64_t dloss_stride, const void* x, int64_t ld, const float* stats,
            const Taught& a, int64_t rows, int64_t cols, void* dx, int64_t ld_dx, void* dt,
            cudaStream_t stream) {
  DeviceInfo dev;
  const int st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  const bool vec = dx == nullptr || same_phase(x, ld, dx, ld_dx, sizeof(T));
  if (dx != nullptr && vec && short_rows(Rows::kGrad, dev, rows, cols * sizeof(T), a.k))
    return run_rows<T, false, true>(x, ld, a, dloss, dloss_stride, rows, cols, nullptr, const_cast<float*>(stats),
                                    dx, ld_dx, dt, stream);
  return with_geometry<T>(cols, a.k, [&](auto ns, auto e) {
    constexpr int NS = decltype(ns)::value, E = decltype(e)::value;
    // chunks of 4 rounds of loads, which hide the list's latency (2048 x 128256
    // bf16: 201 us, 249 us with one round), of 16 for a long list; shorter where
    //     // where rows are few; the teacher's gradient alone is one CTA's work
    const int64_t round = (int64_t)NS * kUnroll * Elem<T>::kVec;
    int64_t chunk = dx == nullptr ? cols : (E == 0 ? 16 : 4) * round;
    while (dx != nullptr && chunk > round && rows * ceil_div(cols, chunk) < 4 * dev.sm_count) chunk /= 2;
    const int64_t chunks = ceil_div(cols, chunk);
    if (rows * chunks > 0x7fffffffLL) return (int)FL_B200_ERR_TOO_LARGE;
    const auto go = [&](auto kern) {
      launch_k(kern, dim3((unsigned)(rows * chunks)), dim3(NS + 32), 0, stream, dloss, dloss_stride,
               reinterpret_cast<const T*>(x), ld, reinterpret_cast<const float2*>(stats), a, (int)cols,
               (int)chunk, (int)chunks, reinterpret_cast<T*>(dx), ld_dx, dt);
      return launch_status();
    };
    return vec ? go(distill_bwd_kernel<T, true, NS, E>) : go(distill_bwd_kernel<T, false, NS, E>);
  });
}

// Clusters of `cluster` CTAs of a kernel that are resident at once, asked for
// once a device; 0 when the kernel cannot run so.
template <typename T, int NT, int E>
int grad_clusters(int cluster, cudaLaunchConfig_t cfg) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][kMaxCluster + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return 0;
  int n = known[dev][cluster].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveClusters(&n, distill_grad_kernel<T, NT, E>, &cfg) != cudaSuccess) n = 0;
    (void)cudaGetLastError();
    known[dev][cluster].store(n > 0 ? n : -1, std::memory_order_relaxed);
  }
  return n > 0 ? n : 0;
}

// The one-pass kernel; returns -1 where it does not apply.
template <typename T, int NT, int E>
int run_grad(const void* x, int64_t ld, const Taught& a, const float* weight, int64_t weight_stride,
             int64_t rows, int64_t cols, float* loss, float* stats, void* dx, int64_t ld_dx,
             cudaStream_t stream) {
  const auto kern = distill_grad_kernel<T, NT, E>;
  const int64_t cluster = ceil_div(cols, (int64_t)NT * kPacks * Elem<T>::kVec);
  if (cluster > kMaxCluster) return -1;
  const size_t smem = sizeof(GradShared<NT>);
  static std::atomic<int> allowed[64];
  if (!allow_smem(kern, smem, cluster > 8, allowed)) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.blockDim = dim3(NT + kHelpers);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int clusters = grad_clusters<T, NT, E>((int)cluster, cfg);
  if (clusters == 0) return -1;
  return launch_cluster(kern, std::min<int64_t>(rows, clusters) * cluster, (int)cluster, NT + kHelpers, smem,
                        stream, reinterpret_cast<const T*>(x), ld, a, weight, weight_stride, rows,
                        (int)cols, loss, reinterpret_cast<float2*>(stats), reinterpret_cast<T*>(dx),
                        ld_dx, g_wait_limit.load(std::memory_order_relaxed));
}

}  // namespace
}  // namespace flb200

extern "C" {

FL_B200_API int64_t fl_b200_set_wait_limit(int64_t nanoseconds) {
  const int64_t ns = std::min<int64_t>(std::max<int64_t>(nanoseconds, 0), 2000000000);
  return flb200::g_wait_limit.exchange((uint32_t)ns, std::memory_order_relaxed);
}

FL_B200_API int fl_b200_lost_waits(uint64_t* count) {
  using namespace flb200;
  FLB_CHECK_ARG(count != nullptr);
  unsigned long long n = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&n, lost_clusters, sizeof n);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    set_last_cuda_error(e);
    return FL_B200_ERR_NO_DEVICE;
  }
  *count = n;
  return FL_B200_OK;
}

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
  // an operand may be read after any row of a gradient is stored
  const Region out[] = {{dlogits, ld_dlogits, cols, rows, dtype_size(dtype)},
                        {dteacher, k, k, rows, dtype_size(t_dtype)}};
  const Region in[] = {{logits, ld, cols, rows, dtype_size(dtype)},
                       {teacher, ld_t, k, rows, dtype_size(t_dtype)},
                       {ids, ld_ids, k, rows, dtype_size(ids_dtype)},
                       {dloss, dloss_stride, 1, rows, 4},
                       {stats, 2, 2, rows, 4}};
  for (const Region& o : out)
    for (const Region& i : in) FLB_CHECK_ARG(!meet(o, i));
  FLB_CHECK_ARG(!meet(out[0], out[1]));
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
  // rows are read and stored in no order
  const Region out[] = {{dlogits, ld_dlogits, cols, rows, dtype_size(dtype)},
                        {loss, 1, 1, rows, 4},
                        {stats, 2, 2, rows, 4}};
  const Region in[] = {{logits, ld, cols, rows, dtype_size(dtype)},
                       {teacher, ld_t, k, rows, dtype_size(t_dtype)},
                       {ids, ld_ids, k, rows, dtype_size(ids_dtype)},
                       {row_weight, weight_stride, 1, rows, 4}};
  for (const Region& o : out)
    for (const Region& i : in) FLB_CHECK_ARG(!meet(o, i));
  FLB_CHECK_ARG(!meet(out[0], out[1]) && !meet(out[0], out[2]));
  if (same_phase(logits, ld, dlogits, ld_dlogits, dtype_size(dtype))) {
    const Taught a = taught(teacher, ld_t, t_dtype, ids, ld_ids, ids_dtype, k, temperature);
    DeviceInfo dev;
    st = current_device_info(&dev);
    if (st != FL_B200_OK) return st;
    st = dispatch_float(dtype, [&](auto t) {
      using T = decltype(t);
      if (short_rows(Rows::kBoth, dev, rows, cols * sizeof(T), k))
        return run_rows<T, true, true>(logits, ld, a, row_weight, weight_stride, rows, cols, loss, stats,
                                       dlogits, ld_dlogits, nullptr, (cudaStream_t)stream);
      const auto go = [&](auto threads) {
        constexpr int NT = decltype(threads)::value;
        const auto each = [&](auto entries) {
          return run_grad<T, NT, decltype(entries)::value>(logits, ld, a, row_weight, weight_stride, rows,
                                                           cols, loss, stats, dlogits, ld_dlogits,
                                                           (cudaStream_t)stream);
        };
        if (k <= 64) return each(std::integral_constant<int, 2>{});
        if (k <= 128) return each(std::integral_constant<int, 4>{});
        return -1;
      };
      constexpr int kHold = kPacks * Elem<T>::kVec;  // elements a thread
      if (cols <= 64 * kHold) return go(std::integral_constant<int, 64>{});
      // clusters of up to 7 CTAs of 128 threads, three an SM, beat half as many
      // of 256, two an SM (16384 x 16384 bf16: 170 us, 191 us; 1001 x 40003 f16:
      // 35 us, 41 us); from 8 on these do (4096 x 65536: 185 us, 175 us)
      if (cols <= 7 * 128 * kHold) return go(std::integral_constant<int, 128>{});
      return go(std::integral_constant<int, 256>{});
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
