// The norm after a block, its gate and scale, the residual add and the norm
// before the next block in one pass, and the gradients.
//
//   n = x / sqrt(mean(x^2) + eps)
//   h = residual + scale * gate * n * (o + post)        (gate 1 where none is given)
//   y = h / sqrt(mean(h^2) + eps) * (o + pre)
//
// o is the weights' offset (0, or 1 for weights stored as differences from
// 1); the gate holds one row for every `rows_per_gate` rows: one for all (a
// gate a channel), one a sequence, or one a token.  Everything is fp32 and h
// and y are rounded once: y is the norm of h before its rounding.
//
// Gradients, with m = h / sqrt(mean(h^2) + eps) from the h that was stored:
//   g         = dh + (dy w - m mean(dy w m)) / sqrt(mean(h^2) + eps),  w = o + pre
//   dresidual = g
//   dpre      = sum over rows of dy m
//   A         = sum over a gate row's rows of g n
//   dgate     = scale (o + post) A,   dpost = scale * sum over gate rows of gate A
//   dx        = (t - n mean(t n)) / sqrt(mean(x^2) + eps),  t = scale gate (o + post) g
//
// Bound by memory: x and the residual are read and h and y written once
// forward; x, h, dy and dh are read and dx and dresidual written backward.
//
// Column sums.  The rows are dealt to chunks in order.  A chunk holds whole
// gate rows, which it finishes itself, and at most two it shares with its
// neighbours (its first and its last), whose A it leaves in the workspace; a
// last kernel adds dpre's and dpost's partial sums and those shared A in the
// order of the chunks.  So every sum has one order, whatever the gate's
// shape, and no atomics.
#include "row_ladder.cuh"

namespace flb200 {
namespace {

// Column counters are ints, and a loop's last step passes the row's end by up
// to 4 turns of 512 threads of 8 elements.
constexpr int64_t kMaxCols = 0x7fff0000;

struct Sandwich {
  const void *x, *res, *post, *pre, *gate;
  int64_t ldx, ldr;
  void *y, *h;
  uint32_t rows, per_gate;
  int cols;
  float eps, scale, off;
  // backward
  const void *dy, *dh, *hs;
  int64_t ldy, ldh, lds;
  void *dx, *dres, *dpost, *dpre, *dgate;
  float* parts;    // [n_parts][2][cols]: dpre, dpost
  float* shared;   // [chunks][2][cols]: A of the first and of the last gate row
  float4* stats;   // [rows]: 1/rms(x), 1/rms(h), mean(dy w m)
  uint32_t chunks, per_chunk, n_parts;
};

template <typename T>
__device__ __forceinline__ const T* gate_row(const Sandwich& a, uint32_t row) {
  return a.gate == nullptr ? nullptr : static_cast<const T*>(a.gate) + (int64_t)(row / a.per_gate) * a.cols;
}

// A 16-byte pack as fp32 pairs and back.
template <typename T>
struct Pairs {
  static constexpr int P = Elem<T>::kVec / 2;
  uint64_t v[P];
  __device__ __forceinline__ Pairs() {}
  __device__ __forceinline__ explicit Pairs(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (std::is_same<T, float>::value) {
      v[0] = f2_make(__uint_as_float(w[0]), __uint_as_float(w[1]));
      v[1] = f2_make(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
#pragma unroll
      for (int p = 0; p < P; ++p) v[p] = pair_from_bits<T>(w[p]);
    }
  }
  __device__ __forceinline__ uint4 bits() const {
    if constexpr (std::is_same<T, float>::value) {
      return make_uint4(__float_as_uint(f2_lo(v[0])), __float_as_uint(f2_hi(v[0])), __float_as_uint(f2_lo(v[1])),
                        __float_as_uint(f2_hi(v[1])));
    } else {
      return make_uint4(pair_to_bits<T>(v[0]), pair_to_bits<T>(v[1]), pair_to_bits<T>(v[2]), pair_to_bits<T>(v[3]));
    }
  }
};
__device__ __forceinline__ uint64_t both(float x) { return f2_make(x, x); }

// Barrier of a team's warps.  Its number is a constant in the instruction: a
// kernel whose barrier stands in a register holds all 16, of which an SM has
// enough for four CTAs.
template <int TPR, int BLOCK>
__device__ __forceinline__ void team_barrier(int team) {
  if constexpr (BLOCK == TPR) {
    __syncthreads();
  } else {
    static_assert(BLOCK / TPR <= 4, "barriers 1 to 4");
    if (team == 0) asm volatile("bar.sync 1, %0;" ::"n"(TPR) : "memory");
    else if (team == 1) asm volatile("bar.sync 2, %0;" ::"n"(TPR) : "memory");
    else if (team == 2) asm volatile("bar.sync 3, %0;" ::"n"(TPR) : "memory");
    else asm volatile("bar.sync 4, %0;" ::"n"(TPR) : "memory");
  }
}

// Sums of K values over the TPR threads of a row or team (TPR a power of two;
// from 64 on its warps meet at named barrier 1 + team), into every thread, in
// warp order.  One barrier: consecutive calls use different halves of `buf`,
// so that no warp overwrites what another still reads.
template <int TPR, int BLOCK, int K>
__device__ __forceinline__ void team_sum(float (&v)[K], float4* buf, int half) {
  static_assert(K <= 4, "a float4 of values");
#pragma unroll
  for (int off = (TPR < 32 ? TPR : 32) / 2; off > 0; off >>= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
  }
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int team = threadIdx.x / TPR;
    if constexpr (K == 1) {
      float* h = reinterpret_cast<float*>(buf + half * (BLOCK / 32));
      if ((threadIdx.x & 31) == 0) h[threadIdx.x >> 5] = v[0];
      team_barrier<TPR, BLOCK>(team);
      v[0] = h[team * W];
#pragma unroll
      for (int i = 1; i < W; ++i) v[0] += h[team * W + i];
    } else {
      float4* h = buf + half * (BLOCK / 32);
      if ((threadIdx.x & 31) == 0)
        h[threadIdx.x >> 5] = make_float4(v[0], v[1], K > 2 ? v[K > 2 ? 2 : 0] : 0.f, K > 3 ? v[K > 3 ? 3 : 0] : 0.f);
      team_barrier<TPR, BLOCK>(team);
      float4 t = h[team * W];
#pragma unroll
      for (int i = 1; i < W; ++i) {
        const float4 o = h[team * W + i];
        t.x += o.x, t.y += o.y, t.z += o.z, t.w += o.w;
      }
      v[0] = t.x, v[1] = t.y;
      if constexpr (K > 2) v[2] = t.z;
      if constexpr (K > 3) v[3] = t.w;
    }
  }
}

// Row in registers: TPR threads, VPT packs of x each; h stays fp32.  65536 x
// 4096 bf16: 348 us at first, 382 us over seconds.  Faster arithmetic is
// slower here: with rsqrtf for the IEEE square root and division, and one
// barrier a sum for two, the same launch takes 383 to 401 us at first, whatever
// the order of its stores; why was not found.
template <typename T, int TPR, int VPT, int BLOCK>
__global__ void __launch_bounds__(BLOCK, ladder_min_blocks<BLOCK>())
sandwich_vec_kernel(const __grid_constant__ Sandwich a) {
  pdl_prologue();
  constexpr int VW = Elem<T>::kVec, P = VW / 2;
  __shared__ float4 sums[2 * BLOCK / 32];
  const int lane = threadIdx.x % TPR;
  const uint64_t row64 = (uint64_t)blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR;
  const bool ok = row64 < a.rows;
  const uint32_t row = ok ? (uint32_t)row64 : a.rows - 1;
  const int nvec = a.cols / VW;
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  const T* rr = static_cast<const T*>(a.res) + row * a.ldr;
  const T* gr = gate_row<T>(a, row);
  uint4 x[VPT], r[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    const bool in = ok && vi < nvec;
    x[i] = in ? ld_stream(xr + (int64_t)vi * VW) : make_uint4(0, 0, 0, 0);
    r[i] = in ? ld_stream(rr + (int64_t)vi * VW) : make_uint4(0, 0, 0, 0);
  }
  uint64_t s2 = both(0.f);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const Pairs<T> f(x[i]);
#pragma unroll
    for (int p = 0; p < P; ++p) s2 = f2_fma(f.v[p], f.v[p], s2);
  }
  float ss[1] = {f2_lo(s2) + f2_hi(s2)};
  ss[0] = row_reduce<SumOp, TPR, BLOCK>(ss[0], reinterpret_cast<float*>(sums));
  const uint64_t rx = both(a.scale / sqrtf(ss[0] / (float)a.cols + a.eps)), off = both(a.off);
  Pairs<T> h[VPT];
  s2 = both(0.f);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    if (!ok || vi >= nvec) continue;
    Pairs<T> f(opaque(x[i]));
    const Pairs<T> w(ld_cached(static_cast<const T*>(a.post) + (int64_t)vi * VW));
#pragma unroll
    for (int p = 0; p < P; ++p) f.v[p] = f2_mul(f2_mul(f.v[p], rx), f2_add(w.v[p], off));
    if (gr != nullptr) {
      const Pairs<T> g(ld_cached(gr + (int64_t)vi * VW));
#pragma unroll
      for (int p = 0; p < P; ++p) f.v[p] = f2_mul(f.v[p], g.v[p]);
    }
    const Pairs<T> q(r[i]);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      h[i].v[p] = f2_add(f.v[p], q.v[p]);
      s2 = f2_fma(h[i].v[p], h[i].v[p], s2);
    }
    st_stream(static_cast<T*>(a.h) + (int64_t)row * a.cols + (int64_t)vi * VW, h[i].bits());
  }
  ss[0] = f2_lo(s2) + f2_hi(s2);
  ss[0] = row_reduce<SumOp, TPR, BLOCK>(ss[0], reinterpret_cast<float*>(sums));
  const uint64_t rh = both(1.0f / sqrtf(ss[0] / (float)a.cols + a.eps));
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    if (!ok || vi >= nvec) continue;
    Pairs<T> w(ld_cached(static_cast<const T*>(a.pre) + (int64_t)vi * VW));
#pragma unroll
    for (int p = 0; p < P; ++p) w.v[p] = f2_mul(f2_mul(h[i].v[p], rh), f2_add(w.v[p], off));
    st_stream(static_cast<T*>(a.y) + (int64_t)row * a.cols + (int64_t)vi * VW, w.bits());
  }
}

// The same rows staged in shared memory: resident CTAs take every gridDim-th
// row, each thread the same VPT packs of every row; the next row's x and
// residual are copied in by cp.async while this one is worked on, and the
// weights stay in registers.  The gate row does while it lasts: a gate a channel
// for good, one a sequence for its rows over the grid's; one a token is loaded
// for every row when the row's turn comes.  65536 x 4096 bf16: 338 us over
// seconds (6.4 TB/s) with three CTAs an SM; two 414 us, four 367 us.
template <int TPR, int VPT>
constexpr int staged_ctas() {
  return VPT > 2 ? 1 : TPR >= 512 ? 2 : 768 / TPR;
}
template <typename T, int TPR, int VPT>
__global__ void __launch_bounds__(TPR, staged_ctas<TPR, VPT>())
sandwich_staged_kernel(const __grid_constant__ Sandwich a) {
  pdl_prologue();
  constexpr int VW = Elem<T>::kVec, P = VW / 2;
  constexpr int STAGE = 2 * VPT * TPR;
  extern __shared__ uint4 dyn[];
  __shared__ float4 sums[2 * TPR / 32];
  uint4* stage = dyn + threadIdx.x;
  const int lane = threadIdx.x;
  const int nvec = a.cols / VW;
  const float inv_n = 1.f / (float)a.cols;
  const uint64_t off = both(a.off);
  uint4 post[VPT], pre[VPT], gate[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = min(lane + i * TPR, nvec - 1);
    post[i] = ld_cached(static_cast<const T*>(a.post) + (int64_t)vi * VW);
    pre[i] = ld_cached(static_cast<const T*>(a.pre) + (int64_t)vi * VW);
  }
  auto fetch = [&](uint32_t row, int st) {
    const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
    const T* rr = static_cast<const T*>(a.res) + row * a.ldr;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int vi = lane + i * TPR;
      if (vi < nvec) {
        cp_async16(stage + st * STAGE + i * TPR, xr + (int64_t)vi * VW);
        cp_async16(stage + st * STAGE + (VPT + i) * TPR, rr + (int64_t)vi * VW);
      }
    }
    cp_async_commit();
  };
  uint32_t row = blockIdx.x;
  fetch(row, 0);
  uint32_t seg = 0xffffffffu;
  int st = 0;
  for (; row < a.rows; row += gridDim.x, st ^= 1) {
    if (row + gridDim.x < a.rows) {
      fetch(row + gridDim.x, st ^ 1);
      cp_async_wait_pending<1>();
    } else {
      cp_async_wait_all();
    }
    const uint4* in = stage + st * STAGE;
    if (a.gate != nullptr && row / a.per_gate != seg) {
      seg = row / a.per_gate;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        gate[i] = ld_cached(static_cast<const T*>(a.gate) + (int64_t)seg * a.cols + (int64_t)min(lane + i * TPR, nvec - 1) * VW);
    }
    uint64_t s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (lane + i * TPR >= nvec) continue;
      const Pairs<T> f(in[i * TPR]);
#pragma unroll
      for (int p = 0; p < P; ++p) s2 = f2_fma(f.v[p], f.v[p], s2);
    }
    float ss[1] = {f2_lo(s2) + f2_hi(s2)};
    team_sum<TPR, TPR>(ss, sums, 0);
    const uint64_t rx = both(a.scale * rsqrtf(fmaf(ss[0], inv_n, a.eps)));
    Pairs<T> h[VPT];
    s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int vi = lane + i * TPR;
      if (vi >= nvec) continue;
      Pairs<T> f(in[i * TPR]);
      const Pairs<T> w(opaque(post[i]));
#pragma unroll
      for (int p = 0; p < P; ++p) f.v[p] = f2_mul(f2_mul(f.v[p], rx), f2_add(w.v[p], off));
      if (a.gate != nullptr) {
        const Pairs<T> g(opaque(gate[i]));
#pragma unroll
        for (int p = 0; p < P; ++p) f.v[p] = f2_mul(f.v[p], g.v[p]);
      }
      const Pairs<T> q(in[(VPT + i) * TPR]);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        h[i].v[p] = f2_add(f.v[p], q.v[p]);
        s2 = f2_fma(h[i].v[p], h[i].v[p], s2);
      }
      st_stream(static_cast<T*>(a.h) + (int64_t)row * a.cols + (int64_t)vi * VW, h[i].bits());
    }
    ss[0] = f2_lo(s2) + f2_hi(s2);
    team_sum<TPR, TPR>(ss, sums, 1);
    const uint64_t rh = both(rsqrtf(fmaf(ss[0], inv_n, a.eps)));
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int vi = lane + i * TPR;
      if (vi >= nvec) continue;
      Pairs<T> w(opaque(pre[i]));
#pragma unroll
      for (int p = 0; p < P; ++p) w.v[p] = f2_mul(f2_mul(h[i].v[p], rh), f2_add(w.v[p], off));
      st_stream(static_cast<T*>(a.y) + (int64_t)row * a.cols + (int64_t)vi * VW, w.bits());
    }
  }
}

// VEC elements (a 16-byte pack, two, or one) as fp32 and back.
template <typename T>
struct alignas(2 * sizeof(T)) Two {
  T v[2];
};
template <typename T, int VEC>
__device__ __forceinline__ void get(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = Elem<T>::to_f(*p);
  } else if constexpr (VEC == 2) {
    const Two<T> u = *reinterpret_cast<const Two<T>*>(p);
    f[0] = Elem<T>::to_f(u.v[0]), f[1] = Elem<T>::to_f(u.v[1]);
  } else {
    unpack<T>(ld_plain(p), f);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void put(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) *p = Elem<T>::from_f(f[0]);
  else if constexpr (VEC == 2) *reinterpret_cast<Two<T>*>(p) = Two<T>{{Elem<T>::from_f(f[0]), Elem<T>::from_f(f[1])}};
  else st_stream(p, pack<T>(f));
}

// Rows of any length (VEC a pack) and alignment (VEC 2, 1): TPR threads a row, x
// and the residual read again from cache.
template <typename T, int VEC, int TPR>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR)
sandwich_loop_kernel(const __grid_constant__ Sandwich a) {
  pdl_prologue();
  constexpr int BLOCK = TPR < 128 ? 128 : TPR, TEAMS = BLOCK / TPR;
  __shared__ float4 sums[2 * BLOCK / 32];
  const T *post = static_cast<const T*>(a.post), *pre = static_cast<const T*>(a.pre);
  const int lane = threadIdx.x % TPR * VEC;
  const float inv_n = 1.f / (float)a.cols;
  for (uint32_t row = blockIdx.x * TEAMS + threadIdx.x / TPR; row < a.rows; row += gridDim.x * TEAMS) {
    const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
    const T* rr = static_cast<const T*>(a.res) + row * a.ldr;
    const T* gr = gate_row<T>(a, row);
    T* hr = static_cast<T*>(a.h) + (int64_t)row * a.cols;
    T* yr = static_cast<T*>(a.y) + (int64_t)row * a.cols;
    float ss[1] = {0.f};
#pragma unroll 4
    for (int c = lane; c < a.cols; c += TPR * VEC) {
      float f[VEC];
      get<T, VEC>(xr + c, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss[0] = fmaf(f[e], f[e], ss[0]);
    }
    team_sum<TPR, BLOCK>(ss, sums, 0);
    const float rx = a.scale * rsqrtf(fmaf(ss[0], inv_n, a.eps));
    auto sum_of = [&](int c, float (&f)[VEC]) {
      float w[VEC];
      get<T, VEC>(xr + c, f);
      get<T, VEC>(post + c, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = f[e] * rx * (w[e] + a.off);
      if (gr != nullptr) {
        get<T, VEC>(gr + c, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] *= w[e];
      }
      get<T, VEC>(rr + c, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] += w[e];
    };
    ss[0] = 0.f;
#pragma unroll 2
    for (int c = lane; c < a.cols; c += TPR * VEC) {
      float f[VEC];
      sum_of(c, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss[0] = fmaf(f[e], f[e], ss[0]);
      put<T, VEC>(hr + c, f);
    }
    team_sum<TPR, BLOCK>(ss, sums, 1);
    const float rh = rsqrtf(fmaf(ss[0], inv_n, a.eps));
#pragma unroll 2
    for (int c = lane; c < a.cols; c += TPR * VEC) {
      float f[VEC], w[VEC];
      sum_of(c, f);
      get<T, VEC>(pre + c, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = f[e] * rh * (w[e] + a.off);
      put<T, VEC>(yr + c, f);
    }
  }
}

// ------------------------------------------------------------- backward ---
// Rows of any length and alignment: the row gradients and the row's
// statistics, then the column sums in a second pass over the operands.
template <typename T, int VEC, int TPR>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR)
sandwich_bwd_rows_kernel(const __grid_constant__ Sandwich a) {
  pdl_prologue();
  constexpr int BLOCK = TPR < 128 ? 128 : TPR, TEAMS = BLOCK / TPR;
  __shared__ float4 sums[2 * BLOCK / 32];
  const T *post = static_cast<const T*>(a.post), *pre = static_cast<const T*>(a.pre);
  const int lane = threadIdx.x % TPR * VEC;
  const float inv_n = 1.f / (float)a.cols;
  for (uint32_t row = blockIdx.x * TEAMS + threadIdx.x / TPR; row < a.rows; row += gridDim.x * TEAMS) {
    const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
    const T* hr = static_cast<const T*>(a.hs) + row * a.lds;
    const T* dyr = static_cast<const T*>(a.dy) + row * a.ldy;
    const T* dhr = a.dh == nullptr ? nullptr : static_cast<const T*>(a.dh) + row * a.ldh;
    const T* gr = gate_row<T>(a, row);
    float v[3] = {0.f, 0.f, 0.f};
#pragma unroll 2
    for (int c = lane; c < a.cols; c += TPR * VEC) {
      float x[VEC], h[VEC], d[VEC], w[VEC];
      get<T, VEC>(xr + c, x);
      get<T, VEC>(hr + c, h);
      get<T, VEC>(dyr + c, d);
      get<T, VEC>(pre + c, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[0] = fmaf(x[e], x[e], v[0]);
        v[1] = fmaf(h[e], h[e], v[1]);
        v[2] = fmaf(d[e] * (w[e] + a.off), h[e], v[2]);
      }
    }
    team_sum<TPR, BLOCK>(v, sums, 0);
    const float rx = rsqrtf(fmaf(v[0], inv_n, a.eps)), rh = rsqrtf(fmaf(v[1], inv_n, a.eps));
    const float mean = v[2] * rh * inv_n;
    auto grad = [&](int c, float (&g)[VEC]) {
      float h[VEC], w[VEC];
      get<T, VEC>(dyr + c, g);
      get<T, VEC>(hr + c, h);
      get<T, VEC>(pre + c, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) g[e] = rh * (g[e] * (w[e] + a.off) - h[e] * rh * mean);
      if (dhr != nullptr) {
        get<T, VEC>(dhr + c, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[e] += w[e];
      }
    };
    auto weigh = [&](int c, float (&g)[VEC]) {
      float w[VEC];
      get<T, VEC>(post + c, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) g[e] *= a.scale * (w[e] + a.off);
      if (gr != nullptr) {
        get<T, VEC>(gr + c, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[e] *= w[e];
      }
    };
    float u[1] = {0.f};
#pragma unroll 2
    for (int c = lane; c < a.cols; c += TPR * VEC) {
      float g[VEC], x[VEC];
      grad(c, g);
      put<T, VEC>(static_cast<T*>(a.dres) + (int64_t)row * a.cols + c, g);
      weigh(c, g);
      get<T, VEC>(xr + c, x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) u[0] = fmaf(g[e], x[e], u[0]);
    }
    team_sum<TPR, BLOCK>(u, sums, 1);
    const float back = rx * rx * (u[0] * rx * inv_n);
#pragma unroll 2
    for (int c = lane; c < a.cols; c += TPR * VEC) {
      float g[VEC], x[VEC];
      grad(c, g);
      weigh(c, g);
      get<T, VEC>(xr + c, x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) g[e] = rx * g[e] - x[e] * back;
      put<T, VEC>(static_cast<T*>(a.dx) + (int64_t)row * a.cols + c, g);
    }
    if (lane == 0) a.stats[row] = make_float4(rx, rh, mean, 0.f);
  }
}

// A thread VEC columns of a chunk of rows (blockIdx.y).
template <typename T, int VEC>
__global__ void __launch_bounds__(128)
sandwich_bwd_cols_kernel(const __grid_constant__ Sandwich a) {
  pdl_prologue();
  const int c = (blockIdx.x * 128 + threadIdx.x) * VEC;
  if (c >= a.cols) return;
  const uint32_t chunk = blockIdx.y;
  const uint32_t r0 = chunk * a.per_chunk, r1 = min(a.rows, r0 + a.per_chunk);
  float pre[VEC], dpre[VEC], dpost[VEC], sum[VEC];
  get<T, VEC>(static_cast<const T*>(a.pre) + c, pre);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    pre[e] += a.off;
    dpre[e] = dpost[e] = sum[e] = 0.f;
  }
  uint32_t row = r0;
  while (row < r1) {  // one gate row a turn
    const uint32_t seg = row / a.per_gate;
    const uint64_t seg_end = (uint64_t)(seg + 1) * a.per_gate;
    const uint32_t end = seg_end < r1 ? (uint32_t)seg_end : r1;
    const bool whole = (uint64_t)seg * a.per_gate >= r0 && (seg_end <= r1 || (r1 == a.rows));
    const bool is_first = seg == r0 / a.per_gate;
#pragma unroll(VEC <= 2 ? 4 : 2)
    for (; row < end; ++row) {
      const float4 s = a.stats[row];
      float dy[VEC], m[VEC], x[VEC], g[VEC];
      get<T, VEC>(static_cast<const T*>(a.dy) + row * a.ldy + c, dy);
      get<T, VEC>(static_cast<const T*>(a.hs) + row * a.lds + c, m);
      get<T, VEC>(static_cast<const T*>(a.x) + row * a.ldx + c, x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        m[e] *= s.y;
        g[e] = s.y * (dy[e] * pre[e] - m[e] * s.z);
        dpre[e] = fmaf(dy[e], m[e], dpre[e]);
      }
      if (a.dh != nullptr) {
        get<T, VEC>(static_cast<const T*>(a.dh) + row * a.ldh + c, m);
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[e] += m[e];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] = fmaf(g[e], x[e] * s.x, sum[e]);
    }
    if (a.gate != nullptr) {
      const int64_t at = (int64_t)seg * a.cols + c;
      float g[VEC], w[VEC];
      get<T, VEC>(static_cast<const T*>(a.gate) + at, g);
      get<T, VEC>(static_cast<const T*>(a.post) + c, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        dpost[e] = fmaf(a.scale * g[e], sum[e], dpost[e]);
        w[e] = a.scale * (w[e] + a.off) * sum[e];
      }
      if (whole) {
        put<T, VEC>(static_cast<T*>(a.dgate) + at, w);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) a.shared[((int64_t)chunk * 2 + (is_first ? 0 : 1)) * a.cols + c + e] = sum[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) dpost[e] = a.scale * sum[e];
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
  }
  const int64_t at = (int64_t)chunk * 2 * a.cols + c;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    a.parts[at + e] = dpre[e];
    a.parts[at + a.cols + e] = dpost[e];
  }
}

// Adds the chunks' partial sums: blockIdx.y == 0 dpre and dpost, y > 0 a gate
// row that chunks share, if there is one: gate row y - 1, or, of more gate
// rows than chunks, the one that begins in chunk y - 1 and reaches into the
// next.  32 columns a CTA, 16 threads a column.
template <typename T>
__global__ void __launch_bounds__(512)
sandwich_bwd_sum_kernel(const __grid_constant__ Sandwich a, int by_gate) {
  pdl_prologue();
  __shared__ float part[2][16][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  const int64_t stride = 2ll * a.cols;
  uint32_t from = 0, to = a.n_parts, seg = 0;
  uint64_t begin = 0;
  if (blockIdx.y > 0) {
    seg = by_gate ? blockIdx.y - 1 : blockIdx.y * a.per_chunk / a.per_gate;
    begin = (uint64_t)seg * a.per_gate;
    from = (uint32_t)(begin / a.per_chunk);
    to = (uint32_t)((min((uint64_t)a.rows, begin + a.per_gate) - 1) / a.per_chunk) + 1;
    if (to - from < 2 || (!by_gate && from != blockIdx.y - 1)) return;  // (the whole CTA)
  }
  float s0 = 0.f, s1 = 0.f;
  if (c < a.cols) {
    if (blockIdx.y == 0) {
#pragma unroll 8
      for (uint32_t k = ty; k < to; k += 16) {
        s0 += a.parts[k * stride + c];
        s1 += a.parts[k * stride + a.cols + c];
      }
    } else {
      // the last gate row of the chunk it begins in (its first where both begin
      // together), the first of the others
#pragma unroll 8
      for (uint32_t k = from + ty; k < to; k += 16)
        s0 += a.shared[k * stride + (k == from && begin != (uint64_t)from * a.per_chunk ? a.cols : 0) + c];
    }
  }
  part[0][ty][tx] = s0;
  part[1][ty][tx] = s1;
  __syncthreads();
  if (ty != 0 || c >= a.cols) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) {
    s0 += part[0][k][tx];
    s1 += part[1][k][tx];
  }
  if (blockIdx.y == 0) {
    static_cast<T*>(a.dpre)[c] = Elem<T>::from_f(s0);
    static_cast<T*>(a.dpost)[c] = Elem<T>::from_f(s1);
  } else {
    const float post = a.scale * (Elem<T>::to_f(static_cast<const T*>(a.post)[c]) + a.off);
    static_cast<T*>(a.dgate)[(int64_t)seg * a.cols + c] = Elem<T>::from_f(post * s0);
  }
}

// Rows staged in shared memory: a team of TPR threads takes a chunk of rows,
// each thread the same VPT packs of every row, whose column sums it holds in
// registers.  The next row's x, h, dy and dh are copied in by cp.async while
// this one is worked on (a thread reads only what it copied, so no barrier
// orders them).  Two barriers a row, for the two sums that hang together.
// dpost's sums, which only the end of a gate row adds to, lie in shared
// memory, and so do the weights as fp32 (converted from their own type for
// every row they took a third of the instructions).
template <typename T, int TPR, int VPT, int BLOCK>
__global__ void __launch_bounds__(BLOCK, BLOCK <= 256 ? 2 : 1)
sandwich_bwd_kernel(const __grid_constant__ Sandwich a) {
  pdl_prologue();
  constexpr int VW = Elem<T>::kVec, P = VW / 2;
  constexpr int TEAMS = BLOCK / TPR;
  constexpr int STAGE = 4 * VPT * BLOCK;  // packs
  extern __shared__ uint4 dyn[];
  __shared__ float4 sums[2 * BLOCK / 32];
  uint4* stage = dyn + threadIdx.x;  // [stage][array][i][thread]
  // dpost's sums, o + pre, and scale * gate * (o + post) of the gate row: pairs
  // 2 k and 2 k + 1 of pack i at [i][k][thread]
  constexpr int QUADS = VPT * (VW / 4) * BLOCK;
  ulonglong2* dpost = reinterpret_cast<ulonglong2*>(dyn + 2 * STAGE) + threadIdx.x;
  ulonglong2 *pre = dpost + QUADS, *post = pre + QUADS;
  const int lane = threadIdx.x % TPR;
  const uint32_t chunk = blockIdx.x * TEAMS + threadIdx.x / TPR;
  const int nvec = a.cols / VW;
  const float inv_n = 1.f / (float)a.cols;
  const uint32_t r0 = min(a.rows, chunk * a.per_chunk), r1 = min(a.rows, r0 + a.per_chunk);
  const uint64_t off = both(a.off), zero = both(0.f);
  uint64_t dpre[VPT][P], sum[VPT][P];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    const Pairs<T> w(vi < nvec ? ld_cached(static_cast<const T*>(a.pre) + (int64_t)vi * VW) : make_uint4(0, 0, 0, 0));
#pragma unroll
    for (int p = 0; p < P; ++p) dpre[i][p] = sum[i][p] = zero;
#pragma unroll
    for (int k = 0; k < P / 2; ++k) {
      dpost[(i * (P / 2) + k) * BLOCK] = make_ulonglong2(zero, zero);
      pre[(i * (P / 2) + k) * BLOCK] = make_ulonglong2(f2_add(w.v[2 * k], off), f2_add(w.v[2 * k + 1], off));
    }
  }
  auto fetch = [&](uint32_t row, int st) {
    const T* src[4] = {static_cast<const T*>(a.x) + row * a.ldx, static_cast<const T*>(a.hs) + row * a.lds,
                       static_cast<const T*>(a.dy) + row * a.ldy,
                       a.dh == nullptr ? nullptr : static_cast<const T*>(a.dh) + row * a.ldh};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (src[k] == nullptr) continue;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int vi = lane + i * TPR;
        if (vi < nvec) cp_async16(stage + st * STAGE + (k * VPT + i) * BLOCK, src[k] + (int64_t)vi * VW);
      }
    }
    cp_async_commit();
  };
  if (r0 < r1) fetch(r0, 0);
  uint32_t seg = r0 / a.per_gate;
  uint64_t seg_end = (uint64_t)(seg + 1) * a.per_gate;
  bool first_seg = true, fresh = true;
  for (uint32_t row = r0; row < r1; ++row) {
    const int st = (row - r0) & 1;
    if (row + 1 < r1) {
      fetch(row + 1, st ^ 1);
      cp_async_wait_pending<1>();
    } else {
      cp_async_wait_all();
    }
    const uint4* in = stage + st * STAGE;
    const T* gr = a.gate == nullptr ? nullptr : static_cast<const T*>(a.gate) + (int64_t)seg * a.cols;
    if (fresh) {  // a gate row begins
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int vi = lane + i * TPR;
        if (vi >= nvec) continue;
        Pairs<T> w(ld_cached(static_cast<const T*>(a.post) + (int64_t)vi * VW));
#pragma unroll
        for (int p = 0; p < P; ++p) w.v[p] = f2_mul(f2_add(w.v[p], off), both(a.scale));
        if (gr != nullptr) {
          const Pairs<T> g(ld_cached(gr + (int64_t)vi * VW));
#pragma unroll
          for (int p = 0; p < P; ++p) w.v[p] = f2_mul(w.v[p], g.v[p]);
        }
#pragma unroll
        for (int k = 0; k < P / 2; ++k) post[(i * (P / 2) + k) * BLOCK] = make_ulonglong2(w.v[2 * k], w.v[2 * k + 1]);
      }
      fresh = false;
    }
    uint64_t vx = zero, vh = zero, vd = zero;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (lane + i * TPR >= nvec) continue;
      const Pairs<T> x(in[i * BLOCK]), h(in[(VPT + i) * BLOCK]), dy(in[(2 * VPT + i) * BLOCK]);
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        const ulonglong2 w = pre[(i * (P / 2) + k) * BLOCK];
        vd = f2_fma(f2_mul(dy.v[2 * k], w.x), h.v[2 * k], vd);
        vd = f2_fma(f2_mul(dy.v[2 * k + 1], w.y), h.v[2 * k + 1], vd);
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        vx = f2_fma(x.v[p], x.v[p], vx);
        vh = f2_fma(h.v[p], h.v[p], vh);
      }
    }
    float v[3] = {f2_lo(vx) + f2_hi(vx), f2_lo(vh) + f2_hi(vh), f2_lo(vd) + f2_hi(vd)};
    team_sum<TPR, BLOCK>(v, sums, 0);
    const float rx = rsqrtf(fmaf(v[0], inv_n, a.eps)), rh = rsqrtf(fmaf(v[1], inv_n, a.eps));
    const uint64_t rx2 = both(rx), rh2 = both(rh), mean2 = both(-(v[2] * rh * inv_n));
    uint64_t t[VPT][P], vt = zero;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int vi = lane + i * TPR;
      if (vi >= nvec) continue;
      const Pairs<T> h(in[(VPT + i) * BLOCK]), dy(in[(2 * VPT + i) * BLOCK]);
      Pairs<T> g;
      if (a.dh != nullptr) {
        g = Pairs<T>(in[(3 * VPT + i) * BLOCK]);
      } else {
#pragma unroll
        for (int p = 0; p < P; ++p) g.v[p] = zero;
      }
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        const ulonglong2 w = pre[(i * (P / 2) + k) * BLOCK];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int p = 2 * k + q;
          const uint64_t m = f2_mul(h.v[p], rh2);
          dpre[i][p] = f2_fma(dy.v[p], m, dpre[i][p]);
          g.v[p] = f2_fma(rh2, f2_fma(m, mean2, f2_mul(dy.v[p], q ? w.y : w.x)), g.v[p]);
        }
      }
      st_stream(static_cast<T*>(a.dres) + (int64_t)row * a.cols + (int64_t)vi * VW, g.bits());
      const Pairs<T> x(in[i * BLOCK]);
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        const ulonglong2 w = post[(i * (P / 2) + k) * BLOCK];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int p = 2 * k + q;
          sum[i][p] = f2_fma(g.v[p], f2_mul(x.v[p], rx2), sum[i][p]);
          t[i][p] = f2_mul(g.v[p], q ? w.y : w.x);
          vt = f2_fma(t[i][p], x.v[p], vt);
        }
      }
    }
    float u[1] = {f2_lo(vt) + f2_hi(vt)};
    team_sum<TPR, BLOCK>(u, sums, 1);
    // rx (t - n mean(t n)) with n = x rx
    const uint64_t back = both(-(rx * rx * (u[0] * rx * inv_n)));
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int vi = lane + i * TPR;
      if (vi >= nvec) continue;
      Pairs<T> x(in[i * BLOCK]);
#pragma unroll
      for (int p = 0; p < P; ++p) x.v[p] = f2_fma(x.v[p], back, f2_mul(t[i][p], rx2));
      st_stream(static_cast<T*>(a.dx) + (int64_t)row * a.cols + (int64_t)vi * VW, x.bits());
    }
    if (row + 1 == seg_end || row + 1 == r1) {  // the gate row ends, or the chunk
      const bool whole = (uint64_t)seg * a.per_gate >= r0 && (row + 1 == seg_end || r1 == a.rows);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int vi = lane + i * TPR;
        if (vi >= nvec) continue;
        const int64_t c = (int64_t)vi * VW;
        Pairs<T> g;
        if (gr != nullptr) {
          g = Pairs<T>(ld_cached(gr + c));
          if (whole) {
            Pairs<T> w(ld_cached(static_cast<const T*>(a.post) + c));
#pragma unroll
            for (int p = 0; p < P; ++p) w.v[p] = f2_mul(f2_mul(f2_add(w.v[p], off), both(a.scale)), sum[i][p]);
            st_stream(static_cast<T*>(a.dgate) + (int64_t)seg * a.cols + c, w.bits());
          } else {
            float* sh = a.shared + ((int64_t)chunk * 2 + (first_seg ? 0 : 1)) * a.cols + c;
#pragma unroll
            for (int p = 0; p < P; ++p) {
              sh[2 * p] = f2_lo(sum[i][p]);
              sh[2 * p + 1] = f2_hi(sum[i][p]);
            }
          }
        } else {
#pragma unroll
          for (int p = 0; p < P; ++p) g.v[p] = both(1.f);
        }
#pragma unroll
        for (int k = 0; k < P / 2; ++k) {
          ulonglong2& d = dpost[(i * (P / 2) + k) * BLOCK];
          d = make_ulonglong2(f2_fma(f2_mul(g.v[2 * k], both(a.scale)), sum[i][2 * k], d.x),
                              f2_fma(f2_mul(g.v[2 * k + 1], both(a.scale)), sum[i][2 * k + 1], d.y));
        }
#pragma unroll
        for (int p = 0; p < P; ++p) sum[i][p] = zero;
      }
      first_seg = false;
      fresh = true;
      ++seg;
      seg_end += a.per_gate;
    }
  }
  // the CTA's partial sums: its teams' in order
  float* part = a.parts + (int64_t)blockIdx.x * 2 * a.cols;
  if constexpr (TEAMS > 1) {
    // dpre laid out as dpost, over the stages that nothing is on its way to any more
    ulonglong2* all = reinterpret_cast<ulonglong2*>(dyn);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int k = 0; k < P / 2; ++k)
        all[(i * (P / 2) + k) * BLOCK + threadIdx.x] = make_ulonglong2(dpre[i][2 * k], dpre[i][2 * k + 1]);
    __syncthreads();
    const float *dp = reinterpret_cast<const float*>(dyn), *dq = reinterpret_cast<const float*>(dyn + 2 * STAGE);
    for (int c = threadIdx.x; c < a.cols; c += BLOCK) {
      const int vi = c / VW;
      const int at = (((vi / TPR) * (P / 2) + c % VW / 4) * BLOCK + vi % TPR) * 4 + c % 4;
      float p = 0.f, q = 0.f;
      for (int k = 0; k < TEAMS; ++k) {
        p += dp[at + k * TPR * 4];
        q += dq[at + k * TPR * 4];
      }
      part[c] = p;
      part[a.cols + c] = q;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int vi = lane + i * TPR;
      if (vi >= nvec) continue;
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        const ulonglong2 d = dpost[(i * (P / 2) + k) * BLOCK];
        const int c = vi * VW + 4 * k;
        *reinterpret_cast<float4*>(part + c) = make_float4(f2_lo(dpre[i][2 * k]), f2_hi(dpre[i][2 * k]),
                                                           f2_lo(dpre[i][2 * k + 1]), f2_hi(dpre[i][2 * k + 1]));
        *reinterpret_cast<float4*>(part + a.cols + c) = make_float4(f2_lo(d.x), f2_hi(d.x), f2_lo(d.y), f2_hi(d.y));
      }
    }
  }
}

// How the column sums are dealt: `team` threads a row (0: rows by single
// elements and a second pass), chunks of rows, CTAs.
struct Plan {
  int team;
  uint32_t chunks, per_chunk, n_parts;
};
Plan deal(int64_t rows, int64_t teams, int per_cta, int team) {
  Plan p;
  p.team = team;
  p.per_chunk = (uint32_t)ceil_div(rows, std::min(rows, teams));
  p.chunks = (uint32_t)ceil_div(rows, p.per_chunk);
  p.n_parts = (uint32_t)ceil_div(p.chunks, per_cta);
  return p;
}
// Teams of 32 to 512 threads of 2 packs, as many as are resident at once (a
// CTA of 256 threads twice an SM, one of 512 once).
constexpr int kBwdVpt = 2;
Plan plan_teams(int64_t rows, int64_t packs, int sms) {
  int team = 32;
  while (team < 512 && (int64_t)team * kBwdVpt < packs) team *= 2;
  const int per_cta = team >= 256 ? 1 : 256 / team;
  return deal(rows, (int64_t)sms * (team == 512 ? 1 : 2) * per_cta, per_cta, team);
}
// About 8 CTAs an SM of 128 columns (or pairs, or packs) and at least 8 rows.
Plan plan_columns(int64_t rows, int64_t units, int sms) {
  return deal(rows, std::max<int64_t>(1, std::min(ceil_div(8ll * sms, ceil_div(std::max<int64_t>(units, 1), 128)), ceil_div(rows, 8))), 1, 0);
}
// All plans' needs (which of them a call takes hangs on its alignment too).
size_t bwd_workspace(int64_t rows, int64_t cols, int64_t packs, int sms) {
  size_t most = 0;
  for (const Plan& p : {plan_teams(rows, packs, sms), plan_columns(rows, cols, sms), plan_columns(rows, cols / 2, sms),
                        plan_columns(rows, packs, sms)})
    most = std::max(most, (size_t)p.chunks + p.n_parts);
  return (size_t)rows * sizeof(float4) + (size_t)2 * cols * sizeof(float) * most;
}

// The most elements at once that every address and stride allows: a pack, two
// or one.
template <typename T>
int width_of(int64_t cols, std::initializer_list<int64_t> strides, std::initializer_list<const void*> pointers) {
  for (const int w : {Elem<T>::kVec, 2}) {
    bool ok = cols % w == 0;
    for (const int64_t s : strides) ok = ok && s % w == 0;
    for (const void* p : pointers) ok = ok && reinterpret_cast<uintptr_t>(p) % (w * sizeof(T)) == 0;
    if (ok) return w;
  }
  return 1;
}
// Calls f(VEC, TPR) for rows read `width` elements at once: at least four of
// these a thread, up to 512 threads.
template <typename T, typename F>
void by_length(int64_t cols, int width, F&& f) {
  using std::integral_constant;
  auto threads = [&](auto vec) {
    const int64_t units = cols / decltype(vec)::value;
    if (units <= 128) f(vec, integral_constant<int, 32>{});
    else if (units <= 1024) f(vec, integral_constant<int, 128>{});
    else f(vec, integral_constant<int, 512>{});
  };
  if (width == Elem<T>::kVec) threads(integral_constant<int, Elem<T>::kVec>{});
  else if (width == 2) threads(integral_constant<int, 2>{});
  else threads(integral_constant<int, 1>{});
}

// The staged kernel where its resident CTAs have at least 8 rows each; -1: too
// few rows.
template <typename T, int TPR, int VPT>
int launch_staged(const Sandwich& a, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kCtas = staged_ctas<TPR, VPT>();
  if (a.rows < 8ll * kCtas * dev.sm_count) return -1;
  auto kern = sandwich_staged_kernel<T, TPR, VPT>;
  constexpr int smem = 2 * 2 * VPT * TPR * 16;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return launch_status();
  launch_k(kern, kCtas * dev.sm_count, TPR, smem, stream, a);
  return launch_status();
}

template <typename T>
int launch_fwd(const Sandwich& a, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int VW = Elem<T>::kVec;
  const int width = width_of<T>(a.cols, {a.ldx, a.ldr}, {a.x, a.res, a.post, a.pre, a.gate, a.y, a.h});
  if (width == VW) {
    // 4096 columns of 16 bits: 256 threads of two packs (65536 rows 346 us; 128 of four 465 us)
    const int64_t n = a.cols / VW;
    // Where staging pays, over seconds, 4.3 GB a launch, against one CTA a row
    // group: 16 bits, 192 packs 358 us (427), 512 335 (377), 640 409 (496), 1024
    // 355 (405), 1280 378 (629), 2048 342 (474); 32 bits, 1280 329 (585), 2048 358
    // (446).  Where not: 16 bits, 256 packs 387 (361); 32 bits, 512 373 (315).  The
    // other 32-bit rows of up to 1024 packs were not measured and take the latter.
    int st = -1;
    if constexpr (sizeof(T) == 2) {
      if (n > 128 && n < 256) st = launch_staged<T, 128, 2>(a, dev, stream);
      else if (n > 256 && n <= 512) st = launch_staged<T, 256, 2>(a, dev, stream);
      else if (n > 512 && n <= 1024) st = launch_staged<T, 512, 2>(a, dev, stream);
    }
    if (n > 1024 && n <= 2048) st = launch_staged<T, 512, 4>(a, dev, stream);
    if (st >= 0) return st;
    const int r = row_ladder<2>(a.cols / VW, [&](auto tpr, auto vpt) -> int {
      constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
      constexpr int BLOCK = ladder_block<TPR>();
      launch_k((sandwich_vec_kernel<T, TPR, VPT, BLOCK>), (unsigned)ceil_div(a.rows, BLOCK / TPR), BLOCK, 0, stream,
               a);
      return launch_status();
    });
    if (r >= 0) return r;
  }
  by_length<T>(a.cols, width, [&](auto vec, auto tpr) {
    constexpr int TPR = decltype(tpr)::value, BLOCK = TPR < 128 ? 128 : TPR;
    launch_k((sandwich_loop_kernel<T, decltype(vec)::value, TPR>),
             (unsigned)std::min<int64_t>(ceil_div(a.rows, BLOCK / TPR), 2048ll / BLOCK * dev.sm_count), BLOCK, 0, stream,
             a);
  });
  return launch_status();
}

template <typename T, int TPR>
int launch_teams(const Sandwich& a, cudaStream_t stream) {
  constexpr int BLOCK = TPR >= 256 ? TPR : 256;
  constexpr int VW = Elem<T>::kVec;
  // two stages of four operands; dpost's sums and the two weights in fp32
  constexpr int smem = (2 * 4 * kBwdVpt * 16 + 3 * kBwdVpt * VW * 4) * BLOCK;
  auto kern = sandwich_bwd_kernel<T, TPR, kBwdVpt, BLOCK>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return launch_status();
  launch_k(kern, a.n_parts, BLOCK, smem, stream, a);
  return launch_status();
}

template <typename T>
int launch_bwd(Sandwich a, const DeviceInfo& dev, float* ws, cudaStream_t stream) {
  constexpr int VW = Elem<T>::kVec;
  const int64_t packs = a.cols / VW;
  const int width = width_of<T>(a.cols, {a.ldx, a.lds, a.ldy, a.ldh},
                                {a.x, a.hs, a.dy, a.dh, a.post, a.pre, a.gate, a.dx, a.dres, a.dgate});
  const Plan p = width == VW && packs <= 512 * kBwdVpt ? plan_teams(a.rows, packs, dev.sm_count)
                                                       : plan_columns(a.rows, a.cols / width, dev.sm_count);
  a.chunks = p.chunks, a.per_chunk = p.per_chunk, a.n_parts = p.n_parts;
  a.parts = ws;
  a.shared = ws + (int64_t)2 * p.n_parts * a.cols;
  int st = FL_B200_OK;
  switch (p.team) {
    case 0:
      by_length<T>(a.cols, width, [&](auto vec, auto tpr) {
        constexpr int VEC = decltype(vec)::value, TPR = decltype(tpr)::value, BLOCK = TPR < 128 ? 128 : TPR;
        launch_k((sandwich_bwd_rows_kernel<T, VEC, TPR>),
                 (unsigned)std::min<int64_t>(ceil_div(a.rows, BLOCK / TPR), 2048ll / BLOCK * dev.sm_count), BLOCK, 0,
                 stream, a);
        launch_k((sandwich_bwd_cols_kernel<T, VEC>), dim3((unsigned)ceil_div(a.cols, 128 * VEC), a.chunks), 128, 0,
                 stream, a);
      });
      break;
    case 32: st = launch_teams<T, 32>(a, stream); break;
    case 64: st = launch_teams<T, 64>(a, stream); break;
    case 128: st = launch_teams<T, 128>(a, stream); break;
    case 256: st = launch_teams<T, 256>(a, stream); break;
    default: st = launch_teams<T, 512>(a, stream); break;
  }
  if (st != FL_B200_OK) return st;
  const int64_t gates = a.gate ? ceil_div(a.rows, a.per_gate) : 0;
  const int by_gate = gates < a.chunks;
  // (chunks of whole gate rows share none)
  const int64_t sums = a.per_chunk % a.per_gate == 0 ? 1 : 1 + std::min<int64_t>(gates, a.chunks - 1);
  launch_k((sandwich_bwd_sum_kernel<T>), dim3((unsigned)ceil_div(a.cols, 32), (unsigned)sums), 512, 0, stream, a, by_gate);
  return launch_status();
}

// The bytes of a row operand (stride in elements of `size` bytes).
struct Range {
  uintptr_t lo, hi;
  Range(const void* p, int64_t ld, int64_t rows, int64_t cols, int64_t size)
      : lo(reinterpret_cast<uintptr_t>(p)), hi(p ? lo + (uintptr_t)(((rows - 1) * ld + cols) * size) : lo) {}
  bool meets(const Range& o) const { return lo < o.hi && o.lo < hi; }
};

int check(Sandwich& a, int64_t rows, int64_t cols, int64_t per_gate, const void* gate, float eps, float scale,
          float off) {
  FLB_CHECK_ARG(gate == nullptr || per_gate >= 1);
  FLB_CHECK_ARG(eps >= 0.f && scale == scale && off == off);
  if (rows > 0x7fffffff || cols > kMaxCols) return FL_B200_ERR_TOO_LARGE;
  a.rows = (uint32_t)rows, a.cols = (int)cols, a.gate = gate;
  a.per_gate = (uint32_t)(gate == nullptr ? rows : std::min(per_gate, rows));
  a.eps = eps, a.scale = scale, a.off = off;
  return FL_B200_OK;
}

}  // namespace
}  // namespace flb200

extern "C" {

FL_B200_API int fl_b200_sandwich_norm(const void* x, int64_t ld_x, const void* residual, int64_t ld_r,
                                      const void* post, const void* pre, const void* gate,
                                      int64_t rows_per_gate, void* y, void* h, int64_t rows, int64_t cols,
                                      float eps, float scale, float weight_offset, int dtype,
                                      fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(rows >= 0 && cols >= 0);
  if (!is_float_dtype(dtype)) return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (rows == 0 || cols == 0) return FL_B200_OK;
  FLB_CHECK_ARG(x && residual && post && pre && y && h && ld_x >= cols && ld_r >= cols);
  Sandwich a = {};
  int st = check(a, rows, cols, rows_per_gate, gate, eps, scale, weight_offset);
  if (st != FL_B200_OK) return st;
  const int64_t size = dtype_size(dtype);
  if (!aligned_to(size, {x, residual, post, pre, gate, y, h})) return FL_B200_ERR_MISALIGNED;
  const Range ry(y, cols, rows, cols, size), rh(h, cols, rows, cols, size);
  const Range in[] = {{x, ld_x, rows, cols, size}, {residual, ld_r, rows, cols, size},
                      {post, cols, 1, cols, size}, {pre, cols, 1, cols, size},
                      {gate, cols, gate ? ceil_div(rows, a.per_gate) : 1, cols, size}};
  FLB_CHECK_ARG(!ry.meets(rh));
  for (const Range& r : in) FLB_CHECK_ARG(!ry.meets(r) && !rh.meets(r));
  a.x = x, a.ldx = ld_x, a.res = residual, a.ldr = ld_r, a.post = post, a.pre = pre, a.y = y, a.h = h;
  DeviceInfo dev;
  st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  return dispatch_float(dtype, [&](auto tag) -> int {
    return launch_fwd<decltype(tag)>(a, dev, static_cast<cudaStream_t>(stream));
  });
}

FL_B200_API size_t fl_b200_sandwich_norm_bwd_workspace_size(int64_t rows, int64_t cols) {
  using namespace flb200;
  DeviceInfo dev;
  if (rows <= 0 || cols <= 0 || current_device_info(&dev) != FL_B200_OK) return 0;
  if (rows > 0x7fffffff || cols > kMaxCols) return 0;
  // (a pack holds 4 or 8 elements: the larger need of the two)
  return std::max(bwd_workspace(rows, cols, cols / 4, dev.sm_count), bwd_workspace(rows, cols, cols / 8, dev.sm_count));
}

FL_B200_API int fl_b200_sandwich_norm_bwd(const void* dy, int64_t ld_dy, const void* dh, int64_t ld_dh,
                                          const void* x, int64_t ld_x, const void* h, int64_t ld_h,
                                          const void* post, const void* pre, const void* gate,
                                          int64_t rows_per_gate, void* dx, void* dresidual, void* dpost,
                                          void* dpre, void* dgate, int64_t rows, int64_t cols, float eps,
                                          float scale, float weight_offset, int dtype, void* workspace,
                                          size_t workspace_bytes, fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(rows >= 0 && cols >= 0);
  if (!is_float_dtype(dtype)) return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (cols == 0) return FL_B200_OK;
  FLB_CHECK_ARG(dpost && dpre);
  const int64_t size = dtype_size(dtype);
  if (!aligned_to(size, {dpost, dpre})) return FL_B200_ERR_MISALIGNED;
  if (rows == 0) {  // sums over no rows
    auto* s = static_cast<cudaStream_t>(stream);
    if (cudaMemsetAsync(dpost, 0, cols * size, s) != cudaSuccess ||
        cudaMemsetAsync(dpre, 0, cols * size, s) != cudaSuccess)
      return launch_status();
    return FL_B200_OK;
  }
  FLB_CHECK_ARG(dy && x && h && post && pre && dx && dresidual && (!gate || dgate));
  FLB_CHECK_ARG(ld_dy >= cols && ld_x >= cols && ld_h >= cols && (!dh || ld_dh >= cols));
  Sandwich a = {};
  int st = check(a, rows, cols, rows_per_gate, gate, eps, scale, weight_offset);
  if (st != FL_B200_OK) return st;
  if (!aligned_to(size, {dy, dh, x, h, post, pre, gate, dx, dresidual, dgate})) return FL_B200_ERR_MISALIGNED;
  const int64_t gates = gate ? ceil_div(rows, a.per_gate) : 1;
  const Range out[] = {{dx, cols, rows, cols, size}, {dresidual, cols, rows, cols, size}, {dpost, cols, 1, cols, size},
                       {dpre, cols, 1, cols, size}, {gate ? dgate : nullptr, cols, gates, cols, size}};
  const Range in[] = {{dy, ld_dy, rows, cols, size}, {dh, ld_dh, rows, cols, size}, {x, ld_x, rows, cols, size},
                      {h, ld_h, rows, cols, size}, {post, cols, 1, cols, size}, {pre, cols, 1, cols, size},
                      {gate, cols, gates, cols, size}};
  for (const Range& o : out) {
    for (const Range& r : in) FLB_CHECK_ARG(!o.meets(r));
    for (const Range& r : out) FLB_CHECK_ARG(&r == &o || !o.meets(r));
  }
  DeviceInfo dev;
  st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  if (workspace == nullptr || workspace_bytes < fl_b200_sandwich_norm_bwd_workspace_size(rows, cols))
    return FL_B200_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FL_B200_ERR_MISALIGNED;
  a.stats = static_cast<float4*>(workspace);
  float* ws = reinterpret_cast<float*>(a.stats + rows);
  a.dy = dy, a.ldy = ld_dy, a.dh = dh, a.ldh = ld_dh, a.x = x, a.ldx = ld_x, a.hs = h, a.lds = ld_h;
  a.post = post, a.pre = pre, a.dx = dx, a.dres = dresidual, a.dpost = dpost, a.dpre = dpre, a.dgate = dgate;
  return dispatch_float(dtype, [&](auto tag) -> int {
    return launch_bwd<decltype(tag)>(a, dev, ws, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
