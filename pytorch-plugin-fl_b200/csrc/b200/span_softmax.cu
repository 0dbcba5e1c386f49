// Softmax of attention scores over each query's span of keys, forward and
// backward.
//
// Row (b, h, q) of the scores x sees the keys j of its span [lo, hi):
//   z_j = scale x_j;  z_j = cap tanh(z_j / cap) where cap > 0;
//   z_j -= slope_h |p - j| where slopes are given, p the query's position;
//   y_j = exp(z_j) / sum over the span of exp(z);  0 outside it.
// Causal and sliding-window masks, packed documents, bidirectional prefixes
// and padded batches are all spans, so there is no mask tensor, and keys
// outside a span are never read.
//   dx_j = scale (1 - tanh^2) y_j (dy_j - sum over the span of y dy).
//
// Bound by memory: the span is read once, the row written once.  A row is
// held in registers (at most 4 packs a thread, one warp for 128 packs, up to
// 1024 threads), its scores as fp32 between the passes.  Rows need not begin
// on a 16-byte boundary: they are walked by the aligned packs that cover
// them, elements outside masked and the row's first and last pack stored by
// element.  (An aligned pack that holds one byte of the row lies in that
// byte's page, so reading all of it is safe.)
//
// Exponentials are ex2.approx (2^-22 relative) of differences from the row's
// maximum.  tanh u = 1 - 2 / (1 + 2^(2 u log2 e)) by ex2.approx and
// rcp.approx: off by some 2^-22 absolutely, as the capped score is by cap
// times that (tanh.approx would be off by 2^-11).
#include "common.cuh"

namespace flb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// e^d.  Scores stay in their own units until they are differences from the
// maximum: times log2 e, a row of the type's lowest value would be -inf.
__device__ __forceinline__ float exp_of(float d) { return ex2(d * kLog2e); }

struct SpanArgs {
  const void* x;
  int64_t ldx;
  const int32_t* spans;
  int64_t spb, spq;
  const int32_t* pos;  // NULL: row q stands at key q + cols - q_len
  int64_t pb, pq;
  const float* slopes;  // NULL: none
  void* out;
  int64_t ldo;
  uint32_t rows, q_len, heads;
  int cols;
  float scale, cap;
  // backward
  const void* dy;
  int64_t ldd;
  const void* y;
  int64_t ldy;
};

struct Row {
  int lo, hi;      // clamped; lo == hi: nothing is seen
  float pos, slope;
};
__device__ __forceinline__ Row row_of(const SpanArgs& a, uint32_t row) {
  const uint32_t bh = row / a.q_len, q = row - bh * a.q_len;
  const uint32_t b = bh / a.heads, h = bh - b * a.heads;
  const int32_t* s = a.spans + b * a.spb + q * a.spq;
  Row r;
  r.lo = max(__ldg(s), 0);
  r.hi = min(__ldg(s + 1), a.cols);
  if (r.hi <= r.lo) r.lo = r.hi = 0;
  r.pos = 0.f;
  r.slope = 0.f;
  if (a.slopes != nullptr) {
    r.slope = __ldg(a.slopes + h);
    r.pos = a.pos != nullptr ? (float)__ldg(a.pos + b * a.pb + q * a.pq)
                             : (float)((int64_t)q + a.cols - (int64_t)a.q_len);
  }
  return r;
}

struct Score {
  float mul, cap;  // cap 0: none
  bool biased;
  __device__ __forceinline__ Score(const SpanArgs& a)
      : mul(a.cap > 0.f ? 2.f * kLog2e * (a.scale / a.cap) : a.scale), cap(a.cap), biased(a.slopes != nullptr) {}
  __device__ __forceinline__ float operator()(float x, int key, const Row& r) const {
    float z = x * mul;
    if (cap != 0.f) z = fmaf(-2.f * cap, rcp(1.f + ex2(z)), cap);
    if (biased) z = fmaf(-r.slope, fabsf(r.pos - (float)key), z);
    return z;
  }
  // d(score) / d(scale x): 1 - tanh^2 = 4 e / (1 + e)^2
  __device__ __forceinline__ float slope(float x) const {
    if (cap == 0.f) return 1.f;
    const float q = rcp(1.f + ex2(x * mul));  // (1 - tanh) / 2
    return 4.f * q * (1.f - q);
  }
};

// N consecutive elements of T at a 16-byte boundary (N * size a multiple of 16).
template <typename T, int N>
struct Elems {
  static constexpr int VW = Elem<T>::kVec;
  uint4 w[N / VW];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N / VW; ++i) w[i] = ld_stream(p + i * VW);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N / VW; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void to(float (&f)[N]) const {
#pragma unroll
    for (int i = 0; i < N / VW; ++i) {
      float g[VW];
      unpack<T>(w[i], g);
#pragma unroll
      for (int e = 0; e < VW; ++e) f[i * VW + e] = g[e];
    }
  }
};
// Stores f at virtual elements [v, v + N) of a row that holds [first, last).
template <typename T, int N>
__device__ __forceinline__ void store(T* row, int v, int first, int last, const float (&f)[N]) {
  constexpr int VW = Elem<T>::kVec;
  if (v >= first && v + N <= last) {
#pragma unroll
    for (int i = 0; i < N / VW; ++i) {
      float g[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) g[e] = f[i * VW + e];
      st_stream(row + v + i * VW, pack<T>(g));
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (v + e >= first && v + e < last) row[v + e] = Elem<T>::from_f(f[e]);
  }
}

// A row's aligned packs: element j of the row is virtual element shift + j,
// and virtual element 0 lies on a 16-byte boundary.
template <typename T>
__device__ __forceinline__ int shift_of(const T* p) {
  return (int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
}

// TPR threads a row, VPT packs each.
template <typename TI, typename TO, int TPR, int VPT, int BLOCK>
__global__ void __launch_bounds__(BLOCK, BLOCK <= 256 ? 4 : 1)
span_softmax_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  constexpr int N = Elem<TI>::kVec;
  constexpr int RPB = BLOCK / TPR;
  __shared__ float smem[BLOCK / 32];
  const int lane = threadIdx.x % TPR;
  const uint64_t row64 = (uint64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const bool ok = row64 < a.rows;
  const uint32_t row = ok ? (uint32_t)row64 : a.rows - 1;
  const Row r = row_of(a, row);
  const Score score(a);
  const TI* xr = static_cast<const TI*>(a.x) + row * a.ldx;
  const int shift = shift_of(xr);
  xr -= shift;
  TO* out = static_cast<TO*>(a.out) + row * a.ldo - shift;
  const int first = shift, last = shift + a.cols;  // of the row, virtual
  const int lo = shift + r.lo, hi = shift + r.hi;  // of the span
  const int p0 = lo / N, n = (hi + N - 1) / N - p0;   // the span's packs
  const int count = r.hi > r.lo ? n : 0;
  Elems<TI, N> v[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    if (ok && vi < count) v[i].load(xr + (int64_t)(p0 + vi) * N);
    else v[i].clear();
  }
  if (ok) {  // what is not seen is 0
    float zero[N];
#pragma unroll
    for (int e = 0; e < N; ++e) zero[e] = 0.f;
    const int packs = (last + N - 1) / N;
    const int until = count ? p0 : packs;
    for (int p = lane; p < until; p += TPR) store<TO, N>(out, p * N, first, last, zero);
    if (count)
      for (int p = p0 + n + lane; p < packs; p += TPR) store<TO, N>(out, p * N, first, last, zero);
  }
  float z[VPT][N];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    if (i * TPR < count) {
      const int at = (p0 + vi) * N;
      float f[N];
      v[i].to(f);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const bool in = at + e >= lo && at + e < hi;
        z[i][e] = in ? score(f[e], at + e - shift, r) : -INFINITY;
        m = fmaxf(m, z[i][e]);
      }
    }
  }
  m = row_reduce<FastMaxOp, TPR, BLOCK>(m, smem);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i * TPR < count) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        z[i][e] = exp_of(z[i][e] - m);
        s += z[i][e];
      }
    }
  }
  s = row_reduce<SumOp, TPR, BLOCK>(s, smem);
  const float inv = 1.f / s;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    if (ok && vi < count) {
      const int at = (p0 + vi) * N;
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = at + e >= lo && at + e < hi ? z[i][e] * inv : 0.f;
      store<TO, N>(out, at, first, last, f);
    }
  }
}

// Rows of any length and alignment: a CTA a row, the span read twice.
template <typename TI, typename TO>
__global__ void __launch_bounds__(512)
span_softmax_loop_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  constexpr int BLOCK = 512;
  __shared__ float smem[BLOCK / 32];
  const Score score(a);
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const Row r = row_of(a, row);
    const TI* xr = static_cast<const TI*>(a.x) + row * a.ldx;
    TO* out = static_cast<TO*>(a.out) + row * a.ldo;
    float m = -INFINITY, s = 0.f;
    bool nan = false;
    for (int j = r.lo + threadIdx.x; j < r.hi; j += BLOCK) {
      const float z = score(Elem<TI>::to_f(xr[j]), j, r);
      nan |= z != z;
      if (z > m) {
        s *= exp_of(m - z);
        m = z;
      }
      s += m == -INFINITY ? 0.f : exp_of(z - m);
    }
    const float top = block_reduce<FastMaxOp, BLOCK>(m, smem);
    // (a row of -inf alone, and one with a NaN or +inf, is NaN as softmax's is)
    s = nan ? NAN : m == -INFINITY ? 0.f : s * exp_of(m - top);
    s = block_reduce<SumOp, BLOCK>(s, smem);
    const float inv = 1.f / s;
    for (int j = threadIdx.x; j < a.cols; j += BLOCK) {
      float y = 0.f;
      if (j >= r.lo && j < r.hi) y = exp_of(score(Elem<TI>::to_f(xr[j]), j, r) - top) * inv;
      out[j] = Elem<TO>::from_f(y);
    }
  }
}

// TI: x's and dx's type, TY: y's and dy's.
template <typename TI, typename TY, int TPR, int VPT, int BLOCK>
__global__ void __launch_bounds__(BLOCK, BLOCK <= 256 ? 2 : 1)
span_softmax_bwd_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  constexpr int N = Elem<TI>::kVec;
  constexpr int RPB = BLOCK / TPR;
  __shared__ float smem[BLOCK / 32];
  const int lane = threadIdx.x % TPR;
  const uint64_t row64 = (uint64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const bool ok = row64 < a.rows;
  const uint32_t row = ok ? (uint32_t)row64 : a.rows - 1;
  const Row r = row_of(a, row);
  const Score score(a);
  const bool capped = score.cap != 0.f;
  TI* out = static_cast<TI*>(a.out) + row * a.ldo;
  const int shift = shift_of(out);
  out -= shift;
  const TY* yr = static_cast<const TY*>(a.y) + row * a.ldy - shift;
  const TY* dr = static_cast<const TY*>(a.dy) + row * a.ldd - shift;
  const TI* xr = static_cast<const TI*>(a.x) + (capped ? row * a.ldx - shift : 0);
  const int first = shift, last = shift + a.cols;
  const int lo = shift + r.lo, hi = shift + r.hi;
  const int p0 = lo / N, n = (hi + N - 1) / N - p0;
  const int count = r.hi > r.lo ? n : 0;
  Elems<TY, N> y[VPT], d[VPT];
  Elems<TI, N> x[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    if (ok && vi < count) {
      y[i].load(yr + (int64_t)(p0 + vi) * N);
      d[i].load(dr + (int64_t)(p0 + vi) * N);
      if (capped) x[i].load(xr + (int64_t)(p0 + vi) * N);
    } else {
      y[i].clear();
      d[i].clear();
    }
  }
  if (ok) {
    float zero[N];
#pragma unroll
    for (int e = 0; e < N; ++e) zero[e] = 0.f;
    const int packs = (last + N - 1) / N;
    const int until = count ? p0 : packs;
    for (int p = lane; p < until; p += TPR) store<TI, N>(out, p * N, first, last, zero);
    if (count)
      for (int p = p0 + n + lane; p < packs; p += TPR) store<TI, N>(out, p * N, first, last, zero);
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i * TPR < count) {
      const int at = (p0 + lane + i * TPR) * N;
      float f[N], g[N];
      y[i].to(f);
      d[i].to(g);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (at + e >= lo && at + e < hi) sum = fmaf(f[e], g[e], sum);
    }
  }
  sum = row_reduce<SumOp, TPR, BLOCK>(sum, smem);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    if (ok && vi < count) {
      const int at = (p0 + vi) * N;
      float f[N], g[N], h[N];
      y[i].to(f);
      d[i].to(g);
      if (capped) x[i].to(h);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        float t = a.scale * f[e] * (g[e] - sum);
        if (capped) t *= score.slope(h[e]);
        f[e] = at + e >= lo && at + e < hi ? t : 0.f;
      }
      store<TI, N>(out, at, first, last, f);
    }
  }
}

template <typename TI, typename TY>
__global__ void __launch_bounds__(512)
span_softmax_bwd_loop_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  constexpr int BLOCK = 512;
  __shared__ float smem[BLOCK / 32];
  const Score score(a);
  const bool capped = score.cap != 0.f;
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const Row r = row_of(a, row);
    const TY* yr = static_cast<const TY*>(a.y) + row * a.ldy;
    const TY* dr = static_cast<const TY*>(a.dy) + row * a.ldd;
    const TI* xr = static_cast<const TI*>(a.x) + (capped ? row * a.ldx : 0);
    TI* out = static_cast<TI*>(a.out) + row * a.ldo;
    float sum = 0.f;
    for (int j = r.lo + threadIdx.x; j < r.hi; j += BLOCK)
      sum = fmaf(Elem<TY>::to_f(yr[j]), Elem<TY>::to_f(dr[j]), sum);
    sum = block_reduce<SumOp, BLOCK>(sum, smem);
    for (int j = threadIdx.x; j < a.cols; j += BLOCK) {
      float t = 0.f;
      if (j >= r.lo && j < r.hi) {
        t = a.scale * Elem<TY>::to_f(yr[j]) * (Elem<TY>::to_f(dr[j]) - sum);
        if (capped) t *= score.slope(Elem<TI>::to_f(xr[j]));
      }
      out[j] = Elem<TI>::from_f(t);
    }
  }
}

// Calls f(TPR, VPT) for rows covered by `packs` packs, at most 4 a thread;
// -1: longer than that.
template <typename F>
int span_ladder(int64_t packs, F&& f) {
  using std::integral_constant;
  using V4 = integral_constant<int, 4>;
  if (packs <= 32) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  if (packs <= 64) return f(integral_constant<int, 32>{}, integral_constant<int, 2>{});
  if (packs <= 128) return f(integral_constant<int, 32>{}, V4{});
  if (packs <= 256) return f(integral_constant<int, 64>{}, V4{});
  if (packs <= 512) return f(integral_constant<int, 128>{}, V4{});
  if (packs <= 1024) return f(integral_constant<int, 256>{}, V4{});
  if (packs <= 2048) return f(integral_constant<int, 512>{}, V4{});
  if (packs <= 4096) return f(integral_constant<int, 1024>{}, V4{});
  return -1;
}

// Whether rows at p and q (strides in elements) begin at the same element of
// a 16-byte pack of the wider type TB, row by row.
template <typename TA, typename TB>
bool in_step(const void* p, int64_t lp, const void* q, int64_t lq, int64_t rows) {
  constexpr int64_t w = Elem<TA>::kVec < Elem<TB>::kVec ? Elem<TA>::kVec : Elem<TB>::kVec;
  const int64_t ep = (int64_t)(reinterpret_cast<uintptr_t>(p) / sizeof(TA));
  const int64_t eq = (int64_t)(reinterpret_cast<uintptr_t>(q) / sizeof(TB));
  return (ep - eq) % w == 0 && (rows <= 1 || (lp - lq) % w == 0);
}

template <typename TI, typename TO>
int launch_fwd(const SpanArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int N = Elem<TI>::kVec;
  if (in_step<TI, TO>(a.x, a.ldx, a.out, a.ldo, a.rows)) {
    const int64_t packs = (a.cols + 2 * (N - 1)) / N;
    const int st = span_ladder(packs, [&](auto tpr, auto vpt) -> int {
      constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
      constexpr int BLOCK = TPR >= 256 ? TPR : 256;
      launch_k((span_softmax_kernel<TI, TO, TPR, VPT, BLOCK>), (unsigned)ceil_div(a.rows, BLOCK / TPR), BLOCK, 0,
               stream, a);
      return launch_status();
    });
    if (st >= 0) return st;
  }
  const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 4ll * dev.sm_count);
  launch_k((span_softmax_loop_kernel<TI, TO>), grid, 512, 0, stream, a);
  return launch_status();
}

template <typename TI, typename TY>
int launch_bwd(const SpanArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int N = Elem<TI>::kVec;
  if (in_step<TI, TY>(a.out, a.ldo, a.y, a.ldy, a.rows) && in_step<TI, TY>(a.out, a.ldo, a.dy, a.ldd, a.rows) &&
      (!(a.cap > 0.f) || in_step<TI, TI>(a.out, a.ldo, a.x, a.ldx, a.rows))) {
    const int64_t packs = (a.cols + 2 * (N - 1)) / N;
    const int st = span_ladder(packs, [&](auto tpr, auto vpt) -> int {
      constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
      constexpr int BLOCK = TPR >= 256 ? TPR : 256;
      launch_k((span_softmax_bwd_kernel<TI, TY, TPR, VPT, BLOCK>), (unsigned)ceil_div(a.rows, BLOCK / TPR), BLOCK,
               0, stream, a);
      return launch_status();
    });
    if (st >= 0) return st;
  }
  const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 4ll * dev.sm_count);
  launch_k((span_softmax_bwd_loop_kernel<TI, TY>), grid, 512, 0, stream, a);
  return launch_status();
}

// Whether two row operands (strides in elements) share memory.
bool overlap(const void* p, int64_t lp, int64_t sp, const void* q, int64_t lq, int64_t sq, int64_t rows,
             int64_t cols) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  const uintptr_t ea = a + (uintptr_t)(((rows - 1) * lp + cols) * sp);
  const uintptr_t eb = b + (uintptr_t)(((rows - 1) * lq + cols) * sq);
  return a < eb && b < ea;
}

int check(SpanArgs& a, const int32_t* spans, int64_t rows, int64_t cols, int64_t heads, int64_t q_len,
          float scale, float cap) {
  FLB_CHECK_ARG(spans && heads > 0 && q_len > 0 && rows % (heads * q_len) == 0);
  FLB_CHECK_ARG(a.spb >= 0 && a.spq >= 0 && a.pb >= 0 && a.pq >= 0);
  FLB_CHECK_ARG(scale == scale && cap >= 0.f && cap <= 3e38f);
  if (rows > 0x7fffffff || cols > 0x7fffff00) return FL_B200_ERR_TOO_LARGE;
  a.spans = spans;
  a.rows = (uint32_t)rows, a.q_len = (uint32_t)q_len, a.heads = (uint32_t)heads;
  a.cols = (int)cols;
  a.scale = scale, a.cap = cap;
  return FL_B200_OK;
}

}  // namespace
}  // namespace flb200

extern "C" {

FL_B200_API int fl_b200_span_softmax(const void* x, int64_t ld_x, const int32_t* spans, int64_t span_sb,
                                     int64_t span_sq, const int32_t* positions, int64_t pos_sb, int64_t pos_sq,
                                     const float* slopes, void* out, int64_t ld_out, int64_t rows, int64_t cols,
                                     int64_t heads, int64_t q_len, float scale, float cap, int in_dtype,
                                     int out_dtype, fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(rows >= 0 && cols >= 0);
  if (!is_float_dtype(in_dtype) || (out_dtype != in_dtype && out_dtype != FL_B200_F32))
    return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (rows == 0 || cols == 0) return FL_B200_OK;
  FLB_CHECK_ARG(x && out && ld_x >= cols && ld_out >= cols);
  SpanArgs a = {};
  a.spb = span_sb, a.spq = span_sq, a.pos = positions, a.pb = pos_sb, a.pq = pos_sq;
  int st = check(a, spans, rows, cols, heads, q_len, scale, cap);
  if (st != FL_B200_OK) return st;
  FLB_CHECK_ARG(!overlap(x, ld_x, dtype_size(in_dtype), out, ld_out, dtype_size(out_dtype), rows, cols));
  a.x = x, a.ldx = ld_x, a.out = out, a.ldo = ld_out, a.slopes = slopes;
  DeviceInfo dev;
  st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  auto* s = static_cast<cudaStream_t>(stream);
  return dispatch_float(in_dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    return out_dtype == in_dtype ? launch_fwd<T, T>(a, dev, s) : launch_fwd<T, float>(a, dev, s);
  });
}

FL_B200_API int fl_b200_span_softmax_bwd(const void* dy, int64_t ld_dy, const void* y, int64_t ld_y,
                                         const void* x, int64_t ld_x, const int32_t* spans, int64_t span_sb,
                                         int64_t span_sq, void* dx, int64_t ld_dx, int64_t rows, int64_t cols,
                                         int64_t heads, int64_t q_len, float scale, float cap, int y_dtype,
                                         int x_dtype, fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(rows >= 0 && cols >= 0);
  if (!is_float_dtype(x_dtype) || (y_dtype != x_dtype && y_dtype != FL_B200_F32))
    return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (rows == 0 || cols == 0) return FL_B200_OK;
  FLB_CHECK_ARG(dy && y && dx && ld_dy >= cols && ld_y >= cols && ld_dx >= cols);
  SpanArgs a = {};
  a.spb = span_sb, a.spq = span_sq;
  int st = check(a, spans, rows, cols, heads, q_len, scale, cap);
  if (st != FL_B200_OK) return st;
  const int sx = dtype_size(x_dtype), sy = dtype_size(y_dtype);
  FLB_CHECK_ARG(!overlap(dx, ld_dx, sx, dy, ld_dy, sy, rows, cols) &&
                !overlap(dx, ld_dx, sx, y, ld_y, sy, rows, cols));
  if (cap > 0.f) {
    FLB_CHECK_ARG(x && ld_x >= cols && !overlap(dx, ld_dx, sx, x, ld_x, sx, rows, cols));
    a.x = x, a.ldx = ld_x;
  }
  a.dy = dy, a.ldd = ld_dy, a.y = y, a.ldy = ld_y, a.out = dx, a.ldo = ld_dx;
  DeviceInfo dev;
  st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  auto* s = static_cast<cudaStream_t>(stream);
  return dispatch_float(x_dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    return y_dtype == x_dtype ? launch_bwd<T, T>(a, dev, s) : launch_bwd<T, float>(a, dev, s);
  });
}

}  // extern "C"
