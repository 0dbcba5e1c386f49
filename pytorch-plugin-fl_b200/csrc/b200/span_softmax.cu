// Softmax of attention scores over each query's span of keys, forward and
// backward.
//
// Row (b, h, q) of the scores x sees the keys j of its span [lo, hi):
//   z_j = scale x_j;  z_j = cap tanh(z_j / cap) where cap > 0;
//   z_j -= slope_h |p - j| where slopes are given, p the query's position;
//   y_j = exp(z_j) / sum over the span of exp(z);  0 outside it.
// Causal and sliding-window masks, packed documents, bidirectional prefixes
// and padded batches are all spans, so there is no mask tensor, and of what
// lies outside a span only the rest of its first and last 16 bytes is read.
//   dx_j = scale (1 - tanh^2) y_j (dy_j - sum over the span of y dy).
//
// The span is read once and the row written once (a row too long for a CTA's
// registers is read a second time, from L2): a warp a row up to 2048 keys of
// 16 bits, then a CTA a row, scores as fp32 between the passes.  Long spans
// are bound by memory (2048 of 2048 keys, bf16: 4.5 TB/s), short ones by the
// instructions a row costs before its first key (340 of the 470 of a row of
// 200 keys, 5.4 TB/s with the zeros around them), capped ones by theirs.
// Rows need not begin on a 16-byte boundary: they are walked by the aligned
// packs that cover them, elements outside masked and the row's first and last
// pack stored by element.  (16 aligned bytes that hold one byte of the row lie
// in that byte's page, so reading all of them is safe; of a pack of 32 bytes,
// fp32 beside 16-bit scores, each half is read only if it does.)
//
// Exponentials are ex2.approx (2^-22 relative) of differences from the row's
// maximum.  Capped scores for 16-bit results take tanh u = 1 - 2 / (1 + 2^(2 u
// log2 e)) by ex2.approx and rcp.approx: off by some 2^-22 absolutely, as the
// score is by cap times that (tanh.approx would be off by 2^-11).  Up to a cap
// of 256 that is an eighth of half a step of fp16; larger caps and fp32
// results, which resolve it, take tanhf, off by a few 2^-24 of the score (4 x 32
// x 2048 x 2048 f32, documents, cap 50: 460 us, 458 with the other).
#include "common.cuh"
#include "span_place.cuh"

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

// Key counters are ints, and a loop's last step passes the row's end.
constexpr int64_t kMaxCols = 0x7fff0000;

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
  uint32_t unit;  // rows a warp takes in order
  float scale, cap;
  // backward
  const void* dy;
  int64_t ldd;
  const void* y;
  int64_t ldy;
};

struct Raw {
  int lo, hi, pos;
  float slope;
};
struct Row {
  int lo, hi;  // clamped; lo == hi: nothing is seen
  int pos;     // whole, so that the distance to a key is exact wherever both lie
  float slope;
  __device__ __forceinline__ Row(const Raw& r, int cols)
      : lo(max(r.lo, 0)), hi(min(r.hi, cols)), pos(min(max(r.pos, -(1 << 30)), 1 << 30)), slope(r.slope) {
    if (hi <= lo) lo = hi = 0;
  }
};
// Row `row`'s head and query, the latter kept up to date while rows are
// walked in order (a division a row is 5 % of a short row's instructions).
struct Walk {
  uint32_t row, q;
  const int32_t *span, *pos;
  float slope;
  __device__ __forceinline__ void to(const SpanArgs& a, uint32_t at) {
    row = at;
    const uint32_t bh = row / a.q_len;
    q = row - bh * a.q_len;
    const uint32_t b = bh / a.heads, h = bh - b * a.heads;
    span = a.spans + b * a.spb + q * a.spq;
    pos = a.pos == nullptr ? nullptr : a.pos + b * a.pb + q * a.pq;
    slope = a.slopes == nullptr ? 0.f : __ldg(a.slopes + h);
  }
  __device__ __forceinline__ void next(const SpanArgs& a) {
    if (q + 1 == a.q_len) return to(a, row + 1);
    ++row;
    ++q;
    span += a.spq;
    if (pos != nullptr) pos += a.pq;
  }
  // What the row's metadata hold, not looked at yet: the loads are on their
  // way while other work goes on.
  __device__ __forceinline__ Raw read(const SpanArgs& a) const {
    Raw r;
    r.lo = __ldg(span);
    r.hi = __ldg(span + 1);
    r.pos = 0;
    if (a.slopes != nullptr) r.pos = pos != nullptr ? __ldg(pos) : (int)(q + (uint32_t)a.cols - a.q_len);
    r.slope = slope;
    return r;
  }
  __device__ __forceinline__ Row get(const SpanArgs& a) const { return Row(read(a), a.cols); }
};
__device__ __forceinline__ Row row_of(const SpanArgs& a, uint32_t row) {
  Walk w;
  w.to(a, row);
  return w.get(a);
}

// EXACT: tanh by tanhf, for capped scores (see above).
template <bool EXACT>
struct Score {
  float mul, cap;  // cap 0: none
  bool biased;
  __device__ __forceinline__ Score(const SpanArgs& a)
      : mul(a.cap > 0.f ? (EXACT ? 1.f : 2.f * kLog2e) * (a.scale / a.cap) : a.scale), cap(a.cap),
        biased(a.slopes != nullptr) {}
  __device__ __forceinline__ float operator()(float x, int key, const Row& r) const {
    float z = x * mul;
    if constexpr (EXACT) z = cap * tanhf(z);
    else if (cap != 0.f) z = fmaf(-2.f * cap, rcp(1.f + ex2(z)), cap);
    if (biased) z = fmaf(-r.slope, fabsf((float)(r.pos - key)), z);
    return z;
  }
  // d(score) / d(scale x): 1 - tanh^2 = 4 e / (1 + e)^2
  __device__ __forceinline__ float slope(float x) const {
    if (cap == 0.f) return 1.f;
    const float q = rcp(1.f + ex2(x * mul));  // (1 - tanh) / 2
    return 4.f * q * (1.f - q);
  }
  // (1 - tanh) / 2 of a pair of x.
  __device__ __forceinline__ uint64_t half_of(uint64_t x) const {
    const uint64_t t = f2_mul(x, f2_make(mul, mul));
    const uint64_t d = f2_add(f2_make(ex2(f2_lo(t)), ex2(f2_hi(t))), f2_make(1.f, 1.f));
    return f2_make(rcp(f2_lo(d)), rcp(f2_hi(d)));
  }
  // P pairs in place, the first element at `key`.  Choices are made for a
  // pack, not for each element.
  template <int P>
  __device__ __forceinline__ void pack(uint64_t (&z)[P], int key, const Row& r) const {
    if constexpr (EXACT) {
#pragma unroll
      for (int e = 0; e < P; ++e) z[e] = f2_make(cap * tanhf(f2_lo(z[e]) * mul), cap * tanhf(f2_hi(z[e]) * mul));
    } else if (cap != 0.f) {
      const uint64_t m = f2_make(-2.f * cap, -2.f * cap), c = f2_make(cap, cap);
#pragma unroll
      for (int e = 0; e < P; ++e) z[e] = f2_fma(half_of(z[e]), m, c);
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e) z[e] = f2_mul(z[e], f2_make(mul, mul));
    }
    if (biased) {
      const float d = (float)(r.pos - key);
#pragma unroll
      for (int e = 0; e < P; ++e)
        z[e] = f2_make(fmaf(-r.slope, fabsf(d - (float)(2 * e)), f2_lo(z[e])),
                       fmaf(-r.slope, fabsf(d - (float)(2 * e + 1)), f2_hi(z[e])));
    }
  }
};

// N consecutive elements of T at a 16-byte boundary (N * size a multiple of
// 16), as fp32 pairs when they are worked on.
template <typename T, int N>
struct Elems {
  static constexpr int VW = Elem<T>::kVec;
  static constexpr int WORDS = N * (int)sizeof(T) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N / VW; ++i) {
      word(i, ld_stream_now(p + i * VW));
    }
  }
  __device__ __forceinline__ void word(int i, const uint4& u) {
    w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
  }
  // Zeros but for elements [from, to).
  __device__ __forceinline__ void keep(int from, int to) {
    constexpr int P = 4 / (int)sizeof(T);  // elements a word
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      uint32_t mask = 0;
#pragma unroll
      for (int e = 0; e < P; ++e)
        if (i * P + e >= from && i * P + e < to) mask |= (P == 1 ? 0xffffffffu : 0xffffu << (16 * e));
      w[i] &= mask;
    }
  }
  __device__ __forceinline__ void to(uint64_t (&f)[N / 2]) const {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      if constexpr (std::is_same<T, float>::value) {
        f[e] = f2_make(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
      } else {
        f[e] = pair_from_bits<T>(w[e]);
      }
    }
  }
};
// Stores pairs at virtual elements [v, v + N) of a row that holds [first, last).
template <typename T, int N>
__device__ __forceinline__ void store(T* row, int v, int first, int last, const uint64_t (&f)[N / 2]) {
  constexpr int VW = Elem<T>::kVec;
  if (v >= first && v + N <= last) {
#pragma unroll
    for (int i = 0; i < N / VW; ++i) {
      uint4 u;
      if constexpr (std::is_same<T, float>::value) {
        u = make_uint4(__float_as_uint(f2_lo(f[2 * i])), __float_as_uint(f2_hi(f[2 * i])),
                       __float_as_uint(f2_lo(f[2 * i + 1])), __float_as_uint(f2_hi(f[2 * i + 1])));
      } else {
        u = make_uint4(pair_to_bits<T>(f[4 * i]), pair_to_bits<T>(f[4 * i + 1]), pair_to_bits<T>(f[4 * i + 2]),
                       pair_to_bits<T>(f[4 * i + 3]));
      }
      st_stream(row + v + i * VW, u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (v + e >= first && v + e < last) row[v + e] = Elem<T>::from_f(e % 2 ? f2_hi(f[e / 2]) : f2_lo(f[e / 2]));
  }
}

// A row's aligned packs: element j of the row is virtual element shift + j,
// and virtual element 0 lies on a 16-byte boundary.
template <typename T>
__device__ __forceinline__ int shift_of(const T* p) {
  return (int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
}

template <int N>
struct Place : Packs<N> {
  using Packs<N>::lo;
  using Packs<N>::hi;
  __device__ __forceinline__ Place(const Row& r, int shift, int cols) : Packs<N>(r.lo, r.hi, shift, cols) {}
  // Pairs of the pack at `at`: `other` outside the span.
  __device__ __forceinline__ void mask(uint64_t (&z)[N / 2], int at, float other) const {
#pragma unroll
    for (int e = 0; e < N / 2; ++e)
      z[e] = f2_make(at + 2 * e >= lo && at + 2 * e < hi ? f2_lo(z[e]) : other,
                     at + 2 * e + 1 >= lo && at + 2 * e + 1 < hi ? f2_hi(z[e]) : other);
  }
};
// Pack `at` of y or dy: its words that hold something of the span, else zeros.
template <typename T, int N>
__device__ __forceinline__ void load_words(Elems<T, N>& v, const T* from, int at, const Place<N>& p) {
  constexpr int VW = Elem<T>::kVec;
#pragma unroll
  for (int k = 0; k < N / VW; ++k)
    v.word(k, N == VW || p.meets(at + k * VW, VW) ? ld_stream_now(from + k * VW) : make_uint4(0, 0, 0, 0));
}
// Where nothing is seen: whole packs [begin, p0) and [p1, end), and the
// row's first and last pack where they are not whole.
template <typename TO, int N>
struct Outside {
  int begin, p0, p1, end;
  __device__ __forceinline__ explicit Outside(const Place<N>& p) {
    begin = p.first > 0 ? 1 : 0;
    end = (int)((uint32_t)p.last / N);
    p0 = p.count ? max(p.p0, begin) : end;
    p1 = p.count ? p.p0 + p.count : end;
  }
  __device__ __forceinline__ void edges(TO* row, const Place<N>& p, int lane) const {
    if (p.first > 0 && (p.count == 0 || p.p0 > 0) && lane >= p.first && lane < N && lane < p.last)
      row[lane] = Elem<TO>::from_f(0.f);
    if ((uint32_t)p.last % N != 0 && end >= begin && (p.count == 0 || p1 <= end) && lane < p.last - end * N)
      row[end * N + lane] = Elem<TO>::from_f(0.f);
  }
};
// Zeros there by the TPR threads of a row.
template <typename TO, int N, int TPR>
__device__ __forceinline__ void clear_outside(TO* row, const Place<N>& p, int lane) {
  const Outside<TO, N> o(p);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const int before = max(o.p0 - o.begin, 0), all = before + max(o.end - o.p1, 0);
#pragma unroll 2
  for (int j = lane; j < all; j += TPR) {
    const int v = j < before ? o.begin + j : o.p1 + (j - before);
#pragma unroll
    for (int i = 0; i < N / Elem<TO>::kVec; ++i) st_stream(row + v * N + i * Elem<TO>::kVec, zero);
  }
  o.edges(row, p, lane);
}
// Zeros there by the warp of a row as bulk copies of 1 KB of zeros in shared
// memory: one instruction for what takes a loop of stores.
constexpr int kZeroBytes = 1024;
template <typename TO, int N>
__device__ __forceinline__ void clear_outside_bulk(TO* row, const Place<N>& p, int lane, uint32_t zeros) {
  const Outside<TO, N> o(p);
  constexpr int kPack = N * (int)sizeof(TO);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    char* to = reinterpret_cast<char*>(row) + (side == 0 ? o.begin : o.p1) * kPack;
    const int bytes = (side == 0 ? o.p0 - o.begin : o.end - o.p1) * kPack;
    const int at = lane * kZeroBytes;  // (a warp's rows have less than 32 KB)
    if (at < bytes)
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to + at), "r"(zeros),
                   "r"(min(kZeroBytes, bytes - at))
                   : "memory");
  }
  o.edges(row, p, lane);
}
// The CTA's zeros; every thread of it calls this once.
__device__ __forceinline__ uint32_t make_zeros(void* smem) {
  for (int i = threadIdx.x; i < kZeroBytes / 16; i += blockDim.x) static_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // seen by the copies
  __syncthreads();
  return (uint32_t)__cvta_generic_to_shared(smem);
}
// Before a thread leaves: its copies have read the zeros.
__device__ __forceinline__ void finish_zeros() {
  asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
}
// Scores of the pack at virtual element `at` from its elements, -inf outside
// the span; returns the larger of m and their maximum.  (What lies outside is
// scored too and then dropped.)
template <int N, bool EXACT>
__device__ __forceinline__ float scores_of(uint64_t (&z)[N / 2], int at, const Place<N>& p, const Row& r,
                                           const Score<EXACT>& score, float m) {
  score.template pack<N / 2>(z, at - p.first, r);
  if (!p.inside(at)) p.mask(z, at, -INFINITY);
#pragma unroll
  for (int e = 0; e < N / 2; ++e) m = fmax3(m, f2_lo(z[e]), f2_hi(z[e]));
  return m;
}
// Turns scores into exponentials of their differences from m; the sum.  One
// FMA an element: the rounding of m log2 e, up to 2^-24 |m| log2 e, is a
// factor 2^that which all of them share.  Where it could overflow, the maximum
// is subtracted first.
constexpr float kWide = 1e6f;
template <int N, int VPT, int TPR>
__device__ __forceinline__ float exps_of(uint64_t (&z)[VPT][N / 2], int count, float m) {
  float shift = m * kLog2e;
  if (!(fabsf(m) < kWide)) {
    shift = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (i * TPR < count) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) z[i][e] = f2_make(f2_lo(z[i][e]) - m, f2_hi(z[i][e]) - m);
      }
  }
  const uint64_t l = f2_make(kLog2e, kLog2e), c = f2_make(-shift, -shift);
  uint64_t s[2] = {f2_make(0.f, 0.f), f2_make(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i * TPR < count) {
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        const uint64_t t = f2_fma(z[i][e], l, c);
        z[i][e] = f2_make(ex2(f2_lo(t)), ex2(f2_hi(t)));
        s[e & 1] = f2_add(s[e & 1], z[i][e]);
      }
    }
  }
  s[0] = f2_add(s[0], s[1]);
  return f2_lo(s[0]) + f2_hi(s[0]);
}
// The same of one pack where a row's exponentials are not all taken from one
// maximum (by threads with their own, and again in a second pass): the
// factor would not be shared, so the difference is rounded first.
template <int N>
__device__ __forceinline__ float exps_from(uint64_t (&z)[N / 2], float m) {
  const uint64_t l = f2_make(kLog2e, kLog2e), c = f2_make(-m, -m);
  uint64_t s = f2_make(0.f, 0.f);
#pragma unroll
  for (int e = 0; e < N / 2; ++e) {
    const uint64_t t = f2_mul(f2_add(z[e], c), l);
    z[e] = f2_make(ex2(f2_lo(t)), ex2(f2_hi(t)));
    s = f2_add(s, z[e]);
  }
  return f2_lo(s) + f2_hi(s);
}
// Exponentials times inv, stored.  Outside the span they are 0, but 0 times
// an inv that is not finite is not.
template <typename TO, int N>
__device__ __forceinline__ void put(TO* out, uint64_t (&z)[N / 2], int at, const Place<N>& p, float inv) {
#pragma unroll
  for (int e = 0; e < N / 2; ++e) z[e] = f2_mul(z[e], f2_make(inv, inv));
  if (!(inv < 3e38f) && !p.inside(at)) p.mask(z, at, 0.f);
  store<TO, N>(out, at, p.first, p.last, z);
}

// A warp takes `unit` rows in order, then those `unit` times the grid's warps
// further on (so that rows that see little and rows that see much are spread).
struct Rows {
  Walk w;
  uint32_t left;  // rows of this unit after this one
  bool more;
  __device__ __forceinline__ explicit Rows(const SpanArgs& a) {
    const uint32_t unit = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    more = (uint64_t)unit * a.unit < a.rows;
    left = a.unit - 1;
    if (more) w.to(a, unit * a.unit);
  }
  __device__ __forceinline__ void next(const SpanArgs& a) {
    if (w.row + 1 >= a.rows) {
      more = false;
    } else if (left > 0) {
      --left;
      w.next(a);
    } else {
      const uint64_t to = (uint64_t)w.row + 1 - a.unit + (uint64_t)gridDim.x * (blockDim.x >> 5) * a.unit;
      more = to < a.rows;
      left = a.unit - 1;
      if (more) w.to(a, (uint32_t)to);
    }
  }
};

// A warp a row.  Spans of up to 64 packs stay in registers; longer ones have
// their scores in shared memory, fp32, between the passes (a lane reads only
// what it wrote, so nothing waits for anything): loops whose length is the
// span's, 80 registers and 24 warps an SM.  All of 2048 scores in registers
// took 110 to 128 of them and 16 warps, code for every length that a short
// span skipped at half the price of running it, and spills, which this much
// shared memory leaves no L1 for: 524288 rows of 2048, packed documents,
// capped, 1431 us with 116 bytes of spills and 672 us without; this 455 to
// 480 us (4.9 TB/s).  The first packs of the next row are loaded while a long span's
// sums go through the warp, and every row's span is read one row ahead.
// Neither an earlier load of the next row, nor more but shorter runs of rows
// for an even end, nor fewer instructions with 20 warps changed that.
template <typename TI, typename TO, bool EXACT>
__global__ void __launch_bounds__(256, 3)
span_softmax_warp_kernel(const __grid_constant__ SpanArgs a, int room) {
  pdl_prologue();
  constexpr int N = Elem<TI>::kVec;
  constexpr int Q = N / 4;  // quads of scores a pack
  extern __shared__ float4 dyn[];
  const int lane = threadIdx.x & 31;
  const uint32_t zeros = make_zeros(dyn);
  // Quad k of pack v at [v / 32][k][v % 32]: neighbouring packs' quads are
  // neighbours.  Lanes past the span's last pack go along (their scores are
  // -inf), so that no pass asks for each lane; room is a multiple of 32.
  constexpr int kBlock = 32 * Q;
  float4* mine = dyn + kZeroBytes / 16 + (threadIdx.x >> 5) * room * Q + lane;
  Rows rows(a);
  if (!rows.more) return;
  const Score<EXACT> score(a);
  uint32_t row = rows.w.row;
  Row r = rows.w.get(a);
  rows.next(a);
  Raw ahead = rows.more ? rows.w.read(a) : Raw{0, 0, 0, 0.f};
  Elems<TI, N> v[2];
  v[0].clear();
  v[1].clear();
  // packs at and at + 32 of a row's span
  auto load = [&](const TI* xr, int at, int count) {
    if (at < count) v[0].load(xr + at * N);
    if (at + 32 < count) v[1].load(xr + (at + 32) * N);
  };
  auto place = [&](uint32_t rw, const Row& rr) {
    return Place<N>(rr, shift_of(static_cast<const TI*>(a.x) + rw * a.ldx), a.cols);
  };
  auto span_at = [&](uint32_t rw, const Place<N>& p) {
    return static_cast<const TI*>(a.x) + rw * a.ldx + (p.p0 * N - p.first);
  };
  Place<N> p = place(row, r);
  const TI* xr = span_at(row, p);
  load(xr, lane, p.count);
  while (true) {
    TO* out = static_cast<TO*>(a.out) + row * a.ldo - p.first;
    clear_outside_bulk<TO, N>(out, p, lane, zeros);
    float m = -INFINITY;
    int at = (p.p0 + lane) * N;
    float4* z4 = mine;
    auto keep = [&](const Elems<TI, N>& in) {
      uint64_t z[N / 2];
      in.to(z);
      m = scores_of<N>(z, at, p, r, score, m);
#pragma unroll
      for (int k = 0; k < Q; ++k)
        z4[k * 32] = make_float4(f2_lo(z[2 * k]), f2_hi(z[2 * k]), f2_lo(z[2 * k + 1]), f2_hi(z[2 * k + 1]));
      z4 += kBlock;
      at += 32 * N;
    };
    const bool more = rows.more;
    const uint32_t then = rows.w.row;
    const Row next(ahead, a.cols);
    Place<N> then_p = p;
    auto turn = [&]() {  // to the next row
      if (!more) return;
      then_p = place(then, next);
      xr = span_at(then, then_p);
      load(xr, lane, then_p.count);
      rows.next(a);
      if (rows.more) ahead = rows.w.read(a);
    };
    if (p.count <= 64) {  // two packs a lane: they stay in registers
      const bool two = p.count > 32;
      uint64_t y[2][1][N / 2];
      v[0].to(y[0][0]);
      m = scores_of<N>(y[0][0], at, p, r, score, m);
      if (two) {
        v[1].to(y[1][0]);
        m = scores_of<N>(y[1][0], at + 32 * N, p, r, score, m);
      }
      m = group_reduce_warp<FastMaxOp, 32>(m);
      float s = exps_of<N, 1, 32>(y[0], 1, m);
      if (two) s += exps_of<N, 1, 32>(y[1], 1, m);
      const float inv = rcp(group_reduce_warp<SumOp, 32>(s));
      if (lane < p.count) put<TO, N>(out, y[0][0], at, p, inv);
      if (lane + 32 < p.count) put<TO, N>(out, y[1][0], at + 32 * N, p, inv);
      turn();
      if (!more) break;
      row = then;
      r = next;
      p = then_p;
      continue;
    }
    for (int done = 0; done < p.count; done += 64) {
      const Elems<TI, N> v0 = v[0], v1 = v[1];
      load(xr, done + 64 + lane, p.count);
      keep(v0);
      if (done + 32 < p.count) keep(v1);
    }
    turn();
    m = group_reduce_warp<FastMaxOp, 32>(m);
    float c = -m * kLog2e;  // as in exps_of
    if (!(fabsf(m) < kWide)) {
      c = 0.f;
      z4 = mine;
      for (int done = 0; done < p.count; done += 32, z4 += kBlock)
        for (int k = 0; k < Q; ++k) {
          const float4 f = z4[k * 32];
          z4[k * 32] = make_float4(f.x - m, f.y - m, f.z - m, f.w - m);
        }
    }
    const uint64_t l2 = f2_make(kLog2e, kLog2e), c2 = f2_make(c, c);
    uint64_t s2[2] = {f2_make(0.f, 0.f), f2_make(0.f, 0.f)};
    z4 = mine;
    for (int done = 0; done < p.count; done += 32, z4 += kBlock) {
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        float4 f = z4[k * 32];
        const uint64_t t0 = f2_fma(f2_make(f.x, f.y), l2, c2), t1 = f2_fma(f2_make(f.z, f.w), l2, c2);
        f = make_float4(ex2(f2_lo(t0)), ex2(f2_hi(t0)), ex2(f2_lo(t1)), ex2(f2_hi(t1)));
        s2[0] = f2_add(s2[0], f2_make(f.x, f.y));
        s2[1] = f2_add(s2[1], f2_make(f.z, f.w));
        z4[k * 32] = f;
      }
    }
    s2[0] = f2_add(s2[0], s2[1]);
    const float inv = rcp(group_reduce_warp<SumOp, 32>(f2_lo(s2[0]) + f2_hi(s2[0])));
    z4 = mine;
    at = (p.p0 + lane) * N;
    for (int left = p.count - lane; left > 0; left -= 32, z4 += kBlock, at += 32 * N) {
      uint64_t z[N / 2];
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        const float4 f = z4[k * 32];
        z[2 * k] = f2_make(f.x, f.y);
        z[2 * k + 1] = f2_make(f.z, f.w);
      }
      put<TO, N>(out, z, at, p, inv);
    }
    if (!more) break;
    row = then;
    r = next;
    p = then_p;
  }
  finish_zeros();
}

// TPR threads a row, VPT packs each, a CTA a row.
template <typename TI, typename TO, bool EXACT, int TPR, int VPT>
__global__ void __launch_bounds__(TPR, TPR <= 256 ? 4 : 1)
span_softmax_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  constexpr int N = Elem<TI>::kVec;
  __shared__ float smem[TPR / 32];
  const int lane = threadIdx.x;
  const uint32_t row = blockIdx.x;
  const Row r = row_of(a, row);
  const Score<EXACT> score(a);
  const TI* xr = static_cast<const TI*>(a.x) + row * a.ldx;
  const int shift = shift_of(xr);
  TO* out = static_cast<TO*>(a.out) + row * a.ldo - shift;
  const Place<N> p(r, shift, a.cols);
  xr += (int64_t)p.p0 * N - shift;
  Elems<TI, N> v[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (lane + i * TPR < p.count) v[i].load(xr + (int64_t)(lane + i * TPR) * N);
    else v[i].clear();
  }
  clear_outside<TO, N, TPR>(out, p, lane);
  uint64_t z[VPT][N / 2];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i * TPR < p.count) {
      v[i].to(z[i]);
      m = scores_of<N>(z[i], (p.p0 + lane + i * TPR) * N, p, r, score, m);
    }
  }
  m = row_reduce<FastMaxOp, TPR, TPR>(m, smem);
  const float inv = 1.f / row_reduce<SumOp, TPR, TPR>(exps_of<N, VPT, TPR>(z, p.count, m), smem);
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (lane + i * TPR < p.count) put<TO, N>(out, z[i], (p.p0 + lane + i * TPR) * N, p, inv);
}

// Rows too long for registers: a CTA of 1024 threads a row, the span read
// twice, the second time from L2.
template <typename TI, typename TO, bool EXACT>
__global__ void __launch_bounds__(1024)
span_softmax_long_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  constexpr int N = Elem<TI>::kVec, TPR = 1024, U = 2;
  __shared__ float smem[TPR / 32];
  const int lane = threadIdx.x;
  const uint32_t row = blockIdx.x;
  const Row r = row_of(a, row);
  const Score<EXACT> score(a);
  const TI* xr = static_cast<const TI*>(a.x) + row * a.ldx;
  const int shift = shift_of(xr);
  TO* out = static_cast<TO*>(a.out) + row * a.ldo - shift;
  const Place<N> p(r, shift, a.cols);
  xr += (int64_t)p.p0 * N - shift;
  float m = -INFINITY, s = 0.f;
  Elems<TI, N> v[U];
  auto load = [&](int vi) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (vi + u * TPR < p.count) v[u].load(xr + (int64_t)(vi + u * TPR) * N);
  };
  load(lane);
  clear_outside<TO, N, TPR>(out, p, lane);
  for (int vi = lane; vi < p.count; vi += U * TPR) {
    Elems<TI, N> w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = v[u];
    load(vi + U * TPR);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (vi + u * TPR >= p.count) continue;
      uint64_t z[1][N / 2];
      w[u].to(z[0]);
      const float top = scores_of<N>(z[0], (p.p0 + vi + u * TPR) * N, p, r, score, m);
      if (top > m) {
        s *= exp_of(m - top);
        m = top;
      }
      // (-inf so far: nothing to add, unless a NaN came without raising the maximum)
      s += exps_from<N>(z[0], m == -INFINITY ? 0.f : m);
    }
  }
  const float top = row_reduce<FastMaxOp, TPR, TPR>(m, smem);
  s = row_reduce<SumOp, TPR, TPR>(m == -INFINITY && s == 0.f ? 0.f : s * exp_of(m - top), smem);
  // (nothing but -inf: 0 / 0 as in softmax)
  const float inv = 1.f / s, base = top == -INFINITY ? 0.f : top;
  for (int vi = lane; vi < p.count; vi += U * TPR) {
    load(vi);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (vi + u * TPR >= p.count) continue;
      uint64_t z[1][N / 2];
      const int at = (p.p0 + vi + u * TPR) * N;
      v[u].to(z[0]);
      (void)scores_of<N>(z[0], at, p, r, score, -INFINITY);
      (void)exps_from<N>(z[0], base);
      put<TO, N>(out, z[0], at, p, inv);
    }
  }
}

// Rows whose output lies otherwise than their input: a CTA a row by single
// elements.
template <typename TI, typename TO, bool EXACT>
__global__ void __launch_bounds__(512)
span_softmax_loop_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  constexpr int BLOCK = 512;
  __shared__ float smem[BLOCK / 32];
  const Score<EXACT> score(a);
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

// One row of the gradient by TPR threads (the CTA, or a warp of it).
// TI: x's and dx's type, TY: y's and dy's.
template <typename TI, typename TY, int TPR, int VPT>
__device__ __forceinline__ void span_bwd_row(const SpanArgs& a, uint32_t row, const Row& r, const Score<false>& score,
                                             int lane, float* smem) {
  constexpr int N = Elem<TI>::kVec;
  const bool capped = score.cap != 0.f;
  TI* out = static_cast<TI*>(a.out) + row * a.ldo;
  const int shift = shift_of(out);
  out -= shift;
  const Place<N> p(r, shift, a.cols);
  const int64_t skip = (int64_t)p.p0 * N - shift;
  const TY* yr = static_cast<const TY*>(a.y) + row * a.ldy + skip;
  const TY* dr = static_cast<const TY*>(a.dy) + row * a.ldd + skip;
  const TI* xr = static_cast<const TI*>(a.x) + (capped ? row * a.ldx + skip : 0);
  Elems<TY, N> y[VPT], d[VPT];
  Elems<TI, N> x[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    if (vi < p.count) {
      load_words(y[i], yr + (int64_t)vi * N, (p.p0 + vi) * N, p);
      load_words(d[i], dr + (int64_t)vi * N, (p.p0 + vi) * N, p);
      if (capped) x[i].load(xr + (int64_t)vi * N);
    } else {
      y[i].clear();
      d[i].clear();
    }
  }
  clear_outside<TI, N, TPR>(out, p, lane);
  uint64_t acc[2] = {f2_make(0.f, 0.f), f2_make(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i * TPR < p.count) {
      const int at = (p.p0 + lane + i * TPR) * N;
      if (!p.inside(at)) {  // what lies outside counts as 0 from here on
        y[i].keep(p.lo - at, p.hi - at);
        d[i].keep(p.lo - at, p.hi - at);
        if (capped) x[i].keep(p.lo - at, p.hi - at);
      }
      uint64_t f[N / 2], g[N / 2];
      y[i].to(f);
      d[i].to(g);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) acc[e & 1] = f2_fma(f[e], g[e], acc[e & 1]);
    }
  }
  acc[0] = f2_add(acc[0], acc[1]);
  const float sum = row_reduce<SumOp, TPR, TPR>(f2_lo(acc[0]) + f2_hi(acc[0]), smem);
  // 1 - tanh^2 = 4 (q - q^2), q = (1 - tanh) / 2
  const float by = capped ? 4.f * a.scale : a.scale;
  const uint64_t minus = f2_make(-sum, -sum), times = f2_make(by, by), one = f2_make(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = lane + i * TPR;
    if (vi < p.count) {
      const int at = (p.p0 + vi) * N;
      uint64_t f[N / 2], g[N / 2];
      y[i].to(f);
      d[i].to(g);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) f[e] = f2_mul(f2_mul(f[e], times), f2_add(g[e], minus));
      if (capped) {
        x[i].to(g);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          const uint64_t q = score.half_of(g[e]);
          f[e] = f2_mul(f[e], f2_fma(f2_mul(q, one), q, q));
        }
      }
      if (!(fabsf(sum) < 3e38f) && !p.inside(at)) p.mask(f, at, 0.f);  // (0 times a sum that is not finite)
      store<TI, N>(out, at, p.first, p.last, f);
    }
  }
}

// A warp a row: y, dy and x (where capped) copied into shared memory by
// cp.async, as many bytes in flight as a row has and no registers for them;
// a lane reads only what it copied.
template <typename TI, typename TY>
__global__ void __launch_bounds__(128, sizeof(TY) == sizeof(TI) ? 7 : 5)
span_softmax_bwd_warp_kernel(const __grid_constant__ SpanArgs a, int room) {
  pdl_prologue();
  constexpr int N = Elem<TI>::kVec;
  constexpr int W = (int)(sizeof(TY) / sizeof(TI));  // 16-byte words of y a pack
  extern __shared__ uint4 words[];
  const int lane = threadIdx.x & 31;
  const Score<false> score(a);
  const bool capped = score.cap != 0.f;
  const uint32_t zeros = make_zeros(words);
  // word k of pack v at [v / 32][k][v % 32]: y's, dy's, x's
  const int kinds = 2 * W + (capped ? 1 : 0);
  uint4* mine = words + kZeroBytes / 16 + (threadIdx.x >> 5) * room * kinds + lane;
  Rows rows(a);
  if (!rows.more) return;
  uint32_t row = rows.w.row;
  Row r = rows.w.get(a);
  const float by = capped ? 4.f * a.scale : a.scale;  // 1 - tanh^2 = 4 (q - q^2), q = (1 - tanh) / 2
  const uint64_t times = f2_make(by, by), minus_one = f2_make(-1.f, -1.f);
  while (true) {
    TI* out = static_cast<TI*>(a.out) + row * a.ldo;
    const int shift = shift_of(out);
    out -= shift;
    const Place<N> p(r, shift, a.cols);
    const int skip = p.p0 * N - shift;
    const TY* yr = static_cast<const TY*>(a.y) + row * a.ldy + skip;
    const TY* dr = static_cast<const TY*>(a.dy) + row * a.ldd + skip;
    const TI* xr = static_cast<const TI*>(a.x) + (capped ? row * a.ldx + skip : 0);
    uint4* w = mine;
    int at = lane * N;
    for (int left = p.count - lane; left > 0; left -= 32, w += 32 * kinds, at += 32 * N) {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        constexpr int VW = Elem<TY>::kVec;
        if (W == 1 || p.meets(p.p0 * N + at + k * VW, VW)) {
          cp_async16(w + k * 32, yr + at + k * VW);
          cp_async16(w + (W + k) * 32, dr + at + k * VW);
        } else {
          w[k * 32] = w[(W + k) * 32] = make_uint4(0, 0, 0, 0);
        }
      }
      if (capped) cp_async16(w + 2 * W * 32, xr + at);
    }
    cp_async_commit();
    rows.next(a);
    const bool more = rows.more;
    const Raw ahead = more ? rows.w.read(a) : Raw{0, 0, 0, 0.f};
    clear_outside_bulk<TI, N>(out, p, lane, zeros);
    cp_async_wait_all();
    Elems<TY, N> y, d;
    auto get = [&]() {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        y.word(k, w[k * 32]);
        d.word(k, w[(W + k) * 32]);
      }
      if (!p.inside(at)) {  // what lies outside counts as 0
        y.keep(p.lo - at, p.hi - at);
        d.keep(p.lo - at, p.hi - at);
      }
    };
    uint64_t acc[2] = {f2_make(0.f, 0.f), f2_make(0.f, 0.f)};
    w = mine;
    at = (p.p0 + lane) * N;
    // (lanes past the span's last pack go along with nothing)
    for (int done = 0; done < p.count; done += 32, w += 32 * kinds, at += 32 * N) {
      get();
      uint64_t f[N / 2], g[N / 2];
      y.to(f);
      d.to(g);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) acc[e & 1] = f2_fma(f[e], g[e], acc[e & 1]);
    }
    acc[0] = f2_add(acc[0], acc[1]);
    const float sum = group_reduce_warp<SumOp, 32>(f2_lo(acc[0]) + f2_hi(acc[0]));
    const uint64_t minus = f2_make(-sum, -sum);
    const bool odd = !(fabsf(sum) < 3e38f);  // 0 times it is not 0
    w = mine;
    at = (p.p0 + lane) * N;
    for (int left = p.count - lane; left > 0; left -= 32, w += 32 * kinds, at += 32 * N) {
      get();
      uint64_t f[N / 2], g[N / 2];
      y.to(f);
      d.to(g);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) f[e] = f2_mul(f2_mul(f[e], times), f2_add(g[e], minus));
      if (capped) {
        Elems<TI, N> x;
        x.word(0, w[2 * W * 32]);
        if (!p.inside(at)) x.keep(p.lo - at, p.hi - at);
        x.to(g);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          const uint64_t q = score.half_of(g[e]);
          f[e] = f2_mul(f[e], f2_fma(f2_mul(q, minus_one), q, q));
        }
      }
      if (odd && !p.inside(at)) p.mask(f, at, 0.f);
      store<TI, N>(out, at, p.first, p.last, f);
    }
    if (!more) break;
    row = rows.w.row;
    r = Row(ahead, a.cols);
  }
  finish_zeros();
}

// A CTA a row.
template <typename TI, typename TY, int TPR, int VPT>
__global__ void __launch_bounds__(TPR, TPR <= 256 ? 2 : 1)
span_softmax_bwd_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  __shared__ float smem[TPR / 32];
  span_bwd_row<TI, TY, TPR, VPT>(a, blockIdx.x, row_of(a, blockIdx.x), Score<false>(a), threadIdx.x, smem);
}

// Rows too long for registers: a CTA of 1024 threads a row, y and dy read
// twice.
template <typename TI, typename TY>
__global__ void __launch_bounds__(1024)
span_softmax_bwd_long_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  constexpr int N = Elem<TI>::kVec, TPR = 1024;
  __shared__ float smem[TPR / 32];
  const int lane = threadIdx.x;
  const uint32_t row = blockIdx.x;
  const Row r = row_of(a, row);
  const Score<false> score(a);
  const bool capped = score.cap != 0.f;
  TI* out = static_cast<TI*>(a.out) + row * a.ldo;
  const int shift = shift_of(out);
  out -= shift;
  const Place<N> p(r, shift, a.cols);
  const int64_t skip = (int64_t)p.p0 * N - shift;
  const TY* yr = static_cast<const TY*>(a.y) + row * a.ldy + skip;
  const TY* dr = static_cast<const TY*>(a.dy) + row * a.ldd + skip;
  const TI* xr = static_cast<const TI*>(a.x) + (capped ? row * a.ldx + skip : 0);
  clear_outside<TI, N, TPR>(out, p, lane);
  uint64_t f[N / 2], g[N / 2], acc[2] = {f2_make(0.f, 0.f), f2_make(0.f, 0.f)};
  auto get = [&](int vi) {
    Elems<TY, N> y, d;
    const int at = (p.p0 + vi) * N;
    load_words(y, yr + (int64_t)vi * N, at, p);
    load_words(d, dr + (int64_t)vi * N, at, p);
    if (!p.inside(at)) {
      y.keep(p.lo - at, p.hi - at);
      d.keep(p.lo - at, p.hi - at);
    }
    y.to(f);
    d.to(g);
  };
#pragma unroll 2
  for (int vi = lane; vi < p.count; vi += TPR) {
    get(vi);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) acc[e & 1] = f2_fma(f[e], g[e], acc[e & 1]);
  }
  acc[0] = f2_add(acc[0], acc[1]);
  const float sum = row_reduce<SumOp, TPR, TPR>(f2_lo(acc[0]) + f2_hi(acc[0]), smem);
  const float by = capped ? 4.f * a.scale : a.scale;
  const uint64_t minus = f2_make(-sum, -sum), times = f2_make(by, by), minus_one = f2_make(-1.f, -1.f);
#pragma unroll 2
  for (int vi = lane; vi < p.count; vi += TPR) {
    const int at = (p.p0 + vi) * N;
    Elems<TI, N> x;
    if (capped) x.load(xr + (int64_t)vi * N);
    get(vi);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) f[e] = f2_mul(f2_mul(f[e], times), f2_add(g[e], minus));
    if (capped) {
      if (!p.inside(at)) x.keep(p.lo - at, p.hi - at);
      x.to(g);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        const uint64_t q = score.half_of(g[e]);
        f[e] = f2_mul(f[e], f2_fma(f2_mul(q, minus_one), q, q));
      }
    }
    if (!(fabsf(sum) < 3e38f) && !p.inside(at)) p.mask(f, at, 0.f);
    store<TI, N>(out, at, p.first, p.last, f);
  }
}

template <typename TI, typename TY>
__global__ void __launch_bounds__(512)
span_softmax_bwd_loop_kernel(const __grid_constant__ SpanArgs a) {
  pdl_prologue();
  constexpr int BLOCK = 512;
  __shared__ float smem[BLOCK / 32];
  const Score<false> score(a);
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

// Calls f(TPR) for rows covered by `packs` packs: a warp up to WARP packs,
// then a CTA of 4 packs a thread; -1: longer than that.
template <int WARP, typename F>
int span_ladder(int64_t packs, F&& f) {
  using std::integral_constant;
  if (packs <= WARP) return f(integral_constant<int, 32>{});
  if constexpr (WARP < 512)
    if (packs <= 512) return f(integral_constant<int, 128>{});
  if (packs <= 1024) return f(integral_constant<int, 256>{});
  if (packs <= 2048) return f(integral_constant<int, 512>{});
  if (packs <= 4096) return f(integral_constant<int, 1024>{});
  return -1;
}
// Packs in whole turns of a warp.
constexpr int room_of(int64_t packs) { return (int)((packs + 31) / 32 * 32); }
// Launches CTAs of BLOCK threads, as many as are resident at once (`most` an
// SM by their registers), with `room` packs of `each` bytes of shared memory a
// warp.  Warps that have many rows take 8 in order.  What the kernel may take
// (MOST bytes) is a constant: it belongs to the function, and another thread
// may be between its own call's setting and launch.
template <int BLOCK, int MOST, typename K>
int launch_warps(K kernel, int most, SpanArgs& a, int room, int each, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kWarps = BLOCK / 32;
  const int smem = room * each * kWarps + kZeroBytes;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST) != cudaSuccess)
    return launch_status();
  const int64_t ctas = (int64_t)std::max(1, std::min(most, 228 * 1024 / (smem + 1024))) * dev.sm_count;
  a.unit = a.rows >= ctas * kWarps * 32 ? 8 : 1;
  launch_k(kernel, (unsigned)std::min<int64_t>(ctas, ceil_div(a.rows, kWarps * a.unit)), BLOCK, smem, stream, a, room);
  return launch_status();
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

// The most packs that cover a row: one more where rows begin inside one.
template <typename T>
int64_t packs_of(const void* p, int64_t ld, int64_t cols, int64_t rows) {
  constexpr int64_t N = Elem<T>::kVec;
  return ceil_div(cols, N) + (aligned16(p) && (rows <= 1 || ld % N == 0) ? 0 : 1);
}

template <typename TI, typename TO, bool EXACT>
int launch_fwd_as(SpanArgs a, const DeviceInfo& dev, cudaStream_t stream) {
  if (in_step<TI, TO>(a.x, a.ldx, a.out, a.ldo, a.rows)) {
    const int64_t packs = packs_of<TI>(a.x, a.ldx, a.cols, a.rows);
    // 65 KB of scores for 8 warps: three CTAs an SM up to 2048 keys
    constexpr int kWarpPacks = 2056 / Elem<TI>::kVec, kEach = Elem<TI>::kVec * 4;
    const int st = span_ladder<kWarpPacks>(packs, [&](auto tpr) -> int {
      constexpr int TPR = decltype(tpr)::value;
      if constexpr (TPR == 32) {
        return launch_warps<256, room_of(kWarpPacks) * kEach * 8 + kZeroBytes>(
            span_softmax_warp_kernel<TI, TO, EXACT>, 3, a, room_of(packs), kEach, dev, stream);
      } else {
        launch_k((span_softmax_kernel<TI, TO, EXACT, TPR, 4>), a.rows, TPR, 0, stream, a);
        return launch_status();
      }
    });
    if (st >= 0) return st;
    launch_k((span_softmax_long_kernel<TI, TO, EXACT>), a.rows, 1024, 0, stream, a);
    return launch_status();
  }
  const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 4ll * dev.sm_count);
  launch_k((span_softmax_loop_kernel<TI, TO, EXACT>), grid, 512, 0, stream, a);
  return launch_status();
}
template <typename TI, typename TO>
int launch_fwd(const SpanArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  const bool exact = a.cap > (std::is_same<TO, float>::value ? 0.f : 256.f);
  return exact ? launch_fwd_as<TI, TO, true>(a, dev, stream) : launch_fwd_as<TI, TO, false>(a, dev, stream);
}

template <typename TI, typename TY>
int launch_bwd(SpanArgs a, const DeviceInfo& dev, cudaStream_t stream) {
  if (in_step<TI, TY>(a.out, a.ldo, a.y, a.ldy, a.rows) && in_step<TI, TY>(a.out, a.ldo, a.dy, a.ldd, a.rows) &&
      (!(a.cap > 0.f) || in_step<TI, TI>(a.out, a.ldo, a.x, a.ldx, a.rows))) {
    const int64_t packs = packs_of<TI>(a.out, a.ldo, a.cols, a.rows);
    // up to 12 KB a warp (20 where y is wider than x): 16 warps an SM
    constexpr int kWarpPacks = 257, kWords = 2 * (int)(sizeof(TY) / sizeof(TI));
    const int st = span_ladder<kWarpPacks>(packs, [&](auto tpr) -> int {
      constexpr int TPR = decltype(tpr)::value;
      if constexpr (TPR == 32) {
        return launch_warps<128, room_of(kWarpPacks) * (kWords + 1) * 16 * 4 + kZeroBytes>(
            span_softmax_bwd_warp_kernel<TI, TY>, sizeof(TY) == sizeof(TI) ? 7 : 5, a, room_of(packs),
            16 * (kWords + (a.cap > 0.f ? 1 : 0)), dev, stream);
      } else {
        launch_k((span_softmax_bwd_kernel<TI, TY, TPR, 4>), a.rows, TPR, 0, stream, a);
        return launch_status();
      }
    });
    if (st >= 0) return st;
    launch_k((span_softmax_bwd_long_kernel<TI, TY>), a.rows, 1024, 0, stream, a);
    return launch_status();
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
  // a score of 0 has to stay one: no infinite factor
  FLB_CHECK_ARG(fabsf(scale) <= 3e38f && (cap == 0.f || fabsf(2.f * kLog2e * (scale / cap)) <= 3e38f));
  if (rows > 0x7fffffff || cols > kMaxCols) return FL_B200_ERR_TOO_LARGE;
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
  // the distance from a position of up to +-2^30 to a key is a 32-bit number
  if (slopes != nullptr && (cols > (1 << 30) - 4096 || q_len > 1 << 30)) return FL_B200_ERR_TOO_LARGE;
  if (!aligned_to(dtype_size(in_dtype), {x}) || !aligned_to(dtype_size(out_dtype), {out}) ||
      !aligned_to(4, {spans, positions, slopes}))
    return FL_B200_ERR_MISALIGNED;
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
  if (!aligned_to(sx, {dx}) || (cap > 0.f && !aligned_to(sx, {x})) || !aligned_to(sy, {dy, y}) || !aligned_to(4, {spans}))
    return FL_B200_ERR_MISALIGNED;
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
