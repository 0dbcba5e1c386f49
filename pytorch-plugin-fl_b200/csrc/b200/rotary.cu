// Rotary positions from positions and frequencies: no table of cosines in
// memory, halves or neighbours paired, the whole head or its first part.
//
//   angle = position * freq[i],  i < rot / 2
//   (a, b) -> scale * (a cos - b sin, b cos + a sin)
//
// with (a, b) = (x[i], x[i + rot/2]) or (x[2i], x[2i+1]); the elements from
// rot on stay as they are.  The inverse turns by -angle and is the adjoint:
// with the same scale it is the gradient.
//
// The angle is taken in fp64 as a fraction of a turn, reduced to half a turn
// there (exact), and only then rounded to fp32 for sincospif: a position of
// 1e6 costs no digit of its cosine (fp32 angles are off by up to 2^-5 of a
// radian there).  The cosines stay fp32 and are scaled once; the rotation is
// fp32 with one rounding to the heads' type.
//
// Bound by memory: every head is read and written once (65536 tokens of 40
// heads of 128 bf16: 212 us, 6.3 TB/s).  A warp takes a token
// (or a part of its heads, for few tokens), its lanes compute the token's
// cosines into shared memory (rot / 64 sincospif a lane, while the first
// packs are on their way) and walk the (head, pack) items; all heads share
// them.  The table's 16-byte chunks of neighbouring packs are neighbours, so
// reading it has no bank conflicts.
#include <numeric>

#include "common.cuh"
#include "heads_place.cuh"

namespace flb200 {
namespace {

struct RotaryArgs {
  const char* in[2];  // q, k
  char* out[2];
  int64_t sb[2], sh[2], ss[2], ob[2], oh[2], os[2];  // bytes
  const void* pos;
  int64_t pb, ps;  // elements
  const float* freq;
  float scale, sign;
  int pos64, q_heads, heads, rot, splits;
  uint32_t tokens, seq;
  int items, copies;        // packs a head that turn (pairs of them where halves are paired) / stay
  uint32_t items_m, copies_m;  // ceil(2^31 / items), ...
  int copy_from, copy_to;   // item range of a token's packs that are copied
  int group;                // tokens a warp
  uint32_t token_m, copy_m;    // ceil(2^31 / a token's items), ... of its copies
  int split_b;              // bytes from a pack to its partner
};

// n / d from m = ceil(2^31 / d), exact while n * d < 2^31.
__device__ __forceinline__ int quotient(int n, uint32_t m) { return (int)(((uint64_t)(uint32_t)n * m) >> 31); }

template <int BYTES>
struct RawOf;
template <>
struct RawOf<16> { using type = uint4; };
template <>
struct RawOf<8> { using type = uint2; };
template <>
struct RawOf<4> { using type = unsigned int; };
template <>
struct RawOf<2> { using type = unsigned short; };

// Loads where they stand, before the work that hides them (an input may be
// its own output: not through the read-only path).
__device__ __forceinline__ void ld_now(uint4& r, const char* p) {
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void ld_now(uint2& r, const char* p) {
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p) : "memory");
}
__device__ __forceinline__ void ld_now(unsigned int& r, const char* p) {
  asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(r) : "l"(p) : "memory");
}
__device__ __forceinline__ void ld_now(unsigned short& r, const char* p) {
  asm volatile("ld.global.L1::no_allocate.u16 %0, [%1];" : "=h"(r) : "l"(p) : "memory");
}

template <typename T, int VEC>
struct Pack {
  using Raw = typename RawOf<VEC * (int)sizeof(T)>::type;
  union {
    Raw raw;
    T e[VEC];
  };
  __device__ __forceinline__ Pack() {}
};

// One chunk of the table: CH of an item's cosines and sines.
template <int CH>
struct alignas(CH * 4) Chunk {
  float v[CH];
};

// VEC elements a pack.  An item is a pack and its partner half a turn part
// away, or (NEIGH) one pack of neighbours; single elements are loaded as
// pairs in both cases.
// 64 registers: 32 warps an SM (65536 tokens of 40 heads of 128 bf16: 212 us,
// with 88 registers and 20 warps 239 us).
// MANY: a warp takes `group` tokens, whose heads have few packs.
template <typename T, int VEC, bool NEIGH, bool MANY>
__global__ void __launch_bounds__(128, 8)
rotary_kernel(const __grid_constant__ RotaryArgs a) {
  pdl_prologue();
  constexpr bool PAIR = !NEIGH || VEC == 1;  // an item is two loads
  constexpr int NE = PAIR ? VEC : VEC / 2;   // angles an item
  constexpr int CH = 2 * NE < 4 ? 2 * NE : 4;
  constexpr int NCH = 2 * NE / CH;
  constexpr int U = PAIR ? 4 : 8;  // items in flight
  constexpr int kSize = (int)sizeof(T);
  extern __shared__ float4 smem4[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = MANY ? a.group : 1;
  float* table = reinterpret_cast<float*>(smem4) + warp * ((group * a.rot + 3) & ~3);
  const uint32_t unit = blockIdx.x * 4u + warp;
  const uint32_t first = MANY ? unit * (uint32_t)group : unit / (uint32_t)a.splits;
  if (first >= a.tokens) return;
  const int part = MANY ? 0 : (int)(unit - first * (uint32_t)a.splits);
  const int here = MANY ? (int)min((uint32_t)group, a.tokens - first) : 1;  // tokens
  const uint32_t b0 = first / a.seq, s0 = first - b0 * a.seq;
  // token `tok` of the warp's
  auto where = [&](int tok, uint32_t* b, uint32_t* s) {
    *b = b0, *s = s0 + tok;
    if constexpr (MANY)
      while (*s >= a.seq) *s -= a.seq, ++*b;
  };
  const char* q_in = a.in[0] + b0 * a.sb[0] + s0 * a.ss[0];
  const char* k_in = a.in[1] + b0 * a.sb[1] + s0 * a.ss[1] - a.q_heads * a.sh[1];
  char* q_out = a.out[0] + b0 * a.ob[0] + s0 * a.os[0];
  char* k_out = a.out[1] + b0 * a.ob[1] + s0 * a.os[1] - a.q_heads * a.oh[1];
  auto head_in = [&](int tok, int h) -> const char* {
    if constexpr (!MANY) return h < a.q_heads ? q_in + h * a.sh[0] : k_in + h * a.sh[1];
    uint32_t b, s;
    where(tok, &b, &s);
    const int t = h >= a.q_heads;
    return (t ? a.in[1] : a.in[0]) + b * a.sb[t] + s * a.ss[t] + (h - (t ? a.q_heads : 0)) * a.sh[t];
  };
  auto head_out = [&](int tok, int h) -> char* {
    if constexpr (!MANY) return h < a.q_heads ? q_out + h * a.oh[0] : k_out + h * a.oh[1];
    uint32_t b, s;
    where(tok, &b, &s);
    const int t = h >= a.q_heads;
    return (t ? a.out[1] : a.out[0]) + b * a.ob[t] + s * a.os[t] + (h - (t ? a.q_heads : 0)) * a.oh[t];
  };
  const int each = a.heads * a.items, copies = a.copy_to - a.copy_from;  // a token's
  const int P = a.items;
  const int total = here * each;
  const int step = a.splits * 32;
  auto offset = [&](int j) { return (NEIGH && VEC == 1 ? 2 * j : j) * VEC * kSize; };
  using Raw = typename Pack<T, VEC>::Raw;
  Pack<T, VEC> lo[U], hi[PAIR ? U : 1];
  auto load = [&](int it0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int it = it0 + u * step;
      if (it < total) {
        const int tok = MANY ? quotient(it, a.token_m) : 0;
        const int of = it - tok * each, h = quotient(of, a.items_m);
        const char* p = head_in(tok, h) + offset(of - h * P);
        ld_now(lo[u].raw, p);
        if constexpr (PAIR) ld_now(hi[u].raw, p + a.split_b);
      }
    }
  };
  int it0 = part * 32 + lane;
  load(it0);
  auto position = [&](uint32_t b, uint32_t s) {
    return a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[b * a.pb + s * a.ps]
                   : (double)static_cast<const int32_t*>(a.pos)[b * a.pb + s * a.ps];
  };
  double pos = MANY ? 0.0 : position(b0, s0);
  for (int f = lane; f < here * (a.rot / 2); f += 32) {
    const int tok = MANY ? f / (a.rot / 2) : 0, i = MANY ? f - tok * (a.rot / 2) : f;
    if constexpr (MANY) {
      uint32_t b, s;
      where(tok, &b, &s);
      pos = position(b, s);
    }
    // in turns; 0.15915494309189535 is 1 / (2 pi)
    double t = pos * (double)__ldg(a.freq + i) * 0.15915494309189535;
    t -= rint(t);
    float sn, cs;
    sincospif((float)(2.0 * t), &sn, &cs);
    float* to = table + tok * a.rot;
    const int j = i / NE, e = i % NE;
    to[((e / CH) * P + j) * CH + e % CH] = cs * a.scale;
    to[(((NE + e) / CH) * P + j) * CH + (NE + e) % CH] = sn * (a.scale * a.sign);
  }
  __syncwarp();
  while (it0 < total) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int it = it0 + u * step;
      if (it >= total) break;
      const int tok = MANY ? quotient(it, a.token_m) : 0;
      const int of = it - tok * each, h = quotient(of, a.items_m), j = of - h * P;
      char* p = head_out(tok, h) + offset(j);
      float cs[2 * NE];
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const Chunk<CH> v = reinterpret_cast<const Chunk<CH>*>(table + tok * a.rot)[c * P + j];
#pragma unroll
        for (int e = 0; e < CH; ++e) cs[c * CH + e] = v.v[e];
      }
      if constexpr (PAIR) {
        Pack<T, VEC> x, y;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float f = Elem<T>::to_f(lo[u].e[e]), g = Elem<T>::to_f(hi[u].e[e]);
          x.e[e] = Elem<T>::from_f(fmaf(f, cs[e], -(g * cs[NE + e])));
          y.e[e] = Elem<T>::from_f(fmaf(g, cs[e], f * cs[NE + e]));
        }
        __stcs(reinterpret_cast<Raw*>(p), x.raw);
        __stcs(reinterpret_cast<Raw*>(p + a.split_b), y.raw);
      } else {
        Pack<T, VEC> x;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const float f = Elem<T>::to_f(lo[u].e[2 * e]), g = Elem<T>::to_f(lo[u].e[2 * e + 1]);
          x.e[2 * e] = Elem<T>::from_f(fmaf(f, cs[e], -(g * cs[NE + e])));
          x.e[2 * e + 1] = Elem<T>::from_f(fmaf(g, cs[e], f * cs[NE + e]));
        }
        __stcs(reinterpret_cast<Raw*>(p), x.raw);
      }
    }
    it0 += U * step;
    load(it0);
  }
  // the rest of each head, where it is not in place already
  for (int c0 = part * 32 + lane; c0 < here * copies; c0 += 8 * step) {
    Raw v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int c = c0 + u * step;
      if (c >= here * copies) break;
      const int tok = MANY ? quotient(c, a.copy_m) : 0;
      const int of = c - tok * copies + a.copy_from, h = quotient(of, a.copies_m);
      ld_now(v[u], head_in(tok, h) + a.rot * kSize + (of - h * a.copies) * (int)sizeof(Raw));
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int c = c0 + u * step;
      if (c >= here * copies) break;
      const int tok = MANY ? quotient(c, a.copy_m) : 0;
      const int of = c - tok * copies + a.copy_from, h = quotient(of, a.copies_m);
      __stcs(reinterpret_cast<Raw*>(head_out(tok, h) + a.rot * kSize) + (of - h * a.copies), v[u]);
    }
  }
}

template <typename T, int VEC, bool NEIGH>
int launch(RotaryArgs a, int64_t head_dim, cudaStream_t stream) {
  DeviceInfo dev;
  int st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  constexpr bool PAIR = !NEIGH || VEC == 1;
  a.items = PAIR ? a.rot / 2 / VEC : a.rot / VEC;
  a.copies = (int)((head_dim - a.rot) / VEC);
  a.split_b = (NEIGH ? 1 : a.rot / 2) * (int)sizeof(T);
  const int64_t most = std::max(a.items, a.copies);
  if (a.heads * most * most >= (1ll << 31)) return FL_B200_ERR_TOO_LARGE;
  a.items_m = (uint32_t)ceil_div(1ll << 31, a.items);
  a.copies_m = a.copies ? (uint32_t)ceil_div(1ll << 31, a.copies) : 0;
  // heads whose rest lies in place already are not copied onto themselves
  a.copy_from = a.in[0] == a.out[0] ? a.q_heads * a.copies : 0;
  a.copy_to = (a.heads > a.q_heads && a.in[1] != a.out[1] ? a.heads : a.q_heads) * a.copies;
  if (a.copy_to < a.copy_from) a.copy_to = a.copy_from;
  const int64_t each = (int64_t)a.heads * a.items;
  // Tokens of few packs (one or two heads) share a warp, whose lanes and loads
  // in flight they would not fill alone, while that leaves 32 warps an SM
  // (100804 tokens of two heads of 80 fp32: 45 us, a warp each 73 us).
  a.group = (int)std::max<int64_t>(1, std::min({(int64_t)8, (int64_t)(128 / each), (int64_t)(2048 / a.rot),
                                                (int64_t)a.tokens / (32 * dev.sm_count)}));
  // (quotients of a warp's copied packs stay exact)
  if (a.copy_to - a.copy_from > 8192) a.group = 1;
  if (a.group > 1) {
    a.splits = 1;
    a.token_m = (uint32_t)ceil_div(1ll << 31, each);
    a.copy_m = a.copy_to > a.copy_from ? (uint32_t)ceil_div(1ll << 31, a.copy_to - a.copy_from) : 0;
    const size_t smem = 4 * ((a.group * a.rot + 3) & ~3) * sizeof(float);
    launch_k((rotary_kernel<T, VEC, NEIGH, true>), (unsigned)ceil_div(ceil_div(a.tokens, a.group), 4), 128, smem,
             stream, a);
    return launch_status();
  }
  // A warp a token leaves most of the GPU idle below 16 warps an SM; then a
  // token's items are dealt to as many warps as have 32 of them.
  const int64_t want = ceil_div(16ll * dev.sm_count, a.tokens);
  a.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, ceil_div(each, 32)));
  const int64_t units = (int64_t)a.tokens * a.splits;
  const size_t smem = 4 * ((a.rot + 3) & ~3) * sizeof(float);
  launch_k((rotary_kernel<T, VEC, NEIGH, false>), (unsigned)ceil_div(units, 4), 128, smem, stream, a);
  return launch_status();
}

template <typename T, bool NEIGH>
int by_width(const RotaryArgs& a, int64_t head_dim, int64_t unit, cudaStream_t stream) {
  const int64_t vec = unit / (int64_t)sizeof(T);
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return launch<T, 8, NEIGH>(a, head_dim, stream);
  if (vec == 4) return launch<T, 4, NEIGH>(a, head_dim, stream);
  if (vec == 2) return launch<T, 2, NEIGH>(a, head_dim, stream);
  return launch<T, 1, NEIGH>(a, head_dim, stream);
}

}  // namespace
}  // namespace flb200

extern "C" FL_B200_API int fl_b200_rotary(
    const void* q, void* q_out, int64_t Hq, int64_t sqb, int64_t sqh, int64_t sqs, int64_t soqb, int64_t soqh,
    int64_t soqs, const void* k, void* k_out, int64_t Hk, int64_t skb, int64_t skh, int64_t sks, int64_t sokb,
    int64_t sokh, int64_t soks, const void* positions, int64_t spb, int64_t sps, int pos_dtype,
    const float* inv_freq, int64_t rot, float scale, int interleaved, int inverse, int64_t B, int64_t S,
    int64_t D, int dtype, fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(B >= 0 && S >= 0 && D >= 0 && Hq >= 0 && Hk >= 0);
  FLB_CHECK_ARG(rot >= 2 && rot % 2 == 0 && rot <= D);
  if (!is_float_dtype(dtype) || (pos_dtype != FL_B200_I32 && pos_dtype != FL_B200_I64))
    return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (k == nullptr) Hk = 0;
  if (B == 0 || S == 0 || D == 0 || Hq + Hk == 0) return FL_B200_OK;
  FLB_CHECK_ARG((Hq == 0 || (q && q_out)) && (Hk == 0 || k_out) && positions && inv_freq);
  FLB_CHECK_ARG(sqb >= 0 && sqh >= 0 && sqs >= 0 && skb >= 0 && skh >= 0 && sks >= 0 && spb >= 0 && sps >= 0 &&
                soqb >= 0 && soqh >= 0 && soqs >= 0 && sokb >= 0 && sokh >= 0 && soks >= 0);
  if (rot > FL_B200_ROTARY_MAX || Hq + Hk > (1 << 20) || D > (1 << 20) || B > 0x7fffffff / S)
    return FL_B200_ERR_TOO_LARGE;
  const int64_t size = dtype_size(dtype);
  if ((Hq && !aligned_to(size, {q, q_out})) || (Hk && !aligned_to(size, {k, k_out})) || !aligned_to(4, {inv_freq}) ||
      !aligned_to(dtype_size(pos_dtype), {positions}))
    return FL_B200_ERR_MISALIGNED;
  RotaryArgs a = {};
  int64_t unit = 16;  // every address is a multiple of it
  Heads ins[2], outs[2];
  const auto meeting = [&](const void* p, const Heads& x, const void* r, const Heads& y) {
    return meet((int64_t)(reinterpret_cast<uintptr_t>(r) - reinterpret_cast<uintptr_t>(p)), x, y, D * size);
  };
  auto tensor = [&](int t, const void* in, void* out, int64_t H, const int64_t (&si)[3], const int64_t (&so)[3]) {
    if (H == 0) return true;
    const bool same = in == out;
    const int64_t n[3] = {B, H, S};
    for (int d = 0; d < 3; ++d) {
      ins[t].n[d] = outs[t].n[d] = n[d];
      ins[t].st[d] = si[d] * size, outs[t].st[d] = so[d] * size;
      if (n[d] == 1) continue;
      if (same && si[d] != so[d]) return false;
      unit = std::gcd(unit, std::gcd(si[d] * size, so[d] * size));
    }
    if (meets_itself(outs[t], D * size) || (!same && meeting(in, ins[t], out, outs[t]))) return false;
    unit = std::gcd(unit, (int64_t)((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15));
    a.in[t] = static_cast<const char*>(in);
    a.out[t] = static_cast<char*>(out);
    a.sb[t] = si[0] * size, a.sh[t] = si[1] * size, a.ss[t] = si[2] * size;
    a.ob[t] = so[0] * size, a.oh[t] = so[1] * size, a.os[t] = so[2] * size;
    return true;
  };
  FLB_CHECK_ARG(tensor(0, q, q_out, Hq, {sqb, sqh, sqs}, {soqb, soqh, soqs}));
  FLB_CHECK_ARG(tensor(1, k, k_out, Hk, {skb, skh, sks}, {sokb, sokh, soks}));
  if (Hq && Hk)
    FLB_CHECK_ARG(!meeting(q_out, outs[0], k_out, outs[1]) && !meeting(q_out, outs[0], k, ins[1]) &&
                  !meeting(k_out, outs[1], q, ins[0]));
  unit = std::gcd(unit, std::gcd((D - rot) * size, (interleaved ? rot : rot / 2) * size));
  a.pos = positions, a.pb = spb, a.ps = sps, a.pos64 = pos_dtype == FL_B200_I64;
  a.freq = inv_freq, a.scale = scale, a.sign = inverse ? -1.f : 1.f;
  a.q_heads = (int)Hq, a.heads = (int)(Hq + Hk), a.rot = (int)rot;
  a.tokens = (uint32_t)(B * S), a.seq = (uint32_t)S;
  auto* s = static_cast<cudaStream_t>(stream);
  return dispatch_float(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    return interleaved ? by_width<T, true>(a, D, unit, s) : by_width<T, false>(a, D, unit, s);
  });
}
