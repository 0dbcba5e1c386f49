// Verification of drafted tokens (speculative sampling) from given uniform
// numbers.
//
// Sequence b has n = lens[b] <= K drafted tokens x_i, the target's
// probabilities p_i over the vocabulary at each of them and after the last,
// and the draft model's q_i.  x_i is kept while u_i q_i(x_i) < p_i(x_i), in
// order; the next token then comes from
//   the residual max(p_i - q_i, 0) at the first token turned down, or
//   p_n when all were kept,
// by the inverse of its cumulative sum at the sequence's last uniform
// number.  Tokens so chosen are distributed as the target's own samples.
//
// Without q (drafts that come with no probabilities) q_i is 1 at x_i: kept
// with probability p_i(x_i), and the residual is p_i without x_i.
//
// The sampled token does not depend on the order of the sums: probabilities
// are held as whole multiples of 2^-36 (rounded to nearest, clamped to
// [0, 1], NaN as 0), differences and sums are 64-bit integers, and the
// uniform number is a whole multiple t of 2^-24, so the token is the first
// whose cumulative sum exceeds floor(t W / 2^24) of the total W.  The product
// u q is compared in fp64, where it is exact.  A residual without mass falls
// back to p; a row of p without mass gives -1.
#include "vocab_rows.cuh"

namespace flb200 {
namespace {

constexpr int kBlock = 256;
constexpr int kWarps = kBlock / 32;

__device__ __forceinline__ long long fixed(float p) {
  return __float2ll_rn(__saturatef(p) * 68719476736.0f);  // 2^36: an exact product
}

template <typename T>
struct VerifyArgs {
  const int64_t* ids;
  int64_t ld_ids;
  const T* p;
  int64_t spb, sps;
  const T* q;
  int64_t sqb, sqs;
  const float* u;
  int64_t ld_u;
  const int64_t* lens;
  int drafts, vocab;
  int64_t* tokens;
  int64_t* accepted;
};

__device__ __forceinline__ long long warp_sum64(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The row that the next token is drawn from: weights p, p - q where that is
// positive, or p without one token.
template <typename T>
struct Row {
  const T* p;
  const T* q;   // null: nothing subtracted
  int without;  // an index whose weight is 0, or -1

  __device__ __forceinline__ static long long excess(T p, T q) {
    const long long d = fixed(Elem<T>::to_f(p)) - fixed(Elem<T>::to_f(q));
    return d > 0 ? d : 0;
  }
  __device__ __forceinline__ long long weight(int i) const {
    if (q != nullptr) return excess(p[i], q[i]);
    return i == without ? 0 : fixed(Elem<T>::to_f(p[i]));
  }

  // This lane's part of the weights of packs [from, to) of the row's split,
  // of which q's are packs too when `packed`.
  __device__ __forceinline__ long long sum(const RowSplit& sp, int from, int to, bool packed) const {
    constexpr int VW = Elem<T>::kVec;
    constexpr int U = 4;
    const int lane = threadIdx.x & 31;
    long long s = 0;
    const uint4* pv = reinterpret_cast<const uint4*>(p + sp.head);
    const auto add = [&](const uint4& a) {
      float f[VW];
      unpack<T>(a, f);
#pragma unroll
      for (int j = 0; j < VW; ++j) s += fixed(f[j]);
    };
    const auto add2 = [&](const uint4& a, const uint4& b) {
      float f[VW], g[VW];
      unpack<T>(a, f);
      unpack<T>(b, g);
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        const long long d = fixed(f[j]) - fixed(g[j]);
        s += d > 0 ? d : 0;
      }
    };
    if (q == nullptr) {
      for (int i = from + lane; i < to; i += 32 * U) {
        uint4 a[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
          a[k] = i + 32 * k < to ? ld_cached(pv + i + 32 * k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < U; ++k) add(a[k]);
      }
      const int x = without - sp.head;  // (a single element's owner leaves it out itself)
      if (lane == 0 && x >= from * VW && x < to * VW) s -= fixed(Elem<T>::to_f(p[without]));
    } else if (packed) {
      const uint4* qv = reinterpret_cast<const uint4*>(q + sp.head);
      // one pack of each ahead: four at once, then summed, were no faster
      const auto get = [&](const uint4* v, int i) {
        return i < to ? ld_cached(v + i) : make_uint4(0, 0, 0, 0);
      };
      int i = from + lane;
      uint4 a = get(pv, i), b = get(qv, i);
      for (; i - lane < to; i += 64) {
        const uint4 c = get(pv, i + 32), d = get(qv, i + 32);
        add2(a, b);
        a = get(pv, i + 64);
        b = get(qv, i + 64);
        add2(c, d);
      }
    } else {
      const int end = sp.head + to * VW;
      for (int e = sp.head + from * VW + lane; e < end; e += 32 * 2 * U) {
        T a[2 * U], b[2 * U];
#pragma unroll
        for (int k = 0; k < 2 * U; ++k) {
          const bool in = e + 32 * k < end;
          a[k] = in ? p[e + 32 * k] : Elem<T>::from_f(0.f);
          b[k] = in ? q[e + 32 * k] : Elem<T>::from_f(0.f);
        }
#pragma unroll
        for (int k = 0; k < 2 * U; ++k) s += excess(a[k], b[k]);
      }
    }
    return s;
  }
};

// A cluster of CTAs a sequence.  Every CTA judges the drafts for itself; the
// row is cut into one segment a warp, in index order, and each warp sums its
// own; the CTAs' totals meet through distributed shared memory, and the CTA
// that has the mark walks the one segment that holds it again.  Bound by the
// latency of these steps in turn, then by HBM: 256 sequences of 5 drafts over
// 128256 fp32 in 47 us (197 MB read: 4.2 TB/s), one over 32000 in 5.2 us.  The
// pipe that converts to 64-bit integers is busy 17% of the time.
template <typename T>
__global__ void __launch_bounds__(kBlock, 4) verify_kernel(VerifyArgs<T> a) {
  constexpr int VW = Elem<T>::kVec;
  __shared__ long long part[kWarps];
  __shared__ long long mine[2];  // this CTA's total, of either attempt
  __shared__ int kept;
  pdl_prologue();
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int64_t b = cluster_id();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t* ids = a.ids + b * a.ld_ids;
  const float* u = a.u + b * a.ld_u;
  int n = a.drafts;
  const int64_t len = a.lens != nullptr ? a.lens[b] : n;
  if (warp == 0) {
    int at = 0;
    // (the loads of a draft do not wait for the length: two trips to memory,
    // not three)
    for (; at < a.drafts; at += 32) {
      const int i = at + lane;
      bool ok = true;
      if (i < a.drafts) {
        const int64_t x = ids[i];
        const float ui = u[i];
        ok = false;
        if (x >= 0 && x < a.vocab) {
          const float pt = __saturatef(Elem<T>::to_f(a.p[b * a.spb + i * a.sps + x]));
          const float qt =
              a.q != nullptr ? __saturatef(Elem<T>::to_f(a.q[b * a.sqb + i * a.sqs + x])) : 1.f;
          ok = (double)fmaxf(ui, 0.f) * (double)qt < (double)pt;
        }
        ok = ok || i >= len;
      }
      const uint32_t no = __ballot_sync(0xffffffffu, !ok);
      if (no != 0) {
        at += __ffs(no) - 1;
        break;
      }
    }
    n = (int)min((int64_t)n, max((int64_t)0, len));
    if (lane == 0) kept = min(at, n);
  }
  n = (int)min((int64_t)a.drafts, max((int64_t)0, len));
  __syncthreads();
  const int count = kept;
  const bool cut = count < n;
  Row<T> r = {a.p + b * a.spb + count * a.sps, nullptr, -1};
  if (cut && a.q != nullptr) r.q = a.q + b * a.sqb + count * a.sqs;
  if (cut && a.q == nullptr) {
    const int64_t x = ids[count];
    r.without = x >= 0 && x < a.vocab ? (int)x : -1;
  }
  const RowSplit sp = split_row(r.p, a.vocab);
  const bool packed = ((reinterpret_cast<uintptr_t>(r.p) ^ reinterpret_cast<uintptr_t>(r.q)) & 15u) == 0;
  const int segments = C * kWarps, seg = rank * kWarps + warp;
  const int per = (sp.nvec + segments - 1) / segments;
  const int from = min(sp.nvec, seg * per), to = min(sp.nvec, from + per);
  long long before = 0, total = 0;  // weights ahead of this CTA's, of the row
  for (int attempt = 0; attempt < 2; ++attempt) {
    long long s = r.sum(sp, from, to, packed);
    // the row's single elements belong to its first and last segment
    if (seg == 0 && lane < sp.head) s += r.weight(lane);
    if (seg == segments - 1 && lane < sp.tail) s += r.weight(a.vocab - sp.tail + lane);
    s = warp_sum64(s);
    if (lane == 0) part[warp] = s;
    __syncthreads();
    before = total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += part[w];
    if (C > 1) {
      if (tid == 0) mine[attempt] = total;
      cluster_sync_all();
      const long long v = lane < C ? ld_remote_s64(remote_smem(&mine[attempt], lane)) : 0;
      before = warp_sum64(lane < rank ? v : 0);
      total = warp_sum64(v);
    }
    if (total > 0 || !cut) break;
    r.q = nullptr;  // nothing left of the residual
    r.without = -1;
    __syncthreads();
  }
  if (C > 1) cluster_sync_all();  // the totals are read: no CTA leaves before
  if (rank == 0) {
    for (int i = tid; i <= a.drafts; i += kBlock) {
      if (i < count) a.tokens[b * (a.drafts + 1) + i] = ids[i];
      if (i > count || (i == count && total == 0)) a.tokens[b * (a.drafts + 1) + i] = -1;
    }
    if (tid == 0) a.accepted[b] = count;
  }
  if (total == 0) return;
  const float us = __saturatef(u[a.drafts]);
  const unsigned long long t = min((unsigned long long)(us * 16777216.0f), 16777215ull);
  const unsigned long long hi = __umul64hi(t, (unsigned long long)total);
  long long mark = (long long)((hi << 40) | ((t * (unsigned long long)total) >> 24)) - before;
  // the warp whose segment holds the mark, if it is one of this CTA's
  int w = 0;
  while (w < kWarps && mark >= part[w]) mark -= part[w++];
  if (mark < 0 || w == kWarps) return;
  const int at = rank * kWarps + w;
  const int first = at == 0 ? 0 : sp.head + min(sp.nvec, at * per) * VW;
  const int last = at == segments - 1 ? a.vocab : sp.head + min(sp.nvec, (at + 1) * per) * VW;
  // the CTA walks that segment again, E elements a thread
  constexpr int E = 8;
  for (int base = first; base < last; base += kBlock * E) {
    const int i = base + tid * E;
    long long v[E], sum = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      v[j] = i + j < last ? r.weight(i + j) : 0;
      sum += v[j];
    }
    long long upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();  // part has been read
    if (lane == 31) part[warp] = upto;
    __syncthreads();
    long long c = upto - sum, round = 0;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      if (x < warp) c += part[x];
      round += part[x];
    }
    if (mark < round) {
      if (c <= mark && mark < c + sum) {
        int more = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          c += v[j];
          more += c <= mark;
        }
        a.tokens[b * (a.drafts + 1) + count] = i + more;
      }
      return;
    }
    mark -= round;
  }
}

}  // namespace
}  // namespace flb200

extern "C" {

FL_B200_API int fl_b200_verify_draft(const int64_t* draft_ids, int64_t ld_ids, const void* p,
                                     int64_t p_stride_b, int64_t p_stride_i, const void* q,
                                     int64_t q_stride_b, int64_t q_stride_i, const float* uniform,
                                     int64_t ld_u, const int64_t* lens, int64_t batch,
                                     int64_t drafts, int64_t vocab, int64_t* tokens,
                                     int64_t* accepted, int dtype, fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(batch >= 0 && drafts >= 0 && vocab >= 0);
  if (!is_float_dtype(dtype)) return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (batch > 0x7fffffffLL || drafts > 0x7fffffLL || vocab > 0x3ffffffLL)
    return FL_B200_ERR_TOO_LARGE;
  if (batch == 0) return FL_B200_OK;
  FLB_CHECK_ARG(vocab > 0 && p && uniform && tokens && accepted && (drafts == 0 || draft_ids));
  FLB_CHECK_ARG(ld_ids >= 0 && p_stride_b >= 0 && p_stride_i >= 0 && q_stride_b >= 0 &&
                q_stride_i >= 0 && ld_u >= 0);
  DeviceInfo dev;
  const int st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  return dispatch_float(dtype, [&](auto t) {
    using T = decltype(t);
    VerifyArgs<T> a = {draft_ids, ld_ids, reinterpret_cast<const T*>(p), p_stride_b, p_stride_i,
                       reinterpret_cast<const T*>(q), q_stride_b, q_stride_i, uniform, ld_u, lens,
                       (int)drafts, (int)vocab, tokens, accepted};
    // up to 8 CTAs a sequence, with three packs a thread at least, while all
    // of them are resident at once (a sequence alone: 5.3 us with 8, 8.5 us
    // with one; 500 sequences over 32000 float32: 24 us with one, 49 us with 8)
    int cluster = 1;
    while (cluster < 8 && batch * cluster * 2 <= 4 * dev.sm_count &&
           vocab / (cluster * 2) >= 3 * kBlock * Elem<T>::kVec)
      cluster *= 2;
    if (batch * cluster > 0x7fffffffLL) return (int)FL_B200_ERR_TOO_LARGE;
    return launch_cluster(verify_kernel<T>, batch * cluster, cluster, kBlock, 0, (cudaStream_t)stream, a);
  });
}

}  // extern "C"
