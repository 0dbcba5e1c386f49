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

constexpr int kBlock = 512;
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

// What the row's weights are made of once the drafts are judged.
template <typename T>
struct Row {
  const T* p;
  const T* q;    // null: no subtraction
  int without;   // an index whose weight is 0, or -1
  __device__ long long weight(int i) const {
    const long long w = fixed(Elem<T>::to_f(p[i]));
    if (q != nullptr) return max(w - fixed(Elem<T>::to_f(q[i])), 0LL);
    return i == without ? 0 : w;
  }
};

__device__ __forceinline__ long long warp_sum64(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One CTA a sequence.  Warp w sums the w-th slice of the row; the warp whose
// slice holds the mark walks it again in index order.
template <typename T>
__global__ void __launch_bounds__(kBlock) verify_kernel(VerifyArgs<T> a) {
  __shared__ long long part[kWarps];
  __shared__ int kept;
  pdl_prologue();
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t* ids = a.ids + b * a.ld_ids;
  const float* u = a.u + b * a.ld_u;
  int n = a.drafts;
  if (a.lens != nullptr) n = (int)min((int64_t)a.drafts, max((int64_t)0, a.lens[b]));
  if (warp == 0) {
    int at = 0;
    for (; at < n; at += 32) {
      const int i = at + lane;
      bool ok = i >= n;
      if (!ok) {
        const int64_t x = ids[i];
        if (x >= 0 && x < a.vocab) {
          const float pt = __saturatef(Elem<T>::to_f(a.p[b * a.spb + i * a.sps + x]));
          const float qt =
              a.q != nullptr ? __saturatef(Elem<T>::to_f(a.q[b * a.sqb + i * a.sqs + x])) : 1.f;
          ok = (double)fmaxf(u[i], 0.f) * (double)qt < (double)pt;
        }
      }
      const uint32_t no = __ballot_sync(0xffffffffu, !ok);
      if (no != 0) {
        at += __ffs(no) - 1;
        break;
      }
    }
    if (lane == 0) kept = min(at, n);
  }
  __syncthreads();
  const int count = kept;
  const bool cut = count < n;
  Row<T> r = {a.p + b * a.spb + count * a.sps, nullptr, -1};
  if (cut && a.q != nullptr) r.q = a.q + b * a.sqb + count * a.sqs;
  if (cut && a.q == nullptr) {
    const int64_t x = ids[count];
    r.without = x >= 0 && x < a.vocab ? (int)x : -1;
  }
  const int per = (a.vocab + kWarps - 1) / kWarps;
  const int from = min(a.vocab, warp * per), to = min(a.vocab, from + per);
  long long total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    long long s = 0;
    for (int i = from + lane; i < to; i += 32) s += r.weight(i);
    s = warp_sum64(s);
    __syncthreads();
    if (lane == 0) part[warp] = s;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kWarps; ++w) total += part[w];
    if (total > 0 || !cut) break;
    r.q = nullptr;  // nothing left of the residual
    r.without = -1;
  }
  for (int i = tid; i <= a.drafts; i += kBlock) {
    if (i < count) a.tokens[b * (a.drafts + 1) + i] = ids[i];
    if (i > count || (i == count && total == 0)) a.tokens[b * (a.drafts + 1) + i] = -1;
  }
  if (tid == 0) a.accepted[b] = count;
  if (total == 0) return;
  const float us = __saturatef(u[a.drafts]);
  const unsigned long long t = min((unsigned long long)(us * 16777216.0f), 16777215ull);
  const unsigned long long hi = __umul64hi(t, (unsigned long long)total);
  const long long mark = (long long)((hi << 40) | ((t * (unsigned long long)total) >> 24));
  long long before = 0;
  for (int w = 0; w < warp; ++w) before += part[w];
  if (mark < before || mark >= before + part[warp]) return;
  for (int i = from; i < to; i += 32) {
    const long long w = i + lane < to ? r.weight(i + lane) : 0;
    long long sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const uint32_t over = __ballot_sync(0xffffffffu, before + sum > mark);
    if (over != 0) {
      if (lane == 0) a.tokens[b * (a.drafts + 1) + count] = i + __ffs(over) - 1;
      return;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
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
  return dispatch_float(dtype, [&](auto t) {
    using T = decltype(t);
    VerifyArgs<T> a = {draft_ids, ld_ids, reinterpret_cast<const T*>(p), p_stride_b, p_stride_i,
                       reinterpret_cast<const T*>(q), q_stride_b, q_stride_i, uniform, ld_u, lens,
                       (int)drafts, (int)vocab, tokens, accepted};
    launch_k(verify_kernel<T>, dim3((unsigned)batch), dim3(kBlock), 0, (cudaStream_t)stream, a);
    return launch_status();
  });
}

}  // extern "C"
