// The k largest elements of each row with their indices, and the gradient.
//
// Order: descending by value; equal values (and -0 and +0) by ascending
// index; NaN counts as larger than everything, as in argmax.  Every element
// therefore has a distinct 64-bit key, (ordered value bits, ~index), and the
// result is the k largest keys in descending order: one right answer.
#include "vocab_rows.cuh"

namespace flb200 {
namespace {

constexpr int kMaxTop = FL_B200_TOPK_MAX;
constexpr int kPacks = 8;     // 16-byte packs a thread has in flight
constexpr int kCap = 2048;    // candidates kept
constexpr int kShared = 512;  // the longest list that clusters exchange
constexpr int kRank = 128;    // up to as many keys are placed by counting the larger ones, more are sorted

// Monotone 32-bit image of a value: unsigned order is float order, NaN on
// top; never 0.
__device__ __forceinline__ uint32_t value_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);  // -0 -> +0
  if (f != f) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// The value with that key (NaN for 0, which no value has).
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ uint64_t element_key(float f, uint32_t index) {
  return ((uint64_t)value_key(f) << 32) | (uint32_t)~index;
}

// NaN-propagating maximum of the elements in two words, element by element
// (two 16-bit elements a word), and of the elements of one word.
template <typename T>
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, float>::value) {
    asm("{ .reg .f32 x, y, z; mov.b32 x, %1; mov.b32 y, %2; max.NaN.f32 z, x, y; mov.b32 %0, z; }"
        : "=r"(r)
        : "r"(a), "r"(b));
  } else if constexpr (std::is_same<T, __half>::value) {
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  } else {
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ float word_top(uint32_t w) {
  if constexpr (std::is_same<T, float>::value) {
    return __uint_as_float(w);
  } else {
    const uint64_t p = pair_from_bits<T>(w);
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(f2_lo(p)), "f"(f2_hi(p)));
    return r;
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack_max(const uint4& u) {
  return word_max<T>(word_max<T>(u.x, u.y), word_max<T>(u.z, u.w));
}
// Word of -infinities.
template <typename T>
__device__ __forceinline__ uint32_t word_lowest() {
  return std::is_same<T, float>::value ? 0xff800000u
         : std::is_same<T, __half>::value ? 0xfc00fc00u
                                          : 0xff80ff80u;
}

// B threads a CTA.
template <int B>
struct Shared {
  static constexpr int kWarps = B / 32;
  static constexpr int kChunk = B * kPacks;  // packs after which the groups repeat
  uint64_t cand[kCap];  // candidates, in no order
  union {
    uint64_t top[kShared];  // this slice's largest, for CTA 0
    uint16_t list[kChunk];  // groups of packs that hold candidates
  };
  int2 sums[2][kWarps];
  uint32_t run[B];  // the threads' maxima
  int hist[256];
  uint32_t least;  // collect's threshold
  int filled, listed, pick, above;
  uint4 stage[kPacks][B];  // packs on their way, each thread its own
};

// `n` more of `*counter`: the old value.  (Inline: these are rare, and what
// the compiler does to share one atomic among a warp's lanes costs more than
// it saves.)
__device__ __forceinline__ int take_slots(int* counter, int n) {
  int slot;
  asm volatile("atom.shared.add.s32 %0, [%1], %2;"
               : "=r"(slot)
               : "r"((uint32_t)__cvta_generic_to_shared(counter)), "r"(n)
               : "memory");
  return slot;
}
__device__ __forceinline__ int take_slot(int* counter) { return take_slots(counter, 1); }

// Sums over the CTA, in every thread, of three counts (at most 2^15 in all)
// given as (first, second << 16) and third.  `parity` alternates between the
// two halves of the scratch, so that one barrier a call is enough.
template <int B>
__device__ __forceinline__ void block_sum3(Shared<B>& s, int& n12, int& n3, int& parity) {
  constexpr int kWarps = B / 32;
  const int lane = threadIdx.x & 31;
  n12 = __reduce_add_sync(0xffffffffu, n12);
  n3 = __reduce_add_sync(0xffffffffu, n3);
  if (lane == 0) s.sums[parity][threadIdx.x >> 5] = make_int2(n12, n3);
  __syncthreads();
  const int2 v = lane < kWarps ? s.sums[parity][lane] : make_int2(0, 0);
  n12 = __reduce_add_sync(0xffffffffu, v.x);
  n3 = __reduce_add_sync(0xffffffffu, v.y);
  parity ^= 1;
}

// A key K that at least k of the counted keys reach, and at most `enough`
// where that is possible: found from the top, two bits a step.  visit(see)
// calls see for each of the thread's own keys.
template <int B, typename F>
__device__ __forceinline__ uint32_t bisect(Shared<B>& s, int k, int enough, int& parity, F visit) {
  uint32_t at = 0;
  for (int bit = 30; bit >= 0; bit -= 2) {
    const uint32_t one = 1u << bit;
    int n12 = 0, n3 = 0;
    visit([&](uint32_t key) {
      n12 += (key >= at + one) + ((key >= at + 2 * one) << 16);
      n3 += key >= at + 3 * one;
    });
    block_sum3(s, n12, n3, parity);
    const int n1 = n12 & 0xffff, n2 = n12 >> 16;
    const int reached = n3 >= k ? n3 : n2 >= k ? n2 : n1 >= k ? n1 : 0;
    at += n3 >= k ? 3 * one : n2 >= k ? 2 * one : n1 >= k ? one : 0;
    if (reached != 0 && reached <= enough) break;
  }
  return at;
}

template <int B>
__device__ __forceinline__ void append(Shared<B>& s, uint64_t key) {
  const int slot = take_slot(&s.filled);
  if (slot < kCap) s.cand[slot] = key;
}

// Descending bitonic sort, N neighbours a thread, t its place.  Partners in
// two lanes meet by shuffles, those in two warps through shared memory (ten
// barriers for eight warps; with one a step, after a search for the cut, 64 x
// 32000 float32, top 1000, took 44 us, now 30).  Above 128 keys it beats
// counting (1 x 5289 float32, top 120: 9.0 us, 11.8), below it does not (4096 x
// 128256 bf16, top 64: 214 us, counted 178).
template <typename K>
__device__ __forceinline__ void order(K& a, K& b, bool larger_first) {
  const K hi = a > b ? a : b, lo = a > b ? b : a;
  a = larger_first ? hi : lo;
  b = larger_first ? lo : hi;
}
// The steps of one merge of `lanes` lanes' keys.
template <int N, typename K>
__device__ __forceinline__ void merge_lanes(K (&v)[N], int lane, int lanes, bool down) {
#pragma unroll 1
  for (int other = lanes >> 1; other > 0; other >>= 1) {
    const bool larger = ((lane & other) == 0) == down;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const K o = __shfl_xor_sync(0xffffffffu, v[i], other);
      v[i] = (o > v[i]) == larger ? o : v[i];
    }
  }
#pragma unroll
  for (int stride = N >> 1; stride > 0; stride >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & stride) == 0) order(v[i], v[i + stride], down);
  }
}
// A warp's 32 N keys, the largest first where bit 5 of t is 0, else last.
template <int N, typename K>
__device__ __forceinline__ void sort_lanes(K (&v)[N], int t) {
#pragma unroll
  for (int size = 2; size <= N; size <<= 1) {
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((i & stride) == 0) order(v[i], v[i + stride], ((t * N + i) & size) == 0);
    }
  }
#pragma unroll 1
  for (int lanes = 2; lanes <= 32; lanes <<= 1) merge_lanes(v, t, lanes, (t & lanes) == 0);
}
// n <= 32 N keys, by a warp.
template <int N>
__device__ __forceinline__ void warp_sort(uint64_t* keys, int n, int lane) {
  uint64_t v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane * N + i < n ? keys[lane * N + i] : 0;
  sort_lanes(v, lane);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < N; ++i) keys[lane * N + i] = v[i];
  __syncwarp();
}
// n <= B N candidates, by the CTA.
template <int N, int B>
__device__ __forceinline__ void block_sort(Shared<B>& s, int n) {
  const int t = threadIdx.x;
  uint64_t v[N];
  uint64_t* mine = s.cand + t * N;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = t * N + i < n ? mine[i] : 0;
  sort_lanes(v, t);
  for (int threads = 64; threads <= B; threads <<= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) mine[i] = v[i];
    for (int stride = threads * N / 2; stride >= 32 * N; stride >>= 1) {
      __syncthreads();
      for (int i = t; i < B * N / 2; i += B) {
        const int lo = 2 * i - (i & (stride - 1));
        order(s.cand[lo], s.cand[lo + stride], (lo & threads * N) == 0);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = mine[i];
    merge_lanes(v, t, 32, (t & threads) == 0);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) mine[i] = v[i];
  __syncthreads();
}
// The CTA's n candidates, in order.
template <int B>
__device__ __noinline__ void sort_desc(Shared<B>& s, int n) {
  static_assert(kCap <= 8 * B, "keys a thread");
  if (n <= B) {
    block_sort<1>(s, n);
  } else if (n <= 2 * B) {
    block_sort<2>(s, n);
  } else if (kCap <= 4 * B || n <= 4 * B) {
    block_sort<4>(s, n);
  } else {
    block_sort<kCap / B>(s, n);
  }
}

// The k largest keys of elements [lo, hi), at least k of which reach s.least,
// whatever they are: for slices whose candidates overflow.  Where fewer than k
// exceed the least of those (long ties, as in a masked row), one pass finds it
// and one more the elements above it, and the first ones equal to it follow in
// index order; else (rows that rise steeply) a histogram of the values' keys 8
// bits at a time finds the k-th largest value first, in two to four passes.
// 4096 x 128256 bf16, top 64, masked but for 20: 916 us (4.8 ms with the
// histograms for these too); 64 rows 30 us (145).
template <typename T, int B>
__device__ __noinline__ void select_any(Shared<B>& s, const T* xr, int lo, int hi, int k) {
  // the upper bits that tell two values' keys apart: 16 of a bf16 value's, 19
  // of an f16 value's (5 + 10 bits and the sign, with fp32's 8 bits of exponent)
  constexpr int kBits = std::is_same<T, float>::value ? 32 : std::is_same<T, __half>::value ? 24 : 16;
  constexpr int VW = Elem<T>::kVec, kWarps = B / 32, U = 2;  // (with 4 the callers' registers spill)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const RowSplit sp = split_row(xr + lo, hi - lo);
  const uint4* body = reinterpret_cast<const uint4*>(xr + lo + sp.head);
  const int single = single_of(sp, tid, VW);
  const uint32_t alone = single >= 0 ? value_key(Elem<T>::to_f(xr[lo + single])) >> (32 - kBits) : 0;
  const auto each = [&](auto see) {  // (keys and elements, in no order)
    if (single >= 0) see(alone, single);
    for (int p = tid; p < sp.nvec; p += U * B) {
      uint4 u[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (p + i * B < sp.nvec) u[i] = ld_cached(body + p + i * B);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (p + i * B >= sp.nvec) break;
        float f[VW];
        unpack<T>(u[i], f);
#pragma unroll
        for (int j = 0; j < VW; ++j)
          see(value_key(f[j]) >> (32 - kBits), sp.head + (p + i * B) * VW + j);
      }
    }
  };
  uint32_t value = 0xffffffffu;
  int above = 0, need = k;
  {
    const uint32_t least = s.least >> (32 - kBits);
    int equal = 0, reach = 0;
    each([&](uint32_t key, int) {
      if (key < least) return;
      ++reach;
      if (key < value) equal = 0;
      value = min(value, key);
      equal += key == value;
    });
    const uint32_t mine = value;
    value = __reduce_min_sync(0xffffffffu, value);
    equal = __reduce_add_sync(0xffffffffu, mine == value ? equal : 0);
    reach = __reduce_add_sync(0xffffffffu, reach);
    if (lane == 0) {
      s.sums[0][warp] = make_int2((int)value, equal);
      s.sums[1][warp].x = reach;
    }
    if (tid == 0) s.filled = 0;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) value = min(value, (uint32_t)s.sums[0][w].x);
    for (int w = 0; w < kWarps; ++w)
      above += s.sums[1][w].x - ((uint32_t)s.sums[0][w].x == value ? s.sums[0][w].y : 0);
    __syncthreads();
  }
  if (above < k) {
    need = k - above;
  } else {
    const int rounds = (hi - lo + B - 1) / B;
    value = 0;
    for (int shift = kBits - 8; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += B) s.hist[i] = 0;
      __syncthreads();
      for (int r = 0; r < rounds; ++r) {
        const int i = lo + r * B + tid;
        const uint32_t key = i < hi ? value_key(Elem<T>::to_f(xr[i])) >> (32 - kBits) : 0;
        const bool in = i < hi && (uint64_t)key >> (shift + 8) == (uint64_t)value >> (shift + 8);
        const uint32_t digit = in ? (key >> shift) & 255 : 256;
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        if (in && __ffs(same) - 1 == lane) atomicAdd(&s.hist[digit], __popc(same));
      }
      __syncthreads();
      if (tid == 0) {
        int sum = 0, d = 255;
        while (d > 0 && sum + s.hist[d] < need) sum += s.hist[d--];
        s.pick = d;
        s.above = sum;
      }
      __syncthreads();
      value |= (uint32_t)s.pick << shift;
      need -= s.above;
    }
  }
  if (need < k) {
    each([&](uint32_t key, int at) {
      if (key > value) append(s, element_key(Elem<T>::to_f(xr[lo + at]), (uint32_t)(lo + at)));
    });
  }
  // the first ones equal to it, in the order of threads: elements at + j
  int parity = 0, taken = 0;
  const auto first_ones = [&](uint32_t mine, int at) {
    const int count = __popc(mine);
    int before = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    if (lane == 31) s.sums[parity][warp].x = before;
    __syncthreads();
    before += taken - count;
    int all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s.sums[parity][w].x;
      all += s.sums[parity][w].x;
    }
    parity ^= 1;
    for (; mine != 0 && before < need; mine &= mine - 1, ++before) {
      const int e = lo + at + __ffs(mine) - 1;
      append(s, element_key(Elem<T>::to_f(xr[e]), (uint32_t)e));
    }
    taken += all;
  };
  first_ones(tid < 8 && single >= 0 && alone == value, single);
  for (int base = 0; base < sp.nvec && taken < need; base += B) {
    uint32_t mine = 0;
    if (base + tid < sp.nvec) {
      float f[VW];
      unpack<T>(ld_cached(body + base + tid), f);
#pragma unroll
      for (int j = 0; j < VW; ++j) mine |= (uint32_t)(value_key(f[j]) >> (32 - kBits) == value) << j;
    }
    first_ones(mine, sp.head + (base + tid) * VW);
  }
  if (taken < need) first_ones(tid >= 8 && single >= 0 && alone == value, single);
  __syncthreads();
}

// The k-th largest of the threads' maxima (or one that a few more reach), by
// the lanes of one warp; 0 when there are fewer.
template <int B>
__device__ __forceinline__ uint32_t kth_maximum(const Shared<B>& s, int k) {
  constexpr int kEach = B / 32;
  const int lane = threadIdx.x & 31;
  uint32_t v[kEach], lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    v[i] = s.run[i * 32 + lane];
    lo = min(lo, v[i]);
    hi = max(hi, v[i]);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  // two bits a step, below those that lo and hi share: the counts of the three
  // larger keys in ten bits each (at most B of them)
  static_assert(B < 1024, "the counts' fields");
  const int top = (32 - __clz(lo ^ hi) + 1) & ~1;
  uint32_t at = top < 32 ? lo >> top << top : 0;
  for (int bit = top - 2; bit >= 0; bit -= 2) {
    const uint32_t one = 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      n += (v[i] >= at + one) + ((v[i] >= at + 2 * one) << 10) + ((v[i] >= at + 3 * one) << 20);
    n = __reduce_add_sync(0xffffffffu, n);
    const int n3 = n >> 20, n2 = (n >> 10) & 1023, n1 = n & 1023;
    const int reached = n3 >= k ? n3 : n2 >= k ? n2 : n1 >= k ? n1 : 0;
    at += n3 >= k ? 3 * one : n2 >= k ? 2 * one : n1 >= k ? one : 0;
    if (reached != 0 && reached <= k + k / 8) break;
  }
  return at;  // (0 among the keys: lo = 0, and `at` stays 0 unless k reach more)
}

// The 16-byte packs of one slice.
struct Packs {
  const uint4* body;
  int nvec;
};
// Copies half `h` of the thread's packs of chunk `base` into its stage slots.
template <int B>
__device__ __forceinline__ void issue(Shared<B>& s, const Packs& src, int base, int h) {
  const uint4* from = src.body + base + threadIdx.x;
  const int left = src.nvec - base - (int)threadIdx.x;
#pragma unroll
  for (int i = h * kPacks / 2; i < (h + 1) * kPacks / 2; ++i)
    if (i * B < left) cp_async16(&s.stage[i][threadIdx.x], from + i * B);
  cp_async_commit();
}

// Candidates of elements [lo, hi) of a row, which hold its k largest keys
// (k <= hi - lo); returns their number, in every thread, more than kCap when
// they did not fit.  The slice's first chunk has been issued; the first chunk
// of `next` is when this returns.
//
// The slice streams through once, each thread keeping one maximum for each of
// its pack slots: groups of every kChunk-th pack.  k groups reach the k-th
// largest of these maxima, so an element below it is not among the k largest,
// and in a row without order little over k elements reach it.  Only the packs
// of the groups that do, about k of kChunk, are read again (from L2) for their
// elements.  Elements equal to the threshold are kept, so ties are settled by
// index at the end.  For k <= 5 B / 8 the k-th largest of the threads' maxima
// serves, which one warp finds: a little lower, and without a barrier a step.
template <typename T, int B>
__device__ __forceinline__ int collect(Shared<B>& s, const T* xr, int lo, int hi, int k,
                                       const Packs& next, int& parity) {
  constexpr int kChunk = Shared<B>::kChunk;
  constexpr int VW = Elem<T>::kVec;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const RowSplit sp = split_row(xr + lo, hi - lo);
  const Packs src = {reinterpret_cast<const uint4*>(xr + lo + sp.head), sp.nvec};
  if (tid == 0) s.filled = s.listed = 0;
  // the slice's single elements, used after the stream
  const int single = single_of(sp, tid, VW);
  const float alone = single >= 0 ? Elem<T>::to_f(xr[lo + single]) : 0.f;
  uint32_t group[kPacks];
#pragma unroll
  for (int i = 0; i < kPacks; ++i) group[i] = word_lowest<T>();
  for (int base = 0; base < max(sp.nvec, 1); base += kChunk) {
    const int left = sp.nvec - base - tid;  // the thread's packs end here
    const bool more = base + kChunk < sp.nvec;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      cp_async_wait_pending<1>();
#pragma unroll
      for (int i = h * kPacks / 2; i < (h + 1) * kPacks / 2; ++i) {
        const uint4 u = s.stage[i][tid];
        if (i * B < left) group[i] = word_max<T>(group[i], pack_max<T>(u));
      }
      if (more) {
        issue(s, src, base + kChunk, h);
      } else {
        issue(s, next, 0, h);
      }
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    group[i] = i * B + tid < sp.nvec ? value_key(word_top<T>(group[i])) : 0;
    most = max(most, group[i]);
  }
  uint32_t least;
  if (k <= 5 * B / 8) {
    s.run[tid] = most;
    __syncthreads();
    if (warp == 0) {
      const uint32_t v = kth_maximum(s, k);
      if (lane == 0) s.least = v;
    }
    __syncthreads();
    least = s.least;
  } else {
    __syncthreads();
    least = bisect(s, k, k + k / 8, parity, [&](auto see) {
#pragma unroll
      for (int i = 0; i < kPacks; ++i) see(group[i]);
    });
    if (tid == 0) s.least = least;
  }
  if (single >= 0) append(s, element_key(alone, (uint32_t)(lo + single)));
#pragma unroll
  for (int i = 0; i < kPacks; ++i)
    if (group[i] >= max(least, 1u)) s.list[take_slot(&s.listed)] = (uint16_t)(i * B + tid);
  __syncthreads();
  const int depth = (sp.nvec + kChunk - 1) / kChunk;  // packs of a group
  const int items = s.listed * depth;
  const float bar = key_value(least);  // (NaN while everything passes, or only NaN does)
  const auto look = [&](const uint4& u, int p) {
    if (word_top<T>(pack_max<T>(u)) < bar) return;
    float f[VW];
    unpack<T>(u, f);
#pragma unroll
    for (int i = 0; i < VW; ++i)
      if (value_key(f[i]) >= least) append(s, element_key(f[i], (uint32_t)(lo + sp.head + p * VW + i)));
  };
  // (a tie of all the row is not counted to the end, one atomic an element)
  const auto more_fit = [&] { return *(volatile int*)&s.filled <= kCap; };
  if (depth == 1 && next.nvec == 0) {
    // the stage still holds them
    for (int j = tid; j < items && more_fit(); j += B) {
      const int p = s.list[j];
      look(s.stage[p / B][p % B], p);
    }
  } else {
    // two packs a thread in flight; n / depth by a multiplication where that is
    // exact (n < 4096 depth, off by less than n depth / 2^32 of a step)
    const uint32_t over = depth < 1024 ? (uint32_t)((0x100000000ull + depth - 1) / depth) : 0;
    for (int j = tid; j < items && more_fit(); j += 2 * B) {
      int p[2];
      uint4 u[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t n = min(j + i * B, items - 1);
        const uint32_t entry = depth == 1 ? n : depth < 1024 ? __umulhi(n, over) : n / depth;
        p[i] = s.list[entry] + (int)(n - entry * depth) * kChunk;
        if (j + i * B >= items || p[i] >= sp.nvec) p[i] = -1;
        u[i] = ld_cached(src.body + max(p[i], 0));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (p[i] >= 0) look(u[i], p[i]);
    }
  }
  __syncthreads();
  return s.filled;
}

// One CTA a row, walking rows, or a cluster with a slice of the row in each
// CTA when there are few: every CTA finds its slice's k largest, CTA 0 takes
// them all and orders the k largest of the row.  Bound by HBM for many rows:
// 4096 x 128256 bf16, top 64, in 178 us (5.9 TB/s, 91% of the measured copy
// rate).  Few rows are bound by the steps after the stream (threshold, second
// look, order: 3 to 5 us): 333 x 40003 fp32, top 50, 17.5 us; 4 x 32000 bf16,
// top 8, 6.0 us.
template <typename T, int B>
__global__ void __launch_bounds__(B, 1024 / B)
topk_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int cols, int k, T* __restrict__ values,
            int64_t* __restrict__ indices) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared<B>& s = *reinterpret_cast<Shared<B>*>(smem);
  pdl_prologue();
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int tid = threadIdx.x;
  int parity = 0;
  // slices of whole groups of 64 elements
  const int per = (int)(ceil_div(ceil_div(cols, C), 64) * 64);
  const int lo = min(cols, rank * per), hi = min(cols, lo + per);
  const int want = min(k, hi - lo);
  const auto packs_of = [&](int64_t row) {
    if (row >= rows) return Packs{nullptr, 0};
    const T* at = x + row * ld + lo;
    const RowSplit sp = split_row(at, hi - lo);
    return Packs{reinterpret_cast<const uint4*>(at + sp.head), sp.nvec};
  };
  const int64_t step = cluster_count();
  issue(s, packs_of(cluster_id()), 0, 0);
  issue(s, packs_of(cluster_id()), 0, 1);
  for (int64_t row = cluster_id(); row < rows; row += step) {
    const T* xr = x + row * ld;
    int n = collect(s, xr, lo, hi, want, packs_of(row + step), parity);
    if (n > kCap) {
      select_any(s, xr, lo, hi, want);
      n = want;
    }
    // few keys: each one's place is the number of keys above it
    const auto place_all = [&](auto put) {
      int shift = 5;  // 2^shift threads a key
      while ((n << shift) > B) --shift;
      const int i = tid >> shift, step = 1 << shift;
      const uint64_t key = i < n ? s.cand[i] : 0;
      int place = 0;
      if (i < n) {
        int j = tid & (step - 1);
        for (; j + 3 * step < n; j += 4 * step)
          place += (s.cand[j] > key) + (s.cand[j + step] > key) + (s.cand[j + 2 * step] > key) +
                   (s.cand[j + 3 * step] > key);
        for (; j < n; j += step) place += s.cand[j] > key;
      }
      __syncwarp();
      for (int o = step >> 1; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
      if (i < n && (tid & (step - 1)) == 0 && place < k) put(place, key);
    };
    if (C > 1) {
      // this slice's k largest, 0 past the last
      if (n <= kRank) {
        for (int i = tid; i < k; i += B) s.top[i] = 0;
        __syncthreads();
        place_all([&](int place, uint64_t key) { s.top[place] = key; });
      } else {
        sort_desc(s, n);
        for (int i = tid; i < k; i += B) s.top[i] = i < n ? s.cand[i] : 0;
      }
      cluster_sync_all();
      if (rank == 0) {
        for (int i = tid; i < C * k; i += B)
          s.cand[i] = (uint64_t)ld_remote_s64(remote_smem(&s.top[i % k], i / k));
        n = C * k;
        __syncthreads();
      }
      cluster_sync_all();  // the others' lists are read
    }
    if (rank == 0) {
      const auto put = [&](int place, uint64_t key) {
        const uint32_t at = ~(uint32_t)key;
        const uint32_t v = (uint32_t)(key >> 32);
        indices[row * k + place] = at;
        // the key tells the value's bits but for a zero's sign and a NaN's payload
        values[row * k + place] =
            v == 0x80000000u || v == 0xffffffffu ? xr[at] : Elem<T>::from_f(key_value(v));
      };
      if (n <= kRank) {
        place_all(put);
      } else {
        sort_desc(s, n);
        for (int i = tid; i < k; i += B) put(i, s.cand[i]);
      }
    }
    __syncthreads();  // the next row's candidates take these ones' place
  }
  cp_async_wait_all();
}

constexpr int kBlock = 512;

// The same with a warp a row, for many short rows: the CTA's barriers, one
// after the other, took most of a short row's time (20000 x 1024 bf16, top 8,
// 411 us against 39; 8192 x 4096, top 64, 192 against 55).  The warp's 256
// slots are the groups; threshold, second look and order run on shuffles and a
// list in shared memory.  Bound by the instructions of these steps: a third
// of the copy rate at 1500 x 12000 bf16, top 20 (17 us), a fifth at 8192 x
// 4096, top 64.
constexpr int kRowWarps = 4;
constexpr int kRowCap = 512;     // candidates listed
constexpr int kRowSorted = 256;  // candidates put in order
constexpr int kRowTop = 128;     // the largest k: half the slots, which some 180 elements reach

struct RowShared {
  uint64_t cand[kRowWarps][kRowCap];
  uint8_t list[kRowWarps][256];  // slots that hold candidates
  int filled[kRowWarps];
};

// The k-th largest of the lanes' maxima, k <= 32.
template <int S>
__device__ __forceinline__ uint32_t kth_lane(const uint32_t (&v)[S], int k, int lane) {
  uint32_t m[1] = {v[0]};
#pragma unroll
  for (int i = 1; i < S; ++i) m[0] = max(m[0], v[i]);
  sort_lanes(m, lane);
  return __shfl_sync(0xffffffffu, m[0], k - 1);
}

// The lowest bits that tell two values' keys apart are from this one up: 16 of
// a bf16 value's, 19 of an f16 value's (two more so that they come in pairs).
template <typename T>
__device__ __forceinline__ constexpr int key_bits_from() {
  return std::is_same<T, float>::value ? 0 : std::is_same<T, __half>::value ? 12 : 16;
}

// The k-th largest of the slots' (or one that a few more reach), as in kth_maximum.
template <typename T, int S>
__device__ __forceinline__ uint32_t search_slots(const uint32_t (&v)[S], int k) {
  constexpr int kLast = key_bits_from<T>();
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    lo = min(lo, v[i] - 1);  // (slots without a pack aside)
    hi = max(hi, v[i]);
  }
  lo = __reduce_min_sync(0xffffffffu, lo) + 1;
  hi = __reduce_max_sync(0xffffffffu, hi);
  const int top = (32 - __clz(lo ^ hi) + 1) & ~1;
  uint32_t least = top < 32 ? lo >> top << top : 0;
  for (int bit = top - 2; bit >= kLast; bit -= 2) {
    const uint32_t one = 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < S; ++i)
      n += (v[i] >= least + one) + ((v[i] >= least + 2 * one) << 10) + ((v[i] >= least + 3 * one) << 20);
    n = __reduce_add_sync(0xffffffffu, n);
    const int n3 = n >> 20, n2 = (n >> 10) & 1023, n1 = n & 1023;
    const int reached = n3 >= k ? n3 : n2 >= k ? n2 : n1 >= k ? n1 : 0;
    least += n3 >= k ? 3 * one : n2 >= k ? 2 * one : n1 >= k ? one : 0;
    if (reached != 0 && reached <= k + k / 8) break;
  }
  return least;
}

// For a row whose candidates did not fit (ties at the threshold `least`, as in
// a masked row, or a row that rises): the elements above a value and the first
// ones equal to it in index order, at least the k largest and at most
// kRowSorted, into cand; their number.  By a warp, in two walks over the row
// where fewer than k elements exceed the least of those that reach `least`, as
// for a mask's; else in one more for two bits of the values' keys.  8192 x 4096
// bf16, top 64, masked but for 20: 128 us (1068 by two bits of a 64-bit key).
template <typename T>
__device__ __forceinline__ int row_select(const T* xr, int cols, int k, uint32_t least, uint64_t* cand,
                                       int* filled) {
  constexpr int VW = Elem<T>::kVec, kFrom = key_bits_from<T>();
  const int lane = threadIdx.x & 31;
  const RowSplit sp = split_row(xr, cols);
  const uint4* body = reinterpret_cast<const uint4*>(xr + sp.head);
  const int single = single_of(sp, lane, VW);
  const uint32_t alone = single >= 0 ? value_key(Elem<T>::to_f(xr[single])) >> kFrom : 0;
  const auto each = [&](auto see) {  // (keys, in no order)
    if (single >= 0) see(alone);
    for (int p = lane; p < sp.nvec; p += 64) {
      uint4 u[2];
      float f[VW];
      u[0] = ld_cached(body + p);
      if (p + 32 < sp.nvec) u[1] = ld_cached(body + p + 32);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (p + 32 * i >= sp.nvec) break;
        unpack<T>(u[i], f);
#pragma unroll
        for (int j = 0; j < VW; ++j) see(value_key(f[j]) >> kFrom);
      }
    }
  };
  // the least key that reaches `least`, how many are it, how many exceed it
  least >>= kFrom;
  uint32_t lowest = 0xffffffffu;
  int equal = 0, reach = 0;
  each([&](uint32_t key) {
    if (key < least) return;
    ++reach;
    if (key < lowest) equal = 0;
    lowest = min(lowest, key);
    equal += key == lowest;
  });
  uint32_t cut = __reduce_min_sync(0xffffffffu, lowest);
  equal = __reduce_add_sync(0xffffffffu, lowest == cut ? equal : 0);
  int above = __reduce_add_sync(0xffffffffu, reach) - equal;
  uint32_t under = cut;  // the keys above this one are all taken
  if (above >= k) {
    cut = 0;
    above = 0;
    bool exact = true;
    for (int bit = 30 - kFrom; bit >= 0; bit -= 2) {
      const uint32_t one = 1u << bit;
      int n1 = 0, n2 = 0, n3 = 0;
      each([&](uint32_t key) {
        n1 += key >= cut + one;
        n2 += key >= cut + 2 * one;
        n3 += key >= cut + 3 * one;
      });
      n1 = __reduce_add_sync(0xffffffffu, n1);
      n2 = __reduce_add_sync(0xffffffffu, n2);
      n3 = __reduce_add_sync(0xffffffffu, n3);
      // (the fewest that are too few: those above the key in the end)
      above = n1 < k ? n1 : n2 < k ? n2 : n3 < k ? n3 : above;
      const int reached = n3 >= k ? n3 : n2 >= k ? n2 : n1 >= k ? n1 : 0;
      cut += n3 >= k ? 3 * one : n2 >= k ? 2 * one : n1 >= k ? one : 0;
      if (reached != 0 && reached <= kRowSorted) {
        above = reached;
        exact = false;
        break;
      }
    }
    under = exact ? cut : cut - 1;
  }
  const int need = max(0, k - above);
  if (lane == 0) *filled = 0;
  __syncwarp();
  int taken = 0;  // of the ones equal to cut; they follow those above it
  const auto first_ones = [&](uint32_t mine, int at) {  // this lane's, elements at + j, in lane order
    const int count = __popc(mine);
    int before = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    const int all = __shfl_sync(0xffffffffu, before, 31);
    before += taken - count;
    for (; mine != 0 && before < need; mine &= mine - 1, ++before) {
      const int e = at + __ffs(mine) - 1;
      cand[above + before] = element_key(Elem<T>::to_f(xr[e]), (uint32_t)e);
    }
    taken += all;
  };
  if (single >= 0 && alone > under) cand[take_slot(filled)] = element_key(Elem<T>::to_f(xr[single]), (uint32_t)single);
  first_ones(lane < 8 && single >= 0 && alone == cut, single);
  for (int base = 0; base < sp.nvec; base += 32) {
    __syncwarp();
    if (taken >= need && *(volatile int*)filled == above) break;
    __syncwarp();
    const int p = base + lane;
    uint32_t mine = 0;
    if (p < sp.nvec) {
      float f[VW];
      unpack<T>(ld_cached(body + p), f);
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        const uint32_t key = value_key(f[j]) >> kFrom;
        mine |= (uint32_t)(key == cut) << j;
        if (key > under) cand[take_slot(filled)] = element_key(f[j], (uint32_t)(sp.head + p * VW + j));
      }
    }
    if (taken < need) first_ones(mine, sp.head + p * VW);
  }
  if (taken < need) first_ones(lane >= 8 && single >= 0 && alone == cut, single);
  __syncwarp();
  return above + need;
}

// The warp's rows that row_select is for: their first index is -1 - least.
// (Apart from the others' loop, whose registers it would take.)
template <typename T>
__device__ __noinline__ void finish_late(const T* x, int64_t ld, int64_t rows, int cols, int k, T* values,
                                         int64_t* indices, uint64_t* cand, int* filled) {
  const int lane = threadIdx.x & 31;
  const int64_t first = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  for (int64_t row = first; row < rows; row += (int64_t)gridDim.x * kRowWarps) {
    int64_t* ids = indices + row * k;
    const int64_t mark = *(volatile int64_t*)ids;
    __syncwarp();
    if (mark >= 0) continue;
    const T* xr = x + row * ld;
    const int n = row_select<T>(xr, cols, k, (uint32_t)(-1 - mark), cand, filled);
    warp_sort<kRowSorted / 32>(cand, n, lane);
    for (int i = lane; i < k; i += 32) {
      const uint32_t at = ~(uint32_t)cand[i];
      ids[i] = at;
      values[row * k + i] = xr[at];
    }
    __syncwarp();
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32, 32 / kRowWarps)
topk_rows_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int cols, int k,
                 T* __restrict__ values, int64_t* __restrict__ indices) {
  constexpr int VW = Elem<T>::kVec;
  constexpr int S = 8, kChunk = 32 * S;
  __shared__ RowShared s;
  pdl_prologue();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t* cand = s.cand[warp];
  uint8_t* list = s.list[warp];
  int* filled = &s.filled[warp];
  const auto keep = [&](uint64_t key) {
    const int slot = take_slot(filled);
    if (slot < kRowCap) cand[slot] = key;
  };
  const int64_t step = (int64_t)gridDim.x * kRowWarps;
  bool late = false;
  for (int64_t row = (int64_t)blockIdx.x * kRowWarps + warp; row < rows; row += step) {
    const T* xr = x + row * ld;
    const RowSplit sp = split_row(xr, cols);
    const uint4* body = reinterpret_cast<const uint4*>(xr + sp.head);
    const int single = single_of(sp, lane, VW);
    const float alone = single >= 0 ? Elem<T>::to_f(xr[single]) : 0.f;
    if (lane == 0) *filled = 0;
    uint32_t v[S];
#pragma unroll
    for (int i = 0; i < S; ++i) v[i] = word_lowest<T>();
    for (int base = lane; base < sp.nvec; base += kChunk) {
      uint4 u[S];
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (base + 32 * i < sp.nvec) u[i] = ld_cached(body + base + 32 * i);
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (base + 32 * i < sp.nvec) v[i] = word_max<T>(v[i], pack_max<T>(u[i]));
    }
#pragma unroll
    for (int i = 0; i < S; ++i) v[i] = lane + 32 * i < sp.nvec ? value_key(word_top<T>(v[i])) : 0;
    // up to k = 16 the lanes' maxima, which 1.4 k elements reach, in a sixth of
    // the search's steps (20000 x 1024 bf16, top 8: 37 us, 45); past that the
    // search, for its fewer candidates (1500 x 12000, top 20: 16.5 us, 17.7 with
    // two maxima a lane)
    const uint32_t least = k <= 16 ? kth_lane(v, k, lane) : search_slots<T>(v, k);
    // the slots that reach it, and their packs' elements
    uint32_t listed = 0;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const bool in = v[i] >= max(least, 1u);
      const uint32_t vote = __ballot_sync(0xffffffffu, in);
      if (in) list[listed + __popc(vote & ((1u << lane) - 1))] = (uint8_t)(lane + 32 * i);
      listed += __popc(vote);
    }
    __syncwarp();
    if (single >= 0) keep(element_key(alone, (uint32_t)single));
    const float bar = key_value(least);  // (NaN while everything passes, or only NaN does)
    const uint32_t depth = (sp.nvec + kChunk - 1) / kChunk, items = listed * depth;
    for (uint32_t base = lane; base < items && *(volatile int*)filled <= kRowCap; base += 64) {
      uint4 u[2];
      int p[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t item = base + 32 * i, chunk = item / listed;
        p[i] = item < items ? list[item - chunk * listed] + (int)(chunk * kChunk) : sp.nvec;
        if (p[i] < sp.nvec) u[i] = ld_cached(body + p[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (p[i] >= sp.nvec) continue;
        float f[VW];
        unpack<T>(u[i], f);
        uint32_t reach = 0;
#pragma unroll
        for (int j = 0; j < VW; ++j) reach |= (uint32_t)!(f[j] < bar) << j;
        if (reach == 0) continue;
        const int first = take_slots(filled, __popc(reach));
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          const int slot = first + __popc(reach & ((1u << j) - 1));
          if ((reach >> j & 1) && slot < kRowCap)
            cand[slot] = element_key(f[j], (uint32_t)(sp.head + p[i] * VW + j));
        }
      }
    }
    __syncwarp();
    int n = *filled;
    if (n > kRowCap) {
      if (lane == 0) indices[row * k] = -1 - (int64_t)least;
      late = true;
      __syncwarp();
      continue;
    }
    if (n > kRowSorted) {
      // a key that k to kRowSorted of the listed ones reach, two bits a walk
      uint64_t at = 0;
      for (int bit = 62; bit >= 0; bit -= 2) {
        const uint64_t one = (uint64_t)1 << bit;
        int n1 = 0, n2 = 0, n3 = 0;
        for (int i = lane; i < n; i += 32) {
          n1 += cand[i] >= at + one;
          n2 += cand[i] >= at + 2 * one;
          n3 += cand[i] >= at + 3 * one;
        }
        n1 = __reduce_add_sync(0xffffffffu, n1);
        n2 = __reduce_add_sync(0xffffffffu, n2);
        n3 = __reduce_add_sync(0xffffffffu, n3);
        const int reached = n3 >= k ? n3 : n2 >= k ? n2 : n1 >= k ? n1 : 0;
        at += n3 >= k ? 3 * one : n2 >= k ? 2 * one : n1 >= k ? one : 0;
        if (reached != 0 && reached <= kRowSorted) break;
      }
      int kept = 0;
      for (int i = 0; i < n; i += 32) {
        const uint64_t key = i + lane < n ? cand[i + lane] : 0;
        const uint32_t vote = __ballot_sync(0xffffffffu, key >= at && key != 0);
        __syncwarp();
        if (vote >> lane & 1) cand[kept + __popc(vote & ((1u << lane) - 1))] = key;
        kept += __popc(vote);
        __syncwarp();
      }
      n = kept;
    }
    if (n <= 32) {
      warp_sort<1>(cand, n, lane);
    } else if (n <= 64) {
      warp_sort<2>(cand, n, lane);
    } else if (n <= 128) {
      warp_sort<4>(cand, n, lane);
    } else {
      warp_sort<8>(cand, n, lane);
    }
    for (int i = lane; i < k; i += 32) {
      const uint64_t key = cand[i];
      const uint32_t at = ~(uint32_t)key, w = (uint32_t)(key >> 32);
      indices[row * k + i] = at;
      values[row * k + i] = w == 0x80000000u || w == 0xffffffffu ? xr[at] : Elem<T>::from_f(key_value(w));
    }
    __syncwarp();  // the next row's candidates take these ones' place
  }
  if (late) finish_late(x, ld, rows, cols, k, values, indices, cand, filled);
}

// Gradient: zeros, and dvalues at the indices (distinct in a row).
template <typename T>
__global__ void __launch_bounds__(kBlock)
topk_bwd_kernel(const T* __restrict__ dv, const int64_t* __restrict__ indices, int cols, int k,
                T* __restrict__ dx) {
  pdl_prologue();
  const int64_t row = blockIdx.x;
  T* dr = dx + row * (int64_t)cols;
  const RowSplit sp = split_row(dr, cols);
  uint4* body = reinterpret_cast<uint4*>(dr + sp.head);
  const int e = single_of(sp, threadIdx.x, Elem<T>::kVec);
  if (e >= 0) dr[e] = Elem<T>::from_f(0.f);
  for (int p = threadIdx.x; p < sp.nvec; p += kBlock) st_stream(body + p, make_uint4(0, 0, 0, 0));
  __syncthreads();
  for (int i = threadIdx.x; i < k; i += kBlock) {
    const int64_t at = indices[row * k + i];
    if (at >= 0 && at < cols) dr[at] = dv[row * k + i];
  }
}

}  // namespace
}  // namespace flb200

extern "C" {

FL_B200_API int fl_b200_topk_lastdim(const void* x, int64_t ld, int64_t rows, int64_t cols,
                                     int64_t k, void* values, int64_t* indices, int dtype,
                                     fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(rows >= 0 && k >= 0 && k <= cols);
  if (!is_float_dtype(dtype)) return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (k > kMaxTop || rows > 0x7fffffffLL || cols > kMaxCols) return FL_B200_ERR_TOO_LARGE;
  if (rows == 0 || k == 0) return FL_B200_OK;
  FLB_CHECK_ARG(x && values && indices && (rows == 1 || ld >= cols));
  DeviceInfo dev;
  const int st = current_device_info(&dev);
  if (st != FL_B200_OK) return st;
  return dispatch_float(dtype, [&](auto t) {
    using T = decltype(t);
    // More rows of at most 32 KB than CTAs of 256 threads fit: a warp a row, if
    // k is at most half the row's packs (1000 x 8000 bf16, top 64: 17.9 us, 28.5
    // with a CTA a row).  Above 16 KB a warp's chain of steps is long: with a
    // large k it takes more rows to hide (600 x 16000, top 64: 27.0 us, 19.0
    // with a CTA a row; 1300 rows, top 128: 51.3 and 54.3).
    const int64_t bytes = cols * (int64_t)sizeof(T);
    if (rows > (bytes <= 16384 || k <= 32 ? 4 : 8) * dev.sm_count && bytes <= 32768 && k <= kRowTop &&
        cols / Elem<T>::kVec >= 2 * k) {
      const int64_t ctas = std::min<int64_t>(ceil_div(rows, kRowWarps), 32 / kRowWarps * dev.sm_count);
      launch_k(topk_rows_kernel<T>, dim3((unsigned)ctas), dim3(kRowWarps * 32), 0, (cudaStream_t)stream,
               reinterpret_cast<const T*>(x), ld, rows, (int)cols, (int)k, reinterpret_cast<T*>(values),
               indices);
      return launch_status();
    }
    const auto go = [&](auto block) {
      constexpr int B = decltype(block)::value;
      // few rows: up to 8 CTAs a row, with two packs a thread at least, whose
      // lists fit CTA 0
      int cluster = 1;
      while (cluster < 8 && rows * cluster < dev.sm_count && cluster * 2 * k <= kCap && k <= kShared &&
             cols / (cluster * 2) >= 2 * B * Elem<T>::kVec)
        cluster *= 2;
      const auto kern = topk_kernel<T, B>;
      static std::atomic<int> allowed[64];
      if (!allow_smem(kern, sizeof(Shared<B>), false, allowed)) return (int)FL_B200_ERR_LAUNCH;
      const int64_t ctas = std::min<int64_t>(rows, 1024 / B * dev.sm_count);
      return launch_cluster(kern, cluster > 1 ? rows * cluster : ctas, cluster, B, sizeof(Shared<B>),
                            (cudaStream_t)stream, reinterpret_cast<const T*>(x), ld, rows, (int)cols,
                            (int)k, reinterpret_cast<T*>(values), indices);
    };
    // 512 threads a row stream fastest (4096 rows of 128256 bf16: 184 us, 203 us
    // with 256); with no more rows than CTAs of 256 threads fit, those end
    // sooner (333 rows of 40003 float32: 18.6 us, 20.4 us with 512)
    return rows > 4 * dev.sm_count ? go(std::integral_constant<int, 512>{})
                                   : go(std::integral_constant<int, 256>{});
  });
}

FL_B200_API int fl_b200_topk_bwd(const void* dvalues, const int64_t* indices, void* dx, int64_t rows,
                                 int64_t cols, int64_t k, int dtype, fl_b200_stream_t stream) {
  using namespace flb200;
  FLB_CHECK_ARG(rows >= 0 && k >= 0 && k <= cols);
  if (!is_float_dtype(dtype)) return FL_B200_ERR_UNSUPPORTED_DTYPE;
  if (k > kMaxTop || rows > 0x7fffffffLL || cols > kMaxCols) return FL_B200_ERR_TOO_LARGE;
  if (rows == 0 || cols == 0) return FL_B200_OK;
  FLB_CHECK_ARG(dx && (k == 0 || (dvalues && indices)));
  return dispatch_float(dtype, [&](auto t) {
    using T = decltype(t);
    launch_k(topk_bwd_kernel<T>, dim3((unsigned)rows), dim3(kBlock), 0, (cudaStream_t)stream,
             reinterpret_cast<const T*>(dvalues), indices, (int)cols, (int)k,
             reinterpret_cast<T*>(dx));
    return launch_status();
  });
}

}  // extern "C"
