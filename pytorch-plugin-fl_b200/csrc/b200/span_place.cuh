// Where a row's packs and its span's words lie: plain arithmetic, which a host
// compiler takes too.
#pragma once

#ifdef __CUDACC__
#define FLB_HD __host__ __device__ __forceinline__
#else
#define FLB_HD inline
#endif

namespace flb200 {

// Element j of a row is virtual element shift + j, and virtual element 0 lies
// on the boundary of a pack of N at or before the row's first one.  The row's
// own (virtual) elements are [first, last), its span's [lo, hi), the span's
// packs p0 ... p0 + count - 1.
template <int N>
struct Packs {
  int first, last, lo, hi, p0, count;
  FLB_HD Packs(int row_lo, int row_hi, int shift, int cols)
      : first(shift), last(shift + cols), lo(shift + row_lo), hi(shift + row_hi), p0((int)((unsigned)lo / N)),
        count(row_hi > row_lo ? (int)((unsigned)(hi + N - 1) / N) - p0 : 0) {}
  FLB_HD bool inside(int at) const { return at >= lo && at + N <= hi; }
  // Whether the n elements at `at` hold one of the span.  A pack of the span
  // does, so in a 16-byte type it is read whole: the aligned 16 bytes lie in
  // the page of the row's byte they hold.  In a wider type a pack is several
  // 16-byte words, and one that holds nothing of the row may lie outside its
  // memory: those are not read.
  FLB_HD bool meets(int at, int n) const { return at < hi && at + n > lo; }
};

}  // namespace flb200
