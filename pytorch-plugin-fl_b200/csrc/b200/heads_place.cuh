// Which operands of heads share memory: plain host arithmetic.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace flb200 {

// A [B, H, S, D] operand: counts and strides (bytes) of its heads' places.
struct Heads {
  int64_t n[3], st[3];
  int64_t bytes(int64_t head) const { return head + (n[0] - 1) * st[0] + (n[1] - 1) * st[1] + (n[2] - 1) * st[2]; }
};
// Whether two operands, `to` bytes from a's first head to b's, share memory.
// Views of one tensor lie inside each other's extent (q and k of a fused
// projection): what repeats at one stride in both is taken apart by the
// multiples of it at which a part of one can meet a part of the other.
// Layouts with nothing in common count as meeting where their extents do.
inline bool meet(int64_t to, Heads a, Heads b, int64_t head) {
  if (to >= a.bytes(head) || -to >= b.bytes(head)) return false;
  int top = -1;
  for (int d = 0; d < 3; ++d) {
    if (a.n[d] == 1) a.st[d] = b.st[d];
    if (b.n[d] == 1) b.st[d] = a.st[d];
    if (a.st[d] == b.st[d] && a.st[d] > 0 && (a.n[d] > 1 || b.n[d] > 1) && (top < 0 || a.st[d] > a.st[top])) top = d;
  }
  if (top < 0) return true;
  const int64_t period = a.st[top], back = a.n[top] - 1, on = b.n[top] - 1;
  a.n[top] = b.n[top] = 1;
  // parts m periods further apart meet where -b's bytes < to + m period < a's bytes
  const auto down = [&](int64_t v) { return v >= 0 ? v / period : -((-v + period - 1) / period); };
  const int64_t lo = std::max(-back, down(-b.bytes(head) - to) + 1), hi = std::min(on, down(a.bytes(head) - 1 - to));
  if (hi - lo > 16) return true;
  for (int64_t m = lo; m <= hi; ++m)
    if (meet(to + m * period, a, b, head)) return true;
  return false;
}
// Whether heads of one operand share memory: every stride has to pass what
// lies at the smaller ones.
inline bool meets_itself(Heads a, int64_t head) {
  int64_t need = head;
  for (int k = 0; k < 3; ++k) {
    int next = -1;
    for (int d = 0; d < 3; ++d)
      if (a.n[d] > 1 && (next < 0 || a.st[d] < a.st[next])) next = d;
    if (next < 0) return false;
    if (a.st[next] < need) return true;
    need += (a.n[next] - 1) * a.st[next];
    a.n[next] = 1;
  }
  return false;
}

}  // namespace flb200
