// The error text of libsffft_ops.so and the checks its entry points share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/sffft_ops.h"

namespace sffft {
namespace ops {

// Records the HIP error of the last failing call on this thread (defined in ops_api.hip).
int hip_status(hipError_t err, const char* what);

inline bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = (uintptr_t)a, z = (uintptr_t)b;
  return a && b && na && nb && x < z + nb && z < x + na;
}
inline bool aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }
inline bool valid_io(int io) { return io == SFFFT_IO_F32 || io == SFFFT_IO_BF16; }

// HIP takes no launch of 2^32 threads or more along a dimension.
inline bool launchable(long long workgroups, int threads) { return workgroups < ((1LL << 32) + threads - 1) / threads; }

// Bytes from the start of a strided [B][T][H][D] array to its end; 0 if an index may leave 62 bits or
// a stride is negative.
inline size_t extent(const long long s[3], int B, int T, int H, int D, int elem) {
  const int n[3] = {B, T, H};
  __int128 e = D;
  for (int i = 0; i < 3; i++) {
    if (s[i] < 0) return 0;
    e += (__int128)s[i] * (n[i] - 1);
  }
  e *= elem;
  return e >= ((__int128)1 << 62) ? 0 : (size_t)e;
}

// Whether no element of an output is written twice. Of two strided arrays [B][T][H or Hk][D] with elements of `elem`
// bytes: neither among their own elements nor between them; of one, with hb = 0. The dimensions are taken by ascending
// stride, each of which has to reach beyond what the smaller ones span; arrays that share their strides, such as parts
// of a fused projection, may lie between each other's rows, and then count as one from the stride on that exceeds their
// distance. (A few arrangements that would be in order are refused.)
inline bool distinct(const void* a, const long long sa[3], int ha, const void* b, const long long sb[3], int hb, int B, int T,
                     int D, int elem) {
  if (hb && a > b) return distinct(b, sb, hb, a, sa, ha, B, T, D, elem);
  const int na[3] = {B, T, ha}, nb[3] = {B, T, hb};
  const auto spans = [&](const long long s[3], const int n[3], __int128* span) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int i, int j) { return s[i] < s[j]; });
    *span = D;
    for (int i : order) {
      if (n[i] > 1 && s[i] < *span) return false;
      *span += (__int128)s[i] * (n[i] - 1);
    }
    return true;
  };
  __int128 span_a, span_b;
  if (!spans(sa, na, &span_a)) return false;
  if (!hb) return true;
  const uintptr_t bytes = (uintptr_t)b - (uintptr_t)a;
  const __int128 gap = bytes / elem;
  if (!spans(sb, nb, &span_b)) return false;
  if (gap >= span_a) return true;
  if (bytes % elem) return false;
  long long s[3];
  int order[3] = {0, 1, 2};
  for (int i = 0; i < 3; i++) {
    if (na[i] > 1 && nb[i] > 1 && sa[i] != sb[i]) return false;
    s[i] = na[i] > 1 ? sa[i] : sb[i];
  }
  std::sort(order, order + 3, [&](int i, int j) { return s[i] < s[j]; });
  bool one = false;
  span_a = span_b = D;
  for (int i : order) {
    const int n = std::max(na[i], nb[i]);
    if (n == 1) continue;
    if (!one && s[i] > gap) {
      if (span_a > gap) return false;
      span_a = gap + span_b, one = true;
    }
    if (one && s[i] < span_a) return false;
    span_a += (__int128)s[i] * ((one ? n : na[i]) - 1);
    span_b += (__int128)s[i] * (nb[i] - 1);
  }
  return one || span_a <= gap;
}

}  // namespace ops
}  // namespace sffft
