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
// stride, each of which has to reach beyond what the smaller ones span. Arrays may lie between each other's rows, such
// as parts of a fused projection: the strides that they share and that exceed their distance step over both. (A few
// arrangements that would be in order are refused.)
inline bool distinct(const void* a, const long long sa[3], int ha, const void* b, const long long sb[3], int hb, int B, int T,
                     int D, int elem) {
  if (hb && a > b) return distinct(b, sb, hb, a, sa, ha, B, T, D, elem);
  // whether dimensions of n elements at strides s step over `span` elements and each other; span: of all
  const auto steps = [](const long long s[3], const int n[3], __int128* span) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int i, int j) { return s[i] < s[j]; });
    for (int i : order) {
      if (n[i] > 1 && s[i] < *span) return false;
      *span += (__int128)s[i] * (n[i] - 1);
    }
    return true;
  };
  const int na[3] = {B, T, ha}, nb[3] = {B, T, hb};
  __int128 span_a = D, span_b = D;
  if (!steps(sa, na, &span_a) || (hb && !steps(sb, nb, &span_b))) return false;
  const uintptr_t bytes = (uintptr_t)b - (uintptr_t)a, gap = bytes / elem;
  if (!hb || gap >= span_a) return true;
  if (bytes % elem) return false;
  // within a row of both: what is left without the shared dimensions
  int in_a[3], in_b[3], shared[3];
  long long s[3];
  for (int i = 0; i < 3; i++) {
    s[i] = na[i] > 1 ? sa[i] : sb[i];
    const bool both = (na[i] == 1 || nb[i] == 1 || sa[i] == sb[i]) && s[i] > (__int128)gap;
    in_a[i] = both ? 1 : na[i], in_b[i] = both ? 1 : nb[i], shared[i] = both ? std::max(na[i], nb[i]) : 1;
  }
  span_a = span_b = D;
  if (!steps(sa, in_a, &span_a) || !steps(sb, in_b, &span_b) || span_a > (__int128)gap) return false;
  __int128 span = gap + span_b;
  return steps(s, shared, &span);
}

}  // namespace ops
}  // namespace sffft
