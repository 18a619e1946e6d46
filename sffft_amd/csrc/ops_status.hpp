// The error text of libsffft_ops.so and the checks its entry points share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

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

}  // namespace ops
}  // namespace sffft
