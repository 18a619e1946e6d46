// Rotary positions of q and k in one launch. A pair (a, b) of channels turns by its position's angle,
//   a' = a cos - b sin,   b' = b cos + a sin,
// with the cosines and sines of a position in one row of a table. Bound by memory: every element is read and written
// once. 65536 tokens, 12 + 12 heads of 64, fp32: 137 us, 5.9 TB/s (partly from the Infinity Cache); 8 x 2048 tokens,
// 12 + 4 heads of 128, bf16, interleaved: 27 to 30 us, 4.5 TB/s.
#pragma once
#include "opsio.hpp"

namespace sffft {
namespace rot {

struct Side {
  const void* x;
  void* y;
  long long sb, st, sh, ob, ot, oh;
};

struct Args {
  Side q, k;
  const float* table;
  const void* pos;
  int pos64, positions;
  unsigned tokens, T;  // T = tokens where one stride leads through all of them
  int H, heads, D, R, inverse;  // heads: of q and k together
  unsigned units, per, wg_tokens, by_units, by_per;  // units of a head, of a token; ceil(2^32 / units), ceil(2^32 / per)
};

// n / d for n * d < 2^32, from m = ceil(2^32 / d)
__device__ __forceinline__ unsigned divide(unsigned n, unsigned d, unsigned m) { return d == 1 ? n : __umulhi(n, m); }

// A lane takes one unit of one head of one token: half layout, PP pairs in two vectors; interleaved, PP pairs in one;
// of the channels that are copied as much. Neighbouring lanes take neighbouring vectors.
template <class T, int PP, bool INTERLEAVED>
__device__ __forceinline__ void rotate_unit(const Args& A, unsigned token, unsigned b, unsigned t, unsigned head, unsigned u) {
  const bool first = head < (unsigned)A.H;
  const Side& s = first ? A.q : A.k;
  const int h = first ? head : head - A.H;
  const T* x = static_cast<const T*>(s.x) + b * s.sb + t * s.st + h * s.sh;
  T* y = static_cast<T*>(s.y) + b * s.ob + t * s.ot + h * s.oh;
  const unsigned turned = A.R / (2 * PP);
  const bool turn = u < turned;
  if (!turn && x == y) return;
  float c[PP], sn[PP];
  if (turn) {
    const long long p = !A.pos ? t : A.pos64 ? static_cast<const long long*>(A.pos)[token] : static_cast<const int*>(A.pos)[token];
    if (p >= 0 && p < A.positions) {
      const float* row = A.table + p * A.R + u * PP;
      ops::load(row, c);
      ops::load(row + A.R / 2, sn);
    } else {
#pragma unroll
      for (int e = 0; e < PP; e++) c[e] = sn[e] = __builtin_nanf("");
    }
    if (A.inverse)
#pragma unroll
      for (int e = 0; e < PP; e++) sn[e] = -sn[e];
  }
  if constexpr (INTERLEAVED) {
    float z[2 * PP];
    ops::load(x + 2 * PP * u, z);
    if (turn)
#pragma unroll
      for (int e = 0; e < PP; e++) {
        const float a = z[2 * e], d = z[2 * e + 1];
        z[2 * e] = a * c[e] - d * sn[e];
        z[2 * e + 1] = d * c[e] + a * sn[e];
      }
    ops::store(y + 2 * PP * u, z);
  } else {
    // the copied channels too in two halves
    const unsigned lo = turn ? PP * u : A.R + PP * (u - turned), hi = lo + (turn ? A.R : A.D - A.R) / 2;
    float v[PP], w[PP];
    ops::load(x + lo, v);
    ops::load(x + hi, w);
    if (turn)
#pragma unroll
      for (int e = 0; e < PP; e++) {
        const float a = v[e], d = w[e];
        v[e] = a * c[e] - d * sn[e];
        w[e] = d * c[e] + a * sn[e];
      }
    ops::store(y + lo, v);
    ops::store(y + hi, w);
  }
}

template <class T, int PP, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(Args A) {
  const unsigned token0 = blockIdx.x * A.wg_tokens, items = min(A.wg_tokens, A.tokens - token0) * A.per;
  for (unsigned i = threadIdx.x; i < items; i += 256) {
    const unsigned k = divide(i, A.per, A.by_per), r = i - k * A.per, head = divide(r, A.units, A.by_units);
    const unsigned token = token0 + k, b = A.T == A.tokens ? 0 : token / A.T;
    rotate_unit<T, PP, INTERLEAVED>(A, token, b, token - b * A.T, head, r - head * A.units);
  }
}

}  // namespace rot
}  // namespace sffft
