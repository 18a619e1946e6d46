// Rotary positions of q and k in one launch. A pair (a, b) of channels turns by its position's angle,
//   a' = a cos - b sin,   b' = b cos + a sin,
// with the cosines and sines of a position in one row of a table. Bound by memory: every element is
// read and written once.
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
  int T, H, heads, D, R, inverse;  // heads: of q and k together
  long long items;
};

// A lane takes PP pairs of one head of one token, or 2 PP of the channels that are copied.
template <class T, int PP, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(Args A) {
  const int units = A.D / (2 * PP), turned = A.R / (2 * PP);
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= A.items) return;
  const long long at = i / units, bt = at / A.heads;
  const int u = (int)(i - at * units), head = (int)(at - bt * A.heads);
  const long long b = bt / A.T;
  const int t = (int)(bt - b * A.T);
  const Side& s = head < A.H ? A.q : A.k;
  const int h = head < A.H ? head : head - A.H;
  const T* x = static_cast<const T*>(s.x) + b * s.sb + t * s.st + h * s.sh;
  T* y = static_cast<T*>(s.y) + b * s.ob + t * s.ot + h * s.oh;
  if (u >= turned) {  // copied
    if (x == y) return;
    float v[2 * PP];
    ops::load(x + u * 2 * PP, v);
    ops::store(y + u * 2 * PP, v);
    return;
  }
  const long long p = !A.pos ? t : A.pos64 ? static_cast<const long long*>(A.pos)[bt] : static_cast<const int*>(A.pos)[bt];
  float c[PP], sn[PP];
  if (p >= 0 && p < A.positions) {
    const float* row = A.table + p * A.R + u * PP;
    ops::load(row, c);
    ops::load(row + A.R / 2, sn);
  } else {
#pragma unroll
    for (int e = 0; e < PP; e++) c[e] = sn[e] = __builtin_nanf("");
  }
  const float sign = A.inverse ? -1.f : 1.f;
  if constexpr (INTERLEAVED) {
    float v[2 * PP], w[2 * PP];
    ops::load(x + u * 2 * PP, v);
#pragma unroll
    for (int e = 0; e < PP; e++) {
      w[2 * e] = v[2 * e] * c[e] - v[2 * e + 1] * (sign * sn[e]);
      w[2 * e + 1] = v[2 * e + 1] * c[e] + v[2 * e] * (sign * sn[e]);
    }
    ops::store(y + u * 2 * PP, w);
  } else {
    float v[PP], w[PP], a[PP], z[PP];
    ops::load(x + u * PP, v);
    ops::load(x + A.R / 2 + u * PP, w);
#pragma unroll
    for (int e = 0; e < PP; e++) {
      a[e] = v[e] * c[e] - w[e] * (sign * sn[e]);
      z[e] = w[e] * c[e] + v[e] * (sign * sn[e]);
    }
    ops::store(y + u * PP, a);
    ops::store(y + A.R / 2 + u * PP, z);
  }
}

}  // namespace rot
}  // namespace sffft
