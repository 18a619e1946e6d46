// The norms before and after a block, fused with its gate, its scale and the residual sum:
//   r = x + s . act(g) . (y ry) . wp,   h = (r rr) . wq,   rz = 1 / sqrt(mean z^2 + eps)
// With gr, gh the gradients of r and h, r^ = r rr and y^ = y ry:
//   dr = gr + rr (gh wq - r^ mean(gh wq r^)),      dx = dr,   dwq = sum gh r^
//   dg = dr s y^ wp act'(g),   dn = dr s act(g),   dy = ry (dn wp - y^ mean(dn wp y^))
//   ds = wp t,  dwp = s t  with  t = sum dr act(g) y^
// The weights leave the sums over rows, so that ds and dwp are one sum; so does a gate that many rows
// share, whose gradient is s wp act'(g) sum dr y^. r is not read back, it is made again from x, y and g: its
// stored value is rounded, and the weights' gradients would be off by that rounding.
//
// A row lies in the registers of one workgroup, 8 channels to a lane (16 beyond 8192 channels): every array crosses
// memory once. Rows of up to 256 channels take 16 or 32 lanes of a wavefront, which has several of them. Rows of
// more than 4096 channels leave a lane 128 registers: their gradients spill up to 87 of them, beyond 8192 channels
// up to 312 (25 M bf16 elements, gradients alone, us: C = 4096 118, 8192 178, 12288 444). A workgroup takes a run of
// rows and reads the next one before it works on this one (up to 4096 channels); sums over rows stay in registers
// until its end, and the parts it leaves are added by a second kernel in a fixed order. Bound by memory: 16384 x 4
// rows of 1536 in bf16, gate for each token, 561 us forward and backward for 2.6 GB.
//
// Rows of an odd width start anywhere between 16-byte boundaries. A workgroup then takes rows that start at the same
// distance from one (every 2nd, 4th or 8th) and reads them from the boundary before the row on: the vectors stay
// aligned and the lane's channels the same in all its rows, so that the sums over rows stay in registers.
#pragma once
#include "opsio.hpp"

namespace sffft {
namespace bn {

struct Args {
  const void *x, *y, *gate, *gr, *gh;
  long long sx, sy, sg, sgr, sgh;
  const float *wq, *wp, *sc;
  void *r, *h;            // forward
  void *dx, *dy, *dgate;  // backward; dgate only where each row has its own gate
  float* parts;           // [quantity][part][C]: dwq, t, and the gate's where rows share one
  long long rows, gate_rows, block_rows;  // block_rows: rows that may share a workgroup
  // A workgroup's part: part_rows rows, each `step` after the one before; `step` of them interleave
  int C, act, part_rows, step, parts_per_block;
  long long nparts;
  float eps;
};

// Rows first, first + step, .. below last of part `part`.
struct Part {
  long long first, last;
  __device__ __forceinline__ Part(const Args& A, int part) {
    const int block = part / A.parts_per_block, k = part - block * A.parts_per_block, group = k / A.step;
    const long long span = (long long)A.part_rows * A.step, base = block * A.block_rows;
    first = base + group * span + (k - group * A.step);
    last = min(min(base + (group + 1) * span, base + A.block_rows), A.rows);
  }
};

// act(g) and its derivative
__device__ __forceinline__ float activate(int act, float g, float* d) {
  if (act == 0) {
    *d = 1.f;
    return g;
  }
  const float s = 1.f / (1.f + __expf(-g));
  if (act == 1) {
    *d = s * (1.f - s);
    return s;
  }
  *d = s * (1.f + g * (1.f - s));
  return g * s;
}

// Sum over the 64 lanes: within 16 by DPP (xor 1, xor 2, and mirrors of 8 and 16), then the four rows.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane(float x, int l) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l));
}
// Sum over the 16 or 32 lanes of a row.
template <int LANES>
__device__ __forceinline__ float row_sum(float x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  x += dpp<0x140>(x);
  if constexpr (LANES == 32) x += __shfl_xor(x, 16);
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
  x = row_sum<16>(x);
  return (lane(x, 0) + lane(x, 16)) + (lane(x, 32) + lane(x, 48));
}

// Sums over the workgroup's W wavefronts. Successive sums use the two buffers in turn, so that one barrier each is
// enough: who writes a buffer again has passed the barrier that follows its last reading.
struct Sums {
  float v[2][2][16];
};
template <int BLK>
struct Reduce {
  Sums& s;
  int W, turn;
  template <int N>
  __device__ __forceinline__ void operator()(float (&v)[N]) {
    if constexpr (BLK < 64) {
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = row_sum<BLK>(v[i]);
      return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = wave_sum(v[i]);
    if (W == 1) return;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; i++) s.v[turn][i][w] = v[i];
    ops::barrier();
#pragma unroll
    for (int i = 0; i < N; i++) {
      v[i] = 0.f;
      for (int j = 0; j < W; j++) v[i] += s.v[turn][i][j];
    }
    turn ^= 1;
  }
};

// Where a lane's N channels lie: vector e of VEC at places (e * lanes + lane) * VEC. The row's channels are the
// places from `lo` to `hi`: it starts lo elements after a 16-byte boundary. (SHIFT; else lo is 0, and VEC divides C.)
// BLK below 64: the lanes of a row, of which a wavefront has several.
template <int VEC, int N, int BLK, bool SHIFT>
struct Places {
  static constexpr int ROWS = BLK < 64 ? 64 / BLK : 1;  // at once
  int lo, hi;
  __device__ __forceinline__ int at(int e) const {
    return (BLK < 64 ? e * BLK + (int)threadIdx.x % BLK : e * (int)blockDim.x + (int)threadIdx.x) * VEC;
  }
  static __device__ __forceinline__ int row() { return BLK < 64 ? (int)threadIdx.x / BLK : 0; }
  __device__ __forceinline__ bool holds(int place) const { return (!SHIFT || place >= lo) && place < hi; }
  // vector e lies in the row with all its elements
  __device__ __forceinline__ bool whole(int e) const { return !SHIFT || (at(e) >= lo && at(e) + VEC <= hi); }
};

// A lane's channels of a row, as they are in memory (bf16 two to a register, unless they come one by one).
template <class T, int VEC, int N, int BLK, bool SHIFT>
struct Row {
  static constexpr int PER = VEC == 1 ? 1 : 4 / (int)sizeof(T), WORDS = VEC / PER;
  typedef Places<VEC, N, BLK, SHIFT> P;
  uint32_t w[N / PER];
  static __device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x); }
  static __device__ __forceinline__ uint32_t bits(uint16_t x) { return x; }
  // element by element: of any alignment, nothing outside the row is read
  __device__ __forceinline__ void load_elements(const T* p, int e, const P& at) {
#pragma unroll
    for (int i = 0; i < VEC; i++)
      if (at.holds(at.at(e) + i)) w[(e * VEC + i) / PER] |= bits(p[at.at(e) + i]) << (sizeof(T) == 4 ? 0 : PER == 1 ? 16 : 16 * (i & 1));
  }
  // `edge`: the array's first or last row. In the others a vector that is not whole is read as a whole, with elements
  // of the neighbouring rows, which mask() clears.
  __device__ __forceinline__ void load(const void* base, long long row, long long stride, const P& at, bool edge, bool on = true) {
    const T* p = static_cast<const T*>(base) + row * stride - (SHIFT ? at.lo : 0);
#pragma unroll
    for (int e = 0; e < N / VEC; e++) {
      uint32_t* d = w + e * WORDS;
#pragma unroll
      for (int i = 0; i < WORDS; i++) d[i] = 0;
      if (on && at.at(e) < at.hi) {
        if constexpr (VEC == 1) {
          load_elements(p, e, at);
        } else if (SHIFT && edge && !at.whole(e)) {
          load_elements(p, e, at);
        } else {
          if constexpr (WORDS == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + at.at(e));
            d[0] = v.x, d[1] = v.y, d[2] = v.z, d[3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(p + at.at(e));
            d[0] = v.x, d[1] = v.y;
          }
        }
      }
    }
  }
  __device__ __forceinline__ void load_any(const void* base, long long row, long long stride, const P& at) {
    const T* p = static_cast<const T*>(base) + row * stride - (SHIFT ? at.lo : 0);
#pragma unroll
    for (int i = 0; i < N / PER; i++) w[i] = 0;
#pragma unroll
    for (int e = 0; e < N / VEC; e++) load_elements(p, e, at);
  }
  __device__ __forceinline__ void mask(const uint32_t (&m)[N / PER]) {
    if constexpr (SHIFT)
#pragma unroll
      for (int i = 0; i < N / PER; i++) w[i] &= m[i];
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (PER == 2) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __uint_as_float(w[i]);
  }
};
template <class T, int VEC, int N, int BLK, bool SHIFT>
__device__ __forceinline__ void put_row(void* base, long long row, int C, const Places<VEC, N, BLK, SHIFT>& at, const float (&x)[N]) {
  T* p = static_cast<T*>(base) + row * C - (SHIFT ? at.lo : 0);
#pragma unroll
  for (int e = 0; e < N / VEC; e++) {
    if (SHIFT && !at.whole(e)) {
#pragma unroll
      for (int i = 0; i < VEC; i++)
        if (at.holds(at.at(e) + i)) ops::put(p + at.at(e) + i, x[e * VEC + i]);
    } else if (at.at(e) < at.hi) {
      float t[VEC];
#pragma unroll
      for (int i = 0; i < VEC; i++) t[i] = x[e * VEC + i];
      ops::store(p + at.at(e), t);
    }
  }
}
// sums, channel by channel where the row is shifted: their rows are aligned in another way
template <int VEC, int N, int BLK, bool SHIFT>
__device__ __forceinline__ void put_sums(float* base, long long part, int C, const Places<VEC, N, BLK, SHIFT>& at, const float (&x)[N]) {
  if constexpr (!SHIFT) {
    put_row<float>(base, part, C, at, x);
  } else {
    float* p = base + part * C - at.lo;
#pragma unroll
    for (int e = 0; e < N / VEC; e++)
#pragma unroll
      for (int i = 0; i < VEC; i++)
        if (at.holds(at.at(e) + i)) p[at.at(e) + i] = x[e * VEC + i];
  }
}
// weights, 1 where there are none; 0 outside the row
template <int VEC, int N, int BLK, bool SHIFT>
__device__ __forceinline__ void weights(const float* p, const Places<VEC, N, BLK, SHIFT>& at, float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N / VEC; e++) {
    if constexpr (SHIFT) {
#pragma unroll
      for (int i = 0; i < VEC; i++) x[e * VEC + i] = !at.holds(at.at(e) + i) ? 0.f : p ? p[at.at(e) + i - at.lo] : 1.f;
    } else {
      float t[VEC];
      const bool in = at.at(e) < at.hi;
      if (p && in) ops::load(p + at.at(e), t);
#pragma unroll
      for (int i = 0; i < VEC; i++) x[e * VEC + i] = !p ? 1.f : in ? t[i] : 0.f;
    }
  }
}

// What both kernels share: the lane's places, the mask of its elements, and the gates that rows share.
template <class T, int VEC, int N, int BLK, bool SHIFT>
struct Lane {
  typedef Row<T, VEC, N, BLK, SHIFT> R;
  Places<VEC, N, BLK, SHIFT> at;
  uint32_t m[N / R::PER];
  __device__ __forceinline__ Lane(const Args& A, long long first) {
    at.lo = 0;
    if constexpr (SHIFT)
      at.lo = (int)((reinterpret_cast<uintptr_t>(A.x) + (uintptr_t)(first * A.sx) * sizeof(T)) % 16 / sizeof(T));
    at.hi = at.lo + A.C;
    if constexpr (SHIFT)
#pragma unroll
      for (int i = 0; i < N / R::PER; i++) {
        const int p = at.at(i / R::WORDS) + i % R::WORDS * R::PER;
        m[i] = R::PER == 1 ? (at.holds(p) ? ~0u : 0u) : (at.holds(p) ? 0xffffu : 0u) | (at.holds(p + 1) ? 0xffff0000u : 0u);
      }
  }
  // gate i, which lies at another distance from a boundary than the rows
  __device__ __forceinline__ void gate(const Args& A, long long i, R& g) const {
    if constexpr (SHIFT) g.load_any(A.gate, i, A.sg, at);
    else g.load(A.gate, i, A.sg, at, false);
  }
};

template <class T, int VEC, int N, int BLK, bool SHIFT, bool Y>
__global__ __launch_bounds__(BLK < 64 ? 64 : BLK, BLK > 512 ? 4 : VEC == 1 || BLK < 64 ? 5 : 6) void fwd_kernel(Args A) {
  constexpr bool AHEAD = BLK <= 512;  // 1024 lanes leave each 128 registers: none for a row in advance
  __shared__ Sums sums;
  Reduce<BLK> reduce = {sums, (int)blockDim.x >> 6, 0};
  const Part part(A, blockIdx.x);
  Lane<T, VEC, N, BLK, SHIFT> lane(A, part.first);
  const auto& at = lane.at;
  const bool shared = A.gate && A.gate_rows > 1;
  float wq[N], ws[N];
  weights(A.wq, at, wq);
  if constexpr (Y) {
    float sc[N];
    weights(A.wp, at, ws);
    weights(A.sc, at, sc);
#pragma unroll
    for (int i = 0; i < N; i++) ws[i] *= sc[i];
  }
  const float inv = 1.f / (float)A.C;
  Row<T, VEC, N, BLK, SHIFT> nx, ny, ng, rg;
  const long long run = (long long)at.ROWS * A.step;
  auto fetch = [&](long long row) {
    row += at.row() * A.step;
    const bool edge = row == 0 || row == A.rows - 1, on = at.ROWS == 1 || row < part.last;
    nx.load(A.x, row, A.sx, at, edge, on);
    if constexpr (Y) {
      ny.load(A.y, row, A.sy, at, edge, on);
      if (A.gate && !shared) ng.load(A.gate, row, A.sg, at, edge, on);
    }
  };
  if (AHEAD && part.first < part.last) fetch(part.first);
  if constexpr (Y)  // rows of a part share theirs
    if (shared && part.first < part.last) lane.gate(A, part.first / A.gate_rows, rg);
  for (long long row0 = part.first; row0 < part.last; row0 += run) {
    if (!AHEAD) fetch(row0);
    const long long row = row0 + at.row() * A.step;
    const bool on = at.ROWS == 1 || row < part.last;
    const float eps = on ? A.eps : 1.f;
    Row<T, VEC, N, BLK, SHIFT> rx = nx, ry = ny;
    rx.mask(lane.m);
    if constexpr (Y) {
      ry.mask(lane.m);
      if (!shared) rg = ng, rg.mask(lane.m);
    }
    if (AHEAD && row0 + run < part.last) fetch(row0 + run);
    float x[N], s[1];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = rx[i];
    if constexpr (Y) {
      float f = 1.f, d;
      if (A.wp) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) s[0] += ry[i] * ry[i];
        reduce(s);
        f = 1.f / sqrtf(s[0] * inv + eps);
      }
#pragma unroll
      for (int i = 0; i < N; i++) {
        float m = ry[i] * f * ws[i];
        if (A.gate) m *= activate(A.act, rg[i], &d);
        x[i] += m;
      }
      if (on) put_row<T>(A.r, row, A.C, at, x);
    }
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) s[0] += x[i] * x[i];
    reduce(s);
    const float f = 1.f / sqrtf(s[0] * inv + eps);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] *= f * wq[i];
    if (on) put_row<T>(A.h, row, A.C, at, x);
  }
}

template <class T, int VEC, int N, int BLK, bool SHIFT, bool Y>
__global__ __launch_bounds__(BLK < 64 ? 64 : BLK) void bwd_kernel(Args A) {
  constexpr bool AHEAD = BLK <= 512;  // 1024 lanes leave each 128 registers: none for a row in advance
  __shared__ Sums sums;
  Reduce<BLK> reduce = {sums, (int)blockDim.x >> 6, 0};
  const Part part(A, blockIdx.x);
  Lane<T, VEC, N, BLK, SHIFT> lane(A, part.first);
  const auto& at = lane.at;
  const bool shared = A.gate && A.gate_rows > 1;
  const float inv = 1.f / (float)A.C;
  float wq[N], wp[N], sc[N], dwq[N], t[N];
  weights(A.wq, at, wq);
#pragma unroll
  for (int i = 0; i < N; i++) dwq[i] = t[i] = 0.f;
  if constexpr (Y) {
    weights(A.wp, at, wp);
    weights(A.sc, at, sc);
  }
  Row<T, VEC, N, BLK, SHIFT> nx, ny, ng, nr, nh;
  const long long run = (long long)at.ROWS * A.step;
  auto fetch = [&](long long row) {
    row += at.row() * A.step;
    const bool edge = row == 0 || row == A.rows - 1, on = at.ROWS == 1 || row < part.last;
    nx.load(A.x, row, A.sx, at, edge, on);
    if constexpr (Y) {
      ny.load(A.y, row, A.sy, at, edge, on);
      if (A.gate && !shared) ng.load(A.gate, row, A.sg, at, edge, on);
    }
    if (A.gr) nr.load(A.gr, row, A.sgr, at, edge, on);
    if (A.gh) nh.load(A.gh, row, A.sgh, at, edge, on);
  };
  if (!A.gr) nr = {};
  if (!A.gh) nh = {};
  if (AHEAD && part.first < part.last) fetch(part.first);
  Row<T, VEC, N, BLK, SHIFT> rg = {};
  if constexpr (Y)  // rows of a part share theirs
    if (shared && part.first < part.last) lane.gate(A, part.first / A.gate_rows, rg);
  for (long long row0 = part.first; row0 < part.last; row0 += run) {
    if (!AHEAD) fetch(row0);
    const long long row = row0 + at.row() * A.step;
    const bool on = at.ROWS == 1 || row < part.last;
    const float eps = on ? A.eps : 1.f;
    Row<T, VEC, N, BLK, SHIFT> rx = nx, ry = ny, rr = nr, rh = nh;
    rx.mask(lane.m), rr.mask(lane.m), rh.mask(lane.m);
    if constexpr (Y) {
      ry.mask(lane.m);
      if (!shared) rg = ng, rg.mask(lane.m);
    }
    if (AHEAD && row0 + run < part.last) fetch(row0 + run);
    float r[N], y[N], act[N], s[1], fy = 1.f, d;
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = rx[i];
    if constexpr (Y) {
      if (A.wp) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) s[0] += ry[i] * ry[i];
        reduce(s);
        fy = 1.f / sqrtf(s[0] * inv + eps);
      }
#pragma unroll
      for (int i = 0; i < N; i++) {
        act[i] = A.gate ? activate(A.act, rg[i], &d) : 1.f;
        y[i] = ry[i] * fy;
        r[i] += y[i] * wp[i] * sc[i] * act[i];
      }
    }
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; i++) q[0] += r[i] * r[i], q[1] += rh[i] * wq[i] * r[i];
    reduce(q);
    const float fr = 1.f / sqrtf(q[0] * inv + eps), mean = q[1] * fr * inv;
    float dr[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      r[i] *= fr;
      dwq[i] += rh[i] * r[i];
      dr[i] = rr[i] + fr * (rh[i] * wq[i] - r[i] * mean);
    }
    if (on) put_row<T>(A.dx, row, A.C, at, dr);
    if constexpr (Y) {
      if (shared) {
#pragma unroll
        for (int i = 0; i < N; i++) t[i] += dr[i] * y[i];
      } else {
#pragma unroll
        for (int i = 0; i < N; i++) t[i] += dr[i] * y[i] * act[i];
      }
      if (A.gate && !shared) {
        float g[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
          activate(A.act, rg[i], &d);
          g[i] = dr[i] * sc[i] * y[i] * wp[i] * d;
        }
        if (on) put_row<T>(A.dgate, row, A.C, at, g);
      }
#pragma unroll
      for (int i = 0; i < N; i++) dr[i] *= sc[i] * act[i];
      if (A.wp) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) {
          dr[i] *= wp[i];
          s[0] += dr[i] * y[i];
        }
        reduce(s);
        const float my = s[0] * inv;
#pragma unroll
        for (int i = 0; i < N; i++) dr[i] = fy * (dr[i] - y[i] * my);
      }
      if (on) put_row<T>(A.dy, row, A.C, at, dr);
    }
  }
  if constexpr (BLK < 64) {  // the sums of a wavefront's rows
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int o = BLK; o < 64; o *= 2) {
        dwq[i] += __shfl_xor(dwq[i], o);
        if constexpr (Y) t[i] += __shfl_xor(t[i], o);
      }
    if (at.row()) return;
  }
  put_sums(A.parts, blockIdx.x, A.C, at, dwq);
  if constexpr (Y) {
    if (shared) {
      float g[N], d;
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float a = activate(A.act, rg[i], &d);
        g[i] = t[i] * sc[i] * wp[i] * d;
        t[i] *= a;
      }
      put_sums(A.parts, 2 * A.nparts + blockIdx.x, A.C, at, g);
    }
    put_sums(A.parts, A.nparts + blockIdx.x, A.C, at, t);
  }
}

// The sums of the parts (1024 parts of three quantities of 1531 channels: 19 MB in 7 us; rows of such widths start
// between cache lines, and the 32 columns of a workgroup lie in two of them: 37 MB are fetched). Workgroups take 32
// columns of one quantity: the nparts parts of dwq and of t, which gives dwp and ds, then for each gate that rows share its
// `per` consecutive parts. There may be more quantities than the grid has rows.
struct SumArgs {
  const float *parts, *wp, *sc;
  float *dwq, *dwp, *ds;
  void* dgate;
  int C, bf16, y;
  long long nparts, per, sums;
};
__global__ __launch_bounds__(1024) void sum_kernel(SumArgs A) {
  __shared__ float lds[32][33];
  const int lc = threadIdx.x & 31, g = threadIdx.x >> 5, c = blockIdx.x * 32 + lc;
  for (long long which = blockIdx.y; which < A.sums; which += gridDim.y) {
    // which: 0 = dwq, 1 = t (where there is a y), then the gates
    const long long gate = which - (A.y ? 2 : 1);
    const long long n = gate < 0 ? A.nparts : A.per, at = gate < 0 ? which * A.nparts : 2 * A.nparts + gate * A.per;
    const float* p = A.parts + at * A.C + c;
    float s = 0.f;
    if (c < A.C) {
      long long i = g;
      for (; i + 7 * 32 < n; i += 8 * 32) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = p[(i + 32 * k) * A.C];
#pragma unroll
        for (int k = 0; k < 8; k++) s += v[k];
      }
      for (; i < n; i += 32) s += p[i * A.C];
    }
    lds[g][lc] = s;
    ops::barrier();
    // 32 lanes add 32 rows: lane (g, lc) of the first wavefronts takes column g
    s = lds[lc][g];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor(s, o);
    const int col = blockIdx.x * 32 + g;
    if (!lc && col < A.C) {
      if (which == 0) {
        A.dwq[col] = s;
      } else if (gate < 0) {
        if (A.dwp) A.dwp[col] = A.sc ? A.sc[col] * s : s;
        if (A.ds) A.ds[col] = A.wp ? A.wp[col] * s : s;
      } else if (A.bf16) {
        ops::put(static_cast<uint16_t*>(A.dgate) + gate * A.C + col, s);
      } else {
        static_cast<float*>(A.dgate)[gate * A.C + col] = s;
      }
    }
    ops::barrier();  // before the next sum takes the array
  }
}

}  // namespace bn
}  // namespace sffft
