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
// memory once. A workgroup takes a run of rows and reads the next one before it works on this one (up to 4096 channels);
// sums over rows stay in registers until its end, and the parts it leaves are added by a second kernel in a
// fixed order. Bound by memory.
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
  int C, act, part_rows, parts_per_block;
  long long nparts;
  float eps;
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
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  x += dpp<0x140>(x);
  return (lane(x, 0) + lane(x, 16)) + (lane(x, 32) + lane(x, 48));
}

// Sums over the workgroup's W wavefronts. Successive sums use the two buffers in turn, so that one barrier each is
// enough: who writes a buffer again has passed the barrier that follows its last reading.
struct Sums {
  float v[2][2][16];
};
struct Reduce {
  Sums& s;
  int W, turn;
  template <int N>
  __device__ __forceinline__ void operator()(float (&v)[N]) {
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

// A lane's N channels of a row, as they are in memory (bf16 two to a register, unless they come one by
// one): vector e of VEC at (e * lanes + lane) * VEC.
template <class T, int VEC, int N>
struct Row {
  static constexpr int PER = VEC == 1 ? 1 : 4 / (int)sizeof(T), WORDS = VEC / PER;
  uint32_t w[N / PER];
  __device__ __forceinline__ void load(const void* base, long long row, long long stride, int C) {
    const T* p = static_cast<const T*>(base) + row * stride;
#pragma unroll
    for (int e = 0; e < N / VEC; e++) {
      const int at = (e * (int)blockDim.x + (int)threadIdx.x) * VEC;
      uint32_t* d = w + e * WORDS;
#pragma unroll
      for (int i = 0; i < WORDS; i++) d[i] = 0;
      if (at < C) {
        if constexpr (WORDS == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(p + at);
          d[0] = v.x, d[1] = v.y, d[2] = v.z, d[3] = v.w;
        } else if constexpr (WORDS == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(p + at);
          d[0] = v.x, d[1] = v.y;
        } else if constexpr (sizeof(T) == 4) {
          d[0] = __float_as_uint(p[at]);
        } else {
          d[0] = (uint32_t)p[at] << 16;
        }
      }
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (PER == 2) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __uint_as_float(w[i]);
  }
};
template <class T, int VEC, int N>
__device__ __forceinline__ void put_row(void* base, long long row, int C, const float (&x)[N]) {
  T* p = static_cast<T*>(base) + row * C;
#pragma unroll
  for (int e = 0; e < N / VEC; e++) {
    const int at = (e * (int)blockDim.x + (int)threadIdx.x) * VEC;
    float t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) t[i] = x[e * VEC + i];
    if (at < C) ops::store(p + at, t);
  }
}
// weights, 1 where there are none
template <int VEC, int N>
__device__ __forceinline__ void weights(const float* p, int C, float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N / VEC; e++) {
    const int at = (e * (int)blockDim.x + (int)threadIdx.x) * VEC;
    float t[VEC];
    if (p && at < C) ops::load(p + at, t);
#pragma unroll
    for (int i = 0; i < VEC; i++) x[e * VEC + i] = !p ? 1.f : at < C ? t[i] : 0.f;
  }
}

template <class T, int VEC, int N, int BLK, bool Y>
__global__ __launch_bounds__(BLK) void fwd_kernel(Args A) {
  constexpr bool AHEAD = BLK <= 512;  // 1024 lanes leave each 128 registers: none for a row in advance
  __shared__ Sums sums;
  Reduce reduce = {sums, (int)blockDim.x >> 6, 0};
  const long long first = (long long)blockIdx.x * A.part_rows, last = min(first + A.part_rows, A.rows);
  float wq[N], ws[N];
  weights<VEC>(A.wq, A.C, wq);
  if constexpr (Y) {
    float sc[N];
    weights<VEC>(A.wp, A.C, ws);
    weights<VEC>(A.sc, A.C, sc);
#pragma unroll
    for (int i = 0; i < N; i++) ws[i] *= sc[i];
  }
  const float inv = 1.f / (float)A.C;
  Row<T, VEC, N> nx, ny, ng;
  auto fetch = [&](long long row) {
    nx.load(A.x, row, A.sx, A.C);
    if constexpr (Y) {
      ny.load(A.y, row, A.sy, A.C);
      if (A.gate) ng.load(A.gate, A.gate_rows == 1 ? row : row / A.gate_rows, A.sg, A.C);
    }
  };
  if (AHEAD) fetch(first);
  for (long long row = first; row < last; row++) {
    if (!AHEAD) fetch(row);
    const Row<T, VEC, N> rx = nx, ry = ny, rg = ng;
    if (AHEAD && row + 1 < last) fetch(row + 1);
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
        f = 1.f / sqrtf(s[0] * inv + A.eps);
      }
#pragma unroll
      for (int i = 0; i < N; i++) {
        float m = ry[i] * f * ws[i];
        if (A.gate) m *= activate(A.act, rg[i], &d);
        x[i] += m;
      }
      put_row<T, VEC>(A.r, row, A.C, x);
    }
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) s[0] += x[i] * x[i];
    reduce(s);
    const float f = 1.f / sqrtf(s[0] * inv + A.eps);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] *= f * wq[i];
    put_row<T, VEC>(A.h, row, A.C, x);
  }
}

template <class T, int VEC, int N, int BLK, bool Y>
__global__ __launch_bounds__(BLK) void bwd_kernel(Args A) {
  constexpr bool AHEAD = BLK <= 512;  // 1024 lanes leave each 128 registers: none for a row in advance
  __shared__ Sums sums;
  Reduce reduce = {sums, (int)blockDim.x >> 6, 0};
  const long long part = blockIdx.x, block = part / A.parts_per_block;
  const long long first = block * A.block_rows + (part - block * A.parts_per_block) * A.part_rows;
  const long long last = min(min(first + A.part_rows, (block + 1) * A.block_rows), A.rows);
  const bool shared = A.gate && A.gate_rows > 1;
  const float inv = 1.f / (float)A.C;
  float wq[N], wp[N], sc[N], dwq[N], t[N];
  weights<VEC>(A.wq, A.C, wq);
#pragma unroll
  for (int i = 0; i < N; i++) dwq[i] = t[i] = 0.f;
  if constexpr (Y) {
    weights<VEC>(A.wp, A.C, wp);
    weights<VEC>(A.sc, A.C, sc);
  }
  Row<T, VEC, N> nx, ny, ng, nr, nh;
  auto fetch = [&](long long row) {
    nx.load(A.x, row, A.sx, A.C);
    if constexpr (Y) {
      ny.load(A.y, row, A.sy, A.C);
      if (A.gate) ng.load(A.gate, shared ? row / A.gate_rows : row, A.sg, A.C);
    }
    if (A.gr) nr.load(A.gr, row, A.sgr, A.C);
    if (A.gh) nh.load(A.gh, row, A.sgh, A.C);
  };
  if (!A.gr) nr = {};
  if (!A.gh) nh = {};
  if (AHEAD) fetch(first);
  Row<T, VEC, N> rg = {};
  for (long long row = first; row < last; row++) {
    if (!AHEAD) fetch(row);
    const Row<T, VEC, N> rx = nx, ry = ny, rr = nr, rh = nh;
    rg = ng;
    if (AHEAD && row + 1 < last) fetch(row + 1);
    float r[N], y[N], act[N], s[1], fy = 1.f, d;
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = rx[i];
    if constexpr (Y) {
      if (A.wp) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) s[0] += ry[i] * ry[i];
        reduce(s);
        fy = 1.f / sqrtf(s[0] * inv + A.eps);
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
    const float fr = 1.f / sqrtf(q[0] * inv + A.eps), mean = q[1] * fr * inv;
    float dr[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      r[i] *= fr;
      dwq[i] += rh[i] * r[i];
      dr[i] = rr[i] + fr * (rh[i] * wq[i] - r[i] * mean);
    }
    put_row<T, VEC>(A.dx, row, A.C, dr);
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
        put_row<T, VEC>(A.dgate, row, A.C, g);
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
      put_row<T, VEC>(A.dy, row, A.C, dr);
    }
  }
  put_row<float, VEC>(A.parts, part, A.C, dwq);
  if constexpr (Y) {
    if (shared) {
      float g[N], d;
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float a = activate(A.act, rg[i], &d);
        g[i] = t[i] * sc[i] * wp[i] * d;
        t[i] *= a;
      }
      put_row<float, VEC>(A.parts, 2 * A.nparts + part, A.C, g);
    }
    put_row<float, VEC>(A.parts, A.nparts + part, A.C, t);
  }
}

// The sums of the parts. Workgroups take 32 columns of one quantity: the nparts parts of dwq and of t, which gives
// dwp and ds, then for each gate that rows share its `per` consecutive parts.
struct SumArgs {
  const float *parts, *wp, *sc;
  float *dwq, *dwp, *ds;
  void* dgate;
  int C, bf16, y;
  long long nparts, per;
};
__global__ __launch_bounds__(1024) void sum_kernel(SumArgs A) {
  __shared__ float lds[32][33];
  const int tiles = (A.C + 31) / 32, which = blockIdx.x / tiles, lc = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int c = (blockIdx.x - which * tiles) * 32 + lc;
  // which: 0 = dwq, 1 = t (where there is a y), then the gates
  const int gate = which - (A.y ? 2 : 1);
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
  const int col = (blockIdx.x - which * tiles) * 32 + g;
  if (lc || col >= A.C) return;
  if (which == 0) {
    A.dwq[col] = s;
  } else if (gate < 0) {
    if (A.dwp) A.dwp[col] = A.sc ? A.sc[col] * s : s;
    if (A.ds) A.ds[col] = A.wp ? A.wp[col] * s : s;
  } else if (A.bf16) {
    ops::put(static_cast<uint16_t*>(A.dgate) + (long long)gate * A.C + col, s);
  } else {
    static_cast<float*>(A.dgate)[(long long)gate * A.C + col] = s;
  }
}

}  // namespace bn
}  // namespace sffft
