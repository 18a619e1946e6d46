// The norms before and after a block, fused with its gate, its scale and the residual sum:
//   r = x + s . act(g) . (y ry) . wp,   h = (r rr) . wq,   rz = 1 / sqrt(mean z^2 + eps)
// With gr, gh the gradients of r and h, r^ = r rr and y^ = y ry:
//   dr = gr + rr (gh wq - r^ mean(gh wq r^)),      dx = dr,   dwq = sum gh r^
//   ds = sum dr act(g) y^ wp,   dg = dr s y^ wp act'(g),   dn = dr s act(g),   dwp = sum dn y^
//   dy = ry (dn wp - y^ mean(dn wp y^))
// r is not read back, it is made again from x, y and g: its stored value is rounded, and the sums over
// rows of the weights' gradients would be off by that rounding.
//
// A row lies in the registers of one wavefront, or of one workgroup where it is longer than 1024
// channels: every array crosses memory once. A workgroup takes a run of rows, so that the weights are
// read once for all of them and the sums over rows stay in registers until its end; the parts it leaves
// are added by a second kernel, in a fixed order.
#pragma once
#include "opsio.hpp"

namespace sffft {
namespace bn {

struct Args {
  const void *x, *y, *gate, *gr, *gh;
  long long sx, sy, sg, sgr, sgh;
  const float *wq, *wp, *sc;
  void *r, *h;           // forward
  void *dx, *dy, *dgate; // backward; dgate only where each row has its own gate
  float* parts;          // [quantity][part][C]: dwq, dwp, ds, and the gate's where rows share one
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

// Sums of N values over the lanes of a row: W wavefronts.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int W, float* lds) {
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int o = 32; o; o >>= 1) v[i] += __shfl_xor(v[i], o);
  if (W == 1) return;
  const int w = threadIdx.x >> 6;
  __syncthreads();  // the last sum has been read
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < N; i++) lds[w * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; i++) {
    v[i] = 0.f;
    for (int j = 0; j < W; j++) v[i] += lds[j * N + i];
  }
}

// The channels of a lane: vector e of VEC at (e * lanes + lane) * VEC.
template <class T, int VEC, int NV>
__device__ __forceinline__ void get(const T* p, int lane, int lanes, int C, float (&v)[NV * VEC], float fill) {
#pragma unroll
  for (int e = 0; e < NV; e++) {
    const int at = (e * lanes + lane) * VEC;
    float t[VEC];
    if (at < C) ops::load(p + at, t);
#pragma unroll
    for (int i = 0; i < VEC; i++) v[e * VEC + i] = at < C ? t[i] : fill;
  }
}
template <class T, int VEC, int NV>
__device__ __forceinline__ void set(T* p, int lane, int lanes, int C, const float (&v)[NV * VEC]) {
#pragma unroll
  for (int e = 0; e < NV; e++) {
    const int at = (e * lanes + lane) * VEC;
    float t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) t[i] = v[e * VEC + i];
    if (at < C) ops::store(p + at, t);
  }
}

template <class T, int VEC, int NV, int BLK, bool Y>
__global__ __launch_bounds__(BLK) void fwd_kernel(Args A) {
  constexpr int N = VEC * NV;
  __shared__ float lds[16 * 2];
  // rows of one wavefront: four to a workgroup; else one row to a workgroup
  const int W = A.C <= 64 * N ? 1 : blockDim.x >> 6, lanes = 64 * W;
  const int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x, group = W == 1 ? threadIdx.x >> 6 : 0;
  const int groups = W == 1 ? blockDim.x >> 6 : 1;
  const long long first = (long long)blockIdx.x * A.part_rows, last = min(first + A.part_rows, A.rows);
  float wq[N], wp[N], sc[N];
  get<float, VEC, NV>(A.wq, lane, lanes, A.C, wq, 0.f);
  if constexpr (Y) {
#pragma unroll
    for (int i = 0; i < N; i++) wp[i] = sc[i] = 1.f;
    if (A.wp) get<float, VEC, NV>(A.wp, lane, lanes, A.C, wp, 0.f);
    if (A.sc) get<float, VEC, NV>(A.sc, lane, lanes, A.C, sc, 0.f);
  }
  const float inv = 1.f / (float)A.C;
  for (long long row = first + group; row < last; row += groups) {
    float x[N], s[1];
    get<T, VEC, NV>(static_cast<const T*>(A.x) + row * A.sx, lane, lanes, A.C, x, 0.f);
    if constexpr (Y) {
      float y[N], g[N], d;
      get<T, VEC, NV>(static_cast<const T*>(A.y) + row * A.sy, lane, lanes, A.C, y, 0.f);
      if (A.gate) get<T, VEC, NV>(static_cast<const T*>(A.gate) + row / A.gate_rows * A.sg, lane, lanes, A.C, g, 0.f);
      float ry = 1.f;
      if (A.wp) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) s[0] += y[i] * y[i];
        row_sum(s, W, lds);
        ry = 1.f / sqrtf(s[0] * inv + A.eps);
      }
#pragma unroll
      for (int i = 0; i < N; i++) {
        float m = y[i] * ry * wp[i] * sc[i];
        if (A.gate) m *= activate(A.act, g[i], &d);
        x[i] += m;
      }
      set<T, VEC, NV>(static_cast<T*>(A.r) + row * A.C, lane, lanes, A.C, x);
    }
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) s[0] += x[i] * x[i];
    row_sum(s, W, lds);
    const float rr = 1.f / sqrtf(s[0] * inv + A.eps);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] *= rr * wq[i];
    set<T, VEC, NV>(static_cast<T*>(A.h) + row * A.C, lane, lanes, A.C, x);
  }
}

// Adds the four wavefronts' values of one quantity and writes the workgroup's part.
template <int VEC, int NV>
__device__ __forceinline__ void put_part(float* part, float* lds, int lane, int lanes, int C, int group, int groups,
                                         float (&v)[NV * VEC]) {
  if (groups > 1) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV * VEC; i++) lds[(group * NV * VEC + i) * 64 + lane] = v[i];
    __syncthreads();
    if (group) return;
    for (int g = 1; g < groups; g++)
#pragma unroll
      for (int i = 0; i < NV * VEC; i++) v[i] += lds[(g * NV * VEC + i) * 64 + lane];
  }
  set<float, VEC, NV>(part, lane, lanes, C, v);
}

template <class T, int VEC, int NV, int BLK, bool Y>
__global__ __launch_bounds__(BLK) void bwd_kernel(Args A) {
  constexpr int N = VEC * NV;
  __shared__ float lds[4 * N * 64];
  const int W = A.C <= 64 * N ? 1 : blockDim.x >> 6, lanes = 64 * W;
  const int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x, group = W == 1 ? threadIdx.x >> 6 : 0;
  const int groups = W == 1 ? blockDim.x >> 6 : 1;
  const long long part = blockIdx.x, block = part / A.parts_per_block;
  const long long first = block * A.block_rows + (part - block * A.parts_per_block) * A.part_rows;
  const long long last = min(min(first + A.part_rows, (block + 1) * A.block_rows), A.rows);
  float wq[N], wp[N], sc[N], dwq[N], dwp[N], dsc[N], dgs[N];
  get<float, VEC, NV>(A.wq, lane, lanes, A.C, wq, 0.f);
#pragma unroll
  for (int i = 0; i < N; i++) wp[i] = sc[i] = 1.f, dwq[i] = dwp[i] = dsc[i] = dgs[i] = 0.f;
  if constexpr (Y) {
    if (A.wp) get<float, VEC, NV>(A.wp, lane, lanes, A.C, wp, 0.f);
    if (A.sc) get<float, VEC, NV>(A.sc, lane, lanes, A.C, sc, 0.f);
  }
  const float inv = 1.f / (float)A.C;
  const bool shared_gate = A.gate_rows > 1;
  for (long long row = first + group; row < last; row += groups) {
    float r[N], y[N], g[N], gr[N], gh[N];
    get<T, VEC, NV>(static_cast<const T*>(A.x) + row * A.sx, lane, lanes, A.C, r, 0.f);
    if constexpr (Y) {
      get<T, VEC, NV>(static_cast<const T*>(A.y) + row * A.sy, lane, lanes, A.C, y, 0.f);
      if (A.gate) get<T, VEC, NV>(static_cast<const T*>(A.gate) + row / A.gate_rows * A.sg, lane, lanes, A.C, g, 0.f);
    }
#pragma unroll
    for (int i = 0; i < N; i++) gr[i] = gh[i] = 0.f;
    if (A.gr) get<T, VEC, NV>(static_cast<const T*>(A.gr) + row * A.sgr, lane, lanes, A.C, gr, 0.f);
    if (A.gh) get<T, VEC, NV>(static_cast<const T*>(A.gh) + row * A.sgh, lane, lanes, A.C, gh, 0.f);
    float ry = 1.f, s[1], act[N], dact[N];
    if constexpr (Y) {
      if (A.wp) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) s[0] += y[i] * y[i];
        row_sum(s, W, lds);
        ry = 1.f / sqrtf(s[0] * inv + A.eps);
      }
#pragma unroll
      for (int i = 0; i < N; i++) {
        act[i] = dact[i] = 1.f;
        if (A.gate) act[i] = activate(A.act, g[i], &dact[i]);
        y[i] *= ry;
        r[i] += y[i] * wp[i] * sc[i] * act[i];
      }
    }
    float t[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; i++) t[0] += r[i] * r[i], t[1] += gh[i] * wq[i] * r[i];
    row_sum(t, W, lds);
    const float rr = 1.f / sqrtf(t[0] * inv + A.eps), mean = t[1] * rr * inv;
#pragma unroll
    for (int i = 0; i < N; i++) {
      r[i] *= rr;
      dwq[i] += gh[i] * r[i];
      gr[i] += rr * (gh[i] * wq[i] - r[i] * mean);
    }
    set<T, VEC, NV>(static_cast<T*>(A.dx) + row * A.C, lane, lanes, A.C, gr);
    if constexpr (Y) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float n = y[i] * wp[i];
        dsc[i] += gr[i] * act[i] * n;
        g[i] = gr[i] * sc[i] * n * dact[i];
        dgs[i] += g[i];
        gr[i] *= sc[i] * act[i];
      }
      if (A.gate && !shared_gate) set<T, VEC, NV>(static_cast<T*>(A.dgate) + row * A.C, lane, lanes, A.C, g);
      if (A.wp) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) {
          dwp[i] += gr[i] * y[i];
          gr[i] *= wp[i];
          s[0] += gr[i] * y[i];
        }
        row_sum(s, W, lds);
        const float my = s[0] * inv;
#pragma unroll
        for (int i = 0; i < N; i++) gr[i] = ry * (gr[i] - y[i] * my);
      }
      set<T, VEC, NV>(static_cast<T*>(A.dy) + row * A.C, lane, lanes, A.C, gr);
    }
  }
  const long long q = A.nparts * A.C;
  float* out = A.parts + part * A.C;
  put_part<VEC, NV>(out, lds, lane, lanes, A.C, group, groups, dwq);
  if constexpr (Y) {
    if (A.wp) put_part<VEC, NV>(out + q, lds, lane, lanes, A.C, group, groups, dwp);
    if (A.sc) put_part<VEC, NV>(out + 2 * q, lds, lane, lanes, A.C, group, groups, dsc);
    if (A.gate && shared_gate) put_part<VEC, NV>(out + 3 * q, lds, lane, lanes, A.C, group, groups, dgs);
  }
}

// out[block][c] = sum of `per` consecutive parts
template <class T>
__global__ __launch_bounds__(256) void sum_kernel(const float* parts, T* out, int C, int per) {
  __shared__ float lds[4][64];
  const int tiles = (C + 63) / 64, block = blockIdx.x / tiles;
  const int c = (blockIdx.x - block * tiles) * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6;
  const float* p = parts + (long long)block * per * C + c;
  float s = 0.f;
  if (c < C)
    for (int i = g; i < per; i += 4) s += p[(long long)i * C];
  lds[g][threadIdx.x & 63] = s;
  __syncthreads();
  if (g == 0 && c < C)
    ops::put(out + (long long)block * C + c,
             lds[0][threadIdx.x] + lds[1][threadIdx.x] + lds[2][threadIdx.x] + lds[3][threadIdx.x]);
}

}  // namespace bn
}  // namespace sffft
