// Linear attention with a decay for each head. Forward and all three gradients are one recurrence
// over a state X [K][V] with operands a, b (K channels) and c (V channels):
//
//   out_i = sum_{j <= i} g^(i-j) (a_i . b_j) c_j + g^(i+1) X0^T a_i        (REV: j >= i, g^(j-i))
//
//   o  : a = q,  b = k,  c = v            dv : a = k, b = q,  c = do, reversed in time
//   dq : a = do, b = v,  c = k, X = S^T   dk : a = v, b = do, c = q,  reversed, X = dS^T
#pragma once
#include "opsio.hpp"

namespace sffft {
namespace la {

// One operand: element strides of (batch, token, head); head h of the march reads head h / div.
struct Operand {
  const void* p;
  long long sb, st, sh;
  int div;
};

// One march: state element (kk, vv) of (b, h) is at s[(b * H + h) * K * V + kk * sk + vv * sv].
// The update adds w b c^T; the products with the entering state take x, those within the march p.
// Forward, the state enters before a token's own update (a_0 sees g X0); reversed, it holds all from the
// token on (the first one sees X0 undecayed, and the update includes the decay of the step).
struct March {
  Operand a, b, c;
  void* out;  // [B][T][H][V], in the operands' type, or fp32 if out_f32
  const float* s0;
  float* s1;
  int K, V, sk, sv;
  int rev, out_f32;
  float p, x, w;
};

struct Shape {
  int B, T, H;
  const float* log_decay;
  const int* lengths;
};

constexpr float LOG2E = 1.44269504088896340736f;

// log2 of the decay; -inf becomes a finite value whose powers are 0, so that the zeroth is 1
__device__ __forceinline__ float decay_log2(const float* log_decay, int h) { return fmaxf(log_decay[h] * LOG2E, -1e4f); }
__device__ __forceinline__ int valid_tokens(const Shape& s, int b) {
  return s.lengths ? min(max(s.lengths[b], 0), s.T) : s.T;
}

// The recurrence token by token: one wavefront holds 16 columns of the state, lane (r, c) the rows
// r, r + 4, ... of column c.
template <class T>
__global__ __launch_bounds__(64) void recur_kernel(March m, Shape s) {
  constexpr int ROWS = 32;
  const int tiles = (m.V + 15) / 16, bh = blockIdx.x / tiles, h = bh % s.H, b = bh / s.H;
  const int r = threadIdx.x >> 4, col = (blockIdx.x - bh * tiles) * 16 + (threadIdx.x & 15);
  const bool in = col < m.V;
  const float g = exp2f(decay_log2(s.log_decay, h));
  const int n = valid_tokens(s, b);
  const T* a = static_cast<const T*>(m.a.p) + b * m.a.sb + (h / m.a.div) * m.a.sh;
  const T* bb = static_cast<const T*>(m.b.p) + b * m.b.sb + (h / m.b.div) * m.b.sh;
  const T* c = static_cast<const T*>(m.c.p) + b * m.c.sb + (h / m.c.div) * m.c.sh;
  const long long at = (long long)bh * m.K * m.V + (long long)col * m.sv;
  float x[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const int kk = r + 4 * i;
    x[i] = in && kk < m.K && m.s0 ? m.s0[at + (long long)kk * m.sk] : 0.f;
  }
  for (int i = 0; i < s.T; i++) {
    const int t = m.rev ? s.T - 1 - i : i;
    float o = 0.f;
    if (t < n) {
      const float cv = in ? ops::to_f32(c[t * m.c.st + col]) : 0.f;
      // reversed, the state's own scale is in it already; what enters and what is added are equal there
      const float up = m.rev ? m.w : 1.f;
#pragma unroll
      for (int e = 0; e < ROWS; e++) {
        const int kk = r + 4 * e;
        if (kk < m.K) {
          if (!m.rev || t < n - 1) x[e] *= g;
          x[e] += up * ops::to_f32(bb[t * m.b.st + kk]) * cv;
          o += ops::to_f32(a[t * m.a.st + kk]) * x[e];
        }
      }
      o *= m.x;
    }
    o += __shfl_xor(o, 16);
    o += __shfl_xor(o, 32);
    if (in && r == 0) {
      const long long q = (((long long)b * s.T + t) * s.H + h) * m.V + col;
      if (m.out_f32) static_cast<float*>(m.out)[q] = o;
      else ops::put(static_cast<T*>(m.out) + q, o);
    }
  }
  if (m.s1)
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int kk = r + 4 * i;
      if (in && kk < m.K) m.s1[at + (long long)kk * m.sk] = m.rev && n ? x[i] * g : x[i];
    }
}

// Sum over the query heads that share a key/value head: out [rows][Hk][D] from in [rows][H][D].
template <class T>
__global__ __launch_bounds__(256) void head_sum_kernel(const float* in, T* out, long long n, int D, int G) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const long long head = i / D;
  const float* p = in + head * G * D + (i - head * D);
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int g = 0; g < G; g++) {
    float y[4];
    ops::load(p + (long long)g * D, y);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] += y[e];
  }
  ops::store(out + i, x);
}

// One token: lane (r, c) takes four columns c of rows r, r + 16, ... of the state.
template <class T>
__global__ __launch_bounds__(256) void step_kernel(Operand q, Operand k, Operand v, const float* log_decay,
                                                   float* state, int slots, const int* slot, T* o, int H, int Dk,
                                                   int Dv, float scale) {
  __shared__ float part[4][64];
  const int h = blockIdx.x % H, b = blockIdx.x / H, r = threadIdx.x >> 4, lc = (threadIdx.x & 15) * 4;
  const int col = blockIdx.y * 64 + lc;
  const int row = slot ? slot[b] : b;
  const bool live = row >= 0 && row < slots, in = col < Dv;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  if (live && in) {
    const float g = exp2f(fmaxf(log_decay[h] * LOG2E, -1e4f));
    const T* qp = static_cast<const T*>(q.p) + b * q.sb + (h / q.div) * q.sh;
    const T* kp = static_cast<const T*>(k.p) + b * k.sb + (h / k.div) * k.sh;
    const T* vp = static_cast<const T*>(v.p) + b * v.sb + (h / v.div) * v.sh;
    float* sp = state + ((long long)row * H + h) * Dk * Dv + col;
    float vv[4], x[8][4];
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (r + 16 * i < Dk) ops::load(sp + (long long)(r + 16 * i) * Dv, x[i]);
    ops::load(vp + col, vv);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int kk = r + 16 * i;
      if (kk < Dk) {
        const float kv = ops::to_f32(kp[kk]), qv = ops::to_f32(qp[kk]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[i][e] = g * x[i][e] + kv * vv[e];
          acc[e] += qv * x[i][e];
        }
        ops::store(sp + (long long)kk * Dv, x[i]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    acc[e] += __shfl_xor(acc[e], 16);
    acc[e] += __shfl_xor(acc[e], 32);
  }
  if ((threadIdx.x & 63) < 16) {
#pragma unroll
    for (int e = 0; e < 4; e++) part[threadIdx.x >> 6][lc + e] = acc[e];
  }
  __syncthreads();
  if (threadIdx.x < 16 && in) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = scale * (part[0][lc + e] + part[1][lc + e] + part[2][lc + e] + part[3][lc + e]);
    ops::store(o + ((long long)b * H + h) * Dv + col, y);
  }
}

}  // namespace la
}  // namespace sffft
