// Linear attention with a decay for each head. Forward and all three gradients are one recurrence
// over a state X [K][V] with operands a, b (K channels) and c (V channels):
//
//   out_i = sum_{j <= i} g^(i-j) (a_i . b_j) c_j + g^(i+1) X0^T a_i        (rev: j >= i, g^(j-i))
//
//   o  : a = q,  b = k,  c = v            dv : a = k, b = q,  c = do, reversed in time
//   dq : a = do, b = v,  c = k, X = S^T   dk : a = v, b = do, c = q,  reversed, X = dS^T
//
// A workgroup marches over the tokens of one head in chunks of 64 (fp32: 32) with the state in its
// registers. For a chunk of n tokens entered with X:
//   P_ij = g^(i-j) (a_i . b_j) for j <= i,   out = P c + g^(i+1) a X,   X' = g^n X + sum_j g^(n-1-j) b_j c_j^T
// all four products on MFMA; every decay is a power of g not above 1, so nothing overflows however fast a head
// forgets. Where the heads alone do not fill the chip the tokens are cut into segments: a first launch sums each
// segment's own state, and the march starts every segment with the decayed sums of those before it, which it joins
// itself or, where they are many, finds joined by a scan.
//
// Operands in 16 bits: bf16 inputs are exact. P and the entering state, operands of products that are rounded to bf16
// in the end, are split into two bf16 parts (17 bits: 2^-9 of that rounding), one product each; in one part each they
// made the outputs' error 2.3e-3 where their own rounding is 1.7e-3, and training 5 to 10% faster. The state is fp32 and
// so are the decayed c_j that are added to it: they are split into three bf16 parts (8 bits each, 24 together), into two
// where the state only serves outputs of 16 bits (three there: the same outputs, 1 to 8% slower). fp32 inputs are split
// so too, and every product of two split operands is the six partial products above 2^-24 (a bf16 product at 1240
// TFLOP/s, an fp32 one at 154).
//
// Measured (bf16, us): 131072 tokens, 12 heads of 128: 577, in a trace sums 177, scan 14 and march 389 at 4.2 TB/s,
// bound by memory (k and v are read twice); training, 8 x 2048 tokens, 12 heads of 64: 130, in a trace sums 13 and 18,
// march 29 forward and 76 for the gradients, whose time is the chain of a chunk's products and barriers with three
// workgroups on a CU; one token of 96 x 12 heads of 128: 26, 5.9 TB/s of states.
#pragma once
#include "opsio.hpp"

namespace sffft {
namespace la {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16;
typedef u16 u16x2 __attribute__((ext_vector_type(2)));

// One operand: element strides of (batch, token, head); head h of the march reads head h / div.
struct Operand {
  const void* p;
  long long sb, st, sh;
  int div;
};

// One march. A state of (b, h) is an array [K][V] with element strides sk, sv: the one it starts from at s0 + (b * H
// + h) * K * V, the sum of segment z alone at sums + ((b * H + h) * nseg + z) * K * V. A segment starts from s0,
// decayed, and the sums of those before it (from the last one on if reversed); where there are many a scan has put
// the entering states in the sums' place (scanned). s1 gets the state after the last segment. The update adds w b
// c^T; the products with the entering state take x, those within the march p. Forward, the state enters before a
// token's own update (a_0 sees g X0); reversed, it holds all from the token on (the first one sees X0 undecayed, and
// the update includes the decay of the step).
struct March {
  Operand a, b, c;
  void* out;  // [B][T][H][V]
  const float* s0;
  float *sums, *s1;
  int K, V, sk, sv;
  int rev;
  float p, x, w;
};

struct Shape {
  int B, T, H;
  const float* log_decay;
  const int* lengths;
};

// A launch: nm marches over B * H heads, nseg segments of seg tokens, vtiles tiles of the V channels. Sums are made of
// all segments, or of all but the last of a march (the first if reversed), whose sum nobody enters with: its
// own workgroups then leave the last state.
struct Launch {
  March m[3];
  Shape s;
  int nm, nseg, seg, vtiles, scanned, all;
};

constexpr float LOG2E = 1.44269504088896340736f;

// log2 of the decay; -inf becomes a finite value whose powers are 0. NaN stays (fmaxf would drop it).
__device__ __forceinline__ float decay_log2(const float* log_decay, int h) {
  const float x = log_decay[h] * LOG2E;
  return x < -1e4f ? -1e4f : x;
}
// the decay over n tokens: 1 over none, whatever it is; 0 for negative n
__device__ __forceinline__ float decay_power(float l2, int n) {
  return n < 0 ? 0.f : __builtin_amdgcn_exp2f(n == 0 ? 0.f : l2 * (float)n);
}
// The decay over n tokens for states that pass it many times over. Rounded to fp32 it would be off by the same part of
// itself each time, 8e-5 after 2048 chunks of a slow head; next() makes up in each factor for what the ones before it
// left out. (A head that forgets half of its state or more in n tokens keeps no such error.)
struct Decay {
  float hi, lo, inv;  // the decay is hi + lo
  __device__ __forceinline__ Decay(const float* log_decay, int h, int n) {
    float e = n == 0 ? 0.f : expm1f(log_decay[h] * (float)n);
    e = e > 3e38f ? 3e38f : e;
    const bool slow = e > -0.5f;
    const float g = slow ? 1.f + e : decay_power(decay_log2(log_decay, h), n);
    hi = uniform(g), lo = uniform(slow && e <= 1.f ? e - (g - 1.f) : 0.f), inv = uniform(slow ? 1.f / g : 0.f);
  }
  static __device__ __forceinline__ float uniform(float x) {
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
  }
  // the next factor; `behind`: by what part of it the product so far is too small
  __device__ __forceinline__ float next(float& behind) const {
    const float t = lo + hi * behind, g = hi + t;
    behind = (t - (g - hi)) * inv;
    return g;
  }
};
__device__ __forceinline__ int valid_tokens(const Shape& s, int b) {
  return s.lengths ? min(max(s.lengths[b], 0), s.T) : s.T;
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// x = h + m + l exactly, 8 bits each, truncated; two values to a dword of each plane
__device__ __forceinline__ void split2(float x, float y, uint32_t& h, uint32_t& m, uint32_t& l) {
  const uint32_t xh = __float_as_uint(x) & 0xffff0000u, yh = __float_as_uint(y) & 0xffff0000u;
  const float xr = x - __uint_as_float(xh), yr = y - __uint_as_float(yh);
  const uint32_t xm = __float_as_uint(xr) & 0xffff0000u, ym = __float_as_uint(yr) & 0xffff0000u;
  const float xl = xr - __uint_as_float(xm), yl = yr - __uint_as_float(ym);
  h = __builtin_amdgcn_perm(yh, xh, 0x07060302);
  m = __builtin_amdgcn_perm(ym, xm, 0x07060302);
  l = __builtin_amdgcn_perm(__float_as_uint(yl), __float_as_uint(xl), 0x07060302);
}

// x = h + m to 16 bits, each rounded
__device__ __forceinline__ void split2(float x, float y, uint32_t& h, uint32_t& m) {
  h = ops::pack_bf16(x, y);
  m = ops::pack_bf16(x - __uint_as_float(h << 16), y - __uint_as_float(h & 0xffff0000u));
}

// NS planes of one operand fragment
template <int NS>
struct Frag {
  bf16x8 p[NS];
};
// d += a b, the products of planes that are not below the last one's bits
template <int NA, int NB>
__device__ __forceinline__ void product(const Frag<NA>& a, const Frag<NB>& b, f32x4& d) {
  constexpr int LAST = (NA > NB ? NA : NB) - 1;
#pragma unroll
  for (int s = LAST; s >= 0; s--)
#pragma unroll
    for (int i = 0; i < NA; i++)
      if (s - i >= 0 && s - i < NB) d = mfma(a.p[i], b.p[s - i], d);
}
// the same for several accumulators at once: products that follow each other do not wait for each other
template <int NA, int NB, int N, class FA, class FB, class FD>
__device__ __forceinline__ void products(FA a, FB b, FD d) {
  constexpr int LAST = (NA > NB ? NA : NB) - 1;
#pragma unroll
  for (int s = LAST; s >= 0; s--)
#pragma unroll
    for (int i = 0; i < NA; i++)
      if (s - i >= 0 && s - i < NB)
#pragma unroll
        for (int n = 0; n < N; n++) d(n) = mfma(a(n).p[i], b(n).p[s - i], d(n));
}
template <int NS>
__device__ __forceinline__ Frag<NS> split8(const float (&x)[8]) {
  Frag<NS> f;
  if constexpr (NS == 1) {
    const uint4 v = make_uint4(ops::pack_bf16(x[0], x[1]), ops::pack_bf16(x[2], x[3]), ops::pack_bf16(x[4], x[5]),
                               ops::pack_bf16(x[6], x[7]));
    f.p[0] = __builtin_bit_cast(bf16x8, v);
  } else if constexpr (NS == 2) {
    uint32_t h[4], m[4];
#pragma unroll
    for (int i = 0; i < 4; i++) split2(x[2 * i], x[2 * i + 1], h[i], m[i]);
    f.p[0] = __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
    f.p[1] = __builtin_bit_cast(bf16x8, make_uint4(m[0], m[1], m[2], m[3]));
  } else {
    uint32_t h[4], m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) split2(x[2 * i], x[2 * i + 1], h[i], m[i], l[i]);
    f.p[0] = __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
    f.p[1] = __builtin_bit_cast(bf16x8, make_uint4(m[0], m[1], m[2], m[3]));
    f.p[2] = __builtin_bit_cast(bf16x8, make_uint4(l[0], l[1], l[2], l[3]));
  }
  return f;
}

// Row-major [C][L] tiles of 16 bits in LDS, NS planes. Rows are padded by 32 bytes: the transposing reads below touch
// 8 rows of 32 bytes at a time, on 64 different banks. SWAP: in rows 8..15 of each 16 neighbouring pieces of 16 bytes
// change places, so that reads of a piece of 16 rows find 64 different banks too (the 8 rows' starts are 8 banks
// apart).
template <int NS, int C, int L, bool SWAP = true>
struct Tile {
  u16 v[NS][C][L];
  static __device__ __forceinline__ int at(int row, int col) { return SWAP ? col ^ (row & 8) : col; }

  // operand whose index is the row: lane (g, i) holds channels at..at+7 of row r0 + i, at = c0 + 8 g
  __device__ __forceinline__ bf16x8 plane(int p, int r0, int c0, int i, int g) const {
    return *reinterpret_cast<const bf16x8*>(&v[p][r0 + i][c0 + at(i, 8 * g)]);
  }
  __device__ __forceinline__ Frag<NS> rows(int r0, int c0, int i, int g) const {
    Frag<NS> f;
#pragma unroll
    for (int p = 0; p < NS; p++) f.p[p] = plane(p, r0, c0, i, g);
    return f;
  }
  // the same with the channels in the order of an accumulator's rows: c0 + 4 g .. + 3 and c0 + 16 + 4 g .. + 3
  __device__ __forceinline__ Frag<NS> rows_acc(int r0, int c0, int i, int g) const {
    Frag<NS> f;
#pragma unroll
    for (int p = 0; p < NS; p++) {
      const uint2 a = *reinterpret_cast<const uint2*>(&v[p][r0 + i][c0 + at(i, 4 * g)]);
      const uint2 b = *reinterpret_cast<const uint2*>(&v[p][r0 + i][c0 + 16 + at(i, 4 * g)]);
      f.p[p] = __builtin_bit_cast(bf16x8, make_uint4(a.x, a.y, b.x, b.y));
    }
    return f;
  }
  // operand whose index is the channel: lane (g, i) holds rows r0 + 4 g .. + 3 and r0 + 16 + 4 g .. + 3 of
  // channel c0 + i. A transposing read takes 4 rows of 16 channels for each 16 lanes: lane i points at
  // row i / 4, channels 4 (i % 4).., and receives channel i of the four rows.
  __device__ __forceinline__ Frag<NS> cols(int r0, int c0, int i, int g) const {
    Frag<NS> f;
#pragma unroll
    for (int p = 0; p < NS; p++) {
      const u16* q = &v[p][r0 + 4 * g + (i >> 2)][c0 + at(4 * g, 4 * (i & 3))];
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)q);
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(q + 16 * L));
      const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
      f.p[p] = __builtin_bit_cast(bf16x8, make_uint4(x.x, x.y, y.x, y.y));
    }
    return f;
  }
};

// A 16-byte store. Its whole offset is the lane's: with a scalar register for a part of it the compiler leaves out the
// wait between the store and the next write to its data registers, and where workgroups shared a CU the
// store then sent what was written after it.
__device__ __forceinline__ void store16(i32x4 x, __amdgpu_buffer_rsrc_t r, uint32_t at) {
  __builtin_amdgcn_raw_buffer_store_b128(x, r, at, 0, 0);
}

// A chunk's rows of one operand on their way from memory to LDS: 16 bytes a piece, rows from n on and channels
// from D on are zero and not read: their lanes' offsets lie beyond the buffer's records. One lane offset serves
// every piece, the rest is in scalar registers.
template <class T, int C, int DT>
struct Stage {
  static constexpr int E = 16 / sizeof(T), PER = DT / E, N = C * PER / 256, ROWS = 256 / PER;
  static constexpr uint32_t RECORDS = 0x7fffffffu, OUTSIDE = 0x80000000u;
  i32x4 v[N];
  // The lane's row among ROWS. Rows of 128 bytes are written two at a time: 4 apart they lie on different banks.
  static __device__ __forceinline__ int row() {
    const int r = threadIdx.x / PER;
    return PER * sizeof(T) * E == 128 && sizeof(T) == 2 ? (r & ~7) | (r & 1) << 2 | (r & 6) >> 1 : r;
  }
  static __device__ __forceinline__ int col() { return threadIdx.x % PER * E; }
  __device__ __forceinline__ void load(const T* p, long long st, int n, int D) {
    const int row = this->row(), col = this->col();
    const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, RECORDS, 0x00027000);
    const uint32_t at = col < D ? (uint32_t)(row * (int)st + col) * sizeof(T) : OUTSIDE;
#pragma unroll
    for (int i = 0; i < N; i++)
      v[i] = __builtin_amdgcn_raw_buffer_load_b128(r, row + i * ROWS < n ? at : OUTSIDE, i * ROWS * (int)st * (int)sizeof(T), 0);
  }
  // whether no value is an infinity or NaN
  __device__ __forceinline__ bool finite() const {
    u16x2 top = {0, 0};
    uint32_t top32 = 0;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if constexpr (sizeof(T) == 2) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[i][k] & 0x7fff7fff));
        else top32 = max(top32, (uint32_t)v[i][k] & 0x7fffffffu);
      }
    return sizeof(T) == 2 ? top.x < 0x7f80 && top.y < 0x7f80 : top32 < 0x7f800000u;
  }
  // (tiles of 96 channels are fetched by the lanes of 128)
  template <int NS, int L>
  __device__ __forceinline__ void store(Tile<NS, C, L>& t) const {
    constexpr int W = L - 16;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int row = this->row() + i * ROWS, col = t.at(row, this->col());
      if (DT > W && this->col() >= W) break;
      if constexpr (NS == 1) {
        *reinterpret_cast<i32x4*>(&t.v[0][row][col]) = v[i];
      } else {
        uint2 h, m, l;
        split2(__int_as_float(v[i].x), __int_as_float(v[i].y), h.x, m.x, l.x);
        split2(__int_as_float(v[i].z), __int_as_float(v[i].w), h.y, m.y, l.y);
        *reinterpret_cast<uint2*>(&t.v[0][row][col]) = h;
        *reinterpret_cast<uint2*>(&t.v[1][row][col]) = m;
        *reinterpret_cast<uint2*>(&t.v[2][row][col]) = l;
      }
    }
  }
};

template <class T>
constexpr int chunk_of() { return sizeof(T) == 4 ? 32 : 64; }

// Four wavefronts; wavefront w holds the columns vv = v0 + w VT/4 .. of the state, in the layout of an
// accumulator (row kk = 16 a + 4 g + r, column lane % 16), which is an operand's too when the other operand
// takes the same order of channels (rows_acc). With !OUT only the state is made. UP: the planes of what is
// added to the state; 2 where it only serves outputs of 16 bits. TO: the output's type (fp32 for parts that are
// summed).
//
// The next chunk is fetched a chunk ahead, and a chunk's outputs leave at the start of the next, before that
// fetch: the wait for it then finds them gone.
template <class T, class TO, int KT, int VT, bool OUT, int UP>
__global__ __launch_bounds__(256, KT <= 64 && VT == 64 ? 3 : 2) void march_kernel(Launch L) {
  constexpr int NS = sizeof(T) == 4 ? 3 : 1, PX = sizeof(T) == 4 ? 3 : 2, C = chunk_of<T>(), MT = C / 16, JS = C / 32, KS = KT / 32, KA = KT / 16;
  constexpr int VW = VT / 64, TILES = MT * (MT + 1) / 2, NP = (TILES + 3) / 4;  // P's tiles, and those of a wavefront (some twice)
  constexpr int E = sizeof(TO);
  constexpr int LK = KT == 96 ? 128 : KT;  // lanes that fetch K channels take these
  // outputs leave through a's tile (below)
  constexpr bool VIA = OUT && NS == 1 && E == 2 && LK == VT;
  struct Tiles {
    Tile<NS, OUT ? C : 1, (VIA ? VT : KT) + 16> a;
    Tile<NS, C, KT + 16> b;
    Tile<NS, C, VT + 16> c;
    Tile<PX, OUT ? C : 1, C + 8, false> p;  // PX: planes of P and X
  };
  __shared__ __attribute__((aligned(16))) Tiles tiles;
  auto& ta = tiles.a;
  auto& tb = tiles.b;
  auto& tc = tiles.c;
  auto& tp = tiles.p;
  __shared__ int odd[2];  // whether this chunk, or the next, has infinities or NaN
  __shared__ __attribute__((aligned(16))) float fi[C], wj[C];  // decays: of the entering state at row i, of token j in the update

  // Workgroups go to the 8 XCDs in turn; the marches and V tiles of one head and segment, which read the same
  // operands, follow each other on one of them.
  const int per = L.nm * L.vtiles, y = blockIdx.x >> 3;
  const int unit = y / per * 8 + (blockIdx.x & 7), sub = y % per;
  const int segments = OUT || L.all ? L.nseg : L.nseg - 1;
  if (unit >= L.s.B * L.s.H * segments) return;
  const March m = L.m[sub / L.vtiles];
  const int v0 = sub % L.vtiles * VT;
  if (v0 >= m.V) return;
  const int h = unit % L.s.H, zb = unit / L.s.H, b = zb / segments, z = zb % segments + (!OUT && !L.all && m.rev);
  const long long bh = (long long)b * L.s.H + h;
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool rev = m.rev;
  const int first = z * L.seg, last = first + min(L.seg, L.s.T - first), chunks = (last - first + C - 1) / C;
  const int end = min(valid_tokens(L.s, b), last);  // of the tokens that count
  const float l2 = decay_log2(L.s.log_decay, h);
  auto power = [&](int n) { return decay_power(l2, n); };
  auto count = [&](int t0) { return __builtin_amdgcn_readfirstlane(min(max(end - t0, 0), C)); };

  // The first chunk: the last one of the segment if reversed. The sums go the other way, so that what they read last
  // is what the march reads first, out of the cache that all XCDs share.
  const bool back = OUT ? rev : !rev;
  const int dir = back ? -C : C;
  int t0 = back ? first + (chunks - 1) * C : first;
  auto token = [&](const Operand& x, int t) { return static_cast<const T*>(x.p) + b * x.sb + (h / x.div) * x.sh + t * x.st; };
  const T *pa = token(m.a, t0), *pb = token(m.b, t0), *pc = token(m.c, t0) + v0;
  const int orow = L.s.H * m.V;
  TO* po = OUT ? static_cast<TO*>(m.out) + (((long long)b * L.s.T + t0) * L.s.H + h) * m.V : nullptr;

  Stage<T, C, LK> ga, gb;
  Stage<T, C, VT> gc;
  auto fetch = [&](int n) {
    if constexpr (OUT) ga.load(pa, m.a.st, n, m.K);
    gb.load(pb, m.b.st, n, m.K);
    gc.load(pc, m.c.st, n, m.V - v0);
    pa += dir * m.a.st, pb += dir * m.b.st, pc += dir * m.c.st;
  };
  int n = count(t0);
  fetch(n);

  // the wavefront's tiles of P: (row tile, column tile), and their decays
  int pi[NP], pj[NP];
  float pd[NP][4];
  if constexpr (OUT) {
#pragma unroll
    for (int t = 0; t < NP; t++) {
      const int idx = min(w + 4 * t, TILES - 1);
      int r = 0;
      while ((r + 1) * (r + 2) / 2 <= idx) r++;
      const int c = idx - r * (r + 1) / 2;
      pi[t] = __builtin_amdgcn_readfirstlane(rev ? c : r), pj[t] = __builtin_amdgcn_readfirstlane(rev ? r : c);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int d = 16 * pi[t] + i16 - (16 * pj[t] + 4 * g + e);
        pd[t][e] = m.p * power(rev ? -d : d);
      }
    }
    // tiles on the other side of the diagonal stay zero
    for (int i = threadIdx.x; i < (int)sizeof(tp) / 16; i += 256) reinterpret_cast<uint4*>(&tp)[i] = make_uint4(0, 0, 0, 0);
  }

  f32x4 S[KA][VW];
  const int kv = m.K * m.V, sv0 = v0 + 16 * w * VW + i16;
  const uint32_t sat = (uint32_t)(4 * g * m.sk + sv0 * m.sv) * 4;
  // f(tile, lane offset, scalar offset) for the tiles of a state; the lanes outside it get an offset outside
  auto state_tiles = [&](auto f) {
#pragma unroll
    for (int a = 0; a < KA; a++)
#pragma unroll
      for (int v = 0; v < VW; v++) {
        const bool in = (16 * a + 4 * g < m.K) & (sv0 + 16 * v < m.V);
        f(a, v, in ? sat : 0x80000000u, (16 * a * m.sk + 16 * v * m.sv) * 4);
      }
  };
  auto load_state = [&](const float* p, f32x4(&x)[KA][VW]) {
    const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p), 0, 0x7fffffff, 0x00027000);
    if (m.sk == 1)  // rows kk next to each other
      state_tiles([&](int a, int v, uint32_t at, int off) {
        x[a][v] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, off, 0));
      });
    else
      state_tiles([&](int a, int v, uint32_t at, int off) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[a][v][e] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, at, off + e * m.sk * 4, 0));
      });
  };
  auto store_state = [&](float* p, const f32x4(&x)[KA][VW]) {
    const auto r = __builtin_amdgcn_make_buffer_rsrc(p, 0, 0x7fffffff, 0x00027000);
    state_tiles([&](int a, int v, uint32_t at, int off) {
#pragma unroll
      for (int e = 0; e < 4; e++) __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(x[a][v][e]), r, at, off + e * m.sk * 4, 0);
    });
  };
#pragma unroll
  for (int a = 0; a < KA; a++)
#pragma unroll
    for (int v = 0; v < VW; v++) S[a][v] = f32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (OUT) {
    const float* sums = m.sums + bh * L.nseg * kv;
    if (L.scanned) {
      load_state(sums + (long long)z * kv, S);
    } else {
      if (m.s0) load_state(m.s0 + bh * kv, S);
      const int total = valid_tokens(L.s, b);
      auto join = [&](int y, f32x4(&x)[KA][VW]) {
        f32x4 u[KA][VW];
        load_state(sums + (long long)y * kv, u);
        const float d = power(min(max(total - y * L.seg, 0), L.seg));
#pragma unroll
        for (int a = 0; a < KA; a++)
#pragma unroll
          for (int v = 0; v < VW; v++) x[a][v] = S[a][v] * d + u[a][v];
      };
      for (int y = rev ? L.nseg - 1 : 0; y != z; y += rev ? -1 : 1) join(y, S);
      if (L.all && m.s1 && z == (rev ? 0 : L.nseg - 1)) {  // the last state
        f32x4 x[KA][VW];
        join(z, x);
        store_state(m.s1 + bh * kv, x);
      }
    }
  }

  // A chunk's outputs, transposed: rows vv, columns i. Where a's tile has their size they go through it, dead
  // by then, so that whole rows leave together (a store of 4 channels in each of 16 rows takes the
  // address unit 64 cycles, of 8 whole rows 16), each lane from the pieces that it will overwrite with the
  // next chunk's a; rows from `left` on are not written.
  f32x4 o[MT][VW] = {};
  int left = 0;
  auto stage_out = [&]() {
    if constexpr (VIA)
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int v = 0; v < VW; v++)
          *reinterpret_cast<uint2*>(&ta.v[0][16 * t + i16][16 * (w * VW + v) + ta.at(i16, 4 * g)]) =
              make_uint2(ops::pack_bf16(o[t][v][0], o[t][v][1]), ops::pack_bf16(o[t][v][2], o[t][v][3]));
  };
  auto store_out = [&]() {
    if constexpr (VIA) {
      typedef Stage<T, C, VT> G;
      const auto r = __builtin_amdgcn_make_buffer_rsrc(po + v0, 0, 0x7fffffff, 0x00027000);
      const int row = G::row(), col = G::col();
      const uint32_t at = v0 + col < m.V ? (uint32_t)(row * orow + col) * E : 0x80000000u;
#pragma unroll
      for (int i = 0; i < G::N; i++) {
        const i32x4 x = *reinterpret_cast<const i32x4*>(&ta.v[0][row + i * G::ROWS][ta.at(row + i * G::ROWS, col)]);
        store16(x, r, row + i * G::ROWS < left ? at + i * G::ROWS * orow * E : 0x80000000u);
      }
    } else {
      const auto r = __builtin_amdgcn_make_buffer_rsrc(po, 0, 0x7fffffff, 0x00027000);
      const int ovv = v0 + 16 * w * VW + 4 * g;
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int v = 0; v < VW; v++) {
          const bool in = (16 * t + i16 < left) & (ovv + 16 * v < m.V);
          const uint32_t to = in ? (uint32_t)(i16 * orow + ovv) * E : 0x80000000u;
          const int off = 16 * (t * orow + v) * E;
          if constexpr (E == 2) {
            const i32x2 x = {(int)ops::pack_bf16(o[t][v][0], o[t][v][1]), (int)ops::pack_bf16(o[t][v][2], o[t][v][3])};
            __builtin_amdgcn_raw_buffer_store_b64(x, r, to, off, 0);
          } else {
            store16(__builtin_bit_cast(i32x4, o[t][v]), r, in ? to + off : to);
          }
        }
    }
  };

  // A chunk token by token, straight from memory: where a product is infinite or NaN the tiles of P that are 0 would
  // carry it to tokens that must not see it. (Looking for such values takes 1 to 3% of a training step.) `from`: the
  // chunk's first token, of which `count` count; rows: those of the output. The state goes through LDS, 16 columns
  // of a wavefront at a time, where the tiles of a, b and c are dead (P's keep their zeros), so that no register is
  // held for this.
  auto by_token = [&](int from, int count, int rows) {
    static_assert(!OUT || sizeof(tiles) - sizeof(tp) >= KT * 64 * sizeof(float), "");
    float* X = reinterpret_cast<float*>(&tiles) + w * KT * 16 + i16;  // row kk of the wavefront's 16 columns at X + 16 kk
    const float decay = power(1), before = rev ? 1.f : decay, after = rev ? decay : 1.f;
#pragma unroll
    for (int v = 0; v < VW; v++) {
#pragma unroll
      for (int a = 0; a < KA; a++)
#pragma unroll
        for (int e = 0; e < 4; e++) X[(16 * a + 4 * g + e) * 16] = S[a][v][e];
      const int vv = sv0 + 16 * v;
      const T *ra = token(m.a, from), *rb = token(m.b, from), *rc = token(m.c, from) + vv;
#pragma unroll 1
      for (int s = 0; s < rows; s++) {
        const int i = rev && s < count ? count - 1 - s : s;
        const float c = s < count && vv < m.V ? m.w * ops::to_f32(rc[i * m.c.st]) : 0.f;
        float sum = 0.f;
#pragma unroll 1
        for (int k = s < count ? 4 * g : m.K; k < m.K; k += 16) {
          const T *a = ra + i * m.a.st + k, *b = rb + i * m.b.st + k;
#pragma unroll 2
          for (int e = 0; e < 4; e++) {
            float& x = X[(k + e) * 16];
            const float y = x * before + ops::to_f32(b[e]) * c;
            sum += ops::to_f32(a[e]) * y;
            x = y * after;
          }
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (g == 0 && vv < m.V) ops::put(po + (long long)i * orow + vv, m.x * sum);
      }
#pragma unroll
      for (int a = 0; a < KA; a++)
#pragma unroll
        for (int e = 0; e < 4; e++) S[a][v][e] = X[(16 * a + 4 * g + e) * 16];
    }
  };

  if (threadIdx.x == 0) odd[0] = 0;
  Decay gn(L.s.log_decay, h, 0);
  float behind = 0.f;
  int have = OUT ? -1 : 0;  // tokens of the chunk that the decays are for; of the chunks before
  for (int c = 0; c < chunks; c++) {
    ops::barrier();
    if constexpr (OUT) {  // the last chunk's
      store_out();
      if (c) po += (long long)dir * orow;
      left = last - t0;
      ga.store(ta);
    }
    gb.store(tb);
    gc.store(tc);
    if constexpr (OUT)
      if (!gc.finite()) odd[c & 1] = 1;
    // The decays depend on the tokens in a chunk; in the sums also on those between the chunk and where the sum is
    // taken.
    if (!OUT || n != have) {
      const int i = threadIdx.x, behind = OUT ? 0 : have;
      if (i < C) {
        if constexpr (OUT) fi[i] = m.x * power(rev ? n - 1 - i : i + 1);
        wj[i] = m.w * power(i >= n ? -1 : behind + (rev ? i + 1 : n - 1 - i));
      }
      if constexpr (OUT) have = n, gn = Decay(L.s.log_decay, h, n);
      else have += n;
    }
    t0 += dir;
    n = c + 1 < chunks ? count(t0) : 0;  // past the last chunk nothing is valid, and nothing is read
    fetch(n);
    ops::barrier();

    if constexpr (OUT) {
      if (threadIdx.x == 0) odd[~c & 1] = 0;
      bool finite = true;  // so are a and b if their products with tokens of their own are
      // P^T tiles: rows j, columns i
#pragma unroll
      for (int t = 0; t < NP; t++) {
        Frag<NS> fb[KS], fa[KS];
#pragma unroll
        for (int k = 0; k < KS; k++) fb[k] = tb.rows(16 * pj[t], 32 * k, i16, g), fa[k] = ta.rows(16 * pi[t], 32 * k, i16, g);
        f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; k++) product(fb[k], fa[k], d);
        // stored in the order of the transposing reads' rows: 16 * (j / 16 % 2) + 4 g + e at 8 g + 4 (j / 16 % 2) + e
        u16* q = &tp.v[0][16 * pi[t] + i16][32 * (pj[t] >> 1) + 8 * g + 4 * (pj[t] & 1)];
        const float x0 = d[0] * pd[t][0], x1 = d[1] * pd[t][1], x2 = d[2] * pd[t][2], x3 = d[3] * pd[t][3];
        finite = finite && __builtin_isfinite(x0) && __builtin_isfinite(x1) && __builtin_isfinite(x2) && __builtin_isfinite(x3);
        if constexpr (PX == 2) {
          uint2 hh, mm;
          split2(x0, x1, hh.x, mm.x);
          split2(x2, x3, hh.y, mm.y);
          *reinterpret_cast<uint2*>(q) = hh;
          *reinterpret_cast<uint2*>(q + C * (C + 8)) = mm;
        } else {
          uint2 hh, mm, ll;
          split2(x0, x1, hh.x, mm.x, ll.x);
          split2(x2, x3, hh.y, mm.y, ll.y);
          *reinterpret_cast<uint2*>(q) = hh;
          *reinterpret_cast<uint2*>(q + C * (C + 8)) = mm;
          *reinterpret_cast<uint2*>(q + 2 * C * (C + 8)) = ll;
        }
      }
      if (!finite) odd[c & 1] = 1;
      // a X, transposed: rows vv, columns i
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int v = 0; v < VW; v++) o[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; k++) {
        Frag<PX> fs[VW];
        Frag<NS> fa[MT];
#pragma unroll
        for (int t = 0; t < MT; t++) fa[t] = ta.rows_acc(16 * t, 32 * k, i16, g);
#pragma unroll
        for (int v = 0; v < VW; v++) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = S[2 * k + (e >> 2)][v][e & 3];
          fs[v] = split8<PX>(x);
        }
        products<PX, NS, MT * VW>([&](int n) -> auto& { return fs[n % VW]; }, [&](int n) -> auto& { return fa[n / VW]; },
                                  [&](int n) -> auto& { return o[n / VW][n % VW]; });
      }
#pragma unroll
      for (int t = 0; t < MT; t++) {
        const float f = fi[16 * t + i16];
#pragma unroll
        for (int v = 0; v < VW; v++) o[t][v] *= f;
      }
      ops::barrier();
      if (__builtin_amdgcn_readfirstlane(odd[c & 1])) {
        by_token(t0 - dir, have, min(left, C));
        left = 0;  // the outputs have left
        continue;
      }
    }

    if constexpr (OUT) {
      const float f = gn.next(behind);
#pragma unroll
      for (int a = 0; a < KA; a++)
#pragma unroll
        for (int v = 0; v < VW; v++) S[a][v] *= f;
    }
#pragma unroll
    for (int s = 0; s < JS; s++) {
      // c's channels as an operand, tokens along the sum; and decayed, to be added to the state
      Frag<NS> fc[VW];
      Frag<UP> fw[VW];
      const f32x4 w0 = *reinterpret_cast<const f32x4*>(&wj[32 * s + 4 * g]), w1 = *reinterpret_cast<const f32x4*>(&wj[32 * s + 16 + 4 * g]);
#pragma unroll
      for (int v = 0; v < VW; v++) {
        fc[v] = tc.cols(32 * s, 16 * (w * VW + v), i16, g);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          x[e] = (float)fc[v].p[NS - 1][e];
#pragma unroll
          for (int p = NS - 2; p >= 0; p--) x[e] += (float)fc[v].p[p][e];
          x[e] *= e < 4 ? w0[e & 3] : w1[e & 3];
        }
        fw[v] = split8<UP>(x);
      }
      if constexpr (OUT) {
        // the zero tiles too: their two products cost less than branches. Where there is one plane of c, P's come one
        // by one, for their registers.
        constexpr int AT_ONCE = NS == 1 ? 1 : PX;
#pragma unroll
        for (int p = PX - AT_ONCE; p >= 0; p -= AT_ONCE) {
          Frag<AT_ONCE> fp[MT];
#pragma unroll
          for (int t = 0; t < MT; t++)
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) fp[t].p[k] = tp.plane(p + k, 16 * t, 32 * s, i16, g);
          products<NS, AT_ONCE, MT * VW>([&](int n) -> auto& { return fc[n % VW]; }, [&](int n) -> auto& { return fp[n / VW]; },
                                         [&](int n) -> auto& { return o[n / VW][n % VW]; });
        }
      }
      constexpr int HALF = 2;
#pragma unroll
      for (int a = 0; a < KA; a += HALF) {
        Frag<NS> fb[HALF];
#pragma unroll
        for (int i = 0; i < HALF; i++) fb[i] = tb.cols(32 * s, 16 * (a + i), i16, g);
        products<NS, UP, HALF * VW>([&](int n) -> auto& { return fb[n / VW]; }, [&](int n) -> auto& { return fw[n % VW]; },
                                    [&](int n) -> auto& { return S[a + n / VW][n % VW]; });
      }
    }
    if constexpr (OUT) {
      // Tokens that do not count give 0, whatever the state holds: their rows of a are 0, but 0 times an infinity is not.
      if (have < C) {
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int v = 0; v < VW; v++)
            if (16 * t + i16 >= have) o[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      stage_out();
    }
  }
  if constexpr (OUT) {
    if constexpr (VIA) ops::barrier();
    store_out();
  }

  if constexpr (!OUT) store_state(m.sums + (bh * L.nseg + z) * kv, S);
  else if (!L.all && m.s1 && z == (rev ? 0 : L.nseg - 1)) store_state(m.s1 + bh * kv, S);
}

// The states that enter the segments, from the sums of those before them, in place. Lane: four elements. Sixteen
// segments are read ahead. Bound by memory: 42 segments of 12 states of 128 x 128, 67 MB, in 14 us.
struct Scan {
  float* sums;  // [bh][nseg][n]
  const float* s0;
  float* s1;  // the last state
  int n, rev;
};
struct ScanLaunch {
  Scan c[2];
  Shape s;
  int nseg, seg;
};
__global__ __launch_bounds__(256) void scan_kernel(ScanLaunch L) {
  const Scan& c = L.c[blockIdx.y];
  const int tiles = (c.n + 1023) / 1024, bh = blockIdx.x / tiles, e = ((blockIdx.x - bh * tiles) * 256 + threadIdx.x) * 4;
  if (e >= c.n) return;
  const int h = bh % L.s.H, b = bh / L.s.H, valid = valid_tokens(L.s, b);
  // of a whole segment, and of the one that the sequence ends in
  const Decay whole(L.s.log_decay, h, L.seg), part(L.s.log_decay, h, valid % L.seg);
  float behind = 0.f;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (c.s0) ops::load(c.s0 + (long long)bh * c.n + e, x);
  float* p = c.sums + (long long)bh * L.nseg * c.n + e;
  constexpr int AHEAD = 16;
  for (int z0 = 0; z0 < L.nseg; z0 += AHEAD) {
    float u[AHEAD][4];
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (z0 + i < L.nseg) ops::load(p + (long long)(c.rev ? L.nseg - 1 - z0 - i : z0 + i) * c.n, u[i]);
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (z0 + i < L.nseg) {
        const int z = c.rev ? L.nseg - 1 - z0 - i : z0 + i;
        const int n = min(max(valid - z * L.seg, 0), L.seg);
        const float d = n == L.seg ? whole.next(behind) : n ? part.hi : 1.f;
        ops::store(p + (long long)z * c.n, x);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = x[k] * d + u[i][k];
      }
  }
  if (c.s1) ops::store(c.s1 + (long long)bh * c.n + e, x);
}

// Sums over the query heads that share a key/value head, of dk and of dv: out [rows][Hk][D] from in [rows][H][D].
// Bound by memory: 47 MB in 8 us. (Adding in the march itself would need an order among its workgroups, or atomics
// without one.)
struct HeadSum {
  const float* in;
  void* out;
  long long n;
  int D;
};
struct HeadSums {
  HeadSum s[2];
  int G;
  unsigned blocks;  // workgroups of the first
};
template <class T>
__global__ __launch_bounds__(256) void head_sum_kernel(HeadSums L) {
  const bool second = blockIdx.x >= L.blocks;
  const HeadSum& A = L.s[second];
  const int D = A.D, G = L.G;
  const long long i = ((long long)(blockIdx.x - (second ? L.blocks : 0)) * 256 + threadIdx.x) * 4;
  if (i >= A.n) return;
  const long long head = i / D;
  const float* p = A.in + head * G * D + (i - head * D);
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int g = 0; g < G; g++) {
    float y[4];
    ops::load(p + (long long)g * D, y);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] += y[e];
  }
  ops::store(static_cast<T*>(A.out) + i, x);
}

// One token: S' = g S + k v^T, o = scale S'^T q. Bound by memory, the state's reading and writing: 96 sequences of 12
// heads of 128 channels take 26 us, 152 MB at 5.9 TB/s (small ones the launch, 4 us). A workgroup takes 64 columns of
// a state, lane (r, c) four of them in rows r, r + 16, ..: all its loads of 16 bytes, up to eight, are on their way
// before the first is used.
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
    const Decay g(log_decay, h, 1);  // in two parts: calls that follow each other would add up the rounding of one
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
          x[i][e] = __builtin_fmaf(g.hi, x[i][e], __builtin_fmaf(g.lo, x[i][e], kv * vv[e]));
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
  ops::barrier();
  if (threadIdx.x < 16 && in) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = scale * (part[0][lc + e] + part[1][lc + e] + part[2][lc + e] + part[3][lc + e]);
    ops::store(o + ((long long)b * H + h) * Dv + col, y);
  }
}

}  // namespace la
}  // namespace sffft
