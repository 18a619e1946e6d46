// Launches and C ABI of the rotary positions (rotary.hpp) and of the norms around a block
// (blocknorm.hpp), and the error text of the library.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <initializer_list>

#include "blocknorm.hpp"
#include "ops_status.hpp"
#include "rotary.hpp"

namespace sffft {
namespace ops {

thread_local char g_last_error[256] = "";

int hip_status(hipError_t err, const char* what) {
  if (err == hipSuccess) return SFFFT_OK;
  snprintf(g_last_error, sizeof(g_last_error), "%s: %s (%d)", what, hipGetErrorString(err), (int)err);
  return SFFFT_EHIP;
}

}  // namespace ops

namespace {

// ---- rotary ----

// Vectors of 16 bytes where everything is aligned to them, else channel by channel (the two workloads of rotary.hpp:
// 137 us against 277, 59 against 148 for two calls). About one unit for each of a workgroup's 256 lanes.
bool rotary_grid(rot::Args& a, int elem, bool interleaved, bool wide) {
  const int V = 16 / elem, pp = !wide ? 1 : interleaved ? V / 2 : V;
  a.units = a.D / (2 * pp), a.per = a.heads * a.units;
  const auto inverse = [](unsigned d) { return (unsigned)((((unsigned long long)1 << 32) + d - 1) / d); };
  a.by_units = inverse(a.units), a.by_per = inverse(a.per);
  // more than one where so many tokens need a launch of 2^32 lanes otherwise; a workgroup's units are divided by
  // `per` in 32 bits
  const unsigned most = (1u << 24) - 1;
  a.wg_tokens = std::max({1u, 256u / a.per, (unsigned)(((unsigned long long)a.tokens + most - 1) / most)});
  return (unsigned long long)a.wg_tokens * a.per * a.per < 1ULL << 32;
}
template <class T>
hipError_t rotary(const rot::Args& a, bool interleaved, bool wide, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const dim3 grid((a.tokens + a.wg_tokens - 1) / a.wg_tokens), block(256);
  if (wide) {
    if (interleaved) hipLaunchKernelGGL((rot::rotary_kernel<T, V / 2, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((rot::rotary_kernel<T, V, false>), grid, block, 0, st, a);
  } else {
    if (interleaved) hipLaunchKernelGGL((rot::rotary_kernel<T, 1, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((rot::rotary_kernel<T, 1, false>), grid, block, 0, st, a);
  }
  return hipGetLastError();
}

// ---- norms ----

// How a row is read: in vectors of 16 bytes; in vectors of 8 (bf16); of 16 from the boundary before the row on
// (SHIFTED); or channel by channel.
enum Access { WHOLE, HALVES, SHIFTED, SINGLE };
// How it lies in registers: n channels to a lane, the fewest wavefronts that hold it. Rows that start at the same
// distance from a boundary are `step` apart.
struct RowShape {
  Access access;
  int n, waves, step;
  // of a row, where a wavefront has several: 16 or 32; else 64. (A training step over 25 M bf16 elements, us, with 64
  // lanes and with these: C = 64 713, 201; 128 369, 139; 256 201, 140.)
  int lanes;
};
RowShape row_shape(const sffft_blocknorm* p, Access access) {
  const int V = p->io ? 8 : 4, places = p->C + (access == SHIFTED ? V - 1 : 0), n = places > 8192 ? 16 : 8;
  int step = 1;
  while (access == SHIFTED && (long long)step * p->C % V) step *= 2;
  return {access, n, (places + 64 * n - 1) / (64 * n), step, places <= 128 ? 16 : places <= 256 ? 32 : 64};
}
constexpr int MAX_WAVES = 16;

// Rows in parts that one workgroup each takes: as many workgroups as `fill` wavefronts on each of 256 CUs hold (one
// round of them: a second one for a few more would double the time), no part across rows of different gates.
struct Parts {
  long long block_rows, blocks, nparts;
  int part_rows, step, per_block;
};
Parts parts_of(const sffft_blocknorm* p, const RowShape& s, bool shared_gate, int fill) {
  Parts q;
  q.block_rows = shared_gate ? p->gate_rows : p->rows;
  q.blocks = p->rows / q.block_rows;
  q.step = (int)std::min<long long>(s.step, q.block_rows);
  const long long groups = std::max<long long>(1, 256 * std::max(1, fill / s.waves) / q.blocks / q.step);
  const long long run = (q.block_rows + q.step - 1) / q.step;  // rows of a class
  const long long rows = 64 / s.lanes, each = (run + groups - 1) / groups;
  q.part_rows = (int)std::min<long long>((each + rows - 1) / rows * rows, INT_MAX / 16);
  q.per_block = (int)std::min<long long>((run + q.part_rows - 1) / q.part_rows * q.step, INT_MAX);
  q.nparts = q.blocks * q.per_block;
  return q;
}
// Registers allow about 12 wavefronts for the backward kernel and 24 for the forward one. (Forward and backward, 4 x
// 16384 rows of 1536: 561 us; half of these 683, double 596.)
constexpr int FILL_FWD = 24, FILL_BWD = 12;

template <class T, int VEC, int N, int BLK, bool SHIFT>
void norm_launch(const bn::Args& a, int waves, bool y, bool backward, dim3 grid, hipStream_t st) {
  const dim3 block(64u * waves);
  if (backward) {
    if (y) hipLaunchKernelGGL((bn::bwd_kernel<T, VEC, N, BLK, SHIFT, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((bn::bwd_kernel<T, VEC, N, BLK, SHIFT, false>), grid, block, 0, st, a);
  } else {
    if (y) hipLaunchKernelGGL((bn::fwd_kernel<T, VEC, N, BLK, SHIFT, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((bn::fwd_kernel<T, VEC, N, BLK, SHIFT, false>), grid, block, 0, st, a);
  }
}
template <class T, int VEC, bool SHIFT = false>
void norm_access(const bn::Args& a, const RowShape& s, bool y, bool backward, dim3 grid, hipStream_t st) {
  if (s.lanes == 16) norm_launch<T, VEC, 8, 16, SHIFT>(a, s.waves, y, backward, grid, st);
  else if (s.lanes == 32) norm_launch<T, VEC, 8, 32, SHIFT>(a, s.waves, y, backward, grid, st);
  else if (s.n == 16) norm_launch<T, VEC, 16, 1024, SHIFT>(a, s.waves, y, backward, grid, st);
  else if (s.waves > 8) norm_launch<T, VEC, 8, 1024, SHIFT>(a, s.waves, y, backward, grid, st);
  else if (s.waves > 4) norm_launch<T, VEC, 8, 512, SHIFT>(a, s.waves, y, backward, grid, st);
  else norm_launch<T, VEC, 8, 256, SHIFT>(a, s.waves, y, backward, grid, st);
}
template <class T>
hipError_t norm(const bn::Args& a, const RowShape& s, bool y, bool backward, dim3 grid, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (s.access == WHOLE) norm_access<T, V>(a, s, y, backward, grid, st);
  else if (s.access == SHIFTED) norm_access<T, V, true>(a, s, y, backward, grid, st);
  else if (s.access == SINGLE) norm_access<T, 1>(a, s, y, backward, grid, st);
  else if constexpr (V == 8) norm_access<T, 4>(a, s, y, backward, grid, st);
  return hipGetLastError();
}

constexpr int MAX_C = 16384;

bool valid_norm(const sffft_blocknorm* p) {
  return p && ops::valid_io(p->io) && p->rows >= 1 && p->rows <= (1LL << 40) && p->C >= 1 && p->C <= MAX_C &&
         p->act >= SFFFT_ACT_NONE && p->act <= SFFFT_ACT_SILU && p->gate_rows >= 1 && p->rows % p->gate_rows == 0 &&
         p->eps >= 0.f && std::isfinite(p->eps);
}

// extents of the rows of a strided array; 0 if invalid
size_t row_bytes(const sffft_blocknorm* p, long long stride, long long rows) {
  if (stride < 0 || (rows > 1 && stride && stride < p->C)) return 0;
  const __int128 e = ((__int128)stride * (rows - 1) + p->C) * (p->io ? 2 : 4);
  return e >= ((__int128)1 << 62) ? 0 : (size_t)e;
}

struct Span {
  const void* p;
  size_t n;
};
// no output overlaps an input or another output
bool apart(const Span* in, int ni, const Span* out, int no) {
  for (int i = 0; i < no; i++) {
    for (int j = 0; j < ni; j++)
      if (ops::overlap(out[i].p, out[i].n, in[j].p, in[j].n)) return false;
    for (int j = 0; j < i; j++)
      if (ops::overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return false;
  }
  return true;
}

// WHOLE (HALVES) where every row starts and ends at a boundary of 16 (8) bytes, SHIFTED where those of all arrays
// start at the same distance from one of 16 (a gate that rows share is read seldom and does not count). A training
// step over 25 M elements with a gate for each token, us: bf16 C = 1531 SINGLE 897, SHIFTED 223; 2047 886, 380; 5001
// 671, 354; 8185 580, 316; 9001 1462, 734; 12289 1164, 646; fp32 1531 312, 303; 2047 343, 435; 5001 476, 467; 9001 1193,
// 937; 12289 1030, 865; bf16 1028 HALVES 192, SHIFTED 248.
struct RowArray {
  const void* p;
  long long stride;
};
Access access_of(const sffft_blocknorm* p, std::initializer_list<RowArray> arrays, RowArray gate, const float* const (&w)[3]) {
  const int elem = p->io ? 2 : 4, V = 16 / elem;
  int vec = p->C % V ? p->C % 4 ? 1 : 4 : V;  // what is aligned
  // (a row of SHIFTED has 16 bytes at least: what is read beside it then lies in its neighbours)
  bool shifted = p->C >= V;
  const auto whole = [&](const RowArray& a) {
    if (!a.p) return;
    while (vec > 1 && (!ops::aligned(a.p, vec * elem) || a.stride % vec)) vec = vec > 4 ? 4 : 1;
  };
  const auto look = [&](const RowArray& a) {
    if (!a.p) return;
    whole(a);
    shifted = shifted && ((uintptr_t)a.p - (uintptr_t)arrays.begin()->p) % 16 == 0 &&
              (p->rows == 1 || (a.stride >= p->C && (a.stride - p->C) % V == 0));
  };
  for (const RowArray& a : arrays) look(a);
  if (p->gate_rows == 1) look(gate);
  else whole(gate);
  for (const float* x : w)
    if (!ops::aligned(x, 16)) vec = 1;
  if (vec == V) return WHOLE;
  if (vec == 4) return HALVES;
  // fp32 rows that would take one more wavefront are faster channel by channel: two workgroups of 5 on a CU instead
  // of three of 4
  const int waves = row_shape(p, SHIFTED).waves;
  return shifted && (p->io ? waves <= MAX_WAVES : waves == row_shape(p, SINGLE).waves) ? SHIFTED : SINGLE;
}

}  // namespace
}  // namespace sffft

using namespace sffft;

extern "C" {

int sffft_rotary_apply(const sffft_rotary* p, const void* q, const void* k, const float* table, const void* pos,
                       void* qo, void* ko, void* stream) {
  if (!p || !ops::valid_io(p->io) || p->B < 1 || p->T < 1 || p->H < 1 || p->Hk < 0 || p->D < 2 || p->D % 2 ||
      p->R < 2 || p->R % 2 || p->R > p->D || p->positions < 1 || (p->interleaved != 0 && p->interleaved != 1) ||
      (p->inverse != 0 && p->inverse != 1) || (pos && p->pos_bits != 32 && p->pos_bits != 64) || !q || !qo || !table ||
      (p->Hk > 0) != (k != nullptr) || (p->Hk > 0) != (ko != nullptr))
    return SFFFT_EINVAL;
  const int elem = p->io ? 2 : 4;
  // a token's pairs are counted in 16 bits, the tokens in 31
  if ((long long)p->B * p->T > INT_MAX || ((long long)p->H + p->Hk) * (p->D / 2) > 65535) return SFFFT_EINVAL;
  const size_t nq = ops::extent(p->q, p->B, p->T, p->H, p->D, elem), mq = ops::extent(p->qo, p->B, p->T, p->H, p->D, elem);
  const size_t nk = k ? ops::extent(p->k, p->B, p->T, p->Hk, p->D, elem) : 1;
  const size_t mk = k ? ops::extent(p->ko, p->B, p->T, p->Hk, p->D, elem) : 1;
  if (!nq || !mq || !nk || !mk || !ops::aligned(q, elem) || !ops::aligned(k, elem) || !ops::aligned(qo, elem) ||
      !ops::aligned(ko, elem) || !ops::aligned(table, 4) || !ops::aligned(pos, p->pos_bits / 8))
    return SFFFT_EINVAL;
  // in place (q itself, with its strides) or apart
  const bool sq = q == qo && std::equal(p->q, p->q + 3, p->qo), sk = k == ko && std::equal(p->k, p->k + 3, p->ko);
  const size_t nt = (size_t)p->positions * p->R * 4, np = pos ? (size_t)p->B * p->T * (p->pos_bits / 8) : 0;
  // (q and k may be views of one array whose extents interleave; what is written in place is no element of another)
  const auto apart_from = [&](const void* a, const long long* sa, int ha, const void* b, const long long* sb, int hb) {
    return ops::distinct(a, sa, ha, b, sb, hb, p->B, p->T, p->D, elem);
  };
  if (!apart_from(qo, p->qo, p->H, ko, p->ko, p->Hk) || (sq && !apart_from(q, p->q, p->H, k, p->k, p->Hk)) ||
      (sk && k && !apart_from(k, p->k, p->Hk, q, p->q, p->H)))
    return SFFFT_EINVAL;
  if ((!sq && (ops::overlap(qo, mq, q, nq) || ops::overlap(qo, mq, k, k ? nk : 0))) ||
      (!sk && (ops::overlap(ko, mk, k, nk) || ops::overlap(ko, k ? mk : 0, q, nq))) || qo == ko ||
      ops::overlap(qo, mq, table, nt) ||
      ops::overlap(ko, mk, table, nt) || ops::overlap(qo, mq, pos, np) || ops::overlap(ko, mk, pos, np))
    return SFFFT_EINVAL;
  rot::Args a = {};
  a.q = {q, qo, p->q[0], p->q[1], p->q[2], p->qo[0], p->qo[1], p->qo[2]};
  a.k = {k, ko, p->k[0], p->k[1], p->k[2], p->ko[0], p->ko[1], p->ko[2]};
  a.table = table, a.pos = pos, a.pos64 = p->pos_bits == 64, a.positions = p->positions;
  a.tokens = (unsigned)((long long)p->B * p->T), a.T = p->T;
  bool flat = pos || p->B == 1;  // one stride leads through all tokens, and no token's place in its sequence matters
  for (const long long* s : {p->q, p->k, p->qo, p->ko}) flat = flat && (p->B == 1 || s[0] == s[1] * p->T || (!k && (s == p->k || s == p->ko)));
  if (flat) a.T = a.tokens;
  a.H = p->H, a.heads = p->H + p->Hk, a.D = p->D, a.R = p->R, a.inverse = p->inverse;
  // 16-byte loads of 8 bf16 or 4 fp32 channels; a lane takes two
  bool wide = p->D % (32 / elem) == 0 && p->R % (32 / elem) == 0 && ops::aligned(q, 16) && ops::aligned(k, 16) &&
              ops::aligned(qo, 16) && ops::aligned(ko, 16) && ops::aligned(table, 16);
  for (int i = 0; i < 3; i++)
    wide = wide && p->q[i] * elem % 16 == 0 && p->qo[i] * elem % 16 == 0 &&
           (!k || (p->k[i] * elem % 16 == 0 && p->ko[i] * elem % 16 == 0));
  if (!rotary_grid(a, elem, p->interleaved, wide)) return SFFFT_EINVAL;
  const auto run = p->io ? rotary<uint16_t> : rotary<float>;
  return ops::hip_status(run(a, p->interleaved, wide, (hipStream_t)stream), "rotary launch");
}

int sffft_rotary_table(int positions, int R, double base, int scaling, double factor, int trained, double magnitude,
                       float* table) {
  if (positions < 1 || R < 2 || R % 2 || !(base > 0) || !std::isfinite(base) || scaling < SFFFT_ROTARY_NONE ||
      scaling > SFFFT_ROTARY_PARTS || !(factor > 0) || !std::isfinite(factor) || !std::isfinite(magnitude) || !table ||
      (scaling == SFFFT_ROTARY_PARTS && trained < 1))
    return SFFFT_EINVAL;
  if (scaling == SFFFT_ROTARY_STRETCHED && R > 2) base *= std::pow(factor, (double)R / (R - 2));
  for (int i = 0; i < R / 2; i++) {
    double f = std::pow(base, -2.0 * i / R);
    if (scaling == SFFFT_ROTARY_LINEAR) f /= factor;
    if (scaling == SFFFT_ROTARY_PARTS) {
      const double turns = trained * f / (2 * M_PI), keep = std::min(1.0, std::max(0.0, (turns - 1) / 31));
      f = f * keep + f / factor * (1 - keep);
    }
    for (int n = 0; n < positions; n++) {
      table[(size_t)n * R + i] = (float)(magnitude * std::cos(n * f));
      table[(size_t)n * R + R / 2 + i] = (float)(magnitude * std::sin(n * f));
    }
  }
  return SFFFT_OK;
}

int sffft_blocknorm_fwd(const sffft_blocknorm* p, const void* x, const void* y, const void* gate, const float* w_pre,
                        const float* w_post, const float* scale, void* r, void* h, void* stream) {
  if (!valid_norm(p) || !x || !h || !w_pre || (y != nullptr) != (r != nullptr) || (!y && (gate || w_post || scale)))
    return SFFFT_EINVAL;
  const int elem = p->io ? 2 : 4;
  const long long gates = p->rows / p->gate_rows;
  const size_t vec = (size_t)p->C * 4, nx = row_bytes(p, p->x, p->rows), ny = y ? row_bytes(p, p->y, p->rows) : 1;
  const size_t ng = gate ? row_bytes(p, p->gate, gates) : 1, no = (size_t)p->rows * p->C * elem;
  if (!nx || !ny || !ng) return SFFFT_EINVAL;
  const Span in[] = {{x, nx}, {y, ny}, {gate, ng}, {w_pre, vec}, {w_post, vec}, {scale, vec}};
  const Span out[] = {{r, no}, {h, no}};
  for (int i = 0; i < 6; i++)
    if (!ops::aligned(in[i].p, i < 3 ? elem : 4)) return SFFFT_EINVAL;
  if (!ops::aligned(r, elem) || !ops::aligned(h, elem) || !apart(in, 6, out, 2)) return SFFFT_EINVAL;
  const RowShape s = row_shape(p, access_of(p, {{x, p->x}, {y, p->y}, {r, p->C}, {h, p->C}}, {gate, p->gate},
                                            {w_pre, w_post, scale}));
  const Parts q = parts_of(p, s, gate && p->gate_rows > 1, FILL_FWD);
  if (q.nparts > INT_MAX || !ops::launchable(q.nparts, 64 * s.waves)) return SFFFT_EINVAL;
  bn::Args a = {};
  a.x = x, a.y = y, a.gate = gate, a.sx = p->x, a.sy = p->y, a.sg = p->gate;
  a.wq = w_pre, a.wp = w_post, a.sc = scale, a.r = r, a.h = h;
  a.rows = p->rows, a.gate_rows = p->gate_rows, a.C = p->C, a.act = p->act, a.eps = p->eps;
  a.block_rows = q.block_rows, a.part_rows = q.part_rows, a.step = q.step, a.parts_per_block = q.per_block;
  const auto run = p->io ? norm<uint16_t> : norm<float>;
  return ops::hip_status(run(a, s, y != nullptr, false, dim3((unsigned)q.nparts), (hipStream_t)stream),
                         "block norm launch");
}

size_t sffft_blocknorm_work_bytes(const sffft_blocknorm* p, int has_y, int has_gate) {
  if (!valid_norm(p)) return 0;
  const bool shared = has_gate && p->gate_rows > 1;
  long long n = 0;  // of any access: where the arrays lie is not known yet
  for (Access a : {WHOLE, SHIFTED}) n = std::max(n, parts_of(p, row_shape(p, a), shared, FILL_BWD).nparts);
  return (size_t)(has_y ? shared ? 3 : 2 : 1) * n * p->C * 4;
}

int sffft_blocknorm_bwd(const sffft_blocknorm* p, const void* x, const void* y, const void* gate, const float* w_pre,
                        const float* w_post, const float* scale, const void* gr, const void* gh, void* dx, void* dy,
                        void* dgate, float* dw_pre, float* dw_post, float* dscale, void* work, size_t work_bytes,
                        void* stream) {
  if (!valid_norm(p) || !x || !w_pre || !dx || !dw_pre || (!gr && !gh) || (y != nullptr) != (dy != nullptr) ||
      (gate != nullptr) != (dgate != nullptr) || (w_post != nullptr) != (dw_post != nullptr) ||
      (scale != nullptr) != (dscale != nullptr) || (!y && (gate || w_post || scale)))
    return SFFFT_EINVAL;
  const int elem = p->io ? 2 : 4;
  const bool shared = gate && p->gate_rows > 1;
  const long long gates = p->rows / p->gate_rows;
  const size_t vec = (size_t)p->C * 4, no = (size_t)p->rows * p->C * elem;
  const size_t nx = row_bytes(p, p->x, p->rows), ny = y ? row_bytes(p, p->y, p->rows) : 1;
  const size_t ng = gate ? row_bytes(p, p->gate, gates) : 1, nr = gr ? row_bytes(p, p->gr, p->rows) : 1;
  const size_t nh = gh ? row_bytes(p, p->gh, p->rows) : 1, need = sffft_blocknorm_work_bytes(p, y != nullptr, gate != nullptr);
  if (!nx || !ny || !ng || !nr || !nh || !work || work_bytes < need || !ops::aligned(work, 16)) return SFFFT_EINVAL;
  const Span in[] = {{x, nx}, {y, ny}, {gate, ng}, {gr, nr}, {gh, nh}, {w_pre, vec}, {w_post, vec}, {scale, vec}};
  const Span out[] = {{dx, no}, {dy, no}, {dgate, (size_t)gates * p->C * elem}, {dw_pre, vec}, {dw_post, vec},
                      {dscale, vec}, {work, need}};
  for (int i = 0; i < 8; i++)
    if (!ops::aligned(in[i].p, i < 5 ? elem : 4)) return SFFFT_EINVAL;
  for (int i = 0; i < 6; i++)
    if (!ops::aligned(out[i].p, i < 3 ? elem : 4)) return SFFFT_EINVAL;
  if (!apart(in, 8, out, 7)) return SFFFT_EINVAL;
  const RowArray gates_in = {gate, p->gate}, gates_out = {shared ? nullptr : dgate, p->C};
  const RowShape s = row_shape(p, access_of(p, {{x, p->x}, {y, p->y}, {gr, p->gr}, {gh, p->gh}, {dx, p->C}, {dy, p->C}, gates_out},
                                            gates_in, {w_pre, w_post, scale}));
  const Parts q = parts_of(p, s, shared, FILL_BWD);
  if (q.nparts > INT_MAX || !ops::launchable(q.nparts, 64 * s.waves)) return SFFFT_EINVAL;
  bn::Args a = {};
  a.x = x, a.y = y, a.gate = gate, a.gr = gr, a.gh = gh;
  a.sx = p->x, a.sy = p->y, a.sg = p->gate, a.sgr = p->gr, a.sgh = p->gh;
  a.wq = w_pre, a.wp = w_post, a.sc = scale, a.dx = dx, a.dy = dy, a.dgate = dgate;
  a.parts = static_cast<float*>(work), a.rows = p->rows, a.gate_rows = gate ? p->gate_rows : 1;
  a.block_rows = q.block_rows, a.C = p->C, a.act = p->act, a.part_rows = q.part_rows, a.step = q.step, a.parts_per_block = q.per_block;
  a.nparts = q.nparts, a.eps = p->eps;
  hipStream_t st = (hipStream_t)stream;
  const auto run = p->io ? norm<uint16_t> : norm<float>;
  hipError_t err = run(a, s, y != nullptr, true, dim3((unsigned)q.nparts), st);
  if (err == hipSuccess) {
    const long long sums = (y ? 2 : 1) + (shared ? q.blocks : 0);
    const bn::SumArgs u = {a.parts, w_post, scale, dw_pre, dw_post, dscale, shared ? dgate : nullptr, p->C, p->io,
                           y != nullptr, q.nparts, q.per_block, sums};
    hipLaunchKernelGGL(bn::sum_kernel, dim3((unsigned)((p->C + 31) / 32), (unsigned)std::min<long long>(sums, 32768)), dim3(1024),
                       0, st, u);
    err = hipGetLastError();
  }
  return ops::hip_status(err, "block norm gradient launch");
}

const char* sffft_ops_last_error(void) { return ops::g_last_error; }

}  // extern "C"
