// Launches and C ABI of linear attention (linattn.hpp).
#include <algorithm>
#include <climits>
#include <initializer_list>

#include "linattn.hpp"
#include "ops_status.hpp"

namespace sffft {
namespace {

using la::March;
using la::Operand;
using la::Shape;

constexpr int MAX_D = 128;
// the rows of a chunk are addressed by 31-bit byte offsets: 64 of them in 2 bytes, 32 in 4
constexpr long long MAX_TOKEN_STRIDE = (1 << 24) - MAX_D;

bool valid_shape(const sffft_linattn* p) {
  if (!p || !ops::valid_io(p->io) || p->B < 1 || p->T < 1 || p->H < 1 || p->Hk < 1 || p->H % p->Hk) return false;
  if (p->Dk < 8 || p->Dv < 8 || p->Dk > MAX_D || p->Dv > MAX_D || p->Dk % 8 || p->Dv % 8) return false;
  return (long long)p->B * p->H <= INT_MAX / 64 && (long long)p->B * p->T <= INT_MAX &&
         (long long)p->H * std::max(p->Dk, p->Dv) <= MAX_TOKEN_STRIDE / 2;
}

// A strided input: 16-byte aligned rows, and its extent.
bool valid_input(const void* x, const long long s[3], const sffft_linattn* p, int heads, int D, size_t* bytes) {
  const int elem = p->io ? 2 : 4;
  if (!x || !ops::aligned(x, 16)) return false;
  for (int i = 0; i < 3; i++)
    if (s[i] * elem % 16) return false;
  if (s[1] > MAX_TOKEN_STRIDE) return false;
  *bytes = ops::extent(s, p->B, p->T, heads, D, elem);
  return *bytes != 0;
}

Operand operand(const void* x, const long long s[3], int div) { return {x, s[0], s[1], s[2], div}; }

// More segments than this are joined by a launch of its own, fewer by each workgroup that follows them. (us at 4, 8,
// 16: training, 8 x 2048 tokens, 12 heads of 64 channels, bf16 134, 130, 130; 5 x 1237 tokens forward 27.9, 26.9,
// 29.1; training, 3 x 1531 tokens, 12 heads on 4 of 96 and 64, fp32 147, 147, 164.)
constexpr int MAX_JOINED = 8;

// How a call is cut: segments of whole chunks, as many as give the chip `fill` workgroups of the march, two or three
// to a CU by their registers (half, these, double: the bf16 training step above 142, 130, 135, the fp32 one 146, 147,
// 172; 131072 tokens of 12 heads of 128 channels 666, 576, 616). No more than MAX_JOINED where these are few chunks longer and as many
// workgroups as the chip runs well: a launch and the states' way through memory less. Measured at 180 sizes of 8 to 96
// heads and 300 to 8192 tokens, forward, time with any number of segments over time with 8: from 160 workgroups (5 for
// every 8 CUs) on 1.0 to 1.3, of 40 to 130 0.64 to 1.14, most below 1. Above 64 channels a second workgroup on a CU
// costs more than the launch (bf16, 2048 tokens: 36 heads, 288 workgroups 55.9 -> 66.9 us; 1200 tokens, 252 45.6 ->
// 40.1), and segments two or more chunks longer only pay in fp32. Up to 64 channels it does not, up to three longer
// ones either (bf16 0.94 to 1.32); fp32's third does (576 to 768 workgroups 0.85 to 1.04).
struct Cut {
  int nseg, seg;
};
Cut cut_of(const sffft_linattn* p, int marches) {
  const int C = p->io ? la::chunk_of<uint16_t>() : la::chunk_of<float>(), D = std::max(p->Dk, p->Dv);
  const int chunks = (p->T - 1) / C + 1, fill = D > 64 ? 512 : 1024;
  const long long heads = (long long)p->B * p->H * marches;
  const int want = (int)std::min<long long>(chunks, std::max<long long>(1, fill / heads));
  const int few = (chunks + MAX_JOINED - 1) / MAX_JOINED, joined = (chunks + few - 1) / few;
  int per = (chunks + want - 1) / want;
  const long long cus = 256, workgroups = joined * heads;
  const bool fits = workgroups >= cus * 5 / 8 && (D > 64 ? workgroups <= cus : p->io || workgroups <= 2 * cus);
  if (few > per && few - per <= (D > 64 ? 1 : 3) && fits) per = few;
  return {(chunks + per - 1) / per, per * C};
}

// Marches of the gradients' smallest launch (see backward): they share one where sizes and types are equal. (Segments
// for three marches also where each has a launch of its own: the fp32 step above 182 us instead of 147.)
int backward_marches(const sffft_linattn* p) { return p->Dk == p->Dv && (p->H == p->Hk || !p->io) ? 3 : 1; }

// Workgroups of nm marches over units of a head and a segment.
long long workgroups(long long units, int nm, int vtiles) { return (units + 7) / 8 * 8 * nm * vtiles; }

template <class T, class TO, int KT, int VT, bool OUT, int UP>
hipError_t launch(la::Launch& L, hipStream_t st) {
  L.vtiles = (L.m[0].V + VT - 1) / VT;
  const int units = L.s.B * L.s.H * (OUT || L.all ? L.nseg : L.nseg - 1);
  hipLaunchKernelGGL((la::march_kernel<T, TO, KT, VT, OUT, UP>), dim3((unsigned)workgroups(units, L.nm, L.vtiles)),
                     dim3(256), 0, st, L);
  return hipGetLastError();
}
// Tiles of 32, 64, 96 or 128 channels of K, 64 or 128 of V. (In the next larger one of K instead, training, 8 x 12
// heads of 600 tokens, us: bf16 heads of 32 channels 58 for 51, of 96 107 for 96; fp32 95 for 74, 227 for 168.) One tile
// of 128 of V wherever it leaves two workgroups on a CU: beside fp32's 128 of K the planes do not, beside 32 of K two of
// 64 leave three. (Two of 64 instead, us: fp32 64 x 96 channels 157 for 139, 96 x 96 199 for 169; bf16 64 x 96 104 for
// 100, 64 x 128 of 8 x 2048 tokens 229 for 210, 128 x 128 of 131072 tokens forward 706 for 576.)
int v_tile(int elem, int K, int V) {
  const bool wide = K > 32 && (elem == 2 || K <= 96);
  return V > 64 && wide ? 128 : 64;
}
template <class T, class TO, bool OUT, int UP>
hipError_t march_planes(la::Launch& L, hipStream_t st) {
  const int K = L.m[0].K;
  const bool wide = v_tile(sizeof(T), K, L.m[0].V) == 128;
  if (K <= 32) return launch<T, TO, 32, 64, OUT, UP>(L, st);
  if (K <= 64) return wide ? launch<T, TO, 64, 128, OUT, UP>(L, st) : launch<T, TO, 64, 64, OUT, UP>(L, st);
  if (K <= 96) return wide ? launch<T, TO, 96, 128, OUT, UP>(L, st) : launch<T, TO, 96, 64, OUT, UP>(L, st);
  if constexpr (sizeof(T) == 2)
    if (wide) return launch<T, TO, 128, 128, OUT, UP>(L, st);
  return launch<T, TO, 128, 64, OUT, UP>(L, st);
}
// nm marches of the same K and V
template <class T, bool OUT, class TO = T>
hipError_t march(la::Launch L, hipStream_t st) {
  bool state = !OUT || sizeof(T) == 4;  // whether states leave in fp32
  for (int i = 0; i < L.nm; i++) state = state || (L.m[i].s1 && !L.all);
  if constexpr (OUT && sizeof(T) == 2)
    if (!state) return march_planes<T, TO, OUT, 2>(L, st);
  return march_planes<T, TO, OUT, 3>(L, st);
}
hipError_t scan(const la::ScanLaunch& L, int n, hipStream_t st) {
  const unsigned tiles = (unsigned)((L.c[0].n + 1023) / 1024);
  hipLaunchKernelGGL(la::scan_kernel, dim3((unsigned)(L.s.B * L.s.H) * tiles, (unsigned)n), dim3(256), 0, st, L);
  return hipGetLastError();
}

long long head_sum_workgroups(long long n) { return (n / 4 + 255) / 256; }
template <class T>
hipError_t head_sums(la::HeadSums L, hipStream_t st) {
  L.blocks = (unsigned)head_sum_workgroups(L.s[0].n);
  hipLaunchKernelGGL(la::head_sum_kernel<T>, dim3(L.blocks + (unsigned)head_sum_workgroups(L.s[1].n)), dim3(256), 0, st, L);
  return hipGetLastError();
}

// The segments' sums, or entering states
size_t state_bytes(const sffft_linattn* p, const Cut& c) {
  return c.nseg == 1 ? 0 : (size_t)p->B * p->H * c.nseg * p->Dk * p->Dv * 4;
}
// From this many segments on the sum of the last one is made too, for the last state: it costs one more of many sums,
// and the march then adds to its state only what outputs of 16 bits need. (Never: 130.7, 27.5 and 146 us in the cases
// above.)
constexpr int MIN_ALL = 4;
// dk and dv of heads that are shared, for each query head, before their sum
size_t shared_bytes(const sffft_linattn* p) {
  return p->H == p->Hk ? 0 : (size_t)p->B * p->T * p->H * (p->Dk + p->Dv) * 4;
}

// Arguments that fit every launch of a forward or backward call, the largest of each size of marches.
bool valid_call(const sffft_linattn* p, int backward) {
  if (!valid_shape(p)) return false;
  const int nseg = cut_of(p, backward ? backward_marches(p) : 1).nseg, elem = p->io ? 2 : 4;
  const auto fits = [&](int nm, int K, int V) {
    const int VT = v_tile(elem, K, V);
    return ops::launchable(workgroups((long long)p->B * p->H * nseg, nm, (V + VT - 1) / VT), 256);
  };
  if (!backward) return fits(1, p->Dk, p->Dv);
  const long long tokens = (long long)p->B * p->T;
  const bool parts = p->H != p->Hk;
  if (parts && !ops::launchable(head_sum_workgroups(tokens * p->Hk * p->Dk) + head_sum_workgroups(tokens * p->Hk * p->Dv), 256))
    return false;
  const int together = parts && p->io ? 1 : 2;  // marches that share a launch where Dk and Dv differ
  return p->Dk == p->Dv ? fits(together + 1, p->Dk, p->Dv)
                        : fits(nseg > 1 ? 2 : 1, p->Dk, p->Dv) && fits(together, p->Dv, p->Dk);
}

template <class T>
hipError_t forward(const sffft_linattn* p, const void* q, const void* k, const void* v, const Shape& s,
                   const float* s0, void* o, float* s1, float* work, hipStream_t st) {
  const int G = p->H / p->Hk;
  const Cut cut = cut_of(p, 1);
  const March m = {operand(q, p->q, 1), operand(k, p->k, G), operand(v, p->v, G), o, s0, work, s1, p->Dk, p->Dv, p->Dv, 1,
                   0, p->scale, p->scale, 1.f};
  // A scan too where the last state takes the initial one's place: workgroups that join the segments read that one
  // while another writes it.
  const bool scanned = cut.nseg > MAX_JOINED || (cut.nseg > 1 && s1 && s1 == s0);
  la::Launch L = {{m}, s, 1, cut.nseg, cut.seg, 1, scanned, scanned || (s1 && cut.nseg >= MIN_ALL)};
  hipError_t e = hipSuccess;
  if (cut.nseg > 1) e = march<T, false>(L, st);
  if (e == hipSuccess && L.scanned) {
    e = scan({{{work, s0, s1, p->Dk * p->Dv, 0}}, s, cut.nseg, cut.seg}, 1, st);
    L.m[0].s1 = nullptr;
  }
  return e == hipSuccess ? march<T, true>(L, st) : e;
}

template <class T>
hipError_t backward(const sffft_linattn* p, const void* q, const void* k, const void* v, const void* go,
                    const Shape& s, const float* s0, const float* ds1, void* dq, void* dk, void* dv, float* ds0,
                    float* work, hipStream_t st) {
  const int G = p->H / p->Hk, Dk = p->Dk, Dv = p->Dv;
  const Operand Q = operand(q, p->q, 1), K = operand(k, p->k, G), V = operand(v, p->v, G), O = operand(go, p->go, 1);
  const size_t rows = (size_t)p->B * p->T;
  const Cut cut = cut_of(p, backward_marches(p));
  const size_t states = state_bytes(p, cut) / 4;
  float *ws = work, *wd = ws + states, *wk = wd + states, *wv = wk + rows * p->H * Dk;
  const float c = p->scale;
  March mv = {K, Q, O, G > 1 ? wv : dv, ds1, wd, ds0, Dk, Dv, Dv, 1, 1, c, 1.f, c};
  la::Launch L = {{{Q, K, V, nullptr, s0, ws, nullptr, Dk, Dv, Dv, 1, 0, c, c, 1.f}, mv}, s, 2, cut.nseg, cut.seg, 1,
                  cut.nseg > MAX_JOINED, cut.nseg > MAX_JOINED || (ds0 && cut.nseg >= MIN_ALL)};
  hipError_t e = hipSuccess;
  if (cut.nseg > 1) e = march<T, false>(L, st);
  if (e == hipSuccess && L.scanned)
    e = scan({{{ws, s0, nullptr, Dk * Dv, 0}, {wd, ds1, ds0, Dk * Dv, 1}}, s, cut.nseg, cut.seg}, 2, st);
  if (e != hipSuccess) return e;
  if (L.scanned) mv.s1 = nullptr;
  const March mq = {O, V, K, dq, s0, ws, nullptr, Dv, Dk, 1, Dv, 0, c, c, 1.f};
  const March mk = {V, O, Q, G > 1 ? wk : dk, ds1, wd, nullptr, Dv, Dk, 1, Dv, 1, c, 1.f, c};
  // One launch where the sizes and the types of the outputs are equal: what is summed afterwards leaves in fp32.
  const auto run = [&](std::initializer_list<March> ms, bool parts) {
    L.nm = 0;
    for (const March& m : ms) L.m[L.nm++] = m;
    if (e == hipSuccess) e = parts ? march<T, true, float>(L, st) : march<T, true>(L, st);
  };
  const bool parts = G > 1, split = parts && sizeof(T) == 2;
  if (Dk == Dv) {
    if (!split) run({mq, mv, mk}, false);
    else run({mq}, false), run({mv, mk}, true);
  } else {
    if (!split) run({mq, mk}, false), run({mv}, false);
    else run({mq}, false), run({mk}, true), run({mv}, true);
  }
  if (!parts || e != hipSuccess) return e;
  return head_sums<T>({{{wk, dk, (long long)rows * p->Hk * Dk, Dk}, {wv, dv, (long long)rows * p->Hk * Dv, Dv}}, G, 0}, st);
}

}  // namespace
}  // namespace sffft

using namespace sffft;

extern "C" {

size_t sffft_linattn_work_bytes(const sffft_linattn* p, int backward) {
  if (!valid_call(p, backward)) return 0;
  return backward ? 2 * state_bytes(p, cut_of(p, backward_marches(p))) + shared_bytes(p) : state_bytes(p, cut_of(p, 1));
}

int sffft_linattn_fwd(const sffft_linattn* p, const void* q, const void* k, const void* v, const float* log_decay,
                      const float* initial_state, const int* lengths, void* o, float* final_state, void* work,
                      size_t work_bytes, void* stream) {
  size_t nq, nk, nv;
  if (!valid_call(p, 0) || !log_decay || !o || !ops::aligned(o, 16) || !valid_input(q, p->q, p, p->H, p->Dk, &nq) ||
      !valid_input(k, p->k, p, p->Hk, p->Dk, &nk) || !valid_input(v, p->v, p, p->Hk, p->Dv, &nv) ||
      !ops::aligned(initial_state, 16) || !ops::aligned(final_state, 16) || !ops::aligned(log_decay, 4) ||
      !ops::aligned(lengths, 4))
    return SFFFT_EINVAL;
  const size_t no = (size_t)p->B * p->T * p->H * p->Dv * (p->io ? 2 : 4), ns = (size_t)p->B * p->H * p->Dk * p->Dv * 4;
  const void* in[] = {q, k, v, initial_state, log_decay, lengths};
  const size_t len[] = {nq, nk, nv, ns, (size_t)p->H * 4, (size_t)p->B * 4};
  for (int i = 0; i < 6; i++)
    if (ops::overlap(o, no, in[i], len[i]) || ((i != 3 || in[i] != final_state) && ops::overlap(final_state, ns, in[i], len[i])))
      return SFFFT_EINVAL;
  if (ops::overlap(o, no, final_state, ns)) return SFFFT_EINVAL;
  const size_t need = sffft_linattn_work_bytes(p, 0);
  if (need && (!work || work_bytes < need || !ops::aligned(work, 16) || ops::overlap(work, need, o, no) ||
               ops::overlap(work, need, final_state, ns)))
    return SFFFT_EINVAL;
  for (int i = 0; i < 6; i++)
    if (need && ops::overlap(work, need, in[i], len[i])) return SFFFT_EINVAL;
  const Shape s = {p->B, p->T, p->H, log_decay, lengths};
  const auto run = p->io ? forward<uint16_t> : forward<float>;
  return ops::hip_status(run(p, q, k, v, s, initial_state, o, final_state, static_cast<float*>(work), (hipStream_t)stream),
                         "linear attention launch");
}

int sffft_linattn_bwd(const sffft_linattn* p, const void* q, const void* k, const void* v, const float* log_decay,
                      const float* initial_state, const int* lengths, const void* go, const float* d_final_state,
                      void* dq, void* dk, void* dv, float* d_initial_state, void* work, size_t work_bytes,
                      void* stream) {
  size_t nq, nk, nv, no;
  if (!valid_call(p, 1) || !log_decay || !dq || !dk || !dv || !valid_input(q, p->q, p, p->H, p->Dk, &nq) ||
      !valid_input(k, p->k, p, p->Hk, p->Dk, &nk) || !valid_input(v, p->v, p, p->Hk, p->Dv, &nv) ||
      !valid_input(go, p->go, p, p->H, p->Dv, &no) || !ops::aligned(initial_state, 16) ||
      !ops::aligned(d_final_state, 16) || !ops::aligned(d_initial_state, 16) || !ops::aligned(dq, 16) ||
      !ops::aligned(dk, 16) || !ops::aligned(dv, 16) || !ops::aligned(log_decay, 4) || !ops::aligned(lengths, 4))
    return SFFFT_EINVAL;
  const size_t elem = p->io ? 2 : 4, rows = (size_t)p->B * p->T, ns = (size_t)p->B * p->H * p->Dk * p->Dv * 4;
  const size_t need = sffft_linattn_work_bytes(p, 1);
  if (need && (!work || work_bytes < need || !ops::aligned(work, 16))) return SFFFT_EINVAL;
  const void* in[] = {q, k, v, go, initial_state, d_final_state, log_decay, lengths};
  const size_t len[] = {nq, nk, nv, no, ns, ns, (size_t)p->H * 4, (size_t)p->B * 4};
  const void* out[] = {dq, dk, dv, d_initial_state, need ? work : nullptr};
  const size_t size[] = {rows * p->H * p->Dk * elem, rows * p->Hk * p->Dk * elem, rows * p->Hk * p->Dv * elem, ns, need};
  for (int i = 0; i < 5; i++) {
    for (int j = 0; j < 8; j++)
      if (ops::overlap(out[i], size[i], in[j], len[j])) return SFFFT_EINVAL;
    for (int j = 0; j < i; j++)
      if (ops::overlap(out[i], size[i], out[j], size[j])) return SFFFT_EINVAL;
  }
  const Shape s = {p->B, p->T, p->H, log_decay, lengths};
  const auto run = p->io ? backward<uint16_t> : backward<float>;
  return ops::hip_status(run(p, q, k, v, go, s, initial_state, d_final_state, dq, dk, dv, d_initial_state,
                             static_cast<float*>(work), (hipStream_t)stream),
                         "linear attention gradient launch");
}

int sffft_linattn_step(const sffft_linattn* p, const void* q, const void* k, const void* v, const float* log_decay,
                       float* state, int slots, const int* slot, void* o, void* stream) {
  size_t nq, nk, nv;
  if (!valid_shape(p) || p->T != 1 || !ops::launchable((long long)p->B * p->H, 256) || !log_decay || !state || !o || slots < 1 || !ops::aligned(state, 16) ||
      !ops::aligned(o, 16) || !valid_input(q, p->q, p, p->H, p->Dk, &nq) ||
      !valid_input(k, p->k, p, p->Hk, p->Dk, &nk) || !valid_input(v, p->v, p, p->Hk, p->Dv, &nv) ||
      !ops::aligned(log_decay, 4) || !ops::aligned(slot, 4))
    return SFFFT_EINVAL;
  const size_t no = (size_t)p->B * p->H * p->Dv * (p->io ? 2 : 4), ns = (size_t)slots * p->H * p->Dk * p->Dv * 4;
  const void* in[] = {q, k, v, log_decay, slot};
  const size_t len[] = {nq, nk, nv, (size_t)p->H * 4, (size_t)p->B * 4};
  for (int i = 0; i < 5; i++)
    if (ops::overlap(o, no, in[i], len[i]) || ops::overlap(state, ns, in[i], len[i])) return SFFFT_EINVAL;
  if (ops::overlap(o, no, state, ns)) return SFFFT_EINVAL;
  const int G = p->H / p->Hk;
  const Operand Q = operand(q, p->q, 1), K = operand(k, p->k, G), V = operand(v, p->v, G);
  const dim3 grid((unsigned)(p->B * p->H), (unsigned)((p->Dv + 63) / 64)), block(256);
  hipStream_t st = (hipStream_t)stream;
  if (p->io)
    hipLaunchKernelGGL(la::step_kernel<uint16_t>, grid, block, 0, st, Q, K, V, log_decay, state, slots, slot,
                       static_cast<uint16_t*>(o), p->H, p->Dk, p->Dv, p->scale);
  else
    hipLaunchKernelGGL(la::step_kernel<float>, grid, block, 0, st, Q, K, V, log_decay, state, slots, slot,
                       static_cast<float*>(o), p->H, p->Dk, p->Dv, p->scale);
  return ops::hip_status(hipGetLastError(), "linear attention step launch");
}

}  // extern "C"
