// C ABI of the attention operators (declared in include/ncn_b200.h): argument checks, choice of kernels, launches.
#include <cmath>

#include "../../include/ncn_b200.h"
#include "attn_common.cuh"
#include "attn_tensor.h"
#include "ncn_common.cuh"
#include "ncn_host.h"
#include "qk_rotary.h"

namespace ncn {
namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kMaxHead = 256;
constexpr long long kMaxGrid = 0x7fffffff;

int round_up(int64_t n, int to) { return (int)((n + to - 1) / to * to); }

// The sizes and tensors of an attention call.  strides: {batch, position} of q, k, v and dy in elements, or null for contiguous ones.
int attn_params(AttnParams& p, const void* q, const void* k, const void* v, const int* ctxlen, const int* q_start, const int64_t* strides,
                int n_strides, int64_t B, int64_t Nq, int64_t Nk, int64_t E, int64_t Ek, int n_head, int64_t window, int64_t n_sink,
                int64_t start, double scale, int dtype) {
  if (dtype != NCN_F32 && dtype != NCN_BF16) return NCN_ERR_DTYPE;
  if (B < 0 || Nq < 0 || Nk < 0 || E <= 0 || Ek <= 0 || n_head <= 0 || E % n_head != 0) return NCN_ERR_SHAPE;
  const int64_t d = E / n_head;
  if (d > kMaxHead || Ek % d != 0 || (E / d) % (Ek / d) != 0) return NCN_ERR_SHAPE;
  if (window < 1 || n_sink < 0 || !std::isfinite(scale) || !(scale > 0)) return NCN_ERR_SHAPE;  // (-inf marks what is masked)
  if (B > kMaxGrid || Nq > kMaxLength || Nk > kMaxLength) return NCN_ERR_SHAPE;
  if (B == 0 || Nq == 0) return NCN_OK;  // (the caller launches nothing)
  if (!q || ((!k || !v) && Nk > 0)) return NCN_ERR_NULL;
  p.q = q, p.k = k, p.v = v;
  p.ctxlen = ctxlen, p.q_start = q_start;
  p.B = (int)B, p.Nq = (int)Nq, p.Nk = (int)Nk, p.H = n_head, p.Hk = (int)(Ek / d), p.G = p.H / p.Hk, p.d = (int)d;
  p.Nqp = round_up(Nq, 128);
  p.window = (int)(window < Nk ? window : (Nk > 0 ? Nk : 1));  // (no two visible positions are further apart)
  p.n_sink = (int)(n_sink < Nk ? n_sink : Nk);
  p.start0 = (int)(start < -Nq ? -Nq : start > Nk ? Nk : start);
  p.scale = (float)scale;
  p.scale_log2 = (float)(scale * 1.4426950408889634074);
  const long long contiguous[8] = {Nq * E, E, Nk * Ek, Ek, Nk * Ek, Ek, Nq * E, E};
  long long s[8];
  for (int i = 0; i < 8; ++i) s[i] = strides && i < n_strides ? strides[i] : contiguous[i];
  p.sq_b = s[0], p.sq_n = s[1], p.sk_b = s[2], p.sk_n = s[3], p.sv_b = s[4], p.sv_n = s[5], p.sdy_b = s[6], p.sdy_n = s[7];
  const int per = dtype == NCN_BF16 ? 8 : 4;  // elements of 16 bytes
  p.vec = d % per == 0 && aligned16(q) && aligned16(k) && aligned16(v);
  for (int i = 0; i < 8; ++i)
    if (s[i] % per) p.vec = 0;
  return NCN_OK;
}

// Tiles of sinks and pieces of the queries beyond the window, for key tiles of T and query tiles of TQ: a piece is about as long as
// what a tile's own window takes, so that the sinks' tiles, which every later query sees, hold nobody up.
void plan_sinks(AttnParams& p, int T, int TQ) {
  p.sink_tiles = p.chunks = p.sink_rows = 0;
  if (p.n_sink == 0 || p.window >= p.Nk) return;
  const int tiles = (p.Nq + TQ - 1) / TQ, own = (p.window + T) / TQ + 2;
  p.sink_tiles = (p.n_sink + T - 1) / T;
  p.sink_rows = p.n_sink < T ? p.n_sink : T;
  p.chunks = (tiles + own - 1) / own;
  const int most = p.sink_tiles < 4 ? 64 : p.sink_tiles < 256 ? 256 / p.sink_tiles : 1;  // (many sink tiles are many items already)
  if (p.chunks > most) p.chunks = most;
}
size_t part_floats(const AttnParams& p) {
  return (size_t)p.B * p.Hk * p.sink_tiles * (p.chunks + 1) * 2 * p.sink_rows * p.d;
}
size_t delta_floats(const AttnParams& p) { return (size_t)p.B * p.H * p.Nqp; }

// key tile, query tile of the backward that these arguments take
void bwd_tiles(const AttnParams& p, int dtype, int& T, int& TQ) {
  if (attn_tensor_covers(p, dtype)) {
    T = TQ = 128;
  } else {
    T = 64;
    TQ = p.d > 128 ? 32 : 64;
  }
}

void set_state(AttnParams& p, void* state, int dtype) {
  p.lse = static_cast<float*>(state);
  p.rest = state && dtype == NCN_BF16 ? reinterpret_cast<__nv_bfloat16*>(p.lse + delta_floats(p)) : nullptr;
}

// Whether a launch's CTAs can be counted: one per 64 queries of a head at most (also in the backward); in the backward one per 64 keys of
// a head and piece of the sinks' queries (after plan_sinks), and one per sink; in decode one per two of the rows that share keys, or per row
// where there is one (several share them only where there are fewer of these than SMs).
bool grid_fwd_ok(const AttnParams& p) { return (p.Nq + 63ll) / 64 * p.H <= kMaxGrid / p.B; }
bool grid_bwd_ok(const AttnParams& p) {
  const long long items = (p.Nk + 63ll) / 64 + (long long)p.sink_tiles * p.chunks;
  return grid_fwd_ok(p) && items * p.Hk <= kMaxGrid / p.B && (p.chunks == 0 || (long long)p.n_sink * p.Hk <= kMaxGrid / p.B);
}
bool grid_decode_ok(const AttnParams& p) {
  const long long rows = (long long)p.G * p.Nq;
  return rows <= 1 << 30 && (rows + 1) / 2 * p.Hk <= kMaxGrid / p.B;
}

}  // namespace
}  // namespace ncn

using namespace ncn;

extern "C" {

size_t ncn_window_state_bytes(int64_t B, int64_t Nq, int64_t E, int n_head, int dtype) {
  if (B <= 0 || Nq <= 0 || E <= 0 || n_head <= 0 || Nq > kMaxLength) return 0;
  return (size_t)B * n_head * round_up(Nq, 128) * sizeof(float) + (dtype == NCN_BF16 ? (size_t)B * Nq * E * 2 : 0);
}

int ncn_window_fwd(const void* q, const void* k, const void* v, void* y, void* state, const int* ctxlen, const int* q_start,
                   const int64_t* strides, int64_t B, int64_t Nq, int64_t Nk, int64_t E, int64_t Ek, int n_head, int64_t window,
                   int64_t n_sink, int64_t start, double scale, int dtype, void* stream) {
  AttnParams p{};
  int rc = attn_params(p, q, k, v, ctxlen, q_start, strides, 6, B, Nq, Nk, E, Ek, n_head, window, n_sink, start, scale, dtype);
  if (rc != NCN_OK || B == 0 || Nq == 0) return rc;
  if (!y) return NCN_ERR_NULL;
  if (!aligned16(state)) return NCN_ERR_ALIGN;
  if (!grid_fwd_ok(p)) return NCN_ERR_TOO_LARGE;
  DevInfo dev;
  if ((rc = get_dev(dev)) != NCN_OK) return rc;
  p.y = y, p.status = dev.status;
  set_state(p, state, dtype);
  cudaError_t e = attn_tensor_covers(p, dtype) ? launch_attn_tensor_fwd(p, (cudaStream_t)stream) : launch_attn_simt_fwd(p, dtype, (cudaStream_t)stream);
  return e == cudaSuccess ? NCN_OK : cuda_fail(e);
}

size_t ncn_window_bwd_workspace_bytes(int64_t B, int64_t Nq, int64_t Nk, int64_t E, int64_t Ek, int n_head, int64_t window, int64_t n_sink,
                                      int dtype) {
  AttnParams p{};
  const char any[16] = {};
  if (attn_params(p, any, any, any, nullptr, nullptr, nullptr, 0, B, Nq, Nk, E, Ek, n_head, window, n_sink, 0, 1.0, dtype) != NCN_OK) return 0;
  if (B == 0 || Nq == 0) return 0;
  size_t most = 0;  // whichever kernels the pointers' alignment will choose
  for (int tensor = 0; tensor < 2; ++tensor) {
    const int T = tensor ? 128 : 64, TQ = tensor ? 128 : p.d > 128 ? 32 : 64;
    plan_sinks(p, T, TQ);
    const size_t n = delta_floats(p) + part_floats(p);
    if (n > most) most = n;
  }
  return most * sizeof(float);
}

int ncn_window_bwd(const void* q, const void* k, const void* v, const void* y, const void* dy, const void* state, void* dq, void* dk, void* dv,
                   const int* ctxlen, const int* q_start, const int64_t* strides, void* workspace, size_t workspace_bytes, int64_t B,
                   int64_t Nq, int64_t Nk, int64_t E, int64_t Ek, int n_head, int64_t window, int64_t n_sink, int64_t start, double scale,
                   int dtype, void* stream) {
  AttnParams p{};
  int rc = attn_params(p, q, k, v, ctxlen, q_start, strides, 8, B, Nq, Nk, E, Ek, n_head, window, n_sink, start, scale, dtype);
  if (rc != NCN_OK || B == 0 || Nq == 0) return rc;
  if (!y || !dy || !state || !dq || ((!dk || !dv) && Nk > 0)) return NCN_ERR_NULL;
  if (!aligned16(state) || !aligned16(workspace)) return NCN_ERR_ALIGN;  // (read by bulk copies and 16 bytes at a time)
  DevInfo dev;
  if ((rc = get_dev(dev)) != NCN_OK) return rc;
  p.y_in = y, p.dy = dy, p.dq = dq, p.dk = dk, p.dv = dv, p.status = dev.status;
  set_state(p, const_cast<void*>(state), dtype);
  if (!aligned16(dy)) p.vec = 0;
  int T, TQ;
  bwd_tiles(p, dtype, T, TQ);
  plan_sinks(p, T, TQ);
  if (!grid_bwd_ok(p)) return NCN_ERR_TOO_LARGE;
  if (!workspace || workspace_bytes < (delta_floats(p) + part_floats(p)) * sizeof(float)) return NCN_ERR_WORKSPACE;
  p.delta = static_cast<float*>(workspace);
  p.part = p.delta + delta_floats(p);
  cudaError_t e = T == 128 ? launch_attn_tensor_bwd(p, (cudaStream_t)stream) : launch_attn_simt_bwd(p, dtype, (cudaStream_t)stream);
  return e == cudaSuccess ? NCN_OK : cuda_fail(e);
}

int ncn_window_decode(const void* q, const void* k, const void* v, void* y, const int* ctxlen, const int64_t* strides, int64_t B, int64_t Nq,
                      int64_t S, int64_t E, int64_t Ek, int n_head, int64_t window, int64_t n_sink, double scale, int dtype, void* stream) {
  AttnParams p{};
  int rc = attn_params(p, q, k, v, ctxlen, nullptr, strides, 6, B, Nq, S, E, Ek, n_head, window, n_sink, 0, scale, dtype);
  if (rc != NCN_OK || B == 0 || Nq == 0) return rc;
  if (!y || !ctxlen) return NCN_ERR_NULL;
  if (!grid_decode_ok(p)) return NCN_ERR_TOO_LARGE;
  DevInfo dev;
  if ((rc = get_dev(dev)) != NCN_OK) return rc;
  p.y = y, p.start_at_end = 1;
  cudaError_t e = launch_attn_decode(p, dtype, dev.sms, (cudaStream_t)stream);
  return e == cudaSuccess ? NCN_OK : cuda_fail(e);
}

}  // extern "C"

namespace ncn {
namespace {

int rotary_params(RotaryParams& p, const double* freqs, const int64_t* pos, int64_t pos_b, int64_t start, int64_t B, int64_t N, int64_t E,
                  int64_t Ek, int n_head, int64_t R, int interleaved, double eps, double magnitude, int dtype) {
  if (dtype != NCN_F32 && dtype != NCN_BF16) return NCN_ERR_DTYPE;
  if (B < 0 || N < 0 || E <= 0 || Ek < 0 || n_head <= 0 || E % n_head != 0) return NCN_ERR_SHAPE;
  const int64_t d = E / n_head;
  if (d > 512 || Ek % d != 0 || R < 0 || R > d || R % 2 != 0) return NCN_ERR_SHAPE;
  if (B > 0x7fffffff || N > 0x7fffffff || !(eps >= 0) || !std::isfinite(eps) || !std::isfinite(magnitude)) return NCN_ERR_SHAPE;
  if (R > 0 && !freqs) return NCN_ERR_NULL;
  p.freqs = freqs;
  p.pos = reinterpret_cast<const long long*>(pos);
  p.pos_b = pos_b, p.start = start;
  p.B = (int)B, p.N = (int)N, p.d = (int)d, p.R = (int)R;
  p.interleaved = interleaved != 0;
  p.eps = (float)eps;
  p.magnitude = (float)magnitude;
  p.t[0].heads = n_head;
  p.t[1].heads = (int)(Ek / d);
  return NCN_OK;
}
int set_vec(RotaryParams& p, int dtype) {
  const int per = dtype == NCN_BF16 ? 8 : 4;
  int vec = p.d % per == 0;
  for (const RotaryTensor& t : p.t) {
    if (!t.heads) continue;
    if (!aligned16(t.x) || !aligned16(t.out) || t.sb % per || t.sn % per) vec = 0;
    if (t.dy && (!aligned16(t.dy) || t.gb % per || t.gn % per)) vec = 0;
  }
  return vec;
}

}  // namespace
}  // namespace ncn

extern "C" {

int ncn_qk_rotary(const void* q, const void* k, const float* wq, const float* wk, const double* freqs, const int64_t* positions,
                  int64_t positions_stride, int64_t start, void* yq, void* yk, const int64_t* strides, int64_t B, int64_t N, int64_t E,
                  int64_t Ek, int n_head, int64_t R, int interleaved, double eps, double magnitude, int inverse, int dtype, void* stream) {
  RotaryParams p{};
  int rc = rotary_params(p, freqs, positions, positions_stride, start, B, N, E, Ek, n_head, R, interleaved, eps, magnitude, dtype);
  if (rc != NCN_OK || B == 0 || N == 0) return rc;
  if (!q || !yq || (Ek && (!k || !yk)) || (Ek && (wq == nullptr) != (wk == nullptr))) return NCN_ERR_NULL;
  if (inverse && wq) return NCN_ERR_UNSUPPORTED;
  DevInfo dev;
  if ((rc = get_dev(dev)) != NCN_OK) return rc;
  const long long s[4] = {strides ? strides[0] : N * E, strides ? strides[1] : E, strides ? strides[2] : N * Ek, strides ? strides[3] : Ek};
  p.t[0].x = q, p.t[0].out = yq, p.t[0].w = wq, p.t[0].sb = s[0], p.t[0].sn = s[1];
  p.t[1].x = k, p.t[1].out = yk, p.t[1].w = wk, p.t[1].sb = s[2], p.t[1].sn = s[3];
  p.backward = inverse != 0;
  p.vec = set_vec(p, dtype);
  const int grid = rotary_plan(p, dev.sms);
  const cudaError_t e = launch_rotary(p, dtype, grid, (cudaStream_t)stream);
  return e == cudaSuccess ? NCN_OK : cuda_fail(e);
}

size_t ncn_qk_norm_rotary_workspace_bytes(int64_t B, int64_t N, int64_t E, int n_head) {
  if (B <= 0 || N <= 0 || E <= 0 || n_head <= 0 || E % n_head != 0) return 0;
  // a row of sums per CTA, of which there are no more than heads of queries
  const long long rows = B > kRotaryMostCtas || N > kRotaryMostCtas || B * N > kRotaryMostCtas ? kRotaryMostCtas : B * N;
  const long long ctas = rows * n_head > kRotaryMostCtas ? kRotaryMostCtas : rows * n_head;
  return (size_t)ctas * 2 * (E / n_head) * sizeof(float);
}

int ncn_qk_norm_rotary_bwd(const void* q, const void* k, const float* wq, const float* wk, const double* freqs, const int64_t* positions,
                           int64_t positions_stride, int64_t start, const void* dyq, const void* dyk, void* dq, void* dk, float* dwq,
                           float* dwk, const int64_t* strides, void* workspace, size_t workspace_bytes, int64_t B, int64_t N, int64_t E,
                           int64_t Ek, int n_head, int64_t R, int interleaved, double eps, double magnitude, int dtype, void* stream) {
  RotaryParams p{};
  int rc = rotary_params(p, freqs, positions, positions_stride, start, B, N, E, Ek, n_head, R, interleaved, eps, magnitude, dtype);
  if (rc != NCN_OK) return rc;
  if (B == 0 || N == 0) return NCN_ERR_SHAPE;
  if (!q || !wq || !dyq || !dq || !dwq || (Ek && (!k || !wk || !dyk || !dk || !dwk))) return NCN_ERR_NULL;
  if (!workspace || workspace_bytes < ncn_qk_norm_rotary_workspace_bytes(B, N, E, n_head)) return NCN_ERR_WORKSPACE;
  DevInfo dev;
  if ((rc = get_dev(dev)) != NCN_OK) return rc;
  const long long c[8] = {N * E, E, N * Ek, Ek, N * E, E, N * Ek, Ek};
  long long s[8];
  for (int i = 0; i < 8; ++i) s[i] = strides ? strides[i] : c[i];
  p.t[0].x = q, p.t[0].dy = dyq, p.t[0].out = dq, p.t[0].w = wq, p.t[0].sb = s[0], p.t[0].sn = s[1], p.t[0].gb = s[4], p.t[0].gn = s[5];
  p.t[1].x = k, p.t[1].dy = dyk, p.t[1].out = dk, p.t[1].w = wk, p.t[1].sb = s[2], p.t[1].sn = s[3], p.t[1].gb = s[6], p.t[1].gn = s[7];
  p.backward = 1;
  p.partial = static_cast<float*>(workspace);
  p.vec = set_vec(p, dtype);
  const int grid = rotary_plan(p, dev.sms);
  const cudaError_t e = launch_rotary(p, dtype, grid, (cudaStream_t)stream);
  if (e != cudaSuccess) return cuda_fail(e);
  const float* partials[2] = {p.partial, p.partial + (size_t)grid * p.d};
  const int rows[2] = {grid, grid};
  float* const out[2] = {dwq, dwk};
  return ncn_reduce_partials(partials, rows, out, Ek ? 2 : 1, p.d, stream);
}

}  // extern "C"
