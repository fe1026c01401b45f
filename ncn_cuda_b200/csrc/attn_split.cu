// Windowed attention in fp32 on the tensor cores: every operand as the sum of two tf32 numbers, three products for one.
//
//   x = hi + lo, hi: x rounded to 11 bits, lo: what is left (12 bits and a sign, of which the products use 11)
//   a b = hi hi + (hi lo + lo hi), the second sum in accumulators of its own; lo lo, 2^-22 of the product at most, is left out
// A product is off by 2^-20.4 of its size at most (2^-22 for each lo that loses its last bit and for lo lo) and by 2^-24 as a rule, as
// far as fp32 additions one after the other are: results are 1.0 to 1.7 times as far from the exact ones as with fp32 products.
// The matrix unit may cut where fp32 additions round: a sum therefore runs over one tile in it, and tiles are added in fp32.
//
// A CTA of 4 warps owns 64 rows (queries; in the backward of the keys: keys), 16 a warp, and walks the tiles of the other side in shared
// memory; two or more CTAs fit on an SM.  Scores never leave registers: the accumulators' columns 2 c and 2 c + 1 of a lane are the
// entries c and c + 4 of the next product's left operand, if its rows are taken in that order (the order of a sum's terms is free).
// A row in shared memory is DP + 4 floats (DP: the head size rounded up to 32, 48, 64, 80, 96 or 128): the 32 lanes of an operand's load hit 32 different banks both ways.  While one tile of
// a pair is worked on, the other's successor is on its way (cp.async).
//
// Measured, 2 x 4096 positions of 8 heads, windows of 1024: heads of 128 forward 616 us (48.8 TFLOP/s), dq 949 (47.5), dk and dv 1262
// (47.7); heads of 80 401, 634, 828 (in tiles of 96 features 472, 733, 983); heads of 64 317, 462, 624 (48); as fp32 products on the FMA pipes
// (attn_simt.cu, when it had tiles of these sizes) 928, 1332, 1761 and 453, 649, 862.  The matrix unit is 50 to 56 % busy (three
// products: 275 TFLOP/s of tf32 would be 92 here); more CTAs, smaller tiles and more independent accumulators change nothing.
#include "attn_common.cuh"
#include "ncn_common.cuh"

namespace ncn {
namespace {

constexpr int kOwn = 64, kCta = 128;
// Rows of the other side's tiles: the backward holds two tiles of its own, and 32 let a second CTA fit beside it where heads are large.
// CTAs per SM that the registers leave room for.  (Heads of 128 forward with 32 rows and three CTAs 642 us, as below 616; heads of
// 64 backward with 32 rows and three CTAs 478 + 641, as below 462 + 624.)
constexpr int kFwdRows = 64;
template <int DP> constexpr int bwd_rows() { return DP > 64 ? 32 : 64; }
template <int DP> constexpr int fwd_ctas() { return DP > 96 ? 2 : 3; }
template <int DP> constexpr int bwd_ctas() { return DP > 32 ? 2 : 3; }

struct Parts {
  uint32_t hi, lo;
};
__device__ __forceinline__ Parts split(float x) {
  Parts p;
  p.hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  p.lo = __float_as_uint(x - __uint_as_float(p.hi));
  return p;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ROWS x d of `src` -> tile [ROWS][DP + 4], asynchronously where rows may be read 16 bytes at a time; rows that `rows` does not
// have and features beyond d are zero.
template <int DP, int ROWS>
__device__ __forceinline__ void send_for(float* dst, const float* src, long long stride, Rows rows, int d, int vec) {
  constexpr int PER = DP / 4;
  if (vec) {
#pragma unroll 4
    for (int e = threadIdx.x; e < ROWS * PER; e += kCta) {
      const int r = e / PER, c = e % PER * 4;
      const bool ok = rows.has(r) && c < d;
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst + r * (DP + 4) + c);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(ok ? src + r * stride + c : src), "r"(ok ? 16 : 0) : "memory");
    }
  } else {
    for (int e = threadIdx.x; e < ROWS * DP; e += kCta) {
      const int r = e / DP, c = e % DP;
      dst[r * (DP + 4) + c] = rows.has(r) && c < d ? src[r * stride + c] : 0.f;
    }
  }
}
__device__ __forceinline__ void sent() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all that was sent for has arrived, but for the last LATER groups
template <int LATER> __device__ __forceinline__ void arrived() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory");
  __syncthreads();
}

// s = A B^T over the features: A the warp's 16 rows, B 8 NB rows
template <int DP, int NB>
__device__ __forceinline__ void rows_by_rows(const float* A, const float* B, float (&s)[NB][4]) {
  const int lane = threadIdx.x % 32, g8 = lane / 4, c4 = lane % 4;
  const float *a_at = A + g8 * (DP + 4) + c4, *b_at = B + g8 * (DP + 4) + c4;
  float small[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[n][i] = small[n][i] = 0.f;
#pragma unroll 2
  for (int k = 0; k < DP; k += 8) {
    uint32_t ah[4], al[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Parts p = split(a_at[k + (i & 1) * 8 * (DP + 4) + (i >> 1) * 4]);
      ah[i] = p.hi, al[i] = p.lo;
    }
    Parts b[NB][2];  // (products that follow each other go to different accumulators)
#pragma unroll
    for (int n = 0; n < NB; ++n) b[n][0] = split(b_at[8 * n * (DP + 4) + k]), b[n][1] = split(b_at[8 * n * (DP + 4) + k + 4]);
#pragma unroll
    for (int n = 0; n < NB; ++n) mma(small[n], al, b[n][0].hi, b[n][1].hi);
#pragma unroll
    for (int n = 0; n < NB; ++n) mma(s[n], ah, b[n][0].hi, b[n][1].hi);
#pragma unroll
    for (int n = 0; n < NB; ++n) mma(small[n], ah, b[n][0].lo, b[n][1].lo);
  }
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[n][i] += small[n][i];
}

// acc = acc keep + w V: w the 16 x 8 KB results of a product as they lie in the accumulators, V 8 KB rows; keep: of rows g8 and g8 + 8
template <int DP, int KB>
__device__ __forceinline__ void add_rows_by_cols(const float (&w)[KB][4], const float* V, float keep0, float keep1, float (&acc)[DP / 8][4]) {
  const int lane = threadIdx.x % 32, g8 = lane / 4, c4 = lane % 4;
  const float* at = V + 2 * c4 * (DP + 4) + g8;
  uint32_t wh[KB][4], wl[KB][4];
#pragma unroll
  for (int k = 0; k < KB; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // entries (row g8, 2 c4), (g8 + 8, 2 c4), (g8, 2 c4 + 1), (g8 + 8, 2 c4 + 1)
      const Parts p = split(w[k][(i & 1) * 2 + (i >> 1)]);
      wh[k][i] = p.hi, wl[k][i] = p.lo;
    }
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    float big[4] = {}, small[4] = {}, other[4] = {};
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const Parts b0 = split(at[8 * k * (DP + 4) + 8 * n]), b1 = split(at[(8 * k + 1) * (DP + 4) + 8 * n]);
      mma(small, wl[k], b0.hi, b1.hi);
      mma(big, wh[k], b0.hi, b1.hi);
      mma(other, wh[k], b0.lo, b1.lo);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = fmaf(acc[n][i], i < 2 ? keep0 : keep1, big[i] + (small[i] + other[i]));
  }
}

// over the four lanes of a row
__device__ __forceinline__ float max4(float x) {
  x = fmaxf(x, __shfl_xor_sync(~0u, x, 1));
  return fmaxf(x, __shfl_xor_sync(~0u, x, 2));
}
__device__ __forceinline__ float sum4(float x) {
  x += __shfl_xor_sync(~0u, x, 1);
  return x + __shfl_xor_sync(~0u, x, 2);
}

template <int DP>
__global__ void __launch_bounds__(kCta, fwd_ctas<DP>()) attn_split_fwd_kernel(const AttnParams p) {
  wait_for_inputs();
  constexpr int BN = kFwdRows, NB = BN / 8;
  extern __shared__ __align__(16) float sm[];
  float *Q = sm, *K = Q + kOwn * (DP + 4), *V = K + BN * (DP + 4);
  const Block at_block = block_of(p.H, (p.Nq + kOwn - 1) / kOwn);
  const int i0 = at_block.last_first * kOwn, h = at_block.head, b = at_block.b, hk = h / p.G;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g8 = lane / 4, c4 = lane % 4;
  const RowGeom g = row_geom(p, b);
  const KeyTiles kt = key_tiles<BN>(p, g, i0, i0 + kOwn);
  const SeenKeys seen = seen_keys(p, g);
  const float* q = static_cast<const float*>(p.q) + b * p.sq_b + i0 * p.sq_n + (long long)h * p.d;
  const float* k = static_cast<const float*>(p.k) + b * p.sk_b + (long long)hk * p.d;
  const float* v = static_cast<const float*>(p.v) + b * p.sv_b + (long long)hk * p.d;
  auto send_keys = [&](int it) {
    const int k0 = kt.tile(it) * BN;
    send_for<DP, BN>(K, k + k0 * p.sk_n, p.sk_n, rows_seen(seen, k0), p.d, p.vec);
  };
  auto send_values = [&](int it) {
    const int k0 = kt.tile(it) * BN;
    send_for<DP, BN>(V, v + k0 * p.sv_n, p.sv_n, rows_seen(seen, k0), p.d, p.vec);
  };
  float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  const int n_tiles = kt.count();
  if (n_tiles) {
    send_for<DP, kOwn>(Q, q, p.sq_n, rows_between(0, p.Nq - i0), p.d, p.vec);
    send_keys(0);
    sent();
    send_values(0);
    sent();
  }
  for (int it = 0; it < n_tiles; ++it) {
    const int k0 = kt.tile(it) * BN;
    arrived<1>();
    float s[NB][4];
    rows_by_rows<DP, NB>(Q + 16 * warp * (DP + 4), K, s);
    __syncthreads();
    if (it + 1 < n_tiles) send_keys(it + 1);
    sent();
    const int pos = g.start + i0 + 16 * warp + g8;
    if (!sees_all(p, g, i0, kOwn, k0, BN)) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!sees(p, g.ctx, pos + (i >> 1) * 8, k0 + 8 * n + 2 * c4 + (i & 1))) s[n][i] = -INFINITY;
    }
    float keep[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < NB; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
      const float now = fmaxf(m[r], max4(mx));
      const float ref = now == -INFINITY ? 0.f : now * p.scale_log2;
      keep[r] = m[r] == -INFINITY ? 0.f : ex2(m[r] * p.scale_log2 - ref);
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 2 * r; i < 2 * r + 2; ++i) {
          s[n][i] = s[n][i] == -INFINITY ? 0.f : ex2(fmaf(s[n][i], p.scale_log2, -ref));
          sum += s[n][i];
        }
      l[r] = l[r] * keep[r] + sum4(sum);
      m[r] = now;
    }
    arrived<1>();
    add_rows_by_cols<DP, NB>(s, V, keep[0], keep[1], o);
    __syncthreads();
    if (it + 1 < n_tiles) send_values(it + 1);
    sent();
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int qi = i0 + 16 * warp + g8 + 8 * r;
    if (qi >= p.Nq) continue;
    const int pos = g.start + qi;
    const bool some = pos >= 0 && pos < g.ctx;  // (it sees its own place; scores that are all minus infinity leave l = 0, and NaN)
    const float inv = 1.f / l[r];
    float* y = static_cast<float*>(p.y) + ((long long)b * p.Nq + qi) * p.H * p.d + (long long)h * p.d;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = 8 * n + 2 * c4 + i;
        if (c < p.d) y[c] = some ? o[n][2 * r + i] * inv : 0.f;
      }
    if (p.lse && c4 == 0) p.lse[((long long)b * p.H + h) * p.Nqp + qi] = some ? m[r] * p.scale_log2 + log2f(l[r]) : INFINITY;
  }
}

// Gradient of the queries; also leaves delta = sum(dy * y) of its rows for the backward of the keys.
template <int DP>
__global__ void __launch_bounds__(kCta, bwd_ctas<DP>()) attn_split_dq_kernel(const AttnParams p) {
  wait_for_inputs();
  constexpr int BN = bwd_rows<DP>(), NB = BN / 8;
  extern __shared__ __align__(16) float sm[];
  float *Q = sm, *dO = Q + kOwn * (DP + 4), *K = dO + kOwn * (DP + 4), *V = K + BN * (DP + 4);
  const Block at_block = block_of(p.H, (p.Nq + kOwn - 1) / kOwn);
  const int i0 = at_block.last_first * kOwn, h = at_block.head, b = at_block.b, hk = h / p.G;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g8 = lane / 4, c4 = lane % 4, row0 = 16 * warp;
  const RowGeom g = row_geom(p, b);
  const KeyTiles kt = key_tiles<BN>(p, g, i0, i0 + kOwn);
  const SeenKeys seen = seen_keys(p, g);
  const float* q = static_cast<const float*>(p.q) + b * p.sq_b + i0 * p.sq_n + (long long)h * p.d;
  const float* dy = static_cast<const float*>(p.dy) + b * p.sdy_b + i0 * p.sdy_n + (long long)h * p.d;
  const float* k = static_cast<const float*>(p.k) + b * p.sk_b + (long long)hk * p.d;
  const float* v = static_cast<const float*>(p.v) + b * p.sv_b + (long long)hk * p.d;
  const int r_lo = max(0, -(g.start + i0)), r_hi = min(p.Nq, g.ctx - g.start) - i0;  // rows that are not padding
  auto send_keys = [&](int it) {
    const int k0 = kt.tile(it) * BN;
    send_for<DP, BN>(K, k + k0 * p.sk_n, p.sk_n, rows_seen(seen, k0), p.d, p.vec);
  };
  auto send_values = [&](int it) {
    const int k0 = kt.tile(it) * BN;
    send_for<DP, BN>(V, v + k0 * p.sv_n, p.sv_n, rows_seen(seen, k0), p.d, p.vec);
  };
  const int n_tiles = kt.count();
  send_for<DP, kOwn>(dO, dy, p.sdy_n, rows_between(r_lo, r_hi), p.d, p.vec);
  send_for<DP, kOwn>(Q, q, p.sq_n, rows_between(r_lo, r_hi), p.d, p.vec);
  if (n_tiles) send_values(0);
  sent();
  if (n_tiles) send_keys(0);
  sent();
  arrived<1>();
  float acc[DP / 8][4], lse[2], delta[2];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = row0 + g8 + 8 * r, qi = i0 + row;
    const long long at = ((long long)b * p.H + h) * p.Nqp + qi;
    const bool live = row >= r_lo && row < r_hi;
    lse[r] = live ? p.lse[at] : INFINITY;
    float sum = 0.f;
    if (live) {
      const float* y = static_cast<const float*>(p.y_in) + ((long long)b * p.Nq + qi) * p.H * p.d + (long long)h * p.d;
      for (int c = c4; c < p.d; c += 4) sum = fmaf(dO[row * (DP + 4) + c], y[c], sum);
    }
    delta[r] = sum4(sum);
    if (c4 == 0 && qi < p.Nq) p.delta[at] = delta[r];
  }
  for (int it = 0; it < n_tiles; ++it) {
    const int k0 = kt.tile(it) * BN;
    if (it) arrived<1>();
    float s[NB][4], dp[NB][4];
    rows_by_rows<DP, NB>(dO + row0 * (DP + 4), V, dp);
    __syncthreads();
    if (it + 1 < n_tiles) send_values(it + 1);
    sent();
    arrived<1>();
    rows_by_rows<DP, NB>(Q + row0 * (DP + 4), K, s);
    const bool all = sees_all(p, g, i0, kOwn, k0, BN);
    const int pos = g.start + i0 + row0 + g8;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = ex2(fmaf(s[n][i], p.scale_log2, -lse[i >> 1]));
        s[n][i] = all || sees(p, g.ctx, pos + (i >> 1) * 8, k0 + 8 * n + 2 * c4 + (i & 1)) ? w * (dp[n][i] - delta[i >> 1]) : 0.f;
      }
    add_rows_by_cols<DP, NB>(s, K, 1.f, 1.f, acc);
    __syncthreads();
    if (it + 1 < n_tiles) send_keys(it + 1);
    sent();
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int qi = i0 + row0 + g8 + 8 * r;
    if (qi >= p.Nq) continue;
    float* dq = static_cast<float*>(p.dq) + ((long long)b * p.Nq + qi) * p.H * p.d + (long long)h * p.d;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = 8 * n + 2 * c4 + i;
        if (c < p.d) dq[c] = acc[n][2 * r + i] * p.scale;
      }
  }
}

// Gradients of the keys and values.  The heads of a group are walked one after the other by the same CTA, so that their sum has
// one order.
template <int DP>
__global__ void __launch_bounds__(kCta, bwd_ctas<DP>()) attn_split_dkv_kernel(const AttnParams p) {
  wait_for_inputs();
  constexpr int BN = bwd_rows<DP>(), NB = BN / 8;
  extern __shared__ __align__(16) float sm[];
  float *K = sm, *V = K + kOwn * (DP + 4), *Q = V + kOwn * (DP + 4), *dO = Q + BN * (DP + 4);
  float *lse_s = dO + BN * (DP + 4), *del_s = lse_s + 2 * BN;  // of this tile and of the next one
  const Block at_block = block_of(p.Hk, (p.Nk + kOwn - 1) / kOwn + p.sink_tiles * p.chunks);
  const int hk = at_block.head, b = at_block.b, lane = threadIdx.x % 32, warp = threadIdx.x / 32, g8 = lane / 4, c4 = lane % 4, row0 = 16 * warp;
  const RowGeom g = row_geom(p, b);
  const KeyItem it = key_item<kOwn, BN>(p, g, at_block.first_last);
  const int k0 = it.tile * kOwn, end = min(g.ctx, g.start + p.Nq);  // (of the queries: the last tile's rows behind them see nothing)
  const float* k = static_cast<const float*>(p.k) + b * p.sk_b + k0 * p.sk_n + (long long)hk * p.d;
  const float* v = static_cast<const float*>(p.v) + b * p.sv_b + k0 * p.sv_n + (long long)hk * p.d;
  auto place = [&](int e, int& h, int& i0, int& r_lo, int& r_hi) {
    h = hk * p.G + e / it.tiles, i0 = (it.first + e % it.tiles) * BN;
    r_lo = max(0, -(g.start + i0)), r_hi = min(p.Nq, g.ctx - g.start) - i0;
  };
  auto send_queries = [&](int e) {
    int h, i0, r_lo, r_hi;
    place(e, h, i0, r_lo, r_hi);
    send_for<DP, BN>(Q, static_cast<const float*>(p.q) + b * p.sq_b + i0 * p.sq_n + (long long)h * p.d, p.sq_n, rows_between(r_lo, r_hi), p.d, p.vec);
  };
  auto send_cotangents = [&](int e, int buffer) {  // and what belongs to their rows
    int h, i0, r_lo, r_hi;
    place(e, h, i0, r_lo, r_hi);
    send_for<DP, BN>(dO, static_cast<const float*>(p.dy) + b * p.sdy_b + i0 * p.sdy_n + (long long)h * p.d, p.sdy_n, rows_between(r_lo, r_hi), p.d, p.vec);
    if (threadIdx.x < BN) {
      const int r = threadIdx.x;
      const long long at = ((long long)b * p.H + h) * p.Nqp + i0 + r;
      const bool live = r >= r_lo && r < r_hi;
      lse_s[buffer * BN + r] = live ? p.lse[at] : INFINITY;
      del_s[buffer * BN + r] = live ? p.delta[at] : 0.f;
    }
  };
  float dk[DP / 8][4], dv[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) dk[n][i] = dv[n][i] = 0.f;
  if (it.begin < it.end) {
    send_for<DP, kOwn>(K, k, p.sk_n, rows_between(0, g.ctx - k0), p.d, p.vec);
    send_for<DP, kOwn>(V, v, p.sv_n, rows_between(0, g.ctx - k0), p.d, p.vec);
    send_cotangents(it.begin, it.begin & 1);
    sent();
    send_queries(it.begin);
    sent();
  }
  for (int e = it.begin; e < it.end; ++e) {
    int h, i0, r_lo, r_hi;
    place(e, h, i0, r_lo, r_hi);
    const float *lse = lse_s + (e & 1) * BN, *delta = del_s + (e & 1) * BN;
    float s[NB][4], dp[NB][4];
    arrived<1>();
    rows_by_rows<DP, NB>(V + row0 * (DP + 4), dO, dp);
    arrived<0>();
    rows_by_rows<DP, NB>(K + row0 * (DP + 4), Q, s);
    const bool all = sees_all(p, g, i0, BN, k0, kOwn);
    const int key = k0 + row0 + g8;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 8 * n + 2 * c4 + (i & 1);
        float w = ex2(fmaf(s[n][i], p.scale_log2, -lse[c])), t = w * (dp[n][i] - delta[c]);
        if (!all && !sees(p, end, g.start + i0 + c, key + (i >> 1) * 8)) w = t = 0.f;
        s[n][i] = w, dp[n][i] = t;
      }
    add_rows_by_cols<DP, NB>(s, dO, 1.f, 1.f, dv);
    __syncthreads();
    if (e + 1 < it.end) send_cotangents(e + 1, (e + 1) & 1);
    sent();
    add_rows_by_cols<DP, NB>(dp, Q, 1.f, 1.f, dk);
    __syncthreads();
    if (e + 1 < it.end) send_queries(e + 1);
    sent();
  }
  const bool sinks = p.chunks > 0 && it.tile < p.sink_tiles;
  float* part = sinks ? part_of(p, b, hk, it.tile, it.chunk < 0 ? p.chunks : it.chunk) : nullptr;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = row0 + g8 + 8 * half, key = k0 + r;
    if (key >= p.Nk) continue;
    const bool partial = sinks && key < p.n_sink;
    if (it.chunk >= 0 && !partial) continue;
    const long long at = ((long long)b * p.Nk + key) * p.Hk * p.d + (long long)hk * p.d;
    float* const to_k = partial ? part + r * p.d : static_cast<float*>(p.dk) + at;
    float* const to_v = partial ? part + (p.sink_rows + r) * p.d : static_cast<float*>(p.dv) + at;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = 8 * n + 2 * c4 + i;
        if (c >= p.d) continue;
        to_k[c] = dk[n][2 * half + i] * p.scale;
        to_v[c] = dv[n][2 * half + i];
      }
  }
}

template <int DP>
cudaError_t run_fwd(const AttnParams& p, cudaStream_t st) {
  static SmemGrant grant;
  constexpr size_t smem = sizeof(float) * (kOwn + 2 * kFwdRows) * (DP + 4);
  const cudaError_t e = grant_smem(grant, attn_split_fwd_kernel<DP>, smem);
  if (e != cudaSuccess) return e;
  return launch_behind(attn_split_fwd_kernel<DP>, dim3((unsigned)((p.Nq + kOwn - 1) / kOwn * p.H * p.B)), kCta, smem, st, p);
}
template <int DP>
cudaError_t run_bwd(const AttnParams& p, cudaStream_t st) {
  static SmemGrant g1, g2;
  constexpr int BN = bwd_rows<DP>();
  constexpr size_t smem = sizeof(float) * ((2 * kOwn + 2 * BN) * (DP + 4) + 4 * BN);
  cudaError_t e = grant_smem(g1, attn_split_dq_kernel<DP>, smem);
  if (e == cudaSuccess) e = grant_smem(g2, attn_split_dkv_kernel<DP>, smem);
  if (e != cudaSuccess) return e;
  e = launch_behind(attn_split_dq_kernel<DP>, dim3((unsigned)((p.Nq + kOwn - 1) / kOwn * p.H * p.B)), kCta, smem, st, p);
  if (e != cudaSuccess || p.Nk == 0) return e;
  const int items = (p.Nk + kOwn - 1) / kOwn + p.sink_tiles * p.chunks;
  return launch_behind(attn_split_dkv_kernel<DP>, dim3((unsigned)(items * p.Hk * p.B)), kCta, smem, st, p);
}

}  // namespace

cudaError_t launch_attn_split_fwd(const AttnParams& p, cudaStream_t st) {
  return p.d <= 32   ? run_fwd<32>(p, st)
         : p.d <= 48 ? run_fwd<48>(p, st)
         : p.d <= 64 ? run_fwd<64>(p, st)
         : p.d <= 80 ? run_fwd<80>(p, st)
         : p.d <= 96 ? run_fwd<96>(p, st)
                     : run_fwd<128>(p, st);
}
cudaError_t launch_attn_split_bwd(const AttnParams& p, cudaStream_t st) {
  return p.d <= 32   ? run_bwd<32>(p, st)
         : p.d <= 48 ? run_bwd<48>(p, st)
         : p.d <= 64 ? run_bwd<64>(p, st)
         : p.d <= 80 ? run_bwd<80>(p, st)
         : p.d <= 96 ? run_bwd<96>(p, st)
                     : run_bwd<128>(p, st);
}

}  // namespace ncn
