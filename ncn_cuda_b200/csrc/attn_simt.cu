// Windowed attention on the FMA pipes: fp32 with heads of more than 128 or at most 16 features, and bf16 with head sizes or alignments that
// the tensor-core kernels do not take.  (fp32 between these: attn_split.cu.)
//
// A CTA of 256 threads owns 64 rows (queries; in the backward of the keys: keys) and walks the tiles of the other side.  Thread
// (ty, tx) of 16 x 16 holds rows 4 ty .. 4 ty + 3.  Tiles are fp32 in shared memory whatever the storage type; a row is DP + 4
// floats, so that eight lanes that read eight rows 16 bytes at a time hit 32 different banks.  DP is the head size, rounded up to
// 32, 64, 96, 128 or 256 (fp32: 32 or 256): without 96, heads of 72 to 96 did a third more products on zeros.
//
// What bounds it: the reads of shared memory.  A product over 4 features takes a thread 8 reads of 16 bytes, which return to a
// warp in 32 cycles, for 64 FMAs, which take 16: half the FMA rate (36 of 72 TFLOP/s) is the most this split can give.  Measured:
// heads of 256, 2 x 2048 positions of 8 heads, windows of 512: fp32 forward 568 us (26.5 TFLOP/s), dq 847 (26.6), dk and dv 1076 (28.0), bf16
// 571, 846, 1046; fp32 heads of 16, 2 x 4096 positions of 8 heads, windows of 1024: 281, 374, 521 us (13 to 15 TFLOP/s: half of a tile's
// features are zeros); bf16 heads of 12, the same: 321, 433, 562.  Tiles of 8 rows a thread would
// lower the reads by a quarter, but with large heads the backward's four tiles then no longer fit in shared memory.
#include "attn_common.cuh"
#include "ncn_common.cuh"

namespace ncn {
namespace {

constexpr int kOwn = 64;
template <int DP> constexpr int other_rows() { return DP > 128 ? 32 : 64; }

// ROWS x d of `src` (row stride in elements) -> fp32 tile [ROWS][DP + 4]; rows that `rows` does not have and features beyond d are zero.
// All of a thread's loads are under way at once: one after the other they took longer than the tile's arithmetic.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void load_tile(float* dst, const T* src, long long stride, Rows rows, int d, int vec) {
  constexpr int V = 16 / sizeof(T), PER = DP / V, COUNT = ROWS * PER, EACH = (COUNT + 255) / 256;
  if (vec) {
    uint4 raw[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int e = threadIdx.x + 256 * i, r = e / PER, c = e % PER * V;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (e < COUNT && rows.has(r) && c < d) raw[i] = *reinterpret_cast<const uint4*>(src + r * stride + c);  // (d is a multiple of V)
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int e = threadIdx.x + 256 * i, r = e / PER, c = e % PER * V;
      if (e >= COUNT) break;
      const T* t = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
      for (int x = 0; x < V; x += 4) *reinterpret_cast<float4*>(dst + r * (DP + 4) + c + x) = make_float4(to_f(t[x]), to_f(t[x + 1]), to_f(t[x + 2]), to_f(t[x + 3]));
    }
  } else {
    for (int e = threadIdx.x; e < ROWS * DP; e += 256) {
      const int r = e / DP, c = e % DP;
      dst[r * (DP + 4) + c] = rows.has(r) && c < d ? to_f(src[r * stride + c]) : 0.f;
    }
  }
}

// acc[i][j] += sum over features of A[4 ty + i][.] * B[tx + 16 j][.]
template <int DP, int CJ>
__device__ __forceinline__ void rows_by_rows(const float* A, const float* B, float (&acc)[4][CJ]) {
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
#pragma unroll 4
  for (int c = 0; c < DP; c += 4) {
    float4 a[4], b[CJ];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(A + (4 * ty + i) * (DP + 4) + c);
#pragma unroll
    for (int j = 0; j < CJ; ++j) b[j] = *reinterpret_cast<const float4*>(B + (tx + 16 * j) * (DP + 4) + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < CJ; ++j) {
        acc[i][j] = fmaf(a[i].x, b[j].x, acc[i][j]);
        acc[i][j] = fmaf(a[i].y, b[j].y, acc[i][j]);
        acc[i][j] = fmaf(a[i].z, b[j].z, acc[i][j]);
        acc[i][j] = fmaf(a[i].w, b[j].w, acc[i][j]);
      }
  }
}

// A thread's features of a row: VW at a time, VW * tx + 16 VW m
template <int DP> constexpr int vec_width() { return DP % 64 == 0 ? 4 : 2; }
template <int DP> __device__ __forceinline__ int feature_of(int e) {
  constexpr int VW = vec_width<DP>();
  return VW * (threadIdx.x % 16) + 16 * VW * (e / VW) + e % VW;
}

// acc[i][.] += sum over n of P[4 ty + i][n] * V[n][features of the thread]; P [64][BN + 4]
template <int DP, int BN>
__device__ __forceinline__ void rows_by_cols(const float* P, const float* V, float (&acc)[4][DP / 16]) {
  constexpr int VW = vec_width<DP>();
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
#pragma unroll 2
  for (int n = 0; n < BN; n += 4) {
    float4 pr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) pr[i] = *reinterpret_cast<const float4*>(P + (4 * ty + i) * (BN + 4) + n);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float x[DP / 16];
#pragma unroll
      for (int m = 0; m < DP / 16; m += VW) {
        const float* at = V + (n + u) * (DP + 4) + VW * tx + 16 * m;
        if constexpr (VW == 4) {
          const float4 t = *reinterpret_cast<const float4*>(at);
          x[m] = t.x, x[m + 1] = t.y, x[m + 2] = t.z, x[m + 3] = t.w;
        } else {
          const float2 t = *reinterpret_cast<const float2*>(at);
          x[m] = t.x, x[m + 1] = t.y;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = u == 0 ? pr[i].x : u == 1 ? pr[i].y : u == 2 ? pr[i].z : pr[i].w;
#pragma unroll
        for (int m = 0; m < DP / 16; ++m) acc[i][m] = fmaf(w, x[m], acc[i][m]);
      }
    }
  }
}

__device__ __forceinline__ float max16(float x) {
#pragma unroll
  for (int s = 8; s; s >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, s));
  return x;
}
__device__ __forceinline__ float sum16(float x) {
#pragma unroll
  for (int s = 8; s; s >>= 1) x += __shfl_xor_sync(~0u, x, s);
  return x;
}

template <typename T, int DP>
__global__ void __launch_bounds__(256) attn_simt_fwd_kernel(const AttnParams p) {
  wait_for_inputs();
  constexpr int BN = other_rows<DP>(), CJ = BN / 16;
  extern __shared__ float sm[];
  float *Q = sm, *K = Q + kOwn * (DP + 4), *V = K + BN * (DP + 4), *P = V + BN * (DP + 4);
  const Block at_block = block_of(p.H, (p.Nq + kOwn - 1) / kOwn);
  const int i0 = at_block.last_first * kOwn, h = at_block.head, b = at_block.b, hk = h / p.G;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const RowGeom g = row_geom(p, b);
  const KeyTiles kt = key_tiles<BN>(p, g, i0, i0 + kOwn);
  const SeenKeys seen = seen_keys(p, g);
  const T* q = static_cast<const T*>(p.q) + b * p.sq_b + i0 * p.sq_n + (long long)h * p.d;
  const T* k = static_cast<const T*>(p.k) + b * p.sk_b + (long long)hk * p.d;
  const T* v = static_cast<const T*>(p.v) + b * p.sv_b + (long long)hk * p.d;
  float o[4][DP / 16], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) o[i][e] = 0.f;
  }
  const int n = kt.count();
  if (n) load_tile<T, DP, kOwn>(Q, q, p.sq_n, rows_between(0, p.Nq - i0), p.d, p.vec);
  for (int it = 0; it < n; ++it) {
    const int k0 = kt.tile(it) * BN;
    __syncthreads();
    load_tile<T, DP, BN>(K, k + k0 * p.sk_n, p.sk_n, rows_seen(seen, k0), p.d, p.vec);
    load_tile<T, DP, BN>(V, v + k0 * p.sv_n, p.sv_n, rows_seen(seen, k0), p.d, p.vec);
    __syncthreads();
    float s[4][CJ] = {};
    rows_by_rows<DP, CJ>(Q, K, s);
    if (!sees_all(p, g, i0, kOwn, k0, BN)) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < CJ; ++j)
          if (!sees(p, g.ctx, g.start + i0 + 4 * ty + i, k0 + tx + 16 * j)) s[i][j] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < CJ; ++j) mx = fmaxf(mx, s[i][j]);
      const float now = fmaxf(m[i], max16(mx));
      const float ref = now == -INFINITY ? 0.f : now * p.scale_log2;
      const float keep = m[i] == -INFINITY ? 0.f : ex2(m[i] * p.scale_log2 - ref);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < CJ; ++j) {
        const float w = s[i][j] == -INFINITY ? 0.f : ex2(fmaf(s[i][j], p.scale_log2, -ref));
        P[(4 * ty + i) * (BN + 4) + tx + 16 * j] = w;
        sum += w;
      }
      l[i] = l[i] * keep + sum16(sum);
      m[i] = now;
#pragma unroll
      for (int e = 0; e < DP / 16; ++e) o[i][e] *= keep;
    }
    __syncwarp();  // a row of P is written and read by the same half warp
    rows_by_cols<DP, BN>(P, V, o);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int qi = i0 + 4 * ty + i;
    if (qi >= p.Nq) continue;
    const int pos = g.start + qi;
    const bool some = pos >= 0 && pos < g.ctx;  // (it sees its own place; scores that are all minus infinity leave l = 0, and NaN)
    const float inv = 1.f / l[i];
    const long long at = ((long long)b * p.Nq + qi) * p.H * p.d + (long long)h * p.d;
    T *y = static_cast<T*>(p.y) + at, *rest = sizeof(T) == 2 && p.rest ? reinterpret_cast<T*>(p.rest) + at : nullptr;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) {
      const int c = feature_of<DP>(e);
      if (c < p.d) put_rest(y + c, rest ? rest + c : nullptr, some ? o[i][e] * inv : 0.f);
    }
    if (p.lse && tx == 0)
      p.lse[((long long)b * p.H + h) * p.Nqp + qi] = some ? m[i] * p.scale_log2 + log2f(l[i]) : INFINITY;
  }
}

// Gradient of the queries; also leaves delta = sum(dy * y) of its rows for the backward of the keys.
template <typename T, int DP>
__global__ void __launch_bounds__(256) attn_simt_dq_kernel(const AttnParams p) {
  wait_for_inputs();
  constexpr int BN = other_rows<DP>(), CJ = BN / 16;
  extern __shared__ float sm[];
  float *Q = sm, *dO = Q + kOwn * (DP + 4), *K = dO + kOwn * (DP + 4), *V = K + BN * (DP + 4), *S = V + BN * (DP + 4);
  const Block at_block = block_of(p.H, (p.Nq + kOwn - 1) / kOwn);
  const int i0 = at_block.last_first * kOwn, h = at_block.head, b = at_block.b, hk = h / p.G;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const RowGeom g = row_geom(p, b);
  const KeyTiles kt = key_tiles<BN>(p, g, i0, i0 + kOwn);
  const SeenKeys seen = seen_keys(p, g);
  const T* q = static_cast<const T*>(p.q) + b * p.sq_b + i0 * p.sq_n + (long long)h * p.d;
  const T* dy = static_cast<const T*>(p.dy) + b * p.sdy_b + i0 * p.sdy_n + (long long)h * p.d;
  const T* k = static_cast<const T*>(p.k) + b * p.sk_b + (long long)hk * p.d;
  const T* v = static_cast<const T*>(p.v) + b * p.sv_b + (long long)hk * p.d;
  const int r_lo = max(0, -(g.start + i0)), r_hi = min(p.Nq, g.ctx - g.start) - i0;  // rows that are not padding
  load_tile<T, DP, kOwn>(Q, q, p.sq_n, rows_between(r_lo, r_hi), p.d, p.vec);
  load_tile<T, DP, kOwn>(dO, dy, p.sdy_n, rows_between(r_lo, r_hi), p.d, p.vec);
  __syncthreads();
  float acc[4][DP / 16] = {}, lse[4], delta[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i, qi = i0 + r;
    const long long at = ((long long)b * p.H + h) * p.Nqp + qi;
    const bool live = r >= r_lo && r < r_hi;
    lse[i] = live ? p.lse[at] : INFINITY;
    float sum = 0.f;
    if (live) {
      const long long row = ((long long)b * p.Nq + qi) * p.H * p.d + (long long)h * p.d;
      const T* y = static_cast<const T*>(p.y_in) + row;
      for (int c = tx; c < p.d; c += 16) {
        const float rest = sizeof(T) == 2 ? to_f(p.rest[row + c]) : 0.f;
        sum = fmaf(dO[r * (DP + 4) + c], to_f(y[c]) + rest, sum);
      }
    }
    delta[i] = sum16(sum);
    if (tx == 0 && qi < p.Nq) p.delta[at] = delta[i];
  }
  const int n = kt.count();
  for (int it = 0; it < n; ++it) {
    const int k0 = kt.tile(it) * BN;
    __syncthreads();
    load_tile<T, DP, BN>(K, k + k0 * p.sk_n, p.sk_n, rows_seen(seen, k0), p.d, p.vec);
    load_tile<T, DP, BN>(V, v + k0 * p.sv_n, p.sv_n, rows_seen(seen, k0), p.d, p.vec);
    __syncthreads();
    float s[4][CJ] = {}, dp[4][CJ] = {};
    rows_by_rows<DP, CJ>(Q, K, s);
    rows_by_rows<DP, CJ>(dO, V, dp);
    const bool all = sees_all(p, g, i0, kOwn, k0, BN);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = g.start + i0 + 4 * ty + i;
#pragma unroll
      for (int j = 0; j < CJ; ++j) {
        const float w = ex2(fmaf(s[i][j], p.scale_log2, -lse[i]));
        S[(4 * ty + i) * (BN + 4) + tx + 16 * j] = all || sees(p, g.ctx, pos, k0 + tx + 16 * j) ? w * (dp[i][j] - delta[i]) : 0.f;
      }
    }
    __syncwarp();
    rows_by_cols<DP, BN>(S, K, acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int qi = i0 + 4 * ty + i;
    if (qi >= p.Nq) continue;
    T* dq = static_cast<T*>(p.dq) + ((long long)b * p.Nq + qi) * p.H * p.d + (long long)h * p.d;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) {
      const int c = feature_of<DP>(e);
      if (c < p.d) put(dq + c, acc[i][e] * p.scale);
    }
  }
}

// Gradients of the keys and values.  The heads of a group are walked one after the other by the same CTA, so that their sum has
// one order.
template <typename T, int DP>
__global__ void __launch_bounds__(256) attn_simt_dkv_kernel(const AttnParams p) {
  wait_for_inputs();
  constexpr int BN = other_rows<DP>(), CJ = BN / 16;
  extern __shared__ float sm[];
  float *K = sm, *V = K + kOwn * (DP + 4), *Q = V + kOwn * (DP + 4), *dO = Q + BN * (DP + 4), *P = dO + BN * (DP + 4), *S = P + kOwn * (BN + 4);
  float *lse_s = S + kOwn * (BN + 4), *del_s = lse_s + BN;
  const Block at_block = block_of(p.Hk, (p.Nk + kOwn - 1) / kOwn + p.sink_tiles * p.chunks);
  const int hk = at_block.head, b = at_block.b, ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const RowGeom g = row_geom(p, b);
  const KeyItem it = key_item<kOwn, BN>(p, g, at_block.first_last);
  const int k0 = it.tile * kOwn, end = min(g.ctx, g.start + p.Nq);  // (of the queries: the last tile's rows behind them see nothing)
  const T* k = static_cast<const T*>(p.k) + b * p.sk_b + k0 * p.sk_n + (long long)hk * p.d;
  const T* v = static_cast<const T*>(p.v) + b * p.sv_b + k0 * p.sv_n + (long long)hk * p.d;
  float dk[4][DP / 16] = {}, dv[4][DP / 16] = {};
  if (it.begin < it.end) {
    load_tile<T, DP, kOwn>(K, k, p.sk_n, rows_between(0, g.ctx - k0), p.d, p.vec);
    load_tile<T, DP, kOwn>(V, v, p.sv_n, rows_between(0, g.ctx - k0), p.d, p.vec);
  }
  for (int e = it.begin; e < it.end; ++e) {
    const int h = hk * p.G + e / it.tiles, i0 = (it.first + e % it.tiles) * BN;
    const int r_lo = max(0, -(g.start + i0)), r_hi = min(p.Nq, g.ctx - g.start) - i0;
    __syncthreads();
    load_tile<T, DP, BN>(Q, static_cast<const T*>(p.q) + b * p.sq_b + i0 * p.sq_n + (long long)h * p.d, p.sq_n, rows_between(r_lo, r_hi), p.d, p.vec);
    load_tile<T, DP, BN>(dO, static_cast<const T*>(p.dy) + b * p.sdy_b + i0 * p.sdy_n + (long long)h * p.d, p.sdy_n, rows_between(r_lo, r_hi), p.d, p.vec);
    if (threadIdx.x < BN) {
      const int r = threadIdx.x;
      const long long at = ((long long)b * p.H + h) * p.Nqp + i0 + r;
      const bool live = r >= r_lo && r < r_hi;
      lse_s[r] = live ? p.lse[at] : INFINITY;
      del_s[r] = live ? p.delta[at] : 0.f;
    }
    __syncthreads();
    float s[4][CJ] = {}, dp[4][CJ] = {};
    rows_by_rows<DP, CJ>(K, Q, s);
    rows_by_rows<DP, CJ>(V, dO, dp);
    const bool all = sees_all(p, g, i0, BN, k0, kOwn);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = k0 + 4 * ty + i;
#pragma unroll
      for (int j = 0; j < CJ; ++j) {
        const int c = tx + 16 * j;
        float w = ex2(fmaf(s[i][j], p.scale_log2, -lse_s[c])), t = w * (dp[i][j] - del_s[c]);
        if (!all && !sees(p, end, g.start + i0 + c, key)) w = t = 0.f;
        P[(4 * ty + i) * (BN + 4) + c] = w;
        S[(4 * ty + i) * (BN + 4) + c] = t;
      }
    }
    __syncwarp();
    rows_by_cols<DP, BN>(P, dO, dv);
    rows_by_cols<DP, BN>(S, Q, dk);
  }
  const bool sinks = p.chunks > 0 && it.tile < p.sink_tiles;
  float* part = sinks ? part_of(p, b, hk, it.tile, it.chunk < 0 ? p.chunks : it.chunk) : nullptr;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i, key = k0 + r;
    if (key >= p.Nk) continue;
    const bool partial = sinks && key < p.n_sink;
    if (it.chunk >= 0 && !partial) continue;
    const long long at = ((long long)b * p.Nk + key) * p.Hk * p.d + (long long)hk * p.d;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) {
      const int c = feature_of<DP>(e);
      if (c >= p.d) continue;
      if (partial) {
        part[r * p.d + c] = dk[i][e] * p.scale;
        part[(p.sink_rows + r) * p.d + c] = dv[i][e];
      } else {
        put(static_cast<T*>(p.dk) + at + c, dk[i][e] * p.scale);
        put(static_cast<T*>(p.dv) + at + c, dv[i][e]);
      }
    }
  }
}

// The sums of the sink keys' partial gradients, piece by piece in one order.  One CTA per key.
template <typename T>
__global__ void __launch_bounds__(256) attn_sink_sum_kernel(const AttnParams p, int tile_rows) {
  wait_for_inputs();
  const Block at_block = block_of(p.Hk, p.n_sink);
  const int key = at_block.first_last, hk = at_block.head, b = at_block.b, tile = key / tile_rows, r = key % tile_rows;
  const float* part = part_of(p, b, hk, tile, 0);
  const long long step = 2ll * p.sink_rows * p.d, at = ((long long)b * p.Nk + key) * p.Hk * p.d + (long long)hk * p.d;
  for (int c = threadIdx.x; c < 2 * p.d; c += 256) {
    const bool is_v = c >= p.d;
    const int f = is_v ? c - p.d : c;
    const float* x = part + ((is_v ? p.sink_rows : 0) + r) * p.d + f;
    float sum = 0.f;
    for (int i = 0; i <= p.chunks; ++i) sum += x[i * step];
    put(static_cast<T*>(is_v ? p.dv : p.dk) + at + f, sum);
  }
}

template <typename T, int DP> constexpr size_t smem_fwd() {
  constexpr int BN = other_rows<DP>();
  return sizeof(float) * ((kOwn + 2 * BN) * (DP + 4) + kOwn * (BN + 4));
}
template <typename T, int DP> constexpr size_t smem_dq() {
  constexpr int BN = other_rows<DP>();
  return sizeof(float) * ((2 * kOwn + 2 * BN) * (DP + 4) + kOwn * (BN + 4));
}
template <typename T, int DP> constexpr size_t smem_dkv() {
  constexpr int BN = other_rows<DP>();
  return sizeof(float) * ((2 * kOwn + 2 * BN) * (DP + 4) + 2 * kOwn * (BN + 4) + 2 * BN);
}

template <typename T, int DP>
cudaError_t run_fwd(const AttnParams& p, cudaStream_t st) {
  static SmemGrant grant;
  cudaError_t e = grant_smem(grant, attn_simt_fwd_kernel<T, DP>, smem_fwd<T, DP>());
  if (e != cudaSuccess) return e;
  return launch_behind(attn_simt_fwd_kernel<T, DP>, dim3((unsigned)((p.Nq + kOwn - 1) / kOwn * p.H * p.B)), 256, smem_fwd<T, DP>(), st, p);
}
template <typename T, int DP>
cudaError_t run_bwd(const AttnParams& p, cudaStream_t st) {
  static SmemGrant g1, g2;
  cudaError_t e = grant_smem(g1, attn_simt_dq_kernel<T, DP>, smem_dq<T, DP>());
  if (e == cudaSuccess) e = grant_smem(g2, attn_simt_dkv_kernel<T, DP>, smem_dkv<T, DP>());
  if (e != cudaSuccess) return e;
  e = launch_behind(attn_simt_dq_kernel<T, DP>, dim3((unsigned)((p.Nq + kOwn - 1) / kOwn * p.H * p.B)), 256, smem_dq<T, DP>(), st, p);
  if (e != cudaSuccess) return e;
  if (p.Nk == 0) return cudaSuccess;
  const int items = (p.Nk + kOwn - 1) / kOwn + p.sink_tiles * p.chunks;
  return launch_behind(attn_simt_dkv_kernel<T, DP>, dim3((unsigned)(items * p.Hk * p.B)), 256, smem_dkv<T, DP>(), st, p);
}
// (With few features the products' error of 2^-22 would stand out against their sum's.)
bool split_covers(const AttnParams& p, int dtype) { return dtype == DT_F32 && p.d > 16 && p.d <= 128; }
template <typename T>
cudaError_t by_size(const AttnParams& p, bool bwd, cudaStream_t st) {
  if (p.d <= 32) return bwd ? run_bwd<T, 32>(p, st) : run_fwd<T, 32>(p, st);
  if constexpr (sizeof(T) == 2) {
    if (p.d <= 64) return bwd ? run_bwd<T, 64>(p, st) : run_fwd<T, 64>(p, st);
    if (p.d <= 96) return bwd ? run_bwd<T, 96>(p, st) : run_fwd<T, 96>(p, st);
    if (p.d <= 128) return bwd ? run_bwd<T, 128>(p, st) : run_fwd<T, 128>(p, st);
  }
  return bwd ? run_bwd<T, 256>(p, st) : run_fwd<T, 256>(p, st);
}

}  // namespace

cudaError_t launch_attn_simt_fwd(const AttnParams& p, int dtype, cudaStream_t st) {
  if (split_covers(p, dtype)) return launch_attn_split_fwd(p, st);
  return dtype == DT_BF16 ? by_size<__nv_bfloat16>(p, false, st) : by_size<float>(p, false, st);
}
cudaError_t launch_attn_simt_bwd(const AttnParams& p, int dtype, cudaStream_t st) {
  cudaError_t e = split_covers(p, dtype) ? launch_attn_split_bwd(p, st)
                  : dtype == DT_BF16     ? by_size<__nv_bfloat16>(p, true, st)
                                         : by_size<float>(p, true, st);
  if (e != cudaSuccess || p.chunks == 0) return e;
  return launch_attn_sink_sum(p, dtype, kOwn, st);
}
cudaError_t launch_attn_sink_sum(const AttnParams& p, int dtype, int tile, cudaStream_t st) {
  const dim3 grid((unsigned)(p.n_sink * p.Hk * p.B));
  return dtype == DT_BF16 ? launch_behind(attn_sink_sum_kernel<__nv_bfloat16>, grid, 256, 0, st, p, tile)
                          : launch_behind(attn_sink_sum_kernel<float>, grid, 256, 0, st, p, tile);
}

}  // namespace ncn
