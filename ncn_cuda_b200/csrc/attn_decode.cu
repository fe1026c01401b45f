// Windowed attention of the last few positions of each row over a cache: the form for single tokens.
//
// Bound by reading the visible keys and values once (64 rows, windows of 4096, 8 heads of 128: 1.08 GB in 184 us, 5.9 of the 6.46 TB/s
// that a plain copy reaches); one row's time is a launch, the latency of its loads and the joins (7 us).
//
// A CTA of 8 warps takes the queries of one key/value head (the heads of its
// group times the new positions, up to 16 rows at a time); the visible keys, sinks first and the window behind them, are dealt out to the
// warps of a cluster of CTAs in blocks, every warp keeps a running softmax of its own, and the parts are joined through shared
// memory, first in the CTA, then in the cluster over distributed shared memory: one launch, no workspace, and one order of sums.
// Keys outside the sinks and the window are not read at all.
#include <cooperative_groups.h>

#include "attn_common.cuh"
#include "ncn_common.cuh"

namespace ncn {
namespace {

namespace cg = cooperative_groups;
constexpr int kWarps = 8;

// The keys that any of a row's queries sees, as blocks of `size`: those of the sinks, then those of the window.
struct KeyBlocks {
  int sinks, first, end, sink_blocks, count;
};
__device__ __forceinline__ KeyBlocks key_blocks(const AttnParams& p, const RowGeom& g, int size) {
  KeyBlocks k;
  const int lo = max(g.start, 0);
  k.end = min(g.start + p.Nq, g.ctx);
  k.first = min(max(lo - p.window + 1, 0), k.end);
  k.sinks = min(p.n_sink, k.first);
  k.sink_blocks = (k.sinks + size - 1) / size;
  k.count = k.end > lo ? k.sink_blocks + (k.end - k.first + size - 1) / size : 0;
  return k;
}
// Block i: its first key; `limit`: the end of its part of the keys
__device__ __forceinline__ int block_start(const KeyBlocks& k, int i, int size, int& limit) {
  const bool sink = i < k.sink_blocks;
  limit = sink ? k.sinks : k.end;
  return sink ? i * size : k.first + (i - k.sink_blocks) * size;
}

// Joins what the warps of a cluster hold.  Os[kWarps][R][DP], ms (log2 units) and ls [kWarps][R] in shared memory.
template <typename T, int R, int DP>
__device__ __forceinline__ void join(const AttnParams& p, float* Os, float* ms, float* ls, int rows, int row0, int hk, int b, int start) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  __syncthreads();
  // the CTA's own, in the place of its first warp's
  for (int e = threadIdx.x; e < rows * DP; e += kWarps * 32) {
    const int r = e / DP;
    float M = -INFINITY;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ms[w * R + r]);
    const float ref = M == -INFINITY ? 0.f : M;
    float sum = 0.f;
    for (int w = 0; w < kWarps; ++w) sum = fmaf(Os[w * R * DP + e], ex2(ms[w * R + r] - ref), sum);
    Os[e] = sum;  // (only this thread reads entry e of any warp)
  }
  __syncthreads();
  if (threadIdx.x < rows) {
    const int r = threadIdx.x;
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ms[w * R + r]);
    const float ref = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < kWarps; ++w) L = fmaf(ls[w * R + r], ex2(ms[w * R + r] - ref), L);
    ms[r] = M;
    ls[r] = L;
  }
  cluster.sync();
  // each rank writes its share of the rows and features
  for (int e = rank * kWarps * 32 + threadIdx.x; e < rows * DP; e += ranks * kWarps * 32) {
    const int r = e / DP, c = e % DP;
    float M = -INFINITY;
    for (int i = 0; i < ranks; ++i) M = fmaxf(M, cluster.map_shared_rank(ms, i)[r]);
    const float ref = M == -INFINITY ? 0.f : M;
    float sum = 0.f, L = 0.f;
    for (int i = 0; i < ranks; ++i) {
      const float f = ex2(cluster.map_shared_rank(ms, i)[r] - ref);
      sum = fmaf(cluster.map_shared_rank(Os, i)[e], f, sum);
      L = fmaf(cluster.map_shared_rank(ls, i)[r], f, L);
    }
    if (c < p.d) {
      const int row = row0 + r, h = hk * p.G + row / p.Nq, i = row % p.Nq;
      put(static_cast<T*>(p.y) + ((long long)b * p.Nq + i) * p.H * p.d + (long long)h * p.d + c, start + i >= 0 ? sum / L : 0.f);  // (scores that are all minus infinity: 0 / 0)
    }
  }
  cluster.sync();  // nobody leaves while its memory is read
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load16(const void* at, bool ok) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (ok) v = __ldcs(static_cast<const uint4*>(at));
  return v;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// a pair of bf16 per lane as an 8 x 8 matrix (lane / 4: row): its transpose
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// bf16, heads of a multiple of 8 features.  Blocks of 16 keys go from global memory straight into the left operands of the matrix
// instructions (m16n8k16), 16 bytes per lane and load, without shared memory; 8 query rows are the columns (TILES of them).
//   scores^T = keys . queries^T    16 keys, 16 features a time
//   sums^T  += values^T . weights^T  16 features, 16 keys a time
// The order of a sum's terms is free: the lane that loads features 8 c .. 8 c + 7 of two keys uses them as its pairs of two products'
// terms, the queries laid out the same way.  For the values the lane's eight features belong to four products' rows, and pairs of keys
// are put together by byte permutes.  (With the queries as left operand, whose 16 rows are half empty, a step took twice the
// instructions and 32 registers more, and one CTA less fitted on an SM.)  Two new tokens in groups of 4 (8 rows) take as long as one, four
// (16 rows: TILES 2, one CTA per SM) 289 us for 184.
template <int DP, int TILES>
__global__ void __launch_bounds__(kWarps * 32, TILES == 1 ? 2 : 1) attn_decode_kernel(const __grid_constant__ AttnParams p) {
  wait_for_inputs();
  constexpr int R = 8 * TILES, TK = DP / 32, TV = DP / 64;
  extern __shared__ float sm[];
  float *Os = sm, *ms = Os + kWarps * R * DP, *ls = ms + kWarps * R;
  const int ranks = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
  const int groups = (p.G * p.Nq + R - 1) / R;
  const int unit = blockIdx.x / ranks, hk = unit % p.Hk, b = unit / p.Hk / groups, row0 = unit / p.Hk % groups * R;
  const int rows = min(R, p.G * p.Nq - row0);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g8 = lane / 4, c4 = lane % 4;
  const RowGeom g = row_geom(p, b);
  const KeyBlocks kb = key_blocks(p, g, 16);
  using bf16 = __nv_bfloat16;

  uint4 q[TILES][TK];
  int pos[TILES][2];  // of the lane's columns 2 c4, 2 c4 + 1
#pragma unroll
  for (int u = 0; u < TILES; ++u) {
    const int r = g8 + 8 * u, row = row0 + r, i = row % p.Nq, h = hk * p.G + row / p.Nq;
#pragma unroll
    for (int t = 0; t < TK; ++t) {
      const int c = (4 * t + c4) * 8;
      q[u][t] = load16(static_cast<const bf16*>(p.q) + b * p.sq_b + i * p.sq_n + (long long)h * p.d + c, r < rows && c < p.d);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int column = 2 * c4 + x + 8 * u;
      pos[u][x] = column < rows ? g.start + (row0 + column) % p.Nq : -1;
    }
  }
  const bf16* kp = static_cast<const bf16*>(p.k) + b * p.sk_b + (long long)hk * p.d + c4 * 8;
  const bf16* vp = static_cast<const bf16*>(p.v) + b * p.sv_b + (long long)hk * p.d + g8 * 8;

  float o[TILES][TV * 4][4], m[TILES][2], l[TILES][2];
#pragma unroll
  for (int u = 0; u < TILES; ++u) {
    m[u][0] = m[u][1] = -INFINITY;
    l[u][0] = l[u][1] = 0.f;
#pragma unroll
    for (int e = 0; e < TV * 4; ++e) o[u][e][0] = o[u][e][1] = o[u][e][2] = o[u][e][3] = 0.f;
  }

  for (int i = rank * kWarps + warp; i < kb.count; i += ranks * kWarps) {
    int limit;
    const int key0 = block_start(kb, i, 16, limit);
    uint4 kf[2][TK], vf[4][TV];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int key = key0 + 8 * n + g8;
#pragma unroll
      for (int t = 0; t < TK; ++t) kf[n][t] = load16(kp + key * p.sk_n + 32 * t, key < limit && 32 * t + 8 * c4 < p.d);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int key = key0 + 2 * c4 + (n & 1) + 8 * (n >> 1);
#pragma unroll
      for (int t = 0; t < TV; ++t) vf[n][t] = load16(vp + key * p.sv_n + 64 * t, key < limit && 64 * t + 8 * g8 < p.d);
    }
    uint32_t w[TILES][2];
#pragma unroll
    for (int u = 0; u < TILES; ++u) {
      float s[4] = {};  // keys g8 (0, 1) and g8 + 8 (2, 3), columns 2 c4 and 2 c4 + 1
#pragma unroll
      for (int t = 0; t < TK; ++t)
#pragma unroll
        for (int half = 0; half < 4; half += 2) {
          const uint32_t a[4] = {word(kf[0][t], half), word(kf[1][t], half), word(kf[0][t], half + 1), word(kf[1][t], half + 1)};
          mma_bf16(s, a, word(q[u][t], half), word(q[u][t], half + 1));
        }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int key = key0 + 8 * n + g8;
          s[2 * n + x] = key < limit && sees(p, g.ctx, pos[u][x], key) ? s[2 * n + x] * p.scale_log2 : -INFINITY;
        }
        float mx = fmaxf(s[x], s[2 + x]);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, d));
        const float now = fmaxf(m[u][x], mx), ref = now == -INFINITY ? 0.f : now, keep = ex2(m[u][x] - ref);
        m[u][x] = now;
        s[x] = ex2(s[x] - ref), s[2 + x] = ex2(s[2 + x] - ref);
        l[u][x] = fmaf(l[u][x], keep, s[x] + s[2 + x]);
#pragma unroll
        for (int e = 0; e < TV * 4; ++e) o[u][e][x] *= keep, o[u][e][2 + x] *= keep;
      }
      w[u][0] = transpose8(pack(s[0], s[1]));
      w[u][1] = transpose8(pack(s[2], s[3]));
    }
#pragma unroll
    for (int t = 0; t < TV; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t a[4] = {__byte_perm(word(vf[0][t], e), word(vf[1][t], e), 0x5410), __byte_perm(word(vf[0][t], e), word(vf[1][t], e), 0x7632),
                               __byte_perm(word(vf[2][t], e), word(vf[3][t], e), 0x5410), __byte_perm(word(vf[2][t], e), word(vf[3][t], e), 0x7632)};
#pragma unroll
        for (int u = 0; u < TILES; ++u) mma_bf16(o[u][t * 4 + e], a, w[u][0], w[u][1]);
      }
  }
  // row g8 and g8 + 8 of product (t, e) are features 64 t + 8 g8 + 2 e and the next one
#pragma unroll
  for (int u = 0; u < TILES; ++u)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = 2 * c4 + x + 8 * u;
#pragma unroll
      for (int d = 4; d < 32; d *= 2) l[u][x] += __shfl_xor_sync(~0u, l[u][x], d);
      if (g8 == 0) ms[warp * R + r] = m[u][x], ls[warp * R + r] = l[u][x];
#pragma unroll
      for (int t = 0; t < TV; ++t)
#pragma unroll
        for (int e = 0; e < 4; e += 2)
          *reinterpret_cast<float4*>(Os + (warp * R + r) * DP + 64 * t + 8 * g8 + 2 * e) =
              make_float4(o[u][t * 4 + e][x], o[u][t * 4 + e][2 + x], o[u][t * 4 + e + 1][x], o[u][t * 4 + e + 1][2 + x]);
    }
  join<bf16, R, DP>(p, Os, ms, ls, rows, row0, hk, b, g.start);
}

// fp32, and bf16 heads that the kernel above does not take.  Eight lanes per key, DP / 8 features each; a warp has four keys at a
// time.  Every group of lanes has its own running softmax; rescaling is rare once the largest score has been met.  Bound by the products and
// the sums over eight lanes, of R rows whether there are as many or not: 64 rows, windows of 4096, 8 heads of 128 each for 4 heads of queries,
// fp32 757 us (2.8 TB/s), with two new tokens 1285, with four 2471; 32 rows, windows of 2048, 8 heads of 256, fp32 412 us, bf16 1953.
template <typename T, int DP, int R>
__global__ void __launch_bounds__(kWarps * 32) attn_decode_any_kernel(const AttnParams p) {
  wait_for_inputs();
  extern __shared__ float sm[];
  float *Os = sm, *ms = Os + kWarps * R * DP, *ls = ms + kWarps * R;
  const int ranks = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
  const int groups = (p.G * p.Nq + R - 1) / R;
  const int unit = blockIdx.x / ranks, hk = unit % p.Hk, b = unit / p.Hk / groups, row0 = unit / p.Hk % groups * R;
  const int rows = min(R, p.G * p.Nq - row0);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, part = lane % 8;
  const RowGeom g = row_geom(p, b);
  const KeyBlocks kb = key_blocks(p, g, 4);
  constexpr int F = DP / 8;  // features of a lane: 4 part + 32 j .. + 3
  auto feature = [&](int e) { return 4 * part + 32 * (e / 4) + e % 4; };
  auto load = [&](const T* at, bool ok, float (&x)[F]) {
#pragma unroll
    for (int e = 0; e < F; e += 4) {
      const int c = feature(e);
      if (sizeof(T) == 4 && p.vec) {
        const float4 v = ok && c < p.d ? *reinterpret_cast<const float4*>(at + c) : make_float4(0, 0, 0, 0);
        x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[e + i] = ok && c + i < p.d ? to_f(at[c + i]) : 0.f;
      }
    }
  };
  float q[R][F], o[R][F], m[R], l[R];
  int pos[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + r, i = row % p.Nq, h = hk * p.G + row / p.Nq;
    pos[r] = r < rows ? g.start + i : -1;
    load(static_cast<const T*>(p.q) + b * p.sq_b + i * p.sq_n + (long long)h * p.d, r < rows, q[r]);
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < F; ++e) o[r][e] = 0.f;
  }
  for (int i = rank * kWarps + warp; i < kb.count; i += ranks * kWarps) {
    int limit;
    const int key = block_start(kb, i, 4, limit) + lane / 8;
    float x[F], v[F];
    load(static_cast<const T*>(p.k) + b * p.sk_b + key * p.sk_n + (long long)hk * p.d, key < limit, x);
    load(static_cast<const T*>(p.v) + b * p.sv_b + key * p.sv_n + (long long)hk * p.d, key < limit, v);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < F; ++e) s = fmaf(q[r][e], x[e], s);
#pragma unroll
      for (int w = 4; w; w >>= 1) s += __shfl_xor_sync(~0u, s, w);
      if (key < limit && sees(p, g.ctx, pos[r], key)) {
        s *= p.scale_log2;
        if (s > m[r]) {
          const float keep = ex2(m[r] - s);
          m[r] = s;
          l[r] *= keep;
#pragma unroll
          for (int e = 0; e < F; ++e) o[r][e] *= keep;
        }
        const float w = s == -INFINITY ? 0.f : ex2(s - (m[r] == -INFINITY ? 0.f : m[r]));
        l[r] += w;
#pragma unroll
        for (int e = 0; e < F; ++e) o[r][e] = fmaf(w, v[e], o[r][e]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {  // the warp's four groups
    float M = fmaxf(m[r], __shfl_xor_sync(~0u, m[r], 8));
    M = fmaxf(M, __shfl_xor_sync(~0u, M, 16));
    const float keep = ex2(m[r] - (M == -INFINITY ? 0.f : M));
    l[r] *= keep;
    l[r] += __shfl_xor_sync(~0u, l[r], 8);
    l[r] += __shfl_xor_sync(~0u, l[r], 16);
#pragma unroll
    for (int e = 0; e < F; ++e) {
      o[r][e] *= keep;
      o[r][e] += __shfl_xor_sync(~0u, o[r][e], 8);
      o[r][e] += __shfl_xor_sync(~0u, o[r][e], 16);
    }
    if (lane == 0) ms[warp * R + r] = M, ls[warp * R + r] = l[r];
    if (lane < 8) {
#pragma unroll
      for (int e = 0; e < F; ++e) Os[(warp * R + r) * DP + feature(e)] = o[r][e];
    }
  }
  join<T, R, DP>(p, Os, ms, ls, rows, row0, hk, b, g.start);
}

// CTAs of a cluster: enough that the SMs have a CTA each, no more than the keys feed, blocks of `size` keys to a warp.  (64 rows of a cache
// of 8192, windows of 4096, 8 heads of keys of 128: 184 us with clusters of 1 and 2, 197 of 4, 242 of 8; one row, windows of 1024: 16.7 us
// with one CTA per head, 7.3 with clusters of 8.)
template <typename K>
cudaError_t launch(K kernel, const AttnParams& p, int R, int DP, int size, int sms, SmemGrant& grant, cudaStream_t st) {
  const size_t smem = sizeof(float) * kWarps * R * (DP + 2);
  cudaError_t e = grant_smem(grant, kernel, smem);
  if (e != cudaSuccess) return e;
  const long long units = (long long)p.B * p.Hk * ((p.G * p.Nq + R - 1) / R);
  const long long keys = min((long long)p.Nk, (long long)p.window + p.Nq - 1 + p.n_sink);
  int ranks = 1;
  while (ranks < 8 && units * ranks < sms && (long long)ranks * kWarps * size < keys) ranks *= 2;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * ranks));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int DP>
cudaError_t run_bf16(const AttnParams& p, int sms, cudaStream_t st) {
  static SmemGrant g8, g16;
  return p.G * p.Nq > 8 ? launch(attn_decode_kernel<DP, 2>, p, 16, DP, 16, sms, g16, st)
                        : launch(attn_decode_kernel<DP, 1>, p, 8, DP, 16, sms, g8, st);
}
template <typename T, int DP>
cudaError_t run_any(const AttnParams& p, int sms, cudaStream_t st) {
  constexpr int R = DP <= 64 ? 8 : DP <= 128 ? 4 : 2;
  static SmemGrant g1, g;
  return p.G * p.Nq == 1 ? launch(attn_decode_any_kernel<T, DP, 1>, p, 1, DP, 4, sms, g1, st)
                         : launch(attn_decode_any_kernel<T, DP, R>, p, R, DP, 4, sms, g, st);
}
template <typename T>
cudaError_t any_size(const AttnParams& p, int sms, cudaStream_t st) {
  if (p.d <= 32) return run_any<T, 32>(p, sms, st);
  if (p.d <= 64) return run_any<T, 64>(p, sms, st);
  if (p.d <= 128) return run_any<T, 128>(p, sms, st);
  return run_any<T, 256>(p, sms, st);
}

}  // namespace

cudaError_t launch_attn_decode(const AttnParams& p, int dtype, int sms, cudaStream_t st) {
  if (dtype == DT_F32) return any_size<float>(p, sms, st);
  if (p.vec && p.d <= 64) return run_bf16<64>(p, sms, st);
  if (p.vec && p.d <= 128) return run_bf16<128>(p, sms, st);
  return any_size<__nv_bfloat16>(p, sms, st);
}

}  // namespace ncn
