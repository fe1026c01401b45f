// Rotary positions, and norms of queries and keys per head with the rotation in the same pass; forward and backward.
//
//   u = x r w,  r = 1 / sqrt(mean(x^2) + eps)          (or u = x, without a norm)
//   (a, b) pair i of u:  a' = M (a cos - b sin),  b' = M (b cos + a sin),  angle = position * frequency_i
// Backward: g = the cotangent rotated by the opposite angle;  dw = sum g x r,  dx = r (g w - x r mean(g w x r)).
//
// One pass over the data: 2 tensors forward, 3 backward, which is what bounds it.  Measured (bf16, 32768 positions, 32 + 8 heads of
// 128): 122 us forward, 194 backward with norms, 5.5 and 5.2 of the 6.46 TB/s that a plain copy reaches, with three quarters of the
// instruction slots in use.  Teams that keep a position and walk its heads need fewer instructions but were slower (131, 207: their
// reads lie 10 KB apart), and so were bulk prefetches of the next span into L2 (139, 228).
//
// Angles are formed in 64 bits as turns
// (position * frequency / 2 pi minus the nearest whole number), so that far positions lose nothing; what is left is below half a
// turn and goes through sincospi in 32 bits.  A sine and cosine cost more instructions than everything else of a pair of
// features: they are formed once per position, into shared memory, for all heads.
#include <cuda_bf16.h>

#include "ncn_common.cuh"
#include "qk_rotary.h"

namespace ncn {
namespace {

__device__ __forceinline__ float2 cos_sin(const RotaryParams& p, long long pos, int pair) {
  const double turns = (double)pos * (p.freqs[pair] * 0.15915494309189533577);  // 1 / (2 pi)
  float s, c;
  sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
  return make_float2(c * p.magnitude, p.backward ? -s * p.magnitude : s * p.magnitude);
}

// 16 features of a lane, two chunks of 8: as they come, and in fp32
template <typename T> struct Chunks {
  static constexpr int V = sizeof(T) / 2;  // 16-byte words of a chunk
  uint4 a[V], c[V];
  __device__ __forceinline__ void load(const T* row, int c0, int c1) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] = __ldcs(reinterpret_cast<const uint4*>(row + c0) + i);
      c[i] = __ldcs(reinterpret_cast<const uint4*>(row + c1) + i);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = c[i] = make_uint4(0, 0, 0, 0);
  }
  static __device__ __forceinline__ void widen(const uint4 (&r)[V], float2 (&x)[4]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
      } else {
        x[2 * i] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
        x[2 * i + 1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
      }
    }
  }
  static __device__ __forceinline__ void store(T* at, const float2 (&x)[4]) {
    if constexpr (sizeof(T) == 2) {
      __nv_bfloat162 h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __float22bfloat162_rn(x[i]);
      *reinterpret_cast<uint4*>(at) = *reinterpret_cast<uint4*>(h);
    } else {
      reinterpret_cast<float4*>(at)[0] = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
      reinterpret_cast<float4*>(at)[1] = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
    }
  }
};
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 minus(float2 x) { return make_float2(-x.x, -x.y); }

template <int W>
__device__ __forceinline__ float team_sum(float x) {
#pragma unroll
  for (int s = W / 2; s; s >>= 1) x += __shfl_xor_sync(~0u, x, s);
  return x;
}

// Heads of d = 16 m features with R a multiple of 16: a team of W >= d / 16 lanes per head, 16 features per lane in two chunks of 8.
// Lane i < R / 16 holds the pairs 8 i .. 8 i + 7 (half layout: features 8 i .. and R / 2 + 8 i ..; interleaved: 16 i ..), the
// lanes behind it features that are not rotated.  A CTA takes p.span positions at a time; the heads of all of them, those of the
// queries first, are dealt out to its teams (and to p.parts CTAs, where there are few positions).  The first head is under way while
// the sines are formed, the next one while one is worked on.
enum Mode : int { PLAIN = 0, NORM = 1, NORM_BWD = 2 };  // PLAIN: either direction
template <typename T, int W, int MODE>
__global__ void __launch_bounds__(256, MODE == NORM_BWD ? 2 : 4) rotary_kernel(const __grid_constant__ RotaryParams p) {
  wait_for_inputs();
  constexpr bool norm = MODE != PLAIN, norm_bwd = MODE == NORM_BWD;
  constexpr int TEAMS = 256 / W;
  __shared__ __align__(16) float table[2 * kRotaryTable];
  __shared__ long long offs[norm_bwd ? 4 : 2][kRotarySpan];  // of the span's positions in q, k and their cotangents
  __shared__ __align__(16) float weight[norm ? 2 * 16 * W : 4];  // W <= 16: the first 2 W threads fill it
  const int lane = threadIdx.x % W, team = threadIdx.x / W, half = p.R / 2;
  const int turning = p.R / 16;
  const bool active = lane < p.d / 16, turn = lane < turning;
  const int c0 = turn && !p.interleaved ? 8 * lane : 16 * lane, c1 = turn && !p.interleaved ? 8 * lane + half : c0 + 8;
  const int part = blockIdx.x % p.parts, step = p.parts * TEAMS, first = part * TEAMS + team;
  const uint32_t N = (uint32_t)p.N;
  const long long rows = (long long)p.B * p.N, stride = (long long)(gridDim.x / p.parts) * p.span;
  const float inv[2] = {1.f / p.t[0].heads, p.t[1].heads ? 1.f / p.t[1].heads : 0.f}, inv_d = 1.f / p.d;
  // position of a row of all of them (32-bit divisions where the batch allows)
  auto split = [&](long long row, long long& b, long long& n) {
    if (rows <= 0xffffffffll) {
      const uint32_t q = (uint32_t)row / N;
      b = q, n = (uint32_t)row - q * N;
    } else {
      b = row / p.N, n = row - b * p.N;
    }
  };
  if (norm && threadIdx.x < 2 * W && active && p.t[team].heads) {  // entry j of a lane: four weights of its features
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) weight[((team * 4 + j) * W + lane) * 4 + e] = p.t[team].w[(j < 2 ? c0 : c1) + j % 2 * 4 + e];
  }
  // NORM_BWD: the sums for the weights of the tensor `of` that is being worked on; what a team has of either is kept in shared memory
  __shared__ __align__(16) float kept[norm_bwd ? 2 : 1][norm_bwd ? TEAMS : 1][norm_bwd ? 16 * W : 4];
  float2 dw[8];
  int of = 0;
  auto keep = [&]() {  // (the lane's own entries)
    float2 *const u = reinterpret_cast<float2*>(&kept[of][team][c0]), *const v = reinterpret_cast<float2*>(&kept[of][team][c1]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u[e] = __fadd2_rn(u[e], dw[e]), v[e] = __fadd2_rn(v[e], dw[4 + e]);
      dw[e] = dw[4 + e] = both(0.f);
    }
  };
  if constexpr (norm_bwd) {
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[e] = both(0.f);
    if (active) {
#pragma unroll
      for (int e = 0; e < 8; ++e) kept[0][team][c0 + e] = kept[0][team][c1 + e] = kept[1][team][c0 + e] = kept[1][team][c1 + e] = 0.f;
    }
  }
  for (long long row0 = (long long)(blockIdx.x / p.parts) * p.span; row0 < rows; row0 += stride) {
    const int span = (int)min((long long)p.span, rows - row0), of_q = span * p.t[0].heads, count = of_q + span * p.t[1].heads;
    const int turns = (count + step - 1) / step;  // the same for every lane: shuffles
    Chunks<T> x_next, g_next;
    int which = 0, at = 0, h = 0, next_which, next_at, next_h;  // of the head that is worked on, of the next one
    auto fetch = [&](int i, bool first_one) {
      x_next.clear();
      if (norm_bwd) g_next.clear();
      // (i < 2^20: the product is off by less than what 0.5 leaves)
      next_which = i >= of_q;
      const int j = next_which ? i - of_q : i;
      next_at = (int)((j + 0.5f) * (next_which ? inv[1] : inv[0]));
      next_h = j - next_at * (next_which ? p.t[1].heads : p.t[0].heads);
      if (active && i < count) {
        const RotaryTensor& t = p.t[next_which];
        long long xo, go = 0;
        if (first_one) {
          long long b, n;
          split(row0 + next_at, b, n);
          xo = b * t.sb + n * t.sn, go = b * t.gb + n * t.gn;
        } else {
          xo = offs[next_which][next_at];
          if (norm_bwd) go = offs[2 + next_which][next_at];
        }
        x_next.load(static_cast<const T*>(t.x) + xo + next_h * p.d, c0, c1);
        if (norm_bwd) g_next.load(static_cast<const T*>(t.dy) + go + next_h * p.d, c0, c1);
      }
    };
    fetch(first, true);
    __syncthreads();  // (the span before is done with the sines)
    for (int e = threadIdx.x; e < span * half; e += 256) {
      const int pos_at = e / half, pair = e - pos_at * half;
      long long b, n;
      split(row0 + pos_at, b, n);
      const float2 cs = cos_sin(p, p.pos ? p.pos[b * p.pos_b + n] : p.start + n, pair);
      // of a lane's 8 pairs: two words of four cosines, two of four sines
      float* const to = table + pos_at * p.R + (pair % 8 / 4 * turning + pair / 8) * 4 + pair % 4;
      to[0] = cs.x;
      to[8 * turning] = cs.y;
    }
    if (threadIdx.x < span) {
      long long b, n;
      split(row0 + threadIdx.x, b, n);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        offs[w][threadIdx.x] = b * p.t[w].sb + n * p.t[w].sn;
        if (norm_bwd) offs[2 + w][threadIdx.x] = b * p.t[w].gb + n * p.t[w].gn;
      }
    }
    __syncthreads();
    for (int k = 0; k < turns; ++k) {
      const int i = first + k * step;
      const bool here = active && i < count;
      which = next_which, at = next_at, h = next_h;
      const float4* w = reinterpret_cast<const float4*>(weight) + which * 4 * W + lane;
      float2 a[4], c[4], ga[4], gc[4];
      Chunks<T>::widen(x_next.a, a);
      Chunks<T>::widen(x_next.c, c);
      if (norm_bwd) {
        Chunks<T>::widen(g_next.a, ga);
        Chunks<T>::widen(g_next.c, gc);
      }
      if (k + 1 < turns) fetch(i + step, false);
      float r = 1.f;
      if (norm) {
        float2 sq = both(0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) sq = __ffma2_rn(a[e], a[e], __ffma2_rn(c[e], c[e], sq));
        r = rsqrtf(team_sum<W>(sq.x + sq.y) * inv_d + p.eps);
        if (!here) r = 0.f;  // (infinite where eps is 0)
      }
      float2 wa[4], wc[4];
      if (norm) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 u = w[e * W], v = w[(2 + e) * W];
          wa[2 * e] = make_float2(u.x, u.y), wa[2 * e + 1] = make_float2(u.z, u.w);
          wc[2 * e] = make_float2(v.x, v.y), wc[2 * e + 1] = make_float2(v.z, v.w);
        }
      }
      if (!norm_bwd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ga[e] = norm ? __fmul2_rn(a[e], __fmul2_rn(both(r), wa[e])) : a[e];
          gc[e] = norm ? __fmul2_rn(c[e], __fmul2_rn(both(r), wc[e])) : c[e];
        }
      }
      if (turn && here) {
        const float4* tab = reinterpret_cast<const float4*>(table + at * p.R) + lane;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float4 cw = tab[q * turning], sw = tab[(2 + q) * turning];
          if (p.interleaved) {  // pairs 4 q .. 4 q + 3: a's for q = 0, c's for q = 1
            float2(&g)[4] = q ? gc : ga;
            const float cs[4] = {cw.x, cw.y, cw.z, cw.w}, sn[4] = {sw.x, sw.y, sw.z, sw.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] = make_float2(g[e].x * cs[e] - g[e].y * sn[e], g[e].y * cs[e] + g[e].x * sn[e]);
          } else {
            const float2 cs[2] = {make_float2(cw.x, cw.y), make_float2(cw.z, cw.w)}, sn[2] = {make_float2(sw.x, sw.y), make_float2(sw.z, sw.w)};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 u = ga[2 * q + e], v = gc[2 * q + e];
              ga[2 * q + e] = __ffma2_rn(u, cs[e], minus(__fmul2_rn(v, sn[e])));
              gc[2 * q + e] = __ffma2_rn(v, cs[e], __fmul2_rn(u, sn[e]));
            }
          }
        }
      }
      if (norm_bwd) {
        if (here && which != of) {  // from the queries to the keys, or to the next span's queries
          keep();
          of = which;
        }
        float2 dot = both(0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = __fmul2_rn(a[e], both(r)), c[e] = __fmul2_rn(c[e], both(r));  // x r
          dw[e] = __ffma2_rn(ga[e], a[e], dw[e]), dw[4 + e] = __ffma2_rn(gc[e], c[e], dw[4 + e]);  // (zeros where nothing is)
          ga[e] = __fmul2_rn(ga[e], wa[e]), gc[e] = __fmul2_rn(gc[e], wc[e]);
          dot = __ffma2_rn(ga[e], a[e], __ffma2_rn(gc[e], c[e], dot));
        }
        const float2 mean = both(-team_sum<W>(here ? dot.x + dot.y : 0.f) * inv_d);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ga[e] = __fmul2_rn(both(r), __ffma2_rn(a[e], mean, ga[e]));
          gc[e] = __fmul2_rn(both(r), __ffma2_rn(c[e], mean, gc[e]));
        }
      }
      if (here) {
        const RotaryTensor& t = p.t[which];
        T* y = static_cast<T*>(t.out) + ((row0 + at) * t.heads + h) * p.d;
        Chunks<T>::store(y + c0, ga);
        Chunks<T>::store(y + c1, gc);
      }
    }
  }
  if constexpr (norm_bwd) {  // the CTA's sums, team after team
    if (active) keep();
    __syncthreads();
    // WAYS threads per column, then their sums
    constexpr int COLUMNS = 16 * W, WAYS = 256 / COLUMNS;
    const int c = threadIdx.x % COLUMNS, way = threadIdx.x / COLUMNS;
    for (int which = 0; which < 2; ++which) {
      if (!p.t[which].heads) continue;
      float sum = 0.f;
      for (int i = way; i < TEAMS; i += WAYS) sum += kept[which][i][c];
      __syncthreads();
      kept[which][way][c] = sum;  // (over what this way alone has read)
      __syncthreads();
      if (way == 0 && c < p.d) {
        for (int i = 1; i < WAYS; ++i) sum += kept[which][i][c];
        p.partial[((long long)which * gridDim.x + blockIdx.x) * p.d + c] = sum;
      }
    }
  }
}

// Any head size and any rotated part: a warp per head of a position, pair by pair.  Feature of pair i: half layout i and i + R / 2.  Bound by
// sines formed for every head (twice in the backward of a norm) and accesses of one feature: 8192 positions, 32 + 8 heads of 80 with 40 turned,
// bf16, 142 us a direction for 105 MB; heads of 40, all turned, 107 us for 52.
constexpr int kAnyMax = 512;  // features of a head
template <typename T>
__global__ void __launch_bounds__(256) rotary_any_kernel(const RotaryParams p) {
  wait_for_inputs();
  __shared__ float sums[8][kAnyMax];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, half = p.R / 2;
  for (int which = 0; which < 2; ++which) {
    const RotaryTensor& t = p.t[which];
    if (!t.heads) continue;
    const bool norm = t.w != nullptr;
    const long long mine = (long long)p.B * p.N * t.heads;
    for (int c = lane; c < p.d; c += 32) sums[warp][c] = 0.f;
    __syncwarp();
    for (long long item = (long long)blockIdx.x * 8 + warp; item < mine; item += (long long)gridDim.x * 8) {
      const int h = (int)(item % t.heads);
      const long long row = item / t.heads, b = row / p.N, n = row % p.N;
      const T* x = static_cast<const T*>(t.x) + b * t.sb + n * t.sn + (long long)h * p.d;
      const T* g = p.backward && norm ? static_cast<const T*>(t.dy) + b * t.gb + n * t.gn + (long long)h * p.d : x;
      T* y = static_cast<T*>(t.out) + (row * t.heads + h) * p.d;
      const long long pos = p.pos ? p.pos[b * p.pos_b + n] : p.start + n;
      auto at = [](const T* q, int c) -> float {
        if constexpr (sizeof(T) == 2) return __bfloat162float(q[c]);
        else return q[c];
      };
      auto put = [&](int c, float v) {
        if constexpr (sizeof(T) == 2) y[c] = __float2bfloat16(v);
        else y[c] = v;
      };
      float r = 1.f;
      if (norm) {
        float sq = 0.f;
        for (int c = lane; c < p.d; c += 32) sq = fmaf(at(x, c), at(x, c), sq);
        r = rsqrtf(team_sum<32>(sq) / p.d + p.eps);
      }
      // u(c): what is rotated; the rotated values of entry i: a pair below R / 2, then one feature each
      auto value = [&](int c) { return p.backward ? at(g, c) : norm ? at(x, c) * r * t.w[c] : at(x, c); };
      const int entries = half + p.d - p.R;
      auto rotated = [&](int i, int& c0, int& c1, float& v0, float& v1) {
        if (i < half) {
          c0 = p.interleaved ? 2 * i : i;
          c1 = p.interleaved ? c0 + 1 : i + half;
          const float2 s = cos_sin(p, pos, i);
          const float u0 = value(c0), u1 = value(c1);
          v0 = u0 * s.x - u1 * s.y;
          v1 = u1 * s.x + u0 * s.y;
        } else {
          c0 = i + half;
          c1 = -1;
          v0 = value(c0);
          v1 = 0.f;
        }
      };
      float mean = 0.f;
      if (p.backward && norm) {
        float dot = 0.f;
        for (int i = lane; i < entries; i += 32) {
          int c0, c1;
          float v0, v1;
          rotated(i, c0, c1, v0, v1);
          dot = fmaf(v0 * t.w[c0], at(x, c0) * r, dot);
          sums[warp][c0] += v0 * (at(x, c0) * r);
          if (c1 >= 0) {
            dot = fmaf(v1 * t.w[c1], at(x, c1) * r, dot);
            sums[warp][c1] += v1 * (at(x, c1) * r);
          }
        }
        mean = team_sum<32>(dot) / p.d;
      }
      for (int i = lane; i < entries; i += 32) {
        int c0, c1;
        float v0, v1;
        rotated(i, c0, c1, v0, v1);
        if (p.backward && norm) {
          v0 = r * (v0 * t.w[c0] - at(x, c0) * r * mean);
          if (c1 >= 0) v1 = r * (v1 * t.w[c1] - at(x, c1) * r * mean);
        }
        put(c0, v0);
        if (c1 >= 0) put(c1, v1);
      }
    }
    if (p.partial && norm) {
      __syncthreads();
      for (int c = threadIdx.x; c < p.d; c += 256) {
        float sum = 0.f;
        for (int i = 0; i < 8; ++i) sum += sums[i][c];
        p.partial[((long long)which * gridDim.x + blockIdx.x) * p.d + c] = sum;
      }
      __syncthreads();
    }
  }
}

bool in_chunks(const RotaryParams& p) {
  return p.vec && p.d % 16 == 0 && p.R % 16 == 0 && p.d <= 256 && p.t[0].heads < 1 << 16 && p.t[1].heads < 1 << 16;
}
int team_width(const RotaryParams& p) {  // lanes per head
  int w = 1;
  while (w < p.d / 16) w *= 2;
  return w;
}

template <typename T, int W>
cudaError_t by_mode(const RotaryParams& p, int grid, cudaStream_t st) {
  if (!p.t[0].w) return launch_behind(rotary_kernel<T, W, PLAIN>, dim3(grid), 256, 0, st, p);
  if (!p.backward) return launch_behind(rotary_kernel<T, W, NORM>, dim3(grid), 256, 0, st, p);
  return launch_behind(rotary_kernel<T, W, NORM_BWD>, dim3(grid), 256, 0, st, p);
}
template <typename T>
cudaError_t by_width(const RotaryParams& p, int grid, cudaStream_t st) {
  if (!in_chunks(p)) return launch_behind(rotary_any_kernel<T>, dim3(grid), 256, 0, st, p);
  switch (team_width(p)) {
    case 1: return by_mode<T, 1>(p, grid, st);
    case 2: return by_mode<T, 2>(p, grid, st);
    case 4: return by_mode<T, 4>(p, grid, st);
    case 8: return by_mode<T, 8>(p, grid, st);
    default: return by_mode<T, 16>(p, grid, st);
  }
}

}  // namespace

// Positions that a CTA takes at a time, CTAs that share one position's heads, and CTAs.  Sines, launch and first loads are the same for
// any span, so a span is as long as leaves two CTAs per SM (5997 positions, 18 heads of 96: 31.5 us with one position per CTA, 16.6 where 8
// CTAs are left per SM, 14.0 with 2; 32768 positions of 40 heads of 128: the same from 2 to 8, 26 % slower with one position), or half a
// one where its heads would not give each team one; with few positions their heads are spread out, a team each.  The
// backward of a norm takes 4 CTAs per SM at most, each with several spans: every CTA leaves a row of sums behind.
int rotary_plan(RotaryParams& p, int sms) {
  const long long rows = (long long)p.B * p.N, heads = p.t[0].heads;
  long long ctas;
  p.span = p.parts = 1;
  if (in_chunks(p)) {
    const int teams = 256 / team_width(p), most = p.R ? kRotaryTable / (p.R / 2) : kRotarySpan;
    auto doubled = [&](long long ctas_left) { return 2 * p.span <= most && 2 * p.span <= kRotarySpan && 2 * rows / (2 * p.span) >= ctas_left; };
    while (doubled(4ll * sms) || (p.span * (heads + p.t[1].heads) < teams && doubled(sms))) p.span *= 2;
    const long long spans = (rows + p.span - 1) / p.span;
    while (p.parts * teams < heads && spans * p.parts < 4ll * sms) ++p.parts;
    ctas = spans * p.parts;
    const long long cap = (p.partial ? 4ll : 1ll << 20) * sms;
    if (ctas > cap) ctas = cap / p.parts * p.parts;
  } else {
    ctas = (rows * heads + 7) / 8;
    if (ctas > kRotaryMostCtas) ctas = kRotaryMostCtas;
  }
  return (int)ctas;
}

cudaError_t launch_rotary(const RotaryParams& p, int dtype, int grid, cudaStream_t st) {
  return dtype == DT_BF16 ? by_width<__nv_bfloat16>(p, grid, st) : by_width<float>(p, grid, st);
}

}  // namespace ncn
