// Rotary positions, and norms of queries and keys per head with the rotation in the same pass; forward and backward.
//
//   u = x r w,  r = 1 / sqrt(mean(x^2) + eps)          (or u = x, without a norm)
//   (a, b) pair i of u:  a' = M (a cos - b sin),  b' = M (b cos + a sin),  angle = position * frequency_i
// Backward: g = the cotangent rotated by the opposite angle;  dw = sum g x r,  dx = r (g w - x r mean(g w x r)).
//
// One pass over the data: 2 tensors forward, 3 backward, which is what bounds it.  Angles are formed in 64 bits as turns
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
  static __device__ __forceinline__ void widen(const uint4 (&r)[V], float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 2) {
          x[2 * e] = __uint_as_float(w[e] << 16);
          x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        } else {
          x[4 * i + e] = __uint_as_float(w[e]);
        }
      }
    }
  }
  static __device__ __forceinline__ void store(T* at, const float (&x)[8]) {
    if constexpr (sizeof(T) == 2) {
      __nv_bfloat162 h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      *reinterpret_cast<uint4*>(at) = *reinterpret_cast<uint4*>(h);
    } else {
      reinterpret_cast<float4*>(at)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(at)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
  }
};

template <int W>
__device__ __forceinline__ float team_sum(float x) {
#pragma unroll
  for (int s = W / 2; s; s >>= 1) x += __shfl_xor_sync(~0u, x, s);
  return x;
}

// Heads of d = 16 m features with R a multiple of 16: a team of W >= d / 16 lanes per head, 16 features per lane in two chunks of 8.
// Lane i < R / 16 holds the pairs 8 i .. 8 i + 7 (half layout: chunks i and i + R / 2 / 8; interleaved: chunks 2 i, 2 i + 1), the
// lanes behind it two chunks of the features that are not rotated.  A CTA takes p.span positions at a time, their heads dealt out to its
// teams (and to p.parts CTAs, where there are few positions); the next head is fetched while one is worked on.
enum Mode : int { PLAIN = 0, NORM = 1, NORM_BWD = 2 };  // PLAIN: either direction
template <typename T, int W, int MODE>
__global__ void __launch_bounds__(256, MODE == NORM_BWD ? 2 : 4) rotary_kernel(const __grid_constant__ RotaryParams p) {
  wait_for_inputs();
  constexpr bool norm = MODE != PLAIN, norm_bwd = MODE == NORM_BWD;
  constexpr int TEAMS = 256 / W;
  __shared__ long long offs[4][kRotarySpan];  // of the span's positions in q, k and their cotangents
  __shared__ __align__(16) float2 table[kRotaryTable];
  const int lane = threadIdx.x % W, team = threadIdx.x / W, half = p.R / 2;
  const bool active = lane < p.d / 16, turn = lane < p.R / 16;
  const int c0 = turn && !p.interleaved ? 8 * lane : 16 * lane, c1 = turn && !p.interleaved ? 8 * lane + half : c0 + 8;
  const int part = blockIdx.x % p.parts;
  const long long rows = (long long)p.B * p.N, stride = (long long)(gridDim.x / p.parts) * p.span;
  float dw[2][16];  // (NORM_BWD)
#pragma unroll
  for (int e = 0; e < 16; ++e) dw[0][e] = dw[1][e] = 0.f;
  for (long long row0 = (long long)(blockIdx.x / p.parts) * p.span; row0 < rows; row0 += stride) {
    const int span = (int)min((long long)p.span, rows - row0);
    __syncthreads();
    for (int e = threadIdx.x; e < span * half; e += 256) {
      const long long row = row0 + e / half, b = row / p.N, n = row - b * p.N;
      table[e] = cos_sin(p, p.pos ? p.pos[b * p.pos_b + n] : p.start + n, e % half);
    }
    if (threadIdx.x < span) {
      const long long row = row0 + threadIdx.x, b = row / p.N, n = row - b * p.N;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        offs[which][threadIdx.x] = b * p.t[which].sb + n * p.t[which].sn;
        offs[2 + which][threadIdx.x] = b * p.t[which].gb + n * p.t[which].gn;
      }
    }
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const RotaryTensor& t = p.t[which];
      if (!t.heads) continue;
      float w[16];
      if (norm && active) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = t.w[c0 + e], w[8 + e] = t.w[c1 + e];
      }
      const int count = span * t.heads, step = p.parts * TEAMS, first = part * TEAMS + team;
      const int turns = (count + step - 1) / step;  // the same for every lane: shuffles
      auto fetch = [&](int i, Chunks<T>& x, Chunks<T>& g) {
        const bool here = active && i < count;
        x.clear();
        if (norm_bwd) g.clear();
        if (here) {
          const int at = i / t.heads, h = i - at * t.heads;
          x.load(static_cast<const T*>(t.x) + offs[which][at] + h * p.d, c0, c1);
          if (norm_bwd) g.load(static_cast<const T*>(t.dy) + offs[2 + which][at] + h * p.d, c0, c1);
        }
      };
      Chunks<T> x_next, g_next;
      fetch(first, x_next, g_next);
      for (int k = 0; k < turns; ++k) {
        const int i = first + k * step, at = i / t.heads;
        const bool here = active && i < count;
        float a[8], c[8], ga[8], gc[8];
        Chunks<T>::widen(x_next.a, a);
        Chunks<T>::widen(x_next.c, c);
        if (norm_bwd) {
          Chunks<T>::widen(g_next.a, ga);
          Chunks<T>::widen(g_next.c, gc);
        }
        if (k + 1 < turns) fetch(i + step, x_next, g_next);
        float r = 1.f;
        if (norm) {
          float sq = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sq = fmaf(a[e], a[e], fmaf(c[e], c[e], sq));
          r = rsqrtf(team_sum<W>(sq) / p.d + p.eps);
        }
        if (!norm_bwd) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            ga[e] = norm ? a[e] * r * w[e] : a[e];
            gc[e] = norm ? c[e] * r * w[8 + e] : c[e];
          }
        }
        if (turn && here) {
          const float4* tab = reinterpret_cast<const float4*>(table + at * half + 8 * lane);  // (two pairs each; half is a multiple of 8)
          if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float4 s = tab[e / 2], u = tab[2 + e / 2];
              float y0 = ga[2 * e], y1 = ga[2 * e + 1];
              ga[2 * e] = y0 * s.x - y1 * s.y, ga[2 * e + 1] = y1 * s.x + y0 * s.y;
              y0 = ga[2 * e + 2], y1 = ga[2 * e + 3];
              ga[2 * e + 2] = y0 * s.z - y1 * s.w, ga[2 * e + 3] = y1 * s.z + y0 * s.w;
              y0 = gc[2 * e], y1 = gc[2 * e + 1];
              gc[2 * e] = y0 * u.x - y1 * u.y, gc[2 * e + 1] = y1 * u.x + y0 * u.y;
              y0 = gc[2 * e + 2], y1 = gc[2 * e + 3];
              gc[2 * e + 2] = y0 * u.z - y1 * u.w, gc[2 * e + 3] = y1 * u.z + y0 * u.w;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float4 s = tab[e / 2];
              float a0 = ga[e], b0 = gc[e];
              ga[e] = a0 * s.x - b0 * s.y, gc[e] = b0 * s.x + a0 * s.y;
              a0 = ga[e + 1], b0 = gc[e + 1];
              ga[e + 1] = a0 * s.z - b0 * s.w, gc[e + 1] = b0 * s.z + a0 * s.w;
            }
          }
        }
        if (norm_bwd) {
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            a[e] *= r, c[e] *= r;  // x r
            if (here) dw[which][e] = fmaf(ga[e], a[e], dw[which][e]), dw[which][8 + e] = fmaf(gc[e], c[e], dw[which][8 + e]);
            ga[e] *= here ? w[e] : 0.f, gc[e] *= here ? w[8 + e] : 0.f;
            dot = fmaf(ga[e], a[e], fmaf(gc[e], c[e], dot));
          }
          const float mean = team_sum<W>(dot) / p.d;
#pragma unroll
          for (int e = 0; e < 8; ++e) ga[e] = r * (ga[e] - a[e] * mean), gc[e] = r * (gc[e] - c[e] * mean);
        }
        if (here) {
          T* y = static_cast<T*>(t.out) + (row0 * t.heads + i) * p.d;
          Chunks<T>::store(y + c0, ga);
          Chunks<T>::store(y + c1, gc);
        }
      }
    }
  }
  if constexpr (norm_bwd) {  // the CTA's sums, team after team
    __shared__ float red[TEAMS][16 * W + 1];
    for (int which = 0; which < 2; ++which) {
      if (!p.t[which].heads) continue;
      __syncthreads();
      if (active) {
#pragma unroll
        for (int e = 0; e < 8; ++e) red[team][c0 + e] = dw[which][e], red[team][c1 + e] = dw[which][8 + e];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < p.d; c += 256) {
        float sum = 0.f;
        for (int i = 0; i < TEAMS; ++i) sum += red[i][c];
        p.partial[((long long)which * gridDim.x + blockIdx.x) * p.d + c] = sum;
      }
    }
  }
}

// Any head size and any rotated part: a warp per head of a position, pair by pair.  Feature of pair i: half layout i and i + R / 2.
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

bool in_chunks(const RotaryParams& p) { return p.vec && p.d % 16 == 0 && p.R % 16 == 0 && p.d <= 256; }
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

// Positions that a CTA takes at a time, CTAs that share one position's heads, and CTAs.  A span is as long as leaves 16 CTAs per SM
// (the last ones are not waited for long), its sines are formed once; with few positions their heads are spread out, a team each.  The
// backward of a norm takes 4 CTAs per SM at most, each with several spans: every CTA leaves a row of sums behind.
int rotary_plan(RotaryParams& p, int sms) {
  const long long rows = (long long)p.B * p.N, heads = p.t[0].heads;
  long long ctas;
  p.span = p.parts = 1;
  if (in_chunks(p)) {
    const int teams = 256 / team_width(p), most = p.R ? kRotaryTable / (p.R / 2) : kRotarySpan;
    while (2 * p.span <= most && 2 * p.span <= kRotarySpan && rows / (2 * p.span) >= 16ll * sms) p.span *= 2;
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
