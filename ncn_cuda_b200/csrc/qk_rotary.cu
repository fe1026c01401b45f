// Rotary positions, and norms of queries and keys per head with the rotation in the same pass; forward and backward.
//
//   u = x r w,  r = 1 / sqrt(mean(x^2) + eps)          (or u = x, without a norm)
//   (a, b) pair i of u:  a' = M (a cos - b sin),  b' = M (b cos + a sin),  angle = position * frequency_i
// Backward: g = the cotangent rotated by the opposite angle;  dw = sum g x r,  dx = r (g w - x r mean(g w x r)).
//
// One pass over the data: 2 tensors forward, 3 backward, which is what bounds it.  Angles are formed in 64 bits as turns
// (position * frequency / 2 pi minus the nearest whole number), so that far positions lose nothing; what is left is below half a
// turn and goes through sincospi in 32 bits.  A sine and cosine cost 40 instructions, more than everything else of a pair of
// features: a team of lanes therefore keeps a position's in registers and walks the heads.
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

template <typename T> struct Chunk8;  // 8 features in registers
template <> struct Chunk8<__nv_bfloat16> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* at, float (&x)[8]) {
    const uint4 r = __ldcs(reinterpret_cast<const uint4*>(at));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* at, const float (&x)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(at) = *reinterpret_cast<uint4*>(h);
  }
};
template <> struct Chunk8<float> {
  static __device__ __forceinline__ void load(const float* at, float (&x)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(at)), b = __ldcs(reinterpret_cast<const float4*>(at) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* at, const float (&x)[8]) {
    reinterpret_cast<float4*>(at)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(at)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
};

template <int W>
__device__ __forceinline__ float team_sum(float x) {
#pragma unroll
  for (int s = W / 2; s; s >>= 1) x += __shfl_xor_sync(~0u, x, s);
  return x;
}

// Heads of d = 16 m features with R a multiple of 16: a team of W >= d / 16 lanes per head, 16 features per lane in two chunks of 8.
// Lane i < R / 16 holds the pairs 8 i .. 8 i + 7 (half layout: chunks i and i + R / 16; interleaved: chunks 2 i, 2 i + 1), the
// lanes behind it two chunks of the features that are not rotated.  `teams` teams share the heads of a position.
enum Mode : int { PLAIN = 0, NORM = 1, NORM_BWD = 2 };  // PLAIN: either direction
template <typename T, int W, int MODE>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  wait_for_inputs();
  constexpr bool norm = MODE != PLAIN, norm_bwd = MODE == NORM_BWD;
  const int lane = threadIdx.x % W, turning = p.R / 16;
  const bool active = lane < p.d / 16, turn = lane < turning;
  const int c0 = turn && !p.interleaved ? 8 * lane : 16 * lane, c1 = turn && !p.interleaved ? 8 * lane + p.R / 2 : c0 + 8;
  const long long per_cta = 256 / W, items = (long long)p.B * p.N * p.teams;
  const long long rounds = (items + per_cta * gridDim.x - 1) / (per_cta * gridDim.x);  // (the same for every lane: shuffles)
  float dw[2][16];  // (NORM_BWD)
#pragma unroll
  for (int e = 0; e < 16; ++e) dw[0][e] = dw[1][e] = 0.f;
  for (long long round = 0; round < rounds; ++round) {
    const long long item = (round * gridDim.x + blockIdx.x) * per_cta + threadIdx.x / W;
    const bool live = item < items;
    const int team = live ? (int)(item % p.teams) : 0;
    const long long row = live ? item / p.teams : 0, b = row / p.N, n = row % p.N;
    float2 cs[8];
    if (turn && live) {
      const long long pos = p.pos ? p.pos[b * p.pos_b + n] : p.start + n;
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[e] = cos_sin(p, pos, 8 * lane + e);
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const RotaryTensor& t = p.t[which];
      if (!t.heads) continue;
      float w[16];
      if (norm && active) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = t.w[c0 + e], w[8 + e] = t.w[c1 + e];
      }
      const int hs = (t.heads + p.teams - 1) / p.teams;
      for (int k = 0; k < hs; ++k) {
        const int h = team + k * p.teams;
        const bool here = live && active && h < t.heads;
        float a[8], c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = c[e] = 0.f;
        if (here) {
          const T* x = static_cast<const T*>(t.x) + b * t.sb + n * t.sn + (long long)h * p.d;
          Chunk8<T>::load(x + c0, a);
          Chunk8<T>::load(x + c1, c);
        }
        float r = 1.f;
        if (norm) {
          float sq = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sq = fmaf(a[e], a[e], fmaf(c[e], c[e], sq));
          r = rsqrtf(team_sum<W>(sq) / p.d + p.eps);
        }
        float ga[8], gc[8];
        if (norm_bwd) {
#pragma unroll
          for (int e = 0; e < 8; ++e) ga[e] = gc[e] = 0.f;
          if (here) {
            const T* g = static_cast<const T*>(t.dy) + b * t.gb + n * t.gn + (long long)h * p.d;
            Chunk8<T>::load(g + c0, ga);
            Chunk8<T>::load(g + c1, gc);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            ga[e] = norm ? a[e] * r * w[e] : a[e];
            gc[e] = norm ? c[e] * r * w[8 + e] : c[e];
          }
        }
        if (turn) {
          if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float2 s = cs[e / 2], u = cs[4 + e / 2];
              const float a0 = ga[e], a1 = ga[e + 1], b0 = gc[e], b1 = gc[e + 1];
              ga[e] = a0 * s.x - a1 * s.y, ga[e + 1] = a1 * s.x + a0 * s.y;
              gc[e] = b0 * u.x - b1 * u.y, gc[e + 1] = b1 * u.x + b0 * u.y;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float a0 = ga[e], b0 = gc[e];
              ga[e] = a0 * cs[e].x - b0 * cs[e].y;
              gc[e] = b0 * cs[e].x + a0 * cs[e].y;
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
          T* y = static_cast<T*>(t.out) + (row * t.heads + h) * p.d;
          Chunk8<T>::store(y + c0, ga);
          Chunk8<T>::store(y + c1, gc);
        }
      }
    }
  }
  if constexpr (norm_bwd) {  // the CTA's sums, team after team
    __shared__ float red[256 / W][16 * W + 1];
    for (int which = 0; which < 2; ++which) {
      if (!p.t[which].heads) continue;
      __syncthreads();
      if (active) {
#pragma unroll
        for (int e = 0; e < 8; ++e) red[threadIdx.x / W][c0 + e] = dw[which][e], red[threadIdx.x / W][c1 + e] = dw[which][8 + e];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < p.d; c += 256) {
        float sum = 0.f;
        for (int i = 0; i < 256 / W; ++i) sum += red[i][c];
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
int team_width(const RotaryParams& p) {
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

// Teams per position and CTAs.  Few positions: each head gets a team of its own.  Many: a team walks several heads with one set of
// sines, and there are still enough CTAs for the last ones not to be waited for.
int rotary_plan(RotaryParams& p, int sms) {
  const long long rows = (long long)p.B * p.N, heads = p.t[0].heads;
  long long ctas;
  if (in_chunks(p)) {
    const long long per_cta = 256 / team_width(p), want = (16ll * sms * per_cta + rows - 1) / rows;
    p.teams = (int)(want < 1 ? 1 : want > heads ? heads : want);
    ctas = (rows * p.teams + per_cta - 1) / per_cta;
  } else {
    p.teams = 1;
    ctas = (rows * heads + 7) / 8;
  }
  return (int)(ctas < kRotaryMostCtas ? ctas : kRotaryMostCtas);
}

cudaError_t launch_rotary(const RotaryParams& p, int dtype, int grid, cudaStream_t st) {
  return dtype == DT_BF16 ? by_width<__nv_bfloat16>(p, grid, st) : by_width<float>(p, grid, st);
}

}  // namespace ncn
