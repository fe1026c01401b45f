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
  __shared__ __align__(16) float2 table[kRotaryTable];
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
  float dw[2][16];  // (NORM_BWD)  of the tensor that is being worked on, of the other
#pragma unroll
  for (int e = 0; e < 16; ++e) dw[0][e] = dw[1][e] = 0.f;
  int of = 0;  // the former
  for (long long row0 = (long long)(blockIdx.x / p.parts) * p.span; row0 < rows; row0 += stride) {
    const int span = (int)min((long long)p.span, rows - row0), of_q = span * p.t[0].heads, count = of_q + span * p.t[1].heads;
    const int turns = (count + step - 1) / step;  // the same for every lane: shuffles
    Chunks<T> x_next, g_next;
    auto place = [&](int i, int& which, int& at, int& h) {  // (i < 2^20: the product is off by less than what 0.5 leaves)
      which = i >= of_q;
      const int j = which ? i - of_q : i, heads = which ? p.t[1].heads : p.t[0].heads;
      at = (int)((j + 0.5f) * (which ? inv[1] : inv[0]));
      h = j - at * heads;
    };
    auto fetch = [&](int i) {
      x_next.clear();
      if (norm_bwd) g_next.clear();
      if (active && i < count) {
        int which, at, h;
        long long b, n;
        place(i, which, at, h);
        split(row0 + at, b, n);
        const RotaryTensor& t = p.t[which];
        x_next.load(static_cast<const T*>(t.x) + b * t.sb + n * t.sn + (long long)h * p.d, c0, c1);
        if (norm_bwd) g_next.load(static_cast<const T*>(t.dy) + b * t.gb + n * t.gn + (long long)h * p.d, c0, c1);
      }
    };
    fetch(first);
    __syncthreads();  // (the span before is done with the sines)
    for (int e = threadIdx.x; e < span * half; e += 256) {
      const int at = e / half;
      long long b, n;
      split(row0 + at, b, n);
      const int pair = e - at * half;
      table[at * half + (pair % 8 / 2 * turning + pair / 8) * 2 + pair % 2] = cos_sin(p, p.pos ? p.pos[b * p.pos_b + n] : p.start + n, pair);
    }
    __syncthreads();
    for (int k = 0; k < turns; ++k) {
      const int i = first + k * step;
      const bool here = active && i < count;
      int which, at, h;
      place(i, which, at, h);
      const float4* w = reinterpret_cast<const float4*>(weight) + which * 4 * W + lane;
      float a[8], c[8], ga[8], gc[8];
      Chunks<T>::widen(x_next.a, a);
      Chunks<T>::widen(x_next.c, c);
      if (norm_bwd) {
        Chunks<T>::widen(g_next.a, ga);
        Chunks<T>::widen(g_next.c, gc);
      }
      if (k + 1 < turns) fetch(i + step);
      float r = 1.f;
      if (norm) {
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sq = fmaf(a[e], a[e], fmaf(c[e], c[e], sq));
        r = rsqrtf(team_sum<W>(sq) * inv_d + p.eps);
        if (!here) r = 0.f;  // (infinite where eps is 0)
      }
      float wa[8], wc[8];
      if (norm) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 u = here ? w[e / 4 * W] : make_float4(0, 0, 0, 0), v = here ? w[(2 + e / 4) * W] : make_float4(0, 0, 0, 0);
          wa[e] = u.x, wa[e + 1] = u.y, wa[e + 2] = u.z, wa[e + 3] = u.w;
          wc[e] = v.x, wc[e + 1] = v.y, wc[e + 2] = v.z, wc[e + 3] = v.w;
        }
      }
      if (!norm_bwd) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ga[e] = norm ? a[e] * r * wa[e] : a[e];
          gc[e] = norm ? c[e] * r * wc[e] : c[e];
        }
      }
      if (turn && here) {
        const float4* tab = reinterpret_cast<const float4*>(table + at * half) + lane;  // (entry e: the lane's pairs 2 e, 2 e + 1)
        if (p.interleaved) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 s = tab[e * turning], u = tab[(2 + e) * turning];
            float y0 = ga[4 * e], y1 = ga[4 * e + 1];
            ga[4 * e] = y0 * s.x - y1 * s.y, ga[4 * e + 1] = y1 * s.x + y0 * s.y;
            y0 = ga[4 * e + 2], y1 = ga[4 * e + 3];
            ga[4 * e + 2] = y0 * s.z - y1 * s.w, ga[4 * e + 3] = y1 * s.z + y0 * s.w;
            y0 = gc[4 * e], y1 = gc[4 * e + 1];
            gc[4 * e] = y0 * u.x - y1 * u.y, gc[4 * e + 1] = y1 * u.x + y0 * u.y;
            y0 = gc[4 * e + 2], y1 = gc[4 * e + 3];
            gc[4 * e + 2] = y0 * u.z - y1 * u.w, gc[4 * e + 3] = y1 * u.z + y0 * u.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float4 s = tab[e / 2 * turning];
            float a0 = ga[e], b0 = gc[e];
            ga[e] = a0 * s.x - b0 * s.y, gc[e] = b0 * s.x + a0 * s.y;
            a0 = ga[e + 1], b0 = gc[e + 1];
            ga[e + 1] = a0 * s.z - b0 * s.w, gc[e + 1] = b0 * s.z + a0 * s.w;
          }
        }
      }
      if (norm_bwd) {
        if (here && which != of) {  // from the queries to the keys, or to the next span's queries
          of = which;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float t = dw[0][e];
            dw[0][e] = dw[1][e];
            dw[1][e] = t;
          }
        }
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[e] *= r, c[e] *= r;  // x r
          dw[0][e] = fmaf(ga[e], a[e], dw[0][e]), dw[0][8 + e] = fmaf(gc[e], c[e], dw[0][8 + e]);  // (zeros where nothing is)
          ga[e] *= wa[e], gc[e] *= wc[e];
          dot = fmaf(ga[e], a[e], fmaf(gc[e], c[e], dot));
        }
        const float mean = team_sum<W>(dot) * inv_d;
#pragma unroll
        for (int e = 0; e < 8; ++e) ga[e] = r * (ga[e] - a[e] * mean), gc[e] = r * (gc[e] - c[e] * mean);
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
    __shared__ float red[TEAMS][16 * W + 1];
    for (int which = 0; which < 2; ++which) {
      if (!p.t[which].heads) continue;
      __syncthreads();
      if (active) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          red[team][c0 + e] = which == of ? dw[0][e] : dw[1][e];
          red[team][c1 + e] = which == of ? dw[0][8 + e] : dw[1][8 + e];
        }
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

// Positions that a CTA takes at a time, CTAs that share one position's heads, and CTAs.  A span is as long as leaves 8 CTAs per SM
// (the last ones are not waited for long), its sines are formed once; with few positions their heads are spread out, a team each.  The
// backward of a norm takes 4 CTAs per SM at most, each with several spans: every CTA leaves a row of sums behind.
int rotary_plan(RotaryParams& p, int sms) {
  const long long rows = (long long)p.B * p.N, heads = p.t[0].heads;
  long long ctas;
  p.span = p.parts = 1;
  if (in_chunks(p)) {
    const int teams = 256 / team_width(p), most = p.R ? kRotaryTable / (p.R / 2) : kRotarySpan;
    while (2 * p.span <= most && 2 * p.span <= kRotarySpan && rows / (2 * p.span) >= 8ll * sms) p.span *= 2;
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
