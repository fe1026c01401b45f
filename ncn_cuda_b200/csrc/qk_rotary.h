// Norms of queries and keys per head, and rotary positions: parameters of the kernels of qk_rotary.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ncn {

struct RotaryTensor {
  const void* x;    // [B, N, heads * d], features of a position contiguous; the cotangent where no norm is walked back
  const void* dy;   // backward of the norm: the cotangent, with strides of its own
  const float* w;   // [d] or null: no norm
  void* out;        // y, or dx in the backward; contiguous
  long long sb, sn, gb, gn;  // strides of x and dy, in elements
  int heads;
};
struct RotaryParams {
  RotaryTensor t[2];        // queries, keys (heads 0: absent)
  const double* freqs;      // [R / 2], radians per position
  const long long* pos;     // positions, [N] or [B, N], or null: start, start + 1, ...
  long long pos_b, start;   // stride of a row of positions (0: the same for all)
  float* partial;           // backward of the norm: [2][grid][d]
  int B, N, d, R;
  int interleaved, backward, vec;
  int span, parts;          // positions that a CTA takes at a time, CTAs that share their heads
  float eps, magnitude;
};

constexpr int kRotarySpan = 16, kRotaryTable = 1024;  // most positions of a span; its pairs of sines
constexpr long long kRotaryMostCtas = 8192;  // of a launch: rows of partial sums
int rotary_plan(RotaryParams& p, int sms);  // sets span and parts; returns the CTAs of a launch
cudaError_t launch_rotary(const RotaryParams& p, int dtype, int grid, cudaStream_t st);

}  // namespace ncn
