// Attention with a sliding window and sink tokens: what its kernels share.
//
// Query i of a row is at position p = start + i, key j at position j.  The query sees the key where
//   j < ctx,  j <= p < ctx  and  (p - j < window or j < n_sink),
// ctx the row's context length.  A query that sees nothing (padding, a position below zero) gives zeros.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ncn {

constexpr int kMaxLength = 1 << 28;  // of queries and keys: sums of three positions stay in 32 bits

struct AttnParams {
  const void *q, *k, *v;       // [B, N, heads * d] with the strides below, features of a position contiguous
  void* y;                     // [B, Nq, H * d], contiguous
  float* lse;                  // [B, H, Nqp], log2 of the softmax sums; +inf where nothing is seen.  May be null in the forward
  __nv_bfloat16* rest;         // bf16, kept with lse: what rounding took off y, itself rounded to bf16, [B, Nq, H * d].  May be null
  const void *dy, *y_in;       // backward: cotangent (strides) and output
  void *dq, *dk, *dv;          // contiguous
  float* delta;                // [B, H, Nqp]: sum(dy * y)
  float* part;                 // partial dk, dv of the sink keys: [B, Hk, sink tiles, chunks + 1, 2, sink rows, d]
  const int *ctxlen, *q_start; // per row, may be null
  long long sq_b, sq_n, sk_b, sk_n, sv_b, sv_n, sdy_b, sdy_n;
  int B, Nq, Nk, H, Hk, G, d, Nqp;
  int window, n_sink, start0, start_at_end;
  int sink_tiles, chunks, sink_rows;  // backward of the keys: tiles with sinks, pieces that queries beyond the window are cut into
  int vec;                     // rows may be read 16 bytes at a time
  float scale, scale_log2;     // of q.k: as it is, and times log2(e)
  int* status;
};

struct RowGeom {
  int ctx, start;
};
__device__ __forceinline__ RowGeom row_geom(const AttnParams& p, int b) {
  RowGeom g;
  g.ctx = p.ctxlen ? min(max(p.ctxlen[b], 0), p.Nk) : p.Nk;
  g.start = p.start_at_end ? g.ctx - p.Nq : min(max(p.q_start ? p.q_start[b] : p.start0, -p.Nq), p.Nk);  // (beyond these
  // no query sees anything, wherever it is)
  return g;
}

// Keys of a row that some query of the call sees: from `first` to `end`, and sinks before that.  What lies in other places (a cache behind
// the last query, in front of the window) may be anything, NaN included: where the weights' zeros would meet it in a product it is
// read as zero.
struct SeenKeys {
  int sinks, first, end;
  __device__ __forceinline__ bool has(int key) const { return key < end && (key >= first || key < sinks); }
  // whether one of keys k0 .. k0 + n - 1 (of Nk) is not seen
  __device__ __forceinline__ bool lacks(int k0, int n, int Nk) const {
    const int k1 = min(k0 + n, Nk);
    return k1 > end || max(k0, sinks) < min(k1, first);
  }
};
__device__ __forceinline__ SeenKeys seen_keys(const AttnParams& p, const RowGeom& g) {
  return SeenKeys{p.n_sink, max(g.start, 0) - p.window + 1, min(g.ctx, g.start + p.Nq)};
}
// Rows of a tile that are read: [lo, hi) without [gap_lo, gap_hi)
struct Rows {
  int lo, hi, gap_lo, gap_hi;
  __device__ __forceinline__ bool has(int r) const { return r >= lo && r < hi && !(r >= gap_lo && r < gap_hi); }
};
__device__ __forceinline__ Rows rows_between(int lo, int hi) { return Rows{lo, hi, 0, 0}; }
__device__ __forceinline__ Rows rows_seen(const SeenKeys& s, int k0) { return Rows{0, s.end - k0, s.sinks - k0, s.first - k0}; }

// A CTA's place: heads next to each other, so that a group reads its keys and values out of L2; then the tiles of a row; then rows.
// last_first counts the tiles from the last, which see the most keys.  One-dimensional, as batches may have more rows than the
// other two dimensions of a grid hold.
struct Block {
  int head, first_last, last_first, b;
};
__device__ __forceinline__ Block block_of(int heads, int tiles) {
  Block k;
  k.head = blockIdx.x % heads;
  const int rest = blockIdx.x / heads;
  k.first_last = rest % tiles;
  k.last_first = tiles - 1 - k.first_last;
  k.b = rest / tiles;
  return k;
}

// Key tiles of size T that queries i0 .. i1-1 need: tiles 0 .. ns-1 hold sinks, t0 .. t1 the window (t0 >= ns).
struct KeyTiles {
  int ns = 0, t0 = 0, t1 = -1, p_lo = 0, p_hi = -1;
  __device__ __forceinline__ int count() const { return ns + max(t1 - t0 + 1, 0); }
  __device__ __forceinline__ int tile(int i) const { return i < ns ? i : t0 + i - ns; }
  __device__ __forceinline__ int entry(int t) const { return t < ns ? t : t - t0 + ns; }  // the list's entry that tile t is
};
template <int T>
__device__ __forceinline__ KeyTiles key_tiles(const AttnParams& p, const RowGeom& g, int i0, int i1) {
  KeyTiles k;
  k.p_lo = max(g.start + i0, 0);
  k.p_hi = min(g.start + min(i1, p.Nq) - 1, g.ctx - 1);
  if (k.p_hi < k.p_lo || i0 >= p.Nq) {
    k.p_hi = k.p_lo - 1;
    return k;
  }
  k.ns = (min(p.n_sink, k.p_hi + 1) + T - 1) / T;
  k.t0 = max(k.ns, max(0, k.p_lo - p.window + 1) / T);
  k.t1 = k.p_hi / T;
  return k;
}

__device__ __forceinline__ bool sees(const AttnParams& p, int ctx, int pos, int key) {
  return key <= pos && pos < ctx && (pos - key < p.window || key < p.n_sink);
}

// whether queries i0 .. i0 + n - 1 see all of keys k0 .. k0 + m - 1
__device__ __forceinline__ bool sees_all(const AttnParams& p, const RowGeom& g, int i0, int n, int k0, int m) {
  const int lo = g.start + i0, hi = lo + n - 1;
  return i0 + n <= p.Nq && k0 + m - 1 <= lo && hi < g.ctx && (k0 > hi - p.window || k0 + m <= p.n_sink);
}

// Work items of the backward of the keys.  Item x < key tiles: the queries within reach of tile x's window (all of their pairs with
// the tile, sinks included).  Beyond these: piece c of the queries that see only the sinks of sink tile st.
// Query tiles of size TQ; `first .. last` of each of the G heads of the group, entries [begin, end) of the list head * tiles + tile.
struct KeyItem {
  int tile, chunk;  // chunk < 0: the window's queries
  int first, tiles, begin, end;
};
template <int T, int TQ>
__device__ __forceinline__ KeyItem key_item(const AttnParams& p, const RowGeom& g, int x) {
  const int key_tiles_n = (p.Nk + T - 1) / T;
  KeyItem it;
  it.chunk = -1;
  it.tile = x;
  if (x >= key_tiles_n) {
    it.tile = (x - key_tiles_n) / p.chunks;
    it.chunk = (x - key_tiles_n) % p.chunks;
  }
  const int k0 = it.tile * T;
  const int i_end = min(p.Nq - 1, g.ctx - 1 - g.start);                        // last query that is not padding
  const int lo = max(max(0, -g.start), k0 - g.start);                          // first one that may see a key of the tile
  const int hi = min(i_end, min(k0 + T - 1, g.ctx - 1) + p.window - 1 - g.start);  // last one within the window
  int first = lo / TQ, last = hi >= lo ? hi / TQ : first - 1;
  if (k0 >= g.ctx || i_end < lo) last = first - 1;
  if (it.chunk >= 0) {
    const bool any = k0 < g.ctx && i_end >= lo;
    first = last + 1;
    last = any ? i_end / TQ : first - 1;
  }
  it.first = first;
  it.tiles = max(last - first + 1, 0);
  it.begin = 0;
  it.end = it.tiles * p.G;
  if (it.chunk >= 0) {
    const int per = (it.end + p.chunks - 1) / p.chunks;
    it.begin = min(it.chunk * per, it.end);
    it.end = min(it.begin + per, it.end);
  }
  return it;
}
__device__ __forceinline__ float* part_of(const AttnParams& p, int b, int hk, int tile, int chunk) {
  const long long at = (((long long)b * p.Hk + hk) * p.sink_tiles + tile) * (p.chunks + 1) + chunk;
  return p.part + at * 2 * p.sink_rows * p.d;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
// A result and what rounding it takes off.  The backward's delta = sum(dy * y) is taken from every dP of a row: with the 8 bits of a bf16
// y it would bring an error as large as dS's own rounding where a query sees few keys (2 visible keys: 1.5 times the error of dq).
__device__ __forceinline__ void put_rest(float* p, float*, float v) { *p = v; }
__device__ __forceinline__ void put_rest(__nv_bfloat16* p, __nv_bfloat16* rest, float v) {
  const __nv_bfloat16 r = __float2bfloat16(v);
  *p = r;
  if (rest) *rest = __float2bfloat16(v - __bfloat162float(r));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// launchers
cudaError_t launch_attn_simt_fwd(const AttnParams& p, int dtype, cudaStream_t st);
cudaError_t launch_attn_simt_bwd(const AttnParams& p, int dtype, cudaStream_t st);
cudaError_t launch_attn_split_fwd(const AttnParams& p, cudaStream_t st);
cudaError_t launch_attn_split_bwd(const AttnParams& p, cudaStream_t st);  // (but for the sum of the sinks' parts)
cudaError_t launch_attn_sink_sum(const AttnParams& p, int dtype, int tile, cudaStream_t st);
cudaError_t launch_attn_decode(const AttnParams& p, int dtype, int sms, cudaStream_t st);

}  // namespace ncn
