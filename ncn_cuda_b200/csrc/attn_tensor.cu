// Windowed attention on the 5th-generation tensor cores: bf16 storage, heads of up to 128 features (a multiple of 8), fp32 sums.
//
// All three kernels have the same parts.  One warp fetches tiles of 128 positions by TMA into a ring of slots in shared memory, one
// warp issues the matrix instructions (tcgen05.mma, one thread), eight warps work on the scores.  Scores and sums stay in
// tensor memory; the weights go back there in bf16, over the scores that they came from, and are the left operand of the second
// product straight from there.  A tile is DP / 64 blocks of [128 positions][64 features], each row of 128 bytes swizzled by the
// TMA unit; the same tile serves as an operand along its features (scores) and along its positions (second products).
// Heads whose size is not 64 or 128 are filled up with zeros by the TMA unit.
//
// Rows of padding (behind ctxlen) and places that no query of the call sees may hold anything, NaN included: scores are masked by
// selection, and the rows that a second product would multiply by zero weights are cleared in shared memory first.
//
// The backward is two kernels, one that owns queries and one that owns keys.  It computes the scores twice, 7 products for 5, and in
// return no sum depends on the order in which CTAs finish.
//
// Rounded to bf16: the weights P and the gradients dS, as operands of the second products (each term off by at
// most 2^-8, like the results' own rounding: results end up about 1.4 times as far from the exact ones as that alone puts them).  Scores,
// softmax sums, delta and all sums over keys or queries are fp32.
//
// Measured (2 x 4096 positions, 16 heads of 128 on 4 of keys, windows of 1024, 4 sinks): forward 89 us, dq 126, dk and dv 123, 680 to 980
// TFLOP/s over the visible pairs; 16384 positions, windows of 4096: forward 428 us, 1120 TFLOP/s (1688 is what plain matrix products
// reach).  Per tile the bound is the exchange between the two sides: 3000 cycles per pair of tiles against 2048 of the products
// alone (score to weight to product, each waiting for the one before).  For short windows it is the CTA: first loads, epilogue
// and uneven ends take some 10 us of each, and 256 or 512 of them on 148 SMs leave the last round part empty.
#include <cuda.h>

#include "attn_tensor.h"
#include "ncn_common.cuh"

namespace ncn {
namespace {

constexpr int kT = 128;               // positions of a tile
constexpr int kThreads = 352;         // backward: warps 0-7 scores, 8 products, 9 TMA, 10 padding
constexpr int kFwdThreads = 608;      // forward: warps 0-15 scores, 16 products, 17 TMA, 18 padding
constexpr uint32_t kBlockBytes = kT * 128;
constexpr uint64_t kWaitLimitNs = 4000000000ull;

// ------------------------------------------------------------------ PTX
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols));
}
__device__ __forceinline__ void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns of the lane's row
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t (&x)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]),
        "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]), "=r"(x[20]),
        "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]), "=r"(x[28]), "=r"(x[29]), "=r"(x[30]),
        "=r"(x[31])
      : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t (&x)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31};" ::"r"(x[0]),
      "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]), "r"(x[9]), "r"(x[10]), "r"(x[11]), "r"(x[12]),
      "r"(x[13]), "r"(x[14]), "r"(x[15]), "r"(x[16]), "r"(x[17]), "r"(x[18]), "r"(x[19]), "r"(x[20]), "r"(x[21]), "r"(x[22]), "r"(x[23]),
      "r"(x[24]), "r"(x[25]), "r"(x[26]), "r"(x[27]), "r"(x[28]), "r"(x[29]), "r"(x[30]), "r"(x[31]), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_load32f(uint32_t at, float (&x)[32]) { tmem_load32(at, reinterpret_cast<uint32_t(&)[32]>(x)); }
__device__ __forceinline__ void tmem_store32f(uint32_t at, float (&x)[32]) { tmem_store32(at, reinterpret_cast<uint32_t(&)[32]>(x)); }
__device__ __forceinline__ void tmem_load16f(uint32_t at, float (&x)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]), "=f"(x[9]),
                 "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15])
               : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(x[0]), "r"(x[1]), "r"(x[2]),
      "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]), "r"(x[9]), "r"(x[10]), "r"(x[11]), "r"(x[12]), "r"(x[13]), "r"(x[14]),
      "r"(x[15]), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t at, const uint32_t (&x)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]),
               "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(at)
               : "memory");
}
// Waits for the loads; the values are tied to it, so that nothing made of them is moved ahead of the wait.
template <int N>
__device__ __forceinline__ void tmem_tie(float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("" : "+f"(x[i]), "+f"(x[i + 1]), "+f"(x[i + 2]), "+f"(x[i + 3]), "+f"(x[i + 4]), "+f"(x[i + 5]), "+f"(x[i + 6]), "+f"(x[i + 7]));
}
template <int N>
__device__ __forceinline__ void tmem_loaded(float (&x)[N][32]) {
  tmem_wait_load();
#pragma unroll
  for (int c = 0; c < N; ++c) tmem_tie(x[c]);
}
template <int N>
__device__ __forceinline__ void tmem_loaded(float (&x)[N]) {
  tmem_wait_load();
  tmem_tie(x);
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// arrives on `bar` when the products issued so far are done
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// One instruction's products.  Operands in shared memory are given by the low halves of their descriptors, the high half is the same for
// all: what the issuing thread computes per instruction is two 32-bit additions.  (With whole descriptors formed for each, an instruction
// took 90 to 130 cycles to issue, and 64 to execute: heads of 128 in windows of 2048, 4300 cycles per pair of tiles.)
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);  // rows of 8 x 128 bytes 1024 apart, version 1, 128-byte swizzle
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((int)add), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((int)add), "n"(kDescHigh)
      : "memory");
}
// one lane of a warp whose lanes are all here
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int c, int head, int row, int b, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                   dst),
               "l"(map), "r"(c), "r"(head), "r"(row), "r"(b), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, int c, int head, int row, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map), "r"(src), "r"(c), "r"(head),
               "r"(row), "r"(b)
               : "memory");
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// Operand descriptors.  Along the features ("k-major") the 16 features of an instruction are 32 bytes on; along the positions
// ("mn-major") the 64-feature blocks are kBlockBytes apart, 16 positions 2048 bytes on.  Addresses and distances in units of 16 bytes.
__device__ __forceinline__ uint32_t desc_low(uint32_t smem, uint32_t lead) { return ((smem & 0x3ffffu) >> 4) | ((lead >> 4) << 16); }
template <int N, bool MN>
__device__ __forceinline__ constexpr uint32_t idesc_of() {  // fp32 sums, bf16 operands, 128 x N
  return (1u << 4) | (1u << 7) | (1u << 10) | (MN ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kT >> 4) << 24);
}
// D[128 x 128] = A B^T over DP features; A, B tiles
template <int DP>
__device__ __forceinline__ void product_scores(uint32_t d, uint32_t a, uint32_t b) {
  const uint32_t la = desc_low(a, 16), lb = desc_low(b, 16);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const uint32_t off = ((k / 4) * kBlockBytes + (k % 4) * 32) >> 4;
    mma_ss(d, la + off, lb + off, idesc_of<kT, false>(), k > 0);
  }
}
// D[128 x DP] (+)= W V over 64 of 128 positions: 0 .. 31 and 64 .. 95 (HALF 0) or the others.  W bf16 in tensor memory, two positions per
// column, positions 64 .. 127 64 columns on; V a tile.  Two threads share a row of weights, and each hands in its first 32 before it
// makes the others.
template <int DP, int HALF>
__device__ __forceinline__ void product_sums(uint32_t d, uint32_t w, uint32_t v, bool add) {
  const uint32_t lv = desc_low(v, kBlockBytes);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = i / 2 * 4 + i % 2 + 2 * HALF;
    mma_ts(d, w + (k / 4) * 64 + (k % 4) * 8, lv + k * (2048 >> 4), idesc_of<DP, true>(), add || i > 0 || HALF > 0);
  }
}

// A wait that gives up: the kernel then leaves an error in the status word, and its other warps stop waiting too.
struct Waiter {
  volatile int* stop;
  int* status;
  __device__ __forceinline__ bool one(uint64_t* bar, uint32_t parity) const {
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    const uint64_t begin = now_ns();
    while (!mbar_try_wait(bar, parity)) {
      if (*stop) return false;
      if (now_ns() - begin > kWaitLimitNs) {
        *stop = 1;
        if (status) atomicExch(status, (int)DEV_WAIT_TIMEOUT);
        return false;
      }
    }
    return true;
  }
  // a whole warp: one answer for all of its lanes
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const { return __all_sync(~0u, one(bar, parity)); }
};

// A ring of tile slots, and a place in it that moves on by one
template <int SLOTS>
struct Ring {
  uint64_t *full, *empty;
  uint32_t mem, bytes;
  struct Place {
    int slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
      if (++slot == SLOTS) slot = 0, parity ^= 1;
    }
  };
  __device__ __forceinline__ Place place(int i) const {
    Place p;
    p.slot = i % SLOTS;
    p.parity = (i / SLOTS) & 1;
    return p;
  }
  __device__ __forceinline__ uint32_t at(const Place& p) const { return mem + p.slot * bytes; }
  __device__ __forceinline__ uint64_t* arrived(const Place& p) const { return full + p.slot; }
  __device__ __forceinline__ bool wait_full(const Waiter& w, const Place& p) const { return w.one(full + p.slot, p.parity); }
  __device__ __forceinline__ bool wait_empty(const Waiter& w, const Place& p) const { return w.one(empty + p.slot, p.parity ^ 1); }  // (free at first)
  __device__ __forceinline__ void release(const Place& p) const { mma_commit(empty + p.slot); }
};

template <int DP>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int head, int row, int b, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) tma_load(dst + c * kBlockBytes, map, c * 64, head, row, b, bar);
}
// Clears the rows of a tile that `keep` does not name; a whole warp.  The thread that issues the products has seen the tile arrive, asks for it
// (`go`) and waits (`cleared`) before it goes on: one tile at a time, so neither can be a phase ahead.
template <int DP, typename Keep>
__device__ __forceinline__ void clear_rows(uint32_t tile, Keep keep, uint64_t* cleared) {
  const int lane = threadIdx.x % 32;
  for (int e = lane; e < kT * DP / 8; e += 32) {
    const int r = e % (kT * 8) / 8;
    if (!keep(r))
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + e / (kT * 8) * kBlockBytes + e % (kT * 8) * 16), "r"(0) : "memory");
  }
  fence_proxy_async();
  __syncwarp();
  if (lane == 0) mbar_arrive(cleared);
}
__device__ __forceinline__ bool have_cleared(const Waiter& wait, uint64_t* go, uint64_t* cleared, uint32_t phase) {
  mbar_arrive(go);
  return wait.one(cleared, phase);
}

__device__ __forceinline__ void lds128(uint32_t at, uint32_t (&x)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Exponentials.  The special-function pipe gives 16 per SM and cycle, 1024 cycles per tile of 128 x 128, as long as both products of heads
// of 128 take; so some pairs (kOnFma of 8; 2 and 3 measured best, 0 and 4 two to four per cent slower) are computed on the FMA pipe instead, two at a time: 2^x = 2^n 2^f, n the nearest whole number,
// |f| <= 1/2, 2^f by the polynomial of degree 4 of least relative error (Remez exchange; 2.6e-6 = 2^-18.6, a thousandth of the weights'
// rounding to bf16).  From -127 down 2^n has the bits of zero, and so has the result, minus infinity's too.  NaN stays NaN.
constexpr int kOnFma = 2;
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.f));
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it leaves the nearest whole number in the low bits
  const float2 t = __fadd2_rn(x, make_float2(kRound, kRound));
  const float2 n = __fadd2_rn(t, make_float2(-kRound, -kRound));
  const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
  float2 p = __ffma2_rn(f, make_float2(0.009570101911f, 0.009570101911f), make_float2(0.05591786032f, 0.05591786032f));
  p = __ffma2_rn(p, f, make_float2(0.2402474483f, 0.2402474483f));
  p = __ffma2_rn(p, f, make_float2(0.6931218147f, 0.6931218147f));
  p = __ffma2_rn(p, f, make_float2(0.9999992614f, 0.9999992614f));
  const float2 two_n = make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000));
  return __fmul2_rn(p, two_n);
}
// a, b = 2^(a scale + bias), 2^(b scale + bias); pair: its number
__device__ __forceinline__ void exp2_pair(float& a, float& b, float2 scale, float2 bias, int pair) {
  float2 x = __ffma2_rn(make_float2(a, b), scale, bias);
  if (pair % 8 < kOnFma)
    x = exp2_fma(x);
  else
    x = make_float2(ex2(x.x), ex2(x.y));
  a = x.x, b = x.y;
}
// Results leave through shared memory and the TMA unit: rows written by their threads straight to global memory, 16 bytes per lane and
// row, took a third of the forward's time in windows of 1024 (15000 of 51000 cycles).  32 features of row r, c0 .. c0 + 31,
// into a tile laid out as the TMA unit has it.
__device__ __forceinline__ void stage_row(uint32_t tile, int r, const float (&x)[32], float f, int c0) {
#pragma unroll
  for (int e = 0; e < 32; e += 8) {
    const int c = c0 + e;
    const uint32_t at = tile + (c / 64) * kBlockBytes + r * 128 + ((c % 64 / 8 ^ (r & 7)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(pack(x[e] * f, x[e + 1] * f)), "r"(pack(x[e + 2] * f, x[e + 3] * f)),
                 "r"(pack(x[e + 4] * f, x[e + 5] * f)), "r"(pack(x[e + 6] * f, x[e + 7] * f))
                 : "memory");
  }
}
// The same for a warp's 32 rows by themselves (rows of 64 bytes), on their way when its lanes are done: no other warp is waited for.  Rows
// and features beyond the tensor are left out.  OTHERS: how many of the sends before may still be reading, from other places.
template <int OTHERS>
__device__ __forceinline__ void send_rows(const CUtensorMap* map, uint32_t at, const float (&x)[32], float f, int c, int head, int row, int b) {
  const int lane = threadIdx.x % 32;
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(OTHERS) : "memory");
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 32; e += 8)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + lane * 64 + ((e / 8 ^ (lane >> 1 & 3)) << 4)),
                 "r"(pack(x[e] * f, x[e + 1] * f)), "r"(pack(x[e + 2] * f, x[e + 3] * f)), "r"(pack(x[e + 4] * f, x[e + 5] * f)),
                 "r"(pack(x[e + 6] * f, x[e + 7] * f))
                 : "memory");
  fence_proxy_async();
  __syncwarp();
  if (lane == 0) {
    tma_store(map, at, c, head, row, b);
    bulk_commit();
  }
}
// what the rounding in stage_row takes off, to be staged itself
__device__ __forceinline__ void keep_rest(float (&x)[32], float f) {
#pragma unroll
  for (int e = 0; e < 32; ++e) x[e] = x[e] * f - __bfloat162float(__float2bfloat16(x[e] * f));
}
// A staged tile (written, fenced and handed in by its threads) to global memory; rows and features beyond the tensor are left out.
template <int DP>
__device__ __forceinline__ void send_tile(const CUtensorMap* map, uint32_t tile, int head, int row, int b) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) tma_store(map, tile + c * kBlockBytes, c * 64, head, row, b);
  bulk_commit();
}
// 32 features of a row to global memory, c0 .. c0 + 31 of d (a multiple of 8)
__device__ __forceinline__ void store_row(__nv_bfloat16* row, const float (&x)[32], float f, int c0, int d) {
#pragma unroll
  for (int e = 0; e < 32; e += 8)
    if (c0 + e < d)
      *reinterpret_cast<uint4*>(row + c0 + e) = make_uint4(pack(x[e] * f, x[e + 1] * f), pack(x[e + 2] * f, x[e + 3] * f),
                                                           pack(x[e + 4] * f, x[e + 5] * f), pack(x[e + 6] * f, x[e + 7] * f));
}

// After a wait that gave up: what is on its way to the last loads' slots arrives before the memory is given up.
template <int SLOTS>
__device__ __forceinline__ void settle(const Ring<SLOTS>& ring, int loads) {
  for (int e = loads > SLOTS ? loads - SLOTS : 0; e < loads; ++e) {
    const auto at = ring.place(e);
    mbar_wait_bounded(ring.full + at.slot, at.parity, 1u << 16);
  }
}

struct Maps {
  CUtensorMap q, k, v, dy, y, rest, dq, dk, dv;  // (the direction's own)
};

// The keys of tile k0 that a query at `pos` sees, as columns: [lo, hi), and those below `sink`
struct Columns {
  int lo, hi, sink;
};
__device__ __forceinline__ Columns columns_of(const AttnParams& p, int pos, int end, int k0) {
  Columns c;
  const bool live = pos >= 0 && pos < end;
  c.hi = live ? pos + 1 - k0 : 0;
  c.lo = pos - p.window + 1 - k0;
  c.sink = p.n_sink - k0;
  return c;
}
// columns x .. x + 31 as bits.  Every tile goes through the same code, and one with a mask through a few selections more: code of its own
// for masked tiles, in short windows met once or twice per CTA, is fetched as often as it is run.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }
__device__ __forceinline__ uint32_t visible32(const Columns& c, int x) { return below(c.hi - x) & (~below(c.lo - x) | below(c.sink - x)); }

// ------------------------------------------------------------------ forward
// Two tiles of 128 queries per CTA: of two heads that share their keys (the tiles need the same ones, at the same time), or, where heads
// do not come in such pairs, one behind the other (the second starts one tile of keys later, and ends later).  Eight warps each: while one's scores are exponentiated, the other's products run.  Two threads own a
// row, 64 keys each (with one, the single warp that a tile then has on each of the SM's four parts waits for its own instructions: 2000
// cycles per tile, and 3400 per pair of tiles where heads of 128 need 2048 for their products).  They agree on the largest score through
// shared memory, read the scores twice from tensor memory rather than keep them, and rescale and write half of the features each.
// Tensor memory: scores of both tiles (128 columns each; the weights over them), sums of both (DP each).
// The running maximum is followed lazily: sums are rescaled only where it has grown by 2^8 since, which bf16 weights and
// fp32 sums carry without loss.
constexpr float kLazy = 8.f;

template <int DP, int SLOTS>
struct FwdSmem {
  static constexpr uint32_t tile = kT * DP * 2;
  static constexpr uint32_t bytes = (2 + SLOTS) * tile + 2048 + 512;
};

template <int DP, int SLOTS>
__global__ void __launch_bounds__(kFwdThreads, 1) attn_tensor_fwd_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ Maps maps) {
  constexpr uint32_t TILE = FwdSmem<DP, SLOTS>::tile;
  extern __shared__ __align__(1024) uint8_t base[];
  if (smem_u32(base) & 1023) {  // (the swizzle goes by the address)
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, (int)DEV_WAIT_TIMEOUT);
    return;
  }
  const uint32_t qs = smem_u32(base);
  float* const shared_row = reinterpret_cast<float*>(base + (2 + SLOTS) * TILE);  // [tile][half][row]
  uint64_t* const bars = reinterpret_cast<uint64_t*>(shared_row + 4 * kT);
  uint64_t *const q_full = bars, *const s_full = bars + 1, *const p_half = bars + 3, *const p_ready = bars + 5, *const o_full = bars + 7, *const go = bars + 9, *const cleared = bars + 10;
  const Ring<SLOTS> ring{bars + 11, bars + 11 + SLOTS, qs + 2 * TILE, TILE};
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 11 + 2 * SLOTS);
  volatile int* const stop = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  // The thread that loads sets the barriers up and sends for the first tiles before it meets the others: the loads are under way while
  // tensor memory is taken and everybody finds out what the item is.
  if (warp == 16) tmem_alloc(tmem_slot, 512);
  if (warp == 17 && elect_one()) {
    mbar_init(q_full, 1), mbar_init(go, 1), mbar_init(cleared, 1);
    for (int x = 0; x < 2; ++x) mbar_init(s_full + x, 1), mbar_init(p_half + x, 2 * kT), mbar_init(p_ready + x, 2 * kT), mbar_init(o_full + x, 1);
    for (int i = 0; i < SLOTS; ++i) mbar_init(ring.full + i, 1), mbar_init(ring.empty + i, 1);
    fence_mbar_init();
    *stop = 0;
  }
  wait_for_inputs();
  const bool by_head = p.G % 2 == 0;
  const Block at = by_head ? block_of(p.H / 2, (p.Nq + kT - 1) / kT) : block_of(p.H, (p.Nq + 2 * kT - 1) / (2 * kT));
  const int i0 = at.last_first * (by_head ? kT : 2 * kT), h0 = by_head ? 2 * at.head : at.head, b = at.b, hk = h0 / p.G;
  auto first_of = [&](int x) { return by_head ? i0 : i0 + x * kT; };  // tile x's first query, and its head
  auto head_of = [&](int x) { return by_head ? h0 + x : h0; };
  const RowGeom g = row_geom(p, b);
  const KeyTiles all = key_tiles<kT>(p, g, i0, first_of(1) + kT);
  const int n = all.count();
  // tiles with places that nobody sees (the last one may end in padding), whose values would meet weights of zero
  const SeenKeys seen = seen_keys(p, g);
  auto unseen = [&](int j) { return seen.lacks(all.tile(j) * kT, kT, p.Nk); };
  const int at_once = min(2 * n, SLOTS);
  auto load = [&](int i) {
    const auto to = ring.place(i);
    mbar_expect_tx(ring.arrived(to), TILE);
    load_tile<DP>(ring.at(to), i & 1 ? &maps.v : &maps.k, hk, all.tile(i >> 1) * kT, b, ring.arrived(to));
  };
  if (warp == 17) {
    __syncwarp();
    if (n > 0 && elect_one()) {
      const int queries = first_of(1) < p.Nq ? 2 : 1;
      mbar_expect_tx(q_full, queries * TILE);
      for (int x = 0; x < queries; ++x) load_tile<DP>(qs + x * TILE, &maps.q, head_of(x), first_of(x), b, q_full);
      for (int i = 0; i < at_once; ++i) load(i);
    }
    __syncwarp();
  }
  tmem_before();
  __syncthreads();
  tmem_after();
  const uint32_t tmem = *tmem_slot;
  const Waiter wait{stop, p.status};

  if (warp == 17) {
    if (elect_one()) {
      for (int i = at_once; i < 2 * n; ++i) {
        if (!ring.wait_empty(wait, ring.place(i))) {
          mbar_wait_bounded(q_full, 0, 1u << 16);
          settle(ring, i);
          break;
        }
        load(i);
      }
    }
    __syncwarp();
  } else if (warp == 18) {
    uint32_t clears = 0;
    for (int j = 0; j < n; ++j) {
      if (!unseen(j)) continue;
      if (!wait(go, clears++ & 1)) break;
      const int k0 = all.tile(j) * kT;
      clear_rows<DP>(ring.at(ring.place(2 * j + 1)), [&](int r) { return seen.has(k0 + r); }, cleared);
    }
  } else if (warp == 16) {
    if (n > 0 && elect_one()) {
      // what tile x needs of the list: entries below ns, and lo .. hi
      int ns[2], lo[2], hi[2], last[2];
      for (int x = 0; x < 2; ++x) {
        const KeyTiles kt = key_tiles<kT>(p, g, first_of(x), first_of(x) + kT);
        ns[x] = kt.ns;
        lo[x] = all.entry(kt.t0);
        hi[x] = kt.t1 >= kt.t0 ? all.entry(kt.t1) : -1;
        last[x] = max(ns[x] - 1, hi[x]);
      }
      uint32_t phase[2] = {0, 0}, clears = 0;
      bool begun[2] = {false, false};
      typename Ring<SLOTS>::Place k_at, v_at;
      v_at.next();
      auto needs = [&](int x, int j) { return j < ns[x] || (j >= lo[x] && j <= hi[x]); };
      auto scores = [&](int x) {
        product_scores<DP>(tmem + x * kT, qs + x * TILE, ring.at(k_at));
        mma_commit(s_full + x);
      };
      bool ok = wait.one(q_full, 0) && ring.wait_full(wait, k_at);
      if (ok) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (needs(x, 0)) scores(x);
        ring.release(k_at);
        k_at.next(), k_at.next();
      }
#pragma unroll 1
      for (int j = 0; ok && j < n; ++j) {
        ok = ring.wait_full(wait, v_at) && (!unseen(j) || have_cleared(wait, go, cleared, clears++ & 1)) && (j + 1 >= n || ring.wait_full(wait, k_at));
        if (!ok) break;
        const uint32_t vs = ring.at(v_at);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (needs(x, j)) {
            if (!(ok = wait.one(p_half + x, phase[x]))) break;
            tmem_after();
            product_sums<DP, 0>(tmem + 2 * kT + x * 128, tmem + x * kT, vs, begun[x]);
            if (!(ok = wait.one(p_ready + x, phase[x]))) break;
            tmem_after();
            product_sums<DP, 1>(tmem + 2 * kT + x * 128, tmem + x * kT, vs, true);
            phase[x] ^= 1;
            begun[x] = true;
            if (j == last[x]) mma_commit(o_full + x);
          }
          if (j + 1 < n && needs(x, j + 1)) scores(x);
        }
        if (!ok) break;
        ring.release(v_at);
        v_at.next(), v_at.next();
        if (j + 1 < n) {
          ring.release(k_at);
          k_at.next(), k_at.next();
        }
      }
    }
    __syncwarp();
  } else {
    const int x = warp / 8, half = warp / 4 % 2, r = threadIdx.x % kT, first = first_of(x), h = head_of(x), qi = first + r, pos = g.start + qi;
    const int end = min(g.ctx, g.start + p.Nq);
    const KeyTiles kt = key_tiles<kT>(p, g, first_of(x), first_of(x) + kT);
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    const uint32_t ts = tmem + x * kT + half * 64 + lanes, to = tmem + 2 * kT + x * 128 + lanes;
    const int p_lo = g.start + first, p_hi = p_lo + kT - 1;  // positions of the tile, padding included
    const int mine = kt.count(), pair_bar = 1 + x * 4 + warp % 4;  // the barrier of the two warps that share rows
    float *const my_row = shared_row + (2 * x + half) * kT + r, *const other_row = shared_row + (2 * x + 1 - half) * kT + r;
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    float ref = -INFINITY, l = 0.f;  // (ref in log2 units)
    bool ok = true;
    for (int j = 0; j < mine; ++j) {
      const int k0 = kt.tile(j) * kT + half * 64;
      const bool whole = k0 + 63 <= p_lo && k0 + 64 <= g.ctx && (k0 > p_hi - p.window || k0 + 64 <= p.n_sink);
      const Columns col = columns_of(p, pos, end, k0);
      if (!(ok = wait(s_full + x, j & 1))) break;
      tmem_after();
      float top;
      {
        float s[2][32];
        tmem_load32f(ts, s[0]);
        tmem_load32f(ts + 32, s[1]);
        tmem_loaded(s);
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t bits = visible32(col, 32 * c);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[c][e] = bits & (1u << e) ? s[c][e] : -INFINITY;
          }
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            mx[2 * c + u] = fmaxf(s[c][u], s[c][u + 2]);
#pragma unroll
            for (int e = u + 4; e < 32; e += 4) mx[2 * c + u] = fmaxf(fmaxf(mx[2 * c + u], s[c][e]), s[c][e + 2]);
          }
        top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
      }
      *my_row = top;
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      top = fmaxf(top, *other_row);  // (written again only when both have handed in this tile's weights)
      const bool grown = top > ref + kLazy;  // (also the first score of a row: ref is -inf)
      if (__any_sync(~0u, grown && ref != -INFINITY)) {  // the sums that the products so far have left: they are done, the scores came after them
        const float keep = grown ? ex2(ref - top) : 1.f;
        l *= keep;
#pragma unroll 1
        for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
          float o[32];
          tmem_load32f(to + c, o);
          tmem_loaded(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= keep;
          tmem_store32f(to + c, o);
        }
      }
      if (grown) ref = top;
      const float bias = ref == -INFINITY ? 0.f : ref;
      const float2 bias2 = make_float2(-bias, -bias);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      float s[2][16];
      tmem_load16f(ts, s[0]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {  // the weights of scores 16 c .. lie over scores 8 c .., which have been used
        float(&t)[16] = s[c % 2];
        tmem_loaded(t);
        if (c < 3) tmem_load16f(ts + 16 * (c + 1), s[(c + 1) % 2]);
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) exp2_pair(t[e], t[e + 1], scale2, bias2, e / 2);
        if (!whole) {
          const uint32_t bits = visible32(col, 16 * c);
#pragma unroll
          for (int e = 0; e < 16; ++e) t[e] = bits & (1u << e) ? t[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          sum[e / 2 % 2] = __fadd2_rn(sum[e / 2 % 2], make_float2(t[e], t[e + 1]));
          w[e / 2] = pack(t[e], t[e + 1]);
        }
        tmem_store8(ts + 8 * c, w);
        if (c == 1) {
          tmem_stored();
          tmem_before();
          mbar_arrive(p_half + x);
        }
      }
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      tmem_stored();
      tmem_before();
      mbar_arrive(p_ready + x);
    }
    if (mine > 0 && ok) ok = wait(o_full + x, 0);
    tmem_after();
    if (!ok) asm volatile("bar.arrive %0, 64;" ::"r"(pair_bar) : "memory");  // given up: the warp that shares the rows does not wait for this one
    if (ok) {
      *my_row = l;
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      l += *other_row;
      // (padding between rows that see a whole tile has had no mask)
      const bool some = mine > 0 && pos >= 0 && pos < end;  // (scores that are all minus infinity leave l = 0, and NaN)
      const float inv = some ? 1.f / l : 0.f;
      if (p.lse && half == 0 && qi < p.Nq) p.lse[((long long)b * p.H + h) * p.Nqp + qi] = some ? ref + log2f(l) : INFINITY;
      // through the place of the tile's queries, 4 KB of it to a warp (2 KB in heads of 64): the last of its products has read them (with no
      // products, they may still be arriving)
      const int row0 = first + warp % 4 * 32;
      if (n > 0 && first < p.Nq) ok = wait(q_full, 0);
      if (ok && row0 < p.Nq) {
        constexpr uint32_t MINE = TILE / 8;
        constexpr int OTHERS = MINE / 2048 - 1;
        const uint32_t place = qs + x * TILE + warp % 8 * MINE, second = place + OTHERS * 2048;
#pragma unroll 1
        for (int c = half * (DP / 2); c < (half + 1) * (DP / 2) && c < p.d; c += 32) {
          float o[32];
          if (mine > 0) {
            tmem_load32f(to + c, o);
            tmem_loaded(o);
          }
          if (!some) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          send_rows<OTHERS>(&maps.y, p.rest || c % 64 == 0 ? place : second, o, inv, c, h, row0, b);
          if (p.rest) {
            keep_rest(o, inv);
            send_rows<OTHERS>(&maps.rest, second, o, 1.f, c, h, row0, b);
          }
        }
        if (lane == 0) bulk_wait_read0();
        __syncwarp();
      }
    }
    tmem_before();
  }
  __syncthreads();
  if (warp == 16) {
    tmem_after();
    tmem_free(tmem, 512);
  }
}

// ------------------------------------------------------------------ backward of the queries
// One tile of 128 queries per CTA.  dP = dy v^T, dS = P (dP - delta), dq = dS k.  Two threads per row, 64 keys each.  Tensor
// memory: two buffers of scores (the next tile's are ready while this one's are worked on; dS over them), dP, dq.
template <int DP, int SLOTS>
struct BwdSmem {
  static constexpr uint32_t tile = kT * DP * 2;
  static constexpr uint32_t bytes = (2 + SLOTS) * tile + 2048 + 512;
};

template <int DP, int SLOTS>
__global__ void __launch_bounds__(kThreads, 1) attn_tensor_dq_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ Maps maps) {
  constexpr uint32_t TILE = BwdSmem<DP, SLOTS>::tile;
  extern __shared__ __align__(1024) uint8_t base[];
  if (smem_u32(base) & 1023) {  // (the swizzle goes by the address)
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, (int)DEV_WAIT_TIMEOUT);
    return;
  }
  const uint32_t qs = smem_u32(base), dys = qs + TILE;
  float* const deltas = reinterpret_cast<float*>(base + (2 + SLOTS) * TILE);  // [128]
  uint64_t* const bars = reinterpret_cast<uint64_t*>(deltas + 512);
  uint64_t *const q_full = bars, *const s_full = bars + 1, *const dp_full = bars + 3, *const ds_half = bars + 4, *const ds_ready = bars + 5, *const done = bars + 6,
           *const go = bars + 7, *const cleared = bars + 8, *const staged = bars + 9;
  const Ring<SLOTS> ring{bars + 10, bars + 10 + SLOTS, qs + 2 * TILE, TILE};
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 10 + 2 * SLOTS);
  volatile int* const stop = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (warp == 8) tmem_alloc(tmem_slot, 512);
  if (warp == 9 && elect_one()) {
    mbar_init(q_full, 1), mbar_init(s_full, 1), mbar_init(s_full + 1, 1), mbar_init(dp_full, 1), mbar_init(ds_half, 256), mbar_init(ds_ready, 256);
    mbar_init(done, 1), mbar_init(go, 1), mbar_init(cleared, 1), mbar_init(staged, 256);
    for (int i = 0; i < SLOTS; ++i) mbar_init(ring.full + i, 1), mbar_init(ring.empty + i, 1);
    fence_mbar_init();
    *stop = 0;
  }
  wait_for_inputs();
  const Block at = block_of(p.H, (p.Nq + kT - 1) / kT);
  const int i0 = at.last_first * kT, h = at.head, b = at.b, hk = h / p.G;
  const RowGeom g = row_geom(p, b);
  const KeyTiles kt = key_tiles<kT>(p, g, i0, i0 + kT);
  const int n = kt.count();

  // tiles with places that nobody sees: keys that would meet a dS of zero
  const SeenKeys seen = seen_keys(p, g);
  auto unseen = [&](int j) { return seen.lacks(kt.tile(j) * kT, kT, p.Nk); };
  // (as in the forward: the first tiles are sent for before the warps meet)
  const int at_once = min(2 * n + 2, SLOTS);
  auto load = [&](int i) {  // y and its rest, for delta, in the ring's first places; then keys and values
    const auto to = ring.place(i);
    mbar_expect_tx(ring.arrived(to), TILE);
    if (i < 2)
      load_tile<DP>(ring.at(to), i ? &maps.rest : &maps.y, h, i0, b, ring.arrived(to));
    else
      load_tile<DP>(ring.at(to), i & 1 ? &maps.v : &maps.k, hk, kt.tile((i >> 1) - 1) * kT, b, ring.arrived(to));
  };
  if (warp == 9) {
    __syncwarp();
    if (n > 0 && elect_one()) {
      mbar_expect_tx(q_full, 2 * TILE);
      load_tile<DP>(qs, &maps.q, h, i0, b, q_full);
      load_tile<DP>(dys, &maps.dy, h, i0, b, q_full);
      for (int i = 0; i < at_once; ++i) load(i);
    }
    __syncwarp();
  }
  tmem_before();
  __syncthreads();
  tmem_after();
  const uint32_t tmem = *tmem_slot, t_dp = tmem + 256, t_dq = tmem + 384;
  const Waiter wait{stop, p.status};

  if (warp == 9) {
    if (n > 0 && elect_one()) {
      for (int i = at_once; i < 2 * n + 2; ++i) {
        if (!ring.wait_empty(wait, ring.place(i))) {
          mbar_wait_bounded(q_full, 0, 1u << 16);
          settle(ring, i);
          break;
        }
        load(i);
      }
    }
    __syncwarp();
  } else if (warp == 10) {
    uint32_t clears = 0;
    for (int j = 0; j < n; ++j) {
      if (!unseen(j)) continue;
      if (!wait(go, clears++ & 1)) break;
      const int k0 = kt.tile(j) * kT;
      clear_rows<DP>(ring.at(ring.place(2 * j + 2)), [&](int r) { return seen.has(k0 + r); }, cleared);
    }
  } else if (warp == 8) {
    if (n > 0 && elect_one()) {
      typename Ring<SLOTS>::Place k_at, v_at, old_k;  // of the next scores, the next dP, the next dS
      k_at = old_k = ring.place(2), v_at = ring.place(3);
      uint32_t clears = 0;
      auto scores = [&](int j) {  // of tile j into buffer j % 2
        if (!(ring.wait_full(wait, k_at) && (!unseen(j) || have_cleared(wait, go, cleared, clears++ & 1)))) return false;
        product_scores<DP>(tmem + (j & 1) * kT, qs, ring.at(k_at));
        mma_commit(s_full + (j & 1));
        k_at.next(), k_at.next();
        return true;
      };
      auto grads = [&]() {
        if (!ring.wait_full(wait, v_at)) return false;
        product_scores<DP>(t_dp, dys, ring.at(v_at));
        mma_commit(dp_full);
        ring.release(v_at);
        v_at.next(), v_at.next();
        return true;
      };
      bool ok = wait.one(q_full, 0) && scores(0) && grads() && (n < 2 || scores(1));
#pragma unroll 1
      for (int j = 0; ok && j < n; ++j) {
        const uint32_t ds = tmem + (j & 1) * kT, ks = ring.at(old_k);
        if (!(ok = wait.one(ds_half, j & 1))) break;
        tmem_after();
        product_sums<DP, 0>(t_dq, ds, ks, j > 0);
        if (!(ok = wait.one(ds_ready, j & 1))) break;
        tmem_after();
        if (j + 1 < n && !(ok = grads())) break;
        product_sums<DP, 1>(t_dq, ds, ks, true);
        ring.release(old_k);
        old_k.next(), old_k.next();
        if (j + 2 < n) ok = scores(j + 2);
      }
      if (ok) mma_commit(done);
    }
    __syncwarp();
  } else {  // warps 0-7
    const int half = warp / 4, r = warp % 4 * 32 + lane, qi = i0 + r, pos = g.start + qi;
    const int end = min(g.ctx, g.start + p.Nq);
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    const int p_lo = g.start + i0, p_hi = p_lo + kT - 1;
    const bool live = pos >= 0 && pos < end;
    const long long head_row = ((long long)b * p.H + h) * p.Nqp + qi;
    const float lse = live ? p.lse[head_row] : INFINITY;
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    float delta = 0.f;
    if (n > 0) {
      // delta = sum(dy * y), of half of the row's features each.  All three are tiles that the TMA unit has fetched: read by the threads
      // themselves, y and its rest took 9000 cycles longer (the cache that is left next to this much shared memory has no room for them).
      ok = wait(q_full, 0) && wait(ring.full, 0) && wait(ring.full + 1, 0);
      const uint32_t ys = qs + 2 * TILE, rests = ys + TILE;
      float sum = 0.f;
      if (ok && live) {
#pragma unroll
        for (int e = 0; e < DP / 2; e += 8) {
          const int c = half * (DP / 2) + e;
          const uint32_t off = (c / 64) * kBlockBytes + r * 128 + ((c % 64 / 8 ^ (r & 7)) << 4);
          uint32_t u[4], t[4], w[4];
          lds128(ys + off, u), lds128(rests + off, t), lds128(dys + off, w);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            sum = fmaf(__uint_as_float(u[x] << 16) + __uint_as_float(t[x] << 16), __uint_as_float(w[x] << 16), sum);
            sum = fmaf(__uint_as_float(u[x] & 0xffff0000u) + __uint_as_float(t[x] & 0xffff0000u), __uint_as_float(w[x] & 0xffff0000u), sum);
          }
        }
      }
      deltas[half * kT + r] = sum;
      asm volatile("bar.sync 1, 256;" ::: "memory");  // (every warp comes here, whatever became of its waits)
      if (threadIdx.x == 0) mbar_arrive(ring.empty), mbar_arrive(ring.empty + 1);
      delta = deltas[r] + deltas[kT + r];
      if (half == 0 && qi < p.Nq) p.delta[head_row] = delta;
    }
    for (int j = 0; ok && j < n; ++j) {
      const int k0 = kt.tile(j) * kT + half * 64;
      const uint32_t ts = tmem + (j & 1) * kT + half * 64 + lanes;
      if (!(ok = wait(s_full + (j & 1), (j >> 1) & 1))) break;
      tmem_after();
      const bool whole = k0 + 63 <= p_lo && p_hi < end && k0 + 64 <= g.ctx && (k0 > p_hi - p.window || k0 + 64 <= p.n_sink);
      const Columns col = columns_of(p, pos, end, k0);
      const float2 bias2 = make_float2(-lse, -lse), delta2 = make_float2(-delta, -delta);
      float s[2][32];
      tmem_load32f(ts, s[0]);
      tmem_load32f(ts + 32, s[1]);
      tmem_loaded(s);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 32; e += 2) exp2_pair(s[c][e], s[c][e + 1], scale2, bias2, e / 2);
      if (!(ok = wait(dp_full, j & 1))) break;
      tmem_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float dp[32];
        uint32_t w[16];
        tmem_load32f(t_dp + half * 64 + 32 * c + lanes, dp);
        tmem_loaded(dp);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 t = __fmul2_rn(make_float2(s[c][e], s[c][e + 1]), __fadd2_rn(make_float2(dp[e], dp[e + 1]), delta2));
          dp[e] = t.x, dp[e + 1] = t.y;
        }
        if (!whole) {
          const uint32_t bits = visible32(col, 32 * c);
#pragma unroll
          for (int e = 0; e < 32; ++e) dp[e] = bits & (1u << e) ? dp[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) w[e / 2] = pack(dp[e], dp[e + 1]);
        tmem_store16(ts + 16 * c, w);
        tmem_stored();
        tmem_before();
        mbar_arrive(c ? ds_ready : ds_half);
      }
    }
    if (n > 0 && ok) ok = wait(done, 0);
    tmem_after();
    if (ok) {
      if (n > 0) ok = wait(q_full, 0);
#pragma unroll 1
      for (int c = half * (DP / 2); ok && c < (half + 1) * (DP / 2); c += 32) {
        float o[32];
        if (n > 0) {
          tmem_load32f(t_dq + c + lanes, o);
          tmem_loaded(o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        stage_row(qs, r, o, p.scale, c);  // (over the queries, which the last product has read)
      }
      fence_proxy_async();
      if (ok) mbar_arrive(staged);
      if (ok && warp == 0 && wait(staged, 0) && lane == 0) {
        send_tile<DP>(&maps.dq, qs, h, i0, b);
        bulk_wait_read0();
      }
      __syncwarp();
    }
    tmem_before();
  }
  __syncthreads();
  if (warp == 8) {
    tmem_after();
    tmem_free(tmem, 512);
  }
}

// ------------------------------------------------------------------ backward of the keys
// One tile of 128 keys per CTA, its group's heads and their query tiles one after the other.  Scores the other way round (keys are
// rows): P^T and dS^T are left operands as they come.  dv = P^T dy, dk = dS^T q.  Two threads per row, 64 queries each.  Tensor
// memory is full: scores (P over them), dP (dS over it), dv, dk; the next tile's scores wait for dv's product only, its dP for
// dk's.
template <int DP, int SLOTS>
__global__ void __launch_bounds__(kThreads, 1) attn_tensor_dkv_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ Maps maps) {
  constexpr uint32_t TILE = BwdSmem<DP, SLOTS>::tile;
  constexpr int STATS = 2;  // tiles whose lse and delta are held
  extern __shared__ __align__(1024) uint8_t base[];
  if (smem_u32(base) & 1023) {  // (the swizzle goes by the address)
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, (int)DEV_WAIT_TIMEOUT);
    return;
  }
  const uint32_t ks = smem_u32(base), vs = ks + TILE;
  float* const stats = reinterpret_cast<float*>(base + (2 + SLOTS) * TILE);  // [STATS][2][128]
  uint64_t* const bars = reinterpret_cast<uint64_t*>(stats + STATS * 2 * kT);
  uint64_t *const kv_full = bars, *const s_full = bars + 1, *const dp_full = bars + 2, *const p_half = bars + 3, *const p_ready = bars + 4, *const ds_half = bars + 5,
           *const ds_ready = bars + 6, *const done = bars + 7, *const go = bars + 8, *const cleared = bars + 9, *const st_full = bars + 10,
           *const st_empty = bars + 10 + STATS, *const staged = bars + 10 + 2 * STATS;
  const Ring<SLOTS> ring{bars + 11 + 2 * STATS, bars + 11 + 2 * STATS + SLOTS, ks + 2 * TILE, TILE};
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 11 + 2 * STATS + 2 * SLOTS);
  volatile int* const stop = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (warp == 8) tmem_alloc(tmem_slot, 512);
  if (warp == 9 && elect_one()) {
    mbar_init(kv_full, 1), mbar_init(s_full, 1), mbar_init(dp_full, 1), mbar_init(done, 1), mbar_init(go, 1), mbar_init(cleared, 1), mbar_init(staged, 256);
    mbar_init(p_half, 256), mbar_init(p_ready, 256), mbar_init(ds_half, 256), mbar_init(ds_ready, 256);
    for (int i = 0; i < STATS; ++i) mbar_init(st_full + i, 1), mbar_init(st_empty + i, 8);
    for (int i = 0; i < SLOTS; ++i) mbar_init(ring.full + i, 1), mbar_init(ring.empty + i, 1);
    fence_mbar_init();
    *stop = 0;
  }
  wait_for_inputs();
  const Block at = block_of(p.Hk, (p.Nk + kT - 1) / kT + p.sink_tiles * p.chunks);
  const int hk = at.head, b = at.b;
  const RowGeom g = row_geom(p, b);
  const KeyItem it = key_item<kT, kT>(p, g, at.first_last);
  const int k0 = it.tile * kT, n = it.end - it.begin;
  // an entry of the list of the item's heads and tiles of queries, and the next one (each role walks the list by itself)
  struct Entry {
    int head, tile, first, end;  // tile: first <= tile < end
    __device__ __forceinline__ int row() const { return tile * kT; }
    __device__ __forceinline__ void next() {
      if (++tile == end) tile = first, ++head;
    }
  };
  Entry entry{hk * p.G, it.first, it.first, it.first + it.tiles};
  if (it.begin > 0 && n > 0) entry.head += it.begin / it.tiles, entry.tile += it.begin % it.tiles;

  // tiles of queries that reach into padding: their rows there would meet weights of zero
  auto padded = [&](const Entry& e) {
    const int first = g.start + e.row();
    return first < 0 || (first + kT > g.ctx && g.start + p.Nq > g.ctx);
  };
  // (as in the forward: the first tiles are sent for before the warps meet)
  const int at_once = min(2 * n, 4);
  auto load = [&](int i, const Entry& e) {  // queries, their cotangents, and with these the stats, whose place is free before that
    const auto to = ring.place(i);
    mbar_expect_tx(ring.arrived(to), TILE);
    load_tile<DP>(ring.at(to), i & 1 ? &maps.dy : &maps.q, e.head, e.row(), b, ring.arrived(to));
    if (i & 1) {
      const int u = i >> 1;
      float* const st = stats + u % STATS * 2 * kT;
      const long long row = ((long long)b * p.H + e.head) * p.Nqp + e.row();
      mbar_expect_tx(st_full + u % STATS, 2 * kT * 4);
      bulk_g2s(st, p.lse + row, kT * 4, st_full + u % STATS);
      bulk_g2s(st + kT, p.delta + row, kT * 4, st_full + u % STATS);
    }
  };
  if (warp == 9) {
    __syncwarp();
    if (n > 0 && elect_one()) {
      mbar_expect_tx(kv_full, 2 * TILE);
      load_tile<DP>(ks, &maps.k, hk, k0, b, kv_full);
      load_tile<DP>(vs, &maps.v, hk, k0, b, kv_full);
      Entry e = entry;
      for (int i = 0; i < at_once; ++i) {
        load(i, e);
        if (i & 1) e.next();
      }
    }
    __syncwarp();
  }
  tmem_before();
  __syncthreads();
  tmem_after();
  const uint32_t tmem = *tmem_slot, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 384;
  const Waiter wait{stop, p.status};

  if (warp == 9) {
    if (n > 0 && elect_one()) {
      for (int i = 0; i < at_once; i += 2) entry.next();
      for (int i = at_once; i < 2 * n; ++i) {
        const int u = i >> 1;
        if (!ring.wait_empty(wait, ring.place(i)) || (i & 1 && !wait.one(st_empty + u % STATS, (u / STATS & 1) ^ 1))) {
          mbar_wait_bounded(kv_full, 0, 1u << 16);
          for (int e = u > STATS ? u - STATS : 0; e < u; ++e) mbar_wait_bounded(st_full + e % STATS, (e / STATS) & 1, 1u << 16);
          settle(ring, i);
          break;
        }
        load(i, entry);
        if (i & 1) entry.next();
      }
    }
    __syncwarp();
  } else if (warp == 10) {
    uint32_t clears = 0;
    for (int i = 0; i < 2 * n; ++i) {
      if (padded(entry)) {
        if (!wait(go, clears++ & 1)) break;
        const int first = g.start + entry.row();
        clear_rows<DP>(ring.at(ring.place(i)), [&](int r) { return first + r >= 0 && first + r < g.ctx; }, cleared);
      }
      if (i & 1) entry.next();
    }
  } else if (warp == 8) {
    if (n > 0 && elect_one()) {
      typename Ring<SLOTS>::Place q_at, dy_at, old_q, old_dy;  // of the next scores, the next dP; of the next dk, the next dv
      dy_at.next(), old_dy.next();
      uint32_t clears = 0;
      auto arrived = [&](const typename Ring<SLOTS>::Place& at) {
        if (!ring.wait_full(wait, at)) return false;
        return !padded(entry) || have_cleared(wait, go, cleared, clears++ & 1);  // (in the order of the loads)
      };
      auto scores = [&]() {
        if (!arrived(q_at)) return false;
        product_scores<DP>(tmem, ks, ring.at(q_at));
        mma_commit(s_full);
        q_at.next(), q_at.next();
        return true;
      };
      auto grads = [&]() {  // (moves on to the next entry)
        if (!arrived(dy_at)) return false;
        product_scores<DP>(t_dp, vs, ring.at(dy_at));
        mma_commit(dp_full);
        dy_at.next(), dy_at.next();
        entry.next();
        return true;
      };
      bool ok = wait.one(kv_full, 0) && scores() && grads();
#pragma unroll 1
      for (int i = 0; ok && i < n; ++i) {
        if (!(ok = wait.one(p_half, i & 1))) break;
        tmem_after();
        product_sums<DP, 0>(t_dv, tmem, ring.at(old_dy), i > 0);
        if (!(ok = wait.one(p_ready, i & 1))) break;
        tmem_after();
        product_sums<DP, 1>(t_dv, tmem, ring.at(old_dy), true);
        ring.release(old_dy);
        old_dy.next(), old_dy.next();
        if (i + 1 < n && !(ok = scores())) break;
        if (!(ok = wait.one(ds_half, i & 1))) break;
        tmem_after();
        product_sums<DP, 0>(t_dk, t_dp, ring.at(old_q), i > 0);
        if (!(ok = wait.one(ds_ready, i & 1))) break;
        tmem_after();
        product_sums<DP, 1>(t_dk, t_dp, ring.at(old_q), true);
        ring.release(old_q);
        old_q.next(), old_q.next();
        if (i + 1 < n) ok = grads();
      }
      if (ok) mma_commit(done);
    }
    __syncwarp();
  } else if (warp < 8) {
    const int half = warp / 4, r = warp % 4 * 32 + lane, key = k0 + r;
    const int end = min(g.ctx, g.start + p.Nq);
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16, ts = tmem + half * 64 + lanes, td = t_dp + half * 64 + lanes;
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int first = g.start + entry.row() + half * 64;  // position of column 0
      entry.next();
      const float *lse = stats + i % STATS * 2 * kT + half * 64, *delta = lse + kT;
      if (!(ok = wait(st_full + i % STATS, (i / STATS) & 1) && wait(s_full, i & 1))) break;
      tmem_after();
      float s[2][32];
      tmem_load32f(ts, s[0]);
      tmem_load32f(ts + 32, s[1]);
      tmem_loaded(s);
      // queries key .. last of the columns see the key
      const int lo = key - first, hi = min(end, key < p.n_sink ? end : key + p.window) - first;
      const bool whole = k0 + kT - 1 <= first && first + 64 <= end && (first + 63 < k0 + p.window || k0 + kT <= p.n_sink);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[16];
        const uint32_t bits = below(hi - 32 * c) & ~below(lo - 32 * c);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 ls = *reinterpret_cast<const float4*>(lse + 32 * c + e);
          exp2_pair(s[c][e], s[c][e + 1], scale2, make_float2(-ls.x, -ls.y), e / 2);
          exp2_pair(s[c][e + 2], s[c][e + 3], scale2, make_float2(-ls.z, -ls.w), e / 2 + 1);
        }
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 32; ++e) s[c][e] = bits & (1u << e) ? s[c][e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) w[e / 2] = pack(s[c][e], s[c][e + 1]);
        tmem_store16(ts + 16 * c, w);
        tmem_stored();
        tmem_before();
        mbar_arrive(c ? p_ready : p_half);
      }
      if (!(ok = wait(dp_full, i & 1))) break;
      tmem_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float dp[32];
        uint32_t w[16];
        tmem_load32f(td + 32 * c, dp);
        tmem_loaded(dp);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 de = *reinterpret_cast<const float4*>(delta + 32 * c + e);
          const float2 t = __fmul2_rn(make_float2(s[c][e], s[c][e + 1]), __fadd2_rn(make_float2(dp[e], dp[e + 1]), make_float2(-de.x, -de.y)));
          const float2 u = __fmul2_rn(make_float2(s[c][e + 2], s[c][e + 3]), __fadd2_rn(make_float2(dp[e + 2], dp[e + 3]), make_float2(-de.z, -de.w)));
          dp[e] = t.x, dp[e + 1] = t.y, dp[e + 2] = u.x, dp[e + 3] = u.y;
        }
        if (!whole) {
          const uint32_t bits = below(hi - 32 * c) & ~below(lo - 32 * c);
#pragma unroll
          for (int e = 0; e < 32; ++e) dp[e] = bits & (1u << e) ? dp[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) w[e / 2] = pack(dp[e], dp[e + 1]);
        tmem_store16(td + 16 * c, w);
        tmem_stored();
        tmem_before();
        mbar_arrive(c ? ds_ready : ds_half);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(st_empty + i % STATS);
    }
    if (n > 0 && ok) ok = wait(done, 0);
    tmem_after();
    const bool sinks = p.chunks > 0 && it.tile < p.sink_tiles, partial = sinks && key < p.n_sink;
    if (ok) {
      float* const part = sinks ? part_of(p, b, hk, it.tile, it.chunk < 0 ? p.chunks : it.chunk) : nullptr;
      const long long row = ((long long)b * p.Nk + key) * p.Hk * p.d + (long long)hk * p.d;
      if (n > 0) ok = wait(kv_full, 0);
#pragma unroll 1
      for (int which = 0; ok && which < 2; ++which)
#pragma unroll 1
        for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
          float o[32];
          if (n > 0) {
            tmem_load32f((which ? t_dv : t_dk) + c + lanes, o);
            tmem_loaded(o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          const float f = which ? 1.f : p.scale;
          if (partial) {
            float* const at_part = part + ((long long)which * p.sink_rows + r) * p.d + c;
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (c + e < p.d) *reinterpret_cast<float4*>(at_part + e) = make_float4(o[e] * f, o[e + 1] * f, o[e + 2] * f, o[e + 3] * f);
          } else if (sinks) {  // (a tile whose rows go two ways)
            if (it.chunk < 0 && key < p.Nk) store_row(static_cast<__nv_bfloat16*>(which ? p.dv : p.dk) + row, o, f, c, p.d);
          } else {
            stage_row(which ? vs : ks, r, o, f, c);  // (over the keys and values, which the last products have read)
          }
        }
      if (!sinks) {
        fence_proxy_async();
        if (ok) mbar_arrive(staged);
        if (ok && warp == 0 && wait(staged, 0) && lane == 0) {
          send_tile<DP>(&maps.dk, ks, hk, k0, b);
          send_tile<DP>(&maps.dv, vs, hk, k0, b);
          bulk_wait_read0();
        }
        __syncwarp();
      }
    }
    tmem_before();
  }
  __syncthreads();
  if (warp == 8) {
    tmem_after();
    tmem_free(tmem, 512);
  }
}

// ------------------------------------------------------------------ host
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* at = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &at, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
      at = nullptr;
    return reinterpret_cast<EncodeFn>(at);
  }();
  return fn;
}
// Tensor maps are encoded by the driver, which wants a context current in the calling thread; a thread of the autograd engine that has
// made no runtime call yet has none.
cudaError_t bind_context() {
  static const auto current = [] {
    void* at = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &at, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
      at = nullptr;
    return reinterpret_cast<CUresult (*)(CUcontext*)>(at);
  }();
  CUcontext ctx = nullptr;
  if (current && current(&ctx) == CUDA_SUCCESS && ctx) return cudaSuccess;
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  return e == cudaSuccess ? cudaSetDevice(dev) : e;
}
// [B, N, heads, d] with boxes of 128 positions x 64 features, or (of_warp) 32 x 32
cudaError_t encode(CUtensorMap& m, const void* at, int d, int heads, int N, int B, long long sn, long long sb, bool of_warp = false) {
  const EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)N, (cuuint64_t)B};
  const cuuint64_t strides[3] = {(cuuint64_t)d * 2, (cuuint64_t)sn * 2, (cuuint64_t)sb * 2};
  const cuuint32_t box[4] = {of_warp ? 32u : 64u, 1, of_warp ? 32u : (cuuint32_t)kT, 1}, step[4] = {1, 1, 1, 1};
  return fn(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(at), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            of_warp ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? cudaSuccess
             : cudaErrorInvalidValue;
}

template <int DP, int SLOTS>
cudaError_t run_fwd(const AttnParams& p, const Maps& maps, cudaStream_t st) {
  static SmemGrant grant;
  constexpr uint32_t smem = FwdSmem<DP, SLOTS>::bytes;
  const cudaError_t e = grant_smem(grant, attn_tensor_fwd_kernel<DP, SLOTS>, smem);
  if (e != cudaSuccess) return e;
  const unsigned items = p.G % 2 == 0 ? (unsigned)((p.Nq + kT - 1) / kT) * (p.H / 2) * p.B : (unsigned)((p.Nq + 2 * kT - 1) / (2 * kT)) * p.H * p.B;
  return launch_behind(attn_tensor_fwd_kernel<DP, SLOTS>, dim3(items), kFwdThreads, smem, st, p, maps);
}
template <int DP, int SLOTS>
cudaError_t run_bwd(const AttnParams& p, const Maps& maps, cudaStream_t st) {
  static SmemGrant g1, g2;
  constexpr uint32_t smem = BwdSmem<DP, SLOTS>::bytes;
  cudaError_t e = grant_smem(g1, attn_tensor_dq_kernel<DP, SLOTS>, smem);
  if (e == cudaSuccess) e = grant_smem(g2, attn_tensor_dkv_kernel<DP, SLOTS>, smem);
  if (e != cudaSuccess) return e;
  e = launch_behind(attn_tensor_dq_kernel<DP, SLOTS>, dim3((unsigned)((p.Nq + kT - 1) / kT * p.H * p.B)), kThreads, smem, st, p, maps);
  if (e != cudaSuccess) return e;
  const int items = (p.Nk + kT - 1) / kT + p.sink_tiles * p.chunks;
  return launch_behind(attn_tensor_dkv_kernel<DP, SLOTS>, dim3((unsigned)(items * p.Hk * p.B)), kThreads, smem, st, p, maps);
}
cudaError_t encode_all(Maps& m, const AttnParams& p, bool bwd) {
  cudaError_t e = bind_context();
  if (e == cudaSuccess) e = encode(m.q, p.q, p.d, p.H, p.Nq, p.B, p.sq_n, p.sq_b);
  if (e == cudaSuccess) e = encode(m.k, p.k, p.d, p.Hk, p.Nk, p.B, p.sk_n, p.sk_b);
  if (e == cudaSuccess) e = encode(m.v, p.v, p.d, p.Hk, p.Nk, p.B, p.sv_n, p.sv_b);
  const long long En = (long long)p.H * p.d, Ek = (long long)p.Hk * p.d;  // results are contiguous
  if (!bwd) {
    if (e == cudaSuccess) e = encode(m.y, p.y, p.d, p.H, p.Nq, p.B, En, En * p.Nq, true);
    if (e == cudaSuccess && p.rest) e = encode(m.rest, p.rest, p.d, p.H, p.Nq, p.B, En, En * p.Nq, true);
    return e;
  }
  if (e == cudaSuccess) e = encode(m.dy, p.dy, p.d, p.H, p.Nq, p.B, p.sdy_n, p.sdy_b);
  if (e == cudaSuccess) e = encode(m.y, p.y_in, p.d, p.H, p.Nq, p.B, En, En * p.Nq);
  if (e == cudaSuccess) e = encode(m.rest, p.rest, p.d, p.H, p.Nq, p.B, En, En * p.Nq);
  if (e == cudaSuccess) e = encode(m.dq, p.dq, p.d, p.H, p.Nq, p.B, En, En * p.Nq);
  if (e == cudaSuccess) e = encode(m.dk, p.dk, p.d, p.Hk, p.Nk, p.B, Ek, Ek * p.Nk);
  if (e == cudaSuccess) e = encode(m.dv, p.dv, p.d, p.Hk, p.Nk, p.B, Ek, Ek * p.Nk);
  return e;
}

}  // namespace

// bf16 rows that a tensor map describes: 16-byte aligned, strides multiples of 16 bytes, not zero and not negative.
bool attn_tensor_covers(const AttnParams& p, int dtype) {
  if (dtype != DT_BF16 || !p.vec || p.d > 128 || p.Nk < 1) return false;
  const long long s[8] = {p.sq_b, p.sq_n, p.sk_b, p.sk_n, p.sv_b, p.sv_n, p.sdy_b, p.sdy_n};
  for (const long long x : s)
    if (x < 8 || x >= (1ll << 38)) return false;
  const void* const out[6] = {p.y, p.y_in, p.dq, p.dk, p.dv, p.lse};  // (rest lies a multiple of 512 bytes behind lse)
  for (const void* o : out)
    if (reinterpret_cast<uintptr_t>(o) & 15u) return false;
  return true;
}

cudaError_t launch_attn_tensor_fwd(const AttnParams& p, cudaStream_t st) {
  Maps m;
  const cudaError_t e = encode_all(m, p, false);
  if (e != cudaSuccess) return e;
  return p.d <= 64 ? run_fwd<64, 8>(p, m, st) : run_fwd<128, 5>(p, m, st);
}
cudaError_t launch_attn_tensor_bwd(const AttnParams& p, cudaStream_t st) {
  Maps m;
  cudaError_t e = encode_all(m, p, true);
  if (e == cudaSuccess) e = p.d <= 64 ? run_bwd<64, 8>(p, m, st) : run_bwd<128, 5>(p, m, st);
  if (e != cudaSuccess || p.chunks == 0) return e;
  return launch_attn_sink_sum(p, DT_BF16, kT, st);
}

}  // namespace ncn
