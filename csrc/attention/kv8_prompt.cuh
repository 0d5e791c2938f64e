// Pieces that the prompt kernels of the 8-bit cache share: how a call is cut into work items, cluster launch control, TMEM access,
// packed arithmetic, the second kernel that joins the splits of long contexts.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "../common/kv8.cuh"
#include "../common/launch.cuh"
#include "../common/ptx.cuh"
#include "../gemm/gemm_common.cuh"

namespace b200 {
namespace kv8prompt {

constexpr int kTile = 128, kPage = 64;
constexpr int kTmemCols = 512;
constexpr float kMaxSlack = 8.f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3e38f;         // log-sum-exp of a split whose scores are all -inf; one without keys has -inf

struct Params {
  void* out;                // [T, Hq, D]
  float* ws_o;              // [splits][T][Hq][D]
  float* ws_lse;            // [splits][T][Hq], log2
  const uint8_t* cache;
  const int* block_tables;
  const int* seq_lens;
  const int* qsl;
  const float* sinks;
  int* status;
  int64_t num_blocks, bt_stride, T;
  int B, Hq, Hkv, g, block_size, max_blocks, window;
  int head0, heads;         // key / value heads that this launch works on
  int toks;                 // tokens of a tile
  int single;               // one stream a CTA
  int row_blocks, splits;
  int max_keys;             // no key is looked for from here on (a multiple of 128)
  int span;                 // nor so many behind the request's first tile
  int take;                 // CTAs may be pending: whoever is done takes their items
  float scale_log2;
};

__device__ __forceinline__ void tmem_ld_x32_p(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32_p(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16_p(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]; issued by ONE thread.  A: lane = row, two 16-bit elements of K per column.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// two fp32 values in one 64-bit register: a fused multiply-add or an add of both is one instruction
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unf2(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 2^x on the special-function unit (-inf -> 0)
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}


// One work item: what the two streams of a CTA share and their own rows.
struct Item {
  int req, qs, q_len, ctx, seq_len, key0, head, split;     // key0: first key of the first tile
  int origin;                                              // first_key of the request
  int tok0[2], toks[2], n[2];                              // per stream: first token within the request, tokens, key tiles
  int n_max;
};
// The first key that a request's queries read, rounded down to tiles of 128: a window hides what is in front of it.
__device__ __forceinline__ int first_key(int ctx, int window, int max_keys) {
  return window > 0 ? min(max(0, ctx - window + 1), max_keys - 1) / kTile * kTile : 0;
}
// Items are ordered by descending row block, so by descending number of key tiles for prompts of one length.
template <int kKeys>       // keys of a tile
__device__ __forceinline__ void get_item(const Params& p, int idx, Item& it) {
  const int heads = p.heads * p.splits, per = p.B * heads, rb = p.row_blocks - 1 - idx / per, rem = idx % per;
  it.req = rem / heads;
  it.head = p.head0 + rem % heads / p.splits;
  it.split = rem % p.splits;
  it.qs = p.qsl[it.req];
  it.q_len = p.qsl[it.req + 1] - it.qs;
  it.seq_len = p.seq_lens[it.req];
  it.ctx = it.seq_len - it.q_len;
  it.origin = first_key(it.ctx, p.window, p.max_keys);
  const int step = p.single ? p.toks : 2 * p.toks;
  int all[2];
  int kv_begin = 0;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    it.tok0[s] = rb * step + s * p.toks;
    it.toks[s] = (s == 1 && p.single) ? 0 : max(0, min(p.toks, it.q_len - it.tok0[s]));
    // a window hides everything in front of the first token's first visible key (whole tiles of it)
    if (s == 0 && p.window > 0)
      kv_begin = it.origin + min(min(max(0, it.ctx + it.tok0[0] - p.window + 1), p.max_keys - 1) - it.origin, p.span - 1) / kKeys * kKeys;
    // keys visible to the tile end with the position of its last token; rows that see nothing have a tile all the same
    const int kv_end = it.origin + min(min(min(it.seq_len, p.max_keys), it.ctx + it.tok0[s] + it.toks[s]) - it.origin, p.span);
    all[s] = it.toks[s] > 0 ? max(1, (kv_end - kv_begin + kKeys - 1) / kKeys) : 0;
  }
  const int each = (max(all[0], all[1]) + p.splits - 1) / p.splits, first = it.split * each;
#pragma unroll
  for (int s = 0; s < 2; ++s) it.n[s] = max(0, min(all[s] - first, each));
  it.key0 = kv_begin + first * kKeys;
  it.n_max = max(it.n[0], it.n[1]);
}

// Asks for the index of a CTA of this grid that has not been started, which then never will be: 16 bytes at `dst`, complete_tx on `bar`.
__device__ __forceinline__ void ask_for_cta(uint32_t dst, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(dst),
               "r"(smem_u32(bar)) : "memory");
}
// The answer: a CTA's index, or -1 when all have been started or taken (then no further question may be asked).
__device__ __forceinline__ int taken_cta(uint32_t src) {
  uint32_t ok, x = 0;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .b64 lo, hi;\n\t.reg .pred p;\n\t"
      "ld.shared.v2.b64 {lo, hi}, [%2];\n\t"
      "mov.b128 r, {lo, hi};\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=r"(ok), "=r"(x) : "r"(src) : "memory");
  return ok ? (int)x : -1;
}

// Joins the splits of a row: out = sum_s w_s O_s / (sum_s w_s [+ sink]), w_s = 2^(lse_s - max).  A warp per (token, head).
template <typename T, int D>
__global__ void __launch_bounds__(256)
kv8_join_kernel(T* __restrict__ out, const float* __restrict__ ws_o, const float* __restrict__ ws_lse, const float* __restrict__ sinks,
                int64_t rows, int Hq, int head0, int heads, int splits, const int* __restrict__ qsl, int B) {
  griddep_launch();
  griddep_wait();
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows || row / Hq < qsl[0] || row / Hq >= qsl[B] || row % Hq < head0 || row % Hq >= head0 + heads) return;
  constexpr int N = D / 32;
  const float mine = lane < splits ? ws_lse[lane * rows + row] : -INFINITY;      // at most 32 splits
  const float M = warp_max(mine), Ms = M == -INFINITY ? 0.f : M;
  float w = mine == -INFINITY ? 0.f : exp2f(mine - Ms);
  float den = warp_sum(w);
  if (sinks != nullptr) den += exp2f(sinks[row % Hq] * kLog2e - Ms);
  w = den == 0.f ? 0.f : w / den;
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float ws = __shfl_sync(0xffffffffu, w, s);
    if (ws == 0.f) continue;             // an empty split's row may hold anything
    const float* src = ws_o + (s * rows + row) * D + lane * N;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 v = *reinterpret_cast<const float2*>(src + j);
      acc[j] += ws * v.x;
      acc[j + 1] += ws * v.y;
    }
  }
  uint32_t* dst = reinterpret_cast<uint32_t*>(out + row * D + lane * N);
#pragma unroll
  for (int j = 0; j < N; j += 2) dst[j / 2] = pack2<T>(acc[j], acc[j + 1]);
}

}  // namespace kv8prompt
}  // namespace b200
