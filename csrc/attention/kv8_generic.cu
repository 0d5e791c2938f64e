// Attention over the 8-bit paged cache (common/kv8.cuh) for any head size, block size and query type, on the CUDA cores and in fp32
// throughout: what the tensor-core kernels do not take (kv8_decode.cu, kv8_prompt.cu), and models in fp32.  Causal, optional
// sliding window, sinks.  One CTA = one (query token, query head).  Each of its four warps walks 32-key tiles of the visible
// range: scores with a lane per key, an online softmax per warp, then P.V with four dims a lane; the warps' states meet at the end.
// 16 requests of 4096 tokens, 32 / 8 heads of 128: 344 us (the tensor-core kernel 33); bound by fp32 instructions, every head reads its keys anew.
// A key whose block is outside the pool is not there.  A row that sees no key gives zeros; a NaN among the keys it sees gives NaN.
#include <math.h>

#include "../api.h"
#include "../common/kv8.cuh"
#include "../common/launch.cuh"

namespace b200 {
namespace {

constexpr int kGenWarps = 4;

template <typename T, int ND>  // ND: groups of four dims a lane, D <= 128 ND
__global__ void __launch_bounds__(kGenWarps * 32)
kv8_generic_kernel(T* __restrict__ out, const T* __restrict__ q, Kv8Cache c, const int* __restrict__ block_tables,
                   const int* __restrict__ seq_lens, const int* __restrict__ qsl, const float* __restrict__ sinks, int B, int Hq,
                   int max_blocks, int64_t bt_stride, int window, float scale, int64_t q_stride) {
  extern __shared__ float sm_gen[];
  const int D = c.D;
  float* sq = sm_gen;                       // [D]
  float* so = sq + D;                       // [kGenWarps][D]
  float* sml = so + kGenWarps * D;          // [kGenWarps][3]
  griddep_launch();
  griddep_wait();
  const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (t < qsl[0] || t >= qsl[B]) return;
  int lo = 0, hi = B;                       // the last request that starts at or before t: empty ones in front of it do not own it
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (qsl[mid] <= t) lo = mid; else hi = mid;
  }
  const int req = lo, kvh = h / (Hq / c.Hkv);
  const int pos = seq_lens[req] - (qsl[req + 1] - t);
  const int first = window > 0 ? max(0, pos - window + 1) : 0;
  for (int i = tid; i < D; i += kGenWarps * 32) sq[i] = to_f(q[(int64_t)t * q_stride + (int64_t)h * D + i]) * scale;
  __syncthreads();
  const int* bt = block_tables + (int64_t)req * bt_stride;
  const int64_t to_v = (int64_t)c.Hkv * c.page_bytes();
  float m = -INFINITY, l = 0.f, acc[ND][4];
  bool sees = false;                        // any key
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  for (int k0 = first + warp * 32; k0 <= pos; k0 += kGenWarps * 32) {
    const int key = k0 + lane;
    int64_t row = -1;                       // byte offset of the key's codes
    float s = -INFINITY, vs = 0.f;
    if (key <= pos) {
      const int bi = key / c.block_size, off = key % c.block_size;
      const int64_t blk = bi < max_blocks ? bt[bi] : -1;
      if (blk >= 0 && blk < c.num_blocks) {
        uint8_t* page = c.page(blk, 0, kvh);
        const uint8_t* kr = c.codes(page, off);
        row = kr - c.base;
        float a0 = 0.f, a1 = 0.f;
        for (int d = 0; d < D; d += 16) {
          const uint4 w = *reinterpret_cast<const uint4*>(kr + d);
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 f = e4m3x2_to_float2((uint16_t)(x[j / 2] >> (16 * (j & 1))));
            a0 += sq[d + 2 * j] * f.x;
            a1 += sq[d + 2 * j + 1] * f.y;
          }
        }
        s = (a0 + a1) * *c.scale(page, off);
        vs = *c.scale(page + to_v, off);
      }
    }
    sees |= __any_sync(0xffffffffu, row >= 0);
    if (__any_sync(0xffffffffu, is_nan_bits(s))) l = NAN;
    const float mn = fmaxf(m, warp_max(s));
    if (mn == -INFINITY) continue;
    const float corr = expf(m - mn);
    const float pr = row >= 0 ? expf(s - mn) : 0.f;
    m = mn;
    l = l * corr + warp_sum(pr);
#pragma unroll
    for (int i = 0; i < ND; ++i) { acc[i][0] *= corr; acc[i][1] *= corr; acc[i][2] *= corr; acc[i][3] *= corr; }
    const float pv = row >= 0 ? pr * vs : 0.f;
    for (int j = 0; j < 32; ++j) {
      const float pj = __shfl_sync(0xffffffffu, pv, j);
      const int64_t rj = __shfl_sync(0xffffffffu, row, j);
      if (rj < 0) continue;
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int d = (i * 32 + lane) * 4;
        if (d >= D) continue;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(c.base + rj + to_v + d);
        const float2 a = e4m3x2_to_float2((uint16_t)w), b = e4m3x2_to_float2((uint16_t)(w >> 16));
        acc[i][0] += pj * a.x;
        acc[i][1] += pj * a.y;
        acc[i][2] += pj * b.x;
        acc[i][3] += pj * b.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int d = (i * 32 + lane) * 4;
    if (d < D) {
#pragma unroll
      for (int j = 0; j < 4; ++j) so[warp * D + d + j] = acc[i][j];
    }
  }
  if (lane == 0) { sml[warp * 3] = m; sml[warp * 3 + 1] = l; sml[warp * 3 + 2] = sees; }
  __syncthreads();
  float M = sinks != nullptr ? sinks[h] : -INFINITY;
#pragma unroll
  for (int w = 0; w < kGenWarps; ++w) { M = fmaxf(M, sml[w * 3]); sees |= sml[w * 3 + 2] != 0.f; }
  const float Ms = M == -INFINITY ? 0.f : M;
  float den = sinks != nullptr ? expf(sinks[h] - Ms) : 0.f, wg[kGenWarps];
#pragma unroll
  for (int w = 0; w < kGenWarps; ++w) { wg[w] = expf(sml[w * 3] - Ms); den += is_nan_bits(sml[w * 3 + 1]) ? NAN : sml[w * 3 + 1] * wg[w]; }
  const float inv = den == 0.f ? (sees ? NAN : 0.f) : 1.f / den;      // NaN stays NaN; keys with scores of -inf alone give one
  for (int d = tid; d < D; d += kGenWarps * 32) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < kGenWarps; ++w) a += so[w * D + d] * wg[w];
    out[((int64_t)t * Hq + h) * D + d] = from_f<T>(a * inv);
  }
}

}  // namespace
}  // namespace b200

extern "C" int b200_kv8_attention_generic(void* out, const void* q, const void* cache, const int* block_tables,
                                          const int* seq_lens, const int* qsl, const float* sinks, int64_t T_, int B, int Hq,
                                          int Hkv, int D, int block_size, int max_blocks, int64_t bt_stride, int64_t num_blocks,
                                          int window, float scale, int64_t q_stride, int dtype, cudaStream_t st) {
  using namespace b200;
  if (B == 0 || T_ == 0) return 0;
  if (Hq % Hkv || Hq > 65535 || window < 0 || D % 16 || D < 16 || D > 512 || block_size % 4 || T_ > 0x7fffffff) return 2;
  const size_t smem = (size_t)(D + kGenWarps * (D + 3)) * sizeof(float);
  const Kv8Cache c{static_cast<uint8_t*>(const_cast<void*>(cache)), num_blocks, Hkv, block_size, D};
  const dim3 grid((unsigned)T_, Hq);
#define B200_KV8_GEN(ND)                                                                                                         \
  B200_DISPATCH_DTYPE(dtype, return (int)launch_pdl(kv8_generic_kernel<T, ND>, grid, dim3(kGenWarps * 32), smem, st, (T*)out,    \
                                                    (const T*)q, c, block_tables, seq_lens, qsl, sinks, B, Hq, max_blocks,       \
                                                    bt_stride, window, scale, q_stride))
  if (D <= 128) { B200_KV8_GEN(1); }
  if (D <= 256) { B200_KV8_GEN(2); }
  B200_KV8_GEN(4);
#undef B200_KV8_GEN
  return 2;
}
