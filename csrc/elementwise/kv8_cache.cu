// Writing keys and values into the 8-bit paged cache and reading them back (layout and number format: common/kv8.cuh).
//
// All kernels are bound by memory, small calls by their launch.  A half-warp holds one row: lane l has elements 8 l .. 8 l + 7 of every 128, so that a
// head of 128 is one 16-byte load a lane, its largest magnitude four shuffles, its codes one 8-byte store.  The two halves of a
// warp take a token's key and value of the same head, because a NaN in either marks both.  Write, 2179 tokens x 8 heads of 128 in fp16 (13.5 MB):
// 6.0 us, two waves of one load and one store; reading 16384 tokens x 8 heads back (102 MB): 20.7 us, 0.75 of a plain copy's rate.
#include <math.h>

#include <algorithm>

#include "../api.h"
#include "../common/kv8.cuh"
#include "../common/launch.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 8;

// a / b of non-negative numbers; a division of 64 bits is some hundred instructions, and few numbers here need it.
__device__ __forceinline__ int64_t quotient(int64_t a, int b) { return a >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b); }

// elements 8 l .. 8 l + 7 of every 128 of a row of D; zeros behind its end
template <typename T, int NI, bool kVec>
__device__ __forceinline__ void load_row(float (&v)[NI][8], const T* src, int D, int l) {
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int at = i * 128 + l * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    if (at >= D) continue;          // D is a multiple of 16
    if constexpr (kVec) {
      constexpr int N = Vec16<T>::N;
#pragma unroll
      for (int p = 0; p < 8; p += N) {
        const Vec16<T> a = ld_vec(src + at + p);
#pragma unroll
        for (int j = 0; j < N; ++j) v[i][p + j] = to_f(a.v[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = to_f(src[at + j]);
    }
  }
}

// Lower half-warp: the key row, upper one: the value row of the same token and head.
template <int NI>
__device__ __forceinline__ void put_row(const float (&v)[NI][8], const Kv8Cache& c, int64_t slot, int h, int half, int l) {
  float amax = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      amax = fmaxf(amax, fabsf(v[i][j]));
      nan |= is_nan_bits(v[i][j]);
    }
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  nan = __any_sync(0xffffffffu, nan);
  if (slot < 0 || slot >= c.num_blocks * c.block_size) return;      // padding: the whole warp
  const float s = kv8_scale(amax), inv = nan ? 0.f : pow2_inv(s);
  const int64_t blk = quotient(slot, c.block_size);
  const int off = (int)(slot - blk * c.block_size);
  uint8_t* page = c.page(blk, half, h);
  uint8_t* dst = c.codes(page, off);
#pragma unroll
  for (int i = 0; i < NI; ++i)
    if (i * 128 + l * 8 < c.D)
      *reinterpret_cast<uint2*>(dst + i * 128 + l * 8) = nan ? make_uint2(0, 0) : kv8_pack8(v[i], inv);
  if (l == 0) *c.scale(page, off) = nan ? __uint_as_float(0x7fffffffu) : s;
}

// k, v [T, Hkv, D] with strided tokens; a warp = (token, head).
template <typename T, int NI, bool kVec>
__global__ void __launch_bounds__(kWarps * 32) kv8_put_kernel(const T* __restrict__ k, const T* __restrict__ v, Kv8Cache c,
                                                              const int64_t* __restrict__ slots, int64_t rows, int64_t k_stride,
                                                              int64_t v_stride) {
  griddep_launch();
  griddep_wait();
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
  const int64_t t = quotient(row, c.Hkv);
  const int h = (int)(row - t * c.Hkv);
  float x[NI][8];
  load_row<T, NI, kVec>(x, (half ? v + t * v_stride : k + t * k_stride) + (int64_t)h * c.D, c.D, l);
  put_row<NI>(x, c, slots[t], h, half, l);
}

// The common case of the kernel below: heads of 128, rotated whole in halves, 16 bits, 16-byte aligned.  Eight lanes have a head, lane l of
// them columns 8 l .. 8 l + 7 and the same behind 64, so that a column meets its partner in its own thread.  With w the norm's weight and 1 / n
// the norm, a column is (x w_x cos - y w_y sin) / n: the products of weights and angles are the token's, not the head's.  A warp takes four
// heads a step, with copies of the next steps in flight; a token has one warp, or more, up to one a step, where there are too few tokens to
// fill the GPU's three CTAs of eight warps an SM.  8192 tokens of 32 + 2 x 4 heads, 164 MB, 25 us of memory: 36 us.  48 us with two heads a
// step and their angles and weights multiplied head by head (twice the instructions); 47 with the next step's loads in registers and two
// warps a token, 38 with four steps in flight in shared memory, 40 with six; 36 with one warp.
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 un2(uint64_t r) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(r));
  return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
constexpr int kRing = 4;
template <typename T>
__device__ __forceinline__ void unpack8(uint4 a, uint64_t (&v)[4]) {
  const T* x = reinterpret_cast<const T*>(&a);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = pk2(to_f(x[2 * j]), to_f(x[2 * j + 1]));
}
template <typename T> __device__ __forceinline__ uint32_t round2(uint64_t v);
template <> __device__ __forceinline__ uint32_t round2<__nv_bfloat16>(uint64_t v) {
  const float2 f = un2(v);
  const __nv_bfloat162 r = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <> __device__ __forceinline__ uint32_t round2<__half>(uint64_t v) {
  const float2 f = un2(v);
  const __half2 r = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T, bool kNorm>
__global__ void __launch_bounds__(kWarps * 32, 3) kv8_qkv128_kernel(
    T* __restrict__ q_out, const T* __restrict__ qkv, const int64_t* __restrict__ positions, const float* __restrict__ cos_sin,
    const T* __restrict__ q_w, const T* __restrict__ k_w, float eps, int Hq, float gemma, Kv8Cache c,
    const int64_t* __restrict__ slots, int64_t max_pos, int64_t qkv_stride, int64_t tokens, int share) {
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31, part = lane >> 3, l = lane & 7;
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5), t = w / share;
  const int q_units = (Hq + 3) / 4, units = q_units + (c.Hkv + 1) / 2;
  int u = (int)(w - t * share);
  if (t >= tokens || u >= units) return;
  const T* row = qkv + t * qkv_stride + l * 8;
  // A unit is four query heads, or the keys and values of two.
  const bool value = part & 1;
  const auto head_of = [&](int u) { return u < q_units ? 4 * u + part : 2 * (u - q_units) + part / 2; };
  // Loads of kRing units are in flight a warp; a lane copies to shared memory what it reads there itself.
  __shared__ uint4 ring[kWarps][kRing][2][32];
  uint4(*const mine)[2][32] = ring[threadIdx.x >> 5];
  const auto fetch = [&](int u, int at) {
    if (u < units) {
      const int h = head_of(u);
      const T* src = row + (int64_t)(u < q_units ? min(h, Hq - 1) : Hq + min(h, c.Hkv - 1) + (value ? c.Hkv : 0)) * 128;
      copy16(&mine[at][0][lane], src);
      copy16(&mine[at][1][lane], src + 64);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kRing; ++i) fetch(u + i * share, i);
  int64_t pos = positions[t];
  const int64_t slot = slots[t];
  pos = pos < 0 ? 0 : (pos >= max_pos ? max_pos - 1 : pos);
  const float* angles = cos_sin + pos * 128 + l * 8;
  uint64_t xc[4], xs[4], yc[4], ys[4];   // weight x cosine and sine of either half, -sine in ys
  const auto turns = [&](const T* weight) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 cs = reinterpret_cast<const float4*>(angles)[j], sn = reinterpret_cast<const float4*>(angles + 64)[j];
      xc[2 * j] = yc[2 * j] = pk2(cs.x, cs.y), xc[2 * j + 1] = yc[2 * j + 1] = pk2(cs.z, cs.w);
      xs[2 * j] = pk2(sn.x, sn.y), xs[2 * j + 1] = pk2(sn.z, sn.w);
      ys[2 * j] = pk2(-sn.x, -sn.y), ys[2 * j + 1] = pk2(-sn.z, -sn.w);
    }
    if constexpr (kNorm) {
      uint64_t wx[4], wy[4];
      unpack8<T>(*reinterpret_cast<const uint4*>(weight + l * 8), wx);
      unpack8<T>(*reinterpret_cast<const uint4*>(weight + l * 8 + 64), wy);
      const uint64_t ones = pk2(1.f, 1.f), g = pk2(gemma, gemma);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        wx[j] = fma2(wx[j], ones, g);
        wy[j] = fma2(wy[j], ones, g);
        xc[j] = mul2(xc[j], wx[j]);
        xs[j] = mul2(xs[j], wx[j]);
        yc[j] = mul2(yc[j], wy[j]);
        ys[j] = mul2(ys[j], wy[j]);
      }
    }
  };
  bool keys = u >= q_units;
  turns(keys ? k_w : q_w);
  int at = 0;
  for (; u < units; u += share) {
    const bool is_q = u < q_units;
    const int h = head_of(u);
    if (kNorm && !is_q && !keys) {
      keys = true;
      turns(k_w);
    }
    uint64_t x[4], y[4];                 // columns 8 l .. and 64 + 8 l ..
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
    unpack8<T>(mine[at][0][lane], x);
    unpack8<T>(mine[at][1][lane], y);
    uint64_t inv2 = 0;
    if constexpr (kNorm) {
      uint64_t sq = mul2(x[0], x[0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) sq = fma2(x[j], x[j], sq);
#pragma unroll
      for (int j = 0; j < 4; ++j) sq = fma2(y[j], y[j], sq);
      const float2 s2 = un2(sq);
      float s = s2.x + s2.y;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      const float inv = rsqrtf(s / 128 + eps);
      inv2 = pk2(inv, inv);
    }
    if (is_q || !value) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint64_t a = fma2(x[j], xc[j], mul2(y[j], ys[j])), b = fma2(y[j], yc[j], mul2(x[j], xs[j]));
        if constexpr (kNorm) a = mul2(a, inv2), b = mul2(b, inv2);
        x[j] = a;
        y[j] = b;
      }
    }
    fetch(u + kRing * share, at);
    at = at + 1 == kRing ? 0 : at + 1;
    if (is_q) {
      if (h >= Hq) continue;
      T* dst = q_out + (t * Hq + h) * (int64_t)128 + l * 8;
      *reinterpret_cast<uint4*>(dst) = make_uint4(round2<T>(x[0]), round2<T>(x[1]), round2<T>(x[2]), round2<T>(x[3]));
      *reinterpret_cast<uint4*>(dst + 64) = make_uint4(round2<T>(y[0]), round2<T>(y[1]), round2<T>(y[2]), round2<T>(y[3]));
      continue;
    }
    float f[2][8], amax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = un2(x[j]), b = un2(y[j]);
      f[0][2 * j] = a.x, f[0][2 * j + 1] = a.y, f[1][2 * j] = b.x, f[1][2 * j + 1] = b.y;
    }
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      amax = fmaxf(amax, fabsf(f[j >> 3][j & 7]));
      nan |= is_nan_bits(f[j >> 3][j & 7]);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    nan = (__ballot_sync(0xffffffffu, nan) >> (lane & 16) & 0xffffu) != 0;   // in the head's key or its value
    if (slot < 0 || slot >= c.num_blocks * c.block_size || h >= c.Hkv) continue;
    const int64_t blk = quotient(slot, c.block_size);
    const int off = (int)(slot - blk * c.block_size);
    const float s = kv8_scale(amax), inv = pow2_inv(s);
    uint8_t* page = c.page(blk, value, h);
    uint8_t* dst = c.codes(page, off) + l * 8;
    *reinterpret_cast<uint2*>(dst) = nan ? make_uint2(0, 0) : kv8_pack8(f[0], inv);
    *reinterpret_cast<uint2*>(dst + 64) = nan ? make_uint2(0, 0) : kv8_pack8(f[1], inv);
    if (l == 0) *c.scale(page, off) = nan ? __uint_as_float(0x7fffffffu) : s;
  }
}

// A fused qkv row: split, optional RMSNorm of query and key heads, rotation, queries out in T, keys and values into the cache.
// A warp takes two query heads, or the key and the value of one head; all in fp32 between the load and the one rounding at the
// end (no rounding to T between norm and rotation, nor in front of the codes).  Columns meet their partners in shared memory, one by one, and
// cosines are read head by head: this is what bounds it.  8192 tokens with norms (25 us of memory): 64 / 8 heads of 64 204 us, 16 / 2 heads
// of 256 165 us.
template <typename T, int NI, bool kVec>
__global__ void __launch_bounds__(kWarps * 32) kv8_qkv_kernel(
    T* __restrict__ q_out, const T* __restrict__ qkv, const int64_t* __restrict__ positions, const float* __restrict__ cos_sin,
    const T* __restrict__ q_w, const T* __restrict__ k_w, float eps, int Hq, int rot, int neox, float gemma, Kv8Cache c,
    const int64_t* __restrict__ slots, int64_t max_pos, int64_t qkv_stride) {
  extern __shared__ float sm_rows[];
  griddep_launch();
  griddep_wait();
  const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
  const int64_t t = blockIdx.x;
  const int D = c.D, q_units = (Hq + 1) / 2, units = q_units + c.Hkv;
  int64_t pos = positions[t];
  pos = pos < 0 ? 0 : (pos >= max_pos ? max_pos - 1 : pos);
  const float* cs = cos_sin + pos * rot;
  const int64_t slot = slots[t];
  for (int u = blockIdx.y * kWarps + wid; u < units; u += gridDim.y * kWarps) {
    const bool is_q = u < q_units;
    const int head = is_q ? 2 * u + half : Hq + (u - q_units) + half * c.Hkv;
    const bool in = !is_q || head < Hq, turn = is_q || half == 0;
    float v[NI][8];
    load_row<T, NI, kVec>(v, qkv + t * qkv_stride + (int64_t)(in ? head : 0) * D, D, l);
    const T* w = is_q ? q_w : k_w;
    if (w != nullptr) {
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sq += v[i][j] * v[i][j];
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      if (turn) {
        const float inv = rsqrtf(sq / D + eps);
        float wv[NI][8];
        load_row<T, NI, kVec>(wv, w, D, l);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * inv * (wv[i][j] + gemma);
        }
      }
    }
    {
      float* buf = sm_rows + (wid * 2 + half) * D;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (i * 128 + l * 8 < D) buf[i * 128 + l * 8 + j] = v[i][j];
      }
      __syncwarp();
      const int hr = rot >> 1;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at = i * 128 + l * 8 + j;
          if (turn && at < 2 * hr) {
            const bool first = neox ? at < hr : (at & 1) == 0;
            const int f = neox ? (at < hr ? at : at - hr) : at >> 1;
            const float other = buf[neox ? (at < hr ? at + hr : at - hr) : at ^ 1];
            v[i][j] = first ? v[i][j] * cs[f] - other * cs[hr + f] : v[i][j] * cs[f] + other * cs[hr + f];
          }
        }
      }
      __syncwarp();       // read before the next unit's rows
    }
    if (is_q) {
      if (!in) continue;
      T* dst = q_out + (t * Hq + head) * (int64_t)D;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int at = i * 128 + l * 8;
        if (at >= D) continue;
        constexpr int N = Vec16<T>::N;
#pragma unroll
        for (int p = 0; p < 8; p += N) {
          Vec16<T> a;
#pragma unroll
          for (int j = 0; j < N; ++j) a.v[j] = from_f<T>(v[i][p + j]);
          st_vec(dst + at + p, a);
        }
      }
    } else {
      put_row<NI>(v, c, slot, u - q_units, half, l);
    }
  }
}

// k, v [M, Hkv, D] (contiguous) = rows `slots` of the cache; a slot outside it gives zeros.  A thread takes 16 elements of a row, the
// grid's y says whether of the key or of the value.  `k8`: the 8-bit cache, otherwise one in T [block][2][kv_head][slot][D].
template <typename T, bool k8>
__global__ void __launch_bounds__(256) kv_gather_kernel(T* __restrict__ k, T* __restrict__ v, Kv8Cache c,
                                                        const int64_t* __restrict__ slots, int64_t chunks) {
  griddep_launch();
  griddep_wait();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= chunks) return;
  const int per = c.D / 16, which = blockIdx.y;
  const int64_t row = quotient(i, per), m = quotient(row, c.Hkv);
  const int at = (int)(i - row * per) * 16, h = (int)(row - m * c.Hkv);
  const int64_t slot = slots[m];
  const bool in = slot >= 0 && slot < c.num_blocks * c.block_size;
  const int64_t blk = in ? quotient(slot, c.block_size) : 0;
  const int off = in ? (int)(slot - blk * c.block_size) : 0;
  T* dst = (which ? v : k) + row * c.D + at;
  alignas(16) T o[16];
  if (!in) {
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = from_f<T>(0.f);
  } else if constexpr (k8) {
    uint8_t* page = c.page(blk, which, h);
    const uint4 w = *reinterpret_cast<const uint4*>(c.codes(page, off) + at);
    const float s = *c.scale(page, off);
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = e4m3x2_to_float2((uint16_t)(x[j / 2] >> (16 * (j & 1))));
      o[2 * j] = from_f<T>(f.x * s);
      o[2 * j + 1] = from_f<T>(f.y * s);
    }
  } else {
    const T* src = reinterpret_cast<const T*>(c.base) + (((blk * 2 + which) * c.Hkv + h) * c.block_size + off) * (int64_t)c.D + at;
#pragma unroll
    for (int j = 0; j < 16; j += Vec16<T>::N) st_vec(o + j, ld_vec(src + j));
  }
#pragma unroll
  for (int j = 0; j < 16; j += Vec16<T>::N) st_vec(dst + j, ld_vec(o + j));
}

Kv8Cache cache_of(void* base, int64_t num_blocks, int Hkv, int block_size, int D) {
  return Kv8Cache{static_cast<uint8_t*>(base), num_blocks, Hkv, block_size, D};
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_kv8_put(const void* k, const void* v, void* cache, const int64_t* slots, int64_t T_, int Hkv, int D,
                            int block_size, int64_t num_blocks, int64_t k_stride, int64_t v_stride, int dtype, cudaStream_t st) {
  if (T_ == 0 || num_blocks == 0) return 0;
  if (D % 16 || D < 16 || D > 512 || Hkv < 1 || block_size % 4 || block_size < 4) return 2;
  const int64_t rows = T_ * Hkv, ctas = (rows + kWarps - 1) / kWarps;
  if (ctas > 0x7fffffff) return 2;
  const Kv8Cache c = cache_of(cache, num_blocks, Hkv, block_size, D);
  const int esize = dtype == kF32 ? 4 : 2;
  const bool vec = aligned16(k) && aligned16(v) && k_stride * esize % 16 == 0 && v_stride * esize % 16 == 0;
#define B200_KV8_PUT(NI, VEC)                                                                                                  \
  B200_DISPATCH_DTYPE(dtype, return (int)launch_pdl(kv8_put_kernel<T, NI, VEC>, dim3((unsigned)ctas), dim3(kWarps * 32), 0, st, \
                                                    (const T*)k, (const T*)v, c, slots, rows, k_stride, v_stride))
#define B200_KV8_PUT_NI(NI) if (vec) { B200_KV8_PUT(NI, true); } else { B200_KV8_PUT(NI, false); }
  if (D <= 128) { B200_KV8_PUT_NI(1) }
  else if (D <= 256) { B200_KV8_PUT_NI(2) }
  else { B200_KV8_PUT_NI(4) }
#undef B200_KV8_PUT_NI
#undef B200_KV8_PUT
  return 2;
}

extern "C" int b200_kv8_qkv(void* q_out, const void* qkv, const int64_t* positions, const float* cos_sin, const void* q_w,
                            const void* k_w, float eps, int64_t T_, int Hq, int Hkv, int D, int rot_dim, int neox, int gemma,
                            void* cache, const int64_t* slots, int block_size, int64_t num_blocks, int64_t max_pos,
                            int64_t qkv_stride, int dtype, int num_sms, cudaStream_t st) {
  if (T_ == 0) return 0;
  if (num_sms < 1 || D % 16 || D < 16 || D > 512 || Hkv < 1 || Hq < 1 || block_size % 4 || block_size < 4 || rot_dim > D || rot_dim % 2 ||
      max_pos < 1 || T_ > 0x7fffffff)
    return 2;
  const Kv8Cache c = cache_of(cache, num_blocks, Hkv, block_size, D);
  const int units = (Hq + 1) / 2 + Hkv, esize = dtype == kF32 ? 4 : 2;
  const bool vec = aligned16(qkv) && qkv_stride * esize % 16 == 0 && aligned16(q_w) && aligned16(k_w);
  const bool fast = vec && D == 128 && rot_dim == 128 && neox && dtype != kF32 && aligned16(cos_sin) && aligned16(q_out) &&
                    (q_w == nullptr) == (k_w == nullptr);
  // Few tokens: a warp per unit, so that a decode step is one turn deep; otherwise a CTA per token, which reads its angles once.  us with
  // a warp per unit and with a CTA per token, 64 / 8 heads of 64: 16 tokens 3.7 and 8.5, 256: 10.4 and 11.1, 320: 12.4 and 11.7, 1024: 33.6 and
  // 27.5; 16 / 2 heads of 256, 64 columns rotated: 16 tokens 4.2 and 6.0, 384: 10.4 and 11.1, 512: 13.0 and 12.8.
  const dim3 grid((unsigned)T_, T_ <= 384 ? (unsigned)((units + kWarps - 1) / kWarps) : 1u);
  if (fast) {
    const int steps = (Hq + 3) / 4 + (Hkv + 1) / 2, fill = num_sms * 3 * kWarps;
    const int share = (int)std::max<int64_t>(1, std::min<int64_t>(steps, (fill + T_ - 1) / T_));
    if (T_ * share > ((int64_t)1 << 33)) return 2;
#define B200_KV8_QKV128(TT, NORM)                                                                                              \
  return (int)launch_pdl(kv8_qkv128_kernel<TT, NORM>, dim3((unsigned)((T_ * share + kWarps - 1) / kWarps)), dim3(kWarps * 32), 0, st, \
                         (TT*)q_out, (const TT*)qkv, positions, cos_sin, (const TT*)q_w, (const TT*)k_w, eps, Hq, gemma ? 1.f : 0.f,   \
                         c, slots, max_pos, qkv_stride, T_, share)
    if (dtype == kBF16) {
      if (q_w != nullptr) B200_KV8_QKV128(__nv_bfloat16, true);
      B200_KV8_QKV128(__nv_bfloat16, false);
    }
    if (q_w != nullptr) B200_KV8_QKV128(__half, true);
    B200_KV8_QKV128(__half, false);
#undef B200_KV8_QKV128
  }
  const size_t smem = (size_t)kWarps * 2 * D * sizeof(float);
#define B200_KV8_QKV(NI, VEC)                                                                                                  \
  B200_DISPATCH_DTYPE(dtype, return (int)launch_pdl(kv8_qkv_kernel<T, NI, VEC>, grid, dim3(kWarps * 32), smem, st,             \
                                                    (T*)q_out, (const T*)qkv, positions, cos_sin, (const T*)q_w, (const T*)k_w, \
                                                    eps, Hq, rot_dim, neox, gemma ? 1.f : 0.f, c, slots, max_pos, qkv_stride))
#define B200_KV8_QKV_NI(NI) if (vec) { B200_KV8_QKV(NI, true); } else { B200_KV8_QKV(NI, false); }
  if (D <= 128) { B200_KV8_QKV_NI(1) }
  else if (D <= 256) { B200_KV8_QKV_NI(2) }
  else { B200_KV8_QKV_NI(4) }
#undef B200_KV8_QKV_NI
#undef B200_KV8_QKV
  return 2;
}

extern "C" int b200_kv_gather(void* k, void* v, const void* cache, const int64_t* slots, int64_t M, int Hkv, int D, int block_size,
                              int64_t num_blocks, int eight, int dtype, cudaStream_t st) {
  if (M == 0) return 0;
  if (D % 16 || D < 16 || Hkv < 1 || block_size < 1 || (eight && block_size % 4)) return 2;
  const int64_t chunks = M * Hkv * (D / 16), ctas = (chunks + 255) / 256;
  if (ctas > 0x7fffffff) return 2;
  const Kv8Cache c = cache_of(const_cast<void*>(cache), num_blocks, Hkv, block_size, D);
  B200_DISPATCH_DTYPE(dtype, {
    if (eight) return (int)launch_pdl(kv_gather_kernel<T, true>, dim3((unsigned)ctas, 2), dim3(256), 0, st, (T*)k, (T*)v, c, slots, chunks);
    return (int)launch_pdl(kv_gather_kernel<T, false>, dim3((unsigned)ctas, 2), dim3(256), 0, st, (T*)k, (T*)v, c, slots, chunks);
  });
  return 2;
}
