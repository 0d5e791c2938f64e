// Prompt and chunk attention over the 8-bit paged cache (common/kv8.cuh) on tcgen05 + TMEM, fed by TMA from the pages: heads of 64 and
// 128, any number of query tokens.
//
// Per 128-key tile and 128-row query tile
//     S[128 rows, 128 keys]  = Q . K_tile^T                 e4m3: codes as cached, queries in pieces
//     O[128 rows, D dims]   += P[128 rows, 128 keys] . V    fp16, P in TMEM over the columns of S
// Queries are sums of three 8-bit pieces as in kv8_decode.cu, so K is an operand as it comes from memory; its scales are multiplied onto the
// scores.  Three pieces at twice the rate of a 16-bit product cost one and a half times what that would.  V and P go the other
// way: pieces of P would have to be made by the softmax warps, which have no time left, so four warps widen V to fp16 between the TMA's
// buffer and the tensor core's.  Every stored value is an exact fp16 number (common/kv8.cuh): its scale is gone then, and P rounds to 11 bits.
// What bounds it: per tile the tensor core needs 1280 cycles, the special-function units 1024 (128 x 128 exponentials at 16 a cycle), shared
// memory more than either (operands, TMA, widening, scales).
// Measured, us, beside the kernel that widens first (kv8_wide.cu), 32 / 8 heads of 128 behind 16000 tokens: one tile 44 and 58, two 57 and 65, four 100
// and 92, ten 328 and 235; 12 requests without context, one tile 12 and 14.  So it takes up to two tiles.  (Two pieces, which hold fewer digits:
// 43, 53, 94, 305.)
//
// A row is (token, head of a group): a tile holds 128 / g tokens of all g heads of one key / value head, so that a few new tokens fill it,
// and K and V are read and converted once for the group.  A persistent CTA works on two tiles ("streams") of consecutive tokens that read
// the same K / V tiles; the tensor core works on one while the other is in its softmax.  A stream's products are issued in the order
// P.V(i), S(i + 1), so the arrival of S(i + 1) also says that O holds P.V(i).  With few tiles behind a long context the keys of an item are
// split over CTAs, whose normalised partial results a second kernel joins.
// 512 threads: warp 0 TMA producer (a lane per 16 keys), warp 1 MMA issuer, warps 4-7 / 8-11 queries, softmax and epilogue of stream 0 / 1
// (thread = row), warps 12-15 widening.  The grid has a CTA per item, in descending order of row blocks; a CTA that is done takes the next
// pending one's item (cluster launch control).  Every wait is bounded; on time-out the status word is set and the CTA unwinds.
#include "../api.h"
#include "kv8_prompt.cuh"

namespace b200 {
namespace kv8prompt {

constexpr int kThreads = 4 * 128;
// Registers a thread of the first and the last warpgroup keeps and one of the softmax warpgroups gets: the launch brings 512 x 128 =
// 65536, and the split takes 128 x (64 + 192 + 192 + 64) = 65536.
constexpr int kRegsFew = 64, kRegsSoft = 192;
constexpr int kVStages = 4;                              // V pages as operands
constexpr int kRing = 4;                                 // K scales and valid masks: more than the K stages

template <typename T> struct Pieces;
template <> struct Pieces<__nv_bfloat16> {
  static constexpr float kTop = 32768.f;
  __host__ __device__ static constexpr bool e5(int) { return true; }
};
template <> struct Pieces<__half> {
  static constexpr float kTop = 16384.f;
  __host__ __device__ static constexpr bool e5(int piece) { return piece < 2; }
};

template <typename T, int D> struct Cfg {
  static constexpr int P = 3;
  static constexpr int kPiece = kTile * D;             // 128 rows of D e4m3 bytes
  static constexpr int kQ = P * kPiece;                // a stream's queries; in 16 bits (2 * kPiece) until they are taken apart
  static constexpr int kKStages = D == 128 ? 2 : 3, kK = kTile * D;
  static constexpr int kB = D / 64;                    // 64-dim blocks of a 16-bit row
  static constexpr int kV = kB * kPage * 128;
  static constexpr int kRaw = D == 128 ? 3 : 4, kCodes = kPage * D;      // V pages as codes
  static constexpr size_t kSmem =
      1024 + 2 * kQ + kKStages * kK + kVStages * kV + kRaw * (kCodes + kPage * 4) + kRing * kTile * 4 + 512;
  static_assert(kSmem <= 227 * 1024 && kKStages < kRing);
};

// four codes -> four fp16 values times a power of two, exact
__device__ __forceinline__ void widen4(uint32_t w, __half2 f, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = e4m3x2_to_f16x2((uint16_t)w), b = e4m3x2_to_f16x2((uint16_t)(w >> 16));
  const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&a), f), y = __hmul2(*reinterpret_cast<const __half2*>(&b), f);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}

// K-major operand whose rows are D e4m3 bytes, swizzled over 128 or 64 bytes; and where 16-byte chunk c of row r lies
template <int D>
__device__ __forceinline__ uint64_t desc_rows(uint32_t addr) {
  if constexpr (D == 128) return umma_desc_k_sw128(addr);
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(512 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)4 << 61;
}
template <int D>
__device__ __forceinline__ int chunk_at(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ (r >> 1 & 3)) << 4);
}

// What a page of V is, for the widening warps: bits 0-3 which 16 keys were read, 4-10 keys in front of the request's end, 12 the end of
// all work.
constexpr uint32_t kMetaEnd = 1u << 12;

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
kv8_prompt_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKV, const __grid_constant__ Params p) {
  using C = Cfg<T, D>;
  constexpr int kB = C::kB, kKStages = C::kKStages, kRaw = C::kRaw;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                  // [2 streams][pieces][128 rows][D B]
  uint8_t* sK = sQ + 2 * C::kQ;                        // [kKStages][128 keys][D B]
  uint8_t* sV = sK + kKStages * C::kK;                 // [kVStages][kB dim blocks][64 keys][128 B]
  uint8_t* sRaw = sV + kVStages * C::kV;               // [kRaw][64 keys][D B]
  float* sScaleV = reinterpret_cast<float*>(sRaw + kRaw * C::kCodes);   // [kRaw][64]
  float* sScaleK = sScaleV + kRaw * kPage;             // [kRing][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sScaleK + kRing * kTile);
  uint64_t* q_full = bars;              // one phase per item
  uint64_t* q_empty = bars + 1;         // the item's last S has been computed
  uint64_t* q_ready = bars + 2;         // [2 streams] in pieces: four warps, a phase per item with work for the stream
  uint64_t* k_full = bars + 4;          // [3]
  uint64_t* k_empty = bars + 7;         // [3] both streams' S of the tile have been computed
  uint64_t* ks_full = bars + 10;        // [kRing] scales and valid mask
  uint64_t* v_full = bars + 14;         // [4] four warps
  uint64_t* v_empty = bars + 18;        // [4]
  uint64_t* raw_full = bars + 22;       // [4]
  uint64_t* raw_empty = bars + 26;      // [4] four warps
  uint64_t* s_full = bars + 30;         // [2 streams]
  uint64_t* p_ready = bars + 32;        // [2 streams][2 halves] one arrival per softmax warp
  uint64_t* o_final = bars + 36;        // [2 streams] one phase per item with work for the stream
  // answers about the next item: question k uses slot k & 1
  uint64_t* next_full = bars + 38;      // [2]
  uint64_t* next_empty = bars + 40;     // [2] read by the MMA thread and the eight softmax warps
  const uint32_t next_at = smem_u32(bars + 42);   // [2] x 16 bytes
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 46);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* sMeta = tmem_slot + 2;      // [4]
  uint32_t* sValid = sMeta + 4;         // [kRing] which 16 keys of a tile are there

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Abort ab{p.status, abort_flag};
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int b = 0; b < kKStages; ++b) { mbar_init(&k_full[b], 1); mbar_init(&k_empty[b], 1); }
    for (int b = 0; b < kRing; ++b) mbar_init(&ks_full[b], 1);
    for (int b = 0; b < kVStages; ++b) { mbar_init(&v_full[b], 4); mbar_init(&v_empty[b], 1); }
    for (int b = 0; b < kRaw; ++b) { mbar_init(&raw_full[b], 1); mbar_init(&raw_empty[b], 4); }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_ready[s], 4);
      mbar_init(&s_full[s], 1);
      mbar_init(&o_final[s], 1);
      for (int h = 0; h < 2; ++h) mbar_init(&p_ready[s * 2 + h], 4);
      mbar_init(&next_full[s], 1);
      mbar_init(&next_empty[s], 9);
    }
    mbar_fence_init();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmKV);
    griddep_launch();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();   // q, the lengths and this step's cache rows come from the preceding kernels
  Item it;
  // MMA thread, softmax warps: answer k.  -1: there is no further item, or a wait gave up (then `ok` is false as well).
  auto next_item = [&](int k, bool whole_warp, bool& ok) {
    if (!p.take) return -1;
    ok = wait_or_abort(&next_full[k & 1], (k >> 1) & 1, ab, 929);
    if (whole_warp) ok = !__any_sync(0xffffffffu, !ok);
    if (!ok) return -1;
    const int idx = taken_cta(next_at + 16 * (k & 1));
    fence_proxy_async_smem();           // read before the next answer is written here
    if (whole_warp) __syncwarp();
    if (!whole_warp || lane == 0) mbar_arrive(&next_empty[k & 1]);
    return idx;
  };

  if (warp < 4 || warp >= 12) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer: lane u = keys 16 u .. of a tile
    const int R = min(kPage, p.block_size & -p.block_size), units = R / 16;      // keys of a box; the host's map agrees
    const int64_t page_bytes = (int64_t)p.block_size * (D + 4);
    int kc = 0, rc = 0, qc = 0, asked = 0;      // K tiles, V pages and items issued, questions asked so far
    bool ok = true;
    auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) { return __all_sync(0xffffffffu, wait_or_abort(bar, parity, ab, code)) != 0; };
    // asked when the item's last loads are due: late enough that a CTA does not hold an item it cannot start, early enough that the
    // answer is there before the last tiles have been worked on
    auto ask = [&]() {
      const int b = asked & 1;
      if (asked >= 2 && !wait_all(&next_empty[b], ((asked >> 1) - 1) & 1, 930)) return false;
      if (lane == 0) {
        mbar_expect_tx(&next_full[b], 16);
        ask_for_cta(next_at + 16 * b, &next_full[b]);
      }
      ++asked;
      return true;
    };
    for (int idx = blockIdx.x; ok && idx >= 0;) {
      get_item<kTile>(p, idx, it);
      const int n_max = it.n_max;
      if (n_max > 0) {
        if (qc > 0 && !wait_all(q_empty, (qc - 1) & 1, 920)) { ok = false; break; }
        if (lane == 0) {
          mbar_expect_tx(q_full, p.toks * p.g * 2 * D * ((it.n[0] > 0) + (it.n[1] > 0)));
#pragma unroll
          for (int s = 0; s < 2; ++s)
            if (it.n[s] > 0) {
#pragma unroll
              for (int h = 0; h < kB; ++h)
                tma_load_3d(sQ + s * C::kQ + h * (kTile * 128), &tmQ, q_full, h * 64, it.head * p.g, it.qs + it.tok0[s]);
            }
        }
        ++qc;
        const int* bt = p.block_tables + (int64_t)it.req * p.bt_stride;
        const int key_end = min(it.seq_len, it.key0 + n_max * kTile);
        auto lookup = [&](int j) -> int {      // block of this lane's 16 keys in tile j, -1: nothing to read
          const int key = it.key0 + j * kTile + lane * 16;
          if (lane >= 8 || j >= n_max || key >= key_end) return -1;
          const int bi = key / p.block_size;
          const int blk = bi < p.max_blocks ? bt[bi] : -1;
          return blk >= 0 && blk < p.num_blocks ? blk : -1;
        };
        // lanes at the start of a box issue it
        auto copy = [&](int key, int blk, int which, uint8_t* codes, float* scales, uint64_t* full_codes, uint64_t* full_scales) {
          const int in = key % p.block_size;
          const int64_t page = ((int64_t)blk * 2 + which) * p.Hkv + it.head;
          tma_load_3d(codes, &tmKV, full_codes, 0, in, (int)page);
          bulk_load_1d(scales, p.cache + page * page_bytes + (int64_t)p.block_size * D + in * 4, R * 4, full_scales);
        };
        auto load_k = [&](int j, int blk) {
          const uint32_t valid = __ballot_sync(0xffffffffu, blk >= 0);
          const bool issuer = blk >= 0 && lane % units == 0;
          const int boxes = __popc(__ballot_sync(0xffffffffu, issuer)), st = kc % kKStages, at = kc % kRing;
          if (kc >= kKStages && !wait_all(&k_empty[st], (kc / kKStages - 1) & 1, 921)) return false;
          if (lane == 0) {
            sValid[at] = valid;
            mbar_expect_tx(&k_full[st], boxes * R * D);
            mbar_expect_tx(&ks_full[at], boxes * R * 4);
          }
          __syncwarp();
          if (issuer)
            copy(it.key0 + j * kTile + lane * 16, blk, 0, sK + st * C::kK + lane * 16 * D, sScaleK + at * kTile + lane * 16, &k_full[st],
                 &ks_full[at]);
          ++kc;
          return true;
        };
        auto load_v = [&](int j, int blk) {
          const uint32_t valid = __ballot_sync(0xffffffffu, blk >= 0);
          const int key0 = it.key0 + j * kTile;
          const bool issuer = blk >= 0 && lane % units == 0;
          const uint32_t starts = __ballot_sync(0xffffffffu, issuer);
#pragma unroll 1
          for (int pg = 0; pg < 2; ++pg) {
            const int st = rc % kRaw;
            if (rc >= kRaw && !wait_all(&raw_empty[st], (rc / kRaw - 1) & 1, 922)) return false;
            if (lane == 0) {
              const int left = max(0, min(kPage, it.seq_len - key0 - pg * kPage));
              sMeta[st] = (valid >> (4 * pg) & 15u) | (uint32_t)left << 4;
              mbar_expect_tx(&raw_full[st], __popc(starts >> (4 * pg) & 15u) * R * (D + 4));
            }
            __syncwarp();
            if (issuer && lane >> 2 == pg)
              copy(key0 + lane * 16, blk, 1, sRaw + st * C::kCodes + (lane & 3) * 16 * D, sScaleV + st * kPage + (lane & 3) * 16,
                   &raw_full[st], &raw_full[st]);
            ++rc;
          }
          return true;
        };
        int blk = lookup(0), blk_v = -1;
        for (int j = 0; ok && j <= n_max; ++j) {      // K(0), K(1), V(0), K(2), V(1), ...
          if (j == n_max - 1 && p.take && !ask()) { ok = false; break; }
          const int after = lookup(j + 1);
          if (j < n_max) ok = load_k(j, blk);
          if (ok && j >= 1) ok = load_v(j - 1, blk_v);
          blk_v = blk;
          blk = after;
        }
      } else if (p.take) {
        ok = ask();
      }
      if (!p.take || !ok) break;
      if (!wait_all(&next_full[(asked - 1) & 1], ((asked - 1) >> 1) & 1, 929)) { ok = false; break; }
      idx = taken_cta(next_at + 16 * ((asked - 1) & 1));
      fence_proxy_async_smem();
      __syncwarp();
    }
    if (ok) {          // the widening warps' end
      const int st = rc % kRaw;
      if (rc >= kRaw) ok = wait_all(&raw_empty[st], (rc / kRaw - 1) & 1, 922);
      if (ok && lane == 0) {
        sMeta[st] = kMetaEnd;
        mbar_arrive(&raw_full[st]);
      }
    }
    if (!ok && lane == 0) {   // let the copies in flight land before the CTA's shared memory goes away (bounded)
      auto drain = [](uint64_t* bar, uint32_t parity) {
        for (uint32_t q = 0; q < (1u << 16); ++q)
          if (mbar_try_wait(bar, parity)) break;
      };
      if (qc > 0) drain(q_full, (qc - 1) & 1);
      for (int i = max(0, kc - kKStages); i < kc; ++i) drain(&k_full[i % kKStages], (i / kKStages) & 1);
      for (int i = max(0, kc - kRing); i < kc; ++i) drain(&ks_full[i % kRing], (i / kRing) & 1);
      for (int i = max(0, rc - kRaw); i < rc; ++i) drain(&raw_full[i % kRaw], (i / kRaw) & 1);
      if (asked > 0) drain(&next_full[(asked - 1) & 1], ((asked - 1) >> 1) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      // A = a piece of Q, B = K tile (e4m3), both K-major
      constexpr uint32_t idesc_s[2] = {umma_idesc(kTile, kTile, 0, 0, 0, 0), umma_idesc(kTile, kTile, 1, 0, 0, 0)};
      constexpr uint32_t idesc_o = umma_idesc(kTile, D, 0, 0, 0, 1);       // A = P (TMEM), B = V tile (MN-major), fp16
      int kc = 0, vc = 0, qc[2] = {0, 0}, tc[2] = {0, 0};   // consumed so far; tc: tiles of each stream whose P has been awaited
      bool ok = true;
      for (int idx = blockIdx.x, round = 0; idx >= 0; idx = ok ? next_item(round++, false, ok) : -1) {
        get_item<kTile>(p, idx, it);
        if (it.n_max == 0) continue;
        const int n_max = it.n_max;
        // S of tile j of the item; the last reader of a K stage (of Q) gives it back
        auto issue_s = [&](int s, int j) {
          const uint32_t q_addr = smem_u32(sQ + s * C::kQ), k_addr = smem_u32(sK + ((kc + j) % kKStages) * C::kK);
#pragma unroll
          for (int c = 0; c < C::P * (D / 32); ++c)
            umma_f8(tmem_base + s * kTile, desc_rows<D>(q_addr + c / (D / 32) * C::kPiece + c % (D / 32) * 32),
                    desc_rows<D>(k_addr + c % (D / 32) * 32), idesc_s[Pieces<T>::e5(c / (D / 32))], c > 0 ? 1u : 0u);
          umma_commit(&s_full[s]);
          const bool last = s == 1 || j >= it.n[1];
          if (last) {
            umma_commit(&k_empty[(kc + j) % kKStages]);
            if (j == n_max - 1) umma_commit(q_empty);
          }
        };
        ok = wait_or_abort(&k_full[kc % kKStages], (kc / kKStages) & 1, ab, 924);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (!ok || it.n[s] == 0) continue;
          ok = wait_or_abort(&q_ready[s], qc[s] & 1, ab, 923);
          if (!ok) break;
          ++qc[s];
          tc_fence_after_sync();
          issue_s(s, 0);
        }
        if (!ok) break;
        for (int i = 0; ok && i < n_max; ++i) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (!ok || i >= it.n[s]) continue;
            // the last stream that reads this V tile gives it back
            const bool last_v = s == 1 || i >= it.n[1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int v = vc + 2 * i + h;
              ok = ok && wait_or_abort(&v_full[v % kVStages], (v / kVStages) & 1, ab, 925) &&
                   wait_or_abort(&p_ready[s * 2 + h], tc[s] & 1, ab, 926);
              if (!ok) break;
              tc_fence_after_sync();
              const uint32_t v_addr = smem_u32(sV + (v % kVStages) * C::kV);
#pragma unroll
              for (int k = 0; k < kPage / 16; ++k)
                umma_f16_ts(tmem_base + (2 + s) * kTile, tmem_base + s * kTile + h * 32 + k * 8,
                            umma_desc_mn_sw128(v_addr + k * 2048, C::kV / kB, 1024), idesc_o,
                            (i > 0 || h > 0 || k > 0) ? 1u : 0u);
              if (last_v) umma_commit(&v_empty[v % kVStages]);
            }
            if (!ok) break;
            ++tc[s];
            if (i == it.n[s] - 1) {
              umma_commit(&o_final[s]);
            } else {
              const int k = kc + i + 1;
              if (!wait_or_abort(&k_full[k % kKStages], (k / kKStages) & 1, ab, 924)) { ok = false; break; }
              tc_fence_after_sync();
              issue_s(s, i + 1);
            }
          }
        }
        kc += n_max;
        vc += 2 * n_max;
      }
    }
  } else if (warp >= 12) {
    // ------------------------------------------------------------------ V in fp16: 16 codes a thread and step
    const int w = warp - 12;
    for (int n = 0;; ++n) {
      const int st = n % kRaw, to = n % kVStages;
      if (__any_sync(0xffffffffu, !wait_or_abort(&raw_full[st], (n / kRaw) & 1, ab, 931))) break;
      const uint32_t meta = sMeta[st];
      if (meta & kMetaEnd) break;
      const int left = meta >> 4 & 127;
      const uint8_t* src = sRaw + st * C::kCodes;
      const float* scale = sScaleV + st * kPage;
      uint8_t* dst = sV + to * C::kV;
      // A warp takes 16 keys.  Eight lanes together must meet eight different 16-byte places of a 128-byte line, when they read (place =
      // chunk ^ row % 8) and when they write (two chunks of eight values, places of one parity for a row).  Heads of 128: the lower four
      // take the lower half of a row's codes, the upper four the upper half of the next row's, and the other halves a step later.  Heads
      // of 64: two rows of 64 bytes.
      constexpr int kSteps = 16 * D / 512;
      auto where = [&](int i, int& key, int& chunk) {    // chunk: 16 codes of a row
        if constexpr (D == 128) {
          key = w * 16 + (i >> 1) * 8 + (lane >> 2);
          chunk = (lane & 3) + 4 * ((lane >> 2 & 1) ^ (i & 1));
        } else {
          key = w * 16 + i * 8 + (lane >> 2);
          chunk = lane & 3;
        }
      };
      uint4 c[kSteps];          // all loads in front of the first store: the compiler cannot tell the buffers apart
      float sc[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        int key, chunk;
        where(i, key, chunk);
        c[i] = *reinterpret_cast<const uint4*>(src + chunk_at<D>(key, chunk));
        sc[i] = scale[key];
      }
      if (n >= kVStages && __any_sync(0xffffffffu, !wait_or_abort(&v_empty[to], (n / kVStages - 1) & 1, ab, 932))) break;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        int key, chunk;
        where(i, key, chunk);
        // rows that were not read, lie behind the end or hold a NaN (whose key says so): zeros, since a weight of zero does not hide one
        const bool there = key < left && (meta >> (key >> 4) & 1u) && !is_nan_bits(sc[i]);
        const __half2 f = __float2half2_rn(there ? sc[i] : 0.f);
        const uint32_t x[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
        uint32_t y[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) widen4(there ? x[q] : 0u, f, y[2 * q], y[2 * q + 1]);
        const int at = 2 * (chunk & 3);
        uint8_t* row = dst + (chunk >> 2) * (kPage * 128) + key * 128;
        *reinterpret_cast<uint4*>(row + ((at ^ (key & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<uint4*>(row + (((at + 1) ^ (key & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_full[to]);
        mbar_arrive(&raw_empty[st]);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ softmax + epilogue: thread = query row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoft));
    const int s = (warp >> 2) - 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;                 // row of the tile = TMEM lane
    const int r_tok = r / p.g, r_head = r % p.g;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem_base + s * kTile + lane_off, tO = tmem_base + (2 + s) * kTile + lane_off;
    int tc = 0, oc = 0, tiles = 0, qc = 0;    // tiles and items of this stream so far, K tiles and items of both
    bool fail = false;
    bool ok = true;
    for (int idx = blockIdx.x, round = 0; idx >= 0; idx = next_item(round++, true, ok)) {
      get_item<kTile>(p, idx, it);
      const int n = s ? it.n[1] : it.n[0], tok0 = s ? it.tok0[1] : it.tok0[0], toks = s ? it.toks[1] : it.toks[0];
      const bool row_ok = r_tok < toks;                // toks <= 128 / g
      const int64_t orow = (int64_t)(it.qs + tok0 + r_tok) * p.Hq + it.head * p.g + r_head;
      if (it.n_max > 0) ++qc;
      if (n == 0) {
        if (p.splits > 1 && row_ok) p.ws_lse[(int64_t)it.split * p.T * p.Hq + orow] = -INFINITY;
        tiles += it.n_max;
        continue;
      }
      const int pos_first = it.ctx + tok0, pos_last = pos_first + toks - 1, pos = pos_first + r_tok;
      float m_used = -INFINITY, l_sum = 0.f, sc;
      // ---- this row's queries in pieces, over the 16-bit ones; sc: what a score is still to be multiplied with
      {
        const bool late = !wait_or_abort(q_full, (qc - 1) & 1, ab, 920);
        uint8_t* q = sQ + s * C::kQ;
        uint4 x[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c) x[c] = *reinterpret_cast<const uint4*>(q + (c >> 3) * (kTile * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
        // magnitudes compare as integers.  Infinities and NaN, and what is too large for its scale to be a number: NaN in every piece, so
        // that the row's scores are NaN before keys that it does not see are taken out
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          top = __vmaxu2(__vmaxu2(__vmaxu2(top, x[c].x & 0x7fff7fffu), x[c].y & 0x7fff7fffu), __vmaxu2(x[c].z & 0x7fff7fffu, x[c].w & 0x7fff7fffu));
        const uint32_t t16 = max(top & 0xffffu, top >> 16);
        const float amax = to_f(__builtin_bit_cast(T, (uint16_t)t16));
        const bool bad = !row_ok || !(amax <= 8.5e37f);
        const float up2 = pow2_ceil(bad ? 1.f : fmaxf(amax, 1e-30f)), up = Pieces<T>::kTop * pow2_inv(up2);
        const __half2 instead = __float2half2_rn(row_ok ? __uint_as_float(0x7fffffffu) : 0.f);      // of the elements of a bad row
        sc = up2 * (1.f / Pieces<T>::kTop) * p.scale_log2;
        if (bar_red_or(1 + s, 128, late)) { fail = true; break; }     // also: rows of pieces and of queries overlap
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          __half2 rest[8];                   // 16 elements, scaled: at most kTop, fp16 holds them
          const uint32_t in[8] = {x[2 * c].x, x[2 * c].y, x[2 * c].z, x[2 * c].w, x[2 * c + 1].x, x[2 * c + 1].y, x[2 * c + 1].z, x[2 * c + 1].w};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float lo = to_f(__builtin_bit_cast(T, (uint16_t)in[j])), hi = to_f(__builtin_bit_cast(T, (uint16_t)(in[j] >> 16)));
            rest[j] = bad ? instead : __floats2half2_rn(lo * up, hi * up);
          }
#pragma unroll
          for (int k = 0; k < C::P; ++k) {
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              constexpr auto e5 = Pieces<T>::e5;
              const uint16_t a = e5(k) ? f16x2_to_e5m2x2(rest[2 * j]) : f16x2_to_e4m3x2(rest[2 * j]);
              const uint16_t b = e5(k) ? f16x2_to_e5m2x2(rest[2 * j + 1]) : f16x2_to_e4m3x2(rest[2 * j + 1]);
              y[j] = a | (uint32_t)b << 16;
              if (k + 1 < C::P) {
                const uint32_t ua = e5(k) ? e5m2x2_to_f16x2(a) : e4m3x2_to_f16x2(a), ub = e5(k) ? e5m2x2_to_f16x2(b) : e4m3x2_to_f16x2(b);
                rest[2 * j] = __hsub2(rest[2 * j], *reinterpret_cast<const __half2*>(&ua));
                rest[2 * j + 1] = __hsub2(rest[2 * j + 1], *reinterpret_cast<const __half2*>(&ub));
              }
            }
            *reinterpret_cast<uint4*>(q + k * C::kPiece + chunk_at<D>(r, c)) = make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_ready[s]);
      }
      for (int i = 0; i < n; ++i, ++tc) {
        if (__any_sync(0xffffffffu, !wait_or_abort(&s_full[s], tc & 1, ab, 927))) { fail = true; break; }
        tc_fence_after_sync();
        const int key0 = it.key0 + i * kTile;
        uint32_t v[kTile];
#pragma unroll
        for (int c = 0; c < kTile; c += 32) tmem_ld_x32_p(tS + c, v + c);
        const int ring = (tiles + i) % kRing;
        if (__any_sync(0xffffffffu, !wait_or_abort(&ks_full[ring], ((tiles + i) / kRing) & 1, ab, 934))) { fail = true; break; }
        const uint32_t valid = sValid[ring];
        const float4* kscale = reinterpret_cast<const float4*>(sScaleK + ring * kTile);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < kTile; e += 4) {
          const float4 f = kscale[e / 4];
          float a, b;
          unf2(mul2(f2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), f2(f.x, f.y)), a, b);
          v[e] = __float_as_uint(a);
          v[e + 1] = __float_as_uint(b);
          unf2(mul2(f2(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), f2(f.z, f.w)), a, b);
          v[e + 2] = __float_as_uint(a);
          v[e + 3] = __float_as_uint(b);
        }
        // a tile that every row of this stream sees in full needs no mask
        const bool full_tile = key0 + kTile - 1 <= pos_first && key0 + kTile <= it.seq_len && valid == 0xffu &&
                               (p.window <= 0 || key0 > pos_last - p.window);
        if (!full_tile) {
          const int hi = min(pos, it.seq_len - 1) - key0, lo = p.window > 0 ? pos - p.window + 1 - key0 : 0;
#pragma unroll
          for (int e = 0; e < kTile; ++e) v[e] = (e <= hi && e >= lo && (valid >> (e >> 4) & 1u)) ? v[e] : 0xff800000u;   // -inf
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kTile; e += 8) {
#pragma unroll
          for (int u = 0; u < 4; ++u) mx[u] = fmaxf(fmaxf(mx[u], __uint_as_float(v[e + u])), __uint_as_float(v[e + u + 4]));
        }
        float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;   // scale > 0: max commutes
        if (!row_ok) tmax = -INFINITY;
        // ---- lazy running maximum (it moves when a tile exceeds it by more than 8 in log2 units); the rescale of O is
        // warp-collective (TMEM access), so the warp decides together.  S(i) has arrived, so P.V(i - 1) is in O.
        const bool bump = tmax > m_used + kMaxSlack;
        const float alpha = bump ? exp2f(m_used - tmax) : 1.f;
        if (bump) { m_used = tmax; l_sum *= alpha; }
        if (__any_sync(0xffffffffu, bump) && i > 0) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {   // rare path: 32 columns at a time keeps the register count down
            uint32_t o[32];
            tmem_ld_x32_p(tO + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_x32_p(tO + c, o);
          }
        }
        // nothing seen so far: every score is -inf or a NaN, and both stay what they are
        const float neg_m = !row_ok ? -INFINITY : m_used == -INFINITY ? 0.f : -m_used;
        const uint64_t sc2 = f2(sc, sc), neg2 = f2(neg_m, neg_m);
        uint64_t ls[4] = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kTile; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float a, b;
            unf2(fma2(f2(__uint_as_float(v[c + e]), __uint_as_float(v[c + e + 1])), sc2, neg2), a, b);
            a = ex2_approx(a);
            b = ex2_approx(b);
            ls[(e >> 1) & 3] = add2(ls[(e >> 1) & 3], f2(a, b));
            pk[e / 2] = pack2<__half>(a, b);
          }
          tmem_st_x16_p(tS + c / 2, pk);
          if (c == 32 || c == 96) {   // 64 keys of P are on their way: hand them over
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[s * 2 + c / 64]);
          }
        }
        float a0, a1, b0, b1;
        unf2(add2(ls[0], ls[1]), a0, a1);
        unf2(add2(ls[2], ls[3]), b0, b1);
        l_sum += (a0 + a1) + (b0 + b1);
      }
      tiles += it.n_max;
      if (fail) break;
      // ---- epilogue
      if (__any_sync(0xffffffffu, !wait_or_abort(&o_final[s], oc & 1, ab, 928))) { fail = true; break; }
      ++oc;
      tc_fence_after_sync();
      float den = l_sum;
      const float ms = m_used == -INFINITY ? 0.f : m_used;
      if (p.splits == 1 && p.sinks != nullptr) den += exp2f(p.sinks[it.head * p.g + r_head] * kLog2e - ms);
      const float inv = den == 0.f ? 0.f : 1.f / den;      // a NaN stays one
      if (p.splits > 1 && row_ok) p.ws_lse[(int64_t)it.split * p.T * p.Hq + orow] = den == 0.f ? -INFINITY : ms + log2f(den);
#pragma unroll
      for (int c = 0; c < D; c += 64) {
        uint32_t o[64];
        tmem_ld_x32_p(tO + c, o);          // warp-collective: every lane loads
        tmem_ld_x32_p(tO + c + 32, o + 32);
        tmem_ld_wait();
        if (row_ok) {
          if (p.splits == 1) {
            T* dst = reinterpret_cast<T*>(p.out) + orow * D;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              uint32_t y[4];
#pragma unroll
              for (int u = 0; u < 4; ++u)
                y[u] = pack2<T>(__uint_as_float(o[q * 8 + 2 * u]) * inv, __uint_as_float(o[q * 8 + 2 * u + 1]) * inv);
              *reinterpret_cast<uint4*>(dst + c + q * 8) = make_uint4(y[0], y[1], y[2], y[3]);
            }
          } else {
            float* dst = p.ws_o + ((int64_t)it.split * p.T * p.Hq + orow) * D;
#pragma unroll
            for (int q = 0; q < 16; ++q)
              *reinterpret_cast<float4*>(dst + c + q * 4) =
                  make_float4(__uint_as_float(o[q * 4]) * inv, __uint_as_float(o[q * 4 + 1]) * inv,
                              __uint_as_float(o[q * 4 + 2]) * inv, __uint_as_float(o[q * 4 + 3]) * inv);
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <typename T, int D>
static int launch(const Params& p, const CUtensorMap& tmQ, const CUtensorMap& tmKV, int64_t items, cudaStream_t st) {
  auto kern = kv8_prompt_kernel<T, D>;
  cudaError_t e = ensure_dynamic_smem((const void*)kern, (int)Cfg<T, D>::kSmem);
  if (e != cudaSuccess) return (int)e;
  e = launch_pdl(kern, dim3((unsigned)items), dim3(kThreads), Cfg<T, D>::kSmem, st, tmQ, tmKV, p);
  if (e != cudaSuccess || p.splits == 1) return (int)e;
  const int64_t rows = p.T * p.Hq;
  return (int)launch_pdl(kv8_join_kernel<T, D>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, (T*)p.out, (const float*)p.ws_o,
                         (const float*)p.ws_lse, p.sinks, rows, p.Hq, 0, p.Hq, p.splits, p.qsl, p.B);
}

}  // namespace kv8prompt
}  // namespace b200

// How a call is cut: tokens of a tile, streams of a CTA, splits of an item's keys.  The scratch of b200_kv8_prompt is splits * T * Hq * (D + 1)
// floats when splits > 1.
extern "C" int b200_kv8_prompt_splits(int B, int Hq, int Hkv, int max_query_len, int64_t max_seq_len, int window, int num_sms) {
  using namespace b200::kv8prompt;
  const int toks = kTile / (Hq / Hkv);
  const int64_t tiles = (int64_t)B * Hkv * ((max_query_len + toks - 1) / toks);
  const int64_t span = window > 0 && window + toks < max_seq_len ? window + toks : max_seq_len, keys = (span + kTile - 1) / kTile;
  // as many as fill the SMs once, four key tiles at least a split
  int64_t s = num_sms / (tiles > 0 ? tiles : 1);
  if (s > keys / 4) s = keys / 4;
  return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}

// Prompt attention over the 8-bit cache.  `tmQ`: q as [T][Hq][D] with boxes of 64 dims, Hq / Hkv heads and 128 / (Hq / Hkv) tokens; `tmKV`: the
// codes as written by b200_encode_tmap_kv8 with boxes of at most 64 keys.  Returns 3 for shapes it does not serve.
extern "C" int b200_kv8_prompt(void* out, const void* cache, const void* tmQ, const void* tmKV, const int* block_tables,
                               const int* seq_lens, const int* qsl, const float* sinks, float* ws_o, float* ws_lse, int splits,
                               int* status, int64_t T_, int B, int Hq, int Hkv, int D, int block_size, int max_blocks,
                               int64_t bt_stride, int64_t num_blocks, int max_query_len, int window, float scale, int dtype,
                               int num_sms, cudaStream_t st) {
  using namespace b200;
  if (B == 0 || max_query_len <= 0 || T_ == 0) return 0;
  if (Hq % Hkv || Hq / Hkv > kv8prompt::kTile || block_size % 16 || (D != 64 && D != 128) || (dtype != kBF16 && dtype != kF16) ||
      num_blocks * 2 * Hkv > 0x7fffffff || window < 0 || num_sms < 1 || splits < 1 || splits > 32 || !(scale > 0.f))
    return 3;
  if (splits > 1 && (ws_o == nullptr || ws_lse == nullptr)) return 2;
  kv8prompt::Params p = {};
  p.out = out; p.ws_o = ws_o; p.ws_lse = ws_lse; p.cache = static_cast<const uint8_t*>(cache); p.block_tables = block_tables;
  p.seq_lens = seq_lens; p.qsl = qsl; p.sinks = sinks; p.status = status; p.num_blocks = num_blocks; p.bt_stride = bt_stride;
  p.T = T_; p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.g = Hq / Hkv; p.block_size = block_size; p.max_blocks = max_blocks; p.window = window;
  p.heads = Hkv;
  p.max_keys = 0x7fffff80;
  p.span = 0x7fffffff;
  p.toks = kv8prompt::kTile / p.g; p.splits = splits; p.scale_log2 = scale * kv8prompt::kLog2e;
  const int64_t tiles = (int64_t)B * Hkv * ((max_query_len + p.toks - 1) / p.toks);
  p.single = tiles * splits <= num_sms;
  const int step = p.single ? p.toks : 2 * p.toks;
  p.row_blocks = (max_query_len + step - 1) / step;
  const int64_t items = (int64_t)B * Hkv * splits * p.row_blocks;
  if (items > (1 << 30)) return 3;
  p.take = items > num_sms;
  const CUtensorMap& q = *reinterpret_cast<const CUtensorMap*>(tmQ);
  const CUtensorMap& kv = *reinterpret_cast<const CUtensorMap*>(tmKV);
  if (dtype == kBF16)
    return D == 64 ? kv8prompt::launch<__nv_bfloat16, 64>(p, q, kv, items, st) : kv8prompt::launch<__nv_bfloat16, 128>(p, q, kv, items, st);
  return D == 64 ? kv8prompt::launch<__half, 64>(p, q, kv, items, st) : kv8prompt::launch<__half, 128>(p, q, kv, items, st);
}
