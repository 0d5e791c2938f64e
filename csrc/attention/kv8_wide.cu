// Prompt and chunk attention over the 8-bit paged cache (common/kv8.cuh) where many query tiles read the same keys: a first kernel writes
// the keys and values that the call needs in 16 bits to scratch, once for all query tiles, a second one multiplies.  Heads of 64, 128, 256.
// (kv8_prompt.cu widens inside the attention kernel, once per pair of query tiles.)
//
// Per key tile and 128-row query tile
//     S[128 rows, N keys]  = Q . K_tile^T           in the queries' type (bf16 or fp16); K is exact in both
//     O[128 rows, D dims] += P[128 rows, N keys] . V    in fp16: V is exact, P rounds to 11 bits; P in TMEM over the columns of S
// A row is (token, head of a group), 128 / g tokens a tile.  Heads of 64 and 128: N = 128, a persistent CTA works on two tiles ("streams") of
// consecutive tokens that read the same K / V tiles, the tensor core on one while the other is in its softmax; a stream's products are
// issued in the order P.V(i), S(i + 1), so the arrival of S(i + 1) says that O holds P.V(i).  Heads of 256: TMEM holds one O of 256 columns,
// so there is one stream with two S buffers of N = 64 keys; S(i + 2) is issued behind P.V(i), the softmax of tile i + 1 meanwhile.
// What bounds it: per 128 keys and tile the tensor core needs 1024 cycles (2048 with heads of 256), the special-function units 1024.
// Widening reads D + 4 and writes 2 D bytes a row; what it writes mostly stays in L2.
// Measured, bf16, 32 / 8 heads of 128: 4 prompts of 2048 tokens 180 us (137 GFLOP of visible scores and values: 760 TFLOP/s); 4096 tokens behind 28672
// 1.83 ms (2.06 TFLOP: 1120 TFLOP/s, 0.69 of what a library product reaches).  Widening inside for every pair of tiles: 239 us and 2.87 ms.
// Warp 0 TMA producer, warp 1 MMA issuer, warps 4-7 and 8-11 softmax and epilogue (thread = row).  The grid has a CTA per item, in descending
// order of row blocks; a CTA that is done takes the next pending one's item (cluster launch control).  Every wait is bounded; on time-out the
// status word is set and the CTA unwinds.
#include "../api.h"
#include "kv8_prompt.cuh"

namespace b200 {
namespace kv8prompt {

template <int D> struct Wide {
  static constexpr int kStreams = D == 256 ? 1 : 2;
  static constexpr int kN = D == 256 ? 64 : 128;           // keys of a tile
  static constexpr int kThreads = 128 + kStreams * 128;
  static constexpr int kB = D / 64;                        // 64-dim blocks of a row
  static constexpr int kQ = kB * kTile * 128, kK = kB * kN * 128, kV = kB * kPage * 128;
  static constexpr int kHalves = kN / kPage;               // P of a tile is handed over 64 keys at a time
  static constexpr int kKStages = 3, kVStages = D == 256 ? 2 : 4;      // V in pages of 64 keys
  // 384 threads: 128 x (104 + 200 + 200) of the 168 x 384 registers that the launch brings
  static constexpr int kRegsFew = 104, kRegsSoft = 200;
  static constexpr int kO = 256;                           // first column of O; S is in front
  static constexpr size_t kSmem = 1024 + kStreams * kQ + kKStages * kK + kVStages * kV + 512;
  static_assert(kSmem <= 227 * 1024);
};

template <typename T> struct Fmt;
template <> struct Fmt<__nv_bfloat16> { static constexpr uint32_t v = 1; };
template <> struct Fmt<__half> { static constexpr uint32_t v = 0; };

// Where the widened rows are: [B][heads][rows][D], rows a multiple of 128 from the request's first_key on, and which 16 keys of every 128 are there.
struct Scratch {
  const void* k;
  const void* v;
  const uint8_t* valid;     // [B][rows / 128]
  int rows;
};

template <typename T, int D>
__global__ void __launch_bounds__(Wide<D>::kThreads, 1)
kv8_wide_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ Params p, const __grid_constant__ Scratch w) {
  using C = Wide<D>;
  constexpr int kB = C::kB, kN = C::kN, kStreams = C::kStreams, kKStages = C::kKStages, kVStages = C::kVStages, kHalves = C::kHalves;
  constexpr bool kOne = kStreams == 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                  // [streams][kB dim blocks][128 rows][128 B]
  uint8_t* sK = sQ + kStreams * C::kQ;                 // [kKStages][kB dim blocks][kN keys][128 B]
  uint8_t* sV = sK + kKStages * C::kK;                 // [kVStages][kB dim blocks][64 keys][128 B]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kVStages * C::kV);
  uint64_t* q_full = bars;              // one phase per item
  uint64_t* q_empty = bars + 1;         // the item's last S has been computed
  uint64_t* k_full = bars + 2;          // [3]
  uint64_t* k_empty = bars + 5;         // [3] S of the tile has been computed for every stream
  uint64_t* v_full = bars + 8;          // [4]
  uint64_t* v_empty = bars + 12;        // [4]
  uint64_t* s_full = bars + 16;         // [2 streams, or buffers of the one]
  uint64_t* p_ready = bars + 18;        // [2][halves] one arrival per softmax warp
  uint64_t* o_final = bars + 22;        // [2 streams] one phase per item with work for the stream
  uint64_t* pv_done = bars + 24;        // one stream: one phase per tile
  // answers about the next item: question k uses slot k & 1
  uint64_t* next_full = bars + 26;      // [2]
  uint64_t* next_empty = bars + 28;     // [2] read by the MMA thread and the softmax warps
  const uint32_t next_at = smem_u32(bars + 30);   // [2] x 16 bytes
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 34);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Abort ab{p.status, abort_flag};
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int b = 0; b < kKStages; ++b) { mbar_init(&k_full[b], 1); mbar_init(&k_empty[b], 1); }
    for (int b = 0; b < kVStages; ++b) { mbar_init(&v_full[b], 1); mbar_init(&v_empty[b], 1); }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&o_final[s], 1);
      for (int h = 0; h < kHalves; ++h) mbar_init(&p_ready[s * kHalves + h], 4);
      mbar_init(&next_full[s], 1);
      mbar_init(&next_empty[s], 1 + 4 * kStreams);
    }
    mbar_init(pv_done, 1);
    mbar_fence_init();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
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
  griddep_wait();   // q, the lengths and the widened rows come from the preceding kernels
  Item it;
  // MMA thread, softmax warps: answer k.  -1: there is no further item, or a wait gave up (then `ok` is false as well).
  auto next_item = [&](int k, bool whole_warp, bool& ok) {
    if (!p.take) return -1;
    ok = wait_or_abort(&next_full[k & 1], (k >> 1) & 1, ab, 959);
    if (whole_warp) ok = !__any_sync(0xffffffffu, !ok);
    if (!ok) return -1;
    const int idx = taken_cta(next_at + 16 * (k & 1));
    fence_proxy_async_smem();           // read before the next answer is written here
    if (whole_warp) __syncwarp();
    if (!whole_warp || lane == 0) mbar_arrive(&next_empty[k & 1]);
    return idx;
  };

  if constexpr (!kOne) {
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsFew));
  }
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int kc = 0, vc = 0, qc = 0, asked = 0;    // K tiles, V pages and items issued, questions asked so far
      bool ok = true;
      // asked when the item's last loads are due: late enough that a CTA does not hold an item it cannot start, early enough that the
      // answer is there before the last tiles have been worked on
      auto ask = [&]() {
        const int b = asked & 1;
        if (asked >= 2 && !wait_or_abort(&next_empty[b], ((asked >> 1) - 1) & 1, ab, 950)) return false;
        mbar_expect_tx(&next_full[b], 16);
        ask_for_cta(next_at + 16 * b, &next_full[b]);
        ++asked;
        return true;
      };
      for (int idx = blockIdx.x; ok && idx >= 0;) {
        get_item<kN>(p, idx, it);
        const int n_max = it.n_max;
        if (n_max > 0) {
          if (qc > 0 && !wait_or_abort(q_empty, (qc - 1) & 1, ab, 951)) { ok = false; break; }
          mbar_expect_tx(q_full, p.toks * p.g * 2 * D * ((it.n[0] > 0) + (it.n[1] > 0)));
#pragma unroll
          for (int s = 0; s < kStreams; ++s)
            if (it.n[s] > 0) {
#pragma unroll
              for (int h = 0; h < kB; ++h)
                tma_load_3d(sQ + s * C::kQ + h * (kTile * 128), &tmQ, q_full, h * 64, it.head * p.g, it.qs + it.tok0[s]);
            }
          ++qc;
          const int row0 = (it.req * p.heads + it.head - p.head0) * w.rows + it.key0 - it.origin;
          for (int j = 0; ok && j <= n_max; ++j) {      // K(0), K(1), V(0), K(2), V(1), ...
            if (j == n_max - 1 && p.take && !ask()) { ok = false; break; }
            if (j < n_max) {
              const int st = kc % kKStages, use = kc / kKStages;
              if (use > 0 && !wait_or_abort(&k_empty[st], (use - 1) & 1, ab, 952)) { ok = false; break; }
              mbar_expect_tx(&k_full[st], C::kK);
#pragma unroll
              for (int h = 0; h < kB; ++h)
                tma_load_2d(sK + st * C::kK + h * (kN * 128), &tmK, &k_full[st], h * 64, row0 + j * kN);
              ++kc;
            }
            if (j >= 1) {
#pragma unroll
              for (int pg = 0; pg < kHalves; ++pg) {
                const int st = vc % kVStages, use = vc / kVStages;
                if (use > 0 && !wait_or_abort(&v_empty[st], (use - 1) & 1, ab, 953)) { ok = false; break; }
                mbar_expect_tx(&v_full[st], C::kV);
#pragma unroll
                for (int h = 0; h < kB; ++h)
                  tma_load_2d(sV + st * C::kV + h * (kPage * 128), &tmV, &v_full[st], h * 64, row0 + (j - 1) * kN + pg * kPage);
                ++vc;
              }
            }
          }
        } else if (p.take) {
          ok = ask();
        }
        if (!p.take || !ok) break;
        if (!wait_or_abort(&next_full[(asked - 1) & 1], ((asked - 1) >> 1) & 1, ab, 959)) { ok = false; break; }
        idx = taken_cta(next_at + 16 * ((asked - 1) & 1));
        fence_proxy_async_smem();
      }
      if (!ok) {   // let the copies in flight land before the CTA's shared memory goes away (bounded)
        auto drain = [](uint64_t* bar, uint32_t parity) {
          for (uint32_t q = 0; q < (1u << 16); ++q)
            if (mbar_try_wait(bar, parity)) break;
        };
        if (qc > 0) drain(q_full, (qc - 1) & 1);
        for (int i = max(0, kc - kKStages); i < kc; ++i) drain(&k_full[i % kKStages], (i / kKStages) & 1);
        for (int i = max(0, vc - kVStages); i < vc; ++i) drain(&v_full[i % kVStages], (i / kVStages) & 1);
        if (asked > 0) drain(&next_full[(asked - 1) & 1], ((asked - 1) >> 1) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t fmt = Fmt<T>::v;
      constexpr uint32_t idesc_s = umma_idesc(kTile, kN, fmt, fmt, 0, 0);  // A = Q, B = K tile, both K-major
      constexpr uint32_t idesc_o = umma_idesc(kTile, D, 0, 0, 0, 1);       // A = P (TMEM), B = V tile (MN-major), fp16
      int kc = 0, vc = 0, qc = 0, tc[2] = {0, 0};   // consumed so far; tc: tiles of each stream whose P has been awaited
      bool ok = true;
      for (int idx = blockIdx.x, round = 0; idx >= 0; idx = ok ? next_item(round++, false, ok) : -1) {
        get_item<kN>(p, idx, it);
        if (it.n_max == 0) continue;
        const int n_max = it.n_max;
        // S of tile j of the item for stream s; the last reader of a K stage (of Q) gives it back
        auto issue_s = [&](int s, int j) {
          const int buf = kOne ? (kc + j) & 1 : s;
          const uint32_t q_addr = smem_u32(sQ + s * C::kQ), k_addr = smem_u32(sK + ((kc + j) % kKStages) * C::kK);
#pragma unroll
          for (int k = 0; k < kB * 4; ++k)
            umma_f16(tmem_base + buf * kN, umma_desc_k_sw128(q_addr + (k / 4) * (kTile * 128) + (k % 4) * 32),
                     umma_desc_k_sw128(k_addr + (k / 4) * (kN * 128) + (k % 4) * 32), idesc_s, k > 0 ? 1u : 0u);
          umma_commit(&s_full[buf]);
          if (kOne || s == 1 || j >= it.n[1]) {
            umma_commit(&k_empty[(kc + j) % kKStages]);
            if (j == n_max - 1) umma_commit(q_empty);
          }
        };
        auto wait_k = [&](int j) {
          const int k = kc + j;
          if (!wait_or_abort(&k_full[k % kKStages], (k / kKStages) & 1, ab, 954)) return false;
          tc_fence_after_sync();
          return true;
        };
        // O of stream s += P of tile i . V
        auto issue_pv = [&](int s, int i, bool last_v) {
          const int buf = kOne ? (kc + i) & 1 : s;
          const uint32_t parity = kOne ? ((kc + i) >> 1) & 1 : tc[s] & 1;
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            const int v = vc + kHalves * i + h;
            if (!wait_or_abort(&v_full[v % kVStages], (v / kVStages) & 1, ab, 955) ||
                !wait_or_abort(&p_ready[buf * kHalves + h], parity, ab, 956))
              return false;
            tc_fence_after_sync();
            const uint32_t v_addr = smem_u32(sV + (v % kVStages) * C::kV);
#pragma unroll
            for (int k = 0; k < kPage / 16; ++k)
              umma_f16_ts(tmem_base + C::kO + s * kTile, tmem_base + buf * kN + h * 32 + k * 8,
                          umma_desc_mn_sw128(v_addr + k * 2048, kPage * 128, 1024), idesc_o, (i > 0 || h > 0 || k > 0) ? 1u : 0u);
            if (last_v) umma_commit(&v_empty[v % kVStages]);
          }
          ++tc[s];
          return true;
        };
        ok = wait_or_abort(q_full, qc & 1, ab, 957) && wait_k(0);
        if (!ok) break;
        ++qc;
        if (it.n[0] > 0) issue_s(0, 0);
        if constexpr (kOne) {
          if (n_max > 1) {
            ok = wait_k(1);
            if (ok) issue_s(0, 1);
          }
          for (int i = 0; ok && i < n_max; ++i) {
            ok = issue_pv(0, i, true);
            if (!ok) break;
            umma_commit(pv_done);
            if (i == n_max - 1) umma_commit(&o_final[0]);
            if (i + 2 < n_max) {
              ok = wait_k(i + 2);
              if (ok) issue_s(0, i + 2);
            }
          }
        } else {
          if (it.n[1] > 0) issue_s(1, 0);
          for (int i = 0; ok && i < n_max; ++i) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              if (!ok || i >= it.n[s]) continue;
              ok = issue_pv(s, i, s == 1 || i >= it.n[1]);
              if (!ok) break;
              if (i == it.n[s] - 1) {
                umma_commit(&o_final[s]);
              } else {
                ok = wait_k(i + 1);
                if (ok) issue_s(s, i + 1);
              }
            }
          }
        }
        kc += n_max;
        vc += kHalves * n_max;
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ softmax + epilogue: thread = query row
    if constexpr (!kOne) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoft));
    const int s = (warp >> 2) - 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;                 // row of the tile = TMEM lane
    const int r_tok = r / p.g, r_head = r % p.g;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tO = tmem_base + C::kO + s * kTile + lane_off;
    const float sc = p.scale_log2;
    int tc = 0, oc = 0;               // tiles and items of this stream so far
    bool fail = false;
    bool ok = true;
    for (int idx = blockIdx.x, round = 0; idx >= 0; idx = next_item(round++, true, ok)) {
      get_item<kN>(p, idx, it);
      const int n = s ? it.n[1] : it.n[0], tok0 = s ? it.tok0[1] : it.tok0[0], toks = s ? it.toks[1] : it.toks[0];
      const bool row_ok = r_tok < toks;                // toks <= 128 / g
      const int64_t orow = (int64_t)(it.qs + tok0 + r_tok) * p.Hq + it.head * p.g + r_head;
      if (n == 0) {
        if (p.splits > 1 && row_ok) p.ws_lse[(int64_t)it.split * p.T * p.Hq + orow] = -INFINITY;
        continue;
      }
      const int pos_first = it.ctx + tok0, pos_last = pos_first + toks - 1, pos = pos_first + r_tok;
      const uint8_t* there = w.valid + (int64_t)it.req * (w.rows / kTile);
      const int key_base = it.origin;
      uint32_t valid_next = there[(it.key0 - key_base) / kTile];
      float m_used = -INFINITY, l_sum = 0.f;
      bool sees = false;               // any key
      for (int i = 0; i < n; ++i, ++tc) {
        const int key0 = it.key0 + i * kN;
        constexpr uint32_t kAll = kN == kTile ? 255u : 15u;
        const uint32_t valid = valid_next >> (key0 % kTile / 16) & kAll;
        if (i + 1 < n) valid_next = there[(key0 + kN - key_base) / kTile];
        const int buf = kOne ? tc & 1 : s;
        const uint32_t tS = tmem_base + buf * kN + lane_off;
        if (__any_sync(0xffffffffu, !wait_or_abort(&s_full[buf], kOne ? (tc >> 1) & 1 : tc & 1, ab, 958))) { fail = true; break; }
        tc_fence_after_sync();
        uint32_t v[kN];
#pragma unroll
        for (int c = 0; c < kN; c += 32) tmem_ld_x32_p(tS + c, v + c);
        tmem_ld_wait();
        // a tile that every row of this stream sees in full needs no mask
        const bool full_tile = key0 + kN - 1 <= pos_first && key0 + kN <= it.seq_len && valid == kAll &&
                               (p.window <= 0 || key0 > pos_last - p.window);
        if (!full_tile) {
          const int hi = min(pos, it.seq_len - 1) - key0, lo = p.window > 0 ? pos - p.window + 1 - key0 : 0;
          const int a = max(lo, 0), b = min(hi, kN - 1);
          if (a <= b) sees |= (valid & (2u << (b >> 4)) - (1u << (a >> 4))) != 0;
#pragma unroll
          for (int e = 0; e < kN; ++e) v[e] = (e <= hi && e >= lo && (valid >> (e >> 4) & 1u)) ? v[e] : 0xff800000u;   // -inf
        } else {
          sees = true;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kN; e += 8) {
#pragma unroll
          for (int u = 0; u < 4; ++u) mx[u] = fmaxf(fmaxf(mx[u], __uint_as_float(v[e + u])), __uint_as_float(v[e + u + 4]));
        }
        float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;   // scale > 0: max commutes
        if (!row_ok) tmax = -INFINITY;
        // ---- lazy running maximum (it moves when a tile exceeds it by more than 8 in log2 units); the rescale of O is warp-collective
        // (TMEM access), so the warp decides together.  Two streams: S(i) has arrived, so P.V(i - 1) is in O; one: P.V(i - 2) is, and the
        // next is waited for.
        const bool bump = tmax > m_used + kMaxSlack;
        const float alpha = bump ? exp2f(m_used - tmax) : 1.f;
        if (bump) { m_used = tmax; l_sum *= alpha; }
        if (__any_sync(0xffffffffu, bump) && i > 0) {
          if constexpr (kOne) {
            if (__any_sync(0xffffffffu, !wait_or_abort(pv_done, (tc - 1) & 1, ab, 960))) { fail = true; break; }
            tc_fence_after_sync();
          }
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
        for (int c = 0; c < kN; c += 32) {
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
          if (c % kPage == 32) {   // 64 keys of P are on their way: hand them over
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[buf * kHalves + c / kPage]);
          }
        }
        float a0, a1, b0, b1;
        unf2(add2(ls[0], ls[1]), a0, a1);
        unf2(add2(ls[2], ls[3]), b0, b1);
        l_sum += (a0 + a1) + (b0 + b1);
      }
      if (fail) break;
      // ---- epilogue
      if (__any_sync(0xffffffffu, !wait_or_abort(&o_final[s], oc & 1, ab, 961))) { fail = true; break; }
      ++oc;
      tc_fence_after_sync();
      float den = l_sum;
      const float ms = m_used == -INFINITY ? 0.f : m_used;
      if (p.splits == 1 && p.sinks != nullptr) den += exp2f(p.sinks[it.head * p.g + r_head] * kLog2e - ms);
      // A NaN stays one.  A row that sees no key gives zeros; one whose scores are all -inf (its query is not finite) NaN, but as a split only if
      // no other has more.
      const float inv = den == 0.f ? (sees ? NAN : 0.f) : 1.f / den;
      if (p.splits > 1 && row_ok)
        p.ws_lse[(int64_t)it.split * p.T * p.Hq + orow] = den != 0.f ? ms + log2f(den) : sees ? kLowest : -INFINITY;
#pragma unroll 1
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

// Keys (in T, even blockIdx.x) or values (in fp16, odd) of a tile of 128 keys of a request and head, as far as the call needs it.  Rows that were not
// written, or whose block is outside the pool: zeros; a NaN stays one in the key and is a zero in the value, since a weight of zero would
// not hide it.  A thread takes 16 codes of a row at a time.
template <typename T, int D>
__global__ void __launch_bounds__(256)
kv8_widen_kernel(T* __restrict__ k, __half* __restrict__ v, uint8_t* __restrict__ valid, int rows, Kv8Cache c,
                 const int* __restrict__ block_tables, int64_t bt_stride, int max_blocks, const int* __restrict__ seq_lens,
                 const int* __restrict__ qsl, int window, int max_keys, int head0) {
  griddep_launch();
  griddep_wait();
  const int tile = blockIdx.x >> 1, which = blockIdx.x & 1, h = head0 + blockIdx.y, req = blockIdx.z;
  const int q_len = qsl[req + 1] - qsl[req], seq_len = seq_lens[req], first = first_key(seq_len - q_len, window, max_keys);
  // a request whose rows see nothing has its first tile read all the same
  if (q_len <= 0 || (tile > 0 && tile * kTile >= min(seq_len, max_keys) - first)) return;
  const int key0 = first + tile * kTile;
  const int* bt = block_tables + (int64_t)req * bt_stride;
  auto block_of = [&](int key) -> int {
    if (key >= seq_len) return -1;
    const int bi = key / c.block_size;
    const int b = bi < max_blocks ? bt[bi] : -1;
    return b >= 0 && b < c.num_blocks ? b : -1;
  };
  if (blockIdx.y == 0 && which == 0 && threadIdx.x < 32) {
    const uint32_t bits = __ballot_sync(0xffffffffu, threadIdx.x < 8 && block_of(key0 + threadIdx.x * 16) >= 0);
    if (threadIdx.x == 0) valid[(int64_t)req * (rows / kTile) + tile] = (uint8_t)bits;
  }
  constexpr int kPer = D / 16, kSteps = kTile * kPer / 256;
  const int64_t out0 = (((int64_t)req * gridDim.y + blockIdx.y) * rows + tile * kTile) * D;
  uint4 codes[kSteps];
  float scale[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int x = i * 256 + threadIdx.x, key = key0 + x / kPer, b = block_of(key);
    codes[i] = make_uint4(0, 0, 0, 0);
    scale[i] = 0.f;
    if (b >= 0) {
      uint8_t* page = c.page(b, which, h);
      const int off = key % c.block_size;
      codes[i] = *reinterpret_cast<const uint4*>(c.codes(page, off) + x % kPer * 16);
      scale[i] = *c.scale(page, off);
    }
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int x = i * 256 + threadIdx.x;
    const uint32_t in[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
    const float f = which && is_nan_bits(scale[i]) ? 0.f : scale[i];
    uint32_t y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 a = e4m3x2_to_float2((uint16_t)(in[j / 2] >> (16 * (j & 1))));
      y[j] = which ? pack2<__half>(a.x * f, a.y * f) : pack2<T>(a.x * f, a.y * f);
    }
    uint4* dst = which ? reinterpret_cast<uint4*>(v + out0 + (int64_t)x * 16) : reinterpret_cast<uint4*>(k + out0 + (int64_t)x * 16);
    dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
    dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
  }
}

template <typename T, int D>
static int launch_wide(const Params& p, const Scratch& w, const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV,
                       int64_t items, cudaStream_t st) {
  const Kv8Cache c{const_cast<uint8_t*>(p.cache), p.num_blocks, p.Hkv, p.block_size, D};
  cudaError_t e = launch_pdl(kv8_widen_kernel<T, D>, dim3(2 * (w.rows / kTile), p.heads, p.B), dim3(256), 0, st, (T*)w.k, (__half*)w.v,
                             (uint8_t*)w.valid, w.rows, c, p.block_tables, p.bt_stride, p.max_blocks, p.seq_lens, p.qsl, p.window,
                             p.max_keys, p.head0);
  if (e != cudaSuccess) return (int)e;
  auto kern = kv8_wide_kernel<T, D>;
  e = ensure_dynamic_smem((const void*)kern, (int)Wide<D>::kSmem);
  if (e != cudaSuccess) return (int)e;
  e = launch_pdl(kern, dim3((unsigned)items), dim3(Wide<D>::kThreads), Wide<D>::kSmem, st, tmQ, tmK, tmV, p, w);
  if (e != cudaSuccess || p.splits == 1) return (int)e;
  const int64_t rows = p.T * p.Hq;
  return (int)launch_pdl(kv8_join_kernel<T, D>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, (T*)p.out, (const float*)p.ws_o,
                         (const float*)p.ws_lse, p.sinks, rows, p.Hq, p.head0 * p.g, p.heads * p.g, p.splits, p.qsl, p.B);
}

}  // namespace kv8prompt
}  // namespace b200

// Prompt attention over the 8-bit cache through scratch, for key / value heads head0 .. head0 + heads - 1: wide_k, wide_v
// [B][heads][rows][D] 16-bit and valid [B][rows / 128] bytes.  max_keys: the
// longest request rounded up to 128; rows: the same, or with a window no less than window + max_query_len + 127 rounded down to it.  `tmQ` as for b200_kv8_prompt, `tmK` / `tmV`: the scratch as 2-D with boxes of 64 columns and 128 (heads of
// 256: 64) and 64 rows.  splits and its scratch as for b200_kv8_prompt.  Returns 3 for shapes it does not serve.
extern "C" int b200_kv8_wide(void* out, const void* cache, const void* tmQ, const void* tmK, const void* tmV, void* wide_k, void* wide_v,
                             void* valid, int rows, int max_keys, const int* block_tables, const int* seq_lens, const int* qsl, const float* sinks,
                             float* ws_o, float* ws_lse, int splits, int* status, int64_t T_, int B, int Hq, int Hkv, int head0, int heads,
                             int D, int block_size, int max_blocks, int64_t bt_stride, int64_t num_blocks, int max_query_len, int window,
                             float scale, int dtype, int num_sms, cudaStream_t st) {
  using namespace b200;
  if (B == 0 || max_query_len <= 0 || T_ == 0) return 0;
  if (Hq % Hkv || Hq / Hkv > kv8prompt::kTile || block_size % 16 || (D != 64 && D != 128 && D != 256) ||
      (dtype != kBF16 && dtype != kF16) || window < 0 || num_sms < 1 || splits < 1 || splits > 32 || !(scale > 0.f) || rows < 128 ||
      rows % 128 || max_keys < rows || max_keys % 128 || max_keys > 0x7fffff80 || (int64_t)B * heads * rows > 0x7fffffff || B > 65535 || heads > 65535 ||
      head0 < 0 || heads < 1 || head0 + heads > Hkv)
    return 3;
  if (splits > 1 && (ws_o == nullptr || ws_lse == nullptr)) return 2;
  kv8prompt::Params p = {};
  p.out = out; p.ws_o = ws_o; p.ws_lse = ws_lse; p.cache = static_cast<const uint8_t*>(cache); p.block_tables = block_tables;
  p.seq_lens = seq_lens; p.qsl = qsl; p.sinks = sinks; p.status = status; p.num_blocks = num_blocks; p.bt_stride = bt_stride;
  p.T = T_; p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.g = Hq / Hkv; p.block_size = block_size; p.max_blocks = max_blocks; p.window = window;
  p.head0 = head0; p.heads = heads;
  p.max_keys = max_keys;
  p.span = rows;
  p.toks = kv8prompt::kTile / p.g; p.splits = splits; p.scale_log2 = scale * kv8prompt::kLog2e;
  const int64_t tiles = (int64_t)B * heads * ((max_query_len + p.toks - 1) / p.toks);
  p.single = D == 256 || tiles * splits <= num_sms;
  const int step = p.single ? p.toks : 2 * p.toks;
  p.row_blocks = (max_query_len + step - 1) / step;
  const int64_t items = (int64_t)B * heads * splits * p.row_blocks;
  if (items > (1 << 30)) return 3;
  p.take = items > num_sms;
  const kv8prompt::Scratch w{wide_k, wide_v, static_cast<const uint8_t*>(valid), rows};
  const CUtensorMap& q = *reinterpret_cast<const CUtensorMap*>(tmQ);
  const CUtensorMap& k = *reinterpret_cast<const CUtensorMap*>(tmK);
  const CUtensorMap& v = *reinterpret_cast<const CUtensorMap*>(tmV);
#define B200_KV8_WIDE(TT, DD) return kv8prompt::launch_wide<TT, DD>(p, w, q, k, v, items, st)
  if (dtype == kBF16) {
    if (D == 64) B200_KV8_WIDE(__nv_bfloat16, 64);
    if (D == 128) B200_KV8_WIDE(__nv_bfloat16, 128);
    B200_KV8_WIDE(__nv_bfloat16, 256);
  }
  if (D == 64) B200_KV8_WIDE(__half, 64);
  if (D == 128) B200_KV8_WIDE(__half, 128);
  B200_KV8_WIDE(__half, 256);
#undef B200_KV8_WIDE
}
