// Decode attention over the 8-bit paged cache (common/kv8.cuh) on tcgen05 + TMEM, fed by TMA straight from the pages: at most 16
// query rows (heads of a group x query tokens) per key / value head, heads of 64, 128 or 256.
//
// What bounds it is reading the cache, D + 4 bytes a row, so nothing is converted on the way: codes go from memory to shared memory to
// the tensor core as e4m3 operands, and the numbers that have more digits are taken apart instead.
//   * Queries: q times a power of two that puts the row's largest element in (2^14, 2^15] (fp16: half of that) is the sum of three pieces, each
//     the rounded rest of those in front of it.  An e5m2 piece has three significant bits, an e4m3 piece four, and rests are signed, so three
//     e5m2 pieces hold the 8 bits of bf16 exactly, off by 2^-32 of the row's largest element for the smallest ones, and two of them with one of
//     e4m3 the 11 bits of fp16, off by 2^-24: no more than fp32 sums with the largest element are.  All pieces add into one accumulator.
//     (Two and three e4m3 pieces, off by 2^-18, made rows with one element 2^11 times the others wrong by up to 5 %.)
//   * Weights: exp2(s - m) * v_scale * 2^lift, m the largest s + log2(v_scale) that the row has seen, so that neither a heavy key with a small
//     value nor a light or hidden one with a large value takes the others' digits.  In fp16 and then in three pieces; each rest is multiplied
//     up so that weights far below the largest keep theirs, and every piece has accumulator columns of its own.  The many keys behind one that
//     holds most of a row count together however little each weighs, so the range matters as much as the digits.  bf16: e5m2 pieces, rests
//     times 2^3, weights up to 2^15: off by 2^-9, and by half the last piece's smallest step, 2^-30 of the largest.  fp16: e4m3 pieces, rests
//     times 2^5, weights up to 2^8: 2^-12, and 2^-25 of the largest, the smallest step of the prompt kernels' fp16 weights.  Two e4m3
//     pieces for bf16 (off by 2^-8, and by 2^-18 of the largest: 32768 keys just below that, 12 % of a row, count as nothing) are no faster:
//     16 x 4096 tokens of 32 / 8 heads of 128 33.9 us, with three pieces 34.1; 48 ragged requests 62.4 and 62.7; 64 requests of two tokens
//     behind 4095, 64 / 8 heads of 64, 215 and 213.
// Few query rows and many keys: keys are the UMMA M side, query rows the N side.
//     S^T[128 rows, 16]        = K[128 rows, 128 B] . Q^T      per piece, K-major as cached
//     O^T[128 dims, 16 pieces] += V^T[128 dims, 128 rows] . P   V MN-major as cached
// Heads of 64: a row of 128 bytes holds two keys, so Q^T has 32 columns, (q, 0) and (0, q): scores of the even and the odd keys; P has the
// even keys' weights in one half of its columns and the odd ones' in the other, and O is the sum of the two matching quadrants.
// Heads of 256: two 128-byte blocks a key, two O^T accumulators.
//
// Work: all tiles of all (request, head) items in one line, cut into equal pieces, one a CTA (two CTAs an SM where shared memory lasts), so
// that uneven requests cost what their sum costs.  Cuts come from the lengths on the device: captured launches adapt.  An item
// that lies in several CTAs is merged by the last of them to arrive, in the order of the cuts: the result does not depend on who that is.
// 192, 320 or 576 threads: warp 0 TMA producer (a lane per box of a tile, which looks its block up a tile ahead), warp 1 MMA issuer, the others
// softmax (thread = row of the tile; TMEM lane = output dim at the end) and queries: groups of four warps that share the scores of a row by
// query rows and, with heads of 64, by keys, so that a thread has eight at most.  What is done once an item is kept short in code as
// well as in time: half of a call's time went into it before, most of that into fetching instructions.  Merging waits for the end of
// the CTA's work, where one fence serves both of its cut items.  Every wait is bounded; on time-out the status word is
// set and the CTA unwinds.
// Measured, us (bf16, caches larger than L2; floor = bytes at 6.56 TB/s): 16 requests of 4096 tokens, 32 / 8 heads of 128: 33 (21); 64 of them 94
// to 101 (85); 48 of up to 8192, 32 / 4 heads: 63 (42); 16 / 2 heads of 256, 16 x 4096: 25 (11); 64 / 8 heads of 64, 16 x 4096: 41 (11), of
// two tokens 65.  The first version, a thread per row of the tile with all its scores: 37 for the first of these.  On the CUDA cores: 344.
#include <cuda.h>
#include <math.h>

#include "../api.h"
#include "../common/kv8.cuh"
#include "../common/launch.cuh"
#include "../common/ptx.cuh"
#include "../gemm/gemm_common.cuh"

namespace b200 {
namespace kv8dec {

constexpr int kM = 128;          // rows of 128 bytes in a tile
constexpr int kRows = 16;        // query rows, zero padded
constexpr int kMaxB = 2048;      // requests a launch
// A cut this close to an item's end moves there (tiles; CTAs of one tile keep theirs): one tile costs less than a merge of 16 rows.  us without
// and with, 12 requests of 600 tokens, 8 heads of 128: 16 rows 26.0 and 23.2, 8 rows 18.3 and 16.6, 4 rows 14.6 and 13.2; of 2000, 16 rows: 39.7 and
// 40.8.
constexpr int kSnap = 1;
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  const void* q;            // [T, Hq, D], token stride q_stride
  void* out;                // [T, Hq, D]
  const uint8_t* cache;
  float* ws_o;              // [2 * grid][16][D]
  float* ws_lse;            // [2 * grid][16]
  int* tickets;             // [B * Hkv], zero between calls
  const int* block_tables;
  const int* seq_lens;
  const int* qsl;
  const float* sinks;
  int* status;
  int64_t num_blocks, bt_stride, q_stride;
  int B, Hq, Hkv, block_size, max_blocks, max_keys, window, slots, early_meta;
  float scale_log2;
};

template <int D> struct Geo {
  static constexpr int kPack = D == 64 ? 2 : 1;        // keys in a row of 128 bytes
  static constexpr int kBlk = D == 256 ? 2 : 1;        // 128-byte blocks of a key
  static constexpr int kKeys = kM * kPack;             // keys of a tile
  static constexpr int kOp = kBlk * kM * 128;          // codes of K or V of a tile
  static constexpr int kNS = kRows * kPack;            // columns of S^T
};
// Pieces of a query (q; of those scaled to at most kTop) and of a weight (w; the rest times kStep from one to the next).  The running maximum moves when a score exceeds it by
// more than kSlack (log2): weights stay below 2^(kLift + kSlack).
template <typename T> struct Pieces;
template <> struct Pieces<__nv_bfloat16> {
  static constexpr int q = 3, w = 3;
  static constexpr bool kE5 = true;
  static constexpr float kTop = 32768.f;
  __host__ __device__ static constexpr bool q_e5(int) { return true; }
  static constexpr float kStep = 8.f, kLift = 7.f, kSlack = 8.f;
};
template <> struct Pieces<__half> {
  static constexpr int q = 3, w = 3;
  static constexpr bool kE5 = false;
  static constexpr float kTop = 16384.f;
  __host__ __device__ static constexpr bool q_e5(int piece) { return piece < 2; }
  static constexpr float kStep = 32.f, kLift = 5.f, kSlack = 3.f;
};

template <typename T, int D, int NR> struct Layout {
  using G = Geo<D>;
  static constexpr int P = Pieces<T>::q, W = Pieces<T>::w;
  // Groups of four softmax warps: heads of 64 a group for the even and one for the odd keys; 16 query rows in halves.  8 rows in halves where
  // one CTA an SM fits anyway (heads of 256), and where a row of heads of 64 brings many instructions (fp16's pieces), which two groups overlap
  // better than two CTAs.  us with 8 rows in one group and in two, 16 requests of 4096 tokens / 128 of 1000: heads of 256 bf16 28.0 and 25.3 / 40.6
  // and 36.1, fp16 30.5 and 27.4 / 43.7 and 38.1; heads of 64 bf16 40.8 and 41.4 / 77.2 and 81.8, fp16 49.3 and 45.5 / 100.0 and 91.7; heads of 128
  // bf16 29.2 and 29.7 / (64 of 4096) 61.1 and 62.8.
  static constexpr int kKeyGroups = G::kPack;
  static constexpr int kRowGroups = NR == 16 || (NR == 8 && (D == 256 || (D == 64 && !Pieces<T>::kE5))) ? 2 : 1;
  static constexpr int kGroups = kKeyGroups * kRowGroups;
  static constexpr int kSoft = 128 * kGroups, kThreads = 64 + kSoft;
  static constexpr int kCtas = D == 256 || kGroups == 4 ? 1 : 2;        // an SM at most: shared memory, registers
  static constexpr int kRowsOf = NR / kRowGroups;                       // query rows of a thread
  static constexpr int kNO = G::kNS * W;                       // columns of an O^T accumulator
  static constexpr int kQ = P * G::kBlk * G::kNS * 128;        // queries
  static constexpr int kP = kNO * 128;                         // one weight buffer
  static constexpr int kCols = 2 * G::kNS + G::kBlk * kNO;
  static constexpr int kTmem = kCols <= 64 ? 64 : kCols <= 128 ? 128 : 256;
  static constexpr int kScales = G::kKeys * 4;
  // barriers, factors, flags, exchange buffers
  static constexpr int kMisc = 2048 + (D == 64 ? kRows * 64 * 4 : 0);
  static size_t smem(int slots, int B) {
    return 1024 + (size_t)slots * (G::kOp + kScales) + kQ + 2 * kP + kMisc + (size_t)(B + 1) * 4;
  }
};

__device__ __forceinline__ void named_bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ float warp_max_redux(float v) {
  int i = __float_as_int(v);
  i = i >= 0 ? i : i ^ 0x7fffffff;
  i = __reduce_max_sync(0xffffffffu, i);
  i = i >= 0 ? i : i ^ 0x7fffffff;
  return __int_as_float(i);
}
// The columns of a thread's rows and no others: the columns next to them are another group's, which may be writing them.
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[8]) { tmem_ld_x8(taddr, r); }
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_rows(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_rows(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// 2^x, results below 2^-126 as zero, which is far below what a weight's pieces hold
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }

// The last request whose tiles start at or before unit `at`: those without tiles lie in front of it.
__device__ __forceinline__ int request_at(const int* pre, int B, int Hkv, int at) {
  int a = 0, b = B;
#pragma unroll 1
  while (b - a > 1) {
    const int mid = (a + b) >> 1;
    if (pre[mid] * Hkv <= at) a = mid; else b = mid;
  }
  return a;
}

// Cut b of the line of units: b * share, moved to the end of an item that is at most `snap` tiles away.
__device__ __forceinline__ int cut_at(const int* pre, int B, int Hkv, int units, int share, int snap, int b) {
  const long long p = (long long)share * b;
  if (p == 0 || p >= units) return p == 0 ? 0 : units;
  const int at = (int)p, a = request_at(pre, B, Hkv, at), n = pre[a + 1] - pre[a];
  const int in = (int)((unsigned)(at - pre[a] * Hkv) % (unsigned)n);
  if (min(in, n - in) > snap) return at;
  return in <= n - in ? at - in : at + n - in;
}

// A CTA's share of the line of tiles, item by item.
struct Walk {
  const int* pre;          // [B + 1] tiles of the requests in front (of one head)
  int at, end;             // units left
  int Hkv, B;
  int req, head, tile, n;  // current item: its tiles, and the first of this CTA's among them
  int count;               // this CTA's tiles of it
  __device__ __forceinline__ void start(const int* pre_, int B_, int Hkv_, int lo, int hi) {
    pre = pre_; B = B_; Hkv = Hkv_; at = lo; end = hi;
    count = 0;
    if (at >= end) return;
    const int a = request_at(pre, B, Hkv, at);
    req = a;
    n = pre[a + 1] - pre[a];
    const unsigned in = at - pre[a] * Hkv;
    head = in / (unsigned)n;
    tile = in - head * n;
    count = min(n - tile, end - at);
  }
  __device__ __forceinline__ bool more() const { return count > 0; }
  __device__ __forceinline__ void next() {
    at += count;
    count = 0;
    if (at >= end) return;
    tile = 0;
    if (++head == Hkv) {
      head = 0;
#pragma unroll 1
      do { ++req; n = pre[req + 1] - pre[req]; } while (n == 0);
    }
    count = min(n, end - at);
  }
};

struct Request {
  int qs, q_len, seq_len, ctx, kv_begin;
};
template <int D>
__device__ __forceinline__ Request request_of(const Params& p, int req) {
  Request r;
  r.qs = p.qsl[req];
  r.q_len = p.qsl[req + 1] - r.qs;
  r.seq_len = p.seq_lens[req];
  r.ctx = r.seq_len - r.q_len;
  r.kv_begin = p.window > 0 ? max(0, r.ctx - p.window + 1) / Geo<D>::kKeys * Geo<D>::kKeys : 0;
  return r;
}

template <typename T, int D, int NR>
__global__ void __launch_bounds__((Layout<T, D, NR>::kThreads), (Layout<T, D, NR>::kCtas))
kv8_decode_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ Params p) {
  using G = Geo<D>;
  using L = Layout<T, D, NR>;
  constexpr int P = L::P, W = L::W, kPack = G::kPack, kBlk = G::kBlk, kKeys = G::kKeys, kNS = G::kNS, kNO = L::kNO, kSoft = L::kSoft, kWarps = kSoft / 32;
  constexpr int kRowsOf = L::kRowsOf, kThreads = L::kThreads;
  using Pc = Pieces<T>;
  constexpr float kLift = Pc::kLift, kSlack = Pc::kSlack;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int ns = p.slots;
  uint8_t* sQ = smem + ns * G::kOp;                          // [P][kBlk][kNS][128 B]
  uint8_t* sP = sQ + L::kQ;                                  // [2][kNO][128 B]
  float* sScale = reinterpret_cast<float*>(sP + 2 * L::kP);  // [ns][kKeys]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sScale + ns * kKeys);
  uint64_t* kv_full = bars;              // [16]
  uint64_t* kv_empty = bars + 16;        // [16] the product that reads the codes, and the warps that read the scales
  uint64_t* s_full = bars + 32;          // [2]
  uint64_t* s_empty = bars + 34;         // [2]
  uint64_t* p_ready = bars + 36;         // [2]
  uint64_t* p_free = bars + 38;          // [2]
  uint64_t* q_ready = bars + 40;         // a phase per item
  uint64_t* o_done = bars + 41;          // a phase per tile
  uint64_t* o_final = bars + 42;         // a phase per item
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 44);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* ok_slot = abort_flag + 1;                    // [16]
  int* s_last = const_cast<int*>(abort_flag) + 17;
  uint32_t* sValid = tmem_slot + 20;                         // [16] boxes of a K slot that were read
  uint32_t* sOdd = sValid + 16;                              // [16] heads of 64: 1 + the row of a K slot whose second key is behind the end
  float* sFactor = reinterpret_cast<float*>(sOdd + 16);      // [2 items][16]
  float* sMax = sFactor + 2 * kRows;                         // [16 warps][8] maxima of a group's rows
  float* sSum = sMax + 16 * 8;                               // [16][8]
  float* sInv = sSum + 16 * 8;                               // [16]
  int* sScan = reinterpret_cast<int*>(sInv + kRows);         // [18]
  int* sPend = sScan + 20;                                   // [2][8] the CTA's cut items: ticket, its CTAs, rows, output
  float* sHalf = reinterpret_cast<float*>(sPend + 16);       // [16][64] (heads of 64)
  int* sPre = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + L::kMisc);   // [B + 1]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Abort ab{p.status, abort_flag};
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < ns; ++s) { mbar_init(&kv_full[s], 1); mbar_init(&kv_empty[s], 1 + kWarps); }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s_full[b], 1); mbar_init(&s_empty[b], kWarps);
      mbar_init(&p_ready[b], kWarps); mbar_init(&p_free[b], 1);
    }
    mbar_init(q_ready, kWarps);
    mbar_init(o_done, 1);
    mbar_init(o_final, 1);
    mbar_fence_init();
    prefetch_tmap(&tm);
    griddep_launch();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmem);
    tmem_relinquish();
  }
  // columns of queries and weights that no row uses, and the halves of heads of 64, stay zero
  for (int c = threadIdx.x; c < (L::kQ + 2 * L::kP) / 16; c += kThreads) reinterpret_cast<uint4*>(sQ)[c] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();

  // With early_meta lengths and block tables were written long before this launch, and old tokens' rows as well: both are read before
  // the wait for the kernels in front.
  if (!p.early_meta) griddep_wait();
  const int g = p.Hq / p.Hkv;
  {
    // tiles of every request, summed up over those in front: a thread has consecutive requests
    const int per = (p.B + kThreads - 1) / kThreads, lo = min(p.B, (int)threadIdx.x * per), hi = min(p.B, lo + per);
    int sum = 0;
    for (int r = lo; r < hi; ++r) {
      const Request q = request_of<D>(p, r);
      const bool served = q.q_len > 0 && q.q_len * g <= NR;
      // a request whose rows see nothing has a tile all the same: it writes their zeros
      const int end = min(q.seq_len, p.max_keys);      // the block table has no more
      const int n = served ? max(1, (end - q.kv_begin + kKeys - 1) / kKeys) : 0;
      sPre[r + 1] = n;
      sum += n;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sScan[warp] = incl;
    __syncthreads();
    int base = incl - sum;
    for (int w = 0; w < warp; ++w) base += sScan[w];
    for (int r = lo; r < hi; ++r) { base += sPre[r + 1]; sPre[r + 1] = base; }
    if (threadIdx.x == 0) sPre[0] = 0;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  const int units = sPre[p.B] * p.Hkv;
  const int share = max((units + (int)gridDim.x - 1) / (int)gridDim.x, 1);
  const int snap = share > 1 ? kSnap : 0;
  const int lo = cut_at(sPre, p.B, p.Hkv, units, share, snap, blockIdx.x), hi = cut_at(sPre, p.B, p.Hkv, units, share, snap, blockIdx.x + 1);
  const int n_tiles = hi - lo;
  Walk it;
  it.start(sPre, p.B, p.Hkv, lo, hi);

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer: lane b = box b of the tile
    const int page_rows = p.block_size / kPack;
    const int box = page_rows & -page_rows, R = min(kM, box), boxes = kM / R;      // power of two rows a box; the host's map agrees
    const int64_t page_bytes = (int64_t)p.block_size * (D + 4);
    int slot = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true, waited = !p.early_meta;
    for (; ok && it.more(); it.next()) {
      const Request r = request_of<D>(p, it.req);
      const int* bt = p.block_tables + (int64_t)it.req * p.bt_stride;
      auto lookup = [&](int i) -> int {      // block of this lane's box in tile i, -1: nothing to read
        const int key = r.kv_begin + i * kKeys + lane * R * kPack;
        if (lane >= boxes || key >= r.seq_len) return -1;
        const int bi = key / p.block_size;
        const int blk = bi < p.max_blocks ? bt[bi] : -1;
        return blk >= 0 && blk < p.num_blocks ? blk : -1;
      };
      int blk = lookup(it.tile);
      for (int i = it.tile; ok && i < it.tile + it.count; ++i) {
        const int key0 = r.kv_begin + i * kKeys;
        const int after = i + 1 < it.tile + it.count ? lookup(i + 1) : -1;
        if (!waited && (issued >= ns || key0 + kKeys > r.ctx)) {   // rows of this step come from the kernels in front
          griddep_wait();
          waited = true;
        }
        const uint32_t valid = __ballot_sync(0xffffffffu, blk >= 0);
        const int row = ((key0 + lane * R * kPack) % p.block_size) / kPack;
        const int64_t page = ((int64_t)max(blk, 0) * 2) * p.Hkv + it.head;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (issued >= ns) {
            if (lane == 0) ok = wait_or_abort(&kv_empty[slot], phase ^ 1, ab, 901);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
          }
          if (lane == 0) {
            if (w == 0) {
              sValid[slot] = valid;
              const int left = r.seq_len - key0;
              if (kPack == 2) sOdd[slot] = left > 0 && left < kKeys && (left & 1) ? 1 + left / 2 : 0;
            }
            mbar_expect_tx(&kv_full[slot], __popc(valid) * (R * 128 * kBlk + R * kPack * 4));
          }
          __syncwarp();
          if (blk >= 0) {
            const int64_t pg = page + (int64_t)w * p.Hkv;
#pragma unroll
            for (int b = 0; b < kBlk; ++b)
              tma_load_3d(smem + slot * G::kOp + b * (kM * 128) + lane * R * 128, &tm, &kv_full[slot], b * 128, row, (int)pg);
            bulk_load_1d(sScale + slot * kKeys + lane * R * kPack,
                         p.cache + pg * page_bytes + (int64_t)p.block_size * D + row * kPack * 4, R * kPack * 4, &kv_full[slot]);
          }
          ++issued;
          if (++slot == ns) { slot = 0; phase ^= 1; }
        }
        blk = after;
      }
    }
    if (!ok && lane == 0) {     // let the copies in flight land before the CTA's shared memory goes away (bounded)
      const int pending = min(issued, ns);
      for (int i = 0; i < pending; ++i) {
        const int s = (slot - 1 - i + 2 * ns) % ns;
        const uint32_t ph = s < slot ? phase : phase ^ 1;
        for (uint32_t k = 0; k < (1u << 16); ++k)
          if (mbar_try_wait(&kv_full[s], ph)) break;
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (p.early_meta) griddep_wait();        // as the queries' warps do: the limit of the waits below is for this kernel's own work alone
    if (elect_one() && n_tiles > 0) {
      // A = K (e4m3, K-major), B = a piece of Q^T (K-major)
      constexpr uint32_t idesc_s[2] = {umma_idesc(kM, kNS, 0, 0, 0, 0), umma_idesc(kM, kNS, 0, 1, 0, 0)};
      constexpr uint32_t idesc_o = umma_idesc(kM, kNO, 0, Pc::kE5 ? 1 : 0, 1, 0);     // A = V (e4m3, MN-major), B = P (K-major)
      const uint32_t tS = tmem_base, tO = tmem_base + 2 * kNS;
      const uint32_t q_addr = smem_u32(sQ), p_addr = smem_u32(sP), kv_addr = smem_u32(smem);
      // S of the next tile and P.V of the current one are independent: whichever is ready is issued
      Walk ws = it, wp = it;
      int s_in = 0, p_in = 0, s_item = 0;            // tiles of the current item issued; items begun
      int ks = 0, vs = 1 % ns;                       // slots of the next K and V
      uint32_t kph = 0, vph = 1 / ns;
      int next_s = 0, next_pv = 0;
      uint32_t spins = 0;
      while (next_pv < n_tiles) {
        bool progressed = false;
        if (next_s < n_tiles && next_s <= next_pv + 1 && (s_in > 0 || mbar_try_wait(q_ready, s_item & 1)) &&
            mbar_try_wait(&kv_full[ks], kph) &&
            (next_s < 2 || mbar_try_wait(&s_empty[next_s & 1], ((next_s >> 1) - 1) & 1))) {
          tc_fence_after_sync();
          if (kPack == 2 && sOdd[ks] != 0) {
            // this key's codes were not written and meet zeros of Q^T in its neighbour's scores, which do not hide a NaN
            const int row = (int)sOdd[ks] - 1;
#pragma unroll
            for (int c = 4; c < 8; ++c)
              *reinterpret_cast<uint4*>(smem + ks * G::kOp + row * 128 + ((c ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
          }
          const uint32_t k_at = kv_addr + ks * G::kOp, q_at = q_addr;
#pragma unroll
          for (int c = 0; c < P * kBlk * 4; ++c) {
            const int piece = c / (kBlk * 4), b = (c / 4) % kBlk, k = c % 4;
            umma_f8(tS + (next_s & 1) * kNS, umma_desc_k_sw128(k_at + b * (kM * 128) + k * 32),
                    umma_desc_k_sw128(q_at + (piece * kBlk + b) * (kNS * 128) + k * 32), idesc_s[Pc::q_e5(piece)], c > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[next_s & 1]);
          umma_commit(&kv_empty[ks]);
          ks += 2;
          if (ks >= ns) { ks -= ns; kph ^= 1; }
          ++next_s;
          if (++s_in == ws.count) {
            s_in = 0;
            ++s_item;
            ws.next();
          }
          progressed = true;
        }
        if (next_pv < next_s && mbar_try_wait(&p_ready[next_pv & 1], (next_pv >> 1) & 1) && mbar_try_wait(&kv_full[vs], vph)) {
          tc_fence_after_sync();
          const uint32_t v_at = kv_addr + vs * G::kOp, w_at = p_addr + (next_pv & 1) * L::kP;
#pragma unroll
          for (int b = 0; b < kBlk; ++b) {
#pragma unroll
            for (int k = 0; k < 4; ++k)       // 32 rows: four groups of eight, 1024 bytes apart
              umma_f8(tO + b * kNO, umma_desc_mn_sw128(v_at + b * (kM * 128) + k * 4096, 1024, 1024),
                      umma_desc_k_sw128(w_at + k * 32), idesc_o, (p_in > 0 || k > 0) ? 1u : 0u);
          }
          // o_done first: whoever has seen p_free of this tile may rely on o_done having advanced as well
          umma_commit(o_done);
          umma_commit(&kv_empty[vs]);
          umma_commit(&p_free[next_pv & 1]);
          vs += 2;
          if (vs >= ns) { vs -= ns; vph ^= 1; }
          ++next_pv;
          if (++p_in == wp.count) {
            umma_commit(o_final);
            p_in = 0;
            wp.next();
          }
          progressed = true;
        }
        if (progressed) { spins = 0; continue; }
        if (++spins > (1u << 20)) { ab.raise(902); break; }
        if ((spins & 255) == 255 && ab.aborted()) break;
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax, queries, epilogue
    if (p.early_meta) griddep_wait();
    const int wi = warp - 2, tid = wi * 32 + lane, group = wi >> 2, quarter = warp & 3;
    const int row_id = quarter * 32 + lane;          // TMEM lane: row of the tile, output dim
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int row_group = group / L::kKeyGroups, key_of = group % L::kKeyGroups, row_of = row_group * kRowsOf;
    const uint32_t tS = tmem_base + lane_off + key_of * kRows + row_of, tO = tmem_base + 2 * kNS + lane_off + key_of * kRows + row_of;
    const uint32_t inv_g = 65536u / g + 1;           // r / g = r * inv_g >> 16 for r < 16
    const int page_rows = p.block_size / kPack, box_rows = min(kM, page_rows & -page_rows);
    const uint32_t all_boxes = (1u << (kM / box_rows)) - 1;              // 16 boxes at most
    const int my_box = row_id / box_rows;
    // byte `row_id` of the thread's first row of P; 16-byte chunks are swizzled by the row's number, of which the thread's part is below 8
    uint8_t* sW = sP + (key_of * kRows + row_of) * 128 + (row_id & 15);
    const int p_ch = (row_id >> 4) ^ (row_of & 7);

    // ---- queries in pieces: 8 elements a thread and step, lanes of a row next to one another
    constexpr int kLanes = D / 8, kQSteps = (NR * kLanes + kSoft - 1) / kSoft;
    uint4 raw[kQSteps];
    auto q_load = [&](const Walk& w, const Request& r) {
#pragma unroll
      for (int i = 0; i < kQSteps; ++i) {
        const int x = i * kSoft + tid, row = x / kLanes;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (row < r.q_len * g) {
          const int tok = (row * inv_g) >> 16;
          raw[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + (r.qs + tok) * p.q_stride +
                                                   (int64_t)(w.head * g + row - tok * g) * D + x % kLanes * 8);
        }
      }
    };
    auto q_store = [&](int item) {
#pragma unroll
      for (int i = 0; i < kQSteps; ++i) {
        const int x = i * kSoft + tid, row = x / kLanes, d = x % kLanes * 8;
        const Vec16<T> a = *reinterpret_cast<const Vec16<T>*>(&raw[i]);
        float v[8], amax = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = to_f(a.v[j]);
          amax = fabsf(v[j]) <= 8.5e37f ? fmaxf(amax, fabsf(v[j])) : INFINITY;
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        // infinities, NaN, and what is too large for its scale to be a number: NaN
        const bool bad = amax == INFINITY;
        const float top = bad ? 1.f : pow2_ceil(fmaxf(amax, 1e-30f)), up = Pc::kTop * pow2_inv(top);
        if (row >= NR) continue;       // whole warps, or the same lanes of every exchange above
        if (d == 0) sFactor[(item & 1) * kRows + row] = bad ? __uint_as_float(0x7fffffffu) : top * (1.f / Pc::kTop) * p.scale_log2;
        __half2 rest[4];               // fp16 holds numbers up to kTop
#pragma unroll
        for (int j = 0; j < 4; ++j) rest[j] = bad ? __float2half2_rn(0.f) : __floats2half2_rn(v[2 * j] * up, v[2 * j + 1] * up);
#pragma unroll
        for (int c = 0; c < P; ++c) {
          uint16_t e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            e[j] = Pc::q_e5(c) ? f16x2_to_e5m2x2(rest[j]) : f16x2_to_e4m3x2(rest[j]);
            if (c + 1 < P) rest[j] = __hsub2(rest[j], as_half2(Pc::q_e5(c) ? e5m2x2_to_f16x2(e[j]) : e4m3x2_to_f16x2(e[j])));
          }
          const uint2 w = make_uint2(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16);
#pragma unroll
          for (int q2 = 0; q2 < kPack; ++q2) {
            const int rr = q2 * kRows + row, byte = kPack == 2 ? q2 * 64 + d : d & 127;
            *reinterpret_cast<uint2*>(sQ + ((c * kBlk + (kBlk == 2 ? d >> 7 : 0)) * kNS + rr) * 128 + (((byte >> 4) ^ (rr & 7)) << 4) +
                                      (byte & 15)) = w;
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    };

    auto out_row = [&](int qs, int head0, int row) {
      const int tok = (int)((row * inv_g) >> 16);
      return ((int64_t)(qs + tok) * p.Hq + head0 + (row - tok * g)) * D + row_id;
    };
    int t = 0;                                       // tiles so far
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true, fail = false;
    Request r = {};
    if (it.more()) {
      r = request_of<D>(p, it.req);
      q_load(it, r);
      q_store(0);
    }
    if (tid < 2) sPend[tid * 8 + 7] = 0;             // no cut item yet
    named_bar_sync(1, kSoft);                        // factors
#pragma unroll 1
    for (int item = 0; it.more(); ++item) {
      const int rows = r.q_len * g, pos_max = r.ctx + r.q_len - 1;
      // weights are 2^(score + base) * v_scale, base = kLift - the reference maximum; rows of `unset` have seen no score yet
      float base[kRowsOf], l_part[kRowsOf];
      uint32_t unset = (1u << kRowsOf) - 1;
#pragma unroll
      for (int i = 0; i < kRowsOf; ++i) { base[i] = kLift; l_part[i] = 0.f; }
      const float* factor = sFactor + (item & 1) * kRows + row_of;
      const Walk cur = it;
      const Request rc = r;
      it.next();
      if (it.more()) {
        r = request_of<D>(p, it.req);
        q_load(it, r);                       // on their way while this item is worked on
      }
      const int tile_end = cur.tile + cur.count;
      bool unset_any = true;
#pragma unroll 1
      for (int i = cur.tile; ok && i < tile_end; ++i, ++t) {
        const int buf = t & 1;
        const int kslot = slot, vslot = slot + 1 == ns ? 0 : slot + 1;
        const uint32_t vphase = slot + 1 == ns ? phase ^ 1 : phase;
        if (!fail && !wait_or_abort(&s_full[buf], (t >> 1) & 1, ab, 905)) fail = true;
        // weight buffer t & 1 is free (P.V of tile t - 2).  Waiting here, before a possible rescale, also keeps o_done at most one phase
        // behind, so that the parity wait on it below cannot pass two phases early.
        if (t >= 2 && !fail && !wait_or_abort(&p_free[buf], ((t >> 1) - 1) & 1, ab, 906)) fail = true;
        if (!fail && !wait_or_abort(&kv_full[kslot], phase, ab, 904)) fail = true;
        if (!fail && !wait_or_abort(&kv_full[vslot], vphase, ab, 904)) fail = true;
        slot += 2;
        if (slot >= ns) { slot -= ns; phase ^= 1; }
        tc_fence_after_sync();
        uint32_t sr[kRowsOf];
        tmem_ld_rows(tS + buf * kNS, sr);
        float kscale = sScale[kslot * kKeys + row_id * kPack + key_of], vscale = sScale[vslot * kKeys + row_id * kPack + key_of];
        const uint32_t valid = sValid[kslot];
        float fac[kRowsOf];
#pragma unroll
        for (int n = 0; n < kRowsOf; n += 4) *reinterpret_cast<float4*>(fac + n) = *reinterpret_cast<const float4*>(factor + n);
        tmem_ld_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s_empty[buf]);
          mbar_arrive(&kv_empty[kslot]);
          mbar_arrive(&kv_empty[vslot]);
        }
        const int key0 = rc.kv_begin + i * kKeys;
        const bool whole = key0 + kKeys <= rc.seq_len && (valid & all_boxes) == all_boxes;
        const bool full = whole && key0 + kKeys - 1 <= rc.ctx && (p.window <= 0 || key0 > pos_max - p.window);
        float y[kRowsOf];                    // log2 of the weights without the values' scale
        bool need = fail || unset_any;
        if (is_nan_bits(vscale)) {           // the row's key gives NaN to those who see it, then, and the value nothing to the others
          kscale = vscale;
          vscale = 0.f;
        }
        if (full) {
          // rows behind the request's have queries of zeros and go along
#pragma unroll
          for (int n = 0; n < kRowsOf; ++n) y[n] = fmaf(__uint_as_float(sr[n]), kscale * fac[n], base[n]);
        } else {
          const int key = key0 + row_id * kPack + key_of;
          const bool there = whole || (key < rc.seq_len && (valid >> my_box & 1));
          if (!there) {
            vscale = 0.f;
            // codes of rows that were not read, or not written, may be anything: zeros, since a weight of zero does not hide a NaN
            uint8_t* v = smem + vslot * G::kOp + row_id * 128;
#pragma unroll
            for (int c = 0; c < 8 / kPack; ++c) {
#pragma unroll
              for (int b = 0; b < kBlk; ++b)
                *reinterpret_cast<uint4*>(v + b * (kM * 128) + (((kPack == 2 ? key_of * 4 + c : c) ^ (row_id & 7)) << 4)) =
                    make_uint4(0, 0, 0, 0);
            }
          }
#pragma unroll
          for (int n = 0; n < kRowsOf; ++n) {
            const int row = row_of + n, pos = row < rows ? rc.ctx + (int)((row * inv_g) >> 16) : -1;
            const bool seen = there && key <= pos && (p.window <= 0 || key > pos - p.window);
            y[n] = seen ? fmaf(__uint_as_float(sr[n]), kscale * fac[n], base[n]) : -INFINITY;
          }
        }
        // log2 of the scale, a power of two; 2^-15 is the smallest that is written
        const float lv = fmaxf((float)((int)(__float_as_uint(vscale) >> 23) - 127), -15.f), limit = kLift + kSlack - lv;
#pragma unroll
        for (int n = 0; n < kRowsOf; ++n) need |= y[n] > limit;
        if (bar_red_or(1, kSoft, need)) {
          // ---- rare after the first tiles: move the reference maxima, rescale O^T
#pragma unroll
          for (int n = 0; n < kRowsOf; ++n) {
            const float wm = warp_max_redux(y[n] + lv);
            if (lane == n) sMax[wi * 8 + n] = wm;
          }
          const bool warp_failed = __any_sync(0xffffffffu, fail);
          if (lane == 0) ok_slot[wi] = warp_failed ? 0 : 1;
          named_bar_sync(1, kSoft);
          bool all_ok = true;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) all_ok &= ok_slot[w] != 0;
          if (!all_ok) { ok = false; break; }
          float alpha[kRowsOf];
          bool rescale = false;
#pragma unroll
          for (int n = 0; n < kRowsOf; ++n) {
            // a group's rows, and the same rows' other keys next to it
            const float* mx = sMax + row_group * L::kKeyGroups * 4 * 8 + n;
            float top = fmaxf(fmaxf(mx[0], mx[8]), fmaxf(mx[16], mx[24]));
            if (L::kKeyGroups == 2) top = fmaxf(top, fmaxf(fmaxf(mx[32], mx[40]), fmaxf(mx[48], mx[56])));
            alpha[n] = 1.f;
            const bool first = unset >> n & 1;
            if (top > kLift + kSlack || (first && top > -INFINITY)) {
              alpha[n] = first ? 0.f : exp2f(kLift - top);       // nothing was added yet
              base[n] -= top - kLift;
              y[n] -= top - kLift;
              l_part[n] *= alpha[n];
              unset &= ~(1u << n);
              rescale = true;
            }
          }
          unset_any = (unset & (rows - row_of >= kRowsOf ? ~0u : (1u << max(0, rows - row_of)) - 1)) != 0;
          // every group has its own columns; the waits of its threads agree because they read the same maxima
          if (rescale && i > cur.tile) {
            if (!wait_or_abort(o_done, (t - 1) & 1, ab, 908)) fail = true;
            __syncwarp();
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < kBlk * W; ++c) {
              const uint32_t at = tO + c / W * kNO + c % W * kPack * kRows;
              uint32_t o[kRowsOf];
              tmem_ld_rows(at, o);
              tmem_ld_wait();
#pragma unroll
              for (int n = 0; n < kRowsOf; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * alpha[n]);
              tmem_st_rows(at, o);
            }
            tmem_st_wait();
          }
          named_bar_sync(1, kSoft);          // sMax has been read
        }
        if (!fail) {
          uint8_t* wbuf = sW + buf * L::kP;
#pragma unroll
          for (int n = 0; n < kRowsOf; n += 2) {
            const float x0 = fast_exp2(y[n]), x1 = fast_exp2(y[n + 1]);
            l_part[n] += x0;
            l_part[n + 1] += x1;
            __half2 rest = __floats2half2_rn(x0 * vscale, x1 * vscale);
#pragma unroll
            for (int c = 0; c < W; ++c) {
              const uint16_t code = Pc::kE5 ? f16x2_to_e5m2x2(rest) : f16x2_to_e4m3x2(rest);
              wbuf[(c * kPack * kRows + n) * 128 + ((p_ch ^ n) << 4)] = (uint8_t)code;
              wbuf[(c * kPack * kRows + n + 1) * 128 + ((p_ch ^ (n + 1)) << 4)] = (uint8_t)(code >> 8);
              if (c + 1 < W) {
                const uint32_t wide = Pc::kE5 ? e5m2x2_to_f16x2(code) : e4m3x2_to_f16x2(code);
                rest = __hmul2(__hsub2(rest, as_half2(wide)), __float2half2_rn(Pc::kStep));
              }
            }
          }
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        const bool warp_failed = __any_sync(0xffffffffu, fail);
        __syncwarp();
        if (lane == 0 && !warp_failed) mbar_arrive(&p_ready[buf]);
      }
      if (fail) ok = false;
      // ---- the next item's queries, so that its first product runs while this one ends: every S of this item has been read
      if (it.more()) q_store(item + 1);
      // ---- row sums
#pragma unroll
      for (int n = 0; n < kRowsOf; ++n) {
        float v = l_part[n];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == n) {
          sSum[wi * 8 + n] = v;
          sMax[wi * 8 + n] = base[n];
        }
      }
      const int first = sPre[cur.req] * p.Hkv + cur.head * cur.n;
      // the CTAs that have tiles of this item: its cuts lie more than `snap` from its ends
      const int c0 = (first + snap) / share, c1 = cur.n > 2 * snap + 1 ? (first + cur.n - snap - 1) / share : 0;
      const bool partial = c0 < c1;
      const int64_t my_slot = 2 * (int64_t)blockIdx.x + ((int)blockIdx.x == c0 ? 1 : 0);
      if (ok && !wait_or_abort(o_final, item & 1, ab, 907)) ok = false;
      ok = bar_red_or(1, kSoft, !ok) == 0;   // one thread's time-out ends the work of all
      tc_fence_after_sync();
      if (tid < NR) {
        const int w0 = tid / kRowsOf * L::kKeyGroups * 4, n = tid % kRowsOf;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4 * L::kKeyGroups; ++w) sum += sSum[(w0 + w) * 8 + n];
        const float lift = sMax[w0 * 8 + n];
        float den = sum;
        if (!partial && p.sinks != nullptr && tid < rows)
          den += exp2f(p.sinks[cur.head * g + ((int)tid - (int)((tid * inv_g) >> 16) * g)] * kLog2e + lift);
        // a row that saw nothing gives zeros, a NaN stays one
        sInv[tid] = !ok || den == 0.f ? 0.f : 1.f / den;
        if (partial) p.ws_lse[my_slot * kRows + tid] = !ok || sum == 0.f ? -INFINITY : log2f(sum) - lift;
      }
      named_bar_sync(1, kSoft);
      // this thread's output dims of its rows: pieces summed; heads of 64: even keys' in lanes 0 .. 63, odd ones' behind
      constexpr bool kBoth = kPack == 2 && L::kKeyGroups == 1;
      const bool reads = L::kKeyGroups == 1 || (row_id >> 6) == key_of;
      float o_mine[kBlk][kRowsOf];
#pragma unroll
      for (int b = 0; b < kBlk; ++b) {
#pragma unroll
        for (int n = 0; n < kRowsOf; ++n) o_mine[b][n] = 0.f;
        if (!ok) continue;
#pragma unroll
        for (int c = 0; c < W; ++c) {
          const uint32_t at = tO + b * kNO + (c * kPack + (kBoth ? row_id >> 6 : 0)) * kRows;
          uint32_t o[kRowsOf];
          tmem_ld_rows(at, o);
          tmem_ld_wait();
          const float unit = c == 0 ? 1.f : c == 1 ? 1.f / Pc::kStep : 1.f / (Pc::kStep * Pc::kStep);
#pragma unroll
          for (int n = 0; n < kRowsOf; ++n) o_mine[b][n] += __uint_as_float(o[n]) * unit;
        }
      }
      if constexpr (kPack == 2) {
        if (row_id >= 64 && reads) {
#pragma unroll
          for (int n = 0; n < kRowsOf; ++n) sHalf[(row_of + n) * 64 + row_id - 64] = o_mine[0][n];
        }
        named_bar_sync(1, kSoft);
        if (row_id < 64 && reads) {
#pragma unroll
          for (int n = 0; n < kRowsOf; ++n) o_mine[0][n] += sHalf[(row_of + n) * 64 + row_id];
        }
      }
      const bool writes = (kPack == 1 || row_id < 64) && reads;
      if (writes) {
#pragma unroll
        for (int n = 0; n < kRowsOf; ++n) {
          const int row = row_of + n;
          const float inv = sInv[row];
          if (row < rows) {
#pragma unroll
            for (int b = 0; b < kBlk; ++b) {
              const float v = inv == 0.f ? 0.f : o_mine[b][n] * inv;
              if (partial) p.ws_o[(my_slot * kRows + row) * D + b * 128 + row_id] = v;
              else reinterpret_cast<T*>(p.out)[out_row(rc.qs, cur.head * g, row) + b * 128] = from_f<T>(v);
            }
          }
        }
      }
      if (partial && tid == 0) {
        int* pend = sPend + (item == 0 ? 0 : 8);      // the first and the last item of a CTA at most
        pend[0] = cur.req * p.Hkv + cur.head;
        pend[1] = c0;
        pend[2] = c1;
        pend[3] = rows;
        pend[4] = rc.qs;
        pend[5] = cur.head * g;
        pend[7] = 1;
      }
      named_bar_sync(1, kSoft);                        // the exchange buffers are free for the next item
    }
    // ---- the last CTA of an item to arrive merges.  The barrier has ordered everyone's stores in front of these threads' releases.
    if (tid < 64 && lane == 0) {
      const bool mine = sPend[tid == 0 ? 7 : 15] != 0;
      int last = 0;
      if (mine) {
        const int* pend = sPend + (tid == 0 ? 0 : 8);
        int seen;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(seen) : "l"(p.tickets + pend[0]) : "memory");
        last = seen == pend[2] - pend[1];
      }
      s_last[tid >> 5] = last;
    }
    named_bar_sync(1, kSoft);
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      if (s_last[k] == 0) continue;
      const int* pend = sPend + k * 8;
      const int c0 = pend[1], n_parts = pend[2] - c0 + 1, rows = pend[3], qs = pend[4], head0 = pend[5];
      const bool writes = (kPack == 1 || row_id < 64) && (L::kKeyGroups == 1 || (row_id >> 6) == key_of);
        // every thread its dims: a few parts' log-sum-exps and results at a time, all in flight, joined in the order of the parts
        
        constexpr int kAtOnce = kRowsOf * kBlk > 8 || L::kGroups > 1 ? 2 : 4;
        float acc[kBlk][kRowsOf], M[kRowsOf], S[kRowsOf];
#pragma unroll
        for (int n = 0; n < kRowsOf; ++n) {
          M[n] = -INFINITY;
          S[n] = 0.f;
#pragma unroll
          for (int b = 0; b < kBlk; ++b) acc[b][n] = 0.f;
        }
        if (writes) {
#pragma unroll 1
          for (int base = 0; base < n_parts; base += kAtOnce) {
            float l[kAtOnce][kRowsOf], v[kAtOnce][kBlk][kRowsOf];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
              const int c = c0 + min(base + u, n_parts - 1);
              const int64_t at = (2 * (int64_t)c + (c == c0 ? 1 : 0)) * kRows + row_of;
#pragma unroll
              for (int n = 0; n < kRowsOf; ++n) {
                const bool in = row_of + n < rows && base + u < n_parts;
                l[u][n] = in ? __ldcg(p.ws_lse + at + n) : -INFINITY;
#pragma unroll
                for (int b = 0; b < kBlk; ++b) v[u][b][n] = in ? __ldcg(p.ws_o + (at + n) * D + b * 128 + row_id) : 0.f;
              }
            }
#pragma unroll
            for (int n = 0; n < kRowsOf; ++n) {
              float top = M[n];
#pragma unroll
              for (int u = 0; u < kAtOnce; ++u) top = fmaxf(top, l[u][n]);
              const float ts = top == -INFINITY ? 0.f : top, old = exp2f(M[n] - ts);
              M[n] = top;
              S[n] *= old;
#pragma unroll
              for (int b = 0; b < kBlk; ++b) acc[b][n] *= old;
#pragma unroll
              for (int u = 0; u < kAtOnce; ++u) {
                const float w = exp2f(l[u][n] - ts);       // a NaN stays one; an empty part weighs nothing, and its result is zeros
                S[n] += w;
#pragma unroll
                for (int b = 0; b < kBlk; ++b) acc[b][n] += v[u][b][n] * w;
              }
            }
          }
#pragma unroll
          for (int n = 0; n < kRowsOf; ++n) {
            const int row = row_of + n;
            if (row >= rows) continue;
            if (p.sinks != nullptr)
              S[n] += exp2f(p.sinks[head0 + (row - (int)((row * inv_g) >> 16) * g)] * kLog2e - (M[n] == -INFINITY ? 0.f : M[n]));
            const float inv = S[n] == 0.f ? 0.f : 1.f / S[n];
#pragma unroll
            for (int b = 0; b < kBlk; ++b) reinterpret_cast<T*>(p.out)[out_row(qs, head0, row) + b * 128] = from_f<T>(acc[b][n] * inv);
          }
        }
      if (tid == 0) p.tickets[pend[0]] = 0;
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, L::kTmem);
  }
}

template <typename T, int D, int NR>
static int launch_nr(Params p, const CUtensorMap& tm, int64_t units, int num_sms, cudaStream_t st) {
  using L = Layout<T, D, NR>;
  auto kern = kv8_decode_kernel<T, D, NR>;
  // two CTAs an SM where four operand slots each fit, otherwise one with as many as fit
  int ctas = L::kCtas, slots = 6;
  while (slots > 4 && L::smem(slots, p.B) > 113 * 1024) --slots;
  if (ctas == 1 || L::smem(slots, p.B) > 113 * 1024) {
    ctas = 1;
    slots = 10;
    while (slots > 4 && L::smem(slots, p.B) > 226 * 1024) --slots;
  }
  const int grid = (int)(units < (int64_t)num_sms * ctas ? units : (int64_t)num_sms * ctas);
  p.slots = slots;
  const size_t smem = L::smem(slots, p.B);
  cudaError_t e = ensure_dynamic_smem((const void*)kern, (int)smem);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(kern, dim3(grid), dim3(L::kThreads), smem, st, tm, p);
}

template <typename T, int D>
static int launch(const Params& p0, const CUtensorMap& tm, int B, int max_rows, int num_sms, int64_t max_tiles, cudaStream_t st) {
  Params p = p0;
  // tiles are counted in 32 bits
  const int64_t most = 0x7fffffff / ((int64_t)p.Hkv * (p.max_keys / Geo<D>::kKeys + 2));
  if (most < 1) return 3;
  const int step = most < kMaxB ? (int)most : kMaxB;
  for (int b0 = 0; b0 < B; b0 += step) {
    p.B = B - b0 < step ? B - b0 : step;
    p.block_tables = p0.block_tables + (int64_t)b0 * p.bt_stride;
    p.seq_lens = p0.seq_lens + b0;
    p.qsl = p0.qsl + b0;
    p.tickets = p0.tickets + (int64_t)b0 * p.Hkv;
    const int64_t units = (int64_t)p.B * p.Hkv * (max_tiles < 1 ? 1 : max_tiles);
    int rc;
    if (max_rows <= 4) rc = launch_nr<T, D, 4>(p, tm, units, num_sms, st);
    else if (max_rows <= 8) rc = launch_nr<T, D, 8>(p, tm, units, num_sms, st);
    else rc = launch_nr<T, D, 16>(p, tm, units, num_sms, st);
    if (rc != 0) return rc;
  }
  return 0;
}

}  // namespace kv8dec
}  // namespace b200

// `tmap`: the codes as written by b200_encode_tmap_kv8.  ws_o: 2 * 2 * num_sms * 16 * D floats, ws_lse: 2 * 2 * num_sms * 16, tickets: B * Hkv zeros (zeros again on return).
// Requests with more than max_query_len queries are left out.  Returns 3 for shapes it does not serve.
extern "C" int b200_kv8_decode(void* out, const void* q, const void* cache, const void* tmap, const int* block_tables,
                               const int* seq_lens, const int* qsl, const float* sinks, float* ws_o, float* ws_lse, int* tickets,
                               int* status, int B, int Hq, int Hkv, int D, int block_size, int max_blocks, int64_t bt_stride,
                               int64_t num_blocks, int max_query_len, int64_t max_seq_len, int window, float scale, int64_t q_stride,
                               int early_meta, int dtype, int num_sms, cudaStream_t st) {
  using namespace b200;
  if (B == 0) return 0;
  if (Hq % Hkv || max_query_len < 1 || (int64_t)max_query_len * (Hq / Hkv) > kv8dec::kRows || block_size % 16 ||
      (D != 64 && D != 128 && D != 256) || (dtype != kBF16 && dtype != kF16) || num_blocks * 2 * Hkv > 0x7fffffff || q_stride % 8 ||
      (reinterpret_cast<uintptr_t>(q) & 15) || window < 0 || num_sms < 1)
    return 3;
  kv8dec::Params p = {};
  p.q = q; p.out = out; p.cache = static_cast<const uint8_t*>(cache); p.ws_o = ws_o; p.ws_lse = ws_lse; p.tickets = tickets;
  p.block_tables = block_tables; p.seq_lens = seq_lens; p.qsl = qsl; p.sinks = sinks; p.status = status;
  p.num_blocks = num_blocks; p.bt_stride = bt_stride; p.q_stride = q_stride; p.Hq = Hq; p.Hkv = Hkv; p.block_size = block_size;
  p.max_blocks = max_blocks; p.max_keys = (int)((int64_t)max_blocks * block_size < 0x7ffffe00 ? max_blocks * block_size : 0x7ffffe00);
  p.window = window; p.early_meta = early_meta;
  p.scale_log2 = scale * kv8dec::kLog2e;
  const CUtensorMap& tm = *reinterpret_cast<const CUtensorMap*>(tmap);
  const int rows = max_query_len * (Hq / Hkv), keys = D == 64 ? 256 : 128;
  const int64_t span = window > 0 && window + max_query_len < max_seq_len ? window + max_query_len + keys : max_seq_len;
  const int64_t tiles = (span + keys - 1) / keys;
#define B200_KV8_DEC(TT, DD) return kv8dec::launch<TT, DD>(p, tm, B, rows, num_sms, tiles, st)
  if (dtype == kBF16) {
    if (D == 64) B200_KV8_DEC(__nv_bfloat16, 64);
    if (D == 128) B200_KV8_DEC(__nv_bfloat16, 128);
    B200_KV8_DEC(__nv_bfloat16, 256);
  }
  if (D == 64) B200_KV8_DEC(__half, 64);
  if (D == 128) B200_KV8_DEC(__half, 128);
  B200_KV8_DEC(__half, 256);
#undef B200_KV8_DEC
}
