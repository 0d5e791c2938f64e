// Prompt and chunk attention over the 8-bit paged cache (common/kv8.cuh) on tcgen05 + TMEM, fed by TMA from the pages: heads of 64 and
// 128, any number of query tokens.
//
// The products are 16-bit: per 128-key tile and 128-row query tile
//     S[128 rows, 128 keys]  = Q . K_tile^T          in the queries' type (bf16 or fp16)
//     O[128 rows, D dims]   += P[128 rows, 128 keys] . V    in fp16, P in TMEM over the columns of S
// Four warps turn codes into operands between the TMA's buffer and the tensor core's: every stored value is an exact bf16 and fp16 number
// (common/kv8.cuh), so nothing is lost, scales are gone before the products, and V and P in fp16 round weights to 11 bits.  Products in e4m3
// would not be faster: queries and weights need two pieces each, twice the work at twice the rate.
// What bounds it: per tile the tensor core needs 1024 cycles (2 x 128^3 products), the special-function units as many (128 x 128
// exponentials at 16 a cycle); conversion is 2 x 128 x 128 values per two tiles.
//
// A row is (token, head of a group): a tile holds 128 / g tokens of all g heads of one key / value head, so that a few new tokens fill it,
// and K and V are read and converted once for the group.  A persistent CTA works on two tiles ("streams") of consecutive tokens that read
// the same K / V tiles; the tensor core works on one while the other is in its softmax.  A stream's products are issued in the order
// P.V(i), S(i + 1), so the arrival of S(i + 1) also says that O holds P.V(i).  With few tiles behind a long context the keys of an item are
// split over CTAs, whose normalised partial results a second kernel joins.
// 512 threads: warp 0 TMA producer (a lane per 16 keys), warp 1 MMA issuer, warps 4-7 / 8-11 softmax and epilogue of stream 0 / 1 (thread =
// row), warps 12-15 conversion.  The grid has a CTA per item, in descending order of row blocks; a CTA that is done takes the next
// pending one's item (cluster launch control).  Every wait is bounded; on time-out the status word is set and the CTA unwinds.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "../api.h"
#include "../common/kv8.cuh"
#include "../common/launch.cuh"
#include "../common/ptx.cuh"
#include "../gemm/gemm_common.cuh"

namespace b200 {
namespace kv8prompt {

constexpr int kThreads = 4 * 128;
// Registers a thread of the first and the last warpgroup keeps and one of the softmax warpgroups gets: the launch brings 512 x 128 =
// 65536, and the split takes 128 x (64 + 192 + 192 + 64) = 65536.
constexpr int kRegsFew = 64, kRegsSoft = 192;
constexpr int kTile = 128, kPage = 64;
constexpr int kKStages = 2, kVStages = 4, kRaw = 4;      // K tiles, V pages, pages of codes
constexpr int kTmemCols = 512;
constexpr float kMaxSlack = 8.f;
constexpr float kLog2e = 1.4426950408889634f;

template <int D> struct Cfg {
  static constexpr int kB = D / 64;                    // 64-dim blocks
  static constexpr int kBlock = kTile * 128;           // one block of a 128-row operand tile
  static constexpr int kQ = kB * kBlock, kK = kB * kBlock, kV = kB * kPage * 128;
  static constexpr int kCodes = kPage * D;
  static constexpr size_t kSmem = 1024 + 2 * kQ + kKStages * kK + kVStages * kV + kRaw * (kCodes + kPage * 4) + 512;
};

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
  int toks;                 // tokens of a tile
  int single;               // one stream a CTA
  int row_blocks, splits;
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
template <typename T> struct FmtOf;
template <> struct FmtOf<__nv_bfloat16> { static constexpr uint32_t v = 1; };
template <> struct FmtOf<__half> { static constexpr uint32_t v = 0; };
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

// Codes -> 16-bit values times a power of two, exact.
template <typename T> struct Widen;
template <> struct Widen<__half> {
  static __device__ __forceinline__ uint32_t factor(float s) { return pack2<__half>(s, s); }
  static __device__ __forceinline__ void four(uint32_t w, uint32_t f, uint32_t& lo, uint32_t& hi) {
    const uint32_t a = e4m3x2_to_f16x2((uint16_t)w), b = e4m3x2_to_f16x2((uint16_t)(w >> 16));
    const __half2 s = *reinterpret_cast<const __half2*>(&f);
    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&a), s), y = __hmul2(*reinterpret_cast<const __half2*>(&b), s);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
};
// Exponent and mantissa of an e4m3 number four places lower in a bf16 number are its value times 2^-120, below the normal range too.
template <> struct Widen<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t factor(float s) {
    const uint32_t b = __float_as_uint(s * 1.329227995784916e36f);      // 2^120
    return __byte_perm(b, b, 0x3232);
  }
  static __device__ __forceinline__ uint32_t two(uint32_t u, uint32_t f) {
    const uint32_t x = ((u >> 4) & 0x07f007f0u) | (u & 0x80008000u);
    const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&f));
    return *reinterpret_cast<const uint32_t*>(&y);
  }
  static __device__ __forceinline__ void four(uint32_t w, uint32_t f, uint32_t& lo, uint32_t& hi) {
    lo = two(__byte_perm(w, 0, 0x1404), f);
    hi = two(__byte_perm(w, 0, 0x3424), f);
  }
};

// One work item: what the two streams of a CTA share and their own rows.
struct Item {
  int req, qs, q_len, ctx, seq_len, key0, head, split;     // key0: first key of the first tile
  int tok0[2], toks[2], n[2];                              // per stream: first token within the request, tokens, key tiles
  int n_max;
};
// Items are ordered by descending row block, so by descending number of key tiles for prompts of one length.
__device__ __forceinline__ void get_item(const Params& p, int idx, Item& it) {
  const int heads = p.Hkv * p.splits, per = p.B * heads, rb = p.row_blocks - 1 - idx / per, rem = idx % per;
  it.req = rem / heads;
  it.head = rem % heads / p.splits;
  it.split = rem % p.splits;
  it.qs = p.qsl[it.req];
  it.q_len = p.qsl[it.req + 1] - it.qs;
  it.seq_len = p.seq_lens[it.req];
  it.ctx = it.seq_len - it.q_len;
  const int step = p.single ? p.toks : 2 * p.toks;
  int all[2];
  int kv_begin = 0;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    it.tok0[s] = rb * step + s * p.toks;
    it.toks[s] = (s == 1 && p.single) ? 0 : max(0, min(p.toks, it.q_len - it.tok0[s]));
    // a window hides everything in front of the first token's first visible key (whole tiles of it)
    if (s == 0) kv_begin = p.window > 0 ? max(0, it.ctx + it.tok0[0] - p.window + 1) / kTile * kTile : 0;
    // keys visible to the tile end with the position of its last token; rows that see nothing have a tile all the same
    const int kv_end = min(it.seq_len, it.ctx + it.tok0[s] + it.toks[s]);
    all[s] = it.toks[s] > 0 ? max(1, (kv_end - kv_begin + kTile - 1) / kTile) : 0;
  }
  const int each = (max(all[0], all[1]) + p.splits - 1) / p.splits, first = it.split * each;
#pragma unroll
  for (int s = 0; s < 2; ++s) it.n[s] = max(0, min(all[s] - first, each));
  it.key0 = kv_begin + first * kTile;
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

// What a page of codes is, for the conversion warps: bits 0-3 which 16 keys were read, 4-10 keys in front of the request's end, 11 V, 12 the
// end of all work; 16-18 the tile's place in the ring of valid masks (K).
constexpr uint32_t kMetaV = 1u << 11, kMetaEnd = 1u << 12;

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
kv8_prompt_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKV, const __grid_constant__ Params p) {
  using C = Cfg<D>;
  constexpr int kB = C::kB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                  // [2 streams][kB dim blocks][128 rows][128 B]
  uint8_t* sK = sQ + 2 * C::kQ;                        // [kKStages][kB dim blocks][128 keys][128 B]
  uint8_t* sV = sK + kKStages * C::kK;                 // [kVStages][kB dim blocks][64 keys][128 B]
  uint8_t* sRaw = sV + kVStages * C::kV;               // [kRaw][64 keys][D B]
  float* sScale = reinterpret_cast<float*>(sRaw + kRaw * C::kCodes);   // [kRaw][64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sScale + kRaw * kPage);
  uint64_t* q_full = bars;              // one phase per item
  uint64_t* q_empty = bars + 1;         // the item's last S has been computed
  uint64_t* k_full = bars + 2;          // [2] four warps, two pages
  uint64_t* k_empty = bars + 4;         // [2] both streams' S of the tile have been computed
  uint64_t* v_full = bars + 6;          // [4] four warps
  uint64_t* v_empty = bars + 10;        // [4]
  uint64_t* raw_full = bars + 14;       // [4]
  uint64_t* raw_empty = bars + 18;      // [4] four warps
  uint64_t* s_full = bars + 22;         // [2 streams]
  uint64_t* p_ready = bars + 24;        // [2 streams][2 halves] one arrival per softmax warp
  uint64_t* o_final = bars + 28;        // [2 streams] one phase per item with work for the stream
  // answers about the next item: question k uses slot k & 1
  uint64_t* next_full = bars + 30;      // [2]
  uint64_t* next_empty = bars + 32;     // [2] read by the MMA thread and the eight softmax warps
  const uint32_t next_at = smem_u32(bars + 34);   // [2] x 16 bytes
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 38);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* sMeta = tmem_slot + 2;      // [kRaw]
  volatile uint32_t* sValid = sMeta + kRaw;   // [8] which 16 keys of a tile are there

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Abort ab{p.status, abort_flag};
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int b = 0; b < kKStages; ++b) { mbar_init(&k_full[b], 8); mbar_init(&k_empty[b], 1); }
    for (int b = 0; b < kVStages; ++b) { mbar_init(&v_full[b], 4); mbar_init(&v_empty[b], 1); }
    for (int b = 0; b < kRaw; ++b) { mbar_init(&raw_full[b], 1); mbar_init(&raw_empty[b], 4); }
    for (int s = 0; s < 2; ++s) {
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
    const int page_rows = p.block_size * D / 128;                        // rows of 128 bytes of a cache page
    const int R = min(kPage * D / 128, page_rows & -page_rows);          // ... of a box; the host's map agrees
    const int box_keys = R * 128 / D, units = box_keys / 16;
    const int64_t page_bytes = (int64_t)p.block_size * (D + 4);
    int rc = 0, qc = 0, asked = 0, tiles = 0;      // pages and items issued, questions asked, K tiles so far
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
      get_item(p, idx, it);
      const int n_max = it.n_max;
      if (n_max > 0) {
        if (qc > 0 && !wait_all(q_empty, (qc - 1) & 1, 920)) { ok = false; break; }
        if (lane == 0) {
          mbar_expect_tx(q_full, p.toks * p.g * 128 * kB * ((it.n[0] > 0) + (it.n[1] > 0)));
#pragma unroll
          for (int s = 0; s < 2; ++s)
            if (it.n[s] > 0) {
#pragma unroll
              for (int h = 0; h < kB; ++h)
                tma_load_3d(sQ + s * C::kQ + h * C::kBlock, &tmQ, q_full, h * 64, it.head * p.g, it.qs + it.tok0[s]);
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
        // pages of tile j: lanes at the start of a box issue it
        auto load = [&](int j, int blk, bool is_v, int place) {
          const uint32_t valid = __ballot_sync(0xffffffffu, blk >= 0);
          const int key0 = it.key0 + j * kTile;
          const bool issuer = blk >= 0 && lane % units == 0;
          const uint32_t starts = __ballot_sync(0xffffffffu, issuer);
#pragma unroll 1
          for (int pg = 0; pg < 2; ++pg) {
            const int st = rc % kRaw;
            if (rc >= kRaw && !wait_all(&raw_empty[st], (rc / kRaw - 1) & 1, 921)) return false;
            if (lane == 0) {
              const int left = max(0, min(kPage, it.seq_len - key0 - pg * kPage));
              sMeta[st] = (valid >> (4 * pg) & 15u) | (uint32_t)left << 4 | (is_v ? kMetaV : 0u) | (uint32_t)place << 16;
              mbar_expect_tx(&raw_full[st], __popc(starts >> (4 * pg) & 15u) * (R * 128 + box_keys * 4));
            }
            __syncwarp();
            if (issuer && lane >> 2 == pg) {
              const int in = (key0 + lane * 16) % p.block_size, at = (lane & 3) * 16;      // key within its block, within the page
              const int64_t page = ((int64_t)blk * 2 + is_v) * p.Hkv + it.head;
              tma_load_3d(sRaw + st * C::kCodes + at * D, &tmKV, &raw_full[st], 0, in * D / 128, (int)page);
              bulk_load_1d(sScale + st * kPage + at, p.cache + page * page_bytes + (int64_t)p.block_size * D + in * 4, box_keys * 4,
                           &raw_full[st]);
            }
            ++rc;
          }
          return true;
        };
        int blk = lookup(0), blk_v = -1;
        for (int j = 0; ok && j <= n_max; ++j) {      // K(0), K(1), V(0), K(2), V(1), ...
          if (j == n_max - 1 && p.take && !ask()) { ok = false; break; }
          const int after = lookup(j + 1);
          if (j < n_max) ok = load(j, blk, false, (tiles + j) & 7);
          if (ok && j >= 1) ok = load(j - 1, blk_v, true, 0);
          blk_v = blk;
          blk = after;
        }
        tiles += n_max;
      } else if (p.take) {
        ok = ask();
      }
      if (!p.take || !ok) break;
      if (!wait_all(&next_full[(asked - 1) & 1], ((asked - 1) >> 1) & 1, 929)) { ok = false; break; }
      idx = taken_cta(next_at + 16 * ((asked - 1) & 1));
      fence_proxy_async_smem();
      __syncwarp();
    }
    if (ok) {          // the conversion warps' end
      const int st = rc % kRaw;
      if (rc >= kRaw) ok = wait_all(&raw_empty[st], (rc / kRaw - 1) & 1, 921);
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
      for (int i = max(0, rc - kRaw); i < rc; ++i) drain(&raw_full[i % kRaw], (i / kRaw) & 1);
      if (asked > 0) drain(&next_full[(asked - 1) & 1], ((asked - 1) >> 1) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc(kTile, kTile, FmtOf<T>::v, FmtOf<T>::v, 0, 0);   // A = Q, B = K tile, both K-major
      constexpr uint32_t idesc_o = umma_idesc(kTile, D, 0, 0, 0, 1);       // A = P (TMEM), B = V tile (MN-major), fp16
      int kc = 0, vc = 0, qc = 0, tc[2] = {0, 0};   // consumed so far; tc: tiles of each stream whose P has been awaited
      bool ok = true;
      for (int idx = blockIdx.x, round = 0; idx >= 0; idx = ok ? next_item(round++, false, ok) : -1) {
        get_item(p, idx, it);
        if (it.n_max == 0) continue;
        const int n_max = it.n_max;
        // S of tile j of the item; the last reader of a K stage (of Q) gives it back
        auto issue_s = [&](int s, int j) {
          const uint32_t q_addr = smem_u32(sQ + s * C::kQ), k_addr = smem_u32(sK + ((kc + j) % kKStages) * C::kK);
#pragma unroll
          for (int k = 0; k < kB * 4; ++k)
            umma_f16(tmem_base + s * kTile, umma_desc_k_sw128(q_addr + (k / 4) * C::kBlock + (k % 4) * 32),
                     umma_desc_k_sw128(k_addr + (k / 4) * C::kBlock + (k % 4) * 32), idesc_s, k > 0 ? 1u : 0u);
          umma_commit(&s_full[s]);
          const bool last = s == 1 || j >= it.n[1];
          if (last) {
            umma_commit(&k_empty[(kc + j) % kKStages]);
            if (j == n_max - 1) umma_commit(q_empty);
          }
        };
        ok = wait_or_abort(q_full, qc & 1, ab, 923) && wait_or_abort(&k_full[kc % kKStages], (kc / kKStages) & 1, ab, 924);
        if (!ok) break;
        ++qc;
        tc_fence_after_sync();
        if (it.n[0] > 0) issue_s(0, 0);
        if (it.n[1] > 0) issue_s(1, 0);
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
    // ------------------------------------------------------------------ conversion: 16 codes a thread and step
    const int w = warp - 12;
    int kp = 0, vp = 0;       // pages of K and V so far
    for (int n = 0;; ++n) {
      const int st = n % kRaw;
      if (__any_sync(0xffffffffu, !wait_or_abort(&raw_full[st], (n / kRaw) & 1, ab, 931))) break;
      const uint32_t meta = sMeta[st];
      if (meta & kMetaEnd) break;
      const bool is_v = (meta & kMetaV) != 0;
      const uint8_t* src = sRaw + st * C::kCodes;
      const float* scale = sScale + st * kPage;
      uint8_t* dst;
      int block_bytes;
      uint64_t* full;
      if (is_v) {
        const int s = vp % kVStages;
        if (vp >= kVStages && __any_sync(0xffffffffu, !wait_or_abort(&v_empty[s], (vp / kVStages - 1) & 1, ab, 932))) break;
        dst = sV + s * C::kV;
        block_bytes = kPage * 128;
        full = &v_full[s];
        ++vp;
      } else {
        const int tile = kp >> 1, s = tile % kKStages;
        if (tile >= kKStages && __any_sync(0xffffffffu, !wait_or_abort(&k_empty[s], (tile / kKStages - 1) & 1, ab, 933))) break;
        dst = sK + s * C::kK + (kp & 1) * (kPage * 128);
        block_bytes = C::kBlock;
        full = &k_full[s];
        if (w == 0 && lane == 0) {       // this half's bits; the first half clears the other's
          const int at = meta >> 16 & 7;
          sValid[at] = (kp & 1) ? sValid[at] | (meta & 15u) << 4 : meta & 15u;
        }
        ++kp;
      }
      const int left = meta >> 4 & 127;
      // A warp takes 16 keys.  Eight lanes together must meet eight different 16-byte places of a 128-byte line, when they read (place =
      // chunk ^ row % 8) and when they write (two chunks of eight values, places of one parity for a row): the lower four take the lower
      // half of a row's codes, the upper four the upper half of the next row's, and the other halves a step later.  Heads of 64: a row of
      // codes is two keys, and its halves are keys of different parity anyway.
#pragma unroll
      for (int i = 0; i < 16 * D / 512; ++i) {
        int key, src_row, chunk, dim;     // chunk: 16 codes of the source row; dim: first dim
        if constexpr (D == 128) {
          const int sub = (lane >> 2 & 1) ^ (i & 1);
          key = w * 16 + (i >> 1) * 8 + (lane >> 2);
          src_row = key;
          chunk = (lane & 3) + 4 * sub;
          dim = chunk * 16;
        } else {
          src_row = w * 8 + i * 4 + (lane >> 3);
          chunk = lane & 7;
          key = 2 * src_row + (chunk >> 2);
          dim = (chunk & 3) * 16;
        }
        const uint4 c = *reinterpret_cast<const uint4*>(src + src_row * 128 + ((chunk ^ (src_row & 7)) << 4));
        const float s = scale[key];
        const uint32_t x[4] = {c.x, c.y, c.z, c.w};
        uint32_t y[8];
        if (is_v) {
          // rows that were not read, lie behind the end or hold a NaN (whose key says so): zeros, since a weight of zero does not hide one
          const bool there = key < left && (meta >> (key >> 4) & 1u) && !is_nan_bits(s);
          const uint32_t f = Widen<__half>::factor(s);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            Widen<__half>::four(x[q], f, y[2 * q], y[2 * q + 1]);
            y[2 * q] = there ? y[2 * q] : 0u;
            y[2 * q + 1] = there ? y[2 * q + 1] : 0u;
          }
        } else {
          const uint32_t f = Widen<T>::factor(s);
#pragma unroll
          for (int q = 0; q < 4; ++q) Widen<T>::four(x[q], f, y[2 * q], y[2 * q + 1]);
        }
        uint8_t* row = dst + (dim >> 6) * block_bytes + key * 128;
        const int at = (dim & 63) >> 3;
        *reinterpret_cast<uint4*>(row + ((at ^ (key & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<uint4*>(row + (((at + 1) ^ (key & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(full);
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
    const float sc = p.scale_log2;
    int tc = 0, oc = 0, tiles = 0;    // tiles and items of this stream so far, K tiles of all items
    bool fail = false;
    bool ok = true;
    for (int idx = blockIdx.x, round = 0; idx >= 0; idx = next_item(round++, true, ok)) {
      get_item(p, idx, it);
      const int n = s ? it.n[1] : it.n[0], tok0 = s ? it.tok0[1] : it.tok0[0], toks = s ? it.toks[1] : it.toks[0];
      const bool row_ok = r_tok < toks;                // toks <= 128 / g
      const int64_t orow = (int64_t)(it.qs + tok0 + r_tok) * p.Hq + it.head * p.g + r_head;
      if (n == 0) {
        if (p.splits > 1 && row_ok) p.ws_lse[(int64_t)it.split * p.T * p.Hq + orow] = -INFINITY;
        tiles += it.n_max;
        continue;
      }
      const int pos_first = it.ctx + tok0, pos_last = pos_first + toks - 1, pos = pos_first + r_tok;
      float m_used = -INFINITY, l_sum = 0.f;
      for (int i = 0; i < n; ++i, ++tc) {
        if (__any_sync(0xffffffffu, !wait_or_abort(&s_full[s], tc & 1, ab, 927))) { fail = true; break; }
        tc_fence_after_sync();
        const int key0 = it.key0 + i * kTile;
        uint32_t v[kTile];
#pragma unroll
        for (int c = 0; c < kTile; c += 32) tmem_ld_x32_p(tS + c, v + c);
        const uint32_t valid = sValid[(tiles + i) & 7];
        tmem_ld_wait();
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

// Joins the splits of a row: out = sum_s w_s O_s / (sum_s w_s [+ sink]), w_s = 2^(lse_s - max).  A warp per (token, head).
template <typename T, int D>
__global__ void __launch_bounds__(256)
kv8_join_kernel(T* __restrict__ out, const float* __restrict__ ws_o, const float* __restrict__ ws_lse, const float* __restrict__ sinks,
                int64_t rows, int Hq, int splits, const int* __restrict__ qsl, int B) {
  griddep_launch();
  griddep_wait();
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows || row / Hq < qsl[0] || row / Hq >= qsl[B]) return;
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

template <typename T, int D>
static int launch(const Params& p, const CUtensorMap& tmQ, const CUtensorMap& tmKV, int64_t items, cudaStream_t st) {
  auto kern = kv8_prompt_kernel<T, D>;
  cudaError_t e = ensure_dynamic_smem((const void*)kern, (int)Cfg<D>::kSmem);
  if (e != cudaSuccess) return (int)e;
  e = launch_pdl(kern, dim3((unsigned)items), dim3(kThreads), Cfg<D>::kSmem, st, tmQ, tmKV, p);
  if (e != cudaSuccess || p.splits == 1) return (int)e;
  const int64_t rows = p.T * p.Hq;
  return (int)launch_pdl(kv8_join_kernel<T, D>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, (T*)p.out, (const float*)p.ws_o,
                         (const float*)p.ws_lse, p.sinks, rows, p.Hq, p.splits, p.qsl, p.B);
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
