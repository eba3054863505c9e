// kvb_paged_decode_fwd: attention of one new token per request over its blocks of the
// pool, sm_100a.  O = softmax(q K^T s) V with GQA, the 16-token blocks read in place.
//
// What bounds it: K and V are read once for 2 * (query heads per KV head) FLOP per byte
// (16-bit pool), so HBM, up to the widest groups; short rows are latency.  The tensor
// cores run through mma.sync: a tcgen05 tile has at least 64 rows of which a group of 8
// query heads would fill an eighth, its accumulators live in TMEM behind a
// tcgen05.ld, and one thread issues for the CTA; here every warp is its own pipeline
// and needs about a tenth of the issue slots that the loads leave it.
//
// Split: a unit of work is one block of one (request, KV head, head tile).  The units of
// all items, laid end to end, are divided evenly over the warps of one CTA per SM from
// the lengths on the device, so ragged batches balance to a block without the host
// knowing a length.  A warp walks its units alone: lane 0 brings each block's K and V
// by TMA into the warp's ring of stages, several blocks ahead, through the block table;
// no CTA-wide step sits in the loop.  Items that a warp holds whole it writes itself
// (short ones are left whole with one warp or the next, not cut);
// the pieces at its range's ends are joined in shared memory at the CTA's end, and what
// still spans CTAs goes to the workspace, where the CTA that finds all of an item's pieces
// joins them.  Short tables take one CTA per item instead, whose warps split the item (split()
// below says when).
//
// Arithmetic (per block, tokens on the MMA's rows, query heads on its columns):
//   S^T = K Q^T; online softmax down the rows against a maximum that is raised only when
//   a score passes it by 2^8 (float16: 2^4; one vote instead of shuffles); O^T += V^T P^T.
// P is carried in two 16-bit halves (p = hi + lo), so the weights keep 16 bits and the
// result's error is that of its final rounding; the second MMA is free here.
// KIVI int8 pools: a code is exact in float16 (as a subnormal, biased by 128; the bias leaves
// through the accumulators' start), so Q (scaled by a power of two per row) and P's halves are
// float16 and the scales act in float32 on S (K, per token) and on each block's product (V, per
// channel): the dequantised values are never rounded.
//
// Measured (B200, us per call in a CUDA graph, of the measured 6.48 TB/s copy): 64 requests of
// 700 .. 16381 tokens, 32/8 heads, D 128, bfloat16: 203 to 207 (6.3 to 6.4 TB/s, 97 to 99 %); 8 x 4096,
// 16/2 heads: 14.6 (start, joins); int8 4 x 32768, 64/8 heads: 60.3 (4.8 TB/s, 74 %; 56.5 with the
// weights' high halves alone, which under bfloat16 left 2.5 % of the outputs a step off); 24 requests
// of 1 .. 2051 tokens, 32 heads of D 96, float16: 23.1 (3.9 TB/s).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <mutex>
#include <string>
#include <type_traits>

#include "kvb_attn.h"
#include "kvb_sm100_ptx.cuh"

int kvb_detail_fail(int code, const std::string& msg);

namespace kvb_pd {

using namespace kvb::ptx;

int fail(int code, const std::string& msg) { return kvb_detail_fail(code, msg); }

constexpr int kSms = 148;
constexpr uint64_t kWaitNs = 2000000000ull;
// Weights are exp2(x - m) with m kept kLift below the running maximum (log2 units), and m is raised
// when a score passes m by kTop.  In bfloat16, with float32's exponents, that is a maximum raised
// when it is passed by 2^8.  A float16 half has nothing below 2^-25, so there the weights lie as high
// as 2^15 and the maximum's own at 2^11 or above: what is lost lies below 2^-36 of the largest (2^-25
// without the lift: 2000 tokens of weight 2^-26 and V 60000 beside some of weight 1 were all lost).
// Raising at every new maximum instead: int8 4 x 32768 tokens 61.2 us, 60.3 so.
template <typename E> constexpr float kLift = std::is_same<E, __half>::value ? 11.f : 0.f;
template <typename E> constexpr float kTop = std::is_same<E, __half>::value ? 15.f : 8.f;
// Warps per CTA, as registers allow.  Items of up to 8 heads: 64 requests of 700 .. 16381 tokens in
// bfloat16 took 211 us with 8 warps of three stages, 209 with 10, 206 with 12 of two; int8 4 x
// 32768 tokens, 64/8 heads: 68.3 with 10, 60.3 with 12, 66.4 with 14, 65.9 with 16 (which spill).
// D 64 needs fewer registers: 16 warps instead of 12 took 32 x 16384 tokens, 8 KV
// heads, from 6.28 to 6.43 TB/s, 64 x 16384 in int8 from 4.32 to 4.61.  Items of 16 heads hold twice
// the accumulators: 8 warps (10: 5.81 TB/s instead of 5.89), 12 for int8 of D 64 (3.12, with 8 2.65).
constexpr int warps_of(int D, bool i8, int tiles8) {
  return tiles8 == 1 ? (D == 64 ? 16 : 12) : (D == 64 && i8 ? 12 : 8);
}
constexpr int kMostWarps = 16;
// What an item's start and end weigh in the split, in blocks: 24 requests of 1 to 2051 tokens,
// 32 heads of D 96: 24.2 us with 0, 19.6 with 1 and 2.
constexpr int kItemCost = 1;
// Places per CTA below which fewer CTAs share a split (one request of 2000 tokens, 2 KV heads:
// 10.3 us with 8, 9.2 with 16, 12.1 with 32), and the most CTAs per item (the join reads them
// all: one request of 32768 tokens, 1 KV head: 20.3 us on 148 CTAs, 13.7 on 64).
constexpr int kMinUnits = 16;
constexpr int kSpan = 64;
// Most blocks of an item that a share's end does not cut, one warp taking all of it: kShort, more
// where the shares are long enough for the uneven ends not to show (kShort 2 up to four shares,
// uncut_of up to two).  D 128, cut and joined / whole: 640 items of 64 tokens 10.3 us / 7.3, of 256
// 21.6 / 17.3 (8 heads 26.4 / 17.6); 2368 of 64 24.8 / 18.3 (int8 27.5 / 18.6), of 256 63.9 /
// 53.8 (50.5 / 45.7), of 512 104.9 / 99.8 (71.1 / 74.2).  With shares of less than two blocks
// the cut is better: 128 items of 256 tokens 12.8 / 15.7.
constexpr int kShort = 8;
constexpr int uncut_of(bool i8) { return i8 ? 16 : 32; }
constexpr int kSplitRows = 8192;           // most rows of a split launch (prefix sums in shared memory)

struct Args {
  int batch, num_q_heads, num_kv_heads, num_blocks, width;
  int group, tiles, items;                 // tiles: head tiles per KV head; items = kv heads * tiles
  int ctas;                                // split launch: CTAs sharing the units
  float scale_log2;
  const void* q;
  void* o;
  float* lse;
  int64_t q_bs, q_hs, o_bs, o_hs, lse_bs, table_stride;
  const __half* k_scale;
  const __half* v_scale;
  const int32_t* tables;
  const int32_t* lens;
  int32_t* status;
  float* part;                             // [ctas][2][NH * D + 2 * NH]
  float* first;                            // [ctas * warps][PIECE]: pieces that start a warp's range
  uint64_t* flags;                         // [ctas][2][NH]: head's piece is in the workspace
  uint64_t nonce;                          // what this call's flags read
};

// ---- warp-level primitives ------------------------------------------------------------------
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float lds_half(uint32_t addr) {
  uint16_t h;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(addr) : "memory");
  return __half2float(__ushort_as_half(h));
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// One arrival on `bar` once this thread's copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// D (16 x 8, float32) += A (16 x 16) B (16 x 8), both operands in E
template <typename E>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<E, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// D = A B + C in float16
__device__ __forceinline__ void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

template <typename E>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {   // lo in the low half
  if constexpr (std::is_same<E, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename E>
__device__ __forceinline__ float2 unpack(uint32_t u) {
  if constexpr (std::is_same<E, __half>::value) {
    __half2 h;
    memcpy(&h, &u, 4);
    return __half22float2(h);
  } else {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
}

// Two of four int8 codes, biased by 128 to 0 .. 255, as float16: under a zero byte a code is
// (code + 128) * 2^-24, exactly (a subnormal, which the tensor core multiplies as any other);
// the bias leaves through the accumulator's start.
constexpr float kCode = 1.f / 16777216.f;  // 2^-24
__device__ __forceinline__ uint32_t codes_to_half(uint32_t biased, uint32_t select) {
  return __byte_perm(biased, 0u, select);
}

// A warp's wait for a phase; false after 2 s (the status word says so).  The lanes vote at each look, so
// all of them get one verdict: what follows is warp-wide.
__device__ __forceinline__ bool wait_full(uint32_t bar, uint32_t parity, int32_t* status) {
  if (__all_sync(~0u, mbar_try_wait(bar, parity))) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!__all_sync(~0u, mbar_try_wait(bar, parity))) {
    if (__any_sync(~0u, globaltimer_ns() - t0 > kWaitNs)) {
      if (status) atomicOr(status, KVB_STATUS_LOAD_WAIT);
      return false;
    }
  }
  return true;
}

// ---- geometry -------------------------------------------------------------------------------
template <int D, bool I8, int NT>
struct Geo {
  static constexpr int WARPS = warps_of(D, I8, NT);
  static constexpr int UNCUT = uncut_of(I8);
  static constexpr int THREADS = WARPS * 32;
  static constexpr int NH = 8 * NT;                          // query heads per item
  static constexpr int HALVES = I8 ? 1 : (D + 63) / 64;      // TMA boxes per block
  static constexpr int ROW = I8 && D == 64 ? 64 : 128;       // bytes of a box row = its swizzle
  static constexpr int BOX = 2 * 16 * ROW;                   // K and V, 16 tokens
  static constexpr int STAGE = HALVES * BOX;
  static constexpr int SCALES = I8 ? 32 + 256 : 0;           // K then V scales of the block
  static constexpr int OS = D + 4;                           // piece row: conflict-free columns
  static constexpr int PIECE = NH * OS + 2 * NH;             // floats: O rows, maxima, sums
  // alignment, notes, warp sums; per stage: data, scales, barrier
  static constexpr int FIXED = 1024 + WARPS * 2 * 16 + WARPS * 4;
  static constexpr int PER_STAGE = WARPS * (STAGE + SCALES + 8);
  static constexpr int FIT = (232448 - FIXED) / PER_STAGE;
  static constexpr int NS = FIT < 6 ? FIT : 6;               // stages per warp
  static constexpr int SMEM = FIXED + NS * PER_STAGE;
  static constexpr int PART = NH * D + 2 * NH;               // floats of a workspace piece
  static_assert(NS >= 2, "at least two stages per warp");
  static_assert(PIECE * 4 <= NS * STAGE, "a last piece goes over the warp's stages");
  static_assert(WARPS * NS * STAGE >= kSplitRows * 4, "prefix sums go over the stages");
};

// total places over `workers`: worker i's first place, and the worker that holds place u.
struct Shares {
  int q, rem;
  __device__ __forceinline__ Shares(int total, int workers) : q(total / workers), rem(total - q * workers) {}
  __device__ __forceinline__ int first(int i) const { return i * q + min(i, rem); }
  __device__ __forceinline__ int holder(int u) const {
    const int big = rem * (q + 1);
    return u < big ? u / (q + 1) : rem + (u - big) / q;
  }
};

__device__ __forceinline__ int row_len(const Args& a, int b) {
  const int len = a.lens[b];
  return len < 0 ? 0 : (int)min((int64_t)len, (int64_t)a.width * 16);
}

// One item's running state in a warp: maximum (log2), sum and O^T, for NT tiles of 8 heads;
// lane (r, c) = (lane / 4, lane % 4) holds heads 2c, 2c + 1 of each tile.
template <int MT, int NT>
struct State {
  float m[NT][2], l[NT][2], acc[NT][MT][4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[t][j][0] = acc[t][j][1] = acc[t][j][2] = acc[t][j][3] = 0.f;
    }
  }
};

// The largest of the warp's values: a float's bits, the negative ones' turned over, order as
// integers.
__device__ __forceinline__ float warp_max(float x) {
  const int i = __float_as_int(x);
  const int top = __reduce_max_sync(~0u, i < 0 ? i ^ 0x7fffffff : i);
  return __int_as_float(top < 0 ? top ^ 0x7fffffff : top);
}

// ln of the weights' sum: the lift leaves both exactly before the logarithm
template <typename E>
__device__ __forceinline__ float lse_of(float m, float sum) {
  constexpr float unlift = 1.f / (1 << (int)kLift<E>);
  return ((m == -INFINITY ? 0.f : m + kLift<E>) + log2f(sum * unlift)) * 0.6931471805599453f;
}

// Writes a joined head: lane i features 4 i .. 4 i + 3; top, kLift below the maximum, in log2 units.
template <typename T, typename E, int D>
__device__ __forceinline__ void write_head(const Args& a, int b, int head, int lane, const float4& o, float top,
                                           float sum) {
  const float inv = 1.f / sum;
  if (lane < D / 4)
    *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + b * a.o_bs + (int64_t)head * a.o_hs + 4 * lane) =
        make_uint2(pack<T>(o.x * inv, o.y * inv), pack<T>(o.z * inv, o.w * inv));
  if (lane == 0 && a.lse)
    a.lse[b * a.lse_bs + head] = lse_of<E>(top, sum);
}

template <typename T, int D, bool I8, int NT, bool SPLIT>
__global__ void __launch_bounds__(Geo<D, I8, NT>::THREADS, 1)
    kvb_paged_decode_kernel(const __grid_constant__ CUtensorMap map, const Args a) {
  using G = Geo<D, I8, NT>;
  using E = typename std::conditional<I8, __half, T>::type;   // MMA operand type
  constexpr int MT = D / 16, KS = D / 16, NS = G::NS, NH = G::NH;
  constexpr int kWarps = G::WARPS, kThreads = G::THREADS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * NS * G::STAGE;
  uint8_t* scales = smem + kWarps * NS * G::STAGE + warp * NS * G::SCALES;
  uint8_t* after = smem + kWarps * NS * (G::STAGE + G::SCALES);
  int32_t* prefix = reinterpret_cast<int32_t*>(smem);                  // before the first load
  uint64_t* bars = reinterpret_cast<uint64_t*>(after);
  // [kWarps][2] pieces: request (-1: none), item, the item's first and last CTA
  int4* notes = reinterpret_cast<int4*>(bars + kWarps * NS);
  int32_t* wsum = reinterpret_cast<int32_t*>(notes + 2 * kWarps);
  const uint32_t ring_u = smem_u32(ring), scales_u = smem_u32(scales), bar_u = smem_u32(bars + warp * NS);

  if (lane == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(bar_u + 8 * s, I8 ? 33 : 1);
    fence_mbar_init();
    notes[2 * warp].x = notes[2 * warp + 1].x = -1;
    prefetch_tmap(&map);
  }
  __syncwarp();
  griddep_wait();
  griddep_launch_dependents();

  // ---- this warp's units -------------------------------------------------------------------
  int b, j, blk, nb;            // the unit to consume: request, item of the request, block
  int left;                     // what is left of this warp's share
  int u = 0, total = 0;         // split launch: the unit's place among all rows' units
  int ctas = 1;                 // split launch: CTAs that get units
  int uncut = 0;                // split launch: items of up to so many blocks stay whole
  // What is left of a share at an item's first block: an item that the share's end would cut
  // belongs to the warp that has the larger part.
  const auto whole = [&](int left, int nb) {
    return left > 0 && left < nb && nb <= uncut ? (2 * left >= nb ? nb : 0) : left;
  };
  if constexpr (SPLIT) {
    // A row weighs its blocks and kItemCost for each of its items; the weights laid end to end
    // are shared out, so u and left count places, of which an item's first nb are its blocks.
    b = j = blk = nb = 0;
    left = 0;
    const int me = blockIdx.x * kWarps + warp;
    int before = 0, weight = 0, err = 0;
    auto row = [&](int i) {
      const int len = max(a.lens[i], 0), n = (len >> 4) + ((len & 15) != 0);
      if (n > a.width) err = KVB_STATUS_BAD_LENGTH;
      return n ? min(n, a.width) + kItemCost : 0;
    };
    auto scan = [&](int x) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
      }
      return x;
    };
    auto share = [&](int rows_weight) {
      total = rows_weight * a.items;                // below 2^31: the host saw to it
      // no CTA without a block, so an item's CTAs are consecutive
      ctas = min(a.ctas, (total + kMinUnits - 1) / kMinUnits);
      if ((int)blockIdx.x < ctas) {
        const Shares sh(total, ctas * kWarps);
        u = sh.first(me);
        left = sh.first(me + 1) - u;
        uncut = max(max(kShort, min(2 * kShort, 4 * sh.q)), min(G::UNCUT, 2 * sh.q));
      }
    };
    if (a.batch <= 32) {                            // every warp for itself, a row a lane
      const int w = lane < a.batch ? row(lane) : 0, sum = scan(w);
      share(__shfl_sync(~0u, sum, 31));
      const uint32_t past = __ballot_sync(~0u, sum * a.items > u);
      b = past ? __ffs(past) - 1 : 0;
      weight = __shfl_sync(~0u, w, b);
      before = __shfl_sync(~0u, sum, b) - weight;
    } else if (a.batch <= 256) {                    // 8 rows a lane
      int w[8], own = 0;
      const int per = (a.batch + 31) >> 5, from = lane * per;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = i < per && from + i < a.batch ? row(from + i) : 0;
        own += w[i];
      }
      const int sum = scan(own);
      share(__shfl_sync(~0u, sum, 31));
      const uint32_t past = __ballot_sync(~0u, sum * a.items > u);
      const int src = past ? __ffs(past) - 1 : 0;
      int row_b = from;                             // on lane src: its row that holds u
      before = sum - own;
      weight = w[0];
#pragma unroll
      for (int i = 1; i < 8; ++i)
        if (row_b == from + i - 1 && i < per && (before + weight) * a.items <= u) {
          ++row_b;
          before += weight;
          weight = w[i];
        }
      b = __shfl_sync(~0u, row_b, src);
      before = __shfl_sync(~0u, before, src);
      weight = __shfl_sync(~0u, weight, src);
    } else {
      int base = 0;
      for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
        const int i = b0 + tid;
        int x = scan(i < a.batch ? row(i) : 0);
        if (lane == 31) wsum[warp] = x;
        __syncthreads();
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) x += wsum[w];
          sum += wsum[w];
        }
        if (i < a.batch) prefix[i] = base + x;      // inclusive
        base += sum;
        __syncthreads();
      }
      share(base);
      if (left > 0) {
        int lo = 0, hi = a.batch - 1;               // first row whose inclusive sum passes u
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (prefix[mid] * a.items > u) hi = mid; else lo = mid + 1;
        }
        b = lo;
        before = lo ? prefix[lo - 1] : 0;
        weight = prefix[lo] - before;
      }
      fence_proxy_async_smem();                     // the loads go over the sums
      __syncthreads();
    }
    if (err && blockIdx.x == 0 && a.status) atomicOr(a.status, err);
    if (left > 0) {
      const int rel = u - before * a.items;
      j = rel / weight;
      blk = rel - j * weight;
      nb = weight - kItemCost;
      if (blk > 0 && 2 * blk < nb && nb <= uncut) { // the item is this warp's from its start
        u -= blk;
        left += blk;
        blk = 0;
      }
      if (blk >= nb || (blk > 0 && nb <= uncut)) {  // between two items, or the one before's: on to the next
        const int skip = weight - blk;
        blk = 0;
        u += skip;
        left -= skip;
        if (left > 0 && ++j == a.items) {
          j = 0;
          do { nb = (row_len(a, ++b) + 15) >> 4; } while (nb == 0);
        }
      }
      if (blk == 0) left = whole(left, nb);
    }
  } else {
    b = blockIdx.x / a.items;
    j = blockIdx.x - b * a.items;
    nb = (row_len(a, b) + 15) >> 4;
    if (tid == 0 && j == 0 && (int64_t)a.lens[b] > (int64_t)a.width * 16 && a.status)
      atomicOr(a.status, KVB_STATUS_BAD_LENGTH);
    blk = (int)((int64_t)nb * warp / kWarps);
    left = (int)((int64_t)nb * (warp + 1) / kWarps) - blk;
  }

  // ---- producer: this warp's loads, NS units ahead -------------------------------------------
  int pb = b, pj = j, pblk = blk, pnb = nb;
  int to_issue = left;
  int ids = 0, cached_b = -1, cached_c = -1;        // 32 table entries, one per lane
  uint32_t issued = 0, ps = 0;                      // loads issued, the next one's stage
  int pkv = a.tiles == 1 ? pj : pj / a.tiles;       // their KV head
  // lanes 0, 1 copy the K scales, the next D / 8 the V scales: 16 bytes each
  const __half* scale_src = nullptr;
  int64_t scale_step = 0;
  if constexpr (I8) {
    scale_src = lane < 2 ? a.k_scale + 8 * lane : a.v_scale + 8 * (lane - 2);
    scale_step = lane < 2 ? 16 : D;
  }
  auto issue = [&]() {
    const int chunk = pblk >> 5;
    if (pb != cached_b || chunk != cached_c) {
      const int at = chunk * 32 + lane;
      ids = at < pnb ? a.tables[pb * a.table_stride + at] : 0;
      cached_b = pb;
      cached_c = chunk;
    }
    const int id = __shfl_sync(~0u, ids, pblk & 31);
    const uint32_t s = ps, bar = bar_u + 8 * s, dst = ring_u + s * G::STAGE;
    ps = ps + 1 == NS ? 0 : ps + 1;
    const bool ok = (unsigned)id < (unsigned)a.num_blocks;
    if (lane == 0) {
      mbar_arrive_expect_tx(bar, G::STAGE);
#pragma unroll
      for (int h = 0; h < G::HALVES; ++h)
        tma_load_4d(dst + h * G::BOX, &map, h * 64, pkv * 16, 0, ok ? id : -1, bar);
    }
    if constexpr (I8) {
      if (ok && lane < 2 + D / 8)
        copy16(scales_u + s * G::SCALES + 16 * lane,
               scale_src + ((int64_t)id * a.num_kv_heads + pkv) * scale_step);
    }
    if (!ok) {                                      // reads as zeros
      if (I8)
        for (int i = lane; i < G::SCALES / 4; i += 32) sts32(scales_u + s * G::SCALES + 4 * i, 0u);
      __syncwarp();
      if (lane == 0 && a.status) atomicOr(a.status, KVB_STATUS_BAD_BLOCK);
    }
    if constexpr (I8) copies_arrive(bar);
    ++issued;
    to_issue -= ++pblk == pnb ? 1 + (SPLIT ? kItemCost : 0) : 1;
    if (pblk == pnb && to_issue > 0) {
      pblk = 0;
      if (++pj == a.items) {
        pj = 0;
        do { pnb = (row_len(a, ++pb) + 15) >> 4; } while (pnb == 0);
      }
      if constexpr (SPLIT) {
        to_issue = whole(to_issue, pnb);
        if (to_issue == 0) return;
      }
      pkv = a.tiles == 1 ? pj : pj / a.tiles;
      // the item's query heads will be wanted NS blocks from now
      const int h = pkv * a.group + (pj - pkv * a.tiles) * NH + (lane >> 1);
      if ((lane >> 1) < NH && h < (pkv + 1) * a.group)
        prefetch_l2(static_cast<const T*>(a.q) + pb * a.q_bs + h * a.q_hs + (lane & 1) * (D / 2));
    }
  };
  // An item's query heads as the MMA's B operand: for 16-bit pools features 16 ks + 2c, + 8; for
  // int8 pools in the order the K codes are read (lane c's 16-byte pieces c, c + 4; of D 96 its words
  // 4 ks + c), still in T.
  auto load_q = [&](uint32_t (&f)[NT][KS][2], int qb, int qj) {
    const int kv = a.tiles == 1 ? qj : qj / a.tiles, hq = kv * a.group + (qj - kv * a.tiles) * NH;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const bool on = hq + t * 8 + r < (kv + 1) * a.group;
      const T* row = static_cast<const T*>(a.q) + qb * a.q_bs + (int64_t)(on ? hq + t * 8 + r : hq) * a.q_hs;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if constexpr (I8) {
          const int d = D == 96 ? 16 * ks + 4 * c : 16 * (c + 4 * (ks >> 2)) + 4 * (ks & 3);
          const uint2 x = on ? *reinterpret_cast<const uint2*>(row + d) : make_uint2(0u, 0u);
          f[t][ks][0] = x.x;
          f[t][ks][1] = x.y;
        } else {
          f[t][ks][0] = on ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 2 * c) : 0u;
          f[t][ks][1] = on ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 8 + 2 * c) : 0u;
        }
      }
    }
  };
  uint32_t qf[NT][KS][2];
  if (left > 0) load_q(qf, b, j);                   // ahead of the loads that will fill the memory's queues
#pragma unroll 1
  for (int s = 0; s < NS && to_issue > 0; ++s) issue();

  // rows without tokens: zeros and -inf
  if constexpr (SPLIT) {
    for (int z = blockIdx.x; z < a.batch; z += a.ctas)
      if (a.lens[z] <= 0)
        for (int i = tid; i < a.num_q_heads * D; i += kThreads) {
          const int h = i / D, d = i - h * D;
          static_cast<T*>(a.o)[z * a.o_bs + h * a.o_hs + d] = T(0.f);
          if (d == 0 && a.lse) a.lse[z * a.lse_bs + h] = -INFINITY;
        }
  } else if (nb == 0) {
    const int kvh = j / a.tiles, h0 = kvh * a.group + (j - kvh * a.tiles) * NH;
    const int n = min(NH, (kvh + 1) * a.group - h0);
    for (int i = tid; i < n * D; i += kThreads) {
      const int h = h0 + i / D, d = i % D;
      static_cast<T*>(a.o)[b * a.o_bs + h * a.o_hs + d] = T(0.f);
      if (d == 0 && a.lse) a.lse[b * a.lse_bs + h] = -INFINITY;
    }
    return;
  }

  // ---- consumer ----------------------------------------------------------------------------
  constexpr bool AHEAD = NT == 1 && !I8;                   // the next item's heads fit in registers too
  State<MT, NT> st;
  uint32_t qn[NT][KS][2];
  float qx[NT][2];              // what turns S into log2 scores, per head of this lane's columns
  float qb[NT][2];              // int8: -128 * 2^-24 * sum q, the codes' bias in S
  uint32_t used = 0, cs = 0, phase = 0;             // loads consumed, the next one's stage and phase
  bool alive = true, fetched = false;
  while (left > 0 && alive) {
    // one item, or the part of it in this warp's range
    if (SPLIT && blk == 0 && (left = whole(left, nb)) == 0) break;
    const int kvh = a.tiles == 1 ? j : j / a.tiles;
    const int h0 = kvh * a.group + (j - kvh * a.tiles) * NH;
    const int heads = min(NH, (kvh + 1) * a.group - h0);
    const int len = row_len(a, b);
    const int first = blk;
    const int stop = min(nb, blk + left);
    const int past = stop == nb && SPLIT ? kItemCost : 0;
    const bool last = left <= stop - first + past;
    st.clear();
    if constexpr (AHEAD) {
      if (fetched) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[0][ks][0] = qn[0][ks][0], qf[0][ks][1] = qn[0][ks][1];
      }
    } else {
      if (fetched) load_q(qf, b, j);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (!I8) {
        qx[t][0] = qx[t][1] = a.scale_log2;
      } else {
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const float2 x = unpack<T>(qf[t][ks][0]), y = unpack<T>(qf[t][ks][1]);
          top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
        }
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
        // a power of two that brings the row's largest magnitude into [1, 4)
        const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 254);
        const float f = __uint_as_float((uint32_t)max(254 - e, 1) << 23);
        const float inv = __uint_as_float((uint32_t)min(e, 253) << 23);
        float sum = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const float2 x = unpack<T>(qf[t][ks][0]), y = unpack<T>(qf[t][ks][1]);
          qf[t][ks][0] = pack<__half>(x.x * f, x.y * f);
          qf[t][ks][1] = pack<__half>(y.x * f, y.y * f);
          const float2 xr = unpack<__half>(qf[t][ks][0]), yr = unpack<__half>(qf[t][ks][1]);
          sum += (xr.x + xr.y) + (yr.x + yr.y);
        }
        sum += __shfl_xor_sync(~0u, sum, 1);
        sum += __shfl_xor_sync(~0u, sum, 2);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          qx[t][i] = __shfl_sync(~0u, inv, 8 * c + 4 * i) * a.scale_log2 * (1.f / kCode);
          qb[t][i] = __shfl_sync(~0u, sum, 8 * c + 4 * i) * (-128.f * kCode);
        }
      }
    }
    // the item after this one
    int b2 = b, j2 = j + 1, nb2 = nb;

#pragma unroll 1
    for (; blk < stop; ++blk) {
      const uint32_t base = ring_u + cs * G::STAGE, sc = scales_u + cs * G::SCALES;
      if (blk + 1 == stop && !last) {
        if (j2 == a.items) {
          j2 = 0;
          do { nb2 = (row_len(a, ++b2) + 15) >> 4; } while (nb2 == 0);
        }
        if constexpr (AHEAD) load_q(qn, b2, j2);
        fetched = true;
      }
      if (!wait_full(bar_u + 8 * cs, phase, a.status)) {
        alive = false;
        break;
      }
      if (++cs == NS) cs = 0, phase ^= 1;
      const int valid = len - blk * 16;             // >= 1; below 16 in the row's last block
      // S^T: two chains of MMAs
      float sa[NT][2][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sa[t][0][i] = I8 ? qb[t][i & 1] : 0.f, sa[t][1][i] = 0.f;
      if constexpr (!I8) {
        const uint32_t ka = base + ((lane & 7) + ((lane >> 3) & 1) * 8) * 128;
        const uint32_t kx = (((lane >> 4) ^ (lane & 7)) << 4);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t f[4];
          ldsm4(ka + (ks >> 2) * G::BOX + (kx ^ ((ks & 3) << 5)), f);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma<E>(sa[t][ks & 1], f, qf[t][ks][0], qf[t][ks][1]);
        }
      } else {
        auto codes = [&](int ks, uint32_t p, uint32_t v) {   // tokens r and r + 8, four features
          p ^= 0x80808080u;
          v ^= 0x80808080u;
          const uint32_t f[4] = {codes_to_half(p, 0x4140), codes_to_half(v, 0x4140),
                                 codes_to_half(p, 0x4342), codes_to_half(v, 0x4342)};
#pragma unroll
          for (int t = 0; t < NT; ++t) mma<E>(sa[t][ks & 1], f, qf[t][ks][0], qf[t][ks][1]);
        };
        if constexpr (D == 96) {                    // 24 words a row: lane c the words 4 ks + c
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const uint32_t at = base + r * 128 + ((ks ^ (r & 7)) << 4) + 4 * c;
            codes(ks, lds32(at), lds32(at + 8 * 128));
          }
        } else
#pragma unroll
        for (int i = 0; i < KS / 4; ++i) {
          const uint32_t at = G::ROW == 128 ? (((c + 4 * i) ^ (r & 7)) << 4) : ((c ^ ((r >> 1) & 3)) << 4);
          const uint4 x = lds128(base + r * G::ROW + at), y = lds128(base + (r + 8) * G::ROW + at);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) codes(4 * i + w, xs[w], ys[w]);
        }
      }
      // log2 scores: [t][0..1] token r, [2..3] token r + 8; heads 2c, 2c + 1
      float x[NT][4];
      float k0 = 1.f, k1 = 1.f;
      if constexpr (I8) {
        k0 = lds_half(sc + 2 * r);
        k1 = lds_half(sc + 2 * (r + 8));
      }
      bool raise = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = sa[t][0][i] + sa[t][1][i];
          v *= I8 ? qx[t][i & 1] * (i < 2 ? k0 : k1) : qx[t][i & 1];
          if (r + (i < 2 ? 0 : 8) >= valid) v = -INFINITY;
          x[t][i] = v;
          raise |= v > st.m[t][i & 1] + kTop<E>;
        }
      if (__any_sync(~0u, raise)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(x[t][i], x[t][i + 2]);
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
            top = fmaxf(top - kLift<E>, st.m[t][i]);
            const float f = top == -INFINITY ? 1.f : ex2(st.m[t][i] - top);
            st.m[t][i] = top;
            st.l[t][i] *= f;
#pragma unroll
            for (int jj = 0; jj < MT; ++jj) {
              st.acc[t][jj][i] *= f;
              st.acc[t][jj][i + 2] *= f;
            }
          }
      }
      // weights, in two 16-bit halves, transposed to the MMA's B operand
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float m = st.m[t][i & 1];
          p[i] = ex2(x[t][i] - (m == -INFINITY ? 0.f : m));
          st.l[t][i & 1] += p[i];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t hi = pack<E>(p[2 * h], p[2 * h + 1]);
          const float2 back = unpack<E>(hi);
          ph[t][h] = transpose8(hi);
          pl[t][h] = transpose8(pack<E>(p[2 * h] - back.x, p[2 * h + 1] - back.y));
        }
      }
      // O^T += V^T P^T
      if constexpr (!I8) {
        const uint32_t va = base + 2048 + ((lane & 7) + (lane >> 4) * 8) * 128;
        const uint32_t vx = ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
        // slots past the row's end may hold anything: their V is cleared, not only their weight
        uint32_t m01 = ~0u, m89 = ~0u;
        if (valid < 16) {
          m01 = (2 * c < valid ? 0xffffu : 0u) | (2 * c + 1 < valid ? 0xffff0000u : 0u);
          m89 = (2 * c + 8 < valid ? 0xffffu : 0u) | (2 * c + 9 < valid ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int jj = 0; jj < MT; ++jj) {
          uint32_t f[4];
          ldsm4t(va + (jj >> 2) * G::BOX + (vx ^ ((jj & 3) << 5)), f);
          f[0] &= m01;
          f[1] &= m01;
          f[2] &= m89;
          f[3] &= m89;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma<E>(st.acc[t][jj], f, ph[t][0], ph[t][1]);
            mma<E>(st.acc[t][jj], f, pl[t][0], pl[t][1]);
          }
        }
      } else {
        // lane r reads features [PR r, PR r + PR) of tokens 2c, 2c + 1, 2c + 8, 2c + 9; MMA row
        // r of tile jj is feature PR r + 2 jj, row r + 8 the next one
        constexpr int W = D / 32;               // 32-bit words of a lane's features
        uint32_t v[4][W];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = 2 * c + (k & 1) + (k >> 1) * 8;
          const uint32_t at = base + 16 * G::ROW + row * G::ROW;
          if constexpr (D == 96) {
#pragma unroll
            for (int w = 0; w < 3; ++w)
              v[k][w] = lds32(at + ((((3 * r + w) >> 2) ^ (row & 7)) << 4) + ((3 * r + w) & 3) * 4) ^ 0x80808080u;
          } else if constexpr (G::ROW == 128) {
            const uint4 z = lds128(at + ((r ^ (row & 7)) << 4));
            v[k][0] = z.x ^ 0x80808080u, v[k][1] = z.y ^ 0x80808080u;
            v[k][2] = z.z ^ 0x80808080u, v[k][3] = z.w ^ 0x80808080u;
          } else {
            const uint2 z = lds64(at + ((((r >> 1) ^ ((row >> 1) & 3)) << 4) | ((r & 1) << 3)));
            v[k][0] = z.x ^ 0x80808080u, v[k][1] = z.y ^ 0x80808080u;
          }
        }
        uint32_t vs[W * 2];                         // the features' scales, float16 pairs
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const uint2 z = lds64(sc + 32 + r * (W * 8) + k * 8);
          vs[2 * k] = z.x, vs[2 * k + 1] = z.y;
        }
        // -128 * 2^-24 * the block's weights: what the codes' bias adds to every feature
        float bias[NT][4];
        const uint32_t minus[4] = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};   // -2^-17
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          bias[t][0] = bias[t][1] = bias[t][2] = bias[t][3] = 0.f;
          mma<E>(bias[t], minus, ph[t][0], ph[t][1]);
          mma<E>(bias[t], minus, pl[t][0], pl[t][1]);
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint32_t t01[2] = {__byte_perm(v[0][w], v[1][w], 0x5140), __byte_perm(v[0][w], v[1][w], 0x7362)};
          const uint32_t t89[2] = {__byte_perm(v[2][w], v[3][w], 0x5140), __byte_perm(v[2][w], v[3][w], 0x7362)};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int jj = 2 * w + h;
            const uint32_t f[4] = {codes_to_half(t01[h], 0x4140), codes_to_half(t01[h], 0x4342),
                                   codes_to_half(t89[h], 0x4140), codes_to_half(t89[h], 0x4342)};
            const float2 z = unpack<__half>(vs[jj]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              float o[4];
              mma_from(o, f, ph[t][0], ph[t][1], bias[t]);
              mma<E>(o, f, pl[t][0], pl[t][1]);
              st.acc[t][jj][0] += z.x * o[0];
              st.acc[t][jj][1] += z.x * o[1];
              st.acc[t][jj][2] += z.y * o[2];
              st.acc[t][jj][3] += z.y * o[3];
            }
          }
        }
      }
      ++used;
      __syncwarp();                                 // every lane has read the stage
      if (to_issue > 0) issue();
    }
    if (!alive) break;

    // ---- the end of the item in this warp ----------------------------------------------------
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float l = st.l[t][i];
        l += __shfl_xor_sync(~0u, l, 4);
        l += __shfl_xor_sync(~0u, l, 8);
        l += __shfl_xor_sync(~0u, l, 16);
        st.l[t][i] = l;
      }
    const int n = stop - first;
    if (n == nb) {
      // whole: normalised and written from here
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float unit = I8 ? 1.f / kCode : 1.f;
        const float i0 = unit / st.l[t][0], i1 = unit / st.l[t][1];
        T* o = static_cast<T*>(a.o) + b * a.o_bs + (int64_t)(h0 + t * 8) * a.o_hs;
        if constexpr (!I8) {
#pragma unroll
          for (int jj = 0; jj < MT; ++jj)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t w = transpose8(pack<T>(st.acc[t][jj][2 * h] * i0, st.acc[t][jj][2 * h + 1] * i1));
              if (t * 8 + r < heads)
                *reinterpret_cast<uint32_t*>(o + r * a.o_hs + jj * 16 + h * 8 + 2 * c) = w;
            }
        } else {
#pragma unroll
          for (int jj = 0; jj < MT; ++jj) {
            const int d = r * (D / 8) + 2 * jj;
            if (t * 8 + 2 * c < heads)
              *reinterpret_cast<uint32_t*>(o + (2 * c) * a.o_hs + d) =
                  pack<T>(st.acc[t][jj][0] * i0, st.acc[t][jj][2] * i0);
            if (t * 8 + 2 * c + 1 < heads)
              *reinterpret_cast<uint32_t*>(o + (2 * c + 1) * a.o_hs + d) =
                  pack<T>(st.acc[t][jj][1] * i1, st.acc[t][jj][3] * i1);
          }
        }
        if (a.lse && r == 0)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (t * 8 + 2 * c + i < heads)
              a.lse[b * a.lse_bs + h0 + t * 8 + 2 * c + i] = lse_of<E>(st.m[t][i], st.l[t][i]);
      }
    } else {
      // a piece: in the workspace, or at the end of the warp's range over its stages (every load
      // it issued has been consumed)
      float* p = last ? reinterpret_cast<float*>(ring)
                      : a.first + ((int64_t)blockIdx.x * kWarps + warp) * G::PIECE;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int h = t * 8 + 2 * c + i;
#pragma unroll
          for (int jj = 0; jj < MT; ++jj)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int d = I8 ? r * (D / 8) + 2 * jj + k : jj * 16 + 8 * k + r;
              p[h * G::OS + d] = st.acc[t][jj][2 * k + i] * (I8 ? 1.f / kCode : 1.f);
            }
          if (r == 0) {
            p[NH * G::OS + h] = st.m[t][i];
            p[NH * G::OS + NH + h] = st.l[t][i];
          }
        }
      if (lane == 0) {
        int c0 = blockIdx.x, c1 = blockIdx.x;
        if constexpr (SPLIT) {
          const Shares sh(total, ctas * kWarps);
          c0 = sh.holder(u - first) / kWarps;
          c1 = sh.holder(u - first + nb - 1) / kWarps;
        }
        notes[2 * warp + (last ? 1 : 0)] = make_int4(b, j, c0, c1);
      }
    }
    u += n + past;
    left -= n + past;
    blk = 0;
    b = b2;
    j = j2;
    nb = nb2;
  }
  if (!alive) {                                     // a wait ran out: drain what is in flight
    while (used < issued) {
      const uint32_t s = used % NS;
      if (!wait_full(bar_u + 8 * s, (used / NS) & 1, nullptr)) break;
      ++used;
    }
  }
  __syncthreads();

  // ---- the CTA's pieces, joined item by item: a warp per head, a lane per four features ---------
  const int4 note = lane < 2 * kWarps ? notes[lane] : make_int4(-1, 0, 0, 0);
  uint32_t todo = __ballot_sync(~0u, note.x >= 0);
  int turn = 0;                                     // (item, head) pairs go round the warps
  int pending = 0;                                  // this warp's heads of items that go on elsewhere
  int4 wait_for = make_int4(0, 0, 0, 0);            // lane i: the i-th (at most two items, two heads)
  while (todo) {
    const int at = __ffs(todo) - 1;
    const int ib = __shfl_sync(~0u, note.x, at), ij = __shfl_sync(~0u, note.y, at);
    const int c0 = __shfl_sync(~0u, note.z, at), c1 = __shfl_sync(~0u, note.w, at);
    const bool mine = note.x == ib && note.y == ij;
    const uint32_t members = __ballot_sync(~0u, mine);
    todo &= ~members;
    const int kvh = a.tiles == 1 ? ij : ij / a.tiles, h0 = kvh * a.group + (ij - kvh * a.tiles) * NH;
    const int heads = min(NH, (kvh + 1) * a.group - h0);
    // an item that continues from the CTA before takes the first workspace slot, one that
    // continues into the next CTA (and began here) the second
    float* part = nullptr;
    if (SPLIT && c0 != c1)
      part = a.part + (2 * (int64_t)blockIdx.x + (c0 == (int)blockIdx.x ? 1 : 0)) * G::PART;
    const int begin = warp >= turn ? warp - turn : warp - turn + kWarps;
    turn = (turn + heads) % kWarps;
    for (int h = begin; h < heads; h += kWarps) {
      // this lane's piece (lane 2 w + 1: warp w's last, over its stages; 2 w: its first, in the
      // workspace), and every last piece's four features, members or not
      float4 v[kWarps];
#pragma unroll
      for (int k = 0; k < kWarps; ++k)
        v[k] = *reinterpret_cast<const float4*>(smem + k * NS * G::STAGE + (h * G::OS + 4 * (lane % (D / 4))) * 4);
      float m = -INFINITY, l = 0.f;
      if (mine) {
        if ((lane & 1) || !SPLIT) {
          const float* p = reinterpret_cast<const float*>(smem + (lane >> 1) * NS * G::STAGE) + NH * G::OS + h;
          m = p[0];
          l = p[NH];
        } else {
          const float* p = a.first + ((int64_t)blockIdx.x * kWarps + (lane >> 1)) * G::PIECE + NH * G::OS + h;
          m = p[0];
          l = p[NH];
        }
      }
      const float top = warp_max(m), w = ex2(m - (top == -INFINITY ? 0.f : top));
      float sum = mine ? l * w : 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float f = __shfl_sync(~0u, w, 2 * k + 1);
        if ((members >> (2 * k + 1)) & 1) o.x += f * v[k].x, o.y += f * v[k].y, o.z += f * v[k].z, o.w += f * v[k].w;
      }
      if constexpr (SPLIT) {
        for (uint32_t firsts = members & 0x55555555u; firsts; firsts &= firsts - 1) {
          const int k = __ffs(firsts) - 1;
          const float f = __shfl_sync(~0u, w, k);
          const float4 x = *reinterpret_cast<const float4*>(
              a.first + ((int64_t)blockIdx.x * kWarps + (k >> 1)) * G::PIECE + h * G::OS + 4 * (lane % (D / 4)));
          o.x += f * x.x, o.y += f * x.y, o.z += f * x.z, o.w += f * x.w;
        }
      }
#pragma unroll
      for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
      if (part) {
        if (lane < D / 4) *reinterpret_cast<float4*>(part + h * D + 4 * lane) = o;
        if (lane == 0) *reinterpret_cast<float2*>(part + NH * D + 2 * h) = make_float2(top, sum);
        if (lane == pending) wait_for = make_int4(ib, ij | h << 24, c0, c1);
        ++pending;
      } else {
        write_head<T, E, D>(a, ib, h0 + h, lane, o, top, sum);
      }
    }
  }
  if (!SPLIT || pending == 0) return;

  // ---- items that span CTAs: whoever finds all pieces of a head there joins them ---------------
  // A warp raises a flag for each head whose piece it wrote, passes a fence and looks at the
  // flags of all CTAs of the item: the last to raise its flag sees all of them.  More than one
  // may, and each then joins the same pieces into the same values.  Nobody waits.  A flag holds
  // this call's nonce, so the workspace needs no clearing; whoever joins takes the flags back,
  // so a replayed graph starts afresh.
  __syncwarp();
  if (lane < pending) {
    const int64_t at = (2 * (int)blockIdx.x + (wait_for.z == (int)blockIdx.x ? 1 : 0)) * NH + (wait_for.y >> 24);
    asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(a.flags + at), "l"(a.nonce) : "memory");
  }
  __syncwarp();
  asm volatile("fence.sc.gpu;" ::: "memory");
  for (int i = 0; i < pending; ++i) {
    const int ib = __shfl_sync(~0u, wait_for.x, i), jh = __shfl_sync(~0u, wait_for.y, i);
    const int c0 = __shfl_sync(~0u, wait_for.z, i), c1 = __shfl_sync(~0u, wait_for.w, i);
    const int ij = jh & 0xffffff, h = jh >> 24, n = c1 - c0 + 1;
    bool all = true;
    for (int k = c0 + lane; k <= c1; k += 32) {
      uint64_t f;
      asm volatile("ld.acquire.gpu.global.u64 %0, [%1];"
                   : "=l"(f) : "l"(a.flags + (2 * k + (k == c0 ? 1 : 0)) * NH + h) : "memory");
      all &= f == a.nonce;
    }
    if (!__all_sync(~0u, all)) continue;
    __syncwarp();                                   // what one lane acquired, all lanes may read
    // pieces c0 .. c1, sixteen at a time in flight; a first one is CTA c0's second slot, the others
    // the first slots of the CTAs after it
    const float* part = a.part + 2 * (int64_t)c0 * G::PART;
    auto piece = [&](int k) { return part + (k == 0 ? 1 : 2 * k) * G::PART; };
    const int x4 = h * D + 4 * (lane % (D / 4));
    float top = -INFINITY, sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int k0 = 0; k0 < n; k0 += 16) {
      const int mine = min(k0 + (lane & 15), n - 1);
      float2 ml = __ldcg(reinterpret_cast<const float2*>(piece(mine) + NH * D + 2 * h));
      float4 v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = __ldcg(reinterpret_cast<const float4*>(piece(min(k0 + k, n - 1)) + x4));
      const float up = fmaxf(top, warp_max(ml.x)), zero = up == -INFINITY ? 0.f : up;
      const float keep = ex2(top - zero), w = ex2(ml.x - zero);
      top = up;
      sum = sum * keep + (lane < 16 && k0 + lane < n ? ml.y * w : 0.f);  // lanes 0 .. 15: shares of the sum
      o.x *= keep, o.y *= keep, o.z *= keep, o.w *= keep;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float f = __shfl_sync(~0u, w, k);
        if (k0 + k < n) o.x += f * v[k].x, o.y += f * v[k].y, o.z += f * v[k].z, o.w += f * v[k].w;
      }
    }
#pragma unroll
    for (int x = 8; x; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
    sum = __shfl_sync(~0u, sum, 0);
    for (int k = c0 + lane; k <= c1; k += 32) a.flags[(2 * k + (k == c0 ? 1 : 0)) * NH + h] = 0;
    const int kvh = a.tiles == 1 ? ij : ij / a.tiles;
    write_head<T, E, D>(a, ib, kvh * a.group + (ij - kvh * a.tiles) * NH + h, lane, o, top, sum);
  }
}

// ---- host -------------------------------------------------------------------------------------

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Query heads per item: 8, or 16 where a group has more.
int head_tiles(const KvbPagedDecodeParams* p) { return p->num_q_heads / p->num_kv_heads > 8 ? 2 : 1; }

int64_t items(const KvbPagedDecodeParams* p) {
  const int nh = 8 * head_tiles(p), group = p->num_q_heads / p->num_kv_heads;
  return (int64_t)p->batch * p->num_kv_heads * ((group + nh - 1) / nh);
}

// One CTA per item, or the blocks split over the GPU.  A CTA per item needs no places to be
// found and no joins, and the hardware hands items to SMs as they come free; but a long row
// keeps its CTA for long, and very many items are as many starts.  What the host knows is the
// table's width (or the caller's bound).  Measured, us per call (CTA per item / split), KV
// heads x requests = items, D 128, 16 bits: 2 items of 256 tokens 5.1 / 7.7, of 1024 9.2 / 8.0,
// of 2048 15.0 / 8.9; 32 of 1024 9.7 / 12.4; 128 of 2048 25.0 / 31.5; 256 of 64 7.0 / 6.7, of 256
// 12.9 / 15.9; 512 of 64 13.0 / 7.4, of 256 24.8 / 18.8, of 512 35.1 / 34.5, of 1024 51.8 / 54.2,
// of 2048 84.9 / 93.5.  int8: 256 of 1024 25.7 / 27.9; 512 of 256 24.5 / 24.5, of 1024 41.9 / 41.8.
bool split(const KvbPagedDecodeParams* p) {
  if (p->batch > kSplitRows) return false;
  // 32-bit places: wider than any pool
  if ((int64_t)p->batch * (p->max_blocks_per_seq + kItemCost) * p->num_q_heads > 0x7fffffff) return false;
  const int64_t width = p->max_seq_len > 0
                            ? std::min<int64_t>(p->max_blocks_per_seq, ((int64_t)p->max_seq_len + 15) / 16)
                            : p->max_blocks_per_seq;
  const int64_t n = items(p);
  if (n > (p->pool_format == KVB_POOL_INT8_KIVI || width <= 32 ? 2 : 4) * kSms) return true;
  return width > (n < 64 ? 64 : 128);
}

// Workspace of a split launch: CTAs' pieces, warps' first pieces, flags.
struct Room {
  int64_t part, first, flags, bytes;
  explicit Room(const KvbPagedDecodeParams* p) {
    const int64_t nh = 8 * head_tiles(p);
    part = 0;
    first = part + 4 * kSms * 2 * (nh * p->head_dim + 2 * nh);
    flags = first + 4 * kSms * kMostWarps * (nh * (p->head_dim + 4) + 2 * nh);
    bytes = flags + kSms * 2 * nh * (int64_t)sizeof(uint64_t);
  }
};

int check(const KvbPagedDecodeParams* p) {
  if (!p) return fail(KVB_ERR_INVALID, "params is NULL");
  if (p->dtype != KVB_DTYPE_BF16 && p->dtype != KVB_DTYPE_FP16)
    return fail(KVB_ERR_INVALID, "dtype must be KVB_DTYPE_BF16 or KVB_DTYPE_FP16");
  if (p->head_dim != 64 && p->head_dim != 96 && p->head_dim != 128)
    return fail(KVB_ERR_INVALID, "head_dim must be 64, 96 or 128");
  if (p->batch < 0) return fail(KVB_ERR_INVALID, "batch must be non-negative");
  if (p->num_kv_heads < 1 || p->num_q_heads < 1 || p->num_q_heads % p->num_kv_heads)
    return fail(KVB_ERR_INVALID, "num_q_heads must be divisible by num_kv_heads, both >= 1");
  if (p->batch > 65535 || p->num_q_heads > 65535)
    return fail(KVB_ERR_UNSUPPORTED, "batch and num_q_heads must be <= 65535");
  if (p->block_size != 16) return fail(KVB_ERR_INVALID, "block_size must be 16");
  if (p->pool_format != KVB_POOL_INT8_KIVI && p->pool_format != KVB_POOL_COMPUTE)
    return fail(KVB_ERR_INVALID, "pool_format must be KVB_POOL_INT8_KIVI or KVB_POOL_COMPUTE");
  if (p->num_blocks < 1) return fail(KVB_ERR_INVALID, "num_blocks must be >= 1");
  if (p->max_blocks_per_seq < 1 || p->block_table_stride < p->max_blocks_per_seq)
    return fail(KVB_ERR_INVALID,
                "max_blocks_per_seq must be >= 1 and block_table_stride at least that");
  if ((int64_t)p->batch * (p->max_blocks_per_seq + kItemCost) > 0x7fffffff || p->max_blocks_per_seq > (1 << 27) - 1)
    return fail(KVB_ERR_UNSUPPORTED, "batch * max_blocks_per_seq must be below 2^31, one row's blocks below 2^27");
  if (p->batch == 0) return KVB_OK;
  if (!p->q || !p->o || !p->kv_pool || !p->block_tables || !p->seq_lens)
    return fail(KVB_ERR_INVALID, "q, o, kv_pool, block_tables and seq_lens must be non-null");
  if (p->pool_format == KVB_POOL_INT8_KIVI && (!p->k_scale16 || !p->v_scale16))
    return fail(KVB_ERR_INVALID, "int8 pools need k_scale16 and v_scale16");
  if (!aligned(p->q, 16) || !aligned(p->o, 16) || !aligned(p->kv_pool, 16) ||
      (p->pool_format == KVB_POOL_INT8_KIVI &&
       (!aligned(p->k_scale16, 16) || !aligned(p->v_scale16, 16))))
    return fail(KVB_ERR_INVALID, "q, o, kv_pool and the scales must be 16-byte aligned");
  if (p->q_batch_stride % 8 || p->q_head_stride % 8 || p->o_batch_stride % 8 ||
      p->o_head_stride % 8)
    return fail(KVB_ERR_INVALID, "strides must be multiples of 8 elements");
  // heads of one request inside its row, or requests of one head inside the head's
  const auto apart = [&](int64_t in, int64_t n_in, int64_t out, int64_t n_out) {
    return (n_in == 1 || in >= p->head_dim) && (n_out == 1 || out >= (n_in > 1 ? (n_in - 1) * in : 0) + p->head_dim);
  };
  if (!apart(p->o_head_stride, p->num_q_heads, p->o_batch_stride, p->batch) &&
      !apart(p->o_batch_stride, p->batch, p->o_head_stride, p->num_q_heads))
    return fail(KVB_ERR_INVALID, "heads of o must not overlap");
  return KVB_OK;
}

// The pool as (feature, KV head and slot, K or V, block); a box is one head's 16 slots of K and
// V, 64 features (16-bit) or all of them (int8, padded to 64 or 128 by the zero fill).
bool pool_map(CUtensorMap* m, const KvbPagedDecodeParams* p, std::string* err) {
  static PFN_cuTensorMapEncodeTiled_v12000 enc = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  if (!enc) {
    *err = "cuTensorMapEncodeTiled unavailable from the CUDA driver";
    return false;
  }
  const bool i8 = p->pool_format == KVB_POOL_INT8_KIVI;
  const cuuint64_t el = i8 ? 1 : 2, row = el * p->head_dim, kv = row * 16 * p->num_kv_heads;
  const cuuint64_t dims[4] = {(cuuint64_t)p->head_dim, (cuuint64_t)p->num_kv_heads * 16, 2,
                              (cuuint64_t)p->num_blocks};
  const cuuint64_t strides[3] = {row, kv, 2 * kv};
  const cuuint32_t box[4] = {(cuuint32_t)(i8 && p->head_dim > 64 ? 128 : 64), 16, 2, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r = enc(
      m, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
            : p->dtype == KVB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
      4, const_cast<void*>(p->kv_pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
      i8 && p->head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    *err = "cuTensorMapEncodeTiled failed with CUresult " + std::to_string((int)r);
    return false;
  }
  return true;
}

template <typename... KArgs, typename... As>
cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, int threads, int smem, cudaStream_t s, As&&... as) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<As>(as)...);
}

template <typename T, int D, bool I8, int NT>
cudaError_t launch(const CUtensorMap& map, const Args& a, bool is_split, cudaStream_t s) {
  using G = Geo<D, I8, NT>;
  auto kern = is_split ? kvb_paged_decode_kernel<T, D, I8, NT, true> : kvb_paged_decode_kernel<T, D, I8, NT, false>;
  // the shared-memory limit is set once per device and instantiation
  static std::atomic<uint64_t> ready[2];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev > 63 || !(ready[is_split].load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
    if (e != cudaSuccess) return e;
    ready[is_split].fetch_or(bit, std::memory_order_release);
  }
  return launch_pdl(kern, dim3(is_split ? a.ctas : a.batch * a.items), G::THREADS, G::SMEM, s, map, a);
}

template <typename T, bool I8, int NT>
cudaError_t launch_d(int D, const CUtensorMap& map, const Args& a, bool is_split, cudaStream_t s) {
  return D == 64 ? launch<T, 64, I8, NT>(map, a, is_split, s)
                 : D == 96 ? launch<T, 96, I8, NT>(map, a, is_split, s)
                           : launch<T, 128, I8, NT>(map, a, is_split, s);
}

template <typename T>
cudaError_t launch_t(const KvbPagedDecodeParams* p, const CUtensorMap& map, const Args& a, bool is_split,
                     cudaStream_t s) {
  const bool i8 = p->pool_format == KVB_POOL_INT8_KIVI;
  if (head_tiles(p) == 1)
    return i8 ? launch_d<T, true, 1>(p->head_dim, map, a, is_split, s)
              : launch_d<T, false, 1>(p->head_dim, map, a, is_split, s);
  return i8 ? launch_d<T, true, 2>(p->head_dim, map, a, is_split, s)
            : launch_d<T, false, 2>(p->head_dim, map, a, is_split, s);
}

}  // namespace kvb_pd

extern "C" int64_t kvb_paged_decode_workspace_bytes(const KvbPagedDecodeParams* p) {
  if (kvb_pd::check(p) != KVB_OK) return -1;
  if (p->batch == 0 || !kvb_pd::split(p)) return 0;
  return kvb_pd::Room(p).bytes;
}

extern "C" int kvb_paged_decode_fwd(const KvbPagedDecodeParams* p, void* stream) {
  if (const int rc = kvb_pd::check(p)) return rc;
  if (p->batch == 0) return KVB_OK;
  const bool is_split = kvb_pd::split(p);
  if (is_split) {
    if (!p->workspace || p->workspace_bytes < kvb_paged_decode_workspace_bytes(p))
      return kvb_pd::fail(KVB_ERR_INVALID, "workspace must hold kvb_paged_decode_workspace_bytes bytes");
    if (!kvb_pd::aligned(p->workspace, 16))
      return kvb_pd::fail(KVB_ERR_INVALID, "workspace must be 16-byte aligned");
  }
  kvb_pd::Args a = {};
  a.batch = p->batch;
  a.num_q_heads = p->num_q_heads;
  a.num_kv_heads = p->num_kv_heads;
  a.num_blocks = p->num_blocks;
  a.width = p->max_blocks_per_seq;
  a.group = p->num_q_heads / p->num_kv_heads;
  const int nh = 8 * kvb_pd::head_tiles(p);
  a.tiles = (a.group + nh - 1) / nh;
  a.items = p->num_kv_heads * a.tiles;
  if ((int64_t)a.items * p->batch > 0x7fffffff)
    return kvb_pd::fail(KVB_ERR_UNSUPPORTED, "too many requests and heads for one call");
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  a.q = p->q;
  a.o = p->o;
  a.lse = p->lse;
  a.q_bs = p->q_batch_stride;
  a.q_hs = p->q_head_stride;
  a.o_bs = p->o_batch_stride;
  a.o_hs = p->o_head_stride;
  a.lse_bs = p->lse_batch_stride;
  a.table_stride = p->block_table_stride;
  a.k_scale = static_cast<const __half*>(p->k_scale16);
  a.v_scale = static_cast<const __half*>(p->v_scale16);
  a.tables = p->block_tables;
  a.lens = p->seq_lens;
  a.status = p->status;
  if (is_split) {
    const int64_t most = (int64_t)p->batch * p->max_blocks_per_seq * a.items;
    a.ctas = (int)std::max<int64_t>(
        1, std::min({(int64_t)kvb_pd::kSms, (most + kvb_pd::kMinUnits - 1) / kvb_pd::kMinUnits,
                     kvb_pd::kSpan * kvb_pd::items(p)}));
    const kvb_pd::Room room(p);
    uint8_t* w = static_cast<uint8_t*>(p->workspace);
    a.part = reinterpret_cast<float*>(w + room.part);
    a.first = reinterpret_cast<float*>(w + room.first);
    a.flags = reinterpret_cast<uint64_t*>(w + room.flags);
    // a different odd number for every call of the process (the odd factor permutes 2^64)
    static std::atomic<uint64_t> calls{0};
    a.nonce = (2 * calls.fetch_add(1, std::memory_order_relaxed) + 1) * 0x9e3779b97f4a7c15ull;
  }
  CUtensorMap map;
  std::string err;
  if (!kvb_pd::pool_map(&map, p, &err)) return kvb_pd::fail(KVB_ERR_CUDA, err);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = p->dtype == KVB_DTYPE_BF16
                            ? kvb_pd::launch_t<__nv_bfloat16>(p, map, a, is_split, s)
                            : kvb_pd::launch_t<__half>(p, map, a, is_split, s);
  if (e != cudaSuccess)
    return kvb_pd::fail(KVB_ERR_CUDA, std::string("kvb_paged_decode_fwd launch: ") + cudaGetErrorString(e));
  return KVB_OK;
}
