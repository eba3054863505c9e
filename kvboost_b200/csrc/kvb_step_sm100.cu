// The small operators of a batched decode step over the block pool, sm_100a:
//
//  * kvb_extend_block_tables: block tables, slots and positions of the step's new
//    tokens, from request lengths on the device;
//  * kvb_append_paged_kv: the new tokens' K/V into the 16-bit pool at those slots;
//  * kvb_process_logits: penalties, biases, temperature and grammar mask in one
//    pass over the logits.
//
// The first is latency, the other two byte work: no data is read on the host.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <string>
#include <type_traits>

#include "kvb_attn.h"

int kvb_detail_fail(int code, const std::string& msg);

namespace kvb_step {

int fail(int code, const std::string& msg) { return kvb_detail_fail(code, msg); }

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return fail(KVB_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return KVB_OK;
}

// ---- block tables and slots -------------------------------------------------------------

struct TablesArgs {
  int batch, width, num_blocks, max_tokens, capacity;
  int64_t stride;
  int32_t* tables;
  const int32_t* seq_lens;
  const int32_t* new_lens;
  const int32_t* free_blocks;
  const int32_t* num_free;
  int32_t* slots;
  int64_t* positions;
  int32_t* cu_new;
  int32_t* seq_lens_out;
  int32_t* num_free_out;
  int32_t* status;
};

// Sums that stop at 2^31 - 1: exact where they are compared with something below.
__device__ __forceinline__ uint32_t add_sat(uint32_t x, uint32_t y) { return min(x + y, 0x7fffffffu); }

__device__ __forceinline__ uint2 scan_sat(uint2 x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t p = __shfl_up_sync(~0u, x.x, o), q = __shfl_up_sync(~0u, x.y, o);
    if (lane >= o) x = make_uint2(add_sat(x.x, p), add_sat(x.y, q));
  }
  return x;
}

// A scan over the rows gives each row's place in the packed arrays and in the free list (one
// scan for both: a row that does not fit in the packed arrays is followed only by rows that
// do not either, or that need nothing).  Then a thread takes four consecutive tokens: one
// search for the row of the first, slots and positions in 16-byte stores, and the table entry
// of each block that a token begins.
// Latency is all there is: two dependent reads, a scan and the stores.  One cluster of up to
// eight CTAs shares the tokens; every CTA scans for itself, and since the new lengths may go
// over the old ones, no CTA writes before all have read.  8 rows of a token each: 4.1 us; 256 rows
// of 43220 tokens 8.4 us, 38.7 with one CTA.
__global__ void __launch_bounds__(1024) kvb_extend_tables_kernel(const TablesArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* cu = sm;                        // [batch + 1] place of the row's tokens
  int32_t* start = cu + a.batch + 1;       // [batch] pops before the row's, -1: does not fit
  int32_t* len = start + a.batch;          // [batch]
  __shared__ uint2 wsum[32];
  __shared__ int taken;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nt = blockDim.x, warps = nt >> 5;
  const int nfree = min(max(*a.num_free, 0), a.capacity);
  uint2 base = make_uint2(0, 0);
  int err = 0;
  if (tid == 0) cu[0] = taken = 0;
  for (int b0 = 0; b0 < a.batch; b0 += nt) {
    const int b = b0 + tid;
    int l = 0, n = 0;
    bool ok = false;
    if (b < a.batch) {
      l = a.seq_lens[b];
      n = a.new_lens[b];
      ok = l >= 0 && n >= 0 && n <= a.max_tokens;
      if (!ok) n = 0;
      ok = ok && (int64_t)l + n <= (int64_t)a.width * 16;
      if (!ok) err |= KVB_STATUS_BAD_LENGTH;
    }
    const int need = ok ? (l + n + 15) / 16 - (l + 15) / 16 : 0;
    uint2 x = scan_sat(make_uint2(n, need), lane);
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    const uint2 w = scan_sat(lane < warps ? wsum[lane] : make_uint2(0, 0), lane);
    const uint32_t before_t = __shfl_sync(~0u, w.x, max(warp - 1, 0));
    const uint32_t before_n = __shfl_sync(~0u, w.y, max(warp - 1, 0));
    if (warp > 0) x = make_uint2(add_sat(x.x, before_t), add_sat(x.y, before_n));
    x = make_uint2(add_sat(x.x, base.x), add_sat(x.y, base.y));
    base = make_uint2(add_sat(base.x, __shfl_sync(~0u, w.x, 31)), add_sat(base.y, __shfl_sync(~0u, w.y, 31)));
    const bool packed = ok && (n == 0 || x.x <= (uint32_t)a.max_tokens);
    const bool fits = packed && (need == 0 || x.y <= (uint32_t)nfree);
    if (ok && !packed) err |= KVB_STATUS_BAD_LENGTH;
    if (packed && !fits) err |= KVB_STATUS_POOL_EMPTY;
    if (b < a.batch) {
      cu[b + 1] = (int)min(x.x, (uint32_t)a.max_tokens);
      start[b] = fits ? (int)x.y - need : -1;
      len[b] = l;
    }
    // rows that fit and need blocks come before all others that need some: the last one's end
    const int end = __reduce_max_sync(~0u, fits && need ? (int)x.y : 0);
    if (lane == 0 && end) atomicMax(&taken, end);
    __syncthreads();
  }
  if (gridDim.x > 1) {                     // every CTA has read the lengths and the free list's
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (blockIdx.x == 0) {
    for (int b = tid; b < a.batch; b += nt) {
      a.cu_new[b + 1] = cu[b + 1];
      a.seq_lens_out[b] = start[b] >= 0 ? len[b] + cu[b + 1] - cu[b] : len[b];
    }
    if (tid == 0) {
      a.cu_new[0] = 0;
      *a.num_free_out = nfree - taken;
    }
  }
  const int total = cu[a.batch], step = gridDim.x * nt * 4;
  for (int t0 = (blockIdx.x * nt + tid) * 4; t0 < a.max_tokens; t0 += step) {
    int row = 0;
    if (t0 < total) {                      // the row with cu[row] <= t0 < cu[row + 1]
      int hi = a.batch - 1;
      while (row < hi) {
        const int mid = (row + hi) >> 1;
        if (cu[mid + 1] <= t0) row = mid + 1; else hi = mid;
      }
    }
    int slot[4];
    int64_t pos[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + i;
      slot[i] = -1;
      pos[i] = 0;
      if (t >= total) continue;
      while (cu[row + 1] <= t) ++row;
      const int s = start[row];
      if (s < 0) continue;
      const int l = len[row], p = l + t - cu[row], have = (l + 15) >> 4, blk = p >> 4;
      int32_t* table = a.tables + (int64_t)row * a.stride;
      int id;
      if (blk < have) {
        id = table[blk];
      } else {
        id = a.free_blocks[nfree - 1 - s - (blk - have)];
        if ((p & 15) == 0) table[blk] = id;
      }
      pos[i] = p;
      if (id >= 0 && id < a.num_blocks) slot[i] = id * 16 + (p & 15);
      else err |= KVB_STATUS_BAD_BLOCK;
    }
    if (t0 + 4 <= a.max_tokens) {
      *reinterpret_cast<int4*>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<longlong2*>(a.positions + t0) = make_longlong2(pos[0], pos[1]);
      *reinterpret_cast<longlong2*>(a.positions + t0 + 2) = make_longlong2(pos[2], pos[3]);
    } else {
      for (int i = 0; i < 4 && t0 + i < a.max_tokens; ++i) {
        a.slots[t0 + i] = slot[i];
        a.positions[t0 + i] = pos[i];
      }
    }
  }
  if (err && a.status) atomicOr(a.status, err);
}

// ---- append ---------------------------------------------------------------------------------

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery's round-up method).
struct Div {
  uint32_t d, mul, shift;
  explicit Div(uint32_t by) : d(by), shift(0) {
    while ((1ull << shift) < by) ++shift;
    mul = (uint32_t)(((((uint64_t)1 << shift) - by) << 32) / by + 1);
  }
  __device__ __forceinline__ uint32_t quot(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct AppendArgs {
  Div per, vecs;                             // 16-byte pieces of a token, of a head's vector
  uint32_t pieces;                           // of all tokens
  int heads, num_blocks;
  const uint4* src[2];
  int64_t token_stride[2], head_stride[2];   // in 16-byte pieces
  uint4* pool;
  const int32_t* slots;
  int32_t* status;
};

// A thread moves one 16-byte piece of K and the same one of V, for one slot and one place
// computed.  Byte work: the 8192-token prefill of 8 heads (D 128) takes 12.4 to 13.0 us (5.2 TB/s, 80 % of
// the measured copy, the launch included), as with two or four such pairs a thread; with K and V
// in CTAs of their own 29.5, and 16.2 with four pieces a thread (a slot read per piece).
__global__ void __launch_bounds__(256) kvb_append_paged_kernel(const AppendArgs a) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.pieces) return;
  const uint32_t t = a.per.quot(i), r = i - t * a.per.d, h = a.vecs.quot(r), x = r - h * a.vecs.d;
  const int slot = a.slots[t];
  const uint4 k = __ldcs(a.src[0] + t * a.token_stride[0] + h * a.head_stride[0] + x);
  const uint4 v = __ldcs(a.src[1] + t * a.token_stride[1] + h * a.head_stride[1] + x);
  if (slot < 0 || slot >= (int64_t)a.num_blocks * 16) {
    if (slot != -1 && r == 0 && a.status) atomicOr(a.status, KVB_STATUS_BAD_BLOCK);
    return;
  }
  uint4* to = a.pool + (((int64_t)(slot >> 4) * 2 * a.heads + h) * 16 + (slot & 15)) * a.vecs.d + x;
  to[0] = k;
  to[(int64_t)a.heads * 16 * a.vecs.d] = v;
}

// ---- logits -----------------------------------------------------------------------------------

struct LogitsArgs {
  int vocab, history_len, num_bias;
  int iters;                              // a CTA's slice in 2048 tokens
  const void* logits;
  void* out;
  int64_t logits_stride, out_stride, history_stride, mask_stride;
  const int32_t* token_ids;
  const int32_t* prompt_lens;
  const int32_t* total_lens;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const float* temperature;
  const int32_t* bias_ids;
  const float* bias_values;
  const uint32_t* mask;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float* p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// A thread's eight values of a turn as they are stored, and as float32: G side by side, then the
// next G 32 G further on; an access moves G values (G 1 needs no alignment).  left: from the first
// value to the slice's end.  Whole 32-byte sectors a thread, or 16 bytes side by side over the
// warp, are what the stores need: two 16-byte stores of float32, 32 bytes apart over the warp,
// took 19.4 us for 150 rows of 100000 where these take 12.5.
template <int G>
__device__ __forceinline__ constexpr int place(int k) { return k / G * 32 * G + k % G; }

struct alignas(32) Wide { uint32_t x[8]; };

template <typename R>
__device__ __forceinline__ R stream_in(const R* p) { return __ldcs(p); }
template <typename R>
__device__ __forceinline__ void stream_out(R* p, R v) { __stcs(p, v); }
__device__ __forceinline__ Wide stream_in(const Wide* p) {
  Wide v;
  asm volatile("ld.global.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.x[0]), "=r"(v.x[1]), "=r"(v.x[2]), "=r"(v.x[3]), "=r"(v.x[4]), "=r"(v.x[5]), "=r"(v.x[6]), "=r"(v.x[7])
               : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void stream_out(Wide* p, Wide v) {
  asm volatile("st.global.L2::evict_first.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.x[0]), "r"(v.x[1]),
               "r"(v.x[2]), "r"(v.x[3]), "r"(v.x[4]), "r"(v.x[5]), "r"(v.x[6]), "r"(v.x[7]) : "memory");
}

template <typename T, int G>
struct Eight {
  static constexpr int B = G * sizeof(T);
  using Run = typename std::conditional<B == 32, Wide, typename std::conditional<B == 16, uint4,
              typename std::conditional<B == 8, uint2, T>::type>::type>::type;
  Run run[8 / G];
  __device__ __forceinline__ void load(const T* p, int left) {
#pragma unroll
    for (int i = 0; i < 8 / G; ++i) {
      const T* q = p + place<G>(i * G);
      if (place<G>(i * G + G - 1) < left) {
        run[i] = stream_in(reinterpret_cast<const Run*>(q));
      } else {
        T h[G];
#pragma unroll
        for (int k = 0; k < G; ++k) {
          from_f32(h + k, 0.f);
          if (place<G>(i * G + k) < left) h[k] = q[k];
        }
        memcpy(&run[i], h, sizeof(Run));
      }
    }
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    T h[8];
    memcpy(h, run, sizeof(run));
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = to_f32(h[k]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[8], int left) {
    T h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) from_f32(h + k, x[k]);
#pragma unroll
    for (int i = 0; i < 8 / G; ++i) {
      T* q = p + place<G>(i * G);
      if (place<G>(i * G + G - 1) < left) {
        Run v;
        memcpy(&v, h + i * G, sizeof(v));
        stream_out(reinterpret_cast<Run*>(q), v);
      } else {
#pragma unroll
        for (int k = 0; k < G; ++k)
          if (place<G>(i * G + k) < left) q[k] = h[i * G + k];
      }
    }
  }
};

constexpr int kBiasRoom = 256;            // a slice's bias entries kept in shared memory
constexpr int kCounts16 = 16383;          // the longest history that a 16-bit note can count

// A CTA takes one slice of a row.  It notes the history's tokens that fall into the slice in
// shared memory (per token a seen bit, a count and a bias bit, in 16 bits, or 32 for long
// histories; integer adds: any order gives the same) and the slice's bias entries in their
// order, then streams the slice, 2048 tokens a turn, 8 a thread, the next turn's logits on their
// way.  Byte work for large batches: the logits once, the result once; the history is read by
// every slice's CTA (from L2), so slices are long there, and short (2048) where few rows have to
// spread over the GPU.  The stream's own work has to stay small beside 6 bytes a token: with the
// penalties' divisions and the bias list in the unrolled stream it took 124 us for 192 rows of
// 151936, waiting for instructions; with 32-bit notes of shorter slices, all of a thread's logits
// in registers, 68 us; so 37.9 us (4.7 TB/s; 28.4 us and 6.3 TB/s with the mask alone), what the
// notes cost being the two barriers with the wait for the history before the first turn, and the
// branches of noted tokens.  A list of the noted tokens, worked on behind the stream, took
// longer (45 us).  The quotients by the repetition penalty and the temperature are products with
// their reciprocals: one more rounding of float32 each (3.5e-8 from the 64-bit result instead of
// 2.5e-8 in the 2-norm); with divisions an eager call takes 47.3 us instead of 38.9.
//
// G 8: rows on 8 values.  G 4: rows on 4 without notes (12.5 us for 150 rows of 100000, 13.5 with
// G 8).  G 1: other rows, odd vocabularies (150 of 100001: 25.4 us with notes, 18.8 for 100000).
template <typename TI, typename TO, typename NT, int G>
__global__ void __launch_bounds__(256, 6) kvb_logits_kernel(const LogitsArgs a) {
  constexpr int PER = 4 / sizeof(NT), BITS = 8 * sizeof(NT);   // notes a word, bits a note
  constexpr uint32_t kBias = 1u << (BITS - 1), kAll = BITS == 32 ? ~0u : 0xffffu;
  extern __shared__ __align__(16) uint32_t note[];
  __shared__ int32_t list_ids[kBiasRoom];
  __shared__ float list_values[kBiasRoom];
  __shared__ int list_len;
  const int b = blockIdx.y, tid = threadIdx.x;
  const int v0 = blockIdx.x * a.iters * 2048, v1 = min(a.vocab, v0 + a.iters * 2048);
  const TI* in = static_cast<const TI*>(a.logits) + b * a.logits_stride;
  TO* out = static_cast<TO*>(a.out) + b * a.out_stride;
  const uint8_t* mask = a.mask ? reinterpret_cast<const uint8_t*>(a.mask + b * a.mask_stride) : nullptr;
  // the thread's first token of a turn, and the first of the eight whose mask byte it loads
  const int first = (tid & ~31) * 8 + (tid & 31) * G, byte = tid * 8;
  Eight<TI, G> next;
  uint32_t next_open = 0xff;
  next.load(in + v0 + first, v1 - v0 - first);
  if (mask && v0 + byte < v1) next_open = mask[(v0 + byte) >> 3];
  const float r = a.repetition ? a.repetition[b] : 1.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f;
  const float pres = a.presence ? a.presence[b] : 0.f;
  const float heat = a.temperature ? fmaxf(a.temperature[b], 1e-5f) : 1.f;
  const int32_t* bias_ids = a.bias_ids ? a.bias_ids + (int64_t)b * a.num_bias : nullptr;
  const float* bias_values = a.bias_values + (int64_t)b * a.num_bias;
  const bool noted = G != 4 && (a.token_ids || bias_ids);
  if (noted) {
    // The first 2048 of the history (before its length is known) and 64 of the bias list are
    // on their way while the notes are cleared.
    const int32_t* ids = a.token_ids + b * a.history_stride;
    const int room = a.token_ids ? a.history_len : 0;
    int total = a.token_ids ? a.total_lens[b] : 0, prompt = a.token_ids && a.prompt_lens ? a.prompt_lens[b] : 0;
    int id[8], bias_id[2] = {-1, -1};
    float bias_value[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; ++k) id[k] = tid + k * 256 < room ? ids[tid + k * 256] : -1;
    if (bias_ids && tid < 32)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (tid + 32 * k < a.num_bias) {
          bias_id[k] = bias_ids[tid + 32 * k];
          bias_value[k] = bias_values[tid + 32 * k];
        }
    for (int i = tid; i < a.iters * 512 / PER; i += 256) reinterpret_cast<uint4*>(note)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    total = min(max(total, 0), room);
    prompt = min(prompt, total);
    for (int i = tid; i < total; i += 8 * 256) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t at = (uint32_t)id[k] - (uint32_t)v0, shift = (at % PER) * BITS;
        if (i + k * 256 < total && id[k] >= 0 && at < (uint32_t)(v1 - v0)) {
          if (i + k * 256 < prompt) atomicOr(&note[at / PER], 1u << shift);
          else atomicAdd(&note[at / PER], 2u << shift);
        }
      }
      if (i + 8 * 256 < total)
#pragma unroll
        for (int k = 0; k < 8; ++k) id[k] = i + (k + 8) * 256 < total ? ids[i + (k + 8) * 256] : -1;
    }
    if (bias_ids && tid < 32) {           // the slice's entries, in their order
      int n = 0;
      for (int e0 = 0; e0 < a.num_bias; e0 += 32) {
        int mine = bias_id[0];
        float value = bias_value[0];
        bias_id[0] = bias_id[1];
        bias_value[0] = bias_value[1];
        if (e0 >= 64) {
          mine = e0 + tid < a.num_bias ? bias_ids[e0 + tid] : -1;
          value = e0 + tid < a.num_bias ? bias_values[e0 + tid] : 0.f;
        }
        const bool here = mine >= v0 && mine < v1;
        const uint32_t some = __ballot_sync(~0u, here);
        if (here) {
          const uint32_t at = mine - v0;
          atomicOr(&note[at / PER], kBias << ((at % PER) * BITS));
          const int place = n + __popc(some & ((1u << tid) - 1));
          if (place < kBiasRoom) {
            list_ids[place] = mine;
            list_values[place] = value;
          }
        }
        n += __popc(some);
      }
      if (tid == 0) list_len = n;
    }
    __syncthreads();
  }
  const float ir = 1.f / r, inv = 1.f / heat;
#pragma unroll 1
  for (int at0 = v0; at0 < v1; at0 += 2048) {
    const int v = at0 + first;
    float x[8];
    next.values(x);
    uint32_t open = 0xff;
    if (G == 8) {
      open = next_open;
    } else if (mask) {                      // from the lanes that hold the bytes
      open = 0;
#pragma unroll
      for (int i = 0; i < 8 / G; ++i) {
        const int bit = place<G>(i * G) + (tid & 31) * G;
        open |= ((__shfl_sync(~0u, next_open, bit / 8) >> (bit % 8)) & ((1u << G) - 1)) << (i * G);
      }
    }
    if (at0 + 2048 < v1) {
      next.load(in + v + 2048, v1 - v - 2048);
      if (mask && at0 + 2048 + byte < v1) next_open = mask[(at0 + 2048 + byte) >> 3];
    }
    if (noted) {
      uint32_t n[8 / PER];
      const NT* one = reinterpret_cast<const NT*>(note) + (v - v0);
      if (G == 8) {
        memcpy(n, __builtin_assume_aligned(one, 16), sizeof(n));
      } else {
#pragma unroll
        for (int i = 0; i < 8 / PER; ++i) {
          n[i] = one[place<G>(i * PER)];
          if (PER == 2) n[i] |= (uint32_t)one[place<G>(i * PER + 1)] << 16;
        }
      }
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < 8 / PER; ++i) any |= n[i];
      if (any) {
        bool biased = false;
#pragma unroll
        for (int w = 0; w < 8 / PER; ++w) {   // a word at a time: few of a warp's 256 tokens are noted
          if (!n[w]) continue;
#pragma unroll
          for (int k = w * PER; k < (w + 1) * PER; ++k) {
            const uint32_t one = (n[w] >> ((k % PER) * BITS)) & kAll, count = (one & ~kBias) >> 1;
            if ((one & ~kBias) && a.repetition) x[k] *= x[k] > 0.f ? ir : r;
            if (count) x[k] = x[k] - freq * (float)count - pres;
            biased |= (one & kBias) != 0;
          }
        }
        if (biased) {
          const bool all = list_len <= kBiasRoom;
          const int len = all ? list_len : a.num_bias;
#pragma unroll 1
          for (int e = 0; e < len; ++e) {
            const uint32_t off = (uint32_t)((all ? list_ids[e] : bias_ids[e]) - v);
            const uint32_t at = off / (32 * G) * G + off % (32 * G);
            if (off < 256 && off % (32 * G) < G) {
              const float w = all ? list_values[e] : bias_values[e];
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] += at == k ? w : 0.f;
            }
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = (open >> k) & 1 ? x[k] * inv : __uint_as_float(0xff800000u);
    Eight<TO, G>::store(out + v, x, v1 - v);
  }
}

// Whether a row of n bytes, `step` bytes from one to the next, of one buffer shares bytes with one of
// the other.  (Rows of two buffers may lie side by side in one wider buffer.)
bool rows_meet(const void* p, int64_t n, int64_t step, const void* q, int64_t m, int64_t other, int rows) {
  const int64_t x = (int64_t)reinterpret_cast<uintptr_t>(p), y = (int64_t)reinterpret_cast<uintptr_t>(q);
  if (x + (rows - 1) * step + n <= y || y + (rows - 1) * other + m <= x) return false;
  for (int i = 0, j = 0; i < rows && j < rows;) {
    const int64_t a = x + i * step, b = y + j * other;
    if (a + n <= b) ++i;
    else if (b + m <= a) ++j;
    else return true;
  }
  return false;
}

template <typename TI, typename TO>
void launch_logits(LogitsArgs a, int batch, cudaStream_t s) {
  // Slices of up to 8192 tokens, as long as every SM gets two CTAs (192 x 151936: 37.9 us with
  // 8192, 41.5 with 16384, 43.8 with 4096; 16 x 128000: 6.0 us with 4096, 7.0 with 2048, 7.8 with
  // 8192), 4096 without notes (192 x 151936: 28.3 us, 27.6 with 2048, 29.5 with 8192).
  for (a.iters = a.token_ids || a.bias_ids ? 4 : 2; a.iters > 1; a.iters /= 2)
    if ((int64_t)batch * ((a.vocab + a.iters * 2048 - 1) / (a.iters * 2048)) >= 2 * 148) break;
  const dim3 grid((a.vocab + a.iters * 2048 - 1) / (a.iters * 2048), batch);
  const auto on = [&](int n) {            // every row on n values
    return aligned(a.logits, n * sizeof(TI)) && aligned(a.out, n * sizeof(TO)) &&
           (batch == 1 || (a.logits_stride % n == 0 && a.out_stride % n == 0));
  };
  const bool few = a.history_len <= kCounts16;
  const int smem = a.iters * (few ? 4096 : 8192);
  if (!a.token_ids && !a.bias_ids && on(4)) kvb_logits_kernel<TI, TO, uint16_t, 4><<<grid, 256, 0, s>>>(a);
  else if (few && on(8)) kvb_logits_kernel<TI, TO, uint16_t, 8><<<grid, 256, smem, s>>>(a);
  else if (few) kvb_logits_kernel<TI, TO, uint16_t, 1><<<grid, 256, smem, s>>>(a);
  else if (on(8)) kvb_logits_kernel<TI, TO, uint32_t, 8><<<grid, 256, smem, s>>>(a);
  else kvb_logits_kernel<TI, TO, uint32_t, 1><<<grid, 256, smem, s>>>(a);
}

}  // namespace kvb_step

using kvb_step::aligned;
using kvb_step::fail;

extern "C" int kvb_extend_block_tables(const KvbExtendTablesParams* p, void* stream) {
  if (!p) return fail(KVB_ERR_INVALID, "params is NULL");
  if (p->batch < 1) return fail(KVB_ERR_INVALID, "batch must be >= 1");
  if (p->batch > KVB_MAX_STEP_ROWS)
    return fail(KVB_ERR_UNSUPPORTED, "batch must be <= " + std::to_string(KVB_MAX_STEP_ROWS));
  if (p->block_size != 16) return fail(KVB_ERR_INVALID, "block_size must be 16");
  if (p->max_blocks_per_seq < 1 || p->max_blocks_per_seq > (1 << 27) ||
      p->block_table_stride < p->max_blocks_per_seq)
    return fail(KVB_ERR_INVALID,
                "max_blocks_per_seq must be in [1, 2^27] and block_table_stride at least that");
  if (p->num_blocks < 1 || p->num_blocks > (1 << 27) - 1)
    return fail(KVB_ERR_INVALID, "num_blocks must be in [1, 2^27 - 1] (32-bit slots)");
  if (p->max_new_tokens < 0 || p->free_capacity < 0)
    return fail(KVB_ERR_INVALID, "max_new_tokens and free_capacity must be >= 0");
  if (p->max_new_tokens > (1 << 30) || p->free_capacity > (1 << 30))
    return fail(KVB_ERR_UNSUPPORTED, "max_new_tokens and free_capacity must be <= 2^30");
  if (!p->block_tables || !p->seq_lens || !p->new_lens || !p->num_free || !p->cu_new ||
      !p->seq_lens_out || !p->num_free_out || (p->free_capacity && !p->free_blocks) ||
      (p->max_new_tokens && (!p->slots || !p->positions)))
    return fail(KVB_ERR_INVALID, "arrays must be non-null");
  kvb_step::TablesArgs a = {p->batch, p->max_blocks_per_seq, p->num_blocks, p->max_new_tokens,
                            p->free_capacity, p->block_table_stride, p->block_tables, p->seq_lens,
                            p->new_lens, p->free_blocks, p->num_free, p->slots, p->positions,
                            p->cu_new, p->seq_lens_out, p->num_free_out, p->status};
  // 16-byte stores of slots and positions
  if (!aligned(p->slots, 16) || !aligned(p->positions, 16))
    return fail(KVB_ERR_INVALID, "slots and positions must be 16-byte aligned");
  const int smem = (3 * p->batch + 1) * 4;
  if (smem > 40 * 1024) {
    // the largest batch's limit, once per device: a limit of each call's own could shrink between
    // another thread's setting and its launch
    static std::atomic<uint64_t> ready{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e == cudaSuccess && (dev > 63 || !(ready.load(std::memory_order_acquire) & bit))) {
      e = cudaFuncSetAttribute(kvb_step::kvb_extend_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (3 * KVB_MAX_STEP_ROWS + 1) * 4);
      if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
    }
    if (e != cudaSuccess)
      return fail(KVB_ERR_CUDA, std::string("kvb_extend_block_tables: ") + cudaGetErrorString(e));
  }
  // a decode step of up to 256 rows is one small CTA's scan; long prefills take up to eight
  // CTAs of four tokens a thread
  const int threads = p->batch <= 256 && p->max_new_tokens <= 4096 ? 256 : 1024;
  const int ctas = std::min(8, std::max(1, p->max_new_tokens / (threads * 4)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kvb_step::kvb_extend_tables_kernel, a);
  return kvb_step::launched("kvb_extend_block_tables");
}

extern "C" int kvb_append_paged_kv(const KvbAppendPagedParams* p, void* stream) {
  if (!p) return fail(KVB_ERR_INVALID, "params is NULL");
  if (p->head_dim < 8 || p->head_dim > 256 || p->head_dim % 8)
    return fail(KVB_ERR_INVALID, "head_dim must be a multiple of 8 up to 256");
  if (p->num_kv_heads < 1 || p->num_kv_heads > 65535)
    return fail(KVB_ERR_INVALID, "num_kv_heads must be in [1, 65535]");
  if (p->num_tokens < 0) return fail(KVB_ERR_INVALID, "num_tokens must be >= 0");
  if (p->num_blocks < 1 || p->num_blocks > (1 << 27) - 1)
    return fail(KVB_ERR_INVALID, "num_blocks must be in [1, 2^27 - 1] (32-bit slots)");
  if (p->num_tokens == 0) return KVB_OK;
  if (!p->k_new || !p->v_new || !p->kv_pool || !p->slots)
    return fail(KVB_ERR_INVALID, "k_new, v_new, kv_pool and slots must be non-null");
  if (!aligned(p->k_new, 16) || !aligned(p->v_new, 16) || !aligned(p->kv_pool, 16))
    return fail(KVB_ERR_INVALID, "k_new, v_new and kv_pool must be 16-byte aligned");
  if (p->k_token_stride % 8 || p->k_head_stride % 8 || p->v_token_stride % 8 ||
      p->v_head_stride % 8)
    return fail(KVB_ERR_INVALID, "strides must be multiples of 8 elements");
  const int64_t pool_bytes = (int64_t)p->num_blocks * 2 * p->num_kv_heads * 16 * p->head_dim * 2;
  const auto in_pool = [&](const void* src, int64_t token_stride, int64_t head_stride) {
    const int64_t from = (int64_t)reinterpret_cast<uintptr_t>(src), pool = (int64_t)reinterpret_cast<uintptr_t>(p->kv_pool);
    const int64_t last = (p->num_tokens - 1) * token_stride + (p->num_kv_heads - 1) * head_stride + p->head_dim;
    return from < pool + pool_bytes && pool < from + last * 2;
  };
  if (in_pool(p->k_new, p->k_token_stride, p->k_head_stride) || in_pool(p->v_new, p->v_token_stride, p->v_head_stride))
    return fail(KVB_ERR_INVALID, "k_new and v_new must not overlap kv_pool");
  const int vecs = p->head_dim / 8;
  const int64_t pieces = (int64_t)p->num_tokens * p->num_kv_heads * vecs;
  if (pieces >= (1ll << 31) - 1024 * 256)
    return fail(KVB_ERR_UNSUPPORTED, "too many tokens for one call (2^31 16-byte pieces)");
  kvb_step::AppendArgs a = {kvb_step::Div(p->num_kv_heads * vecs), kvb_step::Div(vecs), (uint32_t)pieces,
                            p->num_kv_heads, p->num_blocks};
  a.src[0] = static_cast<const uint4*>(p->k_new);
  a.src[1] = static_cast<const uint4*>(p->v_new);
  a.token_stride[0] = p->k_token_stride / 8;
  a.token_stride[1] = p->v_token_stride / 8;
  a.head_stride[0] = p->k_head_stride / 8;
  a.head_stride[1] = p->v_head_stride / 8;
  a.pool = static_cast<uint4*>(p->kv_pool);
  a.slots = p->slots;
  a.status = p->status;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  kvb_step::kvb_append_paged_kernel<<<(unsigned)((pieces + 255) / 256), 256, 0, s>>>(a);
  return kvb_step::launched("kvb_append_paged_kv");
}

extern "C" int kvb_process_logits(const KvbLogitsParams* p, void* stream) {
  if (!p) return fail(KVB_ERR_INVALID, "params is NULL");
  if (p->dtype < KVB_DTYPE_BF16 || p->dtype > KVB_DTYPE_FP32)
    return fail(KVB_ERR_INVALID, "dtype must be KVB_DTYPE_BF16, KVB_DTYPE_FP16 or KVB_DTYPE_FP32");
  if (p->out_dtype != p->dtype && p->out_dtype != KVB_DTYPE_FP32)
    return fail(KVB_ERR_INVALID, "out_dtype must be KVB_DTYPE_FP32 or dtype");
  if (p->batch < 0 || p->vocab < 1 || p->history_len < 0 || p->num_bias < 0)
    return fail(KVB_ERR_INVALID, "batch, history_len and num_bias must be >= 0, vocab >= 1");
  if (p->batch > 65535) return fail(KVB_ERR_UNSUPPORTED, "batch must be <= 65535");
  if (p->vocab > (1 << 30)) return fail(KVB_ERR_UNSUPPORTED, "vocab must be <= 2^30");
  if (p->batch == 0) return KVB_OK;
  if (!p->logits || !p->out) return fail(KVB_ERR_INVALID, "logits and out must be non-null");
  const size_t el_in = p->dtype == KVB_DTYPE_FP32 ? 4 : 2;
  const size_t el_out = p->out_dtype == KVB_DTYPE_FP32 ? 4 : 2;
  if (!aligned(p->logits, el_in) || !aligned(p->out, el_out))
    return fail(KVB_ERR_INVALID, "logits and out must be aligned to their element");
  if (p->batch > 1 && (p->logits_stride < p->vocab || p->out_stride < p->vocab))
    return fail(KVB_ERR_INVALID, "row strides must be >= vocab");
  if (p->logits == p->out && (p->dtype != p->out_dtype || p->logits_stride != p->out_stride))
    return fail(KVB_ERR_INVALID, "processing in place needs the logits' dtype and stride");
  if (p->logits != p->out &&
      kvb_step::rows_meet(p->logits, p->vocab * (int64_t)el_in, p->logits_stride * (int64_t)el_in, p->out,
                          p->vocab * (int64_t)el_out, p->out_stride * (int64_t)el_out, p->batch))
    return fail(KVB_ERR_INVALID, "out must be the logits themselves or not overlap them");
  if (p->token_ids && (!p->total_lens || p->history_stride < p->history_len))
    return fail(KVB_ERR_INVALID, "token_ids needs total_lens and history_stride >= history_len");
  if (!p->token_ids && (p->repetition_penalty || p->frequency_penalty || p->presence_penalty))
    return fail(KVB_ERR_INVALID, "penalties need token_ids");
  if (p->num_bias && (!p->bias_ids || !p->bias_values))
    return fail(KVB_ERR_INVALID, "bias_ids and bias_values must be non-null");
  if (p->allowed_mask && p->mask_stride < (p->vocab + 31) / 32)
    return fail(KVB_ERR_INVALID, "mask_stride must be >= ceil(vocab / 32)");
  kvb_step::LogitsArgs a = {};
  a.vocab = p->vocab;
  a.history_len = p->history_len;
  a.num_bias = p->num_bias;
  a.logits = p->logits;
  a.out = p->out;
  a.logits_stride = p->logits_stride;
  a.out_stride = p->out_stride;
  a.history_stride = p->history_stride;
  a.mask_stride = p->mask_stride;
  a.token_ids = p->history_len ? p->token_ids : nullptr;
  a.prompt_lens = p->prompt_lens;
  a.total_lens = p->total_lens;
  a.repetition = p->repetition_penalty;
  a.frequency = p->frequency_penalty;
  a.presence = p->presence_penalty;
  a.temperature = p->temperature;
  a.bias_ids = p->num_bias ? p->bias_ids : nullptr;
  a.bias_values = p->bias_values;
  a.mask = p->allowed_mask;
  const bool f32 = p->out_dtype == KVB_DTYPE_FP32;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  using bf16 = __nv_bfloat16;
  if (p->dtype == KVB_DTYPE_FP32) kvb_step::launch_logits<float, float>(a, p->batch, s);
  else if (p->dtype == KVB_DTYPE_FP16 && f32) kvb_step::launch_logits<__half, float>(a, p->batch, s);
  else if (p->dtype == KVB_DTYPE_FP16) kvb_step::launch_logits<__half, __half>(a, p->batch, s);
  else if (f32) kvb_step::launch_logits<bf16, float>(a, p->batch, s);
  else kvb_step::launch_logits<bf16, bf16>(a, p->batch, s);
  return kvb_step::launched("kvb_process_logits");
}

extern "C" int kvb_new_status(int32_t** status) {
  if (!status) return fail(KVB_ERR_INVALID, "status must be non-null");
  *status = nullptr;
  // a thread that captures may neither allocate nor wait for other streams unless it says so
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) return fail(KVB_ERR_CUDA, std::string("kvb_new_status: ") + cudaGetErrorString(e));
  int32_t* word = nullptr;
  cudaStream_t s = nullptr;
  e = cudaMalloc(&word, sizeof(*word));
  if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking);
  if (e == cudaSuccess) e = cudaMemsetAsync(word, 0, sizeof(*word), s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (s) cudaStreamDestroy(s);
  if (e != cudaSuccess && word) cudaFree(word);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) return fail(KVB_ERR_CUDA, std::string("kvb_new_status: ") + cudaGetErrorString(e));
  *status = word;
  return KVB_OK;
}
