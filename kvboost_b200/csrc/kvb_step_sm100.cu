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

#include <cstdint>
#include <string>

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

// One CTA: a scan over the rows gives each row's place in the packed arrays and in the
// free list, then one thread per token writes its slot, its position and, for the first
// token of a new block, the table entry.
__global__ void __launch_bounds__(1024) kvb_extend_tables_kernel(const TablesArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* cu = sm;                        // [batch + 1] place of the row's tokens
  int32_t* start = cu + a.batch + 1;       // [batch] pops before the row's, -1: does not fit
  int32_t* len = start + a.batch;          // [batch]
  __shared__ int64_t wsum[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nt = blockDim.x;
  const int nfree = min(max(*a.num_free, 0), a.capacity);
  int64_t base_tok = 0, base_need = 0;
  int err = 0;
  for (int b0 = 0; b0 < a.batch; b0 += nt) {
    const int b = b0 + tid;
    int l = 0, n = 0;
    bool ok = false;
    if (b < a.batch) {
      l = a.seq_lens[b];
      n = a.new_lens[b];
      ok = l >= 0 && n >= 0 && n <= a.max_tokens;
      if (!ok) {
        err |= KVB_STATUS_BAD_LENGTH;
        n = 0;
      }
    }
    const bool wide = ok && (int64_t)l + n <= (int64_t)a.width * 16;
    if (ok && !wide) err |= KVB_STATUS_BAD_LENGTH;
    const int64_t end0 = n;
    int64_t need = wide ? ((int64_t)l + n + 15) / 16 - ((int64_t)l + 15) / 16 : 0;
    // inclusive scans of tokens and needs over the CTA
    int64_t t_in = end0;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(~0u, t_in, o);
      if (lane >= o) t_in += x;
    }
    if (lane == 31) wsum[0][warp] = t_in;
    __syncthreads();
    int64_t tot_tok = 0;
    for (int w = 0; w < (nt >> 5); ++w) {
      if (w < warp) t_in += wsum[0][w];
      tot_tok += wsum[0][w];
    }
    const int64_t tok_end = base_tok + t_in;
    const bool packed = wide && (n == 0 || tok_end <= a.max_tokens);
    if (wide && !packed) {
      err |= KVB_STATUS_BAD_LENGTH;
      need = 0;
    }
    int64_t n_in = need;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(~0u, n_in, o);
      if (lane >= o) n_in += x;
    }
    if (lane == 31) wsum[1][warp] = n_in;
    __syncthreads();
    int64_t tot_need = 0;
    for (int w = 0; w < (nt >> 5); ++w) {
      if (w < warp) n_in += wsum[1][w];
      tot_need += wsum[1][w];
    }
    const int64_t need_end = base_need + n_in;
    const bool fits = packed && (need == 0 || need_end <= nfree);
    if (packed && !fits) err |= KVB_STATUS_POOL_EMPTY;
    if (b < a.batch) {
      cu[b + 1] = (int32_t)min(tok_end, (int64_t)a.max_tokens);
      start[b] = fits ? (int32_t)(need_end - need) : -1;
      len[b] = l;
    }
    base_tok += tot_tok;
    base_need += tot_need;
    __syncthreads();
  }
  if (tid == 0) cu[0] = 0;
  __syncthreads();
  // every read of seq_lens and num_free is done: the outputs may alias them
  if (tid == 0) a.cu_new[0] = 0;
  int taken = 0;
  for (int b = tid; b < a.batch; b += nt) {
    const int n = cu[b + 1] - cu[b], l = len[b];
    a.cu_new[b + 1] = cu[b + 1];
    a.seq_lens_out[b] = start[b] >= 0 ? l + n : l;
    if (start[b] >= 0) taken += (l + n + 15) / 16 - (l + 15) / 16;
  }
  for (int o = 16; o; o >>= 1) taken += __shfl_xor_sync(~0u, taken, o);
  if (lane == 0) wsum[0][warp] = taken;
  __syncthreads();
  if (tid == 0) {
    int64_t t = 0;
    for (int w = 0; w < (nt >> 5); ++w) t += wsum[0][w];
    *a.num_free_out = nfree - (int)t;
  }
  const int total = cu[a.batch];
  for (int t = tid; t < a.max_tokens; t += nt) {
    int slot = -1;
    int64_t pos = 0;
    if (t < total) {
      int lo = 0, hi = a.batch - 1;   // the row with cu[row] <= t < cu[row + 1]
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid + 1] <= t) lo = mid + 1; else hi = mid;
      }
      const int s = start[lo];
      if (s >= 0) {
        const int l = len[lo], p = l + t - cu[lo], have = (l + 15) >> 4, blk = p >> 4;
        int32_t* row = a.tables + (int64_t)lo * a.stride;
        int id;
        if (blk < have) {
          id = row[blk];
        } else {
          id = a.free_blocks[nfree - 1 - s - (blk - have)];
          if ((p & 15) == 0) row[blk] = id;
        }
        pos = p;
        if (id >= 0 && id < a.num_blocks) slot = id * 16 + (p & 15);
        else err |= KVB_STATUS_BAD_BLOCK;
      }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
  if (err && a.status) atomicOr(a.status, err);
}

// ---- append ---------------------------------------------------------------------------------

struct AppendArgs {
  int vecs, heads, tokens, num_blocks;   // vecs: 16-byte pieces of a head's vector
  const uint4* src[2];
  int64_t token_stride[2], head_stride[2];   // in 16-byte pieces
  uint4* pool;
  const int32_t* slots;
  int32_t* status;
};

// One thread per 16-byte piece; blockIdx.y picks K or V.
__global__ void __launch_bounds__(256) kvb_append_paged_kernel(const AppendArgs a) {
  const int kv = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = a.heads * a.vecs;
  const int64_t t = i / per;
  if (t >= a.tokens) return;
  const int r = (int)(i - t * per), h = r / a.vecs, x = r - h * a.vecs;
  const int slot = a.slots[t];
  if (slot < 0 || slot >= (int64_t)a.num_blocks * 16) {
    if (slot != -1 && r == 0 && kv == 0 && a.status) atomicOr(a.status, KVB_STATUS_BAD_BLOCK);
    return;
  }
  const int64_t row = (((int64_t)(slot >> 4) * 2 + kv) * a.heads + h) * 16 + (slot & 15);
  a.pool[row * a.vecs + x] = a.src[kv][t * a.token_stride[kv] + h * a.head_stride[kv] + x];
}

// ---- logits -----------------------------------------------------------------------------------

struct LogitsArgs {
  int vocab, history_len, num_bias, slice;
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

constexpr uint32_t kHasBias = 1u << 31;   // a seen word: bit 0 seen, bits 1..30 count, bit 31

// A CTA takes one slice of one row: it notes the history's tokens that fall into the slice
// in shared memory (seen bit and count, integer adds: any order gives the same), then
// streams the slice.
template <typename TI, typename TO>
__global__ void __launch_bounds__(256) kvb_logits_kernel(const LogitsArgs a) {
  extern __shared__ uint32_t note[];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int v0 = blockIdx.x * a.slice, v1 = min(a.vocab, v0 + a.slice);
  const int32_t* bias_ids = a.bias_ids ? a.bias_ids + (int64_t)b * a.num_bias : nullptr;
  const bool noted = a.token_ids || bias_ids;
  if (noted) {
    for (int i = tid; i < v1 - v0; i += 256) note[i] = 0;
    __syncthreads();
    if (a.token_ids) {
      const int total = min(max(a.total_lens[b], 0), a.history_len);
      const int prompt = a.prompt_lens ? min(max(a.prompt_lens[b], 0), total) : 0;
      const int32_t* ids = a.token_ids + (int64_t)b * a.history_stride;
      for (int i = tid; i < total; i += 256) {
        const int id = ids[i];
        if (id >= v0 && id < v1) {
          if (i < prompt) atomicOr(&note[id - v0], 1u);
          else atomicAdd(&note[id - v0], 2u);
        }
      }
    }
    if (bias_ids) {
      __syncthreads();
      for (int i = tid; i < a.num_bias; i += 256) {
        const int id = bias_ids[i];
        if (id >= v0 && id < v1) atomicOr(&note[id - v0], kHasBias);
      }
    }
    __syncthreads();
  }
  const float r = a.repetition ? a.repetition[b] : 1.f;
  const float freq = a.frequency ? a.frequency[b] : 0.f;
  const float pres = a.presence ? a.presence[b] : 0.f;
  const float temp = a.temperature ? fmaxf(a.temperature[b], 1e-5f) : 1.f;
  const TI* in = static_cast<const TI*>(a.logits) + (int64_t)b * a.logits_stride;
  TO* out = static_cast<TO*>(a.out) + (int64_t)b * a.out_stride;
  for (int v = v0 + tid; v < v1; v += 256) {
    float x = to_f32(in[v]);
    const uint32_t n = noted ? note[v - v0] : 0;
    if (n) {
      const uint32_t count = (n & ~kHasBias) >> 1;
      if ((n & ~kHasBias) && a.repetition) x = x > 0.f ? x / r : x * r;
      if (count) x = x - freq * (float)count - pres;
      if (n & kHasBias)
        for (int i = 0; i < a.num_bias; ++i)
          if (bias_ids[i] == v) x += a.bias_values[(int64_t)b * a.num_bias + i];
    }
    x = x / temp;
    if (a.mask && !((a.mask[(int64_t)b * a.mask_stride + (v >> 5)] >> (v & 31)) & 1))
      x = __uint_as_float(0xff800000u);
    from_f32(out + v, x);
  }
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
  if (!p->block_tables || !p->seq_lens || !p->new_lens || !p->num_free || !p->cu_new ||
      !p->seq_lens_out || !p->num_free_out || (p->free_capacity && !p->free_blocks) ||
      (p->max_new_tokens && (!p->slots || !p->positions)))
    return fail(KVB_ERR_INVALID, "arrays must be non-null");
  kvb_step::TablesArgs a = {p->batch, p->max_blocks_per_seq, p->num_blocks, p->max_new_tokens,
                            p->free_capacity, p->block_table_stride, p->block_tables, p->seq_lens,
                            p->new_lens, p->free_blocks, p->num_free, p->slots, p->positions,
                            p->cu_new, p->seq_lens_out, p->num_free_out, p->status};
  const int smem = (3 * p->batch + 1) * 4;
  if (smem > 40 * 1024)
    cudaFuncSetAttribute(kvb_step::kvb_extend_tables_kernel,
                         cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  kvb_step::kvb_extend_tables_kernel<<<1, 1024, smem, static_cast<cudaStream_t>(stream)>>>(a);
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
  kvb_step::AppendArgs a = {};
  a.vecs = p->head_dim / 8;
  a.heads = p->num_kv_heads;
  a.tokens = p->num_tokens;
  a.num_blocks = p->num_blocks;
  a.src[0] = static_cast<const uint4*>(p->k_new);
  a.src[1] = static_cast<const uint4*>(p->v_new);
  a.token_stride[0] = p->k_token_stride / 8;
  a.token_stride[1] = p->v_token_stride / 8;
  a.head_stride[0] = p->k_head_stride / 8;
  a.head_stride[1] = p->v_head_stride / 8;
  a.pool = static_cast<uint4*>(p->kv_pool);
  a.slots = p->slots;
  a.status = p->status;
  const int64_t pieces = (int64_t)p->num_tokens * p->num_kv_heads * a.vecs;
  const int64_t ctas = (pieces + 255) / 256;
  if (ctas > 0x7fffffff) return fail(KVB_ERR_UNSUPPORTED, "too many tokens for one call");
  kvb_step::kvb_append_paged_kernel<<<dim3((unsigned)ctas, 2), 256, 0,
                                      static_cast<cudaStream_t>(stream)>>>(a);
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
  a.slice = 4096;
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
  void (*kern)(kvb_step::LogitsArgs) = nullptr;
  const bool f32 = p->out_dtype == KVB_DTYPE_FP32;
  if (p->dtype == KVB_DTYPE_FP32) kern = kvb_step::kvb_logits_kernel<float, float>;
  else if (p->dtype == KVB_DTYPE_FP16)
    kern = f32 ? kvb_step::kvb_logits_kernel<__half, float> : kvb_step::kvb_logits_kernel<__half, __half>;
  else
    kern = f32 ? kvb_step::kvb_logits_kernel<__nv_bfloat16, float>
               : kvb_step::kvb_logits_kernel<__nv_bfloat16, __nv_bfloat16>;
  kern<<<dim3((p->vocab + a.slice - 1) / a.slice, p->batch), 256, a.slice * 4,
         static_cast<cudaStream_t>(stream)>>>(a);
  return kvb_step::launched("kvb_process_logits");
}
