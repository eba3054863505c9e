// kvb_paged_decode_fwd: attention of one new token per request over its blocks of the
// pool, sm_100a.  O = softmax(q K^T s) V with GQA; the blocks are read in place.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "kvb_attn.h"

int kvb_detail_fail(int code, const std::string& msg);

namespace kvb_pd {

int fail(int code, const std::string& msg) { return kvb_detail_fail(code, msg); }

struct Args {
  int num_q_heads, num_kv_heads, num_blocks, width;
  float scale;
  const void* q;
  void* o;
  float* lse;
  int64_t q_bs, q_hs, o_bs, o_hs, lse_bs, table_stride;
  const void* pool;
  const __half* k_scale;
  const __half* v_scale;
  const int32_t* tables;
  const int32_t* lens;
  int32_t* status;
};

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(int8_t x) { return (float)x; }
__device__ __forceinline__ void from_f32(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// One CTA per (query head, request): 8 warps take tokens in turn, a lane holds D / 32
// features; running maximum and sum per warp, joined at the end.
template <typename T, typename P, int D>
__global__ void __launch_bounds__(256) kvb_paged_decode_kernel(const Args a) {
  constexpr int N = D / 32;
  __shared__ float sm_m[8], sm_l[8], sm_o[8][D];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kvh = h / (a.num_q_heads / a.num_kv_heads);
  int len = a.lens[b];
  if (len > a.width * 16) {
    len = a.width * 16;
    if (a.status && threadIdx.x == 0) atomicOr(a.status, KVB_STATUS_BAD_LENGTH);
  }
  float q[N], o[N];
  const T* qp = static_cast<const T*>(a.q) + b * a.q_bs + h * a.q_hs;
  for (int i = 0; i < N; ++i) q[i] = to_f32(qp[i * 32 + lane]) * a.scale, o[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int t = warp; t < len; t += 8) {
    const int id = a.tables[b * a.table_stride + (t >> 4)];
    const bool ok = id >= 0 && id < a.num_blocks;
    if (!ok && a.status) atomicOr(a.status, KVB_STATUS_BAD_BLOCK);
    float x = 0.f, v[N];
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    if (ok) {
      const int64_t at = ((int64_t)id * 2 * a.num_kv_heads + kvh) * 16 + (t & 15);
      const P* kp = static_cast<const P*>(a.pool) + at * D;
      const P* vp = kp + (int64_t)a.num_kv_heads * 16 * D;
      for (int i = 0; i < N; ++i) x += q[i] * to_f32(kp[i * 32 + lane]);
      for (int s = 16; s; s >>= 1) x += __shfl_xor_sync(~0u, x, s);
      const int64_t bh = (int64_t)id * a.num_kv_heads + kvh;
      if (a.k_scale) x *= __half2float(a.k_scale[bh * 16 + (t & 15)]);
      for (int i = 0; i < N; ++i) {
        v[i] = to_f32(vp[i * 32 + lane]);
        if (a.v_scale) v[i] *= __half2float(a.v_scale[bh * D + i * 32 + lane]);
      }
    }
    const float mn = fmaxf(m, x), base = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - base), p = expf(x - base);
    m = mn;
    l = l * f + p;
    for (int i = 0; i < N; ++i) o[i] = o[i] * f + p * v[i];
  }
  if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
  for (int i = 0; i < N; ++i) sm_o[warp][i * 32 + lane] = o[i];
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < 8; ++w) top = fmaxf(top, sm_m[w]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int w = 0; w < 8; ++w) total += sm_l[w] * expf(sm_m[w] - base);
  T* op = static_cast<T*>(a.o) + b * a.o_bs + h * a.o_hs;
  for (int d = threadIdx.x; d < D; d += 256) {
    float s = 0.f;
    for (int w = 0; w < 8; ++w) s += sm_o[w][d] * expf(sm_m[w] - base);
    from_f32(op + d, len > 0 ? s / total : 0.f);
  }
  if (a.lse && threadIdx.x == 0) a.lse[b * a.lse_bs + h] = len > 0 ? base + logf(total) : -INFINITY;
}

template <typename T, typename P>
void* pick(int D) {
  return D == 64 ? (void*)kvb_paged_decode_kernel<T, P, 64>
                 : D == 96 ? (void*)kvb_paged_decode_kernel<T, P, 96>
                           : (void*)kvb_paged_decode_kernel<T, P, 128>;
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

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
  if (p->max_blocks_per_seq < 1 || p->max_blocks_per_seq > (1 << 27) - 1 ||
      p->block_table_stride < p->max_blocks_per_seq)
    return fail(KVB_ERR_INVALID,
                "max_blocks_per_seq must be in [1, 2^27 - 1] and block_table_stride at least that");
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
  return KVB_OK;
}

}  // namespace kvb_pd

extern "C" int64_t kvb_paged_decode_workspace_bytes(const KvbPagedDecodeParams* p) {
  if (kvb_pd::check(p) != KVB_OK) return -1;
  return 0;
}

extern "C" int kvb_paged_decode_fwd(const KvbPagedDecodeParams* p, void* stream) {
  if (const int rc = kvb_pd::check(p)) return rc;
  if (p->batch == 0) return KVB_OK;
  kvb_pd::Args a = {};
  a.num_q_heads = p->num_q_heads;
  a.num_kv_heads = p->num_kv_heads;
  a.num_blocks = p->num_blocks;
  a.width = p->max_blocks_per_seq;
  a.scale = p->softmax_scale;
  a.q = p->q;
  a.o = p->o;
  a.lse = p->lse;
  a.q_bs = p->q_batch_stride;
  a.q_hs = p->q_head_stride;
  a.o_bs = p->o_batch_stride;
  a.o_hs = p->o_head_stride;
  a.lse_bs = p->lse_batch_stride;
  a.table_stride = p->block_table_stride;
  a.pool = p->kv_pool;
  const bool int8 = p->pool_format == KVB_POOL_INT8_KIVI;
  a.k_scale = int8 ? static_cast<const __half*>(p->k_scale16) : nullptr;
  a.v_scale = int8 ? static_cast<const __half*>(p->v_scale16) : nullptr;
  a.tables = p->block_tables;
  a.lens = p->seq_lens;
  a.status = p->status;
  void* kern = p->dtype == KVB_DTYPE_BF16
                   ? (int8 ? kvb_pd::pick<__nv_bfloat16, int8_t>(p->head_dim)
                           : kvb_pd::pick<__nv_bfloat16, __nv_bfloat16>(p->head_dim))
                   : (int8 ? kvb_pd::pick<__half, int8_t>(p->head_dim)
                           : kvb_pd::pick<__half, __half>(p->head_dim));
  void* args[] = {&a};
  const cudaError_t e = cudaLaunchKernel(kern, dim3(p->num_q_heads, p->batch), dim3(256), args, 0,
                                         static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess)
    return kvb_pd::fail(KVB_ERR_CUDA, std::string("kvb_paged_decode_fwd launch: ") + cudaGetErrorString(e));
  return KVB_OK;
}
