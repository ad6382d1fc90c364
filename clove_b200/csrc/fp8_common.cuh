// Shared pieces of the 8-bit cache kernels: the pool handle, the scale rule
// and the e4m3 conversions.
#pragma once

#include <cuda_fp8.h>

#include <mutex>

#include "../../include/clove_fp8.h"
#include "common.cuh"
#include "host.h"

struct clove_fp8_pool {
  int device;
  int num_blocks;
  int block_size;
  int num_kv_heads;
  int head_dim;
  int owns_memory;
  unsigned char* codes;  // [2, num_blocks, num_kv_heads, block_size, head_dim]
  float* scales;         // [2, num_blocks, num_kv_heads]
  float* mass;           // [num_blocks, num_kv_heads, block_size] or null
  size_t plane_bytes;    // bytes of one plane of codes
  int32_t* flags;        // device words: check flags of all calls; those that the last status call took off
  std::mutex status_lock;  // held while a status call takes flags off
  int32_t* slot_token;   // append index: a word per slot, then one per block; zero between calls
  int num_sms;
  CUtensorMap map;  // the codes as the decode's copies see them
};

namespace clove {

// 2^e, e >= -126 the smallest with amax <= 448 * 2^e (448 = 1.75 * 2^8, the
// largest e4m3 value): from the bits of amax = 1.m * 2^E, e = E - 8, one more
// when 1.m > 1.75.  amax is finite and >= 0.
__device__ __forceinline__ float fp8_scale_for(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return __int_as_float((max(e, -126) + 127) << 23);
}

// |x| where it is finite, else 0 (infinities and NaN do not count towards a scale).
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// Two floats -> two e4m3 bytes, round to nearest even, +-448 beyond; NaN stays NaN.
__device__ __forceinline__ uint32_t fp8_pack2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ uint2 fp8_pack8(const float (&x)[8]) {
  return make_uint2(fp8_pack2(x[0], x[1]) | fp8_pack2(x[2], x[3]) << 16,
                    fp8_pack2(x[4], x[5]) | fp8_pack2(x[6], x[7]) << 16);
}

// Two e4m3 bytes (the low 16 bits) -> two halves, exact.
__device__ __forceinline__ __half2 fp8_unpack2(uint32_t w) {
  return __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3));
}

__device__ __forceinline__ void fp8_unpack4(uint32_t w, float* o) {
  const float2 a = __half22float2(fp8_unpack2(w)), b = __half22float2(fp8_unpack2(w >> 16));
  o[0] = a.x;
  o[1] = a.y;
  o[2] = b.x;
  o[3] = b.y;
}

__device__ __forceinline__ void fp8_unpack8(uint2 w, float (&o)[8]) {
  fp8_unpack4(w.x, o);
  fp8_unpack4(w.y, o + 4);
}

// Round 8 codes to a scale 1 / ratio times as large.
__device__ __forceinline__ uint2 fp8_rescale8(uint2 w, float ratio) {
  float x[8];
  fp8_unpack8(w, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= ratio;
  return fp8_pack8(x);
}

// ---- launchers (host) -----------------------------------------------------
struct Fp8AppendArgs {
  const void* x[2];  // k, v rows [tokens, heads, dim]
  const int32_t* slots;
  unsigned char* codes;
  float* scales;
  float* mass;
  int32_t* flags;
  int32_t* slot_token;   // the pool's append index
  int32_t* block_state;
  int32_t* leads;        // [tokens] workspace
  size_t plane_bytes;
  int num_tokens, num_blocks, block_size, num_kv_heads;
};

struct Fp8DecodeCall {
  int dtype;
  const void* q;
  const void* k_new;  // null: plain decode
  const void* v_new;
  int num_q_heads;
  const int32_t* block_tables;
  int bt_stride;
  const int32_t* context_lens;
  int batch;
  float scale;
  int max_ctx;
  clove_fp8_scores_t scores;
  float* out;
  void* workspace;
};

struct Fp8EvictCall {
  const int32_t* block_tables;
  int bt_stride;
  const int32_t* context_lens;
  int batch;
  int max_ctx;
  const int32_t* new_tables;
  int new_stride;
  int budget, recent;
  int32_t* kept;
  int32_t* new_lens;
};

// Each returns a CLOVE_* status and sets the last-error text on failure.
size_t fp8_append_workspace(const clove_fp8_pool& pool, int num_tokens);
int launch_fp8_append(const clove_fp8_pool& pool, int dtype, const void* k, const void* v, const int32_t* slots,
                      int num_tokens, void* workspace, cudaStream_t stream);
int launch_fp8_gather(const clove_fp8_pool& pool, const int32_t* block_tables, int bt_stride,
                      const int32_t* context_lens, int batch, int max_ctx, float* k_out, float* v_out,
                      cudaStream_t stream);
int launch_fp8_copy(const clove_fp8_pool& pool, const int32_t* src, const int32_t* dst, int n, cudaStream_t stream);
int fp8_encode_map(clove_fp8_pool& pool);
size_t fp8_decode_workspace(const clove_fp8_pool& pool, int batch, int num_q_heads, int max_ctx, int accumulate);
int launch_fp8_decode(const clove_fp8_pool& pool, const Fp8DecodeCall& call, cudaStream_t stream);
size_t fp8_evict_workspace(const clove_fp8_pool& pool, int batch, int max_ctx, int budget);
int launch_fp8_evict(const clove_fp8_pool& pool, const Fp8EvictCall& call, cudaStream_t stream);

inline int fp8_launch_status(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return CLOVE_OK;
  set_last_error("%s: %s", what, cudaGetErrorString(e));
  return CLOVE_ERR_CUDA;
}

}  // namespace clove
