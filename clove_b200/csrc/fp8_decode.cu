// Decode over the 8-bit cache.
//
// One CTA per (sequence, KV head).  Its warps take the tokens in turn; a
// warp's lanes split head_dim, and each warp keeps the running maximum m, sum
// l and weighted value sum of an online softmax for every query head of the
// group (f32, log2 domain).  The warps' states are merged at the end.  With
// accumulate, a second pass over K turns the scores into weights.
#include <algorithm>

#include "fp8_common.cuh"

namespace clove {

struct Fp8DecodeArgs {
  const void* q;
  const unsigned char* codes;
  const float* scales;
  float* mass;
  const int32_t* block_tables;
  const int32_t* context_lens;
  const float* slopes;
  float* out;
  int32_t* flags;
  size_t plane_bytes;
  int bt_stride, num_kv_heads, num_blocks, block_size, max_ctx, group, append, window, accumulate;
  float scale, softcap;
};

__device__ __forceinline__ float fp8_score(const Fp8DecodeArgs& a, float dot, int hq, int back) {
  float z = dot * a.scale;
  if (a.softcap > 0.f) z = a.softcap * tanhf(z / a.softcap);
  if (a.slopes != nullptr) z -= __ldg(a.slopes + hq) * (float)back;
  return z * kLog2e;
}

constexpr int kDecThreads = 128, kDecWarps = kDecThreads / 32;

template <typename T, int D>
__global__ void __launch_bounds__(kDecThreads) fp8_decode_kernel(const Fp8DecodeArgs a) {
  constexpr int E = D / 32;
  __shared__ float qs[8][D];
  __shared__ float st[kDecWarps][8][D + 2];
  __shared__ float fin[8][2];
  const int h = blockIdx.x, b = blockIdx.y, H = a.num_kv_heads, G = a.group, bs = a.block_size;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int ctx = __ldg(a.context_lens + b);
  if (ctx < 0 || ctx > a.max_ctx - a.append) {
    if (h == 0 && tid == 0) atomicOr(a.flags, CLOVE_FLAG_CTX_RANGE);
    ctx = max(0, min(ctx, a.max_ctx - a.append));
  }
  const int L = ctx + a.append, t0 = a.window > 0 ? max(0, L - a.window) : 0;
  float* out = a.out + ((size_t)b * H + h) * G * D;
  if (L == 0) {
    for (int i = tid; i < G * D; i += kDecThreads) out[i] = 0.f;
    return;
  }
  const T* q = static_cast<const T*>(a.q) + ((size_t)b * H + h) * G * D;
  for (int i = tid; i < G * D; i += kDecThreads) qs[i / D][i % D] = Elem<T>::to_f(q[i]);
  __syncthreads();
  const int32_t* table = a.block_tables + (size_t)b * a.bt_stride;
  auto tile_of = [&](int t) {
    int blk = __ldg(table + t / bs);
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0) atomicOr(a.flags, CLOVE_FLAG_BLOCK_OOB);
      blk = 0;
    }
    return (size_t)blk * H + h;
  };
  auto load = [&](int p, size_t tile, int t, float (&x)[E]) {
    const unsigned char* c = a.codes + p * a.plane_bytes + (tile * bs + t % bs) * D + lane * E;
    const float s = a.scales[(size_t)p * a.num_blocks * H + tile];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 f = __half22float2(fp8_unpack2(*reinterpret_cast<const uint16_t*>(c + e)));
      x[e] = f.x * s;
      x[e + 1] = f.y * s;
    }
  };
  float m[8], l[8], acc[8][E];
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[g][e] = 0.f;
  }
  for (int t = t0 + warp; t < L; t += kDecWarps) {
    const size_t tile = tile_of(t);
    float k[E], v[E];
    load(0, tile, t, k);
    load(1, tile, t, v);
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      if (g >= G) break;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(qs[g][lane * E + e], k[e], s);
      s = fp8_score(a, warp_sum(s), h * G + g, L - 1 - t);
      const float mn = fmaxf(m[g], s), c = exp2f(m[g] - mn), w = exp2f(s - mn);
      m[g] = mn;
      l[g] = l[g] * c + w;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] = fmaf(acc[g][e], c, w * v[e]);
    }
  }
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    if (g >= G) break;
#pragma unroll
    for (int e = 0; e < E; ++e) st[warp][g][lane * E + e] = acc[g][e];
    if (lane == 0) {
      st[warp][g][D] = m[g];
      st[warp][g][D + 1] = l[g];
    }
  }
  __syncthreads();
  for (int g = warp; g < G; g += kDecWarps) {
    float M = -INFINITY, lsum = 0.f, o[E] = {};
    for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, st[w][g][D]);
    for (int w = 0; w < kDecWarps; ++w) {
      const float f = st[w][g][D] == -INFINITY ? 0.f : exp2f(st[w][g][D] - M);
      lsum = fmaf(f, st[w][g][D + 1], lsum);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(f, st[w][g][lane * E + e], o[e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) out[g * D + lane * E + e] = o[e] / lsum;
    if (lane == 0) {
      fin[g][0] = M;
      fin[g][1] = 1.f / lsum;
    }
  }
  if (!a.accumulate) return;
  __syncthreads();
  for (int t = t0 + warp; t < L; t += kDecWarps) {
    const size_t tile = tile_of(t);
    float k[E], w = 0.f;
    load(0, tile, t, k);
    for (int g = 0; g < G; ++g) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(qs[g][lane * E + e], k[e], s);
      s = fp8_score(a, warp_sum(s), h * G + g, L - 1 - t);
      w = fmaf(exp2f(s - fin[g][0]), fin[g][1], w);
    }
    if (lane == 0) a.mass[tile * bs + t % bs] += w;
  }
}

// The slots of the new tokens (-1 where the table has no block for one).
__global__ void fp8_slots_kernel(const int32_t* block_tables, int bt_stride, const int32_t* context_lens, int batch,
                                 int max_ctx, int block_size, int num_blocks, int32_t* slots, int32_t* flags) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= batch) return;
  const int ctx = max(0, min(context_lens[b], max_ctx - 1));
  const int blk = block_tables[(size_t)b * bt_stride + ctx / block_size];
  if (blk < 0 || blk >= num_blocks) {
    atomicOr(flags, CLOVE_FLAG_BLOCK_OOB);
    slots[b] = -1;
  } else {
    slots[b] = blk * block_size + ctx % block_size;
  }
}

size_t fp8_decode_workspace(const clove_fp8_pool&, int batch, int, int, int) { return sizeof(int32_t) * (size_t)batch; }

template <typename T>
static cudaError_t run_decode(const Fp8DecodeArgs& a, int head_dim, int batch, cudaStream_t stream) {
  const dim3 grid(a.num_kv_heads, batch);
  switch (head_dim) {
    case 64: fp8_decode_kernel<T, 64><<<grid, kDecThreads, 0, stream>>>(a); break;
    case 128: fp8_decode_kernel<T, 128><<<grid, kDecThreads, 0, stream>>>(a); break;
    default: fp8_decode_kernel<T, 256><<<grid, kDecThreads, 0, stream>>>(a); break;
  }
  return cudaGetLastError();
}

int launch_fp8_decode(const clove_fp8_pool& pool, const Fp8DecodeCall& c, cudaStream_t stream) {
  if (c.k_new) {
    int32_t* slots = static_cast<int32_t*>(c.workspace);
    fp8_slots_kernel<<<(c.batch + 255) / 256, 256, 0, stream>>>(c.block_tables, c.bt_stride, c.context_lens, c.batch,
                                                                c.max_ctx, pool.block_size, pool.num_blocks, slots,
                                                                pool.flags);
    int rc = fp8_launch_status("fp8_decode slots launch", cudaGetLastError());
    if (rc) return rc;
    count_launches(1);
    rc = launch_fp8_append(pool, c.dtype, c.k_new, c.v_new, slots, c.batch, nullptr, stream);
    if (rc) return rc;
  }
  Fp8DecodeArgs a;
  a.q = c.q;
  a.codes = pool.codes;
  a.scales = pool.scales;
  a.mass = pool.mass;
  a.block_tables = c.block_tables;
  a.context_lens = c.context_lens;
  a.slopes = c.scores.alibi_slopes;
  a.out = c.out;
  a.flags = pool.flags;
  a.plane_bytes = pool.plane_bytes;
  a.bt_stride = c.bt_stride;
  a.num_kv_heads = pool.num_kv_heads;
  a.num_blocks = pool.num_blocks;
  a.block_size = pool.block_size;
  a.max_ctx = c.max_ctx;
  a.group = c.num_q_heads / pool.num_kv_heads;
  a.append = c.k_new ? 1 : 0;
  a.window = c.scores.window;
  a.accumulate = c.scores.accumulate;
  a.scale = c.scale;
  a.softcap = c.scores.softcap;
  cudaError_t e;
  switch (c.dtype) {
    case CLOVE_DTYPE_F32: e = run_decode<float>(a, pool.head_dim, c.batch, stream); break;
    case CLOVE_DTYPE_F16: e = run_decode<__half>(a, pool.head_dim, c.batch, stream); break;
    default: e = run_decode<__nv_bfloat16>(a, pool.head_dim, c.batch, stream); break;
  }
  count_launches(1);
  return fp8_launch_status("fp8_decode launch", e);
}

}  // namespace clove
