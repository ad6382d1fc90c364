// Eviction by accumulated attention weight.
//
// select    one CTA per (sequence, KV head): radix selection of the weight of
//           the last token kept (8 bits of the key per pass), then an ordered
//           write of the kept indices.
// compact   one CTA per (new block, KV head, sequence): gathers the kept rows
//           into the new block, rounding to its scale where that is larger.
#include <algorithm>

#include "fp8_common.cuh"

namespace clove {

// Ascending order of the float as an unsigned key; NaN above everything.
__device__ __forceinline__ uint32_t mass_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 counts as 0
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

struct Fp8EvictArgs {
  unsigned char* codes;
  float* scales;
  float* mass;
  size_t plane_bytes;
  const int32_t* block_tables;
  const int32_t* context_lens;
  const int32_t* new_tables;
  int32_t* kept;
  int32_t* new_lens;
  int32_t* flags;
  int bt_stride, new_stride, max_ctx, budget, recent, num_blocks, block_size, num_kv_heads;
};

__device__ __forceinline__ int evict_len(const Fp8EvictArgs& a, int b) {
  return max(0, min(__ldg(a.context_lens + b), a.max_ctx));
}

constexpr int kSelThreads = 1024;

__device__ __forceinline__ int block_scan(int x, int* warp_tot, int* total) {  // exclusive
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();
  if (lane == 31) warp_tot[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int w = lane < kSelThreads / 32 ? warp_tot[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_tot[lane] = w;
  }
  __syncthreads();
  *total = warp_tot[kSelThreads / 32 - 1];
  return s - x + (warp > 0 ? warp_tot[warp - 1] : 0);
}

__global__ void __launch_bounds__(kSelThreads) fp8_select_kernel(const Fp8EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int warp_tot[32];
  __shared__ int s_digit, s_above;
  const int h = blockIdx.x, b = blockIdx.y, H = a.num_kv_heads, bs = a.block_size, tid = threadIdx.x;
  const int n = evict_len(a, b), m = min(n, a.budget);
  if (h == 0 && tid == 0) {
    a.new_lens[b] = m;
    if (__ldg(a.context_lens + b) != n) atomicOr(a.flags, CLOVE_FLAG_CTX_RANGE);
  }
  int32_t* kept = a.kept + ((size_t)b * H + h) * a.budget;
  for (int i = m + tid; i < a.budget; i += kSelThreads) kept[i] = -1;
  const int last = min(a.recent, n), old = n - last, need = m - last;
  for (int i = tid; i < last; i += kSelThreads) kept[need + i] = old + i;
  if (need == 0) return;
  if (need == old) {
    for (int i = tid; i < need; i += kSelThreads) kept[i] = i;
    return;
  }
  const int32_t* table = a.block_tables + (size_t)b * a.bt_stride;
  auto key = [&](int t) {
    int blk = __ldg(table + t / bs);
    if (blk < 0 || blk >= a.num_blocks) {
      atomicOr(a.flags, CLOVE_FLAG_BLOCK_OOB);
      blk = 0;
    }
    return mass_key(a.mass[((size_t)blk * H + h) * bs + t % bs]);
  };
  // the need-th largest key, 8 bits at a time
  uint32_t prefix = 0;
  int left = need;  // rank of the wanted key among those that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int t = tid; t < old; t += kSelThreads) {
      const uint32_t k = key(t);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    int total;
    const int c = tid < 256 ? hist[255 - tid] : 0;  // from the largest digit down
    const int above = block_scan(c, warp_tot, &total);
    if (tid < 256 && above < left && left <= above + c) {
      s_digit = 255 - tid;
      s_above = above;
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    left -= s_above;
    __syncthreads();
  }
  // keys above the threshold, and the first `left` of those equal to it
  int at = 0, equal = 0;
  for (int base = 0; base < old; base += kSelThreads) {
    const int t = base + tid;
    const uint32_t k = t < old ? key(t) : 0u;
    const int eq = t < old && k == prefix;
    int neq, nkeep;
    const int r = equal + block_scan(eq, warp_tot, &neq);
    const int keep = t < old && (k > prefix || (eq && r < left));
    const int pos = at + block_scan(keep, warp_tot, &nkeep);
    if (keep) kept[pos] = t;
    equal += neq;
    at += nkeep;
  }
}

constexpr int kCompactThreads = 128;

template <int D>
__global__ void __launch_bounds__(kCompactThreads) fp8_compact_kernel(const Fp8EvictArgs a) {
  constexpr int LPR = D / 8;
  __shared__ int row[256];      // source row (tile * block_size + offset) of each new row, -1: bad block
  __shared__ float sc[2][256];  // its scales
  __shared__ float top[2];
  const int j = blockIdx.x, h = blockIdx.y, b = blockIdx.z, H = a.num_kv_heads, bs = a.block_size;
  const int tid = threadIdx.x;
  const int m = min(evict_len(a, b), a.budget), first = j * bs, rows = min(bs, m - first);
  if (rows <= 0) return;
  const int dst = __ldg(a.new_tables + (size_t)b * a.new_stride + j);
  if (dst < 0 || dst >= a.num_blocks) {
    if (tid == 0 && h == 0) atomicOr(a.flags, CLOVE_FLAG_BLOCK_OOB);
    return;
  }
  const size_t to = (size_t)dst * H + h;
  const int32_t* kept = a.kept + ((size_t)b * H + h) * a.budget + first;
  for (int r = tid; r < rows; r += kCompactThreads) {
    const int t = kept[r];
    int blk = __ldg(a.block_tables + (size_t)b * a.bt_stride + t / bs);
    if (blk < 0 || blk >= a.num_blocks) {
      atomicOr(a.flags, CLOVE_FLAG_BLOCK_OOB);
      blk = 0;
    }
    const size_t tile = (size_t)blk * H + h;
    row[r] = (int)(tile * bs) + t % bs;
    sc[0][r] = a.scales[tile];
    sc[1][r] = a.scales[(size_t)a.num_blocks * H + tile];
    a.mass[to * bs + r] = a.mass[tile * bs + t % bs];
  }
  __syncthreads();
  if (tid < 64) {
    float x = 0.f;
    for (int r = tid & 31; r < rows; r += 32) x = fmaxf(x, sc[tid >> 5][r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    if ((tid & 31) == 0) {
      top[tid >> 5] = x;
      a.scales[(size_t)(tid >> 5) * a.num_blocks * H + to] = x;
    }
  }
  __syncthreads();
  for (int i = tid; i < 2 * rows * LPR; i += kCompactThreads) {
    const int p = i / (rows * LPR), k = i - p * rows * LPR, r = k / LPR, w = k - r * LPR;
    unsigned char* plane = a.codes + p * a.plane_bytes;
    uint2 x = *reinterpret_cast<const uint2*>(plane + (size_t)row[r] * D + w * 8);
    if (sc[p][r] != top[p]) x = fp8_rescale8(x, sc[p][r] / top[p]);
    *reinterpret_cast<uint2*>(plane + (to * bs + r) * D + w * 8) = x;
  }
}

size_t fp8_evict_workspace(const clove_fp8_pool&, int, int, int) { return 0; }

int launch_fp8_evict(const clove_fp8_pool& pool, const Fp8EvictCall& c, cudaStream_t stream) {
  Fp8EvictArgs a;
  a.codes = pool.codes;
  a.scales = pool.scales;
  a.mass = pool.mass;
  a.plane_bytes = pool.plane_bytes;
  a.block_tables = c.block_tables;
  a.context_lens = c.context_lens;
  a.new_tables = c.new_tables;
  a.kept = c.kept;
  a.new_lens = c.new_lens;
  a.flags = pool.flags;
  a.bt_stride = c.bt_stride;
  a.new_stride = c.new_stride;
  a.max_ctx = c.max_ctx;
  a.budget = c.budget;
  a.recent = c.recent;
  a.num_blocks = pool.num_blocks;
  a.block_size = pool.block_size;
  a.num_kv_heads = pool.num_kv_heads;
  fp8_select_kernel<<<dim3(pool.num_kv_heads, c.batch), kSelThreads, 0, stream>>>(a);
  int rc = fp8_launch_status("fp8_evict select launch", cudaGetLastError());
  if (rc) return rc;
  count_launches(1);
  const int most = std::min(c.budget, c.max_ctx);
  if (most == 0) return CLOVE_OK;
  const dim3 grid((most + pool.block_size - 1) / pool.block_size, pool.num_kv_heads, c.batch);
  switch (pool.head_dim) {
    case 64: fp8_compact_kernel<64><<<grid, kCompactThreads, 0, stream>>>(a); break;
    case 128: fp8_compact_kernel<128><<<grid, kCompactThreads, 0, stream>>>(a); break;
    default: fp8_compact_kernel<256><<<grid, kCompactThreads, 0, stream>>>(a); break;
  }
  count_launches(1);
  return fp8_launch_status("fp8_evict compact launch", cudaGetLastError());
}

}  // namespace clove
