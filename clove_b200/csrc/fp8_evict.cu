// Eviction by accumulated attention weight.
//
// select    a cluster of 1 to 8 CTAs per (sequence, KV head), each with a part
//           of the tokens.  The weights become ordered 32-bit keys, read from
//           HBM once and kept in shared memory; three histograms of 11, 11 and
//           10 bits, summed over the cluster through distributed shared memory,
//           find the key of the last token kept; then every warp writes its
//           kept tokens at their place, counted from the parts before it.
// compact   one warp per (new block, KV head, sequence): gathers the kept rows
//           into the new block, rounding to its scale where that is larger.
//           All loads of 16 rows are under way at once.
// HBM bounds both: 4 bytes per token and KV head for the first, 4 head_dim
// bytes per kept token and KV head (read and written, K and V) for the second.
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

constexpr int kSelThreads = 512, kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxRoom = 48 * 1024;

// Exclusive sum over the block of one int per thread; *total gets the sum.
__device__ __forceinline__ int block_scan(int x, int* warp_tot, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  if (lane == 31) warp_tot[warp] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    if (w < warp) before += warp_tot[w];
    all += warp_tot[w];
  }
  *total = all;
  __syncthreads();
  return before + s - x;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// The address of `p` (shared) in CTA `rank` of the cluster, and a read of it.
__device__ __forceinline__ uint32_t peer_address(const void* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ int4 peer_int4(uint32_t a) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ int2 peer_int2(uint32_t a) {
  int2 v;
  asm volatile("ld.shared::cluster.v2.s32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}

// Grid (C * heads, batch), clusters of C along x.  `room`: keys that the
// dynamic shared memory holds; a part longer than that is read from the cache
// again in every pass.
__global__ void __launch_bounds__(kSelThreads) fp8_select_kernel(const Fp8EvictArgs a, int C, int room) {
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) int hist[kBins];
  __shared__ int warp_tot[kSelWarps];
  __shared__ int2 warp_cnt[kSelWarps];       // keys above and equal to the threshold
  __shared__ __align__(8) int2 part_cnt;     // the same of this CTA
  __shared__ __align__(8) int2 found;        // digit, keys above it
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.x / C, rank = blockIdx.x - h * C, b = blockIdx.y, H = a.num_kv_heads, bs = a.block_size;
  const int shift = 31 - __clz(bs);
  griddep_wait();
  const int n = evict_len(a, b), m = min(n, a.budget);
  if (h == 0 && rank == 0 && tid == 0) {
    a.new_lens[b] = m;
    if (__ldg(a.context_lens + b) != n) atomicOr(a.flags, CLOVE_FLAG_CTX_RANGE);
  }
  int32_t* kept = a.kept + ((size_t)b * H + h) * a.budget;
  const int self = rank * kSelThreads + tid, all = C * kSelThreads;
  for (int i = m + self; i < a.budget; i += all) kept[i] = -1;
  const int last = min(a.recent, n), old = n - last, need = m - last;
  for (int i = self; i < last; i += all) kept[need + i] = old + i;
  if (need == 0) return;  // (every CTA of the cluster alike)
  if (need == old) {
    for (int i = self; i < need; i += all) kept[i] = i;
    return;
  }
  const int32_t* table = a.block_tables + (size_t)b * a.bt_stride;
  auto load = [&](int t) {
    int blk = __ldg(table + (t >> shift));
    if (blk < 0 || blk >= a.num_blocks) {
      atomicOr(a.flags, CLOVE_FLAG_BLOCK_OOB);
      blk = 0;
    }
    return mass_key(__ldg(a.mass + ((size_t)blk * H + h) * bs + (t & (bs - 1))));
  };
  // this CTA's tokens [t0, t1), a multiple of 32 per warp
  const int part = ((old + C - 1) / C + kSelThreads - 1) / kSelThreads * kSelThreads;
  const int t0 = min(old, rank * part), t1 = min(old, t0 + part), cnt = t1 - t0;
  const bool held = cnt <= room;
  if (held) {
#pragma unroll 4
    for (int i = tid; i < cnt; i += kSelThreads) keys[i] = load(t0 + i);
  }
  auto key = [&](int i) { return held ? keys[i] : load(t0 + i); };

  // ---- the need-th largest key ----
  uint32_t prefix = 0;
  int left = need;  // rank of the wanted key among those that share the prefix
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int low = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < cnt; i += kSelThreads) {
      const uint32_t k = key(i);
      if (pass == 0 || ((k ^ prefix) >> (low + bits)) == 0) atomicAdd(&hist[(k >> low) & ((1u << bits) - 1)], 1);
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    if (rank == 0) {
      // thread i: four bins, from the largest down
      const int first = kBins - 4 - 4 * tid;
      int4 c = *reinterpret_cast<const int4*>(hist + first);
      for (int r = 1; r < C; ++r) {
        const int4 p = peer_int4(peer_address(hist + first, r));
        c.x += p.x;
        c.y += p.y;
        c.z += p.z;
        c.w += p.w;
      }
      int total;
      int above = block_scan(c.x + c.y + c.z + c.w, warp_tot, &total);
      const int v[4] = {c.w, c.z, c.y, c.x};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (above < left && left <= above + v[k]) found = make_int2(first + 3 - k, above);
        above += v[k];
      }
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    const int2 f = C > 1 ? peer_int2(peer_address(&found, 0)) : found;
    prefix |= (uint32_t)f.x << low;
    left -= f.y;
    if (C > 1) cluster_sync();  // (rank 0 may not change `found` before all have read it)
    else __syncthreads();
  }

  // ---- the keys above the threshold, and the first `left` of those equal to it ----
  const int per_warp = part / kSelWarps, w0 = warp * per_warp, w1 = min(cnt, w0 + per_warp);
  int gt = 0, eq = 0;
  for (int base = w0; base < w1; base += 32) {
    const bool in = base + lane < w1;
    const uint32_t k = in ? key(base + lane) : 0u;
    gt += __popc(__ballot_sync(0xffffffffu, in && k > prefix));
    eq += __popc(__ballot_sync(0xffffffffu, in && k == prefix));
  }
  if (lane == 0) warp_cnt[warp] = make_int2(gt, eq);
  __syncthreads();
  int2 sum = make_int2(0, 0), before = make_int2(0, 0);
  for (int w = 0; w < kSelWarps; ++w) {
    if (w == warp) before = sum;
    sum.x += warp_cnt[w].x;
    sum.y += warp_cnt[w].y;
  }
  if (C > 1) {
    if (tid == 0) part_cnt = sum;
    cluster_sync();
    for (int r = 0; r < rank; ++r) {
      const int2 p = peer_int2(peer_address(&part_cnt, r));
      before.x += p.x;
      before.y += p.y;
    }
    cluster_sync();  // no CTA leaves while its shared memory is read
  }
  const unsigned lower = (1u << lane) - 1;
  for (int base = w0; base < w1; base += 32) {
    const bool in = base + lane < w1;
    const uint32_t k = in ? key(base + lane) : 0u;
    const unsigned mg = __ballot_sync(0xffffffffu, in && k > prefix), me = __ballot_sync(0xffffffffu, in && k == prefix);
    const int g = before.x + __popc(mg & lower), e = before.y + __popc(me & lower);
    if (in && (k > prefix || (k == prefix && e < left))) kept[g + min(e, left)] = t0 + base + lane;
    before.x += __popc(mg);
    before.y += __popc(me);
  }
}

constexpr int kCompactWarps = 4;

// Two 16-byte pieces of codes to a scale 1 / ratio times as large.
__device__ __forceinline__ uint4 fp8_rescale16(uint4 c, float ratio) {
  const uint2 lo = fp8_rescale8(make_uint2(c.x, c.y), ratio), hi = fp8_rescale8(make_uint2(c.z, c.w), ratio);
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

template <int D>
__global__ void __launch_bounds__(kCompactWarps * 32) fp8_compact_kernel(const Fp8EvictArgs a) {
  constexpr int LPR = D / 16, RPW = 32 / LPR, STEP = 16 / RPW;  // lanes per row, rows per load, loads of 16 rows
  const int lane = threadIdx.x & 31, sub = lane % LPR, r0 = lane / LPR;
  const int j = blockIdx.x * kCompactWarps + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
  const int H = a.num_kv_heads, bs = a.block_size, shift = 31 - __clz(bs);
  griddep_wait();
  const int m = min(evict_len(a, b), a.budget), first = j * bs, rows = min(bs, m - first);
  if (rows <= 0) return;
  const int dst = __ldg(a.new_tables + (size_t)b * a.new_stride + j);
  if (dst < 0 || dst >= a.num_blocks) {
    if (lane == 0 && h == 0) atomicOr(a.flags, CLOVE_FLAG_BLOCK_OOB);
    return;
  }
  const size_t to = (size_t)dst * H + h, plane = (size_t)a.num_blocks * H;
  const int32_t* kept = a.kept + ((size_t)b * H + h) * a.budget + first;
  // lane r: source tile and offset of row base + r, and its scales
  struct Source {
    int row;
    float s[2];
  };
  auto source = [&](int r, bool move_mass) {
    Source s = {0, {0.f, 0.f}};
    if (r < rows) {
      const int t = __ldcg(kept + r);
      int blk = __ldg(a.block_tables + (size_t)b * a.bt_stride + (t >> shift));
      if (blk < 0 || blk >= a.num_blocks) {
        atomicOr(a.flags, CLOVE_FLAG_BLOCK_OOB);
        blk = 0;
      }
      const size_t tile = (size_t)blk * H + h;
      s.row = (int)(tile * bs) + (t & (bs - 1));
      s.s[0] = a.scales[tile];
      s.s[1] = a.scales[plane + tile];
      if (move_mass) a.mass[to * bs + r] = a.mass[s.row];
    }
    return s;
  };
  Source now = source(lane, true);
  float top[2] = {now.s[0], now.s[1]};
  for (int base = 32; base < rows; base += 32) {
    const Source s = source(base + lane, true);
    top[0] = fmaxf(top[0], s.s[0]);
    top[1] = fmaxf(top[1], s.s[1]);
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top[p] = fmaxf(top[p], __shfl_xor_sync(0xffffffffu, top[p], o));
    if (lane == 0) a.scales[p * plane + to] = top[p];
  }
  for (int base = 0; base < rows; base += 32) {
    if (base > 0) now = source(base + lane, false);
    for (int half = 0; half < 32 && base + half < rows; half += 16) {
      uint4 c[2][STEP];
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        const int r = half + i * RPW + r0, src = __shfl_sync(0xffffffffu, now.row, r);
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if (base + r < rows)
            c[p][i] = *reinterpret_cast<const uint4*>(a.codes + p * a.plane_bytes + (size_t)src * D + sub * 16);
      }
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        const int r = half + i * RPW + r0;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const float s = __shfl_sync(0xffffffffu, now.s[p], r);
          if (base + r < rows) {
            if (s != top[p]) c[p][i] = fp8_rescale16(c[p][i], s / top[p]);
            *reinterpret_cast<uint4*>(a.codes + p * a.plane_bytes + (to * bs + base + r) * D + sub * 16) = c[p][i];
          }
        }
      }
    }
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
  // CTAs per (sequence, head): parts of at most 8192 tokens of the longest sequence, in a cluster of up to 8.  Keys
  // that fit stay in shared memory (room for 8192 to 48 K of them); longer parts are read again.
  const int most = std::min(c.budget, c.max_ctx);
  int C = 1;
  while (C < 8 && (long long)C * 8192 < c.max_ctx) C *= 2;
  const int part = ((c.max_ctx + C - 1) / C + kSelThreads - 1) / kSelThreads * kSelThreads;
  const int room = part <= kMaxRoom ? part : 0, smem = room * (int)sizeof(uint32_t);
  int rc = fp8_launch_status("cudaFuncSetAttribute", cudaFuncSetAttribute(fp8_select_kernel,
                                                                          cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                                          kMaxRoom * (int)sizeof(uint32_t)));
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C * pool.num_kv_heads, c.batch);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)C, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  rc = fp8_launch_status("fp8_evict select launch", cudaLaunchKernelEx(&cfg, fp8_select_kernel, a, C, room));
  if (rc) return rc;
  count_launches(1);
  if (most == 0) return CLOVE_OK;
  const int blocks = (most + pool.block_size - 1) / pool.block_size;
  cfg.gridDim = dim3((blocks + kCompactWarps - 1) / kCompactWarps, pool.num_kv_heads, c.batch);
  cfg.blockDim = dim3(kCompactWarps * 32);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  cudaError_t e;
  switch (pool.head_dim) {
    case 64: e = cudaLaunchKernelEx(&cfg, fp8_compact_kernel<64>, a); break;
    case 128: e = cudaLaunchKernelEx(&cfg, fp8_compact_kernel<128>, a); break;
    default: e = cudaLaunchKernelEx(&cfg, fp8_compact_kernel<256>, a); break;
  }
  count_launches(1);
  return fp8_launch_status("fp8_evict compact launch", e);
}

}  // namespace clove
