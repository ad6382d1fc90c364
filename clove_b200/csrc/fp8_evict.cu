// Eviction by accumulated attention weight.
//
// select    a cluster of 1 to 8 CTAs per (sequence, KV head), each with a part
//           of the tokens.  The weights become ordered 32-bit keys, read from
//           HBM once and kept in shared memory; three histograms of 11, 11 and
//           10 bits, summed over the cluster through distributed shared memory,
//           find the key of the last token kept; then every warp writes its
//           kept tokens at their place, counted from the parts before it.
// compact   a warp moves 32 kept rows of a (sequence, KV head) at a time into
//           their new blocks, rounding to a new block's scale where that is
//           larger; the loads of 32 rows (16 at head_dim 256) are under way at
//           once, and beside them the chain (kept index, table, scales) that
//           the warp's next rows need.
// HBM bounds both: 4 bytes per token and KV head for the first, 4 head_dim
// bytes per kept token and KV head (read and written, K and V) for the second.
// Measured with 8 heads of 128, selection + moving: 128 ragged sequences (16 to
// 8192 tokens) to 512 36 + 50 us, 8 of 32k to 131k tokens to 8192 60 + 56 us: the
// work and the barriers of five passes hold up the first, rows of 128 bytes gathered at
// random (4.5 TB/s) the second.  (Launching the second early costs 12 us: its
// CTAs take the first one's places.)
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

constexpr int kBins = 2048;
constexpr int kMaxRoom = 16 * 1024;  // keys in shared memory: three CTAs on an SM

// Exclusive sum over the block of one int per thread; *total gets the sum.
template <int kSelWarps>
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
// dynamic shared memory holds; what a part has beyond that is read from the
// cache (L2) again in every pass.
template <int kSelThreads, int kPerSm>
__global__ void __launch_bounds__(kSelThreads, kPerSm) fp8_select_kernel(const Fp8EvictArgs a, int C, int room) {
  constexpr int kSelWarps = kSelThreads / 32, kBinsPer = kBins / kSelThreads;
  static_assert(kBinsPer % 4 == 0 && kBinsPer * kSelThreads == kBins, "a thread reads its bins four at a time");
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) int hist[kBins];
  __shared__ int warp_tot[kSelWarps];
  __shared__ int2 warp_cnt[kSelWarps];       // keys above and equal to the threshold
  __shared__ __align__(8) int2 part_cnt;     // the same of this CTA
  __shared__ __align__(16) int4 found;       // digit, keys above it, keys with it
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
#pragma unroll 4
  for (int i = tid; i < min(cnt, room); i += kSelThreads) keys[i] = load(t0 + i);
  auto key = [&](int i) { return i < room ? keys[i] : load(t0 + i); };

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
      // thread i: kBinsPer bins, from the largest down
      const int first = kBins - kBinsPer * (tid + 1);
      int v[kBinsPer], mine = 0;
#pragma unroll
      for (int k = 0; k < kBinsPer; k += 4) {
        int4 c = *reinterpret_cast<const int4*>(hist + first + k);
        for (int r = 1; r < C; ++r) {
          const int4 p = peer_int4(peer_address(hist + first + k, r));
          c.x += p.x;
          c.y += p.y;
          c.z += p.z;
          c.w += p.w;
        }
        v[k] = c.x;
        v[k + 1] = c.y;
        v[k + 2] = c.z;
        v[k + 3] = c.w;
        mine += c.x + c.y + c.z + c.w;
      }
      int total;
      int above = block_scan<kSelWarps>(mine, warp_tot, &total);
#pragma unroll
      for (int k = kBinsPer - 1; k >= 0; --k) {
        if (above < left && left <= above + v[k]) found = make_int4(first + k, above, v[k], 0);
        above += v[k];
      }
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    const int4 f = C > 1 ? peer_int4(peer_address(&found, 0)) : found;
    prefix |= (uint32_t)f.x << low;
    left -= f.y;
    if (left == f.z && prefix > 0) {  // all keys with these digits are kept
      --prefix;
      left = 0;
      break;
    }
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

constexpr int kCompactWarps = 4, kCompactPerSm = 5;

// Two 16-byte pieces of codes to a scale 1 / ratio times as large.
__device__ __forceinline__ uint4 fp8_rescale16(uint4 c, float ratio) {
  const uint2 lo = fp8_rescale8(make_uint2(c.x, c.y), ratio), hi = fp8_rescale8(make_uint2(c.z, c.w), ratio);
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// A warp's item: 32 kept rows of one (sequence, KV head).  `chunks`: items of a
// (sequence, head), enough for the longest one.
template <int D>
__global__ void __launch_bounds__(kCompactWarps * 32, kCompactPerSm)
    fp8_compact_kernel(const Fp8EvictArgs a, int batch, int chunks) {
  constexpr int LPR = D / 16, RPW = 32 / LPR;         // lanes per row, rows per load
  constexpr int STEP = D == 64 ? 4 : 8, ROWS = STEP * RPW;  // loads per plane and rows per batch
  const int lane = threadIdx.x & 31, sub = lane % LPR, r0 = lane / LPR;
  const int H = a.num_kv_heads, bs = a.block_size, shift = 31 - __clz(bs);
  const size_t plane = (size_t)a.num_blocks * H;
  griddep_wait();
  const int total = batch * H * chunks, stride = gridDim.x * kCompactWarps;

  // Lane r of an item: row `from` (tile * block_size + offset) goes to row
  // `to`, its codes times ratio (K, V) rounded; to < 0: nothing.
  struct Move {
    int from, to;
    float ratio[2];
  };
  auto scales_of = [&](int b, int h, int t, float (&s)[2]) {
    int blk = __ldg(a.block_tables + (size_t)b * a.bt_stride + (t >> shift));
    if (blk < 0 || blk >= a.num_blocks) {
      atomicOr(a.flags, CLOVE_FLAG_BLOCK_OOB);
      blk = 0;
    }
    const int tile = blk * H + h;
    s[0] = a.scales[tile];
    s[1] = a.scales[plane + tile];
    return tile * bs + (t & (bs - 1));
  };
  auto prepare = [&](int item) {
    Move v = {0, -1, {1.f, 1.f}};
    if (item >= total) return v;
    const int head = item / chunks, r = (item - head * chunks) * 32 + lane, b = head / H, h = head - b * H;
    const int m = min(evict_len(a, b), a.budget);
    if ((r & ~31) >= m) return v;
    const int32_t* kept = a.kept + (size_t)head * a.budget;
    float s[2] = {0.f, 0.f}, top[2];
    int dst = -1;
    if (r < m) {
      dst = __ldg(a.new_tables + (size_t)b * a.new_stride + (r >> shift));
      v.from = scales_of(b, h, __ldcg(kept + r), s);
    }
    // the new block's scale: the largest of its rows'
    top[0] = s[0];
    top[1] = s[1];
    if (bs > 32) {
      const int first = r >> shift << shift;
      for (int k = first - (first & 31) + lane; k < min(m, first + bs); k += 32) {
        float o[2];
        scales_of(b, h, __ldcg(kept + k), o);
        top[0] = fmaxf(top[0], o[0]);
        top[1] = fmaxf(top[1], o[1]);
      }
    }
    for (int o = min(bs, 32) / 2; o > 0; o >>= 1) {
      top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
      top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
    }
    if (r < m) {
      if (dst < 0 || dst >= a.num_blocks) {
        atomicOr(a.flags, CLOVE_FLAG_BLOCK_OOB);
      } else {
        const int tile = dst * H + h, off = r & (bs - 1);
        v.to = tile * bs + off;
        if (off == 0) {
          a.scales[tile] = top[0];
          a.scales[plane + tile] = top[1];
        }
        a.mass[v.to] = a.mass[v.from];
        if (s[0] != top[0]) v.ratio[0] = s[0] / top[0];
        if (s[1] != top[1]) v.ratio[1] = s[1] / top[1];
      }
    }
    return v;
  };

  int item = blockIdx.x * kCompactWarps + (threadIdx.x >> 5);
  Move now = prepare(item);
  for (; item < total; item += stride) {
    Move next = {0, -1, {1.f, 1.f}};
    bool prepared = false;
    if (__any_sync(0xffffffffu, now.to >= 0)) {
#pragma unroll 1
      for (int at = 0; at < 32; at += ROWS) {
        uint4 c[2][STEP];
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
          const int from = __shfl_sync(0xffffffffu, now.from, at + i * RPW + r0);
#pragma unroll
          for (int p = 0; p < 2; ++p)
            c[p][i] = __ldcg(reinterpret_cast<const uint4*>(a.codes + p * a.plane_bytes + (size_t)from * D + sub * 16));
        }
        if (!prepared) {  // the next item's chain of loads runs beside this one's rows
          next = prepare(item + stride);
          prepared = true;
        }
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
          const int r = at + i * RPW + r0, to = __shfl_sync(0xffffffffu, now.to, r);
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const float ratio = __shfl_sync(0xffffffffu, now.ratio[p], r);
            if (to >= 0) {
              if (ratio != 1.f) c[p][i] = fp8_rescale16(c[p][i], ratio);
              *reinterpret_cast<uint4*>(a.codes + p * a.plane_bytes + (size_t)to * D + sub * 16) = c[p][i];
            }
          }
        }
      }
    }
    if (!prepared) next = prepare(item + stride);
    now = next;
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
  const int most = std::min(c.budget, c.max_ctx);
  const long long heads = (long long)c.batch * pool.num_kv_heads;
  const int chunks = (int)((most + 31LL) / 32);
  if (heads * chunks > 0x7fffffff - (1 << 20)) {
    set_last_error("fp8_evict: %lld rows to move", heads * chunks * 32);
    return CLOVE_ERR_UNSUPPORTED;
  }
  // CTAs per (sequence, head): parts of at most 8192 tokens of the longest sequence (of 2048 while the GPU has room
  // for more CTAs), in a cluster of up to 8.  Short parts alone on a CTA take few threads, so that many fit an SM.
  int C = 1;
  while (C < 8 && (C * 8192LL < c.max_ctx || (C * 2048LL < c.max_ctx && 2 * C * heads <= 2 * pool.num_sms))) C *= 2;
  auto select = C == 1 ? fp8_select_kernel<256, 5> : fp8_select_kernel<512, 3>;
  const unsigned threads = C == 1 ? 256 : 512;
  const long long part = ((c.max_ctx + C - 1LL) / C + 511) / 512 * 512;
  const int room = (int)std::min<long long>(part, kMaxRoom), smem = room * (int)sizeof(uint32_t);
  int rc = fp8_launch_status("cudaFuncSetAttribute",
                             cudaFuncSetAttribute(select, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                  kMaxRoom * (int)sizeof(uint32_t)));
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C * pool.num_kv_heads, c.batch);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)C, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  rc = fp8_launch_status("fp8_evict select launch", cudaLaunchKernelEx(&cfg, select, a, C, room));
  if (rc) return rc;
  count_launches(1);
  if (most == 0) return CLOVE_OK;
  cfg.gridDim = dim3((unsigned)std::min<long long>((heads * chunks + kCompactWarps - 1) / kCompactWarps,
                                                   (long long)pool.num_sms * kCompactPerSm));
  cfg.blockDim = dim3(kCompactWarps * 32);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  cudaError_t e;
  switch (pool.head_dim) {
    case 64: e = cudaLaunchKernelEx(&cfg, fp8_compact_kernel<64>, a, c.batch, chunks); break;
    case 128: e = cudaLaunchKernelEx(&cfg, fp8_compact_kernel<128>, a, c.batch, chunks); break;
    default: e = cudaLaunchKernelEx(&cfg, fp8_compact_kernel<256>, a, c.batch, chunks); break;
  }
  count_launches(1);
  return fp8_launch_status("fp8_evict compact launch", e);
}

}  // namespace clove
