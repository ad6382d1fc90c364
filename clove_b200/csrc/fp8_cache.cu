// Data movement of the 8-bit cache: the quantising append, the gather and
// the block copy.
//
// Append.  The codes of a (block, KV head) tile share one scale, so the tile,
// not the token, is the unit of work: one warp takes a tile with all the rows
// that the call writes to it, finds their largest magnitude, settles the
// scale, and stores the codes (rounding the rows already there when the scale
// grows).  HBM bounds it for prompts (3 bytes per element with 16-bit input:
// read 2, write 1), launch latency for a decode step.  Measured with 8 heads of
// 128, bf16: 8 x 2048 tokens 30 us (3.4 TB/s; ~4 us of it the first kernel),
// 64 x 2048 5.0 TB/s, one token of each of 128 sequences 4 us.
#include <algorithm>
#include <type_traits>

#include "fp8_common.cuh"

namespace clove {

// Eight elements of a row as loaded (16 bytes aligned), and widened.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  // The largest magnitude so far; NaN is passed over, an infinity is not.
  // 16-bit types: of the even and the odd elements, as packed pairs.
  __device__ __forceinline__ void max_into(uint32_t& m) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          m = __float_as_uint(fmaxf(__uint_as_float(m), fabsf(__uint_as_float(v[k]))));
        } else {
          using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
          const T2 x = __habs2(*reinterpret_cast<const T2*>(&v[k]));
          const T2 y = __hmax2(*reinterpret_cast<const T2*>(&m), x);
          m = *reinterpret_cast<const uint32_t*>(&y);
        }
      }
    }
  }
  static __device__ __forceinline__ float max_of(uint32_t m) {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(m);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
      return fmaxf(f.x, f.y);
    } else {
      return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
  }
  __device__ __forceinline__ void widen(float (&o)[8]) const {
    const uint32_t v[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[sizeof(T) / 2 - 1].x, w[sizeof(T) / 2 - 1].y,
                           w[sizeof(T) / 2 - 1].z, w[sizeof(T) / 2 - 1].w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = __uint_as_float(v[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
        o[2 * i] = f.x;
        o[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[2 * i] = __uint_as_float(v[i] << 16);
        o[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
      }
    }
  }
};

// One tile of plane p by `nw` warps (32 rows each; nw = max(1, block_size /
// 32)), this one being the w-th.  Lane r's `tok` > 0: row 32 w + r is written
// from token tok - 1; the other rows are rounded anew if the scale grows.  D /
// 8 lanes share a row.  `red` (2 floats per warp of the group) and barrier
// `bar` serve the group's maximum.  Eight 16-byte loads of a lane are
// under way at once; where its rows are more than that they are read again to
// be rounded, from L2 mostly (keeping twice as many cost more in resident warps).
// ROWS: rows per warp (block_size, at most 32).
template <typename T, int D, int ROWS>
__device__ __forceinline__ void fp8_write_tile(const Fp8AppendArgs& a, int p, int blk, int h, int tok, int nw, int w, float* red, int bar,
                               int lane) {
  constexpr int LPR = D / 8, RPW = 32 / LPR, NI = ROWS / RPW, VEC = (int)sizeof(T) / 2;
  constexpr int STEP = NI * VEC <= 8 ? NI : 8 / VEC;  // rows per lane at once
  constexpr bool kKeep = STEP == NI;
  const int sub = lane % LPR, r0 = lane / LPR;
  const int H = a.num_kv_heads, bs = a.block_size;
  const T* src = static_cast<const T*>(a.x[p]) + (size_t)h * D + sub * 8;
  const size_t tile = (size_t)blk * H + h;
  float* sp = a.scales + (size_t)p * a.num_blocks * H + tile;
  const float before = __ldcg(sp);
  float amax = 0.f;
  Raw8<T> raw[STEP];
  auto fetch = [&](int base) {
#pragma unroll
    for (int k = 0; k < STEP; ++k) {
      const int row = base + k * RPW + r0, t = __shfl_sync(0xffffffffu, tok, row & 31) - 1;
      if (t >= 0)
        raw[k].load(src + (size_t)t * H * D);
      else
        raw[k].zero();
    }
  };
  uint32_t most = 0;
  for (int base = 0; base < ROWS; base += RPW * STEP) {
    fetch(base);
#pragma unroll
    for (int k = 0; k < STEP; ++k) raw[k].max_into(most);
  }
  amax = Raw8<T>::max_of(most);
  if (__any_sync(0xffffffffu, !(amax < INFINITY))) {  // infinities do not count: look again without them
    amax = 0.f;
    for (int base = 0; base < ROWS; base += RPW * STEP) {
      if constexpr (!kKeep) fetch(base);
#pragma unroll
      for (int k = 0; k < STEP; ++k) {
        float x[8];
        raw[k].widen(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(x[i]));
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  bool anew = __shfl_sync(0xffffffffu, tok, 0) > 0;  // row 0 is written: the block starts anew
  if (nw > 1) {
    if (lane == 0) {
      red[2 * w] = amax;
      red[2 * w + 1] = anew ? 1.f : 0.f;
    }
    named_bar_sync(bar, nw * 32);
    for (int k = 0; k < nw; ++k) amax = fmaxf(amax, red[2 * k]);
    anew = red[1] > 0.f;
    named_bar_sync(bar, nw * 32);
  }
  const float old = anew ? 0.f : before;
  const float s = fmaxf(old, fp8_scale_for(amax));
  const float inv = 1.f / s, ratio = old / s;
  const bool grown = old > 0.f && s > old;
  unsigned char* dst = a.codes + p * a.plane_bytes + (tile * bs + 32 * w) * D + sub * 8;
  for (int base = 0; base < ROWS; base += RPW * STEP) {
    if constexpr (!kKeep) fetch(base);
#pragma unroll
    for (int k = 0; k < STEP; ++k) {
      const int row = base + k * RPW + r0, t = __shfl_sync(0xffffffffu, tok, row & 31) - 1;
      uint2* out = reinterpret_cast<uint2*>(dst + row * D);
      if (t >= 0) {
        float x[8];
        raw[k].widen(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= inv;
        *out = fp8_pack8(x);
      } else if (grown) {
        *out = fp8_rescale8(*out, ratio);
      }
    }
  }
  if (w == 0 && lane == 0) *sp = s;
  if (p == 0 && a.mass != nullptr && tok > 0) a.mass[tile * bs + 32 * w + lane] = 0.f;
}

constexpr int kAppendThreads = 256, kAppendWarps = kAppendThreads / 32;

// Few tokens: CTA (i, y).  If token i is the call's first token of its block,
// the CTA takes the block's tiles (its share y of them).  The rows the call
// writes are found by looking through slot_mapping.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kAppendThreads) fp8_append_scan_kernel(const Fp8AppendArgs a) {
  __shared__ int tok[256];
  __shared__ int earlier;
  __shared__ float red[2 * kAppendWarps];
  griddep_wait();
  const int i = blockIdx.x, tid = threadIdx.x, bs = a.block_size;
  const int slot = __ldg(a.slots + i);
  if (slot < 0) return;
  if (slot >= a.num_blocks * (long long)bs) {
    if (tid == 0 && blockIdx.y == 0) atomicOr(a.flags, CLOVE_FLAG_SLOT_OOB);
    return;
  }
  const int shift = 31 - __clz(bs), blk = slot >> shift;
  if (tid == 0) earlier = 0;
  tok[tid] = 0;
  __syncthreads();
  for (int j = tid; j < a.num_tokens; j += kAppendThreads) {
    const int s = __ldg(a.slots + j);
    if (s < 0 || s >> shift != blk) continue;
    if (j < i) earlier = 1;
    atomicMax(&tok[s & (bs - 1)], j + 1);  // of two tokens with one slot the later counts
  }
  __syncthreads();
  if (earlier) return;
  const int warp = tid >> 5, lane = tid & 31;
  const int nw = max(1, bs / 32), group = warp / nw, w = warp - group * nw, groups = kAppendWarps / nw;
  const int mine = tok[(32 * w + lane) & 255], tiles = 2 * a.num_kv_heads;
  for (int k = blockIdx.y * groups + group; k < tiles; k += gridDim.y * groups)
    fp8_write_tile<T, D, ROWS>(a, k & 1, blk, k >> 1, 32 * w + lane < bs ? mine : 0, nw, w, red + 2 * group * nw, 1 + group, lane);
}

// Many tokens, two kernels.  claim: the later of two tokens with one slot
// stays in the pool's slot index, and the first token to reach a block becomes
// its leader.  write: the tiles of the leaders' blocks; the last tile of a
// block puts its entries of the index back to zero, as the next call wants them.
__global__ void __launch_bounds__(256) fp8_append_claim_kernel(const Fp8AppendArgs a) {
  griddep_wait();
  const int i = blockIdx.x * 256 + threadIdx.x, bs = a.block_size;
  if (i >= a.num_tokens) return;
  const int slot = __ldg(a.slots + i);
  int lead = -1;
  if (slot >= a.num_blocks * (long long)bs) {
    atomicOr(a.flags, CLOVE_FLAG_SLOT_OOB);
  } else if (slot >= 0) {
    const int blk = slot / bs;
    atomicMax(a.slot_token + slot, i + 1);
    // of neighbours in one block only the first tries
    const int before = i % 32 > 0 ? __ldg(a.slots + i - 1) : -1;
    if ((before < 0 || before / bs != blk) && atomicExch(a.block_state + blk, 1) == 0) lead = blk;
  }
  a.leads[i] = lead;
}

// CTA (x, y): the leaders among 32 tokens, every gridDim.y-th group of their
// items.  An item (leader, tile) is the work of nw warps.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kAppendThreads, 4) fp8_append_write_kernel(const Fp8AppendArgs a) {
  __shared__ float red[2 * kAppendWarps];
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bs = a.block_size;
  const int nw = max(1, bs / 32), group = warp / nw, w = warp - group * nw, groups = kAppendWarps / nw;
  const int tiles = 2 * a.num_kv_heads;
  const int i = blockIdx.x * 32 + lane;
  const int lead = i < a.num_tokens ? __ldcg(a.leads + i) : -1;
  __shared__ int list[32];
  const unsigned leaders = __ballot_sync(0xffffffffu, lead >= 0);
  if (leaders == 0) return;
  if (warp == 0 && lead >= 0) list[__popc(leaders & ((1u << lane) - 1))] = lead;
  __syncthreads();
  const int n = __popc(leaders) * tiles;
  for (int q = blockIdx.y * groups + group; q < n; q += gridDim.y * groups) {
    const int j = q / tiles, k = q - j * tiles, blk = list[j];
    const int tok = 32 * w + lane < bs ? __ldcg(a.slot_token + (size_t)blk * bs + 32 * w + lane) : 0;
    __syncwarp();
    // a warp that has read its part of the index counts itself off; the last one clears the block's entries
    int done = 0;
    if (lane == 0) {
      __threadfence();
      done = atomicAdd(a.block_state + blk, 1);
    }
    fp8_write_tile<T, D, ROWS>(a, k & 1, blk, k >> 1, tok, nw, w, red + 2 * group * nw, 1 + group, lane);
    done = __shfl_sync(0xffffffffu, done, 0);
    if (done == tiles * nw) {
      for (int r = lane; r < bs; r += 32) a.slot_token[(size_t)blk * bs + r] = 0;
      if (lane == 0) a.block_state[blk] = 0;
    }
  }
}

// One look through n slots per token against two launches: measured equal at
// about 250 tokens (8.3 us each at 8 heads of 128).
constexpr int kScanTokens = 256;

template <typename K, typename... A>
static cudaError_t launch_after(K kern, dim3 grid, unsigned threads, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <typename T, int D, int ROWS>
static cudaError_t run_append(const Fp8AppendArgs& a, cudaStream_t stream) {
  const int groups = kAppendWarps / std::max(1, a.block_size / 32);
  const int ty = std::min((2 * a.num_kv_heads + groups - 1) / groups, 65535);
  if (a.num_tokens <= kScanTokens) {
    count_launches(1);
    return launch_after(fp8_append_scan_kernel<T, D, ROWS>, dim3(a.num_tokens, ty), kAppendThreads, stream, a);
  }
  cudaError_t e = launch_after(fp8_append_claim_kernel, dim3((a.num_tokens + 255) / 256), 256, stream, a);
  if (e != cudaSuccess) return e;
  count_launches(2);
  // 32 tokens of a prompt have one leader or two, of a batch of single tokens up to 32: a chunk's items go to as
  // many CTAs as one leader keeps busy, to more where the chunks are few (512 CTAs in all: most of them find nothing)
  const int chunks = (a.num_tokens + 31) / 32, tiles = 2 * a.num_kv_heads;
  const int one = std::min((tiles + groups - 1) / groups, 8), most = (32 * tiles + groups - 1) / groups;
  return launch_after(fp8_append_write_kernel<T, D, ROWS>, dim3(chunks, std::min(most, std::max(one, 512 / chunks))),
                      kAppendThreads, stream, a);
}

template <typename T, int D>
static cudaError_t append_rows(const Fp8AppendArgs& a, cudaStream_t stream) {
  switch (a.block_size) {
    case 8: return run_append<T, D, 8>(a, stream);
    case 16: return run_append<T, D, 16>(a, stream);
    default: return run_append<T, D, 32>(a, stream);
  }
}

template <typename T>
static cudaError_t append_dim(const Fp8AppendArgs& a, int head_dim, cudaStream_t stream) {
  switch (head_dim) {
    case 64: return append_rows<T, 64>(a, stream);
    case 128: return append_rows<T, 128>(a, stream);
    default: return append_rows<T, 256>(a, stream);
  }
}

size_t fp8_append_workspace(const clove_fp8_pool&, int num_tokens) {
  return num_tokens > kScanTokens ? sizeof(int32_t) * (size_t)num_tokens : 0;
}

int launch_fp8_append(const clove_fp8_pool& pool, int dtype, const void* k, const void* v, const int32_t* slots,
                      int num_tokens, void* workspace, cudaStream_t stream) {
  Fp8AppendArgs a;
  a.x[0] = k;
  a.x[1] = v;
  a.slots = slots;
  a.codes = pool.codes;
  a.scales = pool.scales;
  a.mass = pool.mass;
  a.flags = pool.flags;
  a.slot_token = pool.slot_token;
  a.block_state = pool.slot_token + (size_t)pool.num_blocks * pool.block_size;
  a.leads = static_cast<int32_t*>(workspace);
  a.plane_bytes = pool.plane_bytes;
  a.num_tokens = num_tokens;
  a.num_blocks = pool.num_blocks;
  a.block_size = pool.block_size;
  a.num_kv_heads = pool.num_kv_heads;
  cudaError_t e;
  switch (dtype) {
    case CLOVE_DTYPE_F32: e = append_dim<float>(a, pool.head_dim, stream); break;
    case CLOVE_DTYPE_F16: e = append_dim<__half>(a, pool.head_dim, stream); break;
    default: e = append_dim<__nv_bfloat16>(a, pool.head_dim, stream); break;
  }
  return fp8_launch_status("fp8_append launch", e);
}

// ---------------------------------------------------------------------------
// gather: [batch, max_ctx, heads, dim] f32; eight elements per thread
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
fp8_gather_kernel(const unsigned char* codes, const float* scales, size_t plane_bytes, const int32_t* block_tables,
                  int bt_stride, const int32_t* context_lens, int max_ctx, int block_size, int num_blocks, int H,
                  int D, float* k_out, float* v_out, int32_t* flags) {
  const int p = blockIdx.z, b = blockIdx.y;
  const unsigned char* src = codes + p * plane_bytes;
  const float* sc = scales + (size_t)p * num_blocks * H;
  int ctx = __ldg(context_lens + b);
  if (ctx < 0 || ctx > max_ctx) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && p == 0) atomicOr(flags, CLOVE_FLAG_CTX_RANGE);
    ctx = max(0, min(ctx, max_ctx));
  }
  const int words = H * D / 8, wpr = D / 8;
  const long long total = (long long)max_ctx * words;
  float* out = (p == 0 ? k_out : v_out) + (size_t)b * total * 8;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const int t = (int)(i / words), w = (int)(i - (long long)t * words);
    const int h = w / wpr, d8 = w - h * wpr;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (t < ctx) {
      const int blk = __ldg(block_tables + (long long)b * bt_stride + t / block_size);
      if (blk >= 0 && blk < num_blocks) {
        const size_t tile = (size_t)blk * H + h;
        fp8_unpack8(*reinterpret_cast<const uint2*>(src + (tile * block_size + t % block_size) * D + d8 * 8), x);
        const float s = sc[tile];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= s;
      } else if (w == 0) {
        atomicOr(flags, CLOVE_FLAG_BLOCK_OOB);
      }
    }
    float4* o = reinterpret_cast<float4*>(out + i * 8);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

int launch_fp8_gather(const clove_fp8_pool& pool, const int32_t* block_tables, int bt_stride,
                      const int32_t* context_lens, int batch, int max_ctx, float* k_out, float* v_out,
                      cudaStream_t stream) {
  const long long words = (long long)max_ctx * pool.num_kv_heads * pool.head_dim / 8;
  const unsigned bx = (unsigned)std::max(1LL, std::min((words + 255) / 256, 1024LL));
  fp8_gather_kernel<<<dim3(bx, batch, 2), 256, 0, stream>>>(
      pool.codes, pool.scales, pool.plane_bytes, block_tables, bt_stride, context_lens, max_ctx, pool.block_size,
      pool.num_blocks, pool.num_kv_heads, pool.head_dim, k_out, v_out, pool.flags);
  count_launches(1);
  return fp8_launch_status("fp8_gather launch", cudaGetLastError());
}

// ---------------------------------------------------------------------------
// block copy: CTA (i, plane) copies block src[i]; plane 0 also moves the mass
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
fp8_copy_kernel(unsigned char* codes, float* scales, float* mass, size_t plane_bytes, const int32_t* src,
                const int32_t* dst, int num_blocks, int H, int block_size, int D, int32_t* flags) {
  const int p = blockIdx.y;
  const int s = src[blockIdx.x], d = dst[blockIdx.x];
  if (s < 0 || s >= num_blocks || d < 0 || d >= num_blocks) {
    if (threadIdx.x == 0 && p == 0) atomicOr(flags, CLOVE_FLAG_BLOCK_OOB);
    return;
  }
  if (s == d) return;
  const int words = H * block_size * D / 16;
  uint4* plane = reinterpret_cast<uint4*>(codes + p * plane_bytes);
  for (int w = threadIdx.x; w < words; w += blockDim.x) plane[(size_t)d * words + w] = plane[(size_t)s * words + w];
  float* sc = scales + (size_t)p * num_blocks * H;
  for (int h = threadIdx.x; h < H; h += blockDim.x) sc[(size_t)d * H + h] = sc[(size_t)s * H + h];
  if (p == 0 && mass != nullptr)
    for (int w = threadIdx.x; w < H * block_size; w += blockDim.x)
      mass[(size_t)d * H * block_size + w] = mass[(size_t)s * H * block_size + w];
}

int launch_fp8_copy(const clove_fp8_pool& pool, const int32_t* src, const int32_t* dst, int n, cudaStream_t stream) {
  fp8_copy_kernel<<<dim3((unsigned)n, 2), 256, 0, stream>>>(pool.codes, pool.scales, pool.mass, pool.plane_bytes, src,
                                                            dst, pool.num_blocks, pool.num_kv_heads, pool.block_size,
                                                            pool.head_dim, pool.flags);
  count_launches(1);
  return fp8_launch_status("fp8_copy_blocks launch", cudaGetLastError());
}

}  // namespace clove
