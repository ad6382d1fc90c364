// Data movement of the 8-bit cache: the quantising append, the gather and
// the block copy.
//
// Append.  The codes of a (block, KV head) tile share one scale, so the tile,
// not the token, is the unit of work: one warp takes a tile with all the rows
// that the call writes to it, finds their largest magnitude, settles the
// scale, and stores the codes (rounding the rows already there when the scale
// grows).  HBM bounds it for prompts (3 bytes per element with 16-bit input:
// read 2, write 1), launch latency for a decode step.
#include <algorithm>

#include "fp8_common.cuh"

namespace clove {

// Eight consecutive elements of a row, widened (16-byte aligned).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&o)[8]) {
  load_vec_f32<T, 8>(p, o);
}

// One tile of plane p: rows with tok[r] > 0 are written from token tok[r] - 1,
// the others rescaled if the scale grows.  D / 8 lanes share a row, so a warp
// covers 256 / D rows at a time.
template <typename T, int D>
__device__ void fp8_write_tile(const Fp8AppendArgs& a, int p, int blk, int h, const int* tok, int lane) {
  constexpr int LPR = D / 8, RPW = 32 / LPR;
  const int sub = lane % LPR, r0 = lane / LPR;
  const int H = a.num_kv_heads, bs = a.block_size;
  const T* src = static_cast<const T*>(a.x[p]) + (size_t)h * D + sub * 8;
  float amax = 0.f;
  for (int r = r0; r < bs; r += RPW) {
    const int t = tok[r] - 1;
    if (t < 0) continue;
    float x[8];
    load8<T>(src + (size_t)t * H * D, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(x[i]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const size_t tile = (size_t)blk * H + h;
  float* sp = a.scales + (size_t)p * a.num_blocks * H + tile;
  const float old = tok[0] > 0 ? 0.f : *sp;
  const float s = fmaxf(old, fp8_scale_for(amax));
  const float inv = 1.f / s, ratio = old / s;
  unsigned char* dst = a.codes + p * a.plane_bytes + tile * bs * D + sub * 8;
  for (int r = r0; r < bs; r += RPW) {
    const int t = tok[r] - 1;
    uint2* out = reinterpret_cast<uint2*>(dst + r * D);
    if (t >= 0) {
      float x[8];
      load8<T>(src + (size_t)t * H * D, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= inv;
      *out = fp8_pack8(x);
    } else if (old > 0.f && s > old) {
      *out = fp8_rescale8(*out, ratio);
    }
  }
  __syncwarp();
  if (lane == 0) *sp = s;
  if (p == 0 && a.mass != nullptr) {
    for (int r = lane; r < bs; r += 32)
      if (tok[r] > 0) a.mass[tile * bs + r] = 0.f;
  }
}

constexpr int kAppendThreads = 256;

// CTA (i, y): if token i is the call's first token of its block, its warps
// take the block's tiles.  The rows the call writes are found by looking
// through slot_mapping.
template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) fp8_append_scan_kernel(const Fp8AppendArgs a) {
  __shared__ int tok[256];
  __shared__ int earlier;
  const int i = blockIdx.x, tid = threadIdx.x, bs = a.block_size;
  const int slot = __ldg(a.slots + i);
  if (slot < 0) return;
  if (slot >= a.num_blocks * (long long)bs) {
    if (tid == 0 && blockIdx.y == 0) atomicOr(a.flags, CLOVE_FLAG_SLOT_OOB);
    return;
  }
  const int blk = slot / bs;
  if (tid == 0) earlier = 0;
  for (int r = tid; r < bs; r += kAppendThreads) tok[r] = 0;
  __syncthreads();
  for (int j = tid; j < a.num_tokens; j += kAppendThreads) {
    const int s = __ldg(a.slots + j);
    if (s < 0 || s / bs != blk) continue;
    if (j < i) earlier = 1;
    atomicMax(&tok[s - blk * bs], j + 1);  // of two tokens with one slot the later counts
  }
  __syncthreads();
  if (earlier) return;
  const int warp = tid >> 5, lane = tid & 31;
  const int tiles = 2 * a.num_kv_heads;
  for (int k = blockIdx.y * (kAppendThreads / 32) + warp; k < tiles; k += gridDim.y * (kAppendThreads / 32))
    fp8_write_tile<T, D>(a, k & 1, blk, k >> 1, tok, lane);
}

template <typename T, int D>
static cudaError_t run_append(const Fp8AppendArgs& a, cudaStream_t stream) {
  const int ty = std::min((2 * a.num_kv_heads + 7) / 8, 64);
  fp8_append_scan_kernel<T, D><<<dim3(a.num_tokens, ty), kAppendThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t append_dim(const Fp8AppendArgs& a, int head_dim, cudaStream_t stream) {
  switch (head_dim) {
    case 64: return run_append<T, 64>(a, stream);
    case 128: return run_append<T, 128>(a, stream);
    default: return run_append<T, 256>(a, stream);
  }
}

size_t fp8_append_workspace(const clove_fp8_pool&, int) { return 0; }

int launch_fp8_append(const clove_fp8_pool& pool, int dtype, const void* k, const void* v, const int32_t* slots,
                      int num_tokens, void*, cudaStream_t stream) {
  Fp8AppendArgs a;
  a.x[0] = k;
  a.x[1] = v;
  a.slots = slots;
  a.codes = pool.codes;
  a.scales = pool.scales;
  a.mass = pool.mass;
  a.flags = pool.flags;
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
  count_launches(1);
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
