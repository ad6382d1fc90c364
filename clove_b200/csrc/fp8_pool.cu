// The C ABI of the 8-bit cache (include/clove_fp8.h): argument checks, pool
// lifecycle and error reporting around the kernel launchers.
#include <cfloat>
#include <exception>
#include <new>

#include "fp8_common.cuh"

namespace clove {
namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int kMaxEvict = 0x7fffffff - (1 << 16);

int fail(int rc, const char* what) {
  set_last_error("%s", what);
  return rc;
}

int cuda_fail(const char* what, cudaError_t e) {
  set_last_error("%s: %s", what, cudaGetErrorString(e));
  return CLOVE_ERR_CUDA;
}

// Calls may come from any thread with any device current.
struct OnDevice {
  int prev = -1;
  bool ok = true, changed = false;
  explicit OnDevice(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) {
      changed = true;
      ok = cudaSetDevice(dev) == cudaSuccess;
    }
  }
  ~OnDevice() {
    if (changed && prev >= 0) cudaSetDevice(prev);
  }
};

int check_shape(int num_blocks, int block_size, int num_kv_heads, int head_dim) {
  if (num_blocks <= 0 || num_kv_heads <= 0 || num_kv_heads > 65535) {
    set_last_error("fp8 pool: num_blocks %d, num_kv_heads %d", num_blocks, num_kv_heads);
    return CLOVE_ERR_INVALID_ARG;
  }
  if (block_size < 8 || block_size > 256 || (block_size & (block_size - 1))) {
    set_last_error("fp8 pool: block_size %d must be a power of two in [8, 256]", block_size);
    return CLOVE_ERR_UNSUPPORTED;
  }
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_last_error("fp8 pool: head_dim %d not built (64, 128, 256)", head_dim);
    return CLOVE_ERR_UNSUPPORTED;
  }
  if ((long long)num_blocks * block_size > 0x7fffffffLL)
    return fail(CLOVE_ERR_INVALID_ARG, "fp8 pool: num_blocks * block_size exceeds the int32 slot range");
  if ((long long)num_blocks * num_kv_heads * block_size * (head_dim >= 128 ? head_dim / 128 : 1) > 0x7fffffffLL)
    return fail(CLOVE_ERR_INVALID_ARG, "fp8 pool: more cache rows than a bulk copy's int32 coordinate reaches");
  return CLOVE_OK;
}

int check_device(int device) {
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return fail(CLOVE_ERR_NO_DEVICE, "no CUDA device");
  }
  if (device < 0 || device >= n) {
    set_last_error("device %d out of range [0, %d)", device, n);
    return CLOVE_ERR_NO_DEVICE;
  }
  return CLOVE_OK;
}

bool known_dtype(int dtype) {
  return dtype == CLOVE_DTYPE_F32 || dtype == CLOVE_DTYPE_F16 || dtype == CLOVE_DTYPE_BF16;
}

int finish_pool(clove_fp8_pool* p) {
  cudaError_t e = cudaDeviceGetAttribute(&p->num_sms, cudaDevAttrMultiProcessorCount, p->device);
  if (e != cudaSuccess) return cuda_fail("cudaDeviceGetAttribute", e);
  // the status word, and the append index behind it
  const size_t bytes = 256 + sizeof(int32_t) * (size_t)p->num_blocks * (p->block_size + 1);
  e = cudaMalloc(reinterpret_cast<void**>(&p->flags), bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_last_error("cudaMalloc(status word and append index, %zu): %s", bytes, cudaGetErrorString(e));
    return CLOVE_ERR_OOM;
  }
  p->slot_token = p->flags + 64;
  e = cudaMemset(p->flags, 0, bytes);
  // the first call may come on a stream that does not wait for this one
  if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
  if (e != cudaSuccess) return cuda_fail("cudaMemset(status word and append index)", e);
  return fp8_encode_map(*p);
}

// Takes the flags off in one step: calls on other streams may be raising some.
__global__ void take_flags_kernel(int32_t* flags, int32_t* taken) { *taken = atomicExch(flags, 0); }

// Tables, lengths and bounds that every reading call takes.
int check_tables(const clove_fp8_pool* pool, const char* who, const int32_t* block_tables, int bt_stride,
                 const int32_t* context_lens, int batch, int max_ctx) {
  if (batch < 0 || batch > 65535 || max_ctx < 0 || bt_stride <= 0) {
    set_last_error("%s: batch %d, max_ctx %d, bt_stride %d", who, batch, max_ctx, bt_stride);
    return CLOVE_ERR_INVALID_ARG;
  }
  if ((long long)max_ctx > (long long)bt_stride * pool->block_size) {
    set_last_error("%s: max_ctx %d exceeds block table capacity %d x %d", who, max_ctx, bt_stride, pool->block_size);
    return CLOVE_ERR_INVALID_ARG;
  }
  if (batch > 0 && (!block_tables || !context_lens)) {
    set_last_error("%s: null pointer", who);
    return CLOVE_ERR_INVALID_ARG;
  }
  return CLOVE_OK;
}

}  // namespace
}  // namespace clove

using namespace clove;

extern "C" {

int clove_fp8_pool_wrap(int device, void* codes, float* scales, float* mass, int num_blocks, int block_size,
                        int num_kv_heads, int head_dim, clove_fp8_pool_t* out) {
  if (!out || !codes || !scales) return fail(CLOVE_ERR_INVALID_ARG, "fp8_pool_wrap: null pointer");
  *out = nullptr;
  int rc = check_shape(num_blocks, block_size, num_kv_heads, head_dim);
  if (rc) return rc;
  if (!aligned(codes, 128) || !aligned(scales, 16) || !aligned(mass, 16))
    return fail(CLOVE_ERR_INVALID_ARG, "fp8_pool_wrap: codes must be 128-byte aligned, scales and mass 16-byte aligned");
  rc = check_device(device);
  if (rc) return rc;
  OnDevice g(device);
  if (!g.ok) return cuda_fail("cudaSetDevice", cudaGetLastError());
  clove_fp8_pool* p = new (std::nothrow) clove_fp8_pool();
  if (!p) return fail(CLOVE_ERR_OOM, "fp8_pool_wrap: out of host memory");
  p->device = device;
  p->num_blocks = num_blocks;
  p->block_size = block_size;
  p->num_kv_heads = num_kv_heads;
  p->head_dim = head_dim;
  p->codes = static_cast<unsigned char*>(codes);
  p->scales = scales;
  p->mass = mass;
  p->plane_bytes = (size_t)num_blocks * block_size * num_kv_heads * head_dim;
  rc = finish_pool(p);
  if (rc) {
    clove_fp8_pool_destroy(p);
    return rc;
  }
  *out = p;
  return CLOVE_OK;
}

int clove_fp8_pool_create(int device, int num_blocks, int block_size, int num_kv_heads, int head_dim, int with_mass,
                          clove_fp8_pool_t* out) {
  if (!out) return fail(CLOVE_ERR_INVALID_ARG, "fp8_pool_create: null out");
  *out = nullptr;
  int rc = check_shape(num_blocks, block_size, num_kv_heads, head_dim);
  if (rc) return rc;
  rc = check_device(device);
  if (rc) return rc;
  OnDevice g(device);
  if (!g.ok) return cuda_fail("cudaSetDevice", cudaGetLastError());
  // one allocation: codes, then scales, then mass, each 256-byte aligned
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  const size_t tiles = (size_t)num_blocks * num_kv_heads;
  const size_t codes = up(2 * tiles * block_size * head_dim), scales = up(2 * tiles * sizeof(float));
  const size_t total = codes + scales + (with_mass ? up(tiles * block_size * sizeof(float)) : 0);
  unsigned char* base = nullptr;
  cudaError_t e = cudaMalloc(reinterpret_cast<void**>(&base), total);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_last_error("fp8_pool_create: cudaMalloc(%zu): %s", total, cudaGetErrorString(e));
    return CLOVE_ERR_OOM;
  }
  e = cudaMemset(base, 0, total);
  if (e != cudaSuccess) {
    cudaFree(base);
    return cuda_fail("cudaMemset", e);
  }
  rc = clove_fp8_pool_wrap(device, base, reinterpret_cast<float*>(base + codes),
                           with_mass ? reinterpret_cast<float*>(base + codes + scales) : nullptr, num_blocks,
                           block_size, num_kv_heads, head_dim, out);
  if (rc) {
    cudaFree(base);
    return rc;
  }
  (*out)->owns_memory = 1;
  return CLOVE_OK;
}

int clove_fp8_pool_destroy(clove_fp8_pool_t pool) {
  if (!pool) return CLOVE_OK;
  OnDevice g(pool->device);
  if (pool->owns_memory) cudaFree(pool->codes);
  if (pool->flags) cudaFree(pool->flags);
  delete pool;
  return CLOVE_OK;
}

int clove_fp8_pool_info(clove_fp8_pool_t pool, clove_fp8_pool_info_t* info) {
  if (!pool || !info) return fail(CLOVE_ERR_INVALID_ARG, "fp8_pool_info: null pointer");
  info->device = pool->device;
  info->num_blocks = pool->num_blocks;
  info->block_size = pool->block_size;
  info->num_kv_heads = pool->num_kv_heads;
  info->head_dim = pool->head_dim;
  info->owns_memory = pool->owns_memory;
  info->codes = pool->codes;
  info->scales = pool->scales;
  info->mass = pool->mass;
  info->codes_bytes = 2 * pool->plane_bytes;
  return CLOVE_OK;
}

int clove_fp8_pool_status(clove_fp8_pool_t pool, void* stream, int* flags) {
  if (!pool) return fail(CLOVE_ERR_INVALID_ARG, "fp8_pool_status: null pool");
  OnDevice g(pool->device);
  if (!g.ok) return cuda_fail("cudaSetDevice", cudaGetLastError());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int host = 0;
  try {
    const std::lock_guard<std::mutex> lk(pool->status_lock);  // the word taken off is one per pool
    take_flags_kernel<<<1, 1, 0, s>>>(pool->flags, pool->flags + 1);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaMemcpyAsync(&host, pool->flags + 1, sizeof(int), cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return cuda_fail("fp8_pool_status", e);
  } catch (const std::exception&) {
    return fail(CLOVE_ERR_CUDA, "fp8_pool_status: lock");
  }
  count_launches(1);
  if (flags) *flags = host;
  if (host) {
    set_last_error("device check flags 0x%x", host);
    return CLOVE_ERR_DEVICE_CHECK;
  }
  return CLOVE_OK;
}

size_t clove_fp8_append_workspace_size(clove_fp8_pool_t pool, int num_tokens) {
  return pool && num_tokens > 0 ? fp8_append_workspace(*pool, num_tokens) : 0;
}

int clove_fp8_append(clove_fp8_pool_t pool, int dtype, const void* k, const void* v, const int32_t* slot_mapping,
                     int num_tokens, void* workspace, size_t workspace_bytes, void* stream) {
  if (!pool || num_tokens < 0) return fail(CLOVE_ERR_INVALID_ARG, "fp8_append: bad pool or num_tokens");
  if (!known_dtype(dtype)) return fail(CLOVE_ERR_UNSUPPORTED, "fp8_append: dtype must be f32, f16 or bf16");
  if (num_tokens == 0) return CLOVE_OK;
  if (!k || !v || !slot_mapping) return fail(CLOVE_ERR_INVALID_ARG, "fp8_append: null pointer");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(CLOVE_ERR_INVALID_ARG, "fp8_append: k and v must be 16-byte aligned");
  const size_t need = fp8_append_workspace(*pool, num_tokens);
  if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need)) {
    set_last_error("fp8_append: workspace of %zu bytes, 16-byte aligned, needed", need);
    return CLOVE_ERR_WORKSPACE;
  }
  OnDevice g(pool->device);
  if (!g.ok) return cuda_fail("cudaSetDevice", cudaGetLastError());
  return launch_fp8_append(*pool, dtype, k, v, slot_mapping, num_tokens, workspace, static_cast<cudaStream_t>(stream));
}

int clove_fp8_gather(clove_fp8_pool_t pool, const int32_t* block_tables, int bt_stride, const int32_t* context_lens,
                     int batch, int max_ctx, float* k_out, float* v_out, void* stream) {
  if (!pool) return fail(CLOVE_ERR_INVALID_ARG, "fp8_gather: null pool");
  int rc = check_tables(pool, "fp8_gather", block_tables, bt_stride, context_lens, batch, max_ctx);
  if (rc) return rc;
  if (batch == 0 || max_ctx == 0) return CLOVE_OK;
  if (!k_out || !v_out || !aligned(k_out, 16) || !aligned(v_out, 16))
    return fail(CLOVE_ERR_INVALID_ARG, "fp8_gather: k_out and v_out must be 16-byte aligned, not null");
  OnDevice g(pool->device);
  if (!g.ok) return cuda_fail("cudaSetDevice", cudaGetLastError());
  return launch_fp8_gather(*pool, block_tables, bt_stride, context_lens, batch, max_ctx, k_out, v_out,
                           static_cast<cudaStream_t>(stream));
}

size_t clove_fp8_decode_workspace_size(clove_fp8_pool_t pool, int batch, int num_q_heads, int max_ctx,
                                       int accumulate) {
  if (!pool || batch <= 0 || num_q_heads <= 0 || max_ctx < 0) return 0;
  return fp8_decode_workspace(*pool, batch, num_q_heads, max_ctx, accumulate);
}

int clove_fp8_decode(clove_fp8_pool_t pool, int dtype, const void* q, const void* k_new, const void* v_new,
                     int num_q_heads, const int32_t* block_tables, int bt_stride, const int32_t* context_lens,
                     int batch, float scale, int max_ctx, const clove_fp8_scores_t* scores, float* out,
                     void* workspace, size_t workspace_bytes, void* stream) {
  if (!pool) return fail(CLOVE_ERR_INVALID_ARG, "fp8_decode: null pool");
  if (!known_dtype(dtype)) return fail(CLOVE_ERR_UNSUPPORTED, "fp8_decode: dtype must be f32, f16 or bf16");
  if (num_q_heads <= 0 || num_q_heads % pool->num_kv_heads != 0) {
    set_last_error("fp8_decode: num_q_heads %d not a multiple of num_kv_heads %d", num_q_heads, pool->num_kv_heads);
    return CLOVE_ERR_INVALID_ARG;
  }
  if (num_q_heads / pool->num_kv_heads > 8) {
    set_last_error("fp8_decode: group size %d > 8 not built", num_q_heads / pool->num_kv_heads);
    return CLOVE_ERR_UNSUPPORTED;
  }
  int rc = check_tables(pool, "fp8_decode", block_tables, bt_stride, context_lens, batch, max_ctx);
  if (rc) return rc;
  const clove_fp8_scores_t sc = scores ? *scores : clove_fp8_scores_t{0.f, nullptr, 0, 0};
  // (a cap below float32's normal range has no usable inverse)
  const bool cap_ok = sc.softcap == 0.f || (sc.softcap >= FLT_MIN && sc.softcap < 3.4e38f);
  if (!cap_ok || sc.window < 0) {
    set_last_error("fp8_decode: softcap %g, window %d", (double)sc.softcap, sc.window);
    return CLOVE_ERR_INVALID_ARG;
  }
  if (sc.accumulate && !pool->mass) return fail(CLOVE_ERR_INVALID_ARG, "fp8_decode: accumulate needs a pool with mass");
  if (!k_new != !v_new) return fail(CLOVE_ERR_INVALID_ARG, "fp8_decode: k_new and v_new go together");
  if (k_new && max_ctx < 1) return fail(CLOVE_ERR_INVALID_ARG, "fp8_decode: max_ctx must be >= 1 with append");
  if (batch == 0) return CLOVE_OK;
  if (!q || !out) return fail(CLOVE_ERR_INVALID_ARG, "fp8_decode: null pointer");
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_new, 16) || !aligned(v_new, 16))
    return fail(CLOVE_ERR_INVALID_ARG, "fp8_decode: q, k_new, v_new and out must be 16-byte aligned");
  OnDevice g(pool->device);
  if (!g.ok) return cuda_fail("cudaSetDevice", cudaGetLastError());
  if (max_ctx == 0) {
    cudaError_t e = cudaMemsetAsync(out, 0, sizeof(float) * (size_t)batch * num_q_heads * pool->head_dim,
                                    static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? CLOVE_OK : cuda_fail("cudaMemsetAsync", e);
  }
  const size_t need = fp8_decode_workspace(*pool, batch, num_q_heads, max_ctx, sc.accumulate);
  if (need && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) {
    set_last_error("fp8_decode: workspace of %zu bytes, 256-byte aligned, needed", need);
    return CLOVE_ERR_WORKSPACE;
  }
  Fp8DecodeCall c;
  c.dtype = dtype;
  c.q = q;
  c.k_new = k_new;
  c.v_new = v_new;
  c.num_q_heads = num_q_heads;
  c.block_tables = block_tables;
  c.bt_stride = bt_stride;
  c.context_lens = context_lens;
  c.batch = batch;
  c.scale = scale;
  c.max_ctx = max_ctx;
  c.scores = sc;
  c.out = out;
  c.workspace = workspace;
  try {
    return launch_fp8_decode(*pool, c, static_cast<cudaStream_t>(stream));
  } catch (const std::exception&) {  // (the launch configurations' table)
    return fail(CLOVE_ERR_OOM, "fp8_decode: out of host memory");
  }
}

size_t clove_fp8_evict_workspace_size(clove_fp8_pool_t pool, int batch, int max_ctx, int budget) {
  if (!pool || batch <= 0 || max_ctx < 0 || budget < 0) return 0;
  return fp8_evict_workspace(*pool, batch, max_ctx, budget);
}

int clove_fp8_evict(clove_fp8_pool_t pool, const int32_t* block_tables, int bt_stride, const int32_t* context_lens,
                    int batch, int max_ctx, const int32_t* new_tables, int new_stride, int budget, int recent,
                    int32_t* kept, int32_t* new_lens, void* workspace, size_t workspace_bytes, void* stream) {
  if (!pool) return fail(CLOVE_ERR_INVALID_ARG, "fp8_evict: null pool");
  if (!pool->mass) return fail(CLOVE_ERR_INVALID_ARG, "fp8_evict: needs a pool with mass");
  int rc = check_tables(pool, "fp8_evict", block_tables, bt_stride, context_lens, batch, max_ctx);
  if (rc) return rc;
  if (budget < 1 || recent < 0 || recent > budget) {
    set_last_error("fp8_evict: budget %d, recent %d (0 <= recent <= budget, budget >= 1)", budget, recent);
    return CLOVE_ERR_INVALID_ARG;
  }
  // the selection counts tokens and places in 32 bits, a cluster's threads at a time
  if (budget > kMaxEvict || max_ctx > kMaxEvict) {
    set_last_error("fp8_evict: budget %d, max_ctx %d: more than the selection counts (%d)", budget, max_ctx, kMaxEvict);
    return CLOVE_ERR_UNSUPPORTED;
  }
  const int most = budget < max_ctx ? budget : max_ctx;
  if (new_stride <= 0 || (long long)new_stride * pool->block_size < most) {
    set_last_error("fp8_evict: new tables of %d x %d tokens do not hold %d", new_stride, pool->block_size, most);
    return CLOVE_ERR_INVALID_ARG;
  }
  if (batch == 0) return CLOVE_OK;
  if (!new_tables || !kept || !new_lens) return fail(CLOVE_ERR_INVALID_ARG, "fp8_evict: null pointer");
  const size_t need = fp8_evict_workspace(*pool, batch, max_ctx, budget);
  if (need && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) {
    set_last_error("fp8_evict: workspace of %zu bytes, 256-byte aligned, needed", need);
    return CLOVE_ERR_WORKSPACE;
  }
  OnDevice g(pool->device);
  if (!g.ok) return cuda_fail("cudaSetDevice", cudaGetLastError());
  Fp8EvictCall c;
  c.block_tables = block_tables;
  c.bt_stride = bt_stride;
  c.context_lens = context_lens;
  c.batch = batch;
  c.max_ctx = max_ctx;
  c.new_tables = new_tables;
  c.new_stride = new_stride;
  c.budget = budget;
  c.recent = recent;
  c.kept = kept;
  c.new_lens = new_lens;
  return launch_fp8_evict(*pool, c, static_cast<cudaStream_t>(stream));
}

int clove_fp8_copy_blocks(clove_fp8_pool_t pool, const int32_t* src, const int32_t* dst, int n, void* stream) {
  if (!pool || n < 0) return fail(CLOVE_ERR_INVALID_ARG, "fp8_copy_blocks: bad arguments");
  if (n == 0) return CLOVE_OK;
  if (!src || !dst) return fail(CLOVE_ERR_INVALID_ARG, "fp8_copy_blocks: null pointer");
  OnDevice g(pool->device);
  if (!g.ok) return cuda_fail("cudaSetDevice", cudaGetLastError());
  return launch_fp8_copy(*pool, src, dst, n, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
