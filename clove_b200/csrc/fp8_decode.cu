// Decode over the 8-bit cache.
//
// The work partition, the pipeline (one producer warp, a ring of stages in
// shared memory, consumer warps that own whole stages), the merge and the
// combine are those of the other decodes (decode_common.cuh, combine.cuh).
// The unit of the partition is a slice of up to 32 tokens of one (block, KV
// head) tile: kSlice = min(block_size, 32), so a block of 256 tokens is eight
// slices with one scale.
//
// Mathematics.  HBM bounds this kernel, so the arithmetic is held to what
// float32 would give instead of spending the slack elsewhere:
//   - an e4m3 code is exact in f16, so K and V enter the tensor cores exactly,
//     and their block scales are applied to scores and weights in f32;
//   - a query element is the sum of two halves (f16 queries and, but for
//     elements 2^-31 below the row's largest, bf16 queries are one half), a
//     weight the sum of two halves.  The m16n8k16 MMA has 16 rows and a KV
//     head at most 8 queries: the high halves are rows 0..7, the low halves
//     rows 8..15 of the same instruction, and the two results meet in one
//     thread's registers;
//   - weights are 2^(z - m + 14): the f16 range below the largest weight is 14
//     binades longer than with 2^(z - m), so a weight is off by at most 2^-39
//     of the row's largest however many light tokens there are;
//   - the scales of V differ from block to block: a warp keeps the largest
//     power of two seen, `vref`, in its accumulators' unit (as it keeps the
//     running maximum m), and multiplies weights by v_scale / vref <= 2;
//   - the value sum of 32 tokens starts from zero in the tensor cores and is
//     added to f32 registers, so the chain of truncated tensor-core additions
//     is two long, not as long as the sequence.
//
// Shared memory.  A tile is contiguous in HBM; it is copied as rows of 128
// bytes (64 for head_dim 64) with the hardware swizzle: the 16-byte chunk at
// byte offset x lands at x ^ (((x >> 7) & 7) << 4) (& 3 for 64-byte rows), so
// the 16-byte reads below touch every bank once (the V reads of head_dim 64
// and 256 twice).
#include <algorithm>
#include <cstdlib>
#include <mutex>
#include <unordered_map>

#include "combine.cuh"
#include "common.cuh"
#include "decode_common.cuh"
#include "fp8_common.cuh"

namespace clove {

struct Fp8Args : DecodeArgs {
  static constexpr bool kPublishFlags = false;  // flags go straight to the pool's word
  static constexpr bool kKeepsRowState = true;
  float* scales;       // [2, num_blocks, num_kv_heads]
  float* mass;         // null: the pool keeps none
  const float* slopes;  // null: no distance bias
  float2* row_state;   // [batch, Hq]: (M, 1 / L) of each output row (accumulate only, else null)
  float* z;            // [batch, Hq, z_stride]: scores in the log2 domain (accumulate only, else null)
  long long z_stride;
  int real_block;      // tokens per cache block; DecodeArgs::block_size is the slice
  int sub_shift;       // log2(real_block / slice)
  int window;
  int append_here;     // 1: the producers append the new tokens (see fp8_append_kernel)
  int direct;          // 1: CTA c takes segment c whole, nothing is split
  float scale, softcap;
};

constexpr int kSlice = 32;
constexpr int kMaxSb = 16;  // slices per stage: 128 tokens of 8 (head_dim 64)

// Stage tokens: 16 KB of K and V.
template <int D>
constexpr int stage_tokens() {
  return D == 64 ? 128 : D == 128 ? 64 : 32;
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// First slice of sequence b that the call reads.
__device__ __forceinline__ int first_slice(const Fp8Args& a, int L) {
  return a.window > 0 ? max(0, L - a.window) / a.block_size : 0;
}
__device__ __forceinline__ int num_slices(const Fp8Args& a, int L) {
  return (L + a.block_size - 1) / a.block_size - first_slice(a, L);
}

// partition_prologue (decode_common.cuh) for segments that start at a window.
template <int D>
__device__ void fp8_prologue(const Fp8Args& a, WalkStart* out) {
  const int tid = threadIdx.x, lane = tid & 31, nt = blockDim.x, H = a.num_kv_heads;
  if (a.direct) {
    const int b = blockIdx.x / H, h = blockIdx.x - b * H;
    const int raw = __ldg(a.context_lens + b);
    const int L = clamp_ctx(a.context_lens, b, a.max_ctx, a.append);
    if (h == 0 && tid == 0 && raw != L - a.append) atomicOr(a.err, CLOVE_FLAG_CTX_RANGE);
    if (L == 0)
      for (int i = tid; i < a.group * D; i += nt) a.out[(size_t)blockIdx.x * a.group * D + i] = 0.f;
    if (tid == 0) {
      out->lo = 0;
      out->hi = L > 0 ? num_slices(a, L) + a.seg_cost : 0;
      out->b = L > 0 ? b : -1;
      out->h = h;
      out->off = 0;
    }
    __syncthreads();
    return;
  }
  __shared__ int warp_tot[32];
  __shared__ long long s_sum;
  __shared__ int s_found;
  const int row_floats = H * a.group * D;
  if (tid == 0) {
    s_sum = 0;
    s_found = 0;
  }
  __syncthreads();
  long long mine = 0;
  for (int b = tid; b < a.batch; b += nt) {
    const int raw = __ldg(a.context_lens + b);
    const int L = clamp_ctx(a.context_lens, b, a.max_ctx, a.append);
    if (blockIdx.x == 0 && raw != L - a.append) atomicOr(a.err, CLOVE_FLAG_CTX_RANGE);
    if (L > 0) mine += num_slices(a, L) + a.seg_cost;
    if (L == 0 && b % a.num_ctas == (int)blockIdx.x) {
      float4* row = reinterpret_cast<float4*>(a.out + (size_t)b * row_floats);
      for (int i = 0; i < row_floats / 4; ++i) row[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0 && mine) atomicAdd(reinterpret_cast<unsigned long long*>(&s_sum), (unsigned long long)mine);
  __syncthreads();
  const long long W = s_sum * H, P = a.num_ctas;
  const long long lo = range_begin(blockIdx.x, W, P), hi = range_begin(blockIdx.x + 1, W, P);
  if (tid == 0) {
    out->lo = lo;
    out->hi = hi;
    out->b = -1;
    out->h = 0;
    out->off = 0;
    if (blockIdx.x == 0) *a.total = W;
  }
  if (lo < hi) {
    long long carry = 0;
    for (int base = 0; base < a.batch; base += nt) {
      const int b = base + tid;
      const int L = b < a.batch ? clamp_ctx(a.context_lens, b, a.max_ctx, a.append) : 0;
      const int len = L > 0 ? num_slices(a, L) + a.seg_cost : 0;
      int tot;
      const int excl = block_excl_scan(len, warp_tot, &tot);
      const long long s0 = (carry + excl) * H;
      if (len > 0 && s0 <= lo && lo < s0 + (long long)len * H) {
        const long long r = lo - s0;
        out->b = b;
        out->h = (int)(r / len);
        out->off = (int)(r - (r / len) * len);
        s_found = 1;
      }
      carry += tot;
      __syncthreads();
      if (s_found) break;
    }
  }
  __syncthreads();
  if (tid == 0) {
    int4 d = make_int4(-1, 0, 0, 0);
    if (out->b >= 0)
      d = make_int4(out->b, out->h, out->off,
                    num_slices(a, clamp_ctx(a.context_lens, out->b, a.max_ctx, a.append)) + a.seg_cost);
    a.desc[blockIdx.x] = d;
  }
}

// The new token of head h: settles the block's scale with the row, rounds the
// rows already there if it grew, writes the row.  One warp, D / 8 lanes hold
// the row; nobody else reads or writes this tile before the copies that the
// caller issues next.
template <typename T, int D>
__device__ void fp8_append_row(const Fp8Args& a, int b, int h, int L, int lane) {
  const int bs = a.real_block, H = a.num_kv_heads, pos = L - 1, off = pos & (bs - 1);
  const int phys = __ldg(a.block_tables + (size_t)b * a.bt_stride + pos / bs);
  if (phys < 0 || phys >= a.num_blocks) {
    if (lane == 0) atomicOr(a.err, CLOVE_FLAG_BLOCK_OOB);
    return;
  }
  const size_t tile = (size_t)phys * H + h, src = ((size_t)b * H + h) * D + lane * 8;
  float v[2][8] = {};
  float old[2];
  if (lane < D / 8) {
    load_vec_f32<T, 8>(static_cast<const T*>(a.k_new) + src, v[0]);
    load_vec_f32<T, 8>(static_cast<const T*>(a.v_new) + src, v[1]);
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) old[p] = off == 0 ? 0.f : __ldcg(a.scales + (size_t)p * a.num_blocks * H + tile);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(v[p][i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float s = fmaxf(old[p], fp8_scale_for(amax)), inv = 1.f / s;
    unsigned char* rows = static_cast<unsigned char*>(p ? a.v_cache : a.k_cache) + tile * bs * D;
    if (old[p] > 0.f && s > old[p]) {
      const float ratio = old[p] / s;
      uint4* w = reinterpret_cast<uint4*>(rows);
#pragma unroll 4
      for (int i = lane; i < bs * (D / 16); i += 32) {
        if (i / (D / 16) == off) continue;  // written below
        const uint4 c = __ldcg(w + i);
        const uint2 lo = fp8_rescale8(make_uint2(c.x, c.y), ratio), hi = fp8_rescale8(make_uint2(c.z, c.w), ratio);
        w[i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    }
    if (lane < D / 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[p][i] *= inv;
      *reinterpret_cast<uint2*>(rows + (size_t)off * D + lane * 8) = fp8_pack8(v[p]);
    }
    if (lane == 0) a.scales[(size_t)p * a.num_blocks * H + tile] = s;
  }
  if (lane == 0 && a.mass != nullptr && a.z == nullptr) a.mass[tile * bs + off] = 0.f;
  fence_proxy_async_global();
  __syncwarp();
}

// The new tokens of all sequences, a warp per (KV head, sequence), ahead of
// the decode.  Used where a block is more than one slice: another CTA may then
// stream the earlier slices of the block that an append rescales.
template <typename T, int D>
__global__ void __launch_bounds__(32) fp8_append_kernel(const Fp8Args a) {
  griddep_wait();
  const int b = blockIdx.y;
  fp8_append_row<T, D>(a, b, blockIdx.x, clamp_ctx(a.context_lens, b, a.max_ctx, 1), threadIdx.x);
}

// The producer warp (produce() of decode_common.cuh for this cache): walks
// the CTA's range, posts each piece, appends the new token where the piece
// ends its sequence, and streams the slices.  Table entries and scales are
// loaded 32 slices at a time, half a group ahead of their use.
template <typename T, int D>
__device__ void fp8_produce(const Fp8Args& a, const CUtensorMap* tm_k, const CUtensorMap* tm_v, const SmemPtrs& sm,
                            const SmemPlan& sp, float2* scl, int sb, const WalkStart& ws) {
  constexpr int RPT = D >= 128 ? D / 128 : 1;  // rows of the copies' tensor map per token
  const int lane = threadIdx.x & 31;
  const int vs = a.block_size, H = a.num_kv_heads, Hq = H * a.group;
  const uint32_t tile_bytes = (uint32_t)(vs * D);
  const uint32_t q_bytes = (uint32_t)(a.group * D * (int)sizeof(T));
  const uint64_t pol = policy_evict_first();
  int slot = 0, uk = 0;
  uint32_t phase = 0, uphase = 0;
  bool aborted = false;

  // Lane i: the table entry of slice j0 + i of the piece (unchecked) ...
  auto entry = [&](const Unit& x, int j0) {
    const int j = j0 + lane;
    return j < x.nblk ? __ldg(a.block_tables + (size_t)x.b * a.bt_stride + ((x.blk0 + j) >> a.sub_shift)) : 0;
  };
  // ... and what it leads to: the copy's first row, the scales.  Entries
  // outside the pool are flagged and replaced by block 0 (never followed).
  struct Slice {
    int row;
    float sk, sv;
  };
  auto resolve = [&](const Unit& x, int j0, int phys) {
    const int j = j0 + lane;
    Slice s = {0, 0.f, 0.f};
    if (j < x.nblk) {
      if (phys < 0 || phys >= a.num_blocks) {
        atomicOr(a.err, CLOVE_FLAG_BLOCK_OOB);
        phys = 0;
      }
      const size_t tile = (size_t)phys * H + x.h;
      s.row = ((int)tile * a.real_block + ((x.blk0 + j) & ((1 << a.sub_shift) - 1)) * vs) * RPT;
      s.sk = __ldcg(a.scales + tile);
      s.sv = __ldcg(a.scales + (size_t)a.num_blocks * H + tile);
    }
    return s;
  };

  const int alpha = a.seg_cost;
  int b = ws.b, h = ws.h, off = ws.off, npiece = 0;
  long long pos = ws.lo;
  int L = b >= 0 ? clamp_ctx(a.context_lens, b, a.max_ctx, a.append) : 0;
  int nb = L > 0 ? num_slices(a, L) : 0;
  auto next_piece = [&](Unit& x, int& e0) -> bool {
    while (b >= 0 && pos < ws.hi) {
      const int len = nb + alpha;
      const int span = (int)min((long long)(len - off), ws.hi - pos);
      const int r0 = max(off, alpha), r1 = off + span;
      const bool piece = r1 > r0;
      if (piece) {
        x.u = 0;
        x.b = b;
        x.h = h;
        x.L = L;
        x.blk0 = first_slice(a, L) + r0 - alpha;
        x.nblk = r1 - r0;
        x.nstages = (x.nblk + sb - 1) / sb;
        x.complete = r0 == alpha && r1 == len;
        x.slot = npiece == 0 ? 0 : 1;
        x.last = r1 == len;
      }
      pos += span;
      off += span;
      if (off == len && pos < ws.hi) {
        off = 0;
        if (++h == H) {
          h = 0;
          do {
            if (++b >= a.batch) {  // (cannot happen while pos < hi; bounds the walk regardless)
              b = -1;
              break;
            }
            L = clamp_ctx(a.context_lens, b, a.max_ctx, a.append);
            nb = L > 0 ? num_slices(a, L) : 0;
          } while (L == 0);
        }
      }
      if (piece) {
        e0 = entry(x, 0);
        ++npiece;
        return true;
      }
    }
    return false;
  };

  int e0 = 0;
  Unit x;
  bool have = next_piece(x, e0);
  bool first = true;
  while (true) {
    int ok = 1;
    if (lane == 0) {
      if (*sm.misc || !mbar_wait_bounded(&sm.uempty[uk], uphase ^ 1, a.err, a.wait_limit)) {
        ok = 0;
        *sm.misc = 1;
      } else if (!have) {
        sm.slots[uk].valid = 0;
        mbar_arrive(&sm.ufull[uk]);
      } else {
        sm.slots[uk].x = x;
        sm.slots[uk].valid = 1;
        mbar_arrive_expect_tx(&sm.ufull[uk], q_bytes);
        const T* qsrc = static_cast<const T*>(a.q) + ((size_t)x.b * Hq + (size_t)x.h * a.group) * D;
        bulk_load(sm.qbuf + uk * sp.q_stride, qsrc, q_bytes, &sm.ufull[uk]);
      }
    }
    ok = __shfl_sync(0xffffffffu, ok, 0);
    if (!ok) {
      aborted = true;
      break;
    }
    if (!have) break;
    if (++uk == kUnitRing) {
      uk = 0;
      uphase ^= 1;
    }

    if (a.append_here && x.last) fp8_append_row<T, D>(a, x.b, x.h, x.L, lane);
    Slice cur = resolve(x, 0, e0), nxt = {0, 0.f, 0.f};
    int e1 = x.nblk > 32 ? entry(x, 32) : 0;
    int e2 = 0;
    Unit x2;
    bool have2 = false;
    const int claim_at = min(x.nstages - 1, a.nstage / 2);
    for (int s = 0; s < x.nstages; ++s) {
      const int j0 = s * sb;
      if ((j0 & 31) == 0 && j0 > 0) {
        cur = nxt;
        if (j0 + 32 < x.nblk) e1 = entry(x, j0 + 32);
      }
      if ((j0 & 31) == 16 && j0 + 16 < x.nblk) nxt = resolve(x, j0 + 16, e1);
      const int n = min(sb, x.nblk - j0);
      int ready = 1;
      if (lane == 0 && (*sm.misc || !mbar_wait_bounded(&sm.empty[slot], phase ^ 1, a.err, a.wait_limit))) {
        ready = 0;
        *sm.misc = 1;
      }
      ready = __shfl_sync(0xffffffffu, ready, 0);
      if (!ready) {
        aborted = true;
        break;
      }
      __syncwarp();
      // the stage's scales, zero where it has no slice
      const int from = (j0 + lane) & 31;
      const float sk = __shfl_sync(0xffffffffu, cur.sk, from), sv = __shfl_sync(0xffffffffu, cur.sv, from);
      if (lane < sb) scl[slot * kMaxSb + lane] = lane < n ? make_float2(sk, sv) : make_float2(0.f, 0.f);
      __syncwarp();
      const bool stall = a.inject_stall && first && s == 0;  // test hook: this stage is never filled
      if (lane == 0 && !stall) mbar_arrive_expect_tx(&sm.full[slot], 2u * tile_bytes * (uint32_t)n);
      __syncwarp();
      const int row = __shfl_sync(0xffffffffu, cur.row, from);
      if (lane < n && !stall) {
        unsigned char* st = sm.ring + (size_t)slot * sp.stage_bytes;
        tma_load_2d(st + lane * tile_bytes, tm_k, &sm.full[slot], 0, row, pol);
        tma_load_2d(st + (sb + lane) * tile_bytes, tm_v, &sm.full[slot], 0, row, pol);
      }
      if (++slot == a.nstage) {
        slot = 0;
        phase ^= 1;
      }
      if (s == claim_at) have2 = next_piece(x2, e2);
    }
    if (aborted) break;
    have = have2;
    x = x2;
    e0 = e2;
    first = false;
  }
  if (aborted && lane == 0) {
    // drain: the last nstage stages and unit posts may still be in flight
    int s = slot;
    uint32_t ph = phase;
    for (int k = 0; k < a.nstage; ++k) {
      if (--s < 0) {
        s = a.nstage - 1;
        ph ^= 1;
      }
      for (uint32_t i = 0; i < a.wait_limit; ++i)
        if (mbar_try_wait(&sm.full[s], ph)) break;
    }
    int k2 = uk;
    uint32_t uph = uphase;
    for (int k = 0; k < kUnitRing; ++k) {
      if (--k2 < 0) {
        k2 = kUnitRing - 1;
        uph ^= 1;
      }
      for (uint32_t i = 0; i < a.wait_limit; ++i)
        if (mbar_try_wait(&sm.ufull[k2], uph)) break;
    }
  }
}

__device__ __forceinline__ void fence_proxy_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// D(16x8, f32) += A(16x16, f16) * B(16x8, f16)
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Codes in the low / high 16 bits of w as an f16 pair.
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) { return half2_bits(fp8_unpack2(w)); }
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) { return half2_bits(fp8_unpack2(w >> 16)); }

// x, y = hi + lo, each a pair of halves.
__device__ __forceinline__ void split_halves(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = half2_bits(h);
  lo = half2_bits(__floats2half2_rn(x - f.x, y - f.y));
}

// Byte offset of x within a stage's K (or V) region after the copy's swizzle.
template <int D>
__device__ __forceinline__ uint32_t swz(uint32_t x) {
  return D >= 128 ? x ^ (((x >> 7) & 7) << 4) : x ^ (((x >> 7) & 3) << 4);
}

// The K chunk (16 dims) that lane column tq reads as its j-th: the MMA's
// contraction may take the dims in any order, this one keeps the eight lanes
// of a shared-memory phase on distinct banks.
template <int D>
__device__ __forceinline__ int k_chunk(int tq, int j) {
  if (D == 64) return tq;
  if (D == 128) return 2 * tq + j;
  return (j >> 1) * 8 + (tq & 1) + 4 * (tq >> 1) + 2 * (j & 1);
}

// The power of two at or below x > 0 (within the range whose inverse is normal).
__device__ __forceinline__ float floor_pow2(float x) {
  return __int_as_float(min(max(__float_as_int(x) & 0x7f800000, 1 << 23), 252 << 23));
}
__device__ __forceinline__ float inv_pow2(float x) { return __int_as_float((254 << 23) - __float_as_int(x)); }

template <typename T, int D, int NCW>
__global__ void __launch_bounds__((NCW + 1) * 32)
    fp8_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const Fp8Args a) {
  constexpr int G = 8;
  constexpr bool kTwoHalves = sizeof(T) == 4;  // f32 queries need the low halves
  constexpr int KJ = D / 64;                   // 16-byte K chunks per lane and token
  constexpr int VB = D >= 128 ? 16 : 8;        // V bytes per lane and token (per 128 dims)
  constexpr int VH = D >= 128 ? D / 128 : 1;   // 128-dim halves
  constexpr int NT = D / 8;                    // n-tiles of the value sum
  const int vs = a.block_size, sb = a.stage_blocks, TT = sb * vs, group = a.group;

  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const SmemPlan sp = smem_plan(vs, D, 1, sb, a.nstage, NCW * group * state_stride(D) * (int)sizeof(float),
                                group * D * (int)sizeof(T), a.nscr);
  const SmemPtrs sm = smem_ptrs(smem, sp, a.nstage);
  float2* scl = reinterpret_cast<float2*>(reinterpret_cast<unsigned char*>(sm.scratch) + a.nscr * sp.scratch_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tensor_map(&tm_k);
    prefetch_tensor_map(&tm_v);
  }
  init_barriers(sm, a.nstage, NCW);
  __shared__ WalkStart walk;
  fp8_prologue<D>(a, &walk);

  if (warp == 0) {
    fp8_produce<T, D>(a, &tm_k, &tm_v, sm, sp, scl, sb, walk);
    return;
  }

  const int cw = warp - 1, g = lane >> 2, tq = lane & 3;
  const int vshift = 31 - __clz(vs);
  int gbase = 0, uk = 0, n_done = 0;
  uint32_t uphase = 0;
  UnitSlot us;

  while (wait_unit(a, sm, uk, uphase, us)) {
    const Unit x = us.x;
    // Query fragments: row g scaled by a power of two that puts its largest
    // element in [2^13, 2^14), undone in the score's factor.
    uint32_t qa[KJ * 4][kTwoHalves ? 4 : 2];
    float zf;  // score = dot * K scale * zf
    {
      const T* qrow = reinterpret_cast<const T*>(sm.qbuf + uk * sp.q_stride) + g * D;
      float amax = 0.f;
      if (g < group) {
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
          for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(Elem<T>::to_f(qrow[k_chunk<D>(tq, j) * 16 + i])));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const float unit = floor_pow2(amax);
      const int e = min((__float_as_int(unit) >> 23) - 127 - 13, 126);  // divide by 2^e
      const float up = __int_as_float((127 - max(e, -127)) << 23);
      zf = a.scale * __int_as_float((127 + max(e, -126)) << 23);
      if (e < -126) zf *= 0.5f;
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float f[4] = {0.f, 0.f, 0.f, 0.f};
          if (g < group) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = Elem<T>::to_f(qrow[k_chunk<D>(tq, j) * 16 + w * 4 + i]) * up;
          }
          uint32_t lo0, lo1;
          split_halves(f[0], f[1], qa[j * 4 + w][0], lo0);
          split_halves(f[2], f[3], qa[j * 4 + w][1], lo1);
          if constexpr (kTwoHalves) {
            qa[j * 4 + w][2] = lo0;
            qa[j * 4 + w][3] = lo1;
          }
        }
    }
    const int hq = x.h * group + g;
    const float cap = a.softcap;
    zf = cap > 0.f ? zf / cap : zf * kLog2e;
    const float slope = a.slopes != nullptr && g < group ? __ldg(a.slopes + hq) * kLog2e : 0.f;
    const int t_first = a.window > 0 ? max(0, x.L - a.window) : 0;  // first token attended to
    float* zrow = a.z != nullptr && g < group
                      ? a.z + ((size_t)x.b * a.num_kv_heads * group + hq) * a.z_stride
                      : nullptr;

    float m = -INFINITY, l = 0.f, vref = 0.f;
    float o[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = 0.f;

    bool aborted = false;
    const int ncw = a.ncw;
    // Stage gs belongs to warp gs % ncw; nstage is a multiple of ncw.
    for (int j = cw < ncw ? ((cw - gbase) % ncw + ncw) % ncw : x.nstages; j < x.nstages; j += ncw) {
      const int gs = gbase + j, slot = gs % a.nstage;
      if (!wait_or_abort(a, sm, &sm.full[slot], (uint32_t)(gs / a.nstage) & 1u)) {
        aborted = true;
        break;
      }
      unsigned char* kst = sm.ring + (size_t)slot * sp.stage_bytes;
      unsigned char* vst = kst + sb * sp.tile_stride;
      const float2* sc = scl + slot * kMaxSb;
      const int t_base = (x.blk0 + j * sb) * vs;  // token of the stage's first row
      const int hi = min(TT, min((x.blk0 + x.nblk) * vs, x.L) - t_base), lo = max(0, t_first - t_base);
      const bool ragged = lo > 0 || hi < TT;
      if (ragged) {
        // Rows outside [lo, hi) may hold NaN codes; their weights are 0, but
        // 0 * NaN is NaN, so clear those V rows.
        for (int i = lane; i < TT * (D / 16); i += 32) {
          const int tok = i / (D / 16);
          if (tok < lo || tok >= hi) *reinterpret_cast<uint4*>(vst + swz<D>(i * 16)) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      for (int p0 = 0; p0 < hi; p0 += 32) {
        // ---- scores of 32 tokens: four tiles of 8 ----
        float z[4][2], wv[4];
        float vmax = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint4 kw[KJ];
#pragma unroll
          for (int c = 0; c < KJ; ++c)
            kw[c] = *reinterpret_cast<const uint4*>(
                kst + swz<D>((uint32_t)((p0 + 8 * e + g) * D + k_chunk<D>(tq, c) * 16)));
          float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < KJ; ++c) {
            const uint32_t w[4] = {kw[c].x, kw[c].y, kw[c].z, kw[c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t* q = qa[c * 4 + i];
              if constexpr (kTwoHalves)
                mma_f16(s, q[0], q[2], q[1], q[3], codes_lo(w[i]), codes_hi(w[i]));
              else
                mma_f16(s, q[0], 0u, q[1], 0u, codes_lo(w[i]), codes_hi(w[i]));
            }
          }
          const float2 f = sc[(p0 + 8 * e) >> vshift];
          const float kf = f.x * zf;
          wv[e] = f.y;
          vmax = fmaxf(vmax, f.y);
          z[e][0] = (kTwoHalves ? s[0] + s[2] : s[0]) * kf;
          z[e][1] = (kTwoHalves ? s[1] + s[3] : s[1]) * kf;
        }
        if (cap > 0.f) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            z[e][0] = tanhf(z[e][0]) * (cap * kLog2e);
            z[e][1] = tanhf(z[e][1]) * (cap * kLog2e);
          }
        }
        if (a.slopes != nullptr) {
          const int back = t_base + p0 + 2 * tq - (x.L - 1);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            z[e][0] = fmaf(slope, (float)(back + 8 * e), z[e][0]);
            z[e][1] = fmaf(slope, (float)(back + 8 * e + 1), z[e][1]);
          }
        }
        if (zrow != nullptr) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (p0 + 8 * e + 2 * tq < hi)
              *reinterpret_cast<float2*>(zrow + t_base + p0 + 8 * e + 2 * tq) = make_float2(z[e][0], z[e][1]);
        }
        if (ragged) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int tok = p0 + 8 * e + 2 * tq + c;
              if (tok < lo || tok >= hi) z[e][c] = -INFINITY;
            }
        }
        // ---- online softmax of row g ----
        float mx = z[0][0];
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(z[e][0], z[e][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m, mx);
        const float ms = mn == -INFINITY ? 0.f : mn - 14.f;
        const float corr = m == -INFINITY ? 0.f : exp2f(m - mn);
        m = mn;
        const float vnew = fmaxf(vref, floor_pow2(vmax)), vinv = inv_pow2(vnew);
        const float oc = corr * (vref * vinv);
        vref = vnew;
        float ps = 0.f;
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0e = exp2f(z[e][0] - ms), p1e = exp2f(z[e][1] - ms);
          ps += p0e + p1e;
          const float f = wv[e] * vinv;
          split_halves(p0e * f, p1e * f, ph[e], pl[e]);
        }
        l = fmaf(l, corr, ps);
        // ---- value sum: two 16-token steps ----
        // Lane column g of an n-tile is dims g * VB + byte (of each 128-dim half).
#pragma unroll
        for (int half = 0; half < VH; ++half) {
          uint32_t vw[2][4][VB / 4];
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int tok = p0 + 16 * k + 2 * tq + (i & 1) + 8 * (i >> 1);
              const unsigned char* src = vst + swz<D>((uint32_t)(tok * D + half * 128 + g * VB));
              if constexpr (VB == 16) {
                const uint4 w = *reinterpret_cast<const uint4*>(src);
                vw[k][i][0] = w.x;
                vw[k][i][1] = w.y;
                vw[k][i][2] = w.z;
                vw[k][i][3] = w.w;
              } else {
                const uint2 w = *reinterpret_cast<const uint2*>(src);
                vw[k][i][0] = w.x;
                vw[k][i][1] = w.y;
              }
            }
#pragma unroll
          for (int w = 0; w < VB / 4; ++w) {
            uint32_t b0[2][2], b1[2][2];  // [step][dims 0,1 | 2,3]: token pairs of two dims
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              b0[k][0] = __byte_perm(vw[k][0][w], vw[k][1][w], 0x5140);
              b0[k][1] = __byte_perm(vw[k][0][w], vw[k][1][w], 0x7362);
              b1[k][0] = __byte_perm(vw[k][2][w], vw[k][3][w], 0x5140);
              b1[k][1] = __byte_perm(vw[k][2][w], vw[k][3][w], 0x7362);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const uint32_t x0 = i & 1 ? codes_hi(b0[k][i >> 1]) : codes_lo(b0[k][i >> 1]);
                const uint32_t x1 = i & 1 ? codes_hi(b1[k][i >> 1]) : codes_lo(b1[k][i >> 1]);
                mma_f16(d, ph[2 * k], pl[2 * k], ph[2 * k + 1], pl[2 * k + 1], x0, x1);
              }
              float* on = o[half * 16 + w * 4 + i];
              on[0] = fmaf(on[0], oc, d[0] + d[2]);
              on[1] = fmaf(on[1], oc, d[1] + d[3]);
            }
          }
        }
      }
      if (ragged) fence_proxy_async_smem();  // order the cleared rows before the slot's next copy
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[slot]);
    }
    if (aborted) return;  // the abort flag is up; every other warp leaves at its next wait
    gbase += x.nstages;

    // ---- publish (acc, m - 14, l) of the group's rows, hand off ----
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int sbuf = n_done % a.nscr;
    if (!wait_or_abort(a, sm, &sm.scr_empty[sbuf], ((uint32_t)(n_done / a.nscr) & 1u) ^ 1u)) return;
    float* scr = sm.scratch + sbuf * sm.scratch_floats + (size_t)(cw * group + g) * state_stride(D);
    if (g < group) {
      // thread (g, tq) holds columns 2 tq and 2 tq + 1 of every n-tile
#pragma unroll
      for (int half = 0; half < VH; ++half)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < VB; i += 4)
            *reinterpret_cast<float4*>(scr + half * 128 + (2 * tq + c) * VB + i) =
                make_float4(o[half * 16 + i][c] * vref, o[half * 16 + i + 1][c] * vref, o[half * 16 + i + 2][c] * vref,
                            o[half * 16 + i + 3][c] * vref);
      if (tq == 0) {
        scr[D] = m - 14.f;
        scr[D + 1] = l;
      }
    }
    hand_off<D, G, NCW>(a, sm, us, sbuf, uk, lane);
    ++n_done;
    if (++uk == kUnitRing) {
      uk = 0;
      uphase ^= 1;
    }
  }
}

// ---------------------------------------------------------------------------
// weights: mass += sum over the group of 2^(z - M) / L
// ---------------------------------------------------------------------------
constexpr int kMassThreads = 256, kMassTokens = 1024;

__global__ void __launch_bounds__(kMassThreads) fp8_mass_kernel(const Fp8Args a) {
  const int b = blockIdx.z, h = blockIdx.y, H = a.num_kv_heads, G = a.group, bs = a.real_block;
  griddep_wait();
  const int L = clamp_ctx(a.context_lens, b, a.max_ctx, a.append);
  const int t0 = a.window > 0 ? max(0, L - a.window) : 0;
  const int from = max(t0, (int)blockIdx.x * kMassTokens), to = min(L, ((int)blockIdx.x + 1) * kMassTokens);
  if (from >= to) return;
  const size_t row = (size_t)b * H * G + (size_t)h * G;
  for (int t = from + threadIdx.x; t < to; t += kMassThreads) {
    int blk = __ldg(a.block_tables + (size_t)b * a.bt_stride + t / bs);
    const bool mine = a.append && t == L - 1;
    if (blk < 0 || blk >= a.num_blocks) {
      if (mine) continue;  // the token was not written
      blk = 0;
    }
    float w = 0.f;
#pragma unroll 8
    for (int g = 0; g < G; ++g) {
      const float2 st = __ldg(a.row_state + row + g);
      w = fmaf(exp2f(__ldcs(a.z + (row + g) * a.z_stride + t) - st.x), st.y, w);
    }
    float* dst = a.mass + ((size_t)blk * H + h) * bs + (t & (bs - 1));
    *dst = mine ? w : *dst + w;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int kFp8Warps = 4;
constexpr int kFp8Ring = 96 * 1024;

// Stream positions charged per segment for a piece's fixed cost: 40 KB worth
// of slices, as for the other decodes.
static int fp8_segment_cost(int slice, int head_dim) {
  const int bytes = 2 * slice * head_dim;
  return (40 * 1024 + bytes - 1) / bytes;
}

struct Fp8Layout {
  int max_ctas;
  long long z_stride;
  size_t off_total, off_desc, off_partials, off_rows, off_z, total;
};

static Fp8Layout fp8_layout(const clove_fp8_pool& pool, int batch, int num_q_heads, int max_ctx, int accumulate) {
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  Fp8Layout L;
  L.max_ctas = pool.num_sms * kMaxCtasPerSm;
  L.z_stride = ((long long)max_ctx + 4) & ~3LL;
  const int group = std::max(1, num_q_heads / pool.num_kv_heads);
  L.off_total = 0;
  L.off_desc = 256;
  L.off_partials = up(L.off_desc + sizeof(int4) * (size_t)L.max_ctas);
  L.off_rows = up(L.off_partials + sizeof(float) * (size_t)L.max_ctas * 2 * group * state_stride(pool.head_dim));
  L.off_z = L.off_rows;
  L.total = L.off_rows;
  if (accumulate) {
    L.off_z = up(L.off_rows + sizeof(float2) * (size_t)batch * num_q_heads);
    L.total = up(L.off_z + sizeof(float) * (size_t)batch * num_q_heads * L.z_stride);
  }
  return L;
}

size_t fp8_decode_workspace(const clove_fp8_pool& pool, int batch, int num_q_heads, int max_ctx, int accumulate) {
  return fp8_layout(pool, batch, num_q_heads, max_ctx, accumulate).total;
}

// One plane of codes as rows of 128 bytes (64 for head_dim 64), a box being
// one slice of a tile.
static int fp8_plane_map(CUtensorMap* map, void* base, const clove_fp8_pool& pool, int slice) {
  auto fn = tensor_map_encoder();
  if (!fn) {
    set_last_error("cuTensorMapEncodeTiled unavailable from the driver");
    return CLOVE_ERR_CUDA;
  }
  const cuuint32_t inner = pool.head_dim >= 128 ? 128 : 64, rpt = pool.head_dim / inner;
  cuuint64_t dims[2] = {inner, (cuuint64_t)pool.plane_bytes / inner};
  cuuint64_t strides[1] = {inner};
  cuuint32_t box[2] = {inner, (cuuint32_t)slice * rpt};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r =
      fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         inner == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("cuTensorMapEncodeTiled failed (%d) for head_dim %d block_size %d", (int)r, pool.head_dim,
                   pool.block_size);
    return CLOVE_ERR_CUDA;
  }
  return CLOVE_OK;
}

int fp8_encode_maps(clove_fp8_pool& pool) {
  const int slice = std::min(pool.block_size, kSlice);
  const int rc = fp8_plane_map(&pool.tm_k, pool.codes, pool, slice);
  return rc ? rc : fp8_plane_map(&pool.tm_v, pool.codes + pool.plane_bytes, pool, slice);
}

template <typename K, typename... A>
static cudaError_t launch_chained(K kern, dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Launch configuration of one kernel instance, worked out once per (device,
// slice, group).
struct Fp8Cfg {
  int nstage, smem, ctas;
};

template <typename T, int D>
static int fp8_cfg(const clove_fp8_pool& pool, int slice, int group, int nscr, Fp8Cfg* out) {
  static std::mutex mu;
  static std::unordered_map<long long, Fp8Cfg> cache;
  static std::unordered_map<int, int> attr;  // device -> shared memory the kernel may use there
  auto kern = fp8_decode_kernel<T, D, kFp8Warps>;
  const long long key = ((long long)pool.device << 32) | ((long long)slice << 8) | group;
  std::lock_guard<std::mutex> lk(mu);
  auto it = cache.find(key);
  if (it != cache.end()) {
    *out = it->second;
    return CLOVE_OK;
  }
  static const int ring_kb = [] {
    const char* v = std::getenv("CLOVE_DECODE_RING_KB");
    return v ? std::atoi(v) : 0;
  }();
  const int ring = ring_kb > 0 ? ring_kb * 1024 : kFp8Ring;
  const int sb = stage_tokens<D>() / slice;
  const int scratch = kFp8Warps * group * state_stride(D) * 4, qb = group * D * (int)sizeof(T);
  Fp8Cfg c;
  const int stage = smem_plan(slice, D, 1, sb, 1, scratch, qb, nscr).stage_bytes;
  c.nstage = std::max(1, ring / stage / kFp8Warps) * kFp8Warps;
  c.smem = smem_plan(slice, D, 1, sb, c.nstage, scratch, qb, nscr).total + c.nstage * kMaxSb * (int)sizeof(float2) + 1024;
  if (c.smem > attr[pool.device]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, c.smem);
    if (e != cudaSuccess) return fp8_launch_status("cudaFuncSetAttribute", e);
    attr[pool.device] = c.smem;
  }
  int occ = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, (kFp8Warps + 1) * 32, c.smem) != cudaSuccess ||
      occ < 1) {
    cudaGetLastError();
    occ = 1;
  }
  c.ctas = pool.num_sms * std::min(occ, kMaxCtasPerSm);
  cache[key] = c;
  *out = c;
  return CLOVE_OK;
}

template <typename T, int D>
static int run_fp8(const clove_fp8_pool& pool, Fp8Args& a, cudaStream_t stream) {
  a.stage_blocks = stage_tokens<D>() / a.block_size;
  a.nscr = a.group > 4 ? 2 : 1;
  Fp8Cfg c;
  int rc = fp8_cfg<T, D>(pool, a.block_size, a.group, a.nscr, &c);
  if (rc) return rc;
  a.nstage = c.nstage;
  a.ncw = kFp8Warps;
  a.num_ctas = a.direct ? a.batch * a.num_kv_heads : c.ctas;
  if (!a.direct && (a.num_ctas > pool.num_sms * kMaxCtasPerSm || a.num_ctas > kCombineMaxPieces)) {
    set_last_error("fp8_decode: %d CTAs exceed the workspace bound", a.num_ctas);
    return CLOVE_ERR_UNSUPPORTED;
  }
  if (a.append && !a.append_here) {
    rc = fp8_launch_status("fp8_decode append launch", launch_chained(fp8_append_kernel<T, D>, dim3(a.num_kv_heads, a.batch),
                                                                     32, 0, stream, a));
    if (rc) return rc;
    count_launches(1);
  }
  rc = fp8_launch_status("fp8_decode launch",
                         launch_chained(fp8_decode_kernel<T, D, kFp8Warps>, dim3(a.num_ctas), (kFp8Warps + 1) * 32,
                                        c.smem, stream, pool.tm_k, pool.tm_v, a));
  if (rc) return rc;
  count_launches(1);
  if (!a.direct) {
    rc = fp8_launch_status("fp8_decode combine launch",
                           launch_chained(combine_kernel<D, Fp8Args>, dim3(std::max(1, a.num_ctas - 1)),
                                          kCombineThreads, 0, stream, a));
    if (rc) return rc;
    count_launches(1);
  }
  if (a.z != nullptr) {
    const dim3 grid((a.max_ctx + kMassTokens - 1) / kMassTokens, a.num_kv_heads, a.batch);
    rc = fp8_launch_status("fp8_decode weights launch", launch_chained(fp8_mass_kernel, grid, kMassThreads, 0, stream, a));
    if (rc) return rc;
    count_launches(1);
  }
  return CLOVE_OK;
}

template <typename T>
static int run_fp8_dim(const clove_fp8_pool& pool, Fp8Args& a, cudaStream_t stream) {
  switch (pool.head_dim) {
    case 64: return run_fp8<T, 64>(pool, a, stream);
    case 128: return run_fp8<T, 128>(pool, a, stream);
    default: return run_fp8<T, 256>(pool, a, stream);
  }
}

int launch_fp8_decode(const clove_fp8_pool& pool, const Fp8DecodeCall& c, cudaStream_t stream) {
  const Fp8Layout L = fp8_layout(pool, c.batch, c.num_q_heads, c.max_ctx, c.scores.accumulate);
  unsigned char* ws = static_cast<unsigned char*>(c.workspace);
  const int slice = std::min(pool.block_size, kSlice);
  Fp8Args a = {};
  a.q = c.q;
  a.k_new = c.k_new;
  a.v_new = c.v_new;
  a.k_cache = pool.codes;
  a.v_cache = pool.codes + pool.plane_bytes;
  a.block_tables = c.block_tables;
  a.context_lens = c.context_lens;
  a.out = c.out;
  a.total = reinterpret_cast<long long*>(ws + L.off_total);
  a.desc = reinterpret_cast<int4*>(ws + L.off_desc);
  a.partials = reinterpret_cast<float*>(ws + L.off_partials);
  a.err = pool.flags;
  a.bt_stride = c.bt_stride;
  a.batch = c.batch;
  a.num_kv_heads = pool.num_kv_heads;
  a.num_blocks = pool.num_blocks;
  a.block_size = slice;
  a.seg_cost = fp8_segment_cost(slice, pool.head_dim);
  a.max_ctx = c.max_ctx;
  a.group = c.num_q_heads / pool.num_kv_heads;
  a.append = c.k_new ? 1 : 0;
  a.wait_limit = debug_wait_limit();
  a.inject_stall = debug_inject_stall();
  a.scales = pool.scales;
  a.mass = pool.mass;
  a.slopes = c.scores.alibi_slopes;
  a.real_block = pool.block_size;
  for (a.sub_shift = 0; (slice << a.sub_shift) < pool.block_size;) ++a.sub_shift;
  a.window = c.scores.window;
  a.scale = c.scale;
  a.softcap = c.scores.softcap;
  if (c.scores.accumulate) {
    a.row_state = reinterpret_cast<float2*>(ws + L.off_rows);
    a.z = reinterpret_cast<float*>(ws + L.off_z);
    a.z_stride = L.z_stride;
  }
  a.direct = 0;
  a.append_here = a.append && (a.direct || a.sub_shift == 0);
  switch (c.dtype) {
    case CLOVE_DTYPE_F32: return run_fp8_dim<float>(pool, a, stream);
    case CLOVE_DTYPE_F16: return run_fp8_dim<__half>(pool, a, stream);
    default: return run_fp8_dim<__nv_bfloat16>(pool, a, stream);
  }
}

}  // namespace clove
