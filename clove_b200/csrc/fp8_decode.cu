// Decode over the 8-bit cache.
//
// The work partition, the pipeline (one producer warp, a ring of stages in
// shared memory, consumer warps that own whole stages), the merge and the
// combine are those of the other decodes (decode_common.cuh, combine.cuh).
// The unit of the partition is a slice of one (block, KV head) tile: the tile,
// or the part of it that fills a stage (16 KB of K and V: 64 tokens at head_dim
// 128), so a block of 256 such tokens is four slices with one scale.
//
// Measured (heads of 128, bf16): 8 sequences of 32k to 131k tokens, 64 / 8 heads
// 217 us (0.97 of a copy's rate; 228 to 248 in loops that reach the power
// limit); 128 ragged sequences of 1300 tokens on average, 32 / 8 heads, with
// append 66.5 us (0.72: start, hand-offs and combine); 256 of a window of 1024
// with capped scores 113 us (0.66: hand-offs and instruction fetch).
//
// Mathematics.  HBM bounds this kernel, so its slack goes into arithmetic close
// to float32's.  What is rounded to fewer bits than that is named:
//   - an e4m3 code is exact in f16, so K and V enter the tensor cores exactly,
//     and their block scales are applied to scores and weights in f32;
//   - scores are computed transposed, K (16 tokens) times Q^T (8 queries): the
//     m16n8k16 MMA has no row to spare.  A 16-bit query is one half once its
//     row is scaled to the top of the f16 range (bf16 elements 2^-31 below the
//     row's largest lose bits), an f32 query the sum of two halves and so two
//     MMAs: off by at most 2^-23 of itself or 2^-38 of its row's largest,
//     where float32 has 2^-24 (a third MMA would be half as much work again);
//   - a weight times its block's V scale is the sum of two halves, off by at
//     most 2^-23 of itself, and the value sum is transposed too: V^T (16 dims)
//     times P^T (8 queries).  With up to 4 queries columns 4..7 repeat queries
//     0..3, and one MMA takes the high halves in columns 0..3 and the low
//     halves in 4..7 (their sums meet once a piece); with more, each half has
//     its MMA.  An 8x8 transpose of f16 pairs (movmatrix) turns the score
//     fragment into that operand;
//   - what must not exceed f16 is weight times scale, so the running reference
//     is that of the products: with H the largest exponent of a V scale in the
//     piece so far and e_t a token's, m is the largest z_t + e_t - H, weights
//     are 2^(z_t - m), and the operand is a weight times v_scale 2^(15 - H).
//     A row's largest product is above 2^14 there, whatever blocks of larger
//     scale but no weight lie beside it, and a token is off by at most 2^-25,
//     2^-39 of that largest product;
//   - e_t - H counts as -100 below that, so that weights stay within float32
//     (2^100 at most).  When H rises by d, m falls by d (by less where a block
//     is already 100 below H): the producer, which sees the scales in order,
//     adds these up.  So blocks of one sequence lose nothing to one another
//     while their scales are within 2^100; a scale further below the largest
//     one keeps as many bits less;
//   - m is rounded up to a whole number: all factors between references are
//     then exact powers of two;
//   - the value sum of a pass (64 tokens; 32 for head_dim 256) starts from zero
//     in the tensor cores and is added to f32 registers, so the chain of
//     truncated tensor-core additions is four long (eight where each half has
//     its MMA), not as long as the sequence.
//
// Shared memory.  A tile is contiguous in HBM; it is copied as rows of 128
// bytes (64 for head_dim 64) with the hardware swizzle: the 16-byte chunk at
// byte offset x lands at x ^ (((x >> 7) & 7) << 4) (& 3 for 64-byte rows), so
// the 16-byte reads below touch every bank once (the V reads of head_dim 64
// and 256 twice).
#include <algorithm>
#include <cstdlib>
#include <mutex>
#include <type_traits>
#include <unordered_map>

#include "combine.cuh"
#include "common.cuh"
#include "decode_common.cuh"
#include "fp8_common.cuh"
#include "mma_common.cuh"

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
  int* gave_up;        // [num_ctas + 1]: CTAs that gave up on a wait, then whether any did (accumulate only, else null)
  int real_block;      // tokens per cache block; DecodeArgs::block_size is the slice
  int slice_shift;     // log2 of the slice
  int real_shift;      // log2 of real_block
  int window;
  int append_here;     // 1: the producers append the new tokens (see fp8_append_kernel)
  int direct;          // 1: CTA c takes segment c whole, nothing is split
  float scale, softcap;
};

constexpr int kSclRing = 128;  // slices whose scales the ring holds (see fp8_produce)

// What the consumers need of a slice's scales (see the top).
struct __align__(16) SliceScales {
  float k;       // K scale
  float v;       // V scale * 2^(15 - H)
  float rel;     // the V scale's exponent less H, -kSpan at least
  int units;     // H, and above it the sum of what it lowers m by
};
constexpr int kSpan = 100;

// Stage tokens: 16 KB of K and V.
constexpr int stage_tokens(int head_dim) { return 8192 / head_dim; }

// First slice of sequence b that the call reads.
__device__ __forceinline__ int first_slice(const Fp8Args& a, int L) {
  return a.window > 0 ? max(0, L - a.window) >> a.slice_shift : 0;
}
__device__ __forceinline__ int num_slices(const Fp8Args& a, int L) {
  return ((L + a.block_size - 1) >> a.slice_shift) - first_slice(a, L);
}

__device__ __noinline__ unsigned long long udiv64(unsigned long long a, unsigned b) { return a / b; }

// partition_prologue (decode_common.cuh) for segments that start at a window.
template <int D>
__device__ void fp8_prologue(const Fp8Args& a, WalkStart* out) {
  const int tid = threadIdx.x, lane = tid & 31, nt = blockDim.x, H = a.num_kv_heads;
  if (tid == 0 && a.gave_up != nullptr) a.gave_up[blockIdx.x] = 0;
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
  __shared__ long long s_rest;
  __shared__ int s_found;
  const int row_floats = H * a.group * D;
  if (tid == 0) {
    s_rest = 0;
    s_found = 0;
  }
  // stream positions of each of sequence b's segments; empty sequences get their zero rows on the way
  auto length = [&](int b, bool first_look) {
    if (b >= a.batch) return 0;
    const int L = clamp_ctx(a.context_lens, b, a.max_ctx, a.append);
    if (first_look) {
      if (blockIdx.x == 0 && __ldg(a.context_lens + b) != L - a.append) atomicOr(a.err, CLOVE_FLAG_CTX_RANGE);
      if (L == 0 && b % a.num_ctas == (int)blockIdx.x) {
        float4* row = reinterpret_cast<float4*>(a.out + (size_t)b * row_floats);
        for (int i = 0; i < row_floats / 4; ++i) row[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    return L > 0 ? num_slices(a, L) + a.seg_cost : 0;
  };
  // the first nt sequences by a scan (usually all of them), the sum of the others
  int len = length(tid, true), tot;
  int excl = block_excl_scan(len, warp_tot, &tot);
  if (a.batch > nt) {
    long long mine = 0;
#pragma unroll 1
    for (int b = tid + nt; b < a.batch; b += nt) mine += length(b, true);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0 && mine) atomicAdd(reinterpret_cast<unsigned long long*>(&s_rest), (unsigned long long)mine);
    __syncthreads();
  }
  // floor(c W / P) = c (W / P) + floor(c (W mod P) / P), the last in 32 bits
  const unsigned long long W = (unsigned long long)(s_rest + tot) * H, quot = udiv64(W, a.num_ctas);
  const unsigned rest = (unsigned)(W - quot * a.num_ctas), c = blockIdx.x;
  const long long lo = (long long)(c * quot + c * rest / a.num_ctas);
  const long long hi = (long long)((c + 1) * quot + (c + 1) * rest / a.num_ctas);
  if (tid == 0) {
    out->lo = lo;
    out->hi = hi;
    out->b = -1;
    out->h = 0;
    out->off = 0;
    if (blockIdx.x == 0) *a.total = (long long)W;
  }
  __syncthreads();
  if (lo < hi) {
    long long carry = 0;
#pragma unroll 1
    for (int base = 0;; ) {
      const long long s0 = (carry + excl) * H;
      if (len > 0 && s0 <= lo && lo < s0 + (long long)len * H) {
        const unsigned long long r = lo - s0, hh = udiv64(r, len);
        out->b = base + tid;
        out->h = (int)hh;
        out->off = (int)(r - hh * len);
        s_found = 1;
      }
      carry += tot;
      base += nt;
      __syncthreads();
      if (s_found || base >= a.batch) break;
      len = length(base + tid, false);
      excl = block_excl_scan(len, warp_tot, &tot);
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

// The new token of one (sequence, KV head), held by a warp: lanes 0..15 have
// its K row, lanes 16..31 its V row, D / 16 elements each.
template <int D>
struct NewRow {
  int phys;   // its block, -1: none
  float old;  // the plane's scale before it, after fp8_store_new the scale now
  float v[D / 16];
};

template <typename T, int D>
__device__ __forceinline__ void fp8_load_new(const Fp8Args& a, int b, int h, int L, int phys, int lane, NewRow<D>& n) {
  const int off = (L - 1) & (a.real_block - 1), H = a.num_kv_heads, p = lane >> 4;
  n.phys = phys;
  if (phys < 0 || phys >= a.num_blocks) {
    if (lane == 0) atomicOr(a.err, CLOVE_FLAG_BLOCK_OOB);
    n.phys = -1;
    return;
  }
  n.old = off == 0 ? 0.f : __ldcg(a.scales + ((size_t)p * a.num_blocks + phys) * H + h);
  const T* src = static_cast<const T*>(p ? a.v_new : a.k_new) + ((size_t)b * H + h) * D + (lane & 15) * (D / 16);
#pragma unroll
  for (int i = 0; i < D / 16; i += 4) load_vec_f32<T, 4>(src + i, reinterpret_cast<float(&)[4]>(n.v[i]));
}

// 1 / s: exact for the powers of two that scales are.
__device__ __forceinline__ float fp8_inverse(float s) { return __frcp_rn(s); }

// Rounds a tile's codes, but for row `but`, to a scale 1 / ratio times as
// large.  Sixteen lanes; out of line, for it is rare.
__device__ __noinline__ void fp8_rescale_tile(unsigned char* rows, int chunks, int chunks_per_row, int but, float ratio,
                                              int lane) {
  uint4* w = reinterpret_cast<uint4*>(rows);
#pragma unroll 1
  for (int i = lane; i < chunks; i += 16) {
    if (i / chunks_per_row == but) continue;
    const uint4 c = __ldcg(w + i);
    const uint2 lo = fp8_rescale8(make_uint2(c.x, c.y), ratio), hi = fp8_rescale8(make_uint2(c.z, c.w), ratio);
    w[i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
}

// Settles the block's scale with the row, rounds the rows already there if it
// grew, writes the row.  Nobody else reads or writes this tile before the
// copies that the caller issues next.  The new scales come back in n.old.
template <int D>
__device__ __forceinline__ void fp8_store_new(const Fp8Args& a, int h, int L, int lane, NewRow<D>& n) {
  if (n.phys < 0) return;
  const int bs = a.real_block, H = a.num_kv_heads, off = (L - 1) & (bs - 1), p = lane >> 4;
  const size_t tile = (size_t)n.phys * H + h;
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) amax = fmaxf(amax, finite_abs(n.v[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float s = fmaxf(n.old, fp8_scale_for(amax)), inv = fp8_inverse(s);
  unsigned char* rows = static_cast<unsigned char*>(p ? a.v_cache : a.k_cache) + tile * bs * D;
  if (n.old > 0.f && s > n.old)  // the row itself is written below
    fp8_rescale_tile(rows, bs * (D / 16), D / 16, off, n.old / s, lane & 15);
  uint32_t* dst = reinterpret_cast<uint32_t*>(rows + (size_t)off * D + (lane & 15) * (D / 16));
#pragma unroll
  for (int i = 0; i < D / 16; i += 4)
    dst[i / 4] = fp8_pack2(n.v[i] * inv, n.v[i + 1] * inv) | fp8_pack2(n.v[i + 2] * inv, n.v[i + 3] * inv) << 16;
  if ((lane & 15) == 0) a.scales[(size_t)p * a.num_blocks * H + tile] = s;
  n.old = s;
  if (lane == 0 && a.mass != nullptr) a.mass[tile * bs + off] = 0.f;
  fence_proxy_async_global();
  __syncwarp();
}

__device__ __forceinline__ int new_entry(const Fp8Args& a, int b, int L) {
  return __ldg(a.block_tables + (size_t)b * a.bt_stride + ((L - 1) >> a.real_shift));
}

// The new tokens of all sequences, a warp per (KV head, sequence), ahead of
// the decode.  Used where a block is more than one slice: another CTA may then
// stream the earlier slices of the block that an append rescales.
template <typename T, int D>
__global__ void __launch_bounds__(32) fp8_append_kernel(const Fp8Args a) {
  griddep_wait();
  const int b = blockIdx.y, h = blockIdx.x, lane = threadIdx.x, L = clamp_ctx(a.context_lens, b, a.max_ctx, 1);
  NewRow<D> n;
  fp8_load_new<T, D>(a, b, h, L, new_entry(a, b, L), lane, n);
  fp8_store_new<D>(a, h, L, lane, n);
}

// Shared-memory reads by address (the compiler would take a generic pointer's
// longer way).
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}

// Barrier operations by shared-memory address: the producer's
// per-stage loop has to stay small.
__device__ __forceinline__ bool try_wait_at(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void expect_tx_at(uint32_t bar, uint32_t bytes) {
  asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tma_slice(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %2}], [%4], %5;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(bar), "l"(policy)
      : "memory");
}
// The bounded wait for a ring slot, out of line.  False: it ran out, or the
// CTA has given up.
__device__ __noinline__ bool slot_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, int* err, uint32_t limit) {
  for (uint32_t i = 0; i < limit && *gave_up == 0; ++i)
    if (try_wait_at(bar, parity)) return true;
  if (*gave_up == 0) {
    atomicOr(err, CLOVE_FLAG_TIMEOUT);
    *gave_up = 1;
  }
  return false;
}

// e with x < (2 - 2^-10) 2^e, so that 2^15 x 2^-e stays within f16; -126 <= e <= 127.
__device__ __forceinline__ int scale_exponent(float x) {
  return min(max((__float_as_int(x) + 0x2000) >> 23, 1), 254) - 127;
}

// The producer warp (produce() of decode_common.cuh for this cache): walks
// the CTA's range, posts each piece, appends the new token where the piece
// ends its sequence, and streams the slices.
//
// It must issue a stage every ~1300 clocks beside the consumers, so what runs
// once a stage is short (a loop that leaves the instruction cache costs over
// 1000 clocks here): the warp prepares 32 slices at a time (table entries,
// copy rows, scales; loaded a group ahead), leaves the scales in the ring
// `scl` and issues the copies.
// The scales of slice i of stage gs are at scl[(gs * sb + i) % kSclRing]: a
// group is written when at most nstage stages are unconsumed, so nstage * sb +
// 32 <= kSclRing entries are live.
template <typename T, int D>
__device__ void fp8_produce(const Fp8Args& a, const CUtensorMap* map, const SmemPtrs& sm, const SmemPlan& sp, SliceScales* scl,
                            int sb, const WalkStart& ws) {
  constexpr int RPT = D >= 128 ? D / 128 : 1;  // rows of the copies' tensor map per token
  const int lane = threadIdx.x & 31, sub_shift = a.real_shift - a.slice_shift;
  const int vs = a.block_size, H = a.num_kv_heads, Hq = H * a.group;
  const uint32_t slice_bytes = (uint32_t)(2 * vs * D);
  const uint32_t q_bytes = (uint32_t)(a.group * D * (int)sizeof(T));
  const uint64_t pol = policy_evict_first();
  const uint32_t full = smem_u32(sm.full), empty = smem_u32(sm.empty), ring = smem_u32(sm.ring);
  const uint32_t stage_bytes = (uint32_t)sp.stage_bytes;
  int slot = 0, uk = 0, stage = 0;  // ring slot of the next stage, unit slot, stages issued
  uint32_t phase = 0, uphase = 0;
  bool aborted = false;

  // Lane i: the table entry of slice j0 + i of the piece (unchecked) ...
  auto entry = [&](const Unit& x, int j0) {
    const int j = j0 + lane;
    return j < x.nblk ? __ldg(a.block_tables + (size_t)x.b * a.bt_stride + ((x.blk0 + j) >> sub_shift)) : 0;
  };
  // ... and what it leads to: the copy's first row, the scales (zero behind
  // the piece).  Entries outside the pool are flagged and replaced by block 0
  // (never followed).
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
      s.row = ((int)tile * a.real_block + ((x.blk0 + j) & ((1 << sub_shift) - 1)) * vs) * RPT;
      s.sk = __ldcg(a.scales + tile);
      s.sv = __ldcg(a.scales + (size_t)a.num_blocks * H + tile);
    }
    return s;
  };

  const int alpha = a.seg_cost, sb_shift = 31 - __clz(sb);
  int vmax = 0, vmin = 0, lowered = 0;  // the piece's V exponents so far

  int b = ws.b, h = ws.h, off = ws.off, npiece = 0;
  int left = (int)(ws.hi - ws.lo);  // stream positions of the range still to walk
  int L = b >= 0 ? clamp_ctx(a.context_lens, b, a.max_ctx, a.append) : 0;
  int nb = L > 0 ? num_slices(a, L) : 0;
  // What a piece needs from memory before its first copy, loaded while the
  // piece before it still streams: the first slices and the new token.
  Slice cur = {0, 0.f, 0.f};
  NewRow<D> nr;
  int e0 = 0, ne = 0;
  // The next piece of the walk, with its first table entries under way.
  auto claim = [&](Unit& x) -> bool {
    while (b >= 0 && left > 0) {
      const int len = nb + alpha, span = min(len - off, left);
      const int r0 = max(off, alpha), r1 = off + span;
      const bool piece = r1 > r0;
      if (piece) {
        x.u = 0;
        x.b = b;
        x.h = h;
        x.L = L;
        x.blk0 = first_slice(a, L) + r0 - alpha;
        x.nblk = r1 - r0;
        x.nstages = (x.nblk + sb - 1) >> sb_shift;
        x.complete = r0 == alpha && r1 == len;
        x.slot = npiece == 0 ? 0 : 1;
        x.last = r1 == len;
        e0 = entry(x, 0);
        if (a.append_here && x.last) ne = new_entry(a, b, L);
        ++npiece;
      }
      left -= span;
      off += span;
      if (off == len && left > 0) {
        off = 0;
        if (++h == H) {
          h = 0;
          do {
            if (++b >= a.batch) {  // (cannot happen while positions are left; bounds the walk regardless)
              b = -1;
              break;
            }
            L = clamp_ctx(a.context_lens, b, a.max_ctx, a.append);
            nb = L > 0 ? num_slices(a, L) : 0;
          } while (L == 0);
        }
      }
      if (piece) return true;
    }
    return false;
  };
  auto preload = [&](const Unit& x) {
    cur = resolve(x, 0, e0);
    if (a.append_here && x.last) fp8_load_new<T, D>(a, x.b, x.h, x.L, ne, lane, nr);
  };

  // The walk starts behind an empty piece, so that there is one place in the
  // code that claims and preloads.
  Unit x;
  x.nblk = 0;
  x.last = 0;
  bool have = true, first = true;
  while (true) {
    int ok = 1;
    if (x.nblk > 0 || !have) {
      if (lane == 0) {
        if (!try_wait_at(smem_u32(&sm.uempty[uk]), uphase ^ 1) &&
            !slot_wait(smem_u32(&sm.uempty[uk]), uphase ^ 1, sm.misc, a.err, a.wait_limit)) {
          ok = 0;
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
    }

    if (a.append_here && x.last) {
      fp8_store_new<D>(a, x.h, x.L, lane, nr);
      // the scales loaded for the last block's slices are the old ones
      const float sk = __shfl_sync(0xffffffffu, nr.old, 0), sv = __shfl_sync(0xffffffffu, nr.old, 16);
      if (nr.phys >= 0 && lane < x.nblk && (x.blk0 + lane) >> sub_shift == (x.L - 1) >> a.real_shift) {
        cur.sk = sk;
        cur.sv = sv;
      }
    }
    int e1 = x.nblk > 32 ? entry(x, 32) : 0;
    Unit x2;
    bool have2 = false;
#pragma unroll 1
    for (int j0 = 0; j0 == 0 || j0 < x.nblk; j0 += 32) {
      const int n = min(32, x.nblk - j0);  // slices of this group
      const bool final = j0 + 32 >= x.nblk;
      const int issued = cur.row;
      {
        // behind the piece: its last slice once more
        const float sk = __shfl_sync(0xffffffffu, cur.sk, min(lane, n - 1));
        const float sv = __shfl_sync(0xffffffffu, cur.sv, min(lane, n - 1));
        const int e = scale_exponent(sv);
        const int hi = __reduce_max_sync(0xffffffffu, e), lo = __reduce_min_sync(0xffffffffu, e);
        if (j0 == 0) {
          vmax = hi;
          vmin = lo;
          lowered = 0;
        } else {
          const int was = min(vmax - vmin, kSpan);
          vmax = max(vmax, hi);
          lowered += min(vmax - vmin, kSpan) - was;
          vmin = min(vmin, lo);
        }
        SliceScales f;
        f.k = sk;
        // (2^(15 - H) in two factors: it may be above 2^127)
        f.v = sv * __int_as_float((127 + min(15 - vmax, 127)) << 23) * __int_as_float((127 + max(15 - vmax - 127, 0)) << 23);
        f.rel = (float)max(e - vmax, -kSpan);
        f.units = lowered * 256 + vmax + 128;
        scl[(stage * sb + lane) & (kSclRing - 1)] = f;
      }
      __syncwarp();
      if (final) {
        have2 = claim(x2);
      } else {
        cur = resolve(x, j0 + 32, e1);
        if (j0 + 64 < x.nblk) e1 = entry(x, j0 + 64);
      }
      // issue the group; before a piece's last stages come the next piece's loads
      const int nst = (n + sb - 1) >> sb_shift, cut = final ? (nst + 1) / 2 : nst;
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {
        const int s0 = part == 0 ? 0 : cut, s1 = part == 0 ? cut : nst;
        int s = s0;
        if (first && s < s1) {
          first = false;
          if (a.inject_stall) {  // test hook: the CTA's first stage is never filled
            ++s;
            ++slot;
          }
        }
#pragma unroll 1
        for (; s < s1; ++s) {
          if (slot == a.nstage) {
            slot = 0;
            phase ^= 1;
          }
          // the whole warp waits and counts, one lane issues: operands stay in uniform registers
          if (!__all_sync(0xffffffffu, try_wait_at(empty + slot * 8, phase ^ 1)) &&
              !__all_sync(0xffffffffu, slot_wait(empty + slot * 8, phase ^ 1, sm.misc, a.err, a.wait_limit))) {
            ok = 0;
            break;
          }
          const int m = min(sb, n - s * sb);
          const uint32_t bar = full + slot * 8;
          if (elect_one()) expect_tx_at(bar, slice_bytes * (uint32_t)m);
          uint32_t dst = ring + slot * stage_bytes;
#pragma unroll 1
          for (int i = 0; i < m; ++i) {  // one copy per slice: its K tile, then its V tile
            const int row = __shfl_sync(0xffffffffu, issued, s * sb + i);
            if (elect_one()) tma_slice(dst, map, bar, row, pol);
            dst += slice_bytes;
          }
          ++slot;
        }
        if (part == 0 && final && have2) preload(x2);
      }
      stage += nst;
      if (!ok) break;
    }
    if (!ok) {
      aborted = true;
      break;
    }
    have = have2;
    x = x2;
  }
  if (aborted && lane == 0) {
    if (a.gave_up != nullptr) a.gave_up[blockIdx.x] = 1;
    // drain: the last nstage stages and unit posts may still be in flight
    int s = slot;  // 1 .. nstage: the slot behind the last one issued
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

// D(16x8, f32) += A(16x16, f16) * B(16x8, f16)
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from a zero accumulator.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Four codes -> two f16 pairs (low bytes first), exact.
__device__ __forceinline__ void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

// Two f32 operations in one instruction, each rounded as alone.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// v = hi + lo, each a pair of halves.
__device__ __forceinline__ void split_halves(float2 v, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  const float2 r = fma2(__half22float2(h), both(-1.f), v);
  hi = half2_bits(h);
  lo = half2_bits(__floats2half2_rn(r.x, r.y));
}

// 16 bytes of elements, widened.
template <typename T>
__device__ __forceinline__ void unpack16(uint4 v, float* o) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      o[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      o[2 * i] = f.x;
      o[2 * i + 1] = f.y;
    } else {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
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

// The 8-byte V unit (8 dims of a 128-byte row) that lane row g reads as its
// p-th: as for K, any assignment of dims to MMA columns will do.
template <int D>
__device__ __forceinline__ int v_unit(int g, int p) {
  return D == 64 ? g : 2 * ((g & 1) + 2 * p + 4 * (g >> 2)) + ((g >> 1) & 1);
}

// 2^x; the hardware's, flushing results below 2^-126.  Exact for whole x (all
// of -126 .. 127 tried on the GPU).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh for |x| <= kTanhNear, where scores below a cap mostly are: x + x^3 P(x^2)
// with P of degree 3, fitted so that the largest relative error there is
// smallest (1.6e-8, a quarter of 2^-24; Taylor's coefficients give that up to 0.26).
constexpr float kTanhNear = 0.5f;
__device__ __forceinline__ float2 tanh_near(float2 x) {
  const float2 y = mul2(x, x);
  float2 p = fma2(y, both(0.01724149f), both(-0.05304549f));
  p = fma2(y, p, both(0.13325879f));
  p = fma2(y, p, both(-0.33333144f));
  return fma2(mul2(x, y), p, x);
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh for any x: up to 1.25 the continued fraction x / (1 + x^2 / (3 + x^2 /
// (5 + ..))) cut after the sixth level (off by less than 2^-27), beyond it 1 -
// 2 / (1 + e^2x).
__device__ __forceinline__ float tanh_any(float x) {
  const float y = x * x, e = ex2(fabsf(x) * (2.f * kLog2e));
  const float low = x * fmaf(y, fmaf(y, 21.f, 1260.f), 10395.f) * rcp(fmaf(y, fmaf(y, y + 210.f, 4725.f), 10395.f));
  return fabsf(x) > 1.25f ? copysignf(fmaf(-2.f, rcp(1.f + e), 1.f), x) : low;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}


// kShaped: scores may be capped or biased; kKept: they are written out for the
// weights; kTwin: groups of up to 4 queries.  A variant has none of the others'
// code, run or not: it would crowd the instruction cache (the capped window of
// 256 sequences took 121 us with the code that keeps scores beside it, 111 without).
template <typename T, int D, int NCW, bool kShaped, bool kKept, bool kTwin>
__global__ void __launch_bounds__((NCW + 1) * 32, 2)
    fp8_decode_kernel(const __grid_constant__ CUtensorMap map, const Fp8Args a) {
  static_assert(NCW == 3, "the hand-off sums three warps' states");
  constexpr bool kTwoHalves = sizeof(T) == 4;  // f32 queries need the low halves
  constexpr int KJ = D / 64;                   // 16-byte K chunks per lane and token
  constexpr int VH = D >= 128 ? D / 128 : 1;   // 128-byte rows per token
  constexpr int VP = D >= 128 ? 2 : 1;         // 8-byte V units per lane and row
  constexpr int S = state_stride(D);
  constexpr int PT = D == 256 ? 32 : 64;       // tokens per pass
  constexpr int NG = PT / 16, NE = PT / 8;     // MMA steps and 8-token tiles of a pass
  constexpr int TT = stage_tokens(D);          // tokens per stage
  const int vs = a.block_size, sb = a.stage_blocks, group = a.group;

  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const SmemPlan sp = smem_plan(vs, D, 1, sb, a.nstage, (NCW - 1) * group * S * (int)sizeof(float),
                                group * D * (int)sizeof(T), 1);
  const SmemPtrs sm = smem_ptrs(smem, sp, a.nstage);
  SliceScales* scl = reinterpret_cast<SliceScales*>(reinterpret_cast<unsigned char*>(sm.scratch) + sp.scratch_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) prefetch_tensor_map(&map);
  init_barriers<1, NCW - 1>(sm, a.nstage, NCW);
  __shared__ WalkStart walk;
  fp8_prologue<D>(a, &walk);

  if (warp == 0) {
    fp8_produce<T, D>(a, &map, sm, sp, scl, sb, walk);
    return;
  }

  const int cw = warp - 1, g = lane >> 2, tq = lane & 3;
  const int vshift = a.slice_shift;
  const int gq = kTwin ? g & 3 : g;  // kTwin: columns 4..7 repeat queries 0..3
  // Read offsets within a pass: K rows g (+ 8 e), V rows 2 tq + (i & 1) (+ 8 n);
  // the swizzle's row bits do not change with the multiples of 8 tokens.
  uint32_t koff[KJ], voff[2][VH * VP];
#pragma unroll
  for (int j = 0; j < KJ; ++j) koff[j] = swz<D>((uint32_t)(g * D + k_chunk<D>(tq, j) * 16));
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < VH * VP; ++k)
      voff[i][k] = swz<D>((uint32_t)((2 * tq + i) * D + (k / VP) * 128 + v_unit<D>(g, k % VP) * 8));
  // A stage is slice after slice, K tile then V tile: the K rows of token tok
  // (a multiple of 8) from the stage's start, its V rows one tile further.
  auto tile_at = [&](int tok) { return (uint32_t)((tok + (tok & -vs)) * D); };
  int gbase = 0, uk = 0, n_done = 0;
  uint32_t uphase = 0;
  UnitSlot us;

  while (wait_unit(a, sm, uk, uphase, us)) {
    const Unit x = us.x;
    // Query fragments: row g scaled by a power of two that puts its largest
    // element in [2^13, 2^14), undone in the score's factor.
    uint32_t qh[KJ * 4][2], ql[kTwoHalves ? KJ * 4 : 1][2];
    float2 zf, slope;  // of queries 2 tq and 2 tq + 1: score = dot * K scale * zf, bias per token
    // stage gs belongs to warp gs % NCW (nstage is a multiple of NCW)
    const int j_first = ((cw - gbase) % NCW + NCW) % NCW;
    const bool mine = j_first < x.nstages;
    if (mine) {
      const uint32_t qaddr = smem_u32(sm.qbuf + uk * sp.q_stride) + gq * D * (int)sizeof(T);
      float q[KJ * 16];
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int i = 0; i < 16; i += 16 / (int)sizeof(T)) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (gq < group) w = lds128(qaddr + (k_chunk<D>(tq, j) * 16 + i) * (int)sizeof(T));
          unpack16<T>(w, q + j * 16 + i);
        }
#pragma unroll
      for (int i = 0; i < KJ * 16; ++i) amax = fmaxf(amax, fabsf(q[i]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = min(max(__float_as_int(amax) >> 23, 1), 254) - 127 - 13;  // divide by 2^e
      const float up = __int_as_float((127 - max(e, -127)) << 23);
      float f = a.scale * __int_as_float((127 + max(e, -126)) << 23);
      if (e < -126) f *= 0.5f;
      f = kShaped && a.softcap > 0.f ? f / a.softcap : f * kLog2e;
      const float s = kShaped && a.slopes != nullptr && gq < group ? __ldg(a.slopes + x.h * group + gq) * kLog2e : 0.f;
      zf = make_float2(__shfl_sync(0xffffffffu, f, 8 * tq), __shfl_sync(0xffffffffu, f, 8 * tq + 4));
      slope = make_float2(__shfl_sync(0xffffffffu, s, 8 * tq), __shfl_sync(0xffffffffu, s, 8 * tq + 4));
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float* f4 = q + j * 16 + w * 4;
          uint32_t lo[2];
          split_halves(make_float2(f4[0] * up, f4[1] * up), qh[j * 4 + w][0], lo[0]);
          split_halves(make_float2(f4[2] * up, f4[3] * up), qh[j * 4 + w][1], lo[1]);
          if constexpr (kTwoHalves) {
            ql[j * 4 + w][0] = lo[0];
            ql[j * 4 + w][1] = lo[1];
          }
        }
    }
    const float cap = a.softcap * kLog2e;
    const int t_first = a.window > 0 ? max(0, x.L - a.window) : 0;  // first token attended to
    float* zrow =
        kKept ? a.z + ((size_t)(x.b * a.num_kv_heads + x.h) * group + 2 * tq) * a.z_stride : nullptr;

    float m[2] = {-INFINITY, -INFINITY};
    int units = 128;  // of the passes so far (SliceScales)
    float2 l2 = make_float2(0.f, 0.f);
    // value sums: o[4 i + k] is dim k (of 4) of half i of this lane's V units, queries 2 tq and 2 tq + 1
    float2 o[D / 8];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n] = make_float2(0.f, 0.f);

    bool aborted = false;
    for (int j = j_first; j < x.nstages; j += NCW) {
      const int gs = gbase + j, slot = gs % a.nstage;
      if (!wait_or_abort(a, sm, &sm.full[slot], (uint32_t)(gs / a.nstage) & 1u)) {
        aborted = true;
        break;
      }
      const uint32_t kbase = smem_u32(sm.ring + (size_t)slot * sp.stage_bytes);
      const uint32_t vbase = kbase + sp.tile_stride, sbase = smem_u32(scl);
      const int s_first = gs * sb;                // scale ring index of the stage's first slice
      const int t_base = (x.blk0 + j * sb) * vs;  // token of the stage's first row
      const int hi = min(TT, min((x.blk0 + x.nblk) * vs, x.L) - t_base), lo = max(0, t_first - t_base);
      const bool ragged = lo > 0 || hi < TT;
      if (ragged) {
        // Rows outside [lo, hi) may hold NaN codes; their weights are 0, but
        // 0 * NaN is NaN, so clear those V rows.
        unsigned char* vst = sm.ring + (size_t)slot * sp.stage_bytes + sp.tile_stride;
        for (int i = lane; i < TT * (D / 16); i += 32) {
          const int tok = i / (D / 16);
          if (tok < lo || tok >= hi) *reinterpret_cast<uint4*>(vst + (tok & -vs) * D + swz<D>(i * 16)) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
#pragma unroll 1
      for (int p0 = 0; p0 < (TT == PT ? 1 : hi); p0 += PT) {
        // ---- scores: tile e is tokens p0 + 8 e + g, queries 2 tq + c ----
        float2 z[NE];
        int now = 0;
        float wv[NE], rel[NE];
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          uint4 kw[2][KJ];
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < KJ; ++c) kw[r][c] = lds128(kbase + koff[c] + tile_at(p0 + 16 * k + 8 * r));
          float s[4];
#pragma unroll
          for (int c = 0; c < KJ; ++c) {
            const uint32_t w0[4] = {kw[0][c].x, kw[0][c].y, kw[0][c].z, kw[0][c].w};
            const uint32_t w1[4] = {kw[1][c].x, kw[1][c].y, kw[1][c].z, kw[1][c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a0, a1, a2, a3;
              codes4(w0[i], a0, a2);
              codes4(w1[i], a1, a3);
              if (c == 0 && i == 0)
                mma_f16_first(s, a0, a1, a2, a3, qh[0][0], qh[0][1]);
              else
                mma_f16(s, a0, a1, a2, a3, qh[c * 4 + i][0], qh[c * 4 + i][1]);
              if constexpr (kTwoHalves) mma_f16(s, a0, a1, a2, a3, ql[c * 4 + i][0], ql[c * 4 + i][1]);
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int e = 2 * k + r;
            const uint4 f = lds128(sbase + ((s_first + ((p0 + 8 * e) >> vshift)) & (kSclRing - 1)) * 16);
            wv[e] = __uint_as_float(f.y);
            rel[e] = __uint_as_float(f.z);
            if (e == 0) now = (int)f.w;
            z[e] = mul2(make_float2(s[2 * r], s[2 * r + 1]), mul2(both(__uint_as_float(f.x)), zf));
          }
        }
        if constexpr (kShaped) {
          if (cap > 0.f) {
            float most = 0.f;
#pragma unroll
            for (int e = 0; e < NE; ++e) most = fmaxf(most, fmaxf(fabsf(z[e].x), fabsf(z[e].y)));
            if (__builtin_expect(__any_sync(0xffffffffu, most > kTanhNear), 0)) {
              // a loop of one body, the registers moving through it: unrolled it would crowd the instruction cache
#pragma unroll 1
              for (int i = 0; i < NE; ++i) {
                const float2 w = make_float2(tanh_any(z[0].x) * cap, tanh_any(z[0].y) * cap);
#pragma unroll
                for (int e = 0; e < NE - 1; ++e) z[e] = z[e + 1];
                z[NE - 1] = w;
              }
            } else {
#pragma unroll
              for (int e = 0; e < NE; ++e) z[e] = mul2(tanh_near(z[e]), both(cap));
            }
          }
          if (a.slopes != nullptr) {
            const float back = (float)(t_base + p0 + g - (x.L - 1));  // exact below 2^24
#pragma unroll
            for (int e = 0; e < NE; ++e) z[e] = fma2(slope, both(back + (float)(8 * e)), z[e]);
          }
        }
        if constexpr (kKept) {
          const int left = hi - p0 - g;  // tokens of this lane's column
          float* zt = zrow + t_base + p0 + g;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (2 * tq + c < group) {
#pragma unroll
              for (int e = 0; e < NE; ++e)
                if (8 * e < left) zt[8 * e] = c ? z[e].y : z[e].x;
            }
            zt += a.z_stride;
          }
        }
        if (ragged) {
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            const int tok = p0 + 8 * e + g;
            if (tok < lo || tok >= hi) z[e] = both(-INFINITY);
          }
        }
        // ---- online softmax of queries 2 tq and 2 tq + 1 ----
        const float lowered = (float)((now >> 8) - (units >> 8)), down = ex2((float)((units & 255) - (now & 255)));
        units = now;
        float corr[2], oc[2];
        float2 top = add2(z[0], both(rel[0]));
#pragma unroll
        for (int e = 1; e < NE; ++e) {
          const float2 t = add2(z[e], both(rel[e]));
          top = make_float2(fmaxf(top.x, t.x), fmaxf(top.y, t.y));
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = c ? top.y : top.x;
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
          const float mn = fmaxf(m[c] - lowered, ceilf(mx));
          const float up = fmaxf(m[c] - mn, -1024.f);  // (also where both are -infinity)
          corr[c] = ex2(up);
          oc[c] = corr[c] * down;
          m[c] = mn;
        }
        const float2 ms = make_float2(m[0] == -INFINITY ? 0.f : -m[0], m[1] == -INFINITY ? 0.f : -m[1]);
        l2 = mul2(l2, make_float2(corr[0], corr[1]));
        // the P^T operand (tokens x queries): both halves of the weights, or, where columns 4..7 repeat the queries,
        // the high halves in columns 0..3 and the low ones in 4..7
        uint32_t ph[NE], pl[kTwin ? 1 : NE];
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const float2 d = add2(z[e], ms), w = make_float2(ex2(d.x), ex2(d.y));
          l2 = add2(l2, w);
          uint32_t hi2, lo2;
          split_halves(mul2(w, both(wv[e])), hi2, lo2);
          ph[e] = transpose8x8(kTwin && tq >= 2 ? lo2 : hi2);
          if constexpr (!kTwin) pl[e] = transpose8x8(lo2);
        }
        const float2 oc2 = make_float2(oc[0], oc[1]);
        // ---- value sum, V^T (16 dims) times P^T (8 queries) ----
#pragma unroll
        for (int u = 0; u < VH * VP; ++u) {
          uint2 vw[NG][4];  // tokens 16 k + 2 tq + {0, 1, 8, 9}, 8 dims each
#pragma unroll
          for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              vw[k][i] = lds64(vbase + voff[i & 1][u] + tile_at(p0 + 16 * k + 8 * (i >> 1)));
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            float d[2][4];  // MMA i: rows g and g + 8 are this lane's dims 2 i and 2 i + 1 of the four
#pragma unroll
            for (int k = 0; k < NG; ++k) {
              const uint32_t t0 = w ? vw[k][0].y : vw[k][0].x, t1 = w ? vw[k][1].y : vw[k][1].x;
              const uint32_t t2 = w ? vw[k][2].y : vw[k][2].x, t3 = w ? vw[k][3].y : vw[k][3].x;
              uint32_t v0[4], v1[4];  // token pairs of dims 0..3
              codes4(__byte_perm(t0, t1, 0x5140), v0[0], v0[1]);
              codes4(__byte_perm(t0, t1, 0x7362), v0[2], v0[3]);
              codes4(__byte_perm(t2, t3, 0x5140), v1[0], v1[1]);
              codes4(__byte_perm(t2, t3, 0x7362), v1[2], v1[3]);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                if (k == 0)
                  mma_f16_first(d[i], v0[2 * i], v0[2 * i + 1], v1[2 * i], v1[2 * i + 1], ph[0], ph[1]);
                else
                  mma_f16(d[i], v0[2 * i], v0[2 * i + 1], v1[2 * i], v1[2 * i + 1], ph[2 * k], ph[2 * k + 1]);
              }
              if constexpr (!kTwin) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                  mma_f16(d[i], v0[2 * i], v0[2 * i + 1], v1[2 * i], v1[2 * i + 1], pl[2 * k], pl[2 * k + 1]);
              }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                float2& on = o[(u * 2 + w) * 4 + 2 * i + r];
                on = fma2(on, oc2, make_float2(d[i][2 * r], d[i][2 * r + 1]));
              }
          }
        }
      }
      if (ragged) fence_proxy_async_smem();  // order the cleared rows before the slot's next copy
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[slot]);
    }
    if (aborted) break;  // the abort flag is up; every other warp leaves at its next wait
    gbase += x.nstages;

    // ---- hand-off: the last warp to finish a piece merges the others' states
    // (acc, M, l), left in scratch, with its own, still in registers: acc and l
    // sums of 2^(z - M) v and 2^(z - M), M whole and such that 1 <= l < 2 (or 0).
    // Lane (g, tq) holds queries 2 tq and 2 tq + 1 of its V units' dims. ----
    float l[2] = {l2.x, l2.y};
    float2 unit;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) l[c] += __shfl_xor_sync(0xffffffffu, l[c], s);
      // (o is in units of 2^(H - 15); less is taken off l where that, less k, would leave float32)
      const int h = (units & 255) - 128, k = max(min((__float_as_int(l[c]) >> 23) - 127, h + 111), -15);
      l[c] *= __int_as_float((127 - k) << 23);
      m[c] += (float)k;
      (c ? unit.y : unit.x) = __int_as_float((127 + h - 15 - k) << 23);
    }
    if constexpr (kTwin) {  // high and low halves' sums
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        o[n] = add2(o[n], make_float2(__shfl_xor_sync(0xffffffffu, o[n].x, 2), __shfl_xor_sync(0xffffffffu, o[n].y, 2)));
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n] = mul2(o[n], unit);
    auto sum = [&](int n, int c) { return c ? o[n].y : o[n].x; };
    const uint32_t par = (uint32_t)n_done & 1u;
    if (!wait_or_abort(a, sm, &sm.scr_empty[0], par ^ 1u)) break;
    int order = 0;
    if (lane == 0) {
      order = atomicAdd(&sm.arrive[0], 1);
      mbar_arrive(&sm.uempty[uk]);  // this warp no longer reads the unit's slot
    }
    order = __shfl_sync(0xffffffffu, order, 0);
    if (order < NCW - 1) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (2 * tq + c >= group) continue;
        float* row = sm.scratch + ((size_t)order * group + 2 * tq + c) * S;
        if (mine) {
#pragma unroll
          for (int i = 0; i < VH * VP * 2; ++i)
            *reinterpret_cast<float4*>(row + (i / (2 * VP)) * 128 + v_unit<D>(g, (i >> 1) % VP) * 8 + (i & 1) * 4) =
                make_float4(sum(4 * i, c), sum(4 * i + 1, c), sum(4 * i + 2, c), sum(4 * i + 3, c));
        }
        if (g == 0) {
          row[D] = m[c];
          row[D + 1] = l[c];
          row[D + 2] = (float)cw;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.scr_empty[1]);  // [1]: the others' states are in scratch
    } else {
      if (!wait_or_abort(a, sm, &sm.scr_empty[1], par)) break;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int q = 2 * tq + c;
        if (q >= group) continue;
        // Which warp comes last differs from run to run, the sums must not:
        // they are (warp 0 + warp 1) + warp 2, A and B being the others' states
        // in the order of their warps.
        const float* A = sm.scratch + (size_t)q * S;
        const float* B = A + (size_t)group * S;
        if (A[D + 2] > B[D + 2]) {
          const float* swap = A;
          A = B;
          B = swap;
        }
        const bool own_last = cw == NCW - 1;
        // fo xo + fa xa + fb xb, each product rounded (a contracted one would tell who came last)
        auto add = [&](float wo, float xo, float wa, float xa, float wb, float xb) {
          const float po = __fmul_rn(wo, xo), pb = __fmul_rn(wb, xb);
          return __fadd_rn(__fadd_rn(own_last ? pb : po, __fmul_rn(wa, xa)), own_last ? po : pb);
        };
        const float mo = m[c], M = fmaxf(mo, fmaxf(A[D], B[D]));
        const float fo = mo == -INFINITY ? 0.f : ex2(mo - M);
        const float fa = A[D] == -INFINITY ? 0.f : ex2(A[D] - M), fb = B[D] == -INFINITY ? 0.f : ex2(B[D] - M);
        const float L = add(fo, l[c], fa, A[D + 1], fb, B[D + 1]);
        const float inv = 1.f / L, norm = x.complete ? inv : 1.f;
        const int Hq = a.num_kv_heads * group, hq = x.h * group + q;
        float* dst = x.complete ? a.out + ((size_t)x.b * Hq + hq) * D
                                : a.partials + (((size_t)blockIdx.x * 2 + x.slot) * group + q) * S;
#pragma unroll
        for (int i = 0; i < VH * VP * 2; ++i) {
          const int d = (i / (2 * VP)) * 128 + v_unit<D>(g, (i >> 1) % VP) * 8 + (i & 1) * 4;
          // (a warp without a stage of the piece leaves no acc)
          float4 va = make_float4(0.f, 0.f, 0.f, 0.f), vb = va;
          if (fa > 0.f) va = *reinterpret_cast<const float4*>(A + d);
          if (fb > 0.f) vb = *reinterpret_cast<const float4*>(B + d);
          *reinterpret_cast<float4*>(dst + d) = make_float4(add(fo, sum(4 * i, c), fa, va.x, fb, vb.x) * norm,
                                                            add(fo, sum(4 * i + 1, c), fa, va.y, fb, vb.y) * norm,
                                                            add(fo, sum(4 * i + 2, c), fa, va.z, fb, vb.z) * norm,
                                                            add(fo, sum(4 * i + 3, c), fa, va.w, fb, vb.w) * norm);
        }
        if (g == 0) {
          if (!x.complete) {
            dst[D] = M;
            dst[D + 1] = L;
          } else if (kKept) {
            a.row_state[(size_t)x.b * Hq + hq] = make_float2(M, inv);
          }
        }
      }
      __syncwarp();
      if (lane == 0) {
        sm.arrive[0] = 0;
        mbar_arrive(&sm.scr_empty[0]);
      }
    }
    ++n_done;
    if (++uk == kUnitRing) {
      uk = 0;
      uphase ^= 1;
    }
  }
  if (kKept && sm.misc[0] && lane == 0) a.gave_up[blockIdx.x] = 1;
}

// ---------------------------------------------------------------------------
// weights: mass += sum over the group of 2^(z - M) / L
// ---------------------------------------------------------------------------
constexpr int kMassThreads = 256, kMassCtas = 6;  // CTAs per SM, all resident
constexpr int kMassTokens = 128;                  // tokens per warp and step: four per lane

// The steps of all (sequence, KV head) pairs are one stream, sequence by
// sequence, and every warp takes an equal run of it: with lengths that differ
// the longest sequence would otherwise hold its warps several times as long as
// the others theirs (128 ragged sequences: 4 us more).  Bound by latency: the
// scores come from L2 where they fit it, and a warp has one or two steps; CTAs
// in a second wave cost 3 us there.
__global__ void __launch_bounds__(kMassThreads, kMassCtas) fp8_mass_kernel(const Fp8Args a) {
  constexpr int kWarps = kMassThreads / 32;
  __shared__ int warp_tot[kWarps], start[kMassThreads], count[kMassThreads];
  __shared__ long long s_rest;
  const int H = a.num_kv_heads, G = a.group, bs = a.real_block, tid = threadIdx.x, lane = tid & 31;
  // steps of one KV head of sequence b: from the first attended token's to the last's
  auto first_step = [&](int L) { return a.window > 0 ? max(0, L - a.window) / kMassTokens : 0; };
  auto steps = [&](int b) {
    if (b >= a.batch) return 0;
    const int L = clamp_ctx(a.context_lens, b, a.max_ctx, a.append);
    return (L + kMassTokens - 1) / kMassTokens - first_step(L);
  };
  int n = steps(tid), tot;
  int before = block_excl_scan(n, warp_tot, &tot);
  long long all = tot;
  if (a.batch > kMassThreads) {
    if (tid == 0) s_rest = 0;
    __syncthreads();
    long long mine = 0;
#pragma unroll 1
    for (int b = tid + kMassThreads; b < a.batch; b += kMassThreads) mine += steps(b);
    if (mine) atomicAdd(reinterpret_cast<unsigned long long*>(&s_rest), (unsigned long long)mine);
    __syncthreads();
    all += s_rest;
  }
  all *= H;
  const long long runs = (long long)gridDim.x * kWarps, run = (long long)blockIdx.x * kWarps + (tid >> 5);
  const long long per = (all + runs - 1) / runs, lo = min(all, run * per);
  const long long lo_last = min(all, ((long long)blockIdx.x * kWarps + kWarps - 1) * per);  // the CTA's last warp's
  int left = (int)(min(all, lo + per) - lo);
  // where the run starts
  int b = -1, h = 0, c = 0, len = 0;
  long long carry = 0;
#pragma unroll 1
  for (int base = 0;; ) {
    start[tid] = before;
    count[tid] = n;
    __syncthreads();
    if (left > 0 && b < 0 && lo < (carry + tot) * H) {
#pragma unroll 1
      for (int k = 0; b < 0 && k < kWarps; ++k) {
        const long long s0 = (carry + start[32 * k + lane]) * H;
        const unsigned hit = __ballot_sync(0xffffffffu, s0 <= lo && lo < s0 + (long long)count[32 * k + lane] * H);
        if (hit == 0) continue;
        const int at = 32 * k + __ffs(hit) - 1, r = (int)(lo - (carry + start[at]) * H);
        b = base + at;
        len = count[at];
        h = r / len;
        c = r - h * len;
      }
    }
    carry += tot;
    base += kMassThreads;
    if (base >= a.batch || lo_last < carry * H) break;
    __syncthreads();
    n = steps(base + tid);
    before = block_excl_scan(n, warp_tot, &tot);
  }
  griddep_wait();  // (the lengths were complete before the decode let this kernel be launched)
  // Where a CTA of the decode gave up, scores and row states are not what they
  // should be: the call then adds no weights at all, so that it can be repeated.
  if (b < 0) return;
  int gave_up = 0;
  if (a.direct) {
    for (int i = lane; i < a.num_ctas; i += 32) gave_up |= __ldcg(a.gave_up + i);
    gave_up = __any_sync(0xffffffffu, gave_up);
  } else {
    gave_up = __ldcg(a.gave_up + a.num_ctas);  // the combine has looked through them
  }
  int L = clamp_ctx(a.context_lens, b, a.max_ctx, a.append);
  for (; left > 0; --left, ++c) {
    if (c == len) {  // the next KV head, or the next sequence that has tokens
      c = 0;
      if (++h == H) {
        h = 0;
        do {
          if (++b >= a.batch) return;  // (cannot happen while steps are left)
          len = steps(b);
        } while (len == 0);
        L = clamp_ctx(a.context_lens, b, a.max_ctx, a.append);
      }
    }
    const int head = b * H + h, t0 = a.window > 0 ? max(0, L - a.window) : 0;
    const int t = (first_step(L) + c) * kMassTokens + 4 * lane;
    if (t >= L || t + 4 <= t0) continue;
    const int blk = __ldg(a.block_tables + (size_t)b * a.bt_stride + (t >> a.real_shift));
    if (blk < 0 || blk >= a.num_blocks) continue;  // (flagged by the decode)
    float* dst = a.mass + ((size_t)blk * H + h) * bs + (t & (bs - 1));
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    const float* z = a.z + (size_t)head * G * a.z_stride + t;
#pragma unroll 4
    for (int g = 0; g < G; ++g) {
      const float2 st = __ldg(a.row_state + (size_t)head * G + g);
      const float4 v = __ldcs(reinterpret_cast<const float4*>(z + (size_t)g * a.z_stride));
      w[0] = fmaf(ex2(v.x - st.x), st.y, w[0]);
      w[1] = fmaf(ex2(v.y - st.x), st.y, w[1]);
      w[2] = fmaf(ex2(v.z - st.x), st.y, w[2]);
      w[3] = fmaf(ex2(v.w - st.x), st.y, w[3]);
    }
    if (gave_up) return;  // (not before: the word arrives beside the scores)
    // added atomically: forked sequences share blocks
    if (t >= t0 && t + 4 <= L - a.append) {
      asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(dst), "f"(w[0]), "f"(w[1]), "f"(w[2]), "f"(w[3])
                   : "memory");
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (t + k < t0 || t + k >= L) continue;
        if (!a.append || t + k < L - 1)
          atomicAdd(dst + k, w[k]);
        else
          dst[k] = w[k];  // the new token starts at its own weight
      }
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int kFp8Warps = 3;
constexpr int kDirectTokens = 1024;
constexpr int kFp8Ring = 96 * 1024;
constexpr int kFp8Smem = 227 * 1024 / 2 - 1024;  // of each of two CTAs on an SM

// Stream positions charged per segment for a piece's fixed cost: 40 KB worth
// of slices, as for the other decodes.
static int fp8_segment_cost(int slice, int head_dim) {
  const int bytes = 2 * slice * head_dim;
  return (40 * 1024 + bytes - 1) / bytes;
}

// The most (sequence, KV head) pairs that are taken whole (fp8_direct).
static int direct_ctas(const clove_fp8_pool& pool) { return 4 * pool.num_sms; }

struct Fp8Layout {
  int max_ctas;
  long long z_stride;
  size_t off_total, off_desc, off_partials, off_gave_up, off_rows, off_z, total;
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
  L.off_gave_up = up(L.off_partials + sizeof(float) * (size_t)L.max_ctas * 2 * group * state_stride(pool.head_dim));
  L.off_rows = L.off_z = L.total = L.off_gave_up;
  if (accumulate) {
    L.off_rows = up(L.off_gave_up + sizeof(int) * (size_t)std::max(L.max_ctas + 1, direct_ctas(pool)));
    L.off_z = up(L.off_rows + sizeof(float2) * (size_t)batch * num_q_heads);
    L.total = up(L.off_z + sizeof(float) * (size_t)batch * num_q_heads * L.z_stride);
  }
  return L;
}

// Few and short sequences, each KV head whole on one CTA: no partition to work
// out and nothing to combine.  Measured with 8 heads of 128, blocks of 16, in
// us against the split: 1 sequence of 100 / 1000 / 2000 tokens 9.4 / 16.5 /
// 22.6 against 20.5 / 19.2 / 20.5; 64 sequences (512 heads) of 100 / 1000:
// 18.5 / 37.1 against 22.3 / 40.0; 128 of 100 / 1000: 32.9 / 71.6 against 28.8
// / 60.8, since the CTAs then come in more than two waves.
static bool fp8_direct(const clove_fp8_pool& pool, int batch, int longest) {
  return (long long)batch * pool.num_kv_heads <= direct_ctas(pool) && longest <= kDirectTokens;
}

size_t fp8_decode_workspace(const clove_fp8_pool& pool, int batch, int num_q_heads, int max_ctx, int accumulate) {
  if (!accumulate && fp8_direct(pool, batch, max_ctx)) return 0;
  return fp8_layout(pool, batch, num_q_heads, max_ctx, accumulate).total;
}

// The codes as rows of 128 bytes (64 for head_dim 64) in two planes, a box
// being the K and V parts of one slice.
int fp8_encode_map(clove_fp8_pool& pool) {
  auto fn = tensor_map_encoder();
  if (!fn) {
    set_last_error("cuTensorMapEncodeTiled unavailable from the driver");
    return CLOVE_ERR_CUDA;
  }
  const int slice = std::min(pool.block_size, stage_tokens(pool.head_dim));
  const cuuint32_t inner = pool.head_dim >= 128 ? 128 : 64, rpt = pool.head_dim / inner;
  cuuint64_t dims[3] = {inner, (cuuint64_t)pool.plane_bytes / inner, 2};
  cuuint64_t strides[2] = {inner, (cuuint64_t)pool.plane_bytes};
  cuuint32_t box[3] = {inner, (cuuint32_t)slice * rpt, 2};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(&pool.map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, pool.codes, dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE,
                        inner == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("cuTensorMapEncodeTiled failed (%d) for head_dim %d block_size %d", (int)r, pool.head_dim,
                   pool.block_size);
    return CLOVE_ERR_CUDA;
  }
  return CLOVE_OK;
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

template <typename T, int D, bool kShaped, bool kKept, bool kTwin>
static int fp8_cfg(const clove_fp8_pool& pool, int slice, int group, Fp8Cfg* out) {
  static std::mutex mu;
  static std::unordered_map<long long, Fp8Cfg> cache;
  static std::unordered_map<int, int> attr;  // device -> shared memory the kernel may use there
  auto kern = fp8_decode_kernel<T, D, kFp8Warps, kShaped, kKept, kTwin>;
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
  const int sb = stage_tokens(D) / slice;
  const int scratch = (kFp8Warps - 1) * group * state_stride(D) * 4, qb = group * D * (int)sizeof(T);
  Fp8Cfg c;
  const int stage = smem_plan(slice, D, 1, sb, 1, scratch, qb, 1).stage_bytes;
  auto bytes = [&](int n) {
    return smem_plan(slice, D, 1, sb, n, scratch, qb, 1).total + kSclRing * (int)sizeof(SliceScales) + 1024;
  };
  // as deep a ring as two CTAs on an SM leave room for
  c.nstage = std::max(1, ring / stage / kFp8Warps) * kFp8Warps;
  while (c.nstage > kFp8Warps && (bytes(c.nstage) > kFp8Smem || c.nstage * sb + 32 > kSclRing)) c.nstage -= kFp8Warps;
  c.smem = bytes(c.nstage);
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

template <typename T, int D, bool kShaped, bool kKept, bool kTwin>
static int run_fp8(const clove_fp8_pool& pool, Fp8Args& a, cudaStream_t stream) {
  a.stage_blocks = stage_tokens(D) / a.block_size;
  Fp8Cfg c;
  int rc = fp8_cfg<T, D, kShaped, kKept, kTwin>(pool, a.block_size, a.group, &c);
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
                         launch_chained(fp8_decode_kernel<T, D, kFp8Warps, kShaped, kKept, kTwin>, dim3(a.num_ctas), (kFp8Warps + 1) * 32,
                                        c.smem, stream, pool.map, a));
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
    const long long items = (long long)a.batch * a.num_kv_heads * ((a.max_ctx + kMassTokens - 1LL) / kMassTokens);
    const dim3 grid((unsigned)std::min(items / (kMassThreads / 32) + 1, kMassCtas * (long long)pool.num_sms));
    rc = fp8_launch_status("fp8_decode weights launch", launch_chained(fp8_mass_kernel, grid, kMassThreads, 0, stream, a));
    if (rc) return rc;
    count_launches(1);
  }
  return CLOVE_OK;
}

template <typename T, int D>
static int run_fp8_scores(const clove_fp8_pool& pool, Fp8Args& a, cudaStream_t stream) {
  auto run = [&](auto twin) {
    const bool shaped = a.softcap > 0.f || a.slopes != nullptr;
    if (a.z != nullptr)
      return shaped ? run_fp8<T, D, true, true, twin.value>(pool, a, stream)
                    : run_fp8<T, D, false, true, twin.value>(pool, a, stream);
    return shaped ? run_fp8<T, D, true, false, twin.value>(pool, a, stream)
                  : run_fp8<T, D, false, false, twin.value>(pool, a, stream);
  };
  return a.group <= 4 ? run(std::true_type{}) : run(std::false_type{});
}

template <typename T>
static int run_fp8_dim(const clove_fp8_pool& pool, Fp8Args& a, cudaStream_t stream) {
  switch (pool.head_dim) {
    case 64: return run_fp8_scores<T, 64>(pool, a, stream);
    case 128: return run_fp8_scores<T, 128>(pool, a, stream);
    default: return run_fp8_scores<T, 256>(pool, a, stream);
  }
}

int launch_fp8_decode(const clove_fp8_pool& pool, const Fp8DecodeCall& c, cudaStream_t stream) {
  const Fp8Layout L = fp8_layout(pool, c.batch, c.num_q_heads, c.max_ctx, c.scores.accumulate);
  unsigned char* ws = static_cast<unsigned char*>(c.workspace);
  const int slice = std::min(pool.block_size, stage_tokens(pool.head_dim));
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
  while ((1 << a.slice_shift) < slice) ++a.slice_shift;
  while ((1 << a.real_shift) < pool.block_size) ++a.real_shift;
  a.window = c.scores.window;
  a.scale = c.scale;
  a.softcap = c.scores.softcap;
  if (c.scores.accumulate) {
    a.row_state = reinterpret_cast<float2*>(ws + L.off_rows);
    a.gave_up = reinterpret_cast<int*>(ws + L.off_gave_up);
    a.z = reinterpret_cast<float*>(ws + L.off_z);
    a.z_stride = L.z_stride;
  }
  a.direct = fp8_direct(pool, c.batch, c.scores.window > 0 ? std::min(c.scores.window, c.max_ctx) : c.max_ctx);
  // the partition counts a CTA's share and 128 sequences' slices in 32 bits
  const long long slices = (c.max_ctx + slice - 1LL) / slice + a.seg_cost;
  if (slices > 0x7fffffffLL / 128 || slices * c.batch * pool.num_kv_heads / (2 * pool.num_sms) > 0x7fffffffLL) {
    set_last_error("fp8_decode: batch %d of up to %d tokens is more than the partition counts", c.batch, c.max_ctx);
    return CLOVE_ERR_UNSUPPORTED;
  }
  a.append_here = a.append && (a.direct || slice == pool.block_size);
  switch (c.dtype) {
    case CLOVE_DTYPE_F32: return run_fp8_dim<float>(pool, a, stream);
    case CLOVE_DTYPE_F16: return run_fp8_dim<__half>(pool, a, stream);
    default: return run_fp8_dim<__nv_bfloat16>(pool, a, stream);
  }
}

}  // namespace clove
