// The combine kernel of the decodes (decode_kernels.cu, fp8_decode.cu): merges
// the partial softmax states of the segments that the equal-work partition
// split at CTA boundaries (decode_common.cuh).
#pragma once

#include "common.cuh"
#include "decode_common.cuh"

namespace clove {

// ---------------------------------------------------------------------------
// combine
// ---------------------------------------------------------------------------
// Segments split by CTA boundaries: segment s is split iff some boundary
// range_begin(c), 0 < c < P, falls strictly inside it; its pieces are those
// of CTAs cta_of(S) .. cta_of(S + len - 1).  The CTA whose range starts at
// (or before) S keeps its piece in partial slot 1 (its last piece) unless its
// range starts exactly at S (slot 0); every later CTA keeps it in slot 0 (its
// first piece).  Combine CTAs stride over the boundaries c and merge the
// segment whose first interior boundary is c.
constexpr int kCombineThreads = 128;
constexpr int kCombineMaxPieces = 1024;  // >= P (decode CTAs) - checked on the host

// Pieces merged per pass (more are merged in passes, carrying a running state).
constexpr int kCombinePass = 256;

// Merge the np partial states listed in pieces[] (partial slot indices
// c * 2 + slot) of segment (b, h) and write outputs [o_begin, o_end) of its
// rows (output o = row o / (D/4), dims 4 (o % (D/4)) ..).  All threads of the
// CTA take part; per pass, every load of a phase is independent of the
// others, so a pass costs a few memory round trips whatever the piece count:
//   1. (m, l) of every (piece, row) into shared memory;
//   2. per row g: M = max_i m_i, w_i = 2^(m_i - M), L = sum_i w_i l_i;
//   3. each thread sums four dims of one row over all pieces (16-byte loads).
template <int D, typename Args>
__device__ void combine_segment(const Args& a, int b, int h, const int* pieces, int np, float* pm, float* pl,
                                float* run, float* rowv, int o_begin, int o_end) {
  constexpr int S = state_stride(D);
  constexpr int NW = kCombineThreads / 32;
  const int group = a.group;
  const int Hq = a.num_kv_heads * group;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float* rowM = rowv;         // [8] reference max of the pass
  float* rowL = rowv + 8;     // [8] sum of weights times l (running)
  float* rowR = rowv + 16;    // [8] factor on the running state
  for (int base = 0; base < np; base += kCombinePass) {
    const int n = min(kCombinePass, np - base);
    const bool first = base == 0, last = base + n >= np;
    for (int i = tid; i < n * group; i += kCombineThreads) {
      const int p = i / group, g = i - p * group;
      const float* src = a.partials + ((size_t)pieces[base + p] * group + g) * S;
      pm[i] = __ldcg(src + D);
      pl[i] = __ldcg(src + D + 1);
    }
    __syncthreads();
    for (int g = warp; g < group; g += NW) {
      float M = first ? -INFINITY : rowM[g];
      for (int i = lane; i < n; i += 32) M = fmaxf(M, pm[i * group + g]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      float ls = 0.f;
      for (int i = lane; i < n; i += 32) {
        const float mi = pm[i * group + g];
        const float wi = mi == -INFINITY ? 0.f : exp2f(mi - M);
        pm[i * group + g] = wi;  // the weight replaces m
        ls = fmaf(wi, pl[i * group + g], ls);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o);
      if (lane == 0) {
        const float r = first || rowM[g] == -INFINITY ? 0.f : exp2f(rowM[g] - M);
        rowR[g] = r;
        rowL[g] = (first ? 0.f : rowL[g] * r) + ls;
        rowM[g] = M;
      }
    }
    __syncthreads();
    // Output float4s [o_begin, o_end): kpar threads (lanes of one warp) per
    // output, each summing every kpar-th piece, then a shuffle reduction, so
    // a small slice over many pieces is not one long chain of loads.
    const int nout = o_end - o_begin;
    int kpar = 1;
    while (kpar < 32 && 2 * kpar * nout <= kCombineThreads) kpar *= 2;
    const int sub = tid & (kpar - 1);
    // every lane runs the same number of rounds (the shuffles below are
    // warp-wide); lanes past the slice carry zeros and store nothing
    for (int o0 = o_begin; o0 < o_end; o0 += kCombineThreads / kpar) {
      const int o = o0 + tid / kpar;
      const bool live = o < o_end;
      const int g = live ? o / (D / 4) : 0, d4 = live ? o - g * (D / 4) : 0;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (live && !first && sub == 0) {
        const float r = rowR[g];
        const float4 v = reinterpret_cast<const float4*>(run + g * S)[d4];
        acc = make_float4(v.x * r, v.y * r, v.z * r, v.w * r);
      }
#pragma unroll 4
      for (int i = sub; live && i < n; i += kpar) {
        const float w = pm[i * group + g];
        const float4 v = __ldcg(reinterpret_cast<const float4*>(a.partials + ((size_t)pieces[base + i] * group + g) * S) + d4);
        acc.x = fmaf(w, v.x, acc.x);
        acc.y = fmaf(w, v.y, acc.y);
        acc.z = fmaf(w, v.z, acc.z);
        acc.w = fmaf(w, v.w, acc.w);
      }
      for (int off = kpar / 2; off > 0; off >>= 1) {
        acc.x += __shfl_xor_sync(0xffffffffu, acc.x, off, kpar);
        acc.y += __shfl_xor_sync(0xffffffffu, acc.y, off, kpar);
        acc.z += __shfl_xor_sync(0xffffffffu, acc.z, off, kpar);
        acc.w += __shfl_xor_sync(0xffffffffu, acc.w, off, kpar);
      }
      if (!live || sub != 0) continue;
      if (last) {
        const float inv = 1.f / rowL[g];
        if constexpr (Args::kKeepsRowState) {
          if (a.row_state != nullptr && d4 == 0) a.row_state[(size_t)b * Hq + h * group + g] = make_float2(rowM[g], inv);
        }
        float* dst = a.out + ((size_t)b * Hq + (size_t)h * group + g) * D + 4 * d4;
        dst[0] = acc.x * inv;
        dst[1] = acc.y * inv;
        dst[2] = acc.z * inv;
        dst[3] = acc.w * inv;
      } else {
        reinterpret_cast<float4*>(run + g * S)[d4] = acc;
      }
    }
    __syncthreads();
  }
}

template <int D, typename Args>
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(const Args a) {
  constexpr int S = state_stride(D);
  __shared__ float pm[kCombinePass * 8];
  __shared__ float pl[kCombinePass * 8];
  __shared__ __align__(16) float run[8 * S];  // running merged state between passes
  __shared__ float rowv[24];
  __shared__ int pieces[kCombineMaxPieces];
  __shared__ int s_np;
  // the kernel behind may set itself up now (it waits for this one before it reads results)
  if constexpr (Args::kKeepsRowState) griddep_launch_dependents();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if constexpr (kTrace) {
    if (a.trace && threadIdx.x == 0) atomicMin(a.trace + 2, gtime());
  }
  // The decode grid has finished: publish this call's check flags and clear
  // the accumulating word for the next call (whose decode waits for this
  // grid before it raises anything).
  if constexpr (Args::kPublishFlags) {
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      *a.err_last = *a.err;
      *a.err = 0;
    }
  }
  // did any CTA of the decode give up on a wait? (asked here, told below)
  int gave_up = 0;
  if constexpr (Args::kKeepsRowState) {
    if (blockIdx.x == 0 && a.gave_up != nullptr)
      for (int i = threadIdx.x; i < a.num_ctas; i += kCombineThreads) gave_up |= __ldcg(a.gave_up + i);
  }
  const long long W = *a.total;
  const long long P = a.num_ctas;
  const int alpha = a.seg_cost;
  const int n_out = a.group * (D / 4);  // float4 outputs of a segment
  for (int c = 1 + blockIdx.x; c < P; c += gridDim.x) {
    const int4 d = a.desc[c];
    // empty range, or the boundary does not fall inside the segment's blocks
    if (d.x < 0 || d.z <= alpha) continue;
    // segment (d.x, d.y) starts at stream position S0 and is d.w positions
    // long; its pieces belong to CTAs c_first .. c_last
    const long long S0 = range_begin(c, W, P) - d.z;
    const long long c_first = cta_of(S0 + alpha, W, P);
    const long long c_last = cta_of(S0 + d.w - 1, W, P);
    int helper = 0, helpers = 1, np;
    if (W >= P) {
      // no empty ranges: every boundary inside the segment has a combine
      // CTA, and they share the segment's outputs
      helper = (int)(c - c_first - 1);
      helpers = (int)(c_last - c_first);
      np = (int)(c_last - c_first + 1);
      const int slot_first = range_begin(c_first, W, P) < S0 ? 1 : 0;
      for (int i = threadIdx.x; i < np && i < kCombineMaxPieces; i += kCombineThreads)
        pieces[i] = (int)((c_first + i) * 2 + (i == 0 ? slot_first : 0));
      np = min(np, kCombineMaxPieces);
    } else {
      // less work than CTAs (empty ranges hold no piece): the first boundary
      // inside merges alone
      if (cta_of(range_begin(c, W, P) - 1, W, P) != c_first) continue;
      if (threadIdx.x == 0) {
        int n = 0;
        for (long long k = c_first; k <= c_last && n < kCombineMaxPieces; ++k) {
          if (range_begin(k, W, P) == range_begin(k + 1, W, P)) continue;
          pieces[n++] = (int)(k * 2 + ((k == c_first && range_begin(k, W, P) < S0) ? 1 : 0));
        }
        s_np = n;
      }
      __syncthreads();
      np = s_np;
    }
    __syncthreads();
    const int o_begin = (int)((long long)helper * n_out / helpers);
    const int o_end = (int)((long long)(helper + 1) * n_out / helpers);
    combine_segment<D, Args>(a, d.x, d.y, pieces, np, pm, pl, run, rowv, o_begin, o_end);
  }
  if constexpr (Args::kKeepsRowState) {
    if (blockIdx.x == 0 && a.gave_up != nullptr) {
      gave_up = __syncthreads_or(gave_up);
      if (threadIdx.x == 0) a.gave_up[a.num_ctas] = gave_up;
    }
  }
  if constexpr (kTrace) {
    if (a.trace && threadIdx.x == 0) atomicMax(a.trace + 3, gtime());
  }
}

}  // namespace clove
