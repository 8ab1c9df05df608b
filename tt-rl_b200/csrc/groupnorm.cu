// Group norm with a fused activation over channels-last rows, forward and
// backward.
//
// An image is `spatial` consecutive rows of `channels` floats; its group g
// is the columns [g*Cg, (g+1)*Cg) of all its rows. With mean and variance
// over a group,
//   hat = (x - mean) * rstd,  z = hat * w + b,  y = act(z),
// and with dz = dy * act'(z), d = dz * w (means over the group):
//   dx = rstd * (d - mean(d) - hat * mean(d * hat)),
//   dw = sum over images and rows of dz * hat,  db = the same sum of dz.
//
// The bound is memory: 8 bytes an element forward, 12 backward, if an image
// is read from memory once. So an image stays on chip between its statistics
// and its output, in one of four ways by its length (see pick_plan). Times are
// of B200, forward and backward (with the column sums behind it), shares of
// the measured copy rate in brackets:
//  - one row of up to 1024 floats whose groups are 2^k quads: one warp a row,
//    the next row under way while this one is reduced by shuffles. 32768 x
//    512: 25 us (83%), 50 us (62%);
//  - up to 1024 floats otherwise: one warp an image, group sums through shared
//    memory. 32768 x 488: 79 us (25%), 110 us: the sums of quads that straddle
//    groups are issue, not memory;
//  - up to 8 slots of a block's threads: one block an image, held in
//    registers. A thread's slots have the same columns in every period of the
//    block, so its weights, group indices and column sums are registers too.
//    4096 x 49 x 64: 31 us (51%), 43 us (55%);
//  - longer: one thread-block cluster an image, its rows staged in shared
//    memory forward, read again from L2 backward. 512 x 1764 x 90: 176 us
//    (57%), 341 us (44%): 25 to 30 warps an SM with one barrier of the cluster
//    an image do not cover the loads, the group sums (3000 cycles an image) and
//    the exchange (2500). Tried: the next image's rows fetched while this one
//    is written (the same); images dealt out as clusters finish, by a counter
//    (162 us, but two calls at once would share it) or by cancelling the launch
//    of clusters that have not started (176 us; 4 to 8% faster for images of a
//    quarter of the length); backward both operands staged (446 us), four slots
//    under way (377 us), a ring of slots by cp.async (320 us, and 5 to 12%
//    slower where a thread has fewer than 15 slots);
// and few long images, or rows wider than a block's threads, take three
// passes over global memory with per-column partial sums: 21 images of 5879 x
// 128 46 us and 71 us. (Batches of images whose sums one launch takes while it
// writes the batch before were 1.2 to 1.7 times slower: the sums' tail.)
// Variance is taken about means within a thread and in the passes over global
// memory (merged by the pairwise update of count, mean and sum of squares). The
// threads of a block or cluster add sums and sums of squares in 64 bits and
// subtract there: a mean of 10^k deviations costs 2k of 15 digits, fewer than its
// values' own roundings to float have cost. Every sum
// has a fixed order: results are bit for bit the same from run to run.
#include <algorithm>
#include <cstring>
#include <mutex>

#include "common.cuh"
#include "internal.h"

namespace ttrl {

struct GnArgs {
  const float* x;
  const float* dy;   // backward
  const float* w;    // [C], or null: ones
  const float* b;    // [C], or null: zeros
  float* y;          // forward: y; backward: dx
  float* stats;      // [N][G][2]: mean, rstd (forward may be null)
  float* partial;    // backward: [rows][2][C] sums of dz * hat and dz
  int32_t images, spatial, channels, groups;
  int32_t cg;        // channels of a group
  int32_t act;
  float eps;
  int32_t lpg;       // lanes that share a group's sum
  int32_t reps;      // replicas of the columns in a block's period
  int32_t ctas, rows_per;  // cluster: CTAs an image, rows a CTA
  FastDiv f_c, f_cg;
};

// 1 / (1 + exp(-z)) by the approximate exponential and reciprocal, each within
// two units in the last place of float (the exponent's own rounding adds |z| *
// 2^-24 where z is negative and large, and the value next to nothing), small
// results flushed to zero. The library's expf and division, and the forms that
// keep subnormals, cost 15 to 35 instructions an element more, and the kernels
// are then bound by instruction issue, not memory.
__device__ __forceinline__ float sigmoid_f(float z) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

// 1 / sqrt(x) for x > 0: the approximate root (within two units in the last
// place) and one Newton step.
__device__ __forceinline__ float rsqrt_f(float x) {
  const float r = rsqrtf(x);
  return fmaf(r * 0.5f, fmaf(-x * r, r, 1.f), r);
}

// Rounding may take a sum of squares below zero; NaN stays (fmaxf would drop
// it, and with it an infinity among the values).
__device__ __forceinline__ float at_least_zero(float x) { return x < 0.f ? 0.f : x; }

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if (ACT == TTRL_ACT_RELU) return z > 0.f ? z : 0.f;
  if (ACT == TTRL_ACT_SILU) return z * sigmoid_f(z);
  return z;
}

// dy * act'(z).
template <int ACT>
__device__ __forceinline__ float act_bwd(float dy, float z) {
  if (ACT == TTRL_ACT_RELU) return z > 0.f ? dy : 0.f;
  if (ACT == TTRL_ACT_SILU) {
    const float s = sigmoid_f(z);
    return dy * (s * (1.f + z * (1.f - s)));
  }
  return dy;
}

// z, by the same roundings in every kernel: a ReLU's gate in the backward is the
// forward's, whichever of them ran it.
__device__ __forceinline__ float norm_z(float hat, float w, float b) { return fmaf(hat, w, b); }

// Sum over the `lanes` (a power of two) consecutive lanes a lane belongs to.
__device__ __forceinline__ float seg_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int W>
struct Vec;
template <>
struct Vec<1> {
  float v[1];
  __device__ __forceinline__ void load_last(const float* p) { v[0] = __ldcs(p); }
  __device__ __forceinline__ void store_last(float* p) const { __stcs(p, v[0]); }
  __device__ __forceinline__ void load(const float* p) { v[0] = *p; }
  __device__ __forceinline__ void store(float* p) const { *p = v[0]; }
};
template <>
struct Vec<4> {
  float v[4];
  // Accesses that are a value's last: first to leave the caches.
  __device__ __forceinline__ void load_last(const float* p) {
    const float4 t = __ldcs(reinterpret_cast<const float4*>(p));
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  }
  __device__ __forceinline__ void store_last(float* p) const {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  }
  __device__ __forceinline__ void load(const float* p) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};

// ------------------------------------------------------- one warp an image

constexpr int kGnWarps = 8;

// Group sums of the values in `slot` (a warp's shared array of one image, a
// value for every W elements) divided by `count`, into out[g].
template <int W>
__device__ __forceinline__ void warp_group_sums(const GnArgs& a, const float* slot, float* out,
                                                float count, int lane) {
  const int cq = a.cg / W, row = a.channels / W, units = 32 / a.lpg;
  const int unit = lane / a.lpg, in = lane % a.lpg;
  for (int g0 = 0; g0 < a.groups; g0 += units) {
    const int g = g0 + unit;
    float s = 0.f;
    if (g < a.groups) {
      for (int r = 0; r < a.spatial; ++r)
        for (int i = in; i < cq; i += a.lpg) s += slot[r * row + g * cq + i];
    }
    s = seg_sum(s, a.lpg);
    if (in == 0 && g < a.groups) out[g] = s / count;
  }
  __syncwarp();
}

// Lane `lane` owns the R slots (r * 32 + lane) of W floats. EL: a slot may
// straddle groups or rows, so shared sums and lookups go by element (W = 4
// without EL: groups of whole quads).
template <int W, int R, int ACT, bool BWD, bool EL>
__global__ void __launch_bounds__(kGnWarps * 32) gn_warp_kernel(const __grid_constant__ GnArgs a) {
  extern __shared__ __align__(16) float gn_smem[];
  constexpr int SV = EL ? W : 1;  // shared values a slot
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int len = a.spatial * a.channels, slots = len / W;
  const int gpad = (a.groups + 3) & ~3;
  float* slot = gn_smem + warp * (R * 32 * SV + 2 * gpad);
  float* g1 = slot + R * 32 * SV;
  float* g2 = g1 + gpad;
  int col[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = r * 32 + lane;
    const int at = j < slots ? j * W : 0;
    col[r] = at - fdiv(a.f_c, at) * a.channels;
  }
  // The column and group of element e of slot r.
  auto column = [&](int r, int e) {
    if (!EL) return col[r] + e;
    const int c = col[r] + e;
    return c - fdiv(a.f_c, c) * a.channels;
  };
  auto group = [&](int r, int e) { return fdiv(a.f_cg, EL ? column(r, e) : col[r]); };
  // Values of a slot to the shared array: their sum, or each one.
  auto put = [&](int r, const float(&t)[W]) {
    if (EL && W == 4) {
      *reinterpret_cast<float4*>(slot + (r * 32 + lane) * 4) =
          make_float4(t[0], t[W > 1 ? 1 : 0], t[W > 2 ? 2 : 0], t[W > 3 ? 3 : 0]);
    } else {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < W; ++e) s += t[e];
      slot[r * 32 + lane] = s;
    }
  };
  auto params = [&](int r, const float* p, float none, Vec<W>& v) {
#pragma unroll
    for (int e = 0; e < W; ++e) v.v[e] = none;
    if (p == nullptr) return;
    if (EL) {
#pragma unroll
      for (int e = 0; e < W; ++e) v.v[e] = p[column(r, e)];
    } else {
      v.load(p + col[r]);
    }
  };
  constexpr int GW = EL ? 1 : W;
  float acc_w[BWD ? R : 1][W], acc_b[BWD ? R : 1][W];
#pragma unroll
  for (int r = 0; r < (BWD ? R : 1); ++r)
#pragma unroll
    for (int e = 0; e < W; ++e) acc_w[r][e] = acc_b[r][e] = 0.f;
  pdl_trigger();
  pdl_wait();
  const float count = static_cast<float>(a.spatial * a.cg);
  const int stride = gridDim.x * kGnWarps;
  for (int n = blockIdx.x * kGnWarps + warp; n < a.images; n += stride) {
    const long long base = static_cast<long long>(n) * len;
    Vec<W> x[R], dy[BWD ? R : 1];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = r * 32 + lane;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        x[r].v[e] = 0.f;
        if (BWD) dy[BWD ? r : 0].v[e] = 0.f;
      }
      if (j < slots) {
        x[r].load(a.x + base + j * W);
        if (BWD) dy[BWD ? r : 0].load(a.dy + base + j * W);
      }
    }
    if (!BWD) {
#pragma unroll
      for (int r = 0; r < R; ++r) put(r, x[r].v);
      __syncwarp();
      warp_group_sums<GW>(a, slot, g1, count, lane);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float t[W];
        float m = g1[group(r, 0)];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          if (EL && e > 0) m = g1[group(r, e)];
          x[r].v[e] -= m;
          t[e] = x[r].v[e] * x[r].v[e];
        }
        put(r, t);
      }
      __syncwarp();
      warp_group_sums<GW>(a, slot, g2, count, lane);
      for (int g = lane; g < a.groups; g += 32) {
        const float rstd = rsqrt_f(g2[g] + a.eps);
        g2[g] = rstd;
        if (a.stats != nullptr) {
          float* st = a.stats + (static_cast<long long>(n) * a.groups + g) * 2;
          st[0] = g1[g];
          st[1] = rstd;
        }
      }
      __syncwarp();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = r * 32 + lane;
        if (j >= slots) continue;
        Vec<W> w, b;
        params(r, a.w, 1.f, w);
        params(r, a.b, 0.f, b);
        float rstd = g2[group(r, 0)];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          if (EL && e > 0) rstd = g2[group(r, e)];
          x[r].v[e] = act_fwd<ACT>(norm_z(x[r].v[e] * rstd, w.v[e], b.v[e]));
        }
        x[r].store(a.y + base + j * W);
      }
      __syncwarp();  // the next image rewrites the shared sums
    } else {
      for (int g = lane; g < a.groups; g += 32) {
        const float* st = a.stats + (static_cast<long long>(n) * a.groups + g) * 2;
        g1[g] = st[0];
        g2[g] = st[1];
      }
      __syncwarp();
      float rs[R][EL ? W : 1];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = r * 32 + lane;
        float t[W];
#pragma unroll
        for (int e = 0; e < W; ++e) t[e] = 0.f;
        rs[r][0] = g2[group(r, 0)];
        if (j < slots) {
          Vec<W> w, b;
          params(r, a.w, 1.f, w);
          params(r, ACT == TTRL_ACT_NONE ? nullptr : a.b, 0.f, b);
          float m = g1[group(r, 0)];
#pragma unroll
          for (int e = 0; e < W; ++e) {
            if (EL && e > 0) {
              m = g1[group(r, e)];
              rs[r][EL ? e : 0] = g2[group(r, e)];
            }
            const float hat = (x[r].v[e] - m) * rs[r][EL ? e : 0];
            const float dz = act_bwd<ACT>(dy[BWD ? r : 0].v[e], norm_z(hat, w.v[e], b.v[e]));
            acc_w[BWD ? r : 0][e] = fmaf(dz, hat, acc_w[BWD ? r : 0][e]);
            acc_b[BWD ? r : 0][e] += dz;
            x[r].v[e] = hat;
            t[e] = dz * w.v[e];
            dy[BWD ? r : 0].v[e] = t[e];
          }
        }
        put(r, t);
      }
      __syncwarp();
      warp_group_sums<GW>(a, slot, g1, count, lane);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float t[W];
#pragma unroll
        for (int e = 0; e < W; ++e) t[e] = dy[BWD ? r : 0].v[e] * x[r].v[e];
        put(r, t);
      }
      __syncwarp();
      warp_group_sums<GW>(a, slot, g2, count, lane);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = r * 32 + lane;
        if (j >= slots) continue;
        float m1 = g1[group(r, 0)], m2 = g2[group(r, 0)];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          if (EL && e > 0) {
            m1 = g1[group(r, e)];
            m2 = g2[group(r, e)];
          }
          x[r].v[e] = rs[r][EL ? e : 0] * (dy[BWD ? r : 0].v[e] - m1 - x[r].v[e] * m2);
        }
        x[r].store(a.y + base + j * W);
      }
      __syncwarp();
    }
  }
  if (BWD && a.partial != nullptr) {
    // Column sums of this block: warps in order, then a column's rows.
    __syncthreads();
    float* sums = gn_smem;  // [slots * W] of one kind at a time
    float* out = a.partial + static_cast<long long>(blockIdx.x) * 2 * a.channels;
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      for (int wv = 0; wv < kGnWarps; ++wv) {
        if (warp == wv) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int j = r * 32 + lane;
            if (j >= slots) continue;
#pragma unroll
            for (int e = 0; e < W; ++e) {
              const float v = kind == 0 ? acc_w[BWD ? r : 0][e] : acc_b[BWD ? r : 0][e];
              sums[j * W + e] = wv == 0 ? v : sums[j * W + e] + v;
            }
          }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < a.channels; c += blockDim.x) {
        float s = 0.f;
        for (int r = 0; r < a.spatial; ++r) s += sums[r * a.channels + c];
        out[kind * a.channels + c] = s;
      }
      __syncthreads();
    }
  }
}

// Images of one row whose groups are 2^k quads: a group is a run of lanes (or
// of whole slots), so its sum is a few shuffles (and register adds) and every
// lane has it; the next row is on its way while this one is reduced. The form
// above spends 50 instructions an element on the same rows, this one 17.
template <int R, int ACT, bool BWD>
__global__ void __launch_bounds__(kGnWarps * 32, R <= 4 ? (BWD ? 2 : 3) : 1)
    gn_row_kernel(const __grid_constant__ GnArgs a) {
  extern __shared__ __align__(16) float gn_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slots = a.channels / 4, per = a.cg / 4;
  const int lanes = min(per, 32), span = per <= 32 ? 1 : per / 32;
  const int shift = __ffs(per) - 1;  // slot to group
  auto group_sums = [&](float (&t)[R]) {
#pragma unroll
    for (int o = 1; o < R; o *= 2)
      if (o < span) {
        float u[R];
#pragma unroll
        for (int r = 0; r < R; ++r) u[r] = t[r] + t[r ^ o];
#pragma unroll
        for (int r = 0; r < R; ++r) t[r] = u[r];
      }
    for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int r = 0; r < R; ++r) t[r] += __shfl_xor_sync(0xffffffffu, t[r], o);
  };
  float acc_w[BWD ? R : 1][4], acc_b[BWD ? R : 1][4];
#pragma unroll
  for (int r = 0; r < (BWD ? R : 1); ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc_w[r][e] = acc_b[r][e] = 0.f;
  pdl_trigger();
  pdl_wait();
  const float inv = 1.f / static_cast<float>(a.cg);
  const int stride = gridDim.x * kGnWarps;
  Vec<4> next[R], next_dy[BWD ? R : 1];
  auto fetch = [&](int n) {
    const float* px = a.x + static_cast<long long>(n) * a.channels + lane * 4;
    const float* pd = a.dy + static_cast<long long>(n) * a.channels + lane * 4;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        next[r].v[e] = 0.f;
        if (BWD) next_dy[BWD ? r : 0].v[e] = 0.f;
      }
      if (r * 32 + lane < slots) {
        next[r].load(px + r * 128);
        if (BWD) next_dy[BWD ? r : 0].load(pd + r * 128);
      }
    }
  };
  int n = blockIdx.x * kGnWarps + warp;
  if (n < a.images) fetch(n);
  for (; n < a.images; n += stride) {
    Vec<4> x[R], dy[BWD ? R : 1];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      x[r] = next[r];
      if (BWD) dy[BWD ? r : 0] = next_dy[BWD ? r : 0];
    }
    if (n + stride < a.images) fetch(n + stride);
    const long long base = static_cast<long long>(n) * a.channels;
    float* st = a.stats + static_cast<long long>(n) * a.groups * 2;
    float t1[R], t2[R];
    if (!BWD) {
#pragma unroll
      for (int r = 0; r < R; ++r) t1[r] = (x[r].v[0] + x[r].v[1]) + (x[r].v[2] + x[r].v[3]);
      group_sums(t1);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        t1[r] *= inv;
        t2[r] = 0.f;
        if (r * 32 + lane < slots)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[r].v[e] -= t1[r];
            t2[r] = fmaf(x[r].v[e], x[r].v[e], t2[r]);
          }
      }
      group_sums(t2);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = r * 32 + lane;
        if (j >= slots) continue;
        const float rstd = rsqrt_f(fmaf(t2[r], inv, a.eps));
        if (a.stats != nullptr && (j & (per - 1)) == 0)
          *reinterpret_cast<float2*>(st + (j >> shift) * 2) = make_float2(t1[r], rstd);
        Vec<4> w, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.v[e] = 1.f, b.v[e] = 0.f;
        if (a.w != nullptr) w.load(a.w + j * 4);
        if (a.b != nullptr) b.load(a.b + j * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[r].v[e] = act_fwd<ACT>(norm_z(x[r].v[e] * rstd, w.v[e], b.v[e]));
        x[r].store(a.y + base + j * 4);
      }
    } else {
      float rs[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = r * 32 + lane;
        t1[r] = t2[r] = rs[r] = 0.f;
        if (j >= slots) continue;
        const float2 mr = *reinterpret_cast<const float2*>(st + (j >> shift) * 2);
        rs[r] = mr.y;
        Vec<4> w, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.v[e] = 1.f, b.v[e] = 0.f;
        if (a.w != nullptr) w.load(a.w + j * 4);
        if (ACT != TTRL_ACT_NONE && a.b != nullptr) b.load(a.b + j * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float hat = (x[r].v[e] - mr.x) * mr.y;
          const float dz = act_bwd<ACT>(dy[BWD ? r : 0].v[e], norm_z(hat, w.v[e], b.v[e]));
          acc_w[BWD ? r : 0][e] = fmaf(dz, hat, acc_w[BWD ? r : 0][e]);
          acc_b[BWD ? r : 0][e] += dz;
          const float d = dz * w.v[e];
          x[r].v[e] = hat;
          dy[BWD ? r : 0].v[e] = d;
          t1[r] += d;
          t2[r] = fmaf(d, hat, t2[r]);
        }
      }
      group_sums(t1);
      group_sums(t2);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = r * 32 + lane;
        if (j >= slots) continue;
        const float m1 = t1[r] * inv, m2 = t2[r] * inv;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[r].v[e] = rs[r] * (dy[BWD ? r : 0].v[e] - m1 - x[r].v[e] * m2);
        x[r].store(a.y + base + j * 4);
      }
    }
  }
  if (BWD && a.partial != nullptr) {
    // Column sums of this block, its warps in order.
    float* out = a.partial + static_cast<long long>(blockIdx.x) * 2 * a.channels;
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = r * 32 + lane;
        if (j >= slots) continue;
        const float(&v)[4] = kind == 0 ? acc_w[BWD ? r : 0] : acc_b[BWD ? r : 0];
        *reinterpret_cast<float4*>(gn_smem + warp * a.channels + j * 4) =
            make_float4(v[0], v[1], v[2], v[3]);
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.channels; c += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < kGnWarps; ++q) s += gn_smem[q * a.channels + c];
        out[kind * a.channels + c] = s;
      }
    }
  }
}

// ------------------------------------------------------ one block an image

// Group sums over a block of two per-thread column values, in 64 bits: entry
// j of v1 and v2 (T * W of them) belongs to column j % C. SQUARES: v1 is the
// mean of an entry's values and v2 their sum of squares about it, and the sums
// are those of the values and of their squares (which 64 bits can subtract);
// entry j has `slots` values, and one more below `rest`. Else the plain sums.
// out[g] = the two sums.
template <int W, bool SQUARES>
__device__ __forceinline__ void block_group_sums(const GnArgs& a, const float* v1,
                                                 const float* v2, double2* out, int threads,
                                                 float slots, int rest) {
  const int units = threads / a.lpg;
  const int unit = threadIdx.x / a.lpg, in = threadIdx.x % a.lpg;
  const int items = a.reps * a.cg;
  // A unit lies in one warp (lpg divides 32); threads past the last whole
  // unit and groups past the last add nothing but take part in the shuffle.
  for (int g0 = 0; g0 < a.groups; g0 += units) {
    const int g = g0 + unit;
    double s1 = 0.0, s2 = 0.0;
    if (unit < units && g < a.groups) {
#pragma unroll 4
      for (int i = in; i < items; i += a.lpg) {
        const int rep = fdiv(a.f_cg, i);
        const int j = rep * a.channels + g * a.cg + (i - rep * a.cg);
        if (SQUARES) {
          const double m = v1[j], t = (j < rest ? slots + 1.f : slots) * m;
          s1 += t;
          s2 += fma(t, m, static_cast<double>(v2[j]));
        } else {
          s1 += v1[j];
          s2 += v2[j];
        }
      }
    }
    for (int o = a.lpg >> 1; o > 0; o >>= 1) {
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
      s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    }
    if (in == 0 && unit < units && g < a.groups) out[g] = make_double2(s1, s2);
  }
  __syncthreads();
}

// Mean and 1 / sqrt(variance + eps) from the sum and the sum of squares; inv =
// 1 / count.
__device__ __forceinline__ float2 mean_rstd(double s1, double s2, double inv, float eps) {
  const double m = s1 * inv;
  const float var = at_least_zero(static_cast<float>(fma(s2, inv, -m * m)));
  return make_float2(static_cast<float>(m), rsqrt_f(var + eps));
}

// A block's threads own the slots (r * T + tid), r < R, of W floats of its
// rows, held in registers. T * W is a multiple of the channels, so a
// thread's columns are the same in every slot. blockDim.x is T rounded up to
// whole warps; threads past T own nothing.
template <int W, int R, int ACT, bool BWD>
__global__ void __launch_bounds__(512) gn_block_kernel(const __grid_constant__ GnArgs a) {
  extern __shared__ __align__(16) float gn_smem[];
  const int threads = a.reps * a.channels / W;
  const int tid = threadIdx.x;
  const int len = tid < threads ? a.spatial * a.channels : 0;
  double2* sums = reinterpret_cast<double2*>(gn_smem);     // group sums
  float2* got = reinterpret_cast<float2*>(sums + a.groups);  // what they give
  float* cols = reinterpret_cast<float*>(got + a.groups);  // [threads * W]
  float* cols2 = cols + threads * W;
  int gid[W];
  float w[W], b[W], aw[W], ab[W];
  pdl_trigger();
  pdl_wait();
#pragma unroll
  for (int e = 0; e < W; ++e) {
    const int at = tid * W + e;
    const int c = at - fdiv(a.f_c, at) * a.channels;
    gid[e] = fdiv(a.f_cg, c);
    w[e] = a.w != nullptr ? a.w[c] : 1.f;
    b[e] = a.b != nullptr ? a.b[c] : 0.f;
    aw[e] = ab[e] = 0.f;
  }
  const int step = threads * W;
  const int first = tid * W;
  const double inv_total = 1.0 / (static_cast<double>(a.spatial) * a.cg);
  const int whole = a.spatial * a.channels;
  const float slots = static_cast<float>(whole / step);
  const int rest = whole % step;
  // Slots of this thread.
  const int k = len > first ? (len - first - 1) / step + 1 : 0;
  const float inv = k > 0 ? 1.f / static_cast<float>(k) : 0.f;
  // Forward, the next image's loads are under way while one is reduced.
  Vec<W> next[BWD ? 1 : R];
  if (!BWD && static_cast<int>(blockIdx.x) < a.images) {
    const float* from = a.x + static_cast<long long>(blockIdx.x) * whole + first;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < k) next[BWD ? 0 : r].load(from + r * step);
  }
  for (int n = blockIdx.x; n < a.images; n += gridDim.x) {
    const long long base = static_cast<long long>(n) * whole + first;
    Vec<W> x[R], dy[BWD ? R : 1];
    if (!BWD) {
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = next[BWD ? 0 : r];
      if (n + static_cast<int>(gridDim.x) < a.images) {
        const float* from = a.x + base + static_cast<long long>(gridDim.x) * whole;
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (r < k) next[BWD ? 0 : r].load(from + r * step);
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r < k) {
          x[r].load(a.x + base + r * step);
          dy[BWD ? r : 0].load(a.dy + base + r * step);
        }
    }
    if (!BWD) {
      // Each thread's mean and sum of squares about it, a column at a time:
      // one pass about its own first value (which is one of the at most R
      // values, so the difference of squares loses at most log2 R bits).
#pragma unroll
      for (int e = 0; e < W; ++e) {
        float mt = 0.f, q = 0.f;
        if (k > 0) {
          const float x0 = x[0].v[e];
          float s = 0.f;
#pragma unroll
          for (int r = 1; r < R; ++r) {
            if (r < k) {
              const float d = x[r].v[e] - x0;
              s += d;
              q = fmaf(d, d, q);
            }
          }
          const float d = s * inv;
          mt = x0 + d;
          q = at_least_zero(fmaf(-s, d, q));
        }
        if (tid < threads) {
          cols[first + e] = mt;
          cols2[first + e] = q;
        }
      }
      __syncthreads();
      block_group_sums<W, true>(a, cols, cols2, sums, threads, slots, rest);
      for (int g = tid; g < a.groups; g += blockDim.x) {
        const float2 t = mean_rstd(sums[g].x, sums[g].y, inv_total, a.eps);
        got[g] = t;
        if (a.stats != nullptr)
          *reinterpret_cast<float2*>(a.stats + (static_cast<long long>(n) * a.groups + g) * 2) = t;
      }
      __syncthreads();
      float m[W], rs[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        m[e] = got[gid[e]].x;
        rs[e] = got[gid[e]].y;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= k) continue;
#pragma unroll
        for (int e = 0; e < W; ++e)
          x[r].v[e] = act_fwd<ACT>(norm_z((x[r].v[e] - m[e]) * rs[e], w[e], b[e]));
        x[r].store(a.y + base + r * step);
      }
    } else {
      float m[W], rs[W], t1[W], t2[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float* st = a.stats + (static_cast<long long>(n) * a.groups + gid[e]) * 2;
        m[e] = st[0];
        rs[e] = st[1];
        t1[e] = t2[e] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= k) continue;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float hat = (x[r].v[e] - m[e]) * rs[e];
          const float dz = act_bwd<ACT>(dy[BWD ? r : 0].v[e], norm_z(hat, w[e], b[e]));
          t1[e] += dz;
          t2[e] = fmaf(dz, hat, t2[e]);
          x[r].v[e] = hat;
          dy[BWD ? r : 0].v[e] = dz;
        }
      }
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (tid < threads) {
          cols[first + e] = t1[e] * w[e];
          cols2[first + e] = t2[e] * w[e];
        }
        ab[e] += t1[e];
        aw[e] += t2[e];
      }
      __syncthreads();
      block_group_sums<W, false>(a, cols, cols2, sums, threads, 0.f, 0);
      for (int g = tid; g < a.groups; g += blockDim.x)
        got[g] = make_float2(static_cast<float>(sums[g].x * inv_total),
                             static_cast<float>(sums[g].y * inv_total));
      __syncthreads();
      float m1[W], m2[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        m1[e] = got[gid[e]].x;
        m2[e] = got[gid[e]].y;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= k) continue;
#pragma unroll
        for (int e = 0; e < W; ++e)
          x[r].v[e] = rs[e] * (fmaf(dy[BWD ? r : 0].v[e], w[e], -m1[e]) - x[r].v[e] * m2[e]);
        x[r].store(a.y + base + r * step);
      }
    }
    __syncthreads();  // every thread has read the group sums
  }
  if (BWD && a.partial != nullptr) {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      if (tid < threads) {
        cols[first + e] = aw[e];
        cols2[first + e] = ab[e];
      }
    }
    __syncthreads();
    float* out = a.partial + static_cast<long long>(blockIdx.x) * 2 * a.channels;
    for (int c = tid; c < a.channels; c += blockDim.x) {
      float s1 = 0.f, s2 = 0.f;
      for (int r = 0; r < a.reps; ++r) {
        s1 += cols[r * a.channels + c];
        s2 += cols2[r * a.channels + c];
      }
      out[c] = s1;
      out[a.channels + c] = s2;
    }
  }
}

// ------------------------------------------- longer images: clusters walk

__device__ __forceinline__ void gn_cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void gn_cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Store two doubles at shared address p of cluster CTA `rank`.
__device__ __forceinline__ void st_peer2(double2* p, int rank, double2 v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(remote), "d"(v.x), "d"(v.y)
               : "memory");
}

// An SM holds two CTAs of 512 threads or four of 256, at 64 registers: one's
// barriers hide behind another's loads.
constexpr int kGnMaxCluster = 16;
constexpr int kGnRun = 32;

// An image too long for a block: a cluster of `ctas` CTAs copies its rows to
// shared memory (STAGED), sums them, exchanges the sums (every CTA sends its
// two of each group to all; reading them from one peer after another cost a
// round trip each) and writes the output. An image that 16 CTAs cannot hold is
// read twice instead, the second time from L2 as far as the images under way,
// one a cluster, fit there. A thread's columns are the same in every period,
// as in the block form. Clusters walk over the images, all of them resident.
// recv[rank][group] alternates between two buffers by image: a CTA sends
// image i + 2 after every peer has passed the barrier of image i + 1, and so
// has read image i: one barrier an image is enough.
template <int W, int ACT, bool BWD, bool STAGED>
__global__ void __launch_bounds__(512, 2) gn_cluster_kernel(const __grid_constant__ GnArgs a) {
  extern __shared__ __align__(16) float gn_smem[];
  // Slots whose loads are in flight. Staged, from shared memory, two are enough
  // and four spill: 512 images of 1764 x 90 173 us against 186.
  constexpr int U = BWD || STAGED ? 2 : 4;
  const int threads = a.reps * a.channels / W;
  const int tid = threadIdx.x;
  const int rank = blockIdx.x % a.ctas;
  const int row0 = min(a.spatial, rank * a.rows_per);
  const int rows = min(a.spatial, row0 + a.rows_per) - row0;
  const bool mine = tid < threads;
  const int len = mine ? rows * a.channels : 0;
  const int first = tid * W, step = threads * W;
  const float slots = static_cast<float>(rows * a.channels / step);
  const int rest = rows * a.channels % step;
  double2* sums = reinterpret_cast<double2*>(gn_smem);        // this CTA's group sums
  double2* recv = sums + a.groups;                            // [2][ctas][groups]
  float2* merged = reinterpret_cast<float2*>(recv + 2 * a.ctas * a.groups);
  float* cols = reinterpret_cast<float*>(merged + a.groups);  // [threads * W]
  float* cols2 = cols + step;
  int parity = 0;
  // Peers write into recv only once this block runs: waited for before the
  // first exchange.
  gn_cluster_arrive();
  bool met = false;
  // Column and group of this thread's element e, worked out where needed: a
  // register each would spill.
  auto col = [&](int e) { return first + e - fdiv(a.f_c, first + e) * a.channels; };
  auto gid = [&](int e) { return fdiv(a.f_cg, col(e)); };
  // Backward: this thread's sums of dz * hat and dz over its images.
  float* acc = cols2 + step;  // [2][threads * W]
  // Staged (forward only): this CTA's rows of x.
  float* sx = reinterpret_cast<float*>(
      (reinterpret_cast<uintptr_t>(acc + (BWD ? 2 * step : 0)) + 15) & ~static_cast<uintptr_t>(15));
  if (BWD && mine)
#pragma unroll
    for (int e = 0; e < W; ++e) acc[first + e] = acc[step + first + e] = 0.f;
  // f(live, i) for slots i, i + step, ... below end, U at a time: live(u) says
  // which are there, all of them but in the last turn.
  auto walk = [&](int i, int end, auto&& f) {
    for (; i + (U - 1) * step < end; i += U * step) f([](int) { return true; }, i);
    if (i < end) f([&](int u) { return i + u * step < end; }, i);
  };
  pdl_trigger();
  pdl_wait();
  const double inv_total = 1.0 / (static_cast<double>(a.spatial) * a.cg);
  const int clusters = gridDim.x / a.ctas;
  for (int n = blockIdx.x / a.ctas; n < a.images; n += clusters) {
    const long long base = (static_cast<long long>(n) * a.spatial + row0) * a.channels;
    const float* xs = a.x + base;
    float* ys = a.y + base;
    const float* st = a.stats + static_cast<long long>(n) * a.groups * 2;
    const float* dys = BWD ? a.dy + base : nullptr;
    if (STAGED) {
      // A thread copies the slots it reads; all of them are under way at once.
      for (int i = first; i < len; i += step) {
        if (W == 4)
          cp_async16(smem_u32(sx + i), xs + i, 16);
        else
          cp_async4(smem_u32(sx + i), xs + i, 4);
      }
      cp_async_commit();
      cp_async_wait<0>();
    }
    auto get_x = [&](Vec<W>& v, int i, bool last) {
      if (STAGED)
        v.load(sx + i);
      else if (last)
        v.load_last(xs + i);
      else
        v.load(xs + i);
    };
    auto get_dy = [&](Vec<W>& v, int i, bool last) {
      if (last)
        v.load_last(dys + i);
      else
        v.load(dys + i);
    };
    if (!BWD) {
      // Runs of at most kGnRun slots, each summed about its first value (one
      // of them, so the difference of squares loses at most log2 kGnRun bits)
      // and merged into the thread's mean and squares about it.
      float mt[W], q[W], cnt = 0.f;
#pragma unroll
      for (int e = 0; e < W; ++e) mt[e] = q[e] = 0.f;
      for (int i0 = first; i0 < len; i0 += kGnRun * step) {
        const int stop = min(len, i0 + kGnRun * step);
        float x0[W], s1[W], s2[W];
        Vec<W> v;
        get_x(v, i0, false);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          x0[e] = v.v[e];
          s1[e] = s2[e] = 0.f;
        }
        walk(i0 + step, stop, [&](auto live, int i) {
          Vec<W> x[U];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (live(u)) get_x(x[u], i + u * step, false);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (live(u))
#pragma unroll
              for (int e = 0; e < W; ++e) {
                const float d = x[u].v[e] - x0[e];
                s1[e] += d;
                s2[e] = fmaf(d, d, s2[e]);
              }
        });
        const float n1 = static_cast<float>((stop - i0 + step - 1) / step), all = cnt + n1;
        const float share = __fdividef(n1, all), inv = __fdividef(1.f, n1);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float m = s1[e] * inv;
          const float d = x0[e] + m - mt[e];
          mt[e] = fmaf(d, share, mt[e]);
          q[e] += at_least_zero(fmaf(-s1[e], m, s2[e])) + d * d * (cnt * share);
        }
        cnt = all;
      }
      if (mine)
#pragma unroll
        for (int e = 0; e < W; ++e) {
          cols[first + e] = mt[e];
          cols2[first + e] = q[e];
        }
      __syncthreads();
      block_group_sums<W, true>(a, cols, cols2, sums, threads, slots, rest);
    } else {
      float m[W], rs[W], w[W], b[W], t1[W], t2[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        m[e] = st[gid(e) * 2];
        rs[e] = st[gid(e) * 2 + 1];
        w[e] = a.w != nullptr ? a.w[col(e)] : 1.f;
        b[e] = a.b != nullptr ? a.b[col(e)] : 0.f;
        t1[e] = t2[e] = 0.f;
      }
      walk(first, len, [&](auto live, int i) {
        Vec<W> x[U], dy[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (live(u)) {
            get_x(x[u], i + u * step, false);
            get_dy(dy[u], i + u * step, false);
          }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (live(u))
#pragma unroll
            for (int e = 0; e < W; ++e) {
              const float hat = (x[u].v[e] - m[e]) * rs[e];
              const float dz = act_bwd<ACT>(dy[u].v[e], norm_z(hat, w[e], b[e]));
              t1[e] += dz;
              t2[e] = fmaf(dz, hat, t2[e]);
            }
      });
      if (mine)
#pragma unroll
        for (int e = 0; e < W; ++e) {
          cols[first + e] = t1[e] * w[e];
          cols2[first + e] = t2[e] * w[e];
          acc[first + e] += t2[e];
          acc[step + first + e] += t1[e];
        }
      __syncthreads();
      block_group_sums<W, false>(a, cols, cols2, sums, threads, 0.f, 0);
    }
    if (!met) gn_cluster_wait();
    met = true;
    double2* got = recv + parity * a.ctas * a.groups;
    parity ^= 1;
    for (int i = tid; i < a.groups * a.ctas; i += blockDim.x) {
      const int p = i / a.groups, g = i - p * a.groups;
      st_peer2(got + rank * a.groups + g, p, sums[g]);
    }
    gn_cluster_arrive();
    gn_cluster_wait();
    for (int g = tid; g < a.groups; g += blockDim.x) {
      double s1 = 0.0, s2 = 0.0;
#pragma unroll 4
      for (int p = 0; p < a.ctas; ++p) {
        s1 += got[p * a.groups + g].x;
        s2 += got[p * a.groups + g].y;
      }
      float2 t;
      if (!BWD) {
        t = mean_rstd(s1, s2, inv_total, a.eps);
        if (rank == 0 && a.stats != nullptr)
          *reinterpret_cast<float2*>(a.stats + (static_cast<long long>(n) * a.groups + g) * 2) = t;
      } else {
        t = make_float2(static_cast<float>(s1 * inv_total), static_cast<float>(s2 * inv_total));
      }
      merged[g] = t;
    }
    __syncthreads();
    if (!BWD) {
      float m[W], rs[W], w[W], b[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float2 t = merged[gid(e)];
        m[e] = t.x;
        rs[e] = t.y;
        w[e] = a.w != nullptr ? a.w[col(e)] : 1.f;
        b[e] = a.b != nullptr ? a.b[col(e)] : 0.f;
      }
      walk(first, len, [&](auto live, int i) {
        Vec<W> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (live(u)) get_x(x[u], i + u * step, true);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (live(u)) {
#pragma unroll
            for (int e = 0; e < W; ++e)
              x[u].v[e] = act_fwd<ACT>(norm_z((x[u].v[e] - m[e]) * rs[e], w[e], b[e]));
            x[u].store_last(ys + i + u * step);
          }
      });
    } else {
      float m[W], rs[W], w[W], b[W], m1[W], m2[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        m[e] = st[gid(e) * 2];
        rs[e] = st[gid(e) * 2 + 1];
        w[e] = a.w != nullptr ? a.w[col(e)] : 1.f;
        b[e] = a.b != nullptr ? a.b[col(e)] : 0.f;
        m1[e] = merged[gid(e)].x;
        m2[e] = merged[gid(e)].y;
      }
      walk(first, len, [&](auto live, int i) {
        Vec<W> x[U], dy[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (live(u)) {
            get_x(x[u], i + u * step, true);
            get_dy(dy[u], i + u * step, true);
          }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (live(u)) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
              const float hat = (x[u].v[e] - m[e]) * rs[e];
              const float dz = act_bwd<ACT>(dy[u].v[e], norm_z(hat, w[e], b[e]));
              x[u].v[e] = rs[e] * fmaf(-hat, m2[e], fmaf(dz, w[e], -m1[e]));
            }
            x[u].store_last(ys + i + u * step);
          }
      });
    }
    // The sums are rewritten only behind the next image's barriers, which
    // every thread reaches after its last read of them.
  }
  if (!met) gn_cluster_wait();  // a cluster without an image still owes it
  if (BWD && a.partial != nullptr) {
    __syncthreads();
    float* out = a.partial + static_cast<long long>(blockIdx.x) * 2 * a.channels;
    for (int c = tid; c < a.channels; c += blockDim.x) {
      float s1 = 0.f, s2 = 0.f;
      for (int r = 0; r < a.reps; ++r) {
        s1 += acc[r * a.channels + c];
        s2 += acc[step + r * a.channels + c];
      }
      out[c] = s1;
      out[a.channels + c] = s2;
    }
  }
}

// --------------- few long images, and rows wider than a block has threads

struct GnWideArgs {
  GnArgs a;
  int32_t splits, rows;  // row ranges of an image, rows of one
  int32_t across, down;  // a block's threads over columns and rows
  float* part;           // [N][splits][2][C]
  float* group;          // [N][G][2]: backward's mean(d), mean(d * hat)
};

constexpr int kGnWideThreads = 256;
constexpr int kGnWideRows = 8;  // rows of a column held at once

// Per-column partials of one row range, W columns a thread, its block's
// threads taking the rows in turn. Forward: mean and sum of squares about it,
// blocks of 8 rows merged, then the threads'; backward: sums of dz and dz * hat.
// One column and every row a thread took twice as long (21 images of 5879 x
// 128, both directions: 232 us).
template <int W, int ACT, bool BWD>
__global__ void __launch_bounds__(kGnWideThreads)
    gn_wide_part_kernel(const __grid_constant__ GnWideArgs p) {
  __shared__ float sums[2][kGnWideThreads * W], counts[kGnWideThreads];
  pdl_trigger();
  pdl_wait();
  const GnArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid / p.across;
  const int c = (blockIdx.y * p.across + tid - lane * p.across) * W;
  const bool mine = lane < p.down && c < a.channels;
  const int split = blockIdx.x % p.splits;
  const int n = blockIdx.x / p.splits;
  const int r0 = split * p.rows;
  const int r1 = min(a.spatial, r0 + p.rows);
  const long long base = static_cast<long long>(n) * a.spatial * a.channels + c;
  float s1[W], s2[W], cnt = 0.f;
#pragma unroll
  for (int e = 0; e < W; ++e) s1[e] = s2[e] = 0.f;
  if (!BWD) {
    for (int r = r0 + lane; mine && r < r1; r += kGnWideRows * p.down) {
      Vec<W> v[kGnWideRows];
      const int k = min(kGnWideRows, (r1 - r + p.down - 1) / p.down);
#pragma unroll
      for (int i = 0; i < kGnWideRows; ++i)
        if (i < k) v[i].load(a.x + base + static_cast<long long>(r + i * p.down) * a.channels);
      const float inv = __fdividef(1.f, static_cast<float>(k)), all = cnt + k;
      const float share = __fdividef(static_cast<float>(k), all);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < kGnWideRows; ++i) s += i < k ? v[i].v[e] : 0.f;
        const float bm = s * inv;
#pragma unroll
        for (int i = 0; i < kGnWideRows; ++i)
          q = i < k ? fmaf(v[i].v[e] - bm, v[i].v[e] - bm, q) : q;
        const float d = bm - s1[e];
        s1[e] = fmaf(d, share, s1[e]);
        s2[e] += q + d * d * (cnt * share);
      }
      cnt = all;
    }
  } else if (mine) {
    float m[W], rs[W], w[W], b[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int g = fdiv(a.f_cg, c + e);
      const float* st = a.stats + (static_cast<long long>(n) * a.groups + g) * 2;
      m[e] = st[0];
      rs[e] = st[1];
      w[e] = a.w != nullptr ? a.w[c + e] : 1.f;
      b[e] = a.b != nullptr ? a.b[c + e] : 0.f;
    }
    constexpr int U = 4;
    for (int r = r0 + lane; r < r1; r += U * p.down) {
      Vec<W> x[U], dy[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (r + i * p.down < r1) {
          const long long o = base + static_cast<long long>(r + i * p.down) * a.channels;
          x[i].load(a.x + o);
          dy[i].load(a.dy + o);
        }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (r + i * p.down < r1)
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const float hat = (x[i].v[e] - m[e]) * rs[e];
            const float dz = act_bwd<ACT>(dy[i].v[e], norm_z(hat, w[e], b[e]));
            s1[e] += dz;
            s2[e] = fmaf(dz, hat, s2[e]);
          }
    }
  }
  // The block's threads of a column, halved until one is left.
#pragma unroll
  for (int e = 0; e < W; ++e) {
    sums[0][tid * W + e] = s1[e];
    sums[1][tid * W + e] = s2[e];
  }
  counts[tid] = cnt;
  for (int left = p.down; left > 1;) {
    const int half = (left + 1) / 2;
    __syncthreads();
    if (lane + half < left) {
      const int o = tid + half * p.across;
      const float n2 = counts[o], all = cnt + n2;
      const float share = !BWD && n2 > 0.f ? __fdividef(n2, all) : 0.f;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float x1 = sums[0][o * W + e], x2 = sums[1][o * W + e];
        if (BWD) {
          s1[e] += x1;
          s2[e] += x2;
        } else {
          const float d = x1 - s1[e];
          s1[e] = fmaf(d, share, s1[e]);
          s2[e] += x2 + d * d * (cnt * share);
        }
        sums[0][tid * W + e] = s1[e];
        sums[1][tid * W + e] = s2[e];
      }
      counts[tid] = cnt = all;
    }
    left = half;
  }
  if (lane == 0 && mine) {
    float* out = p.part + (static_cast<long long>(n) * p.splits + split) * 2 * a.channels + c;
#pragma unroll
    for (int e = 0; e < W; ++e) {
      out[e] = BWD ? s2[e] : s1[e];
      out[a.channels + e] = BWD ? s1[e] : s2[e];
    }
  }
}

// Sum of a value over a block of kGnWideThreads, the same for every thread.
__device__ __forceinline__ double gn_block_sum(double v, double* red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; i < kGnWideThreads / 32; ++i) t += red[i];
  return t;
}

// One block a (image, group): the columns' partials merged in 64 bits.
template <bool BWD>
__global__ void __launch_bounds__(kGnWideThreads)
    gn_wide_merge_kernel(const __grid_constant__ GnWideArgs p) {
  __shared__ double red[kGnWideThreads / 32];
  pdl_trigger();
  pdl_wait();
  const GnArgs& a = p.a;
  const long long id = blockIdx.x;
  const int n = static_cast<int>(id / a.groups), g = static_cast<int>(id % a.groups);
  const float* in = p.part + static_cast<long long>(n) * p.splits * 2 * a.channels + g * a.cg;
  const double total = static_cast<double>(a.spatial) * a.cg;
  double s1 = 0.0, s2 = 0.0;
  const int items = p.splits * a.cg;
#pragma unroll 8
  for (int i = threadIdx.x; i < items; i += kGnWideThreads) {
    const int split = fdiv(a.f_cg, i), c = i - split * a.cg;
    const float* q = in + static_cast<long long>(split) * 2 * a.channels;
    if (!BWD) {
      const int rows = min(a.spatial, (split + 1) * p.rows) - split * p.rows;
      s1 += static_cast<double>(q[c]) * rows;
    } else {
      const double w = a.w != nullptr ? a.w[g * a.cg + c] : 1.f;
      s1 += w * q[a.channels + c];
      s2 += w * q[c];
    }
  }
  s1 = gn_block_sum(s1, red);
  if (!BWD) {
    const double mean = s1 / total;
#pragma unroll 8
    for (int i = threadIdx.x; i < items; i += kGnWideThreads) {
      const int split = fdiv(a.f_cg, i), c = i - split * a.cg;
      const float* q = in + static_cast<long long>(split) * 2 * a.channels;
      const int rows = min(a.spatial, (split + 1) * p.rows) - split * p.rows;
      const double d = q[c] - mean;
      s2 += q[a.channels + c] + d * d * rows;
    }
    s2 = gn_block_sum(s2, red);
    if (threadIdx.x == 0) {
      a.stats[id * 2] = static_cast<float>(mean);
      a.stats[id * 2 + 1] = static_cast<float>(1.0 / sqrt(s2 / total + a.eps));
    }
  } else {
    s2 = gn_block_sum(s2, red);
    if (threadIdx.x == 0) {
      p.group[id * 2] = static_cast<float>(s1 / total);
      p.group[id * 2 + 1] = static_cast<float>(s2 / total);
    }
  }
}

// The output pass, laid out as the first.
template <int W, int ACT, bool BWD>
__global__ void __launch_bounds__(kGnWideThreads)
    gn_wide_apply_kernel(const __grid_constant__ GnWideArgs p) {
  pdl_trigger();
  pdl_wait();
  const GnArgs& a = p.a;
  const int lane = threadIdx.x / p.across;
  const int c = (blockIdx.y * p.across + threadIdx.x - lane * p.across) * W;
  if (lane >= p.down || c >= a.channels) return;
  const int split = blockIdx.x % p.splits;
  const int n = blockIdx.x / p.splits;
  const int r0 = split * p.rows;
  const int r1 = min(a.spatial, r0 + p.rows);
  float m[W], rs[W], w[W], b[W], m1[W], m2[W];
#pragma unroll
  for (int e = 0; e < W; ++e) {
    const long long id = static_cast<long long>(n) * a.groups + fdiv(a.f_cg, c + e);
    m[e] = a.stats[id * 2];
    rs[e] = a.stats[id * 2 + 1];
    w[e] = a.w != nullptr ? a.w[c + e] : 1.f;
    b[e] = a.b != nullptr ? a.b[c + e] : 0.f;
    m1[e] = BWD ? p.group[id * 2] : 0.f;
    m2[e] = BWD ? p.group[id * 2 + 1] : 0.f;
  }
  const long long base = static_cast<long long>(n) * a.spatial * a.channels + c;
  constexpr int U = 4;
  for (int r = r0 + lane; r < r1; r += U * p.down) {
    Vec<W> x[U], dy[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (r + i * p.down < r1) {
        const long long o = base + static_cast<long long>(r + i * p.down) * a.channels;
        x[i].load_last(a.x + o);
        if (BWD) dy[i].load_last(a.dy + o);
      }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (r + i * p.down < r1) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float hat = (x[i].v[e] - m[e]) * rs[e], z = norm_z(hat, w[e], b[e]);
          if (BWD)
            x[i].v[e] = rs[e] * fmaf(-hat, m2[e], fmaf(act_bwd<ACT>(dy[i].v[e], z), w[e], -m1[e]));
          else
            x[i].v[e] = act_fwd<ACT>(z);
        }
        x[i].store_last(a.y + base + static_cast<long long>(r + i * p.down) * a.channels);
      }
  }
}

// dw, db = column sums of `rows` partial rows in 64 bits: 32 columns and
// `per` rows a block, its warps taking the rows in turn; the last block of a
// column tile to finish adds the blocks' sums in their order (`counters` are
// zero before and after).
constexpr int kGnParamWarps = 16;
__global__ void __launch_bounds__(kGnParamWarps * 32)
    gn_param_kernel(const float* partial, int rows, int per, int channels, double* sums,
                    int* counters, float* dw, float* db, int acc_w, int acc_b) {
  pdl_trigger();
  pdl_wait();
  __shared__ double s[2][kGnParamWarps][32];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int r1 = min(rows, (static_cast<int>(blockIdx.y) + 1) * per);
  double t1 = 0.0, t2 = 0.0;
  if (c < channels) {
#pragma unroll 4
    for (int r = blockIdx.y * per + warp; r < r1; r += kGnParamWarps) {
      const float* in = partial + static_cast<long long>(r) * 2 * channels + c;
      t1 += in[0];
      t2 += in[channels];
    }
  }
  s[0][warp][lane] = t1;
  s[1][warp][lane] = t2;
  __syncthreads();
  double t = 0.0;
  if (warp < 2)
    for (int q = 0; q < kGnParamWarps; ++q) t += s[warp][q][lane];
  if (gridDim.y > 1) {
    const long long tiles = gridDim.x;
    if (warp < 2)
      sums[((static_cast<long long>(blockIdx.y) * tiles + blockIdx.x) * 2 + warp) * 32 + lane] = t;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      const unsigned prev =
          atomicAdd(reinterpret_cast<unsigned*>(counters) + blockIdx.x, 1u);
      s_last = prev == gridDim.y - 1;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    t = 0.0;
    if (warp < 2)
      for (unsigned q = 0; q < gridDim.y; ++q)
        t += __ldcg(sums + ((q * tiles + blockIdx.x) * 2 + warp) * 32 + lane);
    if (threadIdx.x == 0) counters[blockIdx.x] = 0;
  }
  if (warp < 2 && c < channels) {
    float* out = warp == 0 ? dw : db;
    const int acc = warp == 0 ? acc_w : acc_b;
    if (out != nullptr) {
      const float v = static_cast<float>(t);
      out[c] = acc ? out[c] + v : v;
    }
  }
}

// ------------------------------------------------------------------ host

static bool gn_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

enum class GnPath { kRow, kWarp, kBlock, kCluster, kWide };

struct GnPlan {
  GnPath path;
  int vec;             // 4 or 1 floats a slot
  int regs;            // slots a lane or thread
  bool by_element;     // warp: quads that straddle groups
  bool staged;         // cluster: rows in shared memory
  int threads, reps, ctas, rows_per, lpg;
  int smem;
  int blocks;          // grid
  int splits, rows;    // wide: row ranges of an image, rows of one
  int partial_rows;    // backward's partial sums
};

constexpr int kGnSms = 148;
constexpr int kGnStageMax = 44 * 1024;
constexpr int kGnSmemMax = 112 * 1024;  // two CTAs an SM
// The way an image stays on chip; see the head of this file. `vec` is the
// widest access the caller's pointers allow.
static GnPlan pick_plan(long long images, int spatial, int channels, int groups, int vec,
                        bool bwd) {
  GnPlan p;
  std::memset(&p, 0, sizeof(p));
  const int cg = channels / groups;
  const long long len = static_cast<long long>(spatial) * channels;
  // One warp: up to 8 quads a lane, or 8 floats where quads do not fit the
  // image or the pointers.
  const int w = vec == 4 && len % 4 == 0 ? 4 : 1;
  if (spatial == 1 && w == 4 && len <= 32 * 8 * 4 && cg % 4 == 0 && (cg & (cg - 1)) == 0) {
    p.path = GnPath::kRow;
    p.vec = 4;
    const int need = static_cast<int>((len / 4 + 31) / 32);
    p.regs = need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : 8;
    p.smem = bwd ? kGnWarps * channels * 4 : 0;
    p.threads = kGnWarps * 32;
    const long long want = (images + kGnWarps - 1) / kGnWarps;
    const long long most = kGnSms * (p.regs == 8 ? 1 : bwd ? 2 : 3);
    p.blocks = static_cast<int>(std::min(want, most));
    p.partial_rows = p.blocks;
    return p;
  }
  if (len <= (w == 4 ? 32 * 8 * 4 : 32 * 8)) {
    p.path = GnPath::kWarp;
    p.vec = w;
    p.by_element = w == 4 && cg % 4 != 0;
    const int need = static_cast<int>((len / w + 31) / 32);
    p.regs = w == 1 ? 8 : need <= 2 ? 2 : need <= 4 ? 4 : 8;
    int pow2 = 1;
    while (pow2 < groups) pow2 *= 2;
    p.lpg = pow2 >= 32 ? 1 : 32 / pow2;
    const int gpad = (groups + 3) & ~3;
    const int per_warp = p.regs * 32 * (p.by_element ? 4 : 1) + 2 * gpad;
    p.smem = std::max(kGnWarps * per_warp, p.regs * 32 * w) * 4;
    p.threads = kGnWarps * 32;
    const long long want = (images + kGnWarps - 1) / kGnWarps;
    const long long most = kGnSms * (bwd ? 4 : 8);
    p.blocks = static_cast<int>(std::min(want, most));
    p.partial_rows = p.blocks;
    if (p.smem <= 48 * 1024) return p;
  }
  // Blocks: a period must hold whole rows.
  const int odd = channels % 4 == 0 ? 1 : channels % 2 == 0 ? 2 : 4;  // rows to a whole quad
  const int q = w == 4 ? channels * odd / 4 : channels;  // threads to a whole row (or rows)
  // 8 slots a thread of 256: an SM holds several blocks, and one's loads hide
  // behind another's sums.
  const int top = q <= 256 ? 256 / q * q : q <= 512 ? q : 0;
  const long long slots = len / w;
  const bool whole = slots <= static_cast<long long>(top) * 8;
  // CTAs of a cluster. Forward: as few as bring a CTA's rows to 44 KB (four
  // CTAs an SM), which are then staged. Backward, and forward where 16 do not:
  // 8 slots a thread at least, and not staged (x and dy leave room for two CTAs
  // an SM only: the backward of 512 x 42 x 42 x 96 takes 450 us staged, 340
  // not).
  const long long row_bytes = static_cast<long long>(channels) * 4;
  auto share = [&](int n) {
    const int rows = ((spatial + n - 1) / n + odd - 1) / odd * odd;
    return rows * row_bytes;
  };
  int ctas = 2;
  while (ctas < kGnMaxCluster && share(ctas) > kGnStageMax) ctas *= 2;
  const bool staged = !bwd && share(ctas) <= kGnStageMax;
  if (!staged) {
    ctas = 8;
    while (ctas > 2 && slots < static_cast<long long>(top) * 8 * ctas) ctas /= 2;
  }
  // Fewer images than fill half the SMs' places: the passes over global
  // memory use them all. Backward, where a cluster reads its image from L2 a
  // second time anyway, they win for as long as x and dy fit it in part, and
  // have work enough to outweigh two launches more (us, clusters and passes:
  // 100 images of 441 x 128: 32, 37; 40 of 1764 x 96: 43, 39; 94 of 957 x 132:
  // 68, 56; 300 of 441 x 128: 80, 75; 256 of 1764 x 96: 177, 171).
  const long long floats = images * len;
  const bool few = images * ctas < kGnSms * 2 ||
                   (bwd && channels % 4 == 0 && channels >= 32 && floats >= (6ll << 20) &&
                    floats <= (48ll << 20));
  if (top > 0 && (whole || !few)) {
    int threads = top;
    p.vec = w;
    if (whole) {
      // Many images: 8 slots a thread, the most of an SM's registers in
      // flight. Few: 4, for a shorter walk.
      p.path = GnPath::kBlock;
      p.regs = images <= 2 * kGnSms && slots <= static_cast<long long>(top) * 4 ? 4 : 8;
      threads = static_cast<int>((slots + p.regs - 1) / p.regs + q - 1) / q * q;
      // Blocks that are resident together, at the kernel's 128 registers a
      // thread, walk over the images.
      const long long cap = kGnSms * std::max(1, 512 / ((threads + 31) / 32 * 32));
      p.blocks = static_cast<int>(std::min<long long>(images, cap));
      p.smem = (2 * threads * w + 6 * groups) * 4;
    } else {
      p.path = GnPath::kCluster;
      p.ctas = ctas;
      p.staged = staged;
      p.rows_per = static_cast<int>(share(ctas) / row_bytes);
      p.smem = ((bwd ? 4 : 2) * threads * w + 6 * groups + 8 * ctas * groups) * 4;
      if (staged) p.smem += static_cast<int>(share(ctas)) + 16;
      const long long most = kGnSms * (threads > 256 ? 2 : 4) / ctas;
      p.blocks = static_cast<int>(std::min<long long>(images, most)) * ctas;
    }
    p.partial_rows = p.blocks;
    p.threads = (threads + 31) / 32 * 32;
    p.reps = threads * w / channels;
    int lpg = 32;
    while (lpg > 1 && static_cast<long long>(lpg) * groups > p.threads) lpg /= 2;
    p.lpg = lpg;
    if (p.smem <= (p.path == GnPath::kCluster ? kGnSmemMax : 48 * 1024)) return p;
  }
  p.path = GnPath::kWide;
  p.vec = vec == 4 && channels % 4 == 0 ? 4 : 1;
  p.threads = std::min(kGnWideThreads, channels / p.vec);  // across the columns
  const int col_blocks = (channels / p.vec + p.threads - 1) / p.threads;
  const long long want = std::max(1ll, kGnSms * 8 / (images * col_blocks));
  long long splits = std::min<long long>(want, (spatial + 31) / 32);
  splits = std::max(1ll, splits);
  p.rows = static_cast<int>((spatial + splits - 1) / splits);
  p.splits = (spatial + p.rows - 1) / p.rows;
  p.partial_rows = static_cast<int>(images * p.splits);
  return p;
}

// Row splits of the weight gradients' column sums.
static int gn_param_splits(int rows, int channels) {
  if ((channels + 31) / 32 > static_cast<int>(kCounterBytes / sizeof(int))) return 1;
  return std::max(1, std::min(rows / 64, 64));
}

// The workspace behind the counters: the partial rows (both directions of
// the wide path, the backward of the others), the wide path's group means,
// the column sums of the weight gradients' row splits (at an even float).
struct GnWs {
  size_t group, sums, bytes;  // offsets in floats; total in bytes
};
static GnWs gn_ws(const GnPlan& p, long long images, int channels, int groups, bool bwd) {
  GnWs w;
  size_t n = 0;
  if (bwd || p.path == GnPath::kWide) n += static_cast<size_t>(p.partial_rows) * 2 * channels;
  w.group = n;
  if (p.path == GnPath::kWide) n += static_cast<size_t>(images) * groups * 2;
  n = (n + 1) & ~static_cast<size_t>(1);
  w.sums = n;
  if (bwd)
    n += static_cast<size_t>(gn_param_splits(p.partial_rows, channels)) *
         ((channels + 31) / 32 * 32) * 2 * 2;
  w.bytes = n * sizeof(float);
  return w;
}

// The passes over global memory have a grid row for every 256 channels or quads.
constexpr int kGnMaxChannels = 65535 * kGnWideThreads;

static bool gn_shape_ok(int images, int spatial, int channels, int groups) {
  if (images <= 0 || spatial <= 0 || channels <= 0 || groups <= 0) return false;
  if (channels % groups != 0 || channels > kGnMaxChannels) return false;
  // Counts of rows and images step past their ends by less than 2^16.
  constexpr long long kMost = (1ll << 31) - (1ll << 16);
  return static_cast<long long>(spatial) * channels < kMost &&
         static_cast<long long>(images) * groups < kMost;
}

// The workspace is sized for either access width.
size_t group_norm_ws(int images, int spatial, int channels, int groups, int backward) {
  if (!gn_shape_ok(images, spatial, channels, groups)) return 0;
  size_t most = 0;
  for (int vec : {1, 4})
    most = std::max(most, gn_ws(pick_plan(images, spatial, channels, groups, vec, backward != 0),
                                images, channels, groups, backward != 0)
                              .bytes);
  return kCounterBytes + most;
}

template <int W, int R, int ACT, bool BWD>
static cudaError_t launch_block(const GnPlan& p, const GnArgs& a, cudaStream_t st) {
  return launch_pdl(gn_block_kernel<W, R, ACT, BWD>, dim3(p.blocks), dim3(p.threads), p.smem, st,
                    a);
}

template <int W, int ACT, bool BWD, bool STAGED>
static cudaError_t launch_cluster(const GnPlan& p, const GnArgs& a, int* partial_rows,
                                  cudaStream_t st) {
  // Clusters that are resident at once: fewer than the SM count says where
  // they do not pack into the GPCs. Asked once per device for each cluster
  // size, and number of CTAs an SM by their shared memory and threads: how an
  // image falls to a cluster depends on the call's shape only.
  static std::mutex lock;
  static bool ready[64] = {};
  static int known[64][kGnMaxCluster + 1][2][2] = {};
  const auto kernel = gn_cluster_kernel<W, ACT, BWD, STAGED>;
  const bool wide = p.smem > 56 * 1024, many = p.threads > 256;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.ctas);
  cfg.blockDim = dim3(many ? 512 : 256);
  cfg.dynamicSmemBytes = wide ? kGnSmemMax : 56 * 1024;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  int most = 0;
  {
    std::lock_guard<std::mutex> hold(lock);
    if (!ready[dev]) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGnSmemMax);
      if (e == cudaSuccess)  // clusters above the portable 8
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return e;
      ready[dev] = true;
    }
    most = known[dev][p.ctas][wide][many];
    if (most == 0) {
      e = cudaOccupancyMaxActiveClusters(&most, kernel, &cfg);
      if (e != cudaSuccess) return e;
      if (most < 1) most = 1;
      known[dev][p.ctas][wide][many] = most;
    }
  }
  // As many images for each cluster: one more round for a few of them would
  // leave the others idle.
  int clusters = std::min(most, p.blocks / p.ctas);
  const int walk = (a.images + clusters - 1) / clusters;
  clusters = (a.images + walk - 1) / walk;
  *partial_rows = clusters * p.ctas;
  cfg.gridDim = dim3(clusters * p.ctas);
  cfg.blockDim = dim3(p.threads);
  cfg.dynamicSmemBytes = p.smem;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int W, int R, int ACT, bool BWD, bool EL>
static cudaError_t launch_warp(const GnPlan& p, const GnArgs& a, cudaStream_t st) {
  return launch_pdl(gn_warp_kernel<W, R, ACT, BWD, EL>, dim3(p.blocks), dim3(p.threads), p.smem,
                    st, a);
}

template <int ACT, bool BWD>
static cudaError_t launch_act(const GnPlan& p, const GnArgs& a, float* ws,
                              int* partial_rows, cudaStream_t st) {
  if (p.path == GnPath::kRow) {
    note_launch();
    const auto kernel = p.regs == 1   ? gn_row_kernel<1, ACT, BWD>
                        : p.regs == 2 ? gn_row_kernel<2, ACT, BWD>
                        : p.regs == 4 ? gn_row_kernel<4, ACT, BWD>
                                      : gn_row_kernel<8, ACT, BWD>;
    return launch_pdl(kernel, dim3(p.blocks), dim3(p.threads), p.smem, st, a);
  }
  if (p.path == GnPath::kWarp) {
    note_launch();
    if (p.vec == 1) return launch_warp<1, 8, ACT, BWD, true>(p, a, st);
    if (p.by_element) {
      switch (p.regs) {
        case 2: return launch_warp<4, 2, ACT, BWD, true>(p, a, st);
        case 4: return launch_warp<4, 4, ACT, BWD, true>(p, a, st);
        default: return launch_warp<4, 8, ACT, BWD, true>(p, a, st);
      }
    }
    switch (p.regs) {
      case 2: return launch_warp<4, 2, ACT, BWD, false>(p, a, st);
      case 4: return launch_warp<4, 4, ACT, BWD, false>(p, a, st);
      default: return launch_warp<4, 8, ACT, BWD, false>(p, a, st);
    }
  }
  if (p.path == GnPath::kBlock) {
    note_launch();
    if (p.vec == 1)
      return p.regs == 4 ? launch_block<1, 4, ACT, BWD>(p, a, st)
                         : launch_block<1, 8, ACT, BWD>(p, a, st);
    return p.regs == 4 ? launch_block<4, 4, ACT, BWD>(p, a, st)
                       : launch_block<4, 8, ACT, BWD>(p, a, st);
  }
  if (p.path == GnPath::kCluster) {
    note_launch();
    if constexpr (!BWD)
      if (p.staged)
        return p.vec == 1 ? launch_cluster<1, ACT, false, true>(p, a, partial_rows, st)
                          : launch_cluster<4, ACT, false, true>(p, a, partial_rows, st);
    return p.vec == 1 ? launch_cluster<1, ACT, BWD, false>(p, a, partial_rows, st)
                      : launch_cluster<4, ACT, BWD, false>(p, a, partial_rows, st);
  }
  GnWideArgs l;
  std::memset(&l, 0, sizeof(l));
  l.a = a;
  l.splits = p.splits;
  l.rows = p.rows;
  l.part = ws;
  l.group = ws + gn_ws(p, a.images, a.channels, a.groups, BWD).group;
  if (a.stats == nullptr) l.a.stats = l.group;  // forward without saved statistics
  l.across = p.threads;
  l.down = kGnWideThreads / p.threads;
  const dim3 grid(static_cast<unsigned>(a.images) * p.splits,
                  (a.channels / p.vec + p.threads - 1) / p.threads);
  const unsigned merge = static_cast<unsigned>(a.images) * static_cast<unsigned>(a.groups);
  cudaError_t e = launch_pdl(p.vec == 4 ? gn_wide_part_kernel<4, ACT, BWD>
                                         : gn_wide_part_kernel<1, ACT, BWD>,
                             grid, dim3(kGnWideThreads), 0, st, l);
  note_launch();
  if (e != cudaSuccess) return e;
  e = launch_pdl(gn_wide_merge_kernel<BWD>, dim3(merge), dim3(kGnWideThreads), 0, st, l);
  note_launch();
  if (e != cudaSuccess) return e;
  note_launch();
  return launch_pdl(p.vec == 4 ? gn_wide_apply_kernel<4, ACT, BWD>
                                : gn_wide_apply_kernel<1, ACT, BWD>,
                    grid, dim3(kGnWideThreads), 0, st, l);
}

template <bool BWD>
static cudaError_t launch_any(const GnPlan& p, const GnArgs& a, float* ws,
                              int* partial_rows, cudaStream_t st) {
  switch (a.act) {
    case TTRL_ACT_RELU: return launch_act<TTRL_ACT_RELU, BWD>(p, a, ws, partial_rows, st);
    case TTRL_ACT_SILU: return launch_act<TTRL_ACT_SILU, BWD>(p, a, ws, partial_rows, st);
    default: return launch_act<TTRL_ACT_NONE, BWD>(p, a, ws, partial_rows, st);
  }
}

static int gn_check(const char* what, int images, int spatial, int channels, int groups,
                    int act) {
  if (images < 0 || spatial <= 0 || channels <= 0 || groups <= 0)
    return set_error(TTRL_EINVAL, "%s: bad extents (images %d, spatial %d, channels %d, groups %d)",
                     what, images, spatial, channels, groups);
  if (channels % groups != 0)
    return set_error(TTRL_EINVAL, "%s: %d channels do not divide into %d groups", what, channels,
                     groups);
  if (act != TTRL_ACT_NONE && act != TTRL_ACT_RELU && act != TTRL_ACT_SILU)
    return set_error(TTRL_EINVAL, "%s: unknown activation %d", what, act);
  if (channels > kGnMaxChannels)
    return set_error(TTRL_EUNSUPPORTED, "%s: %d channels, up to %d are served", what, channels,
                     kGnMaxChannels);
  if (images > 0 && !gn_shape_ok(images, spatial, channels, groups))
    return set_error(TTRL_EUNSUPPORTED, "%s: an image of more than 2^31 - 2^16 elements, or as many groups in all",
                     what);
  return TTRL_OK;
}

static GnArgs gn_args(const GnPlan& p, int images, int spatial, int channels, int groups,
                      int act) {
  GnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.images = images;
  a.spatial = spatial;
  a.channels = channels;
  a.groups = groups;
  a.cg = channels / groups;
  a.act = act;
  a.lpg = p.lpg;
  a.reps = p.reps;
  a.ctas = p.ctas;
  a.rows_per = p.rows_per;
  a.f_c = make_fastdiv(channels);
  a.f_cg = make_fastdiv(a.cg);
  return a;
}

// The workspace of a call: kCounterBytes of counters (zero before and after,
// as for every user of the shared workspace), then the partial sums.
static int gn_workspace(const char* what, const GnPlan& p, const GnArgs& a, bool bwd, void* ws,
                        size_t ws_bytes, float** out) {
  const size_t need = gn_ws(p, a.images, a.channels, a.groups, bwd).bytes;
  *out = nullptr;
  if (need == 0) return TTRL_OK;
  if (reinterpret_cast<uintptr_t>(ws) & 15u)
    return set_error(TTRL_EINVAL, "%s: the workspace has to start on a 16-byte boundary", what);
  if (ws == nullptr || ws_bytes < need + kCounterBytes)
    return set_error(TTRL_EWORKSPACE, "%s: needs %zu bytes of workspace, got %zu", what,
                     need + kCounterBytes, ws == nullptr ? static_cast<size_t>(0) : ws_bytes);
  *out = reinterpret_cast<float*>(static_cast<char*>(ws) + kCounterBytes);
  return TTRL_OK;
}

int group_norm_fwd(const float* x, const float* w, const float* b, float* y, float* stats,
                   int images, int spatial, int channels, int groups, float eps, int act,
                   void* ws, size_t ws_bytes, cudaStream_t st) {
  int rc = gn_check("group_norm_fwd", images, spatial, channels, groups, act);
  if (rc) return rc;
  if (!(eps > 0.f)) return set_error(TTRL_EINVAL, "group_norm_fwd: eps has to be positive");
  if (images == 0) return TTRL_OK;
  if (x == nullptr || y == nullptr)
    return set_error(TTRL_EINVAL, "group_norm_fwd: null pointer");
  if (reinterpret_cast<uintptr_t>(stats) & 7u)
    return set_error(TTRL_EINVAL, "group_norm_fwd: stats have to start on an 8-byte boundary");
  const int vec = gn_aligned16(x) && gn_aligned16(y) && gn_aligned16(w) && gn_aligned16(b) ? 4 : 1;
  const GnPlan p = pick_plan(images, spatial, channels, groups, vec, false);
  GnArgs a = gn_args(p, images, spatial, channels, groups, act);
  a.x = x;
  a.w = w;
  a.b = b;
  a.y = y;
  a.stats = stats;
  a.eps = eps;
  float* fws = nullptr;
  if ((rc = gn_workspace("group_norm_fwd", p, a, false, ws, ws_bytes, &fws))) return rc;
  const int64_t all = static_cast<int64_t>(images) * spatial * channels;
  const Span in[] = {{"x", x == y ? nullptr : x, all}, {"weight", w, channels}, {"bias", b, channels}};
  const Span made[] = {{"y", y, all}, {"stats", stats, static_cast<int64_t>(images) * groups * 2}};
  if ((rc = spans_apart("group_norm_fwd", in, made))) return rc;
  int rows = p.partial_rows;
  const cudaError_t e = launch_any<false>(p, a, fws, &rows, st);
  return e == cudaSuccess ? TTRL_OK : set_cuda_error("group_norm_fwd launch", e);
}

int group_norm_bwd(const float* dy, const float* x, const float* w, const float* b,
                   const float* stats, float* dx, float* dw, float* db, int images, int spatial,
                   int channels, int groups, int act, int acc_w, int acc_b, void* ws,
                   size_t ws_bytes, cudaStream_t st) {
  int rc = gn_check("group_norm_bwd", images, spatial, channels, groups, act);
  if (rc) return rc;
  const bool params = dw != nullptr || db != nullptr;
  if (images == 0) {
    // No rows: the weight gradients are zero (or keep what they hold).
    if (!params) return TTRL_OK;
    note_launch();
    const cudaError_t e0 = launch_pdl(
        gn_param_kernel, dim3((channels + 31) / 32), dim3(kGnParamWarps * 32), 0, st,
        static_cast<const float*>(nullptr), 0, 1, channels, static_cast<double*>(nullptr),
        static_cast<int*>(nullptr), dw, db, acc_w, acc_b);
    return e0 == cudaSuccess ? TTRL_OK : set_cuda_error("group_norm_bwd launch", e0);
  }
  if (dy == nullptr || x == nullptr || stats == nullptr || dx == nullptr)
    return set_error(TTRL_EINVAL, "group_norm_bwd: null pointer");
  if (reinterpret_cast<uintptr_t>(stats) & 7u)
    return set_error(TTRL_EINVAL, "group_norm_bwd: stats have to start on an 8-byte boundary");
  const int vec = gn_aligned16(x) && gn_aligned16(dy) && gn_aligned16(dx) && gn_aligned16(w) &&
                          gn_aligned16(b)
                      ? 4
                      : 1;
  const GnPlan p = pick_plan(images, spatial, channels, groups, vec, true);
  GnArgs a = gn_args(p, images, spatial, channels, groups, act);
  a.x = x;
  a.dy = dy;
  a.w = w;
  a.b = b;
  a.y = dx;
  a.stats = const_cast<float*>(stats);
  float* fws = nullptr;
  if ((rc = gn_workspace("group_norm_bwd", p, a, true, ws, ws_bytes, &fws))) return rc;
  const int64_t all = static_cast<int64_t>(images) * spatial * channels;
  const Span in[] = {{"x", x, all},
                     {"dy", dy == dx ? nullptr : dy, all},
                     {"weight", w, channels},
                     {"bias", b, channels},
                     {"stats", stats, static_cast<int64_t>(images) * groups * 2}};
  const Span made[] = {{"dx", dx, all}, {"dweight", dw, channels}, {"dbias", db, channels}};
  if ((rc = spans_apart("group_norm_bwd", in, made))) return rc;
  a.partial = params ? fws : nullptr;
  int rows = p.partial_rows;
  cudaError_t e = launch_any<true>(p, a, fws, &rows, st);
  if (e == cudaSuccess && params) {
    note_launch();
    const int splits = gn_param_splits(rows, channels);
    const int per = (rows + splits - 1) / splits;
    e = launch_pdl(gn_param_kernel, dim3((channels + 31) / 32, splits), dim3(kGnParamWarps * 32),
                   0, st, static_cast<const float*>(fws), rows, per, channels,
                   reinterpret_cast<double*>(fws + gn_ws(p, images, channels, groups, true).sums),
                   static_cast<int*>(ws), dw, db, acc_w, acc_b);
  }
  return e == cudaSuccess ? TTRL_OK : set_cuda_error("group_norm_bwd launch", e);
}

}  // namespace ttrl

using namespace ttrl;

extern "C" {

size_t ttrl_group_norm_workspace_bytes(int images, int spatial, int channels, int groups,
                                       int backward) {
  return group_norm_ws(images, spatial, channels, groups, backward);
}

int ttrl_group_norm_fwd(const float* x, const float* weight, const float* bias, float* y,
                        float* stats, int images, int spatial, int channels, int groups, float eps,
                        int act, void* workspace, size_t workspace_bytes,
                        ttrl_stream_t stream) {
  return group_norm_fwd(x, weight, bias, y, stats, images, spatial, channels, groups, eps, act,
                        workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int ttrl_group_norm_bwd(const float* dy, const float* x, const float* weight, const float* bias,
                        const float* stats, float* dx, float* dweight, float* dbias, int images,
                        int spatial, int channels, int groups, int act, int accumulate_weight,
                        int accumulate_bias, void* workspace, size_t workspace_bytes,
                        ttrl_stream_t stream) {
  return group_norm_bwd(dy, x, weight, bias, stats, dx, dweight, dbias, images, spatial, channels,
                        groups, act, accumulate_weight, accumulate_bias, workspace,
                        workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
