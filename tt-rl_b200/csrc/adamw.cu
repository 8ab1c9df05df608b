// AdamW (decoupled weight decay) over many tensors in one launch, with the
// moments held in 32 bits or in 8.
//
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit moments are kept in blocks of 256 elements that share a 32-bit scale,
// the block's largest magnitude:
//   m = scale * sign(c) * (c / 127)^2,  c in [-127, 127];
//   v = scale * (c / 255)^4,            c in [0, 255], at least 1 where v > 0.
// A uniform code would hold the many small entries beside a large one as
// zero; the square (of sqrt(v) too, which is what the step divides by)
// spaces the codes by the square root of the value. A positive v never
// becomes zero, so m / sqrt(v) cannot blow up. The step itself uses the
// unrounded new moments; only what is kept is rounded, to the nearest code.
// A value that is not finite makes its block's scale, and so the block's
// moments, NaN from then on.
//
// Bound by memory: 28 bytes an element in 32 bits, 16 and 16 a block in 8.
// The unit of work is a block of 256 elements, one warp's: 8 elements a lane
// as two groups of four, so every load of an fp32 array is 16 bytes a lane
// and all of them (8, or 4 and 4 short ones) are in flight together. A thread
// block takes an equal, contiguous run of units, and its warps walk it side
// by side; the tensors' pointers are launch parameters, so a captured launch
// needs no table in memory that could change under it.
//
// Times on B200, shares of the measured copy rate in brackets: 64M elements 326
// us (89%) in 32 bits, 239 us (70%) in 8, where the arithmetic of the codes
// takes about as long as the memory; 320 tensors of 24M in all 129 us (81%);
// 2.3M in 16 tensors 14 us. 100M 8-bit moments read back as floats: 207 us
// (76%).
#include <cstring>

#include "common.cuh"
#include "internal.h"

namespace ttrl {

constexpr int kAwThreads = 256;
constexpr int kAwWarps = kAwThreads / 32;
constexpr int kAwBlock = TTRL_ADAMW_BLOCK;
constexpr int kAwFew = 24;  // tensors of the launch with the short parameter block
constexpr int kAwBlocksPerSM = 4;

template <int MAX>
struct AdamwArgs {
  ttrl_adamw_tensor t[MAX];
  int32_t start[MAX + 1];  // first unit of each tensor
  uint8_t vec[MAX];        // its fp32 buffers are 16-byte aligned
  uint8_t lead[MAX];       // the first tensor of the call with its counter
  int32_t count;
  int32_t* steps;
  int32_t* ticket;
  const float* grad_scale;
  const double* lr_device;
  const double* bias;  // [bias_steps][2]: (1 - b1^t, sqrt((1 - b2) / (1 - b2^t)))
  long long bias_steps;
  double lr, b1, b2, eps, wd;
};
static_assert(sizeof(AdamwArgs<TTRL_ADAMW_MAX_TENSORS>) <= 32764, "launch parameter limit");

struct AdamwScalars {
  float decay, rate, rc2;  // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

// Byte e of a word of codes as a float, and a rounded float's low byte: by
// the bits of 2^23 + n, as the conversion instructions run at an eighth of the
// rate of an addition and there would be four an element.
__device__ __forceinline__ float m_float(uint32_t w, int e) {  // int8
  return __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7440 | e)) -
         (8388608.f + 128.f);
}
__device__ __forceinline__ float v_float(uint32_t w, int e) {  // uint8
  return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | e)) - 8388608.f;
}
// fp32 value of a first-moment code, and of a second-moment code, as a share
// of the block's scale.
__device__ __forceinline__ float m_share(float c) {
  const float r = __fmul_rn(c, 1.0f / 127.0f);
  return __fmul_rn(r, fabsf(r));
}
__device__ __forceinline__ float v_share(float c) {
  float r = __fmul_rn(c, 1.0f / 255.0f);
  r = __fmul_rn(r, r);
  return __fmul_rn(r, r);
}
__device__ __forceinline__ float sqrt_fast(float x) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The code of a value before rounding: of a block whose scale is `scale` (> 0,
// or 0 where all its values are), with inv = 1 / scale. EXACT: the rounded
// quotient, roots and product of IEEE arithmetic, which define the code, so
// that it does not depend on a device's approximations. They cost five
// sequences of a dozen instructions an element; the approximate ones are each
// within one unit in the last place (2^-23), in all within kNear of r, and
// decide where that leaves no doubt (see codes_of).
constexpr float kNear = 5e-7f;
template <bool EXACT>
__device__ __forceinline__ float m_root(float x, float scale, float inv) {
  if (EXACT)
    return copysignf(
        __fmul_rn(__fsqrt_rn(__fdiv_rn(fabsf(x), scale > 0.f ? scale : 1.f)), 127.f), x);
  return copysignf(sqrt_fast(fabsf(x) * inv) * 127.f, x);
}
template <bool EXACT>
__device__ __forceinline__ float v_root(float x, float scale, float inv) {
  const float r =
      EXACT ? __fmul_rn(__fsqrt_rn(__fsqrt_rn(__fdiv_rn(x, scale > 0.f ? scale : 1.f))), 255.f)
            : sqrt_fast(sqrt_fast(x * inv)) * 255.f;
  return x > 0.f ? fmaxf(r, 1.f) : r;
}

// Four values' codes as bytes of a word; `doubt` is set where one lies too
// near the middle of two codes, or is not finite, for the approximations.
template <bool EXACT, bool FIRST>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float scale, float inv,
                                             bool& doubt) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float r = FIRST ? m_root<EXACT>(x[e], scale, inv) : v_root<EXACT>(x[e], scale, inv);
    const float t = r + 12582912.f;  // 1.5 * 2^23: rounds to the nearest integer, ties to even
    w[e] = __float_as_uint(t);
    if (!EXACT) doubt |= !(fabsf(r - (t - 12582912.f)) <= fmaf(-kNear, fabsf(r), 0.5f));
    if (EXACT && !(fabsf(r) <= 255.f)) w[e] = 0;  // NaN: the scale says so too
  }
  return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}

// Largest magnitude over a warp, by the bits: a NaN's are the largest. NaN
// where it is infinite, as no code could hold the block's other values.
__device__ __forceinline__ float warp_abs_max(float v) {
  const uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu);
  return __uint_as_float(b == 0x7f800000u ? 0x7fffffffu : b);
}
__device__ __forceinline__ float abs_max(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}

// Four consecutive elements from i of an array that ends at `end`.
__device__ __forceinline__ void get4(const float* p, long long i, long long end, bool vec,
                                     float (&v)[4]) {
  if (vec && i + 3 < end) {
    const float4 t = *reinterpret_cast<const float4*>(p + i);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = i + e < end ? p[i + e] : 0.f;
}
__device__ __forceinline__ void put4(float* p, long long i, long long end, bool vec,
                                     const float (&v)[4]) {
  if (vec && i + 3 < end) {
    *reinterpret_cast<float4*>(p + i) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (i + e < end) p[i + e] = v[e];
}

// The codes of a lane's two groups of four, stored; code arrays are padded to
// whole blocks, so a word never leaves them.
__device__ __forceinline__ void put_codes(uint8_t* m8, uint8_t* v8, const float (&m)[2][4],
                                          const float (&v)[2][4], float mm, float vm) {
  // A scale too small to invert gives infinities, and those are in doubt; one
  // above 2^126 gives zero, by the fast quotient's definition, and so is that.
  const float minv = mm > 0.f ? __fdividef(1.f, mm) : 0.f;
  const float vinv = vm > 0.f ? __fdividef(1.f, vm) : 0.f;
  bool doubt = fmaxf(mm, vm) > 0x1p126f;
  uint32_t mc[2], vc[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    mc[h] = codes_of<false, true>(m[h], mm, minv, doubt);
    vc[h] = codes_of<false, false>(v[h], vm, vinv, doubt);
  }
  if (doubt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mc[h] = codes_of<true, true>(m[h], mm, minv, doubt);
      vc[h] = codes_of<true, false>(v[h], vm, vinv, doubt);
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    *reinterpret_cast<uint32_t*>(m8 + h * 128) = mc[h];
    *reinterpret_cast<uint32_t*>(v8 + h * 128) = vc[h];
  }
}

template <int MAX>
__global__ void __launch_bounds__(kAwThreads, kAwBlocksPerSM)
    adamw_kernel(const __grid_constant__ AdamwArgs<MAX> a) {
  __shared__ AdamwScalars ks[MAX];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // This block's run of units.
  const int units = a.start[a.count];
  const long long b0 = blockIdx.x, nb = gridDim.x;
  const int u0 = static_cast<int>(b0 * units / nb);
  const int u1 = static_cast<int>((b0 + 1) * units / nb);
  // The tensor of a unit: the last one that starts at or before it.
  auto tensor_of = [&](int u) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.start[mid] <= u)
        lo = mid;
      else
        hi = mid - 1;
    }
    return lo;
  };
  const int t0 = tensor_of(u0), t1 = tensor_of(u1 - 1);
  // The step's scalars in 64 bits, one thread a tensor of the run.
  for (int q = t0 + threadIdx.x; q <= t1; q += kAwThreads) {
    const double lr = a.lr_device != nullptr ? *a.lr_device : a.lr;
    const int step = a.steps[a.t[q].step_index] + 1;
    double bc1, bc2;
    if (a.bias != nullptr) {
      // Host-computed terms; the last row serves every later step.
      const long long t = step < a.bias_steps ? step : a.bias_steps;
      bc1 = a.bias[2 * (t - 1)];
      const double c = a.bias[2 * (t - 1) + 1];
      bc2 = (1.0 - a.b2) / (c * c);
    } else {
      bc1 = 1.0 - pow(a.b1, static_cast<double>(step));
      bc2 = 1.0 - pow(a.b2, static_cast<double>(step));
    }
    ks[q].decay = static_cast<float>(1.0 - lr * a.wd);
    ks[q].rate = static_cast<float>(lr / bc1);
    ks[q].rc2 = static_cast<float>(1.0 / sqrt(bc2));
  }
  const float b1 = static_cast<float>(a.b1), c1 = static_cast<float>(1.0 - a.b1);
  const float b2 = static_cast<float>(a.b2), c2 = static_cast<float>(1.0 - a.b2);
  const float eps = static_cast<float>(a.eps);
  const bool scaled = a.grad_scale != nullptr;
  const float gs = scaled ? *a.grad_scale : 1.f;
  __syncthreads();

  int ti = t0;
  for (int u = u0 + warp; u < u1; u += kAwWarps) {
    while (ti + 1 < a.count && a.start[ti + 1] <= u) ++ti;
    const ttrl_adamw_tensor& T = a.t[ti];
    const AdamwScalars k = ks[ti];
    const bool vec = a.vec[ti] != 0;
    const long long blk = u - a.start[ti];
    const long long at = blk * kAwBlock + lane * 4, end = T.numel;
    const bool codes = T.bits == 8;
    float g[2][4], p[2][4], m[2][4], v[2][4];
    uint32_t mc[2], vc[2];
    float ms = 0.f, vs = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long i = at + h * 128;
      get4(T.grad, i, end, vec, g[h]);
      get4(T.param, i, end, vec, p[h]);
      if (!codes) {
        get4(static_cast<const float*>(T.m), i, end, vec, m[h]);
        get4(static_cast<const float*>(T.v), i, end, vec, v[h]);
      } else {
        mc[h] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(T.m) + i);
        vc[h] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(T.v) + i);
      }
    }
    if (codes) {
      ms = T.m_scale[blk];
      vs = T.v_scale[blk];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m[h][e] = __fmul_rn(m_share(m_float(mc[h], e)), ms);
          v[h][e] = __fmul_rn(v_share(v_float(vc[h], e)), vs);
        }
    }
    float mm = 0.f, vm = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = scaled ? __fmul_rn(g[h][e], gs) : g[h][e];
        m[h][e] = __fadd_rn(__fmul_rn(m[h][e], b1), __fmul_rn(x, c1));
        v[h][e] = __fadd_rn(__fmul_rn(v[h][e], b2), __fmul_rn(__fmul_rn(x, x), c2));
        // The step, a small part of p, by the fast root and quotient: each
        // within two units in the last place of itself.
        const float root = fmaf(sqrt_fast(v[h][e]), k.rc2, eps);
        p[h][e] = __fsub_rn(__fmul_rn(p[h][e], k.decay), __fdividef(m[h][e], root) * k.rate);
        if (codes) {
          mm = abs_max(mm, m[h][e]);
          vm = abs_max(vm, v[h][e]);
        }
      }
    if (codes) {
      mm = warp_abs_max(mm);
      vm = warp_abs_max(vm);
      if (lane == 0) {
        T.m_scale[blk] = mm;
        T.v_scale[blk] = vm;
      }
      // The padding's moments are zero (its gradients read as zero).
      put_codes(static_cast<uint8_t*>(T.m) + at, static_cast<uint8_t*>(T.v) + at, m, v, mm, vm);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long i = at + h * 128;
      put4(T.param, i, end, vec, p[h]);
      if (!codes) {
        put4(static_cast<float*>(T.m), i, end, vec, m[h]);
        put4(static_cast<float*>(T.v), i, end, vec, v[h]);
      }
    }
  }

  // The last block to finish advances the counters of this launch, which all
  // blocks have read by then; tensors that share one advance it once.
  __syncthreads();
  __shared__ bool last;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(reinterpret_cast<unsigned*>(a.ticket), 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  for (int q = threadIdx.x; q < a.count; q += kAwThreads)
    if (a.lead[q]) a.steps[a.t[q].step_index] += 1;
  if (threadIdx.x == 0) *a.ticket = 0;
}

// ------------------------------------------------- 8-bit moments to and from

struct AdamwStateArgs {
  ttrl_adamw_state t[TTRL_ADAMW_MAX_TENSORS];
  int32_t start[TTRL_ADAMW_MAX_TENSORS + 1];
  int32_t count;
  int32_t pack;
};

__global__ void __launch_bounds__(kAwThreads)
    adamw_state_kernel(const __grid_constant__ AdamwStateArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * kAwWarps;
  int ti = 0;
  for (int u = blockIdx.x * kAwWarps + (threadIdx.x >> 5); u < a.start[a.count]; u += warps) {
    while (ti + 1 < a.count && a.start[ti + 1] <= u) ++ti;
    const ttrl_adamw_state& T = a.t[ti];
    const long long blk = u - a.start[ti];
    const long long at = blk * kAwBlock + lane * 4, end = T.numel;
    const bool vec = (reinterpret_cast<uintptr_t>(T.m32) & 15u) == 0 &&
                     (reinterpret_cast<uintptr_t>(T.v32) & 15u) == 0;
    uint8_t* m8 = static_cast<uint8_t*>(T.m8);
    uint8_t* v8 = static_cast<uint8_t*>(T.v8);
    float m[2][4], v[2][4];
    if (!a.pack) {
      const float ms = T.m_scale[blk], vs = T.v_scale[blk];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long i = at + h * 128;
        const uint32_t mc = *reinterpret_cast<const uint32_t*>(m8 + i);
        const uint32_t vc = *reinterpret_cast<const uint32_t*>(v8 + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m[h][e] = __fmul_rn(m_share(m_float(mc, e)), ms);
          v[h][e] = __fmul_rn(v_share(v_float(vc, e)), vs);
        }
        put4(T.m32, i, end, vec, m[h]);
        put4(T.v32, i, end, vec, v[h]);
      }
    } else {
      float mm = 0.f, vm = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        get4(T.m32, at + h * 128, end, vec, m[h]);
        get4(T.v32, at + h * 128, end, vec, v[h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mm = abs_max(mm, m[h][e]);
          vm = abs_max(vm, v[h][e]);
        }
      }
      mm = warp_abs_max(mm);
      vm = warp_abs_max(vm);
      if (lane == 0) {
        T.m_scale[blk] = mm;
        T.v_scale[blk] = vm;
      }
      put_codes(m8 + at, v8 + at, m, v, mm, vm);
    }
  }
}

// ------------------------------------------------------------------ host

static bool aw_aligned(const void* p, uintptr_t n) {
  return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

template <int MAX>
static int adamw_launch(const ttrl_adamw_tensor* tensors, int count, int32_t* steps,
                        int32_t* ticket, const float* grad_scale, const double* lr_device,
                        double lr, double b1, double b2, double eps, double wd,
                        const double* bias, long long bias_steps, cudaStream_t st) {
  AdamwArgs<MAX> a;
  std::memset(&a, 0, sizeof(a));
  long long units = 0;
  int32_t highest = -1;  // counters in rising order need no search for a twin
  for (int i = 0; i < count; ++i) {
    const ttrl_adamw_tensor& t = tensors[i];
    a.t[i] = t;
    bool lead = true;
    if (t.step_index <= highest)
      for (int r = 0; r < i && lead; ++r) lead = tensors[r].step_index != t.step_index;
    highest = t.step_index > highest ? t.step_index : highest;
    a.lead[i] = lead;
    a.start[i] = static_cast<int32_t>(units);
    a.vec[i] = aw_aligned(t.param, 16) && aw_aligned(t.grad, 16) &&
               (t.bits == 8 || (aw_aligned(t.m, 16) && aw_aligned(t.v, 16)));
    units += (t.numel + kAwBlock - 1) / kAwBlock;
    if (units >= (1ll << 31))
      return set_error(TTRL_EUNSUPPORTED, "adamw: more than 2^31 blocks of %d elements", kAwBlock);
  }
  a.start[count] = static_cast<int32_t>(units);
  a.count = count;
  a.steps = steps;
  a.ticket = ticket;
  a.grad_scale = grad_scale;
  a.lr_device = lr_device;
  a.bias = bias;
  a.bias_steps = bias_steps;
  a.lr = lr;
  a.b1 = b1;
  a.b2 = b2;
  a.eps = eps;
  a.wd = wd;
  const long long want = (units + kAwWarps - 1) / kAwWarps;
  const long long wave = 148ll * kAwBlocksPerSM;
  const unsigned blocks = static_cast<unsigned>(want < wave ? want : wave);
  const cudaError_t e = launch_pdl(adamw_kernel<MAX>, dim3(blocks), dim3(kAwThreads), 0, st, a);
  note_launch();
  return e == cudaSuccess ? TTRL_OK : set_cuda_error("adamw launch", e);
}

int adamw_step(const ttrl_adamw_tensor* tensors, int count, int32_t* steps, int32_t* ticket,
               const float* grad_scale, const double* lr_device, double lr, double b1, double b2,
               double eps, double wd, const double* bias, long long bias_steps, cudaStream_t st) {
  if (bias != nullptr && bias_steps < 1)
    return set_error(TTRL_EINVAL, "adamw: a bias table needs at least one step");
  if (count < 0 || count > TTRL_ADAMW_MAX_TENSORS)
    return set_error(TTRL_EINVAL, "adamw: %d tensors, a call takes up to %d", count,
                     TTRL_ADAMW_MAX_TENSORS);
  if (count == 0) return TTRL_OK;
  if (tensors == nullptr || steps == nullptr || ticket == nullptr)
    return set_error(TTRL_EINVAL, "adamw: null tensor list, step counter or ticket");
  if (!(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0))
    return set_error(TTRL_EINVAL, "adamw: betas have to be in [0, 1)");
  // The step divides by sqrt(v) + eps in float, of which 1 / eps has to be one.
  if (!(eps >= 0x1p-126))
    return set_error(TTRL_EINVAL, "adamw: eps has to be at least 2^-126, got %g", eps);
  if (!(wd >= 0.0)) return set_error(TTRL_EINVAL, "adamw: weight decay has to be >= 0");
  for (int i = 0; i < count; ++i) {
    const ttrl_adamw_tensor& t = tensors[i];
    if (t.numel <= 0 || !t.param || !t.grad || !t.m || !t.v || t.step_index < 0)
      return set_error(TTRL_EINVAL, "adamw: tensor %d is empty, has a null buffer or no counter",
                       i);
    if (t.bits != 32 && t.bits != 8)
      return set_error(TTRL_EINVAL, "adamw: tensor %d holds its moments in %d bits, not 32 or 8",
                       i, t.bits);
    if (t.bits == 8 && (!t.m_scale || !t.v_scale || !aw_aligned(t.m, 4) || !aw_aligned(t.v, 4)))
      return set_error(TTRL_EINVAL,
                       "adamw: tensor %d needs scales, and codes on a 4-byte boundary", i);
  }
  return count <= kAwFew
             ? adamw_launch<kAwFew>(tensors, count, steps, ticket, grad_scale, lr_device, lr, b1,
                                    b2, eps, wd, bias, bias_steps, st)
             : adamw_launch<TTRL_ADAMW_MAX_TENSORS>(tensors, count, steps, ticket, grad_scale,
                                                    lr_device, lr, b1, b2, eps, wd, bias,
                                                    bias_steps, st);
}

int adamw_state_convert(const ttrl_adamw_state* tensors, int count, int pack, cudaStream_t st) {
  if (count < 0 || count > TTRL_ADAMW_MAX_TENSORS)
    return set_error(TTRL_EINVAL, "adamw_state: %d tensors, a call takes up to %d", count,
                     TTRL_ADAMW_MAX_TENSORS);
  if (count == 0) return TTRL_OK;
  if (tensors == nullptr) return set_error(TTRL_EINVAL, "adamw_state: null tensor list");
  AdamwStateArgs a;
  std::memset(&a, 0, sizeof(a));
  long long units = 0;
  for (int i = 0; i < count; ++i) {
    const ttrl_adamw_state& t = tensors[i];
    if (t.numel <= 0 || !t.m32 || !t.v32 || !t.m8 || !t.v8 || !t.m_scale || !t.v_scale ||
        !aw_aligned(t.m8, 4) || !aw_aligned(t.v8, 4))
      return set_error(TTRL_EINVAL,
                       "adamw_state: tensor %d is empty, has a null buffer or codes off a 4-byte "
                       "boundary", i);
    a.t[i] = t;
    a.start[i] = static_cast<int32_t>(units);
    units += (t.numel + kAwBlock - 1) / kAwBlock;
    if (units >= (1ll << 31))
      return set_error(TTRL_EUNSUPPORTED, "adamw_state: more than 2^31 blocks of %d elements",
                       kAwBlock);
  }
  a.start[count] = static_cast<int32_t>(units);
  a.count = count;
  a.pack = pack;
  const long long want = (units + kAwWarps - 1) / kAwWarps;
  const long long wave = 148ll * 8;
  const unsigned blocks = static_cast<unsigned>(want < wave ? want : wave);
  const cudaError_t e = launch_pdl(adamw_state_kernel, dim3(blocks), dim3(kAwThreads), 0, st, a);
  note_launch();
  return e == cudaSuccess ? TTRL_OK : set_cuda_error("adamw_state launch", e);
}

}  // namespace ttrl

using namespace ttrl;

extern "C" {

int ttrl_adamw_step(const ttrl_adamw_tensor* tensors, int count, int32_t* steps, int32_t* ticket,
                    const float* grad_scale, const double* lr_device, double lr, double b1,
                    double b2, double eps, double weight_decay, const double* bias_table,
                    int64_t bias_steps, ttrl_stream_t stream) {
  return adamw_step(tensors, count, steps, ticket, grad_scale, lr_device, lr, b1, b2, eps,
                    weight_decay, bias_table, bias_steps, static_cast<cudaStream_t>(stream));
}

int ttrl_adamw_state_convert(const ttrl_adamw_state* tensors, int count, int pack,
                             ttrl_stream_t stream) {
  return adamw_state_convert(tensors, count, pack, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
