// Linear attention with a decay for each head:
//
//   S_t = d_h (1 - start_t) S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t
//
// with S a [K][V] matrix for every lane and head. Rows are time-major, as the
// GRU's: token (t, lane) is row t * batch + lane of [q | k | v], each head by
// head. A start drops the state (it is selected away, not multiplied by zero).
//
// Backward: with R_t the gradient of S_t, the same recurrence runs backwards
// in time, R_t = scale q_t do_t^T + d (1 - start_{t+1}) R_{t+1}, and
//   dq_t = scale do_t S_t^T,  dk_t = v_t R_t^T,  dv_t = k_t R_t,
// so each gradient is a scan of this kind with the operands' places changed:
// one kernel serves all four (scan direction, operand pointers and strides).
//
// Scan. Tokens are taken in chunks of 64. With i, j the places in a chunk,
// c_i = d^(i + 1) and w_ij = d^(i - j) where no start lies in between (0
// elsewhere, and for j > i):
//   o_i = c_i q_i S + sum_j w_ij (q_i . k_j) v_j,
//   S  <- d^64 S + sum_j w_(63)j k_j v_j^T
// four small matrix products a chunk. The state stays in registers (and a
// copy in shared memory) along the chunks, so q, k and v are read once and
// o written once: 4 (2K + 2V) bytes a token and head is the floor.
//
// The products must be good to fp32, on tensor cores. Each row of q, k and v
// gets a power of two that brings its largest value just below 2^15 (the state
// has one for all of it), and each
// value is held as two half-precision numbers, hi and x - hi: 22 bits, down to
// values 2^-18 of the row's largest, and 2^-40 of that below. The powers of k's
// and v's rows go into the weight of their token's scores, and a row of weighted
// scores, split in its turn, is divided by the largest token that it sees: a
// token's error goes by what its own result is made of, not by a larger token in
// the same tile, in an episode that a start has dropped or later in time. (One
// power a tile took 13% less time, and lost all bits of a token beside one 10^12
// times its size; done in fp32, a chunk takes ten times as long. Tokens of e^N(0, 1)
// times a size each: 638 us instead of 637 backward; of e^3N(0, 1), 728.) A product is
// hi hi + hi lo + lo hi, three mma.sync of 16-bit operands at twice the rate
// that two-part tf32 has. k, v and the state are split once, as they are
// stored in shared memory, and ldmatrix reads either orientation; a warp's
// rows of q are its own and stay in registers. The tensor core cuts sums
// off instead of rounding them (measured: 1.3e-6 of the result after 512
// products, all to one side), so no sum runs further than one chunk before
// fp32 additions take over.
//
// This form (mma.sync, chunks of 64, four blocks an SM) serves sequences of up
// to 64 tokens, widths of up to 32 and the sums of segments; longer ones take
// the same mathematics in chunks of 128 on tcgen05.mma, further down.
//
// Times on B200, forward and backward (three scans in one launch, or two where
// key and value pad differently), shares of the measured copy rate in brackets:
//   32 tokens x 16 lanes x 4 heads of 64/64: 12 and 15 us: one chunk's chain of
//     loads, splits and products, mostly first fetches of instructions
//   512 x 256 x 4 of 32/32: 122 (34%) and 328 us
//   1024 x 64 x 8 of 64/64: 240 (35%) and 637 us; of 64/128: 424 and 1086 us
//   2048 x 8 x 8 of 128/128: 173 and 504 us
//   8191 x 2 x 8 of 64/64: 118 and 319 us, in segments
//
// A product with a masked-out factor multiplies by zero, which infinities and
// NaN survive. So a chunk whose results are not all finite is done again
// token by token in fp32, from the recurrence itself (la_exact); so is one whose
// columns differ in size by more than the halves hold (kLaShort).
//
// Few lanes and heads with many tokens: the scan is cut into segments. One
// launch gives each segment's state from nothing, a second adds them up in
// order, a third does the full scan of all segments at once.
#include <algorithm>
#include <cstring>
#include <mutex>

#include <cuda_fp16.h>

#include "common.cuh"
#include "internal.h"

namespace ttrl {

constexpr int kLaChunk = 64;
constexpr int kLaThreads = 128;

struct LaArgs {
  const float *q, *k, *v;  // [steps * batch] rows, head h at + h * (width)
  float* o;
  int64_t ldq, ldk, ldv, ldo;  // floats from row to row
  const float* starts;         // [steps][batch], or null
  const float* decay;          // [heads]
  const float* s_in;           // [batch][heads] matrices, element (k, v) at k * in_k + v * in_v
  float* s_out;                // (may be null)
  float* seg;                  // [sums][batch * heads][K][V]: what each sum's tokens add to the
                               // state; behind a segment's last sum, then, the state itself
  int* seg_start;              // [sums][batch]: a start inside
  int32_t steps, batch, heads, kd, vd;
  int32_t in_k, in_v, out_k, out_v;
  int32_t segments, seg_len;
  int32_t sums, sum_len;  // a segment's parts, seg_len a multiple of sum_len
  int32_t reverse;  // tokens last to first; s_in enters the first without decay,
                    // and s_out leaves the last with one more and its start
  int32_t vq, vk, vv, vo;  // 16-byte loads; 8-byte stores
  float scale, kscale;     // of o, of k
};

// Scans of the same steps, lanes and heads in one launch: the last grid
// dimension goes over the scans, and over their blocks of columns.
// A scan on its own has its arguments at fixed places (with three the forward
// of 4096 x 4 lanes x 4 heads of 128 takes 146 us instead of 133).
template <int N>
struct LaJobs {
  LaArgs j[N];
  int32_t n;  // in use
};

// d^n from log2(d); d^0 is 1 for d = 0 too. The exponent's rounding is 2^-24
// of it, so a power is off by more than 2^-22 only where it is below 2^-4.
__device__ __forceinline__ float decay_pow(float log2_d, int n) {
  return n == 0 ? 1.f : exp2f(n * log2_d);
}

// Two values times a power of two as packed halves: hi, and what is left.
__device__ __forceinline__ void split2(float x, float y, float scale, uint32_t& hi, uint32_t& lo) {
  const float2 t = __fmul2_rn(make_float2(x, y), make_float2(scale, scale));
  const __half2 h = __floats2half2_rn(t.x, t.y);
  const float2 f = __half22float2(h);
  const float2 r = __ffma2_rn(f, make_float2(-1.f, -1.f), t);
  const __half2 l = __floats2half2_rn(r.x, r.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
// Two values as packed halves: hi, and what is left.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ float2 join2(uint32_t hi, uint32_t lo) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  return make_float2(h.x + l.x, h.y + l.y);
}

// The power of two that brings the state's largest magnitude
// to [2^14, 2^15), from 2^-40 to 2^90. Beyond, at either end, the chunk is done
// token by token (tile_fits).
constexpr int kLaTileMost = 90;
__device__ __forceinline__ float tile_scale(uint32_t max_bits) {
  if (max_bits == 0) return 1.f;
  int e = 141 - static_cast<int>(max_bits >> 23);
  e = max(-40, min(kLaTileMost, e));
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}
__device__ __forceinline__ bool tile_fits(uint32_t max_bits) {
  return max_bits < 0x7f800000u && (max_bits == 0 || (max_bits >> 23) >= 141 - kLaTileMost);
}
// Of a power of two. Products of such inverses may run out of range to zero,
// as what they scale does; a product of the powers themselves may not.
__device__ __forceinline__ float pow2_inverse(float s) {
  return __uint_as_float((254u << 23) - __float_as_uint(s));
}

// A row of q, k or v has a power of two of its own, that brings its largest value to
// [2^14, 2^15): from 2^-40 to 2^100 (smaller rows: row_fits), those of a token's k
// and v 2^124 at most. No power
// (kLaNone) for a row of zeros.
constexpr int kLaNone = -128, kLaLeast = -40, kLaMost = 100, kLaBoth = 124;
__device__ __forceinline__ int row_exp(uint32_t max_bits) {
  if (max_bits == 0) return kLaNone;
  return max(kLaLeast, min(kLaMost, 141 - static_cast<int>(max_bits >> 23)));
}
__device__ __forceinline__ bool row_fits(uint32_t max_bits) {
  return max_bits < 0x7f800000u && (max_bits == 0 || (max_bits >> 23) >= 141 - kLaMost);
}
__device__ __forceinline__ float pow2(int e) {  // -126 .. 127
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}
__device__ __forceinline__ float row_scale(int e) { return e == kLaNone ? 1.f : pow2(e); }
// The power of two above x > 0; 1 for 0.
__device__ __forceinline__ float pow2_above(float x) {
  return x == 0.f ? 1.f : pow2(max(-126, static_cast<int>(__float_as_uint(x) >> 23) - 126));
}
// A token's size, the inverse of what its k and v were scaled by, as the
// exponent of a float (3 to 207; 0 where either is zero). `fine` becomes false
// where the token is too small for one.
__device__ __forceinline__ uint32_t token_size(int ek, int ev, bool& fine) {
  if (ek == kLaNone || ev == kLaNone) return 0u;
  fine &= ek + ev <= kLaBoth;
  return static_cast<uint32_t>(127 - min(ek + ev, kLaBoth));
}
__device__ __forceinline__ float size_float(uint32_t size) { return __uint_as_float(size << 23); }
// Tokens alike within 2^8: then the bound of a row's scores is the largest
// token's, which costs them 2^8 of the 2^32 that their halves hold beside the
// typical one.
constexpr uint32_t kLaAlike = 8;
// The largest of the LANES neighbouring lanes that share a row.
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  if constexpr (LANES == 32) {
    return __reduce_max_sync(0xffffffffu, x);
  } else if constexpr (LANES == 16) {
    const bool low = (threadIdx.x & 16) == 0;
    const uint32_t a = __reduce_max_sync(0xffffffffu, low ? x : 0u);
    const uint32_t b = __reduce_max_sync(0xffffffffu, low ? 0u : x);
    return low ? a : b;
  } else {
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) x = max(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
  }
}
// What the halves cannot hold. A scaled value below 2^-3 (kLaShort) keeps fewer
// than 22 bits. One by chance (one normal value in 80,000) does not show in its
// column's norm; columns that differ in size have many, and the small one's
// results need them. So a chunk is done in fp32, token by token, where la_spare
// threads have such values in la_rows of their rows (a column is at least four
// threads'). That q's columns differ does no harm unless k's do too, and that the
// state's do none where every token of the chunk weighs as much as 2^-18 of
// the state: then its column is of that size (la_dwarfs).
constexpr int kLaShort = 127 - 3;  // an exponent as in a float's bits
// Twice the bits of the smaller magnitude, less one: zero is the largest.
__device__ __forceinline__ uint32_t least2(float x, float y) {
  return min(__float_as_uint(x) * 2u - 1u, __float_as_uint(y) * 2u - 1u);
}
// Whether one of the magnitudes behind `least`, times 2^e, is short of bits.
__device__ __forceinline__ int la_short(uint32_t least, int e) {
  return least < (static_cast<uint32_t>(kLaShort - e) << 24) - 1u;
}
__device__ __forceinline__ int la_short(const float (&x)[4], int e) {
  return la_short(min(least2(x[0], x[1]), least2(x[2], x[3])), e == kLaNone ? 0 : e);
}
// Whether a state scaled by 2^es is more than that beside tokens of this least
// size (0: tokens of zeros).
__device__ __forceinline__ bool la_dwarfs(int es, uint32_t least_size) {
  return es + static_cast<int>(least_size) + 30 < 127;
}
__device__ __forceinline__ int la_rows(int len) { return len >= 64 ? 2 : 1; }
__device__ __forceinline__ int la_spare(int len) {
  return len >= 64 ? 2 : max(1, min(4, len / 2));
}

// Scores of two such tiles are below 128 * 2^30: times this, a half.
constexpr float kScoreScale = 1.f / (1 << 22);

__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t saddr) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(saddr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(saddr)
                 : "memory");
}

// A 16 x 16 operand block of a split tile, both parts.
struct Frag {
  uint32_t hi[4], lo[4];
  template <bool TRANS>
  __device__ __forceinline__ void load(uint32_t saddr, uint32_t lo_off) {
    ldsm4<TRANS>(hi, saddr);
    ldsm4<TRANS>(lo, saddr + lo_off);
  }
};
// acc += A B for the two column tiles of B.
__device__ __forceinline__ void mma3(float (&acc0)[4], float (&acc1)[4], const Frag& a,
                                     const Frag& b) {
  mma16(acc0, a.lo, b.hi[0], b.hi[1]);
  mma16(acc1, a.lo, b.hi[2], b.hi[3]);
  mma16(acc0, a.hi, b.lo[0], b.lo[1]);
  mma16(acc1, a.hi, b.lo[2], b.lo[3]);
  mma16(acc0, a.hi, b.hi[0], b.hi[1]);
  mma16(acc1, a.hi, b.hi[2], b.hi[3]);
}

// Shared tiles of halves, hi then lo; a row is 8 halves longer than a multiple
// of 64, so the 8 rows of an ldmatrix lie in different banks.
template <int DK, int DV>
struct LaTile {
  static constexpr int kLdK = DK + 8, kLdV = DV + 8;       // halves
  static constexpr int kK = kLaChunk * kLdK * 2;           // bytes of a part
  static constexpr int kV = kLaChunk * kLdV * 2;
  static constexpr int kS = DK * kLdV * 2;
  static constexpr int kK0 = 0, kV0 = 2 * kK, kS0 = kV0 + 2 * kV;
  // pw, wt, cnt, mask, state maxima, the sum's scale; kf, rows, exponents
  static constexpr int kRest = kS0 + 2 * kS;
  static constexpr int kBytes = kRest + (16 + 3 * kLaChunk + 4 + 2 + 4 + 2) * 4 + 10 * kLaChunk;
};

// One tile of `rows` tokens by `cols` floats (the rest zeros) in registers, 4
// floats a slot: slot u of a thread is floats 4 (u * threads + tid) of the
// padded tile; token r is row (first + r * step).
template <int D>
__device__ __forceinline__ void load_tile(float (&x)[kLaChunk * D / (4 * kLaThreads)][4],
                                              const float* src, int64_t ld, int rows, int cols,
                                              int64_t first, int64_t step, bool vec) {
  constexpr int Q = D / 4, N = kLaChunk * D / (4 * kLaThreads);
  const int r0 = threadIdx.x / Q, c = (threadIdx.x % Q) * 4;
  const float* p = src + (first + r0 * step) * ld + c;
  const int64_t jump = step * ld * (kLaThreads / Q);
#pragma unroll
  for (int u = 0; u < N; ++u, p += jump) {
    const bool in = r0 + u * (kLaThreads / Q) < rows;
    if (vec) {
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in && c < cols) t = *reinterpret_cast<const float4*>(p);
      x[u][0] = t.x, x[u][1] = t.y, x[u][2] = t.z, x[u][3] = t.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[u][e] = in && c + e < cols ? p[e] : 0.f;
    }
  }
}
// The same slots, each row scaled by its own power of two and split, into a
// shared tile; the powers' exponents to exps[row]. False where a row is not
// finite, or too small for the powers there are.
template <int D>
__device__ __forceinline__ bool store_tile(uint32_t base, uint32_t part,
                                           const float (&x)[kLaChunk * D / (4 * kLaThreads)][4],
                                           int8_t* exps, int& lost) {
  constexpr int Q = D / 4, N = kLaChunk * D / (4 * kLaThreads);
  const int r0 = threadIdx.x / Q;
  const uint32_t at = base + (r0 * (D + 8) + (threadIdx.x % Q) * 4) * 2;
  bool fine = true;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[u][e]) & 0x7fffffffu);
    top = row_max<Q>(top);
    const int e = row_exp(top);
    fine &= row_fits(top);
    lost += la_short(x[u], e);
    const float scale = row_scale(e);
    if (threadIdx.x % Q == 0) exps[r0 + u * (kLaThreads / Q)] = static_cast<int8_t>(e);
    uint32_t h0, h1, l0, l1;
    split2(x[u][0], x[u][1], scale, h0, l0);
    split2(x[u][2], x[u][3], scale, h1, l1);
    const uint32_t to = at + u * (kLaThreads / Q) * (D + 8) * 2;
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(h0), "r"(h1) : "memory");
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + part), "r"(l0), "r"(l1) : "memory");
  }
  return fine;
}

// Not zero where a start lies before token `place` of the scan (its own start;
// run backwards, the start of the token after it).
__device__ __forceinline__ float la_start(const LaArgs& a, int place, int lane) {
  if (a.starts == nullptr || (a.reverse && place == 0)) return 0.f;
  const int token = a.reverse ? a.steps - place : place;
  return a.starts[static_cast<int64_t>(token) * a.batch + lane];
}

// A chunk of `len` tokens from the recurrence itself, in fp32: the state is in
// `ss` ([DK][LD]) before and behind it. A thread has one column and DK / (TH /
// DV) rows of it in registers; the sums over rows meet in `part` (32 tokens of
// TH floats), so a token costs no barrier. drop(i): a start before token i.
template <int DK, int DV, int LD, int TH, bool OUT, typename F>
__device__ __forceinline__ void la_exact(const LaArgs& a, float* ss, float* part, int64_t row,
                                         int64_t dir, int len, int lead, int h, int v0, int vcols,
                                         float decay, F&& drop) {
  constexpr int G = TH / DV, R = DK / G, TOKENS = 32;
  const int col = threadIdx.x % DV, grp = threadIdx.x / DV, r0 = grp * R;
  const bool mine = col < vcols;
  float s[R];
#pragma unroll
  for (int r = 0; r < R; ++r) s[r] = ss[(r0 + r) * LD + col];
  for (int i0 = 0; i0 < len; i0 += TOKENS) {
    const int n = min(TOKENS, len - i0);
    for (int i = 0; mine && i < n; ++i) {
      const int64_t at = row + (i0 + i) * dir;
      const float f = i0 + i == 0 && lead == 0 ? 1.f : decay;
      const bool gone = drop(i0 + i);
      const float* k = a.k + at * a.ldk + h * a.kd + r0;
      const float* q = a.q + at * a.ldq + h * a.kd + r0;
      const float v = a.v[at * a.ldv + h * a.vd + v0 + col];
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r0 + r >= a.kd) continue;
        s[r] = fmaf(k[r] * a.kscale, v, gone ? 0.f : s[r] * f);
        if (OUT) sum = fmaf(q[r], s[r], sum);
      }
      if (OUT) part[(i * G + grp) * DV + col] = sum;
    }
    if (OUT) {
      __syncthreads();
      for (int e = threadIdx.x; e < n * DV; e += TH) {
        const int i = e / DV, c = e % DV;
        if (c >= vcols) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < G; ++w) sum += part[(i * G + w) * DV + c];
        a.o[(row + (i0 + i) * dir) * a.ldo + h * a.vd + v0 + c] = sum * a.scale;
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) ss[(r0 + r) * LD + col] = s[r];
  __syncthreads();
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// Lane g = lane / 4, c = lane % 4 of a warp; an accumulator holds (row g | g +
// 8, column 2c | 2c + 1), and two neighbouring ones are, as they are, the A
// fragment of the next product.
template <int DK, int DV, bool OUT, int N>
__global__ void __launch_bounds__(kLaThreads, DK <= 64 ? 4 : DV == 64 ? 2 : 3)
    la_scan_kernel(const __grid_constant__ LaJobs<N> jobs) {
  using T = LaTile<DK, DV>;
  const LaArgs& a = jobs.j[N == 1 ? 0 : blockIdx.z % jobs.n];
  constexpr int LV = T::kLdV;
  constexpr int NV = DV / 8;  // column tiles of o and of the state
  // State tiles: a warp owns MT blocks of 16 rows (K) and NS column tiles.
  constexpr int MT = DK >= 64 ? DK / 64 : 1;
  constexpr int NS = DK >= 64 ? NV : NV / 2;
  constexpr int NK = DK / 16;
  extern __shared__ __align__(16) uint8_t la_smem[];
  float* ss = reinterpret_cast<float*>(la_smem + T::kS0);  // the state in fp32, token by token
  // kScoreScale d^n, n = 0..64, and 16 zeros before.
  float* pw = reinterpret_cast<float*>(la_smem + T::kRest) + 16;
  float* wt = pw + kLaChunk + 4;                         // weight of a token in the state
  int* cnt = reinterpret_cast<int*>(wt + kLaChunk);      // starts up to a token, its own included
  uint32_t* mask = reinterpret_cast<uint32_t*>(cnt + kLaChunk);  // [2]
  uint32_t* maxima = mask + 2;                                   // [4 warps], of the state
  float* sum_up = reinterpret_cast<float*>(maxima + 4);          // [1] of the state's sum
  float* kf = sum_up + 2;        // a token's size
  float* reach = kf + kLaChunk;  // the size of what a row's scores may add up
  int8_t* kexp = reinterpret_cast<int8_t*>(reach + kLaChunk);  // of k's rows, then v's
  const uint32_t sbase = smem_u32(la_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int bh = blockIdx.x, b = bh / a.heads, h = bh - b * a.heads;
  const int seg = blockIdx.y;
  const int v0 = (N == 1 ? blockIdx.z : blockIdx.z / jobs.n) * DV;
  const int vcols = min(DV, a.vd - v0);
  // Scans of fewer columns or segments than another.
  if (vcols <= 0 || seg >= (OUT ? a.segments : a.sums) || (!OUT && a.segments == 1)) return;
  // Rows of the chunk this warp scores: the later ones see more tokens, so
  // neighbouring blocks give them to different quarters of an SM.
  const int rb = ((warp + blockIdx.x) & 3) * 16;
  const int sm = DK >= 64 ? warp * 16 : (warp & 1) * 16;        // first state row (then + 64)
  const int sn = DK >= 64 ? 0 : (warp >> 1) * (DV / 2);         // first state column
  // This lane's row addresses for ldmatrix: plain B (rows of k), transposed A
  // (columns of k) and transposed B (v, the state).
  const uint32_t k_at = sbase + T::kK0 +
                        (((lane & 7) + (lane >> 4) * 8) * T::kLdK + ((lane >> 3) & 1) * 8) * 2;
  const uint32_t kt_at = sbase + T::kK0 +
                         (((lane & 7) + (lane >> 4) * 8) * T::kLdK + sm + ((lane >> 3) & 1) * 8) * 2;
  const uint32_t vt_at = sbase + T::kV0 + ((lane & 15) * LV + (lane >> 4) * 8) * 2;
  const uint32_t st_at = sbase + T::kS0 + ((lane & 15) * LV + (lane >> 4) * 8) * 2;
  pdl_trigger();
  pdl_wait();
  const float decay = a.decay[h];
  for (int n = tid - 16; n <= kLaChunk; n += kLaThreads)
    pw[n] = n < 0 ? 0.f : decay_pow(log2f(decay), n) * kScoreScale;

  // The state entering the segment, in this warp's registers.
  float st[MT][NS][4];
  const int64_t mat = static_cast<int64_t>(bh) * a.kd * a.vd;
  const float* from = nullptr;
  int fk = a.vd, fv = 1;
  if (OUT) {
    if (seg > 0) {
      from = a.seg + mat +
           static_cast<int64_t>(seg * (a.seg_len / a.sum_len) - 1) * a.batch * a.heads * a.kd * a.vd;
    } else if (a.s_in != nullptr) {
      from = a.s_in + mat;
      fk = a.in_k;
      fv = a.in_v;
    }
  }
  // f(held, row, column) over this warp's part of the state.
  auto each_state = [&](auto&& f) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          f(st[m][n][e], sm + m * 64 + g + (e >> 1) * 8, sn + n * 8 + 2 * c + (e & 1));
  };
  each_state([&](float& held, int r, int col) {
    held = from != nullptr && r < a.kd && v0 + col < a.vd
               ? from[static_cast<int64_t>(r) * fk + static_cast<int64_t>(v0 + col) * fv]
               : 0.f;
  });

  const int span = OUT ? a.seg_len : a.sum_len;
  const int begin = seg * span;
  const int end = min(a.steps, begin + span);
  const int64_t dir = a.reverse ? -static_cast<int64_t>(a.batch) : a.batch;
  int any_start = 0;
  for (int c0 = begin; c0 < end; c0 += kLaChunk) {
    const int len = min(kLaChunk, end - c0);
    const int lead = c0 == 0 && a.reverse ? 0 : 1;
    const int64_t row = static_cast<int64_t>(a.reverse ? a.steps - 1 - c0 : c0) * a.batch + b;
    float sst = 1.f;  // the state's power of two
    uint64_t starts;
    int total;
    bool finite;   // and within what the halves hold
    int lost = 0;  // rows with values short of bits
    {
      float xk[kLaChunk * DK / (4 * kLaThreads)][4], xv[kLaChunk * DV / (4 * kLaThreads)][4];
      uint32_t flag = 0;
      if (warp < 2)
        flag = __ballot_sync(0xffffffffu, tid < len && la_start(a, c0 + tid, b) != 0.f);
      load_tile<DK>(xk, a.k + h * a.kd, a.ldk, len, a.kd, row, dir, a.vk);
      load_tile<DV>(xv, a.v + h * a.vd + v0, a.ldv, len, vcols, row, dir, a.vv);
      if (a.kscale != 1.f) {
#pragma unroll
        for (int u = 0; u < kLaChunk * DK / (4 * kLaThreads); ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) xk[u][e] *= a.kscale;
      }
      finite = store_tile<DK>(sbase + T::kK0, T::kK, xk, kexp, lost);
      finite &= store_tile<DV>(sbase + T::kV0, T::kV, xv, kexp + kLaChunk, lost);
      if (OUT) {
        uint32_t top = 0;
        each_state([&](float& held, int, int) {
          top = max(top, __float_as_uint(held) & 0x7fffffffu);
        });
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) maxima[warp] = top;
      }
      if (warp < 2 && lane == 0) mask[warp] = flag;
    }
    __syncthreads();
    starts = mask[0] | static_cast<uint64_t>(mask[1]) << 32;
    total = __popcll(starts);
    uint32_t low = 255;  // the least of the tokens' sizes
    {
      uint32_t size[2], high = 0;
      bool zeros = false;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int j = w * 32 + lane;
        size[w] = token_size(kexp[j], kexp[kLaChunk + j], finite);
        high = max(high, size[w]);
        low = min(low, size[w] == 0 ? 255u : size[w]);
        zeros |= size[w] == 0 && j < len;
      }
      high = __reduce_max_sync(0xffffffffu, high);
      low = __reduce_min_sync(0xffffffffu, zeros ? 0u : low);
      if (tid < kLaChunk) {
        const uint64_t upto = starts & (~0ull >> (63 - tid));
        const float f[2] = {size_float(size[0]), size_float(size[1])};
        const float mine = warp == 0 ? f[0] : f[1];
        const int last = starts == 0 ? 0 : 63 - __clzll(starts);
        const float w = tid >= last && tid < len ? mine * (pw[len - 1 - tid] * (1.f / kScoreScale))
                                                 : 0.f;
        float m = size_float(high), most = m;
        if (high > low + kLaAlike) {
          // The state's sum: against the largest token at its weight.
          const int other = tid ^ 32;
          const float w2 = other >= last && other < len
                               ? (warp == 0 ? f[1] : f[0]) * (pw[len - 1 - other] * (1.f / kScoreScale))
                               : 0.f;
          most = __uint_as_float(
              __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(w, w2))));
          // The largest token that a row sees, at its weight: of the rows before
          // it in the warp, then of the first half.
          const int own = upto == 0 ? -1 : 63 - __clzll(upto);
          m = mine;
#pragma unroll
          for (int o = 1; o < 32; o *= 2) {
            const float before = __shfl_up_sync(0xffffffffu, m, o);
            if (lane >= o && tid - o >= own)
              m = fmaxf(m, before * (pw[o] * (1.f / kScoreScale)));
          }
          if (warp == 1) {
            const uint32_t early = static_cast<uint32_t>(starts);
            const int from = early == 0 ? -1 : 31 - __clz(early);
            const float carry = __uint_as_float(__reduce_max_sync(
                0xffffffffu, __float_as_uint(lane >= from ? f[0] * (pw[32 - lane] *
                                                                    (1.f / kScoreScale))
                                                          : 0.f)));
            if (own < 32) m = fmaxf(m, carry * (pw[lane] * (1.f / kScoreScale)));
          }
        }
        const float up = pow2_above(most);
        cnt[tid] = __popcll(upto);
        kf[tid] = mine;
        wt[tid] = w * pow2_inverse(up);
        reach[tid] = pow2_above(m);
        if (tid == 0) *sum_up = up;
      }
      if constexpr (OUT) {
        const uint32_t top = max(max(maxima[0], maxima[1]), max(maxima[2], maxima[3]));
        finite &= tile_fits(top);
        sst = tile_scale(top);
        const int es = static_cast<int>(__float_as_uint(sst) >> 23) - 127;
        if (la_dwarfs(es, low)) {
          int few = 0;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NS; ++n) {
              few += la_short(least2(st[m][n][0], st[m][n][1]), es);
              few += la_short(least2(st[m][n][2], st[m][n][3]), es);
            }
          if (few >= (a.kd > 8 && vcols > 8 ? 2 : 1)) finite = false;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t hi, lo;
              split2(st[m][n][half * 2] * sst, st[m][n][half * 2 + 1] * sst, hi, lo);
              uint8_t* to = la_smem + T::kS0 +
                            ((sm + m * 64 + g + half * 8) * LV + sn + n * 8 + 2 * c) * 2;
              *reinterpret_cast<uint32_t*>(to) = hi;
              *reinterpret_cast<uint32_t*>(to + T::kS) = lo;
            }
          }
      }
    }
    any_start |= total;
    // The next chunk's rows on their way to L2.
    if (c0 + kLaChunk < end) {
      const int next = min(kLaChunk, end - c0 - kLaChunk);
      const int r = tid >> 1;
      if (r < next) {
        const int64_t at = row + (kLaChunk + r) * dir;
        const int kc = (tid & 1) * 32, kstep = 64;
        for (int i = kc; i < a.kd; i += kstep) {
          if (OUT) prefetch_l2(a.q + at * a.ldq + h * a.kd + i);
          prefetch_l2(a.k + at * a.ldk + h * a.kd + i);
        }
        for (int i = kc; i < vcols; i += kstep)
          prefetch_l2(a.v + at * a.ldv + h * a.vd + v0 + i);
      }
    }
    // The sum of this thread's results: not finite if one of them is not (or,
    // at no harm but time, if it overflows).
    float check = 0.f;
    const float keep = total == 0 ? pw[len - 1 + lead] * (1.f / kScoreScale) : 0.f;
    if constexpr (OUT) {
      // This warp's rows of q, split at their own scales.
      Frag q[NK];
      float sq[2];
      {
        float x[NK][8];
        const int r0 = rb + g, r1 = rb + g + 8;
        const float* p0 = a.q + (row + r0 * dir) * a.ldq + h * a.kd;
        const float* p1 = a.q + (row + r1 * dir) * a.ldq + h * a.kd;
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int col = k * 16 + half * 8 + 2 * c;
            float2 t0 = make_float2(0.f, 0.f), t1 = t0;
            if (a.vq) {
              if (r0 < len && col < a.kd) t0 = *reinterpret_cast<const float2*>(p0 + col);
              if (r1 < len && col < a.kd) t1 = *reinterpret_cast<const float2*>(p1 + col);
            } else {
              if (r0 < len && col < a.kd) t0.x = p0[col];
              if (r0 < len && col + 1 < a.kd) t0.y = p0[col + 1];
              if (r1 < len && col < a.kd) t1.x = p1[col];
              if (r1 < len && col + 1 < a.kd) t1.y = p1[col + 1];
            }
            x[k][half * 4] = t0.x, x[k][half * 4 + 1] = t0.y;
            x[k][half * 4 + 2] = t1.x, x[k][half * 4 + 3] = t1.y;
          }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t top = 0;
#pragma unroll
          for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              top = max(top, __float_as_uint(x[k][(e >> 1) * 4 + half * 2 + (e & 1)]) & 0x7fffffffu);
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          sq[half] = row_scale(row_exp(top));
          finite &= row_fits(top);
        }
        finite &= __syncthreads_count(lost >= la_rows(len)) < la_spare(len);
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            split2(x[k][2 * i] * sq[i & 1], x[k][2 * i + 1] * sq[i & 1], q[k].hi[i], q[k].lo[i]);
      }
      // c_i q_i S, then brought to the scale of the scores' product with v.
      float o[NV][4];
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int n = 0; n < NV; n += 2) {
          Frag s;
          s.load<true>(st_at + (k * 16 * LV + n * 8) * 2, T::kS);
          mma3(o[n], o[n + 1], q[k], s);
        }
      const int n0 = cnt[rb + g], n1 = cnt[rb + g + 8];
      // A row's scores are divided by `reach`.
      const float down0 = reach[rb + g], down1 = reach[rb + g + 8];
      const float up0 = pow2_inverse(down0), up1 = pow2_inverse(down1);
      {
        const float e0 = n0 == 0 ? pw[rb + g + lead] * (pow2_inverse(sst) * up0) : 0.f;
        const float e1 = n1 == 0 ? pw[rb + g + 8 + lead] * (pow2_inverse(sst) * up1) : 0.f;
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][e] *= e < 2 ? e0 : e1;
      }
      // Scores against the tokens up to this warp's last row, 16 at a time:
      // w_ij (q_i . k_j), then their product with v.
      const float* pi = pw + rb + g - 2 * c;
#pragma unroll 1
      for (int j0 = 0; j0 <= rb; j0 += 16) {
        // One accumulator a product: the chains of dependent instructions
        // are what this loop waits for (2060 cycles a turn with one for all
        // three, of which the products need 420).
        float p[2][4], p1[2][4], p2[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) p[n][e] = p1[n][e] = p2[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          Frag k;
          k.load<false>(k_at + (j0 * T::kLdK + kk * 16) * 2, T::kK);
          mma16(p[0], q[kk].hi, k.hi[0], k.hi[1]);
          mma16(p[1], q[kk].hi, k.hi[2], k.hi[3]);
          mma16(p1[0], q[kk].lo, k.hi[0], k.hi[1]);
          mma16(p1[1], q[kk].lo, k.hi[2], k.hi[3]);
          mma16(p2[0], q[kk].hi, k.lo[0], k.lo[1]);
          mma16(p2[1], q[kk].hi, k.lo[2], k.lo[3]);
        }
        // The table is zero before d^0, which leaves later tokens out.
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float* t = pi - j0 - n * 8;
          const float2 f = *reinterpret_cast<const float2*>(kf + j0 + n * 8 + 2 * c);
          p[n][0] = (p[n][0] + (p1[n][0] + p2[n][0])) * t[0] * f.x;
          p[n][1] = (p[n][1] + (p1[n][1] + p2[n][1])) * t[-1] * f.y;
          p[n][2] = (p[n][2] + (p1[n][2] + p2[n][2])) * t[8] * f.x;
          p[n][3] = (p[n][3] + (p1[n][3] + p2[n][3])) * t[7] * f.y;
        }
        if (total != 0) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int2 at = *reinterpret_cast<const int2*>(cnt + j0 + n * 8 + 2 * c);
            p[n][0] = at.x == n0 ? p[n][0] : 0.f;
            p[n][1] = at.y == n0 ? p[n][1] : 0.f;
            p[n][2] = at.x == n1 ? p[n][2] : 0.f;
            p[n][3] = at.y == n1 ? p[n][3] : 0.f;
          }
        }
        Frag f;
        split2(p[0][0], p[0][1], up0, f.hi[0], f.lo[0]);
        split2(p[0][2], p[0][3], up1, f.hi[1], f.lo[1]);
        split2(p[1][0], p[1][1], up0, f.hi[2], f.lo[2]);
        split2(p[1][2], p[1][3], up1, f.hi[3], f.lo[3]);
#pragma unroll
        for (int n = 0; n < NV; n += 2) {
          Frag v;
          v.load<true>(vt_at + (j0 * LV + n * 8) * 2, T::kV);
          mma3(o[n], o[n + 1], f, v);
        }
      }
      // In two steps: the inverses' product alone may be too small for float
      // where the sums that it scales are not.
      const float down_kv[2] = {down0, down1};
      const float down_q[2] = {a.scale * (1.f / kScoreScale) * pow2_inverse(sq[0]),
                               a.scale * (1.f / kScoreScale) * pow2_inverse(sq[1])};
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[n][e] = o[n][e] * down_kv[e >> 1] * down_q[e >> 1];
          check += o[n][e];
        }
      // Stored before it is known whether the chunk has to be done again.
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = rb + g + half * 8;
        if (i >= len) continue;
        float* to = a.o + (row + i * dir) * a.ldo + h * a.vd + v0;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          const int col = n * 8 + 2 * c;
          const float x0 = o[n][half * 2], x1 = o[n][half * 2 + 1];
          if (a.vo && col + 1 < vcols) {
            *reinterpret_cast<float2*>(to + col) = make_float2(x0, x1);
          } else {
            if (col < vcols) to[col] = x0;
            if (col + 1 < vcols) to[col + 1] = x1;
          }
        }
      }
    } else {
      finite &= __syncthreads_count(lost >= la_rows(len)) < la_spare(len);
    }
    // The state behind the chunk: this chunk's sum on its own, then one fp32
    // multiply and add.
    float nx[MT][NS][4];
    const float down = *sum_up;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) nx[m][n][e] = 0.f;
#pragma unroll
      for (int j = 0; j < kLaChunk; j += 16) {
        Frag f;
        f.load<true>(kt_at + (j * T::kLdK + m * 64) * 2, T::kK);
        // w_j k_j: joined, weighted and split again.
        const float2 w0 = *reinterpret_cast<const float2*>(wt + j + 2 * c);
        const float2 w1 = *reinterpret_cast<const float2*>(wt + j + 8 + 2 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 k = join2(f.hi[i], f.lo[i]);
          const float2 w = i < 2 ? w0 : w1;
          split2(k.x * w.x, k.y * w.y, f.hi[i], f.lo[i]);
        }
#pragma unroll
        for (int n = 0; n < NS; n += 2) {
          Frag v;
          v.load<true>(vt_at + (j * LV + sn + n * 8) * 2, T::kV);
          mma3(nx[m][n], nx[m][n + 1], f, v);
        }
      }
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          nx[m][n][e] = fmaf(keep, st[m][n][e], nx[m][n][e] * down);
          check += nx[m][n][e];
        }
    }
    finite &= isfinite(check);
    if (__syncthreads_or(!finite)) {
      // Token by token, with the state entering the chunk in shared memory in
      // fp32 (over its halves) and the operands as they are.
      each_state([&](float& held, int r, int col) { ss[r * LV + col] = held; });
      __syncthreads();
      la_exact<DK, DV, LV, kLaThreads, OUT>(a, ss, reinterpret_cast<float*>(la_smem), row, dir,
                                            len, lead, h, v0, vcols, decay,
                                            [&](int i) { return starts >> i & 1; });
      each_state([&](float& held, int r, int col) { held = ss[r * LV + col]; });
      continue;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[m][n][e] = nx[m][n][e];
  }

  float* to = nullptr;
  int tk = a.vd, tv = 1;
  float f = 1.f;
  if (!OUT) {
    to = a.seg + (static_cast<int64_t>(seg) * a.batch * a.heads) * a.kd * a.vd + mat;
    if (h == 0 && v0 == 0 && tid == 0)
      a.seg_start[static_cast<int64_t>(seg) * a.batch + b] = any_start;
  } else if (a.s_out != nullptr && a.segments == 1) {
    to = a.s_out + mat;
    tk = a.out_k;
    tv = a.out_v;
    if (a.reverse) f = a.starts != nullptr && a.starts[b] != 0.f ? 0.f : a.decay[h];
  }
  if (to == nullptr) return;
  each_state([&](float& held, int r, int col) {
    if (r < a.kd && v0 + col < a.vd)
      to[static_cast<int64_t>(r) * tk + static_cast<int64_t>(v0 + col) * tv] =
          f == 0.f ? 0.f : held * f;
  });
}

// ---------------------------------------------- the scan on tcgen05.mma
//
// The same scan in chunks of 128 tokens, one row of the tensor core's tile a
// token. The scores leave the tensor core in TMEM, are weighted there by the
// threads and go back in as halves, as the next product's operand; q, k, v and
// the state lie in shared memory, split, in the 128-byte swizzle that serves
// both orientations: k is read token by token for the scores and transposed
// for the state.
//
// Bound: the chain of a chunk: loads, scales and splits, the products (6,000
// cycles), weights and output. Two blocks an SM (keys of 64: 113 KB each) fill
// each other's waits, 16,000 cycles a chunk, at 49% of the issue slots and 24% of
// the tensor pipe; memory alone would allow 5,600. Keys of 128 leave room for one
// block, of 512 threads (256: 11% slower). Tried and not kept: k copied ahead
// to shared memory (the same at 64, 12% slower at 128), k ahead in registers
// (spills at 64, 2% at 128), v's and the state's splits behind the first
// product (the same).
constexpr int kTcChunk = 128;

template <int DK>
struct LaTc {
  // A slot is four floats: keys of 64 leave room for two blocks an SM, keys of
  // 128 for one, of twice the threads.
  static constexpr int kThreads = DK * 4, kWarps = kThreads / 32;
  static constexpr int kParts = kWarps / 4;      // of the 64 columns
  static constexpr int kQ = kTcChunk * DK * 2;   // bytes of a part; k alike
  static constexpr int kV = kTcChunk * 64 * 2;
  static constexpr int kS = DK * 64 * 2;
  static constexpr int kBlock = kTcChunk * 128;  // 64 columns of q or k
  static constexpr int kQ0 = 0, kK0 = 2 * kQ, kV0 = 4 * kQ, kS0 = kV0 + 2 * kV;
  static constexpr int kPw = kS0 + 2 * kS;       // d^0 .. d^128
  static constexpr int kMax = kPw + 528;         // [warps], of the state
  static constexpr int kMask = kMax + kWarps * 4;      // [4]
  static constexpr int kExp = kMask + 4 * 4;     // [128] exponents of q's rows
  // [128] tokens' sizes; where a thread's rows of k are not its rows of v, the
  // exponents that they come from.
  static constexpr bool kTwo = DK != 64;
  static constexpr int kSize = kExp + kTcChunk;
  static constexpr int kRows = kSize + kTcChunk;  // [k, v][128]
  static constexpr int kBar = kRows + (kTwo ? 2 * kTcChunk : 0);  // four
  static constexpr int kSlot = kBar + 32;
  static constexpr int kBytes = kSlot + 8;
  // With what the hardware keeps of each block: two blocks an SM, or one.
  static_assert((kBytes + 1024) * (DK == 64 ? 2 : 1) <= 228 * 1024, "shared memory");
};
// TMEM columns: scores (then their halves, hi and lo in turns of 16 columns),
// q S (then the chunk's sum for the state), scores v.
constexpr uint32_t kTcP = 0, kTcO1 = 128, kTcO2 = 192, kTcCols = 256;

// Instruction descriptor for 16-bit halves with an fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((static_cast<uint32_t>(n) >> 3) << 17) | ((static_cast<uint32_t>(m) >> 4) << 24);
}
__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The first operand in TMEM.
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
#define LA_R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), \
                    "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define LA_I8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), \
                    "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
// 32 columns of this thread's own row.
__device__ __forceinline__ void tmem_ld_row(uint32_t (&r)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LA_R8(r, 0), LA_R8(r, 8), LA_R8(r, 16), LA_R8(r, 24)
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_st_row(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::LA_I8(r, 0),
      LA_I8(r, 8), LA_I8(r, 16), LA_I8(r, 24), "r"(at)
      : "memory");
}
// 16 rows by 32 or 16 columns: register 4 n + e is row g + 8 (e >> 1), column
// 8 n + 2 c + (e & 1), for lane 4 g + c.
__device__ __forceinline__ void tmem_ld_frag(uint32_t (&r)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : LA_R8(r, 0), LA_R8(r, 8)
      : "r"(at)
      : "memory");
}

__device__ __forceinline__ void tmem_ld_frag(uint32_t (&r)[8], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LA_R8(r, 0)
      : "r"(at)
      : "memory");
}

// A tile of 128 tokens by D floats as load_tile has it, for THREADS threads.
template <int D, int THREADS>
__device__ __forceinline__ void tc_load(float (&x)[kTcChunk * D / (4 * THREADS)][4],
                                        const float* src, int64_t ld, int rows, int cols,
                                        int64_t first, int64_t step, bool vec) {
  constexpr int Q = D / 4, R = THREADS / Q, N = kTcChunk / R;
  const int r0 = threadIdx.x / Q, c = (threadIdx.x % Q) * 4;
  const float* p = src + (first + r0 * step) * ld + c;
  const int64_t jump = step * ld * R;
  if (vec) {
    const int last = c < cols ? rows - 1 - r0 : -1;  // the slots' rows up to here
#pragma unroll
    for (int u = 0; u < N; ++u, p += jump) {
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
      if (u * R <= last) t = *reinterpret_cast<const float4*>(p);
      x[u][0] = t.x, x[u][1] = t.y, x[u][2] = t.z, x[u][3] = t.w;
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < N; ++u, p += jump)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[u][e] = r0 + u * R < rows && c + e < cols ? p[e] : 0.f;
}
// Byte of this thread's first slot in a swizzled tile (slot u: u * R * 128 on).
template <int D>
__device__ __forceinline__ uint32_t tc_slot() {
  constexpr int Q = D / 4;
  const uint32_t r = threadIdx.x / Q, c = (threadIdx.x % Q) * 4;
  return (c >> 6) * (kTcChunk * 128) + r * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4) + (c & 7) * 2;
}
__device__ __forceinline__ void tc_put(uint32_t to, uint32_t part, const float (&x)[4],
                                       float scale) {
  uint32_t h0, h1, l0, l1;
  split2(x[0], x[1], scale, h0, l0);
  split2(x[2], x[3], scale, h1, l1);
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(h0), "r"(h1) : "memory");
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + part), "r"(l0), "r"(l1) : "memory");
}

// The largest magnitude of four, as bits. NaN is passed over: it reaches the
// results.
__device__ __forceinline__ uint32_t tc_max(const float (&x)[4]) {
  return __float_as_uint(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
}

template <int DK, int N>
__global__ void __launch_bounds__(LaTc<DK>::kThreads, DK == 64 ? 2 : 1)
    la_tc_kernel(const __grid_constant__ LaJobs<N> jobs) {
  using T = LaTc<DK>;
  const LaArgs& a = jobs.j[N == 1 ? 0 : blockIdx.z % jobs.n];
  constexpr int TH = T::kThreads, COLS = 64 / T::kParts, NC = COLS / 8;
  constexpr int MS = DK / 64;  // blocks of 16 rows of the state a warp owns, by COLS
  constexpr int NK = kTcChunk * DK / (4 * TH), RK = TH / (DK / 4);
  constexpr int NV = kTcChunk * 64 / (4 * TH), RV = TH / 16;
  extern __shared__ __align__(1024) uint8_t tc_smem[];
  float* ss = reinterpret_cast<float*>(tc_smem + T::kS0);  // the state in fp32, token by token
  const float* pw = reinterpret_cast<const float*>(tc_smem + T::kPw);  // kScoreScale d^n
  uint32_t* maxima = reinterpret_cast<uint32_t*>(tc_smem + T::kMax);
  uint32_t* mask = reinterpret_cast<uint32_t*>(tc_smem + T::kMask);
  int8_t* qexp = reinterpret_cast<int8_t*>(tc_smem + T::kExp);
  int8_t* kexp = reinterpret_cast<int8_t*>(tc_smem + T::kRows);
  uint8_t* size = tc_smem + T::kSize;
  // What a row's scores may add up to; over the state, when its product is done.
  float* reach = reinterpret_cast<float*>(tc_smem + T::kS0);
  const uint32_t sbase = smem_u32(tc_smem);
  const uint32_t bar = sbase + T::kBar;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int quarter = warp & 3, part = warp >> 2;  // of the rows, of the columns
  const int g = lane >> 2, c = lane & 3;
  const int bh = blockIdx.x, b = bh / a.heads, h = bh - b * a.heads;
  const int seg = blockIdx.y;
  const int v0 = (N == 1 ? blockIdx.z : blockIdx.z / jobs.n) * 64;
  const int vcols = min(64, a.vd - v0);
  if (vcols <= 0 || seg >= a.segments) return;  // fewer than another scan has
  // TMEM is taken before a later kernel's blocks may start, which could
  // otherwise hold what this one's wait for.
  if (warp == 0) {
    tmem_alloc(sbase + T::kSlot, kTcCols);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(bar + i * 8, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<const uint32_t*>(tc_smem + T::kSlot);
  const uint32_t my_rows = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  pdl_trigger();
  pdl_wait();
  const float decay = a.decay[h];
  if (tid <= kTcChunk)
    reinterpret_cast<float*>(tc_smem + T::kPw)[tid] = decay_pow(log2f(decay), tid) * kScoreScale;

  float st[MS][NC][4];
  const int64_t mat = static_cast<int64_t>(bh) * a.kd * a.vd;
  const float* from = nullptr;
  int fk = a.vd, fv = 1;
  if (seg > 0) {
    from = a.seg + mat +
           static_cast<int64_t>(seg * (a.seg_len / a.sum_len) - 1) * a.batch * a.heads * a.kd * a.vd;
  } else if (a.s_in != nullptr) {
    from = a.s_in + mat;
    fk = a.in_k;
    fv = a.in_v;
  }
  // f(held, row, column) over this thread's part of the state.
  auto each_state = [&](auto&& f) {
#pragma unroll
    for (int m = 0; m < MS; ++m)
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          f(st[m][n][e], (quarter * MS + m) * 16 + g + (e >> 1) * 8,
            part * COLS + n * 8 + 2 * c + (e & 1));
  };
  each_state([&](float& held, int r, int col) {
    held = from != nullptr && r < a.kd && v0 + col < a.vd
               ? from[static_cast<int64_t>(r) * fk + static_cast<int64_t>(v0 + col) * fv]
               : 0.f;
  });

  const int begin = seg * a.seg_len;
  const int end = min(a.steps, begin + a.seg_len);
  const int64_t dir = a.reverse ? -static_cast<int64_t>(a.batch) : a.batch;
  uint32_t phase = 0;
  bool dead = false;  // a wait ran out: the rest token by token
  // Fetched a chunk ahead, and not looked at before it is needed.
  float start = tid < min(kTcChunk, end - begin) ? la_start(a, begin + tid, b) : 0.f;
  for (int c0 = begin; c0 < end; c0 += kTcChunk) {
    const int len = min(kTcChunk, end - c0);
    const int lead = c0 == 0 && a.reverse ? 0 : 1;
    const int64_t row = static_cast<int64_t>(a.reverse ? a.steps - 1 - c0 : c0) * a.batch + b;
    float xv[NV][4];
    float sst;
    bool finite = true;  // and within what the halves hold
    int lost = 0;        // rows with values short of bits
    {
      float xk[NK][4];
      tc_load<DK, TH>(xk, a.k + h * a.kd, a.ldk, len, a.kd, row, dir, a.vk);
      tc_load<64, TH>(xv, a.v + h * a.vd + v0, a.ldv, len, vcols, row, dir, a.vv);
      const uint32_t flag = __ballot_sync(0xffffffffu, start != 0.f);
      if (warp < 4 && lane == 0) mask[warp] = flag;
      float most = 0.f;
      each_state([&](float& held, int, int) { most = fmaxf(most, fabsf(held)); });
      const uint32_t top_s = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
      if (lane == 0) maxima[warp] = top_s;
      int ek[NK];
#pragma unroll
      for (int u = 0; u < NK; ++u) {
        if (a.kscale != 1.f)
#pragma unroll
          for (int e = 0; e < 4; ++e) xk[u][e] *= a.kscale;
        const uint32_t top = row_max<DK / 4>(tc_max(xk[u]));
        ek[u] = row_exp(top);
        finite &= row_fits(top);
        lost += la_short(xk[u], ek[u]);
        tc_put(sbase + T::kK0 + tc_slot<DK>() + u * RK * 128, T::kQ, xk[u], row_scale(ek[u]));
        if (T::kTwo && tid % (DK / 4) == 0)
          kexp[tid / (DK / 4) + u * RK] = static_cast<int8_t>(ek[u]);
      }
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const uint32_t top = row_max<16>(tc_max(xv[u]));
        const int ev = row_exp(top);
        finite &= row_fits(top);
        lost += la_short(xv[u], ev);
        const float scale = row_scale(ev);
#pragma unroll
        for (int e = 0; e < 4; ++e) xv[u][e] *= scale;  // and so they stay
        tc_put(sbase + T::kV0 + tc_slot<64>() + u * RV * 128, T::kV, xv[u], 1.f);
        if (tid % 16 == 0) {
          const int r = tid / 16 + u * RV;
          if (T::kTwo)
            kexp[kTcChunk + r] = static_cast<int8_t>(ev);
          else
            size[r] = static_cast<uint8_t>(token_size(ek[u % NK], ev, finite));
        }
      }
    }
    __syncthreads();
    {
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < T::kWarps; w += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(maxima + w);
        top = max(top, max(max(x.x, x.y), max(x.z, x.w)));
      }
      sst = tile_scale(top);
      finite &= tile_fits(top);
    }
    if (T::kTwo && tid < kTcChunk)
      size[tid] = static_cast<uint8_t>(token_size(kexp[tid], kexp[kTcChunk + tid], finite));
    {
#pragma unroll
      for (int m = 0; m < MS; ++m)
#pragma unroll
        for (int n = 0; n < NC; ++n) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t hi, lo;
            split2(st[m][n][i * 2], st[m][n][i * 2 + 1], sst, hi, lo);
            const int r = (quarter * MS + m) * 16 + g + i * 8;
            uint8_t* to = tc_smem + T::kS0 + r * 128 + (((part * NC + n) ^ (r & 7)) << 4) + c * 4;
            *reinterpret_cast<uint32_t*>(to) = hi;
            *reinterpret_cast<uint32_t*>(to + T::kS) = lo;
          }
        }
    }
    const uint32_t starts[4] = {mask[0], mask[1], mask[2], mask[3]};
    {
      float xq[NK][4];
      tc_load<DK, TH>(xq, a.q + h * a.kd, a.ldq, len, a.kd, row, dir, a.vq);
      // A power of two for each row: a slot of a warp is one of 128 columns,
      // two of 64.
#pragma unroll
      for (int u = 0; u < NK; ++u) {
        const uint32_t top = row_max<DK / 4>(tc_max(xq[u]));
        const float sq = row_scale(row_exp(top));
        finite &= row_fits(top);
        if (tid % (DK / 4) == 0)
          qexp[tid / (DK / 4) + u * RK] =
              static_cast<int8_t>(static_cast<int>(__float_as_uint(sq) >> 23) - 127);
        tc_put(sbase + T::kQ0 + tc_slot<DK>() + u * RK * 128, T::kQ, xq[u], sq);
      }
    }
    fence_proxy_async_smem();
    tc_fence_before();
    finite &= __syncthreads_count(lost >= la_rows(len)) < la_spare(len);
    if (tid == 0 && !dead) {
      tc_fence_after();
      const uint64_t qd = umma_desc(sbase + T::kQ0, 16, 1024, kLayoutSw128);
      const uint64_t kd = umma_desc(sbase + T::kK0, 16, 1024, kLayoutSw128);
      const uint64_t sd = umma_desc(sbase + T::kS0, 16, 1024, kLayoutSw128);
#pragma unroll
      for (int p = 0; p < 3; ++p)  // small products first
#pragma unroll
        for (int s = 0; s < DK / 16; ++s) {
          const uint32_t at = (s >> 2) * T::kBlock + (s & 3) * 32;
          umma_f16(tmem + kTcP, qd + (((p == 0 ? T::kQ : 0) + at) >> 4),
                   kd + (((p == 1 ? T::kQ : 0) + at) >> 4), idesc_f16(128, 128, false, false),
                   p | s);
        }
      umma_commit(bar);
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int s = 0; s < DK / 16; ++s) {
          const uint32_t at = (s >> 2) * T::kBlock + (s & 3) * 32;
          umma_f16(tmem + kTcO1, qd + (((p == 0 ? T::kQ : 0) + at) >> 4),
                   sd + (((p == 1 ? T::kS : 0) + s * 2048) >> 4), idesc_f16(128, 64, false, true),
                   p | s);
        }
      umma_commit(bar + 8);
    }
    // The next chunk's rows on their way to L2.
    const int next = min(kTcChunk, end - c0 - kTcChunk);
    start = tid < next ? la_start(a, c0 + kTcChunk + tid, b) : 0.f;
    constexpr int LINES = TH / kTcChunk;  // threads of a row, a line of 32 floats each
    if (tid / LINES < next) {
      const int64_t at = row + (kTcChunk + tid / LINES) * dir;
      const int i = tid % LINES * 32;
      if (i < a.kd) {
        prefetch_l2(a.q + at * a.ldq + h * a.kd + i);
        prefetch_l2(a.k + at * a.ldk + h * a.kd + i);
      }
      if (i < vcols) prefetch_l2(a.v + at * a.ldv + h * a.vd + v0 + i);
    }
    // The first and the last token with a start, and this row's last.
    const uint32_t any = starts[0] | starts[1] | starts[2] | starts[3];
    int first = kTcChunk, last = -1, own = -1;
    if (any != 0) {
      uint32_t low = 0, high = 0, seen = 0;  // the words that hold them
      int at_low = 0, at_high = 0, at_seen = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (starts[3 - w] != 0) low = starts[3 - w], at_low = (3 - w) * 32;
        if (starts[w] != 0) high = starts[w], at_high = w * 32;
        const uint32_t upto =
            w < quarter ? starts[w] : w == quarter ? starts[w] & (0xffffffffu >> (31 - lane)) : 0u;
        if (upto != 0) seen = upto, at_seen = w * 32;
      }
      first = at_low + __ffs(low) - 1;
      last = at_high + 31 - __clz(high);
      if (seen != 0) own = at_seen + 31 - __clz(seen);
    }
    // While the products run: the largest token that this row sees, at its weight,
    // and the state's sum.
    float m, most;
    {
      uint32_t high = 0, low = 255;
      bool zeros = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t own_size = size[w * 32 + lane];
        high = max(high, own_size);
        low = min(low, own_size == 0 ? 255u : own_size);
        zeros |= own_size == 0 && w * 32 + lane < len;
      }
      high = __reduce_max_sync(0xffffffffu, high);
      low = __reduce_min_sync(0xffffffffu, zeros ? 0u : low);
      const int es = static_cast<int>(__float_as_uint(sst) >> 23) - 127;
      if (la_dwarfs(es, low)) {
        int few = 0;
#pragma unroll
        for (int i = 0; i < MS; ++i)
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            few += la_short(least2(st[i][n][0], st[i][n][1]), es);
            few += la_short(least2(st[i][n][2], st[i][n][3]), es);
          }
        if (few >= (a.kd > 8 && vcols > 8 ? 2 : 1)) finite = false;
      }
      m = most = size_float(high);
      if (high > low + kLaAlike) {
        most = 0.f;
        float carry = 0.f;
        int from = -1;  // the last start before this quarter
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (w < quarter && starts[w] != 0) from = w * 32 + 31 - __clz(starts[w]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int j = w * 32 + lane;
          const float f = size_float(size[j]);
          if (w == quarter) m = f;
          if (w < quarter && j >= from)
            carry = fmaxf(carry, f * (pw[quarter * 32 - j] * (1.f / kScoreScale)));
          if (j >= last && j < len) most = fmaxf(most, f * (pw[len - 1 - j] * (1.f / kScoreScale)));
        }
        carry = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(carry)));
        most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
        const int own_row = quarter * 32 + lane;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const float before = __shfl_up_sync(0xffffffffu, m, o);
          if (lane >= o && own_row - o >= own)
            m = fmaxf(m, before * (pw[o] * (1.f / kScoreScale)));
        }
        if (own < quarter * 32) m = fmaxf(m, carry * (pw[lane] * (1.f / kScoreScale)));
      }
    }
    const float down_row = pow2_above(m), up_row = pow2_inverse(down_row);
    const float down_sum = pow2_above(most);
    if (!dead && !mbar_wait(bar, phase)) dead = true;
    tc_fence_after();
    // w_ij (q_i . k_j) in blocks of 32 tokens, at the tokens' sizes, of what the
    // row may add up to.
#pragma unroll 1
    for (int j = part; j < 4; j += T::kParts) {
      uint32_t x[32];
      if (j > quarter) {
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = 0;
      } else {
        uint32_t y[32];
        tmem_ld_row(y, my_rows + kTcP + j * 32);
        const float* t = pw + (quarter - j) * 32 + lane;
        const uint4* sizes = reinterpret_cast<const uint4*>(size + j * 32);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint4 four = sizes[q];
          const uint32_t word[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int at = q * 16 + e;
            const uint32_t w = word[e >> 2];
            // Byte e & 3 as the exponent of a float.
            const uint32_t f = (e & 3) == 3 ? w >> 1 : w << (23 - 8 * (e & 3));
            y[at] = __float_as_uint(__uint_as_float(y[at]) * t[-at] *
                                    __uint_as_float(f & 0x7f800000u));
          }
        }
        // None from before the row's own start, none behind it.
        if (own > j * 32 || j == quarter) {
          uint32_t seen = j == quarter ? 0xffffffffu >> (31 - lane) : 0xffffffffu;
          if (own > j * 32) seen &= own < j * 32 + 32 ? 0xffffffffu << (own - j * 32) : 0u;
#pragma unroll
          for (int e = 0; e < 32; ++e) y[e] = seen >> e & 1 ? y[e] : 0;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
          split2(__uint_as_float(y[2 * e]), __uint_as_float(y[2 * e + 1]), up_row, x[e],
                 x[16 + e]);
      }
      tmem_st_row(my_rows + kTcP + j * 32, x);
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    if (!dead && !mbar_wait(bar + 8, phase)) dead = true;
    tc_fence_after();
    uint32_t o1[2][4 * NC];
#pragma unroll
    for (int m = 0; m < 2; ++m)
      tmem_ld_frag(o1[m], my_rows + (static_cast<uint32_t>(m * 16) << 16) + kTcO1 + part * COLS);
    // v with a token's weight in the state, where q was.
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int r = tid / 16 + u * RV;
      const float w =
          r >= last ? pw[max(len - 1 - r, 0)] * (1.f / kScoreScale) *
                          size_float(size[r]) * pow2_inverse(down_sum)
                    : 0.f;
      tc_put(sbase + T::kQ0 + tc_slot<64>() + u * RV * 128, T::kV, xv[u], w);
    }
    if (part == 0) reach[quarter * 32 + lane] = down_row;
    fence_proxy_async_smem();
    tc_fence_before();
    dead = __syncthreads_or(dead);
    if (tid == 0 && !dead) {
      tc_fence_after();
      const uint64_t vd = umma_desc(sbase + T::kV0, 16, 1024, kLayoutSw128);
      const uint64_t kd = umma_desc(sbase + T::kK0, T::kBlock, 1024, kLayoutSw128);
      const uint64_t wd = umma_desc(sbase + T::kQ0, 16, 1024, kLayoutSw128);
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int s = 0; s < kTcChunk / 16; ++s) {
          umma_f16_ts(tmem + kTcO2, tmem + kTcP + (s >> 1) * 32 + (p == 0 ? 16 : 0) + (s & 1) * 8,
                      vd + (((p == 1 ? T::kV : 0) + s * 2048) >> 4),
                      idesc_f16(128, 64, false, true), p | s);
        }
      umma_commit(bar + 16);
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int s = 0; s < kTcChunk / 16; ++s) {
          umma_f16(tmem + kTcO1, kd + (((p == 0 ? T::kQ : 0) + s * 2048) >> 4),
                   wd + (((p == 1 ? T::kV : 0) + s * 2048) >> 4), idesc_f16(DK, 64, true, true),
                   p | s);
        }
      umma_commit(bar + 24);
    }
    if (!dead && !mbar_wait(bar + 16, phase)) dead = true;
    tc_fence_after();
    // The sum of this thread's results: not finite if one of them is not (or,
    // at no harm but time, if it overflows).
    float check = 0.f;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      uint32_t o2[4 * NC];
      tmem_ld_frag(o2, my_rows + (static_cast<uint32_t>(m * 16) << 16) + kTcO2 + part * COLS);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = quarter * 32 + m * 16 + i * 8 + g;
        const float un = __uint_as_float(static_cast<uint32_t>(127 - qexp[r]) << 23) * a.scale *
                         (1.f / kScoreScale);
        // In two steps: a product of the inverses alone may be too small for
        // float where what they scale is not.
        const float e1 = r < first ? pw[r + lead] * pow2_inverse(sst) : 0.f;
        const float e2 = reach[r];
        float* to = a.o + (row + r * dir) * a.ldo + h * a.vd + v0;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          const float x0 = un * fmaf(e1, __uint_as_float(o1[m][n * 4 + i * 2]),
                                     e2 * __uint_as_float(o2[n * 4 + i * 2]));
          const float x1 = un * fmaf(e1, __uint_as_float(o1[m][n * 4 + i * 2 + 1]),
                                     e2 * __uint_as_float(o2[n * 4 + i * 2 + 1]));
          check += x0 + x1;
          // Stored before it is known whether the chunk has to be done again.
          const int col = part * COLS + n * 8 + 2 * c;
          if (r >= len) continue;
          if (a.vo && col + 1 < vcols) {
            *reinterpret_cast<float2*>(to + col) = make_float2(x0, x1);
          } else {
            if (col < vcols) to[col] = x0;
            if (col + 1 < vcols) to[col + 1] = x1;
          }
        }
      }
    }
    if (!dead && !mbar_wait(bar + 24, phase)) dead = true;
    if (!dead) phase ^= 1;
    tc_fence_after();
    const float keep = any == 0 ? pw[len - 1 + lead] * (1.f / kScoreScale) : 0.f;
    const float down = down_sum;
    float nx[MS][NC][4];
#pragma unroll
    for (int m = 0; m < MS; ++m) {
      uint32_t x[4 * NC];
      tmem_ld_frag(x, my_rows + (static_cast<uint32_t>(m * 16) << 16) + kTcO1 + part * COLS);
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          nx[m][n][e] = fmaf(keep, st[m][n][e], __uint_as_float(x[n * 4 + e]) * down);
          check += nx[m][n][e];
        }
    }
    finite &= static_cast<bool>(isfinite(check));
    tc_fence_before();
    if (__syncthreads_or(!finite || dead)) {
      dead = __syncthreads_or(dead);
      // Token by token, with the state entering the chunk in shared memory in
      // fp32 (over its halves) and the operands as they are.
      each_state([&](float& held, int r, int col) { ss[r * 64 + col] = held; });
      __syncthreads();
      la_exact<DK, 64, 64, TH, true>(a, ss, reinterpret_cast<float*>(tc_smem + T::kK0), row, dir,
                                     len, lead, h, v0, vcols, decay,
                                     [&](int i) { return mask[i >> 5] >> (i & 31) & 1; });
      each_state([&](float& held, int r, int col) { held = ss[r * 64 + col]; });
      continue;
    }
#pragma unroll
    for (int m = 0; m < MS; ++m)
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[m][n][e] = nx[m][n][e];
  }
  if (a.s_out != nullptr && a.segments == 1) {
    const float f = !a.reverse ? 1.f : a.starts != nullptr && a.starts[b] != 0.f ? 0.f : decay;
    each_state([&](float& held, int r, int col) {
      if (r < a.kd && v0 + col < a.vd)
        a.s_out[mat + static_cast<int64_t>(r) * a.out_k + static_cast<int64_t>(v0 + col) * a.out_v] =
            f == 0.f ? 0.f : held * f;
    });
  }
  // A wait that ran out left its products behind it: wait for them again, for
  // as long at most.
  for (int i = 0; dead && i < 4; ++i) mbar_wait(bar + i * 8, phase);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, kTcCols);
}

// The state behind each segment, from the sums in order; the last to s_out.
template <int N>
__global__ void __launch_bounds__(128) la_join_kernel(const __grid_constant__ LaJobs<N> jobs) {
  const LaArgs& a = jobs.j[N == 1 ? 0 : blockIdx.y];
  pdl_trigger();
  pdl_wait();
  const int64_t per = static_cast<int64_t>(a.kd) * a.vd;
  const int64_t all = per * a.batch * a.heads;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
  if (i >= all || a.segments == 1) return;
  const int bh = static_cast<int>(i / per), e = static_cast<int>(i - bh * per);
  const int b = bh / a.heads, h = bh - b * a.heads;
  const int r = e / a.vd, col = e - r * a.vd;
  const float lg = log2f(a.decay[h]);
  const int sub = a.seg_len / a.sum_len;
  const float full = decay_pow(lg, a.sum_len);
  float s = a.s_in != nullptr ? a.s_in[bh * per + static_cast<int64_t>(r) * a.in_k +
                                       static_cast<int64_t>(col) * a.in_v]
                              : 0.f;
  constexpr int kAhead = 8;  // loads in flight
  for (int q0 = 0; q0 < a.sums; q0 += kAhead) {
    float own[kAhead];
    int cut[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool in = q0 + u < a.sums;
      own[u] = in ? a.seg[(q0 + u) * all + i] : 0.f;
      cut[u] = in ? a.seg_start[static_cast<int64_t>(q0 + u) * a.batch + b] : 0;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int q = q0 + u;
      if (q >= a.sums) break;
      float f = full;
      const int len = min(a.sum_len, a.steps - q * a.sum_len);
      if (q == 0 && a.reverse) f = decay_pow(lg, len - 1);
      else if (len < a.sum_len) f = decay_pow(lg, len);
      // A power that float cannot hold is no zero to an infinite state.
      if (f == 0.f && a.decay[h] > 0.f && isinf(s)) f = 1.f;
      s = cut[u] ? own[u] : fmaf(f, s, own[u]);
      if ((q + 1) % sub == 0) a.seg[q * all + i] = s;
    }
  }
  if (a.s_out != nullptr) {
    if (a.reverse) s = a.starts != nullptr && a.starts[b] != 0.f ? 0.f : s * a.decay[h];
    a.s_out[bh * per + static_cast<int64_t>(r) * a.out_k + static_cast<int64_t>(col) * a.out_v] =
        s;
  }
}

// --------------------------------------------------------- a single token

struct LaStepArgs {
  const float* qkv;    // [batch] rows of [q | k | v]
  const float* s_in;   // [batch][heads][K][V]
  float* s_out;        // (may be s_in)
  const float* starts; // [batch] or null
  const float* decay;
  float* out;          // [batch][heads * V]
  int32_t batch, heads, kd, vd;
  int32_t cols;        // column slots: vd / W
  float scale;
};

constexpr int kLaStepThreads = 256;

// One block a lane and head: reads the state once and writes it once (8 K V
// bytes, all that counts), 16 bytes a thread and access where W = 4. A thread
// keeps its columns and walks the rows, so the output's sum over the rows
// needs one exchange at the end.
template <int W>
__global__ void __launch_bounds__(kLaStepThreads) la_step_kernel(const __grid_constant__ LaStepArgs a) {
  __shared__ float sk[128], sq[128];
  __shared__ __align__(16) float red[kLaStepThreads * W];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x;
  const int bh = blockIdx.x, b = bh / a.heads, h = bh - b * a.heads;
  const float* row = a.qkv + static_cast<int64_t>(b) * a.heads * (2 * a.kd + a.vd);
  for (int i = tid; i < a.kd; i += kLaStepThreads) {
    sq[i] = row[h * a.kd + i];
    sk[i] = row[a.heads * a.kd + h * a.kd + i];
  }
  const int groups = kLaStepThreads / a.cols;
  const int col = tid % a.cols, grp = tid / a.cols;
  const bool mine = grp < groups;
  const bool drop = a.starts != nullptr && a.starts[b] != 0.f;
  const float d = a.decay[h];
  const int64_t mat = static_cast<int64_t>(bh) * a.kd * a.vd;
  float v[W], sum[W];
#pragma unroll
  for (int e = 0; e < W; ++e) {
    v[e] = mine ? row[2 * a.heads * a.kd + h * a.vd + col * W + e] : 0.f;
    sum[e] = 0.f;
  }
  __syncthreads();
  if (mine) {
    constexpr int U = 4;
    for (int r0 = grp; r0 < a.kd; r0 += U * groups) {
      float s[U][W];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * groups;
#pragma unroll
        for (int e = 0; e < W; ++e) s[u][e] = 0.f;
        if (r < a.kd && !drop) {
          const float* p = a.s_in + mat + static_cast<int64_t>(r) * a.vd + col * W;
          if (W == 4) {
            const float4 t = *reinterpret_cast<const float4*>(p);
            s[u][0] = t.x, s[u][W > 1 ? 1 : 0] = t.y, s[u][W > 2 ? 2 : 0] = t.z,
            s[u][W > 3 ? 3 : 0] = t.w;
          } else {
            s[u][0] = *p;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * groups;
        if (r >= a.kd) continue;
        const float k = sk[r], q = sq[r];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          s[u][e] = fmaf(k, v[e], drop ? 0.f : s[u][e] * d);
          sum[e] = fmaf(q, s[u][e], sum[e]);
        }
        float* p = a.s_out + mat + static_cast<int64_t>(r) * a.vd + col * W;
        if (W == 4)
          *reinterpret_cast<float4*>(p) =
              make_float4(s[u][0], s[u][W > 1 ? 1 : 0], s[u][W > 2 ? 2 : 0], s[u][W > 3 ? 3 : 0]);
        else
          *p = s[u][0];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < W; ++e) red[tid * W + e] = sum[e];
  __syncthreads();
  for (int i = tid; i < a.vd; i += kLaStepThreads) {
    float t = 0.f;
    for (int q = 0; q < groups; ++q) t += red[q * a.cols * W + i];
    a.out[static_cast<int64_t>(b) * a.heads * a.vd + h * a.vd + i] = t * a.scale;
  }
}

// ------------------------------------------------------------------ host

constexpr int kLaMaxDim = 128;
constexpr int kLaSms = 148;

static int la_pad_k(int kd) { return kd <= 32 ? 32 : kd <= 64 ? 64 : 128; }
// Columns of v a block takes: 64 (two blocks for up to 128). Beside a key of
// 128 that leaves room for two blocks an SM, where 32 columns leave it for
// three, but the scores are computed half as often: 2048 x 8 lanes x 8 heads
// of 128 x 128 in 399 us against 424, the backward in 1209 against 1350.
static int la_pad_v(int vd) { return vd <= 32 ? 32 : 64; }

// The scan that writes results takes the tcgen05 form where its tiles of 128
// tokens and 64 columns are not mostly empty. Times of 64 lanes x 8 heads on
// mma.sync and on tcgen05 in us:
//   64 tokens, 64/64: 24, 33; 65: 39, 33; 128: 44, 36; 1024: 296, 236
//   1024 tokens, key 64, value 32: 190, 226; 128/32: 460, 336;
//   2048 x 8 lanes, 128/128: 426, 168
static bool la_tc(const LaArgs& a) {
  return a.steps > 64 && (a.kd > 64 || (a.kd > 32 && a.vd > 32));
}

// Segments of a scan, one of `jobs`: enough blocks for the SMs' places, each at
// least two chunks long.
static void la_segments(LaArgs& a, int jobs) {
  const int dv = la_pad_v(a.vd);
  const long long blocks =
      static_cast<long long>(a.batch) * a.heads * ((a.vd + dv - 1) / dv) * jobs;
  const bool tc = la_tc(a);
  const int places = kLaSms * (tc ? a.kd <= 64 ? 2 : 1 : a.kd <= 64 ? 4 : dv == 64 ? 2 : 3);
  const int unit = tc ? kTcChunk : kLaChunk;
  a.segments = a.sums = 1;
  a.seg_len = a.sum_len = a.steps;
  if (blocks * 2 > places) return;
  const long long chunks = (a.steps + unit - 1) / unit;
  const long long want = std::min<long long>(places / blocks, chunks / 2);
  if (want < 2) return;
  const long long per = (chunks + want - 1) / want;
  a.seg_len = static_cast<int>(per * unit);
  a.segments = (a.steps + a.seg_len - 1) / a.seg_len;
  // The sums are the smaller blocks' work: parts of a segment, as many as find
  // a place, of two chunks at least.
  const int rooms = kLaSms * (a.kd <= 64 ? 4 : dv == 64 ? 2 : 3);
  int sub = 1;
  while (a.seg_len % (4 * sub * kLaChunk) == 0 && blocks * a.segments * sub * 2 <= rooms) sub *= 2;
  a.sum_len = a.seg_len / sub;
  a.sums = (a.steps + a.sum_len - 1) / a.sum_len;
}

static size_t la_seg_floats(const LaArgs& a) {
  if (a.segments == 1) return 0;
  return a.sums * (static_cast<size_t>(a.batch) * a.heads * a.kd * a.vd + a.batch);
}
static size_t la_scan_ws(LaArgs* jobs, int n) {
  size_t floats = 0;
  for (int i = 0; i < n; ++i) {
    la_segments(jobs[i], n);
    floats += la_seg_floats(jobs[i]);
  }
  return floats * sizeof(float);
}

// One kernel's launch, its shared memory allowed once a device.
template <typename Tag, int N>
static cudaError_t la_launch(void (*kernel)(LaJobs<N>), int bytes, int threads, int columns,
                             const LaJobs<N>& jobs, bool sums, cudaStream_t st) {
  static std::mutex lock;
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    std::lock_guard<std::mutex> hold(lock);
    if (dev < 0 || dev >= 64 || !ready[dev]) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (e != cudaSuccess) return e;
      if (dev >= 0 && dev < 64) ready[dev] = true;
    }
  }
  int segments = 1, wide = 1;
  for (int i = 0; i < jobs.n; ++i) {
    const LaArgs& a = jobs.j[i];
    segments = std::max(segments, sums ? a.sums : a.segments);
    wide = std::max(wide, (a.vd + columns - 1) / columns);
  }
  note_launch();
  return launch_pdl(kernel,
                    dim3(static_cast<unsigned>(jobs.j[0].batch) * jobs.j[0].heads, segments,
                         wide * jobs.n),
                    dim3(threads), bytes, st, jobs);
}
template <int DK, int DV, bool OUT, int N>
static cudaError_t la_scan_launch(const LaJobs<N>& jobs, cudaStream_t st) {
  struct Tag {};
  return la_launch<Tag>(la_scan_kernel<DK, DV, OUT, N>, LaTile<DK, DV>::kBytes, kLaThreads, DV, jobs,
                        !OUT, st);
}
template <int DK, int N>
static cudaError_t la_tc_launch(const LaJobs<N>& jobs, cudaStream_t st) {
  struct Tag {};
  return la_launch<Tag>(la_tc_kernel<DK, N>, LaTc<DK>::kBytes, LaTc<DK>::kThreads, 64, jobs, false, st);
}

template <bool OUT, int N>
static cudaError_t la_pick(const LaJobs<N>& jobs, cudaStream_t st) {
  const LaArgs& a = jobs.j[0];
  const int dk = la_pad_k(a.kd), dv = la_pad_v(a.vd);
  if (OUT && la_tc(a)) return dk == 64 ? la_tc_launch<64>(jobs, st) : la_tc_launch<128>(jobs, st);
  if (dv == 32)
    return dk == 32   ? la_scan_launch<32, 32, OUT>(jobs, st)
           : dk == 64 ? la_scan_launch<64, 32, OUT>(jobs, st)
                      : la_scan_launch<128, 32, OUT>(jobs, st);
  return dk == 32   ? la_scan_launch<32, 64, OUT>(jobs, st)
         : dk == 64 ? la_scan_launch<64, 64, OUT>(jobs, st)
                    : la_scan_launch<128, 64, OUT>(jobs, st);
}

static bool la_vec(const float* p, int64_t ld, int width) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 4 == 0 && width % 4 == 0;
}

// Scans that take the same kernel.
static bool la_alike(const LaArgs& x, const LaArgs& y) {
  return la_pad_k(x.kd) == la_pad_k(y.kd) && la_pad_v(x.vd) == la_pad_v(y.vd) &&
         la_tc(x) == la_tc(y);
}

// n scans that take the same kernel.
template <int N>
static cudaError_t la_scan(LaArgs* scans, int n, char* ws, cudaStream_t st) {
  LaJobs<N> jobs;
  std::memset(&jobs, 0, sizeof(jobs));
  jobs.n = n;
  bool split = false;
  float* room = reinterpret_cast<float*>(ws);
  for (int i = 0; i < n; ++i) {
    LaArgs& a = scans[i];
    a.vq = la_vec(a.q, a.ldq, a.kd);
    a.vk = la_vec(a.k, a.ldk, a.kd);
    a.vv = la_vec(a.v, a.ldv, a.vd);
    a.vo = (reinterpret_cast<uintptr_t>(a.o) & 7u) == 0 && a.ldo % 2 == 0 && a.vd % 2 == 0;
    la_segments(a, n);
    if (a.segments > 1) {
      split = true;
      a.seg = room;
      a.seg_start = reinterpret_cast<int*>(room + la_seg_floats(a)) -
                    static_cast<size_t>(a.sums) * a.batch;
      room += la_seg_floats(a);
    }
    jobs.j[i] = a;
  }
  if (split) {
    cudaError_t e = la_pick<false>(jobs, st);
    if (e != cudaSuccess) return e;
    const int64_t all = static_cast<int64_t>(jobs.j[0].batch) * jobs.j[0].heads * jobs.j[0].kd *
                        jobs.j[0].vd;
    note_launch();
    e = launch_pdl(la_join_kernel<N>, dim3(static_cast<unsigned>((all + 127) / 128), n), dim3(128),
                   0, st, jobs);
    if (e != cudaSuccess) return e;
  }
  return la_pick<true>(jobs, st);
}

static int la_check(const char* what, int steps, int batch, int heads, int kd, int vd) {
  if (steps < 1 || batch < 0 || heads < 1 || kd < 1 || vd < 1)
    return set_error(TTRL_EINVAL, "%s: bad extents (steps %d, batch %d, heads %d, key %d, value %d)",
                     what, steps, batch, heads, kd, vd);
  if (steps > (1 << 30))
    return set_error(TTRL_EUNSUPPORTED, "%s: more than 2^30 steps", what);
  if (kd > kLaMaxDim || vd > kLaMaxDim)
    return set_error(TTRL_EUNSUPPORTED, "%s: key and value widths up to %d, got %d and %d", what,
                     kLaMaxDim, kd, vd);
  if (static_cast<long long>(batch) * heads * kd * vd >= (1ll << 39) ||
      static_cast<long long>(batch) * heads >= (1ll << 31))
    return set_error(TTRL_EUNSUPPORTED, "%s: too many lanes and heads", what);
  // A head's place in its row is a 32-bit number.
  if (static_cast<long long>(heads) * (2 * kd + vd) >= (1ll << 31))
    return set_error(TTRL_EUNSUPPORTED, "%s: a row of 2^31 values or more", what);
  return TTRL_OK;
}

static LaArgs la_args(int steps, int batch, int heads, int kd, int vd, const float* starts,
                      const float* decay) {
  LaArgs a;
  std::memset(&a, 0, sizeof(a));
  a.steps = steps;
  a.batch = batch;
  a.heads = heads;
  a.kd = kd;
  a.vd = vd;
  a.starts = starts;
  a.decay = decay;
  a.scale = 1.f;
  a.kscale = 1.f;
  return a;
}

// The backward's scans, without their operands: dq, dk, then dv; the first
// two always take the same kernel.
static void la_backward(LaArgs (&scan)[3], int steps, int batch, int heads, int kd, int vd,
                        const float* starts, const float* decay) {
  scan[0] = la_args(steps, batch, heads, vd, kd, starts, decay);
  scan[1] = la_args(steps, batch, heads, vd, kd, starts, decay);
  scan[2] = la_args(steps, batch, heads, kd, vd, starts, decay);
}

size_t linear_attention_ws(int steps, int batch, int heads, int kd, int vd) {
  if (la_check("linear_attention", steps, batch, heads, kd, vd) != TTRL_OK || batch == 0) return 0;
  LaArgs one = la_args(steps, batch, heads, kd, vd, nullptr, nullptr);
  LaArgs scan[3];
  la_backward(scan, steps, batch, heads, kd, vd, nullptr, nullptr);
  const size_t forward = la_scan_ws(&one, 1);
  const size_t backward = la_alike(scan[0], scan[2])
                              ? la_scan_ws(scan, 3)
                              : std::max(la_scan_ws(scan, 2), la_scan_ws(scan + 2, 1));
  return kCounterBytes + std::max(forward, backward);
}

static int la_workspace(const char* what, int steps, int batch, int heads, int kd, int vd, void* ws,
                        size_t bytes, char** out) {
  const size_t need = linear_attention_ws(steps, batch, heads, kd, vd);
  *out = nullptr;
  if (need == kCounterBytes) return TTRL_OK;
  if (ws == nullptr || bytes < need)
    return set_error(TTRL_EWORKSPACE, "%s: needs %zu bytes of workspace, got %zu", what, need,
                     ws == nullptr ? static_cast<size_t>(0) : bytes);
  if (reinterpret_cast<uintptr_t>(ws) & 15u)
    return set_error(TTRL_EINVAL, "%s: the workspace has to start on a 16-byte boundary", what);
  *out = static_cast<char*>(ws) + kCounterBytes;
  return TTRL_OK;
}

int linear_attention_step(const float* qkv, const float* s_in, const float* starts,
                          const float* decay, float* out, float* s_out, int batch, int heads,
                          int kd, int vd, float scale, cudaStream_t st) {
  int rc = la_check("linear_attention_step", 1, batch, heads, kd, vd);
  if (rc) return rc;
  if (batch == 0) return TTRL_OK;
  if (!qkv || !s_in || !decay || !out || !s_out)
    return set_error(TTRL_EINVAL, "linear_attention_step: null pointer");
  const int64_t state = static_cast<int64_t>(batch) * heads * kd * vd;
  const Span in[] = {{"qkv", qkv, static_cast<int64_t>(batch) * heads * (2 * kd + vd)},
                       {"state", s_out == s_in ? nullptr : s_in, state},
                       {"starts", starts, batch},
                       {"decay", decay, heads}};
  const Span made[] = {{"out", out, static_cast<int64_t>(batch) * heads * vd},
                         {"new_state", s_out, state}};
  if ((rc = spans_apart("linear_attention_step", in, made))) return rc;
  LaStepArgs a;
  std::memset(&a, 0, sizeof(a));
  a.qkv = qkv;
  a.s_in = s_in;
  a.s_out = s_out;
  a.starts = starts;
  a.decay = decay;
  a.out = out;
  a.batch = batch;
  a.heads = heads;
  a.kd = kd;
  a.vd = vd;
  a.scale = scale;
  const bool vec = vd % 4 == 0 && ((reinterpret_cast<uintptr_t>(s_in) |
                                    reinterpret_cast<uintptr_t>(s_out)) & 15u) == 0;
  a.cols = vec ? vd / 4 : vd;
  note_launch();
  const dim3 grid(static_cast<unsigned>(batch) * heads);
  const cudaError_t e =
      vec ? launch_pdl(la_step_kernel<4>, grid, dim3(kLaStepThreads), 0, st, a)
          : launch_pdl(la_step_kernel<1>, grid, dim3(kLaStepThreads), 0, st, a);
  return e == cudaSuccess ? TTRL_OK : set_cuda_error("linear_attention_step launch", e);
}

int linear_attention_fwd(const float* qkv, const float* s_in, const float* starts,
                         const float* decay, float* out, float* s_out, int steps, int batch,
                         int heads, int kd, int vd, float scale, void* ws, size_t ws_bytes,
                         cudaStream_t st) {
  int rc = la_check("linear_attention_fwd", steps, batch, heads, kd, vd);
  if (rc) return rc;
  if (batch == 0) return TTRL_OK;
  if (!qkv || !decay || !out)
    return set_error(TTRL_EINVAL, "linear_attention_fwd: null pointer");
  const int64_t rows = static_cast<int64_t>(steps) * batch;
  const int64_t state = static_cast<int64_t>(batch) * heads * kd * vd;
  // Results are written while other blocks, and the scans that follow, still
  // read what came in.
  const Span in[] = {{"qkv", qkv, rows * heads * (2 * kd + vd)},
                     {"state", s_in, state},
                     {"starts", starts, rows},
                     {"decay", decay, heads}};
  const Span made[] = {{"out", out, rows * heads * vd}, {"new_state", s_out, state}};
  char* room = nullptr;
  if ((rc = la_workspace("linear_attention_fwd", steps, batch, heads, kd, vd, ws, ws_bytes, &room)))
    return rc;
  if ((rc = spans_apart("linear_attention_fwd", in, made))) return rc;
  LaArgs a = la_args(steps, batch, heads, kd, vd, starts, decay);
  const int64_t ld = static_cast<int64_t>(heads) * (2 * kd + vd);
  a.q = qkv;
  a.k = qkv + static_cast<int64_t>(heads) * kd;
  a.v = qkv + 2 * static_cast<int64_t>(heads) * kd;
  a.o = out;
  a.ldq = a.ldk = a.ldv = ld;
  a.ldo = static_cast<int64_t>(heads) * vd;
  a.s_in = s_in;
  a.s_out = s_out;
  a.in_k = a.out_k = vd;
  a.in_v = a.out_v = 1;
  a.scale = scale;
  const cudaError_t e = la_scan<1>(&a, 1, room, st);
  return e == cudaSuccess ? TTRL_OK : set_cuda_error("linear_attention_fwd launch", e);
}

int linear_attention_bwd(const float* dout, const float* ds_out, const float* qkv,
                         const float* s_in, const float* starts, const float* decay, float* dqkv,
                         float* ds_in, int steps, int batch, int heads, int kd, int vd,
                         float scale, void* ws, size_t ws_bytes, cudaStream_t st) {
  int rc = la_check("linear_attention_bwd", steps, batch, heads, kd, vd);
  if (rc) return rc;
  if (batch == 0) return TTRL_OK;
  if (!dout || !qkv || !decay || !dqkv)
    return set_error(TTRL_EINVAL, "linear_attention_bwd: null pointer");
  const int64_t rows = static_cast<int64_t>(steps) * batch;
  const int64_t state = static_cast<int64_t>(batch) * heads * kd * vd;
  const Span in[] = {{"qkv", qkv, rows * heads * (2 * kd + vd)},
                       {"state", s_in, state},
                       {"dout", dout, rows * heads * vd},
                       {"dnew_state", ds_out, state},
                       {"starts", starts, rows},
                       {"decay", decay, heads}};
  const Span made[] = {{"dqkv", dqkv, rows * heads * (2 * kd + vd)}, {"dstate", ds_in, state}};
  char* room = nullptr;
  if ((rc = la_workspace("linear_attention_bwd", steps, batch, heads, kd, vd, ws, ws_bytes, &room)))
    return rc;
  if ((rc = spans_apart("linear_attention_bwd", in, made))) return rc;
  const int64_t ld = static_cast<int64_t>(heads) * (2 * kd + vd);
  const int64_t ldo = static_cast<int64_t>(heads) * vd;
  const float* q = qkv;
  const float* k = qkv + static_cast<int64_t>(heads) * kd;
  const float* v = qkv + 2 * static_cast<int64_t>(heads) * kd;
  float* dq = dqkv;
  float* dk = dqkv + static_cast<int64_t>(heads) * kd;
  float* dv = dqkv + 2 * static_cast<int64_t>(heads) * kd;
  LaArgs scan[3];
  la_backward(scan, steps, batch, heads, kd, vd, starts, decay);
  {
    // dq = scale do S^T: forward in time, with S^T for its state.
    LaArgs& a = scan[0];
    a.q = dout;
    a.ldq = ldo;
    a.k = v;
    a.v = k;
    a.ldk = a.ldv = ld;
    a.o = dq;
    a.ldo = ld;
    a.s_in = s_in;
    a.in_k = 1;
    a.in_v = vd;
    a.scale = scale;
  }
  {
    // dk = v R^T with R summing scale q do^T, backwards in time.
    LaArgs& a = scan[1];
    a.reverse = 1;
    a.q = v;
    a.ldq = ld;
    a.k = dout;
    a.ldk = ldo;
    a.v = q;
    a.ldv = ld;
    a.o = dk;
    a.ldo = ld;
    a.s_in = ds_out;
    a.in_k = 1;
    a.in_v = vd;
    a.kscale = scale;
  }
  {
    // dv = k R; what it leaves is the gradient of the entering state.
    LaArgs& a = scan[2];
    a.reverse = 1;
    a.q = k;
    a.ldq = ld;
    a.k = q;
    a.ldk = ld;
    a.v = dout;
    a.ldv = ldo;
    a.o = dv;
    a.ldo = ld;
    a.s_in = ds_out;
    a.s_out = ds_in;
    a.in_k = a.out_k = vd;
    a.in_v = a.out_v = 1;
    a.kscale = scale;
  }
  cudaError_t e;
  if (la_alike(scan[0], scan[2])) {
    e = la_scan<3>(scan, 3, room, st);
  } else {
    e = la_scan<3>(scan, 2, room, st);
    if (e == cudaSuccess) e = la_scan<1>(scan + 2, 1, room, st);
  }
  return e == cudaSuccess ? TTRL_OK : set_cuda_error("linear_attention_bwd launch", e);
}

}  // namespace ttrl

using namespace ttrl;

extern "C" {

size_t ttrl_linear_attention_workspace_bytes(int steps, int batch, int heads, int key_dim,
                                             int value_dim) {
  return linear_attention_ws(steps, batch, heads, key_dim, value_dim);
}

int ttrl_linear_attention_fwd(const float* qkv, const float* state, const float* starts,
                              const float* decay, float* out, float* new_state, int steps,
                              int batch, int heads, int key_dim, int value_dim, float scale,
                              void* workspace, size_t workspace_bytes, ttrl_stream_t stream) {
  return linear_attention_fwd(qkv, state, starts, decay, out, new_state, steps, batch, heads,
                              key_dim, value_dim, scale, workspace, workspace_bytes,
                              static_cast<cudaStream_t>(stream));
}

int ttrl_linear_attention_bwd(const float* dout, const float* dnew_state, const float* qkv,
                              const float* state, const float* starts, const float* decay,
                              float* dqkv, float* dstate, int steps, int batch, int heads,
                              int key_dim, int value_dim, float scale, void* workspace,
                              size_t workspace_bytes, ttrl_stream_t stream) {
  return linear_attention_bwd(dout, dnew_state, qkv, state, starts, decay, dqkv, dstate, steps,
                              batch, heads, key_dim, value_dim, scale, workspace,
                              workspace_bytes, static_cast<cudaStream_t>(stream));
}

int ttrl_linear_attention_step(const float* qkv, const float* state, const float* starts,
                               const float* decay, float* out, float* new_state, int batch,
                               int heads, int key_dim, int value_dim, float scale,
                               ttrl_stream_t stream) {
  return linear_attention_step(qkv, state, starts, decay, out, new_state, batch, heads, key_dim,
                               value_dim, scale, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
