// Rows to 8 bits on the way into a matrix product:
//   dsmoe_rms_norm_quant   r = round(x + residual);  v = r / sqrt(mean(r^2) + eps) * w
//   dsmoe_swiglu_quant     v = silu(min(g, limit)) * clamp(u, -limit, limit) [* row weight]
// followed by the quantization of v in the same pass, in one of two forms:
//   e4m3   one fp32 scale per 128 values, s = max(amax, 1e-4) / 448, q = e4m3(v / s)  (act_quant's rule;
//          with pow2 the scale is its power-of-2 ceiling)
//   int8   one fp32 scale per row, s = max(amax, 1e-4) / 127, q = rint(v / s)
//
// Both are bound by memory: every input byte is read once and every output byte written once, the row
// stays in registers between. The norm needs two values of the whole row, sum(r^2) and (int8)
// max|r w|: since amax(v) = max|r w| / sqrt(..), both come out of one block reduction, so a row costs
// one barrier. r is the rounded residual (what the next layer adds to), sums and products are fp32.
// Measured: 4096 rows of 5120 bf16 with residual, codes, scales and normed rows 32.7 us (5.8 TB/s; a copy of those bytes
// 28.9), one row 2.4 to 2.6 us (a launch); swiglu of 12282 rows of 2 x 2048 bf16 24.4 us to e4m3 (5.2 TB/s; 19.3), 26.5 to int8:
// about 22 instructions a value keep the issue slots two thirds busy. Rows that are not a multiple of 16 bytes cost
// shifts and masks: swiglu of 6000 x 2049 to int8 22.4 us (2.7 TB/s), norm of 4000 x 6387 with residual 50.0 (3.6).
// Scales that are not finite are NaN, so that the values read back as NaN: those of a norm's row that holds an infinity
// or NaN or whose squares overflow fp32, and of a swiglu's row (e4m3: block) whose amax is not finite.
#include "common.cuh"

namespace dsmoe {
namespace rows8 {

constexpr float kAmaxFloor = 1e-4f;
constexpr int kMaxHidden = 16384;

struct Args {
  const void* x;      // norm: [rows][n]; swiglu: [rows][2n] (g | u)
  const void* res;    // norm: [rows][n] or null
  const void* w;      // norm: [n] fp32 or bf16; swiglu: [rows] fp32 row weight or null
  void* q;            // [rows][n] 8-bit
  float* s;           // e4m3: [rows][n / 128]; int8: [rows]
  void* res_out;      // norm: [rows][n] or null
  void* normed;       // norm: [rows][n] or null
  long long rows;
  int n;              // values per row
  int tpr, rpc;       // threads per row (a multiple of 32), rows per CTA
  int w_bf16, pow2;
  float eps, limit;
};

// VEC values (16 bytes) as loaded; bf16 stays packed in registers until it is used.
template <typename T>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  // the first n values of p alone
  __device__ __forceinline__ void load_first(const __nv_bfloat16* p, int n) {
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) w[i >> 1] |= (uint32_t)h[i] << (16 * (i & 1));
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
  // values s.. of this chunk followed by the next one's (0 <= s < 8, the same in every lane of a row)
  __device__ __forceinline__ void shift_in(const Raw& next, int s) {
    const uint4 n = next.u;
    switch (s >> 1) {
      case 0: words(u.x, u.y, u.z, u.w, n.x, s); break;
      case 1: words(u.y, u.z, u.w, n.x, n.y, s); break;
      case 2: words(u.z, u.w, n.x, n.y, n.z, s); break;
      default: words(u.w, n.x, n.y, n.z, n.w, s); break;
    }
  }
  __device__ __forceinline__ void words(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, int s) {
    const int half = (s & 1) * 16;
    u = make_uint4(__funnelshift_r(a, b, half), __funnelshift_r(b, c, half), __funnelshift_r(c, d, half),
                   __funnelshift_r(d, e, half));
  }
  __device__ __forceinline__ void get(float (&o)[8]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Raw<float> {
  float4 u;
  __device__ __forceinline__ void load(const float* p) { u = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void zero() { u = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load_first(const float* p, int n) {
    u = make_float4(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, n > 3 ? p[3] : 0.f);
  }
  __device__ __forceinline__ void shift_in(const Raw& next, int s) {
    float w[8] = {u.x, u.y, u.z, u.w, next.u.x, next.u.y, next.u.z, next.u.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = s & 2 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = s & 1 ? w[i + 1] : w[i];
    u = make_float4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void get(float (&o)[4]) const { o[0] = u.x; o[1] = u.y; o[2] = u.z; o[3] = u.w; }
};

// Chunk at element e (a multiple of VEC) of an array of `total` elements; outside it: zeros. inner: the chunk is
// known to lie inside (only rows with less than a chunk behind them reach over the array's end).
template <typename T>
__device__ __forceinline__ Raw<T> load_inside(const T* p, long long e, long long total, bool inner) {
  constexpr int VEC = 16 / sizeof(T);
  Raw<T> r;
  if (inner || (e >= 0 && e + VEC <= total)) r.load(p + e);
  else if (e >= 0 && e < total) r.load_first(p + e, (int)(total - e));
  else r.zero();
  return r;
}
// VEC elements from any element e on: two aligned chunks, shifted (s = e mod VEC, the same for a whole row).
template <typename T>
__device__ __forceinline__ Raw<T> load_any(const T* p, long long e, long long total, bool inner) {
  constexpr int VEC = 16 / sizeof(T);
  const int s = (int)(e & (VEC - 1));
  Raw<T> r = load_inside(p, e - s, total, inner);
  if (s) r.shift_in(load_inside(p, e - s + VEC, total, inner), s);
  return r;
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const float (&v)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
}

// Where a thread's chunk j lies. Rows of a multiple of VEC values: chunks of the row. Others (EDGE): chunks of
// the whole array, aligned in memory, of which a row's first and last belong to it in part, so that loads and
// stores are wide whatever the row length; [lo, hi) are the chunk's values of this row (none: lo = hi = 0).
struct Span {
  long long e;  // first element of the chunk in the array
  int k;        // ... in the row (EDGE: may be negative)
  int lo, hi;
};
template <int VEC, bool EDGE>
__device__ __forceinline__ Span span_of(const Args& a, long long row, int j, int t, bool live) {
  Span p;
  const long long at = row * a.n;
  if (EDGE) {
    p.e = (at & ~(long long)(VEC - 1)) + (long long)(j * a.tpr + t) * VEC;
    p.k = (int)(p.e - at);
    p.lo = p.k < 0 ? -p.k : 0;
    p.hi = a.n - p.k < VEC ? a.n - p.k : VEC;
    if (!live || p.lo >= p.hi) p.lo = p.hi = 0;
  } else {
    p.k = (j * a.tpr + t) * VEC;
    p.e = at + p.k;
    p.lo = 0;
    p.hi = live && p.k < a.n ? VEC : 0;
  }
  return p;
}
template <typename T, bool EDGE>
__device__ __forceinline__ void store_span(T* p, const Span& s, const float (&v)[16 / sizeof(T)]) {
  constexpr int VEC = 16 / sizeof(T);
  if (!EDGE || (s.lo == 0 && s.hi == VEC)) {
    store_chunk<T>(p + s.e, v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= s.lo && i < s.hi) p[s.e + i] = (T)v[i];
  }
}

template <typename T>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(__float2bfloat16_rn(v));
  else return v;
}

// weights of VEC consecutive channels from k on, fp32 or bf16
template <int VEC>
__device__ __forceinline__ void load_w(const Args& a, int k, float (&v)[VEC]) {
  if (a.w_bf16) {
    const __nv_bfloat16* w = reinterpret_cast<const __nv_bfloat16*>(a.w);
    const uint32_t* p = reinterpret_cast<const uint32_t*>(w + k);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const uint32_t u = p[i];
      v[2 * i] = __uint_as_float(u << 16);
      v[2 * i + 1] = __uint_as_float(u & 0xFFFF0000u);
    }
  } else {
    const float* w = reinterpret_cast<const float*>(a.w);
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      Raw<float> u;
      u.load(w + k + 4 * i);
      float f[4];
      u.get(f);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[4 * i + q] = f[q];
    }
  }
}

template <int VEC>
__device__ __forceinline__ void take(const float (&f)[VEC + 4], int s, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = f[i + s];
}
// ... from any k on, zeros outside the row: aligned groups of 4, shifted by a branch that a whole row takes alike
template <int VEC>
__device__ __forceinline__ void load_w_any(const Args& a, int k, float (&v)[VEC]) {
  const __nv_bfloat16* wb = reinterpret_cast<const __nv_bfloat16*>(a.w);
  const float* w = reinterpret_cast<const float*>(a.w);
  if (k < 8 || k + 16 > a.n) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = k + i < 0 || k + i >= a.n ? 0.f : a.w_bf16 ? (float)wb[k + i] : w[k + i];
    return;
  }
  const int s = k & 3;
  float f[VEC + 4];
#pragma unroll
  for (int i = 0; i < VEC / 4 + 1; ++i) {
    if (a.w_bf16) {
      const uint2 u = *reinterpret_cast<const uint2*>(wb + k - s + 4 * i);
      f[4 * i] = __uint_as_float(u.x << 16);
      f[4 * i + 1] = __uint_as_float(u.x & 0xFFFF0000u);
      f[4 * i + 2] = __uint_as_float(u.y << 16);
      f[4 * i + 3] = __uint_as_float(u.y & 0xFFFF0000u);
    } else {
      const float4 u = *reinterpret_cast<const float4*>(w + k - s + 4 * i);
      f[4 * i] = u.x;
      f[4 * i + 1] = u.y;
      f[4 * i + 2] = u.z;
      f[4 * i + 3] = u.w;
    }
  }
  switch (s) {
    case 0: take<VEC>(f, 0, v); break;
    case 1: take<VEC>(f, 1, v); break;
    case 2: take<VEC>(f, 2, v); break;
    default: take<VEC>(f, 3, v); break;
  }
}

// Minimum and maximum that keep a NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// amax / top rounded once, as act_quant's: the same amax gives the same scale to the last bit. The product with the
// reciprocal is a unit off for every second amax; what it leaves over, added, makes it the rounded quotient (division by
// a divisor known in advance, Brisebarre, Muller and Raina 2004; compared with the division over all mantissas). A
// division instruction sequence costs int8 rows of 2048 6 % (26.2, 27.7 us). inf and NaN come out as NaN.
template <int TOP>
__device__ __forceinline__ float scale_of(float amax, int pow2) {
  constexpr float kInv = 1.0f / TOP;
  amax = amax < kAmaxFloor ? kAmaxFloor : amax;  // a NaN stays
  const float p = amax * kInv;
  float s = fmaf(fmaf(-p, (float)TOP, amax), kInv, p);
  if (pow2) {
    int e;
    const float m = frexpf(s, &e);
    if (s < INFINITY) s = ldexpf(1.0f, m == 0.5f ? e - 1 : e);
  }
  return s < INFINITY ? s : __int_as_float(0x7FC00000);
}

// Four values already divided by the scale -> four int8 in a word: adding 1.5 * 2^23 leaves the value,
// rounded to the nearest even integer, in the low bits (|v| <= 127 by the choice of the scale).
__device__ __forceinline__ uint32_t int8x4(float a, float b, float c, float d) {
  constexpr float kMagic = 12582912.0f;
  const uint32_t ia = __float_as_uint(a + kMagic), ib = __float_as_uint(b + kMagic), ic = __float_as_uint(c + kMagic),
                 id = __float_as_uint(d + kMagic);
  return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
}

// One block reduction per row: sum and maximum (not negative) over the row's tpr threads. Numbers that are not
// negative order like their bits, with infinity and NaN on top, so the maximum is an integer one.
template <bool SUM, bool MAX>
__device__ __forceinline__ void row_reduce(float& sum, float& top, int tpr) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (SUM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (MAX) top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7FFFFFFFu));
  if (tpr == 32) return;  // a row is one warp
  __shared__ float ssum[32];
  __shared__ uint32_t smax[32];
  const int lane = threadIdx.x & 31, nw = tpr >> 5, w0 = threadIdx.y * nw, warp = w0 + (threadIdx.x >> 5);
  if (lane == 0) {
    if (SUM) ssum[warp] = sum;
    if (MAX) smax[warp] = __float_as_uint(top);
  }
  __syncthreads();
  if (SUM) {
    sum = lane < nw ? ssum[w0 + lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (MAX) top = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < nw ? smax[w0 + lane] : 0u));
}

// v * mul to 8 bits with its scales; top: the row's max |v| (int8), mul: the row's factor that v still lacks. A code is
// v * (mul * (1 / s)) rounded: one factor for all values instead of a division for each, which is within 6 * 2^-24 of
// v mul / s, so that the code is its neighbour where the quotient lies that near to a tie (e4m3: 10 of 21 million codes).
template <int VEC, int NV, bool FP8, bool EDGE>
__device__ __forceinline__ void quant_store(const Args& a, const float (&v)[NV][VEC], float mul, float top, long long row,
                                            int t, bool live) {
  uint8_t* q = reinterpret_cast<uint8_t*>(a.q);
  if constexpr (FP8) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Span p = span_of<VEC, EDGE>(a, row, j, t, live);
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) m = max_nan(m, fabsf(v[j][i]));
      // the 128 values of a block are 16 (bf16) or 32 (fp32) neighbouring lanes' chunks
#pragma unroll
      for (int o = 64 / VEC; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float s = scale_of<448>(m * fabsf(mul), a.pow2);
      const float f = mul * __fdividef(1.0f, s);
      if (p.hi) {
        if (p.k % 128 == 0) a.s[row * (a.n / 128) + p.k / 128] = s;
        const uint32_t lo = f32x2_to_e4m3x2(v[j][0] * f, v[j][1] * f) | (f32x2_to_e4m3x2(v[j][2] * f, v[j][3] * f) << 16);
        if constexpr (VEC == 8) {
          const uint32_t hi = f32x2_to_e4m3x2(v[j][4] * f, v[j][5] * f) | (f32x2_to_e4m3x2(v[j][6] * f, v[j][7] * f) << 16);
          *reinterpret_cast<uint2*>(q + p.e) = make_uint2(lo, hi);
        } else {
          *reinterpret_cast<uint32_t*>(q + p.e) = lo;
        }
      }
    }
  } else {
    const float s = scale_of<127>(top * fabsf(mul), 0);
    const float f = mul * __fdividef(1.0f, s);
    if (t == 0 && live) a.s[row] = s;
    const bool fine = s == s;  // else the row holds a NaN or an infinity: the code 0 throughout
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Span p = span_of<VEC, EDGE>(a, row, j, t, live);
      if (!p.hi) continue;
      uint32_t w[VEC / 4];
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i)
        w[i] = fine ? int8x4(v[j][4 * i] * f, v[j][4 * i + 1] * f, v[j][4 * i + 2] * f, v[j][4 * i + 3] * f) : 0u;
      if (!EDGE || (p.lo == 0 && p.hi == VEC)) {
        if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q + p.e) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(q + p.e) = w[0];
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (i >= p.lo && i < p.hi) q[p.e + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
      }
    }
  }
}

// NaN where the squares' sum is not finite: a row with an infinity or NaN, or with values past 1e19.
__device__ __forceinline__ float rstd_of(float sum, const Args& a) {
  return sum < INFINITY ? 1.0f / sqrtf(sum / (float)a.n + a.eps) : __int_as_float(0x7FC00000);
}

// One row in registers: residual added and stored, squares and |r w| reduced; v holds r w afterwards.
template <typename T, int NV, bool FP8, bool EDGE>
__device__ __forceinline__ void norm_row(const Args& a, const Raw<T> (&x)[NV], const Raw<T> (&r)[NV],
                                         float (&v)[NV][16 / sizeof(T)], float& sum, float& top, long long row, int t, bool live) {
  constexpr int VEC = 16 / sizeof(T);
  sum = 0.f;
  top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Span p = span_of<VEC, EDGE>(a, row, j, t, live);
    x[j].get(v[j]);
    if (!p.hi) continue;
    if (a.res) {
      float y[VEC];
      r[j].get(y);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = round_to<T>(v[j][i] + y[i]);
      if (a.res_out) store_span<T, EDGE>(reinterpret_cast<T*>(a.res_out), p, v[j]);
    }
    if (EDGE && (p.lo != 0 || p.hi != VEC)) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (i < p.lo || i >= p.hi) v[j][i] = 0.f;  // the neighbouring rows' values
    }
    float w[VEC];
    if constexpr (EDGE) load_w_any<VEC>(a, p.k, w);
    else load_w<VEC>(a, p.k, w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      sum = fmaf(v[j][i], v[j][i], sum);
      v[j][i] *= w[i];
      if (!FP8) top = max_nan(top, fabsf(v[j][i]));
    }
  }
}

template <typename T, int NV, bool EDGE>
__device__ __forceinline__ void store_normed(const Args& a, const float (&v)[NV][16 / sizeof(T)], float rstd, long long row, int t,
                                             bool live) {
  constexpr int VEC = 16 / sizeof(T);
  if (!a.normed) return;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Span p = span_of<VEC, EDGE>(a, row, j, t, live);
    if (!p.hi) continue;
    float y[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) y[i] = v[j][i] * rstd;
    store_span<T, EDGE>(reinterpret_cast<T*>(a.normed), p, y);
  }
}

template <typename T, int NV, bool FP8, bool EDGE>
__global__ void __launch_bounds__(1024) norm_kernel(const Args a) {
  constexpr int VEC = 16 / sizeof(T);
  pdl_wait();
  pdl_launch();
  const int t = threadIdx.x;
  const long long row = (long long)blockIdx.x * a.rpc + threadIdx.y, total = a.rows * a.n;
  const bool live = row < a.rows;
  Raw<T> x[NV], r[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Span p = span_of<VEC, EDGE>(a, row, j, t, live);
    x[j].zero();
    r[j].zero();
    if (p.hi) {
      if constexpr (EDGE) {
        const bool inner = (a.rows - 1 - row) * a.n >= VEC;
        x[j] = load_inside(reinterpret_cast<const T*>(a.x), p.e, total, inner);
        if (a.res) r[j] = load_inside(reinterpret_cast<const T*>(a.res), p.e, total, inner);
      } else {
        x[j].load(reinterpret_cast<const T*>(a.x) + p.e);
        if (a.res) r[j].load(reinterpret_cast<const T*>(a.res) + p.e);
      }
    }
  }
  float v[NV][VEC], sum, top;
  norm_row<T, NV, FP8, EDGE>(a, x, r, v, sum, top, row, t, live);
  row_reduce<true, !FP8>(sum, top, a.tpr);
  const float rstd = rstd_of(sum, a);
  store_normed<T, NV, EDGE>(a, v, rstd, row, t, live);
  quant_store<VEC, NV, FP8, EDGE>(a, v, rstd, top, row, t, live);
}

__device__ __forceinline__ float exp2_hw(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_hw(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two fp32 values in a register pair: one instruction for both on this architecture.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_get(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// silu(g) u of two values, with g <= limit, |u| <= limit, as (-g) (-u) / (1 + exp(-g)). exp(n) of n = -g is
// 2^t (1 + r) with t = n log2(e) rounded and r = n - t ln 2, what the rounding lost, so the hardware's 2^t (2 units in the
// last place) and reciprocal (1) are all that is approximated; the argument's own rounding would cost |g| units. t
// stops at 87 log2(e), before 2^t overflows, but r does not: past it the sum grows on, and from n = 87.5 on (silu(g) above
// -1e-36) its reciprocal is 0 and takes every finite gate to 0 and -inf to the formula's NaN. BIG: limits past 1e38, where t
// needs a floor too; chosen at launch, as the two in one kernel take 29.4 us where one takes 24.4 (e4m3, 12282 x 2048).
// PACKED: both values in one instruction where it exists (the same rows when this was chosen: e4m3 24.2 us, 25.3 one by
// one; int8 rows without an edge are faster one by one, 26.0 and 27.7).
template <bool PACKED, bool BIG>
__device__ __forceinline__ void swiglu2(float& g0, float& g1, float u0, float u1, float limit) {
  const float n0 = max_nan(-g0, -limit), n1 = max_nan(-g1, -limit);
  u0 = max_nan(min_nan(-u0, limit), -limit);
  u1 = max_nan(min_nan(-u1, limit), -limit);
  constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
  float a0 = min_nan(n0, 87.0f), a1 = min_nan(n1, 87.0f);
  if (BIG) {
    a0 = max_nan(a0, -200.0f);
    a1 = max_nan(a1, -200.0f);
  }
  float t0, t1, e0, e1;
  if constexpr (PACKED) {
    const F2 n = f2(n0, n1), t = f2_mul(f2(a0, a1), f2(kLog2e, kLog2e)), r = f2_fma(t, f2(-kLn2, -kLn2), n);
    f2_get(t, t0, t1);
    e0 = exp2_hw(t0);
    e1 = exp2_hw(t1);
    const F2 e = f2(e0, e1);
    f2_get(f2_add(f2_fma(e, r, e), f2(1.0f, 1.0f)), t0, t1);
    f2_get(f2_mul(f2_mul(n, f2(rcp_hw(t0), rcp_hw(t1))), f2(u0, u1)), g0, g1);
  } else {
    t0 = a0 * kLog2e;
    t1 = a1 * kLog2e;
    e0 = exp2_hw(t0);
    e1 = exp2_hw(t1);
    g0 = n0 * rcp_hw(1.0f + fmaf(e0, fmaf(t0, -kLn2, n0), e0)) * u0;
    g1 = n1 * rcp_hw(1.0f + fmaf(e1, fmaf(t1, -kLn2, n1), e1)) * u1;
  }
}

template <typename T, int NV, bool FP8, bool EDGE, bool BIG>
__global__ void __launch_bounds__(1024) swiglu_kernel(const Args a) {
  constexpr int VEC = 16 / sizeof(T);
  pdl_wait();
  pdl_launch();
  const int t = threadIdx.x;
  const long long row = (long long)blockIdx.x * a.rpc + threadIdx.y, total = 2 * a.rows * a.n;
  const bool live = row < a.rows;
  const T* gu = reinterpret_cast<const T*>(a.x);
  Raw<T> x[NV], y[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Span p = span_of<VEC, EDGE>(a, row, j, t, live);
    const long long e = 2 * row * a.n + p.k;
    x[j].zero();
    y[j].zero();
    if (p.hi) {
      if constexpr (EDGE) {  // the codes' chunks are aligned; g and u lie at their own offsets to them
        if ((a.rows - 1 - row) * a.n >= VEC) {  // 2 VEC values behind the row: two whole chunks lie inside
          const long long eg = 2 * row * a.n - (row * a.n & (VEC - 1)), eu = eg + a.n;  // where the row's chunk 0 begins
          const int sg = (int)(eg & (VEC - 1)), su = (int)(eu & (VEC - 1)), c = (j * a.tpr + t) * VEC;
          Raw<T> xn, yn;
          x[j].load(gu + (eg - sg) + c);
          xn.load(gu + (eg - sg) + c + VEC);
          y[j].load(gu + (eu - su) + c);
          yn.load(gu + (eu - su) + c + VEC);
          x[j].shift_in(xn, sg);
          y[j].shift_in(yn, su);
        } else {
          x[j] = load_any(gu, e, total, false);
          y[j] = load_any(gu, e + a.n, total, false);
        }
      } else {
        x[j].load(gu + e);
        y[j].load(gu + e + a.n);
      }
    }
  }
  const float wr = live && a.w ? reinterpret_cast<const float*>(a.w)[row] : 1.0f;
  float v[NV][VEC], top = 0.f, none = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Span p = span_of<VEC, EDGE>(a, row, j, t, live);
    float u[VEC];
    x[j].get(v[j]);
    y[j].get(u);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) swiglu2<FP8 || EDGE, BIG>(v[j][i], v[j][i + 1], u[i], u[i + 1], a.limit);
    if (EDGE && (p.lo != 0 || p.hi != VEC)) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (i < p.lo || i >= p.hi) v[j][i] = 0.f;  // the neighbouring rows' values
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (!FP8) top = max_nan(top, fabsf(v[j][i]));
  }
  if (!FP8) row_reduce<false, true>(none, top, a.tpr);
  quant_store<VEC, NV, FP8, EDGE>(a, v, wr, top, row, t, live);
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <bool NORM, typename T, int NV, bool FP8, bool EDGE>
void launch(const Args& a, cudaStream_t st) {
  const long long grid = (a.rows + a.rpc - 1) / a.rpc;
  launch_pdl(NORM               ? norm_kernel<T, NV, FP8, EDGE>
             : a.limit > 1e38f ? swiglu_kernel<T, NV, FP8, EDGE, true>
                               : swiglu_kernel<T, NV, FP8, EDGE, false>,
             dim3((unsigned)grid), dim3(a.tpr, a.rpc), 0, st, a);
}
template <bool NORM, typename T, bool FP8, bool EDGE>
void launch_nv(const Args& a, int nv, cudaStream_t st) {
  if (nv == 1) launch<NORM, T, 1, FP8, EDGE>(a, st);
  else if (nv == 2) launch<NORM, T, 2, FP8, EDGE>(a, st);
  else if (nv == 4) launch<NORM, T, 4, FP8, EDGE>(a, st);
  else if constexpr (EDGE && sizeof(T) == 4) launch<NORM, T, 8, FP8, EDGE>(a, st);  // the longest: 4097 chunks
}

template <bool NORM, typename T>
int run(Args& a, bool fp8, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool edge = a.n % V != 0;
  const int nchunk = edge ? (a.n - 2) / V + 2 : a.n / V;  // a row's chunks, at most
  // Chunks per thread: one, so that a row's loads go out at once from many threads. The norm's fixed work per thread
  // is worth two where the grid fills the GPU several times (4096 rows of 5120 32.7 us, 34.7 with one), and with an
  // edge, where registers let few threads onto an SM, from about one long row per SM on (4000 rows of 6387 50.9 us, 80.6
  // with one; 160: 4.5, 6.0; but 100 of 5001 3.4, 2.9, and 400 of 1501 3.7, 3.2). The swiglu loses (12282 rows of 2048
  // 24.2 us, 27.6 with two; 6000 of 2049 22.7, 26.0). A row keeps 32 threads.
  int nv = 1;
  while ((nchunk + nv - 1) / nv > 1024) nv *= 2;
  if (NORM && nv == 1 && nchunk >= (edge ? 128 : 64) && a.rows * nchunk >= (edge ? 600LL : 8192LL) * sm_count()) nv = 2;
  a.tpr = ((nchunk + nv - 1) / nv + 31) / 32 * 32;
  a.rpc = a.tpr >= 256 ? 1 : 256 / a.tpr;
  if (a.rpc > a.rows) a.rpc = (int)a.rows;
  if (fp8) launch_nv<NORM, T, true, false>(a, nv, st);
  else if (edge) launch_nv<NORM, T, false, true>(a, nv, st);
  else launch_nv<NORM, T, false, false>(a, nv, st);
  return cuda_status(NORM ? "rms_norm_quant" : "swiglu_quant");
}

int check(const char* name, int dtype, int q_dtype, int pow2, long long rows, long long n, const void* q, const float* s) {
  DSMOE_REQUIRE(q && s, DSMOE_ERR_ARG, "%s: null pointer", name);
  DSMOE_REQUIRE(dtype == DSMOE_DTYPE_F32 || dtype == DSMOE_DTYPE_BF16, DSMOE_ERR_ARG, "%s: dtype %d", name, dtype);
  DSMOE_REQUIRE(q_dtype == DSMOE_DTYPE_E4M3 || q_dtype == DSMOE_DTYPE_I8, DSMOE_ERR_ARG, "%s: q_dtype %d", name, q_dtype);
  DSMOE_REQUIRE(rows > 0 && rows < (1LL << 31), DSMOE_ERR_ARG, "%s: rows %lld", name, rows);
  DSMOE_REQUIRE(n > 0 && n <= kMaxHidden, DSMOE_ERR_ARG, "%s: row length %lld (1..%d)", name, n, kMaxHidden);
  DSMOE_REQUIRE(q_dtype == DSMOE_DTYPE_I8 || n % 128 == 0, DSMOE_ERR_ARG, "%s: e4m3 rows need a multiple of 128 values (%lld)",
                name, n);
  DSMOE_REQUIRE(!pow2 || q_dtype == DSMOE_DTYPE_E4M3, DSMOE_ERR_ARG, "%s: power-of-2 scales are for e4m3", name);
  return DSMOE_OK;
}

}  // namespace rows8
}  // namespace dsmoe

using namespace dsmoe;

extern "C" int dsmoe_rms_norm_quant(const void* x, int dtype, const void* residual, const void* weight, int w_dtype,
                                    long long rows, long long hidden, float eps, int q_dtype, int pow2, void* q, float* s,
                                    void* residual_out, void* normed, void* stream) {
  int rc = rows8::check("rms_norm_quant", dtype, q_dtype, pow2, rows, hidden, q, s);
  if (rc) return rc;
  DSMOE_REQUIRE(x && weight, DSMOE_ERR_ARG, "rms_norm_quant: null pointer");
  DSMOE_REQUIRE(w_dtype == DSMOE_DTYPE_F32 || w_dtype == DSMOE_DTYPE_BF16, DSMOE_ERR_ARG, "rms_norm_quant: w_dtype %d", w_dtype);
  DSMOE_REQUIRE(!residual_out || residual, DSMOE_ERR_ARG, "rms_norm_quant: residual_out without residual");
  const int sz = dtype == DSMOE_DTYPE_F32 ? 4 : 2;
  DSMOE_REQUIRE((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)residual_out | (uintptr_t)normed |
                  (uintptr_t)q) & 15) == 0 && ((uintptr_t)s & 3) == 0,
                DSMOE_ERR_ALIGN, "rms_norm_quant: misaligned pointer");
  // every output is its own memory; only residual_out may be x or residual themselves (element for element)
  const long long nb = rows * hidden * sz, sb = (q_dtype == DSMOE_DTYPE_E4M3 ? rows * (hidden / 128) : rows) * 4;
  DSMOE_REQUIRE(!overlap({{residual_out, nb}, {normed, nb}, {q, rows * hidden}, {s, sb}},
                         {{x == residual_out ? nullptr : x, nb},
                          {residual == residual_out ? nullptr : residual, nb},
                          {weight, hidden * (w_dtype == DSMOE_DTYPE_F32 ? 4 : 2)}}),
                DSMOE_ERR_ARG, "rms_norm_quant: outputs overlap inputs");
  rows8::Args a{};
  a.x = x; a.res = residual; a.w = weight; a.q = q; a.s = s; a.res_out = residual_out; a.normed = normed;
  a.rows = rows; a.n = (int)hidden; a.w_bf16 = w_dtype == DSMOE_DTYPE_BF16; a.pow2 = pow2; a.eps = eps;
  const bool fp8 = q_dtype == DSMOE_DTYPE_E4M3;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == DSMOE_DTYPE_F32 ? rows8::run<true, float>(a, fp8, st) : rows8::run<true, __nv_bfloat16>(a, fp8, st);
}

extern "C" int dsmoe_swiglu_quant(const void* gu, int dtype, const float* row_weight, long long rows, long long inter,
                                  float limit, int q_dtype, int pow2, void* q, float* s, void* stream) {
  int rc = rows8::check("swiglu_quant", dtype, q_dtype, pow2, rows, inter, q, s);
  if (rc) return rc;
  DSMOE_REQUIRE(gu, DSMOE_ERR_ARG, "swiglu_quant: null pointer");
  DSMOE_REQUIRE(limit > 0.f, DSMOE_ERR_ARG, "swiglu_quant: limit must be positive");
  const int sz = dtype == DSMOE_DTYPE_F32 ? 4 : 2;
  DSMOE_REQUIRE((((uintptr_t)gu | (uintptr_t)q) & 15) == 0 && (((uintptr_t)s | (uintptr_t)row_weight) & 3) == 0, DSMOE_ERR_ALIGN,
                "swiglu_quant: misaligned pointer");
  const long long sb = (q_dtype == DSMOE_DTYPE_E4M3 ? rows * (inter / 128) : rows) * 4;
  DSMOE_REQUIRE(!overlap({{q, rows * inter}, {s, sb}}, {{gu, 2 * rows * inter * sz}, {row_weight, rows * 4}}), DSMOE_ERR_ARG,
                "swiglu_quant: outputs overlap inputs");
  rows8::Args a{};
  a.x = gu; a.w = row_weight; a.q = q; a.s = s; a.rows = rows; a.n = (int)inter; a.pow2 = pow2; a.limit = limit;
  const bool fp8 = q_dtype == DSMOE_DTYPE_E4M3;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == DSMOE_DTYPE_F32 ? rows8::run<false, float>(a, fp8, st) : rows8::run<false, __nv_bfloat16>(a, fp8, st);
}
