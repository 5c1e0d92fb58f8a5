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
// A row (e4m3: a block) whose amax is not finite gets the scale NaN, so its values read back as NaN.
#include "common.cuh"

namespace dsmoe {
namespace rows8 {

constexpr float kAmaxFloor = 1e-4f;
constexpr int kMaxHidden = 16384;
constexpr int kStages = 3;              // rows in a persistent CTA's ring
constexpr int kMaxSmem = 227 * 1024;

struct Args {
  const void* x;      // norm: [rows][n]; swiglu: [rows][2n] (g | u)
  const void* res;    // norm: [rows][n] or null
  const void* w;      // norm: [n] fp32 or bf16; swiglu: [rows] fp32 row weight or null
  void* q;            // [rows][n] 8-bit
  float* s;           // e4m3: [rows][n / 128]; int8: [rows]
  void* res_out;      // norm: [rows][n] or null
  void* normed;       // norm: [rows][n] or null
  long long rows;
  int n, nchunk;      // values per row; chunks of VEC values
  int tpr, rpc;       // threads per row (a multiple of 32), rows per CTA
  int w_bf16, pow2;
  float eps, limit;
};

// A chunk as loaded, and its values: bf16 stays packed in registers until it is used.
template <typename T, int VEC>
struct Raw {
  T v;  // VEC == 1
  __device__ __forceinline__ void load(const T* p) { v = p[0]; }
  __device__ __forceinline__ void zero() { v = (T)0.f; }
  __device__ __forceinline__ void get(float (&o)[VEC]) const { o[0] = (float)v; }
};
template <>
struct Raw<__nv_bfloat16, 8> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
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
struct Raw<float, 4> {
  float4 u;
  __device__ __forceinline__ void load(const float* p) { u = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void zero() { u = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&o)[4]) const { o[0] = u.x; o[1] = u.y; o[2] = u.z; o[3] = u.w; }
};

template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(T) == 2) p[0] = __float2bfloat16_rn(v[0]);
    else p[0] = v[0];
  } else if constexpr (sizeof(T) == 2) {
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

template <typename T>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(__float2bfloat16_rn(v));
  else return v;
}

// weights of VEC consecutive channels, fp32 or bf16
template <int VEC>
__device__ __forceinline__ void load_w(const void* w, int w_bf16, int at, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = w_bf16 ? (float)reinterpret_cast<const __nv_bfloat16*>(w)[at] : reinterpret_cast<const float*>(w)[at];
  } else if (w_bf16) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(reinterpret_cast<const __nv_bfloat16*>(w) + at);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const uint32_t u = p[i];
      v[2 * i] = __uint_as_float(u << 16);
      v[2 * i + 1] = __uint_as_float(u & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 u = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + at + 4 * i);
      v[4 * i] = u.x; v[4 * i + 1] = u.y; v[4 * i + 2] = u.z; v[4 * i + 3] = u.w;
    }
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

__device__ __forceinline__ float scale_of(float amax, float inv_top, int pow2) {
  float s = (amax < kAmaxFloor ? kAmaxFloor : amax) * inv_top;  // a NaN stays
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
__device__ __forceinline__ void row_reduce(float& sum, float& top, int tpr, int turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (SUM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (MAX) top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7FFFFFFFu));
  if (tpr == 32 && blockDim.x == 32) {
    __syncwarp();
    return;
  }
  __shared__ float ssums[2][32];  // a second reduction (turn 1) may begin while the first is being read
  __shared__ uint32_t smaxs[2][32];
  float* ssum = ssums[turn];
  uint32_t* smax = smaxs[turn];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = tpr >> 5, w0 = warp / nw * nw;
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

// v * mul to 8 bits with its scales; top: the row's max |v| (int8), mul: the row's factor that v still lacks.
template <int VEC, int NV, bool FP8>
__device__ __forceinline__ void quant_store(const Args& a, const float (&v)[NV][VEC], float mul, float top, long long row,
                                            int t, bool live) {
  if constexpr (FP8) {
    uint8_t* q = reinterpret_cast<uint8_t*>(a.q) + row * a.n;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * a.tpr + t;
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) m = max_nan(m, fabsf(v[j][i]));
      // the 128 values of a block are 16 (bf16) or 32 (fp32) neighbouring lanes' chunks
#pragma unroll
      for (int o = 64 / VEC; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float s = scale_of(m * fabsf(mul), 1.0f / 448.0f, a.pow2);
      const float f = mul * __fdividef(1.0f, s);
      if (live && c < a.nchunk) {
        if ((c * VEC) % 128 == 0) a.s[row * (a.n / 128) + c * VEC / 128] = s;
        const uint32_t lo = f32x2_to_e4m3x2(v[j][0] * f, v[j][1] * f) | (f32x2_to_e4m3x2(v[j][2] * f, v[j][3] * f) << 16);
        if constexpr (VEC == 8) {
          const uint32_t hi = f32x2_to_e4m3x2(v[j][4] * f, v[j][5] * f) | (f32x2_to_e4m3x2(v[j][6] * f, v[j][7] * f) << 16);
          *reinterpret_cast<uint2*>(q + c * VEC) = make_uint2(lo, hi);
        } else {
          *reinterpret_cast<uint32_t*>(q + c * VEC) = lo;
        }
      }
    }
  } else {
    const float s = scale_of(top * fabsf(mul), 1.0f / 127.0f, 0);
    const float f = mul * __fdividef(1.0f, s);
    if (!live) return;
    if (t == 0) a.s[row] = s;
    uint8_t* q = reinterpret_cast<uint8_t*>(a.q) + row * a.n;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * a.tpr + t;
      if (c >= a.nchunk) continue;
      // a row without a scale (NaN or infinity somewhere) has the code 0 throughout
      auto at = [&](int i) { return s == s ? v[j][i] * f : 0.f; };
      if constexpr (VEC == 1) {
        q[c] = (uint8_t)int8x4(at(0), 0.f, 0.f, 0.f);
      } else if constexpr (VEC == 4) {
        *reinterpret_cast<uint32_t*>(q + c * VEC) = int8x4(at(0), at(1), at(2), at(3));
      } else {
        *reinterpret_cast<uint2*>(q + c * VEC) = make_uint2(int8x4(at(0), at(1), at(2), at(3)),
                                                            int8x4(at(4), at(5), at(6), at(7)));
      }
    }
  }
}

// One row in registers: residual added and stored, squares and |r w| reduced; v holds r w afterwards.
template <typename T, int VEC, int NV, bool FP8>
__device__ __forceinline__ void norm_row(const Args& a, const Raw<T, VEC> (&x)[NV], const Raw<T, VEC> (&r)[NV],
                                         float (&v)[NV][VEC], float& sum, float& top, long long at, int t, bool live) {
  sum = 0.f;
  top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * a.tpr + t;
    x[j].get(v[j]);
    if (live && c < a.nchunk) {
      if (a.res) {
        float y[VEC];
        r[j].get(y);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] = round_to<T>(v[j][i] + y[i]);
        if (a.res_out) store_chunk<T, VEC>(reinterpret_cast<T*>(a.res_out) + at + c * VEC, v[j]);
      }
      float w[VEC];
      load_w<VEC>(a.w, a.w_bf16, c * VEC, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        sum = fmaf(v[j][i], v[j][i], sum);
        v[j][i] *= w[i];
        if (!FP8) top = max_nan(top, fabsf(v[j][i]));
      }
    }
  }
}

template <typename T, int VEC, int NV>
__device__ __forceinline__ void store_normed(const Args& a, const float (&v)[NV][VEC], float rstd, long long at, int t, bool live) {
  if (!a.normed || !live) return;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * a.tpr + t;
    if (c >= a.nchunk) continue;
    float y[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) y[i] = v[j][i] * rstd;
    store_chunk<T, VEC>(reinterpret_cast<T*>(a.normed) + at + c * VEC, y);
  }
}

template <typename T, int VEC, int NV, bool FP8>
__global__ void __launch_bounds__(1024) norm_kernel(const Args a) {
  const int g = threadIdx.x / a.tpr, t = threadIdx.x % a.tpr;
  const long long row = (long long)blockIdx.x * a.rpc + g;
  const bool live = row < a.rows;
  const long long at = row * a.n;
  Raw<T, VEC> x[NV], r[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * a.tpr + t;
    x[j].zero();
    r[j].zero();
    if (live && c < a.nchunk) {
      x[j].load(reinterpret_cast<const T*>(a.x) + at + c * VEC);
      if (a.res) r[j].load(reinterpret_cast<const T*>(a.res) + at + c * VEC);
    }
  }
  float v[NV][VEC], sum;
  float top;
  norm_row<T, VEC, NV, FP8>(a, x, r, v, sum, top, at, t, live);
  row_reduce<true, !FP8>(sum, top, a.tpr, 0);
  const float rstd = 1.0f / sqrtf(sum / (float)a.n + a.eps);
  store_normed<T, VEC, NV>(a, v, rstd, at, t, live);
  quant_store<VEC, NV, FP8>(a, v, rstd, top, row, t, live);
}

// Many rows: a persistent CTA walks rows blockIdx.x + i gridDim.x while bulk copies bring the next ones into a
// ring of shared memory, so loads stay in flight over the reductions and stores of the rows before.
constexpr uint64_t kWaitNs = 1000000000ull;

template <typename T, int VEC, int NV, bool FP8>
__global__ void __launch_bounds__(512) norm_stream_kernel(const Args a) {
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ uint64_t full[kStages];
  const int t = threadIdx.x, terms = a.res ? 2 : 1;
  const uint32_t row_bytes = (uint32_t)(a.n * sizeof(T));
  if (t == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  __syncthreads();
  auto fetch = [&](long long row, int s) {
    uint8_t* st = sm + (size_t)s * terms * row_bytes;
    mbar_expect_tx(&full[s], terms * row_bytes);
    bulk_g2s(st, reinterpret_cast<const T*>(a.x) + row * a.n, row_bytes, &full[s]);
    if (a.res) bulk_g2s(st + row_bytes, reinterpret_cast<const T*>(a.res) + row * a.n, row_bytes, &full[s]);
  };
  const long long step = gridDim.x;
  if (t == 0)
    for (int s = 0; s < kStages; ++s)
      if (blockIdx.x + s * step < a.rows) fetch(blockIdx.x + s * step, s);
  int i = 0;
  for (long long row = blockIdx.x; row < a.rows; row += step, ++i) {
    const int s = i % kStages;
    const bool ok = mbar_wait(&full[s], (i / kStages) & 1, kWaitNs);
    const T* st = reinterpret_cast<const T*>(sm + (size_t)s * terms * row_bytes);
    Raw<T, VEC> x[NV], r[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = j * a.tpr + t;
      x[j].zero();
      r[j].zero();
      if (c < a.nchunk) {
        x[j].load(st + c * VEC);
        if (a.res) r[j].load(st + a.n + c * VEC);
      }
    }
    float v[NV][VEC], sum;
    float top;
    norm_row<T, VEC, NV, FP8>(a, x, r, v, sum, top, row * a.n, t, true);
    row_reduce<true, !FP8>(sum, top, a.tpr, i & 1);  // its barrier: every thread has read the stage
    if (t == 0 && row + kStages * step < a.rows) fetch(row + kStages * step, s);
    // an expired wait leaves a row of NaN
    const float rstd = ok ? 1.0f / sqrtf(sum / (float)a.n + a.eps) : __int_as_float(0x7FC00000);
    store_normed<T, VEC, NV>(a, v, rstd, row * a.n, t, true);
    quant_store<VEC, NV, FP8>(a, v, rstd, top, row, t, true);
  }
}

// silu(g) u with g <= limit, |u| <= limit. exp(-g) = 2^t (1 + d ln 2) with t = -g log2(e) rounded and d what the
// rounding lost, so the hardware's 2^t (2 units in the last place) and reciprocal (1) are all that is
// approximated; the argument's own rounding would cost |g| units. exp's argument stops at 87, where silu(g) is
// below 1e-35, so that the reciprocal stays a normal number.
__device__ __forceinline__ float swiglu(float g, float u, float limit) {
  g = min_nan(g, limit);
  u = max_nan(min_nan(u, limit), -limit);
  constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
  const float a = max_nan(g, -87.0f);
  const float t = -a * kLog2e, d = fmaf(-a, kLog2e, -t);
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  e = 1.0f + fmaf(e, d * kLn2, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e));
  return g * r * u;
}

template <typename T, int VEC, int NV, bool FP8>
__global__ void __launch_bounds__(1024) swiglu_kernel(const Args a) {
  const int gidx = threadIdx.x / a.tpr, t = threadIdx.x % a.tpr;
  const long long row = (long long)blockIdx.x * a.rpc + gidx;
  const bool live = row < a.rows;
  const T* g = reinterpret_cast<const T*>(a.x) + row * 2 * a.n;
  Raw<T, VEC> x[NV], y[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = j * a.tpr + t;
    x[j].zero();
    y[j].zero();
    if (live && c < a.nchunk) {
      x[j].load(g + c * VEC);
      y[j].load(g + a.n + c * VEC);
    }
  }
  const float wr = live && a.w ? reinterpret_cast<const float*>(a.w)[row] : 1.0f;
  float v[NV][VEC], top = 0.f, none = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float u[VEC];
    x[j].get(v[j]);
    y[j].get(u);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[j][i] = swiglu(v[j][i], u[i], a.limit);
      if (!FP8) top = max_nan(top, fabsf(v[j][i]));
    }
  }
  if (!FP8) row_reduce<false, true>(none, top, a.tpr, 0);
  quant_store<VEC, NV, FP8>(a, v, wr, top, row, t, live);
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <bool NORM, typename T, int VEC, int NV, bool FP8>
void launch(const Args& a, cudaStream_t st) {
  const long long grid = (a.rows + a.rpc - 1) / a.rpc;
  if (NORM) norm_kernel<T, VEC, NV, FP8><<<(unsigned)grid, a.tpr * a.rpc, 0, st>>>(a);
  else swiglu_kernel<T, VEC, NV, FP8><<<(unsigned)grid, a.tpr * a.rpc, 0, st>>>(a);
}

template <typename T, int NV, bool FP8>
void launch_stream(const Args& a, int ctas, size_t smem, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  auto k = norm_stream_kernel<T, V, NV, FP8>;
  if (smem > 48 * 1024) cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  k<<<ctas, a.tpr, smem, st>>>(a);
}

template <bool NORM, typename T>
int run(Args& a, bool fp8, bool wide, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int vec = wide ? V : 1;
  a.nchunk = (a.n + vec - 1) / vec;
  if (NORM && wide) {
    // ring of whole rows where every CTA of the persistent grid gets several of them
    const int nv = a.nchunk <= 1024 ? 2 : 4;
    const int tpr = ((a.nchunk + nv - 1) / nv + 31) / 32 * 32;
    const size_t smem = (size_t)kStages * (a.res ? 2 : 1) * a.n * sizeof(T);
    const int per_sm = (int)(kMaxSmem / (smem + 2048));  // beside static arrays and what the system keeps
    const int sms = sm_count(), fit = per_sm < 2048 / tpr ? per_sm : 2048 / tpr;
    if (tpr >= 128 && tpr <= 512 && fit >= 1 && a.rows >= 2LL * sms * fit) {
      a.tpr = tpr;
      a.rpc = 1;
      const int ctas = sms * fit;
      if (fp8) {
        if (nv == 2) launch_stream<T, 2, true>(a, ctas, smem, st);
        else launch_stream<T, 4, true>(a, ctas, smem, st);
      } else {
        if (nv == 2) launch_stream<T, 2, false>(a, ctas, smem, st);
        else launch_stream<T, 4, false>(a, ctas, smem, st);
      }
      return cuda_status("rms_norm_quant");
    }
  }
  // chunks per thread: few, so that a row's loads are spread over many threads
  int nv = wide ? 1 : 8;
  while ((a.nchunk + nv - 1) / nv > 1024) nv *= 2;
  a.tpr = ((a.nchunk + nv - 1) / nv + 31) / 32 * 32;
  a.rpc = a.tpr >= 256 ? 1 : 256 / a.tpr;
  if (a.rpc > a.rows) a.rpc = (int)a.rows;
  if (wide) {
    if (fp8) {
      if (nv == 1) launch<NORM, T, V, 1, true>(a, st);
      else if (nv == 2) launch<NORM, T, V, 2, true>(a, st);
      else launch<NORM, T, V, 4, true>(a, st);
    } else {
      if (nv == 1) launch<NORM, T, V, 1, false>(a, st);
      else if (nv == 2) launch<NORM, T, V, 2, false>(a, st);
      else launch<NORM, T, V, 4, false>(a, st);
    }
  } else {
    if (nv == 8) launch<NORM, T, 1, 8, false>(a, st);
    else launch<NORM, T, 1, 16, false>(a, st);
  }
  return cuda_status(NORM ? "rms_norm_quant" : "swiglu_quant");
}

bool overlap(const void* p, long long np, const void* q, long long nq) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return p && q && a < b + (uintptr_t)nq && b < a + (uintptr_t)np;
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
  // every output is its own memory; only residual_out may be x or residual themselves (element for element)
  const long long nb = rows * hidden * sz;
  DSMOE_REQUIRE((residual_out == residual || !rows8::overlap(residual_out, nb, residual, nb)) &&
                    (residual_out == x || !rows8::overlap(residual_out, nb, x, nb)) &&
                    !rows8::overlap(normed, nb, x, nb) && !rows8::overlap(normed, nb, residual, nb) &&
                    !rows8::overlap(normed, nb, residual_out, nb) && !rows8::overlap(q, rows * hidden, x, nb) &&
                    !rows8::overlap(q, rows * hidden, residual, nb) && !rows8::overlap(q, rows * hidden, residual_out, nb) &&
                    !rows8::overlap(q, rows * hidden, normed, nb),
                DSMOE_ERR_ARG, "rms_norm_quant: outputs overlap inputs");
  const uintptr_t any = (uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)residual_out | (uintptr_t)normed;
  DSMOE_REQUIRE((any & (sz - 1)) == 0 && ((uintptr_t)s & 3) == 0 &&
                    ((uintptr_t)weight & (w_dtype == DSMOE_DTYPE_F32 ? 3 : 1)) == 0,
                DSMOE_ERR_ALIGN, "rms_norm_quant: misaligned pointer");
  const bool wide = (any & 15) == 0 && ((uintptr_t)q & 7) == 0 && hidden * sz % 16 == 0;
  DSMOE_REQUIRE(wide || q_dtype == DSMOE_DTYPE_I8, DSMOE_ERR_ALIGN, "rms_norm_quant: e4m3 rows need 16-byte aligned pointers");
  rows8::Args a{};
  a.x = x; a.res = residual; a.w = weight; a.q = q; a.s = s; a.res_out = residual_out; a.normed = normed;
  a.rows = rows; a.n = (int)hidden; a.w_bf16 = w_dtype == DSMOE_DTYPE_BF16; a.pow2 = pow2; a.eps = eps;
  const bool fp8 = q_dtype == DSMOE_DTYPE_E4M3;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == DSMOE_DTYPE_F32 ? rows8::run<true, float>(a, fp8, wide, st) : rows8::run<true, __nv_bfloat16>(a, fp8, wide, st);
}

extern "C" int dsmoe_swiglu_quant(const void* gu, int dtype, const float* row_weight, long long rows, long long inter,
                                  float limit, int q_dtype, int pow2, void* q, float* s, void* stream) {
  int rc = rows8::check("swiglu_quant", dtype, q_dtype, pow2, rows, inter, q, s);
  if (rc) return rc;
  DSMOE_REQUIRE(gu, DSMOE_ERR_ARG, "swiglu_quant: null pointer");
  DSMOE_REQUIRE(limit > 0.f, DSMOE_ERR_ARG, "swiglu_quant: limit must be positive");
  const int sz = dtype == DSMOE_DTYPE_F32 ? 4 : 2;
  DSMOE_REQUIRE(((uintptr_t)gu & (sz - 1)) == 0 && (((uintptr_t)s | (uintptr_t)row_weight) & 3) == 0, DSMOE_ERR_ALIGN,
                "swiglu_quant: misaligned pointer");
  DSMOE_REQUIRE(!rows8::overlap(q, rows * inter, gu, 2 * rows * inter * sz), DSMOE_ERR_ARG, "swiglu_quant: q overlaps gu");
  const bool wide = ((uintptr_t)gu & 15) == 0 && ((uintptr_t)q & 7) == 0 && inter * sz % 16 == 0;
  DSMOE_REQUIRE(wide || q_dtype == DSMOE_DTYPE_I8, DSMOE_ERR_ALIGN, "swiglu_quant: e4m3 rows need 16-byte aligned pointers");
  rows8::Args a{};
  a.x = gu; a.w = row_weight; a.q = q; a.s = s; a.rows = rows; a.n = (int)inter; a.pow2 = pow2; a.limit = limit;
  const bool fp8 = q_dtype == DSMOE_DTYPE_E4M3;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == DSMOE_DTYPE_F32 ? rows8::run<false, float>(a, fp8, wide, st) : rows8::run<false, __nv_bfloat16>(a, fp8, wide, st);
}
