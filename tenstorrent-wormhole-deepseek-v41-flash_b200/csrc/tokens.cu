// Tokens sorted by expert and back, and the gradients of both directions:
//   dsmoe_sort_tokens      idx [P, k] -> pos [P, k], src [P k], offsets [E + 1]
//   dsmoe_dispatch_rows    xs[pos[t, j]] = x[t]                     (rows behind the last: zero)
//   dsmoe_combine_rows     y[t] = sum_j wt[t, j] ys[pos[t, j]]      (wt = 1: the gradient of dispatch)
//   dsmoe_combine_grad     dys[pos[t, j]] = wt[t, j] dy[t],  dwt[t, j] = <dy[t], ys[pos[t, j]]>
// The order is that of (expert, token, choice): a stable counting sort, so nothing depends on the
// order in which threads arrive. Choices outside 0..E-1 are dropped (pos = -1) and the rows behind
// offsets[E] hold zeros.
// The three row kernels are bound by memory: a token's row is read once for all its choices. Measured, bf16 rows of
// 5120, 4096 tokens x 6: dispatch 49 us (6.0 TB/s), combine 48 us (6.1), its gradient 91 us (6.0). The sort is a chain
// of latencies: 48 pairs 3.0 us, 12282 6.5, 131072 16.9.
#include <cooperative_groups.h>

#include <atomic>

#include "common.cuh"

namespace dsmoe {
namespace tokens {

namespace cg = cooperative_groups;

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 64;

// ------------------------------------------------------------------ sort
// One cluster of C CTAs (C = 1 for few pairs). Counting warp w of CTA c owns a contiguous run of pairs and a
// row of counters in shared memory. Count; prefix over the warps of the CTA, the CTAs of the cluster (their
// totals read through distributed shared memory) and the experts; then each warp walks its run again, 32
// pairs at a time, and ranks equal experts among its lanes by match. Bound by latency: a launch, two reads of
// idx, a cluster barrier and the scan; loads are issued kBatch at a time.
struct SortArgs {
  const int64_t* idx;
  int* pos;
  int* src;
  int* offsets;
  int n, E;
  int run, cw;  // pairs per counting warp (a multiple of 32), counting warps of a CTA
};
constexpr int kBatch = 4;
constexpr int kSortSmem = (34 * kMaxExperts + 32) * (int)sizeof(int);  // at most

template <int C>
__global__ void __launch_bounds__(1024) sort_kernel(const SortArgs a) {
  pdl_wait();
  pdl_launch();
  extern __shared__ int sm[];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = C > 1 ? (int)cluster.block_rank() : 0;
  const int nt = blockDim.x, tid = threadIdx.x, nw = nt >> 5, warp = tid >> 5, lane = tid & 31;
  int* hist = sm;                 // [cw][E]
  int* total = hist + a.cw * a.E; // [E] pairs of each expert in this CTA
  int* off = total + a.E;         // [E] first row of this CTA's pairs of each expert
  int* part = off + a.E;          // [32] warp sums of the scan
  long long first = (long long)(rank * a.cw + warp) * a.run;
  if (warp >= a.cw || first > a.n) first = a.n;
  const int lo = (int)first, hi = warp < a.cw && first + a.run < a.n ? (int)(first + a.run) : a.n;
  // the pairs from i0 on, -1 where there is none or its expert is outside
  auto keys = [&](int i0, int (&key)[kBatch]) {
    long long e[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) e[q] = i0 + 32 * q + lane < hi ? a.idx[i0 + 32 * q + lane] : -1;
#pragma unroll
    for (int q = 0; q < kBatch; ++q) key[q] = e[q] >= 0 && e[q] < a.E ? (int)e[q] : -1;
  };
  int key[kBatch];
  if (lo < hi) keys(lo, key);
  for (int i = tid; i < a.cw * a.E; i += nt) hist[i] = 0;
  __syncthreads();
  int* mine = hist + warp * a.E;
  for (int i0 = lo; i0 < hi; i0 += 32 * kBatch) {
    if (i0 > lo) keys(i0, key);
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
      if (key[q] >= 0) atomicAdd(&mine[key[q]], 1);
  }
  __syncthreads();
  for (int e = tid; e < a.E; e += nt) {
    int sum = 0;
    for (int w = 0; w < a.cw; ++w) {
      const int c = hist[w * a.E + e];
      hist[w * a.E + e] = sum;
      sum += c;
    }
    total[e] = sum;
  }
  if (C > 1) cluster.sync();
  // exclusive prefix over the experts of the whole cluster's counts, nt experts at a time
  int carry = 0;
  for (int e0 = 0; e0 < a.E; e0 += nt) {
    const int e = e0 + tid;
    int before = 0, all = 0;
    if (e < a.E) {
      int v[C];
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = C == 1 ? total[e] : cluster.map_shared_rank(total, c)[e];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (c < rank) before += v[c];
        all += v[c];
      }
    }
    int inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    int p = lane < nw ? part[lane] : 0;  // every warp scans the warps' sums
    const int own = p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += v;
    }
    const int start = carry + __shfl_sync(0xffffffffu, p - own, warp) + inc - all;
    carry += __shfl_sync(0xffffffffu, p, 31);
    if (e < a.E) {
      off[e] = start + before;
      if (rank == 0) a.offsets[e] = start;
    }
    __syncthreads();
  }
  if (rank == 0 && tid == 0) a.offsets[a.E] = carry;
  if (hi - lo > 32 * kBatch) keys(lo, key);
  for (int i0 = lo; i0 < hi; i0 += 32 * kBatch) {
    int next[kBatch];
    if (i0 + 32 * kBatch < hi) keys(i0 + 32 * kBatch, next);
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int i = i0 + 32 * q + lane;
      if (i0 + 32 * q >= hi) break;
      const unsigned same = __match_any_sync(0xffffffffu, key[q]);
      const bool ok = key[q] >= 0;
      int p = -1;
      if (ok) p = off[key[q]] + mine[key[q]] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (ok && (same >> lane) == 1u) mine[key[q]] += __popc(same);  // the last lane of each expert
      __syncwarp();
      if (i < hi) {
        a.pos[i] = p;
        if (ok) a.src[p] = i;
      }
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) key[q] = next[q];
  }
  // rows behind the last pair
  for (int i = carry + rank * nt + tid; i < a.n; i += C * nt) a.src[i] = -1;
  if (C > 1) cluster.sync();  // no CTA leaves while another may still read its totals
}

// ------------------------------------------------------------------ rows
// U: the unit of a copy, the widest that divides the row and the addresses. A CTA takes one token and
// a stretch of its row: the token's units are read once and written to its k places.
template <typename U>
__global__ void dispatch_kernel(const U* __restrict__ x, const float* __restrict__ s, const int* __restrict__ pos,
                                const int* __restrict__ offsets, int E, int k, int n, long long units, U* __restrict__ xs,
                                float* __restrict__ ss) {
  pdl_wait();
  pdl_launch();
  const long long t = blockIdx.x;
  __shared__ int place[kMaxTopk];
  if (threadIdx.x < k) {
    const int p = pos[t * k + threadIdx.x];
    place[threadIdx.x] = p >= 0 && p < n ? p : -1;
  }
  __syncthreads();
  const int live = min(max(offsets[E], 0), n);
  const long long c0 = (long long)blockIdx.y * blockDim.x + threadIdx.x, step = (long long)gridDim.y * blockDim.x;
  for (long long c = c0; c < units; c += step) {
    const U v = x[t * units + c];
    for (int j = 0; j < k; ++j)
      if (place[j] >= 0) xs[place[j] * units + c] = v;
  }
  // this CTA's share of the rows behind the last pair: those with its pairs' numbers
  for (int j = 0; j < k; ++j) {
    const long long r = t * k + j;
    if (r < live) continue;
    for (long long c = c0; c < units; c += step) xs[r * units + c] = U{};
    if (ss && c0 == 0) ss[r] = 0.f;
  }
  if (ss && blockIdx.y == 0 && threadIdx.x < k && place[threadIdx.x] >= 0) ss[place[threadIdx.x]] = s[t];
}

// VEC values of a row as loaded (16 bytes, or one value where the row or an address is not a multiple of 16
// bytes): they stay packed until they are used, which keeps registers few and warps many.
template <typename T, int VEC>
struct Raw {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = p[0]; }
  __device__ __forceinline__ void get(float (&o)[VEC]) const { o[0] = (float)v; }
};
template <>
struct Raw<__nv_bfloat16, 8> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
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
  __device__ __forceinline__ void get(float (&o)[4]) const { o[0] = u.x; o[1] = u.y; o[2] = u.z; o[3] = u.w; }
};

template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    p[0] = (T)v[0];
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

// y[t] in fp32, choices added in order j, rounded once.
constexpr int kRows = 4;
template <typename T, int VEC>
__global__ void __launch_bounds__(256, 7) combine_kernel(const T* __restrict__ ys, const int* __restrict__ pos, const float* __restrict__ wt, int k, int n,
                               long long width, T* __restrict__ y) {
  pdl_wait();
  pdl_launch();
  const long long t = blockIdx.x;
  __shared__ int place[kMaxTopk];
  __shared__ float weight[kMaxTopk];
  if (threadIdx.x < k) {
    const int p = pos[t * k + threadIdx.x];
    place[threadIdx.x] = p >= 0 && p < n ? p : -1;
    weight[threadIdx.x] = wt ? wt[t * k + threadIdx.x] : 1.0f;
  }
  __syncthreads();
  const long long step = (long long)gridDim.y * blockDim.x * VEC;
  for (long long c = ((long long)blockIdx.y * blockDim.x + threadIdx.x) * VEC; c < width; c += step) {
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    for (int j0 = 0; j0 < k; j0 += kRows) {  // loads of kRows choices at once
      Raw<T, VEC> raw[kRows];
#pragma unroll
      for (int q = 0; q < kRows; ++q) {
        const int p = j0 + q < k ? place[j0 + q] : -1;
        if (p >= 0) raw[q].load(ys + p * width + c);
      }
#pragma unroll
      for (int q = 0; q < kRows; ++q) {
        if (j0 + q >= k || place[j0 + q] < 0) continue;
        float v[VEC];
        raw[q].get(v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = fmaf(weight[j0 + q], v[i], acc[i]);
      }
    }
    store_row<T, VEC>(y + t * width + c, acc);
  }
}

// One CTA for kRows choices of a token: its dy row is read once for them, their rows of ys are read, their rows
// of dys written, and dwt's dot products summed lane, warp, block, in a fixed order.
template <typename T, int VEC>
__global__ void __launch_bounds__(256, 6) combine_grad_kernel(const T* __restrict__ dy, const T* __restrict__ ys,
                                                              const int* __restrict__ pos, const float* __restrict__ wt,
                                                              const int* __restrict__ offsets, int E, int k, int n,
                                                              long long width, T* __restrict__ dys, float* __restrict__ dwt) {
  pdl_wait();
  pdl_launch();
  const int batches = (k + kRows - 1) / kRows;
  const long long t = blockIdx.x / batches;
  const int j0 = blockIdx.x % batches * kRows;
  __shared__ float part[kRows][32];
  const int live = min(max(offsets[E], 0), n);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int place[kRows];
  float w[kRows], sum[kRows];
#pragma unroll
  for (int q = 0; q < kRows; ++q) {
    const long long r = t * k + j0 + q;
    const int p = j0 + q < k ? pos[r] : -1;
    place[q] = p >= 0 && p < n ? p : -1;
    w[q] = wt && place[q] >= 0 ? wt[r] : 1.0f;
    sum[q] = 0.f;
  }
  for (long long c = threadIdx.x * VEC; c < width; c += blockDim.x * VEC) {
    Raw<T, VEC> rg, rv[kRows];
    rg.load(dy + t * width + c);
    if (dwt) {
#pragma unroll
      for (int q = 0; q < kRows; ++q)
        if (place[q] >= 0) rv[q].load(ys + place[q] * width + c);
    }
    float g[VEC];
    rg.get(g);
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      if (place[q] < 0) continue;
      float v[VEC];
      if (dwt) {
        rv[q].get(v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[q] = fmaf(g[i], v[i], sum[q]);
      }
      if (dys) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = g[i] * w[q];
        store_row<T, VEC>(dys + place[q] * width + c, v);
      }
    }
  }
  if (dys) {
    for (int q = 0; q < kRows && j0 + q < k; ++q) {
      const long long r = t * k + j0 + q;
      if (r < live) continue;  // else this choice's number is that of a row behind the last
      const float zero[VEC] = {};
      for (long long c = threadIdx.x * VEC; c < width; c += blockDim.x * VEC) store_row<T, VEC>(dys + r * width + c, zero);
    }
  }
  if (dwt) {
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      sum[q] = warp_sum(sum[q]);
      if (lane == 0) part[q][warp] = sum[q];
    }
    __syncthreads();
    if (warp < kRows && j0 + warp < k) {
      const float s = warp_sum(lane < nw ? part[warp][lane] : 0.f);
      if (lane == 0) dwt[t * k + j0 + warp] = s;
    }
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// CTAs of one token's row: more than one while the tokens alone leave SMs idle
dim3 row_grid(long long P, long long units, int threads) {
  long long y = (units + threads - 1) / threads;
  const long long want = (4LL * sm_count() + P - 1) / P;
  if (y > want) y = want;
  return dim3((unsigned)P, (unsigned)(y < 1 ? 1 : y));
}

int threads_for(long long units) {
  int t = 32;
  while (t < units && t < 256) t *= 2;
  return t;
}

int check_order(const char* name, long long P, int k, int E) {
  DSMOE_REQUIRE(P > 0 && k > 0 && k <= kMaxTopk && P < (1LL << 30) && P * k < (1LL << 30), DSMOE_ERR_ARG,
                "%s: %lld tokens with %d choices (1..%d choices, fewer than 2^30 pairs)", name, P, k, kMaxTopk);
  DSMOE_REQUIRE(E > 0 && E <= kMaxExperts, DSMOE_ERR_ARG, "%s: %d experts (1..%d)", name, E, kMaxExperts);
  return DSMOE_OK;
}

template <typename U>
void dispatch(const void* x, const float* s, const int* pos, const int* offsets, int E, long long P, int k, long long row_bytes,
              void* xs, float* ss, cudaStream_t st) {
  const long long units = row_bytes / (long long)sizeof(U);
  int th = threads_for(units);
  if (th < k) th = 64;  // the first k threads read the places
  launch_pdl(dispatch_kernel<U>, row_grid(P, units, th), dim3(th), 0, st, (const U*)x, s, pos, offsets, E, k, (int)(P * k), units,
             (U*)xs, ss);
}

template <typename T>
void combine(const void* ys, const int* pos, const float* wt, long long P, int k, long long width, bool wide, void* y,
             cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const long long units = wide ? width / V : width;
  int th = threads_for(units);
  if (th < k) th = 64;
  const dim3 grid = row_grid(P, units, th);
  launch_pdl(wide ? combine_kernel<T, V> : combine_kernel<T, 1>, grid, dim3(th), 0, st, (const T*)ys, pos, wt, k, (int)(P * k),
             width, (T*)y);
}

template <typename T>
void combine_grad(const void* dy, const void* ys, const int* pos, const float* wt, const int* offsets, int E, long long P, int k,
                  long long width, bool wide, void* dys, float* dwt, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  int th = threads_for(wide ? width / V : width);
  if (th < 32 * kRows) th = 32 * kRows;  // a warp joins each choice's sums
  const int n = (int)(P * k), grid = (int)(P * ((k + kRows - 1) / kRows));
  launch_pdl(wide ? combine_grad_kernel<T, V> : combine_grad_kernel<T, 1>, dim3(grid), dim3(th), 0, st, (const T*)dy, (const T*)ys,
             pos, wt, offsets, E, k, n, width, (T*)dys, dwt);
}

// Whether the current device runs clusters of 16 CTAs (more than 8 is not portable); asked once per device.
bool sixteen() {
  static std::atomic<int> known[64];  // 0 unknown, 1 yes, 2 no
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev > 63) return false;
  int is = known[dev].load();
  if (!is) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(1024);
    cfg.dynamicSmemBytes = kSortSmem;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 16;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int n = 0;
    is = cudaFuncSetAttribute(sort_kernel<16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                 cudaFuncSetAttribute(sort_kernel<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSmem) == cudaSuccess &&
                 cudaOccupancyMaxActiveClusters(&n, sort_kernel<16>, &cfg) == cudaSuccess && n > 0
             ? 1
             : 2;
    cudaGetLastError();
    known[dev].store(is);
  }
  return is == 1;
}

}  // namespace tokens
}  // namespace dsmoe

using namespace dsmoe;

extern "C" int dsmoe_sort_tokens(const int64_t* idx, long long P, int k, int n_experts, int* pos, int* src, int* offsets,
                                 void* stream) {
  int rc = tokens::check_order("sort_tokens", P, k, n_experts);
  if (rc) return rc;
  DSMOE_REQUIRE(idx && pos && src && offsets, DSMOE_ERR_ARG, "sort_tokens: null pointer");
  DSMOE_REQUIRE(((uintptr_t)idx & 7) == 0 && (((uintptr_t)pos | (uintptr_t)src | (uintptr_t)offsets) & 3) == 0, DSMOE_ERR_ALIGN,
                "sort_tokens: misaligned pointer");
  const long long pairs = P * k;
  DSMOE_REQUIRE(!overlap({{pos, pairs * 4}, {src, pairs * 4}, {offsets, (n_experts + 1) * 4}}, {{idx, pairs * 8}}), DSMOE_ERR_ARG,
                "sort_tokens: outputs overlap");
  tokens::SortArgs a{idx, pos, src, offsets, (int)(P * k), n_experts, 0, 0};
  // 131072 pairs of 384 experts: 26.8 us with 8 CTAs, 16.9 with 16 (24576 pairs 8.1 and 6.3; 12282: 6.5 and 6.6)
  const int C = a.n > 16384 && tokens::sixteen() ? 16 : a.n > 4096 ? 8 : 1;
  const int cw = (a.n / C + 127) / 128;  // a warp for each 128 pairs
  a.cw = cw < 1 ? 1 : cw > 32 ? 32 : cw;
  a.run = (int)((((long long)a.n + (long long)C * a.cw - 1) / (C * a.cw) + 31) / 32 * 32);
  const int ew = (n_experts + 31) / 32;  // a thread for each expert in the scan
  const int nw = a.cw > ew ? a.cw : ew;
  const size_t smem = ((size_t)(a.cw + 2) * n_experts + 32) * sizeof(int);
  auto kern = C == 1 ? tokens::sort_kernel<1> : C == 8 ? tokens::sort_kernel<8> : tokens::sort_kernel<16>;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, tokens::kSortSmem) != cudaSuccess)
    return cuda_status("sort_tokens");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(C);
  cfg.blockDim = dim3(nw * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = C;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kern, a);
  return cuda_status("sort_tokens");
}

extern "C" int dsmoe_dispatch_rows(const void* x, const float* s, const int* pos, const int* offsets, int n_experts, long long P,
                                   int k, long long row_bytes, void* xs, float* ss, void* stream) {
  int rc = tokens::check_order("dispatch_rows", P, k, n_experts);
  if (rc) return rc;
  DSMOE_REQUIRE(x && pos && offsets && xs && (!s == !ss), DSMOE_ERR_ARG, "dispatch_rows: null pointer");
  DSMOE_REQUIRE(row_bytes > 0 && row_bytes < (1LL << 31), DSMOE_ERR_ARG, "dispatch_rows: row of %lld bytes", row_bytes);
  DSMOE_REQUIRE((((uintptr_t)pos | (uintptr_t)offsets | (uintptr_t)s | (uintptr_t)ss) & 3) == 0, DSMOE_ERR_ALIGN,
                "dispatch_rows: misaligned pointer");
  DSMOE_REQUIRE(!overlap({{xs, P * k * row_bytes}, {ss, P * k * 4}},
                         {{x, P * row_bytes}, {s, P * 4}, {pos, P * k * 4}, {offsets, (n_experts + 1) * 4}}),
                DSMOE_ERR_ARG, "dispatch_rows: outputs overlap inputs");
  cudaStream_t st = (cudaStream_t)stream;
  const uintptr_t any = (uintptr_t)x | (uintptr_t)xs | (uintptr_t)row_bytes;
  if ((any & 15) == 0) tokens::dispatch<uint4>(x, s, pos, offsets, n_experts, P, k, row_bytes, xs, ss, st);
  else if ((any & 3) == 0) tokens::dispatch<uint32_t>(x, s, pos, offsets, n_experts, P, k, row_bytes, xs, ss, st);
  else if ((any & 1) == 0) tokens::dispatch<uint16_t>(x, s, pos, offsets, n_experts, P, k, row_bytes, xs, ss, st);
  else tokens::dispatch<uint8_t>(x, s, pos, offsets, n_experts, P, k, row_bytes, xs, ss, st);
  return cuda_status("dispatch_rows");
}

extern "C" int dsmoe_combine_rows(const void* ys, int dtype, const int* pos, const float* wt, long long P, int k, long long width,
                                  void* y, void* stream) {
  int rc = tokens::check_order("combine_rows", P, k, 1);
  if (rc) return rc;
  DSMOE_REQUIRE(ys && pos && y, DSMOE_ERR_ARG, "combine_rows: null pointer");
  DSMOE_REQUIRE(dtype == DSMOE_DTYPE_F32 || dtype == DSMOE_DTYPE_BF16, DSMOE_ERR_ARG, "combine_rows: dtype %d", dtype);
  DSMOE_REQUIRE(width > 0 && width < (1LL << 29), DSMOE_ERR_ARG, "combine_rows: width %lld", width);
  const int sz = dtype == DSMOE_DTYPE_F32 ? 4 : 2;
  const uintptr_t any = (uintptr_t)ys | (uintptr_t)y;
  DSMOE_REQUIRE((any & (sz - 1)) == 0 && (((uintptr_t)pos | (uintptr_t)wt) & 3) == 0, DSMOE_ERR_ALIGN,
                "combine_rows: misaligned pointer");
  DSMOE_REQUIRE(!overlap({{y, P * width * sz}}, {{ys, P * k * width * sz}, {pos, P * k * 4}, {wt, P * k * 4}}), DSMOE_ERR_ARG,
                "combine_rows: y overlaps an input");
  const bool wide = ((any | (uintptr_t)(width * sz)) & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == DSMOE_DTYPE_F32) tokens::combine<float>(ys, pos, wt, P, k, width, wide, y, st);
  else tokens::combine<__nv_bfloat16>(ys, pos, wt, P, k, width, wide, y, st);
  return cuda_status("combine_rows");
}

extern "C" int dsmoe_combine_grad(const void* dy, const void* ys, int dtype, const int* pos, const float* wt, const int* offsets,
                                  int n_experts, long long P, int k, long long width, void* dys, float* dwt, void* stream) {
  int rc = tokens::check_order("combine_grad", P, k, n_experts);
  if (rc) return rc;
  DSMOE_REQUIRE(dy && pos && offsets && (dys || dwt) && (ys || !dwt), DSMOE_ERR_ARG, "combine_grad: null pointer");
  DSMOE_REQUIRE(dtype == DSMOE_DTYPE_F32 || dtype == DSMOE_DTYPE_BF16, DSMOE_ERR_ARG, "combine_grad: dtype %d", dtype);
  DSMOE_REQUIRE(width > 0 && width < (1LL << 29), DSMOE_ERR_ARG, "combine_grad: width %lld", width);
  const int sz = dtype == DSMOE_DTYPE_F32 ? 4 : 2;
  const uintptr_t any = (uintptr_t)dy | (uintptr_t)ys | (uintptr_t)dys;
  DSMOE_REQUIRE((any & (sz - 1)) == 0 &&
                    (((uintptr_t)pos | (uintptr_t)wt | (uintptr_t)offsets | (uintptr_t)dwt) & 3) == 0,
                DSMOE_ERR_ALIGN, "combine_grad: misaligned pointer");
  const long long nb = P * width * sz;
  DSMOE_REQUIRE(!overlap({{dys, nb * k}, {dwt, P * k * 4}},
                         {{dy, nb}, {ys, nb * k}, {pos, P * k * 4}, {wt, P * k * 4}, {offsets, (n_experts + 1) * 4}}),
                DSMOE_ERR_ARG, "combine_grad: outputs overlap inputs");
  const bool wide = ((any | (uintptr_t)(width * sz)) & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == DSMOE_DTYPE_F32)
    tokens::combine_grad<float>(dy, ys, pos, wt, offsets, n_experts, P, k, width, wide, dys, dwt, st);
  else
    tokens::combine_grad<__nv_bfloat16>(dy, ys, pos, wt, offsets, n_experts, P, k, width, wide, dys, dwt, st);
  return cuda_status("combine_grad");
}
