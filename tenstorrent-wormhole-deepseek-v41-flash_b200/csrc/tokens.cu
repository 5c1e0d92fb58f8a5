// Tokens sorted by expert and back, and the gradients of both directions:
//   dsmoe_sort_tokens      idx [P, k] -> pos [P, k], src [P k], offsets [E + 1]
//   dsmoe_dispatch_rows    xs[pos[t, j]] = x[t]                     (rows behind the last: zero)
//   dsmoe_combine_rows     y[t] = sum_j wt[t, j] ys[pos[t, j]]      (wt = 1: the gradient of dispatch)
//   dsmoe_combine_grad     dys[pos[t, j]] = wt[t, j] dy[t],  dwt[t, j] = <dy[t], ys[pos[t, j]]>
// The order is that of (expert, token, choice): a stable counting sort, so nothing depends on the
// order in which threads arrive. Choices outside 0..E-1 are dropped (pos = -1) and the rows behind
// offsets[E] hold zeros.
#include <cooperative_groups.h>

#include "common.cuh"

namespace dsmoe {
namespace tokens {

namespace cg = cooperative_groups;

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 64;

// ------------------------------------------------------------------ sort
// One cluster of C CTAs (C = 1 for few pairs). Warp w of CTA c owns a contiguous run of pairs and a
// row of counters in shared memory. Count; prefix over the warps of the CTA, the CTAs of the cluster
// (their totals read through distributed shared memory) and the experts; then each warp walks its run
// again, 32 pairs at a time, and ranks equal experts among its lanes by match.
struct SortArgs {
  const int64_t* idx;
  int* pos;
  int* src;
  int* offsets;
  int n, E;
  int run;  // pairs per warp, a multiple of 32
};

__global__ void __launch_bounds__(1024) sort_kernel(const SortArgs a) {
  extern __shared__ int sm[];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int nt = blockDim.x, tid = threadIdx.x, nw = nt >> 5, warp = tid >> 5, lane = tid & 31;
  int* hist = sm;               // [nw][E]
  int* total = hist + nw * a.E; // [E] pairs of each expert in this CTA
  int* off = total + a.E;       // [E] first row of each expert, then of this CTA's pairs of it
  int* part = off + a.E;        // [32] warp sums of the scan
  for (int i = tid; i < nw * a.E; i += nt) hist[i] = 0;
  __syncthreads();
  int* mine = hist + warp * a.E;
  const long long first = (long long)(rank * nw + warp) * a.run;
  const int lo = first < a.n ? (int)first : a.n, hi = first + a.run < a.n ? (int)(first + a.run) : a.n;
  for (int i = lo + lane; i < hi; i += 32) {
    const long long e = a.idx[i];
    if (e >= 0 && e < a.E) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  for (int e = tid; e < a.E; e += nt) {
    int sum = 0;
    for (int w = 0; w < nw; ++w) {
      const int c = hist[w * a.E + e];
      hist[w * a.E + e] = sum;
      sum += c;
    }
    total[e] = sum;
  }
  cluster.sync();
  // exclusive prefix over the experts of the whole cluster's counts, nt experts at a time
  int carry = 0;
  for (int e0 = 0; e0 < a.E; e0 += nt) {
    const int e = e0 + tid;
    int before = 0, all = 0;
    if (e < a.E) {
      for (int c = 0; c < C; ++c) {
        const int v = C == 1 ? total[e] : cluster.map_shared_rank(total, c)[e];
        if (c < rank) before += v;
        all += v;
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
    int below = carry, sum = 0;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) below += part[w];
      sum += part[w];
    }
    __syncthreads();
    if (e < a.E) {
      const int start = below + inc - all;
      off[e] = start + before;
      if (rank == 0) a.offsets[e] = start;
    }
    carry += sum;
  }
  if (rank == 0 && tid == 0) a.offsets[a.E] = carry;
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    long long e = -1;
    if (i < hi) e = a.idx[i];
    const bool ok = e >= 0 && e < a.E;
    const int key = ok ? (int)e : -1;
    const unsigned same = __match_any_sync(0xffffffffu, key);
    int p = -1;
    if (ok) p = off[key] + mine[key] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (ok && (same >> lane) == 1u) mine[key] += __popc(same);  // the last lane of each expert
    __syncwarp();
    if (i < hi) {
      a.pos[i] = p;
      if (ok) a.src[p] = i;
    }
  }
  // rows behind the last pair
  for (int i = carry + rank * nt + tid; i < a.n; i += C * nt) a.src[i] = -1;
  cluster.sync();  // no CTA leaves while another may still read its totals
}

// ------------------------------------------------------------------ rows
// U: the unit of a copy, the widest that divides the row and the addresses. A CTA takes one token and
// a stretch of its row: the token's units are read once and written to its k places.
template <typename U>
__global__ void dispatch_kernel(const U* __restrict__ x, const float* __restrict__ s, const int* __restrict__ pos,
                                const int* __restrict__ offsets, int E, int k, int n, long long units, U* __restrict__ xs,
                                float* __restrict__ ss) {
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

template <typename T, int VEC>
__device__ __forceinline__ void load_row(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = (float)p[0];
  } else if constexpr (sizeof(T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
    const float4 u = *reinterpret_cast<const float4*>(p);
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  }
}

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
template <typename T, int VEC>
__global__ void combine_kernel(const T* __restrict__ ys, const int* __restrict__ pos, const float* __restrict__ wt, int k, int n,
                               long long width, T* __restrict__ y) {
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
    for (int j = 0; j < k; ++j) {
      if (place[j] < 0) continue;
      float v[VEC];
      load_row<T, VEC>(ys + place[j] * width + c, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] = fmaf(weight[j], v[i], acc[i]);
    }
    store_row<T, VEC>(y + t * width + c, acc);
  }
}

// One CTA per token; dwt's dot products are summed lane, warp, block, in a fixed order.
template <typename T, int VEC>
__global__ void combine_grad_kernel(const T* __restrict__ dy, const T* __restrict__ ys, const int* __restrict__ pos,
                                    const float* __restrict__ wt, const int* __restrict__ offsets, int E, int k, int n,
                                    long long width, T* __restrict__ dys, float* __restrict__ dwt) {
  const long long t = blockIdx.x;
  __shared__ int place[kMaxTopk];
  __shared__ float weight[kMaxTopk];
  __shared__ float part[32];
  if (threadIdx.x < k) {
    const int p = pos[t * k + threadIdx.x];
    place[threadIdx.x] = p >= 0 && p < n ? p : -1;
    weight[threadIdx.x] = wt ? wt[t * k + threadIdx.x] : 1.0f;
  }
  __syncthreads();
  const int live = min(max(offsets[E], 0), n);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  for (int j = 0; j < k; ++j) {
    const int p = place[j];
    float sum = 0.f;
    if (p >= 0) {
      for (long long c = threadIdx.x * VEC; c < width; c += blockDim.x * VEC) {
        float g[VEC], v[VEC];
        load_row<T, VEC>(dy + t * width + c, g);
        if (dwt) {
          load_row<T, VEC>(ys + p * width + c, v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum = fmaf(g[i], v[i], sum);
        }
        if (dys) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[i] = g[i] * weight[j];
          store_row<T, VEC>(dys + p * width + c, v);
        }
      }
    }
    if (dwt) {
      sum = warp_sum(sum);
      if (lane == 0) part[warp] = sum;
      __syncthreads();
      if (warp == 0) {
        sum = warp_sum(lane < nw ? part[lane] : 0.f);
        if (lane == 0) dwt[t * k + j] = sum;
      }
      __syncthreads();
    }
    const long long r = t * k + j;
    if (dys && r >= live) {
      const float zero[VEC] = {};
      for (long long c = threadIdx.x * VEC; c < width; c += blockDim.x * VEC) store_row<T, VEC>(dys + r * width + c, zero);
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
  dispatch_kernel<U><<<row_grid(P, units, th), th, 0, st>>>((const U*)x, s, pos, offsets, E, k, (int)(P * k), units, (U*)xs, ss);
}

template <typename T>
void combine(const void* ys, const int* pos, const float* wt, long long P, int k, long long width, bool wide, void* y,
             cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const long long units = wide ? width / V : width;
  int th = threads_for(units);
  if (th < k) th = 64;
  const dim3 grid = row_grid(P, units, th);
  if (wide) combine_kernel<T, V><<<grid, th, 0, st>>>((const T*)ys, pos, wt, k, (int)(P * k), width, (T*)y);
  else combine_kernel<T, 1><<<grid, th, 0, st>>>((const T*)ys, pos, wt, k, (int)(P * k), width, (T*)y);
}

template <typename T>
void combine_grad(const void* dy, const void* ys, const int* pos, const float* wt, const int* offsets, int E, long long P, int k,
                  long long width, bool wide, void* dys, float* dwt, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  int th = threads_for(wide ? width / V : width);
  if (th < k) th = 64;
  if (wide)
    combine_grad_kernel<T, V><<<(unsigned)P, th, 0, st>>>((const T*)dy, (const T*)ys, pos, wt, offsets, E, k, (int)(P * k), width,
                                                          (T*)dys, dwt);
  else
    combine_grad_kernel<T, 1><<<(unsigned)P, th, 0, st>>>((const T*)dy, (const T*)ys, pos, wt, offsets, E, k, (int)(P * k), width,
                                                          (T*)dys, dwt);
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
  tokens::SortArgs a{idx, pos, src, offsets, (int)(P * k), n_experts, 0};
  const int C = a.n > 4096 ? 8 : 1;
  int nw = (a.n / C + 127) / 128;  // a warp for each 128 pairs
  nw = nw < 4 ? 4 : nw > 32 ? 32 : nw;
  a.run = (int)((((long long)a.n + (long long)C * nw - 1) / (C * nw) + 31) / 32 * 32);
  const size_t smem = ((size_t)(nw + 2) * n_experts + 32) * sizeof(int);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(tokens::sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (34 * tokens::kMaxExperts + 32) * (int)sizeof(int)) != cudaSuccess)
    return cuda_status("sort_tokens");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(C);
  cfg.blockDim = dim3(nw * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = C;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, tokens::sort_kernel, a);
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
  const bool wide = ((any | (uintptr_t)(width * sz)) & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == DSMOE_DTYPE_F32)
    tokens::combine_grad<float>(dy, ys, pos, wt, offsets, n_experts, P, k, width, wide, dys, dwt, st);
  else
    tokens::combine_grad<__nv_bfloat16>(dy, ys, pos, wt, offsets, n_experts, P, k, width, wide, dys, dwt, st);
  return cuda_status("combine_grad");
}
