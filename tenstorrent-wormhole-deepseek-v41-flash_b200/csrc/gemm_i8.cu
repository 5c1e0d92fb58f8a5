// Matrix products in 8-bit integers, a scale for each token and each channel:
//   dsmoe_int8_gemm          out[m, n] = (sum_k a[m, k] b[n, k]) a_s[m] b_s[n]
//   dsmoe_int8_grouped_gemm  the same with expert e's weights b[e] for rows offsets[e]..offsets[e+1]-1
// The integer sum is exact (int32: K <= 131071 keeps 128 * 128 * K below 2^31); it is converted to
// fp32 and multiplied by the two scales, and the product is rounded once to the output type.
//
// tcgen05.mma kind::i8 with the accumulators in tensor memory. The MMA's M side (128) holds weight
// rows and its N side (up to 256, in steps of 16) token rows, so an accumulator lane is a channel, a
// column is a token, and the epilogue's stores of one token are contiguous whatever N is. Both
// operands are K-major rows of 128-byte blocks, loaded by TMA with the 128-byte swizzle the MMA reads;
// rows and K behind the tensor's end arrive as zeros. The tokens of a tile start at any row (the TMA's
// row coordinate has no alignment), so a group needs no padding.
//   warp 0      producer: per 128-K block one load of 128 weight rows and one for each BR token rows
//   warp 1      MMA issuer, two accumulators in turn
//   warps 2-9   epilogue (two warps per 32-lane quadrant, splitting the tokens)
// Tiles are dealt round-robin to a persistent grid. Few tokens: SPLIT, a cluster of S CTAs shares a
// tile's K blocks and adds the S integer partials through distributed shared memory (exact, so the
// order does not matter); no workspace, nothing shared between calls.
// Every wait is bounded; where one expired, the outputs are NaN.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace dsmoe {
namespace gemm_i8 {

constexpr int NT = 320;       // 10 warps
constexpr int CT = 256;       // epilogue threads
constexpr int TM = 128;       // weight rows per tile (MMA M)
constexpr int MAXTT = 256;    // tokens per tile (MMA N)
constexpr int SPLIT_TT = 64;  // the same where K is split over a cluster
constexpr int MAXRS = 12;     // ring stages
constexpr int kMaxExperts = 1024;
constexpr int kMaxK = 131071;
constexpr uint64_t kWaitNs = 1000000000ull;

struct Args {
  CUtensorMap tb;      // weights [E N][K], box 128 x 128
  CUtensorMap ta;      // tokens [M][K], box 128 x BR
  const float* a_s;    // [M]
  const float* b_s;    // [E][N]
  const int* offsets;  // [E + 1], or null: one group of all M rows
  void* out;           // [M][N]
  int M, N, K, E, nkb, TT, BR, RS, NTN, S, out_f32;
};

struct Tile {
  int e, n0, m0, cols;  // expert, first channel, first token row, tokens
};

__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* tm, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// 16 accumulator columns of this warp's 32 lanes; load and wait in one statement.
__device__ __forceinline__ void ld16(uint32_t taddr, int (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
// The same address in the shared memory of another CTA of the cluster.
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void peer_arrive(uint64_t* bar, uint32_t rank) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(peer_addr(smem_u32(bar), rank)) : "memory");
}
__device__ __forceinline__ int peer_ld(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// mbar_wait whose success also orders the other CTAs' writes before their arrivals.
__device__ __forceinline__ bool cluster_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  const uint64_t t0 = globaltimer_ns();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (ok) return true;
    if (globaltimer_ns() - t0 > limit_ns) return false;
  }
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <bool SPLIT>
__global__ void __launch_bounds__(NT, 1) gemm_i8_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t gsm[];
  uint8_t* ring = gsm + ((1024 - (smem_u32(gsm) & 1023)) & 1023);
  const int SB = TM * 128 + a.TT * 128;  // stage bytes
  int* part = reinterpret_cast<int*>(ring + a.RS * SB);                       // SPLIT: [2][TT][TM]
  uint64_t* bars = reinterpret_cast<uint64_t*>(part + (SPLIT ? 2 * a.TT * TM : 0));
  uint64_t* full = bars;             // [MAXRS] stage landed
  uint64_t* empty = full + MAXRS;    // [MAXRS] stage read by its MMAs
  uint64_t* accf = empty + MAXRS;    // [2] accumulator complete
  uint64_t* acce = accf + 2;         // [2] accumulator read (8 warps)
  uint64_t* pfull = acce + 2;        // [2] SPLIT: every CTA's partial written
  uint64_t* pempty = pfull + 2;      // [2] SPLIT: this CTA's partial read by every CTA
  uint64_t* mdone = pempty + 2;      // [1] no MMA in flight
  uint32_t* tslot = reinterpret_cast<uint32_t*>(mdone + 1);
  volatile int* abortf = reinterpret_cast<volatile int*>(tslot + 1);
  int* wsum = reinterpret_cast<int*>(tslot + 2);  // [10]
  int* first = wsum + 10;            // [E + 1] first row of each group
  int* pre = first + a.E + 1;        // [E + 1] tiles before each group

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = SPLIT ? a.S : 1;
  const int rank = SPLIT ? blockIdx.x % S : 0;
  const int cid = blockIdx.x / S, ncl = gridDim.x / S;
  const int kb0 = rank * a.nkb / S, kb1 = (rank + 1) * a.nkb / S;

  if (tid == 0) {
    for (int s = 0; s < MAXRS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&accf[s], 1);
      mbar_init(&acce[s], 8);
      mbar_init(&pfull[s], S);
      mbar_init(&pempty[s], S);
    }
    mbar_init(mdone, 1);
    *abortf = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // groups of ceil(rows / TT) tiles, prefix over experts. Offsets that do not rise from 0 to at most M
  // describe no groups: no tile runs and the whole output is NaN.
  int tiles, behind = a.M;
  float fill = 0.f;
  if (a.offsets) {
    int bad = 0;
    for (int e = tid; e <= a.E; e += NT) {
      const int o = a.offsets[e];
      first[e] = o;
      bad |= o < (e ? a.offsets[e - 1] : 0) || o > (e ? a.M : 0);
    }
    bad = __syncthreads_or(bad);
    int carry = 0;
    for (int e0 = 0; e0 < a.E; e0 += NT) {
      const int e = e0 + tid;
      int inc = e < a.E && !bad ? (first[e + 1] - first[e] + a.TT - 1) / a.TT : 0;
      const int own = inc;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) wsum[warp] = inc;
      __syncthreads();
      int below = carry, sum = 0;
      for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) below += wsum[w];
        sum += wsum[w];
      }
      if (e < a.E) pre[e] = below + inc - own;
      carry += sum;
      __syncthreads();
    }
    if (tid == 0) pre[a.E] = carry;
    tiles = carry * a.NTN;
    behind = bad ? 0 : first[a.E];
    if (bad) fill = __int_as_float(0x7FC00000);
  } else {
    if (tid == 0) {
      first[0] = 0;
      first[1] = a.M;
      pre[0] = 0;
      pre[1] = (a.M + a.TT - 1) / a.TT;
    }
    tiles = (a.M + a.TT - 1) / a.TT * a.NTN;
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (SPLIT) cluster_sync();  // every CTA's barriers exist before the first remote arrival
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tslot;
  auto wait = [&](uint64_t* bar, uint32_t par) -> bool {
    if (*abortf) return false;
    if (!mbar_wait(bar, par, kWaitNs)) {
      *abortf = 1;
      return false;
    }
    return true;
  };
  // tile -> expert, channels, tokens. Tiles of one expert are neighbours, the tokens of one weight tile
  // in a row, so its bytes are in L2 when they are read again.
  auto locate = [&](int tile) -> Tile {
    int lo = 0, hi = a.E;  // the expert with pre[e] NTN <= tile < pre[e + 1] NTN
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] * a.NTN <= tile) lo = mid;
      else hi = mid;
    }
    const int mt = pre[lo + 1] - pre[lo], at = tile - pre[lo] * a.NTN;
    const int rows = first[lo + 1] - first[lo];
    const int per = ((rows + mt - 1) / mt + 15) & ~15;  // the group's rows spread evenly over its tiles
    const int m = (at % mt) * per;
    return Tile{lo, at / mt * TM, first[lo] + m, max(min(per, rows - m), 0)};
  };

  if (warp == 0) {
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&a.tb) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&a.ta) : "memory");
      int it = 0;
      bool ok = true;
      for (int tile = cid; tile < tiles && ok; tile += ncl) {
        const Tile t = locate(tile);
        const int nb = max((t.cols + a.BR - 1) / a.BR, 1);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % a.RS;
          if (it >= a.RS && !wait(&empty[s], ((it / a.RS) - 1) & 1)) {
            ok = false;
            break;
          }
          uint8_t* st = ring + s * SB;
          mbar_expect_tx(&full[s], (uint32_t)(TM * 128 + nb * a.BR * 128));
          tma_2d(st, &a.tb, kb * 128, t.e * a.N + t.n0, &full[s]);
          for (int b = 0; b < nb; ++b) tma_2d(st + TM * 128 + b * a.BR * 128, &a.ta, kb * 128, t.m0 + b * a.BR, &full[s]);
        }
      }
      // every copy issued has landed before the CTA may exit (the last use of each stage)
      for (int i = it - 1; i >= 0 && i >= it - a.RS; --i) mbar_wait(&full[i % a.RS], (i / a.RS) & 1, kWaitNs);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // D s32, A and B s8, both K-major
      const uint32_t idesc0 = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TM >> 4) << 24);
      const uint64_t da0 = desc_sw128(smem_u32(ring)), db0 = desc_sw128(smem_u32(ring + TM * 128));
      int it = 0, tc = 0;
      bool ok = true;
      for (int tile = cid; tile < tiles && ok; tile += ncl, ++tc) {
        const Tile t = locate(tile);
        const int ac = tc & 1;
        if (tc >= 2 && !wait(&acce[ac], ((tc >> 1) - 1) & 1)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t idesc = idesc0 | ((uint32_t)(max((t.cols + 15) >> 4, 1) * 2) << 17);
        const uint32_t d = tmem + (uint32_t)(ac * MAXTT);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % a.RS;
          if (!wait(&full[s], (it / a.RS) & 1)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t o = (uint64_t)(s * (SB >> 4));
#pragma unroll
          for (int q = 0; q < 4; ++q) mma_i8(d, da0 + o + 2u * q, db0 + o + 2u * q, idesc, (kb > kb0 || q > 0) ? 1u : 0u);
          commit(&empty[s]);
        }
        commit(&accf[ac]);
      }
      commit(mdone);  // no MMA may still run when the tensor memory is freed
      mbar_wait(mdone, 0, kWaitNs);
    }
  } else {
    const int ct = tid - 64;
    const int qd = warp & 3, half = (warp - 2) >> 2;
    const int row_l = 32 * qd + lane;
    const float nanv = __int_as_float(0x7FC00000);
    auto store = [&](long long t, int n, float v) {
      const long long o = t * a.N + n;
      if (a.out_f32) reinterpret_cast<float*>(a.out)[o] = v;
      else reinterpret_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(v);
    };
    int tc = 0;
    bool ok = true;
    for (int tile = cid; tile < tiles; tile += ncl, ++tc) {
      const Tile t = locate(tile);
      const int ac = tc & 1;
      ok = ok && wait(&accf[ac], (tc >> 1) & 1);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int groups = (t.cols + 15) >> 4;  // 16 tokens at a time, the two warps of a quadrant in turn
      const uint32_t tq = tmem + ((uint32_t)(32 * qd) << 16) + (uint32_t)(ac * MAXTT);
      if (!SPLIT) {
        const int n = t.n0 + row_l;
        const float bs = n < a.N ? a.b_s[(long long)t.e * a.N + n] : 0.f;
        for (int g = half; g < groups; g += 2) {
          int v[16];
          ld16(tq + 16u * g, v);
          const int c = 16 * g + (lane & 15);
          const float as = c < t.cols ? a.a_s[t.m0 + c] : 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float sc = __shfl_sync(0xffffffffu, as, i);
            if (n < a.N && 16 * g + i < t.cols) store(t.m0 + 16 * g + i, n, ok ? (float)v[i] * sc * bs : nanv);
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&acce[ac]);
      } else {
        int* mine = part + ac * a.TT * TM;
        if (ok && tc >= 2) {
          ok = cluster_wait(&pempty[ac], ((tc >> 1) - 1) & 1, kWaitNs);
          if (!ok) *abortf = 1;
        }
        for (int g = half; g < groups; g += 2) {
          int v[16];
          ld16(tq + 16u * g, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) mine[(16 * g + i) * TM + row_l] = v[i];
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&acce[ac]);
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        named_bar_sync(1, CT);
        if (ct < S) peer_arrive(&pfull[ac], (uint32_t)ct);
        if (ok) {
          ok = cluster_wait(&pfull[ac], (tc >> 1) & 1, kWaitNs);
          if (!ok) *abortf = 1;
        }
        // this CTA finishes channels rank TM / S .. of the tile, for every token
        const int rows = TM / S, r = rank * rows + ct % rows, n = t.n0 + r;
        if (n < a.N) {
          const float bs = a.b_s[(long long)t.e * a.N + n];
          for (int c = ct / rows; c < t.cols; c += CT / rows) {
            const uint32_t at = smem_u32(mine + c * TM + r);
            int sum = 0;
            if (ok)
              for (int z = 0; z < S; ++z) sum += peer_ld(peer_addr(at, (uint32_t)z));
            store(t.m0 + c, n, ok ? (float)sum * a.a_s[t.m0 + c] * bs : nanv);
          }
        }
        named_bar_sync(1, CT);
        if (ct < S) peer_arrive(&pempty[ac], (uint32_t)ct);
      }
    }
    // rows behind the last group
    {
      const long long from = (long long)behind * a.N, to = (long long)a.M * a.N;
      for (long long i = from + (long long)blockIdx.x * CT + ct; i < to; i += (long long)gridDim.x * CT) {
        if (a.out_f32) reinterpret_cast<float*>(a.out)[i] = fill;
        else reinterpret_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(fill);
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (SPLIT) cluster_sync();  // no CTA leaves while another may still read its partials
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ------------------------------------------------------------------ host side
std::atomic<void*> g_encode{nullptr};

int encoder(PFN_cuTensorMapEncodeTiled_v12000* fn) {
  void* p = g_encode.load();
  if (!p) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess || !p) {
      cudaGetLastError();
      set_error("int8_gemm: no cuTensorMapEncodeTiled entry point");
      return DSMOE_ERR_CUDA;
    }
    g_encode.store(p);
  }
  *fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  return DSMOE_OK;
}

// The current device's SM count and shared memory limit, and the kernels' attribute set once per device.
int device_limits(const char* name, int* sms, int* optin) {
  static std::atomic<int> known[64][2];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return cuda_status(name);
  const int slot = dev & 63;
  *sms = known[slot][0].load(std::memory_order_acquire);
  *optin = known[slot][1].load(std::memory_order_acquire);
  if (*sms && dev < 64) return DSMOE_OK;
  if (cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      cudaDeviceGetAttribute(optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_i8_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, *optin) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_i8_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, *optin) != cudaSuccess)
    return cuda_status(name);
  known[slot][1].store(*optin, std::memory_order_release);
  known[slot][0].store(*sms, std::memory_order_release);
  return DSMOE_OK;
}

int encode(PFN_cuTensorMapEncodeTiled_v12000 fn, CUtensorMap* m, const void* p, long long K, long long rows, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)K};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  DSMOE_REQUIRE(r == CUDA_SUCCESS, DSMOE_ERR_CUDA, "int8_gemm: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return DSMOE_OK;
}

int run(const char* name, const int8_t* x, const float* a_s, long long M, long long K, const int8_t* b, const float* b_s,
        long long N, const int* offsets, int E, void* out, int out_dtype, void* stream) {
  DSMOE_REQUIRE(x && a_s && b && b_s && out, DSMOE_ERR_ARG, "%s: null pointer", name);
  DSMOE_REQUIRE(M > 0 && N > 0 && M < (1LL << 31) - 512 && N * E < (1LL << 31) - 512, DSMOE_ERR_ARG, "%s: M %lld, N %lld, E %d",
                name, M, N, E);
  DSMOE_REQUIRE(K > 0 && K % 16 == 0 && K <= kMaxK, DSMOE_ERR_ARG, "%s: K (%lld) must be a multiple of 16, at most %d", name, K,
                kMaxK);
  DSMOE_REQUIRE(out_dtype == DSMOE_DTYPE_F32 || out_dtype == DSMOE_DTYPE_BF16, DSMOE_ERR_ARG, "%s: out_dtype %d", name, out_dtype);
  DSMOE_REQUIRE((((uintptr_t)x | (uintptr_t)b) & 15) == 0, DSMOE_ERR_ALIGN, "%s: a and b must be 16-byte aligned", name);
  DSMOE_REQUIRE((((uintptr_t)a_s | (uintptr_t)b_s | (uintptr_t)offsets) & 3) == 0 &&
                    ((uintptr_t)out & (out_dtype == DSMOE_DTYPE_F32 ? 3 : 1)) == 0,
                DSMOE_ERR_ALIGN, "%s: misaligned pointer", name);
  int sms = 0, optin = 0;
  int rc = device_limits(name, &sms, &optin);
  if (rc) return rc;
  PFN_cuTensorMapEncodeTiled_v12000 fn;
  rc = encoder(&fn);
  if (rc) return rc;
  Args a{};
  a.a_s = a_s; a.b_s = b_s; a.offsets = offsets; a.out = out;
  a.M = (int)M; a.N = (int)N; a.K = (int)K; a.E = E;
  a.nkb = (int)((K + 127) / 128);
  a.NTN = (int)((N + TM - 1) / TM);
  a.out_f32 = out_dtype == DSMOE_DTYPE_F32;
  // tokens of a tile: the mean group's, in the next of 16, 32, 64 or 256
  const long long mean = offsets ? (M + E - 1) / E : M;
  a.TT = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : MAXTT;
  const long long groups = offsets ? std::min<long long>(E, M) : 1;
  const long long tiles = a.NTN * (M / a.TT + groups);  // at most
  DSMOE_REQUIRE(tiles < (1LL << 31), DSMOE_ERR_ARG, "%s: too many tiles", name);
  a.S = 1;
  if (a.TT <= SPLIT_TT)
    while (a.S < 8 && a.S * 2 <= a.nkb && tiles * a.S * 2 <= sms) a.S *= 2;
  a.BR = std::min(a.TT, 64);
  rc = encode(fn, &a.tb, b, K, (long long)E * N, TM);
  if (!rc) rc = encode(fn, &a.ta, x, K, M, a.BR);
  if (rc) return rc;
  const int SB = (TM + a.TT) * 128;
  const size_t fixed = 1024 + (a.S > 1 ? 2 * a.TT * TM * 4 : 0) + (2 * MAXRS + 9) * 8 + 48 + 2 * (E + 1) * 4 + 64;
  a.RS = (int)std::min<size_t>(MAXRS, (optin - fixed) / SB);
  const size_t smem = fixed + (size_t)a.RS * SB;
  auto kern = a.S > 1 ? gemm_i8_kernel<true> : gemm_i8_kernel<false>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(std::min<long long>(tiles, std::max(1, sms / a.S)) * a.S));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = a.S;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = a.S > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kern, a);
  return cuda_status(name);
}

}  // namespace gemm_i8
}  // namespace dsmoe

using namespace dsmoe;

extern "C" int dsmoe_int8_gemm(const int8_t* a, const float* a_s, long long M, long long K, const int8_t* b, const float* b_s,
                               long long N, void* out, int out_dtype, void* stream) {
  return gemm_i8::run("int8_gemm", a, a_s, M, K, b, b_s, N, nullptr, 1, out, out_dtype, stream);
}

extern "C" int dsmoe_int8_grouped_gemm(const int8_t* a, const float* a_s, long long M, long long K, const int8_t* b,
                                       const float* b_s, int n_experts, long long N, const int* offsets, void* out, int out_dtype,
                                       void* stream) {
  DSMOE_REQUIRE(offsets, DSMOE_ERR_ARG, "int8_grouped_gemm: null pointer");
  DSMOE_REQUIRE(n_experts > 0 && n_experts <= gemm_i8::kMaxExperts, DSMOE_ERR_ARG, "int8_grouped_gemm: %d experts (1..%d)",
                n_experts, gemm_i8::kMaxExperts);
  return gemm_i8::run("int8_grouped_gemm", a, a_s, M, K, b, b_s, N, offsets, n_experts, out, out_dtype, stream);
}
