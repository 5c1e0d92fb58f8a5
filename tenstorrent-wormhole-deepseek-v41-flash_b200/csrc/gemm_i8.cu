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
//   warp 0      producer: a ring of stages, per 128-K block one load of the weight rows and some of the token rows
//   warp 1      MMA issuer
//   warps 2-9   epilogue (two warps per 32-lane quadrant, splitting the tokens)
// Two kernels. gemm_i8_kernel, for few tokens, is bound by the weights' bytes and by its own latencies: a cluster of up
// to 8 CTAs shares a tile's K blocks and adds the integer partial sums through distributed shared memory (exact, so the
// order does not matter); no workspace, nothing shared between calls. Set-up, first load, barrier and sum are about
// 3.5 us of a call: 8 x 4096 x 5120 takes 7.9 us with weights from memory and 7.3 where three sets of them take turns
// (3.2 are the bytes at copy rate), 64 x 4096 x 5120 9.0, 256 x 4096 x 5120 12.7, 512 x 4096 x 5120 16.2. gemm_i8_pair_kernel, for many, is bound by the tensor pipe and, in a long run, by the power
// limit: CTA pairs on 256 x 512 tiles, as the bytes an SM takes in hold back smaller tiles (4096 x 4096 x 5120: 128 x 256
// by one CTA 98.6 us, 256 x 256 by a pair 69.3, 256 x 480 61.5, 2790 TOP/s; 70 us when it runs for 0.15 s).
// Every wait is bounded; where one expired, the outputs are NaN: those of the whole cluster that shares the sums.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "common.cuh"

namespace dsmoe {
namespace gemm_i8 {

constexpr int NT = 320;       // 10 warps
constexpr int CT = 256;       // epilogue threads
constexpr int TM = 128;       // weight rows of a CTA's tile
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
  int M, N, K, E, nkb, TT, BR, RS, NTN, out_f32;
  unsigned tcols;      // tensor memory columns (one-tile kernel)
  uint64_t land_ns;    // how long the MMA issuer waits for a stage's operands; 0: it gives up before the first
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
__device__ __forceinline__ void ld32(uint32_t taddr, int (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                 "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
                 "=r"(r[30]), "=r"(r[31])
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
__device__ __forceinline__ int4 peer_ld4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int peer_ld(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// mbar_wait whose success also orders the other CTAs' writes before their arrivals.
__device__ __forceinline__ bool cluster_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool cluster_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  if (cluster_test(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!cluster_test(bar, parity)) {
    if (globaltimer_ns() - t0 > limit_ns) return false;
  }
  return true;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Groups of ceil(rows / TT) token tiles each, prefix over experts (every thread of the CTA calls this; the
// caller synchronizes before the tables are read). Offsets that do not rise from 0 to at most M describe no
// groups: no tile runs and the whole output is filled with NaN.
struct Groups {
  int tiles;   // of all groups
  int behind;  // first row of no group
  float fill;  // what the rows from there on hold
};
__device__ __forceinline__ Groups setup_groups(const Args& a, int* first, int* pre, int* wsum) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (!a.offsets) {
    const int mt = (a.M + a.TT - 1) / a.TT;
    if (tid == 0) {
      first[0] = pre[0] = 0;
      first[1] = a.M;
      pre[1] = mt;
    }
    return Groups{mt * a.NTN, a.M, 0.f};
  }
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
  return Groups{carry * a.NTN, bad ? 0 : first[a.E], bad ? __int_as_float(0x7FC00000) : 0.f};
}

// Tile -> expert, channels, tokens. Tiles of one expert are neighbours, the tokens of one weight tile in a
// row, so its bytes are in L2 when they are read again; a group's rows are spread evenly over its tiles, in
// steps of STEP.
template <int STEP>
__device__ __forceinline__ Tile locate_tile(const Args& a, const int* first, const int* pre, int tile, int rows_w) {
  int lo = 0, hi = a.E;  // the expert with pre[e] NTN <= tile < pre[e + 1] NTN
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] * a.NTN <= tile) lo = mid;
    else hi = mid;
  }
  const int mt = pre[lo + 1] - pre[lo], at = tile - pre[lo] * a.NTN;
  const int rows = first[lo + 1] - first[lo];
  const int per = ((rows + mt - 1) / mt + STEP - 1) / STEP * STEP;
  const int m = (at % mt) * per;
  return Tile{lo, at / mt * rows_w, first[lo] + m, max(min(per, rows - m), 0)};
}

// Four neighbouring channels of token t from n (a multiple of 4) on.
__device__ __forceinline__ void store_out4(const Args& a, long long t, int n, const float (&v)[4]) {
  const long long o = t * a.N + n;
  if (a.N % 4 == 0 && ((uintptr_t)a.out & 15) == 0) {
    if (a.out_f32) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + o) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + o) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= a.N) return;
    if (a.out_f32) reinterpret_cast<float*>(a.out)[o + i] = v[i];
    else reinterpret_cast<__nv_bfloat16*>(a.out)[o + i] = __float2bfloat16_rn(v[i]);
  }
}

// Accumulators of this warp's 32 channels and every other 32 tokens from 32 `half` on -> out. sc: the tokens'
// scales in shared memory (padded to 32). The store of one token is 32 neighbouring channels.
template <typename T>
__device__ __forceinline__ void drain(const Args& a, uint32_t tq, int half, int cols, long long m0, int n, float bs,
                                      const float* sc, bool ok) {
  if (!ok) bs = __int_as_float(0x7FC00000);
  const bool live = n < a.N;
  T* p = reinterpret_cast<T*>(a.out) + (m0 + 32 * half) * a.N + n;
  for (int c0 = 32 * half; c0 < cols; c0 += 64, p += 64LL * a.N) {
    int v[32];
    ld32(tq + (uint32_t)c0, v);
    T* o = p;
    if (live && c0 + 32 <= cols) {
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 s = *reinterpret_cast<const float4*>(sc + c0 + i);
        o[0] = (T)((float)v[i] * bs * s.x);
        o += a.N;
        o[0] = (T)((float)v[i + 1] * bs * s.y);
        o += a.N;
        o[0] = (T)((float)v[i + 2] * bs * s.z);
        o += a.N;
        o[0] = (T)((float)v[i + 3] * bs * s.w);
        o += a.N;
      }
    } else if (live) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (c0 + i < cols) o[0] = (T)((float)v[i] * bs * sc[c0 + i]);
        o += a.N;
      }
    }
  }
}
__device__ __forceinline__ void drain(const Args& a, uint32_t tq, int half, int cols, long long m0, int n, float bs,
                                      const float* sc, bool ok) {
  if (a.out_f32) drain<float>(a, tq, half, cols, m0, n, bs, sc, ok);
  else drain<__nv_bfloat16>(a, tq, half, cols, m0, n, bs, sc, ok);
}

// Rows behind the last group, by the epilogue threads of the whole grid.
__device__ __forceinline__ void fill_behind(const Args& a, const Groups& g, int ct) {
  const long long to = (long long)a.M * a.N;
  for (long long i = (long long)g.behind * a.N + (long long)blockIdx.x * CT + ct; i < to; i += (long long)gridDim.x * CT) {
    if (a.out_f32) reinterpret_cast<float*>(a.out)[i] = g.fill;
    else reinterpret_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(g.fill);
  }
}

// A position in a ring of n stages and the parity of its current use, without divisions in the loops.
struct Ring {
  int s = 0;
  uint32_t par = 0;
  __device__ __forceinline__ void next(int n) {
    if (++s == n) {
      s = 0;
      par ^= 1u;
    }
  }
};

// One tile per cluster of S CTAs (S = 1: per CTA): 128 weight rows x up to 256 tokens, each CTA a share of the K
// blocks. The partial sums change hands through the ring's memory once the products have read it.
template <int S>
__global__ void __launch_bounds__(NT) gemm_i8_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t gsm[];
  uint8_t* ring = gsm + ((1024 - (smem_u32(gsm) & 1023)) & 1023);
  const int SB = (TM + a.TT) * 128;  // stage bytes
  int* part = reinterpret_cast<int*>(ring);  // [tokens][TM]
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + a.RS * SB);
  uint64_t* full = bars;             // [MAXRS] stage landed
  uint64_t* empty = full + MAXRS;    // [MAXRS] stage read by its MMAs
  uint64_t* accf = empty + MAXRS;    // [1] accumulator complete
  float* scales = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(accf + 1) + 15) & ~(uintptr_t)15);  // [256]
  uint32_t* tslot = reinterpret_cast<uint32_t*>(scales + 256);
  volatile int* abortf = reinterpret_cast<volatile int*>(tslot + 1);
  int* wsum = reinterpret_cast<int*>(tslot + 2);  // [10]
  int* first = wsum + 10;            // [E + 1] first row of each group
  int* pre = first + a.E + 1;        // [E + 1] tiles before each group

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % S, tile = blockIdx.x / S;
  const int kb0 = rank * a.nkb / S, kb1 = (rank + 1) * a.nkb / S;
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&a.tb) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&a.ta) : "memory");
    for (int s = 0; s < a.RS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(accf, 1);
    *abortf = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(a.tcols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  const Groups g = setup_groups(a, first, pre, wsum);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tslot;
  auto give_up = [&] {
    *abortf = 1;
    __threadfence_block();  // seen by whoever sees an arrival that follows
  };
  auto wait = [&](uint64_t* bar, uint32_t par, uint64_t limit_ns = kWaitNs) -> bool {
    if (*abortf) return false;
    if (!mbar_wait(bar, par, limit_ns)) {
      give_up();
      return false;
    }
    return true;
  };
  // the grid covers the most tiles that M rows in E groups can have
  const bool work = tile < g.tiles;
  const Tile t = work ? locate_tile<16>(a, first, pre, tile, TM) : Tile{0, 0, 0, 0};
  if (warp == 0) {
    if (lane == 0) {
      pdl_launch();
      const int nb = (t.cols + a.BR - 1) / a.BR, yb = t.e * a.N + t.n0;
      const uint32_t bytes = (uint32_t)(TM * 128 + nb * a.BR * 128);
      Ring p;
      int issued = 0;
      for (int kb = kb0; kb < kb1 && work; ++kb, p.next(a.RS), ++issued) {
        if (issued >= a.RS && !wait(&empty[p.s], p.par ^ 1u)) break;
        uint8_t* st = ring + p.s * SB;
        mbar_expect_tx(&full[p.s], bytes);
        tma_2d(st, &a.tb, kb * 128, yb, &full[p.s]);
        for (int b = 0; b < nb; ++b) tma_2d(st + TM * 128 + b * a.BR * 128, &a.ta, kb * 128, t.m0 + b * a.BR, &full[p.s]);
      }
      // every copy issued has landed before the CTA may exit (the last use of each stage)
      for (int i = issued - 1; i >= 0 && i >= issued - a.RS; --i) mbar_wait(&full[i % a.RS], (i / a.RS) & 1, kWaitNs);
    }
  } else if (warp == 1) {
    if (lane == 0 && work) {
      // D s32, A and B s8, both K-major
      const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TM >> 4) << 24) |
                             ((uint32_t)(((t.cols + 15) >> 4) * 2) << 17);
      const uint64_t da0 = desc_sw128(smem_u32(ring)), db0 = desc_sw128(smem_u32(ring + TM * 128));
      Ring p;
      if (!a.land_ns) give_up();
      for (int kb = kb0; kb < kb1; ++kb, p.next(a.RS)) {
        if (!wait(&full[p.s], p.par, a.land_ns)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t o = (uint64_t)(p.s * (SB >> 4));
#pragma unroll
        for (int q = 0; q < 4; ++q) mma_i8(tmem, da0 + o + 2u * q, db0 + o + 2u * q, idesc, (kb > kb0 || q > 0) ? 1u : 0u);
        commit(&empty[p.s]);
      }
      commit(accf);  // also after an abort: no MMA may still run when the tensor memory is freed
      mbar_wait(accf, 0, kWaitNs);
    }
  } else {
    const int ct = tid - 64;
    const int qd = warp & 3, half = (warp - 2) >> 2;
    const int row_l = 32 * qd + lane;
    // S > 1: this CTA finishes channels rank TM / S .. of the tile, a thread four of them for one token at a time
    constexpr int kQuads = TM / S / 4;
    const int r = rank * (TM / S) + ct % kQuads * 4, n = t.n0 + (S > 1 ? r : row_l);
    float bs[S > 1 ? 4 : 1];
    // the scales, while the products are still running
    if (work) {
#pragma unroll
      for (int i = 0; i < (S > 1 ? 4 : 1); ++i) bs[i] = n + i < a.N ? a.b_s[(long long)t.e * a.N + n + i] : 0.f;
      scales[ct] = ct < t.cols ? a.a_s[t.m0 + ct] : 0.f;
    }
    bool ok = work && wait(accf, 0) && !*abortf;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tq = tmem + ((uint32_t)(32 * qd) << 16);
    if (S == 1) {
      named_bar_sync(1, CT);
      if (work) drain(a, tq, half, t.cols, t.m0, n, bs[0], scales, ok);
    } else if (work) {
      for (int c16 = half; 16 * c16 < t.cols; c16 += 2) {
        int v[16];
        ld16(tq + 16u * c16, v);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (16 * c16 + i < t.cols) part[(16 * c16 + i) * TM + row_l] = v[i];
      }
    }
    if (S > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
      if (work && n < a.N) {
        int bad = 0;
#pragma unroll
        for (int z = 0; z < S; ++z) bad |= peer_ld(peer_addr(smem_u32(const_cast<int*>(abortf)), (uint32_t)z));
        for (int c = ct / kQuads; c < t.cols; c += CT / kQuads) {
          const uint32_t at = smem_u32(part + c * TM + r);
          int4 v[S];
          int sum[4] = {0, 0, 0, 0};
          // every CTA begins with its neighbour's partial, so that no CTA's memory is read by all at once
#pragma unroll
          for (int z = 0; z < S; ++z) v[z] = peer_ld4(peer_addr(at, (uint32_t)((rank + 1 + z) % S)));
#pragma unroll
          for (int z = 0; z < S; ++z) {
            sum[0] += v[z].x;
            sum[1] += v[z].y;
            sum[2] += v[z].z;
            sum[3] += v[z].w;
          }
          float o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = bad ? __int_as_float(0x7FC00000) : (float)sum[i] * bs[i] * scales[c];
          store_out4(a, t.m0 + c, n, o);
        }
      }
    }
    fill_behind(a, g, ct);
  }
  __syncwarp();
  if (S > 1 && warp < 2) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  // no CTA leaves while another may still read its partials: those reads are done when their sums are
  if (S > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tcols) : "memory");
  }
}

// ------------------------------------------------------------------ CTA pairs
// Many tokens: two CTAs of a cluster work as a pair (cta_group::2) on a tile of 256 weight rows x up to 512
// tokens. Each CTA loads its own 128 weight rows and half of the token rows, the leader's MMA (M 256, N up to
// 256, one for each half of the tile's tokens) reads both CTAs' shared memory and writes each CTA's 128 rows
// of accumulators into that CTA's tensor memory.
constexpr int PTT = 512;                   // tokens per tile
constexpr int PBR = 64;                    // token rows of one load
// Token rows of one CTA in a stage: half of the tile's, in whole loads; halves of 256 tokens lie 128 rows apart.
__host__ __device__ inline int pair_rows(int TT) { return TT > 256 ? 256 : (TT / 2 + PBR - 1) / PBR * PBR; }

__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Arrives at the barrier of both CTAs when the pair's MMAs so far are complete.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"((unsigned short)3) : "memory");
}
// A load into this CTA's shared memory that reports to a barrier of the pair's leader.
__device__ __forceinline__ void tma_2d_pair(void* dst, const CUtensorMap* tm, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__global__ void __launch_bounds__(NT, 1) gemm_i8_pair_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t gsm[];
  uint8_t* ring = gsm + ((1024 - (smem_u32(gsm) & 1023)) & 1023);
  const int SB = (TM + pair_rows(a.TT)) * 128;  // stage bytes of this CTA: its weight rows, its half of the tokens
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + a.RS * SB);
  uint64_t* full = bars;           // [MAXRS] leader: both CTAs' stage landed
  uint64_t* empty = full + MAXRS;  // [MAXRS] stage read by its MMAs
  uint64_t* accf = empty + MAXRS;  // [2] half of the tensor memory: accumulators complete
  uint64_t* acce = accf + 2;       // [2] leader: accumulators read by both CTAs (8 warps each)
  uint64_t* mdone = acce + 2;      // [1] no MMA in flight
  float* scales = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(mdone + 1) + 15) & ~(uintptr_t)15);  // [2][256]
  uint32_t* tslot = reinterpret_cast<uint32_t*>(scales + 2 * 256);
  volatile int* abortf = reinterpret_cast<volatile int*>(tslot + 1);
  int* wsum = reinterpret_cast<int*>(tslot + 2);  // [10]
  int* first = wsum + 10;          // [E + 1] first row of each group
  int* pre = first + a.E + 1;      // [E + 1] tiles before each group

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x & 1, cid = blockIdx.x >> 1, ncl = gridDim.x >> 1;
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&a.tb) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&a.ta) : "memory");
    for (int s = 0; s < a.RS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&accf[s], 1);
      mbar_init(&acce[s], 16);
    }
    mbar_init(mdone, 1);
    *abortf = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  const Groups g = setup_groups(a, first, pre, wsum);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // both CTAs' barriers and tensor memory exist
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tslot;
  auto give_up = [&] {
    *abortf = 1;
    __threadfence_block();  // seen by whoever sees an arrival that follows
  };
  auto wait = [&](uint64_t* bar, uint32_t par, uint64_t limit_ns = kWaitNs) -> bool {
    if (*abortf) return false;
    if (!cluster_wait(bar, par, limit_ns)) {
      give_up();
      return false;
    }
    return true;
  };
  auto locate = [&](int tile) -> Tile { return locate_tile<32>(a, first, pre, tile, 2 * TM); };
  // A tile's tokens in one or two halves of up to 256, each a multiple of 32 as the MMA wants; half h uses the
  // next half of the tensor memory, so a tile of up to 256 tokens is stored while the next one is computed.
  auto width = [](int cols, int h) -> int {
    const int all = max((cols + 31) & ~31, 32);
    return h == 0 ? min(all, 256) : max(all - 256, 0);
  };

  if (warp == 0) {
    if (lane == 0) {
      pdl_launch();
      int issued = 0;
      Ring p;
      bool ok = true;
      for (int tile = cid; tile < g.tiles && ok; tile += ncl) {
        const Tile t = locate(tile);
        const int w0 = width(t.cols, 0), w1 = width(t.cols, 1);
        const int nb0 = (w0 / 2 + PBR - 1) / PBR, nb1 = (w1 / 2 + PBR - 1) / PBR;
        const int y0 = t.m0 + rank * (w0 / 2), y1 = t.m0 + w0 + rank * (w1 / 2), yb = t.e * a.N + t.n0 + rank * TM;
        const uint32_t bytes = (uint32_t)(2 * (TM * 128 + (nb0 + nb1) * PBR * 128));
        for (int kb = 0; kb < a.nkb; ++kb, p.next(a.RS), ++issued) {
          if (issued >= a.RS && !wait(&empty[p.s], p.par ^ 1u)) {
            ok = false;
            break;
          }
          uint8_t* st = ring + p.s * SB;
          if (rank == 0) mbar_expect_tx(&full[p.s], bytes);
          const uint32_t bar = peer_addr(smem_u32(&full[p.s]), 0);
          tma_2d_pair(st, &a.tb, kb * 128, yb, bar);
          for (int b = 0; b < nb0; ++b) tma_2d_pair(st + TM * 128 + b * PBR * 128, &a.ta, kb * 128, y0 + b * PBR, bar);
          for (int b = 0; b < nb1; ++b) tma_2d_pair(st + TM * 128 + 16384 + b * PBR * 128, &a.ta, kb * 128, y1 + b * PBR, bar);
        }
      }
      // Every copy issued has landed before the pair may exit: both CTAs' report to the leader's barriers, and neither
      // leaves without the other. The follower sees its own only through the MMAs that read them, of which an issuer
      // that gave up runs none: then it waits out the limit, one for all stages.
      const uint64_t t0 = globaltimer_ns();
      for (int i = issued - 1; i >= 0 && i >= issued - a.RS; --i) {
        const uint64_t spent = globaltimer_ns() - t0;
        cluster_wait(rank == 0 ? &full[i % a.RS] : &empty[i % a.RS], (i / a.RS) & 1, spent < kWaitNs ? kWaitNs - spent : 0);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc0 = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(2 * TM >> 4) << 24);
      const uint64_t da0 = desc_sw128(smem_u32(ring)), db0 = desc_sw128(smem_u32(ring + TM * 128));
      int slot = 0;  // halves of the tensor memory used so far
      Ring p;
      bool ok = true;
      if (!a.land_ns) give_up();
      for (int tile = cid; tile < g.tiles && ok; tile += ncl) {
        const Tile t = locate(tile);
        const int w0 = width(t.cols, 0), w1 = width(t.cols, 1), n = w1 ? 2 : 1;
        for (int h = 0; h < n && ok; ++h)
          if (slot + h >= 2) ok = wait(&acce[(slot + h) & 1], (((slot + h) >> 1) - 1) & 1);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t id0 = idesc0 | ((uint32_t)(w0 >> 3) << 17), id1 = idesc0 | ((uint32_t)(w1 >> 3) << 17);
        const uint32_t d0 = tmem + (uint32_t)((slot & 1) * 256), d1 = tmem + (uint32_t)(((slot + 1) & 1) * 256);
        for (int kb = 0; kb < a.nkb; ++kb, p.next(a.RS)) {
          if (!wait(&full[p.s], p.par, a.land_ns)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t o = (uint64_t)(p.s * (SB >> 4));
#pragma unroll
          for (int q = 0; q < 4; ++q) mma_i8_pair(d0, da0 + o + 2u * q, db0 + o + 2u * q, id0, (kb > 0 || q > 0) ? 1u : 0u);
          if (w1) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mma_i8_pair(d1, da0 + o + 2u * q, db0 + o + 1024u + 2u * q, id1, (kb > 0 || q > 0) ? 1u : 0u);
          }
          commit_pair(&empty[p.s]);
        }
        // incomplete sums are not announced: the other CTA does not see this one's flag, its wait for them expires
        if (!ok) break;
        for (int h = 0; h < n; ++h) commit_pair(&accf[(slot + h) & 1]);
        slot += n;
      }
      commit_pair(mdone);  // no MMA may still run when the tensor memory is freed
    }
    if (lane == 0) cluster_wait(mdone, 0, 4 * kWaitNs);
  } else {
    const int ct = tid - 64;
    const int qd = warp & 3, half = (warp - 2) >> 2;
    const int row_l = 32 * qd + lane;
    int slot = 0;
    bool ok = true;
    for (int tile = cid; tile < g.tiles; tile += ncl) {
      const Tile t = locate(tile);
      const int n = t.n0 + rank * TM + row_l;
      const float bs = n < a.N ? a.b_s[(long long)t.e * a.N + n] : 0.f;
      for (int h = 0; h < 2 && width(t.cols, h); ++h, ++slot) {
        const int cols = h ? t.cols - 256 : min(t.cols, 256);
        const long long m0 = t.m0 + 256 * h;
        // the tokens' scales, while the products are still running (the other half of the buffer is being read)
        float* sc = scales + (slot & 1) * 256;
        sc[ct] = ct < cols ? a.a_s[m0 + ct] : 0.f;
        named_bar_sync(1, CT);
        ok = ok && wait(&accf[slot & 1], (slot >> 1) & 1);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t tq = tmem + ((uint32_t)(32 * qd) << 16) + (uint32_t)((slot & 1) * 256);
        drain(a, tq, half, cols, m0, n, bs, sc, ok);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) peer_arrive(&acce[slot & 1], 0);
      }
    }
    fill_behind(a, g, ct);
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other's MMAs or arrivals may reach it
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ------------------------------------------------------------------ host side
std::atomic<void*> g_encode{nullptr};
std::atomic<unsigned long long> g_land_ns{kWaitNs};

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
      cudaFuncSetAttribute(gemm_i8_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, *optin) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_i8_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, *optin) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_i8_kernel<4>, cudaFuncAttributeMaxDynamicSharedMemorySize, *optin) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_i8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, *optin) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_i8_kernel<8>, cudaFuncAttributeMaxDynamicSharedMemorySize, *optin) != cudaSuccess)
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

constexpr size_t kHalfSmem = 113 * 1024;  // of a CTA that shares its SM: with 1 KB each for the system, 228 KB

struct Plan {
  bool pair;
  int TT, S;  // tokens per tile; CTAs of a cluster
};

// Stages of a one-tile CTA's ring: four, which is 64 KB of weights in flight (8 x 4096 x 5120 with four 6.2 us, three
// 6.2, five 6.3, six 7.2: more bytes in flight wait in memory's queues), or what the partials take; no more than K blocks.
int one_tile_stages(int TT, int kb, size_t tables, size_t optin) {
  const size_t SB = (size_t)(TM + TT) * 128;
  const int need = (int)((TT * TM * 4 + SB - 1) / SB);
  return std::min(std::max(std::min(kb, 4), need), (int)((optin - tables) / SB));
}

// Tensor memory columns of a one-tile CTA.
unsigned tile_columns(int TT) { return TT <= 32 ? 32 : TT <= 64 ? 64 : TT <= 128 ? 128 : 256; }

// Groups: their sizes are known to the device alone, so the model takes popularities that fall like rank^-1.1: G
// experts are reached, and tiles of TT tokens number 1.4 for each and one per TT rows. A tile costs its set-up, its K
// blocks (latency, or the bytes an SM takes in) and its store; tiles beyond what the GPU holds at once queue, and so do
// the CTAs of tiles that could have been there; the weights that are reached come from memory. Constants fitted to 227
// cases (1 to 24576 rows, 4 to 384 experts, N 64 to 5120, K 64 to 5120): on the mean 3 % over the best shape of each,
// where a tile of 16 or 32 tokens for up to 64 rows and pairs for more was 17 % (456 rows of 6 experts, N 121, K 2960:
// pairs 13.2 us, 32 x 8 CTAs 7.2; 4285 of 10, N 332, K 112: 11.0, 32 x 1 6.0; 48 of 384, N 512, K 5120: 33, 64 x 2 18.6,
// 16 x 1 21.1). A wider tile must gain 1.5 %, as sizes are not known; pairs on 512 tokens, which are stored before the
// next tile begins, want the mean group to fill half of them (24576 of 64 x 4096 x 5120: 501, 502 with 256; of 384 x 512
// x 5120: 218, 198).
Plan plan_groups(long long M, long long N, int nkb, int E, int sms, size_t tables, size_t optin) {
  const double G = std::min<double>((double)M * E / (M + 1.15 * E - 0.15), std::min<long long>(E, M)), mem = G * N * nkb * 128 / 6.2e6 + M * N * 2 / 6.2e6;
  auto total = [&](double x, double start) {
    return start + std::sqrt(std::sqrt(x * x * x * x + mem * mem * mem * mem));
  };
  Plan best{false, 16, 1};
  double least = 1e30;
  for (int TT = 16; TT <= 256 && (TT == 16 || TT < 2 * M); TT *= 2) {
    const double m = 1.4 * G + (double)M / TT, cols = std::min<double>(TT, M / m), ntn = (N + TM - 1) / TM;
    double t = 1e30;
    int at = 1;
    for (int S = 1; S <= 8 && S <= nkb; S *= 2) {
      const int kb = (nkb + S - 1) / S;
      const size_t ring = tables + (size_t)one_tile_stages(TT, kb, tables, optin) * (TM + TT) * 128;
      const size_t smem = S > 1 ? std::max(ring, kHalfSmem) : ring;
      const int occ = std::min({(int)((optin + 1024) / (smem + 1024)), 3, (int)(512 / tile_columns(TT))});
      const double fit = (S == 8 ? sms * 13 / 15 : S == 4 ? sms * 14 / 15 : sms) * occ, queue = m * ntn * S / fit;
      const double idle = ntn * S * (M / TT + std::min<long long>(E, M)) / fit - std::max(1.0, queue);
      const double block = std::max(0.33, std::max(1.0, occ * std::min(1.0, queue)) * (TM + cols) * 128 / 105e3);
      const double u = total(std::max(1.0, queue) * (3.7 + kb * block + (S > 1 ? 0.033 : 0.0183) * cols) + 4.0 * std::max(0.0, idle), 2.2);
      if (u < t) t = u, at = S;
    }
    if (t < 0.985 * least) least = t, best = Plan{false, TT, at};
  }
  for (int TT = 128; TT <= (M < 256LL * E ? 256 : PTT); TT *= 2) {
    const double m = 1.4 * G + (double)M / TT, cols = std::min<double>(TT, M / m), store = 0.0113 * cols;
    const double blocks = nkb * std::max(0.00105 * cols, (TM * 128 + cols / 2 * 128) / 105e3);
    const double queue = m * ((N + 2 * TM - 1) / (2 * TM)) / (sms / 2);
    const double t = total(std::max(1.0, queue) * (1.45 + (TT > 256 ? blocks + store : std::max(blocks, 1.2 * store))), 6.2);
    if (t < 0.985 * least) least = t, best = Plan{true, TT, 2};
  }
  return best;
}

// The tile shape that should take least time, in us, by a model of what bounds each kernel, its constants fitted to
// measurements on a B200 (M 1..4096, N 72..8192, K 64..8192). An SM takes in at most 105 bytes/ns, and no more than its
// ring's bytes in a round trip (2.2 us for weights that come from memory, 1.4 where other tiles brought them to L2);
// all weights come from memory at 6200 bytes/ns; a K block takes 0.33 us, 0.34 in a pair.
Plan plan(long long M, long long N, int nkb, int E, int sms, size_t tables, size_t optin) {
  if (E) return plan_groups(M, N, nkb, E, sms, tables, optin);
  Plan best{false, 16, 1};
  double least = 1e30;
  const double weights = (double)N * nkb * 128 / 6.2e6;
  const long long ntn = (N + TM - 1) / TM;
  const long long mt0 = (M + 255) / 256, mt1 = std::min<long long>((M + 15) / 16, mt0 + 15);
  for (long long mt = mt0; mt <= mt1; ++mt) {
    const int TT = (int)(((M + mt - 1) / mt + 15) / 16 * 16);
    for (int S = 1; S <= 8 && S <= nkb; S *= 2) {
      const int kb = (nkb + S - 1) / S, rs = one_tile_stages(TT, kb, tables, optin);
      const double SB = (TM + TT) * 128.0;
      const int occ = tables + rs * SB <= kHalfSmem ? 2 : 1;
      const int fit = S == 8 ? sms * 13 / 15 : S == 4 ? sms * 14 / 15 : sms;  // SMs that clusters of S can use
      const long long n = (M + TT - 1) / TT * ntn * S, rounds = (n + fit - 1) / fit, waves = (rounds + occ - 1) / occ;
      const double load = std::max(std::max(kb * SB * std::min<long long>(occ, rounds) / 105e3, ((double)kb / rs - 1) * (1.4 + 0.8 / mt)), 0.33 * kb);
      // joining partials costs a cluster barrier and each CTA's share of the reads
      const double t = 0.8 + std::max(waves * load, weights) + waves * (2.2 + (S > 1 ? 0.4 + 0.0125 * TT + 0.1 * S : 0.008 * TT));
      if (t < least) least = t, best = Plan{false, TT, S};
    }
  }
  if (M > 64) {
    const long long ntp = (N + 2 * TM - 1) / (2 * TM);
    const long long mp0 = (M + PTT - 1) / PTT, mp1 = std::min<long long>((M + 63) / 64, mp0 + 15);
    for (long long mt = mp0; mt <= mp1; ++mt) {
      const int TT = (int)(((M + mt - 1) / mt + 31) / 32 * 32);
      const double SB = (TM + pair_rows(TT)) * 128.0;
      const long long rounds = ((M + TT - 1) / TT * ntp + sms / 2 - 1) / (sms / 2);
      // a K block: its MMAs, or its bytes; a tile of more than 256 tokens is stored before the next one begins
      const double block = std::max(0.34, std::max(TT * 0.00105, SB / 105e3)), store = 0.012 * TT;
      const double tile = TT > 256 ? nkb * block + store : std::max(nkb * block, 1.2 * store);
      const double t = 5.0 + std::max(rounds * tile, weights) + (TT > 256 ? 0.0 : store);
      if (t < least) least = t, best = Plan{true, TT, 2};
    }
  }
  return best;
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
  DSMOE_REQUIRE(!overlap({{out, M * N * (out_dtype == DSMOE_DTYPE_F32 ? 4 : 2)}},
                         {{x, M * K}, {a_s, M * 4}, {b, N * E * K}, {b_s, N * E * 4}, {offsets, (E + 1) * 4}}),
                DSMOE_ERR_ARG, "%s: out overlaps an input", name);
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
  a.land_ns = g_land_ns.load(std::memory_order_relaxed);
  const size_t tables = 1024 + (2 * MAXRS + 9) * 8 + 16 + 2 * 256 * 4 + 48 + 2 * (E + 1) * 4 + 64;
  const Plan p = plan(M, N, a.nkb, offsets ? E : 0, sms, tables, optin);
  a.TT = p.TT;
  a.BR = p.pair ? PBR : offsets ? std::min(p.TT, 64) : p.TT;
  // a one-tile stage holds TT token rows, which its loads fill exactly: a last one in part would write into the next stage
  DSMOE_REQUIRE(p.pair || a.TT % a.BR == 0, DSMOE_ERR_UNSUPPORTED, "%s: tile of %d tokens in loads of %d", name, a.TT, a.BR);
  a.NTN = (int)((N + (p.pair ? 2 : 1) * TM - 1) / ((p.pair ? 2 : 1) * TM));
  const long long tiles = a.NTN * (M / a.TT + (offsets ? std::min<long long>(E, M) : M % a.TT != 0));  // at most
  DSMOE_REQUIRE(tiles * p.S < (1LL << 31), DSMOE_ERR_ARG, "%s: too many tiles", name);
  rc = encode(fn, &a.tb, b, K, (long long)E * N, TM);
  if (!rc) rc = encode(fn, &a.ta, x, K, M, a.BR);
  if (rc) return rc;
  const int SB = (TM + (p.pair ? pair_rows(a.TT) : a.TT)) * 128;
  if (p.pair) {
    a.RS = std::min(MAXRS, (int)((optin - tables) / SB));
  } else {
    a.RS = one_tile_stages(a.TT, (a.nkb + p.S - 1) / p.S, tables, optin);
    a.tcols = tile_columns(a.TT);
  }
  // Shared memory also decides who shares an SM, and with it its tensor memory, whose allocation waits without a limit
  // while CTAs of a cluster wait for one another. A pair (all 512 columns) takes the whole SM; a CTA of a cluster half of
  // it: two such CTAs hold at most 512 columns, and no kernel that takes more than half an SM, as those with pairs of
  // their own do, can stand between the CTAs of one cluster.
  size_t smem = tables + (size_t)a.RS * SB;
  if (p.pair) smem = optin;
  else if (p.S > 1) smem = std::max(smem, kHalfSmem);
  auto kern = p.pair     ? gemm_i8_pair_kernel
              : p.S == 1 ? gemm_i8_kernel<1>
              : p.S == 2 ? gemm_i8_kernel<2>
              : p.S == 4 ? gemm_i8_kernel<4>
                         : gemm_i8_kernel<8>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.pair ? std::min<long long>(tiles, sms / 2) : tiles) * p.S));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = p.S;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.S > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kern, a);
  return cuda_status(name);
}

}  // namespace gemm_i8
}  // namespace dsmoe

using namespace dsmoe;

extern "C" int dsmoe_int8_operand_wait(long long ns) {
  DSMOE_REQUIRE(ns >= 0 && ns <= (long long)gemm_i8::kWaitNs, DSMOE_ERR_ARG, "int8_operand_wait: %lld ns (0..%lld)", ns,
                (long long)gemm_i8::kWaitNs);
  gemm_i8::g_land_ns.store((unsigned long long)ns);
  return DSMOE_OK;
}

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
