// Linear layer with 4-bit weights (format: q4.cuh): y[t, n] = ts sum_k x[t, k] w[n, k] (+ residual[t, n]),
// fp32 accumulation, one rounding to bf16.  Three kernels, by the number of tokens and tiles:
//
// q4_linear_few: the weight tile is the A operand of mma.m16n8k16 (16 output features), the tokens are N = 8, so one
// token costs no more tensor work than eight.  What bounds it is the stream of weight bytes; codes go from global
// memory to registers in 16-byte loads and are dequantised there (exact).
//
// q4_linear_many: tokens are the M = 128 rows of tcgen05.mma, 64 output features its N; x comes by TMA, and four warps
// dequantise the stage's 64 columns of weights into shared memory in the operand's swizzled layout, their codes fetched
// four stages ahead.  With few tiles K is split over a cluster, whose CTAs add up over distributed shared memory.
//
// q4_linear_wide: with enough tiles the products bound it, and shared memory their operands: with x and 256 outputs'
// weights there an SM moves 96 KB for 512 clocks of products (28 us for 4096 x 2048 -> 1024).  So the weights are the
// A operand in tensor memory, 128 outputs, written there by the dequantising warps, and 256 tokens of x the B operand:
// 64 KB per 512 clocks, half of the dequantisation, 550 clocks a stage (15.8 us; 1090 TFLOP/s).  What is left is
// mostly the start and the output of the one tile a CTA has (about 5.7 us).
//
// None has a workspace or a second launch.
#include <cudaTypedefs.h>

#include "../../include/hla_s6.h"
#include "hla_s6_internal.h"
#include "q4.cuh"
#include "tc.cuh"

namespace hla {

struct Q4LinearParams {
  const __nv_bfloat16* x;  // [T, K]
  int64_t x_st;
  const uint8_t* w;
  int T, N, K;
  float ts;
  const __nv_bfloat16* res;  // [T, N] or NULL
  int64_t res_st;
  __nv_bfloat16* out;
  int64_t o_st;
  int vec;    // out (and residual) rows are 16-byte aligned
  int split;  // CTAs of a cluster that share a tile's K (many tokens)
  int* err;   // error word or NULL
  uint64_t wait_ns;
};

// ------------------------------------------------------------------ few tokens
constexpr int kQ4LinWarps = 8;
constexpr int kQ4FewTokens = 64;

// A CTA: RT tiles of 16 output features x 8 NT tokens, K split over its 8 warps, which meet in shared memory.
template <int NT, int RT>
__global__ void __launch_bounds__(kQ4LinWarps * 32, NT == 1 ? 4 : 1) q4_linear_few_kernel(const Q4LinearParams p) {
  __shared__ float red[kQ4LinWarps][RT][NT][4][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int kt_n = (p.K + 127) / 128, t0 = blockIdx.y * (8 * NT), n_tiles = (p.N + 15) / 16;
  float acc[RT][NT][4] = {};
  const int64_t tile_row = static_cast<int64_t>(kt_n) * kQ4WeightTile;
  const uint8_t* tile = p.w + blockIdx.x * RT * tile_row + warp * kQ4WeightTile;
  const bool live0 = t0 + g < p.T;
#pragma unroll 1
  for (int kt = warp; kt < kt_n; kt += kQ4LinWarps, tile += kQ4LinWarps * kQ4WeightTile) {
    uint4 lo[RT], hi[RT];
    uint32_t sb[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const bool ok = blockIdx.x * RT + i < n_tiles;  // tiles past the last read the first one's bytes, unused
      const uint8_t* at = tile + (ok ? i * tile_row : 0);
      lo[i] = __ldg(reinterpret_cast<const uint4*>(at) + lane);
      hi[i] = __ldg(reinterpret_cast<const uint4*>(at + 512) + lane);
      sb[i] = __ldg(reinterpret_cast<const uint16_t*>(at + 1024) + lane);
    }
    uint4 xb[NT][4];
    const int col = kt * 128 + 32 * c;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const bool in = (NT == 1 ? live0 : t0 + 8 * j + g < p.T) && col < p.K;
      const uint4* src = reinterpret_cast<const uint4*>(p.x + static_cast<int64_t>(t0 + 8 * j + g) * p.x_st + col);
#pragma unroll
      for (int i = 0; i < 4; ++i) xb[j][i] = in ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint32_t s2 = e4m3x2_to_bf2(sb[r]);
      const Q4Scale s0(__byte_perm(s2, 0, 0x1010)), s1(__byte_perm(s2, 0, 0x3232));
      const uint32_t wl[4] = {lo[r].x, lo[r].y, lo[r].z, lo[r].w}, wh[4] = {hi[r].x, hi[r].y, hi[r].z, hi[r].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a0[4] = {q4_pair<0>(wl[i], s0), q4_pair<0>(wh[i], s1), q4_pair<1>(wl[i], s0),
                                q4_pair<1>(wh[i], s1)};
        const uint32_t a1[4] = {q4_pair<2>(wl[i], s0), q4_pair<2>(wh[i], s1), q4_pair<3>(wl[i], s0),
                                q4_pair<3>(wh[i], s1)};
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_bf16_16816(acc[r][j], a0, xb[j][i].x, xb[j][i].y);
          mma_bf16_16816(acc[r][j], a1, xb[j][i].z, xb[j][i].w);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][r][j][e][lane] = acc[r][j][e];
  __syncthreads();
  // element (row n, token t) of a tile: lane (n % 8) * 4 + (t % 8) / 2, register 2 (n / 8) + t % 2
  for (int i = threadIdx.x; i < RT * NT * 128; i += blockDim.x) {
    const int nl = i & 15, r = (i >> 4) % RT, tl = i / (16 * RT), t = t0 + tl, n = (blockIdx.x * RT + r) * 16 + nl;
    if (t >= p.T || n >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kQ4LinWarps; ++w)
      v += red[w][r][tl >> 3][2 * (nl >> 3) + (tl & 1)][(nl & 7) * 4 + ((tl & 7) >> 1)];
    v *= p.ts;
    if (p.res) v += __bfloat162float(p.res[static_cast<int64_t>(t) * p.res_st + n]);
    p.out[static_cast<int64_t>(t) * p.o_st + n] = __float2bfloat16_rn(v);
  }
}

template <int NT, int RT>
static int launch_few(const Q4LinearParams& p, cudaStream_t s) {
  q4_linear_few_kernel<NT, RT><<<dim3((p.N + 16 * RT - 1) / (16 * RT), (p.T + 8 * NT - 1) / (8 * NT)), kQ4LinWarps * 32, 0,
                                 s>>>(p);
  return cuda_status(cudaGetLastError(), "q4_linear_few_kernel launch");
}

// ------------------------------------------------------------------ many tokens
struct Q4Many {
  static constexpr int BN = 64;           // outputs of a tile
  static constexpr int A_BYTES = 128 * 64 * 2, B_BYTES = BN * 64 * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int SMEM = 1024 + STAGES * STAGE + 256;
  static constexpr int DQ = BN / 16;      // dequantising warps, one 16-row tile of the stage each
  static constexpr int RED = BN + 4;      // floats per row of the partial tile that a cluster's CTAs exchange
  static_assert(128 * RED * 4 <= STAGES * STAGE, "partial tile");
  static constexpr uint32_t COLS = BN;
};

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_rows(void* dst, const void* tmap, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::
          "r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}

// out[t, n .. n + 15] from the fp32 sums (columns past N left out); `pre`: the residual, where it has been loaded.
__device__ __forceinline__ void store16(const Q4LinearParams& p, int t, int n, float (&v)[16], const uint4* pre = nullptr) {
  __nv_bfloat16* dst = p.out + static_cast<int64_t>(t) * p.o_st + n;
  const __nv_bfloat16* rs = p.res ? p.res + static_cast<int64_t>(t) * p.res_st + n : nullptr;
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] *= p.ts;
  if (p.vec && n + 16 <= p.N) {
    if (rs) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint4 u = pre ? pre[q] : reinterpret_cast<const uint4*>(rs)[q];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[8 * q + 2 * e] += __uint_as_float(w[e] << 16);
          v[8 * q + 2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
      reinterpret_cast<uint4*>(dst)[q] =
          make_uint4(pack_bf16(v[8 * q], v[8 * q + 1]), pack_bf16(v[8 * q + 2], v[8 * q + 3]),
                     pack_bf16(v[8 * q + 4], v[8 * q + 5]), pack_bf16(v[8 * q + 6], v[8 * q + 7]));
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (n + e < p.N) dst[e] = __float2bfloat16_rn(v[e] + (rs ? __bfloat162float(rs[e]) : 0.f));
  }
}

// Called by whole warps (the forms that are not aligned take 0.5 us longer).
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
// 16 bytes of another CTA's shared memory, at the address `p` has in this one.
__device__ __forceinline__ float4 ld_cluster(const void* p, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n"
      ".reg .b32 a;\n"
      "mapa.shared::cluster.u32 a, %4, %5;\n"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n"
      "}\n"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(smem_u32(p)), "r"(rank)
      : "memory");
  return v;
}

// warps 0 .. DQ-1 dequantise, then write the output; warp DQ: TMA of x; warp DQ + 1: products.
__global__ void __launch_bounds__((Q4Many::DQ + 2) * 32) q4_linear_many_kernel(
    const __grid_constant__ CUtensorMap tmap_x, const Q4LinearParams p) {
  using C = Q4Many;
  constexpr int DQ = C::DQ, BN = C::BN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // (an offset, not a rounded pointer: the compiler then knows that these are shared-memory addresses)
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE);  // x copied and weights written
  uint64_t* empty = full + C::STAGES;
  uint64_t* done = empty + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.y * 128, n0 = blockIdx.x * BN, kt_n = (p.K + 127) / 128;
  // this CTA's blocks of 64 columns of K
  const int nk_all = (p.K + 63) / 64;
  const int kfirst = static_cast<int>(stream_start(blockIdx.z, nk_all, p.split));
  const int NK = static_cast<int>(stream_start(blockIdx.z + 1, nk_all, p.split)) - kfirst;

  if (warp == DQ) tc::alloc(tmem_slot, C::COLS);
  if (threadIdx.x == (DQ + 1) * 32) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1 + DQ);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const tc::Waits wait{abort_flag, p.err, p.wait_ns};

  if (warp < DQ) {
    // lane: row 8 half + g of a 16-row tile, columns 32 c .. of the stage's 64
    const int half = lane >> 4, g = (lane >> 1) & 7, c = lane & 1, row = 8 * half + g;
    const int64_t tile_row = static_cast<int64_t>(kt_n) * kQ4WeightTile;
    const bool there = n0 / 16 + warp < (p.N + 15) / 16;
    // a block of 64 columns is half a tile; pairs of blocks advance by a tile
    const uint8_t* src = p.w + (n0 / 16 + warp) * tile_row + static_cast<int64_t>(kfirst >> 1) * kQ4WeightTile;
    const uint32_t code_at = half * 512 + (g * 4 + c) * 16, scale_at = 1024 + (g * 4 + c) * 2 + half;
    constexpr int AHEAD = 4;  // blocks whose codes are in flight
    uint4 code[AHEAD];
    uint32_t sb[AHEAD];
    int kf = kfirst;                     // next block to fetch
    const int kend = there ? kfirst + NK : 0;
    auto fetch = [&](uint4& cd, uint32_t& s) {
      cd = make_uint4(0u, 0u, 0u, 0u);
      s = 0u;
      if (kf < kend) {
        const uint8_t* at = src + (kf & 1) * 32;
        cd = __ldg(reinterpret_cast<const uint4*>(at + code_at));
        s = __ldg(src + (kf & 1) * 4 + scale_at);
      }
      if (kf & 1) src += kQ4WeightTile;
      ++kf;
    };
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) fetch(code[a], sb[a]);
    // the four 16-byte chunks of this thread's row in stage 0 (SWIZZLE_128B)
    uint8_t* const b0 = smem + C::A_BYTES + (warp * 16 + row) * 128;
    uint32_t off[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) off[j] = ((4 * c + j) ^ g) << 4;
    static_assert(AHEAD == C::STAGES, "one fetched block per stage");
    uint32_t phase = 1;
    for (int kb0 = 0; kb0 < NK; kb0 += AHEAD, phase ^= 1) {
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        if (kb0 + a >= NK) break;
        wait(&empty[a], phase, kErrWaitEmpty);
        const Q4Scale sc(e4m3x2_to_bf2(sb[a] | (sb[a] << 8)));
        const uint32_t w[4] = {code[a].x, code[a].y, code[a].z, code[a].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(b0 + a * C::STAGE + off[j]) =
              make_uint4(q4_pair<0>(w[j], sc), q4_pair<1>(w[j], sc), q4_pair<2>(w[j], sc), q4_pair<3>(w[j], sc));
        fetch(code[a], sb[a]);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[a]);
      }
    }
    // ---- output: this warp's 32 rows (tokens), its share of the columns
    wait(done, 0, kErrWaitFull);
    __syncwarp();
    tc::fence_after();
    const int t = m0 + (warp & 3) * 32 + lane;
    constexpr int SHARE = BN * 4 / DQ;  // columns per warp
    const int cw = (warp >> 2) * SHARE;
    const uint32_t acc = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + cw;
#pragma unroll 1
    for (int c0 = 0; c0 < SHARE; c0 += 16) {
      uint32_t r[16];
      tc::ld16(acc + c0, r);
      tc::wait_ld();
      if (p.split > 1) {  // this CTA's part of the sum, for the cluster
        float4* dst = reinterpret_cast<float4*>(smem + ((warp & 3) * 32 + lane) * C::RED * 4 + (cw + c0) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          dst[e] = make_float4(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1]), __uint_as_float(r[4 * e + 2]),
                               __uint_as_float(r[4 * e + 3]));
        continue;
      }
      const int n = n0 + cw + c0;
      if (t >= p.T || n >= p.N) continue;
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(r[e]);
      store16(p, t, n, v);
    }
  } else if (warp == DQ) {
    if (lane == 0) {
      prefetch_tmap(&tmap_x);
      for (int kb = 0; kb < NK; ++kb) {
        const int s = kb % C::STAGES;
        if (kb >= C::STAGES) wait(&empty[s], ((kb / C::STAGES) - 1) & 1, kErrWaitEmpty);
        mbar_arrive_expect_tx(&full[s], C::A_BYTES);
        tma_load_rows(smem + s * C::STAGE, &tmap_x, &full[s], (kfirst + kb) * 64, m0);  // rows and columns past x are zeros
      }
      // the last copies land before the CTA ends, also when a wait has given up
      for (int kb = max(0, NK - C::STAGES); kb < NK; ++kb) mbar_wait(&full[kb % C::STAGES], (kb / C::STAGES) & 1, p.wait_ns);
    }
  } else if (tc::elect()) {
    for (int kb = 0; kb < NK; ++kb) {
      const int s = kb % C::STAGES;
      wait(&full[s], (kb / C::STAGES) & 1, kErrWaitFull);
      tc::fence_after();
      const uint64_t da = tc::desc_sw128(smem_u32(smem + s * C::STAGE));
      const uint64_t db = tc::desc_sw128(smem_u32(smem + s * C::STAGE + C::A_BYTES));
#pragma unroll
      for (int k = 0; k < 4; ++k) mma_ss(tmem, da + 2 * k, db + 2 * k, tc::idesc(1, 128, BN), k ? 1u : kb != 0);
      tc::commit(&empty[s]);
    }
    tc::commit(done);
    mbar_wait(done, 0, p.wait_ns);
  }
  if (warp >= DQ) __syncwarp();  // one lane's branch ends
  if (p.split > 1) {
    // the cluster's CTAs hold a part of the sum each; CTA k adds up and writes every split-th row from k
    cluster_sync();
    const int rows = min(128, p.T - m0);
    for (int u = threadIdx.x; u < ((rows - static_cast<int>(blockIdx.z) + p.split - 1) / p.split) * (BN / 4); u += blockDim.x) {
      const int r = u / (BN / 4) * p.split + blockIdx.z, c0 = u % (BN / 4) * 4, t = m0 + r, n = n0 + c0;
      if (n >= p.N) continue;
      float4 part[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) part[k] = k < p.split ? ld_cluster(smem + (r * C::RED + c0) * 4, k) : make_float4(0.f, 0.f, 0.f, 0.f);
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // in order: the sum does not depend on which CTA adds
        v[0] += part[k].x; v[1] += part[k].y; v[2] += part[k].z; v[3] += part[k].w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (n + e >= p.N) break;
        const float rs = p.res ? __bfloat162float(p.res[static_cast<int64_t>(t) * p.res_st + n + e]) : 0.f;
        p.out[static_cast<int64_t>(t) * p.o_st + n + e] = __float2bfloat16_rn(v[e] * p.ts + rs);
      }
    }
    __syncwarp();
    cluster_sync();  // no CTA's memory goes before the others have read it
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == DQ) tc::dealloc(tmem, C::COLS);
}

// ------------------------------------------------------------------ very many tokens
constexpr int kWideTokens = 256, kWideOut = 128;          // a CTA's tile of the output
constexpr int kWideStages = 6, kWideStage = kWideTokens * 128;  // 64 columns of x, bf16
constexpr int kWideSmem = 1024 + kWideStages * kWideStage + 256;
static_assert(kWideTokens * kWideOut * 4 <= kWideStages * kWideStage, "the output tile replaces the stages");
static_assert(kWideTokens + kWideStages * 32 <= 512, "tensor memory");

// warps 0-7 dequantise (groups of four take turns), then write the output; warp 8: TMA of x; warp 9: products.
__global__ void __launch_bounds__(320, 1) q4_linear_wide_kernel(const __grid_constant__ CUtensorMap tmap_x,
                                                                const Q4LinearParams p) {
  constexpr int S = kWideStages, AHEAD = S / 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  uint64_t* x_full = reinterpret_cast<uint64_t*>(smem + S * kWideStage);  // x of a stage copied
  uint64_t* a_full = x_full + S;                                          // its weights in tensor memory
  uint64_t* empty = a_full + S;                                           // its products done
  uint64_t* done = empty + S;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * kWideOut, m0 = blockIdx.y * kWideTokens, NK = (p.K + 63) / 64;
  if (warp == 8) tc::alloc(tmem_slot, 512);
  if (threadIdx.x == 9 * 32) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&x_full[s], 1);
      mbar_init(&a_full[s], 4);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;  // columns: the output's 256 tokens, then a stage's 64 weight columns each
  const tc::Waits wait{abort_flag, p.err, p.wait_ns};

  if (warp < 8) {
    const int grp = warp >> 2, w = warp & 3, row = 32 * w + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(w * 32) << 16);
    // group 0 takes the first halves of the weight tiles (64 of 128 columns), group 1 the second
    const int own = (NK - grp + 1) / 2, h = (row >> 3) & 1, g = row & 7;
    const bool there = n0 / 16 + row / 16 < (p.N + 15) / 16;
    const uint8_t* src = p.w + (n0 / 16 + row / 16) * (static_cast<int64_t>((p.K + 127) / 128) * kQ4WeightTile);
    const uint8_t *codes = src + h * 512 + g * 64 + grp * 32, *scales = src + 1024 + g * 8 + grp * 4 + h;
    uint4 code[AHEAD][2];
    uint32_t sb[AHEAD][2];
    int next = 0;
    auto fetch = [&](uint4 (&cd)[2], uint32_t (&s)[2]) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        cd[q] = make_uint4(0u, 0u, 0u, 0u);
        s[q] = 0u;
        if (there && next < own) {
          cd[q] = __ldg(reinterpret_cast<const uint4*>(codes + 16 * q));
          s[q] = __ldg(scales + 2 * q);
        }
      }
      codes += kQ4WeightTile;
      scales += kQ4WeightTile;
      ++next;
    };
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) fetch(code[a], sb[a]);
    uint32_t phase = 1;
    for (int i0 = 0; i0 < own; i0 += AHEAD, phase ^= 1) {
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        if (i0 + a >= own) break;
        const int s = 2 * a + grp;
        wait(&empty[s], phase, kErrWaitEmpty);
        __syncwarp();
        tc::fence_after();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const Q4Scale sc(e4m3x2_to_bf2(sb[a][q] | (sb[a][q] << 8)));
          const uint32_t x[4] = {code[a][q].x, code[a][q].y, code[a][q].z, code[a][q].w};
          uint32_t v[16];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[4 * j] = q4_pair<0>(x[j], sc);
            v[4 * j + 1] = q4_pair<1>(x[j], sc);
            v[4 * j + 2] = q4_pair<2>(x[j], sc);
            v[4 * j + 3] = q4_pair<3>(x[j], sc);
          }
          tc::st16(lane_base + kWideTokens + s * 32 + q * 16, v);
        }
        fetch(code[a], sb[a]);
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&a_full[s]);
      }
    }
    // ---- output: through shared memory, where a token's 128 columns lie side by side (16-byte chunks swizzled)
    const int tid = threadIdx.x & 127, seg = tid & 7;  // 16 columns of every 16th token
    uint4 pre[8][2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = m0 + grp * 128 + (tid >> 3) + 16 * i, n = n0 + 16 * seg;
      pre[i][0] = pre[i][1] = make_uint4(0u, 0u, 0u, 0u);
      if (p.res && p.vec && t < p.T && n + 16 <= p.N) {
        const uint4* r = reinterpret_cast<const uint4*>(p.res + static_cast<int64_t>(t) * p.res_st + n);
        pre[i][0] = r[0];
        pre[i][1] = r[1];
      }
    }
    wait(done, 0, kErrWaitFull);
    __syncwarp();
    tc::fence_after();
    uint8_t* tile = smem + grp * 128 * 512;
    {
      const uint32_t at = (8 * w + ((lane >> 2) ^ w)) * 16 + (lane & 3) * 4;
#pragma unroll 2
      for (int c0 = 0; c0 < 128; c0 += 16) {
        uint32_t r[16];
        tc::ld16(lane_base + grp * 128 + c0, r);
        tc::wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) *reinterpret_cast<uint32_t*>(tile + (c0 + e) * 512 + at) = r[e];
      }
    }
    named_bar_sync(1 + grp, 128);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int tl = (tid >> 3) + 16 * i, t = m0 + grp * 128 + tl, n = n0 + 16 * seg;
      float v[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int q = 4 * seg + e;
        const float4 f = *reinterpret_cast<const float4*>(tile + tl * 512 + ((q & ~7) | ((q & 7) ^ (q >> 3))) * 16);
        v[4 * e] = f.x; v[4 * e + 1] = f.y; v[4 * e + 2] = f.z; v[4 * e + 3] = f.w;
      }
      if (t < p.T && n < p.N) store16(p, t, n, v, pre[i]);
    }
  } else if (warp == 8) {
    if (lane == 0) {
      prefetch_tmap(&tmap_x);
      for (int kb = 0; kb < NK; ++kb) {
        const int s = kb % S;
        if (kb >= S) wait(&empty[s], ((kb / S) - 1) & 1, kErrWaitEmpty);
        mbar_arrive_expect_tx(&x_full[s], kWideStage);  // rows and columns past x are zeros
        tma_load_rows(smem + s * kWideStage, &tmap_x, &x_full[s], kb * 64, m0);
        tma_load_rows(smem + s * kWideStage + kWideStage / 2, &tmap_x, &x_full[s], kb * 64, m0 + 128);
      }
      // the last copies land before the CTA ends, also when a wait has given up
      for (int kb = max(0, NK - S); kb < NK; ++kb) mbar_wait(&x_full[kb % S], (kb / S) & 1, p.wait_ns);
    }
  } else if (tc::elect()) {
    uint32_t phase = 0;
    for (int kb0 = 0; kb0 < NK; kb0 += S, phase ^= 1) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (kb0 + s >= NK) break;
        wait(&a_full[s], phase, kErrWaitFull);
        wait(&x_full[s], phase, kErrWaitFull);
        tc::fence_after();
        const uint64_t xd = tc::desc_sw128(smem_u32(smem + s * kWideStage));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc::mma_ts(tmem, tmem + kWideTokens + s * 32 + k * 8, xd + 2 * k, tc::idesc(1, 128, kWideTokens), kb0 + s + k > 0);
        tc::commit(&empty[s]);
      }
    }
    tc::commit(done);
    mbar_wait(done, 0, p.wait_ns);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 8) tc::dealloc(tmem, 512);
}

static int launch_wide(const Q4LinearParams& p, cudaStream_t s) {
  CUtensorMap tx;
  int rc = rows_tmap(&tx, p.x, p.T, p.K, p.x_st);
  if (rc) return rc;
  static unsigned attr_mask = 0;
  ensure_smem_limit(q4_linear_wide_kernel, kWideSmem, attr_mask);
  const dim3 grid((p.N + kWideOut - 1) / kWideOut, (p.T + kWideTokens - 1) / kWideTokens);
  q4_linear_wide_kernel<<<grid, 320, kWideSmem, s>>>(tx, p);
  return cuda_status(cudaGetLastError(), "q4_linear_wide_kernel launch");
}

static int launch_many(const Q4LinearParams& p, cudaStream_t s) {
  using C = Q4Many;
  CUtensorMap tx;
  int rc = rows_tmap(&tx, p.x, p.T, p.K, p.x_st);
  if (rc) return rc;
  static unsigned attr_mask = 0;
  ensure_smem_limit(q4_linear_many_kernel, C::SMEM, attr_mask);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + C::BN - 1) / C::BN, (p.T + 127) / 128, p.split);
  cfg.blockDim = dim3((C::DQ + 2) * 32);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = p.split;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, q4_linear_many_kernel, tx, p), "q4_linear_many_kernel launch");
}

}  // namespace hla

using namespace hla;

extern "C" {

int hla_s6_linear_q4_checked(const void* x, int64_t x_stride_t, const void* packed, int32_t num_tokens,
                             int32_t out_features, int32_t in_features, float scale, const void* residual,
                             int64_t residual_stride_t, void* out, int64_t out_stride_t, int* error_flag, void* stream) {
  if (num_tokens < 0 || out_features < 1 || out_features > 16 * 65535 || in_features < 32 || in_features % 32 ||
      (x_stride_t % 8) || (reinterpret_cast<uintptr_t>(x) % 16) || (reinterpret_cast<uintptr_t>(packed) % 16)) {
    set_error("linear (4 bit) needs in_features %% 32 == 0, 1..1048560 out_features and 16-byte aligned x rows and "
              "weight");
    return kStatusInvalid;
  }
  if (num_tokens > 65535 * kWideTokens) {
    set_error("linear (4 bit): at most %d tokens (got %d)", 65535 * kWideTokens, num_tokens);
    return kStatusInvalid;
  }
  if (out_stride_t < out_features && num_tokens > 1) {
    set_error("linear (4 bit): output rows overlap (stride %lld)", static_cast<long long>(out_stride_t));
    return kStatusInvalid;
  }
  if (!(scale > 0.f && scale <= 3.0e38f)) {
    set_error("linear (4 bit): the weight's tensor scale must be positive and finite");
    return kStatusInvalid;
  }
  if (num_tokens == 0) return kStatusOk;
  Q4LinearParams p;
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.x_st = x_stride_t;
  p.w = static_cast<const uint8_t*>(packed);
  p.T = num_tokens;
  p.N = out_features;
  p.K = in_features;
  p.ts = scale;
  p.res = static_cast<const __nv_bfloat16*>(residual);
  p.res_st = residual_stride_t;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_st = out_stride_t;
  auto a16 = [](const void* q, int64_t st) { return (reinterpret_cast<uintptr_t>(q) % 16) == 0 && st % 8 == 0; };
  p.vec = a16(out, out_stride_t) && (!residual || a16(residual, residual_stride_t));
  p.err = error_flag;
  p.wait_ns = std::max(wait_limit_ns(), tc::kLeastWaitNs);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Few tokens: tiles of 16 outputs x 8 tokens.  One token tile: two row tiles a CTA once there are enough CTAs (1 x 2048
  // -> 12288 5.0 us instead of 5.3; -> 6144 4.7 instead of 4.3).
  if (num_tokens <= 8) return out_features >= 8192 ? launch_few<1, 2>(p, s) : launch_few<1, 1>(p, s);
  // Then two token tiles share a row tile's codes; up to 64 tokens, from 768 tiles on (3 CTAs of two tiles per SM), four
  // share two row tiles' while their CTAs still run at once.  Two by one, four by two and the kernel for many tokens:
  //   48 x 2048 -> 2048 (768 tiles) 6.5, 6.4 us; 64 x 2048 -> 512 (256) 3.8, 6.3; 64 x 2048 -> 2048 (1024) 8.2, 7.0, 7.5
  //   32 x 2048 -> 3616 (904, 113 CTAs) 8.2, 7.1, 9.2; -> 5120 (1280, 160 CTAs) 9.9, 11.6, 12.0
  //   64 x 2048 -> 2560 (1280, 160 CTAs) 10.0, 11.7, 9.4; 48 x 2048 -> 2560 (960, 160) 8.2, 9.5, 9.1; -> 3392 (1272, 212)
  //   10.1, 10.6, 9.2
  // with fewer than 32 tokens 24 x 2048 -> 49152 54, -, 78.  K moves them alike: 64 x 512 -> 2048 4.5, 3.9, 6.2 and 4096
  // -> 2048 13.1, 10.0, 9.7; 48 x 512 -> 3392 4.9, 5.7, 6.0 and 4096 -> 3392 16.1, 15.7, 13.4.  (About 1280 tiles the
  // third is the quicker for long K and 48 tokens or more, the first by more for short K or 32.)
  const int64_t few = static_cast<int64_t>((out_features + 15) / 16) * ((num_tokens + 7) / 8);
  const int64_t four = static_cast<int64_t>((out_features + 31) / 32) * ((num_tokens + 31) / 32);  // CTAs of four by two
  if (num_tokens < 32) return launch_few<2, 1>(p, s);
  if (num_tokens <= kQ4FewTokens && few >= 768 && four <= 148) return launch_few<4, 2>(p, s);
  if (num_tokens <= kQ4FewTokens && few <= 1280) return launch_few<2, 1>(p, s);
  // More tiles of 128 tokens x 64 outputs than SMs: the large tiles, which take the same time however few there are
  // (512 x 2048 -> 2048, 128 of the small ones: 15.0 us with the large, 13.0 with the small; 256 x 2048 -> 6144, 192:
  // 15.4 and 18.7)
  const int64_t tiles = static_cast<int64_t>((num_tokens + 127) / 128) * ((out_features + 63) / 64);
  if (tiles > 148) return launch_wide(p, s);
  // K is split over a cluster while every SM has at most one CTA and each keeps at least 4 blocks of 64 (128 x 2048 ->
  // 2048, 32 tiles: 9.5, 7.5 and 9.5 us split by 2, 4 and 8; -> 6144, 96 tiles: 11.7 whole, 13.2 split by 2)
  p.split = 1;
  while (p.split < 8 && tiles * p.split * 2 <= 148 && (in_features + 63) / 64 >= 8 * p.split) p.split *= 2;
  return launch_many(p, s);
}

int hla_s6_linear_q4(const void* x, int64_t x_stride_t, const void* packed, int32_t num_tokens, int32_t out_features,
                     int32_t in_features, float scale, const void* residual, int64_t residual_stride_t, void* out,
                     int64_t out_stride_t, void* stream) {
  return hla_s6_linear_q4_checked(x, x_stride_t, packed, num_tokens, out_features, in_features, scale, residual,
                                  residual_stride_t, out, out_stride_t, nullptr, stream);
}

}  // extern "C"
