// Linear layer with 4-bit weights (format: q4.cuh): y[t, n] = ts sum_k x[t, k] w[n, k] (+ residual[t, n]),
// fp32 accumulation, one rounding to bf16.  Two kernels, by the number of tokens:
//
// q4_linear_few: the weight tile is the A operand of mma.m16n8k16 (16 output features), the tokens are N = 8, so one
// token costs no more tensor work than eight.  What bounds it is the stream of weight bytes; codes go from global
// memory to registers in 16-byte loads and are dequantised there (exact).
//
// q4_linear_many: tokens are the M = 128 rows of tcgen05.mma, x comes by TMA, and eight warps dequantise the weight
// block of the stage into shared memory in the operand's swizzled layout, one 16-byte load of codes per thread and 16
// rows, three stages ahead.  One launch and no workspace; the weight is dequantised once per 128 tokens.
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
  int vec;  // out (and residual) rows are 16-byte aligned
  uint64_t wait_ns;
};

// ------------------------------------------------------------------ few tokens
constexpr int kQ4LinWarps = 8;

template <int NT>
__global__ void __launch_bounds__(kQ4LinWarps * 32) q4_linear_few_kernel(const Q4LinearParams p) {
  __shared__ float red[kQ4LinWarps][NT][4][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int kt_n = (p.K + 127) / 128, t0 = blockIdx.y * (8 * NT);
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  for (int kt = warp; kt < kt_n; kt += kQ4LinWarps) {
    const uint8_t* tile = p.w + (static_cast<int64_t>(blockIdx.x) * kt_n + kt) * kQ4WeightTile;
    const uint4 lo = __ldg(reinterpret_cast<const uint4*>(tile) + lane);
    const uint4 hi = __ldg(reinterpret_cast<const uint4*>(tile + 512) + lane);
    const uint32_t sb = __ldg(reinterpret_cast<const uint16_t*>(tile + 1024) + lane);
    uint4 xb[NT][4];
    const int col = kt * 128 + 32 * c;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int t = t0 + 8 * j + g;
      const bool in = t < p.T && col < p.K;
      const uint4* src = reinterpret_cast<const uint4*>(p.x + static_cast<int64_t>(t) * p.x_st + col);
#pragma unroll
      for (int i = 0; i < 4; ++i) xb[j][i] = in ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
    }
    const uint32_t s2 = e4m3x2_to_bf2(sb);
    const Q4Scale s0(__byte_perm(s2, 0, 0x1010)), s1(__byte_perm(s2, 0, 0x3232));
    const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a0[4] = {q4_pair<0>(wl[i], s0), q4_pair<0>(wh[i], s1), q4_pair<1>(wl[i], s0),
                              q4_pair<1>(wh[i], s1)};
      const uint32_t a1[4] = {q4_pair<2>(wl[i], s0), q4_pair<2>(wh[i], s1), q4_pair<3>(wl[i], s0),
                              q4_pair<3>(wh[i], s1)};
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma_bf16_16816(acc[j], a0, xb[j][i].x, xb[j][i].y);
        mma_bf16_16816(acc[j], a1, xb[j][i].z, xb[j][i].w);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][j][e][lane] = acc[j][e];
  __syncthreads();
  // element (row n, token t) of tile j: lane (n % 8) * 4 + (t % 8) / 2, register 2 (n / 8) + t % 2
  for (int i = threadIdx.x; i < NT * 128; i += blockDim.x) {
    const int nl = i & 15, tl = i >> 4, t = t0 + tl, n = blockIdx.x * 16 + nl;
    if (t >= p.T || n >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kQ4LinWarps; ++w) v += red[w][tl >> 3][2 * (nl >> 3) + (tl & 1)][(nl & 7) * 4 + ((tl & 7) >> 1)];
    v *= p.ts;
    if (p.res) v += __bfloat162float(p.res[static_cast<int64_t>(t) * p.res_st + n]);
    p.out[static_cast<int64_t>(t) * p.o_st + n] = __float2bfloat16_rn(v);
  }
}

template <int NT>
static int launch_few(const Q4LinearParams& p, cudaStream_t s) {
  q4_linear_few_kernel<NT><<<dim3((p.N + 15) / 16, (p.T + 8 * NT - 1) / (8 * NT)), kQ4LinWarps * 32, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "q4_linear_few_kernel launch");
}

// ------------------------------------------------------------------ many tokens
template <int BN>
struct Q4Many {
  static constexpr int A_BYTES = 128 * 64 * 2, B_BYTES = BN * 64 * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 64 ? 4 : 4;
  static constexpr int SMEM = 1024 + STAGES * STAGE + 256;
  static constexpr int PER = BN / 128 > 0 ? BN / 128 : 1;  // 16-row tiles a dequantising warp takes per stage
  static constexpr int DQ = BN / 16 / PER;                 // dequantising warps: 4 (BN 64) or 8
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

// warps 0 .. DQ-1 dequantise, then write the output; warp DQ: TMA of x; warp DQ + 1: products.
template <int BN>
__global__ void __launch_bounds__((Q4Many<BN>::DQ + 2) * 32) q4_linear_many_kernel(
    const __grid_constant__ CUtensorMap tmap_x, const Q4LinearParams p) {
  using C = Q4Many<BN>;
  constexpr int DQ = C::DQ;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE);  // x copied and weights written
  uint64_t* empty = full + C::STAGES;
  uint64_t* done = empty + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.y * 128, n0 = blockIdx.x * BN, NK = (p.K + 63) / 64, kt_n = (p.K + 127) / 128;

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
  const tc::Waits wait{abort_flag, nullptr, p.wait_ns};

  if (warp < DQ) {
    // lane: row 8 half + g of a 16-row tile, columns 32 c .. of the stage's 64
    const int half = lane >> 4, g = (lane >> 1) & 7, c = lane & 1, row = 8 * half + g;
    const int64_t tile_row = static_cast<int64_t>(kt_n) * kQ4WeightTile;
    const uint8_t* base = p.w + (n0 / 16 + warp * C::PER) * tile_row;
    const int n_tiles = (p.N + 15) / 16;
    bool there[C::PER];
#pragma unroll
    for (int i = 0; i < C::PER; ++i) there[i] = n0 / 16 + warp * C::PER + i < n_tiles;
    constexpr int AHEAD = 3;  // stages whose codes are in flight
    uint4 code[AHEAD][C::PER];
    uint32_t sb[AHEAD][C::PER];
    auto fetch = [&](int kb, uint4 (&cd)[C::PER], uint32_t (&s)[C::PER]) {
#pragma unroll
      for (int i = 0; i < C::PER; ++i) {
        const uint8_t* tile = base + i * tile_row + static_cast<int64_t>(kb >> 1) * kQ4WeightTile;
        const int cc = 2 * (kb & 1) + c;
        const bool ok = there[i] && kb < NK;
        cd[i] = ok ? __ldg(reinterpret_cast<const uint4*>(tile + half * 512 + (g * 4 + cc) * 16)) : make_uint4(0u, 0u, 0u, 0u);
        s[i] = ok ? __ldg(tile + 1024 + (g * 4 + cc) * 2 + half) : 0u;
      }
    };
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) fetch(a, code[a], sb[a]);
    for (int kb0 = 0; kb0 < NK; kb0 += AHEAD) {
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int kb = kb0 + a;
        if (kb >= NK) break;
        const int s = kb % C::STAGES;
        if (kb >= C::STAGES) wait(&empty[s], ((kb / C::STAGES) - 1) & 1, kErrWaitEmpty);
        uint8_t* b = smem + s * C::STAGE + C::A_BYTES;
#pragma unroll
        for (int i = 0; i < C::PER; ++i) {
          const int r = (warp * C::PER + i) * 16 + row;
          const Q4Scale sc(e4m3x2_to_bf2(sb[a][i] | (sb[a][i] << 8)));
          const uint32_t w[4] = {code[a][i].x, code[a][i].y, code[a][i].z, code[a][i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(b + r * 128 + (((4 * c + j) ^ (r & 7)) << 4)) =
                make_uint4(q4_pair<0>(w[j], sc), q4_pair<1>(w[j], sc), q4_pair<2>(w[j], sc), q4_pair<3>(w[j], sc));
        }
        fetch(kb + AHEAD, code[a], sb[a]);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
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
      const int n = n0 + cw + c0;
      if (t >= p.T || n >= p.N) continue;
      __nv_bfloat16* dst = p.out + static_cast<int64_t>(t) * p.o_st + n;
      const __nv_bfloat16* rs = p.res ? p.res + static_cast<int64_t>(t) * p.res_st + n : nullptr;
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(r[e]) * p.ts;
      if (p.vec && n + 16 <= p.N) {
        if (rs) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const uint4 u = reinterpret_cast<const uint4*>(rs)[q];
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
  } else if (warp == DQ) {
    if (lane == 0) {
      prefetch_tmap(&tmap_x);
      for (int kb = 0; kb < NK; ++kb) {
        const int s = kb % C::STAGES;
        if (kb >= C::STAGES) wait(&empty[s], ((kb / C::STAGES) - 1) & 1, kErrWaitEmpty);
        mbar_arrive_expect_tx(&full[s], C::A_BYTES);
        tma_load_rows(smem + s * C::STAGE, &tmap_x, &full[s], kb * 64, m0);  // rows and columns past x are zeros
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
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == DQ) tc::dealloc(tmem, C::COLS);
}

template <int BN>
static int launch_many(const Q4LinearParams& p, cudaStream_t s) {
  using C = Q4Many<BN>;
  CUtensorMap tx;
  int rc = rows_tmap(&tx, p.x, p.T, p.K, p.x_st);
  if (rc) return rc;
  static unsigned attr_mask = 0;
  ensure_smem_limit(q4_linear_many_kernel<BN>, C::SMEM, attr_mask);
  q4_linear_many_kernel<BN><<<dim3((p.N + BN - 1) / BN, (p.T + 127) / 128), (C::DQ + 2) * 32, C::SMEM, s>>>(tx, p);
  return cuda_status(cudaGetLastError(), "q4_linear_many_kernel launch");
}

}  // namespace hla

using namespace hla;

extern "C" {

int hla_s6_linear_q4(const void* x, int64_t x_stride_t, const void* packed, int32_t num_tokens, int32_t out_features,
                     int32_t in_features, float scale, const void* residual, int64_t residual_stride_t, void* out,
                     int64_t out_stride_t, void* stream) {
  if (num_tokens < 0 || out_features < 1 || out_features > 16 * 65535 || in_features < 32 || in_features % 32 ||
      (x_stride_t % 8) || (reinterpret_cast<uintptr_t>(x) % 16) || (reinterpret_cast<uintptr_t>(packed) % 16)) {
    set_error("linear (4 bit) needs in_features %% 32 == 0, 1..1048560 out_features and 16-byte aligned x rows and "
              "weight");
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
  p.wait_ns = wait_limit_ns();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (num_tokens <= 8) return launch_few<1>(p, s);
  if (num_tokens <= 16) return launch_few<2>(p, s);
  if (num_tokens <= 32) return launch_few<4>(p, s);
  const int64_t wide = static_cast<int64_t>((num_tokens + 127) / 128) * ((out_features + 255) / 256);
  return wide >= 64 ? launch_many<256>(p, s) : launch_many<64>(p, s);
}

}  // extern "C"
