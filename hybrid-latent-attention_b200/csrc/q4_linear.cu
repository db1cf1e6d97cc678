// Linear layer with 4-bit weights (format: q4.cuh): y[t, n] = ts sum_k x[t, k] w[n, k] (+ residual[t, n]),
// fp32 accumulation, one rounding to bf16.
//
// Few tokens: the weight tile is the A operand of mma.m16n8k16 (16 output features), the tokens are N = 8,
// so one token costs no more tensor work than eight.  Codes go from global memory to registers in 16-byte
// loads and are dequantised there (exact); the 8 warps of a CTA split K and meet in shared memory.
#include "../../include/hla_s6.h"
#include "gemm_ops.cuh"
#include "hla_s6_internal.h"
#include "q4.cuh"

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
};

constexpr int kQ4LinWarps = 8;

template <int NT>
__global__ void __launch_bounds__(kQ4LinWarps * 32) q4_linear_kernel(const Q4LinearParams p) {
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
static int launch_linear(const Q4LinearParams& p, cudaStream_t s) {
  q4_linear_kernel<NT><<<dim3((p.N + 15) / 16, (p.T + 8 * NT - 1) / (8 * NT)), kQ4LinWarps * 32, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "q4_linear_kernel launch");
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (num_tokens <= 8) return launch_linear<1>(p, s);
  if (num_tokens <= 16) return launch_linear<2>(p, s);
  return launch_linear<4>(p, s);
}

}  // extern "C"
