// Paged latent-history reader over the 4-bit cache (format: q4.cuh): per token t and head h,
//   o[t, h] = v_ts sum_j p_j V[j],  p = softmax_j(scale k_ts q[t, h] . K[j]),  j < ctx[t],
// the operation of history.cu with rows of 17 W / 16 bytes instead of 4 W.  It leaves the same partials
// (slot = CTA + row, slot ranges in meta) in the same workspace, so the reduces and the fused combine of
// history.cu / combine.cu follow it unchanged.
//
// One warp owns 128 latent columns of 16-row tiles; heads are the M = 16 dimension of mma.m16n8k16.
// Codes are dequantised in registers into bf16 fragments (exact).
#include "../../include/hla_s6.h"
#include "hla_s6_internal.h"
#include "q4.cuh"

namespace hla {

struct Q4HistoryParams {
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  const uint8_t* cache;
  int64_t num_blocks, c_sb;
  int page;
  const int32_t* bt;
  int64_t bt_st;
  int32_t max_blocks;
  const int32_t* ctx;
  int32_t T, H;
  float scale_log2;  // softmax scale * k tensor scale * log2(e)
  float v_ts;
  float* ws_o;
  float* ws_lse;
  int2* meta;
  int32_t slots_cap, grid, stream_mode;
  int* err;
};

// The scale bytes of rows row0, row0 + 1 with those at or past `valid` zeroed.
__device__ __forceinline__ uint32_t mask_rows(uint32_t bytes, int row0, int valid) {
  if (row0 >= valid) return 0u;
  return row0 + 1 >= valid ? bytes & 0xffu : bytes;
}

template <int W>
__global__ void __launch_bounds__(W / 4) q4_history_kernel(const Q4HistoryParams p) {
  constexpr int NC = W / 128, G = W / kQ4Group;
  __shared__ float4 xbuf[2][NC][2][32];
  extern __shared__ int pref[];  // [T + 1] page prefix (stream mode)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, c4 = lane & 3;
  const int T = p.T, page = p.page;
  int64_t P = 0, GR = 1, p0 = 0, p1 = 0;
  int r = blockIdx.x;
  if (p.stream_mode) {
    for (int t = tid; t < T; t += blockDim.x) pref[t + 1] = (max(p.ctx[t], 0) + page - 1) / page;
    if (tid == 0) pref[0] = 0;
    __syncthreads();
    if (warp == 0) {
      int carry = 0;
      for (int b = 0; b < T; b += 32) {
        int v = b + lane < T ? pref[b + lane + 1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int n = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += n;
        }
        if (b + lane < T) pref[b + lane + 1] = v + carry;
        carry += __shfl_sync(0xffffffffu, v, 31);
      }
    }
    __syncthreads();
    P = pref[T];
    GR = p.grid < P ? static_cast<int64_t>(p.grid) : P;
    griddep_wait();
    if (blockIdx.x == 0) {
      for (int t = tid; t < T; t += blockDim.x) {
        const int a = pref[t], b = pref[t + 1];
        p.meta[t] = b > a ? make_int2(static_cast<int>(stream_owner(a, P, GR)) + t,
                                      static_cast<int>(stream_owner(b - 1, P, GR)) + t + 1)
                          : make_int2(0, 0);
      }
    }
    if (static_cast<int64_t>(blockIdx.x) >= GR) return;
    p0 = stream_start(blockIdx.x, P, GR);
    p1 = stream_start(blockIdx.x + 1, P, GR);
    int lo = 0, hi = T;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pref[mid] <= p0) lo = mid; else hi = mid;
    }
    r = lo;
  } else {
    griddep_wait();
    p1 = (max(p.ctx[r], 0) + page - 1) / page;
    if (p1 == 0) {
      if (tid < p.H && r < p.slots_cap) p.ws_lse[static_cast<int64_t>(r) * p.H + tid] = -INFINITY;
      return;
    }
  }
  if (tid == 0) griddep_launch_dependents();

  const Q4Tile tl(W);
  int buf = 0;
  for (int64_t pg = p0; pg < p1;) {  // one row's segment at a time
    int64_t base = 0, end = p1;
    if (p.stream_mode) {
      while (pg >= pref[r + 1]) ++r;
      base = pref[r];
      end = min(p1, static_cast<int64_t>(pref[r + 1]));
    }
    const int ctx = max(p.ctx[r], 0);
    const int col0 = warp * 128;
    uint32_t qa[8][4];
    {
      // fragment step s of this thread: latent columns col0 + 32 c4 + 4 s + {0,1} and {2,3}
      const __nv_bfloat16* q0 = p.q + static_cast<int64_t>(r) * p.q_st + static_cast<int64_t>(g8) * p.q_sh + col0 + 32 * c4;
      const __nv_bfloat16* q1 = q0 + 8 * p.q_sh;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        qa[s][0] = g8 < p.H ? *reinterpret_cast<const uint32_t*>(q0 + 4 * s) : 0u;
        qa[s][1] = g8 + 8 < p.H ? *reinterpret_cast<const uint32_t*>(q1 + 4 * s) : 0u;
        qa[s][2] = g8 < p.H ? *reinterpret_cast<const uint32_t*>(q0 + 4 * s + 2) : 0u;
        qa[s][3] = g8 + 8 < p.H ? *reinterpret_cast<const uint32_t*>(q1 + 4 * s + 2) : 0u;
      }
    }
    float o[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
    for (; pg < end; ++pg) {
      const int lp = static_cast<int>(pg - base);
      const int blk = lp < p.max_blocks ? p.bt[static_cast<int64_t>(r) * p.bt_st + lp] : -1;
      const bool present = blk >= 0 && blk < p.num_blocks;  // an entry outside the cache reads as zeros
      if (!present && tid == 0) record_error(p.err, kErrBlock);
      const uint8_t* pb = p.cache + (present ? static_cast<int64_t>(blk) * p.c_sb : 0);
      for (int sub = 0; sub < page; sub += 16) {
        const int valid = min(16, ctx - lp * page - sub);
        if (valid <= 0) break;
        const uint8_t* tb = pb + (sub / 16) * tl.bytes();
        // ---- partial scores over this warp's columns
        float sc[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
          const int row = 8 * j + g8;
          const uint4 kc = __ldg(reinterpret_cast<const uint4*>(tb + tl.k_codes(4 * warp + c4, row)));
          uint32_t sb = __ldg(tb + tl.k_scale(row, 4 * warp + c4));
          if (!present) sb = 0;
          const Q4Scale s(e4m3x2_to_bf2(sb | (sb << 8)));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w = i == 0 ? kc.x : (i == 1 ? kc.y : (i == 2 ? kc.z : kc.w));
            mma_bf16_16816(sc[j], qa[2 * i], q4_pair<0>(w, s), q4_pair<1>(w, s));
            mma_bf16_16816(sc[j], qa[2 * i + 1], q4_pair<2>(w, s), q4_pair<3>(w, s));
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) xbuf[buf][warp][j][lane] = make_float4(sc[j][0], sc[j][1], sc[j][2], sc[j][3]);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
          for (int w = 0; w < NC; ++w) {
            const float4 v = xbuf[buf][w][j][lane];
            sc[j][0] += v.x; sc[j][1] += v.y; sc[j][2] += v.z; sc[j][3] += v.w;
          }
        }
        buf ^= 1;
        // ---- online softmax (log2 domain)
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool in = j * 8 + 2 * c4 + e < valid;
            sc[j][e] = in ? sc[j][e] * p.scale_log2 : -INFINITY;
            sc[j][2 + e] = in ? sc[j][2 + e] * p.scale_log2 : -INFINITY;
            mx0 = fmaxf(mx0, sc[j][e]);
            mx1 = fmaxf(mx1, sc[j][2 + e]);
          }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float mn0 = fmaxf(m_run[0], mx0), mn1 = fmaxf(m_run[1], mx1);
        const float al0 = exp2f(m_run[0] - mn0), al1 = exp2f(m_run[1] - mn1);
        m_run[0] = mn0;
        m_run[1] = mn1;
        float rs0 = 0.f, rs1 = 0.f;
        uint32_t pa[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float e0 = exp2f(sc[j][0] - mn0), e1 = exp2f(sc[j][1] - mn0);
          const float e2 = exp2f(sc[j][2] - mn1), e3 = exp2f(sc[j][3] - mn1);
          rs0 += e0 + e1;
          rs1 += e2 + e3;
          pa[j * 2] = pack_bf16(e0, e1);
          pa[j * 2 + 1] = pack_bf16(e2, e3);
        }
        l_run[0] = l_run[0] * al0 + rs0;
        l_run[1] = l_run[1] * al1 + rs1;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          o[j][0] *= al0; o[j][1] *= al0;
          o[j][2] *= al1; o[j][3] *= al1;
        }
        // ---- O += P . V: rows 2c, 2c + 1 and 8 + 2c, 9 + 2c of the 16 columns col0 + 16 g8 ..
        const int vg = 4 * warp + (g8 >> 1);
        uint32_t sv = *reinterpret_cast<const uint16_t*>(tb + tl.v_scale(vg, 2 * c4));
        uint32_t sw = *reinterpret_cast<const uint16_t*>(tb + tl.v_scale(vg, 8 + 2 * c4));
        // rows past the context (or of an absent page): a zero scale, whatever their bytes are
        sv = mask_rows(present ? sv : 0u, 2 * c4, valid);
        sw = mask_rows(present ? sw : 0u, 8 + 2 * c4, valid);
        const Q4Scale s0(e4m3x2_to_bf2(sv)), s1(e4m3x2_to_bf2(sw));
#pragma unroll
        for (int oc = 0; oc < 2; ++oc) {
          const int octet = 16 * warp + 2 * g8 + oc;
          const uint2 u0 = __ldg(reinterpret_cast<const uint2*>(tb + tl.v_codes(octet, 2 * c4)));
          const uint2 u1 = __ldg(reinterpret_cast<const uint2*>(tb + tl.v_codes(octet, 8 + 2 * c4)));
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // even, odd columns of the octet
            const uint32_t sel = half ? 0x7632 : 0x5410;
            const uint32_t a = __byte_perm(u0.x, u0.y, sel), b = __byte_perm(u1.x, u1.y, sel);
            mma_bf16_16816(o[oc * 8 + half], pa, q4_pair<0>(a, s0), q4_pair<0>(b, s1));
            mma_bf16_16816(o[oc * 8 + 2 + half], pa, q4_pair<1>(a, s0), q4_pair<1>(b, s1));
            mma_bf16_16816(o[oc * 8 + 4 + half], pa, q4_pair<2>(a, s0), q4_pair<2>(b, s1));
            mma_bf16_16816(o[oc * 8 + 6 + half], pa, q4_pair<3>(a, s0), q4_pair<3>(b, s1));
          }
        }
      }
    }
    // ---- segment end: the normalised partial and its lse
    float l0 = l_run[0], l1 = l_run[1];
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const int64_t slot = p.stream_mode ? static_cast<int64_t>(blockIdx.x) + r : r;
    if (slot >= p.slots_cap) {
      if (tid == 0) record_error(p.err, kErrSlots);
    } else {
      const float ln2 = 0.6931471805599453f;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int h = g8 + 8 * hh;
        if (h >= p.H) continue;
        const float inv = p.v_ts / (hh ? l1 : l0);
        float* dst = p.ws_o + (slot * p.H + h) * W + col0 + 32 * c4;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < 16; j += 4)
            *reinterpret_cast<float4*>(dst + 16 * e + j) =
                make_float4(o[j][2 * hh + e] * inv, o[j + 1][2 * hh + e] * inv, o[j + 2][2 * hh + e] * inv,
                            o[j + 3][2 * hh + e] * inv);
        if (warp == 0 && c4 == 0) p.ws_lse[slot * p.H + h] = ((hh ? m_run[1] : m_run[0]) + log2f(hh ? l1 : l0)) * ln2;
      }
    }
  }
}

template <int W>
static int launch_q4(const HistoryArgs& a, const HistoryPlan& plan, float v_ts, cudaStream_t stream) {
  Q4HistoryParams p;
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_st = a.q_st;
  p.q_sh = a.q_sh;
  p.cache = static_cast<const uint8_t*>(a.cache);
  p.num_blocks = a.num_blocks;
  p.c_sb = a.cache_st_block;
  p.page = a.page;
  p.bt = a.block_table;
  p.bt_st = a.bt_st;
  p.max_blocks = a.max_blocks;
  p.ctx = a.ctx;
  p.T = a.T;
  p.H = a.H;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.v_ts = v_ts;
  p.ws_o = plan.ws_o;
  p.ws_lse = plan.ws_lse;
  p.meta = plan.meta;
  p.slots_cap = plan.slots_cap;
  p.grid = plan.grid;
  p.stream_mode = plan.stream_mode;
  p.err = a.err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan.grid);
  cfg.blockDim = dim3(W / 4);
  cfg.dynamicSmemBytes = plan.stream_mode ? (a.T + 1) * sizeof(int) : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.pdl ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, q4_history_kernel<W>, p), "q4_history_kernel launch");
}

// a.scale is the softmax scale times the K tensor scale; a.cache_st_block counts bytes.
int q4_history_split(const HistoryArgs& a, const HistoryPlan& plan, float v_ts, cudaStream_t stream) {
  if (a.T == 0) return kStatusOk;
  switch (a.W) {
    case 256: return launch_q4<256>(a, plan, v_ts, stream);
    case 512: return launch_q4<512>(a, plan, v_ts, stream);
    case 1024: return launch_q4<1024>(a, plan, v_ts, stream);
    default: set_error("unsupported latent width %d (256, 512 or 1024)", a.W); return kStatusInvalid;
  }
}

}  // namespace hla

using namespace hla;

static int q4_args(HistoryArgs& a, const void* q, int64_t q_st, int64_t q_sh, const void* cache, int64_t num_blocks,
                   int64_t st_block, const int32_t* bt, int64_t bt_st, int32_t max_blocks, const int32_t* ctx, int32_t T,
                   int32_t H, int32_t W, int32_t page, float scale, int32_t splits, float* ws, int64_t ws_floats,
                   float k_scale, float v_scale, int* err) {
  if (T < 0 || H < 1 || H > 16 || splits < 1) {
    set_error("history attention (4 bit) needs 1..16 query heads and num_kv_splits >= 1 (got H=%d, T=%d)", H, T);
    return kStatusInvalid;
  }
  if (W != 256 && W != 512 && W != 1024) {
    set_error("history attention (4 bit): latent width %d unsupported (256, 512 or 1024)", W);
    return kStatusInvalid;
  }
  if (page < 16 || page % 16) {
    set_error("history attention (4 bit): page size %d is not a multiple of 16", page);
    return kStatusInvalid;
  }
  if ((q_st % 8) || (q_sh % 8) || (reinterpret_cast<uintptr_t>(q) % 16)) {
    set_error("history attention (4 bit): q_lat needs 16-byte aligned rows and a unit last-dim stride");
    return kStatusInvalid;
  }
  if ((reinterpret_cast<uintptr_t>(cache) % 16) || st_block % 16 || st_block < static_cast<int64_t>(page) * 17 * W / 16 ||
      num_blocks < 1) {
    set_error("history attention (4 bit): the cache needs a 16-byte aligned base and a block stride that is a "
              "multiple of 16 bytes and holds a page (%lld)", static_cast<long long>(st_block));
    return kStatusInvalid;
  }
  if (!(k_scale > 0.f && k_scale <= 3.0e38f && v_scale > 0.f && v_scale <= 3.0e38f)) {
    set_error("history attention (4 bit): tensor scales must be positive and finite");
    return kStatusInvalid;
  }
  if (reinterpret_cast<uintptr_t>(ws) % 16) {
    set_error("history attention (4 bit): the workspace must be 16-byte aligned");
    return kStatusInvalid;
  }
  a.q = q;
  a.q_st = q_st;
  a.q_sh = q_sh;
  a.cache = cache;
  a.num_blocks = num_blocks;
  a.cache_st_block = st_block;
  a.block_table = bt;
  a.bt_st = bt_st;
  a.max_blocks = max_blocks;
  a.ctx = ctx;
  a.T = T;
  a.H = H;
  a.W = W;
  a.page = page;
  a.scale = scale * k_scale;
  a.num_kv_splits = splits;
  a.ws = ws;
  a.ws_floats = ws_floats;
  a.waves = 1;
  a.err = err;
  return kStatusOk;
}

extern "C" {

int hla_s6_history_attention_q4(const void* q_lat, int64_t q_stride_t, int64_t q_stride_h, const void* cache,
                                int64_t num_blocks, int64_t cache_stride_block, const int32_t* block_table,
                                int64_t block_table_stride, int32_t max_blocks, const int32_t* ctx,
                                const uint8_t* empty, int32_t num_tokens, int32_t num_heads, int32_t width,
                                int32_t page, float scale, int32_t num_kv_splits, float* workspace,
                                int64_t workspace_floats, float k_scale, float v_scale, void* out,
                                int64_t out_stride_t, int64_t out_stride_h, float* lse, int* error_flag,
                                void* stream) {
  HistoryArgs a{};
  int rc = q4_args(a, q_lat, q_stride_t, q_stride_h, cache, num_blocks, cache_stride_block, block_table,
                   block_table_stride, max_blocks, ctx, num_tokens, num_heads, width, page, scale, num_kv_splits,
                   workspace, workspace_floats, k_scale, v_scale, error_flag);
  if (rc) return rc;
  HistoryPlan plan;
  if ((rc = history_plan(a, &plan))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((rc = q4_history_split(a, plan, v_scale, s))) return rc;
  return history_reduce(a, plan, empty, out, out_stride_t, out_stride_h, nullptr, lse, s);
}

int hla_s6_history_partials_q4(const void* q_lat, int64_t q_stride_t, int64_t q_stride_h, const void* cache,
                               int64_t num_blocks, int64_t cache_stride_block, const int32_t* block_table,
                               int64_t block_table_stride, int32_t max_blocks, const int32_t* ctx, int32_t num_tokens,
                               int32_t num_heads, int32_t width, int32_t page, float scale, int32_t num_kv_splits,
                               float* workspace, int64_t workspace_floats, float k_scale, float v_scale,
                               int* error_flag, int32_t flags, void* stream) {
  if (flags & ~HLA_S6_PARTIALS_AFTER_QUERY) {
    set_error("history partials: unknown flags 0x%x", flags);
    return kStatusInvalid;
  }
  HistoryArgs a{};
  int rc = q4_args(a, q_lat, q_stride_t, q_stride_h, cache, num_blocks, cache_stride_block, block_table,
                   block_table_stride, max_blocks, ctx, num_tokens, num_heads, width, page, scale, num_kv_splits,
                   workspace, workspace_floats, k_scale, v_scale, error_flag);
  if (rc) return rc;
  a.pdl = (flags & HLA_S6_PARTIALS_AFTER_QUERY) != 0;
  HistoryPlan plan;
  if ((rc = history_plan(a, &plan))) return rc;
  return q4_history_split(a, plan, v_scale, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
