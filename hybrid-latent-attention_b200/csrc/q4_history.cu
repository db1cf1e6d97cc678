// Paged latent-history reader over the 4-bit cache (format: q4.cuh): per token t and head h,
//   o[t, h] = v_ts sum_j p_j V[j],  p = softmax_j(scale k_ts q[t, h] . K[j]),  j < ctx[t],
// the operation of history.cu with rows of 17 W / 16 bytes instead of 4 W.  It leaves the same partials
// (slot = CTA + row, slot ranges in meta) in the same workspace, so the reduces and the fused combine of
// history.cu / combine.cu follow it unchanged.
//
// What bounds it.  A row of 512-wide latents is 544 bytes and 16384 multiply-adds for 16 heads: 60 flop per
// byte, four times the bf16 reader's.  mma.sync runs at 1024 multiply-adds per clock and SM here (8 clocks of
// issue per m16n8k16 and scheduler, measured), which alone is 0.7 of the time HBM gives a row; the codes also
// have to become f16 values, two per register, at about 11 instructions per word of 8.  A first version on
// mma.sync did both on the same schedulers and took 260 us where the bytes take 43 (64 requests of 8160 rows).
// So the products are on tcgen05, which issues asynchronously from one thread, and the schedulers only
// dequantise.  Written to shared memory the dequantised values would need 2 KB a row in and 2 KB out of it
// beside the codes, more than its bandwidth; the A operand of tcgen05.mma may lie in tensor memory instead,
// which the dequantising threads write directly.  Keys (for the scores) and latent columns (for the output)
// are therefore the M = 128 lanes and the heads are N = 16:
//   S^T [128 keys x 16 heads]    = K [128 x W] (tensor memory) . Q^T (shared memory, f16)
//   O^T [128 columns x 16 heads] += V^T [128 x 16 rows] (tensor memory) . P^T (shared memory, f16), W / 128 of them
// One CTA per SM takes 128 rows ("step") at a time:
//   warps 0-7   K: a thread dequantises one row into its lane, 128 columns (a chunk) at a time; the two groups of
//               four warps take turns.
//   warps 8-15  V: thread 4 g + c takes 4 rows x W / 32 columns of a tile as a 16x256b fragment (lane = column);
//               two groups as well.
//   warps 16-23 softmax: a thread has the scores of its key for the 8 heads of its group.  The exponent base of a
//               head only moves when a score passes it by 2^4 (a vote), so the output is rescaled rarely and the
//               common step needs no reduction at all.  They also write the segment's output.
//   warp 24, 25 one thread each issues the score and the value products.
//   warp 26, 27 bulk copies of the tiles' K and V halves into a ring each, of 5 units of 17408 bytes (2, 4 or 8 tiles):
//               K is used a step or more before V, and in one ring of whole tiles its units waited for that.
// Code size is what costs most after the arithmetic: the warps of a scheduler run different roles, whose loops share
// its instruction caches.  So the loops over chunks, tiles and steps are rolled and the short ones inside unrolled (64
// requests of 8160 rows, 79 us as it is: K chunks unrolled 99, V tiles unrolled 94, V octets rolled 86, K halves rolled
// 82, the issuing loops unrolled 5 more).
//
// Measured: 64 requests of 8160 rows, width 512: 79.5 us (3.6 TB/s, 215 TFLOP/s; the bytes alone 43.6); 4 of 65501: 45.5
// us (21.7); 37 of 0 to 16384, width 256: 27.4 us.  A step of 128 rows takes 5200 clocks, its bytes 2980.  It is 14000
// warp instructions, 3500 a scheduler: their issue alone is 1.17 times the bytes.  5600 of them dequantise (11 for each of
// the 16384 words of a step, 32 words a warp); the rest is softmax, tensor-memory and shared-memory traffic, addresses
// and waits, and the other 1700 clocks are hand-overs between the roles that nothing covers.  Slower: two CTAs of 13
// warps per SM (112 us), all on mma.sync (118).
// f16 instead of bf16 because its 10-bit mantissa takes a nibble at either of two places (q4.cuh): both operands
// of an MMA have one type, so q is scaled by a power of two per head into f16's range (exact but for elements
// 2^-26 below the head's largest, whose error is 2^-37 of it), and p is carried as 2^11 p <= 2^15, rounded to 11
// bits or, below p = 2^-25, to a multiple of 2^-35.
#include "../../include/hla_s6.h"
#include "hla_s6_internal.h"
#include "q4.cuh"
#include "tc.cuh"

namespace hla {

struct Q4HistoryParams {
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  const uint8_t* cache;
  int64_t num_blocks, c_sb;
  int tpp;  // 16-row tiles per page
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
  int32_t slots_cap, parts, stream_mode;  // parts: CTAs of the partition (stream mode)
  uint32_t sixteen;  // 16 (q4_word_h)
  int* err;
  uint64_t wait_ns;
};

template <int W>
struct Q4Cfg {
  static constexpr int NB = W / 128;             // blocks of 128 latent columns (output accumulators)
  static constexpr int HALF = 17 * W / 2;        // bytes of a tile's K or V: codes [8 W], scales [W / 2]
  static constexpr int SCALES = 8 * W;           // where the scales begin
  static constexpr int UT = 2048 / W;            // tiles per ring unit
  static constexpr int UNIT = UT * HALF;         // 17408
  static constexpr int UNITS = 5;
  // tiles per V chunk (width 512, 64 x 8160 rows: 85.6, 80.3 and 79.4 us at 1, 2 and 4)
  static constexpr int VT = W == 256 ? 2 : W == 512 ? 4 : 1;
  static constexpr int VCOLS = NB * VT * 8;      // its tensor-memory columns
  static constexpr int KB = 2;                   // K chunks in tensor memory (4 at width 256: no faster)
  static constexpr int VB = W == 256 ? 4 : 2;    // V chunks
  static constexpr int Q_BYTES = 32 * W;
  static constexpr int P_BYTES = 2 * 4096;  // two steps
  // tensor-memory columns: K chunks (128 rows x 128 latent columns), V chunks, two score tiles, output
  static constexpr uint32_t AK = 0, AV = AK + KB * 64, S = AV + VB * VCOLS, O = S + 32;
  static_assert(O + NB * 16 <= 512, "tensor memory");
  static constexpr int SMEM = 1024 + Q_BYTES + P_BYTES + 2 * UNITS * UNIT + 1024;  // + 4 (T + 1) in stream mode
};
constexpr int kQSlots = 4;  // score factors of this many segments: the K warps run at most 3 segments ahead
constexpr int kQ4HistThreads = 28 * 32;
// log2 of how far a score may pass its head's exponent base before the base moves, and of the factor the
// probabilities carry: together they end at 2^15, f16's largest power of two.  A small first term lets small
// probabilities keep f16's precision, a large one makes rescales rare (each costs about one step).
constexpr float kQ4Over = 4.f, kQ4Lift = 11.f;

// Sum or maximum of each of 8 values over a warp: halving exchanges, after which lane l holds value rev8(l % 8)
// of all 32 lanes.
template <bool MAX>
__device__ __forceinline__ float reduce8(float (&v)[8], int lane) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int half = 4 >> k;
    const bool up = (lane >> k) & 1;
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float give = up ? v[j] : v[j + half], keep = up ? v[j + half] : v[j];
      const float got = __shfl_xor_sync(0xffffffffu, give, 1 << k);
      v[j] = MAX ? fmaxf(keep, got) : keep + got;
    }
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) {
    const float got = __shfl_xor_sync(0xffffffffu, v[0], o);
    v[0] = MAX ? fmaxf(v[0], got) : v[0] + got;
  }
  return v[0];
}
__device__ __forceinline__ int rev8(int l) { return ((l & 1) << 2) | (l & 2) | ((l & 4) >> 2); }

// 2^x to 2^-22 relative (0 for -inf and below 2^-126, where it only feeds sums of terms up to 2^15).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Barrier of `threads` threads that returns whether the predicate holds in any of them.
__device__ __forceinline__ bool named_bar_or(int id, int threads, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.u32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, %2, %3, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r)
      : "r"(pred ? 1u : 0u), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}

// The partition over the CTAs (stream mode) counts half steps: a row costs 2 a step of 128 rows and 1 for what its
// segment takes to begin and end, and is only cut between steps (a cut one costs its CTAs a step each).  Cut at pages
// and without that 1, short rows piled up in a CTA, up to 5 segments and 8 steps where 5 were due (37 rows of 0 to
// 16384, width 256: 35 us against 29; 64 rows of 8160, width 512: 102 against 97, both on a form before this one).
__device__ __forceinline__ int q4_cost(int ctx) { return ctx > 0 ? 2 * ((ctx - 1) / 128 + 1) + 1 : 0; }
// The step at cost x of a row: a CTA that starts there begins with it, one that ends there ends before it.
__device__ __forceinline__ int q4_step_at(int x) { return x > 0 ? (x - 1) >> 1 : 0; }

// The steps of a CTA: up to 8 consecutive tiles of one row's segment.  Every role walks them by itself.
struct Q4Walk {
  const Q4HistoryParams& p;
  const int* pref;  // prefix of the rows' costs (stream mode)
  int r, pg, p1, tile, tend, n, ctx, slot;
  bool first, last;
  __device__ Q4Walk(const Q4HistoryParams& p_, const int* pref_, int r0, int p0, int p1_)
      : p(p_), pref(pref_), r(r0), pg(p0), p1(p1_), tile(0), tend(0), n(0), ctx(0), slot(0), first(false), last(false) {}
  __device__ __forceinline__ bool next() {
    tile += n;
    first = tile >= tend;
    if (first) {
      if (p.stream_mode) {
        do {
          if (pg >= p1) return false;
          while (pg >= pref[r + 1]) ++r;
          const int base = pref[r], end = min(p1, pref[r + 1]);
          ctx = p.ctx[r];
          tile = 8 * q4_step_at(pg - base);
          tend = min(8 * q4_step_at(end - base), (ctx + 15) >> 4);
          pg = end;
          slot = blockIdx.x + r;
        } while (tile >= tend);  // the range ends before the row's next step
      } else {
        for (r = pg; r < p.T; r += gridDim.x) {
          ctx = p.ctx[r];
          if (ctx > 0) break;
        }
        if (r >= p.T) return false;
        pg = r + gridDim.x;
        tile = 0;
        tend = (ctx + 15) >> 4;
        slot = r;
      }
    }
    n = min(8, tend - tile);
    last = tile + n >= tend;
    return true;
  }
};

template <int W>
__global__ void __launch_bounds__(kQ4HistThreads, 1) q4_history_kernel(const Q4HistoryParams p) {
  using C = Q4Cfg<W>;
  constexpr int NB = C::NB, UT = C::UT;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // (an offset, not a rounded pointer: the compiler then knows that these are shared-memory addresses)
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  uint8_t* qs = smem;
  uint8_t* ps = qs + C::Q_BYTES;
  uint8_t* k_units = ps + C::P_BYTES;
  uint8_t* v_units = k_units + C::UNITS * C::UNIT;
  uint8_t* ctl = v_units + C::UNITS * C::UNIT;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(ctl);  // [UNITS] unit copied
  uint64_t* k_empty = k_full + C::UNITS;                // [UNITS] unit read
  uint64_t* v_full = k_empty + C::UNITS;
  uint64_t* v_empty = v_full + C::UNITS;
  uint64_t* akf = v_empty + C::UNITS;                 // [KB] K chunk in tensor memory
  uint64_t* ake = akf + C::KB;                        // [KB] its MMAs are done
  uint64_t* avf = ake + C::KB;                        // [VB] V chunk
  uint64_t* ave = avf + C::VB;
  uint64_t* sf = ave + C::VB;                       // [2] scores of a step
  uint64_t* se = sf + 2;                              // [2] read
  uint64_t* qf = se + 2;                              // [kQSlots] score factors of a segment
  uint64_t* pf = qf + kQSlots;                        // [2] probabilities of a step written
  uint64_t* pv = pf + 2;                              // [2] value products of a step done
  uint64_t* drain = pv + 2;                           // [2] every MMA of an issuer is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  float* qscale = reinterpret_cast<float*>(ctl + 512);  // [kQSlots][16] score factor of a head, by segment
  float* red = qscale + kQSlots * 16;                   // [2][4][8] per-warp maxima / sums
  int* pref = reinterpret_cast<int*>(ctl + 1024);       // [T + 1] (stream mode)

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int r0 = 0, p0 = 0, p1 = 0;
  int P = 0, G = 1;
  if (p.stream_mode) {
    for (int t = tid; t < p.T; t += blockDim.x) pref[t + 1] = q4_cost(p.ctx[t]);
    if (tid == 0) pref[0] = 0;
    __syncthreads();
    if (warp == 0) {
      int carry = 0;
      for (int b = 0; b < p.T; b += 32) {
        int v = b + lane < p.T ? pref[b + lane + 1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int n = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += n;
        }
        if (b + lane < p.T) pref[b + lane + 1] = v + carry;
        carry += __shfl_sync(0xffffffffu, v, 31);
      }
    }
    __syncthreads();
    P = pref[p.T];
    G = min(p.parts, max(P / 2, 1));  // ranges of 2 or more: a CTA between the first and the last of a row has a step
    if (P == 0 || static_cast<int>(blockIdx.x) >= G) {
      if (blockIdx.x == 0) {  // no rows at all: every slot range is empty
        griddep_wait();
        for (int t = tid; t < p.T; t += blockDim.x) p.meta[t] = make_int2(0, 0);
      }
      return;
    }
    p0 = static_cast<int>(stream_start(blockIdx.x, P, G));
    p1 = static_cast<int>(stream_start(blockIdx.x + 1, P, G));
    int lo = 0, hi = p.T;  // the row that p0 is in
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pref[mid] <= p0) lo = mid; else hi = mid;
    }
    r0 = lo;
  } else {
    p0 = blockIdx.x;  // rows blockIdx.x, + gridDim.x, ...
  }

  if (warp == 24) tc::alloc(tmem_slot, 512);
  if (tid == 25 * 32) {
    for (int s = 0; s < C::UNITS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], UT);  // the K warps of its tiles (one for two tiles in each group)
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 8);
    }
    for (int b = 0; b < C::KB; ++b) {
      mbar_init(&akf[b], 4);
      mbar_init(&ake[b], 1);
    }
    for (int b = 0; b < C::VB; ++b) {
      mbar_init(&avf[b], 4);
      mbar_init(&ave[b], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sf[b], 1);
      mbar_init(&se[b], 8);
      mbar_init(&pf[b], 8);
      mbar_init(&pv[b], 1);
      mbar_init(&drain[b], 1);
    }
    for (int b = 0; b < kQSlots; ++b) mbar_init(&qf[b], 8);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const tc::Waits wait{abort_flag, p.err, p.wait_ns};
  const uint32_t sixteen = p.sixteen;
  Q4Walk st(p, pref, r0, p0, p1);

  if (warp < 8) {
    // ------------------------------------------------------------------ K rows
    // Launched as a programmatic dependent of the launch that writes q, this grid has been copying tiles
    // meanwhile; q is read only once that launch has completed.
    griddep_wait();
    const int grp = warp >> 2, w = warp & 3;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(w * 32) << 16);
    const int u0 = 2 * w / UT, row = lane & 15;              // the unit of the step with this warp's two tiles
    const int tile_off = (2 * w - u0 * UT + (lane >> 4)) * C::HALF;
    int unit0 = 0;        // ring position of the step's first unit
    uint32_t chunk = 0;   // chunks before this step
    int seg = 0;
    for (uint32_t i = 0; st.next(); ++i) {
      if (st.first) {
        if (i > 0) wait(&sf[(i - 1) & 1], ((i - 1) >> 1) & 1, kErrWaitFull);  // the scores before read Q no more
        // the row's queries: 16 threads per head, W / 16 columns each
        const int h = tid >> 4, part = tid & 15;
        const __nv_bfloat16* src = p.q + static_cast<int64_t>(st.r) * p.q_st + static_cast<int64_t>(h) * p.q_sh + part * (W / 16);
        uint4 v[W / 128];
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < W / 128; ++k) {
          v[k] = h < p.H ? reinterpret_cast<const uint4*>(src)[k] : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t x[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(x[j] << 16)), fabsf(__uint_as_float(x[j] & 0xffff0000u))));
        }
        __syncwarp();
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        // a power of two that puts the head's largest element into [2^12, 2^13) (an infinity stays one)
        int e = static_cast<int>((__float_as_uint(amax) >> 23) & 255u) - 127 - 12;
        e = e > 110 ? 110 : (e < -110 ? -110 : e);
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        if (part == 0) qscale[seg % kQSlots * 16 + h] = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
        for (int k = 0; k < W / 128; ++k) {
          const uint32_t x[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          uint32_t u[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __half2 hh = __floats2half2_rn(__uint_as_float(x[j] << 16) * down, __uint_as_float(x[j] & 0xffff0000u) * down);
            u[j] = *reinterpret_cast<const uint32_t*>(&hh);
          }
          const int col = part * (W / 16) + 8 * k;
          *reinterpret_cast<uint4*>(qs + (col >> 6) * 2048 + tc::sw128(h, (col >> 3) & 7)) = make_uint4(u[0], u[1], u[2], u[3]);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&qf[seg % kQSlots]);
        ++seg;
      } else if (i > 1) {
        // keeps a warp that runs ahead within two steps, so that the wait above never meets an older phase
        wait(&sf[i & 1], ((i - 2) >> 1) & 1, kErrWaitFull);
      }
      const int ring = (unit0 + u0) % C::UNITS;
      const bool unit_there = u0 * UT < st.n;
      const uint8_t* tb = k_units + ring * C::UNIT + tile_off;
      if (unit_there) wait(&k_full[ring], ((unit0 + u0) / C::UNITS) & 1, kErrWaitFull);
#pragma unroll 1
      for (int kc = grp; kc < W / 128; kc += 2) {
        const uint32_t c = chunk + kc, buf = c % C::KB;
        wait(&ake[buf], ((c / C::KB) & 1) ^ 1, kErrWaitEmpty);
        __syncwarp();
        tc::fence_after();
        const uint32_t sc = *reinterpret_cast<const uint32_t*>(tb + C::SCALES + row * (W / 32) + 4 * kc);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          Q4ScaleH s[2];
          q4_scales_h((sc >> (16 * hf)) & 0xffffu, s[0], s[1]);
#pragma unroll
          for (int gi = 0; gi < 2; ++gi) {
            const uint4 x = *reinterpret_cast<const uint4*>(tb + (4 * kc + 2 * hf + gi) * 256 + row * 16);
            uint32_t v[16];
            q4_word_h(x.x, s[gi], sixteen, v[0], v[1], v[2], v[3]);
            q4_word_h(x.y, s[gi], sixteen, v[4], v[5], v[6], v[7]);
            q4_word_h(x.z, s[gi], sixteen, v[8], v[9], v[10], v[11]);
            q4_word_h(x.w, s[gi], sixteen, v[12], v[13], v[14], v[15]);
            tc::st16(lane_base + C::AK + buf * 64 + (2 * hf + gi) * 16, v);
          }
        }
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&akf[buf]);
      }
      if (lane == 0 && unit_there) mbar_arrive(&k_empty[ring]);
      unit0 += (st.n + UT - 1) / UT;
      chunk += W / 128;
    }
  } else if (warp < 16) {
    // ------------------------------------------------------------------ V columns
    const int w = warp & 3, g = lane >> 2, c = lane & 3;
    const uint32_t grp = (warp >> 2) & 1;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(w * 32) << 16);
    const int col0 = (8 * w + g) * 4 * NB;  // this thread's 4 NB columns
    int unit = 0;
    uint32_t chunk = 0;
    while (st.next()) {
      for (int ut = 0; ut < st.n; ut += UT, ++unit) {
        const int ring = unit % C::UNITS;
        const uint8_t* ub = v_units + ring * C::UNIT;
        wait(&v_full[ring], (unit / C::UNITS) & 1, kErrWaitFull);
        const int tiles = min(UT, st.n - ut);
#pragma unroll 1
        for (int t0 = ((chunk + ut / C::VT) & 1) == grp ? 0 : C::VT; t0 < tiles; t0 += 2 * C::VT) {
          // chunks alternate between the groups over all steps, so that a buffer always belongs to the same group:
          // a group that met a buffer's barrier out of turn could take an older phase for the one it waits for
          const uint32_t ch = chunk + (ut + t0) / C::VT, buf = ch % C::VB;
          wait(&ave[buf], ((ch / C::VB) & 1) ^ 1, kErrWaitEmpty);
          __syncwarp();
          tc::fence_after();
#pragma unroll 1
          for (int ti = 0; ti < C::VT && t0 + ti < tiles; ++ti) {
            const uint8_t* tb = ub + (t0 + ti) * C::HALF;
            uint32_t sb = *reinterpret_cast<const uint32_t*>(tb + C::SCALES + (col0 >> 5) * 16 + 4 * c);
            // rows past the context get a zero scale, whatever their bytes are
            if (st.last) {
              const int valid = st.ctx - ((st.tile + ut + t0 + ti) << 4) - 4 * c;
              if (valid < 4) sb = valid <= 0 ? 0u : sb & ((1u << (8 * valid)) - 1u);
            }
            const Q4ScaleH s01 = q4_scale_h(e4m3x2_to_h2(sb & 0xffffu)), s23 = q4_scale_h(e4m3x2_to_h2(sb >> 16));
            const uint32_t at = lane_base + C::AV + buf * C::VCOLS + ti * 8;
            constexpr int OH = NB >= 4 ? NB / 4 : 1;  // octets per half of the lanes (width 256: one for both)
#pragma unroll
            for (int o0 = 0; o0 < NB / 2; o0 += OH) {
              uint32_t v[8 * OH][2];  // [column][rows 4c, 4c+1 | 4c+2, 4c+3]
#pragma unroll
              for (int oc = 0; oc < OH; ++oc) {
                const uint4 x = *reinterpret_cast<const uint4*>(tb + ((col0 >> 3) + o0 + oc) * 64 + 16 * c);
                uint32_t (*d)[2] = v + 8 * oc;
                q4_word_h(__byte_perm(x.x, x.y, 0x5410), s01, sixteen, d[0][0], d[2][0], d[4][0], d[6][0]);
                q4_word_h(__byte_perm(x.x, x.y, 0x7632), s01, sixteen, d[1][0], d[3][0], d[5][0], d[7][0]);
                q4_word_h(__byte_perm(x.z, x.w, 0x5410), s23, sixteen, d[0][1], d[2][1], d[4][1], d[6][1]);
                q4_word_h(__byte_perm(x.z, x.w, 0x7632), s23, sixteen, d[1][1], d[3][1], d[5][1], d[7][1]);
              }
              // block b: columns q NB + b of q = 2 hf (lanes 0..7 of half hf) and 2 hf + 1 (lanes 8..15)
              constexpr int HALVES = NB >= 4 ? 1 : 2;
#pragma unroll
              for (int hl = 0; hl < HALVES; ++hl) {
                const int hf = NB >= 4 ? o0 / OH : hl;
#pragma unroll
                for (int b = 0; b < NB; ++b)
                  tc::st_16x256(at + (static_cast<uint32_t>(hf * 16) << 16) + b * (C::VT * 8), v[2 * hl * NB + b][0],
                                v[2 * hl * NB + b][1], v[(2 * hl + 1) * NB + b][0], v[(2 * hl + 1) * NB + b][1]);
              }
            }
          }
          tc::wait_st();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&avf[buf]);
        }
        if (lane == 0) mbar_arrive(&v_empty[ring]);
      }
      chunk += (st.n + C::VT - 1) / C::VT;
    }
  } else if (warp < 24) {
    // ------------------------------------------------------------------ softmax, output: heads 8 grp .. + 7
    // the workspace may still be read by what runs before the launch this grid waits for
    griddep_wait();
    const int grp = (warp >> 2) & 1, w = warp & 3, h0 = 8 * grp;
    if (warp == 16 && lane == 0) griddep_launch_dependents();
    if (p.stream_mode && blockIdx.x == 0) {
      for (int t = tid - 512; t < p.T; t += 256) {
        const int a = pref[t], b = pref[t + 1];
        // the CTAs of the row's first and last step (its step s ends at cost 2 s + 2)
        p.meta[t] = b > a ? make_int2(static_cast<int>(stream_owner(a + 2, P, G)) + t,
                                      static_cast<int>(stream_owner(b - 1, P, G)) + t + 1)
                          : make_int2(0, 0);
      }
    }
    if (!p.stream_mode && warp == 16) {  // rows without history: their slot says so
      for (int r = blockIdx.x; r < p.T; r += gridDim.x)
        if (p.ctx[r] <= 0 && lane < p.H && r < p.slots_cap) p.ws_lse[static_cast<int64_t>(r) * p.H + lane] = -INFINITY;
    }
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(w * 32) << 16);
    const int key = 32 * w + lane, bar = 1 + grp;
    uint8_t* pk = ps + (key >> 6) * 2048 + grp * 1024 + (key & 7) * 2;  // + swizzled chunk of head h0 + h
    float* myred = red + grp * 32;
    int seg = 0;
    float mm[8], l[8];  // the base of a head minus kQ4Lift; this key's share of the sums
    for (uint32_t i = 0; st.next(); ++i) {
      if (st.first) {
        wait(&qf[seg % kQSlots], (seg / kQSlots) & 1, kErrWaitFull);
        ++seg;
      }
      const float4* fs = reinterpret_cast<const float4*>(qscale + (seg - 1) % kQSlots * 16 + h0);
      const int sb = i & 1;
      wait(&sf[sb], (i >> 1) & 1, kErrWaitFull);
      __syncwarp();
      tc::fence_after();
      uint32_t raw[8];
      tc::ld8(lane_base + C::S + sb * 16 + h0, raw);
      const float4 f0 = fs[0], f1 = fs[1];
      const float f[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
      tc::wait_ld();
      tc::fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&se[sb]);
      // a step that is not full: dead keys score -inf
      const bool dead = st.last && ((st.tile << 4) + key >= st.ctx || key >= (st.n << 4));
      float x[8], over = -INFINITY;
      if (!st.first) {
#pragma unroll
        for (int h = 0; h < 8; ++h) x[h] = fmaf(__uint_as_float(raw[h]), f[h], -mm[h]);
        if (dead) {
#pragma unroll
          for (int h = 0; h < 8; ++h) x[h] = -INFINITY;
        }
#pragma unroll
        for (int h = 0; h < 8; ++h) over = fmaxf(over, x[h]);
      }
      if (i > 1) wait(&pv[sb], ((i - 2) >> 1) & 1, kErrWaitFull);  // these probabilities replace those of step i - 2
      __syncwarp();
      if (named_bar_or(bar, 128, st.first || over > kQ4Lift + kQ4Over)) {
        // new bases: the maximum over the step's keys, per head
#pragma unroll
        for (int h = 0; h < 8; ++h) x[h] = dead ? -INFINITY : __uint_as_float(raw[h]) * f[h];
        float mx[8];
#pragma unroll
        for (int h = 0; h < 8; ++h) mx[h] = x[h];
        const float top = reduce8<true>(mx, lane);
        if (lane < 8) myred[w * 8 + rev8(lane)] = top;
        named_bar_sync(bar, 128);
        float al[8];
#pragma unroll
        for (int h = 0; h < 8; ++h) {
          float mn = fmaxf(fmaxf(myred[h], myred[8 + h]), fmaxf(myred[16 + h], myred[24 + h]));
          if (!st.first) mn = fmaxf(mn, mm[h] + kQ4Lift);
          mn = mn == -INFINITY ? -kQ4Lift : mn - kQ4Lift;  // every score -inf: any finite base
          al[h] = st.first || mn == mm[h] ? 1.f : ex2(mm[h] - mn);
          mm[h] = mn;
          l[h] = st.first ? 0.f : l[h] * al[h];
          x[h] -= mn;
        }
        if (!st.first) {
          wait(&pv[sb ^ 1], ((i - 1) >> 1) & 1, kErrWaitFull);  // no product touches the output meanwhile
          __syncwarp();
          tc::fence_after();
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            uint32_t o[8];
            tc::ld8(lane_base + C::O + b * 16 + h0, o);
            tc::wait_ld();
#pragma unroll
            for (int h = 0; h < 8; ++h) o[h] = __float_as_uint(__uint_as_float(o[h]) * al[h]);
            tc::st8(lane_base + C::O + b * 16 + h0, o);
          }
          tc::wait_st();
          tc::fence_before();
        }
        named_bar_sync(bar, 128);  // myred is read before it is written again
      }
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        const float e = ex2(x[h]);
        l[h] += e;
        *reinterpret_cast<__half*>(pk + sb * 4096 + h * 128 + ((((key >> 3) & 7) ^ h) << 4)) = __float2half_rn(e);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pf[sb]);
      if (!st.last) continue;

      // ---- segment end: the normalised partial and its lse
      float t[8];
#pragma unroll
      for (int h = 0; h < 8; ++h) t[h] = l[h];
      const float sum = reduce8<false>(t, lane);
      if (lane < 8) myred[w * 8 + rev8(lane)] = sum;
      named_bar_sync(bar, 128);
#pragma unroll
      for (int h = 0; h < 8; ++h) t[h] = myred[h] + myred[8 + h] + myred[16 + h] + myred[24 + h];
      const bool room = st.slot < p.slots_cap;
      if (!room && lane == 0) record_error(p.err, kErrSlots);
      if (room && w == 0) {
        // A partial that is NaN says so by an lse of +inf: the reduces and the combine drop a NaN from their maximum and
        // would take a row of such partials alone for one without history; +inf outweighs the others, as exp(inf - inf).
        // (fminf drops it too; as a comparison and a choice this cost 1.2 us of 80 in registers.)
#pragma unroll
        for (int h = 0; h < 8; ++h)
          if (lane == h && h0 + h < p.H)
            p.ws_lse[static_cast<int64_t>(st.slot) * p.H + h0 + h] = fminf((mm[h] + log2f(t[h])) * 0.6931471805599453f, INFINITY);
      }
#pragma unroll
      for (int h = 0; h < 8; ++h) t[h] = t[h] == 0.f ? 0.f : p.v_ts / t[h];  // 0: every score is -inf
      wait(&pv[sb], (i >> 1) & 1, kErrWaitFull);
      __syncwarp();
      tc::fence_after();
      // lane 8 q + g of warp w holds columns (8 w + g) 4 NB + q NB .. + NB - 1, one per block
      constexpr int NV = NB < 4 ? NB : 4;
      const int col = (8 * w + (lane & 7)) * 4 * NB + (lane >> 3) * NB;
#pragma unroll
      for (int b0 = 0; b0 < NB; b0 += NV) {
        uint32_t o[NV][8];
#pragma unroll
        for (int b = 0; b < NV; ++b) tc::ld8(lane_base + C::O + (b0 + b) * 16 + h0, o[b]);
        tc::wait_ld();
        if (room) {
          float* dst = p.ws_o + (static_cast<int64_t>(st.slot) * p.H + h0) * W + col + b0;
#pragma unroll
          for (int h = 0; h < 8; ++h) {
            if (h0 + h >= p.H) continue;
            if constexpr (NV == 4)
              *reinterpret_cast<float4*>(dst + h * W) =
                  make_float4(__uint_as_float(o[0][h]) * t[h], __uint_as_float(o[1][h]) * t[h],
                              __uint_as_float(o[2][h]) * t[h], __uint_as_float(o[3][h]) * t[h]);
            else
              *reinterpret_cast<float2*>(dst + h * W) =
                  make_float2(__uint_as_float(o[0][h]) * t[h], __uint_as_float(o[1][h]) * t[h]);
          }
        }
      }
      tc::fence_before();
      named_bar_sync(bar, 128);  // myred is read before it is written again
    }
  } else if (warp == 24) {
    // ------------------------------------------------------------------ score products
    if (tc::elect()) {
      const uint64_t qd = tc::desc_sw128(smem_u32(qs));
      uint32_t c = 0;
      int seg = 0;
      for (uint32_t i = 0; st.next(); ++i) {
        if (st.first) {
          wait(&qf[seg % kQSlots], (seg / kQSlots) & 1, kErrWaitFull);
          ++seg;
        }
        if (i >= 2) wait(&se[i & 1], ((i >> 1) - 1) & 1, kErrWaitEmpty);
        const uint32_t d = tmem + C::S + (i & 1) * 16;
#pragma unroll 1
        for (int kc = 0; kc < W / 128; ++kc, ++c) {
          const uint32_t buf = c % C::KB;
          wait(&akf[buf], (c / C::KB) & 1, kErrWaitFull);
          tc::fence_after();
          const uint32_t a = tmem + C::AK + buf * 64;
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            tc::mma_ts(d, a + ks * 8, qd + ((kc * 2 + (ks >> 2)) * 2048 + (ks & 3) * 32) / 16, tc::idesc(0, 128, 16),
                       kc | ks);
          tc::commit(&ake[buf]);
        }
        tc::commit(&sf[i & 1]);
      }
      tc::commit(&drain[0]);
      if (!mbar_wait(&drain[0], 0, p.wait_ns)) record_error(p.err, kErrWaitFull);
    }
  } else if (warp == 25) {
    // ------------------------------------------------------------------ value products
    if (tc::elect()) {
      uint32_t c = 0;
      for (uint32_t i = 0; st.next(); ++i) {
        wait(&pf[i & 1], (i >> 1) & 1, kErrWaitFull);
        const uint64_t pd = tc::desc_sw128(smem_u32(ps) + (i & 1) * 4096);
        const uint32_t keep = !st.first;
#pragma unroll 1
        for (int t0 = 0; t0 < 8; t0 += C::VT, ++c) {
          if (t0 >= st.n) break;
          const uint32_t buf = c % C::VB;
          wait(&avf[buf], (c / C::VB) & 1, kErrWaitFull);
          tc::fence_after();
          const uint32_t a = tmem + C::AV + buf * C::VCOLS;
#pragma unroll
          for (int ti = 0; ti < C::VT; ++ti) {
            const int t = t0 + ti;
            if (t >= st.n) break;
#pragma unroll
            for (int b = 0; b < NB; ++b)
              tc::mma_ts(tmem + C::O + b * 16, a + b * (C::VT * 8) + ti * 8, pd + ((t >> 2) * 2048 + (t & 3) * 32) / 16,
                         tc::idesc(0, 128, 16), t ? 1u : keep);
          }
          tc::commit(&ave[buf]);
        }
        tc::commit(&pv[i & 1]);
      }
      tc::commit(&drain[1]);
      if (!mbar_wait(&drain[1], 0, p.wait_ns)) record_error(p.err, kErrWaitFull);
    }
  } else {
    // ------------------------------------------------------------------ copies: warp 26 K, warp 27 V
    // codes are read once: evicted from L2 first, so that the partials and the combine's operands stay
    const uint64_t policy = l2_policy_evict_first();
    const bool is_v = warp == 27;
    uint8_t* units = is_v ? v_units : k_units;
    uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
    const Q4Tile tl(W);
    const int codes_at = is_v ? tl.v_codes(0, 0) : 0, scales_at = is_v ? tl.v_scale(0, 0) : tl.k_scale(0, 0);
    // The lanes look up 32 tiles at once: a lookup per unit, when its slot was free, kept this warp busy for longer
    // than the others took to use the unit up (64 x 8160 rows, on a form with one ring: 95 us against 91).
    int unit = 0;
    while (st.next()) {
      for (int b = st.tile; b < st.tend; b += 32) {
        const int t = b + lane, lp = t / p.tpp;
        int blk = -1;
        if (t < st.tend) {
          if (lp < p.max_blocks) blk = p.bt[static_cast<int64_t>(st.r) * p.bt_st + lp];
          if (blk < 0 || blk >= p.num_blocks) {
            record_error(p.err, kErrBlock);
            blk = -1;
          }
        }
        const uint8_t* src = p.cache + static_cast<int64_t>(blk) * p.c_sb + static_cast<int64_t>(t - lp * p.tpp) * tl.bytes();
        const unsigned absent = __ballot_sync(0xffffffffu, t < st.tend && blk < 0);
        for (int k = 0; k < 32 && b + k < st.tend; k += UT, ++unit) {
          const int ring = unit % C::UNITS, n = min(UT, st.tend - b - k);
          const bool mine = lane >= k && lane < k + n;
          if (unit >= C::UNITS) wait(&empty[ring], ((unit / C::UNITS) - 1) & 1, kErrWaitEmpty);
          __syncwarp();
          uint8_t* dst = units + ring * C::UNIT + (lane - k) * C::HALF;
          if (mine && blk < 0) {  // a page outside the table or the cache reads as zeros
            for (int o = 0; o < C::HALF; o += 16) *reinterpret_cast<uint4*>(dst + o) = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(&full[ring], (n - __popc((absent >> k) & ((1u << n) - 1u))) * C::HALF);
          __syncwarp();
          if (mine && blk >= 0) {
            tc::bulk_load(dst, src + codes_at, C::SCALES, &full[ring], policy);
            tc::bulk_load(dst + C::SCALES, src + scales_at, C::HALF - C::SCALES, &full[ring], policy);
          }
        }
      }
      st.n = st.tend - st.tile;  // the segment's steps are all taken
    }
    // after an abort no role may have waited for the last copies: they must land before the CTA ends
    if (wait.aborted() && lane == 0)
      for (int u = max(0, unit - C::UNITS); u < unit; ++u) mbar_wait(&full[u % C::UNITS], (u / C::UNITS) & 1, p.wait_ns);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 24) tc::dealloc(tmem, 512);
}

template <int W>
static int launch_q4(const HistoryArgs& a, const HistoryPlan& plan, float v_ts, cudaStream_t stream) {
  using C = Q4Cfg<W>;
  Q4HistoryParams p;
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_st = a.q_st;
  p.q_sh = a.q_sh;
  p.cache = static_cast<const uint8_t*>(a.cache);
  p.num_blocks = a.num_blocks;
  p.c_sb = a.cache_st_block;
  p.tpp = a.page / 16;
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
  p.stream_mode = plan.stream_mode;
  p.sixteen = 16;
  p.err = a.err;
  p.wait_ns = std::max(wait_limit_ns(), tc::kLeastWaitNs);
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  // one CTA per SM (its ring and tensor memory fill one); within the slots the plan's workspace holds
  const int grid = std::min(plan.grid, sms);
  p.parts = grid;
  static unsigned attr_mask = 0;
  ensure_smem_limit(q4_history_kernel<W>, C::SMEM + 4 * (kHistoryMaxStreamRows + 1), attr_mask);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kQ4HistThreads);
  cfg.dynamicSmemBytes = C::SMEM + (plan.stream_mode ? 4 * (a.T + 1) : 0);
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
