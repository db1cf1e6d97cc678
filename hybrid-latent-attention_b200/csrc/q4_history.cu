// Paged latent-history reader over the 4-bit cache (format: q4.cuh): per token t and head h,
//   o[t, h] = v_ts sum_j p_j V[j],  p = softmax_j(scale k_ts q[t, h] . K[j]),  j < ctx[t],
// the operation of history.cu with rows of 17 W / 16 bytes instead of 4 W.  It leaves the same partials
// (slot = CTA + row, slot ranges in meta) in the same workspace, so the reduces and the fused combine of
// history.cu / combine.cu follow it unchanged.
//
// What bounds it.  A row of 512-wide latents is 544 bytes and 32768 multiply-adds for 16 heads: 60 flop per
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
// A CTA takes 128 rows ("step") at a time; two CTAs share an SM and fill each other's gaps:
//   warps 0-3  dequantise the step's K rows into tensor memory (thread = row) in chunks of 128 columns, then the
//              first two chunks of V (thread 4 g + c: 4 rows x W / 32 columns as 16x256b fragments, lane = column),
//              which hides the score products' latency; then the softmax (thread = key) and the other V chunks.
//              The exponent base of a head only moves when a score passes it by 2^4 (a vote), so the output is
//              rescaled rarely and the common step needs no reduction at all.
//   warp 4     one thread issues every product.
//   warp 5     bulk copies of the K and V halves of tiles into a ring of units of 17408 bytes (the halves of 2, 4
//              or 8 tiles), in the order in which they are used.
// Roles of their own for K, V and the softmax (28 warps, one CTA per SM) took 102 us instead: each step then
// crosses more barriers than it has work between them, and the roles' code competes for the instruction caches.
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
  int32_t slots_cap, parts, stream_mode;  // parts: CTAs of the page partition (stream mode)
  uint32_t sixteen;  // 16 (q4_word_h)
  int* err;
  uint64_t wait_ns;
};

template <int W>
struct Q4Cfg {
  static constexpr int NB = W / 128;             // blocks of 128 latent columns (output accumulators)
  static constexpr int TILE = 17 * W;            // bytes of 16 rows
  static constexpr int UT = 2048 / W;            // tiles per ring unit
  static constexpr int SCALES = 16384;           // a unit: the codes of its tiles (8 W bytes each), then their scales
  static constexpr int UNIT = SCALES + 1024;
  static constexpr int CTAS = W == 1024 ? 1 : 2; // per SM: 1024 columns of output need half the tensor memory
  static constexpr int UNITS = W == 1024 ? 9 : 5;
  static constexpr int VT = UT / 2;              // tiles per V chunk: 64 columns of tensor memory, as a K chunk
  static constexpr int Q_BYTES = 32 * W;
  static constexpr int P_BYTES = 4096;
  // tensor-memory columns: two chunk buffers (K: 128 rows x 128 columns; V), the scores, the output
  static constexpr uint32_t A = 0, S = 128, O = 144;
  static constexpr uint32_t COLS = W == 1024 ? 512 : 256;
  static_assert(O + NB * 16 <= COLS, "tensor memory");
  static constexpr int SMEM = 1024 + Q_BYTES + P_BYTES + UNITS * UNIT + 768;  // + 4 (T + 1) in stream mode
};
constexpr int kQ4HistThreads = 6 * 32;
// log2 of how far a score may pass its head's exponent base before the base moves, and of the factor the
// probabilities carry: together they end at 2^15, f16's largest power of two.  A small first term lets small
// probabilities keep f16's precision, a large one makes rescales rare (each costs about one step).
constexpr float kQ4Over = 4.f, kQ4Lift = 11.f;

// Sum or maximum of each of 16 values over a warp: halving exchanges, after which lane l holds value rev16(l % 16)
// of all 32 lanes.
template <bool MAX>
__device__ __forceinline__ float reduce16(float (&v)[16], int lane) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int half = 8 >> k;
    const bool up = (lane >> k) & 1;
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float give = up ? v[j] : v[j + half], keep = up ? v[j + half] : v[j];
      const float got = __shfl_xor_sync(0xffffffffu, give, 1 << k);
      v[j] = MAX ? fmaxf(keep, got) : keep + got;
    }
  }
  const float got = __shfl_xor_sync(0xffffffffu, v[0], 16);
  return MAX ? fmaxf(v[0], got) : v[0] + got;
}
__device__ __forceinline__ int rev16(int l) { return ((l & 1) << 3) | ((l & 2) << 1) | ((l & 4) >> 1) | ((l & 8) >> 3); }

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

// The steps of a CTA: up to 8 consecutive tiles of one row's segment.  Every role walks them by itself.
struct Q4Walk {
  const Q4HistoryParams& p;
  const int* pref;  // page prefix (stream mode)
  int r, pg, p1, tile, tend, n, ctx, slot;
  bool first, last;
  __device__ Q4Walk(const Q4HistoryParams& p_, const int* pref_, int r0, int p0, int p1_)
      : p(p_), pref(pref_), r(r0), pg(p0), p1(p1_), tile(0), tend(0), n(0), ctx(0), slot(0), first(false), last(false) {}
  __device__ __forceinline__ bool next() {
    tile += n;
    first = tile >= tend;
    if (first) {
      if (p.stream_mode) {
        if (pg >= p1) return false;
        while (pg >= pref[r + 1]) ++r;
        const int base = pref[r], end = min(p1, pref[r + 1]);
        ctx = p.ctx[r];
        tile = (pg - base) * p.tpp;
        tend = min((end - base) * p.tpp, (ctx + 15) >> 4);
        pg = end;
        slot = blockIdx.x + r;
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
__global__ void __launch_bounds__(kQ4HistThreads, Q4Cfg<W>::CTAS) q4_history_kernel(const Q4HistoryParams p) {
  using C = Q4Cfg<W>;
  constexpr int NB = C::NB, UT = C::UT;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qs = smem;
  uint8_t* ps = qs + C::Q_BYTES;
  uint8_t* units = ps + C::P_BYTES;
  uint8_t* ctl = units + C::UNITS * C::UNIT;
  uint64_t* full = reinterpret_cast<uint64_t*>(ctl);  // [UNITS] unit copied
  uint64_t* empty = full + C::UNITS;                  // [UNITS] unit read
  uint64_t* af = empty + C::UNITS;                    // [2] chunk in tensor memory
  uint64_t* ae = af + 2;                              // [2] its products are done
  uint64_t* sf = ae + 2;                              // scores of a step
  uint64_t* pf = sf + 1;                              // probabilities of a step written
  uint64_t* pv = pf + 1;                              // value products of a step done
  uint64_t* drain = pv + 1;                           // every product is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  float* qscale = reinterpret_cast<float*>(ctl + 256);  // [16] score factor of a head
  float* red = qscale + 16;                             // [4][16] per-warp maxima / sums
  int* pref = reinterpret_cast<int*>(ctl + 768);        // [T + 1] (stream mode)

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int r0 = 0, p0 = 0, p1 = 0;
  int P = 0, G = 1;
  if (p.stream_mode) {
    const int page = 16 * p.tpp;
    for (int t = tid; t < p.T; t += blockDim.x) pref[t + 1] = (max(p.ctx[t], 0) + page - 1) / page;
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
    G = min(p.parts, P);
    if (static_cast<int>(blockIdx.x) >= G) {
      if (blockIdx.x == 0) {  // no rows at all: every slot range is empty
        griddep_wait();
        for (int t = tid; t < p.T; t += blockDim.x) p.meta[t] = make_int2(0, 0);
      }
      return;
    }
    p0 = static_cast<int>(stream_start(blockIdx.x, P, G));
    p1 = static_cast<int>(stream_start(blockIdx.x + 1, P, G));
    int lo = 0, hi = p.T;  // the row holding page p0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pref[mid] <= p0) lo = mid; else hi = mid;
    }
    r0 = lo;
  } else {
    p0 = blockIdx.x;  // rows blockIdx.x, + gridDim.x, ...
  }

  if (warp == 4) tc::alloc(tmem_slot, C::COLS);
  if (tid == 5 * 32) {
    for (int u = 0; u < C::UNITS; ++u) {
      mbar_init(&full[u], 1);
      mbar_init(&empty[u], 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&af[b], 4);
      mbar_init(&ae[b], 1);
    }
    mbar_init(sf, 1);
    mbar_init(pf, 4);
    mbar_init(pv, 1);
    mbar_init(drain, 1);
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

  if (warp < 4) {
    // Launched as a programmatic dependent of the launch that writes q, this grid has been copying tiles
    // meanwhile; q and the workspace (which what runs before that launch may still read) are touched only once
    // that launch has completed.
    griddep_wait();
    if (tid == 0) griddep_launch_dependents();
    if (p.stream_mode && blockIdx.x == 0) {
      for (int t = tid; t < p.T; t += 128) {
        const int a = pref[t], b = pref[t + 1];
        p.meta[t] = b > a ? make_int2(static_cast<int>(stream_owner(a, P, G)) + t,
                                      static_cast<int>(stream_owner(b - 1, P, G)) + t + 1)
                          : make_int2(0, 0);
      }
    }
    if (!p.stream_mode && warp == 0) {  // rows without history: their slot says so
      for (int r = blockIdx.x; r < p.T; r += gridDim.x)
        if (p.ctx[r] <= 0 && lane < p.H && r < p.slots_cap) p.ws_lse[static_cast<int64_t>(r) * p.H + lane] = -INFINITY;
    }
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const int key = tid;
    // K: the unit of the step with this warp's two tiles, and this lane's row in it
    const int u0 = 2 * warp / UT, tiu = 2 * warp - u0 * UT + (lane >> 4), row = lane & 15;
    const int kcode = tiu * 8 * W + row * 16, kscale = C::SCALES + (tiu * 16 + row) * (W / kQ4Group);
    // V: this thread's 4 NB columns
    const int c4 = lane & 3, col0 = (8 * warp + (lane >> 2)) * 4 * NB;
    const int vcode = col0 * 8 + 16 * c4, vscale = C::SCALES + (col0 >> 5) * 16 + 4 * c4;
    uint8_t* pk = ps + (key >> 6) * 2048 + (key & 7) * 2;  // + swizzled chunk of a head
    int slot0 = 0;              // ring slot of the step's first unit
    uint32_t ring_phase = 0;    // and its parity
    uint32_t chunk = 0;         // chunks so far: buffer chunk & 1
    float mm[16], l[16];        // the base of a head minus kQ4Lift; this key's share of the sums

    auto chunk_begin = [&]() {
      wait(&ae[chunk & 1], ((chunk >> 1) & 1) ^ 1, kErrWaitEmpty);
      __syncwarp();
      tc::fence_after();
    };
    auto chunk_end = [&]() {
      tc::wait_st();
      tc::fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&af[chunk & 1]);
      ++chunk;
    };

    for (uint32_t i = 0; st.next(); ++i) {
      const int nu = (st.n + UT - 1) / UT;
      if (st.first) {
        // the row's queries: 8 threads per head, W / 8 columns each (every product with the last row's is done)
        const int h = tid >> 3, part = tid & 7;
        const __nv_bfloat16* src = p.q + static_cast<int64_t>(st.r) * p.q_st + static_cast<int64_t>(h) * p.q_sh + part * (W / 8);
        uint4 v[W / 64];
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < W / 64; ++k) {
          v[k] = h < p.H ? reinterpret_cast<const uint4*>(src)[k] : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t x[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(x[j] << 16)), fabsf(__uint_as_float(x[j] & 0xffff0000u))));
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        // a power of two that puts the head's largest element into [2^12, 2^13) (an infinity stays one)
        int e = static_cast<int>((__float_as_uint(amax) >> 23) & 255u) - 127 - 12;
        e = e > 110 ? 110 : (e < -110 ? -110 : e);
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        if (part == 0) qscale[h] = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
        for (int k = 0; k < W / 64; ++k) {
          const uint32_t x[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          uint32_t u[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __half2 hh = __floats2half2_rn(__uint_as_float(x[j] << 16) * down, __uint_as_float(x[j] & 0xffff0000u) * down);
            u[j] = *reinterpret_cast<const uint32_t*>(&hh);
          }
          const int col = part * (W / 8) + 8 * k;
          *reinterpret_cast<uint4*>(qs + (col >> 6) * 2048 + tc::sw128(h, (col >> 3) & 7)) = make_uint4(u[0], u[1], u[2], u[3]);
        }
        fence_proxy_async();     // ordered before the products by the chunk barriers below
        named_bar_sync(1, 128);  // qscale
      }

      // ---- K: thread = row
      {
        int slot = slot0 + u0;
        const bool wrap = slot >= C::UNITS;
        if (wrap) slot -= C::UNITS;
        const uint8_t* ub = units + slot * C::UNIT;
        if (u0 < nu) wait(&full[slot], ring_phase ^ (wrap ? 1u : 0u), kErrWaitFull);
#pragma unroll 1
        for (int kc = 0; kc < W / 128; ++kc) {
          const uint32_t sc = *reinterpret_cast<const uint32_t*>(ub + kscale + 4 * kc);
          chunk_begin();
          const uint32_t at = lane_base + C::A + (chunk & 1) * 64;
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            Q4ScaleH s[2];
            q4_scales_h((sc >> (16 * hf)) & 0xffffu, s[0], s[1]);
#pragma unroll
            for (int gi = 0; gi < 2; ++gi) {
              const uint4 x = *reinterpret_cast<const uint4*>(ub + kcode + kc * 1024 + (2 * hf + gi) * 256);
              uint32_t v[16];
              q4_word_h(x.x, s[gi], sixteen, v[0], v[1], v[2], v[3]);
              q4_word_h(x.y, s[gi], sixteen, v[4], v[5], v[6], v[7]);
              q4_word_h(x.z, s[gi], sixteen, v[8], v[9], v[10], v[11]);
              q4_word_h(x.w, s[gi], sixteen, v[12], v[13], v[14], v[15]);
              tc::st16(at + (2 * hf + gi) * 16, v);
            }
          }
          chunk_end();
        }
        // the step's K units are free: every warp releases each of them
        if (lane == 0)
          for (int u = 0; u < nu; ++u) mbar_arrive(&empty[slot0 + u < C::UNITS ? slot0 + u : slot0 + u - C::UNITS]);
        slot0 += nu;
        if (slot0 >= C::UNITS) {
          slot0 -= C::UNITS;
          ring_phase ^= 1u;
        }
      }

      // ---- V: thread = 4 rows x 4 NB columns of a tile
      auto dequant_v = [&](int t0) {
        if (t0 % UT == 0) wait(&full[slot0], ring_phase, kErrWaitFull);
        chunk_begin();
        const uint8_t* ub = units + slot0 * C::UNIT;
#pragma unroll 1
        for (int ti = 0; ti < C::VT && t0 + ti < st.n; ++ti) {
          const int tu = (t0 + ti) % UT;
          uint32_t sb = *reinterpret_cast<const uint32_t*>(ub + vscale + tu * (W / 2));
          // rows past the context get a zero scale, whatever their bytes are
          if (st.last) {
            const int valid = st.ctx - ((st.tile + t0 + ti) << 4) - 4 * c4;
            if (valid < 4) sb = valid <= 0 ? 0u : sb & ((1u << (8 * valid)) - 1u);
          }
          const Q4ScaleH s01 = q4_scale_h(e4m3x2_to_h2(sb & 0xffffu)), s23 = q4_scale_h(e4m3x2_to_h2(sb >> 16));
          const uint32_t at = lane_base + C::A + (chunk & 1) * 64 + ti * 8;
          constexpr int OH = NB >= 4 ? NB / 4 : 1;  // octets per half of the lanes (width 256: one for both)
#pragma unroll
          for (int o0 = 0; o0 < NB / 2; o0 += OH) {
            uint32_t v[8 * OH][2];  // [column][rows 4c, 4c+1 | 4c+2, 4c+3]
#pragma unroll
            for (int oc = 0; oc < OH; ++oc) {
              const uint4 x = *reinterpret_cast<const uint4*>(ub + vcode + tu * 8 * W + (o0 + oc) * 64);
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
        chunk_end();
        if ((t0 + C::VT) % UT == 0 || t0 + C::VT >= st.n) {  // the unit's last chunk
          if (lane == 0) mbar_arrive(&empty[slot0]);
          if (++slot0 == C::UNITS) {
            slot0 = 0;
            ring_phase ^= 1u;
          }
        }
      };

      // ---- softmax: thread = key
      auto softmax = [&]() {
        wait(sf, i & 1, kErrWaitFull);
        __syncwarp();
        tc::fence_after();
        uint32_t raw[16];
        tc::ld16(lane_base + C::S, raw);
        float f[16];
#pragma unroll
        for (int h = 0; h < 16; h += 4) {
          const float4 x = *reinterpret_cast<const float4*>(qscale + h);
          f[h] = x.x, f[h + 1] = x.y, f[h + 2] = x.z, f[h + 3] = x.w;
        }
        tc::wait_ld();
        tc::fence_before();
        // a step that is not full: dead keys score -inf
        const bool dead = st.last && ((st.tile << 4) + key >= st.ctx || key >= (st.n << 4));
        float x[16], over = -INFINITY;
        if (!st.first) {
#pragma unroll
          for (int h = 0; h < 16; ++h) x[h] = fmaf(__uint_as_float(raw[h]), f[h], -mm[h]);
          if (dead) {
#pragma unroll
            for (int h = 0; h < 16; ++h) x[h] = -INFINITY;
          }
#pragma unroll
          for (int h = 0; h < 16; ++h) over = fmaxf(over, x[h]);
        }
        if (named_bar_or(1, 128, st.first || over > kQ4Lift + kQ4Over)) {
          // new bases: the maximum over the step's keys, per head
#pragma unroll
          for (int h = 0; h < 16; ++h) x[h] = dead ? -INFINITY : __uint_as_float(raw[h]) * f[h];
          float mx[16];
#pragma unroll
          for (int h = 0; h < 16; ++h) mx[h] = x[h];
          const float top = reduce16<true>(mx, lane);
          if (lane < 16) red[warp * 16 + rev16(lane)] = top;
          named_bar_sync(1, 128);
          float al[16];
#pragma unroll
          for (int h = 0; h < 16; ++h) {
            float mn = fmaxf(fmaxf(red[h], red[16 + h]), fmaxf(red[32 + h], red[48 + h]));
            if (!st.first) mn = fmaxf(mn, mm[h] + kQ4Lift);
            mn = mn == -INFINITY ? -kQ4Lift : mn - kQ4Lift;  // every score -inf: any finite base
            al[h] = st.first || mn == mm[h] ? 1.f : ex2(mm[h] - mn);
            mm[h] = mn;
            l[h] = st.first ? 0.f : l[h] * al[h];
            x[h] -= mn;
          }
          if (!st.first) {
            // the products of the step before are done: their chunks' buffers have been refilled since, or soon are
            wait(pv, (i - 1) & 1, kErrWaitFull);
            __syncwarp();
            tc::fence_after();
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              uint32_t o[16];
              tc::ld16(lane_base + C::O + b * 16, o);
              tc::wait_ld();
#pragma unroll
              for (int h = 0; h < 16; ++h) o[h] = __float_as_uint(__uint_as_float(o[h]) * al[h]);
              tc::st16(lane_base + C::O + b * 16, o);
            }
            tc::wait_st();
            tc::fence_before();
          }
          named_bar_sync(1, 128);  // red is read before it is written again
        }
        if (i > 0) wait(pv, (i - 1) & 1, kErrWaitFull);  // these probabilities replace the last step's
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 16; ++h) {
          const float e = ex2(x[h]);
          l[h] += e;
          *reinterpret_cast<__half*>(pk + (h >> 3) * 1024 + (h & 7) * 128 + ((((key >> 3) & 7) ^ (h & 7)) << 4)) =
              __float2half_rn(e);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(pf);
      };

#pragma unroll 1
      for (int t0 = 0, ck = 0; t0 < st.n; t0 += C::VT, ++ck) {
        dequant_v(t0);
        // two chunks fit the buffers before the first needs probabilities
        if (ck == 1 || (ck == 0 && t0 + C::VT >= st.n)) softmax();
      }
      if (!st.last) continue;

      // ---- segment end: the normalised partial and its lse
      float t[16];
#pragma unroll
      for (int h = 0; h < 16; ++h) t[h] = l[h];
      const float sum = reduce16<false>(t, lane);
      if (lane < 16) red[warp * 16 + rev16(lane)] = sum;
      named_bar_sync(1, 128);
#pragma unroll
      for (int h = 0; h < 16; ++h) t[h] = red[h] + red[16 + h] + red[32 + h] + red[48 + h];
      const bool room = st.slot < p.slots_cap;
      if (!room && lane == 0) record_error(p.err, kErrSlots);
      if (room && warp == 0) {
#pragma unroll
        for (int h = 0; h < 16; ++h)
          if (lane == h && h < p.H)
            p.ws_lse[static_cast<int64_t>(st.slot) * p.H + h] = (mm[h] + log2f(t[h])) * 0.6931471805599453f;
      }
#pragma unroll
      for (int h = 0; h < 16; ++h) t[h] = t[h] == 0.f ? 0.f : p.v_ts / t[h];  // 0: every score is -inf
      wait(pv, i & 1, kErrWaitFull);
      __syncwarp();
      tc::fence_after();
      // lane 8 q + g of warp w holds columns (8 w + g) 4 NB + q NB .. + NB - 1, one per block
      constexpr int NV = NB < 4 ? NB : 4;
      const int col = (8 * warp + (lane & 7)) * 4 * NB + (lane >> 3) * NB;
#pragma unroll
      for (int b0 = 0; b0 < NB; b0 += NV) {
        uint32_t o[NV][16];
#pragma unroll
        for (int b = 0; b < NV; ++b) tc::ld16(lane_base + C::O + (b0 + b) * 16, o[b]);
        tc::wait_ld();
        if (room) {
          float* dst = p.ws_o + static_cast<int64_t>(st.slot) * p.H * W + col + b0;
#pragma unroll
          for (int h = 0; h < 16; ++h) {
            if (h >= p.H) continue;
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
      named_bar_sync(1, 128);  // red and the output are read before they are written again
    }
  } else if (warp == 4) {
    // ------------------------------------------------------------------ products
    if (tc::elect()) {
      const uint64_t qd = tc::desc_sw128(smem_u32(qs)), pd = tc::desc_sw128(smem_u32(ps));
      uint32_t c = 0;
      for (uint32_t i = 0; st.next(); ++i) {
#pragma unroll
        for (int kc = 0; kc < W / 128; ++kc, ++c) {
          wait(&af[c & 1], (c >> 1) & 1, kErrWaitFull);
          tc::fence_after();
          const uint32_t a = tmem + C::A + (c & 1) * 64;
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            tc::mma_ts(tmem + C::S, a + ks * 8, qd + ((kc * 2 + (ks >> 2)) * 2048 + (ks & 3) * 32) / 16,
                       tc::idesc(0, 128, 16), kc | ks);
          tc::commit(&ae[c & 1]);
        }
        tc::commit(sf);
        wait(pf, i & 1, kErrWaitFull);
        const uint32_t keep = !st.first;
#pragma unroll
        for (int t0 = 0; t0 < 8; t0 += C::VT, ++c) {
          if (t0 >= st.n) break;
          wait(&af[c & 1], (c >> 1) & 1, kErrWaitFull);
          tc::fence_after();
          const uint32_t a = tmem + C::A + (c & 1) * 64;
#pragma unroll
          for (int ti = 0; ti < C::VT; ++ti) {
            const int t = t0 + ti;
            if (t >= st.n) break;
#pragma unroll
            for (int b = 0; b < NB; ++b)
              tc::mma_ts(tmem + C::O + b * 16, a + b * (C::VT * 8) + ti * 8, pd + ((t >> 2) * 2048 + (t & 3) * 32) / 16,
                         tc::idesc(0, 128, 16), t ? 1u : keep);
          }
          tc::commit(&ae[c & 1]);
        }
        tc::commit(pv);
      }
      tc::commit(drain);
      if (!mbar_wait(drain, 0, p.wait_ns)) record_error(p.err, kErrWaitFull);
    }
  } else {
    // ------------------------------------------------------------------ tile copies: a step's K units, then its V units
    // codes are read once: evicted from L2 first, so that the partials and the combine's operands stay
    const uint64_t policy = l2_policy_evict_first();
    // lanes 0 .. 15 take the codes of a tile each, lanes 16 .. 31 the scales
    const int mine = lane & 15;
    const uint32_t bytes = lane < 16 ? 8 * W : W / 2;
    const uint32_t dst_off = (lane < 16 ? 0 : C::SCALES) + mine * bytes;
    int unit = 0, ring = 0;
    uint32_t phase = 1;  // parity of a unit's last release
    while (st.next()) {
      const int nu = (st.n + UT - 1) / UT;
      for (int hu = 0; hu < 2 * nu; ++hu, ++unit) {
        const bool v = hu >= nu;
        const int t0 = (v ? hu - nu : hu) * UT, n = min(UT, st.n - t0);
        const int t = st.tile + t0 + mine;
        const int lp = t / p.tpp;
        int blk = -1;
        if (mine < n) {
          if (lp < p.max_blocks) blk = p.bt[static_cast<int64_t>(st.r) * p.bt_st + lp];
          if (blk < 0 || blk >= p.num_blocks) {
            record_error(p.err, kErrBlock);
            blk = -1;
          }
        }
        wait(&empty[ring], phase, kErrWaitEmpty);
        __syncwarp();
        uint8_t* dst = units + ring * C::UNIT + dst_off;
        const unsigned absent = __ballot_sync(0xffffffffu, mine < n && blk < 0);
        if (mine < n && blk < 0) {  // a page outside the table or the cache reads as zeros
          for (uint32_t o = 0; o < bytes; o += 16) *reinterpret_cast<uint4*>(dst + o) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&full[ring], (n - __popc(absent & 0xffffu)) * (C::TILE / 2));
        __syncwarp();
        if (mine < n && blk >= 0)
          tc::bulk_load(dst,
                        p.cache + static_cast<int64_t>(blk) * p.c_sb + static_cast<int64_t>(t - lp * p.tpp) * C::TILE +
                            (lane < 16 ? (v ? 8 * W : 0) : 16 * W + (v ? W / 2 : 0)),
                        bytes, &full[ring], policy);
        if (++ring == C::UNITS) {
          ring = 0;
          phase ^= 1;
        }
      }
    }
    // after an abort no role may have waited for the last copies: they must land before the CTA ends
    if (wait.aborted() && lane == 0)
      for (int u = max(0, unit - C::UNITS); u < unit; ++u) mbar_wait(&full[u % C::UNITS], (u / C::UNITS) & 1, p.wait_ns);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 4) tc::dealloc(tmem, C::COLS);
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
  p.wait_ns = wait_limit_ns();
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  // as many CTAs as shared and tensor memory hold at once; within the slots the plan's workspace holds
  const int grid = std::min(plan.grid, sms * C::CTAS);
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
