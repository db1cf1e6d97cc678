// Rows of the 4-bit latent cache (format: q4.cuh): the committed row - latent RoPE of the K half in the
// torch bf16 order (register.py:73-79), quantise, paged scatter - and the gather that reads rows back for
// the rollout export (cache_export.py:160-174).  Also the one-time quantisation of a weight matrix.
#include "../../include/hla_s6.h"
#include "decode_ops.cuh"
#include "hla_s6_internal.h"
#include "q4.cuh"

namespace hla {

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// Quantise 8 columns of a group whose 32 columns sit in 4 neighbouring lanes: the word, and the scale byte
// (the same in the 4 lanes).  The maximum carries a NaN on, and a group that holds one takes the scale NaN.
__device__ __forceinline__ uint32_t quantize8(const float (&f)[8], float ts, uint32_t& scale) {
  float a = max_nan(fabsf(f[0]), fabsf(f[1]));
#pragma unroll
  for (int i = 2; i < 8; i += 2) a = max_nan(a, fabsf(f[i]), fabsf(f[i + 1]));
  a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));
  a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 2));
  uint32_t w;
  if (q4_pow2(ts)) {
    scale = q4_scale_byte_pow2(a, ts);
    w = q4_word_pow2(f, a, q4_scale_value(scale) * ts);
  } else {
    const float norm = q4_norm(ts);
    ts *= norm;
    scale = q4_scale_byte(a * norm, ts);
    const Q4Coder code(q4_scale_value(scale) * ts);
    uint32_t n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = code(f[i] * norm);
    w = q4_word(n);
  }
  if (a != a) {
    scale = kQ4ScaleNaN;
    w = kQ4Zeros;
  }
  return w;
}

struct Q4CommitArgs {
  const __nv_bfloat16* row;  // [T, 2 W] (K | V)
  int64_t row_st;
  const int64_t* positions;
  const __nv_bfloat16* table;  // [max_pos, W] = [cos | sin]
  int64_t tab_st, max_pos;
  uint8_t* cache;
  int64_t c_sb, num_blocks;
  int page;
  const int32_t* bt;
  int64_t bt_st;
  int max_blocks;
  const int32_t* qsl;
  int R, T;
  float k_ts, v_ts;
  int64_t* slot_out;
  int rounds;
};

// W / 16 threads per row; thread k holds columns 8k .. and W/2 + 8k .. of both halves, i.e. whole RoPE
// pairs and quarters of groups, so the amax of a group is two shuffles.
constexpr int kQ4CommitThreads = 128;
constexpr int kQ4CommitRounds = 4;  // rows of a thread group, one after the other, with many tokens (rule at the launch)
template <int W>
__global__ void __launch_bounds__(kQ4CommitThreads) q4_commit_kernel(const Q4CommitArgs a) {
  constexpr int PER = W / 16;
  __shared__ int32_t qsl_s[kQslCap];
  const int32_t* qsl = stage_qsl(a.qsl, a.R, qsl_s);
  constexpr int ROWS = kQ4CommitThreads / PER;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS * a.rounds;
  const Q4Tile tl(W);
  // One thread looks a row up (token_slot of decode_ops.cuh with 32-bit divisions: a position inside the table is below
  // 2^31, checked).  The row's own threads did it at first, a third of their instructions.
  __shared__ uint8_t* tile_s[ROWS * kQ4CommitRounds];  // NULL: no slot
  __shared__ int row_s[ROWS * kQ4CommitRounds];
  if (threadIdx.x < ROWS * a.rounds) {
    const int64_t t = first + threadIdx.x;
    uint8_t* tile = nullptr;
    if (t < a.T) {
      const int64_t pos = a.positions[t];
      int req;
      int64_t slot = -1;
      if (token_request(qsl, a.R, static_cast<int>(t), req) && pos >= 0 && pos < static_cast<int64_t>(a.max_blocks) * a.page) {
        const uint32_t p32 = static_cast<uint32_t>(pos), page = a.page, col = p32 / page, off = p32 - col * page;
        const int blk = a.bt[static_cast<int64_t>(req) * a.bt_st + col];
        if (blk >= 0 && blk < a.num_blocks) {
          slot = static_cast<int64_t>(blk) * a.page + off;
          tile = a.cache + static_cast<int64_t>(blk) * a.c_sb + static_cast<int64_t>(off / 16) * tl.bytes();
          row_s[threadIdx.x] = static_cast<int>(off % 16);
        }
      }
      if (a.slot_out) a.slot_out[t] = slot;
    }
    tile_s[threadIdx.x] = tile;
  }
  const int k = threadIdx.x % PER;
  for (int round = 0; round < a.rounds; ++round) {
    const int at = round * ROWS + threadIdx.x / PER;
    const int64_t t = first + at;
    uint4 raw[6] = {};
    if (t < a.T) {
      const __nv_bfloat16* src = a.row + t * a.row_st + 8 * k;
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(src + i * (W / 2)));
      const __nv_bfloat16* tab = a.table + clamp_pos(a.positions[t], a.max_pos) * a.tab_st + 8 * k;
      raw[4] = __ldg(reinterpret_cast<const uint4*>(tab));
      raw[5] = __ldg(reinterpret_cast<const uint4*>(tab + W / 2));
    }
    if (round == 0) __syncthreads();  // the lookups, behind the first row's loads
    uint8_t* const tile = tile_s[at];
    const int r = tile ? row_s[at] : 0;
    // latent RoPE of the K half in packed bf16 arithmetic: every operation rounds its exact result once, which on bf16
    // inputs is the fp32 operation rounded to bf16 (a product is exact in fp32; a sum's first rounding is innocuous)
    float x[4][8];
    {
      uint32_t* lo = reinterpret_cast<uint32_t*>(&raw[0]);
      uint32_t* hi = reinterpret_cast<uint32_t*>(&raw[1]);
      const uint32_t* cs = reinterpret_cast<const uint32_t*>(&raw[4]);
      const uint32_t* sn = reinterpret_cast<const uint32_t*>(&raw[5]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 x1 = *reinterpret_cast<const __nv_bfloat162*>(lo + i), x2 = *reinterpret_cast<const __nv_bfloat162*>(hi + i);
        const __nv_bfloat162 c = *reinterpret_cast<const __nv_bfloat162*>(cs + i), s = *reinterpret_cast<const __nv_bfloat162*>(sn + i);
        const __nv_bfloat162 y1 = __hadd2_rn(__hmul2_rn(x1, c), __hneg2(__hmul2_rn(x2, s)));
        const __nv_bfloat162 y2 = __hadd2_rn(__hmul2_rn(x2, c), __hmul2_rn(x1, s));
        lo[i] = *reinterpret_cast<const uint32_t*>(&y1);
        hi[i] = *reinterpret_cast<const uint32_t*>(&y2);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack8(raw[i], x[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t sb;
      const uint32_t w = quantize8(x[i], i < 2 ? a.k_ts : a.v_ts, sb);  // warp-collective: every lane
      if (!tile) continue;
      const int octet = k + (i & 1) * PER, group = octet / 4;
      if (i < 2) {
        *reinterpret_cast<uint32_t*>(tile + tl.k_codes(group, r) + 4 * (octet & 3)) = w;
        if ((k & 3) == 0) tile[tl.k_scale(r, group)] = static_cast<uint8_t>(sb);
      } else {
        *reinterpret_cast<uint32_t*>(tile + tl.v_codes(octet, r)) = w;
        if ((k & 3) == 0) tile[tl.v_scale(group, r)] = static_cast<uint8_t>(sb);
      }
    }
  }
}

struct Q4GatherArgs {
  const uint8_t* cache;
  int64_t c_sb, num_blocks;
  int page;
  const int32_t* blocks;   // block list: row i is row i % page of blocks[i / page]
  const int64_t* slots;    // or slots: row i is slot slots[i] (negative: zeros)
  int64_t rows;
  float k_ts, v_ts;
  __nv_bfloat16* out;      // [rows, 2 W]
  int64_t o_st;
  int* err;
};

constexpr int kQ4GatherMany = 4096;  // rows from which a thread takes four octets

// The 8 values of a word in bf16.  (n - 8) s is exact.  A power-of-two tensor scale goes into s (`folded`; the values
// stay exact, to bf16's smallest numbers), any other is applied in fp32 and rounded once.
__device__ __forceinline__ uint4 q4_values(uint32_t w, uint32_t scale, float ts, bool folded, uint32_t ts2) {
  const uint32_t s2 = e4m3x2_to_bf2(scale | (scale << 8));
  const Q4Scale s(folded ? bf2_mul(s2, ts2) : s2);
  const uint32_t v[4] = {q4_pair<0>(w, s), q4_pair<1>(w, s), q4_pair<2>(w, s), q4_pair<3>(w, s)};
  if (folded) return make_uint4(v[0], v[1], v[2], v[3]);
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = pack_bf16(__uint_as_float(v[i] << 16) * ts, __uint_as_float(v[i] & 0xffff0000u) * ts);
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// PER = W / (8 OCT) threads per row: thread k takes octets k, k + PER .. of the K and of the V half.  With one octet a
// thread a row's look-up and the tensor scale in fp32 made 12 instructions a value, which bound it (32768 rows of width
// 512: 17 us; 14.4 with four octets and the scale folded, 85 MB at 5.9 TB/s).  Few rows keep one octet a thread: they
// need the threads (77 rows of width 256: 1.6 us, 2.2 with four).  At 4096 rows the two take the same time at every width
// (one and four octets: 2.65 and 2.60 us, 3.36 and 3.27, 4.87 and 4.98 for 256, 512 and 1024; at 16384 4.7 and 4.5, 7.4
// and 6.9, 16.9 and 14.0).
template <int W, int OCT>
__global__ void __launch_bounds__(256) q4_gather_kernel(const Q4GatherArgs a) {
  constexpr int PER = W / (8 * OCT);
  const Q4Tile tl(W);
  const int k = threadIdx.x % PER;
  const uint32_t page = a.page, cache_rows = static_cast<uint32_t>(a.num_blocks) * page;  // < 2^31 (checked)
  const bool k_fold = q4_pow2(a.k_ts) && a.k_ts < 1e30f, v_fold = q4_pow2(a.v_ts) && a.v_ts < 1e30f;
  const uint32_t k_ts2 = pack_bf16(a.k_ts, a.k_ts), v_ts2 = pack_bf16(a.v_ts, a.v_ts);
  for (uint32_t i = blockIdx.x * (256 / PER) + threadIdx.x / PER; i < a.rows; i += gridDim.x * (256 / PER)) {
    uint32_t blk, off;
    bool ok, skip = false;
    if (a.slots) {
      const int64_t s = a.slots[i];
      skip = s < 0;  // a padding token: zeros, no error
      ok = !skip && s < cache_rows;
      blk = ok ? static_cast<uint32_t>(s) / page : 0u;
      off = ok ? static_cast<uint32_t>(s) - blk * page : 0u;
    } else {
      const uint32_t b = i / page;
      blk = a.blocks[b];
      off = i - b * page;
      ok = blk < static_cast<uint32_t>(a.num_blocks);  // a negative id is a large one
    }
    __nv_bfloat16* out = a.out + static_cast<int64_t>(i) * a.o_st + 8 * k;
    if (!ok) {
      if (k == 0 && !skip) record_error(a.err, kErrBlock);
#pragma unroll
      for (int j = 0; j < 2 * OCT; ++j) *reinterpret_cast<uint4*>(out + j * 8 * PER) = make_uint4(0u, 0u, 0u, 0u);
      continue;
    }
    const uint8_t* tile = a.cache + static_cast<int64_t>(blk) * a.c_sb + static_cast<int64_t>(off / 16) * tl.bytes();
    const int r = static_cast<int>(off % 16);
    uint32_t kw[OCT], vw[OCT], ks[OCT], vs[OCT];
#pragma unroll
    for (int j = 0; j < OCT; ++j) {
      const int octet = k + j * PER;
      kw[j] = __ldg(reinterpret_cast<const uint32_t*>(tile + tl.k_codes(octet / 4, r) + 4 * (octet & 3)));
      vw[j] = __ldg(reinterpret_cast<const uint32_t*>(tile + tl.v_codes(octet, r)));
      ks[j] = __ldg(tile + tl.k_scale(r, octet / 4));
      vs[j] = __ldg(tile + tl.v_scale(octet / 4, r));
    }
#pragma unroll
    for (int j = 0; j < OCT; ++j) {
      *reinterpret_cast<uint4*>(out + j * 8 * PER) = q4_values(kw[j], ks[j], a.k_ts, k_fold, k_ts2);
      *reinterpret_cast<uint4*>(out + W + j * 8 * PER) = q4_values(vw[j], vs[j], a.v_ts, v_fold, v_ts2);
    }
  }
}

// One 16-row x 128-column weight tile per CTA: thread = (row, octet).
__global__ void __launch_bounds__(256) q4_weight_kernel(const __nv_bfloat16* __restrict__ w, int64_t w_st, int N, int K,
                                                        float ts, uint8_t* __restrict__ packed) {
  const int row = threadIdx.x >> 4, octet = threadIdx.x & 15;
  const int64_t n = static_cast<int64_t>(blockIdx.y) * 16 + row;
  const int col = blockIdx.x * 128 + octet * 8;
  float f[8] = {};
  if (n < N && col < K) unpack8(__ldg(reinterpret_cast<const uint4*>(w + n * w_st + col)), f);
  uint32_t sb;
  const uint32_t word = quantize8(f, ts, sb);
  uint8_t* tile = packed + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * kQ4WeightTile;
  const int half = row >> 3, lane = (row & 7) * 4 + (octet >> 2);
  *reinterpret_cast<uint32_t*>(tile + half * 512 + lane * 16 + 4 * (octet & 3)) = word;
  if ((octet & 3) == 0) tile[1024 + lane * 2 + half] = static_cast<uint8_t>(sb);
}

static bool q4_cache_ok(const void* cache, int64_t st_block, int32_t width, int32_t page, const char* what) {
  if (width != 256 && width != 512 && width != 1024) {
    set_error("%s: latent width %d unsupported (256, 512 or 1024)", what, width);
    return false;
  }
  if (page < 16 || page % 16) {
    set_error("%s: a 4-bit cache page is a multiple of 16 rows (got %d)", what, page);
    return false;
  }
  if (reinterpret_cast<uintptr_t>(cache) % 16 || st_block % 16 || st_block < static_cast<int64_t>(page) * 17 * width / 16) {
    set_error("%s: a 4-bit cache needs a 16-byte aligned base and a block stride that is a multiple of 16 bytes and "
              "holds a page (%lld)", what, static_cast<long long>(st_block));
    return false;
  }
  return true;
}
static bool q4_ts_ok(float a, float b, const char* what) {
  if (a > 0.f && b > 0.f && a <= 3.0e38f && b <= 3.0e38f) return true;
  set_error("%s: tensor scales must be positive and finite", what);
  return false;
}
// To quantise with, a tensor scale is a normal number too.
static bool q4_ts_normal(float a, float b, const char* what) {
  if (!q4_ts_ok(a, b, what)) return false;
  if (a >= 0x1p-126f && b >= 0x1p-126f) return true;
  set_error("%s: tensor scales below 2^-126 cannot be quantised with", what);
  return false;
}

}  // namespace hla

using namespace hla;

extern "C" {

int hla_s6_commit_rows_q4(const void* row, int64_t row_stride_t, int32_t width, const int64_t* positions,
                          const void* table, int64_t table_stride, int64_t max_position, void* cache,
                          int64_t num_blocks, int64_t cache_stride_block, int32_t page, const int32_t* block_table,
                          int64_t block_table_stride, int32_t max_blocks, const int32_t* query_start_loc,
                          int32_t num_reqs, int32_t num_tokens, float k_scale, float v_scale, int64_t* slot_out,
                          void* stream) {
  if (!q4_cache_ok(cache, cache_stride_block, width, page, "commit rows (4 bit)") ||
      !q4_ts_normal(k_scale, v_scale, "commit rows (4 bit)"))
    return kStatusInvalid;
  if (num_tokens < 0 || num_reqs < 1 || max_position < 1 || table_stride < width || max_blocks < 0 ||
      static_cast<int64_t>(max_blocks) * page >= (int64_t(1) << 31) || (table_stride % 8) ||
      (row_stride_t % 8) || (reinterpret_cast<uintptr_t>(row) % 16) || (reinterpret_cast<uintptr_t>(table) % 16)) {
    set_error("commit rows (4 bit) needs >= 1 request, a [max_position, width] table, a block table of fewer than 2^31 "
              "positions and 16-byte aligned row and table rows");
    return kStatusInvalid;
  }
  if (num_tokens == 0) return kStatusOk;
  Q4CommitArgs a;
  a.row = static_cast<const __nv_bfloat16*>(row);
  a.row_st = row_stride_t;
  a.positions = positions;
  a.table = static_cast<const __nv_bfloat16*>(table);
  a.tab_st = table_stride;
  a.max_pos = max_position;
  a.cache = static_cast<uint8_t*>(cache);
  a.c_sb = cache_stride_block;
  a.num_blocks = num_blocks;
  a.page = page;
  a.bt = block_table;
  a.bt_st = block_table_stride;
  a.max_blocks = max_blocks;
  a.qsl = query_start_loc;
  a.R = num_reqs;
  a.T = num_tokens;
  a.k_ts = k_scale;
  a.v_ts = v_scale;
  a.slot_out = slot_out;
  // Rounds from 12 CTAs without them per SM on, at each width (without and with them: 256 wide 9472 rows 6.7 and 7.0 us,
  // 18944 rows 10.3 and 9.0, 75776 37.1 and 29.4; 512 wide 4736 6.9 and 7.3, 9472 10.4 and 9.3, 37888 37.5 and 30.4; 1024
  // wide 4736 10.6 and 9.4, 37888 74 and 57).
  int rows = kQ4CommitThreads / (width / 16);
  a.rounds = num_tokens >= rows * 148 * 12 ? kQ4CommitRounds : 1;
  rows *= a.rounds;
  const int grid = (num_tokens + rows - 1) / rows;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (width == 256) q4_commit_kernel<256><<<grid, kQ4CommitThreads, 0, s>>>(a);
  else if (width == 512) q4_commit_kernel<512><<<grid, kQ4CommitThreads, 0, s>>>(a);
  else q4_commit_kernel<1024><<<grid, kQ4CommitThreads, 0, s>>>(a);
  return cuda_status(cudaGetLastError(), "q4_commit_kernel launch");
}

int hla_s6_gather_rows_q4(const void* cache, int64_t num_blocks, int64_t cache_stride_block, int32_t width,
                          int32_t page, const int32_t* blocks, const int64_t* slots, int64_t num_rows, float k_scale,
                          float v_scale, void* out, int64_t out_stride, int* error_flag, void* stream) {
  if (!q4_cache_ok(cache, cache_stride_block, width, page, "gather rows (4 bit)") ||
      !q4_ts_ok(k_scale, v_scale, "gather rows (4 bit)"))
    return kStatusInvalid;
  if (num_rows < 0 || num_rows >= (int64_t(1) << 31) || num_blocks < 0 || num_blocks * page >= (int64_t(1) << 31) ||
      (!blocks == !slots && num_rows > 0) || (out_stride % 8) || out_stride < 2 * width ||
      (reinterpret_cast<uintptr_t>(out) % 16)) {
    set_error("gather rows (4 bit) needs a block list or slots (one of them), fewer than 2^31 rows and 16-byte aligned "
              "output rows");
    return kStatusInvalid;
  }
  if (num_rows == 0) return kStatusOk;
  Q4GatherArgs a;
  a.cache = static_cast<const uint8_t*>(cache);
  a.c_sb = cache_stride_block;
  a.num_blocks = num_blocks;
  a.page = page;
  a.blocks = blocks;
  a.slots = slots;
  a.rows = num_rows;
  a.k_ts = k_scale;
  a.v_ts = v_scale;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.o_st = out_stride;
  a.err = error_flag;
  const int oct = num_rows >= kQ4GatherMany ? 4 : 1;
  const int64_t per = 256 / (width / (8 * oct)), want = (num_rows + per - 1) / per;
  const int grid = static_cast<int>(std::min<int64_t>(want, 148 * 64));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto few, auto many) { (oct == 1 ? few : many)<<<grid, 256, 0, s>>>(a); };
  if (width == 256) launch(q4_gather_kernel<256, 1>, q4_gather_kernel<256, 4>);
  else if (width == 512) launch(q4_gather_kernel<512, 1>, q4_gather_kernel<512, 4>);
  else launch(q4_gather_kernel<1024, 1>, q4_gather_kernel<1024, 4>);
  return cuda_status(cudaGetLastError(), "q4_gather_kernel launch");
}

int hla_s6_quantize_weight_q4(const void* weight, int64_t weight_stride_n, int32_t out_features, int32_t in_features,
                              float scale, void* packed, void* stream) {
  if (out_features < 1 || in_features < 32 || in_features % 32 || (weight_stride_n % 8) ||
      (reinterpret_cast<uintptr_t>(weight) % 16) || (reinterpret_cast<uintptr_t>(packed) % 16) || out_features > 16 * 65535) {
    set_error("quantize weight (4 bit) needs in_features %% 32 == 0, 1..1048560 out_features and 16-byte aligned rows");
    return kStatusInvalid;
  }
  if (!q4_ts_normal(scale, scale, "quantize weight (4 bit)")) return kStatusInvalid;
  q4_weight_kernel<<<dim3((in_features + 127) / 128, (out_features + 15) / 16), 256, 0,
                     static_cast<cudaStream_t>(stream)>>>(static_cast<const __nv_bfloat16*>(weight), weight_stride_n,
                                                          out_features, in_features, scale,
                                                          static_cast<uint8_t*>(packed));
  return cuda_status(cudaGetLastError(), "q4_weight_kernel launch");
}

}  // extern "C"
