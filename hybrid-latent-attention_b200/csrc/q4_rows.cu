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
// (the same in the 4 lanes).
__device__ __forceinline__ uint32_t quantize8(const float (&f)[8], float ts, uint32_t& scale) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(f[i]));
  a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
  a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
  scale = q4_scale_byte(a, ts);
  const float step = q4_scale_value(scale) * ts;
  uint32_t n[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = q4_code(f[i], step);
  return q4_word(n);
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
};

// W / 16 threads per row; thread k holds columns 8k .. and W/2 + 8k .. of both halves, i.e. whole RoPE
// pairs and quarters of groups, so the amax of a group is two shuffles.
constexpr int kQ4CommitThreads = 128;
template <int W>
__global__ void __launch_bounds__(kQ4CommitThreads) q4_commit_kernel(const Q4CommitArgs a) {
  constexpr int PER = W / 16;
  __shared__ int32_t qsl_s[kQslCap];
  const int32_t* qsl = stage_qsl(a.qsl, a.R, qsl_s);
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kQ4CommitThreads / PER) + threadIdx.x / PER;
  const int k = threadIdx.x % PER;
  const bool in = t < a.T;
  int64_t slot = -1;
  int64_t pos = 0;
  if (in) {
    pos = a.positions[t];
    slot = token_slot(qsl, a.R, static_cast<int>(t), pos, a.bt, a.bt_st, a.max_blocks, a.page, a.num_blocks);
    if (a.slot_out && k == 0) a.slot_out[t] = slot;
  }
  const bool live = slot >= 0;
  uint4 raw[6] = {};
  if (live) {
    const __nv_bfloat16* src = a.row + t * a.row_st + 8 * k;
    const __nv_bfloat16* tab = a.table + clamp_pos(pos, a.max_pos) * a.tab_st + 8 * k;
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(src + i * (W / 2)));
    raw[4] = __ldg(reinterpret_cast<const uint4*>(tab));
    raw[5] = __ldg(reinterpret_cast<const uint4*>(tab + W / 2));
  }
  float x[4][8], c[8], s[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack8(raw[i], x[i]);
  unpack8(raw[4], c);
  unpack8(raw[5], s);
#pragma unroll
  for (int i = 0; i < 8; ++i) rope_pair_torch(x[0][i], x[1][i], c[i], s[i], x[0][i], x[1][i]);
  const Q4Tile tl(W);
  uint8_t* tile = nullptr;
  int r = 0;
  if (live) {
    const int64_t blk = slot / a.page;
    const int off = static_cast<int>(slot - blk * a.page);
    tile = a.cache + blk * a.c_sb + static_cast<int64_t>(off / 16) * tl.bytes();
    r = off % 16;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t sb;
    const uint32_t w = quantize8(x[i], i < 2 ? a.k_ts : a.v_ts, sb);  // warp-collective: every lane
    if (!live) continue;
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

// The 8 values of a word, times scale s (a float) and the tensor scale, in bf16.
__device__ __forceinline__ uint4 q4_values(uint32_t w, uint32_t scale, float ts) {
  const float s = q4_scale_value(scale);
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (static_cast<float>(q4_code_at(w, i)) * s) * ts;
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

template <int W>
__global__ void __launch_bounds__(128) q4_gather_kernel(const Q4GatherArgs a) {
  constexpr int PER = W / 4;  // octets of a row, K and V
  const Q4Tile tl(W);
  for (int64_t idx = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; idx < a.rows * PER;
       idx += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t i = idx / PER;
    const int oc = static_cast<int>(idx % PER);
    int64_t blk, off;
    if (a.slots) {
      const int64_t s = a.slots[i];
      blk = s < 0 ? -1 : s / a.page;
      off = s < 0 ? 0 : s % a.page;
    } else {
      blk = a.blocks[i / a.page];
      off = i % a.page;
    }
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (blk >= 0 && blk < a.num_blocks) {
      const uint8_t* tile = a.cache + blk * a.c_sb + (off / 16) * tl.bytes();
      const int r = static_cast<int>(off % 16);
      const int octet = oc < W / 8 ? oc : oc - W / 8, group = octet / 4;
      if (oc < W / 8)
        v = q4_values(__ldg(reinterpret_cast<const uint32_t*>(tile + tl.k_codes(group, r) + 4 * (octet & 3))),
                      __ldg(tile + tl.k_scale(r, group)), a.k_ts);
      else
        v = q4_values(__ldg(reinterpret_cast<const uint32_t*>(tile + tl.v_codes(octet, r))),
                      __ldg(tile + tl.v_scale(group, r)), a.v_ts);
    } else if (oc == 0 && !(a.slots && blk < 0)) {
      record_error(a.err, kErrBlock);
    }
    *reinterpret_cast<uint4*>(a.out + i * a.o_st + 8 * oc) = v;
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
      !q4_ts_ok(k_scale, v_scale, "commit rows (4 bit)"))
    return kStatusInvalid;
  if (num_tokens < 0 || num_reqs < 1 || max_position < 1 || table_stride < width || (table_stride % 8) ||
      (row_stride_t % 8) || (reinterpret_cast<uintptr_t>(row) % 16) || (reinterpret_cast<uintptr_t>(table) % 16)) {
    set_error("commit rows (4 bit) needs >= 1 request, a [max_position, width] table and 16-byte aligned row and "
              "table rows");
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
  const int rows = kQ4CommitThreads / (width / 16), grid = (num_tokens + rows - 1) / rows;
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
  if (num_rows < 0 || (!blocks == !slots && num_rows > 0) || (out_stride % 8) || out_stride < 2 * width ||
      (reinterpret_cast<uintptr_t>(out) % 16)) {
    set_error("gather rows (4 bit) needs a block list or slots (one of them) and 16-byte aligned output rows");
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
  const int64_t want = (num_rows * (width / 4) + 127) / 128;
  const int grid = static_cast<int>(std::min<int64_t>(want, 148 * 64));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (width == 256) q4_gather_kernel<256><<<grid, 128, 0, s>>>(a);
  else if (width == 512) q4_gather_kernel<512><<<grid, 128, 0, s>>>(a);
  else q4_gather_kernel<1024><<<grid, 128, 0, s>>>(a);
  return cuda_status(cudaGetLastError(), "q4_gather_kernel launch");
}

int hla_s6_quantize_weight_q4(const void* weight, int64_t weight_stride_n, int32_t out_features, int32_t in_features,
                              float scale, void* packed, void* stream) {
  if (out_features < 1 || in_features < 32 || in_features % 32 || (weight_stride_n % 8) ||
      (reinterpret_cast<uintptr_t>(weight) % 16) || (reinterpret_cast<uintptr_t>(packed) % 16) || out_features > 16 * 65535) {
    set_error("quantize weight (4 bit) needs in_features %% 32 == 0, 1..1048560 out_features and 16-byte aligned rows");
    return kStatusInvalid;
  }
  if (!q4_ts_ok(scale, scale, "quantize weight (4 bit)")) return kStatusInvalid;
  q4_weight_kernel<<<dim3((in_features + 127) / 128, (out_features + 15) / 16), 256, 0,
                     static_cast<cudaStream_t>(stream)>>>(static_cast<const __nv_bfloat16*>(weight), weight_stride_n,
                                                          out_features, in_features, scale,
                                                          static_cast<uint8_t*>(packed));
  return cuda_status(cudaGetLastError(), "q4_weight_kernel launch");
}

}  // extern "C"
