// Microscaled 4-bit floating point: quantise and read back (stored layout), weights to and from the operand layout, rows to the
// operand layout.  All of them move bytes; the arithmetic is in mx_quant.cuh.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/tensorfold_b200.h"
#include "mx_layout.h"
#include "mx_quant.cuh"
#include "tf_ptx.cuh"

namespace tf {

int fail_moe(int code, const char* msg);
int cuda_fail_moe(cudaError_t e, const char* what);

namespace {

// Eight values of a stored type (0 bf16, 1 fp16, 2 fp32) as they lie in memory, and rounded.
template <int DTYPE>
struct Piece {
  uint4 p[DTYPE == 2 ? 2 : 1];
  __device__ __forceinline__ void load(const void* from, int64_t at) {
    const uint4* q = reinterpret_cast<const uint4*>(from) + at * (DTYPE == 2 ? 2 : 1);
    p[0] = q[0];
    if (DTYPE == 2) p[DTYPE == 2] = q[1];
  }
  __device__ __forceinline__ void clear() {
    p[0] = make_uint4(0u, 0u, 0u, 0u);
    if (DTYPE == 2) p[DTYPE == 2] = p[0];
  }
  __device__ __forceinline__ uint32_t quantize(uint32_t& scale) const {
    if constexpr (DTYPE == 0) {
      return quantize_block(p[0], scale);
    } else {
      float v[8];
      const uint32_t w[4] = {p[0].x, p[0].y, p[0].z, p[0].w};
      if constexpr (DTYPE == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
      } else {
        const uint32_t u[4] = {p[1].x, p[1].y, p[1].z, p[1].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]), v[4 + i] = __uint_as_float(u[i]);
      }
      return quantize_block(v, scale);
    }
  }
};

// Rows to stored words and scales.  A lane takes eight values, four lanes a block, so loads and stores of a warp are runs.  A thread
// block takes 256 U neighbouring pieces of a run (rows one after another are one run, others one each, by blockIdx.y), its threads
// U each, all in flight at once and at fixed distances: with 64-bit indexes made piece by piece a piece cost 96 instructions, more
// than its bytes.
template <int DTYPE, int U>
__global__ void __launch_bounds__(256, DTYPE == 2 ? 4 : 6) quantize_kernel(const void* __restrict__ x, int64_t ld_bytes, int rows, int64_t pieces,
                                                                           uint32_t* __restrict__ words, uint8_t* __restrict__ scales) {
  constexpr int BYTES = DTYPE == 2 ? 32 : 16;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (256 * U);
  const int64_t left = pieces - first;
  const int here = left < 256 * U ? static_cast<int>(left) : 256 * U;
  for (int row = blockIdx.y; row < rows; row += gridDim.y) {
    const char* from = static_cast<const char*>(x) + row * ld_bytes + (first + threadIdx.x) * BYTES;
    const int64_t to = row * pieces + first + threadIdx.x;
    uint32_t* w = words + to;
    uint8_t* sc = scales + (to >> 2);
    Piece<DTYPE> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {                              // (whole warps: a piece past the end is zeros and stores nothing)
      if (static_cast<int>(threadIdx.x) + 256 * u < here) v[u].load(from, 256 * u);
      else v[u].clear();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t scale;
      const uint32_t codes = v[u].quantize(scale);
      if (static_cast<int>(threadIdx.x) + 256 * u < here) {
        w[256 * u] = codes;
        if ((threadIdx.x & 3) == 0) sc[64 * u] = static_cast<uint8_t>(scale);
      }
    }
  }
}

// Stored words and scales to values, exact in bf16 and fp32 (2^127 times 2 and more overflows).  An e2m1 magnitude m, three
// bits, moved to the top of a fraction field reads as value * 2^-126 (two exponent bits and one of fraction, subnormals alike), so
// two products by powers of two make the value; in bf16 two values go at once.  Pieces as above.
template <int OUT, int U>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint32_t* __restrict__ words, const uint8_t* __restrict__ scales, int64_t pieces,
                                                         void* __restrict__ out) {
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (256 * U);
  const int64_t left = pieces - first;
  const int here = left < 256 * U ? static_cast<int>(left) : 256 * U;
  const int64_t at = first + threadIdx.x;
  words += at, scales += at >> 2;
  char* to = static_cast<char*>(out) + at * (OUT == 2 ? 32 : 16);
  uint32_t w[U], code[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool live = static_cast<int>(threadIdx.x) + 256 * u < here;
    w[u] = live ? words[256 * u] : 0u;
    code[u] = live ? scales[64 * u] : 0u;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (static_cast<int>(threadIdx.x) + 256 * u >= here) break;
    if (OUT == 0) {
      const uint32_t s1 = code[u] == 255u ? 0x7FC0u : code[u] == 0u ? 0x0040u : code[u] << 7, s2 = s1 | (s1 << 16), lift2 = 0x7E807E80u;
      const __nv_bfloat162 lift = *reinterpret_cast<const __nv_bfloat162*>(&lift2), scale = *reinterpret_cast<const __nv_bfloat162*>(&s2);
      uint32_t p[4];                                                 // values j and j + 4
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t q = w[u] >> (4 * j), bits = ((q & 0x00070007u) << 6) | ((q & 0x00080008u) << 12);
        const __nv_bfloat162 t = __hmul2(__hmul2(*reinterpret_cast<const __nv_bfloat162*>(&bits), lift), scale);
        p[j] = *reinterpret_cast<const uint32_t*>(&t);
      }
      reinterpret_cast<uint4*>(to)[256 * u] = make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410),
                                                         __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x7632));
    } else {
      const float scale = __uint_as_float(code[u] == 255u ? 0x7FC00000u : code[u] == 0u ? 0x00400000u : code[u] << 23);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t q = w[u] >> (4 * j);
        v[j] = __uint_as_float(((q & 7u) << 22) | ((q & 8u) << 28)) * 0x1p126f * scale;
      }
      if (OUT == 2) {
        float4* o = reinterpret_cast<float4*>(to) + 512 * u;
        o[0] = make_float4(v[0], v[1], v[2], v[3]), o[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2 t = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
          p[j] = *reinterpret_cast<const uint32_t*>(&t);
        }
        reinterpret_cast<uint4*>(to)[256 * u] = make_uint4(p[0], p[1], p[2], p[3]);
      }
    }
  }
}

// Stored weights to super-blocks and back.  A thread takes 16 bytes of codes (one block); eight neighbours write the 128 bytes of
// one swizzle line.  `up` interleaves a second projection in tiles of 16 rows.  Rows and inputs past the end become zeros.
__global__ void __launch_bounds__(256) pack_kernel(const uint4* __restrict__ words, const uint8_t* __restrict__ scales,
                                                   const uint4* __restrict__ up_words, const uint8_t* __restrict__ up_scales, int n, int blocks,
                                                   int steps, int64_t sb_bytes, uint8_t* __restrict__ tiled) {
  const int padded = 2 * steps, nsb = (n + MX_SB - 1) / MX_SB;
  const int64_t total = static_cast<int64_t>(nsb) * MX_SB * padded, step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t expert = blockIdx.y;
  const bool pair = up_words != nullptr;
  const int each = pair ? n / 2 : n;
  words += expert * each * blocks, scales += expert * each * blocks;
  if (pair) up_words += expert * each * blocks, up_scales += expert * each * blocks;
  tiled += expert * nsb * sb_bytes;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const int row = static_cast<int>(i / padded), b = static_cast<int>(i - static_cast<int64_t>(row) * padded);
    uint4 codes = make_uint4(0u, 0u, 0u, 0u);
    uint8_t scale = 0;
    if (row < n && b < blocks) {
      const bool second = pair && mx_pair_second(row);
      const int64_t at = static_cast<int64_t>(pair ? mx_pair_row(row) : row) * blocks + b;
      codes = (second ? up_words : words)[at];
      scale = (second ? up_scales : scales)[at];
    }
    uint8_t* sb = tiled + (row / MX_SB) * sb_bytes;
    *reinterpret_cast<uint4*>(sb + mx_code_offset(MX_SB, steps, row % MX_SB, b)) = codes;
    sb[mx_scale_offset(MX_SB, steps, row % MX_SB, b)] = scale;
    // a last stage with an odd number of steps has scales for one step more, which no MMA reads: they are left zero all the same
    if (b == padded - 1 && (steps & 1)) {
      sb[mx_scale_offset(MX_SB, steps, row % MX_SB, b) + 1] = 0;
      sb[mx_scale_offset(MX_SB, steps, row % MX_SB, b) + 2] = 0;
    }
  }
}

__global__ void __launch_bounds__(256) unpack_kernel(const uint8_t* __restrict__ tiled, int n, int blocks, int steps, int64_t sb_bytes,
                                                     uint4* __restrict__ words, uint8_t* __restrict__ scales) {
  const int64_t total = static_cast<int64_t>(n) * blocks, step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const int row = static_cast<int>(i / blocks), b = static_cast<int>(i - static_cast<int64_t>(row) * blocks);
    const uint8_t* sb = tiled + (row / MX_SB) * sb_bytes;
    words[i] = *reinterpret_cast<const uint4*>(sb + mx_code_offset(MX_SB, steps, row % MX_SB, b));
    scales[i] = sb[mx_scale_offset(MX_SB, steps, row % MX_SB, b)];
  }
}

// bf16 rows to the operand layout: operand y (blockIdx.y) holds `tile` rows, a warp (a row, as many runs of 1024 inputs as gridDim.z
// leaves it), four 16-byte loads in flight a lane.  With a plan, row r of item y is row members[first + r] / slots of x
// (members[first + r] itself with slots 0).
constexpr int ROWS_SEGMENT = 1024;
__global__ void __launch_bounds__(256) rows_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int m, int k, int steps, int rows, int tile,
                                                   int64_t item_bytes, const int* __restrict__ items, const int* __restrict__ counts,
                                                   const int* __restrict__ members, int slots, int pairs, uint8_t* __restrict__ out) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), y = blockIdx.y;
  int64_t src = static_cast<int64_t>(y) * tile + row;
  if (row >= tile) return;
  if (items != nullptr) {
    if (y >= counts[0] || row >= items[3 * y + 2]) return;
    const int pos = items[3 * y + 1] + row;
    if (pos < 0 || pos >= pairs) return;
    const int pair = members[pos];
    if (pair < 0 || pair >= pairs) return;
    src = slots > 0 ? pair / slots : pair;
  } else if (src >= m) {
    return;
  }
  out += y * item_bytes;
  const uint4* from = reinterpret_cast<const uint4*>(x + src * ldx);
  const int64_t stage_bytes = mx_stage_bytes(rows);
  const int full = steps >> 2, tail = steps & 3;
  uint8_t* const line = out + (row >> 3) * 1024 + (row & 7) * 128;                  // of stage 0
  uint8_t* const scale_line = out + rows * 128 + (row >> 7) * MX_SCALES + (row & 31) * 16 + ((row & 127) >> 5) * 4;
  for (int at = blockIdx.z * (ROWS_SEGMENT / 8); at < steps * 8; at += gridDim.z * (ROWS_SEGMENT / 8)) {
    uint4 p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int piece = at + 32 * j + lane;
      p[j] = piece * 8 < k ? from[piece] : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {                                                    // 32 pieces of a warp are a stage
      const int piece = at + 32 * j + lane, b = piece >> 2, u = (at >> 5) + j;
      uint32_t scale;
      const uint32_t codes = quantize_block(p[j], scale);
      if (u < full) {
        *reinterpret_cast<uint32_t*>(line + u * stage_bytes + (((b & 7) ^ (row & 7)) << 4) + 4 * (piece & 3)) = codes;
        if ((piece & 3) == 0) scale_line[u * stage_bytes + ((b & 7) >> 2) * 512 + (b & 3)] = static_cast<uint8_t>(scale);
      } else if (u == full && (b & 7) < 2 * tail) {              // K may end inside a step: its second block is zeros
        *reinterpret_cast<uint32_t*>(out + mx_code_offset(rows, steps, row, b) + 4 * (piece & 3)) = codes;
        if ((piece & 3) == 0) out[mx_scale_offset(rows, steps, row, b)] = static_cast<uint8_t>(scale);
      }
    }
  }
}

int blocks_for(int64_t threads) {
  const int64_t b = (threads + 255) / 256;
  return static_cast<int>(b < 1 ? 1 : b > 148 * 64 ? 148 * 64 : b);
}

// Pieces from which a thread takes four.  Measured, us from graphs, one / four: 256 x 5120 1.8 / 2.1 (back 1.8 / 2.1), 1024 x 5120 3.7 / 3.3
// (3.3 / 3.3), 2048 x 5120 5.9 / 4.7 (5.1 / 4.7), 17408 x 5120 48 / 34 (47 / 36).
constexpr int64_t MANY = 148 * 2048 * 4;

bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

}  // namespace

// The product's blocks, which take nearly all of an SM's shared memory, start while this kernel runs: an SM that has to change its split
// between cache and shared memory first would wait for this kernel's blocks to leave it.
cudaError_t mx_rows_configure() {
  return cudaFuncSetAttribute(rows_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
}

// Rows quantised into operands of `rows` rows, `tile` of them used, item_bytes apart: the first half of the products.  items null:
// the m rows in order.
cudaError_t mx_rows_launch(const void* x, int64_t ldx, int m, int k, int rows, int tile, int64_t item_bytes, const int* items, const int* counts,
                           const int* members, int slots, int pairs, int max_items, void* out, cudaStream_t stream) {
  const int steps = mx_steps(k), segments = (steps * MX_STEP + ROWS_SEGMENT - 1) / ROWS_SEGMENT;
  const int operands = items ? max_items : (m + tile - 1) / tile, used = items ? tile : std::min(m, tile);
  if (operands > 65535) return cudaErrorInvalidConfiguration;
  // Few rows: a warp a run, for latency, in blocks whose registers leave the product's block room beside them.  Many: two warps a row,
  // or one with a plan, where a warp starts with a chain of look-ups and blocks of short items have nothing to do.
  // Measured, us of the whole product from graphs: the first form / one warp a row: 48 rows by 6144 x 5120 9.3 / 12.4, 391 by 17408 x 5120
  // 28.7 / 35.5, 1000 by 6144 x 5120 24.9 / 31.8; the first form / two warps a row / one: 2048 by 17408 x 5120 87 / 82 / 84, by
  // 5120 x 17408 - / 104 / 121; routed layer, 2048 rows (12288 pairs), 246 / 242 / 237.
  const bool few = static_cast<int64_t>(operands) * used * segments <= 148 * 64;
  const int warps = few ? 4 : 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((used + warps - 1) / warps, operands, few ? segments : items ? 1 : std::min(segments, 2));
  cfg.blockDim = dim3(32 * warps);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, rows_kernel, static_cast<const __nv_bfloat16*>(x), ldx, m, k, steps, rows, tile, item_bytes, items,
                            counts, members, slots, pairs, static_cast<uint8_t*>(out));
}

}  // namespace tf

using namespace tf;

extern "C" {

int64_t tf_mx_tiled_bytes(int n, int k) {
  if (!mx_sizes(n, k)) return TF_ERR_ARG;
  return static_cast<int64_t>((n + MX_SB - 1) / MX_SB) * mx_operand_bytes(MX_SB, mx_steps(k));
}

int tf_mx_quantize(const void* x, int64_t ldx, int dtype, int rows, int k, void* words, void* scales, void* stream) {
  if (dtype < 0 || dtype > 2 || !mx_sizes(rows, k) || ldx < k || !x || !words || !scales)
    return fail_moe(TF_ERR_ARG, "tf_mx_quantize: rows of a positive multiple of 32 values, none null");
  if (misaligned(x, 16) || (rows > 1 && ldx % (dtype == 2 ? 4 : 8)) || misaligned(words, 4))
    return fail_moe(TF_ERR_ALIGN, "tf_mx_quantize: rows must start on 16-byte boundaries");
  const int64_t pieces = static_cast<int64_t>(rows) * (k / 8);
  const bool flat = rows == 1 || ldx == k;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t* w = static_cast<uint32_t*>(words);
  uint8_t* s = static_cast<uint8_t*>(scales);
  const int64_t run = flat ? pieces : k / 8, total = pieces;
  const int64_t ld = ldx * (dtype == 2 ? 4 : 2);
  if (total / 256 > INT32_MAX) return fail_moe(TF_ERR_ARG, "tf_mx_quantize: too many values");
#define TF_MX_QUANTIZE(DT)                                                                                                       \
  if (dtype == DT) {                                                                                                             \
    const dim3 grid(static_cast<unsigned>((run + (total < MANY ? 255 : 1023)) / (total < MANY ? 256 : 1024)), flat ? 1 : std::min(rows, 65535)); \
    if (total < MANY) quantize_kernel<DT, 1><<<grid, 256, 0, st>>>(x, ld, flat ? 1 : rows, run, w, s);                            \
    else quantize_kernel<DT, 4><<<grid, 256, 0, st>>>(x, ld, flat ? 1 : rows, run, w, s);                                         \
  }
  TF_MX_QUANTIZE(0) TF_MX_QUANTIZE(1) TF_MX_QUANTIZE(2)
#undef TF_MX_QUANTIZE
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TF_OK : cuda_fail_moe(e, "tf_mx_quantize");
}

int tf_mx_dequantize(const void* words, const void* scales, int rows, int k, int out_type, void* out, void* stream) {
  if (out_type < 0 || out_type > 2 || !mx_sizes(rows, k) || !words || !scales || !out)
    return fail_moe(TF_ERR_ARG, "tf_mx_dequantize: rows of a positive multiple of 32 values, none null");
  if (misaligned(words, 4) || misaligned(out, 16)) return fail_moe(TF_ERR_ALIGN, "tf_mx_dequantize: out must start on a 16-byte boundary");
  const int64_t pieces = static_cast<int64_t>(rows) * (k / 8);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint32_t* w = static_cast<const uint32_t*>(words);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  if (pieces / 256 > INT32_MAX) return fail_moe(TF_ERR_ARG, "tf_mx_dequantize: too many values");
#define TF_MX_DEQUANTIZE(OUT)                                                                                                  \
  if (out_type == OUT) {                                                                                                       \
    if (pieces < MANY) dequantize_kernel<OUT, 1><<<static_cast<unsigned>((pieces + 255) / 256), 256, 0, st>>>(w, s, pieces, out); \
    else dequantize_kernel<OUT, 4><<<static_cast<unsigned>((pieces + 1023) / 1024), 256, 0, st>>>(w, s, pieces, out);            \
  }
  TF_MX_DEQUANTIZE(0) TF_MX_DEQUANTIZE(1) TF_MX_DEQUANTIZE(2)
#undef TF_MX_DEQUANTIZE
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TF_OK : cuda_fail_moe(e, "tf_mx_dequantize");
}

int tf_mx_pack(const void* words, const void* scales, const void* up_words, const void* up_scales, int experts, int n, int k, void* tiled,
               void* stream) {
  const bool pair = up_words != nullptr;
  if (experts < 1 || experts > 65535 || !mx_sizes(n, k) || !words || !scales || !tiled || pair != (up_scales != nullptr))
    return fail_moe(TF_ERR_ARG, "tf_mx_pack: rows of a positive multiple of 32 values, none null");
  if (pair && n % 32) return fail_moe(TF_ERR_ARG, "tf_mx_pack: a pair interleaves whole tiles of 16 rows");
  if (misaligned(words, 16) || misaligned(up_words, 16) || misaligned(tiled, 16))
    return fail_moe(TF_ERR_ALIGN, "tf_mx_pack: words and units must start on 16-byte boundaries");
  const int steps = mx_steps(k);
  const int64_t total = static_cast<int64_t>((n + MX_SB - 1) / MX_SB) * MX_SB * 2 * steps;
  const dim3 grid(blocks_for(total), experts);
  pack_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint4*>(words), static_cast<const uint8_t*>(scales), static_cast<const uint4*>(up_words),
      static_cast<const uint8_t*>(up_scales), n, k / MX_BLOCK, steps, mx_operand_bytes(MX_SB, steps), static_cast<uint8_t*>(tiled));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TF_OK : cuda_fail_moe(e, "tf_mx_pack");
}

int tf_mx_unpack(const void* tiled, int n, int k, void* words, void* scales, void* stream) {
  if (!mx_sizes(n, k) || !words || !scales || !tiled) return fail_moe(TF_ERR_ARG, "tf_mx_unpack: bad shape or null pointer");
  if (misaligned(words, 16) || misaligned(tiled, 16))
    return fail_moe(TF_ERR_ALIGN, "tf_mx_unpack: words and units must start on 16-byte boundaries");
  const int steps = mx_steps(k);
  unpack_kernel<<<blocks_for(static_cast<int64_t>(n) * (k / MX_BLOCK)), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(tiled), n, k / MX_BLOCK, steps, mx_operand_bytes(MX_SB, steps), static_cast<uint4*>(words),
      static_cast<uint8_t*>(scales));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TF_OK : cuda_fail_moe(e, "tf_mx_unpack");
}

}  // extern "C"
