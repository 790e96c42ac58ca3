// Linears whose weights stay in 4 bits with one fp16 scale (and, optionally, minimum) per row and group of columns:
//   w[n, k] = s[n, k / G] * (c[n, k] - 8)      or      s[n, k / G] * c[n, k] + m[n, k / G],     c in 0..15
// A weight is laid out once for its kernels, in tiles of 16 rows x 64 columns of 512 bytes: lane l = 4 g + t of a warp owns
// the 16 bytes at l * 16, four words j of eight codes.  Word j holds, for rows g and g + 8, the four columns from
// 32 (j / 2) + 8 t + 4 (j % 2) on; nibble i of a word's low half and of its high half are
//   i = 0: row g, columns 0, 1    1: row g + 8, columns 0, 1    2: row g, columns 2, 3    3: row g + 8, columns 2, 3
// so (word >> 4 i) & 0x000f000f is a pair of neighbouring columns of one row.  Scales (and minima) lie in the order in which
// the lanes of a tile want them: [row block][64 columns][g][group of the tile][row g, row g + 8] for groups of 32, one group
// per tile for 64, and one entry per two tiles for 128.  Rows and columns that pad the last tiles have scale 0.
#include <cuda_fp16.h>

#include "common.cuh"
#include "dsb.h"

namespace dsb {

struct Int4Dims {
  int N, K, group;    // weight rows, columns, columns per group (32, 64 or 128)
  int row_blocks, k_tiles;
  int per_tile;       // groups that begin in a tile: 2 (of 32), else 1
  int tile_shift;     // 1 when a group spans two tiles
  int scale_tiles;    // tiles of scales per row block
};

static bool int4_dims(Int4Dims* d, int N, int K, int group) {
  if (N <= 0 || K <= 0 || (K & 1) || (group != 32 && group != 64 && group != 128)) return false;
  d->N = N;
  d->K = K;
  d->group = group;
  d->row_blocks = (N - 1) / 16 + 1;
  d->k_tiles = (K - 1) / 64 + 1;
  d->per_tile = group == 32 ? 2 : 1;
  d->tile_shift = group == 128 ? 1 : 0;
  d->scale_tiles = (d->k_tiles + d->tile_shift) >> d->tile_shift;
  return true;
}

// index of the scale of `row` of a row block and of the group that column `k` is in
__device__ __forceinline__ int64_t scale_index(const Int4Dims& d, int64_t row_block, int row, int k) {
  const int64_t tile = row_block * d.scale_tiles + (k >> (6 + d.tile_shift));
  const int half = d.per_tile == 2 ? (k >> 5) & 1 : 0;
  return ((tile * 8 + (row & 7)) * d.per_tile + half) * 2 + (row >> 3);
}

// ---------------------------------------------------------------------- layout
// One thread per word of the payload.
__global__ void __launch_bounds__(256) int4_pack_kernel(const uint8_t* __restrict__ codes, int64_t ld, Int4Dims d,
                                                        uint32_t* __restrict__ payload) {
  grid_wait();
  const int64_t total = static_cast<int64_t>(d.row_blocks) * d.k_tiles * 128;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t tile = i >> 7;
    const int lane = (i >> 2) & 31, j = i & 3, g = lane >> 2, t = lane & 3;
    const int64_t rb = tile / d.k_tiles;
    const int k = static_cast<int>(tile - rb * d.k_tiles) * 64 + 32 * (j >> 1) + 8 * t + 4 * (j & 1);
    uint32_t w = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t row = rb * 16 + g + 8 * r;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t q = 8;
        if (row < d.N && k + c < d.K) q = (codes[row * ld + ((k + c) >> 1)] >> (4 * (c & 1))) & 15u;
        const int nibble = r + 2 * (c >> 1) + 4 * (c & 1);
        w |= q << (4 * nibble);
      }
    }
    payload[i] = w;
  }
}

// One thread per packed scale.
__global__ void __launch_bounds__(256) int4_pack_scales_kernel(const __half* __restrict__ scales, const __half* __restrict__ mins,
                                                               int64_t ld, Int4Dims d, __half* __restrict__ out_s,
                                                               __half* __restrict__ out_m) {
  grid_wait();
  const int per_block = d.scale_tiles * 8 * d.per_tile * 2;
  const int64_t total = static_cast<int64_t>(d.row_blocks) * per_block;
  const int groups = (d.K - 1) / d.group + 1;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t rb = i / per_block;
    int rest = static_cast<int>(i - rb * per_block);
    const int hi = rest & 1;
    rest >>= 1;
    const int half = rest % d.per_tile;
    rest /= d.per_tile;
    const int64_t row = rb * 16 + (rest & 7) + 8 * hi;
    const int grp = (rest >> 3) * d.per_tile + half;
    const bool in = row < d.N && grp < groups;
    out_s[i] = in ? scales[row * ld + grp] : __ushort_as_half(0);
    if (out_m) out_m[i] = in ? mins[row * ld + grp] : __ushort_as_half(0);
  }
}

// ------------------------------------------------------------------ quantisation
// One warp per (row, group).  Without minima s = amax / 7 and c = clamp(rint(w / s), -8, 7) + 8; with them s = (max - min) /
// 15, m = min and c = clamp(rint((w - m) / s), 0, 15).  s and m are rounded to fp16 first (they saturate at its largest
// value), so the codes are the best ones for the values that will multiply them.
template <bool BF16>
__global__ void __launch_bounds__(256) int4_quantize_kernel(const void* __restrict__ W, int64_t ld_w, Int4Dims d, int has_min,
                                                            uint8_t* __restrict__ codes, int64_t ld_c,
                                                            __half* __restrict__ scales, __half* __restrict__ mins) {
  grid_wait();
  const int groups = (d.K - 1) / d.group + 1, lane = threadIdx.x & 31;
  const int64_t total = static_cast<int64_t>(d.N) * groups;
  for (int64_t i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < total; i += gridDim.x * 8ll) {
    const int64_t row = i / groups;
    const int grp = static_cast<int>(i - row * groups);
    const int k_end = min(d.K, (grp + 1) * d.group);
    auto at = [&](int k) {
      if constexpr (BF16)
        return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(W)[row * ld_w + k]);
      else
        return reinterpret_cast<const float*>(W)[row * ld_w + k];
    };
    float lo = INFINITY, hi = -INFINITY;
    for (int k = grp * d.group + lane; k < k_end; k += 32) {
      const float w = at(k);
      lo = fminf(lo, w);
      hi = fmaxf(hi, w);
    }
    hi = warp_max(hi);
    lo = -warp_max(-lo);
    const float s32 = has_min ? __fdiv_rn(hi - lo, 15.f) : __fdiv_rn(fmaxf(fabsf(hi), fabsf(lo)), 7.f);
    const __half s = __float2half_rn(fminf(s32, 65504.f));
    const __half m = __float2half_rn(fminf(fmaxf(has_min ? lo : 0.f, -65504.f), 65504.f));
    if (lane == 0) {
      scales[i] = s;
      if (has_min) mins[i] = m;
    }
    const float sf = __half2float(s), mf = __half2float(m);
    // two neighbouring columns per lane: they share a byte (K and the group are even)
    for (int k = grp * d.group + 2 * lane; k < k_end; k += 64) {
      uint32_t q[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float u = sf > 0.f ? rintf(__fdiv_rn(at(k + e) - mf, sf)) : 0.f;
        q[e] = static_cast<uint32_t>(has_min ? static_cast<int>(fminf(fmaxf(u, 0.f), 15.f))
                                             : static_cast<int>(fminf(fmaxf(u, -8.f), 7.f)) + 8);
      }
      codes[row * ld_c + (k >> 1)] = static_cast<uint8_t>(q[0] | (q[1] << 4));
    }
  }
}

// ------------------------------------------------------------------ GGUF blocks
// Q4_0, Q4_1 (blocks of 32) and Q4_K (super-blocks of 256 with eight 6-bit scales and minima) as codes, scales and minima.
// The codes are taken over as they are.  Q4_0 and Q4_1 carry fp16 scales and minima themselves; those of Q4_K are products
// d * sc and -dmin * mn of 11 and 6 bits, rounded here to fp16 (at most 2^-11 of the value; the block's own quantisation
// step is 2^-4 of its range).  One thread per 32 weights.
__global__ void __launch_bounds__(256) int4_from_gguf_kernel(int qtype, const uint8_t* __restrict__ raw, int64_t row_bytes, int N,
                                                             int K, uint8_t* __restrict__ codes, int64_t ld_c,
                                                             __half* __restrict__ scales, __half* __restrict__ mins) {
  grid_wait();
  const int groups = K / 32;
  const int64_t total = static_cast<int64_t>(N) * groups;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t row = i / groups;
    const int grp = static_cast<int>(i - row * groups);
    const uint8_t* r = raw + row * row_bytes;
    uint8_t* out = codes + row * ld_c + grp * 16;
    const uint8_t* qs;
    if (qtype == 12) {  // Q4_K
      const uint8_t* blk = r + static_cast<int64_t>(grp >> 3) * 144;
      const uint8_t* s12 = blk + 4;
      const int j = grp & 7;
      const uint32_t sc = j < 4 ? s12[j] & 63u : (s12[j + 4] & 15u) | ((s12[j - 4] >> 6) << 4);
      const uint32_t mn = j < 4 ? s12[j + 4] & 63u : (s12[j + 4] >> 4) | ((s12[j] >> 6) << 4);
      const float d = __half2float(__ushort_as_half(blk[0] | (blk[1] << 8)));
      const float dmin = __half2float(__ushort_as_half(blk[2] | (blk[3] << 8)));
      scales[i] = __float2half_rn(d * static_cast<float>(sc));
      mins[i] = __float2half_rn(-(dmin * static_cast<float>(mn)));
      qs = blk + 16 + (j >> 1) * 32;  // 32 bytes hold group 2 i in their low nibbles and 2 i + 1 in the high ones
      const int sh = (j & 1) * 4;
      for (int b = 0; b < 16; ++b)
        out[b] = static_cast<uint8_t>(((qs[2 * b] >> sh) & 15) | (((qs[2 * b + 1] >> sh) & 15) << 4));
    } else {            // Q4_0 (2), Q4_1 (3): values 0..15 in the low nibbles, 16..31 in the high ones
      const uint8_t* blk = r + static_cast<int64_t>(grp) * (qtype == 2 ? 18 : 20);
      scales[i] = __ushort_as_half(static_cast<unsigned short>(blk[0] | (blk[1] << 8)));
      if (qtype == 3) mins[i] = __ushort_as_half(static_cast<unsigned short>(blk[2] | (blk[3] << 8)));
      qs = blk + (qtype == 2 ? 2 : 4);
      for (int b = 0; b < 8; ++b) {
        out[b] = static_cast<uint8_t>((qs[2 * b] & 15) | ((qs[2 * b + 1] & 15) << 4));
        out[8 + b] = static_cast<uint8_t>((qs[2 * b] >> 4) | (qs[2 * b + 1] & 0xf0));
      }
    }
  }
}

// ------------------------------------------------------------------ dequantisation
// One thread per word of the payload: two rows, four columns each; the value in fp32, rounded once to bf16.
__global__ void __launch_bounds__(256) int4_dequant_kernel(const uint32_t* __restrict__ payload, const __half* __restrict__ scales,
                                                           const __half* __restrict__ mins, Int4Dims d,
                                                           __nv_bfloat16* __restrict__ out, int64_t ld) {
  grid_wait();
  const int64_t total = static_cast<int64_t>(d.row_blocks) * d.k_tiles * 128;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t tile = i >> 7;
    const int lane = (i >> 2) & 31, j = i & 3, g = lane >> 2, t = lane & 3;
    const int64_t rb = tile / d.k_tiles;
    const int k = static_cast<int>(tile - rb * d.k_tiles) * 64 + 32 * (j >> 1) + 8 * t + 4 * (j & 1);
    const uint32_t w = payload[i];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t row = rb * 16 + g + 8 * r;
      if (row >= d.N || k >= d.K) continue;
      const int64_t si = scale_index(d, rb, g + 8 * r, k);
      const float s = __half2float(scales[si]), m = mins ? __half2float(mins[si]) : 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (k + c >= d.K) break;
        const float q = static_cast<float>((w >> (4 * (r + 2 * (c >> 1) + 4 * (c & 1)))) & 15u);
        out[row * ld + k + c] = __float2bfloat16_rn(mins ? __fadd_rn(__fmul_rn(s, q), m) : s * (q - 8.f));
      }
    }
  }
}

// ------------------------------------------------------------------------ product
struct GemvInt4 {
  const uint4* payload;
  const __half* scales;
  const __half* mins;
  const void* x;
  int64_t ld_x;
  const float* bias;
  void* y;
  int64_t ld_y;
  int M, x_bf16, y_bf16, act_in, act_out, accumulate;
};

__device__ __forceinline__ float act_apply(float v, int act) {
  switch (act) {
    case DSB_ACT_GELU_TANH: return gelu_tanh(v);
    case DSB_ACT_SILU: return silu(v);
    case DSB_ACT_GELU: return gelu_erf(v);
    default: return v;
  }
}

// One warp per row block and activation row, fp32 products.
__global__ void __launch_bounds__(256) gemv_int4_kernel(Int4Dims d, GemvInt4 p) {
  grid_wait();
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, m = blockIdx.y;
  const float* xf = reinterpret_cast<const float*>(p.x) + m * p.ld_x;
  const __nv_bfloat16* xb = reinterpret_cast<const __nv_bfloat16*>(p.x) + m * p.ld_x;
  for (int rb = blockIdx.x * 8 + (threadIdx.x >> 5); rb < d.row_blocks; rb += gridDim.x * 8) {
    float acc[2] = {0.f, 0.f};
    for (int kt = 0; kt < d.k_tiles; ++kt) {
      const uint4 q = p.payload[(static_cast<int64_t>(rb) * d.k_tiles + kt) * 32 + lane];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = kt * 64 + 32 * (j >> 1) + 8 * t + 4 * (j & 1);
        float x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x[c] = 0.f;
          if (k + c < d.K) x[c] = p.x_bf16 ? __bfloat162float(xb[k + c]) : xf[k + c];
          if (p.act_in == DSB_ACT_SILU) x[c] = silu(x[c]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int64_t si = scale_index(d, rb, g + 8 * r, k);
          const float s = __half2float(p.scales[si]);
          float a = 0.f, sum = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            a += (static_cast<float>((w[j] >> (4 * (r + 2 * (c >> 1) + 4 * (c & 1)))) & 15u) - 8.f) * x[c];
            sum += x[c];
          }
          acc[r] += s * a;
          if (p.mins) acc[r] += (__half2float(p.mins[si]) + 8.f * s) * sum;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], 1);
      acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], 2);
      const int n = rb * 16 + g + 8 * r;
      if (t == 0 && n < d.N) {
        float v = act_apply(acc[r] + (p.bias ? p.bias[n] : 0.f), p.act_out);
        if (p.y_bf16) {
          __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(p.y) + m * p.ld_y + n;
          *y = __float2bfloat16_rn(p.accumulate ? v + __bfloat162float(*y) : v);
        } else {
          float* y = reinterpret_cast<float*>(p.y) + m * p.ld_y + n;
          *y = p.accumulate ? v + *y : v;
        }
      }
    }
  }
}

}  // namespace dsb

using namespace dsb;

static bool al(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
// CTAs of a grid-stride kernel: what the work needs, at most eight per SM
static unsigned stride_grid(int64_t blocks) {
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  return static_cast<unsigned>(blocks < cap ? blocks : cap);
}

extern "C" int dsb_int4_quantize(const void* W, int64_t ld_w, int w_bf16, int N, int K, int group, uint8_t* codes, int64_t ld_codes,
                                 void* scales, void* mins, void* stream) {
  Int4Dims d;
  if (!W || !codes || !scales || !int4_dims(&d, N, K, group) || ld_w < K || ld_codes < K / 2) return DSB_ERR_ARG;
  if (!al(W, w_bf16 ? 2 : 4) || !al(scales, 2) || !al(mins, 2)) return DSB_ERR_ARG;
  const int64_t warps = static_cast<int64_t>(N) * ((K - 1) / group + 1);
  const cudaError_t err =
      launch_kernel(w_bf16 ? int4_quantize_kernel<true> : int4_quantize_kernel<false>, stride_grid((warps + 7) / 8), 256, 0,
                    reinterpret_cast<cudaStream_t>(stream), W, ld_w, d, mins ? 1 : 0, codes, ld_codes,
                    reinterpret_cast<__half*>(scales), reinterpret_cast<__half*>(mins));
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

extern "C" int dsb_int4_from_gguf(int qtype, const uint8_t* raw, int64_t row_bytes, int N, int K, uint8_t* codes, int64_t ld_codes,
                                  void* scales, void* mins, void* stream) {
  if (!raw || !codes || !scales || N <= 0 || K <= 0 || ld_codes < K / 2 || !al(scales, 2) || !al(mins, 2)) return DSB_ERR_ARG;
  int block, bytes;
  switch (qtype) {
    case 2: block = 32, bytes = 18; break;
    case 3: block = 32, bytes = 20; break;
    case 12: block = 256, bytes = 144; break;
    default: return DSB_ERR_UNSUPPORTED;
  }
  if ((K % block) || row_bytes < static_cast<int64_t>(K / block) * bytes || (qtype == 2) != (mins == nullptr)) return DSB_ERR_ARG;
  const int64_t threads = static_cast<int64_t>(N) * (K / 32);
  const cudaError_t err = launch_kernel(int4_from_gguf_kernel, stride_grid((threads + 255) / 256), 256, 0,
                                        reinterpret_cast<cudaStream_t>(stream), qtype, raw, row_bytes, N, K, codes, ld_codes,
                                        reinterpret_cast<__half*>(scales), reinterpret_cast<__half*>(mins));
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

extern "C" int dsb_int4_pack(const uint8_t* codes, int64_t ld_codes, const void* scales, const void* mins, int64_t ld_scales, int N,
                             int K, int group, void* payload, void* out_scales, void* out_mins, void* stream) {
  Int4Dims d;
  if (!codes || !scales || !payload || !out_scales || (mins == nullptr) != (out_mins == nullptr) ||
      !int4_dims(&d, N, K, group) || ld_codes < K / 2 || ld_scales < (K - 1) / group + 1 || !al(payload, 16) ||
      !al(out_scales, 8) || !al(out_mins, 8) || !al(scales, 2) || !al(mins, 2))
    return DSB_ERR_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t words = static_cast<int64_t>(d.row_blocks) * d.k_tiles * 128;
  const int64_t halves = static_cast<int64_t>(d.row_blocks) * d.scale_tiles * 16 * d.per_tile;
  if (launch_kernel(int4_pack_kernel, stride_grid((words + 255) / 256), 256, 0, st, codes, ld_codes, d,
                    reinterpret_cast<uint32_t*>(payload)) != cudaSuccess)
    return DSB_ERR_CUDA;
  const cudaError_t err = launch_kernel(int4_pack_scales_kernel, stride_grid((halves + 255) / 256), 256, 0, st,
                                        reinterpret_cast<const __half*>(scales), reinterpret_cast<const __half*>(mins), ld_scales, d,
                                        reinterpret_cast<__half*>(out_scales), reinterpret_cast<__half*>(out_mins));
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

extern "C" int dsb_int4_dequant(const void* payload, const void* scales, const void* mins, int N, int K, int group, void* out,
                                int64_t ld_out, void* stream) {
  Int4Dims d;
  if (!payload || !scales || !out || !int4_dims(&d, N, K, group) || ld_out < K || !al(payload, 16) || !al(scales, 8) ||
      !al(mins, 8) || !al(out, 2))
    return DSB_ERR_ARG;
  const int64_t words = static_cast<int64_t>(d.row_blocks) * d.k_tiles * 128;
  const cudaError_t err =
      launch_kernel(int4_dequant_kernel, stride_grid((words + 255) / 256), 256, 0, reinterpret_cast<cudaStream_t>(stream),
                    reinterpret_cast<const uint32_t*>(payload), reinterpret_cast<const __half*>(scales),
                    reinterpret_cast<const __half*>(mins), d, reinterpret_cast<__nv_bfloat16*>(out), ld_out);
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

extern "C" int dsb_gemv_int4(const void* payload, const void* scales, const void* mins, int N, int K, int group, const void* x,
                             int64_t ld_x, int x_bf16, const float* bias, void* y, int64_t ld_y, int y_bf16, int M, int act_in,
                             int act_out, int accumulate, void* stream) {
  Int4Dims d;
  if (M < 0 || M > DSB_INT4_MAX_ROWS || !int4_dims(&d, N, K, group)) return DSB_ERR_ARG;
  if (act_in != DSB_ACT_NONE && act_in != DSB_ACT_SILU) return DSB_ERR_ARG;
  if (act_out < DSB_ACT_NONE || act_out > DSB_ACT_GELU) return DSB_ERR_ARG;
  if (M == 0) return DSB_OK;
  if (!payload || !scales || !x || !y || !al(payload, 16) || !al(scales, 8) || !al(mins, 8) || !al(x, x_bf16 ? 2 : 4) ||
      !al(y, y_bf16 ? 2 : 4) || !al(bias, 4) || (M > 1 && (ld_x < K || ld_y < N)))
    return DSB_ERR_ARG;
  GemvInt4 p = {};
  p.payload = reinterpret_cast<const uint4*>(payload);
  p.scales = reinterpret_cast<const __half*>(scales);
  p.mins = reinterpret_cast<const __half*>(mins);
  p.x = x;
  p.ld_x = ld_x;
  p.bias = bias;
  p.y = y;
  p.ld_y = ld_y;
  p.M = M;
  p.x_bf16 = x_bf16 ? 1 : 0;
  p.y_bf16 = y_bf16 ? 1 : 0;
  p.act_in = act_in;
  p.act_out = act_out;
  p.accumulate = accumulate ? 1 : 0;
  const cudaError_t err = launch_kernel(gemv_int4_kernel, dim3(stride_grid((d.row_blocks + 7) / 8), M), 256, 0,
                                        reinterpret_cast<cudaStream_t>(stream), d, p);
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}
