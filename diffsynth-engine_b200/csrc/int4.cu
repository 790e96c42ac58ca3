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
// One thread per lane of a tile: eight columns of two rows, twice.
__global__ void __launch_bounds__(256) int4_pack_kernel(const uint8_t* __restrict__ codes, int64_t ld, Int4Dims d,
                                                        uint4* __restrict__ payload) {
  grid_wait();
  const bool words = ((reinterpret_cast<uintptr_t>(codes) | ld) & 3) == 0;
  const int64_t total = static_cast<int64_t>(d.row_blocks) * d.k_tiles * 32;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t tile = i >> 5, rb = tile / d.k_tiles;
    const int lane = i & 31, g = lane >> 2, t = lane & 3, k0 = static_cast<int>(tile - rb * d.k_tiles) * 64 + 8 * t;
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t row = rb * 16 + g + 8 * r;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = k0 + 32 * half;
        uint32_t q = 0x88888888u;   // eight codes; those past the last column are 8
        if (row < d.N && k < d.K) {
          const uint8_t* at = codes + row * ld + (k >> 1);
          if (words && k + 8 <= d.K) {
            q = *reinterpret_cast<const uint32_t*>(at);
          } else {
            const int bytes = min(4, (d.K - k) >> 1);
            for (int x = 0; x < bytes; ++x) q = (q & ~(255u << (8 * x))) | (static_cast<uint32_t>(at[x]) << (8 * x));
          }
        }
        // columns c, c + 1, c + 2, c + 3 of a word go to nibbles r, r + 4, r + 2, r + 6
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t h = q >> (16 * j);
          w[2 * half + j] |= ((h & 15u) | ((h >> 4 & 15u) << 16) | ((h >> 8 & 15u) << 8) | ((h >> 12 & 15u) << 24)) << (4 * r);
        }
      }
    }
    payload[i] = make_uint4(w[0], w[1], w[2], w[3]);
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

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Eight codes of a word as four pairs of fp16 numbers c - 8 (or c), exact, in the way that is usual for 4-bit weights: a code in the
// mantissa of 1024 is 1024 + c in its low four bits and 1024 + 16 c in the next four, so that one shift serves four pairs.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {  // one instruction; the compiler makes two of it
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(bits));
  return d;
}
template <bool UNSIGNED>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t (&a)[4]) {
  constexpr uint32_t k1024 = 0x64006400u, kLow = 0x000f000fu, kHigh = 0x00f000f0u;
  const __half2 low = __float2half2_rn(UNSIGNED ? -1024.f : -1032.f), high = __float2half2_rn(UNSIGNED ? -64.f : -72.f), sixteenth = __float2half2_rn(0.0625f);
  auto h2 = [](uint32_t u) { return *reinterpret_cast<const __half2*>(&u); };
  auto u32 = [](__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); };
  a[0] = u32(__hadd2(h2(and_or(w, kLow, k1024)), low));
  a[1] = u32(__hfma2(h2(and_or(w, kHigh, k1024)), sixteenth, high));
  w >>= 8;
  a[2] = u32(__hadd2(h2(and_or(w, kLow, k1024)), low));
  a[3] = u32(__hfma2(h2(and_or(w, kHigh, k1024)), sixteenth, high));
}
__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

__device__ __forceinline__ uint4 load_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// The weights stream through registers once, 512 bytes of a tile per load of a warp, and are multiplied by the tensor cores:
// A = 16 rows x 16 columns of codes (exact in fp16), B = the activation rows as columns of fp16, fp32 sums of one group at a
// time, which are then multiplied by the group's scale and added up in fp32.  Without minima A holds c - 8; with them it holds
// c, and each group adds m * (sum of its activations).
//
// The activations keep their precision: a row (of a share of the columns) is scaled by a power of two that brings its largest
// magnitude to [2^13, 2^14).  A bf16 value is then exact in fp16 if it is at least 2^-30 of that; a smaller one is off by 2^-25, that is
// 2^-38 of the largest, at most.  An fp32 value (and a bf16 one behind an activation) becomes two columns (SPLIT), high = fp16(x) and
// low = fp16(2^12 (x - high)), whose sums are kept apart until the end: x - high is 2^2 at most, so low stays below 2^14.  That leaves
// out 2^-23 of the value, what one fp32 rounding of a product would, or 2^-25 / 2^12, which is 2^-50 of the largest, whichever is more.
//
// Split: a cluster of `n_share` CTAs owns a range of row blocks, each CTA a share of the columns, whose activations are all that
// it stages; a warp takes every eighth row block of the range and streams its tiles without a pause from one to the next.
// Shares meet in shared memory (CLUSTERED), in a fixed order.
//
// Bound by the bytes of the weight where there are many: 491520 x 5120 in groups of 32 takes 265 us (5.4 of 6.55 TB/s) in bursts of
// some 40 launches and 300 when they go on for half a second, at 880 W and unchanged clocks, whether the weight is the same or another;
// 66 instructions for 512 bytes, 20 of them logic (one lop3 for two codes: written as and + or it is two, 292 us).  Small ones are
// latency: 768 x 256 takes 3.7 us, 5120 x 5120 9.5 to 10.5 (2.5 at the copy rate), with minima 11.8: launch 2, activations 1.2, then a few
// batches of loads and cold code, 1.6 for the two cluster barriers.  An e4m3 weight (one byte each, gemv_kernel) takes 12.7 at 5120 x
// 5120, 16.6 at 13824 x 5104 (here 17.2, with minima 19.4) and 385 at 491520 x 5120.  Tried and not kept: a cp.async ring instead of register buffers (342 us for the
// large one), a third CTA per SM (80 registers: spills), each register slot refilled as it is used (the waits share scoreboards:
// 622 with minima), equal runs of tiles for the warps instead of row blocks (+5 %), sums pushed into the owner's memory to save a
// barrier (small 2.9, large 275).
constexpr int kGemvSmemMax = 227 * 1024 - 1024;
constexpr int kGemvCtas = 2;  // per SM
constexpr float kLowUp = 4096.f;  // what a low column is multiplied by
constexpr int kBatch = 4;  // tiles of a warp in one of the two register buffers that the loads in flight fill

__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_u32(smem_u32(p), rank)));
  return v;
}

// The product of columns k0 .. k1 - 1 of an activation row m that has infinities there with row `row` of a row block of a weight with
// minima: an infinity of the sign that s c + m has, or NaN, and no other column but a NaN matters.  (c and m on their own have other
// signs, so the tensor cores' sums are no use.)  All lanes of a warp, each with a row.  Not inlined: a rare case that should not cost
// the others registers.
__device__ __noinline__ float infinite_part(Int4Dims d, GemvInt4 p, int64_t row_block, int row, int m, int k0, int k1) {
  const uint32_t* words = reinterpret_cast<const uint32_t*>(p.payload);
  float sum = 0.f;
  for (int base = k0; base < k1; base += 32) {
    const int mine = base + (threadIdx.x & 31);
    float x = 0.f;
    if (mine < k1) {
      const int64_t at = m * p.ld_x + mine;
      x = p.x_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.x)[at]) : reinterpret_cast<const float*>(p.x)[at];
      if (p.act_in == DSB_ACT_SILU) x = silu(x);
    }
    for (uint32_t hits = __ballot_sync(0xffffffffu, !(fabsf(x) < INFINITY)); hits; hits &= hits - 1) {
      const int src = __ffs(hits) - 1, k = base + src;
      const int j = 2 * ((k >> 5) & 1) + ((k >> 2) & 1), lane = 4 * (row & 7) + ((k >> 3) & 3), nibble = (row >> 3) + (k & 2) + 4 * (k & 1);
      const uint32_t code = words[((row_block * d.k_tiles + (k >> 6)) * 32 + lane) * 4 + j] >> (4 * nibble) & 15u;
      const int64_t si = scale_index(d, row_block, row, k);
      sum += (__half2float(p.scales[si]) * static_cast<float>(code) + __half2float(p.mins[si])) * __shfl_sync(0xffffffffu, x, src);
    }
  }
  return sum;
}

template <int NT, bool SPLIT, int GROUP, bool MINS, bool CLUSTERED>
__global__ void __launch_bounds__(256, kGemvCtas) gemv_int4_kernel(Int4Dims d, GemvInt4 p, int n_share, int share_tiles, int round_blocks) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kRows = NT * (SPLIT ? 4 : 8);  // activation rows that the columns of B have room for
  constexpr int kHalves = GROUP == 32 ? 2 : 1;  // groups of a tile
  constexpr int kScaleBytes = 32 * kHalves;     // of a tile (of two tiles for groups of 128)
  const int cols = p.M * (SPLIT ? 2 : 1);
  // a row's pitch is 64 bytes above a multiple of 128: the 16-byte reads of two neighbouring columns share no bank
  const int x_pitch = share_tiles * 128 + 64;
  const int share_groups = MINS ? (share_tiles * 64 + GROUP - 1) / GROUP : 0;
  uint8_t* xs = smem;                                               // [cols] rows of fp16
  float* xsum = reinterpret_cast<float*>(xs + cols * x_pitch);      // [share_groups][kRows]
  float* red = xsum + kRows * share_groups;                         // CLUSTERED: [round_blocks][M][16 rows]
  __shared__ uint32_t amax_bits[kRows], inf_rows;   // (a bit for each activation row that has infinities; with minima)
  __shared__ float2 up[kRows];  // the power of two that a row's sums are multiplied by, as two factors
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int rank = CLUSTERED ? cluster_ctarank() : 0;
  const int n_ranges = CLUSTERED ? gridDim.x / n_share : gridDim.x, range = CLUSTERED ? blockIdx.x / n_share : blockIdx.x;
  if (tid < kRows) amax_bits[tid] = 0;
  if (MINS && tid == 0) inf_rows = 0;
  grid_wait();
  const int tile0 = rank * share_tiles;
  const int n_tiles = max(0, min(share_tiles, d.k_tiles - tile0));   // of this share in every row block
  const int block0 = static_cast<int>(static_cast<int64_t>(d.row_blocks) * range / n_ranges);
  const int block1 = static_cast<int>(static_cast<int64_t>(d.row_blocks) * (range + 1) / n_ranges);

  uint4 w[2][kBatch];
  uint2 sc[2][kBatch], mn[2][kBatch];
  // the next tile that this warp requests: its payload, its scales, its number in the share
  const uint4* pw;
  const uint8_t* ps;
  int ahead, left;   // ... and how many tiles of the round are not requested yet
  const int64_t min_off = MINS ? reinterpret_cast<const uint8_t*>(p.mins) - reinterpret_cast<const uint8_t*>(p.scales) : 0;
  const int64_t w_jump = (static_cast<int64_t>(d.k_tiles) * 8 - n_tiles) * 32;
  const int64_t s_jump = static_cast<int64_t>(d.scale_tiles) * 8 * kScaleBytes;
  auto load_one = [&](int buf, int u, const uint4* from, int kt) {
    w[buf][u] = load_stream(from);
    const uint8_t* at = ps + (GROUP == 128 ? kt >> 1 : kt) * kScaleBytes;
    if constexpr (GROUP == 32) {
      sc[buf][u] = __ldg(reinterpret_cast<const uint2*>(at));
      if constexpr (MINS) mn[buf][u] = __ldg(reinterpret_cast<const uint2*>(at + min_off));
    } else {
      sc[buf][u].x = __ldg(reinterpret_cast<const uint32_t*>(at));
      if constexpr (MINS) mn[buf][u].x = __ldg(reinterpret_cast<const uint32_t*>(at + min_off));
    }
  };
  auto load = [&](int buf) {
    if (left >= kBatch && ahead + kBatch <= n_tiles) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) load_one(buf, u, pw + u * 32, ahead + u);
      pw += kBatch * 32;
      ahead += kBatch;
      if (ahead == n_tiles) ahead = 0, pw += w_jump, ps += s_jump;
    } else {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (u < left) {
          load_one(buf, u, pw, ahead);
          pw += 32;
          if (++ahead == n_tiles) ahead = 0, pw += w_jump, ps += s_jump;
        }
      }
    }
    left -= kBatch;
  };
  auto begin = [&](int first_block, int blocks) {
    const int mine = blocks > warp ? (blocks - warp - 1) / 8 + 1 : 0;
    const int64_t rb = first_block + warp;
    left = mine * n_tiles;
    ahead = 0;
    pw = p.payload + (rb * d.k_tiles + tile0) * 32 + lane;
    ps = reinterpret_cast<const uint8_t*>(p.scales) + (rb * d.scale_tiles + (GROUP == 128 ? tile0 >> 1 : tile0)) * kScaleBytes +
         g * (kScaleBytes / 8);
    load(0);
    load(1);
  };
  int round0 = block0, in_round = min(round_blocks, block1 - block0);
  begin(round0, in_round);

  // ---- the activations of this share
  auto eight = [&](int m, int e8, float (&v)[8]) {  // eight neighbouring columns of a row; columns past the last are zero
    const int k = tile0 * 64 + e8 * 8;
    const int64_t off = m * p.ld_x + k;
    const uint8_t* at = reinterpret_cast<const uint8_t*>(p.x) + off * (p.x_bf16 ? 2 : 4);
    if (k + 8 <= d.K && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
      const uint4 a = *reinterpret_cast<const uint4*>(at);
      if (!p.x_bf16) {
        const uint4 b = *reinterpret_cast<const uint4*>(at + 16);
        v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y), v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
        v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y), v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
      } else {
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack_bf16x2(u[j]);
          v[2 * j] = f.x, v[2 * j + 1] = f.y;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = 0.f;
        if (k + j < d.K)
          v[j] = p.x_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.x)[off + j]) : reinterpret_cast<const float*>(p.x)[off + j];
      }
    }
    if (SPLIT && p.act_in == DSB_ACT_SILU) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = silu(v[j]);
    }
  };
  auto largest = [&](int m, const float (&v)[8]) {  // of a warp's finite magnitudes, into the row's
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) a = fmaxf(a, fabsf(v[j]));   // (not of a NaN)
    if (a == INFINITY) {
      a = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (fabsf(v[j]) < INFINITY) a = fmaxf(a, fabsf(v[j]));
      if (MINS) atomicOr(&inf_rows, 1u << m);
    }
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(a));
    if (lane == 0) atomicMax(&amax_bits[m], bits);
  };
  auto convert = [&](int m, int e8, bool in, float (&v)[8]) {
    if (MINS && (inf_rows >> m & 1)) {   // (see infinite_part)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (fabsf(v[j]) == INFINITY) v[j] = 0.f;
    }
    // the power of two, as two factors: its exponent may pass 127
    const uint32_t top = amax_bits[m];
    const int e = top ? ilogbf(__uint_as_float(top)) - 13 : 0, half = e / 2;
    const float f0 = pow2f(-half), f1 = pow2f(half - e);
    uint32_t hi[4], lo[4];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = v[2 * j] * f0 * f1, b = v[2 * j + 1] * f0 * f1;
      const __half2 h = __floats2half2_rn(a, b);
      hi[j] = *reinterpret_cast<const uint32_t*>(&h);
      sum += a + b;
      if constexpr (SPLIT) {
        // (an infinity is its high part alone)
        const float ra = fabsf(a) < INFINITY ? a - __low2float(h) : 0.f, rb = fabsf(b) < INFINITY ? b - __high2float(h) : 0.f;
        const __half2 l = __floats2half2_rn(ra * kLowUp, rb * kLowUp);
        lo[j] = *reinterpret_cast<const uint32_t*>(&l);
      }
    }
    uint8_t* at = xs + (SPLIT ? 2 * m : m) * x_pitch + e8 * 16;
    if (in) {
      *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if constexpr (SPLIT) *reinterpret_cast<uint4*>(at + x_pitch) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    if constexpr (MINS) {
#pragma unroll
      for (int o = 1; o < GROUP / 8; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (in && (lane & (GROUP / 8 - 1)) == 0) xsum[e8 / (GROUP / 8) * kRows + m] = sum;
    }
  };
  {
    const int eights = n_tiles * 8, spans = (eights + 31) / 32, units = p.M * spans;  // a unit: 32 x 8 columns of one row
    __syncthreads();
#pragma unroll 1
    for (int u = warp; u < units; u += 8) {
      const int m = u / spans, e8 = (u - m * spans) * 32 + lane;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (e8 < eights) eight(m, e8, x);
      largest(m, x);
    }
    __syncthreads();
    if (tid < p.M) {
      const int e = amax_bits[tid] ? ilogbf(__uint_as_float(amax_bits[tid])) - 13 : 0, half = e / 2;
      up[tid] = make_float2(pow2f(half), pow2f(e - half));
    }
#pragma unroll 1
    for (int u = warp; u < units; u += 8) {
      const int m = u / spans, e8 = (u - m * spans) * 32 + lane;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (e8 < eights) eight(m, e8, x);
      convert(m, e8, e8 < eights, x);
    }
    __syncthreads();
  }

  // ---- products
  // Lanes whose column of B is not there read the last one's: what it gives is never looked at.
  const uint8_t* xb[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) xb[n] = xs + min(n * 8 + g, cols - 1) * x_pitch + t * 16;
  float acc[NT][4];
  auto tile = [&](const uint4& q, const uint2& s2, const uint2& m2, int kt) {
    const uint32_t words[4] = {q.x, q.y, q.z, q.w};
    float c[NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 b[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) b[n] = *reinterpret_cast<const uint4*>(xb[n] + kt * 128 + h * 64);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t a[4];
        codes_to_f16<MINS>(words[2 * h + j], a);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (j == 0 && (h == 0 || GROUP == 32))
            mma_f16_first(c[n], a, b[n].x, b[n].y);
          else
            mma_f16(c[n], a, j ? b[n].z : b[n].x, j ? b[n].w : b[n].y);
        }
      }
      if (h == 1 || GROUP == 32) {
        const uint32_t sw = GROUP == 32 && h == 1 ? s2.y : s2.x;
        const float2 s = __half22float2(*reinterpret_cast<const __half2*>(&sw));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] = fmaf(s.x, c[n][0], acc[n][0]);
          acc[n][1] = fmaf(s.x, c[n][1], acc[n][1]);
          acc[n][2] = fmaf(s.y, c[n][2], acc[n][2]);
          acc[n][3] = fmaf(s.y, c[n][3], acc[n][3]);
        }
        if (MINS && (GROUP != 128 || (kt & 1) == 0)) {  // a group that spans two tiles adds its minimum's term with the first
          const int grp = GROUP == 32 ? kt * 2 + h : GROUP == 64 ? kt : kt >> 1;
          const uint32_t mw = GROUP == 32 && h == 1 ? m2.y : m2.x;
          const float2 mv = __half22float2(*reinterpret_cast<const __half2*>(&mw));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (SPLIT) {
              const float x0 = xsum[grp * kRows + n * 4 + t];
              acc[n][0] = fmaf(mv.x, x0, acc[n][0]);
              acc[n][2] = fmaf(mv.y, x0, acc[n][2]);
            } else {
              const float2 x2 = *reinterpret_cast<const float2*>(xsum + grp * kRows + n * 8 + 2 * t);
              acc[n][0] = fmaf(mv.x, x2.x, acc[n][0]);
              acc[n][1] = fmaf(mv.x, x2.y, acc[n][1]);
              acc[n][2] = fmaf(mv.y, x2.x, acc[n][2]);
              acc[n][3] = fmaf(mv.y, x2.y, acc[n][3]);
            }
          }
        }
      }
    }
  };
  auto emit = [&](int m, int n, float v) {
    v = act_apply(v + (p.bias ? p.bias[n] : 0.f), p.act_out);
    if (p.y_bf16) {
      __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(p.y) + m * p.ld_y + n;
      *y = __float2bfloat16_rn(p.accumulate ? v + __bfloat162float(*y) : v);
    } else {
      float* y = reinterpret_cast<float*>(p.y) + m * p.ld_y + n;
      *y = p.accumulate ? v + *y : v;
    }
  };
  // the sums of a finished row block (its number in the round)
  auto finish = [&](int block) {
    const uint32_t later = MINS && !CLUSTERED ? inf_rows : 0;   // (rows with infinities have their results from infinite_part)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < (SPLIT ? 1 : 2); ++c) {
          const int m = SPLIT ? n * 4 + t : n * 8 + 2 * t + c, row = g + 8 * r;
          if (m < p.M && !(later >> m & 1)) {
            const float v = (SPLIT ? fmaf(acc[n][2 * r + 1], 1.f / kLowUp, acc[n][2 * r]) : acc[n][2 * r + c]) * up[m].x * up[m].y;
            if constexpr (CLUSTERED)
              red[(block * p.M + m) * 16 + row] = v;
            else if ((round0 + block) * 16 + row < d.N)
              emit(m, (round0 + block) * 16 + row, v);
          }
        }
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  };

  for (;;) {
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    int kt = 0, block = warp;
    // (a share without tiles: its sums are zero)
    if (n_tiles == 0)
      for (; block < in_round; block += 8) finish(block);
    int todo = block < in_round ? ((in_round - block - 1) / 8 + 1) * n_tiles : 0;
    auto multiply = [&](int buf) {
      if (todo >= kBatch && kt + kBatch <= n_tiles) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) tile(w[buf][u], sc[buf][u], mn[buf][u], kt + u);
        kt += kBatch;
        if (kt == n_tiles) finish(block), kt = 0, block += 8;
      } else {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (u < todo) {
            tile(w[buf][u], sc[buf][u], mn[buf][u], kt);
            if (++kt == n_tiles) finish(block), kt = 0, block += 8;
          }
        }
      }
      todo -= kBatch;
    };
    while (todo > 0) {
      multiply(0);
      load(0);
      multiply(1);
      load(1);
    }
    if (MINS && inf_rows) {
      __syncwarp();
      for (int at = warp; at < in_round; at += 8)
        for (uint32_t rows = inf_rows; rows; rows &= rows - 1) {
          const int m = __ffs(rows) - 1, row = lane & 15;
          const float part = infinite_part(d, p, round0 + at, row, m, tile0 * 64, min(d.K, (tile0 + n_tiles) * 64));
          if (lane < 16) {
            if constexpr (CLUSTERED)
              red[(at * p.M + m) * 16 + row] = part;
            else if ((round0 + at) * 16 + row < d.N)
              emit(m, (round0 + at) * 16 + row, part);
          }
        }
    }
    const int next = round0 + in_round, next_in = min(round_blocks, block1 - next);
    if constexpr (CLUSTERED) {
      cluster_sync_all();
      if (next_in > 0) {
        begin(next, next_in);
      }
      const int total = in_round * p.M * 16;
      for (int i = rank * 256 + tid; i < total; i += n_share * 256) {
        const int row = i & 15, bm = i >> 4, m = bm % p.M, n = (round0 + bm / p.M) * 16 + row;
        if (n < d.N) {
          float v = 0.f;
          for (int r = 0; r < n_share; ++r) v += ld_cluster(red + i, r);
          emit(m, n, v);
        }
      }
      cluster_sync_all();   // nobody reads this CTA's sums any more
    }
    if (next_in <= 0) break;
    if constexpr (!CLUSTERED) {
      begin(next, next_in);
    }
    round0 = next;
    in_round = next_in;
  }
}

template <int NT, bool SPLIT, int GROUP, bool MINS, bool CLUSTERED>
static int run_gemv_int4(const Int4Dims& d, const GemvInt4& p, int n_share, cudaStream_t st) {
  auto kern = gemv_int4_kernel<NT, SPLIT, GROUP, MINS, CLUSTERED>;
  DSB_ENSURE_SMEM(kern, kGemvSmemMax);
  int share = (d.k_tiles - 1) / n_share + 1;
  if (GROUP == 128) share = (share + 1) & ~1;   // shares end where groups do
  const int cols = p.M * (SPLIT ? 2 : 1), groups = MINS ? (share * 64 + GROUP - 1) / GROUP : 0;
  const int64_t fixed = static_cast<int64_t>(cols) * (share * 128 + 64) + static_cast<int64_t>(groups) * NT * (SPLIT ? 4 : 8) * 4;
  const int block_bytes = CLUSTERED ? p.M * 64 : 0;
  if (fixed + 8 * block_bytes > kGemvSmemMax) return DSB_ERR_UNSUPPORTED;
  // CTAs that run at once, and the row ranges (a CTA's, or a cluster's) that they make
  const int fit = static_cast<int>((227 << 10) / (fixed + 8 * block_bytes + 2048));
  const int occ = fit > kGemvCtas ? kGemvCtas : fit < 1 ? 1 : fit;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = n_share;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTERED ? 2 : 1;
  int ranges = sm_count() * occ;
  if (CLUSTERED) {
    // clusters that run at once: a GPC holds whole ones, so fewer than the SMs would.  Asked once per device, occupancy and size.
    static std::atomic<int> cached[64][kGemvCtas][4];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return DSB_ERR_CUDA;
    std::atomic<int>& c = cached[dev][occ - 1][n_share == 8 ? 3 : n_share >> 1];
    ranges = c.load();
    if (ranges == 0) {
      cfg.gridDim = dim3(sm_count() / n_share * n_share, 1, 1);
      cfg.dynamicSmemBytes = (227 << 10) / occ - 2048;
      if (cudaOccupancyMaxActiveClusters(&ranges, kern, &cfg) != cudaSuccess || ranges <= 0) ranges = sm_count() * occ / n_share;
      c.store(ranges);
    }
  }
  const int most = (d.row_blocks - 1) / 8 + 1;
  if (ranges > most) ranges = most;
  const int per_range = (d.row_blocks - 1) / ranges + 1;
  int round = per_range;
  int64_t bytes = fixed + static_cast<int64_t>(round) * block_bytes;
  if (CLUSTERED) {
    const int64_t room = (227 << 10) / occ - 2048;
    if (bytes > room) {
      round = static_cast<int>((room - fixed) / block_bytes) & ~7;
      if (round < 8) round = 8;
      bytes = fixed + static_cast<int64_t>(round) * block_bytes;
    }
  }
  cfg.gridDim = dim3(ranges * n_share, 1, 1);
  cfg.dynamicSmemBytes = bytes;
  return cudaLaunchKernelEx(&cfg, kern, d, p, n_share, share, round) == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

template <int NT, bool SPLIT, int GROUP, bool MINS>
static int launch_gemv_int4(const Int4Dims& d, const GemvInt4& p, cudaStream_t st) {
  // Shares of the columns, of four tiles at least.  Each costs a CTA less staging and evens out the work, and a pass over the
  // sums through distributed shared memory.  Measured (us; 1, 2, 4, 8 shares): 5120 x 5120 18.2 11.5 9.5 9.6, 13827 x 5104 with
  // minima and five rows 29.9 21.9 18.6 18.3, with 16 rows 67.9 42.9 30.1 28.0, 30720 x 5120 26.5 24.7 23.9 25.9, 491520 x 5120 263 253
  // 273 309, with minima 323 329 334 366, and 1056768 x 48 tiles with minima 416 420 440 512.  Weights with fewer row blocks than four
  // shares need to reach every SM take eight, the largest one: two would be 4 % less without minima and 1 to 2 % more with them.
  int n_share = d.row_blocks * 4 < 8 * sm_count() ? 8 : 4;
  while (n_share > 1 && d.k_tiles < 4 * n_share) n_share /= 2;
  if (d.row_blocks >= 16 * 8 * sm_count()) n_share = 1;
  for (;;) {
    const int rc = n_share == 1 ? run_gemv_int4<NT, SPLIT, GROUP, MINS, false>(d, p, 1, st)
                                : run_gemv_int4<NT, SPLIT, GROUP, MINS, true>(d, p, n_share, st);
    if (rc != DSB_ERR_UNSUPPORTED || n_share == 8) return rc;   // (a share that does not fit is cut further)
    n_share *= 2;
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
  const int64_t lanes = static_cast<int64_t>(d.row_blocks) * d.k_tiles * 32;
  const int64_t halves = static_cast<int64_t>(d.row_blocks) * d.scale_tiles * 16 * d.per_tile;
  if (launch_kernel(int4_pack_kernel, stride_grid((lanes + 255) / 256), 256, 0, st, codes, ld_codes, d,
                    reinterpret_cast<uint4*>(payload)) != cudaSuccess)
    return DSB_ERR_CUDA;
  const cudaError_t err = launch_kernel(int4_pack_scales_kernel, stride_grid((halves + 255) / 256), 256, 0, st,
                                        reinterpret_cast<const __half*>(scales), reinterpret_cast<const __half*>(mins), ld_scales, d,
                                        reinterpret_cast<__half*>(out_scales), reinterpret_cast<__half*>(out_mins));
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

extern "C" int dsb_int4_dequant(const dsb_int4_weight* w, void* out, int64_t ld_out, void* stream) {
  if (!w) return DSB_ERR_ARG;
  const void *payload = w->payload, *scales = w->scales, *mins = w->mins;
  Int4Dims d;
  if (!payload || !scales || !out || !int4_dims(&d, w->N, w->K, w->group) || ld_out < w->K || !al(payload, 16) || !al(scales, 8) ||
      !al(mins, 8) || !al(out, 2))
    return DSB_ERR_ARG;
  const int64_t words = static_cast<int64_t>(d.row_blocks) * d.k_tiles * 128;
  const cudaError_t err =
      launch_kernel(int4_dequant_kernel, stride_grid((words + 255) / 256), 256, 0, reinterpret_cast<cudaStream_t>(stream),
                    reinterpret_cast<const uint32_t*>(payload), reinterpret_cast<const __half*>(scales),
                    reinterpret_cast<const __half*>(mins), d, reinterpret_cast<__nv_bfloat16*>(out), ld_out);
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

extern "C" int dsb_gemv_int4(const dsb_int4_weight* w, const void* x, int64_t ld_x, int x_bf16, const float* bias, void* y, int64_t ld_y,
                             int y_bf16, int M, int act_in, int act_out, int accumulate, void* stream) {
  if (!w) return DSB_ERR_ARG;
  const void *payload = w->payload, *scales = w->scales, *mins = w->mins;
  const int N = w->N, K = w->K, group = w->group;
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // up to 16 columns of B at a time: 16 rows, or 8 of two columns each
  const bool split = !x_bf16 || act_in != DSB_ACT_NONE;
  int most = split ? 8 : 16;
  for (int m0 = 0; m0 < M;) {
    GemvInt4 q = p;
    q.M = M - m0 < most ? M - m0 : most;
    q.x = reinterpret_cast<const uint8_t*>(x) + m0 * ld_x * (x_bf16 ? 2 : 4);
    q.y = reinterpret_cast<uint8_t*>(y) + m0 * ld_y * (y_bf16 ? 2 : 4);
    const bool two = q.M * (split ? 2 : 1) > 8;
    int rc;
#define DSB_G4(NT, SPLIT, GROUP) \
  rc = mins ? launch_gemv_int4<NT, SPLIT, GROUP, true>(d, q, st) : launch_gemv_int4<NT, SPLIT, GROUP, false>(d, q, st)
#define DSB_G4_GROUP(NT, SPLIT) \
  if (group == 32) DSB_G4(NT, SPLIT, 32); \
  else if (group == 64) DSB_G4(NT, SPLIT, 64); \
  else DSB_G4(NT, SPLIT, 128);
    if (!split) {
      if (two) { DSB_G4_GROUP(2, false) } else { DSB_G4_GROUP(1, false) }
    } else {
      if (two) { DSB_G4_GROUP(2, true) } else { DSB_G4_GROUP(1, true) }
    }
#undef DSB_G4_GROUP
#undef DSB_G4
    if (rc == DSB_ERR_UNSUPPORTED && q.M > 1) {   // rows too long for so many at a time (nothing was launched)
      most = (q.M + 1) / 2;
      continue;
    }
    if (rc != DSB_OK) return rc;
    m0 += q.M;
  }
  return DSB_OK;
}
