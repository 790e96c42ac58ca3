// Keys and values in a paged cache of 8 bits: pages of T tokens, [page][head][token][128] in e4m3, with one exponent e for
// the block of each page and head (its values are e4m3 * 2^e).  A power of two as the scale makes three things exact: taking
// the scale on and off, rounding a block again when a later row needs a larger one (but for what falls below e4m3's smallest
// steps), and the values themselves in 16 bits, so the attention multiplies what the cache stands for and nothing else.
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "dsb.h"
#include "kv_index.h"

namespace dsb {

constexpr int kD = 128;

struct KvPool {
  uint8_t* k;
  uint8_t* v;
  int8_t* k_exp;
  int8_t* v_exp;
  int n_pages, heads, T;
};
struct KvTable {
  const int32_t* table;
  int64_t ld;
  int width;
  __device__ __forceinline__ const int32_t* row(int b) const { return table + b * ld; }
  __host__ __device__ __forceinline__ int64_t capacity(int T) const { return static_cast<int64_t>(width) * T; }
};

__device__ __forceinline__ float e4m3_to_float(uint32_t byte) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// ------------------------------------------------------------------------ append
struct KvAppend {
  KvPool pool;
  KvTable tab;
  const __nv_bfloat16* src[2];  // k, v: [B, n, heads, 128]
  int64_t sb[2], sn[2], sh[2];
  int B, n;
  const int32_t* start;
  int start_all;
  const int32_t* counts;
  const float* rope;            // [rope_rows][64][2]
  int rope_rows, rope_row0;
  int* status;
};

// A CTA has the rows that an append puts into one page of one pool (k or v), of some heads, one after the other: a head's rows are
// read once, eight columns a load, and kept in registers (bf16) while the block's exponent is found, with the next head's on their
// way.  The (cos, sin) of the rows are fetched once, into shared memory, and every key is rotated twice: for the exponent, and
// to be written.  CHUNKS: loads of a thread for a whole page.
//
// 256 bytes in and 128 out for a row of a head.  Measured (us): 2 x about 4700 tokens of 40 heads, rotated, 59 to 62 (47 at the copy
// rate), with 73 % of the issue slots of a busy SM taken (rotation and rounding) and 2.1 waves of CTAs at five an SM, a quarter of them without rows; with a CTA for each head, rotations read from L2 by each and kept in fp32 registers, 83; the same with 256
// threads a CTA 81 (pages of 64 tokens) to 131 (16); with each magnitude compared with infinity 69.  512 tokens 5 to 7, one token of
// 16 sequences 3: latency.
template <int THREADS, int CHUNKS, bool ROTATE>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(const __grid_constant__ KvAppend p, int heads_cta) {
  grid_wait();
  extern __shared__ __align__(16) float4 turns[];   // ROTATE: [2 pairs of a float4][row][16]
  __shared__ uint32_t red[2][THREADS / 32], red_finite[THREADS / 32];
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, T = p.pool.T, tid = threadIdx.x;
  const int h0 = blockIdx.y * heads_cta, h1 = min(h0 + heads_cta, p.pool.heads);
  const int start = p.start ? p.start[b] : p.start_all, count = p.counts ? p.counts[b] : p.n;
  if (!kv_append_ok(start, count, p.n, p.tab.capacity(T)) ||
      (p.rope && count > 0 &&
       (start + static_cast<int64_t>(p.rope_row0) < 0 || start + static_cast<int64_t>(p.rope_row0) + count > p.rope_rows))) {
    if (p.status) *p.status = DSB_ERR_ARG;
    return;
  }
  const KvSpan s = kv_span(start, count, T, blockIdx.x);
  if (s.rows == 0) return;
  const int page = kv_page(p.tab.row(b), p.tab.width, p.pool.n_pages, s.index);
  // (the rows are on their way while the page is looked up)
  const __nv_bfloat16* src = p.src[which] + b * p.sb[which] + static_cast<int64_t>(s.row) * p.sn[which];
  const int chunks = s.rows * 16;
  uint4 ahead[CHUNKS];
  auto fetch = [&](int h) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = tid + c * THREADS;
      ahead[c] = make_uint4(0, 0, 0, 0);
      if (i < chunks) {
        const __nv_bfloat16* at = src + h * p.sh[which] + (i >> 4) * p.sn[which] + (i & 15) * 8;
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(ahead[c].x), "=r"(ahead[c].y), "=r"(ahead[c].z), "=r"(ahead[c].w)
                     : "l"(at));
      }
    }
  };
  fetch(h0);
  const bool rotate = ROTATE && which == 0;
  if (rotate) {
    const float4* cs = reinterpret_cast<const float4*>(p.rope) + (static_cast<int64_t>(p.rope_row0) + start + s.row) * 32;
    for (int i = tid; i < s.rows * 32; i += THREADS) turns[(i & 1) * T * 16 + (i >> 1)] = __ldg(cs + i);
    __syncthreads();
  }
  if (page < 0) {
    if (p.status) *p.status = DSB_ERR_ARG;
    return;
  }
  // columns 0..7 of a chunk in fp32, rotated where they are
  auto values = [&](const uint4& w, int i, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack_bf16x2(u[e]);
      v[2 * e] = f.x, v[2 * e + 1] = f.y;
    }
    if (rotate) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4 r = turns[e * T * 16 + i];   // two pairs' (cos, sin)
        float* x = v + 4 * e;
        const float a0 = x[0], a1 = x[1], a2 = x[2], a3 = x[3];
        x[0] = __fsub_rn(__fmul_rn(a0, r.x), __fmul_rn(a1, r.y));
        x[1] = __fadd_rn(__fmul_rn(a0, r.y), __fmul_rn(a1, r.x));
        x[2] = __fsub_rn(__fmul_rn(a2, r.z), __fmul_rn(a3, r.w));
        x[3] = __fadd_rn(__fmul_rn(a2, r.w), __fmul_rn(a3, r.z));
      }
    }
  };
#pragma unroll 1
  for (int h = h0; h < h1; ++h) {
    const int64_t block = static_cast<int64_t>(page) * p.pool.heads + h;
    uint8_t* dst = (which ? p.pool.v : p.pool.k) + block * T * kD;
    int8_t* exps = (which ? p.pool.v_exp : p.pool.k_exp) + block;
    const int was = kv_held_exponent(*exps);
    uint4 raw[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) raw[c] = ahead[c];
    if (h + 1 < h1) fetch(h + 1);
    // the CTA's largest magnitude, as the bits of an fp32 number; FINITE leaves out what is not (NaN is left out anyway)
    auto largest = [&](auto finite, uint32_t* warps) {
      uint32_t top;
      if (rotate) {
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const int i = tid + c * THREADS;
          if (i >= chunks) break;
          float v[8];
          values(raw[c], i, v);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (!finite.value || fabsf(v[e]) < INFINITY) m = fmaxf(m, fabsf(v[e]));
        }
        top = __float_as_uint(m);
      } else {
        uint32_t most = 0;   // two bf16 magnitudes at a time
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const uint32_t u[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t m = u[e] & 0x7fff7fffu;
            most = __vmaxu2(most, finite.value ? m & __vcmpltu2(m, 0x7f807f80u) : m);
          }
        }
        top = max(most & 0xffffu, most >> 16) << 16;
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if ((tid & 31) == 0) warps[tid >> 5] = top;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) top = max(top, warps[i]);
      return top;
    };
    uint32_t top = largest(std::false_type{}, red[h & 1]);
    if (top >= 0x7f800000u) top = largest(std::true_type{}, red_finite);   // (the same for the whole CTA)
    int e = kv_exponent(top);
    if (s.slot > 0) {
      e = max(e, was);
      if (e > was) {
        const float fall = pow2i(max(was - e, -126));   // (2^-127 and 2^-128 too take every e4m3 value to zero)
        for (int i = tid; i < s.slot * (kD / 4); i += THREADS) {
          uint32_t* at = reinterpret_cast<uint32_t*>(dst) + i;
          const uint32_t q = *at;
          *at = e4m3x4(e4m3_to_float(q & 255u) * fall, e4m3_to_float((q >> 8) & 255u) * fall, e4m3_to_float((q >> 16) & 255u) * fall,
                       e4m3_to_float(q >> 24) * fall);
        }
      }
    }
    if (tid == 0) *exps = static_cast<int8_t>(e);
    const float inv = pow2i(-e);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = tid + c * THREADS;
      if (i >= chunks) break;
      float v[8];
      values(raw[c], i, v);
      reinterpret_cast<uint2*>(dst + s.slot * kD)[i] =
          make_uint2(e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv), e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
    }
  }
}

template <bool ROTATE>
static cudaError_t launch_append(const KvAppend& p, cudaStream_t st) {
  // heads of a CTA: one, until there are ten CTAs for every SM
  const int64_t pages = static_cast<int64_t>(kv_span_pages(p.n, p.pool.T)) * p.B * 2, blocks = pages * p.pool.heads;
  int heads = static_cast<int>(blocks / (10 * sm_count()));
  heads = heads < 1 ? 1 : heads > p.pool.heads ? p.pool.heads : heads;
  const dim3 grid(kv_span_pages(p.n, p.pool.T), (p.pool.heads + heads - 1) / heads, p.B * 2);
  const size_t smem = ROTATE ? p.pool.T * 512 : 0;
  switch (p.pool.T) {
    case 16: return launch_kernel(kv_append_kernel<128, 2, ROTATE>, grid, 128, smem, st, p, heads);
    case 32: return launch_kernel(kv_append_kernel<128, 4, ROTATE>, grid, 128, smem, st, p, heads);
    case 64: return launch_kernel(kv_append_kernel<128, 8, ROTATE>, grid, 128, smem, st, p, heads);
    default: {
      auto kern = kv_append_kernel<256, 8, ROTATE>;   // (64 KB of rotations)
      if (ROTATE) {
        static std::atomic<unsigned long long> opted{0};
        int dev = 0;
        cudaError_t err = cudaGetDevice(&dev);
        if (err != cudaSuccess) return err;
        if (!(opted.load() >> (dev & 63) & 1)) {
          if ((err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 512)) != cudaSuccess) return err;
          opted.fetch_or(1ull << (dev & 63));
        }
      }
      return launch_kernel(kern, grid, 256, smem, st, p, heads);
    }
  }
}

// -------------------------------------------------------------------------- read
struct KvRead {
  KvPool pool;
  KvTable tab;
  __nv_bfloat16* dst[2];
  int64_t sb[2], sn[2], sh[2];
  int B, first, n;
  int* status;
};

// Eight lanes per (token, head) and pool, 16 columns each; 1 byte read and 2 written for a value.  e4m3 * 2^e is exact in bf16 (but below 2^-126, where it is rounded).
__global__ void __launch_bounds__(256) kv_read_kernel(KvRead p) {
  grid_wait();
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, T = p.pool.T, c = threadIdx.x & 7;
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 3);
  const int i = static_cast<int>(x / p.pool.heads), h = static_cast<int>(x - static_cast<int64_t>(i) * p.pool.heads);
  if (i >= p.n) return;
  const int tok = p.first + i;
  const int page = kv_page(p.tab.row(b), p.tab.width, p.pool.n_pages, tok / T);
  uint4 q = make_uint4(0, 0, 0, 0);
  float s = 0.f;
  if (page < 0) {
    if (p.status && c == 0) *p.status = DSB_ERR_ARG;
  } else {
    const int64_t block = static_cast<int64_t>(page) * p.pool.heads + h;
    q = reinterpret_cast<const uint4*>((which ? p.pool.v : p.pool.k) + (block * T + tok % T) * kD)[c];
    s = pow2i(kv_held_exponent((which ? p.pool.v_exp : p.pool.k_exp)[block]));
  }
  const uint32_t u[4] = {q.x, q.y, q.z, q.w};
  uint32_t o[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    o[2 * k] = pack_bf16x2(e4m3_to_float(u[k] & 255u) * s, e4m3_to_float((u[k] >> 8) & 255u) * s);
    o[2 * k + 1] = pack_bf16x2(e4m3_to_float((u[k] >> 16) & 255u) * s, e4m3_to_float(u[k] >> 24) * s);
  }
  uint4* dst = reinterpret_cast<uint4*>(p.dst[which] + b * p.sb[which] + i * p.sn[which] + h * p.sh[which]) + 2 * c;
  dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
  dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// --------------------------------------------------------------------- attention
struct KvAttn {
  KvPool pool;
  KvTable tab;
  const __nv_bfloat16* q;
  int64_t q_sb, q_ss, q_sh;
  __nv_bfloat16* o;
  int64_t o_sb, o_ss, o_sh;
  int B, Sq, H, G;
  const int32_t* lens;
  int len_all, causal;
  float scale_log2;
  int* status;
};

// The rows (query, head of a group) of a sequence that share a cache head are taken 16, 32 or 64 at a time (16 for each of up to four
// warps); such a row tile, a cache head and the keys that its rows see make an item, in tiles of 32 keys.  All tiles of all items,
// in order, are dealt out to the grid's streams in equal contiguous shares, whatever the lengths: a stream runs through its share
// without a pause, finishes the items that are its own, and leaves partial results of the (at most two) items that it shares with
// others, which kv_combine_kernel puts together in order.  Sequences of at most kMinShare tiles are not cut.
//
// Per stream: a ring of K and V tiles (TMA, 128-byte swizzle); per warp S = Q K^T and O += P V with 16-bit tensor-core products and
// fp32 sums, fragments taken straight from the e4m3 bytes (exact in fp16).  Q is bf16 times a power of two per row, so exact in
// fp16 too but for values 2^-27 below the row's largest.  The scales: key j's score is t = S * c * 2^(ek + eq) + ev, in powers of
// two, so that p = 2^(t - m) carries the value block's scale, and the row sum adds p * 2^-ev.  p is rounded to fp16: 11 bits,
// three more than bf16 would keep, where it is between 2^-14 and 2^16.  So the reference m of a row is set 2^kStart below its largest t
// and moves only when a t is 2^kHigh above it (moving it with every new maximum cost a rescaling of O in about every second tile), and
// a tile whose largest p of a row is below 2^-kLow - a flat tail behind one large score, or values far smaller than another
// block's - is multiplied apart: p relative to its own largest t, and P V brought to the row's scale and added to O in fp32.  What
// rounding leaves out of a p is at most 2^-11 of it, or 2^-25 / 2^-kLow = 2^-15 of the largest p of its row and tile (of its half
// of the tile, where the halves are of two pages).
//
// What bounds it: one row tile per cache head (a token of each sequence) the cache's bytes, behind about 10 us of start (lengths,
// page table, first tiles, and code that no cache holds yet) and 4 for the combine pass.  A warp's tile takes about 2500 cycles
// (S 780, softmax 560, P V 800, each a chain of dependent steps), and eight warps an SM are just what the memory rate needs; more
// warps would halve the registers.  With more rows the same chains bind: 64 rows share a ring, but each warp converts for itself.
// Measured (us): 77 keys x 24 heads 8; 16 ragged sequences of up to 16384 keys, 8 cache heads 70 (48 at the copy rate); 2 x 131071
// keys, 32 rows 80 (32); 3 x 260 queries over ragged 8100 keys 454 (54 at the tensor rate of tcgen05, which mma.sync does not
// reach).  Without a look at what falls below fp16 the last three are 70, 77 and 433, and wrong where something does; with kStart = 12 and
// kHigh = 15, two powers of two less room, 71, 83 and 465 (more tiles are looked at closely, for no more than that).
// Tried and slower, before that: fragments of V made before the softmax and S in two sums (spills; 75 instead of 71), ten warps with
// shorter rings (same; short calls +1), and converting each tile once for all its warps through shared memory, by warps of its own
// (137 and 518 instead of 87 and 468) or by the consumers in parts (128 and 661).
constexpr int kTile = 32;       // keys
constexpr int kRowTile = 16;
constexpr int kAttnWarps = 4;   // consumers per CTA
constexpr int kAttnThreads = kAttnWarps * 32 + 32;
constexpr int kInfoRing = 32;   // tiles whose description is kept: four rounds of the producer
constexpr int kAttnStages = 3;  // per warp of the stream
constexpr int kStageBytes = 2 * kTile * kD;
constexpr int kAttnRing = kAttnWarps * kAttnStages * kStageBytes;
constexpr int kAttnDynSmem = kAttnRing + 1024;
constexpr int kMinShare = DSB_KV_UNCUT_TOKENS / kTile;  // tiles: fewer are not worth another warp
constexpr float kStart = 13.f, kHigh = 15.9f, kLow = 10.f;
constexpr int kPartRow = 132;   // floats of a partial row: 128 columns, reference exponent, sum, two unused

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// 2^x for x down to -149: value exponents may be 128 apart, and what is 2^-128 of one block's scale is not nothing in its own
__device__ __forceinline__ float exp2_far(float x) {
  const float y = fast_exp2(0.5f * x);
  return y * y;
}
// four e4m3 values as two pairs of fp16
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t q, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}\n" : "=r"(lo), "=r"(hi) : "r"(q));
}
// the four e4m3 values with zeros for NaN, which are noted
__device__ __forceinline__ uint32_t e4m3_drop_nan(uint32_t q, uint32_t& nans) {
  const uint32_t m = __vcmpeq4(q & 0x7f7f7f7fu, 0x7f7f7f7fu);
  nans |= m;
  return q & ~m;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// x / d for x * d < 2^46 (the host sees to it): mul is above 2^46 / d by less than 1, so x * mul / 2^46 is above x / d by less
// than 1 / d.
struct FastDiv {
  uint64_t mul;
  __host__ static FastDiv of(int d) { return {((1ull << 46) + d - 1) / d}; }
  __device__ __forceinline__ int operator()(int x) const { return static_cast<int>(__umul64hi(static_cast<uint64_t>(x) << 18, mul)); }
};
// The work of a call: pairs (sequence, row tile), each with the same number of tiles for every cache head.  (The host keeps the
// number of all tiles below 2^31.)
struct KvWork {
  FastDiv by_G, by_row_tiles, by_heads;
  int Sq, G, heads, T, shift, causal, rows_tile, row_tiles, pairs;   // T = 1 << shift; rows_tile: rows of an item, 16 per warp
  int64_t capacity;
  const int32_t* lens;
  int len_all;
  __device__ __forceinline__ int length(int b) const { return kv_length(lens ? lens[b] : len_all, capacity); }
  // keys that the last row of a row tile sees
  __device__ __forceinline__ int extent(int len, int rt) const {
    if (!causal) return len;
    return kv_visible(len, Sq, by_G(min(rt * rows_tile + rows_tile, Sq * G) - 1), causal);
  }
  __device__ __forceinline__ int extent_of(int pair) const {
    const int b = by_row_tiles(pair);
    return extent(length(b), pair - b * row_tiles);
  }
};
__device__ __forceinline__ int tiles_of(int ext) { return (ext + kTile - 1) / kTile; }
// Tiles of the first n pairs, all heads.  All lanes of a warp.
__device__ __forceinline__ int count_tiles(const KvWork& w, int n) {
  int sum = 0;
  for (int pair = threadIdx.x & 31; pair < n; pair += 32) sum += tiles_of(w.extent_of(pair));
  return __reduce_add_sync(0xffffffffu, sum) * w.heads;
}
__device__ __forceinline__ int count_tiles(const KvWork& w) { return count_tiles(w, w.pairs); }
// tiles per warp, at least `least`
__device__ __forceinline__ int share_of(int total, int warps, int least) { return max(least, (total + warps - 1) / warps); }

// A place in the sequence of tiles: a tile of an item, whose rows see `ext` keys of sequence b.
struct KvCursor {
  int pair, b, h, tile, ext;
  __device__ __forceinline__ void next(const KvWork& w) {
    if (++tile * kTile < ext) return;
    tile = 0;
    if (++h < w.heads) return;
    h = 0;
    do {
      ++pair;
      ext = pair < w.pairs ? w.extent_of(pair) : 1;
    } while (ext == 0);
    b = w.by_row_tiles(pair);
  }
};
// ... the one that is `index` tiles from the first of all (there is one).  All lanes of a warp.
__device__ __forceinline__ KvCursor find_tile(const KvWork& w, int index) {
  const int lane = threadIdx.x & 31;
  KvCursor c = {0, 0, 0, 0, 1};
  int sum = 0;   // tiles of the pairs before these 32, for one head
  for (int base = 0; base < w.pairs; base += 32) {
    const int ext = base + lane < w.pairs ? w.extent_of(base + lane) : 0, n = tiles_of(ext);
    int run = n;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    const uint32_t vote = __ballot_sync(0xffffffffu, (sum + run) * w.heads > index);
    if (vote) {
      const int src = __ffs(vote) - 1;   // the first whose tiles reach beyond `index`
      const int in = index - __shfl_sync(0xffffffffu, sum + run - n, src) * w.heads, tiles = __shfl_sync(0xffffffffu, n, src);
      c.pair = base + src;
      c.b = w.by_row_tiles(c.pair);
      c.ext = __shfl_sync(0xffffffffu, ext, src);
      c.h = in / tiles;
      c.tile = in - c.h * tiles;
      break;
    }
    sum += __shfl_sync(0xffffffffu, run, 31);
  }
  return c;
}

// What a stream leaves for kv_combine_kernel: the item that its share ends in, if that item began in this stream and goes on in
// the `more` streams behind it (pair -1: none).
struct alignas(16) KvCut {
  int pair, h, more, slot;
};

// What the producer warp tells the consumers of a stream about a tile.
struct alignas(16) KvTileInfo {
  int pair, h, tile, ext;
  int there;                  // bit 0, 1: the first and second 16 keys are in the cache
  int k_exp[2], v_exp[2];     // of the two halves
  int b, unused[2];
};

// RW consumer warps share a stream of tiles (the rows of an item are theirs, 16 each); four consumer warps in all, and a
// producer warp that looks up pages and exponents eight tiles ahead, a lane each, and keeps the rings filled.
template <bool T16, int RW>
__global__ void __launch_bounds__(kAttnThreads, 2) kv_attn_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                  const __grid_constant__ CUtensorMap map_v,
                                                                  const __grid_constant__ KvAttn p, const __grid_constant__ KvWork work,
                                                                  float* parts, KvCut* cuts) {
  constexpr int kStreams = kAttnWarps / RW, kStages = kAttnStages * RW;
  extern __shared__ uint8_t dyn[];
  __shared__ uint64_t full[kStreams][kStages], empty[kStreams][kStages];
  __shared__ KvTileInfo infos[kStreams][kInfoRing];
  __shared__ int counts[kStreams], stream_share;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* rings = dyn + ((1024u - (smem_u32(dyn) & 1023u)) & 1023u);
  if (threadIdx.x == 0) abort_flag = 0;
  if (threadIdx.x < kStreams * kStages) {
    mbar_init(&full[0][0] + threadIdx.x, 1);
    mbar_init(&empty[0][0] + threadIdx.x, RW);
    fence_mbar_init();
  }
  grid_wait();
  const int n_streams = gridDim.x * kStreams, stream0 = blockIdx.x * kStreams;

  if (warp == kAttnWarps) {
    // ------------------------------------------------------------------ producer
    constexpr int kLanes = 32 / kStreams, kAhead = 8;   // lanes of a stream; tiles of a round
    const int st = lane / kLanes, j = lane % kLanes;
    KvCursor c = {0, 0, 0, 0, 1};
    int n_mine = 0;
    if (parts) {
      // equal shares of all tiles
      const int total = count_tiles(work), share = share_of(total, n_streams, kMinShare);
#pragma unroll 1
      for (int x = 0; x < kStreams; ++x) {
        const int64_t begin = static_cast<int64_t>(stream0 + x) * share;
        if (begin >= total) break;
        const KvCursor f = find_tile(work, static_cast<int>(begin));
        if (st == x) c = f, n_mine = min(share, total - static_cast<int>(begin));
      }
      if (lane == 0) stream_share = share;
    } else {
      // short sequences: as many whole items for each stream
      const int items = work.pairs * work.heads, per = (items + n_streams - 1) / n_streams;
      const int item0 = min((stream0 + st) * per, items), item1 = min(item0 + per, items);
      c.pair = work.by_heads(item0);
      c.h = item0 - c.pair * work.heads;
      for (int x = item0, pair = c.pair, h = c.h; x < item1; ++x) {
        const int ext = work.extent_of(pair);
        if (n_mine == 0) c.pair = pair, c.h = h, c.ext = ext;   // (the first item with keys)
        n_mine += tiles_of(ext);
        if (++h == work.heads) h = 0, ++pair;
      }
      c.b = work.by_row_tiles(c.pair);
    }
    if (j == 0) counts[st] = n_mine;
    int most = n_mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    // lane j of a stream has its tiles j, j + 8, ...
#pragma unroll 1
    for (int x = 0; x < j && x < kAhead; ++x)
      if (x < n_mine) c.next(work);
    uint8_t* ring = rings + st * (kStages * kStageBytes);
    int stage = 0, phase = 0, next = 0;   // of the stream's next request (its first lane's)
    bool gone = false;
    if (most == 0) __syncthreads();
    for (int i0 = 0; i0 < most && !gone; i0 += kAhead) {
      const int i = i0 + j;
      if (j < kAhead && i < n_mine) {
        KvTileInfo x;
        const int32_t* row = p.tab.row(c.b);
        const int key = c.tile * kTile;
        int page = kv_page(row, p.tab.width, p.pool.n_pages, key >> work.shift);
        int block[2];
        block[0] = block[1] = page < 0 ? -1 : page * work.heads + c.h;
        if (T16) {
          page = kv_page(row, p.tab.width, p.pool.n_pages, (key >> 4) + 1);
          block[1] = page < 0 ? -1 : page * work.heads + c.h;
        }
        if ((block[0] < 0 || (T16 && block[1] < 0 && key + 16 < c.ext)) && p.status) *p.status = DSB_ERR_ARG;
        x.pair = c.pair, x.h = c.h, x.tile = c.tile, x.ext = c.ext, x.b = c.b;
        x.there = (block[0] >= 0 ? 1 : 0) | (block[1] >= 0 ? 2 : 0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          x.k_exp[h] = x.v_exp[h] = 0;
          if (h == 1 && !T16) x.k_exp[1] = x.k_exp[0], x.v_exp[1] = x.v_exp[0];
          else if (block[h] >= 0 && key + 16 * h < c.ext)   // (a page that no key reaches may never have been written)
            x.k_exp[h] = kv_held_exponent(p.pool.k_exp[block[h]]), x.v_exp[h] = kv_held_exponent(p.pool.v_exp[block[h]]);
        }
        x.unused[0] = block[0], x.unused[1] = block[1];
        infos[st][i % kInfoRing] = x;
#pragma unroll 1
        for (int y = 0; y < kAhead; ++y)
          if (i + y + 1 < n_mine) c.next(work);
      }
      if (i0 == 0) __syncthreads();
      __syncwarp();
      // the first lane of each stream requests the round's tiles as stages come free
      const int upto = min(i0 + kAhead, n_mine);
      const long long t0 = clock64();
      while (__any_sync(0xffffffffu, j == 0 && next < upto)) {
        bool moved = false;
        if (j == 0 && next < upto && mbar_try_wait(&empty[st][stage], phase ^ 1)) {
          const KvTileInfo& x = infos[st][next % kInfoRing];
          uint64_t* bar = &full[st][stage];
          uint8_t* k = ring + stage * kStageBytes;
          uint8_t* v = k + kTile * kD;
          const int b0 = x.unused[0], b1 = x.unused[1];
          if (T16) {
            const int bytes = ((b0 >= 0) + (b1 >= 0)) * 2 * 16 * kD;
            if (bytes == 0) {
              mbar_arrive(bar);
            } else {
              mbar_expect_tx(bar, bytes);
              if (b0 >= 0) tma_load_2d(k, &map_k, bar, 0, b0 * 16), tma_load_2d(v, &map_v, bar, 0, b0 * 16);
              if (b1 >= 0) tma_load_2d(k + 16 * kD, &map_k, bar, 0, b1 * 16), tma_load_2d(v + 16 * kD, &map_v, bar, 0, b1 * 16);
            }
          } else if (b0 < 0) {
            mbar_arrive(bar);
          } else {
            const int y = (b0 << work.shift) + ((x.tile * kTile) & (work.T - 1));
            mbar_expect_tx(bar, kStageBytes);
            tma_load_2d(k, &map_k, bar, 0, y);
            tma_load_2d(v, &map_v, bar, 0, y);
          }
          ++next;
          if (++stage == kStages) stage = 0, phase ^= 1;
          moved = true;
        }
        if (!__any_sync(0xffffffffu, moved)) {
          const bool late = clock64() - t0 > kWaitLimitCycles * 2;
          if (__any_sync(0xffffffffu, late || *reinterpret_cast<volatile int*>(&abort_flag) != 0)) {
            abort_flag = 1;
            gone = true;
            break;
          }
        }
      }
    }
    if (gone && lane == 0 && p.status) *p.status = DSB_ERR_TIMEOUT;
    // copies that are still on their way must not land in shared memory of whoever comes next
    if (j == 0)
      for (int back = min(next, kStages); back > 0; --back) {
        const int x = next - back;
        const long long t1 = clock64();
        while (!mbar_try_wait_suspended(&full[st][x % kStages], (x / kStages) & 1) && clock64() - t1 < kWaitLimitCycles) {}
      }
    return;
  }

  // -------------------------------------------------------------------- consumers
  const int g = lane >> 2, t = lane & 3, st = warp / RW, sub = warp % RW;
  // a length outside its table is reported once, by the first warp
  if (blockIdx.x == 0 && warp == 0 && p.lens && p.status)
    for (int b = lane; b < p.B; b += 32)
      if (!kv_length_ok(p.lens[b], work.capacity)) *p.status = DSB_ERR_ARG;
  // rows that see no key
  for (int pair = blockIdx.x * kAttnWarps + warp; pair < work.pairs; pair += gridDim.x * kAttnWarps) {
    if (work.extent_of(pair) > 0) continue;
    const int b = work.by_row_tiles(pair), row0 = (pair - b * work.row_tiles) * work.rows_tile;
#pragma unroll 1
    for (int x = lane; x < work.rows_tile * work.heads * 16; x += 32) {
      const int c = x & 15, r = work.by_heads(x >> 4), h = (x >> 4) - r * work.heads, row = row0 + r, qi = work.by_G(row);
      if (row < work.Sq * work.G)
        reinterpret_cast<uint4*>(p.o + b * p.o_sb + qi * p.o_ss + (h * work.G + row - qi * work.G) * p.o_sh)[c] = make_uint4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  // (before the first wait: where one runs out, the combine pass finds nothing to do for this stream)
  if (parts && sub == 0 && lane == 0) cuts[stream0 + st] = {-1, 0, 0, 0};
  const int n_mine = counts[st];
  const uint8_t* ring = rings + st * (kStages * kStageBytes);

  uint32_t q[8][4];          // A fragments of 8 x 16 columns: lane (g, t) has rows g, g + 8 and columns 32 t + 4 i + 0..3 of them
  float c_row[2];            // sm_scale * log2(e) * the power of two that the row was divided by
  int seen[2], all_see = 0, any_see = 0;  // keys that the rows g, g + 8 see; that every row of the warp sees; that its last one does
  float o[16][4], m_ref[2], l_sum[2];
  int stage = 0, parity = 0, seg_first = 0;
  bool fresh = true;
  auto arrived = [&] {
    if (mbar_wait_all(&full[st][stage], parity, &abort_flag)) return true;
    if (lane == 0 && p.status) *p.status = DSB_ERR_TIMEOUT;
    return false;
  };
  for (int i = 0; i < n_mine; ++i) {
    // (the first round's descriptions were written before the CTA's barrier: the first item's rows are fetched under its keys)
    if (i > 0 && !arrived()) return;
    const int4 info0 = *reinterpret_cast<const int4*>(&infos[st][i % kInfoRing]);      // pair, h, tile, ext
    const int4 info1 = *(reinterpret_cast<const int4*>(&infos[st][i % kInfoRing]) + 1);  // there, k_exp, v_exp[0]
    const int2 info2 = *reinterpret_cast<const int2*>(reinterpret_cast<const int*>(&infos[st][i % kInfoRing]) + 8);   // v_exp[1], b
    const int b = info2.y, rt = info0.x - b * work.row_tiles, head = info0.y, ext = info0.w, key0 = info0.z * kTile;
    const int row0 = rt * work.rows_tile + sub * kRowTile;
    if (fresh) {
      // ---- an item begins: its rows
      seg_first = info0.z;
      const int len = work.length(b), rows = work.Sq * work.G;
      all_see = kv_visible(len, work.Sq, work.by_G(min(row0, rows - 1)), work.causal);
      any_see = row0 < rows ? kv_visible(len, work.Sq, work.by_G(min(row0 + kRowTile, rows) - 1), work.causal) : 0;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = row0 + g + 8 * r, qi = work.by_G(row);
        uint4 raw[4];
        raw[0] = raw[1] = raw[2] = raw[3] = make_uint4(0, 0, 0, 0);
        seen[r] = 0;
        if (row < rows) {
          seen[r] = kv_visible(len, work.Sq, qi, work.causal);
          const uint4* src = reinterpret_cast<const uint4*>(p.q + b * p.q_sb + qi * p.q_ss + (head * work.G + row - qi * work.G) * p.q_sh + 32 * t);
#pragma unroll
          for (int j = 0; j < 4; ++j) raw[j] = src[j];
        }
        uint32_t most = 0;   // magnitudes as bits, two at a time (NaN is more than any: its row is NaN whatever it is divided by)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          most = __vmaxu2(__vmaxu2(most, __vmaxu2(raw[j].x & 0x7fff7fffu, raw[j].y & 0x7fff7fffu)),
                          __vmaxu2(raw[j].z & 0x7fff7fffu, raw[j].w & 0x7fff7fffu));
        most = max(most >> 16, most & 0xffffu);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the row over 2^eq has its largest magnitude in [2^13, 2^14); eq is kept where both 2^eq and 2^-eq are ordinary numbers
        int eq = static_cast<int>(most >> 7) - 127 - 13;
        eq = max(-100, min(114, eq));
        const float down = pow2i(-eq);
        c_row[r] = p.scale_log2 * pow2i(eq);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack_bf16x2(u[e]);
            q[j * 2 + (e >> 1)][r + 2 * (e & 1)] = pack_f16x2(f.x * down, f.y * down);
          }
        }
        m_ref[r] = -INFINITY;
        l_sum[r] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < 16; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
      fresh = false;
    }
    if (i == 0 && !arrived()) return;
    const uint8_t* ks = ring + stage * kStageBytes;
    const uint8_t* vs = ks + kTile * kD;
    const bool whole = key0 + kTile <= all_see && info1.x == 3;
    if (key0 < any_see) {
      // ---- scores: n tile j holds keys 8 j + g as columns
      float s[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t u[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // chunk 2 t + c of the key's row lies at 2 t + c xor g (the swizzle): no two lanes of an eight share banks
          const uint4 w = *reinterpret_cast<const uint4*>(ks + (8 * j + g) * kD + (((2 * t + c) ^ g) << 4));
          u[j][0] = w.x, u[j][1] = w.y, u[j][2] = w.z, u[j][3] = w.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t b0, b1;
            e4m3x4_to_f16(u[j][e], b0, b1);
            mma_16816(s[j], q[c * 4 + e], b0, b1);
          }
      }
      // ---- t = S c + ev, masked; the running reference
      float top[2] = {-INFINITY, -INFINITY}, top_half[2];   // (of the first half too, where the second is of another page)
      const float hi0 = m_ref[0] + kHigh, hi1 = m_ref[1] + kHigh, lo0 = m_ref[0] - kLow, lo1 = m_ref[1] - kLow;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const float kf = pow2i(hf ? info1.z : info1.y), add = static_cast<float>(hf ? info2.x : info1.w);
        const float f0 = c_row[0] * kf, f1 = c_row[1] * kf;
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const int j = 2 * hf + jj;
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] = fmaf(s[j][e], e < 2 ? f0 : f1, add);
          if (!whole) {
            const bool there = info1.x & (1 << hf);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!there || key0 + 8 * j + 2 * t + (e & 1) >= seen[e >> 1]) s[j][e] = -INFINITY;
          }
          top[0] = max3f(top[0], s[j][0], s[j][1]);
          top[1] = max3f(top[1], s[j][2], s[j][3]);
        }
        if (T16 && hf == 0) top_half[0] = top[0], top_half[1] = top[1], top[0] = top[1] = -INFINITY;
      }
      const float least0 = T16 ? fminf(top[0], top_half[0]) : top[0], least1 = T16 ? fminf(top[1], top_half[1]) : top[1];
      if (T16) top[0] = fmaxf(top[0], top_half[0]), top[1] = fmaxf(top[1], top_half[1]);
      bool apart = false;
      if (__any_sync(0xffffffffu, top[0] > hi0 || top[1] > hi1 || least0 < lo0 || least1 < lo1)) {
        bool moves[2], low = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          moves[r] = top[r] > m_ref[r] + kHigh;
        }
        if (__any_sync(0xffffffffu, moves[0] || moves[1])) {
          float f[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            f[r] = moves[r] ? exp2_far(m_ref[r] - (top[r] - kStart)) : 1.f;   // (0 for the first keys of a row)
            m_ref[r] = moves[r] ? top[r] - kStart : m_ref[r];
            l_sum[r] *= f[r];
          }
#pragma unroll
          for (int n = 0; n < 16; ++n) o[n][0] *= f[0], o[n][1] *= f[0], o[n][2] *= f[1], o[n][3] *= f[1];
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          // the smaller of the halves' largest t, if the row sees both; else the one that it sees
          float least = top[r];
          if (T16) {
            float h0 = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
            float h1 = fmaxf(fmaxf(s[2][2 * r], s[2][2 * r + 1]), fmaxf(s[3][2 * r], s[3][2 * r + 1]));
            h0 = fmaxf(h0, __shfl_xor_sync(0xffffffffu, h0, 1)), h0 = fmaxf(h0, __shfl_xor_sync(0xffffffffu, h0, 2));
            h1 = fmaxf(h1, __shfl_xor_sync(0xffffffffu, h1, 1)), h1 = fmaxf(h1, __shfl_xor_sync(0xffffffffu, h1, 2));
            least = h0 == -INFINITY ? h1 : h1 == -INFINITY ? h0 : fminf(h0, h1);
          }
          low |= least > -INFINITY && least < m_ref[r] - kLow;
        }
        apart = __any_sync(0xffffffffu, low);
      }
      // 2^(t - sub) of a half, rounded to fp16, and their sums
      auto probabilities = [&](int hf, float sub0, float sub1, uint32_t (&a)[4], float& sum0, float& sum1) {
        sum0 = sum1 = 0.f;
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const int j = 2 * hf + jj;
          s[j][0] = fast_exp2(s[j][0] - sub0), s[j][1] = fast_exp2(s[j][1] - sub0);
          s[j][2] = fast_exp2(s[j][2] - sub1), s[j][3] = fast_exp2(s[j][3] - sub1);
          sum0 += s[j][0] + s[j][1];
          sum1 += s[j][2] + s[j][3];
          a[2 * jj] = pack_f16x2(s[j][0], s[j][1]);
          a[2 * jj + 1] = pack_f16x2(s[j][2], s[j][3]);
        }
      };
      // O += P V of a half (APART: P V times a number for each row): n tile n holds columns 16 g + n
      uint32_t nans = 0;
      auto products = [&](auto is_apart, int hf, const uint32_t (&a)[4], float unit0, float unit1) {
        uint4 w[4];   // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the half, chunk g
        auto row = [&](int x) { const int key = 16 * hf + 2 * t + (x & 1) + 8 * (x >> 1); return key; };
        if constexpr (!is_apart.value) {
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = *reinterpret_cast<const uint4*>(vs + row(x) * kD + ((g ^ (row(x) & 7)) << 4));
          if (!whole) {
            // behind the last key there may be anything, and 0 * NaN is NaN; so it is for the rows that do not see a key yet
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              if (key0 + row(x) >= ext || !(info1.x & (1 << hf))) w[x] = make_uint4(0, 0, 0, 0);
              w[x].x = e4m3_drop_nan(w[x].x, nans), w[x].y = e4m3_drop_nan(w[x].y, nans);
              w[x].z = e4m3_drop_nan(w[x].z, nans), w[x].w = e4m3_drop_nan(w[x].w, nans);
            }
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if constexpr (is_apart.value) {   // (a word at a time and in order: ahead of their use they cost spills)
              v[x] = *reinterpret_cast<const volatile uint32_t*>(vs + row(x) * kD + ((g ^ (row(x) & 7)) << 4) + 4 * c);
              if (!whole) v[x] = e4m3_drop_nan(key0 + row(x) >= ext || !(info1.x & (1 << hf)) ? 0u : v[x], nans);
            } else {
              v[x] = c == 0 ? w[x].x : c == 1 ? w[x].y : c == 2 ? w[x].z : w[x].w;
            }
          }
          uint32_t b0[4], b1[4];
          e4m3x4_to_f16(__byte_perm(v[0], v[1], 0x5140), b0[0], b0[1]);
          e4m3x4_to_f16(__byte_perm(v[0], v[1], 0x7362), b0[2], b0[3]);
          e4m3x4_to_f16(__byte_perm(v[2], v[3], 0x5140), b1[0], b1[1]);
          e4m3x4_to_f16(__byte_perm(v[2], v[3], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float(&to)[4] = o[4 * c + e];
            if constexpr (is_apart.value) {
              float x[4];
              mma_16816_first(x, a, b0[e], b1[e]);
              to[0] = fmaf(x[0], unit0, to[0]), to[1] = fmaf(x[1], unit0, to[1]);
              to[2] = fmaf(x[2], unit1, to[2]), to[3] = fmaf(x[3], unit1, to[3]);
            } else {
              mma_16816(to, a, b0[e], b1[e]);
            }
          }
        }
      };
      // (a row that has seen no key yet has no reference: its p are 2^-inf)
      if (!apart) {
        const float m0 = m_ref[0] == -INFINITY ? 0.f : m_ref[0], m1 = m_ref[1] == -INFINITY ? 0.f : m_ref[1];
        uint32_t a[2][4];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const float inv_v = pow2i(-(hf ? info2.x : info1.w));
          float sum0, sum1;
          probabilities(hf, m0, m1, a[hf], sum0, sum1);
          l_sum[0] = fmaf(sum0, inv_v, l_sum[0]);
          l_sum[1] = fmaf(sum1, inv_v, l_sum[1]);
        }
        products(std::false_type{}, 0, a[0], 1.f, 1.f);
        products(std::false_type{}, 1, a[1], 1.f, 1.f);
      } else {
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) {   // (the half's scores are always s[0] and s[1])
          const float ev = static_cast<float>(hf ? info2.x : info1.w);
          float most[2], unit[2], sum[2];
          uint32_t a[4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            most[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
            most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 1));
            most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 2));
            most[r] -= kStart;                                                 // (room below it, as for a row's reference)
            unit[r] = most[r] == -INFINITY ? -INFINITY : most[r] - m_ref[r];   // (no key of the half: nothing to add)
            most[r] = most[r] == -INFINITY ? 0.f : most[r];
          }
          probabilities(0, most[0], most[1], a, sum[0], sum[1]);
          l_sum[0] = fmaf(sum[0], exp2_far(unit[0] - ev), l_sum[0]);
          l_sum[1] = fmaf(sum[1], exp2_far(unit[1] - ev), l_sum[1]);
          products(std::true_type{}, hf, a, exp2_far(unit[0]), exp2_far(unit[1]));
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][e] = s[2][e], s[1][e] = s[3][e];
        }
      }
      if (!whole && __any_sync(0xffffffffu, nans != 0)) {
        // the NaN that were left out, for the rows that see them: columns 32 t + n of rows g and g + 8
        uint32_t hit[2] = {0, 0};
#pragma unroll 1
        for (int key = 0; key < kTile; ++key) {
          if (key0 + key >= ext || !(info1.x & (key < 16 ? 1 : 2))) continue;
          uint32_t m = 0;
#pragma unroll 1
          for (int c = 0; c < 32; ++c) {
            const uint32_t byte = vs[key * kD + (((2 * t + (c >> 4)) ^ (key & 7)) << 4) + (c & 15)];
            m |= ((byte & 0x7fu) == 0x7fu ? 1u : 0u) << c;
          }
          hit[0] |= key0 + key < seen[0] ? m : 0;
          hit[1] |= key0 + key < seen[1] ? m : 0;
        }
#pragma unroll
        for (int n = 0; n < 16; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((hit[e >> 1] >> (n + 16 * (e & 1))) & 1u) o[n][e] = __int_as_float(0x7fffffff);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[st][stage]);
    if (++stage == kStages) stage = 0, parity ^= 1;

    // ---- the end of an item, or of this stream's share of it
    const bool last = key0 + kTile >= ext;
    if (last || i + 1 == n_mine) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l_sum[r] += __shfl_xor_sync(0xffffffffu, l_sum[r], 1);
        l_sum[r] += __shfl_xor_sync(0xffffffffu, l_sum[r], 2);
      }
      const bool alone = seg_first == 0 && last;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = row0 + g + 8 * r, qi = work.by_G(row);
        if (row >= work.Sq * work.G) continue;
        // columns 32 t + n of the row are o[n][2 r], columns 32 t + 16 + n are o[n][2 r + 1]
        if (alone) {
          const float inv = l_sum[r] == 0.f ? 0.f : 1.f / l_sum[r];   // (no key: zeros; a row of NaN has no reference, but its sum is NaN)
          uint4* dst = reinterpret_cast<uint4*>(p.o + b * p.o_sb + qi * p.o_ss + (head * work.G + row - qi * work.G) * p.o_sh + 32 * t);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t u[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) u[k] = pack_bf16x2(o[8 * e + 2 * k][2 * r + c] * inv, o[8 * e + 2 * k + 1][2 * r + c] * inv);
              dst[2 * c + e] = make_uint4(u[0], u[1], u[2], u[3]);
            }
        } else {
          // slot 0: the part with which this stream's share begins, 1: the one with which it ends
          const int slot = i == info0.z - seg_first ? 0 : 1;
          float* dst = parts + ((static_cast<int64_t>((stream0 + st) * RW + sub) * 2 + slot) * kRowTile + g + 8 * r) * kPartRow;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<float4*>(dst + 32 * t + 16 * c + 4 * e) =
                  make_float4(o[4 * e][2 * r + c], o[4 * e + 1][2 * r + c], o[4 * e + 2][2 * r + c], o[4 * e + 3][2 * r + c]);
          if (t == 0) dst[128] = m_ref[r] == -INFINITY && l_sum[r] != 0.f ? 0.f : m_ref[r], dst[129] = l_sum[r];
        }
      }
      if (parts && i + 1 == n_mine && sub == 0 && lane == 0) {
        const int border = info0.z + 1, rest = tiles_of(ext) - border;
        cuts[stream0 + st] = {!last && seg_first == 0 ? info0.x : -1, head, (rest + stream_share - 1) / stream_share, i == info0.z ? 0 : 1};
      }
      fresh = true;
    }
  }
}

// Items that several streams shared are brought together from their parts (a stream's each), in order.  Where an item has a few
// parts, CTA (w, y) has eight rows, a warp each, of the item that stream w was the first to leave unfinished.  Where few items
// have many parts, CTA (x, y) has row y of item x, and WARPS warps for it; it finds the item's streams itself.
template <int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : 32 * WARPS) kv_combine_kernel(const __grid_constant__ KvAttn p,
                                                                                  const __grid_constant__ KvWork work, const float* parts,
                                                                                  const KvCut* cuts, int n_streams) {
  grid_wait();
  KvCut cut;
  int w0 = blockIdx.x;
  if constexpr (WARPS == 1) {
    cut = cuts[w0];
    if (!kv_cut_ok(cut.pair, cut.h, cut.more, cut.slot, w0, work.pairs, work.heads, n_streams)) return;
  } else {
    cut.pair = work.by_heads(blockIdx.x);
    cut.h = blockIdx.x - cut.pair * work.heads;
    const int share = share_of(count_tiles(work), n_streams, kMinShare), tiles = tiles_of(work.extent_of(cut.pair));
    const int first = count_tiles(work, cut.pair) + cut.h * tiles;
    w0 = first / share;
    cut.more = (first + tiles - 1) / share - w0;
    cut.slot = first == w0 * share ? 0 : 1;
    if (tiles == 0 || cut.more == 0) return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = work.by_row_tiles(cut.pair), row0 = (cut.pair - b * work.row_tiles) * work.rows_tile;
  const int r = WARPS == 1 ? blockIdx.y * 8 + warp : blockIdx.y, rows = min(work.rows_tile, work.Sq * work.G - row0);
  if (r >= rows) return;
  // the parts of stream w0 + i: of its last slot for i = 0, its first for the others
  const int n = cut.more + 1;
  const int64_t step = static_cast<int64_t>(work.rows_tile) * 2 * kPartRow;
  const float* base = parts + w0 * step + (static_cast<int64_t>(r / kRowTile) * 2 * kRowTile + r % kRowTile) * kPartRow;
  auto part = [&](int i) { return base + i * step + (i == 0 ? cut.slot * (kRowTile * kPartRow) : 0); };
  float m = -INFINITY;
  for (int i = lane; i < n; i += 32) m = fmaxf(m, part(i)[128]);
  m = warp_max(m);
  const int i0 = WARPS == 1 ? 0 : static_cast<int>(static_cast<int64_t>(n) * warp / WARPS);
  const int i1 = WARPS == 1 ? n : static_cast<int>(static_cast<int64_t>(n) * (warp + 1) / WARPS);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int at = i0; at < i1 && m != -INFINITY; at += 32) {
    float f = 0.f;
    if (at + lane < i1) {
      const float2 ml = *reinterpret_cast<const float2*>(part(at + lane) + 128);
      f = exp2_far(ml.x - m);
      l = fmaf(ml.y, f, l);
    }
    const int here = min(32, i1 - at);
#pragma unroll 8
    for (int k = 0; k < here; ++k) {
      const float4 v = reinterpret_cast<const float4*>(part(at + k))[lane];
      const float fk = __shfl_sync(0xffffffffu, f, k);
      o.x = fmaf(v.x, fk, o.x), o.y = fmaf(v.y, fk, o.y), o.z = fmaf(v.z, fk, o.z), o.w = fmaf(v.w, fk, o.w);
    }
  }
  l = warp_sum(l);
  if constexpr (WARPS > 1) {
    __shared__ float4 sums[WARPS][32];
    __shared__ float lens[WARPS];
    sums[warp][lane] = o;
    if (lane == 0) lens[warp] = l;
    __syncthreads();
    if (warp > 0) return;
    for (int i = 1; i < WARPS; ++i) {
      const float4 v = sums[i][lane];
      o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
      l += lens[i];
    }
  }
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  uint2 u;
  u.x = pack_bf16x2(o.x * inv, o.y * inv);
  u.y = pack_bf16x2(o.z * inv, o.w * inv);
  const int row = row0 + r, qi = work.by_G(row);
  reinterpret_cast<uint2*>(p.o + b * p.o_sb + qi * p.o_ss + (cut.h * work.G + row - qi * work.G) * p.o_sh)[lane] = u;
}

}  // namespace dsb

using namespace dsb;

static bool kv_pool(KvPool* out, const dsb_kv_cache* c, int* rc) {
  *rc = DSB_ERR_ARG;
  if (!c || !c->k || !c->v || !c->k_exp || !c->v_exp || c->n_pages <= 0 || c->heads <= 0) return false;
  if ((reinterpret_cast<uintptr_t>(c->k) & 127u) || (reinterpret_cast<uintptr_t>(c->v) & 127u)) return false;
  *rc = DSB_ERR_UNSUPPORTED;
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128) return false;
  if (c->heads > 65535 || static_cast<int64_t>(c->n_pages) * c->heads * c->page_tokens > 0x7fffffff) return false;
  out->k = reinterpret_cast<uint8_t*>(c->k);
  out->v = reinterpret_cast<uint8_t*>(c->v);
  out->k_exp = c->k_exp;
  out->v_exp = c->v_exp;
  out->n_pages = c->n_pages;
  out->heads = c->heads;
  out->T = c->page_tokens;
  *rc = DSB_OK;
  return true;
}
static bool kv_table(KvTable* t, const int32_t* table, int64_t ld, int width, int T) {
  if (!table || (reinterpret_cast<uintptr_t>(table) & 3u) || width <= 0 || ld < width ||
      static_cast<int64_t>(width) * T > 0x7fffff00)
    return false;
  t->table = table;
  t->ld = ld;
  t->width = width;
  return true;
}
static bool rows_ok(const void* p, int64_t sb, int64_t sn, int64_t sh) {
  return p && !(reinterpret_cast<uintptr_t>(p) & 15u) && sb >= 0 && sn >= 0 && sh >= 0 && !((sb | sn | sh) & 7);
}

extern "C" int dsb_kv_append(const dsb_kv_cache* cache, const void* k, int64_t k_stride_b, int64_t k_stride_s, int64_t k_stride_h,
                             const void* v, int64_t v_stride_b, int64_t v_stride_s, int64_t v_stride_h, int B, int n,
                             const int32_t* table, int64_t ld_table, int width, const int32_t* start, int start_all,
                             const int32_t* counts, const float* rope, int rope_rows, int rope_row0, int* status, void* stream) {
  KvAppend p = {};
  int rc;
  if (!kv_pool(&p.pool, cache, &rc)) return rc;
  const int T = p.pool.T;
  if (B < 0 || n < 0 || (rope && ((reinterpret_cast<uintptr_t>(rope) & 15u) || rope_rows < 0))) return DSB_ERR_ARG;
  if (B == 0 || n == 0) return DSB_OK;
  if (!kv_table(&p.tab, table, ld_table, width, T) || !rows_ok(k, k_stride_b, k_stride_s, k_stride_h) ||
      !rows_ok(v, v_stride_b, v_stride_s, v_stride_h) || (!start && !kv_append_ok(start_all, counts ? 0 : n, n, p.tab.capacity(T))))
    return DSB_ERR_ARG;
  if (B > 32767 || n > 0x7fffff00 - T) return DSB_ERR_UNSUPPORTED;
  p.src[0] = reinterpret_cast<const __nv_bfloat16*>(k);
  p.src[1] = reinterpret_cast<const __nv_bfloat16*>(v);
  p.sb[0] = k_stride_b, p.sn[0] = k_stride_s, p.sh[0] = k_stride_h;
  p.sb[1] = v_stride_b, p.sn[1] = v_stride_s, p.sh[1] = v_stride_h;
  p.B = B;
  p.n = n;
  p.start = start;
  p.start_all = start_all;
  p.counts = counts;
  p.rope = rope;
  p.rope_rows = rope_rows;
  p.rope_row0 = rope_row0;
  p.status = status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t err = rope ? launch_append<true>(p, st) : launch_append<false>(p, st);
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

extern "C" int dsb_kv_read(const dsb_kv_cache* cache, const int32_t* table, int64_t ld_table, int width, int B, int first, int n,
                           void* k, int64_t k_stride_b, int64_t k_stride_s, int64_t k_stride_h, void* v, int64_t v_stride_b,
                           int64_t v_stride_s, int64_t v_stride_h, int* status, void* stream) {
  KvRead p = {};
  int rc;
  if (!kv_pool(&p.pool, cache, &rc)) return rc;
  if (B < 0 || n < 0) return DSB_ERR_ARG;
  if (B == 0 || n == 0) return DSB_OK;
  if (!kv_table(&p.tab, table, ld_table, width, p.pool.T) || !rows_ok(k, k_stride_b, k_stride_s, k_stride_h) ||
      !rows_ok(v, v_stride_b, v_stride_s, v_stride_h) || first < 0 || static_cast<int64_t>(first) + n > p.tab.capacity(p.pool.T))
    return DSB_ERR_ARG;
  if (B > 32767) return DSB_ERR_UNSUPPORTED;
  p.dst[0] = reinterpret_cast<__nv_bfloat16*>(k);
  p.dst[1] = reinterpret_cast<__nv_bfloat16*>(v);
  p.sb[0] = k_stride_b, p.sn[0] = k_stride_s, p.sh[0] = k_stride_h;
  p.sb[1] = v_stride_b, p.sn[1] = v_stride_s, p.sh[1] = v_stride_h;
  p.B = B;
  p.first = first;
  p.n = n;
  p.status = status;
  const int64_t blocks = (static_cast<int64_t>(n) * p.pool.heads - 1) / 32 + 1;
  if (blocks > 0x7fffffff) return DSB_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks), 1, B * 2);
  const cudaError_t err = launch_kernel(kv_read_kernel, grid, 256, 0, reinterpret_cast<cudaStream_t>(stream), p);
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

// Warps of the attention kernel that the current device runs at once; 0 on failure.  Also opts the kernels into their shared
// memory.
static int attn_warps() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = cached[dev].load();
  if (n > 0) return n;
  int per_sm = 0;
  auto opt_in = [](auto kern) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kAttnDynSmem) == cudaSuccess;
  };
  if (!opt_in(kv_attn_kernel<false, 1>) || !opt_in(kv_attn_kernel<false, 2>) || !opt_in(kv_attn_kernel<false, 4>) ||
      !opt_in(kv_attn_kernel<true, 1>) || !opt_in(kv_attn_kernel<true, 2>) || !opt_in(kv_attn_kernel<true, 4>) ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kv_attn_kernel<false, 1>, kAttnThreads, kAttnDynSmem) != cudaSuccess ||
      per_sm <= 0)
    return 0;
  n = sm_count() * per_sm * kAttnWarps;
  cached[dev].store(n);
  return n;
}

extern "C" int64_t dsb_kv_attn_workspace_bytes(void) {
  return static_cast<int64_t>(attn_warps()) * (2 * kRowTile * kPartRow * 4 + sizeof(KvCut));
}

extern "C" int dsb_kv_attn(const dsb_kv_cache* cache, const void* q, int64_t q_stride_b, int64_t q_stride_s, int64_t q_stride_h,
                           void* o, int64_t o_stride_b, int64_t o_stride_s, int64_t o_stride_h, int B, int Sq, int H,
                           const int32_t* table, int64_t ld_table, int width, const int32_t* lens, int len_all, int causal,
                           float sm_scale, void* workspace, int64_t workspace_bytes, int* status, void* stream) {
  KvAttn p = {};
  int rc;
  if (!kv_pool(&p.pool, cache, &rc)) return rc;
  if (B < 0 || Sq < 0 || H <= 0 || (H % p.pool.heads)) return DSB_ERR_ARG;
  if (B == 0 || Sq == 0) return DSB_OK;
  if (!kv_table(&p.tab, table, ld_table, width, p.pool.T) || !rows_ok(q, q_stride_b, q_stride_s, q_stride_h) ||
      !rows_ok(o, o_stride_b, o_stride_s, o_stride_h) || (!lens && !kv_length_ok(len_all, p.tab.capacity(p.pool.T))))
    return DSB_ERR_ARG;
  if (B > 65535 || H > 65535) return DSB_ERR_UNSUPPORTED;
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_stride_b, p.q_ss = q_stride_s, p.q_sh = q_stride_h;
  p.o = reinterpret_cast<__nv_bfloat16*>(o);
  p.o_sb = o_stride_b, p.o_ss = o_stride_s, p.o_sh = o_stride_h;
  p.B = B;
  p.Sq = Sq;
  p.H = H;
  p.G = H / p.pool.heads;
  p.lens = lens;
  p.len_all = len_all;
  p.causal = causal ? 1 : 0;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.status = status;
  const int64_t rows = static_cast<int64_t>(Sq) * p.G;
  if (rows > 1 << 30) return DSB_ERR_UNSUPPORTED;
  // 16 rows of an item for each of up to four warps that share its keys
  const int rw = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int64_t row_tiles = (rows - 1) / (kRowTile * rw) + 1, pairs = row_tiles * B;
  if (pairs > 0x3fffffff || pairs * row_tiles >= 1ll << 45) return DSB_ERR_UNSUPPORTED;
  KvWork w = {};
  w.Sq = Sq;
  w.G = p.G;
  w.heads = p.pool.heads;
  w.T = p.pool.T;
  w.shift = w.T == 16 ? 4 : w.T == 32 ? 5 : w.T == 64 ? 6 : 7;
  w.pairs = static_cast<int>(pairs);
  w.causal = p.causal;
  w.rows_tile = kRowTile * rw;
  w.row_tiles = static_cast<int>(row_tiles);
  w.by_G = FastDiv::of(p.G);
  w.by_row_tiles = FastDiv::of(w.row_tiles);
  w.by_heads = FastDiv::of(w.heads);
  w.capacity = p.tab.capacity(p.pool.T);
  w.lens = lens;
  w.len_all = len_all;
  // Short sequences (at most kMinShare tiles): whole items for each warp, nothing to combine.  No more CTAs than the longest
  // possible lengths need.
  const int64_t most_len = lens ? w.capacity : len_all, item_tiles = (most_len + kTile - 1) / kTile;
  const int64_t items = pairs * p.pool.heads;
  const bool cut = item_tiles > kMinShare;
  if (items > 0x3fffffff || items * item_tiles > 0x3fffffff) return DSB_ERR_UNSUPPORTED;
  if (cut && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))) return DSB_ERR_ARG;
  const int warps = attn_warps();
  if (warps <= 0) return DSB_ERR_CUDA;
  if (cut && workspace_bytes < dsb_kv_attn_workspace_bytes()) return DSB_ERR_ARG;
  const int streams_cta = kAttnWarps / rw;
  const int64_t streams = cut ? (items * item_tiles + kMinShare - 1) / kMinShare : items;
  int64_t ctas = (streams + streams_cta - 1) / streams_cta;
  if (ctas < 1) ctas = 1;
  if (ctas > warps / kAttnWarps) ctas = warps / kAttnWarps;
  const uint64_t map_rows = static_cast<uint64_t>(p.pool.n_pages) * p.pool.heads * p.pool.T;
  CUtensorMap mk, mv;
  const uint32_t box = p.pool.T == 16 ? 16 : 32;
  if ((rc = make_tmap_2d(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.pool.k, map_rows, kD, kD, box, kD)) != DSB_OK) return rc;
  if ((rc = make_tmap_2d(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.pool.v, map_rows, kD, kD, box, kD)) != DSB_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  float* parts = cut ? reinterpret_cast<float*>(workspace) : nullptr;
  auto kern = p.pool.T == 16 ? (rw == 1 ? kv_attn_kernel<true, 1> : rw == 2 ? kv_attn_kernel<true, 2> : kv_attn_kernel<true, 4>)
                             : (rw == 1 ? kv_attn_kernel<false, 1> : rw == 2 ? kv_attn_kernel<false, 2> : kv_attn_kernel<false, 4>);
  const int n_streams = static_cast<int>(ctas) * streams_cta;
  KvCut* cuts = reinterpret_cast<KvCut*>(parts + static_cast<int64_t>(warps) * 2 * kRowTile * kPartRow);
  cudaError_t err = launch_kernel(kern, static_cast<unsigned>(ctas), kAttnThreads, kAttnDynSmem, st, mk, mv, p, w, parts, cuts);
  if (err != cudaSuccess) return DSB_ERR_CUDA;
  if (cut && n_streams > 1) {
    const unsigned rows_item = static_cast<unsigned>(rows < w.rows_tile ? rows : w.rows_tile);
    // parts of an item: about as many as there are streams for it.  One sequence of 131000 keys in 512 parts: 16 us with a warp
    // for each row, 6 with 16.
    if (n_streams > 32 * items)
      err = launch_kernel(kv_combine_kernel<16>, dim3(static_cast<unsigned>(items), rows_item), 512, 0, st, p, w,
                          static_cast<const float*>(parts), static_cast<const KvCut*>(cuts), n_streams);
    else
      err = launch_kernel(kv_combine_kernel<1>, dim3(n_streams - 1, (rows_item + 7) / 8), 256, 0, st, p, w,
                          static_cast<const float*>(parts), static_cast<const KvCut*>(cuts), n_streams);
  }
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}
