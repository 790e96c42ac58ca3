// Keys and values in a paged cache of 8 bits: pages of T tokens, [page][head][token][128] in e4m3, with one exponent e for
// the block of each page and head (its values are e4m3 * 2^e).  A power of two as the scale makes three things exact: taking
// the scale on and off, rounding a block again when a later row needs a larger one (but for what falls below e4m3's smallest
// steps), and the values themselves in 16 bits, so the attention multiplies what the cache stands for and nothing else.
#include <cuda_fp16.h>

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
// 2^e for e in [-128, 127)
__device__ __forceinline__ float pow2i(int e) { return e < -126 ? ldexpf(1.f, e) : __int_as_float((e + 127) << 23); }

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

// One CTA per page that the rows of a sequence touch, head, and pool (k or v): its rows are read once, eight columns a load, kept
// (rotated) in registers while the block's exponent is found, and written as e4m3.  CHUNKS: loads of a thread for a whole page.
template <int THREADS, int CHUNKS>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(KvAppend p) {
  grid_wait();
  __shared__ uint32_t red[THREADS / 32];
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, h = blockIdx.y, T = p.pool.T, tid = threadIdx.x;
  const int start = p.start ? p.start[b] : p.start_all, count = p.counts ? p.counts[b] : p.n;
  const bool rotate = which == 0 && p.rope != nullptr;
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
  const __nv_bfloat16* src = p.src[which] + b * p.sb[which] + h * p.sh[which];
  float x[CHUNKS][8];
  uint32_t top = 0;   // largest finite magnitude, as bits
  {
    uint4 raw[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = tid + c * THREADS;
      raw[c] = make_uint4(0, 0, 0, 0);
      if (i < s.rows * 16) {
        const __nv_bfloat16* at = src + static_cast<int64_t>(s.row + (i >> 4)) * p.sn[which] + (i & 15) * 8;
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(raw[c].x), "=r"(raw[c].y), "=r"(raw[c].z), "=r"(raw[c].w)
                     : "l"(at));
      }
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = tid + c * THREADS;
      const uint32_t u[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = unpack_bf16x2(u[e]);
        x[c][2 * e] = v.x, x[c][2 * e + 1] = v.y;
      }
      if (rotate && i < s.rows * 16) {
        const float4* cs = reinterpret_cast<const float4*>(p.rope) +
                           (static_cast<int64_t>(p.rope_row0) + start + s.row + (i >> 4)) * 32 + (i & 15) * 2;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 r = __ldg(cs + e);   // two pairs' (cos, sin)
          float* v = x[c] + 4 * e;
          const float a0 = v[0], a1 = v[1], a2 = v[2], a3 = v[3];
          v[0] = __fsub_rn(__fmul_rn(a0, r.x), __fmul_rn(a1, r.y));
          v[1] = __fadd_rn(__fmul_rn(a0, r.y), __fmul_rn(a1, r.x));
          v[2] = __fsub_rn(__fmul_rn(a2, r.z), __fmul_rn(a3, r.w));
          v[3] = __fadd_rn(__fmul_rn(a2, r.w), __fmul_rn(a3, r.z));
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t bits = __float_as_uint(x[c][e]) & 0x7fffffffu;
        if (bits < 0x7f800000u) top = max(top, bits);
      }
    }
  }
  if (page < 0) {
    if (p.status) *p.status = DSB_ERR_ARG;
    return;
  }
  const int64_t block = static_cast<int64_t>(page) * p.pool.heads + h;
  uint8_t* dst = (which ? p.pool.v : p.pool.k) + block * T * kD;
  int8_t* exps = (which ? p.pool.v_exp : p.pool.k_exp) + block;
  const int was = *exps;
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) top = max(top, red[i]);
  int e = kv_exponent(top);
  if (s.slot > 0) {
    e = max(e, was);
    if (e > was) {
      const float fall = pow2i(was - e);
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
    if (i < s.rows * 16) {
      const float* v = x[c];
      reinterpret_cast<uint2*>(dst + s.slot * kD)[i] =
          make_uint2(e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv), e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
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

// Eight lanes per (token, head) and pool, 16 columns each.  e4m3 * 2^e is exact in bf16 (but below 2^-126, where it is rounded).
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
    s = pow2i((which ? p.pool.v_exp : p.pool.k_exp)[block]);
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

// The rows (query, head of a group) of a sequence that share a cache head are taken 16 at a time; such a row tile, a cache head
// and the keys that its rows see make an item, in tiles of 32 keys.  All tiles of all items, in order, are dealt out to the
// warps of the grid in equal contiguous shares, whatever the lengths: a warp runs through its share without a pause, finishes the
// items that are its own, and leaves partial results of the (at most two) items that it shares with others, which
// kv_combine_kernel puts together in order.
//
// Per warp: a ring of K and V tiles (TMA, 128-byte swizzle); S = Q K^T and O += P V with 16-bit tensor-core products and fp32
// sums, fragments taken straight from the e4m3 bytes (exact in fp16).  Q is bf16 times a power of two per row, so exact in fp16
// too but for values 2^-27 below the row's largest.  The scales: key j's score is t = S * c * 2^(ek + eq) + ev, in powers of two,
// so that p = 2^(t - m) <= 1 carries the value block's scale, and the row sum adds p * 2^-ev.  p is rounded to fp16: 11 bits,
// three more than bf16 would keep.
constexpr int kTile = 32;       // keys
constexpr int kRowTile = 16;
constexpr int kAttnWarps = 4;   // per CTA; they share nothing
constexpr int kAttnStages = 3;
constexpr int kStageBytes = 2 * kTile * kD;
constexpr int kAttnRing = kAttnWarps * kAttnStages * kStageBytes;
constexpr int kAttnDynSmem = kAttnRing + 1024;
constexpr int kMinShare = DSB_KV_UNCUT_TOKENS / kTile;  // tiles: fewer are not worth another warp
constexpr int kPartRow = 132;   // floats of a partial row: 128 columns, reference exponent, sum, two unused

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// four e4m3 values as two pairs of fp16
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t q, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}\n" : "=r"(lo), "=r"(hi) : "r"(q));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The work of a call: pairs (sequence, row tile), each with the same number of tiles for every cache head.
struct KvWork {
  int Sq, G, heads, T, causal, row_tiles;
  int64_t capacity;
  const int32_t* lens;
  int len_all;
  __device__ __forceinline__ int length(int b) const { return kv_length(lens ? lens[b] : len_all, capacity); }
  // keys that the last row of a row tile sees
  __device__ __forceinline__ int extent(int len, int rt) const {
    const int last = min(rt * kRowTile + kRowTile, Sq * G) - 1;
    return kv_visible(len, Sq, last / G, causal);
  }
  __device__ __forceinline__ int extent_of(int pair) const { return extent(length(pair / row_tiles), pair % row_tiles); }
  __device__ __forceinline__ int tiles(int pair) const { return (extent_of(pair) + kTile - 1) / kTile; }
};
// Sum of the tiles of all pairs before `limit`, for one cache head; with `find`, the last pair whose tiles begin at or before
// that many (times heads) tiles.  All lanes of a warp.
__device__ __forceinline__ int64_t count_tiles(const KvWork& w, int pairs, int64_t find, int* found, int64_t* before) {
  const int lane = threadIdx.x & 31;
  int64_t sum = 0;
  for (int base = 0; base < pairs; base += 32) {
    const int pair = base + lane;
    int64_t n = pair < pairs ? w.tiles(pair) : 0, run = n;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int64_t up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (found) {
      const bool mine = n > 0 && (sum + run - n) * w.heads <= find && (sum + run) * w.heads > find;
      const uint32_t vote = __ballot_sync(0xffffffffu, mine);
      if (vote) {
        const int src = __ffs(vote) - 1;
        *found = base + src;
        *before = __shfl_sync(0xffffffffu, sum + run - n, src) * w.heads;
      }
    }
    sum += __shfl_sync(0xffffffffu, run, 31);
  }
  return sum * w.heads;
}
// tiles per warp, at least `least`
__device__ __forceinline__ int64_t share_of(int64_t total, int warps, int least) {
  const int64_t s = (total + warps - 1) / warps;
  return s < least ? least : s;
}

// A place in the sequence of tiles: a tile of an item, whose rows see `ext` keys.
struct KvCursor {
  int pair, h, tile, ext;
  __device__ __forceinline__ void next(const KvWork& w, int pairs) {
    if (++tile * kTile < ext) return;
    tile = 0;
    if (++h < w.heads) return;
    h = 0;
    do {
      ++pair;
      ext = pair < pairs ? w.extent_of(pair) : 1;
    } while (ext == 0);
  }
};
// ... the one that is `index` tiles from the first of all (there is one)
__device__ __forceinline__ KvCursor find_tile(const KvWork& w, int pairs, int64_t index) {
  KvCursor c;
  int64_t before;
  count_tiles(w, pairs, index, &c.pair, &before);
  c.ext = w.extent_of(c.pair);
  const int tiles = (c.ext + kTile - 1) / kTile;
  c.h = static_cast<int>((index - before) / tiles);
  c.tile = static_cast<int>(index - before - static_cast<int64_t>(c.h) * tiles);
  return c;
}

template <bool T16>
__global__ void __launch_bounds__(kAttnWarps * 32, 2) kv_attn_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_v, KvAttn p, KvWork work,
                                                                     int pairs, float* parts) {
  extern __shared__ uint8_t dyn[];
  __shared__ uint64_t full[kAttnWarps][kAttnStages];
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = dyn + ((1024u - (smem_u32(dyn) & 1023u)) & 1023u) + warp * (kAttnStages * kStageBytes);
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane < kAttnStages) mbar_init(&full[warp][lane], 1);
  if (lane == 0) fence_mbar_init();
  __syncthreads();
  grid_wait();
  const int n_warps = gridDim.x * kAttnWarps, me = blockIdx.x * kAttnWarps + warp;
  // a length outside its table is reported once, by the first warp
  if (me == 0 && p.lens && p.status)
    for (int b = lane; b < p.B; b += 32)
      if (!kv_length_ok(p.lens[b], work.capacity)) *p.status = DSB_ERR_ARG;
  // rows that see no key
  for (int pair = me; pair < pairs; pair += n_warps) {
    if (work.extent_of(pair) > 0) continue;
    const int b = pair / work.row_tiles, row0 = (pair - b * work.row_tiles) * kRowTile;
    for (int x = lane; x < kRowTile * work.heads * 16; x += 32) {
      const int c = x & 15, h = (x >> 4) % work.heads, row = row0 + (x >> 4) / work.heads, qi = row / work.G;
      if (row < work.Sq * work.G)
        reinterpret_cast<uint4*>(p.o + b * p.o_sb + qi * p.o_ss + (h * work.G + row - qi * work.G) * p.o_sh)[c] = make_uint4(0, 0, 0, 0);
    }
  }
  const int64_t total = count_tiles(work, pairs, 0, nullptr, nullptr);
  const int64_t share = share_of(total, n_warps, parts ? kMinShare : 1);
  int64_t first = me * share, end = min(first + share, total);
  if (first >= total) return;
  KvCursor fetch = find_tile(work, pairs, first);
  if (!parts) {
    // nothing is cut: the items that begin in this share, to their ends
    if (fetch.tile > 0) {
      first += (fetch.ext + kTile - 1) / kTile - fetch.tile;
      if (first >= end) return;
      fetch = find_tile(work, pairs, first);
    }
    if (end < total) {
      const KvCursor last = find_tile(work, pairs, end);
      if (last.tile > 0) end += (last.ext + kTile - 1) / kTile - last.tile;
    }
  }
  const int n_mine = static_cast<int>(end - first);
  KvCursor at = fetch;

  // block (page * heads + head) of the 16 keys from `key` on, or -1
  auto block_of = [&](const KvCursor& c, int key) {
    const int page = kv_page(p.tab.row(c.pair / work.row_tiles), p.tab.width, p.pool.n_pages, key / work.T);
    return page < 0 ? -1 : page * work.heads + c.h;
  };
  struct Tile {
    int block0, block1;   // of the first and second 16 keys
  };
  auto look_up = [&](const KvCursor& c) {
    Tile x;
    x.block0 = block_of(c, c.tile * kTile);
    x.block1 = x.block0;
    if (T16) x.block1 = c.tile * kTile + 16 < work.capacity ? block_of(c, c.tile * kTile + 16) : -1;
    return x;
  };
  auto issue = [&](const Tile& x, const KvCursor& c, int stage) {
    if (lane == 0) {
      const int tile = c.tile;
      if ((x.block0 < 0 || (T16 && x.block1 < 0 && tile * kTile + 16 < c.ext)) && p.status) *p.status = DSB_ERR_ARG;
      uint64_t* bar = &full[warp][stage];
      uint8_t* k = ring + stage * kStageBytes;
      uint8_t* v = k + kTile * kD;
      const int slot = (tile * kTile) & (work.T - 1);
      if (T16) {
        const int bytes = ((x.block0 >= 0) + (x.block1 >= 0)) * 2 * 16 * kD;
        if (bytes == 0) {
          mbar_arrive(bar);
        } else {
          mbar_expect_tx(bar, bytes);
          if (x.block0 >= 0) tma_load_2d(k, &map_k, bar, 0, x.block0 * 16), tma_load_2d(v, &map_v, bar, 0, x.block0 * 16);
          if (x.block1 >= 0)
            tma_load_2d(k + 16 * kD, &map_k, bar, 0, x.block1 * 16), tma_load_2d(v + 16 * kD, &map_v, bar, 0, x.block1 * 16);
        }
      } else if (x.block0 < 0) {
        mbar_arrive(bar);
      } else {
        mbar_expect_tx(bar, kStageBytes);
        tma_load_2d(k, &map_k, bar, 0, x.block0 * work.T + slot);
        tma_load_2d(v, &map_v, bar, 0, x.block0 * work.T + slot);
      }
    }
  };

  // tiles on their way: [0] is the one to be multiplied next
  Tile line[kAttnStages];
  int issued = 0;
#pragma unroll
  for (int s = 0; s < kAttnStages; ++s) {
    line[s].block0 = line[s].block1 = -1;
    if (s < n_mine) {
      line[s] = look_up(fetch);
      issue(line[s], fetch, s);
      ++issued;
      fetch.next(work, pairs);
    }
  }
  Tile ahead = {-1, -1};
  if (issued < n_mine) ahead = look_up(fetch);
  struct Exps {
    int k0, k1, v0, v1;
  };
  auto exps_of = [&](const Tile& x) {
    Exps e = {0, 0, 0, 0};
    if (x.block0 >= 0) e.k0 = p.pool.k_exp[x.block0], e.v0 = p.pool.v_exp[x.block0];
    if (T16) {
      if (x.block1 >= 0) e.k1 = p.pool.k_exp[x.block1], e.v1 = p.pool.v_exp[x.block1];
    } else {
      e.k1 = e.k0, e.v1 = e.v0;
    }
    return e;
  };
  Exps exps = exps_of(line[0]);

  uint32_t q[8][4];          // A fragments of 8 x 16 columns: lane (g, t) has rows g, g + 8 and columns 32 t + 4 i + 0..3 of them
  float c_row[2];            // sm_scale * log2(e) * the power of two that the row was divided by
  int seen[2], all_see = 0;  // keys that the rows g, g + 8 see; that every row of the tile sees
  float o[16][4], m_ref[2], l_sum[2];

  int stage = 0, parity = 0, seg_first = at.tile;
  bool failed = false, fresh = true;
  for (int i = 0; i < n_mine; ++i) {
    if (fresh) {
      // ---- an item begins: its rows
      const int b = at.pair / work.row_tiles, rt = at.pair - b * work.row_tiles, rows = work.Sq * work.G;
      const int len = work.length(b);
      all_see = kv_visible(len, work.Sq, rt * kRowTile / work.G, work.causal);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = rt * kRowTile + g + 8 * r, qi = row / work.G;
        uint4 raw[4];
        raw[0] = raw[1] = raw[2] = raw[3] = make_uint4(0, 0, 0, 0);
        seen[r] = 0;
        if (row < rows) {
          seen[r] = kv_visible(len, work.Sq, qi, work.causal);
          const uint4* src = reinterpret_cast<const uint4*>(p.q + b * p.q_sb + qi * p.q_ss + (at.h * work.G + row - qi * work.G) * p.q_sh + 32 * t);
#pragma unroll
          for (int j = 0; j < 4; ++j) raw[j] = src[j];
        }
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack_bf16x2(u[e]);
            if (fabsf(f.x) < INFINITY) top = fmaxf(top, fabsf(f.x));
            if (fabsf(f.y) < INFINITY) top = fmaxf(top, fabsf(f.y));
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the row over 2^eq has its largest magnitude in [2^13, 2^14); eq is kept where both 2^eq and 2^-eq are ordinary numbers
        int eq = static_cast<int>(__float_as_uint(top) >> 23) - 127 - 13;
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
    // exponents of the tile after this one, and the place of the one that will be requested after it
    const Exps exps_next = exps_of(line[1]);

    if (!mbar_wait_all(&full[warp][stage], parity, &abort_flag)) {
      failed = true;
      break;
    }
    const uint8_t* ks = ring + stage * kStageBytes;
    const uint8_t* vs = ks + kTile * kD;
    const int key0 = at.tile * kTile;
    const bool whole = key0 + kTile <= all_see && line[0].block0 >= 0 && line[0].block1 >= 0;

    // ---- scores: n tile j holds keys 8 j + g as columns
    float s[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
      const uint8_t* row = ks + (8 * j + g) * kD;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        // chunk 2 t + c of the key's row lies at 2 t + c xor g (the swizzle): no two lanes of an eight share banks
        const uint4 w = *reinterpret_cast<const uint4*>(row + (((2 * t + c) ^ g) << 4));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t b0, b1;
          e4m3x4_to_f16(u[e], b0, b1);
          mma_16816(s[j], q[c * 4 + e], b0, b1);
        }
      }
    }
    // ---- t = S c + ev, masked; the running reference
    float inv_v[2];   // 2^-ev of the two halves
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int ek = hf ? exps.k1 : exps.k0, ev = hf ? exps.v1 : exps.v0;
      inv_v[hf] = pow2i(-ev);
      const float f0 = c_row[0] * pow2i(ek), f1 = c_row[1] * pow2i(ek), add = static_cast<float>(ev);
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const int j = 2 * hf + jj;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = fmaf(s[j][e], e < 2 ? f0 : f1, add);
        if (!whole) {
          const bool there = hf ? line[0].block1 >= 0 : line[0].block0 >= 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!there || key0 + 8 * j + 2 * t + (e & 1) >= seen[e >> 1]) s[j][e] = -INFINITY;
        }
        top[0] = fmaxf(top[0], fmaxf(s[j][0], s[j][1]));
        top[1] = fmaxf(top[1], fmaxf(s[j][2], s[j][3]));
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
    }
    if (__any_sync(0xffffffffu, top[0] > m_ref[0] || top[1] > m_ref[1])) {
      float f[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float m_new = fmaxf(m_ref[r], top[r]);
        f[r] = m_new == m_ref[r] ? 1.f : fast_exp2(m_ref[r] - m_new);   // (0 for the first keys of a row)
        m_ref[r] = m_new;
        l_sum[r] *= f[r];
      }
#pragma unroll
      for (int n = 0; n < 16; ++n) o[n][0] *= f[0], o[n][1] *= f[0], o[n][2] *= f[1], o[n][3] *= f[1];
    }
    // (a row that has seen no key yet has no reference: its p are 2^-inf)
    const float m0 = m_ref[0] == -INFINITY ? 0.f : m_ref[0], m1 = m_ref[1] == -INFINITY ? 0.f : m_ref[1];
    uint32_t a[2][4];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const int j = 2 * hf + jj;
        s[j][0] = fast_exp2(s[j][0] - m0), s[j][1] = fast_exp2(s[j][1] - m0);
        s[j][2] = fast_exp2(s[j][2] - m1), s[j][3] = fast_exp2(s[j][3] - m1);
        sum0 += s[j][0] + s[j][1];
        sum1 += s[j][2] + s[j][3];
        a[hf][2 * jj] = pack_f16x2(s[j][0], s[j][1]);
        a[hf][2 * jj + 1] = pack_f16x2(s[j][2], s[j][3]);
      }
      l_sum[0] = fmaf(sum0, inv_v[hf], l_sum[0]);
      l_sum[1] = fmaf(sum1, inv_v[hf], l_sum[1]);
    }
    // ---- O += P V: n tile n holds columns 16 g + n
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      uint4 w[4];   // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the half, chunk g
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int key = 16 * hf + 2 * t + (x & 1) + 8 * (x >> 1);
        w[x] = *reinterpret_cast<const uint4*>(vs + key * kD + ((g ^ (key & 7)) << 4));
        // behind the last key there may be anything, and 0 * NaN is NaN
        if (!whole && (key0 + key >= at.ext || (hf ? line[0].block1 : line[0].block0) < 0)) w[x] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t v0 = c == 0 ? w[0].x : c == 1 ? w[0].y : c == 2 ? w[0].z : w[0].w;
        const uint32_t v1 = c == 0 ? w[1].x : c == 1 ? w[1].y : c == 2 ? w[1].z : w[1].w;
        const uint32_t v2 = c == 0 ? w[2].x : c == 1 ? w[2].y : c == 2 ? w[2].z : w[2].w;
        const uint32_t v3 = c == 0 ? w[3].x : c == 1 ? w[3].y : c == 2 ? w[3].z : w[3].w;
        uint32_t b0[4], b1[4];
        e4m3x4_to_f16(__byte_perm(v0, v1, 0x5140), b0[0], b0[1]);
        e4m3x4_to_f16(__byte_perm(v0, v1, 0x7362), b0[2], b0[3]);
        e4m3x4_to_f16(__byte_perm(v2, v3, 0x5140), b1[0], b1[1]);
        e4m3x4_to_f16(__byte_perm(v2, v3, 0x7362), b1[2], b1[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) mma_16816(o[4 * c + e], a[hf], b0[e], b1[e]);
      }
    }
    __syncwarp();
    // ---- this stage is free: the next request, and the look-up of the one behind it
#pragma unroll
    for (int x = 0; x + 1 < kAttnStages; ++x) line[x] = line[x + 1];
    line[kAttnStages - 1] = ahead;
    if (issued < n_mine) {
      issue(ahead, fetch, stage);
      ++issued;
      fetch.next(work, pairs);
      if (issued < n_mine) ahead = look_up(fetch);
    }
    exps = exps_next;
    if (++stage == kAttnStages) stage = 0, parity ^= 1;

    // ---- the end of an item, or of this warp's share of it
    const KvCursor here = at;
    at.next(work, pairs);
    if (at.tile == 0 || i + 1 == n_mine) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l_sum[r] += __shfl_xor_sync(0xffffffffu, l_sum[r], 1);
        l_sum[r] += __shfl_xor_sync(0xffffffffu, l_sum[r], 2);
      }
      const int b = here.pair / work.row_tiles, rt = here.pair - b * work.row_tiles;
      const bool alone = seg_first == 0 && (here.tile + 1) * kTile >= here.ext;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = rt * kRowTile + g + 8 * r, qi = row / work.G;
        if (row >= work.Sq * work.G) continue;
        // columns 32 t + n of the row are o[n][2 r], columns 32 t + 16 + n are o[n][2 r + 1]
        if (alone) {
          const float inv = m_ref[r] == -INFINITY ? 0.f : 1.f / l_sum[r];
          uint4* dst = reinterpret_cast<uint4*>(p.o + b * p.o_sb + qi * p.o_ss + (here.h * work.G + row - qi * work.G) * p.o_sh + 32 * t);
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
          // slot 0: the part with which this warp's share begins, 1: the one with which it ends
          const int slot = first + i + 1 - (here.tile + 1 - seg_first) == first ? 0 : 1;
          float* dst = parts + ((static_cast<int64_t>(me) * 2 + slot) * kRowTile + g + 8 * r) * kPartRow;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<float4*>(dst + 32 * t + 16 * c + 4 * e) =
                  make_float4(o[4 * e][2 * r + c], o[4 * e + 1][2 * r + c], o[4 * e + 2][2 * r + c], o[4 * e + 3][2 * r + c]);
          if (t == 0) dst[128] = m_ref[r], dst[129] = l_sum[r];
        }
      }
      seg_first = 0;
      fresh = true;
    }
  }
  if (failed) {
    if (lane == 0 && p.status) *p.status = DSB_ERR_TIMEOUT;
    // copies that are still on their way must not land in shared memory of whoever comes next
    for (int s = 0; s < kAttnStages; ++s) {
      const int st = stage + s < kAttnStages ? stage + s : stage + s - kAttnStages;
      const int64_t t0 = clock64();
      while (!mbar_try_wait(&full[warp][st], st >= stage ? parity : parity ^ 1) && clock64() - t0 < kWaitLimitCycles) {}
    }
  }
}

// Items that several warps shared: CTA w has the one that the border between the shares of warps w and w + 1 cuts, if that is
// its first cut.  One warp per row; the parts, in order, brought to one reference.
__global__ void __launch_bounds__(256) kv_combine_kernel(KvAttn p, KvWork work, int pairs, int n_warps, const float* parts) {
  grid_wait();
  __shared__ KvCursor item;
  __shared__ int64_t item_share;
  if (threadIdx.x < 32) {
    const int64_t total = count_tiles(work, pairs, 0, nullptr, nullptr), share = share_of(total, n_warps, kMinShare);
    const int64_t border = (blockIdx.x + 1) * share;
    KvCursor c = {-1, 0, 0, 0};
    if (border < total) {
      c = find_tile(work, pairs, border);
      if (c.tile == 0 || c.tile > share) c.pair = -1;
    }
    if (threadIdx.x == 0) item = c, item_share = share;
  }
  __syncthreads();
  if (item.pair < 0) return;
  const int lane = threadIdx.x & 31, h = item.h, b = item.pair / work.row_tiles, rt = item.pair - b * work.row_tiles;
  // the item's first tile lies item.tile tiles before the border, in the share of warp blockIdx.x (which starts with it if the
  // whole share is before the border)
  const int64_t w0 = blockIdx.x, tiles = (item.ext + kTile - 1) / kTile;
  const int64_t w1 = ((w0 + 1) * item_share - item.tile + tiles - 1) / item_share;
  const int slot0 = item.tile == item_share ? 0 : 1;
  for (int r = threadIdx.x >> 5; r < kRowTile; r += 8) {
    const int row = rt * kRowTile + r, qi = row / work.G;
    if (row >= work.Sq * work.G) return;
    auto part = [&](int64_t w) { return parts + ((w * 2 + (w == w0 ? slot0 : 0)) * kRowTile + r) * kPartRow; };
    float m = -INFINITY;
    for (int64_t w = w0 + lane; w <= w1; w += 32) m = fmaxf(m, part(w)[128]);
    m = warp_max(m);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    if (m != -INFINITY) {
#pragma unroll 4
      for (int64_t w = w0; w <= w1; ++w) {
        const float* src = part(w);
        const float f = fast_exp2(src[128] - m);
        const float4 v = reinterpret_cast<const float4*>(src)[lane];
        o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
        l = fmaf(src[129], f, l);
      }
    }
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    uint2 u;
    u.x = pack_bf16x2(o.x * inv, o.y * inv);
    u.y = pack_bf16x2(o.z * inv, o.w * inv);
    reinterpret_cast<uint2*>(p.o + b * p.o_sb + qi * p.o_ss + (h * work.G + row - qi * work.G) * p.o_sh)[lane] = u;
  }
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
  const dim3 grid(kv_span_pages(n, T), p.pool.heads, B * 2);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t err;
  switch (T) {
    case 16: err = launch_kernel(kv_append_kernel<128, 2>, grid, 128, 0, st, p); break;
    case 32: err = launch_kernel(kv_append_kernel<128, 4>, grid, 128, 0, st, p); break;
    case 64: err = launch_kernel(kv_append_kernel<128, 8>, grid, 128, 0, st, p); break;
    default: err = launch_kernel(kv_append_kernel<256, 8>, grid, 256, 0, st, p); break;
  }
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
  if (cudaFuncSetAttribute(kv_attn_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kAttnDynSmem) != cudaSuccess ||
      cudaFuncSetAttribute(kv_attn_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kAttnDynSmem) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kv_attn_kernel<false>, kAttnWarps * 32, kAttnDynSmem) != cudaSuccess ||
      per_sm <= 0)
    return 0;
  n = sm_count() * per_sm * kAttnWarps;
  cached[dev].store(n);
  return n;
}

extern "C" int64_t dsb_kv_attn_workspace_bytes(void) {
  return static_cast<int64_t>(attn_warps()) * 2 * kRowTile * kPartRow * 4;
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
  const int64_t rows = static_cast<int64_t>(Sq) * p.G, row_tiles = (rows - 1) / kRowTile + 1, pairs = row_tiles * B;
  if (rows > 0x7fffff00 || pairs > 0x7fffffff) return DSB_ERR_UNSUPPORTED;
  KvWork w = {};
  w.Sq = Sq;
  w.G = p.G;
  w.heads = p.pool.heads;
  w.T = p.pool.T;
  w.causal = p.causal;
  w.row_tiles = static_cast<int>(row_tiles);
  w.capacity = p.tab.capacity(p.pool.T);
  w.lens = lens;
  w.len_all = len_all;
  // Short sequences (at most kMinShare tiles): whole items for each warp, nothing to combine.  No more CTAs than the longest
  // possible lengths need.
  const int64_t most_len = lens ? w.capacity : len_all, item_tiles = (most_len + kTile - 1) / kTile;
  const int64_t items = pairs * p.pool.heads;
  const bool cut = item_tiles > kMinShare;
  if (cut && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))) return DSB_ERR_ARG;
  const int warps = attn_warps();
  if (warps <= 0) return DSB_ERR_CUDA;
  if (cut && workspace_bytes < dsb_kv_attn_workspace_bytes()) return DSB_ERR_ARG;
  int64_t ctas = cut ? (items * item_tiles + kMinShare * kAttnWarps - 1) / (kMinShare * kAttnWarps) : (items + kAttnWarps - 1) / kAttnWarps;
  if (ctas < 1) ctas = 1;
  if (ctas > warps / kAttnWarps) ctas = warps / kAttnWarps;
  const uint64_t map_rows = static_cast<uint64_t>(p.pool.n_pages) * p.pool.heads * p.pool.T;
  CUtensorMap mk, mv;
  const uint32_t box = p.pool.T == 16 ? 16 : 32;
  if ((rc = make_tmap_2d(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.pool.k, map_rows, kD, kD, box, kD)) != DSB_OK) return rc;
  if ((rc = make_tmap_2d(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.pool.v, map_rows, kD, kD, box, kD)) != DSB_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int n_pairs = static_cast<int>(pairs);
  float* parts = cut ? reinterpret_cast<float*>(workspace) : nullptr;
  cudaError_t err = launch_kernel(p.pool.T == 16 ? kv_attn_kernel<true> : kv_attn_kernel<false>, static_cast<unsigned>(ctas),
                                  kAttnWarps * 32, kAttnDynSmem, st, mk, mv, p, w, n_pairs, parts);
  if (err != cudaSuccess) return DSB_ERR_CUDA;
  const int n_warps = static_cast<int>(ctas) * kAttnWarps;
  if (cut && n_warps > 1)
    err = launch_kernel(kv_combine_kernel, n_warps - 1, 256, 0, st, p, w, n_pairs, n_warps, static_cast<const float*>(parts));
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}
