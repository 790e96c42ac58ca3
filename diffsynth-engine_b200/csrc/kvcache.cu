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
__device__ __forceinline__ uint32_t float_to_e4m3(float x) {
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
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

// One CTA per page that the rows of a sequence touch, head, and pool (k or v).
__global__ void __launch_bounds__(128) kv_append_kernel(KvAppend p) {
  grid_wait();
  __shared__ float red[4];
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, h = blockIdx.y, T = p.pool.T;
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
  if (page < 0) {
    if (p.status) *p.status = DSB_ERR_ARG;
    return;
  }
  const int64_t block = static_cast<int64_t>(page) * p.pool.heads + h;
  uint8_t* dst = (which ? p.pool.v : p.pool.k) + block * T * kD;
  int8_t* exps = (which ? p.pool.v_exp : p.pool.k_exp) + block;
  const __nv_bfloat16* src = p.src[which] + b * p.sb[which] + h * p.sh[which];
  auto pair = [&](int i) {  // the i-th pair of neighbouring columns of the rows that go to this page
    const int r = i >> 6, c = (i & 63) * 2;
    const __nv_bfloat16* x = src + static_cast<int64_t>(s.row + r) * p.sn[which] + c;
    float2 v = make_float2(__bfloat162float(x[0]), __bfloat162float(x[1]));
    if (rotate) {
      const float2 cs =
          reinterpret_cast<const float2*>(p.rope)[static_cast<int64_t>(p.rope_row0 + start + s.row + r) * 64 + (c >> 1)];
      v = make_float2(__fsub_rn(__fmul_rn(v.x, cs.x), __fmul_rn(v.y, cs.y)), __fadd_rn(__fmul_rn(v.x, cs.y), __fmul_rn(v.y, cs.x)));
    }
    return v;
  };
  float amax = 0.f;
  for (int i = threadIdx.x; i < s.rows * 64; i += 128) {
    const float2 v = pair(i);
    if (fabsf(v.x) < INFINITY) amax = fmaxf(amax, fabsf(v.x));
    if (fabsf(v.y) < INFINITY) amax = fmaxf(amax, fabsf(v.y));
  }
  amax = warp_max(amax);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  const int was = *exps;
  __syncthreads();
  amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  int e = kv_exponent(__float_as_uint(amax));
  if (s.slot > 0) {
    e = max(e, was);
    if (e > was) {
      const float fall = pow2i(was - e);
      for (int i = threadIdx.x; i < s.slot * kD; i += 128) dst[i] = static_cast<uint8_t>(float_to_e4m3(e4m3_to_float(dst[i]) * fall));
    }
  }
  if (threadIdx.x == 0) *exps = static_cast<int8_t>(e);
  const float inv = pow2i(-e);
  for (int i = threadIdx.x; i < s.rows * 64; i += 128) {
    const float2 v = pair(i);
    uint8_t* d = dst + s.slot * kD + 2 * i;
    d[0] = static_cast<uint8_t>(float_to_e4m3(v.x * inv));
    d[1] = static_cast<uint8_t>(float_to_e4m3(v.y * inv));
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

// One warp per (token, head) and pool; 4 columns a lane.  e4m3 * 2^e is exact in bf16.
__global__ void __launch_bounds__(256) kv_read_kernel(KvRead p) {
  grid_wait();
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, h = blockIdx.y, T = p.pool.T, lane = threadIdx.x & 31;
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= p.n) return;
  const int tok = p.first + i;
  const int page = kv_page(p.tab.row(b), p.tab.width, p.pool.n_pages, tok / T);
  uint32_t q = 0;
  float s = 0.f;
  if (page < 0) {
    if (p.status && lane == 0) *p.status = DSB_ERR_ARG;
  } else {
    const int64_t block = static_cast<int64_t>(page) * p.pool.heads + h;
    q = reinterpret_cast<const uint32_t*>((which ? p.pool.v : p.pool.k) + (block * T + tok % T) * kD)[lane];
    s = pow2i((which ? p.pool.v_exp : p.pool.k_exp)[block]);
  }
  uint2 o;
  o.x = pack_bf16x2(e4m3_to_float(q & 255u) * s, e4m3_to_float((q >> 8) & 255u) * s);
  o.y = pack_bf16x2(e4m3_to_float((q >> 16) & 255u) * s, e4m3_to_float(q >> 24) * s);
  reinterpret_cast<uint2*>(p.dst[which] + b * p.sb[which] + i * p.sn[which] + h * p.sh[which])[lane] = o;
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

// One warp per (sample, query, head): running maximum and sum over the keys, 4 columns a lane.
__global__ void __launch_bounds__(256) kv_attn_kernel(KvAttn p) {
  grid_wait();
  const int lane = threadIdx.x & 31, b = blockIdx.z, h = blockIdx.y, T = p.pool.T;
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= p.Sq) return;
  const int64_t cap = p.tab.capacity(T);
  int len = p.lens ? p.lens[b] : p.len_all;
  if (!kv_length_ok(len, cap) && p.status && lane == 0) *p.status = DSB_ERR_ARG;
  len = kv_length(len, cap);
  const int n = kv_visible(len, p.Sq, i, p.causal);
  const uint2 qv = reinterpret_cast<const uint2*>(p.q + b * p.q_sb + i * p.q_ss + h * p.q_sh)[lane];
  const float2 qa = unpack_bf16x2(qv.x), qb = unpack_bf16x2(qv.y);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j * T < n; ++j) {
    const int page = kv_page(p.tab.row(b), p.tab.width, p.pool.n_pages, j);
    if (page < 0) {
      if (p.status && lane == 0) *p.status = DSB_ERR_ARG;
      continue;
    }
    const int64_t block = static_cast<int64_t>(page) * p.pool.heads + h / p.G;
    const float ks = pow2i(p.pool.k_exp[block]) * p.scale_log2, vs = pow2i(p.pool.v_exp[block]);
    const int rows = min(T, n - j * T);
    for (int r = 0; r < rows; ++r) {
      const uint32_t kq = reinterpret_cast<const uint32_t*>(p.pool.k + (block * T + r) * kD)[lane];
      const uint32_t vq = reinterpret_cast<const uint32_t*>(p.pool.v + (block * T + r) * kD)[lane];
      float d = qa.x * e4m3_to_float(kq & 255u) + qa.y * e4m3_to_float((kq >> 8) & 255u) + qb.x * e4m3_to_float((kq >> 16) & 255u) +
                qb.y * e4m3_to_float(kq >> 24);
      d = warp_sum(d) * ks;
      const float mn = fmaxf(m, d), a = exp2f(m - mn), e = exp2f(d - mn);
      m = mn;
      l = l * a + e;
      const float ev = e * vs;
      o[0] = o[0] * a + ev * e4m3_to_float(vq & 255u);
      o[1] = o[1] * a + ev * e4m3_to_float((vq >> 8) & 255u);
      o[2] = o[2] * a + ev * e4m3_to_float((vq >> 16) & 255u);
      o[3] = o[3] * a + ev * e4m3_to_float(vq >> 24);
    }
  }
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  uint2 w;
  w.x = pack_bf16x2(o[0] * inv, o[1] * inv);
  w.y = pack_bf16x2(o[2] * inv, o[3] * inv);
  reinterpret_cast<uint2*>(p.o + b * p.o_sb + i * p.o_ss + h * p.o_sh)[lane] = w;
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
  const cudaError_t err = launch_kernel(kv_append_kernel, grid, 128, 0, reinterpret_cast<cudaStream_t>(stream), p);
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
  const dim3 grid((n - 1) / 8 + 1, p.pool.heads, B * 2);
  const cudaError_t err = launch_kernel(kv_read_kernel, grid, 256, 0, reinterpret_cast<cudaStream_t>(stream), p);
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}

extern "C" int64_t dsb_kv_attn_workspace_bytes(void) { return 0; }

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
  (void)workspace;
  (void)workspace_bytes;
  const dim3 grid((Sq - 1) / 8 + 1, H, B);
  const cudaError_t err = launch_kernel(kv_attn_kernel, grid, 256, 0, reinterpret_cast<cudaStream_t>(stream), p);
  return err == cudaSuccess ? DSB_OK : DSB_ERR_CUDA;
}
