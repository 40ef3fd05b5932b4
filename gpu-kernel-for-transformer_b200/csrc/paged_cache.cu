// Writing new tokens into a paged KV cache (optionally in 8 bits with a scale
// per token and head) and reading them back as fp16.
//
// Both are one pass over memory. A thread handles 8 consecutive elements
// (16 bytes of fp16) of one (token, head) row of K and of V; the head_dim / 8
// threads of a row sit in one warp and reduce max|x| with shuffles.
//
// Quantisation rounds x / s as if in exact arithmetic, so that a code is the
// nearest one even when the quotient lies within an fp32 rounding of the
// border between two codes:
//  int8: c = rint(x * (1/s)) is the nearest code or, next to a border, its
//        neighbour; e = fma(-c, s, x) is x - c*s exactly (x has 11 bits, and
//        near a border ulp(s) <= ulp(x), so e has at most 24), and |e| against
//        s/2 tells which.
//  e4m3: the quotient's bits behind the 3 of the code decide unless they are
//        within 4 ulp of a half (or the code is subnormal); then the quotient
//        is divided out and rounded to odd, which rounds on correctly.
#include "paged.cuh"

namespace tfx {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int quant_i8(float x, float inv, float s, float half_s) {
  float c = rintf(x * inv);
  const float e = fmaf(-c, s, x);
  if (fabsf(e) >= half_s) {  // rare: next to a border
    if (fabsf(e) > half_s || (static_cast<int>(c) & 1)) c += copysignf(1.0f, e);
  }
  return static_cast<int>(fminf(fmaxf(c, -127.0f), 127.0f));
}

// x / s for a conversion to e4m3 (see the file's comment).
__device__ __forceinline__ float quot_e4m3(float x, float inv, float s) {
  const float y = x * inv;
  const uint32_t bits = __float_as_uint(y) & 0x7fffffffu;
  if (((bits & 0xfffffu) - 0x7fffcu) <= 8u || (bits < 0x3c800000u && x != 0.f)) {  // 2^-6
    const float ax = fabsf(x), q = __fdiv_rn(ax, s), r = fmaf(-q, s, ax);
    uint32_t odd = __float_as_uint(q);
    if (r < 0.f) --odd;
    if (r != 0.f) odd |= 1u;
    return copysignf(__uint_as_float(odd), x);
  }
  return y;
}

// max|x| of a row's elements as fp16 bits, over the CH threads of the row.
template <int CH>
__device__ __forceinline__ uint32_t row_absmax(const uint4& x) {
  uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                        __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
  m = max(m & 0xffffu, m >> 16);
#pragma unroll
  for (int d = 1; d < CH; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  return m;
}

// Eight codes of a row whose max|x| has the fp16 bits `top`; *scale gets s.
template <int CODE>
__device__ __forceinline__ uint2 quantise(const uint4& x, uint32_t top, float* scale) {
  if (top >= 0x7c00u) {
    *scale = __uint_as_float(0x7fc00000u);
    return make_uint2(0u, 0u);
  }
  const float s = __fdiv_rn(__half2float(__ushort_as_half(static_cast<unsigned short>(top))),
                            CODE == kCodeI8 ? 127.0f : 448.0f);
  *scale = s;
  if (top == 0u) return make_uint2(0u, 0u);
  const float inv = __frcp_rn(s), half_s = 0.5f * s;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t out[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(bits_h2(w[i]));
    uint32_t two;
    if constexpr (CODE == kCodeI8) {
      two = (quant_i8(f.x, inv, s, half_s) & 0xff) | ((quant_i8(f.y, inv, s, half_s) & 0xff) << 8);
    } else {
      two = __nv_cvt_float2_to_fp8x2(make_float2(quot_e4m3(f.x, inv, s), quot_e4m3(f.y, inv, s)),
                                     __NV_SATFINITE, __NV_E4M3);
    }
    out[i >> 1] |= two << (16 * (i & 1));
  }
  return make_uint2(out[0], out[1]);
}

template <int CODE, int HD>
__global__ void __launch_bounds__(kThreads)
    paged_append_kernel(const __half* __restrict__ k, int64_t ld_k, const __half* __restrict__ v,
                        int64_t ld_v, Paged p) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int CH = HD / 8;
  const int row = blockIdx.x * (kThreads / CH) + threadIdx.x / CH;  // (token, head)
  const int c = threadIdx.x % CH;
  const int t = row / p.kv_heads, h = row % p.kv_heads;
  int page = -1, pos = 0;
  if (t < p.num_tokens) {
    const int b = paged_seq_of_row(p, t);
    if (b >= 0) {
      const PagedSeq s = paged_seq(p, b);
      pos = s.pos0 + (t - s.row0);
      if (t >= s.row0 && t < s.row0 + s.n) page = paged_page(p, b, pos);
    }
  }
  uint4 xk = make_uint4(0, 0, 0, 0), xv = xk;
  if (page >= 0) {
    xk = __ldcs(reinterpret_cast<const uint4*>(k + t * ld_k + h * HD + c * 8));
    xv = __ldcs(reinterpret_cast<const uint4*>(v + t * ld_v + h * HD + c * 8));
  }
  const int64_t at = paged_offset(p, page, pos) + h * p.head_stride + c * 8;
  if constexpr (CODE == kCodeF16) {
    if (page >= 0) {
      *reinterpret_cast<uint4*>(static_cast<__half*>(p.k) + at) = xk;
      *reinterpret_cast<uint4*>(static_cast<__half*>(p.v) + at) = xv;
    }
  } else {
    const uint32_t tk = row_absmax<CH>(xk), tv = row_absmax<CH>(xv);  // every lane takes part
    if (page >= 0) {
      float sk, sv;
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.k) + at) = quantise<CODE>(xk, tk, &sk);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.v) + at) = quantise<CODE>(xv, tv, &sv);
      if (c == 0) {
        const int64_t so = paged_scale_offset(p, page, h, pos);
        p.k_scale[so] = sk;
        p.v_scale[so] = sv;
      }
    }
  }
}

// Eight codes times the scale, rounded once to fp16.
template <int CODE>
__device__ __forceinline__ uint4 dequantise(uint2 x, float s) {
  uint32_t h[4] = {codes_to_h2<CODE, 0, 1>(x.x), codes_to_h2<CODE, 2, 3>(x.x),
                   codes_to_h2<CODE, 0, 1>(x.y), codes_to_h2<CODE, 2, 3>(x.y)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(bits_h2(h[i]));
    h[i] = pack_half2(f.x * s, f.y * s);
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
}

template <int CODE, int HD>
__global__ void __launch_bounds__(kThreads)
    paged_read_kernel(__half* __restrict__ k, int64_t ld_k, __half* __restrict__ v, int64_t ld_v,
                      Paged p) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int CH = HD / 8;
  const int row = blockIdx.x * (kThreads / CH) + threadIdx.x / CH;
  const int c = threadIdx.x % CH;
  const int t = row / p.kv_heads, h = row % p.kv_heads;
  if (t >= p.num_tokens) return;
  const int b = paged_seq_of_row(p, t);
  if (b < 0) return;
  const PagedSeq s = paged_seq(p, b);
  if (t < s.row0 || t >= s.row0 + s.n) return;
  const int pos = s.pos0 + (t - s.row0);
  const int page = paged_page(p, b, pos);
  uint4 xk = make_uint4(0, 0, 0, 0), xv = xk;
  if (page >= 0) {
    const int64_t at = paged_offset(p, page, pos) + h * p.head_stride + c * 8;
    if constexpr (CODE == kCodeF16) {
      xk = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p.k) + at);
      xv = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p.v) + at);
    } else {
      const int64_t so = paged_scale_offset(p, page, h, pos);
      xk = dequantise<CODE>(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.k) + at),
                            p.k_scale[so]);
      xv = dequantise<CODE>(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.v) + at),
                            p.v_scale[so]);
    }
  }
  __stcs(reinterpret_cast<uint4*>(k + t * ld_k + h * HD + c * 8), xk);
  __stcs(reinterpret_cast<uint4*>(v + t * ld_v + h * HD + c * 8), xv);
}

template <int CODE, int HD>
int launch_copy(bool append, __half* k, int64_t ld_k, __half* v, int64_t ld_v, const Paged& p,
                cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(p.num_tokens) * p.kv_heads;
  constexpr int per_block = kThreads / (HD / 8);
  const dim3 grid(static_cast<unsigned>((rows + per_block - 1) / per_block));
  if (append) {
    launch_pdl(paged_append_kernel<CODE, HD>, grid, dim3(kThreads), 0, stream,
               static_cast<const __half*>(k), ld_k, static_cast<const __half*>(v), ld_v, p);
    return check_launch("paged_append_kernel");
  }
  launch_pdl(paged_read_kernel<CODE, HD>, grid, dim3(kThreads), 0, stream, k, ld_k, v, ld_v, p);
  return check_launch("paged_read_kernel");
}

template <int CODE>
int launch_copy_hd(bool append, int head_dim, __half* k, int64_t ld_k, __half* v, int64_t ld_v,
                   const Paged& p, cudaStream_t stream) {
  switch (head_dim) {
    case 8:
      if constexpr (CODE == kCodeF16)
        return launch_copy<CODE, 8>(append, k, ld_k, v, ld_v, p, stream);
      break;
    case 16: return launch_copy<CODE, 16>(append, k, ld_k, v, ld_v, p, stream);
    case 32: return launch_copy<CODE, 32>(append, k, ld_k, v, ld_v, p, stream);
    case 64: return launch_copy<CODE, 64>(append, k, ld_k, v, ld_v, p, stream);
    case 128: return launch_copy<CODE, 128>(append, k, ld_k, v, ld_v, p, stream);
    case 256: return launch_copy<CODE, 256>(append, k, ld_k, v, ld_v, p, stream);
  }
  return fail(TFX_ERR_UNSUPPORTED, "paged cache: head_dim %d", head_dim);
}

int launch_copy_code(bool append, const tfx_paged_cache* c, __half* k, int64_t ld_k, __half* v,
                     int64_t ld_v, const Paged& p, cudaStream_t stream) {
  switch (c->dtype) {
    case TFX_CACHE_F16:
      return launch_copy_hd<kCodeF16>(append, c->head_dim, k, ld_k, v, ld_v, p, stream);
    case TFX_CACHE_INT8:
      return launch_copy_hd<kCodeI8>(append, c->head_dim, k, ld_k, v, ld_v, p, stream);
    default:
      return launch_copy_hd<kCodeE4M3>(append, c->head_dim, k, ld_k, v, ld_v, p, stream);
  }
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Checks shared by the two copies; packed rows of width kv_heads * head_dim.
int check_copy(const char* fn, const void* k, int64_t ld_k, const void* v, int64_t ld_v,
               const tfx_paged_cache* cache, const tfx_paged_batch* batch, Paged* p) {
  int st = check_paged(fn, cache, batch, p);
  if (st != TFX_OK) return st;
  if (k == nullptr || v == nullptr) return fail(TFX_ERR_INVALID_ARGUMENT, "%s: null tensor", fn);
  const int64_t width = static_cast<int64_t>(cache->kv_heads) * cache->head_dim;
  if (ld_k < width || ld_v < width)
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: leading dimension smaller than kv_heads*head_dim",
                fn);
  if (!aligned(k, 16) || !aligned(v, 16) || ld_k % 8 != 0 || ld_v % 8 != 0)
    return fail(TFX_ERR_MISALIGNED,
                "%s: pointers 16-byte aligned and leading dims multiples of 8 needed", fn);
  return TFX_OK;
}

}  // namespace

int check_paged(const char* fn, const tfx_paged_cache* c, const tfx_paged_batch* b, Paged* p) {
  if (c == nullptr || b == nullptr)
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: null cache or batch", fn);
  if (c->k == nullptr || c->v == nullptr || b->page_table == nullptr ||
      b->query_start == nullptr || b->kv_len == nullptr)
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: null cache, page_table, query_start or kv_len", fn);
  if (c->dtype != TFX_CACHE_F16 && c->dtype != TFX_CACHE_INT8 && c->dtype != TFX_CACHE_E4M3)
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: dtype %d is not a tfx_cache_dtype", fn, c->dtype);
  if (c->num_pages <= 0 || c->kv_heads <= 0 || b->batch <= 0 || b->max_pages <= 0 ||
      b->num_tokens < 0 || b->max_query_len < 0 || b->max_kv_len < 0)
    return fail(TFX_ERR_INVALID_ARGUMENT,
                "%s: num_pages, kv_heads, batch and max_pages must be positive, lengths not "
                "negative", fn);
  const int hd = c->head_dim, ps = c->page_size;
  if (hd != 8 && hd != 16 && hd != 32 && hd != 64 && hd != 128 && hd != 256)
    return fail(TFX_ERR_UNSUPPORTED, "%s: head_dim %d not in {8,16,32,64,128,256}", fn, hd);
  if (c->dtype != TFX_CACHE_F16 && hd < 16)
    return fail(TFX_ERR_UNSUPPORTED, "%s: 8-bit caches need head_dim >= 16", fn);
  if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256)
    return fail(TFX_ERR_UNSUPPORTED, "%s: page_size %d not in {16,32,64,128,256}", fn, ps);
  if (static_cast<int64_t>(b->max_pages) * ps > (1LL << 30))
    return fail(TFX_ERR_UNSUPPORTED, "%s: max_pages * page_size exceeds 2^30 positions", fn);
  if (b->batch > 65535 || c->kv_heads > 65535)
    return fail(TFX_ERR_UNSUPPORTED, "%s: batch and kv_heads must be <= 65535", fn);
  if (static_cast<int64_t>(b->num_tokens) * c->kv_heads > 0x7fffffffLL - kThreads)
    return fail(TFX_ERR_UNSUPPORTED, "%s: num_tokens * kv_heads exceeds 2^31", fn);
  if (b->table_stride < b->max_pages)
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: table_stride smaller than max_pages", fn);
  if (c->page_stride < hd || c->token_stride < hd || c->head_stride < hd)
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: cache strides must be at least head_dim", fn);
  const bool quant = c->dtype != TFX_CACHE_F16;
  if (quant && (c->k_scale == nullptr || c->v_scale == nullptr))
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: 8-bit caches need k_scale and v_scale", fn);
  const int64_t eb = quant ? 1 : 2;
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->page_stride * eb % 16 != 0 ||
      c->token_stride * eb % 16 != 0 || c->head_stride * eb % 16 != 0)
    return fail(TFX_ERR_MISALIGNED, "%s: k and v 16-byte aligned, strides multiples of 16 bytes",
                fn);
  if (!aligned(b->page_table, 4) || !aligned(b->query_start, 4) || !aligned(b->kv_len, 4) ||
      (quant && (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))))
    return fail(TFX_ERR_MISALIGNED, "%s: int32 and scale arrays must be 4-byte aligned", fn);
  p->k = c->k;
  p->v = c->v;
  p->k_scale = quant ? c->k_scale : nullptr;
  p->v_scale = quant ? c->v_scale : nullptr;
  p->page_stride = c->page_stride;
  p->token_stride = c->token_stride;
  p->head_stride = c->head_stride;
  p->num_pages = c->num_pages;
  p->page_shift = ps == 16 ? 4 : ps == 32 ? 5 : ps == 64 ? 6 : ps == 128 ? 7 : 8;
  p->kv_heads = c->kv_heads;
  p->max_pages = b->max_pages;
  p->table = b->page_table;
  p->table_stride = b->table_stride;
  p->query_start = b->query_start;
  p->kv_len = b->kv_len;
  p->batch = b->batch;
  p->num_tokens = b->num_tokens;
  return TFX_OK;
}

}  // namespace tfx

using namespace tfx;

extern "C" {

int tfx_paged_append(const tfx_half* k, int64_t ld_k, const tfx_half* v, int64_t ld_v,
                     const tfx_paged_cache* cache, const tfx_paged_batch* batch,
                     tfx_stream_t stream) {
  fail(TFX_OK, "%s", "");
  Paged p;
  const int st = check_copy("tfx_paged_append", k, ld_k, v, ld_v, cache, batch, &p);
  if (st != TFX_OK || p.num_tokens == 0) return st;
  return launch_copy_code(true, cache, reinterpret_cast<__half*>(const_cast<tfx_half*>(k)), ld_k,
                          reinterpret_cast<__half*>(const_cast<tfx_half*>(v)), ld_v, p,
                          reinterpret_cast<cudaStream_t>(stream));
}

int tfx_paged_read(const tfx_paged_cache* cache, const tfx_paged_batch* batch, tfx_half* k_out,
                   int64_t ld_k, tfx_half* v_out, int64_t ld_v, tfx_stream_t stream) {
  fail(TFX_OK, "%s", "");
  Paged p;
  const int st = check_copy("tfx_paged_read", k_out, ld_k, v_out, ld_v, cache, batch, &p);
  if (st != TFX_OK || p.num_tokens == 0) return st;
  return launch_copy_code(false, cache, reinterpret_cast<__half*>(k_out), ld_k,
                          reinterpret_cast<__half*>(v_out), ld_v, p,
                          reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
