// Writing new tokens into a paged KV cache (optionally in 8 bits with a scale
// per token and head) and reading them back as fp16.
//
// Both are one pass over memory. A CTA takes a few consecutive tokens: its first
// threads look up where each lives (sequence, page, slot) into shared memory,
// then a thread handles 8 consecutive elements (16 bytes of fp16) of one
// (token, head) row of K and of V at a time, two such pieces in flight. The
// head_dim / 8 threads of a row sit in one warp and reduce max|x| with shuffles.
//
// Quantisation rounds x / s as if in exact arithmetic, so that a code is the
// nearest one even when the quotient lies within an fp32 rounding of the
// border between two codes. x times a number just below 1/s and x times one just
// above give the same code, which is then that of x / s, for all but a few
// elements in 10^5; there the 8 elements of the thread are done again:
//  int8: c = rint(x * (1/s)) is the nearest code or, next to a border, its
//        neighbour; e = fma(-c, s, x) is x - c*s exactly (x has 11 bits, and
//        near a border ulp(s) <= ulp(x), so e has at most 24), and |e| against
//        s/2 tells which.
//  e4m3: the quotient is divided out and rounded to odd, which rounds on
//        correctly.
#include "paged.cuh"

namespace tfx {
namespace {

constexpr int kThreads = 256;

// The codes of x, exact (see the file's comment).
__device__ __forceinline__ int exact_i8(float x, float inv, float s, float half_s) {
  float c = rintf(x * inv);
  const float e = fmaf(-c, s, x);
  if (fabsf(e) > half_s || (fabsf(e) == half_s && (static_cast<int>(c) & 1)))
    c += copysignf(1.0f, e);
  return static_cast<int>(fminf(fmaxf(c, -127.0f), 127.0f));
}

__device__ __forceinline__ float exact_quot(float x, float s) {  // rounded to odd
  const float ax = fabsf(x), q = __fdiv_rn(ax, s), r = fmaf(-q, s, ax);
  uint32_t odd = __float_as_uint(q);
  if (r < 0.f) --odd;
  if (r != 0.f) odd |= 1u;
  return copysignf(__uint_as_float(odd), x);
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
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

// x / 127 or x / 448, correctly rounded: a product with the rounded reciprocal and
// one correction by the exact remainder (Markstein's method; equal to the division for
// every fp16).
template <int CODE>
__device__ __forceinline__ float scale_of(float top) {
  constexpr float kTop = CODE == kCodeI8 ? 127.0f : 448.0f, kInv = 1.0f / kTop;
  const float q = top * kInv;
  return fmaf(fmaf(-q, kTop, top), kInv, q);
}

// Eight codes of a row whose max|x| has the fp16 bits `top`; *scale gets s.
template <int CODE>
__device__ __forceinline__ uint2 quantise(const uint4& x, uint32_t top, float* scale) {
  if (top >= 0x7c00u) {
    *scale = __uint_as_float(0x7fc00000u);
    return make_uint2(0u, 0u);
  }
  const float s = scale_of<CODE>(__half2float(__ushort_as_half(static_cast<unsigned short>(top))));
  *scale = s;
  if (top == 0u) return make_uint2(0u, 0u);
  // 1/s lies between lo and hi (the approximation is within 2^-23), so the quotient
  // rounds to the code that x * lo and x * hi have in common.
  constexpr float kWide = CODE == kCodeI8 ? 1.f / (1 << 22) : 1.f / (1 << 21);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const float lo = inv * (1.f - kWide), hi = inv * (1.f + kWide);
  const uint64_t lo2 = f2_pack(lo, lo), hi2 = f2_pack(hi, hi);
  float f[8];
  uint64_t f2[4];
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = __half22float2(bits_h2(w[i]));
    f[2 * i] = y.x;
    f[2 * i + 1] = y.y;
    f2[i] = f2_pack(y.x, y.y);
  }
  uint32_t out[2], differ = 0;
  if constexpr (CODE == kCodeI8) {
    const uint64_t round2 = f2_pack(12582912.0f, 12582912.0f);  // 1.5 * 2^23: the low byte is the code
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a0, a1, b0, b1;
      f2_unpack(f2_fma(f2[i], lo2, round2), a0, a1);
      f2_unpack(f2_fma(f2[i], hi2, round2), b0, b1);
      c[2 * i] = __float_as_uint(a0);
      c[2 * i + 1] = __float_as_uint(a1);
      differ |= c[2 * i] ^ __float_as_uint(b0);
      differ |= c[2 * i + 1] ^ __float_as_uint(b1);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      out[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040),
                           __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
    if (differ != 0u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = exact_i8(f[i], inv, s, 0.5f * s) & 0xff;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        out[i] = c[4 * i] | (c[4 * i + 1] << 8) | (c[4 * i + 2] << 16) | (c[4 * i + 3] << 24);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float a[4], b[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f2_unpack(f2_mul(f2[2 * i + j], lo2), a[2 * j], a[2 * j + 1]);
        f2_unpack(f2_mul(f2[2 * i + j], hi2), b[2 * j], b[2 * j + 1]);
      }
      out[i] = e4m3x2(a[0], a[1]) | (e4m3x2(a[2], a[3]) << 16);
      differ |= out[i] ^ (e4m3x2(b[0], b[1]) | (e4m3x2(b[2], b[3]) << 16));
    }
    if (differ != 0u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = exact_quot(f[i], s);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        out[i] = e4m3x2(f[4 * i], f[4 * i + 1]) | (e4m3x2(f[4 * i + 2], f[4 * i + 3]) << 16);
    }
  }
  return make_uint2(out[0], out[1]);
}

// Where a CTA's tokens live: element offset of the token's first head in k and
// v, and of its first head's scale; -1: no page; -2: a row of no sequence.
constexpr int kMostTokens = 64;
struct Places {
  int64_t at[kMostTokens];
  int64_t scale[kMostTokens];
};

__device__ __forceinline__ void look_up(const Paged& p, int t0, int tokens, Places& out) {
  for (int i = threadIdx.x; i < tokens; i += kThreads) {
    const int t = t0 + i, b = paged_seq_of_row(p, t);
    int64_t at = -2, scale = 0;
    if (b >= 0) {
      const PagedSeq s = paged_seq(p, b);
      if (t >= s.row0 && t < s.row0 + s.n) {
        const int pos = s.pos0 + (t - s.row0), page = paged_page(p, b, pos);
        at = page < 0 ? -1 : paged_offset(p, page, pos);
        scale = page < 0 ? 0 : paged_scale_offset(p, page, 0, pos);
      }
    }
    out.at[i] = at;
    out.scale[i] = scale;
  }
  __syncthreads();
}

// One 8-element piece of the CTA's tokens: piece i is chunk i % CH of row i / CH,
// a row being (token, head). `div`: 2^32 / kv_heads + 1, or 0 for one head (exact:
// rows of a CTA times heads stay below 2^32).
struct Piece {
  int token, head, chunk;
};
template <int CH>
__device__ __forceinline__ Piece piece_of(int i, int heads, uint32_t div) {
  const int row = i / CH;
  const int token = div == 0u ? row : static_cast<int>(__umulhi(static_cast<uint32_t>(row), div));
  return Piece{token, row - token * heads, i % CH};
}

template <int CODE, int HD>
__global__ void __launch_bounds__(kThreads)
    paged_append_kernel(const __half* __restrict__ k, int64_t ld_k, const __half* __restrict__ v,
                        int64_t ld_v, const __grid_constant__ Paged p, int cta_tokens,
                        uint32_t div) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int CH = HD / 8, U = 2;
  __shared__ Places places;
  const int t0 = blockIdx.x * cta_tokens, tokens = min(cta_tokens, p.num_tokens - t0);
  look_up(p, t0, tokens, places);
  const int pieces = tokens * p.kv_heads * CH;
  const int64_t head_scale = static_cast<int64_t>(1) << p.page_shift;
  // (whole warps go through the loop: the rows' threads reduce together)
  for (int i0 = threadIdx.x; i0 - static_cast<int>(threadIdx.x) < pieces; i0 += U * kThreads) {
    Piece pc[U];
    int64_t at[U];
    uint4 xk[U], xv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads;
      pc[u] = piece_of<CH>(min(i, pieces - 1), p.kv_heads, div);
      at[u] = i < pieces ? places.at[pc[u].token] : -1;
      xk[u] = xv[u] = make_uint4(0, 0, 0, 0);
      if (at[u] >= 0) {
        const int64_t t = t0 + pc[u].token;
        xk[u] = __ldcs(reinterpret_cast<const uint4*>(k + t * ld_k + pc[u].head * HD) + pc[u].chunk);
        xv[u] = __ldcs(reinterpret_cast<const uint4*>(v + t * ld_v + pc[u].head * HD) + pc[u].chunk);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t to = at[u] + pc[u].head * p.head_stride + pc[u].chunk * 8;
      if constexpr (CODE == kCodeF16) {
        if (at[u] >= 0) {
          *reinterpret_cast<uint4*>(static_cast<__half*>(p.k) + to) = xk[u];
          *reinterpret_cast<uint4*>(static_cast<__half*>(p.v) + to) = xv[u];
        }
      } else {
        const uint32_t tk = row_absmax<CH>(xk[u]), tv = row_absmax<CH>(xv[u]);  // every lane
        if (at[u] >= 0) {
          float sk, sv;
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.k) + to) = quantise<CODE>(xk[u], tk, &sk);
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.v) + to) = quantise<CODE>(xv[u], tv, &sv);
          if (pc[u].chunk == 0) {
            const int64_t so = places.scale[pc[u].token] + pc[u].head * head_scale;
            p.k_scale[so] = sk;
            p.v_scale[so] = sv;
          }
        }
      }
    }
  }
}

// Eight codes times the scale, in fp32 and then rounded to fp16. (Two roundings, which
// differ from one where the product lies within 2^-24 of itself of the border between
// two fp16 numbers: by a step of fp16, in about one element of 2^14.)
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
                      const __grid_constant__ Paged p, int cta_tokens, uint32_t div) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int CH = HD / 8, U = 2;
  __shared__ Places places;
  const int t0 = blockIdx.x * cta_tokens, tokens = min(cta_tokens, p.num_tokens - t0);
  look_up(p, t0, tokens, places);
  const int pieces = tokens * p.kv_heads * CH;
  const int64_t head_scale = static_cast<int64_t>(1) << p.page_shift;
  for (int i0 = threadIdx.x; i0 < pieces; i0 += U * kThreads) {
    Piece pc[U];
    int64_t at[U];
    uint4 xk[U], xv[U];  // 8 bit: codes in the first half
    float sk[U], sv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads;
      pc[u] = piece_of<CH>(min(i, pieces - 1), p.kv_heads, div);
      at[u] = i < pieces ? places.at[pc[u].token] : -2;
      xk[u] = xv[u] = make_uint4(0, 0, 0, 0);
      sk[u] = sv[u] = 0.f;
      if (at[u] >= 0) {
        const int64_t from = at[u] + pc[u].head * p.head_stride + pc[u].chunk * 8;
        if constexpr (CODE == kCodeF16) {
          xk[u] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const __half*>(p.k) + from));
          xv[u] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const __half*>(p.v) + from));
        } else {
          const uint2 ck = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.k) + from));
          const uint2 cv = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.v) + from));
          const int64_t so = places.scale[pc[u].token] + pc[u].head * head_scale;
          xk[u] = make_uint4(ck.x, ck.y, 0, 0);
          xv[u] = make_uint4(cv.x, cv.y, 0, 0);
          sk[u] = p.k_scale[so];
          sv[u] = p.v_scale[so];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] == -2) continue;
      if constexpr (CODE != kCodeF16) {
        xk[u] = dequantise<CODE>(make_uint2(xk[u].x, xk[u].y), sk[u]);
        xv[u] = dequantise<CODE>(make_uint2(xv[u].x, xv[u].y), sv[u]);
      }
      const int64_t t = t0 + pc[u].token;
      __stcs(reinterpret_cast<uint4*>(k + t * ld_k + pc[u].head * HD) + pc[u].chunk, xk[u]);
      __stcs(reinterpret_cast<uint4*>(v + t * ld_v + pc[u].head * HD) + pc[u].chunk, xv[u]);
    }
  }
}

template <int CODE, int HD>
int launch_copy(bool append, __half* k, int64_t ld_k, __half* v, int64_t ld_v, const Paged& p,
                cudaStream_t stream) {
  // Tokens of a CTA: about 16384 elements of K, fewer where that leaves SMs idle.
  const int width = p.kv_heads * HD;
  int tokens = width < 16384 ? 16384 / width : 1;
  const int spread = (p.num_tokens + 4 * num_sms() - 1) / (4 * num_sms());
  if (tokens > spread) tokens = spread;
  if (tokens > kMostTokens) tokens = kMostTokens;
  const dim3 grid(static_cast<unsigned>((p.num_tokens + tokens - 1) / tokens));
  const uint32_t div =
      p.kv_heads == 1 ? 0u : static_cast<uint32_t>((1ull << 32) / static_cast<uint32_t>(p.kv_heads)) + 1u;
  if (append) {
    launch_pdl(paged_append_kernel<CODE, HD>, grid, dim3(kThreads), 0, stream,
               static_cast<const __half*>(k), ld_k, static_cast<const __half*>(v), ld_v, p, tokens,
               div);
    return check_launch("paged_append_kernel");
  }
  launch_pdl(paged_read_kernel<CODE, HD>, grid, dim3(kThreads), 0, stream, k, ld_k, v, ld_v, p,
             tokens, div);
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

bool rows_overlap(const void* a, int64_t ld_a, const void* b, int64_t ld_b, int64_t rows,
                  int64_t width) {
  if (rows <= 0) return false;
  const int64_t a0 = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a)) / 2;
  const int64_t b0 = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b)) / 2;
  if (a0 + (rows - 1) * ld_a + width <= b0 || b0 + (rows - 1) * ld_b + width <= a0) return false;
  if (ld_a != ld_b) return true;
  const int64_t d = (a0 < b0 ? b0 - a0 : a0 - b0) % ld_a;  // columns apart in a common row
  return d < width || ld_a - d < width;
}

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
      (quant && (!aligned(c->k_scale, 16) || !aligned(c->v_scale, 16))))
    return fail(TFX_ERR_MISALIGNED, "%s: int32 arrays 4-byte, scales 16-byte aligned", fn);
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
  if (st != TFX_OK) return st;
  if (p.k == p.v || (p.k_scale != nullptr && p.k_scale == p.v_scale))
    return fail(TFX_ERR_INVALID_ARGUMENT, "tfx_paged_append: the cache's k and v are one memory");
  if (p.num_tokens == 0) return TFX_OK;
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
  if (rows_overlap(k_out, ld_k, v_out, ld_v, p.num_tokens,
                   static_cast<int64_t>(cache->kv_heads) * cache->head_dim))
    return fail(TFX_ERR_INVALID_ARGUMENT, "tfx_paged_read: k_out and v_out overlap");
  return launch_copy_code(false, cache, reinterpret_cast<__half*>(k_out), ld_k,
                          reinterpret_cast<__half*>(v_out), ld_v, p,
                          reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
