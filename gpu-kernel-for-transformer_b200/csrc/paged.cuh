// Shared by the paged KV cache's kernels: the cache and the batch as the
// kernels take them, lookups that stay in bounds whatever the device arrays
// hold, and the conversions between 8-bit codes and fp16.
#pragma once

#include <cuda_fp8.h>

#include "internal.h"
#include "ptx.cuh"

namespace tfx {

// tfx_cache_dtype as template arguments.
constexpr int kCodeF16 = TFX_CACHE_F16, kCodeI8 = TFX_CACHE_INT8, kCodeE4M3 = TFX_CACHE_E4M3;

constexpr int code_bytes(int code) { return code == kCodeF16 ? 2 : 1; }

// Kernel parameter: tfx_paged_cache and tfx_paged_batch in one.
struct Paged {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t page_stride, token_stride, head_stride;  // elements
  int num_pages, page_shift, kv_heads;
  int max_pages;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* query_start;
  const int32_t* kv_len;
  int batch, num_tokens;
};

// Checks a cache and a batch and fills the kernel parameter (paged_cache.cu).
int check_paged(const char* fn, const tfx_paged_cache* cache, const tfx_paged_batch* batch,
                Paged* p);

// Whether `rows` fp16 rows of `width` elements at a (row pitch ld_a) and at b share
// an element.
bool rows_overlap(const void* a, int64_t ld_a, const void* b, int64_t ld_b, int64_t rows,
                  int64_t width);

// One sequence of the batch, clamped: rows [row0, row0 + n) of the packed
// tensors at positions pos0 + i; len: keys that may be looked up.
struct PagedSeq {
  int row0, n, pos0, len;
};

__device__ __forceinline__ PagedSeq paged_seq(const Paged& p, int b) {
  PagedSeq s;
  s.row0 = min(max(p.query_start[b], 0), p.num_tokens);
  s.n = min(max(p.query_start[b + 1], s.row0), p.num_tokens) - s.row0;
  const int len = min(max(p.kv_len[b], 0), 1 << 30);
  s.pos0 = len - s.n;
  s.len = min(len, p.max_pages << p.page_shift);  // <= 2^30, checked on the host
  return s;
}

// The sequence that owns packed row `row` (the last b with query_start[b] <=
// row), or -1 behind the last one.
__device__ __forceinline__ int paged_seq_of_row(const Paged& p, int row) {
  if (row >= p.query_start[p.batch]) return -1;
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.query_start[mid] <= row) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Page of position pos of sequence b, or -1 when it has none.
__device__ __forceinline__ int paged_page(const Paged& p, int b, int pos) {
  if (pos < 0 || (pos >> p.page_shift) >= p.max_pages) return -1;
  const int page = p.table[b * p.table_stride + (pos >> p.page_shift)];
  return page >= 0 && page < p.num_pages ? page : -1;
}

__device__ __forceinline__ int64_t paged_offset(const Paged& p, int page, int pos) {
  return page * p.page_stride + (pos & ((1 << p.page_shift) - 1)) * p.token_stride;
}

__device__ __forceinline__ int64_t paged_scale_offset(const Paged& p, int page, int head, int pos) {
  return ((static_cast<int64_t>(page) * p.kv_heads + head) << p.page_shift) +
         (pos & ((1 << p.page_shift) - 1));
}

// ------------------------------------------------------- codes -> fp16 pairs
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// Two e4m3 codes (low or high 16 bits) -> two fp16, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
      : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ uint32_t e4m3x2_hi_to_h2(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}"
      : "=r"(r) : "r"(x));
  return r;
}

// Bytes (I, J) of four codes as an fp16 pair, exact. int8: with the sign bit
// flipped a code is u = code + 128; the fp16 with high byte 0x64 and low byte
// u is 1024 + u, and 1024 + u - 1152 = code.
template <int CODE, int I, int J>
__device__ __forceinline__ uint32_t codes_to_h2(uint32_t x) {
  if constexpr (CODE == kCodeI8) {
    const uint32_t u = __byte_perm(x ^ 0x80808080u, 0x64646464u, 0x4040 | (J << 8) | I);
    return h2_bits(__hsub2(bits_h2(u), bits_h2(0x64806480u)));
  } else {
    if constexpr (I == 0 && J == 1) return e4m3x2_to_h2(x);
    if constexpr (I == 2 && J == 3) return e4m3x2_hi_to_h2(x);
    return e4m3x2_to_h2(__byte_perm(x, 0u, 0x4400 | (J << 4) | I));
  }
}

// ------------------------------------------------- scales of cached values
// 8 bit: the second product takes a key's weight times its value's scale, in fp16,
// and one scale may be any power of two away from another. So the scale is an
// exponent, added to the key's score in the log2 domain, and a row's running maximum
// is that of these sums: what is rounded is relative to the largest weight * scale that
// the row itself sees, whatever other keys and rows hold. The sum of weights takes each
// over its scale. (Weights over one unit for all scales of a CTA lost values of 0.01
// beside a token of 65504, seen or not. prompt_parts_grouped_int8: 722 us with the unit,
// 702 so; 758 with the weights first, done again where one has outgrown the reference.)
//
// log2 of a scale, at least -40: values of smaller scales (448 * 2^-40 = 4e-10 at most)
// are nothing in fp16, and a key whose values are zeros (scale 0) needs a weight in
// the sum still. NaN for a scale that is negative or NaN, and +inf for +inf, so that
// a row which sees one is NaN.
__device__ __forceinline__ float value_scale_log2(float scale) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;\n\tmax.NaN.f32 %0, %0, %2;" : "=&f"(y) : "f"(scale), "f"(-40.0f));
  return y;
}
// One over a scale: finite and above 0 whatever it is (a masked key's may be anything).
__device__ __forceinline__ float value_scale_inverse(float scale) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fminf(fmaxf(scale, 0x1p-40f), 0x1p100f)));
  return y;
}
// A scale that makes its token NaN for the rows that see it.
__device__ __forceinline__ bool value_scale_bad(float scale) {
  return !(scale >= 0.f && scale < INFINITY);
}

// True where either fp16 of the pair is an infinity or NaN.
__device__ __forceinline__ bool h2_not_finite(uint32_t w) {
  return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
}

// Clears the halves that are infinities or NaN; true if there was one.
__device__ __forceinline__ bool h2_clear(uint32_t& w) {
  if (!h2_not_finite(w)) return false;
  if ((w & 0x7c00u) == 0x7c00u) w &= 0xffff0000u;
  if ((w & 0x7c000000u) == 0x7c000000u) w &= 0xffffu;
  return true;
}

// Four elements of a row over the sum of its weights; no key seen: zeros (a
// sum that is NaN stays).
__device__ __forceinline__ void store_row4(__half* dst, float4 x, float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(pack_half2(x.x * inv, x.y * inv), pack_half2(x.z * inv, x.w * inv));
}

// One cached value (fp16 bits for kCodeF16, else a code and its scale).
template <int CODE>
__device__ __forceinline__ float paged_value(const void* base, int64_t at, float scale) {
  if constexpr (CODE == kCodeF16) return __half2float(static_cast<const __half*>(base)[at]);
  if constexpr (CODE == kCodeI8) return static_cast<const int8_t*>(base)[at] * scale;
  if constexpr (CODE == kCodeE4M3)
    return static_cast<float>(static_cast<const __nv_fp8_e4m3*>(base)[at]) * scale;
}

// ------------------------------------------------------------- attention
// One attention call as its kernels take it. Sequences with more than
// tc_rows rows (new tokens x group) belong to the tcgen05 kernel, the others to
// the mma.sync kernel. splits_rows (or splits_tc) CTAs share the keys of a row
// block, kps (kps_tc) keys each, a multiple of 256; if more than one, their
// unnormalised results go to part_o [token][q_head][split][head_dim] with the (max,
// sum) in part_ml (room for `splits`, the larger number), and a third kernel joins
// them.
struct PagedAttn {
  const __half* q;
  int64_t ld_q;
  __half* out;
  int64_t ld_out;
  int group;  // query heads per key/value head
  float scale_log2;
  int causal;
  int q_len;  // tokens of a sequence that are attended: max_query_len
  int tc_rows;
  int splits, splits_rows, splits_tc, kps, kps_tc;
  int cluster;  // mma.sync kernel: CTAs of a cluster that share a row block's keys; 0: splits
  float* part_o;
  float2* part_ml;
};

// The sequence as attention takes it: its first q_len tokens (which stay where they are).
__device__ __forceinline__ PagedSeq paged_attn_seq(const Paged& p, const PagedAttn& a, int b) {
  PagedSeq s = paged_seq(p, b);
  s.n = min(s.n, a.q_len);
  return s;
}

__device__ __forceinline__ bool paged_is_tc(const PagedAttn& a, const PagedSeq& s) {
  return s.n * a.group > a.tc_rows;  // below 2^31: checked on the host
}

__device__ __forceinline__ int paged_split_keys(const PagedAttn& a, const PagedSeq& s) {
  return paged_is_tc(a, s) ? a.kps_tc : a.kps;
}

__device__ __forceinline__ int paged_split_count(const PagedAttn& a, const PagedSeq& s) {
  return paged_is_tc(a, s) ? a.splits_tc : a.splits_rows;
}

// Keys are split for this sequence (its partial results are joined later);
// otherwise split 0 holds all of them and writes the rows itself.
__device__ __forceinline__ bool paged_is_split(const PagedAttn& a, const PagedSeq& s) {
  return paged_split_count(a, s) > 1 && s.len > paged_split_keys(a, s);
}

// End of the keys of a split (the last one takes whatever is left: max_kv_len may
// have been less than a sequence's length).
__device__ __forceinline__ int paged_split_end(const PagedAttn& a, const PagedSeq& s, int split,
                                               int k_begin) {
  return split == paged_split_count(a, s) - 1 ? s.len
                                              : min(s.len, k_begin + paged_split_keys(a, s));
}

// Rows of a CTA of the mma.sync kernel for rows = max_query_len * group.
int paged_rows_block(int head_dim, int64_t rows);
template <int CODE>
int launch_paged_rows(const Paged& p, const PagedAttn& a, int head_dim, int block_rows,
                      bool mixed, int64_t rows, cudaStream_t stream);
// tokens: max_query_len.
template <int CODE>
int launch_paged_tc(const tfx_paged_cache* cache, const Paged& p, const PagedAttn& a,
                    int64_t tokens, cudaStream_t stream);

}  // namespace tfx
