// tfx_paged_attention: host-side checks, the choice of kernel and of the split
// over keys, and the kernel that joins the splits.
#include "paged.cuh"

namespace tfx {
namespace {

// Keys of a split: a multiple of every kernel's round of tiles over its warps.
constexpr int kSplitKeys = 256;
// Sequences with more rows (new tokens x query heads per key/value head) may go
// to the tcgen05 kernel, whose tiles have 128: the wider the head, the more the
// mma.sync kernel's registers cost it. us with 64 and with this many: 64 sequences
// with 1 to 8 new tokens and up to 6000 keys, 8 heads in groups of 8, head_dim 64
// fp16 127 and (32) 136, 128 215 and 191, 256 504 and 308; 32 with 3 at head_dim 256
// (32 rows) 314 and 239.
constexpr int tc_rows(int head_dim) { return 4096 / head_dim; }  // from head_dim 64
// Partial results kept for a call at most, where few splits would do as well.
constexpr int64_t kPartBytes = 128 << 20;

// out[row] = sum over splits of partial O scaled to the common maximum, over
// the sum of their sums. `wpr` warps of the CTA per (token, head) row: one when
// there are few splits (more rows per CTA), four when there are many.
template <int HD>
__global__ void __launch_bounds__(128)
    paged_join_kernel(const __grid_constant__ Paged p, const __grid_constant__ PagedAttn a,
                      int64_t rows, int wpr) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int DL = HD >= 32 ? HD / 32 : 1;  // dims of a lane
  __shared__ float sm[4][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (4 / wpr) + warp / wpr;
  const int part = warp % wpr, heads = p.kv_heads * a.group;
  int n = 0, tok = 0, head = 0;
  if (row < rows) {
    tok = static_cast<int>(row / heads);
    head = static_cast<int>(row % heads);
    const int b = paged_seq_of_row(p, tok);
    if (b >= 0) {
      const PagedSeq s = paged_seq(p, b);
      if (paged_is_split(a, s) && tok >= s.row0 && tok < s.row0 + s.n) {
        const int lim = a.causal ? min(s.len, max(0, s.pos0 + (tok - s.row0) + 1)) : s.len;
        n = min(a.splits, (lim + paged_split_keys(a, s) - 1) / paged_split_keys(a, s));
        if (n == 0) n = -1;  // a split sequence's row that sees no key
      }
    }
  }
  const int64_t base = row * a.splits;
  float m = -INFINITY, acc[DL], l = 0.f;
#pragma unroll
  for (int e = 0; e < DL; ++e) acc[e] = 0.f;
  for (int s = lane; s < n; s += 32) m = fmaxf(m, a.part_ml[base + s].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  for (int s = 0; s < n; ++s) {
    const float2 ml = a.part_ml[base + s];
    const float f = ml.x == -INFINITY && ml.y == 0.f ? 0.f : fast_exp2(ml.x - m);
    if (f == 0.f && ml.y == 0.f) continue;
    l += f * ml.y;
    if (s % wpr != part) continue;
    const float* src = a.part_o + (base + s) * HD + lane * DL;
    if (HD >= 32 || lane < HD) {
#pragma unroll
      for (int e = 0; e < DL; ++e) acc[e] += f * src[e];
    }
  }
  if (wpr > 1) {
    if (HD >= 32 || lane < HD) {
#pragma unroll
      for (int e = 0; e < DL; ++e) sm[warp][lane * DL + e] = acc[e];
    }
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < 4; ++w)
#pragma unroll
      for (int e = 0; e < DL; ++e)
        if (HD >= 32 || lane < HD) acc[e] += sm[w][lane * DL + e];
  }
  if (n == 0 || (HD < 32 && lane >= HD)) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __half* dst = a.out + static_cast<int64_t>(tok) * a.ld_out + head * HD + lane * DL;
#pragma unroll
  for (int e = 0; e < DL; ++e) dst[e] = __float2half_rn(acc[e] * inv);
}

template <int HD>
int launch_join(const Paged& p, const PagedAttn& a, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(p.num_tokens) * p.kv_heads * a.group;
  const int wpr = a.splits > 16 ? 4 : 1, per_cta = 4 / wpr;
  launch_pdl(paged_join_kernel<HD>, dim3(static_cast<unsigned>((rows + per_cta - 1) / per_cta)),
             dim3(128), 0, stream, p, a, rows, wpr);
  return check_launch("paged_join_kernel");
}

int join_hd(const Paged& p, const PagedAttn& a, int head_dim, cudaStream_t stream) {
  switch (head_dim) {
    case 8: return launch_join<8>(p, a, stream);
    case 16: return launch_join<16>(p, a, stream);
    case 32: return launch_join<32>(p, a, stream);
    case 64: return launch_join<64>(p, a, stream);
    case 128: return launch_join<128>(p, a, stream);
    default: return launch_join<256>(p, a, stream);
  }
}

struct Plan {
  int64_t q, rows;  // new tokens of the longest sequence, and their rows
  int block_rows;   // of the mma.sync kernel
  int tc_rows;      // sequences with more rows go to the tcgen05 kernel
  bool tc, small;   // which kernels run
  int splits, kps, kps_tc, cluster;
  int64_t ml_offset, bytes;  // workspace
};

// Into how many ranges the keys of `blocks` row blocks are cut, for `slots`
// CTAs at a time, each of which costs `start` keys besides its own; `most`
// ranges at most, of `least` keys at least. Sequences are taken to have any
// length up to kv: the work per slot, and behind it the longest range (alone,
// where all CTAs run at once). More than one range costs `join` keys.
int64_t cut(int64_t blocks, int64_t slots, int64_t kv, int64_t start, int64_t join, int64_t least,
            int64_t most, double* cost) {
  int64_t best = 1;
  *cost = 0.;
  for (int64_t n = 1; n <= most; n += n < 8 ? 1 : n / 4) {
    const int64_t keys = (kv + n - 1) / n;
    if (n > 1 && keys < least) break;
    const double waves = static_cast<double>(blocks) * n / slots;
    const double c = (waves <= 1. ? keys + start : waves * (0.55 * keys + start) + keys) +
                     (n > 1 ? join : 0);
    if (n == 1 || c < *cost) {
      best = n;
      *cost = c;
    }
  }
  return best;
}

int round_keys(int64_t kv, int64_t parts) {
  const int64_t keys = (kv + parts - 1) / parts;
  return static_cast<int>((keys + kSplitKeys - 1) / kSplitKeys * kSplitKeys);
}

// How the work is cut: which kernel, row blocks, and ranges of keys where the
// blocks alone leave SMs idle.
Plan make_plan(const tfx_paged_cache* c, const tfx_paged_batch* b, int q_heads) {
  Plan pl{};
  const int group = q_heads / c->kv_heads, hd = c->head_dim;
  pl.q = b->max_query_len < b->num_tokens ? b->max_query_len : b->num_tokens;
  pl.rows = pl.q * group;
  const bool quant = c->dtype != TFX_CACHE_F16;
  const int64_t pairs = static_cast<int64_t>(b->batch) * c->kv_heads;
  int64_t kv = static_cast<int64_t>(b->max_pages) * c->page_size;
  if (b->max_kv_len < kv) kv = b->max_kv_len;
  if (kv < 1) kv = 1;

  // tcgen05: one CTA to an SM, whose start costs about as much as 768 keys.
  // Whole waves of equal CTAs, and what the partial results of every row cost
  // (written and read once, in units of a key's time): cutting pays where there
  // are few row blocks.
  const int tokens = group <= 128 ? (hd == 256 ? 1 : 2) * (128 / group) : 1;
  const int64_t tc_blocks = pairs * ((pl.q + tokens - 1) / tokens);
  int64_t tc_parts = 1;
  double tc_cost = 0., tc_keys = 0.;
  for (int64_t n = 1; n <= 16 && (n == 1 || (kv + n - 1) / n >= 1024); ++n) {
    const double waves = static_cast<double>((tc_blocks * n + num_sms() - 1) / num_sms());
    const double join = n > 1 ? 500. + 1e-5 * 8. * b->num_tokens * q_heads * n * hd : 0.;
    const double cost = waves * ((kv + n - 1) / n + 768) + join;
    if (n == 1 || cost < tc_cost) {
      tc_parts = n;
      tc_cost = cost;
      tc_keys = waves * ((kv + n - 1) / n + 300);
    }
  }
  pl.kps_tc = round_keys(kv, tc_parts);

  // Which kernel: more than tc_rows rows, and enough work. Times in ns, fitted to
  // both kernels at 1 to 64 sequences of 2 000 to 30 000 tokens, 8 heads, 16 to 128
  // rows; e.g. 128 rows, head_dim 64, fp16: 1 x 2 000 26 us tcgen05, 13 mma.sync;
  // 1 x 30 000 40 and 56; 16 x 3 000 47 and 108; 64 x 4 000 210 and 382.
  pl.tc = hd >= 64 && group <= 128 && pl.rows > tc_rows(hd);
  if (pl.tc) {
    const int i = hd == 64 ? 0 : hd == 128 ? 1 : 2;
    constexpr double kTcKey[2][3] = {{11., 13., 16.}, {12.5, 13., 16.}};
    constexpr double kRowsKey[2][3] = {{.05, .08, .16}, {.06, .09, .18}};  // of 32 rows
    const double tc_ns = 10e3 + tc_keys * kTcKey[quant][i];
    const double rows_ns =
        6e3 + static_cast<double>(pairs) * ((pl.rows + 31) / 32) * kv * kRowsKey[quant][i];
    pl.tc = tc_ns < rows_ns;
  }
  pl.small = !pl.tc || b->batch > 1;  // a single sequence has all the rows
  pl.tc_rows = !pl.tc ? 0x7fffffff : pl.small ? tc_rows(hd) : 0;

  // mma.sync: CTAs to an SM by registers and shared memory; a start costs about
  // as much as 400 keys, a second launch to join as much as 512 and one for every
  // 100 rows that it looks at (beside the tcgen05 kernel: all of its rows).
  const int64_t small_rows = pl.rows < pl.tc_rows ? pl.rows : pl.tc_rows;
  pl.block_rows = paged_rows_block(hd, small_rows);
  const int row_bytes = hd * (quant ? 1 : 2);
  const int64_t slots = num_sms() * (row_bytes >= 512 ? 1 : pl.block_rows >= 32 ? 2 :
                                     pl.block_rows == 16 || row_bytes == 256 ? 3 : 4);
  const int64_t blocks = pairs * ((small_rows + pl.block_rows - 1) / pl.block_rows);
  double alone = 0., joined = 0.;
  const int64_t share = cut(blocks, slots, kv, 400, 0, 128, 8, &alone);
  const int64_t all_rows = static_cast<int64_t>(b->num_tokens) * q_heads;
  int64_t most = kPartBytes / ((all_rows + 1) * (hd + 2) * 4);
  most = most < 1 ? 1 : most > 1024 ? 1024 : most;
  const int64_t parts = cut(blocks, slots, kv, 400, 512 + all_rows / 100, kSplitKeys, most, &joined);
  // (CTAs of a cluster wait for one another at its end: for one wave only)
  if (!pl.tc && alone <= joined && (share == 1 || 4 * blocks * share <= 5 * slots)) {
    pl.cluster = share > 1 ? static_cast<int>(share) : 0;
    pl.kps = round_keys(kv, 1);
  } else {
    pl.kps = round_keys(kv, parts);
  }
  int64_t least = pl.tc ? pl.kps_tc : pl.kps;
  if (pl.small && pl.kps < least) least = pl.kps;
  pl.splits = static_cast<int>((kv + least - 1) / least);
  if (pl.cluster > 0) pl.splits = 1;
  if (pl.splits > 1) {
    const int64_t part_rows = static_cast<int64_t>(b->num_tokens) * q_heads * pl.splits;
    pl.ml_offset = part_rows * hd;  // floats; head_dim is even: float2 stays aligned
    pl.bytes = (part_rows * (hd + 2) * 4 + 255) / 256 * 256;
  }
  return pl;
}

template <int CODE>
int launch_attention_code(const tfx_paged_cache* c, const Paged& p, const PagedAttn& a,
                          const Plan& pl, cudaStream_t stream) {
  int st = TFX_OK;
  if (pl.tc) st = launch_paged_tc<CODE>(c, p, a, pl.q, stream);
  if (st == TFX_OK && pl.small)
    st = launch_paged_rows<CODE>(p, a, c->head_dim, pl.block_rows, pl.tc,
                                 pl.rows < pl.tc_rows ? pl.rows : pl.tc_rows, stream);
  return st;
}

int check_heads(const char* fn, const tfx_paged_cache* c, const tfx_paged_batch* b, int q_heads) {
  if (q_heads <= 0 || q_heads % c->kv_heads != 0)
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: q_heads %d is not a multiple of kv_heads %d", fn,
                q_heads, c->kv_heads);
  if (static_cast<int64_t>(b->num_tokens) * q_heads > 0x7fffffffLL - 1024)
    return fail(TFX_ERR_UNSUPPORTED, "%s: num_tokens * q_heads exceeds 2^31", fn);
  return TFX_OK;
}

}  // namespace

int paged_rows_block(int head_dim, int64_t rows) {
  // Registers hold 32 rows, 16 at head_dim 256. (64 rows up to head_dim 64 halve
  // the reads of K and V from L2 but leave two CTAs to an SM: 48.9 against 33.1 us
  // for 40 sequences of up to 200 new tokens, 4 heads of 32.)
  const int most = head_dim <= 128 ? 32 : 16;
  const int need = rows <= 8 ? 8 : (rows <= 16 ? 16 : 32);
  return need < most ? need : most;
}

}  // namespace tfx

using namespace tfx;

extern "C" {

int64_t tfx_paged_attention_workspace_bytes(const tfx_paged_cache* cache,
                                            const tfx_paged_batch* batch, int q_heads) {
  fail(TFX_OK, "%s", "");
  const char* fn = "tfx_paged_attention_workspace_bytes";
  Paged p;
  if (check_paged(fn, cache, batch, &p) != TFX_OK ||
      check_heads(fn, cache, batch, q_heads) != TFX_OK)
    return -1;
  return make_plan(cache, batch, q_heads).bytes;
}

int tfx_paged_attention(const tfx_half* q, int64_t ld_q, const tfx_paged_cache* cache,
                        const tfx_paged_batch* batch, tfx_half* out, int64_t ld_out, int q_heads,
                        float scale, int causal, void* workspace, size_t workspace_bytes,
                        tfx_stream_t stream_) {
  fail(TFX_OK, "%s", "");
  const char* fn = "tfx_paged_attention";
  Paged p;
  int st = check_paged(fn, cache, batch, &p);
  if (st == TFX_OK) st = check_heads(fn, cache, batch, q_heads);
  if (st != TFX_OK) return st;
  if (q == nullptr || out == nullptr) return fail(TFX_ERR_INVALID_ARGUMENT, "%s: null tensor", fn);
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!(scale > 0.f) || !(scale_log2 < INFINITY))
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: scale must be positive and finite", fn);
  const int64_t width = static_cast<int64_t>(q_heads) * cache->head_dim;
  if (ld_q < width || ld_out < width)
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: leading dimension smaller than q_heads*head_dim",
                fn);
  if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 16 ||
      ld_q % 8 != 0 || ld_out % 8 != 0)
    return fail(TFX_ERR_MISALIGNED,
                "%s: pointers 16-byte aligned and leading dims multiples of 8 needed", fn);
  if (rows_overlap(q, ld_q, out, ld_out, batch->num_tokens, width))
    return fail(TFX_ERR_INVALID_ARGUMENT, "%s: out must not overlap q", fn);
  const Plan pl = make_plan(cache, batch, q_heads);
  if (pl.bytes > 0) {
    if (workspace == nullptr) return fail(TFX_ERR_INVALID_ARGUMENT, "%s: null workspace", fn);
    if (reinterpret_cast<uintptr_t>(workspace) % 256)
      return fail(TFX_ERR_MISALIGNED, "%s: workspace 256-byte alignment", fn);
    if (workspace_bytes < static_cast<size_t>(pl.bytes))
      return fail(TFX_ERR_WORKSPACE, "%s: workspace %zu < required %lld bytes", fn,
                  workspace_bytes, static_cast<long long>(pl.bytes));
  }
  if (pl.rows == 0) return TFX_OK;  // no new token
  PagedAttn a{};
  a.q = reinterpret_cast<const __half*>(q);
  a.ld_q = ld_q;
  a.out = reinterpret_cast<__half*>(out);
  a.ld_out = ld_out;
  a.group = q_heads / cache->kv_heads;
  a.scale_log2 = scale_log2;
  a.causal = causal != 0;
  a.splits = pl.splits;
  a.kps = pl.kps;
  a.kps_tc = pl.kps_tc;
  a.tc_rows = pl.tc_rows;
  a.cluster = pl.cluster;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + pl.ml_offset);
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  switch (cache->dtype) {
    case TFX_CACHE_F16: st = launch_attention_code<kCodeF16>(cache, p, a, pl, stream); break;
    case TFX_CACHE_INT8: st = launch_attention_code<kCodeI8>(cache, p, a, pl, stream); break;
    default: st = launch_attention_code<kCodeE4M3>(cache, p, a, pl, stream); break;
  }
  if (st != TFX_OK || pl.splits == 1) return st;
  return join_hd(p, a, cache->head_dim, stream);
}

}  // extern "C"
