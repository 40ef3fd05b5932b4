// tfx_paged_attention: host-side checks, the choice of kernel and of the split
// over keys, and the kernel that joins the splits.
#include "paged.cuh"

namespace tfx {
namespace {

// Keys of a split: a multiple of every kernel's tile and of the mma.sync kernel's round of
// tiles over its warps (but for its six warps at 512-byte rows, 96 keys a round).
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

// N consecutive floats of a lane, aligned to as many.
template <int N>
__device__ __forceinline__ void load_floats(const float* src, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(src + i);
      v[i] = x.x;
      v[i + 1] = x.y;
      v[i + 2] = x.z;
      v[i + 3] = x.w;
    }
  } else if constexpr (N == 2) {
    const float2 x = *reinterpret_cast<const float2*>(src);
    v[0] = x.x;
    v[1] = x.y;
  } else {
    v[0] = *src;
  }
}

// out[row] = sum over splits of partial O scaled to the common maximum, over the
// sum of their sums, for the rows of sequences whose keys are split. blockIdx.y:
// sequence, whose first CTA-many rows (token, head) go to its CTAs in turn, so that
// sequences without splits cost next to nothing (a search for every row's sequence
// took 33 us behind a batch of prompts that had no splits). `wpr` warps of the CTA
// per row: one when there are few splits (more rows per CTA), four when there are
// many. Bound by latency: lanes hold a split's factor each, the loads of partial O
// do not wait for one another.
template <int HD>
__global__ void __launch_bounds__(128)
    paged_join_kernel(const __grid_constant__ Paged p, const __grid_constant__ PagedAttn a,
                      int wpr) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int DL = HD >= 32 ? HD / 32 : 1;  // dims of a lane
  __shared__ float sm[4][HD];
  const PagedSeq seq = paged_attn_seq(p, a, blockIdx.y);
  if (!paged_is_split(a, seq)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % wpr, heads = p.kv_heads * a.group, per_cta = 4 / wpr;
  const int keys = paged_split_keys(a, seq);
  const bool mine = HD >= 32 || lane < HD;
  const int64_t rows = static_cast<int64_t>(seq.n) * heads;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * per_cta; r0 < rows;
       r0 += static_cast<int64_t>(gridDim.x) * per_cta) {
    const int64_t r = r0 + warp / wpr;
    const bool real = r < rows;  // the same for a warp
    const int i = real ? static_cast<int>(r / heads) : 0, head = static_cast<int>(r % heads);
    const int lim = a.causal ? min(seq.len, max(0, seq.pos0 + i + 1)) : seq.len;
    const int n = real ? min(paged_split_count(a, seq), (lim + keys - 1) / keys) : 0;
    const int64_t base = (static_cast<int64_t>(seq.row0 + i) * heads + head) * a.splits;
    float m = -INFINITY, l = 0.f, acc[DL];
#pragma unroll
    for (int e = 0; e < DL; ++e) acc[e] = 0.f;
    for (int s = lane; s < n; s += 32) m = fmaxf(m, a.part_ml[base + s].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    for (int s0 = 0; s0 < n; s0 += 32) {
      float f = 0.f;
      bool seen = false;  // the split saw a key of this row
      if (s0 + lane < n) {
        const float2 ml = a.part_ml[base + s0 + lane];
        f = ml.x == -INFINITY && ml.y == 0.f ? 0.f : fast_exp2(ml.x - m);
        seen = !(f == 0.f && ml.y == 0.f);
        if (seen) l += f * ml.y;
      }
      const uint32_t used = __ballot_sync(0xffffffffu, seen);
      const int count = min(32, n - s0);
#pragma unroll 4
      for (int j = part; j < count; j += wpr) {
        const float g = __shfl_sync(0xffffffffu, f, j);
        float v[DL];
        if (mine) load_floats<DL>(a.part_o + (base + s0 + j) * HD + lane * DL, v);
        if ((used >> j) & 1u) {
#pragma unroll
          for (int e = 0; e < DL; ++e) acc[e] = mine ? acc[e] + g * v[e] : 0.f;
        }
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    if (wpr > 1) {
      if (mine) {
#pragma unroll
        for (int e = 0; e < DL; ++e) sm[warp][lane * DL + e] = acc[e];
      }
      __syncthreads();
      if (warp == 0 && mine) {
#pragma unroll
        for (int w = 1; w < 4; ++w)
#pragma unroll
          for (int e = 0; e < DL; ++e) acc[e] += sm[w][lane * DL + e];
      }
      __syncthreads();
    }
    if (part != 0 || !real || !mine) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    __half* dst = a.out + static_cast<int64_t>(seq.row0 + i) * a.ld_out + head * HD + lane * DL;
    if constexpr (DL == 1) {
      *dst = __float2half_rn(acc[0] * inv);
    } else {
#pragma unroll
      for (int e = 0; e < DL; e += 2)
        *reinterpret_cast<uint32_t*>(dst + e) = pack_half2(acc[e] * inv, acc[e + 1] * inv);
    }
  }
}

// rows: (token, head) rows of a sequence that may be split, at most.
template <int HD>
int launch_join(const Paged& p, const PagedAttn& a, int64_t rows, cudaStream_t stream) {
  const int64_t all = static_cast<int64_t>(p.num_tokens) * p.kv_heads * a.group;
  const int wpr = a.splits > 16 ? 4 : 1, per_cta = 4 / wpr;
  // A CTA for every per_cta rows of the longest sequence, but not many more in all
  // than there are rows.
  int64_t most = 2 * ((all + per_cta - 1) / per_cta) / p.batch;
  if (most < 4096 / p.batch) most = 4096 / p.batch;
  int64_t x = (rows + per_cta - 1) / per_cta;
  if (x > most) x = most < 1 ? 1 : most;
  launch_pdl(paged_join_kernel<HD>, dim3(static_cast<unsigned>(x), static_cast<unsigned>(p.batch)),
             dim3(128), 0, stream, p, a, wpr);
  return check_launch("paged_join_kernel");
}

int join_hd(const Paged& p, const PagedAttn& a, int head_dim, int64_t rows, cudaStream_t stream) {
  switch (head_dim) {
    case 8: return launch_join<8>(p, a, rows, stream);
    case 16: return launch_join<16>(p, a, rows, stream);
    case 32: return launch_join<32>(p, a, rows, stream);
    case 64: return launch_join<64>(p, a, rows, stream);
    case 128: return launch_join<128>(p, a, rows, stream);
    default: return launch_join<256>(p, a, rows, stream);
  }
}

struct Plan {
  int64_t q, rows;  // new tokens of the longest sequence, and their rows
  int block_rows;   // of the mma.sync kernel
  int tc_rows;      // sequences with more rows go to the tcgen05 kernel
  bool tc, small;   // which kernels run
  int splits, splits_rows, splits_tc, kps, kps_tc, cluster;
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
  // Row blocks x ranges are the launch's gridDim.z. More row blocks than that (from 65536
  // new tokens in groups of 65 at head_dim 256) are the mma.sync kernel's.
  constexpr int64_t kGridZ = 65535;
  const int64_t tc_row_blocks = (pl.q + tokens - 1) / tokens, tc_blocks = pairs * tc_row_blocks;
  int64_t tc_parts = 1;
  double tc_cost = 0., tc_keys = 0.;
  for (int64_t n = 1; n <= 16 && (n == 1 || ((kv + n - 1) / n >= 1024 && tc_row_blocks * n <= kGridZ));
       ++n) {
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
  pl.tc = hd >= 64 && group <= 128 && pl.rows > tc_rows(hd) && tc_row_blocks <= kGridZ;
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
  pl.splits_tc = pl.tc ? static_cast<int>((kv + pl.kps_tc - 1) / pl.kps_tc) : 1;
  pl.splits_rows =
      pl.small && pl.cluster == 0 ? static_cast<int>((kv + pl.kps - 1) / pl.kps) : 1;
  pl.splits = pl.splits_tc > pl.splits_rows ? pl.splits_tc : pl.splits_rows;
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
  a.q_len = static_cast<int>(pl.q);
  a.splits = pl.splits;
  a.splits_rows = pl.splits_rows;
  a.splits_tc = pl.splits_tc;
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
  // (the sequences with more rows are the tcgen05 kernel's)
  const int64_t rows = pl.tc && pl.splits_tc == 1 ? pl.tc_rows : pl.rows;
  return join_hd(p, a, cache->head_dim, rows * cache->kv_heads, stream);
}

}  // extern "C"
