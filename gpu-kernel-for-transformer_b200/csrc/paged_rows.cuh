// Attention of a few query rows over a paged cache, on mma.sync: every
// head_dim, cache type and number of rows. Included by one translation unit
// per cache type.
//
// Rows: the `group` query heads that read one key/value head are rows of the
// same block (row = token * group + head in group), so a cached key is read
// once for all of them. A CTA takes 8 * NT rows of one (sequence, key/value
// head) and one range of its keys. Its warps take the range's KT-key tiles in
// turn, each with a ring of two tiles of its own in shared memory (cp.async,
// no barrier between warps) and its own running maximum and sum per row; they
// are merged through shared memory at the end.
//
// Keys are the products' M: S^T = K Q^T and O^T = V^T P^T, 16 keys (or dims) by
// 8 rows at a time, so that a single row wastes 7 columns and not 15 rows, and
// a cached value is expanded once for all rows. Bound by instructions, not
// by the tensor cores; against rows as M: half the products, scores and
// accumulators per key at up to 8 rows. P^T comes out of the first product with
// keys along lanes and goes into the second with keys along k: movmatrix.
//
// The running maximum moves only when a score exceeds it by more than 2^8
// (weights stay below 2^8, fine in fp16), so that most tiles need neither the
// maximum over lanes nor a rescaled accumulator, only a vote.
//
// 8-bit caches are expanded to fp16 in registers, between ldmatrix and the
// product, without the scales: a key's scale multiplies its row of scores, a
// value's is an exponent added to them (see value_scale_log2), both in fp32.
// The weights, with the values' scales in them, are rounded to fp16 for the second
// product.
//
// Fragment orders. An 8x8 ldmatrix block of 16-bit words holds 8 keys x 16
// codes. Scores: thread (g, t) gets codes 4t..4t+3 of key g and uses (4t, 4t+1)
// and (4t+2, 4t+3) as the k pairs; the sum over k does not depend on the order,
// and Q is stored in the same one. Second product, transposed load: the thread
// gets dims 2g and 2g+1 of keys 2t and 2t+1; the even dims are rows 0-7 of the
// product, the odd dims rows 8-15.
//
// Masked keys. A weight of 0 does not hide an infinity or NaN among the values
// (0 * inf), so values beyond the sequence are loaded as zeros, and in tiles
// that some rows of the block see and others do not, non-finite fp16 values
// (NaN codes) are cleared before the product and added at the end to the rows
// that see them. (A scale that is not finite stays in its row: it makes the score
// NaN, which is replaced where masked.)
//
// Keys over CTAs: either ranges of kps keys whose unnormalised results a second
// kernel joins, or, where 8 ranges are enough, a cluster of CTAs with equal
// shares that reads each other's results from shared memory: one launch and
// no workspace.
#pragma once

#include "paged.cuh"

namespace tfx {
namespace {

__device__ __forceinline__ void rows_cp16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // zero-fill where there is no key
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
__device__ __forceinline__ void rows_cp4(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
__device__ __forceinline__ void rows_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void rows_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void rows_ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void rows_ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void rows_ldsm2(uint32_t addr, uint32_t& r0, uint32_t& r1) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
               : "=r"(r0), "=r"(r1) : "r"(addr) : "memory");
}
__device__ __forceinline__ void rows_ldsm2_t(uint32_t addr, uint32_t& r0, uint32_t& r1) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(r0), "=r"(r1) : "r"(addr) : "memory");
}
// Transposes an 8x8 block of 16-bit words held two to a lane.
__device__ __forceinline__ uint32_t rows_movm_t(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// D(16x8, f32) += A(16x16, f16, row) * B(16x8, f16, col)
__device__ __forceinline__ void rows_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float4 rows_peer4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 rows_peer2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr)
               : "memory");
  return v;
}

constexpr float kRowsRescale = 8.0f;  // log2 units, see the file's comment

template <int CODE, int HD, int NT>
struct RowsCfg {
  static constexpr int kRows = 8 * NT;
  // One CTA to an SM at 512-byte rows: more warps in it.
  static constexpr int kWarps = HD * code_bytes(CODE) >= 512 ? 6 : 4;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kHDP = HD < 16 ? 16 : HD;  // width of the first product (zero padded)
  static constexpr int kRowBytes = HD * code_bytes(CODE);
  static constexpr int kU = kRowBytes / 16;  // 16-byte chunks of a cached row
  // Rows an odd number of chunks apart: ldmatrix without bank conflicts.
  static constexpr int kPitch = ((kHDP * code_bytes(CODE) / 16) | 1) * 16;
  static constexpr int kQPitch = (kHDP + 8) * 2;
  // Keys of a warp's tile: about 2 KB of K (small tiles keep more warps on an
  // SM), 4 KB with more than 8 rows (registers bound the warps there, and a tile's
  // fixed cost is larger: 46 against 40 us for drafts of 2 to 8 tokens in groups of
  // 4, int8, 128); at most 64, and 128 scores to a column of lanes.
  static constexpr int kMost = 128 / NT < 64 ? 128 / NT : 64;
  static constexpr int kWantBytes = NT >= 2 ? 4096 : 2048;
  static constexpr int kWant = kWantBytes / kRowBytes < 16 ? 16 : kWantBytes / kRowBytes;
  static constexpr int kKT = kWant < kMost ? kWant : kMost;
  static constexpr int NS = 2;
  static constexpr int kTileBytes = kKT * kPitch;
  static constexpr int kScaleBytes = CODE == kCodeF16 ? 0 : 2 * kKT * 4;
  // K, V, their scales, the bits of keys that exist
  static constexpr int kStageBytes = 2 * kTileBytes + kScaleBytes + 16;
  static constexpr int kQBytes = kRows * kQPitch;
  static constexpr int kRing = kWarps * NS * kStageBytes;
  // After the loop, over the ring: 8 rows of every warp; the CTA's rows.
  static constexpr int kMP = HD + 4;  // row pitch in floats: spreads the banks
  static constexpr int kMergeRows = kWarps * 8 * kMP * 4;
  static constexpr int kMergeMl = kMergeRows + kWarps * 8 * 8;
  static constexpr int kPart = kMergeMl + kRows * HD * 4;
  static constexpr int kMerge = kPart + kRows * 8;
  static constexpr int kFlag = kQBytes + (kRing > kMerge ? kRing : kMerge);
  static constexpr int kSmem = kFlag + 16;
  static_assert(kSmem <= 227 * 1024, "shared-memory budget");
  static_assert(kKT >= 16 && kKT % 16 == 0, "tile of 16 to 64 keys");
};

// A CTA's work, in the layout C of NTC blocks of 8 rows; NT of them hold rows.
template <int CODE, int HD, int NTC, int NT>
__device__ __forceinline__ void rows_cta(const Paged& p, const PagedAttn& a, const PagedSeq& seq,
                                         int rb, int split) {
  using C = RowsCfg<CODE, HD, NTC>;
  constexpr int KT = C::kKT, NS = C::NS, HDP = C::kHDP, U = C::kU, W = C::kWarps;
  constexpr int KB = KT / 16;                // 16-key blocks of a tile
  constexpr int KS = HDP / 16;               // 16-wide steps of the first product
  constexpr int DB = HD < 16 ? 1 : HD / 16;  // 16-dim blocks of the output
  constexpr int KW = (KT + 31) / 32;         // 32-bit words of key bits
  constexpr bool kQuant = CODE != kCodeF16;
  // Chains of dependent products: several accumulators where there are few.
  constexpr int kAcc0 = NT * KB >= 4 ? 1 : 4 / (NT * KB);
  constexpr int ACC = kAcc0 < KS ? kAcc0 : KS;
  constexpr bool kQInRegs = NT * KS <= 16;
  extern __shared__ __align__(16) uint8_t smem_rows[];
  uint8_t* sQ = smem_rows;
  int* flag = reinterpret_cast<int*>(smem_rows + C::kFlag);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int b = blockIdx.z, hk = blockIdx.y;
  const int parts = a.cluster > 0 ? a.cluster : a.splits_rows;
  const int rows = seq.n * a.group;  // below 2^31: checked on the host
  const int r0 = rb * C::kRows;
  // Keys that row r sees: [0, lim(r)).
  auto lim_of = [&](int r) {
    return a.causal ? min(seq.len, max(0, seq.pos0 + r / a.group + 1)) : seq.len;
  };
  const int lim_first = lim_of(r0), lim_last = lim_of(min(r0 + C::kRows, rows) - 1);
  const bool is_split = a.cluster == 0 && paged_is_split(a, seq);
  int k_begin = 0, k_end = lim_last;
  if (a.cluster > 0) {
    const int share = ((lim_last + parts - 1) / parts + KT - 1) / KT * KT;
    k_begin = min(split * share, lim_last);
    k_end = min(k_begin + share, lim_last);
  } else {
    // Splits behind the sequence.
    if (is_split ? static_cast<int64_t>(split) * a.kps >= lim_last : split > 0) return;
    if (is_split) {
      k_begin = split * a.kps;
      k_end = min(lim_last, paged_split_end(a, seq, split, k_begin));
    }
  }

  // ---- queries as the product's B operand, zero rows behind the last one.
  // 8 bits: dims in the order of the codes' k pairs (see the file's comment).
  for (int i = threadIdx.x; i < 8 * NT * (HD / 8); i += C::kThreads) {
    const int r = i / (HD / 8), c = i % (HD / 8), row = r0 + r;
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows)
      x = *reinterpret_cast<const uint4*>(a.q +
                                          static_cast<int64_t>(seq.row0 + row / a.group) * a.ld_q +
                                          (hk * a.group + row % a.group) * HD + c * 8);
    uint8_t* dst = sQ + r * C::kQPitch;
    if constexpr (!kQuant) {
      *reinterpret_cast<uint4*>(dst + c * 16) = x;
      if (HD < 16) *reinterpret_cast<uint4*>(dst + 16) = make_uint4(0u, 0u, 0u, 0u);
    } else {  // words 0, 2 of the 4 here to the first half of the 16, 1, 3 to the second
      uint8_t* at = dst + (c >> 1) * 32 + (c & 1) * 8;
      *reinterpret_cast<uint2*>(at) = make_uint2(x.x, x.z);
      *reinterpret_cast<uint2*>(at + 16) = make_uint2(x.y, x.w);
    }
  }
  if (threadIdx.x == 0) *flag = 0;

  // ---- this warp's ring
  uint8_t* ring = smem_rows + C::kQBytes + warp * NS * C::kStageBytes;
  if constexpr (HD < 16) {
    for (int i = lane; i < NS * 2 * KT; i += 32)
      *reinterpret_cast<uint4*>(ring + (i / (2 * KT)) * C::kStageBytes + (i % (2 * KT)) * C::kPitch +
                                HD * 2) = make_uint4(0, 0, 0, 0);
  }
  const int n_tiles =
      k_end > k_begin + warp * KT ? (k_end - k_begin - warp * KT + W * KT - 1) / (W * KT) : 0;
  const uint8_t* kb = static_cast<const uint8_t*>(p.k) + hk * p.head_stride * code_bytes(CODE);
  const uint8_t* vb = static_cast<const uint8_t*>(p.v) + hk * p.head_stride * code_bytes(CODE);
  auto tile_key = [&](int i) { return k_begin + (i * W + warp) * KT; };
  // Pages of this lane's keys of tile i (lane and lane + 32), one tile ahead.
  const int32_t* table = p.table + b * p.table_stride;
  int pg[KW];
  auto look_up = [&](int i) {
#pragma unroll
    for (int u = 0; u < KW; ++u) {
      const int key = tile_key(i) + 32 * u + lane;
      int page = -1;
      if (i < n_tiles && key < k_end && (KT % 32 == 0 || lane < KT)) page = table[key >> p.page_shift];
      pg[u] = static_cast<unsigned>(page) < static_cast<unsigned>(p.num_pages) ? page : -1;
    }
  };
  // 16 keys lie in one page. Lane = (row of it, 16-byte chunk); a pass covers
  // RP rows, a group of passes 16 keys (32 where a pass does).
  constexpr int RP = 32 / U, GK = RP > 16 ? RP : 16;
  const int64_t row_step = p.token_stride * code_bytes(CODE);
  const int64_t lane_off = (lane / U) % 16 * row_step + (lane % U) * 16;
  const uint8_t* klane = kb + lane_off;
  const uint8_t* vlane = vb + lane_off;
  const uint32_t lane_dst = smem_u32(ring) + (lane / U) * C::kPitch + (lane % U) * 16;
  auto load = [&](int i) {
    const uint32_t st = (i % NS) * C::kStageBytes;
    const int k0 = tile_key(i);
    uint32_t there[KW];  // keys that exist
#pragma unroll
    for (int u = 0; u < KW; ++u) there[u] = __ballot_sync(0xffffffffu, pg[u] >= 0);
#pragma unroll
    for (int g0 = 0; g0 < KT; g0 += GK) {
      // Byte offset of the group's first key (of each half's, where a pass is two).
      const int page = __shfl_sync(0xffffffffu, pg[g0 / 32], GK == 32 ? lane & 16 : g0 & 16);
      const int first = k0 + g0 + (GK == 32 ? lane & 16 : 0);
      const int64_t from = page >= 0 ? paged_offset(p, page, first & ~15) * code_bytes(CODE) : 0;
      const uint8_t* kp = klane + from;
      const uint8_t* vp = vlane + from;
      const uint32_t dst = lane_dst + st + g0 * C::kPitch;
      constexpr uint32_t kAll = GK >= 32 ? 0xffffffffu : 0xffffu;
      const bool mine = KT % RP == 0 || lane / U < KT;
      if (((there[g0 / 32] >> (g0 & 31)) & kAll) == kAll) {
#pragma unroll
        for (int it = 0; it < GK / RP; ++it) {
          rows_cp16(dst + it * RP * C::kPitch, kp, true);
          rows_cp16(dst + C::kTileBytes + it * RP * C::kPitch, vp, true);
          kp += RP * row_step;
          vp += RP * row_step;
        }
      } else {  // zeros where there is no key
#pragma unroll 1
        for (int it = 0; it < GK / RP; ++it) {
          const int r = g0 + it * RP + lane / U;
          const bool ok = mine && ((there[g0 / 32] >> (r & 31)) & 1u);
          const int64_t off = static_cast<int64_t>(it) * RP * row_step;
          if (mine) {
            rows_cp16(dst + it * RP * C::kPitch, ok ? kp + off : kb, ok);
            rows_cp16(dst + C::kTileBytes + it * RP * C::kPitch, ok ? vp + off : vb, ok);
          }
        }
      }
    }
    uint8_t* at = ring + st + 2 * C::kTileBytes;
    if constexpr (kQuant) {
#pragma unroll
      for (int u = 0; u < KW; ++u) {
        if (KT % 32 == 0 || lane < KT) {
          const bool ok = pg[u] >= 0;
          const int64_t so = ok ? paged_scale_offset(p, pg[u], hk, k0 + 32 * u + lane) : 0;
          rows_cp4(smem_u32(at) + (32 * u + lane) * 4, p.k_scale + so, ok);
          rows_cp4(smem_u32(at) + (KT + 32 * u + lane) * 4, p.v_scale + so, ok);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < KW; ++u)
      if (lane == 0) reinterpret_cast<uint32_t*>(at + C::kScaleBytes)[u] = there[u];
  };
  look_up(0);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    if (i < n_tiles) load(i);
    rows_commit();
    look_up(i + 1);
  }
  __syncthreads();  // the queries

  // Q fragments of two steps at a time (b0, b1 of each).
  auto load_q = [&](int nt, int kk, uint32_t (&f)[4]) {
    const uint32_t row = smem_u32(sQ + (nt * 8 + (lane & 7)) * C::kQPitch + kk * 32);
    if constexpr (KS == 1)
      rows_ldsm2(row + ((lane >> 3) & 1) * 16, f[0], f[1]);
    else
      rows_ldsm4(row + (lane >> 4) * 32 + ((lane >> 3) & 1) * 16, f);
  };
  uint32_t qf[kQInRegs ? NT : 1][kQInRegs ? (KS + 1) / 2 : 1][4];
  if constexpr (kQInRegs) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int kk = 0; kk < KS; kk += 2) load_q(nt, kk, qf[nt][kk / 2]);
  }

  // Rows 2t and 2t+1 of each 8 are this thread's.
  float o[NT][DB][4];
  float m_ref[NT][2], l_run[NT][2];
  int lim[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int n = 0; n < DB; ++n) o[nt][n][0] = o[nt][n][1] = o[nt][n][2] = o[nt][n][3] = 0.f;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m_ref[nt][r] = -INFINITY;  // no key seen yet
      l_run[nt][r] = 0.f;
      lim[nt][r] = lim_of(min(r0 + nt * 8 + 2 * t + r, rows - 1));
    }
  }
  bool cleared = false;

  for (int i = 0; i < n_tiles; ++i) {
    __syncwarp();  // every lane is done with the stage that is loaded next
    if (i + NS - 1 < n_tiles) load(i + NS - 1);
    rows_commit();
    look_up(i + NS);
    rows_wait<NS - 1>();
    __syncwarp();
    uint8_t* st = ring + (i % NS) * C::kStageBytes;
    uint8_t* sv = st + C::kTileBytes;
    const float* sc = reinterpret_cast<const float*>(st + 2 * C::kTileBytes);
    const int k0 = tile_key(i);

    // ---- S^T = K Q^T: key g (values 0, 1) and g + 8 (2, 3) of each 16, rows 2t, 2t+1
    float s[NT][KB][4];
    {
      float part[ACC][NT][KB][4];
#pragma unroll
      for (int x = 0; x < ACC; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < KB; ++j)
            part[x][nt][j][0] = part[x][nt][j][1] = part[x][nt][j][2] = part[x][nt][j][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KS; kk += 2) {
        uint32_t f[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if constexpr (kQInRegs) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[nt][e] = qf[nt][kk / 2][e];
          } else {
            load_q(nt, kk, f[nt]);
          }
        }
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          const uint32_t row =
              smem_u32(st + (j * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * C::kPitch);
          uint32_t k1[4], k2[4];  // steps kk and kk + 1
          if constexpr (!kQuant) {
            rows_ldsm4(row + kk * 32 + (lane >> 4) * 16, k1);
            if constexpr (KS > 1) rows_ldsm4(row + (kk + 1) * 32 + (lane >> 4) * 16, k2);
          } else {
            uint32_t w[4];
            if constexpr (KS > 1)
              rows_ldsm4(row + (kk + (lane >> 4)) * 16, w);
            else
              rows_ldsm2(row, w[0], w[1]);
            k1[0] = codes_to_h2<CODE, 0, 1>(w[0]);
            k1[1] = codes_to_h2<CODE, 0, 1>(w[1]);
            k1[2] = codes_to_h2<CODE, 2, 3>(w[0]);
            k1[3] = codes_to_h2<CODE, 2, 3>(w[1]);
            if constexpr (KS > 1) {
              k2[0] = codes_to_h2<CODE, 0, 1>(w[2]);
              k2[1] = codes_to_h2<CODE, 0, 1>(w[3]);
              k2[2] = codes_to_h2<CODE, 2, 3>(w[2]);
              k2[3] = codes_to_h2<CODE, 2, 3>(w[3]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            rows_mma(part[kk % ACC][nt][j], k1, f[nt][0], f[nt][1]);
            if constexpr (KS > 1) rows_mma(part[(kk + 1) % ACC][nt][j], k2, f[nt][2], f[nt][3]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < KB; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[nt][j][e] = part[0][nt][j][e];
#pragma unroll
            for (int x = 1; x < ACC; ++x) s[nt][j][e] += part[x][nt][j][e];
          }
    }

    // ---- keys that exist; values that must not leak
    uint32_t bits[KW];
    bool full = true;
#pragma unroll
    for (int u = 0; u < KW; ++u) {
      bits[u] = reinterpret_cast<const uint32_t*>(st + 2 * C::kTileBytes + C::kScaleBytes)[u];
      full = full && bits[u] == (KT < 32 ? (1u << (KT & 31)) - 1u : 0xffffffffu);
    }
    const bool need_mask = !full || k0 + KT > lim_first;  // warp-uniform
    if constexpr (CODE != kCodeI8) {
      if (k0 + KT > lim_first && lim_first < lim_last) {
        bool found = false;
        for (int c = lane; c < KT * U; c += 32) {
          uint4* at = reinterpret_cast<uint4*>(sv + (c / U) * C::kPitch + (c % U) * 16);
          uint4 x = *at;
          uint32_t* w = reinterpret_cast<uint32_t*>(&x);
          bool hit = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (CODE == kCodeF16) {
              hit |= h2_clear(w[e]);
            } else {
              const uint32_t nan = __vcmpeq4(w[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              hit = hit || nan != 0u;
              w[e] &= ~nan;
            }
          }
          if (hit) {
            *at = x;
            found = true;
          }
        }
        if (__any_sync(0xffffffffu, found)) cleared = true;
        __syncwarp();
      }
    }

    // ---- scores in the log2 domain, masked; does a maximum grow?
    [[maybe_unused]] float back_x[kQuant ? KB : 1][2];  // 1 / the values' scales
#pragma unroll
    for (int j = 0; j < KB; ++j) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float f = a.scale_log2, e = 0.f;
        if constexpr (kQuant) {
          f *= sc[j * 16 + g + 8 * r];
          const float vs = sc[KT + j * 16 + g + 8 * r];
          e = value_scale_log2(vs);
          back_x[j][r] = value_scale_inverse(vs);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[nt][j][2 * r] = kQuant ? fmaf(s[nt][j][2 * r], f, e) : s[nt][j][2 * r] * f;
          s[nt][j][2 * r + 1] = kQuant ? fmaf(s[nt][j][2 * r + 1], f, e) : s[nt][j][2 * r + 1] * f;
        }
      }
    }
    if (need_mask) {
#pragma unroll
      for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int kk = j * 16 + g + 8 * r;
          const int key = (bits[kk >> 5] >> (kk & 31)) & 1u ? k0 + kk : 0x7fffffff;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (key >= lim[nt][e]) s[nt][j][2 * r + e] = -INFINITY;
        }
    }
    float mx[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[nt][e] = fmaxf(s[nt][0][e], s[nt][0][2 + e]);
#pragma unroll
        for (int j = 1; j < KB; ++j) mx[nt][e] = fmax3(mx[nt][e], s[nt][j][e], s[nt][j][2 + e]);
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      grow = grow || mx[nt][0] > m_ref[nt][0] + kRowsRescale || mx[nt][1] > m_ref[nt][1] + kRowsRescale;
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float corr[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = mx[nt][e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          m = fmaxf(m, m_ref[nt][e]);
          corr[e] = m == m_ref[nt][e] ? 1.f : fast_exp2(m_ref[nt][e] - m);  // from -inf: 0
          m_ref[nt][e] = m;
          l_run[nt][e] *= corr[e];
        }
#pragma unroll
        for (int n = 0; n < DB; ++n) {
          o[nt][n][0] *= corr[0];
          o[nt][n][1] *= corr[1];
          o[nt][n][2] *= corr[0];
          o[nt][n][3] *= corr[1];
        }
      }
    }

    // ---- weights, as the second product's B operand. The sum takes them as rounded
    // to fp16, or a row in which one key has nearly all the weight would carry that
    // key's rounding in full. 8 bit: what is rounded has the value's scale in it, and a
    // key of small values may have all the weight: rounded only where that is a normal
    // fp16 number.
    uint32_t pf[NT][KB][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float m_use[2];  // nothing seen yet: weights 0, no NaN
#pragma unroll
      for (int e = 0; e < 2; ++e) m_use[e] = m_ref[nt][e] == -INFINITY ? 0.f : m_ref[nt][e];
#pragma unroll
      for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) w[e] = fast_exp2(s[nt][j][2 * r + e] - m_use[e]);
          const uint32_t h = pack_half2(w[0], w[1]);
          const float2 hf = __half22float2(bits_h2(h));
          if constexpr (kQuant) {
            l_run[nt][0] += (w[0] < 0x1p-14f ? w[0] : hf.x) * back_x[j][r];
            l_run[nt][1] += (w[1] < 0x1p-14f ? w[1] : hf.y) * back_x[j][r];
          } else {
            l_run[nt][0] += hf.x;
            l_run[nt][1] += hf.y;
          }
          pf[nt][j][r] = rows_movm_t(h);
        }
    }

    // ---- O^T += V^T P^T: 16 dims by 16 keys
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      const uint32_t row = smem_u32(sv + j * 16 * C::kPitch);
      if constexpr (!kQuant) {
        if constexpr (HD < 16) {
          uint32_t v[4] = {0u, 0u, 0u, 0u};
          rows_ldsm2_t(row + (lane & 15) * C::kPitch, v[0], v[2]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) rows_mma(o[nt][0], v, pf[nt][j][0], pf[nt][j][1]);
        } else {
#pragma unroll
          for (int n = 0; n < DB; ++n) {
            uint32_t v[4];
            rows_ldsm4_t(row + ((lane >> 4) * 8 + (lane & 7)) * C::kPitch + n * 32 +
                             ((lane >> 3) & 1) * 16,
                         v);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) rows_mma(o[nt][n], v, pf[nt][j][0], pf[nt][j][1]);
          }
        }
      } else {
        auto block = [&](int n, uint32_t lo, uint32_t hi) {  // 16 dims; keys 0-7, 8-15
          const uint32_t v[4] = {codes_to_h2<CODE, 0, 2>(lo), codes_to_h2<CODE, 1, 3>(lo),
                                 codes_to_h2<CODE, 0, 2>(hi), codes_to_h2<CODE, 1, 3>(hi)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) rows_mma(o[nt][n], v, pf[nt][j][0], pf[nt][j][1]);
        };
        if constexpr (HD == 16) {
          uint32_t lo, hi;
          rows_ldsm2_t(row + (lane & 15) * C::kPitch, lo, hi);
          block(0, lo, hi);
        } else {
#pragma unroll
          for (int n = 0; n < DB; n += 2) {
            uint32_t w[4];
            rows_ldsm4_t(row + (lane & 15) * C::kPitch + (n + (lane >> 4)) * 16, w);
            block(n, w[0], w[1]);
            block(n + 1, w[2], w[3]);
          }
        }
      }
    }
  }
  rows_wait<0>();
  if (cleared && lane == 0) *flag = 1;
  __syncthreads();
  const bool fix = *flag != 0;

  // ---- merge the warps, 8 rows at a time
  uint8_t* area = smem_rows + C::kQBytes;
  float* mo = reinterpret_cast<float*>(area);                      // [warp][8][kMP]
  float2* ml = reinterpret_cast<float2*>(area + C::kMergeRows);    // [warp][8] (max, sum)
  float* cta_o = reinterpret_cast<float*>(area + C::kMergeMl);     // cluster: [kRows][HD]
  float2* cta_ml = reinterpret_cast<float2*>(area + C::kPart);     // cluster: [kRows]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (r0 + nt * 8 >= rows) break;  // uniform
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1)
        l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], d);
      float* dst = mo + (warp * 8 + 2 * t + e) * C::kMP;
#pragma unroll
      for (int n = 0; n < DB; ++n) {
        if constexpr (kQuant) {
          *reinterpret_cast<float2*>(dst + n * 16 + 2 * g) =
              make_float2(o[nt][n][e], o[nt][n][2 + e]);
        } else {
          dst[n * 16 + g] = o[nt][n][e];
          if constexpr (HD >= 16) dst[n * 16 + 8 + g] = o[nt][n][2 + e];
        }
      }
      if (g == 0) ml[warp * 8 + 2 * t + e] = make_float2(m_ref[nt][e], l_run[nt][e]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * (HD / 4); i += C::kThreads) {
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4, row = r0 + nt * 8 + r;
      if (row >= rows) continue;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) m = fmaxf(m, ml[w * 8 + r].x);
      float acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 x = ml[w * 8 + r];
        if (x.x == -INFINITY && x.y == 0.f) continue;  // this warp saw no key
        const float f = fast_exp2(x.x - m);
        const float4 y = *reinterpret_cast<const float4*>(mo + (w * 8 + r) * C::kMP + d);
        acc[0] += f * y.x;
        acc[1] += f * y.y;
        acc[2] += f * y.z;
        acc[3] += f * y.w;
        l += f * x.y;
      }
      if (fix) {  // non-finite values cleared from shared tiles: to the rows that see them
        const int hi = min(lim_of(row), k_end);
        for (int key = max(k_begin, lim_first - KT); key < hi; ++key) {
          const int page = paged_page(p, b, key);
          if (page < 0) continue;
          const int64_t at = paged_offset(p, page, key) + hk * p.head_stride + d;
          const float sv = kQuant ? p.v_scale[paged_scale_offset(p, page, hk, key)] : 1.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = paged_value<CODE>(p.v, at + e, sv);
            if (!isfinite(x)) acc[e] += x;
          }
        }
      }
      const int tok = seq.row0 + row / a.group, head = hk * a.group + row % a.group;
      const float4 y = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (a.cluster > 0) {
        *reinterpret_cast<float4*>(cta_o + (nt * 8 + r) * HD + d) = y;
        if (d == 0) cta_ml[nt * 8 + r] = make_float2(m, l);
      } else if (is_split) {
        const int64_t at =
            (static_cast<int64_t>(tok) * (p.kv_heads * a.group) + head) * a.splits + split;
        *reinterpret_cast<float4*>(a.part_o + at * HD + d) = y;
        if (d == 0) a.part_ml[at] = make_float2(m, l);
      } else {
        store_row4(a.out + static_cast<int64_t>(tok) * a.ld_out + head * HD + d, y, l);
      }
    }
    __syncthreads();
  }
  if (a.cluster == 0) return;

  // ---- join the cluster: every CTA a share of the rows' elements
  cluster_sync_all();
  const int count = min(C::kRows, rows - r0) * (HD / 4);
  for (int i = split * C::kThreads + threadIdx.x; i < count; i += parts * C::kThreads) {
    const int r = i / (HD / 4), d = (i % (HD / 4)) * 4, row = r0 + r;
    const uint32_t at_ml = smem_u32(cta_ml + r), at_o = smem_u32(cta_o + r * HD + d);
    float m = -INFINITY;
    for (int c = 0; c < parts; ++c) m = fmaxf(m, rows_peer2(mapa_shared(at_ml, c)).x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int c = 0; c < parts; ++c) {
      const float2 x = rows_peer2(mapa_shared(at_ml, c));
      if (x.x == -INFINITY && x.y == 0.f) continue;  // this CTA saw no key
      const float f = fast_exp2(x.x - m);
      const float4 y = rows_peer4(mapa_shared(at_o, c));
      acc.x += f * y.x;
      acc.y += f * y.y;
      acc.z += f * y.z;
      acc.w += f * y.w;
      l += f * x.y;
    }
    store_row4(a.out + static_cast<int64_t>(seq.row0 + row / a.group) * a.ld_out +
                   (hk * a.group + row % a.group) * HD + d,
               acc, l);
  }
  cluster_sync_all();  // no CTA leaves while another reads its results
}

// MIXED: launched behind the tcgen05 kernel of the same call, which waited for what
// came before both. This one writes other rows, so it need not wait for that kernel;
// it only ends after it (one CTA stays), so that what follows finds both done. Most
// of its sequences are running ones, with few rows in a batch that has many: they
// take only the blocks of 8 that hold rows. (36 sequences with 1 new token and 4 with
// 200, 8 heads in groups of 4, head_dim 128, 800 to 8000 keys: one behind the other
// and with all blocks 282 us, so 184; int8 309 and 190. In kernels that run alone the
// three bodies cost more, in instructions fetched, than they save: drafts of 2 to 8
// tokens, 55 against 43 us.)
template <int CODE, int HD, int NT, bool MIXED>
__global__ void __launch_bounds__((RowsCfg<CODE, HD, NT>::kThreads))
    paged_rows_kernel(const __grid_constant__ Paged p, const __grid_constant__ PagedAttn a,
                      int row_blocks) {
  if constexpr (!MIXED) grid_dep_wait();
  grid_dep_launch();
  const int parts = a.cluster > 0 ? a.cluster : a.splits_rows;
  const int split = static_cast<int>(blockIdx.x) % parts;  // cluster: also the CTA's rank
  // The last rows see the most keys: they go first.
  const int rb = row_blocks - 1 - static_cast<int>(blockIdx.x) / parts;
  const PagedSeq seq = paged_attn_seq(p, a, blockIdx.z);
  const int left = seq.n * a.group - rb * 8 * NT;
  const bool mine = left > 0 && !paged_is_tc(a, seq);  // the same for a whole cluster
  if constexpr (!MIXED) {
    if (mine) rows_cta<CODE, HD, NT, NT>(p, a, seq, rb, split);
  } else {
    if (!mine) {
    } else if (left <= 8) {
      rows_cta<CODE, HD, NT, 1>(p, a, seq, rb, split);
    } else if (NT >= 4 && left <= 16) {
      rows_cta<CODE, HD, NT, NT >= 4 ? 2 : NT>(p, a, seq, rb, split);
    } else {
      rows_cta<CODE, HD, NT, NT>(p, a, seq, rb, split);
    }
    if ((blockIdx.x | blockIdx.y | blockIdx.z) == 0) grid_dep_wait();
  }
}

template <int CODE, int HD, int NT, bool MIXED>
int launch_rows(const Paged& p, const PagedAttn& a, int64_t rows, cudaStream_t stream) {
  using C = RowsCfg<CODE, HD, NT>;
  static int done[kMaxDevices] = {0};
  auto kern = paged_rows_kernel<CODE, HD, NT, MIXED>;
  int st = ensure_smem(reinterpret_cast<const void*>(kern), C::kSmem, done);
  if (st != TFX_OK) return st;
  const int64_t blocks = (rows + C::kRows - 1) / C::kRows;
  const int parts = a.cluster > 0 ? a.cluster : a.splits_rows;
  if (blocks * parts > 0x7fffffffLL)
    return fail(TFX_ERR_UNSUPPORTED, "tfx_paged_attention: too many rows");
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(parts);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks * parts), p.kv_heads, p.batch);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = a.cluster > 0 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, a, static_cast<int>(blocks));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(TFX_ERR_CUDA, "paged_rows_kernel: %s", cudaGetErrorString(e));
  }
  return TFX_OK;
}

template <int CODE, int HD>
int launch_rows_hd(const Paged& p, const PagedAttn& a, int block_rows, bool mixed, int64_t rows,
                   cudaStream_t stream) {
  // (the tcgen05 kernel has head_dim 64 and more, and leaves 64 rows at most, 16 at 256)
  if constexpr (HD >= 64) {
    if (mixed) return launch_rows<CODE, HD, HD <= 128 ? 4 : 2, true>(p, a, rows, stream);
  }
  if constexpr (HD <= 128) {
    if (block_rows == 32) return launch_rows<CODE, HD, 4, false>(p, a, rows, stream);
  }
  if (block_rows == 16) return launch_rows<CODE, HD, 2, false>(p, a, rows, stream);
  return launch_rows<CODE, HD, 1, false>(p, a, rows, stream);
}

}  // namespace

template <int CODE>
int launch_paged_rows(const Paged& p, const PagedAttn& a, int head_dim, int block_rows,
                      bool mixed, int64_t rows, cudaStream_t stream) {
  switch (head_dim) {
    case 8:
      if constexpr (CODE == kCodeF16) return launch_rows_hd<CODE, 8>(p, a, block_rows, mixed, rows, stream);
      break;
    case 16: return launch_rows_hd<CODE, 16>(p, a, block_rows, mixed, rows, stream);
    case 32: return launch_rows_hd<CODE, 32>(p, a, block_rows, mixed, rows, stream);
    case 64: return launch_rows_hd<CODE, 64>(p, a, block_rows, mixed, rows, stream);
    case 128: return launch_rows_hd<CODE, 128>(p, a, block_rows, mixed, rows, stream);
    case 256: return launch_rows_hd<CODE, 256>(p, a, block_rows, mixed, rows, stream);
  }
  return fail(TFX_ERR_UNSUPPORTED, "tfx_paged_attention: head_dim %d", head_dim);
}

}  // namespace tfx
