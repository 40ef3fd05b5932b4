// Attention of a few query rows over a paged cache, on mma.sync: every
// head_dim, cache type and number of rows. Included by one translation unit
// per cache type.
//
// Rows: the `group` query heads that read one key/value head are rows of the
// same block (row = token * group + head in group), so a cached key is read
// once for all of them. A CTA takes 16 * MT rows of one (sequence, key/value
// head) and one range of its keys. Its 4 warps take the range's KT-key tiles
// in turn, each with a ring of NS tiles of its own in shared memory (cp.async,
// no barrier between warps) and its own running maximum and sum per row; they
// are merged through shared memory at the end.
//
// 8-bit caches are expanded to fp16 in registers, between ldmatrix and the
// product, without the scales: a key's scale multiplies its column of scores,
// a value's scale its column of weights, both in fp32. Weights are rounded to
// fp16 for the second product; so that w * scale neither overflows nor loses
// bits for scales far from 1, it is divided by the largest scale seen so far
// (U, the accumulator's unit), which is put back at the end.
//
// Fragment orders. An 8x8 ldmatrix block of 16-bit words holds 8 keys x 16
// codes. Scores: thread (g, t) gets codes 4t..4t+3 of key g and uses (4t, 4t+1)
// and (4t+2, 4t+3) as the B operand's k pairs; the sum over k does not depend
// on the order as long as Q's fragments take the same one. Second product,
// transposed load: the thread gets dims 2g and 2g+1 of keys 2t and 2t+1; the
// even dims make one 8-wide column block of the product, the odd dims another,
// and the thread ends up with dims 4t..4t+3 of each 16.
//
// Masked keys. A weight of 0 does not hide an infinity or NaN among the values
// (0 * inf), so values beyond the sequence are loaded as zeros, and in tiles
// that some rows of the block see and others do not, non-finite fp16 values
// (NaN codes) are cleared before the product and added at the end to the rows
// that see them. (A scale that is not finite stays in its row: it multiplies
// weights, which are 0 where masked.)
#pragma once

#include "paged.cuh"

namespace tfx {
namespace {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = 32 * kRowsWarps;

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
__device__ __forceinline__ void rows_ldsm2_t(uint32_t addr, uint32_t& r0, uint32_t& r1) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(r0), "=r"(r1) : "r"(addr) : "memory");
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

template <int CODE, int HD, int MT>
struct RowsCfg {
  static constexpr int kHDP = HD < 16 ? 16 : HD;  // width of the first product (zero padded)
  static constexpr int kRowBytes = HD * code_bytes(CODE);
  static constexpr int kU = kRowBytes / 16;  // 16-byte chunks of a cached row
  // Rows an odd number of chunks apart: ldmatrix without bank conflicts.
  static constexpr int kPitch = ((kHDP * code_bytes(CODE) / 16) | 1) * 16;
  static constexpr int kQPitch = (kHDP + 8) * 2;
  // Keys of a warp's tile: about 2 KB of K (small tiles keep more warps on an
  // SM), at most 64 / MT (registers: the scores), at least what one x4
  // ldmatrix of codes covers.
  static constexpr int kWant = 2048 / kRowBytes < 16 ? 16 : 2048 / kRowBytes;
  static constexpr int kMost = 64 / MT;
  static constexpr int kLeast = (CODE != kCodeF16 && HD == 16) ? 32 : 16;
  static constexpr int kKT0 = kWant < kMost ? kWant : kMost;
  static constexpr int kKT = kKT0 < kLeast ? kLeast : kKT0;
  static constexpr int NS = 3;
  static constexpr int kTileBytes = kKT * kPitch;
  static constexpr int kScaleBytes = CODE == kCodeF16 ? 0 : 2 * kKT * 4;
  // K, V, their scales, the bits of keys that exist
  static constexpr int kStageBytes = 2 * kTileBytes + kScaleBytes + 16;
  static constexpr int kQBytes = 16 * MT * kQPitch;
  static constexpr int kRing = kRowsWarps * NS * kStageBytes;
  static constexpr int kMerge = kRowsWarps * 16 * (HD + 4) * 4;  // one 16-row block at a time
  static constexpr int kFlag = kQBytes + (kRing > kMerge ? kRing : kMerge);
  static constexpr int kSmem = kFlag + 16;
  static_assert(kSmem <= 227 * 1024, "shared-memory budget");
  static_assert(kKT <= 64 && kKT % 16 == 0, "tile of 16 to 64 keys");
};

template <int CODE, int HD, int MT>
__global__ void __launch_bounds__(kRowsThreads)
    paged_rows_kernel(const __grid_constant__ Paged p, const __grid_constant__ PagedAttn a,
                      int row_blocks) {
  grid_dep_wait();
  grid_dep_launch();
  using C = RowsCfg<CODE, HD, MT>;
  constexpr int KT = C::kKT, NS = C::NS, HDP = C::kHDP, U = C::kU;
  constexpr int NT_S = KT / 8;                        // 8-key column blocks of the scores
  constexpr int NT_O = HD / 8;                        // 8-dim column blocks of the output
  constexpr int KS = HDP / 16;                        // 16-wide steps of the first product
  constexpr bool kQuant = CODE != kCodeF16;
  extern __shared__ __align__(16) uint8_t smem_rows[];
  uint8_t* sQ = smem_rows;
  int* flag = reinterpret_cast<int*>(smem_rows + C::kFlag);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int b = blockIdx.z, hk = blockIdx.y;
  const int split = blockIdx.x / row_blocks;
  // The last rows see the most keys: they go first.
  const int rb = row_blocks - 1 - static_cast<int>(blockIdx.x) % row_blocks;
  const PagedSeq seq = paged_seq(p, b);
  const int rows = seq.n * a.group;  // below 2^31: checked on the host
  const int r0 = rb * 16 * MT;
  if (r0 >= rows) return;
  // Keys that row r sees: [0, lim(r)).
  auto lim_of = [&](int r) {
    return a.causal ? min(seq.len, max(0, seq.pos0 + r / a.group + 1)) : seq.len;
  };
  const int lim_first = lim_of(r0), lim_last = lim_of(min(r0 + 16 * MT, rows) - 1);
  const bool is_split = paged_is_split(a, seq);
  if (!is_split && split > 0) return;
  const int k_begin = is_split ? split * a.kps : 0;
  const int k_end = is_split ? min(lim_last, k_begin + a.kps) : lim_last;
  if (is_split && k_begin >= lim_last) return;  // not looked at when the splits are joined

  // ---- queries, zero rows behind the last one
  for (int i = threadIdx.x; i < 16 * MT * (HD / 8); i += kRowsThreads) {
    const int r = i / (HD / 8), c = i % (HD / 8), row = r0 + r;
    const bool ok = row < rows;
    const int tok = seq.row0 + (ok ? row / a.group : 0);
    const int head = hk * a.group + (ok ? row % a.group : 0);
    rows_cp16(smem_u32(sQ + r * C::kQPitch + c * 16),
              a.q + static_cast<int64_t>(tok) * a.ld_q + head * HD + c * 8, ok);
  }
  if constexpr (HD < 16) {
    for (int i = threadIdx.x; i < 16 * MT; i += kRowsThreads)
      *reinterpret_cast<uint4*>(sQ + i * C::kQPitch + HD * 2) = make_uint4(0, 0, 0, 0);
  }
  if (threadIdx.x == 0) *flag = 0;
  rows_commit();

  // ---- this warp's ring
  uint8_t* ring = smem_rows + C::kQBytes + warp * NS * C::kStageBytes;
  if constexpr (HD < 16) {
    for (int i = lane; i < NS * 2 * KT; i += 32)
      *reinterpret_cast<uint4*>(ring + (i / (2 * KT)) * C::kStageBytes + (i % (2 * KT)) * C::kPitch +
                                HD * 2) = make_uint4(0, 0, 0, 0);
  }
  const int n_tiles = k_end > k_begin + warp * KT
                          ? (k_end - k_begin - warp * KT + kRowsWarps * KT - 1) / (kRowsWarps * KT)
                          : 0;
  const uint8_t* kb = static_cast<const uint8_t*>(p.k) + hk * p.head_stride * code_bytes(CODE);
  const uint8_t* vb = static_cast<const uint8_t*>(p.v) + hk * p.head_stride * code_bytes(CODE);
  auto tile_key = [&](int i) { return k_begin + (i * kRowsWarps + warp) * KT; };
  // Page of this lane's keys of tile i (lane and lane + 32), one tile ahead.
  int pg[2];
  auto look_up = [&](int i) {
    const int key = tile_key(i) + lane;
    pg[0] = i < n_tiles && key < k_end && lane < KT ? paged_page(p, b, key) : -1;
    if constexpr (KT > 32)
      pg[1] = i < n_tiles && key + 32 < k_end ? paged_page(p, b, key + 32) : -1;
  };
  auto load = [&](int i) {
    uint8_t* st = ring + (i % NS) * C::kStageBytes;
    const int k0 = tile_key(i);
#pragma unroll
    for (int it = 0; it < KT * U / 32 + (KT * U % 32 != 0); ++it) {
      const int c = it * 32 + lane, r = c / U, col = c % U;
      int page = __shfl_sync(0xffffffffu, pg[0], r & 31);
      if constexpr (KT > 32) {
        const int hi = __shfl_sync(0xffffffffu, pg[1], r & 31);
        page = r < 32 ? page : hi;
      }
      if (KT * U % 32 == 0 || c < KT * U) {
        const int64_t off = page >= 0 ? paged_offset(p, page, k0 + r) * code_bytes(CODE) : 0;
        rows_cp16(smem_u32(st + r * C::kPitch + col * 16), kb + off + col * 16, page >= 0);
        rows_cp16(smem_u32(st + C::kTileBytes + r * C::kPitch + col * 16), vb + off + col * 16,
                  page >= 0);
      }
    }
    if constexpr (kQuant) {
      float* sc = reinterpret_cast<float*>(st + 2 * C::kTileBytes);
#pragma unroll
      for (int u = 0; u < (KT + 31) / 32; ++u) {
        if (lane + 32 * u < KT) {
          const bool ok = pg[u] >= 0;
          const int64_t so = ok ? paged_scale_offset(p, pg[u], hk, k0 + 32 * u + lane) : 0;
          rows_cp4(smem_u32(sc + 32 * u + lane), p.k_scale + so, ok);
          rows_cp4(smem_u32(sc + KT + 32 * u + lane), p.v_scale + so, ok);
        }
      }
    }
    uint32_t* bits = reinterpret_cast<uint32_t*>(st + 2 * C::kTileBytes + C::kScaleBytes);
#pragma unroll
    for (int u = 0; u < (KT + 31) / 32; ++u) {
      const uint32_t m = __ballot_sync(0xffffffffu, pg[u] >= 0);
      if (lane == 0) bits[u] = m;
    }
  };
  look_up(0);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    if (i < n_tiles) load(i);
    rows_commit();
    look_up(i + 1);
  }
  rows_wait<NS - 1>();  // the queries (the oldest group)
  __syncthreads();

  // Q fragments; with more than one 16-row block they are read again for each
  // tile (registers).
  uint32_t qf[MT == 1 ? KS : 1][4];
  auto load_q = [&](int mt, int kk, uint32_t (&f)[4]) {
    if constexpr (!kQuant) {
      rows_ldsm4(smem_u32(sQ + (mt * 16 + (lane & 15)) * C::kQPitch + kk * 32 + (lane >> 4) * 16),
                 f);
    } else {  // columns 4t..4t+3 of each 16, see the file's comment
      const uint2 lo = *reinterpret_cast<const uint2*>(sQ + (mt * 16 + g) * C::kQPitch + kk * 32 +
                                                       t * 8);
      const uint2 hi = *reinterpret_cast<const uint2*>(sQ + (mt * 16 + g + 8) * C::kQPitch +
                                                       kk * 32 + t * 8);
      f[0] = lo.x;
      f[1] = hi.x;
      f[2] = lo.y;
      f[3] = hi.y;
    }
  };
  if constexpr (MT == 1) {
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) load_q(0, kk, qf[kk]);
  }

  float o[MT][NT_O][4];
  float m_run[MT][2], l_run[MT][2];
  int lim[MT][2];
  float unit = 1e-37f;  // U (its reciprocal stays finite)
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int i = 0; i < NT_O; ++i) o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.f;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m_run[mt][r] = -INFINITY;
      l_run[mt][r] = 0.f;
      lim[mt][r] = lim_of(min(r0 + mt * 16 + g + 8 * r, rows - 1));
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

    // ---- S = Q K^T
    float s[MT][NT_S][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < NT_S; ++j) s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.f;
    auto product = [&](int j, int kk, uint32_t b0, uint32_t b1) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if constexpr (MT == 1) {
          rows_mma(s[0][j], qf[kk], b0, b1);
        } else {
          uint32_t f[4];
          load_q(mt, kk, f);
          rows_mma(s[mt][j], f, b0, b1);
        }
      }
    };
    if constexpr (!kQuant) {
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        uint32_t f[MT][4];
        if constexpr (MT > 1) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) load_q(mt, kk, f[mt]);
        }
#pragma unroll
        for (int j = 0; j < NT_S; j += 2) {
          uint32_t r[4];
          rows_ldsm4(smem_u32(st + (j * 8 + (lane >> 4) * 8 + (lane & 7)) * C::kPitch + kk * 32 +
                              ((lane >> 3) & 1) * 16),
                     r);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            if constexpr (MT == 1) {
              rows_mma(s[0][j], qf[kk], r[0], r[1]);
              rows_mma(s[0][j + 1], qf[kk], r[2], r[3]);
            } else {
              rows_mma(s[mt][j], f[mt], r[0], r[1]);
              rows_mma(s[mt][j + 1], f[mt], r[2], r[3]);
            }
          }
        }
      }
    } else {
      // Blocks of 8 keys x 16 codes, four at a time: block n is column block
      // n / KS, step n % KS.
#pragma unroll
      for (int n = 0; n < NT_S * KS; n += 4) {
        uint32_t r[4];
        const int mine = n + (lane >> 3);
        rows_ldsm4(smem_u32(st + ((mine / KS) * 8 + (lane & 7)) * C::kPitch + (mine % KS) * 16), r);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          product((n + m) / KS, (n + m) % KS, codes_to_h2<CODE, 0, 1>(r[m]),
                  codes_to_h2<CODE, 2, 3>(r[m]));
      }
    }

    // ---- keys that exist; the accumulator's unit; values that must not leak
    uint32_t bits[(KT + 31) / 32];
    bool full = true;
#pragma unroll
    for (int u = 0; u < (KT + 31) / 32; ++u) {
      bits[u] = reinterpret_cast<const uint32_t*>(st + 2 * C::kTileBytes + C::kScaleBytes)[u];
      full = full && bits[u] == (KT < 32 ? (1u << (KT & 31)) - 1u : 0xffffffffu);
    }
    const bool need_mask = !full || k0 + KT > lim_first;  // warp-uniform
    float unit_corr = 1.f, inv_unit = 0.f;
    if constexpr (kQuant) {
      uint32_t top = 0;
#pragma unroll
      for (int u = 0; u < (KT + 31) / 32; ++u) {
        const uint32_t x = lane + 32 * u < KT ? __float_as_uint(sc[KT + 32 * u + lane]) & 0x7fffffffu
                                              : 0u;
        top = max(top, x < 0x7f800000u ? x : 0u);
      }
      top = __reduce_max_sync(0xffffffffu, top);  // non-negative floats order as integers
      if (__uint_as_float(top) > unit) {
        unit_corr = unit / __uint_as_float(top);
        unit = __uint_as_float(top);
      }
      inv_unit = 1.f / unit;
    }
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
              if (h2_not_finite(w[e])) {
                hit = true;
                if ((w[e] & 0x7c00u) == 0x7c00u) w[e] &= 0xffff0000u;
                if ((w[e] & 0x7c000000u) == 0x7c000000u) w[e] &= 0xffffu;
              }
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

    // ---- mask and running softmax (scores in the log2 domain)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < NT_S; ++j) {
        float f0 = a.scale_log2, f1 = a.scale_log2;
        if constexpr (kQuant) {
          const float2 ks = *reinterpret_cast<const float2*>(sc + j * 8 + 2 * t);
          f0 *= ks.x;
          f1 *= ks.y;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float val = s[mt][j][e] * ((e & 1) ? f1 : f0);
          if (need_mask) {
            const int kk = j * 8 + 2 * t + (e & 1);
            if (k0 + kk >= lim[mt][e >> 1] || !((bits[kk >> 5] >> (kk & 31)) & 1u)) val = -INFINITY;
          }
          s[mt][j][e] = val;
          mx[e >> 1] = fmaxf(mx[e >> 1], val);
        }
      }
      float corr[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float m_new = fmaxf(m_run[mt][r], mx[r]);
        const float m_ref = m_new == -INFINITY ? 0.f : m_new;  // nothing seen yet: weights 0, no NaN
        corr[r] = fast_exp2(m_run[mt][r] - m_ref);
        m_run[mt][r] = m_new;
        mx[r] = m_ref;
      }
      float rs[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NT_S; ++j) {
        float v0 = 1.f, v1 = 1.f;
        if constexpr (kQuant) {
          const float2 vs = *reinterpret_cast<const float2*>(sc + KT + j * 8 + 2 * t);
          v0 = vs.x * inv_unit;
          v1 = vs.y * inv_unit;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w = fast_exp2(s[mt][j][e] - mx[e >> 1]);
          rs[e >> 1] += w;
          if constexpr (kQuant)  // a masked key's scale may be anything
            s[mt][j][e] = w == 0.f ? 0.f : w * ((e & 1) ? v1 : v0);
          else
            s[mt][j][e] = w;
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) l_run[mt][r] = l_run[mt][r] * corr[r] + rs[r];
      if constexpr (kQuant) {
        corr[0] *= unit_corr;
        corr[1] *= unit_corr;
      }
#pragma unroll
      for (int n = 0; n < NT_O; ++n) {
        o[mt][n][0] *= corr[0];
        o[mt][n][1] *= corr[0];
        o[mt][n][2] *= corr[1];
        o[mt][n][3] *= corr[1];
      }
    }

    // ---- O += P V, 16 keys at a time
#pragma unroll
    for (int kk = 0; kk < KT / 16; ++kk) {
      uint32_t pf[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        pf[mt][0] = pack_half2(s[mt][2 * kk][0], s[mt][2 * kk][1]);
        pf[mt][1] = pack_half2(s[mt][2 * kk][2], s[mt][2 * kk][3]);
        pf[mt][2] = pack_half2(s[mt][2 * kk + 1][0], s[mt][2 * kk + 1][1]);
        pf[mt][3] = pack_half2(s[mt][2 * kk + 1][2], s[mt][2 * kk + 1][3]);
      }
      const uint32_t row = smem_u32(sv + (kk * 16 + (lane & 15)) * C::kPitch);
      if constexpr (!kQuant) {
        if constexpr (NT_O == 1) {
          uint32_t b0, b1;
          rows_ldsm2_t(row, b0, b1);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) rows_mma(o[mt][0], pf[mt], b0, b1);
        } else {
#pragma unroll
          for (int n = 0; n < NT_O; n += 2) {
            uint32_t r[4];
            rows_ldsm4_t(row + n * 16 + (lane >> 4) * 16, r);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              rows_mma(o[mt][n], pf[mt], r[0], r[1]);
              rows_mma(o[mt][n + 1], pf[mt], r[2], r[3]);
            }
          }
        }
      } else {
        auto block = [&](int n, uint32_t lo, uint32_t hi) {  // 16 dims; lo, hi: keys 0-7, 8-15
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) {
            const uint32_t b0 = odd ? codes_to_h2<CODE, 1, 3>(lo) : codes_to_h2<CODE, 0, 2>(lo);
            const uint32_t b1 = odd ? codes_to_h2<CODE, 1, 3>(hi) : codes_to_h2<CODE, 0, 2>(hi);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) rows_mma(o[mt][2 * n + odd], pf[mt], b0, b1);
          }
        };
        if constexpr (HD == 16) {
          uint32_t lo, hi;
          rows_ldsm2_t(row, lo, hi);
          block(0, lo, hi);
        } else {
#pragma unroll
          for (int n = 0; n < HD / 16; n += 2) {
            uint32_t r[4];
            rows_ldsm4_t(row + n * 16 + (lane >> 4) * 16, r);
            block(n, r[0], r[1]);
            block(n + 1, r[2], r[3]);
          }
        }
      }
    }
  }
  rows_wait<0>();
  if (cleared && lane == 0) *flag = 1;
  __syncthreads();
  const bool fix = *flag != 0;

  // ---- merge the warps, one 16-row block at a time
  float* mo = reinterpret_cast<float*>(smem_rows + C::kQBytes);  // [warp][16][HD]
  float* mm = mo + kRowsWarps * 16 * HD;                         // [warp][16]
  float* ml = mm + kRowsWarps * 16;
  const float back = kQuant ? unit : 1.f;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (r0 + mt * 16 >= rows) break;  // uniform
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l_run[mt][r] += __shfl_xor_sync(0xffffffffu, l_run[mt][r], 1);
      l_run[mt][r] += __shfl_xor_sync(0xffffffffu, l_run[mt][r], 2);
      float* dst = mo + (warp * 16 + g + 8 * r) * HD;
      if constexpr (!kQuant) {
#pragma unroll
        for (int n = 0; n < NT_O; ++n)
          *reinterpret_cast<float2*>(dst + n * 8 + 2 * t) =
              make_float2(o[mt][n][2 * r], o[mt][n][2 * r + 1]);
      } else {
#pragma unroll
        for (int n = 0; n < HD / 16; ++n)
          *reinterpret_cast<float4*>(dst + n * 16 + 4 * t) =
              make_float4(o[mt][2 * n][2 * r] * back, o[mt][2 * n + 1][2 * r] * back,
                          o[mt][2 * n][2 * r + 1] * back, o[mt][2 * n + 1][2 * r + 1] * back);
      }
      if (t == 0) {
        mm[warp * 16 + g + 8 * r] = m_run[mt][r];
        ml[warp * 16 + g + 8 * r] = l_run[mt][r];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (HD / 4); i += kRowsThreads) {
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4, row = r0 + mt * 16 + r;
      if (row >= rows) continue;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) m = fmaxf(m, mm[w * 16 + r]);
      float acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) {
        const float mw = mm[w * 16 + r];
        if (mw == -INFINITY && ml[w * 16 + r] == 0.f) continue;  // this warp saw no key
        const float f = fast_exp2(mw - m);
        const float4 x = *reinterpret_cast<const float4*>(mo + (w * 16 + r) * HD + d);
        acc[0] += f * x.x;
        acc[1] += f * x.y;
        acc[2] += f * x.z;
        acc[3] += f * x.w;
        l += f * ml[w * 16 + r];
      }
      if (fix) {  // non-finite values cleared from shared tiles: to the rows that see them
        const int hi = min(lim_of(row), k_end);
        for (int key = max(k_begin, lim_first - KT); key < hi; ++key) {
          const int page = paged_page(p, b, key);
          if (page < 0) continue;
          const int64_t at = paged_offset(p, page, key) + hk * p.head_stride + d;
          const float vs = kQuant ? p.v_scale[paged_scale_offset(p, page, hk, key)] : 1.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = paged_value<CODE>(p.v, at + e, vs);
            if (!isfinite(x)) acc[e] += x;
          }
        }
      }
      const int tok = seq.row0 + row / a.group, head = hk * a.group + row % a.group;
      if (is_split) {
        const int64_t at = (static_cast<int64_t>(tok) * (p.kv_heads * a.group) + head) * a.splits +
                           split;
        *reinterpret_cast<float4*>(a.part_o + at * HD + d) =
            make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) a.part_ml[at] = make_float2(m, l);
      } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;  // no key seen: zero (NaN sums stay NaN)
        *reinterpret_cast<uint2*>(a.out + static_cast<int64_t>(tok) * a.ld_out + head * HD + d) =
            make_uint2(pack_half2(acc[0] * inv, acc[1] * inv), pack_half2(acc[2] * inv, acc[3] * inv));
      }
    }
    __syncthreads();
  }
}

template <int CODE, int HD, int MT>
int launch_rows(const Paged& p, const PagedAttn& a, int64_t rows, cudaStream_t stream) {
  using C = RowsCfg<CODE, HD, MT>;
  static int done[kMaxDevices] = {0};
  auto kern = paged_rows_kernel<CODE, HD, MT>;
  int st = ensure_smem(reinterpret_cast<const void*>(kern), C::kSmem, done);
  if (st != TFX_OK) return st;
  const int64_t blocks = (rows + 16 * MT - 1) / (16 * MT);
  if (blocks * a.splits > 0x7fffffffLL)
    return fail(TFX_ERR_UNSUPPORTED, "tfx_paged_attention: too many rows");
  launch_pdl(kern, dim3(static_cast<unsigned>(blocks * a.splits), p.kv_heads, p.batch),
             dim3(kRowsThreads), C::kSmem, stream, p, a, static_cast<int>(blocks));
  return check_launch("paged_rows_kernel");
}

template <int CODE, int HD>
int launch_rows_hd(const Paged& p, const PagedAttn& a, int block_rows, int64_t rows,
                   cudaStream_t stream) {
  if constexpr (HD <= 64) {
    if (block_rows == 64) return launch_rows<CODE, HD, 4>(p, a, rows, stream);
  }
  if constexpr (HD <= 128) {
    if (block_rows == 32) return launch_rows<CODE, HD, 2>(p, a, rows, stream);
  }
  return launch_rows<CODE, HD, 1>(p, a, rows, stream);
}

}  // namespace

template <int CODE>
int launch_paged_rows(const Paged& p, const PagedAttn& a, int head_dim, int block_rows,
                      int64_t rows, cudaStream_t stream) {
  switch (head_dim) {
    case 8:
      if constexpr (CODE == kCodeF16) return launch_rows_hd<CODE, 8>(p, a, block_rows, rows, stream);
      break;
    case 16: return launch_rows_hd<CODE, 16>(p, a, block_rows, rows, stream);
    case 32: return launch_rows_hd<CODE, 32>(p, a, block_rows, rows, stream);
    case 64: return launch_rows_hd<CODE, 64>(p, a, block_rows, rows, stream);
    case 128: return launch_rows_hd<CODE, 128>(p, a, block_rows, rows, stream);
    case 256: return launch_rows_hd<CODE, 256>(p, a, block_rows, rows, stream);
  }
  return fail(TFX_ERR_UNSUPPORTED, "tfx_paged_attention: head_dim %d", head_dim);
}

}  // namespace tfx
