// Attention of many query rows (chunks of prompts) over a paged cache on the
// 5th-generation tensor cores, head_dim 64, 128 and 256. Included by one
// translation unit per cache type.
//
// The `group` query heads that read one key/value head are rows of the same
// tile: a 128-row tile holds 128 / group tokens x group heads (TMA box of q;
// the last 128 % group rows stay unused). CTA = two such tiles A and B of one
// (sequence, key/value head) that share every 128-key tile, and one range of
// the keys; 12 warps (8 bit: 16), one CTA per SM:
//   warps 4..7, 8..11  softmax of A and of B; thread = row = TMEM lane
//   warps 1, 2         MMA issuers of A and of B (one lane)
//   fp16:  warp 0 loads K and V, a TMA box per page and 64 columns (lane =
//          box); warp 3 looks after V tiles that hold keys which not every
//          row sees
//   8 bit: warp 0 loads raw tiles (a box per page), warps 12..15 expand 32 rows
//          each of every K and V tile to fp16, a lane per row (both tiles are
//          swizzled: no bank conflicts), warp 3 brings the scales
// A key tile is 128 consecutive positions, 128 / page_size pages or a part of
// one; pages outside the pool are boxes outside the tensor map and read as
// zeros.
//
// S = Q K^T (128 x N keys) goes to TMEM, the softmax warps write P over it or
// beside it, O += P V takes P from TMEM and V MN-major from the row-major tile.
// A row's reference maximum moves only when it is exceeded by more than 2^8
// (O is then rescaled in TMEM). A tile's S is two parts of N = 64 keys, so that
// one is being exponentiated while the other is multiplied and replaced (with
// N = 128 at head_dim 128 each tile's chain S - P - PV - S was serial: 870 against
// 1029 TFLOP/s, one fp16 head_dim 128 sequence of 16k, not causal). head_dim 64:
// P has columns of its own (S 2 x 128, P 2 x 64, O 2 x 64), so the next S is
// computed as soon as this one is in registers; head_dim 128: O fills half of
// TMEM and P lies over S. head_dim 256: one query tile to a CTA and tiles of 64
// keys (O alone is 256 columns, Q 64 KB), two of them in S.
//
// 8-bit codes are expanded to fp16 exactly, without the scales: a key's scale
// multiplies its column of scores, a value's is an exponent added to it (see
// value_scale_log2), in fp32 (as fp16 factors of the tiles they cost as much, in the
// warps that expand, and five times the error: a key's rounded scale multiplies its
// whole score).
//
// What a row does not see must not reach it, and 0 * inf does: V rows behind
// the sequence are cleared; in tiles that some rows of the CTA see and others
// do not, non-finite values are cleared before the product and added at the
// end to the rows that see them. Rows whose scores hold a NaN or +inf are NaN.
#pragma once

#include <type_traits>

#include "paged.cuh"

namespace tfx {
namespace {

constexpr int kPtConvert = 4;  // 8 bit: warps that expand
constexpr int kPtTile = 128;
constexpr float kPtRescale = 8.0f;  // O is rescaled when a row's maximum grows by more than 2^8
// fp16: of 8 pairs of exponentials, so many on the FMA pipe. 8 bit: none; its warps
// have the scales to multiply as well, and are bound by the instructions that they
// issue (16k int8 sequence, head_dim 64, not causal: 2318, 2447 and 2436 us with 0, 1
// and 2 of 8).
constexpr int kPtPoly = 2;
constexpr uint32_t kPtCols = 512;

template <int CODE, int HD>
struct PtCfg {
  static constexpr bool kQuant = CODE != kCodeF16;
  static constexpr int kThreads = kQuant ? 512 : 384;
  static constexpr int kNT = HD == 256 ? 1 : 2;            // query tiles (TMEM, shared memory)
  static constexpr int kKT = HD == 256 ? 64 : kPtTile;     // keys of a K or V tile
  static constexpr int kStages = HD == 64 ? 4 : 2;
  static constexpr int kBlocks = HD / 64;                  // 64-column blocks, 128-byte rows
  static constexpr int kQBlock = kPtTile * 128, kQBytes = kPtTile * HD * 2;
  static constexpr int kBlockBytes = kKT * 128, kTileBytes = kKT * HD * 2;
  static constexpr int kRaws = kQuant ? (HD == 64 ? 4 : 2) : 0;  // raw tiles: K and V in turn
  static constexpr int kRawRow = HD < 128 ? HD : 128;            // bytes: blocks of 128 columns
  static constexpr int kRawBytes = kKT * HD;
  static constexpr int kQ = 0;
  static constexpr int kK = kNT * kQBytes;
  static constexpr int kV = kK + kStages * kTileBytes;
  static constexpr int kR = kV + kStages * kTileBytes;
  // 8 bit: scales of kSlots parts of tiles: K's times the softmax scale, log2 of V's and
  // one over V's (with two, and slack to align shared memory in, the two query tiles of
  // head_dim 128 wait for one another: 750 against 702 us, prompt_parts_grouped_int8)
  static constexpr int kSlots = 3;
  static constexpr int kSlotFloats = 3 * 64;
  static constexpr int kSc = kR + kRaws * kRawBytes;
  static constexpr int kBar = kSc + (kQuant ? kSlots * kSlotFloats * 4 : 0);
  static constexpr int kBarBytes = HD == 64 ? 1024 : 512;
  static constexpr int kSmem = kBar + kBarBytes;
  static constexpr bool kSepP = HD == 64 && !kQuant;  // P has its own TMEM columns
  static constexpr int kParts = kSepP || kKT == 64 ? 1 : 2;  // a tile's S in so many parts
  static constexpr int kKeys = kKT / kParts;                 // keys of one
  static constexpr int kBufs = kSepP ? 1 : 2;                // parts of S in TMEM at a time
  static constexpr uint32_t kColP = kSepP ? 2 * kPtTile : 0;
  static constexpr uint32_t kPStride = kSepP ? kPtTile / 2 : kPtTile;  // of a query tile
  static constexpr uint32_t kColO = kNT == 1 ? kPtTile : kSepP ? 3 * kPtTile : 2 * kPtTile;
  static_assert(kColO + kNT * HD <= kPtCols, "TMEM budget");
  static_assert(kSmem <= 227 * 1024, "shared-memory budget");
};

__device__ __forceinline__ void pt_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar,
                                           int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// Four codes to two fp16 pairs, exact.
template <int CODE>
__device__ __forceinline__ void pt_expand(uint32_t x, uint32_t& lo, uint32_t& hi) {
  lo = codes_to_h2<CODE, 0, 1>(x);
  hi = codes_to_h2<CODE, 2, 3>(x);
}

// Adds the non-finite values of keys [lo, hi) to a finished row (rare; out of
// the kernel's registers): exactly what its weights, all above 0, make of them.
template <int CODE, int HD>
__device__ __noinline__ void pt_add_cleared(const Paged& p, int b, int hk, int lo, int hi,
                                            float* part, __half* out) {
  for (int key = lo; key < hi; ++key) {
    const int page = paged_page(p, b, key);
    if (page < 0) continue;
    const int64_t at = paged_offset(p, page, key) + hk * p.head_stride;
    float vs = CODE != kCodeF16 ? p.v_scale[paged_scale_offset(p, page, hk, key)] : 1.f;
    if (value_scale_bad(vs)) vs = __uint_as_float(0x7fc00000u);
    for (int d = 0; d < HD; ++d) {
      const float y = paged_value<CODE>(p.v, at + d, vs);
      if (isfinite(y)) continue;
      if (part != nullptr) part[d] += y;
      else out[d] = __float2half_rn(__half2float(out[d]) + y);
    }
  }
}

template <int CODE, int HD>
__global__ void __launch_bounds__((PtCfg<CODE, HD>::kThreads), 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Paged p,
                    const __grid_constant__ PagedAttn a, int row_blocks, int* err) {
  grid_dep_wait();
  grid_dep_launch();
  using L = PtCfg<CODE, HD>;
  constexpr int S = L::kStages;
  constexpr bool kQuant = L::kQuant;
  constexpr int R = L::kRaws > 0 ? L::kRaws : 1;

  // ---- this CTA's work
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.x, b = blockIdx.y;
  const int split = static_cast<int>(blockIdx.z) % a.splits_tc;
  // The last rows of all sequences and heads see the most keys: they go first.
  const int rb = row_blocks - 1 - static_cast<int>(blockIdx.z) / a.splits_tc;
  const int group = a.group, tile_tokens = kPtTile / group;
  const PagedSeq seq = paged_attn_seq(p, a, b);
  const int i0 = rb * L::kNT * tile_tokens;  // first token
  if (i0 >= seq.n || !paged_is_tc(a, seq)) return;
  auto lim_of = [&](int i) {  // token i sees keys [0, lim)
    return a.causal ? min(seq.len, max(0, seq.pos0 + i + 1)) : seq.len;
  };
  const bool is_split = paged_is_split(a, seq);
  // Splits behind the sequence.
  if (is_split ? static_cast<int64_t>(split) * a.kps_tc >= seq.len : split > 0) return;
  const int k_begin = is_split ? split * a.kps_tc : 0;
  const int k_stop = is_split ? paged_split_end(a, seq, split, k_begin) : seq.len;  // of the split
  auto tiles_of = [&](int x) {
    const int first = i0 + x * tile_tokens;
    if (first >= seq.n) return 0;
    const int lim = min(lim_of(min(first + tile_tokens, seq.n) - 1), k_stop);
    return lim > k_begin ? (lim - k_begin + L::kKT - 1) / L::kKT : 0;
  };
  const int nA = tiles_of(0), nB = L::kNT == 2 ? tiles_of(1) : 0, n_iter = max(nA, nB);
  if (is_split && n_iter == 0) return;  // not looked at when the splits are joined
  // Keys from here on are not seen by every row; the first tile that holds one.
  const int lim_first = lim_of(i0);
  const int j_partly = max(0, lim_first - k_begin) / L::kKT;

  // (aligned as declared: there is no room for slack, and addresses are constants.
  // With slack, prompt_part_fp16 549 us and so 494.)
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0u) {
    record_error(err, kDevTimeoutOther);
    return;
  }
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* k_full = q_full + 1;
  uint64_t* v_full = k_full + S;        // fp16: V loaded
  uint64_t* v_seen = v_full + S;        // fp16: and warp 3 knows
  uint64_t* v_ready = v_seen + S;       // V may be multiplied
  uint64_t* k_empty = v_ready + S;      // [2][S]
  uint64_t* v_empty = k_empty + 2 * S;  // [2][S]
  constexpr int N = L::kParts, SB = L::kBufs;
  uint64_t* s_full = v_empty + 2 * S;   // [2][SB] S of a part computed
  uint64_t* s_free = s_full + 2 * SB;   // [2][SB] in registers (separate P only)
  uint64_t* p_full = s_free + 2 * SB;   // [2][SB] its P written
  uint64_t* o_done = p_full + 2 * SB;   // [2][SB] and multiplied
  uint64_t* drain = o_done + 2 * SB;    // [2]
  uint64_t* r_full = drain + 2;         // [R] raw tile loaded
  uint64_t* r_empty = r_full + R;       // [R] raw tile expanded by all its warps
  constexpr int SC = L::kSlots;
  uint64_t* c_full = r_empty + R;       // [SC] scales of a part
  uint64_t* c_empty = c_full + SC;      // [2][SC]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(c_empty + 2 * SC);
  volatile int* cleared = reinterpret_cast<int*>(tmem_slot + 1);
  float* scales = reinterpret_cast<float*>(smem + L::kSc);
  static_assert((1 + 8 * S + 2 + 8 * SB + 2 * R + 3 * SC) * 8 + 8 <= L::kBarBytes, "barrier space");

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    mbar_init(q_full, 1);
    for (int s = 0; s < S; ++s) {
      mbar_init(&k_full[s], kQuant ? kPtConvert : 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_seen[s], 1);
      mbar_init(&v_ready[s], kQuant ? kPtConvert : 1);
      for (int x = 0; x < 2; ++x) {
        mbar_init(&k_empty[x * S + s], 1);
        mbar_init(&v_empty[x * S + s], 1);
      }
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&drain[x], 1);
      for (int h = 0; h < SB; ++h) {
        mbar_init(&s_free[x * SB + h], 4);
        mbar_init(&s_full[x * SB + h], 1);
        mbar_init(&p_full[x * SB + h], 4);
        mbar_init(&o_done[x * SB + h], 1);
      }
    }
    for (int r = 0; r < R; ++r) {
      mbar_init(&r_full[r], 1);
      mbar_init(&r_empty[r], kPtConvert);
    }
    for (int c = 0; c < SC; ++c) {
      mbar_init(&c_full[c], 1);
      mbar_init(&c_empty[c], 4);
      mbar_init(&c_empty[SC + c], 4);
    }
    *cleared = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kPtCols);
    tmem_relinquish();
  }
  // Pages of the range that are outside the pool: rare, so looked for once.
  int hole = 0;
  {
    const int last = min(k_stop, min(seq.len, lim_of(min(i0 + L::kNT * tile_tokens, seq.n) - 1)));
    for (int pos = k_begin + (static_cast<int>(threadIdx.x) << p.page_shift); pos < last;
         pos += L::kThreads << p.page_shift)
      hole |= paged_page(p, b, pos) < 0;
  }
  tc_fence_before();
  const bool holes = __syncthreads_or(hole);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int page_rows = min(1 << p.page_shift, L::kKT);  // of a tile in one page
  const int tile_pages = L::kKT / page_rows;

  // Page of a tile's part, as a coordinate (outside the map: zeros).
  auto page_coord = [&](int j, int part) {
    const int pos = k_begin + j * L::kKT + part * page_rows;
    const int page = j < n_iter && pos < seq.len ? paged_page(p, b, pos) : -1;
    return page < 0 ? p.num_pages : page;
  };
  auto slot_coord = [&](int j, int part) {
    return (k_begin + j * L::kKT + part * page_rows) & ((1 << p.page_shift) - 1);
  };
  auto stage_free = [&](uint64_t* empty, int j) {  // stage of tile j, which held tile j - S
    const uint32_t par = ((j / S) - 1) & 1;
    bool ok = true;
    if (j >= S) {
      if (j - S < nA) ok = mbar_wait_sleep(&empty[j % S], par, err, kDevTimeoutEmpty);
      if (ok && j - S < nB) ok = mbar_wait_sleep(&empty[S + j % S], par, err, kDevTimeoutEmpty);
    }
    return __all_sync(0xffffffffu, ok) != 0;
  };
  auto load_q = [&]() {
    if (lane == 0) {
      const int rows = tile_tokens * group;
      mbar_arrive_expect_tx(q_full, static_cast<uint32_t>(L::kNT * L::kBlocks * rows * 128));
#pragma unroll
      for (int x = 0; x < L::kNT; ++x)
#pragma unroll
        for (int cb = 0; cb < L::kBlocks; ++cb)
          tma_load_3d(smem + L::kQ + x * L::kQBytes + cb * L::kQBlock, &tm_q, q_full,
                      64 * cb, hk * group, seq.row0 + i0 + x * tile_tokens);
    }
  };

  if (warp == 0 || warp == 3 || warp >= 12) {
    if constexpr (!kQuant) {
      if (warp == 0) {
        // -------------------------------------------------- TMA of K and V
        load_q();
        // Lane = (part of the tile, 64-column block).
        const int part = lane % tile_pages, cb = lane / tile_pages;
        const bool mine = cb < L::kBlocks;
        const uint32_t dst = smem_u32(smem) + cb * L::kBlockBytes + part * page_rows * 128;
        int page = page_coord(0, part), k_issued = 0, issued = 0;
        for (int j = 0; j < n_iter; ++j) {
          const int st = j % S;
          const int next = page_coord(j + 1, part);
          if (!stage_free(k_empty, j)) break;
          if (lane == 0) mbar_arrive_expect_tx(&k_full[st], L::kTileBytes);
          __syncwarp();
          if (mine)
            pt_load_4d(dst + L::kK + st * L::kTileBytes, &tm_k, &k_full[st], 64 * cb,
                       slot_coord(j, part), hk, page);
          k_issued = j + 1;
          if (!stage_free(v_empty, j)) break;
          // (a barrier's parity tells only neighbouring phases apart: no load may start
          // before everyone who watches v_full knows of the one before)
          if (j >= S && !__all_sync(0xffffffffu, mbar_wait_sleep(&v_seen[st], ((j / S) - 1) & 1, err,
                                                                 kDevTimeoutEmpty)))
            break;
          if (lane == 0) mbar_arrive_expect_tx(&v_full[st], L::kTileBytes);
          __syncwarp();
          if (mine)
            pt_load_4d(dst + L::kV + st * L::kTileBytes, &tm_v, &v_full[st], 64 * cb,
                       slot_coord(j, part), hk, page);
          issued = j + 1;
          page = next;
        }
        // Our own copies land before the CTA may exit.
        mbar_wait(q_full, 0, nullptr, 0);
        for (int j = max(0, k_issued - S); j < k_issued; ++j)
          mbar_wait(&k_full[j % S], (j / S) & 1, nullptr, 0);
        for (int j = max(0, issued - S); j < issued; ++j)
          mbar_wait(&v_full[j % S], (j / S) & 1, nullptr, 0);
      } else {
        // ---------------------------------------------- V tiles not all see
        for (int j = 0; j < n_iter; ++j) {
          const int st = j % S, key0 = k_begin + j * L::kKT;
          if (!__all_sync(0xffffffffu,
                          mbar_wait_sleep(&v_full[st], (j / S) & 1, err, kDevTimeoutFull)))
            break;
          if (lane == 0) mbar_arrive(&v_seen[st]);
          if (j < j_partly) continue;
          uint8_t* tile = smem + L::kV + st * L::kTileBytes;
          bool found = false;
#pragma unroll 4
          for (int c = lane; c < L::kTileBytes / 16; c += 32) {
            // 16-byte chunk c lies in row (c / 8) % kKT of its 64-column block
            uint4* at = reinterpret_cast<uint4*>(tile) + c;
            const bool behind = key0 + ((c >> 3) & (L::kKT - 1)) >= seq.len;
            uint4 x = *at;
            bool hit = h2_clear(x.x);
            hit |= h2_clear(x.y);
            hit |= h2_clear(x.z);
            hit |= h2_clear(x.w);
            if (behind) *at = make_uint4(0u, 0u, 0u, 0u);
            else if (hit) *at = x;
            found |= hit && !behind;
          }
          if (found) *cleared = 1;
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_ready[st]);
        }
      }
    } else {
      // Raw tiles: K and V in turn, K one tile ahead (K0 K1 V0 K2 V1 .. V), so that
      // the next scores do not wait behind a V that waits for its stage.
      const int total = 2 * n_iter;
      auto is_v = [&](int e) { return e == total - 1 || (e > 0 && !(e & 1)); };
      auto tile_of = [&](int e) { return is_v(e) ? (e - 1) / 2 : (e + 1) / 2; };
      if (warp == 0) {
        // ------------------------------------------------ TMA of raw tiles
        load_q();
        // Lane = (part of the tile, block of 128 columns).
        const int part = lane % tile_pages, cb = lane / tile_pages;
        const uint32_t dst = smem_u32(smem + L::kR) + cb * L::kKT * 128 + part * page_rows * L::kRawRow;
        int v_page = page_coord(0, part), k_page = page_coord(1, part), issued = 0;
        int next = page_coord(2, part);
        for (int e = 0; e < total; ++e) {
          const int j = tile_of(e);
          const bool v = is_v(e);
          if (e >= R && !__all_sync(0xffffffffu, mbar_wait_sleep(&r_empty[e % R], ((e / R) - 1) & 1, err,
                                                           kDevTimeoutEmpty)))
            break;
          if (lane == 0) mbar_arrive_expect_tx(&r_full[e % R], L::kRawBytes);
          __syncwarp();
          if (cb < HD / L::kRawRow)
            pt_load_4d(dst + (e % R) * L::kRawBytes, v ? &tm_v : &tm_k, &r_full[e % R],
                       128 * cb, slot_coord(j, part), hk, v || e == 0 ? v_page : k_page);
          issued = e + 1;
          if (v) {
            v_page = k_page;
            k_page = next;
            next = page_coord(j + 3, part);
          }
        }
        // Our own copies land before the CTA may exit.
        mbar_wait(q_full, 0, nullptr, 0);
        for (int e = max(0, issued - R); e < issued; ++e)
          mbar_wait(&r_full[e % R], (e / R) & 1, nullptr, 0);
      } else if (warp >= 12) {
        // ------------------------------------------------- expansion to fp16
        // This lane's row of every tile (of 64 keys: two lanes, 128 columns each).
        const int r = ((warp - 12) * 32 + lane) % L::kKT, cb = ((warp - 12) * 32 + lane) / L::kKT;
        // Raw rows of 128 bytes: 16-byte chunk c at c ^ (r & 7); of 64 bytes: at
        // c ^ (r >> 1 & 3). fp16 rows: chunk c of a 64-column block at c ^ (r & 7).
        const uint32_t rx = HD >= 128 ? (r & 7) << 4 : ((r >> 1) & 3) << 4;
        const uint32_t dx = (r & 7) << 4;
        for (int e = 0; e < total; ++e) {
          const int j = tile_of(e), st = j % S, key0 = k_begin + j * L::kKT;
          const bool kv = is_v(e);
          if (!__all_sync(0xffffffffu,
                          mbar_wait_sleep(&r_full[e % R], (e / R) & 1, err, kDevTimeoutFull)) ||
              !stage_free(kv ? v_empty : k_empty, j))
            break;
          const uint8_t* src = smem + L::kR + (e % R) * L::kRawBytes + cb * L::kKT * 128 + r * L::kRawRow;
          uint8_t* dst = smem + (kv ? L::kV : L::kK) + st * L::kTileBytes + 2 * cb * L::kBlockBytes + r * 128;
          // Not every row sees all of it: NaN codes must not leak (int8 has none).
          const bool partly = CODE == kCodeE4M3 && kv && key0 + L::kKT > lim_first;
          const bool behind = partly && key0 + r >= seq.len;
          bool found = false;
#pragma unroll
          for (int c0 = 0; c0 < L::kRawRow / 16; c0 += 4) {
            uint4 x[4];
#pragma unroll
            for (int c = 0; c < 4; ++c)
              x[c] = *reinterpret_cast<const uint4*>(src + (((c0 + c) << 4) ^ rx));
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t w[8];
              pt_expand<CODE>(x[c].x, w[0], w[1]);
              pt_expand<CODE>(x[c].y, w[2], w[3]);
              pt_expand<CODE>(x[c].z, w[4], w[5]);
              pt_expand<CODE>(x[c].w, w[6], w[7]);
              if (partly) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const bool hit = h2_clear(w[i]);
                  found |= hit && !behind;
                  if (behind) w[i] = 0u;
                }
              }
              uint8_t* row = dst + (c0 >> 2) * L::kBlockBytes;
              *reinterpret_cast<uint4*>(row + (((2 * c) << 4) ^ dx)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(row + (((2 * c + 1) << 4) ^ dx)) =
                  make_uint4(w[4], w[5], w[6], w[7]);
            }
          }
          if (found) *cleared = 1;
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(kv ? &v_ready[st] : &k_full[st]);
            mbar_arrive(&r_empty[e % R]);
          }
        }
      } else {
        // ------------------------------------------------------ the scales
        // Lane = two consecutive keys of the part, one part ahead.
        float2 ks, vs;
        auto load_scales = [&](int u) {
          const int key = k_begin + u * L::kKeys + 2 * lane;
          const int page = u < n_iter * N && key < seq.len ? paged_page(p, b, key) : -1;
          const int64_t so = page >= 0 ? paged_scale_offset(p, page, hk, key) : 0;
          ks = vs = make_float2(0.f, 0.f);
          if (page >= 0) {
            ks = *reinterpret_cast<const float2*>(p.k_scale + so);
            vs = *reinterpret_cast<const float2*>(p.v_scale + so);
            if (key + 1 >= seq.len) ks.y = vs.y = 0.f;
          }
        };
        load_scales(0);
        for (int u = 0; u < n_iter * N; ++u) {
          const int slot = u % SC;
          const uint32_t par = ((u / SC) - 1) & 1;
          bool ok = true;
          if (u >= SC) {
            if (u - SC < nA * N) ok = mbar_wait_sleep(&c_empty[slot], par, err, kDevTimeoutEmpty);
            if (ok && u - SC < nB * N)
              ok = mbar_wait_sleep(&c_empty[SC + slot], par, err, kDevTimeoutEmpty);
          }
          if (!__all_sync(0xffffffffu, ok)) break;
          if (k_begin + (u + 1) * L::kKeys > lim_first) {
            // A scale that is none must not leak to rows that do not see it.
            const bool x = value_scale_bad(vs.x), y = value_scale_bad(vs.y);
            if (x) vs.x = 0.f;
            if (y) vs.y = 0.f;
            if (x || y) *cleared = 1;
          }
          float* dst = scales + slot * L::kSlotFloats;
          reinterpret_cast<float2*>(dst)[lane] = make_float2(ks.x * a.scale_log2, ks.y * a.scale_log2);
          reinterpret_cast<float2*>(dst + 64)[lane] = make_float2(value_scale_log2(vs.x), value_scale_log2(vs.y));
          reinterpret_cast<float2*>(dst + 128)[lane] =
              make_float2(value_scale_inverse(vs.x), value_scale_inverse(vs.y));
          load_scales(u + 1);
          __syncwarp();
          if (lane == 0) mbar_arrive(&c_full[slot]);
        }
      }
    }
  } else if (warp == 1 || warp == 2) {
    // ------------------------------------------------ MMA issuer of tile x
    const int x = warp == 1 ? 0 : 1;
    if (lane == 0 && x < L::kNT) {
      const int nx = x == 0 ? nA : nB;
      uint64_t* k_free = k_empty + x * S;
      uint64_t* v_free = v_empty + x * S;
      constexpr uint32_t id_qk = idesc_f16_f32(kPtTile, L::kKeys);
      constexpr uint32_t id_pv = idesc_f16_f32_bmn(kPtTile, HD);
      const uint64_t dq0 = sdesc_k_sw128(smem_u32(smem + L::kQ));
      const uint64_t dk0 = sdesc_k_sw128(smem_u32(smem + L::kK));
      const uint64_t dv0 = sdesc_mn_sw128(smem_u32(smem + L::kV), L::kBlockBytes);
      // Part u: rows (u % N) * kKeys .. of K and V of tile u / N, buffer u % SB of S.
      auto rows_of = [&](int u) {
        return static_cast<uint64_t>((u / N % S * L::kTileBytes + u % N * L::kKeys * 128) >> 4);
      };
      auto issue_qk = [&](int u) {
        const uint64_t da = dq0 + static_cast<uint64_t>(x * (L::kQBytes >> 4));
        const uint64_t db = dk0 + rows_of(u);
        const uint32_t d = tmem + x * kPtTile + u % SB * L::kKeys;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          mma_f16_ss(d, da + static_cast<uint64_t>(((k >> 2) * L::kQBlock + (k & 3) * 32) >> 4),
                     db + static_cast<uint64_t>(((k >> 2) * L::kBlockBytes + (k & 3) * 32) >> 4),
                     id_qk, k > 0 ? 1u : 0u);
        mma_commit(&s_full[x * SB + u % SB]);
        if (u % N == N - 1) mma_commit(&k_free[u / N % S]);
      };
      auto issue_pv = [&](int u) {
        const uint64_t db = dv0 + rows_of(u);
        const uint32_t p = tmem + L::kColP + x * L::kPStride + u % SB * L::kKeys;
#pragma unroll
        for (int k = 0; k < L::kKeys / 16; ++k)
          mma_f16_ts(tmem + L::kColO + x * HD, p + 8 * k, db + static_cast<uint64_t>((k * 2048) >> 4),
                     id_pv, (u > 0 || k > 0) ? 1u : 0u);
        mma_commit(&o_done[x * SB + u % SB]);
        if (u % N == N - 1) mma_commit(&v_free[u / N % S]);
      };
      auto wait_k = [&](int u) {  // for the first part of a tile
        const int j = u / N;
        return u % N != 0 || mbar_wait(&k_full[j % S], (j / S) & 1, err, kDevTimeoutFull);
      };
      // fp16: V as loaded, where every row sees all of the tile.
      auto wait_v = [&](int u) {
        const int j = u / N;
        if (u % N != 0) return true;
        if (!kQuant && j < j_partly)
          return mbar_wait(&v_full[j % S], (j / S) & 1, err, kDevTimeoutFull);
        const int uses = kQuant ? j / S : (j - j_partly) / S;  // of v_ready's stage before
        return mbar_wait(&v_ready[j % S], uses & 1, err, kDevTimeoutFull);
      };
      const int parts = nx * N;
      bool ok = mbar_wait(q_full, 0, err, kDevTimeoutFull);
      for (int u = 0; ok && u < min(SB, parts); ++u) {
        ok = wait_k(u);
        if (!ok) break;
        tc_fence_after();
        issue_qk(u);
      }
      for (int u = 0; ok && u < parts; ++u) {
        const int h = u % SB;
        const uint32_t ph = (u / SB) & 1;
        if constexpr (L::kSepP) {
          if (u + SB < parts) {  // the next S, as soon as this one is in registers
            ok = wait_k(u + SB) && mbar_wait(&s_free[x * SB + h], ph, err, kDevTimeoutOther);
            if (!ok) break;
            tc_fence_after();
            issue_qk(u + SB);
          }
        }
        ok = wait_v(u) && mbar_wait(&p_full[x * SB + h], ph, err, kDevTimeoutOther);
        if (!ok) break;
        tc_fence_after();
        issue_pv(u);
        if constexpr (!L::kSepP) {
          if (u + SB < parts) {
            // The next S overwrites this part's P: after the product that reads it.
            ok = wait_k(u + SB) && mbar_wait(&o_done[x * SB + h], ph, err, kDevTimeoutAccum);
            if (!ok) break;
            tc_fence_after();
            issue_qk(u + SB);
          }
        }
      }
      mma_commit(&drain[x]);
      mbar_wait(&drain[x], 0, nullptr, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int x = (warp - 4) >> 2;
    if (x < L::kNT) {
    const int quarter = warp & 3;  // this warp's TMEM lanes [32*quarter, +32)
    const int row = quarter * 32 + lane;
    const int first = i0 + x * tile_tokens;
    const int tok = first + row / group;
    const bool owned = row < tile_tokens * group && tok < seq.n;  // a row of the batch
    const int nx = x == 0 ? nA : nB;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lane_off + x * kPtTile;
    const uint32_t t_p = tmem + lane_off + L::kColP + x * L::kPStride;
    const uint32_t t_o = tmem + lane_off + L::kColO + x * HD;
    const int lim_row = lim_of(min(tok, seq.n - 1));
    const int lim_tile = lim_of(min(first, seq.n - 1));  // smallest of the tile
    float m_ref = -INFINITY;  // -inf: no key seen yet
    float l = 0.f;
    bool ok = true;
    auto wait_o = [&](int u) {  // the product of part u is through
      return mbar_wait(&o_done[x * SB + u % SB], (u / SB) & 1, err, kDevTimeoutAccum);
    };
    auto rescale_o = [&](float f) {  // this lane's row of O
#pragma unroll 1
      for (int c = 0; c < HD; c += 16) {
        uint32_t o[16];
        tmem_ld16(t_o + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tmem_st16(t_o + c, o);
      }
    };
    constexpr int KC = L::kKeys;
    // Which groups of 16 keys of a part exist (page in the pool): bit i.
    auto there_of = [&](int key0) {
      uint32_t there = 0;
#pragma unroll 1
      for (int i = 0; i < KC / 16; ++i)
        there |= static_cast<uint32_t>(key0 + 16 * i < seq.len &&
                                       paged_page(p, b, key0 + 16 * i) >= 0) << i;
      return there;
    };
    auto softmax = [&](auto with_holes) {
    uint64_t lsum0 = 0, lsum1 = 0;
    for (int u = 0; u < nx * N; ++u) {  // parts of the tiles
      const int h = u % SB;
      if (!__all_sync(0xffffffffu,
                      mbar_wait(&s_full[x * SB + h], (u / SB) & 1, err, kDevTimeoutAccum))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int key0 = k_begin + u * KC;
      uint32_t s[KC];
#pragma unroll
      for (int c = 0; c < KC / 32; ++c)
        tmem_ld32(t_s + h * KC + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
      tmem_ld_wait();
      if constexpr (L::kSepP) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[x * SB + h]);
      }
      if (key0 + KC > lim_tile) {  // warp-uniform
        const int c0 = lim_row - key0;
#pragma unroll
        for (int c = 0; c < KC; ++c)
          if (c >= c0) s[c] = 0xff800000u;  // -inf
      }
      if constexpr (decltype(with_holes)::value) {
        const uint32_t there = there_of(key0);
        if (there != (1u << (KC / 16)) - 1u) {
#pragma unroll
          for (int c = 0; c < KC; ++c)
            if (!((there >> (c >> 4)) & 1u)) s[c] = 0xff800000u;
        }
      }
      float mm[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        mm[i] = fmaxf(__uint_as_float(s[i]), __uint_as_float(s[i + 8]));
#pragma unroll
      for (int c = 16; c < KC; c += 16)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          mm[i] = fmax3(mm[i], __uint_as_float(s[c + i]), __uint_as_float(s[c + 8 + i]));
      const float m_new = fmaxf(fmax3(mm[0], mm[1], mm[2]),
                                fmax3(fmax3(mm[3], mm[4], mm[5]), mm[6], mm[7])) * a.scale_log2;
      bool rescale = false;
      float f = 1.f;
      if (u == 0) {
        m_ref = m_new;
      } else if (__any_sync(0xffffffffu, m_new > m_ref + kPtRescale)) {
        const float m_up = fmaxf(m_ref, m_new);
        f = m_ref == m_up ? 1.f : fast_exp2(m_ref - m_up);  // m_ref -inf: 0
        m_ref = m_up;
        const uint64_t f2v = f2_pack(f, f);
        lsum0 = f2_fma(lsum0, f2v, 0);
        lsum1 = f2_fma(lsum1, f2v, 0);
        rescale = true;
      }
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
      const uint64_t c2 = f2_pack(a.scale_log2, a.scale_log2);
      const uint64_t negm2 = f2_pack(-m_use, -m_use);
#pragma unroll
      for (int q = 0; q < KC / 64; ++q) {  // P goes to TMEM 64 keys at a time
        uint32_t pr[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int c = 64 * q + 2 * i;
          const uint64_t arg =
              f2_fma(f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), c2, negm2);
          uint64_t e;
          if ((i & 7) < kPtPoly) {
            uint64_t mant;
            e = exp2_poly_nan_f2(arg, &mant);
            lsum0 = f2_fma(mant, 0, lsum0);  // a NaN score makes the sum NaN
          } else {
            float a0, a1;
            f2_unpack(arg, a0, a1);
            e = f2_pack(fast_exp2(a0), fast_exp2(a1));
          }
          if (i & 1) lsum1 = f2_add(lsum1, e); else lsum0 = f2_add(lsum0, e);
          float e0, e1;
          f2_unpack(e, e0, e1);
          pr[i] = pack_half2(e0, e1);
        }
        if (q == 0) {
          // P's columns are free once the last product that read them is through
          // (P over S: it was before this S was computed); O may be rescaled once
          // the previous part's is.
          if (L::kSepP && u >= SB) ok = wait_o(u - SB);
          if (rescale && ok) ok = wait_o(u - 1);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (rescale) rescale_o(f);
        }
        tmem_st32(t_p + h * KC + 32 * q, pr);
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[x * SB + h]);
    }
    float la, lb, lc, ld;
    f2_unpack(lsum0, la, lb);
    f2_unpack(lsum1, lc, ld);
    l = (la + lb) + (lc + ld);
    };
    // 8 bit: every score and weight meets a scale from shared memory. A lane holds
    // 16 keys of 4 rows (lane / 4 + 8 k: the layout of matrix fragments) and so reads
    // the scales of 16 keys a part; with 64 keys of one row it read those of 64, and that
    // was what bounded the kernel (128 bytes a clock: 1024 of a part's 3100 clocks).
    auto softmax_quant = [&](auto with_holes) {
    static_assert(!kQuant || KC == 64, "one fragment load per 16 rows");
    const int quad = lane & 3, sub = lane >> 2;
    float mr[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    uint64_t ls[4] = {0, 0, 0, 0};
    auto of_row = [&](const float (&v)[4]) {  // from this layout to a lane per row
      float y = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float z = __shfl_sync(0xffffffffu, v[k], (lane & 7) * 4);
        if (lane >> 3 == k) y = z;
      }
      return y;
    };
    for (int u = 0; u < nx * N; ++u) {  // parts of the tiles
      const int h = u % SB, slot = u % SC;
      if (!__all_sync(0xffffffffu,
                      mbar_wait(&s_full[x * SB + h], (u / SB) & 1, err, kDevTimeoutAccum) &&
                          mbar_wait(&c_full[slot], (u / SC) & 1, err, kDevTimeoutOther))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int key0 = k_begin + u * KC;
      uint32_t s[2][32];  // [k / 2][4 c + 2 (k % 2)]: keys 8 c + 2 quad, + 1 of row k
      tmem_ld_16x64(t_s + h * KC, s[0]);
      tmem_ld_16x64(t_s + (16u << 16) + h * KC, s[1]);
      tmem_ld_wait();
      const float2* sk = reinterpret_cast<const float2*>(scales + slot * L::kSlotFloats) + quad;
      const float2* sv = reinterpret_cast<const float2*>(scales + slot * L::kSlotFloats + 128) + quad;
#pragma unroll
      for (int c = 0; c < 8; ++c) {  // scores in the log2 domain from here on
        const float2 f = sk[4 * c], g = sk[32 + 4 * c];
        const uint64_t f2 = f2_pack(f.x, f.y), e2 = f2_pack(g.x, g.y);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t* at = &s[k >> 1][4 * c + 2 * (k & 1)];
          float y0, y1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(at[0]), __uint_as_float(at[1])), f2, e2), y0, y1);
          at[0] = __float_as_uint(y0);
          at[1] = __float_as_uint(y1);
        }
      }
      if (key0 + KC > lim_tile) {  // warp-uniform
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = first + (quarter * 32 + sub + 8 * k) / group;
          const int c0 = lim_of(min(i, seq.n - 1)) - key0 - 2 * quad;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            if (8 * c >= c0) s[k >> 1][4 * c + 2 * (k & 1)] = 0xff800000u;  // -inf
            if (8 * c + 1 >= c0) s[k >> 1][4 * c + 2 * (k & 1) + 1] = 0xff800000u;
          }
        }
      }
      if constexpr (decltype(with_holes)::value) {
        const uint32_t there = there_of(key0);
        if (there != (1u << (KC / 16)) - 1u) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!((there >> (i >> 3)) & 1u)) s[0][i] = s[1][i] = 0xff800000u;
        }
      }
      float mn[4];
      bool more = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t* at = &s[k >> 1][2 * (k & 1)];
        float z = fmaxf(__uint_as_float(at[0]), __uint_as_float(at[1]));
#pragma unroll
        for (int c = 1; c < 8; ++c)
          z = fmax3(z, __uint_as_float(at[4 * c]), __uint_as_float(at[4 * c + 1]));
        mn[k] = z;
      }
#pragma unroll
      for (int m = 1; m <= 2; m *= 2)
#pragma unroll
        for (int k = 0; k < 4; ++k) mn[k] = fmaxf(mn[k], __shfl_xor_sync(0xffffffffu, mn[k], m));
#pragma unroll
      for (int k = 0; k < 4; ++k) more |= mn[k] > mr[k] + kPtRescale;
      bool rescale = false;
      float f = 1.f;  // of this lane's row of O
      if (u == 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) mr[k] = mn[k];
      } else if (__any_sync(0xffffffffu, more)) {
        float fk[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float up = fmaxf(mr[k], mn[k]);
          fk[k] = mr[k] == up ? 1.f : fast_exp2(mr[k] - up);  // mr -inf: 0
          mr[k] = up;
          ls[k] = f2_fma(ls[k], f2_pack(fk[k], fk[k]), 0);
        }
        f = of_row(fk);
        rescale = true;
      }
      uint64_t neg[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float z = mr[k] == -INFINITY ? 0.f : -mr[k];
        neg[k] = f2_pack(z, z);
      }
      uint32_t pr[2][16];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float2 w = sv[4 * c];  // one over the values' scales
        const uint64_t w2 = f2_pack(w.x, w.y);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t* at = &s[k >> 1][4 * c + 2 * (k & 1)];
          const uint64_t arg =
              f2_add(f2_pack(__uint_as_float(at[0]), __uint_as_float(at[1])), neg[k]);
          float a0, a1;
          f2_unpack(arg, a0, a1);
          const float e0 = fast_exp2(a0), e1 = fast_exp2(a1);
          ls[k] = f2_fma(f2_pack(e0, e1), w2, ls[k]);
          pr[k >> 1][2 * c + (k & 1)] = pack_half2(e0, e1);
        }
      }
      // (P lies over S: the product that read these columns was before this S.)
      if (rescale) {
        ok = wait_o(u - 1);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        rescale_o(f);
      }
      tmem_st_16x32(t_p + h * KC, pr[0]);
      tmem_st_16x32(t_p + (16u << 16) + h * KC, pr[1]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&p_full[x * SB + h]);
        mbar_arrive(&c_empty[x * SC + slot]);
      }
    }
    float lk[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float y0, y1;
      f2_unpack(ls[k], y0, y1);
      lk[k] = y0 + y1;
      lk[k] += __shfl_xor_sync(0xffffffffu, lk[k], 1);
      lk[k] += __shfl_xor_sync(0xffffffffu, lk[k], 2);
    }
    l = of_row(lk);
    m_ref = of_row(mr);
    };
    auto run = [&](auto with_holes) {
      if constexpr (kQuant) softmax_quant(with_holes); else softmax(with_holes);
    };
    if (holes) run(std::true_type{}); else run(std::false_type{});
    if (ok && nx > 0) ok = __all_sync(0xffffffffu, wait_o(nx * N - 1));
    if (m_ref == -INFINITY && l == l) l = 0.f;                  // no key seen
    if (m_ref == INFINITY) l = __uint_as_float(0x7fc00000u);  // a score of +inf
    if (ok) {
      const bool fix = *cleared != 0;  // the writer arrived before the last product
      const int head = hk * group + row % group;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t at = (static_cast<int64_t>(seq.row0 + tok) * (p.kv_heads * group) + head) *
                             a.splits + split;
      __half* dst = a.out + static_cast<int64_t>(seq.row0 + tok) * a.ld_out + head * HD;
      if (nx > 0) tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        if (nx > 0) {
          tmem_ld32(t_o + c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        float* of = reinterpret_cast<float*>(o);
        if (owned) {
          if (is_split) {
            float4* d4 = reinterpret_cast<float4*>(a.part_o + at * HD + c);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              d4[i] = make_float4(of[4 * i], of[4 * i + 1], of[4 * i + 2], of[4 * i + 3]);
            if (c == 0) a.part_ml[at] = make_float2(m_ref, l);
          } else {
            uint4* d4 = reinterpret_cast<uint4*>(dst + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float* g = of + 8 * i;
              d4[i] =
                  make_uint4(pack_half2(g[0] * inv, g[1] * inv), pack_half2(g[2] * inv, g[3] * inv),
                             pack_half2(g[4] * inv, g[5] * inv), pack_half2(g[6] * inv, g[7] * inv));
            }
          }
        }
        __syncwarp();  // the next tmem_ld is warp-collective
      }
      if (fix && owned)
        pt_add_cleared<CODE, HD>(p, b, hk, max(k_begin, lim_first - L::kKT), min(lim_row, k_stop),
                                 is_split ? a.part_o + at * HD : nullptr, dst);
    }
    }  // x < kNT
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, kPtCols);
  }
}

template <int CODE, int HD>
int launch_tc_hd(const tfx_paged_cache* c, const Paged& p, const PagedAttn& a, int64_t tokens,
                 cudaStream_t stream) {
  using L = PtCfg<CODE, HD>;
  static int done[kMaxDevices] = {0};
  auto kern = paged_tc_kernel<CODE, HD>;
  int st = ensure_smem(reinterpret_cast<const void*>(kern), L::kSmem, done);
  if (st != TFX_OK) return st;
  const int eb = code_bytes(CODE), page_rows = c->page_size < L::kKT ? c->page_size : L::kKT;
  const uint32_t tile_tokens = static_cast<uint32_t>(kPtTile / a.group);
  CUtensorMap tq, tk, tv;
  const uint64_t qd[3] = {HD, static_cast<uint64_t>(p.kv_heads) * a.group,
                          static_cast<uint64_t>(p.num_tokens)};
  const uint64_t qs[2] = {HD * 2, static_cast<uint64_t>(a.ld_q) * 2};
  const uint32_t qb[3] = {64, static_cast<uint32_t>(a.group), tile_tokens};
  st = make_tmap(&tq, a.q, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, qd, qs, qb,
                 CU_TENSOR_MAP_SWIZZLE_128B);
  // fp16: 64-column boxes in the layout of the products; 8 bit: whole rows.
  const uint64_t kd[4] = {HD, static_cast<uint64_t>(c->page_size),
                          static_cast<uint64_t>(p.kv_heads), static_cast<uint64_t>(p.num_pages)};
  const uint64_t ks[3] = {static_cast<uint64_t>(p.token_stride) * eb,
                          static_cast<uint64_t>(p.head_stride) * eb,
                          static_cast<uint64_t>(p.page_stride) * eb};
  const uint32_t kb[4] = {L::kQuant ? L::kRawRow : 64, static_cast<uint32_t>(page_rows), 1, 1};
  const CUtensorMapDataType dt =
      L::kQuant ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUtensorMapSwizzle sw =
      L::kQuant && HD == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  if (st == TFX_OK) st = make_tmap(&tk, p.k, dt, 4, kd, ks, kb, sw);
  if (st == TFX_OK) st = make_tmap(&tv, p.v, dt, 4, kd, ks, kb, sw);
  if (st != TFX_OK) return st;
  const int64_t blocks = (tokens + L::kNT * tile_tokens - 1) / (L::kNT * tile_tokens);
  launch_pdl(kern, dim3(p.kv_heads, p.batch, static_cast<unsigned>(blocks * a.splits_tc)),
             dim3(L::kThreads), L::kSmem, stream, tq, tk, tv, p, a, static_cast<int>(blocks),
             device_error_word());
  return check_launch("paged_tc_kernel");
}

}  // namespace

template <int CODE>
int launch_paged_tc(const tfx_paged_cache* c, const Paged& p, const PagedAttn& a, int64_t tokens,
                    cudaStream_t stream) {
  switch (c->head_dim) {
    case 64: return launch_tc_hd<CODE, 64>(c, p, a, tokens, stream);
    case 128: return launch_tc_hd<CODE, 128>(c, p, a, tokens, stream);
    default: return launch_tc_hd<CODE, 256>(c, p, a, tokens, stream);
  }
}

}  // namespace tfx
