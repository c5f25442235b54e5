// Parts of the causal prefill kernels that several translation units share
// (gfx950): the kernels' arguments, the search for a workgroup's tile of query
// columns, and the wave of the pipelined long tiles.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attn_device.hpp"

namespace loom_dev {

struct PrefillArgs {
  const uint16_t *__restrict__ q;
  const uint16_t *__restrict__ k;
  const uint16_t *__restrict__ v;
  const int32_t *__restrict__ qo;
  const int32_t *__restrict__ indptr;
  const int32_t *__restrict__ indices;
  const int32_t *__restrict__ last;
  uint16_t *__restrict__ out;
  float *__restrict__ lse;
  int32_t batch;
  int32_t nnz;
  int32_t hq;
  int32_t hkv;
  int32_t group;
  int64_t pool;
  int64_t n_indices;
  float scale_log2;
  int32_t indices_capacity;
  // Ragged (contiguous) K/V: `indptr` is kv_indptr over [nnz_kv, Hkv, 128]
  // rows; `indices` and `last` are unused.
  int32_t nnz_kv;
  // K/V row geometry (NHD: head_elems 128, row_elems Hkv * 128; HND pages:
  // head_elems 16 * 128, row_elems 128): token row t of kv-head h, t a
  // multiple of 16 for pages, starts at t * Hkv * 128 + h * head_elems.
  int32_t head_elems;
  int32_t row_elems;
  // Paged K/V: token rows per page (16, 32 or 64) and log2 of the 16-row
  // blocks per page; the kernel streams 16-row blocks, block j of page p
  // starting at token row p * page_rows + 16 * j.
  int32_t page_rows;
  int32_t blocks_lg;
  // Tiles per dispatch layer (one workgroup on each CU that the kv-heads of
  // one workgroup's XCD share: CUs / Hkv) for the serpentine tile order; 0:
  // plain heaviest-first order.
  int32_t tile_layer;
  // Nonzero (paged long tiles, at most 64 requests): tiles of all requests in
  // order of their distance from their request's end (rank k: the k-th
  // heaviest tile of every request), instead of request by request.
  int32_t tile_interleave;
  // FP8 E4M3 pages: device [k_scale, v_scale] (K = fp8 * k_scale, V = fp8 *
  // v_scale); null for BF16 pages.
  const float *kv_scales;
  // Split row tiles: workgroups per (tile, kv-head), each over an equal share
  // of the tile's blocks, and their column states: state c of tile rank m,
  // kv-head h and split s at ((s * row_tiles + m) * Hkv + h) * 16 + c, as
  // (max_log2, normalizer, 2 pad, acc[128]).
  int32_t splits;
  int32_t row_tiles;
  float *states;
};

// ---- locating a workgroup's tile ------------------------------------------------
// The tile of workgroup blockIdx.x and the request that owns it (wave-uniform).
struct TileLoc {
  int kvh;
  int rank;               // place among the grid's tiles
  int tile0;              // tile within the request's columns
  int32_t qs, qe;         // the request's qo_indptr pair
  int32_t ps, pe;         // its page (ragged: kv) indptr pair
  int32_t tl;             // its last page's rows (paged)
  int32_t fbeg;           // first flattened column it owns
  int32_t ipB;            // indptr[batch]
};

// Tile count given to a request whose qo range is malformed: larger than any
// tile index, so neither it nor any later request owns a tile (the reference's
// request search returns at the first malformed range, prefill.rs:303-313).
constexpr int64_t kNoTiles = (int64_t)1 << 50;

template <int W>
struct LocateSmem {
  int64_t wave_tot[W];
  int32_t wave_max[W];
  int32_t req;
  int32_t tile0;
  // the located request's qo_indptr pair, page (or kv) indptr pair, tail, and
  // the first flattened column it owns
  int32_t meta[6];
};

// Finds the tile of this workgroup (TC flattened columns per tile) and applies
// the global guards (prefill.rs:293-300 paged, :102-108 ragged); false: no
// tile, or a failed guard.
//
// Tiles come in reverse order: a request's later rows see longer causal
// ranges, so the heaviest tiles are dispatched first and the launch does not
// end with a few long tiles running alone (the grid's excess workgroups, which
// find no tile, come first and exit at once).  Workgroup b runs on XCD b % 8;
// with the kv-head fastest, each XCD keeps to a fixed set of kv-heads, whose
// K/V its L2 shares across tiles.
//
// The metadata comes in as few dependent round trips as possible: every
// request's qo range, page (kv) range and tail are loaded together and the
// guards applied afterwards.  Paged (prefill.rs:303-313): rows belong to the
// requests before the first malformed qo range.  Ragged (prefill.rs:111-137):
// row q belongs to the first request r with q < qo_indptr[r+1], i.e. r owns
// the rows from max(qo_indptr[r], max(qo_indptr[1..r])) to qo_indptr[r+1], and
// a request failing its guards keeps its rows' sentinels.
//
// Up to 64 requests every wave holds the whole table, one request per lane,
// and finds the tile by itself with register scans: no LDS and no barrier on
// the way (16 requests of 256 BF16 rows, GQA4 32/8: 35.0 -> 34.3 us; 1 x 1024
// 22.3 -> 21.5, 1 x 512 13.8 -> 12.9; a batch of two on row tiles 14.2 -> 13.5).
//
// EMPTY (paged): a request may have no rows (equal qo_indptr entries).  `block`: the
// workgroup's place, where it is not its number.
template <int W, bool RAGGED, int TC, bool INTERLEAVE, bool EMPTY = false>
__device__ __forceinline__ bool locate_tile(const PrefillArgs &a, LocateSmem<W> &sm, TileLoc &t,
                                            int split = 0, uint32_t block = blockIdx.x) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  t.kvh = (int)(block % a.hkv);
  const int64_t n_tiles = a.row_tiles, m = (int64_t)(block / a.hkv) - split * n_tiles;
  t.rank = (int)m;
  int64_t rank = m;
  if (a.tile_layer > 0) {
    // Serpentine: every other layer of tile_layer workgroups (one per CU of
    // the XCDs this kv-head runs on) takes its tiles in reverse, so a CU's
    // successive workgroups pair heavy tiles with light ones instead of
    // stacking the heaviest of every layer.
    const int64_t L = a.tile_layer, layer = m / L, c = m - layer * L;
    const int64_t width = min(L, n_tiles - layer * L);
    rank = layer * L + ((layer & 1) ? width - 1 - c : c);
  }
  const int64_t tile = n_tiles - 1 - rank;
  const bool interleave = INTERLEAVE && a.tile_interleave != 0;
  auto guards = [&](int32_t qo0, int32_t qoB, int32_t ip0, int32_t ipB) {
    t.ipB = ipB;
    if constexpr (RAGGED) return qo0 == 0 && qoB == a.nnz && ip0 == 0 && ipB == a.nnz_kv;
    return qo0 == 0 && qoB == a.nnz && ip0 == 0 && ipB >= 0 &&
           (a.indices_capacity ? (int64_t)ipB <= a.n_indices : (int64_t)ipB == a.n_indices);
  };
  // Tiles of a request that owns the rows [lo, s1) (ragged: lo past earlier
  // requests' rows); kNoTiles where the paged search ends.
  auto count = [&](int32_t s0, int32_t s1, int32_t p0, int32_t p1, int32_t lo) -> int64_t {
    if constexpr (RAGGED) {
      const bool ok = s0 >= 0 && s1 > s0 && s1 <= a.nnz && p0 >= 0 && p1 > p0 && p1 <= a.nnz_kv &&
                      s1 - s0 <= p1 - p0;
      return ok && s1 > lo ? ((int64_t)(s1 - lo) * a.group + TC - 1) / TC : 0;
    }
    return (s0 >= 0 && (EMPTY ? s1 >= s0 : s1 > s0) && s1 <= a.nnz) ? ((int64_t)(s1 - s0) * a.group + TC - 1) / TC
                                               : kNoTiles;
  };

  if (a.batch <= 64) {
    int32_t s0 = 0, s1 = 0, p0 = 0, p1 = 0, t1 = 0;
    const bool in = lane < a.batch;
    if (in) {
      s0 = a.qo[lane];
      s1 = a.qo[lane + 1];
      p0 = a.indptr[lane];
      p1 = a.indptr[lane + 1];
      if constexpr (!RAGGED) t1 = a.last[lane];
    }
    int32_t lo = s0;
    if constexpr (RAGGED) {
      const int32_t ends = wave_incl_max_i32(in ? s1 : 0);  // running max of the qo ends
      lo = max(s0, __builtin_amdgcn_update_dpp(0, ends, 0x138, 0xf, 0xf, false));  // (of lane - 1)
    }
    const int64_t cnt64 = in ? count(s0, s1, p0, p1, lo) : 0;
    // (saturated: a count or a prefix past UINT32_MAX lies past every tile)
    const uint32_t cnt = (uint32_t)min<int64_t>(cnt64, (int64_t)UINT32_MAX);
    bool mine;
    if (interleave) {
      // Tile `rank` of all requests' tiles in order of their distance from
      // their request's end (after the grid's excess workgroups): the j-th of
      // the tiles k from their request's end, where k is the largest with
      // F(k) = sum of min(k, count) <= it and j counts requests with more
      // than k tiles in request order; requests from the first malformed qo
      // range on own no tile.  Each lane evaluates F at one k, so a round
      // narrows the range of k 64-fold.
      const uint64_t badm = __builtin_amdgcn_ballot_w64(in && cnt64 == kNoTiles);
      const int first_bad = badm ? __builtin_ctzll(badm) : 64;
      const uint32_t c = (in && lane < first_bad) ? cnt : 0u;
      auto F = [&](uint32_t k) {
        uint32_t f = 0;
        for (int r = 0; r < a.batch; ++r)
          f = __builtin_elementwise_add_sat(
              f, (uint32_t)min(k, (uint32_t)__builtin_amdgcn_readlane((int)c, r)));
        return f;
      };
      // F at one wave-uniform k
      auto F1 = [&](uint32_t k) {
        return (uint32_t)__builtin_amdgcn_readlane((int)wave_incl_add_sat_u32(min(k, c)), 63);
      };
      const int64_t rr = rank - (n_tiles - (int64_t)F1(UINT32_MAX));
      if (rr < 0) return false;
      uint32_t base = 0, span = (uint32_t)n_tiles;  // k in [base, base + span)
      while (span > 1) {
        const uint32_t st = (span + 63) >> 6;
        const uint64_t below = __builtin_amdgcn_ballot_w64(lane * st < span &&
                                                           (int64_t)F(base + lane * st) <= rr);
        const uint32_t n = (uint32_t)__builtin_popcountll(below) - 1u;  // F(base) <= rr always
        base += n * st;
        span = min(st, span - n * st);
      }
      const int j = (int)(rr - (int64_t)F1(base));
      const uint64_t more = __builtin_amdgcn_ballot_w64(c > base);
      const int before = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(more >> 32),
                                                        __builtin_amdgcn_mbcnt_lo((uint32_t)more, 0u));
      mine = c > base && before == j;
      t.tile0 = (int)(c - 1u - base);
    } else {
      const uint32_t incl = wave_incl_add_sat_u32(cnt);
      const uint32_t excl = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)incl, 0x138, 0xf, 0xf, false);
      mine = in && cnt64 != kNoTiles && tile < (int64_t)incl && tile >= (int64_t)excl;
      t.tile0 = (int)(tile - (int64_t)excl);
    }
    const uint64_t who = __builtin_amdgcn_ballot_w64(mine);
    const int B1 = a.batch - 1;
    if (!guards(__builtin_amdgcn_readlane(s0, 0), __builtin_amdgcn_readlane(s1, B1),
                __builtin_amdgcn_readlane(p0, 0), __builtin_amdgcn_readlane(p1, B1)))
      return false;
    if (!who) return false;
    const int w = __builtin_ctzll(who);
    t.tile0 = __builtin_amdgcn_readlane(t.tile0, w);
    t.qs = __builtin_amdgcn_readlane(s0, w);
    t.qe = __builtin_amdgcn_readlane(s1, w);
    t.ps = __builtin_amdgcn_readlane(p0, w);
    t.pe = __builtin_amdgcn_readlane(p1, w);
    t.tl = __builtin_amdgcn_readlane(t1, w);
    t.fbeg = RAGGED ? (__builtin_amdgcn_readlane(lo, w) - t.qs) * a.group : 0;
    return true;
  }

  // Larger batches: a workgroup-wide prefix of the requests' tile counts.
  const int32_t qo0 = a.qo[0], qoB = a.qo[a.batch];
  const int32_t ip0 = a.indptr[0], ipB = a.indptr[a.batch];
  if (tid == 0) sm.req = -1;
  int64_t carry = 0;
  int32_t carry_max = 0;
  for (int base = 0; base < a.batch; base += W * 64) {
    const int r = base + tid;
    int32_t s0 = 0, s1 = 0, p0 = 0, p1 = 0, t1 = 0;
    if (r < a.batch) {
      s0 = a.qo[r];
      s1 = a.qo[r + 1];
      p0 = a.indptr[r];
      p1 = a.indptr[r + 1];
      if constexpr (!RAGGED) t1 = a.last[r];
    }
    int32_t lo = s0;
    if constexpr (RAGGED) {
      // exclusive running max of the qo ends before r
      int32_t x = r < a.batch ? s1 : INT32_MIN;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int32_t y = __shfl_up(x, o, 64);
        if (lane >= o) x = max(x, y);
      }
      if (lane == 63) sm.wave_max[wave] = x;
      __syncthreads();
      int32_t before = carry_max, blk = carry_max;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        before = i < wave ? max(before, sm.wave_max[i]) : before;
        blk = max(blk, sm.wave_max[i]);
      }
      const int32_t up = __shfl_up(x, 1, 64);
      lo = max(s0, lane > 0 ? max(before, up) : before);
      carry_max = blk;
    }
    const int64_t cnt = r < a.batch ? count(s0, s1, p0, p1, lo) : 0;
    const int64_t x = wave_incl_scan64(cnt, lane);
    if (lane == 63) sm.wave_tot[wave] = x;
    __syncthreads();
    int64_t before = 0, tot = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int64_t y = sm.wave_tot[i];
      before += (i < wave) ? y : 0;
      tot += y;
    }
    const int64_t incl = carry + before + x;
    if (r < a.batch && tile < incl && tile >= incl - cnt && cnt != kNoTiles) {
      sm.req = r;
      sm.tile0 = (int32_t)(tile - (incl - cnt));
      sm.meta[0] = s0;
      sm.meta[1] = s1;
      sm.meta[2] = p0;
      sm.meta[3] = p1;
      sm.meta[4] = t1;
      sm.meta[5] = RAGGED ? (lo - s0) * a.group : 0;
    }
    carry += tot;
    __syncthreads();
    if (carry > tile) break;
  }
  if (!guards(qo0, qoB, ip0, ipB)) return false;
  if (uni(sm.req) < 0) return false;
  t.tile0 = uni(sm.tile0);
  t.qs = uni(sm.meta[0]);
  t.qe = uni(sm.meta[1]);
  t.ps = uni(sm.meta[2]);
  t.pe = uni(sm.meta[3]);
  t.tl = uni(sm.meta[4]);
  t.fbeg = uni(sm.meta[5]);
  return true;
}

// ---- pipelined long tiles (LOOM_PAGED_PREFILL_LONG_TILE, 64 or 128 columns) -----
// A workgroup owns 32 * NW flattened columns, two 16-column tiles per wave,
// and walks the whole causal range in 32-token blocks (two 16-row blocks),
// which are loaded straight into an LDS ring (buffer loads to LDS: no VGPRs or
// LDS stores).  G groups of NW waves own the same columns and split the blocks
// (block b to group b % G); their states merge at the end.
//
// Bound and shape.  A 16x16x32 MFMA takes 16 cycles of the SIMD's matrix core
// and holds its vector issue for 8 of them, an exponential for 8, other vector
// instructions 4 (measured with register-only loops), and a wave issues in
// order.  Per wave and block: 32 MFMAs (512 cycles) among 101 vector
// instructions, 16 of them exponentials, which fit beside the MFMAs only if
// they are issued between them (a block takes 1061 cycles of its SIMD at 8192
// rows, so the matrix cores are busy 48%; the clock falls to 1.86 GHz).  Hence: the products of one block, the softmax of the
// next and the scores of the one after interleaved by hand (pin()); no maximum
// per block; normalizer sums by dot products with ones; page addresses
// computed per 64 blocks, one per lane; whole rows per load instruction.  Two
// waves per SIMD (241-244 registers; FP8 pages 215-217).  Tried with 32x32x16
// MFMAs: a tenth faster on cool data (zeros), but their energy per flop is
// higher and random data holds the card at its power limit from about 4096 rows
// on, where they lost 3%.
// Measured against the plain long tiles: see long_form.
//
// acc[t][e][i] = O[column of tile t][dim 16 e + 4 quad + i].
//
// A column's reference lies kHeadroomLog2 above the largest score it was taken
// from and moves when a lane's normalizer passes 1 (see step()), so a weight
// never exceeds 1 and |O| stays below four times the largest |V|.  Along with it
// move the columns past kNearRefresh, which would follow within a few blocks; a
// column that has just moved is below it (9 * 2^-12).  Scores of unit variance
// pass 1 only after some 80000 tokens (with 8 for 12, after 5000: 1% of an 8192
// row prompt), and V's smallest normal values keep 11 bits of their products.
constexpr float kHeadroomLog2 = 12.0f, kNearRefresh = 0.0625f;

// HL: P enters the product as a BF16 high part and a BF16 residual (two MFMAs
// per block of V), so the weights carry 16 significant bits and the
// normalizer sums them in FP32.  Otherwise P is rounded once to BF16 and the
// normalizer sums the rounded weights, or (XS) the weights before their rounding.  The
// former keeps a weight that stands alone out of O's error, the latter all roundings out of
// LSE's.
template <int NW, bool FP8, bool HL, int G, bool XS = false>
struct PipeWave {
  const PrefillArgs &a;
  int lane, col, quad;
  int64_t end_col[2];  // causal end (exclusive) of the lane's column of each tile, 0 if unused
  int64_t full_end;    // smallest causal end of the wave's valid columns
  float nmax[2];       // negated reference (log2 domain, scaled); +inf: none yet
  float lsum[2];       // normalizer over the lane's quarter of the tokens
  f32x4 acc[2][8];
  u32x4 qf[2][4];      // B fragments of the query tiles
  const uint8_t *ring;
  int kofs[4], vofs[4];  // the lane's fragments within a ring slot

  // Ring slot: 32 rows of K, then 32 of V, in 1 KB groups of whole rows (4;
  // FP8 8), so that one load instruction covers whole rows (21 cycles of the
  // CU's load path; 64 where it reads 64 bytes of each of 16).  Within a group
  // the 16-byte units of row r are permuted (BF16: unit u at u ^ 4 (r & 3);
  // FP8: u ^ 2 ((r >> 1) & 3)) and the groups are padded, which spreads the
  // fragment reads below over the banks (conflicts are 12% of the CU's cycles at
  // 8192 rows).
  static constexpr int kRowBytes = FP8 ? 128 : 256;
  static constexpr int kUnits = kRowBytes / 16;
  static constexpr int kGroupRows = 1024 / kRowBytes;
  static constexpr int kGroups = 32 / kGroupRows;  // of each of K and V
  static constexpr int kKGroup = 1040;             // group stride of K
  static constexpr int kVGroup = 1056;             // group stride of V (BF16)
  static constexpr int kKBytes = kGroups * kKGroup;
  static constexpr int kSlotBytes = kKBytes + (FP8 ? kGroups * 1024 + 32 : kGroups * kVGroup);
  // Byte offset of V's group g from the slot's start (FP8: 16 bytes of padding per 16 rows).
  static constexpr int v_group(int g) { return kKBytes + (FP8 ? g * 1024 + (g >> 1) * 16 : g * kVGroup); }
  // Two workgroups of four waves per CU, or one of eight: four slots where
  // one group shares the ring, two for each of several groups.
  static constexpr int kSlots = NW;
  // 1 KB loads per wave and block: waves 0 .. NW / 2 - 1 load K, the others V.
  static constexpr int kLoads = 2 * kGroups / NW;

  static __device__ __forceinline__ int swizzle(int r) { return FP8 ? (r & 6) : 4 * (r & 3); }

  __device__ __forceinline__ void reset(const uint8_t *group_ring) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      nmax[t] = INFINITY;
      lsum[t] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[t][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    ring = group_ring;
    // K: row col of a 16-row block.  BF16: 8 dims 32c + 8 quad .. (unit 4c +
    // quad).  FP8: 16 dims 64j + 16 quad .. (unit 4j + quad), which the query
    // fragments 2j and 2j + 1 hold in the same order.
    const int kr = (col / kGroupRows) * kKGroup + (col % kGroupRows) * kRowBytes;
#pragma unroll
    for (int c = 0; c < 4; ++c) kofs[c] = kr + ((4 * (FP8 ? c & 1 : c) + quad) ^ swizzle(col)) * 16;
    // Vᵀ, dims 16 e .. 16 e + 15, tokens 4 quad + [0, 4) of both 16-row blocks
    // in the order of the Pᵀ fragment, e = 2x + y (y: an immediate offset).
    // BF16 (ds_read_b64_tr_b16, one read per 16-row block: within 16 lanes,
    // lane i receives element i % 4 of the 8 bytes lane 4k + i / 4 addresses, k
    // = 0..3): lane i addresses dims 16 e + 4 (i % 4) .. of token row 4 quad +
    // i / 4.  FP8 (ds_read_b64_tr_b8, one read: lane i receives byte i % 8 of
    // the 8 bytes lane 2k + i / 8 addresses, k = 0..7): lane i addresses dims
    // 16 e + 8 (i & 1) .. of token row 4 quad + (i >> 1) % 4 of block i >> 3.
    const int i = col;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if constexpr (FP8) {
        const int r = 4 * quad + ((i >> 1) & 3), g = 2 * (i >> 3) + (r >> 3);
        vofs[x] = v_group(g) + (r & 7) * 128 + (2 * x ^ swizzle(r)) * 16 + 8 * (i & 1);
      } else {
        vofs[x] = v_group(quad) + (i >> 2) * 256 + ((4 * x ^ swizzle(i >> 2)) + ((i & 3) >> 1)) * 16 +
                  8 * (i & 1);
      }
    }
  }

  // Query fragment c: B fragment of S (lane: column, k = 8 quad + [0, 8)).
  static __device__ __forceinline__ int q_dim(int c, int quad) {
    return FP8 ? 64 * (c >> 1) + 16 * quad + 8 * (c & 1) : 32 * c + 8 * quad;
  }

  // K fragments of a block (A fragments of S: token row, k as above), by
  // chunk and 16-row block.
  struct KFrags {
    u32x4 f[FP8 ? 2 : 4][2];
  };
  __device__ __forceinline__ KFrags read_k(int slot) const {
    KFrags k;
#pragma unroll
    for (int c = 0; c < (FP8 ? 2 : 4); ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        k.f[c][h] = *reinterpret_cast<const u32x4 *>(ring + kofs[c] + slot + h * (kGroups / 2) * kKGroup);
    return k;
  }
  // Scores of a block: s[t][h][i] = S[token 16 h + 4 quad + i][column of tile t].
  struct Scores {
    f32x4 s[2][2];
    __device__ __forceinline__ float get(int x) const { return s[x >> 3][(x >> 2) & 1][x & 3]; }
  };
  // S = K·Qᵀ, product x of 8: chunk x >> 1, 16-row block x & 1, both tiles.
  __device__ __forceinline__ void score(const KFrags &k, Scores &sc, int x) const {
    const int c = x >> 1, h = x & 1;
    const u32x4 w = FP8 ? fp8x8_to_bf16x8(u32x2{k.f[c >> 1][h][2 * (c & 1)], k.f[c >> 1][h][2 * (c & 1) + 1]})
                        : k.f[FP8 ? 0 : c][h];
    const f32x4 z = {};
#pragma unroll
    for (int t = 0; t < 2; ++t)
      sc.s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(w), as_bf16x8(qf[t][c]),
                                                           c ? sc.s[t][h] : z, 0, 0, 0);
  }

  // Vᵀ fragments of a block, by 16-dim block.
  struct VFrags {
    u32x4 f[8];
  };
  __device__ __forceinline__ u32x4 read_v(int slot, int e) const {
    const uint8_t *p = ring + vofs[e >> 1] + slot + (e & 1) * (FP8 ? 16 : 32);
    if constexpr (FP8) {
      const u32x2 b = lds_read_tr8(p);
      return u32x4{b[0], b[1], 0, 0};
    } else {
      const u32x2 lo = lds_read_tr16(p), hi = lds_read_tr16(p + (v_group(4) - v_group(0)));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  }

  // Weights as B fragments of the product (lane: column, k = 8 quad + j is
  // token 16 (j >> 2) + 4 quad + (j & 3)), and their residuals.
  struct Weights {
    u32x4 hi[2], lo[2];
  };
  // O += P·V, dims 16 e .. of both tiles.
  __device__ __forceinline__ void product(const VFrags &v, const Weights &p, int e) {
    const bf16x8 w = as_bf16x8(FP8 ? fp8x8_to_bf16x8(u32x2{v.f[e][0], v.f[e][1]}) : v.f[e]);
#pragma unroll
    for (int t = 0; t < 2; ++t)
      acc[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, as_bf16x8(p.hi[t]), acc[t][e], 0, 0, 0);
    if constexpr (HL)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        acc[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, as_bf16x8(p.lo[t]), acc[t][e], 0, 0, 0);
  }

  // Weights 2y, 2y + 1 of the lane's 16 (already exponentiated; 8 per tile)
  // into the fragments, and into the normalizer l of the tile.
  static __device__ __forceinline__ void put(Weights &p, float &l, float x0, float x1, int y) {
    if constexpr (HL) {
      const uint32_t b0 = __float_as_uint(x0), b1 = __float_as_uint(x1);
      p.hi[y >> 2][y & 3] = pack_hi16(b0, b1);
      p.lo[y >> 2][y & 3] = pack_hi16(__float_as_uint(x0 - __uint_as_float(b0 & 0xffff0000u)),
                                      __float_as_uint(x1 - __uint_as_float(b1 & 0xffff0000u)));
      l += x0;
      l += x1;
    } else {
      const uint32_t w = bf16x2_pack(x0, x1);
      p.hi[y >> 2][y & 3] = w;
      if constexpr (XS) {
        l += x0 + x1;
        return;
      }
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w),
                                          __builtin_bit_cast(bf16x2, 0x3F803F80u), l, false);
    }
  }

  // Holds the values' computation at this place of the instruction stream.
  static __device__ __forceinline__ void pin(f32x4 &m, f32x4 &n, float &x, float &y, float &z) {
    asm volatile("" : "+v"(m), "+v"(n), "+v"(x), "+v"(y), "+v"(z));
    __builtin_amdgcn_sched_barrier(0);
  }

  // Masks the scores of tokens at or past a column's causal end (lt0: the
  // block's first token).
  __device__ __forceinline__ void mask(Scores &cur, int64_t lt0) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int vis = (int)max<int64_t>(-1, min<int64_t>(32, end_col[t] - lt0));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cur.s[t][0][i] = (quad * 4 + i < vis) ? cur.s[t][0][i] : -INFINITY;
        cur.s[t][1][i] = (16 + quad * 4 + i < vis) ? cur.s[t][1][i] : -INFINITY;
      }
    }
  }

  // One step of the software pipeline, block j of the wave's group:
  //   products of block j - 1 (v, w)    |  scaling and half the exponentials
  //   scores of block j + 1             |  the rest of block j's softmax, and
  //                                     |  the reads of block j's V
  // `cur`: block j's scores; on return `nxt` holds block j + 1's, v and w
  // block j's.  kslot, vslot: ring offsets of K (j + 1) and V (j).  (After
  // the last block the scores of whatever K's slot holds are not used.)
  __device__ __forceinline__ void step(int kslot, int vslot, Scores &cur, Scores &nxt, VFrags &v,
                                       Weights &w) {
    const KFrags k = read_k(kslot);
    float p[16];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      product(v, w, x);
      p[2 * x] = fmaf(cur.get(2 * x), a.scale_log2, nmax[x >> 2]);
      p[2 * x + 1] = fmaf(cur.get(2 * x + 1), a.scale_log2, nmax[x >> 2]);
      if (x > 0) p[x - 1] = fast_exp2(p[x - 1]);
      pin(acc[0][x], acc[1][x], p[2 * x], p[2 * x + 1], p[x > 0 ? x - 1 : 0]);
    }
    Weights wn;
    float l[2] = {lsum[0], lsum[1]};
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      score(k, nxt, x);
      if (x < 5) {
        p[2 * x + 7] = fast_exp2(p[2 * x + 7]);
        if (x < 4) p[2 * x + 8] = fast_exp2(p[2 * x + 8]);
      }
      if (x < 7) put(wn, l[x >> 2], p[2 * x], p[2 * x + 1], x);
      if (x == 6) put(wn, l[1], p[14], p[15], 7);
      v.f[x] = read_v(vslot, x);
      pin(nxt.s[0][x & 1], nxt.s[1][x & 1], l[x >> 2], p[x < 5 ? 2 * x + 7 : 15],
          p[x < 4 ? 2 * x + 8 : 15]);
    }
    // The reference of a column moves only when its normalizer passes 1 or is
    // not a number (no reference yet): BF16 and FP32 weights keep their relative
    // precision at any magnitude, so a reference above the running max costs
    // none, and the common step needs no max at all.  LSE = reference +
    // log2(normalizer).
    if (__builtin_amdgcn_ballot_w64(!(l[0] <= 1.0f && l[1] <= 1.0f))) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float mx = fmaxf(cur.get(8 * t), cur.get(8 * t + 1));
#pragma unroll
        for (int i = 2; i < 8; ++i) mx = fmaxf(mx, cur.get(8 * t + i));
        mx = quad_max(mx) * a.scale_log2;
        const float m_old = -nmax[t];
        const bool move = !(quad_max_nan(l[t]) <= kNearRefresh);
        const float m_new = move ? fmaxf(m_old, mx) + kHeadroomLog2 : m_old;
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;  // nothing visible yet
        // (a column with nothing visible before has O = 0: nothing to rescale)
        const float al = fast_exp2(m_old - m_use);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[t][e] *= al;
        nmax[t] = -m_new;
        l[t] = lsum[t] * al;
#pragma unroll
        for (int y = 4 * t; y < 4 * t + 4; ++y)
          put(wn, l[t], fast_exp2(fmaf(cur.get(2 * y), a.scale_log2, -m_use)),
              fast_exp2(fmaf(cur.get(2 * y + 1), a.scale_log2, -m_use)), y);
      }
    }
    lsum[0] = l[0];
    lsum[1] = l[1];
    w = wn;
  }

  // The whole causal walk of the wave's group over 16-row blocks 0..n16-1 (the
  // second half of the last 32-token block is empty when n16 is odd: no rows).
  // load(b, slot): the wave's share of block b to the slot at LDS address
  // `slot` (blocks past the end: no rows, zeros).  `loads_k`: the wave loads K
  // rows, else V rows; K runs one block ahead of V, so that one barrier per
  // step publishes K (j + 1) and V (j), the loads of the next kSlots - 1 steps
  // are in flight, and a slot is refilled one step after it was read.
  // first(): called once the first loads are out.
  template <class Load, class First>
  __device__ __forceinline__ void stream(int n16, Load load, First first, uint32_t lds, bool loads_k, int grp,
                                         int64_t own_end) {
    const int nb = (n16 + 1) >> 1;
    const int steps = (nb + G - 1) / G;
    // this group's blocks that the wave computes, and the blocks (of all
    // groups) that need no mask
    const int nbw = uni(max(0, ((int)min<int64_t>((own_end + 31) >> 5, nb) - grp + G - 1) / G));
    const int nfull = uni((int)min<int64_t>(full_end >> 5, nb));
    // (K) block j + kSlots goes to the slot of block j, (V) one less
    const int ahead = uni(kSlots - (loads_k ? 0 : 1));
    auto slot_of = [](int j) { return (j & (kSlots - 1)) * kSlotBytes; };
    if (loads_k) load(grp, lds);
#pragma unroll
    for (int j = 1 - kSlots; j < 0; ++j)
      load(G * (j + ahead) + grp, lds + slot_of(j + ahead));
    first();
    publish<(kSlots - 1) * kLoads>();
    // (s: j, or its slot)
    auto advance = [&](int j, int s) {
      publish<(kSlots - 2) * kLoads>();
      load(G * (j + ahead) + grp, lds + slot_of(s + ahead));
    };
    Scores sa, sb;
    VFrags v = {};
    Weights w = {};
    if (nbw > 0) {
      const KFrags k = read_k(0);
#pragma unroll
      for (int c = 0; c < 8; ++c) score(k, sa, c);
    }
    int j = 0;
    while (j < nbw) {
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        if (s > 0 && j >= nbw) break;
        advance(j, s);
        Scores &cur = s & 1 ? sb : sa, &nxt = s & 1 ? sa : sb;
        if (G * j + grp >= nfull) mask(cur, 32 * (int64_t)(G * j + grp));
        step(slot_of(s + 1), slot_of(s), cur, nxt, v, w);
        ++j;
      }
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) product(v, w, x);
    for (; j < steps; ++j) advance(j, j);
    wait_vmcnt<0>();
  }

  // Waits until at most N of this wave's loads are outstanding (and for its
  // LDS reads, so that a slot read before the barrier may be refilled after
  // it), then meets the workgroup's other waves.
  template <int N>
  static __device__ __forceinline__ void publish() {
    static_assert(N < 64, "vmcnt field");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(((N >> 4) << 14) | (0x0 << 8) | (0x7 << 4) | (N & 15));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

}  // namespace loom_dev
