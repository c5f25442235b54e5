// Attention with a sliding window and sinks over paged K/V for gfx950 (MI355X), D128,
// BF16, FP8 E4M3 or MXFP4 pages of 16-64 rows, NHD or HND (no reference counterpart):
// one new token per request (decode) or ragged rows of new tokens (a chunk).
//
// A row at position p of its request sees token t <= p where t > p - window or t < sinks;
//   O = sum_t softmax(scale q.k_t)_t v_t,   LSE = log2 sum_t 2^(scale log2(e) q.k_t).
// The query rows of a request and the heads of one kv-head's group are flattened, (row, group
// head) -> row * group + head, and cut into tiles of columns, as for paged prefill.  A tile
// walks the 16-row blocks that some column of it sees: the sinks' blocks, then those from
// the first row's window start to the last row's own token.  Blocks in between are never
// touched, nor are their page indices.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "attn_device.hpp"
#include "loom_internal.hpp"
#include "prefill_device.hpp"

using loom::fail;
using namespace loom_dev;

namespace {

enum Kv : int { kBf16, kFp8, kMx4 };
template <Kv KV>
constexpr int kRowBytes = KV == kBf16 ? 256 : KV == kFp8 ? 128 : 64;  // of one head's K or V

struct WindowArgs : PrefillArgs {
  const uint8_t *k_mx;  // MXFP4 scales
  const uint8_t *v_mx;
  int32_t window;       // INT32_MAX: none
  int32_t sinks;
  int32_t head_bytes;   // from one kv-head's rows of a page to the next
  int32_t row_bytes;    // from one token's row to the next
  int32_t head_tiles;   // one-row form: tiles per request
  uint32_t group_inv;   // 2^32 / group, rounded up, where that divides every column; 0: it does not
  uint32_t *arrived;    // splits: arrival words, loom::kMx4JoinBytes apart
  int32_t sorted;       // tiles of the longest walks first (up to 64 requests)
  // Row tiles over MXFP4 pages with an even number of kv-heads: the workgroups of the command,
  // and its blocks are dealt so that two neighbouring heads, whose rows or scales share
  // cache lines, run on one XCD; 0: in order.
  int32_t pair_heads;
};

// Row of column f: f / group.  (A division takes about 35 instructions, and a tile has
// nine of them.)
__device__ __forceinline__ int row_of(const WindowArgs &a, int f) {
  if (a.group == 1) return f;
  return a.group_inv ? (int)__umulhi((uint32_t)f, a.group_inv) : (int)((uint32_t)f / (uint32_t)a.group);
}

// A tile's place and what its columns see (wave-uniform).
struct Tile {
  TileLoc loc;
  int kv_len;
  int group_rows;     // the request's query rows
  int fcols, col0;    // its columns, and the tile's first
  int p_lo, p_hi;     // positions of the tile's first and last row
  int sink_blocks, first_block, blocks;  // the walk, in 16-row blocks
  // 16-row block of the request at place x of the walk
  __device__ __forceinline__ int block(int x) const {
    return x < sink_blocks ? x : x - sink_blocks + first_block;
  }
  // tokens of it that some column may see, from its first row on
  __device__ __forceinline__ int rows(const WindowArgs &a, int x) const {
    const int b = block(x);
    return min(16, (x < sink_blocks ? min(a.sinks, p_hi + 1) : p_hi + 1) - 16 * b);
  }
};

// The tile of this workgroup among those of up to 64 requests: every wave holds the table, a
// request per lane.  Rows belong to the requests before the first falling qo_indptr range.
// A request's last rows come first, and (`sorted`) the request of the longest walks: the
// launch does not end with a few long walks alone (four chunks of 512 rows behind
// 2048-16384 tokens, the longest listed first and so dispatched last: 481 us without the
// order, 440 with it).  A grid of a workgroup per CU needs no order.
template <int TC>
__device__ __forceinline__ bool locate_lanes(const WindowArgs &a, TileLoc &l, int split,
                                                     uint32_t block) {
  const int lane = threadIdx.x & 63;
  const bool in = lane < a.batch;
  int32_t s0 = 0, s1 = 0, p0 = 0, p1 = 0, t1 = 0;
  if (in) {
    s0 = a.qo[lane];
    s1 = a.qo[lane + 1];
    p0 = a.indptr[lane];
    p1 = a.indptr[lane + 1];
    t1 = a.last[lane];
  }
  l.kvh = (int)(block % (uint32_t)a.hkv);
  l.rank = (int)(block / (uint32_t)a.hkv) - split * a.row_tiles;
  const uint64_t falls = __builtin_amdgcn_ballot_w64(in && !(s0 >= 0 && s1 >= s0 && s1 <= a.nnz));
  const int valid = falls ? __builtin_ctzll(falls) : a.batch;
  // (columns fit 31 bits: the plan checks it)
  const uint32_t cnt = lane < valid ? ((uint32_t)(s1 - s0) * (uint32_t)a.group + TC - 1) / TC : 0u;
  int place = lane;
  uint32_t ordered = cnt;
  if (a.sorted) {
    // place among the requests, by pages that the last row sees (up to 2^24), no two alike
    const int pages = max(0, min(min(p1 - p0, a.window / a.page_rows + 1), 1 << 24));
    if (__builtin_amdgcn_ballot_w64(in && pages != __builtin_amdgcn_readfirstlane(pages))) {
      const int key = in ? pages << 6 | (63 - lane) : -1;
      if (in) place = 0;
      for (int r = 0; r < a.batch; ++r) place += in && __builtin_amdgcn_readlane(key, r) > key ? 1 : 0;
      // counts in that order, one per lane (lanes past the batch: places past it)
      ordered = (uint32_t)__builtin_amdgcn_ds_permute(place * 4, (int)cnt);
    }
  }
  const uint32_t incl = wave_incl_add_sat_u32(ordered);
  const uint32_t before = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)incl, 0x138, 0xf, 0xf, false);
  const uint64_t who = __builtin_amdgcn_ballot_w64((uint32_t)l.rank >= before && (uint32_t)l.rank < incl);
  if (__builtin_amdgcn_readlane(s0, 0) != 0 || __builtin_amdgcn_readlane(s1, a.batch - 1) != a.nnz ||
      __builtin_amdgcn_readlane(p0, 0) != 0)
    return false;
  l.ipB = __builtin_amdgcn_readlane(p1, a.batch - 1);
  if (l.ipB < 0 || (a.indices_capacity ? (int64_t)l.ipB > a.n_indices : (int64_t)l.ipB != a.n_indices))
    return false;
  if (!who) return false;
  const int at = __builtin_ctzll(who);
  const int r = __builtin_ctzll(__builtin_amdgcn_ballot_w64(in && place == at));
  l.tile0 = (int)(__builtin_amdgcn_readlane((int)incl, at) - 1u - (uint32_t)l.rank);
  l.qs = __builtin_amdgcn_readlane(s0, r);
  l.qe = __builtin_amdgcn_readlane(s1, r);
  l.ps = __builtin_amdgcn_readlane(p0, r);
  l.pe = __builtin_amdgcn_readlane(p1, r);
  l.tl = __builtin_amdgcn_readlane(t1, r);
  l.fbeg = 0;
  return true;
}

// Finds the workgroup's tile of TC columns; false: none, or a failed guard.
template <int W, int TC>
__device__ __forceinline__ bool find_tile(const WindowArgs &a, LocateSmem<W> &sm, Tile &t, int split,
                                          uint32_t block) {
  TileLoc &l = t.loc;
  if (a.qo) {
    if (a.batch <= 64 ? !locate_lanes<TC>(a, l, split, block)
                      : !locate_tile<W, false, TC, false, true>(a, sm, l, split, block))
      return false;
  } else {
    l.kvh = (int)(block % (uint32_t)a.hkv);
    l.rank = (int)(block / (uint32_t)a.hkv) - split * a.row_tiles;
    const int r = (int)((uint32_t)l.rank / (uint32_t)a.head_tiles);
    l.tile0 = l.rank - r * a.head_tiles;
    l.qs = r;
    l.qe = r + 1;
    l.fbeg = 0;
    const int32_t ip0 = a.indptr[0];
    l.ipB = uni(a.indptr[a.batch]);
    l.ps = uni(a.indptr[r]);
    l.pe = uni(a.indptr[r + 1]);
    l.tl = uni(a.last[r]);
    if (ip0 != 0 || l.ipB < 0 ||
        (a.indices_capacity ? (int64_t)l.ipB > a.n_indices : (int64_t)l.ipB != a.n_indices))
      return false;
  }
  if (l.ps < 0 || l.pe <= l.ps || l.pe > l.ipB || l.tl < 1 || l.tl > a.page_rows) return false;
  // (the enqueue bounds page_indices * page_rows by 2^31 - 1)
  t.kv_len = (l.pe - l.ps - 1) * a.page_rows + l.tl;
  t.group_rows = l.qe - l.qs;
  if (t.group_rows > t.kv_len) return false;
  t.fcols = t.group_rows * a.group;
  t.col0 = l.tile0 * TC;
  const int p0 = t.kv_len - t.group_rows;
  t.p_lo = p0 + row_of(a, t.col0);
  t.p_hi = p0 + row_of(a, min(t.col0 + TC - 1, t.fcols - 1));
  t.first_block = max(0, t.p_lo + 1 - a.window) >> 4;
  t.sink_blocks = min((int)(((uint32_t)a.sinks + 15) >> 4), t.first_block);
  t.blocks = t.sink_blocks + (t.p_hi >> 4) + 1 - t.first_block;
  return true;
}

// The page indices of tokens that some row of the request sees, in order.  (The same for
// every tile of the request.)
struct Pages {
  int first, sinks, n;  // first page of the windows, the sinks' pages, all of them
  __device__ __forceinline__ Pages(const WindowArgs &a, const Tile &t) {
    const int lg = a.blocks_lg + 4;
    first = max(0, t.kv_len - t.group_rows + 1 - a.window) >> lg;
    sinks = min((int)(((uint32_t)a.sinks + (1u << lg) - 1) >> lg), first);
    n = sinks + (t.loc.pe - t.loc.ps) - first;
  }
  __device__ __forceinline__ int32_t index(const WindowArgs &a, const Tile &t, int i) const {
    return a.indices[t.loc.ps + (i < sinks ? i : i - sinks + first)];
  }
};
__device__ __forceinline__ bool bad_page(const WindowArgs &a, int32_t x) {
  return x < 0 || (int64_t)x >= a.pool;
}
// Whether one is out of range: this thread's share, from `i` on, of `threads`.
__device__ __forceinline__ bool bad_pages(const WindowArgs &a, const Tile &t, int i, int threads) {
  const Pages p(a, t);
  bool bad = false;
  for (; i < p.n; i += threads) bad |= bad_page(a, p.index(a, t, i));
  return bad;
}

// Byte offset of row `row` of `page` for kv-head kvh, in K and V alike.
template <Kv KV>
__device__ __forceinline__ uint64_t row_at(const WindowArgs &a, int page, int row, int kvh) {
  return (uint64_t)(uint32_t)page * (uint32_t)(a.page_rows * kRowBytes<KV>) * (uint32_t)a.hkv +
         (uint64_t)(uint32_t)kvh * (uint32_t)a.head_bytes + (uint32_t)row * (uint32_t)a.row_bytes;
}
// The same in the MXFP4 scales.
__device__ __forceinline__ uint64_t scale_at(const WindowArgs &a, int page, int row, int kvh) {
  return (((uint64_t)(uint32_t)page * (uint32_t)a.hkv + (uint32_t)kvh) * (uint32_t)a.page_rows +
          (uint32_t)row) * 4;
}

// FP8: takes the pages' k_scale into scale_log2 and returns what the queries are multiplied
// with besides, exactly: 1, and for a scale of 0 or below 0 or -1.  The kernels mask and
// compare scores before the scale is multiplied in, which has to keep their order.
template <Kv KV>
__device__ __forceinline__ float take_key_scale(WindowArgs &a) {
  if constexpr (KV != kFp8) return 1.0f;
  const float scale = a.scale_log2 * a.kv_scales[0];
  if (scale != 0.0f) a.scale_log2 = fabsf(scale);
  return scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f;
}
__device__ __forceinline__ u32x4 times(const u32x4 &q, float factor) {
  u32x4 r;
#pragma unroll
  for (int x = 0; x < 4; ++x)
    r[x] = pack_hi16(__float_as_uint(bf16_lo(q[x]) * factor), __float_as_uint(bf16_hi(q[x]) * factor));
  return r;
}

// One column's O and LSE token by token, by one wave: for columns whose O is not finite.
// The tiles' products multiply a hidden token's V with a weight of zero, which is not
// zero where V is infinite or NaN; here hidden tokens, and weights of zero, have no part.
// (Not made to be fast: 0.5 us per token, up to the first score that is no number.)
template <Kv KV>
__device__ __forceinline__ void exact_column(const WindowArgs &args, const Tile &t, int f, int lane) {
  WindowArgs a = args;
  const float factor = take_key_scale<KV>(a), v_scale = KV == kFp8 ? a.kv_scales[1] : 1.0f;
  const int qi = row_of(a, f);
  const int64_t row = (int64_t)(t.loc.qs + qi) * a.hq + (int64_t)t.loc.kvh * a.group + (f - qi * a.group);
  const int end = t.kv_len - t.group_rows + qi + 1, beg = max(0, end - a.window);
  const int sinks = min(a.sinks, beg), n = sinks + end - beg;
  const uint32_t qw = *reinterpret_cast<const uint32_t *>(a.q + row * 128 + 2 * lane);
  const float q0 = bf16_lo(qw) * factor, q1 = bf16_hi(qw) * factor;
  float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  auto pair = [&](const uint16_t *base, const uint8_t *mx, uint64_t at, uint64_t sc, float &x, float &y) {
    const uint8_t *b = reinterpret_cast<const uint8_t *>(base) + at;
    if constexpr (KV == kBf16) {
      const uint32_t w = *reinterpret_cast<const uint32_t *>(b + 4 * lane);
      x = bf16_lo(w);
      y = bf16_hi(w);
    } else if constexpr (KV == kFp8) {
      const f32x2 w = __builtin_amdgcn_cvt_pk_f32_fp8(
          *reinterpret_cast<const uint16_t *>(b + 2 * lane), false);
      x = w[0];
      y = w[1];
    } else {
      const uint32_t w = mx4x8_to_bf16x8(b[lane], (uint32_t)mx[sc + (lane >> 4)] << 23)[0];
      x = bf16_lo(w);
      y = bf16_hi(w);
    }
  };
  for (int left = n; left > 0; left -= 64) {  // (counted down: a count up may pass 2^31 - 1)
    const int i = n - left + min(lane, left - 1), tok = i < sinks ? i : i - sinks + beg;
    const int pages = a.indices[t.loc.ps + (tok >> (a.blocks_lg + 4))];
    const int in_page = tok & (a.page_rows - 1);
    const int c = min(64, left);
    for (int j = 0; j < c; ++j) {
      const int page = __builtin_amdgcn_readlane(pages, j), r = __builtin_amdgcn_readlane(in_page, j);
      const uint64_t at = row_at<KV>(a, page, r, t.loc.kvh), sc = scale_at(a, page, r, t.loc.kvh);
      float k0, k1, v0, v1;
      pair(a.k, a.k_mx, at, sc, k0, k1);
      pair(a.v, a.v_mx, at, sc, v0, v1);
      float s = fmaf(q0, k0, q1 * k1);
#pragma unroll
      for (int x = 32; x >= 1; x >>= 1) s += __shfl_xor(s, x, 64);
      s *= a.scale_log2;
      if (s == -INFINITY) continue;
      const float mn = fmax_nan(m, s), old = m == -INFINITY ? 0.0f : fast_exp2(m - mn);
      const float p = fast_exp2(s - mn);  // (NaN at +inf)
      // The mean so far and the token's part of it: O stays within V's range, where sums
      // of p v may pass FP32's.  (What weighs nothing has no part, infinite or not.)
      const float ln = fmaf(l, old, p), keep = l * old / ln, part = p / ln;
      o0 = keep == 0.0f ? 0.0f : o0 * keep;
      o1 = keep == 0.0f ? 0.0f : o1 * keep;
      if (part != 0.0f) {
        o0 = fmaf(part, v0, o0);
        o1 = fmaf(part, v1, o1);
      }
      l = ln;
      m = mn;
      if (!(l == l)) {  // no number, which no later token changes
        left = 0;
        break;
      }
    }
  }
  *reinterpret_cast<uint32_t *>(a.out + row * 128 + 2 * lane) =
      bf16x2_pack(l == 0.0f ? NAN : o0 * v_scale, l == 0.0f ? NAN : o1 * v_scale);
  if (lane == 0) a.lse[row] = m + __log2f(l);
}

// ---- row tiles ---------------------------------------------------------------------
// One workgroup of W waves per (16 or 32 columns, kv-head[, split]).  Wave w takes steps w,
// w + W, ... of the walk (of its split's share of it), of 16 tokens (BF16) or 32, each through
// LDS of its own (PipeWave's slot: whole rows, so a load instruction covers whole lines, in an
// order that spreads the fragment reads over the banks), two of them in flight, and the wave
// states merge in LDS.  Per 32 tokens and 16 columns: S = K.Q^T in 8 MFMAs of 16x16x32, the
// softmax with a running maximum that moves only when a score passes it by 2^8, and O^T +=
// V^T.P^T in 16, P as a BF16 high part and a BF16 residual (16 bits: the roundings of a short
// window's few weights do not average out, see the long tiles').  Memory bounds the long walks (64 single tokens
// under windows of 4096 151 us, 6.5 TB/s, FP8 97, MXFP4 71), three dependent round trips
// (tables, page indices, rows) the short ones: one request's 128 tokens 5.0 us of which an
// empty command is 3.9.
// Rows, codes and scales go straight to LDS.  Widened to BF16 on the way, as the long tiles
// have them, MXFP4 rows cost a wave 360 cycles of LDS per 32 tokens, four times what the
// codes take (8 chunks of a few rows over 4-bit prefixes 39 us, 31 this way).
constexpr int kStash = 132;  // floats between two columns' O in LDS, and of a split's state

template <Kv KV>
using RowPipe = PipeWave<4, KV == kFp8, true, 1>;
// 16-row blocks of a step.
template <Kv KV>
constexpr int kStepBlocks = KV == kBf16 ? 1 : 2;
// A step's rows in LDS.  FP8: PipeWave's slot; BF16: the first half of its K and of its V.
// MXFP4: per block 16 rows of 64 code bytes, K then V, whose four 16-byte pieces are
// permuted by the row (piece c of row r at c ^ (r >> 2)), so that a fragment's read, one
// piece of all rows, and 64 bytes of four neighbouring rows each meet every bank once; then
// per block the K scale words, and the V ones, of rows mx_token(0), mx_token(1), ...
template <Kv KV>
struct RowSlot {
  using Pipe = RowPipe<KV>;
  static constexpr int kGroups = KV == kFp8 ? Pipe::kGroups : Pipe::kGroups / 2;  // of each of K and V
  static constexpr int kVShift = KV == kFp8 ? 0 : -kGroups * Pipe::kKGroup;  // of V, against PipeWave's
  static constexpr int kMxV = 2 * 1024, kMxKs = 4 * 1024, kMxVs = kMxKs + 128;
  static constexpr int kBytes = KV == kMx4   ? kMxVs + 128
                                : KV == kFp8 ? Pipe::kSlotBytes
                                             : kGroups * (Pipe::kKGroup + Pipe::kVGroup);
  static constexpr int kLoads = KV == kMx4 ? 8 : 2 * kGroups;  // instructions of a step
};
// MXFP4: the row of a block that row c of the MFMA tile S = K.Q^T stands for.  S leaves lane
// (col, quad) rows 4 quad + j, which are tokens 4 j + quad, and the V reads of the four
// quads then lie in four neighbouring rows.
__device__ __forceinline__ int mx_token(int c) { return 4 * (c & 3) + (c >> 2); }

template <Kv KV, int CT, int W>
struct RowsSmem {
  using Slot = RowSlot<KV>;
  // a wave's slots, and after its walk its columns' O
  static constexpr int kWaveBytes = (std::max(2 * Slot::kBytes, 16 * CT * kStash * 4) + 15) & ~15;
  __align__(16) uint8_t slots[W][kWaveBytes];
  LocateSmem<W> loc;
  float m[W][16 * CT], l[W][16 * CT];
  uint32_t bad[W];
  uint32_t arrived;
};

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Until this wave's LDS reads have returned: before loads into a slot that it read.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Split states go past L2, which the XCDs do not share.
__device__ __forceinline__ void store_state(float *p, float x, float y) {
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p), __builtin_bit_cast(uint64_t, f32x2{x, y}),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 load_state(const float *p) {
  return __builtin_bit_cast(f32x2, __hip_atomic_load(reinterpret_cast<const uint64_t *>(p),
                                                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

template <Kv KV, int CT, int W, bool NT>
__global__ __launch_bounds__(W * 64, KV == kMx4 && CT == 1 && W == 4 ? 4 : 2)
void window_rows_kernel(WindowArgs args) {
  constexpr int TC = 16 * CT;
  constexpr bool FP8 = KV == kFp8;
  using Pipe = RowPipe<KV>;
  using Slot = RowSlot<KV>;
  constexpr int H = kStepBlocks<KV>, kPlaced = 64 / H;  // steps placed at once
  __shared__ RowsSmem<KV, CT, W> sm;
  WindowArgs a = args;
  const float q_factor = take_key_scale<KV>(a), v_scale = FP8 ? a.kv_scales[1] : 1.0f;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uni(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  uint32_t block = blockIdx.x;
  if (KV == kMx4 && a.pair_heads) {
    block = ((block >> 4) << 4) + 2 * (block & 7) + ((block >> 3) & 1);
    if (block >= (uint32_t)a.pair_heads) return;
  }
  const int split = a.splits > 1 ? (int)(block / (uint32_t)(a.row_tiles * a.hkv)) : 0;
  Tile t;
  if (!find_tile<W, TC>(a, sm.loc, t, split, block)) return;
  const int kvh = t.loc.kvh;
  // tokens [full_beg, full_end) are seen by every column
  const int full_beg = max(0, t.p_hi + 1 - a.window), full_end = t.p_lo + 1;
  Pipe pw{a, lane, col, quad};
  uint8_t *const slots = sm.slots[wave];
  pw.reset(slots);
  // this lane's columns, one of each 16
  int beg_col[CT], end_col[CT];
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    const int f = t.col0 + 16 * x + col;
    const bool valid = f < t.fcols;
    const int qi = valid ? row_of(a, f) : 0;
    end_col[x] = valid ? t.kv_len - t.group_rows + qi + 1 : 0;
    beg_col[x] = max(0, end_col[x] - a.window);
    const uint16_t *qp =
        a.q + ((int64_t)(t.loc.qs + qi) * a.hq + (int64_t)kvh * a.group + (f - qi * a.group)) * 128;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d = KV == kMx4 ? 32 * quad + 8 * c : Pipe::q_dim(c, quad);
      pw.qf[x][c] = valid ? load16(qp + d) : u32x4{0, 0, 0, 0};
    }
  }
  // this split's steps [lo, hi), this wave's lo + wave + W i
  const int steps = (t.blocks + H - 1) / H;
  int lo = 0, hi = steps;
  if (a.splits > 1) {
    lo = (int)((int64_t)steps * split / a.splits);
    hi = (int)((int64_t)steps * (split + 1) / a.splits);
  }
  const int n = hi - lo > wave ? (hi - lo - wave + W - 1) / W : 0;

  // Where the blocks of the wave's steps lie, 64 at a time, one per lane: byte offset of the
  // first row in K and V (and in the MXFP4 scales), and block << 5 | rows (blocks have up to
  // 27 bits: unsigned).
  uint32_t at_lo = 0, at_hi = 0, sc_lo = 0, sc_hi = 0, meta = 0;
  auto locate = [&](int i0) {
    const int x = H * (lo + wave + W * (i0 + lane / H)) + lane % H;
    const bool in = x < t.blocks;
    const int b = t.block(x);
    int rows = in ? t.rows(a, x) : 0;
    const int page = in ? a.indices[t.loc.ps + (b >> a.blocks_lg)] : 0;
    if (page < 0 || (int64_t)page >= a.pool) rows = 0;  // (refused below)
    const int row = (b & ((1 << a.blocks_lg) - 1)) * 16;
    const uint64_t at = row_at<KV>(a, page, row, kvh);
    at_lo = (uint32_t)at;
    at_hi = (uint32_t)(at >> 32);
    if constexpr (KV == kMx4) {
      const uint64_t sc = scale_at(a, page, row, kvh);
      sc_lo = (uint32_t)sc;
      sc_hi = (uint32_t)(sc >> 32);
    }
    meta = (uint32_t)b << 5 | (uint32_t)rows;
  };
  auto lane64 = [&](uint32_t l, uint32_t h, int j) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)h, j) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)l, j);
  };
  auto rsrc = [](const void *base, uint64_t at, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t *>(reinterpret_cast<const uint8_t *>(base) + at), 0, bytes, 0x00020000);
  };
  // The loads of step i (of the placed ones) into the slot at LDS address `slot`
  constexpr int kHalf = Slot::kGroups / H;  // groups of a block (BF16, FP8)
  int lane_off[kHalf], mx_off = 0;
  if constexpr (KV == kMx4) {
    lane_off[0] = (lane >> 2) * a.row_bytes + (((lane & 3) ^ (lane >> 4)) << 4);
    mx_off = 4 * mx_token(lane & 15);
  } else {
    const int unit = (lane & (Pipe::kUnits - 1)) ^ Pipe::swizzle(lane / Pipe::kUnits);
#pragma unroll
    for (int x = 0; x < kHalf; ++x)
      lane_off[x] = (x * Pipe::kGroupRows + lane / Pipe::kUnits) * a.row_bytes + unit * 16;
  }
  auto issue = [&](int i, uint32_t slot) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int j = H * i + h;
      const int rows = __builtin_amdgcn_readlane((int)meta, j) & 31;
      const uint64_t at = lane64(at_lo, at_hi, j);
      const int bytes = rows > 0 ? (rows - 1) * a.row_bytes + kRowBytes<KV> : 0;
      const __amdgpu_buffer_rsrc_t rk = rsrc(a.k, at, bytes), rv = rsrc(a.v, at, bytes);
      if constexpr (KV == kMx4) {
        const uint64_t sc = lane64(sc_lo, sc_hi, j);
        lds_load16_at<NT>(rk, slot + 1024 * h, lane_off[0]);
        lds_load16_at<NT>(rv, slot + Slot::kMxV + 1024 * h, lane_off[0]);
        if (lane < 16) {
          lds_load4_at(rsrc(a.k_mx, sc, 4 * rows), slot + Slot::kMxKs + 64 * h, mx_off);
          lds_load4_at(rsrc(a.v_mx, sc, 4 * rows), slot + Slot::kMxVs + 64 * h, mx_off);
        }
      } else {
#pragma unroll
        for (int x = 0; x < kHalf; ++x) {
          lds_load16_at<NT>(rk, slot + (uint32_t)((h * kHalf + x) * Pipe::kKGroup), lane_off[x]);
          lds_load16_at<NT>(rv, slot + (uint32_t)(Slot::kVShift + Pipe::v_group(x) +
                                                  h * (Pipe::v_group(kHalf) - Pipe::v_group(0))),
                            lane_off[x]);
        }
      }
    }
  };

  float m_run[CT], l_run[CT];
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    m_run[x] = -INFINITY;
    l_run[x] = 0.0f;
  }
  f32x4(&acc)[2][8] = pw.acc;
  // The softmax and products of step i, whose rows lie at `slot`.
  auto process = [&](int i, const uint8_t *slot) {
    f32x4 s[CT][H] = {};  // s[x][h][j]: token 4 quad + j (MXFP4: 4 j + quad) of block h
    u32x4 v[8];           // Vᵀ fragments (FP8: still bytes)
    auto score = [&](const u32x4 &w, int c, int h) {
#pragma unroll
      for (int x = 0; x < CT; ++x)
        s[x][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(w), as_bf16x8(pw.qf[x][c]), s[x][h],
                                                          0, 0, 0);
    };
    if constexpr (KV == kBf16) {
      u32x4 k[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) k[c] = *reinterpret_cast<const u32x4 *>(slot + pw.kofs[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // the same tokens twice: for the weights' two parts
        const u32x2 b = lds_read_tr16(slot + Slot::kVShift + pw.vofs[e >> 1] + (e & 1) * 32);
        v[e] = u32x4{b[0], b[1], b[0], b[1]};
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) score(k[c], c, 0);
    } else if constexpr (FP8) {
      const auto k = pw.read_k((int)(slot - slots));
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = pw.read_v((int)(slot - slots), e);
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const u32x4 &w = k.f[FP8 ? y >> 2 : 0][y & 1];
        const int o = 2 * ((y >> 1) & 1);
        score(fp8x8_to_bf16x8(u32x2{w[o], w[o + 1]}), y >> 1, y & 1);
      }
    } else {
      // K: lane (col, quad) takes dims 32 quad + [0, 32) of row mx_token(col), one scale block.
      // V: dims 8 col + [0, 8) of tokens 4 j + quad; the widened pairs of two tokens make
      // two fragments of one dim each, dims 8 col + e of fragment e.
      u32x4 kw[2], vs[2];
      uint32_t ks[2], vw[2][4];
      const uint8_t *const kp = slot + mx_token(col) * 64 + ((quad ^ (col & 3)) << 4);
      const uint8_t *const vp = slot + Slot::kMxV + quad * 64 + (col & 3) * 4;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        kw[h] = *reinterpret_cast<const u32x4 *>(kp + 1024 * h);
        ks[h] = *reinterpret_cast<const uint32_t *>(slot + Slot::kMxKs + 64 * h + 4 * col);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        vs[h] = *reinterpret_cast<const u32x4 *>(slot + Slot::kMxVs + 64 * h + 16 * quad);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          vw[h][j] = *reinterpret_cast<const uint32_t *>(vp + 1024 * h + 256 * j + (((col >> 2) ^ j) << 4));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t scale = mx_scale(ks[h], quad);
#pragma unroll
        for (int c = 0; c < 4; ++c) score(mx4x8_to_bf16x8(kw[h][c], scale), c, h);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const u32x4 b0 = mx4x8_to_bf16x8(vw[h][j], mx_scale(vs[h][j], col >> 2));
          const u32x4 b1 = mx4x8_to_bf16x8(vw[h][j + 1], mx_scale(vs[h][j + 1], col >> 2));
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            v[e][2 * h + (j >> 1)] = pack_lo16(b0[e >> 1], b1[e >> 1]);
            v[e + 1][2 * h + (j >> 1)] = pack_hi16(b0[e >> 1], b1[e >> 1]);
          }
        }
    }
    int t0[H];
    int t_min = INT32_MAX, t_max = 0;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      t0[h] = (int)((uint32_t)__builtin_amdgcn_readlane((int)meta, H * i + h) >> 5) * 16;
      t_min = min(t_min, t0[h]);
      t_max = max(t_max, t0[h]);
    }
    const bool full = t_min >= full_beg && t_max <= full_end - 16;  // (t0 + 16 may be 2^31)
    if (!full) {
#pragma unroll
      for (int x = 0; x < CT; ++x)
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int tok = t0[h] + (KV == kMx4 ? 4 * j + quad : 4 * quad + j);
            s[x][h][j] =
                tok < end_col[x] && (tok >= beg_col[x] || tok < a.sinks) ? s[x][h][j] : -INFINITY;
          }
    }
    float ml[CT];
    bool above = false;
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      ml[x] = -INFINITY;
#pragma unroll
      for (int h = 0; h < H; ++h)
        ml[x] = fmax_nan(ml[x], fmax_nan(fmax_nan(s[x][h][0], s[x][h][1]), fmax_nan(s[x][h][2], s[x][h][3])));
      above |= ml[x] * a.scale_log2 > m_run[x] + 8.0f;
    }
    if (__builtin_amdgcn_ballot_w64(above)) {
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        const float mx = quad_max_nan(ml[x]) * a.scale_log2;
        const bool grow = mx > m_run[x] + 8.0f;
        const float m_ref = grow ? mx : m_run[x];
        if (__builtin_amdgcn_ballot_w64(grow && m_run[x] != -INFINITY)) {
          const float al = fast_exp2(m_run[x] - (m_ref == -INFINITY ? 0.0f : m_ref));
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[x][e] *= al;
          l_run[x] *= al;
        }
        m_run[x] = m_ref;
      }
    }
    uint32_t ph[CT][2 * H], pl[CT][2 * H];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      const float m_use = m_run[x] == -INFINITY ? 0.0f : m_run[x];  // nothing visible yet
#pragma unroll
      for (int y = 0; y < 2 * H; ++y) {
        const float x0 = fast_exp2(fmaf(s[x][y >> 1][2 * (y & 1)], a.scale_log2, -m_use));
        const float x1 = fast_exp2(fmaf(s[x][y >> 1][2 * (y & 1) + 1], a.scale_log2, -m_use));
        const uint32_t b0 = __float_as_uint(x0), b1 = __float_as_uint(x1);
        ph[x][y] = pack_hi16(b0, b1);
        pl[x][y] = pack_hi16(__float_as_uint(x0 - __uint_as_float(b0 & 0xffff0000u)),
                             __float_as_uint(x1 - __uint_as_float(b1 & 0xffff0000u)));
        l_run[x] += x0 + x1;
      }
    }
    if constexpr (KV == kBf16) {
      // high parts and residuals in the two halves of the contraction
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int x = 0; x < CT; ++x)
          acc[x][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              as_bf16x8(v[e]), as_bf16x8(ph[x][0], ph[x][1], pl[x][0], pl[x][1]), acc[x][e], 0, 0, 0);
    } else {
      bf16x8 w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = as_bf16x8(FP8 ? fp8x8_to_bf16x8(u32x2{v[e][0], v[e][1]}) : v[e]);
#pragma unroll
        for (int x = 0; x < CT; ++x)
          acc[x][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              w[e], as_bf16x8(ph[x][0], ph[x][1], ph[x][2], ph[x][3]), acc[x][e], 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int x = 0; x < CT; ++x)
          acc[x][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              w[e], as_bf16x8(pl[x][0], pl[x][1], pl[x][2], pl[x][3]), acc[x][e], 0, 0, 0);
    }
  };

  const uint32_t ring_at =
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)sm.slots[wave];
  // The thread's first page index comes with those of the walk, and is looked at before
  // the first rows are under way: loads return in order.
  const Pages pages(a, t);
  const int32_t own_page = tid < pages.n ? pages.index(a, t, tid) : 0;
  bool bad = false;
  for (int i0 = 0; i0 == 0 || i0 < n; i0 += kPlaced) {
    const int c = min(kPlaced, n - i0);
    if (c > 0) locate(i0);
    if (i0 == 0) bad = bad_page(a, own_page);
    if (i0 == 0 && q_factor != 1.0f)
#pragma unroll
      for (int x = 0; x < CT; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) pw.qf[x][y] = times(pw.qf[x][y], q_factor);
    // (queries and index words have arrived: no wait of the compiler's in the walk)
#pragma unroll
    for (int x = 0; x < CT; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) asm volatile("" : "+v"(pw.qf[x][y]));
    asm volatile("" : "+v"(at_lo), "+v"(at_hi), "+v"(sc_lo), "+v"(sc_hi), "+v"(meta));
    wait_reads();
    if (c > 0) issue(0, ring_at);
    if (c > 1) issue(1, ring_at + (uint32_t)Slot::kBytes);
    if (i0 == 0 && pages.n > W * 64) {
      bad |= bad_pages(a, t, tid + W * 64, W * 64);
      asm volatile("" ::"s"(__builtin_amdgcn_ballot_w64(bad)));
    }
    for (int i = 0; i < c; ++i) {
      // (of the loads, at most the next step's outstanding)
      if (i + 1 < c)
        wait_loads<Slot::kLoads>();
      else
        wait_loads<0>();
      const int at = (i & 1) * Slot::kBytes;
      process(i, slots + at);
      if (i + 2 < c) {
        wait_reads();
        issue(i + 2, ring_at + (uint32_t)at);
      }
    }
  }

  // The wave's columns to its slot.  acc[x][e][j] = O[column of the x-th 16][16 e + 4 quad + j]
  // (MXFP4: [32 quad + 8 j + e])
  wait_reads();
  wave_lds_fence();
  float *const stash = reinterpret_cast<float *>(sm.slots[wave]);
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    const float l_col = quad_sum(l_run[x]);
    float *const o = stash + (16 * x + col) * kStash;
    if constexpr (KV == kMx4) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<f32x4 *>(o + 32 * quad + 8 * j + e) =
              f32x4{acc[x][e][j], acc[x][e + 1][j], acc[x][e + 2][j], acc[x][e + 3][j]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) *reinterpret_cast<f32x4 *>(o + 16 * e + 4 * quad) = acc[x][e];
    }
    if (quad == 0) {
      sm.m[wave][16 * x + col] = m_run[x];
      sm.l[wave][16 * x + col] = l_col;
    }
  }
  if (block_or(bad, sm.bad)) return;
  const int cols = min(TC, t.fcols - t.col0);
  constexpr int kItems = TC * 32 / (W * 64);  // 4 dims of a column each
  f32x4 o[kItems];
  float ms[kItems], ls[kItems];
#pragma unroll
  for (int y = 0; y < kItems; ++y) {
    const int c = (y * W * 64 + tid) >> 5, d = (tid & 31) * 4;
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) M = fmaxf(M, sm.m[i][c]);
    f32x4 O = {};
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float w = sm.m[i][c] == -INFINITY ? 0.0f : fast_exp2(sm.m[i][c] - M);
      const f32x4 x = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(sm.slots[i]) +
                                                       c * kStash + d);
      L = fmaf(sm.l[i][c], w, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = fmaf(x[e], w, O[e]);
    }
    o[y] = O;
    ms[y] = M;
    ls[y] = L;
  }
  if (a.splits > 1) {
    // Every split writes its columns' states and counts itself at the tile's word; the last
    // one finds them all, merges them and clears the word for the queue's next command.
    // Nobody waits.  Each wave waits for its own stores before the barrier behind which
    // one thread counts the workgroup (a release fence would write the XCD's L2 back).
    const int64_t step = (int64_t)a.row_tiles * a.hkv * TC * kStash;
    float *const tile_states = a.states + ((int64_t)t.loc.rank * a.hkv + kvh) * TC * kStash;
#pragma unroll
    for (int y = 0; y < kItems; ++y) {
      const int c = (y * W * 64 + tid) >> 5, d = (tid & 31) * 4;
      if (c >= cols) continue;
      float *const st = tile_states + split * step + c * kStash;
      store_state(st + 4 + d, o[y][0], o[y][1]);
      store_state(st + 6 + d, o[y][2], o[y][3]);
      if (d == 0) store_state(st, ms[y], ls[y]);
    }
    wait_loads<0>();  // and stores
    __syncthreads();
    uint32_t *const word = a.arrived + (uint64_t)(t.loc.rank * a.hkv + kvh) * (loom::kMx4JoinBytes / 4);
    if (tid == 0)
      sm.arrived = __hip_atomic_fetch_add(word, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (sm.arrived != (uint32_t)a.splits - 1u) return;
    if (tid == 0) __hip_atomic_store(word, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int y = 0; y < kItems; ++y) {
      const int c = min((y * W * 64 + tid) >> 5, cols - 1), d = (tid & 31) * 4;
      float M = -INFINITY, L = 0.0f;
      f32x4 O = {};
      for (int i0 = 0; i0 < a.splits; i0 += 4) {
        f32x2 ml[4], x[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // past the last state: its values again, with no weight
          const float *st = tile_states + min(i0 + i, a.splits - 1) * step + c * kStash;
          ml[i] = load_state(st);
          x[i][0] = load_state(st + 4 + d);
          x[i][1] = load_state(st + 6 + d);
        }
        float mb = M;
#pragma unroll
        for (int i = 0; i < 4; ++i) mb = fmaxf(mb, ml[i][0]);
        const float old = M == -INFINITY ? 0.0f : fast_exp2(M - mb);
        L *= old;
        O *= old;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w =
              i0 + i < a.splits && ml[i][0] != -INFINITY ? fast_exp2(ml[i][0] - mb) : 0.0f;
          L = fmaf(ml[i][1], w, L);
#pragma unroll
          for (int e = 0; e < 4; ++e) O[e] = fmaf(x[i][e >> 1][e & 1], w, O[e]);
        }
        M = mb;
      }
      o[y] = O;
      ms[y] = M;
      ls[y] = L;
    }
  }
  // Columns that are not finite are found token by token.  (The normalizer alone overflows
  // over a V of zeros where scores of 2^31 are off by more than 2^7 in FP32.)
#pragma unroll
  for (int y = 0; y < kItems; ++y) {
    const int c0 = 2 * (y * W + wave);  // the wave's two columns
    const int c = c0 + (lane >> 5), d = (lane & 31) * 4;
    o[y] *= 1.0f / ls[y] * v_scale;
    bool finite = ls[y] < INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) finite &= fabsf(o[y][e]) < INFINITY;
    const uint64_t redo = __builtin_amdgcn_ballot_w64(c < cols && !finite);
    const bool mine = (lane < 32 ? (uint32_t)redo : (uint32_t)(redo >> 32)) == 0;
    if (c < cols && mine) {
      const int fc = t.col0 + c, rc = row_of(a, fc);
      const int64_t row = (int64_t)(t.loc.qs + rc) * a.hq + (int64_t)kvh * a.group + (fc - rc * a.group);
      *reinterpret_cast<u32x2 *>(a.out + row * 128 + d) =
          u32x2{bf16x2_pack(o[y][0], o[y][1]), bf16x2_pack(o[y][2], o[y][3])};
      if (d == 0) a.lse[row] = ms[y] + __log2f(ls[y]);
    }
    if (redo)
#pragma unroll 1
      for (int x = 0; x < 2; ++x)
        if ((uint32_t)(redo >> (32 * x))) exact_column<KV>(args, t, t.col0 + c0 + x, lane);
  }
}

// ---- long tiles --------------------------------------------------------------------
// MXFP4 rows on their way to LDS as BF16: lane l takes 32 values, block mx_block(l) of row
// mx_row(l) of a 16-row block, and the row's scale word.  LDS writes the 16 bytes of 8 lanes at
// once, to 32 banks: two blocks, 64 bytes apart, of rows of the four groups, 16 bytes further
// each in K, 32 in V (where lanes of the last two groups write neighbouring units in turn).
// (Four blocks of two groups shared banks: 122 against 61 million conflict cycles, the rest
// the fragments' reads, for 16384 rows under a window of 4096, 932 against 927 us; rows in
// order took 1.1 ms.)
__device__ __forceinline__ int mx_block(int lane) { return (lane & 1) + ((lane >> 2) & 2); }
__device__ __forceinline__ int mx_group(int lane) { return (lane >> 1) & 3; }
__device__ __forceinline__ int mx_row(int lane) { return 4 * mx_group(lane) + (lane >> 4); }
// A lane's 32 values to a slot as BF16; `group`: where the row's group lies.
template <class Pipe, bool V>
__device__ __forceinline__ void put_mx(uint8_t *group, int lane, const u32x4 &w, uint32_t scales) {
  const int b = mx_block(lane), r3 = lane >> 4;
  const bool turn = V && (lane & 4);
  uint8_t *const dst = group + r3 * 256 + ((4 * b) ^ Pipe::swizzle(r3)) * 16;
  uint8_t *const even = dst + (turn ? 16 : 0), *const odd = dst + (turn ? 0 : 16);
  const uint32_t scale = mx_scale(scales, b);
#pragma unroll
  for (int u = 0; u < 4; u += 2) {
    const uint32_t x = turn ? w[u + 1] : w[u], y = turn ? w[u] : w[u + 1];
    *reinterpret_cast<u32x4 *>(even + 16 * u) = mx4x8_to_bf16x8(x, scale);
    *reinterpret_cast<u32x4 *>(odd + 16 * u) = mx4x8_to_bf16x8(y, scale);
  }
}

// Many rows: the pipelined long tiles of paged prefill (PipeWave: 32 columns per wave, NW
// waves over 32 * NW columns, G = W / NW groups of them that split the walk) over the
// blocks of the walk, in 32-token steps of two blocks each.  A wave masks the sinks' steps,
// those from the walk's begin (the tile's first row's window) to its own last row's, up to
// five where a group is one head, and two at the end; the steps between take PipeWave's
// unmasked path.  (A step whose tokens are all hidden from a column that has seen none yet
// takes the branch that moves the reference.)  P is rounded once to BF16 for the product, as
// in the other long tiles, which adds to O's error against 64 bits (rms, O's own rounding
// among it) 6 to 9% under windows of 2-16 tokens, 3% of 64, 2% of 128 and 1% from 1024 on,
// where the errors of many tokens average out; row tiles (tile_cols 16) add nothing.  The
// normalizer sums the weights before their rounding, so LSE keeps FP32's precision.  (Two
// sums, one for each, take 5 to 20% of the time: registers spill.)  The waves' issue and LDS
// reads bound long walks (16384 rows under a window of 4096, MXFP4: 926 us, 1040 TFLOP/s,
// MFMA busy 42%), a tile's beginning and end the short ones (windows of 128: 9 of a tile's
// 16 us).
//
// BF16 and FP8 blocks are loaded straight into the ring, NW slots deep.  MXFP4 codes go
// through registers, 32 values and their scale per lane and block, two steps ahead, and are
// written to a ring of two slots as BF16: widened once per workgroup instead of once per
// wave (32 conversions per wave and step, and V's scales, which run along the
// contraction's other axis, would have to be applied to P).
template <int W, int NW>
struct LongSmem {
  LocateSmem<W> loc;
  float m[W][32], l[W][32];  // the groups' column states
  uint32_t bad[W];
  uint32_t redo[NW];         // columns of a group's wave whose O is not finite
  int32_t next_idx[W][64];   // page indices of the next 64 blocks
};

template <Kv KV, int W, int NW>
__global__ __launch_bounds__(W * 64, 2) void window_long_kernel(WindowArgs args) {
  constexpr int G = W / NW, TC = 32 * NW;
  constexpr int kOutRow = 256 + 16;  // bytes of a row of O in LDS
  constexpr bool FP8 = KV == kFp8, MX = KV == kMx4;
  using Pipe = PipeWave<NW, FP8, false, G, true>;
  constexpr int kSlot = Pipe::kSlotBytes, kSlots = MX ? 2 : Pipe::kSlots;
  constexpr int kRingBytes = G * kSlots * kSlot;
  constexpr int kMergeBytes = G > 1 ? W * 64 * 64 * 4 : 0;
  constexpr int kOutBytes = W * 32 * kOutRow;
  __shared__ LongSmem<W, NW> sm;
  __shared__ __align__(16) uint8_t ring[std::max({kRingBytes, kMergeBytes, kOutBytes})];
  WindowArgs a = args;
  const float q_factor = take_key_scale<KV>(a), v_scale = FP8 ? a.kv_scales[1] : 1.0f;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uni(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  Tile t;
  if (!find_tile<W, TC>(a, sm.loc, t, 0, blockIdx.x)) return;
  const int kvh = t.loc.kvh;
  const int wq = wave % NW, grp = wave / NW;  // the wave's columns and its group
  const int own0 = t.col0 + 32 * wq;
  const int p0 = t.kv_len - t.group_rows;
  Pipe lw{a, lane, col, quad};
  // this lane's columns, one of each 16: their causal ends (0: no column)
  int end_col[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int f = own0 + 16 * c + col;
    end_col[c] = f < t.fcols ? p0 + row_of(a, f) + 1 : 0;
  }
  // Output row of column f.
  auto out_row = [&](int f) {
    const int qi = row_of(a, f);
    return (t.loc.qs + qi) * a.hq + kvh * a.group + (f - qi * a.group);
  };
  lw.reset(ring + grp * kSlots * kSlot);
  // Steps that need no mask, [first_full, last_full): whose tokens every column of the
  // wave sees; and the steps up to the wave's last column's own token.
  int first_full = 0, last_full = 0, own_steps = 0;
  if (own0 < t.fcols) {
    const int w_lo = p0 + row_of(a, own0), w_hi = p0 + row_of(a, min(own0 + 31, t.fcols - 1));
    const int x0 = t.sink_blocks - t.first_block;  // place of block b of the window: b + x0
    first_full = (((max(0, w_hi + 1 - a.window) + 15) >> 4) + x0 + 1) >> 1;
    last_full = (((w_lo + 1) >> 4) + x0) >> 1;
    own_steps = ((w_hi >> 4) + 1 + x0 + 1) >> 1;
  }
  // The first page indices, then the queries: the first K/V loads wait for the former only.
  const int idx =
      lane < t.blocks ? a.indices[t.loc.ps + (t.block(lane) >> a.blocks_lg)] : 0;
  const Pages pages(a, t);
  const int32_t own_page = tid < pages.n ? pages.index(a, t, tid) : 0;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int f = own0 + 16 * c + col;
    const uint16_t *qp = a.q + (f < t.fcols ? (int64_t)out_row(f) * 128 : 0);
#pragma unroll
    for (int x = 0; x < 4; ++x) lw.qf[c][x] = load16(qp + Pipe::q_dim(x, quad));
  }
  // Lane l holds the place of block 64 win + l of the walk in the wave's matrix (K or V): its
  // first row's address (48 bits), above it the valid rows, and (MXFP4) the block of scales.
  const bool loads_k = wq < NW / 2;
  const uint64_t kv_base = (uint64_t)(loads_k ? a.k : a.v);
  const uint64_t mx_base = MX ? (uint64_t)(loads_k ? a.k_mx : a.v_mx) : 0;
  int win = -1;
  uint32_t blk_lo = 0, blk_hi = 0, blk_mx = 0;
  auto place = [&](int b) {
    if ((b >> 5) == win) return;
    win = b >> 5;
    const int x = 64 * win + lane;
    const int blk = t.block(x);
    int rows = x < t.blocks ? t.rows(a, x) : 0;
    const int pg = win == 0 ? idx : sm.next_idx[wave][lane];
    if (bad_page(a, pg)) rows = 0;  // (the request is refused)
    const int row = (blk & ((1 << a.blocks_lg) - 1)) * 16;
    const uint64_t at = kv_base + row_at<KV>(a, pg, row, kvh);
    blk_lo = (uint32_t)at;
    blk_hi = ((uint32_t)(at >> 32) & 0xffffu) | (uint32_t)rows << 16;
    if constexpr (MX) blk_mx = (uint32_t)(scale_at(a, pg, row, kvh) >> 6);
    asm volatile("" ::"v"(blk_lo), "v"(blk_hi) : "memory");  // next_idx is read
    // (past the walk's end: past the buffer's, or of no use)
    lds_load4(__builtin_amdgcn_make_buffer_rsrc(const_cast<int32_t *>(a.indices + t.loc.ps), 0,
                                                4 * (t.loc.pe - t.loc.ps), 0x00020000),
              &sm.next_idx[wave][0], (t.block(x + 64) >> a.blocks_lg) * 4);
  };
  struct Place {
    uint64_t at, scales;  // addresses of its first row and its first scales
    int rows;
  };
  auto block_at = [&](int x) {
    const int l = x & 63;
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)blk_hi, l);
    return Place{(uint64_t)(hi & 0xffffu) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)blk_lo, l),
                 MX ? mx_base + ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)blk_mx, l) << 6) : 0,
                 (int)(hi >> 16)};
  };
  auto rsrc = [](uint64_t at, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(at), 0, bytes, 0x00020000);
  };
  // Checked and masked while the first blocks are on their way.
  bool bad = false;
  auto first = [&]() {
    bad = bad_page(a, own_page);
    if (pages.n > W * 64) bad |= bad_pages(a, t, tid + W * 64, W * 64);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int x = 0; x < 4; ++x) lw.qf[c][x] = end_col[c] ? lw.qf[c][x] : u32x4{0, 0, 0, 0};
    if (q_factor != 1.0f)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int x = 0; x < 4; ++x) lw.qf[c][x] = times(lw.qf[c][x], q_factor);
  };
  auto mask = [&](typename Pipe::Scores &s, int b) {
    const int t0 = 16 * t.block(2 * b) + 4 * quad, t1 = 16 * t.block(2 * b + 1) + 4 * quad;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int beg = end_col[c] - a.window;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = (h ? t1 : t0) + i;
          s.s[c][h][i] =
              tok < end_col[c] && (tok >= beg || tok < a.sinks) ? s.s[c][h][i] : -INFINITY;
        }
    }
  };
  const int nb = (t.blocks + 1) >> 1, steps = (nb + G - 1) / G;
  const int nbw = uni(max(0, (min(own_steps, nb) - grp + G - 1) / G));
  first_full = uni(first_full);
  last_full = uni(last_full);
  auto slot_of = [](int j) { return (j & (kSlots - 1)) * kSlot; };
  typename Pipe::Scores sa, sb;
  typename Pipe::VFrags v = {};
  typename Pipe::Weights w = {};
  // The walk: at step j the wave's group takes the weights of its j-th block, the scores of
  // the next and the products of the one before; `feed(j, s)` (s: j, or its slot) meets the
  // other waves and refills the ring.
  auto walk = [&](auto feed) {
    if (nbw > 0) {
      const auto k = lw.read_k(0);
#pragma unroll
      for (int c = 0; c < 8; ++c) lw.score(k, sa, c);
    }
    int j = 0;
    while (j < nbw) {
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        if (s > 0 && j >= nbw) break;
        feed(j, s);
        typename Pipe::Scores &cur = s & 1 ? sb : sa, &nxt = s & 1 ? sa : sb;
        const int b = G * j + grp;
        if (b < first_full || b >= last_full) mask(cur, b);
        lw.step(slot_of(s + 1), slot_of(s), cur, nxt, v, w);
        ++j;
      }
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) lw.product(v, w, x);
    for (; j < steps; ++j) {  // (MXFP4: registers are named by j's parity)
      if (!MX || !(j & 1))
        feed(j, MX ? 0 : j);
      else
        feed(j, 1);
    }
  };
  const uint32_t ring_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)ring +
                            (uint32_t)(grp * kSlots * kSlot);
  if constexpr (!MX) {
    // K runs one block ahead of V, so that one barrier per step publishes K (j + 1) and V (j);
    // a slot is refilled one step after it was read.
    int lane_off[16 / Pipe::kGroupRows];
    {
      const int sub = (lane & (Pipe::kUnits - 1)) ^ Pipe::swizzle(lane / Pipe::kUnits);
#pragma unroll
      for (int x = 0; x < 16 / Pipe::kGroupRows; ++x)
        lane_off[x] = (x * Pipe::kGroupRows + lane / Pipe::kUnits) * a.row_bytes + sub * 16;
    }
    auto load = [&](int b, uint32_t slot) {
      place(b);
#pragma unroll
      for (int y = 0; y < (NW == 4 ? 1 : 2); ++y) {
        const int h = NW == 4 ? (wq & 1) : y;
        const Place p = block_at(2 * b + h);
        const __amdgpu_buffer_rsrc_t r =
            rsrc(p.at, p.rows > 0 ? (p.rows - 1) * a.row_bytes + kRowBytes<KV> : 0);
        constexpr int kHalf = Pipe::kGroups / 2;
#pragma unroll
        for (int x = 0; x < kHalf; ++x) {
          const uint32_t kg = (uint32_t)((h * kHalf + x) * Pipe::kKGroup);
          const uint32_t vg = (uint32_t)(Pipe::v_group(x) + h * (Pipe::v_group(kHalf) - Pipe::v_group(0)));
          lds_load16_at(r, slot + (loads_k ? kg : vg), lane_off[x]);
        }
      }
    };
    const int ahead = uni(kSlots - (loads_k ? 0 : 1));
    if (loads_k) load(grp, ring_lds);
#pragma unroll
    for (int j = 1 - kSlots; j < 0; ++j) load(G * (j + ahead) + grp, ring_lds + slot_of(j + ahead));
    first();
    Pipe::template publish<(kSlots - 1) * Pipe::kLoads>();
    walk([&](int j, int s) {
      Pipe::template publish<(kSlots - 2) * Pipe::kLoads>();
      load(G * (j + ahead) + grp, ring_lds + slot_of(s + ahead));
    });
  } else {
    // The wave's share of a block: its 16-row half (NW = 2: both), 32 values per lane.
    constexpr int kHalves = NW == 4 ? 1 : 2;
    struct Share {
      u32x4 w[kHalves];
      uint32_t s[kHalves];
    };
    auto fetch = [&](int b, Share &g) {
      place(b);
#pragma unroll
      for (int y = 0; y < kHalves; ++y) {
        const Place p = block_at(2 * b + (NW == 4 ? (wq & 1) : y));
        g.w[y] = load16_rows<false>(rsrc(p.at, p.rows > 0 ? (p.rows - 1) * a.row_bytes + 64 : 0),
                                    mx_row(lane) * a.row_bytes + mx_block(lane) * 16);
        g.s[y] =
            __builtin_amdgcn_raw_buffer_load_b32(rsrc(p.scales, 4 * p.rows), 4 * mx_row(lane), 0, 0);
      }
    };
    uint8_t *const group_ring = ring + grp * kSlots * kSlot;
    const int half_at = loads_k ? 4 * Pipe::kKGroup : Pipe::v_group(4) - Pipe::v_group(0);
    auto put = [&](int slot, const Share &g) {
      int l = lane;
      // (with both halves of a block in flight, places are worked out anew: no registers)
      if constexpr (kHalves > 1) asm volatile("" : "+v"(l));
      const int group = mx_group(l);
      uint8_t *const at = group_ring + slot + (NW == 4 ? (wq & 1) * half_at : 0) +
                          (loads_k ? group * Pipe::kKGroup : Pipe::v_group(group));
#pragma unroll
      for (int y = 0; y < kHalves; ++y) {
        if (loads_k)
          put_mx<Pipe, false>(at + y * half_at, l, g.w[y], g.s[y]);
        else
          put_mx<Pipe, true>(at + y * half_at, l, g.w[y], g.s[y]);
      }
    };
    // K (j + 2) and V (j + 1) are written at step j, to slots read at step j - 1.
    const int ahead = uni(loads_k ? 2 : 1);
    Share g[2], f0;
    if (loads_k) fetch(grp, f0);
    fetch(G * (ahead - 1) + grp, g[0]);
    fetch(G * ahead + grp, g[1]);
    first();
    if (loads_k) put(0, f0);
    put(slot_of(ahead - 1), g[0]);
    fetch(G * (ahead + 1) + grp, g[0]);
    auto meet = [&]() {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    meet();
    // (g[1]: item ahead, g[0]: ahead + 1; item j + ahead sits in g[(j + 1) & 1])
    walk([&](int j, int s) {
      meet();  // (every wave has read K (j) and V (j - 1))
      put(slot_of(s + ahead), g[(s + 1) & 1]);
      fetch(G * (j + ahead + 2) + grp, g[(s + 1) & 1]);
    });
  }
  wait_loads<0>();

  float L[2], M[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    L[c] = quad_sum(lw.lsum[c]);
    M[c] = -lw.nmax[c];
    if (G > 1 && quad == 0) {
      sm.m[wave][16 * c + col] = M[c];
      sm.l[wave][16 * c + col] = L[c];
    }
  }
  if (tid < NW) sm.redo[tid] = 0;
  if (block_or(bad, sm.bad)) return;
  constexpr int kOwn = 8 / G;  // 16-dim blocks that a group finishes
  if constexpr (G > 1) {
    // The groups' states merge: every wave writes the dims that other groups finish, group
    // g finishes dims 128 g / G .. of its columns.
    static_assert(W * 2 * 8 * 64 * sizeof(f32x4) <= sizeof(ring), "merge staging");
    f32x4 *xs = reinterpret_cast<f32x4 *>(ring) + lane;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e / kOwn != grp) xs[((wave * 2 + c) * 8 + e) * 64] = lw.acc[c][e];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int g = 0; g < G; ++g) M[c] = fmaxf(M[c], sm.m[g * NW + wq][16 * c + col]);
      float f[G];
      L[c] = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float m = sm.m[g * NW + wq][16 * c + col];
        f[g] = m == -INFINITY ? 0.0f : fast_exp2(m - M[c]);
        L[c] = fmaf(sm.l[g * NW + wq][16 * c + col], f[g], L[c]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e / kOwn != grp) continue;
        f32x4 o = {};
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const f32x4 x = g == grp ? lw.acc[c][e] : xs[(((g * NW + wq) * 2 + c) * 8 + e) * 64];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = fmaf(x[i], f[g], o[i]);
        }
        lw.acc[c][e] = o;
      }
    }
  }
  // Columns that are not finite are found token by token.
  uint32_t redo = 0;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float inv = 1.0f / L[c] * v_scale;
    f32x4 zs = {};  // NaN: not finite
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e / kOwn == grp) {
        lw.acc[c][e] *= inv;
#pragma unroll
        for (int i = 0; i < 4; ++i) zs[i] = fmaf(lw.acc[c][e][i], 0.0f, zs[i]);
      }
    const float z = (zs[0] + zs[1]) + (zs[2] + zs[3]);
    const uint64_t b = __builtin_amdgcn_ballot_w64(end_col[c] && !(z == 0.0f && L[c] < INFINITY));
    redo |= (uint32_t)((b | b >> 16 | b >> 32 | b >> 48) & 0xffff) << (16 * c);
  }
  if constexpr (G > 1) {
    if (redo && lane == 0) atomicOr(&sm.redo[wq], redo);
    __syncthreads();
    redo = (uint32_t)uni((int)sm.redo[wq]);
  }
  // O through LDS, each wave its own 32 rows: whole rows go out 16 bytes per lane.
  static_assert(W * 32 * kOutRow <= sizeof(ring), "O staging");
  uint8_t *ot = ring + wave * 32 * kOutRow;
  int own_col = col;  // (found again: held through the walk it would cost registers)
  asm volatile("" : "+v"(own_col));
  int row_head[2];  // output row of each tile's column, -1: none
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const bool mine = end_col[c] && !(redo >> (16 * c + col) & 1);
    row_head[c] = mine ? out_row(own0 + 16 * c + own_col) : -1;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e / kOwn == grp)
        *reinterpret_cast<u32x2 *>(ot + (16 * c + col) * kOutRow + 32 * e + 8 * quad) =
            u32x2{bf16x2_pack(lw.acc[c][e][0], lw.acc[c][e][1]),
                  bf16x2_pack(lw.acc[c][e][2], lw.acc[c][e][3])};
    if (quad == 0 && grp == 0 && mine) a.lse[row_head[c]] = M[c] + __log2f(L[c]);
  }
  wave_lds_fence();
  constexpr int kOwnUnits = 2 * kOwn, kRowsPer = 64 / kOwnUnits;  // 16-byte units of a row
  const int unit = grp * kOwnUnits + (lane & (kOwnUnits - 1));
#pragma unroll
  for (int x = 0; x < 32 / kRowsPer; ++x) {
    const int r = x * kRowsPer + lane / kOwnUnits;  // column of the wave
    const int rh0 = __shfl(row_head[0], r & 15, 64), rh1 = __shfl(row_head[1], r & 15, 64);
    const int rh = r < 16 ? rh0 : rh1;
    if (rh >= 0)
      *reinterpret_cast<u32x4 *>(a.out + (int64_t)rh * 128 + unit * 8) =
          *reinterpret_cast<const u32x4 *>(ot + r * kOutRow + unit * 16);
  }
  if (redo)
    for (int c = grp; c < 32; c += G)
      if (redo >> c & 1) exact_column<KV>(args, t, own0 + c, lane);
}

}  // namespace

// ---- plan / enqueue -------------------------------------------------------------------
struct loom_window_attention_plan {
  loom_window_attention_plan_info_t info{};
  int cus = 0;
  uint32_t groups = 1;  // long tiles: wave groups that split a walk
  bool once = false;    // row tiles: a request has one tile per kv-head, as a rule
  uint64_t least_tiles = 0;  // that the command holds if no request's last one is in part empty
};

// Bytes of a command's rows from which they are loaded past the caches, where each is
// read once: 64 requests under windows of 4096 (1.1 GB) 170 -> 151 us, 8 of 8192 on FP8
// pages (134 MB) 32.5 -> 29.5; but 16 of 1024 (61 MB), which the last-level cache may hold
// still, 14.4 -> 17.1.
constexpr uint64_t kPastCaches = 96ull << 20;

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint64_t kMaxHeads = 4096;  // kv-heads: a row of all of them in a 32-bit stride
constexpr int kMaxSplits = 16;
constexpr uint64_t kLongWalk = 2048;  // tokens, from which a join costs little

// Columns per workgroup, from the number of row tiles of 16 that the command holds (a
// request's last one is about half full).  Microseconds, 16 / 32 / long, rows behind 5000
// tokens 32/8:
//  - one per CU: 16 (8 x 16 rows under windows of 1024 13.7 / 15.0 / 20.0, over the whole
//    prefix 56 / 63 / 82; one request of 8 rows 9.5 / 13.5 / 18.0);
//  - two: 32, which share a walk's rows (8 x 32 rows 23.4 / 17.3 / 20.5, whole 94 / 59 / 80;
//    MXFP4 27.2 / 19.1 / 26.3, whole 81 / 55 / 72, but 8 x 1-32, 300 tiles, 39 / 48: two
//    workgroups of its 16 fit a CU);
//  - more: long tiles (8 x 64 rows under windows of 1024 24 / 21), but where long walks
//    differ (`uneven`), rows balance them: three per CU (8 x 48 rows, whole prefixes of
//    1000-4000 tokens, 45 / 50, FP8 42 / 45, 3 x 100 34 / 43), MXFP4 up to seven (8 x 64 48 /
//    59, 8 x 104 67 / 78, 8 x 128, eight, 76 / 80).
// `uneven` is a guess: the plan sees no lengths, and takes the pool for what the requests
// hold.  Walks over whole prefixes that are all alike lose by it (8 x 48 rows behind 3000
// tokens 58 / 37, MXFP4 58 / 45, 8 x 100 92 / 61), and so do short ones in a pool ten times
// what they need (8 x 48 behind 300 17 / 13, MXFP4 8 x 100 22 / 17, 8 x 64 14 / 16); a
// caller who knows them sets the tile.
uint64_t row_tile_cols(uint64_t tiles, uint64_t cus, bool mx, bool uneven) {
  if (4 * tiles <= (mx ? 6 : 5) * cus) return 16;
  return 4 * tiles <= (uneven ? (mx ? 28 : 14) : 9) * cus ? 32 : 0;
}

// Columns of the long tiles: 128 where they are two per CU, and for MXFP4, whose rows are
// widened once per tile, wherever 64-column ones (a grid of `grid64`) are more than one (8 x
// 80 rows under windows of 1024 30.5 / 37.6, 4 x 300 48 / 58).
uint64_t long_tile_cols(uint64_t tiles128, uint64_t grid64, uint64_t cus, bool mx) {
  return tiles128 >= 2 * cus || (mx && grid64 > cus) ? 128 : 64;
}

// Wave groups of the long tiles, which split a walk: of `tiles` full ones of 128 columns two
// where walks over the whole prefix differ, while two workgroups per CU hold all (4 x 512
// rows behind 2048-16384 tokens 330 us in one group, 253 in two, FP8 338 / 264, MXFP4 404 /
// 290, but under windows of 4096, all alike, 134 / 144, and 8 x 512 277 / 302; with a window
// past the contexts up to one and a half per CU: 4 x 512 of 600-2500 tokens, two per CU, 54 /
// 59), or where one per CU holds them (8 x 128 MXFP4 rows under windows of 1024 37 / 33, 4 x
// 300 48 / 59).  Of 64 columns four where a grid of one per CU holds them, or hardly more
// for uneven walks (8 x 64 rows, whole prefixes of 1000-4000 tokens, 50 in four, 58 in two;
// FP8 45 / 53), else two (8 x 80 rows under windows of 1024 28 / 39).
uint32_t long_groups(uint64_t tile_cols, uint64_t tiles, uint64_t grid, uint64_t cus, uint64_t window,
                     bool uneven) {
  if (tile_cols == 128)
    return tiles <= cus || 2 * tiles <= (window == 0 ? 5 : uneven ? 3 : 0) * cus ? 2 : 1;
  return grid <= cus || (uneven && 2 * grid <= 3 * cus) ? 4 : 2;
}

// Waves of a row-tile workgroup: four where its walks do not wait for the CU, whose two to
// four workgroups then begin and end beside each other's streams (128 single tokens under
// windows of 128 26.2 -> 18.7 us, FP8 21.7 -> 15.6, MXFP4 21.4 -> 10.4; of 4096 337 / 335,
// 194 / 189, 139 / 148); but with hardly more workgroups than CUs a long walk has eight (8
// chunks of 1-32 rows, MXFP4, the whole prefixes of 300-5000 tokens: 31 / 41).  Four as well
// for walks of few steps (`walk` tokens at most, as a rule; 8 x 10 rows under windows of 48
// 5.4 / 5.1, but 8 single tokens under windows of 200 5.5 / 5.9).
uint32_t row_waves(uint64_t grid, uint64_t cus, uint64_t window, uint64_t walk) {
  if (walk <= 112) return 4;
  return grid >= 2 * cus || (grid > cus && window > 0 && window <= 2048) ? 4 : 8;
}

// Workgroups per (tile, kv-head) of a row-tile command of `grid` unsplit ones (`least_grid` at
// least), whose walks hold about `tokens` tokens: at most one per CU, and each with work for
// its join (2 us): the more CUs stream already, the less another one adds.  (8 x 8 rows, 128
// tiles of a grid of 192, over whole prefixes of 2500-5000 tokens 55 -> 37 us, FP8 26.6 ->
// 20.5.)  Walks that may differ (`uneven`) are cut in two up to four tiles on five CUs (24 single
// tokens of 100-8000, 8 kv-heads, 97 -> 67 us, FP8 64 -> 45, MXFP4 43 -> 32; all of 8000 131 ->
// 141, 80 -> 87, 60 -> 67; 32 of 100-8000 would take 105 -> 99, 68 -> 66, 54 -> 55, of 3000 64
// both, 38 both, 27 -> 34).
int row_splits(uint64_t grid, uint64_t least_grid, uint64_t tokens, bool uneven, uint64_t cus, bool mx) {
  const uint64_t blocks = (tokens + 15) / 16;
  uint64_t most = cus / std::max<uint64_t>(tokens >= kLongWalk ? least_grid : grid, 1);
  if (uneven && most == 1 && 5 * grid <= 4 * cus) most = 2;
  most = std::min<uint64_t>(most, kMaxSplits);
  // 16-row blocks per wave
  const uint64_t least = std::max<uint64_t>(1, grid * (mx ? 8 : 16) / cus);
  return (int)std::max<uint64_t>(1, std::min(most, blocks / (least * 8)));
}

// Workgroups that are launched for `workgroups` with work: of MXFP4 row tiles over an even
// number of kv-heads whole groups of 16, see WindowArgs::pair_heads.
bool pairs_heads(bool mx_rows, uint64_t hkv) { return mx_rows && hkv % 2 == 0; }
uint64_t launched(uint64_t workgroups, bool mx_rows, uint64_t hkv) {
  return pairs_heads(mx_rows, hkv) ? (workgroups + 15) / 16 * 16 : workgroups;
}

template <Kv KV>
auto kernel_of(const loom_window_attention_plan &p, uint64_t bytes) {
  if (p.info.algorithm != LOOM_PAGED_PREFILL_LONG_TILE) {
    const bool past = p.once && bytes >= kPastCaches;
    if (p.info.block_threads == 256)
      return p.info.tile_cols == 32 ? window_rows_kernel<KV, 2, 4, false>
             : past                 ? window_rows_kernel<KV, 1, 4, true>
                                    : window_rows_kernel<KV, 1, 4, false>;
    return p.info.tile_cols == 32 ? window_rows_kernel<KV, 2, 8, false>
           : past                 ? window_rows_kernel<KV, 1, 8, true>
                                  : window_rows_kernel<KV, 1, 8, false>;
  }
  if (p.info.tile_cols == 128)
    return p.groups == 2 ? window_long_kernel<KV, 8, 4> : window_long_kernel<KV, 4, 4>;
  if constexpr (KV != kMx4)  // (of 64 columns MXFP4 takes four groups always)
    if (p.groups == 2) return window_long_kernel<KV, 4, 2>;
  return window_long_kernel<KV, 8, 2>;
}

loom_status_t make_plan(const loom::DeviceInfo &dev, const loom_window_attention_spec_t *spec,
                        uint32_t flags, loom_window_attention_plan_t **out, loom_error_t *err) {
  loom_window_attention_spec_t s;
  const loom_status_t rc =
      loom_window_attention_spec_new(&spec->paged, spec->rows, spec->explicit_rows, spec->window,
                                     spec->sinks, &s, err);
  if (rc) return rc;
  const float scale = s.paged.softmax_scale;
  if (!(scale > 0.0f) || !std::isfinite(scale * kLog2e))
    return fail(err, LOOM_PLAN_INVALID_OPTION, "softmax_scale");
  const uint64_t hq = s.paged.num_query_heads, hkv = s.paged.num_kv_heads, group = hq / hkv;
  const uint64_t batch = s.paged.batch_size;
  if (hkv > kMaxHeads) return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "window heads", hkv);
  if (s.rows > (uint64_t)INT32_MAX / hq || batch >= (uint64_t)INT32_MAX)
    return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "window rows", s.rows);
  const uint64_t cols = s.rows * group, cus = (uint64_t)dev.cus;
  // columns of a request, as a rule
  const uint64_t group_cols = s.explicit_rows ? (cols + batch - 1) / batch : group;
  auto tiles_of = [&](uint64_t tc) {
    return s.explicit_rows ? std::min(cols, (cols + (tc - 1) * batch) / tc)
                           : batch * ((group + tc - 1) / tc);
  };
  const bool mx = s.paged.kv_dtype == LOOM_KV_DTYPE_MXFP4;
  // tokens of a request, as a rule (of a pool as large as what it holds), and whether long
  // walks differ with them
  const uint64_t context =
      s.paged.max_num_pages * (s.paged.page_size ? s.paged.page_size : loom::kPageSize) / batch;
  const bool uneven =
      s.explicit_rows && batch > 1 && context >= 1024 && (s.window == 0 || s.window >= context);
  const uint64_t row_cols =
      row_tile_cols((s.explicit_rows ? cols / 16 + (batch + 1) / 2 : tiles_of(16)) * hkv, cus, mx, uneven);
  const bool long_tile =
      flags & LOOM_PLAN_PREFILL_TILE_LONG ||
      (!(flags & LOOM_PLAN_PREFILL_TILE_16) && s.explicit_rows && row_cols == 0);
  const uint64_t tc = long_tile ? long_tile_cols(cols / 128 * hkv, tiles_of(64) * hkv, cus, mx)
                      : row_cols == 16 || group_cols <= 16 ? 16
                                                           : 32;
  const uint64_t tiles = tiles_of(tc), grid = tiles * hkv;
  const uint64_t seen = s.window && s.window < context ? s.window + s.rows / batch : context;
  const uint64_t walk = std::min(context, seen + std::min(s.sinks, context));
  const uint32_t groups = long_tile ? long_groups(tc, cols * hkv / 128, grid, cus, s.window, uneven) : 1;
  const uint32_t waves = !long_tile ? row_waves(grid, cus, s.window, walk) : (uint32_t)tc / 32 * groups;
  if (launched(grid, mx && !long_tile, hkv) * (waves * 64) >= (1ull << 32))
    return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "window rows", s.rows);
  auto *p = new loom_window_attention_plan;
  p->info.spec = s;
  p->info.algorithm = long_tile ? LOOM_PAGED_PREFILL_LONG_TILE : LOOM_PAGED_PREFILL_ROW_TILE;
  p->info.tile_cols = (uint32_t)tc;
  p->info.row_tiles = tiles;
  p->info.grid_blocks = grid;
  p->info.block_threads = waves * 64;
  p->info.flags = flags;
  p->cus = dev.cus;
  p->groups = groups;
  p->once = group_cols <= tc;
  p->least_tiles = s.explicit_rows ? std::min(tiles, std::max(batch, (cols + tc - 1) / tc)) : tiles;
  *out = p;
  return loom::ok(err);
}

}  // namespace

extern "C" {

loom_status_t loom_decode_provider_plan_window_paged_batch(
    const loom_decode_provider_t *provider, const loom_window_attention_spec_t *spec, uint32_t flags,
    loom_window_attention_plan_t **out, loom_error_t *err) {
  if (!provider || !spec || !out) return fail(err, LOOM_NULL_ARGUMENT, "provider");
  if (flags & ~LOOM_PLAN_PAGE_INDICES_CAPACITY)
    return fail(err, LOOM_PLAN_INVALID_OPTION, "flags", flags);
  if (spec->explicit_rows) return fail(err, LOOM_PLAN_INVALID_OPTION, "explicit_rows", 1);
  return make_plan(provider->dev, spec, flags, out, err);
}

loom_status_t loom_prefill_provider_plan_window_paged(const loom_prefill_provider_t *provider,
                                                      const loom_window_attention_spec_t *spec,
                                                      uint32_t flags,
                                                      loom_window_attention_plan_t **out,
                                                      loom_error_t *err) {
  if (!provider || !spec || !out) return fail(err, LOOM_NULL_ARGUMENT, "provider");
  constexpr uint32_t kTiles = LOOM_PLAN_PREFILL_TILE_16 | LOOM_PLAN_PREFILL_TILE_LONG;
  if ((flags & ~(LOOM_PLAN_PAGE_INDICES_CAPACITY | kTiles)) || (flags & kTiles) == kTiles)
    return fail(err, LOOM_PLAN_INVALID_OPTION, "flags", flags);
  if (!spec->explicit_rows) return fail(err, LOOM_PLAN_INVALID_OPTION, "explicit_rows", 0);
  return make_plan(provider->dev, spec, flags, out, err);
}

void loom_window_attention_plan_free(loom_window_attention_plan_t *p) { delete p; }

void loom_window_attention_plan_get_info(const loom_window_attention_plan_t *p,
                                         loom_window_attention_plan_info_t *info) {
  if (p && info) *info = p->info;
}

loom_status_t loom_window_attention_enqueue(const loom_window_attention_plan_t *plan,
                                            loom_command_scope_t *scope,
                                            const loom_window_attention_args_t *args,
                                            loom_error_t *err) {
  if (!plan || !scope || !args) return fail(err, LOOM_NULL_ARGUMENT, "plan");
  const loom_window_attention_spec_t &s = plan->info.spec;
  const loom_paged_decode_spec_t &pg = s.paged;
  const bool fp8 = pg.kv_dtype == LOOM_KV_DTYPE_FP8_E4M3, mx = pg.kv_dtype == LOOM_KV_DTYPE_MXFP4;
  const loom_dtype_t kv_t = fp8 || mx ? LOOM_DTYPE_U8 : LOOM_DTYPE_BF16;
  const uint64_t page_rows = pg.page_size ? pg.page_size : loom::kPageSize;
  const uint64_t head_rows = pg.max_num_pages * page_rows * pg.num_kv_heads;
  const uint64_t kvn = head_rows * (mx ? LOOM_MXFP4_ROW_BYTES : loom::kHeadDim);
  const uint64_t qn = s.rows * pg.num_query_heads * loom::kHeadDim;
  struct Operand {
    loom::OperandSpec spec;
    loom_handle_t handle;
    uint64_t want;
    bool aligned;  // 4-byte boundary
  };
  // the operands of every form, then those of some
  const Operand all[12] = {
      {{"Q", LOOM_DTYPE_BF16, false}, args->query, qn, true},
      {{"K_pages", kv_t, false}, args->key_pages, kvn, true},
      {{"V_pages", kv_t, false}, args->value_pages, kvn, true},
      {{"page_indptr", LOOM_DTYPE_I32, false}, args->page_indptr, pg.batch_size + 1, false},
      {{"page_indices", LOOM_DTYPE_I32, false}, args->page_indices, 0, false},
      {{"last_page_len", LOOM_DTYPE_I32, false}, args->last_page_len, pg.batch_size, false},
      {{"O", LOOM_DTYPE_BF16, true}, args->output, qn, true},
      {{"LSE", LOOM_DTYPE_F32, true}, args->lse, s.rows * pg.num_query_heads, true},
      {{"qo_indptr", LOOM_DTYPE_I32, false}, args->qo_indptr, pg.batch_size + 1, false},
      {{"kv_scales", LOOM_DTYPE_F32, false}, args->kv_scales, 2, true},
      {{"K_scales", LOOM_DTYPE_U8, false}, args->key_scales, head_rows * LOOM_MXFP4_ROW_SCALES, true},
      {{"V_scales", LOOM_DTYPE_U8, false}, args->value_scales, head_rows * LOOM_MXFP4_ROW_SCALES, true}};
  int which[12], n = 0;
  for (int i = 0; i < 12; ++i)
    if (i < 8 || (i == 8 && s.explicit_rows) || (i == 9 && fp8) || (i >= 10 && mx)) which[n++] = i;
  loom::OperandSpec ops[12];
  loom_handle_t hs[12];
  for (int j = 0; j < n; ++j) {
    ops[j] = all[which[j]].spec;
    hs[j] = all[which[j]].handle;
  }
  const loom::Lease *found[12], *l[12] = {};
  loom_status_t rc = loom::resolve_command(scope, hs, ops, n, found, err);
  if (rc) return rc;
  for (int j = 0; j < n; ++j) {
    const Operand &o = all[which[j]];
    l[which[j]] = found[j];
    if (which[j] == 4) {
      if (found[j]->numel < pg.batch_size)
        return fail(err, LOOM_ENQ_PAGE_INDICES_TOO_SHORT, o.spec.name, pg.batch_size, found[j]->numel);
      if (found[j]->numel > (uint64_t)INT32_MAX / page_rows)
        return fail(err, LOOM_ENQ_PAGE_INDICES_TOO_LONG, o.spec.name,
                    (int64_t)((uint64_t)INT32_MAX / page_rows), found[j]->numel);
    } else if (found[j]->numel != o.want) {
      return fail(err, LOOM_ENQ_LENGTH_MISMATCH, o.spec.name, o.want, found[j]->numel);
    }
    if (o.aligned && found[j]->ptr % 4 != 0)
      return fail(err, LOOM_ENQ_MISALIGNED_BUFFER, o.spec.name, (int64_t)found[j]->ptr, 4);
  }
  WindowArgs a{};
  a.q = (const uint16_t *)l[0]->ptr;
  a.k = (const uint16_t *)l[1]->ptr;
  a.v = (const uint16_t *)l[2]->ptr;
  a.indptr = (const int32_t *)l[3]->ptr;
  a.indices = (const int32_t *)l[4]->ptr;
  a.last = (const int32_t *)l[5]->ptr;
  a.out = (uint16_t *)l[6]->ptr;
  a.lse = (float *)l[7]->ptr;
  a.qo = s.explicit_rows ? (const int32_t *)l[8]->ptr : nullptr;
  a.kv_scales = fp8 ? (const float *)l[9]->ptr : nullptr;
  a.k_mx = mx ? (const uint8_t *)l[10]->ptr : nullptr;
  a.v_mx = mx ? (const uint8_t *)l[11]->ptr : nullptr;
  a.batch = (int32_t)pg.batch_size;
  a.nnz = (int32_t)s.rows;
  a.hq = (int32_t)pg.num_query_heads;
  a.hkv = (int32_t)pg.num_kv_heads;
  a.group = a.hq / a.hkv;
  a.pool = (int64_t)pg.max_num_pages;
  a.n_indices = (int64_t)l[4]->numel;
  a.scale_log2 = pg.softmax_scale * kLog2e;
  a.indices_capacity = (plan->info.flags & LOOM_PLAN_PAGE_INDICES_CAPACITY) ? 1 : 0;
  a.page_rows = (int32_t)page_rows;
  a.blocks_lg = page_rows == 64 ? 2 : page_rows == 32 ? 1 : 0;
  const int row = mx ? 64 : fp8 ? 128 : 256;
  const bool hnd = pg.kv_layout == LOOM_KV_LAYOUT_HND;
  a.head_bytes = hnd ? a.page_rows * row : row;
  a.row_bytes = hnd ? row : a.hkv * row;
  a.window = s.window == 0 || s.window > (uint64_t)INT32_MAX ? INT32_MAX : (int32_t)s.window;
  a.sinks = (int32_t)std::min<uint64_t>(s.sinks, INT32_MAX - 64);
  a.row_tiles = (int32_t)plan->info.row_tiles;
  a.head_tiles = (a.group + (int32_t)plan->info.tile_cols - 1) / (int32_t)plan->info.tile_cols;
  // (exact while column * group < 2^32)
  if (a.group > 1 && s.rows * (uint64_t)a.group * (uint64_t)a.group < (1ull << 32))
    a.group_inv = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
  // the tokens that a request's rows see, at most: its window, or the average context
  const uint64_t context = (uint64_t)a.n_indices * page_rows / pg.batch_size;
  const uint64_t tokens =
      std::min<uint64_t>((uint64_t)a.window + (uint64_t)a.sinks + s.rows / pg.batch_size, context);
  const uint64_t grid = plan->info.grid_blocks;
  const bool long_tile = plan->info.algorithm == LOOM_PAGED_PREFILL_LONG_TILE;
  a.splits = long_tile ? 1
                       : row_splits(grid, plan->least_tiles * pg.num_kv_heads, tokens,
                                    pg.batch_size > 1 && (uint64_t)a.window >= context,
                                    (uint64_t)plan->cus, mx);
  if (a.splits > 1) {
    a.arrived = scope->queue->joins;
    a.states = (float *)loom::queue_shares(
        scope, (uint64_t)a.splits * grid * plan->info.tile_cols * kStash * 4);
    if (!a.states || !a.arrived || grid > loom::kMx4Joins) a.splits = 1;
  }
  const uint64_t parts = grid * a.splits, workgroups = launched(parts, mx && !long_tile, pg.num_kv_heads);
  a.pair_heads = pairs_heads(mx && !long_tile, pg.num_kv_heads) ? (int32_t)parts : 0;
  const dim3 blocks((unsigned)workgroups), threads(plan->info.block_threads);
  hipStream_t stream = scope->queue->stream;
  a.sorted = workgroups > (uint64_t)plan->cus;
  const uint64_t bytes = tokens * pg.batch_size * pg.num_kv_heads * 2 * (mx ? 68 : (uint64_t)row);
  const auto kernel = mx    ? kernel_of<kMx4>(*plan, bytes)
                      : fp8 ? kernel_of<kFp8>(*plan, bytes)
                            : kernel_of<kBf16>(*plan, bytes);
  hipLaunchKernelGGL(kernel, blocks, threads, 0, stream, a);
  return loom::record_launch(scope, hipGetLastError(), err);
}

}  // extern "C"
