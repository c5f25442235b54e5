// Paged decode attention over MXFP4 pages for gfx950 (MI355X), D128, 16-64 rows per
// page, NHD or HND (no reference counterpart).
//
// Per query head: S = q.k / sqrt(128), O = softmax(S).V, LSE in log2, over the values
// code * 2^(scale - 127) of the request's tokens.  A token costs 136 bytes per kv-head
// where BF16 pages cost 512, so the arithmetic per byte is four times as dense: a block
// of 32 tokens and one kv-head takes a wave about 375 ns of instructions (VALU busy half
// of the balanced kernel's time).  The step is built for few of them:
//   * 32 tokens at a time, codes and scales loaded straight into LDS, nothing held in
//     registers in flight.  K is read as the MFMA fragment wants it: lane (col, quad)
//     takes the 16 bytes of dims 32 quad + [0, 32) of a row, one scale block, and
//     v_cvt_scalef32_pk_bf16_fp4 widens two codes and applies the block's scale in one
//     instruction, exactly.  (v_mfma_scale_f32_16x16x128_f8f6f4 takes FP4 itself, but
//     sums its 128 products with errors up to 2^-12 of the largest, which LSE does not
//     bear.)
//   * V codes come as 8 dims from 8 col on of rows 4 j + quad.  With up to 4 query heads
//     in a tile the widened pairs are the V^T fragment as they are: an even and an odd
//     dim in neighbouring places of the contraction, where P^T has its weight for the one
//     and a zero for the other, in columns of their own.  With 5 to 8, one byte permute
//     per two tokens turns the pairs into a fragment of one dim.
//   * The running bound of the scores is set kLazy above a new maximum and moves only
//     when a score passes it: the common step has no reduction across lanes and no
//     rescale.  No weight is above 1, so the FP32 sum of weights times V, divided at
//     the end, stays in range for V below 2^128 over the request's tokens; larger V
//     (up to 6 * 2^125) may overflow it although their mean does not.
//   * P keeps 16 bits, a BF16 high part and a BF16 residual, in one MFMA: a tile is at
//     most 8 query heads; columns 0-7 take the high parts, 8-15 the residuals, and the
//     two columns' O are added at the end.
//
// Two decompositions, both independent of the page table's contents:
//   balanced  the 32-token blocks of all valid requests form one virtual list, cut
//             into `teams` equal ranges; a team is one wave per (kv-heads, tile), all
//             walking the same blocks.  Requests that cross a range leave states, which
//             a second kernel merges.  Bound by memory: 64 requests of 512-8192 tokens
//             (32 / 8 heads, 254 MB) 52.3 us, 47.6 without the merge (5.3 TB/s; a large
//             copy reaches 5.1); 8 of 32768 (64 / 8, 286 MB) 56 us.
//   direct    one workgroup per (request, kv-heads, tile[, split]): its waves take the
//             blocks in turn and merge in LDS, the last split of a request the splits.
//             One launch.  Bound by latency: one request of 200 tokens 4.9 us, 16 of
//             256-1536 11.3 (32 / 8 heads), 5 of 1-5003 (28 / 4) 9.5.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attn_device.hpp"
#include "mx4_decode.hpp"

using loom::fail;
using loom::kMx4StateStride;
using loom::Mx4DecodeArgs;
using namespace loom_dev;

namespace {

constexpr int kBlock = 32;  // tokens per step
constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kMaxTile = 8;  // query heads of a tile
// Entries of the balanced kernel's prefix table in LDS; a batch beyond it has one
// entry per 2, 4, ... requests.
constexpr int kPrefix = 512;
constexpr int kMaxBatch = 65536;
// log2 of how far the bound of the scores lies above the maximum that set it.  Weights
// are 2^-8 and less then, which costs no precision in FP32 or in their two BF16 parts.
constexpr float kLazy = 8.0f;
// Normalizer written into a state whose pages failed the guard.
constexpr float kPoisonNormalizer = -1.0f;
// Fewest blocks of a team (a state costs its write and its merge).
constexpr int kMinTeamBlocks = 2;
// Balanced kernel: blocks in flight per wave, and waves per four CUs; one wave per SIMD.
// Three in flight, or more waves, were slower: the pages' order in memory sets the rate,
// and streams that many in number or that far ahead of each other spoil it.
constexpr int kDepth = 2;
constexpr int kWavesPer4Cu = 16;

// decode.rs:233-246: indptr[B] is the page_indices length (at most that length for
// capacity plans).
__device__ __forceinline__ bool batch_ok(const Mx4DecodeArgs &a, int32_t ip0, int32_t ipB) {
  return ip0 == 0 && ipB >= 0 &&
         (a.indices_capacity ? (int64_t)ipB <= a.n_indices : (int64_t)ipB == a.n_indices);
}
// Tokens of a request (0 if it fails the per-request guard of decode.rs:430-478).
__device__ __forceinline__ int64_t request_tokens(const Mx4DecodeArgs &a, int32_t st, int32_t en,
                                                  int32_t tl, int32_t ipB) {
  const bool valid = st >= 0 && en > st && en <= ipB && tl >= 1 && tl <= a.page_rows;
  return valid ? ((int64_t)en - st - 1) * a.page_rows + tl : 0;
}

// floor(n / d) for 0 <= n < 2^53, d > 0: a double-precision estimate, corrected.
__device__ __forceinline__ int64_t floor_div(int64_t n, int64_t d) {
  int64_t q = (int64_t)((double)n / (double)d);
  while (q * d > n) --q;
  while ((q + 1) * d <= n) ++q;
  return q;
}
// The virtual list of `total` blocks in equal ranges: each team in use has `each`
// blocks, the first `more` of them one more.  At most the planned teams are in use, and
// (unless that leaves one) each has at least kMinTeamBlocks.
struct Ranges {
  int64_t each, more;
  int teams;
  __device__ __forceinline__ Ranges(int64_t total, int planned) {
    teams = (int)max<int64_t>(1, min<int64_t>(planned, total / kMinTeamBlocks));
    if (total < INT32_MAX)
      each = (uint32_t)total / (uint32_t)teams;
    else
      each = floor_div(total, teams);
    more = total - each * teams;
  }
  __device__ __forceinline__ int64_t start(int64_t t) const { return t * each + min(t, more); }
  __device__ __forceinline__ int64_t team_of(int64_t v) const {
    const int64_t longer = more * (each + 1);
    return v < longer ? floor_div(v, each + 1) : more + floor_div(v - longer, each);
  }
};

// One 32-token block as a wave stages it in LDS: K and V codes of one or two kv-heads
// and the rows' scale words.  Loads go straight to LDS (nothing is held in registers
// in flight), lane l's 16 bytes to 16 l, so the order within a slot is chosen by the
// addresses the lanes load from.  Two arrangements:
//   kSplit  per head 64-byte rows: HND pages, and single heads.  Lane l takes piece
//           (l & 3) ^ (l >> 4) of row l >> 2 of a half (16 rows).
//   kPair   128-byte rows of two neighbouring heads: NHD pages, whose rows hold them side
//           by side: 64-byte loads take half a cache line each, and every line twice
//           (8 requests of 32768 tokens at 4.5 TB/s, so 5.7).  Lane l takes piece
//           (l & 7) ^ pair_swizzle(row) of row l >> 3 of eight rows.
// Either way the reads below, which take one 16-byte piece of all rows of a half or 64
// bytes of every fourth row, meet each LDS bank once.  Scale word c of a half belongs to
// its row token_of(c).
enum Arrangement : int { kSplit = 0, kPair = 1 };
constexpr int kHalfBytes = 16 * 64;
constexpr int kHeadBytes = 2 * kHalfBytes;  // K (or V) codes of one head's block
// Row of a half that row c of the MFMA tile S = K.Q^T stands for: S leaves lane (col,
// quad) rows 4 quad + i, which are tokens 4 i + quad, and the V reads of the four quads
// then lie in four neighbouring rows.
__host__ __device__ constexpr int token_of(int c) { return 4 * (c & 3) + (c >> 2); }
__host__ __device__ constexpr int pair_swizzle(int row) { return (row & 2) * 2 + (row >> 2); }

// Byte offsets in a slot: K of all heads, V of all heads, then the scales (per half and
// head 16 words).
template <int NH>
struct Slot {
  static constexpr int v = NH * kHeadBytes, ks = 2 * NH * kHeadBytes, vs = ks + NH * 128,
                       bytes = vs + NH * 128;
  // scale words of (head, half): pages of 16 rows load a half of all heads at a time,
  // others both halves of a head
  template <bool P16>
  static __host__ __device__ constexpr int scales(int head, int half) {
    return P16 ? half * NH * 64 + head * 64 : head * 128 + half * 64;
  }
};

// Where a block lies: the cache row (of 64 code bytes; plans hold below 2^32 of them) and
// the scale row (of 4 bytes) of its first token and the wave's first kv-head, for pages of
// 16 rows those of its second half too; and its valid rows (0: none, nothing is read).
// All wave-uniform: found per lane, 64 blocks at a time, since the 64-bit products of
// page, head and row for every block took a fifth of a walk's instructions.
struct Place {
  uint32_t c0, s0, c1, s1;
  int rows;
};
// The two rows of row `row` of `page`, head kvh.
__device__ __forceinline__ void cache_rows(const Mx4DecodeArgs &a, int page, int row, int kvh,
                                           uint32_t &c, uint32_t &s) {
  const uint32_t pg = (uint32_t)page;
  s = (pg * (uint32_t)a.hkv + (uint32_t)kvh) * (uint32_t)a.page_rows + (uint32_t)row;
  c = a.row_bytes == 64 ? s  // HND (and one kv-head): as the scales lie
                        : (pg * (uint32_t)a.page_rows + (uint32_t)row) * (uint32_t)a.hkv + (uint32_t)kvh;
}

// row << N of a wave-uniform row, in scalar registers (the compiler fuses the shift into
// a vector multiply-add of the address otherwise).
template <int N>
__device__ __forceinline__ uint64_t row_bytes(uint32_t row) {
  uint64_t r;
  asm("s_lshl_b64 %0, %1, %2" : "=s"(r) : "s"((uint64_t)row), "n"(N) : "scc");
  return r;
}

// Vector memory instructions that load_block issues, always.
template <bool P16, int NH>
constexpr int kBlockLoads = 4 * NH + (P16 ? 4 : 2);
// Issues the loads of a block of NH neighbouring kv-heads into LDS at byte address
// `slot`.  Rows past the valid ones arrive as zeros and move no bytes.
// NT: nontemporal loads of the codes.
template <bool P16, int NH, int ARR, bool NT>
__device__ __forceinline__ void load_block(const Mx4DecodeArgs &a, const Place &p, uint32_t slot,
                                           int lane) {
  using S = Slot<NH>;
  auto rsrc = [](const uint8_t *base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, bytes, 0x00020000);
  };
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // rows [0, n) of this half (of the whole block where it lies in one page) exist
    const int n = !P16 ? p.rows : h == 0 ? min(p.rows, 16) : max(p.rows - 16, 0);
    const uint32_t c = P16 && h == 1 ? p.c1 : p.c0;
    const int skip = P16 ? 0 : 16 * h * a.row_bytes;
    if constexpr (ARR == kPair) {
      const int bytes = max((n - 1) * a.row_bytes + 128, 0);  // (rows of 128 bytes and more)
      const uint64_t at = row_bytes<6>(c);
      const __amdgpu_buffer_rsrc_t rk = rsrc(a.k + at, bytes), rv = rsrc(a.v + at, bytes);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int row = 8 * t + (lane >> 3);
        const int off = row * a.row_bytes + (((lane & 7) ^ pair_swizzle(row)) << 4) + skip;
        lds_load16_at<NT>(rk, slot + (2 * h + t) * 1024, off);
        lds_load16_at<NT>(rv, slot + S::v + (2 * h + t) * 1024, off);
      }
    } else {
      const int bytes = max((n - 1) * a.row_bytes + 64, 0);
      const int off = (lane >> 2) * a.row_bytes + (((lane & 3) ^ (lane >> 4)) << 4) + skip;
#pragma unroll
      for (int g = 0; g < NH; ++g) {
        const uint64_t head = row_bytes<6>(c + (uint32_t)g * ((uint32_t)a.head_bytes >> 6));
        lds_load16_at<NT>(rsrc(a.k + head, bytes), slot + g * kHeadBytes + h * kHalfBytes, off);
        lds_load16_at<NT>(rsrc(a.v + head, bytes), slot + S::v + g * kHeadBytes + h * kHalfBytes, off);
      }
    }
    // scale words: one lane each, 16 rows (P16) or 32 of every head
    if (P16 || h == 0) {
      constexpr int kRows = P16 ? 16 : 32;
      if (lane < kRows * NH) {
        const int row = token_of(lane & 15) + (P16 ? 0 : lane & 16);
        const uint64_t sc = row_bytes<2>(P16 && h == 1 ? p.s1 : p.s0);
        const int off = row < n ? (lane / kRows) * a.page_rows * 4 + row * 4 : INT32_MAX;
        const int bytes = ((NH - 1) * a.page_rows + n) * 4;
        lds_load4_at(rsrc(a.k_mx + sc, bytes), slot + S::ks + h * NH * 64, off);
        lds_load4_at(rsrc(a.v_mx + sc, bytes), slot + S::vs + h * NH * 64, off);
      }
    }
  }
}
// Until at most N of this wave's vector memory operations are outstanding; LDS reads
// stay behind it.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Until this wave's LDS reads have returned: before loads into a slot that it read.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// One wave's decode of a request for one kv-head and a tile of its query heads: the
// online-softmax states.
// Columns 0-7 of the tiles take P's high parts, 8-15 its residuals.  Tiles of 5 to 8
// heads have a head per column, and acc[e][i] holds O[column col][dim 32 quad + 8 i + e],
// unnormalized.  Tiles of up to 4 (QUADS) have column c & 3, and columns with bit 2 set
// take the odd dims, the others the even ones: acc[e][i] holds dim 32 quad + 8 i + 2 e,
// or + 1.
template <bool QUADS>
struct HeadState {
  float m_run, l_run;  // bound of the scores (log2); sum of this lane's weights
  static constexpr int kAcc = QUADS ? 4 : 8;
  static constexpr int kHeadMask = QUADS ? 3 : 7;  // the head of column c: c & kHeadMask
  f32x4 acc[kAcc];
  u32x4 q[4];  // MFMA c contracts dims 32 quad + 8 c + [0, 8)

  // From the lowest finite maximum, tokens that score -inf weigh nothing.
  __device__ __forceinline__ void reset() {
    m_run = -FLT_MAX;
    l_run = 0.0f;
#pragma unroll
    for (int e = 0; e < kAcc; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void load_q(const uint16_t *row, bool mine, int quad) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      q[c] = mine ? load16(row + quad * 32 + c * 8) : u32x4{0, 0, 0, 0};
  }
  // Ends load_q's loads here: left in flight, they would make every block's first
  // MFMA wait for all loads before it, the pipeline's next blocks among them.
  __device__ __forceinline__ void settle_q() {
#pragma unroll
    for (int c = 0; c < 4; ++c) asm volatile("" : "+v"(q[c]));
  }
  __device__ __forceinline__ float normalizer() const { return quad_sum(l_run); }
  // The 32 dims 32 quad + 8 i + e of this lane's column (a head of the tile), high parts
  // and residuals (lane col ^ 8 of the 16) added.
  __device__ __forceinline__ void columns(f32x4 (&o)[8]) const {
#pragma unroll
    for (int e = 0; e < kAcc; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = acc[e][i] + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
                                        0, (int)__float_as_uint(acc[e][i]), 0x128, 0xf, 0xf, false));
        if constexpr (QUADS) {  // odd dims from lane col + 4
          o[2 * e][i] = x;
          o[2 * e + 1][i] = __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
              0, (int)__float_as_uint(x), 0x12C, 0xf, 0xf, false));
        } else {
          o[e][i] = x;
        }
      }
  }
  // A column of columns() as O and, by quad 0, LSE.
  __device__ __forceinline__ void store(const f32x4 (&x)[8], uint16_t *o, float *lse, float l,
                                        int quad) const {
    const float inv = 1.0f / l;  // (its rounding and the product's are 2^-23 of O)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = bf16x2_pack(x[2 * e][i] * inv, x[2 * e + 1][i] * inv);
      *reinterpret_cast<u32x4 *>(o + quad * 32 + i * 8) = w;
    }
    if (quad == 0) *lse = m_run + __log2f(l);
  }
  // The same column unnormalized.
  static __device__ __forceinline__ void stash(const f32x4 (&x)[8], float *dst, int quad) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float *o = dst + quad * 32 + i * 8;
      *reinterpret_cast<f32x4 *>(o) = f32x4{x[0][i], x[1][i], x[2][i], x[3][i]};
      *reinterpret_cast<f32x4 *>(o + 4) = f32x4{x[4][i], x[5][i], x[6][i], x[7][i]};
    }
  }

  // P^T as B fragments, from a lane's weights p[h][i] of tokens 16 h + 4 i + quad.
  // One fragment: k = 8 quad + 4 h + i is that token.  QUADS, one per half h: k = 8 quad +
  // 2 i is the token for even-dim columns and nothing for the others, + 1 the reverse.
  __device__ __forceinline__ void pack_p(const float (&p)[2][4], int col, bf16x8 (&b)[2]) const {
    const uint32_t taken = col < 8 ? 0u : 0xffff0000u;
    uint32_t x[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[h][i] = __float_as_uint(p[h][i] - __uint_as_float(__float_as_uint(p[h][i]) & taken));
    if constexpr (QUADS) {
      // bytes 3 and 2 of x to the high or the low half, zeros (byte 12: 0) to the other
      const uint32_t sel = col & 4 ? 0x03020c0cu : 0x0c0c0302u;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        b[h] = as_bf16x8(__builtin_amdgcn_perm(0u, x[h][0], sel), __builtin_amdgcn_perm(0u, x[h][1], sel),
                         __builtin_amdgcn_perm(0u, x[h][2], sel), __builtin_amdgcn_perm(0u, x[h][3], sel));
    } else {
      b[0] = as_bf16x8(pack_hi16(x[0][0], x[0][1]), pack_hi16(x[0][2], x[0][3]),
                       pack_hi16(x[1][0], x[1][1]), pack_hi16(x[1][2], x[1][3]));
    }
  }
  // Dims 2 W and 2 W + 1 of O^T += V^T.P^T: V^T's row col is dims 8 col + 2 W and its
  // neighbour, and byte W of the lane's codes holds both.
  template <int W>
  __device__ __forceinline__ void add_pv(const uint32_t (&v)[2][4], const float (&vs)[2][4],
                                         const bf16x8 (&p)[2]) {
    uint32_t x[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[h][j] = __builtin_bit_cast(
            uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[h][j], vs[h][j], W));
    if constexpr (QUADS) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        acc[W] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            as_bf16x8(x[h][0], x[h][1], x[h][2], x[h][3]), p[h], acc[W], 0, 0, 0);
    } else {
      const bf16x8 even =
          as_bf16x8(pack_lo16(x[0][0], x[0][1]), pack_lo16(x[0][2], x[0][3]),
                    pack_lo16(x[1][0], x[1][1]), pack_lo16(x[1][2], x[1][3]));
      const bf16x8 odd =
          as_bf16x8(pack_hi16(x[0][0], x[0][1]), pack_hi16(x[0][2], x[0][3]),
                    pack_hi16(x[1][0], x[1][1]), pack_hi16(x[1][2], x[1][3]));
      acc[2 * W] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, p[0], acc[2 * W], 0, 0, 0);
      acc[2 * W + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, p[0], acc[2 * W + 1], 0, 0, 0);
    }
  }
};

// The block at `slot` (LDS) of which the first `rows` tokens are valid (wave-uniform).
template <bool P16, int NH, int ARR, bool QUADS>
__device__ __forceinline__ void process_block(HeadState<QUADS> (&st)[NH], const uint8_t *slot, int rows,
                                              int col, int quad, float scale_log2) {
  using S = Slot<NH>;
  f32x4 s[NH][2];
#pragma unroll
  for (int g = 0; g < NH; ++g)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // row token_of(col): its low two bits are col >> 2, its high two col & 3
      const uint8_t *kp =
          ARR == kPair ? slot + (16 * h + token_of(col)) * 128 +
                             (((4 * g + quad) ^ pair_swizzle(token_of(col))) << 4)
                       : slot + g * kHeadBytes + h * kHalfBytes + token_of(col) * 64 +
                             ((quad ^ (col & 3)) << 4);
      const u32x4 k = *reinterpret_cast<const u32x4 *>(kp);
      const uint32_t ks = mx_scale(*reinterpret_cast<const uint32_t *>(
                                       slot + S::ks + S::template scales<P16>(g, h) + col * 4),
                                   quad);
      s[g][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        s[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(mx4x8_to_bf16x8(k[c], ks)),
                                                          as_bf16x8(st[g].q[c]), s[g][h], 0, 0, 0);
    }
  // s[g][h][i] = S[token 16 h + 4 i + quad][column col]
  if (rows < kBlock) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (16 * h + 4 * i + quad >= rows) {
#pragma unroll
          for (int g = 0; g < NH; ++g) s[g][h][i] = -INFINITY;
        }
  }
  // (a NaN score makes the maximum NaN, and with it the whole column)
  float mx[NH];
  bool passed = false;
#pragma unroll
  for (int g = 0; g < NH; ++g) {
    mx[g] = fmax_nan(fmax_nan(fmax_nan(s[g][0][0], s[g][0][1]), fmax_nan(s[g][0][2], s[g][0][3])),
                     fmax_nan(fmax_nan(s[g][1][0], s[g][1][1]), fmax_nan(s[g][1][2], s[g][1][3]))) *
            scale_log2;
    passed |= mx[g] > st[g].m_run;
  }
  if (__builtin_amdgcn_ballot_w64(passed)) {
#pragma unroll
    for (int g = 0; g < NH; ++g) {
      const float top = quad_max_nan(mx[g]);
      const float m_new = top > st[g].m_run ? top + kLazy : top == top ? st[g].m_run : top;
      const float al = fast_exp2(st[g].m_run - m_new);
      st[g].m_run = m_new;
      st[g].l_run *= al;
#pragma unroll
      for (int e = 0; e < HeadState<QUADS>::kAcc; ++e) st[g].acc[e] *= al;
    }
  }
#pragma unroll
  for (int g = 0; g < NH; ++g) {
    float pf[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        pf[h][i] = fast_exp2(fmaf(s[g][h][i], scale_log2, -st[g].m_run));
        pf[h][i + 1] = fast_exp2(fmaf(s[g][h][i + 1], scale_log2, -st[g].m_run));
        st[g].l_run += pf[h][i] + pf[h][i + 1];
      }
    bf16x8 p[2];
    st[g].pack_p(pf, col, p);
    // V codes of rows 4 j + quad.  Rows past the valid ones are zeros and weigh nothing.
    uint32_t v[2][4];
    float vs[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(
          slot + S::vs + S::template scales<P16>(g, h) + quad * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        vs[h][j] = __uint_as_float(mx_scale(w[j], col >> 2));
        const uint8_t *vp =
            ARR == kPair ? slot + S::v + (16 * h + 4 * j + quad) * 128 +
                               (((4 * g + (col >> 2)) ^ pair_swizzle(4 * j + quad)) << 4)
                         : slot + S::v + g * kHeadBytes + h * kHalfBytes + (4 * j + quad) * 64 +
                               (((col >> 2) ^ j) << 4);
        v[h][j] = *reinterpret_cast<const uint32_t *>(vp + (col & 3) * 4);
      }
    }
    st[g].template add_pv<0>(v, vs, p);
    st[g].template add_pv<1>(v, vs, p);
    st[g].template add_pv<2>(v, vs, p);
    st[g].template add_pv<3>(v, vs, p);
  }
}

// ---- balanced ---------------------------------------------------------------------
template <int NH>
struct BalancedSmem {
  uint8_t slots[kWaves][kDepth][Slot<NH>::bytes];
  int64_t prefix[kPrefix];  // blocks before request i * stride
  int32_t st[kPrefix];      // with stride 1: indptr[i], and the tokens of its last block
  uint8_t tail[kPrefix];
  int64_t wave_tot[kWaves];
};

// Blocks [v0, v0 + 64) of the virtual list, one per lane.
struct Blocks {
  uint32_t c0, s0, c1, s1;  // as in Place
  int meta;  // valid rows | first block of its request << 8 | last << 9
  int req;
  // Lane i's rows; `meta`: its meta.
  template <bool P16>
  __device__ __forceinline__ Place place(int i, int meta) const {
    Place p;
    p.rows = meta & 255;
    p.c0 = (uint32_t)__builtin_amdgcn_readlane((int)c0, i);
    p.s0 = (uint32_t)__builtin_amdgcn_readlane((int)s0, i);
    p.c1 = P16 ? (uint32_t)__builtin_amdgcn_readlane((int)c1, i) : 0;
    p.s1 = P16 ? (uint32_t)__builtin_amdgcn_readlane((int)s1, i) : 0;
    return p;
  }
  // This lane's rows, from the pages p0 and p1 of its halves; false: an index is invalid.
  template <bool P16>
  __device__ __forceinline__ bool set(const Mx4DecodeArgs &a, int p0, int p1, int row, int kvh) {
    const bool ok = p0 >= 0 && (int64_t)p0 < a.pool && p1 >= 0 && (int64_t)p1 < a.pool;
    if (ok) {
      cache_rows(a, p0, row, kvh, c0, s0);
      if (P16) cache_rows(a, p1, row, kvh, c1, s1);
    }
    return ok;
  }
  // Ends the loads behind them here, as HeadState::settle_q does and for its reason.
  __device__ __forceinline__ void settle() {
    asm volatile("" : "+v"(c0), "+v"(s0), "+v"(c1), "+v"(s1), "+v"(meta), "+v"(req));
  }
};

// The virtual list as a wave knows it.  Up to 64 requests: lane r holds request r's
// inclusive prefix, first page position and tokens of its last block (`in_lanes`).  More:
// the LDS table.
struct List {
  bool in_lanes;
  uint32_t incl, cnt;  // this lane's request
  int32_t st, tail;
  int entries, stride;
  int32_t ipB;
  int64_t total;
};

template <bool P16, class Smem>
__device__ __forceinline__ Blocks find_blocks(const Mx4DecodeArgs &a, const Smem &sm,
                                              const List &list, int64_t v0, int64_t v_end, int lane,
                                              int kvh) {
  Blocks d = {0, 0, 0, 0, 0, -1};
  const int64_t v = v0 + lane;
  const bool in = v < v_end;
  int r = 0;
  int64_t b = 0, cnt = 1;  // block of its request, and that one's blocks
  int32_t st = 0, tail = 0;
  if (list.in_lanes) {
    // the request of v0, then on while later requests begin at or before v
    const uint32_t x = (uint32_t)v, end = (uint32_t)min<int64_t>(v0 + 64, v_end);
    int next = __builtin_ctzll(__builtin_amdgcn_ballot_w64(list.incl > (uint32_t)v0));
    r = next;
    while (true) {
      const uint32_t e = (uint32_t)__builtin_amdgcn_readlane((int)list.incl, next);
      if (e >= end) break;
      ++next;
      if (x >= e) r = next;
    }
    st = __shfl(list.st, r, 64);
    tail = __shfl(list.tail, r, 64);
    const uint32_t c = (uint32_t)__shfl((int)list.cnt, r, 64);
    cnt = c;
    b = x - ((uint32_t)__shfl((int)list.incl, r, 64) - c);
  } else if (in) {
    int lo = 0, n = list.entries;  // the last entry with prefix <= v
    while (n > 1) {
      const int half = n >> 1;
      if (sm.prefix[lo + half] <= v) {
        lo += half;
        n -= half;
      } else {
        n = half;
      }
    }
    r = lo;
    int64_t pre = sm.prefix[lo];
    if (list.stride == 1) {
      cnt = (lo + 1 < list.entries ? sm.prefix[lo + 1] : list.total) - pre;
      st = sm.st[lo];
      tail = sm.tail[lo];
    } else {
      r = lo * list.stride;
      while (true) {
        st = a.indptr[r];
        const int64_t t = request_tokens(a, st, a.indptr[r + 1], a.last[r], list.ipB);
        cnt = (t + kBlock - 1) / kBlock;
        tail = (int)(t - (cnt - 1) * kBlock);
        if (v < pre + cnt || r + 1 >= a.batch) break;
        pre += cnt;
        ++r;
      }
    }
    b = v - pre;
  }
  if (!in) return d;
  const bool last = b == cnt - 1;
  int rows = last ? tail : kBlock;
  // token 32 b lies in the request's page 32 b / P, row 32 b % P
  const int64_t pos = st + (P16 ? 2 * b : a.page_rows == 64 ? b >> 1 : b);
  const int row = !P16 && a.page_rows == 64 ? (int)(b & 1) * kBlock : 0;
  const int p0 = a.indices[pos], p1 = P16 && rows > 16 ? a.indices[pos + 1] : p0;
  if (!d.set<P16>(a, p0, p1, row, kvh)) rows = 0;
  d.meta = rows | (b == 0 ? 256 : 0) | (last ? 512 : 0);
  d.req = r;
  return d;
}

// NH: kv-heads per wave; they divide Hkv.
template <bool P16, int NH, int ARR, bool QUADS>
__global__ __launch_bounds__(kThreads, 2) void mx4_decode_split_kernel(
    Mx4DecodeArgs a) {
  __shared__ BalancedSmem<NH> sm;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uni(tid >> 6);
  const int32_t ip0 = a.indptr[0], ipB = a.indptr[a.batch];
  // ---- the virtual list: prefix of the valid requests' blocks ----------------------
  List list;
  list.ipB = ipB;
  list.in_lanes = false;
  if (a.batch <= 64) {
    // every wave on its own, in registers: no barrier, no LDS round trip
    int64_t t = 0;
    list.st = 0;
    if (lane < a.batch) {
      list.st = a.indptr[lane];
      t = request_tokens(a, list.st, a.indptr[lane + 1], a.last[lane], ipB);
    }
    const int64_t cnt = (t + kBlock - 1) / kBlock;
    list.cnt = (uint32_t)min<int64_t>(cnt, UINT32_MAX);
    list.tail = (int)(t - (cnt - 1) * kBlock);
    list.incl = wave_incl_add_sat_u32(list.cnt);
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)list.incl, 63);
    list.total = total;
    list.in_lanes = total < (uint32_t)INT32_MAX;  // (else the 64-bit table)
    if (list.in_lanes && blockIdx.x == 0 && wave == 0 && lane < a.batch)
      a.header[1 + lane] = list.incl - list.cnt;
  }
  if (!list.in_lanes) {
    int stride = 1;
    while (a.batch > kPrefix * stride) stride <<= 1;
    list.stride = stride;
    list.entries = (a.batch + stride - 1) / stride;
    int64_t carry = 0;
    for (int base = 0; base < a.batch; base += kThreads) {
      const int r = base + tid;
      int64_t cnt = 0;
      int32_t st = 0;
      int tail = 0;
      if (r < a.batch) {
        st = a.indptr[r];
        const int64_t t = request_tokens(a, st, a.indptr[r + 1], a.last[r], ipB);
        cnt = (t + kBlock - 1) / kBlock;
        tail = (int)(t - (cnt - 1) * kBlock);
      }
      const int64_t x = wave_incl_scan64(cnt, lane);
      if (lane == 63) sm.wave_tot[wave] = x;
      __syncthreads();
      int64_t before = carry, tot = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        const int64_t t = sm.wave_tot[i];
        before += i < wave ? t : 0;
        tot += t;
      }
      if (r < a.batch) {
        const int64_t pre = before + x - cnt;
        if (r % stride == 0) sm.prefix[r / stride] = pre;
        if (stride == 1) {
          sm.st[r] = st;
          sm.tail[r] = (uint8_t)tail;
        }
        if (blockIdx.x == 0) a.header[1 + r] = pre;
      }
      carry += tot;
      __syncthreads();
    }
    list.total = uni64(carry);
  }
  const int64_t total = list.total;
  const bool ok = batch_ok(a, ip0, ipB);
  if (blockIdx.x == 0 && tid == 0) {
    a.header[0] = ok ? total : -1;
    a.header[1 + a.batch] = total;
  }
  if (!ok) return;

  // ---- this wave's team and member --------------------------------------------------
  // Workgroup b runs on XCD b % 8; a team's members are consecutive waves of one XCD
  // (one L2, the same blocks at the same time), team t on XCD t % 8.
  const int members = a.hkv / NH * a.tiles;
  const int xcd_wave = (int)(blockIdx.x >> 3) * kWaves + wave;
  const Ranges ranges(total, a.teams);
  const int team = (xcd_wave / members) * 8 + (int)(blockIdx.x & 7);
  const int member = xcd_wave % members;
  if (team >= ranges.teams) return;  // no workgroup barrier follows
  const int kvh = member % (a.hkv / NH) * NH;
  const int g0 = member / (a.hkv / NH) * a.tile;
  const int heads = min(a.tile, a.group - g0);
  const int64_t v_begin = ranges.start(team), v_end = ranges.start(team + 1);
  const int n = uni((int)min<int64_t>(v_end - v_begin, INT32_MAX - 64));
  if (n <= 0) return;

  HeadState<QUADS> w[NH];
  constexpr int kHeadMask = HeadState<QUADS>::kHeadMask;
  const int col = lane & 15, quad = lane >> 4;
  const bool mine = col < heads, loads_q = (col & kHeadMask) < heads;
  const int qh = kvh * a.group + g0 + (col & kHeadMask);  // of the first kv-head

  // ---- one continuous stream of blocks ----------------------------------------------
  // Block i + kDepth - 1 is issued before block i is consumed, across request
  // boundaries.  Blocks are located 64 at a time, one per lane.
  Blocks cur = {0, 0, 0, 0, 0, -1}, next = cur;
  const uint32_t slots = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)sm.slots[wave];
  // Block i into slot i % kDepth; its Blocks::meta and ::req.
  auto issue = [&](int i, int slot, int &meta, int &req) {
    const int j = i & 63;
    if (j == 0) {
      cur = next;  // located 64 blocks ago
      if (i + 64 < n) next = find_blocks<P16>(a, sm, list, v_begin + i + 64, v_end, lane, kvh);
      next.settle();
    }
    meta = uni(i < n ? __builtin_amdgcn_readlane(cur.meta, j) : 0);  // past the range: no rows
    req = __builtin_amdgcn_readlane(cur.req, j);
    load_block<P16, NH, ARR, true>(a, cur.place<P16>(j, meta),
                                   slots + slot * Slot<NH>::bytes, lane);
  };

  int r = -1;
  bool first = false, last = false, bad = false;
  auto finish = [&]() {
#pragma unroll
    for (int g = 0; g < NH; ++g) {
      const float l = w[g].normalizer();
      f32x4 o[8];
      w[g].columns(o);
      if (!mine) continue;
      const int64_t head = qh + g * a.group;
      if (first && last) {  // the whole request; an invalid page index keeps its sentinels
        const int64_t row = (int64_t)r * a.hq + head;
        if (!bad) w[g].store(o, a.out + row * 128, a.lse + row, l, quad);
        continue;
      }
      // One state per (team, request): slot team + r (along the virtual list the team
      // or the request advances at every piece).
      float *st = a.states + ((int64_t)(team + r) * a.hq + head) * kMx4StateStride;
      if (!bad) w[g].stash(o, st + 4, quad);
      if (quad == 0) {
        st[0] = bad ? 0.0f : w[g].m_run;
        st[1] = bad ? kPoisonNormalizer : l;
      }
    }
  };

  int meta[kDepth], req[kDepth];  // of blocks i, i + 1, ..., the last being issued
  next = find_blocks<P16>(a, sm, list, v_begin, v_end, lane, kvh);
  next.settle();
#pragma unroll
  for (int j = 0; j < kDepth - 1; ++j) issue(j, j, meta[j], req[j]);
  int slot = 0;
  for (int i = 0; i < n; ++i) {
    const int ahead = slot == 0 ? kDepth - 1 : slot - 1;  // (slot + kDepth - 1) % kDepth
    wait_reads();
    issue(i + kDepth - 1, ahead, meta[kDepth - 1], req[kDepth - 1]);
    if (req[0] != r) {
      if (r >= 0) finish();
      r = req[0];
#pragma unroll
      for (int g = 0; g < NH; ++g)
        w[g].load_q(a.q + ((int64_t)r * a.hq + qh + g * a.group) * 128, loads_q, quad);
#pragma unroll
      for (int g = 0; g < NH; ++g) {
        w[g].reset();
        w[g].settle_q();
      }
      first = (meta[0] & 256) != 0;
      bad = false;
    }
    last = (meta[0] & 512) != 0;
    const int rows = meta[0] & 255;
    bad |= rows == 0;
    // Block i has arrived once at most the loads issued after it are outstanding
    // (others in between only make the wait longer).
    wait_loads<(kDepth - 1) * kBlockLoads<P16, NH>>();
    process_block<P16, NH, ARR, QUADS>(w, sm.slots[wave][slot], rows, col, quad, a.scale_log2);
#pragma unroll
    for (int j = 0; j + 1 < kDepth; ++j) {
      meta[j] = meta[j + 1];
      req[j] = req[j + 1];
    }
    if (++slot == kDepth) slot = 0;
  }
  finish();
  // loads past the range still write this wave's slots
  wait_loads<0>();
}

// ---- merge ---------------------------------------------------------------------------
// O and LSE of `cols` query heads (query_head(c) of request r) from `count` states of
// consecutive slots, by a workgroup of W waves: `parts` waves per head (a power of two,
// at most W) take every parts-th state, a lane two of the 128 dims, eight states in
// flight; the parts' sums are combined in LDS in order.  A poisoned state leaves the
// head's sentinels.
constexpr int kMergeBatch = 8;
template <bool kArrived>
__device__ __forceinline__ f32x2 load_state(const float *p) {
  if constexpr (kArrived)
    return __builtin_bit_cast(
        f32x2, __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED,
                                 __HIP_MEMORY_SCOPE_AGENT));
  else
    return *reinterpret_cast<const f32x2 *>(p);
}
__device__ __forceinline__ void store_state(float *p, float x, float y) {
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p), __builtin_bit_cast(uint64_t, f32x2{x, y}),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int W>
struct MergeSmem {
  float m[W], l[W];
  f32x2 o[W][64];
};
// kArrived: the states come from workgroups of this launch; they are read as they were
// written, past L2, which other XCDs do not share.
template <int W, bool kArrived, class Head>
__device__ __forceinline__ void merge_heads(const Mx4DecodeArgs &a, MergeSmem<W> &sm, int r,
                                            Head query_head, int cols, int parts, int64_t slot0,
                                            int count) {
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int64_t step = (int64_t)a.hq * kMx4StateStride;
  const int part = wave & (parts - 1);
  for (int c0 = 0; c0 < cols; c0 += W / parts) {
    const int c = c0 + wave / parts;
    const bool in = c < cols;
    const int qh = in ? query_head(c) : 0;
    float M = -FLT_MAX, l = 0.f;
    f32x2 o = {0.f, 0.f};
    bool poisoned = false;
    if (in) {
      const float *base = a.states + slot0 * step + (int64_t)qh * kMx4StateStride;
      for (int t = part; t < count; t += parts * kMergeBatch) {
        float ms[kMergeBatch], ls[kMergeBatch];
        f32x2 xs[kMergeBatch];
#pragma unroll
        for (int u = 0; u < kMergeBatch; ++u) {
          // past the last state: its values again, with no weight
          const float *ss = base + min(t + u * parts, count - 1) * step;
          const f32x2 ml = load_state<kArrived>(ss);
          ms[u] = ml[0];
          ls[u] = ml[1];
          xs[u] = load_state<kArrived>(ss + 4 + 2 * lane);
        }
        float mb = M;
#pragma unroll
        for (int u = 0; u < kMergeBatch; ++u) {
          mb = fmaxf(mb, ms[u]);
          poisoned |= ls[u] < 0.0f;
        }
        const float sc = fast_exp2(M - mb);
        l *= sc;
        o *= sc;
#pragma unroll
        for (int u = 0; u < kMergeBatch; ++u) {
          const float f = t + u * parts < count ? fast_exp2(ms[u] - mb) : 0.f;
          l = fmaf(ls[u], f, l);
          o[0] = fmaf(xs[u][0], f, o[0]);
          o[1] = fmaf(xs[u][1], f, o[1]);
        }
        M = mb;
      }
    }
    if (parts > 1) {
      if (c0) __syncthreads();
      sm.o[wave][lane] = o;
      if (lane == 0) {
        sm.m[wave] = M;
        sm.l[wave] = poisoned ? kPoisonNormalizer : l;
      }
      __syncthreads();
      if (part != 0) continue;
      for (int i = wave; i < wave + parts; ++i) {
        M = fmaxf(M, sm.m[i]);
        poisoned |= sm.l[i] < 0.0f;
      }
      l = 0.f;
      o = f32x2{0.f, 0.f};
      for (int i = wave; i < wave + parts; ++i) {
        const float f = fast_exp2(sm.m[i] - M);
        l = fmaf(sm.l[i], f, l);
        o[0] = fmaf(sm.o[i][lane][0], f, o[0]);
        o[1] = fmaf(sm.o[i][lane][1], f, o[1]);
      }
    }
    if (!in || poisoned) continue;
    const int64_t row = (int64_t)r * a.hq + qh;
    const float inv = 1.0f / l;
    *reinterpret_cast<uint32_t *>(a.out + row * 128 + 2 * lane) =
        bf16x2_pack(o[0] * inv, o[1] * inv);
    if (lane == 0) a.lse[row] = M + __log2f(l);
  }
}

// The requests that span several teams: kWaves / parts query heads per workgroup.
__global__ __launch_bounds__(kThreads) void mx4_decode_merge_kernel(Mx4DecodeArgs a, int parts) {
  __shared__ MergeSmem<kWaves> sm;
  const int wg_heads = kWaves / parts, wgs = (a.hq + wg_heads - 1) / wg_heads;
  const int r = (int)(blockIdx.x / wgs), q0 = (int)(blockIdx.x % wgs) * wg_heads;
  const int64_t total = a.header[0], pre = a.header[1 + r], end = a.header[2 + r];
  if (total <= 0 || end <= pre) return;
  const Ranges ranges(total, a.teams);
  const int64_t t0 = ranges.team_of(pre), t1 = ranges.team_of(end - 1);
  if (t0 == t1) return;
  merge_heads<kWaves, false>(a, sm, r, [&](int c) { return q0 + c; }, min(wg_heads, a.hq - q0), parts, t0 + r,
              (int)(t1 - t0) + 1);
}

// ---- direct --------------------------------------------------------------------------
// Wave w of the workgroup takes blocks w, w + W, ... of its split's share of the request,
// two in flight; the wave states merge in LDS.  (One request of 200 tokens: 4.9 us, of
// 1000 without splits 7.9: a block in each of two waves of a SIMD, about 1 us.)
constexpr int kDirectWaves = 8;
constexpr int kStash = 132;  // floats between two columns' O in LDS

template <bool P16, int NH, int ARR, bool QUADS>
__global__ __launch_bounds__(kDirectWaves * 64) void mx4_decode_direct_kernel(Mx4DecodeArgs a) {
  constexpr int W = kDirectWaves;
  constexpr int kCols = NH * kMaxTile;
  // Each wave's two slots; after its walk its columns' O, kStash floats apart.
  constexpr int kWaveBytes = 2 * Slot<NH>::bytes;
  static_assert(kCols * kStash * 4 <= kWaveBytes, "a wave's columns in its slots");
  __shared__ __align__(16) uint8_t s_wave[W][kWaveBytes];
  __shared__ float s_m[W][kCols], s_l[W][kCols];
  __shared__ uint32_t s_bad[W];
  __shared__ uint32_t s_arrived;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uni(tid >> 6);
  const uint32_t head = blockIdx.x / (uint32_t)a.splits;
  const int split = (int)(blockIdx.x % (uint32_t)a.splits);
  const int kvh = (int)(head % (uint32_t)(a.hkv / NH)) * NH;
  const uint32_t rest = head / (uint32_t)(a.hkv / NH);
  const int g0 = (int)(rest % (uint32_t)a.tiles) * a.tile;
  const int r = (int)(rest / (uint32_t)a.tiles);
  const int heads = min(a.tile, a.group - g0);
  HeadState<QUADS> w[NH];
  constexpr int kHeadMask = HeadState<QUADS>::kHeadMask;
  const int col = lane & 15, quad = lane >> 4;
  // query head of column c of the workgroup's NH * heads
  auto query_head = [&](int c) {
    const int g = NH == 2 && c >= heads ? 1 : 0;
    return (kvh + g) * a.group + g0 + c - g * heads;
  };
  // A split always writes its state (a poisoned one where a guard fails) and arrives, so
  // the last one to arrive at the word of these heads finds them all: it merges them and
  // clears the word for the queue's next command.  Nobody waits.
  auto state_of = [&](int c) {
    return a.states + (((int64_t)r * a.splits + split) * a.hq + query_head(c)) * kMx4StateStride;
  };
  // The states go to memory and come from there (agent-scope accesses); each wave waits
  // for its own to arrive before the barrier behind which one thread counts the
  // workgroup.  A release fence instead writes the XCD's whole L2 back: 40 us here.
  auto arrive = [&]() {
    uint32_t *const arrived = a.arrived + (uint64_t)head * (loom::kMx4JoinBytes / 4);
    wait_loads<0>();  // and stores
    __syncthreads();
    if (tid == 0)
      s_arrived = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_arrived != (uint32_t)a.splits - 1u) return;
    if (tid == 0)
      __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int cols = NH * heads;
    const int parts = cols <= 1 ? 8 : cols <= 2 ? 4 : cols <= 4 ? 2 : 1;
    static_assert(W == 8, "parts");
    merge_heads<W, true>(a, *reinterpret_cast<MergeSmem<W> *>(s_wave), r, query_head, cols, parts,
                (int64_t)r * a.splits, a.splits);
  };
  auto poison = [&]() {
    if (a.splits == 1) return;
    if (tid < NH * heads) store_state(state_of(tid), 0.0f, kPoisonNormalizer);
    arrive();
  };
  // One round trip for the guard words, the queries and, when the page-index array is
  // short, all of it.
#pragma unroll
  for (int g = 0; g < NH; ++g)
    w[g].load_q(a.q + ((int64_t)r * a.hq + (kvh + g) * a.group + g0 + (col & kHeadMask)) * 128,
                (col & kHeadMask) < heads, quad);
  const bool whole_table = a.n_indices <= 128;
  int tbl0 = 0, tbl1 = 0;
  if (whole_table) {
    if (lane < a.n_indices) tbl0 = a.indices[lane];
    if (lane + 64 < a.n_indices) tbl1 = a.indices[lane + 64];
  }
  const int32_t ip0 = a.indptr[0], ipB = a.indptr[a.batch];
  const int32_t st = uni(a.indptr[r]), en = uni(a.indptr[r + 1]), tl = uni(a.last[r]);
  const int64_t tokens = request_tokens(a, st, en, tl, ipB);
  if (!batch_ok(a, ip0, ipB) || tokens == 0) return poison();
  // this split's blocks [lo, hi), this wave's lo + wave + W i
  const int64_t cnt = (tokens + kBlock - 1) / kBlock;
  int64_t lo = 0, hi = cnt;
  if (a.splits > 1) {
    lo = floor_div(cnt * split, a.splits);
    hi = floor_div(cnt * (split + 1), a.splits);
  }
  const int64_t n = hi - lo > wave ? (hi - lo - wave + W - 1) / W : 0;
  bool bad = false;
#pragma unroll
  for (int g = 0; g < NH; ++g) w[g].reset();
  Blocks cur = {0, 0, 0, 0, 0, 0};
  auto locate = [&](int64_t i0) {  // the wave's blocks i0 + [0, 64), one per lane
    const bool in = i0 + lane < n;
    const int64_t b = lo + wave + W * (i0 + lane);
    int rows = in ? (int)min<int64_t>(kBlock, tokens - b * kBlock) : 0;
    const int64_t pos = st + (P16 ? 2 * b : a.page_rows == 64 ? b >> 1 : b);
    const bool two = P16 && rows > 16;
    int p0 = 0, p1 = 0;
    if (whole_table) {  // pos < 128 for blocks that exist
      const int j = (int)pos, lo0 = __shfl(tbl0, j & 63, 64), hi0 = __shfl(tbl1, j & 63, 64);
      const int lo1 = __shfl(tbl0, (j + 1) & 63, 64), hi1 = __shfl(tbl1, (j + 1) & 63, 64);
      p0 = j < 64 ? lo0 : hi0;
      p1 = !two ? p0 : j + 1 < 64 ? lo1 : hi1;
    } else if (in) {
      p0 = a.indices[pos];
      p1 = two ? a.indices[pos + 1] : p0;
    }
    const int row = !P16 && a.page_rows == 64 ? (int)(b & 1) * kBlock : 0;
    if (in && !cur.set<P16>(a, p0, p1, row, kvh)) {
      rows = 0;
      bad = true;
    }
    cur.meta = rows;
  };
  uint8_t *const slots = s_wave[wave];
  const uint32_t slots_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)slots;
  for (int64_t i0 = 0; i0 < n; i0 += 64) {
    locate(i0);
    const int m = uni((int)min<int64_t>(64, n - i0));
    auto issue = [&](int i) {
      const int rows = __builtin_amdgcn_readlane(cur.meta, i);
      load_block<P16, NH, ARR, false>(a, cur.place<P16>(i, rows),
                                      slots_at + (i & 1) * Slot<NH>::bytes, lane);
      return rows;
    };
    cur.settle();
#pragma unroll
    for (int g = 0; g < NH; ++g) w[g].settle_q();
    wait_reads();
    int rows = issue(0);
    for (int i = 0; i < m; ++i) {
      int rows_next = 0;
      if (i + 1 < m) {
        wait_reads();
        rows_next = issue(i + 1);
        wait_loads<kBlockLoads<P16, NH>>();
      } else {
        wait_loads<0>();
      }
      process_block<P16, NH, ARR, QUADS>(w, slots + (i & 1) * Slot<NH>::bytes, rows, col, quad,
                                         a.scale_log2);
      rows = rows_next;
    }
  }
  // The wave's slots become its columns' place.
  wait_reads();
#pragma unroll
  for (int g = 0; g < NH; ++g) {
    const float l = w[g].normalizer();
    f32x4 o[8];
    w[g].columns(o);
    if (col < heads) {
      const int c = g * heads + col;
      w[g].stash(o, reinterpret_cast<float *>(slots) + c * kStash, quad);
      if (quad == 0) {
        s_m[wave][c] = w[g].m_run;
        s_l[wave][c] = l;
      }
    }
  }
  // An invalid page index anywhere in the request keeps its sentinels.
  if (block_or(bad, s_bad)) return poison();
  // Four dims of one column per thread.
  for (int x = tid; x < NH * heads * 32; x += W * 64) {
    const int g = x >> 5, d = (x & 31) * 4;
    float M = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < W; ++i) M = fmax_nan(M, s_m[i][g]);
    float L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float f = fast_exp2(s_m[i][g] - M);
      const f32x4 o = *reinterpret_cast<const f32x4 *>(
          reinterpret_cast<const float *>(s_wave[i]) + g * kStash + d);
      L = fmaf(s_l[i][g], f, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = fmaf(o[e], f, O[e]);
    }
    if (a.splits > 1) {
      float *ss = state_of(g);
      store_state(ss + 4 + d, O[0], O[1]);
      store_state(ss + 6 + d, O[2], O[3]);
      if (d == 0) store_state(ss, M, L);
      continue;
    }
    const int64_t row = (int64_t)r * a.hq + query_head(g);
    const float inv = 1.0f / L;
    *reinterpret_cast<u32x2 *>(a.out + row * 128 + d) =
        u32x2{bf16x2_pack(O[0] * inv, O[1] * inv), bf16x2_pack(O[2] * inv, O[3] * inv)};
    if (d == 0) a.lse[row] = M + __log2f(L);
  }
  if (a.splits > 1) arrive();
}

__global__ void mx4_decode_clear_kernel(uint32_t *arrived) {
  arrived[threadIdx.x * (loom::kMx4JoinBytes / 4)] = 0u;
}

// kv-heads per wave: two neighbours where Hkv is even, in the balanced kernel always.
uint64_t heads_per_wave(uint64_t hkv) { return hkv % 2 == 0 ? 2 : 1; }

}  // namespace

namespace loom {

// The algorithm goes by the tokens a plan covers times Hkv (the rows of K to read).
// Microseconds, direct / balanced, 32x8 heads unless said: 1 x 1000 tokens 7.4 / 11.6;
// 1 x 32000 14.4 / 23.5; 16 x 256-1536 11.5 / 15.5; 64 x 256-1024 15.8 / 21.9; 16 x 4096
// 20.8 / 22.7; 64 x 1024-4096 (1.3 M rows) 45.4 / 40.4; 8 x 1000-32000 (1.1 M) 44.7 /
// 38.4: a direct workgroup has one request's share, so unlike lengths cost it more.
constexpr uint64_t kDirectRows = 1u << 20;
// Direct workgroups over NHD pages take two kv-heads from this many rows on, where whole
// cache lines outweigh the halved parallelism (one / two): 16 x 256-1536 (below it) 11.5 /
// 15.9; 64 x 256-1024 19.1 / 15.8; 16 x 4096 28.3 / 20.8, of 64 / 8 heads 27.8 / 22.2;
// but 32 x 512-4096 of 64 / 8 28.7 / 34.4.
constexpr uint64_t kDirectPairRows = 5u << 16;
// Workgroups per (request, kv-heads, tile), of 8 waves each (4 and 16 were slower).  The
// walk shrinks with the splits and the join grows, so they are doubled while their square
// stays within twice a request's blocks and the CUs hold them (1000 tokens in 8, 16, 32:
// 7.4, 7.4, 8.3 us; 8000: 11.3, 9.4, 9.5; 32000: 23.0, 15.8, 14.4; two per CU: no faster).
// A join costs about 2 us, and 4 where every CU joins at once; a wave's block costs 1.
// Splits that save fewer than kSplitFrom / 8 blocks a wave are left out (one request of
// 700 tokens: 6.9 us, split 8.1; of 1000, 8.1 and in eight 7.4), kSplitFromMany / 8 where
// the requests' own workgroups are more than an eighth of the CUs (8 of 1000: 8.8, in
// four each 10.2; 16 of 2000: 12.6 and 13.1).
constexpr uint64_t kMaxSplits = 64, kSplitFrom = 21, kSplitFromMany = 40;

// kv-heads per direct workgroup.
static uint64_t direct_heads(const loom_paged_decode_plan_info_t &info) {
  const loom_paged_decode_spec_t &s = info.spec;
  const uint64_t page_rows = s.page_size ? s.page_size : kPageSize;
  return s.kv_layout != LOOM_KV_LAYOUT_HND && s.num_kv_heads % 2 == 0 &&
                 info.max_total_pages * page_rows * s.num_kv_heads >= kDirectPairRows
             ? 2
             : 1;
}
uint64_t mx4_direct_grid(const loom_paged_decode_plan_info_t &info, uint64_t splits) {
  const uint64_t grid = info.spec.batch_size * (info.spec.num_kv_heads / direct_heads(info)) *
                        info.group_tiles * splits;
  return grid <= UINT32_MAX / (kDirectWaves * 64) ? grid : 0;
}

// The merge kernel's workgroups and their waves per head: one up to 48 states per request
// on average (64 ragged requests, 5: 52.1 us, with four waves 55.5; 8 of 32k, 33: 56.8 and
// 57.6).
struct MergeGrid {
  uint64_t grid;
  int parts;
};
static MergeGrid merge_grid(uint64_t batch, uint64_t hq, uint64_t teams) {
  const int parts = teams / batch >= 48 ? kWaves : 1;
  const uint64_t heads = kWaves / parts;
  return {batch * ((hq + heads - 1) / heads), parts};
}

loom_status_t plan_mx4_decode(loom_paged_decode_plan_info_t *info, uint32_t teams_option, int cus,
                              loom_error_t *err) {
  const loom_paged_decode_spec_t &s = info->spec;
  const uint64_t B = s.batch_size, hq = s.num_query_heads, hkv = s.num_kv_heads;
  const uint64_t group = hq / hkv;
  const uint32_t tile = (uint32_t)std::min<uint64_t>(group, kMaxTile);
  const uint64_t tiles = (group + tile - 1) / tile;
  const uint64_t page_rows = s.page_size ? s.page_size : kPageSize;
  if (B > (uint64_t)kMaxBatch)
    return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "batch_size", B);
  // the bound of a step is its largest product times the scale, and masked ones are -inf
  if (!(s.softmax_scale > 0.0f) || !std::isfinite(s.softmax_scale))
    return fail(err, LOOM_PLAN_INVALID_OPTION, "softmax_scale");
  uint64_t pool_rows;
  if (__builtin_mul_overflow(s.max_num_pages * page_rows, hkv, &pool_rows) ||
      pool_rows > UINT32_MAX)
    return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "paged batch-decode cache rows", pool_rows);
  info->group_tile = tile;
  info->group_tiles = (uint32_t)tiles;
  info->device_cus = (uint32_t)cus;
  info->header_bytes = 0;
  // blocks of 32 tokens that the plan covers
  const uint64_t blocks = info->max_total_pages * page_rows / kBlock + B;
  if (blocks > (uint64_t)INT32_MAX)
    return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "paged batch-decode blocks", blocks);
  const uint64_t rows = info->max_total_pages * page_rows * hkv;
  if (teams_option == 0 && rows <= kDirectRows) {
    const uint64_t heads = mx4_direct_grid(*info, 1);
    if (heads == 0 || B * hq > (uint64_t)INT32_MAX)
      return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "paged batch-decode", B * hq);
    uint64_t splits = 1;
    const uint64_t each = blocks / B;
    while (heads <= kMx4Joins && splits < kMaxSplits && heads * splits * 2 <= (uint64_t)cus &&
           each >= 2 * splits * splits)
      splits *= 2;
    const uint64_t from = heads * 8 <= (uint64_t)cus ? kSplitFrom : kSplitFromMany;
    if (each * (splits - 1) < from * splits) splits = 1;
    const uint64_t grid = heads * splits;  // (split ones are at most the CUs)
    info->algorithm = LOOM_PAGED_DECODE_DIRECT;
    info->teams = (uint32_t)(splits > 1 ? splits : 0);
    info->state_slots = splits > 1 ? splits * B : 0;
    info->header_bytes = splits > 1 ? kMx4Joins * kMx4JoinBytes : 0;
    info->workspace_bytes =
        splits > 1 ? info->header_bytes + splits * B * hq * kMx4StateStride * 4 : 256;
    info->block_threads = kDirectWaves * 64;
    info->grid_blocks = (uint32_t)grid;
    return LOOM_OK;
  }
  const uint64_t members = hkv / heads_per_wave(hkv) * tiles;
  const uint64_t slots = (uint64_t)cus * kWavesPer4Cu / 4;
  const uint64_t teams = teams_option ? teams_option : std::max<uint64_t>(1, slots / members);
  // Each XCD (every 8th workgroup) holds ceil(teams / 8) whole teams.
  const uint64_t xcd_waves = (teams + 7) / 8 * members;
  const uint64_t grid = (xcd_waves + kWaves - 1) / kWaves * 8;
  // (a launch holds fewer than 2^32 threads)
  if (grid > UINT32_MAX / kThreads || teams > (uint64_t)INT32_MAX ||
      B * hq > (uint64_t)INT32_MAX || merge_grid(B, hq, teams).grid > UINT32_MAX / kThreads)
    return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "paged batch-decode", grid);
  info->algorithm = LOOM_PAGED_DECODE_BALANCED_SPLIT_KV;
  info->teams = (uint32_t)teams;
  info->header_bytes = ((B + 2) * 8 + 255) / 256 * 256;
  info->state_slots = teams + B;
  info->workspace_bytes = info->header_bytes + info->state_slots * hq * kMx4StateStride * 4;
  info->block_threads = kThreads;
  info->grid_blocks = (uint32_t)grid;
  return LOOM_OK;
}

using Mx4Kernel = void (*)(Mx4DecodeArgs);
template <int NH, int ARR, bool QUADS>
static Mx4Kernel direct_kernel(bool p16) {
  return p16 ? mx4_decode_direct_kernel<true, NH, ARR, QUADS>
             : mx4_decode_direct_kernel<false, NH, ARR, QUADS>;
}
template <int NH, int ARR, bool QUADS>
static Mx4Kernel split_kernel(bool p16) {
  return p16 ? mx4_decode_split_kernel<true, NH, ARR, QUADS>
             : mx4_decode_split_kernel<false, NH, ARR, QUADS>;
}

hipError_t launch_mx4_decode(const loom_paged_decode_plan_info_t &info, const Mx4DecodeArgs &a,
                             bool clear, hipStream_t stream) {
  // Tiles of up to 4 heads leave columns for both dims of a code byte: 32 of a block's
  // 200 vector instructions less (16 requests of 256-1536 tokens, 32 / 8 heads: 12.6 us,
  // in the other form 13.7; 64 of 2000-4000, 16 / 4: 30.0 and 33.0; 64 of 512-8192: 52.1
  // and 51.7).
  const bool p16 = a.page_rows == 16, quads = a.tile <= 4;
  if (info.algorithm == LOOM_PAGED_DECODE_DIRECT || !a.states) {
    const dim3 grid((unsigned)mx4_direct_grid(info, (uint64_t)a.splits));
    const bool pair = direct_heads(info) == 2;
    auto kernel = quads ? (pair ? direct_kernel<2, kPair, true>(p16)
                                : direct_kernel<1, kSplit, true>(p16))
                  : pair ? direct_kernel<2, kPair, false>(p16)
                         : direct_kernel<1, kSplit, false>(p16);
    if (clear) {
      hipLaunchKernelGGL(mx4_decode_clear_kernel, dim3(1), dim3(kMx4Joins), 0, stream, a.arrived);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(kDirectWaves * 64), 0, stream, a);
    return hipGetLastError();
  }
  const bool nhd = info.spec.kv_layout != LOOM_KV_LAYOUT_HND, one = heads_per_wave(a.hkv) == 1;
  auto kernel = quads ? (one   ? split_kernel<1, kSplit, true>(p16)
                         : nhd ? split_kernel<2, kPair, true>(p16)
                               : split_kernel<2, kSplit, true>(p16))
                : one ? split_kernel<1, kSplit, false>(p16)
                : nhd ? split_kernel<2, kPair, false>(p16)
                      : split_kernel<2, kSplit, false>(p16);
  hipLaunchKernelGGL(kernel, dim3(info.grid_blocks), dim3(kThreads), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const MergeGrid m = merge_grid((uint64_t)a.batch, (uint64_t)a.hq, (uint64_t)a.teams);
  hipLaunchKernelGGL(mx4_decode_merge_kernel, dim3((unsigned)m.grid), dim3(kThreads), 0, stream, a,
                     m.parts);
  return hipGetLastError();
}

}  // namespace loom
