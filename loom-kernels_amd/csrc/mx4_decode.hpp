// Paged decode over MXFP4 pages: what the planner and the enqueue of paged decode
// need of its kernels (paged_decode_mx4.hip).
#pragma once

#include "loom_internal.hpp"

namespace loom {

struct Mx4DecodeArgs {
  const uint16_t *__restrict__ q;
  const uint8_t *__restrict__ k;
  const uint8_t *__restrict__ v;
  const uint8_t *__restrict__ k_mx;  // E8M0 bytes [pool, Hkv, P, 4]
  const uint8_t *__restrict__ v_mx;
  const int32_t *__restrict__ indptr;
  const int32_t *__restrict__ indices;
  const int32_t *__restrict__ last;
  uint16_t *__restrict__ out;
  float *__restrict__ lse;
  // Workspace: split direct plans first keep kMx4Joins arrival words (used where the
  // queue's may not be); balanced plans first keep header[0] = blocks in the virtual list
  // (-1: batch rejected) and header[1 + r] = virtual block prefix of request r
  // (r = 0..B); then the split states [slot][Hq][kMx4StateStride].
  int64_t *__restrict__ header;
  float *states;  // null: a command without a workspace, run in the direct form unsplit
  // Direct with splits: the word of each (request, kv-heads, tile) at which its
  // workgroups count themselves, zero before the launch and after it.
  uint32_t *arrived;
  int64_t pool;
  int64_t n_indices;
  int32_t indices_capacity;
  int32_t batch;
  int32_t hq;
  int32_t hkv;
  int32_t group;
  int32_t tile;     // query heads per wave: the columns of its MFMA tiles in use
  int32_t tiles;    // ceil(group / tile)
  int32_t teams;    // balanced: ranges of the virtual list
  int32_t splits;   // direct: workgroups per (request, kv-heads, tile); 1 without states
  int32_t page_rows;
  int32_t head_bytes;  // NHD: 64; HND pages: P * 64
  int32_t row_bytes;   // NHD: Hkv * 64; HND pages: 64
  float scale_log2;
};

// FP32 split state: (max_log2, normalizer, 2 pad, acc[128]), 16-byte aligned.
constexpr int kMx4StateStride = 132;

// Fills the algorithm, teams, tiles, workspace and grid of a plan whose spec,
// max_total_pages and flags are set; `teams_option` as in the plan options.
loom_status_t plan_mx4_decode(loom_paged_decode_plan_info_t *info, uint32_t teams_option, int cus,
                              loom_error_t *err);
// Workgroups of a command of the plan in the direct form, `splits` per (request, kv-heads,
// tile).  0: more than a launch holds (it has fewer than 2^32 threads).
uint64_t mx4_direct_grid(const loom_paged_decode_plan_info_t &info, uint64_t splits);
// Launches the command's kernels; `clear`: the arrival words first.
hipError_t launch_mx4_decode(const loom_paged_decode_plan_info_t &info, const Mx4DecodeArgs &args,
                             bool clear, hipStream_t stream);

}  // namespace loom
