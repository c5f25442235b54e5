// Reading MXFP4 pages back as BF16 rows for gfx950 (no reference counterpart).
//
// out[kv_indptr[r] + i] = codes * 2^(scale - 127) of token kv_start[r] + i of
// request r, for K and V and every kv-head: the contiguous rows that a ragged
// prefill reads.
//
// Each head's row is 68 bytes read and 256 written, twice (K and V), with no
// arithmetic but the conversion, so the kernel is bound by the memory rate, four
// fifths of it writes.  A workgroup takes some output rows (64 head rows, or one
// output row): its first wave finds their requests and pages, one row per lane,
// from the table words of 64 requests in its registers (two round trips before the
// rows' own for batches below 64, else a search first), then 16 lanes per head row
// load 4 code bytes each and store 16 bytes, K and V together, the heads of a row
// contiguous.  The stores are streamed past L2: plain ones, whose lines L2 writes
// back in another order, took 41 us instead of 27.1 (31.5k rows of 8 kv-heads, HND
// pages of 64: 6.0 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_device.hpp"
#include "loom_internal.hpp"

using loom::fail;
using namespace loom_dev;

namespace {

constexpr int kReadThreads = 256;
constexpr int kReadMaxRows = 64;  // output rows per workgroup: at most one per lane
constexpr uint64_t kReadMaxHeads = 4096;
// Head rows per workgroup, and how many of them each 16 lanes have in flight.
// Measured with 16 to 256 head rows and 1 to 4 in flight: 64 are within 4% of the
// best from 8k rows of 8 kv-heads (8.3 us) to 31.5k (27.1 us); 256 take 8 us where
// 64 take 4.5 (300 rows of 32 kv-heads), 16 lose 5% of the large ones.  Four in
// flight against one: 64 scattered rows of 8 kv-heads and their append 11.6 and
// 11.8 us, about 1000 14.4 and 14.8.
constexpr int kReadItems = 64;
constexpr int kReadDepth = 4;

struct ReadArgs {
  const uint8_t *k;
  const uint8_t *v;
  const uint8_t *k_mx;
  const uint8_t *v_mx;
  const int32_t *indptr;
  const int32_t *indices;
  const int32_t *last;
  const int32_t *kv_indptr;
  const int32_t *kv_start;  // null: every request from its first token on
  uint16_t *k_out;
  uint16_t *v_out;
  int64_t pool;
  int64_t n_indices;
  int32_t indices_capacity;
  int32_t batch;
  int32_t hkv;
  int32_t nnz;
  int32_t page_rows;
  int32_t head_bytes;  // NHD: 64; HND pages: page_rows * 64
  int32_t row_bytes;   // NHD: hkv * 64; HND pages: 64
  int32_t rows;        // output rows per workgroup
  uint32_t hkv_inv;    // 2^32 / hkv, rounded up
};

// Largest request r <= batch with kv_indptr[r] <= t, by one wave: 64 entries a
// round trip.  (kv_indptr[0] = 0 <= t.)  Wave-uniform.
__device__ __forceinline__ int request_of(const ReadArgs &a, int t, int lane) {
  int lo = 0, n = a.batch + 1;  // the answer is one of [lo, lo + n)
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int at = lane * step;
    const bool le = at < n && a.kv_indptr[lo + at] <= t;
    const int k = __builtin_popcountll(__builtin_amdgcn_ballot_w64(le));
    const int skip = max(k - 1, 0) * step;  // entries 0 .. k - 1 of this round are <= t
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// One head row's part of a lane: 8 codes and their scale byte, of K and of V.
struct Part {
  uint32_t k, v, ks, vs;
};

__global__ __launch_bounds__(kReadThreads) void paged_kv_read_kernel(ReadArgs a) {
  __shared__ int32_t s_page[kReadMaxRows], s_off[kReadMaxRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int t0 = (int)blockIdx.x * a.rows;
  const int rows = min(a.rows, a.nnz - t0);
  if (tid < 64) {
    // Lane l holds the table words of request r0 + l, and finds the place of row l.
    const int r0 = a.batch < 64 ? 0 : uni(request_of(a, t0, lane));
    const int at = min(r0 + lane, a.batch), in = min(at, a.batch - 1);
    const int32_t ip0 = a.indptr[0], ipB = a.indptr[a.batch];
    const int32_t kv0 = a.kv_indptr[0], kvB = a.kv_indptr[a.batch];
    const int32_t w_kv = a.kv_indptr[at], w_ip = a.indptr[at];
    const int32_t w_last = a.last[in], w_start = a.kv_start ? a.kv_start[in] : 0;
    const bool ok = ip0 == 0 && ipB >= 0 && kv0 == 0 && kvB >= 0 && kvB <= a.nnz &&
                    (a.indices_capacity ? (int64_t)ipB <= a.n_indices : (int64_t)ipB == a.n_indices);
    const int t = t0 + lane;
    // the last of the 64 requests that starts at or before row t
    int k = 0;
#pragma unroll
    for (int step = 32; step; step >>= 1)
      if (__shfl(w_kv, k + step, 64) <= t) k += step;
    const int k1 = min(k + 1, 63);
    int32_t st = __shfl(w_ip, k, 64), en = __shfl(w_ip, k1, 64), tl = __shfl(w_last, k, 64);
    int32_t b = __shfl(w_kv, k, 64), e = __shfl(w_kv, k1, 64), start = __shfl(w_start, k, 64);
    int r = min(r0 + k, a.batch);
    int page = -1, off = 0;
    if (ok && lane < rows && r < a.batch) {
      if (k == 63) {  // past 62 short requests: searched, and read, from the table
        int n = a.batch + 1 - r;  // the answer is one of [r, r + n)
        while (n > 1) {
          const int half = n / 2;
          const bool le = a.kv_indptr[r + half] <= t;
          r += le ? half : 0;
          n = le ? n - half : half;
        }
        const int rr = min(r, a.batch - 1);
        st = a.indptr[rr], en = a.indptr[rr + 1], tl = a.last[rr];
        b = a.kv_indptr[rr], e = a.kv_indptr[rr + 1];
        start = a.kv_start ? a.kv_start[rr] : 0;
      }
      const int64_t kv_len = ((int64_t)en - st - 1) * a.page_rows + tl;
      if (st >= 0 && en > st && en <= ipB && tl >= 1 && tl <= a.page_rows && b >= 0 && b <= t &&
          t < e && start >= 0 && (int64_t)start + (e - b) <= kv_len) {
        const uint32_t p = (uint32_t)start + (uint32_t)(t - b);
        const int32_t idx = a.indices[st + (int)(p / (uint32_t)a.page_rows)];
        if (idx >= 0 && (int64_t)idx < a.pool) {
          page = idx;
          off = (int)(p % (uint32_t)a.page_rows);
        }
      }
    }
    s_page[lane] = page;
    s_off[lane] = off;
  }
  __syncthreads();
  const int c = tid & 15;
  const int64_t page_bytes = (int64_t)a.page_rows * a.hkv * 64;
  const int items = rows * a.hkv;
  constexpr int kStep = kReadThreads / 16;
#pragma unroll 1
  for (int i0 = tid >> 4; i0 < items; i0 += kStep * kReadDepth) {
    Part part[kReadDepth];
    int64_t out[kReadDepth];
    // Loads without branches: rows that are not written read some row of the pool.  (A
    // branch round them makes the compiler wait for one turn's before the next.)
#pragma unroll
    for (int u = 0; u < kReadDepth; ++u) {
      const int i = min(i0 + u * kStep, items - 1);
      const int j = a.hkv == 1 ? i : (int)__umulhi((uint32_t)i, a.hkv_inv);
      const int page = s_page[j], off = s_off[j], h = i - j * a.hkv;
      const int64_t pg = max(page, 0);
      out[u] = page < 0 || i0 + u * kStep >= items
                   ? -1
                   : ((int64_t)(t0 + j) * a.hkv + h) * 128 + c * 8;
      const int64_t at =
          pg * page_bytes + (int64_t)h * a.head_bytes + (int64_t)off * a.row_bytes + c * 4;
      const int64_t sc = (((pg * a.hkv + h) * a.page_rows + off) << 2) + (c >> 2);
      part[u] = {*reinterpret_cast<const uint32_t *>(a.k + at),
                 *reinterpret_cast<const uint32_t *>(a.v + at), a.k_mx[sc], a.v_mx[sc]};
    }
#pragma unroll
    for (int u = 0; u < kReadDepth; ++u)
      if (out[u] >= 0) {
        __builtin_nontemporal_store(mx4x8_to_bf16x8(part[u].k, part[u].ks << 23),
                                    reinterpret_cast<u32x4 *>(a.k_out + out[u]));
        __builtin_nontemporal_store(mx4x8_to_bf16x8(part[u].v, part[u].vs << 23),
                                    reinterpret_cast<u32x4 *>(a.v_out + out[u]));
      }
  }
}

}  // namespace

struct loom_paged_kv_read_plan {
  loom_paged_kv_read_spec_t spec{};
  uint32_t flags = 0;
};

extern "C" {

loom_status_t loom_prefill_provider_plan_paged_kv_read(const loom_prefill_provider_t *provider,
                                                       const loom_paged_kv_read_spec_t *spec,
                                                       uint32_t flags,
                                                       loom_paged_kv_read_plan_t **out,
                                                       loom_error_t *err) {
  if (!provider || !spec || !out) return fail(err, LOOM_NULL_ARGUMENT, "provider");
  if (flags & ~LOOM_PLAN_PAGE_INDICES_CAPACITY)
    return fail(err, LOOM_PLAN_INVALID_OPTION, "flags", flags);
  loom_paged_kv_read_spec_t s;
  const loom_status_t rc = loom_paged_kv_read_spec_new(&spec->paged, spec->nnz_kv, &s, err);
  if (rc) return rc;
  // requests and heads are indexed in 32 bits
  if (s.paged.batch_size >= (uint64_t)INT32_MAX)
    return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "K/V read batch", s.paged.batch_size);
  // (head rows of a workgroup are divided by the heads by a 32-bit reciprocal)
  if (s.paged.num_kv_heads > kReadMaxHeads)
    return fail(err, LOOM_PLAN_STATE_COUNT_OUT_OF_RANGE, "K/V read heads", s.paged.num_kv_heads);
  auto *p = new loom_paged_kv_read_plan;
  p->spec = s;
  p->flags = flags;
  *out = p;
  return loom::ok(err);
}

void loom_paged_kv_read_plan_free(loom_paged_kv_read_plan_t *p) { delete p; }

loom_status_t loom_paged_kv_read_enqueue(const loom_paged_kv_read_plan_t *plan,
                                         loom_command_scope_t *scope,
                                         const loom_paged_kv_read_args_t *args,
                                         loom_error_t *err) {
  if (!plan || !scope || !args) return fail(err, LOOM_NULL_ARGUMENT, "plan");
  const loom_paged_decode_spec_t &s = plan->spec.paged;
  const loom::OperandSpec ops[11] = {
      {"K_pages", LOOM_DTYPE_U8, false},      {"V_pages", LOOM_DTYPE_U8, false},
      {"K_scales", LOOM_DTYPE_U8, false},     {"V_scales", LOOM_DTYPE_U8, false},
      {"page_indptr", LOOM_DTYPE_I32, false}, {"page_indices", LOOM_DTYPE_I32, false},
      {"last_page_len", LOOM_DTYPE_I32, false}, {"kv_indptr", LOOM_DTYPE_I32, false},
      {"K", LOOM_DTYPE_BF16, true},           {"V", LOOM_DTYPE_BF16, true},
      {"kv_start", LOOM_DTYPE_I32, false}};
  const loom_handle_t hs[11] = {args->key_pages,    args->value_pages,  args->key_scales,
                                args->value_scales, args->page_indptr,  args->page_indices,
                                args->last_page_len, args->kv_indptr,   args->key,
                                args->value,        args->kv_start};
  const int n = args->kv_start.set_id != 0 ? 11 : 10;
  const loom::Lease *l[11];
  loom_status_t rc = loom::resolve_command(scope, hs, ops, n, l, err);
  if (rc) return rc;
  const uint64_t page_rows = s.page_size ? s.page_size : loom::kPageSize;
  const uint64_t rows = s.max_num_pages * page_rows * s.num_kv_heads;
  const uint64_t on = plan->spec.nnz_kv * s.num_kv_heads * loom::kHeadDim;
  const uint64_t want[11] = {rows * LOOM_MXFP4_ROW_BYTES,
                             rows * LOOM_MXFP4_ROW_BYTES,
                             rows * LOOM_MXFP4_ROW_SCALES,
                             rows * LOOM_MXFP4_ROW_SCALES,
                             s.batch_size + 1,
                             0,
                             s.batch_size,
                             s.batch_size + 1,
                             on,
                             on,
                             s.batch_size};
  for (int i = 0; i < n; ++i) {
    if (i == 5) {
      if (l[5]->numel < s.batch_size)
        return fail(err, LOOM_ENQ_PAGE_INDICES_TOO_SHORT, nullptr, s.batch_size, l[5]->numel);
      continue;
    }
    if (l[i]->numel != want[i])
      return fail(err, LOOM_ENQ_LENGTH_MISMATCH, ops[i].name, want[i], l[i]->numel);
  }
  // 4-byte boundaries, as for the other commands over pages (16-byte accesses
  // need no more on gfx950).
  for (int i : {0, 1, 2, 3, 8, 9})
    if (l[i]->ptr % 4 != 0)
      return fail(err, LOOM_ENQ_MISALIGNED_BUFFER, ops[i].name, (int64_t)l[i]->ptr, 4);
  ReadArgs a{};
  a.k = (const uint8_t *)l[0]->ptr;
  a.v = (const uint8_t *)l[1]->ptr;
  a.k_mx = (const uint8_t *)l[2]->ptr;
  a.v_mx = (const uint8_t *)l[3]->ptr;
  a.indptr = (const int32_t *)l[4]->ptr;
  a.indices = (const int32_t *)l[5]->ptr;
  a.last = (const int32_t *)l[6]->ptr;
  a.kv_indptr = (const int32_t *)l[7]->ptr;
  a.kv_start = n == 11 ? (const int32_t *)l[10]->ptr : nullptr;
  a.k_out = (uint16_t *)l[8]->ptr;
  a.v_out = (uint16_t *)l[9]->ptr;
  a.pool = (int64_t)s.max_num_pages;
  a.n_indices = (int64_t)l[5]->numel;
  a.indices_capacity = (plan->flags & LOOM_PLAN_PAGE_INDICES_CAPACITY) ? 1 : 0;
  a.batch = (int32_t)s.batch_size;
  a.hkv = (int32_t)s.num_kv_heads;
  a.nnz = (int32_t)plan->spec.nnz_kv;
  a.page_rows = (int32_t)page_rows;
  const bool hnd = s.kv_layout == LOOM_KV_LAYOUT_HND;
  a.head_bytes = hnd ? a.page_rows * 64 : 64;
  a.row_bytes = hnd ? 64 : a.hkv * 64;
  a.rows = std::min(std::max(kReadItems / a.hkv, 1), kReadMaxRows);
  a.hkv_inv = (uint32_t)(((1ull << 32) + a.hkv - 1) / a.hkv);  // (hkv = 1: not used)
  const unsigned grid = (unsigned)((plan->spec.nnz_kv + a.rows - 1) / a.rows);
  hipLaunchKernelGGL(paged_kv_read_kernel, dim3(grid), dim3(kReadThreads), 0, scope->queue->stream,
                     a);
  return loom::record_launch(scope, hipGetLastError(), err);
}

}  // extern "C"
