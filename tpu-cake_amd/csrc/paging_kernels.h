// Page allocation on the GPU: request lengths in, page tables, lengths and slot map out.
//
// Mathematics: with have = ceil(len / S), need = ceil((len + new) / S) - have, the inclusive sums
// P(i) of need and T(i) of new over the requests with valid lengths decide admission (P <= free
// pages or need == 0, and T <= max_tokens); a second sum over the admitted gives cu_q_lens.  The
// admitted requests that need pages are a prefix of those that need any, so P(i) - need(i) is also
// the number of pages taken before request i: its j-th new page is free[count - 1 - (P(i) - need(i)) - j].
//
// A step's metadata is tens of bytes a request: launches and dependent loads bound it, not bandwidth.
// So one launch does everything.  Every workgroup writes an entry of the slot map a thread and sums over
// the requests itself, 4 to a thread, until its tokens are covered; workgroup 0 sums over all of them
// and writes the per-request outputs.  Repeating the sums costs a read of 8 N bytes from the L2 for
// each workgroup; a second launch that read them back would cost more than that for N up to thousands.
// The outputs do not overlap the inputs, as the workgroups read the inputs at different times.
//
// Measured: 64 requests 4.4 us (an empty launch takes 2 to 3), 4096 requests and 65 000 tokens 10.4 us.  That is one turn
// of workgroups of 1024 threads, which takes 8.8 us with no token at all, where 1024 requests in workgroups of 256 take
// 5.4 (four barriers over 16 waves instead of 4, and sums over 16 parts a thread); 8192 requests, two turns, take 15.8.
// Tokens add 1.2: the slot map's dependent reads (owner, page).  Release: 3.1 and 4.2 us; trim: 3.7, and 9.8 where 1280
// of 4096 requests give back up to 1186 pages of 16 each.
#pragma once

#include "sparse_common.h"

namespace rpa_sparse {
namespace {

struct AssignParams {
  const int32_t *cached, *fresh;
  int32_t* table;
  const int32_t *free_pages, *free_count;
  int32_t *kv_lens, *cu, *num_seqs, *slots, *positions, *free_out;
  int N, PPS, S, F, max_tokens;
};

constexpr int kItems = 4;  // requests per thread and turn
constexpr int kSmallBatch = 256 * kItems;  // requests that one turn of a 256-thread workgroup sums

template <int THREADS>
__global__ __launch_bounds__(THREADS) void assign_kernel(AssignParams p) {
  constexpr int kWaves = THREADS / 64;
  // the requests with tokens among this workgroup's, at their first token here
  __shared__ int s_req[THREADS], s_first[THREADS], s_page0[THREADS], s_len[THREADS];
  __shared__ Pair s_scan[kWaves];
  __shared__ int s_max[kWaves];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const long long t0 = (long long)blockIdx.x * THREADS;
  const bool lead = blockIdx.x == 0;
  s_req[tid] = -1;
  int count = *p.free_count;
  if (count < 0 || count > p.F) {
    if (lead && tid == 0) flag_error(RPA_SPARSE_ERR_FREE);
    count = count < 0 ? 0 : p.F;
  }
  const long long capacity = (long long)p.PPS * p.S;
  Pair seen = {0, 0};  // needed pages, new tokens of the valid requests so far
  Pair used = {0, 0};  // admitted tokens, pages given
  if (lead && tid == 0) p.cu[0] = 0, *p.num_seqs = p.N;
  for (int c = 0; c < p.N; c += THREADS * kItems) {
    const int base = c + tid * kItems;
    int len[kItems], q[kItems], have[kItems], need[kItems];
    bool valid[kItems];
    Pair sum = {0, 0};
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int i = base + k;
      len[k] = i < p.N ? p.cached[i] : 0;
      q[k] = i < p.N ? p.fresh[i] : 0;
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const long long end = (long long)len[k] + q[k];
      valid[k] = (len[k] >= 0) & (q[k] >= 0) & (end <= capacity);
      have[k] = len[k] >= 0 ? ceil_div(len[k], p.S) : 0;
      need[k] = valid[k] ? ceil_div((int)end, p.S) - have[k] : 0;
      q[k] = valid[k] ? q[k] : 0;
      sum = {sat_add(sum.a, min((uint32_t)need[k], kSumCap)), sat_add(sum.b, min((uint32_t)q[k], kSumCap))};
      if (!valid[k] && lead) flag_error(RPA_SPARSE_ERR_LEN);
    }
    Pair total;
    Pair pre = scan_pairs<kWaves>(sum, total, s_scan);
    pre = {sat_add(seen.a, pre.a), sat_add(seen.b, pre.b)};
    seen = {sat_add(seen.a, total.a), sat_add(seen.b, total.b)};
    int taken[kItems];  // pages needed before the request
    Pair kept = {0, 0};
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      taken[k] = (int)pre.a;
      pre = {sat_add(pre.a, min((uint32_t)need[k], kSumCap)), sat_add(pre.b, min((uint32_t)q[k], kSumCap))};
      // selects, not branches: of `if (!admitted) q[k] = 0, need[k] = 0` with short-circuited conditions clang 22 (ROCm 7.2)
      // makes right IR but, for k = 0, code that clears q and need only where the first two conditions fail and does
      // nothing where the third does: requests turned down for their pages alone kept their tokens
      const bool admitted =
          valid[k] & (pre.b <= (uint32_t)p.max_tokens) & ((need[k] == 0) | (pre.a <= (uint32_t)count));
      q[k] = admitted ? q[k] : 0;
      need[k] = admitted ? need[k] : 0;
      kept = {kept.a + (uint32_t)q[k], kept.b + (uint32_t)need[k]};
    }
    Pair off = scan_pairs<kWaves>(kept, total, s_scan);
    long long first = (long long)used.a + off.a;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int i = base + k;
      if (lead && i < p.N) {
        p.kv_lens[i] = max(len[k], 0) + q[k];
        p.cu[i + 1] = (int)first + q[k];
      }
      if (q[k] > 0 && first < t0 + THREADS && first + q[k] > t0) {
        const int at = first > t0 ? (int)(first - t0) : 0;  // its first token here: no other request's
        s_req[at] = i;
        s_first[at] = (int)first;
        s_page0[at] = count - 1 - taken[k] + have[k];  // page index lp >= have is free[page0 - lp]
        s_len[at] = len[k];
      }
      first += q[k];
    }
    used = {used.a + total.a, used.b + total.b};
    if (!lead && (long long)used.a >= t0 + THREADS) break;  // uniform: the same sums in every thread
  }
  if (lead && tid == 0) *p.free_out = count - (int)used.b;
  __syncthreads();
  // the owner of token t: the last request that starts at or before it
  int at = s_req[tid] >= 0 ? tid : -1;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(at, d);
    if (lane >= d) at = max(at, o);
  }
  if (lane == 63) s_max[wave] = at;
  __syncthreads();
  for (int w = 0; w < wave; ++w) at = max(at, s_max[w]);
  const long long t = t0 + tid;
  if (t >= p.max_tokens) return;
  int slot = -1, pos = 0;
  if (t < used.a && at >= 0) {
    pos = s_len[at] + (int)(t - s_first[at]);
    const int lp = pos / p.S, row = pos % p.S, held = ceil_div(s_len[at], p.S);
    int32_t* entry = p.table + (size_t)s_req[at] * p.PPS + lp;
    const int page = lp < held ? *entry : p.free_pages[s_page0[at] - lp];
    if (row == 0) *entry = page;  // every new page starts with a token of this step
    const long long s = (long long)page * p.S + row;
    if (page >= 0 && s <= 0x7fffffffll)
      slot = (int)s;
    else
      flag_error(RPA_SPARSE_ERR_PAGE);
  }
  p.slots[t] = slot;
  p.positions[t] = pos;
}

struct ReleaseParams {
  const int32_t* cached;
  const uint8_t* finished;
  const int32_t* table;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t *cached_out, *free_out;
  int N, PPS, S, F;
  const int32_t* dropped;  // the trim's: requests longer than `limit` are cut to `budget`
  int32_t* dropped_out;
  int budget, limit;
};

constexpr int kReleaseThreads = 1024;
constexpr int kReleaseSlice = 64;  // requests per workgroup

// A workgroup owns a slice of the requests: it sums the pages that earlier requests give back, then
// copies its own, a wave for each finished request.  The trim (TRIM) gives back the pages of a request past
// its budget's instead: sums and stack are the same.
template <bool TRIM>
__global__ __launch_bounds__(kReleaseThreads) void release_kernel(ReleaseParams p) {
  __shared__ uint32_t s_sum[kReleaseThreads / 64];
  __shared__ uint32_t s_off[kReleaseSlice];
  __shared__ int s_pages[kReleaseSlice];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int i0 = blockIdx.x * kReleaseSlice;
  const long long capacity = (long long)p.PPS * p.S;
  const int first = TRIM ? ceil_div(p.budget, p.S) : 0;  // the first page that goes
  const auto gone = [&](int i, int len) { return TRIM ? len > p.limit : p.finished[i] != 0; };
  const auto pages_of = [&](bool finished, int len) {
    return !finished || len <= 0 ? 0 : max(ceil_div((int)min((long long)len, capacity), p.S) - first, 0);
  };
  uint32_t before = 0;
#pragma unroll 4
  for (int i = tid; i < i0; i += kReleaseThreads) {
    const int len = p.cached[i];
    const bool finished = gone(i, len);  // loaded beside it, not after it
    before = sat_add(before, (uint32_t)pages_of(finished, len));
  }
  for (int d = 32; d; d /= 2) before = sat_add(before, __shfl_xor(before, d));
  if (lane == 0) s_sum[wave] = before;
  __syncthreads();
  if (wave == 0) {
    before = 0;
    for (int w = 0; w < kReleaseThreads / 64; ++w) before = sat_add(before, s_sum[w]);
    const int i = i0 + lane;
    const bool live = i < p.N;
    const int len = live ? p.cached[i] : 0;
    const bool finished = live && gone(i, len);
    const int pages = pages_of(finished, len);
    uint32_t inc = (uint32_t)pages;
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o = __shfl_up(inc, d);
      if (lane >= d) inc = sat_add(inc, o);
    }
    s_pages[lane] = pages;
    s_off[lane] = sat_add(before, inc - (uint32_t)pages);
    if (live) {
      if ((TRIM || finished) && (len < 0 || len > capacity)) flag_error(RPA_SPARSE_ERR_LEN);
      p.cached_out[i] = finished ? (TRIM ? p.budget : 0) : len;
      if (TRIM) p.dropped_out[i] = p.dropped[i] + (finished ? len - p.budget : 0);
    }
    if (i0 + kReleaseSlice >= p.N && lane == 63) {
      const long long end = (long long)max(*p.free_count, 0) + sat_add(before, inc);
      if (end > p.F) flag_error(RPA_SPARSE_ERR_FREE);
      *p.free_out = (int)min(end, (long long)p.F);
    }
  }
  __syncthreads();
  const long long count = max(*p.free_count, 0);
  for (int r = wave; r < kReleaseSlice; r += kReleaseThreads / 64) {
    const int pages = s_pages[r];
    if (pages == 0) continue;
    const int32_t* row = p.table + (size_t)(i0 + r) * p.PPS + first;
    const long long to = count + s_off[r];
    for (int j = lane; j < pages; j += 64)
      if (to + j < p.F) p.free_pages[to + j] = row[j];
  }
}

int check_paging(const rpa_paging_shape_t* s) {
  if (!s) return fail(RPA_E_INVALID, "shape is NULL");
  if (s->num_requests <= 0 || s->pages_per_seq <= 0 || s->page_size <= 0 || s->free_capacity < 0)
    return fail(RPA_E_INVALID, "non-positive dimension in shape");
  if ((long long)s->pages_per_seq * s->page_size > 0x7fffffffll)
    return fail(RPA_E_INVALID, "pages_per_seq * page_size overflows int32");
  if (s->num_requests > kMostIndex || s->pages_per_seq > kMostIndex)
    return fail(RPA_E_UNSUPPORTED, "num_requests and pages_per_seq must be at most 2^31 - 2^16 - 1");
  if (s->free_capacity >= (int)kSumCap || s->max_tokens >= (int)kSumCap || s->max_tokens < 0)
    return fail(RPA_E_INVALID, "free_capacity and max_tokens must be below 2^30");
  return RPA_OK;
}

}  // namespace
}  // namespace rpa_sparse
