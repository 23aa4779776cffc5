// Block tables and slot maps of a paged key/value cache, built on the device from the lengths of the requests.
//
// A request r holds `held[r]` pages (row r of the block table) with room for held[r] * page_size tokens; lens[r]
// tokens are cached and new_lens[r] arrive.  It needs
//     need[r] = max(0, ceil((lens[r] + new_lens[r]) / page_size) - held[r])
// further pages, taken from the top of a free list in request order: with the exclusive prefix sum e[r] of need,
// page j of them is free[count - 1 - (e[r] + j)].  A new token at position p of request r lies in slot
// table[r][p / page_size] * page_size + p % page_size.
//
// One launch, whatever the sizes: every workgroup redoes the two prefix sums over the requests (cumulative tokens,
// pages needed) from the lengths, keeps them in LDS and fills its own share of the token outputs; nothing that one
// workgroup reads is written by another (the new pages' table entries lie behind the held ones, the new counts go to
// buffers of their own), so no workgroup waits for another.  Work: a few dozen bytes per request and 16 per token -
// the launch and three dependent trips to memory are what it costs, not bytes: 6.2 us for 256 requests of one token, 6.8
// for 512 with prompts of up to 611.
#include "mtp_common.h"

namespace {

constexpr int PP_THREADS = 1024;
constexpr int PP_WAVES = PP_THREADS / MTP_WAVE;
constexpr int PP_TOKENS = 1024;        // tokens per workgroup: one per thread
constexpr int PP_MAX_REQUESTS = 4096;  // 8 bytes of LDS per request

struct PlanArgs {
  const int64_t* lens;
  const int64_t* new_lens;
  const int32_t* held;
  int32_t* table;
  const int32_t* free_pages;
  const int32_t* free_count;
  int64_t* slots;
  int64_t* positions;
  int64_t* cu;
  int64_t* kv_lens;
  uint8_t* granted;
  int32_t* held_out;
  int32_t* free_count_out;
  int requests, max_pages, page_size, free_capacity, tokens;
};

__device__ __forceinline__ int64_t wave_scan_incl(int64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t up = __shfl_up((long long)v, o, 64);
    if (lane >= o) v += up;
  }
  return v;
}

// exclusive prefix sum over the workgroup's threads
__device__ __forceinline__ int64_t block_scan_excl(int64_t v, int64_t* sums) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t incl = wave_scan_incl(v);
  __syncthreads();                       // the previous use of `sums` has been read
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int64_t base = 0;
#pragma unroll
  for (int w = 0; w < PP_WAVES; w++)
    if (w < wave) base += sums[w];
  return base + incl - v;
}

__global__ __launch_bounds__(PP_THREADS) void paged_plan_kernel(const PlanArgs p) {
  extern __shared__ int32_t lds[];
  int32_t* cu_l = lds;                   // [R] end of the request's tokens, at most `tokens`
  int32_t* rank_l = lds + p.requests;    // [R] pages handed out before the request's own; -1: refused
  __shared__ int64_t sums[PP_WAVES];
  const int tid = threadIdx.x, R = p.requests;
  const int per = (R + PP_THREADS - 1) / PP_THREADS;   // consecutive requests of this thread
  const int r0 = tid * per < R ? tid * per : R, r1 = r0 + per < R ? r0 + per : R;
  const int64_t room = (int64_t)p.max_pages * p.page_size, cap = p.tokens;
  const int psh = __ffs(p.page_size) - 1;
  int count = *p.free_count;
  count = count < 0 ? 0 : (count > p.free_capacity ? p.free_capacity : count);

  // a request counts at most one token more than the buffers hold: the sums cannot overflow
  auto tokens_of = [&](int r) {
    const int64_t n = p.new_lens[r];
    return n < 0 ? (int64_t)0 : (n > cap ? cap + 1 : n);
  };
  int64_t sum = 0;
  for (int r = r0; r < r1; r++) sum += tokens_of(r);
  int64_t at = block_scan_excl(sum, sums);
  const int64_t at0 = at;
  // pages needed by the requests whose tokens fit the table row and the token buffers; -1: they do not
  auto pages_of = [&](int r, int64_t n, int64_t end) -> int64_t {
    const int64_t len = p.lens[r];
    const int h = p.held[r];
    if (len < 0 || len > room || h < 0 || h > p.max_pages || len + n > room || end > cap) return -1;
    const int64_t want = ((len + n + p.page_size - 1) >> psh) - h;
    return want > 0 ? want : 0;
  };
  sum = 0;
  for (int r = r0; r < r1; r++) {
    const int64_t n = tokens_of(r);
    at += n;
    const int64_t want = pages_of(r, n, at);
    sum += want > 0 ? want : 0;
  }
  int64_t rank = block_scan_excl(sum, sums);
  at = at0;
  const bool lead = blockIdx.x == 0;
  for (int r = r0; r < r1; r++) {
    const int64_t n = tokens_of(r);
    if (lead && r == 0) p.cu[0] = 0;
    at += n;
    const int64_t want = pages_of(r, n, at);
    const bool ok = want == 0 || (want > 0 && rank + want <= count);
    cu_l[r] = (int32_t)(at < cap ? at : cap);
    rank_l[r] = ok ? (int32_t)(want > 0 ? rank : 0) : -1;
    if (lead) {
      const int64_t len = p.lens[r];
      const int h = p.held[r];
      p.cu[r + 1] = at;
      p.kv_lens[r] = ok ? len + n : 0;
      p.granted[r] = ok;
      p.held_out[r] = ok ? h + (int)want : h;
      if (ok && want > 0) {
        // pages that end before the first new token (a table row that lagged behind its length)
        const int first = (int)((len + p.page_size - 1) >> psh);
        for (int j = h; j < first && j < h + (int)want; j++)
          p.table[(int64_t)r * p.max_pages + j] = p.free_pages[count - 1 - (rank + (j - h))];
      }
    }
    if (want > 0) rank += want;
  }
  if (lead) {
    // the granted requests that need pages are the first of those that do: all granted pages are the largest
    // running sum that fits
    int64_t run = rank - sum, taken = 0;
    at = at0;
    for (int r = r0; r < r1; r++) {
      const int64_t n = tokens_of(r);
      at += n;
      const int64_t want = pages_of(r, n, at);
      if (want > 0) {
        run += want;
        if (run <= count) taken += want;
      }
    }
    const int64_t before = block_scan_excl(taken, sums);
    if (tid == PP_THREADS - 1) *p.free_count_out = (int32_t)(count - (before + taken));
    if (R == 0 && tid == 0) p.cu[0] = 0;
  }
  __syncthreads();

  const int64_t t = (int64_t)blockIdx.x * PP_TOKENS + tid;
  if (t >= cap) return;
  int lo = 0, hi = R;                    // first request whose tokens end behind t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu_l[mid] > t) hi = mid; else lo = mid + 1;
  }
  int64_t slot = -1, pos = -1;
  if (lo < R && rank_l[lo] >= 0) {
    const int start = lo ? cu_l[lo - 1] : 0;
    const int64_t len = p.lens[lo];
    const int h = p.held[lo];
    pos = len + (t - start);
    const int j = (int)(pos >> psh);
    int32_t* entry = p.table + (int64_t)lo * p.max_pages + j;
    int page;
    if (j < h) {
      page = *entry;
    } else {
      page = p.free_pages[count - 1 - (rank_l[lo] + (j - h))];
      if ((pos & (p.page_size - 1)) == 0) *entry = page;   // the page's first token writes the table
    }
    slot = ((int64_t)page << psh) + (pos & (p.page_size - 1));
  }
  p.slots[t] = slot;
  p.positions[t] = pos;
}

// Pages of finished requests go back on the free list, in request order and, within a request, in table order.
// One workgroup: a step releases a handful of requests.  16 requests of about 300 pages: 15 us.
__global__ __launch_bounds__(PP_THREADS) void paged_release_kernel(const uint8_t* finished, int32_t* held,
                                                                  const int32_t* table, int32_t* free_pages,
                                                                  int32_t* free_count, int requests, int max_pages,
                                                                  int free_capacity) {
  extern __shared__ int32_t lds[];
  int32_t* rank_l = lds;                 // [R] place of the request's first page behind the list, -1: keeps its pages
  __shared__ int64_t sums[PP_WAVES];
  const int tid = threadIdx.x, R = requests;
  const int per = (R + PP_THREADS - 1) / PP_THREADS;
  const int r0 = tid * per < R ? tid * per : R, r1 = r0 + per < R ? r0 + per : R;
  int count = *free_count;
  count = count < 0 ? 0 : (count > free_capacity ? free_capacity : count);
  auto pages_of = [&](int r) {
    const int h = held[r];
    return finished[r] && h > 0 ? (h < max_pages ? h : max_pages) : 0;
  };
  int64_t sum = 0;
  for (int r = r0; r < r1; r++) sum += pages_of(r);
  int64_t rank = block_scan_excl(sum, sums), kept = 0;
  for (int r = r0; r < r1; r++) {
    const int n = pages_of(r);
    // a list too short for its pages (they were never taken from it) keeps them in the table
    const bool fits = n > 0 && count + rank + n <= free_capacity;
    rank_l[r] = fits ? (int32_t)rank : -1;
    if (fits) kept += n;
    rank += n;
  }
  const int64_t before = block_scan_excl(kept, sums);   // its barriers also publish rank_l
  if (tid == PP_THREADS - 1) *free_count = (int32_t)(count + before + kept);
  for (int r = tid >> 6; r < R; r += PP_WAVES) {        // a wave copies a request's pages
    if (rank_l[r] < 0) continue;
    const int n = pages_of(r);
    for (int j = tid & 63; j < n; j += 64) free_pages[count + rank_l[r] + j] = table[(int64_t)r * max_pages + j];
    __builtin_amdgcn_wave_barrier();
    if ((tid & 63) == 0) held[r] = 0;
  }
}

int check_sizes(const char* what, int64_t requests, int64_t max_pages, int64_t free_capacity) {
  MTP_REQUIRE(requests >= 0 && requests <= PP_MAX_REQUESTS, MTP_EUNSUPPORTED, "%s: %lld requests (at most %d)", what,
              (long long)requests, PP_MAX_REQUESTS);
  MTP_REQUIRE(max_pages > 0 && max_pages <= 0x7fffffffll && free_capacity >= 0 && free_capacity <= 0x7fffffffll,
              MTP_EINVAL, "%s: max_pages=%lld free list of %lld", what, (long long)max_pages, (long long)free_capacity);
  return MTP_OK;
}

}  // namespace

extern "C" int mtp_paged_plan(const int64_t* lens, const int64_t* new_lens, const int32_t* held, int32_t* block_tables,
                              const int32_t* free_pages, const int32_t* free_count, int64_t* slots, int64_t* positions,
                              int64_t* cu, int64_t* kv_lens, uint8_t* granted, int32_t* held_out,
                              int32_t* free_count_out, int64_t requests, int64_t max_pages, int64_t page_size,
                              int64_t free_capacity, int64_t tokens, void* stream) {
  const int rc = check_sizes("paged_plan", requests, max_pages, free_capacity);
  if (rc) return rc;
  MTP_REQUIRE(page_size >= 1 && (page_size & (page_size - 1)) == 0 && max_pages <= 0x7fffffffll / page_size, MTP_EINVAL,
              "paged_plan: page_size=%lld (a power of two), %lld pages a row", (long long)page_size,
              (long long)max_pages);
  MTP_REQUIRE(tokens >= 0 && tokens <= 0x7fffffffll, MTP_EINVAL, "paged_plan: tokens=%lld", (long long)tokens);
  MTP_REQUIRE(cu && free_count && free_count_out && (free_pages || free_capacity == 0), MTP_EINVAL,
              "paged_plan: null pointer");
  MTP_REQUIRE(requests == 0 || (lens && new_lens && held && block_tables && kv_lens && granted && held_out), MTP_EINVAL,
              "paged_plan: null pointer");
  MTP_REQUIRE(tokens == 0 || (slots && positions), MTP_EINVAL, "paged_plan: null pointer");
  MTP_REQUIRE(free_count_out != free_count && (requests == 0 || held_out != held), MTP_EINVAL,
              "paged_plan: the new counts must not share memory with the old ones");
  PlanArgs a = {lens, new_lens, held, block_tables, free_pages, free_count, slots, positions, cu, kv_lens, granted,
                held_out, free_count_out, (int)requests, (int)max_pages, (int)page_size, (int)free_capacity,
                (int)tokens};
  const unsigned grid = (unsigned)(tokens ? (tokens + PP_TOKENS - 1) / PP_TOKENS : 1);
  hipLaunchKernelGGL(paged_plan_kernel, dim3(grid), dim3(PP_THREADS), (size_t)requests * 8,
                     static_cast<hipStream_t>(stream), a);
  MTP_CHECK_LAUNCH("paged_plan");
  return MTP_OK;
}

extern "C" int mtp_paged_release(const uint8_t* finished, int32_t* held, const int32_t* block_tables,
                                 int32_t* free_pages, int32_t* free_count, int64_t requests, int64_t max_pages,
                                 int64_t free_capacity, void* stream) {
  const int rc = check_sizes("paged_release", requests, max_pages, free_capacity);
  if (rc) return rc;
  if (requests == 0) return MTP_OK;
  MTP_REQUIRE(finished && held && block_tables && free_pages && free_count, MTP_EINVAL, "paged_release: null pointer");
  hipLaunchKernelGGL(paged_release_kernel, dim3(1), dim3(PP_THREADS), (size_t)requests * 4,
                     static_cast<hipStream_t>(stream), finished, held, block_tables, free_pages, free_count,
                     (int)requests, (int)max_pages, (int)free_capacity);
  MTP_CHECK_LAUNCH("paged_release");
  return MTP_OK;
}
