// Causal grouped-query attention of the new tokens of many requests over a paged key/value cache, for gfx950: one
// operator for single tokens, drafted tokens and prompts, in any mix.
//
//   out[i,h,:] = sum_t p_t V[t,:] / sum_t p_t,   p_t = exp(scale q[i,h,:] . K[t,:] - max),   t <= kv_len - n + i
//
// in one pass over the keys and values with the running maximum m and sum l of a softmax, in fp32.
//
// Rows.  The g = n_q / n_kv query heads of a key head read the same keys: the rows of a tile are (token, head of the
// group) pairs, token major, so a tile of one request and one key head has n g rows whatever n is, and reads each key
// once for all of them.
//
// Products.  S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16: a lane then owns one row (column lane % 32 of the
// result), the maximum and the sum of a row are in-lane plus one exchange with lane ^ 32, and the 16 scores of a lane
// already sit where the second product takes its right operand, in the k order  4h + {0..3}, 8 + 4h + {0..3}  of each
// 16 tokens (h = lane / 32) - the transposed reads of V follow the same order, so P never moves.
//
// Keys and values go global -> LDS by DMA in blocks of 16 tokens (a page holds at least 16): the block's page id is a
// scalar load, its 64-bit address the base of a buffer resource whose range ends at the request's last token, so
// tokens behind it read as zeros whatever lies there, and an unknown page reads as zeros too.  16-byte chunk c of token
// t sits at chunk position c ^ swz(t) of its row: the fragment reads of K (8 rows, one chunk) and the transposed reads
// of V (4 rows, two neighbouring chunks) then fall into different banks.
//
// Work.  The key/value range of every (request, key head, tile) is counted in units (32 or 64 tokens) plus a constant
// for the tile's start, and the whole sequence of units is dealt to the workgroups in equal runs: lengths may differ by
// any factor, a long context is split over as many workgroups as its share, short ones share a workgroup, and nothing
// depends on what the host knows of the lengths.  Every workgroup finds its run by itself (a prefix sum over the
// requests).  A tile that is cut leaves partial results (O, m, l) in the workspace; the workgroup that delivers last
// merges them in order, so the result does not depend on which one that is.
//
// Two kernels, chosen by the most rows a tile can have:
//   narrow  up to 32 rows, bound by HBM: the waves of a workgroup take turns with the units of its run, each with a ring
//           of LDS slots of its own and no barrier in the loop, and are merged at the end;
//   wide    256 rows, 32 per wave, bound by the matrix cores: the waves share each unit's keys and values.
// With 32 + 8 heads of 128: decode of 64 requests of 200 to 8192 tokens 95 us for 575 MB (6.0 TB/s; read-only streams
// reach 7.0), one token of a request of 130001 88 us (6.0 TB/s), five tokens of 32 requests 60 us (5.0 TB/s), prompts of
// 1900 to 4100 tokens behind up to 5000 562 us for 556 GFLOP (0.99 PFLOP/s; large products reach 1.43): the waves of a
// workgroup meet at a barrier every 64 tokens, so the two of a SIMD multiply and exponentiate at the same time.
#include "gemm_bf16_kernel.h"

namespace {

constexpr int AP_PAGE_MIN = 16;      // tokens per DMA block
// A tile's start (first keys under way, queries, merge, output) in units, as runs are dealt.  Narrow with 2, 8 and 16:
// decode of 64 requests 110, 100 and 102 us, drafts of 32 requests 68, 65 and 66.  Wide with 1, 4 and 12: prompts of 4
// requests 675, 636 and 660 us, 24 tokens of 32 requests 91, 84 and 88.
constexpr int AP_START_NARROW = 8;
constexpr int AP_START_WIDE = 4;
constexpr int64_t AP_COUNTER_BYTES = 4096;     // arrival counters: 4 bytes a workgroup at the head of the workspace

struct PagedArgs {
  const uint16_t* q;         // [T, n_q, D]
  const uint16_t* k;         // [n_pages, n_kv, page_size, D]
  const uint16_t* v;
  const int32_t* table;      // [requests, max_pages]
  const int64_t* cu;         // [requests + 1]
  const int64_t* kv_lens;    // [requests]
  uint16_t* out;
  float* part;               // [2 wgs] partial tiles
  int32_t* arrived;          // [wgs] zero between launches
  int64_t max_pages;
  int T, requests, n_q, n_kv, group, page_shift, n_pages, room, wgs, min_units;
  float scale_log2e;
};

// uniform, read-only data: scalar loads
template <typename T> __device__ __forceinline__ T scalar_load(const T* p) {
  return *(const T __attribute__((address_space(4)))*)(uintptr_t)p;
}

// a value that is the same in every lane, in scalar registers
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// Partial results in the workspace: accesses at device scope (sc1), served at the level all XCDs share
struct Partials {
  static constexpr int SC1 = 16;
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ explicit Partials(float* base) : r(__builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7fffffff, 0x00020000)) {}
  __device__ __forceinline__ void store4(int at, f32x4_t v) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), r, at * 4, 0, SC1);
  }
  __device__ __forceinline__ void store2(int at, float a, float b) const {
    __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(a), __float_as_uint(b)}, r, at * 4, 0, SC1);
  }
  __device__ __forceinline__ f32x4_t load4(int at) const {
    return __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, at * 4, 0, SC1));
  }
  __device__ __forceinline__ f32x2_t load2(int at) const {
    return __builtin_bit_cast(f32x2_t, __builtin_amdgcn_raw_buffer_load_b64(r, at * 4, 0, SC1));
  }
};

template <int N> __device__ __forceinline__ void wait_vm_at_most() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// ---- the sequence of units -----------------------------------------------------------------------------
struct Request {
  int t0, n, kv;             // first row's token, new tokens, cached tokens with them
};
__device__ __forceinline__ int clamp64(int64_t v, int hi) { return v < 0 ? 0 : v > hi ? hi : (int)v; }
__device__ __forceinline__ Request request_of(const PagedArgs& p, int r) {
  const int a = clamp64(scalar_load(p.cu + r), p.T), b = clamp64(scalar_load(p.cu + r + 1), p.T);
  return Request{a, b > a ? b - a : 0, clamp64(scalar_load(p.kv_lens + r), p.room)};
}

// Walks the tiles of a request: tokens that the tile's last row may see, in units of TK.
template <int BM, int TK>
struct Tiles {
  int e0, n, kv, whole, rest, tok, frac, group;
  __device__ __forceinline__ Tiles(const Request& q, int g) {
    e0 = q.kv - q.n;
    n = q.n;
    kv = q.kv;
    group = g;
    whole = BM / g;
    rest = BM % g;
    tok = frac = 0;
  }
  __device__ __forceinline__ int next() {     // units of the next tile
    tok += whole;
    frac += rest;
    if (frac >= group) {
      frac -= group;
      tok++;
    }
    const int upto = tok + (frac > 0 ? 1 : 0);
    const int end = e0 + (upto < n ? upto : n);
    return end <= 0 ? 0 : (end - 1) / TK + 1;      // end + TK - 1 may pass 2^31
  }
};

// quotient of two numbers of 0 or more, with the short division where they fit
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((uint64_t)(a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

struct Run {                 // a workgroup's run of the sequence, and where it starts
  int64_t x, hi, total;      // cost positions
  int wgs;                   // workgroups that have a run
  int r;
  int64_t head_cost, off;    // cost of one key head of request r, position inside the request
};

template <int BM, int TK, int THREADS, int AP_START>
__device__ __forceinline__ bool find_run(const PagedArgs& p, int w, Run& run) {
  __shared__ int64_t sums[THREADS / 64];
  __shared__ int64_t found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (p.requests + THREADS - 1) / THREADS;
  const int r0 = tid * per < p.requests ? tid * per : p.requests;
  const int r1 = r0 + per < p.requests ? r0 + per : p.requests;
  auto cost_of = [&](int r) -> int64_t {      // of one key head
    const Request q = request_of(p, r);
    const int tiles = (int)(((int64_t)q.n * p.group + BM - 1) / BM);
    Tiles<BM, TK> walk(q, p.group);
    int64_t c = 0;
    for (int j = 0; j < tiles; j++) c += walk.next() + AP_START;
    return c;
  };
  int64_t own = 0;
  for (int r = r0; r < r1; r++) own += cost_of(r);
  int64_t incl = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t up = __shfl_up((long long)incl, o, 64);
    if (lane >= o) incl += up;
  }
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int64_t base = 0, total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; i++) {
    if (i < wave) base += sums[i];
    total += sums[i];
  }
  total = uniform(total * p.n_kv);
  int64_t at = (base + incl - own) * p.n_kv;
  const int64_t most = (total + p.min_units - 1) / p.min_units;
  const int wgs = most < p.wgs ? (int)most : p.wgs;
  if (w >= wgs) return false;                 // the same for the whole workgroup
  const int64_t lo = quotient(total * w, wgs);
  if (at <= lo && lo < at + own * p.n_kv) {
    for (int r = r0; r < r1; r++) {
      const int64_t c = cost_of(r);
      if (lo < at + c * p.n_kv) {
        found[0] = r;
        found[1] = c;
        found[2] = lo - at;
        break;
      }
      at += c * p.n_kv;
    }
  }
  __syncthreads();
  run.x = lo;
  run.hi = quotient(total * (w + 1), wgs);
  run.total = total;
  run.wgs = wgs;
  run.r = __builtin_amdgcn_readfirstlane((int)found[0]);
  run.head_cost = uniform(found[1]);
  run.off = uniform(found[2]);
  return true;
}
// workgroup whose run holds position x: the largest w with floor(total w / wgs) <= x
__device__ __forceinline__ int wg_of(const Run& run, int64_t x) { return (int)quotient((x + 1) * run.wgs - 1, run.total); }

// ---- one wave's share of the products -----------------------------------------------------------------
// position of a 16-byte chunk in its token's row of the LDS tile
// (64 banks of 4 bytes: a b128 read serves 16 lanes a cycle - 16 tokens, one chunk -, a transposed b64 read 32 lanes -
// 4 tokens, 4 chunks.  Both want 16 different chunk places; with 64 dims two tokens share the 256 bytes.)
template <int D> __device__ __forceinline__ int swz(int t) {
  return D == 128 ? ((t & 3) << 2) | ((t >> 2) & 3) : (((t >> 1) & 1) << 2) | ((t >> 2) & 3);
}

// maximum over a lane and lane ^ 32
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// place of element d of a row in the merge area
template <int D> __device__ __forceinline__ int merge_at(int row, int d) { return row * D + (d ^ ((row & 7) << 2)); }

template <int D, bool F16, int NB>
struct Wave {
  using X = X16<F16>;
  static constexpr int KS = D / 16, DT = D / 32, ROW = D * 2;
  // Probabilities are held as p 2^SHIFT in the tensors' type; l and O carry the factor alike, so it leaves with their
  // quotient.  bf16 has the exponents of fp32.  Half precision rounds below 2^-14 to whole multiples of 2^-24: without a
  // factor all weights under 2^-25 of the maximum would be lost, and a long flat tail with them (130k keys at 2^-25.1
  // are 0.36 % of the mass).  With 2^11 they are kept down to 2^-36 (n keys: 2^-36 n of the largest value), and
  // LAZY + SHIFT = 15 stays below the largest half, 2^16: the maximum may lag behind by LAZY binary orders.  Times of f16
  // decode of 64 requests and of prompts: 102 and 665 us, with LAZY 8 and SHIFT 7 102 and 669, with 2 and 13 101 and 666.
  static constexpr float LAZY = F16 ? 4.0f : 8.0f, SHIFT = F16 ? 11.0f : 0.0f;
  bf16x8_t qf[KS];
  f32x16_t o[DT];
  float m, l;
  int lim;                   // first token the lane's row does not see
  u32x4_t pf[2 * NB];        // probabilities of the unit, as the second product's operand

  // rows row0 + lane % 32 of the tile, of which `rows` exist
  __device__ __forceinline__ void start(const PagedArgs& p, const Request& q, int kvh, int row0, int rows) {
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    int row = row0 + c;
    if (row >= rows) row = rows - 1;          // a copy of the last row, never stored
    const int tok = row / p.group, g = row - tok * p.group;
    const uint16_t* src = p.q + ((int64_t)(q.t0 + tok) * p.n_q + kvh * p.group + g) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; s++) qf[s] = *reinterpret_cast<const bf16x8_t*>(src + 16 * s);
    // the queries are waited for here, once: left to their first use, the wait would sit in the loop and drain the
    // DMA in flight at every step
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(qf[s]));
    lim = q.kv - q.n + tok + 1;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[dt][i] = 0.0f;
  }

  // scores of the unit's keys (LDS tile `ks`, first token tok0), running maximum and sum, probabilities
  template <bool MASK> __device__ __forceinline__ void scores(const char* ks, int tok0, float c) {
    const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
    f32x16_t s[NB];
    bf16x8_t a[KS][NB];
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int b = 0; b < NB; b++)
        a[k][b] = *reinterpret_cast<const bf16x8_t*>(ks + (32 * b + row) * ROW + (((2 * k + h) ^ swz<D>(row)) << 4));
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 16; i++) s[b][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int b = 0; b < NB; b++)        // neighbouring products add to different blocks: none waits for the one before
        s[b] = X::mfma32(a[k][b], qf[k], s[b]);
    // fragments are read KS products ahead
    __builtin_amdgcn_sched_group_barrier(SG_DS_RD, KS, 0);
#pragma unroll
    for (int i = 0; i < (NB - 1) * KS; i++) {
      __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 0);
      __builtin_amdgcn_sched_group_barrier(SG_DS_RD, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(SG_MFMA, KS, 0);
    if (MASK) {
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (tok0 + 32 * b + 8 * (i >> 2) + 4 * h + (i & 3) >= lim) s[b][i] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[b][i]);
    mx = half_max(mx);
    // The maximum only has to keep the exponentials in range: it is moved (and O and l rescaled) when a row's has
    // grown by more than LAZY binary orders, not at every step.  A row that has seen nothing yet stays at -inf.
    if (__any((mx - m) * c > LAZY)) {
      const float mn = fmaxf(m, mx);
      const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[dt][i] *= f;
    }
    const float mc = SHIFT - (m == -INFINITY ? 0.0f : m * c);
    // the sum takes the probabilities as the second product sees them, rounded: half as many instructions (a dot
    // product with ones adds two), and numerator and denominator then share each rounding
#pragma unroll
    for (int b = 0; b < NB; b++) {
#pragma unroll
      for (int i = 0; i < 16; i++) s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], c, mc));
#pragma unroll
      for (int k = 0; k < 2; k++) {
#pragma unroll
        for (int e = 0; e < 4; e++) pf[2 * b + k][e] = X::pack2(s[b][8 * k + 2 * e], s[b][8 * k + 2 * e + 1]);
        l = X::sum8(__builtin_bit_cast(bf16x8_t, pf[2 * b + k]), l);
      }
    }
  }

  // O^T += V^T P^T from the unit's values (LDS tile `vs`)
  __device__ __forceinline__ void values(const char* vs) {
    const int lane = threadIdx.x & 63, i16 = lane & 15, half = (lane >> 4) & 1, h = lane >> 5;
    const int t = 4 * h + (i16 >> 2);
    auto fragment = [&](int k, int dt) {
      const int chunk = 4 * dt + 2 * half + ((i16 & 3) >> 1);
      const char* a = vs + (16 * k + t) * ROW + ((chunk ^ swz<D>(t)) << 4) + 8 * (i16 & 1);
      const char* b = vs + (16 * k + t + 8) * ROW + ((chunk ^ swz<D>(t + 8)) << 4) + 8 * (i16 & 1);
      const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((bf16x4_t __attribute__((address_space(3)))*)(a));
      const bf16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((bf16x4_t __attribute__((address_space(3)))*)(b));
      return (bf16x8_t)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    bf16x8_t vf[2 * NB][DT];
#pragma unroll
    for (int k = 0; k < 2 * NB; k++)
#pragma unroll
      for (int dt = 0; dt < DT; dt++) vf[k][dt] = fragment(k, dt);
#pragma unroll
    for (int k = 0; k < 2 * NB; k++)
#pragma unroll
      for (int dt = 0; dt < DT; dt++) o[dt] = X::mfma32(vf[k][dt], __builtin_bit_cast(bf16x8_t, pf[k]), o[dt]);
    // 16 tokens' fragments are read while the previous ones' are multiplied
    __builtin_amdgcn_sched_group_barrier(SG_DS_RD, 2 * DT, 1);
#pragma unroll
    for (int i = 0; i < (2 * NB - 1) * DT; i++) {
      __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 1);
      __builtin_amdgcn_sched_group_barrier(SG_DS_RD, 2, 1);
    }
    __builtin_amdgcn_sched_group_barrier(SG_MFMA, DT, 1);
  }

  // four consecutive dims of the lane's row: 32 dt + 8 i + 4 h
  __device__ __forceinline__ f32x4_t quad(int dt, int i) const {
    return f32x4_t{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
  }

  // the rows as fp32 [32][D] and (m, l) per row; groups of four floats are swizzled by the row (merge_at), so that the
  // lanes' rows fall into different banks
  __device__ __forceinline__ void to_lds(float* dst, float* ml) const {
    const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        *reinterpret_cast<f32x4_t*>(dst + merge_at<D>(row, 32 * dt + 8 * i + 4 * h)) = quad(dt, i);
    const float sum = l + __shfl_xor(l, 32, 64);
    if (h == 0) {
      ml[2 * row] = m;
      ml[2 * row + 1] = sum;
    }
  }
};

// DMA of one block of 16 tokens (keys or values) into LDS; `voff` from block_offsets
template <int D> constexpr int block_dmas() { return AP_PAGE_MIN * D * 2 / 1024; }
template <int D> __device__ __forceinline__ void block_offsets(uint32_t* voff) {
  const int lane = threadIdx.x & 63;
  constexpr int CHUNKS = D / 8, ROWS = 64 / CHUNKS;    // chunks per row, rows per DMA instruction
#pragma unroll
  for (int j = 0; j < block_dmas<D>(); j++) {
    const int t = ROWS * j + lane / CHUNKS;
    voff[j] = (uint32_t)(t * D * 2 + (((lane % CHUNKS) ^ swz<D>(t)) << 4));
  }
}
template <int D, bool ONCE>   // ONCE: nothing else in the launch reads these rows
__device__ __forceinline__ void dma_block(const uint16_t* cache, int64_t offset, int tokens, uint32_t lds_addr, const uint32_t* voff) {
  const rsrc_t v = make_rsrc(cache + offset, (int64_t)tokens * (D * 2));
  const rsrc_t r = {__builtin_amdgcn_readfirstlane(v[0]), __builtin_amdgcn_readfirstlane(v[1]),
                    __builtin_amdgcn_readfirstlane(v[2]), v[3]};
#pragma unroll
  for (int j = 0; j < block_dmas<D>(); j++) {
    if (ONCE) dma16_nt(r, lds_addr + j * 1024, voff[j], 0);
    else dma16(r, lds_addr + j * 1024, voff[j], 0);
  }
}

// page of the block of 16 tokens at tok, -1 when it is unknown or the request ends before
__device__ __forceinline__ int page_at(const PagedArgs& p, int r, int kv, int tok) {
  if (tok >= kv) return -1;
  const int page = scalar_load(p.table + (int64_t)r * p.max_pages + (tok >> p.page_shift));
  return page >= 0 && page < p.n_pages ? page : -1;
}
// element offset of the block and the tokens of it that exist
template <int D>
__device__ __forceinline__ int64_t block_at(const PagedArgs& p, int page, int kvh, int kv, int tok, int& tokens) {
  const int left = kv - tok;
  tokens = page < 0 ? 0 : left < AP_PAGE_MIN ? (left < 0 ? 0 : left) : AP_PAGE_MIN;
  const int64_t in_page = tok & ((1 << p.page_shift) - 1);
  return ((((int64_t)(page < 0 ? 0 : page) * p.n_kv + kvh) << p.page_shift) + in_page) * D;
}

// ---- results of a tile --------------------------------------------------------------------------------
// where partial results of a workgroup go: its first tile (started by an earlier workgroup) and its last (its own)
__device__ __forceinline__ int slot_of(int w, int first) { return 2 * w + (w == first ? 1 : 0); }

template <bool F16> __device__ __forceinline__ void store_out(uint16_t* dst, f32x4_t o, float inv) {
  using X = X16<F16>;
  *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{X::pack2(o[0] * inv, o[1] * inv), X::pack2(o[2] * inv, o[3] * inv)};
}
// a sum of zero is a row that sees nothing (NaN is not: it has to be seen)
__device__ __forceinline__ float inverse(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }

template <int D>
__device__ __forceinline__ uint16_t* out_row(const PagedArgs& p, const Request& q, int kvh, int row) {
  const int tok = row / p.group, g = row - tok * p.group;
  return p.out + ((int64_t)(q.t0 + tok) * p.n_q + kvh * p.group + g) * D;
}

// what a partial result with maximum m is multiplied with under the common maximum: one that has seen nothing
// (m = -inf) holds zeros - or NaN, from a NaN in its scores, which has to be seen
__device__ __forceinline__ float part_scale(float m, float common, float c) {
  return m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - common) * c);
}

// After a workgroup has stored its partial tile: the one that delivers last adds all of them up, in order.  Partial
// results travel by device-coherent accesses, so no cache is written back or invalidated: the workgroup waits until
// its stores are acknowledged, then counts itself.
template <int D, bool F16, int BM, int THREADS>
__device__ __forceinline__ void merge_if_last(const PagedArgs& p, const Request& q, int kvh, int tile, int rows, int first, int last) {
  __shared__ int is_last;
  const int tid = threadIdx.x;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const int seen = __hip_atomic_fetch_add(p.arrived + first, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    is_last = seen == last - first;
    if (is_last) __hip_atomic_store(p.arrived + first, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!is_last) return;
  constexpr int STRIDE = BM * (D + 2), BATCH = 8;
  const Partials part(p.part);
  for (int idx = tid; idx < rows * (D / 4); idx += THREADS) {
    const int row = idx / (D / 4), d = idx % (D / 4) * 4;
    float mstar = -INFINITY, sum = 0.0f;
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int w0 = first; w0 <= last; w0 += BATCH) {
      f32x2_t ml[BATCH];
      f32x4_t ov[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; u++) {
        const int src = slot_of(w0 + u <= last ? w0 + u : w0, first) * STRIDE;
        ml[u] = part.load2(src + BM * D + 2 * row);
        ov[u] = part.load4(src + row * D + d);
      }
      float mn = mstar;
#pragma unroll
      for (int u = 0; u < BATCH; u++) {
        if (w0 + u > last) {
          ml[u] = f32x2_t{-INFINITY, 0.0f};
          ov[u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
        mn = fmaxf(mn, ml[u][0]);
      }
      const float keep = part_scale(mstar, mn, p.scale_log2e);
      acc *= keep;
      sum *= keep;
#pragma unroll
      for (int u = 0; u < BATCH; u++) {
        const float f = part_scale(ml[u][0], mn, p.scale_log2e);
        acc += ov[u] * f;
        sum += ml[u][1] * f;
      }
      mstar = mn;
    }
    store_out<F16>(out_row<D>(p, q, kvh, tile * BM + row) + d, acc, inverse(sum));
  }
}

// ---- narrow tiles: the waves take turns with the units ------------------------------------------------------
template <int D, bool F16>
__global__ __launch_bounds__(512) void attn_paged_narrow_kernel(const PagedArgs p) {
  constexpr int WAVES = 8, RING = 2;                     // keys or values of one unit a slot
  constexpr int TK = 32, BM = 32, THREADS = WAVES * 64;
  constexpr int ITEM = TK * D * 2, DMAS = ITEM / 1024;
  static_assert(BM * D * 4 <= RING * ITEM, "merge area");
  __shared__ __attribute__((aligned(1024))) char lds[WAVES * RING * ITEM];
  __shared__ float ml[WAVES][64];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int w = blockIdx.x;
  Run run;
  if (!find_run<BM, TK, THREADS, AP_START_NARROW>(p, w, run)) return;

  uint32_t voff[block_dmas<D>()];
  block_offsets<D>(voff);
  const uint32_t ring0 = __builtin_amdgcn_readfirstlane(lds_addr_of(lds)) + wave * (RING * ITEM);
  const char* ring = lds + wave * (RING * ITEM);
  constexpr int STRIDE = BM * (D + 2);
  const Partials part(p.part);

  int r = run.r;
  int kvh = (int)quotient(run.off, run.head_cost);
  int64_t toff = run.off - kvh * run.head_cost;
  int j = 0;
  bool found = false;
  int64_t x = run.x;
  for (; r < p.requests; r++) {
    const Request q = request_of(p, r);
    const int all = q.n * p.group, tiles = (all + BM - 1) / BM;
    if (tiles == 0) continue;
    for (; kvh < p.n_kv; kvh++) {
      Tiles<BM, TK> walk(q, p.group);
      for (j = 0; j < tiles; j++) {
        const int units = walk.next(), cost = units + AP_START_NARROW;
        if (!found) {                         // the run's first tile
          if (toff >= cost) {
            toff -= cost;
            continue;
          }
          found = true;
        }
        const int64_t left = run.hi - x;
        if (left <= 0) return;
        const int seg = (int)(toff + left < cost ? toff + left : cost);
        const int ua = (int)toff > AP_START_NARROW ? (int)toff - AP_START_NARROW : 0, ub = seg > AP_START_NARROW ? seg - AP_START_NARROW : 0;
        const int64_t tile_x = x - toff;
        const int rows = all - j * BM < BM ? all - j * BM : BM;
        const bool begins = toff == 0;
        x += seg - toff;
        toff = 0;
        if (units == 0) {                     // rows that see nothing
          if (begins)
            for (int idx = tid; idx < rows * D; idx += THREADS) out_row<D>(p, q, kvh, j * BM + idx / D)[idx % D] = 0;
          continue;
        }
        if (ua >= ub) continue;
        const int first = tile_x + AP_START_NARROW >= run.x ? w : wg_of(run, tile_x + AP_START_NARROW);
        const int last = tile_x + cost <= run.hi ? w : wg_of(run, tile_x + cost - 1);

        // ---- this wave's units of [ua, ub) ----
        const int n_my = ub - ua > wave ? (ub - ua - wave + WAVES - 1) / WAVES : 0, n_items = 2 * n_my;
        Wave<D, F16, 1> st;
        st.start(p, q, kvh, j * BM, all);
        int pg[2];
        auto fetch_pages = [&](int i) {
          const int tok = (ua + wave + WAVES * i) * TK;
          pg[0] = page_at(p, r, q.kv, tok);
          pg[1] = page_at(p, r, q.kv, tok + AP_PAGE_MIN);
        };
        auto issue = [&](int it) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slot's earlier contents have been read
          const int tok = (ua + wave + WAVES * (it >> 1)) * TK;
          const uint32_t slot = ring0 + (it % RING) * ITEM;
#pragma unroll
          for (int b = 0; b < 2; b++) {
            int tokens;
            const int64_t at = block_at<D>(p, pg[b], kvh, q.kv, tok + AP_PAGE_MIN * b, tokens);
            dma_block<D, true>((it & 1) ? p.v : p.k, at, tokens, slot + b * (ITEM / 2), voff);
          }
          if ((it & 1) && it + 1 < n_items) fetch_pages((it + 1) >> 1);
        };
        auto wait_item = [&](int it) {        // one item may be under way behind it
          if (it + 1 < n_items) wait_vm_at_most<DMAS>();
          else wait_vm_at_most<0>();
        };
        if (n_my > 0) {
          fetch_pages(0);
          issue(0);
        }
        for (int i = 0; i < n_my; i++) {
          const int tok = (ua + wave + WAVES * i) * TK;
          issue(2 * i + 1);
          wait_item(2 * i);
          // always with the mask: it hides behind the memory, and a second path without it made the compiler copy the
          // accumulators where the two meet (decode of 64 requests 98 -> 114 us)
          st.template scores<true>(ring, tok, p.scale_log2e);
          if (2 * i + 2 < n_items) issue(2 * i + 2);
          wait_item(2 * i + 1);
          st.values(ring + ITEM);
        }

        // ---- the waves' results ----
        __syncthreads();                      // all units read
        st.to_lds(reinterpret_cast<float*>(lds + wave * (RING * ITEM)), ml[wave]);
        __syncthreads();
        for (int idx = tid; idx < rows * (D / 4); idx += THREADS) {
          const int row = idx / (D / 4), d = idx % (D / 4) * 4;
          float mstar = -INFINITY, sum = 0.0f;
#pragma unroll
          for (int i = 0; i < WAVES; i++) mstar = fmaxf(mstar, ml[i][2 * row]);
          f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < WAVES; i++) {
            const float f = part_scale(ml[i][2 * row], mstar, p.scale_log2e);
            acc += *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(lds + i * (RING * ITEM)) + merge_at<D>(row, d)) * f;
            sum += ml[i][2 * row + 1] * f;
          }
          if (first == last) {
            store_out<F16>(out_row<D>(p, q, kvh, j * BM + row) + d, acc, inverse(sum));
          } else {
            const int dst = slot_of(w, first) * STRIDE;
            part.store4(dst + row * D + d, acc);
            if (d == 0) part.store2(dst + BM * D + 2 * row, mstar, sum);
          }
        }
        if (first != last) merge_if_last<D, F16, BM, THREADS>(p, q, kvh, j, rows, first, last);
        __syncthreads();                      // the merge area becomes the rings again
      }
    }
    kvh = 0;
  }
}

// ---- wide tiles: the waves share the units --------------------------------------------------------------
template <int D, bool F16>
__global__ __launch_bounds__(512, 2) void attn_paged_wide_kernel(const PagedArgs p) {
  constexpr int WAVES = 8, STAGES = 4, TK = 64, BM = 32 * WAVES, THREADS = WAVES * 64;
  constexpr int HALF = TK * D * 2, STAGE = 2 * HALF;     // keys, then values of one unit
  constexpr int DMAS = block_dmas<D>();                  // of the unit's 8 blocks (4 of keys, 4 of values) a wave brings one
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * STAGE];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // neighbouring runs share keys and values: keep them on one XCD (workgroups go round robin over the eight)
  const int w = (blockIdx.x & 7) * (p.wgs >> 3) + (blockIdx.x >> 3);
  Run run;
  if (!find_run<BM, TK, THREADS, AP_START_WIDE>(p, w, run)) return;

  uint32_t voff[block_dmas<D>()];
  block_offsets<D>(voff);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr_of(lds)) + (wave & 3) * (AP_PAGE_MIN * D * 2);
  constexpr int STRIDE = BM * (D + 2);
  const Partials part(p.part);

  int r = run.r;
  int kvh = (int)quotient(run.off, run.head_cost);
  int64_t toff = run.off - kvh * run.head_cost;
  bool found = false;
  int64_t x = run.x;
  for (; r < p.requests; r++) {
    const Request q = request_of(p, r);
    const int all = q.n * p.group, tiles = (all + BM - 1) / BM;
    if (tiles == 0) continue;
    for (; kvh < p.n_kv; kvh++) {
      Tiles<BM, TK> walk(q, p.group);
      for (int j = 0; j < tiles; j++) {
        const int units = walk.next(), cost = units + AP_START_WIDE;
        if (!found) {
          if (toff >= cost) {
            toff -= cost;
            continue;
          }
          found = true;
        }
        const int64_t left = run.hi - x;
        if (left <= 0) return;
        const int seg = (int)(toff + left < cost ? toff + left : cost);
        const int ua = (int)toff > AP_START_WIDE ? (int)toff - AP_START_WIDE : 0, ub = seg > AP_START_WIDE ? seg - AP_START_WIDE : 0;
        const int64_t tile_x = x - toff;
        const int rows = all - j * BM < BM ? all - j * BM : BM;
        const bool begins = toff == 0;
        x += seg - toff;
        toff = 0;
        if (units == 0) {
          if (begins)
            for (int idx = tid; idx < rows * D; idx += THREADS) out_row<D>(p, q, kvh, j * BM + idx / D)[idx % D] = 0;
          continue;
        }
        if (ua >= ub) continue;
        const int first = tile_x + AP_START_WIDE >= run.x ? w : wg_of(run, tile_x + AP_START_WIDE);
        const int last = tile_x + cost <= run.hi ? w : wg_of(run, tile_x + cost - 1);

        const int row0 = 32 * wave;
        const bool active = row0 < rows;
        Wave<D, F16, 2> st;
        st.start(p, q, kvh, j * BM + row0, all);
        const int lim0 = q.kv - q.n + (j * BM + row0) / p.group + 1;   // what the wave's first row sees
        int page = page_at(p, r, q.kv, ua * TK + (wave & 3) * AP_PAGE_MIN);
        auto issue = [&](int u) {
          const int tok = u * TK + (wave & 3) * AP_PAGE_MIN;
          int tokens;
          const int64_t at = block_at<D>(p, page, kvh, q.kv, tok, tokens);
          const uint32_t dst = lds0 + (uint32_t)(u % STAGES) * STAGE;
          if (wave < 4) dma_block<D, false>(p.k, at, tokens, dst, voff);
          else dma_block<D, false>(p.v, at, tokens, dst + HALF, voff);
          if (u + 1 < ub) page = page_at(p, r, q.kv, tok + TK);
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++)
          if (ua + i < ub) issue(ua + i);
        auto step = [&](int u) {              // unit u has arrived, unit u - 1 has been read by all
          const int after = ub - 1 - u;       // units requested behind u: up to STAGES - 2
          if (after >= STAGES - 2) wait_vm_at_most<(STAGES - 2) * DMAS>();
          else if (after == 1) wait_vm_at_most<DMAS>();
          else wait_vm_at_most<0>();
          __syncthreads();
          if (u + STAGES - 1 < ub) issue(u + STAGES - 1);
        };
        static_assert(STAGES == 4, "step");
        if (active) {
          int free_of_mask = lim0 <= 0 ? 0 : lim0 / TK;      // units that all of the wave's rows see whole
          if (free_of_mask > ub) free_of_mask = ub;
          int u = ua;
          for (; u < free_of_mask; u++) {
            step(u);
            const char* base = lds + (u % STAGES) * STAGE;
            st.template scores<false>(base, u * TK, p.scale_log2e);
            st.values(base + HALF);
          }
          for (; u < ub; u++) {
            step(u);
            const char* base = lds + (u % STAGES) * STAGE;
            st.template scores<true>(base, u * TK, p.scale_log2e);
            st.values(base + HALF);
          }
        } else {                              // no such rows: the wave brings keys and values for the others
          for (int u = ua; u < ub; u++) step(u);
        }
        __syncthreads();

        if (first == last) {
          const int lane = tid & 63, c = lane & 31, h = lane >> 5;
          const float inv = inverse(st.l + __shfl_xor(st.l, 32, 64));
          if (row0 + c < rows) {
            uint16_t* dst = out_row<D>(p, q, kvh, j * BM + row0 + c);
#pragma unroll
            for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
              for (int i = 0; i < 4; i++) store_out<F16>(dst + 32 * dt + 8 * i + 4 * h, st.quad(dt, i), inv);
          }
        } else {
          // through LDS, 32 dims at a time in the wave's own quarter, for stores of whole lines
          const int dst = slot_of(w, first) * STRIDE;
          const int lane = tid & 63, c = lane & 31, h = lane >> 5;
          float* mine = reinterpret_cast<float*>(lds + wave * (STAGES * STAGE / WAVES));
#pragma unroll
          for (int dt = 0; dt < D / 32; dt++) {
            wave_lds_sync();
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<f32x4_t*>(mine + c * 36 + 8 * i + 4 * h) = st.quad(dt, i);
            wave_lds_sync();
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int row = 8 * i + (lane >> 3), d = 4 * (lane & 7);
              if (row0 + row < rows)
                part.store4(dst + (row0 + row) * D + 32 * dt + d, *reinterpret_cast<const f32x4_t*>(mine + row * 36 + d));
            }
          }
          const float sum = st.l + __shfl_xor(st.l, 32, 64);
          if (lane < 32 && row0 + lane < rows) part.store2(dst + BM * D + 2 * (row0 + lane), st.m, sum);
          merge_if_last<D, F16, BM, THREADS>(p, q, kvh, j, rows, first, last);
        }
        __syncthreads();
      }
    }
    kvh = 0;
  }
}

constexpr int NARROW_WGS = 256;      // one per CU: 128 KiB of LDS each
constexpr int WIDE_WGS = 256;        // one per CU: 128 KiB
static_assert(NARROW_WGS * 4 <= AP_COUNTER_BYTES && WIDE_WGS * 4 <= AP_COUNTER_BYTES, "arrival counters");

// Narrow up to 32 rows a tile: 64 requests of up to 8000 tokens, one token each, 32 + 8 heads: 85 us (wide: 98), 8 tokens
// each 66 (71); one request of 130001 tokens 95 (112), its 8 tokens 100 (113); 12 + 12 heads of 64, 24 tokens 39 (49).
// From 33 rows on wide; a narrow form with two row blocks and four waves was slower nearly everywhere: 9 tokens of 64
// requests 82 (wide: 77), 16 tokens of 4 requests 30 (20), 5 tokens of 96 requests with 64 + 8 heads 81 (71); only one
// request of 130001 tokens gained, 9 tokens 111 (116).
// min_units, the shortest run: few requests then keep to few workgroups.  Narrow with 2, 8 and 32 units: four requests of
// up to 900 tokens 12.2, 12.5 and 21.5 us; wide with 1, 4 and 16: a prompt of 300 tokens 33.5, 35.7 and 51 us, one of 1500
// 60.6, 60.4 and 65.3; the long cases do not depend on it.
template <int D, bool F16>
void launch(const PagedArgs& base, int rows, hipStream_t s) {
  PagedArgs a = base;
  if (rows <= 32) {
    a.wgs = NARROW_WGS;
    a.min_units = 8;
    hipLaunchKernelGGL((attn_paged_narrow_kernel<D, F16>), dim3(a.wgs), dim3(512), 0, s, a);
  } else {
    a.wgs = WIDE_WGS;
    a.min_units = 4;
    hipLaunchKernelGGL((attn_paged_wide_kernel<D, F16>), dim3(a.wgs), dim3(512), 0, s, a);
  }
}

}  // namespace

extern "C" int64_t mtp_attn_paged_workspace_bytes(void) {
  return AP_COUNTER_BYTES + 2ll * WIDE_WGS * 256 * (128 + 2) * (int64_t)sizeof(float);
}

extern "C" int mtp_attn_paged(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                              const int64_t* cu, const int64_t* kv_lens, void* out, void* workspace,
                              int64_t workspace_bytes, int64_t T, int64_t requests, int n_q_heads, int n_kv_heads,
                              int head_dim, int64_t n_pages, int64_t page_size, int64_t max_pages, int64_t max_new,
                              int64_t len_bound, float scale, int dtype, void* stream) {
  MTP_REQUIRE(dtype == MTP_BF16 || dtype == MTP_F16, MTP_EUNSUPPORTED, "attn_paged: dtype %d (bf16 or f16)", dtype);
  MTP_REQUIRE(head_dim == 64 || head_dim == 128, MTP_EUNSUPPORTED, "attn_paged: head_dim %d (64 or 128)", head_dim);
  MTP_REQUIRE(n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0 && n_q_heads <= 4096, MTP_EINVAL,
              "attn_paged: heads %d/%d", n_q_heads, n_kv_heads);
  MTP_REQUIRE(T >= 0 && T <= 0x3fffffffll / n_q_heads && requests >= 0 && requests <= 0x7fffff, MTP_EINVAL,
              "attn_paged: T=%lld requests=%lld", (long long)T, (long long)requests);
  MTP_REQUIRE(page_size >= AP_PAGE_MIN && (page_size & (page_size - 1)) == 0, MTP_EUNSUPPORTED,
              "attn_paged: page_size=%lld (a power of two, at least %d)", (long long)page_size, AP_PAGE_MIN);
  MTP_REQUIRE(n_pages > 0 && n_pages <= 0x7fffffffll && max_pages > 0 && page_size <= 0x40000000ll &&
                  max_pages <= 0x7fffffffll / page_size,
              MTP_EINVAL, "attn_paged: %lld pages of %lld, %lld a row", (long long)n_pages, (long long)page_size,
              (long long)max_pages);
  MTP_REQUIRE(max_new >= 0 && len_bound >= 0, MTP_EINVAL, "attn_paged: max_new=%lld len_bound=%lld", (long long)max_new,
              (long long)len_bound);
  MTP_REQUIRE(scale > 0.0f && scale < INFINITY, MTP_EINVAL, "attn_paged: scale %g", (double)scale);
  if (T == 0 || requests == 0) return MTP_OK;
  MTP_REQUIRE(q && k_cache && v_cache && block_tables && cu && kv_lens && out, MTP_EINVAL, "attn_paged: null pointer");
  MTP_REQUIRE(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) % 16 == 0,
              MTP_EINVAL, "attn_paged: tensors must be 16-byte aligned");
  MTP_REQUIRE(workspace && workspace_bytes >= mtp_attn_paged_workspace_bytes(), MTP_EWORKSPACE,
              "attn_paged: workspace %lld bytes, need %lld", (long long)workspace_bytes,
              (long long)mtp_attn_paged_workspace_bytes());
  PagedArgs a = {};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k_cache);
  a.v = static_cast<const uint16_t*>(v_cache);
  a.table = block_tables;
  a.cu = cu;
  a.kv_lens = kv_lens;
  a.out = static_cast<uint16_t*>(out);
  a.arrived = static_cast<int32_t*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + AP_COUNTER_BYTES);
  a.max_pages = max_pages;
  a.T = (int)T;
  a.requests = (int)requests;
  a.n_q = n_q_heads;
  a.n_kv = n_kv_heads;
  a.group = n_q_heads / n_kv_heads;
  a.page_shift = __builtin_ctzll((unsigned long long)page_size);
  a.n_pages = (int)n_pages;
  a.room = (int)(max_pages * page_size);
  a.scale_log2e = scale * 1.4426950408889634f;
  const int64_t most = (max_new < T ? max_new : T) * a.group;
  const int rows = most > 1 << 20 ? 1 << 20 : (int)most;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f16 = dtype == MTP_F16;
  if (head_dim == 64) {
    if (f16) launch<64, true>(a, rows, s);
    else launch<64, false>(a, rows, s);
  } else {
    if (f16) launch<128, true>(a, rows, s);
    else launch<128, false>(a, rows, s);
  }
  MTP_CHECK_LAUNCH("attn_paged");
  return MTP_OK;
}
