// Verification of drafted tokens against the target model's probabilities, from given random numbers.
//
// Request r has K drafted tokens x_0 .. x_{K-1} (draft_lens[r] of them where given), the target's probabilities p_i for
// the position of each and one more, and the draft's own q_i (none: the draft was certain, q_i(x_i) = 1).  Draft i is
// accepted while u_i q_i(x_i) < p_i(x_i), i.e. with probability min(1, p / q).  At the first rejection, after n
// accepted drafts, the next token is drawn from max(p_n - q_n, 0) normalised; if nothing was rejected, from p_n.  The
// accepted tokens and the drawn one are then distributed as the target's own samples.
// The draw is the inverse CDF in index order: the first index whose cumulative weight exceeds u_K times their sum.
//
// Products and sums are fp64: u q and the comparison are then exact for fp32 inputs, and a cumulative sum over a
// vocabulary moves a border between two tokens by 1e-16 of the mass instead of 1e-7, which would change one draw in
// some thousands.  Weights that are not positive finite numbers count as zero.
//
// Bound: HBM (one row of p, one of q where a draft was rejected), and for a few requests the latency of two launches:
// every row is cut into up to 64 chunks, one workgroup sums each (the first launch), one workgroup per row finds the
// chunk that holds the drawn point and walks it (the second).  A workgroup finds n by itself: K probabilities.  128
// requests of 50257 weights: 10.0 us for the sums (26 MB) and 8.4 for the draw, 8 of 128256: 4.5 and 9.0; the draw is a
// chain of dependent loads (draft, probability, row) whatever the size.
#include "mtp_common.h"

namespace {

constexpr int VD_THREADS = 256;
constexpr int VD_WAVES = VD_THREADS / MTP_WAVE;
constexpr int VD_MAX_DRAFTS = 64;      // one lane each
constexpr int VD_MAX_CHUNKS = 64;      // one lane each
constexpr int VD_STEP = 2048;          // chunk lengths are multiples of this: 8 elements per thread

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<uint16_t>(uint16_t v) { return bf16_bits_to_f32(v); }
template <> __device__ __forceinline__ float to_f32<f16s>(f16s v) { return X16<true>::from_bits(v.bits); }

__device__ __forceinline__ double weight_of(double w) { return w > 0.0 && w < (double)INFINITY ? w : 0.0; }

struct VerifyArgs {
  const int64_t* drafts;       // [R, K]
  const int64_t* draft_lens;   // [R] or null
  const void* target;          // [R, K + 1, V]
  const void* draft;           // [R, K, V] or null
  const float* uniforms;       // [R, K + 1]
  int64_t* tokens;             // [R, K + 1]
  int64_t* accepted;           // [R]
  double* part;                // [R, chunks, 2] sums of the chunk: left over, target
  int64_t V;
  int K, chunks, chunk_len;
};

// accepted drafts of request r, and how many it has; the same in every lane of the wave
template <typename T>
__device__ __forceinline__ int accepted_of(const VerifyArgs& p, int64_t r, int& len) {
  const int i = threadIdx.x & 63;
  len = p.K;
  if (p.draft_lens) {
    const int64_t l = p.draft_lens[r];
    len = l < 0 ? 0 : (l < p.K ? (int)l : p.K);
  }
  bool ok = false;
  if (i < len) {
    const int64_t x = p.drafts[r * p.K + i];
    if (x >= 0 && x < p.V) {
      const double pt = (double)to_f32(static_cast<const T*>(p.target)[(r * (p.K + 1) + i) * p.V + x]);
      const double qt = p.draft ? (double)to_f32(static_cast<const T*>(p.draft)[(r * p.K + i) * p.V + x]) : 1.0;
      ok = (double)p.uniforms[r * (p.K + 1) + i] * qt < pt;
    }
  }
  const uint64_t no = ~__ballot(ok);
  const int n = no ? __ffsll((unsigned long long)no) - 1 : 64;
  return n < len ? n : len;
}

// the weights of the row that the next token is drawn from
template <typename T>
struct Row {
  const T* p;          // target's row
  const T* q;          // draft's row, null: none to take off
  int64_t without;     // index whose weight is taken off whole (a certain draft), -1: none
  __device__ __forceinline__ Row(const VerifyArgs& a, int64_t r, int n, int len) {
    p = static_cast<const T*>(a.target) + (r * (a.K + 1) + n) * a.V;
    const bool rejected = n < len;
    q = rejected && a.draft ? static_cast<const T*>(a.draft) + (r * a.K + n) * a.V : nullptr;
    without = rejected && !a.draft ? a.drafts[r * a.K + n] : -1;
  }
  // weights of the 8 elements at, at + step, ... below end (0 behind it): left over and whole.  All loads are issued
  // together, from clamped places: a branch around each would wait for each.
  __device__ __forceinline__ void load8(int64_t at, int step, int64_t end, double* left, double* whole) const {
    float pv[8], qv[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int64_t v = at + j * step < end ? at + j * step : end - 1;
      pv[j] = to_f32(p[v]);
    }
    if (q) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int64_t v = at + j * step < end ? at + j * step : end - 1;
        qv[j] = to_f32(q[v]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) qv[j] = at + j * step == without ? INFINITY : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const bool in = at + j * step < end;
      whole[j] = in ? weight_of((double)pv[j]) : 0.0;
      left[j] = in ? weight_of((double)pv[j] - (double)qv[j]) : 0.0;
    }
  }
};

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <typename T>
__global__ __launch_bounds__(VD_THREADS) void verify_sum_kernel(const VerifyArgs p) {
  const int64_t r = blockIdx.y;
  int len;
  const int n = accepted_of<T>(p, r, len);
  const Row<T> row(p, r, n, len);
  const int64_t v0 = (int64_t)blockIdx.x * p.chunk_len;
  const int64_t v1 = v0 + p.chunk_len < p.V ? v0 + p.chunk_len : p.V;
  double left = 0.0, whole = 0.0;
  for (int64_t v = v0 + threadIdx.x; v < v1; v += VD_STEP) {
    double l[8], w[8];
    row.load8(v, VD_THREADS, v1, l, w);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      left += l[j];
      whole += w[j];
    }
  }
  __shared__ double acc[VD_WAVES][2];
  left = wave_sum_f64(left);
  whole = wave_sum_f64(whole);
  if ((threadIdx.x & 63) == 0) {
    acc[threadIdx.x >> 6][0] = left;
    acc[threadIdx.x >> 6][1] = whole;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    double v = 0.0;
#pragma unroll
    for (int w = 0; w < VD_WAVES; w++) v += acc[w][threadIdx.x];
    p.part[(r * p.chunks + blockIdx.x) * 2 + threadIdx.x] = v;
  }
}

__device__ __forceinline__ double wave_scan_f64(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(v, o, 64);
    if (lane >= o) v += up;
  }
  return v;
}

template <typename T>
__global__ __launch_bounds__(VD_THREADS) void verify_draw_kernel(const VerifyArgs p) {
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int len;
  const int n = accepted_of<T>(p, r, len);
  const Row<T> row(p, r, n, len);

  // every wave: sums of the chunks, the drawn point, the chunk that holds it
  const double* part = p.part + r * p.chunks * 2;
  const double left = lane < p.chunks ? part[2 * lane] : 0.0;
  const double whole = lane < p.chunks ? part[2 * lane + 1] : 0.0;
  const bool use_left = wave_sum_f64(left) > 0.0;   // nothing left over (p <= q everywhere, by rounding): the target's
  const double mine = use_left ? left : whole;
  const double incl = wave_scan_f64(mine);
  const double total = __shfl(incl, 63, 64);
  const double point = (double)p.uniforms[r * (p.K + 1) + p.K] * total;
  uint64_t hit = __ballot(incl > point && mine > 0.0);
  const uint64_t some = __ballot(mine > 0.0);
  // a point at or behind the end (a uniform of 1, or rounding): the last chunk that holds any weight
  const int chunk = hit ? __ffsll((unsigned long long)hit) - 1 : some ? 63 - __clzll((long long)some) : -1;
  const double before = chunk > 0 ? __shfl(incl, chunk - 1, 64) : 0.0;

  __shared__ double sums[VD_WAVES];
  __shared__ int64_t found, last;
  if (tid == 0) {
    found = p.V;
    last = -1;
  }
  __syncthreads();
  if (chunk >= 0) {
    // 2048 elements at a time, 8 consecutive ones per thread, loaded together and kept: their sum, then the walk to the
    // border in the thread whose range holds it
    const int64_t v0 = (int64_t)chunk * p.chunk_len;
    const int64_t v1 = v0 + p.chunk_len < p.V ? v0 + p.chunk_len : p.V;
    double base = before;
    int64_t last_mine = -1;
    for (int64_t s0 = v0; s0 < v1; s0 += VD_STEP) {
      const int64_t a = s0 + 8 * tid;
      double l[8], x[8], own = 0.0;
      row.load8(a, 1, v1, l, x);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        x[j] = use_left ? l[j] : x[j];
        own += x[j];
        if (x[j] > 0.0) last_mine = a + j;
      }
      const double scan = wave_scan_f64(own);
      if (lane == 63) sums[wave] = scan;
      __syncthreads();
      double mine_at = base;
#pragma unroll
      for (int w = 0; w < VD_WAVES; w++) {
        if (w < wave) mine_at += sums[w];
        base += sums[w];
      }
      if (own > 0.0 && mine_at + scan > point) {
        double run = mine_at + (scan - own);
        int64_t here = p.V;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          run += x[j];
          if (x[j] > 0.0 && run > point && here == p.V) here = a + j;
        }
        // the walk's own rounding may leave it a hair short of the border that the scan has seen
        if (here == p.V) here = last_mine;
        atomicMin(reinterpret_cast<unsigned long long*>(&found), (unsigned long long)here);
      }
      __syncthreads();
      if (found < p.V) break;             // the same for every thread
    }
    if (found == p.V) {                   // no border: the chunk's last weight; waves first: 256 atomics on one word cost 4 us
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const int64_t other = __shfl_xor((long long)last_mine, o, 64);
        last_mine = other > last_mine ? other : last_mine;
      }
      if (lane == 0) atomicMax(reinterpret_cast<long long*>(&last), (long long)last_mine);
      __syncthreads();
    }
  }
  const int64_t token = found < p.V ? found : last;   // -1: the row holds no weight at all
  for (int i = tid; i <= p.K; i += VD_THREADS)
    p.tokens[r * (p.K + 1) + i] = i < n ? p.drafts[r * p.K + i] : i == n ? token : -1;
  if (tid == 0) p.accepted[r] = n;
}

// Chunks of a row: about VD_TARGET workgroups over all rows (128 rows of 50257: 1024 workgroups 24.2 us for both launches,
// 4096 18.5, 8192 18.5), at most one per lane of the wave that scans their sums, and whole steps of 2048 elements.
constexpr int64_t VD_TARGET = 4096;
void pick_chunks(int64_t R, int64_t V, int& chunks, int& chunk_len) {
  const int64_t steps = (V + VD_STEP - 1) / VD_STEP;
  int64_t want = (VD_TARGET + R - 1) / R;
  if (want > VD_MAX_CHUNKS) want = VD_MAX_CHUNKS;
  const int64_t per = (steps + want - 1) / want;
  chunk_len = (int)(per * VD_STEP);
  chunks = (int)((V + chunk_len - 1) / chunk_len);
}

template <typename T>
void launch(const VerifyArgs& a, int64_t R, hipStream_t s) {
  hipLaunchKernelGGL(verify_sum_kernel<T>, dim3(a.chunks, (unsigned)R), dim3(VD_THREADS), 0, s, a);
  hipLaunchKernelGGL(verify_draw_kernel<T>, dim3((unsigned)R), dim3(VD_THREADS), 0, s, a);
}

}  // namespace

extern "C" int64_t mtp_verify_draft_workspace_bytes(int64_t R, int64_t V) {
  if (R <= 0 || V <= 0) return 0;
  int chunks, chunk_len;
  pick_chunks(R, V, chunks, chunk_len);
  return R * chunks * 2 * (int64_t)sizeof(double);
}

extern "C" int mtp_verify_draft(const int64_t* draft_tokens, const int64_t* draft_lens, const void* target_probs,
                                const void* draft_probs, const float* uniforms, int64_t* tokens, int64_t* accepted,
                                void* workspace, int64_t workspace_bytes, int64_t R, int K, int64_t V, int dtype,
                                void* stream) {
  MTP_REQUIRE(dtype == MTP_F32 || dtype == MTP_BF16 || dtype == MTP_F16, MTP_EINVAL, "verify_draft: dtype %d", dtype);
  MTP_REQUIRE(R >= 0 && R <= 65535 && V > 0 && V <= 0x3fffffffll, MTP_EINVAL, "verify_draft: R=%lld V=%lld", (long long)R,
              (long long)V);
  MTP_REQUIRE(K >= 0 && K <= VD_MAX_DRAFTS, MTP_EUNSUPPORTED, "verify_draft: %d drafts (at most %d)", K, VD_MAX_DRAFTS);
  if (R == 0) return MTP_OK;
  MTP_REQUIRE((K == 0 || draft_tokens) && target_probs && uniforms && tokens && accepted, MTP_EINVAL,
              "verify_draft: null pointer");
  const int64_t need = mtp_verify_draft_workspace_bytes(R, V);
  MTP_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 8 == 0, MTP_EWORKSPACE,
              "verify_draft: workspace %lld bytes, need %lld (8-byte aligned)", (long long)workspace_bytes,
              (long long)need);
  VerifyArgs a = {draft_tokens, draft_lens, target_probs, draft_probs, uniforms, tokens, accepted,
                  static_cast<double*>(workspace), V, K, 0, 0};
  pick_chunks(R, V, a.chunks, a.chunk_len);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MTP_F32) launch<float>(a, R, s);
  else if (dtype == MTP_BF16) launch<uint16_t>(a, R, s);
  else launch<f16s>(a, R, s);
  MTP_CHECK_LAUNCH("verify_draft");
  return MTP_OK;
}
