// RMSNorm of every query and key head followed by the rotary embedding, in one pass over the fused QKV rows:
// forward and backward for training, and the serving form that drops keys and values into the pages of a cache.
//
// For a head x of D elements with the norm weight w (shared by the heads of its kind; no weight: no norm), at
// position p with the table rows c = cos[p], s = sin[p], halves written 1 and 2:
//     r = 1 / sqrt(mean(x^2) + eps)     n = x r     z = w n
//     y1 = z1 c1 - z2 s1                y2 = z2 c2 + z1 s2
// and for the gradient dy of y
//     dz1 = dy1 c1 + dy2 s2             dz2 = dy2 c2 - dy1 s1
//     dw  = sum over rows of dz n       dx  = r (w dz - x r^2 mean(w dz x))
// Everything between the load and the store is fp32 and is rounded once, at the store (the separate steps of a tensor
// expression round the normalised head, the product with w and each rotary product; nothing here needs those).
//
// Bound: HBM; every element is read once and written once.  A lane holds 8 consecutive elements of the first half of
// a head and the 8 matching ones of the second half, so both halves of a rotation sit in one lane (no exchange) and
// the mean is three or two butterfly steps over the D / 16 lanes of a head.  One wave walks the heads of one token, so
// the table row is loaded once per token and stays in registers; with few tokens the heads of a token are dealt to
// several waves.  8192 tokens of 32 + 8 heads of 128 in bf16: forward 36 us for 176 MB (5.0 TB/s; a copy of 168 MB runs
// at 5.0 to 5.8), backward 70 us for 294 MB (4.2 TB/s: 200 registers a lane, two waves per SIMD, do not keep enough loads
// under way) and 4.6 us for the weight gradients' sum.  Append of 8191 tokens of 8 + 1 heads 12 us for 50 MB, of 32
// tokens 3.6 us: the launch.
#include "mtp_common.h"

namespace {

constexpr int QN_THREADS = 256;
constexpr int QN_WAVES = QN_THREADS / MTP_WAVE;

// 8 consecutive elements of a tensor as fp32 and back
template <typename T> struct Oct;
template <> struct Oct<uint16_t> {
  u32x4_t v;
  __device__ __forceinline__ void load(const uint16_t* p) { v = *reinterpret_cast<const u32x4_t*>(p); }
  __device__ __forceinline__ void store(uint16_t* p) const { *reinterpret_cast<u32x4_t*>(p) = v; }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int e = 0; e < 4; e++) { f[2 * e] = bf16_lo(v[e]); f[2 * e + 1] = bf16_hi(v[e]); }
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = pack_bf16x2(f[2 * e], f[2 * e + 1]);
  }
  __device__ __forceinline__ void zero() { v = u32x4_t{0u, 0u, 0u, 0u}; }
  static __device__ __forceinline__ uint16_t one(float f) { return f32_to_bf16_bits(f); }
};
template <> struct Oct<f16s> {
  using H = X16<true>;
  u32x4_t v;
  __device__ __forceinline__ void load(const f16s* p) { v = *reinterpret_cast<const u32x4_t*>(p); }
  __device__ __forceinline__ void store(f16s* p) const { *reinterpret_cast<u32x4_t*>(p) = v; }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int e = 0; e < 4; e++) { f[2 * e] = H::lo(v[e]); f[2 * e + 1] = H::hi(v[e]); }
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = H::pack2(f[2 * e], f[2 * e + 1]);
  }
  __device__ __forceinline__ void zero() { v = u32x4_t{0u, 0u, 0u, 0u}; }
  static __device__ __forceinline__ f16s one(float f) { return f16s{H::to_bits(f)}; }
};
template <> struct Oct<float> {
  u32x4_t v[2];
  __device__ __forceinline__ void load(const float* p) {
    v[0] = reinterpret_cast<const u32x4_t*>(p)[0];
    v[1] = reinterpret_cast<const u32x4_t*>(p)[1];
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<u32x4_t*>(p)[0] = v[0];
    reinterpret_cast<u32x4_t*>(p)[1] = v[1];
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = __uint_as_float(v[e >> 2][e & 3]);
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e >> 2][e & 3] = __float_as_uint(f[e]);
  }
  __device__ __forceinline__ void zero() { v[0] = v[1] = u32x4_t{0u, 0u, 0u, 0u}; }
  static __device__ __forceinline__ float one(float f) { return f; }
};

struct RotArgs {
  const void* qkv;            // [T, (n_q + 2 n_kv) D]
  const void* cos_t;          // [max_positions, D], fp32 or the tensors' type
  const void* sin_t;
  const int64_t* positions;   // [T]
  const void* q_weight;       // [D] or null
  const void* k_weight;
  void* q_out;                // [T, n_q, D]
  void* k_out;                // [T, n_kv, D]                     (training form)
  const int64_t* slots;       // [T]                              (serving form)
  void* k_cache;              // [n_pages, n_kv, page_size, D]
  void* v_cache;
  const void* dq;             // gradients                        (backward)
  const void* dk;
  const void* dv;
  void* dqkv;
  float* part;                // [workgroups, 2, D] sums for the weight gradients
  int64_t tokens, max_positions, n_slots;
  int n_q, n_kv, page_shift, table_f32, split;
  float eps;
};

// table row -> 8 floats of each half of cos and sin
template <typename T>
__device__ __forceinline__ void load_table(const void* table, int f32, int64_t row, int d, int half, float* a, float* b) {
  if (f32) {
    Oct<float> o;
    const float* p = static_cast<const float*>(table) + row;
    o.load(p + d);
    o.get(a);
    o.load(p + half + d);
    o.get(b);
  } else {
    Oct<T> o;
    const T* p = static_cast<const T*>(table) + row;
    o.load(p + d);
    o.get(a);
    o.load(p + half + d);
    o.get(b);
  }
}

template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <typename T, int D, bool APPEND>
__global__ __launch_bounds__(QN_THREADS) void qk_norm_rope_kernel(const RotArgs p) {
  constexpr int LANES = D / 16, HEADS = 64 / LANES, HALF = D / 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t item = (int64_t)blockIdx.x * QN_WAVES + wave;
  const int64_t t = item / p.split;
  const int part = (int)(item - t * p.split);
  if (t >= p.tokens) return;
  const int d = 8 * (lane % LANES), sub = lane / LANES;
  const int rotated = p.n_q + p.n_kv, total = APPEND ? rotated + p.n_kv : rotated;
  const T* row = static_cast<const T*>(p.qkv) + t * (int64_t)(p.n_q + 2 * p.n_kv) * D;
  const int64_t pos = p.positions[t];
  const bool known = pos >= 0 && pos < p.max_positions;
  int64_t slot = -1;
  if (APPEND) {
    slot = p.slots[t];
    if (slot >= p.n_slots || !known) slot = -1;
  }
  float c1[8], c2[8], s1[8], s2[8];
  load_table<T>(p.cos_t, p.table_f32, (known ? pos : 0) * D, d, HALF, c1, c2);
  load_table<T>(p.sin_t, p.table_f32, (known ? pos : 0) * D, d, HALF, s1, s2);

  int h = part * HEADS + sub;
  Oct<T> a, b;
  a.zero();
  b.zero();
  if (h < total) {
    a.load(row + (int64_t)h * D + d);
    b.load(row + (int64_t)h * D + HALF + d);
  }
  for (int h0 = part * HEADS; h0 < total; h0 += p.split * HEADS) {
    const int cur = h;
    Oct<T> xa = a, xb = b;
    h += p.split * HEADS;                 // the next heads are on their way while these are turned
    if (h < total) {
      a.load(row + (int64_t)h * D + d);
      b.load(row + (int64_t)h * D + HALF + d);
    }
    float x1[8], x2[8];
    xa.get(x1);
    xb.get(x2);
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) ss += x1[e] * x1[e] + x2[e] * x2[e];
    ss = head_sum<LANES>(ss);
    const T* w = static_cast<const T*>(cur < p.n_q ? p.q_weight : p.k_weight);
    if (w && cur < rotated) {
      // the correctly rounded root and division: an approximate reciprocal root would cost fp32 tensors their last bits
      const float r = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
      Oct<T> wa, wb;
      float w1[8], w2[8];
      wa.load(w + d);
      wb.load(w + HALF + d);
      wa.get(w1);
      wb.get(w2);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        x1[e] *= r * w1[e];
        x2[e] *= r * w2[e];
      }
    }
    float y1[8], y2[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      y1[e] = x1[e] * c1[e] - x2[e] * s1[e];
      y2[e] = x2[e] * c2[e] + x1[e] * s2[e];
    }
    Oct<T> oa, ob;
    oa.set(y1);
    ob.set(y2);
    if (!known) {
      oa.zero();
      ob.zero();
    }
    T* dst = nullptr;
    if (cur < p.n_q) {
      dst = static_cast<T*>(p.q_out) + (t * p.n_q + cur) * D;
    } else if (cur < total) {
      if (!APPEND) {
        dst = static_cast<T*>(p.k_out) + (t * p.n_kv + (cur - p.n_q)) * D;
      } else if (slot >= 0) {
        const bool value = cur >= rotated;
        const int kvh = cur - (value ? rotated : p.n_q);
        const int64_t page = slot >> p.page_shift, at = slot - (page << p.page_shift);
        dst = static_cast<T*>(value ? p.v_cache : p.k_cache) +
              ((((page * p.n_kv + kvh) << p.page_shift) + at) * D);
        if (value) {                      // values are copied
          oa = xa;
          ob = xb;
        }
      }
    }
    if (dst) {
      oa.store(dst + d);
      ob.store(dst + HALF + d);
    }
  }
}

// Backward: dqkv whole (the values' gradient is copied into its place) and, per workgroup, the sums of dz n over the
// workgroup's rows, which dw_kernel adds up in workgroup order (no atomics: the same bits on every run).
template <typename T, int D>
__global__ __launch_bounds__(QN_THREADS) void qk_norm_rope_bwd_kernel(const RotArgs p) {
  constexpr int LANES = D / 16, HEADS = 64 / LANES, HALF = D / 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int d = 8 * (lane % LANES), sub = lane / LANES;
  const int rotated = p.n_q + p.n_kv, total = rotated + p.n_kv;
  const int64_t items = p.tokens * p.split, stride = (int64_t)gridDim.x * QN_WAVES;
  float aq[16], ak[16];
#pragma unroll
  for (int e = 0; e < 16; e++) aq[e] = ak[e] = 0.0f;

  for (int64_t item = (int64_t)blockIdx.x * QN_WAVES + wave; item < items; item += stride) {
    const int64_t t = item / p.split;
    const int part = (int)(item - t * p.split);
    const T* row = static_cast<const T*>(p.qkv) + t * (int64_t)total * D;
    T* out = static_cast<T*>(p.dqkv) + t * (int64_t)total * D;
    const int64_t pos = p.positions[t];
    const bool known = pos >= 0 && pos < p.max_positions;
    float c1[8], c2[8], s1[8], s2[8];
    load_table<T>(p.cos_t, p.table_f32, (known ? pos : 0) * D, d, HALF, c1, c2);
    load_table<T>(p.sin_t, p.table_f32, (known ? pos : 0) * D, d, HALF, s1, s2);
    // gradient of head h of this token; null: it takes none
    auto grad_of = [&](int h) -> const T* {
      if (h < p.n_q) return p.dq ? static_cast<const T*>(p.dq) + (t * p.n_q + h) * D : nullptr;
      if (h < rotated) return p.dk ? static_cast<const T*>(p.dk) + (t * p.n_kv + (h - p.n_q)) * D : nullptr;
      if (h < total) return p.dv ? static_cast<const T*>(p.dv) + (t * p.n_kv + (h - rotated)) * D : nullptr;
      return nullptr;
    };
    Oct<T> xa, xb, ga, gb;
    auto fetch = [&](int h) {
      xa.zero(); xb.zero(); ga.zero(); gb.zero();
      if (h < rotated) {
        xa.load(row + (int64_t)h * D + d);
        xb.load(row + (int64_t)h * D + HALF + d);
      }
      const T* g = grad_of(h);
      if (g) {
        ga.load(g + d);
        gb.load(g + HALF + d);
      }
    };
    int h = part * HEADS + sub;
    fetch(h);
    for (int h0 = part * HEADS; h0 < total; h0 += p.split * HEADS) {
      const int cur = h;
      const Oct<T> va = ga, vb = gb;
      float x1[8], x2[8], g1[8], g2[8];
      xa.get(x1);
      xb.get(x2);
      ga.get(g1);
      gb.get(g2);
      h += p.split * HEADS;
      fetch(h);
      float z1[8], z2[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        z1[e] = known ? g1[e] * c1[e] + g2[e] * s2[e] : 0.0f;
        z2[e] = known ? g2[e] * c2[e] - g1[e] * s1[e] : 0.0f;
      }
      const bool is_q = cur < p.n_q;
      const T* w = static_cast<const T*>(is_q ? p.q_weight : p.k_weight);
      const bool normed = w && known && cur < rotated;   // an unknown position: no gradient, whatever its row holds
      float ss = 0.0f, dot = 0.0f;
      float v1[8], v2[8];
#pragma unroll
      for (int e = 0; e < 8; e++) { v1[e] = z1[e]; v2[e] = z2[e]; }
      if (normed) {
        Oct<T> wa, wb;
        float w1[8], w2[8];
        wa.load(w + d);
        wb.load(w + HALF + d);
        wa.get(w1);
        wb.get(w2);
#pragma unroll
        for (int e = 0; e < 8; e++) { v1[e] *= w1[e]; v2[e] *= w2[e]; }
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        ss += x1[e] * x1[e] + x2[e] * x2[e];
        dot += x1[e] * v1[e] + x2[e] * v2[e];
      }
      ss = head_sum<LANES>(ss);
      dot = head_sum<LANES>(dot);
      if (normed) {
        const float r = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
        const float k = r * r * dot * (1.0f / D);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          v1[e] = r * (v1[e] - x1[e] * k);
          v2[e] = r * (v2[e] - x2[e] * k);
          const float n1 = z1[e] * (x1[e] * r), n2 = z2[e] * (x2[e] * r);
          aq[e] += is_q ? n1 : 0.0f;
          aq[8 + e] += is_q ? n2 : 0.0f;
          ak[e] += is_q ? 0.0f : n1;
          ak[8 + e] += is_q ? 0.0f : n2;
        }
      }
      if (cur < total) {
        Oct<T> oa, ob;
        oa.set(v1);
        ob.set(v2);
        if (cur >= rotated) {
          oa = va;
          ob = vb;
        }
        oa.store(out + (int64_t)cur * D + d);
        ob.store(out + (int64_t)cur * D + HALF + d);
      }
    }
  }
  if (!p.part) return;
  // lanes that hold the same elements, then the waves, in a fixed order
#pragma unroll
  for (int e = 0; e < 16; e++) {
#pragma unroll
    for (int o = LANES; o < 64; o <<= 1) {
      aq[e] += __shfl_xor(aq[e], o, 64);
      ak[e] += __shfl_xor(ak[e], o, 64);
    }
  }
  __shared__ float acc[QN_WAVES][2][D];
  if (sub == 0) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      acc[wave][0][d + e] = aq[e];
      acc[wave][0][HALF + d + e] = aq[8 + e];
      acc[wave][1][d + e] = ak[e];
      acc[wave][1][HALF + d + e] = ak[8 + e];
    }
  }
  __syncthreads();
  const float* flat = &acc[0][0][0];
  for (int i = threadIdx.x; i < 2 * D; i += QN_THREADS) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < QN_WAVES; w++) v += flat[w * 2 * D + i];
    p.part[(int64_t)blockIdx.x * 2 * D + i] = v;
  }
}

constexpr int DW_COLS = 16, DW_ROWS = QN_THREADS / DW_COLS;
template <typename T, int D>
__global__ __launch_bounds__(QN_THREADS) void qk_norm_dw_kernel(const float* part, int n, T* dqw, T* dkw) {
  __shared__ float acc[DW_ROWS][DW_COLS];
  const int c = threadIdx.x % DW_COLS, g = threadIdx.x / DW_COLS, col = blockIdx.x * DW_COLS + c;
  float v = 0.0f;
#pragma unroll 8
  for (int i = g; i < n; i += DW_ROWS) v += part[(int64_t)i * 2 * D + col];
  acc[g][c] = v;
  __syncthreads();
  if (g) return;
  v = 0.0f;
#pragma unroll
  for (int i = 0; i < DW_ROWS; i++) v += acc[i][c];
  T* dst = col < D ? dqw : dkw;
  if (dst) dst[col % D] = Oct<T>::one(v);
}

// Waves per token: one where there are tokens enough to fill the chip with waves that walk all heads (4096 waves are
// 16 per CU), up to one per group of heads below that.
int pick_split(int64_t tokens, int heads, int head_dim) {
  const int groups = (heads * head_dim / 16 + 63) / 64;
  int64_t s = tokens > 0 ? (4096 + tokens - 1) / tokens : 1;
  return (int)(s < 1 ? 1 : s > groups ? groups : s);
}

// two per CU, as many as its registers let run at once: with 1024 the second half starts behind the first (8192 tokens of
// 32 + 8 heads 75 -> 71 us, 1001 tokens of 12 + 12 in fp32 17 -> 12)
constexpr int64_t BWD_WORKGROUPS = 512;
int64_t bwd_grid(int64_t tokens, int split) {
  const int64_t g = (tokens * split + QN_WAVES - 1) / QN_WAVES;
  return g < BWD_WORKGROUPS ? g : BWD_WORKGROUPS;
}

int check_common(const char* what, const RotArgs& a, int head_dim, int table_dtype, int dtype) {
  MTP_REQUIRE(dtype == MTP_F32 || dtype == MTP_BF16 || dtype == MTP_F16, MTP_EINVAL, "%s: dtype %d", what, dtype);
  MTP_REQUIRE(table_dtype == MTP_F32 || table_dtype == dtype, MTP_EINVAL, "%s: tables of dtype %d for tensors of %d",
              what, table_dtype, dtype);
  MTP_REQUIRE(head_dim == 64 || head_dim == 128, MTP_EUNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  MTP_REQUIRE(a.tokens >= 0 && a.n_q > 0 && a.n_kv > 0 && a.n_q <= 4096 && a.n_kv <= 4096 && a.max_positions > 0,
              MTP_EINVAL, "%s: T=%lld heads %d/%d max_positions=%lld", what, (long long)a.tokens, a.n_q, a.n_kv,
              (long long)a.max_positions);
  MTP_REQUIRE(a.tokens <= 1ll << 21, MTP_EUNSUPPORTED, "%s: T=%lld (at most 2^21)", what, (long long)a.tokens);
  MTP_REQUIRE(a.tokens == 0 || (a.qkv && a.cos_t && a.sin_t && a.positions), MTP_EINVAL, "%s: null pointer", what);
  MTP_REQUIRE(((uintptr_t)a.qkv | (uintptr_t)a.cos_t | (uintptr_t)a.sin_t | (uintptr_t)a.q_weight |
               (uintptr_t)a.k_weight | (uintptr_t)a.q_out | (uintptr_t)a.k_out | (uintptr_t)a.k_cache |
               (uintptr_t)a.v_cache | (uintptr_t)a.dq | (uintptr_t)a.dk | (uintptr_t)a.dv | (uintptr_t)a.dqkv) % 16 == 0,
              MTP_EINVAL, "%s: tensors must be 16-byte aligned", what);
  return MTP_OK;
}

template <template <typename, int> class F, typename... A>
void by_type(int dtype, int head_dim, A... args) {
  if (head_dim == 64) {
    if (dtype == MTP_F32) F<float, 64>::run(args...);
    else if (dtype == MTP_BF16) F<uint16_t, 64>::run(args...);
    else F<f16s, 64>::run(args...);
  } else {
    if (dtype == MTP_F32) F<float, 128>::run(args...);
    else if (dtype == MTP_BF16) F<uint16_t, 128>::run(args...);
    else F<f16s, 128>::run(args...);
  }
}
template <typename T, int D> struct Forward {
  static void run(const RotArgs& a, bool append, unsigned grid, hipStream_t s) {
    if (append) hipLaunchKernelGGL((qk_norm_rope_kernel<T, D, true>), dim3(grid), dim3(QN_THREADS), 0, s, a);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<T, D, false>), dim3(grid), dim3(QN_THREADS), 0, s, a);
  }
};
template <typename T, int D> struct Backward {
  static void run(const RotArgs& a, unsigned grid, void* dqw, void* dkw, hipStream_t s) {
    hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<T, D>), dim3(grid), dim3(QN_THREADS), 0, s, a);
    if (a.part)
      hipLaunchKernelGGL((qk_norm_dw_kernel<T, D>), dim3(2 * D / DW_COLS), dim3(QN_THREADS), 0, s, a.part, (int)grid,
                         static_cast<T*>(dqw), static_cast<T*>(dkw));
  }
};

int launch_forward(const char* what, RotArgs a, bool append, int head_dim, int dtype, void* stream) {
  a.split = pick_split(a.tokens, a.n_q + (append ? 2 : 1) * a.n_kv, head_dim);
  const unsigned grid = (unsigned)((a.tokens * a.split + QN_WAVES - 1) / QN_WAVES);
  by_type<Forward>(dtype, head_dim, a, append, grid, static_cast<hipStream_t>(stream));
  MTP_CHECK_LAUNCH(what);
  return MTP_OK;
}

}  // namespace

extern "C" int mtp_qk_norm_rope(const void* qkv, const void* cos_table, const void* sin_table, int table_dtype,
                                const int64_t* positions, const void* q_weight, const void* k_weight, void* q_out,
                                void* k_out, int64_t T, int n_q_heads, int n_kv_heads, int head_dim,
                                int64_t max_positions, float eps, int dtype, void* stream) {
  RotArgs a = {};
  a.qkv = qkv; a.cos_t = cos_table; a.sin_t = sin_table; a.positions = positions;
  a.q_weight = q_weight; a.k_weight = k_weight; a.q_out = q_out; a.k_out = k_out;
  a.tokens = T; a.max_positions = max_positions; a.n_q = n_q_heads; a.n_kv = n_kv_heads;
  a.table_f32 = table_dtype == MTP_F32; a.eps = eps;
  const int rc = check_common("qk_norm_rope", a, head_dim, table_dtype, dtype);
  if (rc) return rc;
  if (T == 0) return MTP_OK;
  MTP_REQUIRE(q_out && k_out, MTP_EINVAL, "qk_norm_rope: null pointer");
  return launch_forward("qk_norm_rope", a, false, head_dim, dtype, stream);
}

extern "C" int mtp_qk_norm_rope_append(const void* qkv, const void* cos_table, const void* sin_table, int table_dtype,
                                       const int64_t* positions, const int64_t* slots, const void* q_weight,
                                       const void* k_weight, void* q_out, void* k_cache, void* v_cache, int64_t T,
                                       int n_q_heads, int n_kv_heads, int head_dim, int64_t max_positions,
                                       int64_t n_pages, int64_t page_size, float eps, int dtype, void* stream) {
  RotArgs a = {};
  a.qkv = qkv; a.cos_t = cos_table; a.sin_t = sin_table; a.positions = positions; a.slots = slots;
  a.q_weight = q_weight; a.k_weight = k_weight; a.q_out = q_out; a.k_cache = k_cache; a.v_cache = v_cache;
  a.tokens = T; a.max_positions = max_positions; a.n_q = n_q_heads; a.n_kv = n_kv_heads;
  a.table_f32 = table_dtype == MTP_F32; a.eps = eps;
  MTP_REQUIRE(dtype == MTP_BF16 || dtype == MTP_F16, MTP_EUNSUPPORTED, "qk_norm_rope_append: dtype %d (bf16 or f16)",
              dtype);
  const int rc = check_common("qk_norm_rope_append", a, head_dim, table_dtype, dtype);
  if (rc) return rc;
  MTP_REQUIRE(n_pages > 0 && n_pages <= 0x7fffffffll && page_size >= 1 && page_size <= (1 << 20) &&
                  (page_size & (page_size - 1)) == 0,
              MTP_EINVAL, "qk_norm_rope_append: %lld pages of %lld (a power of two)", (long long)n_pages,
              (long long)page_size);
  if (T == 0) return MTP_OK;
  MTP_REQUIRE(q_out && k_cache && v_cache && slots, MTP_EINVAL, "qk_norm_rope_append: null pointer");
  a.page_shift = __builtin_ctzll((unsigned long long)page_size);
  a.n_slots = n_pages * page_size;
  return launch_forward("qk_norm_rope_append", a, true, head_dim, dtype, stream);
}

extern "C" int64_t mtp_qk_norm_rope_bwd_workspace_bytes(int64_t T, int n_q_heads, int n_kv_heads, int head_dim) {
  if (T <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  return bwd_grid(T, pick_split(T, n_q_heads + 2 * n_kv_heads, head_dim)) * 2 * head_dim * (int64_t)sizeof(float);
}

extern "C" int mtp_qk_norm_rope_bwd(const void* dq, const void* dk, const void* dv, const void* qkv,
                                    const void* cos_table, const void* sin_table, int table_dtype,
                                    const int64_t* positions, const void* q_weight, const void* k_weight, void* dqkv,
                                    void* dq_weight, void* dk_weight, void* workspace, int64_t workspace_bytes,
                                    int64_t T, int n_q_heads, int n_kv_heads, int head_dim, int64_t max_positions,
                                    float eps, int dtype, void* stream) {
  RotArgs a = {};
  a.dq = dq; a.dk = dk; a.dv = dv; a.dqkv = dqkv;
  a.qkv = qkv; a.cos_t = cos_table; a.sin_t = sin_table; a.positions = positions;
  a.q_weight = q_weight; a.k_weight = k_weight;
  a.tokens = T; a.max_positions = max_positions; a.n_q = n_q_heads; a.n_kv = n_kv_heads;
  a.table_f32 = table_dtype == MTP_F32; a.eps = eps;
  const int rc = check_common("qk_norm_rope_bwd", a, head_dim, table_dtype, dtype);
  if (rc) return rc;
  MTP_REQUIRE((!dq_weight || q_weight) && (!dk_weight || k_weight), MTP_EINVAL,
              "qk_norm_rope_bwd: a weight gradient without its weight");
  MTP_REQUIRE(T > 0 || !(dq_weight || dk_weight), MTP_EINVAL, "qk_norm_rope_bwd: weight gradients of no tokens");
  if (T == 0) return MTP_OK;
  MTP_REQUIRE(dqkv, MTP_EINVAL, "qk_norm_rope_bwd: null pointer");
  a.split = pick_split(T, n_q_heads + 2 * n_kv_heads, head_dim);
  const unsigned grid = (unsigned)bwd_grid(T, a.split);
  if (dq_weight || dk_weight) {
    const int64_t need = (int64_t)grid * 2 * head_dim * (int64_t)sizeof(float);
    MTP_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 4 == 0, MTP_EWORKSPACE,
                "qk_norm_rope_bwd: workspace %lld bytes, need %lld", (long long)workspace_bytes, (long long)need);
    a.part = static_cast<float*>(workspace);
  }
  by_type<Backward>(dtype, head_dim, a, grid, dq_weight, dk_weight, static_cast<hipStream_t>(stream));
  MTP_CHECK_LAUNCH("qk_norm_rope_bwd");
  return MTP_OK;
}
