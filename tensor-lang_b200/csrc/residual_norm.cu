// The norms around a block, its gate and the scaled residual, and their
// gradients:
//
//   y = alpha x + gate * (norm(u) w_post)        n = norm(y) w_pre
//
// with norm the layer norm of kernel_generator.py:1667-1810 (population
// statistics) or the root-mean-square norm.  Unfused this is six passes over
// [rows, cols]; fused, the forward reads x and u and writes y and n, and the
// backward reads x, u, dy, dn and writes dx, du (and a full gate's gradient).
//
// Gradients, with hat(v) = norm(v), r(v) its 1 / scale, c = cols:
//   G    = dy + N(dn w_pre; y)             dx = alpha G
//   P    = G gate                          du = N(P w_post; u)
//   N(g; v) = r(v) (g - [mean g] - hat(v) mean(g hat(v)))   ([.]: layer norm only)
//   dgate = G hat(u) w_post                dw_post = sum_rows P hat(u)
//   dw_pre = sum_rows dn hat(y)
// y is recomputed from x and u in the backward: it costs the same bytes as
// reading a saved y, and is the unrounded value the forward's n came from.
//
// Memory bounds the forward: 65536 x 4096 bf16 353 us, 6.1 TB/s, 0.94 of a
// copy's rate; 4096 x 8192 56 us; float32 8192 x 4096 91 us, 0.91.  The backward's
// 639 us are 5.0 TB/s: registers (column sums and three values an element) leave two
// rows of 256 threads an SM, whose sums over the row wait for one another; issue
// slots are 47% used.  The column sums' second kernel takes 8 us.  (Each kernel alone
// on one set of inputs: 1000 us; with three sets in turn the pass takes 1064.)
// The forwards that hold 16 bf16 a thread spill 24 to 48 bytes of their 64 registers.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "lm_common.cuh"

namespace tl {
namespace {

struct NormArgs {
  int64_t rows, cols;
  const void* x;
  int64_t ldx;
  const void* u;  // null: no block
  int64_t ldu;
  const void* w_post;
  const void* gate;
  int gate_mode;
  int64_t ldg;
  float alpha;
  const void* w_pre;
  float eps;
  // forward
  void* y;
  int64_t ldy;
  void* n;
  int64_t ldn;
  // backward
  const void* dy;
  int64_t lddy;
  const void* dn;
  int64_t lddn;
  void* dx;
  int64_t lddx;
  void* du;
  int64_t lddu;
  void* dgate;
  int64_t lddg;
  void* dw_post;
  void* dw_pre;
  int accumulate;
  float* part;  // [grid][2][cols]: sums over rows of G gate hat(u) (a gate per channel left out) and dn hat(y)
};

// Two float32 operations in one instruction (sm_100): the row kernels hold
// their elements in pairs, since single operations, at 92 instructions per
// element, bounded the backward by instruction issue and not by memory.
__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float hsum(float2 a) { return a.x + a.y; }

// Sums over a row's threads (the whole block), a float each in two buffers
// used in turn: a sum's writes cannot meet the last one's reads, which every
// thread ended before the barrier between them.
template <int NT>
struct RowSum {
  static constexpr int NW = NT / 32, kMost = 3;
  float* sh;  // [2][kMost][NW]
  int turn = 0;
  template <int K>
  __device__ __forceinline__ void operator()(float (&v)[K]) {
    static_assert(K <= kMost, "buffer");
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    float* b = sh + turn * kMost * NW;
    turn ^= 1;
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) b[k * NW + w] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if constexpr (NW <= 8) {
        v[k] = b[k * NW];
#pragma unroll
        for (int i = 1; i < NW; ++i) v[k] += b[k * NW + i];
      } else {
        float t = lane < NW ? b[k * NW + lane] : 0.f;
        v[k] = warp_sum(t);
      }
    }
  }
};

// A thread's elements of a row, in pairs: vector j of VEC elements at
// (j * NT + t) * VEC.
template <typename T, int NT, int VEC, int NV>
struct RowIo {
  static constexpr int E = VEC * NV, H = E / 2;
  int cols;  // at most 16 * NT
  int t;
  int left;  // cols - t * VEC: vector j exists where j * NT * VEC is below
  __device__ __forceinline__ RowIo(int cols_, int t_) : cols(cols_), t(t_), left(cols_ - t_ * VEC) {}
  __device__ __forceinline__ bool has(int j) const { return j * NT * VEC < left; }
  __device__ __forceinline__ bool in(int i) const { return has(i / VEC); }
  __device__ __forceinline__ bool full() const { return has(NV - 1); }
  // column of element i
  __device__ __forceinline__ int col(int i) const { return ((i / VEC) * NT + t) * VEC + i % VEC; }
  __device__ __forceinline__ void store(T* p, const float2 (&v)[H], bool add) const {
    p += t * VEC;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!has(j)) continue;
      float q[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int e = j * VEC + i;
        q[i] = e & 1 ? v[e / 2].y : v[e / 2].x;
      }
      if (add) {
        float o[VEC];
        ld_vec<VEC>(p + j * NT * VEC, o);
#pragma unroll
        for (int i = 0; i < VEC; ++i) q[i] += o[i];
      }
      st_vec<VEC>(p + j * NT * VEC, q);
    }
  }
};

// v becomes hat(v) for the elements a thread holds; returns 1 / scale.
// Elements past the row are zero and stay out of the centred sum.
template <bool LAYER, typename T, int NT, int VEC, int NV, int H>
__device__ __forceinline__ float normalise(const RowIo<T, NT, VEC, NV>& io, float2 (&v)[H], float inv_c,
                                           float eps, RowSum<NT>& sum) {
  float s[1];
  float2 q = pair(0.f);
  if constexpr (LAYER) {
#pragma unroll
    for (int i = 0; i < H; ++i) q = add2(q, v[i]);
    s[0] = hsum(q);
    sum(s);
    // s / cols, by one correction of s * inv_c: the mean of a constant row is
    // that constant where its sum is exact
    float m = s[0] * inv_c;
    m = fmaf(fmaf(-m, (float)io.cols, s[0]), inv_c, m);
#pragma unroll
    for (int i = 0; i < H; ++i) v[i] = add2(v[i], pair(-m));
    if (!io.full()) {
#pragma unroll
      for (int i = 0; i < H; ++i) {
        if (!io.in(2 * i)) v[i].x = 0.f;
        if (!io.in(2 * i + 1)) v[i].y = 0.f;
      }
    }
    q = pair(0.f);
  }
#pragma unroll
  for (int i = 0; i < H; ++i) q = fma2(v[i], v[i], q);
  s[0] = hsum(q);
  sum(s);
  const float r = rsqrtf(fmaf(s[0], inv_c, eps));  // within 2 ulp
#pragma unroll
  for (int i = 0; i < H; ++i) v[i] = mul2(v[i], pair(r));
  return r;
}

// A thread's elements of the rows it will work on, brought into shared memory
// ahead of time by asynchronous copies (each thread copies and reads only its
// own elements, so its own wait is enough): `depth` slots of `na` arrays.
// Element types or alignments that have no asynchronous copy (2 bytes) load
// directly.
template <typename T, int NT, int VEC, int NV, int NA>
struct Ahead {
  using Io = RowIo<T, NT, VEC, NV>;
  static constexpr bool kStaged = VEC * sizeof(T) >= 4;
  static constexpr int kBytes = VEC * sizeof(T);
  static constexpr int kArray = NT * NV * kBytes;  // bytes of one array of one row
  const void* p[NA];
  int64_t ld[NA];
  unsigned char* buf;  // [depth][na][NV][NT] vectors
  int depth, na;

  __device__ __forceinline__ void fetch(const Io& io, int64_t r, int64_t rows, int slot) const {
    if constexpr (kStaged) {
      if (r < rows) {
#pragma unroll
        for (int q = 0; q < NA; ++q) {
          if (!p[q]) continue;
          const T* src = static_cast<const T*>(p[q]) + r * ld[q] + io.t * VEC;
          const uint32_t dst = (uint32_t)__cvta_generic_to_shared(buf + (slot * na + q) * kArray +
                                                                  io.t * kBytes);
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            if (!io.has(j)) continue;
            const uint32_t d = dst + j * NT * kBytes;
            const T* from = src + j * NT * VEC;
            if constexpr (kBytes == 16)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(from) : "memory");
            else
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(from) : "memory");
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");  // an empty group past the last row
    }
  }
  // the oldest of `depth` outstanding rows has arrived
  __device__ __forceinline__ void wait() const {
    if constexpr (kStaged) {
      if (depth >= 4)
        asm volatile("cp.async.wait_group 3;" ::: "memory");
      else if (depth == 3)
        asm volatile("cp.async.wait_group 2;" ::: "memory");
      else if (depth == 2)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      else
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  }
  __device__ __forceinline__ void load(const Io& io, int q, int64_t r, int slot,
                                       float2 (&v)[Io::H]) const {
    const T* src = kStaged ? reinterpret_cast<const T*>(buf + (slot * na + q) * kArray + io.t * kBytes)
                           : static_cast<const T*>(p[q]) + r * ld[q] + io.t * VEC;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = 0.f;
      if (io.has(j)) ld_vec<VEC>(src + j * NT * VEC, e);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int k = j * VEC + i;
        (k & 1 ? v[k / 2].y : v[k / 2].x) = e[i];
      }
    }
  }
};

// A thread's elements of a weight vector, in shared memory as float32; only
// that thread writes and reads them.
template <typename T, int NT, int VEC, int NV>
struct RowWeights {
  using Io = RowIo<T, NT, VEC, NV>;
  static constexpr int H = Io::H;
  static constexpr int kBytes = NT * Io::E * 4;
  float4* p;  // [H / 2][NT]
  // w * g (either may be null: 1)
  __device__ __forceinline__ void fill(const Io& io, const T* w, const T* g) const {
#pragma unroll
    for (int i = 0; i < H / 2; ++i) {
      float e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = io.col(4 * i + k);
        e[k] = c < io.cols ? (w ? to_f32(w[c]) : 1.f) * (g ? to_f32(g[c]) : 1.f) : 0.f;
      }
      p[i * NT + io.t] = make_float4(e[0], e[1], e[2], e[3]);
    }
  }
  __device__ __forceinline__ void load(const Io& io, float2 (&v)[H]) const {
#pragma unroll
    for (int i = 0; i < H / 2; ++i) {
      const float4 q = p[i * NT + io.t];
      v[2 * i] = make_float2(q.x, q.y);
      v[2 * i + 1] = make_float2(q.z, q.w);
    }
  }
};

// One row after another per block (b, b + grid, ...), the next rows of x and u
// on their way while a row is worked on.
template <typename T, int NT, int VEC, int NV, bool LAYER>
__global__ void __launch_bounds__(NT, 1024 / NT) residual_norm_kernel(NormArgs a, int depth) {
  using Io = RowIo<T, NT, VEC, NV>;
  using W = RowWeights<T, NT, VEC, NV>;
  constexpr int H = Io::H;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ float sh[2 * 3 * (NT / 32)];
  RowSum<NT> sum{sh};
  const Io io((int)a.cols, (int)threadIdx.x);
  const float inv_c = 1.f / (float)a.cols;
  const bool full_gate = a.gate_mode == TL_GATE_FULL;
  const Ahead<T, NT, VEC, NV, 3> rows{{a.x, a.u, full_gate ? a.gate : nullptr}, {a.ldx, a.ldu, a.ldg},
                                      dyn + 2 * W::kBytes, depth, full_gate ? 3 : 2};
  wait_for_previous_kernel();
  for (int k = 0; k + 1 < depth; ++k) rows.fetch(io, blockIdx.x + (int64_t)k * gridDim.x, a.rows, k);
  const W w_post{reinterpret_cast<float4*>(dyn)}, w_pre{reinterpret_cast<float4*>(dyn + W::kBytes)};
  int slot = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, slot = slot + 1 == depth ? 0 : slot + 1) {
    rows.fetch(io, r + (int64_t)(depth - 1) * gridDim.x, a.rows, slot == 0 ? depth - 1 : slot - 1);
    if (r == blockIdx.x) {  // while the first row is on its way
      w_post.fill(io, static_cast<const T*>(a.w_post),
                  a.gate_mode == TL_GATE_CHANNEL ? static_cast<const T*>(a.gate) : nullptr);
      w_pre.fill(io, static_cast<const T*>(a.w_pre), nullptr);
    }
    rows.wait();
    float2 y[H];
    rows.load(io, 0, r, slot, y);
#pragma unroll
    for (int i = 0; i < H; ++i) y[i] = mul2(y[i], pair(a.alpha));
    if (a.u) {
      float2 v[H], w[H];
      rows.load(io, 1, r, slot, v);
      normalise<LAYER>(io, v, inv_c, a.eps, sum);
      w_post.load(io, w);
      if (full_gate) {
        float2 g[H];
        rows.load(io, 2, r, slot, g);
#pragma unroll
        for (int i = 0; i < H; ++i) w[i] = mul2(w[i], g[i]);
      } else if (a.gate_mode == TL_GATE_TOKEN) {
        const float g = to_f32(static_cast<const T*>(a.gate)[r]);
#pragma unroll
        for (int i = 0; i < H; ++i) w[i] = mul2(w[i], pair(g));
      }
#pragma unroll
      for (int i = 0; i < H; ++i) y[i] = fma2(v[i], w[i], y[i]);
    }
    if (a.y) io.store(static_cast<T*>(a.y) + r * a.ldy, y, false);
    if (a.n) {
      normalise<LAYER>(io, y, inv_c, a.eps, sum);
      float2 w[H];
      w_pre.load(io, w);
#pragma unroll
      for (int i = 0; i < H; ++i) y[i] = mul2(y[i], w[i]);
      io.store(static_cast<T*>(a.n) + r * a.ldn, y, false);
    }
  }
}

// Block b takes rows b, b + grid, ...: the column sums stay in its threads'
// registers and leave as one row of partials, which norm_sums_kernel adds in
// block order (no atomics: results do not depend on the order blocks end).
// x, u, dy and dn of the next rows are on their way while a row is worked on;
// dn and dy are read from shared memory where they are used, so that only
// hat(u), hat(y) and G are held beside the sums.  A gate per channel needs no
// sum of its own: with S = sum_rows G hat(u), dw_post = gate S and
// dgate = w_post S.
template <typename T, int NT, int VEC, int NV, bool LAYER>
__global__ void __launch_bounds__(NT, NT <= 256 ? 512 / NT : 1)
    residual_norm_bwd_kernel(NormArgs a, int depth) {
  using Io = RowIo<T, NT, VEC, NV>;
  using W = RowWeights<T, NT, VEC, NV>;
  constexpr int H = Io::H;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ float sh[2 * 3 * (NT / 32)];
  RowSum<NT> sum{sh};
  const Io io((int)a.cols, (int)threadIdx.x);
  const bool full_gate = a.gate_mode == TL_GATE_FULL, token_gate = a.gate_mode == TL_GATE_TOKEN;
  const Ahead<T, NT, VEC, NV, 5> rows{{a.u, a.x, a.dn, a.dy, full_gate ? a.gate : nullptr},
                                      {a.ldu, a.ldx, a.lddn, a.lddy, a.ldg},
                                      dyn + 2 * W::kBytes, depth, full_gate ? 5 : 4};
  const float inv_c = 1.f / (float)a.cols;
  wait_for_previous_kernel();
  for (int k = 0; k + 1 < depth; ++k) rows.fetch(io, blockIdx.x + (int64_t)k * gridDim.x, a.rows, k);
  const W w_post{reinterpret_cast<float4*>(dyn)}, w_pre{reinterpret_cast<float4*>(dyn + W::kBytes)};
  float2 s_post[H], s_pre[H];
#pragma unroll
  for (int i = 0; i < H; ++i) s_post[i] = s_pre[i] = pair(0.f);
  int slot = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, slot = slot + 1 == depth ? 0 : slot + 1) {
    rows.fetch(io, r + (int64_t)(depth - 1) * gridDim.x, a.rows, slot == 0 ? depth - 1 : slot - 1);
    if (r == blockIdx.x) {  // while the first row is on its way
      w_post.fill(io, static_cast<const T*>(a.w_post),
                  a.gate_mode == TL_GATE_CHANNEL ? static_cast<const T*>(a.gate) : nullptr);
      w_pre.fill(io, static_cast<const T*>(a.w_pre), nullptr);
    }
    rows.wait();
    const float gate_r = token_gate ? to_f32(static_cast<const T*>(a.gate)[r]) : 1.f;
    // what hat(u) is multiplied by on its way to y: w_post * gate
    auto branch_weight = [&](float2(&w)[H]) {
      w_post.load(io, w);
      if (full_gate) {
        float2 g[H];
        rows.load(io, 4, r, slot, g);
#pragma unroll
        for (int i = 0; i < H; ++i) w[i] = mul2(w[i], g[i]);
      } else if (token_gate) {
#pragma unroll
        for (int i = 0; i < H; ++i) w[i] = mul2(w[i], pair(gate_r));
      }
    };
    float2 hu[H], G[H];
    float ru = 0.f;
    if (a.u) {
      rows.load(io, 0, r, slot, hu);
      ru = normalise<LAYER>(io, hu, inv_c, a.eps, sum);
    }
    if (a.dn) {
      float2 y[H], d[H];
      rows.load(io, 1, r, slot, y);
#pragma unroll
      for (int i = 0; i < H; ++i) y[i] = mul2(y[i], pair(a.alpha));
      if (a.u) {
        branch_weight(d);
#pragma unroll
        for (int i = 0; i < H; ++i) y[i] = fma2(hu[i], d[i], y[i]);
      }
      const float ry = normalise<LAYER>(io, y, inv_c, a.eps, sum);  // y: hat(y)
      rows.load(io, 2, r, slot, d);
      float2 c0 = pair(0.f), c1 = pair(0.f);
      w_pre.load(io, G);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        s_pre[i] = fma2(d[i], y[i], s_pre[i]);
        d[i] = mul2(d[i], G[i]);
        c0 = fma2(d[i], y[i], c0);
        if (LAYER) c1 = add2(c1, d[i]);
      }
      float m[LAYER ? 2 : 1];
      m[0] = hsum(c0);
      if constexpr (LAYER) m[1] = hsum(c1);
      sum(m);
      const float2 m1 = pair(-m[0] * inv_c);
#pragma unroll
      for (int i = 0; i < H; ++i) G[i] = fma2(y[i], m1, d[i]);
      if constexpr (LAYER) {
        const float2 m0 = pair(-m[1] * inv_c);
#pragma unroll
        for (int i = 0; i < H; ++i) G[i] = add2(G[i], m0);
      }
      if (a.dy) {
        rows.load(io, 3, r, slot, d);
#pragma unroll
        for (int i = 0; i < H; ++i) G[i] = fma2(G[i], pair(ry), d[i]);
      } else {
#pragma unroll
        for (int i = 0; i < H; ++i) G[i] = mul2(G[i], pair(ry));
      }
    } else if (a.dy) {
      rows.load(io, 3, r, slot, G);
    } else {
#pragma unroll
      for (int i = 0; i < H; ++i) G[i] = pair(0.f);
    }
    if (a.dx) {
      float2 v[H];
#pragma unroll
      for (int i = 0; i < H; ++i) v[i] = mul2(G[i], pair(a.alpha));
      io.store(static_cast<T*>(a.dx) + r * a.lddx, v, a.accumulate & TL_ACC_DX);
    }
    if (!a.u) continue;
    float c[3] = {0.f, 0.f, 0.f};
    if (full_gate || token_gate) {
      float2 v[H], w[H], t = pair(0.f);
      w_post.load(io, w);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        v[i] = mul2(G[i], hu[i]);
        w[i] = mul2(v[i], w[i]);
        t = add2(t, w[i]);
      }
      c[2] = hsum(t);
      if (full_gate && a.dgate)
        io.store(static_cast<T*>(a.dgate) + r * a.lddg, w, a.accumulate & TL_ACC_DGATE);
      if (full_gate) {
        rows.load(io, 4, r, slot, w);
#pragma unroll
        for (int i = 0; i < H; ++i) s_post[i] = fma2(v[i], w[i], s_post[i]);
      } else {
#pragma unroll
        for (int i = 0; i < H; ++i) s_post[i] = fma2(v[i], pair(gate_r), s_post[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < H; ++i) s_post[i] = fma2(G[i], hu[i], s_post[i]);
    }
    const bool token = token_gate && a.dgate;
    if (!a.du && !token) continue;
    {
      float2 w[H], c0 = pair(0.f), c1 = pair(0.f);
      branch_weight(w);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        G[i] = mul2(G[i], w[i]);
        c0 = fma2(G[i], hu[i], c0);
        if (LAYER) c1 = add2(c1, G[i]);
      }
      c[0] = hsum(c0);
      c[1] = hsum(c1);
    }
    if (token) {
      sum(c);
      if (threadIdx.x == 0) {
        T* p = static_cast<T*>(a.dgate) + r;
        from_f32(p, (a.accumulate & TL_ACC_DGATE) ? to_f32(*p) + c[2] : c[2]);
      }
    } else {
      float m[LAYER ? 2 : 1];
      m[0] = c[0];
      if constexpr (LAYER) m[1] = c[1];
      sum(m);
      c[0] = m[0];
      if constexpr (LAYER) c[1] = m[1];
    }
    if (a.du) {
      const float2 m1 = pair(-c[0] * inv_c), m0 = pair(-c[1] * inv_c);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        G[i] = fma2(hu[i], m1, G[i]);
        if (LAYER) G[i] = add2(G[i], m0);
        G[i] = mul2(G[i], pair(ru));
      }
      io.store(static_cast<T*>(a.du) + r * a.lddu, G, a.accumulate & TL_ACC_DU);
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
  for (int i = 0; i < Io::E; ++i) {
    const int c = io.col(i);
    if (c >= io.cols) continue;
    part[c] = i & 1 ? s_post[i / 2].y : s_post[i / 2].x;
    part[a.cols + c] = i & 1 ? s_pre[i / 2].y : s_pre[i / 2].x;
  }
}

// Adds the partials of `blocks` blocks: 32 columns of one of the outputs per
// block (0 dw_post, 1 dw_pre, 2 dgate of a gate per channel); warp w adds
// partial rows w, w + 32, ... in turn, then the warps in order.
template <typename T>
__global__ void __launch_bounds__(1024) norm_sums_kernel(NormArgs a, int64_t blocks) {
  __shared__ float sh[32][33];
  wait_for_previous_kernel();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, which = blockIdx.y;
  const bool channel = a.gate_mode == TL_GATE_CHANNEL;
  T* out = static_cast<T*>(which == 0 ? a.dw_post : which == 1 ? a.dw_pre : a.dgate);
  if (!out || (which == 2 && !channel)) return;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  const float* part = a.part + (which == 1 ? a.cols : 0);
  float s = 0.f;
  if (c < a.cols) {
#pragma unroll 4
    for (int64_t b = w; b < blocks; b += 32) s += part[b * 2 * a.cols + c];
  }
  sh[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < a.cols) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += sh[k][lane];
    // (no rows: a gate may not exist, and 0 times an infinity is not 0)
    if (which == 0 && channel && blocks > 0) t *= to_f32(static_cast<const T*>(a.gate)[c]);
    if (which == 2 && a.w_post && blocks > 0) t *= to_f32(static_cast<const T*>(a.w_post)[c]);
    const int flag = which == 0 ? TL_ACC_DW_POST : which == 1 ? TL_ACC_DW_PRE : TL_ACC_DGATE;
    from_f32(out + c, (a.accumulate & flag) ? to_f32(out[c]) + t : t);
  }
}

// Rows longer than the register kernels take: every pass reads the row again
// (from L2), one block per row, an element at a time: 8192 x 12288 bf16 762 us
// forward and 3.17 ms with the gradients, where the bytes take 124 and 311.
constexpr int kLong = 1024;

template <typename T, bool LAYER>
struct LongRow {
  const NormArgs& a;
  int64_t r;
  float* sh;
  float inv_c;
  __device__ float sum(float v) const {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    v = warp_sum(v);
    __syncthreads();  // the previous sum's readers are done
    if (lane == 0) sh[w] = v;
    __syncthreads();
    return warp_sum(sh[lane]);
  }
  template <typename F>
  __device__ float total(F f) const {
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < a.cols; c += kLong) s += f(c);
    return sum(s);
  }
  // mean and 1 / scale of the values f(c)
  template <typename F>
  __device__ float2 stats(F f) const {
    const float mean = LAYER ? total(f) / (float)a.cols : 0.f;
    const float q = total([&](int64_t c) { const float d = f(c) - mean; return d * d; });
    return make_float2(mean, 1.f / sqrtf(q * inv_c + a.eps));
  }
  __device__ float at(const void* p, int64_t i) const { return to_f32(static_cast<const T*>(p)[i]); }
  __device__ float w_post(int64_t c) const { return a.w_post ? at(a.w_post, c) : 1.f; }
  __device__ float w_pre(int64_t c) const { return a.w_pre ? at(a.w_pre, c) : 1.f; }
  __device__ float gate(int64_t c) const {
    return a.gate_mode == TL_GATE_CHANNEL ? at(a.gate, c)
           : a.gate_mode == TL_GATE_TOKEN ? at(a.gate, r)
           : a.gate_mode == TL_GATE_FULL  ? at(a.gate, r * a.ldg + c)
                                          : 1.f;
  }
  __device__ float u(int64_t c) const { return at(a.u, r * a.ldu + c); }
  __device__ float y(int64_t c, float2 su) const {
    const float v = a.alpha * at(a.x, r * a.ldx + c);
    return a.u ? v + (u(c) - su.x) * su.y * w_post(c) * gate(c) : v;
  }
};

template <typename T, bool LAYER>
__global__ void __launch_bounds__(kLong) residual_norm_long_kernel(NormArgs a) {
  __shared__ float sh[32];
  wait_for_previous_kernel();
  const float inv_c = 1.f / (float)a.cols;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const LongRow<T, LAYER> R{a, r, sh, inv_c};
    const float2 su = a.u ? R.stats([&](int64_t c) { return R.u(c); }) : make_float2(0.f, 0.f);
    float2 sy = make_float2(0.f, 0.f);
    if (a.n) sy = R.stats([&](int64_t c) { return R.y(c, su); });
    for (int64_t c = threadIdx.x; c < a.cols; c += kLong) {
      const float y = R.y(c, su);
      if (a.y) from_f32(static_cast<T*>(a.y) + r * a.ldy + c, y);
      if (a.n) from_f32(static_cast<T*>(a.n) + r * a.ldn + c, (y - sy.x) * sy.y * R.w_pre(c));
    }
  }
}

template <typename T, bool LAYER>
__global__ void __launch_bounds__(kLong) residual_norm_bwd_long_kernel(NormArgs a) {
  __shared__ float sh[32];
  wait_for_previous_kernel();
  const float inv_c = 1.f / (float)a.cols;
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.cols;
  for (int64_t c = threadIdx.x; c < 2 * a.cols; c += kLong) part[c] = 0.f;
  __syncthreads();  // column c's partials belong to thread c % kLong below
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const LongRow<T, LAYER> R{a, r, sh, inv_c};
    const float2 su = a.u ? R.stats([&](int64_t c) { return R.u(c); }) : make_float2(0.f, 0.f);
    float2 sy = make_float2(0.f, 0.f);
    float m1 = 0.f, m0 = 0.f;
    auto hat_y = [&](int64_t c) { return (R.y(c, su) - sy.x) * sy.y; };
    auto gn = [&](int64_t c) { return R.at(a.dn, r * a.lddn + c) * R.w_pre(c); };
    if (a.dn) {
      sy = R.stats([&](int64_t c) { return R.y(c, su); });
      m1 = R.total([&](int64_t c) { return gn(c) * hat_y(c); }) * inv_c;
      if (LAYER) m0 = R.total(gn) * inv_c;
    }
    auto G = [&](int64_t c) {
      float g = a.dy ? R.at(a.dy, r * a.lddy + c) : 0.f;
      if (a.dn) g += sy.y * (gn(c) - m0 - hat_y(c) * m1);
      return g;
    };
    auto hat_u = [&](int64_t c) { return (R.u(c) - su.x) * su.y; };
    float e1 = 0.f, e0 = 0.f;
    if (a.u) {
      if (a.du) {
        e1 = R.total([&](int64_t c) { return G(c) * R.gate(c) * R.w_post(c) * hat_u(c); }) * inv_c;
        if (LAYER) e0 = R.total([&](int64_t c) { return G(c) * R.gate(c) * R.w_post(c); }) * inv_c;
      }
      if (a.dgate && a.gate_mode == TL_GATE_TOKEN) {
        const float s = R.total([&](int64_t c) { return G(c) * hat_u(c) * R.w_post(c); });
        if (threadIdx.x == 0) {
          T* p = static_cast<T*>(a.dgate) + r;
          from_f32(p, (a.accumulate & TL_ACC_DGATE) ? to_f32(*p) + s : s);
        }
      }
    }
    // every element's inputs are read before its outputs are written (dx may
    // be dy, du may be dn), and no pass over the row follows
    for (int64_t c = threadIdx.x; c < a.cols; c += kLong) {
      const float g = G(c);
      if (a.dn) part[a.cols + c] += R.at(a.dn, r * a.lddn + c) * hat_y(c);
      float du = 0.f, dg = 0.f;
      if (a.u) {
        const float p = g * R.gate(c), h = hat_u(c);
        part[c] += (a.gate_mode == TL_GATE_CHANNEL ? g : p) * h;
        dg = g * h * R.w_post(c);
        du = su.y * (p * R.w_post(c) - e0 - h * e1);
      }
      if (a.dx) {
        T* p = static_cast<T*>(a.dx) + r * a.lddx + c;
        from_f32(p, ((a.accumulate & TL_ACC_DX) ? to_f32(*p) : 0.f) + a.alpha * g);
      }
      if (a.u && a.du) {
        T* p = static_cast<T*>(a.du) + r * a.lddu + c;
        from_f32(p, ((a.accumulate & TL_ACC_DU) ? to_f32(*p) : 0.f) + du);
      }
      if (a.u && a.dgate && a.gate_mode == TL_GATE_FULL) {
        T* p = static_cast<T*>(a.dgate) + r * a.lddg + c;
        from_f32(p, ((a.accumulate & TL_ACC_DGATE) ? to_f32(*p) : 0.f) + dg);
      }
    }
  }
}

// ------------------------------------------------------------- host side ---
constexpr int64_t kMaxCols = 8192;    // of the register kernels
constexpr int kSmemMost = 226 << 10;  // dynamic, beside the sums' few hundred bytes
constexpr int64_t kSmem = 216 << 10;  // of an SM, for weights and rows on their way

// Elements a thread holds: 16 bf16, or 8 float32, whose rows and weights on
// their way take 384 bytes a thread in the backward (16 would leave 288 threads
// an SM).  The longest bf16 rows of a forward take 8 as well: one block of 1024
// threads has room for two rows on their way beside the weights.
template <typename T>
constexpr int kElems = sizeof(T) == 4 ? 8 : 16;

// Threads per row, so that a row fits: 64 to 1024.
template <int E, typename F>
int by_width(int64_t cols, F f) {
  if (cols <= 64 * E) return f(std::integral_constant<int, 64>{});
  if (cols <= 128 * E) return f(std::integral_constant<int, 128>{});
  if (cols <= 256 * E) return f(std::integral_constant<int, 256>{});
  if constexpr (512 * E < kMaxCols) {
    if (cols <= 512 * E) return f(std::integral_constant<int, 512>{});
    return f(std::integral_constant<int, kMaxCols / E>{});
  } else {
    return f(std::integral_constant<int, 512>{});
  }
}

// Blocks of the backward at most (rows of its partials): 512 threads an SM.
int64_t bwd_blocks(int64_t rows, int64_t cols) {
  const int64_t per_sm = cols > 4096 ? 1 : cols > 2048 ? 2 : cols > 1024 ? 4 : 8;
  return std::max<int64_t>(1, std::min<int64_t>(rows, per_sm * sm_count()));
}

// Blocks an SM holds and rows each has on its way: two rows (the one worked on
// and the next) where that leaves at least 256 threads an SM, else one; at most
// four rows.
struct Shape {
  int64_t grid;
  int depth;
};
Shape launch_shape(int64_t rows, int nt, int64_t most_threads, int64_t row_bytes, int64_t weight_bytes,
                   int64_t most_blocks) {
  int64_t per_sm = std::max<int64_t>(1, most_threads / nt);
  auto fit = [&](int64_t blocks) { return (kSmem / blocks - weight_bytes - 1024) / row_bytes; };
  while (per_sm > 1 && (fit(per_sm) < 1 || (fit(per_sm) < 2 && (per_sm - 1) * nt >= 256 && nt <= 256))) --per_sm;
  Shape q;
  q.grid = std::min<int64_t>({rows, per_sm * sm_count(), most_blocks});
  q.depth = (int)std::max<int64_t>(1, std::min<int64_t>({fit(per_sm), 4, (rows + q.grid - 1) / q.grid}));
  return q;
}

template <auto Kern>
int launch_rows(const NormArgs& a, Shape q, int nt, int64_t row_bytes, int64_t weight_bytes,
                cudaStream_t st) {
  const size_t smem = (size_t)(weight_bytes + q.depth * row_bytes);
  if (smem > kSmemMost) return TL_ERR_UNSUPPORTED;
  TL_TRY((allow_smem<Kern, kSmemMost>()));
  // not ahead of the previous kernel's end: blocks that came early would crowd
  // the SMs free at that moment, and each block has its share of the rows
  // (3001 x 1021 float32 training pass 72 us instead of 56)
  Kern<<<(unsigned)q.grid, nt, smem, st>>>(a, q.depth);
  return after_launch();
}

template <typename T, int VEC, int E>
int forward(const NormArgs& a, int kind, cudaStream_t st) {
  return by_width<E>(a.cols, [&](auto threads) {
    constexpr int NT = decltype(threads)::value, NV = E / VEC;
    using A = Ahead<T, NT, VEC, NV, 3>;
    const int64_t w = 2 * RowWeights<T, NT, VEC, NV>::kBytes;
    const int64_t row = A::kStaged ? (a.gate_mode == TL_GATE_FULL ? 3 : 2) * A::kArray : 16;
    const Shape q = launch_shape(a.rows, NT, 1024, row, w, INT32_MAX);
    return kind == TL_NORM_LAYER
               ? launch_rows<residual_norm_kernel<T, NT, VEC, NV, true>>(a, q, NT, row, w, st)
               : launch_rows<residual_norm_kernel<T, NT, VEC, NV, false>>(a, q, NT, row, w, st);
  });
}

// grid: the partials' rows
template <typename T, int VEC>
int backward(const NormArgs& a, int kind, cudaStream_t st, int64_t* grid) {
  constexpr int E = kElems<T>;
  return by_width<E>(a.cols, [&](auto threads) {
    constexpr int NT = decltype(threads)::value, NV = E / VEC;
    using A = Ahead<T, NT, VEC, NV, 5>;
    const int64_t w = 2 * RowWeights<T, NT, VEC, NV>::kBytes;
    const int64_t row = A::kStaged ? (a.gate_mode == TL_GATE_FULL ? 5 : 4) * A::kArray : 16;
    const Shape q = launch_shape(a.rows, NT, 512, row, w, bwd_blocks(a.rows, a.cols));
    *grid = q.grid;
    return kind == TL_NORM_LAYER
               ? launch_rows<residual_norm_bwd_kernel<T, NT, VEC, NV, true>>(a, q, NT, row, w, st)
               : launch_rows<residual_norm_bwd_kernel<T, NT, VEC, NV, false>>(a, q, NT, row, w, st);
  });
}

// Whether rows of p (leading dimension ld) take 128-bit accesses.
bool vec_rows(const void* p, int64_t ld, int64_t vec) {
  return !p || (aligned_to(p, 16) && ld % vec == 0);
}

bool vec_ok(const NormArgs& a, int64_t vec) {
  if (a.cols % vec) return false;
  const bool gate_rows = a.gate_mode == TL_GATE_FULL, gate_vec = a.gate_mode == TL_GATE_CHANNEL;
  if (gate_rows && !(vec_rows(a.gate, a.ldg, vec) && vec_rows(a.dgate, a.lddg, vec))) return false;
  if (gate_vec && !(vec_rows(a.gate, 0, vec))) return false;
  return vec_rows(a.x, a.ldx, vec) && vec_rows(a.u, a.ldu, vec) && vec_rows(a.w_post, 0, vec) &&
         vec_rows(a.w_pre, 0, vec) && vec_rows(a.y, a.ldy, vec) && vec_rows(a.n, a.ldn, vec) &&
         vec_rows(a.dy, a.lddy, vec) && vec_rows(a.dn, a.lddn, vec) &&
         vec_rows(a.dx, a.lddx, vec) && vec_rows(a.du, a.lddu, vec);
}

template <typename T>
int run_forward(const NormArgs& a, int kind, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (a.cols > kMaxCols) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 2LL * sm_count());
    if (kind == TL_NORM_LAYER)
      residual_norm_long_kernel<T, true><<<grid, kLong, 0, st>>>(a);
    else
      residual_norm_long_kernel<T, false><<<grid, kLong, 0, st>>>(a);
    return after_launch();
  }
  constexpr int E = kElems<T>;
  if (vec_ok(a, V))
    return a.cols > 4096 ? forward<T, V, 8>(a, kind, st) : forward<T, V, E>(a, kind, st);
  return a.cols > 4096 ? forward<T, 1, 8>(a, kind, st) : forward<T, 1, E>(a, kind, st);
}

template <typename T>
int run_backward(const NormArgs& a, int kind, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  int64_t blocks = 0;
  if (a.rows > 0) {
    if (a.cols > kMaxCols) {
      blocks = bwd_blocks(a.rows, a.cols);
      const unsigned grid = (unsigned)blocks;
      if (kind == TL_NORM_LAYER)
        residual_norm_bwd_long_kernel<T, true><<<grid, kLong, 0, st>>>(a);
      else
        residual_norm_bwd_long_kernel<T, false><<<grid, kLong, 0, st>>>(a);
      TL_TRY(after_launch());
    } else {
      TL_TRY((vec_ok(a, V) ? backward<T, V>(a, kind, st, &blocks) : backward<T, 1>(a, kind, st, &blocks)));
    }
  }
  if (a.dw_post || a.dw_pre || (a.dgate && a.gate_mode == TL_GATE_CHANNEL)) {
    TL_TRY(launch(norm_sums_kernel<T>, dim3((unsigned)((a.cols + 31) / 32), 3), 1024, 0, st, a, blocks));
  }
  return TL_OK;
}

// Arguments common to both directions.
int check(int dtype, int kind, const NormArgs& a) {
  if (!dtype_ok(dtype) || (kind != TL_NORM_LAYER && kind != TL_NORM_RMS)) return TL_ERR_INVALID_ARG;
  if (a.rows < 0 || a.cols <= 0 || a.rows > INT32_MAX || a.cols > INT32_MAX)
    return TL_ERR_INVALID_ARG;
  if (a.rows > 0 && !a.x) return TL_ERR_INVALID_ARG;
  if (a.gate_mode < TL_GATE_NONE || a.gate_mode > TL_GATE_FULL) return TL_ERR_INVALID_ARG;
  if (a.rows > 0 && a.u && a.gate_mode != TL_GATE_NONE && !a.gate) return TL_ERR_INVALID_ARG;
  if (!(a.eps >= 0.f) || a.alpha != a.alpha) return TL_ERR_INVALID_ARG;
  if (a.ldx < a.cols || (a.u && a.ldu < a.cols)) return TL_ERR_INVALID_ARG;
  if (a.u && a.gate_mode == TL_GATE_FULL && a.ldg < a.cols) return TL_ERR_INVALID_ARG;
  return TL_OK;
}

}  // namespace
}  // namespace tl

extern "C" {

int tl_residual_norm(int dtype, int kind, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                     const void* u, int64_t ldu, const void* w_post, const void* gate,
                     int gate_mode, int64_t ldg, float alpha, const void* w_pre, float eps, void* y,
                     int64_t ldy, void* n, int64_t ldn, void* stream) {
  tl::NormArgs a{};
  a.rows = rows; a.cols = cols; a.x = x; a.ldx = ldx; a.u = u; a.ldu = ldu;
  a.w_post = u ? w_post : nullptr;
  a.gate_mode = u ? gate_mode : TL_GATE_NONE;
  a.gate = a.gate_mode == TL_GATE_NONE ? nullptr : gate;
  a.ldg = ldg; a.alpha = alpha; a.w_pre = w_pre; a.eps = eps;
  a.y = y; a.ldy = ldy; a.n = n; a.ldn = ldn;
  if (gate_mode < TL_GATE_NONE || gate_mode > TL_GATE_FULL) return TL_ERR_INVALID_ARG;
  TL_TRY(tl::check(dtype, kind, a));
  if ((rows > 0 && !y && !n) || (y && ldy < cols) || (n && ldn < cols)) return TL_ERR_INVALID_ARG;
  if (y && y == n) return TL_ERR_INVALID_ARG;
  // an output over an operand: row on row
  auto other_rows = [&](const void* p, int64_t ldp, const void* q, int64_t ldq) {
    return p && p == q && ldp != ldq && rows > 1;
  };
  if (other_rows(y, ldy, x, ldx) || other_rows(y, ldy, u, ldu) || other_rows(n, ldn, x, ldx) ||
      other_rows(n, ldn, u, ldu))
    return TL_ERR_INVALID_ARG;
  if (rows == 0) return TL_OK;
  cudaStream_t st = tl::stream_or_default(stream);
  return dtype == TL_BF16 ? tl::run_forward<__nv_bfloat16>(a, kind, st)
                          : tl::run_forward<float>(a, kind, st);
}

size_t tl_residual_norm_scratch_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols <= 0) return 0;
  return (size_t)tl::bwd_blocks(rows, cols) * 2 * (size_t)cols * sizeof(float);
}

int tl_residual_norm_backward(int dtype, int kind, int64_t rows, int64_t cols, const void* x,
                              int64_t ldx, const void* u, int64_t ldu, const void* w_post,
                              const void* gate, int gate_mode, int64_t ldg, float alpha,
                              const void* w_pre, float eps, const void* dy, int64_t lddy,
                              const void* dn, int64_t lddn, void* dx, int64_t lddx, void* du,
                              int64_t lddu, void* dgate, int64_t lddg, void* dw_post, void* dw_pre,
                              int accumulate, void* scratch, size_t scratch_bytes, void* stream) {
  tl::NormArgs a{};
  a.rows = rows; a.cols = cols; a.x = x; a.ldx = ldx; a.u = u; a.ldu = ldu;
  const bool block = u || rows == 0;  // arrays of no rows are null as well
  a.w_post = block ? w_post : nullptr;
  a.gate_mode = block ? gate_mode : TL_GATE_NONE;
  a.gate = a.gate_mode == TL_GATE_NONE ? nullptr : gate;
  a.ldg = ldg; a.alpha = alpha; a.w_pre = w_pre; a.eps = eps;
  a.dy = dy; a.lddy = lddy; a.dn = dn; a.lddn = lddn;
  a.dx = dx; a.lddx = lddx; a.du = du; a.lddu = lddu; a.dgate = dgate; a.lddg = lddg;
  a.dw_post = dw_post; a.dw_pre = dw_pre; a.accumulate = accumulate;
  a.part = static_cast<float*>(scratch);
  if (gate_mode < TL_GATE_NONE || gate_mode > TL_GATE_FULL) return TL_ERR_INVALID_ARG;
  TL_TRY(tl::check(dtype, kind, a));
  if ((dy && lddy < cols) || (dn && lddn < cols) || (dx && lddx < cols) || (du && lddu < cols))
    return TL_ERR_INVALID_ARG;
  // gradients of what the call does not have
  if (!block && (du || dw_post || dgate)) return TL_ERR_INVALID_ARG;
  if (dgate && (gate_mode == TL_GATE_NONE || dgate == gate)) return TL_ERR_INVALID_ARG;
  if (dgate && gate_mode == TL_GATE_FULL && lddg < cols) return TL_ERR_INVALID_ARG;
  if (accumulate < 0 || accumulate > 31) return TL_ERR_INVALID_ARG;
  if ((dx && dx == du) || (dw_post && dw_post == dw_pre)) return TL_ERR_INVALID_ARG;
  // an output over an operand: row on row, and only where it is read first
  auto other_rows = [&](const void* p, int64_t ldp, const void* q, int64_t ldq) {
    return p && p == q && ldp != ldq && rows > 1;
  };
  if (other_rows(dx, lddx, dy, lddy) || other_rows(du, lddu, dn, lddn)) return TL_ERR_INVALID_ARG;
  if (dgate && (dgate == dx || dgate == du || dgate == dw_post || dgate == dw_pre)) return TL_ERR_INVALID_ARG;
  if (gate_mode == TL_GATE_FULL && gate && (dx == gate || du == gate)) return TL_ERR_INVALID_ARG;
  if (gate_mode == TL_GATE_CHANNEL && ((dw_post && (dw_post == gate || dw_post == w_post)) ||
                                       (dgate && dgate == w_post)))
    return TL_ERR_INVALID_ARG;
  if (rows > 0 && !dx && !du && !dgate && !dw_post && !dw_pre) return TL_ERR_INVALID_ARG;
  if (!scratch || !tl::aligned_to(scratch, 16) ||
      scratch_bytes < tl_residual_norm_scratch_bytes(rows, cols))
    return TL_ERR_INVALID_ARG;
  cudaStream_t st = tl::stream_or_default(stream);
  return dtype == TL_BF16 ? tl::run_backward<__nv_bfloat16>(a, kind, st)
                          : tl::run_backward<float>(a, kind, st);
}

}  // extern "C"
