// The products of linear_ce.cu for few rows of float32: W is read once for each
// (4 bytes an element, what bounds them), by the ordinary float32 units.  The
// tensor cores' way writes W as three bf16 terms first and reads those, 16 bytes
// an element in all, and multiplies 128 rows however few exist.  Forward / whole
// training pass, us, here and there: 20000 classes x 2048, 1 row 47 / 171 and 198 /
// 531, 16 rows 81 / 367 and 200 / 525, 24 rows 129 / 739 and 204 / 530 (here the
// multiplications bound it by then, so 16 rows are the most); 32000 x 4096, 8 rows
// 179 / 677 and 604 / 1609; 50021 x 1000, 16 rows 117 / 465 and 197 / 597; 131072 x
// 1024, 16 rows 209 / 905 and 516 / 1438; 2000 x 512, 16 rows, training 82 and 89.
// A training pass reads W three times (the logits, again in the backward, dx) and
// writes dW: 101 us of the 171 at one row are those 655 MB.
//
//   few_rowdot_kernel   out[t][r] = sum_c a[t][c] W[r][c]
//   few_coldot_kernel   out[t][c] = sum_r a[t][r] W[r][c]
//   few_outer_kernel    O[r][c] = scale sum_t p[t][r] q[t][c] (+ O)
//
// The first two leave a sum per split of the long axis, [split][t][.], so that
// few outputs still fill the GPU; the reader adds them in order.  The logits of
// few rows are small beside W, so they are kept in scratch within a call.
#pragma once

namespace tl {
namespace {

constexpr int kFewRows = 16;
constexpr int64_t kStatBlocks = 64;  // partials of a row at most
constexpr int kFewThreads = 256, kFewWarps = 8;
constexpr int kFewPerWarp = 8;  // rows of W a warp of few_rowdot_kernel works on

// Four elements of a row of n from column c: consecutive (VEC 4) or 32 apart.
template <int VEC>
__device__ __forceinline__ void load4(const float* row, int64_t c, int64_t n, float (&v)[4]) {
  if (VEC == 4 && c + 4 <= n) {
    const float4 q = ld_stream4(row + c);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = VEC == 4 ? c + j : c + 32 * j;
      v[j] = i < n ? __ldcs(row + i) : 0.f;
    }
  }
}

// A warp works on RW rows of W at once, its lanes along the columns; the a of
// 128 columns in shared memory for the block's warps.
template <int TT, int VEC>
__global__ void __launch_bounds__(kFewThreads)
    few_rowdot_kernel(const float* __restrict__ W, int64_t ldw, int64_t R, int64_t C, const float* __restrict__ a,
                      int64_t lda, int T, float* __restrict__ out, int64_t ldo) {
  constexpr int RW = kFewPerWarp, N = TT * RW, PER = (TT * 128 + kFewThreads - 1) / kFewThreads;
  __shared__ __align__(16) float xs[2][TT][128];
  wait_for_previous_kernel();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int64_t r0 = ((int64_t)blockIdx.x * kFewWarps + w) * RW;
  const int64_t chunks = (C + 127) / 128;
  const int64_t begin = chunks * blockIdx.y / gridDim.y, end = chunks * (blockIdx.y + 1) / gridDim.y;
  float acc[N], wv[RW][4], px[PER];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  auto fetch_w = [&](int64_t ch) {
#pragma unroll
    for (int k = 0; k < RW; ++k) {
      if (r0 + k < R)
        load4<VEC>(W + (r0 + k) * ldw, ch * 128 + (VEC == 4 ? 4 * lane : lane), C, wv[k]);
      else
        wv[k][0] = wv[k][1] = wv[k][2] = wv[k][3] = 0.f;
    }
  };
  auto fetch_x = [&](int64_t ch) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * kFewThreads + tid, t = e >> 7;
      const int64_t c = ch * 128 + (e & 127);
      px[i] = t < T && c < C ? a[t * lda + c] : 0.f;
    }
  };
  auto keep_x = [&](int buf) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * kFewThreads + tid;
      if (e < TT * 128) xs[buf][e >> 7][e & 127] = px[i];
    }
  };
  if (begin < end) {
    fetch_w(begin);
    fetch_x(begin);
    keep_x(0);
  }
  __syncthreads();
  int buf = 0;
  for (int64_t ch = begin; ch < end; ++ch, buf ^= 1) {
    float cur[RW][4];
#pragma unroll
    for (int k = 0; k < RW; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) cur[k][j] = wv[k][j];
    if (ch + 1 < end) {
      fetch_w(ch + 1);
      fetch_x(ch + 1);
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float x[4];
      if constexpr (VEC == 4) {
        const float4 q = *reinterpret_cast<const float4*>(&xs[buf][t][4 * lane]);
        x[0] = q.x; x[1] = q.y; x[2] = q.z; x[3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = xs[buf][t][lane + 32 * j];
      }
#pragma unroll
      for (int k = 0; k < RW; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t * RW + k] = fmaf(cur[k][j], x[j], acc[t * RW + k]);
    }
    if (ch + 1 < end) keep_x(buf ^ 1);
    __syncthreads();
  }
  // value i of every 32 (or all N) ends in lane i
  constexpr int G = N < 32 ? N : 32;
#pragma unroll
  for (int g = 0; g < N; g += G) {
    float s = column_sum_of<G>(acc + g, lane);
#pragma unroll
    for (int o = G; o < 32; o *= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int i = g + lane, t = i / RW;
    const int64_t r = r0 + i % RW;
    if (lane < G && t < T && r < R) out[((int64_t)blockIdx.y * T + t) * ldo + r] = s;
  }
}

// The terms of rows r0 .. r0 + ROWS of W as pairs (v, v), a row's together: the
// operands of two multiplications by one instruction.
template <int TT>
struct FewPairs {
  static constexpr int ROWS = 64;
  static constexpr int LD = TT + 2;  // pairs; rows begin at other banks
  static constexpr int PER = (TT * ROWS + kFewThreads - 1) / kFewThreads;
  float2 v[ROWS][LD];
};

// 128 columns per block, its warps take rows in turn.
template <int TT, int VEC>
__global__ void __launch_bounds__(kFewThreads)
    few_coldot_kernel(const float* __restrict__ W, int64_t ldw, int64_t R, int64_t C, const float* __restrict__ a,
                      int64_t lda, int T, float* __restrict__ out, int64_t ldo) {
  using Pairs = FewPairs<TT>;
  constexpr int PER = Pairs::PER, ROWS = Pairs::ROWS, RW = ROWS / kFewWarps;
  __shared__ __align__(16) Pairs as;
  __shared__ float red[TT][128];
  wait_for_previous_kernel();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int64_t c = (int64_t)blockIdx.x * 128 + (VEC == 4 ? 4 * lane : lane);
  const int64_t begin = R * blockIdx.y / gridDim.y, end = R * (blockIdx.y + 1) / gridDim.y;
  float2 acc[TT][2];
  float wv[RW][4], pa[PER];
#pragma unroll
  for (int t = 0; t < TT; ++t) acc[t][0] = acc[t][1] = make_float2(0.f, 0.f);
  auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int k = 0; k < RW; ++k) {
      const int64_t r = r0 + w * RW + k;
      if (r < end)
        load4<VEC>(W + r * ldw, c, C, wv[k]);
      else
        wv[k][0] = wv[k][1] = wv[k][2] = wv[k][3] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * kFewThreads + tid, t = e / ROWS;
      const int64_t r = r0 + e % ROWS;
      pa[i] = t < T && r < end ? a[t * lda + r] : 0.f;
    }
  };
  if (begin < end) fetch(begin);
  for (int64_t r0 = begin; r0 < end; r0 += ROWS) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * kFewThreads + tid;
      if (e < TT * ROWS) as.v[e % ROWS][e / ROWS] = make_float2(pa[i], pa[i]);
    }
    __syncthreads();
    float2 cur[RW][2];
#pragma unroll
    for (int k = 0; k < RW; ++k) {
      cur[k][0] = make_float2(wv[k][0], wv[k][1]);
      cur[k][1] = make_float2(wv[k][2], wv[k][3]);
    }
    if (r0 + ROWS < end) fetch(r0 + ROWS);
#pragma unroll
    for (int k = 0; k < RW; ++k) {
      const float2* p = as.v[w * RW + k];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const float2 q = p[t];
        acc[t][0] = __ffma2_rn(cur[k][0], q, acc[t][0]);
        acc[t][1] = __ffma2_rn(cur[k][1], q, acc[t][1]);
      }
    }
  }
  for (int turn = 0; turn < kFewWarps; ++turn) {  // the warps' sums, in order
    if (w == turn) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const float v[4] = {acc[t][0].x, acc[t][0].y, acc[t][1].x, acc[t][1].y};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float& s = red[t][VEC == 4 ? 4 * lane + j : lane + 32 * j];
          s = turn == 0 ? v[j] : s + v[j];
        }
      }
    }
    __syncthreads();
  }
  for (int e = tid; e < T * 128; e += kFewThreads) {
    const int64_t at = (int64_t)blockIdx.x * 128 + (e & 127);
    if (at < C) out[((int64_t)blockIdx.y * T + (e >> 7)) * ldo + at] = red[e >> 7][e & 127];
  }
}

// 128 columns by kFewOuterRows rows per block; a thread's q stay in registers.
constexpr int kFewOuterRows = 256;
template <int TT, int VEC>
__global__ void __launch_bounds__(kFewThreads)
    few_outer_kernel(const float* __restrict__ p, int64_t ldp, const float* __restrict__ q, int64_t ldq, int T,
                     Targets keep, int64_t R, int64_t C, const float* scale, float* __restrict__ O, int64_t ldo,
                     int accumulate) {
  using Pairs = FewPairs<TT>;
  constexpr int PER = Pairs::PER, ROWS = Pairs::ROWS, RW = ROWS / kFewWarps;
  __shared__ __align__(16) Pairs as;
  __shared__ int kept[TT];
  wait_for_previous_kernel();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (tid < TT) kept[tid] = tid < T && keep.at(tid) >= 0;  // others: no NaN of theirs meets g = 0
  __syncthreads();
  const float k = *scale;
  const int64_t c = (int64_t)blockIdx.x * 128 + (VEC == 4 ? 4 * lane : lane);
  const int64_t begin = (int64_t)blockIdx.y * kFewOuterRows, end = min(R, begin + kFewOuterRows);
  float2 v[TT][2];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    v[t][0] = v[t][1] = make_float2(0.f, 0.f);
    if (kept[t]) {
      float* f = reinterpret_cast<float*>(v[t]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t i = VEC == 4 ? c + j : c + 32 * j;
        f[j] = i < C ? k * q[t * ldq + i] : 0.f;
      }
    }
  }
  for (int64_t r0 = begin; r0 < end; r0 += ROWS) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * kFewThreads + tid, t = e / ROWS;
      const int64_t r = r0 + e % ROWS;
      if (e >= TT * ROWS) continue;
      const float x = kept[t] && r < end ? p[t * ldp + r] : 0.f;
      as.v[e % ROWS][t] = make_float2(x, x);
    }
    __syncthreads();
#pragma unroll 2
    for (int i = 0; i < RW; ++i) {
      const int64_t r = r0 + w * RW + i;
      if (r >= end) break;
      float2 o[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      const float2* a = as.v[w * RW + i];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        o[0] = __ffma2_rn(v[t][0], a[t], o[0]);
        o[1] = __ffma2_rn(v[t][1], a[t], o[1]);
      }
      float* dst = O + r * ldo;
      if (VEC == 4 && c + 4 <= C) {
        float4* d = reinterpret_cast<float4*>(dst + c);
        float4 s = make_float4(o[0].x, o[0].y, o[1].x, o[1].y);
        if (accumulate) {
          const float4 old = *d;
          s.x += old.x; s.y += old.y; s.z += old.z; s.w += old.w;
        }
        *d = s;
      } else {
        const float f[4] = {o[0].x, o[0].y, o[1].x, o[1].y};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t at = VEC == 4 ? c + j : c + 32 * j;
          if (at < C) dst[at] = accumulate ? dst[at] + f[j] : f[j];
        }
      }
    }
  }
}

// logit v of row t: the splits' sums and the bias
__device__ __forceinline__ float few_logit(const float* z, int splits, int T, int64_t ld, int t, int64_t v,
                                           const float* bias) {
  float s = bias ? __ldg(bias + v) : 0.f;
  for (int i = 0; i < splits; ++i) s += z[((int64_t)i * T + t) * ld + v];
  return s;
}

// (maximum, sum of exponentials) of a row's classes, a partial per block, and
// the target's logit
__global__ void __launch_bounds__(256) few_stats_kernel(const float* __restrict__ z, int splits, int64_t ld,
                                                        const float* __restrict__ bias, Targets target,
                                                        float2* part, int64_t part_ld, float* zt) {
  __shared__ float2 sh[8];
  wait_for_previous_kernel();
  const int t = blockIdx.x, T = (int)target.rows;
  const int64_t n = target.classes, begin = n * blockIdx.y / gridDim.y, end = n * (blockIdx.y + 1) / gridDim.y;
  float m = -INFINITY, s = 0.f;
  for (int64_t v = begin + threadIdx.x; v < end; v += 4 * 256) {  // four at a time
    float q[4], M = m;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      q[j] = v + 256 * j < end ? few_logit(z, splits, T, ld, t, v + 256 * j, bias) : -INFINITY;
      M = fmaxf(M, q[j]);
    }
    const float base = M == -INFINITY ? 0.f : M;
    s *= exp_fast(m - base);
#pragma unroll
    for (int j = 0; j < 4; ++j) s += exp_fast(q[j] - base);
    m = M;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    join(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) join(m, s, sh[i].x, sh[i].y);
    part[(int64_t)blockIdx.y * part_ld + t] = make_float2(m, s);
    const int64_t c = target.at(t);
    if (blockIdx.y == 0 && c >= 0) zt[t] = few_logit(z, splits, T, ld, t, c, bias);
  }
}

// g = softmax - onehot of every row (0 without a target), the gradients' scale,
// and dbias; a thread a class.
__global__ void __launch_bounds__(256) few_grad_kernel(const float* __restrict__ z, int splits, int64_t ld,
                                                       const float* __restrict__ bias, Targets target,
                                                       const float* __restrict__ lse, float divisor,
                                                       const float* upstream, float* scale_out,
                                                       float* __restrict__ g, int64_t ldg, float* dbias,
                                                       int accumulate) {
  __shared__ int64_t cls[kFewRows];
  __shared__ float off[kFewRows];
  wait_for_previous_kernel();
  const int T = (int)target.rows;
  const bool counts = (int)threadIdx.x < T && target.at(threadIdx.x) >= 0;
  if ((int)threadIdx.x < T) {
    cls[threadIdx.x] = target.at(threadIdx.x);
    const float l = lse[threadIdx.x];
    off[threadIdx.x] = l == -INFINITY ? INFINITY : l;  // nothing left of the row: p = 0
  }
  const int n = __syncthreads_count(counts);
  const float scale = (upstream ? *upstream : 1.f) / (divisor > 0.f ? divisor : fmaxf(1.f, (float)n));
  if (blockIdx.x == 0 && threadIdx.x == 0) *scale_out = scale;
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (v >= target.classes) return;
  float sum = 0.f;
#pragma unroll 4
  for (int t = 0; t < T; ++t) {
    float q = 0.f;
    if (cls[t] >= 0) {
      q = exp_fast(few_logit(z, splits, T, ld, t, v, bias) - off[t]);
      if (v == cls[t]) q -= 1.f;
    }
    g[t * ldg + v] = q;
    sum += q;
  }
  if (dbias) dbias[v] = (accumulate ? dbias[v] : 0.f) + scale * sum;
}

// calls f(rows as a constant, vector accesses as a constant)
template <typename F>
int few_rows(int64_t T, bool vec, F f) {
  auto with = [&](auto tt) {
    return vec ? f(tt, std::integral_constant<int, 4>{}) : f(tt, std::integral_constant<int, 1>{});
  };
  if (T == 1) return with(std::integral_constant<int, 1>{});
  if (T <= 4) return with(std::integral_constant<int, 4>{});
  if (T <= 8) return with(std::integral_constant<int, 8>{});
  return with(std::integral_constant<int, 16>{});
}

// splits of the long axis: about `waves` blocks an SM
int few_splits(int64_t blocks, int64_t most, int waves) {
  const int64_t want = (int64_t)waves * std::max(1, sm_count());
  return (int)std::max<int64_t>(1, std::min<int64_t>({(want + blocks - 1) / blocks, most, 64}));
}
int64_t rowdot_blocks(int64_t R) { return (R + kFewWarps * kFewPerWarp - 1) / (kFewWarps * kFewPerWarp); }
int rowdot_splits(int64_t R, int64_t C) { return few_splits(rowdot_blocks(R), C / 512, 4); }
int coldot_splits(int64_t R, int64_t C) { return few_splits((C + 127) / 128, R / 256, 6); }

// out [split][T][ldo] = a W^T (by_rows: W's rows give the outputs) or a W
int few_product(bool by_rows, const float* W, int64_t ldw, int64_t R, int64_t C, const float* a, int64_t lda,
                int64_t T, float* out, int64_t ldo, cudaStream_t st) {
  const bool vec = ldw % 4 == 0 && aligned_to(W, 16);
  return few_rows(T, vec, [&](auto tt, auto v) {
    constexpr int TT = decltype(tt)::value, VEC = decltype(v)::value;
    if (by_rows)
      return launch(few_rowdot_kernel<TT, VEC>,
                    dim3((unsigned)rowdot_blocks(R), (unsigned)rowdot_splits(R, C)), kFewThreads, 0, st, W, ldw, R,
                    C, a, lda, (int)T, out, ldo);
    return launch(few_coldot_kernel<TT, VEC>, dim3((unsigned)((C + 127) / 128), (unsigned)coldot_splits(R, C)),
                  kFewThreads, 0, st, W, ldw, R, C, a, lda, (int)T, out, ldo);
  });
}

}  // namespace
}  // namespace tl
