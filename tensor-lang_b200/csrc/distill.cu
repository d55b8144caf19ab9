// Distillation from a teacher's top logits, forward and gradient.
//
// Per row, with the list (i_k, t_k) and tau the temperature:
//   q = softmax(t / tau) over the list,  p = softmax(z / tau) over all classes
//   row_loss = tau^2 sum_k q_k (log q_k - log p[i_k])
//            = tau^2 (sum_k q_k log q_k + lse - sum_k q_k z[i_k] / tau)
//   dz = tau (p - q) upstream / divisor
// (the second form of the loss uses sum q = 1: it needs no log p, so the
// list's part is summed before lse is known).
//
// z is read once and dz written once: the memory's floor.  A row of a
// large vocabulary does not fit one SM's registers beside other rows, so a
// cluster of up to eight CTAs holds it in shared memory: each CTA brings its
// segment in with asynchronous copies, takes the segment's maximum and sum of
// exponentials from shared memory, exchanges four numbers (maximum, sum,
// the list's sums of q and q z) with the other CTAs through distributed shared memory,
// and writes its segment's gradient from the same copy.  Segments are 32 to
// 64 KB, so several CTAs share an SM and one's copy overlaps another's
// exponentials and stores.
//
// Listed classes: the gradient there is p - q with the q of equal indices
// added, rounded once.  Their cells in shared memory are replaced by the
// number of the list entry that came first, and a mark says so; the store
// pass looks the entry up.  (No atomics on values: sums are in list
// order.)
//
// 8192 x 131072 bf16 with lists of 64: 984 us, 4.4 TB/s of the 6.5 a copy
// reaches; 1537 x 50021 float32 141 us, 4.4 TB/s.  What bounds it now is
// instruction issue (70% of the slots): 13 instructions an element (two passes
// over shared memory, the exponential in each) and about 500 a warp for the
// list, the reductions and the exchange.
#include <math.h>

#include <algorithm>

#include "lm_common.cuh"

namespace tl {
namespace {

constexpr int kMaxTop = 1024;
constexpr int64_t kSegTarget = 16384;       // classes of a row a CTA aims at
constexpr int64_t kSegMax = 192 << 10;      // and the most it takes
constexpr int kMaxCluster = 8;
constexpr int kSmemMost = 226 << 10;        // dynamic, beside a few hundred bytes

struct DistillArgs {
  int64_t rows, classes;
  int top;
  const void* z;
  int64_t ldz;
  const void* teacher;
  int64_t ldt;
  const void* index;
  int64_t ldi;
  int index_type;
  float temperature, divisor;
  float k2, inv_tau;    // exp(v / temperature) = 2^(v k2); 1 / temperature
  const float* upstream;
  float* loss;
  float* row_loss;      // the caller's, or scratch when only the mean is wanted
  float* lse;
  void* dz;
  int64_t lddz;
  int accumulate;
  unsigned* counters;   // [0] rows that count, [1] rows done; 0 between calls
  int64_t seg;          // classes per CTA
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t saddr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a float into the same shared variable of CTA `rank`
__device__ __forceinline__ void st_peer(float* p, uint32_t rank, float v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr(p)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}

// 2^x within 2 ulp (results below the smallest normal float are 0)
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Entry k of row r: its class in [0, classes) with a teacher logit above -inf
// (t), or -1.
template <typename T>
__device__ __forceinline__ int entry(const DistillArgs& a, int64_t r, int k, float& t) {
  t = to_f32(static_cast<const T*>(a.teacher)[r * a.ldt + k]);
  const int64_t c = class_index(a.index, a.index_type, r * a.ldi + k, a.classes);
  return t == -INFINITY ? -1 : (int)c;
}

// the larger of m and 16 bytes of elements
__device__ __forceinline__ float max_vec(const float* p, float m) {
  const float4 q = *reinterpret_cast<const float4*>(p);
  return fmaxf(fmaxf(fmaxf(m, q.x), fmaxf(q.y, q.z)), q.w);
}
__device__ __forceinline__ float max_vec(const __nv_bfloat16* p, float m) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  auto b2 = [](const uint32_t& w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
  const __nv_bfloat162 a = __hmax2(__hmax2(b2(q.x), b2(q.y)), __hmax2(b2(q.z), b2(q.w)));
  return fmaxf(fmaxf(m, __low2float(a)), __high2float(a));
}
// sum and maximum of the first N lanes' values, in every lane
template <int N>
__device__ __forceinline__ float few_sum(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return __shfl_sync(0xffffffffu, v, 0);
}
template <int N>
__device__ __forceinline__ float few_max(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return __shfl_sync(0xffffffffu, v, 0);
}

// Words of the marks of a segment: a byte per vector, one before the middle and
// one behind it besides.
__host__ __device__ constexpr int mark_words(int seg, int vec) { return (seg / vec + 2 + 3) / 4; }

// Whether row r has a valid entry (asked by a whole warp).
template <typename T>
__device__ __forceinline__ bool row_counts(const DistillArgs& a, int64_t r) {
  const int lane = threadIdx.x & 31;
  bool any = false;
  for (int k0 = 0; k0 < a.top && !any; k0 += 32) {
    float t;
    any = __any_sync(0xffffffffu, k0 + lane < a.top && entry<T>(a, r, k0 + lane, t) >= 0);
  }
  return any;
}

// Rows with a valid entry, one warp per row.
template <typename T>
__global__ void __launch_bounds__(256) distill_count_kernel(DistillArgs a) {
  wait_for_previous_kernel();
  const int lane = threadIdx.x & 31;
  unsigned n = 0;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < a.rows; r += 8LL * gridDim.x)
    n += row_counts<T>(a, r);
  if (lane == 0 && n) atomicAdd(&a.counters[0], n);  // a whole number: any order
}

// ALONE: few rows; every CTA counts them itself and the last row's adds up.
template <typename T, int NT, bool ALONE>
__global__ void __launch_bounds__(NT) distill_kernel(DistillArgs a) {
  constexpr int V = 16 / sizeof(T), NW = NT / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  // [list: class, q, first entry's q sum, its z] [marks of the listed cells] [segment]
  // (offsets from the array, not pointer casts: the compiler keeps to shared
  // memory instructions)
  int* li = reinterpret_cast<int*>(smem);
  float* lq = reinterpret_cast<float*>(smem + 4 * a.top);
  float* lsum = reinterpret_cast<float*>(smem + 8 * a.top);
  float* lz = reinterpret_cast<float*>(smem + 12 * a.top);
  // per vector of V cells a byte with the listed ones' bits; the vectors are
  // those of the middle (below), the cells before it are vector 0
  unsigned char* mark_of = smem + 16 * a.top;
  uint32_t* marks = reinterpret_cast<uint32_t*>(mark_of);
  const int nmarks = mark_words((int)a.seg, V);
  T* cells = reinterpret_cast<T*>(smem + ((16 * a.top + 4 * nmarks + 15) & ~15));
  __shared__ float peer[4][kMaxCluster];
  __shared__ float sh[2][NW], lsh[5][NW], list[3];
  __shared__ int few[NW];

  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int64_t r = blockIdx.x / size;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int64_t c0 = (int64_t)rank * a.seg;
  const int n = (int)max((int64_t)0, min(a.seg, a.classes - c0));
  const T* src = static_cast<const T*>(a.z) + r * a.ldz + c0;
  // the segment sits in shared memory at the offset within 16 bytes that it
  // has in memory, so that its middle is copied 16 bytes at a time
  const int phase = (int)(((uintptr_t)src & 15) / sizeof(T));
  T* cell = cells + phase;
  const int head = min(n, phase ? V - phase : 0), mid = (n - head) / V * V;
  if (size > 1) cluster_arrive_relaxed();  // every CTA of the cluster runs: waited for before the exchange
  wait_for_previous_kernel();

  // each thread brings in what it reads in the first pass, so waiting for its
  // own copies is enough; the row's ends, outside the 16-byte copies, are one
  // element for each of the first threads (fewer than 2 V)
  for (int i = head + tid * V; i < head + mid; i += NT * V)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(saddr(cell + i)), "l"(src + i)
                 : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");
  const int end = tid < n - mid ? (tid < head ? tid : mid + tid) : -1;
  float end_z = -INFINITY;
  if (end >= 0) {
    cell[end] = src[end];
    end_z = to_f32(cell[end]);
  }
  for (int i = tid; i < nmarks; i += NT) marks[i] = 0u;
  const float up = a.upstream ? *a.upstream : 1.f;
  const float k2 = a.k2, inv_tau = a.inv_tau;
  float div = a.divisor;
  if (ALONE && a.divisor == 0.f) {
    int counted = 0;
    for (int64_t i = w; i < a.rows; i += NW) counted += row_counts<T>(a, i);
    if (lane == 0) few[w] = counted;
    __syncthreads();
    counted = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) counted += few[i];
    div = fmaxf(1.f, (float)counted);
  } else {
    if (a.divisor == 0.f) div = fmaxf(1.f, (float)a.counters[0]);
    __syncthreads();
  }

  // while they are on their way (and while the other warps work on the
  // segment), the first warps prepare the teacher's list: q = softmax(t / tau)
  const int list_warps = min(NW, (a.top + 31) / 32), LT = 32 * list_warps;
  if (w < list_warps) {
    auto list_sync = [&] { asm volatile("bar.sync 1, %0;" ::"r"(LT) : "memory"); };
    float tm = -INFINITY, tnan = 0.f;
    for (int k = tid; k < a.top; k += LT) {
      float t;
      li[k] = entry<T>(a, r, k, t);
      lq[k] = t;
      if (li[k] >= 0) {
        tm = fmaxf(tm, t);
        if (t != t) tnan = 1.f;
      }
    }
    tm = warp_max(tm);
    tnan = warp_max(tnan);
    if (lane == 0) {
      lsh[0][w] = tm;
      lsh[1][w] = tnan;
    }
    list_sync();
    tm = few_max<NW>(lane < list_warps ? lsh[0][lane] : -INFINITY);
    tnan = few_max<NW>(lane < list_warps ? lsh[1][lane] : 0.f);
    float tsum = 0.f, tdot = 0.f;
    for (int k = tid; k < a.top; k += LT) {
      float e = 0.f;
      if (li[k] >= 0) {
        const float d = (lq[k] - tm) * inv_tau;
        e = expf(d);
        tsum += e;
        tdot += e > 0.f ? e * d : 0.f;
      }
      lq[k] = e;  // q times the sum
    }
    tsum = warp_sum(tsum);
    tdot = warp_sum(tdot);
    if (lane == 0) {
      lsh[2][w] = tsum;
      lsh[3][w] = tdot;
    }
    // listed cells are marked; where a class is met again (its bit is there
    // already), the q of equal classes are added, in list order, for the first
    // of them (the others: -1)
    bool again = false;
    for (int k = tid; k < a.top; k += LT) {
      const int c = li[k];
      if (c < c0 || c >= c0 + n) continue;
      const int at = c - (int)c0 - head + V;  // byte at / V, bit at % V
      const uint32_t bit = 1u << (8 * (at / V & 3) + at % V);
      again |= (atomicOr(&marks[at / V >> 2], bit) & bit) != 0;
    }
    again = __any_sync(0xffffffffu, again);
    if (lane == 0) lsh[4][w] = again ? 1.f : 0.f;
    list_sync();
    tsum = few_sum<NW>(lane < list_warps ? lsh[2][lane] : 0.f);
    tdot = few_sum<NW>(lane < list_warps ? lsh[3][lane] : 0.f);
    again = few_max<NW>(lane < list_warps ? lsh[4][lane] : 0.f) > 0.f;
    const bool some = tm > -INFINITY || tnan > 0.f;
    const float inv_t = some ? 1.f / tsum : 0.f;
    for (int k = tid; k < a.top; k += LT) {
      const int c = li[k];
      if (c < c0 || c >= c0 + n) continue;
      float sum = lq[k];
      bool first = true;
      if (again) {
        sum = 0.f;
        for (int j = 0; j < a.top; ++j)
          if (li[j] == c) {
            first = first && j >= k;
            sum += lq[j];
          }
      }
      lsum[k] = first ? sum * inv_t : -1.f;
    }
    if (tid == 0) {
      list[0] = some ? 1.f : 0.f;
      list[1] = inv_t;
      list[2] = some ? tdot * inv_t - logf(tsum) : 0.f;  // sum q log q = sum e d / S - log S
    }
  }

  // the segment: each thread's maximum and sum of exponentials, then the warp's
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  float m = end_z, s;
#pragma unroll 4
  for (int i = head + tid * V; i < head + mid; i += NT * V) m = max_vec(cell + i, m);
  {
    const float base = m == -INFINITY ? 0.f : m;
    const float2 nb = make_float2(-base, -base), kk = make_float2(k2, k2);
    float2 t = make_float2(end >= 0 ? exp2_fast((end_z - base) * k2) : 0.f, 0.f);
#pragma unroll 2
    for (int i = head + tid * V; i < head + mid; i += NT * V) {
      float v[V];
      ld_vec<V>(cell + i, v);
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const float2 x = __fmul2_rn(__fadd2_rn(make_float2(v[j], v[j + 1]), nb), kk);
        t = __fadd2_rn(t, make_float2(exp2_fast(x.x), exp2_fast(x.y)));
      }
    }
    s = t.x + t.y;
    const float wm = warp_max(m), wbase = wm == -INFINITY ? 0.f : wm;
    s = warp_sum(s * exp2_fast((m - wbase) * k2));
    m = wm;
  }
  if (lane == 0) {
    sh[0][w] = m;
    sh[1][w] = s;
  }
  __syncthreads();
  const bool some = list[0] > 0.f;
  if (w == 0) {
    const float inv_t = list[1];
    m = lane < NW ? sh[0][lane] : -INFINITY;
    s = lane < NW ? sh[1][lane] : 0.f;
    const float sm = few_max<NW>(m), base = sm == -INFINITY ? 0.f : sm;
    s = few_sum<NW>(s * exp2_fast((m - base) * k2));
    // the list's entries in this segment: the sums of q and of q (z - m) / tau
    // (differences to the maximum: logits of the type's lowest value cancel
    // exactly); their cells make way for the entry's number
    float dot = 0.f, qs = 0.f;
    for (int k = lane; k < a.top; k += 32) {
      const int c = li[k];
      if (c < c0 || c >= c0 + n) continue;
      const float q = lq[k] * inv_t, z = to_f32(cell[c - c0]);
      lz[k] = z;
      if (q > 0.f || q != q) {
        dot += q * ((z - base) * inv_tau);
        qs += q;
      }
    }
    dot = warp_sum(dot);  // every lane has read its cells
    qs = warp_sum(qs);
    for (int k = lane; k < a.top; k += 32) {
      const int c = li[k] - (int)c0;
      if (li[k] < 0 || c < 0 || c >= n || lsum[k] < 0.f) continue;
      if constexpr (sizeof(T) == 2)
        reinterpret_cast<uint16_t*>(cell)[c] = (uint16_t)k;
      else
        reinterpret_cast<uint32_t*>(cell)[c] = (uint32_t)k;
    }
    if (size > 1) cluster_wait();
    if (lane < (int)size) {
      st_peer(&peer[0][rank], lane, sm);
      st_peer(&peer[1][rank], lane, s);
      st_peer(&peer[2][rank], lane, dot);
      st_peer(&peer[3][rank], lane, qs);
    }
    __syncwarp();
    if (size > 1) cluster_arrive();
  } else if (size > 1) {
    // nothing of these warps is for other CTAs, and their own has them since
    // the last barrier
    cluster_wait();
    cluster_arrive_relaxed();
  }
  if (size > 1) {
    cluster_wait();
  } else {
    __syncthreads();
  }
  const bool there = lane < (int)size;
  const float pm = there ? peer[0][lane] : -INFINITY, ps = there ? peer[1][lane] : 0.f;
  m = few_max<kMaxCluster>(pm);
  const float base = m == -INFINITY ? 0.f : m, pb = pm == -INFINITY ? 0.f : pm;
  s = few_sum<kMaxCluster>(ps == 0.f ? 0.f : ps * exp2_fast((pb - base) * k2));
  float dot = 0.f;
  if (rank == 0 && w == 0) {
    const float pq = there ? peer[3][lane] : 0.f;
    dot = few_sum<kMaxCluster>(pq == 0.f ? 0.f : peer[2][lane] + pq * ((pb - base) * inv_tau));
  }
  if (rank == 0 && tid == 0) {
    const float log_s = logf(s);  // a row of -inf: -inf
    if (a.lse) a.lse[r] = m * inv_tau + log_s;
    float l = 0.f;
    if (some) l = dot == -INFINITY ? INFINITY : a.temperature * a.temperature * (list[2] + (log_s - dot));
    if (a.row_loss) a.row_loss[r] = l;
    if (ALONE && a.loss) {  // the last row to get here adds them up, in order
      __threadfence();
      if (atomicAdd(&a.counters[1], 1u) == (unsigned)(a.rows - 1)) {
        __threadfence();
        double t = 0.0;
        for (int64_t i = 0; i < a.rows; ++i) t += (double)__ldcg(a.row_loss + i);
        a.loss[0] = (float)(t / (double)div);
        a.counters[1] = 0u;
      }
    }
  }
  if (!a.dz) return;
  const float cf = some ? __fdividef(a.temperature * up, div) : 0.f;
  // p = exp((z - m) / tau) / s: nearer than exp(z / tau - lse), whose lse is rounded
  const float inv_s = s > 0.f || s != s ? __fdividef(1.f, s) : 0.f;
  auto grad = [&](int c) {  // of cell c
    const int at = c - head + V;
    float z = to_f32(cell[c]), q = 0.f;
    if (marks[at / V >> 2] >> (8 * (at / V & 3) + at % V) & 1u) {
      const int k = sizeof(T) == 2 ? (int)reinterpret_cast<const uint16_t*>(cell)[c]
                                   : (int)reinterpret_cast<const uint32_t*>(cell)[c];
      z = lz[k];
      q = lsum[k];
    }
    return cf * (exp2_fast((z - base) * k2) * inv_s - q);
  };
  T* dst = static_cast<T*>(a.dz) + r * a.lddz + c0;
  const bool add_to = a.accumulate != 0;
  if (!some) {
    if (!add_to)
      for (int i = tid; i < n; i += NT) from_f32(dst + i, 0.f);
    return;
  }
  if (((uintptr_t)(dst + head) & 15) != 0) {
    for (int c = tid; c < n; c += NT) from_f32(dst + c, (add_to ? to_f32(dst[c]) : 0.f) + grad(c));
    return;
  }
  const float2 nb = make_float2(-base, -base), kk = make_float2(k2, k2);
  const float2 cs = make_float2(cf * inv_s, cf * inv_s);
  for (int i = head + tid * V; i < head + mid; i += NT * V) {
    float v[V], o[V];
    ld_vec<V>(cell + i, v);
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 x = __fmul2_rn(__fadd2_rn(make_float2(v[j], v[j + 1]), nb), kk);
      const float2 y = __fmul2_rn(make_float2(exp2_fast(x.x), exp2_fast(x.y)), cs);
      o[j] = y.x;
      o[j + 1] = y.y;
    }
    if (const unsigned listed = mark_of[(i - head) / V + 1]) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (listed >> j & 1u) o[j] = grad(i + j);
    }
    if (add_to) {
      ld_vec<V>(dst + i, v);
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] += v[j];
    }
    st_vec<V>(dst + i, o);
  }
  if (end >= 0) from_f32(dst + end, (add_to ? to_f32(dst[end]) : 0.f) + grad(end));
}

// The mean, in double, and the counter cleared for the next call.
__global__ void __launch_bounds__(1024) distill_mean_kernel(DistillArgs a) {
  __shared__ double sh[32];
  wait_for_previous_kernel();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  double t = 0.0;
  if (a.loss)
    for (int64_t i = threadIdx.x; i < a.rows; i += 1024) t += (double)a.row_loss[i];
  t = warp_sum(t);
  if (lane == 0) sh[w] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    t = 0.0;
    for (int i = 0; i < 32; ++i) t += sh[i];
    const float div = a.divisor > 0.f ? a.divisor : fmaxf(1.f, (float)a.counters[0]);
    if (a.loss) a.loss[0] = (float)(t / (double)div);
    a.counters[0] = 0u;
  }
}

// ------------------------------------------------------------- host side ---
// About 16384 classes a CTA: 32 KB of bf16 (six CTAs an SM) or 64 KB of float32.
// With 8192, 16384 and 32768 classes, us (131072 and 100000 have eight segments at
// most in the first two): 8192 x 131072 bf16 947, 947, 1020; 4096 x 65536 bf16 341,
// 238, 249; 4096 x 100000 bf16 436, 436, 421; 4096 x 32000 float32 228, 212, 328;
// 1537 x 50021 float32 142, 146, 164.
// Few rows are spread wider: 8 x 32000 float32 takes 7.5 us in 4096 classes a
// CTA, 8.9 us in 16384.
int cluster_for(int64_t rows, int64_t classes) {
  const int64_t target = rows * kMaxCluster <= 2 * sm_count() ? kSegTarget / 4 : kSegTarget;
  int c = 1;
  while (c < kMaxCluster && classes > c * target) c *= 2;
  return c;
}

template <typename T, int NT, bool ALONE>
int launch_rows(const DistillArgs& a, int cluster, cudaStream_t st) {
  const size_t smem = (size_t)a.top * 16 + (size_t)mark_words((int)a.seg, 16 / sizeof(T)) * 4 + 16 +
                      (size_t)a.seg * sizeof(T) + 16;
  constexpr auto kern = distill_kernel<T, NT, ALONE>;
  TL_TRY((allow_smem<kern, kSmemMost>()));
  return launch_in_clusters(cluster, kern, dim3((unsigned)(a.rows * cluster)), NT, smem, st, a);
}

template <typename T>
int run(DistillArgs a, cudaStream_t st) {
  // one launch instead of three: 8 x 32000 float32 takes 10.9 us a call instead of 17.4
  const bool alone = a.rows <= 16 && a.rows * a.top <= 4096;
  if (a.divisor == 0.f && !alone) {
    const int64_t blocks = std::min<int64_t>((a.rows + 7) / 8, 4LL * sm_count());
    TL_TRY(launch(distill_count_kernel<T>, dim3((unsigned)blocks), 256, 0, st, a));
  }
  constexpr int64_t V = 16 / sizeof(T);
  const int cluster = cluster_for(a.rows, a.classes);
  // segments start at multiples of 32 classes: 16-byte aligned in an aligned row
  a.seg = ((a.classes + cluster - 1) / cluster + 31) / 32 * 32;
  static_assert(32 % V == 0, "aligned segments");
  if (alone)
    return a.seg <= 2048 ? launch_rows<T, 128, true>(a, cluster, st) : launch_rows<T, 256, true>(a, cluster, st);
  if (a.seg <= 2048)
    TL_TRY((launch_rows<T, 128, false>(a, cluster, st)));
  else
    TL_TRY((launch_rows<T, 256, false>(a, cluster, st)));
  if (a.loss || a.divisor == 0.f) {
    TL_TRY(launch(distill_mean_kernel, dim3(1), 1024, 0, st, a));
  }
  return TL_OK;
}

int check(int dtype, const DistillArgs& a, int64_t top) {
  if (!dtype_ok(dtype) || !index_ok(a.index_type)) return TL_ERR_INVALID_ARG;
  if (a.rows < 0 || a.classes <= 0 || top <= 0) return TL_ERR_INVALID_ARG;
  if (a.classes > INT32_MAX || a.rows > INT32_MAX / kMaxCluster) return TL_ERR_UNSUPPORTED;
  if (top > kMaxTop) return TL_ERR_UNSUPPORTED;
  if (a.classes * (int64_t)elem_bytes(dtype) > kMaxCluster * kSegMax) return TL_ERR_UNSUPPORTED;
  if (a.rows > 0 && (!a.z || !a.teacher || !a.index)) return TL_ERR_INVALID_ARG;
  if (a.ldz < a.classes || a.ldt < top || a.ldi < top) return TL_ERR_INVALID_ARG;
  if (a.dz && a.lddz < a.classes) return TL_ERR_INVALID_ARG;
  // dz over z: only row on row
  if (a.dz == a.z && a.dz && (a.lddz != a.ldz || a.accumulate)) return TL_ERR_INVALID_ARG;
  // its square is a factor, its inverse another
  if (!(a.temperature >= 1e-18f && a.temperature <= 1e18f) || !(a.divisor >= 0.f)) return TL_ERR_INVALID_ARG;
  return TL_OK;
}

}  // namespace
}  // namespace tl

extern "C" {

size_t tl_distill_topk_scratch_bytes(int64_t rows) {
  return 256 + (size_t)std::max<int64_t>(rows, 0) * sizeof(float);
}

int tl_distill_topk(int dtype, int64_t rows, int64_t classes, int64_t top, const void* z,
                    int64_t ldz, const void* teacher, int64_t ldt, const void* index, int64_t ldi,
                    int index_type, float temperature, float divisor, const float* upstream,
                    float* loss, float* row_loss, float* lse, void* dz, int64_t lddz,
                    int accumulate, void* scratch, size_t scratch_bytes, void* stream) {
  tl::DistillArgs a{};
  a.rows = rows; a.classes = classes; a.top = (int)(top > 0 && top <= tl::kMaxTop ? top : 0);
  a.z = z; a.ldz = ldz; a.teacher = teacher; a.ldt = ldt; a.index = index; a.ldi = ldi;
  a.index_type = index_type; a.temperature = temperature; a.divisor = divisor;
  a.upstream = upstream; a.loss = loss; a.lse = lse; a.dz = dz; a.lddz = lddz;
  a.accumulate = accumulate;
  TL_TRY(tl::check(dtype, a, top));
  a.k2 = (float)(1.4426950408889634 / (double)temperature);
  a.inv_tau = (float)(1.0 / (double)temperature);
  if (rows > 0 && !loss && !row_loss && !lse && !dz) return TL_ERR_INVALID_ARG;
  if (!scratch || !tl::aligned_to(scratch, 16) || scratch_bytes < tl_distill_topk_scratch_bytes(rows))
    return TL_ERR_INVALID_ARG;
  a.counters = static_cast<unsigned*>(scratch);
  a.row_loss = row_loss ? row_loss : reinterpret_cast<float*>(static_cast<char*>(scratch) + 256);
  cudaStream_t st = tl::stream_or_default(stream);
  if (rows == 0) {
    if (loss) TL_CUDA_TRY(cudaMemsetAsync(loss, 0, sizeof(float), st));
    return TL_OK;
  }
  return dtype == TL_BF16 ? tl::run<__nv_bfloat16>(a, st) : tl::run<float>(a, st);
}

}  // extern "C"
