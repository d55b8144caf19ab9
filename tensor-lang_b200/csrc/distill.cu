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
// Bound by the memory system: z is read once and dz written once.  A row of a
// large vocabulary does not fit one SM's registers beside other rows, so a
// cluster of up to eight CTAs holds it in shared memory: each CTA brings its
// segment in with asynchronous copies, takes the segment's maximum and sum of
// exponentials from shared memory, exchanges four numbers (maximum, sum,
// the list's sums of q and q z) with the other CTAs through distributed shared memory,
// and writes its segment's gradient from the same copy.  Segments are about
// 32 KB, so several CTAs share an SM and one's copy overlaps another's
// exponentials and stores.
//
// Listed classes: the gradient there is p - q with the q of equal indices
// added, rounded once.  Their cells in shared memory are replaced by the
// number of the list entry that came first, and a bit per cell says so; the
// store pass looks the entry up.  (No atomics on values: sums are in list
// order.)
#include <math.h>

#include <algorithm>

#include "lm_common.cuh"

namespace tl {
namespace {

constexpr int kMaxTop = 1024;
constexpr int64_t kSegTarget = 32 << 10;    // bytes of a row a CTA aims at
constexpr int64_t kSegMax = 192 << 10;      // and the most it takes
constexpr int kMaxCluster = 8;

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
  const float* upstream;
  float* loss;
  float* row_loss;      // the caller's, or scratch when only the mean is wanted
  float* lse;
  void* dz;
  int64_t lddz;
  int accumulate;
  unsigned* counters;   // [0] rows that count, [1] rows done
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
// (m, s) <- the maximum and the sum of exp(k (v - m)) of both parts
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2, float k) {
  const float M = fmaxf(m, m2);
  const float base = M == -INFINITY ? 0.f : M;  // both empty: 0 + 0
  s = s * exp2_fast((m - base) * k) + s2 * exp2_fast((m2 - base) * k);
  m = M;
}

// Entry k of row r: its class in [0, classes) with a teacher logit above -inf
// (t), or -1.
template <typename T>
__device__ __forceinline__ int entry(const DistillArgs& a, int64_t r, int k, float& t) {
  t = to_f32(static_cast<const T*>(a.teacher)[r * a.ldt + k]);
  const int64_t c = class_index(a.index, a.index_type, r * a.ldi + k, a.classes);
  return t == -INFINITY ? -1 : (int)c;
}

// Rows with a valid entry, one warp per row.
template <typename T>
__global__ void __launch_bounds__(256) distill_count_kernel(DistillArgs a) {
  const int lane = threadIdx.x & 31;
  unsigned n = 0;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < a.rows; r += 8LL * gridDim.x) {
    bool any = false;
    for (int k0 = 0; k0 < a.top && !any; k0 += 32) {
      float t;
      any = __any_sync(0xffffffffu, k0 + lane < a.top && entry<T>(a, r, k0 + lane, t) >= 0);
    }
    n += any;
  }
  if (lane == 0 && n) atomicAdd(&a.counters[0], n);  // a whole number: any order
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_kernel(DistillArgs a) {
  constexpr int V = 16 / sizeof(T), NW = NT / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  // [list: class, q, first entry's q sum, its z] [bits of the listed cells] [segment]
  int* li = reinterpret_cast<int*>(smem);
  float* lq = reinterpret_cast<float*>(li + a.top);
  float* lsum = lq + a.top;
  float* lz = lsum + a.top;
  uint32_t* bits = reinterpret_cast<uint32_t*>(lz + a.top);
  const int nbits = (int)((a.seg + 31) / 32);
  unsigned char* cells = reinterpret_cast<unsigned char*>(
      ((uintptr_t)(bits + nbits) + 15) & ~(uintptr_t)15);
  __shared__ float peer[4][kMaxCluster];
  __shared__ float sh[4][NW];
  __shared__ unsigned ticket;

  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int64_t r = blockIdx.x / size;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int64_t c0 = (int64_t)rank * a.seg;
  const int n = (int)max((int64_t)0, min(a.seg, a.classes - c0));
  const T* src = static_cast<const T*>(a.z) + r * a.ldz + c0;
  // the segment sits in shared memory at the offset within 16 bytes that it
  // has in memory, so that its middle is copied 16 bytes at a time
  const int phase = (int)(((uintptr_t)src & 15) / sizeof(T));
  T* cell = reinterpret_cast<T*>(cells) + phase;
  const int head = min(n, phase ? V - phase : 0), mid = (n - head) / V * V;
  if (size > 1) cluster_arrive();  // every CTA of the cluster runs: waited for before the exchange

  // each thread brings in the vectors it reads in the first pass, so waiting
  // for its own copies is enough
  for (int i = head + tid * V; i < head + mid; i += NT * V)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(saddr(cell + i)), "l"(src + i)
                 : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");
  // the row's ends, outside the 16-byte copies
  for (int i = tid; i < n - mid; i += NT) {
    const int c = i < head ? i : mid + i;
    cell[c] = src[c];
  }
  for (int i = tid; i < nbits; i += NT) bits[i] = 0u;

  // the teacher's list: q = softmax(t / tau)
  const float k2 = 1.4426950408889634f / a.temperature;  // exp(v / tau) = 2^(v k2)
  const float inv_tau = 1.f / a.temperature;
  float tm = -INFINITY;
  bool tnan = false;
  for (int k = tid; k < a.top; k += NT) {
    float t;
    li[k] = entry<T>(a, r, k, t);
    lq[k] = t;
    if (li[k] >= 0) {
      tm = fmaxf(tm, t);
      tnan |= t != t;
    }
  }
  tm = warp_max(tm);
  if (lane == 0) sh[0][w] = tm;
  const bool some = __syncthreads_or(tm > -INFINITY || tnan);
  tm = sh[0][0];
#pragma unroll
  for (int i = 1; i < NW; ++i) tm = fmaxf(tm, sh[0][i]);
  float tsum = 0.f, tdot = 0.f;
  for (int k = tid; k < a.top; k += NT) {
    if (li[k] < 0) continue;
    const float d = (lq[k] - tm) * inv_tau, e = expf(d);
    tsum += e;
    tdot += e > 0.f ? e * d : 0.f;
  }
  tsum = warp_sum(tsum);
  tdot = warp_sum(tdot);
  if (lane == 0) {
    sh[1][w] = tsum;
    sh[2][w] = tdot;
  }
  __syncthreads();
  tsum = tdot = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    tsum += sh[1][i];
    tdot += sh[2][i];
  }
  const float inv_t = some ? 1.f / tsum : 0.f;
  // sum q log q = sum e d / S - log S
  const float qlogq = some ? tdot * inv_t - logf(tsum) : 0.f;
  for (int k = tid; k < a.top; k += NT)
    lq[k] = li[k] >= 0 ? expf((lq[k] - tm) * inv_tau) * inv_t : 0.f;

  // the segment is here: its maximum and sum of exponentials
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float m = -INFINITY, s = 0.f;
  for (int i = head + tid * V; i < head + mid; i += NT * V) {
    float v[V];
    ld_vec<V>(cell + i, v);
    float mm = m;
#pragma unroll
    for (int j = 0; j < V; ++j) mm = fmaxf(mm, v[j]);
    const float base = mm == -INFINITY ? 0.f : mm;
    s *= exp2_fast((m - base) * k2);
#pragma unroll
    for (int j = 0; j < V; ++j) s += exp2_fast((v[j] - base) * k2);
    m = mm;
  }
  for (int i = tid; i < n - mid; i += NT) {
    const float v = to_f32(cell[i < head ? i : mid + i]);
    merge(m, s, v, v == -INFINITY ? 0.f : 1.f, k2);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    merge(m, s, m2, s2, k2);
  }
  __syncthreads();  // sh's earlier readers are done
  if (lane == 0) {
    sh[0][w] = m;
    sh[1][w] = s;
  }
  __syncthreads();
  m = sh[0][0];
  s = sh[1][0];
#pragma unroll
  for (int i = 1; i < NW; ++i) merge(m, s, sh[0][i], sh[1][i], k2);
  // the list's entries in this segment: the sums of q and of q (z - m) / tau
  // (differences to the maximum: logits of the type's lowest value cancel
  // exactly); equal classes are handled by the first of them
  float dot = 0.f, qs = 0.f;
  {
    const float base = m == -INFINITY ? 0.f : m;
    for (int k = tid; k < a.top; k += NT) {
      const int c = li[k];
      if (c < c0 || c >= c0 + n) continue;
      const float zc = to_f32(cell[c - c0]);
      if (lq[k] > 0.f || lq[k] != lq[k]) {
        dot += lq[k] * ((zc - base) * inv_tau);
        qs += lq[k];
      }
      float sum = 0.f;
      bool first = true;
      for (int j = 0; j < a.top; ++j)
        if (li[j] == c) {
          first = first && j >= k;
          sum += lq[j];
        }
      lz[k] = zc;
      lsum[k] = first ? sum : -1.f;
    }
  }
  dot = warp_sum(dot);
  qs = warp_sum(qs);
  if (lane == 0) {
    sh[2][w] = dot;
    sh[3][w] = qs;
  }
  __syncthreads();
  for (int k = tid; k < a.top; k += NT) {
    const int c = li[k] - (int)c0;
    if (li[k] < 0 || c < 0 || c >= n || lsum[k] < 0.f) continue;
    atomicOr(&bits[c >> 5], 1u << (c & 31));
    if constexpr (sizeof(T) == 2)
      reinterpret_cast<uint16_t*>(cell)[c] = (uint16_t)k;
    else
      reinterpret_cast<uint32_t*>(cell)[c] = (uint32_t)k;
  }
  dot = sh[2][0];
  qs = sh[3][0];
#pragma unroll
  for (int i = 1; i < NW; ++i) {
    dot += sh[2][i];
    qs += sh[3][i];
  }
  if (size > 1) {
    cluster_wait();
    if (tid < (int)size) {
      st_peer(&peer[0][rank], tid, m);
      st_peer(&peer[1][rank], tid, s);
      st_peer(&peer[2][rank], tid, dot);
      st_peer(&peer[3][rank], tid, qs);
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    m = peer[0][0];
    s = peer[1][0];
    for (uint32_t i = 1; i < size; ++i) merge(m, s, peer[0][i], peer[1][i], k2);
    const float base = m == -INFINITY ? 0.f : m;
    dot = 0.f;
    for (uint32_t i = 0; i < size; ++i) {
      const float mi = peer[0][i] == -INFINITY ? 0.f : peer[0][i];
      dot += peer[3][i] == 0.f ? 0.f : peer[2][i] + peer[3][i] * ((mi - base) * inv_tau);
    }
  } else {
    __syncthreads();  // the marked cells are seen by all
  }
  if (rank == 0 && tid == 0) {
    const float log_s = logf(s);  // a row of -inf: -inf
    if (a.lse) a.lse[r] = m * inv_tau + log_s;
    float l = 0.f;
    if (some)
      l = dot == -INFINITY ? INFINITY : a.temperature * a.temperature * (qlogq + (log_s - dot));
    a.row_loss[r] = l;
  }
  const unsigned counted = a.counters[0];
  const float div = a.divisor > 0.f ? a.divisor : fmaxf(1.f, (float)counted);
  if (a.dz) {
    const float up = a.upstream ? *a.upstream : 1.f;
    const float cf = some ? a.temperature * up / div : 0.f;
    // p = exp((z - m) / tau) / s: nearer than exp(z / tau - lse), whose lse is rounded
    const float inv_s = s > 0.f || s != s ? 1.f / s : 0.f;
    const float base = m == -INFINITY ? 0.f : m;
    auto grad = [&](int c) {  // of cell c
      float z = to_f32(cell[c]), q = 0.f;
      if (bits[c >> 5] >> (c & 31) & 1u) {
        const int k = sizeof(T) == 2 ? (int)reinterpret_cast<const uint16_t*>(cell)[c]
                                     : (int)reinterpret_cast<const uint32_t*>(cell)[c];
        z = lz[k];
        q = lsum[k];
      }
      return cf * (exp2_fast((z - base) * k2) * inv_s - q);
    };
    T* dst = static_cast<T*>(a.dz) + r * a.lddz + c0;
    const bool add_to = a.accumulate != 0;
    const bool vec = ((uintptr_t)(dst + head) & 15) == 0;
    if (!some && !add_to) {
      for (int i = tid; i < n; i += NT) from_f32(dst + i, 0.f);
    } else if (some) {
      if (vec) {
        for (int i = head + tid * V; i < head + mid; i += NT * V) {
          float v[V], o[V];
          ld_vec<V>(cell + i, v);
          uint32_t b = 0;
          // V cells' bits may lie in two words
          const int w0 = i >> 5, w1 = (i + V - 1) >> 5, sft = i & 31;
          b = bits[w0] >> sft;
          if (w1 != w0) b |= bits[w1] << (32 - sft);
          b &= (1u << V) - 1u;
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = cf * (exp2_fast((v[j] - base) * k2) * inv_s);
          if (b) {
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (b >> j & 1u) o[j] = grad(i + j);
          }
          if (add_to) {
            ld_vec<V>(dst + i, v);
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] += v[j];
          }
          st_vec<V>(dst + i, o);
        }
        for (int i = tid; i < n - mid; i += NT) {
          const int c = i < head ? i : mid + i;
          from_f32(dst + c, (add_to ? to_f32(dst[c]) : 0.f) + grad(c));
        }
      } else {
        for (int c = tid; c < n; c += NT)
          from_f32(dst + c, (add_to ? to_f32(dst[c]) : 0.f) + grad(c));
      }
    }
  }
  // the last row's cluster to finish writes the mean and clears the counters
  if (rank == 0 && tid == 0) {
    __threadfence();
    ticket = atomicAdd(&a.counters[1], 1u);
  }
  if (rank != 0) return;
  __syncthreads();
  if (ticket != (unsigned)(a.rows - 1)) return;
  if (a.loss) {
    __threadfence();
    double t = 0.0;
    for (int64_t i = tid; i < a.rows; i += NT) t += (double)__ldcg(a.row_loss + i);
    t = warp_sum(t);
    __shared__ double shd[NW];
    if (lane == 0) shd[w] = t;
    __syncthreads();
    if (tid == 0) {
      t = 0.0;
      for (int i = 0; i < NW; ++i) t += shd[i];
      a.loss[0] = (float)(t / (double)div);
    }
  }
  __syncthreads();
  if (tid == 0) a.counters[0] = a.counters[1] = 0u;
}

// ------------------------------------------------------------- host side ---
int cluster_for(int64_t row_bytes) {
  int c = 1;
  while (c < kMaxCluster && row_bytes > c * kSegTarget) c *= 2;
  return c;
}

template <typename T, int NT>
int launch(const DistillArgs& a, int cluster, cudaStream_t st) {
  const size_t smem = (size_t)a.top * 16 + (size_t)((a.seg + 31) / 32) * 4 + 16 +
                      (size_t)a.seg * sizeof(T) + 16;
  auto kern = distill_kernel<T, NT>;
  TL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * cluster));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  TL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a));
  return after_launch();
}

template <typename T>
int run(DistillArgs a, cudaStream_t st) {
  if (a.divisor == 0.f) {
    const int64_t blocks = std::min<int64_t>((a.rows + 7) / 8, 4LL * sm_count());
    distill_count_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(a);
    TL_TRY(after_launch());
  }
  constexpr int64_t V = 16 / sizeof(T);
  const int cluster = cluster_for(a.classes * (int64_t)sizeof(T));
  // segments start at multiples of 32 classes: 16-byte aligned in an aligned row
  a.seg = ((a.classes + cluster - 1) / cluster + 31) / 32 * 32;
  static_assert(32 % V == 0, "aligned segments");
  if (a.seg <= 2048) return launch<T, 128>(a, cluster, st);
  return launch<T, 256>(a, cluster, st);
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
  if (!(a.temperature > 0.f) || a.temperature > 3e38f || !(a.divisor >= 0.f))
    return TL_ERR_INVALID_ARG;
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
  if (!loss && !row_loss && !lse && !dz) return TL_ERR_INVALID_ARG;
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
