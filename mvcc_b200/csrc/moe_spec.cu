// moe_spec.cu -- probabilities of a step's logits and the verification of drafted tokens (include/moe_spec.h).
//
//   softmax_rows_kernel  short rows: a CTA (or a cluster) a row, its values in registers; one read, one write.
//   softmax_ring_kernel  long rows: a row is a cluster of up to 8 CTAs. Each CTA walks its share of row after row: a
//                        bulk copy brings the next row's share into shared memory while this row's, in registers, is
//                        reduced and stored. The CTAs' (maximum, sum of 2^((x - max) c)) pairs meet through distributed
//                        shared memory behind one cluster barrier a row, and each CTA rescales what it holds. Two CTAs
//                        an SM: one's barriers hide behind the other's stores (192 rows of 151936: 52 us; one CTA an SM
//                        with two buffers 60 us; a CTA per row share without the walk 95 us). Bound by the row's bytes,
//                        8 V.
//   verify_kernel        CTA (chunk, sequence): which drafts are accepted (a few gathered values, found by every warp
//                        alone), then each warp's fp64 sum of the weights of its stretch of the chunk; the sequence's
//                        last CTA to finish finds the stretch and, in it, the token whose running sum passes u times
//                        the total. Only the row that the token is drawn from is read: 8 V bytes a sequence. fp64,
//                        because a running sum in fp32 is off by more than the smallest gap between two tokens of a
//                        large vocabulary, and the choice would depend on the order of the sum. 64 sequences of 4
//                        drafts over 151936 tokens: 19 us (12 us of them bytes, 5 us the two chains of dependent
//                        loads before and after); one sequence 7 us.
#include <algorithm>
#include <atomic>

#include "../../include/moe_spec.h"
#include "moe_device.cuh"
#include "moe_paged.h"
#include "moe_sync.cuh"

namespace moe {
namespace {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------ softmax

constexpr int kSmThreads = 512;
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kSmMaxCluster = 8;

struct SoftmaxArgs {
  const float* x;
  float* y;
  const float* temperature;
  int64_t ldx, ldy;
  int R, V;
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
// Stores v to the same shared variable of CTA `rank` of the cluster.
__device__ __forceinline__ void store_peer(float* p, uint32_t rank, float v) {
  uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, %1;\n\tst.shared::cluster.f32 [r], %2;\n\t}" ::"r"(
                   addr),
               "r"(rank), "f"(v)
               : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}

// log2(e) / t, but never zero: at an infinite temperature a logit of -infinity keeps its weight of zero.
__device__ __forceinline__ float soft_factor(float t) { return fmaxf(1.4426950408889634f / t, 1.4e-45f); }
// 2^((v - m) c) for v <= m, neither a NaN. Where m or c is infinite the difference or the product may be no number: then
// one at the maximum itself, zero below it.
__device__ __forceinline__ float soft_weight(float v, float m, float c) { return ex2((v - m) * c); }
__device__ __forceinline__ float soft_weight_any(float v, float m, float c) {
  return v == m ? 1.f : ex2((v - m) * c);
}
__device__ __forceinline__ bool soft_plain(float m, float c) { return fabsf(m) < INFINITY && c < INFINITY; }
// A NaN never wins: it counts as -infinity.
__device__ __forceinline__ float soft_clean(float v) { return fmaxf(v, -INFINITY); }

// VEC floats a load (4 when rows and length allow it), N loads a thread; N = 0 reads the row again in every pass.
template <int VEC, int N>
__global__ void __launch_bounds__(kSmThreads, VEC == 4 ? 2 : 1) softmax_rows_kernel(
    const __grid_constant__ SoftmaxArgs a) {
  __shared__ float red[2][kSmWarps];
  __shared__ float peer[3][kSmMaxCluster];  // of each CTA of the row: maximum, sum, index of the maximum
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int CL = (int)cluster_size(), rank = (int)cluster_rank();
  cluster_arrive();  // a CTA's shared memory may be written by the others once it has started: waited for before they do
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x / CL;
  const float* x = a.x + row * a.ldx;
  float* y = a.y + row * a.ldy;
  const float t = a.temperature ? a.temperature[row] : 1.f;
  const bool greedy = !(t > 0.f);
  const float c = greedy ? 0.f : soft_factor(t);
  const int chunk = ((a.V + CL - 1) / CL + 3) & ~3;
  const int b0 = min(a.V, rank * chunk), b1 = min(a.V, b0 + chunk);
  auto weight = [&](float v, float m) { return soft_weight_any(v, m, c); };

  float r[N ? N * VEC : 1];
  float m = -INFINITY;
  if constexpr (N > 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = b0 + (k * kSmThreads + tid) * VEC;
      if constexpr (VEC == 4) {
        const float4 v = i < b1 ? __ldcs(reinterpret_cast<const float4*>(x + i)) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        r[4 * k] = v.x;
        r[4 * k + 1] = v.y;
        r[4 * k + 2] = v.z;
        r[4 * k + 3] = v.w;
      } else {
        r[k] = i < b1 ? __ldcs(x + i) : -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < N * VEC; ++k) {
      r[k] = soft_clean(r[k]);
      m = fmaxf(m, r[k]);
    }
  } else {
    for (int i = b0 + tid; i < b1; i += kSmThreads) m = fmaxf(m, x[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
  m = red[0][lane & (kSmWarps - 1)];
#pragma unroll
  for (int o = kSmWarps / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));

  // sum of the weights relative to this CTA's maximum, or the first index that holds it (below 2^24: exact in a float)
  float s;
  if (!greedy) {
    s = 0.f;
    if constexpr (N > 0) {
      float z = m, cz = c;
      if (!soft_plain(m, c)) {  // one at the maximum, zero below it (or everywhere): exponents 0 and -infinity
#pragma unroll
        for (int k = 0; k < N * VEC; ++k) r[k] = r[k] == m && m != -INFINITY ? 0.f : -INFINITY;
        z = 0.f;
        cz = 1.f;
      }
#pragma unroll
      for (int k = 0; k < N * VEC; ++k) {
        r[k] = soft_weight(r[k], z, cz);
        s += r[k];
      }
    } else {
      for (int i = b0 + tid; i < b1; i += kSmThreads) s += m == -INFINITY ? 0.f : weight(soft_clean(x[i]), m);
    }
    s = warp_sum(s);
  } else {
    int first = 1 << 24;
    if constexpr (N > 0) {
#pragma unroll
      for (int k = N * VEC - 1; k >= 0; --k)
        if (r[k] == m) first = min(first, b0 + (k / VEC * kSmThreads + tid) * VEC + k % VEC);
    } else {
      for (int i = b0 + tid; i < b1; i += kSmThreads)
        if (x[i] == m) first = min(first, i);
    }
    s = (float)__reduce_min_sync(0xffffffffu, first);
  }
  if (lane == 0) red[1][warp] = s;
  __syncthreads();
  s = red[1][lane & (kSmWarps - 1)];
#pragma unroll
  for (int o = kSmWarps / 2; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, s, o);
    s = greedy ? fminf(s, v) : s + v;
  }
  cluster_wait();  // every CTA of the cluster has started
  if (tid < CL) {
    store_peer(&peer[0][rank], tid, m);
    store_peer(&peer[1][rank], tid, s);
  }
  cluster_sync();
  float M = -INFINITY;
  for (int k = 0; k < CL; ++k) M = fmaxf(M, peer[0][k]);
  if (!greedy) {
    float total = 0.f;
    for (int k = 0; k < CL; ++k)
      if (peer[0][k] != -INFINITY) total += peer[1][k] * weight(peer[0][k], M);
    const float f = M == -INFINITY || m == -INFINITY ? 0.f : weight(m, M) / total;
    if constexpr (N > 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int i = b0 + (k * kSmThreads + tid) * VEC;
        if (i < b1) {
          if constexpr (VEC == 4)
            __stcs(reinterpret_cast<float4*>(y + i),
                   make_float4(r[4 * k] * f, r[4 * k + 1] * f, r[4 * k + 2] * f, r[4 * k + 3] * f));
          else __stcs(y + i, r[k] * f);
        }
      }
    } else {
      for (int i = b0 + tid; i < b1; i += kSmThreads) y[i] = f == 0.f ? 0.f : weight(soft_clean(x[i]), m) * f;
    }
  } else {
    float best = (float)(1 << 24);
    for (int k = CL - 1; k >= 0; --k)
      if (peer[0][k] == M && M != -INFINITY) best = peer[1][k];
    const int at = (int)best;
    if constexpr (N > 0 && VEC == 4) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int i = b0 + (k * kSmThreads + tid) * 4;
        if (i < b1)
          __stcs(reinterpret_cast<float4*>(y + i), make_float4(i == at ? 1.f : 0.f, i + 1 == at ? 1.f : 0.f,
                                                               i + 2 == at ? 1.f : 0.f, i + 3 == at ? 1.f : 0.f));
      }
    } else {
      for (int i = b0 + tid; i < b1; i += kSmThreads) y[i] = i == at ? 1.f : 0.f;
    }
  }
}

// Long rows. VEC: 4 where every row and share is 16-byte aligned, else 1 (a share is then fetched with the bytes around
// it that complete its 16-byte words, and read from where it begins). N: groups of four values a thread.
template <int VEC, int N>
__global__ void __launch_bounds__(kSmThreads, N <= 10 ? 2 : 1) softmax_ring_kernel(const __grid_constant__ SoftmaxArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full;
  __shared__ float red[2][kSmWarps];
  __shared__ float peer[2][2][kSmMaxCluster];  // by row parity: maxima and sums (or indices) of the row's CTAs
  __shared__ int broken;  // a wait for a copy gave up: this row and those after it are no numbers
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int CL = (int)cluster_size(), rank = (int)cluster_rank();
  const int first = blockIdx.x / CL, step = gridDim.x / CL;
  const int chunk = ((a.V + CL - 1) / CL + 3) & ~3;
  const int b0 = min(a.V, rank * chunk), n = min(a.V, b0 + chunk) - b0;
  cluster_arrive();
  if (tid == 0) {
    broken = 0;
    mbar_init(&full, 1);
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  int issued = 0;  // copies that thread 0 has started
  auto fetch = [&](int64_t row) {  // thread 0
    if (row >= a.R || n == 0) return;
    ++issued;
    const float* src = a.x + row * a.ldx + b0;
    expect_tx(&full, span_bytes(src, n * 4));
    bulk_span(smem, src, n * 4, &full);
  };
  if (tid == 0) fetch(first);
  int turn = 0;
  bool ok = true;
  for (int row = first; row < a.R; row += step, ++turn) {
    if (n > 0 && ok) ok = bar_wait(&full, turn & 1);
    const float* x = a.x + row * a.ldx + b0;
    const float* sh = reinterpret_cast<const float*>(smem + (VEC == 4 ? 0 : span_delta(x)));
    float r[N * 4];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < N * 4 / VEC; ++k) {
      const int i = (k * kSmThreads + tid) * VEC;
      if constexpr (VEC == 4) {
        const float4 v = i < n ? *reinterpret_cast<const float4*>(sh + i)
                               : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        r[4 * k] = v.x;
        r[4 * k + 1] = v.y;
        r[4 * k + 2] = v.z;
        r[4 * k + 3] = v.w;
      } else {
        r[k] = i < n ? sh[i] : -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < N * 4; ++k) {
      r[k] = soft_clean(r[k]);
      m = fmaxf(m, r[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[0][warp] = m;
    if (!ok) broken = 1;
    __syncthreads();  // the buffer has been read
    if (tid == 0 && !broken) fetch((int64_t)row + step);
    __syncwarp();
    m = red[0][lane & (kSmWarps - 1)];
#pragma unroll
    for (int o = kSmWarps / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float t = a.temperature ? a.temperature[row] : 1.f;
    const bool greedy = !(t > 0.f);
    const float c = greedy ? 0.f : soft_factor(t);
    float s;
    if (!greedy) {
      float z = m, cz = c;
      if (!soft_plain(m, c)) {  // one at the maximum, zero below it (or everywhere): exponents 0 and -infinity
#pragma unroll
        for (int k = 0; k < N * 4; ++k) r[k] = r[k] == m && m != -INFINITY ? 0.f : -INFINITY;
        z = 0.f;
        cz = 1.f;
      }
      float ss[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < N * 4; ++k) {
        r[k] = soft_weight(r[k], z, cz);
        ss[k & 1] += r[k];
      }
      s = warp_sum(ss[0] + ss[1]);
    } else {
      int at = 1 << 24;
#pragma unroll
      for (int k = N * 4 - 1; k >= 0; --k)
        if (r[k] == m) at = min(at, b0 + (k / VEC * kSmThreads + tid) * VEC + k % VEC);
      s = (float)__reduce_min_sync(0xffffffffu, at);
    }
    if (lane == 0) red[1][warp] = s;
    __syncthreads();
    s = red[1][lane & (kSmWarps - 1)];
#pragma unroll
    for (int o = kSmWarps / 2; o > 0; o >>= 1) {
      const float v = __shfl_xor_sync(0xffffffffu, s, o);
      s = greedy ? fminf(s, v) : s + v;
    }
    float(*pr)[kSmMaxCluster] = peer[turn & 1];
    if (turn == 0) cluster_wait();  // every CTA of the cluster has started
    if (tid < CL) {
      // a copy that never came: a maximum that takes part everywhere, and a sum (or index) that is no number
      store_peer(&pr[0][rank], tid, broken ? INFINITY : m);
      store_peer(&pr[1][rank], tid, broken ? __int_as_float(0x7fc00000) : s);
    }
    cluster_sync();  // the other parity's values are written again only after the next row's barrier
    float M = -INFINITY;
    for (int k = 0; k < CL; ++k) M = fmaxf(M, pr[0][k]);
    float* y = a.y + row * a.ldy + b0;
    float f = 0.f;
    int at = -1;
    if (!greedy) {
      float total = 0.f;
      for (int k = 0; k < CL; ++k)
        if (pr[0][k] != -INFINITY) total += pr[1][k] * soft_weight_any(pr[0][k], M, c);
      f = M == -INFINITY || m == -INFINITY ? 0.f : soft_weight_any(m, M, c) / total;
    } else {
      float index = -1.f;
      for (int k = CL - 1; k >= 0; --k)
        if (pr[0][k] == M && M != -INFINITY) index = pr[1][k];
      f = index == index ? 1.f : index;
      at = (int)index - b0;
#pragma unroll
      for (int k = 0; k < N * 4; ++k) r[k] = (k / VEC * kSmThreads + tid) * VEC + k % VEC == at ? 1.f : 0.f;
    }
#pragma unroll
    for (int k = 0; k < N * 4 / VEC; ++k) {
      const int i = (k * kSmThreads + tid) * VEC;
      if (i < n) {
        if constexpr (VEC == 4)
          __stcs(reinterpret_cast<float4*>(y + i),
                 make_float4(r[4 * k] * f, r[4 * k + 1] * f, r[4 * k + 2] * f, r[4 * k + 3] * f));
        else __stcs(y + i, r[k] * f);
      }
    }
  }
  if (tid == 0 && issued > 0) bar_wait(&full, (issued - 1) & 1);  // the last copy may still be landing, if a wait gave up
}

template <int VEC, int N>
cudaError_t launch_softmax(const SoftmaxArgs& args, int R, int cluster, cudaStream_t s) {
  SoftmaxArgs a = args;
  void* p[] = {&a};
  return paged_launch(reinterpret_cast<const void*>(softmax_rows_kernel<VEC, N>), dim3((unsigned)R * cluster),
                      dim3(kSmThreads), 0, s, p, cluster);
}

template <int VEC, int N>
cudaError_t launch_ring(const SoftmaxArgs& args, int cluster, cudaStream_t s) {
  const void* fn = reinterpret_cast<const void*>(softmax_ring_kernel<VEC, N>);
  constexpr int kSmem = kSmThreads * 4 * N * 4 + 16;
  static SmemGrant granted;
  cudaError_t e = grant_smem(fn, kSmem, 0, granted);
  if (e != cudaSuccess) return e;
  // as many clusters as the device holds at once, asked once per device and cluster size
  constexpr int kDevices = 64;
  static std::atomic<int> resident[kDevices][4];
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int lg = cluster == 8 ? 3 : (cluster == 4 ? 2 : (cluster == 2 ? 1 : 0));
  int n = dev < kDevices ? resident[dev][lg].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cluster);
    cfg.blockDim = dim3(kSmThreads);
    cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&n, fn, &cfg);
    if (e != cudaSuccess) return e;
    n = std::max(n, 1);
    if (dev < kDevices) resident[dev][lg].store(n, std::memory_order_relaxed);
  }
  SoftmaxArgs a = args;
  void* p[] = {&a};
  return paged_launch(fn, dim3((unsigned)(std::min(n, a.R) * cluster)), dim3(kSmThreads), kSmem, s, p, cluster);
}

// ------------------------------------------------------------------ verification

constexpr int kVfThreads = 256;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfMaxK = 64;
constexpr int kVfMaxChunks = 1024;   // CTAs of a sequence at most
constexpr int kVfStretch = 128;      // a warp's stretch is a multiple of this many values (a float4 a lane)

struct VerifyArgs {
  const float* p;
  const float* q;
  int64_t ldp, ldq;
  const int32_t* drafted;
  const int32_t* n_drafted;
  const float* u;
  int K, V, stretch, stretches;  // values of a warp's stretch; stretches of a row
  int32_t* tokens;
  int32_t* accepted;
  uint32_t* ticket;  // [B], zero between calls
  double* sums;      // [B][stretches]
};

// A probability as it counts: NaN, negative and infinite entries are zero.
__device__ __forceinline__ float prob(float v) {
  return __float_as_uint(v) < 0x7f800000u ? v : 0.f;  // below infinity's bits and without a sign
}

// Four values of a row from i on, as they count; zero behind V.
template <bool VEC>
__device__ __forceinline__ float4 load_probs(const float* row, int i, int V) {
  float4 x;
  if (VEC) {  // V a multiple of four
    x = i < V ? __ldcs(reinterpret_cast<const float4*>(row + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
    x.x = i < V ? row[i] : 0.f;
    x.y = i + 1 < V ? row[i + 1] : 0.f;
    x.z = i + 2 < V ? row[i + 2] : 0.f;
    x.w = i + 3 < V ? row[i + 3] : 0.f;
  }
  return x;
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A non-negative finite fp32 as fp64, by moving its fields (a conversion instruction has an eighth of the rate). Zero
// becomes 2^-127 and values below 2^-126 are off by less than that. The weights below are differences of two such values:
// equal ones cancel exactly, and a row's sum is off by less than 2^24 2^-126, which 53 bits do not show unless the sum
// itself is below kTiny. Such a row is weighed again by conversion (18.9 us for 64 x 4 drafts; with the small values put
// right in every weight, 26.8).
constexpr double kTiny = 0x1p-40;
template <bool EXACT>
__device__ __forceinline__ double widen(float v) {
  if (EXACT) return (double)v;
  const uint32_t u = __float_as_uint(v);
  return __hiloint2double((int)((u >> 3) + 0x38000000u), (int)(u << 29));
}

// The weights of four values, i on: the residual of p over q, or p itself (q = 0). max(p, q) - q is exact, not negative,
// and zero where p = q.
struct Weights {
  const float* p;
  const float* q;  // null: q is zero but for `hit`, where it is one
  int hit;
  template <bool EXACT>
  __device__ __forceinline__ void of(int i, const float4& pv, const float4& qv, double (&w)[4]) const {
    const float a[4] = {pv.x, pv.y, pv.z, pv.w}, b[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float y = q ? prob(b[k]) : (i + k == hit ? 1.f : 0.f);
      w[k] = widen<EXACT>(fmaxf(prob(a[k]), y)) - widen<EXACT>(y);
    }
  }
};

// Sum of the weights of [i0, i1), over the warp.
template <bool VEC>
__device__ double stretch_sum(const Weights& W, int i0, int i1, int V, int lane) {
  constexpr int kU = 4;
  double s = 0.0;
  for (int base = i0; base < i1; base += kU * 128) {
    float4 p[kU], q[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = base + u * 128 + lane * 4;
      p[u] = i < i1 ? load_probs<VEC>(W.p, i, V) : make_float4(0.f, 0.f, 0.f, 0.f);
      q[u] = W.q && i < i1 ? load_probs<VEC>(W.q, i, V) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      double w[4];
      W.of<false>(base + u * 128 + lane * 4, p[u], q[u], w);
      s += (w[0] + w[1]) + (w[2] + w[3]);
    }
  }
  return warp_sum_f64(s);
}

// The same by conversion, for rows whose sum is tiny: out of line, so that its instructions are not among those of the rest.
template <bool VEC>
__device__ __noinline__ double stretch_sum_exact(const Weights& W, int i0, int i1, int V, int lane) {
  double s = 0.0;
#pragma unroll 1
  for (int i = i0 + lane * 4; i < i1; i += 128) {
    double w[4];
    W.of<true>(i, load_probs<VEC>(W.p, i, V), W.q ? load_probs<VEC>(W.q, i, V) : make_float4(0.f, 0.f, 0.f, 0.f), w);
    s += (w[0] + w[1]) + (w[2] + w[3]);
  }
  return warp_sum_f64(s);
}

template <bool VEC>
__global__ void __launch_bounds__(kVfThreads) verify_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double wsum[kVfWarps];
  __shared__ int last, found, stretch_s, some_s;
  __shared__ double base_s, target_s, total_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y, K = a.K;
  pdl_wait();
  pdl_launch_dependents();
  // the accepted drafts, found by every warp: lane i looks at drafts i and i + 32
  const int n = a.n_drafted ? min(max(a.n_drafted[b], 0), K) : K;
  const float* P = a.p + (int64_t)b * (K + 1) * a.ldp;
  const float* Q = a.q ? a.q + (int64_t)b * K * a.ldq : nullptr;
  int acc = n;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    bool ok = true;
    if (i < n) {
      const int x = a.drafted[(int64_t)b * K + i];
      ok = false;
      if (x >= 0 && x < a.V) {
        const double px = prob(P[i * a.ldp + x]), qx = Q ? prob(Q[i * a.ldq + x]) : 1.f;
        ok = (double)a.u[(int64_t)b * (K + 1) + i] * qx < px;
      }
    }
    const uint32_t no = ~__ballot_sync(0xffffffffu, ok);
    if (no) {
      acc = i0 + __ffs(no) - 1;
      break;
    }
  }
  const bool rejected = acc < n;
  Weights W;
  W.p = P + acc * a.ldp;
  W.q = rejected && Q ? Q + acc * a.ldq : nullptr;
  W.hit = rejected && !Q ? a.drafted[(int64_t)b * K + acc] : -1;
  double* sums = a.sums + (int64_t)b * a.stretches;
  {
    const int k = blockIdx.x * kVfWarps + warp;
    if (k < a.stretches) {
      const double s = stretch_sum<VEC>(W, k * a.stretch, min(a.V, (k + 1) * a.stretch), a.V, lane);
      if (lane == 0) __stcg(sums + k, s);
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicInc(&a.ticket[b], gridDim.x - 1) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
  }
  // the first stretch whose running sum passes the target; where rounding leaves none, the last one that holds weight.
  // A thread takes neighbouring stretches, up to 32 of them.
  const int each = (a.stretches + kVfThreads - 1) / kVfThreads;
  auto choose = [&]() {
    const int k0 = min(a.stretches, tid * each), k1 = min(a.stretches, k0 + each);
    double mine = 0.0;
    for (int k = k0; k < k1; ++k) mine += __ldcg(sums + k);
    double run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (lane == 31) wsum[warp] = run;
    if (tid == 0) {
      stretch_s = 0x7fffffff;
      some_s = -1;
    }
    __syncthreads();
    double before = 0.0, total = 0.0;
    for (int k = 0; k < kVfWarps; ++k) {
      if (k < warp) before += wsum[k];
      total += wsum[k];
    }
    before += run - mine;
    const double target = (double)a.u[(int64_t)b * (K + 1) + K] * total;
    int hit = -1, some = -1;
    double at = before, hit_base = 0.0, some_base = 0.0;
    for (int k = k0; k < k1; ++k) {
      const double v = __ldcg(sums + k);
      if (v > 0.0) {
        if (hit < 0 && at + v > target) {
          hit = k;
          hit_base = at;
        }
        some = k;
        some_base = at;
      }
      at += v;
    }
    if (hit >= 0) atomicMin(&stretch_s, hit);
    if (some >= 0) atomicMax(&some_s, some);
    __syncthreads();
    const bool none = stretch_s == 0x7fffffff;
    const int pick = none ? some_s : stretch_s;
    if (pick >= k0 && pick < k1) base_s = none ? some_base : hit_base;
    if (tid == 0) {
      target_s = target;
      total_s = total;
      found = 0x7fffffff;
    }
    __syncthreads();
    return pick;
  };
  int stretch;
  bool exact = false, residual = rejected;
  while (true) {
    stretch = choose();
    if (stretch < 0 && residual) {  // no residual anywhere: the row itself
      residual = false;
      W.q = nullptr;
      W.hit = -1;
    } else if (stretch >= 0 && total_s < kTiny && !exact) {
      exact = true;
    } else {
      break;
    }
    for (int k = warp; k < a.stretches; k += kVfWarps) {
      const int i0 = k * a.stretch, i1 = min(a.V, i0 + a.stretch);
      const double s = exact ? stretch_sum_exact<VEC>(W, i0, i1, a.V, lane) : stretch_sum<VEC>(W, i0, i1, a.V, lane);
      if (lane == 0) __stcg(sums + k, s);
    }
    __syncthreads();
  }
  int token = -1;
  if (stretch >= 0) {
    // the stretch, 1024 values at a time: four a thread, running sums over the CTA
    const int end = min(a.V, (stretch + 1) * a.stretch);
    double base = base_s;
    int lastpos = -1;
    for (int i0 = stretch * a.stretch; i0 < end; i0 += kVfThreads * 4) {
      const int i = i0 + tid * 4;
      double w[4] = {0.0, 0.0, 0.0, 0.0};
      if (i < end) {
        const float4 p = load_probs<VEC>(W.p, i, a.V);
        const float4 q = W.q ? load_probs<VEC>(W.q, i, a.V) : make_float4(0.f, 0.f, 0.f, 0.f);
        if (exact) W.of<true>(i, p, q, w);
        else W.of<false>(i, p, q, w);
      }
      const double mine = (w[0] + w[1]) + (w[2] + w[3]);
      double run = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      if (lane == 31) wsum[warp] = run;
      __syncthreads();
      double at = base;
      for (int k = 0; k < kVfWarps; ++k) {
        if (k < warp) at += wsum[k];
        base += wsum[k];
      }
      at += run - mine;
      int first = 0x7fffffff;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        at += w[k];
        if (w[k] > 0.0) {
          lastpos = i + k;
          if (at > target_s) first = min(first, i + k);
        }
      }
      if (first != 0x7fffffff) atomicMin(&found, first);
      __syncthreads();
      if (found != 0x7fffffff) break;
    }
    if (found == 0x7fffffff) {  // rounding left the target at the stretch's end: its last value with weight
      __syncthreads();
      if (tid == 0) found = -1;
      __syncthreads();
      if (lastpos >= 0) atomicMax(&found, lastpos);
      __syncthreads();
    }
    token = found;
  }
  for (int i = tid; i <= K; i += kVfThreads)
    a.tokens[(int64_t)b * (K + 1) + i] = i < acc ? a.drafted[(int64_t)b * K + i] : (i == acc ? token : -1);
  if (tid == 0) a.accepted[b] = acc;
}

// The tickets lead the workspace and have room for every sequence, so that they are where they were whatever batch or
// vocabulary a call has, and the chunks' sums never land on one.
constexpr int kSpecMaxB = 65535;
struct SpecWs {
  size_t ticket, sums, total;
};
SpecWs spec_ws(int B) {
  SpecWs L;
  L.ticket = 0;
  L.sums = ws_align(4 * (size_t)kSpecMaxB);
  L.total = ws_align(L.sums + sizeof(double) * (size_t)B * kVfMaxChunks * kVfWarps);
  return L;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_softmax_rows(const float* logits, int64_t ld_logits, int R, int V, const float* temperature, float* probs,
                     int64_t ld_probs, moe_stream_t stream) {
  if (R < 0 || R > (1 << 28) - 1 || V < 1 || V >= (1 << 24) || ld_logits < V || ld_probs < V)
    return (int)cudaErrorInvalidValue;
  if (R == 0) return (int)cudaSuccess;
  if (!logits || !probs || (logits == probs && ld_logits != ld_probs)) return (int)cudaErrorInvalidValue;
  SoftmaxArgs a;
  a.x = logits;
  a.y = probs;
  a.temperature = temperature;
  a.ldx = ld_logits;
  a.ldy = ld_probs;
  a.R = R;
  a.V = V;
  const cudaStream_t s = (cudaStream_t)stream;
  const bool vec = V % 4 == 0 && ld_logits % 4 == 0 && ld_probs % 4 == 0 && paged_al16(logits) && paged_al16(probs);
  // CTAs a row: as many as its values need at 40 a thread, and more, down to 4096 values each, where the rows alone do
  // not fill the GPU
  int cl = 1;
  while (cl < kSmMaxCluster && ((int64_t)cl * kSmThreads * 40 < V || ((int64_t)R * cl * 2 <= paged_sms() && V > cl * 8192)))
    cl *= 2;
  const int chunk = ((V + cl - 1) / cl + 3) & ~3;
  const int per = (chunk + kSmThreads * 4 - 1) / (kSmThreads * 4);  // groups of four values a thread
  if (vec) {
    if (per <= 2) return (int)launch_softmax<4, 2>(a, R, cl, s);
    if (per <= 5) return (int)launch_softmax<4, 5>(a, R, cl, s);
    if (per <= 10) return (int)launch_ring<4, 10>(a, cl, s);
    if (per <= 14) return (int)launch_ring<4, 14>(a, cl, s);
  } else {
    if (per <= 2) return (int)launch_softmax<1, 8>(a, R, cl, s);
    if (per <= 5) return (int)launch_softmax<1, 20>(a, R, cl, s);
    if (per <= 10) return (int)launch_ring<1, 10>(a, cl, s);
    if (per <= 14) return (int)launch_ring<1, 14>(a, cl, s);
  }
  // longer than eight CTAs hold: three reads of each row (128 rows of 229376 take 57 us above, of 229380 here 105)
  return (int)launch_softmax<1, 0>(a, R, cl, s);
}

size_t moe_spec_workspace_bytes(int max_B, int V) {
  if (max_B < 1 || max_B > kSpecMaxB || V < 1 || V >= (1 << 24)) return 0;
  return spec_ws(max_B).total;
}

int moe_spec_verify(const float* target, int64_t ld_target, const float* draft, int64_t ld_draft,
                    const int32_t* drafted, const int32_t* n_drafted, const float* u, int B, int K, int V,
                    int32_t* tokens, int32_t* accepted, void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  if (B < 0 || B > kSpecMaxB || K < 0 || K > kVfMaxK || V < 1 || V >= (1 << 24) || ld_target < V || (draft && ld_draft < V))
    return (int)cudaErrorInvalidValue;
  if (B == 0) return (int)cudaSuccess;
  if (!target || (!drafted && K > 0) || !u || !tokens || !accepted || !workspace || !paged_al16(workspace))
    return (int)cudaErrorInvalidValue;
  if (workspace_bytes < spec_ws(B).total) return (int)cudaErrorInvalidValue;
  VerifyArgs a;
  a.p = target;
  a.q = draft;
  a.ldp = ld_target;
  a.ldq = ld_draft;
  a.drafted = drafted;
  a.n_drafted = n_drafted;
  a.u = u;
  a.K = K;
  a.V = V;
  // CTAs a sequence: four an SM over the batch (as many as fit at once; six: 64 x 4 drafts take 22.5 instead of 19.3 us),
  // so that what a CTA does once, finding the accepted drafts, is paid over as many values as the batch allows, but at
  // least 1024 values each
  const int want = std::max(1, (paged_sms() * 4 + B - 1) / B);
  const int most = std::min(kVfMaxChunks, (V + 1023) / 1024);
  a.stretch = (V + std::min(want, most) * kVfWarps - 1) / (std::min(want, most) * kVfWarps);
  a.stretch = (a.stretch + kVfStretch - 1) / kVfStretch * kVfStretch;
  a.stretches = (V + a.stretch - 1) / a.stretch;
  const int chunks = (a.stretches + kVfWarps - 1) / kVfWarps;
  a.tokens = tokens;
  a.accepted = accepted;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const SpecWs L = spec_ws(B);
  a.ticket = reinterpret_cast<uint32_t*>(ws + L.ticket);
  a.sums = reinterpret_cast<double*>(ws + L.sums);
  const bool vec = V % 4 == 0 && ld_target % 4 == 0 && (!draft || ld_draft % 4 == 0) && paged_al16(target) && paged_al16(draft);
  void* p[] = {&a};
  return (int)paged_launch(vec ? reinterpret_cast<const void*>(verify_kernel<true>)
                               : reinterpret_cast<const void*>(verify_kernel<false>),
                           dim3(chunks, B), dim3(kVfThreads), 0, (cudaStream_t)stream, p);
}

}  // extern "C"
