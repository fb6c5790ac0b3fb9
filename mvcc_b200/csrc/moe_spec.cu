// moe_spec.cu -- probabilities of a step's logits and the verification of drafted tokens (include/moe_spec.h).
//
//   softmax_rows_kernel  a row is a cluster of 1 to 8 CTAs, each with its share of the row in registers: one read and
//                        one write of the row. Each CTA takes its own maximum and the sum of 2^((x - max) c), the pairs
//                        meet through distributed shared memory behind one cluster barrier, and every CTA rescales
//                        what it holds. Bound by the row's bytes: 8 V.
//   verify_kernel        CTA (chunk, sequence): which drafts are accepted (a few gathered values, found by every CTA
//                        alone), then the fp64 sum of the chunk's weights; the sequence's last CTA to finish finds the
//                        chunk and, in it, the token whose running sum passes u times the total. Only the row that the
//                        token is drawn from is read: 8 V bytes a sequence. fp64, because a running sum in fp32 is off
//                        by more than the smallest gap between two tokens of a large vocabulary, and the choice would
//                        depend on the order of the sum.
#include <algorithm>

#include "../../include/moe_spec.h"
#include "moe_device.cuh"
#include "moe_paged.h"

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
  int V;
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
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// VEC floats a load (4 when rows and length allow it), N loads a thread; N = 0 reads the row again in every pass.
template <int VEC, int N>
__global__ void __launch_bounds__(kSmThreads, N * VEC <= 40 ? 2 : 1) softmax_rows_kernel(
    const __grid_constant__ SoftmaxArgs a) {
  __shared__ float red[2][kSmWarps];
  __shared__ float peer[3][kSmMaxCluster];  // of each CTA of the row: maximum, sum, index of the maximum
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int CL = (int)cluster_size(), rank = (int)cluster_rank();
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x / CL;
  const float* x = a.x + row * a.ldx;
  float* y = a.y + row * a.ldy;
  const float t = a.temperature ? a.temperature[row] : 1.f;
  const bool greedy = !(t > 0.f);
  const float c = greedy ? 0.f : 1.4426950408889634f / t;
  const int chunk = ((a.V + CL - 1) / CL + 3) & ~3;
  const int b0 = min(a.V, rank * chunk), b1 = min(a.V, b0 + chunk);
  auto weight = [&](float v, float m) { return v == m ? 1.f : (v != v ? 0.f : ex2((v - m) * c)); };

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
    for (int k = 0; k < N * VEC; ++k) m = fmaxf(m, r[k]);
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
#pragma unroll
      for (int k = 0; k < N * VEC; ++k) {
        r[k] = m == -INFINITY ? 0.f : weight(r[k], m);
        s += r[k];
      }
    } else {
      for (int i = b0 + tid; i < b1; i += kSmThreads) s += m == -INFINITY ? 0.f : weight(x[i], m);
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
      for (int i = b0 + tid; i < b1; i += kSmThreads) y[i] = f == 0.f ? 0.f : weight(x[i], m) * f;
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

template <int VEC, int N>
cudaError_t launch_softmax(const SoftmaxArgs& args, int R, int cluster, cudaStream_t s) {
  SoftmaxArgs a = args;
  void* p[] = {&a};
  return paged_launch(reinterpret_cast<const void*>(softmax_rows_kernel<VEC, N>), dim3((unsigned)R * cluster),
                      dim3(kSmThreads), 0, s, p, cluster);
}

// ------------------------------------------------------------------ verification

constexpr int kVfThreads = 256;
constexpr int kVfPer = 16;                      // values a thread
constexpr int kVfChunk = kVfThreads * kVfPer;   // values a CTA
constexpr int kVfMaxK = 64;

struct VerifyArgs {
  const float* p;
  const float* q;
  int64_t ldp, ldq;
  const int32_t* drafted;
  const int32_t* n_drafted;
  const float* u;
  int K, V, chunks;
  int32_t* tokens;
  int32_t* accepted;
  uint32_t* ticket;  // [B], zero between calls
  double2* sums;     // [B][chunks]: sum of w, sum of p
};

// A probability as it counts: NaN, negative and infinite entries are zero.
__device__ __forceinline__ float prob(float v) { return v > 0.f && v < INFINITY ? v : 0.f; }

// kVfPer values from i0 on, zero behind V.
template <bool VEC>
__device__ __forceinline__ void load_probs(const float* row, int i0, int V, float (&v)[kVfPer]) {
  if (VEC && i0 + kVfPer <= V) {
#pragma unroll
    for (int k = 0; k < kVfPer; k += 4) {
      const float4 x = *reinterpret_cast<const float4*>(row + i0 + k);
      v[k] = x.x;
      v[k + 1] = x.y;
      v[k + 2] = x.z;
      v[k + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < kVfPer; ++k) v[k] = i0 + k < V ? row[i0 + k] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < kVfPer; ++k) v[k] = prob(v[k]);
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <bool VEC>
__global__ void __launch_bounds__(kVfThreads) verify_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double wsum[2][kVfThreads / 32];
  __shared__ int last, found, chunk_s;
  __shared__ double base_s, target_s;
  __shared__ int use_p_s;
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
  const float* prow = P + acc * a.ldp;
  const bool rejected = acc < n;
  const float* qrow = rejected && Q ? Q + acc * a.ldq : nullptr;
  const int hit = rejected && !Q ? a.drafted[(int64_t)b * K + acc] : -1;  // q is 1 at this token alone
  auto weights = [&](int i0, float (&p)[kVfPer], double (&w)[kVfPer]) {
    load_probs<VEC>(prow, i0, a.V, p);
    if (qrow) {
      float q[kVfPer];
      load_probs<VEC>(qrow, i0, a.V, q);
#pragma unroll
      for (int k = 0; k < kVfPer; ++k) w[k] = fmax((double)p[k] - (double)q[k], 0.0);
    } else {
#pragma unroll
      for (int k = 0; k < kVfPer; ++k) w[k] = i0 + k == hit ? fmax((double)p[k] - 1.0, 0.0) : (double)p[k];
    }
  };
  {
    float p[kVfPer];
    double w[kVfPer], sw = 0.0, sp = 0.0;
    weights(blockIdx.x * kVfChunk + tid * kVfPer, p, w);
#pragma unroll
    for (int k = 0; k < kVfPer; ++k) {
      sw += w[k];
      sp += p[k];
    }
    sw = warp_sum_f64(sw);
    sp = warp_sum_f64(sp);
    if (lane == 0) {
      wsum[0][warp] = sw;
      wsum[1][warp] = sp;
    }
    __syncthreads();
    if (tid == 0) {
      double2 t = make_double2(0.0, 0.0);
      for (int k = 0; k < kVfThreads / 32; ++k) {
        t.x += wsum[0][k];
        t.y += wsum[1][k];
      }
      a.sums[(int64_t)b * a.chunks + blockIdx.x] = t;
      __threadfence();
      last = atomicInc(&a.ticket[b], gridDim.x - 1) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
  }
  // the chunk: warp 0 walks the chunks' sums, 32 at a time
  if (warp == 0) {
    const double2* sums = a.sums + (int64_t)b * a.chunks;
    double tw = 0.0, tp = 0.0;
    for (int k = lane; k < a.chunks; k += 32) {
      const double2 v = __ldcg(sums + k);
      tw += v.x;
      tp += v.y;
    }
    tw = warp_sum_f64(tw);
    tp = warp_sum_f64(tp);
    const bool use_p = !(tw > 0.0);
    const double total = use_p ? tp : tw, target = (double)a.u[(int64_t)b * (K + 1) + K] * total;
    // the first chunk whose running sum passes the target; if rounding leaves none, the last one that holds weight
    int chunk = -1, some = -1;
    double base = 0.0, before = 0.0, some_before = 0.0;
    for (int k0 = 0; k0 < a.chunks && chunk < 0; k0 += 32) {
      const int k = k0 + lane;
      double v = 0.0;
      if (k < a.chunks) {
        const double2 t = __ldcg(sums + k);
        v = use_p ? t.y : t.x;
      }
      double run = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      const uint32_t over = __ballot_sync(0xffffffffu, v > 0.0 && base + run > target);
      const uint32_t pos = __ballot_sync(0xffffffffu, v > 0.0);
      const double prev = base + (run - v);
      if (over) {
        chunk = k0 + __ffs(over) - 1;
        before = __shfl_sync(0xffffffffu, prev, __ffs(over) - 1);
      } else if (pos) {
        some = k0 + 31 - __clz(pos);
        some_before = __shfl_sync(0xffffffffu, prev, 31 - __clz(pos));
      }
      base += __shfl_sync(0xffffffffu, run, 31);
    }
    if (lane == 0) {
      chunk_s = chunk >= 0 ? chunk : some;
      base_s = chunk >= 0 ? before : some_before;
      target_s = target;
      use_p_s = use_p;
      found = 0x7fffffff;
    }
  }
  __syncthreads();
  int token = -1;
  if (chunk_s >= 0) {
    const int i0 = chunk_s * kVfChunk + tid * kVfPer;
    float p[kVfPer];
    double w[kVfPer];
    weights(i0, p, w);
    double mine = 0.0;
    int lastpos = -1;
#pragma unroll
    for (int k = 0; k < kVfPer; ++k) {
      if (use_p_s) w[k] = p[k];
      mine += w[k];
      if (w[k] > 0.0) lastpos = i0 + k;
    }
    double run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (lane == 31) wsum[0][warp] = run;
    __syncthreads();
    double at = base_s;
    for (int k = 0; k < warp; ++k) at += wsum[0][k];
    at += run - mine;
    int first = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < kVfPer; ++k) {
      at += w[k];
      if (w[k] > 0.0 && at > target_s) first = min(first, i0 + k);
    }
    if (first != 0x7fffffff) atomicMin(&found, first);
    __syncthreads();
    if (found == 0x7fffffff) {  // rounding left the target at the chunk's end: its last value with weight
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

int verify_chunks(int V) { return (V + kVfChunk - 1) / kVfChunk; }

// The tickets lead the workspace and have room for every sequence, so that they are where they were whatever batch or
// vocabulary a call has, and the chunks' sums never land on one.
constexpr int kSpecMaxB = 65535;
struct SpecWs {
  size_t ticket, sums, total;
};
SpecWs spec_ws(int B, int V) {
  SpecWs L;
  L.ticket = 0;
  L.sums = ws_align(4 * (size_t)kSpecMaxB);
  L.total = ws_align(L.sums + sizeof(double2) * (size_t)B * verify_chunks(V));
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
  a.V = V;
  const cudaStream_t s = (cudaStream_t)stream;
  const bool vec = V % 4 == 0 && ld_logits % 4 == 0 && ld_probs % 4 == 0 && paged_al16(logits) && paged_al16(probs);
  // CTAs a row: as many as its values need at 40 a thread
  int cl = 1;
  while (cl < kSmMaxCluster && (int64_t)cl * kSmThreads * 40 < V) cl *= 2;
  const int chunk = ((V + cl - 1) / cl + 3) & ~3;
  const int per = (chunk + kSmThreads * 4 - 1) / (kSmThreads * 4);  // groups of four values a thread
  if (vec) {
    if (per <= 2) return (int)launch_softmax<4, 2>(a, R, cl, s);
    if (per <= 5) return (int)launch_softmax<4, 5>(a, R, cl, s);
    if (per <= 10) return (int)launch_softmax<4, 10>(a, R, cl, s);
    if (per <= 16) return (int)launch_softmax<4, 16>(a, R, cl, s);
  } else {
    if (per <= 2) return (int)launch_softmax<1, 8>(a, R, cl, s);
    if (per <= 5) return (int)launch_softmax<1, 20>(a, R, cl, s);
    if (per <= 10) return (int)launch_softmax<1, 40>(a, R, cl, s);
    if (per <= 16) return (int)launch_softmax<1, 64>(a, R, cl, s);
  }
  return (int)launch_softmax<1, 0>(a, R, cl, s);
}

size_t moe_spec_workspace_bytes(int max_B, int V) {
  if (max_B < 1 || max_B > kSpecMaxB || V < 1 || V >= (1 << 24)) return 0;
  return spec_ws(max_B, V).total;
}

int moe_spec_verify(const float* target, int64_t ld_target, const float* draft, int64_t ld_draft,
                    const int32_t* drafted, const int32_t* n_drafted, const float* u, int B, int K, int V,
                    int32_t* tokens, int32_t* accepted, void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  if (B < 0 || B > kSpecMaxB || K < 1 || K > kVfMaxK || V < 1 || V >= (1 << 24) || ld_target < V || (draft && ld_draft < V))
    return (int)cudaErrorInvalidValue;
  if (B == 0) return (int)cudaSuccess;
  if (!target || !drafted || !u || !tokens || !accepted || !workspace || !paged_al16(workspace))
    return (int)cudaErrorInvalidValue;
  if (workspace_bytes < spec_ws(B, V).total) return (int)cudaErrorInvalidValue;
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
  a.chunks = verify_chunks(V);
  a.tokens = tokens;
  a.accepted = accepted;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const SpecWs L = spec_ws(B, V);
  a.ticket = reinterpret_cast<uint32_t*>(ws + L.ticket);
  a.sums = reinterpret_cast<double2*>(ws + L.sums);
  const bool vec = ld_target % 4 == 0 && (!draft || ld_draft % 4 == 0) && paged_al16(target) && paged_al16(draft);
  void* p[] = {&a};
  return (int)paged_launch(vec ? reinterpret_cast<const void*>(verify_kernel<true>)
                               : reinterpret_cast<const void*>(verify_kernel<false>),
                           dim3(a.chunks, B), dim3(kVfThreads), 0, (cudaStream_t)stream, p);
}

}  // extern "C"
