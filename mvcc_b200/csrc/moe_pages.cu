// moe_pages.cu -- the pages of a paged key-value cache (include/moe_paged.h): growing, shrinking, forking, compacting
// and copying, and the write of a step's new keys and values.
//
// A page call is a plan and a move. The plan (which pages change hands) is integer work over lists, tables and the
// holder counts: one CTA of 1024 threads, so that its steps are separated by block barriers and its result depends on
// the inputs alone. The move is pure traffic: the plan's (source, destination, rows) triples times layers times {k, v},
// cut into 16 KB pieces that the whole GPU takes in turn. The move is a launch of its own, programmatically dependent
// on the plan's: as one cooperative launch with a barrier between them, forking 32 sequences and growing them took 36 us
// instead of 24.
//
// Measured on a B200: 32 children forked from 4 sequences of 2087 tokens, freed, and grown by a token over 10 layers
// (25 MB copied) 24 us: 10 us of it the move, the rest the latency of three plans; compaction of a pool of 3001 pages,
// 40 % live, over 4 layers (377 MB moved) 131 us, 5.8 TB/s read and written.
#include <algorithm>
#include <cstring>

#include <cuda_fp8.h>

#include "moe_device.cuh"
#include "moe_paged.h"

namespace moe {
namespace {

constexpr int kPlanThreads = 1024;

struct PageArgs {
  int32_t* tables;
  int32_t* refs;
  int32_t* lens;
  int32_t num_pages, page, max_seqs, max_pages;
  const int32_t* a;  // seqs, or src
  const int32_t* b;  // new_lens, or dst
  int n;
  uint32_t* err;
  int32_t* ncopy;
  int32_t* copies;  // [.][3]: source page, destination page, rows
  int32_t* list;
  int32_t* map;
};

// The lowest `want` free pages in ascending order into list (all of them when want >= their number); returns how many
// were found, the same in every thread. Each warp looks at 32 k pages a turn, lane by lane, so that a ballot gives
// the order. `ahead`: the first turn's holder counts, read before.
constexpr int kFreeU = 4;
struct Ahead {
  int refs[kFreeU];
  __device__ __forceinline__ void read(const int32_t* r, int num_pages) {
    const int w0 = (threadIdx.x >> 5) * 32 * kFreeU + (threadIdx.x & 31);
#pragma unroll
    for (int u = 0; u < kFreeU; ++u) refs[u] = w0 + u * 32 < num_pages ? __ldcg(r + w0 + u * 32) : 1;
  }
};
__device__ int find_free(const int32_t* refs, int num_pages, int want, int32_t* list, int* sm, const Ahead* ahead) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int found = 0;
  for (int base = 0; base < num_pages && found < want; base += kPlanThreads * kFreeU) {
    const int w0 = base + warp * 32 * kFreeU;
    uint32_t free_mask[kFreeU];
    int mine = 0;
#pragma unroll
    for (int u = 0; u < kFreeU; ++u) {
      const int p = w0 + u * 32 + lane;
      const int r = base == 0 && ahead ? ahead->refs[u] : (p < num_pages ? __ldcg(refs + p) : 1);
      free_mask[u] = __ballot_sync(0xffffffffu, r == 0);
      mine += __popc(free_mask[u]);
    }
    int total;
    const int before = block_excl_scan(lane == 0 ? mine : 0, sm, &total);
    int at = found + __shfl_sync(0xffffffffu, before, 0);
#pragma unroll
    for (int u = 0; u < kFreeU; ++u) {
      if (free_mask[u] >> lane & 1) {
        const int i = at + __popc(free_mask[u] & ((1u << lane) - 1));
        if (i < want) list[i] = w0 + u * 32 + lane;
      }
      at += __popc(free_mask[u]);
    }
    found += total;
    __syncthreads();
  }
  return min(found, want);
}

__device__ __forceinline__ bool page_ok(const PageArgs& a, int p) { return p >= 0 && p < a.num_pages; }

// moe_paged_resize. Shared memory: five ints a list entry and a bit a sequence.
__global__ void __launch_bounds__(kPlanThreads) resize_plan_kernel(const __grid_constant__ PageArgs a) {
  extern __shared__ int sh[];
  __shared__ int sm[32];
  __shared__ int bad, copies, released;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = kPlanThreads / 32, n = a.n, pg = a.page;
  int* seq = sh;
  int* old = seq + n;
  int* neu = old + n;
  int* last = neu + n;   // the page that must be held alone, or -1
  int* start = last + n; // the sequence's first entry of the free list; bit 31: it copies
  uint32_t* seen = reinterpret_cast<uint32_t*>(start + n);
  pdl_wait();
  pdl_launch_dependents();
  Ahead ahead;
  ahead.read(a.refs, a.num_pages);
  if (tid == 0) {
    bad = 0;
    copies = 0;
    released = 0;
    *a.ncopy = 0;
  }
  for (int i = tid; i < (a.max_seqs + 31) / 32; i += kPlanThreads) seen[i] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kPlanThreads) {
    const int s = a.a[i], m = a.b[i];
    bool fine = s >= 0 && s < a.max_seqs && m >= 0 && m <= a.max_pages * pg;
    if (fine) fine = !(atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1);
    int o = fine ? a.lens[s] : 0;
    fine = fine && o >= 0 && o <= a.max_pages * pg;
    if (!fine) bad = 1;
    seq[i] = s;
    old[i] = o;
    neu[i] = m;
  }
  __syncthreads();
  if (bad) {
    if (tid == 0) atomicOr(a.err, (uint32_t)MOE_ERR_SEQ_ID);
    return;
  }
  // 1. the holders of the pages behind the new ends (tables follow once the call is certain)
  for (int i = warp; i < n; i += nw) {
    const int held = (old[i] + pg - 1) / pg, want = (neu[i] + pg - 1) / pg;
    for (int j = want + lane; j < held; j += 32) {
      const int p = a.tables[(int64_t)seq[i] * a.max_pages + j];
      if (page_ok(a, p)) atomicSub(&a.refs[p], 1);
      else atomicOr(a.err, (uint32_t)MOE_ERR_PAGE_ID);
    }
    if (lane == 0 && want < held) released = 1;
  }
  // 2. the partly filled page at the end of what stays
  for (int i = tid; i < n; i += kPlanThreads) {
    const int kept = min(old[i], neu[i]);
    int p = -1;
    if (kept % pg) {
      p = a.tables[(int64_t)seq[i] * a.max_pages + kept / pg];
      if (!page_ok(a, p)) {
        p = -1;
        atomicOr(a.err, (uint32_t)MOE_ERR_PAGE_ID);
      }
    }
    last[i] = p;
  }
  __syncthreads();
  // 3. who copies it: the listed holders but the last, unless others hold it too; and what each sequence takes
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int need = 0, copy = 0;
    if (i < n) {
      const int held = (old[i] + pg - 1) / pg, want = (neu[i] + pg - 1) / pg;
      if (last[i] >= 0) {
        const int r = __ldcg(&a.refs[last[i]]);
        if (r > 1) {
          int before = 0;
          for (int j = 0; j < i; ++j) before += last[j] == last[i];
          copy = before < r - 1;
        }
      }
      need = min(copy + max(0, want - held), a.num_pages + 1);  // enough to fail, too little to overflow a sum
    }
    int total;
    const int ex = block_excl_scan(need, sm, &total);
    if (i < n) start[i] = (base + ex) | (copy << 31);
    base += total;
    __syncthreads();
    if (base > a.num_pages) break;  // more than there can be: no sum may pass the list
  }
  const int want_all = base;
  const int found = want_all > a.num_pages ? -1
                                           : find_free(a.refs, a.num_pages, want_all, a.list, sm,
                                                       released ? nullptr : &ahead);
  __syncthreads();
  if (found < want_all) {  // nothing is changed: the holders come back
    for (int i = warp; i < n; i += nw) {
      const int held = (old[i] + pg - 1) / pg, want = (neu[i] + pg - 1) / pg;
      for (int j = want + lane; j < held; j += 32) {
        const int p = a.tables[(int64_t)seq[i] * a.max_pages + j];
        if (page_ok(a, p)) atomicAdd(&a.refs[p], 1);
      }
    }
    if (tid == 0) atomicOr(a.err, (uint32_t)MOE_ERR_NO_PAGES);
    return;
  }
  // 4. tables, holders and lengths
  for (int i = warp; i < n; i += nw) {
    const int held = (old[i] + pg - 1) / pg, want = (neu[i] + pg - 1) / pg, copy = (uint32_t)start[i] >> 31;
    const int32_t* take = a.list + (start[i] & 0x7fffffff);
    int32_t* row = a.tables + (int64_t)seq[i] * a.max_pages;
    for (int j = want + lane; j < held; j += 32) row[j] = -1;
    for (int j = held + lane; j < want; j += 32) {
      const int p = take[copy + j - held];
      row[j] = p;
      a.refs[p] = 1;
    }
    if (lane == 0) {
      if (copy) {
        const int kept = min(old[i], neu[i]), p = take[0];
        row[kept / pg] = p;
        a.refs[p] = 1;
        atomicSub(&a.refs[last[i]], 1);
        const int k = atomicAdd(&copies, 1);  // the copies are disjoint: their order does not matter
        a.copies[3 * k] = last[i];
        a.copies[3 * k + 1] = p;
        a.copies[3 * k + 2] = kept % pg;
      }
      a.lens[seq[i]] = neu[i];
    }
  }
  __syncthreads();
  if (tid == 0) *a.ncopy = copies;
}

// moe_paged_fork: every CTA checks the lists, the cluster agrees, then the rows are shared out.
constexpr int kForkCluster = 8;
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__global__ void __launch_bounds__(kPlanThreads) fork_kernel(const __grid_constant__ PageArgs a) {
  extern __shared__ uint32_t seen[];  // a bit a sequence: it is a dst
  __shared__ int bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = kPlanThreads / 32;
  pdl_wait();
  pdl_launch_dependents();
  if (tid == 0) bad = 0;
  for (int i = tid; i < (a.max_seqs + 31) / 32; i += kPlanThreads) seen[i] = 0;
  __syncthreads();
  for (int i = tid; i < a.n; i += kPlanThreads) {
    const int d = a.b[i], s = a.a[i];
    const bool dst = d >= 0 && d < a.max_seqs, src = s >= 0 && s < a.max_seqs;
    const int dn = dst ? a.lens[d] : 1, sn = src ? a.lens[s] : -1;
    if (dn != 0 || sn < 0 || sn > a.max_pages * a.page) bad = 1;
    if (dst && (atomicOr(&seen[d >> 5], 1u << (d & 31)) >> (d & 31) & 1)) bad = 1;
  }
  __syncthreads();
  for (int i = tid; i < a.n; i += kPlanThreads) {
    const int s = a.a[i];
    if (s >= 0 && s < a.max_seqs && (seen[s >> 5] >> (s & 31) & 1)) bad = 1;
  }
  __syncthreads();
  cluster_sync();  // no CTA changes a length before every CTA has looked at them
  if (bad) {
    if (tid == 0 && blockIdx.x == 0) atomicOr(a.err, (uint32_t)MOE_ERR_SEQ_ID);
    return;
  }
  for (int i = blockIdx.x * nw + warp; i < a.n; i += kForkCluster * nw) {
    const int s = a.a[i], d = a.b[i], len = a.lens[s], held = (len + a.page - 1) / a.page;
    const int32_t* from = a.tables + (int64_t)s * a.max_pages;
    int32_t* to = a.tables + (int64_t)d * a.max_pages;
    for (int j = lane; j < held; j += 32) {
      const int p = from[j];
      to[j] = p;
      if (page_ok(a, p)) atomicAdd(&a.refs[p], 1);
      else atomicOr(a.err, (uint32_t)MOE_ERR_PAGE_ID);
    }
    if (lane == 0) a.lens[d] = len;
  }
}

// moe_paged_compact: the free ids below the number of live pages (list) and the live ids behind it meet in order.
// map[p] is where the live page p >= n_live goes; no other entry is read.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const __grid_constant__ PageArgs a) {
  constexpr int kU = 4;
  __shared__ int sm[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();
  int mine = 0;
  for (int p = tid; p < a.num_pages; p += kPlanThreads) mine += a.refs[p] != 0;
  int live;
  block_excl_scan(mine, sm, &live);
  const int holes = find_free(a.refs, live, live, a.list, sm, nullptr);
  __syncthreads();
  int found = 0;
  for (int base = live; base < a.num_pages && found < holes; base += kPlanThreads * kU) {
    const int w0 = base + warp * 32 * kU;
    uint32_t mask[kU];
    int cnt = 0;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int p = w0 + u * 32 + lane;
      mask[u] = __ballot_sync(0xffffffffu, p < a.num_pages && __ldcg(a.refs + p) != 0);
      cnt += __popc(mask[u]);
    }
    int total;
    const int before = block_excl_scan(lane == 0 ? cnt : 0, sm, &total);
    int at = found + __shfl_sync(0xffffffffu, before, 0);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int p = w0 + u * 32 + lane;
      if (mask[u] >> lane & 1) {
        const int i = at + __popc(mask[u] & ((1u << lane) - 1));
        const int d = a.list[i];  // i < holes: as many live pages lie behind the bound as free ones before it
        a.copies[3 * i] = p;
        a.copies[3 * i + 1] = d;
        a.copies[3 * i + 2] = a.page;
        a.map[p] = d;
        a.refs[d] = a.refs[p];
        a.refs[p] = 0;
      } else if (p < a.num_pages) {
        a.map[p] = p;  // free: in no table
      }
      at += __popc(mask[u]);
    }
    found += total;
    __syncthreads();
  }
  if (tid == 0) {
    *a.ncopy = holes;
    a.list[0] = live;  // the bound, for the tables
  }
}

// The move: piece by piece of every copied plane. A copy of `rows` rows touches rows * D values of each kv head; a
// whole page is one run of Hkv * page * D values.
struct CopyArgs {
  uint8_t* k;
  uint8_t* v;
  int64_t layer_bytes;
  int32_t layers, Hkv, page, row_bytes, num_pages;
  const int32_t* ncopy;   // count on the device, or null: n
  const int32_t* copies;  // triples, or null: src and dst lists
  const int32_t* src;
  const int32_t* dst;
  int n;
  uint32_t* err;
  // compaction: the tables follow (null otherwise)
  int32_t* tables;
  const int32_t* map;
  const int32_t* bound;
  int64_t entries;
};

constexpr int kCopyThreads = 256;
constexpr int kPiece = kCopyThreads * 16 * 4;  // bytes: four 16-byte words a thread

__global__ void __launch_bounds__(kCopyThreads) plane_copy_kernel(const __grid_constant__ CopyArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int n = a.ncopy ? *a.ncopy : a.n;
  const int tid = threadIdx.x;
  const int64_t head_bytes = (int64_t)a.page * a.row_bytes, page_bytes = a.Hkv * head_bytes;
  // pieces of one plane (page of one layer's k or v): a run per head, each cut into pieces; a whole page is one run
  const int per_page = (int)((page_bytes + kPiece - 1) / kPiece), per_head = (int)((head_bytes + kPiece - 1) / kPiece);
  const bool whole_only = a.copies == nullptr || a.tables != nullptr;
  const int per_plane = whole_only ? per_page : a.Hkv * per_head;
  const int64_t items = (int64_t)n * a.layers * 2 * per_plane;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int piece = (int)(it % per_plane);
    const int64_t rest = it / per_plane;
    const int plane = (int)(rest % (2 * a.layers)), c = (int)(rest / (2 * a.layers));
    const int s = a.copies ? a.copies[3 * c] : a.src[c], d = a.copies ? a.copies[3 * c + 1] : a.dst[c];
    if (s < 0 || s >= a.num_pages || d < 0 || d >= a.num_pages) {
      if (tid == 0) atomicOr(a.err, (uint32_t)MOE_ERR_PAGE_ID);
      continue;
    }
    int64_t off, len;
    if (whole_only) {
      off = (int64_t)piece * kPiece;
      len = page_bytes - off;
    } else {
      const int h = piece / per_head;
      off = (int64_t)(piece % per_head) * kPiece;
      len = (int64_t)a.copies[3 * c + 2] * a.row_bytes - off;
      off += h * head_bytes;
    }
    uint8_t* base = (plane & 1 ? a.v : a.k) + (plane >> 1) * a.layer_bytes;
    const uint4* from = reinterpret_cast<const uint4*>(base + s * page_bytes + off);
    uint4* to = reinterpret_cast<uint4*>(base + d * page_bytes + off);
    const int words = (int)(len < kPiece ? len : kPiece) / 16;  // rows are multiples of 128 bytes
    uint4 w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u * kCopyThreads + tid < words) w[u] = __ldcs(from + u * kCopyThreads + tid);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u * kCopyThreads + tid < words) __stcs(to + u * kCopyThreads + tid, w[u]);
  }
  if (!a.tables || n == 0) return;
  const int bound = *a.bound;
  for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + tid; i < a.entries; i += (int64_t)gridDim.x * kCopyThreads) {
    const int p = a.tables[i];
    if (p >= bound && p < a.num_pages) a.tables[i] = a.map[p];
  }
}

// ------------------------------------------------------------------ the write of new keys and values

struct AppendArgs {
  const uint16_t* qkv;
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  const double* inv_freq;
  uint16_t* q_out;
  uint8_t* k;
  uint8_t* v;
  const float* k_scale;  // of this layer
  const float* v_scale;
  const int32_t* seqs;
  const int32_t* tables;
  const int32_t* refs;
  const int32_t* lens;
  uint32_t* err;
  int32_t B, Tq, Hq, Hkv, page, num_pages, max_seqs, max_pages, rope_dim;
  int32_t per;  // tokens a CTA
  float eps;
};

constexpr int kAppendWarps = 8;
constexpr int kAppendCtas = 4;  // an SM (five, with 48 registers a thread: 22.8 us instead of 18.6 for the prompt below)
constexpr int kAppendMany = 8;  // tokens a CTA at most, where there are many

// Packed pairs of fp32 (sm_100a): two roundings to nearest an instruction.
__device__ __forceinline__ u64 pair(float lo, float hi) {
  return ((u64)__float_as_uint(hi) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ u64 mul2(u64 x, u64 y) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 x, u64 y, u64 z) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}

// A CTA takes up to TT tokens: their positions are looked up and their angles formed once (in fp64: position times frequency,
// in half turns, reduced to [-1, 1] before the fp32 sine and cosine), while the first rows are on their way. A head is
// L = D / 16 lanes of 16 values, the chunks of eight lane and lane + L; a warp takes 32 / L heads of a token at a time
// and fetches the next ones before it works on these. The pairs of the rotation meet by shuffles, in one lane (rope_dim
// = D), or in shared memory where they lie at different places of two lanes. TT = 1 and several CTAs a token where two
// tokens a CTA would be too few for every SM; else every CTA takes the same share, in as few full rounds of the GPU as
// eight tokens a CTA allow (four a CTA and a last round of any size: 8 to 10 % slower). 4095 tokens of 16 + 2 + 2 heads
// of 256 take 18.4 us (4.6 TB/s; about 170 instructions a warp for every two heads bound it, not memory), into e4m3 12 %
// more (the division and the conversion, value by value), 64 tokens 3.1.
template <int D, bool F8, int TT>
__global__ void __launch_bounds__(kAppendWarps * 32, kAppendCtas) append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int L = D / 16, kHeads = 32 / L;
  __shared__ __align__(16) float cs[TT][D / 2], sn[TT][D / 2];
  __shared__ __align__(16) float rows[kAppendWarps][kHeads][D];
  __shared__ int seq_s[TT], pos_s[TT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hl = lane % L, hw = lane / L;
  const int per = TT == 1 ? 1 : a.per, tok0 = blockIdx.x * per, T = a.B * a.Tq, here = min(per, T - tok0);
  const int heads = a.Hq + 2 * a.Hkv, half = a.rope_dim >> 1;
  // this CTA's share of the (token, group of heads) items, token by token, a warp every kAppendWarps-th
  const int groups = (heads + kHeads - 1) / kHeads, items = here * groups;
  const int begin = (int)((int64_t)items * blockIdx.y / gridDim.y);
  const int end = (int)((int64_t)items * (blockIdx.y + 1) / gridDim.y);
  struct Item {
    int k, g, left;  // token, group, items from this one to the end
    __device__ __forceinline__ void on(int groups) {
      left -= kAppendWarps;
      for (g += kAppendWarps; g >= groups; g -= groups) ++k;
    }
  };
  Item cur, ahead;
  ahead.k = (begin + warp) / groups;
  ahead.g = begin + warp - ahead.k * groups;
  ahead.left = end - begin - warp;
  cur = ahead;
  pdl_wait();
  pdl_launch_dependents();
  const uint4* const qkv0 = reinterpret_cast<const uint4*>(a.qkv + (int64_t)tok0 * heads * D) + hl;
  auto fetch = [&](const Item& it, uint4 (&x)[2]) {
    const int h = it.g * kHeads + hw;
    if (it.left > 0 && h < heads) {
      const uint4* src = qkv0 + (it.k * heads + h) * (D / 8);
      x[0] = src[0];
      x[1] = src[L];
    }
  };
  uint4 next[2];
  fetch(ahead, next);
  // the tokens: sequence and position (-1: none, or a fault)
  if (tid < here) {
    const int tok = tok0 + tid, b = tok / a.Tq, t = tok - b * a.Tq;
    int pos = -1;
    const int s = a.seqs[b];
    if (s >= 0 && s < a.max_seqs) {
      const int len = a.lens[s];
      if (len >= 0 && len <= a.max_pages * a.page) pos = max(-1, len - a.Tq + t);
      else atomicOr(a.err, (uint32_t)MOE_ERR_SEQ_ID);
    } else if (s != -1) {
      atomicOr(a.err, (uint32_t)MOE_ERR_SEQ_ID);
    }
    seq_s[tid] = s;
    pos_s[tid] = pos;
  }
  __syncthreads();
  for (int i = tid; i < here * half; i += kAppendWarps * 32) {
    const int k = i / half, d = i - k * half;
    double x = (double)pos_s[k] * a.inv_freq[d] * 0.31830988618379067154;  // 1 / pi
    x -= 2.0 * rint(0.5 * x);
    sincospif((float)x, &sn[k][d], &cs[k][d]);
  }
  __syncthreads();
  const bool by_lane = half == D / 2, by_shuffle = half % 8 == 0 && 4 * half <= D;
  for (; cur.left > 0; cur = ahead) {
    uint4 raw[2] = {next[0], next[1]};
    ahead.on(groups);
    fetch(ahead, next);
    const int k = cur.k, h = cur.g * kHeads + hw, pos = pos_s[k];
    if (pos < 0) continue;  // the same for the whole warp
    const bool there = h < heads, is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    // a key's or value's page (-1: not to be written)
    int page = -1;
    if (there && !is_q) {
      page = a.tables[(int64_t)seq_s[k] * a.max_pages + pos / a.page];
      if (page < 0 || page >= a.num_pages) {
        atomicOr(a.err, (uint32_t)MOE_ERR_PAGE_ID);
        page = -1;
      } else if (a.refs[page] != 1) {
        atomicOr(a.err, (uint32_t)MOE_ERR_SHARED);
        page = -1;
      }
    }
    float v[2][8];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      v[c][0] = lo_bf(raw[c].x); v[c][1] = hi_bf(raw[c].x); v[c][2] = lo_bf(raw[c].y); v[c][3] = hi_bf(raw[c].y);
      v[c][4] = lo_bf(raw[c].z); v[c][5] = hi_bf(raw[c].z); v[c][6] = lo_bf(raw[c].w); v[c][7] = hi_bf(raw[c].w);
    }
    if (a.q_norm) {
      u64 s2 = 0ull;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const u64 x = pair(v[i >> 3][i & 7], v[i >> 3][(i & 7) + 1]);
        s2 = fma2(x, x, s2);
      }
      float ss = lo_f(s2) + hi_f(s2);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (!is_v) {
        const float inv = rsqrtf(ss * (1.f / (float)D) + a.eps);
        const u64 inv2 = pair(inv, inv);
        const uint4* norm = reinterpret_cast<const uint4*>(is_q ? a.q_norm : a.k_norm);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint4 w4 = norm[hl + c * L];
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const u64 x = mul2(mul2(pair(v[c][2 * i], v[c][2 * i + 1]), inv2), pair(lo_bf(w[i]), hi_bf(w[i])));
            v[c][2 * i] = lo_f(x);
            v[c][2 * i + 1] = hi_f(x);
          }
        }
      }
    }
    if (by_lane) {
      if (!is_v) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 c4 = *reinterpret_cast<const float4*>(&cs[k][hl * 8 + i]);
          const float4 s4 = *reinterpret_cast<const float4*>(&sn[k][hl * 8 + i]);
          const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = v[0][i + j], y = v[1][i + j];
            v[0][i + j] = x * cc[j] - y * ss[j];
            v[1][i + j] = y * cc[j] + x * ss[j];
          }
        }
      }
    } else if (by_shuffle && half) {
      const int hc = half / 8;  // the pair's second chunk is hc lanes on
      const bool low = hl < hc, rot = hl < 2 * hc;
      const int from = low ? lane + hc : (rot ? lane - hc : lane), d0 = (low ? hl : hl - hc) * 8;
      float other[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, v[0][i], from);
      if (rot && !is_v) {
        const float sign = low ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 c4 = *reinterpret_cast<const float4*>(&cs[k][d0 + i]);
          const float4 s4 = *reinterpret_cast<const float4*>(&sn[k][d0 + i]);
          v[0][i] = fmaf(v[0][i], c4.x, sign * other[i] * s4.x);
          v[0][i + 1] = fmaf(v[0][i + 1], c4.y, sign * other[i + 1] * s4.y);
          v[0][i + 2] = fmaf(v[0][i + 2], c4.z, sign * other[i + 2] * s4.z);
          v[0][i + 3] = fmaf(v[0][i + 3], c4.w, sign * other[i + 3] * s4.w);
        }
      }
    } else if (half) {
      float* r = rows[warp][hw];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) r[(i >> 3) * (D / 2) + hl * 8 + (i & 7)] = v[i >> 3][i & 7];
      __syncwarp();
      if (!is_v) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int d = (i >> 3) * (D / 2) + hl * 8 + (i & 7);
          float& x = v[i >> 3][i & 7];
          if (d < half) x = x * cs[k][d] - r[d + half] * sn[k][d];
          else if (d < 2 * half) x = x * cs[k][d - half] + r[d - half] * sn[k][d - half];
        }
      }
    }
    if (!there) continue;
    auto two = [](float x, float y) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
      return *reinterpret_cast<const uint32_t*>(&p);
    };
    if (is_q || !F8) {
      if (!is_q && page < 0) continue;
      const int kvh = h - a.Hq - (is_v ? a.Hkv : 0);
      uint16_t* dst = is_q ? a.q_out + ((int64_t)(tok0 + k) * a.Hq + h) * D
                           : reinterpret_cast<uint16_t*>(is_v ? a.v : a.k) +
                                 (((int64_t)page * a.Hkv + kvh) * a.page + pos % a.page) * D;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        reinterpret_cast<uint4*>(dst)[hl + c * L] = make_uint4(two(v[c][0], v[c][1]), two(v[c][2], v[c][3]),
                                                               two(v[c][4], v[c][5]), two(v[c][6], v[c][7]));
    } else if (page >= 0) {
      const int kvh = h - a.Hq - (is_v ? a.Hkv : 0);
      const float* sp = is_v ? a.v_scale : a.k_scale;
      const float sc = sp ? sp[kvh] : 1.f;
      uint8_t* dst = (is_v ? a.v : a.k) + (((int64_t)page * a.Hkv + kvh) * a.page + pos % a.page) * D;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t q[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          q[i] = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            q[i] |= (uint32_t)__nv_cvt_float_to_fp8(__fdiv_rn(v[c][4 * i + j], sc), __NV_SATFINITE, __NV_E4M3)
                    << (8 * j);
        }
        reinterpret_cast<uint2*>(dst)[hl + c * L] = make_uint2(q[0], q[1]);
      }
    }
  }
}

template <int D, bool F8>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t s) {
  AppendArgs arg = a;
  void* args[] = {&arg};
  const int T = a.B * a.Tq, per_token = (a.Hq + 2 * a.Hkv + 512 / D - 1) / (512 / D);
  // whole rounds of the CTAs that the GPU holds at once, with equal shares
  const int slots = paged_sms() * kAppendCtas, rounds = (T + slots * kAppendMany - 1) / (slots * kAppendMany);
  const bool many = T > slots * 2;
  arg.per = many ? (T + slots * rounds - 1) / (slots * rounds) : 1;
  const void* fn = many ? reinterpret_cast<const void*>(append_kernel<D, F8, kAppendMany>)
                        : reinterpret_cast<const void*>(append_kernel<D, F8, 1>);
  const dim3 grid((T + arg.per - 1) / arg.per, many ? 1 : (per_token + kAppendWarps - 1) / kAppendWarps);
  return paged_launch(fn, grid, dim3(kAppendWarps * 32), 0, s, args);
}

PageArgs page_args(const moe_paged_cache* c, const int32_t* x, const int32_t* y, int n, void* workspace,
                   const PagedWs& L) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PageArgs a;
  a.tables = c->tables;
  a.refs = c->refs;
  a.lens = c->lens;
  a.num_pages = c->num_pages;
  a.page = c->page;
  a.max_seqs = c->max_seqs;
  a.max_pages = c->max_pages;
  a.a = x;
  a.b = y;
  a.n = n;
  a.err = reinterpret_cast<uint32_t*>(ws + L.err);
  a.ncopy = reinterpret_cast<int32_t*>(ws + L.ncopy);
  a.copies = reinterpret_cast<int32_t*>(ws + L.copies);
  a.list = reinterpret_cast<int32_t*>(ws + L.list);
  a.map = reinterpret_cast<int32_t*>(ws + L.map);
  return a;
}

// The workspace a call with lists of n entries needs is there and aligned.
bool ws_ok(const moe_paged_cache* c, int n, void* workspace, size_t bytes, PagedWs* L) {
  if (!paged_ok(c) || !workspace || !paged_al16(workspace)) return false;
  *L = paged_ws(c, c->Hkv, n < 1 ? 1 : n, 1);
  return bytes >= L->total;
}

// The move of a plan (counted on the device; with the tables for a compaction), or of the caller's lists.
CopyArgs copy_args(const moe_paged_cache* c, const PageArgs& p, bool planned, bool tables) {
  CopyArgs a;
  memset(&a, 0, sizeof a);
  a.k = static_cast<uint8_t*>(c->k);
  a.v = static_cast<uint8_t*>(c->v);
  a.layer_bytes = paged_layer_bytes(c);
  a.layers = c->layers;
  a.Hkv = c->Hkv;
  a.page = c->page;
  a.row_bytes = c->D * kv_size(c->kv_type);
  a.num_pages = c->num_pages;
  a.err = p.err;
  if (planned) {
    a.ncopy = p.ncopy;
    a.copies = p.copies;
  } else {
    a.src = p.a;
    a.dst = p.b;
    a.n = p.n;
  }
  if (tables) {
    a.tables = c->tables;
    a.map = p.map;
    a.bound = p.list;
    a.entries = (int64_t)c->max_seqs * c->max_pages;
  }
  return a;
}

cudaError_t launch_copy(const CopyArgs& args, cudaStream_t s) {
  CopyArgs a = args;
  void* p[] = {&a};
  return paged_launch(reinterpret_cast<const void*>(plane_copy_kernel), dim3(paged_sms() * 4), dim3(kCopyThreads), 0, s,
                      p);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_paged_check(const moe_paged_cache* c) { return paged_ok(c) ? (int)cudaSuccess : (int)cudaErrorInvalidValue; }

size_t moe_paged_workspace_bytes(const moe_paged_cache* c, int Hq, int max_batch, int max_new) {
  if (!paged_shape_ok(c) || Hq < 1 || Hq > 128 || Hq % c->Hkv != 0 || max_batch < 1 || max_batch > kPagedMaxBatch ||
      max_new < 1)
    return 0;
  return paged_ws(c, Hq, max_batch, max_new).total;
}

int moe_paged_workspace_error(void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  return moe_attn_workspace_error(workspace, workspace_bytes, stream);  // the error word leads both layouts
}

int moe_paged_resize(const moe_paged_cache* c, const int32_t* seqs, const int32_t* new_lens, int n, void* workspace,
                     size_t workspace_bytes, moe_stream_t stream) {
  PagedWs L;
  if (n < 0 || n > kPagedMaxBatch || !ws_ok(c, n, workspace, workspace_bytes, &L)) return (int)cudaErrorInvalidValue;
  if (n == 0) return (int)cudaSuccess;
  if (!seqs || !new_lens) return (int)cudaErrorInvalidValue;
  PageArgs a = page_args(c, seqs, new_lens, n, workspace, L);
  const size_t smem = (size_t)n * 5 * 4 + ((size_t)c->max_seqs + 31) / 32 * 4;
  static SmemGrant granted;
  cudaError_t e = grant_smem(reinterpret_cast<const void*>(resize_plan_kernel), smem, 64 * 1024, granted);
  if (e != cudaSuccess) return (int)e;
  void* args[] = {&a};
  e = paged_launch(reinterpret_cast<const void*>(resize_plan_kernel), dim3(1), dim3(kPlanThreads), smem,
                   (cudaStream_t)stream, args);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_copy(copy_args(c, a, true, false), (cudaStream_t)stream);
}

int moe_paged_fork(const moe_paged_cache* c, const int32_t* src, const int32_t* dst, int n, void* workspace,
                   size_t workspace_bytes, moe_stream_t stream) {
  PagedWs L;
  if (n < 0 || n > kPagedMaxBatch || !ws_ok(c, n, workspace, workspace_bytes, &L)) return (int)cudaErrorInvalidValue;
  if (n == 0) return (int)cudaSuccess;
  if (!src || !dst) return (int)cudaErrorInvalidValue;
  PageArgs a = page_args(c, src, dst, n, workspace, L);
  void* args[] = {&a};
  return (int)paged_launch(reinterpret_cast<const void*>(fork_kernel), dim3(kForkCluster), dim3(kPlanThreads),
                           ((size_t)c->max_seqs + 31) / 32 * 4, (cudaStream_t)stream, args, kForkCluster);
}

int moe_paged_compact(const moe_paged_cache* c, void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  PagedWs L;
  if (!ws_ok(c, 1, workspace, workspace_bytes, &L)) return (int)cudaErrorInvalidValue;
  PageArgs a = page_args(c, nullptr, nullptr, 0, workspace, L);
  void* args[] = {&a};
  cudaError_t e = paged_launch(reinterpret_cast<const void*>(compact_plan_kernel), dim3(1), dim3(kPlanThreads), 0,
                               (cudaStream_t)stream, args);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_copy(copy_args(c, a, true, true), (cudaStream_t)stream);
}

int moe_paged_copy(const moe_paged_cache* c, const int32_t* src, const int32_t* dst, int n, void* workspace,
                   size_t workspace_bytes, moe_stream_t stream) {
  PagedWs L;
  if (n < 0 || !ws_ok(c, 1, workspace, workspace_bytes, &L)) return (int)cudaErrorInvalidValue;
  if (n == 0) return (int)cudaSuccess;
  if (!src || !dst) return (int)cudaErrorInvalidValue;
  return (int)launch_copy(copy_args(c, page_args(c, src, dst, n, workspace, L), false, false), (cudaStream_t)stream);
}

int moe_paged_append(const moe_paged_cache* c, int layer, const int32_t* seqs, int B, int Tq, const uint16_t* qkv,
                     int Hq, const uint16_t* q_norm, const uint16_t* k_norm, const double* inv_freq, int rope_dim,
                     float eps, uint16_t* q_out, void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  PagedWs L;
  if (B < 0 || B > kPagedMaxBatch || Tq < 1 || (int64_t)B * Tq >= (1 << 24) ||
      !ws_ok(c, B, workspace, workspace_bytes, &L) || layer < 0 || layer >= c->layers || Hq < 1 || Hq > 128 ||
      Hq % c->Hkv != 0 || rope_dim < 0 || rope_dim > c->D || rope_dim % 2 != 0)
    return (int)cudaErrorInvalidValue;
  if (B == 0) return (int)cudaSuccess;
  if (!seqs || !qkv || !q_out || !paged_al16(qkv) || !paged_al16(q_out) || !paged_al16(q_norm) ||
      !paged_al16(k_norm) || (q_norm == nullptr) != (k_norm == nullptr) || (rope_dim > 0) != (inv_freq != nullptr))
    return (int)cudaErrorInvalidValue;
  const int64_t off = layer * paged_layer_bytes(c);
  AppendArgs a;
  a.qkv = qkv;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.inv_freq = inv_freq;
  a.q_out = q_out;
  a.k = static_cast<uint8_t*>(c->k) + off;
  a.v = static_cast<uint8_t*>(c->v) + off;
  a.k_scale = c->k_scale ? c->k_scale + (int64_t)layer * c->Hkv : nullptr;
  a.v_scale = c->v_scale ? c->v_scale + (int64_t)layer * c->Hkv : nullptr;
  a.seqs = seqs;
  a.tables = c->tables;
  a.refs = c->refs;
  a.lens = c->lens;
  a.err = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + L.err);
  a.B = B;
  a.Tq = Tq;
  a.Hq = Hq;
  a.Hkv = c->Hkv;
  a.page = c->page;
  a.num_pages = c->num_pages;
  a.max_seqs = c->max_seqs;
  a.max_pages = c->max_pages;
  a.rope_dim = rope_dim;
  a.per = 1;
  a.eps = eps;
  const cudaStream_t s = (cudaStream_t)stream;
  if (c->kv_type == MOE_KV_E4M3)
    return (int)(c->D == 256 ? launch_append<256, true>(a, s) : launch_append<128, true>(a, s));
  if (c->D == 256) return (int)launch_append<256, false>(a, s);
  return (int)(c->D == 128 ? launch_append<128, false>(a, s) : launch_append<64, false>(a, s));
}

}  // extern "C"
