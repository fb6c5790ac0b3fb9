// moe_paged_attn.cu -- attention of a batch's new tokens over a paged key-value cache (moe_paged_attend,
// include/moe_paged.h).
//
// o = sum_j softmax_j(scale q . k_j) v_j for the G = Hq / Hkv query heads and Tq new tokens that share a kv head: each
// cached value is read once and used by G Tq rows, so up to 64 rows the call is bound by the cache's bytes.
//
// Work split: a unit is NG x KT keys of one (sequence, kv head, row block) job, and a job costs a few units more. Every
// CTA of a persistent grid counts the batch's units itself (a scan over the lengths, which only the device knows) and
// takes an equal, contiguous share of the flattened list, whatever the lengths: a long cache is split over many CTAs,
// many short ones share a CTA. A CTA has partial results for its first and its last job at most; they go to the workspace
// as (max, sum, accumulator), and paged_join_kernel merges each split job's parts in CTA order, so the result does not
// depend on timing. A job that lies in one CTA is finished there. A job of n parts holds n - 1 of the borders between
// CTAs: the join runs a CTA a border, and those of one job share its rows. (Joined by the same launch behind a barrier
// over the grid, a call took 3 us less of the host but 2 us more of the GPU: a cooperative launch does not overlap the
// kernel before it.)
//
// CTA: four or eight consumer warps and four producer warps (a thread issues a TMA copy every 95 cycles or so: one an SM
// fetches 3.2 TB/s over the GPU in 2 KB boxes, four 6.4 TB/s). Producer w takes every NP-th of the CTA's tiles (KT keys of
// k and v each), looks up their pages eight tiles ahead and fetches them by TMA (boxes of 128 bytes x 16 or KT rows inside
// one page, 128-byte swizzle) into a ring of NS slots, mbarrier-counted. Consumer warp (g, mt) holds 16 query rows as MMA
// fragments and takes every NG-th tile: S = Q K^T, the running maximum and sum of the softmax, O += P V, all in
// registers; at a job's end the NG warps of a row tile merge through shared memory.
//
// mma.sync and not tcgen05: at 16 rows the register MMA needs under a half of the cycles that a tile's bytes take to
// arrive, so a tcgen05.mma (at least 64 rows of the cache as M, and P through TMEM) would only add two TMEM round trips to
// the softmax of each tile. At 64 rows that no longer holds: there the register MMAs bound the call.
//
// Measured on a B200 (16 query and 2 kv heads of 256, bf16, unless said otherwise; the device copy moves 6.45 TB/s): one
// sequence of 131071 keys 51 us (5.3 TB/s), 48 ragged sequences of up to 8192 keys 69 us (5.4 TB/s), with 4 and 8 new
// tokens each 83 and 147 us, over e4m3 49, 81 and 143 us; 24 sequences of up to 16000 keys, 32 over 8 heads of 128, 4
// tokens, pages of 16: 124 us in bf16 (5.8 TB/s), 70 us in e4m3 (5.1 TB/s). The batch's tables take room from the ring: 8
// over 2 heads of 128, 260000 keys in all, 52 us for 256 sequences (12 slots), 71 for 1024 (8 slots, and jobs of
// 256 keys on average), 184 for 4096 (4 slots, jobs of 64 keys). The loop over the tiles runs at the read bandwidth for
// bf16 and one row tile; around it lie 2 us for the units, 1.5 us for the first queries and pages, 2 us for the last merge, 1 to
// 4 us for the slowest CTA and 3 us for the join. With e4m3 the consumers' latency a tile (2000 cycles, two warps a
// scheduler) bounds it, with four row tiles their products, and the k and v fragments that every row tile loads again.
#include <algorithm>
#include <cstring>
#include <mutex>

#include <cuda.h>
#include <cuda_fp8.h>

#include "moe_paged.h"
#include "moe_sync.cuh"

namespace moe {
namespace {

constexpr int kSmemOne = 226 * 1024;           // dynamic shared memory of a CTA alone on its SM
constexpr int kSmemTwo = 112 * 1024;           // of one of two

struct PAttnArgs {
  const uint16_t* q;
  uint16_t* out;
  const float* k_scale;  // of this layer, or null
  const float* v_scale;
  const int32_t* seqs;
  const int32_t* tables;
  const int32_t* lens;
  int32_t* joins;  // [ctas][JOIN_INTS]: the split job at the border before each CTA
  float* ml;       // [2 ctas][rows][2]
  float* acc;      // [2 ctas][rows][D]
  uint32_t* err;
  int32_t B, Tq, Hq, Hkv, G, page, num_pages, max_seqs, max_pages, box_rows, row_blocks, rows, ctas, ns;
  float scale, inv_G;
};

// The token of row r of a kv head, r / G for r < 2^12 and G <= 128: half a row off, the product stays clear of the next
// whole number by 0.5 / G, far more than its rounding.
__device__ __forceinline__ int token_of(const PAttnArgs& a, int r) { return __float2int_rd(((float)r + 0.5f) * a.inv_G); }

// Three shapes of a CTA. Heads of 64 and 128: two CTAs an SM, four consumer warps each. Heads of 256, one row tile of
// bf16: one CTA an SM, four consumer warps with queries and accumulator in 255 registers, which keep up with memory.
// Heads of 256 otherwise ("wide"): the conversion of e4m3 or the second to fourth row tile doubles to quadruples the
// work a byte, so eight consumer warps, which share the queries in shared memory.
template <int D, bool F8, int MT>
struct Cfg {
  static constexpr int kEs = F8 ? 1 : 2;
  static constexpr int kRow = D * kEs;                    // bytes of a cached row
  static constexpr int kSegs = kRow / 128;                // 128-byte column segments of a tile
  static constexpr int KT = kRow <= 128 ? 32 : 16;        // keys of a tile
  static constexpr int kSeg = KT * 128;                   // bytes of a segment
  static constexpr int kTile = KT * kRow;                 // bytes of a k or v tile
  static constexpr int kSlot = 2 * kTile;                 // 8 KB, or 16 KB for rows of 512 bytes
  static constexpr int kPerSm = D == 256 ? 1 : 2;         // CTAs an SM: registers (accumulator D / 2 a lane)
  static constexpr bool kWide = D == 256 && (F8 || MT > 1);
  static constexpr int kWarps = kWide ? 8 : 4;            // consumer warps
  static constexpr int NG = kWarps / MT;                  // key groups
  static constexpr int NP = 4;                            // producer warps
  static constexpr int kThreads = (kWarps + NP) * 32;
  // But for the narrow CTA alone, the producers hand most of a launch's registers to the consumers.
  static constexpr bool kHandOver = kPerSm == 2 || kWide;
  static constexpr int kConsumerRegs = kWide ? 232 : 216, kProducerRegs = 40;
  static_assert(!kHandOver || (kWarps * kConsumerRegs + NP * kProducerRegs) * 32 <=
                                  65536 / kPerSm / kThreads / 8 * 8 * kThreads, "registers of a launch");
  static constexpr int kQueries = kWide ? MT * (D / 16 * 512 + 64) : 0;  // bytes: fragments and row factors
  static constexpr int kMergeCols = D == 256 && !kWide ? 64 : 32;   // columns that meet at a time at a job's end
  static constexpr int kMergeRow = kMergeCols + 4;        // floats of a row in the merge buffer, padded
  static constexpr int kMerge = kWarps * 16 * (kMergeRow + 2) * 4;  // every warp's columns; maxima and sums
  static constexpr int kMaxNS = 24;
  // Ring slots for a batch of B: what shared memory leaves beside the merge buffer and three ints a slot of the batch.
  // At least three a key group keep two tiles on their way while one is worked on (two: 15 % less of the bandwidth).
  // A multiple of the producers and of the key groups, so that a ring slot is always filled by one producer and read by
  // one group: barrier waits tell phases apart by parity alone, and two producers on one slot could be two turns apart.
  static constexpr int fixed_bytes(int B) { return 2048 + kMerge + kQueries + (3 * B + 1) * 4; }
  static constexpr int slots(int B) {
    const int fit = ((kPerSm == 1 ? kSmemOne : kSmemTwo) - fixed_bytes(B)) / kSlot;
    constexpr int kMul = NG > NP ? NG : NP;
    return (fit > kMaxNS ? kMaxNS : fit) / kMul * kMul;
  }
  static_assert(NG >= 1 && (NG % NP == 0 || NP % NG == 0), "a ring slot has one producer and one group");
};

// D (16x8, fp32) += A (16x16) B (16x8); bf16 or f16 operands.
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Four e4m3 values as f16 pairs (bytes 0 and 1, 2 and 3), exactly.
__device__ __forceinline__ void e4m3x4_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* mbar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(mbar))
      : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* mbar) {
  asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(smem_u32(mbar)) : "memory");
}
template <int kT>
__device__ __forceinline__ void consumers_bar() {
  asm volatile("bar.sync 1, %0;" ::"n"(kT) : "memory");
}

// Whether one of the values in w (two bf16, or four e4m3) is NaN or infinite.
template <bool F8>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  if constexpr (F8) return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;  // e4m3 has no infinity
  else return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// Keys of slot b: its sequence's length, 0 for an unused slot or a bad entry (recorded).
__device__ __forceinline__ int slot_keys(const PAttnArgs& a, int b, int* seq) {
  const int own = b < a.max_seqs ? a.lens[b] : 0;  // slot b is often sequence b: its length is asked for at once
  const int s = a.seqs[b];
  *seq = 0;
  if (s == -1) return 0;
  if (s < 0 || s >= a.max_seqs) {
    atomicOr(a.err, (uint32_t)MOE_ERR_SEQ_ID);
    return 0;
  }
  *seq = s;
  const int n = s == b ? own : a.lens[s];
  if (n < 0 || n > a.max_pages * a.page) {
    atomicOr(a.err, (uint32_t)MOE_ERR_SEQ_ID);
    return 0;
  }
  return n;
}

// The split job at the border before a CTA: its parts (0: none), its first CTA, whether its part is that CTA's second,
// slot, kv head and row block.
enum { JOIN_PARTS = 0, JOIN_FIRST, JOIN_SECOND, JOIN_SLOT, JOIN_HEAD, JOIN_BLOCK, JOIN_INTS = 8 };

// The share of one CTA: [u, end) of the flattened list, walked job by job. A job counts kSetup units of its own before
// its units of keys: its queries, its first tile's latency and its merge cost a CTA about as much, and a batch with
// many short sequences would otherwise pile them up in a few CTAs. (setup_units, moe_paged.h)
template <int kSetup>
struct Walk {
  int u, end;           // what is left of the share
  int b, job, W;        // the slot, its job (kv head and row block), units of each of its jobs
  int base;             // first unit of the slot
  int lu, run;          // units of keys of the job that are this CTA's: [lu, lu + run)
  // The next job of the share that has keys here; false at the end.
  __device__ __forceinline__ bool next(const int* S, int B, int HR) {
    while (u < end) {
      seek(S, B, HR);
      const int at = u - base - job * W, n = min(end - u, W - at);
      lu = max(0, at - kSetup);
      run = max(0, at + n - kSetup) - lu;
      u += n;
      if (run > 0) return true;
    }
    return false;
  }
  __device__ __forceinline__ void seek(const int* S, int B, int HR) {
    int lo = 0, hi = B - 1;  // the last slot whose first unit is not behind u; empty slots before it are passed
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (S[mid] * HR <= u) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    base = S[b] * HR;
    W = S[b + 1] - S[b];
    job = (u - base) / W;
  }
};

template <int D, bool F8, int MT>
__global__ void __launch_bounds__(Cfg<D, F8, MT>::kThreads, Cfg<D, F8, MT>::kPerSm)
    paged_attn_kernel(const __grid_constant__ PAttnArgs a, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v) {
  using C = Cfg<D, F8, MT>;
  constexpr int kWarps = C::kWarps, NG = C::NG, KT = C::KT, UK = NG * KT, NP = C::NP, kThreads = C::kThreads;
  constexpr int kSetup = setup_units(UK);
  auto consumers_sync = [] { consumers_bar<kWarps * 32>(); };
  const int NS = a.ns;
  constexpr int NT = D / 8;     // accumulator tiles of 8 columns
  constexpr int KC = C::kRow / 16;  // 16-byte chunks of a cached row
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[C::kMaxNS], empty[C::kMaxNS];
  __shared__ int sm[32];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* merge = reinterpret_cast<float*>(ring + (size_t)NS * C::kSlot);
  float2* merge_ml = reinterpret_cast<float2*>(merge + kWarps * 16 * C::kMergeRow);
  uint4* q_sm = reinterpret_cast<uint4*>(merge_ml + kWarps * 16);  // wide: [row tile][k step][lane], row factors behind
  float* q_fac = reinterpret_cast<float*>(q_sm + MT * (D / 16) * 32);
  int* S = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(q_sm) + C::kQueries);
  int* keys = S + a.B + 1;
  int* seqs = keys + a.B;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], MT);
    }
    mbar_fence_init();
  }
  if (warp == kWarps && lane < 2)
    asm volatile("prefetch.tensormap [%0];" ::"l"(lane ? &map_v : &map_k) : "memory");
  pdl_wait();
  pdl_launch_dependents();
  // units of the slots before each slot
  {
    const int per = (a.B + kThreads - 1) / kThreads, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
      const int n = slot_keys(a, b, &seqs[b]);
      keys[b] = n;
      S[b] = sum;
      sum += n > 0 ? (n + UK - 1) / UK + kSetup : 0;
    }
    int total;
    const int before = block_excl_scan(sum, sm, &total);
    for (int b = b0; b < b1; ++b) S[b] += before;
    if (tid == 0) S[a.B] = total;
  }
  __syncthreads();
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {  // no keys: zero rows
    if (S[b + 1] != S[b]) continue;
    uint4* o = reinterpret_cast<uint4*>(a.out + (int64_t)b * a.Tq * a.Hq * D);
    for (int i = tid; i < a.Tq * a.Hq * (D / 8); i += kThreads) o[i] = make_uint4(0, 0, 0, 0);
  }
  const int HR = a.Hkv * a.row_blocks, total = S[a.B] * HR;
  const int per = max(1, (total + a.ctas - 1) / a.ctas);
  Walk<kSetup> w;
  w.u = min(total, (int)blockIdx.x * per);
  w.end = min(total, w.u + per);
  if (warp >= kWarps) {
    // ---------------------------------------------------------------- producer
    if constexpr (C::kHandOver) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kProducerRegs));
    const int none = a.num_pages * a.Hkv;  // a page that is not there: outside the map, reads as zero
    const int nbox = KT / a.box_rows;      // 1 or 2
    const int own = warp - kWarps;
    int slot = own, turn = 0;              // of this warp's next tile, the slot for the turn-th time
    int next = own, before = 0;            // that tile's number; tiles of the jobs so far
    bool ok = true;
    while (ok && w.next(S, a.B, HR)) {
      const int lu = w.lu, run = w.run, h = w.job / a.row_blocks;
      const int n = keys[w.b];
      const int32_t* row = a.tables + (int64_t)seqs[w.b] * a.max_pages;
      const int key_end = (lu + run) * UK;
      // Pages of this warp's next eight tiles, a lane a box, and the lane of the next box. (32 at a time: 52.3 us for one
      // sequence of 131071 keys, 8: 51.8.)
      int z = 0, y = 0, at = 8 * nbox;
      for (; next < before + run * NG; next += NP) {
        const int key = lu * UK + (next - before) * KT;
        if (turn > 0) {
          ok = bar_wait(&empty[slot], (turn - 1) & 1);
          if (!ok) {
            if (lane == 0) atomicOr(a.err, (uint32_t)MOE_ERR_TIMEOUT);
            break;
          }
        }
        if (key >= n) {  // a unit's tile behind the sequence's end
          if (lane == 0) mbar_arrive(&full[slot]);
        } else {
          if (at == 8 * nbox) {
            at = 0;
            const int k = key + (nbox == 2 ? (lane >> 1) * NP * KT + (lane & 1) * a.box_rows : lane * NP * KT);
            z = none;
            y = 0;
            if (lane < 8 * nbox && k < n && k < key_end) {
              const int pid = row[k / a.page];
              if (pid >= 0 && pid < a.num_pages) z = pid * a.Hkv + h;
              else atomicOr(a.err, (uint32_t)MOE_ERR_PAGE_ID);
              y = k % a.page;
            }
          }
          const int boxes = min(nbox, (n - key + a.box_rows - 1) / a.box_rows);
          uint8_t* dst = ring + (size_t)slot * C::kSlot;
          if (lane == 0) expect_tx(&full[slot], (uint32_t)(2 * boxes * a.box_rows * C::kRow));
          __syncwarp();
          for (int x = 0; x < boxes; ++x) {
            const int bz = __shfl_sync(0xffffffffu, z, at + x), by = __shfl_sync(0xffffffffu, y, at + x);
            // one lane issues every copy: the operands of a TMA instruction are uniform, lanes would take turns
            if (lane == 0) {
#pragma unroll
              for (int sg = 0; sg < C::kSegs; ++sg) {
                uint8_t* to = dst + sg * C::kSeg + x * a.box_rows * 128;
                tma_load_3d(to, &map_k, sg * (128 / C::kEs), by, bz, &full[slot]);
                tma_load_3d(to + C::kTile, &map_v, sg * (128 / C::kEs), by, bz, &full[slot]);
              }
            }
          }
          __syncwarp();
          at += nbox;
        }
        if ((slot += NP) >= NS) {
          slot = own;
          ++turn;
        }
      }
      before += run * NG;
    }
    if (!ok)  // no copy may still be landing when the CTA exits: this warp's last tiles
      for (int k = own; k < NS; k += NP) {
        const int t = k < slot ? turn : turn - 1;  // the slot's last turn
        if (t >= 0) bar_wait(&full[k], t & 1);
      }
    return;
  }

  // ------------------------------------------------------------------ consumers
  if constexpr (C::kHandOver) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kConsumerRegs));
  // The split job at the border before this CTA, for the join; off the others' way while the first tile travels.
  if (tid == 64) {
    int4 j0 = make_int4(0, 0, 0, 0);
    Walk<kSetup> at = w;
    if (at.u < at.end) {
      at.seek(S, a.B, HR);
      const int u0 = at.base + at.job * at.W + kSetup;  // the job's first unit of keys
      if (u0 < at.u) {
        const int c0 = u0 / per;
        // its part in CTA c0 is that CTA's second if another job's units lie before it there
        j0 = make_int4((u0 - kSetup + at.W - 1) / per - c0 + 1, c0, u0 - kSetup > c0 * per, at.b);
        *reinterpret_cast<int2*>(a.joins + blockIdx.x * JOIN_INTS + 4) =
            make_int2(at.job / a.row_blocks, at.job % a.row_blocks);
      }
    }
    *reinterpret_cast<int4*>(a.joins + blockIdx.x * JOIN_INTS) = j0;
  }

  const int g = warp / MT, mt = warp % MT, qr = lane >> 2, ql = lane & 3;
  const uint32_t ring32 = smem_u32(ring);
  // this lane's row of an ldmatrix: k takes the four 8x8 blocks (keys 0-7, chunk c), (0-7, c+1), (8-15, c), (8-15, c+1);
  // v, transposed, (0-7, c), (8-15, c), (0-7, c+1), (8-15, c+1)
  const int kk_row = (lane >> 4) * 8 + (lane & 7), kk_ch = (lane >> 3) & 1;
  const int vv_row = ((lane >> 3) & 1) * 8 + (lane & 7), vv_ch = lane >> 4;
  // Offset of chunk pair 0 in a tile, swizzled; pair i of the four in a 128-byte segment is the same with bits 5-6
  // flipped by i, row group j (16 keys) 2048 bytes further on
  const uint32_t k_lane = kk_row * 128 + ((kk_ch ^ (kk_row & 7)) << 4);
  const uint32_t v_lane = vv_row * 128 + ((vv_ch ^ (vv_row & 7)) << 4);
  auto chunk_addr = [&](const uint32_t (&base)[4], int j, int c) {
    return base[(c >> 1) & 3] + (c >> 3) * C::kSeg + j * 2048;
  };
  int slot = g, turn = 0;  // of this group's next tile
  int njob = 0;
  bool ok = true;
  while (w.next(S, a.B, HR)) {
    const int lu = w.lu, run = w.run, h = w.job / a.row_blocks, rb = w.job - h * a.row_blocks;
    const int n = keys[w.b];
    const bool whole = run == w.W - kSetup;
    // this lane's two rows: query row r of the kv head is token r / G, head h G + r % G
    const int rA = rb * a.rows + mt * 16 + qr, rB = rA + 8, M = a.G * a.Tq;
    const int tA = token_of(a, rA), tB = token_of(a, rB);
    const int limA = rA < M ? n - a.Tq + tA + 1 : 0, limB = rB < M ? n - a.Tq + tB + 1 : 0;  // keys the row sees
    auto q_row = [&](int r, int t) {
      return a.q + (((int64_t)w.b * a.Tq + t) * a.Hq + h * a.G + (r - t * a.G)) * D;
    };
    // scores in units of log 2 are S times fA or fB, kept above zero (a masked score is -infinity times it): a negative
    // scale turns the queries' signs, and one of zero is as good as the smallest factor; a NaN stays one
    auto above_zero = [](float f) { return f < 1.1754944e-38f ? 1.1754944e-38f : f; };
    float fA = a.scale * 1.4426950408889634f, fB;
    if (a.k_scale) fA *= a.k_scale[h];
    const uint32_t flip = fA < 0.f ? 0x80008000u : 0u;
    fA = fB = above_zero(fabsf(fA));
    uint32_t qf[C::kWide ? 1 : D / 16][4];
    auto load_queries = [&](uint32_t (&q)[D / 16][4]) {
      const uint16_t* pA = q_row(rA < M ? rA : 0, rA < M ? tA : 0);
      const uint16_t* pB = q_row(rB < M ? rB : 0, rB < M ? tB : 0);
      if constexpr (!F8) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          q[c][0] = *reinterpret_cast<const uint32_t*>(pA + c * 16 + 2 * ql) ^ flip;
          q[c][1] = *reinterpret_cast<const uint32_t*>(pB + c * 16 + 2 * ql) ^ flip;
          q[c][2] = *reinterpret_cast<const uint32_t*>(pA + c * 16 + 8 + 2 * ql) ^ flip;
          q[c][3] = *reinterpret_cast<const uint32_t*>(pB + c * 16 + 8 + 2 * ql) ^ flip;
        }
      } else {
        // e4m3 keys become f16, so the queries do too: scaled by the power of two that brings the row's largest into
        // [1, 2) (exact), what then falls below f16's range is under 2^-24 of it. A 16-byte chunk of a key is one
        // k-step here: lane ql holds its values 4 ql .. + 3, and the queries are laid out to match.
        float xA = 0.f, xB = 0.f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const uint2 va = *reinterpret_cast<const uint2*>(pA + c * 16 + 4 * ql);
          const uint2 vb = *reinterpret_cast<const uint2*>(pB + c * 16 + 4 * ql);
          q[c][0] = va.x ^ flip; q[c][2] = va.y ^ flip; q[c][1] = vb.x ^ flip; q[c][3] = vb.y ^ flip;
          xA = fmaxf(fmaxf(xA, fmaxf(fabsf(lo_bf(va.x)), fabsf(hi_bf(va.x)))), fmaxf(fabsf(lo_bf(va.y)), fabsf(hi_bf(va.y))));
          xB = fmaxf(fmaxf(xB, fmaxf(fabsf(lo_bf(vb.x)), fabsf(hi_bf(vb.x)))), fmaxf(fabsf(lo_bf(vb.y)), fabsf(hi_bf(vb.y))));
        }
        // exponents in [1, 252], so that the factor and its inverse are normal numbers
        const uint32_t eA = min(max(__float_as_uint(quad_max(xA)) >> 23, 1u), 252u);
        const uint32_t eB = min(max(__float_as_uint(quad_max(xB)) >> 23, 1u), 252u);
        const float iA = __uint_as_float((254u - eA) << 23), iB = __uint_as_float((254u - eB) << 23);
        fA = above_zero(fA * __uint_as_float(eA << 23));  // the product may be too small for a number
        fB = above_zero(fB * __uint_as_float(eB << 23));
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          q[c][0] = pack2<true>(lo_bf(q[c][0]) * iA, hi_bf(q[c][0]) * iA);
          q[c][2] = pack2<true>(lo_bf(q[c][2]) * iA, hi_bf(q[c][2]) * iA);
          q[c][1] = pack2<true>(lo_bf(q[c][1]) * iB, hi_bf(q[c][1]) * iB);
          q[c][3] = pack2<true>(lo_bf(q[c][3]) * iB, hi_bf(q[c][3]) * iB);
        }
      }
    };
    if constexpr (!C::kWide) {
      load_queries(qf);
    } else {  // the first group's warps share theirs (all are behind the last job's use of the buffer: its merge)
      if (g == 0) {
        uint32_t q[D / 16][4];
        load_queries(q);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) q_sm[(mt * (D / 16) + c) * 32 + lane] = make_uint4(q[c][0], q[c][1], q[c][2], q[c][3]);
        if (ql == 0) {
          q_fac[mt * 16 + qr] = fA;
          q_fac[mt * 16 + qr + 8] = fB;
        }
      }
      consumers_sync();
      fA = q_fac[mt * 16 + qr];
      fB = q_fac[mt * 16 + qr + 8];
    }
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    float lsum[4] = {0.f, 0.f, 0.f, 0.f};  // the weights' sums, as one more accumulator tile: P times a column of ones
    constexpr uint32_t kOnes = F8 ? 0x3c003c00u : 0x3f803f80u;
    float mA = -INFINITY, mB = -INFINITY;  // the maxima of S

    for (int r = 0; r < run; ++r) {
      const int key0 = (lu + r) * UK + g * KT;
      if (ok && !bar_wait(&full[slot], turn & 1)) {
        ok = false;
        if (lane == 0) atomicOr(a.err, (uint32_t)MOE_ERR_TIMEOUT);
      }
      if (ok && key0 < n) {
        const uint32_t kt = ring32 + slot * C::kSlot, vt = kt + C::kTile;
        const uint32_t k0 = kt + k_lane, v0 = vt + v_lane;
        const uint32_t kb[4] = {k0, k0 ^ 32, k0 ^ 64, k0 ^ 96}, vb[4] = {v0, v0 ^ 32, v0 ^ 64, v0 ^ 96};
        // S = Q K^T. Two chains of accumulators per 8 keys where a tile's 16 keys alone give too few to hide an MMA's
        // latency (21 cycles against 8 of issue)
        constexpr int kChains = KT == 16 ? 2 : 1;
        float s[KT / 8][4], s2[kChains == 2 ? KT / 8 : 1][4];
#pragma unroll
        for (int j = 0; j < KT / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[j][e] = 0.f;
            if constexpr (kChains == 2) s2[j][e] = 0.f;
          }
        auto other = [&](int j) -> float(&)[4] {
          if constexpr (kChains == 2) return s2[j];
          else return s[j];
        };
#pragma unroll
        for (int c = 0; c < KC; c += 2) {
          // the queries of k step k: in registers, or the row tile's in shared memory
          auto query = [&](int k, uint32_t (&q)[4]) {
            if constexpr (!C::kWide) {
              q[0] = qf[k][0]; q[1] = qf[k][1]; q[2] = qf[k][2]; q[3] = qf[k][3];
            } else {
              const uint4 x = q_sm[(mt * (D / 16) + k) * 32 + lane];
              q[0] = x.x; q[1] = x.y; q[2] = x.z; q[3] = x.w;
            }
          };
          uint32_t qa[4], qb[4];
          query(F8 ? c : c / 2, qa);
          if constexpr (F8) query(c + 1, qb);
#pragma unroll
          for (int j = 0; j < KT / 16; ++j) {
            uint32_t kf[4];
            ldsm4(kf, chunk_addr(kb, j, c));
            if constexpr (!F8) {
              mma16816<false>((c / 2) & 1 ? other(2 * j) : s[2 * j], qa, kf[0], kf[1]);
              mma16816<false>((c / 2) & 1 ? other(2 * j + 1) : s[2 * j + 1], qa, kf[2], kf[3]);
            } else {
              uint32_t b[4][2];
#pragma unroll
              for (int e = 0; e < 4; ++e) e4m3x4_f16(kf[e], b[e][0], b[e][1]);
              mma16816<true>(s[2 * j], qa, b[0][0], b[0][1]);
              mma16816<true>(s[2 * j + 1], qa, b[2][0], b[2][1]);
              mma16816<true>(other(2 * j), qb, b[1][0], b[1][1]);
              mma16816<true>(other(2 * j + 1), qb, b[3][0], b[3][1]);
            }
          }
        }
        const bool masked = key0 + KT > n - a.Tq + 1;  // some row does not see all of the tile
        if constexpr (kChains == 2) {
#pragma unroll
          for (int j = 0; j < KT / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] += s2[j][e];
        }
        if (masked) {
#pragma unroll
          for (int j = 0; j < KT / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + j * 8 + 2 * ql + (e & 1) >= (e < 2 ? limA : limB)) s[j][e] = -INFINITY;
        }
        // running maximum
        float nA = mA, nB = mB;
#pragma unroll
        for (int j = 0; j < KT / 8; ++j) {
          nA = fmaxf(nA, fmaxf(s[j][0], s[j][1]));
          nB = fmaxf(nB, fmaxf(s[j][2], s[j][3]));
        }
        nA = quad_max(nA);
        nB = quad_max(nB);
        // The maximum that the weights refer to moves only when a row's grows by more than kSlack (in units of log 2), for
        // moving it rescales the whole accumulator: with the true maximum, every other tile does for some row of a warp.
        // A common factor 2^kLift of the weights cancels in the division. bf16 weights take 2^-24, so that none passes 2^-20
        // and the sums over a million keys of the type's largest value are finite, as their mean is; fp32 and bf16 have the
        // exponents to spare (a weight below 2^-102 of the largest is lost). f16 weights take 2^11: they end below 2^15, and
        // what a long row's many small weights lose below f16's normal range stays under 2^-35 of the largest each; e4m3
        // values leave their sums far from fp32's range.
        constexpr float kSlack = 4.f, kLift = F8 ? 11.f : -20.f - kSlack;
        if (__any_sync(0xffffffffu, (nA - mA) * fA > kSlack || (nB - mB) * fB > kSlack)) {
          const float cA = mA == nA ? 1.f : ex2((mA - nA) * fA), cB = mB == nB ? 1.f : ex2((mB - nB) * fB);
          lsum[0] *= cA;
          lsum[2] *= cB;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            acc[j][0] *= cA;
            acc[j][1] *= cA;
            acc[j][2] *= cB;
            acc[j][3] *= cB;
          }
          mA = nA;
          mB = nB;
        }
        const float zA = mA == -INFINITY ? 0.f : mA * fA, zB = mB == -INFINITY ? 0.f : mB * fB;
        // P in the cache's MMA type; the sums take the same weights, so that a row's still add up to one. f16 keeps 11 bits
        // of a weight, finer than the output. bf16 keeps 8, as few as the output, which would show in rows whose values
        // nearly cancel (the error's mean square over 48 ragged sequences 1.35 times that of the output's rounding alone):
        // what it leaves over goes into a second operand and a second product, 16 bits together. Up to 16 rows a kv head
        // that costs nothing (48 sequences: 68.1 against 69.0 us), with four tokens 83.0 against 81.0, with eight, where
        // the products bound the call, 146 against 126. Over e4m3 the 11 bits leave 1.0015 times the rounding's error. The first part is cut off below the weight, never at it, so that
        // a weight above zero has two parts above zero: an infinite value times them is infinite, not no number.
        uint32_t pf[KT / 16][4], pr[F8 ? 1 : KT / 16][4];
        const float yA = kLift - zA, yB = kLift - zB;
        auto weights = [&](int j, int e, float x, float y) {
          uint32_t& w = pf[j >> 1][(j & 1) * 2 + e];
          if constexpr (F8) {
            w = pack2<true>(x, y);
          } else {
            constexpr float kBelow = 1.f - 0x1p-22f;
            w = __byte_perm(__float_as_uint(x * kBelow), __float_as_uint(y * kBelow), 0x7632);
            pr[j >> 1][(j & 1) * 2 + e] = pack2<false>(x - lo_bf(w), y - hi_bf(w));
          }
        };
#pragma unroll
        for (int j = 0; j < KT / 8; ++j) {
          weights(j, 0, ex2(fmaf(s[j][0], fA, yA)), ex2(fmaf(s[j][1], fA, yA)));
          weights(j, 1, ex2(fmaf(s[j][2], fB, yB)), ex2(fmaf(s[j][3], fB, yB)));
        }
#pragma unroll
        for (int ks = 0; ks < KT / 16; ++ks) {
          mma16816<F8>(lsum, pf[ks], kOnes, kOnes);
          if constexpr (!F8) mma16816<false>(lsum, pr[ks], kOnes, kOnes);
        }
        // O += P V. B fragments of the 16 keys from key0 + 16 ks, the columns of chunk pair c
        auto pv = [&](auto&& keep, auto&& add) {
#pragma unroll
          for (int ks = 0; ks < KT / 16; ++ks) {
#pragma unroll
            for (int c = 0; c < KC; c += 2) {
              uint32_t vf[4];
              ldsm4t(vf, chunk_addr(vb, ks, c));
#pragma unroll
              for (int e = 0; e < 4; ++e) vf[e] &= keep(ks, e & 1);
              if constexpr (!F8) {
                add(acc[c], pf[ks], vf[0], vf[1]);
                add(acc[c + 1], pf[ks], vf[2], vf[3]);
                add(acc[c], pr[ks], vf[0], vf[1]);
                add(acc[c + 1], pr[ks], vf[2], vf[3]);
              } else {
                // a 16-bit unit holds two columns of one key: even columns to one MMA, odd ones to the next
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  uint32_t even0, odd0, even1, odd1;  // keys 0-7 and 8-15
                  e4m3x4_f16(__byte_perm(vf[2 * e], 0, 0x3120), even0, odd0);
                  e4m3x4_f16(__byte_perm(vf[2 * e + 1], 0, 0x3120), even1, odd1);
                  add(acc[2 * (c + e)], pf[ks], even0, even1);
                  add(acc[2 * (c + e) + 1], pf[ks], odd0, odd1);
                }
              }
            }
          }
        };
        // A weight of zero does not silence a NaN or an infinity, so what lies behind the sequence is made zero where
        // it lies, and a row that some tokens see and others do not is looked through for such values first.
        bool careful = false;
        if (masked) {
          uint8_t* v8 = ring + (size_t)slot * C::kSlot + C::kTile;
          for (int r = max(0, n - key0); r < KT; ++r)
            if (lane < C::kRow / 16)
              *reinterpret_cast<uint4*>(v8 + (lane >> 3) * C::kSeg + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
          bool odd = false;
          for (int r = max(0, n - a.Tq + 1 - key0); r < min(KT, n - key0); ++r)
            if (lane < C::kRow / 16) {
              const uint4 x = *reinterpret_cast<const uint4*>(v8 + (lane >> 3) * C::kSeg + r * 128 + (lane & 7) * 16);
              odd |= not_finite<F8>(x.x) || not_finite<F8>(x.y) || not_finite<F8>(x.z) || not_finite<F8>(x.w);
            }
          careful = __any_sync(0xffffffffu, odd);
          fence_proxy_async_smem();  // the next copy into the slot comes after these writes
          __syncwarp();
        }
        if (!careful) {
          pv([](int, int) { return 0xffffffffu; },
             [](float (&d)[4], const uint32_t (&p)[4], uint32_t b0, uint32_t b1) { mma16816<F8>(d, p, b0, b1); });
        } else {
          // one pass per token of these rows, over the keys that token sees, kept by its rows alone
          const int r0 = rb * a.rows + mt * 16, t0 = token_of(a, r0), t1 = min(a.Tq - 1, token_of(a, r0 + 15));
#pragma unroll 1
          for (int t = t0; t <= t1; ++t) {
            const int vis = n - a.Tq + t + 1 - key0;  // keys of the tile that token t sees
            pv([&](int ks, int hi) {
                 const int k = ks * 16 + hi * 8 + 2 * ql;
                 return (k < vis ? 0xffffu : 0u) | (k + 1 < vis ? 0xffff0000u : 0u);
               },
               [&](float (&d)[4], const uint32_t (&p)[4], uint32_t b0, uint32_t b1) {
                 float x[4] = {d[0], d[1], d[2], d[3]};
                 mma16816<F8>(x, p, b0, b1);
                 if (tA == t) {
                   d[0] = x[0];
                   d[1] = x[1];
                 }
                 if (tB == t) {
                   d[2] = x[2];
                   d[3] = x[3];
                 }
               });
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot]);
      if ((slot += NG) >= NS) {
        slot = g;
        ++turn;
      }
    }
    const float lA = lsum[0], lB = lsum[2];
    // maxima in units of log 2 from here on
    mA = mA == -INFINITY ? mA : mA * fA;
    mB = mB == -INFINITY ? mB : mB * fB;

    // The job's end: the NG warps of a row tile exchange their maxima and sums, scale what they hold to the common
    // maximum, and add up in shared memory, kMergeCols columns at a time; a thread then holds four columns of a row.
    if (ql == 0) {
      merge_ml[warp * 16 + qr] = make_float2(mA, lA);
      merge_ml[warp * 16 + qr + 8] = make_float2(mB, lB);
    }
    consumers_sync();
    float sA, sB;  // this warp's factors
    {
      float xA = -INFINITY, xB = -INFINITY;
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        xA = fmaxf(xA, merge_ml[(k * MT + mt) * 16 + qr].x);
        xB = fmaxf(xB, merge_ml[(k * MT + mt) * 16 + qr + 8].x);
      }
      sA = ex2(mA - (xA == -INFINITY ? 0.f : xA));
      sB = ex2(mB - (xB == -INFINITY ? 0.f : xB));
    }
    constexpr int kLanes = C::kMergeCols / 4, kRows = kWarps * 32 / kLanes;  // threads of a row, rows a turn
    const int ocol = (tid % kLanes) * 4;
    const float vs = a.v_scale ? a.v_scale[h] : 1.f;
#pragma unroll
    for (int c0 = 0; c0 < D; c0 += C::kMergeCols) {
      float* mine = merge + (warp * 16 + qr) * C::kMergeRow;
#pragma unroll
      for (int j = c0 / 8; j < (c0 + C::kMergeCols) / 8; j += F8 ? 2 : 1) {
        // columns of accumulator tile j: bf16 8 j + 2 ql, + 1; e4m3 (tiles j, j + 1) 8 j + 4 ql + {0, 2}, + {1, 3}
        if constexpr (!F8) {
          float* at = mine + 8 * j - c0 + 2 * ql;
          *reinterpret_cast<float2*>(at) = make_float2(acc[j][0] * sA, acc[j][1] * sA);
          *reinterpret_cast<float2*>(at + 8 * C::kMergeRow) = make_float2(acc[j][2] * sB, acc[j][3] * sB);
        } else {
          float* at = mine + 8 * j - c0 + 4 * ql;
          *reinterpret_cast<float4*>(at) = make_float4(acc[j][0] * sA, acc[j + 1][0] * sA, acc[j][1] * sA, acc[j + 1][1] * sA);
          *reinterpret_cast<float4*>(at + 8 * C::kMergeRow) =
              make_float4(acc[j][2] * sB, acc[j + 1][2] * sB, acc[j][3] * sB, acc[j + 1][3] * sB);
        }
      }
      consumers_sync();
#pragma unroll 1
      for (int lr = tid / kLanes; lr < min(MT * 16, M - rb * a.rows); lr += kRows) {
        const int x = lr >> 4, row = rb * a.rows + lr;  // row tile; row in the job's kv head
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          const float4 p =
              *reinterpret_cast<const float4*>(merge + ((k * MT + x) * 16 + (lr & 15)) * C::kMergeRow + ocol);
          o.x += p.x;
          o.y += p.y;
          o.z += p.z;
          o.w += p.w;
        }
        float m = -INFINITY, l = 0.f;
        if (whole || (c0 == 0 && ocol == 0)) {
          float2 ml[NG];
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            ml[k] = merge_ml[(k * MT + x) * 16 + (lr & 15)];
            m = fmaxf(m, ml[k].x);
          }
#pragma unroll
          for (int k = 0; k < NG; ++k) l = fmaf(ml[k].y, ex2(ml[k].x - (m == -INFINITY ? 0.f : m)), l);
        }
        if (whole) {
          const float d = l == 0.f ? 0.f : vs / l;  // an empty row is zero; a NaN sum stays
          const int t = token_of(a, row);
          uint16_t* dst = a.out + (((int64_t)w.b * a.Tq + t) * a.Hq + h * a.G + (row - t * a.G)) * D + c0 + ocol;
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<false>(o.x * d, o.y * d), pack2<false>(o.z * d, o.w * d));
        } else {
          const int64_t at = ((int64_t)blockIdx.x * 2 + (njob > 0)) * a.rows + lr;
          if (c0 == 0 && ocol == 0) *reinterpret_cast<float2*>(a.ml + at * 2) = make_float2(m, l);
          *reinterpret_cast<float4*>(a.acc + at * D + c0 + ocol) = o;
        }
      }
      consumers_sync();
    }
    ++njob;
  }
  if (!ok)  // no copy may still be landing when the CTA exits: this group's last tiles once more
    for (int k = g; k < NS; k += NG) {
      const int t = k < slot ? turn : turn - 1;  // the slot's last turn
      if (t >= 0) bar_wait(&full[k], t & 1);
    }
}

// The join. CTA c, of the border before the attention's CTA c, takes the (c - c0 - 1)-th of c1 - c0 equal shares of the
// (row, four columns) items of the job that lies across it, the work of CTAs c0 .. c1. An item's parts, one per CTA of the
// job in order, are weighted by 2^(m_i - m) and added; a share of few items has its parts spread over the threads.
constexpr int kJoinThreads = 256;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PAttnArgs a) {
  constexpr int kCols = D / 4, kT = kJoinThreads, kMaxRows = 64;
  __shared__ float4 red[kT];
  // weights of the share's rows: rows * parts <= (64 / (parts - 1) + 2) * parts
  __shared__ float wt[2 * kMaxRows + 2 * kPagedMaxCtas];
  __shared__ float inv[kMaxRows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.x + 1;
  pdl_wait();
  pdl_launch_dependents();
  const int4 j0 = *reinterpret_cast<const int4*>(a.joins + c * JOIN_INTS);
  const int2 j1 = *reinterpret_cast<const int2*>(a.joins + c * JOIN_INTS + 4);
  const int parts = j0.x, c0 = j0.y, second = j0.z, b = j0.w, h = j1.x, rb = j1.y;
  if (parts == 0) return;
  const int rows = min(a.rows, a.G * a.Tq - rb * a.rows), all = rows * kCols, share = c - c0 - 1;
  const int i0 = all * share / (parts - 1), i1 = all * (share + 1) / (parts - 1);  // all <= 2^12, parts <= 320
  if (i0 >= i1) return;
  const int r0 = i0 / kCols, r1 = (i1 - 1) / kCols + 1;
  auto part = [&](int i) { return (int64_t)(c0 + i) * 2 + (i == 0 ? second : 0); };
  // Few items (many parts): the parts of an item over `slices` threads, a power of two up to 32. Many items (few parts):
  // kItems items a thread at a time. Either way each thread's first kAhead values are on their way while the weights are
  // found: eight parts of one item, or two of each of four.
  constexpr int kAhead = 8, kItems = 4;
  int lg = 0;
  while (lg < 5 && (i1 - i0) << (lg + 1) <= kT) ++lg;
  const int slices = 1 << lg, lanes = kT >> lg, sl = (tid << lg) / kT, mine = i0 + (tid & (lanes - 1));
  auto load = [&](int it, int i) {
    const int r = it / kCols, col = it % kCols;
    return it < i1 && i < parts ? __ldcg(reinterpret_cast<const float4*>(a.acc + (part(i) * a.rows + r) * D + col * 4))
                                : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  auto weight = [&](int it, int i) { return it < i1 && i < parts ? wt[(it / kCols - r0) * parts + i] : 0.f; };
  auto add = [](float4& s, const float4& x, float f) {
    s.x = fmaf(x.x, f, s.x);
    s.y = fmaf(x.y, f, s.y);
    s.z = fmaf(x.z, f, s.z);
    s.w = fmaf(x.w, f, s.w);
  };
  auto store = [&](int it, const float4& s) {
    if (it >= i1) return;
    const int r = it / kCols, col = it % kCols, q = rb * a.rows + r, t = token_of(a, q);
    const float d = inv[r - r0];
    *reinterpret_cast<uint2*>(a.out + (((int64_t)b * a.Tq + t) * a.Hq + h * a.G + (q - t * a.G)) * D + col * 4) =
        make_uint2(pack2<false>(s.x * d, s.y * d), pack2<false>(s.z * d, s.w * d));
  };
  float4 ahead[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    ahead[k] = slices > 1 ? load(mine, sl + k * slices) : load(mine + k % kItems * kT, k / kItems);
  for (int r = r0 + warp; r < r1; r += kT / 32) {
    constexpr int kHeld = 3;  // a lane's parts that stay in registers
    float2 x[kHeld];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int i = lane + 32 * k;
      x[k] = i < parts ? __ldcg(reinterpret_cast<const float2*>(a.ml + (part(i) * a.rows + r) * 2))
                       : make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) m = fmaxf(m, x[k].x);
    for (int i = lane + 32 * kHeld; i < parts; i += 32) m = fmaxf(m, __ldcg(a.ml + (part(i) * a.rows + r) * 2));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float z = m == -INFINITY ? 0.f : m;
    float l = 0.f;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int i = lane + 32 * k;
      const float f = ex2(x[k].x - z);
      if (i < parts) wt[(r - r0) * parts + i] = f;
      l = fmaf(x[k].y, f, l);
    }
    for (int i = lane + 32 * kHeld; i < parts; i += 32) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(a.ml + (part(i) * a.rows + r) * 2));
      const float f = ex2(v.x - z);
      wt[(r - r0) * parts + i] = f;
      l = fmaf(v.y, f, l);
    }
    l = warp_sum(l);
    if (lane == 0) inv[r - r0] = l == 0.f ? 0.f : (a.v_scale ? a.v_scale[h] : 1.f) / l;
  }
  __syncthreads();
  if (slices > 1) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) add(s, ahead[k], weight(mine, sl + k * slices));
#pragma unroll 4
    for (int i = sl + kAhead * slices; i < parts; i += slices) add(s, load(mine, i), weight(mine, i));
    red[tid] = s;
    __syncthreads();
    if (sl != 0) return;
    for (int k = 1; k < slices; ++k) add(s, red[k * lanes + tid], 1.f);
    store(mine, s);
  } else {
    for (int base = mine; base < i1; base += kItems * kT) {
      float4 s[kItems];
#pragma unroll
      for (int k = 0; k < kItems; ++k) s[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = 0; i < parts; i += 2) {
        if (i > 0 || base != mine) {
#pragma unroll
          for (int k = 0; k < kAhead; ++k) ahead[k] = load(base + k % kItems * kT, i + k / kItems);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          add(s[k % kItems], ahead[k], weight(base + k % kItems * kT, i + k / kItems));
      }
#pragma unroll
      for (int k = 0; k < kItems; ++k) store(base + k * kT, s[k]);
    }
  }
}

// ------------------------------------------------------------------ host side

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static EncodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(f);
  });
  return fn;
}

// One layer's k or v as [page, head][row][value], fetched in boxes of 128 bytes x box_rows rows.
bool pool_map(CUtensorMap* m, const moe_paged_cache* c, const void* base, int box_rows) {
  memset(m, 0, sizeof *m);
  const EncodeTiled enc = encode_tiled();
  if (!enc) return false;
  const int es = kv_size(c->kv_type);
  const cuuint64_t dims[3] = {(cuuint64_t)c->D, (cuuint64_t)c->page, (cuuint64_t)c->num_pages * c->Hkv};
  const cuuint64_t strides[2] = {(cuuint64_t)c->D * es, (cuuint64_t)c->page * c->D * es};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base),
             dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool F8, int MT>
cudaError_t launch_attn(const PAttnArgs& args, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t s) {
  using C = Cfg<D, F8, MT>;
  static_assert(C::slots(kPagedMaxBatch) >= std::max(C::NG, C::NP), "each group and producer has a slot");
  const void* fn = reinterpret_cast<const void*>(paged_attn_kernel<D, F8, MT>);
  static SmemGrant granted;
  PAttnArgs a = args;
  a.ns = C::slots(a.B);
  const int smem = C::fixed_bytes(a.B) + a.ns * C::kSlot;
  cudaError_t e = grant_smem(fn, smem, C::kPerSm == 1 ? kSmemOne : kSmemTwo, granted);
  if (e != cudaSuccess) return e;
  static_assert(paged_max_ctas(D) * 2 == kPagedMaxCtas * C::kPerSm, "the partials' room");
  a.ctas = std::min(paged_max_ctas(D), paged_sms() * C::kPerSm);
  CUtensorMap k = mk, v = mv;
  void* p[] = {&a, &k, &v};
  e = paged_launch(fn, dim3(a.ctas), dim3(C::kThreads), smem, s, p);
  if (e != cudaSuccess) return e;
  void* j[] = {&a};
  return paged_launch(reinterpret_cast<const void*>(paged_join_kernel<D>), dim3(a.ctas - 1), dim3(kJoinThreads), 0, s, j);
}

template <int D, bool F8>
cudaError_t launch_rows(const PAttnArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t s) {
  if (a.rows == 16) return launch_attn<D, F8, 1>(a, mk, mv, s);
  if (a.rows == 32) return launch_attn<D, F8, 2>(a, mk, mv, s);
  return launch_attn<D, F8, 4>(a, mk, mv, s);
}

int tile_keys(int row_bytes) { return row_bytes <= 128 ? 32 : 16; }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_paged_attend(const moe_paged_cache* c, int layer, const int32_t* seqs, int B, int Tq, const uint16_t* q, int Hq,
                     float scale, uint16_t* out, void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  if (!paged_ok(c) || layer < 0 || layer >= c->layers || B < 0 || B > kPagedMaxBatch || Tq < 1 || Tq > kPagedMaxNew ||
      Hq < 1 || Hq > 128 || Hq % c->Hkv != 0 || !workspace || !paged_al16(workspace) || !paged_work_fits(c, Hq, B, Tq))
    return (int)cudaErrorInvalidValue;
  if (B == 0) return (int)cudaSuccess;
  if (!seqs || !q || !out || !paged_al16(q) || !paged_al16(out)) return (int)cudaErrorInvalidValue;
  const PagedWs L = paged_ws(c, Hq, B, Tq);
  if (workspace_bytes < L.total) return (int)cudaErrorInvalidValue;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PAttnArgs a;
  a.q = q;
  a.out = out;
  a.k_scale = c->kv_type == MOE_KV_E4M3 && c->k_scale ? c->k_scale + (int64_t)layer * c->Hkv : nullptr;
  a.v_scale = c->kv_type == MOE_KV_E4M3 && c->v_scale ? c->v_scale + (int64_t)layer * c->Hkv : nullptr;
  a.seqs = seqs;
  a.tables = c->tables;
  a.lens = c->lens;
  a.joins = reinterpret_cast<int32_t*>(ws + L.joins);
  a.ml = reinterpret_cast<float*>(ws + L.ml);
  a.acc = reinterpret_cast<float*>(ws + L.acc);
  a.err = reinterpret_cast<uint32_t*>(ws + L.err);
  a.B = B;
  a.Tq = Tq;
  a.Hq = Hq;
  a.Hkv = c->Hkv;
  a.G = Hq / c->Hkv;
  a.page = c->page;
  a.num_pages = c->num_pages;
  a.max_seqs = c->max_seqs;
  a.max_pages = c->max_pages;
  a.rows = paged_block_rows(a.G, Tq);
  a.row_blocks = (a.G * Tq + a.rows - 1) / a.rows;
  a.scale = scale;
  a.inv_G = 1.f / (float)a.G;
  a.ctas = 0;
  const int kt = tile_keys(c->D * kv_size(c->kv_type));
  a.box_rows = c->page % kt == 0 ? kt : 16;
  CUtensorMap mk, mv;
  const int64_t off = layer * paged_layer_bytes(c);
  if (!pool_map(&mk, c, static_cast<const uint8_t*>(c->k) + off, a.box_rows) ||
      !pool_map(&mv, c, static_cast<const uint8_t*>(c->v) + off, a.box_rows))
    return (int)cudaErrorNotSupported;
  const cudaStream_t s = (cudaStream_t)stream;
  if (c->kv_type == MOE_KV_E4M3)
    return (int)(c->D == 256 ? launch_rows<256, true>(a, mk, mv, s) : launch_rows<128, true>(a, mk, mv, s));
  if (c->D == 256) return (int)launch_rows<256, false>(a, mk, mv, s);
  return (int)(c->D == 128 ? launch_rows<128, false>(a, mk, mv, s) : launch_rows<64, false>(a, mk, mv, s));
}

}  // extern "C"
