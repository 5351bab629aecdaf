// Decode attention for sequences that share a prefix: every sequence's own
// keys (those behind its group's prefix, or all of them), and the merge.
//
// HBM-bound: each K / V byte of these keys belongs to one sequence and is read
// once.  An item is a stretch of up to 512 keys (1024 where the batch's own
// keys are long, fewer when every warp would otherwise not get one) of one
// sequence and kv head; the G = Hq / Hkv query heads that share the kv head
// are the columns of the MMAs (S^T = K Q^T, O^T = V^T P^T on mma.sync: with 8
// columns at most there is nothing a larger tile could be filled with).
//
// A CTA has kOwnWarps pairs of warps.  A producer takes items from a global
// queue, looks up their pages and keeps its consumer's ring of 32-key K / V
// tiles (TMA, 128-byte swizzle, one mbarrier each way) full, so that the queue's
// and the tables' latency never stops the arithmetic; the consumer's chain of
// products and shuffles is what a tile costs an SM, and six of them in flight
// with two tiles each beat four with three.  A row with several parts leaves them
// as fp32 partials (m, l, o).
//
// Measured (32 query and 8 kv heads): 256 sequences behind one prefix of 8k keys,
// 526 MB of own keys beside 64 jobs of 32 tiles, 99 us and 6 for the merge (the
// bytes alone: 87); 256 sequences in 9 groups and without one, 665 MB, 126 us and
// 8 (119); 32 sequences behind 2k keys, 48 MB, 18.5 and 6 (8.9: the plan takes 4
// us, an item's first tile 3, the merge waits for the launch and two trips to L2).
#pragma once
#include "common.cuh"
#include "shared_prefix.cuh"

namespace b200 {

constexpr int kOwnHD = 128;
constexpr int kOwnItem = 512;        // keys of an item; sizes the workspace
constexpr int kOwnItemLong = 1024;   // with kOwnLongMean own keys a sequence or more
constexpr int kOwnLongMean = 2048;
constexpr int kOwnItemLeast = 64;
constexpr int kOwnTile = 32;         // keys of a ring stage
constexpr int kOwnWarps = 6;         // consumer warps, each with a producer warp
constexpr int kOwnStages = 2;
constexpr int kOwnThreads = kOwnWarps * 64;
// stage: K [2 dim halves][32 keys][128 B] | V same | Q [2 halves][8 heads][128 B] (with an item's first tile)
constexpr int kOwnK = 0, kOwnV = 8192, kOwnQ = 16384;
constexpr int kOwnStageBytes = 18432;
constexpr int kOwnWarpBytes = kOwnStages * kOwnStageBytes;
constexpr int kOwnQueueBytes = 256;  // {next item, producers out of the queue, items + 1}: zero between calls

struct OwnTile {
  int b, h, c, qrow;
  int ntok;   // valid keys of the tile; -1: no more tiles
  int first, last, alone;  // of its item; the item is all of its row
};

struct OwnPlan {
  uint64_t full[kOwnWarps][kOwnStages], empty[kOwnWarps][kOwnStages];
  OwnTile tile[kOwnWarps][kOwnStages];
  long long keys[kOwnThreads / 32];
  int sums[kOwnThreads / 32];
  int item;                   // keys of an item
  int late;
  int start[kSpMaxSeqs + 1];  // first item (of one kv head) of each sequence
  int prefix[kSpMaxSeqs];     // keys of its shared prefix
};
static_assert(kOwnThreads == kSpThreads, "one CTA does both");
constexpr int kOwnPlanAt = kOwnWarps * kOwnWarpBytes;
static_assert(kOwnPlanAt >= kSpPlanAt + (int)sizeof(SpPlan), "behind all that the jobs use");
static_assert(kOwnPlanAt + (int)sizeof(OwnPlan) <= kSpBar, "the jobs' barriers stay");
constexpr int kSharedSmemBytes = 1024 + kSpBar + 256;
static_assert(kSharedSmemBytes <= 227 * 1024, "shared memory of one CTA");

// Tiled load of keys that no one else will read: they leave L2 first, before
// the shared prefixes, the partials and the kernels' own instructions.
__device__ __forceinline__ uint64_t own_read_once() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void own_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t c0, int32_t c1,
                                            int32_t c2, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
      : "memory");
}

// byte offset of 16-byte chunk ch (0..15 over 128 dims) of row r in a tile of [2 halves][rows][128 B]
__device__ __forceinline__ uint32_t own_at(int half_bytes, int r, int ch) {
  return (uint32_t)((ch >> 3) * half_bytes + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
}

// `n` producers are done with the queue; the last of all resets it for the next call.
__device__ __forceinline__ void own_leave(const SharedArgs& a, int n) {
  if (atomicAdd(&a.queue[1], n) + n == (int)gridDim.x * kOwnWarps) {
    atomicExch(&a.queue[0], 0);
    atomicExch(&a.queue[2], 0);
    atomicExch(&a.queue[1], 0);
  }
}

// The own keys, as many items as this CTA gets from the queue.  All threads call
// it, after the jobs of the prefixes; `sp` is the plan of those, whose memory the
// rings take.
__device__ __forceinline__ void own_run(const SharedArgs& a, uint8_t* smem, const SpPlan& sp, const CUtensorMap& tmK,
                                        const CUtensorMap& tmV, const CUtensorMap& tmQ) {
  OwnPlan& s = *reinterpret_cast<OwnPlan*>(smem + kOwnPlanAt);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the CTA whose number no job has, unless every SM has one, writes what the merge reads
  const bool writer = blockIdx.x == gridDim.x - 1;
  // A CTA that comes late (it had a job) and finds the queue empty needs no plan.
  if (!writer) {
    if (tid == 0) {
      const int items = *reinterpret_cast<volatile int*>(&a.queue[2]) - 1;
      s.late = items >= 0 && *reinterpret_cast<volatile int*>(&a.queue[0]) >= items;
    }
    __syncthreads();
    if (s.late) {
      if (tid == 0) own_leave(a, kOwnWarps);
      return;
    }
  }
  // ---- plan (every CTA the same): shared keys, then the prefix sum of items
  {
    const int per = (a.B + kOwnThreads - 1) / kOwnThreads;
    const int beg = min(a.B, tid * per), end = min(a.B, beg + per);
    long long keys = 0;
    int active = 0;
    for (int b = beg; b < end; ++b) {
      const int g = sp_group_of(a, b);
      const int p = g >= 0 ? sp.tiles[g] * kSpTile : 0;
      const int q0 = a.cu_q[b], nq = a.cu_q[b + 1] - q0;
      const int nk = a.cu_k[b + 1] - a.cu_k[b] - p;
      s.prefix[b] = p;
      // own keys, for now (a row outside q, or of several queries, has no place to go: sp_group_of reports it)
      s.start[b] = nq == 1 && q0 >= 0 && q0 < a.num_q_rows ? max(nk, 0) : 0;
      keys += s.start[b];
      active += s.start[b] > 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      keys += __shfl_xor_sync(0xffffffffu, keys, o);
      active += __shfl_xor_sync(0xffffffffu, active, o);
    }
    if (lane == 0) {
      s.keys[warp] = keys;
      s.sums[warp] = active;
    }
    fence_proxy_async_smem();
    __syncthreads();
    keys = 0;
    active = 0;
    for (int w = 0; w < kOwnThreads / 32; ++w) {
      keys += s.keys[w];
      active += s.sums[w];
    }
    // keys of an item: short ones where every warp would not get one of 512,
    // long ones (half the fixed work) on long sequences
    const long long warps = (long long)gridDim.x * kOwnWarps;
    const long long each = (keys * a.Hkv + warps - 1) / warps;
    int len = kOwnItem;
    if (each < kOwnItem) len = max(kOwnItemLeast, (int)(each + kOwnTile - 1) / kOwnTile * kOwnTile);
    else if (keys >= (long long)kOwnLongMean * active) len = kOwnItemLong;
    __syncthreads();  // sums are used again
    int local = 0;
    for (int b = beg; b < end; ++b) local += (s.start[b] + len - 1) / len;
    int incl = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s.sums[warp] = incl;
    __syncthreads();
    int run = incl - local;
    for (int w = 0; w < warp; ++w) run += s.sums[w];
    for (int b = beg; b < end; ++b) {
      const int n = (s.start[b] + len - 1) / len;
      s.start[b] = run;
      run += n;
    }
    if (tid == kOwnThreads - 1) s.start[a.B] = run;
    if (tid == 0) s.item = len;
    __syncthreads();
  }
  const int total = s.start[a.B], len = s.item;
  if (writer)
    for (int b = tid; b <= a.B; b += kOwnThreads) a.starts[b] = s.start[b];
  if ((long long)total > a.cap_items) {  // lengths past max_seqlen_k
    if (writer && tid == 0) raise_error(a.err, ERR_BAD_INDEX);
    return;
  }
  const int w = warp % kOwnWarps;
  uint8_t* ring = smem + w * kOwnWarpBytes;

  if (warp >= kOwnWarps) {
    // ---- producer
    const int items = total * a.Hkv;
    if (w == 0 && lane == 0) {  // for late CTAs; in place before this thread leaves the queue
      atomicExch(&a.queue[2], items + 1);
      __threadfence();
    }
    const int q_rows = min(a.Hq, 8);
    const uint64_t once = own_read_once();
    int it = 0;  // tiles issued; tile it is in stage it % kOwnStages
    bool ok = true;
    auto stage_free = [&]() {
      if (it < kOwnStages) return true;
      return mbar_wait(&s.empty[w][it % kOwnStages], (uint32_t)(it / kOwnStages + 1) & 1u, a.err);
    };
    while (ok) {
      int i = 0;
      if (lane == 0) i = atomicAdd(&a.queue[0], 1);
      i = __shfl_sync(0xffffffffu, i, 0);
      if (i >= items) break;
      const int c = i / a.Hkv, h = i - c * a.Hkv;
      int lo = 0, hi = a.B - 1;  // the last sequence that starts at c or before it
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s.start[mid] <= c) lo = mid; else hi = mid - 1;
      }
      const int b = lo;
      const int prefix = s.prefix[b];
      const int j0 = prefix + (c - s.start[b]) * len;
      const int n = min(len, a.cu_k[b + 1] - a.cu_k[b] - j0);
      // pages of the item, one a lane: at most 1024 keys over pages of 256 slots or more
      const int col0 = j0 / a.page;
      int page = -1;
      if (lane < 6 && col0 + lane < a.bt_width) page = a.block_tables[(size_t)b * a.bt_stride + col0 + lane];
      OwnTile d;
      d.b = b; d.h = h; d.c = c;
      d.qrow = a.cu_q[b];
      d.alone = s.start[b + 1] - s.start[b] == 1 && prefix == 0;
      const int tiles = (n + kOwnTile - 1) / kOwnTile;
      int col = 0, off = j0 - col0 * a.page;  // page of the item, slot in it
      for (int k = 0; k < tiles; ++k) {
        const int blk = __shfl_sync(0xffffffffu, page, col);
        const int m = min(kOwnTile, n - k * kOwnTile);
        const long long row = (long long)blk * a.page + off;
        const bool there = blk >= 0 && row + m <= a.num_slots;
        off += kOwnTile;
        if (off >= a.page) {  // (pages are whole numbers of tiles, and items start on one)
          off = 0;
          ++col;
        }
        ok = __all_sync(0xffffffffu, stage_free());  // (each lane has a clock of its own: they leave together)
        if (!ok) break;
        if (lane == 0) {
          if (!there) raise_error(a.err, ERR_BAD_INDEX);
          const int st = it % kOwnStages;
          d.ntok = there ? m : 0;  // a missing page: row 0 is loaded and every key masked
          d.first = k == 0;
          d.last = k == tiles - 1;
          s.tile[w][st] = d;
          const uint32_t at = smem_u32(ring) + (uint32_t)st * kOwnStageBytes, bar = smem_u32(&s.full[w][st]);
          const int r = there ? (int)row : 0;
          mbar_arrive_expect_tx(&s.full[w][st], 4 * 4096 + (k == 0 ? 256 * q_rows : 0));
          own_load_3d(at + kOwnK, &tmK, bar, 0, h, r, once);
          own_load_3d(at + kOwnK + 4096, &tmK, bar, 64, h, r, once);
          own_load_3d(at + kOwnV, &tmV, bar, 0, h, r, once);
          own_load_3d(at + kOwnV + 4096, &tmV, bar, 64, h, r, once);
          if (k == 0) {
            tma_load_3d(at + kOwnQ, &tmQ, bar, 0, h * a.G, d.qrow);
            tma_load_3d(at + kOwnQ + 1024, &tmQ, bar, 64, h * a.G, d.qrow);
          }
        }
        ++it;
      }
    }
    if (lane == 0) {
      own_leave(a, 1);
      if (ok && stage_free()) {
        s.tile[w][it % kOwnStages].ntok = -1;
        mbar_arrive(&s.full[w][it % kOwnStages]);
        ++it;
      }
      // every load has landed before the CTA may end (a consumer that gave up leaves some unread)
      for (int i = it > kOwnStages ? it - kOwnStages : 0; i < it; ++i)
        mbar_wait(&s.full[w][i % kOwnStages], (uint32_t)(i / kOwnStages) & 1u, a.err);
    }
    __syncwarp();
  } else {
    // ---- consumer.  Tokens are the MMA rows, heads the columns: 0..G-1 are
    // the item's, the others carry unrelated rows and are never stored (every
    // column is independent of the others).
    const int g = lane >> 2, tq = lane & 3;  // fragment row group / column pair
    const uint32_t base = smem_u32(ring);
    uint32_t qb[8][2];                       // B fragments of Q^T, 8 k-steps of 16 dims
    float ot[8][4];                          // O^T: 8 tiles of 16 dims
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};  // head columns 2tq, 2tq + 1
    for (int it = 0;; ++it) {
      const int st = it % kOwnStages;
      bool ok = mbar_wait(&s.full[w][st], (uint32_t)(it / kOwnStages) & 1u, a.err);
      if (!__all_sync(0xffffffffu, ok)) break;
      const OwnTile d = s.tile[w][st];
      if (d.ntok < 0) break;
      const uint32_t sK = base + (uint32_t)st * kOwnStageBytes + kOwnK, sV = sK + kOwnV, sQ = sK + kOwnQ;
      if (d.ntok < kOwnTile) {
        // slots behind the sequence hold other data of the page, possibly
        // never written: zero their V so that P = 0 cannot meet a NaN
        for (int i = lane; i < (kOwnTile - d.ntok) * 16; i += 32)
          *reinterpret_cast<uint4*>(ring + st * kOwnStageBytes + kOwnV + own_at(4096, d.ntok + (i >> 4), i & 15)) =
              make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();  // before the next load into this stage
        __syncwarp();
      }
      if (d.first) {
#pragma unroll
        for (int p = 0; p < 4; ++p)
          ldmatrix_x4(sQ + own_at(1024, lane & 7, 4 * p + (lane >> 3)), qb[2 * p][0], qb[2 * p][1], qb[2 * p + 1][0],
                      qb[2 * p + 1][1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) ot[i][0] = ot[i][1] = ot[i][2] = ot[i][3] = 0.f;
        m_run[0] = m_run[1] = -INFINITY;
        l_run[0] = l_run[1] = 0.f;
      }
      // S^T: 2 token tiles of 16, each as two chains over the dims
      float sc[2][2][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i >> 3][(i >> 2) & 1][i & 3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t ka[4];
          ldmatrix_x4(sK + own_at(4096, 16 * mt + (lane & 7) + 8 * ((lane >> 3) & 1), 2 * kk + (lane >> 4)), ka[0],
                      ka[1], ka[2], ka[3]);
          mma_bf16_16816(sc[mt][kk & 1], ka, qb[kk][0], qb[kk][1]);
        }
      }
      // online softmax per head column (its 32 tokens live in the 8 lanes
      // that share tq: reduce over lane bits 2..4); the sum stays a lane's own
      // until the item ends
      float x[2][4], cm[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = 16 * mt + g + 8 * (i >> 1);
          // (never fused with the difference below: see kSpFused)
          x[mt][i] = tok < d.ntok ? __fmul_rn(sc[mt][0][i] + sc[mt][1][i], a.scale_log2) : -INFINITY;
          cm[i & 1] = fmaxf(cm[i & 1], x[mt][i]);
        }
      }
      float alpha[2], mm[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        cm[e] = fmaxf(cm[e], __shfl_xor_sync(0xffffffffu, cm[e], 4));
        cm[e] = fmaxf(cm[e], __shfl_xor_sync(0xffffffffu, cm[e], 8));
        cm[e] = fmaxf(cm[e], __shfl_xor_sync(0xffffffffu, cm[e], 16));
        const float m_new = fmaxf(m_run[e], cm[e]);
        mm[e] = m_new == -INFINITY ? 0.f : m_new;  // nothing but -inf so far: P = 0
        alpha[e] = sp_exp2(m_run[e] - mm[e]);
        m_run[e] = m_new;
      }
      // P (bf16, the PV operand) -> B fragments of P^T through 8x8 transposes
      float ls[2] = {0.f, 0.f};
      uint32_t pb[2][2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = sp_exp2(x[mt][i] - mm[i & 1]);
          ls[i & 1] += p[i];
        }
        pb[mt][0] = movmatrix_trans(pack_bf16x2(p[0], p[1]));  // tokens 16mt + 2tq, +1
        pb[mt][1] = movmatrix_trans(pack_bf16x2(p[2], p[3]));  // tokens 16mt + 8 + 2tq, +1
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) l_run[e] = l_run[e] * alpha[e] + ls[e];
      // O^T += V^T P^T: 8 dim tiles x 2 token steps
#pragma unroll
      for (int md = 0; md < 8; ++md) {
        ot[md][0] *= alpha[0]; ot[md][1] *= alpha[1];
        ot[md][2] *= alpha[0]; ot[md][3] *= alpha[1];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t va[4];
          ldmatrix_x4_trans(sV + own_at(4096, 16 * ks + (lane & 7) + 8 * (lane >> 4), 2 * md + ((lane >> 3) & 1)),
                            va[0], va[1], va[2], va[3]);
          mma_bf16_16816(ot[md], va, pb[ks][0], pb[ks][1]);
        }
      }
      __syncwarp();  // every lane has read the stage
      if (lane == 0) mbar_arrive(&s.empty[w][st]);
      if (!d.last) continue;
      // ---- the item's result: the row itself, or a part of it
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 4);
        l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 8);
        l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 16);
      }
      if (d.alone) {
        // O / l, transposed back to [head][dim] rows: the transposes are
        // warp-wide, then the lanes of the G live heads store
        const float inv0 = l_run[0] == 0.f ? 0.f : 1.f / l_run[0];
        const float inv1 = l_run[1] == 0.f ? 0.f : 1.f / l_run[1];
        __nv_bfloat16* dst = a.out + (size_t)d.qrow * a.out_stride + (size_t)(d.h * a.G + g) * kOwnHD;
#pragma unroll
        for (int md = 0; md < 8; ++md) {
          const uint32_t lo = movmatrix_trans(pack_bf16x2(ot[md][0] * inv0, ot[md][1] * inv1));
          const uint32_t hi = movmatrix_trans(pack_bf16x2(ot[md][2] * inv0, ot[md][3] * inv1));
          if (g < a.G) {
            *reinterpret_cast<uint32_t*>(dst + 16 * md + 2 * tq) = lo;
            *reinterpret_cast<uint32_t*>(dst + 16 * md + 8 + 2 * tq) = hi;
          }
        }
        continue;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = 2 * tq + e;
        if (col < a.G) {
          const size_t row = (size_t)d.c * a.Hq + (size_t)d.h * a.G + col;
          float* po = a.part_o + row * kOwnHD;
#pragma unroll
          for (int md = 0; md < 8; ++md) {
            po[16 * md + g] = ot[md][e];
            po[16 * md + 8 + g] = ot[md][2 + e];
          }
          if (g == 0) a.part_ml[row] = make_float2(m_run[e], l_run[e]);
        }
      }
    }
  }
}

// Jobs of the shared prefixes, then own keys: a CTA without a job starts on the
// own keys at once.  (Two kernels that overlapped took 1 to 3 us more: the second
// one's CTAs began where the first one's ended, and made the plan once more.  The
// merge behind a barrier of all CTAs in this kernel, instead of a launch of its
// own, took 1 to 3 us more, too: 12 resident warps an SM, not 36.)
__global__ void __launch_bounds__(kSpThreads, 1)
    shared_attention_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                            const __grid_constant__ CUtensorMap tmQ, const SharedArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const SpSmem sm(smem);
  const int tid = threadIdx.x;
  if (tid == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmQ);
    sm.init();
  }
  if (tid >= 32 && tid < 32 + kOwnWarps * kOwnStages) {
    OwnPlan& s = *reinterpret_cast<OwnPlan*>(smem + kOwnPlanAt);
    mbar_init(&s.full[0][tid - 32], 1);
    mbar_init(&s.empty[0][tid - 32], 1);
  }
  fence_mbar_init();
  griddep_wait();
  SpDraft& draft = *reinterpret_cast<SpDraft*>(smem + kSpRing);
  sp_build_plan(a, sm.plan(), draft);
  const int jobs = sm.plan().off[a.groups];
  if (blockIdx.x == gridDim.x - 1) sp_write_records(a, sm.plan(), draft);
  // the ring, with the draft in it, is the TMA's from here on
  fence_proxy_async_smem();
  __syncthreads();
  if ((int)blockIdx.x < jobs) sp_run_jobs(a, sm, jobs, tmK, tmV);
  own_run(a, smem, sm.plan(), tmK, tmV, tmQ);
  griddep_launch_dependents();
}

// ---------------------------------------------------------------------------
// The parts of a row of attention with shared prefixes: the prefix's pieces,
// then the items of the sequence's own keys, always in that order.  kLanes lanes
// to a (sequence, query head).  The parts come from L2, so it is latency that
// counts: kFlight parts are in flight at once.  A warp to a row and 8 parts where
// rows are few (often of many pieces: with half a warp 4 sequences behind 16k keys
// 33.0 us, not 30.9), half a warp and 4 parts where there are more than 24 rows an
// SM, so that twice as many are under way (256 sequences of 32 heads: 106.9, not
// 108.5).
// ---------------------------------------------------------------------------
constexpr int kMergeWarps = 4;

template <int kFlight, int kLanes>
__global__ void __launch_bounds__(kMergeWarps * 32, kFlight == 8 ? 6 : 7) shared_merge_kernel(const SharedArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kVecs = 32 / kLanes;  // of 4 dims a lane
  const int row = (blockIdx.x * kMergeWarps * 32 + threadIdx.x) / kLanes, lane = threadIdx.x % kLanes;
  if (row >= a.B * a.Hq) return;
  const int b = row / a.Hq, hq = row - b * a.Hq, h = hq / a.G;
  const int q0 = a.cu_q[b], nq = a.cu_q[b + 1] - q0;
  const int c0 = a.starts[b], own = a.starts[b + 1] - c0;
  const SpRec rc = a.rec[b];
  if (nq != 1 || (own == 1 && rc.keys == 0)) return;  // padding, or reported with the plan; written by its one item
  if (q0 < 0 || q0 >= a.num_q_rows) return;            // reported with the plan
  if (c0 < 0 || own < 0 || (long long)c0 + own > a.cap_items) {  // lengths past max_seqlen_k: no such parts
    if (lane == 0) raise_error(a.err, ERR_BAD_INDEX);
    return;
  }
  const int pieces = rc.keys > 0 ? rc.split : 0;  // of the prefix: the first, then those of the next jobs
  const int job = rc.off + (h * rc.blocks + rc.rank / a.members) * rc.split;
  const size_t first = ((size_t)rc.start * a.Hkv + (size_t)h * rc.members + rc.rank) * a.G + (hq - h * a.G);
  const size_t in_block = (size_t)(rc.rank % a.members) * a.G + (hq - h * a.G);
  const int n = pieces + own;
  float M = -INFINITY, L = 0.f;
  float4 acc[kVecs];
#pragma unroll
  for (int e = 0; e < kVecs; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += kFlight) {
    float2 ml[kFlight];
    float4 o[kFlight][kVecs];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int i = i0 + u;
      const float2* pm;
      const float* po;
      if (i < pieces) {
        const size_t at = i == 0 ? first : (size_t)(job + i) * kSpRows + in_block;
        pm = (i == 0 ? a.first_ml : a.rest_ml) + at;
        po = (i == 0 ? a.first_o : a.rest_o) + at * kOwnHD;
      } else {
        const size_t at = (size_t)(c0 + i - pieces) * a.Hq + hq;
        pm = a.part_ml + at;
        po = a.part_o + at * kOwnHD;
      }
      ml[u] = i < n ? __ldcg(pm) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int e = 0; e < kVecs; ++e)
        o[u][e] = i < n ? __ldcg(reinterpret_cast<const float4*>(po) + e * kLanes + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if (ml[u].y == 0.f) continue;  // no key there, or none of a finite score
      const float mn = fmaxf(M, ml[u].x);
      const float s = fast_exp2(M - mn), w = fast_exp2(ml[u].x - mn);
      L = L * s + w * ml[u].y;
#pragma unroll
      for (int e = 0; e < kVecs; ++e) {
        acc[e].x = acc[e].x * s + w * o[u][e].x;
        acc[e].y = acc[e].y * s + w * o[u][e].y;
        acc[e].z = acc[e].z * s + w * o[u][e].z;
        acc[e].w = acc[e].w * s + w * o[u][e].w;
      }
      M = mn;
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint2* out = reinterpret_cast<uint2*>(a.out + (size_t)q0 * a.out_stride + (size_t)hq * kOwnHD);
#pragma unroll
  for (int e = 0; e < kVecs; ++e)
    out[e * kLanes + lane] =
        make_uint2(pack_bf16x2(acc[e].x * inv, acc[e].y * inv), pack_bf16x2(acc[e].z * inv, acc[e].w * inv));
}

}  // namespace b200
