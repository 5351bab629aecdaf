// Decode attention for sequences that share a prefix: the shared part.
//
// The sequences of a group have the same pages at the head of their block
// tables (prefix-cache hits, samples or beams of one prompt).  Softmax over
// keys A + B is the combination of partials over A and over B,
//   (m, l, o) = (max s, sum 2^(s - m), sum 2^(s - m) v),
//   m = max(m_A, m_B), l = l_A 2^(m_A - m) + l_B 2^(m_B - m), o likewise,
// so this kernel computes the partials of all members over the group's prefix
// at once -- a dense product of (members x heads) query rows with the prefix
// keys on the tensor cores, each K / V byte read once for up to 256 rows --,
// the same CTAs then stream every sequence's own keys (own_keys.cuh).
//
// Work: a row block is up to 256 rows of one group and kv head (256 / G members x
// the G = Hq / Hkv heads) and its prefix in tiles of 128 keys.  A job is a row
// block's whole prefix, or one of the equal pieces it is cut into so that no
// SM idles: a CTA (one on each SM) does one job as long as there are no more
// jobs than SMs.  How long the pieces are is weighed against the own keys,
// on which the SMs without a job start at once (sp_choose_piece).  The piece
// that starts a row block leaves its partial in the rows of the sequences, the
// others in a slot of their job: no place is written twice, and the merge finds
// them by the same arithmetic, in a fixed order.
//
// Roles (three warpgroups): warp 0 loads K and V tiles by TMA (a ring of 32 KB
// slots), warp 1 issues the MMAs (warps 2 and 3 only complete their
// warpgroup, which gives most of its registers away); warps 4-7 and 8-11 are
// the softmax of two tiles of 128 rows, one thread per row (its TMEM lane),
// whose 128 scores stay in registers:
//   S_t = Q_t K^T (TMEM, 128 x 128 fp32) -> registers -> P_t = 2^(s - m) as
//   bf16 over S_t's own columns -> O_t += P_t V (P_t read from TMEM).
// The tensor cores work on one tile while the other is in its softmax.  O_t is
// rescaled only when the row maximum grew by more than kSpLazy (log2): P then
// stays below 2^kSpLazy, which costs nothing in fp32 sums and in bf16's
// relative rounding, and the rescale all but disappears after the first tile.
// P is rounded to bf16 (the operand type of the PV product, as in the other
// attention kernels); maxima, sums and O are fp32.
//
// Bound by the softmax, whose exponentials and TMEM traffic take longer than the
// MMAs of the other tile: 2.2 us for 256 rows x 128 keys, and 14 us a job for the
// plan, the query rows, the first tile and the partial.  64 jobs of 32 tiles in 85
// us are 404 TFLOP/s on 64 SMs, 55 % of their part of the measured 1712.
#pragma once
#include "common.cuh"
#include "prefill_tc.cuh"

namespace b200 {

constexpr int kSpMaxSeqs = 1024;
constexpr int kSpMaxGroups = 512;  // groups of two at least
constexpr int kSpTile = 128;       // keys of a tile
constexpr int kSpRows = 256;       // rows of a block: two tiles of 128
constexpr int kSpSlots = 4;        // ring slots of 32 KB (K, V, K, V)
constexpr int kSpThreads = 384;
// registers: 168 a thread at launch (64 K over 12 warps), then 88 for the first
// warpgroup and 208 for the softmax: 128 x (88 + 208 + 208) = 384 x 168
constexpr int kSpRegsLaunch = 168, kSpRegsIssue = 88, kSpRegsSoftmax = 208;
static_assert(kSpRegsIssue + 2 * kSpRegsSoftmax == 3 * kSpRegsLaunch, "the shares are what the launch has");
constexpr float kSpLazy = 8.f;
constexpr float kSpFused = 4096.f;  // maxima (log2) beyond which scores are scaled before the difference
constexpr int kSpQ = 0;                            // [2 tiles][2 dim halves][128 rows][128 B]
constexpr int kSpRing = 65536;
constexpr int kSpPlanAt = kSpRing + kSpSlots * 32768;
constexpr int kSpBar = 226 * 1024 - 256;           // behind everything else: no other use of the memory

// The groups of a call, in shared memory.
struct SpPlan {
  int off[kSpMaxGroups + 1];        // first job of each group
  int tiles[kSpMaxGroups];          // 128-key tiles of the prefix (0: nothing shared)
  short start[kSpMaxGroups + 1];    // first member
  short split[kSpMaxGroups];        // pieces of a row block
  short member[kSpMaxSeqs];         // sequences by group, in batch order
};
// Only while the plan is made; lies in the ring, before its first load.
struct SpDraft {
  unsigned long long keys;          // of all live sequences
  int cnt[kSpMaxGroups];
  int least[kSpMaxGroups];          // shortest member (keys)
  short group[kSpMaxSeqs];
  short rank[kSpMaxSeqs];
  short seen[kSpMaxGroups];         // members numbered so far
};
static_assert(sizeof(SpDraft) <= kSpSlots * 32768, "the draft fits the ring");

// What the merge needs of a sequence; keys = 0: no shared part.
struct SpRec {
  int keys, split;            // shared keys; pieces of a row block
  int off, blocks;            // the group's first job; row blocks of a kv head
  int start, members, rank;   // members of the groups before; members of the group; this one's number
  int pad;
};
constexpr size_t kSpRecBytes = kSpMaxSeqs * sizeof(SpRec);

struct SharedArgs {
  const __nv_bfloat16* q;
  long long q_stride;
  int num_q_rows;
  const int* cu_q;
  const int* cu_k;
  const int* block_tables;
  int bt_stride, bt_width;
  const int* prefix_group;  // [B], -1: none
  const int* prefix_len;    // [groups]
  int groups;
  int always;               // share whatever it costs
  int B, Hq, Hkv, G, page, members;  // members: of a row block, kSpRows / G
  long long num_slots;
  float scale_log2;
  SpRec* rec;
  // own keys (own_keys.cuh)
  int* queue;         // kOwnQueueBytes, zero between calls
  int* starts;        // [B + 1]            first item of each sequence
  float2* part_ml;    // [items][Hq]
  float* part_o;      // [items][Hq][128]
  long long cap_items;
  __nv_bfloat16* out;
  long long out_stride;
  float2* first_ml;   // [B * Hq]           pieces that start a row block: rows by group, kv head, member, head
  float* first_o;     // [B * Hq][128]
  float2* rest_ml;    // [SMs][kSpRows]     the others, by job: rows of the block
  float* rest_o;      // [SMs][kSpRows][128]
  unsigned* err;
};

__device__ __forceinline__ float sp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
struct F2 {
  float x, y;
};
__device__ __forceinline__ F2 sp_fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ F2 sp_add2(F2 a, F2 b) {
  F2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// One lane of a converged warp, always the same one.
__device__ __forceinline__ bool sp_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ float sp_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 32 columns of this warp's TMEM lanes into registers that hold floats from
// the start: nothing may touch them before tmem_ld_wait().
__device__ __forceinline__ void sp_tmem_ld(uint32_t taddr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}

// O of this row times f, 16 columns at a time (the scores stay in registers meanwhile).
__device__ __forceinline__ void sp_tmem_scale(uint32_t taddr, float f) {
  uint32_t r[16];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr + (uint32_t)(c * 16)));
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      asm volatile("" : "+r"(r[i]));
      r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
    }
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(taddr + (uint32_t)(c * 16)),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
  }
}

// D[tmem] (+)= A[tmem] * B[smem]: the A operand's rows are TMEM lanes, two bf16 to a column.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// a / b for 0 <= a < 2^24 and b > 0: the float quotient is off by one at most.
__device__ __forceinline__ int sp_div(int a, int b) {
  int q = (int)__fdiv_rn((float)a, (float)b);
  const int r = a - q * b;
  return q + (r >= b) - (r < 0);
}

// The group that sequence b counts in (-1: none): live rows only.  `flag`: report what is out of range.
__device__ __forceinline__ int sp_group_of(const SharedArgs& a, int b, bool flag = false) {
  const int g = a.prefix_group[b];
  const int q0 = a.cu_q[b], nq = a.cu_q[b + 1] - q0, nk = a.cu_k[b + 1] - a.cu_k[b];
  if (g < -1 || g >= a.groups || nq > 1 || (nq == 1 && (q0 < 0 || q0 >= a.num_q_rows))) {
    if (flag) raise_error(a.err, ERR_BAD_INDEX);
    return -1;
  }
  return nq < 1 || nk <= 0 ? -1 : g;  // padding rows of a captured batch, rows without keys
}

// Groups, their members and shortest member (keys), and the keys of all live
// sequences.  All threads of the CTA call it.
__device__ __forceinline__ void sp_count_groups(const SharedArgs& a, int* cnt, int* least, unsigned long long* keys,
                                                short* group) {
  constexpr int threads = kSpThreads;
  const int tid = threadIdx.x;
  auto row = [&](int b, int& nk) {
    nk = 0;
    if (b >= a.B) return -1;
    nk = a.cu_q[b + 1] - a.cu_q[b] == 1 ? max(a.cu_k[b + 1] - a.cu_k[b], 0) : 0;
    return sp_group_of(a, b, blockIdx.x == 0);
  };
  int nk, g = row(tid, nk);  // (the loads of the first rows are on their way during the barrier)
  for (int i = tid; i < a.groups; i += threads) {
    cnt[i] = 0;
    least[i] = 0x7fffffff;
  }
  if (tid == 0) *keys = 0;
  __syncthreads();
  for (int b0 = 0; b0 < a.B; b0 += threads) {
    if (b0 > 0) g = row(b0 + tid, nk);
    if (b0 + tid < a.B) group[b0 + tid] = (short)g;
    if (g >= 0) {
      atomicAdd(&cnt[g], 1);
      atomicMin(&least[g], nk);
    }
    unsigned long long sum = nk;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((tid & 31) == 0 && sum > 0) atomicAdd(keys, sum);
  }
  __syncthreads();
}

// A job takes about kSpCostJob + kSpCostTile a tile (us), own keys begin after kSpCostOwn.
constexpr float kSpCostJob = 14.f, kSpCostTile = 2.2f, kSpCostOwn = 10.f;

// Tiles of a group's prefix: of whole pages that every member sees.
__device__ __forceinline__ int sp_prefix_tiles(const SharedArgs& a, int given, int members, int least) {
  return members < 2 ? 0 : min(max(min(given, least), 0) / a.page, a.bt_width) * (a.page / kSpTile);
}

// A prefix is shared where that pays, by times in us:
// - Reading a tile (64 KB) once and not once a member saves 1.59 of an SM for
//   each member but one; a row block costs 15 beside the reads and 0.6 a tile.
// - A job, cut into as many pieces as the SMs have room for, has to be over before
//   the batch without sharing would be (`alone` to read all keys, of which a
//   part is shared elsewhere: 0.6 of it; 2 more than a job's start).
// Measured, shared / not: 64 pairs behind 0.1 to 0.5k keys 79 / 57, 0.5 to 2k
// 122 / 125, 1 to 4k 183 / 210; 128 pairs behind 1 to 4k 344 / 431; 16 pairs behind 1
// to 4k 71 / 54 (the second rule: 128 jobs, uncut); 64 groups of 4 behind 0.5 to 2k
// 140 / 211.
__device__ __forceinline__ bool sp_pays(const SharedArgs& a, int tiles, int members, int blocks, int pieces,
                                        float alone) {
  const float saved = 1.59f * (float)(members - 1) * (float)tiles;
  const float cost = (float)blocks * (15.f + 0.6f * (float)tiles);
  const float job = kSpCostJob + kSpCostTile * (float)sp_div(tiles + pieces - 1, pieces);
  return saved > cost && job < 0.6f * alone + kSpCostJob + 2.f;
}

// Tiles of a piece, chosen by one warp: each lane weighs one number of pieces of
// the longest prefix by a model of the call, fitted to measurements (us, on 148
// SMs): an SM streams own keys at 60 GB/s, all of them together at 6.1 TB/s, the
// SMs without a job from the start and the others when their jobs end.
__device__ __forceinline__ int sp_choose_piece(const SharedArgs& a, const SpPlan& s, const SpDraft& d, int longest,
                                              long long own_keys) {
  const int lane = threadIdx.x & 31, sms = gridDim.x;
  const int pieces = lane < 16 ? lane + 1 : 8 * lane - 104;  // 1 .. 16, 24, 32 .. 144
  const int len = max(1, sp_div(longest + pieces - 1, pieces));
  float jobs = 0.f;  // (their number can pass 31 bits before it is refused)
  for (int g = 0; g < a.groups; ++g)
    if (s.tiles[g] > 0)
      jobs += (float)(sp_div(d.cnt[g] + a.members - 1, a.members) * a.Hkv) * (float)sp_div(s.tiles[g] + len - 1, len);
  const float bytes = (float)own_keys * a.Hkv * 512.f;
  const float shared = (kSpCostJob + kSpCostTile * len) * ceilf(__fdividef(jobs, (float)sms));
  const float rate = fminf(fmaxf(sms - jobs, 0.f) * 60e3f, 6.1e6f);     // bytes / us beside the jobs
  const float left = bytes - fmaxf(shared - kSpCostOwn, 0.f) * rate;     // when they end
  float cost = left > 0.f ? shared + 2.f + left / 6.1e6f : shared;
  if (jobs > sms && pieces > 1) cost = 3e38f;  // cut only what fits the SMs
  // the least cost, and of equals the fewest pieces
  float best = cost;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fminf(best, __shfl_xor_sync(0xffffffffu, best, o));
  const int who = __ffs(__ballot_sync(0xffffffffu, cost == best)) - 1;
  return __shfl_sync(0xffffffffu, len, max(who, 0));
}

// The MMA warp, which allocates TMEM, and the softmax warps, which use it.
__device__ __forceinline__ void sp_bar_tmem() { asm volatile("bar.sync 1, 288;" ::: "memory"); }

// Builds the plan (every CTA the same) in shared memory.  All threads call it.
__device__ __forceinline__ void sp_build_plan(const SharedArgs& a, SpPlan& s, SpDraft& d) {
  const int tid = threadIdx.x, lane = tid & 31;
  for (int g = tid; g < a.groups; g += kSpThreads) s.tiles[g] = a.prefix_len[g];
  sp_count_groups(a, d.cnt, d.least, &d.keys, d.group);
  // member numbers in batch order, by the last warp, beside the first one's work below
  if (tid >= kSpThreads - 32) {
    for (int g = lane; g < a.groups; g += 32) d.seen[g] = 0;
    __syncwarp();
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int b = b0 + lane;
      const int g = b < a.B ? d.group[b] : -1;
      const unsigned same = __match_any_sync(0xffffffffu, g);
      const int before = __popc(same & ((1u << lane) - 1u));
      int n = 0;
      if (g >= 0) {
        n = d.seen[g];
        d.rank[b] = (short)(n + before);
      }
      __syncwarp();
      if (g >= 0 && before == 0) d.seen[g] = (short)(n + __popc(same));
      __syncwarp();
    }
  }
  if (tid < 32) {
    // prefixes, then the length of a piece, then first members and jobs
    int longest = 0, blocks = 0;
    long long shared_keys = 0;
    for (int g = lane; g < a.groups; g += 32) {
      s.tiles[g] = sp_prefix_tiles(a, s.tiles[g], d.cnt[g], d.least[g]);
      if (s.tiles[g] > 0) blocks += sp_div(d.cnt[g] + a.members - 1, a.members);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) blocks += __shfl_xor_sync(0xffffffffu, blocks, o);
    const int room = blocks > 0 ? max(1, sp_div(gridDim.x, blocks * a.Hkv)) : 1;
    const float alone = (float)d.keys * (float)(a.Hkv * 512) / 6.1e6f;
    for (int g = lane; g < a.groups; g += 32) {
      int tiles = s.tiles[g];
      if (!a.always && !sp_pays(a, tiles, d.cnt[g], sp_div(d.cnt[g] + a.members - 1, a.members), room, alone)) tiles = 0;
      s.tiles[g] = tiles;
      longest = max(longest, tiles);
      shared_keys += (long long)d.cnt[g] * tiles * kSpTile;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
      shared_keys += __shfl_xor_sync(0xffffffffu, shared_keys, o);
    }
    __syncwarp();
    const int len = sp_choose_piece(a, s, d, longest, (long long)d.keys - shared_keys);
    int members = 0, jobs = 0;
    for (int g0 = 0; g0 < a.groups; g0 += 32) {
      const int g = g0 + lane;
      int n = 0, split = 0, j = 0;
      if (g < a.groups) {
        n = d.cnt[g];
        split = sp_div(s.tiles[g] + len - 1, len);
        j = sp_div(n + a.members - 1, a.members) * a.Hkv * split;
      }
      int ni = n, ji = j;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, ni, o), y = __shfl_up_sync(0xffffffffu, ji, o);
        if (lane >= o) {
          ni += x;
          ji += y;
        }
      }
      if (g < a.groups) {
        s.start[g] = (short)(members + ni - n);
        s.off[g] = jobs + ji - j;
        s.split[g] = (short)split;
      }
      members += __shfl_sync(0xffffffffu, ni, 31);
      jobs += __shfl_sync(0xffffffffu, ji, 31);
    }
    if (lane == 0) {
      s.start[a.groups] = (short)members;
      s.off[a.groups] = jobs;
    }
  }
  __syncthreads();
  for (int b = tid; b < a.B; b += kSpThreads)
    if (d.group[b] >= 0) s.member[s.start[d.group[b]] + d.rank[b]] = (short)b;
  __syncthreads();
}

// A job: a run of tiles of one row block.
struct SpSeg {
  int g, h, block;   // group, kv head, row block
  int k0, k1;        // tiles of the prefix
  int rows, nt;      // valid rows; tiles of 128 rows in use
};

__device__ __forceinline__ SpSeg sp_segment(const SharedArgs& a, const SpPlan& s, int job) {
  int lo = 0, hi = a.groups - 1;  // the last group that starts at the job or before it
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.off[mid] <= job) lo = mid; else hi = mid - 1;
  }
  SpSeg g;
  g.g = lo;
  const int n = s.start[lo + 1] - s.start[lo], split = s.split[lo], tiles = s.tiles[lo];
  const int blocks = sp_div(n + a.members - 1, a.members);
  const int at = sp_div(job - s.off[lo], split), piece = job - s.off[lo] - at * split;
  const int each = sp_div(tiles, split), more = tiles - each * split;  // the first `more` pieces have one tile more
  g.k0 = piece * each + min(piece, more);
  g.k1 = g.k0 + each + (piece < more);
  g.h = sp_div(at, blocks);
  g.block = at - g.h * blocks;
  g.rows = min(a.members, n - g.block * a.members) * a.G;
  g.nt = g.rows > 128 ? 2 : 1;
  return g;
}

// First cache row of tile k of the group's prefix, from its first member's table; -1: no such page.
__device__ __forceinline__ long long sp_tile_row(const SharedArgs& a, int leader, int k) {
  const int per = a.page / kSpTile;
  const int col = k / per;
  const long long blk = a.block_tables[(size_t)leader * a.bt_stride + col];
  const long long row = blk * a.page + (long long)(k - col * per) * kSpTile;
  return blk >= 0 && row + kSpTile <= a.num_slots ? row : -1;
}

// Shared memory of the jobs, aligned to 1024 bytes.
struct SpSmem {
  uint8_t* smem;
  uint64_t* bars;
  __device__ __forceinline__ explicit SpSmem(uint8_t* p) : smem(p), bars(reinterpret_cast<uint64_t*>(p + kSpBar)) {}
  __device__ __forceinline__ uint64_t* full() const { return bars; }                   // [kSpSlots]
  __device__ __forceinline__ uint64_t* empty() const { return bars + kSpSlots; }       // [kSpSlots]
  // [2] a job's query rows are in shared memory, O may be overwritten
  __device__ __forceinline__ uint64_t* q_full() const { return bars + 2 * kSpSlots; }
  __device__ __forceinline__ uint64_t* s_full() const { return q_full() + 2; }         // [2]
  __device__ __forceinline__ uint64_t* p_full() const { return q_full() + 4; }         // [2]
  __device__ __forceinline__ uint64_t* o_done() const { return q_full() + 6; }         // [2]
  __device__ __forceinline__ uint64_t* p_half() const { return q_full() + 8; }         // [2] the first 64 keys of P are there
  __device__ __forceinline__ uint64_t* drain() const { return q_full() + 10; }
  __device__ __forceinline__ uint32_t* tmem_slot() const { return reinterpret_cast<uint32_t*>(q_full() + 11); }
  // some page is missing: the softmax looks which
  __device__ __forceinline__ volatile int* bad() const { return reinterpret_cast<int*>(q_full() + 12); }
  __device__ __forceinline__ SpPlan& plan() const { return *reinterpret_cast<SpPlan*>(smem + kSpPlanAt); }
  // One thread; the barrier that ends the plan shows them to the others.
  __device__ __forceinline__ void init() const {
    for (int i = 0; i < 2 * kSpSlots; ++i) mbar_init(&bars[i], 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full()[t], 4);  // a warp's lane 0 arrives for its rows
      mbar_init(&s_full()[t], 1);
      mbar_init(&p_full()[t], 4);
      mbar_init(&p_half()[t], 4);
      mbar_init(&o_done()[t], 1);
    }
    mbar_init(drain(), 1);
    *bad() = 0;
  }
};

// What the merge needs of the sequences; all threads of a CTA call it after the plan.
__device__ __forceinline__ void sp_write_records(const SharedArgs& a, const SpPlan& plan, const SpDraft& draft) {
  for (int b = threadIdx.x; b < a.B; b += kSpThreads) {
    SpRec r{};
    const int g = draft.group[b];
    if (g >= 0 && plan.tiles[g] > 0) {
      r.keys = plan.tiles[g] * kSpTile;
      r.split = plan.split[g];
      r.off = plan.off[g];
      r.start = plan.start[g];
      r.members = plan.start[g + 1] - plan.start[g];
      r.blocks = sp_div(r.members + a.members - 1, a.members);
      r.rank = draft.rank[b];
    }
    a.rec[b] = r;
  }
}

// This CTA's jobs: number blockIdx.x, and every gridDim.x-th after it.  All
// threads call it, with the registers of the launch, and have those again after it.
__device__ __forceinline__ void sp_run_jobs(const SharedArgs& a, const SpSmem& sm, int jobs, const CUtensorMap& tmK,
                                            const CUtensorMap& tmV) {
  uint8_t* smem = sm.smem;
  uint64_t *full = sm.full(), *empty = sm.empty(), *q_full = sm.q_full(), *s_full = sm.s_full(),
           *p_full = sm.p_full(), *o_done = sm.o_done(), *p_half = sm.p_half(), *drain = sm.drain();
  uint32_t* tmem_slot = sm.tmem_slot();
  volatile int* bad = sm.bad();
  SpPlan& plan = sm.plan();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t base = smem_u32(smem);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSpRegsIssue));
    // ---- producer
    if (warp == 0 && lane == 0) {
      int it = 0;      // loads issued; load it is in slot it % kSpSlots
      bool ok = true;
      for (int job = blockIdx.x; ok && job < jobs; job += gridDim.x) {
        const SpSeg g = sp_segment(a, plan, job);
        const int leader = plan.member[plan.start[g.g]];
        for (int k = g.k0; ok && k < g.k1; ++k) {
          long long row = sp_tile_row(a, leader, k);
          if (row < 0) {
            raise_error(a.err, ERR_BAD_INDEX);
            *bad = 1;
            row = a.num_slots;  // behind the cache: the load fills zeros (the softmax masks the tile)
          }
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int sl = it % kSpSlots;
            if (it >= kSpSlots && !mbar_wait(&empty[sl], (uint32_t)(it / kSpSlots + 1) & 1u, a.err)) {
              ok = false;
              break;
            }
            const uint32_t dst = base + kSpRing + (uint32_t)sl * 32768u, bar = smem_u32(&full[sl]);
            mbar_arrive_expect_tx(&full[sl], 32768);
            // (boxes of 32 keys: the tensor maps are those of the own keys)
#pragma unroll
            for (int r = 0; r < kSpTile; r += 32) {
              tma_load_3d(dst + r * 128, kv ? &tmV : &tmK, bar, 0, g.h, (int)row + r);
              tma_load_3d(dst + 16384 + r * 128, kv ? &tmV : &tmK, bar, 64, g.h, (int)row + r);
            }
            ++it;
          }
        }
      }
      // every load has landed before the CTA may end (a wait that gave up leaves some unread)
      for (int i = it > kSpSlots ? it - kSpSlots : 0; i < it; ++i)
        mbar_wait(&full[i % kSpSlots], (uint32_t)(i / kSpSlots) & 1u, a.err);
    }
    __syncwarp();
    // ---- MMA issuer: the whole warp walks the loop, so that descriptors live in
    // uniform registers, and one elected lane issues
    if (warp == 1) {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
      tc_fence_before();
      sp_bar_tmem();
      tc_fence_after();
      const uint32_t tmem = *tmem_slot;
      const uint32_t idesc_s = umma_idesc_bf16(128, kSpTile);
      const uint32_t idesc_o = umma_idesc_bf16(128, 128) | (1u << 16);  // B (V) MN-major
      // descriptors count in 16 bytes: 2048 a ring slot or Q tile, 1024 a half of the dims
      const uint64_t dq = umma_desc_sw128(base + kSpQ), dk = umma_desc_sw128(base + kSpRing),
                     dv = umma_desc_sw128_mn(base + kSpRing, 16384u);
      const bool leader = sp_elect();
      int it = 0, seg[2] = {0, 0}, step[2] = {0, 0};
      bool ok = true;
      // (each lane has a clock of its own: they give up together)
      auto wait_slot = [&](int i) {
        return __all_sync(0xffffffffu, mbar_wait(&full[i % kSpSlots], (uint32_t)(i / kSpSlots) & 1u, a.err)) != 0;
      };
      auto scores = [&](int t, int i) {  // S_t = Q_t K^T, K in load i
        const uint64_t q = dq + (uint32_t)t * 2048u, k = dk + (uint32_t)(i % kSpSlots) * 2048u;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t o = (uint32_t)(kk >> 2) * 1024u + (uint32_t)(kk & 3) * 2u;
            tc_mma_f16(tmem + (uint32_t)t * 128u, q + o, k + o, idesc_s, kk > 0 ? 1u : 0u);
          }
          tc_commit(&s_full[t]);
        }
      };
      auto values = [&](int t, int i, int half, bool acc) {  // O_t (+)= P_t V over 64 keys, V in load i
        const uint64_t v = dv + (uint32_t)(i % kSpSlots) * 2048u;
        if (leader) {
#pragma unroll
          for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
            tc_mma_f16_ts(tmem + 256u + (uint32_t)t * 128u, tmem + (uint32_t)t * 128u + (uint32_t)kk * 8u,
                          v + (uint32_t)kk * 128u, idesc_o, (acc || kk > 0) ? 1u : 0u);
        }
      };
      auto commit = [&](uint64_t* bar) {
        if (leader) tc_commit(bar);
      };
      for (int job = blockIdx.x; ok && job < jobs; job += gridDim.x) {
        const SpSeg g = sp_segment(a, plan, job);
        // the first scores of both tiles
        ok = wait_slot(it);
        for (int t = 0; ok && t < g.nt; ++t) {
          ok = mbar_wait(&q_full[t], (uint32_t)seg[t] & 1u, a.err);
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after();
          if (ok) scores(t, it);
        }
        if (!ok) break;
        commit(&empty[it % kSpSlots]);
        for (int k = g.k0; k < g.k1; ++k, it += 2) {
          const bool more = k + 1 < g.k1;
          ok = wait_slot(it + 1);
          for (int t = 0; t < g.nt; ++t) {
            ok = ok && mbar_wait(&p_half[t], (uint32_t)step[t] & 1u, a.err);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            values(t, it + 1, 0, k > g.k0);
            ok = mbar_wait(&p_full[t], (uint32_t)step[t] & 1u, a.err);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            ++step[t];
            tc_fence_after();
            values(t, it + 1, 1, true);
            // S_t's next scores overwrite P_t: MMAs of one thread run in the order of issue
            if (more && t == 0) {
              ok = wait_slot(it + 2);
              if (!ok) break;
            }
            if (more) scores(t, it + 2);
            else commit(&o_done[t]);
          }
          if (!ok) break;
          commit(&empty[(it + 1) % kSpSlots]);
          if (more) commit(&empty[(it + 2) % kSpSlots]);
        }
        if (!ok) break;
        for (int t = 0; t < g.nt; ++t) ++seg[t];
      }
      // every MMA issued has completed before TMEM can be released
      commit(drain);
      mbar_wait(drain, 0u, a.err);
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSpRegsSoftmax));
    // ---- softmax: one thread per row of its tile
    const int t = warp >= 8;
    const int q4 = warp & 3;             // TMEM lane quarter of this warp
    const int row = q4 * 32 + lane;      // of the tile
    uint32_t ts = 0, to = 0;             // S / P and O of the row, once TMEM is allocated
    bool have_tmem = false;
    int seg = 0, step = 0;
    bool ok = true;
    for (int job = blockIdx.x; ok && job < jobs; job += gridDim.x) {
      const SpSeg g = sp_segment(a, plan, job);
      if (t >= g.nt) continue;
      const int m0 = plan.start[g.g] + g.block * a.members;  // first member of the block
      uint8_t* qrows = smem + kSpQ + t * 32768 + q4 * 4096;  // this warp's 32 rows (64 dims; the others 16 KB on)
      {
        // the rows in the swizzled K-major layout of the MMA, two rows of 256 bytes a load
        const int r = t * 128 + row;  // row of the block: member r / G, head r % G (zeros behind the last member)
        const int i = r / a.G;
        // (every lane loads, from the block's first row where there is none: a
        // load under a condition would be waited for before the next one)
        const long long from = r < g.rows ? (long long)a.cu_q[plan.member[m0 + i]] * a.q_stride +
                                                (g.h * a.G + r - i * a.G) * 128
                                          : (long long)a.cu_q[plan.member[m0]] * a.q_stride + g.h * a.G * 128;
        uint4 v[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const long long at = __shfl_sync(0xffffffffu, from, 2 * c + (lane >> 4));
          v[c] = __ldg(reinterpret_cast<const uint4*>(a.q + at) + (lane & 15));
        }
        if (!have_tmem) {
          sp_bar_tmem();  // (while the rows are on their way)
          tc_fence_after();
          ts = *tmem_slot + ((uint32_t)(q4 * 32) << 16) + (uint32_t)t * 128u;
          to = ts + 256u;
          have_tmem = true;
        }
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const int rr = 2 * c + (lane >> 4), ch = lane & 15;
          if (t * 128 + q4 * 32 + rr >= g.rows) v[c] = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(qrows + (ch >> 3) * 16384 + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4)) = v[c];
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[t]);
      }
      const int leader = plan.member[plan.start[g.g]];
      float m = -INFINITY, l = 0.f;
      for (int k = g.k0; ok && k < g.k1; ++k, ++step) {
        ok = mbar_wait(&s_full[t], (uint32_t)step & 1u, a.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) sp_tmem_ld(ts + (uint32_t)(c * 32), s + c * 32);
        tmem_ld_wait();
        // every use of s stays behind the wait
#pragma unroll
        for (int i = 0; i < 128; ++i) asm volatile("" : "+f"(s[i]));
        const bool there = !*bad || sp_tile_row(a, leader, k) >= 0;
        float mx[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mx[i] = sp_max3(s[i], s[i + 8], s[i + 16]);
#pragma unroll
        for (int i = 24; i < 120; i += 16) {
#pragma unroll
          for (int e = 0; e < 8; ++e) mx[e] = sp_max3(mx[e], s[i + e], s[i + 8 + e]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) mx[i] = fmaxf(mx[i], s[120 + i]);
        float mt = fmaxf(sp_max3(sp_max3(mx[0], mx[1], mx[2]), mx[3], mx[4]), sp_max3(mx[5], mx[6], mx[7]));
        mt = there ? mt * a.scale_log2 : -INFINITY;
        if (!there) {
#pragma unroll
          for (int i = 0; i < 128; ++i) s[i] = -INFINITY;
        }
        // S complete means that O_t += P V of the tile before is too: rescale O in place
        if (__any_sync(0xffffffffu, mt > m + kSpLazy)) {
          const float m_new = fmaxf(m, mt);
          const float alpha = m == -INFINITY ? 0.f : sp_exp2(m - m_new);
          if (k > g.k0) sp_tmem_scale(to, alpha);
          l *= alpha;
          m = m_new;
        }
        const float mm = m == -INFINITY ? 0.f : m;  // nothing but -inf so far: P = 0
        F2 scale2 = {a.scale_log2, a.scale_log2};
        const F2 minus = {-mm, -mm};
        // The fused s scale - mm keeps what was rounded off in mm, up to 2^-24 of it:
        // nothing beside the rounding of P as long as mm is small, but at the
        // lowest value of a type (masked keys) 2^100 and more.  There the product is
        // rounded first, as the maximum and the own keys' scores are.
        if (__any_sync(0xffffffffu, fabsf(mm) > kSpFused)) {
#pragma unroll
          for (int i = 0; i < 128; ++i) s[i] *= a.scale_log2;
          scale2 = {1.f, 1.f};
        }
        F2 sum[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const F2 y = sp_fma2({s[c * 64 + 2 * i], s[c * 64 + 2 * i + 1]}, scale2, minus);
            // (a polynomial on the FMA pipe for some of the pairs: 2 % faster for
            // one of eight, 5 % slower for three, the warps then lack issue slots)
            const F2 e = {sp_exp2(y.x), sp_exp2(y.y)};
            sum[i & 3] = sp_add2(sum[i & 3], e);
            pk[i] = pack_bf16x2(e.x, e.y);
          }
          tmem_st_32x32b_x32(ts + (uint32_t)(c * 32), pk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          // the PV product of the first 64 keys runs while the others are exponentiated
          if (lane == 0) mbar_arrive(c ? &p_full[t] : &p_half[t]);
        }
        const F2 rs = sp_add2(sp_add2(sum[0], sum[1]), sp_add2(sum[2], sum[3]));
        l += rs.x + rs.y;
      }
      if (!ok) break;
      // ---- the job's partial
      ok = mbar_wait(&o_done[t], (uint32_t)seg & 1u, a.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ++seg;
      tc_fence_after();
      const bool first = g.k0 == 0;
      const size_t at = first ? ((size_t)plan.start[g.g] * a.Hkv +
                                 (size_t)g.h * (plan.start[g.g + 1] - plan.start[g.g]) + g.block * a.members) * a.G
                              : (size_t)job * kSpRows;  // (cut only when there are no more jobs than SMs)
      const int r0 = t * 128 + q4 * 32;  // this warp's first row of the block
      if (r0 + lane < g.rows) (first ? a.first_ml : a.rest_ml)[at + r0 + lane] = make_float2(m, l);
      float* po = (first ? a.first_o : a.rest_o) + (at + r0) * 128;
      // 32 columns at a time through this warp's part of the Q tile (its MMAs
      // are done), so that a store writes whole 128-byte lines
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float x[32];
        sp_tmem_ld(to + (uint32_t)(c * 32), x);
        tmem_ld_wait();
        uint8_t* stage = qrows + (c & 1) * 16384;
#pragma unroll
        for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(x[i]));
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<float4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) =
              make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = 4 * i + (lane >> 3);
          const float4 y = *reinterpret_cast<const float4*>(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
          if (r0 + rr < g.rows) *reinterpret_cast<float4*>(po + rr * 128 + c * 32 + (lane & 7) * 4) = y;
        }
        __syncwarp();
      }
    }
    if (!have_tmem) sp_bar_tmem();  // (no job had rows for these warps: the barrier still counts them)
  }
  tc_fence_before();
  __syncthreads();
  if (warp < 4) {
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(*tmem_slot, 512);
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSpRegsLaunch));
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSpRegsLaunch));
  }
}

}  // namespace b200
