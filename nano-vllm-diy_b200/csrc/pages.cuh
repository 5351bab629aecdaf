// Pages of the KV cache: taking, forking, freeing, compacting and copying.
//
// State (all on the device, so that a step can change it without the host):
//   block_tables int32 [rows][width]  pages of each row in order, -1 behind them
//   seq_lens     int32 [rows]         tokens of each row: it holds ceil(len / page) pages
//   refs         int32 [pages]        rows that hold the page; 0 is a free page
//   cache        planes x pages       (plane = K or V of one layer)
//
// Two kinds of work:
//   * decisions (which free page goes where): one CTA, latency-bound.  Free
//     pages are taken lowest first: every thread owns a contiguous stretch of
//     refs, counts its free pages, one scan over the CTA gives each stretch
//     its first rank, and a second walk hands page k of the free list to the
//     request whose prefix sum of needs covers k (a binary search in shared
//     memory).  No order depends on a race, so results are the same every time.
//   * contents: HBM-bound copies of page heads over all planes in pieces of 32 KB,
//     one CTA each, handed out by the hardware: 6.41 TB/s with 24 ragged page
//     pairs of 72 planes, 6.53 with whole pages (99 % of a plain copy), where a
//     resident grid that strides over the pieces stayed at 4.9 to 5.9 and bulk
//     copies through shared memory at 5.7: pieces that start together then lie
//     together.  More than kPgGrid pieces share the CTAs (measured: within 1 %).
// A fork or a compaction is a decision launch and a content launch, in stream
// order; what the second needs lies in a plan array of the caller's.
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int kPgMax = 1024;            // requests of one call: one thread each in the deciding CTA
constexpr int kPgHash = 4 * kPgMax;     // slots of the table that finds repeated rows
constexpr int kPgThreads = 256;         // content kernels
constexpr int kPgPieceVecs = 2048;      // 16-byte vectors of one piece (32 KB: 8 a thread, all in flight)
constexpr int kPgGrid = 16384;          // CTAs of a content launch
constexpr int kPgGridUnknown = 8192;    // where only the device knows how many have work (empty ones: 6 us)
constexpr int kPgPlanWords = 4;         // fork plan: {source page, fresh page, tokens of the last page, full pages (-1: no fork)}

struct PageTables {
  int* tables;
  long long stride;
  int rows, width;
  int* lens;
  int* refs;
  int pages, page;
  unsigned* err;
};

struct PageCache {
  uint4* base;
  long long s0, s1, page_stride;  // in 16-byte vectors
  int n1;                         // planes = n0 * n1, plane p at (p / n1) * s0 + (p % n1) * s1
  int planes;
  int page_vecs, slot_vecs;
};

// Inclusive sum over the CTA's 1024 threads; `total` gets the whole.  `warp_sums`: 32 ints.
__device__ __forceinline__ int pg_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // warp_sums may still be read from an earlier scan
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int w = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return x + (warp > 0 ? before : 0);
}

// The stretch of refs that this thread of 1024 owns: a multiple of 4 pages long.
__device__ __forceinline__ void pg_stretch(int pages, int& beg, int& end) {
  const int per = (((pages + kPgMax - 1) / kPgMax) + 3) & ~3;
  const long long b = (long long)per * threadIdx.x;
  beg = (int)(b < pages ? b : pages);
  end = (int)(b + per < pages ? b + per : pages);
}

// refs[p .. p + 3] of a stretch; pages behind its end count as held (1).
__device__ __forceinline__ int4 pg_refs4(const int* refs, int p, int end) {
  if (p + 4 <= end && (reinterpret_cast<uintptr_t>(refs + p) & 15u) == 0)
    return *reinterpret_cast<const int4*>(refs + p);
  int4 v = make_int4(1, 1, 1, 1);
  if (p < end) v.x = refs[p];
  if (p + 1 < end) v.y = refs[p + 1];
  if (p + 2 < end) v.z = refs[p + 2];
  if (p + 3 < end) v.w = refs[p + 3];
  return v;
}

// The free pages of a stretch: as bits where 64 cover it, else read again for
// each walk.
struct PgFree {
  int beg, end;
  unsigned long long bits;
  int count;
};
__device__ __forceinline__ PgFree pg_free_pages(const int* refs, int pages) {
  PgFree f;
  pg_stretch(pages, f.beg, f.end);
  f.bits = 0;
  f.count = 0;
  const bool few = f.end - f.beg <= 64;
  for (int p = f.beg; p < f.end; p += 4) {
    const int4 v = pg_refs4(refs, p, f.end);
    const unsigned m = (v.x == 0) | (v.y == 0) << 1 | (v.z == 0) << 2 | (v.w == 0) << 3;
    f.count += __popc(m);
    if (few) f.bits |= (unsigned long long)m << (p - f.beg);
  }
  return f;
}
// take(rank, page) for the free pages of the stretch, the first of which has
// rank `rank`, as far as ranks below `asked` go.
template <typename F>
__device__ __forceinline__ void pg_walk(const PgFree& f, const int* refs, int rank, int asked, F take) {
  if (f.end - f.beg <= 64) {
    for (unsigned long long m = f.bits; m != 0 && rank < asked; m &= m - 1) take(rank++, f.beg + __ffsll(m) - 1);
    return;
  }
  for (int p = f.beg; p < f.end && rank < asked; ++p)
    if (refs[p] == 0) take(rank++, p);
}

// First index t from `lo` on with incl[t] > k (incl ascending, n entries, incl[n - 1] > k).
__device__ __forceinline__ int pg_owner(const int* incl, int n, int k, int lo) {
  if (incl[lo] > k) return lo;
  int hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (incl[mid] > k) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// Of the threads that hold the same row, the lowest owns it.  All threads of
// the CTA call it; row < 0 takes no part.  keys / first: kPgHash ints each.
__device__ __forceinline__ bool pg_owns_row(int row, int* keys, int* first) {
  for (int i = threadIdx.x; i < kPgHash; i += blockDim.x) {
    keys[i] = -1;
    first[i] = 0x7fffffff;
  }
  __syncthreads();
  int slot = -1;
  if (row >= 0) {
    slot = (int)(((unsigned)row * 2654435761u) >> 20);  // 4096 slots for at most 1024 rows: the walk ends
    static_assert(kPgHash == 4096, "the hash keeps 12 bits");
    while (true) {
      const int seen = atomicCAS(&keys[slot], -1, row);
      if (seen == -1 || seen == row) break;
      slot = (slot + 1) & (kPgHash - 1);
    }
    atomicMin(&first[slot], (int)threadIdx.x);
  }
  __syncthreads();
  return row >= 0 && first[slot] == (int)threadIdx.x;
}

struct PgShared {
  int keys[kPgHash];
  int first[kPgHash];
  int incl[kPgMax];
  int sums[32];
};

// ---------------------------------------------------------------------------
// take: row rows[t] grows to new_lens[t] tokens
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kPgMax, 1)
    take_pages_kernel(const PageTables a, const int* __restrict__ rows, const int* __restrict__ new_lens, int n,
                      int* __restrict__ done_out) {
  __shared__ PgShared s;
  griddep_wait();
  griddep_launch_dependents();
  const int t = threadIdx.x;
  int row = -1, len = 0, want = 0;
  if (t < n) {
    row = rows[t];
    want = new_lens[t];
    if (row < -1 || row >= a.rows) {
      raise_error(a.err, ERR_BAD_INDEX);
      row = -1;
    }
  }
  bool ok = pg_owns_row(row, s.keys, s.first);
  int held = 0, need = 0;
  if (ok) {
    len = a.lens[row];
    held = len / a.page + (len % a.page > 0);
    const int to = want / a.page + (want % a.page > 0);
    ok = len >= 0 && want >= len && to <= a.width;
    need = ok ? to - held : 0;
  }
  int asked, free_pages;
  const PgFree f = pg_free_pages(a.refs, a.pages);
  const int incl = pg_scan(need, s.sums, asked);
  s.incl[t] = incl;
  const int rank = pg_scan(f.count, s.sums, free_pages) - f.count;
  // a row is served when the needs up to and with its own fit the free pages
  const bool done = ok && (need == 0 || incl <= free_pages);
  if (t < n) done_out[t] = done;
  // what each request writes: its row (or -1) and the place of its first page
  s.keys[t] = done && need > 0 ? row : -1;
  s.first[t] = held - (incl - need);
  if (done) a.lens[row] = want;
  __syncthreads();
  int o = 0;
  pg_walk(f, a.refs, rank, asked, [&](int k, int p) {
    o = pg_owner(s.incl, kPgMax, k, o);
    if (s.keys[o] < 0) return;
    a.tables[(long long)s.keys[o] * a.stride + s.first[o] + k] = p;
    a.refs[p] = 1;
  });
}

// ---------------------------------------------------------------------------
// free: every entry of rows[i] gives its page back, once however often the
// row is listed (the exchange empties the entry for whoever comes second)
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kPgThreads) free_pages_kernel(const PageTables a, const int* __restrict__ rows) {
  griddep_wait();
  griddep_launch_dependents();
  const int row = rows[blockIdx.x];
  if (row < 0 || row >= a.rows) {
    if (row != -1 && threadIdx.x == 0) raise_error(a.err, ERR_BAD_INDEX);
    return;
  }
  for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
    int* e = a.tables + (long long)row * a.stride + c;
    if (*e == -1) continue;  // (only ever turned to -1 in this launch)
    const int p = atomicExch(e, -1);
    if (p == -1) continue;
    if (p < 0 || p >= a.pages) {
      raise_error(a.err, ERR_BAD_INDEX);
      continue;
    }
    if (atomicSub(&a.refs[p], 1) <= 0) {  // a page that nobody held: left as it was
      atomicAdd(&a.refs[p], 1);
      raise_error(a.err, ERR_BAD_INDEX);
    }
  }
  if (threadIdx.x == 0) a.lens[row] = 0;
}

// ---------------------------------------------------------------------------
// fork, decisions: child children[t] becomes a copy of parent parents[t]
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kPgMax, 1)
    fork_plan_kernel(const PageTables a, const int* __restrict__ parents, const int* __restrict__ children, int n,
                     int* __restrict__ plan, int* __restrict__ done_out) {
  __shared__ PgShared s;
  griddep_wait();
  griddep_launch_dependents();
  const int t = threadIdx.x;
  int parent = -1, child = -1;
  if (t < n) {
    parent = parents[t];
    child = children[t];
    if (parent < -1 || parent >= a.rows || child < -1 || child >= a.rows) {
      raise_error(a.err, ERR_BAD_INDEX);
      parent = -1;
    }
    if (parent < 0) child = -1;
  }
  bool ok = pg_owns_row(child, s.keys, s.first);
  int len = 0, full = 0, part = 0, last = -1;
  if (ok) {
    len = a.lens[parent];
    ok = a.lens[child] == 0;  // a row that still holds pages would lose them
    if (ok && (len < 0 || (long long)len > (long long)a.width * a.page)) {
      raise_error(a.err, ERR_BAD_INDEX);
      ok = false;
    }
    if (ok) {
      full = len / a.page;
      part = len - full * a.page;
      if (part > 0) {
        last = a.tables[(long long)parent * a.stride + full];
        if (last < 0 || last >= a.pages) {
          raise_error(a.err, ERR_BAD_INDEX);
          ok = false;
        }
      }
    }
  }
  const int need = ok && part > 0;
  int asked, free_pages;
  const PgFree f = pg_free_pages(a.refs, a.pages);
  const int incl = pg_scan(need, s.sums, asked);
  s.incl[t] = incl;
  const int rank = pg_scan(f.count, s.sums, free_pages) - f.count;
  const bool done = ok && (!need || incl <= free_pages);
  if (t < n) {
    done_out[t] = done;
    int4* out = reinterpret_cast<int4*>(plan) + t;
    *out = make_int4(last, -1, done && need ? part : 0, done ? full : -1);
  }
  // every length was read before the scans' barriers: parents count as they came in
  if (done) a.lens[child] = len;
  s.keys[t] = done && need;
  __syncthreads();
  int o = 0;
  pg_walk(f, a.refs, rank, asked, [&](int k, int p) {
    o = pg_owner(s.incl, kPgMax, k, o);
    if (!s.keys[o]) return;
    plan[o * kPgPlanWords + 1] = p;
    a.refs[p] = 1;
  });
}

// ---------------------------------------------------------------------------
// contents
// ---------------------------------------------------------------------------
// One piece of a page's head, all loads of a thread in flight before its first store.
__device__ __forceinline__ void pg_copy_piece(const uint4* src, uint4* dst, int vecs) {
  constexpr int kEach = kPgPieceVecs / kPgThreads;
  uint4 v[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (threadIdx.x + i * kPgThreads < vecs) v[i] = src[threadIdx.x + i * kPgThreads];
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (threadIdx.x + i * kPgThreads < vecs) dst[threadIdx.x + i * kPgThreads] = v[i];
}

__device__ __forceinline__ long long pg_plane(const PageCache& c, int plane) {
  return (long long)(plane / c.n1) * c.s0 + (long long)(plane % c.n1) * c.s1;
}

// Piece w of the copy of `tokens` slots of page src into page dst (all planes, plane by plane).
__device__ __forceinline__ void pg_copy_unit(const PageCache& c, int src, int dst, int tokens, int unit, int pieces) {
  const int plane = unit / pieces, piece = unit - plane * pieces;
  const int vecs = tokens * c.slot_vecs - piece * kPgPieceVecs;
  if (vecs <= 0) return;
  uint4* at = c.base + pg_plane(c, plane) + (long long)piece * kPgPieceVecs;
  pg_copy_piece(at + (long long)src * c.page_stride, at + (long long)dst * c.page_stride, min(vecs, kPgPieceVecs));
}

__global__ void __launch_bounds__(kPgThreads)
    copy_pages_kernel(const PageCache c, const int* __restrict__ src, const int* __restrict__ dst,
                      const int* __restrict__ tokens, int n, int pages, int page, unsigned* err) {
  griddep_wait();
  griddep_launch_dependents();
  const int pieces = (c.page_vecs + kPgPieceVecs - 1) / kPgPieceVecs;
  const int per = c.planes * pieces;
  const long long units = (long long)n * per;
  for (long long w = blockIdx.x; w < units; w += gridDim.x) {
    const int i = (int)(w / per), unit = (int)(w - (long long)i * per);
    const int a = src[i], b = dst[i];
    if (a == -1 || b == -1) continue;
    int m = tokens ? tokens[i] : page;
    if (a < 0 || a >= pages || b < 0 || b >= pages || m < 0 || m > page) {
      if (unit == 0 && threadIdx.x == 0) raise_error(err, ERR_BAD_INDEX);
      continue;
    }
    if (a != b) pg_copy_unit(c, a, b, m, unit, pieces);
  }
}

// fork, contents: the children's tables and the references of the shared pages (units [0, n)), then the last pages
__global__ void __launch_bounds__(kPgThreads)
    fork_apply_kernel(const PageTables a, const PageCache c, const int* __restrict__ parents,
                      const int* __restrict__ children, int n, const int* __restrict__ plan) {
  griddep_wait();
  griddep_launch_dependents();
  const int pieces = (c.page_vecs + kPgPieceVecs - 1) / kPgPieceVecs;
  const int per = c.planes * pieces;
  const long long units = n + (long long)n * per;
  for (long long w = blockIdx.x; w < units; w += gridDim.x) {
    if (w < n) {
      const int4 p = reinterpret_cast<const int4*>(plan)[w];
      if (p.w < 0) continue;
      const int* from = a.tables + (long long)parents[w] * a.stride;
      int* to = a.tables + (long long)children[w] * a.stride;
      for (int col = threadIdx.x; col < p.w; col += kPgThreads) {
        const int e = from[col];
        if (e < 0 || e >= a.pages) {
          raise_error(a.err, ERR_BAD_INDEX);
          continue;
        }
        to[col] = e;
        atomicAdd(&a.refs[e], 1);
      }
      if (threadIdx.x == 0 && p.z > 0) to[p.w] = p.y;
      continue;
    }
    const int i = (int)((w - n) / per), unit = (int)(w - n - (long long)i * per);
    const int4 p = reinterpret_cast<const int4*>(plan)[i];
    if (p.z > 0) pg_copy_unit(c, p.x, p.y, p.z, unit, pieces);
  }
}

// ---------------------------------------------------------------------------
// compact, decisions: with n live pages, the k-th live page behind the first
// n places moves into the k-th free one of them.  place[p]: where page p's
// contents are afterwards (-1: free); moves: {count, then (from, to) pairs}
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kPgMax, 1)
    compact_plan_kernel(const PageTables a, int* __restrict__ place, int* __restrict__ moves) {
  __shared__ int sums[32];
  __shared__ int s_holes;
  griddep_wait();
  griddep_launch_dependents();
  int free_pages;
  const PgFree mine = pg_free_pages(a.refs, a.pages);
  const int beg = mine.beg, end = mine.end;
  const bool few = end - beg <= 64;
  auto free_at = [&](int p) { return few ? (mine.bits >> (p - beg) & 1) != 0 : a.refs[p] == 0; };
  const int before = pg_scan(mine.count, sums, free_pages) - mine.count;  // free pages before the stretch
  const int live = a.pages - free_pages;
  // holes: free pages among the first `live` places
  if (threadIdx.x == 0 && live == a.pages) s_holes = 0;
  if (beg <= live && live < end) {
    int h = before;
    for (int p = beg; p < live; ++p) h += free_at(p);
    s_holes = h;
  }
  __syncthreads();
  const int holes = s_holes;
  if (threadIdx.x == 0) moves[0] = holes;
  int f = before;
  for (int p = beg; p < end; ++p) {
    const bool is_free = free_at(p);
    if (p < live) {
      if (is_free) moves[2 + 2 * f + 1] = p;  // the f-th hole
      place[p] = is_free ? -1 : p;
    } else {
      // live pages of [live, p): those before p less the ones of the first places
      if (!is_free) moves[2 + 2 * ((p - f) - (live - holes))] = p;
      if (is_free) place[p] = -1;
    }
    f += is_free;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < holes; k += blockDim.x) {
    const int from = moves[2 + 2 * k], to = moves[2 + 2 * k + 1];
    place[from] = to;
    a.refs[to] = a.refs[from];
    a.refs[from] = 0;
  }
}

// compact, contents: tables (units of kPgThreads entries), then the moved pages
__global__ void __launch_bounds__(kPgThreads)
    compact_apply_kernel(const PageTables a, const PageCache c, const int* __restrict__ place,
                         const int* __restrict__ moves) {
  griddep_wait();
  griddep_launch_dependents();
  const int pieces = (c.page_vecs + kPgPieceVecs - 1) / kPgPieceVecs;
  const int per = c.planes * pieces;
  const int count = moves[0];
  const long long entries = (long long)a.rows * a.width;
  const long long table_units = (entries + kPgThreads - 1) / kPgThreads;
  const long long units = table_units + (long long)count * per;
  for (long long w = blockIdx.x; w < units; w += gridDim.x) {
    if (w < table_units) {
      const long long i = w * kPgThreads + threadIdx.x;
      if (i >= entries || count == 0) continue;
      int* e = a.tables + (i / a.width) * a.stride + i % a.width;
      const int p = *e;
      if (p == -1) continue;
      const int to = p >= 0 && p < a.pages ? place[p] : -1;
      if (to < 0) raise_error(a.err, ERR_BAD_INDEX);  // no page, or a free one: left as it was
      else if (to != p) *e = to;
      continue;
    }
    const long long u = w - table_units;
    const int i = (int)(u / per), unit = (int)(u - (long long)i * per);
    pg_copy_unit(c, moves[2 + 2 * i], moves[2 + 2 * i + 1], a.page, unit, pieces);
  }
}

}  // namespace b200
