// Pages of a cache for gfx950: forking, growing, shrinking and freeing sequences, and compaction.
//
// Which pages are free is kept in one place, the counts (0: free), so a call begins by compacting the
// indices of free pages: the counts are tallied in spans, a second launch adds up the spans before
// its own and writes the indices in ascending order, as far as they are wanted.  Requests are served
// by a prefix sum over what they want; request i takes free pages start[i] .. start[i] + need[i] - 1.
// Nothing depends on the order in which workgroups run.
//
// What bounds it: with data to move, memory, each byte read and written once (500 forks of 48 pools,
// 786 MB: 153 us of copying, 5.1 TB/s, and 14 us of the launches before it; 16 KiB a workgroup at a time,
// four 16-byte loads of a thread in flight).  Without, the launches: 1500 sequences freed and replaced on
// 2^20 pages 27.4 us in five, of which listing 4 MB of counts is 6; a cache of up to 8192 pages with up to
// 64 requests is planned by one workgroup in one launch (9 sequences replaced on 300 pages: three launches
// instead of five, 16 us instead of 24 when that was done).  Every request is compared with all before it:
// 16384 take 66 us, 65536 387.
#include "lm_types.h"

namespace tcd {

constexpr int kPageBlock = 256;
constexpr int kPagesPerThread = 8;
constexpr int kPageSweep = kPageBlock * kPagesPerThread;  // counts that a workgroup looks at in one go
constexpr int kCopyUnit = kPageBlock * 16 * 4;            // bytes that a workgroup copies in one go
constexpr int kMaxSpans = 8192;
constexpr int64_t kMaxRequests = (int64_t(1) << 23);  // a launch counts its threads in 32 bits, 256 of them a request
constexpr int kRequestWaves = kPageBlock / kWave;
// A cache of this size with this many requests is planned by one workgroup of 16 wavefronts: a launch
// costs the host about 3 us and the device 2 us, the loops over pages and requests less than that.
constexpr int kSmallBlock = 1024;
constexpr int kSmallPages = kSmallBlock * kPagesPerThread;
constexpr int kSmallRequests = kWave;

struct PageCache {
  const uint64_t* pools;
  int64_t page_bytes;
  int num_pools, num_pages, page_size, num_sequences, max_pages;
  int32_t* tables;
  int32_t* lengths;
  int32_t* refs;
};

// the temporary storage of a call
struct PageTemp {
  int64_t* head;       // [0] moves of a compaction, [1] free pages
  int32_t* span_free;  // free pages of each span
  int32_t* need;       // pages a request wants; -1: refused
  int64_t* start;      // pages wanted by the requests before it
  int32_t* copied;     // resize: the page that a growing sequence gets a copy of; -1: none; -2 - j: it keeps a shared
                       // page if request j, the last one that leaves it, is served
  int32_t* free_list;  // free pages, ascending; a compaction's holes
  int32_t* movers;     // a compaction's pages that move, descending, and their counts
  int32_t* mover_refs;
  int32_t* place;      // page -> its index among the movers, -1: none
  int spans, span;
};

__device__ inline int clamped_length(const PageCache& c, int s) {
  const int64_t most = (int64_t)c.max_pages * c.page_size;
  const int64_t n = c.lengths[s];
  return (int)(n < 0 ? 0 : n > most ? most : n);
}
__device__ inline int pages_of(const PageCache& c, int length) { return (int)(((int64_t)length + c.page_size - 1) / c.page_size); }
__device__ inline bool is_page(const PageCache& c, int q) { return q >= 0 && q < c.num_pages; }
__device__ inline void add_count(const PageCache& c, int q, int v) { atomicAdd(reinterpret_cast<uint32_t*>(c.refs) + q, (uint32_t)v); }

// ---------------------------------------------------------------------------------------
// Sums over the workgroup
// ---------------------------------------------------------------------------------------
template <int BLOCK>
struct BlockSum {
  static constexpr int kThreads = BLOCK;
  int64_t wave_total[BLOCK / kWave];
};
// exclusive prefix of v over the threads, and the total
template <int BLOCK, class T>
__device__ inline T block_exclusive(BlockSum<BLOCK>& sm, T v, T& total) {
  const int w = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const T incl = wave_inclusive_scan(v, T(0), [](T a, T b) { return a + b; });
  __syncthreads();  // the last call's totals have been read
  if (lane == kWave - 1) sm.wave_total[w] = incl;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < BLOCK / kWave; k++) {
    if (k < w) before += (T)sm.wave_total[k];
    total += (T)sm.wave_total[k];
  }
  return before + incl - v;
}
// the sum of the positive ones of n values, the same in all threads
template <int BLOCK>
__device__ inline int64_t block_sum(BlockSum<BLOCK>& sm, const int32_t* v, int64_t n) {
  constexpr int N = 8;  // values of a thread in flight
  int64_t mine = 0, total;
  for (int64_t i = threadIdx.x; i < n; i += N * BLOCK) {
    int u[N];
#pragma unroll
    for (int k = 0; k < N; k++) u[k] = v[i + k * BLOCK < n ? i + k * BLOCK : i];
#pragma unroll
    for (int k = 0; k < N; k++) mine += i + k * BLOCK < n && u[k] > 0 ? u[k] : 0;
  }
  block_exclusive(sm, mine, total);
  return total;
}

// ---------------------------------------------------------------------------------------
// Free pages
// ---------------------------------------------------------------------------------------
__device__ inline void tally_span(const PageCache& c, const PageTemp& t, int span) {
  __shared__ BlockSum<kPageBlock> sm;
  const int64_t begin = (int64_t)span * t.span;
  const int64_t end = begin + t.span < c.num_pages ? begin + t.span : c.num_pages;
  int mine = 0;
  for (int64_t q = begin + threadIdx.x; q < end; q += kPageBlock) mine += c.refs[q] == 0;
  int total;
  block_exclusive(sm, mine, total);
  if (threadIdx.x == 0) t.span_free[span] = total;
}

// f(q, count, free pages before q) for every page of a span, by the whole workgroup
template <int BLOCK, class F>
__device__ inline void sweep_span(const PageCache& c, const PageTemp& t, BlockSum<BLOCK>& sm, int span, int64_t before, F f) {
  const int64_t begin = (int64_t)span * t.span;
  const int64_t end = begin + t.span < c.num_pages ? begin + t.span : c.num_pages;
  for (int64_t at = begin; at < end; at += BLOCK * kPagesPerThread) {
    int n[kPagesPerThread];
    const int64_t q0 = at + (int64_t)threadIdx.x * kPagesPerThread;
    int mine = 0;
#pragma unroll
    for (int k = 0; k < kPagesPerThread; k++) {
      n[k] = q0 + k < end ? c.refs[q0 + k] : 1;
      mine += n[k] == 0;
    }
    int total;
    int64_t rank = before + block_exclusive(sm, mine, total);
#pragma unroll
    for (int k = 0; k < kPagesPerThread; k++) {
      if (q0 + k < end) f(q0 + k, n[k], rank);
      rank += n[k] == 0;
    }
    before += total;
  }
}

// f(q, count, free pages before q, free pages) for every page of a small cache
template <int BLOCK, class F>
__device__ inline int64_t sweep_once(const PageCache& c, BlockSum<BLOCK>& sm, F f) {
  int n[kPagesPerThread];
  const int q0 = (int)threadIdx.x * kPagesPerThread;
  int mine = 0;
#pragma unroll
  for (int k = 0; k < kPagesPerThread; k++) n[k] = q0 + k < c.num_pages ? c.refs[q0 + k] : 1;
#pragma unroll
  for (int k = 0; k < kPagesPerThread; k++) mine += n[k] == 0;
  int total;
  int rank = block_exclusive(sm, mine, total);
#pragma unroll
  for (int k = 0; k < kPagesPerThread; k++) {
    if (q0 + k < c.num_pages) f(q0 + k, n[k], rank, total);
    rank += n[k] == 0;
  }
  return total;
}

// ---------------------------------------------------------------------------------------
// Requests
// ---------------------------------------------------------------------------------------
// whether an earlier request names the same sequence (all lanes of a wavefront ask for the same one):
// 16 bytes a lane and four of them in flight, 1024 requests a trip
__device__ inline bool named_before(const int32_t* named, int64_t i, int s) {
  bool found = false;
  if (i < 4) {
    if (lane_id() < i) found = named[lane_id()] == s;
  } else {
    for (int64_t q0 = (int64_t)lane_id() * 4; q0 < i; q0 += 4 * 4 * kWave) {
      tcd_v4u v[4];  // behind the end, the last four again
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int64_t q = q0 + k * 4 * kWave;
        v[k] = *reinterpret_cast<const tcd_v4u_anywhere*>(named + (q + 4 <= i ? q : i - 4));
      }
#pragma unroll
      for (int k = 0; k < 4; k++)
        found = found || (int)v[k][0] == s || (int)v[k][1] == s || (int)v[k][2] == s || (int)v[k][3] == s;
    }
  }
  return __ballot(found) != 0;
}

enum : int { kFork = 0, kForkShared = 1, kResize = 2 };

struct Requests {
  const int32_t* first;   // parents, or the lengths of a resize (NULL: 0)
  const int32_t* named;   // children, or the sequences of a resize
  int64_t n;
  int kind;
  uint8_t* done;
};

__device__ inline bool valid_resize(const PageCache& c, int s, int64_t want) {
  return s >= 0 && s < c.num_sequences && want >= 0 && want <= (int64_t)c.max_pages * c.page_size;
}
// Shrinks and frees, a wavefront for a sequence.
__device__ inline void shrink_rows(const PageCache& c, int s, int want) {
  const int lane = lane_id();
  const int old = __builtin_amdgcn_readfirstlane(clamped_length(c, s));
  if (want >= old) return;
  int32_t* row = c.tables + (int64_t)s * c.max_pages;
  constexpr int N = 4;  // entries of a lane in flight
  const int end = pages_of(c, old);
  for (int j0 = pages_of(c, want) + lane; j0 < end; j0 += N * kWave) {
    int q[N];
#pragma unroll
    for (int k = 0; k < N; k++) q[k] = row[j0 + k * kWave < end ? j0 + k * kWave : j0];
#pragma unroll
    for (int k = 0; k < N; k++) {
      if (j0 + k * kWave < end) {
        if (is_page(c, q[k])) add_count(c, q[k], -1);
        row[j0 + k * kWave] = -1;
      }
    }
  }
  if (lane == 0) c.lengths[s] = want;
}
// need[i] = 0, or -1 where the request is refused
__device__ inline void shrink(const PageCache& c, const PageTemp& t, const Requests& r, int64_t i) {
  const int s = r.named[i], want = r.first ? r.first[i] : 0;
  const bool ok = valid_resize(c, s, want) && !named_before(r.named, i, s);
  if (lane_id() == 0) {
    if (t.need) t.need[i] = ok ? 0 : -1;
    else if (r.done) r.done[i] = ok;  // pages_free: nothing is left to do
  }
  if (ok) shrink_rows(c, s, want);
}
__global__ __launch_bounds__(kPageBlock) void pages_shrink_kernel(PageCache c, PageTemp t, Requests r) {
  const int64_t i = (int64_t)blockIdx.x * kRequestWaves + threadIdx.x / kWave;
  if (i < r.n) shrink(c, t, r, i);
}

// The last page of a growing sequence when others name it too and something of it is free.  Requests are
// served in their order: each that grows into a page gets a copy and leaves it, until the one whose turn
// comes is alone with it and keeps it.  So with n names before the call, the n-th that grows into it keeps it;
// but for that all before it must be served, and those which copy are refused from one on.
__device__ inline int shared_page(const PageCache& c, int s, int old, int want) {
  if (want <= old || old % c.page_size == 0) return -1;
  const int q = c.tables[(int64_t)s * c.max_pages + old / c.page_size];
  return is_page(c, q) && c.refs[q] > 1 ? q : -1;
}

__device__ inline int shared_page(const PageCache& c, const Requests& r, int64_t i) {
  return shared_page(c, r.named[i], clamped_length(c, r.named[i]), r.first[i]);
}
// What becomes of it: `before` requests grow into it earlier in the call, the last of them `last`.
__device__ inline int copied_page(const PageCache& c, int q, int before, int last) {
  return q < 0 ? -1 : before < c.refs[q] - 1 ? q : -2 - last;
}
// What a valid resize wants
__device__ inline int wanted_by_resize(const PageCache& c, const Requests& r, int64_t i, int copied) {
  const int old = clamped_length(c, r.named[i]), want = r.first[i];
  return want <= old ? 0 : pages_of(c, want) - pages_of(c, old) + (copied >= 0);
}
// The same by a wavefront for one of many requests.  need[j] is replaced meanwhile by what request j wants, but
// stays -1 where it is refused.
__device__ inline bool refused(const PageTemp& t, int64_t j) { return (int)ld_agent(reinterpret_cast<const uint32_t*>(t.need + j)) < 0; }
__device__ inline void plan_resize(const PageCache& c, const PageTemp& t, const Requests& r, int64_t i) {
  if (refused(t, i)) return;
  const int q = __builtin_amdgcn_readfirstlane(shared_page(c, r, i));
  int before = 0, last = -1;
  if (q >= 0) {  // rare: a sequence was cut back into what it shares
    for (int64_t j0 = 0; j0 < i; j0 += kWave) {
      const int64_t j = j0 + lane_id();
      const uint64_t same = __ballot(j < i && !refused(t, j) && shared_page(c, r, j) == q);
      before += __popcll(same);
      if (same) last = (int)(j0 + kWave - 1 - __builtin_clzll(same));
    }
  }
  if (lane_id() == 0) {
    const int copied = copied_page(c, q, before, last);
    t.copied[i] = copied;
    st_agent(reinterpret_cast<uint32_t*>(t.need + i), (uint32_t)wanted_by_resize(c, r, i, copied));
  }
}
// What a fork wants that names its child first and no parent as child; -1: refused.
__device__ inline int wanted_by_fork(const PageCache& c, int kind, int parent, int child) {
  if (c.lengths[child] != 0) return -1;
  const int n = clamped_length(c, parent);
  return kind == kForkShared ? (n % c.page_size != 0) : pages_of(c, n);
}
__device__ inline bool valid_fork(const PageCache& c, int parent, int child) {
  return parent >= 0 && parent < c.num_sequences && child >= 0 && child < c.num_sequences;
}

// Tallies the free pages and what each request wants.
__global__ __launch_bounds__(kPageBlock) void pages_tally_kernel(PageCache c, PageTemp t, Requests r) {
  if ((int)blockIdx.x < t.spans) return tally_span(c, t, (int)blockIdx.x);
  const int64_t i = (int64_t)(blockIdx.x - t.spans) * kRequestWaves + threadIdx.x / kWave;  // a wavefront for a request
  if (i >= r.n) return;
  if (r.kind == kResize) {
    plan_resize(c, t, r, i);
  } else {
    const int parent = r.first[i], child = r.named[i];
    const bool ok = valid_fork(c, parent, child) && !named_before(r.named, i, child) && !named_before(r.first, r.n, child);
    if (lane_id() == 0) t.need[i] = ok ? wanted_by_fork(c, r.kind, parent, child) : -1;
  }
}

// Lists the free pages, as many as are wanted, and adds up the requests.
__global__ __launch_bounds__(kPageBlock) void pages_list_kernel(PageCache c, PageTemp t, int64_t n) {
  __shared__ BlockSum<kPageBlock> sm;
  if ((int)blockIdx.x == t.spans) {
    constexpr int N = 8;  // requests of a thread, next to one another
    int64_t sum = 0;
    for (int64_t at = 0; at < n; at += N * kPageBlock) {
      const int64_t i0 = at + (int64_t)threadIdx.x * N;
      int need[N];
      int64_t mine = 0, total;
#pragma unroll
      for (int k = 0; k < N; k++) need[k] = t.need[i0 + k < n ? i0 + k : n - 1];
#pragma unroll
      for (int k = 0; k < N; k++) mine += need[k] = i0 + k < n && need[k] > 0 ? need[k] : 0;
      int64_t start = sum + block_exclusive(sm, mine, total);
#pragma unroll
      for (int k = 0; k < N; k++) {
        if (i0 + k < n) t.start[i0 + k] = start;
        start += need[k];
      }
      sum += total;
    }
    const int64_t free = block_sum(sm, t.span_free, t.spans);
    if (threadIdx.x == 0) t.head[1] = free;
    return;
  }
  const int64_t before = block_sum(sm, t.span_free, blockIdx.x);
  const int64_t wanted = block_sum(sm, t.need, n);
  if (before >= wanted) return;
  sweep_span(c, t, sm, (int)blockIdx.x, before, [&](int64_t q, int count, int64_t rank) {
    if (count == 0 && rank < wanted) t.free_list[rank] = (int)q;
  });
}

// All of that for a small cache and up to 64 requests, in one workgroup instead of two or three
// launches.  The first wavefront has a request in each lane and compares them in registers.
__global__ __launch_bounds__(kSmallBlock) void pages_plan_small_kernel(PageCache c, PageTemp t, Requests r) {
  __shared__ BlockSum<kSmallBlock> sm;
  __shared__ int s_need[kWave];
  const int w = threadIdx.x / kWave, i = threadIdx.x, n = (int)r.n;
  if (w == 0) {
    const int first = r.first[i < n ? i : 0], named = r.named[i < n ? i : 0];
    bool again = false, parent = false;
    for (int j = 0; j < n; j++) {
      const int child_j = __builtin_amdgcn_readlane(named, j), first_j = __builtin_amdgcn_readlane(first, j);
      again = again || (j < i && child_j == named);
      parent = parent || first_j == named;
    }
    int need = -1;
    if (i < n && !again) {
      if (r.kind == kResize) need = valid_resize(c, named, first) ? 0 : -1;
      else if (!parent && valid_fork(c, first, named)) need = wanted_by_fork(c, r.kind, first, named);
    }
    s_need[i] = need;
  }
  __syncthreads();
  if (r.kind == kResize) {
    for (int k = w; k < n; k += kSmallBlock / kWave)
      if (s_need[k] == 0) shrink_rows(c, r.named[k], r.first[k]);
    __threadfence();  // lengths, tables and counts are read by other wavefronts below
    __syncthreads();
  }
  int need = i < n ? s_need[i] : 0;
  if (r.kind == kResize && w == 0) {
    const bool valid = i < n && need == 0;
    const int q = valid ? shared_page(c, r, i) : -1;
    int before = 0, last = -1;
    if (__ballot(q >= 0)) {
      for (int j = 0; j < n; j++) {
        const bool same = __builtin_amdgcn_readlane(q, j) == q && j < i;
        before += same;
        if (same) last = j;
      }
    }
    if (valid) {
      const int copied = copied_page(c, q, before, last);
      t.copied[i] = copied;
      need = wanted_by_resize(c, r, i, copied);
    }
  }
  if (i < n) t.need[i] = need;
  int64_t wanted;
  const int64_t start = block_exclusive(sm, (int64_t)(need > 0 ? need : 0), wanted);
  if (i < n) t.start[i] = start;
  const int64_t free = sweep_once(c, sm, [&](int q, int count, int rank, int) {
    if (count == 0 && rank < wanted) t.free_list[rank] = q;
  });
  if (i == 0) t.head[1] = free;
}

// bytes [at, at + n) of a page, n <= kCopyUnit, by the whole workgroup
__device__ inline void copy_unit(const char* from, char* to, int64_t at, int64_t n) {
  const int nvec = (int)(n / 16);
  tcd_v4u v[4];
  if (n == kCopyUnit) {
#pragma unroll
    for (int k = 0; k < 4; k++)
      v[k] = __builtin_nontemporal_load(reinterpret_cast<const tcd_v4u_anywhere*>(from + at + (threadIdx.x + k * kPageBlock) * 16));
#pragma unroll
    for (int k = 0; k < 4; k++)
      __builtin_nontemporal_store(v[k], reinterpret_cast<tcd_v4u_anywhere*>(to + at + (threadIdx.x + k * kPageBlock) * 16));
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int64_t i = threadIdx.x + k * kPageBlock;
    if (i < nvec) v[k] = __builtin_nontemporal_load(reinterpret_cast<const tcd_v4u_anywhere*>(from + at + i * 16));
  }
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int64_t i = threadIdx.x + k * kPageBlock;
    if (i < nvec) __builtin_nontemporal_store(v[k], reinterpret_cast<tcd_v4u_anywhere*>(to + at + i * 16));
  }
  for (int64_t i = (int64_t)nvec * 16 + threadIdx.x; i < n; i += kPageBlock) to[at + i] = from[at + i];
}
__device__ inline void copy_page_unit(const PageCache& c, int pool, int from, int to, int64_t unit) {
  const int64_t at = unit * kCopyUnit;
  const int64_t n = c.page_bytes - at < kCopyUnit ? c.page_bytes - at : kCopyUnit;
  char* base = reinterpret_cast<char*>(c.pools[pool]);
  copy_unit(base + (int64_t)from * c.page_bytes, base + (int64_t)to * c.page_bytes, at, n);
}

// Serves the requests: workgroup (request, piece); piece 0 writes tables, counts and lengths, all of them copy.
__global__ __launch_bounds__(kPageBlock) void pages_serve_kernel(PageCache c, PageTemp t, Requests r, int pieces) {
  const int64_t i = blockIdx.x / (unsigned)pieces;
  const int piece = (int)(blockIdx.x % (unsigned)pieces);
  const int need = t.need[i];
  const int64_t start = t.start[i];
  const auto served = [&](int need, int64_t start) { return need == 0 || (need > 0 && start + need <= t.head[1]); };
  bool ok = served(need, start);
  if (ok && r.kind == kResize && t.copied[i] <= -2) ok = served(t.need[-2 - t.copied[i]], t.start[-2 - t.copied[i]]);
  if (piece == 0 && threadIdx.x == 0 && r.done) r.done[i] = ok;
  if (!ok) return;
  const int32_t* mine = t.free_list + start;
  const int s = r.named[i];
  int32_t* row = c.tables + (int64_t)s * c.max_pages;
  const int64_t units = (c.page_bytes + kCopyUnit - 1) / kCopyUnit;
  if (r.kind == kResize) {
    const int want = r.first[i];
    if (need == 0) {  // it shrank before, or grows within its last page
      if (piece == 0 && threadIdx.x == 0 && want > clamped_length(c, s)) c.lengths[s] = want;
      return;
    }
    const int q = t.copied[i], own = q >= 0;
    if (piece == 0) {
      // its pages from the first one behind the old length: `had` comes from what is wanted, not from the
      // length, which a thread of this workgroup may have replaced
      const int have = pages_of(c, want), had = have - (need - own);
      for (int j = had + (int)threadIdx.x; j < have; j += kPageBlock) {
        const int page = mine[own + j - had];
        row[j] = page;
        c.refs[page] = 1;
      }
      if (threadIdx.x == 0) {
        if (own) {
          row[had - 1] = mine[0];
          c.refs[mine[0]] = 1;
          add_count(c, q, -1);
        }
        c.lengths[s] = want;
      }
    }
    if (own) {
      for (int64_t u = piece; u < units * c.num_pools; u += pieces) copy_page_unit(c, (int)(u / units), q, mine[0], u % units);
    }
    return;
  }
  const int parent = r.first[i];
  const int n = clamped_length(c, parent), held = pages_of(c, n);
  const int32_t* from = c.tables + (int64_t)parent * c.max_pages;
  const int shared = held - need;  // copies are the last pages
  if (piece == 0) {
    for (int j = threadIdx.x; j < held; j += kPageBlock) {
      const int q = j < shared ? from[j] : mine[j - shared];
      row[j] = q;
      if (j >= shared) c.refs[q] = 1;
      else if (is_page(c, q)) add_count(c, q, 1);
    }
    if (threadIdx.x == 0) c.lengths[s] = n;
  }
  const int64_t all = (int64_t)need * c.num_pools * units;
  for (int64_t u = piece; u < all; u += pieces) {
    const int64_t page = u / units;
    const int j = (int)(page / c.num_pools);
    const int q = from[shared + j];
    if (is_page(c, q)) copy_page_unit(c, (int)(page % c.num_pools), q, mine[j], u % units);
  }
}

// ---------------------------------------------------------------------------------------
// Compaction.  With `live` pages in use, the free ones below `live` (holes) are as many as the ones in
// use from there on (movers).  Holes are numbered from below by the free pages before them, movers
// from above by the pages in use behind them; mover k moves to hole k.  No page is both.
// ---------------------------------------------------------------------------------------
__global__ __launch_bounds__(kPageBlock) void pages_tally_only_kernel(PageCache c, PageTemp t) { tally_span(c, t, (int)blockIdx.x); }

__device__ inline void rank_page(const PageTemp& t, int64_t q, int count, int64_t rank, int64_t live, int32_t* refs_out) {
  if (q == live) t.head[0] = rank;  // holes below
  if (q < live) {
    if (count == 0) t.free_list[rank] = (int)q;
    else refs_out[q] = count;
  } else {
    int k = -1;
    if (count != 0) {
      k = (int)(live - 1 - (q - rank));
      t.movers[k] = (int)q;
      t.mover_refs[k] = count;
    }
    t.place[q] = k;
    refs_out[q] = 0;
  }
}
__device__ inline void publish_live(const PageCache& c, const PageTemp& t, int64_t live, int32_t* live_out) {
  *live_out = (int)live;
  if (live == c.num_pages) t.head[0] = 0;  // no page is the first one behind
}
__global__ __launch_bounds__(kPageBlock) void pages_rank_kernel(PageCache c, PageTemp t, int32_t* refs_out, int32_t* live_out) {
  __shared__ BlockSum<kPageBlock> sm;
  const int64_t before = block_sum(sm, t.span_free, blockIdx.x);
  const int64_t live = c.num_pages - block_sum(sm, t.span_free, t.spans);
  if (blockIdx.x == 0 && threadIdx.x == 0) publish_live(c, t, live, live_out);
  sweep_span(c, t, sm, (int)blockIdx.x, before, [&](int64_t q, int count, int64_t rank) { rank_page(t, q, count, rank, live, refs_out); });
}
// The same for a small cache, in one workgroup that needs no tally of spans.
__global__ __launch_bounds__(kSmallBlock) void pages_rank_small_kernel(PageCache c, PageTemp t, int32_t* refs_out, int32_t* live_out) {
  __shared__ BlockSum<kSmallBlock> sm;
  const int64_t free = sweep_once(c, sm, [&](int q, int count, int rank, int total) { rank_page(t, q, count, rank, c.num_pages - total, refs_out); });
  if (threadIdx.x == 0) publish_live(c, t, c.num_pages - free, live_out);
}

__global__ __launch_bounds__(kPageBlock) void pages_move_kernel(PageCache c, PageTemp t, int32_t* tables_out, int32_t* refs_out,
                                                                const int32_t* live_at, int table_blocks) {
  const int live = *live_at;
  if ((int)blockIdx.x < table_blocks) {  // renumbers the tables
    const int64_t all = (int64_t)c.num_sequences * c.max_pages;
    for (int64_t e = (int64_t)blockIdx.x * kPageBlock + threadIdx.x; e < all; e += (int64_t)table_blocks * kPageBlock) {
      int q = c.tables[e];
      if (!is_page(c, q)) q = -1;
      else if (q >= live) {
        const int k = t.place[q];
        q = k >= 0 ? t.free_list[k] : -1;
      }
      tables_out[e] = q;
    }
    return;
  }
  const int64_t moves = t.head[0];
  const int64_t blocks = gridDim.x - table_blocks, block = blockIdx.x - table_blocks;
  for (int64_t k = block * kPageBlock + threadIdx.x; k < moves; k += blocks * kPageBlock) refs_out[t.free_list[k]] = t.mover_refs[k];
  const int64_t units = (c.page_bytes + kCopyUnit - 1) / kCopyUnit, all = moves * c.num_pools * units;
  for (int64_t u = block; u < all; u += blocks) {
    const int64_t page = u / units;
    const int k = (int)(page / c.num_pools);
    copy_page_unit(c, (int)(page % c.num_pools), t.movers[k], t.free_list[k], u % units);
  }
}

// ---------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------
static bool cache_of(const thrust_cdna4_page_cache* a, PageCache& c) {
  if (!a || a->num_pools < 0 || a->num_pages < 0 || a->page_bytes < 0 || a->page_size <= 0 || a->num_sequences < 0 || a->max_pages < 0) return false;
  if ((int64_t)a->max_pages * a->page_size > 0x7fffffff) return false;  // lengths are 32-bit
  c = PageCache{a->pools, a->page_bytes, a->num_pools, a->num_pages, a->page_size, a->num_sequences, a->max_pages, a->tables, a->lengths, a->refs};
  return true;
}
static bool cache_usable(const PageCache& c) {
  return (c.num_pages == 0 || c.refs) && (c.num_sequences == 0 || (c.lengths && (c.max_pages == 0 || c.tables))) &&
         (c.num_pools == 0 || c.page_bytes == 0 || c.pools);
}

// carves the storage; returns its size
static size_t page_temp(const PageCache& c, int64_t n, bool compact, void* temp, PageTemp& t) {
  t.span = (int)(ceil_div(ceil_div(c.num_pages, (int64_t)kMaxSpans), (int64_t)kPageSweep) * kPageSweep);
  if (t.span == 0) t.span = kPageSweep;
  t.spans = (int)ceil_div(c.num_pages, (int64_t)t.span);
  char* base = static_cast<char*>(temp);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* p = base ? base + at : nullptr;
    at += align_up(bytes, 256);
    return p;
  };
  t.head = reinterpret_cast<int64_t*>(take(16));
  t.span_free = reinterpret_cast<int32_t*>(take((size_t)t.spans * 4));
  t.need = reinterpret_cast<int32_t*>(take((size_t)n * 4));
  t.start = reinterpret_cast<int64_t*>(take((size_t)n * 8));
  t.copied = reinterpret_cast<int32_t*>(take((size_t)n * 4));
  t.free_list = reinterpret_cast<int32_t*>(take((size_t)c.num_pages * 4));
  t.movers = t.mover_refs = t.place = nullptr;
  if (compact) {
    t.movers = reinterpret_cast<int32_t*>(take((size_t)c.num_pages * 4));
    t.mover_refs = reinterpret_cast<int32_t*>(take((size_t)c.num_pages * 4));
    t.place = reinterpret_cast<int32_t*>(take((size_t)c.num_pages * 4));
  }
  return at;
}

static hipError_t grant(const PageCache& c, const PageTemp& t, const Requests& r, hipStream_t s) {
  // enough workgroups to fill the device, none without a unit to copy; a resize copies a page at most, and rarely
  const int64_t units = ceil_div(c.page_bytes, (int64_t)kCopyUnit) * c.num_pools * (r.kind == kFork ? c.max_pages : 1);
  int64_t pieces = ceil_div((int64_t)device_cu_count() * (r.kind == kResize ? 2 : 16), r.n);
  if (pieces > units) pieces = units;
  if (pieces < 1) pieces = 1;
  TCD_LAUNCH("pages_serve_kernel", pages_serve_kernel, dim3((unsigned)(r.n * pieces)), dim3(kPageBlock), s, c, t, r, (int)pieces);
  return hipGetLastError();
}

static hipError_t serve(const PageCache& c, const PageTemp& t, const Requests& r, hipStream_t s) {
  if (r.n <= kSmallRequests && c.num_pages <= kSmallPages) {
    TCD_LAUNCH("pages_plan_small_kernel", pages_plan_small_kernel, dim3(1), dim3(kSmallBlock), s, c, t, r);
    return grant(c, t, r, s);
  }
  if (r.kind == kResize)
    TCD_LAUNCH("pages_shrink_kernel", pages_shrink_kernel, dim3((unsigned)ceil_div(r.n, (int64_t)kRequestWaves)), dim3(kPageBlock), s, c, t, r);
  const int64_t request_blocks = ceil_div(r.n, (int64_t)kRequestWaves);
  TCD_LAUNCH("pages_tally_kernel", pages_tally_kernel, dim3((unsigned)(t.spans + request_blocks)), dim3(kPageBlock), s, c, t, r);
  TCD_LAUNCH("pages_list_kernel", pages_list_kernel, dim3((unsigned)t.spans + 1u), dim3(kPageBlock), s, c, t, r.n);
  return grant(c, t, r, s);
}

}  // namespace tcd

extern "C" int thrust_cdna4_pages_fork(void* temp, size_t* temp_bytes, const thrust_cdna4_page_cache* cache, const int32_t* parents,
                                       const int32_t* children, int64_t n, int share, uint8_t* done, void* stream) {
  using namespace tcd;
  PageCache c;
  if (!temp_bytes || temp_misaligned(temp) || n < 0 || n > kMaxRequests || !cache_of(cache, c)) return hipErrorInvalidValue;
  PageTemp t;
  const size_t bytes = page_temp(c, n, false, temp, t);
  if (!temp) {
    *temp_bytes = bytes;
    return hipSuccess;
  }
  if (n == 0) return hipSuccess;
  if (*temp_bytes < bytes || !parents || !children || !done || !cache_usable(c)) return hipErrorInvalidValue;
  return (int)serve(c, t, Requests{parents, children, n, share ? kForkShared : kFork, done}, static_cast<hipStream_t>(stream));
}

extern "C" int thrust_cdna4_pages_resize(void* temp, size_t* temp_bytes, const thrust_cdna4_page_cache* cache, const int32_t* sequences,
                                         const int32_t* lengths, int64_t n, uint8_t* done, void* stream) {
  using namespace tcd;
  PageCache c;
  if (!temp_bytes || temp_misaligned(temp) || n < 0 || n > kMaxRequests || !cache_of(cache, c)) return hipErrorInvalidValue;
  PageTemp t;
  const size_t bytes = page_temp(c, n, false, temp, t);
  if (!temp) {
    *temp_bytes = bytes;
    return hipSuccess;
  }
  if (n == 0) return hipSuccess;
  if (*temp_bytes < bytes || !sequences || !lengths || !done || !cache_usable(c)) return hipErrorInvalidValue;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Requests r{lengths, sequences, n, kResize, done};
  return (int)serve(c, t, r, s);
}

extern "C" int thrust_cdna4_pages_free(const thrust_cdna4_page_cache* cache, const int32_t* sequences, int64_t n, uint8_t* done, void* stream) {
  using namespace tcd;
  PageCache c;
  if (n < 0 || n > kMaxRequests || !cache_of(cache, c)) return hipErrorInvalidValue;
  if (n == 0) return hipSuccess;
  if (!sequences || !cache_usable(c)) return hipErrorInvalidValue;
  hipStream_t s = static_cast<hipStream_t>(stream);
  TCD_LAUNCH("pages_shrink_kernel", pages_shrink_kernel, dim3((unsigned)ceil_div(n, (int64_t)kRequestWaves)), dim3(kPageBlock), s, c, PageTemp{},
             (Requests{nullptr, sequences, n, kResize, done}));
  return (int)hipGetLastError();
}

extern "C" int thrust_cdna4_pages_compact(void* temp, size_t* temp_bytes, const thrust_cdna4_page_cache* cache, int32_t* tables_out,
                                          int32_t* refs_out, int32_t* live_out, void* stream) {
  using namespace tcd;
  PageCache c;
  if (!temp_bytes || temp_misaligned(temp) || !cache_of(cache, c)) return hipErrorInvalidValue;
  PageTemp t;
  const size_t bytes = page_temp(c, 0, true, temp, t);
  if (!temp) {
    *temp_bytes = bytes;
    return hipSuccess;
  }
  const int64_t entries = (int64_t)c.num_sequences * c.max_pages;
  if (*temp_bytes < bytes || !live_out || !cache_usable(c) || (c.num_pages > 0 && !refs_out) || (entries > 0 && !tables_out))
    return hipErrorInvalidValue;
  // the outputs may be the cache's own arrays, and meet nothing else
  const size_t table_bytes = (size_t)entries * 4, ref_bytes = (size_t)c.num_pages * 4, length_bytes = (size_t)c.num_sequences * 4;
  auto meet = [](const void* a, size_t na, const void* b, size_t nb) { return na && nb && ranges_overlap(a, na, b, nb); };
  if ((tables_out != c.tables && meet(tables_out, table_bytes, c.tables, table_bytes)) || meet(tables_out, table_bytes, c.refs, ref_bytes) ||
      (refs_out != c.refs && meet(refs_out, ref_bytes, c.refs, ref_bytes)) || meet(refs_out, ref_bytes, c.tables, table_bytes) ||
      meet(tables_out, table_bytes, refs_out, ref_bytes) || meet(tables_out, table_bytes, c.lengths, length_bytes) ||
      meet(refs_out, ref_bytes, c.lengths, length_bytes))
    return hipErrorInvalidValue;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (c.num_pages == 0) {  // nothing to move; tables name nothing
    hipError_t e = zero_async(live_out, 4, s);
    if (e != hipSuccess) return (int)e;
    e = zero_async(t.head, 16, s);
    if (e != hipSuccess) return (int)e;
  } else if (c.num_pages <= kSmallPages) {
    TCD_LAUNCH("pages_rank_small_kernel", pages_rank_small_kernel, dim3(1), dim3(kSmallBlock), s, c, t, refs_out, live_out);
  } else {
    TCD_LAUNCH("pages_tally_only_kernel", pages_tally_only_kernel, dim3((unsigned)t.spans), dim3(kPageBlock), s, c, t);
    TCD_LAUNCH("pages_rank_kernel", pages_rank_kernel, dim3((unsigned)t.spans), dim3(kPageBlock), s, c, t, refs_out, live_out);
  }
  int64_t table_blocks = ceil_div(entries, (int64_t)kPageBlock * 4);
  if (table_blocks > 2048) table_blocks = 2048;
  const int64_t units = ceil_div(c.page_bytes, (int64_t)kCopyUnit) * c.num_pools * (c.num_pages / 2);  // at most: half of the pages move
  int64_t copy_blocks = (int64_t)device_cu_count() * 16;
  if (copy_blocks > units) copy_blocks = units;
  if (copy_blocks < 1) copy_blocks = 1;
  TCD_LAUNCH("pages_move_kernel", pages_move_kernel, dim3((unsigned)(table_blocks + copy_blocks)), dim3(kPageBlock), s, c, t, tables_out,
             refs_out, live_out, (int)table_blocks);
  return (int)hipGetLastError();
}
