// pa_pages.cu -- page accounting of paged K/V caches on the device (sm_100a).
//
// A pool counts the users of each page (refs) and keeps one bit per free page.
// Block tables, lengths and both of these live in device memory and are changed
// by kernels on the caller's stream: a step that frees, takes, shares, copies or
// moves pages needs no host round trip and can be captured into a graph.
//
//   resize   rows change their lengths: pages behind the new length and pages
//            that left the window are released, missing pages are taken, a
//            partly filled last page that others use too is replaced by a copy
//   fork     a row continued by another: full pages are shared, the used slots
//            of the partly filled last page are copied in every layer
//   compact  the live pages move in front of the free ones in every layer
//
// Every choice is deterministic: the free pages are taken in ascending order,
// in the order of the rows (or pairs); sums over atomics are whole numbers.
//
// What bounds them: resize and the plans of fork and compact are a few dependent
// round trips to L2 (lengths, table entries, counts, bitmap); the copies are
// bound by HBM: each moved byte is read once and written once.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <climits>

#include "pa_decode.h"

namespace pa_pages {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kPlanThreads = 1024;
// Table entries one warp releases per work item: 16 loads in flight per lane.
constexpr int kReleaseSpan = 512;
// Taken pages listed in shared memory; longer lists go through the scratch.
constexpr int kListSmem = 4096;
// Copy kernel: 256 threads x 8 x 16 bytes per unit.
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;
// Three blocks an SM (96 KB of loads in flight): compacting 4096 pages of 16 layers
// (2.06 GB moved) 349 us, with four blocks 378, two 357, four loads a thread 361;
// grids of 8 to 64 blocks an SM differ by 5 %.
constexpr int kCopyBlocks = 3;
constexpr int kCopyGrid = 16;
constexpr int kCopyChunks = kCopyThreads * kCopyUnroll;   // 16-byte chunks of one unit

// Scratch header (int32): zero between launches except kHCopies, which the plan
// kernel sets for the copy kernel that follows it, and kHLive.
constexpr int kHArrive = 0;   // arrivals of the release phase
constexpr int kHCopies = 1;   // entries of the copy list
constexpr int kHLive = 2;     // live pages (compact)
constexpr int kHeader = 32;

struct Pool {
  char* const* caches;        // 2 x layers: K, V of each layer
  int layers;
  long long sb[2], ss[2], sh[2];   // bytes: page, slot, head strides of K and V
  int NB, bs, Hkv, chunks;    // chunks: 16-byte pieces of one (slot, head) row
  int dense;                  // a page's slots and heads are contiguous in K and V
  int* refs;
  unsigned* words;            // bit set: free
  int nwords;
  int* scratch;
  unsigned* status;
  // carve-up of the scratch
  __host__ __device__ int* copies() const { return scratch + kHeader; }          // [3 * NB]
  __host__ __device__ int* list() const { return copies() + 3 * static_cast<size_t>(NB); }  // [NB]
  __host__ __device__ int* plan() const { return list() + NB; }                  // [2 * pairs] (fork)
};

struct Table {
  int* bt;
  long long sb;               // row stride, elements
  int rows, width;
  int* lens;
};

__device__ __forceinline__ void flag(const Pool& p, unsigned bits) {
  if (p.status) atomicOr(p.status, bits);
}
__device__ __forceinline__ bool in_pool(const Pool& p, int page) {
  return static_cast<unsigned>(page) < static_cast<unsigned>(p.NB);
}
__device__ __forceinline__ void grid_wait() {
  // Dependent launch: nothing before this touches global memory.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Inclusive sum over the block's threads in thread order; `total` gets the sum.
// Ends with a barrier, so that back-to-back calls may share `sh` (32 entries).
template <class I>
__device__ __forceinline__ I block_scan(I v, I* sh, I& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I u = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) sh[warp] = v;
  __syncthreads();
  if (warp == 0) {
    I w = lane < nw ? sh[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const I u = __shfl_up_sync(kFull, w, o);
      if (lane >= o) w += u;
    }
    sh[lane] = w;
  }
  __syncthreads();
  const I before = warp ? sh[warp - 1] : 0;
  total = sh[nw - 1];
  __syncthreads();
  return before + v;
}

// The words of this thread: an equal contiguous share of the bitmap.
struct Share { int lo, hi; };
__device__ __forceinline__ Share word_share(const Pool& p) {
  const int per = (p.nwords + blockDim.x - 1) / blockDim.x;
  Share s;
  s.lo = min(p.nwords, static_cast<int>(threadIdx.x) * per);
  s.hi = min(p.nwords, s.lo + per);
  return s;
}
__device__ __forceinline__ int count_free(const Pool& p, const Share& s) {
  int n = 0;
  for (int w = s.lo; w < s.hi; ++w) n += __popc(__ldcg(p.words + w));
  return n;
}
// Takes the free pages of rank [from, to) in ascending order: list[k] = the one
// of rank from + k, its bit cleared and its count set to 1. `rank`: the rank of
// this thread's lowest free page that has not been taken, advanced past those
// taken here.
__device__ __forceinline__ void take_free(const Pool& p, const Share& s, int& rank, int from, int to,
                                          int* list) {
  for (int w = s.lo; w < s.hi && rank < to; ++w) {
    unsigned bits = __ldcg(p.words + w);
    if (!bits) continue;
    while (bits && rank < to) {
      const int page = w * 32 + __ffs(bits) - 1;
      bits &= bits - 1;
      list[rank++ - from] = page;
      p.refs[page] = 1;
    }
    p.words[w] = bits;
  }
}

// ----------------------------------------------------------------------------
// resize
// ----------------------------------------------------------------------------
struct Resize {
  Pool p;
  Table t;
  const int* new_lens;
  int window, sinks;          // window 0: none
  int spans;                  // ceil(width / kReleaseSpan)
};

struct RowChange {
  bool active;
  int S, n;                   // length before and after
  int used, want;             // pages before and after
  int keep_sinks, first;      // pages [keep_sinks, first) hold no visible token
};

// A row's change of length; `bad`: a length outside the table.
__device__ __forceinline__ RowChange row_change(const Resize& a, int r, bool& bad) {
  RowChange c;
  c.S = __ldcg(a.t.lens + r);
  c.n = __ldg(a.new_lens + r);
  const long long cap = static_cast<long long>(a.t.width) * a.p.bs;
  bad = c.n >= 0 && (c.S < 0 || c.S > cap || c.n > cap);
  c.active = c.n >= 0 && !bad;
  c.used = c.S > 0 ? (c.S - 1) / a.p.bs + 1 : 0;
  c.want = c.n > 0 ? (c.n - 1) / a.p.bs + 1 : 0;
  c.keep_sinks = c.first = 0;
  if (c.active && a.window) {
    // The next query sits at min(S, n) or later and sees nothing before
    // token min(S, n) - window + 1 but the sinks.
    c.keep_sinks = a.sinks > 0 ? (a.sinks - 1) / a.p.bs + 1 : 0;
    const int low = min(c.S, c.n) - a.window + 1;
    c.first = low > 0 ? low / a.p.bs : 0;
  }
  return c;
}

__global__ void __launch_bounds__(kPlanThreads) resize_kernel(const Resize a) {
  __shared__ int s_scan[32];
  __shared__ long long s_needs[32];        // rows may ask for more than 2^31 pages together
  __shared__ int s_list[kListSmem];
  __shared__ int s_last, s_copies;
  const Pool& p = a.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  grid_wait();

  // Release, spread over the grid: one warp per 512 entries of a row.
  const long long items = static_cast<long long>(a.t.rows) * a.spans;
  for (long long it = blockIdx.x * static_cast<long long>(nw) + warp; it < items;
       it += static_cast<long long>(gridDim.x) * nw) {
    const int r = static_cast<int>(it / a.spans);
    const int span = static_cast<int>(it - static_cast<long long>(r) * a.spans);
    bool bad;
    const RowChange c = row_change(a, r, bad);
    if (bad && span == 0 && lane == 0) flag(p, PA_STATUS_BAD_SEQLEN);
    if (!c.active) continue;
    int* row = a.t.bt + r * a.t.sb;
    const int j0 = span * kReleaseSpan + lane;
    // nothing to release in this span: no loads
    const int lo = span * kReleaseSpan, hi = min(lo + kReleaseSpan, c.used);
    const bool cut = max(lo, c.want) < hi;
    const bool old = max(lo, c.keep_sinks) < min(hi, c.first);
    if (!cut && !old) continue;
    int e[kReleaseSpan / 32];
#pragma unroll
    for (int i = 0; i < kReleaseSpan / 32; ++i) {
      const int j = j0 + i * 32;
      const bool drop = j < c.used && (j >= c.want || (j >= c.keep_sinks && j < c.first));
      e[i] = drop ? __ldcg(row + j) : -1;
    }
#pragma unroll
    for (int i = 0; i < kReleaseSpan / 32; ++i) {
      if (e[i] == -1) continue;
      row[j0 + i * 32] = -1;
      if (!in_pool(p, e[i])) {
        flag(p, PA_STATUS_BAD_BLOCK);
        continue;
      }
      const int users = atomicSub(p.refs + e[i], 1);
      if (users == 1) {
        atomicOr(p.words + (e[i] >> 5), 1u << (e[i] & 31));
      } else if (users <= 0) {              // freed already: the count stays 0
        atomicAdd(p.refs + e[i], 1);
        flag(p, PA_STATUS_BAD_BLOCK);
      }
    }
  }

  // The last block to arrive takes the missing pages.
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(p.scratch + kHArrive, 1) == static_cast<int>(gridDim.x) - 1;
    __threadfence();
  }
  __syncthreads();
  if (!s_last) return;

  const Share sh = word_share(p);
  const int mine = count_free(p, sh);
  int avail;
  int rank = block_scan(mine, s_scan, avail) - mine;
  if (threadIdx.x == 0) {
    p.scratch[kHArrive] = 0;
    s_copies = 0;
  }

  // In row order, a row all of its pages or none; 1024 rows at a time, one
  // thread each (a step's rows miss a page or two: with a warp per row, eight
  // rows in turn per warp and their lengths read again, this phase took 10 of
  // the call's 18 us for 256 rows).
  long long carry = 0;        // pages asked for so far, refused rows' among them
  int given = 0;              // pages given out so far
  for (int r0 = 0; r0 < a.t.rows; r0 += blockDim.x) {
    const int r = r0 + threadIdx.x;
    long long need = 0;
    int cow = 0, tail = 0;
    bool bad;
    RowChange c;
    c.active = false;
    int* row = a.t.bt + r * a.t.sb;
    if (r < a.t.rows) c = row_change(a, r, bad);
    if (c.active && c.n > c.S) {
      need = c.want - c.used;
      if (c.S % p.bs) {                     // grows into its partly filled last page
        tail = __ldcg(row + c.S / p.bs);
        if (!in_pool(p, tail))
          flag(p, PA_STATUS_BAD_BLOCK);
        else
          cow = __ldcg(p.refs + tail) > 1;  // others use it too: a copy of its own
      }
    }
    need += cow;
    long long total;
    const long long all = carry + block_scan(need, s_needs, total);
    const bool ok = need == 0 || all <= avail;
    if (c.active && !ok) flag(p, PA_STATUS_NO_PAGES);
    // the pages of these rows: up to the largest end of a row that gets its pages
    const unsigned top = __reduce_max_sync(kFull, need > 0 && ok ? static_cast<unsigned>(all) : 0u);
    if (lane == 0) s_scan[warp] = static_cast<int>(top);
    __syncthreads();
    int end = given;
    for (int w = 0; w < nw; ++w) end = max(end, s_scan[w]);
    int* list = end - given <= kListSmem ? s_list : p.list();
    take_free(p, sh, rank, given, end, list);
    __syncthreads();
    int at = static_cast<int>(all - need) - given;     // the row's place in the list
    if (c.active && ok) {
      if (cow) {
        const int dst = list[at];
        row[c.S / p.bs] = dst;
        int* e = p.copies() + 3 * atomicAdd(&s_copies, 1);   // (in any order)
        e[0] = tail;
        e[1] = dst;
        e[2] = c.S % p.bs;
        ++at;
      }
      a.t.lens[r] = c.n;
    }
    // New entries: a few by the row's own thread, many by its warp.
    const int fresh = c.active && ok ? max(0, c.want - c.used) : 0;
    if (fresh <= 4)
      for (int i = 0; i < fresh; ++i) row[c.used + i] = list[at + i];
    for (unsigned big = __ballot_sync(kFull, fresh > 4); big; big &= big - 1) {
      const int src = __ffs(big) - 1;
      const int cnt = __shfl_sync(kFull, fresh, src), first = __shfl_sync(kFull, c.used, src);
      const int from = __shfl_sync(kFull, at, src);
      int* to = a.t.bt + (r - lane + src) * a.t.sb + first;
      for (int i = lane; i < cnt; i += 32) to[i] = list[from + i];
    }
    carry += total;
    given = end;
    __syncthreads();
  }
  // The copied pages lose these users. Only here, so that the free pages numbered
  // above stay the ones they were, and every row found the counts that the releases
  // left, whichever 1024 rows it was among.
  for (int k = threadIdx.x; k < s_copies; k += blockDim.x) {
    const int src = p.copies()[3 * k];
    if (atomicSub(p.refs + src, 1) == 1) atomicOr(p.words + (src >> 5), 1u << (src & 31));
  }
  if (threadIdx.x == 0) p.scratch[kHCopies] = s_copies;
}

// ----------------------------------------------------------------------------
// adopt
// ----------------------------------------------------------------------------
struct Adopt {
  Pool p;
  const int* bt;
  long long sb;
  int rows, width;
  const int* lens;
};

// Counts the entries in use (the counts start at zero); the last block to arrive
// makes the free bits from the counts.
__global__ void __launch_bounds__(kPlanThreads) adopt_kernel(const Adopt a) {
  __shared__ int s_last;
  const Pool& p = a.p;
  grid_wait();
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int S = __ldg(a.lens + r);
    const long long cap = static_cast<long long>(a.width) * p.bs;
    if ((S < 0 || S > cap) && threadIdx.x == 0) flag(p, PA_STATUS_BAD_SEQLEN);
    const int used = S <= 0 ? 0 : S > cap ? a.width : (S - 1) / p.bs + 1;
    for (int j = threadIdx.x; j < used; j += blockDim.x) {
      const int e = __ldg(a.bt + r * a.sb + j);
      if (in_pool(p, e))
        atomicAdd(p.refs + e, 1);
      else if (e != -1)
        flag(p, PA_STATUS_BAD_BLOCK);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(p.scratch + kHArrive, 1) == static_cast<int>(gridDim.x) - 1;
    __threadfence();
  }
  __syncthreads();
  if (!s_last) return;
  if (threadIdx.x == 0) p.scratch[kHArrive] = 0;
  // a warp per word: lane = bit
  const int lane = threadIdx.x & 31;
  for (int w = threadIdx.x >> 5; w < p.nwords; w += blockDim.x >> 5) {
    const int page = w * 32 + lane;
    const unsigned bits = __ballot_sync(kFull, page < p.NB && __ldcg(p.refs + page) == 0);
    if (lane == 0) p.words[w] = bits;
  }
}

// ----------------------------------------------------------------------------
// Copies
// ----------------------------------------------------------------------------
// A unit is one 32 KB part of the used slots of one page in one cache: all eight
// loads of a thread are issued before its stores. A block runs several units in
// turn and reads the next one's list entry during the current one, so that the
// list's latency stays off the path of the data.
struct CopyUnit { int src, dst, slots, cache, part; };
__device__ __forceinline__ CopyUnit load_unit(const Pool& p, long long u, int parts) {
  CopyUnit c;
  const int per_entry = 2 * p.layers * parts;
  long long entry;
  int rest;
  if (u <= 0xffffffffll) {                          // 32-bit divisions nearly always
    const unsigned q = static_cast<unsigned>(u) / static_cast<unsigned>(per_entry);
    entry = q;
    rest = static_cast<int>(static_cast<unsigned>(u) - q * per_entry);
  } else {
    entry = u / per_entry;
    rest = static_cast<int>(u - entry * per_entry);
  }
  c.cache = rest / parts;
  c.part = rest - c.cache * parts;
  const int* e = p.copies() + 3 * entry;
  c.src = __ldcg(e);
  c.dst = __ldcg(e + 1);
  c.slots = __ldcg(e + 2);
  return c;
}
__device__ __forceinline__ void copy_unit(const Pool& p, const CopyUnit& u) {
  const int row = p.Hkv * p.chunks;                 // chunks of one slot
  const int n = u.slots * row;
  if (u.part * kCopyChunks >= n) return;
  const int c0 = u.part * kCopyChunks + threadIdx.x;
  const bool v_cache = u.cache & 1;
  const long long sb = v_cache ? p.sb[1] : p.sb[0];
  char* base = p.caches[u.cache];
  const char* from = base + u.src * sb;
  char* to = base + u.dst * sb;
  uint4 v[kCopyUnroll];
  if (p.dense) {
    from += c0 * 16ll;
    to += c0 * 16ll;
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i)
      if (c0 + i * kCopyThreads < n)
        v[i] = __ldcs(reinterpret_cast<const uint4*>(from) + i * kCopyThreads);
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i)
      if (c0 + i * kCopyThreads < n) reinterpret_cast<uint4*>(to)[i * kCopyThreads] = v[i];
    return;
  }
  const long long ss = v_cache ? p.ss[1] : p.ss[0], sh = v_cache ? p.sh[1] : p.sh[0];
  auto off = [&](int c) {
    const int slot = c / row;
    const int h = (c - slot * row) / p.chunks;
    return slot * ss + h * sh + (c - slot * row - h * p.chunks) * 16ll;
  };
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i)
    if (c0 + i * kCopyThreads < n)
      v[i] = __ldcs(reinterpret_cast<const uint4*>(from + off(c0 + i * kCopyThreads)));
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i)
    if (c0 + i * kCopyThreads < n)
      *reinterpret_cast<uint4*>(to + off(c0 + i * kCopyThreads)) = v[i];
}

__device__ __forceinline__ int page_parts(const Pool& p) {
  return (p.bs * p.Hkv * p.chunks + kCopyChunks - 1) / kCopyChunks;
}

// The copy list's units from `first` on, `step` apart.
__device__ __forceinline__ void copy_all(const Pool& p, long long first, long long step) {
  const int parts = page_parts(p);
  const long long units = static_cast<long long>(__ldcg(p.scratch + kHCopies)) * 2 * p.layers * parts;
  if (first >= units) return;
  CopyUnit next = load_unit(p, first, parts);
  for (long long u = first; u < units; u += step) {
    const CopyUnit cur = next;
    if (u + step < units) next = load_unit(p, u + step, parts);
    copy_unit(p, cur);
  }
}

__global__ void __launch_bounds__(kCopyThreads, kCopyBlocks) copy_kernel(const Pool p) {
  grid_wait();
  copy_all(p, blockIdx.x, gridDim.x);
}

// ----------------------------------------------------------------------------
// fork
// ----------------------------------------------------------------------------
struct Fork {
  Pool p;
  Table t;
  const int* parents;
  const int* children;
  int n;
};

// One block: which pairs go through, their new pages and the copy list.
// plan[2i] = length of the parent (-1: the pair does nothing), plan[2i + 1] =
// the new last page (-1: none).
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const Fork a) {
  __shared__ int s_scan[32];
  __shared__ int s_list[kListSmem];
  const Pool& p = a.p;
  grid_wait();
  const Share sh = word_share(p);
  const int mine = count_free(p, sh);
  int avail;
  int rank = block_scan(mine, s_scan, avail) - mine;
  int* plan = p.plan();

  // A child row has to be empty. Pairs that name the same child: the first one
  // gets it; it is the one whose claim, a length far below zero, is lowest.
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
    const int pr = __ldg(a.parents + i), ch = __ldg(a.children + i);
    plan[2 * i] = -1;
    if (pr < 0 || ch < 0) continue;        // padding
    if (pr >= a.t.rows || ch >= a.t.rows) {
      flag(p, PA_STATUS_BAD_ROW);
      continue;
    }
    const int have = __ldcg(a.t.lens + ch);
    if (have != 0 && have >= INT_MIN + a.n) {
      flag(p, PA_STATUS_BAD_ROW);
      continue;
    }
    atomicMin(a.t.lens + ch, INT_MIN + i);
    plan[2 * i] = 0;
  }
  __syncthreads();

  // Who won, how long the parents are, who needs a page for a copied tail.
  long long carry = 0;
  int granted = 0;
  for (int i0 = 0; i0 < a.n; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    int need = 0, S = -1;
    if (i < a.n && plan[2 * i] == 0) {
      const int pr = __ldg(a.parents + i), ch = __ldg(a.children + i);
      if (__ldcg(a.t.lens + ch) != INT_MIN + i) {
        flag(p, PA_STATUS_BAD_ROW);
      } else {
        S = __ldcg(a.t.lens + pr);
        if (S < INT_MIN + a.n) S = 0;      // itself a child of this call: it was empty
        if (S < 0 || S > static_cast<long long>(a.t.width) * p.bs) {
          flag(p, PA_STATUS_BAD_SEQLEN);
          S = -2;                          // the child stays empty
        } else if (S % p.bs) {
          if (in_pool(p, __ldcg(a.t.bt + pr * a.t.sb + S / p.bs))) {
            need = 1;
          } else {
            flag(p, PA_STATUS_BAD_BLOCK);
            S = -2;
          }
        }
      }
    }
    int total;
    const int end = block_scan(need, s_scan, total);
    const long long all = carry + end;
    if (need && all > avail) {
      flag(p, PA_STATUS_NO_PAGES);
      S = -2;
      need = 0;
    }
    if (i < a.n) {
      plan[2 * i] = S;
      plan[2 * i + 1] = need ? static_cast<int>(all - 1) : -1;   // place in the list
    }
    carry += total;
  }
  granted = static_cast<int>(min(carry, static_cast<long long>(avail)));
  int* list = granted <= kListSmem ? s_list : p.list();
  take_free(p, sh, rank, 0, granted, list);
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
    const int S = plan[2 * i];
    if (S == -1) continue;
    const int k = plan[2 * i + 1];
    a.t.lens[__ldg(a.children + i)] = max(S, 0);
    if (S < 0) {
      plan[2 * i] = -1;
    } else if (k >= 0) {
      const int page = list[k];
      plan[2 * i + 1] = page;
      int* e = p.copies() + 3 * k;
      e[0] = __ldcg(a.t.bt + __ldg(a.parents + i) * a.t.sb + S / p.bs);
      e[1] = page;
      e[2] = S % p.bs;
    }
  }
  if (threadIdx.x == 0) p.scratch[kHCopies] = granted;
}

// The children's table rows (each shared page counted once more), and the copies.
__global__ void __launch_bounds__(kCopyThreads, kCopyBlocks) fork_apply_kernel(const Fork a) {
  const Pool& p = a.p;
  grid_wait();
  const int* plan = p.plan();
  const int spans = (a.t.width + kCopyThreads - 1) / kCopyThreads;
  const long long rows = static_cast<long long>(a.n) * spans;
  for (long long u = blockIdx.x; u < rows; u += gridDim.x) {
    const int i = static_cast<int>(u / spans);
    const int S = __ldcg(plan + 2 * i);
    const int j = static_cast<int>(u - static_cast<long long>(i) * spans) * kCopyThreads + threadIdx.x;
    if (S < 0 || j >= a.t.width) continue;
    const int full = S / p.bs;
    int e = -1;
    if (j < full) {
      e = __ldcg(a.t.bt + __ldg(a.parents + i) * a.t.sb + j);
      if (in_pool(p, e)) atomicAdd(p.refs + e, 1);
    } else if (j == full && S % p.bs) {
      e = __ldcg(plan + 2 * i + 1);
    }
    a.t.bt[__ldg(a.children + i) * a.t.sb + j] = e;
  }
  copy_all(p, (blockIdx.x + gridDim.x - rows % gridDim.x) % gridDim.x, gridDim.x);
}

// ----------------------------------------------------------------------------
// compact
// ----------------------------------------------------------------------------
struct Compact {
  Pool p;
  Table t;                    // lens unused
  int* live;                  // out: number of live pages
};

// One block: the k-th live page at or behind the live count goes to the k-th
// free page before it. map[page] (in the list's place) is a moved page's new
// index, -1 for a free page behind the count.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const Compact a) {
  __shared__ int s_scan[32];
  const Pool& p = a.p;
  grid_wait();
  const Share sh = word_share(p);
  int avail;
  block_scan(count_free(p, sh), s_scan, avail);
  const int live = p.NB - avail;
  int holes = 0, movers = 0;
  for (int w = sh.lo; w < sh.hi; ++w) {
    const unsigned fr = __ldcg(p.words + w);
    const int left = min(32, p.NB - w * 32);               // pages of this word
    const unsigned valid = left == 32 ? kFull : (1u << left) - 1;
    const int front = max(0, min(32, live - w * 32));      // of them before the live count
    const unsigned fm = front == 32 ? kFull : (1u << front) - 1;
    holes += __popc(fr & fm & valid);
    movers += __popc(~fr & ~fm & valid);
  }
  int total;
  int kh = block_scan(holes, s_scan, total) - holes;
  int km = block_scan(movers, s_scan, total) - movers;     // as many as holes
  int* map = p.list();
  for (int w = sh.lo; w < sh.hi; ++w) {
    const unsigned fr = __ldcg(p.words + w);
    const int left = min(32, p.NB - w * 32);
    const unsigned valid = left == 32 ? kFull : (1u << left) - 1;
    const int front = max(0, min(32, live - w * 32));
    const unsigned fm = front == 32 ? kFull : (1u << front) - 1;
    for (unsigned b = fr & fm & valid; b; b &= b - 1) {
      p.copies()[3 * kh + 1] = w * 32 + __ffs(b) - 1;
      ++kh;
    }
    for (unsigned b = ~fm & valid; b; b &= b - 1) {
      const int i = __ffs(b) - 1;
      if (fr >> i & 1u) {
        map[w * 32 + i] = -1;
      } else {
        p.copies()[3 * km] = w * 32 + i;
        p.copies()[3 * km + 2] = p.bs;
        ++km;
      }
    }
    p.words[w] = ~fm & valid;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < total; k += blockDim.x) {
    const int src = p.copies()[3 * k], dst = p.copies()[3 * k + 1];
    map[src] = dst;
    p.refs[dst] = __ldcg(p.refs + src);
    p.refs[src] = 0;
  }
  if (threadIdx.x == 0) {
    p.scratch[kHCopies] = total;
    p.scratch[kHLive] = live;
    *a.live = live;
  }
}

__global__ void __launch_bounds__(kCopyThreads, kCopyBlocks) compact_apply_kernel(const Compact a) {
  const Pool& p = a.p;
  grid_wait();
  const int live = __ldcg(p.scratch + kHLive);
  const int* map = p.list();
  const int spans = (a.t.width + kCopyThreads - 1) / kCopyThreads;
  const long long rows = static_cast<long long>(a.t.rows) * spans;
  for (long long u = blockIdx.x; u < rows; u += gridDim.x) {
    const int r = static_cast<int>(u / spans);
    const int j = static_cast<int>(u - static_cast<long long>(r) * spans) * kCopyThreads + threadIdx.x;
    if (j >= a.t.width) continue;
    int* at = a.t.bt + r * a.t.sb + j;
    const int e = __ldcg(at);
    if (e < live) continue;                 // -1, or a page that stays
    const int to = e < p.NB ? __ldcg(map + e) : -1;
    if (to < 0)
      flag(p, PA_STATUS_BAD_BLOCK);         // a free page, or none of the pool
    else
      *at = to;
  }
  copy_all(p, (blockIdx.x + gridDim.x - rows % gridDim.x) % gridDim.x, gridDim.x);
}

// ----------------------------------------------------------------------------
// Host side
// ----------------------------------------------------------------------------
static size_t scratch_ints(const pa_page_pool* p, int32_t rows, int32_t pairs) {
  return kHeader + 4 * static_cast<size_t>(p->num_blocks) +
         std::max(static_cast<size_t>(rows), 2 * static_cast<size_t>(pairs));
}

static pa_status_t make_pool(const pa_page_pool* q, int32_t rows, int32_t pairs, Pool& p) {
  if (!q || rows < 0 || pairs < 0) return PA_ERR_ARG;
  if (q->num_blocks <= 0 || q->block_size <= 0 || q->num_kv_heads <= 0 || q->head_dim <= 0 ||
      q->num_layers < 0)
    return PA_ERR_ARG;
  if (q->head_dim % 8) return PA_ERR_UNSUPPORTED;
  // a page's 16-byte pieces are counted in int32
  if (static_cast<long long>(q->block_size) * q->num_kv_heads * (q->head_dim / 8) > (1 << 30))
    return PA_ERR_UNSUPPORTED;
  if (q->num_blocks > (1 << 29)) return PA_ERR_UNSUPPORTED;
  const int64_t strides[6] = {q->k_stride_block, q->k_stride_slot, q->k_stride_head,
                              q->v_stride_block, q->v_stride_slot, q->v_stride_head};
  for (int i = 0; i < 6; ++i)
    if (strides[i] % 8) return PA_ERR_ARG;
  if (!q->refs || !q->free_words || !q->scratch || (q->num_layers && !q->caches))
    return PA_ERR_ARG;
  if (q->scratch_ints < scratch_ints(q, rows, pairs)) return PA_ERR_WORKSPACE;
  p.caches = reinterpret_cast<char* const*>(q->caches);
  p.layers = q->num_layers;
  p.sb[0] = q->k_stride_block * 2;
  p.ss[0] = q->k_stride_slot * 2;
  p.sh[0] = q->k_stride_head * 2;
  p.sb[1] = q->v_stride_block * 2;
  p.ss[1] = q->v_stride_slot * 2;
  p.sh[1] = q->v_stride_head * 2;
  p.NB = q->num_blocks;
  p.bs = q->block_size;
  p.Hkv = q->num_kv_heads;
  p.chunks = q->head_dim / 8;
  p.dense = 1;
  for (int i = 0; i < 2; ++i)
    if (p.ss[i] != static_cast<long long>(p.Hkv) * p.chunks * 16 ||
        (p.Hkv > 1 && p.sh[i] != p.chunks * 16ll))
      p.dense = 0;
  p.refs = q->refs;
  p.words = q->free_words;
  p.nwords = (q->num_blocks + 31) / 32;
  p.scratch = q->scratch;
  p.status = q->status;
  return PA_OK;
}

static pa_status_t make_table(int32_t* bt, int64_t stride, int32_t rows, int32_t width,
                              int32_t* lens, bool need_lens, Table& t) {
  if (rows < 0 || width < 0) return PA_ERR_ARG;
  if (rows > 0 && ((width > 0 && !bt) || (need_lens && !lens))) return PA_ERR_ARG;
  t.bt = bt;
  t.sb = stride;
  t.rows = rows;
  t.width = width;
  t.lens = lens;
  return PA_OK;
}

// Programmatic dependent launch: the kernel's griddepcontrol.wait orders its
// memory accesses after the previous kernel in the stream.
template <class Arg>
static cudaError_t launch(void (*kernel)(const Arg), long long grid, int threads, const Arg& arg,
                          cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(std::max<long long>(1, grid)));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, arg);
}

// Blocks of a kernel that copies up to `entries` pages and walks `row_units`
// table parts: one per unit, at most kCopyGrid per SM.
static long long copy_grid(const Pool& p, long long entries, long long row_units, int sms) {
  const long long parts =
      (static_cast<long long>(p.bs) * p.Hkv * p.chunks + kCopyChunks - 1) / kCopyChunks;
  return std::min<long long>(static_cast<long long>(kCopyGrid) * sms, entries * 2 * p.layers * parts + row_units);
}

}  // namespace pa_pages

using namespace pa_pages;

extern "C" {

pa_status_t pa_pages_scratch(const pa_page_pool* pool, int32_t rows, int32_t pairs, size_t* ints) {
  if (!pool || !ints || pool->num_blocks <= 0 || rows < 0 || pairs < 0) return PA_ERR_ARG;
  *ints = scratch_ints(pool, rows, pairs);
  return PA_OK;
}

pa_status_t pa_pages_adopt(const pa_page_pool* pool, const int32_t* block_table,
                           int64_t bt_stride_b, int32_t rows, int32_t max_blocks,
                           const int32_t* seq_lens, cudaStream_t stream) {
  Adopt a;
  const pa_status_t s = make_pool(pool, rows, 0, a.p);
  if (s != PA_OK) return s;
  if (max_blocks < 0 || (rows > 0 && (!seq_lens || (max_blocks > 0 && !block_table))))
    return PA_ERR_ARG;
  const int sms = pa_device_sm_count();
  if (sms <= 0) return PA_ERR_LAUNCH;
  a.bt = block_table;
  a.sb = bt_stride_b;
  a.rows = rows;
  a.width = max_blocks;
  a.lens = seq_lens;
  cudaError_t e = cudaMemsetAsync(a.p.refs, 0, sizeof(int32_t) * static_cast<size_t>(a.p.NB), stream);
  if (e == cudaSuccess) e = launch(adopt_kernel, std::min(rows, sms), kPlanThreads, a, stream);
  return e == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

pa_status_t pa_pages_resize(const pa_page_pool* pool, int32_t* block_table, int64_t bt_stride_b,
                            int32_t rows, int32_t max_blocks, int32_t* seq_lens,
                            const int32_t* new_lens, int32_t window, int32_t num_sinks,
                            cudaStream_t stream) {
  Resize a;
  pa_status_t s = make_pool(pool, rows, 0, a.p);
  if (s != PA_OK) return s;
  s = make_table(block_table, bt_stride_b, rows, max_blocks, seq_lens, true, a.t);
  if (s != PA_OK) return s;
  if (window < 0 || num_sinks < 0 || (window == 0 && num_sinks != 0)) return PA_ERR_ARG;
  if (rows == 0) return PA_OK;
  if (!new_lens) return PA_ERR_ARG;
  const int sms = pa_device_sm_count();
  if (sms <= 0) return PA_ERR_LAUNCH;
  a.new_lens = new_lens;
  a.window = window;
  a.sinks = num_sinks;
  a.spans = std::max(1, (max_blocks + kReleaseSpan - 1) / kReleaseSpan);
  const long long warps = static_cast<long long>(rows) * a.spans;
  cudaError_t e = launch(resize_kernel, std::min<long long>(sms, (warps + 31) / 32), kPlanThreads, a,
                         stream);
  if (e == cudaSuccess && a.p.layers)
    e = launch(copy_kernel, copy_grid(a.p, rows, 0, sms), kCopyThreads, a.p, stream);
  return e == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

pa_status_t pa_pages_fork(const pa_page_pool* pool, int32_t* block_table, int64_t bt_stride_b,
                          int32_t rows, int32_t max_blocks, int32_t* seq_lens,
                          const int32_t* parents, const int32_t* children, int32_t num_pairs,
                          cudaStream_t stream) {
  Fork a;
  pa_status_t s = make_pool(pool, rows, num_pairs, a.p);
  if (s != PA_OK) return s;
  s = make_table(block_table, bt_stride_b, rows, max_blocks, seq_lens, true, a.t);
  if (s != PA_OK) return s;
  if (num_pairs > (1 << 29)) return PA_ERR_UNSUPPORTED;
  if (num_pairs == 0 || rows == 0) return PA_OK;
  if (!parents || !children) return PA_ERR_ARG;
  const int sms = pa_device_sm_count();
  if (sms <= 0) return PA_ERR_LAUNCH;
  a.parents = parents;
  a.children = children;
  a.n = num_pairs;
  const long long spans = (max_blocks + kCopyThreads - 1) / kCopyThreads;
  cudaError_t e = launch(fork_plan_kernel, 1, kPlanThreads, a, stream);
  if (e == cudaSuccess)
    e = launch(fork_apply_kernel, copy_grid(a.p, num_pairs, spans * num_pairs, sms), kCopyThreads, a,
               stream);
  return e == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

pa_status_t pa_pages_compact(const pa_page_pool* pool, int32_t* block_table, int64_t bt_stride_b,
                             int32_t rows, int32_t max_blocks, int32_t* live, cudaStream_t stream) {
  Compact a;
  pa_status_t s = make_pool(pool, rows, 0, a.p);
  if (s != PA_OK) return s;
  s = make_table(block_table, bt_stride_b, rows, max_blocks, nullptr, false, a.t);
  if (s != PA_OK) return s;
  if (!live) return PA_ERR_ARG;
  const int sms = pa_device_sm_count();
  if (sms <= 0) return PA_ERR_LAUNCH;
  a.live = live;
  const long long spans = (max_blocks + kCopyThreads - 1) / kCopyThreads;
  cudaError_t e = launch(compact_plan_kernel, 1, kPlanThreads, a, stream);
  if (e == cudaSuccess)
    e = launch(compact_apply_kernel, copy_grid(a.p, a.p.NB / 2 + 1, spans * rows, sms), kCopyThreads,
               a, stream);
  return e == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // extern "C"
