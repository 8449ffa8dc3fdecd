// How one attention call's work is cut over a grid, computed by every CTA from the lengths on
// the device (the host does not know them).
//
// A segment is (sequence b, key head or part of one vh, row tile qt): the rows of tq tokens x gs
// query heads against the keys those tokens can see, in tiles of BK keys.  Two ways to share the
// segments out, both balanced whatever the lengths:
//  - pieces, where there are few: every segment of t tiles is cut into ceil(t / T) pieces of equal
//    length, one CTA each, with T the least number of tiles for which the pieces fit the grid (and no
//    less than min_tiles: a shorter piece costs more in its start and its join than it saves).  A CTA
//    has one segment to start and to finish, which is what a short call spends its time on.
//  - the line, where T would exceed an even share by more than a few tiles: the segments in the order
//    (b, vh, qt) form a line, each seg_cost units for its start and its end and one unit for each tile,
//    of which CTA c takes the c-th part; the parts' lengths differ by one unit.
// A segment that one CTA has to itself is finished there.  One that is cut leaves a partial result in
// at most two slots per CTA (2c, and on the line 2c + 1 for the segment a share ends in), and a
// second kernel joins the parts in the order of their CTAs, so the result does not depend on timing.
// The slots' size follows the grid and not the lengths.  The CTA with the first part of a cut segment
// leaves a record of it, so the second kernel plans nothing.
#pragma once

#include "common.cuh"
#include "paged.h"

namespace smb {

constexpr int kPlanThreads = 128;  // threads that share the scan over the sequences

struct Seq {
  int s0, n, L;  // first row of q, new tokens, keys
};

__device__ __forceinline__ Seq seq_at(const AttnArgs& a, int b) {
  Seq s;
  const int lo = min(max(a.q_starts[b], 0), a.N);
  const int hi = min(max(a.q_starts[b + 1], lo), a.N);
  s.s0 = lo;
  s.n = hi - lo;
  const long long cap = min(static_cast<long long>(a.max_pages) << a.c.page_shift, 0x7fffffffll);
  s.L = min(max(a.kv_lens[b], 0), static_cast<int>(cap));
  return s;
}

__device__ __forceinline__ int row_tiles(const AttnArgs& a, const Seq& s) {
  return s.n <= a.tq ? (s.n > 0) : (s.n + a.tq - 1) / a.tq;
}

// Keys that row tile qt can see (all of them for a tree, up to its last token otherwise).
__device__ __forceinline__ int keys_of_tile(const AttnArgs& a, const Seq& s, int qt) {
  if (a.tree != nullptr) return s.L;
  const long long end = static_cast<long long>(s.L) - s.n + min(static_cast<long long>(s.n), (qt + 1ll) * a.tq);
  return static_cast<int>(max(end, 0ll));
}

template <int BK>
__device__ __forceinline__ int tiles_of(int keys) {
  return max(1, keys / BK + (keys % BK != 0));
}

// a / b for a >= 0, b > 0, in 32 bits where both fit (a 64-bit division takes some 100 instructions).
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

// sum over i < n of floor((step * i + b) / BK), b >= 0
template <int BK>
__device__ __forceinline__ long long floor_sum(long long n, long long step, long long b) {
  long long sum = 0, m = BK, a = step;
  if (n < 65536 && step < 65536 && b < 0x7fffffff) {  // (then everything but the sum is below 2^32)
    unsigned un = static_cast<unsigned>(n), ua = static_cast<unsigned>(step), ub = static_cast<unsigned>(b), um = BK;
    while (un > 0) {
      const unsigned qa = ua / um, qb = ub / um;
      sum += static_cast<long long>(un * (un - 1) / 2) * qa + static_cast<long long>(un) * qb;
      ua -= qa * um;
      ub -= qb * um;
      const unsigned y = ua * un + ub;
      if (y < um) break;
      un = y / um;
      ub = y - un * um;
      const unsigned t = um;
      um = ua;
      ua = t;
    }
    return sum;
  }
  while (n > 0) {
    const long long qa = quotient(a, m), qb = quotient(b, m);
    sum += (n - 1) * n / 2 * qa + n * qb;
    a -= qa * m;
    b -= qb * m;
    const long long y = a * n + b;
    if (y < m) break;
    n = quotient(y, m);
    b = y - n * m;
    const long long t = m;
    m = a;
    a = t;
  }
  return sum;
}

// Units of row tiles [0, qt) of one (sequence, vh).
template <int BK>
__device__ __forceinline__ long long units_before(const AttnArgs& a, const Seq& s, int qt) {
  if (qt <= 0) return 0;
  if (s.n <= a.tq) return tiles_of<BK>(keys_of_tile(a, s, 0)) + a.seg_cost;
  if (a.tree != nullptr) return static_cast<long long>(qt) * (tiles_of<BK>(s.L) + a.seg_cost);
  const int all = row_tiles(a, s);
  long long sum = static_cast<long long>(qt) * a.seg_cost;
  int whole = qt;
  if (qt == all) {  // the last row tile may be short
    sum += tiles_of<BK>(keys_of_tile(a, s, all - 1));
    whole = all - 1;
  }
  // row tile i ends at key base + (i + 1) tq; those that end at or before key 0 still take a tile
  const long long base = static_cast<long long>(s.L) - s.n;
  long long none = 0;
  if (base + a.tq <= 0) none = min(static_cast<long long>(whole), -base / a.tq);
  sum += none;
  const long long first = base + (none + 1) * a.tq;  // > 0
  if (whole > none) sum += floor_sum<BK>(whole - none, a.tq, first + BK - 1);
  return sum;
}

// Sums over the sequences before each of kPlanThreads runs of consecutive sequences.
struct PlanShared {
  long long before[kPlanThreads + 1];  // units (line) or pieces
  long long warp_sum[kPlanThreads / 32];
  Seq seq[kPlanThreads];               // one run, one sequence: up to kPlanThreads sequences
  int fit[kPlanThreads / 32][4];
  int piece;                           // T, 0: the line
};

struct Cursor {
  int b, vh, qt;         // segment
  int keys, tiles;       // of the segment
  long long start;       // first unit of the segment on the line
  Seq s;
};

template <int BK>
__device__ __forceinline__ long long seq_units(const AttnArgs& a, const Seq& s) {
  return units_before<BK>(a, s, row_tiles(a, s)) * (a.c.Hkv * a.nsub);
}

// Exclusive prefix sums of v over the first kPlanThreads threads into sh->before; every thread calls.
__device__ __forceinline__ void plan_scan(PlanShared* sh, long long v) {
  const int t = threadIdx.x;
  long long inc = v;
  if (t < kPlanThreads) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if ((t & 31) >= o) inc += up;
    }
    if ((t & 31) == 31) sh->warp_sum[t >> 5] = inc;
  }
  __syncthreads();
  if (t < kPlanThreads) {
    long long add = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w)
      if (w < (t >> 5)) add += sh->warp_sum[w];
    sh->before[t] = add + inc - v;
    if (t == kPlanThreads - 1) sh->before[kPlanThreads] = add + inc;
  }
  __syncthreads();
}

// The i-th piece length to try, for an even share of `even` tiles.
__device__ __forceinline__ int piece_length(const AttnArgs& a, long long even, int i) {
  return static_cast<int>(max(even, static_cast<long long>(a.min_tiles))) + (i == 0 ? 0 : 1 << i);
}
__device__ __forceinline__ int pieces_of(int tiles, int T) { return (tiles + T - 1) / T; }

// Every thread of the CTA calls it; the first kPlanThreads do the work.  Returns the units W of the
// line.
template <int BK>
__device__ long long plan_build(const AttnArgs& a, PlanShared* sh, int grid) {
  const int per = (a.B + kPlanThreads - 1) / kPlanThreads;
  const int t = threadIdx.x;
  long long v = 0;
  bool single = per == 1;  // every sequence has a run of its own and at most one row tile
  Seq s{0, 0, 0};
  if (t < kPlanThreads) {
    for (int b = t * per; b < min(a.B, (t + 1) * per); ++b) {
      s = seq_at(a, b);
      v += seq_units<BK>(a, s);
      single = single && s.n <= a.tq;
    }
    sh->seq[t] = s;
  }
  plan_scan(sh, v);
  const long long W = sh->before[kPlanThreads];
  const long long even = quotient(W + grid - 1, grid);
  if (t == 0) sh->piece = 0;
  if (!__syncthreads_and(single) || W == 0 || even > 0x3fffffff) return W;
  const int Hv = a.c.Hkv * a.nsub;
  const int tiles = t < kPlanThreads && s.n > 0 ? tiles_of<BK>(keys_of_tile(a, s, 0)) : 0;
  if (t < kPlanThreads) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (sums that matter are at most the grid's size)
      int n = min(pieces_of(tiles, piece_length(a, even, i)), 1 << 12) * Hv;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      if ((t & 31) == 0) sh->fit[t >> 5][i] = n;
    }
  }
  __syncthreads();
  int T = 0;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    int n = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) n += sh->fit[w][i];
    if (n <= grid) T = piece_length(a, even, i);
  }
  if (T > 0) {  // (uniform)
    if (t == 0) sh->piece = T;
    plan_scan(sh, static_cast<long long>(tiles > 0 ? pieces_of(tiles, T) * Hv : 0));
  }
  return W;
}

// The last run that starts at or before w.
__device__ __forceinline__ int plan_run(const PlanShared* sh, long long w) {
  int lo = 0, hi = kPlanThreads;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (sh->before[mid] <= w) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The segment that holds unit w of the line (0 <= w < W).  Called by whole warps, with the same w.
template <int BK>
__device__ Cursor plan_locate(const AttnArgs& a, const PlanShared* sh, long long w) {
  const int per = (a.B + kPlanThreads - 1) / kPlanThreads;
  const int run = plan_run(sh, w);
  long long at = sh->before[run];
  Cursor c;
  c.b = run * per;
  c.s = per == 1 ? sh->seq[run] : seq_at(a, c.b);
  for (int i = 1; i < per && c.b + 1 < a.B; ++i) {  // w < W, so a sequence that holds it comes before B
    const long long here = seq_units<BK>(a, c.s);
    if (w < at + here) break;
    at += here;
    ++c.b;
    c.s = seq_at(a, c.b);
  }
  const int qts = row_tiles(a, c.s);
  const long long per_head = max(1ll, units_before<BK>(a, c.s, qts));
  c.vh = static_cast<int>(quotient(w - at, per_head));
  at += c.vh * per_head;
  int l = 0, h = qts;  // the last row tile that begins at or before w is in [l, h)
  while (h - l > 1) {  // a lane a candidate
    const int step = (h - l + 31) / 32, mine = l + static_cast<int>(threadIdx.x & 31) * step;
    const bool before = mine < h && at + units_before<BK>(a, c.s, mine) <= w;
    const int k = __popc(__ballot_sync(0xffffffffu, before)) - 1;
    l += k * step;
    h = min(h, l + step);
  }
  c.qt = l;
  c.start = at + units_before<BK>(a, c.s, l);
  c.keys = keys_of_tile(a, c.s, l);
  c.tiles = tiles_of<BK>(c.keys);
  return c;
}

// The segment after c's (only called while one exists).
template <int BK>
__device__ __forceinline__ void plan_next(const AttnArgs& a, Cursor& c) {
  c.start += c.tiles + a.seg_cost;
  if (++c.qt >= row_tiles(a, c.s)) {
    c.qt = 0;
    if (++c.vh >= a.c.Hkv * a.nsub) {
      c.vh = 0;
      do {
        ++c.b;
        c.s = seq_at(a, min(c.b, a.B - 1));
      } while (c.s.n == 0 && c.b + 1 < a.B);
    }
  }
  c.keys = keys_of_tile(a, c.s, c.qt);
  c.tiles = tiles_of<BK>(c.keys);
}

// The line's shares: CTA c of `ctas` takes [begin(c), begin(c + 1)), the first `more` one unit more
// than the others.  No share is below min_tiles while that leaves CTAs idle.
struct Shares {
  long long each;
  int more, ctas;
  __device__ __forceinline__ Shares(const AttnArgs& a, long long W, int grid) {
    ctas = static_cast<int>(min(static_cast<long long>(grid), max(1ll, quotient(W + a.min_tiles - 1, a.min_tiles))));
    each = quotient(W, ctas);
    more = static_cast<int>(W - each * ctas);
  }
  __device__ __forceinline__ long long begin(int c) const { return c * each + min(c, more); }
  __device__ __forceinline__ int owner(long long w) const {
    const long long head = more * (each + 1);
    return static_cast<int>(w < head ? quotient(w, each + 1) : more + quotient(w - head, each));
  }
};

// The segments of one CTA, one after the other.
struct Work {
  Cursor cur;
  int t0, t1;     // key tiles of the segment that are this CTA's
  int slot;       // where its partial result goes, -1: the segment is this CTA's alone
  int last;       // last CTA with a part of it, if this one has the first of several; -1 otherwise
  bool final;     // no other segment follows
  long long w, w_hi;
};

// Opens the next segment of the share [k.w, k.w_hi) of which a tile is in it, k.cur being the one that
// holds unit k.w; false if there is none.
template <int BK>
__device__ __forceinline__ bool work_open(const AttnArgs& a, const Shares& sh, int cta, Work& k) {
  while (k.w < k.w_hi) {
    const long long first = k.cur.start + a.seg_cost, end = first + k.cur.tiles;
    k.t0 = static_cast<int>(max(k.w - first, 0ll));
    k.t1 = static_cast<int>(min(k.w_hi, end) - first);
    k.w = end;
    k.final = end >= k.w_hi;
    if (k.t1 > k.t0) {
      const bool whole = k.t0 == 0 && k.t1 == k.cur.tiles;
      k.slot = whole ? -1 : 2 * cta + (k.t0 == 0);
      k.last = k.t0 == 0 && !whole ? sh.owner(end - 1) : -1;
      return true;
    }
    if (!k.final) plan_next<BK>(a, k.cur);
  }
  k.last = -1;
  return false;
}

// This CTA's first segment; false if it has none.
template <int BK>
__device__ bool work_begin(const AttnArgs& a, const PlanShared* sh, long long W, int cta, int grid, Work& k) {
  k.last = -1;
  if (sh->piece > 0) {
    if (cta >= sh->before[kPlanThreads]) return false;
    k.cur.b = plan_run(sh, cta);
    k.cur.s = sh->seq[k.cur.b];
    k.cur.qt = 0;
    k.cur.keys = keys_of_tile(a, k.cur.s, 0);
    k.cur.tiles = tiles_of<BK>(k.cur.keys);
    const int pieces = pieces_of(k.cur.tiles, sh->piece), i = static_cast<int>(cta - sh->before[k.cur.b]);
    k.cur.vh = i / pieces;
    const int p = i % pieces, len = k.cur.tiles / pieces, more = k.cur.tiles % pieces;
    k.t0 = p * len + min(p, more);
    k.t1 = k.t0 + len + (p < more);
    k.slot = pieces == 1 ? -1 : 2 * cta;
    if (p == 0 && pieces > 1) k.last = cta + pieces - 1;
    k.final = true;
    return true;
  }
  const Shares line(a, W, grid);
  if (W == 0 || cta >= line.ctas) return false;
  k.w = line.begin(cta);
  k.w_hi = line.begin(cta + 1);
  k.cur = plan_locate<BK>(a, sh, k.w);
  return work_open<BK>(a, line, cta, k);
}

// The next one (only called after one that is not final).
template <int BK>
__device__ __forceinline__ bool work_next(const AttnArgs& a, long long W, int cta, int grid, Work& k) {
  plan_next<BK>(a, k.cur);
  return work_open<BK>(a, Shares(a, W, grid), cta, k);
}

// Notes for the join, by one thread: k.last and the segment it belongs to (the CTA's last one), or
// that there is none.
__device__ __forceinline__ void leave_record(const AttnArgs& a, int cta, const Work& k) {
  JoinRecord r;
  r.last = k.last;
  if (k.last >= 0) {
    const Cursor& c = k.cur;
    r.slot = k.slot;
    const int kvh = c.vh / a.nsub, sub = c.vh % a.nsub;
    r.heads = min(a.gs, a.g - sub * a.gs);
    r.head = kvh * a.g + sub * a.gs;
    r.rows = min(a.tq, c.s.n - c.qt * a.tq) * a.gs;
    r.tok = c.s.s0 + c.qt * a.tq;
  }
  a.records[cta] = r;
}

}  // namespace smb
