// kk3_cache.cuh - the paged latent cache of the MLA layers: argument blocks, address arithmetic and the work split
// shared by its kernels (kk3_cache.cu: append, evict, the join of attention tiles; kk3_cache_tc.cu: attention and
// attention weight).
//
// A cached position is 512 latent values and 64 rope values (BF16), in a page of `page_size` positions found
// through the sequence's row of the page table. Everything a kernel reads from the device (lengths, cu_new, the
// table) is clamped before it becomes an address: a page number outside the pool reads as zeros, is never written,
// and raises the caller's error word.
#pragma once

#include "kk3_common.cuh"

namespace kk3 {

constexpr int kLat = 512;            // latent values of a position
constexpr int kRope = 64;            // rope values of a position
constexpr int kEntry = kLat + kRope; // 576
constexpr int kMaxSeqs = 4096;       // sequences per call: their tile prefix is kept in shared memory
constexpr int kMaxHeads = 128;

struct CachePages {
  bf16* kv;
  bf16* pe;
  long long kv_page, kv_row, pe_page, pe_row;   // strides in elements
  const int* table;
  long long table_stride;
  int num_pages, page_size, columns, batch;
  unsigned page_magic;   // floor(2^32 / page_size) + 1: position / page_size = mulhi(position, magic) (see page_of)
  int* error_word;
};

// position / page_size for positions below 2^27 and page sizes up to 2^16 without a division: the estimate by the
// rounded-up reciprocal is at most one too large, and one compare mends it.
KK3_DEV int page_of(const CachePages& c, int pos) {
  if (c.page_size == 1) return pos;
  int p = (int)__umulhi((unsigned)pos, c.page_magic);
  if (p * c.page_size > pos) --p;
  return p;
}

KK3_DEV void cache_error(const CachePages& c) {
  if (c.error_word) *reinterpret_cast<volatile int*>(c.error_word) = kErrDevice;
}

// Page of position `pos` of sequence `b`, or -1 (and the error word) when the table names no page of the pool.
KK3_DEV int page_at(const CachePages& c, int b, int pos, int* slot) {
  const int col = page_of(c, pos);
  *slot = pos - col * c.page_size;
  const int page = c.table[(long long)b * c.table_stride + col];
  if ((unsigned)page >= (unsigned)c.num_pages) {
    cache_error(c);
    return -1;
  }
  return page;
}

// Wait for the kernel before this one on the stream (cache_launch_after) and see what it wrote.
KK3_DEV void cache_follow() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The next kernel's CTAs may come in where there is room (they wait in cache_follow until all of this one is written).
// Said at the start: from there to the next kernel's first instruction it takes 3.7 us.
KK3_DEV void cache_go_on() { asm volatile("griddepcontrol.launch_dependents;"); }

// A sequence of one call: its rows in the packed token arrays and its cached positions (new ones included).
struct Seq {
  int q0, n, len;
};
// The sequences of one call, as the device tensors give them.
struct CallSeqs {
  CachePages c;
  const long long* lengths;
  const int* cu_new;
  int tokens;
  int workers;   // CTAs (or CTA pairs) that share the call
  // [workers][4], of the tile that this worker begins and leaves: attention: its first row among all, its rows; weight:
  // its sequence, its first position, and last the sequence's length; both: how many workers share it (0: no such tile)
  int* meta;
  KK3_DEV Seq seq(int b) const {
    Seq s;
    const int a = min(max(cu_new[b], 0), tokens), e = min(max(cu_new[b + 1], a), tokens);
    const long long cap = (long long)c.columns * c.page_size, l = lengths[b];
    s.q0 = a;
    s.n = e - a;
    s.len = (int)(l < 0 ? 0 : l > cap ? cap : l);
    if (l < 0 || l > cap) cache_error(c);
    return s;
  }
};

// --- attention ---------------------------------------------------------------------------------------------

struct AttendArgs : CallSeqs {
  const bf16* q_lat;
  const bf16* q_pe;
  long long ql_tok, ql_head, qp_tok, qp_head;   // strides in elements
  int heads;
  float scale_log2;      // scale * log2(e): the softmax runs on powers of two
  bf16* out;             // [tokens, heads, 512]
  float* lse;            // [tokens, heads]
  float* part;           // [workers][2][tile rows][kPartRow]: running sums of tiles that several workers share
};
constexpr int kFewRows = 16, kPairRows = 128;   // tiles of the two attention kernels
constexpr int kMaxWorkers = 160;                // that the join keeps the statistics of in registers
constexpr int kPartRow = kLat + 4;   // 512 sums, running maximum, running sum, padding to 16 bytes

struct MassArgs : CallSeqs {
  const bf16* q_lat;
  const bf16* q_pe;
  long long ql_tok, ql_head, qp_tok, qp_head;
  const float* lse;      // [tokens, heads]
  int heads;
  float scale_log2;
  const float* mass;     // null: zeros
  long long mass_row;
  float* out;            // [batch, columns * page_size]
  float* part;           // [workers][2][128]: sums of tiles that several workers share
};

// The work of one call is cut into tiles, laid end to end; a tile takes a number of units, one at least, and every
// worker takes an equal run of units, so that short and long sequences, one token and many, all fill the GPU. A tile
// that is cut is joined afterwards from the sums of its workers, in their order.

// One worker's run of units [begin, end) of the call's `total`, and the tile it begins in.
struct Share {
  long long begin, end, total;
  long long at;      // units before the first tile
  int b, t;          // first tile: its sequence and its number within it
  int workers;       // workers that take part (this one does not when its number is not below)
  Seq seq;           // the first tile's sequence
  KK3_DEV int holder(long long end) const { return (int)((end * workers + total - 1) / total) - 1; }   // of the unit before `end`
};

// Attention: a tile is `rows` (token, head) rows of one sequence over the positions that its last row sees, a unit
// `unit` positions.
struct AttendSplit {
  int rows, heads, unit;
  int cost;   // what a tile costs besides its units, in units: they lie before the tile's own
  KK3_DEV int tiles(const Seq& s) const { return (s.n * heads + rows - 1) / rows; }
  KK3_DEV int sees(const Seq& s, int t) const {   // positions that the tile's last row sees, 0 or less: none
    return s.len - s.n + min(s.n - 1, (int)(((unsigned)(t + 1) * rows - 1) / (unsigned)heads)) + 1;
  }
  KK3_DEV int units(const Seq& s, int t) const {
    const int n = sees(s, t);
    return n > unit ? (n + unit - 1) / unit : 1;
  }
  KK3_DEV int size(const Seq& s, int t) const { return units(s, t) + cost; }
  KK3_DEV long long all(const Seq& s) const {   // of its tiles
    long long n = 0;
    for (int t = 0; t < tiles(s); ++t) n += size(s, t);
    return n;
  }
  // the tile's units that a worker takes, of a tile that begins at `at`
  KK3_DEV int from(const Share& sh, long long at, int units) const { return (int)min((long long)units, max(0ll, sh.begin - at - cost)); }
  KK3_DEV int to(const Share& sh, long long at, int units) const { return (int)min((long long)units, max(0ll, sh.end - at - cost)); }
};
// Attention weight: a tile is `positions` positions of one sequence over the rows that see its first, a unit `rows`
// (token, head) rows.
struct MassSplit {
  int positions, rows, heads;
  KK3_DEV int tiles(const Seq& s) const { return s.n > 0 ? (s.len + positions - 1) / positions : 0; }
  KK3_DEV int first_unit(const Seq& s, int t) const {   // first rows that see position t * positions
    return max(0, t * positions - (s.len - s.n)) * heads / rows;
  }
  KK3_DEV int units(const Seq& s, int t) const { return (s.n * heads + rows - 1) / rows - first_unit(s, t); }
  KK3_DEV int size(const Seq& s, int t) const { return units(s, t); }
  KK3_DEV long long all(const Seq& s) const {   // of its tiles: every row sees the first ones whole
    const int count = tiles(s), whole = min(count, max(0, s.len - s.n) / positions + 1);
    long long n = count ? (long long)whole * units(s, 0) : 0;
    for (int t = whole; t < count; ++t) n += size(s, t);
    return n;
  }
};

// inclusive sums over the lanes of a warp
template <class T>
KK3_DEV T lane_sums(T v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += u;
  }
  return v;
}

// Sum over the threads of a block of NT (a multiple of 32) threads before this one; *total over all of them. `red`
// is shared memory of NT / 32 + 1 long longs.
template <int NT>
KK3_DEV long long block_scan(long long mine, long long* red, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long v = lane_sums(mine);
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  long long before = v - mine, all = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  *total = all;
  return before;
}

// The worker's part of `total` units: false if it has none. A worker takes min_units units at least: shorter pieces cost
// more to join than they save.
KK3_DEV bool plan_part(Share& sh, long long total, int worker, int min_units, int workers) {
  const long long most = (total + min_units - 1) / min_units;
  sh.total = total;
  sh.workers = (int)(most > workers ? workers : most);
  sh.begin = sh.end = sh.at = 0;
  sh.b = sh.t = 0;
  sh.seq = Seq{0, 0, 0};
  if (worker >= sh.workers) return false;
  if (total < 1 << 22) {   // 32-bit divisions: the 64-bit ones take 600 clocks
    sh.begin = (unsigned)total * (unsigned)worker / (unsigned)sh.workers;
    sh.end = (unsigned)total * (unsigned)(worker + 1) / (unsigned)sh.workers;
  } else {
    sh.begin = total * worker / sh.workers;
    sh.end = total * (worker + 1) / sh.workers;
  }
  return true;
}

// The plan of up to 128 sequences of up to 32 tiles each, by every warp for itself, four sequences a lane; false: there
// are more. (A plan by the whole CTA has four barriers and takes 4700 clocks where this takes 1500, a third of the
// time of a small call.)
constexpr int kPlanDeep = 4;
template <class Split>
KK3_DEV bool plan_small(const CallSeqs& a, const Split& split, int worker, int min_units, Share& sh) {
  const int lane = threadIdx.x & 31, B = a.c.batch;
  if (B > 32 * kPlanDeep) return false;
  const int per = (B + 31) / 32, lo = lane * per;
  Seq s[kPlanDeep];
  long long size[kPlanDeep], mine = 0;
  bool small = true;
#pragma unroll
  for (int i = 0; i < kPlanDeep; ++i) {
    s[i] = i < per && lo + i < B ? a.seq(lo + i) : Seq{0, 0, 0};
    small = small && split.tiles(s[i]) <= 32;
  }
  if (!__all_sync(0xffffffffu, small)) return false;
#pragma unroll
  for (int i = 0; i < kPlanDeep; ++i) {
    size[i] = split.all(s[i]);
    mine += size[i];
  }
  const long long incl = lane_sums(mine);
  if (!plan_part(sh, __shfl_sync(0xffffffffu, incl, 31), worker, min_units, a.workers)) return true;
  // the sequence: of the first lane whose units end behind `begin`, and there the first one
  long long u = incl - mine;
  int i = 0;
  Seq mine_seq = s[0];
#pragma unroll
  for (int k = 0; k + 1 < kPlanDeep; ++k)
    if (i == k && u + size[k] <= sh.begin) {
      u += size[k];
      i = k + 1;
      mine_seq = s[k + 1];
    }
  const int from = __ffs(__ballot_sync(0xffffffffu, incl > sh.begin)) - 1;
  sh.b = from * per + __shfl_sync(0xffffffffu, i, from);
  u = __shfl_sync(0xffffffffu, u, from);
  sh.seq = Seq{__shfl_sync(0xffffffffu, mine_seq.q0, from), __shfl_sync(0xffffffffu, mine_seq.n, from),
               __shfl_sync(0xffffffffu, mine_seq.len, from)};
  // its tile: lane t looks at tile t
  const int k = lane < split.tiles(sh.seq) ? split.size(sh.seq, lane) : 0;
  u += lane_sums(k);
  sh.t = __ffs(__ballot_sync(0xffffffffu, u > sh.begin)) - 1;
  sh.at = __shfl_sync(0xffffffffu, u - k, sh.t);
  return true;
}

// Computed by every CTA for itself; all NT threads take part. `room` is shared memory of kPlanBytes, `red` of
// NT / 32 + 4 long longs.
constexpr int kPlanBytes = kMaxSeqs * (int)sizeof(Seq) + (kMaxSeqs + 1) * 4;
template <int NT, class Split>
KK3_DEV Share plan_share(const CallSeqs& a, const Split& split, int worker, int min_units, void* room, long long* red) {
  Share sh;
  if (plan_small(a, split, worker, min_units, sh)) return sh;
  const int tid = threadIdx.x, B = a.c.batch;
  Seq* seqs = reinterpret_cast<Seq*>(room);
  int* prefix = reinterpret_cast<int*>(seqs + B);
  const int per = (B + NT - 1) / NT, lo_b = min(B, tid * per), hi_b = min(B, lo_b + per);
  long long mine = 0, all;
  for (int b = lo_b; b < hi_b; ++b) {
    seqs[b] = a.seq(b);
    mine += split.tiles(seqs[b]);
  }
  int at = (int)block_scan<NT>(mine, red, &all);
  const int tiles = (int)all;
  for (int b = lo_b; b < hi_b; ++b) {
    prefix[b] = at;
    at += split.tiles(seqs[b]);
  }
  if (tid == 0) prefix[B] = tiles;
  __syncthreads();
  // units before each thread's run of tiles
  const int run = (tiles + NT - 1) / NT, g0 = min(tiles, tid * run), g1 = min(tiles, g0 + run);
  int b0 = 0;
  if (g0 < g1) {   // the last sequence whose tiles begin at or before g0
    int hi = B;
    while (hi - b0 > 1) {
      const int mid = (b0 + hi) >> 1;
      if (prefix[mid] <= g0) b0 = mid; else hi = mid;
    }
  }
  mine = 0;
  if (g0 < g1) {
    int b = b0;
    for (int g = g0; g < g1; ++g) {
      while (g >= prefix[b + 1]) ++b;
      mine += split.size(seqs[b], g - prefix[b]);
    }
  }
  long long total;
  const long long before = block_scan<NT>(mine, red, &total);
  if (!plan_part(sh, total, worker, min_units, a.workers)) return sh;
  long long* found = red + NT / 32;
  if (before <= sh.begin && sh.begin < before + mine) {   // exactly one thread
    int b = b0;
    long long u = before;
    for (int g = g0; g < g1; ++g) {
      while (g >= prefix[b + 1]) ++b;
      const int k = split.size(seqs[b], g - prefix[b]);
      if (u + k > sh.begin) {
        found[0] = b;
        found[1] = g - prefix[b];
        found[2] = u;
        break;
      }
      u += k;
    }
  }
  __syncthreads();
  sh.b = (int)found[0];
  sh.t = (int)found[1];
  sh.at = found[2];
  sh.seq = seqs[sh.b];
  __syncthreads();
  return sh;
}

}  // namespace kk3
