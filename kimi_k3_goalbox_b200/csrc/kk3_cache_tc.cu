// kk3_cache_tc.cu - tensor-core kernels of the paged latent cache (tcgen05 on CTA pairs, sm_100a): attention of new
// tokens and the accumulated attention weight.
//
// Operands come through the page table by TMA, in blocks of 64 dims in the 128-byte swizzled form that the matrix
// instructions read: boxes of as many rows as divide a page and a tile, or gathers of four rows where that is below
// eight (odd page sizes) and where rows behind a sequence's end have to arrive as zeros. A gather costs its issuing
// warp as much as a box of any size (about 100 clocks), so boxes carry the bulk. Two CTAs of a cluster work as one
// (cta_group::2): each loads half of the second operand, which halves the shared-memory reads per matrix instruction,
// the bound of these shapes at 128 bytes a clock.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <limits.h>
#include <string.h>

#include <type_traits>

#include "kk3_cache.cuh"
#include "kk3_cache_host.h"
#include "kk3_tcgen05.cuh"

namespace kk3 {

constexpr int kBlocks = kEntry / 64;                    // 64-dim blocks of an entry
constexpr unsigned long long kWaitNs = 2000000000ull;   // bound of every wait; a healthy one takes microseconds

// The tensors of a call: cached entries in boxes of `box` rows and row by row, query rows in boxes. Cached rows are
// numbered page * ratio + slot, query rows token * heads + head.
struct PairMaps {
  CUtensorMap kv_box, pe_box, kv_row, pe_row, ql, qp;
};
struct PairRows {
  int kv_ratio, pe_ratio;   // rows from one page to the next
  int kv_end, pe_end;       // number of the first row behind the pool: reads as zeros
  int box;                  // rows of a box: divides a page and 64, 8 at least; 0: gathers only
};

// Thread i of the CTA has map i fetched, before the first copy needs it.
KK3_DEV void fetch_maps(const PairMaps& maps) {
  if (threadIdx.x < sizeof(PairMaps) / sizeof(CUtensorMap))
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<const CUtensorMap*>(&maps) + threadIdx.x) : "memory");
}
KK3_DEV unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
KK3_DEV unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// shared::cluster address of `addr` in CTA `rank` of the cluster
KK3_DEV unsigned in_cta(unsigned addr, unsigned rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
KK3_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
KK3_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
KK3_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrival on a barrier of either CTA. What these arrivals hand over stays in this SM: tensor memory that was read or
// written to the end (tcgen05.wait, tcgen05.fence) and shared memory that was fenced towards the matrix instructions
// (fence.proxy.async), both of which this SM's half of the instruction then uses; no other CTA reads it. So they are
// released at CTA scope: at cluster scope an arrival waits about 1800 clocks for all of the thread's memory traffic.
KK3_DEV void arrive_cluster(unsigned addr) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Bounded wait; false when it ran out or another role of the CTA gave up (*dead). The part that waits is not inlined:
// the roles' loops stay short.
static __device__ __noinline__ bool pair_wait_on(int* error_word, unsigned bar, unsigned parity, volatile int* dead) {
  const unsigned long long t0 = globaltimer();
  for (unsigned spin = 1;; ++spin) {
    if (mbar_test(bar, parity)) return true;
    if ((spin & 15) == 0 || spin == 1) {
      if (*dead) return false;
      if (globaltimer() - t0 > kWaitNs) {
        *dead = 1;
        if (error_word) *reinterpret_cast<volatile int*>(error_word) = kErrTimeout;
        return false;
      }
    }
  }
}
// What a tile's sums become when a wait of the CTA has run out, so that no caller takes what was allocated or half done
// for a result: NaN, which the division by a row's sum and the join of cut tiles carry to all that the tile gives. All
// of the tile's waits lie before a barrier that its threads pass before they ask.
KK3_DEV float or_lost(float v, volatile int* dead) { return *dead ? __int_as_float(0x7fffffff) : v; }
KK3_DEV bool pair_wait(const CachePages& c, unsigned bar, unsigned parity, volatile int* dead) {
  return mbar_test(bar, parity) || pair_wait_on(c.error_word, bar, parity, dead);
}
// Copies are issued by one lane (`me`) of a converged warp: 50 clocks each, against 90 in a branch of one lane, where
// every operand moves to the uniform registers anew.
KK3_DEV bool elect_one() {
  unsigned p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
// Rows row[0..3] of 64 elements from column x into 512 bytes of this CTA's shared memory; the bytes are counted on
// `bar`, a barrier of either CTA of the pair.
KK3_DEV void gather4(bool me, unsigned dst, const CUtensorMap* map, int x, const int4& row, unsigned bar) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %8, 0;\n"
      " @p cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7];\n}"
      ::"r"(dst), "l"(map), "r"(x), "r"(row.x), "r"(row.y), "r"(row.z), "r"(row.w), "r"(bar), "r"((unsigned)me)
      : "memory");
}
// A box of the map's rows from `row` on, likewise.
KK3_DEV void load_box(bool me, unsigned dst, const CUtensorMap* map, int x, int row, unsigned bar) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n"
      " @p cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
      "[%1, {%2, %3}], [%4];\n}"
      ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(bar), "r"((unsigned)me)
      : "memory");
}
KK3_DEV void pair_mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// one arrival on `bar` of both CTAs when the matrix instructions issued so far are done
KK3_DEV void pair_commit(unsigned bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((unsigned short)3) : "memory");
}
KK3_DEV void pair_alloc(unsigned dst, unsigned ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(ncols) : "memory");
}
KK3_DEV void pair_dealloc(unsigned taddr, unsigned ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
KK3_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 TMEM lanes (one per thread of the warp) x 32 consecutive 32-bit columns
KK3_DEV void tmem_ld32(unsigned taddr, float (&v)[32]) {
  unsigned r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// instruction descriptor: kind::f16, D = F32, A = B = BF16, M rows and N columns over the pair, operands K-major
KK3_DEV constexpr unsigned pair_idesc(int m, int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24);
}

// The rows of 256 cached positions of a sequence, behind `end` or without a page: the first past the pool. A copying
// warp looks them up together (eight positions a lane, which lie in one page unless pages have odd sizes), one table
// ahead: fetch() only reads the page table, write() turns what came into rows, from which all copies are issued.
struct RowTab {
  alignas(16) int kv[256];
  alignas(16) int pe[256];
};
struct PageIds {
  int id[8] = {};
  KK3_DEV void fetch(const CachePages& c, const PairRows& pr, int b, int pos, int end) {
    pos += (threadIdx.x & 31) * 8;
    const int* table = c.table + (long long)b * c.table_stride;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((i == 0 || !pr.box) && pos + i < end) id[i] = table[page_of(c, pos + i)];
  }
  template <bool BOXED>
  KK3_DEV void write(const CachePages& c, const PairRows& pr, int pos, int end, RowTab& tab) const {
    const int lane = threadIdx.x & 31;
    pos += lane * 8;
    int kv[8], pe[8];
    if (BOXED) {
      const bool fine = (unsigned)id[0] < (unsigned)c.num_pages;
      const int slot = pos - page_of(c, pos) * c.page_size, left = fine ? end - pos : 0;
      const int kv0 = id[0] * pr.kv_ratio + slot, pe0 = id[0] * pr.pe_ratio + slot;
      if (!fine && pos < end) cache_error(c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        kv[i] = i < left ? kv0 + i : pr.kv_end;
        pe[i] = i < left ? pe0 + i : pr.pe_end;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        kv[i] = pr.kv_end;
        pe[i] = pr.pe_end;
        if (pos + i < end) {
          const int in = pos + i - page_of(c, pos + i) * c.page_size;
          if ((unsigned)id[i] < (unsigned)c.num_pages) {
            kv[i] = id[i] * pr.kv_ratio + in;
            pe[i] = id[i] * pr.pe_ratio + in;
          } else {
            cache_error(c);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<int4*>(&tab.kv[lane * 8 + i]) = make_int4(kv[i], kv[i + 1], kv[i + 2], kv[i + 3]);
      *reinterpret_cast<int4*>(&tab.pe[lane * 8 + i]) = make_int4(pe[i], pe[i + 1], pe[i + 2], pe[i + 3]);
    }
  }
};
// COUNT positions of the table in boxes of BOX rows, their row numbers in registers; BOX 0: row by row, from the table.
template <int COUNT, int BOX>
struct Boxes {
  static constexpr int kMany = BOX ? COUNT / (BOX ? BOX : 1) : 1;
  int kv[kMany], pe[kMany];
  const RowTab* tab;
  int off;
  KK3_DEV void take(const RowTab& t, int from) {
    tab = &t;
    off = from;
#pragma unroll
    for (int i = 0; i < kMany; ++i) {
      kv[i] = t.kv[from + i * BOX];
      pe[i] = t.pe[from + i * BOX];
    }
  }
  // 64-dim block `d` of them into [COUNT][64] at `dst`
  KK3_DEV void load(bool me, const PairMaps& m, int d, unsigned dst, unsigned bar) const {
    const bool rope = d == kBlocks - 1;
    const int x = rope ? 0 : d * 64;
    if (BOX) {
#pragma unroll
      for (int i = 0; i < kMany; ++i)
        load_box(me, dst + i * BOX * 128, rope ? &m.pe_box : &m.kv_box, x, rope ? pe[i] : kv[i], bar);
    } else {
      const int* rows = (rope ? tab->pe : tab->kv) + off;
#pragma unroll 4
      for (int k = 0; k < COUNT; k += 4)
        gather4(me, dst + k * 128, rope ? &m.pe_row : &m.kv_row, x, *reinterpret_cast<const int4*>(&rows[k]), bar);
    }
  }
};
// f(integral constant of the call's box)
template <class F>
KK3_DEV void with_box(int box, const F& f) {
  switch (box) {
    case 64: return f(std::integral_constant<int, 64>());
    case 32: return f(std::integral_constant<int, 32>());
    case 16: return f(std::integral_constant<int, 16>());
    case 8: return f(std::integral_constant<int, 8>());
    default: return f(std::integral_constant<int, 0>());
  }
}

// ---------------------------------------------------------------------------------------------
// Attention weight of cached positions: w_p = sum over rows of 2^(s_p - lse), s_p = q . e_p.
//
// One product, positions x rows, with the positions as the 256 rows of the pair's matrix instruction: a thread then
// owns a position (its TMEM lane) and adds up its columns in registers, in row order; no reduction crosses threads
// and no atomic is needed. A tile is 256 positions, 147 KB in each CTA, that stay in shared memory while the
// sequence's rows pass through a ring in units of `rows` x 576 dims, half of them in each CTA; two accumulators let
// the sums of one unit run under the products of the next. Where the rows fit one unit (single tokens) the tile's
// blocks are freed one by one instead, and the kernel streams the cache with up to 147 KB in flight in each SM.
//
// Bounds of a unit of 256 rows: 4608 clocks of tensor time (256 x 256 x 576 products at 4096 a clock and SM), as many
// of shared-memory reads (16 KB per 128-clock instruction), and 2048 of exponentials (16 a clock). Measured: 32 tokens
// x 96 heads over four sequences of up to 8192 positions 70 us, 1130 TFLOP/s (47 us at the rate of a plain product): the
// ring's four slots of 16 KB cover 2048 clocks of products, and a slot's turn takes about that;
// 16 single tokens x 12 heads, bound by the cache's bytes, 29 us, 3.7 TB/s: 3 us for the work split, 7 until the first
// tile's sums, then 3.7 us a tile, the rate of HBM.

constexpr int kMassPos = 256;
constexpr int kMassSums = 256, kMassThreads = kMassSums + 64;   // warps 0-7 sums, 8 copies, 9 matrix instructions and TMEM
constexpr int kMassKBlock = 128 * 128;
constexpr int kMassRing = 65536;
constexpr int kMassSlots = 16;
struct MassCtl {
  unsigned long long full[kMassSlots], empty[kMassSlots], kempty[kBlocks], dfull[2], dempty[2], done;
  unsigned tmem;
  int dead;
  long long red[kMassThreads / 32 + 4];
  alignas(16) float lse[2][256];   // read four at a time
  alignas(16) int sees[2][256];
  float sum[128];
  RowTab rows;
};
constexpr int kMassSmem = kBlocks * kMassKBlock + kMassRing + (int)sizeof(MassCtl) + 1024;
static_assert(kMassSmem <= 232448, "shared memory of a CTA");

// What the call leaves as it is: positions behind the sequences' ends, and sequences without new tokens. The CTAs are
// dealt out to the sequences; the first kMassSums threads of each take part, in CTAs with tiles and without alike: the
// CTAs of a sequence take its positions in turn, so their steps have to be of one width.
KK3_DEV void mass_rest(const MassArgs& a, int tid) {
  if (tid >= kMassSums) return;
  const long long cap = (long long)a.c.columns * a.c.page_size;
  const int per = max(1, (int)gridDim.x / a.c.batch), groups = gridDim.x / per;
  if ((int)blockIdx.x >= groups * per) return;
  for (int b = blockIdx.x / per; b < a.c.batch; b += groups) {
    const Seq s = a.seq(b);
    const float* from = a.mass ? a.mass + b * a.mass_row : nullptr;
#pragma unroll 4
    for (long long p = (s.n > 0 ? s.len : 0) + (int)(blockIdx.x % per) * kMassSums + tid; p < cap; p += per * kMassSums)
      a.out[b * cap + p] = from ? from[p] : 0.0f;
  }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMassThreads, 1)
    kk3_cache_mass_kernel(const MassArgs a, const PairRows pr, const __grid_constant__ PairMaps maps, int rows) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  MassCtl& ctl = *reinterpret_cast<MassCtl*>(base + kBlocks * kMassKBlock + kMassRing);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, worker = blockIdx.x >> 1;
  const unsigned rank = cluster_rank();
  const unsigned kbase = smem_u32(base), qbase = kbase + kBlocks * kMassKBlock;
  fetch_maps(maps);
  const int half = rows / 2, slot_bytes = half * 128, slots = min(kMassSlots, kMassRing / slot_bytes);
  const MassSplit split{kMassPos, rows, a.heads};
  const unsigned full = smem_u32(ctl.full), empty = smem_u32(ctl.empty), kempty = smem_u32(ctl.kempty),
                 dfull = smem_u32(ctl.dfull), dempty = smem_u32(ctl.dempty), done = smem_u32(&ctl.done);
  volatile int* dead = &ctl.dead;
  if (tid == 0) {
    for (int i = 0; i < kMassSlots; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kBlocks; ++i) mbar_init(kempty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(dfull + 8 * i, 1);
      mbar_init(dempty + 8 * i, 16);   // eight warps of either CTA
    }
    mbar_init(done, 1);
    ctl.dead = 0;
    fence_mbar_init();
  }
  __syncwarp();
  cluster_arrive();   // the peer's barriers are needed after the plan
  const Share sh = plan_share<kMassThreads>(a, split, worker, 1, base, ctl.red);
  fence_async_smem();   // the plan of a large call lay where the copies come
  cache_go_on();
  if (tid == 0 && rank == 0) a.meta[worker * 4 + 2] = 0;
  if (worker >= sh.workers) {   // both CTAs of the pair
    mass_rest(a, tid);
    cluster_wait();
    return;
  }
  if (warp == 9) pair_alloc(smem_u32(&ctl.tmem), 512);
  tc_fence_before();
  __syncthreads();
  cluster_wait();
  tc_fence_after();
  const unsigned tmem = *reinterpret_cast<volatile unsigned*>(&ctl.tmem);

  int b = sh.b, t = sh.t;
  long long at = sh.at;
  if (warp == 8) {
    // ---- copies
    const unsigned lead_full = in_cta(full, 0);
    const bool me = elect_one();
    int slot = 0, phase = 0, tile = 0, ahead_b = -1, ahead_t = -1;   // the tile whose page ids are there
    PageIds ids;
    bool ok = true;
    Seq s = sh.seq;
    while (ok && at < sh.end) {
      for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
      const int units = split.units(s, t), first = split.first_unit(s, t);
      const int u0 = (int)max(0ll, sh.begin - at), u1 = (int)min((long long)units, sh.end - at);
      if (ahead_b != b || ahead_t != t) ids.fetch(a.c, pr, b, t * kMassPos, s.len);
      if (pr.box) ids.write<true>(a.c, pr, t * kMassPos, s.len, ctl.rows);
      else ids.write<false>(a.c, pr, t * kMassPos, s.len, ctl.rows);
      __syncwarp();
      ids.fetch(a.c, pr, b, (t + 1) * kMassPos, s.len);
      ahead_b = b;
      ahead_t = t + 1;
      with_box(pr.box, [&](auto box) {
        Boxes<128, decltype(box)::value> boxes;
        boxes.take(ctl.rows, (int)rank * 128);
        for (int u = u0; ok && u < u1; ++u) {
          const int q = s.q0 * a.heads + (first + u) * rows + (int)rank * half;   // rows behind the sequence's: masked
#pragma unroll 1
          for (int d = 0; d < kBlocks; ++d) {
            const unsigned bar = lead_full + 8 * slot, qd = qbase + slot * slot_bytes;
            ok = pair_wait(a.c, empty + 8 * slot, phase ^ 1, dead);
            if (u == u0) ok = pair_wait(a.c, kempty + 8 * d, (tile & 1) ^ 1, dead) && ok;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (rank == 0 && me) mbar_arrive_tx(full + 8 * slot, 2 * (slot_bytes + (u == u0 ? kMassKBlock : 0)));
            __syncwarp();
            if (u == u0) boxes.load(me, maps, d, kbase + d * kMassKBlock, bar);
            load_box(me, qd, d < kBlocks - 1 ? &maps.ql : &maps.qp, d < kBlocks - 1 ? d * 64 : 0, q, bar);
            if (++slot == slots) {
              slot = 0;
              phase ^= 1;
            }
          }
        }
      });
      __syncwarp();   // the table is read
      at += units;
      ++t;
      ++tile;
    }
    // after a failed wait: a bounded time for the copies in flight (else their consumers waited for them)
    if (!ok && rank == 0 && lane == 0)
      for (int i = 0; i < slots; ++i) mbar_wait_for(full + 8 * i, i < slot ? phase : phase ^ 1, kWaitNs);
    __syncwarp();
  } else if (warp == 9) {
    // ---- matrix instructions: one thread of the pair
    if (lane == 0 && rank == 0) {
      const unsigned idesc = pair_idesc(256, rows);
      int job = 0, unit = 0;
      bool ok = true;
      Seq s = sh.seq;
      while (ok && at < sh.end) {
        for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
        const int units = split.units(s, t);
        const int u0 = (int)max(0ll, sh.begin - at), u1 = (int)min((long long)units, sh.end - at);
        for (int u = u0; ok && u < u1; ++u, ++unit) {
          const int buf = unit & 1;
          ok = pair_wait(a.c, dempty + 8 * buf, ((unit >> 1) & 1) ^ 1, dead);
          tc_fence_after();
          for (int d = 0; ok && d < kBlocks; ++d, ++job) {
            const int slot = job % slots;
            ok = pair_wait(a.c, full + 8 * slot, (job / slots) & 1, dead);
            if (!ok) break;
            tc_fence_after();
            const unsigned long long ka = sdesc_sw128(kbase + d * kMassKBlock), qa = sdesc_sw128(qbase + slot * slot_bytes);
#pragma unroll
            for (int k = 0; k < 4; ++k) pair_mma(tmem + buf * 256, ka + k * 2, qa + k * 2, idesc, (unsigned)(d | k));
            pair_commit(empty + 8 * slot);
            if (u == u1 - 1) pair_commit(kempty + 8 * d);
          }
          if (ok) pair_commit(dfull + 8 * buf);
        }
        at += units;
        ++t;
      }
      pair_commit(done);   // all matrix instructions end before TMEM is given back
      mbar_wait_for(done, 0, kWaitNs);
    }
    __syncwarp();
  } else {
    // ---- sums: thread = position; warps 0-3 take the first half of the columns, warps 4-7 the second
    mass_rest(a, tid);
    const unsigned tlane = (unsigned)((warp & 3) * 32) << 16, lead_dempty = in_cta(dempty, 0);
    const int group = warp >> 2, row = tid & 127;
    int unit = 0;
    bool ok = true;
    Seq s = sh.seq;
    while (at < sh.end) {   // after a failed wait the rounds go on without work: the warps meet at barriers
      for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
      const int units = split.units(s, t), first = split.first_unit(s, t);
      const int u0 = (int)max(0ll, sh.begin - at), u1 = (int)min((long long)units, sh.end - at);
      const int pos = t * kMassPos + (int)rank * 128 + row;
      const long long all = (long long)s.n * a.heads;
      // a thread fetches one row's log sum, one unit ahead (rows that do not exist or see nothing: -infinity)
      const auto fetch = [&](int u) {
        const long long g = (long long)(first + u) * rows + tid;
        return tid < rows && u < u1 && g < all ? a.lse[(long long)s.q0 * a.heads + g] : -INFINITY;
      };
      float next = fetch(u0), sum = 0.0f;
      for (int u = u0; u < u1; ++u, ++unit) {
        const int buf = unit & 1;
        const long long g0 = (long long)(first + u) * rows;
        if (tid < rows) {
          ctl.lse[buf][tid] = next == -INFINITY ? -INFINITY : -next * 1.4426950408889634f;
          ctl.sees[buf][tid] = g0 + tid < all ? s.len - s.n + (int)((g0 + tid) / a.heads) + 1 : 0;
        }
        next = fetch(u + 1);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        // rows that see not all of the tile, or are another sequence's or no one's: select
        const bool causal = g0 + rows > all || s.len - s.n + (int)(g0 / a.heads) + 1 < min(s.len, (t + 1) * kMassPos);
        ok = pair_wait(a.c, dfull + 8 * buf, (unit >> 1) & 1, dead) && ok;
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        if (ok) {
#pragma unroll 1
          for (int c = group * 32; c < rows; c += 64) {
            float v[32];
            tmem_ld32(tmem + tlane + buf * 256 + c, v);
            tmem_ld_wait();
            float part[4] = {};
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 l = *reinterpret_cast<const float4*>(&ctl.lse[buf][c + i]);
              float w[4] = {ex2(fmaf(v[i], a.scale_log2, l.x)), ex2(fmaf(v[i + 1], a.scale_log2, l.y)),
                            ex2(fmaf(v[i + 2], a.scale_log2, l.z)), ex2(fmaf(v[i + 3], a.scale_log2, l.w))};
              if (causal) {
                const int4 n = *reinterpret_cast<const int4*>(&ctl.sees[buf][c + i]);
                w[0] = pos < n.x ? w[0] : 0.0f;
                w[1] = pos < n.y ? w[1] : 0.0f;
                w[2] = pos < n.z ? w[2] : 0.0f;
                w[3] = pos < n.w ? w[3] : 0.0f;
              }
#pragma unroll
              for (int k = 0; k < 4; ++k) part[k] += w[k];
            }
            sum += (part[0] + part[1]) + (part[2] + part[3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(lead_dempty + 8 * buf);
      }
      if (group == 1) ctl.sum[row] = sum;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (group == 0) {
        sum = or_lost(sum + ctl.sum[row], dead);
        if (u0 == 0 && u1 == units) {
          if (pos < s.len) {
            const long long cap = (long long)a.c.columns * a.c.page_size;
            a.out[b * cap + pos] = (a.mass ? a.mass[b * a.mass_row + pos] : 0.0f) + sum;
          }
        } else {
          a.part[(worker * 2 + (u0 == 0 ? 1 : 0)) * kMassPos + rank * 128 + row] = sum;
          if (u0 == 0 && tid == 0 && rank == 0) {
            a.meta[worker * 4] = b;
            a.meta[worker * 4 + 1] = t * kMassPos;
            a.meta[worker * 4 + 2] = sh.holder(at + units) - worker + 1;
            a.meta[worker * 4 + 3] = s.len;
          }
        }
      }
      at += units;
      ++t;
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // neither CTA gives up its memory while the other's instructions may use it
  if (warp == 9) pair_dealloc(tmem, 512);
}

__global__ void __launch_bounds__(kMassPos) kk3_cache_mass_join_kernel(const MassArgs a) {
  cache_follow();
  const int worker = blockIdx.x, n = a.meta[worker * 4 + 2];
  if (n == 0) return;
  const int b = a.meta[worker * 4], pos = a.meta[worker * 4 + 1] + threadIdx.x;
  if (pos >= a.meta[worker * 4 + 3]) return;
  float sum = 0.0f;
#pragma unroll 4
  for (int w = 0; w < n; ++w) sum += a.part[((worker + w) * 2 + (w == 0 ? 1 : 0)) * kMassPos + threadIdx.x];
  const long long cap = (long long)a.c.columns * a.c.page_size;
  a.out[b * cap + pos] = (a.mass ? a.mass[b * a.mass_row + pos] : 0.0f) + sum;
}

// ---------------------------------------------------------------------------------------------
// Attention: s = scale (q . e_p), running maximum m and sum l per row, O = O 2^(m - m') + sum_p 2^(s_p - m') c_p.
//
// A tile is 128 (token, head) rows of one sequence, 64 in each CTA, a unit 256 positions. The FP32 sums of 512 output
// dims for 128 rows would fill TMEM; the pair's M = 128 form spreads them over both CTAs (64 rows in either, half of
// an instruction's columns in lanes 0-63 and half in lanes 64-127), 256 columns in all, next to two score buffers of
// 128. Every instruction has 256 columns: one takes 64 clocks then, and about as much to issue whatever its size (57
// clocks measured, 175 more for a commit), so narrower ones would leave the tensor cores waiting.
//
// Per unit each CTA loads 128 of the positions (nine blocks of 64 dims) for the scores, and half of the output dims of
// all 256 (eight pieces of 64 positions x 128 dims) for the sums, 16 KB each, through a ring of four and one of three.
// Scores run one unit ahead of sums, and a thread each issues them: what one spends in commits is the other's.
//
// Softmax: four threads per row, 64 of a unit's positions each, that exchange maxima through shared memory. The running
// maximum moves only when it is exceeded by more than 2^8 (probabilities stay below 256, harmless in BF16 and FP32), so
// the sums in TMEM are rarely rescaled. Probabilities are rounded to BF16 for the second product, the type that the
// instruction takes with BF16 latents; the running sum adds them unrounded, since lse is an FP32 result.
//
// Both CTAs bring their part of every block and piece, if only zeros for positions behind the end (rows past the pool,
// which cost no traffic): a CTA that sat a slot's turn out could be passed by two of its phases and wait for good.
//
// Bounds of a unit: 4352 clocks of tensor time (128 x 256 x 1088 products at 4096 a clock and SM), 4200 to issue its
// scores, 278 KB of loads in each SM (mostly from L2). Measured: two chunks of 1024 tokens x 12 heads over up to 8192
// positions 299 us, 1090 TFLOP/s (a plain product: 1679; back to back, at lower clocks, 312 us), 8600 clocks a unit, the
// tensor pipe active for half of them: a slot's turn (copy issued, L2, instructions, commit) takes more than 2000 clocks,
// which seven slots do not cover, and there is no shared memory for more (an eighth in place of half of P took 311 us,
// since the halves then wait for one another). Three prompts of 900 tokens x 24 heads 99 to 107 us: tiles of two or three
// units each, whose first scores, last sums and epilogue (6 us) nothing overlaps.
// Eight single tokens x 96 heads over up to 8192 positions 36 us: 7 us to the first scores, three units of 3.6 us, 8 us for
// the last sums and the running sums' way out, 8 us for their join.

constexpr int kPaUnit = 256;
constexpr int kPaThreads = 384;        // warps 0-7 softmax, 8 and 9 copies and instructions of scores, 10 and 11 of sums
constexpr int kPaQBlock = 64 * 128;    // 64 rows of 64 dims
constexpr int kPaBlock = 128 * 128;    // 128 positions x 64 dims, or 64 positions x 128 dims
constexpr int kPaKSlots = 4, kPaVSlots = 3;   // 16 KB each: nine blocks and eight pieces a unit
constexpr int kPaMinUnits = 3;
constexpr int kPaTileCost = 2;   // what a tile costs besides its units, in units: query load, first and last latencies
constexpr float kPaSlack = 8.0f;
struct PaCtl {
  unsigned long long qfull, qempty, kfull[kPaKSlots], kempty[kPaKSlots], vfull[kPaVSlots], vempty[kPaVSlots], sfull[2],
      sfree[2], oready[2], pfull[4], pfree[4], pvdone[2], done;
  unsigned tmem;
  int dead;
  long long red[kPaThreads / 32 + 4];
  RowTab rows[4];        // entries of a unit: the scores' (two, in turn) and the sums' (two)
  float top[2][4][64];   // [unit parity][64 positions of 256][row]: maxima (at the end: sums) of a row's four threads
};
constexpr int kPaQ = 0, kPaP = kPaQ + kBlocks * kPaQBlock, kPaK = kPaP + 4 * kPaQBlock,
              kPaV = kPaK + kPaKSlots * kPaBlock, kPaCtl = kPaV + kPaVSlots * kPaBlock;
constexpr int kPaSmem = kPaCtl + (int)sizeof(PaCtl);
static_assert(kPaSmem <= 232448, "shared memory of a CTA");

// MN-major operand with the 128-byte swizzle: 64-element blocks `lbo` bytes apart, 8 K-rows in 1024 bytes
KK3_DEV unsigned long long sdesc_mn(unsigned addr, unsigned lbo) {
  return (unsigned long long)((addr & 0x3ffffu) >> 4) | ((unsigned long long)(lbo >> 4) << 16) |
         ((unsigned long long)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
KK3_DEV void tmem_st32(unsigned taddr, const float (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]),
        "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]),
        "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]),
        "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
      : "memory");
}
KK3_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPaThreads, 1)
    kk3_cache_attend_pair_kernel(const AttendArgs a, const PairRows pr, const __grid_constant__ PairMaps maps) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  PaCtl& ctl = *reinterpret_cast<PaCtl*>(smem_raw + kPaCtl);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, worker = blockIdx.x >> 1;
  const unsigned rank = cluster_rank(), base = smem_u32(smem_raw);
  const unsigned qfull = smem_u32(&ctl.qfull), qempty = smem_u32(&ctl.qempty), kfull = smem_u32(ctl.kfull),
                 kempty = smem_u32(ctl.kempty), vfull = smem_u32(ctl.vfull), vempty = smem_u32(ctl.vempty),
                 sfull = smem_u32(ctl.sfull), sfree = smem_u32(ctl.sfree), oready = smem_u32(ctl.oready),
                 pfull = smem_u32(ctl.pfull), pfree = smem_u32(ctl.pfree), pvdone = smem_u32(ctl.pvdone),
                 done = smem_u32(&ctl.done);
  volatile int* dead = &ctl.dead;
  fetch_maps(maps);
  if (tid == 0) {
    mbar_init(qfull, 1);
    mbar_init(qempty, 1);
    for (int i = 0; i < kPaKSlots; ++i) {
      mbar_init(kfull + 8 * i, 1);
      mbar_init(kempty + 8 * i, 1);
    }
    for (int i = 0; i < kPaVSlots; ++i) {
      mbar_init(vfull + 8 * i, 1);
      mbar_init(vempty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sfull + 8 * i, 1);
      mbar_init(sfree + 8 * i, 16);   // the softmax warps of both CTAs
    }
    mbar_init(oready, 16);   // units in turn: one CTA's warps may be a unit ahead of the other's, never two
    mbar_init(oready + 8, 16);
    for (int i = 0; i < 4; ++i) {
      mbar_init(pfull + 8 * i, 4);   // the warps of these 64 positions, of both CTAs
      mbar_init(pfree + 8 * i, 1);
    }
    mbar_init(pvdone, 1);   // units in turn
    mbar_init(pvdone + 8, 1);
    mbar_init(done, 2);
    ctl.dead = 0;
    fence_mbar_init();
  }
  if (warp == 9) pair_alloc(smem_u32(&ctl.tmem), 512);
  __syncwarp();
  cluster_arrive();   // the peer's barriers are needed after the plan
  const AttendSplit split{kPairRows, a.heads, kPaUnit, kPaTileCost};
  const Share sh = plan_share<kPaThreads>(a, split, worker, kPaMinUnits, smem_raw, ctl.red);
  fence_async_smem();   // the plan of a large call lay where the copies come
  cache_go_on();
  if (tid == 0 && rank == 0) a.meta[worker * 4 + 2] = 0;
  tc_fence_before();
  __syncthreads();
  cluster_wait();
  tc_fence_after();
  const unsigned tmem = *reinterpret_cast<volatile unsigned*>(&ctl.tmem);
  const unsigned tmem_s = tmem + 256;   // two score buffers of 128 columns; the sums have 256 before them
  if ((base & 1023u) && tid == 0) cache_error(a.c);   // dynamic shared memory begins on the swizzled blocks' boundary
  const bool takes_part = worker < sh.workers && (base & 1023u) == 0;   // alike in both CTAs of the pair

  int b = sh.b, t = sh.t;
  long long at = sh.at;
  int n = 0, tile = 0;   // units and tiles so far
  bool ok = true;
  if (!takes_part) {
  } else if (warp == 8) {
    // ---- queries, and the entries' blocks for the scores
    const unsigned lead_q = in_cta(qfull, 0), lead_k = in_cta(kfull, 0);
    const bool me = elect_one();
    with_box(pr.box, [&](auto box) {
      int slot = 0, phase = 0;
      Seq s = sh.seq;
      for (; ok && at < sh.end; ++t, ++tile) {
        for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
        const int units = split.units(s, t), end = split.sees(s, t);
        const int u0 = split.from(sh, at, units), u1 = split.to(sh, at, units);
        if (u0 == u1) break;   // only a tile's cost is left: the next worker's
        PageIds ids;
        ids.fetch(a.c, pr, b, u0 * kPaUnit, end);
        ok = __all_sync(0xffffffffu, pair_wait(a.c, qempty, (tile & 1) ^ 1, dead));
        if (!ok) break;
        if (rank == 0 && me) mbar_arrive_tx(qfull, 2 * kBlocks * kPaQBlock);
        __syncwarp();
        const int q = s.q0 * a.heads + t * kPairRows + (int)rank * 64;   // rows behind the sequence's are not written
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
          load_box(me, base + kPaQ + d * kPaQBlock, d < kBlocks - 1 ? &maps.ql : &maps.qp, d < kBlocks - 1 ? d * 64 : 0, q, lead_q);
        ids.write<decltype(box)::value != 0>(a.c, pr, u0 * kPaUnit, end, ctl.rows[0]);
        __syncwarp();
        ids.fetch(a.c, pr, b, (u0 + 1) * kPaUnit, end);
        Boxes<128, decltype(box)::value> boxes, next;
        next.take(ctl.rows[0], (int)rank * 128);
        for (int u = u0; ok && u < u1; ++u) {
          boxes = next;
#pragma unroll 1
          for (int d = 0; d < kBlocks; ++d) {
            ok = __all_sync(0xffffffffu, pair_wait(a.c, kempty + 8 * slot, phase ^ 1, dead));
            if (!ok) break;
            if (rank == 0 && me) mbar_arrive_tx(kfull + 8 * slot, 2 * kPaBlock);
            __syncwarp();
            boxes.load(me, maps, d, base + kPaK + slot * kPaBlock, lead_k + 8 * slot);
            if (++slot == kPaKSlots) {
              slot = 0;
              phase ^= 1;
            }
            if (d == 3 && u + 1 < u1) {   // the next unit's rows, while copies are on their way
              RowTab& tab = ctl.rows[(u + 1 - u0) & 1];
              ids.write<decltype(box)::value != 0>(a.c, pr, (u + 1) * kPaUnit, end, tab);
              __syncwarp();
              ids.fetch(a.c, pr, b, (u + 2) * kPaUnit, end);
              next.take(tab, (int)rank * 128);
            }
          }
        }
        __syncwarp();   // the tables are read
        at += units + kPaTileCost;
      }
    });
    if (rank == 0 && lane == 0 && !ok) {   // after a failed wait: a bounded time for the copies in flight
      mbar_wait_for(qfull, (tile & 1) ^ 1, kWaitNs);
      for (int i = 0; i < 2 * kPaKSlots; ++i) mbar_wait_for(kfull + 8 * (i / 2), i & 1, kWaitNs / 8);
    }
    __syncwarp();
  } else if (warp == 10) {
    // ---- the entries' pieces for the sums: piece (g, h) is dims 256 h + 128 rank .. + 127 of positions 64 g .. + 63 of
    // the unit. Positions behind the sequence's end must be zeros, whatever the page holds there: a group that the end cuts
    // comes row by row (3.4 us; the entries of tokens that come after the tile's have values and weights of zero).
    const unsigned lead_v = in_cta(vfull, 0);
    const bool me = elect_one();
    with_box(pr.box, [&](auto box) {
      int slot = 0, phase = 0;
      Seq s = sh.seq;
      for (; ok && at < sh.end; ++t) {
        for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
        const int units = split.units(s, t), end = min(s.len, (split.sees(s, t) + 63) & ~63);
        const int u0 = split.from(sh, at, units), u1 = split.to(sh, at, units);
        if (u0 == u1) break;
        PageIds ids;
        ids.fetch(a.c, pr, b, u0 * kPaUnit, end);
        ids.write<decltype(box)::value != 0>(a.c, pr, u0 * kPaUnit, end, ctl.rows[2]);
        __syncwarp();
        ids.fetch(a.c, pr, b, (u0 + 1) * kPaUnit, end);
        for (int u = u0; ok && u < u1; ++u) {
          const RowTab& tab = ctl.rows[2 + ((u - u0) & 1)];
#pragma unroll 1
          for (int g = 0; g < 4; ++g) {
            const int left = end - (u * kPaUnit + g * 64);
            const auto pieces = [&](auto boxes) {
              boxes.take(tab, g * 64);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const unsigned dst = base + kPaV + slot * kPaBlock, bar = lead_v + 8 * slot;
                ok = ok && __all_sync(0xffffffffu, pair_wait(a.c, vempty + 8 * slot, phase ^ 1, dead));
                if (!ok) return;
                if (rank == 0 && me) mbar_arrive_tx(vfull + 8 * slot, 2 * kPaBlock);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 2; ++j) boxes.load(me, maps, 4 * h + 2 * (int)rank + j, dst + j * (kPaBlock / 2), bar);
                if (++slot == kPaVSlots) {
                  slot = 0;
                  phase ^= 1;
                }
              }
            };
            if (left > 0 && left < 64) pieces(Boxes<64, 0>());
            else pieces(Boxes<64, decltype(box)::value>());
            if (!ok) break;
            if (g == 1 && u + 1 < u1) {   // the next unit's rows, while copies are on their way
              ids.write<decltype(box)::value != 0>(a.c, pr, (u + 1) * kPaUnit, end, ctl.rows[2 + ((u + 1 - u0) & 1)]);
              __syncwarp();
              ids.fetch(a.c, pr, b, (u + 2) * kPaUnit, end);
            }
          }
        }
        __syncwarp();   // the tables are read
        at += units + kPaTileCost;
      }
    });
    if (rank == 0 && lane == 0 && !ok)
      for (int i = 0; i < 2 * kPaVSlots; ++i) mbar_wait_for(vfull + 8 * (i / 2), i & 1, kWaitNs / 8);
    __syncwarp();
  } else if (warp == 9 || warp == 11) {
    // ---- matrix instructions: two threads of the pair. Issuing costs as much as the instructions take, so the loops are
    // unrolled over the slots and the descriptors are sums of 16-byte offsets.
    if (lane == 0 && rank == 0) {
      constexpr unsigned id_s = pair_idesc(128, 256), id_o = id_s | (1u << 16);   // values are MN-major
      Seq s = sh.seq;
      for (; ok && at < sh.end; ++t, ++tile) {
        for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
        const int units = split.units(s, t), sees = split.sees(s, t);
        const int u0 = split.from(sh, at, units), u1 = split.to(sh, at, units);
        if (u0 == u1) break;
        if (warp == 9) {
          const unsigned long long qd = sdesc_sw128(base + kPaQ), kd = sdesc_sw128(base + kPaK);
          ok = pair_wait(a.c, qfull, tile & 1, dead);
          for (int u = u0; ok && u < u1; ++u, ++n) {
            const int buf = n & 1;
            const unsigned d = tmem_s + buf * 128;
            ok = pair_wait(a.c, sfree + 8 * buf, ((n >> 1) & 1) ^ 1, dead);
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
              const int use = n * kBlocks + i, slot = use % kPaKSlots;
              if (ok) ok = pair_wait(a.c, kfull + 8 * slot, (use / kPaKSlots) & 1, dead);
              if (!ok) break;
              tc_fence_after();
              const unsigned long long ka = kd + slot * (kPaBlock >> 4);
#pragma unroll
              for (int k = 0; k < 4; ++k) pair_mma(d, qd + i * (kPaQBlock >> 4) + k * 2, ka + k * 2, id_s, (unsigned)(i | k));
              pair_commit(kempty + 8 * slot);
            }
            if (ok) pair_commit(sfull + 8 * buf);
          }
          if (ok) pair_commit(qempty);
        } else {
          const unsigned long long pd = sdesc_sw128(base + kPaP), vd = sdesc_mn(base + kPaV, kPaBlock / 2);
          for (int u = u0; ok && u < u1; ++u, ++n) {
            ok = pair_wait(a.c, oready + 8 * (n & 1), (n >> 1) & 1, dead);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int use = n * 8 + i, slot = use % kPaVSlots;
              if (ok && !(i & 1)) ok = pair_wait(a.c, pfull + 4 * i, n & 1, dead);
              if (ok) ok = pair_wait(a.c, vfull + 8 * slot, (use / kPaVSlots) & 1, dead);
              if (!ok) break;
              tc_fence_after();
              const unsigned long long va = vd + slot * (kPaBlock >> 4);
              if (i < 2 || u * kPaUnit + (i >> 1) * 64 < sees) {   // a unit's first group always: it sets the sums
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  pair_mma(tmem + (i & 1) * 128, pd + (i >> 1) * (kPaQBlock >> 4) + k * 2, va + k * 128, id_o, (unsigned)(u > u0 || i > 1 || k));
              }
              pair_commit(vempty + 8 * slot);
              if (i & 1) pair_commit(pfree + 4 * (i - 1));
            }
            if (ok) pair_commit(pvdone + 8 * (n & 1));
          }
        }
        at += units + kPaTileCost;
      }
      pair_commit(done);   // all matrix instructions end before TMEM is given back
      mbar_wait_for(done, 0, kWaitNs);
    }
    __syncwarp();
  } else {
    // ---- softmax: a row's four threads are in the warps of equal parity, 64 positions of a unit each; after a failed
    // wait the rounds go on without work, since they meet at barriers
    const int wg = warp >> 2, quarter = warp & 3, row = (quarter & 1) * 32 + lane;
    const int part64 = (quarter >> 1) * 2 + wg;   // which 64 positions of the unit
    const unsigned tlane = (unsigned)(quarter * 32) << 16, meet = 1 + (quarter & 1);
    const unsigned lead_sfree = in_cta(sfree, 0), lead_oready = in_cta(oready, 0),
                   lead_pfull = in_cta(pfull + 8 * part64, 0);
    const unsigned p_row = base + kPaP + part64 * kPaQBlock + row * 128;
    // Units before number m have been added to O. A barrier's parity only tells a phase from its neighbours: each of the
    // two has every other unit, and where this is asked, the unit three before is known to be added (this thread's part
    // of P was free again from the one two before) and the next one waits for this thread.
    const auto all_added = [&](int m) {
      __all_sync(0xffffffffu, m == 0 || pair_wait(a.c, pvdone + 8 * ((m - 1) & 1), ((m - 1) >> 1) & 1, dead));
    };
    const float sign = a.scale_log2 < 0.0f ? -1.0f : 1.0f, size = fabsf(a.scale_log2);
    Seq s = sh.seq;
    for (; at < sh.end; ++t) {
      for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
      const int units = split.units(s, t);
      const int u0 = split.from(sh, at, units), u1 = split.to(sh, at, units);
      if (u0 == u1) break;
      const int g = t * kPairRows + (int)rank * 64 + row;
      const bool live = g < s.n * a.heads;
      // rows behind the last are computed without a mask (it would cost every unit) and not written
      const int sees = live ? s.len - s.n + g / a.heads + 1 : INT_MAX;
      float m = -INFINITY, l = 0.0f;
      for (int u = u0; u < u1; ++u, ++n) {
        const int buf = n & 1;
        __all_sync(0xffffffffu, pair_wait(a.c, sfull + 8 * buf, (n >> 1) & 1, dead));
        tc_fence_after();
        float v[2][32];
        tmem_ld32(tmem_s + buf * 128 + wg * 64 + tlane, v[0]);
        tmem_ld32(tmem_s + buf * 128 + wg * 64 + 32 + tlane, v[1]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(lead_sfree + 8 * buf);
        const int left = sees - u * kPaUnit - part64 * 64;   // positions of this thread's 64 that the row sees
        const bool cut = !__all_sync(0xffffffffu, left >= 64);
        if (a.scale_log2 < 0.0f) {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i >> 5][i & 31] *= sign;
        }
        if (cut) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= left) v[i >> 5][i & 31] = -INFINITY;
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; ++i) tops[i & 3] = fmaxf(tops[i & 3], v[i >> 5][i & 31]);
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        ctl.top[buf][part64][row] = top;
        asm volatile("bar.sync %0, 128;" ::"r"(meet) : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, ctl.top[buf][i][row]);
        if (top != -INFINITY) top *= size;
        float alpha = 1.0f;
        if (top > m + kPaSlack || m == -INFINITY) {
          if (m != -INFINITY) alpha = ex2(m - top);
          m = top;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        if (u > u0 && __any_sync(0xffffffffu, alpha != 1.0f)) {   // rescale, once the unit before has been added
          all_added(n);
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 128; c += 32) {
            float o[32];
            tmem_ld32(tmem + wg * 128 + tlane + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= alpha;
            tmem_st32(tmem + wg * 128 + tlane + c, o);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(lead_oready + 8 * buf);
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          float& x = v[i >> 5][i & 31];
          x = ex2(fmaf(x, size, -ref));
        }
        if (cut && size == 0.0f) {   // -infinity times a scale of zero is no -infinity
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= left) v[i >> 5][i & 31] = 0.0f;
        }
        float sum[4] = {};
#pragma unroll
        for (int i = 0; i < 64; ++i) sum[i & 3] += v[i >> 5][i & 31];
        l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        unsigned w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const __nv_bfloat162 h2 = __floats2bfloat162_rn(v[i >> 4][(i & 15) * 2], v[i >> 4][(i & 15) * 2 + 1]);
          w[i] = *reinterpret_cast<const unsigned*>(&h2);
        }
        // the sums of the unit before have read this part of P
        if (n > 0) __all_sync(0xffffffffu, pair_wait(a.c, pfree + 8 * part64, (n - 1) & 1, dead));
#pragma unroll
        for (int c = 0; c < 8; ++c)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                       ::"r"(p_row + ((c ^ (row & 7)) << 4)), "r"(w[c * 4]), "r"(w[c * 4 + 1]), "r"(w[c * 4 + 2]), "r"(w[c * 4 + 3])
                       : "memory");
        fence_async_smem();
        __syncwarp();
        if (lane == 0) arrive_cluster(lead_pfull);
      }
      all_added(n);
      tc_fence_after();
      asm volatile("bar.sync %0, 128;" ::"r"(meet) : "memory");   // the last maxima are read
      ctl.top[0][part64][row] = l;
      asm volatile("bar.sync %0, 128;" ::"r"(meet) : "memory");
      l = or_lost((ctl.top[0][0][row] + ctl.top[0][1][row]) + (ctl.top[0][2][row] + ctl.top[0][3][row]), dead);
      const bool whole = u0 == 0 && u1 == units;
      const long long out_row = (long long)s.q0 * a.heads + g;
      float* part = a.part + (((long long)worker * 2 + (u0 == 0 ? 1 : 0)) * kPairRows + rank * 64 + row) * kPartRow;
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      // through 2 KB of the part of P that this warp fills (the instructions have read it, and no other warp's next
      // probabilities come there), so that a row's dims leave in pieces of 64 bytes: 32 rows x 32 dims of results, 16
      // dims of running sums
      unsigned char* stage = smem_raw + kPaP + part64 * kPaQBlock + (quarter & 1) * 4096;
      const int dim0 = wg * 256 + (quarter >> 1) * 128, rows_here = s.n * a.heads - (g - lane);
      const int put = lane * 64, turn = (lane >> 1) & 3;
#pragma unroll 1
      for (int c = 0; c < 128; c += 32) {
        float o[32];
        tmem_ld32(tmem + wg * 128 + tlane + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (whole) {
            if (h) break;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              __nv_bfloat162 w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = __floats2bfloat162_rn(o[i * 8 + k * 2] * inv, o[i * 8 + k * 2 + 1] * inv);
              *reinterpret_cast<uint4*>(stage + put + (i ^ turn) * 16) = *reinterpret_cast<const uint4*>(w);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<float4*>(stage + put + (i ^ turn) * 16) =
                  make_float4(o[h * 16 + i * 4], o[h * 16 + i * 4 + 1], o[h * 16 + i * 4 + 2], o[h * 16 + i * 4 + 3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 2), ch = lane & 3;   // row of this warp's 32, and 16 bytes of it
            const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 64 + (ch ^ ((r >> 1) & 3)) * 16);
            if (r < rows_here) {
              if (whole) *reinterpret_cast<uint4*>(a.out + (out_row - lane + r) * kLat + dim0 + c + ch * 8) = v;
              else *reinterpret_cast<uint4*>(part + (long long)(r - lane) * kPartRow + dim0 + c + h * 16 + ch * 4) = v;
            }
          }
          __syncwarp();
        }
      }
      if (live && part64 == 0) {
        if (whole) {
          a.lse[out_row] = (m + log2f(l)) * 0.69314718055994531f;
        } else {
          part[kLat] = m;
          part[kLat + 1] = l;
        }
      }
      if (u0 == 0 && u1 < units && tid == 0 && rank == 0) {
        a.meta[worker * 4] = s.q0 * a.heads + t * kPairRows;
        a.meta[worker * 4 + 1] = min(kPairRows, s.n * a.heads - t * kPairRows);
        a.meta[worker * 4 + 2] = sh.holder(at + kPaTileCost + units) - worker + 1;
      }
      at += units + kPaTileCost;
      tc_fence_before();   // TMEM is read before the next tile's first sums, which wait for its probabilities
      asm volatile("bar.sync %0, 128;" ::"r"(meet) : "memory");   // the sums are read before the next maxima
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // neither CTA gives up its memory while the other's instructions may use it
  if (warp == 9) pair_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------------------------
// Attention of few rows (single tokens on one rank): a tile is 16 (token, head) rows, a unit 32 cached positions.
//
// The call is bound by the cache's bytes, so each entry comes into shared memory once, by TMA, and serves both products
// from there at warp level (m16n8k16): 32 positions are 36.9 KB, 1600 clocks at one SM's share of HBM. What the work on a
// unit takes is latency, so 16 warps, four to a scheduler, run three units at a time: between two barriers they add the
// values of one unit, take the softmax of the next and the scores of the one after it. In the first product a warp holds
// the query's fragments of a quarter of the 576 dims in registers and takes 8 positions, in the second it owns 32 of the
// output dims, in the softmax a row; half of the warps begin with the scores, so that not all want the same at once. Four
// more warps copy, one unit to a stage of five, and run ahead over the tiles.
// Measured: 64 single tokens x 12 heads over 8192 positions 123 us, 4.9 TB/s, and 119 us where the cache stays in L2: the
// 1800 clocks of a unit's instructions and shared-memory traffic, the start, the workers' uneven ends and the join (25 us
// for the last three); one token over 517 positions 15 us. Before the last two steps: with copies by the 16 warps themselves,
// between the products, the 64 took 142 us; with six stages, scores of one unit in shared memory and two barriers a unit 134.
// Probabilities are rounded to BF16 for the second product, the type that the instruction takes with BF16 latents; the
// running sum adds them unrounded, since lse is an FP32 result.

constexpr int kFewUnit = 32, kFewStages = 5;
constexpr int kFewWork = 512, kFewCopies = 4, kFewThreads = kFewWork + 32 * kFewCopies;
constexpr int kFewBlock = kFewUnit * 128;               // 32 positions x 64 dims
constexpr int kFewStageBytes = kBlocks * kFewBlock;
constexpr int kFewMinUnits = 4;
constexpr int kFewQuarter = 5;   // pairs of k-steps of a quarter of the 18: 5, 5, 4, 4
struct FewCtl {
  // scores of two units, a part from each quarter of the dims; column c of row r at c ^ 8 (r % 4)
  float s[2][4][kFewRows][kFewUnit];
  alignas(16) bf16 p[2][kFewRows][kFewUnit + 8];
  float alpha[2][kFewRows], m[kFewRows], l[kFewRows];
  unsigned long long full[kFewStages], empty[kFewStages];
  int dead;
};
constexpr int kFewSmem = kFewStages * kFewStageBytes + (int)sizeof(FewCtl);
static_assert(kFewSmem <= 232448, "shared memory of a CTA");
static_assert(kFewStages * kFewStageBytes >= kPlanBytes + 16 + (kFewThreads / 32 + 4) * 8, "the plan lies in the ring");

KK3_DEV void ldsm4(unsigned (&r)[4], unsigned a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
KK3_DEV void ldsm4t(unsigned (&r)[4], unsigned a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// m16n8k16 without the order that a volatile one keeps: loads of operands may go ahead of it
KK3_DEV void mma_free(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
KK3_DEV float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
KK3_DEV void few_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kFewWork) : "memory"); }
// single-CTA copies
KK3_DEV void load_box1(bool me, unsigned dst, const CUtensorMap* map, int x, int row, unsigned bar) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n"
      " @p cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}"
      ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(bar), "r"((unsigned)me) : "memory");
}
KK3_DEV void gather4_1(bool me, unsigned dst, const CUtensorMap* map, int x, int r0, int r1, int r2, int r3, unsigned bar) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %8, 0;\n"
      " @p cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7];\n}"
      ::"r"(dst), "l"(map), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar), "r"((unsigned)me) : "memory");
}

// Pages of 256 positions from `first` on, looked up ahead: position first + 8 lane and its slot in its page (boxes
// begin at multiples of 8).
struct FewPages {
  int id, slot;
  KK3_DEV void fetch(const CachePages& c, int b, int first, int end) {
    const int pos = first + 8 * (threadIdx.x & 31), col = page_of(c, pos);
    slot = pos - col * c.page_size;
    id = -1;
    if (pos < end) id = c.table[(long long)b * c.table_stride + col];
  }
};

// A copy warp's part of a unit: every kFewCopies-th 64-dim block. Box by box where the unit lies within the tile's
// positions, else row by row, with zeros for what lies behind (so that nothing there can reach the products).
KK3_DEV void few_load(const AttendArgs& a, const PairRows& pr, const PairMaps& maps, int b, const FewPages& pages, int unit, int end,
                      int part, unsigned stage, unsigned bar) {
  const int lane = threadIdx.x & 31, pos0 = unit * kFewUnit, lane0 = (unit & 7) * 4;
  const bool me = elect_one();
  if (me) mbar_arrive_tx(bar, ((kBlocks - 1 - part) / kFewCopies + 1) * kFewBlock);
  if (pr.box && pos0 + kFewUnit <= end) {
    const bool fine = (unsigned)pages.id < (unsigned)a.c.num_pages;
    if (!fine && lane >= lane0 && lane < lane0 + 4) cache_error(a.c);
    const int kv = fine ? pages.id * pr.kv_ratio + pages.slot : pr.kv_end, pe = fine ? pages.id * pr.pe_ratio + pages.slot : pr.pe_end;
#pragma unroll 1
    for (int k = 0; k < kFewUnit; k += pr.box) {
      const int row = __shfl_sync(0xffffffffu, kv, lane0 + (k >> 3)), rope = __shfl_sync(0xffffffffu, pe, lane0 + (k >> 3));
#pragma unroll 1
      for (int d = part; d < kBlocks - 1; d += kFewCopies) load_box1(me, stage + d * kFewBlock + k * 128, &maps.kv_box, d * 64, row, bar);
      if (part == 0) load_box1(me, stage + (kBlocks - 1) * kFewBlock + k * 128, &maps.pe_box, 0, rope, bar);
    }
  } else {
    const int pos = pos0 + lane;
    int kv = pr.kv_end, pe = pr.pe_end;
    if (pos < end) {
      int slot;
      const int page = page_at(a.c, b, pos, &slot);
      if (page >= 0) {
        kv = page * pr.kv_ratio + slot;
        pe = page * pr.pe_ratio + slot;
      }
    }
#pragma unroll 1
    for (int d = part; d < kBlocks; d += kFewCopies) {
      const bool rope = d == kBlocks - 1;
      const int row = rope ? pe : kv;
#pragma unroll 1
      for (int k = 0; k < kFewUnit; k += 4)
        gather4_1(me, stage + d * kFewBlock + k * 128, rope ? &maps.pe_row : &maps.kv_row, rope ? 0 : d * 64,
                  __shfl_sync(0xffffffffu, row, k), __shfl_sync(0xffffffffu, row, k + 1), __shfl_sync(0xffffffffu, row, k + 2),
                  __shfl_sync(0xffffffffu, row, k + 3), bar);
    }
  }
}

__global__ void __launch_bounds__(kFewThreads, 1)
    kk3_cache_attend_few_kernel(const AttendArgs a, const PairRows pr, const __grid_constant__ PairMaps maps) {
  static_assert(kBlocks % kFewCopies == 1, "the rope block falls to the first copy warp");
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  FewCtl& ctl = *reinterpret_cast<FewCtl*>(smem_raw + kFewStages * kFewStageBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, worker = blockIdx.x;
  const unsigned base = smem_u32(smem_raw), full = smem_u32(ctl.full), empty = smem_u32(ctl.empty);
  volatile int* dead = &ctl.dead;
  fetch_maps(maps);
  const AttendSplit split{kFewRows, a.heads, kFewUnit, 0};
  if (tid == 0) {
    for (int i = 0; i < kFewStages; ++i) {
      mbar_init(full + 8 * i, kFewCopies);
      mbar_init(empty + 8 * i, kFewWork / 32);
    }
    ctl.dead = 0;
    fence_mbar_init();
  }
  const Share sh = plan_share<kFewThreads>(a, split, worker, kFewMinUnits, smem_raw,
                                           reinterpret_cast<long long*>(smem_raw + (kPlanBytes + 15) / 16 * 16));
  cache_go_on();
  if (tid == 0) a.meta[worker * 4 + 2] = 0;
  if (base & 1023u) {   // dynamic shared memory begins on the swizzled blocks' boundary
    if (tid == 0) cache_error(a.c);
    return;
  }
  if (worker >= sh.workers) return;
  int b = sh.b, t = sh.t;
  long long at = sh.at;
  int slot = 0;   // the ring's stage, in turn `phase`
  unsigned phase = 0;
  bool ok = true;
  fence_async_smem();   // the plan of a large call lay where the copies come
  __syncthreads();      // its readers are done with the ring

  if (warp >= kFewWork / 32) {
    const int part = warp - kFewWork / 32;
    Seq s = sh.seq;
    for (; at < sh.end && ok; ++t) {
      for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
      const int units = split.units(s, t), end = split.sees(s, t);
      const int u0 = split.from(sh, at, units), u1 = split.to(sh, at, units);
      FewPages pages, next;
      next.fetch(a.c, b, (u0 & ~7) * kFewUnit, end);
      for (int u = u0; u < u1 && ok; ++u) {
        if (u == u0 || (u & 7) == 0) {
          pages = next;
          next.fetch(a.c, b, ((u & ~7) + 8) * kFewUnit, end);
        }
        ok = pair_wait(a.c, empty + 8 * slot, phase ^ 1, dead);
        __syncwarp();
        if (ok) few_load(a, pr, maps, b, pages, u, end, part, base + slot * kFewStageBytes, full + 8 * slot);
        if (++slot == kFewStages) {
          slot = 0;
          phase ^= 1;
        }
      }
      at += units;
    }
    // after a failed wait: a bounded time for the copies in flight
    if (*dead)
      for (int i = 0; i < 2 * kFewStages; ++i) mbar_wait_for(full + 8 * (i / 2), i & 1, kWaitNs / 16);
  } else {
    const int ntile = warp & 3, quarter = warp >> 2;   // 8 positions of the unit; pairs quarter, quarter + 4 .. of the 18 pairs of k-steps
    const bool fifth = quarter < 2, scores_first = quarter >= 2;
    // this lane's addresses in a stage: score operands (block quarter / 2 + 2 i for pair quarter + 4 i), values
    const unsigned kat = (quarter >> 1) * kFewBlock + (ntile * 8 + (lane & 7)) * 128 + ((((quarter & 1) * 4 + (lane >> 3)) ^ (lane & 7)) << 4);
    const unsigned vat = (warp >> 1) * kFewBlock + (lane & 15) * 128 + ((((warp & 1) * 4 + (lane >> 4)) ^ (lane & 7)) << 4);
    const unsigned pat = smem_u32(&ctl.p[0][lane & 15][(lane >> 4) * 8]);
    Seq s = sh.seq;
    for (; at < sh.end; ++t) {
      for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
      const int units = split.units(s, t);
      const int u0 = split.from(sh, at, units), u1 = split.to(sh, at, units);
      const bool whole = u0 == 0 && u1 == units;
      const int row0 = t * kFewRows, rows = min(kFewRows, s.n * a.heads - row0);
      // Query fragments through the memory of the scores and probabilities, half of the dims at a time, zeros below the
      // last row. (From memory straight into fragments, four bytes a load, took 4400 clocks instead of 1600.)
      static_assert(kFewRows * (kEntry / 8) <= 3 * kFewWork && kFewRows * 5 * 128 <= sizeof(ctl.s) + sizeof(ctl.p), "queries on their way");
      unsigned char* const q_smem = reinterpret_cast<unsigned char*>(ctl.s);
      uint4 qv[3];
#pragma unroll
      for (int j = 0; j < 3; ++j) {   // 16 bytes each: the pieces of blocks 0 .. 3, then those of the others
        const int i = tid + j * kFewWork, r = i >= 512 ? (i - 512) / 40 : i / 32, ch = i >= 512 ? 32 + (i - 512) % 40 : i % 32;
        qv[j] = uint4{};
        if (i < kFewRows * (kEntry / 8) && r < rows) {
          const int g = row0 + r, tok = s.q0 + g / a.heads, head = g % a.heads;
          qv[j] = *reinterpret_cast<const uint4*>(ch < kLat / 8 ? a.q_lat + tok * a.ql_tok + head * a.ql_head + ch * 8
                                                                : a.q_pe + tok * a.qp_tok + head * a.qp_head + (ch - kLat / 8) * 8);
        }
      }
      unsigned qf[2 * kFewQuarter][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        few_sync();   // the scores of the tile before, or the other half, are read
#pragma unroll
        for (int j = h; j < 1 + 2 * h; ++j) {
          const int i = tid + j * kFewWork, r = h ? (i - 512) / 40 : i / 32, ch = h ? (i - 512) % 40 : i % 32;
          if (r < kFewRows) *reinterpret_cast<uint4*>(q_smem + (ch >> 3) * (kFewRows * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = qv[j];
        }
        few_sync();
#pragma unroll
        for (int k = h * 4; k < (h ? 2 * kFewQuarter : 4); ++k) {   // step k % 2 of pair quarter + 4 (k / 2)
          const int pair = quarter + 4 * (k >> 1), block = (pair >> 1) - 4 * h, r = lane & 15, ch = (pair & 1) * 4 + (k & 1) * 2 + (lane >> 4);
          if (k < 8 || fifth) ldsm4(qf[k], smem_u32(q_smem) + block * (kFewRows * 128) + r * 128 + ((ch ^ (r & 7)) << 4));
        }
      }
      few_sync();   // the fragments are taken
      float acc[4][4] = {};
      float m = -INFINITY, l = 0.0f;   // softmax: row `warp`, a position a lane
      const int sees = warp < rows ? s.len - s.n + (row0 + warp) / a.heads + 1 : 0;
      // unit u0 + i: scores, softmax, values; `in` is the stage of the unit whose scores come next, `out` of the one whose values do
      int in = slot, out = slot;
      const auto scores = [&](int i) {
        float c[2][4];
        pair_wait(a.c, full + 8 * in, phase, dead);
        const unsigned kb = base + in * kFewStageBytes + kat;
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j >> 2][j & 3] = 0.0f;   // two chains: a product waits for the one before it on its sums
#pragma unroll
        for (int k = 0; k < kFewQuarter; ++k) {
          if (k < 4 || fifth) {
            unsigned bf[4];
            ldsm4(bf, kb + k * 2 * kFewBlock);
            mma_free(c[0], qf[2 * k], bf[0], bf[1]);
            mma_free(c[1], qf[2 * k + 1], bf[2], bf[3]);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) c[0][j] += c[1][j];
        float* to = &ctl.s[i & 1][quarter][lane >> 2][(ntile * 8 + (lane & 3) * 2) ^ ((lane >> 2 & 3) << 3)];
        *reinterpret_cast<float2*>(to) = make_float2(c[0][0], c[0][1]);
        *reinterpret_cast<float2*>(to + 8 * kFewUnit) = make_float2(c[0][2], c[0][3]);
        if (++in == kFewStages) {
          in = 0;
          phase ^= 1;
        }
      };
      const auto softmax = [&](int i) {
        const float* from = &ctl.s[i & 1][0][warp][lane ^ ((warp & 3) << 3)];
        constexpr int kPart = kFewRows * kFewUnit;
        float v = ((from[0] + from[kPart]) + (from[2 * kPart] + from[3 * kPart])) * a.scale_log2;
        if ((u0 + i) * kFewUnit + lane >= sees) v = -INFINITY;
        const float top = fmaxf(m, redux_max(v)), ref = top == -INFINITY ? 0.0f : top;
        const float al = ex2(m - ref), p = ex2(v - ref);
        l = l * al + p;
        m = top;
        ctl.p[i & 1][warp][lane] = f2bf(p);
        if (lane == 0) ctl.alpha[i & 1][warp] = al;
      };
      const auto values = [&](int i) {
        const float a0 = ctl.alpha[i & 1][lane >> 2], a1 = ctl.alpha[i & 1][(lane >> 2) + 8];
        const unsigned vb = base + out * kFewStageBytes + vat, pb = pat + (i & 1) * (kFewRows * (kFewUnit + 8) * 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[j][0] *= a0;
          acc[j][1] *= a0;
          acc[j][2] *= a1;
          acc[j][3] *= a1;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          unsigned pf[4], b0[4], b1[4];
          ldsm4(pf, pb + k * 32);
          ldsm4t(b0, vb + k * 16 * 128);
          ldsm4t(b1, (vb ^ 32u) + k * 16 * 128);
          mma_free(acc[0], pf, b0[0], b0[1]);
          mma_free(acc[1], pf, b0[2], b0[3]);
          mma_free(acc[2], pf, b1[0], b1[1]);
          mma_free(acc[3], pf, b1[2], b1[3]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * out);
        if (++out == kFewStages) out = 0;
      };
      const int n = u1 - u0;
      scores(0);
      few_sync();
      for (int i = 0; i < n; ++i) {
        if (scores_first && i + 1 < n) scores(i + 1);
        softmax(i);
        if (i > 0) values(i - 1);
        if (!scores_first && i + 1 < n) scores(i + 1);
        few_sync();   // the unit's probabilities and the next one's scores are written, what they replace is read
      }
      values(n - 1);
      slot = in;
      l = warp_sum(l);
      if (lane == 0) {
        ctl.m[warp] = m;
        ctl.l[warp] = or_lost(l, dead);
      }
      few_sync();
      const long long g = (long long)s.q0 * a.heads + row0;
      // running sums for the join: slot 1 for the tile this worker begins and leaves, slot 0 for one it comes into
      float* part = a.part + ((long long)worker * 2 + (u0 == 0 ? 1 : 0)) * kFewRows * kPartRow;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = (lane >> 2) + 8 * h;
        if (r < rows) {
          const int dim = warp * 32 + (lane & 3) * 2;
          const float lr = ctl.l[r], inv = lr > 0.0f || lr != lr ? 1.0f / lr : 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = acc[i][h * 2], y = acc[i][h * 2 + 1];
            if (whole) *reinterpret_cast<__nv_bfloat162*>(a.out + (g + r) * kLat + dim + i * 8) = __floats2bfloat162_rn(x * inv, y * inv);
            else *reinterpret_cast<float2*>(part + r * kPartRow + dim + i * 8) = make_float2(x, y);
          }
        }
      }
      if (tid < rows) {
        if (whole) {
          a.lse[g + tid] = (ctl.m[tid] + log2f(ctl.l[tid])) * 0.69314718055994531f;
        } else {
          part[tid * kPartRow + kLat] = ctl.m[tid];
          part[tid * kPartRow + kLat + 1] = ctl.l[tid];
        }
      }
      if (!whole && u0 == 0 && tid == 0) {
        a.meta[worker * 4] = (int)g;
        a.meta[worker * 4 + 1] = rows;
        a.meta[worker * 4 + 2] = sh.holder(at + units) - worker + 1;
      }
      at += units;
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------
// host side

static int encode_rows(CUtensorMap* map, const void* base, int cols, int64_t rows, int64_t pitch, int box) {
  static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> known{nullptr};
  PFN_cuTensorMapEncodeTiled_v12000 fn = known.load(std::memory_order_acquire);
  if (!fn) {
    cudaDriverEntryPointQueryResult qr;
    const int rc = cache_cuda(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", (void**)&fn, cudaEnableDefault, &qr),
                              "cudaGetDriverEntryPoint(cuTensorMapEncodeTiled)");
    if (rc) return rc;
    if (qr != cudaDriverEntryPointSuccess || !fn) return KK3_ERR_CUDA;
    known.store(fn, std::memory_order_release);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch * 2};
  const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, steps[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, boxes, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? KK3_OK : KK3_ERR_ARG;
}

// maps of all the rows of a [pages, page_size, cols] tensor: in boxes and row by row
static int map_pages(CUtensorMap* by_box, CUtensorMap* by_row, int* ratio, int* end, const void* base, int cols,
                     const kk3_cache* c, int64_t page_stride, int64_t row_stride, int box) {
  const int64_t pages = c->num_pages;
  if (c->page_size == 1 && pages > 1) row_stride = page_stride;
  const int64_t r = pages > 1 ? page_stride / row_stride : c->page_size, rows = (pages - 1) * r + c->page_size;
  if (row_stride < cols || (pages > 1 && page_stride % row_stride) || rows >= INT32_MAX) return KK3_ERR_UNSUPPORTED;
  *ratio = (int)r;
  *end = (int)rows;
  const int rc = encode_rows(by_row, base, cols, rows, row_stride, 1);
  return rc || !box ? rc : encode_rows(by_box, base, cols, rows, row_stride, box);
}

// map of the rows of a [tokens, heads, cols] tensor whose (token, head) rows lie at one pitch
static int map_queries(CUtensorMap* map, const void* base, int cols, int64_t tokens, int64_t heads, int64_t tok_stride,
                       int64_t head_stride, int box) {
  if (heads == 1) head_stride = tokens == 1 ? cols : tok_stride;
  if (head_stride < cols || (tokens > 1 && tok_stride != heads * head_stride)) return KK3_ERR_UNSUPPORTED;
  return encode_rows(map, base, cols, tokens * heads, head_stride, box);
}

// the cache's maps, in boxes of at most `most` rows
static int cache_maps(const kk3_cache* c, int most, PairMaps* m, PairRows* r) {
  memset(m, 0, sizeof(*m));
  r->box = most;
  while (c->page_size % r->box) r->box /= 2;
  if (r->box < 8) r->box = 0;
  const int rc = map_pages(&m->kv_box, &m->kv_row, &r->kv_ratio, &r->kv_end, c->kv, kLat, c, c->kv_page_stride, c->kv_row_stride, r->box);
  return rc ? rc : map_pages(&m->pe_box, &m->pe_row, &r->pe_ratio, &r->pe_end, c->pe, kRope, c, c->pe_page_stride, c->pe_row_stride, r->box);
}

static int pair_maps(const kk3_cache* c, const void* q_latent, int64_t ql_token, int64_t ql_head, const void* q_pe,
                     int64_t qp_token, int64_t qp_head, int tokens, int heads, int q_box, PairMaps* m, PairRows* r) {
  int rc = cache_maps(c, 64, m, r);
  if (!rc) rc = map_queries(&m->ql, q_latent, kLat, tokens, heads, ql_token, ql_head, q_box);
  if (!rc) rc = map_queries(&m->qp, q_pe, kRope, tokens, heads, qp_token, qp_head, q_box);
  return rc;
}

int attend_pair(const kk3_cache* c, const AttendArgs& a, cudaStream_t st) {
  PairMaps maps;
  PairRows pr;
  int r = pair_maps(c, a.q_lat, a.ql_tok, a.ql_head, a.q_pe, a.qp_tok, a.qp_head, a.tokens, a.heads, 64, &maps, &pr);
  if (r) return r;
  static std::atomic<bool> ready[kCacheMaxDevices];
  r = cache_allow_smem(kk3_cache_attend_pair_kernel, kPaSmem, ready, "cudaFuncSetAttribute(kk3_cache_attend_pair_kernel)");
  if (r) return r;
  kk3_cache_attend_pair_kernel<<<a.workers * 2, kPaThreads, kPaSmem, st>>>(a, pr, maps);
  return cache_cuda(cudaGetLastError(), "kk3_cache_attend_pair_kernel");
}

int attend_few(const kk3_cache* c, const AttendArgs& a, cudaStream_t st) {
  PairMaps maps;
  PairRows pr;
  int r = cache_maps(c, kFewUnit, &maps, &pr);
  if (r) return r;
  static std::atomic<bool> ready[kCacheMaxDevices];
  r = cache_allow_smem(kk3_cache_attend_few_kernel, kFewSmem, ready, "cudaFuncSetAttribute(kk3_cache_attend_few_kernel)");
  if (r) return r;
  kk3_cache_attend_few_kernel<<<a.workers, kFewThreads, kFewSmem, st>>>(a, pr, maps);
  return cache_cuda(cudaGetLastError(), "kk3_cache_attend_few_kernel");
}

// rows of a matrix instruction for the average rows of a sequence: the smallest of 32, 64, 128 and 256 that holds
// them, 256 for more. A unit's products take as long as its rows are many, and each unit reads the tile's blocks from
// shared memory anew: 16 sequences of up to 8192 positions with 12 rows each took 31 us with 32 rows and 37 with
// 256, four with 96 rows each 19 us with 128, 21 with 256 and 29 with 32.
static int mass_rows(int64_t tokens, int64_t heads, int64_t batch) {
  int rows = 32;
  while (rows < 256 && (int64_t)rows * batch < tokens * heads) rows *= 2;
  return rows;
}

}  // namespace kk3

using namespace kk3;

extern "C" int64_t kk3_cache_mass_workspace(void) {
  int sms = 0;
  if (cache_sms(&sms)) return 0;
  return (int64_t)(sms / 2) * (16 + 2 * kMassPos * 4);
}

extern "C" int kk3_cache_mass(const kk3_cache_mass_args* x, void* stream) {
  if (!x) return KK3_ERR_ARG;
  MassArgs a;
  const int rc = cache_pages(&x->cache, &a.c, x->error_word);
  if (rc) return rc;
  const int tokens = x->tokens, heads = x->heads;
  if (tokens < 0 || heads < 1 || !cache_aligned(x->lengths, 8) || !cache_aligned(x->cu_new, 4) || !cache_scale(x->scale) ||
      !cache_aligned(x->new_mass, 4) || (x->mass && ((uintptr_t)x->mass % 4 || x->mass_stride < 0)))
    return KK3_ERR_ARG;
  // in place only row by row: with another stride a row is written while a CTA reads the one that lies there
  if (x->mass == x->new_mass && a.c.batch > 1 && x->mass_stride != (int64_t)a.c.columns * a.c.page_size) return KK3_ERR_ARG;
  if (heads > kMaxHeads || (int64_t)tokens * heads > INT32_MAX / 2) return KK3_ERR_UNSUPPORTED;
  if (tokens > 0 && (!cache_queries(x->q_latent, x->ql_token, x->ql_head, x->q_pe, x->qp_token, x->qp_head) ||
                     !cache_aligned(x->lse, 4)))
    return KK3_ERR_ARG;
  int sms = 0;
  if (cache_sms(&sms)) return KK3_ERR_CUDA;
  if (!cache_aligned(x->workspace, 16) || x->workspace_bytes < kk3_cache_mass_workspace()) return KK3_ERR_ARG;
  a.q_lat = (const bf16*)x->q_latent;
  a.q_pe = (const bf16*)x->q_pe;
  a.ql_tok = x->ql_token;
  a.ql_head = x->ql_head;
  a.qp_tok = x->qp_token;
  a.qp_head = x->qp_head;
  a.lse = x->lse;
  a.lengths = (const long long*)x->lengths;
  a.cu_new = x->cu_new;
  a.tokens = tokens;
  a.heads = heads;
  a.scale_log2 = x->scale * 1.4426950408889634f;
  a.mass = x->mass;
  a.mass_row = x->mass_stride;
  a.out = x->new_mass;
  a.workers = sms / 2;
  a.meta = (int*)x->workspace;
  a.part = (float*)((char*)x->workspace + (size_t)a.workers * 16);
  PairMaps maps;
  PairRows pr;
  const int rows = mass_rows(tokens, heads, a.c.batch);
  if (tokens > 0) {
    const int r = pair_maps(&x->cache, x->q_latent, x->ql_token, x->ql_head, x->q_pe, x->qp_token, x->qp_head, tokens, heads, rows / 2, &maps, &pr);
    if (r) return r;
  } else {
    memset(&maps, 0, sizeof(maps));   // no tile reads them
    memset(&pr, 0, sizeof(pr));
  }
  static std::atomic<bool> ready[kCacheMaxDevices];
  int r = cache_allow_smem(kk3_cache_mass_kernel, kMassSmem, ready, "cudaFuncSetAttribute(kk3_cache_mass_kernel)");
  if (r) return r;
  const cudaStream_t st = (cudaStream_t)stream;
  kk3_cache_mass_kernel<<<a.workers * 2, kMassThreads, kMassSmem, st>>>(a, pr, maps, rows);
  r = cache_cuda(cudaGetLastError(), "kk3_cache_mass_kernel");
  if (r) return r;
  return cache_launch_after(kk3_cache_mass_join_kernel, dim3(a.workers), kMassPos, st, "kk3_cache_mass_join_kernel", a);
}
