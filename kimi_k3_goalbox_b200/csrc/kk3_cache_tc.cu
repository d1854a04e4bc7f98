// kk3_cache_tc.cu - tensor-core kernels of the paged latent cache (tcgen05, sm_100a): the accumulated attention weight.
//
// Operands are gathered row by row through the page table with 16-byte cp.async (any page size; rows behind a
// sequence's end arrive as zeros, whatever their page holds) straight into the 128-byte swizzled form that the
// matrix instructions read, in blocks of 64 dims (128 bytes a row).
#include <cuda_runtime.h>

#include "kk3_cache.cuh"
#include "kk3_cache_host.h"
#include "kk3_tcgen05.cuh"

namespace kk3 {

constexpr int kBlocks = kEntry / 64;                    // 64-dim blocks of an entry
constexpr unsigned long long kWaitNs = 2000000000ull;   // bound of every wait; a healthy one takes microseconds

KK3_DEV unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }

// Bounded wait; false when it ran out or another role of the CTA gave up (*dead).
KK3_DEV bool bar_wait(const CachePages& c, unsigned bar, unsigned parity, volatile int* dead) {
  if (mbar_test(bar, parity)) return true;
  const unsigned long long t0 = globaltimer();
  for (unsigned spin = 1;; ++spin) {
    if (mbar_test(bar, parity)) return true;
    if ((spin & 15) == 0) {
      if (*dead) return false;
      if (globaltimer() - t0 > kWaitNs) {
        *dead = 1;
        if (c.error_word) *reinterpret_cast<volatile int*>(c.error_word) = kErrTimeout;
        return false;
      }
    }
  }
}
KK3_DEV void cp16(unsigned dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
KK3_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
KK3_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// 16-byte piece `ch` of row `r` in a 128-byte swizzled block (1024-byte aligned)
KK3_DEV unsigned sw128(int r, int ch) { return (unsigned)(r * 128 + ((ch ^ (r & 7)) << 4)); }
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

// ---------------------------------------------------------------------------------------------
// Attention weight of cached positions: w_p = sum over rows of 2^(s_p - lse), s_p = q . e_p.
//
// One product, positions x rows, with the positions as the 128 rows of the matrix instruction: a thread then owns a
// position (its TMEM lane) and adds up its columns in registers, in row order; no reduction crosses threads and
// no atomic is needed. A tile is 128 positions: its 147 KB stay in shared memory while the sequence's rows pass
// through a ring in units of NR rows x 576 dims; two accumulators let the sums of one unit run under the products
// of the next. When the rows fit one unit (single tokens) the tile's blocks are freed block by block instead and
// the kernel streams the cache: LAG blocks of 16 KB are in flight.
//
// Bounds, per unit of 128 x 128 x 576: shared memory feeds the instructions 295 KB, 2304 clocks at 128 bytes a
// clock, against 1152 clocks of tensor time; exponentials take 1024.

constexpr int kMassPos = 128;
constexpr int kMassThreads = 288;   // warps 0-3 sums, 4-7 copies, 8 matrix instructions and TMEM
constexpr int kMassKBlock = kMassPos * 128;
constexpr int kMassRing = 65536;

template <int NR>
struct MassLayout {
  static constexpr int kSlotBytes = NR * 128;
  static constexpr int kSlots = kMassRing / kSlotBytes < 16 ? kMassRing / kSlotBytes : 16;
  static constexpr int kLag = kSlots - 1 < kBlocks - 1 ? kSlots - 1 : kBlocks - 1;   // groups in flight behind the newest
  static constexpr int kCtl = kBlocks * kMassKBlock + kSlots * kSlotBytes;           // byte offset of the control block
};
struct MassCtl {
  unsigned long long full[16], empty[16], kempty[kBlocks], dfull[2], dempty[2], done;
  unsigned tmem;
  int dead;
  long long red[kMassThreads / 32 + 4];
  float lse[2][128];
  int sees[2][128];
};

template <int NR>
__global__ void __launch_bounds__(kMassThreads, 1) kk3_cache_mass_kernel(const MassArgs a) {
  using L = MassLayout<NR>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  MassCtl& ctl = *reinterpret_cast<MassCtl*>(base + L::kCtl);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, worker = blockIdx.x;
  const unsigned kbase = smem_u32(base), qbase = kbase + kBlocks * kMassKBlock;
  const MassSplit split{kMassPos, NR, a.heads};
  const Share sh = plan_share<kMassThreads>(a, split, worker, 1, reinterpret_cast<int*>(base), ctl.red);
  if (tid == 0) a.meta[worker * 4 + 2] = 0;
  // what the call leaves as it is: positions behind the sequences' ends, and sequences without new tokens
  {
    const long long cap = (long long)a.c.columns * a.c.page_size;
    for (int b = worker; b < a.c.batch; b += gridDim.x) {
      const Seq s = a.seq(b);
      for (long long p = (s.n > 0 ? s.len : 0) + tid; p < cap; p += kMassThreads)
        a.out[b * cap + p] = a.mass ? a.mass[b * a.mass_row + p] : 0.0f;
    }
  }
  if (worker >= sh.workers || sh.total == 0) return;
  const unsigned full = smem_u32(ctl.full), empty = smem_u32(ctl.empty), kempty = smem_u32(ctl.kempty),
                 dfull = smem_u32(ctl.dfull), dempty = smem_u32(ctl.dempty), done = smem_u32(&ctl.done);
  volatile int* dead = &ctl.dead;
  if (tid == 0) {
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(full + 8 * i, 4);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kBlocks; ++i) mbar_init(kempty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(dfull + 8 * i, 1);
      mbar_init(dempty + 8 * i, 4);
    }
    mbar_init(done, 1);
    ctl.dead = 0;
    fence_mbar_init();
  }
  if (warp == 8) tmem_alloc(smem_u32(&ctl.tmem), 2 * NR);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = *reinterpret_cast<volatile unsigned*>(&ctl.tmem);

  int b = sh.b, t = sh.t;
  long long at = sh.at;
  if (warp >= 4 && warp < 8) {
    // ---- copies
    const int pw = warp - 4, sub = lane >> 3, ch = lane & 7;
    int job = 0, tile = 0;
    bool ok = true;
    while (ok && at < sh.end) {
      Seq s = a.seq(b);
      for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
      const int units = split.units(s, t), first = split.first_unit(s, t);
      const int u0 = (int)max(0ll, sh.begin - at), u1 = (int)min((long long)units, sh.end - at);
      long long koff[8], poff[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pos = t * kMassPos + pw * 32 + i * 4 + sub;
        koff[i] = poff[i] = -1;
        if (pos < s.len) {
          int slot;
          const int page = page_at(a.c, b, pos, &slot);
          if (page >= 0) {
            koff[i] = (long long)page * a.c.kv_page + (long long)slot * a.c.kv_row + ch * 8;
            poff[i] = (long long)page * a.c.pe_page + (long long)slot * a.c.pe_row + ch * 8;
          }
        }
      }
      for (int u = u0; ok && u < u1; ++u) {
        long long qoff[NR / 16], roff[NR / 16];
#pragma unroll
        for (int i = 0; i < NR / 16; ++i) {
          const long long g = (long long)(first + u) * NR + pw * (NR / 4) + i * 4 + sub;
          qoff[i] = roff[i] = -1;
          if (g < (long long)s.n * a.heads) {
            const int tok = s.q0 + (int)(g / a.heads), head = (int)(g % a.heads);
            qoff[i] = tok * a.ql_tok + head * a.ql_head + ch * 8;
            roff[i] = tok * a.qp_tok + head * a.qp_head + ch * 8;
          }
        }
        for (int d = 0; d < kBlocks; ++d) {
          const int slot = job % L::kSlots;
          ok = bar_wait(a.c, empty + 8 * slot, ((job / L::kSlots) & 1) ^ 1, dead);
          if (ok && u == u0) ok = bar_wait(a.c, kempty + 8 * d, (tile & 1) ^ 1, dead);
          if (!ok) break;
          if (u == u0) {
            const unsigned dst = kbase + d * kMassKBlock;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const long long o = d < kBlocks - 1 ? koff[i] : poff[i];
              const bf16* src = d < kBlocks - 1 ? a.c.kv + o + d * 64 : a.c.pe + o;
              cp16(dst + sw128(pw * 32 + i * 4 + sub, ch), o >= 0 ? src : a.c.kv, o >= 0);
            }
          }
          const unsigned dst = qbase + slot * L::kSlotBytes;
#pragma unroll
          for (int i = 0; i < NR / 16; ++i) {
            const long long o = d < kBlocks - 1 ? qoff[i] : roff[i];
            const bf16* src = d < kBlocks - 1 ? a.q_lat + o + d * 64 : a.q_pe + o;
            cp16(dst + sw128(pw * (NR / 4) + i * 4 + sub, ch), o >= 0 ? src : a.q_lat, o >= 0);
          }
          cp_commit();
          if (job >= L::kLag) {
            cp_wait<L::kLag>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * ((job - L::kLag) % L::kSlots));
          }
          ++job;
        }
      }
      at += units;
      ++t;
      ++tile;
    }
    cp_wait<0>();
    fence_async_smem();
    __syncwarp();
    if (lane == 0)
      for (int j = max(0, job - L::kLag); j < job; ++j) mbar_arrive(full + 8 * (j % L::kSlots));
  } else if (warp == 8) {
    // ---- matrix instructions (one thread)
    if (lane == 0) {
      constexpr unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(NR >> 3) << 17) | ((128u >> 4) << 24);
      int job = 0, unit = 0;
      bool ok = true;
      while (ok && at < sh.end) {
        Seq s = a.seq(b);
        for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
        const int units = split.units(s, t);
        const int u0 = (int)max(0ll, sh.begin - at), u1 = (int)min((long long)units, sh.end - at);
        for (int u = u0; ok && u < u1; ++u, ++unit) {
          const int buf = unit & 1;
          ok = bar_wait(a.c, dempty + 8 * buf, ((unit >> 1) & 1) ^ 1, dead);
          tc_fence_after();
          for (int d = 0; ok && d < kBlocks; ++d, ++job) {
            const int slot = job % L::kSlots;
            ok = bar_wait(a.c, full + 8 * slot, (job / L::kSlots) & 1, dead);
            if (!ok) break;
            tc_fence_after();
            const unsigned ka = kbase + d * kMassKBlock, qa = qbase + slot * L::kSlotBytes;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              asm volatile(
                  "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                  " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                  ::"r"(tmem + buf * NR), "l"(sdesc_sw128(ka + k * 32)), "l"(sdesc_sw128(qa + k * 32)), "r"(idesc),
                    "r"((unsigned)(d | k))
                  : "memory");
            }
            umma_commit(empty + 8 * slot);
            if (u == u1 - 1) umma_commit(kempty + 8 * d);
          }
          if (ok) umma_commit(dfull + 8 * buf);
        }
        at += units;
        ++t;
      }
      umma_commit(done);   // all matrix instructions end before TMEM is given back
      mbar_wait_for(done, 0, kWaitNs);
    }
    __syncwarp();
  } else {
    // ---- sums: thread = position
    const unsigned tlane = (unsigned)(warp * 32) << 16;
    int unit = 0;
    bool ok = true;
    while (ok && at < sh.end) {
      Seq s = a.seq(b);
      for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
      const int units = split.units(s, t), first = split.first_unit(s, t);
      const int u0 = (int)max(0ll, sh.begin - at), u1 = (int)min((long long)units, sh.end - at);
      const int pos = t * kMassPos + tid;
      float sum = 0.0f;
      for (int u = u0; ok && u < u1; ++u, ++unit) {
        const int buf = unit & 1;
        // this unit's rows: negative log sums (rows that do not exist or see nothing: the products vanish)
        const long long g0 = (long long)(first + u) * NR, all = (long long)s.n * a.heads;
        if (tid < NR) {
          const long long g = g0 + tid;
          const float l = g < all ? a.lse[(long long)s.q0 * a.heads + g] : -INFINITY;
          ctl.lse[buf][tid] = l == -INFINITY ? -INFINITY : -l * 1.4426950408889634f;
          ctl.sees[buf][tid] = g < all ? s.len - s.n + (int)(g / a.heads) + 1 : 0;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const bool causal = s.len - s.n + (int)(g0 / a.heads) + 1 < min(s.len, (t + 1) * kMassPos);
        ok = bar_wait(a.c, dfull + 8 * buf, (unit >> 1) & 1, dead);
        tc_fence_after();
        if (ok) {
#pragma unroll 1
          for (int c = 0; c < NR; c += 32) {
            float v[32];
            tmem_ld32(tmem + tlane + buf * NR + c, v);
            tmem_ld_wait();
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 l = *reinterpret_cast<const float4*>(&ctl.lse[buf][c + i]);
              const float w0 = ex2(fmaf(v[i], a.scale_log2, l.x)), w1 = ex2(fmaf(v[i + 1], a.scale_log2, l.y));
              const float w2 = ex2(fmaf(v[i + 2], a.scale_log2, l.z)), w3 = ex2(fmaf(v[i + 3], a.scale_log2, l.w));
              if (causal) {
                const int4 n = *reinterpret_cast<const int4*>(&ctl.sees[buf][c + i]);
                part += (pos < n.x ? w0 : 0.0f) + (pos < n.y ? w1 : 0.0f) + (pos < n.z ? w2 : 0.0f) + (pos < n.w ? w3 : 0.0f);
              } else {
                part += (w0 + w1) + (w2 + w3);
              }
            }
            sum += part;
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dempty + 8 * buf);
      }
      if (ok) {
        if (u0 == 0 && u1 == units) {
          if (pos < s.len) {
            const long long cap = (long long)a.c.columns * a.c.page_size;
            a.out[b * cap + pos] = (a.mass ? a.mass[b * a.mass_row + pos] : 0.0f) + sum;
          }
        } else {
          a.part[(worker * 2 + (u0 == 0 ? 1 : 0)) * kMassPos + tid] = sum;
          if (u0 == 0 && tid == 0) {   // the workers of this tile: up to the one that holds its last unit
            int last = worker;
            while (sh.total * (last + 1) / sh.workers < at + units) ++last;
            a.meta[worker * 4] = b;
            a.meta[worker * 4 + 1] = t;
            a.meta[worker * 4 + 2] = last - worker + 1;
          }
        }
      }
      at += units;
      ++t;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 2 * NR);
}

__global__ void __launch_bounds__(kMassPos) kk3_cache_mass_join_kernel(const MassArgs a) {
  const int worker = blockIdx.x, n = a.meta[worker * 4 + 2];
  if (n == 0) return;
  const int b = a.meta[worker * 4], pos = a.meta[worker * 4 + 1] * kMassPos + threadIdx.x;
  if (pos >= a.seq(b).len) return;
  float sum = 0.0f;
  for (int w = 0; w < n; ++w) sum += a.part[((worker + w) * 2 + (w == 0 ? 1 : 0)) * kMassPos + threadIdx.x];
  const long long cap = (long long)a.c.columns * a.c.page_size;
  a.out[b * cap + pos] = (a.mass ? a.mass[b * a.mass_row + pos] : 0.0f) + sum;
}

template <int NR>
static int mass_launch(const MassArgs& a, cudaStream_t st) {
  const size_t smem = MassLayout<NR>::kCtl + sizeof(MassCtl) + 1024;
  int r = cache_cuda(cudaFuncSetAttribute(kk3_cache_mass_kernel<NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                     "cudaFuncSetAttribute(kk3_cache_mass_kernel)");
  if (r) return r;
  kk3_cache_mass_kernel<NR><<<a.workers, kMassThreads, smem, st>>>(a);
  r = cache_cuda(cudaGetLastError(), "kk3_cache_mass_kernel");
  if (r) return r;
  kk3_cache_mass_join_kernel<<<a.workers, kMassPos, 0, st>>>(a);
  return cache_cuda(cudaGetLastError(), "kk3_cache_mass_join_kernel");
}

}  // namespace kk3

using namespace kk3;

extern "C" int64_t kk3_cache_mass_workspace(int batch, int tokens, int heads) {
  if (batch < 1 || tokens < 0 || heads < 1 || heads > kMaxHeads) return 0;
  int sms = 0;
  if (cache_sms(&sms)) return 0;
  return (int64_t)sms * (16 + 2 * kMassPos * 4);
}

extern "C" int kk3_cache_mass(const kk3_cache* cache, const void* q_latent, int64_t ql_token, int64_t ql_head,
                              const void* q_pe, int64_t qp_token, int64_t qp_head, const float* lse,
                              const int64_t* lengths, const int32_t* cu_new, int tokens, int heads, float scale,
                              const float* mass, int64_t mass_stride, float* new_mass, void* workspace,
                              int64_t workspace_bytes, int* error_word, void* stream) {
  MassArgs a;
  const int rc = cache_pages(cache, &a.c, error_word);
  if (rc) return rc;
  if (tokens < 0 || heads < 1 || !cache_aligned(lengths, 8) || !cache_aligned(cu_new, 4) || !(scale == scale) ||
      !cache_aligned(new_mass, 4) || (mass && ((uintptr_t)mass % 4 || mass_stride < 0)))
    return KK3_ERR_ARG;
  if (heads > kMaxHeads || (int64_t)tokens * heads > INT32_MAX / 2) return KK3_ERR_UNSUPPORTED;
  if (tokens > 0 && (!cache_aligned(q_latent, 16) || !cache_aligned(q_pe, 16) || !cache_aligned(lse, 4) || ql_token % 8 ||
                     ql_head % 8 || qp_token % 8 || qp_head % 8 || ql_token < 0 || ql_head < 0 || qp_token < 0 || qp_head < 0))
    return KK3_ERR_ARG;
  int sms = 0;
  if (cache_sms(&sms)) return KK3_ERR_CUDA;
  if (!cache_aligned(workspace, 16) || workspace_bytes < kk3_cache_mass_workspace(a.c.batch, tokens, heads)) return KK3_ERR_ARG;
  a.q_lat = (const bf16*)q_latent;
  a.q_pe = (const bf16*)q_pe;
  a.ql_tok = ql_token;
  a.ql_head = ql_head;
  a.qp_tok = qp_token;
  a.qp_head = qp_head;
  a.lse = lse;
  a.lengths = (const long long*)lengths;
  a.cu_new = cu_new;
  a.tokens = tokens;
  a.heads = heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.mass = mass;
  a.mass_row = mass_stride;
  a.out = new_mass;
  a.workers = sms;
  a.meta = (int*)workspace;
  a.part = (float*)((char*)workspace + (size_t)sms * 16);
  // rows per unit: 32 where a sequence's rows fit (single tokens on a rank: the ring then holds more cache blocks in
  // flight), 128 otherwise
  const bool few = (int64_t)tokens * heads <= (int64_t)32 * a.c.batch;
  return few ? mass_launch<32>(a, (cudaStream_t)stream) : mass_launch<128>(a, (cudaStream_t)stream);
}
