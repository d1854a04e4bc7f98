// kk3_cache.cu - kernels and C entry points of the paged latent cache (include/kk3.h, kk3_cache_*): append, attention
// of new tokens at warp level, the join of split attention tiles, eviction.
#include <cuda_runtime.h>

#include "kk3_cache.cuh"
#include "kk3_cache_host.h"

namespace kk3 {

KK3_DEV void cp_async16_zfill(void* smem, const void* src, bool live) {
  const unsigned dst = (unsigned)__cvta_generic_to_shared(smem);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
KK3_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
KK3_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
KK3_DEV void ldsm4(unsigned (&r)[4], const void* p) {
  const unsigned a = (unsigned)__cvta_generic_to_shared(p);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
KK3_DEV void ldsm4t(unsigned (&r)[4], const void* p) {
  const unsigned a = (unsigned)__cvta_generic_to_shared(p);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

// ---------------------------------------------------------------------------------------------
// append: latent = x[:512] / rms(x[:512]) * weight (FP32, rounded to BF16 once), rope = x[512:], into the page of the
// token's position. One warp per token, bound by its 2304 bytes of traffic; 16-byte accesses throughout (lane l owns
// the latent values 8 l .. 8 l + 7 and 256 + 8 l ..; eight lanes copy the rope part).

struct AppendArgs {
  CachePages c;
  const bf16* raw;
  long long raw_row;
  const bf16* weight;
  const long long* lengths;
  long long* new_lengths;
  const int* cu_new;
  int tokens;
  float eps;
};

constexpr int kAppendWarps = 4;

__global__ void __launch_bounds__(kAppendWarps * 32) kk3_cache_append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int tok = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  const int B = a.c.batch;
  const long long cap = (long long)a.c.columns * a.c.page_size;
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
      const int q0 = min(max(a.cu_new[b], 0), a.tokens), q1 = min(max(a.cu_new[b + 1], q0), a.tokens);
      const long long l = a.lengths[b], sum = (l < 0 ? 0 : l) + (q1 - q0);
      if (l < 0 || sum > cap) cache_error(a.c);
      a.new_lengths[b] = sum > cap ? cap : sum;
    }
  }
  if (tok >= a.tokens) return;
  int lo = 0, hi = B;   // the sequence of this token: cu_new[lo] <= tok < cu_new[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_new[mid] <= tok) lo = mid; else hi = mid;
  }
  const int first = a.cu_new[lo];
  if (tok < first || tok >= a.cu_new[lo + 1] || first < 0) return;   // behind the last sequence: no one's token
  const long long pos = max(a.lengths[lo], 0ll) + (tok - first);
  if (pos >= cap) return;
  int slot;
  const int page = page_at(a.c, lo, (int)pos, &slot);
  if (page < 0) return;
  const bf16* x = a.raw + (long long)tok * a.raw_row;
  uint4 v[2], w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v[h] = *reinterpret_cast<const uint4*>(x + h * 256 + lane * 8);
    w[h] = *reinterpret_cast<const uint4*>(a.weight + h * 256 + lane * 8);
  }
  uint4 rope = {};
  if (lane < 8) rope = *reinterpret_cast<const uint4*>(x + kLat + lane * 8);
  float sum = 0.0f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v[h]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(p[i]);
      sum = fmaf(f.x, f.x, fmaf(f.y, f.y, sum));
    }
  }
  const float r = rsqrtf(warp_sum(sum) * (1.0f / kLat) + a.eps);
  bf16* kv = a.c.kv + (long long)page * a.c.kv_page + (long long)slot * a.c.kv_row;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&v[h]);
    const __nv_bfloat162* q = reinterpret_cast<const __nv_bfloat162*>(&w[h]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(p[i]), g = __bfloat1622float2(q[i]);
      p[i] = __floats2bfloat162_rn(f.x * r * g.x, f.y * r * g.y);
    }
    *reinterpret_cast<uint4*>(kv + h * 256 + lane * 8) = v[h];
  }
  if (lane < 8)
    *reinterpret_cast<uint4*>(a.c.pe + (long long)page * a.c.pe_page + (long long)slot * a.c.pe_row + lane * 8) = rope;
}

// ---------------------------------------------------------------------------------------------
// Attention at warp level: a tile is 16 or 32 (MT = 1, 2) (token, head) rows, a unit 64 cached positions.
//
//   s = scale (q . e_p), running maximum m and sum l per row, O = O 2^(m - m') + sum_p 2^(s - m') c_p
//
// Each cached entry is read once per tile and serves both products from shared memory, so few rows per sequence leave
// the call bound by the cache's bytes: 64 positions are 73.7 KB, 3200 clocks at one SM's share of HBM, against some
// 1400 (MT = 1) of work. 8 warps; the query's fragments stay in registers (each warp holds one half of the 576 dims: 18
// k-steps) and 16 of the unit's positions are a warp's in the first product; warp w owns the output dims
// 64 w .. 64 w + 63 in the second. Stages of 32 positions (36.5 KB) arrive by cp.async, three and more ahead; the page
// numbers they need are looked up one unit before that.
// Probabilities are rounded to BF16 for the second product, the type that the instruction takes with BF16 latents; the
// running sum adds them unrounded, since lse is an FP32 result.

constexpr int kWaUnit = 64, kWaStage = 32;
constexpr int kWaPitch = kEntry + 8;      // 1168-byte rows: consecutive rows fall on different banks (ldmatrix)
constexpr int kWaPPitch = kWaUnit + 8;
constexpr int kWaThreads = 256;
constexpr int kWaMinUnits = 2;
template <int MT>
struct WaSmem {
  static constexpr int kRows = 16 * MT, kStages = MT == 1 ? 5 : 4;
  bf16 ring[kStages][kWaStage][kWaPitch];
  bf16 q[kRows][kWaPitch];
  float s[2][kRows][kWaUnit + 4];
  bf16 p[kRows][kWaPPitch];
  float alpha[kRows];
  float m[kRows], l[kRows];
  long long red[kWaThreads / 32 + 4];
};
static_assert(sizeof(WaSmem<1>) <= 232448 && sizeof(WaSmem<2>) <= 232448, "shared memory of a CTA");

// Page of this lane's position (lanes 0 .. 3: the warp's four) of stage `st`, -1 where the tile sees none.
KK3_DEV int wa_page(const CachePages& c, int b, int st, int sees) {
  const int lane = threadIdx.x & 31, pos = st * kWaStage + (threadIdx.x >> 5) * 4 + lane;
  return lane < 4 && pos < sees ? c.table[(long long)b * c.table_stride + page_of(c, pos)] : -1;
}
// Copy stage `st` into `ring`, rows without a page as zeros. `page`: wa_page's.
KK3_DEV void wa_load(const CachePages& c, bf16 (*ring)[kWaPitch], int st, int sees, int page) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long kv = -1, pe = -1;
  if (lane < 4) {
    const int pos = st * kWaStage + warp * 4 + lane;
    if (pos < sees) {
      if ((unsigned)page < (unsigned)c.num_pages) {
        const int slot = pos - page_of(c, pos) * c.page_size;
        kv = (long long)page * c.kv_page + (long long)slot * c.kv_row;
        pe = (long long)page * c.pe_page + (long long)slot * c.pe_row;
      } else {
        cache_error(c);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = i >> 1, chunk = (i & 1) * 32 + lane;
    const long long o = __shfl_sync(0xffffffffu, kv, row);
    cp_async16_zfill(&ring[warp * 4 + row][chunk * 8], o >= 0 ? c.kv + o + chunk * 8 : c.kv, o >= 0);
  }
  const long long o = __shfl_sync(0xffffffffu, pe, lane >> 3);
  cp_async16_zfill(&ring[warp * 4 + (lane >> 3)][kLat + (lane & 7) * 8], o >= 0 ? c.pe + o + (lane & 7) * 8 : c.pe, o >= 0);
}

template <int MT>
__global__ void __launch_bounds__(kWaThreads, 1) kk3_cache_attend_warp_kernel(const AttendArgs a) {
  constexpr int kRows = 16 * MT, kStages = WaSmem<MT>::kStages;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  WaSmem<MT>& sm = *reinterpret_cast<WaSmem<MT>*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int worker = blockIdx.x;
  static_assert(sizeof(sm.ring) >= (kMaxSeqs + 1) * sizeof(int), "the sequences' tile prefix lies in the ring");
  const AttendSplit split{kRows, a.heads, kWaUnit, 0};
  const Share sh = plan_share<kWaThreads>(a, split, worker, kWaMinUnits, reinterpret_cast<int*>(&sm.ring[0][0][0]),
                                          sm.red);
  if (tid == 0) a.meta[worker * 4 + 2] = 0;
  if (worker >= sh.workers) return;
  int b = sh.b, t = sh.t;
  long long at = sh.at;
  while (at < sh.end) {
    Seq s = a.seq(b);
    for (; t >= split.tiles(s); t = 0) s = a.seq(++b);
    const int units = split.units(s, t);
    const int u0 = split.from(sh, at, units), u1 = split.to(sh, at, units);
    const bool whole = u0 == 0 && u1 == units;
    const int row0 = t * kRows, rows = min(kRows, s.n * a.heads - row0);
    const int sees_max = split.sees(s, t);
    __syncthreads();   // the previous tile's readers are done with q, p and the ring
    // stages 2 u0 .. 2 u1 - 1; stage st is in slot (st - 2 u0) % kStages
    const int st0 = 2 * u0, st1 = 2 * u1;
    int page[2] = {wa_page(a.c, b, st0, sees_max), wa_page(a.c, b, st0 + 1, sees_max)};
    // query rows, zeros below the last
    for (int i = tid; i < kRows * (kEntry / 8); i += kWaThreads) {
      const int r = i / (kEntry / 8), ch = i % (kEntry / 8);
      const int g = row0 + min(r, rows - 1), tok = s.q0 + g / a.heads, head = g % a.heads;
      const bf16* src = ch < kLat / 8 ? a.q_lat + tok * a.ql_tok + head * a.ql_head + ch * 8
                                      : a.q_pe + tok * a.qp_tok + head * a.qp_head + (ch - kLat / 8) * 8;
      cp_async16_zfill(&sm.q[r][ch * 8], src, r < rows);
    }
    cp_async_commit();
#pragma unroll
    for (int i = 0; i < kStages - 2; ++i) {
      if (st0 + i < st1) wa_load(a.c, sm.ring[i], st0 + i, sees_max, page[i & 1]);
      cp_async_commit();
      if (st0 + i + 2 < st1) page[i & 1] = wa_page(a.c, b, st0 + i + 2, sees_max);
    }
    cp_async_wait<kStages - 2>();
    __syncthreads();
    // this warp's query fragments: k-steps 18 (warp / 4) .. + 17
    const int ntile = warp & 3, khalf = warp >> 2;
    unsigned qf[MT][18][4];
#pragma unroll
    for (int h = 0; h < MT; ++h)
#pragma unroll
      for (int k = 0; k < 18; ++k)
        ldsm4(qf[h][k], &sm.q[h * 16 + (lane & 15)][(khalf * 18 + k) * 16 + (lane >> 4) * 8]);
    float acc[MT][8][4] = {};
    // softmax rows of this warp: 2 MT warp .. + 2 MT - 1, two positions a lane
    float m[2 * MT], l[2 * MT];
    int sees[2 * MT];
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) {
      const int r = warp * 2 * MT + j;
      m[j] = -INFINITY;
      l[j] = 0.0f;
      sees[j] = r < rows ? s.len - s.n + (row0 + r) / a.heads + 1 : 0;
    }
    int slot = 0;   // of the unit's first stage
    for (int u = u0; u < u1; ++u) {
      // copies so far: stages up to 2 u + kStages - 3; those of this unit are in when kStages - 4 are left
      cp_async_wait<kStages - 4>();
      __syncthreads();   // and every warp is done with the unit before, whose slots are filled again
      const int next = 2 * u + kStages - 2;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int st = next + i, sl = (slot + kStages - 2 + i) % kStages;
        constexpr int kTurn = kStages & 1;   // page[] holds stages in turn
        if (st < st1) wa_load(a.c, sm.ring[sl], st, sees_max, page[(i + kTurn) & 1]);
        cp_async_commit();
        if (st + 2 < st1) page[(i + kTurn) & 1] = wa_page(a.c, b, st + 2, sees_max);
      }
      const int slot1 = (slot + 1) % kStages;
      {
        float c[MT][2][2][4] = {};   // [16 rows][8 positions][chain]
        const bf16(*ring)[kWaPitch] = sm.ring[ntile < 2 ? slot : slot1];
        const int prow = (ntile & 1) * 16;
#pragma unroll
        for (int k = 0; k < 18; k += 2) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            unsigned bf[4];
            ldsm4(bf, &ring[prow + n * 8 + (lane & 7)][(khalf * 18 + k) * 16 + (lane >> 3) * 8]);
#pragma unroll
            for (int h = 0; h < MT; ++h) {
              mma_bf16(c[h][n][0], qf[h][k][0], qf[h][k][1], qf[h][k][2], qf[h][k][3], bf[0], bf[1]);
              mma_bf16(c[h][n][1], qf[h][k + 1][0], qf[h][k + 1][1], qf[h][k + 1][2], qf[h][k + 1][3], bf[2], bf[3]);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < MT; ++h)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int r = h * 16 + (lane >> 2), col = ntile * 16 + n * 8 + (lane & 3) * 2;
            const float(*x)[4] = c[h][n];
            *reinterpret_cast<float2*>(&sm.s[khalf][r][col]) = make_float2(x[0][0] + x[1][0], x[0][1] + x[1][1]);
            *reinterpret_cast<float2*>(&sm.s[khalf][r + 8][col]) = make_float2(x[0][2] + x[1][2], x[0][3] + x[1][3]);
          }
      }
      __syncthreads();
      {
        float v[2 * MT][2], top[2 * MT];
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) {
          const int r = warp * 2 * MT + j;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int col = i * 32 + lane;
            v[j][i] = (sm.s[0][r][col] + sm.s[1][r][col]) * a.scale_log2;
            if (u * kWaUnit + col >= sees[j]) v[j][i] = -INFINITY;
          }
          top[j] = fmaxf(v[j][0], v[j][1]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int j = 0; j < 2 * MT; ++j) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) {
          const int r = warp * 2 * MT + j;
          top[j] = fmaxf(m[j], top[j]);
          const float ref = top[j] == -INFINITY ? 0.0f : top[j];
          const float al = exp2f(m[j] - ref);
          const float p0 = exp2f(v[j][0] - ref), p1 = exp2f(v[j][1] - ref);
          l[j] = l[j] * al + (p0 + p1);
          m[j] = top[j];
          sm.p[r][lane] = f2bf(p0);
          sm.p[r][32 + lane] = f2bf(p1);
          if (lane == 0) sm.alpha[r] = al;
        }
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < MT; ++h) {
        const float a0 = sm.alpha[h * 16 + (lane >> 2)], a1 = sm.alpha[h * 16 + (lane >> 2) + 8];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          acc[h][n][0] *= a0;
          acc[h][n][1] *= a0;
          acc[h][n][2] *= a1;
          acc[h][n][3] *= a1;
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        unsigned pf[MT][4];
#pragma unroll
        for (int h = 0; h < MT; ++h) ldsm4(pf[h], &sm.p[h * 16 + (lane & 15)][k * 16 + (lane >> 4) * 8]);
        const bf16(*ring)[kWaPitch] = sm.ring[k < 2 ? slot : slot1];
#pragma unroll
        for (int n = 0; n < 8; n += 2) {
          unsigned bf[4];
          ldsm4t(bf, &ring[(k & 1) * 16 + (lane & 15)][warp * 64 + n * 8 + (lane >> 4) * 8]);
#pragma unroll
          for (int h = 0; h < MT; ++h) {
            mma_bf16(acc[h][n], pf[h][0], pf[h][1], pf[h][2], pf[h][3], bf[0], bf[1]);
            mma_bf16(acc[h][n + 1], pf[h][0], pf[h][1], pf[h][2], pf[h][3], bf[2], bf[3]);
          }
        }
      }
      slot = (slot + 2) % kStages;
    }
    cp_async_wait<0>();
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) {
      l[j] = warp_sum(l[j]);
      if (lane == 0) {
        sm.m[warp * 2 * MT + j] = m[j];
        sm.l[warp * 2 * MT + j] = l[j];
      }
    }
    __syncthreads();
    const long long g = (long long)s.q0 * a.heads + row0;
    // running sums for the join: slot 1 for the tile this worker begins and leaves, slot 0 for one it comes into
    float* part = a.part + ((long long)worker * 2 + (u0 == 0 ? 1 : 0)) * kRows * kPartRow;
#pragma unroll
    for (int h = 0; h < 2 * MT; ++h) {
      const int rr = (h >> 1) * 16 + (h & 1) * 8 + (lane >> 2);
      if (rr < rows) {
        const float(*x)[4] = acc[h >> 1];
        if (whole) {
          const float lr = sm.l[rr], inv = lr > 0.0f || lr != lr ? 1.0f / lr : 0.0f;
          bf16* o = a.out + (g + rr) * kLat + warp * 64 + (lane & 3) * 2;
#pragma unroll
          for (int n = 0; n < 8; ++n)
            *reinterpret_cast<__nv_bfloat162*>(o + n * 8) = __floats2bfloat162_rn(x[n][(h & 1) * 2] * inv, x[n][(h & 1) * 2 + 1] * inv);
        } else {
          float* o = part + rr * kPartRow + warp * 64 + (lane & 3) * 2;
#pragma unroll
          for (int n = 0; n < 8; ++n) *reinterpret_cast<float2*>(o + n * 8) = make_float2(x[n][(h & 1) * 2], x[n][(h & 1) * 2 + 1]);
        }
      }
    }
    if (tid < rows) {
      if (whole) {
        a.lse[g + tid] = (sm.m[tid] + log2f(sm.l[tid])) * 0.69314718055994531f;
      } else {
        part[tid * kPartRow + kLat] = sm.m[tid];
        part[tid * kPartRow + kLat + 1] = sm.l[tid];
      }
    }
    if (!whole && u0 == 0 && tid == 0) {   // the workers of this tile: up to the one that holds its last unit
      int last = worker;
      while (sh.total * (last + 1) / sh.workers < at + units) ++last;
      a.meta[worker * 4] = b;
      a.meta[worker * 4 + 1] = t;
      a.meta[worker * 4 + 2] = last - worker + 1;
    }
    at += units;
    ++t;
  }
}

// ---------------------------------------------------------------------------------------------
// Join of a split tile: out = sum_w 2^(m_w - m) O_w / sum_w 2^(m_w - m) l_w over the tile's workers in order. grid.x is
// the worker that begins the tile, grid.y deals out its rows. Bound by the pieces' bytes in flight: a warp takes a row
// of few pieces (16 dims a lane, four pieces at a time), the eight warps of a CTA share a row of many.
constexpr int kJoinThreads = 256, kJoinFew = 8;

// sums of pieces w0 .. w1 - 1 of a row, weighted; dims 4 lane + 128 j .. + 3 in sum[j]
KK3_DEV void join_pieces(const float* first, const float* rest, long long pitch, int w0, int w1, float ref, float4 (&sum)[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int w = w0; w < w1; ++w) {
    const float* p = w == 0 ? first : rest + (w - 1) * pitch;
    const float f = exp2f(p[kLat] - ref);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 v = *reinterpret_cast<const float4*>(p + j * 128 + lane * 4);
      sum[j].x = fmaf(f, v.x, sum[j].x);
      sum[j].y = fmaf(f, v.y, sum[j].y);
      sum[j].z = fmaf(f, v.z, sum[j].z);
      sum[j].w = fmaf(f, v.w, sum[j].w);
    }
  }
}

__global__ void __launch_bounds__(kJoinThreads) kk3_cache_join_kernel(const AttendArgs a, int tile_rows) {
  __shared__ float4 shared_sum[kJoinThreads / 32][4][32];
  const int worker = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kJoinThreads / 32;
  cache_follow();
  const int n = a.meta[worker * 4 + 2];
  if (n == 0) return;
  const int b = a.meta[worker * 4], t = a.meta[worker * 4 + 1];
  const Seq s = a.seq(b);
  const int rows = (int)min((long long)tile_rows, (long long)s.n * a.heads - (long long)t * tile_rows);
  const bool few = n <= kJoinFew;
  const long long pitch = 2ll * tile_rows * kPartRow;   // from one worker's piece to the next one's
  for (int row = few ? blockIdx.y * kWarps + warp : blockIdx.y; row < rows; row += gridDim.y * (few ? kWarps : 1)) {
    // the piece of the worker that begins the tile, and those of the workers that it continues into
    const float* first = a.part + (worker * 2ll + 1) * tile_rows * kPartRow + (long long)row * kPartRow;
    const float* rest = a.part + (worker + 1) * pitch + (long long)row * kPartRow;
    const auto piece = [&](int w) { return w == 0 ? first : rest + (w - 1) * pitch; };
    float top = -INFINITY;
    for (int w = lane; w < n; w += 32) top = fmaxf(top, piece(w)[kLat]);
    top = warp_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float l = 0.0f;
    for (int w = lane; w < n; w += 32) l += exp2f(piece(w)[kLat] - ref) * piece(w)[kLat + 1];
    l = warp_sum(l);
    float4 sum[4];
    if (few) {
      join_pieces(first, rest, pitch, 0, n, ref, sum);
    } else {
      const int per = (n + kWarps - 1) / kWarps;
      join_pieces(first, rest, pitch, min(n, warp * per), min(n, (warp + 1) * per), ref, sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) shared_sum[warp][j][lane] = sum[j];
      __syncthreads();
      if (warp < 4) {   // warp j adds up dims 128 j .. 128 j + 127
        sum[0] = shared_sum[0][warp][lane];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
          const float4 v = shared_sum[w][warp][lane];
          sum[0].x += v.x;
          sum[0].y += v.y;
          sum[0].z += v.z;
          sum[0].w += v.w;
        }
      }
      __syncthreads();
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const long long g = (long long)s.q0 * a.heads + (long long)t * tile_rows + row;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!few && (j > 0 || warp >= 4)) break;
      __nv_bfloat162 o[2] = {__floats2bfloat162_rn(sum[j].x * inv, sum[j].y * inv), __floats2bfloat162_rn(sum[j].z * inv, sum[j].w * inv)};
      *reinterpret_cast<uint2*>(a.out + g * kLat + (few ? j : warp) * 128 + lane * 4) = *reinterpret_cast<const uint2*>(o);
    }
    if (lane == 0 && (few || warp == 0)) a.lse[g] = (ref + log2f(l)) * 0.69314718055994531f;
  }
}

// ---------------------------------------------------------------------------------------------
// Eviction, selection: one CTA per sequence. The positions are ordered by (protected, weight, lowest index); the
// weights' bits are mapped to unsigned keys of the same order, the key of the last kept position is found digit by
// digit (four histograms of 8 bits), and one pass in ascending position writes the kept ones.

struct EvictArgs {
  CachePages c;
  const long long* lengths;
  const float* mass;
  long long mass_row;
  int budget, sinks, recent;
  const int* dst;          // destination table, or null: in place
  long long dst_row;
  long long* new_lengths;
  float* new_mass;         // [batch, columns * page_size]
  int* kept;               // [batch, budget]
};

constexpr int kEvThreads = 1024;

// unsigned key in the order of the floats; every NaN above +infinity, -0 equal to 0
KK3_DEV unsigned mass_key(float v) {
  if (v != v) return 0xffffffffu;
  const unsigned u = __float_as_uint(v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kEvThreads) kk3_cache_select_kernel(const EvictArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ int hist[256];
  __shared__ int tell[2];
  __shared__ int sums[32], ties[32];
  const long long cap = (long long)a.c.columns * a.c.page_size;
  long long len64 = a.lengths[b];
  if (len64 < 0 || len64 > cap) {
    if (tid == 0) cache_error(a.c);
    len64 = len64 < 0 ? 0 : cap;
  }
  const int len = (int)len64;
  const int keep = min(len, a.budget);
  const float* mass = a.mass + (long long)b * a.mass_row;
  float* out = a.new_mass + (long long)b * cap;
  int* kept = a.kept + (long long)b * a.budget;
  const int sinks = min(a.sinks, len), tail = max(sinks, len - a.recent);   // free positions: [sinks, tail)
  unsigned border = 0;   // key of the last kept free position
  int want = keep - (sinks + len - tail);   // free positions to keep; at the end: those of the border's key
  const bool all = keep == len;
  if (!all && want > 0) {
    unsigned prefix = 0, mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int p = sinks + tid; p < tail; p += kEvThreads) {
        const unsigned k = mass_key(mass[p]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (warp == 0) {   // digits from the top: lane l owns 255 - 8 l .. 248 - 8 l
        int c[8], mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine += c[i] = hist[255 - lane * 8 - i];
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += u;
        }
        before -= mine;
        if (before < want && want <= before + mine) {
          int i = 0;
          while (before + c[i] < want) before += c[i++];
          tell[0] = 255 - lane * 8 - i;
          tell[1] = want - before;
        }
      }
      __syncthreads();
      prefix |= (unsigned)tell[0] << shift;
      mask |= 255u << shift;
      want = tell[1];
      __syncthreads();
    }
    border = prefix;
  }
  // ascending pass: thread t owns a run of positions
  const int run = (len + kEvThreads - 1) / kEvThreads, p0 = min(len, tid * run), p1 = min(len, p0 + run);
  const auto state = [&](int p) -> int {   // 0 dropped, 1 kept, 2 kept if among the first `want` of the border's key
    if (all || p < sinks || p >= tail) return 1;
    if (want <= 0) return 0;
    const unsigned k = mass_key(mass[p]);
    return k > border ? 1 : k == border ? 2 : 0;
  };
  int sure = 0, tie = 0;
  for (int p = p0; p < p1; ++p) {
    const int v = state(p);
    sure += v == 1;
    tie += v == 2;
  }
  int x = sure, y = tie;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) {
      x += u;
      y += v;
    }
  }
  if (lane == 31) {
    sums[warp] = x;
    ties[warp] = y;
  }
  __syncthreads();
  x -= sure;
  y -= tie;
  for (int w = 0; w < warp; ++w) {
    x += sums[w];
    y += ties[w];
  }
  // x certain ones and y ties lie before this run; a tie is kept while fewer than `want` came before it
  int j = x + min(y, max(want, 0));
  for (int p = p0; p < p1; ++p) {
    const int v = state(p);
    if (v == 1 || (v == 2 && y < want)) {
      kept[j] = p;
      out[j] = mass[p];
      ++j;
    }
    y += v == 2;
  }
  for (int i = keep + tid; i < a.budget; i += kEvThreads) kept[i] = -1;
  for (long long i = keep + tid; i < cap; i += kEvThreads) out[i] = 0.0f;
  if (tid == 0) a.new_lengths[b] = keep;
}

// Eviction, move into pages of their own: one warp per kept entry (1152 bytes), bound by the traffic.
constexpr int kMoveWarps = 8;
__global__ void __launch_bounds__(kMoveWarps * 32) kk3_cache_move_kernel(const EvictArgs a) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int j = blockIdx.x * kMoveWarps + (threadIdx.x >> 5);
  if (j >= a.budget) return;
  cache_follow();
  const int from = a.kept[(long long)b * a.budget + j];
  if (from < 0) return;
  CachePages d = a.c;
  d.table = a.dst;
  d.table_stride = a.dst_row;
  int slot, to_slot;
  const int page = page_at(a.c, b, from, &slot), to = page_at(d, b, j, &to_slot);
  if (page < 0 || to < 0) return;
  const bf16* kv = a.c.kv + (long long)page * a.c.kv_page + (long long)slot * a.c.kv_row + lane * 8;
  const bf16* pe = a.c.pe + (long long)page * a.c.pe_page + (long long)slot * a.c.pe_row + lane * 8;
  const uint4 v0 = ldg_stream16(kv), v1 = ldg_stream16(kv + 256);
  uint4 v2 = {};
  if (lane < 8) v2 = ldg_stream16(pe);
  bf16* okv = a.c.kv + (long long)to * a.c.kv_page + (long long)to_slot * a.c.kv_row + lane * 8;
  *reinterpret_cast<uint4*>(okv) = v0;
  *reinterpret_cast<uint4*>(okv + 256) = v1;
  if (lane < 8)
    *reinterpret_cast<uint4*>(a.c.pe + (long long)to * a.c.pe_page + (long long)to_slot * a.c.pe_row + lane * 8) = v2;
}

// Eviction, move in place: entry kept[j] >= j goes to slot j, so batches in ascending j are safe when a batch is read
// whole before it is written: later batches read slots at or above their own j, which earlier ones did not write.
// The order holds per (sequence, 64-byte slice of the entry); the 18 slices of a sequence run side by side.
constexpr int kSlideThreads = 512;
constexpr int kSlideDeep = 8;    // rows in flight per thread: 1024 rows a batch
__global__ void __launch_bounds__(kSlideThreads) kk3_cache_slide_kernel(const EvictArgs a) {
  const int b = blockIdx.y, ch = blockIdx.x * 4 + (threadIdx.x & 3);   // 16-byte piece of the entry: 0 .. 71
  cache_follow();
  const int keep = (int)a.new_lengths[b];
  const int* kept = a.kept + (long long)b * a.budget;
  constexpr int kRows = kSlideThreads / 4;
  const auto where = [&](int pos) -> bf16* {
    int slot;
    const int page = page_at(a.c, b, pos, &slot);
    if (page < 0) return nullptr;
    return ch < kLat / 8 ? a.c.kv + (long long)page * a.c.kv_page + (long long)slot * a.c.kv_row + ch * 8
                         : a.c.pe + (long long)page * a.c.pe_page + (long long)slot * a.c.pe_row + (ch - kLat / 8) * 8;
  };
  for (int j0 = 0; j0 < keep; j0 += kRows * kSlideDeep) {
    uint4 v[kSlideDeep];
    bool move[kSlideDeep];
#pragma unroll
    for (int i = 0; i < kSlideDeep; ++i) {
      const int j = j0 + i * kRows + (threadIdx.x >> 2);
      move[i] = false;
      if (j < keep) {
        const int from = kept[j];
        const bf16* src = from != j ? where(from) : nullptr;
        if (src) {
          v[i] = *reinterpret_cast<const uint4*>(src);
          move[i] = true;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSlideDeep; ++i) {
      if (move[i]) {
        bf16* dst = where(j0 + i * kRows + (threadIdx.x >> 2));
        if (dst) *reinterpret_cast<uint4*>(dst) = v[i];
      }
    }
    __syncthreads();
  }
}

}  // namespace kk3

// ---------------------------------------------------------------------------------------------
// C entry points

using namespace kk3;

namespace kk3 {



int cache_cuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return KK3_OK;
  fprintf(stderr, "kk3: %s: %s\n", what, cudaGetErrorString(e));
  (void)cudaGetLastError();
  return KK3_ERR_CUDA;
}

int cache_pages(const kk3_cache* c, CachePages* out, int* error_word) {
  if (!c || !cache_aligned(c->kv, 16) || !cache_aligned(c->pe, 16) || !cache_aligned(c->table, 4)) return KK3_ERR_ARG;
  if (c->batch < 1 || c->columns < 1 || c->page_size < 1 || c->num_pages < 1 || c->table_stride < 0) return KK3_ERR_ARG;
  if (c->kv_row_stride < kLat || c->pe_row_stride < kRope || c->kv_page_stride < 0 || c->pe_page_stride < 0 ||
      c->kv_row_stride % 8 || c->pe_row_stride % 8 || c->kv_page_stride % 8 || c->pe_page_stride % 8)
    return KK3_ERR_ARG;
  if (c->batch > kMaxSeqs || c->page_size > 65536 || (long long)c->columns * c->page_size > (1ll << 27))
    return KK3_ERR_UNSUPPORTED;
  out->kv = (bf16*)c->kv;
  out->pe = (bf16*)c->pe;
  out->kv_page = c->kv_page_stride;
  out->kv_row = c->kv_row_stride;
  out->pe_page = c->pe_page_stride;
  out->pe_row = c->pe_row_stride;
  out->table = c->table;
  out->table_stride = c->table_stride;
  out->num_pages = c->num_pages;
  out->page_size = c->page_size;
  out->columns = c->columns;
  out->batch = c->batch;
  out->page_magic = c->page_size > 1 ? (unsigned)((1ull << 32) / (unsigned)c->page_size + 1) : 0;
  out->error_word = error_word;
  return KK3_OK;
}

int cache_sms(int* sms) {
  static std::atomic<int> known[kCacheMaxDevices];
  int dev = 0;
  int rc = cache_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  if (dev < kCacheMaxDevices && (*sms = known[dev].load(std::memory_order_relaxed)) > 0) return KK3_OK;
  rc = cache_cuda(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
  if (rc == KK3_OK && dev < kCacheMaxDevices) known[dev].store(*sms, std::memory_order_relaxed);
  return rc;
}

}  // namespace kk3

extern "C" int kk3_cache_append(const kk3_cache_append_args* x, void* stream) {
  if (!x) return KK3_ERR_ARG;
  AppendArgs a;
  const int rc = cache_pages(&x->cache, &a.c, x->error_word);
  if (rc) return rc;
  if (x->tokens < 0 || (x->tokens > 0 && !cache_aligned(x->raw, 16)) || x->raw_stride % 8 || x->raw_stride < kEntry ||
      !cache_aligned(x->norm_weight, 16) || !cache_aligned(x->lengths, 8) || !cache_aligned(x->cu_new, 4) ||
      !cache_aligned(x->new_lengths, 8) || x->lengths == x->new_lengths || !(x->eps >= 0.0f))
    return KK3_ERR_ARG;
  a.raw = (const bf16*)x->raw;
  a.raw_row = x->raw_stride;
  a.weight = (const bf16*)x->norm_weight;
  a.lengths = (const long long*)x->lengths;
  a.new_lengths = (long long*)x->new_lengths;
  a.cu_new = x->cu_new;
  a.tokens = x->tokens;
  a.eps = x->eps;
  const int grid = x->tokens > 0 ? (x->tokens + kAppendWarps - 1) / kAppendWarps : 1;
  kk3_cache_append_kernel<<<grid, kAppendWarps * 32, 0, (cudaStream_t)stream>>>(a);
  return cache_cuda(cudaGetLastError(), "kk3_cache_append_kernel");
}

// The kernel for a call's average rows per sequence, and its workers: the warp-level ones up to 16 and 32 rows, CTA pairs
// above.
struct Plan {
  int workers, rows;
};
static Plan attend_plan(int64_t batch, int64_t tokens, int64_t heads, int sms) {
  const int64_t total = tokens * heads;
  if (total <= 16 * batch) return Plan{sms, 16};
  if (total <= 32 * batch) return Plan{sms, 32};
  return Plan{sms / 2, kPairRows};
}
template <int MT>
static int attend_warp(const AttendArgs& a, cudaStream_t st) {
  static std::atomic<bool> done[kCacheMaxDevices];
  const int r = cache_allow_smem(kk3_cache_attend_warp_kernel<MT>, sizeof(WaSmem<MT>), done,
                                 "cudaFuncSetAttribute(kk3_cache_attend_warp_kernel)");
  if (r) return r;
  kk3_cache_attend_warp_kernel<MT><<<a.workers, kWaThreads, sizeof(WaSmem<MT>), st>>>(a);
  return cache_cuda(cudaGetLastError(), "kk3_cache_attend_warp_kernel");
}

extern "C" int64_t kk3_cache_attend_workspace(void) {
  int sms = 0;
  if (cache_sms(&sms)) return 0;
  const int64_t pair = (int64_t)(sms / 2) * (16 + 2 * kPairRows * kPartRow * 4), warp = (int64_t)sms * (16 + 2 * 32 * kPartRow * 4);
  return pair > warp ? pair : warp;
}

extern "C" int kk3_cache_attend(const kk3_cache_attend_args* x, void* stream) {
  if (!x) return KK3_ERR_ARG;
  AttendArgs a;
  const int rc = cache_pages(&x->cache, &a.c, x->error_word);
  if (rc) return rc;
  const int tokens = x->tokens, heads = x->heads;
  if (tokens < 0 || heads < 1 || !cache_aligned(x->lengths, 8) || !cache_aligned(x->cu_new, 4) || !(x->scale == x->scale))
    return KK3_ERR_ARG;
  if (heads > kMaxHeads || (int64_t)tokens * heads > INT32_MAX / 2) return KK3_ERR_UNSUPPORTED;
  if (tokens == 0) return KK3_OK;
  if (!cache_queries(x->q_latent, x->ql_token, x->ql_head, x->q_pe, x->qp_token, x->qp_head) || !cache_aligned(x->out, 16) ||
      !cache_aligned(x->lse, 4))
    return KK3_ERR_ARG;
  int sms = 0;
  if (cache_sms(&sms)) return KK3_ERR_CUDA;
  if (!cache_aligned(x->workspace, 16) || x->workspace_bytes < kk3_cache_attend_workspace()) return KK3_ERR_ARG;
  a.q_lat = (const bf16*)x->q_latent;
  a.q_pe = (const bf16*)x->q_pe;
  a.ql_tok = x->ql_token;
  a.ql_head = x->ql_head;
  a.qp_tok = x->qp_token;
  a.qp_head = x->qp_head;
  a.lengths = (const long long*)x->lengths;
  a.cu_new = x->cu_new;
  a.tokens = tokens;
  a.heads = heads;
  a.scale_log2 = x->scale * 1.4426950408889634f;
  a.out = (bf16*)x->out;
  a.lse = x->lse;
  const Plan p = attend_plan(a.c.batch, tokens, heads, sms);
  a.workers = p.workers;
  a.meta = (int*)x->workspace;
  a.part = (float*)((char*)x->workspace + (size_t)p.workers * 16);
  const cudaStream_t st = (cudaStream_t)stream;
  const int r = p.rows == 16 ? attend_warp<1>(a, st) : p.rows == 32 ? attend_warp<2>(a, st) : attend_pair(&x->cache, a, st);
  if (r) return r;
  return cache_launch_after(kk3_cache_join_kernel, dim3(p.workers, 16), kJoinThreads, st, "kk3_cache_join_kernel", a, p.rows);
}

extern "C" int kk3_cache_evict(const kk3_cache_evict_args* x, void* stream) {
  if (!x) return KK3_ERR_ARG;
  EvictArgs a;
  const int rc = cache_pages(&x->cache, &a.c, x->error_word);
  if (rc) return rc;
  const int budget = x->budget;
  if (!cache_aligned(x->lengths, 8) || !cache_aligned(x->mass, 4) || x->mass_stride < 0 || budget < 1 || x->sinks < 0 ||
      x->recent < 0 || (int64_t)x->sinks + x->recent > budget || !cache_aligned(x->new_lengths, 8) ||
      !cache_aligned(x->new_mass, 4) || !cache_aligned(x->kept, 4) || x->lengths == x->new_lengths || x->mass == x->new_mass)
    return KK3_ERR_ARG;
  const int64_t cap = (int64_t)x->cache.columns * x->cache.page_size;
  if (budget > cap) return KK3_ERR_ARG;
  if (x->dst_table && (((uintptr_t)x->dst_table % 4) || x->dst_stride < 0 || (int64_t)x->dst_columns * x->cache.page_size < budget))
    return KK3_ERR_ARG;
  a.lengths = (const long long*)x->lengths;
  a.mass = x->mass;
  a.mass_row = x->mass_stride;
  a.budget = budget;
  a.sinks = x->sinks;
  a.recent = x->recent;
  a.dst = x->dst_table;
  a.dst_row = x->dst_stride;
  a.new_lengths = (long long*)x->new_lengths;
  a.new_mass = x->new_mass;
  a.kept = x->kept;
  const cudaStream_t st = (cudaStream_t)stream;
  kk3_cache_select_kernel<<<a.c.batch, kEvThreads, 0, st>>>(a);
  int r = cache_cuda(cudaGetLastError(), "kk3_cache_select_kernel");
  if (r) return r;
  if (x->dst_table)
    return cache_launch_after(kk3_cache_move_kernel, dim3((budget + kMoveWarps - 1) / kMoveWarps, a.c.batch),
                              kMoveWarps * 32, st, "kk3_cache_move_kernel", a);
  return cache_launch_after(kk3_cache_slide_kernel, dim3(kEntry / 32, a.c.batch), kSlideThreads, st,
                            "kk3_cache_slide_kernel", a);
}
