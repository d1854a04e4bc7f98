// kk3_cache.cu - kernels and C entry points of the paged latent cache (include/kk3.h, kk3_cache_*): append, the
// join of split attention tiles, eviction.
#include <cuda_runtime.h>

#include "kk3_cache.cuh"
#include "kk3_cache_host.h"

namespace kk3 {

// ---------------------------------------------------------------------------------------------
// append: latent = x[:512] / rms(x[:512]) * weight, rope = x[512:], into the page of the token's position. In FP32, rounded
// to BF16 once, or (STEP) as the decode step and the model round it: to BF16 before the product with the weight, and
// after it (kimi.py:265-270, common.py:13-21), so that the entry is the one that the step would have cached. One warp per
// token, bound by its 2304 bytes of traffic; 16-byte accesses throughout (lane l owns the latent values 8 l .. 8 l + 7 and
// 256 + 8 l ..; eight lanes copy the rope part). Five chunks of up to 4096 tokens take 6.8 us, 5.5 TB/s (STEP 7.2); eight
// single tokens 2.4 us, a launch.

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

template <bool STEP>
__global__ void __launch_bounds__(kAppendWarps * 32) kk3_cache_append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int tok = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  const int B = a.c.batch;
  const long long cap = (long long)a.c.columns * a.c.page_size;
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
      const int q0 = min(max(a.cu_new[b], 0), a.tokens), q1 = min(max(a.cu_new[b + 1], q0), a.tokens);
      const long long l = a.lengths[b], sum = min(max(l, 0ll), cap) + (q1 - q0);
      if (l < 0 || l > cap || sum > cap) cache_error(a.c);
      a.new_lengths[b] = min(sum, cap);
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
  const long long held = a.lengths[lo], pos = min(held, cap) + (tok - first);
  if (held < 0 || pos >= cap) return;   // no place that the sequence could mean
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
      float2 f = __bfloat1622float2(p[i]);
      const float2 g = __bfloat1622float2(q[i]);
      f = make_float2(f.x * r, f.y * r);
      if (STEP) f = make_float2(round_bf(f.x), round_bf(f.y));
      p[i] = __floats2bfloat162_rn(f.x * g.x, f.y * g.y);
    }
    *reinterpret_cast<uint4*>(kv + h * 256 + lane * 8) = v[h];
  }
  if (lane < 8)
    *reinterpret_cast<uint4*>(a.c.pe + (long long)page * a.c.pe_page + (long long)slot * a.c.pe_row + lane * 8) = rope;
}

// ---------------------------------------------------------------------------------------------
// Join of split tiles: out = sum_w 2^(m_w - m) O_w / sum_w 2^(m_w - m) l_w over a tile's workers in order. Bound by the
// pieces' bytes in flight: a warp takes a row of few pieces (16 dims a lane, four pieces at a time), the eight warps of
// a CTA share a row of many. Every CTA finds the cut tiles among the workers' notes and takes its share of their rows,
// so that the grid fits the GPU at once (16 CTAs for each worker, most with nothing to do, began 2.7 us later).
constexpr int kJoinThreads = 256, kJoinFew = 8, kJoinPerSm = 3;
static_assert(kMaxWorkers <= kJoinThreads, "a thread looks at a worker");

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

__global__ void __launch_bounds__(kJoinThreads, kJoinPerSm) kk3_cache_join_kernel(const AttendArgs a, int tile_rows) {
  __shared__ float4 shared_sum[kJoinThreads / 32][4][32];
  __shared__ int4 cut[kMaxWorkers];    // a worker's tile: first row among all, rows, pieces, items before it
  __shared__ int sums[kJoinThreads / 32];
  constexpr int kWarps = kJoinThreads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cache_follow();
  // an item: a row of many pieces, or eight rows of few
  int4 mine = tid < a.workers ? reinterpret_cast<const int4*>(a.meta)[tid] : make_int4(0, 0, 0, 0);
  const int items = mine.z == 0 ? 0 : mine.z <= kJoinFew ? (mine.y + kWarps - 1) / kWarps : mine.y;
  int before = items;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += u;
  }
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  mine.w = before - items;
  if (tid < a.workers) cut[tid] = mine;
  __syncthreads();
  for (int item = blockIdx.x; item < total; item += gridDim.x) {
    int worker = 0;   // the last one whose items begin at or before this one: those without any lie before it
    for (int hi = a.workers; hi - worker > 1;) {
      const int mid = (worker + hi) >> 1;
      if (cut[mid].w <= item) worker = mid; else hi = mid;
    }
    const int g0 = cut[worker].x, rows = cut[worker].y, n = cut[worker].z;
    const bool few = n <= kJoinFew;
    const int row = few ? (item - cut[worker].w) * kWarps + warp : item - cut[worker].w;
    const long long pitch = 2ll * tile_rows * kPartRow;   // from one worker's piece to the next one's
    if (row >= rows) continue;   // some warps' rows of few pieces
    // the piece of the worker that begins the tile, and those of the workers that it continues into
    const float* first = a.part + (worker * 2ll + 1) * tile_rows * kPartRow + (long long)row * kPartRow;
    const float* rest = a.part + (worker + 1) * pitch + (long long)row * kPartRow;
    float2 ml[kMaxWorkers / 32];   // maximum and sum of pieces lane, lane + 32, ..
    float top = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxWorkers / 32; ++i) {
      const int w = lane + 32 * i;
      ml[i] = w < n ? *reinterpret_cast<const float2*>((w == 0 ? first : rest + (w - 1) * pitch) + kLat) : make_float2(-INFINITY, 0.0f);
      top = fmaxf(top, ml[i].x);
    }
    top = warp_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < kMaxWorkers / 32; ++i) l += exp2f(ml[i].x - ref) * ml[i].y;
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
    const long long g = g0 + row;
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
// digit (four histograms of 8 bits), and one pass in ascending position writes the kept ones. Bound by latency: the keys
// of up to kEvHeld positions are read once and stay in shared memory, the search ends with the first digit whose
// positions all stay, and in the last pass a warp takes 32 neighbours at a time. A pass over 8192 positions takes 1.4 us,
// most of it the instructions of one SM. (Adding a warp's equal digits up by match before they are counted took 0.9 us
// more a pass than the plain atomics, and four positions of a thread at a time nothing less.)

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
constexpr int kEvHeld = 32768;

// unsigned key in the order of the floats; every NaN above +infinity, -0 equal to 0
KK3_DEV unsigned mass_key(float v) {
  if (v != v) return 0xffffffffu;
  const unsigned u = __float_as_uint(v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kEvThreads) kk3_cache_select_kernel(const EvictArgs a) {
  extern __shared__ unsigned held_keys[];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ int hist[4][256];
  __shared__ int tell[4][2];
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
  const int sinks = min(a.sinks, keep), tail = max(sinks, len - a.recent);   // free positions: [sinks, tail)
  unsigned border = 0xffffffffu;   // what stays lies above
  int want = keep - (sinks + len - tail);   // free positions to keep; at the end: those at the border
  const int end = len + min(want, 0);   // of the protected positions that stay: the lowest ones where not all can
  want = max(want, 0);
  const bool all = keep == len, held = len <= kEvHeld;
  const auto key = [&](int p) { return held ? held_keys[p] : mass_key(mass[p]); };
  if (!all && want > 0) {
    if (held) {
#pragma unroll 8
      for (int p = tid; p < len; p += kEvThreads) held_keys[p] = mass_key(mass[p]);
    }
    hist[tid >> 8][tid & 255] = 0;
    __syncthreads();
    unsigned prefix = 0, mask = 0;
#pragma unroll 1
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
      for (int p = sinks + tid; p < tail; p += kEvThreads) {
        const unsigned k = key(p);
        if ((k & mask) == prefix) atomicAdd(&hist[pass][(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (warp == 0) {   // digits from the top: lane l owns 255 - 8 l .. 248 - 8 l
        int c[8], mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine += c[i] = hist[pass][255 - lane * 8 - i];
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += u;
        }
        before -= mine;
        if (before < want && want <= before + mine) {
          int digit = -1;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (digit < 0 && want <= before + c[i]) {
              digit = 255 - lane * 8 - i;
              tell[pass][0] = digit;
              tell[pass][1] = want - before;
            }
            before += c[i];
          }
        }
      }
      __syncthreads();
      prefix |= (unsigned)tell[pass][0] << shift;
      mask |= 255u << shift;
      want = tell[pass][1];
      if (want == hist[pass][tell[pass][0]]) {   // all of these stay, no ties: some free position is dropped, so prefix > 0
        --prefix;
        want = 0;
        break;
      }
    }
    border = prefix;
  }
  // ascending pass: a warp owns a run of positions
  const int run = (len + kEvThreads - 1) / kEvThreads * 32, w0 = min(len, warp * run), w1 = min(len, w0 + run);
  const bool keyed = border != 0xffffffffu || want > 0;   // else no free position stays, or all do
  const auto state = [&](int p) -> int {   // 0 dropped, 1 kept, 2 kept if among the first `want` at the border
    if (p >= w1) return 0;
    if (all || p < sinks) return 1;
    if (p >= tail) return p < end;
    if (!keyed) return 0;
    const unsigned k = key(p);
    return k > border ? 1 : k == border && want > 0 ? 2 : 0;
  };
  int sure = 0, tie = 0;
  for (int p = w0; p < w1; p += 32) {
    const int v = state(p + lane);
    sure += __popc(__ballot_sync(0xffffffffu, v == 1));
    tie += __popc(__ballot_sync(0xffffffffu, v == 2));
  }
  if (lane == 0) {
    sums[warp] = sure;
    ties[warp] = tie;
  }
  __syncthreads();
  // x certain ones and y ties lie before; a tie is kept while fewer than `want` came before it
  int x = lane < warp ? sums[lane] : 0, y = lane < warp ? ties[lane] : 0;
  x = __reduce_add_sync(0xffffffffu, x);
  y = __reduce_add_sync(0xffffffffu, y);
  const unsigned lower = (1u << lane) - 1;
  for (int p0 = w0; p0 < w1; p0 += 32) {
    const int p = p0 + lane, v = state(p);
    const float weight = p < w1 ? mass[p] : 0.0f;
    const unsigned certain = __ballot_sync(0xffffffffu, v == 1), tied = __ballot_sync(0xffffffffu, v == 2);
    const int ties_before = y + __popc(tied & lower);
    if (v == 1 || (v == 2 && ties_before < want)) {
      const int j = x + __popc(certain & lower) + min(ties_before, want);
      kept[j] = p;
      out[j] = weight;
    }
    x += __popc(certain);
    y += __popc(tied);
  }
  for (int i = keep + tid; i < a.budget; i += kEvThreads) kept[i] = -1;
  for (long long i = keep + tid; i < cap; i += kEvThreads) out[i] = 0.0f;
  if (tid == 0) a.new_lengths[b] = keep;
}

// Eviction, move into pages of their own: one warp per kept entry (1152 bytes), bound by the traffic: 65000 entries 23 us,
// 6.5 TB/s.
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
// The order holds per (sequence, 64-byte slice of the entry); the 18 slices of a sequence run side by side, bound by the
// batches' latencies: 16 sequences of up to 8192 positions cut down to 4096 take 46 us in place, 38 into other pages.
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

template <bool STEP>
static int cache_append(const kk3_cache_append_args* x, void* stream) {
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
  kk3_cache_append_kernel<STEP><<<grid, kAppendWarps * 32, 0, (cudaStream_t)stream>>>(a);
  return cache_cuda(cudaGetLastError(), "kk3_cache_append_kernel");
}

extern "C" int kk3_cache_append(const kk3_cache_append_args* x, void* stream) { return cache_append<false>(x, stream); }
extern "C" int kk3_cache_append_step(const kk3_cache_append_args* x, void* stream) { return cache_append<true>(x, stream); }

// The kernel and its workers. Up to 16 rows a sequence on average fill the small tile: 64 sequences of 8192 positions
// with 12 rows each take 123 us in it and 187 us in CTA pairs; with 24 rows, two small tiles that read the cache twice,
// 243 and 195 us. A small call is faster in the small tile whatever its rows, since that begins and ends sooner: 48 rows
// of one sequence take 20.5 against 24.0 us over 517 positions and 24.0 against 26.0 over 8192, 96 rows 27.4 against 26.7.
// The host does not know the lengths, only what the table can hold.
struct Plan {
  int workers, rows;
};
static Plan attend_plan(int64_t batch, int64_t tokens, int64_t heads, int64_t capacity, int sms) {
  const int workers = sms < kMaxWorkers ? sms : kMaxWorkers;
  const int64_t rows = tokens * heads;
  return rows <= kFewRows * batch || (rows <= 4 * kFewRows && capacity <= 8192) ? Plan{workers, kFewRows} : Plan{workers / 2, kPairRows};
}

extern "C" int64_t kk3_cache_attend_workspace(void) {
  int sms = 0;
  if (cache_sms(&sms)) return 0;
  const int64_t pair = (int64_t)(sms / 2) * (16 + 2 * kPairRows * kPartRow * 4), few = (int64_t)sms * (16 + 2 * kFewRows * kPartRow * 4);
  return pair > few ? pair : few;
}

extern "C" int kk3_cache_attend(const kk3_cache_attend_args* x, void* stream) {
  if (!x) return KK3_ERR_ARG;
  AttendArgs a;
  const int rc = cache_pages(&x->cache, &a.c, x->error_word);
  if (rc) return rc;
  const int tokens = x->tokens, heads = x->heads;
  if (tokens < 0 || heads < 1 || !cache_aligned(x->lengths, 8) || !cache_aligned(x->cu_new, 4) || !cache_scale(x->scale))
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
  const Plan p = attend_plan(a.c.batch, tokens, heads, (int64_t)a.c.columns * a.c.page_size, sms);
  a.workers = p.workers;
  a.meta = (int*)x->workspace;
  a.part = (float*)((char*)x->workspace + (size_t)p.workers * 16);
  const cudaStream_t st = (cudaStream_t)stream;
  const int r = p.rows == kFewRows ? attend_few(&x->cache, a, st) : attend_pair(&x->cache, a, st);
  if (r) return r;
  return cache_launch_after(kk3_cache_join_kernel, dim3(kJoinPerSm * sms), kJoinThreads, st, "kk3_cache_join_kernel", a, p.rows);
}

extern "C" int kk3_cache_evict(const kk3_cache_evict_args* x, void* stream) {
  if (!x) return KK3_ERR_ARG;
  EvictArgs a;
  const int rc = cache_pages(&x->cache, &a.c, x->error_word);
  if (rc) return rc;
  const int budget = x->budget;
  if (!cache_aligned(x->lengths, 8) || !cache_aligned(x->mass, 4) || x->mass_stride < 0 || budget < 1 || x->sinks < 0 ||
      x->recent < 0 || !cache_aligned(x->new_lengths, 8) ||
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
  static std::atomic<bool> ready[kCacheMaxDevices];
  int r = cache_allow_smem(kk3_cache_select_kernel, kEvHeld * 4, ready, "cudaFuncSetAttribute(kk3_cache_select_kernel)");
  if (r) return r;
  kk3_cache_select_kernel<<<a.c.batch, kEvThreads, (cap < kEvHeld ? cap : kEvHeld) * 4, st>>>(a);
  r = cache_cuda(cudaGetLastError(), "kk3_cache_select_kernel");
  if (r) return r;
  if (x->dst_table)
    return cache_launch_after(kk3_cache_move_kernel, dim3((budget + kMoveWarps - 1) / kMoveWarps, a.c.batch),
                              kMoveWarps * 32, st, "kk3_cache_move_kernel", a);
  return cache_launch_after(kk3_cache_slide_kernel, dim3(kEntry / 32, a.c.batch), kSlideThreads, st,
                            "kk3_cache_slide_kernel", a);
}
