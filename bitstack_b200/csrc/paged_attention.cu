// One new token per request over a paged key/value cache: rotary embedding of q and k, k and v written into the request's
// page, softmax(q K^T / sqrt(D)) V over the request's pages.
//
// Bound by reading K and V once (4 flops per byte and head of a group; the floor is their bytes at copy bandwidth).  Measured: 64
// requests of 1 to 8192 positions, 32 / 8 heads of 128: 121 us, 5.9 TB/s (copy 6.55); one request of 131071: 91 us, 5.9 TB/s.  The
// prefix sums take shared memory: from about 310 requests on, heads of 64 keep three CTAs of a multiprocessor instead of
// four (300 requests of 1500, 16 / 4 heads: 5.6 TB/s, 320: 4.6); heads of 128 do not notice (5.7 TB/s on both sides).
//  * Work split: a request's length is cut into tiles of 64 positions; the tiles of all (request, kv head) pairs form one
//    sequence, of which every CTA takes the same number.  Lengths are only known on the device, so every CTA finds its place
//    by a prefix sum over the requests.  A pair that several CTAs share leaves partial results (maximum, sum, unnormalised
//    output), which a second kernel joins in CTA order: no atomics, no state between calls, the same bits every time.
//  * A CTA is four warps (eight: see kManyWarps), and a warp is on its own: it streams its 16 positions of every tile through a ring of its own in
//    shared memory (16-byte cp.async, rows looked up page by page, so a page may end anywhere) and needs no barrier with the
//    others until the pair ends.  Rows behind the last position are filled with zeros, whatever the page holds there.
//  * All query heads of a group share the K and V that were read.  The products are taken transposed, scores^T = K Q^T and
//    output^T = V^T P^T, so that positions and dimensions fill the 16 rows of mma.sync m16n8k16 and the heads its 8 columns: a
//    group of up to 8 heads wastes nothing (half the MMAs, exponentials and accumulators of the untransposed form), one of up
//    to 16 takes two column blocks.  q after its rotation and the weights go in as two values of the type each, the nearest one
//    and what that leaves: twice the MMAs, 1 % of the time (117 -> 118 us, 64 requests).  Beside the output's rounding that leaves
//    2^-22 of a value (bf16 2^-16), below fp16's normal range 2^-25 in q and 2^-38 of the largest weight (see Exponents); single
//    values had twice the error.  Scores and output are accumulated in fp32; one pass keeps the running maximum and sum.
//  * The new position's K and V come from the projection's output: turned, stored to the page and to the ring by the warp
//    that meets the position, so nothing is read back.
#include <climits>
#include <math.h>

#include "common.cuh"
#include "numeric.cuh"

namespace bsb {
namespace {

// Warps of a CTA; a tile is 16 positions of each.  Eight where every pair has a multiprocessor to itself: half the rounds of
// latency of a pair (1 request of 200: 6.6 -> 5.6 us, of 512: 9.4 -> 7.9).
constexpr int kManyWarps = 8;
constexpr int kRows = 16;                // most query heads of one pass
constexpr int kMaxBatch = 2048;          // requests of one launch: their prefix sums stay in shared memory
// What a pair costs a CTA beside its tiles, in tiles (64 ragged requests up to 8192 positions / 128 up to 1500, heads of 64: cost 0
// 143 / 37 us, 1 126 / 29.5, 3 120 / 23.3, 6 120 / 25.4).
constexpr int kPairCost = 3;
// Weights are 2^(score - reference + bias), the reference being a running maximum that may fall behind by 2^slack; bias cancels in
// the division.  fp16 holds weights from 2^-24 on only: without a bias those of a few thousand positions 17 nats below the leading
// one vanished from the product, and not from the sum.  With 2 and 13 the largest weight lies in 2^13 .. 2^15, and what two
// values of the type leave of a weight stays below 2^-38 of it.  bf16 has fp32's exponents.
template <typename T> struct Exponents;
template <> struct Exponents<__half> { static constexpr float slack = 2.f, bias = 13.f; };
template <> struct Exponents<__nv_bfloat16> { static constexpr float slack = 6.f, bias = 0.f; };
// Requests that cannot be longer than this by the width of their table get one CTA per (request, kv head) and no join (short ones
// in a wide table take the shared form: 1 request of 200 8.1 us instead of 5.8, 16 up to 384 with 64 / 8 heads 12.3 instead of
// 7.4).  32 / 8 heads of 128, one CTA per pair
// against equal shares: 1 request of 200 5.6 / 8.0 us, of 512 7.9 / 8.1; 16 requests of 512 7.8 / 10.9; 64 requests of 200 (four warps)
// 11.2 / 15.2; with four warps throughout, 1 request of 1000 14.6 / 8.7, 16 of 1000 14.7 / 12.0.
constexpr int64_t kWholePositions = 512;
// Stages of a warp's ring, CTAs of a multiprocessor (64 ragged requests: 2 x 3 141 us, 3 x 2 147, 4 x 1 183, before the last steps).
template <int D> struct Shape;
template <> struct Shape<128> { static constexpr int stages = 2, ctas = 3; };
template <> struct Shape<64> { static constexpr int stages = 3, ctas = 4; };
constexpr int kMaxCtas = 4;              // per multiprocessor, for the scratch

struct AttnParams {
  const void *q, *k, *v, *cos_t, *sin_t;
  void *k_pages, *v_pages, *out;
  int64_t q_stride, k_stride, v_stride, k_page_stride, v_page_stride, table_len, num_pages, table_stride;
  const int64_t* positions;
  const int32_t* table;
  int64_t most;                          // positions that a table row can hold, at most 2^31 - 64
  int batch, Hq, Hkv, group, chunks, rows_kept, page_size;
  uint32_t page_mul, page_shift;         // p / page_size = (p * page_mul) >> page_shift for p < 2^31
  int whole;                             // one CTA per (request, kv head)
  float scale_log2;
  float* part;                           // [CTA][2]: 16 maxima, 16 sums, rows_kept x D outputs (every part 16-byte aligned)
  int4* plan;                            // [CTA][2]: pairs shared with other CTAs, the one that this CTA continues and the one that begins
                                         // in it: first output row, heads (0: there is none), first and last CTA
  int* status;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool keep) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(keep ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {   // an 8 x 8 block of 16-bit values across the warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const typename Pair<T>::type p = Pair<T>::make(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// a / b, in 32 bits where they do (a 64-bit division is a long chain of instructions)
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
// tokens a request holds after this step; -1: its position is behind its table row or the cos / sin tables
__device__ __forceinline__ int length_of(const AttnParams& P, int b) {
  const int64_t pos = P.positions[b];
  if (pos < 0) return 0;
  return pos < P.most && pos < P.table_len ? (int)pos + 1 : -1;
}
template <int TILE>
__device__ __forceinline__ int tiles_of(int n) { return n <= 0 ? 1 : (n + TILE - 1) / TILE; }   // idle rows too have an output

// four values of the type as fp32; and back, leaving in x what the rounding took
template <typename T>
__device__ __forceinline__ void load4(const T* src, float (&x)[4]) {
  const uint2 raw = *reinterpret_cast<const uint2*>(src);
  const typename Pair<T>::type* p = reinterpret_cast<const typename Pair<T>::type*>(&raw);
  const float2 a = to_f2(p[0]), b = to_f2(p[1]);
  x[0] = a.x;
  x[1] = a.y;
  x[2] = b.x;
  x[3] = b.y;
}
template <typename T>
__device__ __forceinline__ void store4(uint8_t* dst, float (&x)[4]) {
  uint2 raw;
  typename Pair<T>::type* p = reinterpret_cast<typename Pair<T>::type*>(&raw);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    p[i] = Pair<T>::make(x[2 * i], x[2 * i + 1]);
    const float2 f = to_f2(p[i]);
    x[2 * i] -= f.x;
    x[2 * i + 1] -= f.y;
  }
  *reinterpret_cast<uint2*>(dst) = raw;
}

// rotary embedding of eight pairs (i, i + D/2): x*cos + rotate_half(x)*sin with rotate_half(x) = [-x1, x0]
template <typename T, int D>
__device__ __forceinline__ void turn8(const T* src, const T* cos_t, const T* sin_t, float (&x0)[8], float (&x1)[8]) {
  float c0[8], c1[8], s0[8], s1[8];
  load8(src, x0);
  load8(src + D / 2, x1);
  load8(cos_t, c0);
  load8(cos_t + D / 2, c1);
  load8(sin_t, s0);
  load8(sin_t + D / 2, s1);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = x0[e], b = x1[e];
    x0[e] = a * c0[e] - b * s0[e];
    x1[e] = b * c1[e] + a * s1[e];
  }
}

// dynamic shared memory: [warp][stage][K 16 rows, V 16 rows], q [16 rows], maxima and sums [2][warp][16], prefix sums [batch + 1]
template <int D, int W> constexpr int ring_bytes() { return W * Shape<D>::stages * 2 * 16 * D * 2; }
template <int D, int W> constexpr int fixed_bytes() { return ring_bytes<D, W>() + 2 * kRows * D * 2 + 2 * W * kRows * 4; }

// NB: column blocks of 8 heads.  ALIGNED: pages are a multiple of 16 rows, so the 16 positions of a warp lie in one page.
template <typename T, int D, int NB, bool ALIGNED, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps == kManyWarps ? 1 : NB == 1 ? Shape<D>::ctas : 2) paged_attention_kernel(const __grid_constant__ AttnParams P) {
  constexpr int kThreads = kWarps * 32, kTile = 16 * kWarps;
  constexpr int kStages = Shape<D>::stages;
  constexpr int kChunks = D / 8;                 // 16-byte pieces of a row
  constexpr int kStep = 32 / kChunks;            // rows that one warp-wide copy covers
  constexpr int kHalf = 16 * D * 2;              // bytes of the K (or V) rows of a stage
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* s_q = smem + ring_bytes<D, kWarps>();
  float* s_m = reinterpret_cast<float*>(s_q + 2 * kRows * D * 2);
  float* s_l = s_m + kWarps * kRows;
  int64_t* s_before = reinterpret_cast<int64_t*>(s_l + kWarps * kRows);
  __shared__ int64_t s_sum[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pairs = P.Hkv * P.chunks;            // (kv head, chunk of its query heads)
  pdl_wait();   // (the join is let in at the end: its waiting CTAs cost this kernel 10 % when they come early)

  // ---- this CTA's share of the tiles ------------------------------------------------------------------------------
  // The sequence is counted in units: a pair is kPairCost units in front of its tiles.  Short requests then do not pile up in one
  // CTA's share, where each of them would cost a round of latencies for a tile or two.
  int64_t first, end, share = 0;
  int b, pair, u0 = 0;
  const int cost = P.whole ? 0 : kPairCost;
  if (P.whole) {
    b = blockIdx.x / pairs;
    pair = blockIdx.x - b * pairs;
    first = 0;
    end = tiles_of<kTile>(length_of(P, b));
  } else {
    const int each = (P.batch + kThreads - 1) / kThreads;
    const int lo = min(tid * each, P.batch), hi = min(lo + each, P.batch);
    int64_t mine = 0;
    for (int i = lo; i < hi; ++i) mine += cost + tiles_of<kTile>(length_of(P, i));
    int64_t upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += s_sum[w];
    int64_t run = upto - mine;
    for (int i = lo; i < hi; ++i) {
      s_before[i] = run;
      run += cost + tiles_of<kTile>(length_of(P, i));
    }
    if (tid == kThreads - 1) s_before[P.batch] = upto;
    __syncthreads();
    const int64_t total = s_before[P.batch] * pairs;
    share = divide(total + gridDim.x - 1, gridDim.x);
    first = min(blockIdx.x * share, total);
    end = min(first + share, total);
    if (tid < 2) P.plan[2 * blockIdx.x + tid] = make_int4(0, 0, 0, 0);
    __syncthreads();                             // (thread 0 may fill in either of them)
    if (first == end) return;
    int l = 0, h = P.batch - 1;                  // the request of unit `first`
    while (l < h) {
      const int mid = (l + h + 1) >> 1;
      if (s_before[mid] * pairs <= first) l = mid;
      else h = mid - 1;
    }
    b = l;
    const int64_t in = first - s_before[b] * pairs;
    const int units = (int)(s_before[b + 1] - s_before[b]);
    pair = (int)divide(in, units);
    u0 = (int)(in - (int64_t)pair * units);
    if (u0 + (end - first) <= cost) return;      // nothing but the cost of a pair that begins further on
  }

  uint8_t* ring = smem + warp * (kStages * 2 * kHalf);
  const uint32_t ring_at = smem_u32(ring);
  const int gid = lane >> 2, t4 = lane & 3;
  const float nan = __int_as_float(0x7FC00000);
  // this lane's piece of a warp-wide copy: rows copy_row, copy_row + kStep, ..; the swizzle of a row r is r & 7
  const int copy_row = lane / kChunks, copy_c = lane % kChunks;
  const uint32_t ring_copy = ring_at + copy_row * D * 2 + ((copy_c ^ copy_row) << 4);
  // where this lane's rows of K (row = position) and V (transposed) fragments begin; pieces 2j on are 32 j bytes on, swizzled alike
  const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, v_row = (lane & 7) + (lane >> 4) * 8;
  const uint32_t k_frag = ring_at + k_row * D * 2 + (((lane >> 4) ^ (k_row & 7)) << 4);
  const uint32_t v_frag = ring_at + kHalf + v_row * D * 2 + ((((lane >> 3) & 1) ^ (v_row & 7)) << 4);

  // ---- the stretch of one pair that is worked on: tiles t0 .. t0 + nt - 1 of request b, units u0 .. u0 + used - 1 of the pair, from
  // unit `at` of the sequence
  int64_t at = first;
  int n, tiles, t0, nt, used, hk, head0, heads, base0;
  const int32_t* pages;
  const T *cos_t, *sin_t;
  bool bad;
  auto enter = [&]() {
    const int len = length_of(P, b);
    n = max(len, 0);
    bad = len < 0;
    tiles = tiles_of<kTile>(len);
    used = (int)min((int64_t)(tiles + cost - u0), end - at);
    t0 = max(u0 - cost, 0);
    nt = u0 + used - cost - t0;
    hk = pair / P.chunks;
    head0 = hk * P.group + (pair - hk * P.chunks) * kRows;
    heads = min(kRows, (hk + 1) * P.group - head0);
    base0 = t0 * kTile + warp * 16;
    pages = P.table + (int64_t)b * P.table_stride;
    cos_t = (const T*)P.cos_t + (int64_t)(n - 1) * D;
    sin_t = (const T*)P.sin_t + (int64_t)(n - 1) * D;
  };
  enter();

  // ---- the ring ------------------------------------------------------------------------------------------------------
  auto page_of = [&](int p) { return (int)(((uint64_t)(uint32_t)p * P.page_mul) >> P.page_shift); };
  int page_next = 0;
  // Tile i of a stretch goes to stage (i + 1) % stages.  All but the last stage's worth of a stretch is asked for while the one
  // before it is being joined, which uses stage 0.
  auto stage_of = [&](int i) { return (uint32_t)((i + 1) % kStages) * (2 * kHalf); };
  // ALIGNED: the page of the 16 positions; else lane r (and r + 16) that of row r.  Loaded one tile ahead of its use.
  auto look_up = [&](int i) {
    const int p = base0 + i * kTile + (ALIGNED ? 0 : lane & 15);
    page_next = i < nt && p < n ? pages[page_of(p)] : 0;
  };
  auto issue = [&](int i) {
    const int base = base0 + i * kTile;
    if (i < nt && base < n) {
      const int page = page_next;
      look_up(i + 1);
      const uint32_t dst = ring_copy + stage_of(i);
      const int fresh = n - 1 - base;           // row of the new position, if it is one of these 16
      if (ALIGNED && fresh >= 16 && page >= 0 && page < P.num_pages) {   // 16 rows of one page: nothing to decide
        const int64_t off = ((int64_t)hk * P.page_size + (base - page_of(base) * P.page_size) + copy_row) * D + copy_c * 8;
        const T* ks = (const T*)P.k_pages + page * P.k_page_stride + off;
        const T* vs = (const T*)P.v_pages + page * P.v_page_stride + off;
#pragma unroll
        for (int j = 0; j < 16; j += kStep) {   // (the swizzle of row j + copy_row is that of copy_row, turned by j)
          cp_async16((dst + j * D * 2) ^ ((j & 7) << 4), ks + j * D);
          cp_async16((dst + kHalf + j * D * 2) ^ ((j & 7) << 4), vs + j * D);
        }
        cp_async_commit();
        return;
      }
      const int p = base + (lane & 15);
      const bool valid = p < n, found = valid && page >= 0 && page < P.num_pages;
      bad |= valid && !found;
      const int in_page = p - page_of(p) * P.page_size;
      const int code = found ? page : -1;
#pragma unroll
      for (int j = 0; j < 16; j += kStep) {
        const int r = j + copy_row;
        const int pg = __shfl_sync(0xFFFFFFFFu, code, r), rw = __shfl_sync(0xFFFFFFFFu, in_page, r);
        const bool keep = pg >= 0 && r < fresh;
        const int64_t off = ((int64_t)hk * P.page_size + rw) * D + copy_c * 8;
        const uint32_t d = (dst + j * D * 2) ^ ((j & 7) << 4);
        if (r != fresh) {                       // rows behind the last position: zeros
          cp_async16(d, (const T*)P.k_pages + (keep ? pg * P.k_page_stride + off : 0), keep);
          cp_async16(d + kHalf, (const T*)P.v_pages + (keep ? pg * P.v_page_stride + off : 0), keep);
        }
      }
      const int fresh_page = __shfl_sync(0xFFFFFFFFu, code, fresh & 15), fresh_row = __shfl_sync(0xFFFFFFFFu, in_page, fresh & 15);
      if (fresh < 16) {                         // the new position: turned, stored to the page and to the ring
        const bool write = fresh_page >= 0 && pair == hk * P.chunks;
        const int64_t off = ((int64_t)hk * P.page_size + fresh_row) * D;
        T* kd = (T*)P.k_pages + (write ? fresh_page * P.k_page_stride + off : 0);
        T* vd = (T*)P.v_pages + (write ? fresh_page * P.v_page_stride + off : 0);
        uint8_t* row = ring + stage_of(i) + fresh * D * 2;
        const int sw = fresh & 7;
        if (lane < D / 16) {
          float x0[8], x1[8];
          turn8<T, D>((const T*)P.k + b * P.k_stride + (int64_t)hk * D + lane * 8, cos_t + lane * 8, sin_t + lane * 8, x0, x1);
          const uint4 lo = pack8<T>(x0), hi = pack8<T>(x1);
          *reinterpret_cast<uint4*>(row + ((lane ^ sw) << 4)) = lo;
          *reinterpret_cast<uint4*>(row + (((lane + D / 16) ^ sw) << 4)) = hi;
          if (write) {
            *reinterpret_cast<uint4*>(kd + lane * 8) = lo;
            *reinterpret_cast<uint4*>(kd + lane * 8 + D / 2) = hi;
          }
        } else if (lane >= 16 && lane < 16 + D / 8) {
          const int c = lane - 16;
          const uint4 x = *reinterpret_cast<const uint4*>((const T*)P.v + b * P.v_stride + (int64_t)hk * D + c * 8);
          *reinterpret_cast<uint4*>(row + kHalf + ((c ^ sw) << 4)) = x;
          if (write) *reinterpret_cast<uint4*>(vd + c * 8) = x;
        }
      }
    }
    cp_async_commit();
  };

  // ---- q: turned, as the type's nearest value and what that leaves (the products see q as exactly as fp32 does); rows behind the
  // group zero.  A thread takes four pairs (i, i + D/2).
  auto stage_q = [&]() {
    for (int it = tid; it < NB * 8 * (D / 8); it += kThreads) {
      const int r = it / (D / 8), c = (it - r * (D / 8)) * 4;
      float x0[4] = {0.f, 0.f, 0.f, 0.f}, x1[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < heads && n > 0) {
        const T* src = (const T*)P.q + b * P.q_stride + (int64_t)(head0 + r) * D + c;
        float a0[4], a1[4], c0[4], c1[4], s0[4], s1[4];
        load4(src, a0);
        load4(src + D / 2, a1);
        load4(cos_t + c, c0);
        load4(cos_t + c + D / 2, c1);
        load4(sin_t + c, s0);
        load4(sin_t + c + D / 2, s1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x0[e] = a0[e] * c0[e] - a1[e] * s0[e];
          x1[e] = a1[e] * c1[e] + a0[e] * s1[e];
        }
      }
      const int at0 = (((c >> 3) ^ (r & 7)) << 4) + (c & 4) * 2, at1 = ((((c + D / 2) >> 3) ^ (r & 7)) << 4) + (c & 4) * 2;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        uint8_t* row = s_q + (part * kRows + r) * D * 2;
        store4<T>(row + at0, x0);
        store4<T>(row + at1, x1);
      }
    }
  };

  auto begin = [&]() {
    look_up(0);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);
  };
  begin();
  stage_q();
  __syncthreads();
  issue(kStages - 1);

  while (true) {
    uint32_t qf[NB][D / 32][4], qr[NB][D / 32][4];   // columns = heads: two k steps per load; and what the rounding of q left
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      const int r = h * 8 + (lane & 7);
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        ldsm4(smem_u32(s_q) + r * D * 2 + (((4 * ks + (lane >> 3)) ^ (r & 7)) << 4), qf[h][ks]);
        ldsm4(smem_u32(s_q) + kRows * D * 2 + r * D * 2 + (((4 * ks + (lane >> 3)) ^ (r & 7)) << 4), qr[h][ks]);
      }
    }

    // heads 8h + 2 t4 and + 1 of this lane: running maximum (of the raw scores) and sum; output^T, rows = dimensions
    float m[NB][2], limit[NB][2], l[NB][2], o[NB][D / 16][4];
    const float slack = Exponents<T>::slack / P.scale_log2;
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      m[h][0] = m[h][1] = limit[h][0] = limit[h][1] = -INFINITY;
      l[h][0] = l[h][1] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][j][e] = 0.f;
    }
    for (int i = 0; i < nt; ++i) {
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const int left = n - (base0 + i * kTile);   // positions of these 16 that exist, if positive
      if (left > 0) {
        const uint32_t stage = stage_of(i);
        float s[NB][4], s_rest[NB][4];            // (position gid, heads), (position gid + 8, heads)
#pragma unroll
        for (int h = 0; h < NB; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][e] = s_rest[h][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t kf[4];
          ldsm4((k_frag + stage) ^ (ks << 5), kf);
#pragma unroll
          for (int h = 0; h < NB; ++h) {
            mma16816<T>(s[h], kf, qf[h][ks / 2][(ks & 1) * 2], qf[h][ks / 2][(ks & 1) * 2 + 1]);
            mma16816<T>(s_rest[h], kf, qr[h][ks / 2][(ks & 1) * 2], qr[h][ks / 2][(ks & 1) * 2 + 1]);
          }
        }
#pragma unroll
        for (int h = 0; h < NB; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][e] += s_rest[h][e];   // (two chains of products, half as long)
        if (left < 16) {
#pragma unroll
          for (int h = 0; h < NB; ++h) {
            if (gid >= left) s[h][0] = s[h][1] = -INFINITY;
            if (gid + 8 >= left) s[h][2] = s[h][3] = -INFINITY;
          }
        }
        // The reference that the exponents are taken against moves only when a score has passed it by more than the slack:
        // weights up to that are as exact in every type here, and most tiles need no reduction over the positions.
        bool moved = false;
#pragma unroll
        for (int h = 0; h < NB; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) moved |= fmaxf(s[h][e], s[h][e + 2]) > limit[h][e];
        if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
          for (int h = 0; h < NB; ++h) {
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = fmaxf(s[h][e], s[h][e + 2]);
#pragma unroll
              for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, w));
              top = fmaxf(top, m[h][e]);
              f[e] = fast_exp2((m[h][e] - top) * P.scale_log2);
              m[h][e] = top;
              limit[h][e] = top + slack;
              l[h][e] *= f[e];
            }
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              o[h][j][0] *= f[0];
              o[h][j][1] *= f[1];
              o[h][j][2] *= f[0];
              o[h][j][3] *= f[1];
            }
          }
        }
        uint32_t pf[NB][2], pr[NB][2];            // weights^T, rows = positions, columns = heads; and what their rounding left
#pragma unroll
        for (int h = 0; h < NB; ++h) {
          // (the difference first: the two products apart round by more than one from scores of 10^8 on)
          const float m0 = m[h][0], m1 = m[h][1];
          s[h][0] = fast_exp2(fmaf(s[h][0] - m0, P.scale_log2, Exponents<T>::bias));
          s[h][1] = fast_exp2(fmaf(s[h][1] - m1, P.scale_log2, Exponents<T>::bias));
          s[h][2] = fast_exp2(fmaf(s[h][2] - m0, P.scale_log2, Exponents<T>::bias));
          s[h][3] = fast_exp2(fmaf(s[h][3] - m1, P.scale_log2, Exponents<T>::bias));
          l[h][0] += s[h][0] + s[h][2];
          l[h][1] += s[h][1] + s[h][3];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t p = pack2<T>(s[h][2 * e], s[h][2 * e + 1]);
            const float2 f = to_f2(*reinterpret_cast<const typename Pair<T>::type*>(&p));
            pf[h][e] = transpose8(p);
            pr[h][e] = transpose8(pack2<T>(s[h][2 * e] - f.x, s[h][2 * e + 1] - f.y));
          }
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t vf[4];
          ldsm4_t((v_frag + stage) ^ (j << 5), vf);
#pragma unroll
          for (int h = 0; h < NB; ++h) {
            mma16816<T>(o[h][j], vf, pf[h][0], pf[h][1]);
            mma16816<T>(o[h][j], vf, pr[h][0], pr[h][1]);
          }
        }
      }
      __syncwarp();                               // every lane has read the stage before it is filled again
      issue(i + kStages);
    }
    cp_async_wait<0>();
    __syncwarp();
    // ---- on to the next stretch, while this one's results are joined -----------------------------------------------------
    const int done_n = n, done_heads = heads;
    const bool begins = t0 == 0, ends = t0 + nt == tiles, last = at + used + cost >= end;
    const int64_t pair_begin = at - u0 + cost, pair_end = pair_begin + tiles, out_row = (int64_t)b * P.Hq + head0;
    const bool failed = bad;
    if (!last) {
      at += used;
      u0 = 0;
      if (++pair == pairs) {
        pair = 0;
        ++b;
      }
      enter();
      begin();
    }
    float* mine = reinterpret_cast<float*>(ring);   // [heads][D] fp32, no more than the ring: dimension d of head r at d ^ 8 (r & 7)
#pragma unroll
    for (int h = 0; h < NB; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[h][e] += __shfl_xor_sync(0xFFFFFFFFu, l[h][e], w);
        const int r = h * 8 + t4 * 2 + e;
        if (gid == 0) {
          s_m[warp * kRows + r] = m[h][e];
          s_l[warp * kRows + r] = l[h][e];
        }
        if (r < done_heads) {
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            mine[r * D + ((j * 16 + gid) ^ ((r & 7) * 8))] = o[h][j][e];
            mine[r * D + ((j * 16 + gid + 8) ^ ((r & 7) * 8))] = o[h][j][e + 2];
          }
        }
      }
    if (failed) atomicCAS(P.status, 0, 61);
    const bool any_failed = __syncthreads_or(failed);
    const int slot_floats = 2 * kRows + P.rows_kept * D;
    float* part = P.whole ? nullptr : P.part + ((int64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * slot_floats;
    for (int it = tid; it < done_heads * (D / 4); it += kThreads) {
      const int r = it / (D / 4), c = (it - r * (D / 4)) * 4;
      float top = s_m[r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w * kRows + r]);
      float sum = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = s_m[w * kRows + r], f = mw == -INFINITY ? 0.f : fast_exp2((mw - top) * P.scale_log2);
        const float4 x = *reinterpret_cast<const float4*>(smem + w * (kStages * 2 * kHalf) + (r * D + (c ^ ((r & 7) * 8))) * 4);
        sum += s_l[w * kRows + r] * f;
        a.x += x.x * f;
        a.y += x.y * f;
        a.z += x.z * f;
        a.w += x.w * f;
      }
      if (any_failed) sum = nan;
      if (begins && ends) {
        const float inv = done_n > 0 || any_failed ? 1.f / sum : 0.f;          // idle: zeros
        uint2 packed;
        packed.x = pack2<T>(a.x * inv, a.y * inv);
        packed.y = pack2<T>(a.z * inv, a.w * inv);
        *reinterpret_cast<uint2*>((T*)P.out + (out_row + r) * D + c) = packed;
      } else {
        *reinterpret_cast<float4*>(part + 2 * kRows + r * D + c) = a;
        if (c == 0) {
          part[r] = top;
          part[kRows + r] = sum;
        }
      }
    }
    if (!(begins && ends) && tid == 0)
      P.plan[2 * blockIdx.x + (begins ? 1 : 0)] = make_int4((int)out_row, done_heads, (int)divide(pair_begin, share), (int)divide(pair_end - 1, share));
    if (last) {
      if (!P.whole) pdl_trigger();                // (without a join, the next kernel starts when the new rows are in the pages)
      return;
    }
    stage_q();
    __syncthreads();                              // stage 0 is free again, and q is there
    issue(kStages - 1);
  }
}

// Pairs that several CTAs share: each of them joins a slice of the outputs.  A float4 of an output is added up by as many
// lanes as there are parts (up to 32), so that all loads of a slice are in flight at once.
constexpr int kJoinThreads = 128;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(const __grid_constant__ AttnParams P) {
  pdl_enter();
  const int slot = 2 * kRows + P.rows_kept * D;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int4 plan = P.plan[2 * blockIdx.x + which];
    if (plan.y == 0) continue;
    const int c0 = plan.z, count = plan.w - plan.z + 1, units = plan.y * (D / 4);
    const int lo = (int)((int64_t)units * ((int)blockIdx.x - c0) / count), hi = (int)((int64_t)units * ((int)blockIdx.x - c0 + 1) / count);
    int lanes = 2;                                // of a unit
    while (lanes < 32 && lanes < count) lanes *= 2;
    const int sub = threadIdx.x % lanes;
    for (int u0 = lo; u0 < hi; u0 += kJoinThreads / lanes) {   // the same trips for the whole CTA
      const int u = min(u0 + (int)threadIdx.x / lanes, hi - 1), r = u / (D / 4), c = (u - r * (D / 4)) * 4;
      float m = -INFINITY, l = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = sub; i < count; i += lanes) {
        const float* part = P.part + ((int64_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * slot;
        const float mi = part[r], li = part[kRows + r];
        const float4 o = *reinterpret_cast<const float4*>(part + 2 * kRows + r * D + c);
        const float top = fmaxf(m, mi);
        const float f = m == -INFINITY ? 0.f : fast_exp2((m - top) * P.scale_log2), g = mi == -INFINITY ? 0.f : fast_exp2((mi - top) * P.scale_log2);
        m = top;
        l = l * f + li * g;
        a = make_float4(a.x * f + o.x * g, a.y * f + o.y * g, a.z * f + o.z * g, a.w * f + o.w * g);
      }
      float top = m;
      for (int w = 1; w < lanes; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, w));
      const float f = m == -INFINITY ? 0.f : fast_exp2((m - top) * P.scale_log2);
      l *= f;
      a = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
      for (int w = 1; w < lanes; w <<= 1) {
        l += __shfl_xor_sync(0xFFFFFFFFu, l, w);
        a.x += __shfl_xor_sync(0xFFFFFFFFu, a.x, w);
        a.y += __shfl_xor_sync(0xFFFFFFFFu, a.y, w);
        a.z += __shfl_xor_sync(0xFFFFFFFFu, a.z, w);
        a.w += __shfl_xor_sync(0xFFFFFFFFu, a.w, w);
      }
      if (sub == 0 && u0 + (int)threadIdx.x / lanes < hi) {
        const float inv = 1.f / l;
        uint2 packed;
        packed.x = pack2<T>(a.x * inv, a.y * inv);
        packed.y = pack2<T>(a.z * inv, a.w * inv);
        *reinterpret_cast<uint2*>((T*)P.out + ((int64_t)plan.x + r) * D + c) = packed;
      }
    }
  }
}

template <typename T, int D, int NB, bool ALIGNED, int W>
int launch_paged_attention(const AttnParams& P, int grid, cudaStream_t s) {
  constexpr int kMost = fixed_bytes<D, W>() + (W == kManyWarps ? 0 : (kMaxBatch + 1) * 8);
  static bool attr_set[64] = {false};
  int dev = 0;
  BSB_CUDA(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    BSB_CUDA(cudaFuncSetAttribute(paged_attention_kernel<T, D, NB, ALIGNED, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    attr_set[dev] = true;
  }
  const size_t smem = fixed_bytes<D, W>() + (P.whole ? 0 : (size_t)(P.batch + 1) * 8);
  BSB_CUDA(launch_pdl(paged_attention_kernel<T, D, NB, ALIGNED, W>, dim3(grid), dim3(W * 32), smem, s, P));
  return check_launch("paged_attention_kernel");
}
template <typename T, int D, int NB, bool ALIGNED>
int launch_paged_attention(AttnParams P, cudaStream_t s) {
  const int pairs = P.Hkv * P.chunks;
  P.whole = P.most <= kWholePositions;
  if (P.whole) {
    const int grid = P.batch * pairs;
    if constexpr (NB == 1)
      if (grid <= sm_count()) return launch_paged_attention<T, D, NB, ALIGNED, kManyWarps>(P, grid, s);
    return launch_paged_attention<T, D, NB, ALIGNED, 4>(P, grid, s);
  }
  const int grid = sm_count() * (NB == 1 ? Shape<D>::ctas : 2);
  if (int rc = launch_paged_attention<T, D, NB, ALIGNED, 4>(P, grid, s)) return rc;
  BSB_CUDA(launch_pdl(paged_attention_join_kernel<T, D>, dim3(grid), dim3(kJoinThreads), 0, s, P));
  return check_launch("paged_attention_join_kernel");
}
template <typename T, int D>
int launch_paged_attention(const AttnParams& P, cudaStream_t s) {
  const bool aligned = P.page_size % 16 == 0;
  if (P.group <= 8) return aligned ? launch_paged_attention<T, D, 1, true>(P, s) : launch_paged_attention<T, D, 1, false>(P, s);
  return aligned ? launch_paged_attention<T, D, 2, true>(P, s) : launch_paged_attention<T, D, 2, false>(P, s);
}

}  // namespace
}  // namespace bsb

using namespace bsb;

extern "C" {

int64_t bsb_paged_attention_scratch_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  if (batch < 0 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || q_heads % kv_heads != 0) return -1;
  const int rows = q_heads / kv_heads < kRows ? q_heads / kv_heads : kRows;
  return (int64_t)sm_count() * kMaxCtas * (32 + 2 * (2 * kRows + (int64_t)rows * head_dim) * 4);
}

int bsb_paged_decode_attention(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                               const void* cos_table, const void* sin_table, int64_t table_len, const int64_t* positions,
                               const int32_t* block_table, int64_t table_stride, int32_t table_width, void* k_pages, void* v_pages,
                               int64_t num_pages, int64_t k_page_stride, int64_t v_page_stride, void* out, int32_t batch, int32_t q_heads,
                               int32_t kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype, void* scratch, int64_t scratch_bytes,
                               void* stream) {
  BSB_CHECK_ARG(batch >= 0 && q_heads >= 1 && kv_heads >= 1 && q_heads % kv_heads == 0, "bad attention shape");
  BSB_CHECK_ARG(dtype == BSB_F16 || dtype == BSB_BF16, "paged attention: fp16 or bf16 (got dtype code %d)", dtype);
  BSB_CHECK_ARG(head_dim == 128 || head_dim == 64, "paged attention is built for head_dim 64 and 128 (got %d)", head_dim);
  BSB_CHECK_ARG(page_size >= 1 && num_pages >= 1 && num_pages <= INT_MAX && table_len >= 1 && table_width >= 1 && table_stride >= table_width,
                "bad page shape");
  if (batch == 0) return BSB_OK;
  BSB_CHECK_ARG(q && k && v && cos_table && sin_table && positions && block_table && k_pages && v_pages && out, "NULL buffer");
  const int64_t page = (int64_t)kv_heads * page_size * head_dim;
  BSB_CHECK_ARG((batch == 1 || (q_stride >= (int64_t)q_heads * head_dim && k_stride >= (int64_t)kv_heads * head_dim && v_stride >= (int64_t)kv_heads * head_dim)) &&
                (num_pages == 1 || (k_page_stride >= page && v_page_stride >= page)), "stride smaller than the row or page");
  BSB_CHECK_ARG((q_stride | k_stride | v_stride | k_page_stride | v_page_stride) % 8 == 0, "strides must be multiples of 8 elements");
  BSB_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cos_table | (uintptr_t)sin_table | (uintptr_t)out |
                 (uintptr_t)k_pages | (uintptr_t)v_pages) % 16 == 0, "buffers must be 16-byte aligned");
  BSB_CHECK_ARG((int64_t)batch * q_heads <= INT_MAX, "batch * q_heads too large");
  const int64_t need = bsb_paged_attention_scratch_bytes(batch, q_heads, kv_heads, head_dim);
  BSB_CHECK_ARG(scratch != nullptr && (uintptr_t)scratch % 16 == 0, "scratch is NULL or not 16-byte aligned");
  if (scratch_bytes < need) {
    set_error("scratch of %lld bytes needed, %lld given", (long long)need, (long long)scratch_bytes);
    return BSB_EWORKSPACE;
  }
  AttnParams P;
  P.status = device_index_word();
  if (P.status == nullptr) return BSB_ECUDA;
  P.cos_t = cos_table;
  P.sin_t = sin_table;
  P.k_pages = k_pages;
  P.v_pages = v_pages;
  P.q_stride = q_stride;
  P.k_stride = k_stride;
  P.v_stride = v_stride;
  P.k_page_stride = k_page_stride;
  P.v_page_stride = v_page_stride;
  P.table_len = table_len;
  P.num_pages = num_pages;
  P.table_stride = table_stride;
  P.most = (int64_t)table_width * page_size;
  if (P.most > INT_MAX - 63) P.most = INT_MAX - 63;
  P.page_shift = 31;                     // mul = ceil(2^shift / page_size) < 2^32 with 2^(shift - 31) >= page_size: exact below 2^31
  while ((1ll << (P.page_shift - 31)) < page_size) ++P.page_shift;
  P.page_mul = (uint32_t)(((1ull << P.page_shift) + page_size - 1) / page_size);
  P.Hq = q_heads;
  P.Hkv = kv_heads;
  P.group = q_heads / kv_heads;
  P.chunks = (P.group + kRows - 1) / kRows;
  P.rows_kept = P.group < kRows ? P.group : kRows;
  P.page_size = page_size;
  P.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  P.plan = reinterpret_cast<int4*>(scratch);
  P.part = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(scratch) + (int64_t)sm_count() * kMaxCtas * 32);
  // more requests than a launch keeps prefix sums of: launch after launch, in stream order, on the same scratch
  for (int32_t b0 = 0; b0 < batch; b0 += kMaxBatch) {
    P.batch = batch - b0 < kMaxBatch ? batch - b0 : kMaxBatch;
    P.q = (const uint16_t*)q + b0 * q_stride;
    P.k = (const uint16_t*)k + b0 * k_stride;
    P.v = (const uint16_t*)v + b0 * v_stride;
    P.out = (uint16_t*)out + (int64_t)b0 * q_heads * head_dim;
    P.positions = positions + b0;
    P.table = block_table + b0 * table_stride;
    const cudaStream_t s = (cudaStream_t)stream;
    int rc;
    if (dtype == BSB_F16) rc = head_dim == 128 ? launch_paged_attention<__half, 128>(P, s) : launch_paged_attention<__half, 64>(P, s);
    else rc = head_dim == 128 ? launch_paged_attention<__nv_bfloat16, 128>(P, s) : launch_paged_attention<__nv_bfloat16, 64>(P, s);
    if (rc) return rc;
  }
  return BSB_OK;
}

}  // extern "C"
