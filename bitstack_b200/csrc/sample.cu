// The next token of every row: temperature, top-k, top-p and min-p on the logits, drawn with a given uniform number.
//
// Weights.  w(x) = 2^((x - max) log2(e) / T), as an integer in units of 2^-S: sums of integers do not depend on their order,
// so the kept set and the token are the same bits run to run whatever adds them up, and the cumulative weights next to a
// border are right to 2^-S per term (S = 45 for a 128256-token vocabulary, 2^62 is never passed).  The exponential is
// evaluated in 64 bits from a table of 256 powers and a polynomial on |r| <= 1/512 (table-driven evaluation after Tang, 1989;
// the remainder (ln 2 / 512)^5 / 120 is 4e-17).
// Kept set.  All three filters cut the tokens sorted by logit (ties: lowest index first) behind some place, so the set is
// given by a value and a number of tokens with exactly that value.  No sort: a histogram over equal steps of (max - x) / T finds
// the step in which the count (or weight) from the top passes what is wanted; the few tokens of that step are gathered and
// compared with one another.  A step that holds too many (near-equal logits) is taken apart by the bits of its values first.
// Draw.  The first index in vocabulary order whose cumulative kept weight exceeds u times the total: weights of runs of 256
// tokens, the run by a scan, the token inside it by one warp.
//
// Measured: one row of 128256 fp16 logits, top-k 50 and top-p 0.9: 14 us; 64 rows, each with settings of its own: 51-76 us, by how many
// have a wide top-p; all with top-p 0.9 at temperature 1: 86 us; 256 rows of 32000 fp32 logits, top-p: 76 us.  Bound by the
// instructions on the tokens that top-p looks at (their exponentials, three limb additions each in shared memory) and by barriers,
// for few rows those of the cluster; 64 registers, with 172-204 bytes of spills.  bf16 logits of a wide top-p take 125 us where
// fp16 ones take 86: more than kList tokens share the border's value, which is then taken apart by its bits to the last.
//
// A row is a cluster of up to 8 CTAs, each with its part of the row in shared memory: the logits are read once, and
// histograms, totals and results are exchanged through distributed shared memory.
#include <cooperative_groups.h>

#include <climits>
#include <math.h>

#include "common.cuh"
#include "numeric.cuh"

namespace cg = cooperative_groups;

namespace bsb {
namespace {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kRun = 256;                       // tokens of a run (one warp, eight per lane)
constexpr int kBins = 1024;
constexpr int kMaxCluster = 8;
constexpr int kMaxPart = 32768;                 // tokens of one CTA: 2^15 limbs of 17 bits add up below 2^32
constexpr int kMaxVocab = kMaxCluster * kMaxPart;
constexpr int kList = 128;                      // tokens that are compared with one another (256: 64 rows alike, 256
                                                // rows of 32000 cut by top-k 1000 and top-p 94 us instead of 90)
constexpr float kSpan = 32.f;                   // the histogram's steps cover this many temperatures below the maximum

// values in shared memory: the logits' own type, NaN as -infinity
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }
__device__ __forceinline__ __half clean(__half x) { return __hmax(x, __ushort_as_half(0xFC00)); }
__device__ __forceinline__ __nv_bfloat16 clean(__nv_bfloat16 x) { return __hmax(x, __ushort_as_bfloat16(0xFF80)); }
template <typename T> __device__ __forceinline__ T make(float x);
template <> __device__ __forceinline__ float make<float>(float x) { return x; }
template <> __device__ __forceinline__ __half make<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 make<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
// order-preserving bits of a value; -0 as +0
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_order_bits(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// S of the weights' unit 2^-S: vocab * 2^S <= 2^62.  The sums of all weights have to stay there: past 2^64 they are no longer
// ordered, the CTAs of a row take different ways, and one may leave while the others still read its shared memory.
constexpr int unit_of(int64_t vocab) {
  int s = 50;
  while (vocab > (1ll << (62 - s))) --s;         // (vocab << s would itself pass 64 bits)
  return s;
}
static_assert(unit_of(1) == 50 && unit_of(4096) == 50 && unit_of(4097) == 49 && unit_of(128256) == 45 && unit_of(kMaxVocab) == 44, "");

struct Weigher {
  const double* powers;   // 2^(i/256)
  double c256, top;       // exponent in 256ths: (x - top) c256, c256 = 256 log2(e) / T
  uint32_t vanish;        // high word of the (negative) exponent from which on a weight is below half a unit
  int unit;               // S
  __device__ __forceinline__ uint64_t operator()(float x) const {
    // No branch: callers take several values side by side, and the chain of 64-bit operations is long.
    const double t = ((double)x - top) * c256;    // (never NaN: infinite maxima were mapped away, and c256 > 0)
    const double magic = 6755399441055744.0;      // 1.5 * 2^52: adding it leaves the nearest integer in the low word
    const double s = t + magic;
    const double r = t - (s - magic);             // at most a half, in 256ths
    const int i = __double2loint(s);
    const double h = 0.6931471805599453094 / 256.0;
    double p = fma(r, h * h * h * h / 24.0, h * h * h / 6.0);
    p = fma(r, p, h * h / 2.0);
    p = fma(r, p, h);
    p = fma(r, p, 1.0);
    const double w = powers[i & 255] * p;         // times 2^(S + i / 256), by its exponent
    const double scaled = __hiloint2double(__double2hiint(w) + ((i >> 8) + unit) * (1 << 20), __double2loint(w));
    const uint64_t rounded = (uint64_t)__double_as_longlong(scaled + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;   // a whole number of units
    return (uint32_t)__double2hiint(t) >= vanish ? 0 : rounded;
  }
};

struct Found {            // the bin in which the count (or weight) from the top reaches what is wanted
  uint64_t above_mass, mass;   // weight of the bins in front of it, and its own
  double want;
  uint32_t above, count;  // tokens in front of it, tokens in it
  int bin;
};
struct Cut {              // kept: logits above x, and of those equal to x the first `ties` (all of them: !partial)
  float x;
  uint32_t ties, partial;
};

// what the CTAs of a cluster tell one another; peers write into it
struct Exchange {
  uint64_t kept[kMaxCluster];
  float top[kMaxCluster];
  uint32_t at[kMaxCluster], ties[kMaxCluster];
  Cut cut;
  uint32_t listed;        // the leader's list
};

struct SampleShared {
  double powers[256];
  uint32_t hist[4][kBins];              // count, and the weight in three limbs of 17 bits; peers read it
  uint64_t list_w[kList];
  float list_x[kList], own_x[kList];
  uint32_t list_at[kList], own_at[kList];
  uint64_t run_mass[kMaxPart / kRun];
  uint32_t run_ties[kMaxPart / kRun];
  uint64_t red[kSampleWarps];
  uint32_t red2[kSampleWarps];
  float warp_top[kSampleWarps];
  uint32_t own_listed, list_from;
  Found found;
  Exchange ex;
};

struct SampleParams {
  const void* logits;
  int64_t vocab, stride;
  const float *uniforms, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int64_t *tokens, *pos;
  float* logprobs;
  int unit, part;         // part: tokens of a CTA, a multiple of kRun
};

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleParams P) {
  constexpr int kPer = 16 / sizeof(T);            // values of a 16-byte vector
  extern __shared__ __align__(16) uint8_t smem[];
  SampleShared& S = *reinterpret_cast<SampleShared*>(smem);
  T* vals = reinterpret_cast<T*>(smem + ((sizeof(SampleShared) + 15) / 16) * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto row_sync = [&]() {
    if (C == 1) __syncthreads();
    else cluster.sync();
  };
  const int64_t b = blockIdx.x / C;
  const int64_t base = (int64_t)rank * P.part;
  const int n = (int)max(min(P.vocab - base, (int64_t)P.part), (int64_t)0);
  const int runs = (n + kRun - 1) / kRun, vecs = runs * kRun / kPer;

  if (tid < 256) S.powers[tid] = exp2(tid / 256.0);
  if (tid == 0) S.ex.listed = 0;
  row_sync();   // every CTA of the row runs before another one writes into its shared memory
  pdl_wait();   // no early release: this kernel writes *pos, which the dense decode attention reads in front of its own wait

  // the row's settings, asked for together and in front of its values (one after the other where they are used, each is a wait)
  const float temp = P.temperature ? __ldg(P.temperature + b) : 1.f, mp = P.min_p ? __ldg(P.min_p + b) : 0.f, number = __ldg(P.uniforms + b);
  float p = P.top_p ? __ldg(P.top_p + b) : 1.f;
  int32_t k = P.top_k ? __ldg(P.top_k + b) : 0;
  // ---- the row's values and their maximum; tokens that fill up the last run are -infinity -------------------------------
  const T* row = (const T*)P.logits + b * P.stride + base;
  float top = -INFINITY;
  {
    const int nv = reinterpret_cast<uintptr_t>(row) % 16 == 0 ? n / kPer : 0;
#pragma unroll 4
    for (int i = tid; i < nv; i += kSampleThreads) {
      uint4 raw = __ldcs(reinterpret_cast<const uint4*>(row) + i);
      T* x = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        x[e] = clean(x[e]);
        top = fmaxf(top, to_f(x[e]));
      }
      reinterpret_cast<uint4*>(vals)[i] = raw;
    }
    for (int i = nv * kPer + tid; i < runs * kRun; i += kSampleThreads) {
      const T x = i < n ? clean(row[i]) : make<T>(-INFINITY);
      vals[i] = x;
      top = fmaxf(top, to_f(x));
    }
  }
  auto block_sum = [&](uint64_t v) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if (lane == 0) S.red[warp] = v;
    __syncthreads();
    v = S.red[lane % kSampleWarps];
    for (int o = kSampleWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
  };
  auto each_vec = [&](auto&& f) {                // f(the vector's values, index of the first in this CTA's part)
    for (int i = tid; i < vecs; i += kSampleThreads) {
      const uint4 raw = reinterpret_cast<const uint4*>(vals)[i];
      f(reinterpret_cast<const T*>(&raw), i * kPer);
    }
  };
  auto each = [&](auto&& f) {
    each_vec([&](const T* x, int) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) f(to_f(x[e]));
    });
  };
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (lane == 0) S.warp_top[warp] = top;
  __syncthreads();
  top = S.warp_top[lane % kSampleWarps];
  for (int o = kSampleWarps / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (tid < C) cluster.map_shared_rank(&S, tid)->ex.top[rank] = top;
  row_sync();
  for (int i = 0; i < C; ++i) top = fmaxf(top, S.ex.top[i]);
  if (b == 0 && rank == 0 && tid == 0 && P.pos != nullptr) *P.pos += 1;
  if (top == -INFINITY) {                        // a row that its mask leaves nothing of: token 0, as the greedy step gives
    if (rank == 0 && tid == 0) {
      P.tokens[b] = 0;
      if (P.logprobs) P.logprobs[b] = -INFINITY;
    }
    return;
  }
  if (!(temp > 0.f)) {                           // greedy: the first maximum
    uint32_t at = 0xFFFFFFFFu;
    each_vec([&](const T* x, int i) {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (to_f(x[e]) == top) at = min(at, (uint32_t)(i + e));
    });
    at = __reduce_min_sync(0xFFFFFFFFu, at);
    if (lane == 0) S.red2[warp] = at;
    __syncthreads();
    for (int w = 0; w < kSampleWarps; ++w) at = min(at, S.red2[w]);
    if (tid < C) cluster.map_shared_rank(&S, tid)->ex.at[rank] = at;
    row_sync();
    if (rank == 0 && tid == 0) {
      for (int i = 0; i < C; ++i)
        if (S.ex.at[i] != 0xFFFFFFFFu) {
          P.tokens[b] = (int64_t)i * P.part + S.ex.at[i];
          break;
        }
      if (P.logprobs) P.logprobs[b] = 0.f;
    }
    return;
  }
  if (top == INFINITY) {                         // infinities share everything
    for (int i = tid; i < runs * kRun; i += kSampleThreads) vals[i] = make<T>(to_f(vals[i]) == INFINITY ? 0.f : -INFINITY);
    top = 0.f;
    __syncthreads();
  }
  const double per_logit = fmax(1.4426950408889634074 / (double)temp, 1e-290);
  const Weigher weigh{S.powers, per_logit * 256.0, (double)top, (uint32_t)__double2hiint(-256.0 * (P.unit + 2)), P.unit};

  const double least = mp > 0.f ? (double)fminf(mp, 1.f) * (double)(1ull << P.unit) : 0.0;   // the likeliest token always stays
  const uint64_t fewest = (uint64_t)ceil(least);   // units of a token that stays
  const double u = number > 0.f ? (double)fminf(number, 0.99999994f) : 0.0;
  auto chosen = [&](int64_t token, float x, uint64_t total) {
    P.tokens[b] = token;
    if (P.logprobs) P.logprobs[b] = (float)(((double)x - (double)top) * per_logit * 0.6931471805599453094 - log((double)total / (double)(1ull << P.unit)));
  };

  // ---- the kept set ------------------------------------------------------------------------------------------------
  const float steps = fminf((float)kBins / (kSpan * temp), 1e30f);
  auto step_of = [&](float x) { return fminf((top - x) * steps, (float)(kBins - 1)); };   // (NaN, from 0 * infinity: the last)
  auto whole = [&](float q) { return (int)(__float_as_uint(q + 8388608.f) & 0x7FFFFFu); };  // to the nearest, by the bits of 2^23 + q
  // Bins of a round, from the highest values down: equal steps below the maximum; equal steps inside one of those; then ten
  // bits of the value at a time.  Every bin holds a stretch of values, and `inside` the tokens of the bins chosen so far.
  int coarse = 0, fine = 0, round = 0;
  uint32_t mask = 0, bits = 0;
  constexpr int kRounds = 6;
  auto shift_of = [](int round) { return max(42 - 10 * round, 0); };   // 22, 12, 2, 0 in rounds 2 .. 5
  auto fine_of = [&](float q) { return whole(fminf(fmaxf((q - ((float)coarse - 0.5f)) * (float)kBins, 0.f), (float)(kBins - 1))); };
  auto inside = [&](float x) {
    const float q = step_of(x);
    if (whole(q) != coarse) return false;
    if (round < 2) return true;
    return fine_of(q) == fine && (order_bits(x) & mask) == bits;
  };
  auto bin_of = [&](float x) {
    if (round == 0) return whole(step_of(x));
    if (round == 1) return fine_of(step_of(x));
    return kBins - 1 - (int)((order_bits(x) & ~mask) >> shift_of(round) & 1023u);
  };

  Cut cut{-INFINITY, 0, 0};                      // nothing is cut (tokens at -infinity have no weight)
  if (k < 0 || k >= P.vocab) k = 0;
  if (p <= 0.f) {                                // the likeliest token alone
    cut = Cut{top, 1, 1};
    p = 1.f;
    k = 0;
  }
#pragma unroll 1
  for (int stage = 0; stage < 2; ++stage) {      // by count (top-k), then by weight (top-p)
    const bool by_mass = stage == 1;
    if (by_mass ? !(p < 1.f) : k == 0) continue;
    Found f{0, 0, by_mass ? 0.0 : (double)k, 0, 0, 0};
    double want_all = f.want;
    mask = bits = 0;
    // Bounds of the tokens that a pass has to look at: the cut, and from the second round on the chosen step with a margin (rounding
    // is monotone, and a step's rounding errors stay far below 0.01); two comparisons where the step itself takes six instructions
    // (64 rows of 128256, top-k 1000 and top-p 64 -> 59 us, each with its own settings 66 -> 64).
    float lowest = cut.x, highest = INFINITY;
#pragma unroll 1
    for (round = 0;; ++round) {
      if (round > 0) row_sync();                 // (every CTA has read the histograms of the round before)
      for (int i = tid; i < kBins; i += kSampleThreads) reinterpret_cast<uint4*>(&S.hist[0][0])[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      auto add_mass = [&](int q, uint64_t w) {
        atomicAdd(&S.hist[1][q], (uint32_t)w & 0x1FFFFu);
        atomicAdd(&S.hist[2][q], (uint32_t)(w >> 17) & 0x1FFFFu);
        atomicAdd(&S.hist[3][q], (uint32_t)(w >> 34));
      };
      // (the share of the ties that a top-k cut leaves is added below, once: only what lies above the cut has its weight added)
      if (round == 0 && !by_mass) {
        each([&](float x) { atomicAdd(&S.hist[0][whole(step_of(x))], 1u); });
      } else if (round == 0 && cut.x == -INFINITY) {
        each_vec([&](const T* v, int) {
#pragma unroll
          for (int e0 = 0; e0 < kPer; e0 += 4) {  // four values side by side: a weight is a long chain of 64-bit operations
            uint64_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = weigh(to_f(v[e0 + e]));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int q = whole(step_of(to_f(v[e0 + e])));
              atomicAdd(&S.hist[0][q], 1u);
              if (w[e] != 0) add_mass(q, w[e]);
            }
          }
        });
      } else {                                   // few tokens are left by top-k, or inside the bins chosen so far
        each_vec([&](const T* v, int at) {
          uint32_t in = 0;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const float x = to_f(v[e]);
            in |= (x >= lowest && x <= highest ? 1u : 0u) << e;
          }
          for (; in != 0; in &= in - 1) {
            const float x = to_f(vals[at + __ffs(in) - 1]);
            if (round > 0 && !inside(x)) continue;
            const int q = bin_of(x);
            atomicAdd(&S.hist[0][q], 1u);
            if (by_mass && x > cut.x) add_mass(q, weigh(x));
          }
        });
      }
      __syncthreads();
      if (by_mass && rank == 0 && tid == 0 && (round == 0 || inside(cut.x))) {
        const int q = bin_of(cut.x);
        const uint64_t w = weigh(cut.x) * cut.ties;   // up to 62 bits: limbs of 17, 17 and 28; the sums stay below 2^32
        S.hist[1][q] += (uint32_t)w & 0x1FFFFu;
        S.hist[2][q] += (uint32_t)(w >> 17) & 0x1FFFFu;
        S.hist[3][q] += (uint32_t)(w >> 34);
      }
      row_sync();
      // every CTA adds up all bins of the row and scans them
      constexpr int kEach = 4;                   // (16-byte loads from the peers, by half the threads)
      uint64_t m[kEach] = {0, 0, 0, 0}, um = 0;
      uint32_t c[kEach] = {0, 0, 0, 0}, uc = 0;
      if (tid < kBins / kEach)
        for (int peer = 0; peer < C; ++peer) {
          const SampleShared* o = cluster.map_shared_rank(&S, peer);
          uint4 part[4];
#pragma unroll
          for (int l = 0; l < 4; ++l)
            part[l] = l == 0 || by_mass ? *reinterpret_cast<const uint4*>(&o->hist[l][tid * kEach]) : make_uint4(0, 0, 0, 0);
          const uint32_t* word = reinterpret_cast<const uint32_t*>(part);
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
            c[i] += word[i];
            m[i] += (uint64_t)word[4 + i] + ((uint64_t)word[8 + i] << 17) + ((uint64_t)word[12 + i] << 34);
          }
        }
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        um += m[i];
        uc += c[i];
      }
      const uint64_t own_m = um;
      const uint32_t own_c = uc;
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, um, o);
        const uint32_t z = __shfl_up_sync(0xFFFFFFFFu, uc, o);
        if (lane >= o) { um += y; uc += z; }
      }
      if (lane == 31) { S.red[warp] = um; S.red2[warp] = uc; }
      if (tid == 0) S.found = Found{0, 0, 0.0, 0, 0, -1};
      __syncthreads();
      uint64_t total = 0;
      for (int w = 0; w < kSampleWarps; ++w) {
        if (w == warp) { um += total; }
        total += S.red[w];
        if (w < warp) uc += S.red2[w];
      }
      const double want = round > 0 ? f.want : by_mass ? (double)p * (double)total : f.want;
      um -= own_m;
      uc -= own_c;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const double upto = by_mass ? (double)(um + m[i]) : (double)(uc + c[i]), from = by_mass ? (double)um : (double)uc;
        if (tid < kBins / kEach && upto >= want && from < want) S.found = Found{um, m[i], want, uc, c[i], tid * kEach + i};
        um += m[i];
        uc += c[i];
      }
      __syncthreads();
      const Found g = S.found;
      f.above += g.above;
      f.above_mass += g.above_mass;
      f.count = g.count;
      if (round == 0) want_all = want;
      // what is wanted of the bin; never more than it holds, whichever way 2^62 rounds
      f.want = by_mass ? fmin(want - (double)g.above_mass, (double)g.mass) : want - (double)g.above;
      if (round == 0) {
        coarse = g.bin;
        if (coarse < kBins - 1) lowest = fmaxf(lowest, top - ((float)coarse + 0.51f) / steps);
        highest = top - ((float)coarse - 0.51f) / steps;
      } else if (round == 1) fine = g.bin;
      else {
        bits |= (uint32_t)(kBins - 1 - g.bin) << shift_of(round);
        mask |= 1023u << shift_of(round);
      }
      if (f.count <= kList || round == kRounds - 1) break;
    }
    ++round;                                     // `inside` counts the bin that was found last
    if (f.count > kList) {                       // one value, many tokens
      Cut c{of_order_bits(bits), 0, 0};
      const double left = by_mass ? ceil(f.want / (double)weigh(c.x)) : f.want;
      c.ties = (uint32_t)fmin(fmax(left, 1.0), (double)f.count);
      if (c.x == cut.x && cut.ties < c.ties) c.ties = cut.ties;
      c.partial = c.ties < f.count;
      cut = c;
      row_sync();                                // (the histograms have been read)
      continue;
    }
    // The tokens of the bin into the leader's list; where all from the top on are few, those: then the leader finishes alone.
    const bool all = round == 1 && f.above + f.count <= kList;
    if (all) highest = INFINITY;
    if (tid == 0) S.own_listed = 0;
    __syncthreads();
    each_vec([&](const T* v, int at) {
      uint32_t in = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const float x = to_f(v[e]);
        in |= (x >= lowest && x <= highest ? 1u : 0u) << e;
      }
      for (; in != 0; in &= in - 1) {
        const int e = __ffs(in) - 1;
        const float x = to_f(vals[at + e]);
        if (all ? whole(step_of(x)) > coarse : !inside(x)) continue;
        const uint32_t i = atomicAdd(&S.own_listed, 1u);
        if (i < kList) {
          S.own_x[i] = x;
          S.own_at[i] = (uint32_t)(base + at + e);
        }
      }
    });
    __syncthreads();
    const uint32_t listed = min(S.own_listed, (uint32_t)kList);
    SampleShared* leader = cluster.map_shared_rank(&S, 0);
    if (tid == 0 && listed > 0) S.list_from = atomicAdd(&leader->ex.listed, listed);
    __syncthreads();
    for (uint32_t i = tid; i < listed; i += kSampleThreads) {
      const uint32_t at = S.list_from + i;
      if (at < kList) {
        leader->list_x[at] = S.own_x[i];
        leader->list_at[at] = S.own_at[i];
        leader->list_w[at] = weigh(S.own_x[i]);
      }
    }
    row_sync();
    if (rank == 0) {                             // the listed tokens are compared with one another
      const int size = (int)min(S.ex.listed, (uint32_t)kList);
      int lanes = 1;                             // threads that share a token's comparisons
      while (lanes < 32 && lanes * 2 * size <= kSampleThreads) lanes *= 2;
      const int i = tid / lanes, sub = tid % lanes;
      const bool mine = i < size;
      const float x = mine ? S.list_x[i] : 0.f;
      const uint32_t at = mine ? S.list_at[i] : 0;
      const uint64_t w = mine ? S.list_w[i] : 0;
      uint32_t higher = 0, equal = 0, first = 0;
      uint64_t heavier = 0;
      if (mine) {
        if (all) {
#pragma unroll 4
          for (int j = sub; j < size; j += lanes) {
            const float other = S.list_x[j];
            higher += other > x;
            equal += other == x;
            first += other == x && S.list_at[j] < at;
          }
        } else {
#pragma unroll 4
          for (int j = sub; j < size; j += lanes) {
            const float other = S.list_x[j];
            higher += other > x;
            equal += other == x;
          }
        }
        if (by_mass || (all && p < 1.f)) {
#pragma unroll 4
          for (int j = sub; j < size; j += lanes) heavier += S.list_x[j] > x ? S.list_w[j] : 0;
        }
      }
      for (int o = 1; o < lanes; o <<= 1) {
        higher += __shfl_xor_sync(0xFFFFFFFFu, higher, o);
        equal += __shfl_xor_sync(0xFFFFFFFFu, equal, o);
        first += __shfl_xor_sync(0xFFFFFFFFu, first, o);
        heavier += __shfl_xor_sync(0xFFFFFFFFu, heavier, o);
      }
      if (tid == 0) S.ex.cut = cut;
      __syncthreads();
      bool weight = by_mass;
      double want = f.want;
      if (!by_mass) {
        const uint32_t left = (uint32_t)k - (all ? 0 : f.above);
        if (mine && higher < left && left <= higher + equal) S.ex.cut = Cut{x, left - higher, left - higher < equal};
        __syncthreads();
        if (all && p < 1.f) {                    // top-p at once: the weight that the first cut leaves is all in the list
          cut = S.ex.cut;
          weight = true;
          want = (double)p * (double)block_sum(mine && sub == 0 && (x > cut.x || (x == cut.x && first < cut.ties)) ? w : 0);
        }
      } else if (all) {
        want = want_all;
      }
      if (weight) {
        if (mine && sub == 0 && x >= cut.x) {
          const uint32_t ties = x == cut.x ? min(cut.ties, equal) : equal;
          if ((double)heavier < want && !((double)(heavier + ties * w) < want)) {
            const double r = ceil((want - (double)heavier) / (double)w);
            const uint32_t left = r < 1.0 ? 1u : r > (double)ties ? ties : (uint32_t)r;
            S.ex.cut = Cut{x, left, left < equal};
          }
        }
        __syncthreads();
      }
      const Cut c = S.ex.cut;
      if (all) {                                 // the draw, among the listed
        const bool keep = mine && (x > c.x || (x == c.x && first < c.ties)) && w >= fewest;
        if (mine && sub == 0) S.list_w[i] = keep ? w : 0;
        __syncthreads();
        uint64_t before = 0, total = 0;
        if (mine)
          for (int j = sub; j < size; j += lanes) {
            const uint64_t o = S.list_w[j];
            total += o;
            before += S.list_at[j] < at ? o : 0;
          }
        for (int o = 1; o < lanes; o <<= 1) {
          total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
          before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
        }
        const double target = u * (double)total;
        if (keep && sub == 0 && (double)(before + w) > target && !((double)before > target)) chosen(at, x, total);
      } else if (tid == 0) {
        S.ex.listed = 0;
        for (int peer = 1; peer < C; ++peer) cluster.map_shared_rank(&S, peer)->ex.cut = c;
      }
    }
    if (all) return;
    row_sync();
    cut = S.ex.cut;
  }

  // ---- the draw: kept weight of every run, then the run and the token ------------------------------------------------
  auto run_vals = [&](int r, float (&x)[8]) {
    __align__(16) T raw[8];
    const uint4* src = reinterpret_cast<const uint4*>(vals + r * kRun + lane * 8);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(raw)[i] = src[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f(raw[e]);
  };
  uint32_t ties_before = 0;                      // tokens equal to the cut in front of this CTA's part
  if (cut.partial) {
    uint32_t mine = 0;
    for (int r = warp; r < runs; r += kSampleWarps) {
      float x[8];
      run_vals(r, x);
      uint32_t ties = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) ties += x[e] == cut.x;
      ties = __reduce_add_sync(0xFFFFFFFFu, ties);
      if (lane == 0) S.run_ties[r] = ties;
      mine += ties;
    }
    const uint32_t total = (uint32_t)block_sum(lane == 0 ? mine : 0);
    if (tid < C) cluster.map_shared_rank(&S, tid)->ex.ties[rank] = total;
    row_sync();
    for (int i = 0; i < rank; ++i) ties_before += S.ex.ties[i];
    if (warp == 0) {                             // running counts over the runs
      uint32_t carry = ties_before;
      for (int r0 = 0; r0 < runs; r0 += 32) {
        const uint32_t own = r0 + lane < runs ? S.run_ties[r0 + lane] : 0;
        uint32_t upto = own;
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
          if (lane >= o) upto += y;
        }
        if (r0 + lane < runs) S.run_ties[r0 + lane] = carry + upto - own;
        carry += __shfl_sync(0xFFFFFFFFu, upto, 31);
      }
    }
    __syncthreads();
  }
  auto kept_of = [&](int r, float (&x)[8]) {      // this lane's values of a run, and which of them are kept
    run_vals(r, x);
    uint32_t keep = 0;
    if (!cut.partial) {
#pragma unroll
      for (int e = 0; e < 8; ++e) keep |= (x[e] > cut.x || x[e] == cut.x ? 1u : 0u) << e;
      return keep;
    }
    uint32_t own = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) own += x[e] == cut.x;
    uint32_t upto = own;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += y;
    }
    uint32_t tie_rank = S.run_ties[r] + upto - own;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool tie = x[e] == cut.x;
      keep |= (x[e] > cut.x || (tie && tie_rank < cut.ties) ? 1u : 0u) << e;
      tie_rank += tie;
    }
    return keep;
  };
  auto run_weights = [&](const float (&x)[8], uint32_t keep, uint64_t (&w)[8]) {
    uint64_t sum = 0;
#pragma unroll
    for (int e0 = 0; e0 < 8; e0 += 4) {
#pragma unroll
      for (int e = e0; e < e0 + 4; ++e) w[e] = weigh(x[e]);
#pragma unroll
      for (int e = e0; e < e0 + 4; ++e) {
        if (!(keep >> e & 1) || w[e] < fewest) w[e] = 0;
        sum += w[e];
      }
    }
    return sum;
  };
  uint64_t mine = 0;
  for (int r = warp; r < runs; r += kSampleWarps) {
    float x[8];
    uint32_t keep = kept_of(r, x);
    uint64_t sum = 0;
    if (__reduce_max_sync(0xFFFFFFFFu, __popc(keep)) > 2) {
      uint64_t w[8];
      sum = run_weights(x, keep, w);
    } else {                                     // few are: one after the other is shorter than all side by side
      for (; keep != 0; keep &= keep - 1) {
        const uint64_t w = weigh(to_f(vals[r * kRun + lane * 8 + __ffs(keep) - 1]));
        sum += w < fewest ? 0 : w;
      }
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) S.run_mass[r] = sum;
    mine += sum;
  }
  const uint64_t own = block_sum(lane == 0 ? mine : 0);
  if (tid < C) cluster.map_shared_rank(&S, tid)->ex.kept[rank] = own;
  row_sync();
  uint64_t total = 0, before = 0;
  for (int i = 0; i < C; ++i) {
    if (i < rank) before += S.ex.kept[i];
    total += S.ex.kept[i];
  }
  const double target = u * (double)total;
  if (warp != 0 || !((double)(before + own) > target) || (double)before > target) return;
  int run = -1;
  for (int r0 = 0; r0 < runs && run < 0; r0 += 32) {
    const uint64_t m = r0 + lane < runs ? S.run_mass[r0 + lane] : 0;
    uint64_t upto = m;
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += y;
    }
    const uint32_t vote = __ballot_sync(0xFFFFFFFFu, (double)(before + upto) > target);
    const int who = vote ? __ffs(vote) - 1 : 31;
    if (vote) run = r0 + who;
    before += __shfl_sync(0xFFFFFFFFu, vote ? upto - m : upto, who);
  }
  if (run < 0) return;
  float x[8];
  uint64_t w[8];
  const uint32_t keep = kept_of(run, x);
  const uint64_t sum = run_weights(x, keep, w);
  uint64_t upto = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= o) upto += y;
  }
  before += upto - sum;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (w[e] > 0 && (double)(before + w[e]) > target && !((double)before > target)) {
      chosen(base + run * kRun + lane * 8 + e, x[e], total);
    }
    before += w[e];
  }
}

template <typename T>
int launch_sample(SampleParams P, int64_t batch, cudaStream_t s) {
  // CTAs of a row: enough that two parts fit a multiprocessor side by side, and more while all rows still run at once and a
  // CTA keeps 2048 tokens (one row of 128256: 8 CTAs 13.9 us, 4 CTAs 15.5; 64 rows, top-p: 4 CTAs 80 us, 8 CTAs 125; 32000 fp32
  // logits, 64 rows: 1 CTA 42 us, 2 CTAs 33, 4 CTAs 35, 8 CTAs 76; 256 rows: 1 or 2 CTAs 76 us, 4 CTAs 109)
  int cluster = 1;
  while (cluster < kMaxCluster && (P.vocab > (int64_t)kMaxPart * cluster || P.vocab * (int64_t)sizeof(T) > 80 * 1024 * cluster)) cluster *= 2;
  while (cluster < kMaxCluster && P.vocab > 2048 * cluster && batch * cluster <= sm_count()) cluster *= 2;
  P.part = (int)(ceil_div64(ceil_div64(P.vocab, cluster), kRun) * kRun);
  const size_t smem = (sizeof(SampleShared) + 15) / 16 * 16 + (size_t)P.part * sizeof(T);
  static bool attr_set[64] = {false};
  int dev = 0;
  BSB_CUDA(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    BSB_CUDA(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((sizeof(SampleShared) + 15) / 16 * 16 + kMaxPart * sizeof(T))));
    attr_set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * cluster));
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = g_pdl_enabled ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  BSB_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T>, P));
  return check_launch("sample_kernel");
}

}  // namespace
}  // namespace bsb

using namespace bsb;

extern "C" {

int bsb_sample_step(const void* logits, int64_t batch, int64_t vocab, int64_t row_stride, int32_t dtype, const float* uniforms,
                    const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, int64_t* tokens, int64_t* pos,
                    float* logprobs, void* stream) {
  BSB_CHECK_ARG(batch >= 0 && vocab >= 1 && row_stride >= vocab, "bad shape");
  BSB_CHECK_ARG(dtype == BSB_F16 || dtype == BSB_BF16 || dtype == BSB_F32, "sample_step: fp16, bf16 or fp32 logits (got dtype code %d)", dtype);
  if (batch == 0) return BSB_OK;
  BSB_CHECK_ARG(logits && uniforms && tokens, "NULL buffer");
  if (batch > (1 << 24) || vocab > kMaxVocab) {
    set_error("sample_step: at most %d rows of %d tokens", 1 << 24, kMaxVocab);
    return BSB_ELIMIT;
  }
  SampleParams P;
  P.logits = logits;
  P.vocab = vocab;
  P.stride = row_stride;
  P.uniforms = uniforms;
  P.temperature = temperature;
  P.top_k = top_k;
  P.top_p = top_p;
  P.min_p = min_p;
  P.tokens = tokens;
  P.pos = pos;
  P.logprobs = logprobs;
  P.unit = unit_of(vocab);
  if (dtype == BSB_F16) return launch_sample<__half>(P, batch, (cudaStream_t)stream);
  if (dtype == BSB_BF16) return launch_sample<__nv_bfloat16>(P, batch, (cudaStream_t)stream);
  return launch_sample<float>(P, batch, (cudaStream_t)stream);
}

}  // extern "C"
