// The next token of every row: temperature, top-k, top-p and min-p on the logits, drawn with a given uniform number.
//
// Weights.  w(x) = 2^((x - max) log2(e) / T), as an integer in units of 2^-S: sums of integers do not depend on their order,
// so the kept set and the token are the same bits run to run whatever adds them up, and the cumulative weights next to a
// border are right to 2^-S per term (S = 45 for a 128256-token vocabulary, 2^62 is never passed).  The exponential is
// evaluated in 64 bits from a table of 256 powers and a polynomial on |r| <= 1/512 (table-driven evaluation after Tang, 1989;
// the remainder (ln 2 / 512)^5 / 120 is 4e-17).
// Kept set.  All three filters cut the tokens sorted by logit (ties: lowest index first) behind some place, so the set is
// given by a key and a number of tokens with exactly that key.  No sort: a histogram over equal steps of (max - x) / T finds
// the step in which the count (or weight) from the top passes what is wanted; the few tokens of that step are gathered and
// compared with one another.  A step that holds too many (near-equal logits) is taken apart by the bits of its keys first.
// Draw.  The first index in vocabulary order whose cumulative kept weight exceeds u times the total: weights of runs of 256
// tokens, the run by a scan, the token inside it by one warp.
//
// A row is a cluster of up to 8 CTAs, each with its part of the row as keys in shared memory: the logits are read once, and
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
constexpr int kList = 256;                      // tokens that are compared with one another
constexpr float kSpan = 32.f;                   // the histogram's steps cover this many temperatures below the maximum

// order-preserving keys: NaN counts as -infinity, -0 as +0; 0 stands for no token
template <typename T> struct Keys;
template <> struct Keys<float> {
  using K = uint32_t;
  static constexpr int bits = 32;
  static __device__ __forceinline__ K of(float x) {
    x = x == x ? x + 0.f : -INFINITY;
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static __device__ __forceinline__ float logit(K key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
};
template <uint16_t MINUS_INF> struct Keys16 {
  using K = uint16_t;
  static constexpr int bits = 16;
  static __device__ __forceinline__ K of_bits(uint32_t b) {
    const uint32_t mag = b & 0x7FFFu;
    b = mag > (MINUS_INF & 0x7FFFu) ? MINUS_INF : mag == 0 ? 0u : b;
    return (K)(b & 0x8000u ? ~b : b | 0x8000u);
  }
  static __device__ __forceinline__ uint32_t bits_of(K key) { return key & 0x8000u ? key & 0x7FFFu : (uint32_t)(uint16_t)~key; }
};
template <> struct Keys<__half> : Keys16<0xFC00> {
  static __device__ __forceinline__ K of(__half x) { return of_bits(__half_as_ushort(x)); }
  static __device__ __forceinline__ float logit(K key) { return __half2float(__ushort_as_half((unsigned short)bits_of(key))); }
};
template <> struct Keys<__nv_bfloat16> : Keys16<0xFF80> {
  static __device__ __forceinline__ K of(__nv_bfloat16 x) { return of_bits(__bfloat16_as_ushort(x)); }
  static __device__ __forceinline__ float logit(K key) { return __uint_as_float(bits_of(key) << 16); }
};

struct Weigher {
  const double* powers;   // 2^(i/256)
  double per_logit;       // log2(e) / T
  float top;              // the row's maximum
  int unit;               // S
  __device__ __forceinline__ double exponent(float x) const { return x == top ? 0.0 : ((double)x - (double)top) * per_logit; }
  __device__ __forceinline__ uint64_t operator()(float x) const {
    const double t = exponent(x);
    if (!(t > -(double)(unit + 2))) return 0;   // below half a unit; also -infinity, and NaN from 0 * infinity
    const double magic = 6755399441055744.0;    // 1.5 * 2^52: adding it leaves the nearest integer in the low word
    const double s = fma(t, 256.0, magic);
    const int i = __double2loint(s);
    const double r = fma(s - magic, -1.0 / 256.0, t);
    const double ln2 = 0.6931471805599453094;
    double p = fma(r, ln2 * ln2 * ln2 * ln2 / 24.0, ln2 * ln2 * ln2 / 6.0);
    p = fma(r, p, ln2 * ln2 / 2.0);
    p = fma(r, p, ln2);
    p = fma(r, p, 1.0);
    const double w = powers[i & 255] * p * __hiloint2double((1023 + unit + (i >> 8)) << 20, 0);
    return (uint64_t)__double_as_longlong(w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;   // rounded to a whole number of units
  }
};

struct Found {            // the bin in which the count (or weight) from the top reaches what is wanted
  uint64_t above_mass;    // of the bins in front of it
  uint32_t above, count;  // tokens in front of it, tokens in it
  int bin;
};
struct Cut {              // kept: key > `key`, or key == `key` and among the first `ties` such tokens (all of them: !partial)
  uint32_t key, ties, partial;
};

// what the CTAs of a cluster tell one another; peers write into it
struct Exchange {
  uint64_t top[kMaxCluster], mass[kMaxCluster], sum[kMaxCluster], kept[kMaxCluster];
  uint32_t count[kMaxCluster], ties[kMaxCluster];
  Found found;
  Cut cut;
  uint32_t listed;        // the leader's list
};

struct SampleShared {
  double powers[256];
  uint32_t hist[4][kBins];              // count, and the weight in three limbs of 17 bits
  uint64_t bin_mass[kBins];             // of the bins this CTA adds up for the cluster
  uint32_t bin_count[kBins];
  uint64_t list_w[kList];
  uint32_t list_key[kList], own_key[kList];
  uint64_t run_mass[kMaxPart / kRun];
  uint32_t run_ties[kMaxPart / kRun];
  uint64_t red[kSampleWarps];
  uint32_t own_listed, list_at;
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
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleParams P) {
  using KT = Keys<T>;
  using K = typename KT::K;
  extern __shared__ __align__(16) uint8_t smem[];
  SampleShared& S = *reinterpret_cast<SampleShared*>(smem);
  K* keys = reinterpret_cast<K*>(smem + ((sizeof(SampleShared) + 15) / 16) * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t b = blockIdx.x / C;
  const int64_t base = (int64_t)rank * P.part;
  const int n = (int)max(min(P.vocab - base, (int64_t)P.part), (int64_t)0);
  const int runs = (n + kRun - 1) / kRun;

  if (tid < 256) S.powers[tid] = exp2(tid / 256.0);
  if (tid == 0) S.ex.listed = 0;
  cluster.sync();   // every CTA of the row runs before another one writes into its shared memory
  pdl_wait();   // no early release: this kernel writes *pos, which the dense decode attention reads in front of its own wait

  // ---- the row's keys, its maximum and where it is first -----------------------------------------------------------
  const T* row = (const T*)P.logits + b * P.stride + base;
  uint64_t best = 0;   // key in front, then the complement of the index: the largest is the first maximum
  auto meet = [&](K key, int i) {
    const uint64_t v = (uint64_t)key << 32 | (0xFFFFFFFFu - (uint32_t)(base + i));
    best = v > best ? v : best;
  };
  {
    constexpr int kPer = 16 / sizeof(T);
    const bool aligned = reinterpret_cast<uintptr_t>(row) % 16 == 0;
    const int nv = aligned ? n / kPer : 0;
    for (int i = tid; i < nv; i += kSampleThreads) {
      const uint4 raw = reinterpret_cast<const uint4*>(row)[i];
      const T* x = reinterpret_cast<const T*>(&raw);
      uint4 packed;
      K* k = reinterpret_cast<K*>(&packed);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        k[e] = KT::of(x[e]);
        meet(k[e], i * kPer + e);
      }
      reinterpret_cast<uint4*>(keys)[i] = packed;
    }
    for (int i = nv * kPer + tid; i < runs * kRun; i += kSampleThreads) {
      const K k = i < n ? KT::of(row[i]) : (K)0;
      keys[i] = k;
      if (i < n) meet(k, i);
    }
  }
  auto block_sum = [&](uint64_t v, bool is_max) {
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t x = __shfl_xor_sync(0xFFFFFFFFu, v, o);
      v = is_max ? (x > v ? x : v) : v + x;
    }
    __syncthreads();
    if (lane == 0) S.red[warp] = v;
    __syncthreads();
    v = S.red[0];
#pragma unroll
    for (int w = 1; w < kSampleWarps; ++w) v = is_max ? (S.red[w] > v ? S.red[w] : v) : v + S.red[w];
    return v;
  };
  best = block_sum(best, true);
  if (tid < C) cluster.map_shared_rank(&S, tid)->ex.top[rank] = best;
  cluster.sync();
  for (int i = 0; i < C; ++i) best = S.ex.top[i] > best ? S.ex.top[i] : best;
  const K top = (K)(best >> 32);
  const float top_x = KT::logit(top);
  const float temp = P.temperature ? P.temperature[b] : 1.f;
  if (b == 0 && rank == 0 && tid == 0 && P.pos != nullptr) *P.pos += 1;
  if (!(temp > 0.f) || top_x == -INFINITY) {   // greedy; a row that its mask leaves nothing of: token 0, as the greedy step gives
    if (rank == 0 && tid == 0) {
      P.tokens[b] = top_x == -INFINITY ? 0 : (int64_t)(0xFFFFFFFFu - (uint32_t)best);
      if (P.logprobs) P.logprobs[b] = top_x == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  const Weigher weigh{S.powers, 1.4426950408889634074 / (double)temp, top_x, P.unit};

  // ---- the kept set ------------------------------------------------------------------------------------------------
  const float steps = (float)kBins / (kSpan * temp);
  auto bin_of = [&](K key) {   // never falls from a higher key to a lower one
    if (key == top) return 0;
    const float q = (top_x - KT::logit(key)) * steps;
    return q < (float)(kBins - 1) ? (int)q : kBins - 1;
  };
  // a subset of the tokens: a bin (or it and those in front of it), key bits, nothing below `floor`
  struct Part { int bin; bool upto; uint32_t mask, bits, floor; };
  auto in_part = [&](K key, const Part& p) {
    if (key < p.floor || key == 0 || (key & p.mask) != p.bits) return false;
    if (p.bin < 0) return true;
    const int q = bin_of(key);
    return p.upto ? q <= p.bin : q == p.bin;
  };
  auto clear = [&]() {
    for (int i = tid; i < 4 * kBins; i += kSampleThreads) (&S.hist[0][0])[i] = 0;
    __syncthreads();
  };
  auto add_mass = [&](int q, uint64_t w) {
    atomicAdd(&S.hist[1][q], (uint32_t)w & 0x1FFFFu);
    atomicAdd(&S.hist[2][q], (uint32_t)(w >> 17) & 0x1FFFFu);
    atomicAdd(&S.hist[3][q], (uint32_t)(w >> 34));
  };
  // the cluster's histogram, added up by bins, and the bin where `want` (tokens, or weight in units) is reached
  auto find = [&](bool by_mass, double want) {
    cluster.sync();                              // every CTA's histogram is complete
    const int slice = kBins / C, first = rank * slice;
    uint64_t mass = 0;
    uint32_t count = 0;
    for (int i = tid; i < slice; i += kSampleThreads) {
      uint64_t m = 0;
      uint32_t c = 0;
      for (int p = 0; p < C; ++p) {
        const SampleShared* peer = cluster.map_shared_rank(&S, p);
        c += peer->hist[0][first + i];
        if (by_mass) m += (uint64_t)peer->hist[1][first + i] + ((uint64_t)peer->hist[2][first + i] << 17) + ((uint64_t)peer->hist[3][first + i] << 34);
      }
      S.bin_count[i] = c;
      S.bin_mass[i] = m;
      count += c;
      mass += m;
    }
    mass = block_sum(mass, false);
    count = (uint32_t)block_sum(count, false);
    if (tid < C) {
      Exchange& ex = cluster.map_shared_rank(&S, tid)->ex;
      ex.mass[rank] = mass;
      ex.count[rank] = count;
    }
    cluster.sync();
    uint64_t m = 0;
    uint32_t c = 0;
    int owner = 0;
    for (; owner < C - 1; ++owner) {
      const double upto = by_mass ? (double)(m + S.ex.mass[owner]) : (double)(c + S.ex.count[owner]);
      if (upto >= want) break;
      m += S.ex.mass[owner];
      c += S.ex.count[owner];
    }
    if (rank == owner && warp == 0) {            // inside the slice: each lane a stretch of bins, then the stretch bin by bin
      const int each = slice / 32;
      uint64_t lm = 0;
      uint32_t lc = 0;
      for (int i = 0; i < each; ++i) { lm += S.bin_mass[lane * each + i]; lc += S.bin_count[lane * each + i]; }
      uint64_t um = lm;
      uint32_t uc = lc;
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, um, o);
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, uc, o);
        if (lane >= o) { um += x; uc += y; }
      }
      const bool reached = (by_mass ? (double)(m + um) : (double)(c + uc)) >= want;
      const uint32_t vote = __ballot_sync(0xFFFFFFFFu, reached);
      const int who = vote ? __ffs(vote) - 1 : 31;
      if (lane == who) {
        m += um - lm;
        c += uc - lc;
        int i = lane * each;
        for (; i < (lane + 1) * each - 1; ++i) {
          if ((by_mass ? (double)(m + S.bin_mass[i]) : (double)(c + S.bin_count[i])) >= want) break;
          m += S.bin_mass[i];
          c += S.bin_count[i];
        }
        const Found f{m, c, S.bin_count[i], first + i};
        for (int p = 0; p < C; ++p) cluster.map_shared_rank(&S, p)->ex.found = f;
      }
    }
    cluster.sync();
    return S.ex.found;
  };
  // all tokens of a part (no more than kList) into the leader's list, with their weights; the caller knows how many
  auto gather = [&](const Part& part) {
    if (tid == 0) S.own_listed = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
      const K key = keys[i];
      if (in_part(key, part)) {
        const uint32_t at = atomicAdd(&S.own_listed, 1u);
        if (at < kList) S.own_key[at] = key;
      }
    }
    __syncthreads();
    SampleShared* leader = cluster.map_shared_rank(&S, 0);
    if (tid == 0 && S.own_listed > 0) S.list_at = atomicAdd(&leader->ex.listed, S.own_listed);
    __syncthreads();
    for (uint32_t i = tid; i < min(S.own_listed, (uint32_t)kList); i += kSampleThreads) {
      const uint32_t at = S.list_at + i;
      if (at < kList) {
        leader->list_key[at] = S.own_key[i];
        leader->list_w[at] = weigh(KT::logit((K)S.own_key[i]));
      }
    }
    cluster.sync();
  };
  // The leader compares the listed tokens with one another.  By count: the cut leaves `k` of them.  By weight: the cut behind
  // the token with which the weight from the top reaches share * (weight of what `cut` leaves of the list), or `want`.
  auto refine = [&](bool by_count, uint32_t k, bool by_mass, double share, double want, uint64_t above_mass, Cut cut) {
    if (rank == 0) {
      const int m = (int)min(S.ex.listed, (uint32_t)kList);
      int lanes = 1;                             // threads that share a token's comparisons
      while (lanes < 32 && lanes * 2 * m <= kSampleThreads) lanes *= 2;
      const int i = tid / lanes, sub = tid % lanes;
      const uint32_t key = i < m ? S.list_key[i] : 0;
      const uint64_t w = i < m ? S.list_w[i] : 0;
      uint32_t higher = 0, equal = 0;
      uint64_t heavier = 0;
      if (i < m)
        for (int j = sub; j < m; j += lanes) {
          const uint32_t other = S.list_key[j];
          higher += other > key;
          equal += other == key;
          heavier += other > key ? S.list_w[j] : 0;
        }
      for (int o = 1; o < lanes; o <<= 1) {
        higher += __shfl_xor_sync(0xFFFFFFFFu, higher, o);
        equal += __shfl_xor_sync(0xFFFFFFFFu, equal, o);
        heavier += __shfl_xor_sync(0xFFFFFFFFu, heavier, o);
      }
      if (tid == 0) S.ex.cut = cut;
      __syncthreads();
      if (by_count && i < m && higher < k && k <= higher + equal) S.ex.cut = Cut{key, k - higher, k - higher < equal};
      __syncthreads();
      if (by_mass) {
        if (by_count) {                          // the whole kept set is in the list: its weight
          cut = S.ex.cut;
          uint64_t mine = i < m && sub == 0 && key > cut.key ? w : 0;
          if (i < m && sub == 0 && key == cut.key) {   // the ties' share, by the first listed one of them
            bool first = true;
            for (int j = 0; j < i; ++j) first = first && S.list_key[j] != key;
            if (first) mine = cut.ties * w;
          }
          want = share * (double)block_sum(mine, false);
        }
        if (i < m && sub == 0 && key >= cut.key) {
          const uint32_t ties = key == cut.key ? min(cut.ties, equal) : equal;
          const double before = (double)(above_mass + heavier);
          if (before < want && !((double)(above_mass + heavier + ties * w) < want)) {
            const double r = ceil((want - before) / (double)w);
            const uint32_t left = r < 1.0 ? 1u : r > (double)ties ? ties : (uint32_t)r;
            S.ex.cut = Cut{key, left, left < equal};
          }
        }
        __syncthreads();
      }
      if (tid == 0) {
        const Cut c = S.ex.cut;
        S.ex.listed = 0;
        for (int p = 1; p < C; ++p) cluster.map_shared_rank(&S, p)->ex.cut = c;
      }
    }
    cluster.sync();
    return S.ex.cut;
  };
  // tokens of `part` by the next bits of their keys, highest first, until few enough are left to be listed, or one key
  auto by_bits = [&](Part part, bool by_mass, double want, Found f, Cut cut) {
    for (int shift = KT::bits - 10; f.count > kList;) {
      const uint32_t field = 1023u << shift & (KT::bits == 32 ? 0xFFFFFFFFu : 0xFFFFu);
      clear();
      for (int i = tid; i < n; i += kSampleThreads) {
        const K key = keys[i];
        if (!in_part(key, part)) continue;
        const int q = kBins - 1 - (int)((key & field & ~part.mask) >> shift);
        atomicAdd(&S.hist[0][q], 1u);
        if (by_mass && key > cut.key) add_mass(q, weigh(KT::logit(key)));
      }
      __syncthreads();
      if (by_mass && rank == 0 && tid == 0 && cut.key > 0 && in_part((K)cut.key, part)) {
        const int q = kBins - 1 - (int)((cut.key & field & ~part.mask) >> shift);
        const uint64_t w = weigh(KT::logit((K)cut.key)) * cut.ties;
        S.hist[1][q] += (uint32_t)w & 0x1FFFFu;   // (a product of up to 62 bits: limbs of 17, 17 and 28; the sums stay below 2^32)
        S.hist[2][q] += (uint32_t)(w >> 17) & 0x1FFFFu;
        S.hist[3][q] += (uint32_t)(w >> 34);
      }
      const Found g = find(by_mass, by_mass ? want - (double)f.above_mass : want - (double)f.above);
      f.above += g.above;
      f.above_mass += g.above_mass;
      f.count = g.count;
      part.bits |= (uint32_t)(kBins - 1 - g.bin) << shift;
      part.mask |= field;
      if (shift == 0) break;
      shift = shift > 10 ? shift - 10 : 0;
    }
    if (f.count <= kList) {
      gather(part);
      return by_mass ? refine(false, 0, true, 0.0, want, f.above_mass, cut) : refine(true, (uint32_t)want - f.above, false, 0.0, 0.0, 0, cut);
    }
    Cut c{part.bits, 0, 0};                       // one key, many tokens
    double left = by_mass ? ceil((want - (double)f.above_mass) / (double)weigh(KT::logit((K)part.bits))) : want - (double)f.above;
    left = fmin(fmax(left, 1.0), (double)f.count);
    c.ties = (uint32_t)left;
    if (c.key == cut.key && cut.ties < c.ties) c.ties = cut.ties;
    c.partial = c.ties < f.count;
    return c;
  };

  Cut cut{0, 0, 0};
  const int32_t k = P.top_k ? P.top_k[b] : 0;
  float p = P.top_p ? P.top_p[b] : 1.f;
  if (p <= 0.f) {                                // the likeliest token alone
    cut = Cut{top, 1, 1};
    p = 1.f;
  } else if (k > 0 && k < P.vocab) {
    clear();
    for (int i = tid; i < n; i += kSampleThreads) atomicAdd(&S.hist[0][bin_of(keys[i])], 1u);
    __syncthreads();
    const Found f = find(false, (double)k);
    if (f.above + f.count <= kList) {            // everything from the top on is few: both cuts at once
      gather(Part{f.bin, true, 0, 0, 0});
      cut = refine(true, (uint32_t)k, p < 1.f, (double)p, 0.0, 0, cut);
      p = 1.f;
    } else {
      const Part part{f.bin, false, 0, 0, 0};
      if (f.count <= kList) {
        gather(part);
        cut = refine(true, (uint32_t)k - f.above, false, 0.0, 0.0, 0, cut);
      } else {
        cut = by_bits(part, false, (double)k, f, cut);
      }
    }
  }
  if (p < 1.f) {
    clear();
    uint64_t mine = 0;
    for (int i = tid; i < n; i += kSampleThreads) {
      const K key = keys[i];
      if (key < cut.key) continue;
      const int q = bin_of(key);
      atomicAdd(&S.hist[0][q], 1u);
      if (key == cut.key) continue;              // its ties' share is added below, once
      const uint64_t w = weigh(KT::logit(key));
      mine += w;
      if (w > 0) add_mass(q, w);
    }
    __syncthreads();
    if (rank == 0 && tid == 0 && cut.key > 0) {
      const uint64_t w = weigh(KT::logit((K)cut.key)) * cut.ties;
      const int q = bin_of((K)cut.key);
      mine += w;
      S.hist[1][q] += (uint32_t)w & 0x1FFFFu;
      S.hist[2][q] += (uint32_t)(w >> 17) & 0x1FFFFu;
      S.hist[3][q] += (uint32_t)(w >> 34);
    }
    mine = block_sum(mine, false);
    if (tid < C) cluster.map_shared_rank(&S, tid)->ex.sum[rank] = mine;
    cluster.sync();
    uint64_t sum = 0;
    for (int i = 0; i < C; ++i) sum += S.ex.sum[i];
    const double want = (double)p * (double)sum;
    const Found f = find(true, want);
    const Part part{f.bin, false, 0, 0, cut.key};
    if (f.count <= kList) {
      gather(part);
      cut = refine(false, 0, true, 0.0, want, f.above_mass, cut);
    } else {
      cut = by_bits(part, true, want, f, cut);
    }
  }
  const float mp = P.min_p ? P.min_p[b] : 0.f;
  const double least = mp > 0.f ? (double)fminf(mp, 1.f) * (double)(1ull << P.unit) : 0.0;   // the likeliest token always stays

  // ---- the draw: kept weight of every run, then the run and the token ------------------------------------------------
  auto run_keys = [&](int r, K (&x)[8]) {
    const uint4* src = reinterpret_cast<const uint4*>(keys + r * kRun + lane * 8);
#pragma unroll
    for (int i = 0; i < (int)sizeof(K) / 2; ++i) reinterpret_cast<uint4*>(x)[i] = src[i];
  };
  uint32_t ties_before = 0;                      // tokens with the cut's key in front of this CTA's part
  if (cut.partial) {
    uint32_t mine = 0;
    for (int r = warp; r < runs; r += kSampleWarps) {
      __align__(16) K x[8];
      run_keys(r, x);
      uint32_t ties = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) ties += x[e] == cut.key;
      ties = __reduce_add_sync(0xFFFFFFFFu, ties);
      if (lane == 0) S.run_ties[r] = ties;
      mine += ties;
    }
    const uint32_t total = (uint32_t)block_sum(lane == 0 ? mine : 0, false);
    if (tid < C) cluster.map_shared_rank(&S, tid)->ex.ties[rank] = total;
    cluster.sync();
    for (int i = 0; i < rank; ++i) ties_before += S.ex.ties[i];
    if (warp == 0) {                             // running counts over the runs
      uint32_t carry = ties_before;
      for (int r0 = 0; r0 < runs; r0 += 32) {
        const uint32_t own = r0 + lane < runs ? S.run_ties[r0 + lane] : 0;
        uint32_t upto = own;
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
          if (lane >= o) upto += x;
        }
        if (r0 + lane < runs) S.run_ties[r0 + lane] = carry + upto - own;
        carry += __shfl_sync(0xFFFFFFFFu, upto, 31);
      }
    }
    __syncthreads();
  }
  auto run_weights = [&](int r, K (&x)[8], uint64_t (&w)[8]) {
    run_keys(r, x);
    uint32_t tie_rank = 0;
    if (cut.partial) {
      uint32_t own = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) own += x[e] == cut.key;
      uint32_t upto = own;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += y;
      }
      tie_rank = S.run_ties[r] + upto - own;
    }
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool tie = x[e] == cut.key;
      w[e] = 0;
      if (x[e] > cut.key || (tie && x[e] != 0 && (!cut.partial || tie_rank < cut.ties))) {
        w[e] = weigh(KT::logit(x[e]));
        if ((double)w[e] < least) w[e] = 0;
      }
      tie_rank += tie;
      sum += w[e];
    }
    return sum;
  };
  uint64_t mine = 0;
  for (int r = warp; r < runs; r += kSampleWarps) {
    __align__(16) K x[8];
    uint64_t w[8];
    uint64_t sum = run_weights(r, x, w);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) S.run_mass[r] = sum;
    mine += sum;
  }
  const uint64_t own = block_sum(lane == 0 ? mine : 0, false);
  if (tid < C) cluster.map_shared_rank(&S, tid)->ex.kept[rank] = own;
  cluster.sync();
  uint64_t total = 0, before = 0;
  for (int i = 0; i < C; ++i) {
    if (i < rank) before += S.ex.kept[i];
    total += S.ex.kept[i];
  }
  const float u = P.uniforms[b];
  const double target = (u > 0.f ? (double)fminf(u, 0.99999994f) : 0.0) * (double)total;
  if (warp != 0 || !((double)(before + own) > target) || (double)before > target) return;
  int run = -1;
  for (int r0 = 0; r0 < runs && run < 0; r0 += 32) {
    const uint64_t m = r0 + lane < runs ? S.run_mass[r0 + lane] : 0;
    uint64_t upto = m;
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= o) upto += x;
    }
    const uint32_t vote = __ballot_sync(0xFFFFFFFFu, (double)(before + upto) > target);
    const int who = vote ? __ffs(vote) - 1 : 31;
    if (vote) run = r0 + who;
    before += __shfl_sync(0xFFFFFFFFu, vote ? upto - m : upto, who);
  }
  if (run < 0) return;
  __align__(16) K x[8];
  uint64_t w[8];
  const uint64_t sum = run_weights(run, x, w);
  uint64_t upto = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= o) upto += y;
  }
  before += upto - sum;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (w[e] > 0 && (double)(before + w[e]) > target && !((double)before > target)) {
      P.tokens[b] = base + run * kRun + lane * 8 + e;
      if (P.logprobs)
        P.logprobs[b] = (float)(weigh.exponent(KT::logit(x[e])) * 0.6931471805599453094 - log((double)total / (double)(1ull << P.unit)));
    }
    before += w[e];
  }
}

template <typename T>
int launch_sample(SampleParams P, int64_t batch, cudaStream_t s) {
  using K = typename Keys<T>::K;
  // CTAs of a row: as many as its part still keeps a CTA's threads busy for (2048 tokens each)
  int cluster = 1;
  while (cluster < kMaxCluster && P.vocab > 2048 * cluster) cluster *= 2;
  P.part = (int)(ceil_div64(ceil_div64(P.vocab, cluster), kRun) * kRun);
  const size_t smem = (sizeof(SampleShared) + 15) / 16 * 16 + (size_t)P.part * sizeof(K);
  static bool attr_set[64] = {false};
  int dev = 0;
  BSB_CUDA(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    BSB_CUDA(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((sizeof(SampleShared) + 15) / 16 * 16 + kMaxPart * sizeof(K))));
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
  P.unit = 50;                                          // vocab * 2^unit <= 2^62
  while ((vocab << P.unit) > (1ll << 62)) --P.unit;
  if (dtype == BSB_F16) return launch_sample<__half>(P, batch, (cudaStream_t)stream);
  if (dtype == BSB_BF16) return launch_sample<__nv_bfloat16>(P, batch, (cudaStream_t)stream);
  return launch_sample<float>(P, batch, (cudaStream_t)stream);
}

}  // extern "C"
