// The next token of every row: temperature, top-k, top-p and min-p on the logits, drawn with a given uniform number.
//
// Weights.  w(x) = 2^((x - max) log2(e) / T), as an integer in units of 2^-S: sums of integers do not depend on their order,
// so the kept set and the token are the same bits run to run whatever adds them up, and the cumulative weights next to a
// border are right to 2^-S per term (S = 44 for a 128256-token vocabulary, 2^62 is never passed).  The exponential is
// evaluated in 64 bits from a table of 256 powers and a polynomial on |r| <= 1/512 (table-driven evaluation after Tang, 1989;
// the remainder (ln 2 / 512)^5 / 120 is 4e-17).
// Kept set.  All three filters cut the tokens sorted by logit (ties: lowest index first) behind some place, so the set is
// given by a key and a number of tokens with exactly that key: no sort, a radix descent over the key's bits finds them.
// Draw.  The first index in vocabulary order whose cumulative kept weight exceeds u times the total.
#include <climits>
#include <math.h>

#include "common.cuh"
#include "numeric.cuh"

namespace bsb {
namespace {

constexpr int kSampleThreads = 1024;

// order-preserving key of a logit: NaN counts as -infinity, -0 as +0
__device__ __forceinline__ uint32_t key_of(float x) {
  x = x == x ? x + 0.f : -INFINITY;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

struct Weigher {
  const double* powers;   // 2^(i/256)
  double per_logit;       // log2(e) / T
  float top;              // the row's maximum
  int unit;               // S
  __device__ __forceinline__ double exponent(float x) const { return x == top ? 0.0 : ((double)x - (double)top) * per_logit; }
  __device__ __forceinline__ uint64_t operator()(uint32_t key) const {
    const double t = exponent(logit_of(key));
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

// One CTA per row, every pass reads the row again.
template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const T* __restrict__ logits, int64_t V, int64_t stride, const float* __restrict__ uniforms,
                                                                const float* __restrict__ temperature, const int32_t* __restrict__ top_k,
                                                                const float* __restrict__ top_p, const float* __restrict__ min_p,
                                                                int64_t* __restrict__ tokens, int64_t* __restrict__ pos, float* __restrict__ logprobs, int unit) {
  __shared__ double s_powers[256];
  __shared__ uint64_t s_mass[256], s_red[32], s_pick[4];
  __shared__ uint32_t s_count[256], s_redk[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t b = blockIdx.x;
  if (tid < 256) s_powers[tid] = exp2(tid / 256.0);
  pdl_wait();   // no early release: this kernel writes *pos, which the dense decode attention reads in front of its own wait
  const T* row = logits + b * stride;
  uint32_t top = 0;
  int64_t at = LLONG_MAX;
  for (int64_t i = tid; i < V; i += kSampleThreads) {
    const uint32_t key = key_of(to_f(row[i]));
    if (key > top) { top = key; at = i; }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const uint32_t ok = __shfl_xor_sync(0xFFFFFFFFu, top, o);
    const int64_t oa = __shfl_xor_sync(0xFFFFFFFFu, at, o);
    if (ok > top || (ok == top && oa < at)) { top = ok; at = oa; }
  }
  if (lane == 0) { s_redk[warp] = top; s_red[warp] = (uint64_t)at; }
  __syncthreads();
  for (int w = 0; w < 32; ++w)
    if (s_redk[w] > top || (s_redk[w] == top && (int64_t)s_red[w] < at)) { top = s_redk[w]; at = (int64_t)s_red[w]; }
  __syncthreads();
  const float temp = temperature ? temperature[b] : 1.f;
  const float top_x = logit_of(top);
  if (b == 0 && tid == 0 && pos != nullptr) *pos += 1;
  if (!(temp > 0.f) || top_x == -INFINITY) {   // greedy; a row that its mask leaves nothing of: token 0, as the greedy step gives
    if (tid == 0) {
      tokens[b] = top_x == -INFINITY ? 0 : at;
      if (logprobs) logprobs[b] = top_x == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  const Weigher weigh{s_powers, 1.4426950408889634074 / (double)temp, top_x, unit};

  // kept: key > cut_key, or key == cut_key and among the first cut_ties such tokens
  uint32_t cut_key = 0;
  uint64_t cut_ties = (uint64_t)V;
  auto descend = [&](bool by_mass, double want, uint64_t limit_ties, uint32_t limit_key) {
    // the key at which the running count (or weight) from the top reaches `want`, and what lies above it
    uint32_t prefix = 0, mask = 0;
    uint64_t above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) { s_count[tid] = 0; s_mass[tid] = 0; }
      __syncthreads();
      for (int64_t i = tid; i < V; i += kSampleThreads) {
        const uint32_t key = key_of(to_f(row[i]));
        if ((key & mask) != prefix || key < limit_key) continue;
        atomicAdd(&s_count[(key >> shift) & 255], 1u);
        if (by_mass && key > limit_key) atomicAdd((unsigned long long*)&s_mass[(key >> shift) & 255], (unsigned long long)weigh(key));
      }
      __syncthreads();
      if (by_mass && tid == 0 && (limit_key & mask) == prefix) s_mass[(limit_key >> shift) & 255] += limit_ties * weigh(limit_key);
      __syncthreads();
      if (tid == 0) {
        int bin = 255, last = -1;
        uint64_t sum = above;
        for (; bin >= 0; --bin) {
          if (s_count[bin] == 0) continue;
          last = bin;
          const uint64_t v = by_mass ? s_mass[bin] : s_count[bin];
          if ((double)(sum + v) >= want) break;
          if (bin > 0) sum += v;
        }
        s_pick[0] = bin >= 0 ? bin : last;
        s_pick[1] = bin >= 0 ? sum : sum - 0;
        s_pick[2] = bin >= 0;
        s_pick[3] = s_count[s_pick[0]];
      }
      __syncthreads();
      prefix |= (uint32_t)s_pick[0] << shift;
      mask |= 255u << shift;
      above = s_pick[1];
      const bool found = s_pick[2] != 0;
      const uint64_t ties = s_pick[3];
      __syncthreads();
      if (!found) return;   // rounding: the whole set is smaller than `want`; nothing is cut
      if (shift == 0) {
        double r = want - (double)above;
        if (by_mass) r = ceil(r / (double)weigh(prefix));
        cut_key = prefix;
        cut_ties = r < 1.0 ? 1 : (r > (double)ties ? ties : (uint64_t)r);
        if (prefix == limit_key && cut_ties > limit_ties) cut_ties = limit_ties;
      }
    }
  };
  const int32_t k = top_k ? top_k[b] : 0;
  if (k > 0 && k < V) descend(false, (double)k, (uint64_t)V, 0);
  const float p = top_p ? top_p[b] : 1.f;
  if (p < 1.f) {
    uint64_t sum = 0;
    for (int64_t i = tid; i < V; i += kSampleThreads) {
      const uint32_t key = key_of(to_f(row[i]));
      if (key > cut_key) sum += weigh(key);
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) s_red[warp] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < 32; ++w) sum += s_red[w];
    __syncthreads();
    if (cut_key > 0) sum += cut_ties * weigh(cut_key);
    const double want = (double)p * (double)sum;
    if (want > 0.0) descend(true, want, cut_ties, cut_key);
    else { cut_key = top; cut_ties = 1; }
  }
  const float mp = min_p ? min_p[b] : 0.f;
  const double least = mp > 0.f ? (double)fminf(mp, 1.f) * (double)(1ull << unit) : 0.0;   // the likeliest token always stays

  // kept weight in vocabulary order: total first, then the place where it passes u * total
  uint64_t total = 0;
  double target = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    uint64_t before = 0, ties_before = 0;
    for (int64_t base = 0; base < V; base += kSampleThreads) {
      const int64_t i = base + tid;
      uint32_t key = 0;
      if (i < V) key = key_of(to_f(row[i]));
      const bool tie = i < V && key == cut_key;
      const uint32_t vote = __ballot_sync(0xFFFFFFFFu, tie);
      if (lane == 0) s_redk[warp] = __popc(vote);
      __syncthreads();
      uint64_t rank = ties_before + __popc(vote & ((1u << lane) - 1));
      for (int w = 0; w < 32; ++w) { if (w < warp) rank += s_redk[w]; ties_before += s_redk[w]; }
      uint64_t w8 = 0;
      if (i < V && (key > cut_key || (tie && rank < cut_ties))) {
        w8 = weigh(key);
        if ((double)w8 < least) w8 = 0;
      }
      uint64_t upto = w8;
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += x;
      }
      if (lane == 31) s_red[warp] = upto;
      __syncthreads();
      uint64_t chunk = 0;
      for (int w = 0; w < 32; ++w) { if (w < warp) upto += s_red[w]; chunk += s_red[w]; }
      if (pass == 1 && w8 > 0 && (double)(before + upto) > target && !((double)(before + upto - w8) > target)) {
        tokens[b] = i;
        if (logprobs) logprobs[b] = (float)(weigh.exponent(logit_of(key)) * 0.6931471805599453094 - log((double)total / (double)(1ull << unit)));
      }
      before += chunk;
      __syncthreads();
    }
    if (pass == 0) {
      total = before;
      const float u = uniforms[b];
      target = (u > 0.f ? (double)fminf(u, 0.99999994f) : 0.0) * (double)total;
    }
  }
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
  if (batch > 65535 || vocab > (1 << 20)) {
    set_error("sample_step: at most 65535 rows of %d tokens", 1 << 20);
    return BSB_ELIMIT;
  }
  int unit = 50;                                        // vocab * 2^unit <= 2^62
  while (unit > 0 && (vocab << unit) > (1ll << 62)) --unit;
  auto go = [&](auto kernel, auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_pdl(kernel, dim3((unsigned)batch), dim3(kSampleThreads), 0, (cudaStream_t)stream, (const T*)logits, vocab, row_stride, uniforms,
                      temperature, top_k, top_p, min_p, tokens, pos, logprobs, unit);
  };
  if (dtype == BSB_F16) BSB_CUDA(go(sample_kernel<__half>, (__half*)nullptr));
  else if (dtype == BSB_BF16) BSB_CUDA(go(sample_kernel<__nv_bfloat16>, (__nv_bfloat16*)nullptr));
  else BSB_CUDA(go(sample_kernel<float>, (float*)nullptr));
  return check_launch("sample_kernel");
}

}  // extern "C"
