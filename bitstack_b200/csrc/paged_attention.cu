// One new token per request over a paged key/value cache: rotary embedding of q and k, k and v written into the request's
// page, softmax(q K^T / sqrt(D)) V over the request's pages.
#include <climits>
#include <math.h>

#include "common.cuh"
#include "numeric.cuh"

namespace bsb {
namespace {

// One CTA per (query head, request); a warp takes every fourth position, its lanes share the row.  One pass with the
// running maximum and sum of the softmax; the four warps are joined in shared memory.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_attention_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                              int64_t q_stride, int64_t k_stride, int64_t v_stride, const T* __restrict__ cos_t,
                                                              const T* __restrict__ sin_t, int64_t table_len, const int64_t* __restrict__ positions,
                                                              const int32_t* __restrict__ table, int64_t table_stride, int width, T* __restrict__ k_pages,
                                                              T* __restrict__ v_pages, int64_t num_pages, int64_t k_page_stride, int64_t v_page_stride,
                                                              T* __restrict__ out, int Hq, int Hkv, int page_size, float scale, int* __restrict__ status) {
  constexpr int E = D / 32;
  __shared__ float s_q[D], s_k[D], s_o[4][D], s_m[4], s_l[4];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_enter();
  const int64_t pos = positions[b];
  T* o = out + ((int64_t)b * Hq + h) * D;
  const float nan = __int_as_float(0x7FC00000);
  if (pos < 0) {
    if (tid < D) o[tid] = Pair<T>::one(0.f);
    return;
  }
  if (pos >= table_len || pos >= (int64_t)width * page_size) {
    if (tid < D) o[tid] = Pair<T>::one(nan);
    if (tid == 0) atomicCAS(status, 0, 61);
    return;
  }
  const int g = Hq / Hkv, hk = h / g;
  const T* qs = q + b * q_stride + (int64_t)h * D;
  const T* ks = k + b * k_stride + (int64_t)hk * D;
  const T* vs = v + b * v_stride + (int64_t)hk * D;
  const int32_t* pages = table + b * table_stride;
  for (int i = tid; i < D / 2; i += 128) {
    const float c0 = to_f(cos_t[pos * D + i]), c1 = to_f(cos_t[pos * D + i + D / 2]);
    const float s0 = to_f(sin_t[pos * D + i]), s1 = to_f(sin_t[pos * D + i + D / 2]);
    float x0 = to_f(qs[i]), x1 = to_f(qs[i + D / 2]);
    s_q[i] = (x0 * c0 - x1 * s0) * scale;
    s_q[i + D / 2] = (x1 * c1 + x0 * s1) * scale;
    x0 = to_f(ks[i]);
    x1 = to_f(ks[i + D / 2]);
    s_k[i] = to_f(Pair<T>::one(x0 * c0 - x1 * s0));
    s_k[i + D / 2] = to_f(Pair<T>::one(x1 * c1 + x0 * s1));
  }
  __syncthreads();
  bool bad = false;
  const int page_new = pages[pos / page_size];
  if (page_new < 0 || page_new >= num_pages) bad = true;
  else if (h % g == 0 && tid < D) {
    k_pages[page_new * k_page_stride + ((int64_t)hk * page_size + pos % page_size) * D + tid] = Pair<T>::one(s_k[tid]);
    v_pages[page_new * v_page_stride + ((int64_t)hk * page_size + pos % page_size) * D + tid] = vs[tid];
  }
  float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int64_t p = warp; p <= pos; p += 4) {
    float kv[E], vv[E];
    if (p == pos) {
#pragma unroll
      for (int e = 0; e < E; ++e) { kv[e] = s_k[lane + 32 * e]; vv[e] = to_f(vs[lane + 32 * e]); }
    } else {
      const int page = pages[p / page_size];
      if (page < 0 || page >= num_pages) { bad = true; break; }
      const int64_t row = ((int64_t)hk * page_size + p % page_size) * D;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        kv[e] = to_f(k_pages[page * k_page_stride + row + lane + 32 * e]);
        vv[e] = to_f(v_pages[page * v_page_stride + row + lane + 32 * e]);
      }
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(kv[e], s_q[lane + 32 * e], s);
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, w);
    const float mn = fmaxf(m, s), f = __expf(m - mn), e1 = __expf(s - mn);
    l = l * f + e1;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * f + e1 * vv[e];
    m = mn;
  }
  if (bad) { l = nan; if (lane == 0) atomicCAS(status, 0, 61); }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  if (tid < D) {
    float mm = -INFINITY, ll = 0.f, oo = 0.f;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, s_m[w]);
    for (int w = 0; w < 4; ++w) {
      const float f = s_m[w] == -INFINITY ? 0.f : __expf(s_m[w] - mm);
      ll += s_l[w] * f;
      oo += s_o[w][tid] * f;
      if (s_l[w] != s_l[w]) ll = nan;
    }
    o[tid] = Pair<T>::one(oo / ll);
  }
}

}  // namespace
}  // namespace bsb

using namespace bsb;

extern "C" {

int64_t bsb_paged_attention_scratch_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  if (batch < 0 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || q_heads % kv_heads != 0) return -1;
  return 0;
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
  if (batch > 65535) {
    set_error("paged attention: at most 65535 requests per call (got %d)", batch);
    return BSB_ELIMIT;
  }
  (void)scratch;
  (void)scratch_bytes;
  int* status = device_status_word();
  if (status == nullptr) return BSB_ECUDA;
  const float scale = 1.0f / sqrtf((float)head_dim);
  auto go = [&](auto kernel, auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_pdl(kernel, dim3(q_heads, batch), dim3(128), 0, (cudaStream_t)stream, (const T*)q, (const T*)k, (const T*)v, q_stride, k_stride,
                      v_stride, (const T*)cos_table, (const T*)sin_table, table_len, positions, block_table, table_stride, table_width,
                      (T*)k_pages, (T*)v_pages, num_pages, k_page_stride, v_page_stride, (T*)out, q_heads, kv_heads, page_size, scale, status);
  };
  if (dtype == BSB_F16) BSB_CUDA(head_dim == 128 ? go(paged_attention_kernel<__half, 128>, (__half*)nullptr) : go(paged_attention_kernel<__half, 64>, (__half*)nullptr));
  else BSB_CUDA(head_dim == 128 ? go(paged_attention_kernel<__nv_bfloat16, 128>, (__nv_bfloat16*)nullptr) : go(paged_attention_kernel<__nv_bfloat16, 64>, (__nv_bfloat16*)nullptr));
  return check_launch("paged_attention_kernel");
}

}  // extern "C"
