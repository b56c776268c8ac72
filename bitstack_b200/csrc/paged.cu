// Bookkeeping and cache writes of a paged key/value cache: pages handed out and slots mapped from the requests'
// lengths, pages taken back, rotary embedding of a batch of tokens with their K and V written into pages.
// The reference has no cache of any kind (its model calls are whole-sequence evaluations).
#include <climits>

#include "common.cuh"
#include "numeric.cuh"

namespace bsb {
namespace {

constexpr int kTableThreads = 1024;
constexpr int kTableRows = 8192;         // requests of one call: their prefix sums stay in shared memory
// Longer token lists are written by a second, wider launch (64 requests, one launch against two: 355 tokens 4.5 / 5.7 us, 2148
// tokens 6.6 / 6.0, 8547 tokens 12.2 / 6.4, 21872 tokens 24.6 / 6.8).
constexpr int64_t kTokensInOne = 1536;

// inclusive scan of two counters over the CTA; `tot` receives the totals
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t (*red)[2], int64_t& tot_a, int64_t& tot_b) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xFFFFFFFFu, a, o), y = __shfl_up_sync(0xFFFFFFFFu, b, o);
    if (lane >= o) { a += x; b += y; }
  }
  __syncthreads();   // `red` may still be read from the scan before
  if (lane == 31) { red[warp][0] = a; red[warp][1] = b; }
  __syncthreads();
  if (warp == 0) {
    int64_t x = red[lane][0], y = red[lane][1];
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t p = __shfl_up_sync(0xFFFFFFFFu, x, o), q = __shfl_up_sync(0xFFFFFFFFu, y, o);
      if (lane >= o) { x += p; y += q; }
    }
    red[lane][0] = x;
    red[lane][1] = y;
  }
  __syncthreads();
  if (warp > 0) { a += red[warp - 1][0]; b += red[warp - 1][1]; }
  tot_a = red[31][0];
  tot_b = red[31][1];
}

// largest i in [0, n) with start[i] <= x (start is non-decreasing, start[0] <= x)
__device__ __forceinline__ int row_of(const int32_t* start, int n, int64_t x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// the slot and position of token t of the list: its request is found from the offsets, its position counts from the request's
// first new one (the offset behind the request may have been held at 2^31 - 1), its page is in the table
__device__ __forceinline__ void token_entry(int64_t t, const int32_t* offsets, int batch, const int32_t* new_tokens, const int64_t* last,
                                            const int32_t* table, int64_t table_stride, int page_size, int64_t* slots, int64_t* positions) {
  int64_t slot = -1, pos = -1;
  if (t < offsets[batch]) {
    const int row = row_of(offsets, batch, t);
    const int64_t end = last[row];
    if (end >= 0) {
      pos = end + 1 - new_tokens[row] + (t - offsets[row]);
      const int page = table[row * table_stride + (int)pos / page_size];
      slot = page < 0 ? -1 : (int64_t)page * page_size + (int)pos % page_size;
    }
  }
  slots[t] = slot;
  positions[t] = pos;
}

// One CTA: the whole step is two scans over the requests and a scatter, all of it latency (256 requests of one token: 4.8 us in a
// graph, of which the launch is about half).  lens_out may be lens, and
// free_count_out may be free_count: everything is read before the barriers in front of the writes.
__global__ void __launch_bounds__(kTableThreads) page_tables_kernel(
    const int32_t* lens, const int32_t* __restrict__ new_tokens, int batch, int32_t* __restrict__ table, int64_t table_stride,
    int width, const int32_t* __restrict__ free_pages, const int32_t* free_count, int capacity, int page_size,
    int64_t max_tokens, int64_t* __restrict__ slots, int64_t* __restrict__ positions, int32_t* __restrict__ offsets,
    int64_t* __restrict__ last, int32_t* lens_out, int32_t* free_count_out, int* __restrict__ status) {
  extern __shared__ int32_t s_rows[];    // [batch] pages handed out before the request's own, [batch] pages it holds already
  __shared__ int64_t red[32][2];
  int32_t* s_first = s_rows;
  int32_t* s_held = s_rows + batch;
  pdl_wait();   // no early release: the kernels behind read what this one writes, some of it in front of their own wait
  const int64_t count = min(max(*free_count, 0), capacity);
  int64_t need0 = 0, tok0 = 0, taken = 0;   // totals of the requests before this chunk
  for (int base = 0; base < batch; base += kTableThreads) {
    const int i = base + threadIdx.x;
    int64_t len = 0, add = 0, held = 0, after = 0;
    if (i < batch) {
      len = max(lens[i], 0);
      add = max(new_tokens[i], 0);
      held = (len + page_size - 1) / page_size;
      after = (len + add + page_size - 1) / page_size;
    }
    const bool fits = after <= width && len + add <= INT_MAX;
    const int64_t need = fits ? after - held : 0;
    int64_t upto = need, tok = add, need_tot, tok_tot;
    block_scan2(upto, tok, red, need_tot, tok_tot);
    const bool served = fits && (need == 0 || need0 + upto <= count);
    if (i < batch) {
      // pages of refused requests are not taken; all requests behind the first refused one that need pages are refused too
      s_first[i] = (int32_t)min(need0 + upto - need, count);
      s_held[i] = (int32_t)held;
      offsets[i] = (int32_t)min(tok0 + tok - add, (int64_t)INT_MAX);
      last[i] = served && add > 0 ? len + add - 1 : -1;
      lens_out[i] = (int32_t)(served ? len + add : len);
    }
    taken += served ? need : 0;
    need0 += need_tot;
    tok0 += tok_tot;
  }
  {
    int64_t none = 0, taken_tot, none_tot;
    block_scan2(taken, none, red, taken_tot, none_tot);
    taken = taken_tot;
  }
  if (threadIdx.x == 0) {
    offsets[batch] = (int32_t)min(tok0, (int64_t)INT_MAX);
    *free_count_out = (int32_t)(count - taken);
    if (max_tokens > 0 && tok0 > max_tokens) atomicCAS(status, 0, 63);
  }
  for (int64_t a = threadIdx.x; a < taken; a += kTableThreads) {
    const int row = row_of(s_first, batch, a);
    table[row * table_stride + s_held[row] + (a - s_first[row])] = free_pages[count - 1 - a];
  }
  if (max_tokens > kTokensInOne) return;
  __syncthreads();
  for (int64_t t = threadIdx.x; t < max_tokens; t += kTableThreads)
    token_entry(t, offsets, batch, new_tokens, last, table, table_stride, page_size, slots, positions);
}

__global__ void __launch_bounds__(256) page_tokens_kernel(const int32_t* __restrict__ offsets, int batch, const int32_t* __restrict__ new_tokens,
                                                          const int64_t* __restrict__ last, const int32_t* __restrict__ table,
                                                          int64_t table_stride, int page_size, int64_t max_tokens,
                                                          int64_t* __restrict__ slots, int64_t* __restrict__ positions) {
  pdl_wait();
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (t < max_tokens) token_entry(t, offsets, batch, new_tokens, last, table, table_stride, page_size, slots, positions);
}

// pages of the requests that are done go back on the stack, in the order of the requests and of their pages
__global__ void __launch_bounds__(kTableThreads) release_pages_kernel(const uint8_t* __restrict__ done, int32_t* __restrict__ lens, int batch,
                                                                      const int32_t* __restrict__ table, int64_t table_stride, int width,
                                                                      int32_t* __restrict__ free_pages, int32_t* __restrict__ free_count,
                                                                      int capacity, int page_size, int* __restrict__ status) {
  extern __shared__ int32_t s_rows[];    // [batch] pages given back before the request's own
  __shared__ int64_t red[32][2];
  pdl_wait();
  const int64_t count = min(max(*free_count, 0), capacity);
  int64_t total = 0;
  for (int base = 0; base < batch; base += kTableThreads) {
    const int i = base + threadIdx.x;
    int64_t n = 0, none = 0, n_tot, none_tot;
    if (i < batch && done[i]) n = min((max(lens[i], 0) + (int64_t)page_size - 1) / page_size, (int64_t)width);
    const int64_t mine = n;
    block_scan2(n, none, red, n_tot, none_tot);
    if (i < batch) {
      s_rows[i] = (int32_t)min(total + n - mine, (int64_t)INT_MAX);
      if (done[i]) lens[i] = 0;
    }
    total += n_tot;
  }
  __syncthreads();
  const int64_t put = min(total, capacity - count);
  if (threadIdx.x == 0) {
    *free_count = (int32_t)(count + put);
    if (put < total) atomicCAS(status, 0, 64);
  }
  for (int64_t a = threadIdx.x; a < put; a += kTableThreads) {
    const int row = row_of(s_rows, batch, a);
    free_pages[count + a] = table[row * table_stride + (a - s_rows[row])];
  }
}

// One CTA per token; a thread takes eight pairs (i, i + D/2) of a head: two 16-byte loads, two 16-byte stores, and the
// token's cosines and sines from L1.  Bound by the copy: every byte of q, k and v is read once and written once (2047 tokens of
// 32 / 8 heads of 128: 10.9 us, 4.5 TB/s).  The values are asked for in front of the token's position, which the table rows and
// the destination wait for, and every thread gets the same number of items (12.6 us with 256 threads and 1.5 items each; two tokens per CTA 12.2).
constexpr int kRopeThreads = 512;   // at most; the launch takes as many as give every thread the same number of items
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_paged_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                         int64_t q_stride, int64_t k_stride, int64_t v_stride, const T* __restrict__ cos_t,
                                                         const T* __restrict__ sin_t, int64_t table_len, const int64_t* __restrict__ positions,
                                                         const int64_t* __restrict__ slots, T* __restrict__ q_out, T* __restrict__ k_pages,
                                                         T* __restrict__ v_pages, int64_t num_pages, int64_t k_page_stride,
                                                         int64_t v_page_stride, int Hq, int Hkv, int D, int page_size, int* __restrict__ status) {
  pdl_wait();   // no early release: the dense decode attention reads older cache rows, which may be these pages, in front of its own wait
  const int64_t t = blockIdx.x;
  const int parts = D / 16, items = (Hq + 2 * Hkv) * parts;
  for (int it = threadIdx.x; it < items; it += blockDim.x) {
    const int head = it / parts, c = (it - head * parts) * 8;
    const T* src = head < Hq         ? q + t * q_stride + (int64_t)head * D + c
                   : head < Hq + Hkv ? k + t * k_stride + (int64_t)(head - Hq) * D + c
                                     : v + t * v_stride + (int64_t)(head - Hq - Hkv) * D + c;
    const uint4 lo = __ldcs(reinterpret_cast<const uint4*>(src)), hi = __ldcs(reinterpret_cast<const uint4*>(src + D / 2));
    const int64_t pos = positions[t], slot = slots[t];
    const bool bad = pos >= table_len || slot >= num_pages * page_size;
    if (bad && it == 0) atomicCAS(status, 0, 62);
    const bool turn = pos >= 0 && pos < table_len, keep = slot >= 0 && slot < num_pages * page_size && turn;
    if (head >= Hq && !keep) continue;
    const int64_t page = keep ? slot / page_size : 0, row = keep ? slot % page_size : 0;
    if (head >= Hq + Hkv) {   // v: copied
      T* dst = v_pages + page * v_page_stride + ((int64_t)(head - Hq - Hkv) * page_size + row) * D + c;
      *reinterpret_cast<uint4*>(dst) = lo;
      *reinterpret_cast<uint4*>(dst + D / 2) = hi;
      continue;
    }
    float a[8], b[8];
    if (turn) {
      float c0[8], c1[8], s0[8], s1[8];
      load8(cos_t + pos * D + c, c0);
      load8(cos_t + pos * D + c + D / 2, c1);
      load8(sin_t + pos * D + c, s0);
      load8(sin_t + pos * D + c + D / 2, s1);
      unpack8<T>(lo, a);
      unpack8<T>(hi, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x0 = a[e], x1 = b[e];   // x*cos + rotate_half(x)*sin with rotate_half(x) = [-x1, x0]
        a[e] = x0 * c0[e] - x1 * s0[e];
        b[e] = x1 * c1[e] + x0 * s1[e];
      }
    } else {
      const float fill = bad ? __int_as_float(0x7FC00000) : 0.f;   // padding: zeros; a position behind the tables: NaN
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = b[e] = fill;
    }
    T* dst = head < Hq ? q_out + (t * Hq + head) * (int64_t)D + c
                       : k_pages + page * k_page_stride + ((int64_t)(head - Hq) * page_size + row) * D + c;
    store8(dst, a);
    store8(dst + D / 2, b);
  }
}

}  // namespace
}  // namespace bsb

using namespace bsb;

extern "C" {

int bsb_page_tables(const int32_t* lens, const int32_t* new_tokens, int32_t batch, int32_t* block_table, int64_t table_stride,
                    int32_t table_width, const int32_t* free_pages, const int32_t* free_count, int32_t capacity, int32_t page_size,
                    int64_t max_tokens, int64_t* slots, int64_t* positions, int32_t* offsets, int64_t* last, int32_t* lens_out,
                    int32_t* free_count_out, void* stream) {
  BSB_CHECK_ARG(lens && new_tokens && block_table && free_pages && free_count && offsets && last && lens_out && free_count_out, "NULL buffer");
  BSB_CHECK_ARG(batch >= 1 && table_width >= 1 && table_stride >= table_width && page_size >= 1 && capacity >= 1, "bad table shape");
  BSB_CHECK_ARG(max_tokens >= 0 && max_tokens <= INT_MAX && (max_tokens == 0 || (slots && positions)), "bad token list");
  if (batch > kTableRows) {
    set_error("page tables: at most %d requests per call (got %d)", kTableRows, batch);
    return BSB_ELIMIT;
  }
  int* status = device_index_word();
  if (status == nullptr) return BSB_ECUDA;
  const size_t smem = (size_t)batch * 8;
  if (smem > 40 * 1024)                  // (48 KB without it, the kernel's static part included)
    BSB_CUDA(cudaFuncSetAttribute(page_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTableRows * 8));
  BSB_CUDA(launch_pdl(page_tables_kernel, dim3(1), dim3(kTableThreads), smem, (cudaStream_t)stream, lens, new_tokens, batch, block_table,
                      table_stride, table_width, free_pages, free_count, capacity, page_size, max_tokens, slots, positions, offsets, last,
                      lens_out, free_count_out, status));
  if (int rc = check_launch("page_tables_kernel")) return rc;
  if (max_tokens <= kTokensInOne) return BSB_OK;
  BSB_CUDA(launch_pdl(page_tokens_kernel, dim3((unsigned)ceil_div64(max_tokens, 256)), dim3(256), 0, (cudaStream_t)stream,
                      (const int32_t*)offsets, batch, new_tokens, (const int64_t*)last, (const int32_t*)block_table, table_stride, page_size,
                      max_tokens, slots, positions));
  return check_launch("page_tokens_kernel");
}

int bsb_release_pages(const uint8_t* done, int32_t* lens, int32_t batch, const int32_t* block_table, int64_t table_stride, int32_t table_width,
                      int32_t* free_pages, int32_t* free_count, int32_t capacity, int32_t page_size, void* stream) {
  BSB_CHECK_ARG(done && lens && block_table && free_pages && free_count, "NULL buffer");
  BSB_CHECK_ARG(batch >= 1 && table_width >= 1 && table_stride >= table_width && page_size >= 1 && capacity >= 1, "bad table shape");
  if (batch > kTableRows) {
    set_error("release pages: at most %d requests per call (got %d)", kTableRows, batch);
    return BSB_ELIMIT;
  }
  int* status = device_index_word();
  if (status == nullptr) return BSB_ECUDA;
  BSB_CUDA(launch_pdl(release_pages_kernel, dim3(1), dim3(kTableThreads), (size_t)batch * 4, (cudaStream_t)stream, done, lens, batch,
                      block_table, table_stride, table_width, free_pages, free_count, capacity, page_size, status));
  return check_launch("release_pages_kernel");
}

int bsb_rope_paged_cache(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                         const void* cos_table, const void* sin_table, int64_t table_len, const int64_t* positions, const int64_t* slots,
                         void* q_out, void* k_pages, void* v_pages, int64_t num_pages, int64_t k_page_stride, int64_t v_page_stride,
                         int64_t tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype, void* stream) {
  BSB_CHECK_ARG(tokens >= 0, "negative token count");
  BSB_CHECK_ARG(dtype == BSB_F16 || dtype == BSB_BF16, "rope_paged_cache: fp16 or bf16 (got dtype code %d)", dtype);
  BSB_CHECK_ARG(q_heads >= 1 && kv_heads >= 1 && head_dim >= 16 && head_dim % 16 == 0 && head_dim <= 512 && page_size >= 1 &&
                num_pages >= 1 && table_len >= 1, "bad shape (head_dim must be a multiple of 16 up to 512)");
  if (tokens == 0) return BSB_OK;
  BSB_CHECK_ARG(q && k && v && cos_table && sin_table && positions && slots && q_out && k_pages && v_pages, "NULL buffer");
  const int64_t page = (int64_t)kv_heads * page_size * head_dim;
  BSB_CHECK_ARG((tokens == 1 || (q_stride >= (int64_t)q_heads * head_dim && k_stride >= (int64_t)kv_heads * head_dim && v_stride >= (int64_t)kv_heads * head_dim)) &&
                (num_pages == 1 || (k_page_stride >= page && v_page_stride >= page)), "stride smaller than the row or page");
  BSB_CHECK_ARG((q_stride | k_stride | v_stride | k_page_stride | v_page_stride) % 8 == 0, "strides must be multiples of 8 elements");
  BSB_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cos_table | (uintptr_t)sin_table | (uintptr_t)q_out |
                 (uintptr_t)k_pages | (uintptr_t)v_pages) % 16 == 0, "buffers must be 16-byte aligned");
  BSB_CHECK_ARG(tokens <= INT_MAX, "too many tokens");
  int* status = device_index_word();
  if (status == nullptr) return BSB_ECUDA;
  const dim3 grid((unsigned)tokens);
  const int64_t items = ((int64_t)q_heads + 2 * (int64_t)kv_heads) * (head_dim / 16), trips = ceil_div64(items, kRopeThreads);
  const dim3 block((unsigned)(ceil_div64(ceil_div64(items, trips), 32) * 32));
  if (dtype == BSB_F16)
    BSB_CUDA(launch_pdl(rope_paged_kernel<__half>, grid, block, 0, (cudaStream_t)stream, (const __half*)q, (const __half*)k, (const __half*)v,
                        q_stride, k_stride, v_stride, (const __half*)cos_table, (const __half*)sin_table, table_len, positions, slots,
                        (__half*)q_out, (__half*)k_pages, (__half*)v_pages, num_pages, k_page_stride, v_page_stride, q_heads, kv_heads,
                        head_dim, page_size, status));
  else
    BSB_CUDA(launch_pdl(rope_paged_kernel<__nv_bfloat16>, grid, block, 0, (cudaStream_t)stream, (const __nv_bfloat16*)q, (const __nv_bfloat16*)k,
                        (const __nv_bfloat16*)v, q_stride, k_stride, v_stride, (const __nv_bfloat16*)cos_table, (const __nv_bfloat16*)sin_table,
                        table_len, positions, slots, (__nv_bfloat16*)q_out, (__nv_bfloat16*)k_pages, (__nv_bfloat16*)v_pages, num_pages,
                        k_page_stride, v_page_stride, q_heads, kv_heads, head_dim, page_size, status));
  return check_launch("rope_paged_kernel");
}

}  // extern "C"
