// Tensor front end of the serving entry points: argument checks, outputs and scratch from PyTorch's allocator, the current
// stream.  At small sizes these calls are a few microseconds of GPU work, less than the same steps take in Python
// (19 us a call there, 6-9 us here).  The kernels are reached through the C ABI only, at the addresses that bind() is given,
// so that this module and the ctypes binding share one library.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <initializer_list>
#include <optional>
#include <string>

#include "../../include/bitstack_b200.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

decltype(&bsb_page_tables) page_tables_fn = nullptr;
decltype(&bsb_release_pages) release_pages_fn = nullptr;
decltype(&bsb_rope_paged_cache) rope_paged_cache_fn = nullptr;
decltype(&bsb_paged_attention_scratch_bytes) scratch_bytes_fn = nullptr;
decltype(&bsb_paged_decode_attention) paged_decode_attention_fn = nullptr;
decltype(&bsb_sample_step) sample_step_fn = nullptr;

void bind(const py::dict& address) {
  auto at = [&](const char* name) { return reinterpret_cast<void*>(address[name].cast<uintptr_t>()); };
  page_tables_fn = reinterpret_cast<decltype(page_tables_fn)>(at("bsb_page_tables"));
  release_pages_fn = reinterpret_cast<decltype(release_pages_fn)>(at("bsb_release_pages"));
  rope_paged_cache_fn = reinterpret_cast<decltype(rope_paged_cache_fn)>(at("bsb_rope_paged_cache"));
  scratch_bytes_fn = reinterpret_cast<decltype(scratch_bytes_fn)>(at("bsb_paged_attention_scratch_bytes"));
  paged_decode_attention_fn = reinterpret_cast<decltype(paged_decode_attention_fn)>(at("bsb_paged_decode_attention"));
  sample_step_fn = reinterpret_cast<decltype(sample_step_fn)>(at("bsb_sample_step"));
}

constexpr int64_t kAny = -1;

[[noreturn]] void refuse(const std::string& text) { throw py::value_error(text); }

// CUDA tensor on device `index` of this type and shape, contiguous, or with `strided` only in its last dimension
void need(const Tensor& t, const char* name, at::ScalarType type, std::initializer_list<int64_t> shape, int index, bool strided = false) {
  if (!t.defined() || !t.is_cuda() || t.get_device() != index)
    refuse(std::string(name) + " must be a CUDA tensor on cuda:" + std::to_string(index));
  if (t.scalar_type() != type) refuse(std::string(name) + " must be " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
  bool fits = t.dim() == (int64_t)shape.size();
  if (fits) {
    int64_t d = 0;
    for (int64_t want : shape) {
      fits = fits && (want == kAny || t.size(d) == want);
      ++d;
    }
  }
  if (!fits) {
    std::string want, got;
    for (int64_t n : shape) want += (want.empty() ? "" : ", ") + (n == kAny ? std::string("any") : std::to_string(n));
    for (int64_t n : t.sizes()) got += (got.empty() ? "" : ", ") + std::to_string(n);
    refuse(std::string(name) + " must have shape [" + want + "], got [" + got + "]");
  }
  if (!t.is_contiguous() && !(strided && (t.size(-1) <= 1 || t.stride(-1) == 1)))
    refuse(std::string(name) + " must be contiguous" + (strided ? " in its last dimension" : ""));
}

int index_of(const Tensor& t, const char* name) {
  if (!t.defined() || !t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
  return t.get_device();
}
int32_t small(int64_t v, const char* name) {
  if (v < 0 || v > INT32_MAX) refuse(std::string(name) + " is out of range");
  return (int32_t)v;
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* stream_of(int index) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); }
void check(int rc, const char* what) {
  if (rc != 0) py::module_::import("bitstack_b200._lib").attr("check")(rc, what);
}
template <typename T> T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T> T* ptr(const Maybe& t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

int code_of(at::ScalarType type) { return type == at::kHalf ? BSB_F16 : type == at::kBFloat16 ? BSB_BF16 : BSB_F32; }

struct Lists { int index; int32_t batch, width; };
Lists page_lists(const Tensor& lens, const Tensor& table, const Tensor& free_pages, const Tensor& free_count) {
  const int index = index_of(lens, "lens");
  need(lens, "lens", at::kInt, {kAny}, index);
  need(table, "block_table", at::kInt, {lens.size(0), kAny}, index, true);
  need(free_pages, "free_pages", at::kInt, {kAny}, index);
  need(free_count, "free_count", at::kInt, {1}, index);
  return {index, small(lens.size(0), "the number of requests"), small(table.size(1), "the table's width")};
}

py::tuple page_tables(const Tensor& lens, const Tensor& new_tokens, const Tensor& table, const Tensor& free_pages, const Tensor& free_count,
                      int64_t page_size, int64_t max_tokens, const Maybe& lens_out, const Maybe& free_count_out) {
  const Lists l = page_lists(lens, table, free_pages, free_count);
  need(new_tokens, "new_tokens", at::kInt, {l.batch}, l.index);
  if (lens_out) need(*lens_out, "lens_out", at::kInt, {l.batch}, l.index);
  if (free_count_out) need(*free_count_out, "free_count_out", at::kInt, {1}, l.index);
  small(max_tokens, "max_tokens");       // (in front of the lists' allocation)
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)l.index);
  const auto longs = lens.options().dtype(at::kLong);
  Tensor slots = at::empty({max_tokens}, longs), positions = at::empty({max_tokens}, longs), last = at::empty({l.batch}, longs);
  Tensor offsets = at::empty({l.batch + 1}, lens.options());
  check(page_tables_fn(ptr<int32_t>(lens), ptr<int32_t>(new_tokens), l.batch, ptr<int32_t>(table), row_stride(table), l.width,
                       ptr<int32_t>(free_pages), ptr<int32_t>(free_count), small(free_pages.size(0), "the stack's size"),
                       small(page_size, "page_size"), max_tokens, ptr<int64_t>(slots), ptr<int64_t>(positions), ptr<int32_t>(offsets),
                       ptr<int64_t>(last), lens_out ? ptr<int32_t>(*lens_out) : ptr<int32_t>(lens),
                       free_count_out ? ptr<int32_t>(*free_count_out) : ptr<int32_t>(free_count), stream_of(l.index)),
        "bsb_page_tables");
  return py::make_tuple(slots, positions, offsets, last);
}

void release_pages(const Tensor& done, const Tensor& lens, const Tensor& table, const Tensor& free_pages, const Tensor& free_count, int64_t page_size) {
  const Lists l = page_lists(lens, table, free_pages, free_count);
  need(done, "done", at::kBool, {l.batch}, l.index);
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)l.index);
  check(release_pages_fn(ptr<uint8_t>(done), ptr<int32_t>(lens), l.batch, ptr<int32_t>(table), row_stride(table), l.width, ptr<int32_t>(free_pages),
                         ptr<int32_t>(free_count), small(free_pages.size(0), "the stack's size"), small(page_size, "page_size"), stream_of(l.index)),
        "bsb_release_pages");
}

// what the two calls that take q, k, v and the page pool have in common
struct Rows {
  int index, dtype;
  int64_t rows, pages, k_page, v_page;
  int32_t q_heads, kv_heads, dim, page_size;
};
Rows rows_and_pages(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos, const Tensor& sin, const Tensor& k_pages, const Tensor& v_pages,
                    int64_t q_heads, int64_t kv_heads, int64_t dim) {
  if (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16) refuse(std::string("q must be fp16 or bf16, got ") + c10::toString(q.scalar_type()));
  const at::ScalarType type = q.scalar_type();
  Rows r;
  r.index = index_of(q, "q");
  r.dtype = code_of(type);
  r.q_heads = small(q_heads, "q_heads");
  r.kv_heads = small(kv_heads, "kv_heads");
  r.dim = small(dim, "head_dim");
  need(q, "q", type, {kAny, q_heads * dim}, r.index, true);
  r.rows = q.size(0);
  need(k, "k", type, {r.rows, kv_heads * dim}, r.index, true);
  need(v, "v", type, {r.rows, kv_heads * dim}, r.index, true);
  need(cos, "cos", type, {kAny, dim}, r.index);
  need(sin, "sin", type, {cos.size(0), dim}, r.index);
  need(k_pages, "k_pages", type, {kAny, kv_heads, kAny, dim}, r.index, true);
  r.pages = k_pages.size(0);
  r.page_size = small(k_pages.size(2), "page_size");
  need(v_pages, "v_pages", type, {r.pages, kv_heads, r.page_size, dim}, r.index, true);
  if (r.pages < 1 || r.page_size < 1) refuse("the page pool is empty");
  const int64_t inner = kv_heads * r.page_size * dim;
  for (const Tensor* t : {&k_pages, &v_pages}) {   // pages [kv_heads, page_size, dim] are contiguous; they may lie apart
    if (t->is_contiguous()) continue;
    const bool whole = (t->size(1) == 1 || t->stride(1) == r.page_size * dim) && (t->size(2) == 1 || t->stride(2) == dim);
    if (!whole || (r.pages > 1 && t->stride(0) < inner))
      refuse(std::string(t == &k_pages ? "k_pages" : "v_pages") + ": every page [kv_heads, page_size, head_dim] must be contiguous and apart from the next");
  }
  r.k_page = r.pages > 1 ? k_pages.stride(0) : inner;
  r.v_page = r.pages > 1 ? v_pages.stride(0) : inner;
  return r;
}

Tensor rope_paged_cache(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos, const Tensor& sin, const Tensor& positions, const Tensor& slots,
                        const Tensor& k_pages, const Tensor& v_pages, int64_t q_heads, int64_t kv_heads, int64_t dim) {
  const Rows r = rows_and_pages(q, k, v, cos, sin, k_pages, v_pages, q_heads, kv_heads, dim);
  need(positions, "positions", at::kLong, {r.rows}, r.index);
  need(slots, "slots", at::kLong, {r.rows}, r.index);
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)r.index);
  Tensor out = at::empty({r.rows, q_heads * dim}, q.options());
  check(rope_paged_cache_fn(q.data_ptr(), k.data_ptr(), v.data_ptr(), row_stride(q), row_stride(k), row_stride(v), cos.data_ptr(), sin.data_ptr(),
                            cos.size(0), ptr<int64_t>(positions), ptr<int64_t>(slots), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), r.pages,
                            r.k_page, r.v_page, r.rows, r.q_heads, r.kv_heads, r.dim, r.page_size, r.dtype, stream_of(r.index)),
        "bsb_rope_paged_cache");
  return out;
}

Tensor paged_decode_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos, const Tensor& sin, const Tensor& positions,
                              const Tensor& table, const Tensor& k_pages, const Tensor& v_pages, int64_t q_heads, int64_t kv_heads, int64_t dim) {
  const Rows r = rows_and_pages(q, k, v, cos, sin, k_pages, v_pages, q_heads, kv_heads, dim);
  need(positions, "positions", at::kLong, {r.rows}, r.index);
  need(table, "block_table", at::kInt, {r.rows, kAny}, r.index, true);
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)r.index);
  Tensor out = at::empty({r.rows, q_heads * dim}, q.options());
  // scratch of this call alone, from the caching allocator: calls on other streams and other captured graphs have theirs
  const int64_t bytes = std::max<int64_t>(scratch_bytes_fn(small(r.rows, "the batch"), r.q_heads, r.kv_heads, r.dim), 16);
  Tensor scratch = at::empty({bytes}, q.options().dtype(at::kByte));
  check(paged_decode_attention_fn(q.data_ptr(), k.data_ptr(), v.data_ptr(), row_stride(q), row_stride(k), row_stride(v), cos.data_ptr(), sin.data_ptr(),
                                  cos.size(0), ptr<int64_t>(positions), ptr<int32_t>(table), row_stride(table), small(table.size(1), "the table's width"),
                                  k_pages.data_ptr(), v_pages.data_ptr(), r.pages, r.k_page, r.v_page, out.data_ptr(), (int32_t)r.rows, r.q_heads,
                                  r.kv_heads, r.dim, r.page_size, r.dtype, scratch.data_ptr(), bytes, stream_of(r.index)),
        "bsb_paged_decode_attention");
  return out;
}

void sample_step(const Tensor& logits, const Tensor& uniforms, const Tensor& tokens, const Maybe& temperature, const Maybe& top_k, const Maybe& top_p,
                 const Maybe& min_p, const Maybe& pos, const Maybe& logprobs) {
  const at::ScalarType type = logits.scalar_type();
  if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) refuse(std::string("logits must be fp16, bf16 or fp32, got ") + c10::toString(type));
  const int index = index_of(logits, "logits");
  need(logits, "logits", type, {kAny, kAny}, index, true);
  const int64_t batch = logits.size(0);
  need(uniforms, "uniforms", at::kFloat, {batch}, index);
  need(tokens, "tokens", at::kLong, {batch}, index);
  if (temperature) need(*temperature, "temperature", at::kFloat, {batch}, index);
  if (top_k) need(*top_k, "top_k", at::kInt, {batch}, index);
  if (top_p) need(*top_p, "top_p", at::kFloat, {batch}, index);
  if (min_p) need(*min_p, "min_p", at::kFloat, {batch}, index);
  if (logprobs) need(*logprobs, "logprobs", at::kFloat, {batch}, index);
  if (pos) need(*pos, "pos", at::kLong, {1}, index);
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)index);
  check(sample_step_fn(logits.data_ptr(), batch, logits.size(1), row_stride(logits), code_of(type), ptr<float>(uniforms), ptr<float>(temperature),
                       ptr<int32_t>(top_k), ptr<float>(top_p), ptr<float>(min_p), ptr<int64_t>(tokens), ptr<int64_t>(pos), ptr<float>(logprobs),
                       stream_of(index)),
        "bsb_sample_step");
}

}  // namespace

PYBIND11_MODULE(_serving, m) {
  m.def("bind", &bind);
  m.def("page_tables", &page_tables);
  m.def("release_pages", &release_pages);
  m.def("rope_paged_cache", &rope_paged_cache);
  m.def("paged_decode_attention", &paged_decode_attention);
  m.def("sample_step", &sample_step);
}
