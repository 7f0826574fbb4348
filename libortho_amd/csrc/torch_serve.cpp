// The serving operators' part of the compiled torch binding: page_step,
// cache_append, paged_attention and adapter_add over the C ABI, with the
// checks and messages of libortho_amd/_C_ops.py.  Host code only.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <initializer_list>
#include <string>
#include <tuple>

#include "orth_hip.h"

void check_rc(int rc);  // torch_ops.cpp

namespace {

using Opt = c10::optional<at::Tensor>;

void req(bool cond, const char *msg) {
    if (!cond) throw std::runtime_error(msg);
}

bool given(const Opt &t) { return t.has_value() && t->defined(); }

int64_t stride_of(const at::Tensor &t, int64_t d);

void *ptr(const at::Tensor &t) { return t.numel() > 0 ? t.data_ptr() : nullptr; }

// None of the operators has a gradient: a tensor that wants one is refused
// rather than forgotten.
struct Named {
    const char *name;
    const at::Tensor *t;
};
Named named(const char *name, const at::Tensor &t) { return {name, &t}; }
Named named(const char *name, const Opt &t) { return {name, given(t) ? &*t : nullptr}; }
void no_gradient(const char *op, std::initializer_list<Named> tensors) {
    if (!at::GradMode::is_enabled()) return;
    for (const Named &n : tensors)
        if (n.t && n.t->requires_grad())
            throw std::runtime_error(std::string(op) + " has no gradient: " + n.name +
                                     " requires one (detach it, or call under torch.no_grad())");
}

hipStream_t stream_of(const at::Device &dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

int32_t dtype16(const at::Tensor &t, const char *msg) {
    req(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, msg);
    return t.scalar_type() == at::kHalf ? ORTH_DT_F16 : ORTH_DT_BF16;
}

void index_tensor(const at::Tensor &t, const at::Device &dev, int64_t n, at::ScalarType type, const char *msg) {
    req(t.device() == dev && t.scalar_type() == type && t.dim() == 1 && t.is_contiguous() && (n < 0 || t.size(0) == n), msg);
}

orth_hip_cache_t cache_of(const at::Tensor &k, const at::Tensor &v) {
    req(k.is_cuda() && v.device() == k.device(), "k_cache and v_cache must be on one ROCm GPU");
    req(k.dim() == 4 && v.sizes() == k.sizes(), "k_cache and v_cache must be [pages, page_size, kv_heads, head_dim]");
    req(v.scalar_type() == k.scalar_type(), "k_cache and v_cache must have one dtype");
    req(k.stride(3) == 1 && v.stride(3) == 1, "the cache's last dimension must be contiguous");
    orth_hip_cache_t c{};
    c.dtype = dtype16(k, "the cache must be float16 or bfloat16");
    c.k_cache = ptr(k);
    c.v_cache = ptr(v);
    req(k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX, "the cache's page_size or kv_heads is too large");
    c.pages = k.size(0);
    c.page_size = (int32_t)k.size(1);
    c.kv_heads = (int32_t)k.size(2);
    req(k.size(3) <= 256, "head_dim must be a multiple of 8, at most 256");
    c.head_dim = (int32_t)k.size(3);
    for (int i = 0; i < 3; i++) {
        c.k_strides[i] = stride_of(k, i);
        c.v_strides[i] = stride_of(v, i);
    }
    return c;
}

// [tokens, heads, head_dim] of the cache's dtype, elements contiguous
void vectors(const at::Tensor &t, const at::Tensor &cache, int64_t tokens, const char *msg) {
    req(t.device() == cache.device() && t.scalar_type() == cache.scalar_type() && t.dim() == 3 && t.size(0) == tokens &&
            t.size(2) == cache.size(3) && (t.stride(2) == 1 || t.numel() == 0), msg);
}

// A dimension of one element has whatever stride torch gave it: none.
int64_t stride_of(const at::Tensor &t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

void strides2(const at::Tensor &t, int64_t *s) {
    s[0] = stride_of(t, 0);
    s[1] = stride_of(t, 1);
}

// n elements of an int32 tensor's storage from *at on, as a tensor of `type`.
at::Tensor part_of(const at::Tensor &all, int64_t *at, int64_t n, at::ScalarType type) {
    const int64_t words = type == at::kLong ? 2 : 1;
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(),
                                                            c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    t.unsafeGetTensorImpl()->set_storage_offset(*at / words);
    *at += n * words;
    return t;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>
page_step(const at::Tensor &lengths, const at::Tensor &new_tokens, const at::Tensor &table, const at::Tensor &free_pages,
          const at::Tensor &pool, int64_t page_size, int64_t tokens) {
    req(lengths.is_cuda(), "lengths must be on a ROCm GPU");
    const at::Device dev = lengths.device();
    const int64_t R = lengths.dim() == 1 ? lengths.size(0) : -1;
    index_tensor(lengths, dev, -1, at::kInt, "lengths must be a contiguous int32 vector");
    index_tensor(new_tokens, dev, R, at::kInt, "new_tokens must be a contiguous int32 vector as long as lengths");
    req(table.device() == dev && table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == R &&
            (table.numel() == 0 || (table.stride(1) == 1 && (R < 2 || table.stride(0) >= table.size(1)))),
        "block_table must be int32 [requests, pages] with contiguous rows that do not overlap");
    index_tensor(free_pages, dev, -1, at::kInt, "free_pages must be a contiguous int32 vector");
    index_tensor(pool, dev, 2, at::kInt, "pool must be a contiguous int32 vector of 2");
    req(page_size >= 1 && page_size <= INT32_MAX, "page_size must be positive");
    req(tokens >= 0 && tokens <= INT32_MAX, "tokens must not be negative, at most 2^31 - 1");
    c10::DeviceGuard guard(dev);
    // Views of one allocation (each of its own takes longer than the launch),
    // or, where the step's arrays take more than a megabyte, of two: lengths and
    // pool are kept between steps and would hold them all (a second allocation
    // takes 0.8 us: 16 requests 5.8 and 6.6).
    const int64_t own = 4 * tokens, rest = 2 * R + 3;
    const bool apart = own > (1 << 18);
    const at::Tensor step = at::empty({apart ? own : own + rest}, lengths.options());
    const at::Tensor kept = apart ? at::empty({rest}, lengths.options()) : step;
    int64_t at = 0, in = apart ? 0 : own;
    const at::Tensor slots = part_of(step, &at, tokens, at::kLong), rows = part_of(step, &at, tokens, at::kInt),
                     positions = part_of(step, &at, tokens, at::kInt), lengths_out = part_of(kept, &in, R, at::kInt),
                     start = part_of(kept, &in, R + 1, at::kInt), pool_out = part_of(kept, &in, 2, at::kInt);
    orth_hip_step_t s{};
    s.lengths = static_cast<const int32_t *>(ptr(lengths));
    s.new_tokens = static_cast<const int32_t *>(ptr(new_tokens));
    s.block_table = static_cast<int32_t *>(ptr(table));
    s.free_pages = static_cast<const int32_t *>(ptr(free_pages));
    s.pool = static_cast<const int32_t *>(ptr(pool));
    s.lengths_out = static_cast<int32_t *>(ptr(lengths_out));
    s.pool_out = static_cast<int32_t *>(ptr(pool_out));
    s.query_start = static_cast<int32_t *>(ptr(start));
    s.rows = static_cast<int32_t *>(ptr(rows));
    s.positions = static_cast<int32_t *>(ptr(positions));
    s.slots = static_cast<int64_t *>(ptr(slots));
    s.requests = R;
    s.table_width = table.size(1);
    s.table_stride = R < 2 || table.numel() == 0 ? table.size(1) : table.stride(0);
    s.free_count = free_pages.size(0);
    s.tokens = tokens;
    s.page_size = (int32_t)page_size;
    check_rc(orth_page_step_hip(&s, stream_of(dev)));
    return {lengths_out, pool_out, start, rows, positions, slots};
}

Opt cache_append(const at::Tensor &k, const at::Tensor &v, const at::Tensor &k_cache, const at::Tensor &v_cache,
                 const at::Tensor &slots, const Opt &q, const Opt &positions, const Opt &cos_sin, bool interleaved,
                 const Opt &q_out) {
    no_gradient("cache_append", {named("k", k), named("v", v), named("k_cache", k_cache), named("v_cache", v_cache),
                                 named("q", q), named("cos_sin", cos_sin), named("q_out", q_out)});
    const orth_hip_cache_t c = cache_of(k_cache, v_cache);
    const at::Device dev = k_cache.device();
    req(k.dim() == 3, "k must be [tokens, kv_heads, head_dim] of the cache's dtype on its device, vectors contiguous");
    const int64_t T = k.size(0);
    vectors(k, k_cache, T, "k must be [tokens, kv_heads, head_dim] of the cache's dtype on its device, vectors contiguous");
    vectors(v, k_cache, T, "v must be [tokens, kv_heads, head_dim] of the cache's dtype on its device, vectors contiguous");
    req(k.size(1) == c.kv_heads && v.size(1) == c.kv_heads, "k and v must have the cache's kv_heads");
    index_tensor(slots, dev, T, at::kLong, "slots must be a contiguous int64 vector of tokens");
    req(given(cos_sin) || !given(q), "q needs cos_sin");
    req(!given(q_out) || given(q), "q_out needs q");
    orth_hip_append_t a{};
    if (given(cos_sin)) {
        req(given(positions), "cos_sin needs positions");
        index_tensor(*positions, dev, T, at::kInt, "positions must be a contiguous int32 vector of tokens");
        req(cos_sin->device() == dev && cos_sin->scalar_type() == at::kFloat && cos_sin->dim() == 2 && cos_sin->is_contiguous(),
            "cos_sin must be a contiguous float32 [positions, rot]");
        req(cos_sin->size(1) % 2 == 0 && cos_sin->size(1) <= c.head_dim, "rot must be even and at most head_dim");
        a.positions = static_cast<const int32_t *>(ptr(*positions));
        // an empty table still turns the call: no position lies inside it
        static const float none = 0.f;
        a.cos_sin = cos_sin->numel() > 0 ? static_cast<const float *>(ptr(*cos_sin)) : &none;
        a.cos_sin_rows = cos_sin->size(0);
        a.rot = (int32_t)cos_sin->size(1);
    }
    c10::DeviceGuard guard(dev);
    Opt out;
    if (given(q)) {
        vectors(*q, k_cache, T, "q must be [tokens, q_heads, head_dim] of the cache's dtype on its device, vectors contiguous");
        req(q->size(1) >= 1 && q->size(1) <= INT32_MAX, "q must have heads");
        if (given(q_out)) {
            vectors(*q_out, k_cache, T, "q_out must be like q");
            req(q_out->size(1) == q->size(1), "q_out must be like q");
            out = *q_out;
        } else {
            out = at::empty({T, q->size(1), q->size(2)}, q->options());
        }
        a.q = ptr(*q);
        a.q_out = ptr(*out);
        strides2(*q, a.q_strides);
        strides2(*out, a.q_out_strides);
        a.q_heads = (int32_t)q->size(1);
    }
    a.k = ptr(k);
    a.v = ptr(v);
    strides2(k, a.k_strides);
    strides2(v, a.v_strides);
    a.slots = static_cast<const int64_t *>(ptr(slots));
    a.tokens = T;
    a.interleaved = interleaved;
    check_rc(orth_cache_append_hip(&c, &a, stream_of(dev)));
    return out;
}

at::Tensor paged_attention(const at::Tensor &q, const at::Tensor &k_cache, const at::Tensor &v_cache,
                           const at::Tensor &table, const at::Tensor &positions, const Opt &rows,
                           const c10::optional<double> &scale, int64_t window, const Opt &out_) {
    no_gradient("paged_attention", {named("q", q), named("k_cache", k_cache), named("v_cache", v_cache), named("out", out_)});
    const orth_hip_cache_t c = cache_of(k_cache, v_cache);
    const at::Device dev = k_cache.device();
    req(q.dim() == 3, "q must be [tokens, q_heads, head_dim] of the cache's dtype on its device, vectors contiguous");
    const int64_t T = q.size(0);
    vectors(q, k_cache, T, "q must be [tokens, q_heads, head_dim] of the cache's dtype on its device, vectors contiguous");
    req(c.kv_heads > 0 && q.size(1) > 0 && q.size(1) % c.kv_heads == 0 && q.size(1) <= INT32_MAX,
        "q_heads must be a multiple of kv_heads");
    req(table.device() == dev && table.scalar_type() == at::kInt && table.dim() == 2 &&
            (table.numel() == 0 || (table.stride(1) == 1 && (table.size(0) < 2 || table.stride(0) >= table.size(1)))),
        "block_table must be int32 [requests, pages] with contiguous rows that do not overlap");
    index_tensor(positions, dev, T, at::kInt, "positions must be a contiguous int32 vector of tokens");
    if (given(rows)) index_tensor(*rows, dev, T, at::kInt, "rows must be a contiguous int32 vector of tokens");
    req(window >= 0 && window <= INT32_MAX, "window must not be negative");
    c10::DeviceGuard guard(dev);
    at::Tensor out;
    if (given(out_)) {
        vectors(*out_, k_cache, T, "out must be like q");
        req(out_->size(1) == q.size(1), "out must be like q");
        out = *out_;
    } else {
        out = at::empty({T, q.size(1), q.size(2)}, q.options());
    }
    orth_hip_attend_t a{};
    a.q = ptr(q);
    a.out = ptr(out);
    strides2(q, a.q_strides);
    strides2(out, a.out_strides);
    a.block_table = static_cast<const int32_t *>(ptr(table));
    a.positions = static_cast<const int32_t *>(ptr(positions));
    a.rows = given(rows) ? static_cast<const int32_t *>(ptr(*rows)) : nullptr;
    a.table_rows = table.size(0);
    a.table_width = table.size(1);
    a.table_stride = table.size(0) < 2 || table.numel() == 0 ? table.size(1) : table.stride(0);
    a.tokens = T;
    a.q_heads = (int32_t)q.size(1);
    a.window = (int32_t)window;
    a.scale = (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)c.head_dim));
    check_rc(orth_paged_attention_hip(&c, &a, stream_of(dev)));
    return out;
}

at::Tensor adapter_add(const at::Tensor &y, const at::Tensor &x, const at::Tensor &a, const at::Tensor &b,
                       const at::Tensor &adapters, const Opt &scales, const Opt &out_) {
    no_gradient("adapter_add", {named("y", y), named("x", x), named("a", a), named("b", b), named("scales", scales),
                                named("out", out_)});
    req(x.is_cuda(), "x must be on a ROCm GPU");
    const at::Device dev = x.device();
    orth_hip_adapter_t g{};
    g.dtype = dtype16(x, "adapters take float16 or bfloat16 activations");
    req(x.dim() == 2 && y.dim() == 2 && y.size(0) == x.size(0), "x and y must be 2-D [M, K] / [M, N]");
    req(a.dim() == 3 && b.dim() == 3 && b.size(0) == a.size(0) && b.size(2) == a.size(1) && a.size(2) == x.size(1) &&
            b.size(1) == y.size(1),
        "a must be [adapters, rank, K] and b [adapters, N, rank]");
    req(y.device() == dev && a.device() == dev && b.device() == dev, "x, y, a and b must be on one device");
    req(y.scalar_type() == x.scalar_type() && a.scalar_type() == x.scalar_type() && b.scalar_type() == x.scalar_type(),
        "x, y, a and b must have one dtype");
    req(a.is_contiguous() && b.is_contiguous(), "a and b must be contiguous");
    const int64_t M = x.size(0);
    req((x.stride(1) == 1 || x.numel() == 0) && (y.stride(1) == 1 || y.numel() == 0), "the rows of x and y must be contiguous");
    index_tensor(adapters, dev, M, at::kInt, "adapters must be a contiguous int32 vector of tokens");
    if (given(scales))
        req(scales->device() == dev && scales->scalar_type() == at::kFloat && scales->dim() == 1 && scales->is_contiguous() &&
                scales->size(0) == a.size(0),
            "scales must be a contiguous float32 vector of adapters");
    c10::DeviceGuard guard(dev);
    at::Tensor out;
    if (given(out_)) {
        req(out_->device() == dev && out_->scalar_type() == x.scalar_type() && out_->sizes() == y.sizes() &&
                (out_->stride(1) == 1 || out_->numel() == 0),
            "out must be like y");
        out = *out_;
    } else {
        out = at::empty(y.sizes(), y.options());
    }
    g.x = ptr(x);
    g.y = ptr(y);
    g.out = ptr(out);
    g.a = ptr(a);
    g.b = ptr(b);
    g.adapters = static_cast<const int32_t *>(ptr(adapters));
    g.scales = given(scales) ? static_cast<const float *>(ptr(*scales)) : nullptr;
    g.x_stride = stride_of(x, 0);
    g.y_stride = stride_of(y, 0);
    g.out_stride = stride_of(out, 0);
    g.tokens = M;
    g.in_features = x.size(1);
    g.out_features = y.size(1);
    g.count = a.size(0);
    req(a.size(1) >= 1 && a.size(1) <= ORTH_ADAPTER_RANK, "rank must lie in 1..256");
    g.rank = (int32_t)a.size(1);
    check_rc(orth_adapter_add_hip(&g, stream_of(dev)));
    return out;
}

}  // namespace

void bind_serving(pybind11::module_ &m) {
    m.def("page_step", &page_step, "pages, slots and positions of a step's tokens", py::arg("lengths"),
          py::arg("new_tokens"), py::arg("block_table"), py::arg("free_pages"), py::arg("pool"), py::arg("page_size"),
          py::arg("tokens"));
    m.def("cache_append", &cache_append, "rotary positions, keys and values into their slots", py::arg("k"), py::arg("v"),
          py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"), py::arg("q") = py::none(),
          py::arg("positions") = py::none(), py::arg("cos_sin") = py::none(), py::arg("interleaved") = false,
          py::arg("q_out") = py::none());
    m.def("paged_attention", &paged_attention, "attention of single tokens over the paged cache", py::arg("q"),
          py::arg("k_cache"), py::arg("v_cache"), py::arg("block_table"), py::arg("positions"),
          py::arg("rows") = py::none(), py::arg("scale") = py::none(), py::arg("window") = 0, py::arg("out") = py::none());
    m.def("adapter_add", &adapter_add, "low-rank adapters beside a projection's output", py::arg("y"), py::arg("x"),
          py::arg("a"), py::arg("b"), py::arg("adapters"), py::arg("scales") = py::none(), py::arg("out") = py::none());
}
