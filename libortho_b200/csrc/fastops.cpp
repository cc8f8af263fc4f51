// Host path of the operators around the projections (_C_ops.page_step, rotary_append, paged_attention, low_rank_add): argument checks,
// outputs and scratch, the C record, the launch.  Part of the extension module of fastcall.cpp; wrong arguments raise here, with the
// device guard, the current stream and torch's allocator taken as any torch operator takes them.
#include <Python.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/torch.h>

#include <limits>

#include "../../include/ortho_b200.h"

namespace {

int (*page_step_c)(const ortho_b200_page_step_desc *, void *) = nullptr;
int (*rotary_append_c)(const ortho_b200_rotary_append_desc *, void *) = nullptr;
int (*attention_c)(const ortho_b200_paged_attention_desc *, void *, int64_t, void *) = nullptr;
int64_t (*attention_ws_c)(const ortho_b200_paged_attention_desc *) = nullptr;
int (*low_rank_c)(const ortho_b200_low_rank_desc *, void *, int64_t, void *) = nullptr;
int64_t (*low_rank_ws_c)(const ortho_b200_low_rank_desc *) = nullptr;
const char *(*strerror_c)(int) = nullptr;
int (*last_cuda_error_c)() = nullptr;

void check_status(int st, const char *where)
{
    if (st == ORTHO_B200_ERR_CUDA) TORCH_CHECK(false, where, ": ", strerror_c(st), " [cudaError ", last_cuda_error_c(), "] (status ", st, ")");
    TORCH_CHECK(st == ORTHO_B200_OK, where, ": ", strerror_c(st), " (status ", st, ")");
}

const at::Tensor &tensor(PyObject *o, const char *name)
{
    TORCH_CHECK_TYPE(o && THPVariable_Check(o), name, " must be a tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    TORCH_CHECK(t.defined() && t.is_cuda(), "libortho_b200 has no CPU path: `", name, "` must be a CUDA tensor");
    TORCH_CHECK_TYPE(t.layout() == at::kStrided && t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch(), name, " must be a plain strided tensor");
    return t;
}
// one that is read; `like`: on the device of the call
at::Tensor input(PyObject *o, const char *name, at::ScalarType type, const at::Tensor *like = nullptr)
{
    const at::Tensor &t = tensor(o, name);
    TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, ", not ", t.scalar_type());
    TORCH_CHECK(!like || t.device() == like->device(), name, " must live on the device of the other tensors");
    return t.is_neg() ? t.resolve_neg() : t;
}
at::Tensor output(PyObject *o, const char *name, at::ScalarType type, const at::Tensor &like)
{
    const at::Tensor &t = tensor(o, name);
    TORCH_CHECK_TYPE(t.scalar_type() == type && !t.is_neg(), name, " must be ", type, ", not ", t.scalar_type());
    TORCH_CHECK(t.device() == like.device(), name, " must live on the device of the other tensors");
    return t;
}
at::ScalarType half_type(const at::Tensor &t, const char *name)
{
    TORCH_CHECK_TYPE(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name, " must be float16 or bfloat16, not ", t.scalar_type());
    return t.scalar_type();
}
int type_number(at::ScalarType t) { return t == at::kHalf ? ORTHO_B200_TYPE_F16 : ORTHO_B200_TYPE_BF16; }
int64_t integer(PyObject *o, const char *name, int64_t least)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_VALUE(v >= least, name, " must be at least ", least);
    return v;
}
// a list of whole numbers, one after the other in memory
at::Tensor list_of(PyObject *o, const char *name, at::ScalarType type, int64_t n, const at::Tensor &like)
{
    at::Tensor t = input(o, name, type, &like);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, name, " must have ", n, " entries");
    return t.is_contiguous() ? t : t.contiguous();
}
void result_list(const at::Tensor &t, const char *name, int64_t n)
{
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name, " must be contiguous with ", n, " entries");
}
// heads of width D one after the other in the last dimension
void three_dims(const at::Tensor &t, const char *name, int64_t T, int64_t D)
{
    TORCH_CHECK_VALUE(t.dim() == 3 && (T < 0 || t.size(0) == T) && (D < 0 || t.size(2) == D), name, " must be [tokens, heads, head_dim] like the others");
}
bool aligned(const at::Tensor &t) { return ((uintptr_t)t.const_data_ptr() & 15u) == 0; }
// data pointers may be null for empty tensors; the library only looks at them where there is something to read
template <class P> P *ptr(const at::Tensor &t) { return static_cast<P *>(const_cast<void *>(t.const_data_ptr())); }
void *current_stream(const at::Tensor &t) { return (void *)c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
at::Tensor scratch(int64_t bytes, const at::Tensor &like)
{
    return at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(like.device()));
}
bool given(PyObject *o) { return o != Py_None; }

struct Cache { at::Tensor k, v; int64_t pages, page_size, heads, D; };
Cache cache_of(PyObject *k, PyObject *v, at::ScalarType type, const at::Tensor &like)
{
    Cache c;
    c.k = output(k, "k_cache", type, like);
    c.v = output(v, "v_cache", type, like);
    TORCH_CHECK_VALUE(c.k.dim() == 4 && c.v.sizes() == c.k.sizes(), "k_cache and v_cache must be [pages, page_size, kv_heads, head_dim] alike");
    TORCH_CHECK_VALUE(c.k.stride(3) == 1 && c.v.stride(3) == 1, "the caches' last dimension must be contiguous");
    c.pages = c.k.size(0); c.page_size = c.k.size(1); c.heads = c.k.size(2); c.D = c.k.size(3);
    TORCH_CHECK_VALUE(c.page_size >= 1 && c.heads >= 1 && c.D >= 1, "k_cache and v_cache must have pages of at least one token");
    return c;
}

// page_step(cached, fresh, block_table, free_pages, available, page_size, tokens, out or None) -> six tensors
PyObject *page_step(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 8, "page_step takes 8 arguments");
    at::Tensor cached = input(a[0], "cached", at::kInt);
    TORCH_CHECK_VALUE(cached.dim() == 1, "cached must be one-dimensional");
    const int64_t B = cached.size(0);
    if (!cached.is_contiguous()) cached = cached.contiguous();
    const at::Tensor fresh = list_of(a[1], "fresh", at::kInt, B, cached);
    const at::Tensor table = output(a[2], "block_table", at::kInt, cached);
    TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == B && (table.size(1) <= 1 || table.stride(1) == 1) && (B <= 1 || table.stride(0) >= table.size(1)),
                      "block_table must be [requests, pages] with contiguous rows");
    at::Tensor free_pages = input(a[3], "free_pages", at::kInt, &cached);
    TORCH_CHECK_VALUE(free_pages.dim() == 1, "free_pages must be one-dimensional");
    if (!free_pages.is_contiguous()) free_pages = free_pages.contiguous();
    const at::Tensor available = input(a[4], "available", at::kInt, &cached);
    TORCH_CHECK_VALUE(available.numel() == 1, "available must have one entry");
    const int64_t P = integer(a[5], "page_size", 1), T = integer(a[6], "tokens", 0);
    TORCH_CHECK_VALUE(P <= std::numeric_limits<int32_t>::max() && T <= std::numeric_limits<int32_t>::max(), "page_size and tokens must fit 32 bits");
    static const char *names[6] = {"lengths", "starts", "slots", "positions", "requests", "counts"};
    const int64_t sizes[6] = {B, B + 1, T, T, T, 3};
    at::Tensor out[6];
    const c10::cuda::CUDAGuard guard(cached.device());
    if (given(a[7])) {
        TORCH_CHECK_TYPE(PyTuple_Check(a[7]) && PyTuple_GET_SIZE(a[7]) == 6, "out must be the result of an earlier call");
        for (int i = 0; i < 6; i++) {
            out[i] = output(PyTuple_GET_ITEM(a[7], i), names[i], i == 2 ? at::kLong : at::kInt, cached);
            result_list(out[i], names[i], sizes[i]);
        }
    } else {
        for (int i = 0; i < 6; i++) out[i] = at::empty({sizes[i]}, cached.options().dtype(i == 2 ? at::kLong : at::kInt));
    }
    ortho_b200_page_step_desc d;
    memset(&d, 0, sizeof(d));
    d.cached = ptr<int32_t>(cached); d.fresh = ptr<int32_t>(fresh); d.block_table = ptr<int32_t>(table);
    d.free_pages = ptr<int32_t>(free_pages); d.available = ptr<int32_t>(available);
    d.lengths = ptr<int32_t>(out[0]); d.starts = ptr<int32_t>(out[1]); d.slots = ptr<int64_t>(out[2]);
    d.positions = ptr<int32_t>(out[3]); d.request_of = ptr<int32_t>(out[4]); d.counts = ptr<int32_t>(out[5]);
    d.requests = B; d.width = table.size(1); d.table_stride = table.stride(0); d.free_count = free_pages.size(0);
    d.tokens = T; d.page_size = P;
    void *stream = current_stream(cached);
    int st;
    Py_BEGIN_ALLOW_THREADS
    st = page_step_c(&d, stream);
    Py_END_ALLOW_THREADS
    check_status(st, "ortho_b200_page_step");
    if (given(a[7])) return Py_NewRef(a[7]);
    PyObject *r = PyTuple_New(6);
    if (!r) return nullptr;
    for (int i = 0; i < 6; i++) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(out[i]));
    return r;
    END_HANDLE_TH_ERRORS
}

// rotary_append(q or None, k, v, k_cache, v_cache, slots, positions, table, sections, interleaved, out) -> q_out or None
PyObject *rotary_append(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 11, "rotary_append takes 11 arguments");
    const auto type = half_type(tensor(a[1], "k"), "k");
    auto heads = [&](PyObject *o, const char *name, const at::Tensor *like) {
        at::Tensor t = input(o, name, type, like);
        three_dims(t, name, like ? like->size(0) : -1, like ? like->size(2) : -1);
        return t.stride(2) == 1 || t.size(2) <= 1 ? t : t.contiguous();
    };
    const at::Tensor k = heads(a[1], "k", nullptr), v = heads(a[2], "v", &k);
    TORCH_CHECK_VALUE(v.size(1) == k.size(1), "k and v must have the same heads");
    const Cache c = cache_of(a[3], a[4], type, k);
    const int64_t T = k.size(0);
    TORCH_CHECK_VALUE(c.heads == k.size(1) && c.D == k.size(2), "k and v must have the caches' heads and head_dim");
    TORCH_CHECK_VALUE(c.D <= 8192, "head_dim must be at most 8192");
    const at::Tensor slots = list_of(a[5], "slots", at::kLong, T, k);
    const c10::cuda::CUDAGuard guard(k.device());
    ortho_b200_rotary_append_desc d;
    memset(&d, 0, sizeof(d));
    at::Tensor positions, table, q, out;
    TORCH_CHECK_VALUE(given(a[6]) == given(a[7]), "positions and table go together");
    if (given(a[7])) {
        positions = input(a[6], "positions", at::kInt, &k);
        TORCH_CHECK_VALUE((positions.dim() == 1 || positions.dim() == 2) && positions.size(-1) == T, "positions must be [tokens] or [axes, tokens]");
        if (positions.stride(-1) != 1 && T > 1) positions = positions.contiguous();
        table = input(a[7], "table", at::kFloat, &k);
        TORCH_CHECK_VALUE(table.dim() == 2 && table.size(1) >= 2 && table.size(1) % 2 == 0 && table.size(1) <= c.D, "table must be [positions, rotary_dim], rotary_dim even and at most head_dim");
        if (!table.is_contiguous()) table = table.contiguous();
        d.axes = positions.dim() == 1 ? 1 : (int32_t)positions.size(0);
        TORCH_CHECK_VALUE(d.axes >= 1 && d.axes <= ORTHO_B200_MAX_AXES, "positions must have one to ", ORTHO_B200_MAX_AXES, " axes");
        d.position_stride = positions.dim() == 1 ? 0 : positions.stride(0);
        d.rotary = table.size(1);
        if (given(a[8])) {
            PyObject *seq = PySequence_Fast(a[8], "sections must be a sequence of whole numbers");
            if (!seq) throw python_error();
            const THPObjectPtr hold(seq);
            TORCH_CHECK_VALUE(PySequence_Fast_GET_SIZE(seq) == d.axes, "sections must have one entry per axis");
            int64_t end = 0;
            for (int i = 0; i < d.axes; i++) {
                end += integer(PySequence_Fast_GET_ITEM(seq, i), "a section", 0);
                TORCH_CHECK_VALUE(end <= d.rotary / 2, "sections must add up to rotary_dim / 2");
                d.section_ends[i] = (int32_t)end;
            }
            TORCH_CHECK_VALUE(end == d.rotary / 2, "sections must add up to rotary_dim / 2");
        } else {
            TORCH_CHECK_VALUE(d.axes == 1, "several axes need sections");
            d.section_ends[0] = (int32_t)(d.rotary / 2);
        }
        d.positions = ptr<int32_t>(positions); d.table = ptr<float>(table); d.table_rows = table.size(0);
    }
    if (given(a[0])) {
        TORCH_CHECK_VALUE(given(a[7]), "without positions there is nothing to do for q");
        q = heads(a[0], "q", &k);
        if (given(a[10])) {
            out = output(a[10], "out", type, k);
            TORCH_CHECK_VALUE(out.sizes() == q.sizes() && (out.stride(2) == 1 || out.size(2) <= 1), "out must have q's shape and a contiguous last dimension");
        } else {
            out = at::empty(q.sizes(), q.options());
        }
        d.q = ptr<void>(q); d.q_out = ptr<void>(out); d.q_heads = q.size(1);
        d.q_token_stride = q.stride(0); d.q_head_stride = q.stride(1); d.out_token_stride = out.stride(0); d.out_head_stride = out.stride(1);
    } else {
        TORCH_CHECK_VALUE(!given(a[10]), "out is for q");
    }
    const int truth = PyObject_IsTrue(a[9]);
    if (truth < 0) throw python_error();
    d.k = ptr<void>(k); d.v = ptr<void>(v); d.k_cache = ptr<void>(c.k); d.v_cache = ptr<void>(c.v); d.slots = ptr<int64_t>(slots);
    d.tokens = T; d.kv_heads = c.heads; d.head_dim = c.D; d.pages = c.pages; d.page_size = c.page_size;
    d.k_token_stride = k.stride(0); d.k_head_stride = k.stride(1); d.v_token_stride = v.stride(0); d.v_head_stride = v.stride(1);
    d.k_page_stride = c.k.stride(0); d.k_slot_stride = c.k.stride(1); d.k_cache_head_stride = c.k.stride(2);
    d.v_page_stride = c.v.stride(0); d.v_slot_stride = c.v.stride(1); d.v_cache_head_stride = c.v.stride(2);
    d.interleaved = truth; d.type = type_number(type);
    void *stream = current_stream(k);
    int st = 0;
    if (c.pages > 0 || d.q_heads > 0) {          // (a cache without pages keeps nothing)
        Py_BEGIN_ALLOW_THREADS
        st = rotary_append_c(&d, stream);
        Py_END_ALLOW_THREADS
    }
    check_status(st, "ortho_b200_rotary_append");
    if (!out.defined()) Py_RETURN_NONE;
    return given(a[10]) ? Py_NewRef(a[10]) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_cache, v_cache, block_table, lengths, scale or None, window, rows or None, out or None, lse or None) -> out
PyObject *paged_attention(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 10, "paged_attention takes 10 arguments");
    const auto type = half_type(tensor(a[0], "q"), "q");
    at::Tensor q = input(a[0], "q", type);
    three_dims(q, "q", -1, -1);
    const Cache c = cache_of(a[1], a[2], type, q);
    const int64_t B = q.size(0), H = q.size(1), D = q.size(2);
    TORCH_CHECK_VALUE(D == c.D && H >= 1 && H % c.heads == 0, "q must have the caches' head_dim and a multiple of their heads");
    TORCH_CHECK_VALUE(D % 8 == 0 && D <= 256, "head_dim must be a multiple of 8 up to 256");
    for (const at::Tensor *t : {&c.k, &c.v})
        TORCH_CHECK_VALUE(aligned(*t) && t->stride(0) % 8 == 0 && t->stride(1) % 8 == 0 && t->stride(2) % 8 == 0,
                          "the caches must be 16-byte aligned, with strides that are multiples of 8");
    const at::Tensor table = input(a[3], "block_table", at::kInt, &q);
    TORCH_CHECK_VALUE(table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1), "block_table must be [requests, pages] with contiguous rows");
    const at::Tensor lengths = list_of(a[4], "lengths", at::kInt, B, q);
    at::Tensor rows;
    if (given(a[7])) rows = list_of(a[7], "rows", at::kInt, B, q);
    else TORCH_CHECK_VALUE(table.size(0) == B, "block_table must have a row per query, or `rows` has to name them");
    double scale = 1.0 / std::sqrt((double)D);
    if (given(a[5])) {
        scale = PyFloat_AsDouble(a[5]);
        if (scale == -1.0 && PyErr_Occurred()) throw python_error();
    }
    const int64_t window = integer(a[6], "window", 0);
    const c10::cuda::CUDAGuard guard(q.device());
    if (q.stride(2) != 1 || !aligned(q) || q.stride(0) % 8 || q.stride(1) % 8) q = q.clone(at::MemoryFormat::Contiguous);
    at::Tensor out;
    if (given(a[8])) {
        out = output(a[8], "out", type, q);
        TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.stride(2) == 1 && aligned(out) && out.stride(0) % 8 == 0 && out.stride(1) % 8 == 0,
                          "out must have q's shape, a contiguous last dimension, 16-byte alignment and strides that are multiples of 8");
    } else {
        out = at::empty(q.sizes(), q.options());
    }
    ortho_b200_paged_attention_desc d;
    memset(&d, 0, sizeof(d));
    if (given(a[9])) {
        const at::Tensor lse = output(a[9], "lse", at::kFloat, q);
        TORCH_CHECK_VALUE(lse.dim() == 2 && lse.size(0) == B && lse.size(1) == H && lse.is_contiguous(), "lse must be a contiguous [requests, heads] tensor");
        d.lse = ptr<float>(lse);
    }
    d.q = ptr<void>(q); d.k_cache = ptr<void>(c.k); d.v_cache = ptr<void>(c.v); d.out = ptr<void>(out);
    d.block_table = ptr<int32_t>(table); d.lengths = ptr<int32_t>(lengths); d.row_of = rows.defined() ? ptr<int32_t>(rows) : nullptr;
    d.batch = B; d.q_heads = H; d.kv_heads = c.heads; d.head_dim = D; d.rows = table.size(0); d.width = table.size(1); d.table_stride = table.stride(0);
    d.pages = c.pages; d.page_size = c.page_size; d.window = window;
    d.q_token_stride = q.stride(0); d.q_head_stride = q.stride(1); d.out_token_stride = out.stride(0); d.out_head_stride = out.stride(1);
    d.k_page_stride = c.k.stride(0); d.k_slot_stride = c.k.stride(1); d.k_head_stride = c.k.stride(2);
    d.v_page_stride = c.v.stride(0); d.v_slot_stride = c.v.stride(1); d.v_head_stride = c.v.stride(2);
    d.scale = (float)scale; d.type = type_number(type);
    if (c.pages == 0) { d.width = 0; d.k_cache = d.v_cache = d.q; }        // nothing is cached: no row has a key
    int st = 0;
    if (B) {
        const int64_t need = attention_ws_c(&d);
        at::Tensor ws;
        if (need > 0) ws = scratch(need, q);
        void *wsp = need > 0 ? ws.mutable_data_ptr() : nullptr, *stream = current_stream(q);
        Py_BEGIN_ALLOW_THREADS
        st = attention_c(&d, wsp, need, stream);
        Py_END_ALLOW_THREADS
    }
    check_status(st, "ortho_b200_paged_attention");
    return given(a[8]) ? Py_NewRef(a[8]) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// low_rank_add(x, y, down, up, ids, scales or None, ranks or None, out or None) -> out
PyObject *low_rank_add(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 8, "low_rank_add takes 8 arguments");
    const auto type = half_type(tensor(a[0], "x"), "x");
    at::Tensor x = input(a[0], "x", type), y = input(a[1], "y", type, &x);
    const at::Tensor down = input(a[2], "down", type, &x), up = input(a[3], "up", type, &x);
    TORCH_CHECK_VALUE(down.dim() == 3 && up.dim() == 3 && up.size(0) == down.size(0) && up.size(2) == down.size(1) && down.size(0) >= 1,
                      "down must be [adapters, rank, in_features] and up [adapters, out_features, rank]");
    TORCH_CHECK_VALUE(down.is_contiguous() && up.is_contiguous() && aligned(down) && aligned(up), "down and up must be contiguous and 16-byte aligned");
    const int64_t E = down.size(0), R = down.size(1), K = down.size(2), N = up.size(1);
    TORCH_CHECK_VALUE(R >= 8 && R % 8 == 0 && R <= 256 && K >= 8 && K % 8 == 0 && N >= 1, "rank must be a multiple of 8 up to 256 and in_features a multiple of 8");
    TORCH_CHECK_VALUE(E <= 8192, "at most 8192 adapters");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == K && y.dim() == x.dim() && y.size(-1) == N, "x must be [..., in_features] and y [..., out_features]");
    for (int64_t i = 0; i + 1 < x.dim(); i++) TORCH_CHECK_VALUE(x.size(i) == y.size(i), "x and y must have the same tokens");
    const int64_t T = x.numel() / K;
    const at::Tensor ids = list_of(a[4], "ids", at::kInt, T, x);
    at::Tensor scales, ranks;
    if (given(a[5])) scales = list_of(a[5], "scales", at::kFloat, E, x);
    if (given(a[6])) ranks = list_of(a[6], "ranks", at::kInt, E, x);
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out;
    if (given(a[7])) {
        out = output(a[7], "out", type, x);
        TORCH_CHECK_VALUE(out.sizes() == y.sizes() && (out.is_contiguous() || (out.dim() == 2 && out.stride(1) == 1 && out.stride(0) >= N)),
                          "out must have y's shape and contiguous rows");
    } else {
        out = at::empty(y.sizes(), y.options().memory_format(at::MemoryFormat::Contiguous));
    }
    // rows of tokens; those that lie otherwise are copied
    if (x.dim() != 2) x = x.reshape({T, K});
    if (y.dim() != 2) y = y.reshape({T, N});
    const at::Tensor out2 = out.dim() == 2 ? out : out.view({T, N});
    if ((x.stride(1) != 1 && K > 1) || !aligned(x) || x.stride(0) % 8) x = x.clone(at::MemoryFormat::Contiguous);
    if (y.stride(1) != 1 && N > 1) y = y.contiguous();
    ortho_b200_low_rank_desc d;
    memset(&d, 0, sizeof(d));
    d.x = ptr<void>(x); d.y = ptr<void>(y); d.out = ptr<void>(out2); d.down = ptr<void>(down); d.up = ptr<void>(up);
    d.scales = scales.defined() ? ptr<float>(scales) : nullptr; d.ranks = ranks.defined() ? ptr<int32_t>(ranks) : nullptr; d.ids = ptr<int32_t>(ids);
    d.tokens = T; d.K = K; d.N = N; d.adapters = E; d.rank = R;
    d.x_stride = x.stride(0); d.y_stride = y.stride(0); d.out_stride = out2.stride(0); d.type = type_number(type);
    int st = 0;
    if (T) {
        const int64_t need = low_rank_ws_c(&d);
        at::Tensor ws;
        if (need > 0) ws = scratch(need, x);
        void *wsp = need > 0 ? ws.mutable_data_ptr() : nullptr, *stream = current_stream(x);
        Py_BEGIN_ALLOW_THREADS
        st = low_rank_c(&d, wsp, need, stream);
        Py_END_ALLOW_THREADS
    }
    check_status(st, "ortho_b200_low_rank_add");
    return given(a[7]) ? Py_NewRef(a[7]) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// addresses in the loaded library, in the order below
PyObject *set_operators(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    if (n != 8) { PyErr_SetString(PyExc_TypeError, "set_operators takes 8 arguments"); return nullptr; }
    void *p[8];
    for (int i = 0; i < 8; i++) p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
    page_step_c = reinterpret_cast<decltype(page_step_c)>(p[0]);
    rotary_append_c = reinterpret_cast<decltype(rotary_append_c)>(p[1]);
    attention_c = reinterpret_cast<decltype(attention_c)>(p[2]);
    attention_ws_c = reinterpret_cast<decltype(attention_ws_c)>(p[3]);
    low_rank_c = reinterpret_cast<decltype(low_rank_c)>(p[4]);
    low_rank_ws_c = reinterpret_cast<decltype(low_rank_ws_c)>(p[5]);
    strerror_c = reinterpret_cast<decltype(strerror_c)>(p[6]);
    last_cuda_error_c = reinterpret_cast<decltype(last_cuda_error_c)>(p[7]);
    Py_RETURN_NONE;
}

}  // namespace

PyMethodDef ortho_operator_methods[] = {
    {"page_step", (PyCFunction)(void (*)(void))page_step, METH_FASTCALL, nullptr},
    {"rotary_append", (PyCFunction)(void (*)(void))rotary_append, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
    {"low_rank_add", (PyCFunction)(void (*)(void))low_rank_add, METH_FASTCALL, nullptr},
    {"set_operators", (PyCFunction)(void (*)(void))set_operators, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
