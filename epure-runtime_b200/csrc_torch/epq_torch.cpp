// The Python binding of include/epq_paged.h and include/epq_sampling.h: module epure._epq_torch.
//
// The calls of a decode step are a few microseconds of GPU work each, so what a call
// costs on the host is what a small step costs.  These functions take tensors straight
// from their Python objects, check them, allocate outputs and make the C call in 1.4 us
// besides the launch (4 to 5 with it); the same through ctypes took 20 to 30.  libepq.so is
// bound by address (bind()), so the library that EPURE_LIBEPQ names is the one called.
// Every failure raises: TypeError for a type that no kernel takes, RuntimeError for the
// rest.  Python's side of it is epure/_native.py.
#include <Python.h>
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <map>
#include <sstream>
#include <stdexcept>
#include <string>

#include "epq_paged.h"
#include "epq_sampling.h"

namespace {

using at::Tensor;

struct TypeProblem : std::runtime_error {
    using std::runtime_error::runtime_error;
};

// An exception that Python has already set.
struct PythonError {};

template <typename... A> std::string text(const A&... a) {
    std::ostringstream o;
    o << "epure: ";
    (o << ... << a);
    return o.str();
}
template <typename... A> [[noreturn]] void refuse(const A&... a) { throw std::runtime_error(text(a...)); }

// ---------------------------------------------------------------- libepq.so
struct Library {
    decltype(&epq_last_error) last_error = nullptr;
    decltype(&epq_rope) rope = nullptr;
    decltype(&epq_paged_write) write = nullptr;
    decltype(&epq_paged_read) read = nullptr;
    decltype(&epq_paged_attend) attend = nullptr;
    decltype(&epq_paged_attend_workspace_bytes) attend_bytes = nullptr;
    decltype(&epq_paged_attend_blocks) attend_blocks = nullptr;
    decltype(&epq_paged_attend_shared) attend_shared = nullptr;
    decltype(&epq_paged_attend_shared_workspace_bytes) shared_bytes = nullptr;
    decltype(&epq_paged_bounds) bounds = nullptr;
    decltype(&epq_paged_select) select = nullptr;
    decltype(&epq_paged_select_workspace_bytes) select_bytes = nullptr;
    decltype(&epq_verify_drafts) verify = nullptr;
} lib;

template <typename F> void find(void* h, const char* name, F& f) {
    f = reinterpret_cast<F>(dlsym(h, name));
    if (!f) refuse("libepq.so does not export ", name);
}

void check(int rc, const char* what) {
    if (rc != EPQ_OK) refuse(what, " failed (status ", rc, "): ", lib.last_error());
}

// ---------------------------------------------------------------- arguments
const Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) throw TypeProblem(text(what, " must be a tensor"));
    return THPVariable_Unpack(o);
}
const Tensor* maybe(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

int64_t integer(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw TypeProblem("epure: an integer is expected");
    }
    return v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw TypeProblem("epure: a number is expected");
    }
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PythonError();
    return v == 1;
}

int dtype_code(at::ScalarType t) {
    if (t == at::kFloat) return EPQ_F32;
    if (t == at::kHalf) return EPQ_F16;
    if (t == at::kBFloat16) return EPQ_BF16;
    throw TypeProblem(text("dtype ", t, " is not supported by the CUDA kernels"));
}

// These calls record nothing for autograd: a tensor whose derivative they would drop is refused, as torch's own
// out= functions refuse it.  (rope's gradient is _RopeFn's, whose calls come without grad mode.)
struct Named {
    const Tensor* t;
    const char* name;
};
void no_gradient(const char* call, std::initializer_list<Named> tensors) {
    const bool grads = c10::GradMode::is_enabled();
    for (const Named& n : tensors) {
        if (!n.t) continue;
        if (grads && n.t->requires_grad())
            refuse(n.name, " requires a gradient, which ", call, " does not pass on; detach it or call under torch.no_grad()");
        if (n.t->_fw_grad(0).defined())
            refuse(n.name, " has a forward-mode tangent, which ", call, " does not pass on");
    }
}

// Counts a write into a tensor that the caller gave, so that a backward which saved its old values finds out.
// (Inference tensors have no count.)
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The stride of a dimension, or `alone` where it has one element and its stride says nothing.
int64_t step(const Tensor& t, int d, int64_t alone) { return t.size(d) > 1 ? t.stride(d) : alone; }

// A strided tensor [rows, heads, head_dim]; negative sizes are not checked.
epq_heads heads_of(const Tensor& t, const char* what, const at::Device& dev, at::ScalarType dtype, int64_t rows,
                   int64_t heads, int64_t head_dim) {
    if (t.dim() != 3 || t.device() != dev || t.scalar_type() != dtype)
        refuse(what, " must be [rows, heads, head_dim], ", dtype, " on ", dev, "; got ", t.sizes(), ", ", t.scalar_type(),
               " on ", t.device());
    if ((rows >= 0 && t.size(0) != rows) || (heads >= 0 && t.size(1) != heads) || (head_dim >= 0 && t.size(2) != head_dim))
        refuse(what, " is ", t.sizes(), "; expected [", rows, ", ", heads, ", ", head_dim, "] (-1: any)");
    if (t.size(1) > INT32_MAX) refuse(what, " has ", t.size(1), " heads");
    if (t.numel() && t.stride(2) != 1) refuse("the values of a head of ", what, " must be contiguous (stride ", t.stride(2), ")");
    return {t.data_ptr(), step(t, 0, 0), step(t, 1, 0), (int32_t)t.size(1), 0};
}

const Tensor& index_of(const Tensor& t, const char* what, const at::Device& dev, at::ScalarType dtype, int64_t n) {
    if (t.scalar_type() != dtype || t.device() != dev || t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1))
        refuse(what, " must be ", n, " contiguous ", dtype, " on ", dev, "; got ", t.sizes(), ", ", t.scalar_type(), " on ",
               t.device());
    return t;
}

struct Tables {
    const float* cos = nullptr;
    const float* sin = nullptr;
    int64_t max_len = 0;
    int32_t rotary_dim = 0;
};
Tables tables_of(const Tensor& c, const Tensor& s, const at::Device& dev, int64_t head_dim) {
    if (c.dim() != 2 || c.sizes() != s.sizes() || c.scalar_type() != at::kFloat || s.scalar_type() != at::kFloat ||
        c.device() != dev || s.device() != dev || !c.is_contiguous() || !s.is_contiguous())
        refuse("cos and sin must be contiguous float32 [max_len, rotary_dim / 2] tables on the tensors' device");
    if (c.size(1) < 1 || c.size(1) > head_dim / 2 || c.size(0) < 1)
        refuse("rotary tables of ", c.sizes(), " for a head of ", head_dim);
    return {c.const_data_ptr<float>(), s.const_data_ptr<float>(), c.size(0), (int32_t)(2 * c.size(1))};
}

// A cache from five arguments: k, v, table, k_scale, v_scale.
struct Cache {
    epq_pages p;
    at::ScalarType dtype;
    at::Device device = at::kCPU;
};
Cache cache_of(PyObject* const* a) {
    const Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &table = tensor(a[2], "table");
    const Tensor *ks = maybe(a[3], "k_scale"), *vs = maybe(a[4], "v_scale");
    Cache c;
    c.dtype = k.scalar_type();
    c.device = k.device();
    int fmt;
    if (c.dtype == at::kChar) fmt = EPQ_CACHE_INT8;
    else if (c.dtype == at::kFloat8_e4m3fn) fmt = EPQ_CACHE_FP8;
    else if (c.dtype == at::kBFloat16 || c.dtype == at::kHalf || c.dtype == at::kFloat) fmt = EPQ_CACHE_SAME;
    else throw TypeProblem(text("a cache of ", c.dtype, " is not supported"));
    if (!k.is_cuda()) refuse("the paged cache needs CUDA tensors");
    if (k.dim() != 4 || v.sizes() != k.sizes() || v.scalar_type() != c.dtype || v.device() != c.device)
        refuse("k and v must be alike, [pages, kv_heads, page_size, head_dim]");
    const int64_t kv = k.size(1), ps = k.size(2), hd = k.size(3), page = step(k, 0, kv * ps * hd);
    for (const Tensor* t : {&k, &v})
        if (step(*t, 3, 1) != 1 || step(*t, 2, hd) != hd || step(*t, 1, ps * hd) != ps * hd)
            refuse("the heads, slots and values of a page must be contiguous (strides ", t->strides(), ")");
    if (step(v, 0, page) != page) refuse("k and v must be alike: pages ", page, " and ", v.stride(0), " values apart");
    if (table.dim() != 2 || table.scalar_type() != at::kInt || table.device() != c.device || step(table, 1, 1) != 1)
        refuse("the page table must be int32 [seqs, max_pages] on the cache's device");
    if (std::max({kv, ps, hd, table.size(0), table.size(1)}) > INT32_MAX) refuse("a size of the cache is past 2^31");
    int64_t stride = 0;
    if (fmt != EPQ_CACHE_SAME) {
        if (!ks || !vs) refuse("an 8-bit cache needs k_scale and v_scale");
        for (const Tensor* s : {ks, vs})
            if (s->dim() != 3 || s->size(0) != k.size(0) || s->size(1) != kv || s->size(2) != ps || s->scalar_type() != at::kFloat ||
                s->device() != c.device || step(*s, 2, 1) != 1 || step(*s, 1, ps) != ps ||
                step(*s, 0, kv * ps) != step(*ks, 0, kv * ps))
                refuse("scales must be float32 [pages, kv_heads, page_size], pages contiguous");
        stride = step(*ks, 0, kv * ps);
    } else if (ks || vs) {
        refuse("a cache of ", c.dtype, " has no scales");
    }
    c.p = {k.data_ptr(), v.data_ptr(), ks ? ks->data_ptr<float>() : nullptr, vs ? vs->data_ptr<float>() : nullptr,
           table.const_data_ptr<int32_t>(), page, stride, step(table, 0, table.size(1)), k.size(0), (int32_t)table.size(0),
           (int32_t)table.size(1), (int32_t)ps, (int32_t)kv, (int32_t)hd, fmt};
    return c;
}

// The tensors' device as the current one, for the length of a call.
struct OnDevice {
    int before = -1;
    explicit OnDevice(const at::Device& dev) {
        const int now = c10::cuda::current_device();
        if (dev.index() != now) {
            before = now;
            c10::cuda::set_device(dev.index());
        }
    }
    ~OnDevice() {
        if (before >= 0) c10::cuda::set_device((c10::DeviceIndex)before);
    }
};
cudaStream_t stream_of(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, const at::Device& dev) {
    // at::empty's own function for CUDA: outputs need no dispatch (about 0.4 us each)
    return at::detail::empty_cuda(sizes, dtype, dev, std::nullopt);
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap2(const Tensor& a, const Tensor& b) {
    PyObject* x = wrap(a);
    PyObject* y = x ? wrap(b) : nullptr;
    PyObject* t = y ? PyTuple_New(2) : nullptr;
    if (!t) {
        Py_XDECREF(x);
        Py_XDECREF(y);
        return nullptr;
    }
    PyTuple_SET_ITEM(t, 0, x);
    PyTuple_SET_ITEM(t, 1, y);
    return t;
}

// The attention's zeroed workspace: one a stream, grown on demand; inside a capture one a
// capture, zeroed in the graph at every replay, so that a graph shares none with what
// runs outside it.
Tensor workspace(const at::Device& dev, cudaStream_t st, int64_t bytes) {
    struct Held {
        Tensor t;
        unsigned long long capture = 0;
    };
    // never destroyed: at exit the CUDA context may be gone first
    static auto* eager = new std::map<std::pair<int, cudaStream_t>, Held>();
    static auto* captured = new std::map<std::pair<int, cudaStream_t>, Held>();
    cudaStreamCaptureStatus status;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(st, &status, &id) != cudaSuccess) refuse("cudaStreamGetCaptureInfo failed");
    const bool capturing = status == cudaStreamCaptureStatusActive;
    Held& h = (capturing ? *captured : *eager)[{dev.index(), st}];
    if (!h.t.defined() || h.t.numel() < bytes || (capturing && h.capture != id)) {
        h.t = at::zeros({bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
        h.capture = id;
    }
    return h.t;
}

// ---------------------------------------------------------------- calls
// rope(q, k | None, pos, cos, sin, interleaved, inverse, q_out | None, k_out | None)
PyObject* rope(PyObject* const* a) {
    const Tensor& q = tensor(a[0], "q");
    const Tensor* k = maybe(a[1], "k");
    const Tensor *qo = maybe(a[7], "q_out"), *ko = maybe(a[8], "k_out");
    if (!q.is_cuda()) refuse("rope needs CUDA tensors");
    no_gradient(qo || ko ? "rope with out" : "rope", {{&q, "q"}, {k, "k"}, {&tensor(a[3], "cos"), "cos"}, {&tensor(a[4], "sin"), "sin"},
                                                      {qo, "out"}, {ko, "out"}});
    if (q.dim() != 3) refuse("a rope input must be [rows, heads, head_dim]; got ", q.sizes());
    const at::Device dev = q.device();
    const at::ScalarType dt = q.scalar_type();
    const int64_t m = q.size(0), hd = q.size(2);
    const int code = dtype_code(dt);
    if (hd > INT32_MAX) refuse("heads of ", hd, " values");
    OnDevice on(dev);
    epq_heads in[2], out[2];
    in[0] = heads_of(q, "a rope input", dev, dt, m, -1, hd);
    if (k) in[1] = heads_of(*k, "a rope input", dev, dt, m, -1, hd);
    const Tensor& pos = index_of(tensor(a[2], "pos"), "pos", dev, at::kLong, m);
    const Tables t = tables_of(tensor(a[3], "cos"), tensor(a[4], "sin"), dev, hd);
    const Tensor y = qo ? *qo : empty(q.sizes(), dt, dev);
    const Tensor z = !k ? Tensor() : ko ? *ko : empty(k->sizes(), dt, dev);
    out[0] = heads_of(y, "a rope output", dev, dt, m, q.size(1), hd);
    if (k) out[1] = heads_of(z, "a rope output", dev, dt, m, k->size(1), hd);
    check(lib.rope(in, out, k ? 2 : 1, pos.const_data_ptr<int64_t>(), m, (int32_t)hd, t.rotary_dim, t.cos, t.sin, t.max_len,
                   truth(a[5]), truth(a[6]), code, stream_of(dev)),
          "epq_rope");
    if (qo) written(*qo);
    if (k && ko) written(*ko);
    return k ? wrap2(y, z) : wrap(y);
}

// write(k_pool, v_pool, table, k_scale, v_scale, k, v, seq, pos, q | None, q_out | None, cos | None, sin | None,
//       interleaved, qk_norm, eps)
PyObject* write(PyObject* const* a) {
    const Cache c = cache_of(a);
    const Tensor &k = tensor(a[5], "k"), &v = tensor(a[6], "v");
    const Tensor *q = maybe(a[9], "q"), *qo = maybe(a[10], "q_out"), *cs = maybe(a[11], "cos"), *sn = maybe(a[12], "sin");
    no_gradient("write", {{&tensor(a[0], "k"), "the k pool"}, {&tensor(a[1], "v"), "the v pool"}, {maybe(a[3], "k_scale"), "k_scale"},
                          {maybe(a[4], "v_scale"), "v_scale"}, {&k, "k"}, {&v, "v"}, {q, "q"}, {qo, "q_out"}, {cs, "cos"}, {sn, "sin"}});
    const at::ScalarType dt = k.scalar_type();
    const int code = dtype_code(dt);
    if (c.p.format == EPQ_CACHE_SAME && c.dtype != dt) refuse("rows of ", dt, " for a cache of ", c.dtype);
    OnDevice on(c.device);
    const epq_heads kh = heads_of(k, "k", c.device, dt, -1, c.p.kv_heads, c.p.head_dim);
    const int64_t m = k.size(0);
    const epq_heads vh = heads_of(v, "v", c.device, dt, m, c.p.kv_heads, c.p.head_dim);
    const Tensor& seq = index_of(tensor(a[7], "seq"), "seq", c.device, at::kInt, m);
    const Tensor& pos = index_of(tensor(a[8], "pos"), "pos", c.device, at::kLong, m);
    if (!cs != !sn) refuse("cos and sin come together");
    if (qo && !q) refuse("q_out needs q");
    const Tables t = cs ? tables_of(*cs, *sn, c.device, c.p.head_dim) : Tables();
    epq_heads qh, oh;
    Tensor y;
    if (q) {
        qh = heads_of(*q, "q", c.device, dt, m, -1, c.p.head_dim);
        y = qo ? *qo : empty(q->sizes(), dt, c.device);
        oh = heads_of(y, "q_out", c.device, dt, m, q->size(1), c.p.head_dim);
    }
    check(lib.write(&c.p, q ? &qh : nullptr, q ? &oh : nullptr, &kh, &vh, seq.const_data_ptr<int32_t>(),
                    pos.const_data_ptr<int64_t>(), m, t.cos, t.sin, t.max_len, t.rotary_dim, truth(a[13]), truth(a[14]),
                    (float)number(a[15]), code, stream_of(c.device)),
          "epq_paged_write");
    for (int i : {0, 1, 3, 4})
        if (const Tensor* t = maybe(a[i], "a pool")) written(*t);
    if (q && qo) written(*qo);
    if (!q) Py_RETURN_NONE;
    return wrap(y);
}

// read(k_pool, v_pool, table, k_scale, v_scale, seq, pos, dtype | None)
PyObject* read(PyObject* const* a) {
    const Cache c = cache_of(a);
    no_gradient("read", {{&tensor(a[0], "k"), "the k pool"}, {&tensor(a[1], "v"), "the v pool"}, {maybe(a[3], "k_scale"), "k_scale"},
                         {maybe(a[4], "v_scale"), "v_scale"}});
    at::ScalarType dt = c.p.format == EPQ_CACHE_SAME ? c.dtype : at::kBFloat16;
    if (a[7] != Py_None) {
        if (!THPDtype_Check(a[7])) throw TypeProblem("epure: dtype must be a torch.dtype");
        dt = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
    }
    const int code = dtype_code(dt);
    if (c.p.format == EPQ_CACHE_SAME && c.dtype != dt) refuse("a cache of ", c.dtype, " is read as ", c.dtype, ", not ", dt);
    OnDevice on(c.device);
    const Tensor& pos = tensor(a[6], "pos");
    const int64_t m = pos.dim() == 1 ? pos.size(0) : -1;
    index_of(pos, "pos", c.device, at::kLong, m);
    const Tensor& seq = index_of(tensor(a[5], "seq"), "seq", c.device, at::kInt, m);
    const Tensor k = empty({m, c.p.kv_heads, c.p.head_dim}, dt, c.device), v = empty({m, c.p.kv_heads, c.p.head_dim}, dt, c.device);
    check(lib.read(&c.p, seq.const_data_ptr<int32_t>(), pos.const_data_ptr<int64_t>(), m, k.data_ptr(), v.data_ptr(),
                   code, stream_of(c.device)),
          "epq_paged_read");
    return wrap2(k, v);
}

// The tensors that the attentions have in common; `a` holds the cache, q and lengths, then what a form has of its own.
struct Attention {
    Cache c;
    Tensor q, out, lse;
    epq_heads heads;
    const int64_t* lengths;
    const int32_t* seq;
    int64_t batch;
    double scale;
    int dtype;
    // `align`: bytes that q is read at once; another q is copied
    Attention(PyObject* const* a, PyObject* seq_, PyObject* scale_, PyObject* out_, PyObject* lse_, const char* call, int align)
        : c(cache_of(a)), q(tensor(a[5], "q")) {
        const Tensor& n = tensor(a[6], "lengths");
        const Tensor *s = maybe(seq_, "seq"), *to = maybe(out_, "out");
        no_gradient(call, {{&tensor(a[0], "k"), "the k pool"}, {&tensor(a[1], "v"), "the v pool"}, {maybe(a[3], "k_scale"), "k_scale"},
                           {maybe(a[4], "v_scale"), "v_scale"}, {&q, "q"}, {to, "out"}});
        const at::ScalarType dt = q.scalar_type();
        if (dt != at::kBFloat16 && dt != at::kHalf)
            throw TypeProblem(text("paged attention takes float16 or bfloat16 queries, not ", dt));
        if (c.p.format == EPQ_CACHE_SAME && c.dtype != dt) refuse("queries of ", dt, " for a cache of ", c.dtype);
        heads = heads_of(q, "q", c.device, dt, -1, -1, c.p.head_dim);
        batch = q.size(0);
        const int64_t H = q.size(1), hd = c.p.head_dim;
        lengths = index_of(n, "lengths", c.device, at::kLong, batch).const_data_ptr<int64_t>();
        seq = s ? index_of(*s, "seq", c.device, at::kInt, batch).const_data_ptr<int32_t>() : nullptr;
        if (to && (to->dim() != 3 || to->size(0) != batch || to->size(1) != H || to->size(2) != hd || to->scalar_type() != dt ||
                   to->device() != c.device || !to->is_contiguous()))
            refuse("out must be contiguous [", batch, ", ", H, ", ", hd, "], ", dt, " on ", c.device);
        scale = scale_ == Py_None ? 1.0 / std::sqrt((double)hd) : number(scale_);
        dtype = dtype_code(dt);
        OnDevice on(c.device);
        const bool expanded = (batch > 1 && heads.stride_row == 0) || (H > 1 && heads.stride_head == 0);
        if (((uintptr_t)heads.data | (uintptr_t)(2 * heads.stride_row) | (uintptr_t)(2 * heads.stride_head)) % align ||
            (expanded && align == 16)) {
            q = q.clone(at::MemoryFormat::Contiguous);
            heads = heads_of(q, "q", c.device, dt, batch, H, hd);
        }
        given = to;
        out = to ? *to : empty({batch, H, hd}, dt, c.device);
        if (truth(lse_)) lse = empty({batch, H}, at::kFloat, c.device);
    }
    float* lse_to() const { return lse.defined() ? lse.data_ptr<float>() : nullptr; }
    PyObject* results() const {
        if (given) written(*given);
        return lse.defined() ? wrap2(out, lse) : wrap(out);
    }

  private:
    const Tensor* given;
};

// attend(k_pool, v_pool, table, k_scale, v_scale, q, lengths, seq | None, scale | None, window, out | None, return_lse,
//        blocks | None)
PyObject* attend(PyObject* const* a) {
    const int64_t window = integer(a[9]);
    const Tensor* blocks = maybe(a[12], "blocks");
    const Attention t(a, a[7], a[8], a[10], a[11], "attend", 4);
    const Cache& c = t.c;
    if (blocks) {
        if (blocks->dim() != 3 || blocks->size(0) != t.batch || blocks->size(1) != c.p.kv_heads || blocks->scalar_type() != at::kInt ||
            blocks->device() != c.device || !blocks->is_contiguous() || blocks->size(2) > INT32_MAX)
            refuse("blocks must be contiguous int32 [", t.batch, ", ", c.p.kv_heads, ", count] on ", c.device, "; got ",
                   blocks->sizes(), ", ", blocks->scalar_type(), " on ", blocks->device());
        if (window) refuse("attention over listed blocks has no window");
    }
    OnDevice on(c.device);
    const int64_t need = lib.attend_bytes(&c.p, t.batch, t.heads.heads);
    if (need < 0) check((int)need, "epq_paged_attend_workspace_bytes");
    const cudaStream_t st = stream_of(c.device);
    const Tensor ws = workspace(c.device, st, need);
    if (blocks)
        check(lib.attend_blocks(&c.p, &t.heads, t.seq, t.lengths, t.batch, blocks->const_data_ptr<int32_t>(),
                                (int32_t)blocks->size(2), (float)t.scale, t.out.data_ptr(), t.lse_to(), t.dtype, ws.data_ptr(),
                                ws.numel(), st),
              "epq_paged_attend_blocks");
    else
        check(lib.attend(&c.p, &t.heads, t.seq, t.lengths, t.batch, (float)t.scale, window, t.out.data_ptr(), t.lse_to(), t.dtype,
                         ws.data_ptr(), ws.numel(), st),
              "epq_paged_attend");
    return t.results();
}

// attend_shared(k_pool, v_pool, table, k_scale, v_scale, q, lengths, starts, prefix, seq | None, scale | None, out | None,
//               return_lse, always)
PyObject* attend_shared(PyObject* const* a) {
    const Tensor &starts = tensor(a[7], "starts"), &prefix = tensor(a[8], "prefix");
    const Attention t(a, a[9], a[10], a[11], a[12], "attend_shared", 16);
    const Cache& c = t.c;
    const int64_t groups = prefix.dim() == 1 ? prefix.size(0) : -1;
    index_of(prefix, "prefix", c.device, at::kLong, groups);
    index_of(starts, "starts", c.device, at::kInt, groups + 1);
    OnDevice on(c.device);
    const int always = truth(a[13]);
    const int64_t need = lib.shared_bytes(&c.p, t.batch, t.heads.heads, groups, always);
    if (need < 0) check((int)need, "epq_paged_attend_shared_workspace_bytes");
    const cudaStream_t st = stream_of(c.device);
    const Tensor ws = workspace(c.device, st, need);
    check(lib.attend_shared(&c.p, &t.heads, t.seq, t.lengths, t.batch, starts.const_data_ptr<int32_t>(),
                            prefix.const_data_ptr<int64_t>(), groups, always, (float)t.scale, t.out.data_ptr(), t.lse_to(), t.dtype,
                            ws.data_ptr(), ws.numel(), st),
          "epq_paged_attend_shared");
    return t.results();
}

// The bounds of a cache's pages: [pages, kv_heads, 2, head_dim] of its own type, bfloat16 for 8-bit ones.
int64_t check_bounds(const Tensor& t, const Cache& c) {
    const at::ScalarType dt = c.p.format == EPQ_CACHE_SAME ? c.dtype : at::kBFloat16;
    if (dt == at::kFloat) throw TypeProblem("epure: a float32 cache has no bounds");
    const int64_t hd = c.p.head_dim, page = c.p.kv_heads * 2 * hd;
    if (t.dim() != 4 || t.size(0) != c.p.pages || t.size(1) != c.p.kv_heads || t.size(2) != 2 || t.size(3) != hd ||
        t.scalar_type() != dt || t.device() != c.device || step(t, 3, 1) != 1 || step(t, 2, hd) != hd || step(t, 1, 2 * hd) != 2 * hd)
        refuse("bounds must be [", c.p.pages, ", ", c.p.kv_heads, ", 2, ", hd, "], ", dt, " on ", c.device,
               ", the values of a page contiguous; got ", t.sizes(), ", ", t.scalar_type(), " on ", t.device());
    return step(t, 0, page);
}

// bounds(k_pool, v_pool, table, k_scale, v_scale, bounds, lengths, seq | None, first | None)
PyObject* bounds(PyObject* const* a) {
    const Cache c = cache_of(a);
    const Tensor &to = tensor(a[5], "bounds"), &lengths = tensor(a[6], "lengths");
    const Tensor *seq = maybe(a[7], "seq"), *first = maybe(a[8], "first");
    no_gradient("summarise", {{&tensor(a[0], "k"), "the k pool"}, {&tensor(a[1], "v"), "the v pool"}, {maybe(a[3], "k_scale"), "k_scale"},
                              {maybe(a[4], "v_scale"), "v_scale"}, {&to, "bounds"}});
    const int64_t stride = check_bounds(to, c), B = lengths.dim() == 1 ? lengths.size(0) : -1;
    index_of(lengths, "lengths", c.device, at::kLong, B);
    if (seq) index_of(*seq, "seq", c.device, at::kInt, B);
    if (first) index_of(*first, "first", c.device, at::kLong, B);
    OnDevice on(c.device);
    check(lib.bounds(&c.p, to.data_ptr(), stride, dtype_code(to.scalar_type()), seq ? seq->const_data_ptr<int32_t>() : nullptr,
                     first ? first->const_data_ptr<int64_t>() : nullptr, lengths.const_data_ptr<int64_t>(), B, stream_of(c.device)),
          "epq_paged_bounds");
    written(to);
    Py_RETURN_NONE;
}

// select(k_pool, v_pool, table, k_scale, v_scale, bounds, q, lengths, count, seq | None, sinks, recent)
PyObject* select(PyObject* const* a) {
    const Cache c = cache_of(a);
    const Tensor &from = tensor(a[5], "bounds"), &q = tensor(a[6], "q"), &lengths = tensor(a[7], "lengths");
    const Tensor* seq = maybe(a[9], "seq");
    const int64_t count = integer(a[8]), sinks = integer(a[10]), recent = integer(a[11]), most = INT32_MAX;
    const int64_t stride = check_bounds(from, c);
    const at::ScalarType dt = q.scalar_type();
    if (dt != at::kBFloat16 && dt != at::kHalf) throw TypeProblem(text("selection takes float16 or bfloat16 queries, not ", dt));
    const epq_heads qh = heads_of(q, "q", c.device, dt, -1, -1, c.p.head_dim);
    const int64_t B = q.size(0);
    index_of(lengths, "lengths", c.device, at::kLong, B);
    if (seq) index_of(*seq, "seq", c.device, at::kInt, B);
    if (count < 1 || sinks < 0 || recent < 0 || sinks > count || recent > count - sinks || count > most)
        refuse("count=", count, " blocks with sinks=", sinks, " and recent=", recent, " (sinks + recent <= count)");
    OnDevice on(c.device);
    const int64_t need = lib.select_bytes(&c.p, B);
    if (need < 0) check((int)need, "epq_paged_select_workspace_bytes");
    const Tensor chosen = empty({B, c.p.kv_heads, count}, at::kInt, c.device);
    const cudaStream_t st = stream_of(c.device);
    const Tensor ws = workspace(c.device, st, need);
    check(lib.select(&c.p, from.data_ptr(), stride, dtype_code(from.scalar_type()), &qh, dtype_code(dt),
                     seq ? seq->const_data_ptr<int32_t>() : nullptr, lengths.const_data_ptr<int64_t>(), B, (int32_t)count,
                     (int32_t)sinks, (int32_t)recent, chosen.data_ptr<int32_t>(), ws.data_ptr(), ws.numel(), st),
          "epq_paged_select");
    return wrap(chosen);
}

// verify(target, draft | None, tokens, uniforms)
PyObject* verify(PyObject* const* a) {
    const Tensor &p = tensor(a[0], "target"), &tokens = tensor(a[2], "tokens"), &u = tensor(a[3], "uniforms");
    const Tensor* q = maybe(a[1], "draft");
    if (!p.is_cuda()) refuse("verify needs CUDA tensors");
    const at::Device dev = p.device();
    const at::ScalarType dt = p.scalar_type();
    const int code = dtype_code(dt);
    if (p.dim() != 3 || p.size(1) < 1 || p.size(2) < 1 || step(p, 2, 1) != 1)
        refuse("target must be [batch, drafts + 1, vocab] with contiguous rows; got ", p.sizes(), ", strides ", p.strides());
    const int64_t B = p.size(0), K = p.size(1) - 1, V = p.size(2);
    if (K > INT32_MAX) refuse(K, " drafts");
    if (q && (q->dim() != 3 || q->size(0) != B || q->size(1) != K || q->size(2) != V || q->scalar_type() != dt || q->device() != dev ||
              (q->numel() && step(*q, 2, 1) != 1)))
        refuse("draft must be [", B, ", ", K, ", ", V, "] with contiguous rows, ", dt, " on ", dev, "; got ", q->sizes(), ", ",
               q->scalar_type(), " on ", q->device());
    if (tokens.dim() != 2 || tokens.size(0) != B || tokens.size(1) != K || tokens.scalar_type() != at::kLong || tokens.device() != dev ||
        step(tokens, 1, 1) != 1)
        refuse("tokens must be int64 [", B, ", ", K, "] on ", dev, ", rows contiguous; got ", tokens.sizes(), ", ",
               tokens.scalar_type(), " on ", tokens.device());
    if (u.dim() != 2 || u.size(0) != B || u.size(1) != K + 1 || u.scalar_type() != at::kFloat || u.device() != dev || step(u, 1, 1) != 1)
        refuse("uniforms must be float32 [", B, ", ", K + 1, "] on ", dev, ", rows contiguous; got ", u.sizes(), ", ",
               u.scalar_type(), " on ", u.device());
    OnDevice on(dev);
    const Tensor out = empty({B, K + 1}, at::kLong, dev), n = empty({B}, at::kLong, dev);
    const epq_probs target = {p.data_ptr(), step(p, 0, 0), step(p, 1, 0)};
    const epq_probs draft = q ? epq_probs{q->data_ptr(), step(*q, 0, 0), step(*q, 1, 0)} : epq_probs{};
    check(lib.verify(&target, q ? &draft : nullptr, tokens.const_data_ptr<int64_t>(), step(tokens, 0, 0), u.const_data_ptr<float>(),
                     step(u, 0, 0), B, (int32_t)K, V, code, out.data_ptr<int64_t>(), n.data_ptr<int64_t>(), stream_of(dev)),
          "epq_verify_drafts");
    return wrap2(out, n);
}

PyObject* out_of_memory = nullptr;         // torch.OutOfMemoryError

// bind(path of libepq.so, torch.OutOfMemoryError)
PyObject* bind(PyObject* const* a) {
    const char* path = PyUnicode_AsUTF8(a[0]);
    if (!path) {
        PyErr_Clear();
        throw TypeProblem("epure: a path is expected");
    }
    void* h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    if (!h) refuse(dlerror());
    find(h, "epq_last_error", lib.last_error);
    find(h, "epq_rope", lib.rope);
    find(h, "epq_paged_write", lib.write);
    find(h, "epq_paged_read", lib.read);
    find(h, "epq_paged_attend", lib.attend);
    find(h, "epq_paged_attend_workspace_bytes", lib.attend_bytes);
    find(h, "epq_paged_attend_blocks", lib.attend_blocks);
    find(h, "epq_paged_attend_shared", lib.attend_shared);
    find(h, "epq_paged_attend_shared_workspace_bytes", lib.shared_bytes);
    find(h, "epq_paged_bounds", lib.bounds);
    find(h, "epq_paged_select", lib.select);
    find(h, "epq_paged_select_workspace_bytes", lib.select_bytes);
    find(h, "epq_verify_drafts", lib.verify);
    Py_INCREF(a[1]);
    Py_XSETREF(out_of_memory, a[1]);
    Py_RETURN_NONE;
}

// Python's call of F with N arguments; no exception leaves it.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != N) throw TypeProblem(text(N, " arguments are expected, ", n, " were given"));
        if (F != bind && !lib.last_error) refuse("libepq.so is not bound");
        return F(args);
    } catch (const PythonError&) {
    } catch (const TypeProblem& e) {
        PyErr_SetString(PyExc_TypeError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(out_of_memory ? out_of_memory : PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

#define EPQ_METHOD(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&call<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {EPQ_METHOD(bind, 2),    EPQ_METHOD(rope, 9),           EPQ_METHOD(write, 16),
                         EPQ_METHOD(read, 8),    EPQ_METHOD(attend, 13),        EPQ_METHOD(attend_shared, 14),
                         EPQ_METHOD(bounds, 9),  EPQ_METHOD(select, 12),        EPQ_METHOD(verify, 4),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_epq_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__epq_torch() { return PyModule_Create(&module); }
