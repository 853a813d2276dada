// Python binding of the 4-bit KV cache operators (gb_kv_q4_*, include/ggmlc_b200.h) for torch
// tensors: the class behind ggmlc_b200.kv_q4.Q4KVCache.  It checks the tensors, finds the current
// stream and calls the C ABI; a decode step's calls are a few microseconds long, so none of that is
// left to the interpreter (the same in Python took 8 to 12 us a call, here 3 to 5).
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <optional>
#include <stdexcept>
#include <string>

#include "ggmlc_b200.h"

namespace py = pybind11;

namespace {

void require(bool ok, const char* what) {
    if (!ok) throw py::value_error(what);
}

int type_id(at::ScalarType t) {  // ggml type ids
    switch (t) {
        case at::kFloat: return 0;
        case at::kHalf: return 1;
        case at::kBFloat16: return 30;
        default: return -1;
    }
}

void check(int rc) {
    if (rc != 0) throw std::runtime_error(gb_last_error());
}

class Cache {
  public:
    Cache(at::Tensor k, at::Tensor v, int64_t head_dim, std::optional<at::Tensor> pages)
        : k_(std::move(k)), v_(std::move(v)), pages_(std::move(pages)) {
        for (const at::Tensor* t : {&k_, &v_})
            require(t->scalar_type() == at::kByte && t->dim() == 3 && t->is_contiguous() &&
                        t->is_cuda(),
                    "k and v must be contiguous uint8 CUDA tensors [n_pages, n_kv_heads, page_bytes]");
        require(k_.sizes() == v_.sizes() && k_.device() == v_.device(),
                "k and v must have one shape and device");
        require(head_dim > 0 && head_dim % 32 == 0, "head_dim must be a multiple of 32");
        const int64_t row = head_dim / 2 + head_dim / 16;
        const int64_t page_len = k_.size(2) / row;
        require(k_.size(2) % row == 0 && page_len > 0 && page_len % 16 == 0,
                "page_bytes must hold a multiple of 16 positions");
        c_.k = k_.data_ptr();
        c_.v = v_.data_ptr();
        c_.n_pages = k_.size(0);
        c_.page_len = page_len;
        c_.n_kv_heads = k_.size(1);
        c_.head_dim = head_dim;
        c_.pages = nullptr;
        c_.n_slots = 0;
        c_.pages_per_slot = 0;
        if (pages_) {
            require(pages_->scalar_type() == at::kInt && pages_->dim() == 2 &&
                        pages_->is_contiguous() && pages_->device() == k_.device(),
                    "pages must be a contiguous int32 tensor [n_slots, pages_per_slot] on the "
                    "cache's device");
            c_.pages = pages_->data_ptr<int32_t>();
            c_.n_slots = pages_->size(0);
            c_.pages_per_slot = pages_->size(1);
        }
        if (shared().handles++ == 0) shared().work = new ScratchMap;
    }
    Cache(const Cache&) = delete;
    Cache& operator=(const Cache&) = delete;
    ~Cache() {
        if (--shared().handles == 0) {
            delete shared().work;
            shared().work = nullptr;
        }
    }

    void write(const at::Tensor& k, const at::Tensor& v, const py::object& pos,
               const py::object& slot) {
        const int64_t n = rows_of(k, c_.n_kv_heads, "k");
        require(rows_of(v, c_.n_kv_heads, "v") == n && v.scalar_type() == k.scalar_type(),
                "k and v must have the same rows and dtype");
        const gb_kv_rows r = rows(n, pos, slot);
        const c10::cuda::OptionalCUDAGuard guard(k_.device());
        check(gb_kv_q4_write(&c_, &r, type_id(k.scalar_type()), k.data_ptr(), k.stride(0),
                             k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), stream()));
    }

    std::pair<at::Tensor, at::Tensor> read(const py::object& pos, const py::object& slot,
                                           at::ScalarType dtype, std::optional<int64_t> n_rows) {
        int64_t n = n_rows.value_or(-1);
        for (const py::object* x : {&pos, &slot})
            if (n < 0 && THPVariable_Check(x->ptr()) && THPVariable_Unpack(x->ptr()).dim() == 1)
                n = THPVariable_Unpack(x->ptr()).size(0);
        require(n >= 0, "rows must be given when pos and slot are ints");
        const int type = type_id(dtype);
        require(type >= 0, "dtype must be float32, float16 or bfloat16");
        const gb_kv_rows r = rows(n, pos, slot);
        const c10::cuda::OptionalCUDAGuard guard(k_.device());
        const int64_t shape[3] = {n, c_.n_kv_heads, c_.head_dim};
        at::Tensor k = at::detail::empty_cuda(shape, dtype, k_.device(), std::nullopt);
        at::Tensor v = at::detail::empty_cuda(shape, dtype, k_.device(), std::nullopt);
        check(gb_kv_q4_read(&c_, &r, type, k.data_ptr(), v.data_ptr(), stream()));
        return {std::move(k), std::move(v)};
    }

    at::Tensor attend(const at::Tensor& q, const py::object& pos, const py::object& slot,
                      std::optional<double> scale, int64_t max_kv, std::optional<at::Tensor> out) {
        const int64_t n = rows_of(q, -1, "q");
        const gb_kv_rows r = rows(n, pos, slot);
        const c10::cuda::OptionalCUDAGuard guard(k_.device());
        at::Tensor o;
        if (out) {
            o = *out;
            require(o.sizes() == q.sizes() && o.scalar_type() == q.scalar_type() &&
                        o.is_contiguous() && o.device() == k_.device(),
                    "out must be contiguous, of q's shape, dtype and device");
        } else {
            o = at::detail::empty_cuda(q.sizes(), q.scalar_type(), k_.device(), std::nullopt);
        }
        const cudaStream_t st = stream();
        const size_t need =
            gb_kv_q4_attend_workspace_bytes(&c_, r.pos || r.slot ? std::min<int64_t>(n, 1) : n, q.size(1));
        const at::Tensor& work = scratch(k_.device(), st, (int64_t)need);
        check(gb_kv_q4_attend(&c_, &r, type_id(q.scalar_type()), q.data_ptr(), q.stride(0),
                              q.stride(1), q.size(1), max_kv,
                              (float)scale.value_or(1.0 / std::sqrt((double)c_.head_dim)),
                              o.data_ptr(), work.data_ptr(), (size_t)work.numel(), st));
        return o;
    }

    at::Tensor k() const { return k_; }
    at::Tensor v() const { return v_; }
    std::optional<at::Tensor> pages() const { return pages_; }
    int64_t head_dim() const { return c_.head_dim; }
    int64_t page_len() const { return c_.page_len; }
    int64_t n_kv_heads() const { return c_.n_kv_heads; }
    int64_t capacity() const { return c_.page_len * (pages_ ? c_.pages_per_slot : 1); }

  private:
    cudaStream_t stream() const {
        return c10::cuda::getCurrentCUDAStream(k_.device().index()).stream();
    }

    // Split scratch, one per device and stream for all handles: calls on a stream run one after the
    // other (a handle a layer would hold 1.2 GB for 32 layers).  A call under capture never
    // gets the memory of eager calls, which a larger call replaces, nor another capture's, which may
    // replay at the same time or before it: each capture has its own, from the graph's pool, whose
    // counters its first call zeroes as a node of that graph.  The pool keeps it for as long as the
    // graph lives, also after the next capture on the stream has taken its place here.
    static const at::Tensor& scratch(at::Device device, cudaStream_t st, int64_t need) {
        cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
        unsigned long long id = 0;
        if (cudaStreamGetCaptureInfo(st, &status, &id) != cudaSuccess)
            throw std::runtime_error("Q4KVCache: the stream's capture status cannot be read");
        Scratch& s = (*shared().work)[{device.index(), st}];
        const bool capturing = status == cudaStreamCaptureStatusActive;
        at::Tensor& work = capturing ? s.captured : s.eager;
        if (!work.defined() || work.numel() < need || (capturing && s.capture != id)) {
            work = at::empty({need}, at::TensorOptions().dtype(at::kByte).device(device));
            // the counters are zero before the first call and after every one
            work.narrow(0, 0, std::min<int64_t>(need, GB_KV_Q4_WORK_ZEROED)).zero_();
            if (capturing) s.capture = id;
        }
        return work;
    }

    int64_t rows_of(const at::Tensor& x, int64_t heads, const char* what) const {
        if (x.dim() != 3 || x.size(2) != c_.head_dim || x.device() != k_.device() ||
            (heads >= 0 && x.size(1) != heads))
            throw py::value_error(std::string(what) + " must be [rows, heads, " +
                                  std::to_string(c_.head_dim) + "] on the cache's device");
        if (type_id(x.scalar_type()) < 0)
            throw py::value_error(std::string(what) + " must be float32, float16 or bfloat16");
        if (x.stride(2) != 1)
            throw py::value_error(std::string(what) + ": dims must be contiguous");
        return x.size(0);
    }

    // pos / slot: an int, or an int32 tensor of one value a row
    bool of(const py::object& x, int64_t n, const int32_t** array, int64_t* value) const {
        *array = nullptr;
        *value = 0;
        if (THPVariable_Check(x.ptr())) {
            const at::Tensor& t = THPVariable_Unpack(x.ptr());
            if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n ||
                !t.is_contiguous() || t.device() != k_.device())
                return false;
            *array = t.data_ptr<int32_t>();
            return true;
        }
        PyObject* i = PyNumber_Index(x.ptr());
        if (i) {
            *value = PyLong_AsLongLong(i);
            Py_DECREF(i);
        }
        if (PyErr_Occurred()) {
            PyErr_Clear();
            return false;
        }
        return true;
    }
    gb_kv_rows rows(int64_t n, const py::object& pos, const py::object& slot) const {
        gb_kv_rows r;
        r.n = n;
        require(of(pos, n, &r.pos, &r.pos0),
                "pos must be an int or a contiguous int32 tensor of one value a row on the cache's "
                "device");
        require(of(slot, n, &r.slot, &r.slot0),
                "slot must be an int or a contiguous int32 tensor of one value a row on the "
                "cache's device");
        return r;
    }

    at::Tensor k_, v_;
    std::optional<at::Tensor> pages_;
    gb_kv_q4 c_{};
    struct Scratch {
        at::Tensor eager, captured;
        unsigned long long capture = 0;  // the capture `captured` belongs to
    };
    using ScratchMap = std::map<std::pair<int, cudaStream_t>, Scratch>;
    // of the process, freed with its last handle; under the interpreter's lock, like every call here
    struct Shared {
        int handles = 0;
        ScratchMap* work = nullptr;
    };
    static Shared& shared() {
        static Shared s;
        return s;
    }
};

}  // namespace

PYBIND11_MODULE(_kv_q4, m) {
    py::class_<Cache>(m, "Cache")
        .def(py::init<at::Tensor, at::Tensor, int64_t, std::optional<at::Tensor>>(), py::arg("k"),
             py::arg("v"), py::arg("head_dim"), py::arg("pages") = py::none())
        .def("write", &Cache::write, py::arg("k"), py::arg("v"), py::arg("pos"),
             py::arg("slot") = py::int_(0),
             "Quantise rows k, v [rows, n_kv_heads, head_dim] (any row and head strides) into "
             "positions pos of sequences slot; rows outside the cache are skipped.")
        .def("read", &Cache::read, py::arg("pos"), py::arg("slot") = py::int_(0),
             py::arg("dtype") = at::kFloat, py::arg("rows") = py::none(),
             "The values of rows as (k, v), each [rows, n_kv_heads, head_dim]; rows outside the "
             "cache are zeros.  rows is needed when pos and slot are both ints.")
        .def("attend", &Cache::attend, py::arg("q"), py::arg("pos"), py::arg("slot") = py::int_(0),
             py::arg("scale") = py::none(), py::arg("max_kv") = 0, py::arg("out") = py::none(),
             "Attention of q [rows, heads, head_dim]: row r sees positions 0 .. pos[r] of sequence "
             "slot[r] (at most max_kv of them when positive).  scale: 1 / sqrt(head_dim) unless "
             "given.  Returns [rows, heads, head_dim] of q's dtype (out when given).")
        .def_property_readonly("k", &Cache::k)
        .def_property_readonly("v", &Cache::v)
        .def_property_readonly("pages", &Cache::pages)
        .def_property_readonly("head_dim", &Cache::head_dim)
        .def_property_readonly("page_len", &Cache::page_len)
        .def_property_readonly("n_kv_heads", &Cache::n_kv_heads)
        .def_property_readonly("capacity", &Cache::capacity, "Positions a sequence can hold.")
        .def_property_readonly("device", [](const Cache& c) { return c.k().device(); });
}
