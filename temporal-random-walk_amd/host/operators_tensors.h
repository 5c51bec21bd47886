// operators_tensors.h -- what the operators' PyTorch modules share: argument
// checks, rows that the kernels can read, the terms of a score, and results that
// have no gradient.
#ifndef TRW_OPERATORS_TENSORS_H
#define TRW_OPERATORS_TENSORS_H

#include <ATen/ATen.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/custom_class.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>

#include "trw_operators.h"

namespace py = pybind11;
using at::Tensor;
using OptionalTensor = std::optional<Tensor>;

namespace {

constexpr int64_t kMaxRows = int64_t{1} << 30;
// Rows lie at most this far apart (elements); others are copied.
constexpr int64_t kMaxRowStride = int64_t{1} << 22;

struct OutOfMemory : py::builtin_exception {
    using py::builtin_exception::builtin_exception;
    void set_error() const override { PyErr_SetString(PyExc_MemoryError, what()); }
};

#define REQUIRE(ok, message) \
    do {                     \
        if (!(ok)) throw py::value_error(message); \
    } while (0)

void check_status(trw_status status) {
    if (status == TRW_OK) return;
    const char* message = trw_ops_last_error();
    if (status == TRW_ERR_INVALID_ARGUMENT) throw py::value_error(message);
    if (status == TRW_ERR_OUT_OF_MEMORY) throw OutOfMemory(message);
    throw std::runtime_error(message);
}

void on_gpu(const char* name, const Tensor& x) {
    if (!x.is_cuda()) throw py::value_error(std::string(name) + " must be on the GPU");
}
void on_gpu(const char* name, const Tensor& x, const Tensor& beside) {
    on_gpu(name, x);
    if (x.device() != beside.device())
        throw py::value_error(std::string(name) + " is on another device");
}
bool has_shape(const Tensor& x, at::IntArrayRef shape) { return x.sizes() == shape; }
[[noreturn]] void wrong_shape(const char* name, at::IntArrayRef shape) {
    std::string s;
    for (int64_t n : shape) s += (s.empty() ? "" : ", ") + std::to_string(n);
    throw py::value_error(std::string(name) + " must have the shape [" + s + "]");
}

// An int64 tensor of one shape (a view or a copy of what was given).
Tensor ints(const char* name, const Tensor& x, at::IntArrayRef shape, const Tensor& beside) {
    on_gpu(name, x, beside);
    if (!at::isIntegralType(x.scalar_type(), /*includeBool=*/false))
        throw py::value_error(std::string(name) + " must hold whole numbers");
    if (!has_shape(x, shape)) wrong_shape(name, shape);
    return (x.scalar_type() == at::kLong ? x : x.to(at::kLong)).contiguous();
}

Tensor floats(const char* name, const Tensor& x, at::IntArrayRef shape, const Tensor& beside) {
    on_gpu(name, x, beside);
    if (x.scalar_type() != at::kFloat)
        throw py::value_error(std::string(name) + " must be float32");
    if (!has_shape(x, shape)) wrong_shape(name, shape);
    if (x.requires_grad() && at::GradMode::is_enabled())
        throw py::value_error(std::string(name) + " has no gradient here");
    return x.contiguous();
}

int dtype_of(const Tensor& x, const char* message) {
    switch (x.scalar_type()) {
        case at::kFloat: return TRW_F32;
        case at::kHalf: return TRW_F16;
        case at::kBFloat16: return TRW_BF16;
        default: throw py::value_error(message);
    }
}

// Whether rows of the last dimension can be read 16 bytes at a time.
bool in_pieces(const Tensor& x) {
    if (x.stride(-1) != 1 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) return false;
    const int64_t per = 16 / x.element_size();
    for (int64_t d = 0; d + 1 < x.dim(); ++d)
        if (x.stride(d) % per) return false;
    return true;
}
// [rows, heads, dim] that the kernels can read: the tensor, or a copy where its
// rows are not 16-byte pieces or lie further apart than they count.
Tensor readable(const Tensor& x) {
    if (x.numel() == 0 || (in_pieces(x) && x.stride(0) <= kMaxRowStride)) return x;
    return x.clone(at::MemoryFormat::Contiguous);
}
trw_rows rows_of(const Tensor& x) { return trw_rows{x.data_ptr(), x.stride(0), x.stride(1)}; }

template <typename T>
T* pointer(const OptionalTensor& x) {
    return x ? static_cast<T*>(x->data_ptr()) : nullptr;
}
template <typename T>
T* pointer(const Tensor& x) {
    return x.defined() ? static_cast<T*>(x.data_ptr()) : nullptr;
}

Tensor bytes(uint64_t n, const Tensor& beside) {
    return at::empty({static_cast<int64_t>(n)}, beside.options().dtype(at::kByte));
}

// The tensors' device and its current stream, for the calls in a scope.
struct OnDevice {
    c10::hip::OptionalHIPGuard guard;
    void* stream;
    explicit OnDevice(const Tensor& x) {
        if (c10::hip::current_device() != x.get_device()) guard.set_index(x.get_device());
        stream = c10::hip::getCurrentHIPStream(x.get_device()).stream();
    }
};

Tensor as_rows(const Tensor& x) { return readable(x.dim() == 4 ? x.flatten(0, 1) : x); }

bool differentiable(const Tensor& x) {
    return at::GradMode::is_enabled() && x.requires_grad();
}
// Which of the arguments a gradient is asked of.  none: what says that there is none.
torch::autograd::variable_list differentiated_of(const char* none,
                                                 std::initializer_list<OptionalTensor> given) {
    torch::autograd::variable_list which;
    for (const OptionalTensor& x : given) {
        if (!x || !x->defined()) continue;
        if (x->_fw_grad(/*level=*/0).defined()) throw std::runtime_error(none);
        if (differentiable(*x)) which.push_back(*x);
    }
    return which;
}
// The result, which says that it has no gradient where one of those is reached
// through it.
Tensor without_gradient(const char* none, const Tensor& out,
                        const torch::autograd::variable_list& differentiated) {
    if (differentiated.empty()) return out;
    torch::autograd::variable_list all{out};
    all.insert(all.end(), differentiated.begin(), differentiated.end());
    torch::autograd::DelayedError error(none, static_cast<int64_t>(all.size()));
    at::AutoGradMode grad(true);
    return error(std::move(all))[0];
}

// A kernel wrote to the tensor: who saved it for a backward pass is to know.
void wrote(const Tensor& x) {
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

// ---- scores -------------------------------------------------------------------------------------
void check_ids(const Tensor& buckets) {
    REQUIRE(buckets.scalar_type() == at::kInt && buckets.dim() == 1 && buckets.size(0) % 2 == 1,
            "buckets must be an int32 tensor of 2 reach + 1 ids");
    REQUIRE(buckets.size(0) / 2 <= TRW_OPS_MAX_REACH, "reach must be 0 to 1024");
}
void check_num_buckets(int64_t n) {
    REQUIRE(n >= 1 && n <= TRW_OPS_MAX_BUCKETS, "1 to 256 buckets");
}

// The checked terms of a score besides the products; holds their tensors.
struct Terms {
    Tensor buckets, slopes, times, k_times;
    trw_score score{};

    Terms(const Tensor& beside, int64_t heads, int64_t dim, std::optional<double> scale,
          double softcap, const OptionalTensor& table, const OptionalTensor& buckets_,
          const OptionalTensor& slopes_, const OptionalTensor& times_,
          const OptionalTensor& k_times_, at::IntArrayRef q_shape, at::IntArrayRef k_shape) {
        REQUIRE(table.has_value() == buckets_.has_value(), "bias_table and buckets go together");
        score.scale = static_cast<float>(scale.value_or(1.0 / std::sqrt(static_cast<double>(dim))));
        score.softcap = static_cast<float>(softcap);
        if (table) {
            on_gpu("bias_table", *table, beside);
            on_gpu("buckets", *buckets_, beside);
            REQUIRE(table->dim() == 2 && table->size(0) == heads,
                    "bias_table must be [heads, num_buckets]");
            (void)dtype_of(*table, "bias_table must be float32, float16 or bfloat16");
            check_num_buckets(table->size(1));
            check_ids(*buckets_);
            buckets = buckets_->contiguous();
            score.buckets = pointer<int32_t>(buckets);
            score.num_buckets = static_cast<int32_t>(table->size(1));
            score.reach = static_cast<int32_t>(buckets.size(0) / 2);
        }
        if (slopes_) slopes = floats("slopes", *slopes_, {heads}, beside);
        score.slopes = pointer<float>(slopes);
        REQUIRE(!times_ || slopes_, "times are for slopes");
        REQUIRE(!k_times_ || times_, "k_times go with times");
        if (times_) {
            times = floats("times", *times_, q_shape, beside);
            k_times = k_times_ ? floats("k_times", *k_times_, k_shape, beside) : times;
            if (!has_shape(k_times, k_shape)) wrong_shape("k_times", k_shape);
            score.q_times = pointer<float>(times);
            score.k_times = pointer<float>(k_times);
        }
    }
};

void check_qkv(const Tensor& q, const Tensor& k, const Tensor& v, int64_t dims) {
    on_gpu("q", q);
    on_gpu("k", k, q);
    on_gpu("v", v, q);
    if (q.dim() != dims) throw py::value_error("q must have " + std::to_string(dims) + " dimensions");
    REQUIRE(k.sizes() == v.sizes(), "k and v must have the same shape");
    REQUIRE(k.dim() == dims && q.size(-1) == k.size(-1), "q and k must have the same head size");
    (void)dtype_of(q, "q must be float32, float16 or bfloat16");
    REQUIRE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
            "q, k and v must have the same type");
    const int64_t heads = q.size(-2), kv_heads = k.size(-2), dim = q.size(-1);
    REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0,
            "heads must be a positive multiple of the key heads");
    REQUIRE(dim > 0 && dim <= 128 && dim % 8 == 0,
            "the head size must be a multiple of 8 up to 128");
}

}  // namespace

#endif  // TRW_OPERATORS_TENSORS_H
