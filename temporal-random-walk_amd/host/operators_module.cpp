// operators_module.cpp -- the operators of include/trw_operators.h on PyTorch
// tensors: what temporal_random_walk/operators.py calls.
//
// A small batch of walks is a few microseconds of GPU time, so the way there is
// C++: argument checks, outputs and workspaces from PyTorch's allocator, the
// current stream of the tensors' device, and the backward passes as autograd
// functions that run without the interpreter.
#include "operators_tensors.h"

// serving_module.cpp
void define_serving(py::module& m);

namespace {

// ---- masks -------------------------------------------------------------------------------------
struct Mask : torch::CustomClassHolder {
    Tensor info;  // rows' and documents' intervals, one after another
    int32_t *q_info, *k_info, *docs_info;
    int64_t docs, q_rows, k_rows;
    std::vector<int64_t> q_shape, k_shape;  // leading dimensions of q; of k and v
    int64_t longest;  // of any document, where the host knows it
    bool own_causal;
};
using MaskPtr = c10::intrusive_ptr<Mask>;

int kind_of(const std::string& kind, const OptionalTensor& prefix) {
    const int k = kind == "full" ? TRW_MASK_FULL
                  : kind == "causal" ? TRW_MASK_CAUSAL
                  : kind == "prefix" ? TRW_MASK_PREFIX
                                     : -1;
    REQUIRE(k >= 0, "kind must be one of full, causal, prefix");
    REQUIRE(prefix.has_value() == (k == TRW_MASK_PREFIX), "prefix is for the prefix mask");
    return k;
}

MaskPtr make_mask(trw_walk_mask_params p, const OptionalTensor& prefix, const Tensor& beside) {
    auto m = c10::make_intrusive<Mask>();
    Tensor lens;
    if (prefix) {
        lens = ints("prefix", *prefix, {p.docs}, beside);
        p.prefix = pointer<int64_t>(lens);
    }
    m->info = at::empty({4 * (p.q_rows + p.k_rows) + 8 * p.docs},
                        beside.options().dtype(at::kInt));
    m->q_info = static_cast<int32_t*>(m->info.data_ptr());
    m->k_info = m->q_info + 4 * p.q_rows;
    m->docs_info = m->k_info + 4 * p.k_rows;
    m->docs = p.docs;
    m->q_rows = p.q_rows;
    m->k_rows = p.k_rows;
    const bool packed = p.q_offsets != nullptr;
    m->longest = packed ? 0 : std::max(p.q_length, p.k_length);
    m->own_causal = p.kind == TRW_MASK_CAUSAL && !p.k_lens && !p.k_offsets;
    p.q_rows_info = m->q_info;
    p.k_rows_info = m->k_info;
    p.docs_info = m->docs_info;
    OnDevice on(beside);
    check_status(trw_ops_walk_mask(&p, on.stream));
    return m;
}

MaskPtr padded_mask(const Tensor& lens_, int64_t length, const OptionalTensor& k_lens_,
                    std::optional<int64_t> k_length, const std::string& kind,
                    const OptionalTensor& prefix) {
    on_gpu("lens", lens_);
    REQUIRE(lens_.dim() == 1, "lens must have one dimension");
    REQUIRE(lens_.size(0) < kMaxRows, "docs must be 0 to 2^30 - 1");
    REQUIRE(length >= 0 && k_length.value_or(0) >= 0, "lengths must not be negative");
    REQUIRE(length < kMaxRows && k_length.value_or(0) < kMaxRows, "rows must be 0 to 2^30 - 1");
    REQUIRE(k_lens_.has_value() == k_length.has_value(), "k_lens and k_length go together");
    trw_walk_mask_params p{};
    p.kind = kind_of(kind, prefix);
    p.docs = lens_.size(0);
    p.q_length = length;
    p.k_length = k_length.value_or(length);
    p.q_rows = p.docs * length;
    p.k_rows = p.docs * p.k_length;
    const Tensor lens = ints("lens", lens_, {p.docs}, lens_);
    Tensor k_lens;
    if (k_lens_) k_lens = ints("k_lens", *k_lens_, {p.docs}, lens_);
    p.q_lens = pointer<int64_t>(lens);
    p.k_lens = pointer<int64_t>(k_lens);
    MaskPtr m = make_mask(p, prefix, lens_);
    m->q_shape = {p.docs, length};
    m->k_shape = {p.docs, p.k_length};
    return m;
}

MaskPtr packed_mask(const Tensor& offsets_, int64_t rows, const OptionalTensor& k_offsets_,
                    std::optional<int64_t> k_rows, const std::string& kind,
                    const OptionalTensor& prefix) {
    on_gpu("offsets", offsets_);
    REQUIRE(offsets_.dim() == 1 && offsets_.size(0) >= 1,
            "offsets must have one dimension and an entry more than documents");
    REQUIRE(k_offsets_.has_value() == k_rows.has_value(), "k_offsets and k_rows go together");
    REQUIRE(rows >= 0 && k_rows.value_or(0) >= 0, "rows must not be negative");
    REQUIRE(rows < kMaxRows && k_rows.value_or(0) < kMaxRows, "rows must be 0 to 2^30 - 1");
    trw_walk_mask_params p{};
    p.kind = kind_of(kind, prefix);
    p.docs = offsets_.size(0) - 1;
    p.q_rows = rows;
    p.k_rows = k_rows.value_or(rows);
    const Tensor offsets = ints("offsets", offsets_, {p.docs + 1}, offsets_);
    Tensor k_offsets;
    if (k_offsets_) k_offsets = ints("k_offsets", *k_offsets_, {p.docs + 1}, offsets_);
    p.q_offsets = pointer<int64_t>(offsets);
    p.k_offsets = pointer<int64_t>(k_offsets);
    MaskPtr m = make_mask(p, prefix, offsets_);
    m->q_shape = {rows};
    m->k_shape = {p.k_rows};
    return m;
}

// ---- attention ------------------------------------------------------------------------------------
// What one call's passes share.  The tensors are saved variables: changes between
// the passes are noticed, and with hooks on them (checkpointing, offloading) the
// backward pass gets others than the forward pass had, which may be gone.
struct Call : torch::CustomClassHolder {
    MaskPtr mask;
    std::optional<Terms> terms;  // until they are saved
    trw_attention_params params{};
    std::vector<int64_t> q_shape, k_shape;
    bool tabled = false, with_low = false, sloped = false, timed = false;
};
using CallPtr = c10::intrusive_ptr<Call>;

Tensor workspace(trw_attention_params& p, int backward, const Tensor& beside) {
    uint64_t n = 0;
    check_status(trw_ops_attention_workspace(&p, backward, &n));
    Tensor space;
    if (n) {
        space = bytes(n, beside);
        p.workspace = space.data_ptr();
    }
    p.workspace_bytes = n;
    return space;
}

// Autograd saves no tensors of the inference mode.
Tensor saveable(const Tensor& x) { return x.defined() && x.is_inference() ? x.clone() : x; }

// What was saved as a tensor of this shape, type and device, as a hook gave it
// back.
const Tensor& unpacked(const Tensor& x, at::IntArrayRef shape, at::ScalarType type,
                       const Tensor& beside) {
    if (!x.defined() || !has_shape(x, shape) || x.scalar_type() != type ||
        x.device() != beside.device())
        throw std::runtime_error(
            "a saved tensor came back from its hook with another shape, type or device");
    return x;
}

// A backward pass's results, which say so where they are differentiated again.
torch::autograd::variable_list once(torch::autograd::variable_list grads, bool again) {
    if (!again) return grads;
    torch::autograd::variable_list given;
    for (const Tensor& g : grads)
        if (g.defined()) given.push_back(g);
    torch::autograd::DelayedError error(
        "trying to differentiate twice a function that can be differentiated once",
        static_cast<int64_t>(given.size()));
    at::AutoGradMode grad(true);
    for (Tensor& g : given) g.requires_grad_();
    auto marked = error(std::move(given));
    size_t n = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = marked[n++];
    return grads;
}

struct WalkAttention : torch::autograd::Function<WalkAttention> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q_, const Tensor& k_,
                          const Tensor& v_, const OptionalTensor& table, const CallPtr& call,
                          bool train) {
        call->q_shape = q_.sizes().vec();
        call->k_shape = k_.sizes().vec();
        const Tensor q = as_rows(q_), k = as_rows(k_), v = as_rows(v_);
        const Mask& mask = *call->mask;
        const Tensor result = at::empty(call->q_shape, q.options());
        const Tensor out = result.view(q.sizes());
        trw_attention_params& p = call->params;
        p.dtype = dtype_of(q, "");
        p.heads = static_cast<int32_t>(q.size(1));
        p.kv_heads = static_cast<int32_t>(k.size(1));
        p.dim = static_cast<int32_t>(q.size(2));
        p.q_rows = mask.q_rows;
        p.k_rows = mask.k_rows;
        p.q_rows_info = mask.q_info;
        p.k_rows_info = mask.k_info;
        p.docs_info = mask.docs_info;
        p.docs = mask.docs;
        p.longest = mask.longest;
        p.covered = mask.longest > 0;  // padded
        p.own_causal = mask.own_causal;
        p.score = call->terms->score;
        p.score.table = pointer<float>(table);
        p.q = rows_of(q);
        p.k = rows_of(k);
        p.v = rows_of(v);
        p.out = rows_of(out);
        Tensor stats, low;
        if (train) {
            stats = at::empty({2, q.size(1), mask.q_rows}, q.options().dtype(at::kFloat));
            p.stats = pointer<float>(stats);
            // Walks that go a wave each sum there what the backward pass needs of the output
            // (those of up to 8 rows may go through tiles, under a wide cap all do)
            const int64_t wave = p.dim <= 64 ? 96 : 64;
            if (p.dtype != TRW_F32 && !(mask.longest > 8 && mask.longest <= wave &&
                                        p.score.softcap <= TRW_OPS_WIDE_CAP)) {
                low = at::empty_like(out);
                p.out_low = rows_of(low);
            }
        }
        {
            OnDevice on(q);
            const Tensor space = workspace(p, 0, q);  // held until the call has queued
            check_status(trw_ops_attention_forward(&p, on.stream));
        }
        if (train) {
            call->tabled = table.has_value();
            call->with_low = low.defined();
            // the output itself and no view of it, which would keep it, and so this node, alive
            const Terms& terms = *call->terms;
            ctx->save_for_backward({q, k, v, table.value_or(Tensor()), result, stats, low,
                                    saveable(terms.buckets), saveable(terms.slopes),
                                    saveable(terms.times), saveable(terms.k_times)});
            call->sloped = terms.slopes.defined();
            call->timed = terms.times.defined();
            call->terms.reset();
            ctx->saved_data["call"] = c10::IValue::make_capsule(call);
        }
        return result;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto call = c10::static_intrusive_pointer_cast<Call>(
            ctx->saved_data["call"].toCapsule());
        const bool again = differentiable(grads[0]);
        at::AutoGradMode no_grad(false);
        trw_attention_params p = call->params;
        const at::ScalarType type = grads[0].scalar_type();
        const auto back = [&](int n, at::IntArrayRef shape, at::ScalarType of) {
            return unpacked(saved[n], shape, of, grads[0]);
        };
        const Tensor q = readable(back(0, {p.q_rows, p.heads, p.dim}, type));
        const Tensor k = readable(back(1, {p.k_rows, p.kv_heads, p.dim}, type));
        const Tensor v = readable(back(2, {p.k_rows, p.kv_heads, p.dim}, type));
        const Tensor out = as_rows(back(4, call->q_shape, type));
        const Tensor stats = back(5, {2, p.heads, p.q_rows}, at::kFloat).contiguous();
        p.q = rows_of(q);
        p.k = rows_of(k);
        p.v = rows_of(v);
        p.out = rows_of(out);
        p.stats = pointer<float>(stats);
        Tensor table, low, buckets, slopes, times, k_times;
        if (call->tabled) {
            table = back(3, {p.heads, p.score.num_buckets}, at::kFloat).contiguous();
            buckets = back(7, {2 * p.score.reach + 1}, at::kInt).contiguous();
            p.score.table = pointer<float>(table);
            p.score.buckets = pointer<int32_t>(buckets);
        }
        if (call->sloped) {
            slopes = back(8, {p.heads}, at::kFloat).contiguous();
            p.score.slopes = pointer<float>(slopes);
        }
        if (call->timed) {
            times = back(9, call->mask->q_shape, at::kFloat).contiguous();
            k_times = back(10, call->mask->k_shape, at::kFloat).contiguous();
            p.score.q_times = pointer<float>(times);
            p.score.k_times = pointer<float>(k_times);
        }
        if (call->with_low) {
            low = readable(back(6, {p.q_rows, p.heads, p.dim}, type));
            p.out_low = rows_of(low);
        }
        const Tensor d_out = as_rows(grads[0]);
        Tensor d_q = at::empty(q.sizes(), q.options()), d_k = at::empty(k.sizes(), k.options()),
               d_v = at::empty(v.sizes(), v.options()), d_table;
        p.d_out = rows_of(d_out);
        p.d_q = rows_of(d_q);
        p.d_k = rows_of(d_k);
        p.d_v = rows_of(d_v);
        if (table.defined()) {
            d_table = at::empty(table.sizes(), table.options());
            p.d_table = pointer<float>(d_table);
        }
        {
            OnDevice on(q);
            p.workspace = nullptr;
            const Tensor space = workspace(p, 1, q);
            check_status(trw_ops_attention_backward(&p, on.stream));
        }
        return once({d_q.view(call->q_shape), d_k.view(call->k_shape), d_v.view(call->k_shape),
                     d_table, Tensor(), Tensor()},
                    again);
    }
};

bool wants_grad(const Tensor& x) { return x.requires_grad(); }

Tensor walk_attention(const Tensor& q, const Tensor& k, const Tensor& v, const MaskPtr& mask,
                      std::optional<double> scale, double softcap, const OptionalTensor& bias_table,
                      const OptionalTensor& buckets, const OptionalTensor& slopes,
                      const OptionalTensor& times, const OptionalTensor& k_times) {
    const int64_t lead = static_cast<int64_t>(mask->q_shape.size());
    check_qkv(q, k, v, lead + 2);
    REQUIRE(q.device() == mask->info.device(), "q is on another device than the mask");
    if (q.sizes().slice(0, lead) != at::IntArrayRef(mask->q_shape) ||
        k.sizes().slice(0, lead) != at::IntArrayRef(mask->k_shape))
        throw py::value_error("q and k must be the mask's rows of heads");
    auto call = c10::make_intrusive<Call>();
    call->mask = mask;
    call->terms.emplace(q, q.size(-2), q.size(-1), scale, softcap, bias_table, buckets, slopes,
                        times, k_times, mask->q_shape, mask->k_shape);
    OptionalTensor table;
    if (bias_table) table = bias_table->to(at::kFloat).contiguous();
    const bool train = at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) ||
                                                      wants_grad(v) || (table && wants_grad(*table)));
    return WalkAttention::apply(q, k, v, table, call, train);
}

constexpr char kNoGradient[] = "walk_attention_step has no gradient";

Tensor walk_attention_step(const Tensor& q_, const Tensor& k_, const Tensor& v_,
                           const Tensor& k_cache, const Tensor& v_cache, const Tensor& lens_,
                           std::optional<double> scale, double softcap,
                           const OptionalTensor& bias_table, const OptionalTensor& buckets,
                           const OptionalTensor& slopes, const OptionalTensor& times,
                           const OptionalTensor& k_times) {
    const auto differentiated = differentiated_of(
        kNoGradient, {q_, k_, v_, k_cache, v_cache, bias_table, slopes, times, k_times});
    at::AutoGradMode no_grad(false);
    check_qkv(q_, k_, v_, 3);
    const int64_t batch = q_.size(0), heads = q_.size(1), kv_heads = k_.size(1), dim = q_.size(2);
    REQUIRE(k_.size(0) == batch, "q and k must have the same batch");
    for (const Tensor* x : {&k_cache, &v_cache}) {
        on_gpu("a cache", *x, q_);
        REQUIRE(x->scalar_type() == q_.scalar_type() && x->dim() == 4 && x->size(0) == batch &&
                    x->size(2) == kv_heads && x->size(3) == dim,
                "a cache must be [batch, capacity, kv_heads, dim] of q's type");
        REQUIRE(x->numel() == 0 || in_pieces(*x), "a cache's rows must be 16-byte pieces");
    }
    REQUIRE(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache must have the same shape");
    const int64_t capacity = k_cache.size(1);
    const Tensor lens = ints("lens", lens_, {batch}, q_);
    REQUIRE(times.has_value() == k_times.has_value(), "times and k_times go together");
    REQUIRE(!k_times || k_times->is_contiguous(), "k_times must be contiguous");
    const Terms terms(q_, heads, dim, scale, softcap, bias_table, buckets, slopes, times, k_times,
                      {batch}, {batch, capacity});
    Tensor table;
    if (bias_table) table = bias_table->to(at::kFloat).contiguous();
    const Tensor q = readable(q_), k = readable(k_), v = readable(v_);
    Tensor out = at::empty(q.sizes(), q.options());
    trw_attention_step_params p{};
    p.dtype = dtype_of(q, "");
    p.heads = static_cast<int32_t>(heads);
    p.kv_heads = static_cast<int32_t>(kv_heads);
    p.dim = static_cast<int32_t>(dim);
    p.batch = batch;
    p.capacity = capacity;
    p.lens = pointer<int64_t>(lens);
    p.score = terms.score;
    p.score.table = pointer<float>(table);
    p.q = rows_of(q);
    p.k = rows_of(k);
    p.v = rows_of(v);
    p.out = rows_of(out);
    p.k_cache = k_cache.data_ptr();
    p.v_cache = v_cache.data_ptr();
    p.k_batch_stride = k_cache.stride(0);
    p.k_pos_stride = k_cache.stride(1);
    p.k_head_stride = k_cache.stride(2);
    p.v_batch_stride = v_cache.stride(0);
    p.v_pos_stride = v_cache.stride(1);
    p.v_head_stride = v_cache.stride(2);
    OnDevice on(q);
    check_status(trw_ops_attention_step_workspace(&p, &p.workspace_bytes));
    Tensor space;
    if (p.workspace_bytes) {
        space = bytes(p.workspace_bytes, q);
        p.workspace = space.data_ptr();
    }
    check_status(trw_ops_attention_step(&p, on.stream));
    wrote(k_cache);
    wrote(v_cache);
    if (k_times) wrote(*k_times);
    return without_gradient(kNoGradient, out, differentiated);
}

// ---- the dense bias ---------------------------------------------------------------------------------
struct RelativeBias : torch::autograd::Function<RelativeBias> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& table_,
                          const Tensor& buckets, int64_t q_len, int64_t k_len, int64_t q_offset) {
        const Tensor table = table_.contiguous();
        Tensor out = at::empty({table.size(0), q_len, k_len}, table.options());
        trw_relative_bias_params p = params(table, buckets, q_len, k_len, q_offset);
        p.out = out.data_ptr();
        OnDevice on(table);
        check_status(trw_ops_relative_bias(&p, on.stream));
        ctx->save_for_backward({table, saveable(buckets)});
        ctx->saved_data["q_offset"] = q_offset;
        ctx->saved_data["num_buckets"] = table.size(1);
        ctx->saved_data["ids"] = buckets.size(0);
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const bool again = differentiable(grads[0]);
        at::AutoGradMode no_grad(false);
        Tensor d_out = grads[0];
        const Tensor table =
            unpacked(saved[0], {d_out.size(0), ctx->saved_data["num_buckets"].toInt()},
                     d_out.scalar_type(), d_out).contiguous();
        const Tensor buckets =
            unpacked(saved[1], {ctx->saved_data["ids"].toInt()}, at::kInt, d_out).contiguous();
        if (d_out.stride(-1) != 1) d_out = d_out.contiguous();
        Tensor d_table = at::empty(table.sizes(), table.options());
        trw_relative_bias_params p = params(table, buckets, d_out.size(1), d_out.size(2),
                                            ctx->saved_data["q_offset"].toInt());
        p.d_out = d_out.data_ptr();
        p.d_out_head_stride = d_out.stride(0);
        p.d_out_row_stride = d_out.stride(1);
        p.d_table = d_table.data_ptr();
        OnDevice on(table);
        check_status(trw_ops_relative_bias_workspace(&p, &p.workspace_bytes));
        const Tensor space = bytes(std::max<uint64_t>(p.workspace_bytes, 16), table);
        p.workspace = space.data_ptr();
        check_status(trw_ops_relative_bias_backward(&p, on.stream));
        return once({d_table, Tensor(), Tensor(), Tensor(), Tensor()}, again);
    }
    static trw_relative_bias_params params(const Tensor& table, const Tensor& buckets,
                                           int64_t q_len, int64_t k_len, int64_t q_offset) {
        trw_relative_bias_params p{};
        p.dtype = dtype_of(table, "");
        p.heads = static_cast<int32_t>(table.size(0));
        p.num_buckets = static_cast<int32_t>(table.size(1));
        p.reach = static_cast<int32_t>(buckets.size(0) / 2);
        p.q_len = q_len;
        p.k_len = k_len;
        p.q_offset = q_offset;
        p.table = table.data_ptr();
        p.buckets = pointer<int32_t>(buckets);
        return p;
    }
};

Tensor relative_bias(const Tensor& table, const Tensor& buckets, int64_t q_len, int64_t k_len,
                     int64_t q_offset) {
    on_gpu("table", table);
    on_gpu("buckets", buckets, table);
    REQUIRE(table.dim() == 2 && table.size(0) > 0, "table must be [heads, num_buckets]");
    (void)dtype_of(table, "table must be float32, float16 or bfloat16");
    check_num_buckets(table.size(1));
    check_ids(buckets);
    REQUIRE(q_len >= 0 && k_len >= 0, "lengths must not be negative");
    return RelativeBias::apply(table, buckets.contiguous(), q_len, k_len, q_offset);
}

}  // namespace

PYBIND11_MODULE(_operators, m) {
    if (trw_ops_abi_version() != TRW_OPS_ABI_VERSION)
        throw py::import_error("libtrw_operators.so has another ABI than _operators: build again");
    py::class_<Mask, MaskPtr>(m, "Mask")
        .def_readonly("info", &Mask::info)
        .def_readonly("q_rows", &Mask::q_rows)
        .def_readonly("k_rows", &Mask::k_rows)
        .def_readonly("q_shape", &Mask::q_shape)
        .def_readonly("k_shape", &Mask::k_shape);
    m.def("padded_mask", torch::wrap_pybind_function_no_gil(&padded_mask));
    m.def("packed_mask", torch::wrap_pybind_function_no_gil(&packed_mask));
    m.def("walk_attention", torch::wrap_pybind_function_no_gil(&walk_attention));
    m.def("walk_attention_step", torch::wrap_pybind_function_no_gil(&walk_attention_step));
    m.def("relative_bias", torch::wrap_pybind_function_no_gil(&relative_bias));
    define_serving(m);
}
