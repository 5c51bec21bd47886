// serving_module.cpp -- pages and beam search on PyTorch tensors: the second
// part of what temporal_random_walk/operators.py calls.
#include <tuple>
#include <vector>

#include "operators_tensors.h"

namespace {

// ---- pages -----------------------------------------------------------------------------------------
// k, v and, of 8 bits, their scales
using PageTensors = std::tuple<Tensor, Tensor, OptionalTensor, OptionalTensor>;

// Elements from page to page.
int64_t page_stride(const Tensor& x) {
    return x.size(0) > 1 ? x.stride(0) : x.numel();
}
// Whether a page's own elements lie one after another.
bool pages_whole(const Tensor& x) { return x.size(0) == 0 || x.select(0, 0).is_contiguous(); }

trw_pages pages_of(const PageTensors& t, const Tensor& beside) {
    const Tensor &k = std::get<0>(t), &v = std::get<1>(t);
    const OptionalTensor &k_scale = std::get<2>(t), &v_scale = std::get<3>(t);
    on_gpu("pages", k, beside);
    on_gpu("pages", v, beside);
    REQUIRE(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
            "k and v of pages must be [pages, kv_heads, page_rows, dim] of one type");
    REQUIRE(pages_whole(k) && pages_whole(v), "a page must be contiguous");
    const bool eight = k.scalar_type() == at::kFloat8_e4m3fn;
    REQUIRE(k_scale.has_value() == eight && v_scale.has_value() == eight,
            "pages of float8_e4m3fn, and no others, have scales");
    trw_pages p{};
    p.dtype = eight ? TRW_E4M3
                    : dtype_of(k, "pages must be float8_e4m3fn, float32, float16 or bfloat16");
    p.pages = k.size(0);
    REQUIRE(k.size(1) <= 4096 && k.size(2) <= 1024 && k.size(3) <= 128,
            "pages have up to 4096 heads, 1024 rows and 128 elements");
    p.kv_heads = static_cast<int32_t>(k.size(1));
    p.page_rows = static_cast<int32_t>(k.size(2));
    p.dim = static_cast<int32_t>(k.size(3));
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.k_stride = page_stride(k);
    p.v_stride = page_stride(v);
    if (eight) {
        for (const Tensor* s : {&*k_scale, &*v_scale}) {
            on_gpu("scales", *s, beside);
            REQUIRE(s->scalar_type() == at::kByte && has_shape(*s, k.sizes().slice(0, 3)),
                    "scales must be uint8 [pages, kv_heads, page_rows]");
            REQUIRE(pages_whole(*s), "a page's scales must be contiguous");
        }
        p.k_scale = pointer<uint8_t>(k_scale);
        p.v_scale = pointer<uint8_t>(v_scale);
        p.k_scale_stride = page_stride(*k_scale);
        p.v_scale_stride = page_stride(*v_scale);
    }
    return p;
}

// The table's rows one after another (a view or a copy of what was given).
Tensor set_table(trw_pages& p, const Tensor& table_, const Tensor& beside) {
    on_gpu("table", table_, beside);
    REQUIRE(table_.scalar_type() == at::kInt && table_.dim() == 2,
            "table must be int32 [walks, pages of a walk]");
    const Tensor table =
        table_.size(1) <= 1 || table_.stride(1) == 1 ? table_ : table_.contiguous();
    p.table = pointer<int32_t>(table);
    p.walks = table.size(0);
    p.table_pages = table.size(1);
    p.table_stride = table.stride(0);
    return table;
}

void wrote_pages(const PageTensors& t) {
    wrote(std::get<0>(t));
    wrote(std::get<1>(t));
    if (std::get<2>(t)) wrote(*std::get<2>(t));
    if (std::get<3>(t)) wrote(*std::get<3>(t));
}

// Times of the pages' positions, in place.
Tensor page_times(const Tensor& x, const trw_pages& p, const Tensor& beside) {
    const Tensor times = floats("k_times", x, {p.pages, p.page_rows}, beside);
    REQUIRE(x.is_contiguous(), "k_times must be contiguous");
    return times;
}

void paged_write(const PageTensors& tensors, const Tensor& table_, const OptionalTensor& starts_,
                 const Tensor& k_, const Tensor& v_, const OptionalTensor& counts_,
                 const OptionalTensor& offsets_, const OptionalTensor& times_,
                 const OptionalTensor& k_times_) {
    constexpr char kNone[] =
        "paged_write has no gradient: call it under torch.no_grad(), or with detached rows";
    REQUIRE(differentiated_of(kNone, {k_, v_, times_, std::get<0>(tensors), std::get<1>(tensors)})
                .empty(),
            kNone);
    at::AutoGradMode no_grad(false);
    on_gpu("k", k_);
    on_gpu("v", v_, k_);
    REQUIRE(k_.sizes() == v_.sizes() && k_.scalar_type() == v_.scalar_type(),
            "k and v must have the same shape and type");
    trw_paged_copy_params p{};
    p.pages = pages_of(tensors, k_);
    p.dtype = dtype_of(k_, "k must be float32, float16 or bfloat16");
    const Tensor table = set_table(p.pages, table_, k_);
    const int64_t walks = p.pages.walks;
    REQUIRE(!offsets_ || !counts_, "counts are for padded walks, offsets for packed ones");
    const bool packed = offsets_.has_value();
    REQUIRE(k_.dim() == (packed ? 3 : 4) && k_.size(-2) == p.pages.kv_heads &&
                k_.size(-1) == p.pages.dim && (packed || k_.size(0) == walks),
            "k must be [walks, length, kv_heads, dim], or [rows, kv_heads, dim] with offsets");
    Tensor starts, counts, offsets, times, k_times;
    if (starts_) starts = ints("starts", *starts_, {walks}, k_);
    if (counts_) counts = ints("counts", *counts_, {walks}, k_);
    if (offsets_) offsets = ints("offsets", *offsets_, {walks + 1}, k_);
    REQUIRE(times_.has_value() == k_times_.has_value(), "times and k_times go together");
    if (times_) {
        times = floats("times", *times_, k_.sizes().slice(0, packed ? 1 : 2), k_);
        k_times = page_times(*k_times_, p.pages, k_);
    }
    const Tensor k = as_rows(k_), v = as_rows(v_);
    p.rows = k.size(0);
    p.length = packed ? 0 : k_.size(1);
    p.counts = pointer<int64_t>(counts);
    p.offsets = pointer<int64_t>(offsets);
    p.starts = pointer<int64_t>(starts);
    p.k = rows_of(k);
    p.v = rows_of(v);
    p.times = pointer<float>(times);
    p.k_times = pointer<float>(k_times);
    OnDevice on(k);
    check_status(trw_ops_paged_write(&p, on.stream));
    wrote_pages(tensors);
    if (k_times_) wrote(*k_times_);
}

std::tuple<Tensor, Tensor, OptionalTensor> paged_read(
    const PageTensors& tensors, const Tensor& table_, const OptionalTensor& lens_,
    std::optional<int64_t> length, const OptionalTensor& offsets_, std::optional<int64_t> rows,
    std::optional<at::ScalarType> dtype, const OptionalTensor& k_times_) {
    constexpr char kNone[] = "paged_read has no gradient";
    const auto differentiated =
        differentiated_of(kNone, {std::get<0>(tensors), std::get<1>(tensors)});
    at::AutoGradMode no_grad(false);
    const Tensor& beside = std::get<0>(tensors);
    trw_paged_copy_params p{};
    p.pages = pages_of(tensors, beside);
    const bool eight = p.pages.dtype == TRW_E4M3;
    const at::ScalarType type = dtype.value_or(eight ? at::kBFloat16 : beside.scalar_type());
    REQUIRE(type == at::kFloat || type == at::kHalf || type == at::kBFloat16,
            "dtype must be float32, float16 or bfloat16");
    const Tensor table = set_table(p.pages, table_, beside);
    const int64_t walks = p.pages.walks;
    REQUIRE(lens_.has_value() == length.has_value() && offsets_.has_value() == rows.has_value() &&
                lens_.has_value() != offsets_.has_value(),
            "either lens and length are given or offsets and rows");
    REQUIRE(length.value_or(0) >= 0 && length.value_or(0) < kMaxRows && rows.value_or(0) >= 0 &&
                walks < kMaxRows && walks * length.value_or(0) < kMaxRows &&
                rows.value_or(0) < kMaxRows,
            "rows must be 0 to 2^30 - 1");
    Tensor lens, offsets, k_times, times;
    std::vector<int64_t> shape;
    if (lens_) {
        lens = ints("lens", *lens_, {walks}, beside);
        p.length = *length;
        p.rows = walks * *length;
        shape = {walks, *length};
    } else {
        offsets = ints("offsets", *offsets_, {walks + 1}, beside);
        p.rows = *rows;
        shape = {*rows};
    }
    const auto options = beside.options().dtype(type);
    if (k_times_) {
        k_times = page_times(*k_times_, p.pages, beside);
        times = at::empty(shape, beside.options().dtype(at::kFloat));
    }
    shape.push_back(p.pages.kv_heads);
    shape.push_back(p.pages.dim);
    const Tensor k = at::empty(shape, options), v = at::empty(shape, options);
    p.dtype = dtype_of(k, "");
    const int64_t head = p.pages.dim, row = head * p.pages.kv_heads;
    p.counts = pointer<int64_t>(lens);
    p.offsets = pointer<int64_t>(offsets);
    p.k = trw_rows{k.data_ptr(), row, head};
    p.v = trw_rows{v.data_ptr(), row, head};
    p.times = pointer<float>(times);
    p.k_times = pointer<float>(k_times);
    OnDevice on(beside);
    check_status(trw_ops_paged_read(&p, on.stream));
    OptionalTensor read_times;
    if (k_times_) read_times = times;
    return {without_gradient(kNone, k, differentiated), without_gradient(kNone, v, differentiated),
            read_times};
}

Tensor paged_attention_step(const Tensor& q_, const Tensor& k_, const Tensor& v_,
                            const PageTensors& tensors, const Tensor& table_, const Tensor& lens_,
                            const OptionalTensor& first_, std::optional<double> scale,
                            double softcap, const OptionalTensor& bias_table,
                            const OptionalTensor& buckets, const OptionalTensor& slopes,
                            const OptionalTensor& times, const OptionalTensor& k_times) {
    constexpr char kNone[] = "paged_attention_step has no gradient";
    const auto differentiated =
        differentiated_of(kNone, {q_, k_, v_, std::get<0>(tensors), std::get<1>(tensors),
                                  bias_table, slopes, times, k_times});
    at::AutoGradMode no_grad(false);
    check_qkv(q_, k_, v_, 3);
    const int64_t batch = q_.size(0), heads = q_.size(1), dim = q_.size(2);
    REQUIRE(k_.size(0) == batch, "q and k must have the same batch");
    trw_paged_step_params p{};
    p.pages = pages_of(tensors, q_);
    REQUIRE(k_.size(1) == p.pages.kv_heads && dim == p.pages.dim,
            "k and v must be rows of the pages' heads");
    const Tensor table = set_table(p.pages, table_, q_);
    REQUIRE(p.pages.walks == batch, "table must have a row for each of the batch");
    const Tensor lens = ints("lens", lens_, {batch}, q_);
    Tensor first;
    if (first_) first = ints("first", *first_, {batch}, q_);
    REQUIRE(times.has_value() == k_times.has_value(), "times and k_times go together");
    REQUIRE(!k_times || k_times->is_contiguous(), "k_times must be contiguous");
    const Terms terms(q_, heads, dim, scale, softcap, bias_table, buckets, slopes, times, k_times,
                      {batch}, {p.pages.pages, p.pages.page_rows});
    Tensor bias;
    if (bias_table) bias = bias_table->to(at::kFloat).contiguous();
    const Tensor q = readable(q_), k = readable(k_), v = readable(v_);
    Tensor out = at::empty({batch, heads, dim}, q.options());
    p.dtype = dtype_of(q, "");
    p.heads = static_cast<int32_t>(heads);
    p.lens = pointer<int64_t>(lens);
    p.first = pointer<int64_t>(first);
    p.score = terms.score;
    p.score.table = pointer<float>(bias);
    p.q = rows_of(q);
    p.k = rows_of(k);
    p.v = rows_of(v);
    p.out = rows_of(out);
    OnDevice on(q);
    check_status(trw_ops_paged_step_workspace(&p, &p.workspace_bytes));
    Tensor space;
    if (p.workspace_bytes) {
        space = bytes(p.workspace_bytes, q);
        p.workspace = space.data_ptr();
    }
    check_status(trw_ops_paged_step(&p, on.stream));
    wrote_pages(tensors);
    if (k_times) wrote(*k_times);
    return without_gradient(kNone, out, differentiated);
}

// ---- beams -----------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor, Tensor> beam_select(const Tensor& logits_, const Tensor& scores_,
                                                       int64_t width,
                                                       const OptionalTensor& ended_,
                                                       std::optional<int64_t> end_token) {
    constexpr char kNone[] = "beam_select has no gradient";
    const auto differentiated = differentiated_of(kNone, {logits_, scores_});
    at::AutoGradMode no_grad(false);
    on_gpu("logits", logits_);
    REQUIRE(logits_.dim() == 3, "logits must be [groups, beams, nodes]");
    trw_beam_select_params p{};
    p.dtype = dtype_of(logits_, "logits must be float32, float16 or bfloat16");
    const int64_t groups = logits_.size(0), beams = logits_.size(1);
    REQUIRE(beams >= 1 && beams <= TRW_OPS_BEAMS && width >= 1 && width <= TRW_OPS_BEAMS,
            "beams and width must be 1 to 32");
    on_gpu("scores", scores_, logits_);
    REQUIRE(scores_.scalar_type() == at::kFloat, "scores must be float32");
    if (!has_shape(scores_, {groups, beams})) wrong_shape("scores", {groups, beams});
    const Tensor scores = scores_.contiguous();
    Tensor ended;
    if (ended_) {
        on_gpu("ended", *ended_, logits_);
        REQUIRE(ended_->scalar_type() == at::kBool, "ended must hold truth values");
        if (!has_shape(*ended_, {groups, beams})) wrong_shape("ended", {groups, beams});
        ended = ended_->contiguous();
    }
    REQUIRE(!ended_ || end_token, "ended beams need an end_token");
    REQUIRE(!end_token || *end_token >= 0, "end_token must be a node");
    const Tensor logits = logits_.size(2) <= 1 || logits_.stride(2) == 1 ? logits_
                                                                         : logits_.contiguous();
    p.beams = static_cast<int32_t>(beams);
    p.width = static_cast<int32_t>(width);
    p.groups = groups;
    p.nodes = logits.size(2);
    p.logits = logits.data_ptr();
    p.group_stride = logits.stride(0);
    p.beam_stride = logits.stride(1);
    p.scores = pointer<float>(scores);
    p.ended = pointer<uint8_t>(ended);
    p.end_token = end_token.value_or(-1);
    const auto longs = logits.options().dtype(at::kLong);
    Tensor out_scores = at::empty({groups, width}, scores.options());
    Tensor tokens = at::empty({groups, width}, longs), parents = at::empty({groups, width}, longs);
    Tensor out_ended = at::empty({groups, width}, logits.options().dtype(at::kBool));
    p.out_scores = pointer<float>(out_scores);
    p.out_tokens = pointer<int64_t>(tokens);
    p.out_parents = pointer<int64_t>(parents);
    p.out_ended = pointer<uint8_t>(out_ended);
    OnDevice on(logits);
    check_status(trw_ops_beam_select_workspace(&p, &p.workspace_bytes));
    const Tensor space = bytes(std::max<uint64_t>(p.workspace_bytes, 16), logits);
    p.workspace = space.data_ptr();
    check_status(trw_ops_beam_select(&p, on.stream));
    return {without_gradient(kNone, out_scores, differentiated), tokens, parents, out_ended};
}

std::tuple<Tensor, Tensor> beam_reorder(const Tensor& table_, const Tensor& lens_,
                                        const Tensor& parents_,
                                        const std::vector<PageTensors>& caches,
                                        const OptionalTensor& k_times_) {
    constexpr char kNone[] = "beam_reorder has no gradient";
    for (const PageTensors& t : caches)
        REQUIRE(differentiated_of(kNone, {std::get<0>(t), std::get<1>(t)}).empty(), kNone);
    at::AutoGradMode no_grad(false);
    on_gpu("parents", parents_);
    REQUIRE(parents_.dim() == 2, "parents must be [groups, beams]");
    REQUIRE(!caches.empty(), "pages of at least one cache are needed");
    const int64_t groups = parents_.size(0), beams = parents_.size(1);
    REQUIRE(beams >= 1 && beams <= TRW_OPS_BEAMS, "beams must be 1 to 32");
    const Tensor parents = ints("parents", parents_, {groups, beams}, parents_);
    const Tensor lens = ints("lens", lens_, {groups * beams}, parents_);
    std::vector<trw_pages> pages;
    for (const PageTensors& t : caches) pages.push_back(pages_of(t, parents_));
    const Tensor table = set_table(pages[0], table_, parents_);
    REQUIRE(pages[0].walks == groups * beams, "table must have a row for each beam");
    Tensor k_times;
    if (k_times_) k_times = page_times(*k_times_, pages[0], parents_);
    Tensor out_table = at::empty(table.sizes(), table.options());
    Tensor out_lens = at::empty(lens.sizes(), lens.options());
    trw_beam_reorder_params p{};
    p.beams = static_cast<int32_t>(beams);
    p.page_rows = pages[0].page_rows;
    p.count = static_cast<int32_t>(pages.size());
    p.groups = groups;
    p.pages = pages[0].pages;
    p.table_pages = pages[0].table_pages;
    p.table_stride = pages[0].table_stride;
    p.table = pages[0].table;
    p.out_table = pointer<int32_t>(out_table);
    p.lens = pointer<int64_t>(lens);
    p.out_lens = pointer<int64_t>(out_lens);
    p.parents = pointer<int64_t>(parents);
    p.caches = pages.data();
    p.k_times = pointer<float>(k_times);
    OnDevice on(parents);
    check_status(trw_ops_beam_reorder(&p, on.stream));
    for (const PageTensors& t : caches) wrote_pages(t);
    if (k_times_) wrote(*k_times_);
    return {out_table, out_lens};
}

}  // namespace

void define_serving(py::module& m) {
    m.def("paged_write", torch::wrap_pybind_function_no_gil(&paged_write));
    m.def("paged_read", torch::wrap_pybind_function_no_gil(&paged_read));
    m.def("paged_attention_step", torch::wrap_pybind_function_no_gil(&paged_attention_step));
    m.def("beam_select", torch::wrap_pybind_function_no_gil(&beam_select));
    m.def("beam_reorder", torch::wrap_pybind_function_no_gil(&beam_reorder));
}
