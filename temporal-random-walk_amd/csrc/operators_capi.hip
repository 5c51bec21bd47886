// operators_capi.hip -- the extern "C" boundary declared in
// include/trw_operators.h: checks every argument that the host can see, maps
// C++ exceptions to trw_status and keeps the message in a thread-local buffer.
#include <cmath>
#include <new>

#include "operators.h"

namespace {

using trw::ops::require;

thread_local std::string g_last_error;

trw_status failed(trw_status status, const char* message) {
    try {
        g_last_error = message;
    } catch (...) {  // out of memory for the message itself
        g_last_error.clear();
    }
    return status;
}

template <typename F>
trw_status guarded(F&& f) {
    try {
        f();
        return TRW_OK;
    } catch (const trw::ops::InvalidArgument& ex) {
        return failed(TRW_ERR_INVALID_ARGUMENT, ex.what());
    } catch (const std::bad_alloc& ex) {
        return failed(TRW_ERR_OUT_OF_MEMORY, ex.what());
    } catch (const std::exception& ex) {
        return failed(TRW_ERR_RUNTIME, ex.what());
    } catch (...) {
        return failed(TRW_ERR_RUNTIME, "unknown error");
    }
}

constexpr int64_t kMaxRows = int64_t{1} << 30;

void check_dtype(int dtype) {
    require(dtype == TRW_F32 || dtype == TRW_F16 || dtype == TRW_BF16,
            "dtype must be float32, float16 or bfloat16");
}

void check_heads(int dtype, int heads, int kv_heads, int dim) {
    check_dtype(dtype);
    require(heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
            "heads must be a positive multiple of kv_heads");
    require(heads <= 4096, "at most 4096 heads");
    require(dim > 0 && dim <= 128 && dim % 8 == 0, "head size must be a multiple of 8 up to 128");
}

void check_aligned(const void* p, const char* message) {
    require(reinterpret_cast<uintptr_t>(p) % 16 == 0, message);
}

// Rows that are read as 16-byte pieces.
void check_rows(const trw_rows& r, int dtype, int64_t rows, const char* null_message) {
    if (rows == 0) return;
    const int64_t piece = 16 / static_cast<int64_t>(trw::ops::element_size(dtype));
    require(r.data != nullptr, null_message);
    check_aligned(r.data, "rows must be 16-byte aligned");
    require(r.row_stride % piece == 0 && r.head_stride % piece == 0,
            "row and head strides must be multiples of 16 bytes");
    require(r.row_stride >= 0 && r.row_stride <= (int64_t{1} << 22) && r.head_stride >= 0,
            "row strides must be 0 to 2^22 elements");
}

void check_buckets(const float* table, const int32_t* buckets, int num_buckets, int reach) {
    require(table != nullptr && buckets != nullptr, "a bias needs a table and its bucket ids");
    require(num_buckets > 0 && num_buckets <= TRW_OPS_MAX_BUCKETS, "1 to 256 buckets");
    require(reach >= 0 && reach <= TRW_OPS_MAX_REACH, "reach must be 0 to 1024");
}

// Times of no rows may be NULL (an empty tensor's address is).
void check_score(const trw_score& s, int64_t q_rows, int64_t k_rows) {
    require(std::isfinite(s.scale), "scale must be finite");
    require(std::isfinite(s.softcap) && s.softcap >= 0, "softcap must be finite and not negative");
    if (s.table || s.buckets)
        check_buckets(s.table, s.buckets, s.num_buckets, s.reach);
    const bool times = s.q_times || s.k_times;
    require(!times || ((s.q_times || q_rows == 0) && (s.k_times || k_rows == 0)),
            "times are needed for the queries and the keys");
    require(!times || s.slopes, "times are for slopes");
}

const trw_attention_params& checked(const trw_attention_params* p) {
    require(p != nullptr, "null argument");
    check_heads(p->dtype, p->heads, p->kv_heads, p->dim);
    require(p->q_rows >= 0 && p->k_rows >= 0 && p->q_rows < kMaxRows && p->k_rows < kMaxRows,
            "rows must be 0 to 2^30 - 1");
    require(((p->q_rows + 127) / 128 + 8) * p->heads < (int64_t{1} << 31) &&
                ((p->k_rows + 127) / 128 + 8) * p->heads < (int64_t{1} << 31),
            "too many rows and heads");
    require(p->docs >= 0 && p->docs < kMaxRows && p->longest >= 0,
            "docs must be 0 to 2^30 - 1, longest not negative");
    require((p->docs + 7) * p->kv_heads < (int64_t{1} << 31), "too many documents and heads");
    check_score(p->score, p->q_rows, p->k_rows);
    return *p;
}

void check_forward(const trw_attention_params& p) {
    check_rows(p.q, p.dtype, p.q_rows, "q is null");
    check_rows(p.k, p.dtype, p.k_rows, "k is null");
    check_rows(p.v, p.dtype, p.k_rows, "v is null");
    check_rows(p.out, p.dtype, p.q_rows, "out is null");
    if (p.out_low.data) check_rows(p.out_low, p.dtype, p.q_rows, "out_low is null");
    require(p.q_rows == 0 || p.q_rows_info, "q_rows_info is null");
    check_aligned(p.q_rows_info, "q_rows_info must be 16-byte aligned");
    require(p.docs == 0 || p.docs_info, "docs_info is null");
    check_aligned(p.docs_info, "docs_info must be 16-byte aligned");
    require(reinterpret_cast<uintptr_t>(p.stats) % 8 == 0, "stats must be 8-byte aligned");
}

const trw_attention_step_params& checked(const trw_attention_step_params* p) {
    require(p != nullptr, "null argument");
    check_heads(p->dtype, p->heads, p->kv_heads, p->dim);
    require(p->batch >= 0 && p->batch < kMaxRows, "batch must be 0 to 2^30 - 1");
    require(p->capacity >= 0 && p->capacity < kMaxRows, "capacity must be 0 to 2^30 - 1");
    require(p->batch * p->heads < (int64_t{1} << 31) / 1024, "too many walks and heads");
    check_score(p->score, p->batch, p->batch * p->capacity);
    return *p;
}

const trw_relative_bias_params& checked(const trw_relative_bias_params* p) {
    require(p != nullptr, "null argument");
    check_dtype(p->dtype);
    require(p->heads > 0 && p->heads <= 4096, "1 to 4096 heads");
    require(p->q_len >= 0 && p->k_len >= 0 && p->q_len < kMaxRows && p->k_len < kMaxRows,
            "lengths must be 0 to 2^30 - 1");
    require(p->q_offset > -kMaxRows && p->q_offset < kMaxRows, "q_offset is out of range");
    check_buckets(static_cast<const float*>(p->table), p->buckets, p->num_buckets, p->reach);
    return *p;
}

}  // namespace

extern "C" {

trw_status trw_ops_walk_mask(const trw_walk_mask_params* params, void* stream) {
    return guarded([&] {
        require(params != nullptr, "null argument");
        const trw_walk_mask_params& p = *params;
        require(p.docs >= 0 && p.docs < kMaxRows, "docs must be 0 to 2^30 - 1");
        require(p.q_rows >= 0 && p.k_rows >= 0 && p.q_rows < kMaxRows && p.k_rows < kMaxRows,
                "rows must be 0 to 2^30 - 1");
        require(p.kind == TRW_MASK_FULL || p.kind == TRW_MASK_CAUSAL || p.kind == TRW_MASK_PREFIX,
                "unknown kind of mask");
        if (p.q_offsets) {
            require(!p.q_lens && !p.k_lens, "lens are for padded walks, offsets for packed ones");
            require(p.k_offsets || p.k_rows == p.q_rows,
                    "k_rows must be q_rows where k_offsets is null");
        } else {
            require(!p.k_offsets, "k_offsets need q_offsets");
            require(p.q_length >= 0 && (p.q_length > 0 || p.q_rows == 0) &&
                        p.q_rows == p.docs * p.q_length,
                    "q_rows must be docs * q_length");
            const bool own = !p.k_lens;
            require(own ? p.k_rows == p.q_rows
                        : p.k_length >= 0 && (p.k_length > 0 || p.k_rows == 0) &&
                              p.k_rows == p.docs * p.k_length,
                    "k_rows must be docs * k_length");
        }
        require(p.kind != TRW_MASK_PREFIX || p.prefix || p.docs == 0, "prefix is null");
        require((p.q_rows == 0 || p.q_rows_info) && (p.k_rows == 0 || p.k_rows_info),
                "the rows' info is null");
        check_aligned(p.q_rows_info, "q_rows_info must be 16-byte aligned");
        check_aligned(p.k_rows_info, "k_rows_info must be 16-byte aligned");
        require(p.docs == 0 || p.docs_info, "docs_info is null");
        check_aligned(p.docs_info, "docs_info must be 16-byte aligned");
        trw::ops::walk_mask(p, static_cast<hipStream_t>(stream));
    });
}

trw_status trw_ops_attention_workspace(const trw_attention_params* params, int32_t backward,
                                       uint64_t* bytes) {
    return guarded([&] {
        require(bytes != nullptr, "null argument");
        trw::ops::require_grids(checked(params), backward != 0);
        *bytes = trw::ops::attention_workspace(*params, backward != 0);
    });
}

trw_status trw_ops_attention_forward(const trw_attention_params* params, void* stream) {
    return guarded([&] {
        const trw_attention_params& p = checked(params);
        check_forward(p);
        check_aligned(p.workspace, "workspace must be 16-byte aligned");
        trw::ops::require_grids(p, false);
        trw::ops::attention_forward(p, static_cast<hipStream_t>(stream));
    });
}

trw_status trw_ops_attention_backward(const trw_attention_params* params, void* stream) {
    return guarded([&] {
        const trw_attention_params& p = checked(params);
        check_forward(p);
        check_rows(p.d_out, p.dtype, p.q_rows, "d_out is null");
        check_rows(p.d_q, p.dtype, p.q_rows, "d_q is null");
        check_rows(p.d_k, p.dtype, p.k_rows, "d_k is null");
        check_rows(p.d_v, p.dtype, p.k_rows, "d_v is null");
        require(p.q_rows == 0 || p.stats, "stats is null");
        require(p.k_rows == 0 || p.k_rows_info, "k_rows_info is null");
        require(!p.score.table || p.d_table, "d_table is null");
        check_aligned(p.k_rows_info, "k_rows_info must be 16-byte aligned");
        check_aligned(p.workspace, "workspace must be 16-byte aligned");
        trw::ops::require_grids(p, true);
        trw::ops::attention_backward(p, static_cast<hipStream_t>(stream));
    });
}

trw_status trw_ops_attention_step_workspace(const trw_attention_step_params* params,
                                            uint64_t* bytes) {
    return guarded([&] {
        require(bytes != nullptr, "null argument");
        *bytes = trw::ops::attention_step_workspace(checked(params));
    });
}

trw_status trw_ops_attention_step(const trw_attention_step_params* params, void* stream) {
    return guarded([&] {
        const trw_attention_step_params& p = checked(params);
        check_rows(p.q, p.dtype, p.batch, "q is null");
        check_rows(p.k, p.dtype, p.batch, "k is null");
        check_rows(p.v, p.dtype, p.batch, "v is null");
        check_rows(p.out, p.dtype, p.batch, "out is null");
        require(p.batch == 0 || p.lens, "lens is null");
        const int64_t slots = p.batch * p.capacity;
        check_rows(trw_rows{p.k_cache, p.k_pos_stride, p.k_head_stride}, p.dtype, slots,
                   "k_cache is null");
        check_rows(trw_rows{p.v_cache, p.v_pos_stride, p.v_head_stride}, p.dtype, slots,
                   "v_cache is null");
        // Walks write their new rows at once: no two may be one.
        const auto apart = [](int64_t n, int64_t stride) { return n <= 1 || stride != 0; };
        require(apart(p.batch, p.k_batch_stride) && apart(p.batch, p.v_batch_stride) &&
                    apart(p.capacity, p.k_pos_stride) && apart(p.capacity, p.v_pos_stride) &&
                    apart(p.kv_heads, p.k_head_stride) && apart(p.kv_heads, p.v_head_stride),
                "a cache's rows must not share memory");
        const int64_t piece = 16 / static_cast<int64_t>(trw::ops::element_size(p.dtype));
        require(p.k_batch_stride % piece == 0 && p.v_batch_stride % piece == 0,
                "batch strides must be multiples of 16 bytes");
        check_aligned(p.workspace, "workspace must be 16-byte aligned");
        trw::ops::attention_step(p, static_cast<hipStream_t>(stream));
    });
}

trw_status trw_ops_relative_bias(const trw_relative_bias_params* params, void* stream) {
    return guarded([&] {
        const trw_relative_bias_params& p = checked(params);
        require(p.q_len * p.k_len == 0 || p.out, "out is null");
        check_aligned(p.out, "out must be 16-byte aligned");
        trw::ops::relative_bias(p, static_cast<hipStream_t>(stream));
    });
}

trw_status trw_ops_relative_bias_workspace(const trw_relative_bias_params* params,
                                           uint64_t* bytes) {
    return guarded([&] {
        require(bytes != nullptr, "null argument");
        *bytes = trw::ops::relative_bias_workspace(checked(params));
    });
}

trw_status trw_ops_relative_bias_backward(const trw_relative_bias_params* params, void* stream) {
    return guarded([&] {
        const trw_relative_bias_params& p = checked(params);
        require(p.q_len * p.k_len == 0 || p.d_out, "d_out is null");
        require(p.d_table != nullptr, "d_table is null");
        require(reinterpret_cast<uintptr_t>(p.d_out) % trw::ops::element_size(p.dtype) == 0,
                "d_out is misaligned");
        trw::ops::relative_bias_backward(p, static_cast<hipStream_t>(stream));
    });
}

const char* trw_ops_last_error(void) { return g_last_error.c_str(); }

int32_t trw_ops_abi_version(void) { return TRW_OPS_ABI_VERSION; }

}  // extern "C"
