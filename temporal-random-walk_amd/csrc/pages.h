// pages.h -- caches of keys and values in pages of a common pool: where a walk's
// position lies, and rows in 8 bits.
//
// A page holds page_rows positions of every key head, [kv_heads, page_rows, D],
// so that a head's positions of a page are one piece of memory; the table names
// each walk's pages in order.  8 bits: a row x of one head is kept as e4m3 codes
// c and one exponent, x = c 2^e, with the smallest e that brings the row's
// largest value to 448 (e4m3's) or less.  Multiplying by 2^-e is exact, so that
// the code's rounding is the only one.
#ifndef TRW_PAGES_H
#define TRW_PAGES_H

#include "operators.h"

namespace trw {
namespace ops {

struct Pages {
    char *k, *v;
    uint8_t *k_scale, *v_scale;
    int64_t k_page, v_page, k_scale_page, v_scale_page;  // bytes from page to page
    const int32_t* table;
    int64_t table_stride;
    int table_pages, pages, shift;  // a page has 1 << shift rows

    // The page of a walk's position >= 0, or -1 where the walk has none.
    __device__ __forceinline__ int page_of(int64_t walk, int64_t position) const {
        const int64_t n = position >> shift;
        if (n >= table_pages) return -1;
        const int id = table[walk * table_stride + n];
        return id >= 0 && id < pages ? id : -1;
    }
};

inline size_t page_element_size(int dtype) { return dtype == TRW_E4M3 ? 1 : element_size(dtype); }

inline Pages make_pages(const trw_pages& p) {
    Pages r;
    const int64_t size = static_cast<int64_t>(page_element_size(p.dtype));
    r.k = static_cast<char*>(p.k);
    r.v = static_cast<char*>(p.v);
    r.k_scale = p.k_scale;
    r.v_scale = p.v_scale;
    r.k_page = p.k_stride * size;
    r.v_page = p.v_stride * size;
    r.k_scale_page = p.k_scale_stride;
    r.v_scale_page = p.v_scale_stride;
    r.table = p.table;
    r.table_stride = p.table_stride;
    r.table_pages = static_cast<int>(p.table_pages);
    r.pages = static_cast<int>(p.pages);
    r.shift = 0;
    while ((1 << r.shift) < p.page_rows) ++r.shift;
    return r;
}

// Whether blocks of a and of b, `count` of each and each `stride` bytes (its size or
// more) from the next, share memory; where strides differ, whether the ranges do.
inline bool share_memory(const void* a, int64_t a_size, int64_t a_stride, const void* b,
                         int64_t b_size, int64_t b_stride, int64_t count) {
    // (a range may not end inside the addresses that there are: __int128 holds its end)
    const __int128 d = static_cast<__int128>(reinterpret_cast<uintptr_t>(b)) -
                       static_cast<__int128>(reinterpret_cast<uintptr_t>(a));
    if (d >= static_cast<__int128>(count - 1) * a_stride + a_size ||
        -d >= static_cast<__int128>(count - 1) * b_stride + b_size)
        return false;
    if (count == 1 || a_stride != b_stride) return true;
    const int64_t at = static_cast<int64_t>((d % a_stride + a_stride) % a_stride);
    return at < a_size || at + b_size > a_stride;
}
// The last of the checks of pages that are written or read.
inline void require_apart(const trw_pages& p) {
    if (p.pages == 0) return;
    const int64_t size = static_cast<int64_t>(page_element_size(p.dtype));
    const int64_t lines = int64_t{p.kv_heads} * p.page_rows;
    struct {
        const void* at;
        int64_t size, stride;
    } const blocks[] = {{p.k, lines * p.dim * size, p.k_stride * size},
                        {p.v, lines * p.dim * size, p.v_stride * size},
                        {p.k_scale, lines, p.k_scale_stride},
                        {p.v_scale, lines, p.v_scale_stride}};
    const int count = p.dtype == TRW_E4M3 ? 4 : 2;
    for (int i = 0; i < count; ++i)
        for (int j = i + 1; j < count; ++j)
            require(!share_memory(blocks[i].at, blocks[i].size, blocks[i].stride, blocks[j].at,
                                  blocks[j].size, blocks[j].stride, p.pages),
                    "k, v and their scales must not share memory");
}

// ---- rows in 8 bits ------------------------------------------------------------------------------
// The exponents that a row may have: codes' smallest step stays a normal number
// of float32 and bfloat16 (2^-9 2^-117), and 2^-e is one.
constexpr int kLowestExponent = -117, kHighestExponent = 120;

// What a value counts for its row's largest: nothing where it is not finite.
__device__ __forceinline__ float size_of(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}
// The exponent of a row whose largest size is `top`, as it is kept: e + 127.
__device__ __forceinline__ int scale_byte(float top) {
    const uint32_t bits = __float_as_uint(top);
    // 448 = 1.75 2^8
    const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
    return min(max(e, kLowestExponent), kHighestExponent) + 127;
}
__device__ __forceinline__ float power_of(int byte) { return __uint_as_float(byte << 23); }
// 2^-e of a byte that scale_byte made.
__device__ __forceinline__ float inverse_power(int byte) { return __uint_as_float((254 - byte) << 23); }

// Eight values as codes, each times `by`; what is not finite becomes NaN.
__device__ __forceinline__ u32x2 eight_codes(const float (&x)[8], float by) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
        y[e] = fabsf(x[e]) <= 3.402823466e38f ? x[e] * by : __uint_as_float(0x7fc00000);
    u32x2 c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w, true);
        c[h] = static_cast<uint32_t>(w);
    }
    return c;
}
__device__ __forceinline__ void eight_values(u32x2 c, float (&x)[8]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[h]), false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[h]), true);
        x[4 * h] = lo[0];
        x[4 * h + 1] = lo[1];
        x[4 * h + 2] = hi[0];
        x[4 * h + 3] = hi[1];
    }
}

// Eight elements of a row in memory, as float32.
template <typename T>
__device__ __forceinline__ void load8(const T* from, float (&x)[8]) {
    union {
        u32x4 u[sizeof(T) / 2];
        Frag<T> f;
    } in;
#pragma unroll
    for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h)
        in.u[h] = reinterpret_cast<const u32x4*>(from)[h];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(in.f[e]);
}
template <typename T>
__device__ __forceinline__ void store8(T* to, const float (&x)[8]) {
    union {
        u32x4 u[sizeof(T) / 2];
        Frag<T> f;
    } out;
#pragma unroll
    for (int e = 0; e < 8; ++e) out.f[e] = static_cast<T>(x[e]);
#pragma unroll
    for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h)
        reinterpret_cast<u32x4*>(to)[h] = out.u[h];
}

// The largest over groups of `lanes` lanes (a power of two), in every one of them.
template <int kLanes>
__device__ __forceinline__ float group_max(float x) {
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

// f<T>() for a type of rows.
template <typename F>
void by_type(int dtype, F&& f) {
    if (dtype == TRW_F32)
        f(float{});
    else if (dtype == TRW_F16)
        f(_Float16{});
    else
        f(__bf16{});
}

void paged_copy(const trw_paged_copy_params& p, bool write, hipStream_t stream);
uint64_t paged_step_workspace(const trw_paged_step_params& p);
void paged_step(const trw_paged_step_params& p, hipStream_t stream);

}  // namespace ops
}  // namespace trw
#endif  // TRW_PAGES_H
