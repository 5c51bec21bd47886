// paged_copy.hip -- rows of walks to their pages, and back.
//
// Nothing is computed but a row's largest value and the codes: the operators are
// bound by memory.  Lanes hold eight elements each, a group of 4, 8 or 16 lanes a
// row of one head, so that a row's largest value is a few exchanges inside the
// group; a workgroup takes as many consecutive rows as its groups hold (16 to 64)
// of one head after the other: consecutive rows of a head are one piece of their
// page, and whole lines are written at once.
//
// Measured: 201,899 rows of 8 heads of 128 from bfloat16 to 8 bits 250 us, 4.97 TB/s of
// the 1.24 GB that are read and written; 120,065 back 146 us, 5.03 TB/s (a large copy:
// 5.17).  A few hundred rows take 4 us, the latency of three loads.
#include <algorithm>

#include "pages.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;

struct CopyArgs {
    Pages pages;
    Rows k, v;
    const int64_t *counts, *offsets, *starts;
    float *times, *k_times;
    int64_t rows, walks;
    int length, heads, dim;
};

// The last of offsets [first, last] that is `row` or less (`first` if none is),
// by a wave: 64 at once, so that thousands of walks take two or three loads one
// after the other.
__device__ __forceinline__ int64_t last_at_most(const int64_t* offsets, int64_t walks, int64_t row,
                                                int lane) {
    int64_t lo = 0, hi = walks;  // the answer is in [lo, hi)
    while (hi - lo > 1) {
        const int64_t step = (hi - lo + 63) / 64;
        const int64_t at = lo + lane * step;
        const bool here = at < hi && offsets[at] <= row;
        const int count = __popcll(__ballot(here));
        lo += max(count - 1, 0) * step;
        hi = min(lo + step, hi);
    }
    return lo;
}

template <typename T, int kGroup, bool kWrite, bool kEight>
__global__ __launch_bounds__(kThreads) void paged_copy_kernel(CopyArgs a) {
    constexpr int kRows = kThreads / kGroup;
    const int thread = threadIdx.x, sub = thread % kGroup;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + thread / kGroup;

    // whose row, and which of its rows
    int64_t walk = -1, number = 0;
    bool mine = row < a.rows;
    if (a.offsets) {
        if (a.walks > 0) {
            const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows;
            const int lane = thread & 63;
            walk = last_at_most(a.offsets, a.walks, first, lane);
            int64_t end = last_at_most(a.offsets, a.walks, min(first + kRows, a.rows) - 1, lane) + 1;
            while (end - walk > 1) {
                const int64_t mid = walk + (end - walk) / 2;
                if (a.offsets[mid] <= row) walk = mid;
                else end = mid;
            }
            number = row - a.offsets[walk];
            mine = mine && number >= 0 && number < a.rows && row < a.offsets[walk + 1];
        } else {
            mine = false;
        }
    } else if (mine) {
        walk = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.length);
        number = row - walk * a.length;
        if (a.counts) mine = number < a.counts[walk];
    }
    const int64_t start = mine && a.starts ? a.starts[walk] : 0;
    mine = mine && start >= 0 && start < (int64_t{1} << 31);
    const int64_t position = start + number;
    const int page = mine ? a.pages.page_of(walk, position) : -1;
    const int slot = static_cast<int>(position & ((1 << a.pages.shift) - 1));
    mine = page >= 0;
    if (kWrite && !mine) return;  // (whole groups: a group has one row)
    if (!kWrite && row >= a.rows) return;

    if (a.times && blockIdx.y == 0 && sub == 0) {
        float* held = a.k_times + (static_cast<int64_t>(page) << a.pages.shift) + slot;
        if (kWrite) *held = a.times[row];
        else a.times[row] = mine ? *held : 0.0f;
    }
    const int col = sub * 8;
    const bool in = col < a.dim;
    const int size = kEight ? 1 : sizeof(T);
    for (int head = blockIdx.y; head < a.heads; head += gridDim.y) {
        const int64_t line = (static_cast<int64_t>(head) << a.pages.shift) + slot;
        const int64_t k_at = page * a.pages.k_page + (line * a.dim + col) * size;
        const int64_t v_at = page * a.pages.v_page + (line * a.dim + col) * size;
        T* k_row = row_of<T>(a.k, row, head) + col;
        T* v_row = row_of<T>(a.v, row, head) + col;
        if constexpr (!kEight) {
            if (!in) continue;
            constexpr int kPieces = sizeof(T) / 2;
            u32x4* k_page = reinterpret_cast<u32x4*>(a.pages.k + k_at);
            u32x4* v_page = reinterpret_cast<u32x4*>(a.pages.v + v_at);
            u32x4 *k_to = kWrite ? k_page : reinterpret_cast<u32x4*>(k_row);
            u32x4 *v_to = kWrite ? v_page : reinterpret_cast<u32x4*>(v_row);
            const u32x4 *k_from = kWrite ? reinterpret_cast<u32x4*>(k_row) : k_page;
            const u32x4 *v_from = kWrite ? reinterpret_cast<u32x4*>(v_row) : v_page;
            u32x4 k[kPieces] = {}, v[kPieces] = {};
            if (mine) {
#pragma unroll
                for (int n = 0; n < kPieces; ++n) {
                    k[n] = k_from[n];
                    v[n] = v_from[n];
                }
            }
#pragma unroll
            for (int n = 0; n < kPieces; ++n) {
                k_to[n] = k[n];
                v_to[n] = v[n];
            }
        } else if constexpr (kWrite) {
            float k[8] = {}, v[8] = {}, k_top = 0.0f, v_top = 0.0f;
            if (in) {
                load8(k_row, k);
                load8(v_row, v);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                k_top = fmaxf(k_top, size_of(k[e]));
                v_top = fmaxf(v_top, size_of(v[e]));
            }
            const int k_byte = scale_byte(group_max<kGroup>(k_top));
            const int v_byte = scale_byte(group_max<kGroup>(v_top));
            if (in) {
                *reinterpret_cast<u32x2*>(a.pages.k + k_at) = eight_codes(k, inverse_power(k_byte));
                *reinterpret_cast<u32x2*>(a.pages.v + v_at) = eight_codes(v, inverse_power(v_byte));
            }
            if (sub == 0) {
                a.pages.k_scale[page * a.pages.k_scale_page + line] = k_byte;
                a.pages.v_scale[page * a.pages.v_scale_page + line] = v_byte;
            }
        } else if (in) {
            float k[8] = {}, v[8] = {};
            if (mine) {
                const u32x2 kc = *reinterpret_cast<const u32x2*>(a.pages.k + k_at);
                const u32x2 vc = *reinterpret_cast<const u32x2*>(a.pages.v + v_at);
                const float kf = power_of(a.pages.k_scale[page * a.pages.k_scale_page + line]);
                const float vf = power_of(a.pages.v_scale[page * a.pages.v_scale_page + line]);
                eight_values(kc, k);
                eight_values(vc, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    k[e] *= kf;
                    v[e] *= vf;
                }
            }
            store8(k_row, k);
            store8(v_row, v);
        }
    }
}

}  // namespace

void paged_copy(const trw_paged_copy_params& p, bool write, hipStream_t stream) {
    require_apart(p.pages);
    if (p.rows == 0) return;
    CopyArgs a;
    a.pages = make_pages(p.pages);
    a.k = make_rows(p.k);
    a.v = make_rows(p.v);
    a.counts = p.counts;
    a.offsets = p.offsets;
    a.starts = p.starts;
    a.times = p.times;
    a.k_times = p.k_times;
    a.rows = p.rows;
    a.walks = p.pages.walks;
    a.length = static_cast<int>(p.length);
    a.heads = p.pages.kv_heads;
    a.dim = p.pages.dim;
    const int group = a.dim <= 32 ? 4 : a.dim <= 64 ? 8 : 16;
    const int64_t chunks = (p.rows + kThreads / group - 1) / (kThreads / group);
    // Heads are taken one after the other, by as many workgroups as fill the device.
    const int split = static_cast<int>(
        std::min<int64_t>(a.heads, std::max<int64_t>(1, (4096 + chunks - 1) / chunks)));
    require_grid(chunks * split, kThreads);
    const dim3 grid(static_cast<unsigned>(chunks), split);
    const bool eight = p.pages.dtype == TRW_E4M3;
    by_type(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        auto launch = [&](auto lanes, auto writes, auto codes) {
            hipLaunchKernelGGL((paged_copy_kernel<T, decltype(lanes)::value, decltype(writes)::value,
                                                  decltype(codes)::value>),
                               grid, dim3(kThreads), 0, stream, a);
        };
        auto by_codes = [&](auto lanes, auto writes) {
            if (eight) launch(lanes, writes, std::true_type());
            else launch(lanes, writes, std::false_type());
        };
        auto by_way = [&](auto lanes) {
            if (write) by_codes(lanes, std::true_type());
            else by_codes(lanes, std::false_type());
        };
        if (group == 4) by_way(std::integral_constant<int, 4>());
        else if (group == 8) by_way(std::integral_constant<int, 8>());
        else by_way(std::integral_constant<int, 16>());
    });
    check_launch(write ? "paged_write" : "paged_read");
}

}  // namespace ops
}  // namespace trw
