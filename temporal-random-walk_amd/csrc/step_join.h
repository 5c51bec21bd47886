// step_join.h -- the second half of a step that several workgroups share: their
// sums over parts of a walk become one row.
#ifndef TRW_STEP_JOIN_H
#define TRW_STEP_JOIN_H

#include "operators.h"

namespace trw {
namespace ops {
namespace {

struct StepJoin {
    const float* partial;      // [batch, heads, splits, dim]
    const float2* part_stats;  // [batch, heads, splits]: maximum (base 2) and sum
    Rows out;
    const int64_t* lens;  // of a step over dense caches: what has no output; null: a sum of NaN says so
    int64_t capacity;
    int heads, dim, splits;
};

constexpr int kJoinThreads = 256;

// Joins the workgroups of one walk and head: 32 threads for the elements, four
// each, and eight shares of the workgroups.
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void join_step_kernel(StepJoin a) {
    __shared__ f32x4 s_sum[8][32];
    __shared__ float s_total[8], s_top[4];
    const int head = blockIdx.x % a.heads;
    const int b = blockIdx.x / a.heads;
    const int thread = threadIdx.x, share = thread >> 5, d = (thread & 31) * 4;
    const int64_t part = (static_cast<int64_t>(b) * a.heads + head) * a.splits;
    float top = kFloor;
    for (int s = thread; s < a.splits; s += kJoinThreads) top = fmaxf(top, a.part_stats[part + s].x);
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((thread & 63) == 0) s_top[thread >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    float total = 0.0f;
    f32x4 sum = {0, 0, 0, 0};
    // No branch inside, so that eight workgroups' loads are in flight (128 of them:
    // 4.8 us, 9.4 with a branch): threads past the head size read its last elements
    // again and store nothing.
    const float* from = a.partial + part * a.dim + min(d, a.dim - 4);
#pragma unroll 8
    for (int s = share; s < a.splits; s += 8) {
        const float2 st = a.part_stats[part + s];
        const f32x4 x = *reinterpret_cast<const f32x4*>(from + static_cast<int64_t>(s) * a.dim);
        const float by = exp2_fast(st.x - top);
        total = fmaf(by, st.y, total);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = fmaf(by, x[e], sum[e]);
    }
    s_sum[share][thread & 31] = sum;
    if ((thread & 31) == 0) s_total[share] = total;
    __syncthreads();
    if (share || d >= a.dim) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) {
        total += s_total[w];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += s_sum[w][thread & 31][e];
    }
    const int64_t n = a.lens ? a.lens[b] : 0;
    const bool full = a.lens && n >= a.capacity;
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        out[e] = static_cast<T>(n < 0             ? 0.0f
                                : full            ? NAN
                                : total != 0.0f   ? sum[e] / total
                                                  : 0.0f);
    *reinterpret_cast<t4*>(row_of<T>(a.out, b, head) + d) = out;
}

}  // namespace
}  // namespace ops
}  // namespace trw
#endif  // TRW_STEP_JOIN_H
