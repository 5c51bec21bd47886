// relative_bias.hip -- a learned bias by buckets of distance, dense, and its
// gradient.
//
//   out[h, i, j] = table[h, buckets[reach + clamp(i + offset - j)]]
//
// Both directions are one pass over [heads, q_len, k_len] and bound by memory.
//
// Forward: a row is a window of one line, the biases by falling distance.  A
// thread stores 16 bytes; the chunks of a row all start at the same place
// modulo a chunk, so a workgroup keeps the line once for each such place in
// LDS, and every chunk is one aligned 16-byte read of the right copy.
//
// Backward: a wave walks down the rows with its lanes at fixed distances, eight
// (float32: four) consecutive ones each, and sums them in registers; the loads
// slide by one element a row.  The sums are taken to buckets once per tile of
// rows, and the tiles' sums added in a fixed order.
#include "operators.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerWave = 64;  // backward: of one tile

struct BiasArgs {
    trw_relative_bias_params p;
    int rows_per_group;  // forward
    int row_tiles, bands;
    int64_t first_distance;  // of band 0
    float* partial;
};

// Chunks of a copy of the line: the first and the last are the ends alone, in
// every copy.
__host__ __device__ constexpr int copy_chunks(int reach, int elems) {
    return (2 * reach + 1 + 4 * elems - 1) / elems;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void relative_bias_kernel(BiasArgs a) {
    constexpr int kElems = 16 / sizeof(T);
    extern __shared__ u32x4 s_copies[];  // [kElems][chunks]
    const trw_relative_bias_params& p = a.p;
    const int line = 2 * p.reach + 1;
    const int chunks = copy_chunks(p.reach, kElems);
    const int head = blockIdx.y;
    const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6;
    const T* table = static_cast<const T*>(p.table) + static_cast<int64_t>(head) * p.num_buckets;

    // copy c, entry n: the line's entry n + c - 2 kElems, the ends repeated
    T* s = reinterpret_cast<T*>(s_copies);
    for (int n = thread; n < chunks * kElems; n += kThreads)
        for (int c = 0; c < kElems; ++c) {
            const int at = min(max(n + c - 2 * kElems, 0), line - 1);
            const int bucket = min(max(p.buckets[line - 1 - at], 0), p.num_buckets - 1);
            s[c * chunks * kElems + n] = table[bucket];
        }
    __syncthreads();

    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.rows_per_group;
    const int64_t row1 = min(row0 + a.rows_per_group, p.q_len);
    for (int64_t i = row0 + wave; i < row1; i += kThreads / 64) {
        const int64_t flat = (head * p.q_len + i) * p.k_len;
        T* row = static_cast<T*>(p.out) + flat;
        // chunk g: elements kElems g - lead ..
        const int lead = static_cast<int>(flat % kElems);
        const int64_t count = (lead + p.k_len + kElems - 1) / kElems;
        // line entry of column j: j + shift (distance i + q_offset - j falls)
        const int64_t shift = p.reach - (i + p.q_offset);
        for (int64_t g = lane; g < count; g += 64) {
            const int64_t j = g * kElems - lead;
            int64_t entry = j + shift + 2 * kElems;  // in copy 0
            const int c = static_cast<int>(((entry % kElems) + kElems) % kElems);
            entry = (entry - c) / kElems;
            const int64_t chunk = min(max(entry, int64_t{0}), static_cast<int64_t>(chunks - 1));
            union {
                u32x4 u;
                T t[kElems];
            } x;
            x.u = s_copies[c * chunks + chunk];
            if (j >= 0 && j + kElems <= p.k_len) {
                *reinterpret_cast<u32x4*>(row + j) = x.u;
            } else {
#pragma unroll
                for (int e = 0; e < kElems; ++e)
                    if (j + e >= 0 && j + e < p.k_len) row[j + e] = x.t[e];
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void relative_bias_backward_kernel(BiasArgs a) {
    constexpr int kElems = 16 / sizeof(T);
    constexpr int kBand = 64 * kElems;  // distances of a wave
    __shared__ float s_sum[4][kBand];
    const trw_relative_bias_params& p = a.p;
    const int band = blockIdx.x % a.bands;
    const int tile = blockIdx.x / a.bands;
    const int head = blockIdx.y;
    const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6;

    // this lane's elements of row i: columns i + j0 .., distances falling
    const int64_t top_d = a.first_distance + static_cast<int64_t>(band + 1) * kBand - 1;
    const int64_t j0 = p.q_offset - top_d + lane * kElems;
    float sum[kElems];
#pragma unroll
    for (int e = 0; e < kElems; ++e) sum[e] = 0.0f;
    const T* base = static_cast<const T*>(p.d_out) + head * p.d_out_head_stride;
    const int64_t row0 = (static_cast<int64_t>(tile) * 4 + wave) * kRowsPerWave;
    const int64_t row1 = min(row0 + kRowsPerWave, p.q_len);
    typedef u32x4 loose __attribute__((aligned(2)));  // slides by one element a row
#pragma unroll 4
    for (int64_t i = row0; i < row1; ++i) {
        const int64_t j = i + j0;
        const T* at = base + i * p.d_out_row_stride + j;
        union {
            u32x4 u;
            T t[kElems];
        } x;
        if (j >= 0 && j + kElems <= p.k_len) {
            x.u = *reinterpret_cast<const loose*>(at);
        } else {
#pragma unroll
            for (int e = 0; e < kElems; ++e)
                x.t[e] = j + e >= 0 && j + e < p.k_len ? at[e] : static_cast<T>(0.0f);
        }
#pragma unroll
        for (int e = 0; e < kElems; ++e) sum[e] += static_cast<float>(x.t[e]);
    }
#pragma unroll
    for (int e = 0; e < kElems; ++e) s_sum[wave][lane * kElems + e] = sum[e];
    __syncthreads();
    for (int n = thread; n < kBand; n += kThreads)
        s_sum[0][n] += s_sum[1][n] + s_sum[2][n] + s_sum[3][n];
    __syncthreads();
    // to buckets, each by 8 threads; entry n is distance top_d - n
    const int part = thread & 7;
    for (int b = thread >> 3; b < p.num_buckets; b += kThreads / 8) {
        float total = 0.0f;
        for (int n = part; n < kBand; n += 8) {
            const int64_t d =
                min(max(top_d - n, -static_cast<int64_t>(p.reach)), static_cast<int64_t>(p.reach));
            const int of = min(max(p.buckets[d + p.reach], 0), p.num_buckets - 1);
            if (of == b) total += s_sum[0][n];
        }
        total += __shfl_xor(total, 1);
        total += __shfl_xor(total, 2);
        total += __shfl_xor(total, 4);
        if (part == 0)
            a.partial[(static_cast<int64_t>(head) * gridDim.x + blockIdx.x) * p.num_buckets + b] =
                total;
    }
}

// One workgroup per entry of the table sums the tiles' sums.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_table_kernel(const float* partial, int64_t tiles,
                                                              int num_buckets, T* d_table) {
    const int bucket = blockIdx.x % num_buckets;
    const int64_t head = blockIdx.x / num_buckets;
    double sum = 0.0;
    for (int64_t t = threadIdx.x; t < tiles; t += kThreads)
        sum += partial[(head * tiles + t) * num_buckets + bucket];
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    __shared__ double s[4];
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        d_table[head * num_buckets + bucket] =
            static_cast<T>(static_cast<float>(s[0] + s[1] + s[2] + s[3]));
}

void shape_backward(BiasArgs& a) {
    const int band = 64 * 16 / static_cast<int>(element_size(a.p.dtype));
    a.first_distance = a.p.q_offset - a.p.k_len + 1;
    a.bands = static_cast<int>((a.p.q_len + a.p.k_len - 1 + band - 1) / band);
    a.row_tiles = static_cast<int>((a.p.q_len + 4 * kRowsPerWave - 1) / (4 * kRowsPerWave));
}

template <typename F>
void by_type(int dtype, F&& f) {
    if (dtype == TRW_F32) f(float{});
    else if (dtype == TRW_F16) f(_Float16{});
    else f(__bf16{});
}

}  // namespace

void join_table(const float* partial, int64_t tiles, int heads, int num_buckets, int dtype,
                void* d_table, hipStream_t stream) {
    by_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL((join_table_kernel<T>), dim3(static_cast<unsigned>(heads * num_buckets)),
                           dim3(kThreads), 0, stream, partial, tiles, num_buckets,
                           static_cast<T*>(d_table));
    });
    check_launch("join_table");
}

void relative_bias(const trw_relative_bias_params& p, hipStream_t stream) {
    if (p.q_len == 0 || p.k_len == 0 || p.heads == 0) return;
    BiasArgs a{};
    a.p = p;
    const int elems = 16 / static_cast<int>(element_size(p.dtype));
    // rows of a workgroup: 256 KB of output or more, so that filling the
    // copies (16 bytes for each of 2 reach + 1 entries) stays small beside it
    const int64_t row_bytes = p.k_len * static_cast<int64_t>(element_size(p.dtype));
    int64_t rows = (int64_t{256} << 10) / row_bytes;
    rows = rows < 4 ? 4 : rows > p.q_len ? p.q_len : rows;
    // but at least four workgroups for each of the 256 compute units
    const int64_t fair = p.q_len * p.heads / 1024;
    if (rows > fair) rows = fair < 4 ? 4 : fair;
    a.rows_per_group = static_cast<int>(rows);
    const int chunks = copy_chunks(p.reach, elems);
    const dim3 grid(static_cast<unsigned>((p.q_len + rows - 1) / rows),
                    static_cast<unsigned>(p.heads));
    by_type(p.dtype, [&](auto t) {
        hipLaunchKernelGGL((relative_bias_kernel<decltype(t)>), grid, dim3(kThreads),
                           static_cast<size_t>(chunks) * 16 * elems, stream, a);
    });
    check_launch("relative_bias");
}

uint64_t relative_bias_workspace(const trw_relative_bias_params& p) {
    if (p.q_len == 0 || p.k_len == 0) return 0;
    BiasArgs a{};
    a.p = p;
    shape_backward(a);
    return static_cast<uint64_t>(p.heads) * a.bands * a.row_tiles * p.num_buckets * sizeof(float);
}

void relative_bias_backward(const trw_relative_bias_params& p, hipStream_t stream) {
    require(p.workspace_bytes >= relative_bias_workspace(p), "workspace is too small");
    if (p.heads == 0) return;
    BiasArgs a{};
    a.p = p;
    a.partial = static_cast<float*>(p.workspace);
    int64_t tiles = 0;
    if (p.q_len && p.k_len) {
        shape_backward(a);
        tiles = static_cast<int64_t>(a.bands) * a.row_tiles;
        by_type(p.dtype, [&](auto t) {
            hipLaunchKernelGGL((relative_bias_backward_kernel<decltype(t)>),
                               dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(p.heads)),
                               dim3(kThreads), 0, stream, a);
        });
        check_launch("relative_bias_backward");
    }
    join_table(a.partial, tiles, p.heads, p.num_buckets, p.dtype, p.d_table, stream);
}

}  // namespace ops
}  // namespace trw
