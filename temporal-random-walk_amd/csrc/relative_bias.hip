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
// Backward: sums by distance first, in lanes' registers and lines of LDS that
// one wave adds to in its own order; workgroups' lines are joined in a fixed
// order, and distances become buckets once, at the end.
//
// 16 heads, 4096 rows of 4199 columns, bfloat16 (550 MB a direction): 90 us
// forward (6.1 TB/s, a fill reaches 6.9), 180 us for the sums by distance (3.1
// TB/s; a large library sum reaches 3.8, an attention step over caches 4.6), 21 for
// the two joins.
#include "operators.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;

struct BiasArgs {
    trw_relative_bias_params p;
    int rows_per_group;
    float* partial;  // backward: [heads, workgroups, 2 reach + 1]
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

// Sums by distance: wave w walks down every fourth row of the workgroup's, its
// lanes at consecutive 16-byte pieces.  Past the reach a sum in
// registers is enough.  Within it a piece's elements go to the wave's own line
// in LDS, distance d of it in slot (d % kElems) (line / kElems) + d / kElems, so
// that lanes (kElems apart in distance) meet neither in a slot nor in a bank.
template <typename T>
__global__ __launch_bounds__(kThreads, 8) void relative_bias_backward_kernel(BiasArgs a) {
    constexpr int kElems = 16 / sizeof(T);
    constexpr int kAhead = 2;  // pieces of a lane in flight
    extern __shared__ float s_lines[];  // [4][kElems * pieces]
    const trw_relative_bias_params& p = a.p;
    const int reach = p.reach, line = 2 * reach + 1;
    const int pieces = (line + kElems - 1) / kElems;
    const int head = blockIdx.y;
    const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6;
    for (int n = thread; n < 4 * kElems * pieces; n += kThreads) s_lines[n] = 0.0f;
    __syncthreads();
    float* s = s_lines + wave * kElems * pieces;

    // Pieces begin at multiples of kElems whatever the rows' alignment, so that
    // a gradient's layout does not change its bits.
    typedef u32x4 loose __attribute__((aligned(2)));
    union Piece {
        u32x4 u;
        T t[kElems];
    };
    const T* base = static_cast<const T*>(p.d_out) + head * p.d_out_head_stride;
    const int k_len = static_cast<int>(p.k_len);
    const int row0 = static_cast<int>(blockIdx.x * static_cast<int64_t>(a.rows_per_group)) + wave;
    const int row1 = static_cast<int>(min((blockIdx.x + int64_t{1}) * a.rows_per_group, p.q_len));
    auto fetch = [&](int i, int j) {
        Piece x;
        const T* at = base + i * p.d_out_row_stride + j;
        if (j + kElems <= k_len) {
            x.u = *reinterpret_cast<const loose*>(at);
        } else {
            x.u = u32x4{0, 0, 0, 0};
            if (j < k_len) {
#pragma unroll
                for (int e = 0; e < kElems; ++e)
                    if (j + e < k_len) x.t[e] = at[e];
            }
        }
        return x;
    };
    // A wave's pieces in order, the next kAhead of them on their way
    Piece x[kAhead];
    int load_i = row0, load_g = 0;
    auto advance = [&](int& i, int& g) {
        g += 64 * kElems;
        if (g >= k_len) {
            g = 0;
            i += kThreads / 64;
        }
    };
#pragma unroll
    for (int n = 0; n < kAhead; ++n)
        if (load_i < row1) {
            x[n] = fetch(load_i, load_g + lane * kElems);
            advance(load_i, load_g);
        }
    float before = 0.0f, after = 0.0f;
    for (int i = row0, g = 0; i < row1;) {
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            if (i >= row1) break;
            const Piece now = x[n];
            if (load_i < row1) {
                x[n] = fetch(load_i, load_g + lane * kElems);
                advance(load_i, load_g);
            }
            // distances of the wave's pieces: first .. first - 64 kElems + 1
            const int first = i + static_cast<int>(p.q_offset) - g;
            if (first - 64 * kElems + 1 >= reach || first <= -reach) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < kElems; ++e) sum += static_cast<float>(now.t[e]);
                if (first <= -reach) after += sum;
                else before += sum;
            } else {
                // Read, add, write: no two elements of a wave's pieces share a
                // slot, and float atomics of LDS take 100 cycles an instruction.
                const int mine = first - lane * kElems + reach;  // slot of element 0
                float line_value[kElems];
                int slot[kElems];
#pragma unroll
                for (int e = 0; e < kElems; ++e) {
                    const int at = mine - e;
                    const float value = static_cast<float>(now.t[e]);
                    // each once, also where reach 0 makes the two ends one
                    before += at >= 2 * reach ? value : 0.0f;
                    after += at <= 0 && at < 2 * reach ? value : 0.0f;
                    const unsigned in = at > 0 && at < 2 * reach ? at : 0;  // 0: read only
                    slot[e] = in % kElems * pieces + in / kElems;
                    line_value[e] = s[slot[e]] + value;
                }
#pragma unroll
                for (int e = 0; e < kElems; ++e)
                    if (slot[e]) s[slot[e]] = line_value[e];
            }
            advance(i, g);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        before += __shfl_xor(before, o);
        after += __shfl_xor(after, o);
    }
    __syncthreads();
    if (lane == 0) {
        const int at = 2 * reach;
        s[at % kElems * pieces + at / kElems] += before;
        s[0] += after;
    }
    __syncthreads();
    float* out = a.partial + (static_cast<int64_t>(head) * gridDim.x + blockIdx.x) * line;
    for (int n = thread; n < line; n += kThreads) {
        const int at = n % kElems * pieces + n / kElems;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) sum += s_lines[w * kElems * pieces + at];
        out[n] = sum;
    }
}

// Sums tiles' lines into `groups` lines per head: a thread per distance, every
// groups-th tile.
__global__ __launch_bounds__(kThreads) void join_lines_kernel(const float* partial, int64_t tiles,
                                                              int short_line, int groups,
                                                              float* lines, int first, int count,
                                                              int line) {
    const int group = blockIdx.x % groups;
    const int64_t head = blockIdx.x / groups;
    float* out = lines + (head * count + first + group) * line;
    for (int n = threadIdx.x; n < line; n += kThreads) {
        const int at = n - (line - short_line) / 2;
        float sum = 0.0f;
        if (at >= 0 && at < short_line) {
#pragma unroll 8
            for (int64_t t = group; t < tiles; t += groups)
                sum += partial[(head * tiles + t) * short_line + at];
        }
        out[n] = sum;
    }
}

// A head's lines to its table: distances first, in float64, then each bucket's
// by sixteen threads (bucket ids may come in any order).  One workgroup a head:
// it waits for memory, not for arithmetic, so it is as large as can be.  16
// heads, 64 lines of 1025 distances: 14 us, 38 with 256 threads, 8 loads in
// flight and 8 threads a bucket.
constexpr int kTableThreads = 1024;
constexpr int kBucketThreads = 16;
// Lines in flight; past the last one it is read again, so that no remainder goes
// one latency after the other.
constexpr int kAtOnce = 16;

template <typename T>
__global__ __launch_bounds__(kTableThreads) void join_table_kernel(
    const float* lines, int count, const int32_t* buckets, int line, int num_buckets, T* d_table) {
    extern __shared__ double s_sum[];  // [line], then the ids
    int* s_id = reinterpret_cast<int*>(s_sum + line);
    const int64_t head = blockIdx.x;
    for (int n = threadIdx.x; n < line; n += kTableThreads) {
        const float* from = lines + head * count * line + n;
        double sum = 0.0;
        for (int t = 0; t < count; t += kAtOnce) {
            float x[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                x[u] = from[static_cast<int64_t>(min(t + u, count - 1)) * line];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) sum += t + u < count ? x[u] : 0.0f;
        }
        s_sum[n] = sum;
        s_id[n] = min(max(buckets[n], 0), num_buckets - 1);
    }
    __syncthreads();
    const int part = threadIdx.x % kBucketThreads;
    for (int b = threadIdx.x / kBucketThreads; b < num_buckets; b += kTableThreads / kBucketThreads) {
        double sum = 0.0;
        for (int n = part; n < line; n += kBucketThreads)
            if (s_id[n] == b) sum += s_sum[n];
#pragma unroll
        for (int o = 1; o < kBucketThreads; o *= 2) sum += __shfl_xor(sum, o);
        if (part == 0) d_table[head * num_buckets + b] = static_cast<T>(static_cast<float>(sum));
    }
}

int64_t row_groups(const trw_relative_bias_params& p, int* rows_per_group) {
    // as many rows as leave 2048 workgroups, in whole rounds of the four waves
    int64_t rows = (p.q_len * p.heads + 2047) / 2048;
    rows = (rows + 3) / 4 * 4;
    *rows_per_group = static_cast<int>(rows);
    return (p.q_len + rows - 1) / rows;
}

template <typename F>
void by_type(int dtype, F&& f) {
    if (dtype == TRW_F32) f(float{});
    else if (dtype == TRW_F16) f(_Float16{});
    else f(__bf16{});
}

}  // namespace

void join_lines(const float* partial, int64_t tiles, int short_line, int heads, int groups,
                float* lines, int first, int count, int reach, hipStream_t stream) {
    hipLaunchKernelGGL(join_lines_kernel, dim3(static_cast<unsigned>(heads * groups)),
                       dim3(kThreads), 0, stream, partial, tiles, short_line, groups, lines, first,
                       count, 2 * reach + 1);
    check_launch("join_lines");
}

void join_table(const float* lines, int count, int heads, const int32_t* buckets, int reach,
                int num_buckets, int dtype, void* d_table, hipStream_t stream) {
    const int line = 2 * reach + 1;
    by_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL((join_table_kernel<T>), dim3(static_cast<unsigned>(heads)),
                           dim3(kTableThreads), line * (sizeof(double) + sizeof(int)), stream, lines,
                           count, buckets, line, num_buckets, static_cast<T*>(d_table));
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
    require_grid((p.q_len + rows - 1) / rows, kThreads);
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
    int rows;
    const uint64_t groups = row_groups(p, &rows);
    return (groups + kJoinGroups) * p.heads * (2 * static_cast<uint64_t>(p.reach) + 1) *
           sizeof(float);
}

void relative_bias_backward(const trw_relative_bias_params& p, hipStream_t stream) {
    require(p.workspace_bytes >= relative_bias_workspace(p), "workspace is too small");
    BiasArgs a{};
    a.p = p;
    a.partial = static_cast<float*>(p.workspace);
    int64_t groups = 0;
    if (p.q_len && p.k_len) {
        groups = row_groups(p, &a.rows_per_group);
        by_type(p.dtype, [&](auto t) {
            constexpr int kElems = 16 / sizeof(t);
            const int pieces = (2 * p.reach + 1 + kElems - 1) / kElems;
            hipLaunchKernelGGL((relative_bias_backward_kernel<decltype(t)>),
                               dim3(static_cast<unsigned>(groups), static_cast<unsigned>(p.heads)),
                               dim3(kThreads), 4 * kElems * pieces * sizeof(float), stream, a);
        });
        check_launch("relative_bias_backward");
    }
    const int line = 2 * p.reach + 1;
    float* lines = a.partial;
    if (groups > kJoinGroups) {
        lines = a.partial + groups * p.heads * line;
        join_lines(a.partial, groups, line, p.heads, kJoinGroups, lines, 0, kJoinGroups, p.reach,
                   stream);
        groups = kJoinGroups;
    }
    join_table(lines, static_cast<int>(groups), p.heads, p.buckets, p.reach, p.num_buckets, p.dtype,
               p.d_table, stream);
}

}  // namespace ops
}  // namespace trw
