// beams.hip -- beam search over a walk's next nodes: the best continuations of
// each group's beams, and the beams' pages put in their order.
//
// Choice.  log p of node x after beam b is score_b + x - log sum exp(row b), and
// inside a row the order is that of the logits alone, so one pass over them does:
// a wave takes 8 x 16 bytes a lane, keeps their maximum, the sum of their
// exponentials and its best candidates; a workgroup joins four waves' and writes
// one list.  A second launch joins a group's lists and adds scores in float64,
// where candidates of different beams meet.  Lanes hold the same nodes whatever the
// row's alignment, so that equal rows have equal sums and ties go to the lowest
// index.
//
// A wave's best `width` of its nodes: at least `width` of them reach the width-th
// largest of the 64 lanes' largest ones, and hardly more do.  Those are listed and
// ranked by counting.
#include <algorithm>
#include <cmath>

#include "beams.h"
#include "pages.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kPieces = 8;   // 16-byte pieces of a lane
constexpr int kListed = 256; // candidates of a wave before the best are taken from them
constexpr int kMost = TRW_OPS_BEAMS;

typedef unsigned long long u64;

struct SelectArgs {
    const char* logits;
    int64_t group_stride, beam_stride;  // elements
    const float* scores;
    const uint8_t* ended;
    int64_t end_token;
    int groups, beams, width, nodes, parts;
    u64* lists;      // [groups, beams, parts, width]
    float2* sums;    // [groups, beams, parts] maximum and sum
    float* out_scores;
    int64_t *out_tokens, *out_parents;
    uint8_t* out_ended;
};

// A candidate as one number: greater is better, and of equal logits the lower node.
// 0: none.
__device__ __forceinline__ u64 key_of(float x, uint32_t node) {
    const uint32_t bits = __float_as_uint(x + 0.0f);  // -0 is 0
    const uint32_t order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return static_cast<u64>(order) << 32 | (0xffffffffu - node);
}
__device__ __forceinline__ float logit_of(u64 key) {
    const uint32_t order = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint32_t node_of(u64 key) {
    return 0xffffffffu - static_cast<uint32_t>(key);
}

__device__ __forceinline__ float wave_top(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// The first `width` of `count` keys (different ones, or 0) in order, to `best` (0
// where there are none left), by one wave.  keys and best: LDS, apart; width up to
// 64, count up to kListed.
__device__ __forceinline__ void take_best(const u64* keys, int count, u64* best, int width,
                                          int lane) {
    u64 mine[kListed / 64];
    int rank[kListed / 64];
#pragma unroll
    for (int i = 0; i < kListed / 64; ++i) {
        const int at = i * 64 + lane;
        mine[i] = at < count ? keys[at] : 0;
        rank[i] = 0;
    }
    if (count <= 64) {
        for (int j = 0; j < count; ++j) rank[0] += keys[j] > mine[0];
    } else {
        for (int j = 0; j < count; ++j) {
            const u64 other = keys[j];
#pragma unroll
            for (int i = 0; i < kListed / 64; ++i) rank[i] += other > mine[i];
        }
    }
    if (lane < width) best[lane] = 0;
#pragma unroll
    for (int i = 0; i < kListed / 64; ++i)
        if (mine[i] && rank[i] < width) best[rank[i]] = mine[i];
}

template <typename T>
struct Piece {
    static constexpr int kElems = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(kElems)));
    vec x;
    __device__ __forceinline__ float at(int e) const { return static_cast<float>(x[e]); }
};

// One row's nodes of a workgroup: four waves of 64 lanes of 128 bytes.
template <typename T>
__global__ __launch_bounds__(kThreads) void select_rows_kernel(SelectArgs a) {
    constexpr int kElems = Piece<T>::kElems;
    constexpr int kWaveNodes = 64 * kPieces * kElems;
    __shared__ u64 s_listed[kWaves][kListed];
    __shared__ u64 s_best[kWaves][kMost];
    __shared__ u64 s_joined[kMost];
    __shared__ float s_top[kWaves], s_sum[kWaves];

    const int part = blockIdx.x % a.parts;
    const int64_t row = blockIdx.x / a.parts;  // group and beam
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // No candidates come of a beam that has ended or that is none: it is not read.
    if (a.ended && a.ended[row]) return;
    if (!(fabsf(a.scores[row]) <= 3.402823466e38f)) return;

    const T* logits = reinterpret_cast<const T*>(a.logits) +
                      row / a.beams * a.group_stride + row % a.beams * a.beam_stride;
    const int begin = (part * kWaves + wave) * kWaveNodes;
    Piece<T> x[kPieces];
    if (begin + kWaveNodes <= a.nodes) {
#pragma unroll
        for (int c = 0; c < kPieces; ++c)  // 16 bytes of any alignment
            __builtin_memcpy(&x[c], logits + begin + (c * 64 + lane) * kElems, 16);
    } else {
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = begin + (c * 64 + lane) * kElems;
            if (at + kElems <= a.nodes) {
                __builtin_memcpy(&x[c], logits + at, 16);
            } else {
#pragma unroll
                for (int e = 0; e < kElems; ++e)
                    x[c].x[e] = at + e < a.nodes ? logits[at + e] : static_cast<T>(-INFINITY);
            }
        }
    }
    float mine = -INFINITY;
#pragma unroll
    for (int c = 0; c < kPieces; ++c)
#pragma unroll
        for (int e = 0; e < kElems; ++e) mine = fmaxf(mine, x[c].at(e));
    const float top = wave_top(mine);
    // NaN and +inf make the sum NaN; -inf, and a row of nothing else, add 0
    const float base = fmaxf(top, -3.402823466e38f);
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < kPieces; ++c)
#pragma unroll
        for (int e = 0; e < kElems; ++e) sum += exp2_fast((x[c].at(e) - base) * kLog2e);
    sum = wave_sum(sum);

    // the width-th largest of the lanes' largest ones, by their values and lanes
    float bound = -INFINITY;
    {
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < 64; ++j) {
            const float other = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), j));
            rank += other > mine || (other == mine && j < lane);
        }
        const u64 here = __ballot(rank == a.width - 1);
        bound = __uint_as_float(
            __builtin_amdgcn_readlane(__float_as_uint(mine), here ? __ffsll(here) - 1 : 0));
    }
    u64* listed = s_listed[wave];
    int count = 0;
    u64 least = 0;  // candidates have to be above it
#pragma unroll 1
    for (int c = 0; c < kPieces; ++c) {
        Piece<T> now = x[0];
#pragma unroll
        for (int d = 1; d < kPieces; ++d)
            if (c == d) now = x[d];
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
            const float v = now.at(e);
            const u64 key = key_of(v, begin + (c * 64 + lane) * kElems + e);
            const bool in = v >= bound && v > -INFINITY && key > least;
            const u64 all = __ballot(in);
            if (!all) continue;
            if (in) listed[count + __popcll(all & ((u64{1} << lane) - 1))] = key;
            count += __popcll(all);
            if (count > kListed - 64) {  // many equal ones: the best so far, and on from there
                take_best(listed, count, s_best[wave], a.width, lane);
                if (lane < a.width) listed[lane] = s_best[wave][lane];
                count = a.width;
                least = s_best[wave][a.width - 1];
            }
        }
    }
    take_best(listed, count, s_best[wave], a.width, lane);
    if (lane == 0) {
        s_top[wave] = top;
        s_sum[wave] = sum;
    }
    __syncthreads();
    if (wave) return;
    // four lists in one
    u64* all = s_listed[0];
    for (int i = lane; i < kWaves * a.width; i += 64) all[i] = s_best[i / a.width][i % a.width];
    take_best(all, kWaves * a.width, s_joined, a.width, lane);
    const int64_t at = row * a.parts + part;
    if (lane < a.width) a.lists[at * a.width + lane] = s_joined[lane];
    if (lane == 0) {
        float m = s_top[0], l = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_top[w]);
        const float to = fmaxf(m, -3.402823466e38f);
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            l += s_sum[w] * exp2_fast((fmaxf(s_top[w], -3.402823466e38f) - to) * kLog2e);
        a.sums[at] = make_float2(to, l);
    }
}

// A group's lists become its new beams.
constexpr int kJoinBlock = 1024;

// Candidates by their values, and by beam * nodes + node where those are equal.
__device__ __forceinline__ bool before(double a, int64_t ai, double b, int64_t bi) {
    return a > b || (a == b && ai < bi);
}

__global__ __launch_bounds__(kJoinBlock) void select_join_kernel(SelectArgs a) {
    __shared__ double s_off[kMost];    // score less the log of the sum; NaN: no candidates
    __shared__ double s_value[kJoinBlock / 64];
    __shared__ int64_t s_index[kJoinBlock / 64];
    const int group = blockIdx.x, thread = threadIdx.x, lane = thread & 63, wave = thread >> 6;
    const int64_t first = static_cast<int64_t>(group) * a.beams;
    for (int b = wave; b < a.beams; b += kJoinBlock / 64) {
        const float score = a.scores[first + b];
        const bool ended = a.ended && a.ended[first + b];
        const bool is = fabsf(score) <= 3.402823466e38f;
        double off = NAN;
        if (ended) {
            if (is) off = score;
        } else if (is) {
            float m = -INFINITY;
            for (int p = lane; p < a.parts; p += 64) m = fmaxf(m, a.sums[(first + b) * a.parts + p].x);
            m = wave_top(m);
            double sum = 0.0;
            for (int p = lane; p < a.parts; p += 64) {
                const float2 part = a.sums[(first + b) * a.parts + p];
                sum += static_cast<double>(part.y) * exp2_fast((part.x - m) * kLog2e);
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
            if (sum > 0.0) off = static_cast<double>(score) - (static_cast<double>(m) + log(sum));
        }
        if (lane == 0) s_off[b] = off;
    }
    __syncthreads();
    const int each = a.parts * a.width;
    const int64_t entries = static_cast<int64_t>(a.beams) * each;
    // entry n: of beam n / each
    auto entry = [&](int64_t n, double& value, int64_t& index) {
        const int b = static_cast<int>(n / each);
        value = -INFINITY;
        index = INT64_MAX;
        const double off = s_off[b];
        if (!(fabs(off) <= 1.7e308)) return;
        if (a.ended && a.ended[first + b]) {
            if (n % each) return;
            value = off;
            index = static_cast<int64_t>(b) * a.nodes + a.end_token;
            return;
        }
        const u64 key = a.lists[first * each + n];
        if (!key) return;
        value = off + static_cast<double>(logit_of(key));
        index = static_cast<int64_t>(b) * a.nodes + node_of(key);
    };
    double last = INFINITY;
    int64_t last_index = -1;
    for (int place = 0; place < a.width; ++place) {
        double best = -INFINITY;
        int64_t best_index = INT64_MAX;
        for (int64_t n = thread; n < entries; n += kJoinBlock) {
            double value;
            int64_t index;
            entry(n, value, index);
            if (before(last, last_index, value, index) && before(value, index, best, best_index)) {
                best = value;
                best_index = index;
            }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const double value = __shfl_xor(best, o);
            const int64_t index = __shfl_xor(static_cast<long long>(best_index), o);
            if (before(value, index, best, best_index)) {
                best = value;
                best_index = index;
            }
        }
        __syncthreads();
        if (lane == 0) {
            s_value[wave] = best;
            s_index[wave] = best_index;
        }
        __syncthreads();
        best = s_value[0];
        best_index = s_index[0];
#pragma unroll
        for (int w = 1; w < kJoinBlock / 64; ++w)
            if (before(s_value[w], s_index[w], best, best_index)) {
                best = s_value[w];
                best_index = s_index[w];
            }
        if (thread == 0) {
            const int64_t at = static_cast<int64_t>(group) * a.width + place;
            const bool none = best_index == INT64_MAX;
            const int64_t parent = none ? 0 : best_index / a.nodes;
            const int64_t token = none ? max(a.end_token, int64_t{0}) : best_index % a.nodes;
            a.out_scores[at] = static_cast<float>(best);
            a.out_tokens[at] = token;
            a.out_parents[at] = parent;
            a.out_ended[at] =
                none || token == a.end_token || (a.ended && a.ended[first + parent]);
        }
        last = best;
        last_index = best_index;
    }
}

int64_t parts_of(const trw_beam_select_params& p) {
    const int64_t nodes = kWaves * 64 * kPieces * (16 / static_cast<int64_t>(element_size(p.dtype)));
    return (p.nodes + nodes - 1) / nodes;
}

// ---- reordering ----------------------------------------------------------------------------------
constexpr int kCaches = 8;  // of one launch

struct Cache {
    char *k, *v;
    uint8_t *k_scale, *v_scale;
    int64_t k_page, v_page, k_scale_page, v_scale_page;
    int row_bytes, heads;
};
struct ReorderArgs {
    Cache caches[kCaches];
    const int32_t* table;
    int64_t table_stride;
    int32_t* out_table;
    const int64_t *lens, *parents;
    int64_t* out_lens;
    float* k_times;
    int beams, table_pages, pages, shift, count, first;
};

__device__ __forceinline__ void copy_bytes(char* to, const char* from, int bytes, int thread) {
    for (int at = thread * 16; at < bytes; at += kThreads * 16)
        *reinterpret_cast<u32x4*>(to + at) = *reinterpret_cast<const u32x4*>(from + at);
}

// One child of a group, and (grid y) one head of one cache; y = 0 writes the table too.
__global__ __launch_bounds__(kThreads) void reorder_kernel(ReorderArgs a) {
    const int child = blockIdx.x % a.beams;
    const int64_t group = static_cast<int64_t>(blockIdx.x / a.beams) * a.beams;
    const int thread = threadIdx.x, lane = thread & 63;
    int parent_of = -1;  // this lane's child's
    if (lane < a.beams) {
        const int64_t p = a.parents[group + lane];
        parent_of = static_cast<int>(min(max(p, int64_t{0}), static_cast<int64_t>(a.beams - 1)));
    }
    // beams without children, and children that are not their parent's first
    uint32_t childless = 0, further = 0;
    for (int b = 0; b < a.beams; ++b) {
        const uint32_t children = static_cast<uint32_t>(__ballot(parent_of == b));
        if (!children) childless |= 1u << b;
        further |= children & (children - 1);
    }
    const int parent = __builtin_amdgcn_readlane(parent_of, child);
    const bool moves = further >> child & 1;
    int taken = parent;
    if (moves) {  // as many beams are without children as children are further ones
        uint32_t left = childless;
        for (int n = __popc(further & ((1u << child) - 1)); n; --n) left &= left - 1;
        taken = __ffs(left) - 1;
    }
    const int64_t len = a.lens[group + parent];
    const int64_t full = len > 0 ? len >> a.shift : 0;
    const int32_t* from = a.table + (group + parent) * a.table_stride;
    const int32_t* rest = a.table + (group + taken) * a.table_stride;
    if (blockIdx.y == 0 && a.first) {
        int32_t* to = a.out_table + (group + child) * a.table_pages;
        for (int p = thread; p < a.table_pages; p += kThreads) to[p] = p < full ? from[p] : rest[p];
        if (thread == 0) a.out_lens[group + child] = len;
    }
    const int rows = len > 0 ? static_cast<int>(len & ((1 << a.shift) - 1)) : 0;
    if (!moves || !rows || full >= a.table_pages) return;
    const int source = from[full], target = rest[full];
    if (source < 0 || source >= a.pages || target < 0 || target >= a.pages || source == target) return;
    if (blockIdx.y == 0 && a.first && a.k_times)
        for (int r = thread; r < rows; r += kThreads)
            a.k_times[(static_cast<int64_t>(target) << a.shift) + r] =
                a.k_times[(static_cast<int64_t>(source) << a.shift) + r];
    int head = blockIdx.y, c = 0;
    while (c < a.count && head >= a.caches[c].heads) head -= a.caches[c++].heads;
    if (c == a.count) return;
    const Cache& cache = a.caches[c];
    const int64_t line = static_cast<int64_t>(head) << a.shift;
    const int bytes = rows * cache.row_bytes;
    copy_bytes(cache.k + target * cache.k_page + line * cache.row_bytes,
               cache.k + source * cache.k_page + line * cache.row_bytes, bytes, thread);
    copy_bytes(cache.v + target * cache.v_page + line * cache.row_bytes,
               cache.v + source * cache.v_page + line * cache.row_bytes, bytes, thread);
    if (cache.k_scale)
        for (int r = thread; r < rows; r += kThreads) {
            cache.k_scale[target * cache.k_scale_page + line + r] =
                cache.k_scale[source * cache.k_scale_page + line + r];
            cache.v_scale[target * cache.v_scale_page + line + r] =
                cache.v_scale[source * cache.v_scale_page + line + r];
        }
}

}  // namespace

uint64_t beam_select_workspace(const trw_beam_select_params& p) {
    const uint64_t lists = static_cast<uint64_t>(p.groups) * p.beams * parts_of(p);
    return lists * (p.width * sizeof(u64) + sizeof(float2));
}

void beam_select(const trw_beam_select_params& p, hipStream_t stream) {
    if (p.groups == 0) return;
    require(p.workspace_bytes >= beam_select_workspace(p), "workspace is too small");
    SelectArgs a;
    a.logits = static_cast<const char*>(p.logits);
    a.group_stride = p.group_stride;
    a.beam_stride = p.beam_stride;
    a.scores = p.scores;
    a.ended = p.ended;
    a.end_token = p.end_token;
    a.groups = static_cast<int>(p.groups);
    a.beams = p.beams;
    a.width = p.width;
    a.nodes = static_cast<int>(p.nodes);
    a.parts = static_cast<int>(parts_of(p));
    a.lists = static_cast<u64*>(p.workspace);
    a.sums = reinterpret_cast<float2*>(a.lists + p.groups * p.beams * a.parts * p.width);
    a.out_scores = p.out_scores;
    a.out_tokens = p.out_tokens;
    a.out_parents = p.out_parents;
    a.out_ended = p.out_ended;
    const int64_t grid = p.groups * p.beams * a.parts;
    require_grid(grid, kThreads);
    require_grid(p.groups, kJoinBlock);
    by_type(p.dtype, [&](auto t) {
        hipLaunchKernelGGL((select_rows_kernel<decltype(t)>), dim3(static_cast<unsigned>(grid)),
                           dim3(kThreads), 0, stream, a);
    });
    check_launch("beam_select");
    hipLaunchKernelGGL(select_join_kernel, dim3(static_cast<unsigned>(p.groups)), dim3(kJoinBlock), 0,
                       stream, a);
    check_launch("beam_select");
}

void beam_reorder(const trw_beam_reorder_params& p, hipStream_t stream) {
    if (p.groups == 0) return;
    ReorderArgs a;
    a.table = p.table;
    a.table_stride = p.table_stride;
    a.out_table = p.out_table;
    a.lens = p.lens;
    a.parents = p.parents;
    a.out_lens = p.out_lens;
    a.k_times = p.k_times;
    a.beams = p.beams;
    a.table_pages = static_cast<int>(p.table_pages);
    a.pages = static_cast<int>(p.pages);
    a.shift = 0;
    while ((1 << a.shift) < p.page_rows) ++a.shift;
    const int64_t rows = p.groups * p.beams;
    int done = 0;
    do {
        a.count = std::min(kCaches, p.count - done);
        a.first = done == 0;
        int heads = 0;
        for (int c = 0; c < a.count; ++c) {
            const trw_pages& from = p.caches[done + c];
            const Pages pages = make_pages(from);
            a.caches[c] = Cache{pages.k, pages.v, pages.k_scale, pages.v_scale, pages.k_page,
                                pages.v_page, pages.k_scale_page, pages.v_scale_page,
                                static_cast<int>(from.dim * page_element_size(from.dtype)),
                                from.kv_heads};
            heads += from.kv_heads;
        }
        require_grid(rows * std::max(heads, 1), kThreads);
        hipLaunchKernelGGL(reorder_kernel, dim3(static_cast<unsigned>(rows), std::max(heads, 1)),
                           dim3(kThreads), 0, stream, a);
        check_launch("beam_reorder");
        done += a.count;
    } while (done < p.count);
}

}  // namespace ops
}  // namespace trw
