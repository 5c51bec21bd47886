// attention_step.hip -- one new event of each walk over its cache.
//
// Per walk and key head: read the cache once, at memory speed.  The query
// heads that share a key head are the columns of the products (up to 32 of
// them; the matrix instructions are idle most of the time either way), a wave
// takes blocks of 32 positions, and four waves and, where walks are few, many
// workgroups share a walk: each keeps a maximum, a sum and an output of its
// own, joined at the end.  Positions past the walk's length are never read.
//
// The new key and value are taken from the call's arguments, not from the
// cache, by the workgroup whose positions include them, and written to the
// cache by the walk's first workgroup: no launch and no wait between the two.
//
// 64 walks of up to 4095 events (32 heads of 128 over 8 key heads, bfloat16) take
// 123 us, 4.5 TB/s of cache; a large copy reaches 4.9, a sum 3.8.
#include <algorithm>

#include "operators.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kKeys = 32;  // positions of a wave's block

struct StepArgs {
    Rows q, k, v, out;
    char *k_cache, *v_cache;
    int64_t k_batch, k_pos, k_head, v_batch, v_pos, v_head;
    const int64_t* lens;
    float* k_times;
    Score score;
    int64_t capacity;
    int batch, heads, kv_heads, group, columns, dim, splits;
    float* partial;  // [batch, heads, splits, dim]
    float2* part_stats;  // [batch, heads, splits]
};

// All but this wave's last kLater copies to LDS have landed.
template <int kLater>
__device__ __forceinline__ void copies_landed() {
    static_assert(kLater < 64, "counted in six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70 | (kLater & 15) | (kLater >> 4 << 14));
    asm volatile("" ::: "memory");
}

// The call's own row, in every row of a tile from `from` on.
template <typename T, int DB>
__device__ __forceinline__ void put_row(u32x4* tile, const T* row, int from, int dim, int lane) {
    typedef Tile<T, DB> G;
    for (int n = from * G::kUsed + lane; n < kKeys * G::kUsed; n += 64) {
        const int col = n % G::kUsed * G::kElems;
        tile[G::slot(n / G::kUsed, n % G::kUsed)] =
            col < dim ? *reinterpret_cast<const u32x4*>(row + col) : u32x4{0, 0, 0, 0};
    }
}

// Two workgroups a compute unit where their tiles (66 KB at head size 128 in 16
// bits) leave room: left to itself the compiler takes 298 registers there, one
// workgroup, and 238 walks of 350 events (8 heads of 128, bfloat16) take 113 us
// for 83 (4.1 TB/s).
template <typename T, int DB, bool kWide>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 || DB <= 2 ? 2 : 1)
void attention_step_kernel(StepArgs a) {
    typedef Tile<T, DB> G;
    constexpr size_t kTileBytes = G::bytes(kKeys);
    constexpr size_t kJoinBytes = kWaves * 32 * 33 * sizeof(float);
    constexpr size_t kBytes =
        2 * kWaves * kTileBytes > kJoinBytes ? 2 * kWaves * kTileBytes : kJoinBytes;
    __shared__ u32x4 s_mem[kBytes / 16];
    __shared__ float s_m[kWaves][32], s_l[kWaves][32], s_times[kWaves][64];

    // Consecutive workgroups go to the eight XCDs in turn: each takes all key
    // heads of some positions, which lie side by side.
    int rest = blockIdx.x / 8;
    const int col_group = rest % a.columns;
    rest /= a.columns;
    const int kv_head = rest % a.kv_heads;
    const int item = rest / a.kv_heads * 8 + blockIdx.x % 8;
    const int split = item % a.splits;
    const int b = item / a.splits;
    if (b >= a.batch) return;
    const int thread = threadIdx.x, lane = thread & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const Score& sc = a.score;

    const int64_t n = a.lens[b];  // position of the new event
    const bool idle = n < 0 || n >= a.capacity;
    const int col = col_group * 32 + (lane & 31);
    const int head = kv_head * a.group + col;
    const bool any = !idle && col < a.group;
    const T* fresh_k = row_of<const T>(a.k, b, kv_head);
    const T* fresh_v = row_of<const T>(a.v, b, kv_head);
    T* cache_k = reinterpret_cast<T*>(a.k_cache) + b * a.k_batch + kv_head * a.k_head;
    T* cache_v = reinterpret_cast<T*>(a.v_cache) + b * a.v_batch + kv_head * a.v_head;
    const float q_time = sc.q_times ? sc.q_times[b] : 0.0f;

    if (!idle && split == 0 && col_group == 0) {
        constexpr int kElems = G::kElems;
        const int at = thread * kElems;
        if (at < a.dim) {
            *reinterpret_cast<u32x4*>(cache_k + n * a.k_pos + at) =
                *reinterpret_cast<const u32x4*>(fresh_k + at);
            *reinterpret_cast<u32x4*>(cache_v + n * a.v_pos + at) =
                *reinterpret_cast<const u32x4*>(fresh_v + at);
        }
        if (a.k_times && kv_head == 0 && thread == 0) a.k_times[b * a.capacity + n] = q_time;
    }

    // this workgroup's blocks of positions
    const int64_t blocks = idle ? 0 : n / kKeys + 1;
    const int64_t block_begin = blocks * split / a.splits;
    const int64_t block_end = blocks * (split + 1) / a.splits;

    Frag<T> q[G::kSteps];
    load_operand<T, DB>(q, row_of<const T>(a.q, b, any ? head : 0), any, a.dim, half);
    const float slope = sc.slopes && any ? sc.slopes[head] * kLog2e : 0.0f;
    const float far_bias = sc.table && any ? table_entry(sc, head, 2 * sc.reach) : 0.0f;
    const float* k_times = sc.k_times ? sc.k_times + b * a.capacity : nullptr;

    f32x16 o[DB];
#pragma unroll
    for (int c = 0; c < DB; ++c) o[c] = zero16();
    float m = kFloor, l = 0.0f;
    // The wave's tile of keys and of values.  The next keys are on their way
    // while this block's softmax and values are worked on, the next values
    // while the next scores are: each is waited for by the number of copies
    // asked for after it.
    u32x4* s_k = s_mem + wave * 2 * (kTileBytes / 16);
    u32x4* s_v = s_k + kTileBytes / 16;
    const uint32_t at_k = lds_address(s_mem) + wave * 2 * kTileBytes;
    const Loader<T, DB, kKeys, 64> k_load(a.k_pos, a.dim, lane), v_load(a.v_pos, a.dim, lane);
    constexpr int kCopies = Loader<T, DB, kKeys, 64>::kMine;
    const int length = static_cast<int>(n);  // rows of the cache
    auto fetch_k = [&](int j) {
        k_load.load(cache_k, j, 0, length, at_k, lane);
        if (k_times) load_floats(k_times, j, 0, length, lds_address(s_times) + wave * 256, lane);
    };
    auto fetch_v = [&](int j) { v_load.load(cache_v, j, 0, length, at_k + kTileBytes, lane); };
    int block = static_cast<int>(block_begin) + wave;
    if (block < block_end && block * kKeys < length) {
        fetch_k(block * kKeys);
        fetch_v(block * kKeys);
    }
#pragma unroll 1
    for (; block < block_end; block += kWaves) {
        const int j0 = block * kKeys;
        const int j1 = j0 + kWaves * kKeys;
        const bool more = block + kWaves < block_end && j1 < length;
        int at_lane = lane;  // LDS addresses are not held over the loop
        asm volatile("" : "+v"(at_lane));
        copies_landed<kCopies>();  // keys; the values, asked for last, may be on their way
        if (j0 + kKeys > length) {
            copies_landed<0>();
            put_row<T, DB>(s_k, fresh_k, length - j0, a.dim, at_lane);
            put_row<T, DB>(s_v, fresh_v, length - j0, a.dim, at_lane);
        }
        f32x16 x = zero16();
#pragma unroll
        for (int st = 0; st < G::kSteps; ++st)
            x = mma(G::row(s_k, at_lane & 31, st, at_lane >> 5), q[st], x);
        float s[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float unused;
            s[r] = sc.softcap > 0 ? capped<T, kWide>(sc, x[r], unused) : x[r] * sc.scale2;
        }
        float time[16];
        if (k_times) {
#pragma unroll
            for (int r = 0; r < 16; ++r) time[r] = s_times[wave][acc_row(r) + 4 * half];
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): read, so the next keys may come
        if (more) fetch_k(j1);
        // distances from the new event of register r's position: last_d - acc_row(r)
        const int last_d = length - j0 - 4 * half;
        if (sc.table) {
            if (length - (j0 + kKeys - 1) >= sc.reach) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] += far_bias;
            } else if (any) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = min(max(last_d - acc_row(r), 0), sc.reach);
                    s[r] += table_entry(sc, head, d + sc.reach);
                }
            }
        }
        if (sc.slopes) {
            if (k_times) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    // the new event's own time is not in the cache yet: it is 0 away
                    const float gap = q_time - time[r];
                    s[r] = fmaf(-slope, last_d == acc_row(r) ? 0.0f : fabsf(gap), s[r]);
                }
            } else {
                const float from = static_cast<float>(last_d);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = fmaf(-slope, fabsf(from - acc_row(r)), s[r]);
            }
        }
        if (j0 + kKeys > length + 1) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (acc_row(r) > last_d) s[r] = -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any(top > m)) {
            const float grown = fmaxf(m, top);
            const float by = exp2_fast(m - grown);
            m = grown;
            l *= by;
#pragma unroll
            for (int c = 0; c < DB; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[c][r] *= by;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2_fast(s[r] - m);
            l += s[r];
        }
        if (more) copies_landed<kCopies>();  // values; the next keys may be on their way
        else copies_landed<0>();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            Frag<T> p;
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = static_cast<T>(s[8 * t + e]);
#pragma unroll
            for (int c = 0; c < DB; ++c) o[c] = mma(G::columns(s_v, 16 * t, c, at_lane), p, o[c]);
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        if (more) fetch_v(j1);
    }
    l += __shfl_xor(l, 32);

    // join the waves
    if (half == 0) {
        s_m[wave][lane] = m;
        s_l[wave][lane] = l;
    }
    __syncthreads();  // also: the tiles are done with
    float* s_join = reinterpret_cast<float*>(s_mem);
    const int jc = thread >> 3, jd = (thread & 7) * 4;  // a column and four of its elements
    float top = s_m[0][jc], by[kWaves], total = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_m[w][jc]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        by[w] = exp2_fast(s_m[w][jc] - top);
        total += by[w] * s_l[w][jc];
    }
    const int join_col = col_group * 32 + jc;
    const int join_head = kv_head * a.group + join_col;
    const int64_t part = (static_cast<int64_t>(b) * a.heads + join_head) * a.splits + split;
    const float scale = a.splits > 1 ? 1.0f : 1.0f / total;
#pragma unroll
    for (int c = 0; c < DB; ++c) {
        if (c) __syncthreads();
#pragma unroll
        for (int r = 0; r < 16; ++r)
            s_join[(wave * 32 + (lane & 31)) * 33 + acc_row(r) + 4 * half] = o[c][r];
        __syncthreads();
        const int d = 32 * c + jd;
        if (join_col < a.group && d < a.dim) {
            f32x4 sum = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sum[e] = fmaf(by[w], s_join[(w * 32 + jc) * 33 + jd + e], sum[e]);
            if (a.splits > 1) {
                *reinterpret_cast<f32x4*>(a.partial + part * a.dim + d) = sum;
            } else {
                typedef T t4 __attribute__((ext_vector_type(4)));
                t4 out;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // a total of 0: the bias masks every position
                    const float value =
                        n < 0 ? 0.0f : idle ? NAN : total != 0.0f ? sum[e] * scale : 0.0f;
                    out[e] = static_cast<T>(value);
                }
                *reinterpret_cast<t4*>(row_of<T>(a.out, b, join_head) + d) = out;
            }
        }
    }
    if (a.splits > 1 && jd == 0 && join_col < a.group)
        a.part_stats[part] = make_float2(top, total);
}

// Joins the workgroups of one walk and head: 32 threads for the elements, four
// each, and eight shares of the workgroups.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_step_kernel(StepArgs a) {
    __shared__ f32x4 s_sum[8][32];
    __shared__ float s_total[8], s_top[4];
    const int head = blockIdx.x % a.heads;
    const int b = blockIdx.x / a.heads;
    const int thread = threadIdx.x, share = thread >> 5, d = (thread & 31) * 4;
    const int64_t part = (static_cast<int64_t>(b) * a.heads + head) * a.splits;
    float top = kFloor;
    for (int s = thread; s < a.splits; s += kThreads) top = fmaxf(top, a.part_stats[part + s].x);
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
    const int64_t n = a.lens[b];
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        out[e] = static_cast<T>(n < 0              ? 0.0f
                                : n >= a.capacity  ? NAN
                                : total != 0.0f    ? sum[e] / total
                                                   : 0.0f);
    *reinterpret_cast<t4*>(row_of<T>(a.out, b, head) + d) = out;
}

// Workgroups of one walk and key head: each with at least four blocks a wave
// where the cache is full.  Few walks: 1536 in all (768 where heads are large and
// fewer fit), two or three times what the compute units hold, and no more, since
// each has a sum to join: 3 histories of 100k events (2 key heads of 128) take 59
// us with 768 and 66 with 1536, 50 walks of up to 58k (4 of 16) 228 with 1536 and
// 334 with 512.  More walks: three each up to 3072 in all, which evens out their
// lengths: 64 walks of up to 4k events (8 of 128) take 121 us with three each,
// 131 with two.
int splits_of(const trw_attention_step_params& p) {
    const int group = p.heads / p.kv_heads;
    const int64_t items = p.batch * p.kv_heads * ((group + 31) / 32);
    const int64_t most = (p.capacity + 4 * kWaves * kKeys - 1) / (4 * kWaves * kKeys);
    const int64_t enough = p.dim > 64 ? 768 : 1536, n = std::max<int64_t>(items, 1);
    const int64_t want = std::max((enough + n - 1) / n, std::min<int64_t>(3, 3072 / n));
    return static_cast<int>(std::max<int64_t>(1, std::min(want, most)));
}

}  // namespace

uint64_t attention_step_workspace(const trw_attention_step_params& p) {
    const int splits = splits_of(p);
    if (splits == 1) return 0;
    return static_cast<uint64_t>(p.batch) * p.heads * splits * (p.dim + 2) * sizeof(float);
}

void attention_step(const trw_attention_step_params& p, hipStream_t stream) {
    if (p.batch == 0) return;
    require(p.workspace_bytes >= attention_step_workspace(p), "workspace is too small");
    StepArgs a;
    a.q = make_rows(p.q);
    a.k = make_rows(p.k);
    a.v = make_rows(p.v);
    a.out = make_rows(p.out);
    a.k_cache = static_cast<char*>(p.k_cache);
    a.v_cache = static_cast<char*>(p.v_cache);
    a.k_batch = p.k_batch_stride;
    a.k_pos = p.k_pos_stride;
    a.k_head = p.k_head_stride;
    a.v_batch = p.v_batch_stride;
    a.v_pos = p.v_pos_stride;
    a.v_head = p.v_head_stride;
    a.lens = p.lens;
    a.k_times = const_cast<float*>(p.score.k_times);
    a.score = make_score(p.score);
    a.capacity = p.capacity;
    a.batch = static_cast<int>(p.batch);
    a.heads = p.heads;
    a.kv_heads = p.kv_heads;
    a.group = p.heads / p.kv_heads;
    a.columns = (a.group + 31) / 32;
    a.dim = p.dim;
    a.splits = splits_of(p);
    a.partial = static_cast<float*>(p.workspace);
    a.part_stats = reinterpret_cast<float2*>(a.partial + static_cast<int64_t>(p.batch) * p.heads *
                                                             a.splits * p.dim);
    const int64_t grid = xcd_grid(p.batch * a.splits) * p.kv_heads * a.columns;
    require_grid(grid, kThreads);
    dispatch(p.dtype, p.dim, [&](auto t, auto db) {
        typedef decltype(t) T;
        by_cap<T>(p.dtype, p.score, [&](auto wide) {
            hipLaunchKernelGGL(
                (attention_step_kernel<T, decltype(db)::value, decltype(wide)::value>),
                dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, a);
        });
        check_launch("attention_step");
        if (a.splits > 1)
            hipLaunchKernelGGL((join_step_kernel<T>), dim3(static_cast<unsigned>(a.batch * a.heads)),
                               dim3(kThreads), 0, stream, a);
        check_launch("attention_step");
    });
}

}  // namespace ops
}  // namespace trw
