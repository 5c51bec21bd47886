// attention.hip -- attention of query rows over intervals of key rows, forward.
//
//   s_ij = cap(scale q_i . k_j) + bias(i, j),   o_i = sum_j softmax_j(s_ij) v_j
//
// One pass over the keys with a running maximum m and sum l per row: when m
// grows to m', what was summed is scaled by exp2(m - m').  A workgroup of four
// waves takes 128 rows of one head, 32 a wave; tiles of keys and values go
// through LDS, the next one loading into registers beside the products of this
// one.  Rows of several walks share a workgroup (walks are short), so a tile's
// keys are the union of its rows' intervals, each wave skips the tiles that
// none of its rows sees, and only tiles at an interval's end pay for the
// masking.
//
// Scores, maxima, sums and the output accumulate in float32; P is rounded to
// the inputs' type for the product with V (as the matrix instructions take
// it), the sum l is of the unrounded values.
//
// Arithmetic per pair (exponential, bias, conversion) and matrix products, and
// the waits between them: 16384 rows in one causal walk (16 heads of 128 over 4 key
// heads, a bias by distance, bfloat16) take 1.32 to 1.35 ms, 816 to 833 TFLOP/s, with
// the vector units busy 0.63 of the time and the matrix units 0.35; a large library
// product reaches 1260.  Tiles that reach LDS past the registers, two at a time, and
// tiles of few rows sharing long keys took it from 3.3 ms.  23 walks of up to 1999
// rows (8 heads of 80, capped scores with a bias, float16) take 170 us (0.47 and
// 0.14 busy).
#include <algorithm>

#include "operators.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerWave = 32;
constexpr int kTileRows = 128;

// A running maximum is raised once a score passes it by this much (base 2):
// P is then at most 2^8, which every type holds as well as 1, and the output is
// rarely scaled.
constexpr float kSlack = 8.0f;
// Keys that a workgroup takes at least, where several share a tile's.
constexpr int kShare = 512;

struct ForwardArgs {
    Rows q, k, v, out, out_low;
    const int4* q_info;
    float* stats;
    Score score;
    int q_rows, k_rows, heads, group, dim;
    int tiles, splits;
    int walk_limit;      // documents up to here go a wave each (attention_walks.hip)
    // where splits > 1
    float* part_out;     // [splits, heads, q_rows, dim]
    float2* part_stats;  // [splits, heads, q_rows]
    int* part_count;     // [tiles] workgroups that a tile's keys were shared by
};

// What the backward pass takes from a score to have log2 P: m + log2 l at once,
// or in two where a bias can make scores so low that log2 l would be lost in
// the sum.
__device__ __forceinline__ void store_stats(const ForwardArgs& a, int64_t stat, bool seen, float m,
                                            float l) {
    if (!a.stats) return;
    const float log_l = seen ? __builtin_amdgcn_logf(l) : INFINITY;
    const bool apart = a.score.biased();
    a.stats[stat] = apart ? m : m + log_l;
    if (apart) a.stats[static_cast<int64_t>(a.heads) * a.q_rows + stat] = log_l;
}

template <typename T, int DB, bool kWide>
__global__ __launch_bounds__(kThreads, 2) void attention_forward_kernel(ForwardArgs a) {
    typedef Tile<T, DB> G;
    constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;  // of a tile
    constexpr int kBlocks = kKeys / 32;
    constexpr int kTileChunks = kKeys * G::kSlots;
    __shared__ u32x4 s_kv[2][2][kTileChunks];  // two tiles of keys and values
    __shared__ float s_times[2][64];
    __shared__ int s_reduce[4][4];
    extern __shared__ float s_lut[];

    const int64_t items = static_cast<int64_t>(a.tiles) * a.heads * a.splits;
    const int64_t item = xcd_item(blockIdx.x, items);
    if (item >= items) return;
    const int split = static_cast<int>(item % a.splits);
    const int head = static_cast<int>(item / a.splits / a.tiles);
    // the last rows of a causal walk see most: first
    const int tile = a.tiles - 1 - static_cast<int>(item / a.splits % a.tiles);
    const int kv_head = head / a.group;
    const int thread = threadIdx.x, lane = thread & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const Score& sc = a.score;

    const int i = tile * kTileRows + wave * kRowsPerWave + (lane & 31);
    int4 info = {0, 0, 0, 0};
    if (i < a.q_rows) info = a.q_info[i];
    const bool tiled_row = i < a.q_rows && tiled(info.w, a.walk_limit);
    if (!__syncthreads_or(tiled_row)) return;
    int lo = info.x, hi = tiled_row ? max(info.x, min(info.y, a.k_rows)) : info.x;
    const int diag = info.z;
    const bool any = lo < hi;

    Frag<T> q[G::kSteps];
    load_operand<T, DB>(q, row_of<const T>(a.q, i, head), any, a.dim, half);

    // the wave's and the workgroup's intervals
    int w_lo = wave_min(any ? lo : kNone), w_hi = wave_max(any ? hi : 0);
    const int w_diag_lo = wave_min(any ? diag : kNone), w_diag_hi = wave_max(any ? diag : -kNone);
    const int w_last_lo = wave_max(any ? lo : 0);
    if (lane == 0) {
        s_reduce[wave][0] = w_lo;
        s_reduce[wave][1] = w_hi;
        s_reduce[wave][2] = w_last_lo;
    }
    if (sc.table) fill_bias(s_lut, sc, head, thread, kThreads);
    __syncthreads();
    int k_begin = kNone, k_end = 0, last_lo = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        k_begin = min(k_begin, s_reduce[w][0]);
        k_end = max(k_end, s_reduce[w][1]);
        last_lo = max(last_lo, s_reduce[w][2]);
    }
    k_begin = __builtin_amdgcn_readfirstlane(k_begin);
    k_end = __builtin_amdgcn_readfirstlane(k_end);
    const bool mixed = k_begin < last_lo;  // rows of more than one walk
    // this split's tiles of the workgroup's keys: as many splits as have kShare
    // tiles each
    int j_first = k_begin, j_last = k_end;
    bool shared = false;
    if (a.splits > 1) {
        const int count = k_begin < k_end ? (k_end - k_begin + kKeys - 1) / kKeys : 0;
        const int used = min(a.splits, max((count * kKeys + kShare - 1) / kShare, 1));
        if (split >= used) return;
        if (split == 0 && head == 0 && thread == 0) a.part_count[tile] = used;
        shared = used > 1;
        if (shared) {
            j_first = k_begin + static_cast<int>(static_cast<int64_t>(count) * split / used) * kKeys;
            j_last = min(k_end, k_begin + static_cast<int>(static_cast<int64_t>(count) *
                                                           (split + 1) / used) * kKeys);
        }
    }

    const float slope = sc.slopes ? sc.slopes[head] * kLog2e : 0.0f;
    const float q_time = sc.q_times && any ? sc.q_times[i] : 0.0f;
    const T* k_base = row_of<const T>(a.k, 0, kv_head);
    const T* v_base = row_of<const T>(a.v, 0, kv_head);
    const uint32_t at_kv = lds_address(s_kv), at_times = lds_address(s_times);
    const Loader<T, DB, kKeys, kThreads> k_load(a.k.row, a.dim, thread);
    const Loader<T, DB, kKeys, kThreads> v_load(a.v.row, a.dim, thread);
    // Scores that are only products are scaled inside the exponential
    const bool plain = !sc.biased() && !(sc.softcap > 0) && sc.scale2 > 0;
    const float in_exp = plain ? sc.scale2 : 1.0f;

    const int j_begin = j_first, j_end = j_last;

    int only = -1;  // -1: every row; else the rows whose keys begin there, again
    for (;;) {
        f32x16 o[DB];
#pragma unroll
        for (int b = 0; b < DB; ++b) o[b] = zero16();
        float m = kFloor, l = 0.0f;
        // Every row must be inside a tile for it to go unmasked
        const int full_lo = wave_max(any ? lo : kNone), full_hi = wave_min(any ? hi : 0);

        auto fetch = [&](int j0, int buffer) {
            k_load.load(k_base, j0, k_begin, k_end, at_kv + buffer * 2 * kTileChunks * 16, thread);
            v_load.load(v_base, j0, k_begin, k_end, at_kv + (buffer * 2 + 1) * kTileChunks * 16, thread);
            if (sc.k_times && wave == 0)
                load_floats(sc.k_times, j0, k_begin, k_end, at_times + buffer * 256, lane);
        };
        int buffer = 0;
        if (j_first < j_last) fetch(j_first, 0);
        for (int j0 = j_first; j0 < j_last; j0 += kKeys, buffer ^= 1) {
            landed();  // and the other buffer is done with
            if (j0 + kKeys < j_last) fetch(j0 + kKeys, buffer ^ 1);
            if (j0 >= w_hi || j0 + kKeys <= w_lo) continue;
            const u32x4* s_k = s_kv[buffer][0];
            const u32x4* s_v = s_kv[buffer][1];
            const float* s_time = s_times[buffer];
            float s[kBlocks][16];
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                f32x16 x = zero16();
#pragma unroll
                for (int st = 0; st < G::kSteps; ++st)
                    x = mma(G::row(s_k, 32 * b + (lane & 31), st, half), q[st], x);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] = x[r];
            }
            const int j_lane = j0 + 4 * half;  // register r's key: + 32 b + acc_row(r)
            if (!plain) {
                cap_scores<T, kWide>(sc, s);
                add_biases(sc, s, s_lut, slope, diag, w_diag_lo, w_diag_hi, q_time, s_time, j0, half);
            }
            if (j0 < full_lo || j0 + kKeys > full_hi) {
                const unsigned span = static_cast<unsigned>(hi - lo);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = j_lane + 32 * b + acc_row(r);
                        if (static_cast<unsigned>(j - lo) >= span) s[b][r] = -INFINITY;
                    }
            }
            float top = s[0][0];
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
            top = fmaxf(top, __shfl_xor(top, 32)) * in_exp;
            if (__any(top > m + kSlack)) {
                // by its own scores alone: a row's bits do not depend on its neighbours
                const float grown = top > m + kSlack ? top : m;
                const float by = exp2_fast(m - grown);
                m = grown;
                l *= by;
#pragma unroll
                for (int b = 0; b < DB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[b][r] *= by;
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[b][r] = exp2_fast(fmaf(s[b][r], in_exp, -m));
                    l += s[b][r];
                }
            }
#pragma unroll
            for (int t = 0; t < 2 * kBlocks; ++t) {
                Frag<T> p;
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = static_cast<T>(s[t >> 1][8 * (t & 1) + e]);
#pragma unroll
                for (int b = 0; b < DB; ++b) o[b] = mma(G::columns(s_v, 16 * t, b, lane), p, o[b]);
            }
        }

        l += __shfl_xor(l, 32);
        const bool mine = tiled_row && (only < 0 || (any && info.x == only));
        if (mine) {
            const bool seen = any && l != 0.0f;  // 0: the bias masks every key
            const int64_t stat = static_cast<int64_t>(head) * a.q_rows + i;
            if (shared) {
                const int64_t part = static_cast<int64_t>(split) * a.heads * a.q_rows + stat;
                store_row<float, DB>(a.part_out + part * a.dim, o, seen, 1.0f, a.dim, half);
                if (half == 0) a.part_stats[part] = make_float2(m, seen ? l : 0.0f);
            } else {
                store_row<T, DB>(row_of<T>(a.out, i, head), o, seen, 1.0f / l, a.dim, half,
                                 a.out_low.data ? row_of<T>(a.out_low, i, head) : nullptr);
                if (half == 0) store_stats(a, stat, seen, m, l);
            }
        }
        if (!mixed) break;

        // Walks share this workgroup's tiles, and 0 times the infinity or NaN
        // of one walk's value would reach the rows of another.  Where that
        // happened, the rows of each walk in turn go once more over keys that
        // are theirs alone: what is not finite stays in its walk.
        bool off = false;
        if (any && info.x > only) {
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += o[b][r] * 0.0f;
            off = only < 0 ? sum != 0.0f : true;
        }
        if (only < 0 && !__syncthreads_or(off)) break;
        int w_next = wave_min(any && info.x > only ? info.x : kNone);
        __syncthreads();
        if (lane == 0) s_reduce[wave][0] = w_next;
        __syncthreads();
        int seg = kNone;
#pragma unroll
        for (int w = 0; w < 4; ++w) seg = min(seg, s_reduce[w][0]);
        if (seg == kNone) break;
        only = seg;
        const bool in_seg = any && info.x == only;
        lo = in_seg ? info.x : 0;
        hi = in_seg ? max(info.x, min(info.y, a.k_rows)) : 0;
        w_lo = wave_min(in_seg ? lo : kNone);
        w_hi = wave_max(in_seg ? hi : 0);
        if (lane == 0) s_reduce[wave][1] = w_hi;
        __syncthreads();
        k_begin = only;
        k_end = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) k_end = max(k_end, s_reduce[w][1]);
        k_begin = __builtin_amdgcn_readfirstlane(k_begin);
        k_end = __builtin_amdgcn_readfirstlane(k_end);
        // the same tiles: the same bits
        j_first = j_begin + max(k_begin - j_begin, 0) / kKeys * kKeys;
        j_last = min(j_end, k_end);
    }
}

// Joins the splits of a row: four elements a thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_forward_kernel(ForwardArgs a) {
    const int64_t t = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
    const int pieces = a.dim / 4;
    const int64_t rows = static_cast<int64_t>(a.heads) * a.q_rows;
    if (t >= rows * pieces) return;
    const int64_t stat = t / pieces;  // head, row
    const int count = a.part_count[stat % a.q_rows / kTileRows];
    if (count == 1) return;  // written by its one workgroup
    const int col = static_cast<int>(t % pieces) * 4;
    float m = kFloor;
    for (int s = 0; s < count; ++s) {
        const float2 st = a.part_stats[s * rows + stat];
        m = st.y != 0.0f ? fmaxf(m, st.x) : m;
    }
    f32x4 o = {0, 0, 0, 0};
    float l = 0.0f;
    for (int s = 0; s < count; ++s) {
        const float2 st = a.part_stats[s * rows + stat];
        if (st.y == 0.0f) continue;
        const float by = exp2_fast(st.x - m);
        const f32x4 part = *reinterpret_cast<const f32x4*>(a.part_out + (s * rows + stat) * a.dim + col);
        l = fmaf(by, st.y, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(by, part[e], o[e]);
    }
    const bool seen = l != 0.0f;
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 out, low;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x = seen ? o[e] / l : 0.0f;
        out[e] = static_cast<T>(x);
        low[e] = static_cast<T>(x - static_cast<float>(out[e]));
    }
    const int head = static_cast<int>(stat / a.q_rows);
    *reinterpret_cast<t4*>(row_of<T>(a.out, stat % a.q_rows, head) + col) = out;
    if (a.out_low.data)
        *reinterpret_cast<t4*>(row_of<T>(a.out_low, stat % a.q_rows, head) + col) = low;
    if (col == 0) store_stats(a, stat, seen, m, l);
}

// Workgroups that may share one tile's keys: where tiles and heads are no more
// than two workgroups for each of the 256 compute units, enough for eight, for
// each tile as its keys (which the device knows) allow.
int splits_of(const trw_attention_params& p) {
    const int64_t items = (p.q_rows + kTileRows - 1) / kTileRows * p.heads;
    if (items == 0 || items > 512 || walk_blocks(p)) return 1;
    const int64_t splits = std::min<int64_t>({2048 / items, p.k_rows / kShare, 32});
    return static_cast<int>(std::max<int64_t>(splits, 1));
}

}  // namespace

uint64_t attention_backward_workspace(const trw_attention_params& p);

uint64_t attention_workspace(const trw_attention_params& p, bool backward) {
    if (backward) return attention_backward_workspace(p);
    const int splits = splits_of(p);
    if (splits == 1) return 0;
    return static_cast<uint64_t>(splits) * p.heads * p.q_rows * (p.dim + 2) * sizeof(float) +
           (p.q_rows + kTileRows - 1) / kTileRows * sizeof(int);
}

// Tiles' workgroups are shared between several only where they are few, so that
// this holds for all their launches; of the walks' the backward pass has a wave
// for each block.
void require_grids(const trw_attention_params& p, bool backward) {
    const int blocks = walk_blocks(p);
    if (blocks) require_grid(walk_grid(p), 64 * (backward ? blocks : 1));
    if (blocks && !walk_rest(p, blocks)) return;
    const auto tiles = [](int64_t rows) { return (rows + kTileRows - 1) / kTileRows; };
    require_grid(xcd_grid(tiles(p.q_rows) * p.heads), kThreads);
    if (backward) require_grid(xcd_grid(tiles(p.k_rows) * p.kv_heads), kThreads);
}

void attention_forward(const trw_attention_params& p, hipStream_t stream) {
    if (p.q_rows == 0) return;
    require(p.workspace_bytes >= attention_workspace(p, false), "workspace is too small");
    const int blocks = walk_blocks(p);
    if (blocks) {
        walk_forward(p, blocks, stream);
        if (!walk_rest(p, blocks)) return;
    }
    ForwardArgs a;
    a.walk_limit = 32 * blocks;
    a.q = make_rows(p.q);
    a.k = make_rows(p.k);
    a.v = make_rows(p.v);
    a.out = make_rows(p.out);
    a.out_low = make_rows(p.out_low);
    a.q_info = reinterpret_cast<const int4*>(p.q_rows_info);
    a.stats = p.stats;
    a.score = make_score(p.score);
    a.q_rows = static_cast<int>(p.q_rows);
    a.k_rows = static_cast<int>(p.k_rows);
    a.heads = p.heads;
    a.group = p.heads / p.kv_heads;
    a.dim = p.dim;
    a.tiles = static_cast<int>((p.q_rows + kTileRows - 1) / kTileRows);
    a.splits = splits_of(p);
    const int64_t rows = static_cast<int64_t>(a.heads) * a.q_rows;
    a.part_out = static_cast<float*>(p.workspace);
    a.part_stats = reinterpret_cast<float2*>(a.part_out + a.splits * rows * a.dim);
    a.part_count = reinterpret_cast<int*>(a.part_stats + a.splits * rows);
    const int64_t grid = xcd_grid(static_cast<int64_t>(a.tiles) * a.heads * a.splits);
    const size_t lds = p.score.table ? (2 * a.score.reach + 1) * sizeof(float) : 0;
    dispatch(p.dtype, p.dim, [&](auto t, auto db) {
        by_cap<decltype(t)>(p.dtype, p.score, [&](auto wide) {
            hipLaunchKernelGGL(
                (attention_forward_kernel<decltype(t), decltype(db)::value, decltype(wide)::value>),
                dim3(static_cast<unsigned>(grid)), dim3(kThreads), lds, stream, a);
        });
        check_launch("attention_forward");
        if (a.splits > 1) {
            const int64_t threads = rows * (a.dim / 4);
            hipLaunchKernelGGL((join_forward_kernel<decltype(t)>),
                               dim3(static_cast<unsigned>((threads + kThreads - 1) / kThreads)),
                               dim3(kThreads), 0, stream, a);
            check_launch("attention_forward");
        }
    });
}

}  // namespace ops
}  // namespace trw
