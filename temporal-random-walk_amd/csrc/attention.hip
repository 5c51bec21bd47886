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
#include "operators.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerWave = 32;
constexpr int kTileRows = 128;

struct ForwardArgs {
    Rows q, k, v, out;
    const int4* q_info;
    float2* stats;
    Score score;
    int q_rows, k_rows, heads, group, dim;
    int tiles;
};

template <typename T, int DB>
__global__ __launch_bounds__(kThreads) void attention_forward_kernel(ForwardArgs a) {
    typedef Tile<T, DB> G;
    constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;  // of a tile
    constexpr int kBlocks = kKeys / 32;
    __shared__ u32x4 s_k[G::bytes(kKeys) / 16], s_v[G::bytes(kKeys) / 16];
    __shared__ float s_time[kKeys];
    __shared__ int s_reduce[4][4];
    extern __shared__ float s_lut[];

    const int64_t item = xcd_item(blockIdx.x, static_cast<int64_t>(a.tiles) * a.heads);
    if (item >= static_cast<int64_t>(a.tiles) * a.heads) return;
    const int head = static_cast<int>(item / a.tiles);
    // the last rows of a causal walk see most: first
    const int tile = a.tiles - 1 - static_cast<int>(item % a.tiles);
    const int kv_head = head / a.group;
    const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6, half = lane >> 5;
    const Score& sc = a.score;

    const int i = tile * kTileRows + wave * kRowsPerWave + (lane & 31);
    int4 info = {0, 0, 0, 0};
    if (i < a.q_rows) info = a.q_info[i];
    int lo = info.x, hi = max(info.x, min(info.y, a.k_rows));
    const int diag = info.z;
    const bool any = lo < hi;

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
    const bool mixed = k_begin < last_lo;  // rows of more than one walk

    Frag<T> q[G::kSteps];
    load_operand<T, DB>(q, row_of<const T>(a.q, i, head), any, a.dim, half);
    const float slope = sc.slopes ? sc.slopes[head] * kLog2e : 0.0f;
    const float q_time = sc.q_times && any ? sc.q_times[i] : 0.0f;
    const T* k_base = row_of<const T>(a.k, 0, kv_head);
    const T* v_base = row_of<const T>(a.v, 0, kv_head);

    int only = -1;  // -1: every row; else the rows whose keys begin there, again
    int j_first = k_begin;
    for (;;) {
        f32x16 o[DB];
#pragma unroll
        for (int b = 0; b < DB; ++b) o[b] = zero16();
        float m = kFloor, l = 0.0f;
        // Every row must be inside a tile for it to go unmasked
        const int full_lo = wave_max(any ? lo : kNone), full_hi = wave_min(any ? hi : 0);

        Staged<T, DB, kKeys, kThreads> next_k, next_v;
        next_k.load(k_base, a.k.row, a.dim, j_first, k_begin, k_end, thread);
        next_v.load(v_base, a.v.row, a.dim, j_first, k_begin, k_end, thread);
        for (int j0 = j_first; j0 < k_end; j0 += kKeys) {
            __syncthreads();  // the tile before is done with
            next_k.store(s_k, thread);
            next_v.store(s_v, thread);
            if (sc.k_times && thread < kKeys)
                s_time[thread] = j0 + thread < k_end ? sc.k_times[j0 + thread] : 0.0f;
            __syncthreads();
            if (j0 + kKeys < k_end) {
                next_k.load(k_base, a.k.row, a.dim, j0 + kKeys, k_begin, k_end, thread);
                next_v.load(v_base, a.v.row, a.dim, j0 + kKeys, k_begin, k_end, thread);
            }
            if (j0 >= w_hi || j0 + kKeys <= w_lo) continue;

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
            if (sc.softcap > 0) {
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float unused;
                        s[b][r] = capped<T>(sc, s[b][r], unused);
                    }
            } else {
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[b][r] *= sc.scale2;
            }
            const int j_lane = j0 + 4 * half;  // register r's key: + 32 b + acc_row(r)
            if (sc.table) {
                const int far_lo = w_diag_lo - (j0 + kKeys - 1), far_hi = w_diag_hi - j0;
                if (far_lo >= sc.reach || far_hi <= -sc.reach) {
                    const float bias = s_lut[far_lo >= sc.reach ? 2 * sc.reach : 0];
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[b][r] += bias;
                } else {
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int d = diag - (j_lane + 32 * b + acc_row(r));
                            s[b][r] += s_lut[min(max(d, -sc.reach), sc.reach) + sc.reach];
                        }
                }
            }
            if (sc.slopes) {
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int at = 32 * b + acc_row(r);
                        const float gap = sc.k_times
                                              ? q_time - s_time[at + 4 * half]
                                              : static_cast<float>(diag - (j_lane + at));
                        s[b][r] = fmaf(-slope, fabsf(gap), s[b][r]);
                    }
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
            top = fmaxf(top, __shfl_xor(top, 32));
            if (__any(top > m)) {
                const float grown = fmaxf(m, top);
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
                    s[b][r] = exp2_fast(s[b][r] - m);
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
        const bool mine = i < a.q_rows && (only < 0 || (any && info.x == only));
        if (mine) {
            const bool seen = any && l != 0.0f;  // 0: the bias masks every key
            store_row<T, DB>(row_of<T>(a.out, i, head), o, seen, 1.0f / l, a.dim, half);
            if (a.stats && half == 0)
                a.stats[static_cast<int64_t>(head) * a.q_rows + i] =
                    seen ? make_float2(m, __builtin_amdgcn_logf(l)) : make_float2(0.0f, INFINITY);
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
        j_first += (only - j_first) / kKeys * kKeys;  // the same tiles: the same bits
        k_begin = only;
        k_end = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) k_end = max(k_end, s_reduce[w][1]);
    }
}

}  // namespace

uint64_t attention_backward_workspace(const trw_attention_params& p);

uint64_t attention_workspace(const trw_attention_params& p, bool backward) {
    return backward ? attention_backward_workspace(p) : 0;
}

void attention_forward(const trw_attention_params& p, hipStream_t stream) {
    if (p.q_rows == 0) return;
    ForwardArgs a;
    a.q = make_rows(p.q);
    a.k = make_rows(p.k);
    a.v = make_rows(p.v);
    a.out = make_rows(p.out);
    a.q_info = reinterpret_cast<const int4*>(p.q_rows_info);
    a.stats = reinterpret_cast<float2*>(p.stats);
    a.score = make_score(p.score);
    a.q_rows = static_cast<int>(p.q_rows);
    a.k_rows = static_cast<int>(p.k_rows);
    a.heads = p.heads;
    a.group = p.heads / p.kv_heads;
    a.dim = p.dim;
    a.tiles = static_cast<int>((p.q_rows + kTileRows - 1) / kTileRows);
    const int64_t grid = xcd_grid(static_cast<int64_t>(a.tiles) * a.heads);
    const size_t lds = p.score.table ? (2 * a.score.reach + 1) * sizeof(float) : 0;
    dispatch(p.dtype, p.dim, [&](auto t, auto db) {
        hipLaunchKernelGGL((attention_forward_kernel<decltype(t), decltype(db)::value>),
                           dim3(static_cast<unsigned>(grid)), dim3(kThreads), lds, stream, a);
    });
    check_launch("attention_forward");
}

}  // namespace ops
}  // namespace trw
