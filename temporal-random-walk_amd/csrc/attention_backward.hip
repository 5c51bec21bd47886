// attention_backward.hip -- gradients of attention.hip's formula.
//
//   P_ij = exp2(s_ij - m_i) / l_i           (m, l from the forward pass)
//   D_i = dO_i . o_i,  dS_ij = P_ij (dO_i . v_j - D_i)
//   dx_ij = dS_ij (1 - tanh^2)              (1 without a cap)
//   dq_i = scale sum_j dx_ij k_j,  dk_j = scale sum_i dx_ij q_i
//   dv_j = sum_i P_ij dO_i,  dtable[b] = sum of dS over pairs of bucket b
//
// Two kernels, one over tiles of query rows (dq, D, the table) and one over
// tiles of keys (dk, dv): the scores are computed twice, which costs two
// products of seven, and no sum is shared between workgroups, so nothing
// depends on the order they run in and no float32 copy of a gradient goes
// through memory.  Heads that share keys are one sum in registers.
//
// Bound by what two (over keys: one) workgroups a compute unit can hide of the
// waits between products and arithmetic: one causal walk of 8192 rows (16 heads of 128 over 4 key
// heads, capped scores, bfloat16) takes 0.78 ms over query rows (vector units busy
// 0.45 of the time, matrix units 0.22) and 0.98 over keys (0.34 and 0.23), where
// two operands and two sums of 128 columns leave room for one workgroup.
#include <algorithm>

#include "operators.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kTileRows = 128;  // query rows or keys of a workgroup

struct BackwardArgs {
    Rows q, k, v, out, out_low, d_out, d_q, d_k, d_v;
    const int4* q_info;
    const int4* k_info;
    const float* stats;
    float* delta;    // [heads, q_rows] D
    float* partial;  // [heads, q tiles, 2 reach + 1] dS by distance
    Score score;
    int q_rows, k_rows, heads, group, dim;
    int q_tiles, k_tiles;
    int splits;          // workgroups that share a key head's query heads
    int walk_limit;      // documents up to here go a wave each (attention_walks.hip)
    float *part_k, *part_v;  // [splits, k_rows, kv_heads, dim], where splits > 1
};

// Scores in base 2 of one block's products, and the slope that the cap left.
template <typename T, bool kWide>
__device__ __forceinline__ void score_block(const Score& sc, const f32x16& product,
                                            float (&x)[1][16], float (&slope)[16]) {
    if (sc.softcap > 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[0][r] = capped<T, kWide>(sc, product[r], slope[r]);
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[0][r] = product[r] * sc.scale2;
            slope[r] = 1.0f;
        }
    }
}

// ---- over query rows: dq, D, the table -------------------------------------------------------
//
// A lane holds one query row (column) and 16 keys at a time.  The table's
// gradient is dS by distance, along a block's diagonals (add_diagonals); pairs
// past the reach are summed in registers.  Rows whose walks' queries and keys
// are not one distance apart (prompts of several walks) have no common diagonals
// and take float atomics on the wave's own line.
template <typename T, int DB, bool kWide>
__global__ __launch_bounds__(kThreads, 2) void attention_backward_q_kernel(BackwardArgs a) {
    typedef Tile<T, DB> G;
    constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;
    __shared__ u32x4 s_kv[2][2][kKeys * G::kSlots];
    __shared__ float s_times[2][64];
    __shared__ int s_reduce[4][4];
    extern __shared__ float s_dyn[];  // bias by distance; 4 lines of its gradient, 4 squares

    const int64_t items = static_cast<int64_t>(a.q_tiles) * a.heads;
    const int64_t item = xcd_item(blockIdx.x, items);
    if (item >= items) return;
    const int head = static_cast<int>(item / a.q_tiles);
    const int tile = a.q_tiles - 1 - static_cast<int>(item % a.q_tiles);
    const int kv_head = head / a.group;
    const int thread = threadIdx.x, lane = thread & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const Score& sc = a.score;
    const int line = 2 * sc.reach + 1;
    float* s_lut = s_dyn;
    float* s_sum = s_dyn + line + wave * line;
    float* s_square = s_dyn + 5 * line + wave * kSquare;

    const int i = tile * kTileRows + wave * 32 + (lane & 31);
    int4 info = {0, 0, 0, 0};
    if (i < a.q_rows) info = a.q_info[i];
    const bool mine = i < a.q_rows && tiled(info.w, a.walk_limit);
    // Nothing here for most workgroups of a batch whose walks go a wave each
    if (!__syncthreads_or(mine)) {
        if (sc.table)
            for (int n = thread; n < line; n += kThreads)
                a.partial[(static_cast<int64_t>(head) * a.q_tiles + tile) * line + n] = 0.0f;
        return;
    }
    int lo = info.x, hi = mine ? max(info.x, min(info.y, a.k_rows)) : info.x;
    const int diag = info.z;
    const bool any = lo < hi;

    Frag<T> q[G::kSteps], d_o[G::kSteps];
    load_operand<T, DB>(q, row_of<const T>(a.q, i, head), any, a.dim, half);
    load_operand<T, DB>(d_o, row_of<const T>(a.d_out, i, head), any, a.dim, half);

    int w_lo = wave_min(any ? lo : kNone), w_hi = wave_max(any ? hi : 0);
    const int w_diag_lo = wave_min(any ? diag : kNone), w_diag_hi = wave_max(any ? diag : -kNone);
    // distance of lane's row from key j: apart + i - j, where all rows agree
    const int apart = wave_min(any ? diag - i : kNone);
    const bool diagonal = apart == wave_max(any ? diag - i : -kNone);
    const int w_last_lo = wave_max(any ? lo : 0);
    if (lane == 0) {
        s_reduce[wave][0] = w_lo;
        s_reduce[wave][1] = w_hi;
        s_reduce[wave][2] = w_last_lo;
    }
    if (sc.table) {
        fill_bias(s_lut, sc, head, thread, kThreads);
        for (int n = thread; n < 4 * (line + kSquare); n += kThreads) s_dyn[line + n] = 0.0f;
    }
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
    const bool mixed = k_begin < last_lo;

    float delta = 0.0f;
    {
        Frag<T> o[G::kSteps];
        load_operand<T, DB>(o, row_of<const T>(a.out, i, head), any, a.dim, half);
#pragma unroll
        for (int s = 0; s < G::kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                delta = fmaf(static_cast<float>(o[s][e]), static_cast<float>(d_o[s][e]), delta);
        if (a.out_low.data) {
            // of o before it was rounded: an error of D is one of every dS of
            // its row, all of one sign, which a table's sums would keep
            load_operand<T, DB>(o, row_of<const T>(a.out_low, i, head), any, a.dim, half);
#pragma unroll
            for (int s = 0; s < G::kSteps; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    delta = fmaf(static_cast<float>(o[s][e]), static_cast<float>(d_o[s][e]), delta);
        }
        delta += __shfl_xor(delta, 32);
    }
    const int64_t stat = static_cast<int64_t>(head) * a.q_rows + i;
    float m = INFINITY, log_l = INFINITY;
    if (any) {
        m = a.stats[stat];
        log_l = sc.biased() ? a.stats[static_cast<int64_t>(a.heads) * a.q_rows + stat] : 0.0f;
    }
    if (mine && half == 0) a.delta[stat] = delta;
    const float slope = sc.slopes ? sc.slopes[head] * kLog2e : 0.0f;
    const float q_time = sc.q_times && any ? sc.q_times[i] : 0.0f;
    const T* k_base = row_of<const T>(a.k, 0, kv_head);
    const T* v_base = row_of<const T>(a.v, 0, kv_head);
    constexpr int kTileBytes = kKeys * G::kSlots * 16;
    const uint32_t at_kv = lds_address(s_kv), at_times = lds_address(s_times);
    const Loader<T, DB, kKeys, kThreads> k_load(a.k.row, a.dim, thread);
    const Loader<T, DB, kKeys, kThreads> v_load(a.v.row, a.dim, thread);
    float far_before = 0.0f, far_after = 0.0f;  // dS past the reach, either way

    int only = -1;
    const int j_begin = k_begin;
    int j_first = k_begin;
    for (;;) {
        f32x16 dq[DB];
#pragma unroll
        for (int b = 0; b < DB; ++b) dq[b] = zero16();
        const int full_lo = wave_max(any ? lo : kNone), full_hi = wave_min(any ? hi : 0);
        auto fetch = [&](int j0, int buffer) {
            k_load.load(k_base, j0, k_begin, k_end, at_kv + buffer * 2 * kTileBytes, thread);
            v_load.load(v_base, j0, k_begin, k_end, at_kv + (buffer * 2 + 1) * kTileBytes, thread);
            if (sc.k_times && wave == 0)
                load_floats(sc.k_times, j0, k_begin, k_end, at_times + buffer * 256, lane);
        };
        int buffer = 0;
        if (j_first < k_end) fetch(j_first, 0);
        for (int jt = j_first; jt < k_end; jt += kKeys, buffer ^= 1) {
            landed();
            if (jt + kKeys < k_end) fetch(jt + kKeys, buffer ^ 1);
#pragma unroll 1
            for (int sub = 0; sub < kKeys; sub += 32) {
                const int j0 = jt + sub;
                if (j0 >= w_hi || j0 + 32 <= w_lo) continue;
                const u32x4* s_k = s_kv[buffer][0] + sub * G::kSlots;
                const u32x4* s_v = s_kv[buffer][1] + sub * G::kSlots;
                // LDS addresses are worked out for each block: held over the
                // loop, they would take the registers of the sums
                int at_lane = lane;
                asm volatile("" : "+v"(at_lane));

                f32x16 product = zero16(), dp = zero16();
#pragma unroll
                for (int st = 0; st < G::kSteps; ++st) {
                    product = mma(G::row(s_k, lane & 31, st, half), q[st], product);
                    dp = mma(G::row(s_v, lane & 31, st, half), d_o[st], dp);
                }
                float x[1][16], cap_slope[16];
                score_block<T, kWide>(sc, product, x, cap_slope);
                const int j_lane = j0 + 4 * half;
                if (sc.biased()) {
                    add_biases(sc, x, s_lut, slope, diag, w_diag_lo, w_diag_hi, q_time,
                               s_times[buffer] + sub, j0, half);
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[0][r] = (x[0][r] - m) - log_l;
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[0][r] -= m;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) x[0][r] = exp2_fast(x[0][r]) * (dp[r] - delta);
                if (j0 < full_lo || j0 + 32 > full_hi) {
                    const unsigned span = static_cast<unsigned>(hi - lo);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = j_lane + acc_row(r);
                        if (static_cast<unsigned>(j - lo) >= span) x[0][r] = 0.0f;
                    }
                }
                if (sc.table && only < 0) {
                    const int far_lo = w_diag_lo - (j0 + 31), far_hi = w_diag_hi - j0;
                    if (far_lo >= sc.reach || far_hi <= -sc.reach) {
                        float sum = 0.0f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) sum += x[0][r];
                        if (far_lo >= sc.reach) far_before += sum;
                        else far_after += sum;
                    } else if (diagonal) {
                        const int at = tile * kTileRows + wave * 32 + apart - j0;
                        add_diagonals(x[0], s_square, s_sum, sc.reach, at, at + 31, lane, half);
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int d = diag - (j_lane + acc_row(r));
                            far_before += d >= sc.reach ? x[0][r] : 0.0f;
                            far_after += d <= -sc.reach && d < sc.reach ? x[0][r] : 0.0f;
                            if (abs(d) < sc.reach) atomicAdd(&s_sum[d + sc.reach], x[0][r]);
                        }
                    }
                }
                if (sc.softcap > 0) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[0][r] *= cap_slope[r];
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    Frag<T> ds;
#pragma unroll
                    for (int e = 0; e < 8; ++e) ds[e] = static_cast<T>(x[0][8 * t + e]);
#pragma unroll
                    for (int b = 0; b < DB; ++b)
                        dq[b] = mma(G::columns(s_k, 16 * t, b, at_lane), ds, dq[b]);
                }
            }
        }
        if (mine && (only < 0 || (any && info.x == only)))
            store_row<T, DB>(row_of<T>(a.d_q, i, head), dq, any, sc.scale, a.dim, half);
        if (!mixed) break;

        // As in the forward kernel: what is not finite stays in its walk.
        bool off = false;
        if (any && info.x > only) {
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += dq[b][r] * 0.0f;
            off = sum != 0.0f;
        }
        if (only < 0 && !__syncthreads_or(off)) break;
        const int w_next = wave_min(any && info.x > only ? info.x : kNone);
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
        j_first = j_begin + (k_begin - j_begin) / kKeys * kKeys;  // the same tiles: the same bits
    }

    if (!sc.table) return;
    // this tile's line: lanes' far sums first
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        far_before += __shfl_xor(far_before, o);
        far_after += __shfl_xor(far_after, o);
    }
    if (lane == 0) {
        s_sum[2 * sc.reach] += far_before;
        s_sum[0] += far_after;
    }
    __syncthreads();
    float* s_line = s_dyn + line;
    float* out = a.partial + (static_cast<int64_t>(head) * a.q_tiles + tile) * line;
    for (int n = thread; n < line; n += kThreads) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) sum += s_line[w * line + n];
        out[n] = sum;
    }
}

// ---- over keys: dk, dv -------------------------------------------------------------------------
//
// A lane holds one key (column) and 16 query rows at a time; q and dO pass
// through LDS and are read both ways.
template <typename T, int DB, bool kWide>
__global__ __launch_bounds__(kThreads, DB < 4 ? 2 : 1) void attention_backward_kv_kernel(
    BackwardArgs a) {
    typedef Tile<T, DB> G;
    constexpr int kRows = sizeof(T) == 2 ? 64 : 32;
    __shared__ u32x4 s_rows[2][2][kRows * G::kSlots];  // q and dO
    __shared__ float s_stats[2][4][64];                // m, log l, D, times
    __shared__ int4 s_infos[2][64];
    __shared__ int s_reduce[4][4];
    extern __shared__ float s_lut[];

    const int kv_heads = a.heads / a.group;
    const int64_t items = static_cast<int64_t>(a.k_tiles) * kv_heads * a.splits;
    const int64_t item = xcd_item(blockIdx.x, items);
    if (item >= items) return;
    const int split = static_cast<int>(item / a.k_tiles) % a.splits;
    const int kv_head = static_cast<int>(item / a.k_tiles) / a.splits;
    const int tile = static_cast<int>(item % a.k_tiles);  // the first keys are seen most: first
    const int thread = threadIdx.x, lane = thread & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const Score& sc = a.score;

    const int j = tile * kTileRows + wave * 32 + (lane & 31);
    int4 info = {0, 0, 0, 0};
    if (j < a.k_rows) info = a.k_info[j];
    const bool mine = j < a.k_rows && tiled(info.w, a.walk_limit);
    if (!__syncthreads_or(mine)) return;
    int first = info.x, last = mine ? max(info.x, min(info.y, a.q_rows)) : info.x;
    const bool any = first < last;
    const int doc = last;  // no two walks with pairs end at one query

    Frag<T> k[G::kSteps], v[G::kSteps];
    load_operand<T, DB>(k, row_of<const T>(a.k, j, kv_head), any, a.dim, half);
    load_operand<T, DB>(v, row_of<const T>(a.v, j, kv_head), any, a.dim, half);

    int w_lo = wave_min(any ? first : kNone), w_hi = wave_max(any ? last : 0);
    const int w_first_doc = wave_min(any ? doc : kNone);
    if (lane == 0) {
        s_reduce[wave][0] = w_lo;
        s_reduce[wave][1] = w_hi;
        s_reduce[wave][2] = w_first_doc;
    }
    __syncthreads();
    int q_begin = kNone, q_end = 0, first_doc = kNone;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        q_begin = min(q_begin, s_reduce[w][0]);
        q_end = max(q_end, s_reduce[w][1]);
        first_doc = min(first_doc, s_reduce[w][2]);
    }
    q_begin = __builtin_amdgcn_readfirstlane(q_begin);
    q_end = __builtin_amdgcn_readfirstlane(q_end);
    const bool mixed = q_begin < q_end && first_doc < q_end;

    const float k_time = sc.k_times && any ? sc.k_times[j] : 0.0f;
    const int heads_each = (a.group + a.splits - 1) / a.splits;
    const int head_begin = kv_head * a.group + split * heads_each;
    const int head_end = min(head_begin + heads_each, (kv_head + 1) * a.group);
    constexpr int kTileBytes = kRows * G::kSlots * 16;
    const uint32_t at_rows = lds_address(s_rows), at_stats = lds_address(s_stats),
                   at_infos = lds_address(s_infos);
    const Loader<T, DB, kRows, kThreads> q_load(a.q.row, a.dim, thread);
    const Loader<T, DB, kRows, kThreads> do_load(a.d_out.row, a.dim, thread);
    const bool positions = sc.table || (sc.slopes && !sc.k_times);

    int only = -1;
    const int i_begin = q_begin;
    int i_first = q_begin;
    for (;;) {
        f32x16 dk[DB], dv[DB];
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            dk[b] = zero16();
            dv[b] = zero16();
        }
        const int full_lo = wave_max(any ? first : kNone), full_hi = wave_min(any ? last : 0);
#pragma unroll 1
        for (int head = head_begin; head < head_end; ++head) {
            const T* q_base = row_of<const T>(a.q, 0, head);
            const T* do_base = row_of<const T>(a.d_out, 0, head);
            const float* m_base = a.stats + static_cast<int64_t>(head) * a.q_rows;
            const float* log_l_base = m_base + static_cast<int64_t>(a.heads) * a.q_rows;
            const float* delta_base = a.delta + static_cast<int64_t>(head) * a.q_rows;
            const float slope = sc.slopes ? sc.slopes[head] * kLog2e : 0.0f;
            __syncthreads();  // the head before is done with its biases and tiles
            if (sc.table) fill_bias(s_lut, sc, head, thread, kThreads);
            auto fetch = [&](int i0, int buffer) {
                q_load.load(q_base, i0, q_begin, q_end, at_rows + buffer * 2 * kTileBytes, thread);
                do_load.load(do_base, i0, q_begin, q_end, at_rows + (buffer * 2 + 1) * kTileBytes,
                             thread);
                if (wave == 0) {
                    load_floats(m_base, i0, q_begin, q_end, at_stats + (buffer * 4 + 0) * 256, lane);
                    if (sc.biased())
                        load_floats(log_l_base, i0, q_begin, q_end, at_stats + (buffer * 4 + 1) * 256, lane);
                } else if (wave == 1) {
                    load_floats(delta_base, i0, q_begin, q_end, at_stats + (buffer * 4 + 2) * 256, lane);
                } else if (wave == 2) {
                    if (sc.q_times)
                        load_floats(sc.q_times, i0, q_begin, q_end, at_stats + (buffer * 4 + 3) * 256, lane);
                } else if (positions) {
                    const int from = min(max(i0, q_begin), q_end - 1);
                    const int at = min(max(i0 + lane, q_begin), q_end - 1) - from;
                    copy_to_lds(a.q_info + from, static_cast<uint32_t>(at) * 16,
                                at_infos + buffer * 1024);
                }
            };
            int buffer = 0;
            if (i_first < q_end) fetch(i_first, 0);
            for (int it = i_first; it < q_end; it += kRows, buffer ^= 1) {
                landed();
                if (it + kRows < q_end) fetch(it + kRows, buffer ^ 1);
#pragma unroll 1
                for (int sub = 0; sub < kRows; sub += 32) {
                    const int i0 = it + sub;
                    if (i0 >= w_hi || i0 + 32 <= w_lo) continue;
                    const u32x4* s_q = s_rows[buffer][0] + sub * G::kSlots;
                    const u32x4* s_do = s_rows[buffer][1] + sub * G::kSlots;
                    int at_lane = lane;  // as above
                    if (DB == 3) asm volatile("" : "+v"(at_lane));
                    // row of register r: acc_row(r) of these
                    const float* s_m = s_stats[buffer][0] + sub + 4 * half;
                    const float* s_log_l = s_stats[buffer][1] + sub + 4 * half;
                    const float* s_delta = s_stats[buffer][2] + sub + 4 * half;
                    const float* s_time = s_stats[buffer][3] + sub + 4 * half;
                    const int4* s_info = s_infos[buffer] + sub + 4 * half;

                    f32x16 product = zero16(), dp = zero16();
#pragma unroll
                    for (int st = 0; st < G::kSteps; ++st) {
                        product = mma(G::row(s_q, at_lane & 31, st, at_lane >> 5), k[st], product);
                        dp = mma(G::row(s_do, at_lane & 31, st, at_lane >> 5), v[st], dp);
                        if (DB == 3 && st % 2) hold_reads();
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) dp[r] -= s_delta[acc_row(r)];
                    float x[16];
                    if (sc.softcap > 0) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            float cap_slope;
                            x[r] = capped<T, kWide>(sc, product[r], cap_slope);
                            dp[r] *= cap_slope;
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[r] = product[r] * sc.scale2;
                    }
                    if (sc.table) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int d = s_info[acc_row(r)].z - j;
                            x[r] += s_lut[min(max(d, -sc.reach), sc.reach) + sc.reach];
                        }
                    }
                    if (sc.slopes) {
                        if (sc.k_times) {
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                x[r] = fmaf(-slope, fabsf(s_time[acc_row(r)] - k_time), x[r]);
                        } else {
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                x[r] = fmaf(-slope,
                                            fabsf(static_cast<float>(s_info[acc_row(r)].z - j)),
                                            x[r]);
                        }
                    }
                    if (sc.biased()) {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            x[r] = (x[r] - s_m[acc_row(r)]) - s_log_l[acc_row(r)];
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[r] -= s_m[acc_row(r)];
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        x[r] = exp2_fast(x[r]);
                        dp[r] *= x[r];
                    }
                    if (i0 < full_lo || i0 + 32 > full_hi) {
                        const unsigned span = static_cast<unsigned>(last - first);
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int i = i0 + acc_row(r) + 4 * half;
                            if (static_cast<unsigned>(i - first) >= span) x[r] = dp[r] = 0.0f;
                        }
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        Frag<T> p, ds;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            p[e] = static_cast<T>(x[8 * t + e]);
                            ds[e] = static_cast<T>(dp[8 * t + e]);
                        }
#pragma unroll
                        for (int b = 0; b < DB; ++b) {
                            dv[b] = mma(G::columns(s_do, 16 * t, b, at_lane), p, dv[b]);
                            dk[b] = mma(G::columns(s_q, 16 * t, b, at_lane), ds, dk[b]);
                            if (DB == 3) hold_reads();
                        }
                    }
                }
            }
        }
        if (mine && (only < 0 || (any && doc == only))) {
            if (a.splits > 1) {
                const int64_t at =
                    ((static_cast<int64_t>(split) * a.k_rows + j) * kv_heads + kv_head) * a.dim;
                store_row<float, DB>(a.part_k + at, dk, any, sc.scale, a.dim, half);
                store_row<float, DB>(a.part_v + at, dv, any, 1.0f, a.dim, half);
            } else {
                store_row<T, DB>(row_of<T>(a.d_k, j, kv_head), dk, any, sc.scale, a.dim, half);
                store_row<T, DB>(row_of<T>(a.d_v, j, kv_head), dv, any, 1.0f, a.dim, half);
            }
        }
        if (!mixed) break;

        // As in the forward kernel: what is not finite stays in its walk.
        bool off = false;
        if (any && doc > only) {
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += dk[b][r] * 0.0f + dv[b][r] * 0.0f;
            off = sum != 0.0f;
        }
        if (only < 0 && !__syncthreads_or(off)) break;
        const int w_next = wave_min(any && doc > only ? doc : kNone);
        __syncthreads();
        if (lane == 0) s_reduce[wave][0] = w_next;
        __syncthreads();
        int seg = kNone;
#pragma unroll
        for (int w = 0; w < 4; ++w) seg = min(seg, s_reduce[w][0]);
        if (seg == kNone) break;
        only = seg;
        const bool in_seg = any && doc == only;
        first = in_seg ? info.x : 0;
        last = in_seg ? doc : 0;
        w_lo = wave_min(in_seg ? first : kNone);
        w_hi = wave_max(in_seg ? last : 0);
        if (lane == 0) s_reduce[wave][1] = w_lo;
        __syncthreads();
        q_begin = kNone;
        q_end = __builtin_amdgcn_readfirstlane(only);
#pragma unroll
        for (int w = 0; w < 4; ++w) q_begin = min(q_begin, s_reduce[w][1]);
        q_begin = __builtin_amdgcn_readfirstlane(q_begin);
        i_first = i_begin + (q_begin - i_begin) / kRows * kRows;  // the same tiles: the same bits
    }
}

// dk, dv of a key head whose query heads were split over workgroups.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_splits_kernel(BackwardArgs a) {
    const int kv_heads = a.heads / a.group;
    const int64_t n = static_cast<int64_t>(a.k_rows) * kv_heads * (a.dim / 4);
    const int64_t t = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
    if (t >= n) return;
    const int col = static_cast<int>(t % (a.dim / 4)) * 4;
    const int64_t rest = t / (a.dim / 4);
    const int head = static_cast<int>(rest % kv_heads);
    const int64_t row = rest / kv_heads;
    if (!tiled(a.k_info[row].w, a.walk_limit)) return;
    const int64_t step = static_cast<int64_t>(a.k_rows) * kv_heads * a.dim;
    f32x4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
    for (int s = 0; s < a.splits; ++s) {
        const f32x4 pk = *reinterpret_cast<const f32x4*>(a.part_k + s * step + t * 4);
        const f32x4 pv = *reinterpret_cast<const f32x4*>(a.part_v + s * step + t * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            k[e] += pk[e];
            v[e] += pv[e];
        }
    }
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 ok, ov;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        ok[e] = static_cast<T>(k[e]);
        ov[e] = static_cast<T>(v[e]);
    }
    *reinterpret_cast<t4*>(row_of<T>(a.d_k, row, head) + col) = ok;
    *reinterpret_cast<t4*>(row_of<T>(a.d_v, row, head) + col) = ov;
}

int tiles_of(int64_t rows) { return static_cast<int>((rows + kTileRows - 1) / kTileRows); }

// Workgroups that share a key head's query heads: one workgroup per key tile
// and key head sums them in registers; where those are fewer than two for each
// of the 256 compute units (long walks, few key heads), every query head has
// its own, through a float32 copy of dk and dv.
int splits_of(const trw_attention_params& p) {
    const int group = p.heads / p.kv_heads;
    const int64_t items = static_cast<int64_t>(tiles_of(p.k_rows)) * p.kv_heads;
    return group > 1 && items < 512 ? group : 1;
}

uint64_t align256(uint64_t n) { return (n + 255) / 256 * 256; }

struct Layout {
    uint64_t delta, partial = 0, walk_partial = 0, lines = 0, part_k, part_v, bytes;
};
Layout layout_of(const trw_attention_params& p) {
    Layout l;
    uint64_t at = 0;
    const int blocks = walk_blocks(p);
    const bool tiles = blocks == 0 || walk_rest(p, blocks);  // else the walks' kernels do it all
    auto take = [&](uint64_t floats) {
        const uint64_t here = at;
        at += align256(floats * sizeof(float));
        return here;
    };
    l.delta = take(tiles ? static_cast<uint64_t>(p.heads) * p.q_rows : 0);
    if (p.score.table) {
        const uint64_t heads = p.heads, line = 2 * static_cast<uint64_t>(p.score.reach) + 1;
        l.partial = take(tiles ? heads * tiles_of(p.q_rows) * line : 0);
        l.walk_partial = take(blocks ? heads * p.docs * walk_line(p, blocks) : 0);
        l.lines = take(heads * 2 * kJoinGroups * line);
    }
    const int splits = tiles ? splits_of(p) : 1;
    const uint64_t part =
        splits > 1 ? static_cast<uint64_t>(splits) * p.k_rows * p.kv_heads * p.dim : 0;
    l.part_k = take(part);
    l.part_v = take(part);
    l.bytes = at;
    return l;
}

}  // namespace

uint64_t attention_backward_workspace(const trw_attention_params& p) { return layout_of(p).bytes; }

void attention_backward(const trw_attention_params& p, hipStream_t stream) {
    const Layout l = layout_of(p);
    require(p.workspace_bytes >= l.bytes, "workspace is too small");
    char* ws = static_cast<char*>(p.workspace);
    BackwardArgs a;
    a.q = make_rows(p.q);
    a.k = make_rows(p.k);
    a.v = make_rows(p.v);
    a.out = make_rows(p.out);
    a.out_low = make_rows(p.out_low);
    a.d_out = make_rows(p.d_out);
    a.d_q = make_rows(p.d_q);
    a.d_k = make_rows(p.d_k);
    a.d_v = make_rows(p.d_v);
    a.q_info = reinterpret_cast<const int4*>(p.q_rows_info);
    a.k_info = reinterpret_cast<const int4*>(p.k_rows_info);
    a.stats = p.stats;
    a.delta = reinterpret_cast<float*>(ws + l.delta);
    a.partial = reinterpret_cast<float*>(ws + l.partial);
    a.part_k = reinterpret_cast<float*>(ws + l.part_k);
    a.part_v = reinterpret_cast<float*>(ws + l.part_v);
    a.score = make_score(p.score);
    a.q_rows = static_cast<int>(p.q_rows);
    a.k_rows = static_cast<int>(p.k_rows);
    a.heads = p.heads;
    a.group = p.heads / p.kv_heads;
    a.dim = p.dim;
    a.q_tiles = tiles_of(p.q_rows);
    a.k_tiles = tiles_of(p.k_rows);
    a.splits = splits_of(p);
    const int blocks = walk_blocks(p);
    const bool tiles = blocks == 0 || walk_rest(p, blocks);
    a.walk_limit = 32 * blocks;
    float* walk_partial = reinterpret_cast<float*>(ws + l.walk_partial);
    if (blocks) walk_backward(p, blocks, walk_partial, stream);
    const size_t line = p.score.table ? (2 * a.score.reach + 1) * sizeof(float) : 0;
    if (tiles)
        dispatch(p.dtype, p.dim, [&](auto t, auto db) {
            typedef decltype(t) T;
            constexpr int DB = decltype(db)::value;
            by_cap<T>(p.dtype, p.score, [&](auto wide) {
                constexpr bool kWide = decltype(wide)::value;
                if (a.q_tiles)
                    hipLaunchKernelGGL((attention_backward_q_kernel<T, DB, kWide>),
                                       dim3(static_cast<unsigned>(
                                           xcd_grid(static_cast<int64_t>(a.q_tiles) * a.heads))),
                                       dim3(kThreads),
                                       line ? 5 * line + 4 * kSquare * sizeof(float) : 0, stream,
                                       a);
                check_launch("attention_backward");
                if (a.k_tiles)
                    hipLaunchKernelGGL(
                        (attention_backward_kv_kernel<T, DB, kWide>),
                        dim3(static_cast<unsigned>(xcd_grid(
                            static_cast<int64_t>(a.k_tiles) * p.kv_heads * a.splits))),
                        dim3(kThreads), line, stream, a);
                check_launch("attention_backward");
            });
            if (a.k_tiles && a.splits > 1) {
                const int64_t n = p.k_rows * p.kv_heads * (p.dim / 4);
                hipLaunchKernelGGL((join_splits_kernel<T>),
                                   dim3(static_cast<unsigned>((n + kThreads - 1) / kThreads)),
                                   dim3(kThreads), 0, stream, a);
                check_launch("attention_backward");
            }
        });
    if (!p.score.table) return;
    // the table: tiles' and walks' lines, in up to 64 sums of each
    const int reach = a.score.reach;
    const int64_t walks = blocks ? p.docs : 0, q_tiles = tiles ? a.q_tiles : 0;
    const float* lines = a.partial;
    int count = static_cast<int>(q_tiles);
    if (walks || q_tiles > kJoinGroups) {
        float* joined = reinterpret_cast<float*>(ws + l.lines);
        const int tile_groups = static_cast<int>(std::min<int64_t>(q_tiles, kJoinGroups));
        const int walk_groups = static_cast<int>(std::min<int64_t>(walks, kJoinGroups));
        count = tile_groups + walk_groups;
        if (tile_groups)
            join_lines(a.partial, q_tiles, 2 * reach + 1, p.heads, tile_groups, joined, 0, count,
                       reach, stream);
        if (walk_groups)
            join_lines(walk_partial, walks, walk_line(p, blocks), p.heads, walk_groups, joined,
                       tile_groups, count, reach, stream);
        lines = joined;
    }
    join_table(lines, count, p.heads, p.score.buckets, reach, p.score.num_buckets, TRW_F32,
               p.d_table, stream);
}

}  // namespace ops
}  // namespace trw
