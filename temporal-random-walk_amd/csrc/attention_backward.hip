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
#include "operators.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kTileRows = 128;  // query rows or keys of a workgroup

struct BackwardArgs {
    Rows q, k, v, out, d_out, d_q, d_k, d_v;
    const int4* q_info;
    const int2* k_info;
    const float2* stats;
    float* delta;    // [heads, q_rows] D
    float* partial;  // [heads, q tiles, num_buckets]
    Score score;
    int q_rows, k_rows, heads, group, dim;
    int q_tiles, k_tiles;
    int splits;          // workgroups that share a key head's query heads
    float *part_k, *part_v;  // [splits, k_rows, kv_heads, dim], where splits > 1
};

// Scores of 16 pairs in base 2 from their products, and the slope the cap left.
template <typename T>
__device__ __forceinline__ void score_block(const Score& sc, float (&x)[16], float (&slope)[16]) {
    if (sc.softcap > 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = capped<T>(sc, x[r], slope[r]);
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[r] *= sc.scale2;
            slope[r] = 1.0f;
        }
    }
}

// ---- over query rows: dq, D, the table -------------------------------------------------------
//
// A lane holds one query row (column) and 16 keys at a time.  The table's
// gradient is summed by distance in LDS: the rows of a half wave lie at
// distinct distances from one key, so each half of each wave has a line of
// sums of its own and adds to it without two lanes meeting; pairs past the
// reach, which share two buckets, are summed in registers.
template <typename T, int DB>
__global__ __launch_bounds__(kThreads) void attention_backward_q_kernel(BackwardArgs a) {
    typedef Tile<T, DB> G;
    constexpr int kKeys = 32;
    __shared__ u32x4 s_k[G::bytes(kKeys) / 16], s_v[G::bytes(kKeys) / 16];
    __shared__ float s_time[kKeys];
    __shared__ int s_reduce[4][4];
    extern __shared__ float s_dyn[];  // bias by distance, then 8 lines of its gradient

    const int64_t items = static_cast<int64_t>(a.q_tiles) * a.heads;
    const int64_t item = xcd_item(blockIdx.x, items);
    if (item >= items) return;
    const int head = static_cast<int>(item / a.q_tiles);
    const int tile = a.q_tiles - 1 - static_cast<int>(item % a.q_tiles);
    const int kv_head = head / a.group;
    const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6, half = lane >> 5;
    const Score& sc = a.score;
    const int line = 2 * sc.reach + 1;
    float* s_lut = s_dyn;
    float* s_sum = s_dyn + line + (wave * 2 + half) * line;

    const int i = tile * kTileRows + wave * 32 + (lane & 31);
    int4 info = {0, 0, 0, 0};
    if (i < a.q_rows) info = a.q_info[i];
    int lo = info.x, hi = max(info.x, min(info.y, a.k_rows));
    const int diag = info.z;
    const bool any = lo < hi;
    int w_lo = wave_min(any ? lo : kNone), w_hi = wave_max(any ? hi : 0);
    const int w_diag_lo = wave_min(any ? diag : kNone), w_diag_hi = wave_max(any ? diag : -kNone);
    const int w_last_lo = wave_max(any ? lo : 0);
    if (lane == 0) {
        s_reduce[wave][0] = w_lo;
        s_reduce[wave][1] = w_hi;
        s_reduce[wave][2] = w_last_lo;
    }
    if (sc.table) {
        fill_bias(s_lut, sc, head, thread, kThreads);
        for (int n = thread; n < 8 * line; n += kThreads) s_dyn[line + n] = 0.0f;
    }
    __syncthreads();
    int k_begin = kNone, k_end = 0, last_lo = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        k_begin = min(k_begin, s_reduce[w][0]);
        k_end = max(k_end, s_reduce[w][1]);
        last_lo = max(last_lo, s_reduce[w][2]);
    }
    const bool mixed = k_begin < last_lo;

    Frag<T> q[G::kSteps], d_o[G::kSteps];
    load_operand<T, DB>(q, row_of<const T>(a.q, i, head), any, a.dim, half);
    load_operand<T, DB>(d_o, row_of<const T>(a.d_out, i, head), any, a.dim, half);
    float delta = 0.0f;
    {
        Frag<T> o[G::kSteps];
        load_operand<T, DB>(o, row_of<const T>(a.out, i, head), any, a.dim, half);
#pragma unroll
        for (int s = 0; s < G::kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                delta = fmaf(static_cast<float>(o[s][e]), static_cast<float>(d_o[s][e]), delta);
        delta += __shfl_xor(delta, 32);
    }
    const int64_t stat = static_cast<int64_t>(head) * a.q_rows + i;
    float m = 0.0f, log_l = INFINITY;
    if (any) {
        const float2 st = a.stats[stat];
        m = st.x;
        log_l = st.y;
    }
    if (i < a.q_rows && half == 0) a.delta[stat] = delta;
    const float slope = sc.slopes ? sc.slopes[head] * kLog2e : 0.0f;
    const float q_time = sc.q_times && any ? sc.q_times[i] : 0.0f;
    const T* k_base = row_of<const T>(a.k, 0, kv_head);
    const T* v_base = row_of<const T>(a.v, 0, kv_head);
    float far_before = 0.0f, far_after = 0.0f;  // dS past the reach, either way

    int only = -1;
    int j_first = k_begin;
    for (;;) {
        f32x16 dq[DB];
#pragma unroll
        for (int b = 0; b < DB; ++b) dq[b] = zero16();
        const int full_lo = wave_max(any ? lo : kNone), full_hi = wave_min(any ? hi : 0);
        Staged<T, DB, kKeys, kThreads> next_k, next_v;
        next_k.load(k_base, a.k.row, a.dim, j_first, k_begin, k_end, thread);
        next_v.load(v_base, a.v.row, a.dim, j_first, k_begin, k_end, thread);
        for (int j0 = j_first; j0 < k_end; j0 += kKeys) {
            __syncthreads();
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

            f32x16 x16 = zero16(), dp = zero16();
#pragma unroll
            for (int st = 0; st < G::kSteps; ++st) {
                x16 = mma(G::row(s_k, lane & 31, st, half), q[st], x16);
                dp = mma(G::row(s_v, lane & 31, st, half), d_o[st], dp);
            }
            float x[16], cap_slope[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = x16[r];
            score_block<T>(sc, x, cap_slope);
            const int j_lane = j0 + 4 * half;
            const int far_lo = w_diag_lo - (j0 + kKeys - 1), far_hi = w_diag_hi - j0;
            const bool far = far_lo >= sc.reach || far_hi <= -sc.reach;
            if (sc.table) {
                if (far) {
                    const float bias = s_lut[far_lo >= sc.reach ? 2 * sc.reach : 0];
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] += bias;
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int d = diag - (j_lane + acc_row(r));
                        x[r] += s_lut[min(max(d, -sc.reach), sc.reach) + sc.reach];
                    }
                }
            }
            if (sc.slopes) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float gap = sc.k_times
                                          ? q_time - s_time[acc_row(r) + 4 * half]
                                          : static_cast<float>(diag - (j_lane + acc_row(r)));
                    x[r] = fmaf(-slope, fabsf(gap), x[r]);
                }
            }
            // m apart from log l: next to a score near the type's lowest, log l
            // would be lost
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                x[r] = exp2_fast((x[r] - m) - log_l) * (dp[r] - delta);
            }
            if (j0 < full_lo || j0 + kKeys > full_hi) {
                const unsigned span = static_cast<unsigned>(hi - lo);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = j_lane + acc_row(r);
                    if (static_cast<unsigned>(j - lo) >= span) x[r] = 0.0f;
                }
            }
            if (sc.table && only < 0) {
                if (far) {
                    float sum = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum += x[r];
                    if (far_lo >= sc.reach) far_before += sum;
                    else far_after += sum;
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int d = diag - (j_lane + acc_row(r));
                        if (d >= sc.reach) far_before += x[r];
                        else if (d <= -sc.reach) far_after += x[r];
                        else if (any) atomicAdd(&s_sum[d + sc.reach], x[r]);
                    }
                }
            }
            if (sc.softcap > 0) {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] *= cap_slope[r];
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag<T> ds;
#pragma unroll
                for (int e = 0; e < 8; ++e) ds[e] = static_cast<T>(x[8 * t + e]);
#pragma unroll
                for (int b = 0; b < DB; ++b) dq[b] = mma(G::columns(s_k, 16 * t, b, lane), ds, dq[b]);
            }
        }
        if (i < a.q_rows && (only < 0 || (any && info.x == only)))
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
        j_first += (only - j_first) / kKeys * kKeys;  // the same tiles: the same bits
        k_begin = only;
        k_end = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) k_end = max(k_end, s_reduce[w][1]);
    }

    if (!sc.table) return;
    // this tile's sums by bucket: lanes' far sums first
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
    for (int n = thread; n < line; n += kThreads) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += s_line[w * line + n];
        s_line[n] = sum;
    }
    __syncthreads();
    // buckets in any order: 8 threads look through the distances for each
    const int part = thread & 7;
    for (int b = thread >> 3; b < sc.num_buckets; b += kThreads / 8) {
        float sum = 0.0f;
        for (int n = part; n < line; n += 8) {
            const int of = min(max(sc.buckets[n], 0), sc.num_buckets - 1);
            if (of == b) sum += s_line[n];
        }
        sum += __shfl_xor(sum, 1);
        sum += __shfl_xor(sum, 2);
        sum += __shfl_xor(sum, 4);
        if (part == 0)
            a.partial[(static_cast<int64_t>(head) * a.q_tiles + tile) * sc.num_buckets + b] = sum;
    }
}

// ---- over keys: dk, dv -------------------------------------------------------------------------
//
// A lane holds one key (column) and 16 query rows at a time; q and dO pass
// through LDS and are read both ways.
template <typename T, int DB>
__global__ __launch_bounds__(kThreads) void attention_backward_kv_kernel(BackwardArgs a) {
    typedef Tile<T, DB> G;
    constexpr int kRows = 32;
    __shared__ u32x4 s_q[G::bytes(kRows) / 16], s_do[G::bytes(kRows) / 16];
    __shared__ float s_m[kRows], s_log_l[kRows], s_delta[kRows], s_time[kRows];
    __shared__ int s_diag[kRows];
    __shared__ int s_reduce[4][4];
    extern __shared__ float s_lut[];

    const int kv_heads = a.heads / a.group;
    const int64_t items = static_cast<int64_t>(a.k_tiles) * kv_heads * a.splits;
    const int64_t item = xcd_item(blockIdx.x, items);
    if (item >= items) return;
    const int split = static_cast<int>(item / a.k_tiles) % a.splits;
    const int kv_head = static_cast<int>(item / a.k_tiles) / a.splits;
    const int tile = static_cast<int>(item % a.k_tiles);  // the first keys are seen most: first
    const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6, half = lane >> 5;
    const Score& sc = a.score;

    const int j = tile * kTileRows + wave * 32 + (lane & 31);
    int2 info = {0, 0};
    if (j < a.k_rows) info = a.k_info[j];
    int first = info.x, last = max(info.x, min(info.y, a.q_rows));
    const bool any = first < last;
    const int doc = last;  // no two walks with pairs end at one query
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
    const bool mixed = q_begin < q_end && first_doc < q_end;

    Frag<T> k[G::kSteps], v[G::kSteps];
    load_operand<T, DB>(k, row_of<const T>(a.k, j, kv_head), any, a.dim, half);
    load_operand<T, DB>(v, row_of<const T>(a.v, j, kv_head), any, a.dim, half);
    const float k_time = sc.k_times && any ? sc.k_times[j] : 0.0f;
    const int heads_each = (a.group + a.splits - 1) / a.splits;
    const int head_begin = kv_head * a.group + split * heads_each;
    const int head_end = min(head_begin + heads_each, (kv_head + 1) * a.group);

    int only = -1;
    int i_first = q_begin;
    for (;;) {
        f32x16 dk[DB], dv[DB];
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            dk[b] = zero16();
            dv[b] = zero16();
        }
        const int full_lo = wave_max(any ? first : kNone), full_hi = wave_min(any ? last : 0);
        for (int head = head_begin; head < head_end; ++head) {
            const T* q_base = row_of<const T>(a.q, 0, head);
            const T* do_base = row_of<const T>(a.d_out, 0, head);
            const int64_t stat = static_cast<int64_t>(head) * a.q_rows;
            const float slope = sc.slopes ? sc.slopes[head] * kLog2e : 0.0f;
            if (sc.table) {
                __syncthreads();
                fill_bias(s_lut, sc, head, thread, kThreads);
            }
            Staged<T, DB, kRows, kThreads> next_q, next_do;
            next_q.load(q_base, a.q.row, a.dim, i_first, q_begin, q_end, thread);
            next_do.load(do_base, a.d_out.row, a.dim, i_first, q_begin, q_end, thread);
            for (int i0 = i_first; i0 < q_end; i0 += kRows) {
                __syncthreads();
                next_q.store(s_q, thread);
                next_do.store(s_do, thread);
                if (thread < kRows) {
                    const int i = i0 + thread;
                    const bool in = i < q_end;
                    const float2 st = in ? a.stats[stat + i] : make_float2(0.0f, INFINITY);
                    s_m[thread] = st.x;
                    s_log_l[thread] = st.y;
                    s_delta[thread] = in ? a.delta[stat + i] : 0.0f;
                    s_time[thread] = in && sc.q_times ? sc.q_times[i] : 0.0f;
                    s_diag[thread] = in ? a.q_info[i].z : 0;
                }
                __syncthreads();
                if (i0 + kRows < q_end) {
                    next_q.load(q_base, a.q.row, a.dim, i0 + kRows, q_begin, q_end, thread);
                    next_do.load(do_base, a.d_out.row, a.dim, i0 + kRows, q_begin, q_end, thread);
                }
                if (i0 >= w_hi || i0 + kRows <= w_lo) continue;

                f32x16 x16 = zero16(), dp = zero16();
#pragma unroll
                for (int st = 0; st < G::kSteps; ++st) {
                    x16 = mma(G::row(s_q, lane & 31, st, half), k[st], x16);
                    dp = mma(G::row(s_do, lane & 31, st, half), v[st], dp);
                }
                float x[16], cap_slope[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = x16[r];
                score_block<T>(sc, x, cap_slope);
                if (sc.table) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int d = s_diag[acc_row(r) + 4 * half] - j;
                        x[r] += s_lut[min(max(d, -sc.reach), sc.reach) + sc.reach];
                    }
                }
                if (sc.slopes) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int at = acc_row(r) + 4 * half;
                        const float gap = sc.k_times ? s_time[at] - k_time
                                                     : static_cast<float>(s_diag[at] - j);
                        x[r] = fmaf(-slope, fabsf(gap), x[r]);
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = acc_row(r) + 4 * half;
                    x[r] = exp2_fast((x[r] - s_m[at]) - s_log_l[at]);
                }
                float ds[16];
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    ds[r] = x[r] * (dp[r] - s_delta[acc_row(r) + 4 * half]);
                if (i0 < full_lo || i0 + kRows > full_hi) {
                    const unsigned span = static_cast<unsigned>(last - first);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int i = i0 + acc_row(r) + 4 * half;
                        if (static_cast<unsigned>(i - first) >= span) x[r] = ds[r] = 0.0f;
                    }
                }
                if (sc.softcap > 0) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] *= cap_slope[r];
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    Frag<T> p, s;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        p[e] = static_cast<T>(x[8 * t + e]);
                        s[e] = static_cast<T>(ds[8 * t + e]);
                    }
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        dv[b] = mma(G::columns(s_do, 16 * t, b, lane), p, dv[b]);
                        dk[b] = mma(G::columns(s_q, 16 * t, b, lane), s, dk[b]);
                    }
                }
            }
        }
        if (j < a.k_rows && (only < 0 || (any && doc == only))) {
            if (a.splits > 1) {
                const int64_t at =
                    ((static_cast<int64_t>(split) * a.k_rows + j) * kv_heads + kv_head) * a.dim;
                store_row<float, DB>(a.part_k + at, dk, any, sc.scale, a.dim, half);
                store_row<float, DB>(a.part_v + at, dv, any, 1.0f, a.dim, half);
            } else {
                store_row<T, DB>(row_of<T>(a.d_k, j, kv_head), dk, any, sc.scale, a.dim,
                                 half);
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
        q_end = only;
#pragma unroll
        for (int w = 0; w < 4; ++w) q_begin = min(q_begin, s_reduce[w][1]);
        i_first += (q_begin - i_first) / kRows * kRows;  // the same tiles: the same bits
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
    uint64_t delta, partial, part_k, part_v, bytes;
};
Layout layout_of(const trw_attention_params& p) {
    Layout l;
    uint64_t at = 0;
    auto take = [&](uint64_t floats) {
        const uint64_t here = at;
        at += align256(floats * sizeof(float));
        return here;
    };
    l.delta = take(static_cast<uint64_t>(p.heads) * p.q_rows);
    l.partial = take(p.score.table ? static_cast<uint64_t>(p.heads) * tiles_of(p.q_rows) *
                                         p.score.num_buckets
                                   : 0);
    const int splits = splits_of(p);
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
    a.d_out = make_rows(p.d_out);
    a.d_q = make_rows(p.d_q);
    a.d_k = make_rows(p.d_k);
    a.d_v = make_rows(p.d_v);
    a.q_info = reinterpret_cast<const int4*>(p.q_rows_info);
    a.k_info = reinterpret_cast<const int2*>(p.k_rows_info);
    a.stats = reinterpret_cast<const float2*>(p.stats);
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
    const size_t line = p.score.table ? (2 * a.score.reach + 1) * sizeof(float) : 0;
    dispatch(p.dtype, p.dim, [&](auto t, auto db) {
        typedef decltype(t) T;
        constexpr int DB = decltype(db)::value;
        if (a.q_tiles)
            hipLaunchKernelGGL(
                (attention_backward_q_kernel<T, DB>),
                dim3(static_cast<unsigned>(xcd_grid(static_cast<int64_t>(a.q_tiles) * a.heads))),
                dim3(kThreads), 9 * line, stream, a);
        check_launch("attention_backward");
        if (a.k_tiles)
            hipLaunchKernelGGL((attention_backward_kv_kernel<T, DB>),
                               dim3(static_cast<unsigned>(xcd_grid(
                                   static_cast<int64_t>(a.k_tiles) * p.kv_heads * a.splits))),
                               dim3(kThreads), line, stream, a);
        check_launch("attention_backward");
        if (a.k_tiles && a.splits > 1) {
            const int64_t n = p.k_rows * p.kv_heads * (p.dim / 4);
            hipLaunchKernelGGL((join_splits_kernel<T>),
                               dim3(static_cast<unsigned>((n + kThreads - 1) / kThreads)),
                               dim3(kThreads), 0, stream, a);
            check_launch("attention_backward");
        }
    });
    if (p.score.table) {
        join_table(a.partial, a.q_tiles, p.heads, p.score.num_buckets, TRW_F32, p.d_table, stream);
    }
}

}  // namespace ops
}  // namespace trw
