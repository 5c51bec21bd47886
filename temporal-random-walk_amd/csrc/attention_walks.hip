// attention_walks.hip -- attention.hip's formula, forward and backward, for
// walks short enough that one wave holds all their scores.
//
// The walks that the sampler makes have tens of events.  Their attention is
// bound by the memory that q, k, v and the outputs move, if enough of it is on
// its way: tiles of 128 rows that several walks share spend their time in
// barriers, in masking other walks' keys and in waiting for one tile after the
// next.  Here a wave takes one walk and key head by itself: its keys and values
// (up to 32 kNB of them) lie in LDS, all scores of 32 query rows in registers,
// and there is no barrier, no running maximum and, in the backward pass, one
// computation of the scores for all gradients (five products instead of seven)
// and no reading of the output: D_i = sum_j P_ij dP_ij is summed from the same
// registers, in float32, which is also more exact than dO . o of a rounded o.
//
// P and dS are needed both with a lane per query row (for dq, as the registers
// hold them) and with a lane per key (for dk and dv): they go through 2 KB
// squares of LDS in the inputs' type and are read back transposed.
//
// 20000 walks of up to 80 rows (8 heads of 64, bfloat16) take 1.00 ms forward (4.9
// TB/s of the rows' and the padding's bytes; a large copy reaches as much) and 2.6
// backward (by length).
#include <algorithm>

#include "operators.h"

namespace trw {
namespace ops {
namespace {

struct WalkArgs {
    Rows q, k, v, out, d_out, d_q, d_k, d_v;
    const int4* docs;  // two per document: q begin, len, rows, k begin | k len, rows, prefix, kind
    float* stats;      // as attention.hip writes them
    float* partial;    // backward: [heads, docs, stride] dS by distance
    int stride;
    Score score;
    int heads, kv_heads, group, dim;
    int q_rows;
    int doc_count;
    int limit;     // this launch's walks: up to so many rows
    int above;     // backward: and more than these
    int last;      // backward: no launch takes longer ones
    int triangle;  // backward: a causal walk over its own keys has no tiles above the diagonal
    int time_at;   // backward: where in LDS the floats begin, in 16 bytes
};

struct Doc {
    int q_begin, q_len, q_rows, k_begin, k_len, k_rows, prefix, kind;

    // Keys that local query row i sees: [0, seen).
    __device__ __forceinline__ int seen(int i) const {
        const int past = min(max(k_len - q_len + i + 1, 0), k_len);
        return kind == TRW_MASK_FULL ? k_len
                                     : max(past, kind == TRW_MASK_PREFIX ? prefix : 0);
    }
    // The first local query row that sees key j.
    __device__ __forceinline__ int first(int j) const {
        if (kind == TRW_MASK_FULL || (kind == TRW_MASK_PREFIX && j < prefix)) return 0;
        return min(max(j - (k_len - q_len), 0), q_len);
    }
};

// Consecutive workgroups go to the eight XCDs in turn: each takes all key heads
// of a walk, whose rows lie side by side.
__device__ __forceinline__ int head_of(const WalkArgs& a, int id) { return id / 8 % a.kv_heads; }
__device__ __forceinline__ int doc_of(const WalkArgs& a, int id) {
    return id / (8 * a.kv_heads) * 8 + id % 8;
}
__device__ __forceinline__ Doc load_doc(const int4* docs, int doc) {
    const int4 a = docs[2 * doc], b = docs[2 * doc + 1];
    Doc d;
    d.q_begin = __builtin_amdgcn_readfirstlane(a.x);
    d.q_len = __builtin_amdgcn_readfirstlane(a.y);
    d.q_rows = __builtin_amdgcn_readfirstlane(a.z);
    d.k_begin = __builtin_amdgcn_readfirstlane(a.w);
    d.k_len = __builtin_amdgcn_readfirstlane(b.x);
    d.k_rows = __builtin_amdgcn_readfirstlane(b.y);
    d.prefix = __builtin_amdgcn_readfirstlane(b.z);
    d.kind = __builtin_amdgcn_readfirstlane(b.w);
    return d;
}

// Zeros in rows [from, to) of one head, which nobody else writes.
template <typename T, int DB>
__device__ __forceinline__ void zero_rows(const Rows& r, int64_t begin, int from, int to, int head,
                                          int dim, int lane) {
    typedef Tile<T, DB> G;
    static_assert(G::kUsed <= 64, "a row at a time at least");
    constexpr int kRows = 64 / G::kUsed;  // at a time
    const int col = lane % G::kUsed * G::kElems;
    if (col >= dim || lane >= kRows * G::kUsed) return;
    T* row = row_of<T>(r, begin + from + lane / G::kUsed, head) + col;
    for (int i = from + lane / G::kUsed; i < to; i += kRows, row += kRows * r.row)
        *reinterpret_cast<u32x4*>(row) = u32x4{0, 0, 0, 0};
}

// A row as B operands, as load_operand, of a row that is there: columns from
// `dim` on are zeros.
template <typename T, int DB>
__device__ __forceinline__ void load_whole_operand(Frag<T> (&f)[2 * DB], const T* row, int dim,
                                                   int half) {
    typedef Tile<T, DB> G;
#pragma unroll
    for (int s = 0; s < 2 * DB; ++s) {
        union {
            u32x4 u[sizeof(T) / 2];
            Frag<T> f;
        } x;
        const int col = 16 * s + 8 * half < dim ? 16 * s + 8 * half : 0;
#pragma unroll
        for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h)
            x.u[h] = *reinterpret_cast<const u32x4*>(row + col + h * G::kElems);
        f[s] = x.f;
    }
    if (dim < 32 * DB) {
#pragma unroll
        for (int s = 0; s < 2 * DB; ++s)
            if (16 * s + 8 * half >= dim) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[s][e] = static_cast<T>(0.0f);
            }
    }
}

// Byte of elements 8 g + 4 half .. + 4 of a row of a tile.
template <typename G, typename T>
__device__ __forceinline__ int four_at(int row, int g, int half) {
    if (sizeof(T) == 4) return G::slot(row, 2 * g + half) * 16;
    return G::slot(row, g) * 16 + half * 8;
}

// A block's accumulators (a column each a row of the output) as rows of global
// memory, times `by`, zeros where a lane's row has nothing: through a tile of
// the wave's own in LDS, so that a store instruction writes whole rows and not
// 16 bytes of each of 32.
template <typename T, int DB>
__device__ __forceinline__ void store_rows(u32x4* tile, const f32x16 (&acc)[DB], bool any, float by,
                                           const Rows& r, int64_t begin, int count, int head,
                                           int dim, int lane) {
    typedef Tile<T, DB> G;
    typedef T t4 __attribute__((ext_vector_type(4)));
    const int half = lane >> 5;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            t4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = static_cast<T>(any ? acc[b][4 * g + e] * by : 0.0f);
            *reinterpret_cast<t4*>(reinterpret_cast<char*>(tile) +
                                   four_at<G, T>(lane & 31, 4 * b + g, half)) = v;
        }
    T* base = row_of<T>(r, begin, head);
#pragma unroll
    for (int n = 0; n < (32 * G::kUsed + 63) / 64; ++n) {
        const int at = lane + 64 * n, row = at / G::kUsed, col = at % G::kUsed * G::kElems;
        if (row < count && col < dim)
            *reinterpret_cast<u32x4*>(base + row * r.row + col) = tile[G::slot(row, at % G::kUsed)];
    }
}

// All copies of this wave have landed (the tiles are the wave's own).
__device__ __forceinline__ void wave_landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    asm volatile("" ::: "memory");
}

// Distances in a walk of at most 32 kNB keys and queries: the line of biases
// needs no more of the table's reach than that.
template <int kNB>
__device__ __forceinline__ int walk_reach(const Score& sc) {
    return min(sc.reach, 32 * kNB);
}
template <int kNB>
__device__ __forceinline__ void fill_walk_bias(float* lut, const Score& sc, int head, int lane) {
    const int reach = walk_reach<kNB>(sc);
    for (int n = lane; n < 2 * reach + 1; n += 64)
        lut[n] = table_entry(sc, head, n - reach + sc.reach);
}

template <typename T, int DB, int kNB>
__global__ __launch_bounds__(64, DB < 3 ? 2 : 1) void walk_forward_kernel(WalkArgs a) {
    typedef Tile<T, DB> G;
    constexpr int kBlock = 32 * G::kSlots;
    __shared__ u32x4 s_v[kNB * kBlock], s_out[kBlock];
    __shared__ float s_time[128];
    __shared__ float s_lut[64 * kNB + 1];

    int lane = threadIdx.x;
    const int kv_head = head_of(a, blockIdx.x), doc = doc_of(a, blockIdx.x);
    if (doc >= a.doc_count) return;
    const Doc d = load_doc(a.docs, doc);
    if (max(d.q_len, d.k_len) > a.limit) return;  // the tiles' kernel has it
    const int first_head = kv_head * a.group;
    Score sc = a.score;
    sc.reach = walk_reach<kNB>(sc);

    const int q_blocks = (d.q_len + 31) / 32, k_blocks = (d.k_len + 31) / 32;
    const int steps = q_blocks * a.group;
    // Keys stay in registers for all query rows and heads, values, which are
    // read transposed, in LDS.
    Frag<T> k[kNB][G::kSteps], q[G::kSteps], next[G::kSteps];
    auto load_q = [&](Frag<T>(&f)[G::kSteps], int step) {
        const int i = min(step % q_blocks * 32 + (lane & 31), d.q_len - 1);
        load_whole_operand<T, DB>(
            f, row_of<const T>(a.q, d.q_begin + i, first_head + step / q_blocks), a.dim, lane >> 5);
    };
    if (steps > 0 && k_blocks > 0) {
#pragma unroll
        for (int b = 0; b < kNB; ++b)
            if (b < k_blocks)
                load_whole_operand<T, DB>(
                    k[b],
                    row_of<const T>(a.k, d.k_begin + min(32 * b + (lane & 31), d.k_len - 1), kv_head),
                    a.dim, lane >> 5);
        const Loader<T, DB, 32, 64> v_load(a.v.row, a.dim, lane);
        const T* v_base = row_of<const T>(a.v, d.k_begin, kv_head);
        for (int b = 0; b < k_blocks; ++b)
            v_load.load(v_base, 32 * b, 0, d.k_len, lds_address(s_v) + b * kBlock * 16, lane);
        if (sc.k_times)
            for (int j = 0; j < d.k_len; j += 64)
                load_floats(sc.k_times + d.k_begin, j, 0, d.k_len, lds_address(s_time) + j * 4,
                            lane);
        load_q(next, 0);
    }
    for (int step = 0; step < steps; ++step) {
        const int head = first_head + step / q_blocks, i0 = step % q_blocks * 32;
        // What follows from the lane is worked out for every step: held over the
        // loop, it would take the registers that the scores need.
        asm volatile("" : "+v"(lane));
        const int half = lane >> 5;
        if (sc.table && i0 == 0) fill_walk_bias<kNB>(s_lut, a.score, head, lane);
#pragma unroll
        for (int s = 0; s < G::kSteps; ++s) q[s] = next[s];
        if (k_blocks > 0) {
            if (step == 0) wave_landed();
            if (step + 1 < steps) load_q(next, step + 1);
        }
        const int i = i0 + (lane & 31);
        const bool in = i < d.q_len;
        const int row = min(i, d.q_len - 1);  // rows past the walk's end are not stored
        const int seen = d.seen(row);
        const int least = d.seen(i0), most = d.seen(min(i0 + 31, d.q_len - 1));
        const int diag = d.k_len - d.q_len + row;
        const int diag_lo = d.k_len - d.q_len + i0, diag_hi = diag_lo + 31;
        const float slope = sc.slopes ? sc.slopes[head] * kLog2e : 0.0f;
        const float q_time = sc.q_times ? sc.q_times[d.q_begin + row] : 0.0f;

        float s[kNB][1][16];
        float m = kFloor;
#pragma unroll
        for (int b = 0; b < kNB; ++b) {
            if (32 * b >= most) continue;
            f32x16 x = zero16();
#pragma unroll
            for (int st = 0; st < G::kSteps; ++st)
                x = mma(k[b][st], q[st], x);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][0][r] = x[r];
            cap_scores<T>(sc, s[b]);
            add_biases(sc, s[b], s_lut, slope, diag, diag_lo, diag_hi, q_time, s_time + 32 * b,
                       32 * b, half);
            if (32 * b + 32 > least) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * b + acc_row(r) + 4 * half >= seen) s[b][0][r] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) m = fmaxf(m, s[b][0][r]);
        }
        m = fmaxf(m, __shfl_xor(m, 32));
        float l = 0.0f;
        f32x16 o[DB];
#pragma unroll
        for (int c = 0; c < DB; ++c) o[c] = zero16();
#pragma unroll
        for (int b = 0; b < kNB; ++b) {
            if (32 * b >= most) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[b][0][r] = exp2_fast(s[b][0][r] - m);
                l += s[b][0][r];
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag<T> p;
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = static_cast<T>(s[b][0][8 * t + e]);
#pragma unroll
                for (int c = 0; c < DB; ++c)
                    o[c] = mma(G::columns(s_v + b * kBlock, 16 * t, c, lane), p, o[c]);
            }
        }
        l += __shfl_xor(l, 32);
        {
            const bool any = l != 0.0f;
            store_rows<T, DB>(s_out, o, any, 1.0f / l, a.out, d.q_begin + i0, d.q_len - i0, head,
                              a.dim, lane);
            if (a.stats && in && half == 0) {
                const int64_t at = static_cast<int64_t>(head) * a.q_rows + d.q_begin + i;
                const float log_l = any ? __builtin_amdgcn_logf(l) : INFINITY;
                a.stats[at] = sc.biased() ? m : m + log_l;
                if (sc.biased()) a.stats[static_cast<int64_t>(a.heads) * a.q_rows + at] = log_l;
            }
        }
    }
    for (int h = first_head; h < first_head + a.group; ++h)
        zero_rows<T, DB>(a.out, d.q_begin, d.q_len, d.q_rows, h, a.dim, lane);
}

// Backward: a wave for each 32 rows of the walk.  First the wave owns query
// rows: scores, P, dP, D and dq.  Then, P and dS having gone through LDS, it
// owns keys: dk and dv.  Of a causal walk's blocks the first wave has the fewest
// in the first half and the most in the second, the last wave the other way
// round.  P and dS lie where the keys and values were.
template <typename T, int DB, int kNB, bool kShared>
__global__ __launch_bounds__(64 * kNB, kShared && (DB * kNB > (sizeof(T) == 4 ? 2 : 4) || DB == 4) ? 1
                                                                              : 2) void walk_backward_kernel(WalkArgs a) {
    typedef Tile<T, DB> G;
    typedef Tile<T, 1> S;  // P and dS of a block: rows of queries, columns of keys
    constexpr int kBlock = 32 * G::kSlots;
    constexpr int kTile = 32 * S::kSlots;
    extern __shared__ u32x4 s_mem[];

    int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv_head = head_of(a, blockIdx.x), doc = doc_of(a, blockIdx.x);
    if (doc >= a.doc_count) return;
    const Doc d = load_doc(a.docs, doc);
    const int first_head = kv_head * a.group;
    Score sc = a.score;
    sc.reach = walk_reach<kNB>(sc);
    const int line = 2 * sc.reach + 1;
    if (max(d.q_len, d.k_len) <= a.above) return;  // another launch has it
    if (max(d.q_len, d.k_len) > a.limit) {  // another launch or the tiles' kernels have it
        if (sc.table && a.last)
            for (int h = first_head; h < first_head + a.group; ++h)
                for (int n = threadIdx.x; n < a.stride; n += 64 * kNB)
                    a.partial[(static_cast<int64_t>(h) * a.doc_count + doc) * a.stride + n] = 0.0f;
        return;
    }
    const uint32_t at_mem = lds_address(s_mem);
    u32x4* s_q = s_mem;
    u32x4* s_do = s_q + kNB * kBlock;
    u32x4* s_k = s_do + kNB * kBlock;
    u32x4* s_v = s_k + kNB * kBlock;
    u32x4* s_p = s_k;  // [tiles][P, dS]
    float* s_time = reinterpret_cast<float*>(s_mem + a.time_at);  // 64 kNB
    float* s_lut = s_time + 64 * kNB;
    float* s_sum = s_lut + line + wave * line;
    float* s_square = s_lut + (1 + kNB) * line + wave * kSquare;

    const int q_blocks = (d.q_len + 31) / 32, k_blocks = (d.k_len + 31) / 32;
    // the tile of query block q and key block k
    auto tile_of = [&](int q, int k) {
        return s_p + (a.triangle ? q * (q + 1) / 2 + k : q * kNB + k) * 2 * kTile;
    };
    auto most_of = [&](int q) { return d.seen(min(32 * q + 31, d.q_len - 1)); };
    const bool q_mine = wave < q_blocks && k_blocks > 0;
    const int i0 = 32 * wave;
    const int least = i0 + 32 <= d.q_len ? d.seen(i0) : 0;
    const int most = q_mine ? most_of(wave) : 0;
    const int diag_lo = d.k_len - d.q_len + i0, diag_hi = diag_lo + 31;

    const T* k_base = row_of<const T>(a.k, d.k_begin, kv_head);
    const T* v_base = row_of<const T>(a.v, d.k_begin, kv_head);
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int c = 0; c < DB; ++c) {
        dk[c] = zero16();
        dv[c] = zero16();
    }
    if (sc.table)
        for (int n = lane; n < kSquare; n += 64) s_square[n] = 0.0f;

    const int heads = q_blocks > 0 && k_blocks > 0 ? (kShared ? a.group : 1) : 0;
#pragma unroll 1
    for (int g = 0; g < heads; ++g) {
        const int head = first_head + g;
        // What follows from the lane is worked out for every head: held over
        // the loop, it would take the registers that the scores need.
        if (kShared) asm volatile("" : "+v"(lane));
        const int half = lane >> 5;
        const int i = i0 + (lane & 31);
        const bool in = i < d.q_len;
        const int row = min(i, d.q_len - 1);
        const int seen = in && q_mine ? d.seen(row) : 0;  // rows past the end have no part in dk, dv
        const int diag = d.k_len - d.q_len + row;
        if (kShared && g) __syncthreads();  // the head before is done with its tiles
        if (q_mine) {
            const Loader<T, DB, 32, 64> q_load(a.q.row, a.dim, lane);
            const Loader<T, DB, 32, 64> do_load(a.d_out.row, a.dim, lane);
            q_load.load(row_of<const T>(a.q, d.q_begin, head), i0, 0, d.q_len,
                        at_mem + wave * kBlock * 16, lane);
            do_load.load(row_of<const T>(a.d_out, d.q_begin, head), i0, 0, d.q_len,
                         at_mem + (kNB + wave) * kBlock * 16, lane);
        }
        if (wave < k_blocks) {
            const Loader<T, DB, 32, 64> k_load(a.k.row, a.dim, lane), v_load(a.v.row, a.dim, lane);
            k_load.load(k_base, 32 * wave, 0, d.k_len, at_mem + (2 * kNB + wave) * kBlock * 16,
                        lane);
            v_load.load(v_base, 32 * wave, 0, d.k_len, at_mem + (3 * kNB + wave) * kBlock * 16,
                        lane);
            if (sc.k_times)
                load_floats(sc.k_times + d.k_begin, 32 * wave, 0, d.k_len,
                            at_mem + a.time_at * 16 + 128 * wave, lane);
        }
        float m = 0.0f, log_l = 0.0f, q_time = 0.0f;
        if (q_mine) {
            const int64_t at = static_cast<int64_t>(head) * a.q_rows + d.q_begin + row;
            m = a.stats[at];
            if (sc.biased()) log_l = a.stats[static_cast<int64_t>(a.heads) * a.q_rows + at];
            if (sc.q_times) q_time = sc.q_times[d.q_begin + row];
        }
        const float slope = sc.slopes ? sc.slopes[head] * kLog2e : 0.0f;
        if (sc.table) {
            if (wave == 0) fill_walk_bias<kNB>(s_lut, a.score, head, lane);
            for (int n = lane; n < line; n += 64) s_sum[n] = 0.0f;
        }
        landed();

        Frag<T> ps[kNB][2], dss[kNB][2];  // P and dS of this wave's rows
        if (q_mine) {
            Frag<T> q[G::kSteps], d_o[G::kSteps];
#pragma unroll
            for (int st = 0; st < G::kSteps; ++st) {
                q[st] = G::row(s_q + wave * kBlock, lane & 31, st, half);
                d_o[st] = G::row(s_do + wave * kBlock, lane & 31, st, half);
            }
            // columns from dim on hold copies of others: zeros on this side
            if (a.dim < 32 * DB) {
#pragma unroll
                for (int st = 0; st < G::kSteps; ++st)
                    if (16 * st + 8 * half >= a.dim) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) q[st][e] = d_o[st][e] = static_cast<T>(0.0f);
                    }
            }
            // P and dP of every key, and D
            float p[kNB][16], dp[kNB][16];
            float delta = 0.0f;
#pragma unroll
            for (int b = 0; b < kNB; ++b) {
                if (32 * b >= most) continue;
                f32x16 x = zero16(), y = zero16();
#pragma unroll
                for (int st = 0; st < G::kSteps; ++st) {
                    x = mma(G::row(s_k + b * kBlock, lane & 31, st, half), q[st], x);
                    y = mma(G::row(s_v + b * kBlock, lane & 31, st, half), d_o[st], y);
                }
                float s[1][16];
#pragma unroll
                for (int r = 0; r < 16; ++r) s[0][r] = x[r];
                cap_scores<T>(sc, s);
                if (sc.biased()) {
                    add_biases(sc, s, s_lut, slope, diag, diag_lo, diag_hi, q_time,
                               s_time + 32 * b, 32 * b, half);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[0][r] = (s[0][r] - m) - log_l;
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[0][r] -= m;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    p[b][r] = exp2_fast(s[0][r]);
                    dp[b][r] = y[r];
                }
                if (32 * b + 32 > least) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (32 * b + acc_row(r) + 4 * half >= seen) p[b][r] = dp[b][r] = 0.0f;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) delta = fmaf(p[b][r], dp[b][r], delta);
            }
            delta += __shfl_xor(delta, 32);

            f32x16 dq[DB];
#pragma unroll
            for (int c = 0; c < DB; ++c) dq[c] = zero16();
#pragma unroll
            for (int b = 0; b < kNB; ++b) {
                if (32 * b >= most) continue;
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[b][r] = p[b][r] * (dp[b][r] - delta);
                if (sc.table)
                    add_diagonals(dp[b], s_square, s_sum, sc.reach, diag_lo - 32 * b,
                                  diag_hi - 32 * b, lane, half);
                if (sc.softcap > 0) {
                    // the cap's slope once more from the products, which costs
                    // less than holding it
                    f32x16 x = zero16();
#pragma unroll
                    for (int st = 0; st < G::kSteps; ++st)
                        x = mma(G::row(s_k + b * kBlock, lane & 31, st, half), q[st], x);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float cap_slope;
                        (void)capped<T, false>(sc, x[r], cap_slope);
                        dp[b][r] *= cap_slope;
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        ps[b][t][e] = static_cast<T>(p[b][8 * t + e]);
                        dss[b][t][e] = static_cast<T>(dp[b][8 * t + e]);
                    }
#pragma unroll
                    for (int c = 0; c < DB; ++c)
                        dq[c] = mma(G::columns(s_k + b * kBlock, 16 * t, c, lane), dss[b][t], dq[c]);
                }
            }
            if (in)
                store_row<T, DB>(row_of<T>(a.d_q, d.q_begin + i, head), dq, seen > 0, sc.scale,
                                 a.dim, half);
        }
        __syncthreads();  // keys and values are done with: P and dS take their place
        if (q_mine) {
            typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int b = 0; b < kNB; ++b) {
                if (32 * b >= most) continue;
                char* at = reinterpret_cast<char*>(tile_of(wave, b));
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int byte = four_at<S, T>(lane & 31, c, half);
                    t4 vp, vs;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        vp[e] = ps[b][c >> 1][4 * (c & 1) + e];
                        vs[e] = dss[b][c >> 1][4 * (c & 1) + e];
                    }
                    *reinterpret_cast<t4*>(at + byte) = vp;
                    *reinterpret_cast<t4*>(at + kTile * 16 + byte) = vs;
                }
            }
        }
        __syncthreads();
        if (wave < k_blocks) {
#pragma unroll
            for (int b = 0; b < kNB; ++b) {
                if (b >= q_blocks || 32 * wave >= most_of(b)) continue;
                const u32x4* at = tile_of(b, wave);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const Frag<T> pt = S::columns(at, 16 * t, 0, lane);
                    const Frag<T> st = S::columns(at + kTile, 16 * t, 0, lane);
#pragma unroll
                    for (int c = 0; c < DB; ++c) {
                        dv[c] = mma(G::columns(s_do + b * kBlock, 16 * t, c, lane), pt, dv[c]);
                        dk[c] = mma(G::columns(s_q + b * kBlock, 16 * t, c, lane), st, dk[c]);
                    }
                }
            }
        }
        if (sc.table) {  // the waves' sums, by the first (they are in: two barriers ago)
            float* out = a.partial + (static_cast<int64_t>(head) * a.doc_count + doc) * a.stride;
            for (int n = threadIdx.x; n < a.stride; n += 64 * kNB) {
                const int at = n - (a.stride - line) / 2;
                float sum = 0.0f;
                if (at >= 0 && at < line) {
#pragma unroll
                    for (int w = 0; w < kNB; ++w) sum += s_lut[(1 + w) * line + at];
                }
                out[n] = sum;
            }
        }
    }
    const int j = 32 * wave + (lane & 31);
    __syncthreads();  // queries are done with
    {
        const bool any = heads > 0 && d.first(j) < d.q_len;
        u32x4* s_out = s_q + wave * kBlock;
        store_rows<T, DB>(s_out, dk, any, sc.scale, a.d_k, d.k_begin + i0, d.k_len - i0, kv_head,
                          a.dim, lane);
        store_rows<T, DB>(s_out, dv, any, 1.0f, a.d_v, d.k_begin + i0, d.k_len - i0, kv_head, a.dim,
                          lane);
    }
    if (wave == 0) zero_rows<T, DB>(a.d_k, d.k_begin, d.k_len, d.k_rows, kv_head, a.dim, lane);
    if (wave == kNB - 1) zero_rows<T, DB>(a.d_v, d.k_begin, d.k_len, d.k_rows, kv_head, a.dim, lane);
    for (int h = first_head; h < first_head + a.group; ++h) {
        // queries over no keys at all, and padding
        if (wave == kNB / 2)
            zero_rows<T, DB>(a.d_q, d.q_begin, heads > 0 ? d.q_len : 0, d.q_rows, h, a.dim, lane);
        if (sc.table && heads == 0)
            for (int n = threadIdx.x; n < a.stride; n += 64 * kNB)
                a.partial[(static_cast<int64_t>(h) * a.doc_count + doc) * a.stride + n] = 0.0f;
    }
}

WalkArgs make_args(const trw_attention_params& p) {
    WalkArgs a;
    a.q = make_rows(p.q);
    a.k = make_rows(p.k);
    a.v = make_rows(p.v);
    a.out = make_rows(p.out);
    a.d_out = make_rows(p.d_out);
    a.d_q = make_rows(p.d_q);
    a.d_k = make_rows(p.d_k);
    a.d_v = make_rows(p.d_v);
    a.docs = reinterpret_cast<const int4*>(p.docs_info);
    a.stats = p.stats;
    a.partial = nullptr;
    a.stride = 0;
    a.score = make_score(p.score);
    a.heads = p.heads;
    a.kv_heads = p.kv_heads;
    a.group = p.heads / p.kv_heads;
    a.dim = p.dim;
    a.q_rows = static_cast<int>(p.q_rows);
    a.doc_count = static_cast<int>(p.docs);
    a.above = -1;
    a.limit = 0;
    a.last = 1;
    a.triangle = 0;
    a.time_at = 0;
    return a;
}

// Whether the backward pass goes by the length of walks, a launch for each number
// of blocks of 32 rows.  A workgroup has a wave and 16 KB of LDS or more for each
// block that a walk may have, and walks that have fewer leave them idle; a launch
// costs each walk that is not its own a workgroup that reads its length and ends.
// Backward alone, walks of up to 80 (8 key heads of 64, bfloat16): 8192 of them
// 1155 us in one launch and 1058 by length, 2048 of them 295 and 301; walks of 50
// to 60 in one of two launches: 1595 and 1635.  Packed walks of up to 40 (2 key
// heads), of which the host knows the mean alone: 8192 of them 677 and 560 us,
// 2048 203 and 161, 512 86 and 117.  Other head sizes and counts go by the same rule,
// unmeasured.  (The forward pass, whose workgroups are one
// wave either way: 435 and 484, 185 and 194 us; it has one launch.)
bool by_length(const trw_attention_params& p) {
    return p.docs * p.kv_heads >= (p.longest > 0 ? 65536 : 2048);
}

// f<T, DB, NB>() for the walks that go a wave each: up to 96 rows at head sizes
// to 64, up to 64 rows at larger ones.
template <typename F>
void walk_dispatch(int dtype, int dim, int blocks, F&& f) {
    auto by_blocks = [&](auto t, auto db, auto most) {
        if (blocks == 1) {
            f(t, db, std::integral_constant<int, 1>());
            return;
        }
        if constexpr (decltype(most)::value >= 2)
            if (blocks == 2) f(t, db, std::integral_constant<int, 2>());
        if constexpr (decltype(most)::value >= 3)
            if (blocks == 3) f(t, db, std::integral_constant<int, 3>());
    };
    auto by_dim = [&](auto t) {
        switch ((dim + 31) / 32) {
            case 1: by_blocks(t, std::integral_constant<int, 1>(), std::integral_constant<int, 3>()); break;
            case 2: by_blocks(t, std::integral_constant<int, 2>(), std::integral_constant<int, 3>()); break;
            case 3: by_blocks(t, std::integral_constant<int, 3>(), std::integral_constant<int, 2>()); break;
            default: by_blocks(t, std::integral_constant<int, 4>(), std::integral_constant<int, 2>()); break;
        }
    };
    if (dtype == TRW_F32)
        by_dim(float{});
    else if (dtype == TRW_F16)
        by_dim(_Float16{});
    else
        by_dim(__bf16{});
}

}  // namespace

// Blocks of 32 rows that walks of this batch may have to go a wave each; 0: the
// batch is the tiles' kernels' alone.  Lengths are the device's; the host
// knows the padded length, or the mean of packed walks, whose double should
// fit.  Longer walks of such a batch still go to the tiles.
//
// Where many walks have a few rows each, most of a wave's 32 columns would be
// idle, and tiles that several walks share are better: 8192 walks (8 heads of 64
// over 4 key heads, a bias, bfloat16), forward and backward, take 426 us with a
// wave each and 185 with tiles at 4 rows, 457 and 371 at 8, 504 and 708 at 12; in
// float32 at head size 128, 3.7 and 1.2 ms at 4 rows, 3.8 and 2.3 at 8, 3.9 and
// 4.0 at 12.  64 such walks of 4 rows, which do not fill the device either way,
// take 105 and 169 us there.
//
// Wide caps of the 16-bit types, which nobody's scores come near, are the tiles'
// too: their kernels for those would be as many again.
constexpr int64_t kTinyRows = 8;
constexpr int64_t kTinyGroups = 2048;

int walk_blocks(const trw_attention_params& p) {
    if (p.docs == 0 || wide_cap(p.dtype, p.score)) return 0;
    const int db = (p.dim + 31) / 32;
    const int most = db <= 2 ? 3 : 2;
    const int64_t rows = std::max(p.q_rows, p.k_rows);
    const int64_t mean = (rows + p.docs - 1) / p.docs;
    const int64_t length = p.longest > 0 ? p.longest : 2 * mean;
    if (mean <= kTinyRows && p.docs * p.kv_heads >= kTinyGroups) return 0;
    if (mean > 32 * most || (p.longest > 0 && p.longest > 32 * most)) return 0;
    return static_cast<int>(std::min<int64_t>(std::max<int64_t>((length + 31) / 32, 1), most));
}

// Workgroups over walks and key heads.
int64_t walk_grid(const trw_attention_params& p) { return (p.docs + 7) / 8 * 8 * p.kv_heads; }

// Whether walks longer than those can be in the batch, or rows of no walk, which
// the tiles' kernels leave zero.
bool walk_rest(const trw_attention_params& p, int blocks) {
    return !p.covered || p.longest <= 0 || p.longest > 32 * blocks;
}

void walk_forward(const trw_attention_params& p, int blocks, hipStream_t stream) {
    WalkArgs a = make_args(p);
    a.limit = 32 * blocks;
    const unsigned grid = static_cast<unsigned>(walk_grid(p));
    walk_dispatch(p.dtype, p.dim, blocks, [&](auto t, auto db, auto nb) {
        hipLaunchKernelGGL(
            (walk_forward_kernel<decltype(t), decltype(db)::value, decltype(nb)::value>),
            dim3(grid), dim3(64), 0, stream, a);
    });
    check_launch("walk_forward");
}

int walk_line(const trw_attention_params& p, int blocks) {
    return 2 * std::min(p.score.reach, 32 * blocks) + 1;
}

void walk_backward(const trw_attention_params& p, int blocks, float* partial, hipStream_t stream) {
    WalkArgs a = make_args(p);
    a.partial = partial;
    a.stride = walk_line(p, blocks);
    a.triangle = p.own_causal;
    const unsigned grid = static_cast<unsigned>(walk_grid(p));
    for (int n = by_length(p) ? 1 : blocks; n <= blocks; ++n, a.above = a.limit) {
        a.limit = 32 * n;
        a.last = n == blocks;
        const int line = walk_line(p, n);
        walk_dispatch(p.dtype, p.dim, n, [&](auto t, auto db, auto nb) {
            typedef decltype(t) T;
            constexpr int DB = decltype(db)::value, kNB = decltype(nb)::value;
            constexpr int kBlock = 32 * Tile<T, DB>::kSlots, kTile = 32 * Tile<T, 1>::kSlots;
            const int tiles = (a.triangle ? kNB * (kNB + 1) / 2 : kNB * kNB) * 2 * kTile;
            a.time_at = 2 * kNB * kBlock + std::max(2 * kNB * kBlock, tiles);
            size_t lds = a.time_at * size_t{16} + 64 * kNB * sizeof(float);
            if (p.score.table) lds += ((1 + kNB) * line + kNB * kSquare) * sizeof(float);
            if (a.group > 1)
                hipLaunchKernelGGL((walk_backward_kernel<T, DB, kNB, true>), dim3(grid),
                                   dim3(64 * kNB), lds, stream, a);
            else
                hipLaunchKernelGGL((walk_backward_kernel<T, DB, kNB, false>), dim3(grid),
                                   dim3(64 * kNB), lds, stream, a);
        });
    }
    check_launch("walk_backward");
}

}  // namespace ops
}  // namespace trw
