// beams.hip -- beam search over a walk's next nodes: the best continuations of
// each group's beams, and the beams' pages put in their order.
//
// Choice.  log p of node x after beam b is score_b + x - log sum exp(row b).  One pass
// over the logits leaves the maximum and the sum of exponentials of every chunk of a
// row (what a wave holds: 64 lanes of 8 x 16 bytes).  With them a group's workgroup
// knows each beam's sum and the best continuation of every chunk, and the `width` best
// ones are all in the `width` chunks whose best ones come first: of any other chunk's,
// `width` come before.  Those few chunks are read again, and what reaches the last
// one's best is ranked by counting.  What follows the chunks' sums is float64 (but for
// the exponentials that join them), for the order of candidates of different beams:
// scores are 1.05 to 1.12 times as far from 64 bits as their last rounding, with a
// logarithm of float32 1.25 to 1.7 times.  Lanes hold the same nodes whatever the row's
// alignment, so that equal rows have equal sums and ties go to the lowest index.
//
// Measured: 64 groups of 8 beams over 50021 nodes in bfloat16 (51 MB, 9.9 us at a copy's
// rate) 20.6 us: 12.9 for the sums and 8.8 for the choice, whose few loads follow each
// other.  Rows in a worse order for it, all equal or ascending, take 33 to 38.  4 groups
// of 4 beams over 4000 nodes are one launch of 8.4 to 10.8 us, by their numbers.
//
// Order.  A beam's pages but the last one are full, so beams share them by their table
// alone.  The last page is written to next, so each beam owns its own: a parent's first
// child keeps it, further children copy its rows to the pages of beams without children
// (unless another beam's past lies there, or another child's copy of other rows, which
// is not so for a beam that still grows).
#include <algorithm>
#include <cmath>

#include "beams.h"
#include "pages.h"

namespace trw {
namespace ops {
namespace {

constexpr int kPieces = 8;    // 16-byte pieces of a lane
constexpr int kListed = 128;  // candidates of a chunk before the best are taken from them
constexpr int kMost = TRW_OPS_BEAMS;
constexpr int kJoinWaves = 16;    // of a group's workgroup, at most
constexpr int kRanked = 256;      // chunks that are ranked without a bound
constexpr float kMax = 3.402823466e38f;
// Up to here a maximum's product with log2 e is off by 2^-13 at most, and its rounding
// is taken from a sum of exponentials as (1 - ln2 rounding), good to 2^-27.
constexpr float kNear = 2048.0f;

typedef unsigned long long u64;

struct SelectArgs {
    const char* logits;
    int64_t group_stride, beam_stride;  // elements
    const float* scores;
    const uint8_t* ended;
    int64_t end_token;
    int groups, beams, width, nodes, chunks;
    float2* sums;  // [groups, beams, chunks] maximum and sum
    float* out_scores;
    int64_t *out_tokens, *out_parents;
    uint8_t* out_ended;
};

// float32 in the order of whole numbers.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t bits = __float_as_uint(x);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
// A float32 just below, for a bound that is to be reached.
__device__ __forceinline__ float under(double x) {
    const float near = static_cast<float>(x);
    return near > -kMax ? value_of(ordered(near) - 1) : -INFINITY;
}
// A candidate of one row as one number: greater is better, and of equal logits the
// lower node.  0: none.
__device__ __forceinline__ u64 key_of(float x, uint32_t node) {
    return static_cast<u64>(ordered(x + 0.0f)) << 32 | (0xffffffffu - node);  // -0 is 0
}
__device__ __forceinline__ float logit_of(u64 key) { return value_of(key >> 32); }
__device__ __forceinline__ uint32_t node_of(u64 key) {
    return 0xffffffffu - static_cast<uint32_t>(key);
}
// Candidates of beams: by their values, and by beam and node where those are equal.
__device__ __forceinline__ bool before(double a, u64 at_a, double b, u64 at_b) {
    return a > b || (a == b && at_a < at_b);
}
__device__ __forceinline__ u64 place_of(int beam, uint32_t node) {
    return static_cast<u64>(beam) << 32 | node;
}

// Of the lanes in a mask, how many come before this one.
__device__ __forceinline__ int before_me(u64 mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}
// Over a wave, by moves between lanes' registers: 0x111 .. 0x118 are shifts by 1, 2,
// 4 and 8 lanes inside rows of 16, 0x142 and 0x143 broadcast a row's and two rows'
// last lane to the next.  The last lane has the whole.
template <int kMove, int kRows>
__device__ __forceinline__ float moved(float x, float old) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(old), __float_as_uint(x),
                                                       kMove, kRows, 0xf, false));
}
__device__ __forceinline__ float last_lane(float x) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
__device__ __forceinline__ float wave_top(float x) {
    x = fmaxf(x, moved<0x111, 0xf>(x, x));
    x = fmaxf(x, moved<0x112, 0xf>(x, x));
    x = fmaxf(x, moved<0x114, 0xf>(x, x));
    x = fmaxf(x, moved<0x118, 0xf>(x, x));
    x = fmaxf(x, moved<0x142, 0xf>(x, x));
    x = fmaxf(x, moved<0x143, 0xf>(x, x));
    return last_lane(x);
}
__device__ __forceinline__ float wave_sum(float x) {
    x += moved<0x111, 0xf>(x, 0.0f);
    x += moved<0x112, 0xf>(x, 0.0f);
    x += moved<0x114, 0xf>(x, 0.0f);
    x += moved<0x118, 0xf>(x, 0.0f);
    x += moved<0x142, 0xa>(x, 0.0f);
    x += moved<0x143, 0xc>(x, 0.0f);
    return last_lane(x);
}
template <int kMove>
__device__ __forceinline__ uint32_t less_of(uint32_t x) {
    return min(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
                      static_cast<int>(x), static_cast<int>(x), kMove, 0xf, 0xf, false)));
}
__device__ __forceinline__ uint32_t wave_least(uint32_t x) {
    x = less_of<0x111>(x);
    x = less_of<0x112>(x);
    x = less_of<0x114>(x);
    x = less_of<0x118>(x);
    x = less_of<0x142>(x);
    x = less_of<0x143>(x);
    return __builtin_amdgcn_readlane(x, 63);
}
// Over groups of eight lanes, in every one of them: by pairs, by fours, mirrored.
__device__ __forceinline__ float eight_top(float x) {
    x = fmaxf(x, moved<0xb1, 0xf>(x, x));
    x = fmaxf(x, moved<0x4e, 0xf>(x, x));
    return fmaxf(x, moved<0x141, 0xf>(x, x));
}
template <int kMove>
__device__ __forceinline__ double moved(double x) {
    const u64 bits = static_cast<u64>(__double_as_longlong(x));
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), kMove, 0xf, 0xf, false);
    const uint32_t hi =
        __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), kMove, 0xf, 0xf, false);
    return __longlong_as_double(static_cast<long long>(static_cast<u64>(hi) << 32 | lo));
}
__device__ __forceinline__ double eight_sum(double x) {
    x += moved<0xb1>(x);
    x += moved<0x4e>(x);
    return x + moved<0x141>(x);
}
// The first `width` of `count` different keys in order, to `best` (may be `keys`), by
// one wave.  count: width to kListed.
__device__ __forceinline__ void take_best(const u64* keys, int count, u64* best, int width,
                                          int lane) {
    u64 mine[kListed / 64];
    int rank[kListed / 64] = {};
#pragma unroll
    for (int i = 0; i < kListed / 64; ++i)
        mine[i] = i * 64 + lane < count ? keys[i * 64 + lane] : 0;
    for (int j = 0; j < count; ++j) {
        const u64 other = keys[j];
#pragma unroll
        for (int i = 0; i < kListed / 64; ++i) rank[i] += other > mine[i];
    }
#pragma unroll
    for (int i = 0; i < kListed / 64; ++i)
        if (mine[i] && rank[i] < width) best[rank[i]] = mine[i];
}

// A number that the largest `width` of a wave's numbers reach, and hardly more: between
// the least and the greatest by halves, until just `width` do.  0: no bound (0 is none
// of them).
__device__ __forceinline__ uint32_t bound_of(uint32_t order, int width) {
    uint32_t lo = wave_least(order), hi = ~wave_least(~order);
    int reach = 64;
    while (lo < hi && reach != width) {
        const uint32_t mid = lo + ((hi - lo) >> 1) + 1;
        const int n = __popcll(__ballot(order >= mid));
        if (n >= width) {
            lo = mid;
            reach = n;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

// ---- chunks of a row ------------------------------------------------------------------------------
template <typename T>
struct Piece {
    static constexpr int kElems = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(kElems)));
    vec x;
    __device__ __forceinline__ float at(int e) const { return static_cast<float>(x[e]); }
};
template <typename T>
constexpr int kChunk = 64 * kPieces * Piece<T>::kElems;  // nodes of a wave

template <typename T>
__device__ __forceinline__ const T* row_of(const SelectArgs& a, int64_t group, int beam) {
    return reinterpret_cast<const T*>(a.logits) + group * a.group_stride + beam * a.beam_stride;
}

// Piece c of lane l holds the nodes begin + (64 c + l) kElems ..; -inf past the row's end.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int nodes, int begin, int lane,
                                           Piece<T> (&x)[kPieces], int first_piece = 0,
                                           int last_piece = kPieces) {
    constexpr int kElems = Piece<T>::kElems;
    if (begin + kChunk<T> <= nodes) {
#pragma unroll
        for (int c = 0; c < kPieces; ++c)  // 16 bytes of any alignment
            if (c >= first_piece && c < last_piece)
                __builtin_memcpy(&x[c], row + begin + (c * 64 + lane) * kElems, 16);
        return;
    }
    // The row's end: whole pieces, then the one that it cuts, all on their way at once.
    const T none = static_cast<T>(-INFINITY);
    if (nodes >= kElems) {
#pragma unroll
        for (int c = 0; c < kPieces; ++c)
            __builtin_memcpy(&x[c], row + min(begin + (c * 64 + lane) * kElems, nodes - kElems), 16);
    }
    const int cut = (nodes - begin) / kElems;  // its number among the wave's
    T end[kElems];
#pragma unroll
    for (int e = 0; e < kElems; ++e) end[e] = row[min(begin + cut * kElems + e, nodes - 1)];
#pragma unroll
    for (int c = 0; c < kPieces; ++c)
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
            const int number = c * 64 + lane;
            const T last = begin + cut * kElems + e < nodes ? end[e] : none;
            x[c].x[e] = number < cut ? x[c].x[e] : number == cut ? last : none;
        }
}

// A chunk's maximum (-inf: it has no candidates) and the sum of the exponentials of what
// its logits are less than it; NaN where one is NaN or +inf.
template <typename T>
__device__ __forceinline__ void sum_chunk(const T* row, const uint8_t* ended, int nodes, int begin,
                                          int lane, float2* stats) {
    constexpr int kElems = Piece<T>::kElems;
    const uint8_t at_end = ended ? *ended : 0;  // looked at when the nodes are on their way
    Piece<T> x[kPieces];
    load_chunk(row, nodes, begin, lane, x);
    if (at_end) return;
    float top = -INFINITY;
#pragma unroll
    for (int c = 0; c < kPieces; ++c)
#pragma unroll
        for (int e = 0; e < kElems; ++e) top = fmaxf(top, x[c].at(e));
    top = wave_top(top);
    float sum = 0.0f;
    if (fabsf(top) <= kNear) {
        // less base2, whose rounding the sum is then freed of
        const float base2 = top * kLog2e;
#pragma unroll
        for (int c = 0; c < kPieces; ++c)
#pragma unroll
            for (int e = 0; e < kElems; ++e) sum += exp2_fast(fmaf(x[c].at(e), kLog2e, -base2));
        sum = fmaf(-kLn2 * fmaf(top, kLog2e, -base2), sum, sum);
    } else {
        // differences first, which are exact where their exponentials are not 0; -inf, and a
        // chunk of nothing else, add 0
        const float base = fmaxf(top, -kMax);
#pragma unroll
        for (int c = 0; c < kPieces; ++c)
#pragma unroll
            for (int e = 0; e < kElems; ++e) sum += exp2_fast((x[c].at(e) - base) * kLog2e);
    }
    sum = wave_sum(sum);
    if (lane == 0) *stats = make_float2(top, sum);
}

// The nodes of a chunk's pieces [first_piece, last_piece) whose logits are `from` or
// above, `width` best ones at most, as keys; returns how many.  Logits whose values
// off + (logit - top) are one float64 are one logit, so that the lower node comes first.
template <typename T>
__device__ __forceinline__ int scan_chunk(const T* row, int nodes, int begin, int first_piece,
                                          int last_piece, float from, double off, double top,
                                          int width, int lane, u64* listed) {
    constexpr int kElems = Piece<T>::kElems;
    auto key_at = [&](float v, uint32_t node) {
        const double value = off + (static_cast<double>(v) - top);
        return key_of(static_cast<float>(value - off + top), node);
    };
    Piece<T> x[kPieces];
    load_chunk(row, nodes, begin, lane, x, first_piece, last_piece);
    int count = 0;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
        if (c < first_piece || c >= last_piece) continue;
        float most = x[c].at(0);
#pragma unroll
        for (int e = 1; e < kElems; ++e) most = fmaxf(most, x[c].at(e));
        if (!__any(most >= from)) continue;
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
            const float v = x[c].at(e);
            const u64 some = __ballot(v >= from);
            if (!some) continue;
            if (v >= from)
                listed[min(count + before_me(some), kListed - 1)] =
                    key_at(v, begin + (c * 64 + lane) * kElems + e);
            count += __popcll(some);
        }
    }
    if (count > kListed) {
        // Too many for the list: once more, and the best whenever it is full.
        u64 last = 0;
        count = 0;
        const int end = min(nodes, begin + last_piece * 64 * kElems);
        for (int first = begin + first_piece * 64 * kElems + lane; first < end + lane;
             first += 8 * 64) {
            float v[8];  // on their way at once
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = static_cast<float>(row[min(first + 64 * i, end - 1)]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int node = first + 64 * i;
                const u64 key = key_at(v[i], node);
                const bool in = node < end && v[i] >= from && key > last;
                const u64 some = __ballot(in);
                if (in) listed[count + before_me(some)] = key;
                count += __popcll(some);
                if (count > kListed - 64) {
                    take_best(listed, count, listed, width, lane);
                    count = width;
                    last = listed[width - 1];
                }
            }
        }
    }
    if (count > width) {
        take_best(listed, count, listed, width, lane);
        count = width;
    }
    return count;
}

// ---- a group's choice -----------------------------------------------------------------------------
constexpr int kItems = kMost * kMost;  // chunks that are ranked at once, and candidates

struct JoinScratch {
    // of each beam: score less the log of the sum (NaN: no candidates), and the maximum
    // of its logits, which is taken from them first
    double off[kMost];
    float top[kMost];
    bool ended[kMost];
    float bound[kJoinWaves];
    // items that are ranked: chunks, then candidates
    double value[kItems];
    u64 index[kItems];
    int rank[2][kItems];
    int count[2];
    double best_value[kMost];  // the chunks that are looked at
    int best_chunk[kMost];
    u64 listed[kJoinWaves][kListed];
};

// Adds to `rank` how many of `count` items come before each (barriers around).
__device__ __forceinline__ void rank_items(const JoinScratch& s, int count, int* rank) {
    const int thread = threadIdx.x, threads = blockDim.x;
    if (2 * count > threads) {
        for (int i = thread; i < count; i += threads) {
            const double value = s.value[i];
            const u64 index = s.index[i];
            int n = 0;
            for (int j = 0; j < count; ++j) n += before(s.value[j], s.index[j], value, index);
            rank[i] = n;
        }
        return;
    }
    // several threads an item, each for a part of the others
    const int shift = 32 - __clz(max(count - 1, 0)), i = thread & ((1 << shift) - 1);
    const int parts = threads >> shift, part = thread >> shift;
    if (i >= count || part >= parts) return;
    const int each = (count + parts - 1) / parts;
    const double value = s.value[i];
    const u64 index = s.index[i];
    int n = 0;
#pragma unroll 4
    for (int j = part * each; j < min(count, (part + 1) * each); ++j)
        n += before(s.value[j], s.index[j], value, index);
    if (n) atomicAdd(&rank[i], n);
}

// The new beams of a group from its chunks' sums, by a workgroup of whole waves.
template <typename T>
__device__ __forceinline__ void choose(const SelectArgs& a, int64_t group, const float2* sums,
                                       JoinScratch& s) {
    const int thread = threadIdx.x, threads = blockDim.x, lane = thread & 63;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6), waves = threads / 64;
    const int64_t first = group * a.beams;
    const int all = a.beams * a.chunks;
    // This thread's first chunk, and its beam's first sums, are on their way at once.
    const float near_top = sums[min(thread, all - 1)].x;
    float2 near[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        near[i] = sums[min(thread / 8, a.beams - 1) * a.chunks +
                       min((thread & 7) + 8 * i, a.chunks - 1)];
    auto sum_of = [&](int b, int p) {
        if (b == thread / 8 && p < 16) return p < 8 ? near[0] : near[1];
        return sums[b * a.chunks + p];
    };
    for (int i = thread; i < kItems; i += threads) s.rank[0][i] = s.rank[1][i] = 0;
    if (thread < kMost) s.best_chunk[thread] = -1;
    if (thread < 2) s.count[thread] = 0;
    for (int b0 = 0; b0 < a.beams; b0 += threads / 8) {  // eight lanes a beam
        const int b = b0 + thread / 8, sub = thread & 7;
        if (b0 + wave * 8 >= a.beams) break;  // whole waves
        const bool in = b < a.beams;
        const int64_t beam = first + min(b, a.beams - 1);
        const float score = a.scores[beam];
        const bool ended = a.ended && a.ended[beam];
        const bool is = in && fabsf(score) <= kMax, grows = is && !ended;
        float m = -kMax;
        double sum = 0.0;
        if (grows)
            for (int p = sub; p < a.chunks; p += 8) m = fmaxf(m, sum_of(b, p).x);
        m = eight_top(m);
        if (grows)
            for (int p = sub; p < a.chunks; p += 8) {
                const float2 part = sum_of(b, p);
                sum += static_cast<double>(part.y) * exp2_fast((fmaxf(part.x, -kMax) - m) * kLog2e);
            }
        sum = eight_sum(sum);
        if (in && sub == 0) {
            double off = NAN;
            if (grows && sum > 0.0) off = static_cast<double>(score) - log(sum);
            else if (is && ended) off = score;
            s.off[b] = off;
            s.top[b] = m;
            s.ended[b] = ended;
        }
    }
    __syncthreads();

    // Chunk n's best value (-inf: none); a beam that has ended is its first chunk.
    const float per_chunk = 1.0f / a.chunks;
    auto beam_of = [&](int n) {
        int b = static_cast<int>(n * per_chunk);  // n / chunks, n below 2^24, or one beside
        b += (b + 1) * a.chunks <= n;
        return b - (b * a.chunks > n);
    };
    auto chunk_value = [&](int n) {
        const int b = beam_of(n);
        const double off = s.off[b];
        if (!(fabs(off) <= 1.7e308)) return static_cast<double>(-INFINITY);
        if (s.ended[b]) return n == b * a.chunks ? off : -INFINITY;
        const float top = n == thread ? near_top : sums[n].x;
        return off + (static_cast<double>(top) - s.top[b]);
    };
    // The `width` chunks that come first, in order.
    int items = all;
    if (all <= kRanked) {
        for (int n = thread; n < all; n += threads) {
            s.value[n] = chunk_value(n);
            s.index[n] = n;
        }
    } else {
        // Those that reach a bound: in each wave one for its lanes' best ones, and of the
        // waves the greatest.
        double best = -INFINITY;
        for (int n = thread; n < all; n += threads) best = fmax(best, chunk_value(n));
        // (the lower bits would be halves more that change little)
        const uint32_t bound = bound_of(best > -INFINITY ? ordered(under(best)) >> 12 : 0, a.width);
        if (lane == 0) s.bound[wave] = bound >= 0x800 ? value_of(bound << 12) : -INFINITY;  // -kMax
        __syncthreads();
        float least = -INFINITY;
        for (int w = 0; w < waves; ++w) least = fmaxf(least, s.bound[w]);
        for (int n = thread; n < all; n += threads) {
            const double value = chunk_value(n);
            if (value >= least && value > -INFINITY) {
                const int place = atomicAdd(&s.count[0], 1);  // in any order: they are ranked
                if (place < kItems) {
                    s.value[place] = value;
                    s.index[place] = n;
                }
            }
        }
        __syncthreads();
        items = s.count[0];
    }
    if (items <= kItems) {
        __syncthreads();
        rank_items(s, items, s.rank[0]);
        __syncthreads();
        for (int i = thread; i < items; i += threads)
            if (s.rank[0][i] < a.width && s.value[i] > -INFINITY) {
                s.best_chunk[s.rank[0][i]] = static_cast<int>(s.index[i]);
                s.best_value[s.rank[0][i]] = s.value[i];
            }
    } else {  // so many equal ones: one place after the other
        double last = INFINITY;
        int last_number = -1;
        for (int place = 0; place < a.width; ++place) {
            double top = -INFINITY;
            int top_number = INT32_MAX;
            for (int n = thread; n < all; n += threads) {
                const double value = chunk_value(n);
                if (before(last, last_number, value, n) && before(value, n, top, top_number)) {
                    top = value;
                    top_number = n;
                }
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) {
                const double value = __shfl_xor(top, o);
                const int n = __shfl_xor(top_number, o);
                if (before(value, n, top, top_number)) {
                    top = value;
                    top_number = n;
                }
            }
            if (lane == 0) {
                s.value[wave] = top;
                s.index[wave] = top_number;
            }
            __syncthreads();
            top = s.value[0];
            u64 at = s.index[0];
            for (int w = 1; w < waves; ++w)
                if (before(s.value[w], s.index[w], top, at)) {
                    top = s.value[w];
                    at = s.index[w];
                }
            if (thread == 0) {
                s.best_value[place] = top;
                s.best_chunk[place] = static_cast<int>(at);
            }
            __syncthreads();
            last = top;
            last_number = static_cast<int>(at);
        }
    }
    __syncthreads();

    // Their nodes that reach the last one's best: a chunk a wave, or, where there are
    // waves for it, several for its pieces.
    const double least = s.best_chunk[a.width - 1] >= 0 ? s.best_value[a.width - 1] : -INFINITY;
    const int shares = max(1, min(kPieces, 1 << (31 - __clz(max(1, waves / a.width)))));
    for (int i = wave; i < a.width * shares; i += waves) {
        const int n = __builtin_amdgcn_readfirstlane(s.best_chunk[i / shares]);
        if (n < 0) break;
        const int b = __builtin_amdgcn_readfirstlane(beam_of(n));
        const double off = s.off[b];
        const float top = s.top[b];
        const int share = i % shares;
        if (s.ended[b]) {
            if (lane == 0 && share == 0) {
                const int place = atomicAdd(&s.count[1], 1);
                s.value[place] = off;
                s.index[place] = place_of(b, static_cast<uint32_t>(a.end_token));
            }
            continue;
        }
        // (less than float64 may lose between numbers of very different sizes)
        const double lost = (fabs(least) + fabs(off) + fabsf(top)) * 0x1p-50;
        const float from = least > -INFINITY ? fmaxf(under(least - off + top - lost), -kMax) : -kMax;
        u64* listed = s.listed[wave];
        const int found = scan_chunk<T>(row_of<T>(a, group, b), a.nodes, (n - b * a.chunks) * kChunk<T>,
                                        kPieces / shares * share, kPieces / shares * (share + 1),
                                        from, off, top, a.width, lane, listed);
        int place = 0;
        if (lane == 0) place = atomicAdd(&s.count[1], found);  // in any order: they are ranked
        place = __builtin_amdgcn_readfirstlane(place);
        if (lane < found) {
            s.value[place + lane] = off + (static_cast<double>(logit_of(listed[lane])) - top);
            s.index[place + lane] = place_of(b, node_of(listed[lane]));
        }
    }
    __syncthreads();

    const int count = s.count[1];
    rank_items(s, count, s.rank[1]);
    __syncthreads();
    const int64_t to = group * a.width;
    for (int i = thread; i < max(count, a.width); i += threads) {
        const bool none = i >= count;
        const int place = none ? i : s.rank[1][i];
        if (place >= a.width) continue;
        const u64 index = none ? 0 : s.index[i];
        const int parent = static_cast<int>(index >> 32);
        const int64_t token =
            none ? max(a.end_token, int64_t{0}) : static_cast<int64_t>(index & 0xffffffffu);
        a.out_scores[to + place] = none ? -INFINITY : static_cast<float>(s.value[i]);
        a.out_tokens[to + place] = token;
        a.out_parents[to + place] = parent;
        a.out_ended[to + place] = none || token == a.end_token || s.ended[parent];
    }
}

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Whether a beam's score is finite: no candidates come of others.  By the scalar
// cache, past the queue of loads of the waves that are ahead (all of them ask for
// their nodes at once).
__device__ __forceinline__ bool scored(const SelectArgs& a, int64_t beam) {
    typedef __attribute__((address_space(4))) const float* scalar;
    return fabsf(((scalar)(reinterpret_cast<uintptr_t>(a.scores)))[beam]) <= kMax;
}

// One chunk a wave, four of a row a workgroup.
template <typename T>
__global__ __launch_bounds__(kThreads) void select_sums_kernel(SelectArgs a, int parts) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunk = blockIdx.x % parts * kWaves + wave;
    const int64_t row = blockIdx.x / parts;  // group and beam
    if (chunk >= a.chunks || !scored(a, row)) return;
    sum_chunk<T>(row_of<T>(a, row / a.beams, row % a.beams), a.ended ? a.ended + row : nullptr,
                 a.nodes, chunk * kChunk<T>, lane, a.sums + row * a.chunks + chunk);
}

template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void select_kernel(SelectArgs a) {
    __shared__ JoinScratch s_join;
    choose<T>(a, blockIdx.x, a.sums + static_cast<int64_t>(blockIdx.x) * a.beams * a.chunks, s_join);
}

// A whole group a workgroup, where it has few chunks: one launch.
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void select_group_kernel(SelectArgs a) {
    __shared__ float2 s_sums[kJoinWaves];
    __shared__ JoinScratch s_join;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t group = blockIdx.x;
    const int beam = wave / a.chunks, chunk = wave % a.chunks;
    const int64_t row = group * a.beams + beam;
    if (beam < a.beams && scored(a, row))
        sum_chunk<T>(row_of<T>(a, group, beam), a.ended ? a.ended + row : nullptr, a.nodes,
                     chunk * kChunk<T>, lane, s_sums + wave);
    __syncthreads();
    choose<T>(a, group, s_sums, s_join);
}

int64_t chunks_of(const trw_beam_select_params& p) {
    const int64_t nodes = p.dtype == TRW_F32 ? kChunk<float> : kChunk<__bf16>;
    return (p.nodes + nodes - 1) / nodes;
}
bool fused(const trw_beam_select_params& p) { return p.beams * chunks_of(p) <= kJoinWaves; }

// ---- reordering ----------------------------------------------------------------------------------
constexpr int kCaches = 8;  // of one launch

struct Matrix {  // keys or values of one cache
    char* data;
    uint8_t* scale;  // or null
    int64_t page, scale_page;
    int row_bytes, heads;
};
struct ReorderArgs {
    Matrix matrix[2 * kCaches];
    const int32_t* table;
    int64_t table_stride;
    int32_t* out_table;
    const int64_t *lens, *parents;
    int64_t* out_lens;
    float* k_times;
    int beams, table_pages, pages, shift, first, matrices, heads, share;
};

// `share` workgroups a group.  Every wave works out the group's plan, a child a lane;
// the rows that move, of every head of every cache's keys and values, are then dealt
// out to the workgroups piece by piece, which evens out how many children a group's
// parents have.
__global__ __launch_bounds__(kThreads) void reorder_kernel(ReorderArgs a) {
    const int part = blockIdx.x % a.share;
    const int64_t group = static_cast<int64_t>(blockIdx.x / a.share) * a.beams;
    const int thread = threadIdx.x, lane = thread & 63;
    int parent = -1;
    int64_t len = 0;  // of this lane's beam, then of its child
    if (lane < a.beams) {
        const int64_t p = a.parents[group + lane];
        len = a.lens[group + lane];
        parent = static_cast<int>(min(max(p, int64_t{0}), static_cast<int64_t>(a.beams - 1)));
    }
    // beams without children, and children that are not their parent's first
    uint32_t childless = 0, further = 0;
    for (int b = 0; b < a.beams; ++b) {
        const uint32_t children = static_cast<uint32_t>(__ballot(parent == b));
        if (!children) childless |= 1u << b;
        further |= children & (children - 1);
    }
    const int held = static_cast<int>(
        min(max(len, int64_t{0}) >> a.shift, static_cast<int64_t>(a.table_pages)));
    len = __shfl(len, max(parent, 0));
    const int full = __shfl(held, max(parent, 0));
    const int rows = len > 0 ? static_cast<int>(len & ((1 << a.shift) - 1)) : 0;
    int taken = parent, source = -1, target = -1, kept = full;
    if (lane < a.beams && further >> lane & 1) {
        // as many beams are without children as children are further ones
        uint32_t left = childless;
        for (int n = __popc(further & ((1u << lane) - 1)); n; --n) left &= left - 1;
        taken = __ffs(left) - 1;
    }
    // Further children's copies, those of equal lengths at once: a lane a beam's page.
    const u64 fill = __ballot(rows && full < a.table_pages) & further;
    for (u64 left = fill; left;) {
        const int at = __builtin_amdgcn_readlane(full, __ffsll(left) - 1);
        const u64 these = left & __ballot(full == at);
        const int page = lane < a.beams ? a.table[(group + lane) * a.table_stride + at] : -1;
        const int from = __shfl(page, max(parent, 0)), to = __shfl(page, max(taken, 0));
        // A parent that ended before others: the page may be part of what another beam with
        // children holds.  Then the child reads the parent's, which grows no more.  Beams without
        // children may share a page as well: it takes one child's rows, and later children of
        // other parents read their parents'.
        const uint32_t reads = static_cast<uint32_t>(__ballot(lane < a.beams && held >= at)) & ~childless;
        uint32_t equal = 0;  // beams whose page is this child's
        for (int b0 = 0; b0 < a.beams; b0 += 8)
#pragma unroll
            for (int b = 0; b < 8; ++b)
                equal |= __builtin_amdgcn_readlane(page, b0 + b) == to ? 1u << (b0 + b) : 0u;
        bool others = equal & reads;
        const bool again = equal & childless & ~(1u << max(taken, 0));
        if (__builtin_expect((__ballot(again && !others) & these) != 0, 0)) {
            for (u64 b = these; b; b &= b - 1) {
                const int n = __ffsll(b) - 1;
                const bool copies = !__builtin_amdgcn_readlane(static_cast<int>(others), n);
                others |= copies && lane > n && __builtin_amdgcn_readlane(to, n) == to &&
                          __builtin_amdgcn_readlane(from, n) != from;
            }
        }
        others = others && to >= 0 && to < a.pages;
        if (these >> lane & 1) {
            source = from;
            target = others ? -1 : to;
            kept = full + others;
        }
        left &= ~these;
    }
    // what moves: between pages of the pool
    const u64 moving = __ballot(source >= 0 && source < a.pages && target >= 0 && target < a.pages &&
                                source != target);

    if (a.first) {
        for (int child = part; child < a.beams; child += a.share) {
            const int whole = __builtin_amdgcn_readlane(kept, child);
            const int32_t* from =
                a.table + (group + __builtin_amdgcn_readlane(parent, child)) * a.table_stride;
            const int32_t* rest =
                a.table + (group + __builtin_amdgcn_readlane(taken, child)) * a.table_stride;
            int32_t* to = a.out_table + (group + child) * a.table_pages;
            for (int p = thread; p < a.table_pages; p += kThreads)
                to[p] = p < whole ? from[p] : rest[p];
        }
        if (part == 0 && thread < a.beams) a.out_lens[group + thread] = len;
    }

    const int each = a.matrices * a.heads, items = __popcll(moving) * each;
    constexpr int kAtOnce = 4;
    for (int i0 = part; i0 < items; i0 += kAtOnce * a.share) {
        const char* read[kAtOnce];
        char* write[kAtOnce];
        const uint8_t* read_scale[kAtOnce];
        uint8_t* write_scale[kAtOnce];
        u32x4 data[kAtOnce];
        uint8_t scale[kAtOnce];
        int pieces[kAtOnce], scales[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {  // all on their way at once
            const int item = i0 + i * a.share;
            pieces[i] = scales[i] = 0;
            if (item >= items) continue;
            u64 left = moving;
            for (int n = item / each; n; --n) left &= left - 1;
            const int child = __ffsll(left) - 1, head = item % each % a.heads;
            const Matrix& x = a.matrix[item % each / a.heads];
            if (head >= x.heads) continue;
            const int from = __builtin_amdgcn_readlane(source, child);
            const int to = __builtin_amdgcn_readlane(target, child);
            const int count = __builtin_amdgcn_readlane(rows, child);
            const int64_t line = static_cast<int64_t>(head) << a.shift;
            read[i] = x.data + from * x.page + line * x.row_bytes;
            write[i] = x.data + to * x.page + line * x.row_bytes;
            pieces[i] = count * x.row_bytes / 16;
            if (thread < pieces[i]) data[i] = reinterpret_cast<const u32x4*>(read[i])[thread];
            if (x.scale) {
                read_scale[i] = x.scale + from * x.scale_page + line;
                write_scale[i] = x.scale + to * x.scale_page + line;
                scales[i] = count;
                if (thread < count) scale[i] = read_scale[i][thread];
            }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (thread < pieces[i]) reinterpret_cast<u32x4*>(write[i])[thread] = data[i];
            if (thread < scales[i]) write_scale[i][thread] = scale[i];
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {  // what is more than a thread's piece
#pragma unroll 4
            for (int n = thread + kThreads; n < pieces[i]; n += kThreads)
                reinterpret_cast<u32x4*>(write[i])[n] = reinterpret_cast<const u32x4*>(read[i])[n];
            for (int n = thread + kThreads; n < scales[i]; n += kThreads)
                write_scale[i][n] = read_scale[i][n];
        }
    }
    if (a.first && a.k_times)
        for (int n = part; n < __popcll(moving); n += a.share) {
            u64 left = moving;
            for (int i = n; i; --i) left &= left - 1;
            const int child = __ffsll(left) - 1;
            const int64_t from = __builtin_amdgcn_readlane(source, child);
            const int64_t to = __builtin_amdgcn_readlane(target, child);
            const int count = __builtin_amdgcn_readlane(rows, child);
            for (int r = thread; r < count; r += kThreads)
                a.k_times[(to << a.shift) + r] = a.k_times[(from << a.shift) + r];
        }
}

}  // namespace

uint64_t beam_select_workspace(const trw_beam_select_params& p) {
    if (fused(p)) return 0;
    return static_cast<uint64_t>(p.groups) * p.beams * chunks_of(p) * sizeof(float2);
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
    a.chunks = static_cast<int>(chunks_of(p));
    a.sums = static_cast<float2*>(p.workspace);
    a.out_scores = p.out_scores;
    a.out_tokens = p.out_tokens;
    a.out_parents = p.out_parents;
    a.out_ended = p.out_ended;
    require_grid(p.groups, 64 * kJoinWaves);
    if (fused(p)) {
        by_type(p.dtype, [&](auto t) {
            hipLaunchKernelGGL((select_group_kernel<decltype(t)>),
                               dim3(static_cast<unsigned>(p.groups)),
                               dim3(64 * p.beams * a.chunks), 0, stream, a);
        });
        check_launch("beam_select");
        return;
    }
    const int parts = (a.chunks + kWaves - 1) / kWaves;
    const int64_t grid = p.groups * p.beams * parts;
    require_grid(grid, kThreads);
    by_type(p.dtype, [&](auto t) {
        hipLaunchKernelGGL((select_sums_kernel<decltype(t)>), dim3(static_cast<unsigned>(grid)),
                           dim3(kThreads), 0, stream, a, parts);
        check_launch("beam_select");
        hipLaunchKernelGGL((select_kernel<decltype(t)>), dim3(static_cast<unsigned>(p.groups)),
                           dim3(64 * kJoinWaves), 0, stream, a);
        check_launch("beam_select");
    });
}

void beam_reorder(const trw_beam_reorder_params& p, hipStream_t stream) {
    for (int c = 0; c < p.count; ++c) require_apart(p.caches[c]);
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
    int done = 0;
    do {
        const int count = std::min(kCaches, p.count - done);
        a.first = done == 0;
        int heads = 1;
        for (int c = 0; c < count; ++c) {
            const trw_pages& from = p.caches[done + c];
            const Pages pages = make_pages(from);
            const int row_bytes = static_cast<int>(from.dim * page_element_size(from.dtype));
            a.matrix[2 * c] = Matrix{pages.k,      pages.k_scale, pages.k_page, pages.k_scale_page,
                                  row_bytes, from.kv_heads};
            a.matrix[2 * c + 1] = Matrix{pages.v,      pages.v_scale, pages.v_page, pages.v_scale_page,
                                      row_bytes, from.kv_heads};
            heads = std::max(heads, from.kv_heads);
        }
        // As many workgroups as the device holds at once: 32 groups of 8 beams, 4 caches of
        // 8 heads, 46 MB: 15.2 us with 2048, 17.4 with 1024, 17.5 with 4096 (before pages to
        // copy to were looked up among other beams': 16.7 with it).
        a.matrices = 2 * count;
        a.heads = heads;
        const int64_t most = static_cast<int64_t>(std::max(1, p.beams - 1)) * a.matrices * heads;
        a.share = static_cast<int>(std::min(most, std::max<int64_t>(1, 2048 / p.groups)));
        require_grid(p.groups * a.share, kThreads);
        hipLaunchKernelGGL(reorder_kernel, dim3(static_cast<unsigned>(p.groups * a.share)),
                           dim3(kThreads), 0, stream, a);
        check_launch("beam_reorder");
        done += count;
    } while (done < p.count);
}

}  // namespace ops
}  // namespace trw
