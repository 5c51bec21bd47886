// attention_paged.hip -- one new event of each walk over its pages.
//
// Per walk and key head: read the pages once, at memory speed.  The query heads
// that share a key head are the columns of the products, 16 of them; a wave takes
// blocks of 32 positions (two halves of 16, each in one page), four waves share a
// walk, each with a maximum, a sum and an output of its own, joined at the end.
// Positions that the walk does not see are never read.
//
// Walks differ in length, and only the device knows how much, so the positions of
// all walks are put in one line and dealt out evenly to as many workgroups as the
// device holds at once.  Where that cuts a walk, its parts are joined by a second
// launch.  With walks' own workgroups, three of them each, 64 walks of 100 to 4095
// events (8 heads of 128, 8 bits) took 76.7 us, 67.3 so.  Where no walk can be long for
// its batch, each has a workgroup and there is no second launch: the device evens them
// out (512 walks of 0 to 511 events in tables of 512, 8 bits: 87 us, dealt out 93).
//
// Measured, both launches: 64 walks of 4095 events each, 5.2 TB/s in 16 bits and 4.9 in
// 8 (a large copy: 5.17).  Of the mixed 64 above, 283 MB and 54.7 us at a copy's rate,
// the walk over the pages takes 64.5 us and the join 4.9; 3 walks of 260k events
// together, 135 MB and 26.2 us, 38.8 and 8.1.  What is over is the start (four loads
// one after the other before the first tile, 5 to 7 us) and the second launch.  In 8
// bits the vector units are busy 0.37 of the time, the matrix units 0.08.  Tiles are 32,
// 64 or 128 columns wide, in 8 bits 64 or 128; heads between those use part of one: 32
// columns in 8 bits read at 2.2 TB/s, 96 in 16 bits at 3.9.
//
// v_mfma_f32_16x16x32 with keys as rows leaves lane l with keys 4 (l / 16) .. + 4
// of column l & 15.  Two halves give eight, which are the B operand of the next
// product without moving: its element e of lane l is key 4 (l / 16) + e of the
// first half, e < 4, or key 4 (l / 16) + e - 4 of the second, and the values are
// read from LDS in the same order.
//
// 8 bits: codes are exact in bfloat16, and the products are bfloat16's whatever
// the type of q.  Keys' scales multiply scores and values' scales the softmax's
// weights, in float32 and exactly (they are powers of two).  q of longer types goes
// as two (float16) or three (float32) bfloat16 parts, which lose nothing.
//
// The softmax's weights go as two bfloat16 parts as well, or three where q is
// float32, so that nothing but the output is rounded as far as bfloat16 is (one part:
// outputs up to 1.75 times as far from exact ones; it costs no time that is seen, the
// kernel waits for memory).  Over pages of float16 they go as two float16 parts, and the
// largest weight is 2^15 instead of 1 (the sum too, so that it cancels): float16 ends at
// 2^-24, and what many keys of less than that share would be lost next to one of 1.
//
// The new row is taken from the call's arguments by the workgroup whose positions
// include it (in 8 bits as the codes that the pages get), and written to the pages
// by the same one (of several for a key head's columns, the first): no launch and no
// wait between the two.
#include <algorithm>

#include "pages.h"

namespace trw {
namespace ops {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kKeys = 32;    // positions of a wave's block
constexpr int kHalf = 16;    // of them in one page for sure
constexpr int kColumns = 16;

struct PagedArgs {
    Pages pages;
    Rows q, k, v, out;
    const int64_t *lens, *first;
    float* k_times;  // [pages, page_rows]
    Score score;
    int batch, heads, kv_heads, group, columns, dim;
    int even;            // workgroups of a key head that share all walks evenly; 0: one a walk
    // of walks that are cut: each workgroup's first and last part
    float* partial;      // [workgroups, 2, columns, dim]
    float2* part_stats;  // [workgroups, 2, columns]: maximum (base 2) and sum
    int64_t* begins;     // [batch + 1] where each walk begins in the line of units
};

constexpr int kUnit = kWaves;  // blocks that a workgroup takes at once

// Units of a walk: one at least, which writes what an idle one answers.
struct Length {
    int n, first, units;  // the new event's position, the first that is seen
    bool in;              // whether the table has a place for the new event
};
__device__ __forceinline__ Length length_of(const PagedArgs& a, int64_t b) {
    const int64_t at = a.lens[b], begin = a.first ? a.first[b] : 0;
    Length r;
    r.in = at >= 0 && at < static_cast<int64_t>(a.pages.table_pages) << a.pages.shift;
    r.n = r.in ? static_cast<int>(at) : 0;
    r.first = static_cast<int>(min(max(begin, int64_t{0}), static_cast<int64_t>(r.n)));
    r.units = (r.n / kKeys - r.first / kKeys) / kUnit + 1;
    return r;
}

__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// All but this wave's last kLater copies to LDS have landed.
template <int kLater>
__device__ __forceinline__ void copies_landed() {
    static_assert(kLater < 64, "counted in six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70 | (kLater & 15) | (kLater >> 4 << 14));
    asm volatile("" ::: "memory");
}
// 4 bytes of each lane's own address, to LDS at `lds` + 4 lane.
__device__ __forceinline__ void copy_far_word_to_lds(const void* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\t"
                 "s_nop 0\n\t"
                 "global_load_lds_dword %1, off"
                 :
                 : "s"(lds), "v"(from)
                 : "memory", "m0");
}

// A block's rows in LDS, in 16-byte chunks: chunk c of row r in slot c ^ swizzle(r),
// which spreads 16 rows' chunk c over the 256 bytes that the banks span.
template <int kBytes, int DB>
struct PageTile {
    static constexpr int kElems = 16 / kBytes;  // of a chunk
    // 16 rows are whole copies of a wave: 64 bytes of a row at least
    static constexpr int kWidth = DB > 2 ? 128 : DB == 2 ? 64 : kBytes == 1 ? 64 : 32;
    static constexpr int kSlots = kWidth / kElems;
    static constexpr int kHalfCopies = kHalf * kSlots / 64;
    static constexpr int kStep = 64 / kSlots;  // rows from one copy of a lane to the next
    static constexpr size_t kSize = size_t(kKeys) * kSlots * 16;

    __device__ static __forceinline__ int swizzle(int r) {
        return kSlots == 4 ? (r >> 2) & 3 : kSlots == 8 ? (r >> 1) & 7 : r & 15;
    }
    __device__ static __forceinline__ int slot(int row, int chunk) {
        return row * kSlots + (chunk ^ swizzle(row));
    }
};

// Operands of the products from a tile: elements 32 step + 8 quarter .. + 8 of a
// row, and column `col` of the keys 4 quarter + e (e < 4), 16 + 4 quarter + e - 4.
template <typename T, int DB>
struct Wide {  // rows of the products' type
    typedef PageTile<sizeof(T), DB> G;
    typedef Frag<T> F;

    __device__ static __forceinline__ F row(const u32x4* lds, int row, int step, int quarter) {
        union {
            u32x4 u[sizeof(T) / 2];
            F f;
        } x;
        constexpr int kChunks = sizeof(T) / 2;  // of eight elements
#pragma unroll
        for (int h = 0; h < kChunks; ++h)
            x.u[h] = lds[G::slot(row, (4 * step + quarter) * kChunks + h)];
        return x.f;
    }
    __device__ static __forceinline__ F columns(const u32x4* lds, int block, int lane) {
        const int quarter = lane >> 4;
        if constexpr (sizeof(T) == 2) {
            // each group of 16 lanes reads 4 rows of 16 columns and receives its own column
            const int s = lane & 15;
            const int col = 16 * block + 4 * (s & 3);
            union {
                s16x4 s[2];
                F f;
            } x;
            typedef __attribute__((address_space(3))) s16x4* lds4;
            const char* at = reinterpret_cast<const char*>(lds);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = kHalf * h + 4 * quarter + (s >> 2);
                const int byte = G::slot(r, col >> 3) * 16 + (col & 7) * 2;
                x.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds4)(const_cast<char*>(at) + byte));
            }
            return x.f;
        } else {
            const float* at = reinterpret_cast<const float*>(lds);
            const int col = 16 * block + (lane & 15);
            F f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = kHalf * (e >> 2) + 4 * quarter + (e & 3);
                f[e] = at[G::slot(r, col >> 2) * 4 + (col & 3)];
            }
            return f;
        }
    }
};

// Eight codes as bfloat16.
__device__ __forceinline__ bf16x8 widened(u32x2 c) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    union {
        bf16x2 p[4];
        bf16x8 f;
    } x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        x.p[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[h], 1.0f, false);
        x.p[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[h], 1.0f, true);
    }
    return x.f;
}

template <int DB>
struct Eight {  // rows of codes
    typedef PageTile<1, DB> G;
    typedef bf16x8 F;

    __device__ static __forceinline__ F row(const u32x4* lds, int row, int step, int quarter) {
        const char* at = reinterpret_cast<const char*>(lds);
        const int byte = G::slot(row, 2 * step + (quarter >> 1)) * 16 + (quarter & 1) * 8;
        return widened(*reinterpret_cast<const u32x2*>(at + byte));
    }
    __device__ static __forceinline__ F columns(const u32x4* lds, int block, int lane) {
        // each group of 16 lanes reads 8 rows of 16 columns, lane s addressing eight
        // columns of row s / 2, and receives its own column
        const int s = lane & 15, quarter = lane >> 4;
        const int r = 4 * quarter + ((s >> 1) & 3) + kHalf * (s >> 3);
        typedef int s32x2 __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) s32x2* lds2;
        const char* at = reinterpret_cast<const char*>(lds);
        const int byte = G::slot(r, block) * 16 + (s & 1) * 8;
        union {
            s32x2 s;
            u32x2 u;
        } x;
        x.s = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds2)(const_cast<char*>(at) + byte));
        return widened(x.u);
    }
};

template <typename F>
struct ElementOf {
    typedef __bf16 type;
};
template <>
struct ElementOf<f16x8> {
    typedef _Float16 type;
};
template <>
struct ElementOf<f32x8> {
    typedef float type;
};

// float32 values as kParts operands whose sum they are, nearly.
template <int kParts, typename F>
__device__ __forceinline__ void in_parts(const float (&x)[8], F (&parts)[kParts]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float rest = x[e];
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            parts[p][e] = static_cast<typename ElementOf<F>::type>(rest);
            if (p + 1 < kParts) rest -= static_cast<float>(parts[p][e]);
        }
    }
}

// Weights as two operands whose sum they are, nearly, and both of which are positive where
// the weight is, so that an infinity among the values stays one: the first is the greatest
// number of fewer bits that is less than the weight.  (What is left is 2^-7 of it in
// bfloat16 and 2^-10 in float16 at most, and rounded to half a step of as many bits; in
// float16 both are its smallest number or more, 2^-39 of the largest weight.)
__device__ __forceinline__ void in_positive_parts(const float (&x)[8], bf16x8 (&parts)[2]) {
    union {
        uint32_t u[4];
        bf16x8 f;
    } high;
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        uint32_t bits[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t all = __float_as_uint(x[e + i]);
            bits[i] = (all - min(all, 1u)) & 0xffff0000u;
            rest[e + i] = x[e + i] - __uint_as_float(bits[i]);
        }
        high.u[e / 2] = bits[0] >> 16 | bits[1];
    }
    parts[0] = high.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) parts[1][e] = static_cast<__bf16>(rest[e]);
}
__device__ __forceinline__ void in_positive_parts(const float (&x)[8], f16x8 (&parts)[2]) {
    typedef __fp16 h16x2 __attribute__((ext_vector_type(2)));
    union {
        h16x2 h[4];
        f16x8 f;
    } high;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float below[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t all = __float_as_uint(x[e + i]);
            below[i] = __uint_as_float(all - min(all, 1u));
            if (x[e + i] > 0.0f) below[i] = fmaxf(below[i], 0x1p-24f);
        }
        high.h[e / 2] = __builtin_amdgcn_cvt_pkrtz(below[0], below[1]);  // towards 0
    }
    parts[0] = high.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float rest = x[e] - static_cast<float>(high.f[e]);
        parts[1][e] = static_cast<_Float16>(x[e] > 0.0f ? fmaxf(rest, 0x1p-24f) : rest);
    }
}

// A pointer that is the same in every lane, as a scalar.
__device__ __forceinline__ const char* uniform(const char* p) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
    return reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// What was asked of LDS is here: copies may take its place.
__device__ __forceinline__ void reads_done() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}

// How `all` units are dealt out to `many` workgroups: the first ones get one more.
struct Share {
    int64_t each, more;
    __device__ __forceinline__ Share(int64_t all, int many) {
        if (all < (int64_t{1} << 31)) {  // a division of 32 bits
            each = static_cast<uint32_t>(all) / static_cast<uint32_t>(many);
        } else {
            each = all / many;
        }
        more = all - each * many;
    }
    __device__ __forceinline__ int64_t begin(int item) const {
        return item * each + min(static_cast<int64_t>(item), more);
    }
    // Who has unit x.
    __device__ __forceinline__ int owner(int64_t x) const {
        const int64_t big = more * (each + 1);
        return static_cast<int>(x < big ? x / (each + 1) : more + (x - big) / each);
    }
};

// Sums of the lanes up to each: by shifts inside rows of 16, then the rows' sums.
template <int kMove, int kRows>
__device__ __forceinline__ int moved(int x) {
    return __builtin_amdgcn_update_dpp(0, x, kMove, kRows, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int x) {
    x += moved<0x111, 0xf>(x);
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);
    x += moved<0x143, 0xc>(x);
    return x;
}

// The kernel's arguments once more, from memory: what is not needed all the time is not
// held in registers all the time (held, the arguments took more scalar registers than
// there are, and some 700 moves between them and vector registers).
typedef __attribute__((address_space(4))) const PagedArgs* ArgsAgain;
__device__ __forceinline__ ArgsAgain args_again() {
    ArgsAgain p = (ArgsAgain)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// Rows lo .. hi - 1 of a half as bits.
__device__ __forceinline__ uint32_t bits_of(int lo, int hi) {
    return hi > lo ? ((1u << hi) - 1) & ~((1u << lo) - 1) : 0u;
}

// Workgroups that a compute unit holds: their tiles' room in LDS, and registers.
template <typename T, int DB, bool kEight>
constexpr int kResident = kEight           ? (DB <= 2 ? 4 : 3)
                          : sizeof(T) == 2 ? (DB <= 2 ? 4 : 2)
                                           : (DB == 1 ? 4 : DB == 2 ? 2 : 1);

template <typename T, int DB, bool kWide, bool kEight>
__global__ __launch_bounds__(kThreads, (kResident<T, DB, kEight>))
void paged_step_kernel(PagedArgs a) {
    typedef std::conditional_t<kEight, Eight<DB>, Wide<T, DB>> In;
    typedef typename In::G G;
    typedef typename In::F F;
    constexpr int kBytes = kEight ? 1 : sizeof(T);
    constexpr bool kShort = std::is_same<T, __bf16>::value;
    constexpr int kParts = !kEight || kShort ? 1 : sizeof(T) == 4 ? 3 : 2;  // of q
    // parts of a weight, and what the largest one is
    constexpr int kWeights = sizeof(T) == 4 ? kParts : 2;
    constexpr float kLargest = std::is_same<F, f16x8>::value ? 32768.0f : 1.0f;
    constexpr int kJoinPitch = 32 * DB + 4;
    constexpr size_t kJoinBytes = size_t(kWaves) * kColumns * kJoinPitch * sizeof(float);
    constexpr size_t kTileBytes = 2 * kWaves * G::kSize;
    __shared__ u32x4 s_mem[(kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes) / 16];
    __shared__ float s_m[kWaves][kColumns], s_l[kWaves][kColumns];
    __shared__ float s_times[kWaves][64];
    __shared__ uint32_t s_scales[kEight ? kWaves : 1][64];  // keys' 32 bytes, values' 32
    __shared__ int64_t s_sums[kWaves];
    __shared__ int64_t s_start;
    __shared__ int s_walk;

    // Consecutive workgroups go to the eight XCDs in turn: each takes all key
    // heads of some positions.
    int rest = blockIdx.x / 8;
    const int col_group = rest % a.columns;
    rest /= a.columns;
    const int kv_head = rest % a.kv_heads;
    const int item = rest / a.kv_heads * 8 + blockIdx.x % 8;
    const int thread = threadIdx.x, lane = thread & 63, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int shift = a.pages.shift, page_mask = (1 << shift) - 1, dim = a.dim;
    const int col = col_group * kColumns + (lane & 15);
    const int head = kv_head * a.group + col;
    const bool any = col < a.group;
    const bool biased = a.score.table, sloped = a.score.slopes, timed = a.k_times;
    const float softcap = a.score.softcap, scale2 = a.score.scale2;
    const float slope = sloped && any ? a.score.slopes[head] * kLog2e : 0.0f;
    const float far_bias = biased && any ? table_entry(a.score, head, 2 * a.score.reach) : 0.0f;
    const int pitch = dim * kBytes;
    uint32_t offset[G::kHalfCopies];  // bytes from a half's first row
#pragma unroll
    for (int c = 0; c < G::kHalfCopies; ++c) {
        const int row = lane / G::kSlots + c * G::kStep;
        const int chunk = (lane % G::kSlots) ^ G::swizzle(row);
        offset[c] = row * pitch + (chunk * 16 < pitch ? chunk * 16 : 0);
    }

    // Units [unit, unit + left) of this workgroup, counted from walk b's first.
    int b = item;
    int64_t unit = 0, left = INT64_MAX;
    const bool few = a.even && a.batch <= 64;  // a walk a lane
    Length mine{};
    if (a.even) {
        if (item >= a.even) return;
        const bool notes = item == 0 && kv_head == 0 && col_group == 0;
        if (few) {
            if (lane < a.batch) mine = length_of(a, lane);
            const int till = wave_scan(mine.units);
            const int all = __builtin_amdgcn_readlane(till, 63);
            const Share share(all, a.even);
            const int begin = static_cast<int>(share.begin(item));
            left = share.begin(item + 1) - begin;
            if (notes && thread < a.batch) a.begins[thread] = till - mine.units;
            if (notes && thread == 0) a.begins[a.batch] = all;
            if (left <= 0) return;
            b = __popcll(__ballot(till <= begin));
            unit = begin - __builtin_amdgcn_readlane(till - mine.units, b);
        } else {
            // each thread some walks one after the other
            const int each = (a.batch + kThreads - 1) / kThreads;
            const int walk = min(thread * each, a.batch), end = min(walk + each, a.batch);
            int64_t sum = 0;
            for (int w = walk; w < end; ++w) sum += length_of(a, w).units;
            int64_t before = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int64_t other = __shfl_up(static_cast<long long>(before), o);
                if (lane >= o) before += other;
            }
            if (lane == 63) s_sums[wave] = before;
            __syncthreads();
            int64_t all = 0;
            before -= sum;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                if (w < wave) before += s_sums[w];
                all += s_sums[w];
            }
            const Share share(all, a.even);
            const int64_t begin = share.begin(item);
            left = share.begin(item + 1) - begin;
            if (notes && thread == 0) a.begins[a.batch] = all;
            for (int w = walk; w < end; ++w) {
                const int units = length_of(a, w).units;
                if (notes) a.begins[w] = before;
                if (before <= begin && begin < before + units) {
                    s_walk = w;
                    s_start = begin - before;
                }
                before += units;
            }
            if (left <= 0) return;
            __syncthreads();
            b = s_walk;
            unit = s_start;
        }
    } else if (item >= a.batch) {
        return;
    }
    b = __builtin_amdgcn_readfirstlane(b);

  for (int part = 0; left > 0; part = 1) {
    Length length;
    if (few) {
        length.n = __builtin_amdgcn_readlane(mine.n, b);
        length.first = __builtin_amdgcn_readlane(mine.first, b);
        length.units = __builtin_amdgcn_readlane(mine.units, b);
        length.in = __builtin_amdgcn_readlane(mine.in, b);
    } else {
        length = length_of(a, b);
    }
    const int n = __builtin_amdgcn_readfirstlane(length.n);
    const int first = __builtin_amdgcn_readfirstlane(length.first);
    const int units = __builtin_amdgcn_readfirstlane(length.units);
    const int from_unit = __builtin_amdgcn_readfirstlane(static_cast<int>(unit));
    const int till_unit =
        __builtin_amdgcn_readfirstlane(static_cast<int>(min(unit + left, static_cast<int64_t>(units))));
    const bool idle = !length.in;
    const float q_time = timed ? a.score.q_times[b] : 0.0f;

    // this part's blocks of positions
    const int first_block = first / kKeys, last_block = idle ? first_block : n / kKeys + 1;
    const int block_begin = first_block + from_unit * kUnit;
    const int block_end = min(last_block, first_block + till_unit * kUnit);

    f32x4 o[2 * DB];
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c) o[c] = f32x4{0, 0, 0, 0};
    float m = kFloor, l = 0.0f;

    // The wave's tile of keys and of values.  The next keys are on their way
    // while this block's softmax and values are worked on, the next values
    // while the next scores are: each is waited for by the number of copies
    // asked for after it.
    u32x4* s_k = s_mem + wave * 2 * (G::kSize / 16);
    u32x4* s_v = s_k + G::kSize / 16;
    const uint32_t at_k = lds_address(s_mem) + wave * 2 * static_cast<uint32_t>(G::kSize);
    const uint32_t at_v = at_k + static_cast<uint32_t>(G::kSize);
    constexpr int kCopies = 2 * G::kHalfCopies;

    // Pages of the wave's next 64 blocks, one block's two halves a lane.
    int ids[2];
    auto fetch_ids = [&](int block) {
        const ArgsAgain g = args_again();
        const int32_t* table = g->pages.table + b * g->pages.table_stride;
        const int table_pages = g->pages.table_pages, pages = g->pages.pages;
        const int64_t j = (static_cast<int64_t>(block) + lane * kWaves) * kKeys;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t at = (j + kHalf * h) >> shift;
            const int id = j + kHalf * h <= n && at < table_pages ? table[at] : -1;
            ids[h] = id < pages ? id : -1;
        }
    };
    // The rows of a half that are in the pages and seen: [lo, hi), none where hi <= lo.
    struct Span {
        int page, lo, hi;
    };
    auto span_of = [&](int number, int h, int j0) {
        Span s;
        s.page = __builtin_amdgcn_readlane(ids[h], number);
        const int j = j0 + kHalf * h;
        s.lo = max(first - j, 0);
        s.hi = s.page < 0 ? 0 : min(n - j, kHalf);
        return s;
    };
    // A head's row of a page, in rows.
    auto line_of = [&](int j) { return (static_cast<int64_t>(kv_head) << shift) + (j & page_mask); };
    // Copies of a block's keys or values; rows that are not seen repeat the nearest one
    // that is, and a half without any asks for the query's first 16 bytes, which nothing
    // reads.
    auto fetch = [&](const Span (&s)[2], const char* pool, int64_t page_bytes, int j0, uint32_t to) {
        const ArgsAgain g = args_again();
        const char* nothing = g->q.data + static_cast<int64_t>(b) * g->q.row * sizeof(T);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool none = s[h].hi <= s[h].lo;
            const char* base = uniform(
                none ? nothing : pool + s[h].page * page_bytes + line_of(j0 + kHalf * h) * pitch);
            uint32_t at[G::kHalfCopies];
#pragma unroll
            for (int c = 0; c < G::kHalfCopies; ++c) at[c] = offset[c];
            if (s[h].lo > 0 || s[h].hi < kHalf) {
#pragma unroll
                for (int c = 0; c < G::kHalfCopies; ++c) {
                    const int row = lane / G::kSlots + c * G::kStep;
                    const int near = min(max(row, s[h].lo), s[h].hi - 1);
                    at[c] = none ? 0u : offset[c] + (near - row) * pitch;
                }
            }
#pragma unroll
            for (int c = 0; c < G::kHalfCopies; ++c)
                copy_to_lds(base, at[c], __builtin_amdgcn_readfirstlane(
                                             to + (h * G::kHalfCopies + c) * 1024));
        }
    };
    auto fetch_k = [&](const Span (&s)[2], int j0) {
        const ArgsAgain g = args_again();
        fetch(s, g->pages.k, g->pages.k_page, j0, at_k);
        if constexpr (kEight) {
            // lanes 0 .. 3 and 4 .. 7: four keys' scales each, of the two halves; 8 .. 15:
            // values'; the rest repeat them
            const int h = (lane >> 2) & 1, page = h ? s[1].page : s[0].page;
            const int64_t line = line_of(j0 + kHalf * h) + 4 * (lane & 3);
            const uint8_t* from = lane & 8 ? g->pages.v_scale + page * g->pages.v_scale_page + line
                                           : g->pages.k_scale + page * g->pages.k_scale_page + line;
            if (page < 0) from = reinterpret_cast<const uint8_t*>(g->lens + b);
            copy_far_word_to_lds(from, __builtin_amdgcn_readfirstlane(
                                           lds_address(s_scales) + wave * 256));
        }
        if (timed) {
            const int h = (lane >> 4) & 1, page = h ? s[1].page : s[0].page;
            const float* from = g->k_times + (static_cast<int64_t>(page) << shift) +
                                ((j0 + kHalf * h) & page_mask) + (lane & 15);
            if (page < 0) from = g->score.q_times + b;
            copy_far_word_to_lds(
                from, __builtin_amdgcn_readfirstlane(lds_address(s_times) + wave * 256));
        }
    };
    auto fetch_v = [&](const Span (&s)[2], int j0) {
        const ArgsAgain g = args_again();
        fetch(s, g->pages.v, g->pages.v_page, j0, at_v);
    };
    // The new row takes its place in the wave's tiles, and goes to its page.
    auto put_new = [&](int row, int page, int at_lane) {
        const ArgsAgain g = args_again();
        const T* fresh_k = reinterpret_cast<const T*>(g->k.data) + static_cast<int64_t>(b) * g->k.row +
                           kv_head * g->k.head;
        const T* fresh_v = reinterpret_cast<const T*>(g->v.data) + static_cast<int64_t>(b) * g->v.row +
                           kv_head * g->v.head;
        const bool writes = col_group == 0 && page >= 0;
        const int64_t line = line_of(n);
        char* k_row = g->pages.k + page * g->pages.k_page + line * pitch;
        char* v_row = g->pages.v + page * g->pages.v_page + line * pitch;
        if constexpr (kEight) {
            // eight codes in each lane, by its number in 16
            const int at = at_lane & 15;
            float k[8] = {}, v[8] = {}, k_top = 0.0f, v_top = 0.0f;
            if (at * 8 < dim) {
                load8(fresh_k + at * 8, k);
                load8(fresh_v + at * 8, v);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                k_top = fmaxf(k_top, size_of(k[e]));
                v_top = fmaxf(v_top, size_of(v[e]));
            }
            const int byte_k = scale_byte(group_max<16>(k_top));
            const int byte_v = scale_byte(group_max<16>(v_top));
            const u32x2 codes_k = eight_codes(k, inverse_power(byte_k));
            const u32x2 codes_v = eight_codes(v, inverse_power(byte_v));
            if (at_lane < 16 && at < G::kSlots * 2) {
                const int byte = G::slot(row, at >> 1) * 16 + (at & 1) * 8;
                *reinterpret_cast<u32x2*>(reinterpret_cast<char*>(s_k) + byte) = codes_k;
                *reinterpret_cast<u32x2*>(reinterpret_cast<char*>(s_v) + byte) = codes_v;
            }
            uint8_t* scales = reinterpret_cast<uint8_t*>(s_scales[wave]);
            if (at_lane == 0) {
                scales[row] = byte_k;
                scales[32 + row] = byte_v;
            }
            if (writes && at_lane * 8 < dim) {
                *reinterpret_cast<u32x2*>(k_row + at_lane * 8) = codes_k;
                *reinterpret_cast<u32x2*>(v_row + at_lane * 8) = codes_v;
            }
            if (writes && at_lane == 0) {
                g->pages.k_scale[page * g->pages.k_scale_page + line] = byte_k;
                g->pages.v_scale[page * g->pages.v_scale_page + line] = byte_v;
            }
        } else {
            const u32x4* k_from = reinterpret_cast<const u32x4*>(fresh_k);
            const u32x4* v_from = reinterpret_cast<const u32x4*>(fresh_v);
            if (at_lane < G::kSlots) {
                const int at = at_lane * G::kElems < dim ? at_lane : 0;
                s_k[G::slot(row, at_lane)] = k_from[at];
                s_v[G::slot(row, at_lane)] = v_from[at];
            }
            if (writes && at_lane * G::kElems < dim) {
                reinterpret_cast<u32x4*>(k_row)[at_lane] = k_from[at_lane];
                reinterpret_cast<u32x4*>(v_row)[at_lane] = v_from[at_lane];
            }
        }
        if (writes && timed && kv_head == 0 && at_lane == 0)
            g->k_times[(static_cast<int64_t>(page) << shift) + (n & page_mask)] = q_time;
    };

    // Each round works on a block and asks for the next; the first one only asks (so
    // that the code is there once, which matters where a call is short).
    int block = block_begin + wave - kWaves, number = -1;
    if (block + kWaves < block_end) fetch_ids(block + kWaves);
    F q[DB][kParts];
    {
        const T* row = row_of<const T>(a.q, b, any ? head : 0);
#pragma unroll
        for (int st = 0; st < DB; ++st) {
            const int at = 32 * st + 8 * quarter;
            float x[8] = {};
            if (any && at < dim) load8(row + at, x);
            in_parts<kParts>(x, q[st]);
        }
    }
    Span span[2] = {};
    int works = 0;
#pragma unroll 1
    for (;;) {
        const int j0 = block * kKeys, j1 = j0 + kWaves * kKeys;
        const bool more = block + kWaves < block_end;
        int at_lane = lane;  // LDS addresses are not held over the loop
        asm volatile("" : "+v"(at_lane));
        uint32_t seen = 0;
        uint32_t scales[2][2] = {};  // of keys and values: four bytes a half
        float s[8] = {}, time[8] = {};
        if (works) {
            // keys that count: those of the pages, and the new one
            const bool news = n - j0 < kKeys;
            seen = bits_of(span[0].lo, span[0].hi) | bits_of(span[1].lo, span[1].hi) << 16 |
                   (news ? 1u << (n - j0) : 0u);
            copies_landed<kCopies>();  // keys; the values, asked for last, may be on their way
            if (seen != 0xffffffffu || news) {
                copies_landed<0>();
                // Values of rows that are not seen meet a weight of 0: they may not be NaN,
                // nor infinite.
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    for (int c = at_lane; c < kHalf * G::kSlots; c += 64)
                        if (c / G::kSlots < span[h].lo || c / G::kSlots >= span[h].hi)
                            s_v[h * kHalf * G::kSlots + c] = u32x4{0, 0, 0, 0};
                if (news) {
                    const int page = n - j0 < kHalf ? span[0].page : span[1].page;
                    put_new(n - j0, page, at_lane);
                    if (page < 0) l = NAN;  // no page for the new event: no answer
                }
            }
            f32x4 x[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
            for (int st = 0; st < DB; ++st)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    F k = In::row(s_k, kHalf * h + (at_lane & 15), st, at_lane >> 4);
                    // Past the head size a row repeats its start: an infinity there times q's 0
                    // would be NaN (in 8 bits it is NaN where it is).
                    if (!kEight && st == DB - 1 && 32 * st + 8 * (at_lane >> 4) >= dim) k = F{};
#pragma unroll
                    for (int p = 0; p < kParts; ++p) x[h] = mma16(k, q[st][p], x[h]);
                }
            if constexpr (kEight) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    scales[0][h] = s_scales[wave][4 * h + (at_lane >> 4)];
                    scales[1][h] = s_scales[wave][8 + 4 * h + (at_lane >> 4)];
                }
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                s[r] = x[r >> 2][r & 3];
                if constexpr (kEight) s[r] *= power_of((scales[0][r >> 2] >> (8 * (r & 3))) & 255);
            }
            if (timed) {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    time[r] = s_times[wave][kHalf * (r >> 2) + 4 * (at_lane >> 4) + (r & 3)];
            }
            reads_done();  // so the next keys may come
        }
        if (more) {
            number = (number + 1) & 63;
            if (number == 0 && works) fetch_ids(block + kWaves);
#pragma unroll
            for (int h = 0; h < 2; ++h) span[h] = span_of(number, h, j1);
            fetch_k(span, j1);
        }
        if (works) {
            if (softcap > 0) {
                const ArgsAgain g = args_again();
                Score sc;
                sc.cap_in = g->score.cap_in;
                sc.cap_out = g->score.cap_out;
                sc.scale = g->score.scale;
                sc.scale2 = scale2;
                sc.softcap = softcap;
                float unused;
#pragma unroll
                for (int r = 0; r < 8; ++r) s[r] = capped<T, kWide>(sc, s[r], unused);
            } else {
#pragma unroll
                for (int r = 0; r < 8; ++r) s[r] *= scale2;
            }
            // distances from the new event of register r's key: last_d - at(r)
            const int last_d = n - j0 - 4 * quarter;
            auto at = [](int r) { return kHalf * (r >> 2) + (r & 3); };
            if (biased) {
                const ArgsAgain g = args_again();
                Score sc;
                sc.table = g->score.table;
                sc.buckets = g->score.buckets;
                sc.num_buckets = g->score.num_buckets;
                sc.reach = g->score.reach;
                if (n - (j0 + kKeys - 1) >= sc.reach) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) s[r] += far_bias;
                } else if (any) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const int d = min(max(last_d - at(r), 0), sc.reach);
                        s[r] += table_entry(sc, head, d + sc.reach);
                    }
                }
            }
            if (sloped) {
                if (timed) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        // the new event's own time is not in the pages yet: it is 0 away
                        const float gap = q_time - time[r];
                        s[r] = fmaf(-slope, last_d == at(r) ? 0.0f : fabsf(gap), s[r]);
                    }
                } else {
                    const float from = static_cast<float>(last_d);
#pragma unroll
                    for (int r = 0; r < 8; ++r) s[r] = fmaf(-slope, fabsf(from - at(r)), s[r]);
                }
            }
            const uint32_t mine = seen >> (4 * quarter);
            if (seen != 0xffffffffu) {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (!(mine >> at(r) & 1)) s[r] = -INFINITY;
            }
            float top = s[0];
#pragma unroll
            for (int r = 1; r < 8; ++r) top = fmaxf(top, s[r]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            if (__any(top > m)) {
                const float grown = fmaxf(m, top);
                const float by = exp2_fast(m - grown);
                m = grown;
                l *= by;
#pragma unroll
                for (int c = 0; c < 2 * DB; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[c][r] *= by;
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                s[r] = exp2_fast(s[r] - m) * kLargest;
                l += s[r];
            }
            if constexpr (kEight) {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    s[r] *= power_of((scales[1][r >> 2] >> (8 * (r & 3))) & 255);
                if (seen != 0xffffffffu) {  // whatever is in the place of a scale
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (!(mine >> at(r) & 1)) s[r] = 0.0f;
                }
            }
            F p[kWeights];
            if constexpr (kEight || sizeof(T) == 4) in_parts<kWeights>(s, p);
            else in_positive_parts(s, p);
            if (more) copies_landed<kCopies>();  // values; the next keys may be on their way
            else copies_landed<0>();
#pragma unroll
            for (int c = 0; c < 2 * DB; ++c) {
                const F v = In::columns(s_v, c, at_lane);
#pragma unroll
                for (int w = 0; w < kWeights; ++w) o[c] = mma16(v, p[w], o[c]);
            }
            reads_done();
        }
        if (!more) break;
        fetch_v(span, j1);
        block += kWaves;
        asm volatile("s_mov_b32 %0, 1" : "=s"(works));
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // join the waves
    if (quarter == 0) {
        s_m[wave][lane] = m;
        s_l[wave][lane] = l;
    }
    __syncthreads();  // also: the tiles are done with
    float* s_join = reinterpret_cast<float*>(s_mem);
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c)
        *reinterpret_cast<f32x4*>(s_join + (wave * kColumns + (lane & 15)) * kJoinPitch + 16 * c +
                                  4 * quarter) = o[c];
    __syncthreads();
    const int columns = min(a.group - col_group * kColumns, kColumns);
    const int pieces = dim / 4;
    for (int i = thread; i < columns * pieces; i += kThreads) {
        const int jc = i / pieces, d = i % pieces * 4;
        float top = s_m[0][jc], total = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_m[w][jc]);
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float by = exp2_fast(s_m[w][jc] - top);
            total = fmaf(by, s_l[w][jc], total);
            const f32x4 part =
                *reinterpret_cast<const f32x4*>(s_join + (w * kColumns + jc) * kJoinPitch + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = fmaf(by, part[e], sum[e]);
        }
        if (idle && a.lens[b] >= 0) total = NAN;  // no room for the new event: no answer
        if (from_unit > 0 || till_unit < units) {
            const int64_t at = (static_cast<int64_t>(blockIdx.x) * 2 + part) * kColumns + jc;
            *reinterpret_cast<f32x4*>(a.partial + at * dim + d) = sum;
            if (d == 0) a.part_stats[at] = make_float2(top, total);
        } else {
            const int join_head = kv_head * a.group + col_group * kColumns + jc;
            typedef T t4 __attribute__((ext_vector_type(4)));
            t4 out;
#pragma unroll
            for (int e = 0; e < 4; ++e)  // a total of 0: an idle row, or the bias masks everything
                out[e] = static_cast<T>(total != 0.0f ? sum[e] / total : 0.0f);
            *reinterpret_cast<t4*>(row_of<T>(a.out, b, join_head) + d) = out;
        }
    }
    if (!a.even) return;
    left -= till_unit - from_unit;
    unit = 0;
    ++b;
    __syncthreads();  // the join's room is the next part's tiles
  }
}

// Joins the parts of walks that were cut: 32 threads for the elements of a head, four
// each, and kShares shares of the parts.
template <typename T, int kShares, int kSize>
__global__ __launch_bounds__(kSize) void join_parts_kernel(PagedArgs a) {
    constexpr int kHeads = kSize / 32 / kShares;
    __shared__ f32x4 s_sum[kHeads][kShares][32];
    __shared__ float s_total[kHeads][kShares];
    const int thread = threadIdx.x, lane = thread & 31, share = thread / 32 % kShares;
    const int mine = thread / 32 / kShares, groups = (a.heads + kHeads - 1) / kHeads;
    const int b = blockIdx.x / groups;
    const int head = min(static_cast<int>(blockIdx.x % groups) * kHeads + mine, a.heads - 1);
    const int64_t begin = a.begins[b], end = a.begins[b + 1], all = a.begins[a.batch];
    const Share share_of(all, a.even);
    const int first = share_of.owner(begin), parts = share_of.owner(end - 1) - first + 1;
    if (parts == 1) return;
    const int kv_head = head / a.group, col = head % a.group;
    // The first workgroup's part is its last one, unless the walk begins it; the others'
    // is their first one.
    const int begun = share_of.begin(first) < begin;
    auto part_of = [&](int s) {
        const int item = first + s;
        const int64_t block =
            (static_cast<int64_t>(item / 8 * a.kv_heads + kv_head) * a.columns + col / kColumns) * 8 +
            item % 8;
        return (block * 2 + (s == 0 ? begun : 0)) * kColumns + col % kColumns;
    };
    const int d = lane * 4;
    float top = kFloor;
    for (int s = lane; s < parts; s += 32) top = fmaxf(top, a.part_stats[part_of(s)].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    float total = 0.0f;
    f32x4 sum = {0, 0, 0, 0};
    // No branch inside, so that several parts' loads are in flight: threads past the
    // head size read its last elements again and store nothing.
    const int from = min(d, a.dim - 4);
#pragma unroll 4
    for (int s = share; s < parts; s += kShares) {
        const int64_t at = part_of(s);
        const float2 st = a.part_stats[at];
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.partial + at * a.dim + from);
        const float by = exp2_fast(st.x - top);
        total = fmaf(by, st.y, total);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = fmaf(by, x[e], sum[e]);
    }
    if constexpr (kShares > 1) {
        s_sum[mine][share][lane] = sum;
        if (lane == 0) s_total[mine][share] = total;
        __syncthreads();
        if (share) return;
#pragma unroll
        for (int w = 1; w < kShares; ++w) {
            total += s_total[mine][w];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += s_sum[mine][w][lane][e];
        }
    }
    if (d >= a.dim) return;
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = static_cast<T>(total != 0.0f ? sum[e] / total : 0.0f);
    *reinterpret_cast<t4*>(row_of<T>(a.out, b, head) + d) = out;
}

// Workgroups of a key head among which all walks are evened out; 0: one a walk.
// A workgroup takes some 20 ns for each position of a walk that it has alone, and tables say
// how many that can be.  Evened out there is a second launch, and each workgroup adds up all
// lengths, 5 ns a walk.  So walks have a workgroup each where none can have more than 512
// positions, than 128 for each walk that a workgroup's place takes in turn (then one that
// is that long adds up to 28 %), or than a quarter of the walks' number.  One each and
// evened out, us in 16 bits with 8 heads of 128: 512 walks of 0 to 511 events, room for
// 2048, 125 and 133, with one of 100,000 among them 1769 and 217; 512 of 0 to 2000 361 and
// 366; 1024 of 0 to 1000 370 and 378; 1024 of 0 to 100 and one of 1900 152 and 119; 4096 of
// 0 to 200 and one of 20,000 940 and 609; 100,000 of 0 to 100, one head of 64, 749 and 1244.
int even_of(const trw_paged_step_params& p, int resident) {
    const int group = p.heads / p.pages.kv_heads;
    const int64_t heads = int64_t{p.pages.kv_heads} * ((group + kColumns - 1) / kColumns);
    const int64_t slots = 256 * resident, walks = p.pages.walks;
    const int64_t room = p.pages.table_pages * p.pages.page_rows;
    if (room <= std::max({int64_t{4 * kUnit * kKeys}, 128 * walks * heads / slots, walks / 4}))
        return 0;
    return static_cast<int>(std::max<int64_t>(1, slots / heads));
}
int even_of(const trw_paged_step_params& p) {
    int even = 0;
    dispatch(p.dtype, p.pages.dim, [&](auto t, auto db) {
        typedef decltype(t) T;
        constexpr int DB = decltype(db)::value;
        even = even_of(p, p.pages.dtype == TRW_E4M3 ? kResident<T, DB, true> : kResident<T, DB, false>);
    });
    return even;
}
int64_t grid_of(const trw_paged_step_params& p, int even) {
    const int group = p.heads / p.pages.kv_heads;
    const int columns = (group + kColumns - 1) / kColumns;
    return xcd_grid(even ? even : p.pages.walks) * p.pages.kv_heads * columns;
}

}  // namespace

uint64_t paged_step_workspace(const trw_paged_step_params& p) {
    const int even = even_of(p);
    if (!even) return 0;
    return grid_of(p, even) * 2 * kColumns * (p.pages.dim + 2) * sizeof(float) +
           (p.pages.walks + 1) * sizeof(int64_t);
}

void paged_step(const trw_paged_step_params& p, hipStream_t stream) {
    const int64_t batch = p.pages.walks;
    require(batch == 0 || p.workspace_bytes >= paged_step_workspace(p), "workspace is too small");
    require_apart(p.pages);
    if (batch == 0) return;
    PagedArgs a;
    a.pages = make_pages(p.pages);
    a.q = make_rows(p.q);
    a.k = make_rows(p.k);
    a.v = make_rows(p.v);
    a.out = make_rows(p.out);
    a.lens = p.lens;
    a.first = p.first;
    a.k_times = const_cast<float*>(p.score.k_times);
    a.score = make_score(p.score);
    a.batch = static_cast<int>(batch);
    a.heads = p.heads;
    a.kv_heads = p.pages.kv_heads;
    a.group = p.heads / p.pages.kv_heads;
    a.columns = (a.group + kColumns - 1) / kColumns;
    a.dim = p.pages.dim;
    a.even = even_of(p);
    const int64_t grid = grid_of(p, a.even);
    require_grid(grid, kThreads);
    a.partial = static_cast<float*>(p.workspace);
    a.part_stats = reinterpret_cast<float2*>(a.partial + grid * 2 * kColumns * a.dim);
    a.begins = reinterpret_cast<int64_t*>(a.part_stats + grid * 2 * kColumns);
    dispatch(p.dtype, a.dim, [&](auto t, auto db) {
        typedef decltype(t) T;
        by_cap<T>(p.dtype, p.score, [&](auto wide) {
            constexpr int DB = decltype(db)::value;
            constexpr bool kWide = decltype(wide)::value;
            if (p.pages.dtype == TRW_E4M3)
                hipLaunchKernelGGL((paged_step_kernel<T, DB, kWide, true>),
                                   dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, a);
            else
                hipLaunchKernelGGL((paged_step_kernel<T, DB, kWide, false>),
                                   dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, a);
        });
        check_launch("paged_attention_step");
        if (a.even) {
            // Parts of a walk: a head's by 32 shares where there are many (3 walks of
            // 260k events together, 128 parts each: 7.8 us), else eight heads a workgroup
            // (64 walks over 96 workgroups: 4.7 us).
            const bool many = a.even > 8 * batch;
            const int64_t joins = batch * (many ? a.heads : (a.heads + 7) / 8);
            require_grid(joins, many ? 1024 : 256);
            if (many)
                hipLaunchKernelGGL((join_parts_kernel<T, 32, 1024>),
                                   dim3(static_cast<unsigned>(joins)), dim3(1024), 0, stream, a);
            else
                hipLaunchKernelGGL((join_parts_kernel<T, 1, 256>),
                                   dim3(static_cast<unsigned>(joins)), dim3(256), 0, stream, a);
            check_launch("paged_attention_step");
        }
    });
}

}  // namespace ops
}  // namespace trw
