// attention_paged.hip -- one new event of each walk over its pages.
//
// Per walk and key head: read the pages once, at memory speed.  The query heads
// that share a key head are the columns of the products, 16 of them; a wave takes
// blocks of 32 positions (two halves of 16, each in one page), four waves and,
// where walks are few, many workgroups share a walk: each keeps a maximum, a sum
// and an output of its own, joined at the end.  Positions that the walk does not
// see are never read.
//
// v_mfma_f32_16x16x32 with keys as rows leaves lane l with keys 4 (l / 16) .. + 4
// of column l & 15.  Two halves give eight, which are the B operand of the next
// product without moving: its element e of lane l is key 4 (l / 16) + e of the
// first half, e < 4, or key 4 (l / 16) + e - 4 of the second, and the values are
// read from LDS in the same order.
//
// 8 bits: codes are exact in bfloat16, and the products are bfloat16's whatever
// the type of q.  Keys' scales multiply scores and values' scales the softmax's
// weights, in float32 and exactly (they are powers of two).  q and the weights of
// longer types go as two (float16) or three (float32) bfloat16 parts, which lose
// nothing of q and 2^-16 and 2^-24 of a weight.
//
// The new row is taken from the call's arguments by the workgroup whose positions
// include it (in 8 bits as the codes that the pages get), and written to the pages
// by the walk's first workgroup: no launch and no wait between the two.
#include <algorithm>

#include "pages.h"
#include "step_join.h"

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
    int batch, heads, kv_heads, group, columns, dim, splits;
    float* partial;      // [batch, heads, splits, dim]
    float2* part_stats;  // [batch, heads, splits]
};

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

// Rows lo .. hi - 1 of a half as bits.
__device__ __forceinline__ uint32_t bits_of(int lo, int hi) {
    return hi > lo ? ((1u << hi) - 1) & ~((1u << lo) - 1) : 0u;
}

template <typename T, int DB, bool kWide, bool kEight>
__global__ __launch_bounds__(kThreads, kEight ? (DB <= 2 ? 4 : 3) : sizeof(T) == 2 ? (DB <= 2 ? 4 : 2) : 1)
void paged_step_kernel(PagedArgs a) {
    typedef std::conditional_t<kEight, Eight<DB>, Wide<T, DB>> In;
    typedef typename In::G G;
    typedef typename In::F F;
    constexpr int kBytes = kEight ? 1 : sizeof(T);
    constexpr int kParts = !kEight ? 1 : sizeof(T) == 4 ? 3 : std::is_same<T, __bf16>::value ? 1 : 2;
    constexpr int kJoinPitch = 32 * DB + 4;
    constexpr size_t kJoinBytes = size_t(kWaves) * kColumns * kJoinPitch * sizeof(float);
    constexpr size_t kTileBytes = 2 * kWaves * G::kSize;
    __shared__ u32x4 s_mem[(kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes) / 16];
    __shared__ float s_m[kWaves][kColumns], s_l[kWaves][kColumns];
    __shared__ float s_times[kWaves][64];
    __shared__ uint32_t s_scales[kEight ? kWaves : 1][64];  // keys' 32 bytes, values' 32

    // Consecutive workgroups go to the eight XCDs in turn: each takes all key
    // heads of some positions.
    int rest = blockIdx.x / 8;
    const int col_group = rest % a.columns;
    rest /= a.columns;
    const int kv_head = rest % a.kv_heads;
    const int item = rest / a.kv_heads * 8 + blockIdx.x % 8;
    const int split = item % a.splits;
    const int b = item / a.splits;
    if (b >= a.batch) return;
    const int thread = threadIdx.x, lane = thread & 63, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const Score& sc = a.score;
    const Pages& pages = a.pages;
    const int shift = pages.shift, page_mask = (1 << shift) - 1;

    const int64_t at_n = a.lens[b];  // position of the new event
    const int64_t room = static_cast<int64_t>(pages.table_pages) << shift;
    const int new_page = at_n >= 0 && at_n < room ? pages.page_of(b, at_n) : -1;
    const bool idle = new_page < 0;
    const int n = idle ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(at_n));
    const int64_t at_first = a.first ? a.first[b] : 0;
    const int first = __builtin_amdgcn_readfirstlane(
        static_cast<int>(min(max(at_first, int64_t{0}), static_cast<int64_t>(n))));
    const int col = col_group * kColumns + (lane & 15);
    const int head = kv_head * a.group + col;
    const bool any = !idle && col < a.group;
    const T* fresh_k = row_of<const T>(a.k, b, kv_head);
    const T* fresh_v = row_of<const T>(a.v, b, kv_head);
    const float q_time = sc.q_times ? sc.q_times[b] : 0.0f;

    // The new row as codes, eight of them in each lane by its number in 16.
    u32x2 codes_k = {0, 0}, codes_v = {0, 0};
    int byte_k = 0, byte_v = 0;
    auto encode = [&]() {
        const int from = (lane & 15) * 8;
        float k[8] = {}, v[8] = {}, k_top = 0.0f, v_top = 0.0f;
        if (from < a.dim) {
            load8(fresh_k + from, k);
            load8(fresh_v + from, v);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            k_top = fmaxf(k_top, size_of(k[e]));
            v_top = fmaxf(v_top, size_of(v[e]));
        }
        byte_k = scale_byte(group_max<16>(k_top));
        byte_v = scale_byte(group_max<16>(v_top));
        codes_k = eight_codes(k, inverse_power(byte_k));
        codes_v = eight_codes(v, inverse_power(byte_v));
    };

    if (!idle && split == 0 && col_group == 0 && wave == 0) {
        const int64_t line = (static_cast<int64_t>(kv_head) << shift) + (n & page_mask);
        char* k_row = pages.k + new_page * pages.k_page + line * a.dim * kBytes;
        char* v_row = pages.v + new_page * pages.v_page + line * a.dim * kBytes;
        if constexpr (kEight) {
            encode();
            if (lane * 8 < a.dim) {
                *reinterpret_cast<u32x2*>(k_row + lane * 8) = codes_k;
                *reinterpret_cast<u32x2*>(v_row + lane * 8) = codes_v;
            }
            if (lane == 0) {
                pages.k_scale[new_page * pages.k_scale_page + line] = byte_k;
                pages.v_scale[new_page * pages.v_scale_page + line] = byte_v;
            }
        } else if (lane * G::kElems < a.dim) {
            reinterpret_cast<u32x4*>(k_row)[lane] = reinterpret_cast<const u32x4*>(fresh_k)[lane];
            reinterpret_cast<u32x4*>(v_row)[lane] = reinterpret_cast<const u32x4*>(fresh_v)[lane];
        }
        if (a.k_times && kv_head == 0 && lane == 0)
            a.k_times[(static_cast<int64_t>(new_page) << shift) + (n & page_mask)] = q_time;
    }

    // this workgroup's blocks of positions
    const int first_block = first / kKeys;
    const int64_t blocks = idle ? 0 : n / kKeys + 1 - first_block;
    const int block_begin = first_block + static_cast<int>(blocks * split / a.splits);
    const int block_end = first_block + static_cast<int>(blocks * (split + 1) / a.splits);

    F q[DB][kParts];
    {
        const T* row = row_of<const T>(a.q, b, any ? head : 0);
#pragma unroll
        for (int st = 0; st < DB; ++st) {
            const int at = 32 * st + 8 * quarter;
            float x[8] = {};
            if (any && at < a.dim) load8(row + at, x);
            in_parts<kParts>(x, q[st]);
        }
    }
    const float slope = sc.slopes && any ? sc.slopes[head] * kLog2e : 0.0f;
    const float far_bias = sc.table && any ? table_entry(sc, head, 2 * sc.reach) : 0.0f;

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
    const int pitch = a.dim * kBytes;
    constexpr int kCopies = 2 * G::kHalfCopies;
    uint32_t offset[G::kHalfCopies];  // bytes from a half's first row
#pragma unroll
    for (int c = 0; c < G::kHalfCopies; ++c) {
        const int row = lane / G::kSlots + c * G::kStep;
        const int chunk = (lane % G::kSlots) ^ G::swizzle(row);
        offset[c] = row * pitch + (chunk * 16 < pitch ? chunk * 16 : 0);
    }

    // Pages of the wave's next 64 blocks, one block's two halves a lane.
    int ids[2];
    auto fetch_ids = [&](int block) {
        const int64_t j = (static_cast<int64_t>(block) + lane * kWaves) * kKeys;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            ids[h] = j + kHalf * h <= n ? pages.page_of(b, j + kHalf * h) : -1;
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
    // Copies of one half; rows that are not seen repeat the nearest one that is,
    // and a half without any asks for the query's first 16 bytes, which nothing reads.
    auto fetch_half = [&](const Span& s, const char* pool, int64_t page_bytes, int j, uint32_t to) {
        const bool none = s.hi <= s.lo;
        const int64_t line = (static_cast<int64_t>(kv_head) << shift) + (j & page_mask);
        const char* base = uniform(none ? a.q.data + static_cast<int64_t>(b) * a.q.row * sizeof(T)
                                        : pool + s.page * page_bytes + line * pitch);
        if (s.lo == 0 && s.hi == kHalf) {
#pragma unroll
            for (int c = 0; c < G::kHalfCopies; ++c) copy_to_lds(base, offset[c], to + c * 1024);
        } else {
#pragma unroll
            for (int c = 0; c < G::kHalfCopies; ++c) {
                const int row = lane / G::kSlots + c * G::kStep;
                const int near = min(max(row, s.lo), s.hi - 1);
                copy_to_lds(base, none ? 0u : offset[c] + (near - row) * pitch, to + c * 1024);
            }
        }
    };
    auto fetch_k = [&](const Span (&s)[2], int j0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            fetch_half(s[h], pages.k, pages.k_page, j0 + kHalf * h,
                       __builtin_amdgcn_readfirstlane(at_k + h * (uint32_t(G::kSize) / 2)));
        if constexpr (kEight) {
            // lanes 0 .. 3 and 4 .. 7: four keys' scales each, of the two halves; 8 .. 15:
            // values'; the rest repeat them
            const int h = (lane >> 2) & 1;
            const Span mine = h ? s[1] : s[0];
            const int64_t line = (static_cast<int64_t>(kv_head) << shift) +
                                 ((j0 + kHalf * h) & page_mask) + 4 * (lane & 3);
            const uint8_t* from = lane & 8 ? pages.v_scale + mine.page * pages.v_scale_page + line
                                           : pages.k_scale + mine.page * pages.k_scale_page + line;
            if (mine.page < 0) from = reinterpret_cast<const uint8_t*>(a.lens + b);
            copy_far_word_to_lds(from, __builtin_amdgcn_readfirstlane(
                                           lds_address(s_scales) + wave * 256));
        }
        if (a.k_times) {
            const int h = (lane >> 4) & 1;
            const Span mine = h ? s[1] : s[0];
            const float* from = a.k_times + (static_cast<int64_t>(mine.page) << shift) +
                                ((j0 + kHalf * h) & page_mask) + (lane & 15);
            if (mine.page < 0) from = sc.q_times + b;
            copy_far_word_to_lds(
                from, __builtin_amdgcn_readfirstlane(lds_address(s_times) + wave * 256));
        }
    };
    auto fetch_v = [&](const Span (&s)[2], int j0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            fetch_half(s[h], pages.v, pages.v_page, j0 + kHalf * h,
                       __builtin_amdgcn_readfirstlane(at_v + h * (uint32_t(G::kSize) / 2)));
    };

    int block = block_begin + wave, number = 0;
    Span span[2];
    if (block < block_end) {
        fetch_ids(block);
#pragma unroll
        for (int h = 0; h < 2; ++h) span[h] = span_of(0, h, block * kKeys);
        fetch_k(span, block * kKeys);
        fetch_v(span, block * kKeys);
    }
#pragma unroll 1
    for (; block < block_end; block += kWaves) {
        const int j0 = block * kKeys, j1 = j0 + kWaves * kKeys;
        const bool more = block + kWaves < block_end;
        int at_lane = lane;  // LDS addresses are not held over the loop
        asm volatile("" : "+v"(at_lane));
        // keys that count: those of the pages, and the new one
        const uint32_t seen = bits_of(span[0].lo, span[0].hi) | bits_of(span[1].lo, span[1].hi) << 16 |
                              (n - j0 < kKeys ? 1u << (n - j0) : 0u);
        copies_landed<kCopies>();  // keys; the values, asked for last, may be on their way
        if (seen != 0xffffffffu || n - j0 < kKeys) {
            copies_landed<0>();
            // Values of rows that are not seen meet a weight of 0: they may not be NaN.
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (span[h].hi <= span[h].lo)
                    for (int c = at_lane; c < kHalf * G::kSlots; c += 64)
                        s_v[h * kHalf * G::kSlots + c] = u32x4{0, 0, 0, 0};
            if (n - j0 < kKeys) {  // the new row, from its place on
                const int from = n - j0;
                if constexpr (kEight) {
                    encode();
                    const int at = at_lane & 15;
                    for (int row = from + (at_lane >> 4); row < kKeys; row += 4) {
                        if (at < G::kSlots * 2) {
                            const int byte = G::slot(row, at >> 1) * 16 + (at & 1) * 8;
                            *reinterpret_cast<u32x2*>(reinterpret_cast<char*>(s_k) + byte) = codes_k;
                            *reinterpret_cast<u32x2*>(reinterpret_cast<char*>(s_v) + byte) = codes_v;
                        }
                        uint8_t* scales = reinterpret_cast<uint8_t*>(s_scales[wave]);
                        scales[row] = byte_k;
                        scales[32 + row] = byte_v;
                    }
                } else {
                    for (int c = from * G::kSlots + at_lane; c < kKeys * G::kSlots; c += 64) {
                        const int row = c / G::kSlots, chunk = c % G::kSlots;
                        const int at = chunk * G::kElems < a.dim ? chunk : 0;
                        s_k[G::slot(row, chunk)] = reinterpret_cast<const u32x4*>(fresh_k)[at];
                        s_v[G::slot(row, chunk)] = reinterpret_cast<const u32x4*>(fresh_v)[at];
                    }
                }
            }
        }
        f32x4 x[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int st = 0; st < DB; ++st)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const F k = In::row(s_k, kHalf * h + (at_lane & 15), st, at_lane >> 4);
#pragma unroll
                for (int p = 0; p < kParts; ++p) x[h] = mma16(k, q[st][p], x[h]);
            }
        uint32_t scales[2][2];  // of keys and values: four bytes a half
        if constexpr (kEight) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                scales[0][h] = s_scales[wave][4 * h + (at_lane >> 4)];
                scales[1][h] = s_scales[wave][8 + 4 * h + (at_lane >> 4)];
            }
        }
        float s[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            float product = x[r >> 2][r & 3];
            if constexpr (kEight) product *= power_of((scales[0][r >> 2] >> (8 * (r & 3))) & 255);
            float unused;
            s[r] = sc.softcap > 0 ? capped<T, kWide>(sc, product, unused) : product * sc.scale2;
        }
        float time[8];
        if (a.k_times) {
#pragma unroll
            for (int r = 0; r < 8; ++r)
                time[r] = s_times[wave][kHalf * (r >> 2) + 4 * (at_lane >> 4) + (r & 3)];
        }
        reads_done();
        if (more) {
            number = (number + 1) & 63;
            if (number == 0) fetch_ids(block + kWaves);
#pragma unroll
            for (int h = 0; h < 2; ++h) span[h] = span_of(number, h, j1);
            fetch_k(span, j1);
        }
        // distances from the new event of register r's key: last_d - at(r)
        const int last_d = n - j0 - 4 * quarter;
        auto at = [](int r) { return kHalf * (r >> 2) + (r & 3); };
        if (sc.table) {
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
        if (sc.slopes) {
            if (a.k_times) {
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
            s[r] = exp2_fast(s[r] - m);
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
        F p[kParts];
        in_parts<kParts>(s, p);
        if (more) copies_landed<kCopies>();  // values; the next keys may be on their way
        else copies_landed<0>();
#pragma unroll
        for (int c = 0; c < 2 * DB; ++c) {
            const F v = In::columns(s_v, c, at_lane);
#pragma unroll
            for (int part = 0; part < kParts; ++part) o[c] = mma16(v, p[part], o[c]);
        }
        reads_done();
        if (more) fetch_v(span, j1);
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
    const int pieces = a.dim / 4;
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
        // no page for the new event: no answer
        if (idle && at_n >= 0) total = NAN;
        const int join_head = kv_head * a.group + col_group * kColumns + jc;
        const int64_t part = (static_cast<int64_t>(b) * a.heads + join_head) * a.splits + split;
        if (a.splits > 1) {
            *reinterpret_cast<f32x4*>(a.partial + part * a.dim + d) = sum;
            if (d == 0) a.part_stats[part] = make_float2(top, total);
        } else {
            typedef T t4 __attribute__((ext_vector_type(4)));
            t4 out;
#pragma unroll
            for (int e = 0; e < 4; ++e)  // a total of 0: an idle row, or the bias masks everything
                out[e] = static_cast<T>(total != 0.0f ? sum[e] / total : 0.0f);
            *reinterpret_cast<t4*>(row_of<T>(a.out, b, join_head) + d) = out;
        }
    }
}

// Workgroups of one walk and key head: each with at least four blocks a wave
// where the table is full; few walks: 1536 workgroups in all, more: three each up
// to 3072, which evens out their lengths.
int splits_of(const trw_paged_step_params& p) {
    const int group = p.heads / p.pages.kv_heads;
    const int64_t items = p.pages.walks * p.pages.kv_heads * ((group + kColumns - 1) / kColumns);
    const int64_t capacity = p.pages.table_pages * p.pages.page_rows;
    const int64_t most = (capacity + 4 * kWaves * kKeys - 1) / (4 * kWaves * kKeys);
    const int64_t n = std::max<int64_t>(items, 1);
    const int64_t want = std::max((1536 + n - 1) / n, std::min<int64_t>(3, 3072 / n));
    return static_cast<int>(std::max<int64_t>(1, std::min(want, most)));
}

}  // namespace

uint64_t paged_step_workspace(const trw_paged_step_params& p) {
    const int splits = splits_of(p);
    if (splits == 1) return 0;
    return static_cast<uint64_t>(p.pages.walks) * p.heads * splits * (p.pages.dim + 2) *
           sizeof(float);
}

void paged_step(const trw_paged_step_params& p, hipStream_t stream) {
    const int64_t batch = p.pages.walks;
    if (batch == 0) return;
    require(p.workspace_bytes >= paged_step_workspace(p), "workspace is too small");
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
    a.splits = splits_of(p);
    a.partial = static_cast<float*>(p.workspace);
    a.part_stats = reinterpret_cast<float2*>(a.partial + batch * p.heads * a.splits * a.dim);
    const int64_t grid = xcd_grid(batch * a.splits) * a.kv_heads * a.columns;
    require_grid(grid, kThreads);
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
        if (a.splits > 1) {
            const StepJoin join{a.partial, a.part_stats, a.out, nullptr, 0, a.heads, a.dim, a.splits};
            hipLaunchKernelGGL((join_step_kernel<T>), dim3(static_cast<unsigned>(batch * a.heads)),
                               dim3(kJoinThreads), 0, stream, join);
            check_launch("paged_attention_step");
        }
    });
}

}  // namespace ops
}  // namespace trw
