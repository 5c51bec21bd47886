// operators.h -- what the operator kernels share: element types, matrix
// instructions, tiles in LDS, scores.
//
// All attention kernels hold the matrix products the same way round.  A wave
// owns 32 columns (query rows in the forward and dQ kernels, keys in the dK/dV
// kernel), one per lane of each half wave, whose vectors stay in registers as
// the B operand; the other side's rows pass through LDS and are the A operand.
// v_mfma_f32_32x32x16 then leaves lane l with 16 rows of column l & 31 (and
// lane l ^ 32 with the other 16), so a softmax over rows is a sum over a
// lane's own registers and one exchange with lane l ^ 32, and the 16 values
// are, two by two, the B operand of the next product without moving: register
// 8 t + e is row 16 t + 8 (e / 4) + 4 (l / 32) + e % 4, and the A operand of
// that product is read from LDS in the same order of rows.
#ifndef TRW_OPERATORS_KERNELS_H
#define TRW_OPERATORS_KERNELS_H

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>
#include <type_traits>

#include "tile_rows.h"
#include "trw_operators.h"

namespace trw {
namespace ops {

struct InvalidArgument : std::invalid_argument {
    using std::invalid_argument::invalid_argument;
};
inline void require(bool ok, const char* message) {
    if (!ok) throw InvalidArgument(message);
}
// A launch has fewer than 2^32 threads.
inline void require_grid(int64_t groups, int threads) {
    require(groups < (int64_t{1} << 32) / threads, "too many rows, documents or heads for a launch");
}
inline void check_launch(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) throw std::runtime_error(std::string(what) + ": " + hipGetErrorString(e));
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Where a running maximum starts: below every finite score (scores are clamped
// to kLowest), above the -inf of masked ones, so that exp2(score - maximum) is
// 0 for those and never NaN.
constexpr float kFloor = -3.0e38f;
constexpr float kLowest = -1.0e38f;

// The first row of an interval that has none: past every row (rows are below
// 2^30), and row indices counted up from it do not overflow.
constexpr int kNone = 1 << 30;

// Eight values of one lane: one operand of a product over 16.
template <typename T>
struct Lane8;
template <>
struct Lane8<__bf16> {
    typedef bf16x8 vec;
};
template <>
struct Lane8<_Float16> {
    typedef f16x8 vec;
};
template <>
struct Lane8<float> {
    typedef f32x8 vec;
};
template <typename T>
using Frag = typename Lane8<T>::vec;

// c += A B over 16: lane l holds elements 8 (l / 32) .. + 8 of row (column)
// l & 31 of A (B).
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.0f;
    return z;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// No LDS read moves across: where the compiler would read all operands of a
// chain of products ahead and run out of registers for them.
__device__ __forceinline__ void hold_reads() { asm volatile("" ::: "memory"); }

// Row of accumulator register r: 8 (r / 4) + 4 (lane / 32) + r % 4.
__device__ __forceinline__ constexpr int acc_row(int r) { return 8 * (r >> 2) + (r & 3); }

// ---- tiles of rows in LDS --------------------------------------------------------------------
//
// Rows of 32, 64 or 128 elements as 16-byte chunks, chunk c of row r in slot
// c ^ swizzle(r) of the row.  Both ways the tiles are read then touch every
// bank once: 16 consecutive rows' chunk c (row reads) lie in 16 slots of the
// 256 bytes that the banks span, and so do 4 consecutive rows' 64-byte pieces
// (transposing reads).
template <typename T, int DB>
struct Tile {
    static constexpr int kElems = 16 / sizeof(T);  // of a chunk
    static constexpr int kWidth = DB == 1 ? 32 : DB == 2 ? 64 : 128;
    static constexpr int kSlots = kWidth / kElems;    // per row
    static constexpr int kUsed = DB * 32 / kElems;    // chunks per row that are read
    static constexpr int kSteps = DB * 2;             // products over 16 in a row

    static constexpr size_t bytes(int rows) { return size_t(rows) * kSlots * 16; }

    __device__ static __forceinline__ int swizzle(int r) {
        if (kSlots == 4) return (r >> 2) & 3;
        if (kSlots == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        return ((r & 3) << 2) | ((r >> 2) & 3);
    }
    __device__ static __forceinline__ int slot(int row, int chunk) {
        return row * kSlots + (chunk ^ swizzle(row));
    }

    // Elements 16 step + 8 half .. + 8 of a row.
    __device__ static __forceinline__ Frag<T> row(const u32x4* lds, int row, int step, int half) {
        union {
            u32x4 u[sizeof(T) / 2];
            Frag<T> f;
        } x;
        if constexpr (sizeof(T) == 2) {
            x.u[0] = lds[slot(row, 2 * step + half)];
        } else {
            x.u[0] = lds[slot(row, 4 * step + 2 * half)];
            x.u[1] = lds[slot(row, 4 * step + 2 * half + 1)];
        }
        return x.f;
    }

    // The transposed operand: column 32 block + (lane & 31) of the rows first
    // + 8 (e / 4) + 4 (lane / 32) + e % 4, e = 0..7 -- the order in which an
    // accumulator's registers hold them.
    __device__ static __forceinline__ Frag<T> columns(const u32x4* lds, int first, int block,
                                                      int lane) {
        if constexpr (sizeof(T) == 2) {
            // Each group of 16 lanes reads 4 rows of 16 columns, lane s
            // addressing columns 4 (s % 4) .. + 4 of row s / 4, and receives
            // its own column of the 4 rows.
            const int s = lane & 15;
            const int r = first + 4 * (lane >> 5) + (s >> 2);
            const int col = 32 * block + 16 * ((lane >> 4) & 1) + 4 * (s & 3);
            union {
                s16x4 s[2];
                Frag<T> f;
            } x;
            typedef __attribute__((address_space(3))) s16x4* lds4;
            const char* at = reinterpret_cast<const char*>(lds);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int byte = slot(r + 8 * h, col >> 3) * 16 + (col & 7) * 2;
                x.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds4)(const_cast<char*>(at) + byte));
            }
            return x.f;
        } else {
            const float* at = reinterpret_cast<const float*>(lds);
            const int col = 32 * block + (lane & 31);
            Frag<T> f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = first + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                f[e] = at[slot(r, col >> 2) * 4 + (col & 3)];
            }
            return f;
        }
    }
};

// 16 bytes a lane from global memory to LDS at `lds` + 16 lane, past the
// registers.  Written as text because the compiler, given its builtin, waits for
// the copy before the next LDS read of any address, which is what copying
// beside the products is to avoid.  It has no register to write; landed() waits
// for it, and the statements around stay in order.
__device__ __forceinline__ void copy_to_lds(const void* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\t"
                 "s_nop 0\n\t"
                 "global_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(offset), "s"(base)
                 : "memory", "m0");
}
// The same of 4 bytes a lane.
__device__ __forceinline__ void copy_word_to_lds(const void* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\t"
                 "s_nop 0\n\t"
                 "global_load_lds_dword %1, %2"
                 :
                 : "s"(lds), "v"(offset), "s"(base)
                 : "memory", "m0");
}
// The LDS address of a __shared__ array (pass the array itself: of a pointer
// that came a longer way the compiler does not know that it is one).
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    typedef __attribute__((address_space(3))) const void* lds_ptr;
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)(p)));
}
// Every copy of this wave has landed, and every wave is here.
__device__ __forceinline__ void landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
}
// floats first .. first + 63 of [begin, end), the nearest for those outside, by
// one wave.
__device__ __forceinline__ void load_floats(const float* base, int first, int begin, int end,
                                            uint32_t lds, int lane) {
    const int from = min(max(first, begin), end - 1);
    const int at = min(max(first + lane, begin), end - 1) - from;
    copy_word_to_lds(base + from, static_cast<uint32_t>(at) * 4, lds);
}

// A tile's way from global memory to LDS beside the products of the tile before
// it: each lane names the 16 bytes that land in its slot, which is where the
// swizzle is made.  Rows outside [begin, end) repeat its nearest row, columns
// from `dim` on the row's first ones: they meet a P of 0, a q of 0 or an output
// that is not stored, and hold nothing that the interval does not hold itself.
template <typename T, int DB, int kRows, int kThreads>
struct Loader {
    typedef Tile<T, DB> G;
    static constexpr int kSlots = kRows * G::kSlots;
    static constexpr int kMine = kSlots / kThreads;
    static_assert(kSlots % kThreads == 0, "whole waves fill a tile");
    static constexpr int kStep = kThreads / G::kSlots;  // rows from one copy of a lane to the next
    int pitch;                // bytes of a row: 64 of them fit 31 bits (checked on the host)
    int first_row;            // bytes from the tile's first row to that of copy 0
    uint32_t offset[kMine];   // bytes from the tile's first row to copy n

    // row_stride * kRows elements fit 31 bits of bytes (checked on the host)
    __device__ __forceinline__ Loader(int64_t row_stride, int dim, int thread)
        : pitch(static_cast<int>(row_stride * sizeof(T))),
          first_row(thread / G::kSlots * pitch) {
#pragma unroll
        for (int n = 0; n < kMine; ++n) {
            const int row = thread / G::kSlots + n * kStep;
            const int chunk = ((thread + n * kThreads) % G::kSlots) ^ G::swizzle(row);
            const int col = chunk * G::kElems < dim ? chunk * G::kElems : 0;
            offset[n] = first_row + n * kStep * pitch + col * static_cast<int>(sizeof(T));
        }
    }
    // To the LDS address `lds`.  begin < end; first and lds are a wave's scalars.
    __device__ __forceinline__ void load(const T* base, int first, int begin, int end, uint32_t lds,
                                         int thread) const {
        const int from = min(max(first, begin), end - 1);
        const char* at = reinterpret_cast<const char*>(base) + static_cast<int64_t>(from) * pitch;
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds + (thread & ~63) * 16);
        if (first >= begin && first + kRows <= end) {
#pragma unroll
            for (int n = 0; n < kMine; ++n) copy_to_lds(at, offset[n], to + n * kThreads * 16);
        } else {
            // rows as bytes from row `from`, kept between it and the last one
            const EdgeRows edge = edge_rows(first, from, end, kRows, pitch);
#pragma unroll
            for (int n = 0; n < kMine; ++n) {
                const int row = first_row + n * kStep * pitch;
                copy_to_lds(at, offset[n] + (edge_row(edge, row) - row), to + n * kThreads * 16);
            }
        }
    }
};

// A row of global memory as B operands: lane's elements 16 s + 8 half .. + 8
// for every step s; zeros where `in` is false and from column dim on.
template <typename T, int DB>
__device__ __forceinline__ void load_operand(Frag<T> (&f)[2 * DB], const T* row, bool in, int dim,
                                             int half) {
#pragma unroll
    for (int s = 0; s < 2 * DB; ++s) {
        union {
            u32x4 u[sizeof(T) / 2];
            Frag<T> f;
        } x;
        const int col = 16 * s + 8 * half;
#pragma unroll
        for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h)
            x.u[h] = in && col < dim
                         ? *reinterpret_cast<const u32x4*>(row + col + h * (16 / sizeof(T)))
                         : u32x4{0, 0, 0, 0};
        f[s] = x.f;
    }
}

// Writes a column's accumulators (rows of the transposed product = elements of
// the row) as a row of global memory, times `by`; zeros where `any` is false,
// whatever was accumulated.  low: a row for what rounding took from each, or
// null.
template <typename T, int DB>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&acc)[DB], bool any, float by,
                                          int dim, int half, T* low = nullptr) {
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int col = 32 * b + 8 * g + 4 * half;
            if (col >= dim) continue;
            t4 v, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = any ? acc[b][4 * g + e] * by : 0.0f;
                v[e] = static_cast<T>(x);
                l[e] = static_cast<T>(x - static_cast<float>(v[e]));
            }
            *reinterpret_cast<t4*>(row + col) = v;
            if (low) *reinterpret_cast<t4*>(low + col) = l;
        }
}

// ---- reductions -------------------------------------------------------------------------------
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = min(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = max(x, __shfl_xor(x, o));
    return x;
}

// ---- scores -----------------------------------------------------------------------------------
// What a kernel needs of trw_score, everything in base 2 (exp2 of it is the
// softmax's numerator).
struct Score {
    float scale2;    // scale log2 e
    float softcap;   // 0: none
    float cap_in;    // 2 scale log2 e / softcap: tanh(x) = 1 - 2 / (1 + exp2(2 log2 e x))
    float cap_out;   // softcap log2 e
    float scale;
    const float* table;
    const int32_t* buckets;
    int num_buckets, reach;
    const float* slopes;
    const float *q_times, *k_times;

    __device__ __forceinline__ bool biased() const { return table || slopes; }
};

inline Score make_score(const trw_score& s) {
    Score r;
    r.scale = s.scale;
    r.scale2 = s.scale * kLog2e;
    r.softcap = s.softcap;
    r.cap_in = s.softcap > 0 ? 2.0f * kLog2e * s.scale / s.softcap : 0.0f;
    r.cap_out = s.softcap * kLog2e;
    r.table = s.table;
    r.buckets = s.buckets;
    r.num_buckets = s.num_buckets;
    r.reach = s.table ? s.reach : 0;
    r.slopes = s.slopes;
    r.q_times = s.q_times;
    r.k_times = s.k_times;
    return r;
}

// The biases of distances -reach..reach of one head, in base 2.  The type's
// lowest value and its like stay finite (a row of nothing else is a uniform
// row); -inf masks.
__device__ __forceinline__ float table_entry(const Score& s, int head, int at) {
    const int b = min(max(s.buckets[at], 0), s.num_buckets - 1);
    const float raw = s.table[static_cast<int64_t>(head) * s.num_buckets + b];
    const float t = raw * kLog2e;
    return raw != -INFINITY && t < kLowest ? kLowest : t;
}
__device__ __forceinline__ void fill_bias(float* lut, const Score& s, int head, int thread,
                                          int threads) {
    for (int i = thread; i < 2 * s.reach + 1; i += threads) lut[i] = table_entry(s, head, i);
}

// log2 e softcap tanh(scale x / softcap), and 1 - tanh^2.  float32 calls tanhf.
// The 16-bit types take tanh from exp2 and a reciprocal: its error of some 1e-7 is
// absolute, so one of 1e-7 softcap in the score, far below what their scores
// carry while the cap is not wide.  kWide: below 1/16 of the cap, the first terms
// of tanh's series, as exact as x (the next is 17/315 (1/16)^6 < 2^-28 of it).
// Kernels of their own: as a branch in the others it costs registers that they
// need (8192 rows, 16 heads of 128, backward: 1.72 -> 1.90 ms, 1.48 -> 1.67
// without a cap).
template <typename T, bool kWide>
__device__ __forceinline__ float capped(const Score& s, float x, float& slope) {
    if constexpr (sizeof(T) == 4) {
        const float t = tanhf(x * s.scale / s.softcap);
        slope = 1.0f - t * t;
        return s.cap_out * t;
    } else {
        const float in = x * s.cap_in;
        const float u = __builtin_amdgcn_rcpf(1.0f + exp2_fast(in));
        slope = 4.0f * u * (1.0f - u);
        const float far = fmaf(-2.0f * s.cap_out, u, s.cap_out);
        if (!kWide) return far;
        const float y = in * (0.5f * kLn2), y2 = y * y;
        const float series = fmaf(y2, fmaf(y2, 2.0f / 15.0f, -1.0f / 3.0f), 1.0f);
        return fabsf(y) < 0.0625f ? x * s.scale2 * series : far;
    }
}

inline bool wide_cap(int dtype, const trw_score& s) {
    return dtype != TRW_F32 && s.softcap > TRW_OPS_WIDE_CAP;
}
// f(kWide) for a type and a score.
template <typename T, typename F>
void by_cap(int dtype, const trw_score& s, F&& f) {
    if constexpr (sizeof(T) == 2) {
        if (wide_cap(dtype, s)) {
            f(std::true_type());
            return;
        }
    }
    f(std::false_type());
}

// Products to scores in base 2, without biases and mask.
template <typename T, bool kWide = false, int kBlocks>
__device__ __forceinline__ void cap_scores(const Score& sc, float (&s)[kBlocks][16]) {
    if (sc.softcap > 0) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float unused;
                s[b][r] = capped<T, kWide>(sc, s[b][r], unused);
            }
    } else {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] *= sc.scale2;
    }
}

// Adds table and slope terms where a lane's column is a query (position `diag`
// among the keys, time q_time; the wave's positions lie in [diag_lo, diag_hi])
// and register (b, r) is key j0 + 32 b + acc_row(r) + 4 half.
template <int kBlocks>
__device__ __forceinline__ void add_biases(const Score& sc, float (&s)[kBlocks][16],
                                           const float* lut, float slope, int diag, int diag_lo,
                                           int diag_hi, float q_time, const float* k_time, int j0,
                                           int half) {
    const int at = diag - (j0 + 4 * half);  // distance of register (b, r): at - 32 b - acc_row(r)
    if (sc.table) {
        const int far_lo = diag_lo - (j0 + 32 * kBlocks - 1), far_hi = diag_hi - j0;
        if (far_lo >= sc.reach || far_hi <= -sc.reach) {
            const float bias = lut[far_lo >= sc.reach ? 2 * sc.reach : 0];
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] += bias;
        } else {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = at - (32 * b + acc_row(r));
                    s[b][r] += lut[min(max(d, -sc.reach), sc.reach) + sc.reach];
                }
        }
    }
    if (sc.slopes) {
        if (sc.k_times) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[b][r] = fmaf(-slope, fabsf(q_time - k_time[32 * b + acc_row(r) + 4 * half]),
                                   s[b][r]);
        } else {
            const float from = static_cast<float>(at);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[b][r] = fmaf(-slope, fabsf(from - (32 * b + acc_row(r))), s[b][r]);
        }
    }
}

// Sums of a block's dS by distance, along its diagonals.  Float atomics of LDS
// take some 100 cycles an instruction (counted), so a wave writes 8 keys at a
// time to a square of its own, each row followed by zeros, and every lane reads
// one diagonal (rows kPitch + 1 apart, at constant offsets) and adds its sum to
// the wave's line of distances -reach .. reach.  Pairs past the reach share the
// line's ends: sums over lanes.
constexpr int kPitch = 40;  // 32 values and 8 zeros; two half waves' rows in other banks
constexpr int kSquare = 9 * kPitch;

// v: register r is key acc_row(r) + 4 half, the lane's column a query row; lo,
// hi: distances of the first and last row from the block's first key.
__device__ __forceinline__ void add_diagonals(const float (&v)[16], float* square, float* line,
                                              int reach, int lo, int hi, int lane, int half) {
    // lane's diagonal: its row less its key is at (lanes 0 .. 38)
    const int at = min(lane, 39) - 7;
    const bool mine = lane < 39;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            square[(1 + r + 4 * half) * kPitch + (lane & 31)] = v[4 * g + r];
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r) sum += square[(1 + r) * kPitch + r + at];
        const int d = lo - 8 * g + at;
        if (mine && abs(d) < reach) line[d + reach] += sum;
        if (hi - 8 * g >= reach || lo - 8 * g - 7 <= -reach) {
            // each once, also where reach 0 makes the two ends one
            float before = mine && d >= reach ? sum : 0.0f;
            float after = mine && d <= -reach && d < reach ? sum : 0.0f;
#pragma unroll
            for (int o = 32; o; o >>= 1) {
                before += __shfl_xor(before, o);
                after += __shfl_xor(after, o);
            }
            if (lane == 0) {
                line[2 * reach] += before;
                line[0] += after;
            }
        }
    }
}

// Whether a document of `size` rows (0: a row of no document) belongs to the
// kernels of tiles, when documents up to `limit` go a wave each.
__device__ __forceinline__ bool tiled(int size, int limit) { return size == 0 || size > limit; }

struct Rows {
    char* data;
    int64_t row, head;  // strides in elements
};
inline Rows make_rows(const trw_rows& r) {
    return Rows{static_cast<char*>(r.data), r.row_stride, r.head_stride};
}
template <typename T>
__device__ __forceinline__ T* row_of(const Rows& r, int64_t row, int head) {
    return reinterpret_cast<T*>(r.data) + row * r.row + head * r.head;
}

// Consecutive workgroup ids go to the eight XCDs in turn, each with an L2 of
// its own: XCD x takes the x-th eighth of the items, so that workgroups that
// read the same keys share one.
__device__ __forceinline__ int64_t xcd_item(int64_t id, int64_t items) {
    const int64_t per = (items + 7) / 8;
    return (id & 7) * per + (id >> 3);
}
inline int64_t xcd_grid(int64_t items) { return (items + 7) / 8 * 8; }

// f<T, DB>() for a dtype and a head size.
template <typename F>
void dispatch(int dtype, int dim, F&& f) {
    const int db = (dim + 31) / 32;
    auto by_dim = [&](auto t) {
        switch (db) {
            case 1: f(t, std::integral_constant<int, 1>()); break;
            case 2: f(t, std::integral_constant<int, 2>()); break;
            case 3: f(t, std::integral_constant<int, 3>()); break;
            default: f(t, std::integral_constant<int, 4>()); break;
        }
    };
    if (dtype == TRW_F32)
        by_dim(float{});
    else if (dtype == TRW_F16)
        by_dim(_Float16{});
    else
        by_dim(__bf16{});
}

inline size_t element_size(int dtype) { return dtype == TRW_F32 ? 4 : 2; }

// Implementations behind the C ABI (operators_capi.hip checks the arguments).
void walk_mask(const trw_walk_mask_params& p, hipStream_t stream);
uint64_t attention_workspace(const trw_attention_params& p, bool backward);
// Short walks (attention_walks.hip): how many blocks of 32 rows one may have
// (0: none go there), whether longer ones or rows of none may be in the batch,
// floats of one line of the table's gradient.
int walk_blocks(const trw_attention_params& p);
bool walk_rest(const trw_attention_params& p, int blocks);
int walk_line(const trw_attention_params& p, int blocks);
int64_t walk_grid(const trw_attention_params& p);
void walk_forward(const trw_attention_params& p, int blocks, hipStream_t stream);
void walk_backward(const trw_attention_params& p, int blocks, float* partial, hipStream_t stream);
// That every launch of a pass can be made, before the first one.
void require_grids(const trw_attention_params& p, bool backward);
void attention_forward(const trw_attention_params& p, hipStream_t stream);
void attention_backward(const trw_attention_params& p, hipStream_t stream);
// A table's gradient from sums by distance: join_lines adds up to `groups`
// lines per head from `partial` [heads, tiles, short_line] (distances
// -short_line / 2 ..) at line `first` of `lines` [heads, count, 2 reach + 1];
// join_table makes d_table [heads, num_buckets] of `dtype` of those.
void join_lines(const float* partial, int64_t tiles, int short_line, int heads, int groups,
                float* lines, int first, int count, int reach, hipStream_t stream);
void join_table(const float* lines, int count, int heads, const int32_t* buckets, int reach,
                int num_buckets, int dtype, void* d_table, hipStream_t stream);
constexpr int kJoinGroups = 64;
uint64_t attention_step_workspace(const trw_attention_step_params& p);
void attention_step(const trw_attention_step_params& p, hipStream_t stream);
uint64_t relative_bias_workspace(const trw_relative_bias_params& p);
void relative_bias(const trw_relative_bias_params& p, hipStream_t stream);
void relative_bias_backward(const trw_relative_bias_params& p, hipStream_t stream);

}  // namespace ops
}  // namespace trw
#endif  // TRW_OPERATORS_KERNELS_H
