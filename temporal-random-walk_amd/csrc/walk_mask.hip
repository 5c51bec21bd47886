// walk_mask.hip -- which keys each query row of a batch of walks sees, and
// which query rows see each key.
//
// Every mask here (a walk's own keys, causal, prefix, padding) leaves a query
// an interval of key rows, and, the documents being in order in both, leaves a
// key an interval of query rows.  The attention kernels work from these
// intervals alone (a wave with a walk of its own, from the walk's spans).  One
// thread per row of either side and per document; a packed row finds its
// document by a binary search of the offsets.
//
// 32 bytes written per row: 3 us for a small batch (one launch), 14 us for 1.6
// million rows of padded walks (3.6 TB/s), once for all layers of a batch.
#include "operators.h"

namespace trw {
namespace ops {
namespace {

constexpr int kB = 256;

struct Span {
    int64_t begin, len;
};

struct MaskArgs {
    trw_walk_mask_params p;

    __device__ __forceinline__ Span span(int64_t w, const int64_t* lens, const int64_t* offsets,
                                         int64_t length, int64_t rows) const {
        if (offsets) {
            const int64_t a = min(max(offsets[w], int64_t{0}), rows);
            const int64_t b = min(max(offsets[w + 1], a), rows);
            return Span{a, b - a};
        }
        return Span{w * length, lens ? min(max(lens[w], int64_t{0}), length) : length};
    }
    __device__ __forceinline__ Span q_span(int64_t w) const {
        return span(w, p.q_lens, p.q_offsets, p.q_length, p.q_rows);
    }
    // k_offsets / k_lens default to the queries' own (set on the host)
    __device__ __forceinline__ Span k_span(int64_t w) const {
        return span(w, p.k_lens, p.k_offsets, p.k_length, p.k_rows);
    }
    // The document of a row: the last one that begins at or before it.
    __device__ __forceinline__ int64_t doc_of(int64_t row, const int64_t* offsets,
                                              int64_t length) const {
        if (!offsets) return row / length;
        int64_t a = 0, b = p.docs;  // offsets[a] <= row < offsets[b], where they hold
        while (b - a > 1) {
            const int64_t m = (a + b) / 2;
            if (offsets[m] <= row) a = m;
            else b = m;
        }
        return a;
    }
    __device__ __forceinline__ int64_t prefix_of(int64_t w, int64_t len) const {
        return p.kind == TRW_MASK_PREFIX ? min(max(p.prefix[w], int64_t{0}), len) : 0;
    }
};

__global__ __launch_bounds__(kB) void walk_mask_kernel(MaskArgs a, unsigned q_blocks,
                                                            unsigned k_blocks) {
    const trw_walk_mask_params& p = a.p;
    if (blockIdx.x < q_blocks) {
        const int64_t i = blockIdx.x * static_cast<int64_t>(kB) + threadIdx.x;
        if (i >= p.q_rows) return;
        int4 info = {0, 0, 0, 0};
        if (p.docs > 0) {
            const int64_t w = a.doc_of(i, p.q_offsets, p.q_length);
            const Span q = a.q_span(w), k = a.k_span(w);
            const int64_t local = i - q.begin;
            if (local >= 0 && local < q.len) {
                const int64_t pos = k.len - q.len + local;
                int64_t seen = k.len;
                if (p.kind != TRW_MASK_FULL)
                    seen = max(min(max(pos + 1, int64_t{0}), k.len), a.prefix_of(w, k.len));
                info.x = static_cast<int>(k.begin);
                info.y = static_cast<int>(k.begin + seen);
                info.z = static_cast<int>(k.begin + pos);
            }
            if (local >= 0 && (local < q.len || !p.q_offsets))
                info.w = static_cast<int>(max(max(q.len, k.len), int64_t{1}));
        }
        reinterpret_cast<int4*>(p.q_rows_info)[i] = info;
    } else if (blockIdx.x < q_blocks + k_blocks) {
        const int64_t j = (blockIdx.x - q_blocks) * static_cast<int64_t>(kB) + threadIdx.x;
        if (j >= p.k_rows) return;
        int4 info = {0, 0, 0, 0};
        if (p.docs > 0) {
            const int64_t w = a.doc_of(j, p.k_offsets, p.k_length);
            const Span q = a.q_span(w), k = a.k_span(w);
            const int64_t local = j - k.begin;
            if (local >= 0 && local < k.len) {
                int64_t first = 0;
                if (p.kind != TRW_MASK_FULL && local >= a.prefix_of(w, k.len))
                    first = min(max(local - (k.len - q.len), int64_t{0}), q.len);
                info.x = static_cast<int>(q.begin + first);
                info.y = static_cast<int>(q.begin + q.len);
            }
            if (local >= 0 && (local < k.len || !p.k_offsets))
                info.w = static_cast<int>(max(max(q.len, k.len), int64_t{1}));
        }
        reinterpret_cast<int4*>(p.k_rows_info)[j] = info;
    } else {
        const int64_t w = (blockIdx.x - q_blocks - k_blocks) * static_cast<int64_t>(kB) + threadIdx.x;
        if (w >= p.docs) return;
        const Span q = a.q_span(w), k = a.k_span(w);
        int4* out = reinterpret_cast<int4*>(p.docs_info) + 2 * w;
        // rows of padding are the document's as well
        out[0] = int4{static_cast<int>(q.begin), static_cast<int>(q.len),
                      static_cast<int>(p.q_offsets ? q.len : p.q_length),
                      static_cast<int>(k.begin)};
        out[1] = int4{static_cast<int>(k.len), static_cast<int>(p.k_offsets ? k.len : p.k_length),
                      static_cast<int>(a.prefix_of(w, k.len)), p.kind};
    }
}

}  // namespace

void walk_mask(const trw_walk_mask_params& p, hipStream_t stream) {
    MaskArgs a{p};
    if (!p.k_offsets && !p.k_lens) {
        a.p.k_offsets = p.q_offsets;
        a.p.k_lens = p.q_lens;
        if (!p.q_offsets) a.p.k_length = p.q_length;
    }
    const unsigned qb = static_cast<unsigned>((p.q_rows + kB - 1) / kB);
    const unsigned kb = static_cast<unsigned>((p.k_rows + kB - 1) / kB);
    const unsigned db = static_cast<unsigned>((p.docs + kB - 1) / kB);
    if (qb + kb + db == 0) return;
    hipLaunchKernelGGL(walk_mask_kernel, dim3(qb + kb + db), dim3(kB), 0, stream, a, qb, kb);
    check_launch("walk_mask");
}

}  // namespace ops
}  // namespace trw
