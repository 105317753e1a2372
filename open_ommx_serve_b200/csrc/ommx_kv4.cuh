// The 4-bit cache: its record format, and what its kernels share.
//
// One record of 20 D bytes per (page, kv head, 16 tokens); G = D / 32 groups of channels, g = lane / 4, t = lane % 4:
//   K codes   8 D bytes: word (tau * 4 + t) * G + j      = channels 32 j + 8 t + 0..7 of token tau, one nibble each
//   V codes   8 D bytes: word (32 h + 4 g + t) * G + j   = channels 32 j + 4 g + 0..3 of tokens 8 h + 2 t | 8 h + 2 t + 1 << 16
//   K params  2 D bytes: word tau * G + j                = bf16 scale << 16 | bf16 zero
//   V params  2 D bytes: the same
// value = zero + scale * code.  This is the order in which the lanes of a warp hold m16n8k16 A fragments, so attention reads codes
// in 16-byte pieces and masks them in place: K as [token][channel] with the nibbles i and i + 4 of a word in one register, V as
// [channel][token] with the two tokens of a word in one register.  A token owns whole bytes everywhere: a row is stored without
// reading what lies beside it.
#pragma once

#include "ommx_common.cuh"

namespace ommx {
namespace kv4 {

constexpr float LARGEST = 0x1p126f;               // the quantizer takes values to be at most this
constexpr float SMALLEST = 0x1p-96f;              // a smaller scale counts as none
constexpr float SHRINK = 1.0f - 0x1p-20f;         // of quotients before they are rounded: ties go down whatever their last bit

template <int G> struct Rec {
    static constexpr int D = 32 * G, V = 8 * D, KP = 16 * D, VP = 18 * D, BYTES = 20 * D;
};
template <int G> struct Words;                    // a lane's piece of codes, a token's parameters: G words
template <> struct Words<2> { using T = uint2; };
template <> struct Words<4> { using T = uint4; };

// Sequence lengths, page table and record array as every kernel here is given them.
struct Cache {
    uint8_t *records;
    int32_t num_pages, H, page, parts;            // parts: records of 16 tokens per page and head
};
struct Seqs {
    const int32_t *len;                           // tokens, the appended ones among them
    const void *table;
    int64_t table_stride;
    int32_t table64, max_pages, B;
};
__device__ __forceinline__ int64_t page_id(const Seqs &s, int b, int p) {
    const int64_t at = (int64_t)b * s.table_stride + p;
    return s.table64 ? reinterpret_cast<const int64_t *>(s.table)[at] : reinterpret_cast<const int32_t *>(s.table)[at];
}

// Every kernel is launched as a programmatic dependent of the one before it in the stream and touches no global memory before this.
__device__ __forceinline__ void wait_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_in() { asm volatile("griddepcontrol.launch_dependents;"); }

template <typename K, typename... A>
int launch_dependent(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream, int cluster, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    OMMX_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
    count_launch();
    return 0;
}

__device__ __forceinline__ int warp_inclusive_scan(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// eight channels of a query; P: parameters with q, whether it is fp16 (else bf16) and whether all rows start on 16-byte boundaries
template <typename P> __device__ __forceinline__ void load_q8(const P &p, int64_t at, float *x) {
    alignas(16) uint16_t v[8];
    if (p.q_wide) {
        *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(p.q) + at);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = reinterpret_cast<const uint16_t *>(p.q)[at + i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p.q16 ? __half2float(__ushort_as_half(v[i])) : __uint_as_float((uint32_t)v[i] << 16);
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Rows of a call that belong to a sequence: [first, end) of the row tensors; the sequence's last rows, in order.
struct Rows {
    const int32_t *row_start;                     // [B + 1], or null: row b is sequence b's
    int32_t T;
    // end < first: no range of these rows. (Bounds compared without the clamps are as right and 1 us slower: three chunks of 333..1025 rows
    // 13.1 us, 12.0 so.)
    __device__ __forceinline__ void of(int b, int *first, int *end) const {
        if (!row_start) { *first = min(b, T); *end = min(b + 1, T); return; }
        *first = min(max(row_start[b], 0), T);
        *end = min(max(row_start[b + 1], *first), T);
        if (*first != row_start[b] || *end != row_start[b + 1]) *end = *first - 1;
    }
};

// The `index`-th run of rows that lie in one block of `size` tokens (a power of two) of one sequence, counted over the sequences in
// order: sequence, first position, one past the last, and the row of the first.  A whole warp calls it; false when there are fewer.
// A sequence whose range is none of the call's rows, or whose rows are more than its length, has none, and is reported.
struct Run { int b, p0, p1, row; };
__device__ __forceinline__ bool find_run(const Seqs &s, const Rows &rows, int shift, int index, int lane, Run *run, int32_t *status) {
    for (int b0 = 0; b0 < s.B; b0 += 32) {
        int n = 0, first = 0, end = 0, len = 0;
        if (b0 + lane < s.B) {
            rows.of(b0 + lane, &first, &end);
            len = s.len[b0 + lane];
            if (end != first) {
                if (end < first || len < end - first) or_status(status, OMMX_ST_BAD_LENGTH);
                else n = ((len - 1) >> shift) - ((len - (end - first)) >> shift) + 1;
            }
        }
        const int sum = warp_inclusive_scan(n, lane);
        const int all = __shfl_sync(~0u, sum, 31);
        if (index < all) {
            const int from = __ffs(__ballot_sync(~0u, sum > index)) - 1;
            const int before = __shfl_sync(~0u, sum - n, from);
            first = __shfl_sync(~0u, first, from);
            end = __shfl_sync(~0u, end, from);
            len = __shfl_sync(~0u, len, from);
            const int start = len - (end - first);
            const int block = (start >> shift) + index - before;
            run->b = b0 + from;
            run->p0 = max(start, block << shift);
            run->p1 = (int)min((int64_t)len, ((int64_t)block + 1) << shift);
            run->row = first + run->p0 - start;
            return true;
        }
        index -= all;
    }
    return false;
}

// ---- host: arguments every entry point checks ----
inline int shift_of(int page) { int s = 0; while ((1 << s) < page) ++s; return s; }
inline int read_cache(const char *who, const ommx_kv4_cache &c, Cache *to) {
    if (c.head_dim != 64 && c.head_dim != 128) return fail(OMMX_E_UNSUPPORTED, "%s: head_dim %d (this build serves 64 and 128)", who, c.head_dim);
    if (c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1)))
        return fail(OMMX_E_UNSUPPORTED, "%s: page_size %d (this build serves 16, 32, 64, 128 and 256)", who, c.page_size);
    if (c.num_pages < 0 || c.n_kv_heads <= 0 || c.n_kv_heads > 4096) return fail(OMMX_E_ARG, "%s: %d pages of %d kv heads", who, c.num_pages, c.n_kv_heads);
    if ((c.num_pages && !c.records) || reinterpret_cast<uintptr_t>(c.records) % 16) return fail(OMMX_E_ARG, "%s: records must be given and 16-byte aligned", who);
    if (reinterpret_cast<uintptr_t>(c.summary) % 16) return fail(OMMX_E_ARG, "%s: summary must be 16-byte aligned", who);
    *to = {(uint8_t *)c.records, c.num_pages, c.n_kv_heads, c.page_size, c.page_size / 16};
    return 0;
}
inline int read_seqs(const char *who, const ommx_kv4_seqs &s, const Cache &c, Seqs *to) {
    if (s.batch < 0 || s.pages_per_seq < 0) return fail(OMMX_E_ARG, "%s: batch and pages_per_seq must not be negative", who);
    if (s.batch && (!s.b_seq_len || (!s.page_table && s.pages_per_seq))) return fail(OMMX_E_ARG, "%s: b_seq_len and page_table must not be null", who);
    // places are counted in 32 bits, a page and more to spare
    const int32_t most = 0x7FFFFC00 / c.page;
    *to = {s.b_seq_len, s.page_table, s.page_table_stride, s.table_is_int64, s.pages_per_seq < most ? s.pages_per_seq : most, s.batch};
    return 0;
}

// at most this many runs
inline int64_t most_runs(int64_t T, int64_t B, int64_t size, bool one_row_each) {
    const int64_t n = T / size + 2 * B;
    return one_row_each ? (T < B ? T : B) : (n < T ? n : T);
}

}  // namespace kv4
}  // namespace ommx
