// The 4-bit cache: which pages of a sequence attention reads.
//
// score(page) = max over the query heads of a kv head of  sum_c max(q_c M_c, q_c m_c) = q+ . M + q- . m  (M, m: the page's channel
// maxima and minima, q+ and q-: q where it is above and below 0): no key of the page has a larger product with q. It is computed
// in whole numbers, q in 8 bits and M, m in 7, on the tensor cores: exact in any order, so the choice repeats on every device and
// however the work is cut. M and m are read once, 4 D bytes a page and kv head.
#include "ommx_kv4.cuh"

namespace ommx {
namespace kv4 {

constexpr int SCORE_WARPS = 4, PICK_THREADS = 1024;

struct SelectParams {
    Cache c;
    Seqs s;
    const uint16_t *summary;
    const void *q;
    int64_t q_b, q_h;
    uint32_t *keys;                               // [B][H][max_pages]
    int32_t *selected;
    int32_t q16, group, col_blocks, n, first, last, page_shift;
    int32_t *status;
};

__device__ __forceinline__ int pages_of(const SelectParams &p, int b) {
    const int len = p.s.len[b];
    const int64_t most = (int64_t)p.s.max_pages << p.page_shift;
    if (len < 0 || len > most) { or_status(p.status, OMMX_ST_BAD_LENGTH); return len < 0 ? 0 : p.s.max_pages; }
    return (int)(((int64_t)len + p.c.page - 1) >> p.page_shift);
}
// unsigned order as of the numbers
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float load_q(const SelectParams &p, int64_t at) {
    if (p.q16) return __half2float(reinterpret_cast<const __half *>(p.q)[at]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p.q)[at]);
}
__device__ __forceinline__ void mma_u8s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// 64 + x c rounded, of four bf16 x: 192 + x c lies between 128 and 256, where bf16 has whole numbers only
__device__ __forceinline__ uint32_t bytes_of(uint32_t x01, uint32_t x23, uint32_t cc) {
    constexpr uint32_t MAGIC = 0x43404340u;       // 192, twice
    return __byte_perm(fma_bf16x2(x01, cc, MAGIC), fma_bf16x2(x23, cc, MAGIC), 0x6420) & 0x7F7F7F7Fu;
}

// Grid: (blocks of a sequence's pages, kv heads, sequences). A warp scores 16 pages at a time: lane (g, t) holds channels
// 32 j + 8 t + 0..7 of pages g and g + 8 as the rows of m16n8k32 products, up to eight query heads are the columns.
template <int G> __global__ void __launch_bounds__(32 * SCORE_WARPS) kv4_score_kernel(const __grid_constant__ SelectParams p) {
    constexpr int D = 32 * G;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y, b = blockIdx.z;
    wait_earlier();
    let_next_in();
    const int pages = pages_of(p, b);
    if (pages <= p.n) return;                                               // all of them: nothing to compare
    const int tile0 = blockIdx.x * SCORE_WARPS + warp, tiles = (pages + 15) >> 4;
    if (tile0 >= tiles) return;
    // the kv head's queries in 8 bits
    float top = 0.0f;
    for (int i = lane; i < p.group * D; i += 32) top = fmaxf(top, fabsf(load_q(p, b * p.q_b + (int64_t)(h * p.group + i / D) * p.q_h + i % D)));
#pragma unroll
    for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    const int e = (int)(__float_as_uint(top) >> 23) - 127;                  // q of subnormal size: all 0 either way
    const float up = top > 0.0f ? __uint_as_float((uint32_t)min(max(6 - e + 127, 1), 254) << 23) : 0.0f;

    for (int tile = tile0; tile < tiles; tile += gridDim.x * SCORE_WARPS) {
        uint32_t a[2][2][G][2];                                             // [page g, g + 8][M, m][j][half]
        float weight[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int page = tile * 16 + 8 * r + g;
            uint4 x[2][G];
            int64_t id = -1;
            if (page < pages) {
                id = page_id(p.s, b, page);
                if (id < 0 || id >= p.c.num_pages) { or_status(p.status, OMMX_ST_BAD_PAGE); id = -1; }
            }
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < G; ++j)
                    x[m][j] = id < 0 ? make_uint4(0, 0, 0, 0)
                                     : *reinterpret_cast<const uint4 *>(p.summary + ((id * p.c.H + h) * 2 + m) * D + 32 * j + 8 * t);
            uint32_t most = 0;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    most = max_bf16x2(max_bf16x2(most, x[m][j].x & 0x7FFF7FFFu), x[m][j].y & 0x7FFF7FFFu);
                    most = max_bf16x2(max_bf16x2(most, x[m][j].z & 0x7FFF7FFFu), x[m][j].w & 0x7FFF7FFFu);
                }
            uint32_t one = max(most & 0xFFFFu, most >> 16);
            one = max(one, __shfl_xor_sync(~0u, one, 1));
            one = max(one, __shfl_xor_sync(~0u, one, 2));
            const int f = max((int)(one >> 7) - 127, -100);
            const uint32_t c = ((uint32_t)(5 - f - 1 + 127) << 7) | 0x7Cu;  // (63 / 64) 2^(5 - f) = (63 / 32) 2^(4 - f) in bf16
            weight[r] = __uint_as_float((uint32_t)(f - 26 + 127) << 23);
            if (id < 0) weight[r] = 0.0f;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    a[r][m][j][0] = bytes_of(x[m][j].x, x[m][j].y, c | c << 16);
                    a[r][m][j][1] = bytes_of(x[m][j].z, x[m][j].w, c | c << 16);
                }
        }
        int best[2] = {INT32_MIN, INT32_MIN};
        for (int cb = 0; cb < p.col_blocks; ++cb) {
            const int n = min(8, p.group - 8 * cb);
            int sum = 0, acc[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < G; ++j) {
                uint32_t plus[2] = {0, 0}, minus[2] = {0, 0};
                if (g < n) {
                    const int64_t at = b * p.q_b + (int64_t)(h * p.group + 8 * cb + g) * p.q_h + 32 * j + 8 * t;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int v = max(-127, min(127, __float2int_rn(load_q(p, at + i) * up)));
                        sum += v;
                        plus[i >> 2] |= (uint32_t)max(v, 0) << (8 * (i & 3));
                        minus[i >> 2] |= ((uint32_t)min(v, 0) & 255u) << (8 * (i & 3));
                    }
                }
                mma_u8s8(acc, a[0][0][j][0], a[1][0][j][0], a[0][0][j][1], a[1][0][j][1], plus[0], plus[1]);
                mma_u8s8(acc, a[0][1][j][0], a[1][1][j][0], a[0][1][j][1], a[1][1][j][1], minus[0], minus[1]);
            }
            sum += __shfl_xor_sync(~0u, sum, 1);
            sum += __shfl_xor_sync(~0u, sum, 2);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int off = 64 * __shfl_sync(~0u, sum, 8 * t + 4 * i);  // the bytes are 64 too large
                if (2 * t + i < n) { best[0] = max(best[0], acc[i] - off); best[1] = max(best[1], acc[2 + i] - off); }
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            best[r] = max(best[r], __shfl_xor_sync(~0u, best[r], 1));
            best[r] = max(best[r], __shfl_xor_sync(~0u, best[r], 2));
            const int page = tile * 16 + 8 * r + g;
            if (t == 0 && page < pages)
                p.keys[((int64_t)b * p.c.H + h) * p.s.max_pages + page] =
                    page < p.first || page >= pages - p.last ? ~0u : ordered(__int2float_rn(best[r]) * weight[r]);
        }
    }
}

__device__ __forceinline__ int2 block_exclusive_scan(int2 v, int2 *shared, int2 *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 s = make_int2(warp_inclusive_scan(v.x, lane), warp_inclusive_scan(v.y, lane));
    if (lane == 31) shared[warp] = s;
    __syncthreads();
    int2 before = make_int2(0, 0), all = before;
    for (int w = 0; w < PICK_THREADS / 32; ++w) {
        if (w == warp) before = all;
        all.x += shared[w].x;
        all.y += shared[w].y;
    }
    __syncthreads();
    *total = all;
    return make_int2(before.x + s.x - v.x, before.y + s.y - v.y);
}

// The n largest keys of a row, ties to the lowest page: a digit of eight bits at a time from the top, then one ordered pass.
__global__ void __launch_bounds__(PICK_THREADS) kv4_pick_kernel(const __grid_constant__ SelectParams p) {
    __shared__ int histogram[256];
    __shared__ int2 scan[PICK_THREADS / 32];
    __shared__ uint32_t chosen;
    __shared__ int left;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    wait_earlier();
    let_next_in();
    const int pages = pages_of(p, b);
    int32_t *out = p.selected + ((int64_t)b * p.c.H + h) * p.n;
    if (pages <= p.n) {
        for (int i = tid; i < p.n; i += PICK_THREADS) out[i] = i < pages ? i : -1;
        return;
    }
    const uint32_t *keys = p.keys + ((int64_t)b * p.c.H + h) * p.s.max_pages;
    uint32_t prefix = 0, mask = 0;
    int want = p.n;                               // how many of the keys that begin with `prefix` are taken
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) histogram[tid] = 0;
        __syncthreads();
        for (int i = tid; i < pages; i += PICK_THREADS) {
            const uint32_t k = keys[i];
            if ((k & mask) == prefix) atomicAdd(&histogram[k >> shift & 255u], 1);
        }
        __syncthreads();
        if (tid < 32) {                           // lane l: digits 255 - 8 l .. 248 - 8 l
            int mine = 0;
            for (int i = 0; i < 8; ++i) mine += histogram[255 - 8 * tid - i];
            const int upto = warp_inclusive_scan(mine, tid);
            if (upto >= want && upto - mine < want) {
                int above = upto - mine, d = 255 - 8 * tid;
                while (above + histogram[d] < want) above += histogram[d--];
                chosen = prefix | (uint32_t)d << shift;
                left = want - above;
            }
        }
        __syncthreads();
        prefix = chosen;
        want = left;
        mask |= 255u << shift;
        __syncthreads();
    }
    // keys above `prefix`, and the first `want` equal to it, in order
    const int each = (pages + PICK_THREADS - 1) / PICK_THREADS, from = min(pages, tid * each), to = min(pages, from + each);
    int2 mine = make_int2(0, 0), total;
    for (int i = from; i < to; ++i) { mine.x += keys[i] > prefix; mine.y += keys[i] == prefix; }
    int2 at = block_exclusive_scan(mine, scan, &total);
    for (int i = from; i < to; ++i) {
        const bool more = keys[i] > prefix, same = keys[i] == prefix;
        if (more || (same && at.y < want)) out[at.x + min(at.y, want)] = i;
        at.x += more;
        at.y += same;
    }
}

static int64_t select_workspace(int64_t B, int64_t H, int64_t pages) { return (B * H * pages * 4 + 15) / 16 * 16; }

static int select(const ommx_kv4_select_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv4_select: null args");
    SelectParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv4_select", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv4_select", a->seqs, &p.s)) return rc;
    if (a->q_dtype != OMMX_DT_BF16 && a->q_dtype != OMMX_DT_F16) return fail(OMMX_E_UNSUPPORTED, "kv4_select: q must be bfloat16 or float16");
    if (a->n_q_heads < p.c.H || a->n_q_heads % p.c.H)
        return fail(OMMX_E_UNSUPPORTED, "kv4_select: %d query heads are not a multiple of %d kv heads", a->n_q_heads, p.c.H);
    if (a->first_pages < 0 || a->last_pages < 0 || (int64_t)a->first_pages + a->last_pages > a->num_selected)
        return fail(OMMX_E_ARG, "kv4_select: first_pages %d and last_pages %d must fit into %d selected ones", a->first_pages, a->last_pages, a->num_selected);
    if (p.s.B > 65535) return fail(OMMX_E_UNSUPPORTED, "kv4_select: a batch of %d", p.s.B);
    if (p.s.B == 0 || a->num_selected == 0) return 0;
    if (!a->q || !a->selected) return fail(OMMX_E_ARG, "kv4_select: q and selected must not be null");
    if (!a->cache.summary && a->cache.num_pages) return fail(OMMX_E_ARG, "kv4_select: the cache has no page summary");
    const int64_t need = select_workspace(p.s.B, p.c.H, p.s.max_pages);
    if (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_bytes < need))
        return fail(OMMX_E_ARG, "kv4_select: workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
    p.summary = (const uint16_t *)a->cache.summary;
    p.q = a->q; p.q16 = a->q_dtype == OMMX_DT_F16; p.q_b = a->q_stride_b; p.q_h = a->q_stride_h;
    p.keys = (uint32_t *)a->workspace;
    p.selected = a->selected; p.n = a->num_selected; p.first = a->first_pages; p.last = a->last_pages;
    p.group = a->n_q_heads / p.c.H; p.col_blocks = (p.group + 7) / 8;
    p.page_shift = shift_of(p.c.page);
    p.status = a->status;
    if (p.s.max_pages > p.n) {
        const int64_t rows = (int64_t)p.s.B * p.c.H, most = (p.s.max_pages + 16LL * SCORE_WARPS - 1) / (16 * SCORE_WARPS);
        const int64_t fill = (8LL * sm_count() + rows - 1) / rows;          // eight blocks to an SM
        const dim3 grid((unsigned)(most < fill ? most : fill), p.c.H, p.s.B);
        const int rc = a->cache.head_dim == 64 ? launch_dependent(kv4_score_kernel<2>, grid, 32 * SCORE_WARPS, 0, st, p)
                                               : launch_dependent(kv4_score_kernel<4>, grid, 32 * SCORE_WARPS, 0, st, p);
        if (rc) return rc;
    }
    return launch_dependent(kv4_pick_kernel, dim3(p.c.H, p.s.B), PICK_THREADS, 0, st, p);
}

}  // namespace kv4
}  // namespace ommx

extern "C" int64_t ommx_b200_kv4_select_workspace_bytes(int32_t batch, int32_t n_kv_heads, int32_t pages_per_seq) {
    return batch < 0 || n_kv_heads < 0 || pages_per_seq < 0 ? 0 : ommx::kv4::select_workspace(batch, n_kv_heads, pages_per_seq);
}
extern "C" int ommx_b200_kv4_select(const ommx_kv4_select_args *args, void *stream) { return ommx::kv4::select(args, (cudaStream_t)stream); }
