// The 4-bit cache: which pages of a sequence attention reads.
//
// score(page) = max over the query heads of a kv head of  sum_c max(q_c M_c, q_c m_c) = q+ . M + q- . m  (M, m: the page's channel
// maxima and minima of the keys that were stored, q+ and q-: q where it is above and below 0). With those numbers as they are no key has a
// larger product with q; the score is an estimate of that bound: q is rounded to 8 bits and M, m to 7, and the cached keys' codes may lie
// half a step outside. It is computed in whole numbers on the tensor cores: exact in any order, so the choice repeats on every device and
// however the work is cut. M and m are read once, 4 D bytes a page and kv head: 8192 pages x 8 heads (33.6 MB) 7.4 us where the L2 holds
// them, 14.5 from HBM, as a model's layers in turn find them; and 7.6 (12) to pick 256 of them, a block to a kv head, which is latency:
// lengths, keys, five rounds of the block.
#include "ommx_kv4.cuh"

namespace ommx {
namespace kv4 {

constexpr int SCORE_WARPS = 8, PICK_THREADS = 1024;
constexpr int MOST_HEADS = 160;                   // query heads to a kv head: their fragments lie in 40 KB of shared memory

struct SelectParams {
    Cache c;
    Seqs s;
    const uint16_t *summary;
    const void *q;
    int64_t q_b, q_h;
    uint32_t *keys;                               // [B][H][max_pages]
    int32_t *selected;
    int32_t q16, q_wide, group, col_blocks, n, first, last, page_shift;
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
__device__ __forceinline__ void mma_u8s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// A kv head's queries in 8 bits, as B fragments of lane (g, t) = head g, channels 32 j + 8 t + 0..7: what is above 0, and what is below.
// The whole block calls it; sums: of a head's channels.
template <int G> __device__ __forceinline__ void quantize_query(const SelectParams &p, int b, int h, uint4 *frag, int *sums, uint32_t *top) {
    constexpr int D = 32 * G, CHUNKS = D / 8, THREADS = 32 * SCORE_WARPS;
    const int chunks = p.group * CHUNKS;
    for (int i = threadIdx.x; i < p.col_blocks * 8; i += THREADS) sums[i] = 0;
    if (threadIdx.x == 0) *top = 0;
    for (int i = chunks + threadIdx.x; i < p.col_blocks * 8 * CHUNKS; i += THREADS)         // heads that are not there
        frag[((i / CHUNKS / 8) * G + i % CHUNKS / 4) * 32 + (i / CHUNKS % 8) * 4 + i % 4] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int64_t at = b * p.q_b + (int64_t)h * p.group * p.q_h;
    float x[8];
    uint32_t most = 0;
    for (int i = threadIdx.x; i < chunks; i += THREADS) {
        load_q8(p, at + (int64_t)(i / CHUNKS) * p.q_h + i % CHUNKS * 8, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) most = max(most, x[k] == x[k] ? __float_as_uint(fabsf(x[k])) : 0u);
    }
    most = __reduce_max_sync(~0u, most);
    if ((threadIdx.x & 31) == 0) atomicMax(top, most);
    __syncthreads();
    const float pre = *top < 0x0D800000u ? 0x1p64f : 1.0f;                  // below 2^-100: 2^(6 - e) would pass 32 bits, or e is not in a subnormal's exponent
    const float largest = __uint_as_float(*top) * pre;
    const int e = (int)(__float_as_uint(largest) >> 23) - 127;
    const float up = largest > 0.0f ? __uint_as_float((uint32_t)min(max(6 - e + 127, 1), 254) << 23) : 0.0f;
    for (int i = threadIdx.x; i < chunks; i += THREADS) {
        if (chunks > THREADS) load_q8(p, at + (int64_t)(i / CHUNKS) * p.q_h + i % CHUNKS * 8, x);
        uint32_t plus[2] = {0, 0}, minus[2] = {0, 0};
        int sum = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int v = max(-127, min(127, __float2int_rn(x[k] * pre * up)));
            sum += v;
            plus[k >> 2] |= (uint32_t)max(v, 0) << (8 * (k & 3));
            minus[k >> 2] |= ((uint32_t)min(v, 0) & 255u) << (8 * (k & 3));
        }
        const int head = i / CHUNKS, c = i % CHUNKS;
        frag[((head / 8) * G + c / 4) * 32 + (head % 8) * 4 + c % 4] = make_uint4(plus[0], plus[1], minus[0], minus[1]);
        atomicAdd(&sums[head], sum);
    }
    __syncthreads();
}

// Grid: (blocks of a sequence's pages, kv heads, sequences). A warp scores 16 pages at a time: lane (g, t) holds channels
// 32 j + 8 t + 0..7 of pages g and g + 8 as the rows of m16n8k32 products, up to eight query heads are the columns. The first pages
// are on their way while the block works out the queries.
template <int G> __global__ void __launch_bounds__(32 * SCORE_WARPS) kv4_score_kernel(const __grid_constant__ SelectParams p) {
    constexpr int D = 32 * G;
    extern __shared__ uint4 frag[];               // [col_blocks][G][32]
    int *sums = reinterpret_cast<int *>(frag + p.col_blocks * G * 32);      // [col_blocks][8], and the largest |q|
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y, b = blockIdx.z;
    wait_earlier();
    let_next_in();
    const int pages = pages_of(p, b), tiles = (pages + 15) >> 4;
    if (pages <= p.n || blockIdx.x * SCORE_WARPS >= tiles) return;          // all of them: nothing to compare; or none for this block
    uint4 x[2][2][G];                             // [page g, g + 8][M, m][j]
    uint32_t there = 0;
    auto load = [&](int tile) {
        there = 0;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int page = tile * 16 + 8 * r + g;
            int64_t id = -1;
            if (page < pages) {
                id = page_id(p.s, b, page);
                if (id < 0 || id >= p.c.num_pages) { or_status(p.status, OMMX_ST_BAD_PAGE); id = -1; }
            }
            there |= (uint32_t)(id >= 0) << r;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < G; ++j)
                    x[r][m][j] = id < 0 ? make_uint4(0, 0, 0, 0)
                                        : *reinterpret_cast<const uint4 *>(p.summary + ((id * p.c.H + h) * 2 + m) * D + 32 * j + 8 * t);
        }
    };
    int tile = blockIdx.x * SCORE_WARPS + warp;
    if (tile < tiles) load(tile);
    quantize_query<G>(p, b, h, frag, sums, reinterpret_cast<uint32_t *>(sums + p.col_blocks * 8));
    for (; tile < tiles; tile += gridDim.x * SCORE_WARPS) {
        uint32_t a[2][2][G][2];                                             // [page g, g + 8][M, m][j][half]
        float weight[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            uint32_t most = 0;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    const uint4 v = x[r][m][j];
                    most = max_bf16x2(max_bf16x2(most, v.x & 0x7FFF7FFFu), v.y & 0x7FFF7FFFu);
                    most = max_bf16x2(max_bf16x2(most, v.z & 0x7FFF7FFFu), v.w & 0x7FFF7FFFu);
                }
            uint32_t one = max(most & 0xFFFFu, most >> 16);
            one = max(one, __shfl_xor_sync(~0u, one, 1));
            one = max(one, __shfl_xor_sync(~0u, one, 2));
            const int f = max((int)(one >> 7) - 127, -100);
            const uint32_t c = ((uint32_t)(5 - f - 1 + 127) << 7) | 0x7Cu;  // (63 / 64) 2^(5 - f) = (63 / 32) 2^(4 - f) in bf16
            weight[r] = there >> r & 1 ? __uint_as_float((uint32_t)(f - 26 + 127) << 23) : 0.0f;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    a[r][m][j][0] = bytes_of(x[r][m][j].x, x[r][m][j].y, c | c << 16);
                    a[r][m][j][1] = bytes_of(x[r][m][j].z, x[r][m][j].w, c | c << 16);
                }
        }
        const int next = tile + gridDim.x * SCORE_WARPS;
        if (next < tiles) load(next);
        int best[2] = {INT32_MIN, INT32_MIN};
        for (int cb = 0; cb < p.col_blocks; ++cb) {
            int acc[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const uint4 q = frag[(cb * G + j) * 32 + lane];
                mma_u8s8(acc, a[0][0][j][0], a[1][0][j][0], a[0][0][j][1], a[1][0][j][1], q.x, q.y);
                mma_u8s8(acc, a[0][1][j][0], a[1][1][j][0], a[0][1][j][1], a[1][1][j][1], q.z, q.w);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int head = 8 * cb + 2 * t + i, off = 64 * sums[head];  // the bytes are 64 too large
                if (head < p.group) { best[0] = max(best[0], acc[i] - off); best[1] = max(best[1], acc[2 + i] - off); }
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            best[r] = max(best[r], __shfl_xor_sync(~0u, best[r], 1));
            best[r] = max(best[r], __shfl_xor_sync(~0u, best[r], 2));
            const int page = tile * 16 + 8 * r + g;
            if (t == 0 && page < pages) p.keys[((int64_t)b * p.c.H + h) * p.s.max_pages + page] = ordered(__int2float_rn(best[r]) * weight[r]);
        }
    }
}

// Sums of a block's threads before this one's, of two small numbers at once (each sum below 2^31). `shared`: one value a warp.
__device__ __forceinline__ int2 block_exclusive_scan(int2 v, int2 *shared) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int2 s = make_int2(warp_inclusive_scan(v.x, lane), warp_inclusive_scan(v.y, lane));
    if (lane == 31) shared[warp] = s;
    __syncthreads();
    const int2 w = shared[lane];                  // as many warps as lanes
    const int x = __reduce_add_sync(~0u, lane < warp ? w.x : 0), y = __reduce_add_sync(~0u, lane < warp ? w.y : 0);
    return make_int2(x + s.x - v.x, y + s.y - v.y);
}

// The n largest keys of a row, ties to the lowest page. What lies between the smallest key and the largest is cut into BINS equal
// parts, the part that holds the last key taken again, until no more than a warp's worth are in it, which then rank themselves: the
// keys of a row share their leading bits, and counts by those would be atomics on a few words. Up to KEPT keys a thread stay in
// registers.
constexpr int BINS = 2048, KEPT = 8;
__global__ void __launch_bounds__(PICK_THREADS) kv4_pick_kernel(const __grid_constant__ SelectParams p) {
    static_assert(PICK_THREADS == 1024 && BINS == 2 * PICK_THREADS, "a warp to a lane, two bins to a thread");
    __shared__ int histogram[BINS];
    __shared__ int2 scan[32];
    __shared__ uint32_t few[32], low, high;
    __shared__ int left, inside, listed;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    if (tid == 0) { low = ~0u; high = 0; listed = 0; }
    histogram[tid] = histogram[tid + PICK_THREADS] = 0;
    // behind the scores' kernel the lengths are there before the wait: this one starts when all its blocks have waited for what came earlier
    const bool scored = p.s.max_pages > p.n;
    int pages = scored ? pages_of(p, b) : 0;
    wait_earlier();
    let_next_in();
    if (!scored) pages = pages_of(p, b);
    int32_t *out = p.selected + ((int64_t)b * p.c.H + h) * p.n;
    if (pages <= p.n) {
        for (int i = tid; i < p.n; i += PICK_THREADS) out[i] = i < pages ? i : -1;
        return;
    }
    // thread t has keys t * each .. : the order of the threads is the order of the pages
    const uint32_t *keys = p.keys + ((int64_t)b * p.c.H + h) * p.s.max_pages;
    const int each = (pages + PICK_THREADS - 1) / PICK_THREADS, from = min(pages, tid * each), to = min(pages, from + each);
    uint32_t kept[KEPT];
#pragma unroll
    for (int i = 0; i < KEPT; ++i) kept[i] = from + i < to ? keys[from + i] : 0;
    // f(key) for each of the thread's keys that are not taken anyway
    auto each_key = [&](auto f) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i)
            if (from + i < to && from + i >= p.first && from + i < pages - p.last) f(kept[i]);
        for (int i = max(from + KEPT, p.first); i < min(to, pages - p.last); ++i) f(keys[i]);
    };
    uint32_t a = ~0u, z = 0;
    each_key([&](uint32_t k) { a = min(a, k); z = max(z, k); });
    a = __reduce_min_sync(~0u, a);
    z = __reduce_max_sync(~0u, z);
    __syncthreads();
    if (lane == 0) { atomicMin(&low, a); atomicMax(&high, z); }
    __syncthreads();
    a = low;
    int width = 32 - __clz(high - a);             // bits of what the keys span
    int want = p.n - p.first - p.last;            // how many of the keys from `a` on, below a + 2^width, are taken
    auto within = [&](uint32_t k) { return width == 32 || (k - a) >> width == 0; };
    while (width > 0 && want > 0) {
        const int shift = max(0, width - 11);
        each_key([&](uint32_t k) { if (within(k)) atomicAdd(&histogram[(k - a) >> shift], 1); });
        __syncthreads();
        // from the top: thread t has bins BINS - 1 - 2 t and the one below
        const int hi = histogram[BINS - 1 - 2 * tid], lo = histogram[BINS - 2 - 2 * tid];
        const int before = block_exclusive_scan(make_int2(hi + lo, 0), scan).x;
        if (before < want && before + hi + lo >= want) {
            const bool upper = before + hi >= want;
            left = want - before - (upper ? 0 : hi);
            inside = upper ? hi : lo;
            low = a + ((uint32_t)(BINS - (upper ? 1 : 2) - 2 * tid) << shift);
        }
        histogram[BINS - 1 - 2 * tid] = histogram[BINS - 2 - 2 * tid] = 0;
        __syncthreads();
        a = low;
        want = left;
        width = shift;
        if (inside <= 32) break;
        __syncthreads();
    }
    if (width > 0 && want > 0) {                  // the `want`-th of the few that lie in this part
        const int count = inside;
        each_key([&](uint32_t k) { if (within(k)) few[atomicAdd(&listed, 1)] = k; });
        __syncthreads();
        const uint32_t mine = lane < count ? few[lane] : 0;
        int above = 0, same = 0;
        for (int i = 0; i < count; ++i) {
            const uint32_t k = __shfl_sync(~0u, mine, i);
            above += k > mine;
            same += k == mine;
        }
        const uint32_t found = __ballot_sync(~0u, lane < count && above < want && above + same >= want);
        const int one = __ffs(found) - 1;         // equal ones all say so
        a = __shfl_sync(~0u, mine, one);
        want -= __shfl_sync(~0u, above, one);
    }
    if (p.n == p.first + p.last) a = ~0u;         // keys are below that
    // keys above `a`, and the first `want` equal to it, in order
    auto taken = [&](int i) { return i < p.first || i >= pages - p.last; };
    int2 mine = make_int2(0, 0);
    auto count = [&](int i, uint32_t k) { mine.x += taken(i) || k > a; mine.y += !taken(i) && k == a; };
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
        if (from + i < to) count(from + i, kept[i]);
    for (int i = from + KEPT; i < to; ++i) count(i, keys[i]);
    __syncthreads();                              // `scan` is read above
    int2 at = block_exclusive_scan(mine, scan);
    auto put = [&](int i, uint32_t k) {
        const bool more = taken(i) || k > a, same = !taken(i) && k == a;
        if (more || (same && at.y < want)) out[at.x + min(at.y, want)] = i;
        at.x += more;
        at.y += same;
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
        if (from + i < to) put(from + i, kept[i]);
    for (int i = from + KEPT; i < to; ++i) put(i, keys[i]);
}

static int64_t select_workspace(int64_t B, int64_t H, int64_t pages) { return (B * H * pages * 4 + 15) / 16 * 16; }

static int select(const ommx_kv4_select_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv4_select: null args");
    SelectParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv4_select", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv4_select", a->seqs, p.c, &p.s)) return rc;
    if (a->q_dtype != OMMX_DT_BF16 && a->q_dtype != OMMX_DT_F16) return fail(OMMX_E_UNSUPPORTED, "kv4_select: q must be bfloat16 or float16");
    if (a->n_q_heads < p.c.H || a->n_q_heads % p.c.H)
        return fail(OMMX_E_UNSUPPORTED, "kv4_select: %d query heads are not a multiple of %d kv heads", a->n_q_heads, p.c.H);
    if (a->n_q_heads / p.c.H > MOST_HEADS)
        return fail(OMMX_E_UNSUPPORTED, "kv4_select: %d query heads to a kv head (this build serves %d)", a->n_q_heads / p.c.H, MOST_HEADS);
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
    p.q_wide = (reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)(2 * p.q_b) | (uintptr_t)(2 * p.q_h)) % 16 == 0;
    p.keys = (uint32_t *)a->workspace;
    p.selected = a->selected; p.n = a->num_selected; p.first = a->first_pages; p.last = a->last_pages;
    p.group = a->n_q_heads / p.c.H; p.col_blocks = (p.group + 7) / 8;
    p.page_shift = shift_of(p.c.page);
    p.status = a->status;
    if (p.s.max_pages > p.n) {
        const int64_t rows = (int64_t)p.s.B * p.c.H, most = (p.s.max_pages + 16LL * SCORE_WARPS - 1) / (16 * SCORE_WARPS);
        const int64_t fill = (2LL * sm_count() + rows - 1) / rows;          // two blocks to an SM, which is what it holds
        const size_t smem = (size_t)p.col_blocks * (a->cache.head_dim * 16 + 32) + 16;
        const dim3 grid((unsigned)(most < fill ? most : fill), p.c.H, p.s.B);
        const int rc = a->cache.head_dim == 64 ? launch_dependent(kv4_score_kernel<2>, grid, 32 * SCORE_WARPS, smem, st, 1, p)
                                               : launch_dependent(kv4_score_kernel<4>, grid, 32 * SCORE_WARPS, smem, st, 1, p);
        if (rc) return rc;
    }
    return launch_dependent(kv4_pick_kernel, dim3(p.c.H, p.s.B), PICK_THREADS, 0, st, 1, p);
}

}  // namespace kv4
}  // namespace ommx

extern "C" int64_t ommx_b200_kv4_select_workspace_bytes(int32_t batch, int32_t n_kv_heads, int32_t pages_per_seq) {
    return batch < 0 || n_kv_heads < 0 || pages_per_seq < 0 ? 0 : ommx::kv4::select_workspace(batch, n_kv_heads, pages_per_seq);
}
extern "C" int ommx_b200_kv4_select(const ommx_kv4_select_args *args, void *stream) { return ommx::kv4::select(args, (cudaStream_t)stream); }
