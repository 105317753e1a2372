// The 8-bit cache: appending rows and reading rows back.
#include "ommx_kv8.cuh"

namespace ommx {
namespace kv8 {

// ---- runs ---------------------------------------------------------------------------------------
// A run: rows of one sequence that lie in one record. The same answer as kv4::find_run, by a whole block: a thread to a sequence where a
// warp would walk over them 32 at a time. All threads call it; false (for all) when there are fewer than `index` + 1 runs.
constexpr int MOST_WARPS = 8, GATHER_WARPS = 8;
struct RunMemory { int sum[MOST_WARPS]; Run run; };
__device__ __forceinline__ bool find_record(const Seqs &s, const Rows &rows, int index, Run *run, int32_t *status, RunMemory &m) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (!rows.row_start) {                        // one row each: sequence `index`
        if (index >= s.B) return false;
        const int len = s.len[index];
        if (len < 1) { or_status(status, OMMX_ST_BAD_LENGTH); return false; }
        *run = {index, len - 1, len, index};
        return true;
    }
    if (s.B <= 32) return kv4::find_run(s, rows, 4, index, lane, run, status);
    for (int b0 = 0; b0 < s.B; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        int n = 0, first = 0, end = 0, len = 0;
        if (b < s.B) {
            rows.of(b, &first, &end);
            len = s.len[b];
            if (end != first) {
                if (end < first || len < end - first) or_status(status, OMMX_ST_BAD_LENGTH);
                else n = ((len - 1) >> 4) - ((len - (end - first)) >> 4) + 1;
            }
        }
        int sum = warp_inclusive_scan(n, lane);
        if (lane == 31) m.sum[warp] = sum;
        __syncthreads();
        const int w = lane < warps ? m.sum[lane] : 0;
        const int all = __reduce_add_sync(~0u, w);
        sum += __reduce_add_sync(~0u, lane < warp ? w : 0);
        if (index < all) {
            if (sum > index && sum - n <= index) {                          // one thread
                const int start = len - (end - first), block = (start >> 4) + index - (sum - n);
                const int p0 = max(start, block << 4);
                m.run = {b, p0, (int)min((int64_t)len, ((int64_t)block + 1) << 4), first + p0 - start};
            }
            __syncthreads();
            *run = m.run;
            return true;
        }
        index -= all;
        __syncthreads();                          // `sum` is read
    }
    return false;
}
// The page of the run's record, or -1
template <typename P> __device__ __forceinline__ int64_t page_of(const P &p, const Run &run) {
    const int at = run.p0 >> p.page_shift;
    if (at >= p.s.max_pages) { or_status(p.status, OMMX_ST_BAD_LENGTH); return -1; }
    const int64_t id = page_id(p.s, run.b, at);
    if (id < 0 || id >= p.c.num_pages) { or_status(p.status, OMMX_ST_BAD_PAGE); return -1; }
    return id;
}

// ---- rows in and out ----------------------------------------------------------------------------
// eight channels of a type, as words
template <typename T> struct alignas(16) Eight { uint32_t w[2 * sizeof(T)]; };
template <typename T, bool WIDE> __device__ __forceinline__ void fetch8(const T *p, Eight<T> &x) {
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(x) / 16; ++i) reinterpret_cast<uint4 *>(&x)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
        T *to = reinterpret_cast<T *>(&x);
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = p[i];
    }
}
template <typename T> __device__ __forceinline__ float channel(const Eight<T> &x, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(x.w[i]);
    else {
        const uint32_t h = i & 1 ? x.w[i / 2] >> 16 : x.w[i / 2] & 0xFFFFu;
        if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((uint16_t)h));
        else return __uint_as_float(h << 16);
    }
}
// magnitudes as whole numbers, which are in the same order: two to a word, or one
template <typename T> __device__ __forceinline__ uint32_t larger(uint32_t top, uint32_t w) {
    if constexpr (sizeof(T) == 4) return max(top, w & 0x7FFFFFFFu);
    else return __vmaxu2(top, w & 0x7FFF7FFFu);
}
template <typename T> constexpr uint32_t INFINITE = sizeof(T) == 4 ? 0x7F800000u : std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
template <typename T> __device__ __forceinline__ float magnitude(uint32_t bits) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
    else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((uint16_t)bits));
    else return __uint_as_float(bits << 16);
}
__device__ __forceinline__ float tame(float x) { return x != x ? 0.0f : fminf(fmaxf(x, -LARGEST), LARGEST); }

struct AppendParams {
    Cache c;
    Seqs s;
    Rows rows;
    const void *k, *v;
    int64_t k_t, k_h, v_t, v_h;
    int32_t page_shift;
    int32_t *status;
};

// Grid: (records that take rows, shares of their 2 H items); an item is the keys or the values of a head, a warp to it. The warp holds its
// rows (16 at most), whose largest magnitude is an integer maximum, and writes each once. Tokens that the record holds already are read
// again only where the new rows need a larger scale.
// What bounds it: memory where rows are many (8192 of 8 kv heads, D = 128, bf16 9.6 us and fp32 13.5, in graph replays; 50 MB take 7.7 of a copy's rate;
// 65536 rows 69 us, 89 % of it), the chain of launch, lengths, table and rows where they are few (one of one sequence 2.5 us, of 61 too). A row each of many
// sequences is that chain in every block: 1024 are 2048 blocks, 592 at once, 3.5 turns (10.1 us, for 6.3 MB); with ranges every block also looks
// through those of all sequences (14.8).
template <typename T, int G, bool E4M3, bool WIDE>
__global__ void __launch_bounds__(32 * MOST_WARPS, sizeof(T) == 4 ? 2 : 4) kv8_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int D = 32 * G, LANES = D / 8, ROWS = 32 / LANES, TURNS = BLOCK / ROWS;
    __shared__ RunMemory memory;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    wait_earlier();
    let_next_in();
    Run run;
    if (!find_record(p.s, p.rows, blockIdx.x, &run, p.status, memory)) return;
    const int n = run.p1 - run.p0, tau0 = run.p0 & 15, row = lane / LANES, c = 8 * (lane % LANES);
    const int part = (run.p0 >> 4) & (p.c.parts - 1);
    auto rows_of = [&](int item) {
        const int head = item >> 1;
        return item & 1 ? reinterpret_cast<const T *>(p.v) + (int64_t)run.row * p.v_t + (int64_t)head * p.v_h
                        : reinterpret_cast<const T *>(p.k) + (int64_t)run.row * p.k_t + (int64_t)head * p.k_h;
    };
    Eight<T> x[TURNS];
    auto fetch = [&](int item) {
        const T *from = rows_of(item);
        const int64_t step = item & 1 ? p.v_t : p.k_t;
#pragma unroll
        for (int i = 0; i < TURNS; ++i)
            if (i * ROWS + row < n) fetch8<T, WIDE>(from + (i * ROWS + row) * step + c, x[i]);
    };
    const int item0 = blockIdx.y * warps + warp;
    if (item0 < 2 * p.c.H) fetch(item0);          // on their way while the page is looked up
    const int64_t id = page_of(p, run);
    if (id < 0) return;
    bool bad = false;
    for (int item = item0; item < 2 * p.c.H; item += gridDim.y * warps) {
        const int head = item >> 1, which = item & 1;
        const int64_t record = (id * p.c.H + head) * p.c.parts + part;
        const int held = tau0 ? p.c.scales[2 * record + which] : 0;
        if (item != item0) fetch(item);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < TURNS; ++i)
            if (i * ROWS + row < n) {
#pragma unroll
                for (int e = 0; e < (int)(2 * sizeof(T)); ++e) top = larger<T>(top, x[i].w[e]);
            }
        if constexpr (sizeof(T) == 2) top = max(top & 0xFFFFu, top >> 16);
        top = __reduce_max_sync(~0u, top);
        float most = magnitude<T>(top);
        const bool wild = !(most <= LARGEST);     // infinities, NaN, and what is taken to be LARGEST
        if (wild) {
            bad |= top >= INFINITE<T>;
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < TURNS; ++i)
                if (i * ROWS + row < n) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(tame(channel(x[i], e))));
                }
            most = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(m)));
        }
        const int E = max(held, exponent_for<E4M3>(most));
        uint8_t *codes = p.c.codes + record * (32 * D) + which * (16 * D);
        if (tau0 && E > held) {                   // what is there moves to the larger scale
            const Rescale by = rescale_by(held, E);
            for (int at = 16 * lane; at < tau0 * D; at += 512) {
                uint4 *w = reinterpret_cast<uint4 *>(codes + at);
                *w = rescaled<E4M3>(*w, by);
            }
        }
        const float up = __uint_as_float((uint32_t)(254 - min(E, 254)) << 23);                // 2^(127 - E)
#pragma unroll
        for (int i = 0; i < TURNS; ++i)
            if (i * ROWS + row < n) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = channel(x[i], e);
                if (wild) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = tame(f[e]);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= up;
                *reinterpret_cast<uint2 *>(codes + (tau0 + i * ROWS + row) * D + c) =
                    make_uint2(codes_of<E4M3>(f[0], f[1], f[2], f[3]), codes_of<E4M3>(f[4], f[5], f[6], f[7]));
            }
        if (lane == 0 && (!tau0 || E != held)) p.c.scales[2 * record + which] = (uint8_t)E;
        // nothing has attended to the new tokens yet
        if (p.c.weight && which == 0 && lane < n) p.c.weight[record * BLOCK + tau0 + lane] = 0.0f;
    }
    if (bad && lane == 0) or_status(p.status, OMMX_ST_NONFINITE);
}

// ---- reading rows back --------------------------------------------------------------------------
struct GatherParams {
    Cache c;
    Seqs s;
    Rows rows;
    void *k, *v;
    int64_t k_t, k_h, v_t, v_h;
    int32_t page_shift;
    int32_t *status;
};
template <typename T> __device__ __forceinline__ uint32_t two_of(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
// eight channels
template <typename T, bool WIDE> __device__ __forceinline__ void store8(T *to, const float (&x)[8]) {
    constexpr int WORDS = 2 * sizeof(T);
    alignas(16) uint32_t w[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(x[i]);
        else w[i] = two_of<T>(x[2 * i], x[2 * i + 1]);
    }
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) reinterpret_cast<uint4 *>(to)[i] = reinterpret_cast<const uint4 *>(w)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = reinterpret_cast<const T *>(w)[i];
    }
}

// Grid as above; a lane reads 8 codes at a time, so that a warp's store of 16-bit rows is whole rows: 8192 rows x 8 heads 10.8 us, 14.5 with 16 codes a lane,
// whose stores left gaps and which took 64 registers. Since then 7.6 in graph replays (outputs of 34 MB that stay in the cache), 65536 rows 67.4: what it reads
// and writes bounds it, 91 % of a copy's rate. fp32 rows are two stores a lane, each of every other 16 bytes: 8192 rows 20.9 us, for bytes of 12.8.
template <typename T, int G, bool E4M3, bool WIDE>
__global__ void __launch_bounds__(32 * GATHER_WARPS, 6) kv8_gather_kernel(const __grid_constant__ GatherParams p) {
    constexpr int D = 32 * G, LANES = D / 8, ROWS = 32 / LANES, TURNS = BLOCK / ROWS;
    __shared__ RunMemory memory;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    wait_earlier();
    let_next_in();
    Run run;
    if (!find_record(p.s, p.rows, blockIdx.x, &run, p.status, memory)) return;
    const int n = run.p1 - run.p0, tau0 = run.p0 & 15, row = lane / LANES, c = 8 * (lane % LANES);
    const int64_t id = page_of(p, run);
    if (id < 0) return;
    const int part = (run.p0 >> 4) & (p.c.parts - 1);
    for (int item = blockIdx.y * warps + warp; item < 2 * p.c.H; item += gridDim.y * warps) {
        const int head = item >> 1, which = item & 1;
        const int64_t record = (id * p.c.H + head) * p.c.parts + part;
        const uint8_t *codes = p.c.codes + record * (32 * D) + which * (16 * D) + (tau0 + row) * D + c;
        T *to = which ? reinterpret_cast<T *>(p.v) + (int64_t)run.row * p.v_t + (int64_t)head * p.v_h + c
                      : reinterpret_cast<T *>(p.k) + (int64_t)run.row * p.k_t + (int64_t)head * p.k_h + c;
        const int64_t step = which ? p.v_t : p.k_t;
        uint2 w[TURNS];
#pragma unroll
        for (int i = 0; i < TURNS; ++i)
            if (i * ROWS + row < n) w[i] = *reinterpret_cast<const uint2 *>(codes + i * ROWS * D);
        const float scale = scale_of(p.c.scales[2 * record + which]);
#pragma unroll
        for (int i = 0; i < TURNS; ++i)
            if (i * ROWS + row < n) {
                float a[4], b[4];
                numbers_of<E4M3>(w[i].x, a);
                numbers_of<E4M3>(w[i].y, b);
                const float x[8] = {a[0] * scale, a[1] * scale, a[2] * scale, a[3] * scale, b[0] * scale, b[1] * scale, b[2] * scale, b[3] * scale};
                store8<T, WIDE>(to + (i * ROWS + row) * step, x);
            }
    }
}

// ---- host ---------------------------------------------------------------------------------------
static bool aligned16(const void *p, int64_t a, int64_t b, int64_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(a * bytes) | (uintptr_t)(b * bytes)) % 16 == 0;
}
static bool known_dtype(int32_t d) { return d == OMMX_DT_F32 || d == OMMX_DT_BF16 || d == OMMX_DT_F16; }

// kernel<T, G, E4M3, WIDE> of a type, a head size, a code and whether all rows start on 16-byte boundaries
#define KV8_OF_WIDE(kernel, T, G, code, wide) ((wide) ? kernel<T, G, code, true> : kernel<T, G, code, false>)
#define KV8_OF_CODE(kernel, T, G, code, wide) ((code) == OMMX_KV8_E4M3 ? KV8_OF_WIDE(kernel, T, G, true, wide) : KV8_OF_WIDE(kernel, T, G, false, wide))
#define KV8_OF_SIZE(kernel, T, G, code, wide) ((G) == 4 ? KV8_OF_CODE(kernel, T, 4, code, wide) : KV8_OF_CODE(kernel, T, 2, code, wide))
#define KV8_PICK(kernel, dtype, G, code, wide)                                          \
    ((dtype) == OMMX_DT_F32 ? KV8_OF_SIZE(kernel, float, G, code, wide)                 \
                            : ((dtype) == OMMX_DT_F16 ? KV8_OF_SIZE(kernel, __half, G, code, wide) : KV8_OF_SIZE(kernel, __nv_bfloat16, G, code, wide)))

// Blocks of up to eight warps, an item to a warp where there are not many more of them than the SMs hold
static int grid_of(const char *who, int64_t runs, int H, dim3 *grid, int *threads) {
    const int items = 2 * H, warps = items < MOST_WARPS ? items : MOST_WARPS, blocks = (items + warps - 1) / warps;
    if (runs >= 1LL << 31) return fail(OMMX_E_UNSUPPORTED, "%s: %lld runs of rows in one call", who, (long long)runs);
    *threads = 32 * warps;
    *grid = dim3((unsigned)runs, (unsigned)(runs * blocks <= 16LL * sm_count() ? blocks : blocks > 4 ? blocks / 4 : 1));
    return 0;
}

static int append(const ommx_kv8_append_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv8_append: null args");
    AppendParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv8_append", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv8_append", a->seqs, p.c, &p.s)) return rc;
    if (a->num_rows < 0) return fail(OMMX_E_ARG, "kv8_append: num_rows must not be negative");
    if (!known_dtype(a->dtype)) return fail(OMMX_E_ARG, "kv8_append: dtype %d is none of float32, bfloat16, float16", a->dtype);
    if (p.s.B == 0 || a->num_rows == 0) return 0;
    if (!a->k_new || !a->v_new) return fail(OMMX_E_ARG, "kv8_append: k_new and v_new must not be null");
    if (!a->row_start && a->num_rows != p.s.B) return fail(OMMX_E_ARG, "kv8_append: without row_start there is one row for each of the %d sequences, not %d rows", p.s.B, a->num_rows);
    p.rows = {a->row_start, a->num_rows};
    p.k = a->k_new; p.v = a->v_new;
    p.k_t = a->k_stride_t; p.k_h = a->k_stride_h; p.v_t = a->v_stride_t; p.v_h = a->v_stride_h;
    p.page_shift = shift_of(p.c.page);
    p.status = a->status;
    const int bytes = a->dtype == OMMX_DT_F32 ? 4 : 2;
    const bool wide = aligned16(a->k_new, p.k_t, p.k_h, bytes) && aligned16(a->v_new, p.v_t, p.v_h, bytes);
    int threads;
    dim3 grid;
    if (int rc = grid_of("kv8_append", kv4::most_runs(a->num_rows, p.s.B, BLOCK, a->row_start == nullptr), p.c.H, &grid, &threads)) return rc;
    return launch_dependent(KV8_PICK(kv8_append_kernel, a->dtype, a->cache.head_dim / 32, a->cache.code, wide), grid, threads, 0, st, 1, p);
}

static int gather(const ommx_kv8_gather_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv8_gather: null args");
    GatherParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv8_gather", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv8_gather", a->seqs, p.c, &p.s)) return rc;
    if (a->num_rows < 0) return fail(OMMX_E_ARG, "kv8_gather: num_rows must not be negative");
    if (!known_dtype(a->dtype)) return fail(OMMX_E_ARG, "kv8_gather: dtype %d is none of float32, bfloat16, float16", a->dtype);
    if (p.s.B == 0 || a->num_rows == 0) return 0;
    if (!a->k || !a->v) return fail(OMMX_E_ARG, "kv8_gather: k and v must not be null");
    if (!a->row_start && a->num_rows != p.s.B) return fail(OMMX_E_ARG, "kv8_gather: without row_start there is one row for each of the %d sequences, not %d rows", p.s.B, a->num_rows);
    p.rows = {a->row_start, a->num_rows};
    p.k = a->k; p.v = a->v;
    p.k_t = a->k_stride_t; p.k_h = a->k_stride_h; p.v_t = a->v_stride_t; p.v_h = a->v_stride_h;
    p.page_shift = shift_of(p.c.page);
    p.status = a->status;
    const int bytes = a->dtype == OMMX_DT_F32 ? 4 : 2;
    const bool wide = aligned16(a->k, p.k_t, p.k_h, bytes) && aligned16(a->v, p.v_t, p.v_h, bytes);
    int threads;
    dim3 grid;
    if (int rc = grid_of("kv8_gather", kv4::most_runs(a->num_rows, p.s.B, BLOCK, a->row_start == nullptr), p.c.H, &grid, &threads)) return rc;
    return launch_dependent(KV8_PICK(kv8_gather_kernel, a->dtype, a->cache.head_dim / 32, a->cache.code, wide), grid, threads, 0, st, 1, p);
}

}  // namespace kv8
}  // namespace ommx

extern "C" int ommx_b200_kv8_append(const ommx_kv8_append_args *args, void *stream) { return ommx::kv8::append(args, (cudaStream_t)stream); }
extern "C" int ommx_b200_kv8_gather(const ommx_kv8_gather_args *args, void *stream) { return ommx::kv8::gather(args, (cudaStream_t)stream); }
