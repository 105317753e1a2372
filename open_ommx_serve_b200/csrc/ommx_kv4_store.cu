// The 4-bit cache: appending rows (rotation, quantization, page summaries) and reading rows back.
#include <type_traits>

#include "ommx_kv4.cuh"
#include "ommx_kv_device.cuh"

namespace ommx {
namespace kv4 {

using kv::max3_nan;

// ---- rows in and out ----------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// eight channels; WIDE: the address is a multiple of 16 bytes
template <typename T> struct alignas(16) Eight { T v[8]; };
template <typename T, bool WIDE> __device__ __forceinline__ void fetch8(const T *p, Eight<T> &x) {
    if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x.v[i] = p[i];
    } else {
#pragma unroll
        for (int i = 0; i < (int)sizeof(x) / 16; ++i) reinterpret_cast<uint4 *>(&x)[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
}
template <typename T> __device__ __forceinline__ void unpack8(const Eight<T> &e, float *x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(e.v[i]);
}
template <typename T, bool WIDE> __device__ __forceinline__ void store8(T *p, const float *x) {
    if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = from_f32<T>(x[i]);
    } else {
        alignas(16) T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = from_f32<T>(x[i]);
#pragma unroll
        for (int i = 0; i < (int)sizeof(v) / 16; ++i) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(v)[i];
    }
}
template <int N> __device__ __forceinline__ void load_f32(const float *p, float *x) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(p + i);
        x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
}

// x1' = x1 c - x2 s, x2' = x2 c + x1 s: every product and sum rounded by itself, as a rotation written out in 32 bits has it
__device__ __forceinline__ void turn(float &x1, float &x2, float c, float s) {
    const float a = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
    x2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
    x1 = a;
}

// ---- the quantizer ------------------------------------------------------------------------------
// Bits of the largest bf16 not above x, and of the smallest not below it; x finite
__device__ __forceinline__ uint32_t floor_bf16(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b + ((int32_t)b < 0 ? 0xFFFFu : 0u)) >> 16;
}
__device__ __forceinline__ uint32_t ceil_bf16(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b + ((int32_t)b < 0 ? 0u : 0xFFFFu)) >> 16;
}

struct AppendParams {
    Cache c;
    Seqs s;
    Rows rows;
    uint16_t *summary;
    const void *k, *v, *q;
    void *q_out;
    int64_t k_t, k_h, v_t, v_h, q_t, q_h, o_t, o_h;
    const float *cos, *sin;
    int64_t cs_stride;
    const void *positions;
    int32_t positions64, num_positions, rot, interleaved, Hq, page_shift, kv_blocks, blocks, q_rows, split;
    int32_t *status;
};

// Position of a row in the rotation tables; -1 (reported) outside them. 0 without a rotation.
__device__ __forceinline__ int rope_row(const AppendParams &p, int row, int pos) {
    if (!p.rot) return 0;
    int64_t at = pos;
    if (p.positions) at = p.positions64 ? reinterpret_cast<const int64_t *>(p.positions)[row] : reinterpret_cast<const int32_t *>(p.positions)[row];
    if (at < 0 || at >= p.num_positions) { or_status(p.status, OMMX_ST_BAD_LENGTH); return -1; }
    return (int)at;
}

// Rotation of eight channels c .. c + 7 of a key, below p.rot. Pairs (c, c + rot / 2): y holds the partners; pairs (2 i, 2 i + 1): both
// lie here.
__device__ __forceinline__ void rotate_key(const AppendParams &p, float (&x)[8], const float (&y)[8], int at, int c) {
    const int half = p.rot / 2;
    if (p.interleaved) {
        float cs[4], sn[4];
        load_f32<4>(p.cos + at * p.cs_stride + c / 2, cs);
        load_f32<4>(p.sin + at * p.cs_stride + c / 2, sn);
#pragma unroll
        for (int i = 0; i < 4; ++i) turn(x[2 * i], x[2 * i + 1], cs[i], sn[i]);
        return;
    }
    const bool upper = c >= half;
    const int64_t from = at * p.cs_stride + (upper ? c - half : c);
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
        float cs[4], sn[4];
        load_f32<4>(p.cos + from + k, cs);
        load_f32<4>(p.sin + from + k, sn);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float s = __fmul_rn(y[k + i], sn[i]);
            x[k + i] = __fadd_rn(__fmul_rn(x[k + i], cs[i]), upper ? s : -s);
        }
    }
}

// of three, NaN if one is
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Codes and parameters of one group of 32 channels, eight in each of the four lanes of a row: the lane's word of codes, and the
// group's word of parameters. `bad`: x held a value that is not finite.
__device__ __forceinline__ uint32_t quantize_group(float (&x)[8], uint32_t *params, bool *bad) {
    float lo = min3_nan(min3_nan(min3_nan(x[0], x[1], x[2]), x[3], x[4]), x[5], fminf(x[6], x[7]));
    float hi = max3_nan(max3_nan(max3_nan(x[0], x[1], x[2]), x[3], x[4]), x[5], max3_nan(x[6], x[7], x[7]));
    if (!(hi <= LARGEST && lo >= -LARGEST)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            *bad = *bad || !(fabsf(x[i]) < INFINITY);
            x[i] = x[i] != x[i] ? 0.0f : fminf(fmaxf(x[i], -LARGEST), LARGEST);
        }
        lo = hi = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); }
    }
#pragma unroll
    for (int d = 1; d < 4; d *= 2) {
        lo = fminf(lo, __shfl_xor_sync(~0u, lo, d));
        hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, d));
    }
    lo += 0.0f;                                                            // -0 -> 0, whichever lane held it
    const uint32_t zb = floor_bf16(lo);
    const float zero = __uint_as_float(zb << 16);
    uint32_t sb = ceil_bf16(__fmul_rn(__fsub_rn(hi, zero), SHRINK / 15.0f));
    const float scale = __uint_as_float(sb << 16);
    float inverse = __fdiv_rn(SHRINK, scale);
    if (scale < SMALLEST) { inverse = 0.0f; sb = 0; }
    *params = sb << 16 | zb;
    // 2^23 + code in the float's last bits; the shifted leading parts are taken off at once
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word += __float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(x[i], zero), inverse), 8388608.0f)) << (4 * i);
    constexpr uint32_t LEAD = 0x4B000000u;
    return word - (LEAD + (LEAD << 4));                                    // higher shifts push it out of 32 bits
}

// Summary: two bf16 in a register, maxima in the first half of the array and negated minima in the second, so both grow
constexpr uint32_t NOTHING = 0xFF80FF80u;                                  // -inf twice

// One warp appends up to 16 rows that share a record, ROWS of them at a time: lane ((row, j), t) has channels 32 j + 8 t + 0..7, so a
// group's extremes meet in two shuffles. A key's partners in the rotation are loaded too (from the first-level cache), not exchanged.
// Bounds: a row of K and V is 512 bytes in and 160 out at D = 128, and some 285 instructions of a warp: 8192 rows x 8 heads take 24 us
// (64 % of the issue slots; fp32 rows 35) where their bytes take 7 (12), one row 4.0. Eight rows at a time with all groups to a lane (127 registers)
// took 22, and 7.0 for one row; the next rows' loads ahead of these rows' work 25.5 (96 registers, fewer warps). With 72 registers 16-bit rows
// spill some: 14 loads and stores of the 550 instructions for two rows of K and V.
template <typename T, int G, bool WIDE>
__device__ __forceinline__ void append_part(const AppendParams &p, uint8_t *rec, int head, int first_row, int first_pos, int tau0, int n,
                                            int lane, uint32_t (&best)[2][4]) {
    constexpr int ROWS = 8 / G;
    const int t = lane & 3, j = lane / 4 % G, odd = lane / (4 * G) & 1, c = 32 * j + 8 * t;
    const bool rotates = c < p.rot, partner = rotates && !p.interleaved;
    const int other = c < p.rot / 2 ? p.rot / 2 : -p.rot / 2;               // where the partners lie
    bool bad = false;
    Eight<T> kk = {}, yy = {}, vv = {};
    int tau = tau0 / ROWS * ROWS + lane / (4 * G);                          // the lane's token of the record; row tau - tau0 of the n
    const T *k = reinterpret_cast<const T *>(p.k) + (int64_t)(first_row + tau - tau0) * p.k_t + (int64_t)head * p.k_h + c;
    const T *v = reinterpret_cast<const T *>(p.v) + (int64_t)(first_row + tau - tau0) * p.v_t + (int64_t)head * p.v_h + c;
    const int64_t k_step = ROWS * p.k_t, v_step = ROWS * p.v_t;
    uint32_t *words = reinterpret_cast<uint32_t *>(rec) + (tau * 4 + t) * G + j;         // of the lane's token
    uint32_t *params = reinterpret_cast<uint32_t *>(rec + Rec<G>::KP) + tau * G + j;
    uint8_t *const quads = rec + Rec<G>::V + 4 * (G * 8 * t + j);
    const bool summary = p.summary, placed = !p.positions;
    // places in their sequences are rotation positions, all of them in the tables: nothing to look at row by row
    const bool sure = !p.rot || (placed && first_pos + n <= p.num_positions);
    auto fetch = [&] {
        if (tau >= tau0 && tau < tau0 + n) {
            fetch8<T, WIDE>(k, kk);
            if (partner) fetch8<T, WIDE>(k + other, yy);
            fetch8<T, WIDE>(v, vv);
        }
        k += k_step;
        v += v_step;
    };
#pragma unroll 1
    for (int last = tau0 + n - 1, base = tau0 / ROWS * ROWS; base <= last; base += ROWS) {
        const int here = tau, i = here - tau0;
        bool on = i >= 0 && i < n;
        int at = first_pos + i;
        if (!sure) {
            at = on ? rope_row(p, first_row + i, at) : 0;
            on = on && at >= 0;
        }
        fetch();
        tau += ROWS;
        float x[8], y[8];
        unpack8(kk, x);
        if (rotates) {
            unpack8(yy, y);
            rotate_key(p, x, y, on ? at : 0, c);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = to_f32(from_f32<T>(x[e]));   // what a separate rotation would have stored
        }
        uint32_t par, word = quantize_group(x, &par, &bad);
        if (on) {
            *words = word;
            if (t == 0) *params = par;
            if (summary) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = x[2 * e], b = x[2 * e + 1];
                    uint32_t up, down;
                    if constexpr (std::is_same<T, __nv_bfloat16>::value) {          // what came from bf16 is bf16
                        up = down = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
                    } else {
                        up = ceil_bf16(a) | ceil_bf16(b) << 16;
                        down = floor_bf16(a) | floor_bf16(b) << 16;
                    }
                    best[0][e] = max_bf16x2(best[0][e], up);
                    best[1][e] = max_bf16x2(best[1][e], down ^ 0x80008000u);
                }
            }
        }
        // values: a word holds four channels of two tokens; the even token's lane makes those of channel quad 2 t, the odd one's of 2 t + 1
        unpack8(vv, x);
        word = quantize_group(x, &par, &bad);
        const bool both = __shfl_xor_sync(~0u, (int)on, 4 * G) && on;
        const uint32_t theirs = __shfl_xor_sync(~0u, word, 4 * G);
        uint8_t *quad = quads + 4 * G * (32 * (here >> 3) + (here >> 1 & 3));
        if (both) {
            *reinterpret_cast<uint32_t *>(quad + 16 * G * odd) = odd ? __byte_perm(theirs, word, 0x7632) : __byte_perm(word, theirs, 0x5410);
        } else if (on) {
            *reinterpret_cast<uint16_t *>(quad + 2 * odd) = (uint16_t)word;
            *reinterpret_cast<uint16_t *>(quad + 16 * G + 2 * odd) = (uint16_t)(word >> 16);
        }
        if (on && t == 0) params[(Rec<G>::VP - Rec<G>::KP) / 4] = par;
        words += ROWS * 4 * G;
        params += ROWS * G;
    }
    if (bad) or_status(p.status, OMMX_ST_NONFINITE);
}

constexpr int WARPS = 4;

// Grid: `blocks` for each run of rows that share a page. The first kv_blocks of a run take its keys and values, a warp to 16 tokens of a
// head (pages over 64 tokens: a warp to several of them); the others rotate the query rows, q_rows each. The two lie side
// by side in the grid, but do not hide each other: 8192 rows x 8 kv heads take 24 us, with 32 query heads 48 (their bytes 7 and 28).
// A run is found by every warp in turn over 32 sequences at a time, which is what a step of many sequences costs: one row each of 61
// sequences 5.0 us, of 512 21, of 1024 49.
template <typename T, int G, bool WIDE>
__global__ void __launch_bounds__(32 * WARPS, sizeof(T) == 4 ? 5 : 7) kv4_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int D = 32 * G;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    wait_earlier();
    let_next_in();
    Run run;
    const int runs_at = blockIdx.x / p.blocks, block = blockIdx.x - runs_at * p.blocks;
    if (!find_run(p.s, p.rows, p.page_shift, runs_at, lane, &run, p.status)) return;
    const int page = 1 << p.page_shift;

    if (block >= p.kv_blocks) {                                   // ---- query rows
        int p0 = run.p0, p1 = run.p1;
        if (p.q_rows < page) {
            const int from = (run.p0 & -page) + (block - p.kv_blocks) * p.q_rows;
            p0 = max(p0, from);
            p1 = min(p1, from + p.q_rows);
        }
        // a thread to sixteen channels of a row: their angles are loaded once for all heads, and two heads are on their way
        constexpr int CHUNKS = D / 16, TURNS = 2;
        const int slots = 32 * WARPS / CHUNKS, rows = p1 - p0, lots = max(1, slots / max(rows, 1));   // threads to a chunk: rows x lots
        const int c = threadIdx.x % CHUNKS, slot = threadIdx.x / CHUNKS;
        for (int r = slot / lots; r < rows; r += slots / lots) {
            const int row = run.row + p0 - run.p0 + r, at = rope_row(p, row, p0 + r);
            if (at < 0) continue;
            const bool turned = 16 * c < p.rot;
            const int first = turned && !p.interleaved ? 8 * c : 16 * c, second = turned && !p.interleaved ? 8 * c + p.rot / 2 : 16 * c + 8;
            float cs[8], sn[8];
            if (turned) {
                load_f32<8>(p.cos + at * p.cs_stride + 8 * c, cs);
                load_f32<8>(p.sin + at * p.cs_stride + 8 * c, sn);
            }
            const T *in = reinterpret_cast<const T *>(p.q) + (int64_t)row * p.q_t;
            T *out = reinterpret_cast<T *>(p.q_out) + (int64_t)row * p.o_t;
            for (int h0 = slot % lots; h0 < p.Hq; h0 += TURNS * lots) {
                Eight<T> raw[TURNS][2];
#pragma unroll
                for (int u = 0; u < TURNS; ++u)
                    if (h0 + u * lots < p.Hq) {
                        fetch8<T, WIDE>(in + (h0 + u * lots) * p.q_h + first, raw[u][0]);
                        fetch8<T, WIDE>(in + (h0 + u * lots) * p.q_h + second, raw[u][1]);
                    }
#pragma unroll
                for (int u = 0; u < TURNS; ++u)
                    if (h0 + u * lots < p.Hq) {
                        float x[16];
                        unpack8(raw[u][0], x);
                        unpack8(raw[u][1], x + 8);
                        if (turned) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                if (p.interleaved) turn(x[2 * e], x[2 * e + 1], cs[e], sn[e]);
                                else turn(x[e], x[8 + e], cs[e], sn[e]);
                            }
                        }
                        store8<T, WIDE>(out + (h0 + u * lots) * p.o_h + first, x);
                        store8<T, WIDE>(out + (h0 + u * lots) * p.o_h + second, x + 8);
                    }
            }
        }
        return;
    }

    // ---- keys and values
    const int pieces = p.c.parts * p.split, warps_a_head = min(pieces, WARPS), heads = WARPS / warps_a_head, size = 16 / p.split;
    const int head = block * heads + warp / warps_a_head;
    const int at = run.p0 >> p.page_shift;
    int64_t id = -1;
    if (at < p.s.max_pages) id = page_id(p.s, run.b, at);
    else or_status(p.status, OMMX_ST_BAD_LENGTH);
    if (at < p.s.max_pages && (id < 0 || id >= p.c.num_pages)) { or_status(p.status, OMMX_ST_BAD_PAGE); id = -1; }
    if (id < 0) return;                                                     // the whole block: one run, one page
    uint32_t best[2][4];                          // maxima and negated minima of the lane's eight channels
#pragma unroll
    for (int i = 0; i < 4; ++i) best[0][i] = best[1][i] = NOTHING;
    if (head < p.c.H)
        for (int piece = warp % warps_a_head; piece < pieces; piece += warps_a_head) {
            const int part = piece / p.split, base = (run.p0 & -page) + 16 * part;
            const int p0 = max(run.p0, base + piece % p.split * size), p1 = min(run.p1, base + (piece % p.split + 1) * size);
            if (p0 >= p1) continue;
            uint8_t *rec = p.c.records + ((id * p.c.H + head) * p.c.parts + part) * Rec<G>::BYTES;
            append_part<T, G, WIDE>(p, rec, head, run.row + p0 - run.p0, p0, p0 - base, p1 - p0, lane, best);
        }
    if (!p.summary) return;
#pragma unroll
    for (int d = 4 * G; d < 32; d *= 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            best[0][i] = max_bf16x2(best[0][i], __shfl_xor_sync(~0u, best[0][i], d));
            best[1][i] = max_bf16x2(best[1][i], __shfl_xor_sync(~0u, best[1][i], d));
        }
    // the first row's lanes go on with the maxima, the second's with the minima
    __shared__ uint4 shared[WARPS][32];
    const bool low = lane / (4 * G) & 1;
    uint4 own = low ? make_uint4(best[1][0], best[1][1], best[1][2], best[1][3]) : make_uint4(best[0][0], best[0][1], best[0][2], best[0][3]);
    if (warps_a_head > 1) {
        shared[warp][lane] = own;
        __syncthreads();
        if (warp % warps_a_head) return;
        for (int w = 1; w < warps_a_head; ++w) {
            const uint4 o = shared[warp + w][lane];
            own = make_uint4(max_bf16x2(own.x, o.x), max_bf16x2(own.y, o.y), max_bf16x2(own.z, o.z), max_bf16x2(own.w, o.w));
        }
    }
    if (head >= p.c.H || lane >= 8 * G) return;
    if (own.x == NOTHING) return;                                           // none of its rows was stored
    uint4 *to = reinterpret_cast<uint4 *>(p.summary + ((id * p.c.H + head) * 2 + low) * D + 32 * (lane / 4 % G) + 8 * (lane & 3));
    const uint32_t sign = low ? 0x80008000u : 0u;
    if (run.p0 & (page - 1)) {                                              // the page held tokens before: theirs count too
        const uint4 o = *to;
        own = make_uint4(max_bf16x2(own.x, o.x ^ sign), max_bf16x2(own.y, o.y ^ sign), max_bf16x2(own.z, o.z ^ sign), max_bf16x2(own.w, o.w ^ sign));
    }
    *to = make_uint4(own.x ^ sign, own.y ^ sign, own.z ^ sign, own.w ^ sign);
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

// Grid: runs of rows that share a record of 16 tokens; a warp to a head of it (up to GATHER_WARPS at once).
constexpr int GATHER_WARPS = 8;
template <typename T, int G, bool WIDE>
__global__ void __launch_bounds__(32 * GATHER_WARPS) kv4_gather_kernel(const __grid_constant__ GatherParams p) {
    using W = typename Words<G>::T;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    wait_earlier();
    let_next_in();
    Run run;
    if (!find_run(p.s, p.rows, 4, blockIdx.x, lane, &run, p.status)) return;
    const int at = run.p0 >> p.page_shift, part = (run.p0 >> 4) & (p.c.parts - 1);
    if (at >= p.s.max_pages) { or_status(p.status, OMMX_ST_BAD_LENGTH); return; }
    const int64_t id = page_id(p.s, run.b, at);
    if (id < 0 || id >= p.c.num_pages) { or_status(p.status, OMMX_ST_BAD_PAGE); return; }
    const int tau0 = run.p0 & 15, n = run.p1 - run.p0;
    for (int head = warp; head < p.c.H; head += blockDim.x / 32) {
        const uint8_t *rec = p.c.records + ((id * p.c.H + head) * p.c.parts + part) * Rec<G>::BYTES;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int tau = 8 * half + g, i = tau - tau0;
            alignas(16) uint32_t kw[G], vw[G], kp[G], vp[G];
            *reinterpret_cast<W *>(kw) = reinterpret_cast<const W *>(rec)[32 * half + lane];
            *reinterpret_cast<W *>(vw) = reinterpret_cast<const W *>(rec + Rec<G>::V)[32 * half + lane];
            *reinterpret_cast<W *>(kp) = reinterpret_cast<const W *>(rec + Rec<G>::KP)[tau];
            // a value word holds four channels of two tokens: with the lane of the next four, eight channels of one
            const int token = 8 * half + 2 * t + (g & 1), iv = token - tau0;
            *reinterpret_cast<W *>(vp) = reinterpret_cast<const W *>(rec + Rec<G>::VP)[token];
            T *k = reinterpret_cast<T *>(p.k) + (int64_t)(run.row + i) * p.k_t + (int64_t)head * p.k_h + 8 * t;
            T *v = reinterpret_cast<T *>(p.v) + (int64_t)(run.row + iv) * p.v_t + (int64_t)head * p.v_h + 8 * (g >> 1);
#pragma unroll
            for (int j = 0; j < G; ++j) {
                float x[8];
                const uint32_t other = __shfl_xor_sync(~0u, vw[j], 4);
                const uint32_t w = g & 1 ? __byte_perm(other, vw[j], 0x7632) : __byte_perm(vw[j], other, 0x5410);
                if (i >= 0 && i < n) {
                    const float s = __uint_as_float(kp[j] & 0xFFFF0000u), z = __uint_as_float(kp[j] << 16);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)(kw[j] >> (4 * e) & 15u), s, z);
                    store8<T, WIDE>(k + 32 * j, x);
                }
                if (iv >= 0 && iv < n) {
                    const float s = __uint_as_float(vp[j] & 0xFFFF0000u), z = __uint_as_float(vp[j] << 16);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)(w >> (4 * e) & 15u), s, z);
                    store8<T, WIDE>(v + 32 * j, x);
                }
            }
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------
static bool aligned16(const void *p, int64_t a, int64_t b, int64_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(a * bytes) | (uintptr_t)(b * bytes)) % 16 == 0;
}
static bool known_dtype(int32_t d) { return d == OMMX_DT_F32 || d == OMMX_DT_BF16 || d == OMMX_DT_F16; }

// kernel<T, G, WIDE> of a type code, a head size and whether all rows start on 16-byte boundaries
#define KV4_OF_TYPE(kernel, T, G, wide) ((G) == 4 ? ((wide) ? kernel<T, 4, true> : kernel<T, 4, false>) : ((wide) ? kernel<T, 2, true> : kernel<T, 2, false>))
#define KV4_PICK(kernel, dtype, G, wide)                                             \
    ((dtype) == OMMX_DT_F32 ? KV4_OF_TYPE(kernel, float, G, wide)                    \
                            : ((dtype) == OMMX_DT_F16 ? KV4_OF_TYPE(kernel, __half, G, wide) : KV4_OF_TYPE(kernel, __nv_bfloat16, G, wide)))

static int append(const ommx_kv4_append_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv4_append: null args");
    AppendParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv4_append", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv4_append", a->seqs, p.c, &p.s)) return rc;
    if (a->num_rows < 0) return fail(OMMX_E_ARG, "kv4_append: num_rows must not be negative");
    if (!known_dtype(a->dtype)) return fail(OMMX_E_ARG, "kv4_append: dtype %d is none of float32, bfloat16, float16", a->dtype);
    if (p.s.B == 0 || a->num_rows == 0) return 0;
    if (!a->k_new || !a->v_new) return fail(OMMX_E_ARG, "kv4_append: k_new and v_new must not be null");
    if (!a->row_start && a->num_rows != p.s.B) return fail(OMMX_E_ARG, "kv4_append: without row_start there is one row for each of the %d sequences, not %d rows", p.s.B, a->num_rows);
    const int D = a->cache.head_dim, G = D / 32;
    if (a->rot_dim != 0) {
        if (a->rot_dim != 32 && a->rot_dim != 64 && a->rot_dim != 128)
            return fail(OMMX_E_UNSUPPORTED, "kv4_append: rot_dim %d (this build rotates 32, 64 or 128 channels)", a->rot_dim);
        if (a->rot_dim > D) return fail(OMMX_E_ARG, "kv4_append: rot_dim %d of heads of %d", a->rot_dim, D);
        if (!a->cos || !a->sin || a->num_positions <= 0) return fail(OMMX_E_ARG, "kv4_append: a rotation needs cos, sin and at least one position");
        if (!aligned16(a->cos, a->cs_stride, 0, 4) || !aligned16(a->sin, 0, 0, 4) || a->cs_stride < a->rot_dim / 2)
            return fail(OMMX_E_ARG, "kv4_append: rows of cos and sin must start on 16-byte boundaries and hold rot_dim / 2 values");
    }
    if (a->q && (!a->q_out || a->n_q_heads <= 0)) return fail(OMMX_E_ARG, "kv4_append: q needs q_out and n_q_heads");
    if (a->q && a->rot_dim == 0) return fail(OMMX_E_ARG, "kv4_append: q without a rotation");
    p.rows = {a->row_start, a->num_rows};
    p.summary = (uint16_t *)a->cache.summary;
    p.k = a->k_new; p.v = a->v_new; p.q = a->q; p.q_out = a->q_out;
    p.k_t = a->k_stride_t; p.k_h = a->k_stride_h; p.v_t = a->v_stride_t; p.v_h = a->v_stride_h;
    p.q_t = a->q_stride_t; p.q_h = a->q_stride_h; p.o_t = a->qo_stride_t; p.o_h = a->qo_stride_h;
    p.cos = a->cos; p.sin = a->sin; p.cs_stride = a->cs_stride;
    p.positions = a->positions; p.positions64 = a->positions_is_int64; p.num_positions = a->num_positions;
    p.rot = a->rot_dim; p.interleaved = a->interleaved; p.Hq = a->q ? a->n_q_heads : 0;
    p.page_shift = shift_of(p.c.page);
    p.status = a->status;
    // A record to a warp, or to two or four where there are fewer records than warps that the SMs hold (2049 rows of 4 heads: 14.8 us
    // with one, 10.2 with four)
    p.split = 1;
    while (p.split < 4 && a->num_rows >= 16LL * p.split * p.s.B && (int64_t)a->num_rows * p.c.H / (16 * p.split) < 28LL * sm_count()) p.split *= 2;
    const int pieces = p.c.parts * p.split, heads = WARPS / (pieces < WARPS ? pieces : WARPS);
    p.kv_blocks = (p.c.H + heads - 1) / heads;
    // Query rows to a block: at most 8 (8192 rows 48.4 us, 50.8 with 16, 52.4 with 4), and fewer until there are two blocks to an SM, but no more blocks to a run than it has rows
    const int64_t runs = most_runs(a->num_rows, p.s.B, p.c.page, a->row_start == nullptr);
    p.q_rows = p.c.page;
    while (p.c.page / p.q_rows < a->num_rows / runs && (p.q_rows > 8 || runs * (p.c.page / p.q_rows) < 2LL * sm_count())) p.q_rows /= 2;
    const int q_blocks = !a->q ? 0 : p.c.page / p.q_rows;
    p.blocks = p.kv_blocks + q_blocks;
    if (runs * p.blocks >= 1LL << 31) return fail(OMMX_E_UNSUPPORTED, "kv4_append: %d rows of %d kv heads in one call", a->num_rows, p.c.H);
    const int bytes = a->dtype == OMMX_DT_F32 ? 4 : 2;
    const bool wide = aligned16(a->k_new, p.k_t, p.k_h, bytes) && aligned16(a->v_new, p.v_t, p.v_h, bytes) &&
                      (!a->q || (aligned16(a->q, p.q_t, p.q_h, bytes) && aligned16(a->q_out, p.o_t, p.o_h, bytes)));
    return launch_dependent(KV4_PICK(kv4_append_kernel, a->dtype, G, wide), dim3((unsigned)(runs * p.blocks)), 32 * WARPS, 0, st, 1, p);
}

static int gather(const ommx_kv4_gather_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv4_gather: null args");
    GatherParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv4_gather", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv4_gather", a->seqs, p.c, &p.s)) return rc;
    if (a->num_rows < 0) return fail(OMMX_E_ARG, "kv4_gather: num_rows must not be negative");
    if (!known_dtype(a->dtype)) return fail(OMMX_E_ARG, "kv4_gather: dtype %d is none of float32, bfloat16, float16", a->dtype);
    if (p.s.B == 0 || a->num_rows == 0) return 0;
    if (!a->k || !a->v) return fail(OMMX_E_ARG, "kv4_gather: k and v must not be null");
    if (!a->row_start && a->num_rows != p.s.B) return fail(OMMX_E_ARG, "kv4_gather: without row_start there is one row for each of the %d sequences, not %d rows", p.s.B, a->num_rows);
    p.rows = {a->row_start, a->num_rows};
    p.k = a->k; p.v = a->v;
    p.k_t = a->k_stride_t; p.k_h = a->k_stride_h; p.v_t = a->v_stride_t; p.v_h = a->v_stride_h;
    p.page_shift = shift_of(p.c.page);
    p.status = a->status;
    const int bytes = a->dtype == OMMX_DT_F32 ? 4 : 2;
    const bool wide = aligned16(a->k, p.k_t, p.k_h, bytes) && aligned16(a->v, p.v_t, p.v_h, bytes);
    const int64_t runs = most_runs(a->num_rows, p.s.B, 16, a->row_start == nullptr);
    // a warp to each head where a wave of blocks takes all (one row of 8 heads: 2.8 us, 3.9 with four warps), four warps where there
    // are several, which then overlap (64K tokens, D = 64: 34.8 us, 37.9 with eight)
    const int warps = runs < 4LL * sm_count() ? GATHER_WARPS : GATHER_WARPS / 2;
    return launch_dependent(KV4_PICK(kv4_gather_kernel, a->dtype, a->cache.head_dim / 32, wide), dim3((unsigned)runs), 32 * (p.c.H < warps ? p.c.H : warps), 0, st, 1, p);
}

}  // namespace kv4
}  // namespace ommx

extern "C" int ommx_b200_kv4_append(const ommx_kv4_append_args *args, void *stream) { return ommx::kv4::append(args, (cudaStream_t)stream); }
extern "C" int ommx_b200_kv4_gather(const ommx_kv4_gather_args *args, void *stream) { return ommx::kv4::gather(args, (cudaStream_t)stream); }
