// The 4-bit cache: appending rows (rotation, quantization, page summaries) and reading rows back.
#include "ommx_kv4.cuh"

namespace ommx {
namespace kv4 {

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
template <typename T, bool WIDE> __device__ __forceinline__ void load8(const T *p, float *x) {
    if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
    } else {
        alignas(16) T v[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(v) / 16; ++i) reinterpret_cast<uint4 *>(v)[i] = reinterpret_cast<const uint4 *>(p)[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
    }
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
    int32_t positions64, num_positions, rot, interleaved, Hq, page_shift, kv_blocks, q_rows;
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

// Rotation of a lane's channels 32 j + 8 t + 0..7 of a key, the four lanes t of a row together. Pairs (c, c + rot / 2) lie in one
// lane for rot >= 64, in lanes t and t ^ 2 for rot = 32; pairs (2 i, 2 i + 1) always in one.
template <int G> __device__ __forceinline__ void rotate_key(const AppendParams &p, float (&x)[G][8], int at, int t) {
    const float *cos = p.cos + at * p.cs_stride, *sin = p.sin + at * p.cs_stride;
    if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < G; ++j)
            if (32 * j < p.rot) {
                float c[4], s[4];
                load_f32<4>(cos + 16 * j + 4 * t, c);
                load_f32<4>(sin + 16 * j + 4 * t, s);
#pragma unroll
                for (int i = 0; i < 4; ++i) turn(x[j][2 * i], x[j][2 * i + 1], c[i], s[i]);
            }
        return;
    }
    if (p.rot == 32) {
        float c[8], s[8];
        load_f32<8>(cos + 8 * (t & 1), c);
        load_f32<8>(sin + 8 * (t & 1), s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float mine = x[0][i], other = __shfl_xor_sync(~0u, mine, 2);
            if (t < 2) turn(mine, other, c[i], s[i]);
            else { turn(other, mine, c[i], s[i]); }
            x[0][i] = mine;
        }
        return;
    }
    // rot = 64: groups 0, 1; rot = 128: groups 0, 2 and 1, 3
#pragma unroll
    for (int j = 0; j < G / 2; ++j)
        if (64 * j < p.rot) {
            float c[8], s[8];
            load_f32<8>(cos + 32 * j + 8 * t, c);
            load_f32<8>(sin + 32 * j + 8 * t, s);
            if (G == 2 || p.rot == 64) {
#pragma unroll
                for (int i = 0; i < 8; ++i) turn(x[0][i], x[1][i], c[i], s[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) turn(x[j][i], x[j + G / 2][i], c[i], s[i]);
            }
        }
}

// Codes and parameters of one group of 32 channels, eight in each of the four lanes of a row: the lane's word of codes, and the
// group's word of parameters. `bad`: x held a value that is not finite.
__device__ __forceinline__ uint32_t quantize_group(float (&x)[8], uint32_t *params, bool *bad) {
    float check = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) check = fmaf(x[i], 0.0f, check);           // NaN as soon as one of them is not finite
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); }
    if (check != 0.0f || hi > LARGEST || lo < -LARGEST) {
        *bad = *bad || check != 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] != x[i] ? 0.0f : fminf(fmaxf(x[i], -LARGEST), LARGEST);
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
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
constexpr uint32_t NOTHING = 0xFF80FF80u;                                  // -inf twice

template <int G> __device__ __forceinline__ void store_words(void *to, const uint32_t (&w)[G]) {
    if constexpr (G == 4) *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
}

// One warp appends up to 16 rows that share a record. Four lanes to a row, eight rows at a time; eight channels of every group to
// a lane, so that key words, parameters and pairs of the rotation need no exchange beyond two shuffles of a group's extremes.
template <typename T, int G, bool WIDE>
__device__ __forceinline__ void append_part(const AppendParams &p, uint8_t *rec, int head, int first_row, int first_pos, int tau0, int n,
                                            int lane, uint32_t (&best)[2 * G * 4]) {
    const int g = lane >> 2, t = lane & 3;
    bool bad = false;
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
        const int tau = 8 * half + g, i = tau - tau0;                       // the lane's token of the record, its row of the n
        if (tau0 + n <= 8 * half || tau0 >= 8 * half + 8) continue;
        bool on = i >= 0 && i < n;
        const int at = on ? rope_row(p, first_row + i, first_pos + i) : 0;
        on = on && at >= 0;
        float x[G][8];
        uint32_t word[G], par[G];
        const T *k = reinterpret_cast<const T *>(p.k) + (int64_t)(first_row + i) * p.k_t + (int64_t)head * p.k_h + 8 * t;
        const T *v = reinterpret_cast<const T *>(p.v) + (int64_t)(first_row + i) * p.v_t + (int64_t)head * p.v_h + 8 * t;
#pragma unroll
        for (int j = 0; j < G; ++j) {
            if (on) load8<T, WIDE>(k + 32 * j, x[j]);
            else for (int e = 0; e < 8; ++e) x[j][e] = 0.0f;
        }
        if (p.rot) {
            rotate_key<G>(p, x, max(at, 0), t);
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = to_f32(from_f32<T>(x[j][e]));   // what a separate rotation would have stored
        }
#pragma unroll
        for (int j = 0; j < G; ++j) word[j] = quantize_group(x[j], &par[j], &bad);
        if (on) {
            store_words<G>(rec + 4 * G * (tau * 4 + t), word);
            if (t == 0) store_words<G>(rec + Rec<G>::KP + 4 * G * tau, par);
            if (p.summary) {
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a = x[j][2 * e], b = x[j][2 * e + 1];
                        uint32_t &hi = best[j * 4 + e], &lo = best[(G + j) * 4 + e];
                        hi = max_bf16x2(hi, ceil_bf16(a) | ceil_bf16(b) << 16);
                        lo = max_bf16x2(lo, (floor_bf16(a) | floor_bf16(b) << 16) ^ 0x80008000u);
                    }
            }
        }
        // values: a word needs two tokens, and a lane's word of eight channels is two half words of four
#pragma unroll
        for (int j = 0; j < G; ++j) {
            if (on) load8<T, WIDE>(v + 32 * j, x[j]);
            else for (int e = 0; e < 8; ++e) x[j][e] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < G; ++j) word[j] = quantize_group(x[j], &par[j], &bad);
        const bool both = __shfl_xor_sync(~0u, (int)on, 4) && on;
        const int pair = g >> 1, odd = g & 1;                               // tokens 8 half + 2 pair + {0, 1}
        uint32_t two[G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
            // the even token's lane makes the words of channel quad 2 t, the odd one's those of 2 t + 1
            const uint32_t other = __shfl_xor_sync(~0u, word[j], 4);
            two[j] = odd ? __byte_perm(other, word[j], 0x7632) : __byte_perm(word[j], other, 0x5410);
        }
        uint8_t *vc = rec + Rec<G>::V;
        if (both) {
            store_words<G>(vc + 4 * G * (32 * half + 4 * (2 * t + odd) + pair), two);
        } else if (on) {
#pragma unroll
            for (int j = 0; j < G; ++j) {
                *reinterpret_cast<uint16_t *>(vc + 4 * (G * (32 * half + 4 * (2 * t) + pair) + j) + 2 * odd) = (uint16_t)word[j];
                *reinterpret_cast<uint16_t *>(vc + 4 * (G * (32 * half + 4 * (2 * t + 1) + pair) + j) + 2 * odd) = (uint16_t)(word[j] >> 16);
            }
        }
        if (on && t == 0) store_words<G>(rec + Rec<G>::VP + 4 * G * tau, par);
    }
    if (bad) or_status(p.status, OMMX_ST_NONFINITE);
}

// Largest over the eight rows of a warp, halving what a lane holds at every step. Lane (g, t) ends with four registers (eight
// channels): of 2 G runs of four, run g for G = 4, run g / 2 for G = 2.
template <int G> __device__ __forceinline__ void reduce_rows(uint32_t (&a)[2 * G * 4], int lane) {
    int n = 2 * G * 4;
#pragma unroll
    for (int d = 16; d >= 4; d /= 2) {
        if (n > 4) {
            n /= 2;
#pragma unroll
            for (int i = 0; i < G * 4; ++i)
                if (i < n) {
                    const bool up = lane & d;
                    const uint32_t give = up ? a[i] : a[i + n], keep = up ? a[i + n] : a[i];
                    a[i] = max_bf16x2(keep, __shfl_xor_sync(~0u, give, d));
                }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = max_bf16x2(a[i], __shfl_xor_sync(~0u, a[i], d));
        }
    }
}

constexpr int WARPS = 4, Q_ROWS = 4;

// Grid: (runs of rows that share a page, kv_blocks + query blocks). The first kv_blocks blocks of a run take its keys and values, a
// warp to 16 tokens of a head (pages over 64 tokens: a warp to several of them); the others rotate the query rows, q_rows each.
template <typename T, int G, bool WIDE>
__global__ void __launch_bounds__(32 * WARPS) kv4_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int D = 32 * G;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    wait_earlier();
    let_next_in();
    Run run;
    if (!find_run(p.s, p.rows, p.page_shift, blockIdx.x, lane, &run, p.status)) return;
    const int page = 1 << p.page_shift;

    if ((int)blockIdx.y >= p.kv_blocks) {                                   // ---- query rows
        int p0 = run.p0, p1 = run.p1;
        if (p.q_rows < page) {
            const int from = (run.p0 & -page) + ((int)blockIdx.y - p.kv_blocks) * p.q_rows;
            p0 = max(p0, from);
            p1 = min(p1, from + p.q_rows);
        }
        const int items = (p1 - p0) * p.Hq * (D / 16);
#pragma unroll 2
        for (int i = threadIdx.x; i < items; i += 32 * WARPS) {
            const int c = i % (D / 16), r = i / (D / 16) / p.Hq, h = i / (D / 16) - r * p.Hq;
            const int row = run.row + p0 - run.p0 + r, at = rope_row(p, row, p0 + r);
            if (at < 0) continue;
            const bool turned = 16 * c < p.rot;
            const int first = turned && !p.interleaved ? 8 * c : 16 * c, second = turned && !p.interleaved ? 8 * c + p.rot / 2 : 16 * c + 8;
            const T *in = reinterpret_cast<const T *>(p.q) + (int64_t)row * p.q_t + (int64_t)h * p.q_h;
            T *out = reinterpret_cast<T *>(p.q_out) + (int64_t)row * p.o_t + (int64_t)h * p.o_h;
            float x[16];
            load8<T, WIDE>(in + first, x);
            load8<T, WIDE>(in + second, x + 8);
            if (turned) {
                float cs[8], sn[8];
                load_f32<8>(p.cos + at * p.cs_stride + 8 * c, cs);
                load_f32<8>(p.sin + at * p.cs_stride + 8 * c, sn);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (p.interleaved) turn(x[2 * e], x[2 * e + 1], cs[e], sn[e]);
                    else turn(x[e], x[8 + e], cs[e], sn[e]);
                }
            }
            store8<T, WIDE>(out + first, x);
            store8<T, WIDE>(out + second, x + 8);
        }
        return;
    }

    // ---- keys and values
    const int warps_a_head = min(p.c.parts, WARPS), heads = WARPS / warps_a_head;
    const int head = blockIdx.y * heads + warp / warps_a_head;
    const int at = run.p0 >> p.page_shift;
    int64_t id = -1;
    if (at < p.s.max_pages) id = page_id(p.s, run.b, at);
    else or_status(p.status, OMMX_ST_BAD_LENGTH);
    if (at < p.s.max_pages && (id < 0 || id >= p.c.num_pages)) { or_status(p.status, OMMX_ST_BAD_PAGE); id = -1; }
    if (id < 0) return;                                                     // the whole block: one run, one page
    uint32_t best[2 * G * 4];
#pragma unroll
    for (int i = 0; i < 2 * G * 4; ++i) best[i] = NOTHING;
    if (head < p.c.H)
        for (int part = warp % warps_a_head; part < p.c.parts; part += warps_a_head) {
            const int base = (run.p0 & -page) + 16 * part, p0 = max(run.p0, base), p1 = min(run.p1, base + 16);
            if (p0 >= p1) continue;
            uint8_t *rec = p.c.records + ((id * p.c.H + head) * p.c.parts + part) * Rec<G>::BYTES;
            append_part<T, G, WIDE>(p, rec, head, run.row + p0 - run.p0, p0, p0 - base, p1 - p0, lane, best);
        }
    if (!p.summary) return;
    reduce_rows<G>(best, lane);
    __shared__ uint4 shared[WARPS][32];
    uint4 own = make_uint4(best[0], best[1], best[2], best[3]);
    if (warps_a_head > 1) {
        shared[warp][lane] = own;
        __syncthreads();
        if (warp % warps_a_head) return;
        for (int w = 1; w < warps_a_head; ++w) {
            const uint4 o = shared[warp + w][lane];
            own = make_uint4(max_bf16x2(own.x, o.x), max_bf16x2(own.y, o.y), max_bf16x2(own.z, o.z), max_bf16x2(own.w, o.w));
        }
    }
    if (head >= p.c.H) return;
    const int g = lane >> 2, t = lane & 3, r = G == 4 ? g : g >> 1;         // r: run of four of 2 G
    if (G == 2 && (g & 1)) return;
    const bool low = r >= G;
    uint4 *to = reinterpret_cast<uint4 *>(p.summary + ((id * p.c.H + head) * 2 + low) * D + 32 * (r % G) + 8 * t);
    const uint32_t sign = low ? 0x80008000u : 0u;
    if (own.x == NOTHING) return;                                           // none of its rows was stored
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

// Grid: runs of rows that share a record of 16 tokens; a warp to a head of it.
template <typename T, int G, bool WIDE>
__global__ void __launch_bounds__(32 * WARPS) kv4_gather_kernel(const __grid_constant__ GatherParams p) {
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
    for (int head = warp; head < p.c.H; head += WARPS) {
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
    if (int rc = read_seqs("kv4_append", a->seqs, &p.s)) return rc;
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
    const int heads = WARPS / (p.c.parts < WARPS ? p.c.parts : WARPS);
    p.kv_blocks = (p.c.H + heads - 1) / heads;
    p.q_rows = a->row_start ? Q_ROWS : p.c.page;
    const int q_blocks = !a->q ? 0 : a->row_start ? p.c.page / Q_ROWS : 1;
    const int64_t runs = most_runs(a->num_rows, p.s.B, p.c.page, a->row_start == nullptr);
    if (p.kv_blocks + q_blocks > 65535) return fail(OMMX_E_UNSUPPORTED, "kv4_append: %d kv heads", p.c.H);
    const int bytes = a->dtype == OMMX_DT_F32 ? 4 : 2;
    const bool wide = aligned16(a->k_new, p.k_t, p.k_h, bytes) && aligned16(a->v_new, p.v_t, p.v_h, bytes) &&
                      (!a->q || (aligned16(a->q, p.q_t, p.q_h, bytes) && aligned16(a->q_out, p.o_t, p.o_h, bytes)));
    return launch_dependent(KV4_PICK(kv4_append_kernel, a->dtype, G, wide), dim3((unsigned)runs, p.kv_blocks + q_blocks), 32 * WARPS, 0, st, p);
}

static int gather(const ommx_kv4_gather_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv4_gather: null args");
    GatherParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv4_gather", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv4_gather", a->seqs, &p.s)) return rc;
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
    return launch_dependent(KV4_PICK(kv4_gather_kernel, a->dtype, a->cache.head_dim / 32, wide), dim3((unsigned)runs), 32 * WARPS, 0, st, p);
}

}  // namespace kv4
}  // namespace ommx

extern "C" int ommx_b200_kv4_append(const ommx_kv4_append_args *args, void *stream) { return ommx::kv4::append(args, (cudaStream_t)stream); }
extern "C" int ommx_b200_kv4_gather(const ommx_kv4_gather_args *args, void *stream) { return ommx::kv4::gather(args, (cudaStream_t)stream); }
