// The 8-bit cache: attention of one query row per sequence, over all tokens or the first ones and a sliding window, with an account of
// each token's weight where it is asked for.
//
// For query head h of a sequence, over its visible tokens t:  x_t = sm_scale q.K_t,  o = sum_t exp(x_t) V_t / sum_t exp(x_t), with
// K_t = 2^ek a_t and V_t = 2^ev b_t for the 16 tokens of a record: a record's scales are two numbers. Products have the codes as A (tokens as rows
// for K, channels for V) and up to eight query heads that share the kv head as columns:
//   logits   int8: 8-bit products (m16n8k32) of the codes as they are and the three bytes of a query row as whole numbers of 23 bits, exact from there
//            on; a channel is rounded by 2^-22 of the row's largest at most. Fp16 products, whose operands have to be made, took 33 us more of 166 (8 x 64K
//            tokens, copies left out). e4m3: fp16 products, since 8-bit ones of this type have their operands converted each time (three pieces of a
//            query: 32 ragged sequences 71 us with fp16, 81 with e4m3); a query row times a power of two is an fp16 number, bf16 channels below 2^-30
//            of the largest and fp16 ones below 2^-27 are rounded by 2^-38 of it at most;
//   values   fp16 (m16n8k16), in which the codes are made exactly; weights times scales, y 2^ev, go to fp16 in a unit that the largest of them sets,
//            a power of two for each head: a token whose weight times scale is 2^-25 of the largest keeps its bits (11), so values of any size
//            leave no token out but those whose weight is below 2^-126 of the heaviest, which fp32 holds as 0. Where the output is finer than bf16 a
//            second product takes what the rounding left (FINE).
// The tensor cores cut what they add to a sum 24 bits below it, so an output is off by 2^-25 of itself for each record of a warp, 2^-18 for 110 of them
// (8 x 64K tokens).
//
// What bounds it: a record's 32 D bytes are read once for each eight query heads of its kv head, and a warp spends 343 instructions on one (D = 128, int8): the
// copies alone take 165 us of 8 x 64K tokens, 8 kv heads, the products alone 133, both 170 to 182 by card (5.9 to 6.3 TB/s, 90 to 97 % of what a copy
// reaches); 32 ragged sequences of 700 to 8191 tokens 57, 57 and 62 to 64. A warp has a ring of its own, so that no barrier stands between a copy and its use: two slots and 16
// warps to an SM (8 x 64K tokens: 183 us; three slots 192, 12 warps and three slots 188, 20 warps 208). Few and short rows are bound by
// the chain of launch, lengths, table, records and join: 6.9 us for one of 333 tokens, of which a launch alone takes 2.5. Many short rows are a block
// each, with that chain in every block: 512 sequences of 100 to 500 tokens are 4096 blocks, 592 at once, 7 turns of 11.4 us (80 us, 49 of them bytes).
#include <cmath>
#include <type_traits>

#include "ommx_kv8.cuh"
#include "ommx_kv8_deal.cuh"
#include "ommx_kv_device.cuh"

namespace ommx {
namespace kv8 {

using namespace kv;

constexpr int WARPS_PER_SM = 16;                  // a block is NW of them, each with records of its own
constexpr int STAGES = 2, AHEAD = STAGES - 1;     // records that a warp holds, and those of them on their way
constexpr uint32_t ALL = 0xFFFFu;                 // sixteen visible tokens
constexpr int COLS = 8;                           // query heads side by side
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LOWEST = -1e30f;
constexpr int MOST_PARTS = 768;                   // blocks of a call that shares rows
constexpr int WHOLE = 32;                         // records of a row that one block takes at most where it could share it

// Weights w = 2^(x - ref) begin near 1; one past HEAVY moves the reference. Products w 2^(ev - 127) k go to fp16: the largest lies in (2^(TOP - 1), 2^TOP]
// when the references have moved, and may grow to ROOM before they move again.
constexpr float HEAVY = 128.0f, ROOM = 60000.0f;
constexpr int TOP = 11;

struct DecodeParams {
    Cache c;
    Seqs s;
    const void *q;
    void *o;
    float *lse, *work;
    float *logits;                                // [row of group heads' units][16][group], or null
    float2 *stats;                                // [B][Hq]: reference and 1 / sum
    const float *before;                          // what weights add to
    int64_t q_b, q_h, o_b, o_h, lse_b;
    int32_t q16, q_wide, o_type, group, col_blocks, page_shift, least, whole, dealt, window, sinks, most_units;
    float scale, cap, keep;                       // scale 2^scale_e: sm_scale in powers of two, or with a cap in its units; 0.5 to 1 in size, times LOG2E
    int32_t scale_e;
    int32_t *status;
};

__device__ __forceinline__ int length_of(const DecodeParams &p, int b) {
    const int len = p.s.len[b];
    const int64_t most = (int64_t)p.s.max_pages << p.page_shift;
    if (len < 0 || len > most) { or_status(p.status, OMMX_ST_BAD_LENGTH); return len < 0 ? 0 : (int)most; }
    return len;
}
// The records of a sequence that hold visible tokens: the first `head`, and those from `head` + `skip` on.
struct Span { int units, head, skip; };
__device__ __forceinline__ Span span_of(const DecodeParams &p, int len) {
    const int all = (len + 15) >> 4;
    Span s = {all, 0, 0};
    if (p.window && len > p.window) {
        const int tail = (len - p.window) >> 4;
        s.head = min((int)(((uint32_t)p.sinks + 15) >> 4), tail);
        s.skip = tail - s.head;
        s.units = all - s.skip;
    }
    return s;
}
__device__ __forceinline__ int units_of(const DecodeParams &p, int len) { return span_of(p, len).units; }
// Which of a record's tokens are visible, a bit each
__device__ __forceinline__ uint32_t visible(const DecodeParams &p, int len, int record) {
    const int first = 16 * record;
    auto below = [](int n) { return n >= 16 ? ALL : n <= 0 ? 0u : (1u << n) - 1; };
    uint32_t mask = below(len - first);
    if (p.window && len > p.window) mask &= ~below(len - p.window - first) | below(p.sinks - first);
    return mask;
}

__device__ __forceinline__ void store_o(const DecodeParams &p, int64_t at, float v) {
    if (p.o_type == OMMX_DT_F32) reinterpret_cast<float *>(p.o)[at] = v;
    else if (p.o_type == OMMX_DT_F16) reinterpret_cast<__half *>(p.o)[at] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16 *>(p.o)[at] = __float2bfloat16_rn(v);
}
template <int G> __device__ __forceinline__ void store_o(const DecodeParams &p, int64_t at, const float (&v)[G]) {
#pragma unroll
    for (int i = 0; i < G; ++i) store_o(p, at + i, v[i]);
}
// A head's reference and sum of weights
__device__ __forceinline__ void store_sum(const DecodeParams &p, int b, int hq, float ref, float sum) {
    p.lse[b * p.lse_b + hq] = sum != 0.0f ? (ref + log2f(sum)) * LN2 : -INFINITY;
    if (p.stats) p.stats[(int64_t)b * p.c.H * p.group + hq] = make_float2(ref, sum != 0.0f ? 1.0f / sum : 0.0f);
}

// ---- pieces ---------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Products of bytes. Sums stay below 2^22, so one that begins with the bits of 1.5 * 2^23 is, as a float, that number and the sum
constexpr float BEGIN_VALUE = 12582912.0f;
__device__ __forceinline__ void mma_s8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
    uint32_t d[4] = {__float_as_uint(c[0]), __float_as_uint(c[1]), __float_as_uint(c[2]), __float_as_uint(c[3])};
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __uint_as_float(d[i]);
}

// The codes of four channels of two tokens (their words) to fp16 pairs, a channel to each
template <bool E4M3> __device__ __forceinline__ void value_pairs(uint32_t a, uint32_t b, uint32_t (&pair)[4]) {
    const uint32_t two[2] = {__byte_perm(a, b, 0x5140), __byte_perm(a, b, 0x7362)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (E4M3) {
            pair[2 * i] = half2_of_e4m3x2(two[i]);
            pair[2 * i + 1] = half2_of_e4m3x2(two[i] >> 16);
        } else {
            const uint32_t u = two[i] ^ 0x80808080u;                        // 1024 + 128 + code as an fp16 number
            const __half2 off = __float2half2_rn(1152.0f);
            const uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
            const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&lo), off), y = __hsub2(*reinterpret_cast<const __half2 *>(&hi), off);
            pair[2 * i] = *reinterpret_cast<const uint32_t *>(&x);
            pair[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&y);
        }
    }
}

// A kv head's queries as B fragments: lane (g, t) holds head g, channels 8 G t + 8 s + 0..7 for the products s. int8: [s][byte][half of the eight];
// e4m3: [s][half of the eight][two pairs]
constexpr int PIECES = 3;
template <int G, bool E4M3> struct Query {
    uint32_t frag[G][E4M3 ? 2 : PIECES][2];
    float factor[2];                              // of heads 2 t and 2 t + 1: the products' units, in powers of two or with a cap in its units,
    int exponent[2];                              // without the powers of two of `exponent` where they are `apart`
    bool apart;                                   // a factor times a scale may leave fp32's range
};
// The lane's channels as they are, on their way while records are looked up
template <int G> struct Raw { uint4 v[G]; };
template <int G> __device__ __forceinline__ void fetch_query(const DecodeParams &p, int b, int first_head, int n, int lane, Raw<G> &raw) {
    const uint16_t *from = reinterpret_cast<const uint16_t *>(p.q) + b * p.q_b + (first_head + min(lane >> 2, n - 1)) * p.q_h + 8 * G * (lane & 3);
#pragma unroll
    for (int i = 0; i < G; ++i) {
        if (p.q_wide) {
            raw.v[i] = reinterpret_cast<const uint4 *>(from)[i];
        } else {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = from[8 * i + 2 * j] | (uint32_t)from[8 * i + 2 * j + 1] << 16;
            raw.v[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}
template <int G, bool E4M3> __device__ __forceinline__ void make_query(const DecodeParams &p, const Raw<G> &raw, int lane, Query<G, E4M3> &q) {
    const int t = lane & 3;
    float x[8 * G];
    uint32_t largest = 0;                         // magnitudes in the order of their bits, two at a time
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const uint32_t w[4] = {raw.v[i].x, raw.v[i].y, raw.v[i].z, raw.v[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = p.q16 ? __half22float2(*reinterpret_cast<const __half2 *>(&w[j])) : make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
            x[8 * i + 2 * j] = f.x;
            x[8 * i + 2 * j + 1] = f.y;
            largest = __vmaxu2(largest, w[j] & 0x7FFF7FFFu);
        }
    }
    largest = max(largest & 0xFFFFu, largest >> 16);
    largest = max(largest, __shfl_xor_sync(~0u, largest, 1));
    largest = max(largest, __shfl_xor_sync(~0u, largest, 2));
    float top = p.q16 ? __half2float(__ushort_as_half((uint16_t)largest)) : __uint_as_float(largest << 16);
    const bool wild = !(top < INFINITY);          // whole numbers hold neither NaN nor infinities: the head's logits are NaN then
    constexpr int BITS = E4M3 ? 13 : 21;          // the largest channel lies below 2^(BITS + 1)
    constexpr float SMALL = 0x1p-100f;            // rows below it, subnormal ones among them, are raised first: 2^BITS over them is no fp32 number
    constexpr int RAISE = 64;
    const bool small = top > 0.0f && top < SMALL;
    if (__any_sync(~0u, small)) {
        const float by = small ? power_of_two(RAISE) : 1.0f;
        top *= by;
#pragma unroll
        for (int i = 0; i < 8 * G; ++i) x[i] *= by;
    }
    const int e = top > 0.0f ? exponent_of(top) : 0;
    const float up = power_of_two(BITS - e);
#pragma unroll
    for (int s = 0; s < G; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float *f = x + 8 * s + 4 * h;
            if constexpr (E4M3) {
                q.frag[s][h][0] = half2_bits(f[0] * up, f[1] * up);
                q.frag[s][h][1] = half2_bits(f[2] * up, f[3] * up);
            } else {
                // a whole number and 128 in each of three bytes: what is over in a byte is a digit of -128 .. 127
                uint32_t r[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(fmaf(f[i], up, BEGIN_VALUE)) - __float_as_uint(BEGIN_VALUE) + 0x808080u;
#pragma unroll
                for (int j = 0; j < PIECES; ++j) {
                    const uint32_t byte = PIECES - 1 - j, pick = byte | (byte + 4) << 4;
                    q.frag[s][j][h] = __byte_perm(__byte_perm(r[0], r[1], pick), __byte_perm(r[2], r[3], pick), 0x5410) ^ 0x80808080u;
                }
            }
        }
    // A factor of 2^-100 to 1 keeps its bits beside every scale, or the logit is nothing, and stays finite
    const int exponent = p.scale_e + e - BITS - (small ? RAISE : 0);
    q.apart = __any_sync(~0u, exponent > 0 || exponent < -100);
    const float factor = wild ? NAN : q.apart ? p.scale : p.scale * power_of_two(exponent);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        q.factor[i] = __shfl_sync(~0u, factor, 8 * t + 4 * i);
        q.exponent[i] = __shfl_sync(~0u, exponent, 8 * t + 4 * i);
    }
}

// A warp's running state. acc[i]: channels 4 G g + 2 i (rows g) and the next one (rows g + 8) of heads 2 t, 2 t + 1, in units of unit[]
template <int G> struct State {
    float acc[2 * G][4], sum[2], ref[2];
    float unit[2];                                // a power of two that only `acc` has in it
};
template <int G> __device__ __forceinline__ void clear(State<G> &s) {
#pragma unroll
    for (int i = 0; i < 2 * G; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s.acc[i][j] = 0.0f;
    s.sum[0] = s.sum[1] = 0.0f;
    s.ref[0] = s.ref[1] = LOWEST;
    s.unit[0] = s.unit[1] = 1.0f;
}
// The references of head i move to `ref`, a whole number as the one before, so that nothing is rounded. E: exponent of a record's scale, `top`: its
// largest logit less `ref`.
template <int G> __device__ __forceinline__ void move(State<G> &s, int i, float ref, float top, int E) {
    const int was = exponent_of(s.unit[i]);
    const float over = ceilf(fmaxf((s.ref[i] - ref) + (float)(TOP - was), top + (float)(E - 127)));       // 2^over: the largest product
    const int now = min(TOP - (int)fminf(fmaxf(over, -1000.0f), 1000.0f), 253 - E);                       // a scale times the unit is finite
    const int held = min(max(now, -126), 126);
    const float f = exp2_approx(s.ref[i] - ref), a = exp2_approx(s.ref[i] - ref + (float)(held - was));
    s.ref[i] = ref;
    s.unit[i] = power_of_two(held);
    s.sum[i] *= f;
#pragma unroll
    for (int j = 0; j < 2 * G; ++j) { s.acc[j][i] *= a; s.acc[j][i + 2] *= a; }
}

// ---- a warp's ring of records: 16 bytes a lane at a time, a group of copies for each record ----
// In shared memory a record's 128-byte lines have their 16-byte chunks exchanged, chunk c of line l at c ^ (l & 7) (D = 128) or
// c ^ (2 l & 6) (two tokens to a line, D = 64), so that both ways of reading - a token's row by four lanes, and a chunk of
// eight tokens - meet all banks.
template <int G> __device__ __forceinline__ uint32_t swizzle(int token, int chunk) {
    if constexpr (G == 4) return 128 * token + 16 * (chunk ^ (token & 7));
    else return 128 * (token >> 1) + 16 * ((4 * (token & 1) + chunk) ^ (token & 6));
}
template <int G> __device__ __forceinline__ void fetch(uint32_t to, const uint8_t *rec, int lane) {
    // 512 bytes are four lines; every other four the same exchange
    const int line = lane >> 3, chunk = lane & 7;
    const uint32_t even = 128 * line + 16 * (G == 4 ? chunk ^ line : chunk ^ (2 * line)), odd = G == 4 ? even ^ 64 : even;
#pragma unroll
    for (int i = 0; i < 2 * G; ++i)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 512 * i + (i & 1 ? odd : even)), "l"(rec + 512 * i + 16 * lane) : "memory");
}
__device__ __forceinline__ void close_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void fetched() {                // all but the last N groups
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    __syncwarp();
}

// One record in shared memory; info: which tokens are visible, and above that the exponents of K's and V's scales. `put`: where its logits
// go, or null
template <int G, bool E4M3, bool FINE> __device__ __forceinline__ void attend(const DecodeParams &p, const uint8_t *rec, uint32_t info, int lane, const Query<G, E4M3> &q, State<G> &s,
                                                                   float *put, int n) {
    constexpr int D = 32 * G;
    const int g = lane >> 2, t = lane & 3;
    // ---- logits: x[0], x[1] of token g and heads 2 t, 2 t + 1; x[2], x[3] of token g + 8
    constexpr int SUMS = E4M3 ? 2 : PIECES;       // of half the products each; of a byte each
    float c[SUMS][4], x[4];
#pragma unroll
    for (int j = 0; j < SUMS; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[j][i] = E4M3 ? 0.0f : BEGIN_VALUE;
#pragma unroll
    for (int i = 0; i < G / 2; ++i) {
        const uint4 a = *reinterpret_cast<const uint4 *>(rec + swizzle<G>(g, G / 2 * t + i));
        const uint4 b = *reinterpret_cast<const uint4 *>(rec + swizzle<G>(g + 8, G / 2 * t + i));
        if constexpr (E4M3) {
            const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t k[4] = {half2_of_e4m3x2(wa[j]), half2_of_e4m3x2(wb[j]), half2_of_e4m3x2(wa[j] >> 16), half2_of_e4m3x2(wb[j] >> 16)};
                mma_f16(c[j & 1], k, q.frag[2 * i + j / 2][j & 1][0], q.frag[2 * i + j / 2][j & 1][1]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) mma_s8(c[j], a.x, b.x, a.y, b.y, q.frag[2 * i][j]);
#pragma unroll
            for (int j = 0; j < PIECES; ++j) mma_s8(c[j], a.z, b.z, a.w, b.w, q.frag[2 * i + 1][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (E4M3) x[i] = c[0][i] + c[1][i];
        else x[i] = fmaf(fmaf(c[0][i] - BEGIN_VALUE, 256.0f, c[1][i] - BEGIN_VALUE), 256.0f, c[SUMS - 1][i] - BEGIN_VALUE);
    }
    const int EK = info >> 16 & 255u;
    float unit[2] = {q.factor[0] * scale_of(EK), q.factor[1] * scale_of(EK)};
    if (q.apart) {                                // |factor| <= LOG2E: finite; a sum of 0 stays 0, and one below 2^36 times 2^-126 is nothing
#pragma unroll
        for (int i = 0; i < 2; ++i) unit[i] = q.factor[i] * scale_of(EK ? min(max(EK + q.exponent[i], 1), 254) : 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= unit[i & 1];
    if (p.cap > 0.0f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = tanhf(x[i]) * (p.cap * LOG2E);
    }
    if (put) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            float *to = put + (g + 4 * i) * p.group + 2 * t;
            const float2 two = make_float2(fmaxf(x[i], LOWEST), fmaxf(x[i + 1], LOWEST));    // the account has no NaN
            if (p.group % 2 == 0 && 2 * t < n) *reinterpret_cast<float2 *>(to) = two;
            else if (2 * t < n) {
                to[0] = two.x;
                if (2 * t + 1 < n) to[1] = two.y;
            }
        }
    }
    const uint32_t mask = info & ALL;
    if (mask != ALL) {                            // what is not visible may be anything
        if (!(mask >> g & 1)) x[0] = x[1] = -INFINITY;
        if (!(mask >> (g + 8) & 1)) x[2] = x[3] = -INFINITY;
    }

    // ---- weights
    const int E = info >> 24;
    float y[4], f[2], z[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) f[i] = scale_of(E) * s.unit[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) { y[i] = exp2_approx(x[i] - s.ref[i & 1]); z[i] = y[i] * f[i & 1]; }
    // A unit held at its largest while values were zero or tiny may meet a scale with which it is infinite; a weight of 0 then makes a NaN, which
    // counts as too large: a unit that has moved is finite with the record's scale.
    const float heavy = fmaxf(max3(y[0], y[1], y[2]), y[3]), most = max3_nan(max3_nan(z[0], z[1], z[2]), z[3], z[3]);
    if (__any_sync(~0u, !(heavy <= HEAVY && most <= ROOM))) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float l = fmaxf(x[i], x[i + 2]);
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l = fmaxf(l, __shfl_xor_sync(~0u, l, d));
            const float ref = fmaxf(s.ref[i], ceilf(l));
            move(s, i, ref, l - ref, E);
            f[i] = scale_of(E) * s.unit[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) { y[i] = exp2_approx(x[i] - s.ref[i & 1]); z[i] = y[i] * f[i & 1]; }
    }
    s.sum[0] += y[0] + y[2];
    s.sum[1] += y[1] + y[3];
    const uint32_t h0 = half2_bits(z[0], z[1]), h1 = half2_bits(z[2], z[3]);
    const uint32_t b0 = transpose8x8(h0), b1 = transpose8x8(h1);
    uint32_t r0 = 0, r1 = 0;
    if constexpr (FINE) {
        const float2 n0 = __half22float2(*reinterpret_cast<const __half2 *>(&h0)), n1 = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
        r0 = transpose8x8(half2_bits(z[0] - n0.x, z[1] - n0.y));
        r1 = transpose8x8(half2_bits(z[2] - n1.x, z[3] - n1.y));
    }

    // ---- values
    uint32_t w[4][G];                             // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9: channels 4 G g + 0 .. 4 G - 1
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int token = 2 * t + (i & 1) + 4 * (i & 2);
        if constexpr (G == 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(rec + 16 * D + swizzle<G>(token, g));
            w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(rec + 16 * D + swizzle<G>(token, g >> 1) + 8 * (g & 1));
            w[i][0] = v.x; w[i][1] = v.y;
        }
        if (E4M3 && mask != ALL && !(mask >> token & 1)) {                  // a weight of 0 times NaN is not 0
#pragma unroll
            for (int j = 0; j < G; ++j) w[i][j] = 0;
        }
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
        uint32_t near[4], far[4];                 // of tokens 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
        value_pairs<E4M3>(w[0][j], w[1][j], near);
        value_pairs<E4M3>(w[2][j], w[3][j], far);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t a[4] = {near[2 * u], near[2 * u + 1], far[2 * u], far[2 * u + 1]};
            if constexpr (FINE) mma_f16(s.acc[2 * j + u], a, r0, r1);
            mma_f16(s.acc[2 * j + u], a, b0, b1);
        }
    }
}

template <int G> constexpr int PART = COLS * 32 * G + 2 * COLS;            // floats of a part in the workspace: outputs, references, sums
template <int G, int NW> struct Shared {
    static constexpr int D = 32 * G;
    float o[NW][COLS][D + 4];                     // the padding spreads the heads over the banks
};
template <int G> struct Floats;
template <> struct Floats<2> { using T = float2; };
template <> struct Floats<4> { using T = float4; };

// The warps' states of a row to its output, or to a part: [COLS][D] outputs of its own tokens, [COLS] references, [COLS] sums. A warp
// finishes every NW-th head, a lane G channels.
template <int G, int NW>
__device__ __forceinline__ void finish(const DecodeParams &p, State<G> &s, Shared<G, NW> &sh, float (&ref)[COLS][NW], float (&sum)[COLS][NW], int b,
                                       int first_head, int n, float *part, int warp, int lane) {
    using V = typename Floats<G>::T;
    constexpr int D = 32 * G;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) s.sum[i] += __shfl_xor_sync(~0u, s.sum[i], d);
        if (g == 0) { ref[2 * t + i][warp] = s.ref[i]; sum[2 * t + i][warp] = s.sum[i]; }
    }
    __syncthreads();                              // and the ring, whose memory `sh` is, is done with
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float back = s.sum[i] != 0.0f ? 1.0f / s.sum[i] : 0.0f, unit = power_of_two(-exponent_of(s.unit[i]));
        float *to = &sh.o[warp][2 * t + i][4 * G * g];
#pragma unroll
        for (int j = 0; j < 2 * G; j += 2)
            *reinterpret_cast<float4 *>(to + 2 * j) = make_float4(s.acc[j][i] * back * unit, s.acc[j][i + 2] * back * unit,
                                                                  s.acc[j + 1][i] * back * unit, s.acc[j + 1][i + 2] * back * unit);
    }
    __syncthreads();
    for (int h = warp; h < COLS; h += NW) {
        float top = ref[h][0], all = 0.0f;
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, ref[h][w]);
#pragma unroll
        for (int w = 0; w < NW; ++w) all = fmaf(sum[h][w], exp2_approx(ref[h][w] - top), all);
        const float inverse = all != 0.0f ? 1.0f / all : 0.0f;
        float v[G];
#pragma unroll
        for (int i = 0; i < G; ++i) v[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const V x = *reinterpret_cast<const V *>(&sh.o[w][h][lane * G]);
            const float f = sum[h][w] * exp2_approx(ref[h][w] - top) * inverse;
#pragma unroll
            for (int i = 0; i < G; ++i) v[i] = fmaf(reinterpret_cast<const float *>(&x)[i], f, v[i]);
        }
        if (part) {
            *reinterpret_cast<V *>(part + h * D + lane * G) = *reinterpret_cast<const V *>(v);
            if (lane == 0) { part[COLS * D + h] = top; part[COLS * D + COLS + h] = all; }
        } else if (h < n) {
            store_o(p, b * p.o_b + (first_head + h) * p.o_h + lane * G, v);
            if (lane == 0) store_sum(p, b, first_head + h, top, all);
        }
    }
    __syncthreads();
}

template <int G, int NW> struct Memory {
    union {
        Shared<G, NW> sh;
        uint8_t ring[NW][STAGES][1024 * G];
    };
    alignas(16) float merged[PART<G>];            // of this block, where a cluster shares a row
    float ref[COLS][NW], sum[COLS][NW];
    uint32_t fits[NW];                            // of the deal
};

__device__ __forceinline__ bool too_many(const DecodeParams &p, uint32_t units, uint32_t rows) {
    const bool over = (uint64_t)units * rows >> 31;
    if (over) or_status(p.status, OMMX_ST_BAD_LENGTH);
    return over;
}
// A row of no tokens
template <int G> __device__ __forceinline__ void nothing(const DecodeParams &p, int b, int row) {
    const int cb = row % p.col_blocks, first = (row / p.col_blocks) * p.group + cb * COLS, n = min(COLS, p.group - cb * COLS);
    for (int i = threadIdx.x; i < n * 32 * G; i += blockDim.x) store_o(p, b * p.o_b + (first + i / (32 * G)) * p.o_h + i % (32 * G), 0.0f);
    if (threadIdx.x < n) store_sum(p, b, first + threadIdx.x, LOWEST, 0.0f);
}

// ---- a row shared by a cluster's blocks: their parts meet in distributed shared memory ----
// Head h is finished by block h mod n of the cluster, by its warp h.
constexpr int MOST_CLUSTER = 8;
template <int G> __device__ __forceinline__ void merge_cluster(const DecodeParams &p, const float *merged, int b, int first_head, int heads, int h, int lane) {
    constexpr int D = 32 * G, LANES = D / 4;      // lanes that have four channels
    const uint32_t n = cluster_size(), at = (uint32_t)__cvta_generic_to_shared(merged);
    cluster_barrier();
    if (h < heads && h % n == cluster_rank()) {
        float4 v[MOST_CLUSTER];
        float ref[MOST_CLUSTER], sum[MOST_CLUSTER];
#pragma unroll
        for (int r = 0; r < MOST_CLUSTER; ++r) {
            const uint32_t from = r < (int)n ? r : 0;
            v[r] = peer_float4(at + 4 * (h * D + 4 * (lane % LANES)), from);
            ref[r] = r < (int)n ? peer_float(at + 4 * (COLS * D + h), from) : LOWEST;
            sum[r] = r < (int)n ? peer_float(at + 4 * (COLS * D + COLS + h), from) : 0.0f;
        }
        float top = ref[0], all = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 1; r < MOST_CLUSTER; ++r) top = fmaxf(top, ref[r]);
#pragma unroll
        for (int r = 0; r < MOST_CLUSTER; ++r) { sum[r] *= exp2_approx(ref[r] - top); all += sum[r]; }
        const float inverse = all != 0.0f ? 1.0f / all : 0.0f;
#pragma unroll
        for (int r = 0; r < MOST_CLUSTER; ++r) {
            const float f = sum[r] * inverse;
            o[0] = fmaf(v[r].x, f, o[0]); o[1] = fmaf(v[r].y, f, o[1]); o[2] = fmaf(v[r].z, f, o[2]); o[3] = fmaf(v[r].w, f, o[3]);
        }
        if (lane < LANES) store_o(p, b * p.o_b + (first_head + h) * p.o_h + 4 * lane, o);
        if (lane == 0) store_sum(p, b, first_head + h, top, all);
    }
    cluster_barrier();                            // no block leaves before its peers have read its part
}

template <int G, bool E4M3, bool FINE, int NW, bool CLUSTER>
__global__ void __launch_bounds__(32 * NW, WARPS_PER_SM / NW) kv8_decode_kernel(const __grid_constant__ DecodeParams p) {
    extern __shared__ __align__(128) uint8_t memory[];
    Memory<G, NW> &m = *reinterpret_cast<Memory<G, NW> *>(memory);
    constexpr int BYTES = 1024 * G;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint8_t *ring = m.ring[warp][0];
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    wait_earlier();
    let_next_in();
    const uint32_t rows = p.c.H * p.col_blocks;
    uint32_t u, end, base = 0;                    // this block's units; units before sequence b
    uint32_t second = ~0u;                        // a row that begins here or later leaves its part in the second slot
    int b = 0, len = 0;
    Span span = {0, 0, 0};
    if (CLUSTER) {                                // a cluster to a row
        const uint32_t n = cluster_size(), rank = cluster_rank(), at = blockIdx.x / n;
        b = at / rows;
        len = length_of(p, b);
        span = span_of(p, len);
        if (too_many(p, span.units, rows)) span.units = 0;
        if (span.units == 0) {                    // for all of the cluster
            if (rank == 0) nothing<G>(p, b, at - b * rows);
            return;
        }
        u = (at - b * rows) * span.units;
        end = u + (uint64_t)span.units * (rank + 1) / n;
        u += (uint64_t)span.units * rank / n;
    } else if (p.whole) {                         // a block to a row
        b = blockIdx.x / rows;
        len = length_of(p, b);
        span = span_of(p, len);
        if (too_many(p, span.units, rows)) span.units = 0;
        u = (blockIdx.x - b * rows) * span.units;
        end = u + span.units;
        if (span.units == 0) { nothing<G>(p, b, blockIdx.x - b * rows); return; }
    } else {
        const Lengths own = lengths_of(p, lane);
        const Deal d = deal(p, own, rows, gridDim.x, lane, warp, NW, m.fits);
        if (blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<uint2 *>(p.work) = make_uint2(d.per, d.over ? OVER : d.pieces);
        // the sequence that this block's (first) unit lies in; `at`, `before`: this block and the first of the sequence, in pieces or units
        const uint32_t at = d.pieces ? blockIdx.x : blockIdx.x * d.per;
        if (!d.pieces && at >= d.total) return;
        uint32_t before = 0;
        for (int b0 = 0;; b0 += 32) {
            if (b0 >= p.s.B) return;              // no piece for this block (or lengths past max_seq_len, more than 32 bits count)
            int l;
            uint32_t n;
            if (b0 < 64) {
                l = b0 ? own.len[1] : own.len[0];
                n = b0 ? own.units[1] : own.units[0];
            } else {
                l = b0 + lane < p.s.B ? length_of(p, b0 + lane) : 0;
                n = units_of(p, l);
            }
            const uint32_t v = d.pieces ? pieces_of(n, d.per) : n, sum = warp_inclusive_scan(v, lane), past = __ballot_sync(~0u, before + sum * rows > at);
            if (past) {
                const int from = __ffs(past) - 1;
                b = b0 + from;
                before += __shfl_sync(~0u, sum - v, from) * rows;
                len = __shfl_sync(~0u, l, from);
                span = span_of(p, len);
                break;
            }
            before += __shfl_sync(~0u, sum, 31) * rows;
        }
        const uint32_t units = span.units;
        if (d.pieces) {                           // piece `part` of `parts` of a row; units are counted from the sequence's first
            const uint32_t parts = pieces_of(units, d.per), row = (at - before) / parts, part = at - before - row * parts;
            const uint32_t each = units / parts, more = units - each * parts;    // the first `more` have one more
            u = row * units + part * each + min(part, more);
            end = u + each + (part < more);
        } else {
            base = before;
            second = u = at;
            end = min(u + d.per, d.total);
        }
    }
    while (CLUSTER || u < end) {
        while (u >= base + span.units * rows) {   // the next sequence that has any
            base += span.units * rows;
            len = length_of(p, ++b);
            span = span_of(p, len);
        }
        const int units = span.units, row = (u - base) / units, i0 = u - base - row * units, i1 = min((uint32_t)units, i0 + (end - u));
        const int head = p.col_blocks == 1 ? row : row / p.col_blocks, cb = row - head * p.col_blocks;
        const int first_head = head * p.group + cb * COLS, n = min(COLS, p.group - cb * COLS);
        // 32 of the warp's records at a time are looked up by a lane each, while the 32 before are on their way: which one it is, which of
        // its tokens are visible (none: there is no record) and its scales.
        const int mine = (i1 - i0 - warp + NW - 1) / NW;
        auto place_of = [&](int k) { const int i = i0 + warp + (k + lane) * NW; return i < span.head ? i : i + span.skip; };
        auto page_at = [&](int k) -> int64_t {    // -1: none
            return i0 + warp + (k + lane) * NW < i1 ? page_id(p.s, b, place_of(k) >> (p.page_shift - 4)) : -1;
        };
        auto record_at = [&](int k, int64_t page) -> uint32_t {             // one that is not meant is fetched too, and not used
            if (page >= p.c.num_pages || (page < 0 && i0 + warp + (k + lane) * NW < i1)) or_status(p.status, OMMX_ST_BAD_PAGE);
            const bool on = page >= 0 && page < p.c.num_pages;
            return on ? (uint32_t)((page * p.c.H + head) * p.c.parts + (place_of(k) & (p.c.parts - 1))) : 0u;     // below 2^32: there is no memory for more
        };
        auto info_at = [&](int k, int64_t page, uint32_t rec) -> uint32_t {
            return page >= 0 && page < p.c.num_pages ? visible(p, len, place_of(k)) | (uint32_t)reinterpret_cast<const uint16_t *>(p.c.scales)[rec] << 16 : 0u;
        };
        // `rec`, `info`: of the AHEAD first ones, then of 32 at a time, AHEAD of those in use
        uint32_t rec, next_rec, info, next_info, flying[AHEAD];             // flying: of those on their way
        Raw<G> raw;
        {
            const int64_t page = page_at(0), next = page_at(AHEAD);
            fetch_query(p, b, first_head, n, lane, raw);
            rec = record_at(0, page);
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                if (k < mine) fetch<G>(ring_at + k * BYTES, p.c.codes + (uint64_t)__shfl_sync(~0u, rec, k) * BYTES, lane);
                close_group();
            }
            info = info_at(0, page, rec);
            next_rec = record_at(AHEAD, next);
            next_info = info_at(AHEAD, next, next_rec);
        }
        Query<G, E4M3> q;
        State<G> s;
        make_query<G, E4M3>(p, raw, lane, q);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) flying[k] = __shfl_sync(~0u, info, k);
        clear(s);
        float *put = nullptr;
        if (p.logits) put = p.logits + (((int64_t)b * p.c.H + head) * p.most_units * 16) * p.group + cb * COLS;
        // the slot in use and the one that is filled next, which is the one used before
        int read = 0, write = AHEAD * BYTES;
        for (int k0 = 0; k0 < mine; k0 += 32) {
            rec = next_rec;
            info = next_info;
            {
                const int64_t page = page_at(k0 + 32 + AHEAD);
                next_rec = record_at(k0 + 32 + AHEAD, page);
                next_info = info_at(k0 + 32 + AHEAD, page, next_rec);
            }
            const int left = mine - k0, now = min(32, left);
            for (int k = 0; k < now; ++k) {
                if (k + AHEAD < left) fetch<G>(ring_at + write, p.c.codes + (uint64_t)__shfl_sync(~0u, rec, k) * BYTES, lane);
                close_group();
                fetched<AHEAD>();
                if (flying[0] & ALL) {
                    float *to = nullptr;
                    if (put) {
                        const int i = i0 + warp + (k0 + k) * NW;
                        if (i < p.most_units) to = put + (int64_t)i * 16 * p.group;
                        else or_status(p.status, OMMX_ST_BAD_LENGTH);
                    }
                    attend<G, E4M3, FINE>(p, ring + read, flying[0], lane, q, s, to, n);
                }
#pragma unroll
                for (int j = 0; j + 1 < AHEAD; ++j) flying[j] = flying[j + 1];
                flying[AHEAD - 1] = __shfl_sync(~0u, info, k);
                write = read;
                read = read == AHEAD * BYTES ? 0 : read + BYTES;
                __syncwarp();                     // before the slot is filled again
            }
        }
        fetched<0>();
        if constexpr (CLUSTER) {
            finish<G, NW>(p, s, m.sh, m.ref, m.sum, b, first_head, n, m.merged, warp, lane);
            merge_cluster<G>(p, m.merged, b, first_head, n, warp, lane);
            return;
        }
        float *part = nullptr;
        if (i0 > 0 || i1 < units) part = p.work + HEAD + (2 * (int64_t)blockIdx.x + (base + row * units >= second)) * PART<G>;
        finish<G, NW>(p, s, m.sh, m.ref, m.sum, b, first_head, n, part, warp, lane);
        u += i1 - i0;
    }
}

// ---- parts ----------------------------------------------------------------------------------------
template <int G> __device__ __forceinline__ const float *part_at(const DecodeParams &p, const Parts &r, int i) {
    return p.work + HEAD + (2 * (int64_t)(r.first + i) + (i == 0 && r.late)) * PART<G>;
}
// Reference and sum of a head over the parts that `threads` threads of this one's kind look at, met in a warp
template <int G> __device__ __forceinline__ void meet(const DecodeParams &p, const Parts &r, int h, int from, int threads, float &top, float &sum) {
    constexpr int D = 32 * G;
    top = LOWEST;
    sum = 0.0f;
    for (int i = from; i < (int)r.count; i += threads) {
        const float *part = part_at<G>(p, r, i);
        const float ref = part[COLS * D + h], s = part[COLS * D + COLS + h], m = fmaxf(top, ref);
        sum = fmaf(s, exp2_approx(ref - m), sum * exp2_approx(top - m));
        top = m;
    }
#pragma unroll
    for (int d = 16; d; d /= 2) {
        const float ref = __shfl_xor_sync(~0u, top, d), s = __shfl_xor_sync(~0u, sum, d), m = fmaxf(top, ref);
        sum = fmaf(s, exp2_approx(ref - m), sum * exp2_approx(top - m));
        top = m;
    }
}
template <int G> __device__ __forceinline__ void zeros(const DecodeParams &p, int b, int hq, int lane) {      // a head of no tokens
#pragma unroll
    for (int i = 0; i < G; ++i) store_o(p, b * p.o_b + hq * p.o_h + lane * G + i, 0.0f);
    if (lane == 0) store_sum(p, b, hq, LOWEST, 0.0f);
}

// Rows of which several blocks have a part, and those of no tokens, where rows are many: a block to a row, a warp to a head, a lane
// to G channels. `at`: the row of the sequence.
template <int G> __device__ __forceinline__ void combine_row(const DecodeParams &p, int b, int row) {
    using V = typename Floats<G>::T;
    constexpr int D = 32 * G;
    const int lane = threadIdx.x & 31, h = threadIdx.x >> 5;
    const int head = row / p.col_blocks, cb = row % p.col_blocks, hq = head * p.group + cb * COLS + h;
    const Parts r = parts_of(p, b, row, lane);
    let_next_in();
    if (h >= p.group - cb * COLS || r.count == 1) return;                   // not a head, or finished where it was computed
    if (r.count == 0) { zeros<G>(p, b, hq, lane); return; }
    float top, sum, o[G];
    constexpr int EACH = 4;                       // parts on their way, the first ones while the references meet
    V v[EACH];
    float ref[EACH], add[EACH];
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const bool on = i0 + u < (int)r.count;
            const float *part = part_at<G>(p, r, on ? i0 + u : i0);
            v[u] = reinterpret_cast<const V *>(part + h * D)[lane];
            ref[u] = part[COLS * D + h];
            add[u] = on ? part[COLS * D + COLS + h] : 0.0f;
        }
    };
    load(0);
    meet<G>(p, r, h, lane, 32, top, sum);
    const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < G; ++i) o[i] = 0.0f;
    for (int i0 = 0; i0 < (int)r.count; i0 += EACH) {
        if (i0) load(i0);
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const float f = add[u] * exp2_approx(ref[u] - top) * inverse;
#pragma unroll
            for (int i = 0; i < G; ++i) o[i] = fmaf(reinterpret_cast<const float *>(&v[u])[i], f, o[i]);
        }
    }
    store_o(p, b * p.o_b + hq * p.o_h + lane * G, o);
    if (lane == 0) store_sum(p, b, hq, top, sum);
}

// The same where rows are few and their parts many: a block to a head. The references and sums of all parts are read at once; then a
// warp takes every CW-th part, UNROLL of them on their way.
constexpr int CW = 8, UNROLL = 5;
template <int G> __device__ __forceinline__ void combine_head(const DecodeParams &p, int b, int row, int h) {
    constexpr int D = 32 * G;
    using V = typename Floats<G>::T;
    __shared__ float so[CW][D], weight[MOST_PARTS], sr[CW], ss[CW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = row / p.col_blocks, cb = row % p.col_blocks, hq = head * p.group + cb * COLS + h;
    const Parts r = parts_of(p, b, row, lane);
    let_next_in();
    const int n = r.count;
    if (h >= p.group - cb * COLS || n == 1) return;                         // not a head, or finished where it was computed
    if (n == 0) {
        if (warp == 0) zeros<G>(p, b, hq, lane);
        return;
    }
    V v[UNROLL];
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (i0 + u * CW < n) v[u] = reinterpret_cast<const V *>(part_at<G>(p, r, i0 + u * CW) + h * D)[lane];
    };
    load(warp);                                   // on their way while the references meet
    float top = LOWEST, sum = 0.0f;
    for (int i = threadIdx.x; i < n; i += 32 * CW) {
        const float *part = part_at<G>(p, r, i);
        weight[i] = part[COLS * D + h];
    }
    meet<G>(p, r, h, threadIdx.x, 32 * CW, top, sum);
    if (lane == 0) { sr[warp] = top; ss[warp] = sum; }
    __syncthreads();
    top = sr[0];
#pragma unroll
    for (int w = 1; w < CW; ++w) top = fmaxf(top, sr[w]);
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < CW; ++w) sum = fmaf(ss[w], exp2_approx(sr[w] - top), sum);
    const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;
    float o[G];
#pragma unroll
    for (int i = 0; i < G; ++i) o[i] = 0.0f;
    for (int i0 = warp; i0 < n; i0 += CW * UNROLL) {
        if (i0 != warp) load(i0);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (i0 + u * CW < n) {
                const float f = part_at<G>(p, r, i0 + u * CW)[COLS * D + COLS + h] * exp2_approx(weight[i0 + u * CW] - top) * inverse;
                const float *x = reinterpret_cast<const float *>(&v[u]);
#pragma unroll
                for (int i = 0; i < G; ++i) o[i] = fmaf(x[i], f, o[i]);
            }
    }
#pragma unroll
    for (int i = 0; i < G; ++i) so[warp][lane * G + i] = o[i];
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += 32 * CW) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < CW; ++w) x += so[w][c];
        store_o(p, b * p.o_b + hq * p.o_h + c, x);
    }
    if (threadIdx.x == 0) store_sum(p, b, hq, top, sum);
}

// ---- the account ----------------------------------------------------------------------------------
// weight = keep * before + the sum of a kv head's query heads' weights, by a thread to four tokens of a record: the logits are there. Heads are added
// in order. PARTS: their references and sums are not, and the block makes them of the parts.
constexpr int THREADS = 256, SHARED_HEADS = 64, QUAD = 4, STRETCH = THREADS * QUAD;
// references and sums of `n` heads from h0 on, by all warps
template <int G, bool PARTS> __device__ __forceinline__ void stats_of(const DecodeParams &p, int b, int head, int h0, int n, float2 (&stats)[SHARED_HEADS]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // A head whose query row is not finite is left out: its NaN would stay for all steps to come. Its logits are LOWEST here.
    auto counted = [&](float2 s) {
        if (s.y == s.y) return s;
        or_status(p.status, OMMX_ST_NONFINITE);
        return make_float2(0.0f, 0.0f);
    };
    if constexpr (PARTS) {
        for (int h = warp; h < n; h += THREADS / 32) {
            const int row = head * p.col_blocks + (h0 + h) / COLS;
            const Parts r = parts_of(p, b, row, lane);
            float2 s = make_float2(LOWEST, 0.0f);
            if (r.count == 1) s = p.stats[((int64_t)b * p.c.H + head) * p.group + h0 + h];
            else if (r.count > 1) {
                float top, sum;
                meet<G>(p, r, (h0 + h) % COLS, lane, 32, top, sum);
                s = make_float2(top, sum != 0.0f ? 1.0f / sum : 0.0f);
            }
            if (lane == 0) stats[h] = counted(s);
        }
    } else {
        for (int h = threadIdx.x; h < n; h += THREADS) stats[h] = counted(p.stats[((int64_t)b * p.c.H + head) * p.group + h0 + h]);
    }
    __syncthreads();
}
// Block `block` of `blocks` of a kv head's; it takes every blocks-th stretch, so that references and sums are made once where there are many.
template <int G, bool PARTS> __device__ __forceinline__ void weigh(const DecodeParams &p, int b, int head, int block, int blocks) {
    __shared__ __align__(16) float2 stats[SHARED_HEADS];
    wait_earlier();
    let_next_in();
    const int len = length_of(p, b);
    if ((int64_t)block * STRETCH >= len) return;
    const Span span = span_of(p, len);
    // a sequence of more records than are counted was not attended to, or where they are dealt out none was: reported
    if (p.dealt ? reinterpret_cast<const uint2 *>(p.work)->y == OVER : too_many(p, span.units, p.c.H * p.col_blocks)) return;
    const bool few = p.group <= SHARED_HEADS, wide = p.group % 4 == 0;
    const int64_t step = (int64_t)blocks * STRETCH;
    auto page_of = [&](int64_t first) -> int64_t {
        const int64_t t = first + QUAD * threadIdx.x;
        return t < len ? page_id(p.s, b, (int)(t >> p.page_shift)) : -1;
    };
    int64_t next_page = page_of((int64_t)block * STRETCH);                  // of the stretch to come, on its way
    if (few) stats_of<G, PARTS>(p, b, head, 0, p.group, stats);
    for (int64_t first = (int64_t)block * STRETCH; first < len; first += step) {
        const int t = (int)first + QUAD * threadIdx.x, record = t >> 4, unit = record < span.head ? record : record - span.skip;
        const int64_t page = next_page;
        next_page = page_of(first + step);
        const bool there = page >= 0 && page < p.c.num_pages;               // if not, it is reported
        uint32_t seen = there ? visible(p, len, record) >> (t & 15) & 15u : 0u;
        uint32_t kept = !there ? 0u : len - t >= QUAD ? 15u : (1u << (len - t)) - 1;
        if (seen && unit >= p.most_units) { kept &= ~seen; seen = 0; }      // past max_seq_len: reported
        const int64_t at = (page * p.c.H + head) * p.c.page + (t & (p.c.page - 1));
        const float *x = p.logits + ((((int64_t)b * p.c.H + head) * p.most_units + unit) * 16 + (t & 15)) * p.group;
        float4 before = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (kept && p.keep != 0.0f) before = *reinterpret_cast<const float4 *>(p.before + at);
        float add[QUAD] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float *from[QUAD];                  // what is not seen is read from where there is something
#pragma unroll
        for (int u = 0; u < QUAD; ++u) from[u] = seen >> u & 1 ? x + u * p.group : p.logits;
        for (int h0 = 0; h0 < p.group; h0 += SHARED_HEADS) {
            const int n = min(SHARED_HEADS, p.group - h0);
            if (!few) {
                __syncthreads();
                stats_of<G, PARTS>(p, b, head, h0, n, stats);
            }
            if (wide) {
                for (int h = 0; h < n; h += 4) {
                    float4 v[QUAD];
#pragma unroll
                    for (int u = 0; u < QUAD; ++u) v[u] = *reinterpret_cast<const float4 *>(from[u] + h0 + h);
                    const float4 s01 = *reinterpret_cast<const float4 *>(&stats[h]), s23 = *reinterpret_cast<const float4 *>(&stats[h + 2]);
#pragma unroll
                    for (int u = 0; u < QUAD; ++u) {
                        add[u] = fmaf(exp2_approx(v[u].x - s01.x), s01.y, add[u]);
                        add[u] = fmaf(exp2_approx(v[u].y - s01.z), s01.w, add[u]);
                        add[u] = fmaf(exp2_approx(v[u].z - s23.x), s23.y, add[u]);
                        add[u] = fmaf(exp2_approx(v[u].w - s23.z), s23.w, add[u]);
                    }
                }
            } else {
                for (int h = 0; h < n; ++h) {
                    const float2 s = stats[h];
#pragma unroll
                    for (int u = 0; u < QUAD; ++u) add[u] = fmaf(exp2_approx(from[u][h0 + h] - s.x), s.y, add[u]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < QUAD; ++u) add[u] = seen >> u & 1 ? add[u] : 0.0f;
        const float4 now = p.keep != 0.0f ? make_float4(fmaf(p.keep, before.x, add[0]), fmaf(p.keep, before.y, add[1]), fmaf(p.keep, before.z, add[2]), fmaf(p.keep, before.w, add[3]))
                                          : make_float4(add[0], add[1], add[2], add[3]);
        if (kept == 15u) {
            *reinterpret_cast<float4 *>(p.c.weight + at) = now;
        } else {
#pragma unroll
            for (int u = 0; u < QUAD; ++u)
                if (kept >> u & 1) p.c.weight[at + u] = u == 0 ? now.x : u == 1 ? now.y : u == 2 ? now.z : now.w;
        }
    }
}

// Behind the first kernel: what joins the parts (BY: nothing, a block to a row, a block to a head), and the account's blocks.
// Grid: (joining blocks of a sequence + blocks of tokens x H, sequences).
enum { NONE, ROW, HEAD_BLOCKS };
template <int G, int BY> __global__ void __launch_bounds__(THREADS, BY == NONE ? 6 : 4) kv8_second_kernel(const __grid_constant__ DecodeParams p, int joining) {
    static_assert(THREADS == 32 * COLS && THREADS == 32 * CW, "one size of blocks");
    const int b = blockIdx.y, i = blockIdx.x;
    if (i < joining) {
        if constexpr (BY == ROW) combine_row<G>(p, b, i);
        if constexpr (BY == HEAD_BLOCKS) combine_head<G>(p, b, i / COLS, i % COLS);
        return;
    }
    const int blocks = (gridDim.x - joining) / p.c.H, at = i - joining, head = at / blocks;
    weigh<G, BY != NONE>(p, b, head, at - head * blocks, blocks);
}

// ---- host ---------------------------------------------------------------------------------------
static int64_t most_blocks(int warps) {
    const int n = WARPS_PER_SM / warps * sm_count();
    return n < MOST_PARTS ? n : MOST_PARTS;
}
static int64_t parts_floats(int head_dim) {
    const int64_t part = head_dim == 64 ? PART<2> : PART<4>;
    return HEAD + 2 * part * most_blocks(4);
}
// tokens that a sequence of the call can have, and records of a row
static int64_t most_tokens(const ommx_kv8_decode_args *a) {
    const int64_t n = (int64_t)a->seqs.pages_per_seq * a->cache.page_size;
    return a->max_seq_len > 0 && a->max_seq_len < n ? a->max_seq_len : n;
}
static int64_t most_units(const ommx_kv8_decode_args *a) {
    const int64_t n = (most_tokens(a) + 15) / 16;
    if (a->window <= 0) return n;
    const int64_t seen = (a->sink_tokens + 15LL) / 16 + (a->window + 15LL) / 16 + 1;
    return n < seen ? n : seen;
}
static int64_t workspace_floats(const ommx_kv8_decode_args *a) {
    const int64_t units = most_units(a);
    int64_t n = units <= WHOLE ? 0 : parts_floats(a->cache.head_dim);
    if (a->cache.weight) n += 2LL * a->seqs.batch * a->n_q_heads + units * 16 * a->seqs.batch * a->n_q_heads;
    return (n + 3) / 4 * 4;
}

template <int G, bool E4M3, bool FINE, int NW, bool CLUSTER> static int launch_decode(const DecodeParams &p, int64_t blocks, int cluster, int64_t tokens, cudaStream_t st) {
    static std::atomic<uint64_t> allowed{0};      // devices on which the kernel may take its shared memory
    int dev = 0;
    if (int rc = current_device(&dev)) return rc;
    if (!(allowed.load(std::memory_order_acquire) >> dev & 1)) {
        OMMX_CUDA_TRY(cudaFuncSetAttribute(kv8_decode_kernel<G, E4M3, FINE, NW, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Memory<G, NW>)));
        allowed.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (int rc = launch_dependent(kv8_decode_kernel<G, E4M3, FINE, NW, CLUSTER>, dim3((unsigned)blocks), 32 * NW, sizeof(Memory<G, NW>), st, cluster, p)) return rc;
    // a row has some blocks / rows parts
    const int rows = p.c.H * p.col_blocks;
    // The account's blocks: at most as many as the SMs hold. Where there are stretches for no more than that they stand beside those that join the
    // parts, and make references and sums themselves; else they come behind them (8 x 64K tokens: 234 us beside, 215 behind; one of 64K 41.4 and 43.0).
    const int64_t heads = (int64_t)p.c.H * p.s.B, stretches = (tokens + STRETCH - 1) / STRETCH;
    const bool joins = p.dealt, beside = joins && stretches * heads <= 4LL * sm_count();
    const int64_t fill = (6LL * sm_count() + heads - 1) / heads;
    const int account = (int)(stretches < fill ? stretches : fill) * p.c.H;
    if (joins) {
        const bool by_row = (int64_t)rows * p.s.B * COLS >= blocks;
        const int joining = by_row ? rows : rows * COLS;
        const dim3 grid(joining + (beside ? account : 0), p.s.B);
        const int rc = by_row ? launch_dependent(kv8_second_kernel<G, ROW>, grid, THREADS, 0, st, 1, p, joining)
                              : launch_dependent(kv8_second_kernel<G, HEAD_BLOCKS>, grid, THREADS, 0, st, 1, p, joining);
        if (rc) return rc;
    }
    if (beside || !account) return 0;
    return launch_dependent(kv8_second_kernel<G, NONE>, dim3(account, p.s.B), THREADS, 0, st, 1, p, 0);
}

static int decode(const ommx_kv8_decode_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv8_decode: null args");
    DecodeParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv8_decode", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv8_decode", a->seqs, p.c, &p.s)) return rc;
    if (a->q_dtype != OMMX_DT_BF16 && a->q_dtype != OMMX_DT_F16) return fail(OMMX_E_UNSUPPORTED, "kv8_decode: q must be bfloat16 or float16");
    if (a->o_dtype != OMMX_DT_F32 && a->o_dtype != OMMX_DT_BF16 && a->o_dtype != OMMX_DT_F16) return fail(OMMX_E_ARG, "kv8_decode: o dtype %d", a->o_dtype);
    if (a->n_q_heads < p.c.H || a->n_q_heads % p.c.H)
        return fail(OMMX_E_UNSUPPORTED, "kv8_decode: %d query heads are not a multiple of %d kv heads", a->n_q_heads, p.c.H);
    if (!(a->logit_cap >= 0.0f) || !std::isfinite(a->logit_cap)) return fail(OMMX_E_ARG, "kv8_decode: logit_cap must be finite and not negative");
    if (!std::isfinite(a->sm_scale)) return fail(OMMX_E_ARG, "kv8_decode: sm_scale must be finite");
    if (a->window < 0 || a->sink_tokens < 0 || a->max_seq_len < 0) return fail(OMMX_E_ARG, "kv8_decode: window, sink_tokens and max_seq_len must not be negative");
    if (a->cache.weight && (!std::isfinite(a->keep) || (a->keep != 0.0f && !a->weight_before))) return fail(OMMX_E_ARG, "kv8_decode: keep must be finite, and what is kept must be given");
    if (reinterpret_cast<uintptr_t>(a->weight_before) % 16) return fail(OMMX_E_ARG, "kv8_decode: weight_before must be 16-byte aligned");
    const int64_t weights = (int64_t)p.c.num_pages * p.c.H * p.c.page;
    if (a->cache.weight && a->keep != 0.0f && a->weight_before != a->cache.weight && a->weight_before < a->cache.weight + weights && a->cache.weight < a->weight_before + weights)
        return fail(OMMX_E_ARG, "kv8_decode: weight_before must be weight itself or apart from it");
    if (p.s.B > 65535) return fail(OMMX_E_UNSUPPORTED, "kv8_decode: a batch of %d", p.s.B);
    if (p.s.B == 0) return 0;
    if (!a->q || !a->o || !a->lse) return fail(OMMX_E_ARG, "kv8_decode: q, o and lse must not be null");
    const int64_t need = workspace_floats(a);
    if (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_floats < need))
        return fail(OMMX_E_ARG, "kv8_decode: workspace must be 16-byte aligned and hold %lld floats", (long long)need);
    p.q = a->q; p.q16 = a->q_dtype == OMMX_DT_F16; p.q_b = a->q_stride_b; p.q_h = a->q_stride_h;
    p.q_wide = (reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)(2 * p.q_b) | (uintptr_t)(2 * p.q_h)) % 16 == 0;
    p.o = a->o; p.o_type = a->o_dtype; p.o_b = a->o_stride_b; p.o_h = a->o_stride_h;
    p.lse = a->lse; p.lse_b = a->lse_stride_b;
    p.group = a->n_q_heads / p.c.H; p.col_blocks = (p.group + COLS - 1) / COLS;
    p.page_shift = shift_of(p.c.page);
    p.window = a->window; p.sinks = a->sink_tokens;
    // a cap past 2^40 moves a logit of 2^24 by less than its last bit (x^3 / 3 cap^2), and is none: in powers of two the largest ones are infinite
    p.cap = a->logit_cap <= 0x1p40f ? a->logit_cap : 0.0f;
    p.status = a->status;
    p.scale = (float)std::frexp(p.cap > 0.0f ? (double)a->sm_scale / p.cap : (double)a->sm_scale, &p.scale_e);
    if (!(p.cap > 0.0f)) p.scale *= LOG2E;
    if (p.c.num_pages == 0) return fail(OMMX_E_ARG, "kv8_decode: a cache of no pages");   // what is fetched for a page that is not there
    // as many blocks as the SMs hold, no more than the work can have
    const int64_t units = most_units(a);
    const int64_t rows = (int64_t)p.s.B * p.c.H * p.col_blocks;
    if (units * rows >= 1LL << 31 || rows * COLS >= 1LL << 31)
        return fail(OMMX_E_UNSUPPORTED, "kv8_decode: %lld rows of up to %lld records (2^31 in all are counted): give max_seq_len", (long long)rows, (long long)units);
    p.most_units = (int)units;
    p.work = a->workspace;
    if (p.c.weight) {
        p.stats = reinterpret_cast<float2 *>(a->workspace + (units <= WHOLE ? 0 : parts_floats(a->cache.head_dim)));
        p.logits = reinterpret_cast<float *>(p.stats + (int64_t)p.s.B * a->n_q_heads);
        p.before = a->weight_before; p.keep = a->keep;
    }
    // Blocks of eight warps where rows are few, so that a row has few parts, of four where they are many: then blocks often go on from
    // one row to the next, and an SM's others work meanwhile. As many blocks as the SMs hold, no more than the work can have. Rows that
    // are short for certain go whole to a block each, and the second kernel is not needed.
    const int warps = rows >= 64 ? 4 : 8;
    p.least = 2 * warps;
    const int64_t most = (units * rows + p.least - 1) / p.least, hold = most_blocks(warps);
    // Rows of middling length, and few, go to a cluster of eight-warp blocks each, as many as fit at once: no second kernel
    int cluster = 1;
    static AtOnce known[2];                       // of eight and sixteen warps; D = 64 takes less
    while (cluster < MOST_CLUSTER && 2 * cluster * rows <= most_blocks(8) && rows <= clusters_at_once(known[0], kv8_decode_kernel<4, false, false, 8, true>, 256, sizeof(Memory<4, 8>), 2 * cluster)) cluster *= 2;
    // of sixteen warps where a row has more records than eight of eight warps should take, up to where all SMs and a join are faster, which is later the more
    // rows there are. us with eight warps, sixteen and a join: 8 rows of 4600 tokens 10.3, 10.8, 12.7, of 6000 11.1, 11.3, 13.4, 8000 12.5, 12.5, 13.6,
    // 10000 14.2, 13.5, 13.9, 12000 15.6, 14.6, 14.5; where sixteen and a join meet: one row 5900 tokens (10.9), two 6700 (11.6), four 6500 (11.5), eight
    // 11500 (14.4), twelve 20000 (19.2), fifteen past 20000 (19.4 and 21.6). The line lies within 0.6 us of the better one up to eight rows; past
    // its end twelve rows of 16000 take 17.9 for 17.1, fifteen of 20000 21.6 for 19.4
    const bool wide = cluster == MOST_CLUSTER && units > 36 * cluster && units <= (40 + 6 * rows) * cluster &&
                      rows <= clusters_at_once(known[1], kv8_decode_kernel<4, false, false, 16, true>, 512, sizeof(Memory<4, 16>), cluster);
    if (units > 36 * cluster && !wide) cluster = 1;
    // A window makes rows alike, so where there is a block for each and not two they go whole too. us whole and dealt, for 304, 360, 488 and 584 rows of 8 kv heads
    // whose sequences have 300 to 20000 tokens: windows of 600 17.1 and 17.5, 17.6 and 21.4, 18.2 and 22.1, 18.8 and 23.5, of 1400 30.7 and 25.7, 31.4 and
    // 28.8, 33.5 and 37.1, 36.0 and 41.4; 580 rows of one kv head 18.8 and 32.7, 35.4 and 50.8. Where five sequences in six are shorter than the window it is
    // slower below some 450 rows and windows past 1000 (360 rows of 1025 23.0 and 20.7, of 1400 29.2 and 24.3; 488 rows 23.9 and 25.6): lengths are
    // not known here
    const bool alike = a->window > 0 && cluster == 1 && rows <= hold && 2 * rows > hold && units <= 3 * WHOLE;
    p.whole = units <= WHOLE / 2 || (units <= WHOLE && cluster == 1) || alike;
    if (p.whole) cluster = 1;
    p.dealt = !p.whole && cluster == 1;
    const int64_t blocks = p.whole ? rows : cluster > 1 ? cluster * rows : most < 1 ? 1 : most < hold ? most : hold;
    const int64_t tokens = p.c.weight ? most_tokens(a) : 0;                 // that weights are kept of
    auto launch = [&](auto g, auto e4m3, auto fine) {
        constexpr int G = decltype(g)::value;
        constexpr bool E4M3 = decltype(e4m3)::value, FINE = decltype(fine)::value;
        if (cluster > 1 && wide) return launch_decode<G, E4M3, FINE, 16, true>(p, blocks, cluster, tokens, st);
        if (cluster > 1) return launch_decode<G, E4M3, FINE, 8, true>(p, blocks, cluster, tokens, st);
        return warps == 4 ? launch_decode<G, E4M3, FINE, 4, false>(p, blocks, 1, tokens, st) : launch_decode<G, E4M3, FINE, 8, false>(p, blocks, 1, tokens, st);
    };
    using std::integral_constant;
    auto of_size = [&](auto e4m3, auto fine) {
        return a->cache.head_dim == 128 ? launch(integral_constant<int, 4>(), e4m3, fine) : launch(integral_constant<int, 2>(), e4m3, fine);
    };
    auto of_code = [&](auto fine) { return a->cache.code == OMMX_KV8_E4M3 ? of_size(std::true_type(), fine) : of_size(std::false_type(), fine); };
    return a->o_dtype != OMMX_DT_BF16 ? of_code(std::true_type()) : of_code(std::false_type());
}

}  // namespace kv8
}  // namespace ommx

extern "C" int64_t ommx_b200_kv8_decode_workspace_floats(const ommx_kv8_decode_args *args) {
    return !args || (args->cache.head_dim != 64 && args->cache.head_dim != 128) ? 0 : ommx::kv8::workspace_floats(args);
}
extern "C" int ommx_b200_kv8_decode(const ommx_kv8_decode_args *args, void *stream) { return ommx::kv8::decode(args, (cudaStream_t)stream); }
