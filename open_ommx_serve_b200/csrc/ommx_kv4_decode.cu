// The 4-bit cache: attention of one query row per sequence.
//
// For query head h of a sequence, over its tokens t:  x_t = sm_scale q.K_t,  o = sum_t exp(x_t) V_t / sum_t exp(x_t), with
// K_tc = z_tj + s_tj a_tc and V the same (j: the group of 32 channels that c is in, a: codes 0..15). So
//   q.K_t = sum_j s_tj (sum_c q_c a_tc) + z_tj (sum_c q_c),      o_c = sum_t (p_t s_tj) a_tc + sum_t p_t z_tj:
// the codes go into the tensor cores as they are. A nibble masked in place is the fp16 subnormal code * 2^-24 (or 2^-20), exact and
// one LOP3 for two of them; the tokens (of K) and channels (of V) are the rows of an m16n8k16 product and up to eight query heads
// that share the kv head its columns. Scales meet the sums of K's groups behind the product and the weights of V before it, zeros
// are fp32 multiply-adds. Queries keep all their bits: a head's are scaled by a power of two into fp16's range.
//
// A weight w_t = exp(x_t) stays fp32 where it meets a zero and in the sum, against a reference of the logits alone: values of any size the
// cache holds leave no token out. Products w_t s_tj are rounded to fp16, by 2^-11 at most, in a unit that the largest of them sets: below
// 2^-23 of it they have fewer bits (fp16's smallest step is 2^-24), and are off by 2^-34 of it at most. That is less than a bf16 output's own
// rounding; where the output is finer (fp16, fp32), a second product takes what the rounding left (FINE: 32 ragged sequences 58 us
// without, 66 with; 8 x 64K tokens 139 and 165). Sums of weights and zeros stay fp32.
//
// What the tensor cores cut is then the largest error of a record: they line the addends of a product up with the largest and cut them 25 bits
// below its leading one (an emulation of that gives the kernel's errors to a fifth), where a subnormal counts as 2^-14. A masked nibble lies 10 bits
// below that (the odd ones, 16 times as large, 6), so an addend loses up to 2^-15 of one code of the record's heaviest token - or, in a
// logit, of the group's largest |q| -: 2^-14 of a group's range a record at most (17 addends), of the heaviest token's share in the
// output. Nibbles moved up to bits 6..9 would lose 2^-21, for some 48 shifts a record.
//
// What bounds it: a record's 160 bytes a token are read once for each eight query heads of its kv head, so HBM, and beside it the schedulers:
// a record is some 330 instructions of a warp, 17 of them products that hold a scheduler 8 cycles, in which its multiply-adds wait. 8 x 64K
// tokens, 8 kv heads, 32 or 64 query heads: 139 us (4.8 TB/s, 74 % of the copy rate), 260 with 128 heads; an earlier form of 136 us took 110
// with the copies left out, 112 with the arithmetic left out. e4m3 products for K (half the masks, twice the depth) were slower, 173: their
// operands are converted. The D = 128 forms spill a few registers, outside the loop over records: 33 loads and stores of a warp in 2 x 64K
// tokens, of 10 thousand instructions.
#include <cmath>
#include <type_traits>

#include "ommx_kv4.cuh"
#include "ommx_kv_device.cuh"

namespace ommx {
namespace kv4 {

using namespace kv;

constexpr int WARPS_PER_SM = 16;                  // as many as the registers hold; a block is NW of them, each with records of its own
constexpr int STAGES = 3, AHEAD = STAGES - 1;     // records that a warp holds, and those of them on their way
constexpr int FULL = 0x1010;                      // sixteen tokens in each of those
constexpr int COLS = 8;                           // query heads side by side
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Weights w = 2^(x - ref) are held near 2^-ABOVE: they meet zeros of up to 2^126, and a sum of 2^24 such products at HEAVY stays below 2^127.
// Products of weights and scales, w s unit, go to fp16: the largest one lies above 2^(TOP - 2) when the references have moved, and may grow to ROOM
// before they move again. More of fp16's range below it would cost moves (8 x 64K tokens 137.9 us with TOP 8, 139.3 with 12).
constexpr int ABOVE = 30, TOP = 11;
constexpr float HEAVY = 0x1p-23f, ROOM = 60000.0f;
constexpr float LOWEST = -1e30f;
constexpr int MOST_PARTS = 768;                   // blocks of a call that shares rows
constexpr int WHOLE = 32;                         // records of a row that one block takes at most where it could share it

struct DecodeParams {
    Cache c;
    Seqs s;
    const void *q;
    void *o;
    float *lse, *work;
    const int32_t *selected;
    int64_t q_b, q_h, o_b, o_h, lse_b;
    int32_t q16, q_wide, o_type, group, col_blocks, num_selected, page_shift, least, whole;
    float sm_scale, cap;
    int32_t *status;
};

// ---- how the work is dealt ------------------------------------------------------------------------
// Units are records (16 tokens of a kv head, for a block of COLS of its query heads); a row (sequence, kv head, block of heads) is a
// run of them. Lengths are known on the device alone, so every block works the same deal out, and leaves it for the
// second kernel:
// * a block to a row, where the host knows that rows are short (`whole`), or a cluster of blocks, which exchange their parts themselves;
// * else every row is cut into pieces of at most `per` units, a block to a piece, with the smallest `per` for which there are blocks
//   enough;
// * or, where that would leave a block with over BEGIN units more than an even share, all rows end to end are cut into such shares,
//   whatever rows they touch. A second piece costs a block some 4 us, half of it hidden by the SM's other blocks (64K tokens: 26.7 us
//   with seven such blocks of 296, 24.4 with none; 64 sequences of 200..2000 tokens: 43.3 with even shares, 38.3 with pieces).
// A piece that is a whole row is finished where it is computed; the others' parts meet in the second kernel. A block has at most two
// of those, of the row that an earlier block began (its slot 0) and of the one that a later block goes on with (slot 1).
constexpr uint32_t OVER = 2;                      // in the deal's place: there is none
constexpr int BEGIN = 64, HEAD = 4;               // HEAD: floats in front of the parts, which hold the deal
__device__ __forceinline__ int pages_of(const DecodeParams &p, int len) { return (len + p.c.page - 1) >> p.page_shift; }
__device__ __forceinline__ int length_of(const DecodeParams &p, int b) {
    const int len = p.s.len[b];
    const int64_t most = (int64_t)p.s.max_pages << p.page_shift;
    if (len < 0 || len > most) { or_status(p.status, OMMX_ST_BAD_LENGTH); return len < 0 ? 0 : (int)most; }
    return len;
}
__device__ __forceinline__ int units_of(const DecodeParams &p, int len) {
    if (p.selected) return min(pages_of(p, len), p.num_selected) * p.c.parts;
    return (len + 15) >> 4;
}
struct Deal { uint32_t per, total; bool pieces, over; };   // over: lengths far past max_seq_len, of more units than 32 bits count
__device__ __forceinline__ uint32_t pieces_of(uint32_t units, uint32_t per) { return (units + per - 1) / per; }
__device__ __forceinline__ Deal deal(const DecodeParams &p, uint32_t rows, uint32_t blocks, int lane) {
    uint64_t sum = 0;
    uint32_t some = 0, most = 0;
    const uint32_t own = lane < p.s.B ? units_of(p, length_of(p, lane)) : 0;
    for (int b = lane; b < p.s.B; b += 32) {
        const uint32_t n = b == lane ? own : units_of(p, length_of(p, b));
        sum += n;
        some += n > 0;
        most = max(most, n);
    }
    Deal d;
#pragma unroll
    for (int i = 16; i; i /= 2) sum += __shfl_xor_sync(~0u, sum, i);
    d.over = sum * rows >> 31;
    d.total = d.over ? 0 : (uint32_t)sum * rows;
    const uint32_t full = __reduce_add_sync(~0u, some) * rows;
    most = __reduce_max_sync(~0u, most);
    const uint32_t even = max((d.total + blocks - 1) / blocks, (uint32_t)p.least);
    d.per = even;
    d.pieces = false;
    if (d.over) or_status(p.status, OMMX_ST_BAD_LENGTH);
    if (d.over || full == 0 || full > blocks) return d;
    // pieces of `per` take total / per + full blocks at most; fewer may do
    uint32_t lo = even, hi = min(max(most, even), full < blocks ? max(even, d.total / (blocks - full) + 1) : 0xFFFFFFFFu);
#pragma unroll 1
    for (int i = 0; i < 6 && lo < hi; ++i) {
        const uint32_t per = i == 0 ? lo : (lo + hi) / 2;
        uint32_t n = pieces_of(own, per);
        for (int b = lane + 32; b < p.s.B; b += 32) n += pieces_of(units_of(p, length_of(p, b)), per);
        if (__reduce_add_sync(~0u, n) * rows <= blocks) hi = per;
        else lo = per + 1;
    }
    if (hi <= even + BEGIN) { d.per = hi; d.pieces = true; }
    return d;
}

// ---- pieces ---------------------------------------------------------------------------------------
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ float scale_of(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ float zero_of(uint32_t w) { return __uint_as_float(w << 16); }
// of a reference and a sum of weights, which lie near 2^-ABOVE
__device__ __forceinline__ float log_sum(float ref, float sum) {
    return sum != 0.0f ? ((ref - ABOVE) + log2f(sum * power_of_two(ABOVE))) * LN2 : -INFINITY;
}

__device__ __forceinline__ void store_o(const DecodeParams &p, int64_t at, float v) {
    if (p.o_type == OMMX_DT_F32) reinterpret_cast<float *>(p.o)[at] = v;
    else if (p.o_type == OMMX_DT_F16) reinterpret_cast<__half *>(p.o)[at] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16 *>(p.o)[at] = __float2bfloat16_rn(v);
}

// A kv head's queries as B fragments. Lane (g, t): head g, channels 32 j + 8 t + 0..7; frag[j][k] holds the channels (0, 4), (1, 5),
// (2, 6), (3, 7); the second and fourth meet nibbles that are 16 times as large. What meets the zeros is the sum of a group's
// channels: three bf16 numbers add up to it, so that one bf16 product of the zeros, as they are stored, and them is exact.
template <int G> struct Query {
    uint32_t frag[G][4], sums[2];
    float factor[2], raw[2];                      // of heads 2 t and 2 t + 1: the products' units in powers of two; with a cap: in its units
};
// Warp j < G takes group j of all heads; largest values, sums and fragments meet in shared memory. All warps call it.
template <int G> struct QueryMemory {
    uint4 frag[G][32];
    float top[COLS][G], sum[COLS][G];
};
template <int G>
__device__ __forceinline__ void load_query(const DecodeParams &p, int b, int first_head, int n, int warp, int lane, QueryMemory<G> &m, Query<G> &q) {
    const int g = lane >> 2, t = lane & 3;
    float x[8];
    if (warp < G) {
        load_q8(p, b * p.q_b + (first_head + min(g, n - 1)) * p.q_h + 32 * warp + 8 * t, x);
        float top = fabsf(x[0]), sum = 0x1p-8f * x[0];                      // 32 of the largest numbers would not have a finite sum
#pragma unroll
        for (int i = 1; i < 8; ++i) { top = fmaxf(top, fabsf(x[i])); sum += 0x1p-8f * x[i]; }
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
        sum += __shfl_xor_sync(~0u, sum, 1);
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
        sum += __shfl_xor_sync(~0u, sum, 2);
        if (t == 0) { m.top[g][warp] = top; m.sum[g][warp] = sum; }
    }
    __syncthreads();
    float top = m.top[g][0];
#pragma unroll
    for (int j = 1; j < G; ++j) top = fmaxf(top, m.top[g][j]);
    const int e = top > 0.0f ? max(exponent_of(top), -100) : 0;
    const float up = power_of_two(13 - e);
    if (warp < G) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= i & 1 ? up * 0.0625f : up;      // odd nibbles are 16 times as large
        m.frag[warp][lane] = make_uint4(half2_bits(x[0], x[4]), half2_bits(x[1], x[5]), half2_bits(x[2], x[6]), half2_bits(x[3], x[7]));
    }
    // two powers of two: one would pass 32 bits for |q| from 2^117 on
    const float most = 3.4e38f, factor = fminf(fmaxf(p.sm_scale * 2048.0f * power_of_two(e), -most), most);         // 2^11: 24 - 13
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float f = __shfl_sync(~0u, factor, 8 * t + 4 * i);
        q.raw[i] = fminf(fmaxf(f / p.cap, -most), most);
        // never 0, so that a masked logit can be an infinity of the other sign: without a cap |x| < 2^124, and x times this is nothing
        q.factor[i] = p.cap > 0.0f ? p.cap * LOG2E : f * LOG2E != 0.0f ? fminf(fmaxf(f * LOG2E, -most), most) : 0x1p-149f;
    }
    // rows of the product: term r of group j at G r + j; lane t holds rows 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
    const int j = G == 4 ? 2 * (t & 1) : 0;
    const float a = m.sum[g][j] * (up * 0x1p-16f), c = m.sum[g][j + 1] * (up * 0x1p-16f);
    const float a1 = bf16_round_f32(a), c1 = bf16_round_f32(c), a2 = bf16_round_f32(a - a1), c2 = bf16_round_f32(c - c1);
    const uint32_t term1 = f32_to_bf16_bits(a1) | f32_to_bf16_bits(c1) << 16, term2 = f32_to_bf16_bits(a2) | f32_to_bf16_bits(c2) << 16,
                   term3 = f32_to_bf16_bits(a - a1 - a2) | f32_to_bf16_bits(c - c1 - c2) << 16;
    if constexpr (G == 4) {
        q.sums[0] = t < 2 ? term1 : term2;
        q.sums[1] = t < 2 ? term3 : 0u;
    } else {
        q.sums[0] = t == 0 ? term1 : t == 1 ? term2 : t == 2 ? term3 : 0u;
        q.sums[1] = 0u;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const uint4 f = m.frag[i][lane];
        q.frag[i][0] = f.x; q.frag[i][1] = f.y; q.frag[i][2] = f.z; q.frag[i][3] = f.w;
    }
}

// A warp's running state. acc[j][u]: 2^-24 channel 32 j + 4 g + 2 u (rows g), 2^-20 the next one (rows g + 8); heads 2 t, 2 t + 1.
// The tensor cores cut what they add to a sum, so long sums of codes, none of them negative, fall short: by some 2^-26 of the sum a
// record, which is much of an output that the zeros nearly cancel (8e-4 of it after 110 records of 64K tokens that weigh alike). So
// `acc` is added to `whole` in shared memory every 64 records, every 32 where the output is finer than bf16 and a record
// is two products (2 % of the time).
template <int G> struct State {
    float acc[G][2][4], zero[G][2], sum[2], ref[2];
    float unit[2];                                // a power of two that only `acc` has in it
    float *whole;                                 // the lane's first of 8 G values, 32 apart
    bool some;                                    // there is something there
};

template <int G> __device__ __forceinline__ void clear(State<G> &s, float *whole) {
    s.whole = whole;
    s.some = false;
#pragma unroll
    for (int j = 0; j < G; ++j) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) s.acc[j][u][i] = 0.0f;
        s.zero[j][0] = s.zero[j][1] = 0.0f;
    }
    s.sum[0] = s.sum[1] = 0.0f;
    s.ref[0] = s.ref[1] = LOWEST;
    s.unit[0] = s.unit[1] = 1.0f;
}
// The references of head i move to `ref`, a whole number as the one before, so that nothing is rounded. `product`: the record's largest logit
// plus exponent of its scales, less `ref` (logits may be so large that an exponent added to one is lost). A unit stays within normal
// numbers: where scales are the smallest (2^-96), products stay below 2^TOP. The largest logit less `ref` is off by half a step of `ref`, 32 at
// 2^30: up to there a weight is a finite number whatever that is.
template <int G> __device__ __forceinline__ void move(State<G> &s, int i, float ref, float product) {
    const int was = exponent_of(s.unit[i]);
    const float over = ceilf(fmaxf((s.ref[i] - ref) + (float)(TOP - was), product));       // 2^over: the largest product
    const int now = TOP - (int)fminf(fmaxf(over, (float)(TOP - 126)), (float)(TOP + 126));
    const float f = exp2_approx(s.ref[i] - ref), a = exp2_approx(s.ref[i] - ref + (float)(now - was));
    s.ref[i] = ref;
    s.unit[i] = power_of_two(now);
#pragma unroll
    for (int j = 0; j < G; ++j) {
#pragma unroll
        for (int u = 0; u < 2; ++u) { s.acc[j][u][i] *= a; s.acc[j][u][i + 2] *= a; }
        s.zero[j][i] *= f;
    }
    s.sum[i] *= f;
    if (s.some)
#pragma unroll 1
        for (int k = i; k < 8 * G; k += 2) s.whole[32 * k] *= a;
}
template <int G> __device__ __forceinline__ void put_by(State<G> &s) {      // acc to `whole`
#pragma unroll
    for (int i = 0; i < 8 * G; ++i) {
        float &a = s.acc[i / 8][i / 4 % 2][i % 4];
        s.whole[32 * i] = s.some ? s.whole[32 * i] + a : a;
        a = 0.0f;
    }
    s.some = true;
}
template <int G> __device__ __forceinline__ void take_back(State<G> &s) {
    if (s.some)
#pragma unroll
        for (int i = 0; i < 8 * G; ++i) s.acc[i / 8][i / 4 % 2][i % 4] += s.whole[32 * i];
}

// ---- a warp's ring of records: 16 bytes a lane at a time, a group of copies for each record ----
// Bulk copies counted by mbarriers move the same bytes with fewer instructions, but a record's arrival, wait and copy held a scheduler
// longer than five of these do (8 x 64K tokens, 8 kv heads: 146.6 us against 141.9 when both were tried).
template <int G> __device__ __forceinline__ void fetch(uint32_t to, const uint8_t *rec, int lane) {   // both at the lane's 16 bytes
#pragma unroll
    for (int i = 0; i < Rec<G>::BYTES; i += 512)
        if (i + 512 <= Rec<G>::BYTES || i + 16 * lane < Rec<G>::BYTES)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i), "l"(rec + i) : "memory");
}
__device__ __forceinline__ void close_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void fetched() {                // all but the last N groups
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    __syncwarp();
}

// One record in shared memory, n of its tokens valid (1..16)
template <int G, bool FINE> __device__ __forceinline__ void attend(const DecodeParams &p, const uint8_t *rec, int n, int lane, const Query<G> &q, State<G> &s) {
    using W = typename Words<G>::T;
    const int g = lane >> 2;
    constexpr uint32_t LO = 0x000F000Fu, HI = 0x00F000F0u;
    alignas(16) uint32_t k0[G], k1[G], kp0[G], kp1[G], vp0[G], vp1[G];
    *reinterpret_cast<W *>(k0) = reinterpret_cast<const W *>(rec)[lane];
    *reinterpret_cast<W *>(k1) = reinterpret_cast<const W *>(rec)[32 + lane];
    *reinterpret_cast<W *>(kp0) = reinterpret_cast<const W *>(rec + Rec<G>::KP)[g];
    *reinterpret_cast<W *>(kp1) = reinterpret_cast<const W *>(rec + Rec<G>::KP)[g + 8];
    *reinterpret_cast<W *>(vp0) = reinterpret_cast<const W *>(rec + Rec<G>::VP)[g];
    *reinterpret_cast<W *>(vp1) = reinterpret_cast<const W *>(rec + Rec<G>::VP)[g + 8];

    // ---- logits: x[0], x[1] of token g and heads 2 t, 2 t + 1; x[2], x[3] of token g + 8
    float x[4];
    {
        const bool up = G == 4 && (lane & 1);
        const uint32_t z0 = __byte_perm(up ? kp0[G - 2] : kp0[0], up ? kp0[G - 1] : kp0[1], 0x5410);
        const uint32_t z1 = __byte_perm(up ? kp1[G - 2] : kp1[0], up ? kp1[G - 1] : kp1[1], 0x5410);
        mma_bf16(x, z0, z1, z0, z1, q.sums[0], q.sums[1]);
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
        float c[4];
        mma_first(c, k0[j] & LO, k1[j] & LO, k0[j] & HI, k1[j] & HI, q.frag[j][0], q.frag[j][1]);
        const uint32_t a = k0[j] >> 8, b = k1[j] >> 8;
        mma(c, a & LO, b & LO, a & HI, b & HI, q.frag[j][2], q.frag[j][3]);
        const float s0 = scale_of(kp0[j]), s1 = scale_of(kp1[j]);
        x[0] = fmaf(s0, c[0], x[0]);
        x[1] = fmaf(s0, c[1], x[1]);
        x[2] = fmaf(s1, c[2], x[2]);
        x[3] = fmaf(s1, c[3], x[3]);
    }
    if (p.cap > 0.0f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = tanhf(x[i] * q.raw[i & 1]);
    }
    const float f0 = q.factor[0], f1 = q.factor[1];                         // x f: logits in powers of two
    if (n < 16) {                                 // what lies behind the last token may be anything
        const float out0 = copysignf(INFINITY, -f0), out1 = copysignf(INFINITY, -f1);   // logits of -inf, whatever the scale's sign
        if (g >= n) {
            x[0] = out0;
            x[1] = out1;
#pragma unroll
            for (int j = 0; j < G; ++j) vp0[j] = 0;
        }
        if (g + 8 >= n) {
            x[2] = out0;
            x[3] = out1;
#pragma unroll
            for (int j = 0; j < G; ++j) vp1[j] = 0;
        }
    }

    // ---- weights
    // the largest scale of each token; a word taken as a number is its scale and less than a hundredth of it more
    float top0 = 0.0f, top1 = 0.0f;
#pragma unroll
    for (int j = 0; j < G; j += 2) {
        top0 = max3(top0, __uint_as_float(vp0[j]), __uint_as_float(vp0[j + 1]));
        top1 = max3(top1, __uint_as_float(vp1[j]), __uint_as_float(vp1[j + 1]));
    }
    float w[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { w[i] = exp2_approx(fmaf(x[i], i & 1 ? f1 : f0, -s.ref[i & 1])); y[i] = w[i] * s.unit[i & 1]; }
    const float heavy = fmaxf(max3(w[0], w[1], w[2]), w[3]), most = fmaxf(fmaxf(y[0], y[1]) * top0, fmaxf(y[2], y[3]) * top1);
    if (__any_sync(~0u, !(heavy <= HEAVY && most <= ROOM))) {
        const float e0 = (float)(exponent_of(top0) + 1), e1 = (float)(exponent_of(top1) + 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float f = i ? f1 : f0;
            float l = fmaxf(x[i] * f, x[i + 2] * f);
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l = fmaxf(l, __shfl_xor_sync(~0u, l, d));
            const float ref = fmaxf(s.ref[i], ceilf(l) + ABOVE);
            float r = fmaxf(fmaf(x[i], f, -ref) + e0, fmaf(x[i + 2], f, -ref) + e1);
#pragma unroll
            for (int d = 4; d < 32; d *= 2) r = fmaxf(r, __shfl_xor_sync(~0u, r, d));
            move(s, i, ref, r);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) { w[i] = exp2_approx(fmaf(x[i], i & 1 ? f1 : f0, -s.ref[i & 1])); y[i] = w[i] * s.unit[i & 1]; }
    }
    s.sum[0] += w[0] + w[2];
    s.sum[1] += w[1] + w[3];

    // ---- values
    alignas(16) uint32_t v0[G], v1[G];
    *reinterpret_cast<W *>(v0) = reinterpret_cast<const W *>(rec + Rec<G>::V)[lane];
    *reinterpret_cast<W *>(v1) = reinterpret_cast<const W *>(rec + Rec<G>::V)[32 + lane];
#pragma unroll
    for (int j = 0; j < G; ++j) {
        const float s0 = scale_of(vp0[j]), s1 = scale_of(vp1[j]), z0 = zero_of(vp0[j]), z1 = zero_of(vp1[j]);
        s.zero[j][0] = fmaf(z1, w[2], fmaf(z0, w[0], s.zero[j][0]));
        s.zero[j][1] = fmaf(z1, w[3], fmaf(z0, w[1], s.zero[j][1]));
        const float m[4] = {y[0] * s0, y[1] * s0, y[2] * s1, y[3] * s1};
        const uint32_t h0 = half2_bits(m[0], m[1]), h1 = half2_bits(m[2], m[3]);
        const uint32_t a = v0[j] >> 8, b = v1[j] >> 8;
        const uint32_t b0 = transpose8x8(h0), b1 = transpose8x8(h1);
        mma(s.acc[j][0], v0[j] & LO, v0[j] & HI, v1[j] & LO, v1[j] & HI, b0, b1);
        mma(s.acc[j][1], a & LO, a & HI, b & LO, b & HI, b0, b1);
        if constexpr (FINE) {
            const float2 r0 = half2_floats(h0), r1 = half2_floats(h1);
            const uint32_t d0 = transpose8x8(half2_bits(m[0] - r0.x, m[1] - r0.y)), d1 = transpose8x8(half2_bits(m[2] - r1.x, m[3] - r1.y));
            mma(s.acc[j][0], v0[j] & LO, v0[j] & HI, v1[j] & LO, v1[j] & HI, d0, d1);
            mma(s.acc[j][1], a & LO, a & HI, b & LO, b & HI, d0, d1);
        }
    }
}

template <int G> constexpr int PART = COLS * 32 * G + 2 * COLS;            // floats of a part in the workspace
template <int G, int NW> struct Shared {
    static constexpr int D = 32 * G;
    float o[NW][COLS][D + 4];                     // the padding spreads the heads over the banks
};
template <int G> struct Floats;
template <> struct Floats<2> { using T = float2; };
template <> struct Floats<4> { using T = float4; };
template <int G> __device__ __forceinline__ void store_o(const DecodeParams &p, int64_t at, const float (&v)[G]) {
#pragma unroll
    for (int i = 0; i < G; ++i) store_o(p, at + i, v[i]);
}

// The warps' states of a row to its output, or to a part: [COLS][D] weighted values, [COLS] references, [COLS] sums. A warp
// finishes every NW-th head, a lane G channels.
template <int G, int NW>
__device__ __forceinline__ void finish(const DecodeParams &p, State<G> &s, Shared<G, NW> &sh, float (&ref)[COLS][NW], float (&sum)[COLS][NW], int b,
                                       int first_head, int n, float *part, int warp, int lane) {
    static_assert(NW >= G, "a warp to a group of channels when queries are loaded");
    using V = typename Floats<G>::T;
    constexpr int D = 32 * G;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int d = 4; d < 32; d *= 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) s.sum[i] += __shfl_xor_sync(~0u, s.sum[i], d);
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) s.zero[j][i] += __shfl_xor_sync(~0u, s.zero[j][i], d);
    }
    if (g == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) { ref[2 * t + i][warp] = s.ref[i]; sum[2 * t + i][warp] = s.sum[i]; }
    }
    __syncthreads();                              // and the ring, whose memory `sh` is, is done with
    float f[2], back[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float top = ref[2 * t + i][0];
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, ref[2 * t + i][w]);
        f[i] = exp2_approx(s.ref[i] - top);
        back[i] = power_of_two(20 - exponent_of(s.unit[i]));                // 2^20 / unit
    }
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float *to = &sh.o[warp][2 * t + i][32 * j + 4 * g];
            const float z = s.zero[j][i], even = 16.0f * back[i];
            *reinterpret_cast<float4 *>(to) = make_float4(f[i] * fmaf(s.acc[j][0][i], even, z), f[i] * fmaf(s.acc[j][0][i + 2], back[i], z),
                                                          f[i] * fmaf(s.acc[j][1][i], even, z), f[i] * fmaf(s.acc[j][1][i + 2], back[i], z));
        }
    __syncthreads();
    for (int h = warp; h < COLS; h += NW) {
        float top = ref[h][0], all = 0.0f;
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, ref[h][w]);
#pragma unroll
        for (int w = 0; w < NW; ++w) all = fmaf(sum[h][w], exp2_approx(ref[h][w] - top), all);
        float v[G];
#pragma unroll
        for (int i = 0; i < G; ++i) v[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const V x = *reinterpret_cast<const V *>(&sh.o[w][h][lane * G]);
#pragma unroll
            for (int i = 0; i < G; ++i) v[i] += reinterpret_cast<const float *>(&x)[i];
        }
        if (part) {
            *reinterpret_cast<V *>(part + h * D + lane * G) = *reinterpret_cast<const V *>(v);
            if (lane == 0) { part[COLS * D + h] = top; part[COLS * D + COLS + h] = all; }
        } else if (h < n) {
            const float inverse = all != 0.0f ? 1.0f / all : 0.0f;
#pragma unroll
            for (int i = 0; i < G; ++i) v[i] = all != 0.0f ? v[i] * inverse : 0.0f;
            store_o(p, b * p.o_b + (first_head + h) * p.o_h + lane * G, v);
            if (lane == 0) p.lse[b * p.lse_b + first_head + h] = log_sum(top, all);
        }
    }
    __syncthreads();
}

template <int G, int NW> struct Memory {
    union {
        Shared<G, NW> sh;
        uint8_t ring[NW][STAGES][Rec<G>::BYTES];
    };
    // two blocks of eight warps stay below 196 KB, past which the first-level cache is halved (64K tokens took 1 us more); four blocks of four
    // warps are 2 KB over, and take the smaller cache
    union {
        float whole[NW][8 * G][32];
        alignas(16) float merged[PART<G>];        // of this block, where a cluster shares a row; its warps have taken theirs back
    };
    QueryMemory<G> query;
    float ref[COLS][NW], sum[COLS][NW];
};
static_assert(2 * (sizeof(Memory<4, 8>) + 1024) <= 196 * 1024, "1 KB of each block is the system's");

__device__ __forceinline__ bool too_many(const DecodeParams &p, uint32_t units, uint32_t rows) {
    const bool over = (uint64_t)units * rows >> 31;
    if (over) or_status(p.status, OMMX_ST_BAD_LENGTH);
    return over;
}
// A row of no tokens
template <int G> __device__ __forceinline__ void nothing(const DecodeParams &p, int b, int row) {
    const int cb = row % p.col_blocks, first = (row / p.col_blocks) * p.group + cb * COLS, n = min(COLS, p.group - cb * COLS);
    for (int i = threadIdx.x; i < n * 32 * G; i += blockDim.x) store_o(p, b * p.o_b + (first + i / (32 * G)) * p.o_h + i % (32 * G), 0.0f);
    if (threadIdx.x < n) p.lse[b * p.lse_b + first + threadIdx.x] = -INFINITY;
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
        for (int r = 0; r < MOST_CLUSTER; ++r)
            if (r < (int)n) {
                const float f = exp2_approx(ref[r] - top);
                all = fmaf(sum[r], f, all);
                o[0] = fmaf(v[r].x, f, o[0]); o[1] = fmaf(v[r].y, f, o[1]); o[2] = fmaf(v[r].z, f, o[2]); o[3] = fmaf(v[r].w, f, o[3]);
            }
        const float inverse = all != 0.0f ? 1.0f / all : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = all != 0.0f ? o[i] * inverse : 0.0f;
        if (lane < LANES) store_o(p, b * p.o_b + (first_head + h) * p.o_h + 4 * lane, o);
        if (lane == 0) p.lse[b * p.lse_b + first_head + h] = log_sum(top, all);
    }
    cluster_barrier();                            // no block leaves before its peers have read its part
}

template <int G, bool FINE, int NW, bool CLUSTER>
__global__ void __launch_bounds__(32 * NW, WARPS_PER_SM / NW) kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
    extern __shared__ __align__(128) uint8_t memory[];
    Memory<G, NW> &m = *reinterpret_cast<Memory<G, NW> *>(memory);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int BY = FINE ? 32 : 64;            // records to a partial sum
    const uint8_t *ring = m.ring[warp][0];
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + 16 * lane;
    const uint8_t *records = p.c.records + 16 * lane;
    wait_earlier();
    let_next_in();
    const uint32_t rows = p.c.H * p.col_blocks;
    uint32_t u, end, base = 0;                    // this block's units; units before sequence b
    uint32_t second = ~0u;                        // a row that begins here or later leaves its part in the second slot
    int b = 0, units = 0, len = 0;
    if (CLUSTER) {                                // a cluster to a row
        const uint32_t n = cluster_size(), rank = cluster_rank(), at = blockIdx.x / n;
        b = at / rows;
        len = length_of(p, b);
        units = units_of(p, len);
        if (too_many(p, units, rows)) units = 0;
        if (units == 0) {                         // for all of the cluster
            if (rank == 0) nothing<G>(p, b, at - b * rows);
            return;
        }
        u = (at - b * rows) * units;
        end = u + units * (rank + 1) / n;
        u += units * rank / n;
    } else if (p.whole) {                         // a block to a row
        b = blockIdx.x / rows;
        len = length_of(p, b);
        units = units_of(p, len);
        if (too_many(p, units, rows)) units = 0;
        u = (blockIdx.x - b * rows) * units;
        end = u + units;
        if (units == 0) { nothing<G>(p, b, blockIdx.x - b * rows); return; }
    } else {
        const Deal d = deal(p, rows, gridDim.x, lane);
        if (blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<uint2 *>(p.work) = make_uint2(d.per, d.over ? OVER : d.pieces);
        // the sequence that this block's (first) unit lies in; `at`, `base`: this block and the first of the sequence, in pieces or units
        const uint32_t at = d.pieces ? blockIdx.x : blockIdx.x * d.per;
        if (!d.pieces && at >= d.total) return;
        uint32_t before = 0;
        for (int b0 = 0;; b0 += 32) {
            if (b0 >= p.s.B) return;              // no piece for this block (or lengths past max_seq_len, more than 32 bits count)
            const int l = b0 + lane < p.s.B ? length_of(p, b0 + lane) : 0, n = units_of(p, l);
            const uint32_t v = d.pieces ? pieces_of(n, d.per) : n, sum = warp_inclusive_scan(v, lane), past = __ballot_sync(~0u, before + sum * rows > at);
            if (past) {
                const int from = __ffs(past) - 1;
                b = b0 + from;
                before += __shfl_sync(~0u, sum - v, from) * rows;
                units = __shfl_sync(~0u, n, from);
                len = __shfl_sync(~0u, l, from);
                break;
            }
            before += __shfl_sync(~0u, sum, 31) * rows;
        }
        if (d.pieces) {                           // piece `part` of `parts` of a row; units are counted from the sequence's first
            const uint32_t parts = pieces_of(units, d.per), row = (at - before) / parts, part = at - before - row * parts;
            u = row * units + (uint32_t)((uint64_t)units * part / parts);
            end = row * units + (uint32_t)((uint64_t)units * (part + 1) / parts);
        } else {
            base = before;
            second = u = at;
            end = min(u + d.per, d.total);
        }
    }
    while (CLUSTER || u < end) {
        while (u >= base + units * rows) {        // the next sequence that has any
            base += units * rows;
            len = length_of(p, ++b);
            units = units_of(p, len);
        }
        const int row = (u - base) / units, i0 = u - base - row * units, i1 = min((uint32_t)units, i0 + (end - u));
        const int head = row / p.col_blocks, cb = row % p.col_blocks;
        const int first_head = head * p.group + cb * COLS, n = min(COLS, p.group - cb * COLS);
        const int32_t *sel = p.selected ? p.selected + ((int64_t)b * p.c.H + head) * p.num_selected : nullptr;
        // 32 of the warp's records at a time are looked up by a lane each, while the 32 before are on their way: which one it is and how
        // many of its tokens are valid (0: there is none). `odd`: those of less than 16.
        const int mine = (i1 - i0 - warp + NW - 1) / NW, part_shift = p.page_shift - 4;
        auto look_up = [&](int k, uint32_t &rec, int &valid) {
            const int i = i0 + warp + (k + lane) * NW, slot = i >> part_shift, part = i & (p.c.parts - 1);
            rec = 0;                                  // a record that is not meant is fetched too, and not used
            valid = 0;
            if (i >= i1) return;
            const int place = sel ? sel[slot] : slot;
            const int64_t first = ((int64_t)place << p.page_shift) + 16 * part;
            if (place < 0 || first >= len) return;
            const int64_t page = page_id(p.s, b, place);
            if (page < 0 || page >= p.c.num_pages) { or_status(p.status, OMMX_ST_BAD_PAGE); return; }
            rec = (uint32_t)((page * p.c.H + head) * p.c.parts + part);    // below 2^32: there is no memory for more
            valid = (int)min((int64_t)16, len - first);
        };
        // `rec`, `valid`: of the AHEAD first ones, then of 32 at a time, AHEAD of those in use
        uint32_t rec, next_rec;
        int valid, next_valid, flying = 0;            // flying: valid tokens of those on their way, eight bits each, the next one lowest
        look_up(0, rec, valid);
        look_up(AHEAD, next_rec, next_valid);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (k < mine) fetch<G>(ring_at + k * Rec<G>::BYTES, records + (uint64_t)__shfl_sync(~0u, rec, k) * Rec<G>::BYTES, lane);
            flying |= __shfl_sync(~0u, valid, k) << (8 * k);
            close_group();
        }
        Query<G> q;
        State<G> s;
        load_query<G>(p, b, first_head, n, warp, lane, m.query, q);
        clear(s, m.whole[warp][0] + lane);
        // the slot in use and the one that is filled next, which is the one used before
        int read = 0, write = AHEAD * Rec<G>::BYTES;
        auto advance = [&] { write = read; read = read == AHEAD * Rec<G>::BYTES ? 0 : read + Rec<G>::BYTES; };
        for (int k0 = 0; k0 < mine; k0 += 32) {
            if (k0 % BY == 0 && k0) put_by(s);
            rec = next_rec;
            valid = next_valid;
            look_up(k0 + 32 + AHEAD, next_rec, next_valid);
            const int left = mine - k0, now = min(32, left);
            if (flying == FULL && __all_sync(~0u, valid == 16 || lane + AHEAD >= left)) {
                for (int k = 0; k < now; ++k) {
                    if (k + AHEAD < left)
                        fetch<G>(ring_at + write, records + (uint64_t)__shfl_sync(~0u, rec, k) * Rec<G>::BYTES, lane);
                    close_group();
                    fetched<AHEAD>();
                    attend<G, FINE>(p, ring + read, 16, lane, q, s);
                    advance();
                    __syncwarp();                     // before the slot is filled again
                }
            } else {
                for (int k = 0; k < now; ++k) {
                    if (k + AHEAD < left)
                        fetch<G>(ring_at + write, records + (uint64_t)__shfl_sync(~0u, rec, k) * Rec<G>::BYTES, lane);
                    close_group();
                    fetched<AHEAD>();
                    if (flying & 255) attend<G, FINE>(p, ring + read, flying & 255, lane, q, s);
                    advance();
                    flying = flying >> 8 | __shfl_sync(~0u, valid, k) << (8 * (AHEAD - 1));
                    __syncwarp();
                }
            }
        }
        fetched<0>();
        take_back(s);
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

// Where the parts of a row are: those of blocks first .. first + count - 1, the first one in its slot 1 if `late`. A whole warp calls
// it, before the wait for the first kernel: this one starts when every block of that has waited for what came earlier, so the lengths
// are there, and only the deal is not.
struct Parts { uint32_t first, count; bool late; };
__device__ __forceinline__ Parts parts_of(const DecodeParams &p, int b, uint32_t row, int lane) {
    const uint32_t rows = p.c.H * p.col_blocks, units = units_of(p, length_of(p, b)), own = lane < b ? units_of(p, length_of(p, lane)) : 0;
    wait_earlier();
    const uint2 d = *reinterpret_cast<const uint2 *>(p.work);
    uint32_t before = d.y ? pieces_of(own, d.x) : own;
    for (int i = lane + 32; i < b; i += 32) {
        const uint32_t v = units_of(p, length_of(p, i));
        before += d.y ? pieces_of(v, d.x) : v;
    }
    before = __reduce_add_sync(~0u, before) * rows;
    Parts r;
    if (units == 0 || d.y == OVER) return {0, 0, false};
    if (d.y) {
        r.count = pieces_of(units, d.x);
        r.first = before + row * r.count;
        r.late = false;
    } else {
        const uint32_t r0 = before + row * units;
        r.first = r0 / d.x;
        r.count = (r0 + units - 1) / d.x - r.first + 1;
        r.late = true;                            // the first part's block is the one that holds the row's first unit
    }
    return r;
}
template <int G> __device__ __forceinline__ const float *part_at(const DecodeParams &p, const Parts &r, int i) {
    return p.work + HEAD + (2 * (int64_t)(r.first + i) + (i == 0 && r.late)) * PART<G>;
}
template <int G> __device__ __forceinline__ void zeros(const DecodeParams &p, int b, int hq, int lane) {      // a head of no tokens
#pragma unroll
    for (int i = 0; i < G; ++i) store_o(p, b * p.o_b + hq * p.o_h + lane * G + i, 0.0f);
    if (lane == 0) p.lse[b * p.lse_b + hq] = -INFINITY;
}

// Rows of which several blocks have a part, and those of no tokens, where rows are many: a block to a row, a warp to a head, a lane
// to G channels. Grid: (rows of a sequence, sequences).
template <int G> __global__ void __launch_bounds__(32 * COLS) kv4_combine_row_kernel(const __grid_constant__ DecodeParams p) {
    using V = typename Floats<G>::T;
    constexpr int D = 32 * G;
    const int lane = threadIdx.x & 31, h = threadIdx.x >> 5, b = blockIdx.y, row = blockIdx.x;
    const int head = row / p.col_blocks, cb = row % p.col_blocks, hq = head * p.group + cb * COLS + h;
    const Parts r = parts_of(p, b, row, lane);
    let_next_in();
    if (h >= p.group - cb * COLS || r.count == 1) return;                   // not a head, or finished where it was computed
    if (r.count == 0) { zeros<G>(p, b, hq, lane); return; }
    float top = LOWEST, sum = 0.0f, o[G];
#pragma unroll
    for (int i = 0; i < G; ++i) o[i] = 0.0f;
    for (int i0 = 0; i0 < (int)r.count; i0 += 4) {
        V v[4];
        float ref[4], add[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool on = i0 + u < (int)r.count;
            const float *part = part_at<G>(p, r, on ? i0 + u : i0);
            v[u] = reinterpret_cast<const V *>(part + h * D)[lane];
            ref[u] = on ? part[COLS * D + h] : LOWEST;
            add[u] = on ? part[COLS * D + COLS + h] : 0.0f;
        }
        const float next = fmaxf(fmaxf(fmaxf(ref[0], ref[1]), fmaxf(ref[2], ref[3])), top), keep = exp2_approx(top - next);
        sum *= keep;
#pragma unroll
        for (int i = 0; i < G; ++i) o[i] *= keep;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u < (int)r.count) {
                const float f = exp2_approx(ref[u] - next);
                sum = fmaf(add[u], f, sum);
#pragma unroll
                for (int i = 0; i < G; ++i) o[i] = fmaf(reinterpret_cast<const float *>(&v[u])[i], f, o[i]);
            }
        top = next;
    }
    const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < G; ++i) o[i] = sum != 0.0f ? o[i] * inverse : 0.0f;
    store_o(p, b * p.o_b + hq * p.o_h + lane * G, o);
    if (lane == 0) p.lse[b * p.lse_b + hq] = log_sum(top, sum);
}

// The same where rows are few and their parts many: a block to a head. The references and sums of all parts are read at once; then a
// warp takes every CW-th part, UNROLL of them on their way. Grid: (rows of a sequence x COLS, sequences).
constexpr int CW = 8, UNROLL = 5;
template <int G> __global__ void __launch_bounds__(32 * CW) kv4_combine_head_kernel(const __grid_constant__ DecodeParams p) {
    constexpr int D = 32 * G;
    using V = typename Floats<G>::T;
    __shared__ float so[CW][D], weight[MOST_PARTS], sr[CW], ss[CW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.y, row = blockIdx.x / COLS, h = blockIdx.x % COLS;
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
        const float ref = part[COLS * D + h], s = part[COLS * D + COLS + h], m = fmaxf(top, ref);
        weight[i] = ref;
        sum = fmaf(s, exp2_approx(ref - m), sum * exp2_approx(top - m));
        top = m;
    }
#pragma unroll
    for (int d = 16; d; d /= 2) {
        const float ref = __shfl_xor_sync(~0u, top, d), s = __shfl_xor_sync(~0u, sum, d), m = fmaxf(top, ref);
        sum = fmaf(s, exp2_approx(ref - m), sum * exp2_approx(top - m));
        top = m;
    }
    if (lane == 0) { sr[warp] = top; ss[warp] = sum; }
    __syncthreads();
    top = sr[0];
#pragma unroll
    for (int w = 1; w < CW; ++w) top = fmaxf(top, sr[w]);
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < CW; ++w) sum = fmaf(ss[w], exp2_approx(sr[w] - top), sum);
    float o[G];
#pragma unroll
    for (int i = 0; i < G; ++i) o[i] = 0.0f;
    for (int i0 = warp; i0 < n; i0 += CW * UNROLL) {
        if (i0 != warp) load(i0);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (i0 + u * CW < n) {
                const float f = exp2_approx(weight[i0 + u * CW] - top);
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
        store_o(p, b * p.o_b + hq * p.o_h + c, sum != 0.0f ? x / sum : 0.0f);
    }
    if (threadIdx.x == 0) p.lse[b * p.lse_b + hq] = log_sum(top, sum);
}

// ---- host ---------------------------------------------------------------------------------------
static int64_t most_blocks(int warps) {
    const int n = WARPS_PER_SM / warps * sm_count();
    return n < MOST_PARTS ? n : MOST_PARTS;
}
static int64_t workspace_floats(int head_dim) {
    const int64_t part = head_dim == 64 ? PART<2> : PART<4>;
    return HEAD + 2 * part * most_blocks(4);
}

template <int G, bool FINE, int NW, bool CLUSTER> static int launch_decode(const DecodeParams &p, int64_t blocks, int cluster, cudaStream_t st) {
    static std::atomic<uint64_t> allowed{0};      // devices on which the kernel may take its shared memory
    int dev = 0;
    if (int rc = current_device(&dev)) return rc;
    if (!(allowed.load(std::memory_order_acquire) >> dev & 1)) {
        OMMX_CUDA_TRY(cudaFuncSetAttribute(kv4_decode_kernel<G, FINE, NW, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Memory<G, NW>)));
        allowed.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (int rc = launch_dependent(kv4_decode_kernel<G, FINE, NW, CLUSTER>, dim3((unsigned)blocks), 32 * NW, sizeof(Memory<G, NW>), st, cluster, p)) return rc;
    if (p.whole || CLUSTER) return 0;
    // a row has some blocks / rows parts
    const int rows = p.c.H * p.col_blocks;
    if ((int64_t)rows * p.s.B * COLS >= blocks) return launch_dependent(kv4_combine_row_kernel<G>, dim3(rows, p.s.B), 32 * COLS, 0, st, 1, p);
    return launch_dependent(kv4_combine_head_kernel<G>, dim3(rows * COLS, p.s.B), 32 * CW, 0, st, 1, p);
}

// records that a row of the call can have
static int64_t most_units(const ommx_kv4_decode_args *a) {
    const int64_t parts = a->cache.page_size / 16;
    int64_t n = a->seqs.pages_per_seq * parts;
    if (a->max_seq_len > 0) n = n < (a->max_seq_len + 15LL) / 16 ? n : (a->max_seq_len + 15LL) / 16;
    if (a->selected) n = n < a->num_selected * parts ? n : a->num_selected * parts;
    return n;
}
static int64_t workspace_floats(const ommx_kv4_decode_args *a) { return most_units(a) <= WHOLE ? 0 : workspace_floats(a->cache.head_dim); }

static int decode(const ommx_kv4_decode_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv4_decode: null args");
    DecodeParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv4_decode", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv4_decode", a->seqs, p.c, &p.s)) return rc;
    if (a->q_dtype != OMMX_DT_BF16 && a->q_dtype != OMMX_DT_F16) return fail(OMMX_E_UNSUPPORTED, "kv4_decode: q must be bfloat16 or float16");
    if (a->o_dtype != OMMX_DT_F32 && a->o_dtype != OMMX_DT_BF16 && a->o_dtype != OMMX_DT_F16) return fail(OMMX_E_ARG, "kv4_decode: o dtype %d", a->o_dtype);
    if (a->n_q_heads < p.c.H || a->n_q_heads % p.c.H)
        return fail(OMMX_E_UNSUPPORTED, "kv4_decode: %d query heads are not a multiple of %d kv heads", a->n_q_heads, p.c.H);
    if (!(a->logit_cap >= 0.0f) || !std::isfinite(a->logit_cap)) return fail(OMMX_E_ARG, "kv4_decode: logit_cap must be finite and not negative");
    if (!std::isfinite(a->sm_scale)) return fail(OMMX_E_ARG, "kv4_decode: sm_scale must be finite");
    if (a->selected && a->num_selected < 0) return fail(OMMX_E_ARG, "kv4_decode: num_selected must not be negative");
    if (p.s.B > 65535) return fail(OMMX_E_UNSUPPORTED, "kv4_decode: a batch of %d", p.s.B);
    if (p.s.B == 0) return 0;
    if (!a->q || !a->o || !a->lse) return fail(OMMX_E_ARG, "kv4_decode: q, o and lse must not be null");
    const int64_t need = workspace_floats(a);
    if (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_floats < need))
        return fail(OMMX_E_ARG, "kv4_decode: workspace must be 16-byte aligned and hold %lld floats", (long long)need);
    p.q = a->q; p.q16 = a->q_dtype == OMMX_DT_F16; p.q_b = a->q_stride_b; p.q_h = a->q_stride_h;
    p.q_wide = (reinterpret_cast<uintptr_t>(a->q) | (uintptr_t)(2 * p.q_b) | (uintptr_t)(2 * p.q_h)) % 16 == 0;
    p.o = a->o; p.o_type = a->o_dtype; p.o_b = a->o_stride_b; p.o_h = a->o_stride_h;
    p.lse = a->lse; p.lse_b = a->lse_stride_b;
    p.work = a->workspace;
    p.selected = a->selected; p.num_selected = a->num_selected;
    p.group = a->n_q_heads / p.c.H; p.col_blocks = (p.group + COLS - 1) / COLS;
    p.page_shift = shift_of(p.c.page);
    p.sm_scale = a->sm_scale; p.status = a->status;
    p.cap = a->logit_cap <= 0x1p126f ? a->logit_cap : 0.0f;                 // past that it changes no logit, and is infinite in powers of two
    if (p.c.num_pages == 0) return fail(OMMX_E_ARG, "kv4_decode: a cache of no pages");   // what is fetched for a page that is not there
    // as many blocks as the SMs hold, no more than the work can have
    const int64_t units = most_units(a);
    const int64_t rows = (int64_t)p.s.B * p.c.H * p.col_blocks;
    if (units * rows >= 1LL << 31 || rows * COLS >= 1LL << 31)
        return fail(OMMX_E_UNSUPPORTED, "kv4_decode: %lld rows of up to %lld records (2^31 in all are counted): give max_seq_len", (long long)rows, (long long)units);
    // Blocks of eight warps where rows are few, so that a row has few parts, of four where they are many: then blocks often go on from
    // one row to the next, and an SM's others work meanwhile (64 sequences of 200..2000 tokens, 8 kv heads: 43 us with four, 54 with
    // eight; one of 64K: 25.4 and 24.4). As many blocks as the SMs hold, no more than the work can have. Rows that are short for
    // certain go whole to a block each, and the second kernel is not needed.
    const int warps = rows >= 64 ? 4 : 8;
    p.least = 2 * warps;
    const int64_t most = (units * rows + p.least - 1) / p.least, hold = most_blocks(warps);
    // Rows of middling length, and few, go to a cluster of eight-warp blocks each, as many as fit at once: no second kernel
    // (4096 tokens, 8 kv heads: 10.4 us with two, 8.3 with clusters; past 256 records the blocks that stay idle cost more)
    int cluster = 1;
    while (cluster < MOST_CLUSTER && 2 * cluster * rows <= most_blocks(8)) cluster *= 2;
    if (units > 32 * cluster) cluster = 1;
    p.whole = units <= WHOLE / 2 || (units <= WHOLE && cluster == 1);       // 333 tokens: 6.9 us whole, 6.4 in clusters; 100: 5.2
    if (p.whole) cluster = 1;
    const int64_t blocks = p.whole ? rows : cluster > 1 ? cluster * rows : most < 1 ? 1 : most < hold ? most : hold;
    auto launch = [&](auto g, auto fine) {
        constexpr int G = decltype(g)::value;
        constexpr bool FINE = decltype(fine)::value;
        if (cluster > 1) return launch_decode<G, FINE, 8, true>(p, blocks, cluster, st);
        return warps == 4 ? launch_decode<G, FINE, 4, false>(p, blocks, 1, st) : launch_decode<G, FINE, 8, false>(p, blocks, 1, st);
    };
    using std::integral_constant;
    if (a->o_dtype == OMMX_DT_BF16)
        return a->cache.head_dim == 128 ? launch(integral_constant<int, 4>(), std::false_type()) : launch(integral_constant<int, 2>(), std::false_type());
    return a->cache.head_dim == 128 ? launch(integral_constant<int, 4>(), std::true_type()) : launch(integral_constant<int, 2>(), std::true_type());
}

}  // namespace kv4
}  // namespace ommx

extern "C" int64_t ommx_b200_kv4_decode_workspace_floats(const ommx_kv4_decode_args *args) {
    return !args || (args->cache.head_dim != 64 && args->cache.head_dim != 128) ? 0 : ommx::kv4::workspace_floats(args);
}
extern "C" int64_t ommx_b200_kv4_workspace_floats(int32_t head_dim) { return head_dim == 64 || head_dim == 128 ? ommx::kv4::workspace_floats(head_dim) : 0; }
extern "C" int ommx_b200_kv4_decode(const ommx_kv4_decode_args *args, void *stream) { return ommx::kv4::decode(args, (cudaStream_t)stream); }
