// How the 8-bit cache's attention deals its work out, and where a row's parts are.  P: a kernel's parameters, with s.B, c.H, col_blocks, least,
// work and status, for which length_of(p, b) and units_of(p, length) say how many units sequence b has.
#pragma once

#include "ommx_kv8.cuh"

namespace ommx {
namespace kv8 {

// Units are records (16 tokens of a kv head, for a block of its query heads); a row (sequence, kv head, block of heads) is a run of
// them. Lengths are known on the device alone, so every block works the same deal out, and leaves it for the second kernel:
// * a block to a row, where the host knows that rows are short (`whole`), or a cluster of blocks, which exchange their parts themselves;
// * else every row is cut into pieces of at most `per` units, a block to a piece, with the smallest `per` for which there are blocks
//   enough;
// * or, where that would leave a block with over BEGIN units more than an even share, all rows end to end are cut into such shares,
//   whatever rows they touch. A second piece costs a block some 4 us, half of it hidden by the SM's other blocks. us with pieces only up to 0, 16, 32, 64
//   and 256 units above an even share, and always: 8 x 64K tokens, 8 kv heads 206, 183, 180, 181, 181, 179; 64 sequences of 200 to 2000 44, 42, 42, 39, 39,
//   39; 100 of 500 to 4000, 2 kv heads 39.5, then 30; 61 of 300 to 20000 159 up to 256, always 179; 32, 40 and 20 ragged ones within 3 %.
// A piece that is a whole row is finished where it is computed; the others' parts meet in the second kernel. A block has at most two
// of those, of the row that an earlier block began (its slot 0) and of the one that a later block goes on with (slot 1).
constexpr uint32_t OVER = 2;                      // in the deal's place: there is none
constexpr int BEGIN = 64, HEAD = 4;               // HEAD: floats in front of the parts, which hold the deal
struct Deal { uint32_t per, total; bool pieces, over; };   // over: lengths far past max_seq_len, of more units than 32 bits count
// units / per, rounded up. Shares are no smaller than an even one, so quotients are at most as many as there are blocks, and one in 32 bits that is
// put right by one is enough: the search below took 1.5 us with divisions, 0.5 so.
__device__ __forceinline__ uint32_t pieces_of(uint32_t units, uint32_t per) {
    const uint32_t n = units + per - 1;
    const uint32_t q = (uint32_t)__fdividef((float)n, (float)per);
    const int32_t rest = (int32_t)(n - q * per);
    return rest < 0 ? q - 1 : rest >= (int32_t)per ? q + 1 : q;
}
// The lengths of the first 64 sequences, two to a lane of each warp, and their units
struct Lengths { int len[2]; uint32_t units[2]; };
template <typename P> __device__ __forceinline__ Lengths lengths_of(const P &p, int lane) {
    Lengths l;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int b = lane + 32 * i;
        l.len[i] = b < p.s.B ? length_of(p, b) : 0;
        l.units[i] = b < p.s.B ? units_of(p, l.len[i]) : 0;
    }
    return l;
}
// All warps of a block call it. `shared`: a word for each.
template <typename P> __device__ __forceinline__ Deal deal(const P &p, const Lengths &own, uint32_t rows, uint32_t blocks, int lane, int warp, int warps, uint32_t *shared) {
    uint64_t sum = (uint64_t)own.units[0] + own.units[1];
    uint32_t some = (own.units[0] > 0) + (own.units[1] > 0), most = max(own.units[0], own.units[1]);
    for (int b = lane + 64; b < p.s.B; b += 32) {
        const uint32_t n = units_of(p, length_of(p, b));
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
    // Pieces of `per` take total / per + full blocks at most; fewer may do. Each warp tries one of as many sizes between, and the range is cut to
    // the one before the smallest that will do (one size after the other: 1.0 us of 32 sequences, 1.7 of 61; so 0.4).
    uint32_t lo = even, hi = min(max(most, even), full < blocks ? max(even, d.total / (blocks - full) + 1) : 0xFFFFFFFFu);
#pragma unroll 1
    for (int span = 1; span < 64 && lo < hi; span *= warps) {
        const uint32_t step = (hi - lo + warps - 1) / warps, per = lo + warp * step;        // the first is `lo`
        uint32_t n = pieces_of(own.units[0], per) + pieces_of(own.units[1], per);
        for (int b = lane + 64; b < p.s.B; b += 32) n += pieces_of(units_of(p, length_of(p, b)), per);
        n = __reduce_add_sync(~0u, n);
        if (lane == 0) shared[warp] = n * rows <= blocks && per < hi;
        __syncthreads();
        const uint32_t fits = __ballot_sync(~0u, lane < warps && shared[lane]);
        const int first = fits ? __ffs(fits) - 1 : warps;
        if (fits) hi = lo + first * step;
        if (first) lo = min(lo + (first - 1) * step + 1, hi);
        __syncthreads();
    }
    if (hi <= even + BEGIN) { d.per = hi; d.pieces = true; }
    return d;
}

// Where the parts of a row are: those of blocks first .. first + count - 1, the first one in its slot 1 if `late`. A whole warp calls
// it, before the wait for the first kernel: this one starts when every block of that has waited for what came earlier, so the lengths
// are there, and only the deal is not.
struct Parts { uint32_t first, count; bool late; };
template <typename P> __device__ __forceinline__ Parts parts_of(const P &p, int b, uint32_t row, int lane) {
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

}  // namespace kv8
}  // namespace ommx
