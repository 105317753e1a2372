// The 8-bit cache: eviction by what tokens were attended to with.
//
// Of a sequence of more than `budget` tokens each kv head keeps the first `sinks`, the last `recent` and, of those between, the ones of the
// largest weight (ties to the lowest place), and they move to the places 0 .. budget - 1 in their order. A cluster of blocks to a row
// (sequence, kv head):
// * picks: the weights' order is that of whole numbers, of which the want-th largest is found by counting: those above 0 (all, where it is none of
//   these) are cut into 2048 equal parts, and the part that holds it again, until so few are left that each block takes all of them and goes on
//   alone. A thread holds its first keys in registers; counts meet in distributed shared memory.
// * moves: places ascend, and a token never moves up. So once a cluster has read all that a stretch of places takes into its shared
//   memory it can write that stretch where the tokens lie, and go on to the next.
// What bounds it: where rows are many what moves (64 sequences of 4608 to 4096 tokens, 8 kv heads 210 us; 1.1 GB there and back take 165 of a copy's rate),
// where they are few the chain: 64K to 4096 tokens, 8 kv heads 26 us in graph replays (19 MB are 2.9), of which reading weights takes 2, the first count and its
// exchange 4.5, the rest of the choice 5, the list 3 and the move 6.5, on 64 of the SMs, since a cluster has eight blocks at most. Short rows are the same
// chain (700 to 500 tokens 14.4 us). Of 8 x 64K to 4096 (68 us, 23.6 in bytes) a block has 32K keys, which pass through shared memory again at
// each count and in the list.
#include "ommx_kv8.cuh"
#include "ommx_kv_device.cuh"

namespace ommx {
namespace kv8 {

using namespace kv;

// Blocks of 1024 threads, one to an SM, or of 512, two to an SM: where there are more rows than SMs, since they fill each other's waits (64 sequences of 4608
// to 4096 tokens, 8 kv heads: 259 us with one size, 228 so when that was done), and for rows of up to SHORT tokens, whose blocks wait for barriers (4
// sequences of 300 to 200 tokens, 4 kv heads 12.3 us with 1024 and 11.5 with 512; one of 700 to 500 14.4 and 14.6).
constexpr int BINS = 2048, MOST_CLUSTER = 8, SHORT = 640;
constexpr int HELD = 8;                           // keys that a thread holds, of consecutive tokens of a page; TURN: a block's turn of keys
constexpr int LOWEST_BIN = (1 << 30) - 1;         // what the lowest part, which is not counted, is taken to hold
constexpr int FEW = 4096;                         // keys that each block of a cluster finishes for itself
template <int THREADS> struct Sizes {
    static constexpr int TURN = THREADS * HELD;
    static constexpr int PLACES = THREADS / 2;    // that a block moves at a time
    static constexpr int MOST_KEYS = 36 * THREADS;                          // further keys that a block holds in shared memory; it reads others again
};
constexpr int MOST_TOKENS = (1 << 30) - (1 << 16);  // a count of them and one that stands for all (LOWEST_BIN) fit into 32 bits together

struct EvictParams {
    Cache c;
    Seqs s, to;                                   // `to`: where kept tokens go; only its table
    int32_t *kept, *len_out;
    int32_t budget, sinks, recent, keys, page_shift, in_place;              // keys: behind its first turn that a block holds
    int32_t *status;
};
// row `at` of a sequence's kv head: 16 to a record. Below 2^32: there is no memory for more
__device__ __forceinline__ uint32_t row_of(const EvictParams &p, int64_t page, int head, int at) {
    return (uint32_t)((page * p.c.H + head) * p.c.page) + (at & (p.c.page - 1));
}
// weights as whole numbers in their order; NaN comes last, and zeros are one
__device__ __forceinline__ uint32_t ordered(float w) {
    const uint32_t b = __float_as_uint(w + 0.0f);
    return w != w ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint32_t peer_word(const void *at, uint32_t rank) {
    return __float_as_uint(peer_float((uint32_t)__cvta_generic_to_shared(at), rank));
}

// What a block knows of the places that it moves
struct Place { uint32_t from, to; float weight; uint16_t own, scales; };    // rows; exponents of what it takes, and of its record

__device__ __forceinline__ int peer_half(const uint16_t *at, uint32_t rank) {
    uint32_t there;
    uint16_t v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(rank));
    asm volatile("ld.shared::cluster.u16 %0, [%1];" : "=h"(v) : "r"(there) : "memory");
    return v;
}

// Grid: (cluster x H, B).
template <int G, bool E4M3, int THREADS> __global__ void __launch_bounds__(THREADS, 1024 / THREADS) kv8_evict_kernel(const __grid_constant__ EvictParams p) {
    constexpr int D = 32 * G, TURN = Sizes<THREADS>::TURN, PLACES = Sizes<THREADS>::PLACES;
    constexpr int EACH = BINS / THREADS;          // bins of a thread
    extern __shared__ __align__(16) uint8_t memory[];                       // keys, then rows
    uint32_t *keys = reinterpret_cast<uint32_t *>(memory);
    __shared__ __align__(16) int histograms[2][BINS];                       // the one of a round is read by peers until the next round's barrier
    __shared__ uint32_t few[FEW];
    __shared__ Place places[PLACES];
    __shared__ int warp_sum[2][32], starts[MOST_CLUSTER + 1], bin, left, inside, listed, more, same, above_here, equal_here, first_place, bad, spoilt;
    __shared__ int firsts[MOST_CLUSTER];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t n = cluster_size(), rank = cluster_rank();
    const int head = blockIdx.x / n, b = blockIdx.y;
    if (tid == 0) bad = listed = more = 0;
    if (tid < 64) warp_sum[tid / 32][tid % 32] = 0;                         // of warps that there are not
    auto clear = [&](int *histogram) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) histogram[tid + i * THREADS] = 0;
    };
    clear(histograms[0]);
    clear(histograms[1]);
    wait_earlier();
    let_next_in();
    const int given = p.s.len[b];
    const int64_t room = min((int64_t)p.s.max_pages << p.page_shift, (int64_t)MOST_TOKENS);
    int faults = given < 0 || given > room ? OMMX_ST_BAD_LENGTH : 0;
    const int len = faults ? 0 : given, keep = min(len, p.budget);
    if (keep > (int64_t)p.to.max_pages << p.page_shift) faults |= OMMX_ST_BAD_LENGTH;
    __syncthreads();
    const bool all = len <= p.budget;
    int32_t *out = p.kept + ((int64_t)b * p.c.H + head) * p.budget;
    auto there = [&](int64_t id) { return id >= 0 && id < p.c.num_pages; };
    // A sequence whose pages are not all there stays as it is, for all of its heads: every block looks at some, and hears of the others'
    if (!faults) {
        bool off = false;
        for (int i = rank * THREADS + tid; (int64_t)i << p.page_shift < keep; i += n * THREADS) off |= !there(page_id(p.to, b, i));
        if (all)
            for (int i = rank * THREADS + tid; (int64_t)i << p.page_shift < len; i += n * THREADS) off |= !there(page_id(p.s, b, i));
        if (off) bad = 1;
    }
    auto hear = [&] {                             // behind a barrier of the cluster
        if (warp == 0) {
            const bool off = __any_sync(~0u, lane < (int)n && peer_word(&bad, lane % n) != 0);
            if (lane == 0) spoilt = off;
        }
    };
    auto leave = [&](bool listed) {               // the list and the length of a sequence that is not evicted from
        if (rank == 0 && tid == 0) {
            if (faults) or_status(p.status, faults);
            if (head == 0 && p.len_out) p.len_out[b] = faults ? given : keep;
        }
        if (listed)
            for (int64_t i = rank * THREADS + tid; i < p.budget; i += n * THREADS) out[i] = !faults && i < len ? (int)i : -1;
    };
    if (faults) { leave(true); return; }
    const int share = ((len + (int)n - 1) / (int)n + 31) & ~31;
    const bool short_row = share <= TURN;         // a block lists its tokens in shared memory, behind the rows; else the list is the caller's
    uint16_t *list = reinterpret_cast<uint16_t *>(memory + PLACES * 2 * D);
    if (all) {
        __syncthreads();
        cluster_barrier();
        hear();
        cluster_barrier();
        if (spoilt) faults = OMMX_ST_BAD_PAGE;
        leave(true);
        if (faults || p.in_place) return;
    } else {
        // block `rank` has the keys lo .. hi - 1; first .. last - 1 of them are not kept anyway
        const int lo = min(len, (int)rank * share), hi = min(len, lo + share);
        const int first = max(lo, p.sinks), last = min(hi, len - p.recent);
        const float *weight = p.c.weight;
        auto load = [&](int i) {
            const int64_t page = page_id(p.s, b, i >> p.page_shift);
            return there(page) ? ordered(weight[row_of(p, page, head, i)]) : 0u;
        };
        auto place = [&](int turn, int u) { return lo + turn * TURN + tid * HELD + u; };      // `lo` is a multiple of 32
        const int turns = (hi - lo + TURN - 1) / TURN;
        uint32_t held[HELD];
        bool off = false;
        for (int turn = 0; turn < turns; ++turn) {
            const int i0 = place(turn, 0);
            float4 w[HELD / 4];
#pragma unroll
            for (int u = 0; u < HELD / 4; ++u) w[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i0 < hi) {
                const int64_t page = page_id(p.s, b, i0 >> p.page_shift);
                off |= !there(page);
                if (there(page)) {                // tokens behind the last one lie on its page too
#pragma unroll
                    for (int u = 0; u < HELD / 4; ++u) w[u] = *reinterpret_cast<const float4 *>(weight + row_of(p, page, head, i0) + 4 * u);
                }
            }
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
                const uint32_t k = ordered(u % 4 == 0 ? w[u / 4].x : u % 4 == 1 ? w[u / 4].y : u % 4 == 2 ? w[u / 4].z : w[u / 4].w);
                const int i = place(turn, u) - lo - TURN;
                if (turn == 0) held[u] = k;
                else if (i < hi - lo - TURN && i < p.keys) keys[i] = k;
            }
        }
        auto key_at = [&](int i) { return i - lo - TURN < p.keys ? keys[i - lo - TURN] : load(i); };      // behind the first turn
        // of `held`, a bit each: those that there are, and those that are not kept anyway
        uint32_t have = 0, live = 0;
#pragma unroll
        for (int u = 0; u < HELD; ++u) {
            have |= (uint32_t)(place(0, u) < hi) << u;
            live |= (uint32_t)(place(0, u) >= first && place(0, u) < last) << u;
        }
        const bool any_held = __any_sync(~0u, have != 0);                   // warps of a short row have none
        // f(key) for each of the thread's keys that is not kept anyway
        auto each_key = [&](auto f) {
            if (any_held) {
#pragma unroll
                for (int u = 0; u < HELD; ++u)
                    if (live >> u & 1) f(held[u]);
            }
            for (int turn = 1; turn < turns; ++turn)
                for (int u = 0; u < HELD; ++u)
                    if (place(turn, u) >= first && place(turn, u) < last) f(key_at(place(turn, u)));
        };
        if (off) bad = 1;
        __syncthreads();
        // The want-th largest of the keys from `a` on, below a + 2^width. First of those above 0, all others taken for the lowest of them; of all
        // where it is one of these.
        constexpr uint32_t ZERO = 0x80000000u;
        const int wanted = p.budget - p.sinks - p.recent;
        int want = wanted, width = 31;
        uint32_t a = ZERO;
        bool placed = false;                      // the block knows where its first token goes
        int *histogram = histograms[0], *other = histograms[1];             // `other`: all zeros but while peers read it
        for (bool begun = false; width > 0; begun = true) {
            const int shift = max(0, width - 11);
            // the lowest part is not counted: what is not above it is in it, and often it is the one that most are in
            each_key([&](uint32_t key) {
                const uint32_t k = key - a;
                if (key >= a && (width == 32 || k >> width == 0) && k >> shift) atomicAdd(&histogram[k >> shift], 1);
            });
            __syncthreads();
            cluster_barrier();
            if (!begun) hear();
            else clear(other);
            // from the top: thread t has bins BINS - 1 - 4 t and the three below
            int4 mine = make_int4(0, 0, 0, 0);
            if (tid < BINS / 4) {
                const uint32_t at = (uint32_t)__cvta_generic_to_shared(&histogram[BINS - 4 - 4 * tid]);
                float4 v[MOST_CLUSTER];
#pragma unroll
                for (int r = 0; r < MOST_CLUSTER; ++r) v[r] = r < (int)n ? peer_float4(at, r) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int r = 0; r < MOST_CLUSTER; ++r) {
                    mine.x += __float_as_int(v[r].x); mine.y += __float_as_int(v[r].y); mine.z += __float_as_int(v[r].z); mine.w += __float_as_int(v[r].w);
                }
                if (tid == BINS / 4 - 1) mine.x = LOWEST_BIN;
            }
            const int sum = mine.x + mine.y + mine.z + mine.w;
            int before = warp_inclusive_scan(sum, lane);
            if (lane == 31) warp_sum[0][warp] = before;
            __syncthreads();
            before += __reduce_add_sync(~0u, lane < warp ? warp_sum[0][lane] : 0) - sum;
            if (before < want && before + sum >= want) {                    // one thread, but where none is wanted
                const int up[4] = {mine.w, mine.z, mine.y, mine.x};
                int j = 0;
                while (before + up[j] < want) before += up[j++];
                left = want - before;
                inside = up[j];
                bin = BINS - 1 - 4 * tid - j;
            }
            __syncthreads();
            if (!begun && spoilt) {
                cluster_barrier();                // all peers have read
                faults = OMMX_ST_BAD_PAGE;
                break;
            }
            if (wanted == 0) { a = ~0u; break; }
            if (!begun && bin == 0) { a = 0; width = 32; }                  // `want` as it was
            else { a += (uint32_t)bin << shift; want = left; width = shift; }
            if (width > 0 && inside <= FEW) {     // all blocks say so
                int over = 0;                     // keys above those
                each_key([&](uint32_t key) {
                    if ((key - a) >> width == 0) few[atomicAdd(&listed, 1)] = key;
                    else over += key > a;
                });
                over = __reduce_add_sync(~0u, over);
                if (lane == 0 && over) atomicAdd(&more, over);
                __syncthreads();
                cluster_barrier();
                if (warp == 0) {
                    const int mine = lane < (int)n ? (int)peer_word(&listed, lane % n) : 0, sum = warp_inclusive_scan(mine, lane);
                    if (lane < MOST_CLUSTER) starts[lane + 1] = sum;
                    if (lane == 0) starts[0] = 0;
                }
                if (warp == 1) {                  // what the blocks before this one keep whatever the last key is
                    const int r = lane, from = min(len, r * share), to = min(len, from + share);
                    const int pinned = to - from - max(0, min(to, len - p.recent) - max(from, p.sinks));
                    const int sure = __reduce_add_sync(~0u, r < (int)rank ? (int)peer_word(&more, r % n) + pinned : 0);
                    if (lane == 0) above_here = sure;
                    if (lane == 1) equal_here = 0;
                }
                __syncthreads();
                const int count = starts[n];
                uint32_t k[FEW / THREADS];
#pragma unroll
                for (int j = 0; j < FEW / THREADS; ++j) {
                    const int i = tid + j * THREADS;
                    int r = 0;
                    while (r + 1 < (int)n && i >= starts[r + 1]) ++r;
                    k[j] = i < count ? peer_word(&few[i - starts[r]], r) - a : 0u;
                }
                while (width > 0) {
                    const int cut = max(0, width - 11);
#pragma unroll
                    for (int j = 0; j < FEW / THREADS; ++j)
                        if (tid + j * THREADS < count && k[j] >> width == 0) atomicAdd(&other[k[j] >> cut], 1);
                    __syncthreads();
                    // from the top: thread t has bins BINS - 1 - EACH t and those below
                    int mine[EACH], all_mine = 0;
#pragma unroll
                    for (int j = 0; j < EACH; ++j) { mine[j] = other[BINS - 1 - EACH * tid - j]; all_mine += mine[j]; }
                    int over = warp_inclusive_scan(all_mine, lane);
                    if (lane == 31) warp_sum[0][warp] = over;
                    __syncthreads();
                    over += __reduce_add_sync(~0u, lane < warp ? warp_sum[0][lane] : 0) - all_mine;
                    if (over < want && over + all_mine >= want) {
                        bool found = false;
#pragma unroll
                        for (int j = 0; j < EACH; ++j) {
                            if (!found && over + mine[j] >= want) { found = true; left = want - over; bin = BINS - 1 - EACH * tid - j; }
                            over += mine[j];
                        }
                    }
                    clear(other);
                    __syncthreads();
                    const uint32_t from = (uint32_t)bin << cut;
#pragma unroll
                    for (int j = 0; j < FEW / THREADS; ++j) k[j] -= from;   // what was below wraps around, and is out of reach
                    a += from;
                    want = left;
                    width = cut;
                    __syncthreads();
                }
                // and of these few: what is left of a key is by how much it is above the last one
                int m = 0, e = 0;
#pragma unroll
                for (int j = 0; j < FEW / THREADS; ++j) {
                    const bool theirs = tid + j * THREADS < starts[rank];
                    m += theirs && (int)k[j] > 0;
                    e += theirs && k[j] == 0;
                }
                m = __reduce_add_sync(~0u, m);
                e = __reduce_add_sync(~0u, e);
                if (lane == 0 && m) atomicAdd(&above_here, m);
                if (lane == 0 && e) atomicAdd(&equal_here, e);
                placed = true;
                break;
            }
            __syncthreads();
            int *const t = histogram;
            histogram = other;
            other = t;
        }
        leave(faults);
        if (faults) return;
        // keys above `a`, and the first `want` equal to it, in order: by turns and threads. Counts of both are summed in the halves of a word.
        uint32_t ms, es;                          // of a thread's keys of a turn, a bit each
        auto look = [&](int turn) {
            ms = es = 0;
            if (turn == 0) {
                if (any_held) {
#pragma unroll
                    for (int u = 0; u < HELD; ++u) {
                        ms |= (uint32_t)(held[u] > a) << u;
                        es |= (uint32_t)(held[u] == a) << u;
                    }
                    ms = (ms & live) | (have & ~live);
                    es &= live;
                }
            } else {
#pragma unroll
                for (int u = 0; u < HELD; ++u) {
                    const int i = place(turn, u);
                    const uint32_t k = i >= hi ? 0u : key_at(i);
                    const bool pinned = i < p.sinks || i >= len - p.recent;
                    ms |= (uint32_t)(i < hi && (pinned || k > a)) << u;
                    es |= (uint32_t)(i < hi && !pinned && k == a) << u;
                }
            }
            return __popc(ms) | __popc(es) << 16;
        };
        int above = 0, equal = 0;
        for (int turn = turns - 1; turn > 0; --turn) {                      // the first turn's bits stay
            const int c = look(turn);
            above += __reduce_add_sync(~0u, c & 0xFFFF);
            equal += __reduce_add_sync(~0u, c >> 16);
        }
        const int counts = look(0), scanned = warp_inclusive_scan(counts, lane);
        if (lane == 31) { warp_sum[0][warp] = above + (scanned & 0xFFFF); warp_sum[1][warp] = equal + (scanned >> 16); }
        __syncthreads();
        if (!placed) {
            if (warp == 0) {
                const int m = __reduce_add_sync(~0u, warp_sum[0][lane]), e = __reduce_add_sync(~0u, warp_sum[1][lane]);
                if (lane == 0) { more = m; same = e; }
            }
            __syncthreads();
            cluster_barrier();
            if (warp == 0) {
                const int m = __reduce_add_sync(~0u, lane < (int)rank ? (int)peer_word(&more, lane % n) : 0);
                const int e = __reduce_add_sync(~0u, lane < (int)rank ? (int)peer_word(&same, lane % n) : 0);
                if (lane == 0) { above_here = m; equal_here = e; }
            }
            __syncthreads();
        }
        int above_all = above_here, equal_all = equal_here;
        const int first_here = above_all + min(equal_all, want);
        if (tid == 0) first_place = first_here;
        for (int turn = 0; turn < turns; ++turn) {
            const int c = turn > 0 ? look(turn) : counts, scan = turn > 0 ? warp_inclusive_scan(c, lane) : scanned;
            if (turns > 1) {
                __syncthreads();                  // `warp_sum` is read
                if (lane == 31) { warp_sum[0][warp] = scan & 0xFFFF; warp_sum[1][warp] = scan >> 16; }
                __syncthreads();
            }
            const int m = warp_sum[0][lane], e = warp_sum[1][lane];
            above = above_all + __reduce_add_sync(~0u, lane < warp ? m : 0) + ((scan - c) & 0xFFFF);
            equal = equal_all + __reduce_add_sync(~0u, lane < warp ? e : 0) + ((scan - c) >> 16);
            if (turns > 1) {
                above_all += __reduce_add_sync(~0u, m);
                equal_all += __reduce_add_sync(~0u, e);
            }
            for (uint32_t bits = ms | es; bits; bits &= bits - 1) {
                const int u = __ffs(bits) - 1;
                const uint32_t below = (1u << u) - 1;
                const int like = equal + __popc(es & below), to = above + __popc(ms & below) + min(like, want);
                if (ms >> u & 1 || like < want) {
                    if (short_row) list[to - first_here] = (uint16_t)(place(turn, u) - lo);
                    else out[to] = place(turn, u);
                }
            }
        }
        __syncthreads();
        cluster_barrier();                        // the list is there, and no peer reads this block's sums any more
        if (short_row) {
            if (tid < (int)n) firsts[tid] = (int)peer_word(&first_place, tid);
            __syncthreads();
            const int end = rank + 1 < n ? firsts[rank + 1] : p.budget;
            for (int i = first_here + tid; i < end; i += THREADS) out[i] = lo + list[i - first_here];
        }
    }
    // ---- the move. In shared memory a row is D bytes of keys and D of values; 16 bytes to a thread.
    constexpr int CHUNKS = D / 8;                 // of a row
    const int chunk = tid % CHUNKS, which = chunk / (CHUNKS / 2);
    uint8_t *codes = p.c.codes + which * (16 * D) + 16 * (chunk % (CHUNKS / 2));
    const uint32_t rows_at = (uint32_t)__cvta_generic_to_shared(memory);
    for (int base = 0; base < keep; base += n * PLACES) {
        const int start = base + rank * PLACES, count = max(0, min(PLACES, keep - start));
        __syncthreads();                          // what the pass before wrote out of here
        Place x = {0, 0, 0.0f, 0, 0};
        if (tid < count) {
            const int i = start + tid;
            int at = i;
            if (!all && short_row) {              // from the list of the block that it is in
                int r = 0;
#pragma unroll
                for (int j = 1; j < MOST_CLUSTER; ++j) r = j < (int)n && firsts[j] <= i ? j : r;
                at = r * share + peer_half(list + (i - firsts[r]), r);
            } else if (!all) {
                at = __ldcg(out + i);
            }
            const int64_t page = page_id(p.s, b, at >> p.page_shift), to = page_id(p.to, b, i >> p.page_shift);
            x.from = row_of(p, page, head, at);
            x.to = row_of(p, to, head, i);
            places[tid].from = x.from;
            x.own = reinterpret_cast<const uint16_t *>(p.c.scales)[x.from / BLOCK];            // on its way beside the rows
            x.weight = p.c.weight[x.from];
        }
        __syncthreads();
        for (int i = tid / CHUNKS; i < count; i += THREADS / CHUNKS) {
            const uint32_t from = places[i].from;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(rows_at + 16 * (i * CHUNKS + chunk)),
                         "l"(codes + (int64_t)(from / BLOCK) * (32 * D) + (from % BLOCK) * D) : "memory");
        }
        if (tid < PLACES) {
            uint32_t most = x.own;
#pragma unroll
            for (int d = 1; d < 16; d *= 2) most = __vmaxu4(most, __shfl_xor_sync(~0u, most, d));
            x.scales = (uint16_t)most;
            places[tid] = x;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        cluster_barrier();                        // all of the pass is read
#pragma unroll 4
        for (int i = tid / CHUNKS; i < count; i += THREADS / CHUNKS) {
            const Place x = places[i];
            const int own = x.own >> (8 * which) & 255, E = x.scales >> (8 * which) & 255;
            if (own == E && x.from == x.to) continue;
            uint4 w = reinterpret_cast<const uint4 *>(memory)[i * CHUNKS + chunk];
            if (own != E) w = rescaled<E4M3>(w, rescale_by(own, E));
            *reinterpret_cast<uint4 *>(codes + (int64_t)(x.to / BLOCK) * (32 * D) + (x.to % BLOCK) * D) = w;
        }
        if (tid < count) {
            const Place x = places[tid];
            p.c.weight[x.to] = x.weight;
            if (x.to % BLOCK == 0) reinterpret_cast<uint16_t *>(p.c.scales)[x.to / BLOCK] = x.scales;
        }
    }
}

// The new lengths where they take the place of the old ones, which other blocks read
__global__ void kv8_shorten_kernel(const __grid_constant__ EvictParams p, int32_t *len, const int32_t *kept) {
    wait_earlier();
    let_next_in();
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    // the list of a sequence that stayed as it is begins with -1
    if (b < p.s.B && len[b] > p.budget && kept[(int64_t)b * p.c.H * p.budget] >= 0) len[b] = p.budget;
}

// ---- host ---------------------------------------------------------------------------------------
template <int G, bool E4M3, int THREADS> static int launch_evict(EvictParams p, int64_t tokens, int cluster, cudaStream_t st) {
    using S = Sizes<THREADS>;
    static std::atomic<uint64_t> allowed{0};      // devices on which the kernel may take its shared memory
    int dev = 0;
    if (int rc = current_device(&dev)) return rc;
    if (!(allowed.load(std::memory_order_acquire) >> dev & 1)) {
        OMMX_CUDA_TRY(cudaFuncSetAttribute(kv8_evict_kernel<G, E4M3, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * S::MOST_KEYS));
        allowed.fetch_or(1ull << dev, std::memory_order_release);
    }
    const int64_t share = (tokens + cluster - 1) / cluster + 32;
    p.keys = (int)(share <= S::TURN ? 0 : share - S::TURN < S::MOST_KEYS ? share - S::TURN : S::MOST_KEYS);
    const size_t keys = 4 * (size_t)p.keys, rows = (size_t)S::PLACES * 64 * G + 2 * S::TURN;                 // rows and a list
    static_assert(S::PLACES * 64 * G + 2 * S::TURN <= 4 * S::MOST_KEYS, "the limit that is asked for");
    return launch_dependent(kv8_evict_kernel<G, E4M3, THREADS>, dim3(cluster * p.c.H, p.s.B), THREADS, keys > rows ? keys : rows, st, cluster, p);
}

static int evict(const ommx_kv8_evict_args *a, cudaStream_t st) {
    if (!a) return fail(OMMX_E_ARG, "kv8_evict: null args");
    EvictParams p;
    memset(&p, 0, sizeof(p));
    if (int rc = read_cache("kv8_evict", a->cache, &p.c)) return rc;
    if (int rc = read_seqs("kv8_evict", a->seqs, p.c, &p.s)) return rc;
    if (a->budget < 1) return fail(OMMX_E_ARG, "kv8_evict: budget must be at least 1");
    if (a->sink_tokens < 0 || a->recent_tokens < 0 || (int64_t)a->sink_tokens + a->recent_tokens > a->budget)
        return fail(OMMX_E_ARG, "kv8_evict: %d first and %d last tokens must fit into the %d that are kept", a->sink_tokens, a->recent_tokens, a->budget);
    if (a->max_seq_len < 0) return fail(OMMX_E_ARG, "kv8_evict: max_seq_len must not be negative");
    if (p.s.B > 65535 || p.c.H > 65535) return fail(OMMX_E_UNSUPPORTED, "kv8_evict: a batch of %d", p.s.B);
    if (p.s.B == 0) return 0;
    if (p.c.num_pages == 0) return fail(OMMX_E_ARG, "kv8_evict: a cache of no pages");
    if (!p.c.weight) return fail(OMMX_E_ARG, "kv8_evict: the cache has no weights");
    if (!a->kept) return fail(OMMX_E_ARG, "kv8_evict: kept must not be null");
    p.in_place = a->to_table == nullptr;
    p.to = p.s;
    if (a->to_table) {
        ommx_kv8_seqs to = a->seqs;
        to.page_table = a->to_table; to.page_table_stride = a->to_table_stride; to.table_is_int64 = a->to_table_is_int64; to.pages_per_seq = a->to_pages_per_seq;
        if (int rc = read_seqs("kv8_evict", to, p.c, &p.to)) return rc;
    }
    const bool shortens = a->len_out == a->seqs.b_seq_len;
    if (a->len_out && !shortens && a->len_out < a->seqs.b_seq_len + p.s.B && a->seqs.b_seq_len < a->len_out + p.s.B)
        return fail(OMMX_E_ARG, "kv8_evict: len_out must be b_seq_len itself or apart from it");
    p.kept = a->kept; p.len_out = shortens ? nullptr : a->len_out;
    p.budget = a->budget; p.sinks = a->sink_tokens; p.recent = a->recent_tokens;
    p.page_shift = shift_of(p.c.page);
    p.status = a->status;
    // a cluster to a row where rows are few, but no block for less than 512 tokens (8 kv heads: 4608 to 4096 tokens
    // 23.0 us so and 27.0 with 1024; 4 sequences of 3000 to 2000 20.9 and 25.5; 1200 to 1000 19.1 and 20.3),
    // and as many as run at once (16 rows of 20000 to 4096 tokens: 51.3 us in clusters of eight, of which 15 do, 28.9 in clusters of four)
    int64_t tokens = (int64_t)p.s.max_pages * p.c.page;
    if (a->max_seq_len > 0 && a->max_seq_len < tokens) tokens = a->max_seq_len;
    const int64_t rows = (int64_t)p.s.B * p.c.H;
    int cluster = 1;
    static AtOnce known;                          // all forms of 1024 threads take all of an SM's registers
    auto fit = [&](int n) { return clusters_at_once(known, kv8_evict_kernel<4, false, 1024>, 1024, 4 * Sizes<1024>::MOST_KEYS, n); };
    while (cluster < MOST_CLUSTER && 2 * cluster * rows <= sm_count() && rows <= fit(2 * cluster) && tokens >= 1024LL * cluster) cluster *= 2;
    auto launch = [&](auto g, auto e4m3) {
        constexpr int G = decltype(g)::value;
        constexpr bool E4M3 = decltype(e4m3)::value;
        return rows > sm_count() || tokens <= SHORT ? launch_evict<G, E4M3, 512>(p, tokens, cluster, st) : launch_evict<G, E4M3, 1024>(p, tokens, cluster, st);
    };
    using std::integral_constant;
    int rc;
    if (a->cache.code == OMMX_KV8_E4M3)
        rc = a->cache.head_dim == 128 ? launch(integral_constant<int, 4>(), std::true_type()) : launch(integral_constant<int, 2>(), std::true_type());
    else
        rc = a->cache.head_dim == 128 ? launch(integral_constant<int, 4>(), std::false_type()) : launch(integral_constant<int, 2>(), std::false_type());
    if (rc || !shortens) return rc;
    return launch_dependent(kv8_shorten_kernel, dim3((p.s.B + 127) / 128), 128, 0, st, 1, p, a->len_out, (const int32_t *)a->kept);
}

}  // namespace kv8
}  // namespace ommx

extern "C" int ommx_b200_kv8_evict(const ommx_kv8_evict_args *args, void *stream) { return ommx::kv8::evict(args, (cudaStream_t)stream); }
