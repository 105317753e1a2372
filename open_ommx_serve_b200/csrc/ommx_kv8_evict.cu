// The 8-bit cache: eviction by what tokens were attended to with.
//
// Of a sequence of more than `budget` tokens each kv head keeps the first `sinks`, the last `recent` and, of those between, the ones of the
// largest weight (ties to the lowest place), and they move to the places 0 .. budget - 1 in their order. Two kernels:
// * pick: the weights' order is that of whole numbers, of which the want-th largest is found by counting: what lies between the smallest
//   and the largest is cut into 2048 equal parts, and the part that holds it again, three times at most. A cluster of blocks shares a
//   long row, each with a stretch of its keys in shared memory; counts meet in distributed shared memory. It also notes down what the
//   moved rows' scales are and will be, so that the scales in the cache are read before they are written.
// * move: places ascend, and a token never moves up, so a block that reads what a stretch of places takes before it writes that stretch
//   can work where the tokens lie. Channels do not meet: a row (sequence, kv head) is cut into columns of 32 bytes, a block to each.
#include "ommx_kv8.cuh"
#include "ommx_kv_deal.cuh"

namespace ommx {
namespace kv8 {

using namespace kv;

constexpr int PICK_THREADS = 1024, PICK_WARPS = PICK_THREADS / 32, BINS = 2048, MOST_CLUSTER = 8;
constexpr int MOST_KEYS = 48 * 1024;              // keys that a block holds at most; it reads others again

struct EvictParams {
    Cache c;
    Seqs s, to;                                   // `to`: where kept tokens go; only its table
    int32_t *kept, *len_out;
    int2 *counts;                                 // [B][H]: tokens to move, tokens that are left
    uint16_t *scales;                             // [B][H][places, places / 16]: of what a place takes, and of its record
    int32_t budget, sinks, recent, places, keys, page_shift, in_place;      // places: budget up to whole records; keys: that a block holds
    int32_t *status;
};
__device__ __forceinline__ int64_t record_of(const EvictParams &p, const Seqs &s, int b, int head, int at) {
    const int64_t page = page_id(s, b, at >> p.page_shift);
    return (page * p.c.H + head) * p.c.parts + (at >> 4 & (p.c.parts - 1));
}
// weights as whole numbers in their order; NaN comes last, and zeros are one
__device__ __forceinline__ uint32_t ordered(float w) {
    const uint32_t b = __float_as_uint(w + 0.0f);
    return w != w ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint32_t peer_word(const void *at, uint32_t rank) {
    return __float_as_uint(peer_float((uint32_t)__cvta_generic_to_shared(at), rank));
}

// Grid: (cluster x H, B).
__global__ void __launch_bounds__(PICK_THREADS) kv8_pick_kernel(const __grid_constant__ EvictParams p) {
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ int histogram[BINS], warp_sum[2][PICK_WARPS];
    __shared__ uint32_t low, high;
    __shared__ int bin, left, more, same, bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t n = cluster_size(), rank = cluster_rank();
    const int head = blockIdx.x / n, b = blockIdx.y;
    if (tid == 0) { low = ~0u; high = 0; bad = 0; more = same = 0; }
    histogram[tid] = histogram[tid + PICK_THREADS] = 0;
    wait_earlier();
    let_next_in();
    int len = p.s.len[b];
    const int64_t room = (int64_t)p.s.max_pages << p.page_shift;
    int faults = len < 0 || len > room ? OMMX_ST_BAD_LENGTH : 0;
    if (faults) len = len < 0 ? 0 : (int)room;
    const int keep = min(len, p.budget);
    if (keep > (int64_t)p.to.max_pages << p.page_shift) faults |= OMMX_ST_BAD_LENGTH;
    __syncthreads();
    // a sequence whose pages are not all there stays as it is: every block of it sees that
    if (!faults) {
        bool off = false;
        for (int i = tid; (int64_t)i << p.page_shift < len; i += PICK_THREADS) { const int64_t id = page_id(p.s, b, i); off |= id < 0 || id >= p.c.num_pages; }
        for (int i = tid; (int64_t)i << p.page_shift < keep; i += PICK_THREADS) { const int64_t id = page_id(p.to, b, i); off |= id < 0 || id >= p.c.num_pages; }
        if (off) bad = 1;
        __syncthreads();
        if (bad) faults = OMMX_ST_BAD_PAGE;
    }
    int32_t *out = p.kept + ((int64_t)b * p.c.H + head) * p.budget;
    const int share = ((len + (int)n - 1) / (int)n + 31) & ~31, lo = min(len, (int)rank * share), hi = min(len, lo + share);
    const int moved = faults || (p.in_place && len <= p.budget) ? 0 : keep;
    if (rank == 0 && tid == 0) {
        p.counts[(int64_t)b * p.c.H + head] = make_int2(moved, faults ? p.s.len[b] : keep);
        if (faults) or_status(p.status, faults);
    }
    if (faults || len <= p.budget) {
        for (int i = rank * PICK_THREADS + tid; i < p.budget; i += n * PICK_THREADS) out[i] = !faults && i < len ? i : -1;
        if (!moved) return;
    } else {
        const float *weight = p.c.weight;
        auto load = [&](int i) { return ordered(weight[record_of(p, p.s, b, head, i) * BLOCK + (i & 15)]); };
        auto key_at = [&](int i) { return i - lo < p.keys ? keys[i - lo] : load(i); };
        // keys that are not kept anyway: [first, last) of this block's
        const int first = max(lo, p.sinks), last = min(hi, len - p.recent);
        uint32_t a = ~0u, z = 0;
        for (int i = lo + tid; i < hi; i += PICK_THREADS) {
            const uint32_t k = load(i);
            if (i - lo < p.keys) keys[i - lo] = k;
            if (i >= first && i < last) { a = min(a, k); z = max(z, k); }
        }
        a = __reduce_min_sync(~0u, a);
        z = __reduce_max_sync(~0u, z);
        if (lane == 0) { atomicMin(&low, a); atomicMax(&high, z); }
        __syncthreads();
        cluster_barrier();
        for (uint32_t r = 0; r < n; ++r) { a = min(a, peer_word(&low, r)); z = max(z, peer_word(&high, r)); }
        a = __reduce_min_sync(~0u, a);
        z = __reduce_max_sync(~0u, z);
        // the want-th largest of the keys from `a` on, below a + 2^width
        int want = p.budget - p.sinks - p.recent, width = 32 - __clz(z - a);
        if (want == 0) a = ~0u, width = 0;
        while (width > 0) {
            const int shift = max(0, width - 11);
            for (int i = first + tid; i < last; i += PICK_THREADS) {
                const uint32_t k = key_at(i) - a;
                if (width == 32 || k >> width == 0) atomicAdd(&histogram[k >> shift], 1);
            }
            __syncthreads();
            cluster_barrier();
            // from the top: thread t has bins BINS - 1 - 2 t and the one below
            int upper = 0, lower = 0;
            for (uint32_t r = 0; r < n; ++r) {
                upper += (int)peer_word(&histogram[BINS - 1 - 2 * tid], r);
                lower += (int)peer_word(&histogram[BINS - 2 - 2 * tid], r);
            }
            int before = warp_inclusive_scan(upper + lower, lane);
            if (lane == 31) warp_sum[0][warp] = before;
            __syncthreads();
            before += __reduce_add_sync(~0u, lane < warp ? warp_sum[0][lane] : 0) - upper - lower;
            if (before < want && before + upper + lower >= want) {          // one thread
                const bool up = before + upper >= want;
                left = want - before - (up ? 0 : upper);
                bin = BINS - (up ? 1 : 2) - 2 * tid;
            }
            cluster_barrier();                    // all peers have read
            histogram[tid] = histogram[tid + PICK_THREADS] = 0;
            a += (uint32_t)bin << shift;
            want = left;
            width = shift;
            __syncthreads();
        }
        // keys above `a`, and the first `want` equal to it, in order. A warp has a stretch of its own.
        const int stretch = ((hi - lo + PICK_WARPS - 1) / PICK_WARPS + 31) & ~31, from = min(hi, lo + warp * stretch), to = min(hi, from + stretch);
        auto look = [&](int i, bool &is_more, bool &is_same) {
            const uint32_t k = i < to ? key_at(i) : 0;
            const bool pinned = i < p.sinks || i >= len - p.recent;
            is_more = i < to && (pinned || k > a);
            is_same = i < to && !pinned && k == a;
        };
        int above = 0, equal = 0;
        for (int i0 = from; i0 < to; i0 += 32) {
            bool is_more, is_same;
            look(i0 + lane, is_more, is_same);
            above += __popc(__ballot_sync(~0u, is_more));
            equal += __popc(__ballot_sync(~0u, is_same));
        }
        if (lane == 0) { warp_sum[0][warp] = above; warp_sum[1][warp] = equal; }
        __syncthreads();
        if (warp == 0) {
            const int m = __reduce_add_sync(~0u, warp_sum[0][lane]), e = __reduce_add_sync(~0u, warp_sum[1][lane]);
            if (lane == 0) { more = m; same = e; }
        }
        __syncthreads();
        cluster_barrier();
        above = __reduce_add_sync(~0u, lane < warp ? warp_sum[0][lane] : 0);
        equal = __reduce_add_sync(~0u, lane < warp ? warp_sum[1][lane] : 0);
        for (uint32_t r = 0; r < rank; ++r) { above += (int)peer_word(&more, r); equal += (int)peer_word(&same, r); }
        for (int i0 = from; i0 < to; i0 += 32) {
            bool is_more, is_same;
            look(i0 + lane, is_more, is_same);
            const uint32_t m = __ballot_sync(~0u, is_more), e = __ballot_sync(~0u, is_same), below = (1u << lane) - 1;
            const int at = above + __popc(m & below), eq = equal + __popc(e & below);
            if (is_more || (is_same && eq < want)) out[at + min(eq, want)] = i0 + lane;
            above += __popc(m);
            equal += __popc(e);
        }
        cluster_barrier();                        // the list is there; and no block leaves before its peers have read its sums
    }
    // ---- scales of what each place takes, and of its record
    __syncthreads();
    uint16_t *scales = p.scales + ((int64_t)b * p.c.H + head) * (p.places + p.places / BLOCK);
    const bool listed = len > p.budget;
    for (int i0 = (rank * PICK_WARPS + warp) * 32; i0 < keep; i0 += n * PICK_THREADS) {
        const int i = i0 + lane;
        uint32_t E = 0;
        if (i < keep) {
            const int at = listed ? __ldcg(out + i) : i;
            E = reinterpret_cast<const uint16_t *>(p.c.scales)[record_of(p, p.s, b, head, at)];
            scales[i] = (uint16_t)E;
        }
        uint32_t most = E;
#pragma unroll
        for (int d = 1; d < 16; d *= 2) most = __vmaxu4(most, __shfl_xor_sync(~0u, most, d));
        if ((lane & 15) == 0 && i < keep) scales[p.places + i / BLOCK] = (uint16_t)most;
    }
}

// Grid: (2 D / 32 columns, H, B).  A pass takes MOVE_THREADS / 2 * MOVES places, 16 bytes to a thread and turn.
constexpr int MOVE_THREADS = 512, MOVES = 4;
template <int G, bool E4M3>
__global__ void __launch_bounds__(MOVE_THREADS) kv8_move_kernel(const __grid_constant__ EvictParams p) {
    constexpr int D = 32 * G, PLACES = MOVE_THREADS / 2 * MOVES;
    const int which = blockIdx.x / G, column = blockIdx.x % G, head = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    wait_earlier();
    let_next_in();
    const int2 count = p.counts[(int64_t)b * p.c.H + head];
    if (p.len_out && blockIdx.x == 0 && head == 0 && tid == 0) p.len_out[b] = count.y;
    const int32_t *kept = p.kept + ((int64_t)b * p.c.H + head) * p.budget;
    const uint16_t *scales = p.scales + ((int64_t)b * p.c.H + head) * (p.places + p.places / BLOCK);
    const int part = which * 16 * D + column * 32 + (tid & 1) * 16;
    const bool weighs = which == 0 && column == 0 && (tid & 1) == 0, scaled = column == 0 && (tid & 1) == 0;
    for (int base = 0; base < count.x; base += PLACES) {
        uint4 w[MOVES];
        float weight[MOVES];
        uint8_t *to[MOVES];
        int64_t record[MOVES];
#pragma unroll
        for (int u = 0; u < MOVES; ++u) {
            const int i = base + u * (MOVE_THREADS / 2) + tid / 2;
            to[u] = nullptr;
            if (i >= count.x) continue;
            const int at = kept[i];
            const int64_t from = record_of(p, p.s, b, head, at);
            const uint8_t *source = p.c.codes + from * (32 * D) + part + (at & 15) * D;
            record[u] = record_of(p, p.to, b, head, i);
            w[u] = *reinterpret_cast<const uint4 *>(source);
            if (weighs) weight[u] = p.c.weight[from * BLOCK + (at & 15)];
            to[u] = p.c.codes + record[u] * (32 * D) + part + (i & 15) * D;
            const int own = scales[i] >> (8 * which) & 255, E = scales[p.places + i / BLOCK] >> (8 * which) & 255;
            if (own != E) w[u] = rescaled<E4M3>(w[u], ratio_of(own, E));
        }
        __syncthreads();                          // all of the pass is read
#pragma unroll
        for (int u = 0; u < MOVES; ++u) {
            const int i = base + u * (MOVE_THREADS / 2) + tid / 2;
            if (!to[u]) continue;
            *reinterpret_cast<uint4 *>(to[u]) = w[u];
            if (weighs) p.c.weight[record[u] * BLOCK + (i & 15)] = weight[u];
            if (scaled && (i & 15) == 0) p.c.scales[2 * record[u] + which] = (uint8_t)(scales[p.places + i / BLOCK] >> (8 * which));
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------
static int64_t places_of(int64_t budget) { return (budget + BLOCK - 1) / BLOCK * BLOCK; }
static int64_t workspace_bytes(int64_t B, int64_t H, int64_t budget) {
    return (B * H * 8 + B * H * (places_of(budget) + places_of(budget) / BLOCK) * 2 + 15) / 16 * 16;
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
    const int64_t need = workspace_bytes(p.s.B, p.c.H, a->budget);
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_bytes < need)
        return fail(OMMX_E_ARG, "kv8_evict: workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
    p.in_place = a->to_table == nullptr;
    p.to = p.s;
    if (a->to_table) {
        ommx_kv8_seqs to = a->seqs;
        to.page_table = a->to_table; to.page_table_stride = a->to_table_stride; to.table_is_int64 = a->to_table_is_int64; to.pages_per_seq = a->to_pages_per_seq;
        if (int rc = read_seqs("kv8_evict", to, p.c, &p.to)) return rc;
    }
    p.kept = a->kept; p.len_out = a->len_out;
    p.budget = a->budget; p.sinks = a->sink_tokens; p.recent = a->recent_tokens;
    p.places = (int)places_of(a->budget);
    p.counts = (int2 *)a->workspace;
    p.scales = (uint16_t *)(p.counts + (int64_t)p.s.B * p.c.H);
    p.page_shift = shift_of(p.c.page);
    p.status = a->status;
    // a cluster to a row where rows are few, but no block for less than 2048 tokens
    int64_t tokens = (int64_t)p.s.max_pages * p.c.page;
    if (a->max_seq_len > 0 && a->max_seq_len < tokens) tokens = a->max_seq_len;
    const int64_t rows = (int64_t)p.s.B * p.c.H;
    int cluster = 1;
    while (cluster < MOST_CLUSTER && 2 * cluster * rows <= sm_count() && tokens >= 4096LL * cluster) cluster *= 2;
    const int64_t share = (tokens + cluster - 1) / cluster + 32;
    p.keys = (int)(share < MOST_KEYS ? share : MOST_KEYS);
    static std::atomic<uint64_t> allowed{0};      // devices on which the kernel may take its shared memory
    int dev = 0;
    if (int rc = current_device(&dev)) return rc;
    if (!(allowed.load(std::memory_order_acquire) >> dev & 1)) {
        OMMX_CUDA_TRY(cudaFuncSetAttribute(kv8_pick_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * MOST_KEYS));
        allowed.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (int rc = launch_dependent(kv8_pick_kernel, dim3(cluster * p.c.H, p.s.B), PICK_THREADS, 4 * (size_t)p.keys, st, cluster, p)) return rc;
    const int G = a->cache.head_dim / 32;
    const dim3 grid(2 * G, p.c.H, p.s.B);
    if (a->cache.code == OMMX_KV8_E4M3)
        return G == 4 ? launch_dependent(kv8_move_kernel<4, true>, grid, MOVE_THREADS, 0, st, 1, p) : launch_dependent(kv8_move_kernel<2, true>, grid, MOVE_THREADS, 0, st, 1, p);
    return G == 4 ? launch_dependent(kv8_move_kernel<4, false>, grid, MOVE_THREADS, 0, st, 1, p) : launch_dependent(kv8_move_kernel<2, false>, grid, MOVE_THREADS, 0, st, 1, p);
}

}  // namespace kv8
}  // namespace ommx

extern "C" int64_t ommx_b200_kv8_evict_workspace_bytes(int32_t batch, int32_t n_kv_heads, int32_t budget) {
    return batch < 0 || n_kv_heads < 0 || budget < 0 ? 0 : ommx::kv8::workspace_bytes(batch, n_kv_heads, budget);
}
extern "C" int ommx_b200_kv8_evict(const ommx_kv8_evict_args *args, void *stream) { return ommx::kv8::evict(args, (cudaStream_t)stream); }
