// The 8-bit cache: its record format, and what its kernels share.
//
// One record of 32 D bytes per (page, kv head, 16 tokens): 16 rows of D key codes, then 16 rows of D value codes, int8 or e4m3; two
// exponents E per record beside them, of the keys and of the values.  value = code * 2^(E - 127); E = 0 where all are zero.
// Powers of two: every product of a code and a scale is exact, codes are the same however they are computed, and codes that
// move to a larger scale lose their last bits only.
#pragma once

#include <type_traits>

#include "ommx_kv4.cuh"

namespace ommx {
namespace kv8 {

using kv4::Rows;
using kv4::Run;
using kv4::Seqs;
using kv4::launch_dependent;
using kv4::let_next_in;
using kv4::page_id;
using kv4::shift_of;
using kv4::wait_earlier;
using kv4::warp_inclusive_scan;

constexpr float LARGEST = 0x1p126f;               // the quantizer takes values to be at most this
constexpr int BLOCK = 16;                         // tokens to a scale

struct Cache {
    uint8_t *codes, *scales;
    float *weight;                                // [pages][H][page], or null
    int32_t num_pages, H, page, parts;            // parts: records per page and head
};

// 2^(E - 127); 0 for E = 0
__device__ __forceinline__ float scale_of(int E) { return __uint_as_float((uint32_t)E << 23); }
// 2^(E - over), E <= over: what codes are multiplied with to be held in the larger scale
__device__ __forceinline__ float ratio_of(int E, int over) { return E == 0 || over - E > 126 ? 0.0f : __uint_as_float((uint32_t)(127 + E - over) << 23); }
// The smallest E from 1 on with top <= TOP 2^(E - 127), TOP = 127 (1.984375 * 2^6) or 448 (1.75 * 2^8); 0 for 0. Past the mantissa of TOP a
// number's exponent counts one more.
template <bool E4M3> __device__ __forceinline__ int exponent_for(float top) {
    const uint32_t bits = __float_as_uint(top), past = 0x800000u - 1u - (E4M3 ? 0x600000u : 0x7E0000u);
    return top > 0.0f ? max((int)((bits + past) >> 23) - (E4M3 ? 8 : 6), 1) : 0;
}

// two numbers in units to two e4m3 codes (the first in the low byte) and back; nearest, ties to even
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t half2_of_e4m3x2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    return r;
}
// four numbers in units, at most 127 or 448, to a word of codes. int8: the number lands in the last byte of 1.5 * 2^23 + it, rounded as
// a sum is.
template <bool E4M3> __device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d) {
    if constexpr (E4M3) {
        return to_e4m3x2(a, b) | to_e4m3x2(c, d) << 16;
    } else {
        constexpr float ROUND = 12582912.0f;
        const uint32_t lo = __byte_perm(__float_as_uint(a + ROUND), __float_as_uint(b + ROUND), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(c + ROUND), __float_as_uint(d + ROUND), 0x0040);
        return __byte_perm(lo, hi, 0x5410);
    }
}
// a word of codes to four numbers in units
template <bool E4M3> __device__ __forceinline__ void numbers_of(uint32_t w, float (&x)[4]) {
    if constexpr (E4M3) {
        const uint32_t h[2] = {half2_of_e4m3x2(w), half2_of_e4m3x2(w >> 16)};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    } else {
        const uint32_t u = w ^ 0x80808080u;       // code + 128, in the last byte of 2^23 + it
        x[0] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440)) - 8388736.0f;
        x[1] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7441)) - 8388736.0f;
        x[2] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7442)) - 8388736.0f;
        x[3] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7443)) - 8388736.0f;
    }
}
// The same codes in a scale 2^by times as large, by >= 1; all is fp16: codes are fp16 numbers, and where a product has more bits than they
// it rounds to 0 either way. E = 0: the codes stand for zeros.
struct Rescale { __half2 ratio; };
__device__ __forceinline__ Rescale rescale_by(int held, int E) {
    return {__float2half2_rn(ratio_of(held, E))};  // below 2^-24 it is 0, and so are the codes
}
template <bool E4M3> __device__ __forceinline__ uint32_t rescaled(uint32_t w, const Rescale &by) {
    if constexpr (E4M3) {
        const uint32_t h[2] = {half2_of_e4m3x2(w), half2_of_e4m3x2(w >> 16)};
        uint32_t r[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const __half2 x = __hmul2(*reinterpret_cast<const __half2 *>(&h[i]), by.ratio);
            uint16_t e;
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(e) : "r"(*reinterpret_cast<const uint32_t *>(&x)));
            r[i] = e;
        }
        return r[0] | r[1] << 16;
    } else {
        const uint32_t u = w ^ 0x80808080u;       // 1024 + 128 + code as an fp16 number; the last byte of 1536 + code, rounded as a sum is
        const __half2 off = __float2half2_rn(1152.0f), round = __float2half2_rn(1536.0f);
        const uint32_t h[2] = {__byte_perm(u, 0x64646464u, 0x4140), __byte_perm(u, 0x64646464u, 0x4342)};
        uint32_t r[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const __half2 x = __hfma2(__hsub2(*reinterpret_cast<const __half2 *>(&h[i]), off), by.ratio, round);
            r[i] = *reinterpret_cast<const uint32_t *>(&x);
        }
        return __byte_perm(r[0], r[1], 0x6420);
    }
}
template <bool E4M3> __device__ __forceinline__ uint4 rescaled(uint4 w, const Rescale &by) {
    return make_uint4(rescaled<E4M3>(w.x, by), rescaled<E4M3>(w.y, by), rescaled<E4M3>(w.z, by), rescaled<E4M3>(w.w, by));
}

// ---- host: arguments every entry point checks ----
inline int read_cache(const char *who, const ommx_kv8_cache &c, Cache *to) {
    if (c.head_dim != 64 && c.head_dim != 128) return fail(OMMX_E_UNSUPPORTED, "%s: head_dim %d (this build serves 64 and 128)", who, c.head_dim);
    if (c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1)))
        return fail(OMMX_E_UNSUPPORTED, "%s: page_size %d (this build serves 16, 32, 64, 128 and 256)", who, c.page_size);
    if (c.code != OMMX_KV8_INT8 && c.code != OMMX_KV8_E4M3) return fail(OMMX_E_ARG, "%s: code type %d is none of int8, e4m3", who, c.code);
    if (c.num_pages < 0 || c.n_kv_heads <= 0 || c.n_kv_heads > 4096) return fail(OMMX_E_ARG, "%s: %d pages of %d kv heads", who, c.num_pages, c.n_kv_heads);
    if (c.num_pages && (!c.codes || !c.scales)) return fail(OMMX_E_ARG, "%s: codes and scales must be given", who);
    if (reinterpret_cast<uintptr_t>(c.codes) % 16 || reinterpret_cast<uintptr_t>(c.scales) % 2) return fail(OMMX_E_ARG, "%s: codes must be 16-byte aligned and scales 2-byte", who);
    if (reinterpret_cast<uintptr_t>(c.weight) % 16) return fail(OMMX_E_ARG, "%s: weight must be 16-byte aligned", who);
    *to = {(uint8_t *)c.codes, c.scales, c.weight, c.num_pages, c.n_kv_heads, c.page_size, c.page_size / BLOCK};
    return 0;
}
// How many clusters of a size (2, 4 or 8) the device holds at once, asked for once: fewer than blocks / size, since a cluster lies on SMs of one
// group (148 SMs: 33 of eight blocks, two to an SM, and 15 with one). One cluster more than that is a second turn for all.
struct AtOnce { std::atomic<int> count[MAX_DEVICES][4]; };
template <typename K> int clusters_at_once(AtOnce &known, K kernel, int threads, size_t smem, int cluster) {
    int dev = 0, size = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return 0;
    while (1 << size < cluster) ++size;
    if (const int held = known.count[dev][size].load(std::memory_order_acquire)) return held - 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = cluster;
    cfg.blockDim = threads;
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 0) {
        (void)cudaGetLastError();
        n = 0;
    }
    known.count[dev][size].store(n + 1, std::memory_order_release);
    return n;
}
inline int read_seqs(const char *who, const ommx_kv8_seqs &s, const Cache &c, Seqs *to) {
    kv4::Cache like = {nullptr, c.num_pages, c.H, c.page, c.parts};
    return kv4::read_seqs(who, s, like, to);
}

}  // namespace kv8
}  // namespace ommx
