// q4_common.cuh - the packed 4-bit weight layout and the code and slice conversions shared by its kernels.
//
// Packed weights of E experts of N x K: codes, then (at the next multiple of 256 bytes) the scales.
//   codes   code = q + 8, q = -7..7 (8 where N is padded to 16 rows or K to 64): tiles of 16 rows x 64 values of K, 512
//           bytes each, ordered [expert][row block][k block]. The 16 bytes of lane (g, t) = 4g + t of a tile are four
//           words: row g, k = 8t..8t+7; row g + 8, the same k; row g, k = 32 + 8t..; row g + 8, the same. In a word the
//           nibbles from the lowest up are k = 0, 2, 4, 6, 1, 3, 5, 7.
//   scales  bf16, [expert][row block][group][8][2]: rows g and g + 8 in one 32-bit word; 0 in padding rows.
// A warp's 16-byte load of a tile is one coalesced 512-byte access, and lane (g, t) then holds exactly the A fragment
// of m16n8k16 (rows g and g + 8) for a K order in which each lane's B values are 16 contiguous bytes of a row of x.
#pragma once

#include "emugemm_internal.h"

#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace emu {

// Runs its argument (a cudaFuncSetAttribute call, a cudaError_t as int) until it has succeeded once on the current
// device. Calls from several threads may run it more than once.
struct OncePerDevice {
    std::atomic<unsigned long long> done{0};
    template <typename F>
    int operator()(F&& f) {
        int dev = 0;
        const cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return (int)e;
        const unsigned long long bit = 1ull << (dev & 63);
        if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return 0;
        const int r = f();
        if (!r && dev < 64) done.fetch_or(bit, std::memory_order_release);
        return r;
    }
};

// Clusters that the current device holds at once, by CTAs resident on an SM (1 .. 3) and CTAs per cluster (1 .. 8): fewer
// than the SMs would make, since a cluster stays within one GPC. Null: a CUDA error.
struct ClusterFits { int of[4][9]; };
const ClusterFits* cluster_fits();   // k_q4.cu

namespace q4 {

struct Layout {
    long nb, kb, groups;        // row blocks of 16, k blocks of 64, scale groups along K
    size_t codes;               // bytes of the codes of all experts
    size_t scales_at;           // byte offset of the scales
    size_t bytes;               // of the whole
};
inline __host__ __device__ Layout layout(long E, long N, long K, int group) {
    Layout l;
    l.nb = (N + 15) / 16;
    l.kb = (K + 63) / 64;
    l.groups = (K + group - 1) / group;
    l.codes = (size_t)E * l.nb * l.kb * 512;
    l.scales_at = (l.codes + 255) / 256 * 256;
    l.bytes = l.scales_at + (size_t)E * l.nb * l.groups * 32;
    return l;
}

// The values q of all eight codes of a word as 16-bit floats times 1 / code_unit, exact: v[p] holds nibbles p and p + 4
// (the lower k in the low half). Masked in place, without a shift each (the integer pipe, at half the rate of the
// others, bounds the unpacking: 5 operations on it per word, against 7 with every nibble shifted to bit 0).
//   bf16: the low byte u of a half is a subnormal or first-binade bf16, u * 2^-133 for all 256 values; one fused
//         multiply-add by 2^127 (nibble at bit 0) or 2^123 (at bit 4) and minus 8 * 2^-6 gives q * 2^-6;
//   fp16: the nibble as low mantissa bits of 1024: 1024 + u or 1024 + 16 u, minus 1032, or times 1/16 minus 72 (the
//         conversion by an exponent's offset, as in Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run", 2022).
template <bool BF16>
__device__ __forceinline__ constexpr float code_unit() { return BF16 ? 64.f : 1.f; }
template <bool BF16>
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t (&v)[4]) {
    const uint32_t h = w >> 8;
    if (BF16) {
        const uint32_t lo = 0x7f007f00u, hi = 0x7d007d00u, off = 0xbe00be00u;   // 2^127, 2^123, -2^-3
        auto f = [&](uint32_t x, uint32_t m) {
            uint32_t r;
            asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(m), "r"(off));
            return r;
        };
        v[0] = f(w & 0x000F000Fu, lo);
        v[1] = f(w & 0x00F000F0u, hi);
        v[2] = f(h & 0x000F000Fu, lo);
        v[3] = f(h & 0x00F000F0u, hi);
    } else {
        const uint32_t one = 0x3c003c00u, sixteenth = 0x2c002c00u, lo = 0xe408e408u, hi = 0xd480d480u;   // -1032, -72
        auto f = [&](uint32_t x, uint32_t m, uint32_t off) {
            uint32_t r;
            asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(m), "r"(off));
            return r;
        };
        v[0] = f((w & 0x000F000Fu) | 0x64006400u, one, lo);
        v[1] = f((w & 0x00F000F0u) | 0x64006400u, sixteenth, hi);
        v[2] = f((h & 0x000F000Fu) | 0x64006400u, one, lo);
        v[3] = f((h & 0x00F000F0u) | 0x64006400u, sixteenth, hi);
    }
}

// x = hi + mid + lo, each slice the leading 8 significant bits of what is left (truncated, so that nothing overflows and
// the sum is exact down to the smallest bf16). Inf stays Inf in hi with zero slices below; NaN stays NaN.
__device__ __forceinline__ void slice3(float x, uint16_t& hi, uint16_t& mid, uint16_t& lo) {
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7f800000u) == 0x7f800000u) {
        hi = (uint16_t)((b >> 16) | ((b & 0x007fffffu) ? 0x40u : 0u));
        mid = lo = 0;
        return;
    }
    const uint32_t h = b & 0xffff0000u;
    const float r = x - __uint_as_float(h);
    const uint32_t m = __float_as_uint(r) & 0xffff0000u;
    hi = (uint16_t)(h >> 16);
    mid = (uint16_t)(m >> 16);
    lo = (uint16_t)(__float_as_uint(r - __uint_as_float(m)) >> 16);
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

}  // namespace q4
}  // namespace emu
