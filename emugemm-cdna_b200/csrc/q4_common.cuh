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

// The values q of nibbles p and p + 4 of a word of codes as two 16-bit floats (the lower k in the low half), exact: the
// nibble as the low mantissa bits of 128 (bf16) or 1024 (fp16), minus that plus 8.
template <bool BF16>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int p) {
    const uint32_t v = ((w >> (4 * p)) & 0x000F000Fu) | (BF16 ? 0x43004300u : 0x64006400u);
    if (BF16) {
        const uint32_t c = 0x43084308u;   // 136, 136
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                         *reinterpret_cast<const __nv_bfloat162*>(&c));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    const uint32_t c = 0x64086408u;       // 1032, 1032
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
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
