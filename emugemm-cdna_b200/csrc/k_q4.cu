// k_q4.cu - 4-bit weights with group scales: packing, unpacking, and the product for few rows.
#include "q4_common.cuh"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace emu {

namespace {

using namespace q4;

// ------------------------------------------------------------------------------------------------- pack and unpack
// s = bf16(fp32(max|w| / 7)) of a group, q = w / s rounded to the nearest integer (even on a tie), at most 7 away.
// w * (1 / s) in FP32 can round onto or across a tie that w / s itself is not on, so q is checked with the residual
// w - q s, which fmaf gives exactly where it matters (|w| <= 7.1 s: at most 24 significant bits at half a step).
struct Scale {
    float s, inv, half;     // the scale and its half times up, 1 / (scale * up)
    float up;               // 2^64 for groups below 2^-90: of their scales half and inverse would not be normal floats
    uint32_t bits;          // bf16
    bool slow;              // values may be more than 7.5 scales away, or there is nothing to divide by
    bool none;              // the group reads as zeros, or as NaN
};
// m / 7 rounded to the nearest float, m normal with m / 7 normal: the product with the rounded reciprocal, corrected by its
// exact residual (Markstein's division step; 1 / 7 is the correctly rounded reciprocal it asks for).
__device__ __forceinline__ float seventh(float m) {
    const float y = 1.f / 7.f, q = m * y;
    return fmaf(fmaf(-7.f, q, m), y, q);
}
__device__ __forceinline__ Scale scale_of(unsigned absmax_bits) {   // Inf and NaN compare above every number
    Scale c;
    const float m = __uint_as_float(absmax_bits);
    c.slow = !(m >= 0x1p-90f) || absmax_bits >= 0x7f800000u;
    if (!c.slow) {
        c.none = false;
        c.up = 1.f;
        c.s = __bfloat162float(__float2bfloat16_rn(seventh(m)));
        c.bits = __float_as_uint(c.s) >> 16;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(c.inv) : "f"(c.s));   // the codes are checked by their residuals
    } else {
        const bool bad = absmax_bits >= 0x7f800000u;
        const float s = bad ? __uint_as_float(0x7fc00000u) : __bfloat162float(__float2bfloat16_rn(__fdiv_rn(m, 7.f)));
        c.bits = __float_as_uint(s) >> 16;
        c.none = bad || s == 0.f;
        c.up = 0x1p64f;
        c.s = s * c.up;
        c.inv = 1.f / c.s;
    }
    c.half = 0.5f * c.s;
    return c;
}
__device__ __forceinline__ uint32_t code_slow(float w, const Scale& c) {   // q + 8
    if (c.none) return 8u;
    w *= c.up;
    float q = rintf(w * c.inv);
    const float r = fmaf(-q, c.s, w);
    const bool odd = ((int)q) & 1;
    if (r > c.half || (r == c.half && odd)) q += 1.f;
    else if (r < -c.half || (r == -c.half && odd)) q -= 1.f;
    return (uint32_t)((int)fminf(fmaxf(q, -7.f), 7.f) + 8);
}
// q + 8 in the low four bits of w / s + 1.5 * 2^23 + 8; `off` grows to the largest residual seen: at or beyond half a
// step the value needs code_exact.
__device__ __forceinline__ uint32_t code_fast(float w, const Scale& c, float& off) {
    const float t = fmaf(w, c.inv, 12582920.f);
    off = fmaxf(off, fabsf(fmaf(-(t - 12582920.f), c.s, w)));
    return __float_as_uint(t) & 15u;
}
// The same with the step towards the residual where it is beyond half a step, or half a step of an odd q: for the
// FP32 words that code_fast finds one in (very rarely), and for 16-bit weights, where ties are common.
__device__ __forceinline__ uint32_t code_exact(float w, const Scale& c) {
    const float t = fmaf(w, c.inv, 12582920.f);
    const float r = fmaf(-(t - 12582920.f), c.s, w);
    const uint32_t u = __float_as_uint(t);
    const bool step = fabsf(r) > c.half || (fabsf(r) == c.half && (u & 1u));
    return (u + (step ? (r > 0.f ? 1u : ~0u) : 0u)) & 15u;
}

// W on 16-byte boundaries: one warp per 16 rows x 128 values of K. Lane (g, t) reads rows g and g + 8 at k = 32i + 8t ..
// +7 (i = 0..3): the values its own words of the two tiles hold. A group of 32 is one i of four lanes, so the group
// maximum is two shuffles, for groups of 64 and 128 after combining i in registers. Bound for FP32: the read of W (8192 x
// 8192, groups of 128: 53 us, 69 % of DRAM). For 16-bit W, whose codes are all checked against their residual, the arithmetic
// per value (87, 78 and 84 us for groups of 128, 64 and 32; 27 instructions a value, integer pipe 67 %, DRAM 22 %).
template <typename T, int GROUP>
__global__ void __launch_bounds__(256, 4) k_q4_pack(const T* __restrict__ W, long ldw, int E, int N, long K, Layout l,
                                                 uint8_t* __restrict__ packed) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long kp = (l.kb + 1) / 2;
    const long units = (long)E * l.nb * kp;
    constexpr int PER = GROUP / 32;   // values of i per group
    uint32_t* scales = reinterpret_cast<uint32_t*>(packed + l.scales_at);
    for (long u = (long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (long)gridDim.x * 8) {
        const long b = u / kp, k128 = u - b * kp;     // b = expert * nb + row block
        const long e = b / l.nb;
        const int n0 = (int)(b - e * l.nb) * 16;
        uint32_t word[2][4], sc[2][4 / PER];          // [half of the rows]
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int n = n0 + g + 8 * half;
            const T* row = W + ((size_t)e * N + n) * ldw;
#pragma unroll
            for (int gi = 0; gi < 4 / PER; ++gi) {
                __align__(16) float v[PER][8];
                static_assert(__alignof__(v) >= 16, "written 16 bytes at a time");
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const long k = k128 * 128 + GROUP * gi + 32 * i + 8 * t;
                    if (n < N && k + 8 <= K) {
                        if (sizeof(T) == 4) {
                            *reinterpret_cast<float4*>(v[i]) = __ldg(reinterpret_cast<const float4*>(row + k));
                            *reinterpret_cast<float4*>(v[i] + 4) = __ldg(reinterpret_cast<const float4*>(row + k) + 1);
                        } else {
                            const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + k));
                            const T* p = reinterpret_cast<const T*>(&a);
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[i][j] = to_float<T>(p[j]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[i][j] = (n < N && k + j < K) ? to_float<T>(row[k + j]) : 0.f;
                    }
                }
                unsigned m = 0;
#pragma unroll
                for (int i = 0; i < PER; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[i][j]) & 0x7fffffffu);
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const Scale c = scale_of(m);
                sc[half][gi] = n < N ? c.bits : 0u;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    float off = 0.f;
                    uint32_t w = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        w |= (sizeof(T) == 4 ? code_fast(v[i][j], c, off) : code_exact(v[i][j], c)) << (4 * (j / 2 + 4 * (j & 1)));
                    if (c.slow || off >= c.half) {
                        w = 0;
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            w |= (c.slow ? code_slow(v[i][j], c) : code_exact(v[i][j], c)) << (4 * (j / 2 + 4 * (j & 1)));
                    }
                    word[half][gi * PER + i] = w;
                }
            }
        }
        uint4* tile = reinterpret_cast<uint4*>(packed) + (size_t)(b * l.kb + 2 * k128) * 32 + lane;
        tile[0] = make_uint4(word[0][0], word[1][0], word[0][1], word[1][1]);
        if (2 * k128 + 1 < l.kb) tile[32] = make_uint4(word[0][2], word[1][2], word[0][3], word[1][3]);
        if (t == 0) {
#pragma unroll
            for (int gi = 0; gi < 4 / PER; ++gi) {
                const long kg = k128 * (4 / PER) + gi;
                if (kg < l.groups) scales[((size_t)b * l.groups + kg) * 8 + g] = sc[0][gi] | (sc[1][gi] << 16);
            }
        }
    }
}

// W on other boundaries: one warp per 128 values of rows r and r + 8 of a row block, a lane per value of each 32, so that
// the loads stay contiguous whatever the alignment; the group maximum is one warp reduction per 32 values, and a word is
// put together by three shuffles among its eight lanes. Bound: the instructions, 63 a value (8192 x 8191 bf16 155 us, 78 % of
// the issue slots, 12 % of DRAM). (With the mapping above and 2-byte loads 16 bytes apart, 5 x 1000 x 1111 bf16 weights took
// 61 us with their read back.)
template <typename T, int GROUP>
__global__ void __launch_bounds__(256) k_q4_pack_rows(const T* __restrict__ W, long ldw, int E, int N, long K, Layout l,
                                                      uint8_t* __restrict__ packed) {
    const int lane = threadIdx.x & 31;
    const long kp = (l.kb + 1) / 2, rows = l.nb * 8;
    const long units = (long)E * rows * kp;
    constexpr int PER = GROUP / 32;
    uint2* codes = reinterpret_cast<uint2*>(packed);
    uint32_t* scales = reinterpret_cast<uint32_t*>(packed + l.scales_at);
    for (long u = (long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (long)gridDim.x * 8) {
        const long rr = u / kp, k128 = u - rr * kp;
        const long b = rr >> 3, e = b / l.nb;
        const int r = (int)(rr & 7), n = (int)(b - e * l.nb) * 16 + r;
        const T* row = W + ((size_t)e * N + n) * ldw + k128 * 128 + lane;
        const long left = K - k128 * 128 - lane;
        float v[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[half][i] = n + 8 * half < N && 32 * i < left ? to_float<T>(row[8 * half * ldw + 32 * i]) : 0.f;
        uint32_t word[2][4];
#pragma unroll
        for (int gi = 0; gi < 4 / PER; ++gi) {
            uint32_t sc[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                unsigned m = 0;
#pragma unroll
                for (int i = gi * PER; i < (gi + 1) * PER; ++i) m = max(m, __float_as_uint(v[half][i]) & 0x7fffffffu);
                const Scale c = scale_of(__reduce_max_sync(0xffffffffu, m));
                sc[half] = n + 8 * half < N ? c.bits : 0u;
#pragma unroll
                for (int i = gi * PER; i < (gi + 1) * PER; ++i) {
                    const int j = lane & 7;
                    uint32_t w = (c.slow ? code_slow(v[half][i], c) : code_exact(v[half][i], c)) << (4 * (j / 2 + 4 * (j & 1)));
                    w |= __shfl_xor_sync(0xffffffffu, w, 1);
                    w |= __shfl_xor_sync(0xffffffffu, w, 2);
                    w |= __shfl_xor_sync(0xffffffffu, w, 4);
                    word[half][i] = w;
                }
            }
            const long kg = k128 * (4 / PER) + gi;
            if (lane == 0 && kg < l.groups) scales[((size_t)b * l.groups + kg) * 8 + r] = sc[0] | (sc[1] << 16);
        }
        if ((lane & 7) == 0)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long kb = 2 * k128 + (i >> 1);
                if (kb < l.kb) codes[(size_t)(b * l.kb + kb) * 64 + (r * 4 + (lane >> 3)) * 2 + (i & 1)] = make_uint2(word[0][i], word[1][i]);
            }
    }
}

// W = s q in FP32 (8 + 3 significant bits: exact). One warp per tile: the tile comes in as one 512-byte access and goes out
// as rows, their words and scales handed to the lanes by shuffles. Bound: the write. VEC: rows on 16-byte boundaries, a
// lane writes four values and a warp two rows at a time; else a value per lane, so that 32 stay one 128-byte access at any
// alignment (70 us against 45 for 8192 x 8192).
template <bool VEC>
__global__ void __launch_bounds__(256) k_q4_unpack(const uint8_t* __restrict__ packed, int E, int N, long K, int group,
                                                   Layout l, float* __restrict__ W, long ldw) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(packed + l.scales_at);
    const long units = (long)E * l.nb * l.kb;
    // 2^23 + u - (2^23 + 8)
    auto value = [](uint32_t u) { return __uint_as_float((u & 15u) | 0x4b000000u) - 8388616.f; };
    for (long u = (long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (long)gridDim.x * 8) {
        const long b = u / l.kb, kb = u - b * l.kb, e = b / l.nb;
        const int n0 = (int)(b - e * l.nb) * 16;
        const uint4 c = __ldg(reinterpret_cast<const uint4*>(packed) + (size_t)u * 32 + lane);
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        uint32_t sw[2];   // the scales of rows g and g + 8 for the two halves of the tile
#pragma unroll
        for (int h = 0; h < 2; ++h)
            sw[h] = kb * 64 + 32 * h < K ? __ldg(scales + ((size_t)b * l.groups + (kb * 64 + 32 * h) / group) * 8 + g) : 0u;
        if (VEC) {
            // lane: row 2j + (lane >> 4), values 4 (lane & 15) .. + 3, half a word
            const int k = 4 * (lane & 15), h = k >> 5, from = (k >> 3) & 3, shift = 8 * ((k >> 2) & 1);
            float* out = W + ((size_t)e * N + n0) * ldw + kb * 64 + k;
            const long left = K - kb * 64 - k;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = 2 * j + (lane >> 4), hi = j >> 2;
                const uint32_t w0 = __shfl_sync(0xffffffffu, w[hi], (row & 7) * 4 + from);
                const uint32_t w1 = __shfl_sync(0xffffffffu, w[2 + hi], (row & 7) * 4 + from);
                const uint32_t s0 = __shfl_sync(0xffffffffu, sw[0], (row & 7) * 4);
                const uint32_t s1 = __shfl_sync(0xffffffffu, sw[1], (row & 7) * 4);
                const uint32_t word = (h ? w1 : w0) >> shift, sp = h ? s1 : s0;
                const float s = hi ? bf16_hi(sp) : bf16_lo(sp);
                if (n0 + row < N && left > 0)
                    *reinterpret_cast<float4*>(out + (size_t)row * ldw) =
                        make_float4(s * value(word), s * value(word >> 16), s * value(word >> 4), s * value(word >> 20));
            }
        } else {
            const int shift = 4 * ((lane & 7) / 2 + 4 * (lane & 1));
            float* out = W + ((size_t)e * N + n0) * ldw + kb * 64 + lane;
            const long left = K - kb * 64 - lane;
#pragma unroll
            for (int i = 0; i < 4; ++i) {                // word i: rows 8 (i & 1) .. +7, half i >> 1 of the tile
                const int h = i >> 1;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const uint32_t word = __shfl_sync(0xffffffffu, w[i], r * 4 + (lane >> 3));
                    const uint32_t sp = __shfl_sync(0xffffffffu, sw[h], r * 4);
                    const int n = 8 * (i & 1) + r;
                    if (n0 + n < N && 32 * h < left)
                        out[(size_t)n * ldw + 32 * h] = ((i & 1) ? bf16_hi(sp) : bf16_lo(sp)) * value(word >> shift);
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------- product, few rows
// C[m, n] = sum over groups of s[n, group] * (sum over the group of q[n, k] A[m, k]).
//
// One warp multiplies row blocks of 16 weights rows with up to 8 NT columns by m16n8k16 products: the weights are the
// 16-row operand (their integers are exact in bf16 and fp16), the columns are rows of A, and for FP32 A the three bf16
// slices of each row (exact to 24 bits). A group's sum is kept apart and added to the row's FP32 sum times its scale,
// so no weight is ever rounded. What bounds it is the read of the codes (and, beyond about 16 columns, the products):
// each warp keeps the codes of its next D x 128 values of K in flight in registers, the first of them from before the
// columns are staged. The columns of the block's K range lie in shared memory (rows 64 bytes apart modulo 128, so that
// the 16-byte fragment loads of 8 rows x 4 lanes meet no bank conflict); the WK warps of a row block take 128 values
// of K in turn, their sums are added in order, and where there are few row blocks a cluster of CTAs splits K and adds
// its parts over distributed shared memory.
constexpr int kWarps = 8;
constexpr int kRowsSmem = 110 * 1024;

struct RowsParams {
    const void* A; long lda;
    const uint8_t* packed; Layout l;
    void* C; long ldc;
    const int* offsets;       // experts: E + 1 row offsets; null: one matrix, rows 0 .. R - 1
    int R, E, N; long K;
    int kspan;                // K values per CTA of the cluster (a multiple of 128)
    int kstage;               // K values staged at a time (a multiple of 128)
    int vec;                  // rows of A on 16-byte boundaries
};

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool BF16>
__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {   // d = a * b
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint4 ld_codes(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {   // whole warps (.aligned): lanes may have left a loop early
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
    uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r));
    return v;
}

// Expert and rows of blockIdx.y: the i-th expert that has rows (all lanes of a warp call it; false: there is none).
__device__ __forceinline__ bool nth_expert(const int* offsets, int E, int i, int R, int& e, int& r0, int& r1) {
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < E; base += 128) {
        int a[4], b[4];                          // 128 experts at a time: one wait for their offsets
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int x = base + 32 * j + lane;
            a[j] = x < E ? __ldg(offsets + x) : 0;
            b[j] = x < E ? __ldg(offsets + x + 1) : 0;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned some = __ballot_sync(0xffffffffu, b[j] > a[j]);
            const int n = __popc(some);
            if (i < n) {
                const int src = __fns(some, 0, i + 1);
                e = base + 32 * j + src;
                r0 = max(0, __shfl_sync(0xffffffffu, a[j], src));
                r1 = min(R, __shfl_sync(0xffffffffu, b[j], src));   // a bad offset reads and writes no row outside of A and C
                return true;
            }
            i -= n;
        }
    }
    return false;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {   // the rest of 16 is zeroed
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Rows of A (toks rows of `len` values) into shared memory as 16-bit columns, zeros from len to span; a warp takes 256 values
// of a row at a time. Rows on 16-byte boundaries: 8 values per lane, 16-bit ones as asynchronous copies; others: a value
// per lane at a time, so that the loads stay contiguous.
template <typename T>
__device__ __forceinline__ void stage_rows(uint16_t* xs, int pitch, const T* rows, long lda, int toks, int span, int len,
                                           int vec) {
    constexpr int SL = sizeof(T) == 4 ? 3 : 1;
    const int lane = threadIdx.x & 31;
    int m = 0, k0 = (threadIdx.x >> 5) * 256;
    while (true) {
        while (k0 >= span) {
            k0 -= (span + 255) / 256 * 256;
            if (++m >= toks) return;
        }
        const T* row = rows + (size_t)m * lda;
        if (vec) {
            const int k = k0 + lane * 8, left = len - k;
            if (k < span) {
                if (SL == 1) {
                    cp_async16(static_cast<uint32_t>(__cvta_generic_to_shared(xs + m * pitch + k)), left > 0 ? row + k : rows,
                               left <= 0 ? 0 : left >= 8 ? 16 : 2 * left);
                } else {
                    __align__(16) float x[8];
                    if (left >= 8) {
                        *reinterpret_cast<float4*>(x) = __ldg(reinterpret_cast<const float4*>(row + k));
                        *reinterpret_cast<float4*>(x + 4) = __ldg(reinterpret_cast<const float4*>(row + k) + 1);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = j < left ? to_float<T>(row[k + j]) : 0.f;
                    }
                    __align__(16) uint16_t s[3][8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) slice3(x[j], s[0][j], s[1][j], s[2][j]);
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        *reinterpret_cast<uint4*>(xs + (3 * m + i) * pitch + k) = *reinterpret_cast<const uint4*>(s[i]);
                }
            }
        } else {
            T x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int k = k0 + 32 * j + lane;
                x[j] = k < len ? row[k] : from_float<T>(0.f);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int k = k0 + 32 * j + lane;
                if (k >= span) break;
                if (SL == 3) {
                    uint16_t s[3];
                    slice3(to_float<T>(x[j]), s[0], s[1], s[2]);
#pragma unroll
                    for (int i = 0; i < 3; ++i) xs[(3 * m + i) * pitch + k] = s[i];
                } else {
                    xs[m * pitch + k] = *reinterpret_cast<const uint16_t*>(&x[j]);
                }
            }
        }
        k0 += 256 * kWarps;
    }
}

// T: type of A and C; NT: column tiles of 8; WR: warps over row blocks; RBW: row blocks per warp; D: units of 128
// values of K in flight per warp; CTAS: resident on an SM; GROUP.
template <typename T, int NT, int WR, int RBW, int D, int CTAS, int GROUP>
__global__ void __launch_bounds__(32 * kWarps, CTAS) k_q4_rows(RowsParams p) {
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    constexpr int SL = sizeof(T) == 4 ? 3 : 1;
    constexpr int WK = kWarps / WR;
    constexpr int COLS = 8 * NT;
    constexpr int TOK = COLS / SL;               // rows of A per pass
    constexpr int ROWS = WR * RBW * 16;          // weight rows of the CTA
    constexpr int FLUSH = GROUP / 32;            // 32-value steps per group
    extern __shared__ __align__(16) uint8_t smem[];
    const int pitch = p.kstage + 32;             // 16-bit values between columns
    uint16_t* xs = reinterpret_cast<uint16_t*>(smem);
    float* red = reinterpret_cast<float*>(smem); // reused after the last product: [WK][COLS][ROWS]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wr = warp % WR, wk = warp / WR;
    const uint32_t rank = cluster_rank(), csize = cluster_size();
    int e = 0, r0 = 0, r1 = p.R;
    if (p.offsets && !nth_expert(p.offsets, p.E, blockIdx.y, p.R, e, r0, r1)) return;   // the whole cluster returns
    const long rb0 = (long)(blockIdx.x / csize) * (WR * RBW);
    const long kbeg = (long)rank * p.kspan, kend = min(p.K, kbeg + p.kspan);
    const int units = (int)((kend - kbeg + 127) / 128);          // of the CTA; this warp's are wk, wk + WK, ...
    const T* A = static_cast<const T*>(p.A);
    // The lane's codes and scale words of this warp's row blocks, at the CTA's first value of K. What lies behind the
    // last row block, tile or group is not guarded against but read again from the last one: its products belong to
    // rows that are not stored or meet the zeros staged behind K.
    const uint4* codes[RBW];
    const uint32_t* scales[RBW];
#pragma unroll
    for (int r = 0; r < RBW; ++r) {
        const size_t b = (size_t)e * p.l.nb + min(rb0 + wr * RBW + r, p.l.nb - 1);
        codes[r] = reinterpret_cast<const uint4*>(p.packed) + (b * p.l.kb + kbeg / 64) * 32 + lane;
        scales[r] = reinterpret_cast<const uint32_t*>(p.packed + p.l.scales_at) + (b * p.l.groups + kbeg / GROUP) * 8 + g;
    }
    const int kb1 = (int)(p.l.kb - kbeg / 64) - 1, gr1 = (int)(p.l.groups - kbeg / GROUP) - 1;

    uint4 cd[D][RBW][2];
    uint32_t sc[D][RBW][4 / FLUSH];
    auto load = [&](int d, int unit) {
#pragma unroll
        for (int r = 0; r < RBW; ++r) {
            cd[d][r][0] = ld_codes(codes[r] + 64 * unit);
            cd[d][r][1] = ld_codes(codes[r] + 32 * min(2 * unit + 1, kb1));
#pragma unroll
            for (int j = 0; j < 4 / FLUSH; ++j)
                sc[d][r][j] = __ldg(scales[r] + 8 * (j ? min(unit * (4 / FLUSH) + j, gr1) : unit * (4 / FLUSH)));
        }
    };

    for (int c0 = r0; c0 < r1; c0 += TOK) {
        const int toks = min(TOK, r1 - c0), cols = toks * SL;
        float acc[RBW][NT][4];
#pragma unroll
        for (int r = 0; r < RBW; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[r][n][j] = 0.f;
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (wk + d * WK < units) load(d, wk + d * WK);

        int unit = wk;
        for (int u0 = 0; u0 < units; u0 += p.kstage / 128) {     // a multiple of WK * D units, or all of them
            const int u1 = min(units, u0 + p.kstage / 128);
            const int span = (u1 - u0) * 128;
            const long ks = kbeg + (long)u0 * 128;
            if (u0) __syncthreads();
            stage_rows<T>(xs, pitch, A + (size_t)c0 * p.lda + ks, p.lda, toks, span, (int)min((long)span, p.K - ks), p.vec);
            if (SL == 1) asm volatile("cp.async.wait_all;" ::: "memory");
            __syncthreads();
            // columns that are not there repeat the last one; their products are not stored
            const uint16_t* xk[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) xk[n] = xs + min(8 * n + g, cols - 1) * pitch + 8 * t - u0 * 128;
            while (unit < u1) {
#pragma unroll
                for (int d = 0; d < D; ++d) {
                    if (unit >= u1) break;
                    float tmp[RBW][NT][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {   // 32 values of K: half i & 1 of tile i >> 1
                        uint32_t a[RBW][2][4];
#pragma unroll
                        for (int r = 0; r < RBW; ++r) {
                            const uint4 c = cd[d][r][i >> 1];
                            const uint32_t w0 = (i & 1) ? c.z : c.x, w1 = (i & 1) ? c.w : c.y;
                            code_pairs<BF16>(w0, a[r][0]);
                            code_pairs<BF16>(w1, a[r][1]);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint4 x = *reinterpret_cast<const uint4*>(xk[n] + unit * 128 + 32 * i);
#pragma unroll
                            for (int r = 0; r < RBW; ++r) {
                                if (i % FLUSH == 0) mma16816_zero<BF16>(tmp[r][n], a[r][0][0], a[r][1][0], a[r][0][1], a[r][1][1], x.x, x.y);
                                else mma16816<BF16>(tmp[r][n], a[r][0][0], a[r][1][0], a[r][0][1], a[r][1][1], x.x, x.y);
                                mma16816<BF16>(tmp[r][n], a[r][0][2], a[r][1][2], a[r][0][3], a[r][1][3], x.z, x.w);
                            }
                        }
                        if (i % FLUSH == FLUSH - 1)
#pragma unroll
                            for (int r = 0; r < RBW; ++r) {
                                const float s0 = bf16_lo(sc[d][r][i / FLUSH]), s1 = bf16_hi(sc[d][r][i / FLUSH]);
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    acc[r][n][0] = fmaf(s0, tmp[r][n][0], acc[r][n][0]);
                                    acc[r][n][1] = fmaf(s0, tmp[r][n][1], acc[r][n][1]);
                                    acc[r][n][2] = fmaf(s1, tmp[r][n][2], acc[r][n][2]);
                                    acc[r][n][3] = fmaf(s1, tmp[r][n][3], acc[r][n][3]);
                                }
                            }
                    }
                    if (unit + D * WK < units) load(d, unit + D * WK);
                    unit += WK;
                }
            }
        }
        // partial sums: the warps of a row block in order, then the CTAs of the cluster in order
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RBW; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = (wr * RBW + r) * 16 + g + 8 * (j >> 1), col = 8 * n + 2 * t + (j & 1);
                    red[(wk * COLS + col) * ROWS + row] = acc[r][n][j];
                }
        if (csize > 1) cluster_sync();
        else __syncthreads();
        for (int i = rank * 32 * kWarps + threadIdx.x; i < ROWS * toks; i += csize * 32 * kWarps) {
            const int m = i / ROWS, row = i - m * ROWS;
            const long n = rb0 * 16 + row;
            float y = 0.f;
#pragma unroll
            for (int s = SL - 1; s >= 0; --s) {
                const float* q = red + (m * SL + s) * ROWS + row;
                if (csize == 1) {
#pragma unroll
                    for (int k = 0; k < WK; ++k) y += q[k * COLS * ROWS];
                } else if (WK >= 4) {                // the parts of a CTA, or of the cluster, on their way together
                    for (uint32_t c = 0; c < csize; ++c) {
                        float v[WK];
#pragma unroll
                        for (int k = 0; k < WK; ++k) v[k] = ld_cluster(q + k * COLS * ROWS, c);
#pragma unroll
                        for (int k = 0; k < WK; ++k) y += v[k];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < WK; ++k) {
                        float v[8];
#pragma unroll
                        for (uint32_t c = 0; c < 8; ++c) v[c] = c < csize ? ld_cluster(q + k * COLS * ROWS, c) : 0.f;
#pragma unroll
                        for (uint32_t c = 0; c < 8; ++c)
                            if (c < csize) y += v[c];
                    }
                }
            }
            if (n < p.N) static_cast<T*>(p.C)[(size_t)(c0 + m) * p.ldc + n] = from_float<T>(y * code_unit<BF16>());
        }
        // the next pass, or the exit, waits for the others' reads
        if (csize > 1) cluster_sync();
        else __syncthreads();
    }
}

__global__ void k_cluster_probe() {}   // never launched: what cluster_fits asks about, with shared memory for 1 to 3 CTAs per SM

// CTAs of a cluster that split K, among those whose clusters all run at once, by the work on the busiest SM: a CTA's units
// of 128 values of K per warp, 1.8 times as long for two CTAs on an SM and 2.5 for three, and about five units' time for
// what a CTA does besides. Of equals the larger cluster. Rows x N, K = 4096, groups of 128, against powers of two up to two
// CTAs per SM: 8 x 9216 11.7 -> 8.6 us (7 CTAs), 16 x 5120 9.8 -> 8.6 (6), 48 x 5120 20.1 -> 16.5 (6), 48 x 9216 30.8 -> 25.8 (2).
int k_cluster(long clusters, long K, int step, int wk, int most_per_sm, const ClusterFits& fits) {
    const int slowed[4] = {0, 10, 18, 25};
    int best = 1;
    long least = 0;
    for (int ck = 1; ck <= 8 && (ck == 1 || K >= (long)ck * step); ++ck) {
        const long units = ((K + ck - 1) / ck + 128L * wk - 1) / (128L * wk);
        int per_sm = 1;
        while (per_sm < most_per_sm && clusters > fits.of[per_sm][ck]) ++per_sm;
        if (ck > 1 && clusters > fits.of[per_sm][ck]) continue;
        const long cost = 50 + units * slowed[per_sm];
        if (ck == 1 || cost <= least) {
            least = cost;
            best = ck;
        }
    }
    return best;
}

template <typename T, int NT, int WR, int RBW, int D, int CTAS, int GROUP>
int launch_rows_g(RowsParams p, int num_sms, cudaStream_t st) {
    constexpr int SL = sizeof(T) == 4 ? 3 : 1;
    constexpr int STEP = kWarps / WR * D * 128;                // values of K that the warps hold in flight
    const long groups = (p.l.nb + WR * RBW - 1) / (WR * RBW);
    const int experts = p.offsets ? std::min(p.E, p.R) : 1;
    const ClusterFits* fits = cluster_fits();
    if (!fits) return (int)cudaErrorUnknown;
    // single rows: only while there is an SM for every CTA (a cluster of two takes about 2 us longer to launch than its
    // CTAs alone)
    int ck = 1;
    if (NT == 1 && WR == 1) {
        while (ck < 8 && groups * experts * ck * 2 <= num_sms && p.K >= 2L * ck * STEP) ck *= 2;
    } else {
        ck = k_cluster(groups * experts, p.K, STEP, kWarps / WR, CTAS, *fits);
    }
    p.kspan = (int)(((p.K + ck - 1) / ck + 127) / 128 * 128);
    ck = (int)((p.K + p.kspan - 1) / p.kspan);
    const int cols = SL * std::min(p.R, 8 * NT / SL);
    const int most = std::max(STEP, (218 * 1024 / CTAS / (2 * cols) - 32) / STEP * STEP);
    p.kstage = std::min(p.kspan, most);
    p.vec = (reinterpret_cast<uintptr_t>(p.A) & 15) == 0 && (p.lda * sizeof(T)) % 16 == 0;
    const size_t smem = std::max((size_t)cols * (p.kstage + 32) * 2,
                                 (size_t)(kWarps / WR) * WR * RBW * 16 * 8 * NT * 4);
    auto kern = k_q4_rows<T, NT, WR, RBW, D, CTAS, GROUP>;
    static OncePerDevice once;
    const int e0 = once([&] { return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem); });
    if (e0) return e0;
    if (smem > (size_t)kRowsSmem) return (int)cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ck;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(groups * ck), (unsigned)experts, 1);
    cfg.blockDim = dim3(32 * kWarps, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = ck > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    count_launch();
    if (e != cudaSuccess) return (int)e;
    return (int)cudaGetLastError();
}

template <typename T, int NT, int WR, int RBW, int D, int CTAS>
int launch_rows_n(const RowsParams& p, int group, int num_sms, cudaStream_t st) {
    switch (group) {
        case 32: return launch_rows_g<T, NT, WR, RBW, D, CTAS, 32>(p, num_sms, st);
        case 64: return launch_rows_g<T, NT, WR, RBW, D, CTAS, 64>(p, num_sms, st);
        default: return launch_rows_g<T, NT, WR, RBW, D, CTAS, 128>(p, num_sms, st);
    }
}

// Tiles by the columns of a pass (rows of A, three times as many for FP32). With experts: twice the mean, since rows are
// never dealt evenly and a second pass reads the codes again; and for up to 8 columns few row blocks per CTA until the CTAs
// fill the GPU anyway (8 tokens x 4 of 64 experts, 2048 x 4096: 23 us with 4 row blocks against 25 with 16 and 27 with 2;
// 64 x 8 of 256, 2048 x 1024: 68 us with 4, 59 with 16).
template <typename T>
int launch_rows_t(const RowsParams& p, int group, int num_sms, cudaStream_t st) {
    const int experts = p.offsets ? std::min(p.E, p.R) : 1;
    const long cols = (long)((p.R + experts - 1) / experts) * (sizeof(T) == 4 ? 3 : 1) * (p.offsets ? 2 : 1);
    if (p.offsets && cols <= 8 && p.l.nb * experts < 32L * num_sms)
        return launch_rows_n<T, 1, 2, 2, 2, 2>(p, group, num_sms, st);
    if (!p.offsets && cols <= 3) return launch_rows_n<T, 1, 1, 2, 2, 2>(p, group, num_sms, st);
    if (cols <= 8) return launch_rows_n<T, 1, 8, 2, 2, 2>(p, group, num_sms, st);
    if (cols <= 16) return launch_rows_n<T, 2, 8, 2, 2, 2>(p, group, num_sms, st);
    if (cols <= 24) {
        // scales of four groups per unit and two row blocks do not fit the registers beside three column tiles
        // (24 x 5001 x 7013, groups of 32: 23.0 against 20.8 us; 24 x 8192 x 8192, groups of 128: 19.7 against 26.0)
        if (group == 32) return launch_rows_g<T, 3, 8, 1, 1, 3, 32>(p, num_sms, st);
        if (group == 64) return launch_rows_g<T, 3, 8, 2, 1, 2, 64>(p, num_sms, st);
        return launch_rows_g<T, 3, 8, 2, 1, 2, 128>(p, num_sms, st);
    }
    if (cols <= 32) return launch_rows_n<T, 4, 8, 1, 2, 2>(p, group, num_sms, st);
    return launch_rows_n<T, 6, 8, 1, 2, 2>(p, group, num_sms, st);
}

}  // namespace

const ClusterFits* cluster_fits() {
    static ClusterFits known[64];
    static std::atomic<unsigned long long> have{0};
    static std::mutex lock;
    static thread_local ClusterFits other;           // devices past 64
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (have.load(std::memory_order_acquire) & bit)) return &known[dev];
    std::lock_guard<std::mutex> hold(lock);
    ClusterFits& f = dev < 64 ? known[dev] : other;
    if (dev < 64 && (have.load(std::memory_order_acquire) & bit)) return &f;
    if (cudaFuncSetAttribute(k_cluster_probe, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) return nullptr;
    for (int per_sm = 1; per_sm <= 3; ++per_sm)
        for (int ctas = 1; ctas <= 8; ++ctas) {
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = ctas;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3(ctas, 1, 1);
            cfg.blockDim = dim3(256, 1, 1);
            cfg.dynamicSmemBytes = 200 * 1024 / per_sm;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&f.of[per_sm][ctas], k_cluster_probe, &cfg) != cudaSuccess) return nullptr;
        }
    if (dev < 64) have.fetch_or(bit, std::memory_order_release);
    return &f;
}

size_t q4_bytes(int E, int N, long K, int group) { return layout(E, N, K, group).bytes; }

template <typename T, int GROUP>
static int pack_g(const T* W, long ldw, int E, int N, long K, uint8_t* packed, int num_sms, cudaStream_t st) {
    const Layout l = layout(E, N, K, GROUP);
    const long pairs = (long)E * l.nb * ((l.kb + 1) / 2);
    if ((reinterpret_cast<uintptr_t>(W) & 15) == 0 && (ldw * sizeof(T)) % 16 == 0) {
        const int grid = (int)std::min((pairs + 7) / 8, 16L * num_sms);
        k_q4_pack<T, GROUP><<<grid, 256, 0, st>>>(W, ldw, E, N, K, l, packed);
    } else {
        const int grid = (int)std::min(pairs, 32L * num_sms);
        k_q4_pack_rows<T, GROUP><<<grid, 256, 0, st>>>(W, ldw, E, N, K, l, packed);
    }
    count_launch();
    return (int)cudaGetLastError();
}

template <typename T>
static int pack_t(const void* W, long ldw, int E, int N, long K, int group, void* packed, int num_sms, cudaStream_t st) {
    const T* w = static_cast<const T*>(W);
    uint8_t* o = static_cast<uint8_t*>(packed);
    if (group == 32) return pack_g<T, 32>(w, ldw, E, N, K, o, num_sms, st);
    if (group == 64) return pack_g<T, 64>(w, ldw, E, N, K, o, num_sms, st);
    return pack_g<T, 128>(w, ldw, E, N, K, o, num_sms, st);
}

int launch_q4_pack(const void* W, long ldw, int dtype, int E, int N, long K, int group, void* packed, int num_sms,
                   void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == EMU_DTYPE_F32) return pack_t<float>(W, ldw, E, N, K, group, packed, num_sms, st);
    if (dtype == EMU_DTYPE_F16) return pack_t<__half>(W, ldw, E, N, K, group, packed, num_sms, st);
    return pack_t<__nv_bfloat16>(W, ldw, E, N, K, group, packed, num_sms, st);
}

int launch_q4_unpack(const void* packed, int E, int N, long K, int group, float* W, long ldw, int num_sms,
                     void* stream) {
    const Layout l = layout(E, N, K, group);
    const long units = (long)E * l.nb * l.kb;
    const int grid = (int)std::min((units + 7) / 8, 32L * num_sms);
    const bool vec = (reinterpret_cast<uintptr_t>(W) & 15) == 0 && ldw % 4 == 0 && K % 4 == 0;
    auto kern = vec ? k_q4_unpack<true> : k_q4_unpack<false>;
    kern<<<grid, 256, 0, (cudaStream_t)stream>>>(static_cast<const uint8_t*>(packed), E, N, K, group, l, W, ldw);
    count_launch();
    return (int)cudaGetLastError();
}

int launch_q4_rows(const Q4GemmArgs& a, void* stream) {
    RowsParams p{};
    p.A = a.A; p.lda = a.lda;
    p.packed = static_cast<const uint8_t*>(a.packed);
    p.l = layout(a.E, a.N, a.K, a.group);
    p.C = a.C; p.ldc = a.ldc;
    p.offsets = a.offsets;
    p.R = a.R; p.E = a.E; p.N = a.N; p.K = a.K;
    cudaStream_t st = (cudaStream_t)stream;
    if (a.dtype == EMU_DTYPE_F32) return launch_rows_t<float>(p, a.group, a.num_sms, st);
    if (a.dtype == EMU_DTYPE_F16) return launch_rows_t<__half>(p, a.group, a.num_sms, st);
    return launch_rows_t<__nv_bfloat16>(p, a.group, a.num_sms, st);
}

}  // namespace emu
