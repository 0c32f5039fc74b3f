// k_q4.cu - 4-bit weights with group scales: packing, unpacking, and the product for few rows.
#include "q4_common.cuh"

#include <algorithm>
#include <type_traits>

namespace emu {

namespace {

using namespace q4;

// ------------------------------------------------------------------------------------------------- pack and unpack
// s = bf16(fp32(max|w| / 7)) of a group, q = w / s rounded to the nearest integer (even on a tie), at most 7 away.
// The quotient in FP32 can round onto a tie that w / s itself is not on, so q is checked with the residual w - q s:
// |w| <= 7.1 s, so it has at most 24 significant bits where it matters and fmaf gives it exactly.
// s below 2^-100: w and s times 2^64 first, so that 1 / s and s / 2 are normal floats; the quotient is the same.
__device__ __forceinline__ int quantise(float w, float s, float inv) {
    float q = rintf(w * inv);
    const float r = fmaf(-q, s, w), h = 0.5f * s;
    const bool odd = ((int)q) & 1;
    if (r > h || (r == h && odd)) q += 1.f;
    else if (r < -h || (r == -h && odd)) q -= 1.f;
    return (int)fminf(fmaxf(q, -7.f), 7.f);
}

// One warp per tile pair: 16 rows x 128 values of K (two tiles, 4, 2 or 1 groups per row). Lane (g, t) reads rows g and
// g + 8 at k = 32i + 8t .. +7 (i = 0..3): the values its own words of the two tiles hold. A group of 32 is then one i of
// four lanes, so the group maximum is two shuffles, for groups of 64 and 128 after combining i pairwise in registers.
// Bound: the read of W (4 or 2 bytes a value against half a byte written).
template <typename T, int GROUP>
__global__ void __launch_bounds__(256) k_q4_pack(const T* __restrict__ W, long ldw, int E, int N, long K, Layout l,
                                                 uint8_t* __restrict__ packed, int vec) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long kp = (l.kb + 1) / 2;
    const long units = (long)E * l.nb * kp;
    uint16_t* scales = reinterpret_cast<uint16_t*>(packed + l.scales_at);
    for (long u = (long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (long)gridDim.x * 8) {
        const long k128 = u % kp, b = u / kp;     // b = expert * nb + row block
        const long e = b / l.nb;
        const int n0 = (int)(b % l.nb) * 16;
        float v[2][32];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int n = n0 + g + 8 * half;
            const T* row = W + ((size_t)e * N + n) * ldw;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long k = k128 * 128 + 32 * i + 8 * t;
                float* x = v[half] + 8 * i;
                if (n < N && vec && k + 8 <= K) {
                    if (sizeof(T) == 4) {
                        const float4 a = *reinterpret_cast<const float4*>(row + k);
                        const float4 c = *reinterpret_cast<const float4*>(row + k + 4);
                        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
                        x[4] = c.x; x[5] = c.y; x[6] = c.z; x[7] = c.w;
                    } else {
                        const uint4 a = *reinterpret_cast<const uint4*>(row + k);
                        const T* p = reinterpret_cast<const T*>(&a);
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = to_float<T>(p[j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = (n < N && k + j < K) ? to_float<T>(row[k + j]) : 0.f;
                }
            }
        }
        uint32_t word[2][4];   // [half of the rows][i]
        constexpr int PER = GROUP / 32;   // values of i per group
        float sc[2][4 / PER];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int gi = 0; gi < 4 / PER; ++gi) {
                // the maximum of the magnitudes' bits, in which Inf and NaN come out above every number
                unsigned m = 0;
#pragma unroll
                for (int j = 0; j < 8 * PER; ++j)
                    m = max(m, __float_as_uint(v[half][8 * PER * gi + j]) & 0x7fffffffu);
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const bool bad = m >= 0x7f800000u;
                float s = bad ? __uint_as_float(0x7fc00000u)
                              : __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__uint_as_float(m), 7.f)));
                sc[half][gi] = s;
                const bool tiny = s < 0x1p-100f;
                const float up = tiny ? 0x1p64f : 1.f;
                const float su = s * up, inv = 1.f / su;
                const bool none = bad || s == 0.f;
#pragma unroll
                for (int ii = 0; ii < PER; ++ii) {
                    const int i = gi * PER + ii;
                    uint32_t w = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int q = none ? 0 : quantise(v[half][8 * i + j] * up, su, inv);
                        w |= (uint32_t)(q + 8) << (4 * (j / 2 + 4 * (j & 1)));
                    }
                    word[half][i] = w;
                }
            }
        uint4* tile = reinterpret_cast<uint4*>(packed) + (size_t)(b * l.kb + 2 * k128) * 32 + lane;
        tile[0] = make_uint4(word[0][0], word[1][0], word[0][1], word[1][1]);
        if (2 * k128 + 1 < l.kb) tile[32] = make_uint4(word[0][2], word[1][2], word[0][3], word[1][3]);
        if (t == 0) {
#pragma unroll
            for (int gi = 0; gi < 4 / PER; ++gi) {
                const long kg = k128 * (4 / PER) + gi;
                if (kg < l.groups) {
                    const uint32_t lo = n0 + g < N ? __float_as_uint(sc[0][gi]) >> 16 : 0u;
                    const uint32_t hi = n0 + g + 8 < N ? __float_as_uint(sc[1][gi]) & 0xffff0000u : 0u;
                    reinterpret_cast<uint32_t*>(scales)[((size_t)b * l.groups + kg) * 8 + g] = lo | hi;
                }
            }
        }
    }
}

// W = s q in FP32 (8 + 3 significant bits: exact). One warp per tile; bound by the write.
__global__ void __launch_bounds__(256) k_q4_unpack(const uint8_t* __restrict__ packed, int E, int N, long K, int group,
                                                   Layout l, float* __restrict__ W, long ldw, int vec) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint16_t* scales = reinterpret_cast<const uint16_t*>(packed + l.scales_at);
    const long units = (long)E * l.nb * l.kb;
    for (long u = (long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (long)gridDim.x * 8) {
        const long kb = u % l.kb, b = u / l.kb, e = b / l.nb;
        const int n0 = (int)(b % l.nb) * 16;
        const uint4 c = reinterpret_cast<const uint4*>(packed)[(size_t)u * 32 + lane];
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + g + 8 * (i & 1);
            const long k = kb * 64 + 32 * (i >> 1) + 8 * t;
            if (n >= N || k >= K) continue;
            const float s = __uint_as_float(
                (uint32_t)scales[(((size_t)b * l.groups + k / group) * 8 + g) * 2 + (i & 1)] << 16);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = s * (float)((int)((w[i] >> (4 * (j / 2 + 4 * (j & 1)))) & 15u) - 8);
            float* row = W + ((size_t)e * N + n) * ldw + k;
            if (vec && k + 8 <= K) {
                reinterpret_cast<float4*>(row)[0] = make_float4(x[0], x[1], x[2], x[3]);
                reinterpret_cast<float4*>(row)[1] = make_float4(x[4], x[5], x[6], x[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k + j < K) row[j] = x[j];
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
constexpr int kRowsSmem = 100 * 1024;

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
__device__ __forceinline__ void cluster_sync() {
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
    for (int base = 0; base < E; base += 32) {
        const int x = base + lane;
        const int a = x < E ? offsets[x] : 0, b = x < E ? offsets[x + 1] : 0;
        const unsigned some = __ballot_sync(0xffffffffu, b > a);
        const int n = __popc(some);
        if (i < n) {
            unsigned m = some;
            for (int j = 0; j < i; ++j) m &= m - 1;
            const int src = __ffs(m) - 1;
            e = base + src;
            r0 = max(0, __shfl_sync(0xffffffffu, a, src));
            r1 = min(R, __shfl_sync(0xffffffffu, b, src));   // a bad offset reads and writes no row outside of A and C
            return true;
        }
        i -= n;
    }
    return false;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {   // the rest of 16 is zeroed
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
            for (int m = 0; m < toks; ++m) {
                const T* row = A + (size_t)(c0 + m) * p.lda + ks;
                const int len = (int)min((long)span, p.K - ks);
                for (int k = threadIdx.x * 8; k < span; k += 256 * kWarps) {
                    if (SL == 1 && p.vec) {
                        const int left = len - k;
                        cp_async16(static_cast<uint32_t>(__cvta_generic_to_shared(xs + m * pitch + k)),
                                   left > 0 ? row + k : A, left <= 0 ? 0 : left >= 8 ? 16 : 2 * left);
                        continue;
                    }
                    T x[8];
                    if (p.vec && k + 8 <= len) {
#pragma unroll
                        for (int j = 0; j < 8 * (int)sizeof(T) / 16; ++j)
                            reinterpret_cast<uint4*>(x)[j] = __ldg(reinterpret_cast<const uint4*>(row + k) + j);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = k + j < len ? row[k + j] : from_float<T>(0.f);
                    }
                    if (SL == 3) {
                        __align__(16) uint16_t s[3][8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) slice3(to_float<T>(x[j]), s[0][j], s[1][j], s[2][j]);
#pragma unroll
                        for (int q = 0; q < 3; ++q)
                            *reinterpret_cast<uint4*>(xs + (3 * m + q) * pitch + k) = *reinterpret_cast<const uint4*>(s[q]);
                    } else {
                        *reinterpret_cast<uint4*>(xs + m * pitch + k) = *reinterpret_cast<const uint4*>(x);
                    }
                }
            }
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
                        if (i % FLUSH == 0)
#pragma unroll
                            for (int r = 0; r < RBW; ++r)
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int j = 0; j < 4; ++j) tmp[r][n][j] = 0.f;
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
                                mma16816<BF16>(tmp[r][n], a[r][0][0], a[r][1][0], a[r][0][1], a[r][1][1], x.x, x.y);
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
            for (int s = SL - 1; s >= 0; --s)
                for (uint32_t c = 0; c < csize; ++c)
#pragma unroll
                    for (int k = 0; k < WK; ++k) {
                        const float* q = red + (k * COLS + m * SL + s) * ROWS + row;
                        y += csize > 1 ? ld_cluster(q, c) : *q;
                    }
            if (n < p.N) static_cast<T*>(p.C)[(size_t)(c0 + m) * p.ldc + n] = from_float<T>(y * code_unit<BF16>());
        }
        // the next pass, or the exit, waits for the others' reads
        if (csize > 1) cluster_sync();
        else __syncthreads();
    }
}

template <typename T, int NT, int WR, int RBW, int D, int CTAS, int GROUP>
int launch_rows_g(RowsParams p, int num_sms, cudaStream_t st) {
    constexpr int SL = sizeof(T) == 4 ? 3 : 1;
    constexpr int STEP = kWarps / WR * D * 128;                // values of K that the warps hold in flight
    const long groups = (p.l.nb + WR * RBW - 1) / (WR * RBW);
    const int experts = p.offsets ? std::min(p.E, p.R) : 1;
    // K split over a cluster while all CTAs are resident at once and each keeps a step of its warps
    int ck = 1;
    while (ck < 8 && groups * experts * ck * 2 <= (long)CTAS * num_sms && p.K >= 2L * ck * STEP) ck *= 2;
    p.kspan = (int)(((p.K + ck - 1) / ck + 127) / 128 * 128);
    ck = (int)((p.K + p.kspan - 1) / p.kspan);
    const int cols = SL * std::min(p.R, 8 * NT / SL);
    const int most = std::max(STEP, (196 * 1024 / CTAS / (2 * cols) - 32) / STEP * STEP);
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

template <typename T>
int launch_rows_t(const RowsParams& p, int group, int num_sms, cudaStream_t st) {
    const int experts = p.offsets ? std::min(p.E, p.R) : 1;
    const long cols = (long)((p.R + experts - 1) / experts) * (sizeof(T) == 4 ? 3 : 1);
    if (cols <= 3) return launch_rows_n<T, 1, 1, 1, 2, 4>(p, group, num_sms, st);
    if (cols <= 8) return launch_rows_n<T, 1, 4, 1, 2, 4>(p, group, num_sms, st);
    if (cols <= 16) return launch_rows_n<T, 2, 4, 1, 2, 3>(p, group, num_sms, st);
    if (cols <= 24) return launch_rows_n<T, 3, 4, 2, 1, 2>(p, group, num_sms, st);
    if (cols <= 32) return launch_rows_n<T, 4, 4, 2, 1, 2>(p, group, num_sms, st);
    return launch_rows_n<T, 6, 4, 1, 2, 2>(p, group, num_sms, st);
}

}  // namespace

size_t q4_bytes(int E, int N, long K, int group) { return layout(E, N, K, group).bytes; }

template <typename T>
static int pack_t(const void* W, long ldw, int E, int N, long K, int group, void* packed, int num_sms, cudaStream_t st) {
    const Layout l = layout(E, N, K, group);
    const long units = (long)E * l.nb * ((l.kb + 1) / 2);
    const int vec = (reinterpret_cast<uintptr_t>(W) & 15) == 0 && (ldw * sizeof(T)) % 16 == 0;
    const int grid = (int)std::min((units + 7) / 8, 8L * num_sms);
    const T* w = static_cast<const T*>(W);
    uint8_t* o = static_cast<uint8_t*>(packed);
    if (group == 32) k_q4_pack<T, 32><<<grid, 256, 0, st>>>(w, ldw, E, N, K, l, o, vec);
    else if (group == 64) k_q4_pack<T, 64><<<grid, 256, 0, st>>>(w, ldw, E, N, K, l, o, vec);
    else k_q4_pack<T, 128><<<grid, 256, 0, st>>>(w, ldw, E, N, K, l, o, vec);
    count_launch();
    return (int)cudaGetLastError();
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
    const int vec = (reinterpret_cast<uintptr_t>(W) & 15) == 0 && ldw % 4 == 0;
    const int grid = (int)std::min((units + 7) / 8, 16L * num_sms);
    k_q4_unpack<<<grid, 256, 0, (cudaStream_t)stream>>>(static_cast<const uint8_t*>(packed), E, N, K, group, l, W, ldw,
                                                        vec);
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
