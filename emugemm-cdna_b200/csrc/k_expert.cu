// k_expert.cu - rows to their experts and back: stable sort of the slots by expert, the two row movements, and their
// gradients. A slot is one (token, choice) pair, s = token * topk + choice; place[s] is its row among the rows sorted
// by expert, -1 when its expert id is outside [0, E).
#include "emugemm_internal.h"

#include <algorithm>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace emu {

namespace {

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
__device__ __forceinline__ int ld_cluster(const int* p, uint32_t rank) {
    uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(r));
    return v;
}

// ------------------------------------------------------------------------------------------------------------- sort
// Counting sort in one launch of one cluster, with no atomics, so that slots of one expert keep their order: every warp
// owns a contiguous range of slots, counts its slots per expert (32 at a time, equal ids found by match), the counts
// become starting rows by a scan over experts, then CTAs, then warps, and the warp walks its range again handing out
// rows. Bound: the latency of the two walks and the scans.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;

__global__ void __launch_bounds__(kSortThreads) k_expert_sort(const int* __restrict__ expert, int S, int E, int per_warp,
                                                              int* __restrict__ order, int* __restrict__ place,
                                                              int* __restrict__ offsets) {
    extern __shared__ int sm[];
    int* count = sm;                         // [warps][E]
    int* total = sm + (blockDim.x / 32) * E; // [E] of this CTA
    int* base = total + E;                   // [E] first row of this CTA's slots
    __shared__ int part[kSortWarps + 1];
    const int warps = blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), csize = cluster_size();
    for (int i = threadIdx.x; i < warps * E; i += blockDim.x) count[i] = 0;
    __syncthreads();
    const long first = ((long)rank * warps + warp) * per_warp;
    const int s0 = (int)min((long)S, first), s1 = (int)min((long)S, first + per_warp);
    int* mine = count + warp * E;
    for (int s = s0; s < s1; s += 32) {
        const int id = s + lane < s1 ? expert[s + lane] : -1;
        const bool ok = id >= 0 && id < E;
        const unsigned same = __match_any_sync(0xffffffffu, ok ? id : -1);
        if (ok && lane == __ffs(same) - 1) mine[id] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (int x = threadIdx.x; x < E; x += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < warps; ++w) {
            const int c = count[w * E + x];
            count[w * E + x] = sum;
            sum += c;
        }
        total[x] = sum;
    }
    cluster_sync();
    // exclusive scan over experts of the totals of all CTAs, plus the totals of the CTAs before this one
    int run = 0;
    for (int x0 = 0; x0 < E; x0 += blockDim.x) {
        const int x = x0 + threadIdx.x;
        int all = 0, before = 0;
        if (x < E)
            for (uint32_t c = 0; c < csize; ++c) {
                const int v = ld_cluster(total + x, c);
                all += v;
                if (c < rank) before += v;
            }
        int inc = all;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += v;
        }
        if (lane == 31) part[warp] = inc;
        __syncthreads();
        if (warp == 0) {
            int v = lane < warps ? part[lane] : 0;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v += u;
            }
            part[lane] = v;   // inclusive over warps
        }
        __syncthreads();
        const int start = run + (warp ? part[warp - 1] : 0) + inc - all;
        if (x < E) {
            base[x] = start + before;
            if (rank == 0) offsets[x] = start;
        }
        run += part[warps - 1];
        __syncthreads();
    }
    if (rank == 0 && threadIdx.x == 0) offsets[E] = run;
    for (int s = s0; s < s1; s += 32) {
        const int id = s + lane < s1 ? expert[s + lane] : -1;
        const bool ok = id >= 0 && id < E;
        const unsigned same = __match_any_sync(0xffffffffu, ok ? id : -1);
        if (ok) {
            const int row = base[id] + mine[id] + __popc(same & ((1u << lane) - 1));
            place[s + lane] = row;
            order[row] = s + lane;
        } else if (s + lane < s1) {
            place[s + lane] = -1;
        }
        __syncwarp();
        if (ok && lane == __ffs(same) - 1) mine[id] += __popc(same);
        __syncwarp();
    }
    for (long r = run + (long)rank * blockDim.x + threadIdx.x; r < S; r += (long)csize * blockDim.x) order[r] = -1;
    cluster_sync();   // no CTA leaves while another still reads its totals
}

// ---------------------------------------------------------------------------------------------------- row movements
template <int BYTES> struct Vec;
template <> struct Vec<16> { using type = uint4; };
template <> struct Vec<8> { using type = uint2; };
template <> struct Vec<4> { using type = uint32_t; };
template <> struct Vec<2> { using type = uint16_t; };

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// XS[place[t, j]] = X[t]: every row of X is read once and written topk times. V: bytes per access.
template <int V>
__global__ void __launch_bounds__(256) k_expert_gather(const uint8_t* __restrict__ X, long ldx, const int* __restrict__ place,
                                                       uint8_t* __restrict__ XS, long ldxs, long T, int topk, int chunks,
                                                       int slots) {
    using U = typename Vec<V>::type;
    const long n = T * chunks;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long t = i / chunks;
        const long c = (i - t * chunks) * V;
        const U v = *reinterpret_cast<const U*>(X + t * ldx + c);
        for (int j = 0; j < topk; ++j) {
            const int r = place[t * topk + j];
            if (r >= 0 && r < slots) *reinterpret_cast<U*>(XS + (long)r * ldxs + c) = v;
        }
    }
}

// Y[t] = sum over j in order of w[t, j] YS[place[t, j]] in FP32, rounded once (w null: 1). Bound: the read of YS.
template <typename T, int V>
__global__ void __launch_bounds__(256) k_expert_combine(const uint8_t* __restrict__ YS, long ldys, const int* __restrict__ place,
                                                        const float* __restrict__ w, uint8_t* __restrict__ Y, long ldy,
                                                        long T_, int topk, int chunks, int slots) {
    using U = typename Vec<V>::type;
    constexpr int N = V / sizeof(T);
    const long n = T_ * chunks;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long t = i / chunks;
        const long c = (i - t * chunks) * V;
        float acc[N];
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = 0.f;
        for (int j = 0; j < topk; ++j) {
            const int r = place[t * topk + j];
            if (r < 0 || r >= slots) continue;
            const float f = w ? w[t * topk + j] : 1.f;
            const U u = *reinterpret_cast<const U*>(YS + (long)r * ldys + c);
            const T* x = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] = fmaf(f, to_f<T>(x[k]), acc[k]);
        }
        U o;
        T* y = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int k = 0; k < N; ++k) y[k] = from_f<T>(acc[k]);
        *reinterpret_cast<U*>(Y + t * ldy + c) = o;
    }
}

// dYS[place[t, j]] = w[t, j] dY[t] and dw[t, j] = <dY[t], YS[place[t, j]]>: one CTA per token, every row read once, the
// products of a slot added per thread, then by shuffles and over the warps in order (no atomics).
template <typename T, int V>
__global__ void __launch_bounds__(256) k_expert_combine_bwd(const uint8_t* __restrict__ dY, long lddy,
                                                            const uint8_t* __restrict__ YS, long ldys,
                                                            const int* __restrict__ place, const float* __restrict__ w,
                                                            uint8_t* __restrict__ dYS, long lddys, float* __restrict__ dw,
                                                            long T_, int topk, int chunks, int slots) {
    using U = typename Vec<V>::type;
    constexpr int N = V / sizeof(T), J = 4;
    __shared__ float part[8][J];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
    for (long t = blockIdx.x; t < T_; t += gridDim.x) {
        for (int j0 = 0; j0 < topk; j0 += J) {
            int r[J];
            float f[J], dot[J];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                r[j] = j0 + j < topk ? place[t * topk + j0 + j] : -1;
                if (r[j] >= slots) r[j] = -1;
                f[j] = w && j0 + j < topk ? w[t * topk + j0 + j] : 1.f;
                dot[j] = 0.f;
            }
            for (int i = threadIdx.x; i < chunks; i += blockDim.x) {
                const long c = (long)i * V;
                const U u = *reinterpret_cast<const U*>(dY + t * lddy + c);
                const T* d = reinterpret_cast<const T*>(&u);
                U ys[J];
#pragma unroll
                for (int j = 0; j < J; ++j)
                    if (r[j] >= 0) ys[j] = *reinterpret_cast<const U*>(YS + (long)r[j] * ldys + c);
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (r[j] < 0) continue;
                    const T* y = reinterpret_cast<const T*>(&ys[j]);
                    U o;
                    T* q = reinterpret_cast<T*>(&o);
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const float a = to_f<T>(d[k]);
                        dot[j] = fmaf(a, to_f<T>(y[k]), dot[j]);
                        q[k] = from_f<T>(f[j] * a);
                    }
                    *reinterpret_cast<U*>(dYS + (long)r[j] * lddys + c) = o;
                }
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], s);
                if (lane == 0) part[warp][j] = dot[j];
            }
            __syncthreads();
            if (threadIdx.x < J && j0 + threadIdx.x < topk) {
                float sum = 0.f;
                for (int k = 0; k < warps; ++k) sum += part[k][threadIdx.x];
                if (dw) dw[t * topk + j0 + threadIdx.x] = sum;
            }
            __syncthreads();
        }
    }
}

// The widest access (16, 8, 4 or 2 bytes) that all of these addresses and byte strides allow.
int access_bytes(std::initializer_list<uintptr_t> of, int size) {
    uintptr_t all = 16;
    for (uintptr_t v : of) all |= v;
    const int v = (int)(all & (~all + 1));
    return std::max(v, size);
}

int row_grid(long work, int num_sms) { return (int)std::max(1L, std::min((work + 255) / 256, 16L * num_sms)); }

template <typename T, int V>
int combine_v(const ExpertRows& a, cudaStream_t st) {
    const int chunks = (int)(a.H * sizeof(T) / V);
    k_expert_combine<T, V><<<row_grid(a.T * chunks, a.num_sms), 256, 0, st>>>(
        (const uint8_t*)a.S, a.lds * (long)sizeof(T), a.place, a.w, (uint8_t*)a.Y, a.ldy * (long)sizeof(T), a.T, a.topk,
        chunks, (int)(a.T * a.topk));
    count_launch();
    return (int)cudaGetLastError();
}

template <typename T, int V>
int combine_bwd_v(const ExpertRows& a, cudaStream_t st) {
    const int chunks = (int)(a.H * sizeof(T) / V);
    const int threads = std::min(256, std::max(32, (chunks + 31) / 32 * 32));
    const int grid = (int)std::min(a.T, 16L * a.num_sms);
    k_expert_combine_bwd<T, V><<<grid, threads, 0, st>>>(
        (const uint8_t*)a.X, a.ldx * (long)sizeof(T), (const uint8_t*)a.S, a.lds * (long)sizeof(T), a.place, a.w,
        (uint8_t*)a.DS, a.ldds * (long)sizeof(T), a.dw, a.T, a.topk, chunks, (int)(a.T * a.topk));
    count_launch();
    return (int)cudaGetLastError();
}

template <typename T>
int combine_t(const ExpertRows& a, cudaStream_t st) {
    const long s = sizeof(T);
    switch (access_bytes({(uintptr_t)a.S, (uintptr_t)(a.lds * s), (uintptr_t)a.Y, (uintptr_t)(a.ldy * s),
                          (uintptr_t)(a.H * s)}, (int)s)) {
        case 16: return combine_v<T, 16>(a, st);
        case 8: return combine_v<T, 8>(a, st);
        case 4: return combine_v<T, 4>(a, st);
        default: return combine_v<T, (int)sizeof(T)>(a, st);
    }
}

template <typename T>
int combine_bwd_t(const ExpertRows& a, cudaStream_t st) {
    const long s = sizeof(T);
    switch (access_bytes({(uintptr_t)a.S, (uintptr_t)(a.lds * s), (uintptr_t)a.X, (uintptr_t)(a.ldx * s), (uintptr_t)a.DS,
                          (uintptr_t)(a.ldds * s), (uintptr_t)(a.H * s)}, (int)s)) {
        case 16: return combine_bwd_v<T, 16>(a, st);
        case 8: return combine_bwd_v<T, 8>(a, st);
        case 4: return combine_bwd_v<T, 4>(a, st);
        default: return combine_bwd_v<T, (int)sizeof(T)>(a, st);
    }
}

}  // namespace

int launch_expert_sort(const int* expert, int S, int E, int* order, int* place, int* offsets, void* stream) {
    // one CTA up to 8192 slots (8 walks of a warp), else a cluster of 8
    const int ctas = S <= 8192 ? 1 : 8;
    const int warps = ctas > 1 ? kSortWarps : std::max(1, std::min(kSortWarps, (S + 31) / 32));
    const long warps_all = (long)ctas * warps;
    const int per_warp = (int)(((S + warps_all - 1) / warps_all + 31) / 32 * 32);
    const size_t smem = (size_t)(warps + 2) * E * 4;
    cudaError_t e = cudaFuncSetAttribute(k_expert_sort, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (kSortWarps + 2) * kMaxExperts * 4);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(ctas, 1, 1);
    cfg.blockDim = dim3(32 * warps, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, k_expert_sort, expert, S, E, per_warp, order, place, offsets);
    count_launch();
    if (e != cudaSuccess) return (int)e;
    return (int)cudaGetLastError();
}

int launch_expert_gather(const ExpertRows& a, int dtype, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    const long s = dtype == EMU_DTYPE_F32 ? 4 : 2;
    const int v = access_bytes({(uintptr_t)a.X, (uintptr_t)(a.ldx * s), (uintptr_t)a.DS, (uintptr_t)(a.ldds * s),
                                (uintptr_t)(a.H * s)}, (int)s);
    const int chunks = (int)(a.H * s / v), grid = row_grid(a.T * chunks, a.num_sms), slots = (int)(a.T * a.topk);
    const uint8_t* X = (const uint8_t*)a.X;
    uint8_t* XS = (uint8_t*)a.DS;
    if (v == 16) k_expert_gather<16><<<grid, 256, 0, st>>>(X, a.ldx * s, a.place, XS, a.ldds * s, a.T, a.topk, chunks, slots);
    else if (v == 8) k_expert_gather<8><<<grid, 256, 0, st>>>(X, a.ldx * s, a.place, XS, a.ldds * s, a.T, a.topk, chunks, slots);
    else if (v == 4) k_expert_gather<4><<<grid, 256, 0, st>>>(X, a.ldx * s, a.place, XS, a.ldds * s, a.T, a.topk, chunks, slots);
    else k_expert_gather<2><<<grid, 256, 0, st>>>(X, a.ldx * s, a.place, XS, a.ldds * s, a.T, a.topk, chunks, slots);
    count_launch();
    return (int)cudaGetLastError();
}

int launch_expert_combine(const ExpertRows& a, int dtype, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == EMU_DTYPE_F32) return combine_t<float>(a, st);
    if (dtype == EMU_DTYPE_F16) return combine_t<__half>(a, st);
    return combine_t<__nv_bfloat16>(a, st);
}

int launch_expert_combine_bwd(const ExpertRows& a, int dtype, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == EMU_DTYPE_F32) return combine_bwd_t<float>(a, st);
    if (dtype == EMU_DTYPE_F16) return combine_bwd_t<__half>(a, st);
    return combine_bwd_t<__nv_bfloat16>(a, st);
}

}  // namespace emu
