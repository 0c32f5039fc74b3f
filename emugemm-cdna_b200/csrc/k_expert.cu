// k_expert.cu - rows to their experts and back: stable sort of the slots by expert, the two row movements, and their
// gradients. A slot is one (token, choice) pair, s = token * topk + choice; place[s] is its row among the rows sorted
// by expert, -1 when its expert id is outside [0, E).
#include "q4_common.cuh"

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
__device__ __forceinline__ void cluster_sync() {   // whole warps (.aligned): lanes may have left a loop early
    __syncwarp();
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
// owns a contiguous range of slots, counts its slots per expert (32 at a time, equal ids found by one vote per bit of an
// id: match.any took 23 us for 8192 slots of 256 experts, the votes 9), the counts become starting rows by a scan over
// experts, then CTAs, then warps, and the warp walks its range again handing out rows. Bound: the latency of the two walks
// and the scans.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;

// The lanes whose id is this lane's; `ok` lanes only (the others get an arbitrary mask).
__device__ __forceinline__ unsigned same_id(int id, bool ok, int bits) {
    unsigned m = __ballot_sync(0xffffffffu, ok);
    for (int b = 0; b < bits; ++b) {
        const bool one = (id >> b) & 1;
        const unsigned v = __ballot_sync(0xffffffffu, one);
        m &= one ? v : ~v;
    }
    return m;
}

__global__ void __launch_bounds__(kSortThreads) k_expert_sort(const int* __restrict__ expert, int S, int E, int bits, int per_warp,
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
    auto id_at = [&](int s) { return s + lane < s1 ? __ldg(expert + s + lane) : -1; };
    int next = s0 < s1 ? id_at(s0) : -1;
    for (int s = s0; s < s1; s += 32) {
        const int id = next;
        if (s + 32 < s1) next = id_at(s + 32);
        const bool ok = id >= 0 && id < E;
        const unsigned same = same_id(id, ok, bits);
        if (ok && lane == __ffs(same) - 1) mine[id] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (int x = threadIdx.x; x < E; x += blockDim.x) {
        int sum = 0;
        for (int w0 = 0; w0 < warps; w0 += 8) {
            int c[8];
#pragma unroll
            for (int w = 0; w < 8; ++w) c[w] = w0 + w < warps ? count[(w0 + w) * E + x] : 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                if (w0 + w < warps) count[(w0 + w) * E + x] = sum;
                sum += c[w];
            }
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
    next = s0 < s1 ? id_at(s0) : -1;
    for (int s = s0; s < s1; s += 32) {
        const int id = next;
        if (s + 32 < s1) next = id_at(s + 32);
        const bool ok = id >= 0 && id < E;
        const unsigned same = same_id(id, ok, bits);
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

// A group of 2^lw lanes takes a token's row (2^lw >= 32 lanes only where the row has that many accesses), so that no access
// needs a division to find its row; U accesses of a lane are in flight at a time.
struct RowMap { int lw, per; };   // log2 of lanes per row; rows per CTA of 256 threads

// XS[place[t, j]] = X[t]: every row of X is read once and written topk times. V: bytes per access.
template <int V>
__global__ void __launch_bounds__(256) k_expert_gather(const uint8_t* __restrict__ X, long ldx, const int* __restrict__ place,
                                                       uint8_t* __restrict__ XS, long ldxs, long T, int topk, int chunks,
                                                       int slots, RowMap map) {
    using A = typename Vec<V>::type;
    constexpr int U = 4;
    const int lanes = 1 << map.lw, lane = threadIdx.x & (lanes - 1);
    for (long t = (long)blockIdx.x * map.per + (threadIdx.x >> map.lw); t < T; t += (long)gridDim.x * map.per) {
        const A* x = reinterpret_cast<const A*>(X + t * ldx);
        for (int c0 = lane; c0 < chunks; c0 += U * lanes) {
            A v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c0 + u * lanes < chunks) v[u] = x[c0 + u * lanes];
            for (int j = 0; j < topk; ++j) {
                const int r = __ldg(place + t * topk + j);
                if (r < 0 || r >= slots) continue;
                A* o = reinterpret_cast<A*>(XS + (long)r * ldxs);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (c0 + u * lanes < chunks) o[c0 + u * lanes] = v[u];
            }
        }
    }
}

// Y[t] = sum over j in order of w[t, j] YS[place[t, j]] in FP32, rounded once (w null: 1). Bound: the read of YS.
template <typename T, int V>
__global__ void __launch_bounds__(256) k_expert_combine(const uint8_t* __restrict__ YS, long ldys, const int* __restrict__ place,
                                                        const float* __restrict__ w, uint8_t* __restrict__ Y, long ldy,
                                                        long T_, int topk, int chunks, int slots, RowMap map) {
    using A = typename Vec<V>::type;
    constexpr int N = V / sizeof(T), J = 4, U = V >= 8 ? 1 : 4;
    const int lanes = 1 << map.lw, lane = threadIdx.x & (lanes - 1);
    for (long t = (long)blockIdx.x * map.per + (threadIdx.x >> map.lw); t < T_; t += (long)gridDim.x * map.per) {
        for (int c0 = lane; c0 < chunks; c0 += U * lanes) {
            float acc[U][N];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < N; ++k) acc[u][k] = 0.f;
            for (int j0 = 0; j0 < topk; j0 += J) {   // J rows read before any is added
                A v[J][U];
                float f[J];
                bool on[J];
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int r = j0 + j < topk ? __ldg(place + t * topk + j0 + j) : -1;
                    on[j] = r >= 0 && r < slots;
                    f[j] = on[j] && w ? __ldg(w + t * topk + j0 + j) : 1.f;
                    if (on[j]) {
                        const A* x = reinterpret_cast<const A*>(YS + (long)r * ldys);
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (c0 + u * lanes < chunks) v[j][u] = x[c0 + u * lanes];
                    }
                }
#pragma unroll
                for (int j = 0; j < J; ++j)
                    if (on[j])
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            if (c0 + u * lanes >= chunks) continue;
                            const T* x = reinterpret_cast<const T*>(&v[j][u]);
#pragma unroll
                            for (int k = 0; k < N; ++k) acc[u][k] = fmaf(f[j], to_f<T>(x[k]), acc[u][k]);
                        }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                A o;
                T* y = reinterpret_cast<T*>(&o);
#pragma unroll
                for (int k = 0; k < N; ++k) y[k] = from_f<T>(acc[u][k]);
                if (c0 + u * lanes < chunks) reinterpret_cast<A*>(Y + t * ldy)[c0 + u * lanes] = o;
            }
        }
    }
}

// dYS[place[t, j]] = w[t, j] dY[t] and dw[t, j] = <dY[t], YS[place[t, j]]>: every row read once (dY once per four choices),
// the products of a slot added per lane, then by shuffles and, where a row has a whole CTA, over the warps in order (no
// atomics). CTA: a CTA per token, else a warp.
template <typename T, int V, bool CTA>
__global__ void __launch_bounds__(256) k_expert_combine_bwd(const uint8_t* __restrict__ dY, long lddy,
                                                            const uint8_t* __restrict__ YS, long ldys,
                                                            const int* __restrict__ place, const float* __restrict__ w,
                                                            uint8_t* __restrict__ dYS, long lddys, float* __restrict__ dw,
                                                            long T_, int topk, int chunks, int slots) {
    using A = typename Vec<V>::type;
    constexpr int N = V / sizeof(T), J = 4, U = V >= 8 ? 2 : 4;
    __shared__ float part[8][J];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
    const int step = CTA ? blockDim.x : 32;
    for (long t = CTA ? (long)blockIdx.x : (long)blockIdx.x * warps + warp; t < T_; t += CTA ? (long)gridDim.x : (long)gridDim.x * warps) {
        for (int j0 = 0; j0 < topk; j0 += J) {
            int r[J];
            float f[J], dot[J];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                r[j] = j0 + j < topk ? __ldg(place + t * topk + j0 + j) : -1;
                if (r[j] >= slots) r[j] = -1;
                f[j] = j0 + j < topk ? __ldg(w + t * topk + j0 + j) : 1.f;
                dot[j] = 0.f;
            }
            for (int i = CTA ? threadIdx.x : lane; i < chunks; i += U * step) {
                A dv[U], ys[U][J];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int c = i + u * step;
                    if (c >= chunks) continue;
                    dv[u] = reinterpret_cast<const A*>(dY + t * lddy)[c];
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        if (r[j] >= 0) ys[u][j] = reinterpret_cast<const A*>(YS + (long)r[j] * ldys)[c];
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int c = i + u * step;
                    if (c >= chunks) continue;
                    const T* d = reinterpret_cast<const T*>(&dv[u]);
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        if (r[j] < 0) continue;
                        const T* y = reinterpret_cast<const T*>(&ys[u][j]);
                        A o;
                        T* q = reinterpret_cast<T*>(&o);
#pragma unroll
                        for (int k = 0; k < N; ++k) {
                            const float x = to_f<T>(d[k]);
                            dot[j] = fmaf(x, to_f<T>(y[k]), dot[j]);
                            q[k] = from_f<T>(f[j] * x);
                        }
                        reinterpret_cast<A*>(dYS + (long)r[j] * lddys)[c] = o;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], s);
                if (CTA && lane == 0) part[warp][j] = dot[j];
                if (!CTA && lane == j && j0 + j < topk) dw[t * topk + j0 + j] = dot[j];
            }
            if (CTA) {
                __syncthreads();
                if (threadIdx.x < J && j0 + threadIdx.x < topk) {
                    float sum = 0.f;
                    for (int k = 0; k < warps; ++k) sum += part[k][threadIdx.x];
                    dw[t * topk + j0 + threadIdx.x] = sum;
                }
                __syncthreads();
            }
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

RowMap row_map(int chunks) {
    RowMap m{5, 8};
    while (m.lw < 8 && (1 << m.lw) < chunks) ++m.lw;      // a row of up to 256 accesses in one step
    while (m.lw > 1 && (1 << (m.lw - 1)) >= chunks) --m.lw;
    m.per = 256 >> m.lw;
    return m;
}
int row_grid(long T, const RowMap& m, int num_sms) { return (int)std::max(1L, std::min((T + m.per - 1) / m.per, 32L * num_sms)); }

template <typename T, int V>
int combine_v(const ExpertRows& a, cudaStream_t st) {
    const int chunks = (int)(a.H * sizeof(T) / V);
    const RowMap m = row_map(chunks);
    k_expert_combine<T, V><<<row_grid(a.T, m, a.num_sms), 256, 0, st>>>(
        (const uint8_t*)a.S, a.lds * (long)sizeof(T), a.place, a.w, (uint8_t*)a.Y, a.ldy * (long)sizeof(T), a.T, a.topk,
        chunks, (int)(a.T * a.topk), m);
    count_launch();
    return (int)cudaGetLastError();
}

template <typename T, int V>
int combine_bwd_v(const ExpertRows& a, cudaStream_t st) {
    const int chunks = (int)(a.H * sizeof(T) / V);
    const long s = sizeof(T);
    // A warp walks a short row, and a row of narrow accesses where there are tokens enough for 16 warps on each SM
    // (8192 rows of 1111 fp16: 22 us against 27 with a CTA each); a CTA of 128 threads the others (8192 x 4 rows of 4096
    // bf16: 95 us against 101 with a warp each or with 256 threads).
    if ((chunks <= 128 && a.T >= 2L * a.num_sms) || (V <= 4 && a.T >= 16L * a.num_sms)) {
        const int grid = (int)std::min((a.T + 7) / 8, 32L * a.num_sms);
        k_expert_combine_bwd<T, V, false><<<grid, 256, 0, st>>>(
            (const uint8_t*)a.X, a.ldx * s, (const uint8_t*)a.S, a.lds * s, a.place, a.w, (uint8_t*)a.DS, a.ldds * s, a.dw, a.T,
            a.topk, chunks, (int)(a.T * a.topk));
    } else {
        const int threads = std::min(128, std::max(32, (chunks + 31) / 32 * 32));
        const int grid = (int)std::min(a.T, 16L * a.num_sms);
        k_expert_combine_bwd<T, V, true><<<grid, threads, 0, st>>>(
            (const uint8_t*)a.X, a.ldx * s, (const uint8_t*)a.S, a.lds * s, a.place, a.w, (uint8_t*)a.DS, a.ldds * s, a.dw, a.T,
            a.topk, chunks, (int)(a.T * a.topk));
    }
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
    // one CTA up to 4096 slots (4 walks of a warp), else a cluster of 8
    const int ctas = S <= 4096 ? 1 : 8;
    const int warps = ctas > 1 ? kSortWarps : std::max(1, std::min(kSortWarps, (S + 31) / 32));
    const long warps_all = (long)ctas * warps;
    const int per_warp = (int)(((S + warps_all - 1) / warps_all + 31) / 32 * 32);
    int bits = 0;
    while ((1 << bits) < E) ++bits;
    const size_t smem = (size_t)(warps + 2) * E * 4;
    static OncePerDevice once;
    const int e0 = once([] {
        return (int)cudaFuncSetAttribute(k_expert_sort, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (kSortWarps + 2) * kMaxExperts * 4);
    });
    if (e0) return e0;
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
    cfg.numAttrs = ctas > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k_expert_sort, expert, S, E, bits, per_warp, order, place, offsets);
    count_launch();
    if (e != cudaSuccess) return (int)e;
    return (int)cudaGetLastError();
}

int launch_expert_gather(const ExpertRows& a, int dtype, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    const long s = dtype == EMU_DTYPE_F32 ? 4 : 2;
    const int v = access_bytes({(uintptr_t)a.X, (uintptr_t)(a.ldx * s), (uintptr_t)a.DS, (uintptr_t)(a.ldds * s),
                                (uintptr_t)(a.H * s)}, (int)s);
    const int chunks = (int)(a.H * s / v), slots = (int)(a.T * a.topk);
    const RowMap m = row_map(chunks);
    const int grid = row_grid(a.T, m, a.num_sms);
    const uint8_t* X = (const uint8_t*)a.X;
    uint8_t* XS = (uint8_t*)a.DS;
    if (v == 16) k_expert_gather<16><<<grid, 256, 0, st>>>(X, a.ldx * s, a.place, XS, a.ldds * s, a.T, a.topk, chunks, slots, m);
    else if (v == 8) k_expert_gather<8><<<grid, 256, 0, st>>>(X, a.ldx * s, a.place, XS, a.ldds * s, a.T, a.topk, chunks, slots, m);
    else if (v == 4) k_expert_gather<4><<<grid, 256, 0, st>>>(X, a.ldx * s, a.place, XS, a.ldds * s, a.T, a.topk, chunks, slots, m);
    else k_expert_gather<2><<<grid, 256, 0, st>>>(X, a.ldx * s, a.place, XS, a.ldds * s, a.T, a.topk, chunks, slots, m);
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
