// k_q4_tc.cu - the product with 4-bit weights for many rows, on CTA pairs (tcgen05, cta_group::2).
//
// D (256 weight rows x TN rows of A, in TMEM) += Q (integers of the codes) * A^T: the weights are the MMA's A operand, so
// a thread of the epilogue owns one weight row and a group's scale is one register. Every scale group gets a fresh
// accumulator; the epilogue warps add it to FP32 registers times the scale, so no weight is rounded and the tensor
// cores' truncating accumulation never runs over more than 128 values of K. FP32 A is three bf16 slices (lo, mid, hi
// multiplied in this order into the same accumulator).
//
// Per CTA of a pair: 128 weight rows, TN / 2 rows of A. Six converter warps turn the codes (one 16-byte load is rows g
// and g + 8 at two 8-value chunks) into the 128-byte-swizzled K-major operand in shared memory, rows of A come by TMA,
// each CTA's part completing on the leader's barrier. Warps: 0 = TMA producer, 1 = MMA issuer (leader) and TMEM
// allocator, 2-7 converters, warpgroups 2-3 = scale, sum and store. Registers per warpgroup with setmaxnreg: 80 / 80 / 176 / 176 of
// the launch's 512 x 128. The peer's converters report to the leader by 16-byte bulk copies (as in k_tc_fused.cu).
// All waits are bounded.
#include "device_utils.cuh"
#include "q4_common.cuh"

#include <algorithm>
#include <cuda.h>
#include <cudaTypedefs.h>
#include <type_traits>

namespace emu {

bool tc_get_encode(PFN_cuTensorMapEncodeTiled_v12000* out);

namespace {

using namespace dev;
using namespace q4;

constexpr int kThreads = 512;
constexpr int kEpiWarps = 8, kConvPairs = 3;  // converter warps 2 .. 7 in pairs, a pair per panel in turn
constexpr int kRegEpi = 176, kRegOther = 80;
static_assert(2 * 128 * kRegEpi + 2 * 128 * kRegOther == kThreads * 128, "register split");
constexpr int kPanelA = 128 * 128;            // bytes of a panel of the weights: 128 rows x 64 values of K
constexpr int kMaxStages = 8, kMaxBufs = 4;
constexpr int kSmemMax = 227 * 1024;
constexpr int kSmemFixed = 1024 + 1024 + (kMaxExperts + 1) * 4;   // alignment, barriers, row tiles of the experts

// A stage is one panel: 128 converted weight rows and TN / 2 rows of A (SL slices).
template <int SL, int TN>
struct Cfg {
    static constexpr int PANEL_B = TN / 2 * 128;                  // bytes of one slice
    static constexpr int B_BYTES = SL * PANEL_B;
    static constexpr int STAGE = kPanelA + B_BYTES;
    static constexpr int FIT = (kSmemMax - kSmemFixed) / STAGE;
    static constexpr int STAGES = FIT < kMaxStages ? FIT : kMaxStages;
    static constexpr int BUFS = 512 / TN < kMaxBufs ? 512 / TN : kMaxBufs;
    static constexpr int SMEM = STAGES * STAGE + kSmemFixed;
    static_assert(SMEM <= kSmemMax && TN * 128 * 4 <= STAGES * STAGE, "shared memory");
    // A wait tells apart only two neighbouring phases of a barrier: when a converter warp comes to a stage, the use before
    // the last must be known to be over. It knows of the panels up to STAGES before its previous one, kConvPairs back.
    static_assert(STAGES >= kConvPairs, "phases of the empty barriers");
    static_assert(PANEL_B % 1024 == 0, "swizzle atoms");
};

struct Ctl {
    uint64_t full[kMaxStages];      // leader: the rows of A of both CTAs have landed, both CTAs' weights are converted
    uint64_t empty[kMaxStages];     // both: the leader's commit
    uint64_t tmem_full[kMaxBufs];   // both: the leader's commit
    uint64_t tmem_empty[kMaxBufs];  // leader: 2 x 8 epilogue warps
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
    alignas(16) uint32_t sig_src[4];
    alignas(16) uint32_t sig_dst[2 * kConvPairs][4];
};
static_assert(sizeof(Ctl) <= 1024, "barriers");

struct Params {
    const uint8_t* packed; Layout l;
    void* C; long ldc;
    const int* offsets;             // null: one matrix
    int R, E, N;
    int num_n;                      // 256-row tiles of the weights
    int np;                         // panels per tile (even)
    int ks, span;                   // K splits (pairs per cluster, at most 4), panels of each (even; the last may have fewer)
    int wide;                       // 16-bit C that 16-byte stores of 8 columns fit
    int plane;                      // rows between the slices of A (SL = 3)
    unsigned* err;
};

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
    const uint32_t a = smem_u32(bar);
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(a, parity))
        if (globaltimer() - t0 > 200000000ull) return;
}
__device__ __forceinline__ void abort_pair(Ctl* ctl, uint32_t peer) {
    ctl->abort = 1;
    st_shared_cluster_u32(mapa_shared(smem_u32(&ctl->abort), peer), 1u);
}
__device__ __forceinline__ float ld_shared_cluster(const float* p, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
    return v;
}
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// The bounded wait of device_utils.cuh with everything but the first try out of line: the loops of the roles stay short
// straight code (with the waits' loops inlined, fetching instructions held the MMA issuer to 280 cycles per k16 step).
__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort, unsigned* err, unsigned bit) {
    return mbar_wait(bar, parity, abort, err, bit);
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort, unsigned* err, unsigned bit) {
    return mbar_try_wait(smem_u32(bar), parity) || wait_slow(bar, parity, abort, err, bit);
}

// One lane of the (converged) warp, always the same one.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// wait::ld that the values read depend on, so that no use of them can be moved before it.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// 32 lanes' columns of H rows of C (y[j]: row j, this lane's column) as 16-byte stores: three rounds of exchanges between
// lanes 1, 2 and 4 apart turn pairs of rows into pairs of columns, so that lane l ends with columns 8 (l >> 3) .. + 7 of row
// 8 q + (l & 7) for each q. (2-byte stores, 64 contiguous bytes a warp, took about 80 cycles each: 28 % of 16384 rows over 16
// experts, 4096 x 2048.) c: row 0, the warp's first column.
template <typename T, int H>
__device__ __forceinline__ void store_wide(T* c, long ldc, int rows, int cols, const float (&y)[H], float unit) {
    const int lane = threadIdx.x & 31;
    const bool o1 = lane & 1, o2 = lane & 2, o3 = lane & 4;
    uint32_t w[H / 2];
#pragma unroll
    for (int i = 0; i < H / 2; ++i) {
        const float a = y[2 * i] * unit, b = y[2 * i + 1] * unit;
        if (std::is_same<T, __half>::value) {
            const __half2 h = __floats2half2_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        const uint32_t other = __shfl_xor_sync(0xffffffffu, w[i], 1);
        w[i] = __byte_perm(w[i], other, o1 ? 0x3276 : 0x5410);
    }
#pragma unroll
    for (int q = 0; q < H / 4; ++q) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, o2 ? w[2 * q] : w[2 * q + 1], 2);
        if (o2) w[2 * q] = other;
        else w[2 * q + 1] = other;
    }
    T* to = c + (size_t)(lane & 7) * ldc + 8 * (lane >> 3);
    const bool in = 8 * (lane >> 3) < cols;
#pragma unroll
    for (int q = 0; q < H / 8; ++q) {
        const uint32_t r0 = __shfl_xor_sync(0xffffffffu, o3 ? w[4 * q] : w[4 * q + 2], 4);
        const uint32_t r1 = __shfl_xor_sync(0xffffffffu, o3 ? w[4 * q + 1] : w[4 * q + 3], 4);
        const uint4 v = o3 ? make_uint4(r0, r1, w[4 * q + 2], w[4 * q + 3]) : make_uint4(w[4 * q], w[4 * q + 1], r0, r1);
        if (in && 8 * q + (lane & 7) < rows) *reinterpret_cast<uint4*>(to) = v;
        to += 8 * ldc;
    }
}

// The tile's expert, 256-row block of weights, and rows [m0, m1) of A. first[e] is the first row tile of expert e.
struct Tile { int e, nb, m0, m1; };
template <int TN>
__device__ __forceinline__ Tile tile_of(const Params& p, const int* first, int t) {
    Tile r;
    r.nb = t % p.num_n;
    const int mt = t / p.num_n;
    if (!p.offsets) {
        r.e = 0;
        r.m0 = mt * TN;
        r.m1 = min(p.R, r.m0 + TN);
        return r;
    }
    int lo = 0, hi = p.E;            // first[lo] <= mt < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= mt) lo = mid;
        else hi = mid;
    }
    r.e = lo;
    r.m0 = max(0, p.offsets[lo]) + (mt - first[lo]) * TN;
    r.m1 = min(min(p.R, p.offsets[lo + 1]), r.m0 + TN);
    return r;
}

// T: type of A and C. TN: rows of A per tile of the pair. GROUP: values of K per scale.
template <typename T, int TN, int GROUP>
__global__ void __launch_bounds__(kThreads, 1) k_q4_pair(const __grid_constant__ CUtensorMap tm_x, Params p) {
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    constexpr int SL = sizeof(T) == 4 ? 3 : 1;
    using C_ = Cfg<SL, TN>;
    constexpr int ST = C_::STAGES, NB = C_::BUFS;
    constexpr uint32_t kIdesc = idesc_f16(256, TN, BF16);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Ctl* ctl = reinterpret_cast<Ctl*>(smem + ST * C_::STAGE);
    int* first = reinterpret_cast<int*>(ctl + 1);
    float* red = reinterpret_cast<float*>(smem);   // ks > 1: [TN][128] sums of this pair's part of K, after the last product
    constexpr int H = TN / 2;
    volatile int* abort = &ctl->abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a cluster is one pair, or ks of them that share a tile and split its K
    const uint32_t crank = cluster_ctarank(), peer = crank ^ 1u, lead = crank & ~1u, rank = crank & 1u;
    const bool leader = rank == 0;
    const int pair = blockIdx.x / (2 * p.ks), num_pairs = gridDim.x / (2 * p.ks);
    const int p0 = (int)(crank >> 1) * p.span, np = min(p.np, p0 + p.span) - p0;   // panels of this pair
    const uint16_t both = (uint16_t)(3u << lead);

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(&ctl->full[s], 3);       // the producer and the leader's two converter warps of the panel
            mbar_init(&ctl->empty[s], 1);
        }
        for (int b = 0; b < NB; ++b) {
            mbar_init(&ctl->tmem_full[b], 1);
            mbar_init(&ctl->tmem_empty[b], 2 * kEpiWarps);
        }
        mbar_init(&ctl->drain, 1);
        ctl->abort = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) prefetch_tmap(&tm_x);
    if (warp == 1) {
        tmem_alloc_pair(&ctl->tmem_base, 512);
        tmem_relinquish_pair();
    }
    if (warp == 2 && p.offsets) {
        // offsets that run backwards or overlap make no more tiles than the host counted for (tile_count)
        const int cap = min(p.E, p.R) + (p.R + TN - 1) / TN;
        int run = 0;
        for (int x0 = 0; x0 < p.E; x0 += 32) {
            const int x = x0 + lane;
            const int r0 = x < p.E ? max(0, p.offsets[x]) : 0, r1 = x < p.E ? min(p.R, p.offsets[x + 1]) : 0;
            const int n = r1 > r0 ? (r1 - r0 + TN - 1) / TN : 0;
            int inc = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, inc, d);
                if (lane >= d) inc += v;
            }
            if (x < p.E) first[x] = min(run + inc - n, cap);
            run = min(run + __shfl_sync(0xffffffffu, inc, 31), cap);
        }
        if (lane == 0) first[p.E] = run;
    }
    __syncwarp();                                  // the barriers below are .aligned: whole warps
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = ctl->tmem_base;
    const int num_tiles = (p.offsets ? first[p.E] : (p.R + TN - 1) / TN) * p.num_n;   // ks > 1: at most one per cluster

    if (warp < 8) {
        reg_dec<kRegOther>();
        if (warp == 0 && lane == 0) {
            // ---------------- TMA producer: this CTA's half of the rows of A ----------------
            const uint32_t lead_full0 = mapa_shared(smem_u32(&ctl->full[0]), lead);
            long it = 0;
            bool ok = true;
            for (int t = pair; t < num_tiles && ok; t += num_pairs) {
                const Tile tl = tile_of<TN>(p, first, t);
                const int row = tl.m0 + (int)rank * (TN / 2);
                for (int k = 0; k < np; ++k, ++it) {
                    const int s = (int)(it % ST);
                    if (!wait(&ctl->empty[s], (uint32_t)((it / ST) & 1) ^ 1u, abort, p.err, kErrTimeoutProducer)) {
                        ok = false;
                        break;
                    }
                    // both CTAs' rows, and the 16-byte signals of the peer's two converter warps
                    if (leader) mbar_arrive_expect_tx(&ctl->full[s], 2 * C_::B_BYTES + 2 * 16);
                    const uint32_t fb = lead_full0 + (uint32_t)(s * sizeof(uint64_t));
                    uint8_t* st = smem + s * C_::STAGE + kPanelA;
#pragma unroll
                    for (int sl = 0; sl < SL; ++sl)
                        tma_load_2d_pair(st + sl * C_::PANEL_B, &tm_x, fb, (p0 + k) * 64, sl * p.plane + row);
                }
            }
            // The leader's last commits arrive here, also those of stages that nobody waits for again: no CTA leaves before
            // they have. Where a role gave up, the loads in flight are waited for instead.
            const long last = it > ST ? it - ST : 0;
            for (long j = last; j < it && ok; ++j)
                ok = wait(&ctl->empty[j % ST], (uint32_t)((j / ST) & 1), abort, p.err, kErrTimeoutProducer);
            if (!ok) {
                abort_pair(ctl, peer);
                if (leader)
                    for (long j = last; j < it; ++j) drain_wait(&ctl->full[j % ST], (uint32_t)((j / ST) & 1));
            }
        } else if (warp == 1 && leader) {
            // ---------------- leader: pair MMA issuer ----------------
            // The whole warp runs the loop and one elected lane issues: descriptors and addresses then are warp-uniform
            // (one lane alone in a divergent loop took twice as long per panel as its four MMAs).
            constexpr int GPP = GROUP < 64 ? 64 / GROUP : 1, PPG = GROUP > 64 ? GROUP / 64 : 1;
            const uint64_t a00 = sdesc_kmajor(smem_u32(smem), 128);
            int s = 0, u = 0;                      // stage and accumulator, with their phases
            uint32_t ph = 0, pu = 1;
            bool ok = true;
            for (int t = pair; t < num_tiles && ok; t += num_pairs) {
                for (int k = 0; k < np && ok; k += PPG) {
#pragma unroll
                    for (int h = 0; h < PPG && ok; ++h) {
                        bool ready = wait(&ctl->full[s], ph, abort, p.err, kErrTimeoutMma);
                        const uint64_t a0 = a00 + (uint64_t)(uint32_t)((s * C_::STAGE) >> 4);
#pragma unroll
                        for (int q = 0; q < GPP; ++q) {
                            if (h == 0) ready = ready && wait(&ctl->tmem_empty[u], pu, abort, p.err, kErrTimeoutMma);
                            if (!__all_sync(0xffffffffu, ready)) { ok = false; break; }
                            tc_fence_after();
                            const uint32_t d = tmem_base + (uint32_t)(u * TN);
                            if (elect_one()) {
#pragma unroll
                                for (int j = 0; j < 4 / GPP; ++j)
#pragma unroll
                                    for (int sl = SL - 1; sl >= 0; --sl) {
                                        const uint64_t a = a0 + (uint64_t)(((q * (4 / GPP) + j) * 32) >> 4);
                                        mma_f16_ss_pair(d, a, a + (uint64_t)((kPanelA + sl * C_::PANEL_B) >> 4), kIdesc,
                                                        h != 0 || j != 0 || sl != SL - 1 ? 1u : 0u);
                                    }
                                if (h == PPG - 1) mma_commit_pair_both(&ctl->tmem_full[u], both);
                                if (q == GPP - 1) mma_commit_pair_both(&ctl->empty[s], both);
                            }
                            if (h == PPG - 1 && ++u == NB) { u = 0; pu ^= 1u; }
                        }
                        if (++s == ST) { s = 0; ph ^= 1u; }
                    }
                }
            }
            if (!ok && elect_one()) {
                abort_pair(ctl, peer);
                mma_commit_pair(&ctl->drain);
                drain_wait(&ctl->drain, 0);
            }
        } else if (warp >= 2) {
            // ---------------- converters: codes -> integers in the swizzled K-major operand ----------------
            // A pair of warps takes every third panel of the pair's tiles, each warp 64 of the CTA's 128 weight rows.
            const int cp = (warp - 2) >> 1, cw = warp & 1, g = lane >> 2, t4 = lane & 3;
            const uint32_t lead_full0 = mapa_shared(smem_u32(&ctl->full[0]), lead);
            const uint32_t lead_slot = mapa_shared(smem_u32(&ctl->sig_dst[2 * cp + cw][0]), lead);
            const uint32_t sig_src = smem_u32(&ctl->sig_src[0]);
            const uint4 none = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
            const uint4* codes = reinterpret_cast<const uint4*>(p.packed);
            const bool odd = g & 1;
            int t = pair, k = cp;                  // tile and panel to load next
            const uint4* src = nullptr;
            int rows = 0;                          // row blocks of 16 that this warp has in the tile
            auto enter = [&]() {
                const Tile tl = tile_of<TN>(p, first, t);
                const long rb = (long)tl.nb * 16 + (long)rank * 8 + 4 * cw;
                rows = (int)min(4L, p.l.nb - rb);
                src = codes + (((size_t)tl.e * p.l.nb + rb) * p.l.kb) * 32 + lane;
            };
            auto load = [&](uint4 (&c)[4]) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    c[r] = r < rows && p0 + k < p.l.kb ? __ldg(src + ((size_t)r * p.l.kb + p0 + k) * 32) : none;
            };
            auto settle = [&]() {                  // the panel's tile, when k has run past the end of one
                bool moved = false;
                while (k >= np && t < num_tiles) {
                    k -= np;
                    t += num_pairs;
                    moved = true;
                }
                if (moved && t < num_tiles) enter();
            };
            uint4 next[4] = {none, none, none, none};
            if (t < num_tiles) {
                enter();
                settle();
                if (t < num_tiles) load(next);
            }
            for (long it = cp; t < num_tiles; it += kConvPairs) {
                const int s = (int)(it % ST);
                uint4 c[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) c[r] = next[r];
                k += kConvPairs;
                settle();
                const bool more = t < num_tiles;
                if (more) load(next);
                const bool ready = wait(&ctl->empty[s], (uint32_t)((it / ST) & 1) ^ 1u, abort, p.err, kErrTimeoutConvert);
                if (!__all_sync(0xffffffffu, ready)) {
                    if (lane == 0) abort_pair(ctl, peer);
                    break;
                }
                uint8_t* st = smem + s * C_::STAGE + cw * 64 * 128;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // rows g and g + 8, chunks t4 and 4 + t4; odd rows store the upper chunk first, so that the eight
                    // lanes of a store phase (two rows) touch all eight 16-byte columns
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t lo = half ? c[r].y : c[r].x, hi = half ? c[r].w : c[r].z;
                        const uint32_t w0 = odd ? hi : lo, w1 = odd ? lo : hi;
                        const int c0 = odd ? 4 + t4 : t4, c1 = c0 ^ 4;
                        uint8_t* o = st + (r * 16 + g + 8 * half) * 128;
                        uint32_t v[4];
                        code_pairs<BF16>(w0, v);
                        *reinterpret_cast<uint4*>(o + ((c0 ^ g) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
                        code_pairs<BF16>(w1, v);
                        *reinterpret_cast<uint4*>(o + ((c1 ^ g) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (leader) mbar_arrive(&ctl->full[s]);
                    else bulk_signal_cluster(lead_slot, sig_src, 16, lead_full0 + (uint32_t)(s * sizeof(uint64_t)));
                }
            }
        }
    } else {
        reg_inc<kRegEpi>();
        // ---------------- scale, sum, store: one weight row and half of the tile's rows of A per thread ----------------
        const int sp = warp & 3, half = (warp - 8) >> 2;
        const int row_in_tile = (int)rank * 128 + sp * 32 + lane;
        const uint32_t lane_off = (uint32_t)(sp * 32) << 16;
        const uint32_t lead_te0 = mapa_shared(smem_u32(&ctl->tmem_empty[0]), lead);
        const uint16_t* scales = reinterpret_cast<const uint16_t*>(p.packed + p.l.scales_at);
        const int g0 = p0 * 64 / GROUP, groups = np * 64 / GROUP;   // of the padded K
        long ch = 0;
        bool ok = true;
        for (int t = pair; t < num_tiles && ok; t += num_pairs) {
            const Tile tl = tile_of<TN>(p, first, t);
            const int n = tl.nb * 256 + row_in_tile;
            const bool there = n < p.N;
            const uint16_t* sc = scales + (((size_t)tl.e * p.l.nb + (n >> 4)) * p.l.groups + g0) * 16 + (n & 7) * 2 + ((n >> 3) & 1);
            float sum[H];
#pragma unroll
            for (int j = 0; j < H; ++j) sum[j] = 0.f;
            float s_next = there ? __uint_as_float((uint32_t)__ldg(sc) << 16) : 0.f;
            for (int gi = 0; gi < groups; ++gi, ++ch) {
                const int u = (int)(ch % NB);
                const float s = s_next;
                s_next = there && g0 + gi + 1 < p.l.groups ? __uint_as_float((uint32_t)__ldg(sc + (gi + 1) * 16) << 16) : 0.f;
                const bool ready = mbar_wait(&ctl->tmem_full[u], (uint32_t)((ch / NB) & 1), abort, p.err,
                                             kErrTimeoutEpilogue);   // inline: a call would save the sums around it
                if (!__all_sync(0xffffffffu, ready)) { ok = false; break; }
                tc_fence_after();
                const uint32_t tb = tmem_base + lane_off + (uint32_t)(u * TN + half * H);
                uint32_t r[2][16];                 // a read runs while the previous one is added
                tmem_ld_32x32b_x16(tb, r[0]);
#pragma unroll
                for (int q = 0; q < H / 16; ++q) {
                    tmem_ld_wait_for(r[q & 1]);
                    if (q + 1 < H / 16) tmem_ld_32x32b_x16(tb + (uint32_t)((q + 1) * 16), r[(q + 1) & 1]);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        sum[q * 16 + j] = fmaf(s, __uint_as_float(r[q & 1][j]), sum[q * 16 + j]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(lead_te0 + (uint32_t)(u * sizeof(uint64_t)));
            }
            if (!ok) break;
            if (p.ks > 1) {                        // the stages are free: this pair's last product is done
#pragma unroll
                for (int j = 0; j < H; ++j) red[(half * H + j) * 128 + sp * 32 + lane] = sum[j];
            } else if (SL == 1 && p.wide) {
                const int n0 = n - lane;
                store_wide<T, H>(static_cast<T*>(p.C) + (size_t)(tl.m0 + half * H) * p.ldc + n0, p.ldc,
                                 tl.m1 - tl.m0 - half * H, p.N - n0, sum, code_unit<BF16>());
            } else if (there) {
                T* c = static_cast<T*>(p.C) + (size_t)(tl.m0 + half * H) * p.ldc + n;
                const int rows = tl.m1 - tl.m0 - half * H;
#pragma unroll
                for (int j = 0; j < H; ++j)
                    if (j < rows) c[(size_t)j * p.ldc] = from_float<T>(sum[j] * code_unit<BF16>());
            }
        }
        if (!ok && lane == 0) abort_pair(ctl, peer);
    }

    __syncwarp();
    tc_fence_before();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
    if (p.ks > 1) {
        // every split adds the parts of its share of the tile's rows of A, in the order of the splits
        if (warp >= 8 && pair < num_tiles) {
            const Tile tl = tile_of<TN>(p, first, pair);
            const int row = (warp & 3) * 32 + lane, n = tl.nb * 256 + (int)rank * 128 + row;
            const int share = (H + p.ks - 1) / p.ks, j0 = (int)(crank >> 1) * 2 * share + ((warp - 8) >> 2) * share;
            const int j1 = n < p.N ? min(j0 + share, tl.m1 - tl.m0) : j0;
            T* c = static_cast<T*>(p.C) + (size_t)tl.m0 * p.ldc + n;
            for (int j = j0; j < j1; j += 4) {       // the parts of four rows of A on their way together
                float v[4][4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        v[q][i] = q < p.ks && j + i < j1 ? ld_shared_cluster(red + (j + i) * 128 + row, 2u * q + rank) : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (j + i < j1)
                        c[(size_t)(j + i) * p.ldc] = from_float<T>((v[0][i] + v[1][i] + v[2][i] + v[3][i]) * code_unit<BF16>());
            }
        }
        __syncwarp();                              // lanes behind column N - 1 left the loop early
        cluster_sync_all();                        // no CTA leaves while its parts are read
    }
}

// Rows of A as TMA can read them: 16-bit rows of Kp values (zeros behind K), FP32 rows as three planes of bf16 slices. With
// offsets only up to the last row that an expert claims (the largest offset: the last one, unless they run backwards).
template <typename T>
__global__ void __launch_bounds__(256) k_q4_stage(const T* __restrict__ A, long lda, int R, long K, long Kp,
                                                  uint16_t* __restrict__ X, int vec, const int* __restrict__ offsets, int E) {
    __shared__ int claimed[8];
    int rows = R;
    if (offsets) {
        rows = 0;
        for (int e = threadIdx.x; e < E; e += 256) rows = max(rows, min(R, __ldg(offsets + e + 1)));
        __syncwarp();
        rows = __reduce_max_sync(0xffffffffu, rows);
        if ((threadIdx.x & 31) == 0) claimed[threadIdx.x >> 5] = rows;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) rows = max(rows, claimed[w]);
    }
    const long chunks = Kp / 8, n = rows * chunks;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long m = i / chunks, k = (i - m * chunks) * 8;
        const T* a = A + (size_t)m * lda + k;
        __align__(16) T x[8];
        static_assert(__alignof__(x) >= 16, "written and read 16 bytes at a time");
        if (sizeof(T) == 4 && vec && k + 8 <= K) {
            reinterpret_cast<float4*>(x)[0] = reinterpret_cast<const float4*>(a)[0];
            reinterpret_cast<float4*>(x)[1] = reinterpret_cast<const float4*>(a)[1];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = k + j < K ? a[j] : from_float<T>(0.f);
        }
        if (sizeof(T) == 4) {
            __align__(16) uint16_t s[3][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) slice3(to_float<T>(x[j]), s[0][j], s[1][j], s[2][j]);
#pragma unroll
            for (int q = 0; q < 3; ++q)
                *reinterpret_cast<uint4*>(X + ((size_t)q * R + m) * Kp + k) = *reinterpret_cast<const uint4*>(s[q]);
        } else {
            *reinterpret_cast<uint4*>(X + (size_t)m * Kp + k) = *reinterpret_cast<const uint4*>(x);
        }
    }
}

long tile_count(const Q4GemmArgs& a, int TN) {
    return ((a.offsets ? std::min(a.E, a.R) : 0) + ((long)a.R + TN - 1) / TN) * ((a.N + 255) / 256);
}
// Few tiles: the pairs of a cluster share a tile and split its K, as many as leave each 512 values of it and let all
// clusters run at once (33, 22 and 15 of 2, 3 and 4 pairs on a B200). 128 rows, K = 4096: 15 tiles 18.3 us with two, 13.0
// with four; 16 tiles 24.6 with one, 18.3 with two, 15.0 with three, 24.2 with four, which do not all fit; 34 tiles 24.8 with
// one, 35.8 with two.
int k_splits(long tiles, int np, const ClusterFits& f) {
    for (int ks = 4; ks > 1; --ks)
        if (tiles <= f.of[1][2 * ks] && np >= 8 * ks) return ks;
    return 1;
}

template <typename T, int TN, int GROUP>
int launch_pair_g(const Q4GemmArgs& a, const void* X, long ldx, int rows, long kx, int plane, int ks, cudaStream_t st) {
    constexpr int SL = sizeof(T) == 4 ? 3 : 1;
    using C_ = Cfg<SL, TN>;
    PFN_cuTensorMapEncodeTiled_v12000 enc = nullptr;
    if (!tc_get_encode(&enc)) return (int)cudaErrorNotSupported;
    CUtensorMap tm;
    cuuint64_t dims[2] = {(cuuint64_t)kx, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ldx * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)(TN / 2)};
    cuuint32_t estr[2] = {1, 1};
    if (enc(&tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(X), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return (int)cudaErrorInvalidValue;
    Params p{};
    p.packed = static_cast<const uint8_t*>(a.packed);
    p.l = layout(a.E, a.N, a.K, a.group);
    p.C = a.C; p.ldc = a.ldc;
    p.offsets = a.offsets;
    p.R = a.R; p.E = a.E; p.N = a.N;
    p.num_n = (a.N + 255) / 256;
    p.np = (int)((a.K + 127) / 128 * 2);
    p.plane = plane;
    p.wide = SL == 1 && (reinterpret_cast<uintptr_t>(a.C) & 15) == 0 && a.ldc % 8 == 0 && a.N % 8 == 0;
    p.err = a.err;
    auto kern = k_q4_pair<T, TN, GROUP>;
    static OncePerDevice once;
    const int e0 = once([&] { return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C_::SMEM); });
    if (e0) return e0;
    // with offsets the number of tiles is known on the device only: at most one partly filled tile per expert
    const long tiles = tile_count(a, TN);
    p.ks = ks;
    p.span = (p.np / 2 + p.ks - 1) / p.ks * 2;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2 * p.ks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(2 * p.ks * (p.ks > 1 ? tiles : std::min((long)a.num_sms / 2, tiles))), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = C_::SMEM;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tm, p);
    count_launch();
    if (e != cudaSuccess) return (int)e;
    return (int)cudaGetLastError();
}

template <typename T, int TN>
int launch_pair(const Q4GemmArgs& a, const void* X, long ldx, int rows, long kx, int plane, int ks, cudaStream_t st) {
    if (a.group == 32) return launch_pair_g<T, TN, 32>(a, X, ldx, rows, kx, plane, ks, st);
    if (a.group == 64) return launch_pair_g<T, TN, 64>(a, X, ldx, rows, kx, plane, ks, st);
    return launch_pair_g<T, TN, 128>(a, X, ldx, rows, kx, plane, ks, st);
}

template <typename T>
int launch_t(const Q4GemmArgs& a, cudaStream_t st) {
    constexpr int SL = sizeof(T) == 4 ? 3 : 1;
    const void* X = a.A;
    long ldx = a.lda, kx = a.K;
    int rows = a.R, plane = 0;
    if (a.stage) {
        kx = ldx = (a.K + 63) / 64 * 64;
        rows = plane = a.R;
        rows *= SL;
        const long n = (long)a.R * (kx / 8);
        const int grid = (int)std::min((n + 255) / 256, 16L * a.num_sms);
        const int vec = (reinterpret_cast<uintptr_t>(a.A) & 15) == 0 && (a.lda * sizeof(T)) % 16 == 0;
        k_q4_stage<T><<<grid, 256, 0, st>>>(static_cast<const T*>(a.A), a.lda, a.R, a.K, kx,
                                            static_cast<uint16_t*>(a.stage), vec, a.offsets, a.E);
        count_launch();
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return (int)e;
        X = a.stage;
    }
    // 256 or 128 rows of A per tile, whichever is done sooner: rounds of the pairs times a panel's time, 1.3 times as long
    // for 256 (0.49 against 0.375 us at 8192 x 8192).
    const int pairs = a.num_sms / 2, np = (int)((a.K + 127) / 128 * 2);
    const long t128 = tile_count(a, 128), t256 = tile_count(a, 256);
    const ClusterFits* fits = cluster_fits();
    if (!fits) return (int)cudaErrorUnknown;
    const int ks = k_splits(t128, np, *fits);
    const double c128 = (double)((t128 * ks + pairs - 1) / pairs) / ks, c256 = 1.3 * (double)((t256 + pairs - 1) / pairs);
    if (c256 <= c128) return launch_pair<T, 256>(a, X, ldx, rows, kx, plane, 1, st);
    return launch_pair<T, 128>(a, X, ldx, rows, kx, plane, ks, st);
}

}  // namespace

size_t q4_stage_bytes(const void* A, long lda, int dtype, int R, long K) {
    if (dtype == EMU_DTYPE_F32) return (size_t)R * ((K + 63) / 64 * 64) * 6;
    if (lda % 8 == 0 && (reinterpret_cast<uintptr_t>(A) & 15) == 0) return 0;
    return (size_t)R * ((K + 63) / 64 * 64) * 2;
}

int launch_q4_tiles(const Q4GemmArgs& a, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    if (a.dtype == EMU_DTYPE_F32) return launch_t<float>(a, st);
    if (a.dtype == EMU_DTYPE_F16) return launch_t<__half>(a, st);
    return launch_t<__nv_bfloat16>(a, st);
}

}  // namespace emu
