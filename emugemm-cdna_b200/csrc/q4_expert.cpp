// q4_expert.cpp - C entry points of the 4-bit weight products and of the expert routing around them: argument checks
// and dispatch. The kernels are in k_q4.cu and k_expert.cu.
#include "emugemm_internal.h"

#include <cuda_runtime.h>

#include <cstdint>

namespace emu {
namespace {

int dtype_size(int dtype) {
    return dtype == EMU_DTYPE_F32 ? 4 : dtype == EMU_DTYPE_F16 || dtype == EMU_DTYPE_BF16 ? 2 : 0;
}
bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }
// a pointer the kernels may access with its element's (or the packed layout's) alignment
bool bad_ptr(const void* p, int align) { return !p || (reinterpret_cast<uintptr_t>(p) & (align - 1)); }

// Sizes of packed weights: E experts of N x K, of which no count of bytes or tiles passes 63 bits
bool q4_size_ok(int E, int N, long K) {
    return E >= 1 && E <= kMaxExperts && N >= 1 && N <= (1 << 30) && K >= 1 && K <= (1L << 30) &&
           (long)E * N <= (1L << 50) / K;
}
// Sizes of the routing calls: at most 2^30 slots
bool slots_ok(long T, int topk) { return T >= 0 && topk >= 1 && (T == 0 || topk <= (1L << 30) / T); }

emugemm_status_t q4_product(emugemm_handle_t handle, int R, int E, int N, long K, const void* A, long lda, int dtype,
                            const int* offsets, bool experts, const void* packed, int group, void* C, long ldc) {
    Handle* h = reinterpret_cast<Handle*>(handle);
    if (!h) return EMUGEMM_STATUS_INVALID_HANDLE;
    const int size = dtype_size(dtype);
    if (!size || !group_ok(group)) return EMUGEMM_STATUS_INVALID_VALUE;
    if (R < 0 || R > (1 << 30) || !q4_size_ok(E, N, K) || lda < K || ldc < N) return EMUGEMM_STATUS_INVALID_SIZE;
    if (R == 0) return EMUGEMM_STATUS_SUCCESS;
    if (bad_ptr(A, size) || bad_ptr(C, size) || bad_ptr(packed, 16) || (experts && bad_ptr(offsets, 4)))
        return EMUGEMM_STATUS_INVALID_POINTER;
    DeviceGuard g(h->device);
    if (!g.ok) return EMUGEMM_STATUS_INTERNAL_ERROR;
    Q4GemmArgs a{};
    a.R = R; a.E = E; a.N = N; a.K = K; a.group = group; a.dtype = dtype;
    a.A = A; a.lda = lda; a.C = C; a.ldc = ldc;
    a.packed = packed;
    a.offsets = experts ? offsets : nullptr;
    a.num_sms = h->num_sms;
    a.err = h->err_dev;
    const int with = experts ? (E < R ? E : R) : 1;   // experts that can have rows
    const long cols = (long)(R / with) * (dtype == EMU_DTYPE_F32 ? 3 : 1);
    // Few columns: one pass over the codes per 48 of them (k_q4.cu; of experts by the mean, since the rows of each are known on
    // the device only, and the passes of one expert follow one another), else tiles of CTA pairs (k_q4_tc.cu), in us:
    //   48 columns, groups of 128:  4096 x 4096 13.7 against 15.0, 8192 x 4096 20.3 / 19.0, 8192 x 8192 35.4 / 29.4
    //   32 columns, groups of 128:  8192 x 8192 26.1 / 28.8;  48 columns, groups of 64:  11008 x 4096 29.8 / 37.8
    //   16 rows FP32 (48 columns):  4096 x 4096 13.1 / 19.4;  64 columns, groups of 128:  4096 x 4096 23 / 15
    //   groups of 32, an accumulator each on the tiles:  64 columns, 4096 x 4096 25.7 / 27.6, 8192 x 8192 74.5 / 82.6,
    //   11008 x 4096 56.5 / 69.7;  96 columns 29.2 / 27.8, 83.3 / 83.2, 64.6 / 70.9;  2048 x 2048: 17.3 / 14.4, 20.0 / 14.4
    const long weights = (long)with * N * K;
    const bool large = group == 128 && dtype != EMU_DTYPE_F32 && !experts && weights >= (1L << 25);
    // More than 8 experts: rows are seldom dealt evenly among them, and the passes of 48 columns of the fullest expert follow
    // one another, so the 96 of groups of 32 do not hold for them (mean rows; even, mildly and strongly uneven):
    //   16 x 2048 x 4096: 52 rows 136, 186, 376 against 139, 139, 142, 96 rows 159, 284, 667 against 184, 184, 183;  16 x 1024 x
    //   1024: 64 rows 31, 45, 103 against 23;  32 x 4096 x 2048: 52 rows 251, 223, 268 against 276, 276, 310, 96 rows 302, 379,
    //   497 against 337, 336, 382;  FP32 16 x 2048 x 4096: 24 rows 149, 204, 495 against 200.  4 x 2048 x 2048: 64 rows 29, 29,
    //   30 against 36, 96 rows 33, 41, 42 against 37;  8 x 1024 x 4096: 90 rows 48, 64, 71 against 64
    const long most = group == 32 && weights >= (1L << 24) && with <= 8 ? 96 : large ? 32 : 48;
    if (cols <= most) {
        ProfScope ps(h, kProfQ4);
        return from_cuda(launch_q4_rows(a, h->stream));
    }
    if (const size_t bytes = q4_stage_bytes(A, lda, dtype, R, K)) {
        a.stage = ws_get_kept(h, kWsQ4X, bytes);
        if (!a.stage) return EMUGEMM_STATUS_MEMORY_ERROR;
    }
    ProfScope ps(h, kProfQ4);
    return from_cuda(launch_q4_tiles(a, h->stream));
}

emugemm_status_t rows_checked(Handle* h, int T, int topk, int H, int dtype, long ld1, long ld2, long ld3) {
    if (!h) return EMUGEMM_STATUS_INVALID_HANDLE;
    if (!dtype_size(dtype)) return EMUGEMM_STATUS_INVALID_VALUE;
    if (!slots_ok(T, topk) || H < 0 || H > (1 << 30) || ld1 < H || ld2 < H || ld3 < H) return EMUGEMM_STATUS_INVALID_SIZE;
    return EMUGEMM_STATUS_SUCCESS;
}

emugemm_status_t combine(emugemm_handle_t handle, int T, int topk, int H, const void* S, long lds, int dtype,
                         const int* place, const float* w, bool weighted, void* Y, long ldy) {
    Handle* h = reinterpret_cast<Handle*>(handle);
    emugemm_status_t s = rows_checked(h, T, topk, H, dtype, lds, ldy, ldy);
    if (s != EMUGEMM_STATUS_SUCCESS || T == 0 || H == 0) return s;
    const int size = dtype_size(dtype);
    if (bad_ptr(S, size) || bad_ptr(Y, size) || bad_ptr(place, 4) || (weighted && bad_ptr(w, 4)))
        return EMUGEMM_STATUS_INVALID_POINTER;
    DeviceGuard g(h->device);
    if (!g.ok) return EMUGEMM_STATUS_INTERNAL_ERROR;
    ExpertRows a{};
    a.T = T; a.topk = topk; a.H = H; a.num_sms = h->num_sms;
    a.S = S; a.lds = lds; a.Y = Y; a.ldy = ldy;
    a.place = place; a.w = weighted ? w : nullptr;
    ProfScope ps(h, kProfExpert);
    return from_cuda(launch_expert_combine(a, dtype, h->stream));
}

}  // namespace
}  // namespace emu

using emu::Handle;

extern "C" {

size_t emugemm_q4_bytes(int E, int N, long K, int group) {
    return emu::group_ok(group) && emu::q4_size_ok(E, N, K) ? emu::q4_bytes(E, N, K, group) : 0;
}

emugemm_status_t emugemm_q4_pack(emugemm_handle_t handle, int E, int N, long K, const void* W, long ldw, int dtype,
                                 int group, void* packed) {
    Handle* h = reinterpret_cast<Handle*>(handle);
    if (!h) return EMUGEMM_STATUS_INVALID_HANDLE;
    const int size = emu::dtype_size(dtype);
    if (!size || !emu::group_ok(group)) return EMUGEMM_STATUS_INVALID_VALUE;
    if (!emu::q4_size_ok(E, N, K) || ldw < K) return EMUGEMM_STATUS_INVALID_SIZE;
    if (emu::bad_ptr(W, size) || emu::bad_ptr(packed, 16)) return EMUGEMM_STATUS_INVALID_POINTER;
    emu::DeviceGuard g(h->device);
    if (!g.ok) return EMUGEMM_STATUS_INTERNAL_ERROR;
    emu::ProfScope ps(h, emu::kProfQ4);
    return emu::from_cuda(emu::launch_q4_pack(W, ldw, dtype, E, N, K, group, packed, h->num_sms, h->stream));
}

emugemm_status_t emugemm_q4_unpack(emugemm_handle_t handle, int E, int N, long K, int group, const void* packed, float* W,
                                   long ldw) {
    Handle* h = reinterpret_cast<Handle*>(handle);
    if (!h) return EMUGEMM_STATUS_INVALID_HANDLE;
    if (!emu::group_ok(group)) return EMUGEMM_STATUS_INVALID_VALUE;
    if (!emu::q4_size_ok(E, N, K) || ldw < K) return EMUGEMM_STATUS_INVALID_SIZE;
    if (emu::bad_ptr(W, 4) || emu::bad_ptr(packed, 16)) return EMUGEMM_STATUS_INVALID_POINTER;
    emu::DeviceGuard g(h->device);
    if (!g.ok) return EMUGEMM_STATUS_INTERNAL_ERROR;
    emu::ProfScope ps(h, emu::kProfQ4);
    return emu::from_cuda(emu::launch_q4_unpack(packed, E, N, K, group, W, ldw, h->num_sms, h->stream));
}

emugemm_status_t emugemm_q4_gemm(emugemm_handle_t handle, int M, int N, long K, const void* A, long lda, int dtype,
                                 const void* packed, int group, void* C, long ldc) {
    return emu::q4_product(handle, M, 1, N, K, A, lda, dtype, nullptr, false, packed, group, C, ldc);
}

emugemm_status_t emugemm_q4_gemm_experts(emugemm_handle_t handle, int R, int E, int N, long K, const void* A, long lda,
                                         int dtype, const int* offsets, const void* packed, int group, void* C,
                                         long ldc) {
    return emu::q4_product(handle, R, E, N, K, A, lda, dtype, offsets, true, packed, group, C, ldc);
}

emugemm_status_t emugemm_expert_sort(emugemm_handle_t handle, int T, int topk, int E, const int* expert, int* order,
                                     int* place, int* offsets) {
    Handle* h = reinterpret_cast<Handle*>(handle);
    if (!h) return EMUGEMM_STATUS_INVALID_HANDLE;
    if (!emu::slots_ok(T, topk) || E < 1 || E > emu::kMaxExperts) return EMUGEMM_STATUS_INVALID_SIZE;
    if (emu::bad_ptr(offsets, 4) || (T > 0 && (emu::bad_ptr(expert, 4) || emu::bad_ptr(order, 4) || emu::bad_ptr(place, 4))))
        return EMUGEMM_STATUS_INVALID_POINTER;
    emu::DeviceGuard g(h->device);
    if (!g.ok) return EMUGEMM_STATUS_INTERNAL_ERROR;
    emu::ProfScope ps(h, emu::kProfExpert);
    return emu::from_cuda(emu::launch_expert_sort(expert, T * topk, E, order, place, offsets, h->stream));
}

emugemm_status_t emugemm_expert_gather(emugemm_handle_t handle, int T, int topk, int H, const void* X, long ldx, int dtype,
                                       const int* place, void* XS, long ldxs) {
    Handle* h = reinterpret_cast<Handle*>(handle);
    emugemm_status_t s = emu::rows_checked(h, T, topk, H, dtype, ldx, ldxs, ldxs);
    if (s != EMUGEMM_STATUS_SUCCESS || T == 0 || H == 0) return s;
    const int size = emu::dtype_size(dtype);
    if (emu::bad_ptr(X, size) || emu::bad_ptr(XS, size) || emu::bad_ptr(place, 4)) return EMUGEMM_STATUS_INVALID_POINTER;
    emu::DeviceGuard g(h->device);
    if (!g.ok) return EMUGEMM_STATUS_INTERNAL_ERROR;
    emu::ExpertRows a{};
    a.T = T; a.topk = topk; a.H = H; a.num_sms = h->num_sms;
    a.X = X; a.ldx = ldx; a.DS = XS; a.ldds = ldxs; a.place = place;
    emu::ProfScope ps(h, emu::kProfExpert);
    return emu::from_cuda(emu::launch_expert_gather(a, dtype, h->stream));
}

emugemm_status_t emugemm_expert_gather_backward(emugemm_handle_t handle, int T, int topk, int H, const void* dXS,
                                                long lddxs, int dtype, const int* place, void* dX, long lddx) {
    return emu::combine(handle, T, topk, H, dXS, lddxs, dtype, place, nullptr, false, dX, lddx);
}

emugemm_status_t emugemm_expert_combine(emugemm_handle_t handle, int T, int topk, int H, const void* YS, long ldys,
                                        int dtype, const int* place, const float* weights, void* Y, long ldy) {
    return emu::combine(handle, T, topk, H, YS, ldys, dtype, place, weights, true, Y, ldy);
}

emugemm_status_t emugemm_expert_combine_backward(emugemm_handle_t handle, int T, int topk, int H, const void* dY,
                                                 long lddy, const void* YS, long ldys, int dtype, const int* place,
                                                 const float* weights, void* dYS, long lddys, float* dweights) {
    Handle* h = reinterpret_cast<Handle*>(handle);
    emugemm_status_t s = emu::rows_checked(h, T, topk, H, dtype, lddy, ldys, lddys);
    if (s != EMUGEMM_STATUS_SUCCESS || T == 0) return s;
    const int size = emu::dtype_size(dtype);
    if (emu::bad_ptr(place, 4) || emu::bad_ptr(weights, 4) || emu::bad_ptr(dweights, 4) ||
        (H > 0 && (emu::bad_ptr(dY, size) || emu::bad_ptr(YS, size) || emu::bad_ptr(dYS, size))))
        return EMUGEMM_STATUS_INVALID_POINTER;
    emu::DeviceGuard g(h->device);
    if (!g.ok) return EMUGEMM_STATUS_INTERNAL_ERROR;
    emu::ExpertRows a{};
    a.T = T; a.topk = topk; a.H = H; a.num_sms = h->num_sms;
    a.X = dY; a.ldx = lddy; a.S = YS; a.lds = ldys; a.DS = dYS; a.ldds = lddys;
    a.place = place; a.w = weights; a.dw = dweights;
    emu::ProfScope ps(h, emu::kProfExpert);
    return emu::from_cuda(emu::launch_expert_combine_bwd(a, dtype, h->stream));
}

}  // extern "C"
