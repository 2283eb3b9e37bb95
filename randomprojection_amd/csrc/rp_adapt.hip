// rp_adapt.hip — low-rank adapters of many requests beside the dense projection, and their gradients.
//
// The dense projection Y = X C^T (rp_dense.hip) has one frozen matrix C for every row. Here row i also
// has an adapter a = ids[i] of rank R (none where ids[i] is outside 0..G-1), G of them in two banks
// `down` (G x R x m) and `up` (G x R x p), both with the long axis contiguous:
//
//   hidden_i = down[a] x_i,                 y_i = C x_i + scale[a] up[a]^T hidden_i
//   t_i = scale[a] up[a] dy_i,              dx_i = C^T dy_i + down[a]^T t_i
//   d_down[a] = sum_i t_i x_i^T,            d_up[a] = scale[a] sum_i hidden_i dy_i^T
//
// so both directions are made of three products over rows that share an adapter, whatever the bank:
//   shrink  H = Z W^T      (n x q, R x q -> n x R)
//   expand  O += H W       (n x R, R x q -> n x q)
//   outer   dW = H^T Z     (per adapter, over its rows)
#include "rp_common.h"

using namespace rpd;

namespace {

constexpr int kMaxRank = 128;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
// round to nearest even; a NaN stays one
__device__ __forceinline__ uint16_t to_bf16(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ void store_as(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_as(uint16_t* p, float x) { *p = to_bf16(x); }

// H[i][r] = (mul ? mul[a] : 1) sum_q Z[i][q] W[a][r][q]; zeros where row i has no adapter. One wave a row.
template <typename T>
__global__ void __launch_bounds__(256)
shrink_kernel(const T* __restrict__ Z, int64_t ldz, int64_t n, int64_t q, const T* __restrict__ W, int64_t ldw, int64_t G,
              int R, const float* __restrict__ mul, const int32_t* __restrict__ ids, float* __restrict__ H) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= n) return;
    const int64_t a = ids[row];
    const bool has = a >= 0 && a < G;
    for (int r = 0; r < R; ++r) {
        float s = 0.f;
        if (has)
            for (int64_t c = lane; c < q; c += 64) s = fmaf(to_f32(Z[row * ldz + c]), to_f32(W[(a * R + r) * ldw + c]), s);
        for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) H[row * R + r] = has ? (mul ? s * mul[a] : s) : 0.f;
    }
}

// O[i][c] = P[i][c] + (mul ? mul[a] : 1) sum_r H[i][r] W[a][r][c]
template <typename T, typename O>
__global__ void __launch_bounds__(256)
expand_kernel(const float* P, int64_t ldp, O* out, int64_t ldo, int64_t n, int64_t q, const T* __restrict__ W, int64_t ldw,
              int64_t G, int R, const float* __restrict__ mul, const int32_t* __restrict__ ids, const float* __restrict__ H) {
    const int64_t row = blockIdx.x;
    const int64_t a = ids[row];
    const bool has = a >= 0 && a < G;
    for (int64_t c = threadIdx.x; c < q; c += 256) {
        float s = 0.f;
        if (has)
            for (int r = 0; r < R; ++r) s = fmaf(H[row * R + r], to_f32(W[(a * R + r) * ldw + c]), s);
        store_as(out + row * ldo + c, P[row * ldp + c] + (has ? (mul ? s * mul[a] : s) : 0.f));
    }
}

// D[g][r][c] = (mul ? mul[g] : 1) sum over rows of adapter g of H[i][r] Z[i][c]
template <typename T>
__global__ void __launch_bounds__(256)
outer_kernel(const T* __restrict__ Z, int64_t ldz, int64_t n, int64_t q, int64_t G, int R, const float* __restrict__ mul,
             const int32_t* __restrict__ ids, const float* __restrict__ H, float* __restrict__ D, int64_t ldd, int64_t sdd) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= q) return;
    for (int64_t k = blockIdx.y; k < G * R; k += gridDim.y) {
        const int64_t g = k / R, r = k % R;
        float s = 0.f;
        for (int64_t i = 0; i < n; ++i)
            if (ids[i] == g) s = fmaf(H[i * R + r], to_f32(Z[i * ldz + c]), s);
        D[g * sdd + r * ldd + c] = mul ? s * mul[g] : s;
    }
}

int64_t padded(int64_t w, int32_t dtype) {
    const int64_t step = dtype == RP_BF16 ? 64 : 32;
    return (w + step - 1) / step * step;
}

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// the arguments both directions share
int check_shared(int32_t dtype, int64_t n, int64_t m, int64_t p, int64_t G, int32_t R) {
    if (dtype != RP_F32 && dtype != RP_BF16) return fail(RP_ERR_INVALID, "dtype must be RP_F32 or RP_BF16");
    if (n < 0 || m <= 0 || p <= 0 || G <= 0 || R <= 0) return fail(RP_ERR_INVALID, "bad shape");
    if (R > kMaxRank) return fail(RP_ERR_UNSUPPORTED, "rank %d is over %d", (int)R, kMaxRank);
    if (n > INT32_MAX || m > INT32_MAX - 64 || p > INT32_MAX - 64 || G > 65535)
        return fail(RP_ERR_UNSUPPORTED, "n, m, p or the number of adapters too large");
    return RP_OK;
}

int check_operand(const char* name, const void* p, int64_t ld, int64_t width, int32_t dtype) {
    if (!p) return fail(RP_ERR_INVALID, "NULL %s", name);
    if (ld < width) return fail(RP_ERR_INVALID, "%s: row stride %lld is under its padded width %lld", name, (long long)ld,
                                (long long)width);
    if (((uintptr_t)p & 15) || (ld * (dtype == RP_BF16 ? 2 : 4)) % 16)
        return fail(RP_ERR_INVALID, "%s must have 16-byte aligned rows", name);
    return RP_OK;
}

template <typename T>
int project(int device, const T* X, int64_t ldx, int64_t n, int64_t m, const T* C, int64_t p, const T* down, const T* up,
            int64_t G, int R, const float* scale, const int32_t* ids, float* Y, int64_t ldy, float* hidden, hipStream_t st) {
    constexpr int32_t dt = sizeof(T) == 2 ? RP_BF16 : RP_F32;
    const int64_t mk = padded(m, dt), pk = padded(p, dt);
    if (ldx != mk) return fail(RP_ERR_UNSUPPORTED, "rows of X must be contiguous");
    int rc = rp_dense_project_device(device, X, dt, n, mk, C, p, Y, ldy, st, -1);
    if (rc) return rc;
    hipLaunchKernelGGL(shrink_kernel<T>, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, X, ldx, n, mk, down, mk, G, R,
                       (const float*)nullptr, ids, hidden);
    HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL((expand_kernel<T, float>), dim3((unsigned)n), dim3(256), 0, st, Y, ldy, Y, ldy, n, p, up, pk, G, R,
                       scale, ids, hidden);
    HIP_TRY(hipGetLastError());
    return RP_OK;
}

template <typename T>
int gradients(int device, const T* dY, int64_t lddy, const T* X, int64_t ldx, int64_t n, int64_t m, int64_t p, const T* Ct,
              const T* down, const T* up, int64_t G, int R, const float* scale, const int32_t* ids, const float* hidden, T* dX,
              int64_t lddx, float* d_down, int64_t ldd, int64_t sdd, float* d_up, int64_t ldu, int64_t sdu, char* ws,
              hipStream_t st) {
    constexpr int32_t dt = sizeof(T) == 2 ? RP_BF16 : RP_F32;
    const int64_t mk = padded(m, dt), pk = padded(p, dt);
    float* t = (float*)ws;
    if (n) {
        hipLaunchKernelGGL(shrink_kernel<T>, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, dY, lddy, n, pk, up, pk, G, R, scale,
                           ids, t);
        HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL(outer_kernel<T>, dim3((unsigned)((m + 255) / 256), (unsigned)std::min<int64_t>(G * R, 65535)), dim3(256), 0, st, X, ldx, n, m, G, R,
                       (const float*)nullptr, ids, t, d_down, ldd, sdd);
    HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(outer_kernel<T>, dim3((unsigned)((p + 255) / 256), (unsigned)std::min<int64_t>(G * R, 65535)), dim3(256), 0, st, dY, lddy, n, p, G,
                       R, scale, ids, hidden, d_up, ldu, sdu);
    HIP_TRY(hipGetLastError());
    if (dX && n) {
        if (lddy != pk) return fail(RP_ERR_UNSUPPORTED, "rows of dY must be contiguous");
        float* tmp = (float*)(ws + align256((size_t)n * R * 4));
        int rc = rp_dense_project_device(device, dY, dt, n, pk, Ct, m, tmp, m, st, -1);
        if (rc) return rc;
        hipLaunchKernelGGL((expand_kernel<T, T>), dim3((unsigned)n), dim3(256), 0, st, tmp, m, dX, lddx, n, m, down, mk, G, R,
                           (const float*)nullptr, ids, t);
        HIP_TRY(hipGetLastError());
    }
    return RP_OK;
}

}  // namespace

extern "C" {

int64_t rp_adapt_workspace_bytes(int32_t dtype, int64_t n, int64_t m, int64_t p, int64_t adapters, int32_t rank,
                                 int32_t what) {
    if (check_shared(dtype, n, m, p, adapters, rank)) return -1;
    size_t b = align256((size_t)n * rank * 4);
    if (what == RP_ADAPT_GRADIENTS_DX) b += (size_t)n * m * 4;
    return (int64_t)b;
}

int rp_adapt_project_device(int device, const void* X, int64_t ldx, int32_t dtype, int64_t n, int64_t m, const void* C,
                            int64_t p, const void* down, const void* up, int64_t adapters, int32_t rank, const float* scale,
                            const int32_t* ids, float* Y, int64_t ldy, float* hidden, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    int rc = check_shared(dtype, n, m, p, adapters, rank);
    if (rc) return rc;
    const int64_t mk = padded(m, dtype), pk = padded(p, dtype);
    if ((rc = check_operand("X", X, ldx, mk, dtype)) || (rc = check_operand("C", C, mk, mk, dtype)) ||
        (rc = check_operand("down", down, mk, mk, dtype)) || (rc = check_operand("up", up, pk, pk, dtype)))
        return rc;
    if (!ids || !Y) return fail(RP_ERR_INVALID, "NULL ids or Y");
    if (ldy < p) return fail(RP_ERR_INVALID, "Y: row stride %lld is under p=%lld", (long long)ldy, (long long)p);
    if (n == 0) return RP_OK;
    const int64_t need = rp_adapt_workspace_bytes(dtype, n, m, p, adapters, rank, RP_ADAPT_PROJECT);
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need)
        return fail(RP_ERR_INVALID, "workspace must be 256-byte aligned and hold %lld bytes", (long long)need);
    DeviceGuard guard;
    if ((rc = guard.enter(device))) return rc;
    if (!hidden) hidden = (float*)workspace;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == RP_BF16)
        return project<uint16_t>(device, (const uint16_t*)X, ldx, n, m, (const uint16_t*)C, p, (const uint16_t*)down,
                                 (const uint16_t*)up, adapters, rank, scale, ids, Y, ldy, hidden, st);
    return project<float>(device, (const float*)X, ldx, n, m, (const float*)C, p, (const float*)down, (const float*)up, adapters,
                          rank, scale, ids, Y, ldy, hidden, st);
}

int rp_adapt_gradients_device(int device, const void* dY, int64_t lddy, const void* X, int64_t ldx, int32_t dtype, int64_t n,
                              int64_t m, int64_t p, const void* Ct, const void* down, const void* up, int64_t adapters,
                              int32_t rank, const float* scale, const int32_t* ids, const float* hidden, void* dX,
                              int64_t lddx, float* d_down, int64_t d_down_row, int64_t d_down_adapter, float* d_up,
                              int64_t d_up_row, int64_t d_up_adapter, void* workspace, int64_t workspace_bytes,
                              void* stream) {
    int rc = check_shared(dtype, n, m, p, adapters, rank);
    if (rc) return rc;
    const int64_t mk = padded(m, dtype), pk = padded(p, dtype);
    if (n && ((rc = check_operand("dY", dY, lddy, pk, dtype)) || (rc = check_operand("X", X, ldx, mk, dtype)))) return rc;
    if ((rc = check_operand("down", down, mk, mk, dtype)) || (rc = check_operand("up", up, pk, pk, dtype))) return rc;
    if (!Ct != !dX) return fail(RP_ERR_INVALID, "Ct and dX go together");
    if (Ct && ((rc = check_operand("Ct", Ct, pk, pk, dtype)))) return rc;
    if (dX && lddx < m) return fail(RP_ERR_INVALID, "dX: row stride %lld is under m=%lld", (long long)lddx, (long long)m);
    if (!d_down || !d_up || (n && (!ids || !hidden))) return fail(RP_ERR_INVALID, "NULL ids, hidden, d_down or d_up");
    if (d_down_row < m || d_down_adapter < d_down_row * rank || d_up_row < p || d_up_adapter < d_up_row * rank)
        return fail(RP_ERR_INVALID, "d_down or d_up: strides under the shape");
    const int64_t need = rp_adapt_workspace_bytes(dtype, n, m, p, adapters, rank,
                                                  dX ? RP_ADAPT_GRADIENTS_DX : RP_ADAPT_GRADIENTS);
    if (need && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need))
        return fail(RP_ERR_INVALID, "workspace must be 256-byte aligned and hold %lld bytes", (long long)need);
    DeviceGuard guard;
    if ((rc = guard.enter(device))) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == RP_BF16)
        return gradients<uint16_t>(device, (const uint16_t*)dY, lddy, (const uint16_t*)X, ldx, n, m, p, (const uint16_t*)Ct,
                                   (const uint16_t*)down, (const uint16_t*)up, adapters, rank, scale, ids, hidden, (uint16_t*)dX,
                                   lddx, d_down, d_down_row, d_down_adapter, d_up, d_up_row, d_up_adapter, (char*)workspace, st);
    return gradients<float>(device, (const float*)dY, lddy, (const float*)X, ldx, n, m, p, (const float*)Ct, (const float*)down,
                            (const float*)up, adapters, rank, scale, ids, hidden, (float*)dX, lddx, d_down, d_down_row,
                            d_down_adapter, d_up, d_up_row, d_up_adapter, (char*)workspace, st);
}

}  // extern "C"
