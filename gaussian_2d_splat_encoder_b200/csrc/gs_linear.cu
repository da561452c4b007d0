// gs_linear.cu -- linear layer with bias, activation and residual, forward and backward (sm_100a).
//
//   z = x W^T + b,  y = act(z) + residual        x [M][K], W [N][K], y and z [M][N]
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz,  dresidual = dy
//
// First form: one tiled fp32 product with free strides serves the three matrix products.
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "../../include/gsplat_b200.h"
#include "gs_act.cuh"
#include "gs_prof.cuh"

void gs_set_last_error(const char *msg);

namespace {

__device__ __forceinline__ float act_rt(float z, int act) {
    return act == ACT_GELU ? gs_act<ACT_GELU>(z) : act == ACT_SILU ? gs_act<ACT_SILU>(z) : z;
}
__device__ __forceinline__ float slope_rt(float z, int act) {
    return act == ACT_GELU ? gs_act_slope<ACT_GELU>(z) : act == ACT_SILU ? gs_act_slope<ACT_SILU>(z) : 1.f;
}

// out[i][j] = act(sum_k A[i ai + k ak] B[j bj + k bk] + bias[j]) + residual[i][j]; z before the activation.
// 64 x 64 outputs per block, 4 x 4 per thread; long sums fold every 1024 terms.
template <typename T>
__global__ void __launch_bounds__(256) k_product(const T *A, long long ai, long long ak, const T *B, long long bj,
                                                 long long bk, long long I, int J, long long K, const T *bias,
                                                 const T *residual, long long ldr, int act, T *out, T *z) {
    __shared__ float sa[16][65], sb[16][65];
    const long long i0 = (long long)blockIdx.x * 64;
    const int j0 = blockIdx.y * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {}, tot[4][4] = {};
    for (long long k0 = 0; k0 < K; k0 += 16) {
        for (int e = threadIdx.x; e < 1024; e += 256) {
            // neighbouring threads walk the adjacent axis
            const int ka = ak == 1 ? e & 15 : e >> 6, ia = ak == 1 ? e >> 4 : e & 63;
            sa[ka][ia] = i0 + ia < I && k0 + ka < K ? to_f32(A[(i0 + ia) * ai + (k0 + ka) * ak]) : 0.f;
            const int kb = bk == 1 ? e & 15 : e >> 6, jb = bk == 1 ? e >> 4 : e & 63;
            sb[kb][jb] = j0 + jb < J && k0 + kb < K ? to_f32(B[(j0 + jb) * bj + (k0 + kb) * bk]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
        if ((k0 & 1023) == 1008 || k0 + 16 >= K)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                (&tot[0][0])[i] += (&acc[0][0])[i];
                (&acc[0][0])[i] = 0.f;
            }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long r = i0 + ty * 4 + i;
            const int c = j0 + tx * 4 + j;
            if (r >= I || c >= J) continue;
            float v = tot[i][j] + (bias ? to_f32(bias[c]) : 0.f);
            if (z) from_f32(v, z[r * J + c]);
            // (an explicit addition: no fusing with the activation in one of the branches and not in another)
            v = act_rt(v, act);
            if (residual) v = __fadd_rn(v, to_f32(residual[r * ldr + c]));
            from_f32(v, out[r * J + c]);
        }
}

template <typename T>
__global__ void __launch_bounds__(256) k_dz(const T *dy, long long ldy, const T *z, T *dz, long long M, int N, int act) {
    const long long n = M * N;
    for (long long k = blockIdx.x * 256LL + threadIdx.x; k < n; k += gridDim.x * 256LL) {
        const long long r = k / N;
        const int c = (int)(k - r * N);
        from_f32(to_f32(dy[r * ldy + c]) * (z ? slope_rt(to_f32(z[k]), act) : 1.f), dz[k]);
    }
}
// column sums: 32 columns per block, 32 row lanes
template <typename T>
__global__ void __launch_bounds__(1024) k_colsum(const T *dz, T *db, long long M, int N) {
    __shared__ float s[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
    float t = 0.f;
    if (c < N)
        for (long long r = ty; r < M; r += 32) t += to_f32(dz[r * N + c]);
    s[ty][tx] = t;
    __syncthreads();
    if (ty == 0 && c < N) {
        for (int k = 1; k < 32; k++) t += s[k][tx];
        from_f32(t, db[c]);
    }
}

bool valid(const gs_linear_desc *d) {
    return d && d->M >= 0 && d->M <= (1LL << 31) && d->N >= 1 && d->K >= 1 && d->N <= GS_LINEAR_MAX_DIM &&
           d->K <= GS_LINEAR_MAX_DIM && d->dtype >= GS_F32 && d->dtype <= GS_F16 && d->act >= GS_ACT_NONE &&
           d->act <= GS_ACT_SILU;
}
size_t elem(const gs_linear_desc *d) { return d->dtype == GS_F32 ? 4 : 2; }
size_t al(size_t n) { return (n + 255) & ~(size_t)255; }

int done(const char *where) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return GS_OK;
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", where, cudaGetErrorString(e));
    gs_set_last_error(msg);
    return GS_ERR_CUDA;
}

template <typename T>
void product(const void *A, long long ai, long long ak, const void *B, long long bj, long long bk, long long I, int J,
             long long K, const void *bias, const void *res, long long ldr, int act, void *out, void *z,
             cudaStream_t s) {
    dim3 grid((unsigned)((I + 63) / 64), (unsigned)((J + 63) / 64));
    k_product<T><<<grid, 256, 0, s>>>((const T *)A, ai, ak, (const T *)B, bj, bk, I, J, K, (const T *)bias,
                                      (const T *)res, ldr, act, (T *)out, (T *)z);
}

template <typename T>
int forward(const gs_linear_desc *d, const void *x, const void *w, const void *bias, const void *res, void *y, void *z,
            cudaStream_t s) {
    product<T>(x, d->ldx, 1, w, d->ldw, 1, d->M, d->N, d->K, bias, res, d->ldr, d->act, y, z, s);
    gs_count_launch(1);
    return done("gs_linear_act_fwd");
}
template <typename T>
int backward(const gs_linear_desc *d, const void *x, const void *w, const void *z, const void *dy, void *dx, void *dw,
             void *db, void *ws, cudaStream_t s) {
    const long long n = d->M * d->N;
    T *dz = (T *)al((uintptr_t)ws);
    k_dz<T><<<(unsigned)std::min<long long>((n + 255) / 256, 4096), 256, 0, s>>>((const T *)dy, d->ldy, (const T *)z,
                                                                                 dz, d->M, d->N, d->act);
    if (dx) product<T>(dz, d->N, 1, w, 1, d->ldw, d->M, d->K, d->N, nullptr, nullptr, 0, 0, dx, nullptr, s);
    if (dw) product<T>(dz, 1, d->N, x, 1, d->ldx, d->N, d->K, d->M, nullptr, nullptr, 0, 0, dw, nullptr, s);
    if (db) k_colsum<T><<<(unsigned)((d->N + 31) / 32), 1024, 0, s>>>(dz, (T *)db, d->M, d->N);
    gs_count_launch(1 + (dx != nullptr) + (dw != nullptr) + (db != nullptr));
    return done("gs_linear_act_bwd");
}

}  // namespace

extern "C" size_t gs_linear_act_workspace_size(const gs_linear_desc *d, int backward) {
    if (!valid(d)) return 0;
    return 256 + (backward ? al((size_t)d->M * d->N * elem(d)) : 0);
}

extern "C" int gs_linear_act_fwd(const gs_linear_desc *d, const void *x, const void *w, const void *bias,
                                 const void *residual, void *y, void *z, void *workspace, size_t workspace_bytes,
                                 void *stream) {
    if (!valid(d) || d->ldx < d->K || d->ldw < d->K || (residual && d->ldr < d->N)) return GS_ERR_BAD_ARGUMENT;
    if (d->M == 0) return GS_OK;
    if (!x || !w || !y) return GS_ERR_BAD_ARGUMENT;
    if (!workspace || workspace_bytes < gs_linear_act_workspace_size(d, 0)) return GS_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    if (d->dtype == GS_F32) return forward<float>(d, x, w, bias, residual, y, z, s);
    if (d->dtype == GS_BF16) return forward<__nv_bfloat16>(d, x, w, bias, residual, y, z, s);
    return forward<__half>(d, x, w, bias, residual, y, z, s);
}

extern "C" int gs_linear_act_bwd(const gs_linear_desc *d, const void *x, const void *w, const void *z, const void *dy,
                                 void *dx, void *dw, void *dbias, void *workspace, size_t workspace_bytes,
                                 void *stream) {
    if (!valid(d) || d->ldx < d->K || d->ldw < d->K || d->ldy < d->N) return GS_ERR_BAD_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    if (d->M == 0) {
        if (dw) cudaMemsetAsync(dw, 0, (size_t)d->N * d->K * elem(d), s);
        if (dbias) cudaMemsetAsync(dbias, 0, (size_t)d->N * elem(d), s);
        return done("gs_linear_act_bwd");
    }
    if (!x || !w || !dy || (d->act != GS_ACT_NONE && !z)) return GS_ERR_BAD_ARGUMENT;
    if (!workspace || workspace_bytes < gs_linear_act_workspace_size(d, 1)) return GS_ERR_WORKSPACE;
    if (d->act == GS_ACT_NONE) z = nullptr;
    if (d->dtype == GS_F32) return backward<float>(d, x, w, z, dy, dx, dw, dbias, workspace, s);
    if (d->dtype == GS_BF16) return backward<__nv_bfloat16>(d, x, w, z, dy, dx, dw, dbias, workspace, s);
    return backward<__half>(d, x, w, z, dy, dx, dw, dbias, workspace, s);
}
