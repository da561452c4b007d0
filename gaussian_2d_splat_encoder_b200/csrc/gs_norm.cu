// gs_norm.cu -- GroupNorm with an activation on channels-last maps, forward and backward (sm_100a).
//
// x is [B][rows][C] (an image's pixels are rows; row and image strides are free, channels are adjacent),
// G groups of cpg = C / G channels.  With m, v the mean and biased variance of a group of one image and
// r = 1 / sqrt(v + eps):
//   act after  (act_first 0):  xh = (x - m) r,       y = act(w xh + b)
//   act before (act_first 1):  xh = (act(x) - m) r,  y = w xh + b
// Backward, dz the gradient of w xh + b (dy act'(z), or dy itself) and n = rows cpg:
//   db = sum dz,  dw = sum dz xh  (over images and rows),
//   du = r (w dz - mean(w dz) - xh mean(w dz xh)),  dx = du, or du act'(x)
// where the two group means follow from the image's channel sums: sum_c w_c db_c and sum_c w_c dw_c.
//
// The operator moves bytes: x is needed twice (statistics, then the map) and fits no SM, so each direction
// is two launches over the same slices, the second of which finds what L2 (126 MB) still holds.  A block
// takes a run of rows of one image (and, where there are many groups, a chunk of whole groups); a thread
// keeps one 16-byte vector of channels for all its rows, so parameters and sums stay in registers and a
// warp reads contiguous memory.  Statistics are two passes over the slice in fp32 around the slice's own
// mean, joined across slices as (n, mean, M2): no difference of large squares.  All sums run in a fixed order.
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

constexpr int MAX_T = 512;       // threads of a block

struct NormArgs {
    const void *x, *dy, *w, *b;
    void *y, *dx, *dw, *db;
    float *stats;   // [B][G][2] mean, 1 / sqrt(var + eps)
    float *part;    // forward [B][splits][G][2] mean, M2; backward the two group sums
    float *cpart;   // backward [B][splits][C][2] channel sums of dz and dz xh
    long long rows, x_row, x_img, dy_row, dy_img;
    int B, C, G, cpg, splits;
    int chunk, nchunk, cvec, rl;  // channels per block, blocks over channels, vectors per row, rows in flight
    int nslice;                   // blocks of the backward's second launch that map slices
    int param_f32;
    float eps;
};

template <typename T>
__device__ __forceinline__ float param(const void *p, int f32, int c) {
    return f32 ? reinterpret_cast<const float *>(p)[c] : to_f32(reinterpret_cast<const T *>(p)[c]);
}
template <typename T>
__device__ __forceinline__ void set_param(void *p, int f32, int c, float v) {
    if (f32) reinterpret_cast<float *>(p)[c] = v;
    else from_f32(v, reinterpret_cast<T *>(p)[c]);
}

// one vector of channels; without 16-byte alignment (or at a ragged end) element by element, zeros beyond
template <typename T, bool VEC>
__device__ __forceinline__ void load(const T *p, int valid, float *v) {
    if (VEC) {
        unpack16<T>(*reinterpret_cast<const uint4 *>(p), v);
    } else {
#pragma unroll
        for (int i = 0; i < Vec<T>::N; i++) v[i] = i < valid ? to_f32(p[i]) : 0.f;
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store(T *p, int valid, const float *v) {
    if (VEC) {
        *reinterpret_cast<uint4 *>(p) = pack16<T>(v);
    } else {
#pragma unroll
        for (int i = 0; i < Vec<T>::N; i++)
            if (i < valid) from_f32(v[i], p[i]);
    }
}

// The slice of a block and the place of a thread in it.
struct Slice {
    int b, s, c0, cc;   // image, split, first channel, channels of this chunk
    int r, cv, c, valid;  // row lane, vector, its first channel, its channels (<= 0: idle thread)
    long long lo, hi;   // rows
    __device__ Slice(const NormArgs &a, int V) {
        int t = blockIdx.x;
        const int k = t % a.nchunk;
        t /= a.nchunk;
        s = t % a.splits;
        b = t / a.splits;
        c0 = k * a.chunk;
        cc = min(a.chunk, a.C - c0);
        r = (int)threadIdx.x / a.cvec;
        cv = (int)threadIdx.x - r * a.cvec;
        c = c0 + cv * V;
        valid = r < a.rl ? min(V, cc - cv * V) : 0;
        lo = a.rows * s / a.splits;
        hi = a.rows * (s + 1) / a.splits;
    }
};

// Sums of the block's threads by channel: the row lanes fold in a tree, buf[0..cvec*V) holds the result.
template <int V>
__device__ __forceinline__ void fold_rows(float *buf, const float *v, const NormArgs &a, const Slice &sl) {
    const int w = a.cvec * V;
    __syncthreads();
    if (sl.r < a.rl)
#pragma unroll
        for (int i = 0; i < V; i++) buf[sl.r * w + sl.cv * V + i] = i < sl.valid ? v[i] : 0.f;
    int n = a.rl;
    while (n > 1) {
        const int h = (n + 1) >> 1;
        __syncthreads();
        if (sl.r < n - h)
#pragma unroll
            for (int i = 0; i < V; i++) buf[sl.r * w + sl.cv * V + i] += buf[(sl.r + h) * w + sl.cv * V + i];
        n = h;
    }
    __syncthreads();
}
// Sums of the chunk's groups from channel sums, a warp per group; f maps a channel's sum.
template <typename F>
__device__ __forceinline__ void fold_groups(float *gsum, int groups, int cpg, F f) {
    for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
        float s = 0.f;
        for (int c = threadIdx.x & 31; c < cpg; c += 32) s += f(g * cpg + c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if ((threadIdx.x & 31) == 0) gsum[g] = s;
    }
    __syncthreads();
}

// ---- forward, first launch: mean and M2 of the slice's groups
template <typename T, bool VEC, int PRE>
__global__ void __launch_bounds__(MAX_T) k_gn_stats(NormArgs a) {
    constexpr int V = Vec<T>::N;
    extern __shared__ float sm[];
    const Slice sl(a, V);
    const int groups = sl.cc / a.cpg, w = a.cvec * V;
    float *buf = sm, *gsum = sm + (size_t)a.rl * w, *gsq = gsum + a.chunk / a.cpg;
    const T *x = reinterpret_cast<const T *>(a.x) + sl.b * a.x_img + sl.c;
    float s[V], v[V];
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = 0.f;
    if (sl.valid > 0)
#pragma unroll 4
        for (long long r = sl.lo + sl.r; r < sl.hi; r += a.rl) {
            load<T, VEC>(x + r * a.x_row, sl.valid, v);
#pragma unroll
            for (int i = 0; i < V; i++) s[i] += gs_act<PRE>(v[i]);
        }
    fold_rows<V>(buf, s, a, sl);
    fold_groups(gsum, groups, a.cpg, [&](int c) { return buf[c]; });
    // second pass around the slice's mean; its first moment corrects the mean's own rounding
    const float inv = 1.0f / ((float)(sl.hi - sl.lo) * (float)a.cpg);
    float m[V], q[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        m[i] = i < sl.valid ? gsum[(sl.cv * V + i) / a.cpg] * inv : 0.f;
        s[i] = q[i] = 0.f;
    }
    if (sl.valid > 0)
#pragma unroll 4
        for (long long r = sl.lo + sl.r; r < sl.hi; r += a.rl) {
            load<T, VEC>(x + r * a.x_row, sl.valid, v);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float d = gs_act<PRE>(v[i]) - m[i];
                s[i] += d;
                q[i] = fmaf(d, d, q[i]);
            }
        }
    fold_rows<V>(buf, q, a, sl);
    fold_groups(gsq, groups, a.cpg, [&](int c) { return buf[c]; });
    fold_rows<V>(buf, s, a, sl);
    for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
        float d = 0.f;
        for (int c = threadIdx.x & 31; c < a.cpg; c += 32) d += buf[g * a.cpg + c];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        if ((threadIdx.x & 31) == 0) {
            float2 *out = reinterpret_cast<float2 *>(a.part) + ((long long)sl.b * a.splits + sl.s) * a.G;
            out[sl.c0 / a.cpg + g] = make_float2(gsum[g] * inv + d * inv, gsq[g] - d * d * inv);
        }
    }
}

// mean and 1 / sqrt(var + eps) of the chunk's groups from the slices' (n, mean, M2), a warp per group
__device__ __forceinline__ void join_stats(const NormArgs &a, const Slice &sl, float *mean, float *rstd) {
    const int groups = sl.cc / a.cpg, lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
        const int gg = sl.c0 / a.cpg + g;
        const float2 *p = reinterpret_cast<const float2 *>(a.part) + (long long)sl.b * a.splits * a.G + gg;
        const float m0 = p[0].x;
        const float inv = 1.0f / (float)a.rows;
        float d = 0.f;
        for (int s = lane; s < a.splits; s += 32) {
            const float n = (float)(a.rows * (s + 1) / a.splits - a.rows * s / a.splits);
            d = fmaf(n * inv, p[(long long)s * a.G].x - m0, d);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        const float m = m0 + d;
        float q = 0.f;
        for (int s = lane; s < a.splits; s += 32) {
            const float n = (float)(a.rows * (s + 1) / a.splits - a.rows * s / a.splits);
            const float2 e = p[(long long)s * a.G];
            q += fmaf(n * (float)a.cpg * (e.x - m), e.x - m, e.y) * (inv / (float)a.cpg);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
        if (lane == 0) {
            mean[g] = m;
            rstd[g] = 1.0f / sqrtf(q + a.eps);
            if (sl.s == 0 && a.stats)
                reinterpret_cast<float2 *>(a.stats)[(long long)sl.b * a.G + gg] = make_float2(m, rstd[g]);
        }
    }
    __syncthreads();
}

// ---- forward, second launch: the map
template <typename T, bool VEC, int PRE, int POST>
__global__ void __launch_bounds__(MAX_T) k_gn_map(NormArgs a) {
    constexpr int V = Vec<T>::N;
    extern __shared__ float sm[];
    const Slice sl(a, V);
    float *mean = sm, *rstd = sm + a.chunk / a.cpg;
    join_stats(a, sl, mean, rstd);
    if (sl.valid <= 0) return;
    float m[V], k[V], b[V], v[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int c = sl.c + min(i, sl.valid - 1), g = (c - sl.c0) / a.cpg;
        m[i] = mean[g];
        k[i] = rstd[g] * (a.w ? param<T>(a.w, a.param_f32, c) : 1.f);
        b[i] = a.b ? param<T>(a.b, a.param_f32, c) : 0.f;
    }
    const T *x = reinterpret_cast<const T *>(a.x) + sl.b * a.x_img + sl.c;
    T *y = reinterpret_cast<T *>(a.y) + sl.b * a.rows * a.C + sl.c;
#pragma unroll 4
    for (long long r = sl.lo + sl.r; r < sl.hi; r += a.rl) {
        load<T, VEC>(x + r * a.x_row, sl.valid, v);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = gs_act<POST>(fmaf(gs_act<PRE>(v[i]) - m[i], k[i], b[i]));
        store<T, VEC>(y + r * a.C, sl.valid, v);
    }
}

// xh, and dz from dy, of one element; w, b are read only where the activation comes after
template <int PRE, int POST>
__device__ __forceinline__ void grad_of(float x, float dy, float m, float rs, float w, float b, float &xh, float &dz) {
    xh = (gs_act<PRE>(x) - m) * rs;
    dz = POST ? dy * gs_act_slope<POST>(fmaf(xh, w, b)) : dy;
}

// ---- backward, first launch: channel sums of dz and dz xh, and their group sums weighted by w
template <typename T, bool VEC, int PRE, int POST>
__global__ void __launch_bounds__(MAX_T) k_gn_grad_sums(NormArgs a) {
    constexpr int V = Vec<T>::N;
    extern __shared__ float sm[];
    const Slice sl(a, V);
    const int groups = sl.cc / a.cpg, w = a.cvec * V;
    float *buf = sm, *g0 = sm + (size_t)a.rl * w, *g1 = g0 + a.chunk / a.cpg;
    float sz[V], sx[V];
#pragma unroll
    for (int i = 0; i < V; i++) sz[i] = sx[i] = 0.f;
    if (sl.valid > 0) {
        float m[V], rs[V], wt[V], bs[V], v[V], d[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = sl.c + min(i, sl.valid - 1);
            const float2 st = reinterpret_cast<const float2 *>(a.stats)[(long long)sl.b * a.G + c / a.cpg];
            m[i] = st.x;
            rs[i] = st.y;
            wt[i] = a.w ? param<T>(a.w, a.param_f32, c) : 1.f;
            bs[i] = a.b ? param<T>(a.b, a.param_f32, c) : 0.f;
        }
        const T *x = reinterpret_cast<const T *>(a.x) + sl.b * a.x_img + sl.c;
        const T *dy = reinterpret_cast<const T *>(a.dy) + sl.b * a.dy_img + sl.c;
#pragma unroll 2
        for (long long r = sl.lo + sl.r; r < sl.hi; r += a.rl) {
            load<T, VEC>(x + r * a.x_row, sl.valid, v);
            load<T, VEC>(dy + r * a.dy_row, sl.valid, d);
#pragma unroll
            for (int i = 0; i < V; i++) {
                float xh, dz;
                grad_of<PRE, POST>(v[i], d[i], m[i], rs[i], wt[i], bs[i], xh, dz);
                sz[i] += dz;
                sx[i] = fmaf(dz, xh, sx[i]);
            }
        }
    }
    float2 *cp = reinterpret_cast<float2 *>(a.cpart) + ((long long)sl.b * a.splits + sl.s) * a.C;
    float2 *gp = reinterpret_cast<float2 *>(a.part) + ((long long)sl.b * a.splits + sl.s) * a.G + sl.c0 / a.cpg;
    auto weight = [&](int c) { return a.w ? param<T>(a.w, a.param_f32, sl.c0 + c) : 1.f; };
    fold_rows<V>(buf, sz, a, sl);
    for (int c = threadIdx.x; c < sl.cc; c += blockDim.x) cp[sl.c0 + c].x = buf[c];
    fold_groups(g0, groups, a.cpg, [&](int c) { return buf[c] * weight(c); });
    fold_rows<V>(buf, sx, a, sl);
    for (int c = threadIdx.x; c < sl.cc; c += blockDim.x) cp[sl.c0 + c].y = buf[c];
    fold_groups(g1, groups, a.cpg, [&](int c) { return buf[c] * weight(c); });
    for (int g = threadIdx.x; g < groups; g += blockDim.x) gp[g] = make_float2(g0[g], g1[g]);
}

// ---- backward, second launch: dx; the blocks after the slices' fold the channel sums into dw and db
template <typename T, bool VEC, int PRE, int POST>
__global__ void __launch_bounds__(MAX_T) k_gn_grad_map(NormArgs a) {
    constexpr int V = Vec<T>::N;
    extern __shared__ float sm[];
    if ((int)blockIdx.x >= a.nslice) {
        // 32 channels per block, the (image, split) sums dealt to the warps, joined in order
        float2 *red = reinterpret_cast<float2 *>(sm);
        const int lane = threadIdx.x & 31, nw = blockDim.x >> 5, c = ((int)blockIdx.x - a.nslice) * 32 + lane;
        const float2 *cp = reinterpret_cast<const float2 *>(a.cpart);
        float2 t = make_float2(0.f, 0.f);
        if (c < a.C)
#pragma unroll 4
            for (int k = threadIdx.x >> 5; k < a.B * a.splits; k += nw) {
                const float2 e = cp[(long long)k * a.C + c];
                t.x += e.x;
                t.y += e.y;
            }
        red[threadIdx.x] = t;
        __syncthreads();
        if (threadIdx.x < 32 && c < a.C) {
            for (int k = 1; k < nw; k++) {
                t.x += red[k * 32 + lane].x;
                t.y += red[k * 32 + lane].y;
            }
            if (a.db) set_param<T>(a.db, a.param_f32, c, t.x);
            if (a.dw) set_param<T>(a.dw, a.param_f32, c, t.y);
        }
        return;
    }
    const Slice sl(a, V);
    const int groups = sl.cc / a.cpg;
    float *g0 = sm, *g1 = sm + a.chunk / a.cpg;
    const float inv = 1.0f / ((float)a.rows * (float)a.cpg);
    for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
        const float2 *p = reinterpret_cast<const float2 *>(a.part) + (long long)sl.b * a.splits * a.G + sl.c0 / a.cpg + g;
        float s0 = 0.f, s1 = 0.f;
        for (int s = threadIdx.x & 31; s < a.splits; s += 32) {
            const float2 e = p[(long long)s * a.G];
            s0 += e.x;
            s1 += e.y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s0 += __shfl_xor_sync(0xffffffffu, s0, o);
            s1 += __shfl_xor_sync(0xffffffffu, s1, o);
        }
        if ((threadIdx.x & 31) == 0) {
            g0[g] = s0 * inv;
            g1[g] = s1 * inv;
        }
    }
    __syncthreads();
    if (sl.valid <= 0) return;
    float m[V], rs[V], wt[V], bs[V], m0[V], m1[V], v[V], d[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int c = sl.c + min(i, sl.valid - 1), g = (c - sl.c0) / a.cpg;
        const float2 st = reinterpret_cast<const float2 *>(a.stats)[(long long)sl.b * a.G + c / a.cpg];
        m[i] = st.x;
        rs[i] = st.y;
        wt[i] = a.w ? param<T>(a.w, a.param_f32, c) : 1.f;
        bs[i] = a.b ? param<T>(a.b, a.param_f32, c) : 0.f;
        m0[i] = g0[g];
        m1[i] = g1[g];
    }
    const T *x = reinterpret_cast<const T *>(a.x) + sl.b * a.x_img + sl.c;
    const T *dy = reinterpret_cast<const T *>(a.dy) + sl.b * a.dy_img + sl.c;
    T *dx = reinterpret_cast<T *>(a.dx) + sl.b * a.rows * a.C + sl.c;
#pragma unroll 2
    for (long long r = sl.lo + sl.r; r < sl.hi; r += a.rl) {
        load<T, VEC>(x + r * a.x_row, sl.valid, v);
        load<T, VEC>(dy + r * a.dy_row, sl.valid, d);
#pragma unroll
        for (int i = 0; i < V; i++) {
            float xh, dz;
            grad_of<PRE, POST>(v[i], d[i], m[i], rs[i], wt[i], bs[i], xh, dz);
            const float du = rs[i] * (fmaf(wt[i], dz, -m0[i]) - xh * m1[i]);
            v[i] = PRE ? du * gs_act_slope<PRE>(v[i]) : du;
        }
        store<T, VEC>(dx + r * a.C, sl.valid, v);
    }
}

// ---- host
int elem_size(int dtype) { return dtype == GS_F32 ? 4 : 2; }

constexpr int SMS = 148;  // of a B200: the split of the work, and with it the workspace, is a matter of sizes alone

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// Fills sizes and the split of the work; false for arguments outside the operator's range.
bool plan(const gs_norm_desc *d, NormArgs &a) {
    memset(&a, 0, sizeof(a));
    if (!d || d->B < 0 || d->rows < 0 || d->C < 1 || d->groups < 1 || d->C % d->groups) return false;
    if (d->dtype < GS_F32 || d->dtype > GS_F16 || d->act < GS_ACT_NONE || d->act > GS_ACT_SILU) return false;
    if (d->param_dtype != GS_F32 && d->param_dtype != d->dtype) return false;
    if (!(d->eps >= 0.f) || d->C > GS_NORM_MAX_C || d->rows > (1LL << 40)) return false;
    a.B = d->B; a.C = d->C; a.G = d->groups; a.cpg = d->C / d->groups; a.rows = d->rows;
    a.x_row = d->x_row; a.x_img = d->x_img; a.dy_row = d->dy_row; a.dy_img = d->dy_img;
    a.param_f32 = d->param_dtype == GS_F32;
    a.eps = d->eps;
    const int V = 16 / elem_size(d->dtype);
    // many groups: a block takes whole groups of about 64 channels (128 contiguous bytes a row in 16 bits), so
    // the second launch joins only those groups' sums
    a.chunk = a.C;
    if (a.G > 32) {
        const int unit = a.cpg / gcd(a.cpg, V) * V;  // whole groups and whole vectors
        const int want = (64 + unit - 1) / unit * unit;
        if (want < a.C) a.chunk = want;
    }
    a.nchunk = (a.C + a.chunk - 1) / a.chunk;
    a.cvec = (a.chunk + V - 1) / V;
    a.rl = std::max(1, 256 / a.cvec);
    // four blocks of 256 threads per SM, but no fewer than four rows a thread
    const long long most = std::max<long long>(1, a.rows / (4LL * a.rl));
    const long long want = std::max<long long>(1, 4LL * SMS / std::max<long long>(1, (long long)a.B * a.nchunk));
    a.splits = (int)std::min({most, want, 1024LL});
    return (long long)a.B * a.splits * a.nchunk < (1LL << 30);
}

size_t al(size_t n) { return (n + 255) & ~(size_t)255; }
size_t part_bytes(const NormArgs &a) { return al((size_t)a.B * a.splits * a.G * 8); }

bool aligned(const void *p, long long row, long long img, int V) {
    return ((uintptr_t)p & 15) == 0 && row % V == 0 && img % V == 0;
}

int done(const char *where) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return GS_OK;
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", where, cudaGetErrorString(e));
    gs_set_last_error(msg);
    return GS_ERR_CUDA;
}

int threads(const NormArgs &a) { return (a.rl * a.cvec + 31) / 32 * 32; }
// shared memory of the kernels that fold sums, and of those that only join group values
template <typename T>
size_t fold_smem(const NormArgs &a) {
    return ((size_t)a.rl * a.cvec * Vec<T>::N + 2 * (size_t)(a.chunk / a.cpg)) * sizeof(float);
}
size_t join_smem(const NormArgs &a) {
    return std::max<size_t>(2 * (size_t)(a.chunk / a.cpg) * sizeof(float), (size_t)MAX_T * sizeof(float2));
}

template <typename T, bool VEC, int PRE, int POST>
int forward(const NormArgs &a, cudaStream_t s) {
    const unsigned grid = (unsigned)(a.B * a.splits * a.nchunk);
    k_gn_stats<T, VEC, PRE><<<grid, threads(a), fold_smem<T>(a), s>>>(a);
    k_gn_map<T, VEC, PRE, POST><<<grid, threads(a), join_smem(a), s>>>(a);
    gs_count_launch(2);
    return done("gs_group_norm_act_fwd");
}
template <typename T, bool VEC, int PRE, int POST>
int backward(const NormArgs &a, cudaStream_t s) {
    const unsigned grid = (unsigned)(a.B * a.splits * a.nchunk), fold = a.dw || a.db ? (a.C + 31) / 32 : 0;
    if (a.nslice + fold == 0) return GS_OK;
    k_gn_grad_sums<T, VEC, PRE, POST><<<grid, threads(a), fold_smem<T>(a), s>>>(a);
    k_gn_grad_map<T, VEC, PRE, POST><<<a.nslice + fold, threads(a), join_smem(a), s>>>(a);
    gs_count_launch(2);
    return done("gs_group_norm_act_bwd");
}

template <bool BWD, typename T, bool VEC>
int by_act(const gs_norm_desc *d, const NormArgs &a, cudaStream_t s) {
    const int mode = d->act == GS_ACT_NONE ? 0 : d->act_first ? d->act : 2 + d->act;
    switch (mode) {
        case 0: return BWD ? backward<T, VEC, 0, 0>(a, s) : forward<T, VEC, 0, 0>(a, s);
        case 1: return BWD ? backward<T, VEC, ACT_GELU, 0>(a, s) : forward<T, VEC, ACT_GELU, 0>(a, s);
        case 2: return BWD ? backward<T, VEC, ACT_SILU, 0>(a, s) : forward<T, VEC, ACT_SILU, 0>(a, s);
        case 3: return BWD ? backward<T, VEC, 0, ACT_GELU>(a, s) : forward<T, VEC, 0, ACT_GELU>(a, s);
        default: return BWD ? backward<T, VEC, 0, ACT_SILU>(a, s) : forward<T, VEC, 0, ACT_SILU>(a, s);
    }
}
template <bool BWD>
int by_type(const gs_norm_desc *d, const NormArgs &a, bool vec, cudaStream_t s) {
    if (d->dtype == GS_F32) return vec ? by_act<BWD, float, true>(d, a, s) : by_act<BWD, float, false>(d, a, s);
    if (d->dtype == GS_BF16)
        return vec ? by_act<BWD, __nv_bfloat16, true>(d, a, s) : by_act<BWD, __nv_bfloat16, false>(d, a, s);
    return vec ? by_act<BWD, __half, true>(d, a, s) : by_act<BWD, __half, false>(d, a, s);
}

}  // namespace

extern "C" size_t gs_group_norm_act_workspace_size(const gs_norm_desc *d, int backward) {
    NormArgs a;
    if (!plan(d, a)) return 0;
    return part_bytes(a) + (backward ? al((size_t)a.B * a.splits * a.C * 8) : 0) + 256;
}

extern "C" int gs_group_norm_act_fwd(const gs_norm_desc *d, const void *x, const void *weight, const void *bias,
                                     void *y, float *stats, void *workspace, size_t workspace_bytes, void *stream) {
    NormArgs a;
    if (!plan(d, a)) return GS_ERR_BAD_ARGUMENT;
    if (a.B == 0 || a.rows == 0) return GS_OK;
    if (!x || !y) return GS_ERR_BAD_ARGUMENT;
    if (!workspace || workspace_bytes < gs_group_norm_act_workspace_size(d, 0)) return GS_ERR_WORKSPACE;
    a.x = x; a.w = weight; a.b = bias; a.y = y; a.stats = stats;
    a.part = reinterpret_cast<float *>(al((uintptr_t)workspace));
    const int V = 16 / elem_size(d->dtype);
    const bool vec = aligned(x, a.x_row, a.x_img, V) && aligned(y, a.C, 0, V);
    return by_type<false>(d, a, vec, (cudaStream_t)stream);
}

extern "C" int gs_group_norm_act_bwd(const gs_norm_desc *d, const void *x, const void *weight, const void *bias,
                                     const float *stats, const void *dy, void *dx, void *dweight, void *dbias,
                                     void *workspace, size_t workspace_bytes, void *stream) {
    NormArgs a;
    if (!plan(d, a)) return GS_ERR_BAD_ARGUMENT;
    if (a.B == 0 || a.rows == 0) {
        const size_t n = (size_t)a.C * elem_size(d->param_dtype);
        if (dweight) cudaMemsetAsync(dweight, 0, n, (cudaStream_t)stream);
        if (dbias) cudaMemsetAsync(dbias, 0, n, (cudaStream_t)stream);
        return done("gs_group_norm_act_bwd");
    }
    if (!x || !stats || !dy) return GS_ERR_BAD_ARGUMENT;
    if (!workspace || workspace_bytes < gs_group_norm_act_workspace_size(d, 1)) return GS_ERR_WORKSPACE;
    a.x = x; a.w = weight; a.b = bias; a.stats = const_cast<float *>(stats); a.dy = dy; a.dx = dx; a.dw = dweight;
    a.db = dbias;
    a.nslice = dx ? a.B * a.splits * a.nchunk : 0;
    a.part = reinterpret_cast<float *>(al((uintptr_t)workspace));
    a.cpart = reinterpret_cast<float *>(reinterpret_cast<char *>(a.part) + part_bytes(a));
    const int V = 16 / elem_size(d->dtype);
    const bool vec = aligned(x, a.x_row, a.x_img, V) && aligned(dy, a.dy_row, a.dy_img, V) && (!dx || aligned(dx, a.C, 0, V));
    return by_type<true>(d, a, vec, (cudaStream_t)stream);
}
