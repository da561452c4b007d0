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
// The operator moves bytes: x is needed twice (statistics, then the map) and a map of training size fits no
// SM, so each direction is two launches over the same slices, the second of which finds what L2 (126 MB)
// still holds.  A block takes a run of rows of one image (and, where there are many groups, a chunk of
// whole groups); a thread keeps one 16-byte vector of channels for all its rows, so parameters and sums stay
// in registers and a warp reads contiguous memory.  A forward whose image and group chunk fit the shared
// memory of a cluster's CTAs is one launch: values are read once, the cluster joins its sums over distributed
// shared memory.  Statistics are taken around means, never as a difference of large squares: two rows at a time
// exactly around their own mean, joined as (n, mean, M2).  All sums run in a fixed order.
//
// Each launch evaluates an activation once per element (GELU: 0.125 cycles of an SM's MUFU).  Measured: 4x384x384x64
// bf16 with SiLU 44 us (its bytes take 23): statistics 18 to 20, x at half of memory's rate, its warps waiting for
// loads; the map 24, MUFU busy 61 to 68 % of the time, warps queued before it and shared memory.  A training step of
// 4x192x192x128 with GELU first 79 us (19, 18, 21, 26; bytes 23): issue slots 56 to 62 %, MUFU 36 to 56 %, FMA 46 to 52 %,
// memory 21 to 39 %, so no unit is full: latency, with three to five warps a scheduler.  96x96x256 in one launch 13.4 us
// against 27 in two.
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

constexpr int MAX_T = 256;  // threads of a block
constexpr int V = 8;        // channels of a thread's vector
constexpr int FUSED_T = 512, FUSED_R = 12;  // one-launch form: threads, most vectors a thread holds

struct NormArgs {
    const void *x, *dy, *w, *b;
    void *y, *dx, *dw, *db;
    float *stats;   // [B][G][2] mean, 1 / sqrt(var + eps)
    float *part;    // forward [B][splits][G][2] mean, M2; backward the two group sums
    float *cpart;   // backward [B][splits][C][2] channel sums of dz and dz xh
    long long x_row, x_img, dy_row, dy_img;
    int rows, per;  // rows of an image, of a slice
    int B, C, G, cpg, splits;
    int chunk, nchunk, cvec, rl;  // channels per block, blocks over channels, vectors per row, rows in flight
    int nslice;                   // blocks of the backward's second launch that map slices
    int param_f32, fused, held;  // held: vectors a thread of the one-launch form holds
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
__device__ __forceinline__ Raw8<T> fetch(const T *p, int valid) {
    if constexpr (VEC) {
        return *reinterpret_cast<const Raw8<T> *>(p);
    } else {
        union {
            Raw8<T> q;
            T e[V];
        } u;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < valid) u.e[i] = p[i];
            else from_f32(0.f, u.e[i]);
        return u.q;
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store(T *p, int valid, const f2 *v) {
    if (VEC) {
        *reinterpret_cast<Raw8<T> *>(p) = pack8<T>(v);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < valid) from_f32(at(v, i), p[i]);
    }
}

// The slice of a block and the place of a thread in it.
struct Slice {
    int b, s, c0, cc;     // image, split, first channel, channels of this chunk
    int r, cv, c, valid;  // row lane, vector, its first channel, its channels (<= 0: idle thread)
    int lo, hi;           // rows
    __device__ Slice(const NormArgs &a, bool cluster = false) {
        int t = blockIdx.x, k;
        if (cluster) {  // the splits of a chunk are neighbours
            s = t % a.splits;
            t /= a.splits;
            k = t % a.nchunk;
            b = t / a.nchunk;
        } else {
            k = t % a.nchunk;
            t /= a.nchunk;
            s = t % a.splits;
            b = t / a.splits;
        }
        c0 = k * a.chunk;
        cc = min(a.chunk, a.C - c0);
        r = (int)threadIdx.x / a.cvec;
        cv = (int)threadIdx.x - r * a.cvec;
        c = c0 + cv * V;
        valid = r < a.rl ? min(V, cc - cv * V) : 0;
        lo = s * a.per;
        hi = min(lo + a.per, a.rows);
    }
    // rows of this thread: lo + r, lo + r + rl, ...
    __device__ int rows(const NormArgs &a) const { return valid > 0 && r < hi - lo ? (hi - 1 - lo - r) / a.rl + 1 : 0; }
};
// f(i, group of channel i) for a thread's channels, groups counted from the chunk's first
template <typename F>
__device__ __forceinline__ void each_channel(const NormArgs &a, const Slice &sl, F f) {
    const int g = (sl.c - sl.c0) / a.cpg;
    if (a.cpg % V == 0) {
#pragma unroll
        for (int i = 0; i < V; i++) f(i, g);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) f(i, (sl.c - sl.c0 + min(i, sl.valid - 1)) / a.cpg);
    }
}

// A thread's rows of S tensors, fed through a ring of its own in shared memory: NB batches of B rows, cp.async
// keeps NB - 1 of them in flight without holding registers.  Unaligned rows are read in place.
__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
                 : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// NB, a power of two, so a batch's place is a mask away and a row's an immediate offset from it
template <typename T>
constexpr int ring_batches() {
    return sizeof(T) == 4 ? 2 : 4;  // fp32 rows are twice as wide
}
template <typename T, bool VEC, int S, int B, bool KEEP = false>
struct Feed {
    // KEEP: room for all rows, as fp32
    static constexpr int NB = KEEP ? FUSED_R / B : ring_batches<T>();
    static constexpr int threads() { return KEEP ? FUSED_T : MAX_T; }
    static constexpr int pieces() { return KEEP ? 2 : (int)sizeof(T) / 2; }
    static constexpr int place(int batch) { return KEEP ? batch : batch & (NB - 1); }
    static constexpr int row() { return S * pieces() * threads(); }  // 16-byte pieces of one row of all threads
    const T *next[S], *here[S];  // of the next batch to issue; unaligned: of the batch to read
    long long step[S];           // row to row
    int n, valid;                // rows of this thread
    uint4 *ring;                 // + this thread

    __device__ __forceinline__ Feed(uint8_t *smem, int rows, int valid_) : n(rows), valid(valid_) {
        ring = reinterpret_cast<uint4 *>(smem) + threadIdx.x;
    }
    __device__ __forceinline__ void tensor(int s, const T *p, long long st) {
        next[s] = here[s] = p;
        step[s] = st;
    }
    __device__ __forceinline__ void issue(int batch) {
        if constexpr (VEC) {
            uint4 *const to = ring + place(batch) * (B * row());
            const int left = n - batch * B;
#pragma unroll
            for (int s = 0; s < S; s++) {
                const T *p = next[s];
#pragma unroll
                for (int k = 0; k < B; k++) {
                    if (k < left)
#pragma unroll
                        for (int q = 0; q < (int)sizeof(T) / 2; q++)
                            cp_async16(to + k * row() + (s * pieces() + q) * threads(),
                                       reinterpret_cast<const uint4 *>(p) + q);
                    p += step[s];
                }
                next[s] = p;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    }
    __device__ __forceinline__ void start() {
#pragma unroll
        for (int t = 0; t < NB - 1; t++) issue(t);
    }
    // batch t is here, batch t + NB - 1 on its way
    __device__ __forceinline__ void turn(int t) {
        issue(t + NB - 1);
        if (VEC) cp_async_wait<NB - 1>();
    }
    // row k of batch t
    __device__ __forceinline__ Raw8<T> get(int t, int k, int s) const {
        if constexpr (VEC) {
            const uint4 *const from = ring + place(t) * (B * row()) + k * row() + s * pieces() * threads();
            Raw8<T> r;
#pragma unroll
            for (int q = 0; q < (int)sizeof(T) / 2; q++) r.q[q] = from[q * threads()];
            return r;
        } else {
            return fetch<T, false>(here[s] + (long long)(t * B + k) * step[s], valid);
        }
    }
};
template <typename T, int S, int B>
constexpr size_t ring_bytes() {
    return (size_t)ring_batches<T>() * B * S * V * sizeof(T) * MAX_T;
}

// Sums over the row lanes of W values per thread (0 from idle ones): entry cv * W + i of the returned array, in
// buf[0..2 W threads).  Where a warp's lanes repeat the vectors evenly: by shuffles, then over the warps.  Else
// one plane per value in shared memory, its rows dealt to as many threads as there are, their parts added in order.
template <int W>
__device__ __forceinline__ const float *fold_rows(float *buf, float *v, const NormArgs &a, const Slice &sl) {
    const int w = a.cvec * W, T = blockDim.x;
    __syncthreads();
    if (32 % a.cvec == 0) {
        for (int o = a.cvec; o < 32; o <<= 1)
#pragma unroll
            for (int i = 0; i < W; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = T >> 5;
        if (lane < a.cvec)
#pragma unroll
            for (int i = 0; i < W; i++) buf[warp * w + lane * W + i] = v[i];
        __syncthreads();
        for (int k = threadIdx.x; k < w; k += T) {
            float s = buf[k];
            for (int q = 1; q < nw; q++) s += buf[q * w + k];
            buf[k] = s;
        }
        __syncthreads();
        return buf;
    }
    const int plane = a.rl * a.cvec;
    if (sl.r < a.rl)
#pragma unroll
        for (int i = 0; i < W; i++) buf[i * plane + threadIdx.x] = v[i];
    __syncthreads();
    float *const out = buf + W * T;
    const int parts = max(1, min(T / w, a.rl));
    for (int t = threadIdx.x; t < parts * w; t += T) {
        const int part = t / w, o = t - part * w, i = o / a.cvec, cv = o - i * a.cvec;
        float s = 0.f;
#pragma unroll 4
        for (int r = part; r < a.rl; r += parts) s += buf[i * plane + r * a.cvec + cv];
        out[parts > 1 ? t : cv * W + i] = s;
    }
    __syncthreads();
    if (parts == 1) return out;
    for (int o = threadIdx.x; o < w; o += T) {
        float s = out[o];
        for (int part = 1; part < parts; part++) s += out[part * w + o];
        const int i = o / a.cvec, cv = o - i * a.cvec;
        buf[cv * W + i] = s;
    }
    __syncthreads();
    return buf;
}
// Sums over each group's `per` consecutive entries, a warp per group; f gives an entry.
template <typename F>
__device__ __forceinline__ void fold_groups(float *gsum, int groups, int per, F f) {
    for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
        float s = 0.f;
        for (int c = threadIdx.x & 31; c < per; c += 32) s += f(g * per + c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if ((threadIdx.x & 31) == 0) gsum[g] = s;
    }
    __syncthreads();
}

// Running statistics of one thread: count, mean, sum of squares around the mean; W of them with one count
// (W = 1: the thread's vector lies in one group; else one per channel).
template <int W>
struct Running {
    float n, mean[W], m2[W];
    // joins a batch of `k` values with mean m and square sum q, k the same for all W
    __device__ __forceinline__ void join(float k, const float *m, const float *q) {
        if (n == 0.f) {
            n = k;
#pragma unroll
            for (int i = 0; i < W; i++) {
                mean[i] = m[i];
                m2[i] = q[i];
            }
            return;
        }
        const float t = n + k, f = k * gs_rcp(t);
#pragma unroll
        for (int i = 0; i < W; i++) {
            const float d = m[i] - mean[i];
            mean[i] = fmaf(d, f, mean[i]);
            m2[i] = fmaf(d * d, n * f, m2[i] + q[i]);
        }
        n = t;
    }
};
// One batch of R rows of a vector, already activated
template <int W, int R>
__device__ __forceinline__ void take(Running<W> &run, const f2 (*u)[V / 2]) {
    float m[W], q[W];
    if (W == 1) {
        f2 s = u[0][0];
#pragma unroll
        for (int k = 1; k < R * V / 2; k++) s = add2(s, u[k / (V / 2)][k % (V / 2)]);
        m[0] = (s.x + s.y) * (1.0f / (R * V));
        f2 t = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < R * V / 2; k++) {
            const f2 d = add2(u[k / (V / 2)][k % (V / 2)], both(-m[0]));
            t = fma2(d, d, t);
        }
        q[0] = t.x + t.y;
        run.join((float)(R * V), m, q);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; i++) {
            f2 s = u[0][i];
#pragma unroll
            for (int k = 1; k < R; k++) s = add2(s, u[k][i]);
            s = mul2(s, both(1.0f / R));
            f2 t = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < R; k++) {
                const f2 d = fma2(s, both(-1.0f), u[k][i]);
                t = fma2(d, d, t);
            }
            m[2 * i % W] = s.x;
            m[(2 * i + 1) % W] = s.y;
            q[2 * i % W] = t.x;
            q[(2 * i + 1) % W] = t.y;
        }
        run.join((float)R, m, q);
    }
}

// Mean and M2 of the slice's groups, W = 1 where a vector lies in one group: emit(group, mean, M2), one lane
// per group.  KEEP: the ring holds all rows, and the activated values
// replace them there.
template <typename T, bool VEC, int PRE, int W, bool KEEP, typename Emit>
__device__ __forceinline__ void slice_stats(const NormArgs &a, const Slice &sl, uint8_t *ring, float *buf, Emit emit) {
    constexpr int R = 2, THREADS = KEEP ? FUSED_T : MAX_T;
    const int groups = sl.cc / a.cpg, per = W == 1 ? a.cpg / V : a.cpg;
    float *gmean = buf + 2 * THREADS * W, *gsum = gmean + a.chunk / a.cpg;
    const Act<PRE> act;
    Running<W> run;
    run.n = 0.f;
#pragma unroll
    for (int i = 0; i < W; i++) run.mean[i] = run.m2[i] = 0.f;
    Feed<T, VEC, 1, R, KEEP> feed(ring, sl.rows(a), sl.valid);
    feed.tensor(0, reinterpret_cast<const T *>(a.x) + sl.b * a.x_img + sl.c + (long long)(sl.lo + sl.r) * a.x_row, a.rl * a.x_row);
    feed.start();
    auto value = [&](int t, int k, f2 *u) {
        unpack8<T>(feed.get(t, k, 0), u);
#pragma unroll
        for (int i = 0; i < V / 2; i++) u[i] = act(u[i]);
        if (KEEP) {
            float4 *to = reinterpret_cast<float4 *>(ring) + threadIdx.x + (t * R + k) * 2 * THREADS;
            to[0] = make_float4(u[0].x, u[0].y, u[1].x, u[1].y);
            to[THREADS] = make_float4(u[2].x, u[2].y, u[3].x, u[3].y);
        }
    };
    int t = 0;
    f2 u[R][V / 2];
    for (; t * R + R <= feed.n; t++) {
        feed.turn(t);
#pragma unroll
        for (int k = 0; k < R; k++) value(t, k, u[k]);
        take<W, R>(run, u);
    }
    feed.turn(t);
    for (int k = 0; t * R + k < feed.n; k++) {
        value(t, k, u[0]);
        take<W, 1>(run, u);
    }
    // the slice's group means, then square sums around them; the first moments correct the means' own rounding
    float v[W], m[W];
#pragma unroll
    for (int i = 0; i < W; i++) v[i] = W == 1 || i < sl.valid ? run.n * run.mean[i] : 0.f;
    const float inv = sl.hi > sl.lo ? 1.0f / ((float)(sl.hi - sl.lo) * (float)a.cpg) : 0.f;
    const float *f = fold_rows<W>(buf, v, a, sl);
    fold_groups(gmean, groups, per, [&](int c) { return f[c] * inv; });
#pragma unroll
    for (int i = 0; i < W; i++) {
        const bool live = W == 1 ? sl.valid > 0 : i < sl.valid;
        m[i] = live && run.n > 0.f ? run.mean[i] - gmean[(sl.cv * W + i) / per] : 0.f;
        v[i] = live ? run.n * m[i] : 0.f;
    }
    f = fold_rows<W>(buf, v, a, sl);
    fold_groups(gsum, groups, per, [&](int c) { return f[c]; });
#pragma unroll
    for (int i = 0; i < W; i++) v[i] = (W == 1 ? sl.valid > 0 : i < sl.valid) ? fmaf(run.n * m[i], m[i], run.m2[i]) : 0.f;
    f = fold_rows<W>(buf, v, a, sl);
    for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
        float q = 0.f;
        for (int c = threadIdx.x & 31; c < per; c += 32) q += f[g * per + c];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
        const float d = gsum[g] * inv;
        if ((threadIdx.x & 31) == 0) emit(g, gmean[g] + d, fmaf(-d, gsum[g], q));
    }
}

// ---- forward, first launch
template <typename T, bool VEC, int PRE, int W>
__global__ void __launch_bounds__(MAX_T, W == 1 ? 3 : 2) k_gn_stats(NormArgs a) {
    extern __shared__ __align__(16) uint8_t dsm[];
    gs_let_follow();
    const Slice sl(a);
    float2 *out = reinterpret_cast<float2 *>(a.part) + ((long long)sl.b * a.G + sl.c0 / a.cpg) * a.splits + sl.s;
    slice_stats<T, VEC, PRE, W, false>(a, sl, dsm, reinterpret_cast<float *>(dsm + ring_bytes<T, 1, 2>()),
                                       [&](int g, float mean, float m2) { out[(long long)g * a.splits] = make_float2(mean, m2); });
}

__device__ __forceinline__ float slice_rows(const NormArgs &a, int s) {
    return (float)max(0, min(a.per, a.rows - s * a.per));
}
// mean and 1 / sqrt(var + eps) of the chunk's groups from the slices' (n, mean, M2), a warp per group: entry s
// of group g is part[g * gs + s * ss]
__device__ __forceinline__ void join_stats(const NormArgs &a, const Slice &sl, const float2 *part, int gs, int ss,
                                           float *mean, float *rstd) {
    const int groups = sl.cc / a.cpg, lane = threadIdx.x & 31;
    const float inv = 1.0f / (float)a.rows;
    for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
        const float2 *p = part + (long long)g * gs;
        const float m0 = p[0].x;
        // weights n_s / n: the mean first, then the square sums around it
        float d = 0.f, q = 0.f;
#pragma unroll 4
        for (int s = lane; s < a.splits; s += 32) d = fmaf(slice_rows(a, s) * inv, p[s * ss].x - m0, d);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        d += m0;
#pragma unroll 4
        for (int s = lane; s < a.splits; s += 32) {
            const float2 e = p[s * ss];
            const float t = e.x - d;
            q += fmaf(slice_rows(a, s) * inv * t, t, e.y * (inv / (float)a.cpg));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
        if (lane == 0) {
            mean[g] = d;
            rstd[g] = 1.0f / sqrtf((q < 0.f ? 0.f : q) + a.eps);
            if (sl.s == 0 && a.stats)
                reinterpret_cast<float2 *>(a.stats)[(long long)sl.b * a.G + sl.c0 / a.cpg + g] = make_float2(d, rstd[g]);
        }
    }
    __syncthreads();
}

// A thread's coefficients of the map: y = act((u + m) k + b), m the negative mean
template <typename T>
struct Map {
    f2 m[V / 2], k[V / 2], b[V / 2];
    __device__ __forceinline__ Map(const NormArgs &a, const Slice &sl, const float *mean, const float *rstd) {
        each_channel(a, sl, [&](int i, int g) {
            const int c = sl.c + min(i, sl.valid - 1);
            at(m, i) = -mean[g];
            at(k, i) = rstd[g] * (a.w ? param<T>(a.w, a.param_f32, c) : 1.f);
            at(b, i) = a.b ? param<T>(a.b, a.param_f32, c) : 0.f;
        });
    }
    __device__ __forceinline__ f2 operator()(f2 u, int i) const { return fma2(add2(u, m[i]), k[i], b[i]); }
};

// ---- forward, second launch: the map
template <typename T, bool VEC, int PRE, int POST>
__global__ void __launch_bounds__(MAX_T, 3) k_gn_map(NormArgs a) {
    constexpr int B = 4;
    extern __shared__ __align__(16) uint8_t dsm[];
    const Slice sl(a);
    float *mean = reinterpret_cast<float *>(dsm + ring_bytes<T, 1, B>()), *rstd = mean + a.chunk / a.cpg;
    // from the end of the slice: L2 holds what the first launch read last
    const int n = sl.rows(a);
    const long long last = sl.lo + sl.r + (long long)(n - 1) * a.rl;
    Feed<T, VEC, 1, B> feed(dsm, n, sl.valid);
    feed.tensor(0, reinterpret_cast<const T *>(a.x) + sl.b * a.x_img + sl.c + last * a.x_row, -a.rl * a.x_row);
    feed.start();  // (x does not come from the first launch)
    gs_wait_leader();
    join_stats(a, sl, reinterpret_cast<const float2 *>(a.part) + ((long long)sl.b * a.G + sl.c0 / a.cpg) * a.splits,
               a.splits, 1, mean, rstd);
    if (n == 0) return;
    const Map<T> map(a, sl, mean, rstd);
    const Act<PRE> pre;
    const Act<POST> post;
    T *y = reinterpret_cast<T *>(a.y) + ((long long)sl.b * a.rows + last) * a.C + sl.c;
    const long long ystep = -(long long)a.rl * a.C;
    auto one = [&](int t, int k) {
        f2 u[V / 2];
        unpack8<T>(feed.get(t, k, 0), u);
#pragma unroll
        for (int i = 0; i < V / 2; i++) u[i] = post(map(pre(u[i]), i));
        store<T, VEC>(y, sl.valid, u);
        y += ystep;
    };
    int t = 0;
    for (; t * B + B <= n; t++) {
        feed.turn(t);
#pragma unroll
        for (int k = 0; k < B; k++) one(t, k);
    }
    feed.turn(t);
    for (int k = 0; t * B + k < n; k++) one(t, k);
}

// writes v to the place of this CTA's shared address p in rank `rank` of the cluster
__device__ __forceinline__ void put(const float2 *p, int rank, float2 v) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(a)
                 : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(v.x), "f"(v.y) : "memory");
}

// ---- forward in one launch: the CTAs of a cluster hold one image's chunk of groups in shared memory,
// activated, in fp32.  Slices are the cluster's ranks; every rank gets all ranks' (mean, M2) and joins them alike.
__host__ __device__ constexpr size_t held_bytes(int rows) { return (size_t)rows * 32 * FUSED_T; }  // [row][half][thread]
template <typename T, int PRE, int POST, int W>
__global__ void __launch_bounds__(FUSED_T, 1) k_gn_fused(NormArgs a) {
    extern __shared__ __align__(16) uint8_t dsm[];
    const Slice sl(a, true);
    const int gmax = a.chunk / a.cpg;
    float *buf = reinterpret_cast<float *>(dsm + held_bytes(a.held)), *mean = buf + 2 * FUSED_T * W + 2 * gmax, *rstd = mean + gmax;
    float2 *all = reinterpret_cast<float2 *>(rstd + gmax);  // [ranks][gmax]
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    slice_stats<T, true, PRE, W, true>(a, sl, dsm, buf,
                                       [&](int g, float m, float m2) { all[sl.s * gmax + g] = make_float2(m, m2); });
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every rank runs: its memory may be written
    for (int t = threadIdx.x; t < gmax * a.splits; t += blockDim.x) {
        const int rank = t / gmax, at = sl.s * gmax + t - rank * gmax;
        if (rank != sl.s && t - rank * gmax < sl.cc / a.cpg) put(all + at, rank, all[at]);
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    join_stats(a, sl, all, 1, gmax, mean, rstd);
    const int n = sl.rows(a);
    if (n == 0) return;
    const Map<T> map(a, sl, mean, rstd);
    const Act<POST> post;
    T *y = reinterpret_cast<T *>(a.y) + ((long long)sl.b * a.rows + sl.lo + sl.r) * a.C + sl.c;
    const float4 *keep = reinterpret_cast<const float4 *>(dsm) + threadIdx.x;
#pragma unroll 2
    for (int k = 0; k < n; k++) {
        const float4 p = keep[2 * k * FUSED_T], q = keep[(2 * k + 1) * FUSED_T];
        f2 u[V / 2] = {{p.x, p.y}, {p.z, p.w}, {q.x, q.y}, {q.z, q.w}};
#pragma unroll
        for (int i = 0; i < V / 2; i++) u[i] = post(map(u[i], i));
        store<T, true>(y + (long long)k * a.rl * a.C, V, u);
    }
}

// A thread's coefficients of the backward: statistics and parameters of its channels.  SLOPE: the first
// activation's slope too, for dx.
template <typename T, int PRE, int POST, bool SLOPE>
struct Grad {
    Act<PRE, SLOPE> pre;
    Act<POST, true> post;
    f2 m[V / 2], rs[V / 2], w[V / 2], b[V / 2];
    __device__ __forceinline__ Grad(const NormArgs &a, const Slice &sl) {
        const float2 *st = reinterpret_cast<const float2 *>(a.stats) + (long long)sl.b * a.G + sl.c0 / a.cpg;
        each_channel(a, sl, [&](int i, int g) {
            const int c = sl.c + min(i, sl.valid - 1);
            at(m, i) = -st[g].x;
            at(rs, i) = st[g].y;
            at(w, i) = a.w ? param<T>(a.w, a.param_f32, c) : 1.f;
            at(b, i) = a.b ? param<T>(a.b, a.param_f32, c) : 0.f;
        });
    }
    // xh and dz of one pair
    __device__ __forceinline__ f2 operator()(f2 x, f2 dy, int i, f2 &xh, f2 &slope) const {
        const f2 u = SLOPE ? pre(x, slope) : pre(x);
        xh = mul2(add2(u, m[i]), rs[i]);
        if (POST == ACT_NONE) return dy;
        f2 s;
        post(fma2(xh, w[i], b[i]), s);
        return mul2(dy, s);
    }
};

// ---- backward, first launch: channel sums of dz and dz xh, and their group sums weighted by w
template <typename T, bool VEC, int PRE, int POST>
__global__ void __launch_bounds__(MAX_T, 3) k_gn_grad_sums(NormArgs a) {
    extern __shared__ __align__(16) uint8_t dsm[];
    gs_let_follow();
    const Slice sl(a);
    const int groups = sl.cc / a.cpg;
    // (the sums fold in the ring's place, drained by then)
    static_assert(ring_bytes<T, 2, 2>() >= 2 * MAX_T * V * sizeof(float), "room to fold");
    float *buf = reinterpret_cast<float *>(dsm), *g0 = reinterpret_cast<float *>(dsm + ring_bytes<T, 2, 2>()),
          *g1 = g0 + a.chunk / a.cpg;
    f2 sz[V / 2], sx[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; i++) sz[i] = sx[i] = both(0.f);
    constexpr int B = 2;
    const int n = sl.rows(a);
    Feed<T, VEC, 2, B> feed(dsm, n, sl.valid);
    feed.tensor(0, reinterpret_cast<const T *>(a.x) + sl.b * a.x_img + sl.c + (long long)(sl.lo + sl.r) * a.x_row, a.rl * a.x_row);
    feed.tensor(1, reinterpret_cast<const T *>(a.dy) + sl.b * a.dy_img + sl.c + (long long)(sl.lo + sl.r) * a.dy_row, a.rl * a.dy_row);
    feed.start();
    if (n > 0) {
        const Grad<T, PRE, POST, false> grad(a, sl);
        auto one = [&](int t, int k) {
            f2 v[V / 2], d[V / 2];
            unpack8<T>(feed.get(t, k, 0), v);
            unpack8<T>(feed.get(t, k, 1), d);
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                f2 xh, none;
                const f2 dz = grad(v[i], d[i], i, xh, none);
                sz[i] = add2(sz[i], dz);
                sx[i] = fma2(dz, xh, sx[i]);
            }
        };
        int t = 0;
        for (; t * B + B <= n; t++) {
            feed.turn(t);
#pragma unroll
            for (int k = 0; k < B; k++) one(t, k);
        }
        feed.turn(t);
        for (int k = 0; t * B + k < n; k++) one(t, k);
    }
    cp_async_wait<0>();
    float2 *cp = reinterpret_cast<float2 *>(a.cpart) + ((long long)sl.b * a.splits + sl.s) * a.C;
    float2 *gp = reinterpret_cast<float2 *>(a.part) + ((long long)sl.b * a.G + sl.c0 / a.cpg) * a.splits + sl.s;
    auto weight = [&](int c) { return a.w ? param<T>(a.w, a.param_f32, sl.c0 + c) : 1.f; };
    float v[V];
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = i < sl.valid ? at(sz, i) : 0.f;
    const float *f = fold_rows<V>(buf, v, a, sl);
    for (int c = threadIdx.x; c < sl.cc; c += blockDim.x) cp[sl.c0 + c].x = f[c];
    fold_groups(g0, groups, a.cpg, [&](int c) { return f[c] * weight(c); });
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = i < sl.valid ? at(sx, i) : 0.f;
    f = fold_rows<V>(buf, v, a, sl);
    for (int c = threadIdx.x; c < sl.cc; c += blockDim.x) cp[sl.c0 + c].y = f[c];
    fold_groups(g1, groups, a.cpg, [&](int c) { return f[c] * weight(c); });
    for (int g = threadIdx.x; g < groups; g += blockDim.x) gp[(long long)g * a.splits] = make_float2(g0[g], g1[g]);
}

// ---- backward, second launch: dx; the blocks after the slices' fold the channel sums into dw and db
template <typename T, bool VEC, int PRE, int POST>
__global__ void __launch_bounds__(MAX_T, 2) k_gn_grad_map(NormArgs a) {
    extern __shared__ __align__(16) uint8_t dsm[];
    float *sm = reinterpret_cast<float *>(dsm + ring_bytes<T, 2, 2>());
    if ((int)blockIdx.x >= a.nslice) {
        gs_wait_leader();
        // 32 channels per block, the (image, split) sums dealt to the warps, joined in order
        float2 *red = reinterpret_cast<float2 *>(sm);
        const int lane = threadIdx.x & 31, nw = blockDim.x >> 5, c = ((int)blockIdx.x - a.nslice) * 32 + lane;
        const float2 *cp = reinterpret_cast<const float2 *>(a.cpart);
        float2 t = make_float2(0.f, 0.f);
        if (c < a.C)
#pragma unroll 8
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
    const Slice sl(a);
    const int groups = sl.cc / a.cpg;
    float *g0 = sm, *g1 = sm + a.chunk / a.cpg;
    // from the end of the slice, as the forward's map
    constexpr int B = 2;
    const int n = sl.rows(a);
    const long long last = sl.lo + sl.r + (long long)(n - 1) * a.rl;
    Feed<T, VEC, 2, B> feed(dsm, n, sl.valid);
    feed.tensor(0, reinterpret_cast<const T *>(a.x) + sl.b * a.x_img + sl.c + last * a.x_row, -a.rl * a.x_row);
    feed.tensor(1, reinterpret_cast<const T *>(a.dy) + sl.b * a.dy_img + sl.c + last * a.dy_row, -a.rl * a.dy_row);
    feed.start();
    gs_wait_leader();
    const float inv = 1.0f / ((float)a.rows * (float)a.cpg);
    for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
        const float2 *p = reinterpret_cast<const float2 *>(a.part) + ((long long)sl.b * a.G + sl.c0 / a.cpg + g) * a.splits;
        float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
        for (int s = threadIdx.x & 31; s < a.splits; s += 32) {
            const float2 e = p[s];
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
    if (n == 0) return;
    const Grad<T, PRE, POST, true> grad(a, sl);
    f2 m0[V / 2], m1[V / 2];
    each_channel(a, sl, [&](int i, int g) {
        at(m0, i) = -g0[g];
        at(m1, i) = -g1[g];
    });
    T *dx = reinterpret_cast<T *>(a.dx) + ((long long)sl.b * a.rows + last) * a.C + sl.c;
    const long long ystep = -(long long)a.rl * a.C;
    auto one = [&](int t, int k) {
        f2 v[V / 2], d[V / 2];
        unpack8<T>(feed.get(t, k, 0), v);
        unpack8<T>(feed.get(t, k, 1), d);
#pragma unroll
        for (int i = 0; i < V / 2; i++) {
            f2 xh, slope;
            const f2 dz = grad(v[i], d[i], i, xh, slope);
            const f2 du = mul2(grad.rs[i], fma2(xh, m1[i], fma2(grad.w[i], dz, m0[i])));
            v[i] = PRE ? mul2(du, slope) : du;
        }
        store<T, VEC>(dx, sl.valid, v);
        dx += ystep;
    };
    int t = 0;
    for (; t * B + B <= n; t++) {
        feed.turn(t);
#pragma unroll
        for (int k = 0; k < B; k++) one(t, k);
    }
    feed.turn(t);
    for (int k = 0; t * B + k < n; k++) one(t, k);
}

// ---- host
int elem_size(int dtype) { return dtype == GS_F32 ? 4 : 2; }

constexpr int SMS = 148;  // of a B200: the split of the work, and with it the workspace, is a matter of sizes alone

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// Slices of equal length (the last may be shorter, none is empty).
void split(NormArgs &a, int want) {
    a.per = std::max(1, (a.rows + want - 1) / want);
    a.splits = std::max(1, (a.rows + a.per - 1) / a.per);
}

// Chunks of whole groups and whole vectors, of at least `want` channels.
void chunks(NormArgs &a, int want) {
    const int unit = a.cpg / gcd(a.cpg, V) * V;
    const int n = (want + unit - 1) / unit * unit;
    a.chunk = n < a.C ? n : a.C;
    a.nchunk = (a.C + a.chunk - 1) / a.chunk;
    a.cvec = (a.chunk + V - 1) / V;
}

// Fills sizes and the split of the work; false for arguments outside the operator's range.
bool plan(const gs_norm_desc *d, NormArgs &a) {
    memset(&a, 0, sizeof(a));
    if (!d || d->B < 0 || d->rows < 0 || d->C < 1 || d->groups < 1 || d->C % d->groups) return false;
    if (d->dtype < GS_F32 || d->dtype > GS_F16 || d->act < GS_ACT_NONE || d->act > GS_ACT_SILU) return false;
    if (d->param_dtype != GS_F32 && d->param_dtype != d->dtype) return false;
    if (!(d->eps >= 0.f) || d->C > GS_NORM_MAX_C || d->rows > GS_NORM_MAX_ROWS) return false;
    a.B = d->B; a.C = d->C; a.G = d->groups; a.cpg = d->C / d->groups;
    a.rows = (int)d->rows;
    a.x_row = d->x_row; a.x_img = d->x_img; a.dy_row = d->dy_row; a.dy_img = d->dy_img;
    a.param_f32 = d->param_dtype == GS_F32;
    a.eps = d->eps;
    // many groups: a block takes whole groups of about 64 channels (128 contiguous bytes a row in 16 bits), so
    // the second launch joins only those groups' sums
    chunks(a, a.G > 32 ? 64 : a.C);
    a.rl = std::max(1, MAX_T / a.cvec);
    // Three blocks per SM, but no fewer than four rows a thread: one wave of the launches that hold three an SM, one
    // and a half of the others (statistics off eight channels a group, the backward's map).  444, 296 and 592
    // slices: 4x384x384x64 44, 52.5, 45.9 us, the training step of 4x192x192x128 78.5, 81.3, 87.4.
    const long long most = std::max<long long>(1, a.rows / (4LL * a.rl));
    const long long want = std::max<long long>(1, 3LL * SMS / std::max<long long>(1, (long long)a.B * a.nchunk));
    split(a, (int)std::min(most, want));
    return (long long)a.B * a.splits * a.nchunk < (1LL << 30);
}

// The one-launch form's split: chunks of whole groups of at least 64 contiguous bytes a row, over a cluster of
// as few CTAs as hold them, or as many (to 8) as find SMs idle.  False where eight CTAs do not hold a chunk
// (clusters of 16 wait for whole GPCs to be free).
bool fused_plan(const gs_norm_desc *d, NormArgs &a) {
    if (a.C % V) return false;
    chunks(a, 64 / elem_size(d->dtype));
    if (a.cvec > FUSED_T) return false;
    a.rl = FUSED_T / a.cvec;
    int n = 1;
    while (n <= 8 && (a.rows + n - 1) / n > a.rl * FUSED_R) n *= 2;
    if (n > 8) return false;
    while (n < 8 && (long long)a.B * a.nchunk * n * 2 <= SMS && a.rows / (2 * n) >= a.rl) n *= 2;
    a.splits = n;
    a.per = (a.rows + n - 1) / n;
    a.rl = std::min(a.rl, a.per);
    a.held = (a.per + a.rl - 1) / a.rl;
    return (long long)a.B * a.splits * a.nchunk < (1LL << 30);
}

size_t al(size_t n) { return (n + 255) & ~(size_t)255; }
size_t part_bytes(const NormArgs &a) { return al((size_t)a.B * a.splits * a.G * 8); }

bool aligned(const void *p, long long row, long long img) {
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
template <typename K>
int launch(K kern, unsigned grid, const NormArgs &a, size_t smem, cudaStream_t s, bool follows, const char *where) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return done(where);
    gs_launch(kern, dim3(grid), threads(a), smem, s, follows, 1, a);
    gs_count_launch(1);
    return done(where);
}

constexpr const char *FWD = "gs_group_norm_act_fwd", *BWD_ = "gs_group_norm_act_bwd";

template <typename T, int PRE, int POST>
int forward_fused(const NormArgs &a, cudaStream_t s) {
    const int W = a.cpg % V == 0 ? 1 : V;
    auto kern = W == 1 ? k_gn_fused<T, PRE, POST, 1> : k_gn_fused<T, PRE, POST, V>;
    const size_t smem = held_bytes(a.held) + ((size_t)2 * FUSED_T * W + (4 + 2 * (size_t)a.splits) * (a.chunk / a.cpg)) * sizeof(float);
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return done(FWD);
    gs_launch(kern, dim3((unsigned)(a.B * a.splits * a.nchunk)), threads(a), smem, s, false, a.splits, a);
    gs_count_launch(1);
    return done(FWD);
}
template <typename T, bool VEC, int PRE, int POST>
int forward(const NormArgs &a, cudaStream_t s) {
    if (a.fused) return forward_fused<T, PRE, POST>(a, s);
    const unsigned grid = (unsigned)(a.B * a.splits * a.nchunk);
    const size_t groups = 2 * (size_t)(a.chunk / a.cpg) * sizeof(float);
    const int W = a.cpg % V == 0 ? 1 : V;
    const int st = launch(W == 1 ? k_gn_stats<T, VEC, PRE, 1> : k_gn_stats<T, VEC, PRE, V>, grid, a,
                          ring_bytes<T, 1, 2>() + 2 * MAX_T * W * sizeof(float) + groups, s, false, FWD);
    return st != GS_OK ? st : launch(k_gn_map<T, VEC, PRE, POST>, grid, a, ring_bytes<T, 1, 4>() + groups, s, true, FWD);
}
template <typename T, bool VEC, int PRE, int POST>
int backward(const NormArgs &a, cudaStream_t s) {
    const unsigned grid = (unsigned)(a.B * a.splits * a.nchunk), fold = a.dw || a.db ? (a.C + 31) / 32 : 0;
    const size_t groups = 2 * (size_t)(a.chunk / a.cpg) * sizeof(float), ring = ring_bytes<T, 2, 2>();
    if (a.nslice + fold == 0) return GS_OK;
    const int st = launch(k_gn_grad_sums<T, VEC, PRE, POST>, grid, a, ring + groups, s, false, BWD_);
    return st != GS_OK ? st
                       : launch(k_gn_grad_map<T, VEC, PRE, POST>, a.nslice + fold, a,
                                ring + std::max(groups, MAX_T * sizeof(float2)), s, true, BWD_);
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
    const bool vec = aligned(x, a.x_row, a.x_img) && aligned(y, a.C, 0);
    NormArgs f = a;
    if (vec && fused_plan(d, f)) {
        a = f;
        a.fused = 1;
    }
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
    // (whole vectors of channels too: without dx no tightly packed row says so)
    const bool vec = a.C % V == 0 && aligned(x, a.x_row, a.x_img) && aligned(dy, a.dy_row, a.dy_img) &&
                     (!dx || aligned(dx, a.C, 0));
    return by_type<true>(d, a, vec, (cudaStream_t)stream);
}
