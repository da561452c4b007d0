// gs_linear.cu -- linear layer with bias, activation and residual, forward and backward (sm_100a).
//
//   z = x W^T + b,  y = act(z) + residual        x [M][K], W [N][K], y [M][N]
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz,  dresidual = dy
//
// All three products run in one kernel, D[i][j] = sum_k A(i, k) B(j, k) on tcgen05.mma (kind::f16, fp32
// accumulators in TMEM); an operand is read as it lies in memory, with k adjacent (K-major: x and W of the
// forward, dz of dx) or with i / j adjacent (MN-major: W of dx, dz and x of dW), so nothing is transposed.
// fp32 operands enter as three bf16 terms (x = h + m + l, exact to 2^-24 of x) and a product as the six of
// the nine term products that reach 2^-24: the same kernel runs over six times the k-blocks.
//
// The forward keeps, for the backward, the activation's slope instead of z: the epilogue has its parts at
// hand and the backward needs no activation.  It is kept in fp32: in 16 bits either the small slopes of units
// far below zero or those near one lose bits.  dz enters its products in two terms of the operand type, dz = hi + lo
// (rounding it once would add as much error as rounding the result does); db sums the unrounded values.  A training
// step of 36864x256->1024 bf16 takes 243 us for it (169 with 16-bit slopes and dz in one term).
//
// Sums over a long k with few output tiles are split along k over the SMs; the parts go to the workspace
// in fp32 and a second kernel adds them in order (the same bits every time) and applies the epilogue.  What the
// parts of one product take there is bounded: a forward or dx runs over panels of rows, dW over groups of parts
// whose sum so far is kept in the first part's place.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "../../include/gsplat_b200.h"
#include "gs_act.cuh"
#include "gs_prof.cuh"
#include "gs_tc.cuh"

void gs_set_last_error(const char *msg);

using namespace gs_tc;

namespace {

constexpr int SMS = 148;  // of a B200: tiles, splits and the workspace are a matter of sizes alone
constexpr int BM = 128, BK = 64;

struct GemmArgs {
    long long I;          // rows of D
    int J;                // columns of D
    int kb, npair;        // k-blocks of 64 per term product, term products: 1, 2 (A in two terms), 6 (fp32)
    int a_mn, b_mn;       // operand has i / j adjacent instead of k
    int f16;              // operands fp16 (else bf16)
    int splits;           // > 1: parts of the k sum, raw fp32
    int first, nparts, slot;  // of them the launch's: the first, their number, the place of the first
    int tiles_i, tiles_j;
    // epilogue
    int out_f16;          // 16-bit output type
    int out_tma, res_tma; // whole 16-byte rows: TMA boxes, else element by element
    const void *bias, *residual;
    void *out;
    float *slope;
    long long ldr;
    int *wait_error;      // host word for the code of a bounded wait that gives up
};

// term products, small ones first: (a term, b term), 0 = high; the six of fp32, then the two of A in two terms
// fp16 has no exponents below its subnormals: lo is kept times 2^LO_BITS (at most 2^4 2^11 for the largest dz) and
// its sum scaled back when the products with hi begin.  Nor above 65504, which dz passes by the slope's 1.13: both terms
// are of dz / 2, and the epilogue doubles the sum.
constexpr int LO_BITS = 11;
__constant__ const unsigned char PAIR_A[8] = {2, 0, 1, 1, 0, 0, 1, 0}, PAIR_B[8] = {0, 2, 1, 0, 1, 0, 0, 0};

// What an epilogue does with z = acc + bias: nothing, an activation, or an activation and its slope.
constexpr int EPI_WARPS = 16, UNIT = 2048, GEMM_THREADS = 64 + 32 * EPI_WARPS;
enum { EPI_NONE = 0, EPI_GELU = 1, EPI_SILU = 2, EPI_GELU_SLOPE = 3, EPI_SILU_SLOPE = 4 };

// Persistent and warp-specialised, one CTA per SM.  Work item = a tile of D times a k split; CTAs (or pairs)
// stride over the items, neighbours on neighbouring columns of the same rows (A from L2).
//   warp 0   TMA producer: A and B k-blocks into a STAGES-deep ring of 128-byte-swizzled tiles
//   warp 1   TMEM owner, MMA issuer; accumulators double-buffered, so the epilogue runs under the next item
//   warps 2..17 epilogue: quarter warp % 4 of the CTA's 128 rows; a quarter (BN = 256) or half (128) of the
//            columns, and every second (128) or fourth (64) item.  16 warps, because two per scheduler left
//            it idle 60 % of the time.  A unit is 32 rows x 64 bytes of the output, staged in shared memory in the
//            64-byte swizzle (a thread writes its row without bank conflicts) and moved by TMA; the residual
//            comes by TMA into the same place, a unit ahead, and is added in registers before the only rounding.
// PAIR: two CTAs share a 256 x 256 tile (cta_group::2): each loads its 128 rows of A and half of B's rows, so an
// output costs half of the L2 reads and half of the issued MMAs of a 128 x 128 tile (16384x4096->4096 with a
// residual: 387 us, 1420 TFLOP/s, against 569).  The leader issues all MMAs.
// Bound by: long sums, the tensor cores at the clock that the power limit leaves (busy 83 % of the time at 1.5 GHz);
// short ones, the epilogue's latency: 36864x128->512 with GELU takes 23.3 us where its bytes take 7.3 with half of the
// issue slots used (20 instructions an output, 11 of them GELU's) and no pipe above 42 %, its warps waiting in turn
// for accumulators, shared memory and their own chains.
// Every wait is bounded; one that gives up writes its code to wait_error and raises the CTA's abort flag.
template <int BN, bool PAIR, bool OUT32, int EPI>
struct Shape {
    static constexpr int BROWS = PAIR ? BN / 2 : BN;  // rows of B in this CTA
    static constexpr uint32_t A_BYTES = BM * BK * 2, B_BYTES = BROWS * BK * 2, STAGE = A_BYTES + B_BYTES;
    static constexpr int CS = BN / 64;                // warps sharing a row quarter's columns
    static constexpr int PAR = 4 / CS;                // groups of warps taking turns at the items
    static constexpr int NBUF = PAR > 2 ? PAR : 2;    // accumulators
    static constexpr int EC = OUT32 ? 16 : 32;        // columns of a unit
    static constexpr int UNITS = 64 / EC;
    static constexpr bool SLOPE = EPI >= EPI_GELU_SLOPE;
    static constexpr int SLOPES = SLOPE ? EC / 16 : 0;       // 64-byte rows of fp32 hold 16 slopes
    static constexpr uint32_t SLOTS = (2 + SLOPES) * UNIT;   // per epilogue warp: two for outputs and residuals
    static constexpr int STAGES = (229376 - EPI_WARPS * SLOTS) / STAGE;  // 3 to 6
    static constexpr size_t SMEM = 1024 + STAGES * STAGE + EPI_WARPS * SLOTS;
    static constexpr int TILE_I = PAIR ? 2 * BM : BM;
};

struct Pipe {  // one CTA's barriers
    uint64_t full[6], empty[6], tfull[4], tempty[4], mdone, rbar[EPI_WARPS][2];
    uint32_t tmem_base;
    volatile int abort_flag;
    int issued, consumed;
    __align__(16) float bias[EPI_WARPS][16];  // read as float4
};

// row tile, column tile, part (counted from the launch's first) of an item
struct Item {
    int i, j, s;
    __device__ __forceinline__ Item(const GemmArgs &a, int item) {
        j = item % a.tiles_j;
        item /= a.tiles_j;
        i = item % a.tiles_i;
        s = item / a.tiles_i;
    }
    // its k-blocks, and how many it multiplies over all term products
    __device__ __forceinline__ int from(const GemmArgs &a) const { return (int)((long long)a.kb * (a.first + s) / a.splits); }
    __device__ __forceinline__ int to(const GemmArgs &a) const { return (int)((long long)a.kb * (a.first + s + 1) / a.splits); }
    __device__ __forceinline__ int blocks(const GemmArgs &a) const { return (to(a) - from(a)) * a.npair; }
};

template <int BN, bool PAIR, bool OUT32, int EPI, bool LO>
__device__ __forceinline__ void epilogue(const GemmArgs &a, Pipe &p, uint8_t *ring_end, const CUtensorMap *tmO,
                                         const CUtensorMap *tmS, const CUtensorMap *tmR, int first, int stride, int n_items,
                                         int rank) {
    using S = Shape<BN, PAIR, OUT32, EPI>;
    constexpr int EC = S::EC;
    constexpr bool SLOPE = S::SLOPE;
    constexpr int ACT = EPI == EPI_NONE ? ACT_NONE : EPI == EPI_GELU || EPI == EPI_GELU_SLOPE ? ACT_GELU : ACT_SILU;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = warp - 2, q = warp & 3;
    const int part = (e >> 2) % S::CS, turn = (e >> 2) / S::CS;
    uint8_t *const slots = ring_end + e * S::SLOTS, *const slo = slots + 2 * UNIT;
    const uint32_t tbase = p.tmem_base + ((uint32_t)(q * 32) << 16);
    const bool has_res = a.residual != nullptr, res_tma = has_res && a.res_tma;
    const Act<ACT, SLOPE> act;
    const int step = S::PAR * stride;
    int item = first + turn * stride, tc = turn, use = 0;

    // byte b of row r in a unit: rows of 64 bytes, 16-byte chunks exchanged by the 64-byte swizzle
    auto swizzled = [](int r, int b) { return r * 64 + (((b >> 4) ^ ((r >> 1) & 3)) << 4) + (b & 15); };
    auto place_of = [&](int r, int c) { return swizzled(r, c * (OUT32 ? 4 : 2)); };
    auto place = [&](int it, int u, int &col0, long long &row0) {
        const Item t(a, it);
        col0 = t.j * BN + part * 64 + u * EC;
        row0 = (long long)t.i * S::TILE_I + rank * BM + q * 32;
        return col0 < a.J && row0 < a.I;
    };
    // the residual of the first live unit from (it, u) on goes to slot s
    auto prefetch = [&](int it, int u, int s) {
        int col0;
        long long row0;
        for (; it < n_items; it += step, u = 0)
            for (; u < S::UNITS; u++)
                if (place(it, u, col0, row0)) {
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&p.rbar[e][s], UNIT);
                        tma_load_3d(slots + s * UNIT, tmR, &p.rbar[e][s], col0, (int)row0, 0);
                    }
                    return true;
                }
        return false;
    };
    bool pending = res_tma && prefetch(item, 0, 0);  // a residual is on its way to the next unit's place
    // bias of this warp's 64 columns of an item, two a lane, loaded an item ahead
    float ahead[2] = {0.f, 0.f};
    auto load_bias = [&](int it) {
        if (!a.bias || it >= n_items) return;
        const int c = Item(a, it).j * BN + part * 64 + lane;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int cc = c + 32 * k;
            ahead[k] = cc >= a.J   ? 0.f
                       : OUT32     ? reinterpret_cast<const float *>(a.bias)[cc]
                       : a.out_f16 ? to_f32(reinterpret_cast<const __half *>(a.bias)[cc])
                                   : to_f32(reinterpret_cast<const __nv_bfloat16 *>(a.bias)[cc]);
        }
    };
    load_bias(item);
    bool dead = false;
    for (; item < n_items && !dead; item += step, tc += S::PAR) {
        const int buf = tc % S::NBUF;
        const float bias[2] = {ahead[0], ahead[1]};
        load_bias(item + step);
        const Item tile(a, item);
        const int sp = a.slot + tile.s, base = tile.j * BN + part * 64;
        const long long row0 = (long long)tile.i * S::TILE_I + rank * BM + q * 32;
#pragma unroll 1
        for (int u = 0; u < S::UNITS && !dead; u++) {
            const int col0 = base + u * EC;
            const bool live = col0 < a.J && row0 < a.I;
            const int sl = use & 1;
            uint8_t *const out = slots + sl * UNIT;
            if (live) {
                // the slots this unit writes are no longer read by their stores
                if (lane == 0) {
                    if (SLOPE) bulk_wait_read<0>();
                    else bulk_wait_read<1>();
                }
                __syncwarp();
                if (has_res && !res_tma) {
                    for (int r = lane / EC; r < 32 && row0 + r < a.I; r += 32 / EC)
                        if (const int c = lane % EC; col0 + c < a.J) {
                                const long long at = (row0 + r) * a.ldr + col0 + c;
                                uint8_t *d = out + place_of(r, c);
                                if (OUT32) *reinterpret_cast<float *>(d) = reinterpret_cast<const float *>(a.residual)[at];
                                else *reinterpret_cast<uint16_t *>(d) = reinterpret_cast<const uint16_t *>(a.residual)[at];
                            }
                    __syncwarp();
                }
            }
            if (u == 0) {
                if (!mbar_wait_or_abort(&p.tfull[buf], (tc / S::NBUF) & 1, &p.abort_flag, a.wait_error, 5)) dead = true;
                tc_fence_after();
            }
            if (live && pending) {
                // (after an abort too: the copy lands in this CTA's shared memory)
                if (!mbar_wait(&p.rbar[e][sl], (use >> 1) & 1, a.wait_error, 6)) {
                    p.abort_flag = 1;
                    dead = true;
                }
                pending = false;
            }
            // 16 columns at a time
#pragma unroll
            for (int h = 0; h < EC / 16; h++) {
                f2 v[8];
                if (live && !dead) {
                    uint32_t r[16];
                    tmem_issue16(tbase + (uint32_t)(buf * BN + part * 64 + u * EC + 16 * h), r);
                    __syncwarp();
                    // columns 16 k.. of the 64: half of the lanes hold them
                    const int k = u * (EC / 16) + h;
                    if (lane >> 4 == (k & 1)) p.bias[e][lane & 15] = k < 2 ? bias[0] : bias[1];
                    __syncwarp();
                    tmem_wait16(r);
                    const float4 *b = reinterpret_cast<const float4 *>(p.bias[e]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float4 f = b[i];
                        v[2 * i] = add2({__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1])}, {f.x, f.y});
                        v[2 * i + 1] = add2({__uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3])}, {f.z, f.w});
                    }
                }
                if (LO && live && !dead)
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = add2(v[i], v[i]);
                if (u == S::UNITS - 1 && h == EC / 16 - 1) {  // this warp's part of the accumulator is drained
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (PAIR && rank) mbar_arrive_cluster(in_rank(&p.tempty[buf], 0));
                        else mbar_arrive(&p.tempty[buf]);
                    }
                }
                if (!live || dead) continue;
                // 16 bytes of a row: chunk c of the unit
                auto chunk = [&](uint8_t *base, int c) {
                    return reinterpret_cast<uint4 *>(base + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
                };
                if (SLOPE) {
                    f2 s[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = act(v[i], s[i]);
#pragma unroll
                    for (int i = 0; i < 4; i++) *chunk(slo + h * UNIT, i) = pack16<float>(s + 2 * i);
                } else if (ACT != ACT_NONE) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = act(v[i]);
                }
                if (OUT32) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint4 *c = chunk(out, i);
                        if (has_res) {
                            f2 f[2];
                            unpack16<float>(*c, f);
                            v[2 * i] = add2(v[2 * i], f[0]);
                            v[2 * i + 1] = add2(v[2 * i + 1], f[1]);
                        }
                        *c = pack16<float>(v + 2 * i);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        uint4 *c = chunk(out, 2 * h + i);
                        if (has_res) {
                            f2 f[4];
                            if (a.out_f16) unpack16<__half>(*c, f);
                            else unpack16<__nv_bfloat16>(*c, f);
#pragma unroll
                            for (int k = 0; k < 4; k++) v[4 * i + k] = add2(v[4 * i + k], f[k]);
                        }
                        *c = a.out_f16 ? pack16<__half>(v + 4 * i) : pack16<__nv_bfloat16>(v + 4 * i);
                    }
                }
            }
            if (!live || dead) continue;
            fence_proxy_async();
            __syncwarp();
            if (res_tma) {
                if (lane == 0) bulk_wait_read<0>();  // the other slot's store, a unit ago
                pending = prefetch(item, u + 1, (use + 1) & 1);
            }
            if (a.out_tma) {
                if (lane == 0) {
                    tma_store_3d(tmO, out, col0, (int)row0, sp);
#pragma unroll
                    for (int h = 0; h < S::SLOPES; h++)
                        if (col0 + 16 * h < a.J) tma_store_3d(tmS, slo + h * UNIT, col0 + 16 * h, (int)row0, 0);
                    bulk_commit();
                }
            } else {
                for (int r = lane / EC; r < 32 && row0 + r < a.I; r += 32 / EC)
                    if (const int c = lane % EC; col0 + c < a.J) {
                        const long long at = (row0 + r) * a.J + col0 + c;
                        const int off = place_of(r, c);
                        if (OUT32) reinterpret_cast<float *>(a.out)[at] = *reinterpret_cast<const float *>(out + off);
                        else reinterpret_cast<uint16_t *>(a.out)[at] = *reinterpret_cast<const uint16_t *>(out + off);
                        if (SLOPE)
                            a.slope[at] = *reinterpret_cast<const float *>(slo + (c >> 4) * UNIT + swizzled(r, (c & 15) * 4));
                    }
                fence_proxy_async();  // the next residual's copy overwrites what was just read
                __syncwarp();
            }
            use++;
        }
    }
    if (pending) mbar_wait(&p.rbar[e][use & 1], (use >> 1) & 1, a.wait_error, 8);
    if (lane == 0) bulk_wait<0>();
    __syncwarp();
}

// LO: fp16's dz in two terms, the first scaled (a kernel of its own: the test for it in every k-block cost 5 % of
// 16384x4096->4096, 382 us without and 404 with)
template <int BN, bool PAIR, bool OUT32, int EPI, bool LO>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
    k_gemm(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
           const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmS,
           const __grid_constant__ CUtensorMap tmR, const GemmArgs a) {
    using S = Shape<BN, PAIR, OUT32, EPI>;
    constexpr int STAGES = S::STAGES;
    extern __shared__ uint8_t dsmem[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(16) Pipe p;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)cluster_rank() : 0;
    const int first = PAIR ? blockIdx.x / 2 : blockIdx.x, stride = PAIR ? gridDim.x / 2 : gridDim.x;
    const int n_items = a.tiles_i * a.tiles_j * a.nparts;

    if (warp == 1) {
        if (PAIR) {
            tmem_alloc_pair(&p.tmem_base, S::NBUF * BN);
        } else {
            tmem_alloc(&p.tmem_base, S::NBUF * BN);
            tmem_relinquish();
        }
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&p.full[s], 1);
            mbar_init(&p.empty[s], 1);
        }
        for (int j = 0; j < S::NBUF; j++) {
            mbar_init(&p.tfull[j], 1);
            mbar_init(&p.tempty[j], 4 * S::CS * (PAIR ? 2 : 1));
        }
        for (int w = 0; w < EPI_WARPS; w++)
            for (int j = 0; j < 2; j++) mbar_init(&p.rbar[w][j], 1);
        mbar_init(&p.mdone, 1);
        p.abort_flag = 0;
        p.issued = 0;
        p.consumed = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmA);
        prefetch_tensormap(&tmB);
    }
    gs_let_follow();
    gs_wait_leader();  // operands and residents of the workspace come from the launch before
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_arrive_wait();  // both CTAs' barriers exist
    tc_fence_after();
    const uint32_t tbase = p.tmem_base;

    // (these two loops run in one thread each, and an instruction of theirs costs a few cycles: a stage's place,
    // phase and descriptors are stepped, not computed)
    if (warp == 0) {
        if (lane == 0) {
            int it = 0, st = 0, parity = 1;  // of the ring's previous round; the first finds it complete
            for (int item = first; item < n_items && !p.abort_flag; item += stride) {
                const Item t(a, item);
                const int j0 = t.j * BN + (PAIR ? rank * S::BROWS : 0), i0 = t.i * S::TILE_I + rank * BM;
                const int k0 = t.from(a) * BK, k1 = t.to(a) * BK;
                int kk = k0, pr = a.npair == 2 ? 6 : 0, left = t.blocks(a);
                int ta = a.npair > 1 ? PAIR_A[pr] : 0, tb = a.npair > 1 ? PAIR_B[pr] : 0;
                for (; left > 0; left--, it++) {
                    if (!mbar_wait_or_abort(&p.empty[st], parity, &p.abort_flag, a.wait_error, 1)) break;
                    uint8_t *sa = smem + st * S::STAGE, *sb = sa + S::A_BYTES;
                    // both CTAs' copies complete on the leader's barrier
                    if (rank == 0) mbar_arrive_expect_tx(&p.full[st], S::STAGE * (PAIR ? 2 : 1));
                    const uint32_t bar = PAIR ? in_rank(&p.full[st], 0) : 0;
                    auto load = [&](uint8_t *dst, const CUtensorMap *tm, int c0, int c1, int c2) {
                        if (PAIR) tma_load_3d_pair(dst, tm, bar, c0, c1, c2);
                        else tma_load_3d(dst, tm, &p.full[st], c0, c1, c2);
                    };
                    if (a.a_mn) {
#pragma unroll
                        for (int c = 0; c < BM / 64; c++) load(sa + c * 64 * 128, &tmA, i0 + 64 * c, kk, ta);
                    } else {
                        load(sa, &tmA, kk, i0, ta);
                    }
                    if (a.b_mn) {
#pragma unroll
                        for (int c = 0; c < S::BROWS / 64; c++) load(sb + c * 64 * 128, &tmB, j0 + 64 * c, kk, tb);
                    } else {
                        load(sb, &tmB, kk, j0, tb);
                    }
                    p.issued = it + 1;
                    if (++st == STAGES) {
                        st = 0;
                        parity ^= 1;
                    }
                    kk += BK;
                    if (kk == k1 && left > 1) {  // the next term product
                        kk = k0;
                        pr++;
                        ta = PAIR_A[pr];
                        tb = PAIR_B[pr];
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t fmt = a.f16 ? 0u : 1u;
            const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a.a_mn << 15) |
                                   ((uint32_t)a.b_mn << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(S::TILE_I >> 4) << 24);
            // per 16 of k: 32 bytes inside the swizzled row (K-major), two 8-row groups (MN-major); in a
            // descriptor's units of 16 bytes, whose low word holds the address
            const uint64_t stepA = a.a_mn ? 128u : 2u, stepB = a.b_mn ? 128u : 2u;
            const uint32_t s0 = smem_u32(smem);
            const uint64_t descA = a.a_mn ? sdesc_mn(s0, 8192, 1024) : sdesc(s0, 1024, 2);
            const uint64_t descB = a.b_mn ? sdesc_mn(s0 + S::A_BYTES, 8192, 1024) : sdesc(s0 + S::A_BYTES, 1024, 2);
            int it = 0, tc = 0, st = 0, parity = 0;
            for (int item = first; item < n_items && !p.abort_flag; item += stride, tc++) {
                int left = Item(a, item).blocks(a);
                const int hi = left / 2;  // LO: k-blocks left when hi follows lo
                const int buf = tc % S::NBUF;
                if (tc >= S::NBUF && !mbar_wait_or_abort(&p.tempty[buf], (tc / S::NBUF - 1) & 1, &p.abort_flag,
                                                         a.wait_error, 2))
                    break;
                tc_fence_after();
                const uint32_t dcol = tbase + (uint32_t)buf * BN;
                bool ok = true;
                uint32_t more = 0;
                for (; left > 0; left--, it++) {
                    if (!mbar_wait_or_abort(&p.full[st], parity, &p.abort_flag, a.wait_error, 3)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    uint64_t ad = descA + (uint32_t)st * (S::STAGE >> 4), bd = descB + (uint32_t)st * (S::STAGE >> 4);
#pragma unroll
                    for (int q = 0; q < BK / 16; q++) {
                        if (LO && q == 0 && left == hi) mma_scaled<PAIR ? 2 : 1, LO_BITS>(dcol, ad, bd, idesc);
                        else if (PAIR) mma_pair(dcol, ad, bd, idesc, more);
                        else mma_bf16(dcol, ad, bd, idesc, more);
                        more = 1;
                        ad += stepA;
                        bd += stepB;
                    }
                    if (PAIR) mma_commit_pair(&p.empty[st]);
                    else mma_commit(&p.empty[st]);
                    p.consumed = it + 1;
                    if (++st == STAGES) {
                        st = 0;
                        parity ^= 1;
                    }
                }
                if (!ok) break;
                if (PAIR) mma_commit_pair(&p.tfull[buf]);
                else mma_commit(&p.tfull[buf]);
            }
            // all MMAs of this CTA or pair (also those of an aborted item) have finished once mdone flips
            if (PAIR) mma_commit_pair(&p.mdone);
            else mma_commit(&p.mdone);
            mbar_wait(&p.mdone, 0, a.wait_error, 4);
        }
    } else {
        epilogue<BN, PAIR, OUT32, EPI, LO>(a, p, smem + STAGES * S::STAGE, &tmO, &tmS, &tmR, first, stride, n_items, rank);
    }

    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_arrive_wait();  // no CTA leaves while its peer's copies, MMAs or arrivals may reach it
    if (p.abort_flag && threadIdx.x == 0 && rank == 0)
        // copies that were issued but never consumed still land in shared memory: wait for them
        for (int j = p.consumed; j < p.issued; j++) mbar_wait(&p.full[j % STAGES], (j / STAGES) & 1, a.wait_error, 7);
    __syncthreads();
    if (PAIR) cluster_arrive_wait();
    tc_fence_after();
    if (warp == 1) {
        if (PAIR) tmem_dealloc_pair(tbase, S::NBUF * BN);
        else tmem_dealloc(tbase, S::NBUF * BN);
    }
}

// ---- operands that TMA cannot read in place (rows not on 16 bytes, fp32): rows padded to a multiple of eight
// elements, fp32 as three bf16 terms
struct PrepJob {
    const void *src;
    void *dst;
    long long rows, ld;  // source row stride
    int cols, ldp;       // destination row stride
};
__device__ __forceinline__ void split3(float x, float &h, float &m, float &l) {
    h = __bfloat162float(__float2bfloat16_rn(x));
    const float r = x - h;
    m = __bfloat162float(__float2bfloat16_rn(r));
    l = r - m;
}
// The same where a head would be infinite.  What lies beyond bf16's largest number has that for its head.  An infinity
// is in the last term alone, which meets only the other operand's head (0 where the value is 0, or infinite itself):
// in the first it would meet that operand's lower terms too, zeros and either sign, and give NaN.
__device__ __forceinline__ void split3_large(float x, float &h, float &m, float &l) {
    constexpr float MOST = 3.3895313892515355e38f;  // (2 - 2^-7) 2^127
    const bool inf = fabsf(x) > 3.4028234e38f;
    h = inf ? 0.f : fabsf(x) > MOST ? copysignf(MOST, x) : __bfloat162float(__float2bfloat16_rn(x));
    m = inf ? 0.f : __bfloat162float(__float2bfloat16_rn(x - h));
    l = x - h - m;
}
__device__ __forceinline__ void store_terms(const f2 *v, __nv_bfloat16 *dst, long long term_stride) {
    f2 h[4], m[4], l[4];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        split3(at(v, i), at(h, i), at(m, i), at(l, i));
        most = fmaxf(most, fabsf(at(h, i)));
    }
    if (most > 3.4028234e38f) {  // (one test for the vector: it is not the common case)
#pragma unroll
        for (int i = 0; i < 8; i++) split3_large(at(v, i), at(h, i), at(m, i), at(l, i));
    }
    *reinterpret_cast<uint4 *>(dst) = pack16<__nv_bfloat16>(h);
    *reinterpret_cast<uint4 *>(dst + term_stride) = pack16<__nv_bfloat16>(m);
    *reinterpret_cast<uint4 *>(dst + 2 * term_stride) = pack16<__nv_bfloat16>(l);
}
template <typename T>
__device__ __forceinline__ void prep_operand(const PrepJob &j, int block, int blocks) {
    const int nv = j.ldp / 8;
    const long long n = j.rows * nv;
    for (long long t = block * 256LL + threadIdx.x; t < n; t += blocks * 256LL) {
        const long long r = t / nv;
        const int c = (int)(t - r * nv) * 8;
        const T *p = reinterpret_cast<const T *>(j.src) + r * j.ld + c;
        if (sizeof(T) == 4) {
            f2 v[4];
#pragma unroll
            for (int i = 0; i < 8; i++) at(v, i) = c + i < j.cols ? to_f32(p[i]) : 0.f;
            store_terms(v, reinterpret_cast<__nv_bfloat16 *>(j.dst) + r * j.ldp + c, j.rows * j.ldp);
        } else {
            uint32_t w[4];
            const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
            for (int i = 0; i < 4; i++)
                w[i] = (c + 2 * i < j.cols ? h[2 * i] : 0u) | (c + 2 * i + 1 < j.cols ? (uint32_t)h[2 * i + 1] << 16 : 0u);
            *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(j.dst) + r * j.ldp + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}
// the operands of one call that need it, x and W
struct PrepJobs {
    PrepJob job[2];
    int n, blocks;
};
template <typename T>
__global__ void __launch_bounds__(256) k_prep_operands(const __grid_constant__ PrepJobs p) {
    gs_let_follow();
    prep_operand<T>(p.job[blockIdx.y], blockIdx.x, gridDim.x);
}

// ---- dz = dy slope as an operand (dz NULL: not written, dy serves), and its column sums per block of rows.
// Blocks from `rows` on prepare x and W for the backward's products: a launch less.
struct DzArgs {
    const void *dy;
    const float *slope;
    void *dz;
    float *colsum;  // [blocks][N], or NULL
    long long M, ldy;
    int N, ldp, cvec, rl;  // vectors of eight columns per block, row lanes
    int rows;              // blocks over the rows
    int terms;             // of dz in 16-bit types
    PrepJobs prep;
};
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_dz(const __grid_constant__ DzArgs a) {
    __shared__ float buf[256 * 8];
    gs_let_follow();
    if ((int)blockIdx.x >= a.rows) {
        for (int k = blockIdx.y; k < a.prep.n; k += gridDim.y) prep_operand<T>(a.prep.job[k], blockIdx.x - a.rows, a.prep.blocks);
        return;
    }
    const int r = threadIdx.x / a.cvec, cv = threadIdx.x - r * a.cvec;
    const int c = (blockIdx.y * a.cvec + cv) * 8;
    const bool live = r < a.rl && c < a.ldp;
    const long long lo = a.M * blockIdx.x / a.rows, hi = a.M * (blockIdx.x + 1LL) / a.rows;
    const T *dy = reinterpret_cast<const T *>(a.dy) + c;
    const float *slope = a.slope + c;
    f2 s[4] = {both(0.f), both(0.f), both(0.f), both(0.f)};
    // dy and its slope g, in row m
    auto one = [&](long long m, const Raw8<T> &d, const Raw8<float> &g) {
        f2 v[4];
        unpack8<T>(d, v);
        if (a.slope) {
            f2 f[4];
            unpack8<float>(g, f);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = mul2(v[i], f[i]);  // (rounded: db's bits do not depend on dz being written)
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = add2(s[i], v[i]);
        if (a.dz) {
            if (sizeof(T) == 4)
                store_terms(v, reinterpret_cast<__nv_bfloat16 *>(a.dz) + m * a.ldp + c, a.M * a.ldp);
            else {
                constexpr bool HALF = std::is_same_v<T, __half>;
                if (HALF && a.terms == 2)
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = mul2(v[i], both(0.5f));
                Raw8<T> *to = reinterpret_cast<Raw8<T> *>(reinterpret_cast<T *>(a.dz) + m * a.ldp + c);
                const Raw8<T> high = pack8<T>(v);
                *to = high;
                if (a.terms == 2) {  // lo: what the first term leaves; nothing of an infinity or NaN
                    f2 h[4];
                    unpack8<T>(high, h);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        constexpr float scale = HALF ? (float)(1 << LO_BITS) : 1.f;
                        at(v, i) = fabsf(at(h, i)) <= 3.4028234e38f ? (at(v, i) - at(h, i)) * scale : 0.f;
                    }
                    *reinterpret_cast<Raw8<T> *>(reinterpret_cast<T *>(to) + a.M * a.ldp) = pack8<T>(v);
                }
            }
        }
    };
    auto fetch = [&](const auto *p, auto &o) {
        using E = std::decay_t<decltype(*p)>;
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(E) / 2; k++) o.q[k] = __ldcs(reinterpret_cast<const uint4 *>(p) + k);  // read once
        } else {
            union {
                Raw8<E> q;
                E e[8];
            } u;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c + i < a.N) u.e[i] = p[i];
                else from_f32(0.f, u.e[i]);
            o = u.q;
        }
    };
    if (live) {
        long long m = lo + r;
        constexpr int R = 4;  // rows in flight
        for (; m + (R - 1) * a.rl < hi; m += R * a.rl) {
            Raw8<T> d[R];
            Raw8<float> g[R];
#pragma unroll
            for (int k = 0; k < R; k++) {
                fetch(dy + (m + k * a.rl) * a.ldy, d[k]);
                if (a.slope) fetch(slope + (m + k * a.rl) * a.N, g[k]);
            }
#pragma unroll
            for (int k = 0; k < R; k++) one(m + k * a.rl, d[k], g[k]);
        }
        for (; m < hi; m += a.rl) {
            Raw8<T> d;
            Raw8<float> g;
            fetch(dy + m * a.ldy, d);
            if (a.slope) fetch(slope + m * a.N, g);
            one(m, d, g);
        }
    }
    if (!a.colsum) return;
    const int w = a.cvec * 8;
    if (r < a.rl)
#pragma unroll
        for (int i = 0; i < 8; i++) buf[r * w + cv * 8 + i] = at(s, i);
    for (int n = a.rl; n > 1;) {
        const int h = (n + 1) >> 1;
        __syncthreads();
        if (r < n - h)
#pragma unroll
            for (int i = 0; i < 8; i++) buf[r * w + cv * 8 + i] += buf[(r + h) * w + cv * 8 + i];
        n = h;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < w; k += 256) {
        const int cc = blockIdx.y * w + k;
        if (cc < a.N) a.colsum[(long long)blockIdx.x * a.N + cc] = buf[k];
    }
}

// ---- adds the k splits' parts in order and applies the epilogue; blocks from sum_blocks on fold the column
// sums of dz into db
struct JoinArgs {
    float *part;
    long long I, ldr, part_stride;
    int J, ldp, parts, sum_blocks, act;
    int more;  // other parts follow: the sum so far goes to the first's place
    const void *bias, *residual;
    void *out;
    float *slope;
    const float *colsum;
    int ncol, nsum;  // columns, and blocks that were summed
    void *db;
};
template <typename T>
__global__ void __launch_bounds__(256) k_join(JoinArgs a) {
    gs_let_follow();
    gs_wait_leader();
    if ((int)blockIdx.x >= a.sum_blocks) {
        __shared__ float red[8][33];
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = ((int)blockIdx.x - a.sum_blocks) * 32 + lane;
        float t = 0.f;
        if (c < a.ncol)
#pragma unroll 16
            for (int k = w; k < a.nsum; k += 8) t += a.colsum[(long long)k * a.ncol + c];
        red[w][lane] = t;
        __syncthreads();
        if (w == 0 && c < a.ncol) {
            for (int k = 1; k < 8; k++) t += red[k][lane];
            from_f32(t, reinterpret_cast<T *>(a.db)[c]);
        }
        return;
    }
    const Act<ACT_GELU, true> gelu;
    const Act<ACT_SILU, true> silu;
    const int nv = a.ldp / 4;
    const long long n = a.I * nv;
    for (long long t = blockIdx.x * 256LL + threadIdx.x; t < n; t += a.sum_blocks * 256LL) {
        const long long i = t / nv;
        const int c = (int)(t - i * nv) * 4;
        float *p = a.part + i * a.ldp + c;
        float4 s = *reinterpret_cast<const float4 *>(p);
#pragma unroll 8
        for (int k = 1; k < a.parts; k++) {
            const float4 e = *reinterpret_cast<const float4 *>(p + k * a.part_stride);
            s.x += e.x;
            s.y += e.y;
            s.z += e.z;
            s.w += e.w;
        }
        if (a.more) {
            *reinterpret_cast<float4 *>(p) = s;
            continue;
        }
        f2 v[2] = {{s.x, s.y}, {s.z, s.w}}, sl[2];
        const int n = min(4, a.J - c);
        if (a.bias) {
            const T *b = reinterpret_cast<const T *>(a.bias) + c;
            v[0] = add2(v[0], {to_f32(b[0]), n > 1 ? to_f32(b[1]) : 0.f});
            v[1] = add2(v[1], {n > 2 ? to_f32(b[2]) : 0.f, n > 3 ? to_f32(b[3]) : 0.f});
        }
        if (a.act == ACT_GELU) {
            v[0] = gelu(v[0], sl[0]);
            v[1] = gelu(v[1], sl[1]);
        } else if (a.act == ACT_SILU) {
            v[0] = silu(v[0], sl[0]);
            v[1] = silu(v[1], sl[1]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (k >= n) break;
            const long long at = i * a.J + c + k;
            float z = k & 1 ? v[k >> 1].y : v[k >> 1].x;
            if (a.slope) a.slope[at] = k & 1 ? sl[k >> 1].y : sl[k >> 1].x;
            if (a.residual) z = __fadd_rn(z, to_f32(reinterpret_cast<const T *>(a.residual)[i * a.ldr + c + k]));
            from_f32(z, reinterpret_cast<T *>(a.out)[at]);
        }
    }
}

// ================================================================================================ host
size_t al(size_t n) { return (n + 255) & ~(size_t)255; }
int up8(int n) { return (n + 7) & ~7; }
long long cdiv(long long a, long long b) { return (a + b - 1) / b; }

bool valid(const gs_linear_desc *d) {
    return d && d->M >= 0 && d->M <= GS_LINEAR_MAX_ROWS && d->N >= 1 && d->K >= 1 && d->N <= GS_LINEAR_MAX_DIM &&
           d->K <= GS_LINEAR_MAX_DIM && d->dtype >= GS_F32 && d->dtype <= GS_F16 && d->act >= GS_ACT_NONE &&
           d->act <= GS_ACT_SILU && d->ldx >= d->K && d->ldw >= d->K && (d->unaligned & ~7) == 0 &&
           d->ldx <= GS_LINEAR_MAX_LD && d->ldw <= GS_LINEAR_MAX_LD && d->ldr <= GS_LINEAR_MAX_LD &&
           d->ldy <= GS_LINEAR_MAX_LD && d->M * std::max(d->N, d->K) <= 1LL << 40;
}

// The tile of one product: pairs on 256 x 256, single CTAs on 128 x 128 or 128 x 64, whichever costs least, in SM
// cycles as measured: a k-block 720, 600 and 590 (16384x4096->4096: 387, 569, 1099 us); a tile's epilogue 7100, 2500
// and 1650 without an activation (36864x256->1024: 35.5, 43.3, 74.7 us), 9900, 3000 and 2050 with one (48.2, 50.6,
// 81.9 us; 36864x128->512: 25.6, 23.3, 31.5).  A pair's epilogue runs under the next tile's k-blocks; a single
// CTA's warps come back to the same accumulator, so theirs adds to them.  k splits while SMs are left over and a part
// keeps at least four k-blocks: their join costs a launch, 5 us of the host's time, and the parts' bytes or, where
// the output is small, a thread's walk over them (dweight of 100000x64->64: 31.8 us in 148 parts, 22.9 in 74, 26.3
// in 37).  Over 12 sizes, their three products, bf16 and fp32, the choice takes at most 1.1 times the best's time but
// for nine of the smallest (15 to 38 us): 1.1 to 1.36.
//
// A part has at most so many k-blocks as its type allows, because the accumulators cut what they add up rather than
// round it: by 1.7e-6 of the result over 1536 terms, 7e-4 over 131072 of one sign, 6e-3 over 2^20; the join rounds.
// 512 terms in fp32 (six products each), in 16-bit types 16384 (9e-5, where fp16's rounding is up to 5e-4).
constexpr int FP32_CHAIN = 8, CHAIN = 256;
struct Tiling {
    int bn, pair, splits;
    long long rows;  // of D a launch takes
    int slots;       // places for parts in the workspace
};
Tiling tiling(long long I, int J, long long kb, int npair, bool act) {
    Tiling best{64, 0, 1, I, 1};
    double least = 0;
    const int widths[3] = {256, 128, 64};
    const double block[3] = {720, 600, 590}, epi[3] = {act ? 9900. : 7100., act ? 3000. : 2500., act ? 2050. : 1650.};
    for (int w = 0; w < 3; w++) {
        const int bn = widths[w], pair = bn == 256, ti = pair ? 256 : 128, units = pair ? SMS / 2 : SMS;
        if (bn > 64 && J <= bn / 2) continue;
        const long long tiles = cdiv(I, ti) * cdiv(J, bn);
        // as few parts as the chain allows, or one for every second or every idle SM
        const long long few = cdiv(kb, npair == 6 ? FP32_CHAIN : CHAIN);
        const long long many = tiles < units ? std::min({units / tiles, kb * npair / 4, kb}) : 1;
        for (long long s : {few, std::max(few, many / 2), std::max(few, many)}) {
            const double waves = (double)cdiv(tiles * s, units), k = (double)cdiv(kb, s) * npair * block[w];
            const double join = s > 1 ? 9000 + s * std::max((double)I * J * 8 / 3000, 100.) : 0;
            const double cost = (pair ? waves * std::max(k, epi[w]) + std::min(k, epi[w]) : waves * (k + epi[w])) + join;
            if (least == 0 || cost < least) {
                least = cost;
                best = Tiling{bn, pair, (int)s, I, (int)s};
            }
        }
    }
    return best;
}

// The parts of one product take PART_BYTES of the workspace, or what 256 rows or two parts do where that is more:
// unbounded, 16384x4096->4096 in fp32 took 2.15 GB, and dW as many times its size as there are 512 rows.  What goes
// over it by k-blocks alone (parts are then as many as a sum may have terms) is cut into panels of rows, which
// multiply nearly as fast while a panel fills the SMs (the same size 3,088 us, 2,968 in one), or, where `rows` is false (dW, whose k is long), into groups of parts.
constexpr long long PART_BYTES = 256 << 20;
Tiling bounded(long long I, int J, long long kb, int npair, bool act, bool rows) {
    Tiling t = tiling(I, J, kb, npair, act);
    const long long row = (long long)t.splits * ((J + 3) & ~3) * 4;  // bytes of one row's parts
    if (t.splits == 1 || row * I <= PART_BYTES) return t;
    if (rows) {
        const long long most = std::max(256LL, PART_BYTES / row / 256 * 256);
        if (most < I) {
            t = tiling(most, J, kb, npair, act);
            t.rows = most;
        }
    } else {
        t.slots = (int)std::min<long long>(t.splits, std::max(2LL, PART_BYTES / (row / t.splits * I)));
    }
    return t;
}

// Workspace of a call: padded or split operands, the parts of split sums, column sums.
struct Plan {
    int es, terms, dz_terms;  // element size of the operands' source; terms of x and W, of dz
    int ldx, ldw, ldn;     // row strides of the padded x, W and dz
    bool prep_x, prep_w, need_dz;
    Tiling fwd, gx, gw;
    int dz_rows, dz_cols, dz_cvec, dz_rl;
    size_t o_x, o_w, o_dz, o_part, o_col, bytes;
};
bool ragged(long long ld, int unaligned) { return unaligned || ld % 8 != 0; }

size_t parts(const Tiling &t, int J) {
    return t.splits > 1 ? al((size_t)t.slots * t.rows * ((J + 3) & ~3) * 4) : 0;
}
Plan plan(const gs_linear_desc *d, bool bwd) {
    Plan p;
    memset(&p, 0, sizeof(p));
    const bool f32 = d->dtype == GS_F32;
    p.es = f32 ? 4 : 2;
    p.terms = f32 ? 3 : 1;
    p.ldx = p.ldw = up8(d->K);
    p.ldn = up8(d->N);
    p.prep_x = f32 || ragged(d->ldx, d->unaligned & 1);
    p.prep_w = f32 || ragged(d->ldw, d->unaligned & 2);
    p.bytes = 256;
    if (d->M == 0) return p;
    size_t o = 0;
    auto take = [&](size_t n) {
        const size_t at = o;
        o += al(n);
        return at;
    };
    p.o_x = take(p.prep_x ? (size_t)d->M * p.ldx * 2 * p.terms : 0);
    p.o_w = take(p.prep_w ? (size_t)d->N * p.ldw * 2 * p.terms : 0);
    if (!bwd) {
        p.fwd = bounded(d->M, d->N, cdiv(d->K, BK), f32 ? 6 : 1, d->act != GS_ACT_NONE, true);
        p.o_part = take(parts(p.fwd, d->N));
    } else {
        p.need_dz = f32 || d->act != GS_ACT_NONE || ragged(d->ldy, d->unaligned & 4);
        p.dz_terms = f32 ? 3 : d->act != GS_ACT_NONE ? 2 : 1;  // (without an activation dz is dy)
        p.o_dz = take(p.need_dz ? (size_t)d->M * p.ldn * 2 * p.dz_terms : 0);
        p.gx = bounded(d->M, d->K, cdiv(d->N, BK), f32 ? 6 : p.dz_terms, false, true);
        p.gw = bounded(d->N, d->K, cdiv(d->M, BK), f32 ? 6 : p.dz_terms, false, false);
        p.o_part = take(std::max(parts(p.gx, d->K), parts(p.gw, d->K)));
        // dz: blocks of 256 threads, up to 256 column vectors each, about four blocks per SM
        const int nv = p.ldn / 8;
        p.dz_cvec = std::min(nv, 256);
        p.dz_cols = (int)cdiv(nv, p.dz_cvec);
        p.dz_rl = 256 / p.dz_cvec;
        p.dz_rows = (int)std::max<long long>(1, std::min<long long>(cdiv(4 * SMS, p.dz_cols), d->M / (4 * p.dz_rl)));
        p.o_col = take((size_t)p.dz_rows * d->N * 4);
    }
    p.bytes = o + 256;
    return p;
}

int cuda_error(const char *where, const char *what) {
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", where, what);
    gs_set_last_error(msg);
    return GS_ERR_CUDA;
}
int done(const char *where) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? GS_OK : cuda_error(where, cudaGetErrorString(e));
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void *p = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}
// [terms][rows][cols] elements of es bytes with row stride ld and term stride `term`: boxes of box_cols x box_rows,
// swizzled
bool make_map(CUtensorMap *tm, CUtensorMapDataType type, int es, const void *base, long long cols, long long rows,
              long long ld, int terms, long long term, int box_cols, int box_rows) {
    // rows of operand boxes are 128 bytes, of output and residual units 64
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)terms};
    const cuuint64_t str[2] = {(cuuint64_t)ld * es, (cuuint64_t)(terms > 1 ? term : ld) * es};
    const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1}, one[3] = {1, 1, 1};
    auto fn = encode_fn();
    return fn && fn(tm, type, 3, const_cast<void *>(base), dims, str, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    box_cols * es == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The word that waits report to: pinned host memory that every device sees, so that the host reads it without a copy
// or a wait.  NULL where there is no device.
int *wait_error() {
    static int *const word = [] {
        // (an allocation is no work of a stream: made while one is captured too)
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        const bool set = cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
        int *p = nullptr;
        if (cudaHostAlloc(reinterpret_cast<void **>(&p), sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess) p = nullptr;
        if (set) cudaThreadExchangeStreamCaptureMode(&mode);
        if (p) *p = 0;
        return p;
    }();
    return word;
}
int take_wait_error(int *word) { return __atomic_load_n(word, __ATOMIC_RELAXED) ? __atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL) : 0; }
// reports what an earlier call's waits left, once
int check_waits(const char *where) {
    int *const word = wait_error();
    if (!word) return cuda_error(where, "no pinned host memory");
    const int code = take_wait_error(word);
    if (!code) return GS_OK;
    char msg[128];
    snprintf(msg, sizeof(msg), "%s: a device wait of an earlier linear call gave up (code %d), its outputs are not valid", where, code);
    gs_set_last_error(msg);
    return GS_ERR_TIMEOUT;
}

// The driver encodes tensor maps only on a thread with a context.  One that has made no such call yet (a new thread's
// first linear call, autograd's in a backward that begins with a product) gets its device's here.
int bind_device(const char *where) {
    static thread_local int bound = -1;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev == bound) return GS_OK;
    if (e == cudaSuccess) e = cudaSetDevice(dev);
    if (e != cudaSuccess) return cuda_error(where, cudaGetErrorString(e));
    bound = dev;
    return GS_OK;
}

template <int BN, bool PAIR, bool OUT32, int EPI, bool LO>
int launch(const CUtensorMap *m, const GemmArgs &a, bool follows, cudaStream_t s) {
    using S = Shape<BN, PAIR, OUT32, EPI>;
    auto kern = k_gemm<BN, PAIR, OUT32, EPI, LO>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM) != cudaSuccess)
        return done("gs_linear_act");
    const int items = a.tiles_i * a.tiles_j * a.nparts;
    gs_launch(kern, dim3(PAIR ? 2 * std::min(items, SMS / 2) : std::min(items, SMS)), GEMM_THREADS, S::SMEM, s, follows,
              PAIR ? 2 : 1, m[0], m[1], m[2], m[3], m[4], a);
    gs_count_launch(1);
    return GS_OK;
}
template <bool OUT32, int EPI, bool LO = false>
int launch_tile(int bn, const CUtensorMap *m, const GemmArgs &a, bool follows, cudaStream_t s) {
    return bn == 256   ? launch<256, true, OUT32, EPI, LO>(m, a, follows, s)
           : bn == 128 ? launch<128, false, OUT32, EPI, LO>(m, a, follows, s)
                       : launch<64, false, OUT32, EPI, LO>(m, a, follows, s);
}
template <bool OUT32>
int launch_epi(int epi, int bn, const CUtensorMap *m, const GemmArgs &a, bool follows, cudaStream_t s) {
    switch (epi) {
        case EPI_NONE:
            return a.f16 && a.npair == 2 ? launch_tile<OUT32, EPI_NONE, true>(bn, m, a, follows, s)
                                         : launch_tile<OUT32, EPI_NONE>(bn, m, a, follows, s);
        case EPI_GELU: return launch_tile<OUT32, EPI_GELU>(bn, m, a, follows, s);
        case EPI_SILU: return launch_tile<OUT32, EPI_SILU>(bn, m, a, follows, s);
        case EPI_GELU_SLOPE: return launch_tile<OUT32, EPI_GELU_SLOPE>(bn, m, a, follows, s);
        default: return launch_tile<OUT32, EPI_SILU_SLOPE>(bn, m, a, follows, s);
    }
}

// one operand of a product: [terms][rows][cols], row stride ld
struct Operand {
    const void *p;
    long long rows, cols, ld;
    int mn;  // the product's own axis is adjacent (else k is)
    int terms;
    long long term;  // stride of the terms
};
struct Epilogue {
    const void *bias, *residual;
    long long ldr;
    int act;
    void *out;
    float *slope;
};

// Parts first.. of D [I][J] over k = K, one after the other from place `slot` of `part` on for the caller to join; a
// product of one part is finished
int product(const gs_linear_desc *d, const Tiling &t, long long I, int J, long long K, const Operand &A, const Operand &B,
            const Epilogue &e, void *part, int first, int nparts, int slot, bool follows, cudaStream_t s) {
    GemmArgs a;
    memset(&a, 0, sizeof(a));
    const bool f32 = d->dtype == GS_F32, raw = t.splits > 1, out32 = f32 || raw;
    a.I = I; a.J = J;
    a.kb = (int)cdiv(K, BK);
    a.npair = f32 ? 6 : A.terms;
    a.a_mn = A.mn; a.b_mn = B.mn;
    a.f16 = d->dtype == GS_F16;
    a.out_f16 = a.f16;
    a.splits = t.splits; a.first = first; a.nparts = nparts; a.slot = slot;
    a.tiles_i = (int)cdiv(I, t.pair ? 256 : 128);
    a.tiles_j = (int)cdiv(J, t.bn);
    a.wait_error = wait_error();
    CUtensorMap m[5];
    const CUtensorMapDataType in = a.f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    bool ok = make_map(&m[0], in, 2, A.p, A.cols, A.rows, A.ld, A.terms, A.term, 64, A.mn ? BK : BM) &&
              make_map(&m[1], in, 2, B.p, B.cols, B.rows, B.ld, B.terms, B.term, 64, B.mn ? BK : t.pair ? t.bn / 2 : t.bn);
    m[2] = m[3] = m[4] = m[0];
    if (raw) {
        a.out_tma = 1;
        const long long ldp = (J + 3) & ~3;
        ok = ok && make_map(&m[2], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, part, J, I, ldp, slot + nparts, I * ldp, 16, 32);
    } else {
        const int es = f32 ? 4 : 2, ec = f32 ? 16 : 32;
        const CUtensorMapDataType ty = f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
        a.bias = e.bias; a.residual = e.residual; a.ldr = e.ldr; a.out = e.out; a.slope = e.slope;
        const auto whole = [&](const void *q, long long ld) { return ((uintptr_t)q & 15) == 0 && ld * es % 16 == 0; };
        a.out_tma = whole(e.out, J) && ((uintptr_t)e.slope & 15) == 0;  // (rows of slopes are as long or longer)
        a.res_tma = e.residual && whole(e.residual, e.ldr);
        if (a.out_tma) ok = ok && make_map(&m[2], ty, es, e.out, J, I, J, 1, 0, ec, 32);
        if (a.out_tma && e.slope) ok = ok && make_map(&m[3], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, e.slope, J, I, J, 1, 0, 16, 32);
        if (a.res_tma) ok = ok && make_map(&m[4], ty, es, e.residual, J, I, e.ldr, 1, 0, ec, 32);
    }
    if (!ok) return cuda_error("gs_linear_act", "cuTensorMapEncodeTiled refused a tensor");
    const int epi = raw || e.act == GS_ACT_NONE ? EPI_NONE : e.act == GS_ACT_GELU ? (e.slope ? EPI_GELU_SLOPE : EPI_GELU)
                                                                                   : (e.slope ? EPI_SILU_SLOPE : EPI_SILU);
    return out32 ? launch_epi<true>(epi, t.bn, m, a, follows, s) : launch_epi<false>(epi, t.bn, m, a, follows, s);
}

// db from the column sums of dz
struct Fold {
    const float *colsum;
    int ncol, nsum;
    void *db;  // NULL: nothing
};
// Adds `parts` parts of D [I][J] (0: none), to the sum so far or to the epilogue, and folds db beside it.
template <typename T>
void join(long long I, int J, int parts, bool more, const Epilogue &e, void *part, const Fold &f, cudaStream_t s) {
    JoinArgs a;
    memset(&a, 0, sizeof(a));
    if (parts) {
        a.part = reinterpret_cast<float *>(part);
        a.I = I; a.J = J; a.ldp = (J + 3) & ~3; a.part_stride = I * a.ldp; a.parts = parts; a.more = more;
        a.sum_blocks = (int)std::min<long long>(cdiv(I * (a.ldp / 4), 256), 8 * SMS);
        a.bias = e.bias; a.residual = e.residual; a.ldr = e.ldr; a.act = e.act; a.out = e.out; a.slope = e.slope;
    }
    a.colsum = f.colsum; a.ncol = f.ncol; a.nsum = f.nsum; a.db = f.db;
    const int fold = f.db ? (int)cdiv(f.ncol, 32) : 0;
    if (a.sum_blocks + fold == 0) return;
    gs_launch(k_join<T>, dim3((unsigned)(a.sum_blocks + fold)), 256, 0, s, true, 1, a);  // (a product or dz came before)
    gs_count_launch(1);
}
// D [I][J] over k = K, panel by panel and group by group, each joined; db is folded by the last join
template <typename T>
int whole_product(const gs_linear_desc *d, const Tiling &t, long long I, int J, long long K, const Operand &A,
                  const Operand &B, const Epilogue &e, void *part, const Fold &f, bool follows, cudaStream_t s) {
    const size_t es = sizeof(T);
    auto at = [](auto *p, long long bytes) {
        using P = decltype(p);
        return p ? (P)((const char *)p + bytes) : p;
    };
    for (long long r = 0; r < I; r += t.rows) {
        const long long rows = std::min(t.rows, I - r);
        Operand a = A;
        if (t.rows < I) {  // (A is then read along k: its rows are D's)
            a.p = at(A.p, r * A.ld * 2);
            a.rows = rows;
        }
        const Epilogue ep{e.bias, at(e.residual, r * e.ldr * (long long)es), e.ldr, e.act, at(e.out, r * J * (long long)es),
                          at(e.slope, r * J * 4)};
        for (int first = 0; first < t.splits;) {
            const int slot = first ? 1 : 0, n = std::min(t.slots - slot, t.splits - first);
            if (const int st = product(d, t, rows, J, K, a, B, ep, part, first, n, slot, follows, s)) return st;
            follows = true;
            first += n;
            const bool more = first < t.splits, last = !more && r + rows == I;
            if (t.splits > 1) join<T>(rows, J, slot + n, more, ep, part, last ? f : Fold{}, s);
        }
    }
    if (t.splits == 1) join<T>(0, 0, 0, false, e, nullptr, f, s);
    return GS_OK;
}

char *base_of(void *ws) { return reinterpret_cast<char *>(al((uintptr_t)ws)); }

// x and W as the products read them: in place, or prepared in the workspace by the jobs
PrepJobs operands(const gs_linear_desc *d, const Plan &p, const void *x, const void *w, char *ws, bool want_x, bool want_w,
                  Operand &X, Operand &W) {
    PrepJobs jobs;
    memset(&jobs, 0, sizeof(jobs));
    X = Operand{x, d->M, d->K, d->ldx, 0, p.terms, d->M * p.ldx};
    W = Operand{w, d->N, d->K, d->ldw, 0, p.terms, (long long)d->N * p.ldw};
    if (want_x && p.prep_x) {
        jobs.job[jobs.n++] = PrepJob{x, ws + p.o_x, d->M, d->ldx, d->K, p.ldx};
        X.p = ws + p.o_x;
        X.ld = p.ldx;
    }
    if (want_w && p.prep_w) {
        jobs.job[jobs.n++] = PrepJob{w, ws + p.o_w, d->N, d->ldw, d->K, p.ldw};
        W.p = ws + p.o_w;
        W.ld = p.ldw;
    }
    long long most = 0;
    for (int k = 0; k < jobs.n; k++) most = std::max(most, jobs.job[k].rows * (jobs.job[k].ldp / 8));
    jobs.blocks = (int)std::min<long long>(cdiv(most, 256), 8 * SMS);
    return jobs;
}

template <typename T>
int forward(const gs_linear_desc *d, const Plan &p, const void *x, const void *w, const Epilogue &e, void *workspace,
            cudaStream_t s) {
    char *ws = base_of(workspace);
    Operand X, W;
    const PrepJobs jobs = operands(d, p, x, w, ws, true, true, X, W);
    if (jobs.n) {
        k_prep_operands<T><<<dim3((unsigned)jobs.blocks, (unsigned)jobs.n), 256, 0, s>>>(jobs);
        gs_count_launch(1);
    }
    const int st = whole_product<T>(d, p.fwd, d->M, d->N, d->K, X, W, e, ws + p.o_part, Fold{}, jobs.n > 0, s);
    return st != GS_OK ? st : done("gs_linear_act_fwd");
}

template <typename T>
int backward(const gs_linear_desc *d, const Plan &p, const void *x, const void *w, const float *slope, const void *dy,
             void *dx, void *dw, void *db, void *workspace, cudaStream_t s) {
    char *ws = base_of(workspace);
    Operand X, W;
    const PrepJobs jobs = operands(d, p, x, w, ws, dw != nullptr, dx != nullptr, X, W);
    Operand Z{dy, d->M, d->N, d->ldy, 0, p.dz_terms, d->M * p.ldn};
    const bool make_dz = p.need_dz && (dx || dw);
    float *colsum = db ? reinterpret_cast<float *>(ws + p.o_col) : nullptr;
    if (make_dz) {
        Z.p = ws + p.o_dz;
        Z.ld = p.ldn;
    }
    const bool rows = make_dz || db;
    if (rows || jobs.n) {
        const DzArgs a{dy, slope, make_dz ? ws + p.o_dz : nullptr, colsum, d->M, d->ldy, d->N, p.ldn, p.dz_cvec, p.dz_rl,
                       rows ? p.dz_rows : 0, p.dz_terms, jobs};
        // whole 16-byte vectors of dy and of the kept slope
        const bool vec = !ragged(d->ldy, d->unaligned & 4) && d->N % 8 == 0 && ((uintptr_t)slope & 15) == 0;
        const dim3 grid((unsigned)(a.rows + jobs.blocks), (unsigned)(rows ? p.dz_cols : 1));
        if (vec) k_dz<T, true><<<grid, 256, 0, s>>>(a);
        else k_dz<T, false><<<grid, 256, 0, s>>>(a);
        gs_count_launch(1);
    }
    const bool first = rows || jobs.n;  // a launch of this call came before the products
    const Fold fold{colsum, d->N, p.dz_rows, db};
    if (dx) {
        Operand B = W;
        B.mn = 1;
        const Epilogue e{nullptr, nullptr, 0, 0, dx, nullptr};
        if (const int st = whole_product<T>(d, p.gx, d->M, d->K, d->N, Z, B, e, ws + p.o_part, dw ? Fold{} : fold, first, s)) return st;
    }
    if (dw) {
        Operand A = Z, B = X;
        A.mn = B.mn = 1;
        const Epilogue e{nullptr, nullptr, 0, 0, dw, nullptr};
        if (const int st = whole_product<T>(d, p.gw, d->N, d->K, d->M, A, B, e, ws + p.o_part, fold, first || dx, s)) return st;
    }
    if (!dx && !dw) join<T>(0, 0, 0, false, Epilogue{}, nullptr, fold, s);
    return done("gs_linear_act_bwd");
}

}  // namespace

extern "C" size_t gs_linear_act_workspace_size(const gs_linear_desc *d, int backward) {
    return valid(d) ? plan(d, backward != 0).bytes : 0;
}

extern "C" int gs_linear_act_debug_tiles(const gs_linear_desc *d, int product, int64_t *out) {
    if (!valid(d) || d->M == 0 || product < 0 || product > 2 || !out) return GS_ERR_BAD_ARGUMENT;
    const Plan p = plan(d, product > 0);
    const Tiling &t = product == 0 ? p.fwd : product == 1 ? p.gx : p.gw;
    out[0] = t.bn; out[1] = t.splits; out[2] = t.rows; out[3] = t.slots;
    return GS_OK;
}

extern "C" int gs_linear_act_fwd(const gs_linear_desc *d, const void *x, const void *w, const void *bias,
                                 const void *residual, void *y, float *slope, void *workspace, size_t workspace_bytes,
                                 void *stream) {
    if (!valid(d) || (residual && d->ldr < d->N)) return GS_ERR_BAD_ARGUMENT;
    if (d->M == 0) return GS_OK;
    if (!x || !w || !y) return GS_ERR_BAD_ARGUMENT;
    if ((((uintptr_t)x & 15) && !(d->unaligned & 1)) || (((uintptr_t)w & 15) && !(d->unaligned & 2)))
        return GS_ERR_BAD_ARGUMENT;
    const Plan p = plan(d, false);
    if (p.bytes > 256 && (!workspace || workspace_bytes < p.bytes)) return GS_ERR_WORKSPACE;
    if (const int st = bind_device("gs_linear_act_fwd")) return st;
    if (const int st = check_waits("gs_linear_act_fwd")) return st;
    cudaStream_t s = (cudaStream_t)stream;
    const Epilogue e{bias, residual, d->ldr, d->act, y, d->act == GS_ACT_NONE ? nullptr : slope};
    if (d->dtype == GS_F32) return forward<float>(d, p, x, w, e, workspace, s);
    if (d->dtype == GS_BF16) return forward<__nv_bfloat16>(d, p, x, w, e, workspace, s);
    return forward<__half>(d, p, x, w, e, workspace, s);
}

extern "C" int gs_linear_act_bwd(const gs_linear_desc *d, const void *x, const void *w, const float *slope,
                                 const void *dy, void *dx, void *dw, void *dbias, void *workspace,
                                 size_t workspace_bytes, void *stream) {
    if (!valid(d) || d->ldy < d->N) return GS_ERR_BAD_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    const size_t es = d->dtype == GS_F32 ? 4 : 2;
    if (d->M == 0) {
        if (dw) cudaMemsetAsync(dw, 0, (size_t)d->N * d->K * es, s);
        if (dbias) cudaMemsetAsync(dbias, 0, (size_t)d->N * es, s);
        return done("gs_linear_act_bwd");
    }
    if (!x || !w || !dy || (d->act != GS_ACT_NONE && !slope)) return GS_ERR_BAD_ARGUMENT;
    if ((((uintptr_t)x & 15) && !(d->unaligned & 1)) || (((uintptr_t)w & 15) && !(d->unaligned & 2)) ||
        (((uintptr_t)dy & 15) && !(d->unaligned & 4)))
        return GS_ERR_BAD_ARGUMENT;
    const Plan p = plan(d, true);
    if (p.bytes > 256 && (!workspace || workspace_bytes < p.bytes)) return GS_ERR_WORKSPACE;
    if (const int st = bind_device("gs_linear_act_bwd")) return st;
    if (const int st = check_waits("gs_linear_act_bwd")) return st;
    if (d->act == GS_ACT_NONE) slope = nullptr;
    if (d->dtype == GS_F32) return backward<float>(d, p, x, w, slope, dy, dx, dw, dbias, workspace, s);
    if (d->dtype == GS_BF16) return backward<__nv_bfloat16>(d, p, x, w, slope, dy, dx, dw, dbias, workspace, s);
    return backward<__half>(d, p, x, w, slope, dy, dx, dw, dbias, workspace, s);
}

extern "C" int gs_linear_error_flag(int *flag_host) {
    if (!flag_host) return GS_ERR_BAD_ARGUMENT;
    const cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return cuda_error("gs_linear_error_flag", cudaGetErrorString(e));
    int *const word = wait_error();
    if (!word) return cuda_error("gs_linear_error_flag", "no pinned host memory");
    *flag_host = take_wait_error(word);
    return GS_OK;
}

// one thread waits for a barrier that nothing arrives at, and reports as k_gemm does
__global__ void k_wait_in_vain(unsigned limit, int *err) {
    __shared__ uint64_t bar;
    mbar_init(&bar, 1);
    fence_barrier_init();
    mbar_wait(&bar, 0, err, 255, limit);
}
extern "C" int gs_linear_debug_wait(uint32_t limit, void *stream) {
    if (limit > 1024) return GS_ERR_BAD_ARGUMENT;
    int *const word = wait_error();
    if (!word) return cuda_error("gs_linear_debug_wait", "no pinned host memory");
    k_wait_in_vain<<<1, 1, 0, (cudaStream_t)stream>>>(limit, word);
    gs_count_launch(1);
    return done("gs_linear_debug_wait");
}
