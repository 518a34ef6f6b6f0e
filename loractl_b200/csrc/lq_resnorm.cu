// The seam between two sub-blocks as one pass: the norm behind a sub-block, its gate and residual
// scale, and the modulated norm before the next one,
//
//   u = y                                   or  y * q * (1 + pw),   q = rsqrt(mean(y^2) + eps)
//   r = alpha * x + gate * u                (x alone when there is no y)
//   z = (r - mu) * s * (1 + w) * (1 + scale) + shift,   s = rsqrt(mean((r - mu)^2) + eps)
//
// with mu = 0 for the RMS norm (crates/loractl-core/src/mmdit.rs:282-330) and mu = mean(r) for the
// layer norm; gate, shift, scale are [samples, h] and broadcast over the tokens of their sample
// (crates/loractl-core/src/mmdit.rs:857-869 runs these as separate broadcast tensor ops).
// Statistics, r and every sum are f32; r and z are rounded once, when stored, and z is formed from
// the unrounded r.
//
// Backward (gz = dz (1 + w)(1 + scale), rh = (r - mu) s, yh = y q, m(.) = mean over the row):
//   D  = dr + s (gz - [m(gz)] - rh m(gz rh))        the bracket for the layer norm only
//   dx = alpha D,   du = gate D,   dy = du   or   q (du (1 + pw) - yh m(du (1 + pw) yh))
//   S = sum_t dz rh,  T = sum_t dz,  G = sum_t D yh      per sample and column
//   dscale = S (1 + w),  dshift = T,  dgate = G (1 + pw),  dw = sum_b S (1 + scale),  dpw = sum_b gate G
// r is formed again from x and y instead of being read back: y is needed for G anyway, so it costs no
// byte more than reading r and keeps rh at f32 accuracy.  Forward and backward form it by the same operations in the same
// order, fma(gate (1 + pw), y q, alpha x), since s and mu are those of the forward's r: where x and y nearly cancel, another
// rounding of r would no longer fit them.
#include <algorithm>
#include <atomic>

#include <cuda_bf16.h>

#include "lq_internal.cuh"
#include "lq_prof.cuh"
#include "lq_resnorm_plan.cuh"
#include "lq_tc.cuh"
#include "lq_umma.cuh"

namespace {

using namespace resnorm_plan;

typedef lq_residual_norm_args Args;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }

// One value of a modulation vector (f32 or bf16 by the call).
__device__ __forceinline__ float mod_at(const void* p, int f32, int64_t i) {
    return f32 ? ((const float*)p)[i] : to_f(((const __nv_bfloat16*)p)[i]);
}

// Sums of NV values over the threads of a block, in a fixed order.  `area` has two halves that take turns, so that
// one barrier per reduction is enough: whoever writes a half again has passed the barrier of the reduction between.
// Its places behind the last warp hold zeros.
constexpr int kMaxWarps = 32;
template <int NV>
__device__ __forceinline__ void warp_sum(float (&v)[NV]) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1)
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
}
template <int MAXT, int NV>
__device__ __forceinline__ void block_sum(float (&v)[NV], float (*area)[2][kMaxWarps], int& half) {
    warp_sum<NV>(v);
    if (MAXT <= 128 && blockDim.x == 32) {
        __syncwarp();
        return;
    }
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < NV; ++k) area[half][k][threadIdx.x >> 5] = v[k];
    __syncthreads();
    if (MAXT <= 256) {  // up to 8 partial sums: two vector reads are shorter than five exchanges
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            v[k] = 0.f;
#pragma unroll
            for (int w = 0; w < MAXT / 32; w += 4) {
                const float4 q = *(const float4*)&area[half][k][w];
                v[k] += (q.x + q.y) + (q.z + q.w);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] = area[half][k][threadIdx.x & 31];
        warp_sum<NV>(v);
    }
    half ^= 1;
}
__device__ __forceinline__ void clear_area(float (*area)[2][kMaxWarps]) {
    for (int i = threadIdx.x; i < 2 * 2 * kMaxWarps; i += blockDim.x) (&area[0][0][0])[i] = 0.f;
    __syncthreads();
}

// 1 / sqrt(v) for v >= eps: the hardware's estimate and one Newton step (the IEEE square root and quotient are forty
// instructions that every thread of a row would run).  0 for a sum of squares that overflowed.
__device__ __forceinline__ float rsqrt_f32(float v) {
    const float y = rsqrtf(v);
    return y == 0.f ? y : y * fmaf(-0.5f * v * y, y, 1.5f);
}

// The rows of one block: chunk `blockIdx.x % chunks` of a sample.
struct Rows {
    int64_t b, t0, t1;
    __device__ __forceinline__ Rows(int64_t tokens, int chunks, int64_t per) {
        b = blockIdx.x / chunks;
        t0 = (blockIdx.x - b * chunks) * per;
        t1 = min(tokens, t0 + per);
    }
};

// ---- rows that start on 16 bytes ------------------------------------------------------------------
// HBM-bound, so what counts is bytes in flight.  A block walks the rows of its chunk; a few threads keep a ring of
// rows in shared memory filled with bulk copies (a row of each input per stage), and no other thread waits for HBM
// itself.  A thread owns 8 columns for good: it keeps the modulation of the sample and, in the backward, its column
// sums in registers, so that the only exchange is the row's own sums, and a stage may be refilled after the barrier
// of the first of them.
// Register rows instead of the ring (one row per block, loads straight to registers) took 29 us forward and 95 us
// backward on 1536 rows of 6144 bf16 columns, where this takes 17 and 25; the modulation read again from L1 for every row
// was part of that.  At 4096 rows 34 us and 63 us: 89 % and 73 % of the measured HBM rate; 8 x 4096 x 2048 with the layer
// norm 93 us and 150 us: 88 % and 82 %.  The backward's column sums and modulation spill 16-140 bytes a thread at 80 registers, 144-296
// at the 64 of 1024 threads.

// Eight elements as they are stored (four registers in bf16): what is needed again behind a barrier waits like this.
template <typename T>
struct Raw8 {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void ld(const uint8_t* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = ((const uint4*)p)[i];
    }
    __device__ __forceinline__ float operator[](int e) const {
        const uint4 q = v[sizeof(T) == 4 ? e >> 2 : 0];
        const int k = sizeof(T) == 4 ? e & 3 : e >> 1;
        const uint32_t w = k == 0 ? q.x : (k == 1 ? q.y : (k == 2 ? q.z : q.w));
        return sizeof(T) == 4 ? __uint_as_float(w) : __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16);
    }
};
template <typename T>
__device__ __forceinline__ void ld8(const uint8_t* p, float (&f)[8]) {
    Raw8<T> r;
    r.ld(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = r[e];
}
__device__ __forceinline__ void st8(__nv_bfloat16* p, const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *(const uint32_t*)&h;
    }
    *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void st8(float* p, const float (&f)[8]) {
    *(float4*)p = make_float4(f[0], f[1], f[2], f[3]);
    *(float4*)(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
// Pairs of f32 in one 64-bit register pair: one instruction for two products or sums, each rounded as its scalar form
// is.  A row's arithmetic was two thirds of the issue slots of the backward.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ f2 both(float v) { return pack2(v, v); }
__device__ __forceinline__ void unpack2(f2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float sum2(f2 v) {
    float lo, hi;
    unpack2(v, lo, hi);
    return lo + hi;
}
template <typename T>
__device__ __forceinline__ f2 pair_of(const Raw8<T>& r, int k) { return pack2(r[2 * k], r[2 * k + 1]); }
template <typename T>
__device__ __forceinline__ void st8(T* p, const f2 (&v)[4]) {
    float f[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) unpack2(v[k], f[2 * k], f[2 * k + 1]);
    st8(p, f);
}
__device__ __forceinline__ void pack8(const float (&f)[8], f2 (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = pack2(f[2 * k], f[2 * k + 1]);
}

__device__ __forceinline__ void ld_mod8(const void* p, int f32, int64_t i, float (&f)[8]) {
    if (f32) ld8<float>((const uint8_t*)p + i * 4, f);
    else ld8<__nv_bfloat16>((const uint8_t*)p + i * 2, f);
}

// The ring's filling: thread i < inputs copies input i's row of a stage (the same instruction of one warp), thread 0
// announces the bytes.
struct Feed {
    const uint8_t* src;
    int64_t step;
    __device__ __forceinline__ void of(const void* p, int64_t first, int64_t token, int esz) {
        src = (const uint8_t*)p + first * esz;
        step = token * esz;
    }
    __device__ __forceinline__ void fill(uint32_t bar, uint32_t stage, uint32_t row_bytes, uint32_t stage_bytes) {
        if (threadIdx.x == 0) umma::mbar_expect_tx(bar, stage_bytes);
        umma::bulk_load(stage + threadIdx.x * row_bytes, src, row_bytes, bar);
        src += step;
    }
};

extern __shared__ __align__(128) uint8_t ring_smem[];

template <typename T, bool POST, bool LAYER, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) resnorm_fwd_ring_kernel(const Args a, int chunks, int64_t per, int stages, int* status) {
    __shared__ __align__(16) float area[2][2][kMaxWarps];
    __shared__ __align__(8) uint64_t bars[kMaxStages];
    __shared__ int abort_flag;
    const Rows rows(a.tokens, chunks, per);
    const int h = (int)a.h, c = threadIdx.x * 8;
    const bool in = c < h;
    const float inv_h = 1.f / (float)h;
    const int n = (int)(rows.t1 - rows.t0);
    if (n <= 0) return;
    const int inputs = a.y ? 2 : 1;
    const uint32_t row_bytes = (uint32_t)h * sizeof(T), stage_bytes = row_bytes * inputs;
    const uint32_t ring = umma::smem_u32(ring_smem);
    Feed feed;
    if (threadIdx.x == 0) feed.of(a.x, rows.b * a.x_sample + rows.t0 * a.x_token, a.x_token, sizeof(T));
    else feed.of(a.y, rows.b * a.y_sample + rows.t0 * a.y_token, a.y_token, sizeof(T));
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) umma::mbar_init(umma::smem_u32(&bars[s]), 1);
        abort_flag = 0;
        umma::fence_barrier_init();
        umma::fence_proxy_async_smem();
    }
    if (threadIdx.x < 32) {
        __syncwarp();  // the barriers are there before any of the copying threads names one
        if (threadIdx.x < inputs)
            for (int s = 0; s < min(stages, n); ++s) feed.fill(umma::smem_u32(&bars[s]), ring + s * stage_bytes, row_bytes, stage_bytes);
    }
    clear_area(area);
    f2 gate[4] = {0, 0, 0, 0}, shift[4] = {0, 0, 0, 0}, mul[4] = {0, 0, 0, 0};  // of this thread's columns; mul = (1 + w)(1 + scale)
    if (in) {
        float f[8], w[8];
        ld_mod8(a.shift, a.mod_f32, rows.b * a.shift_sample + c, f);
        pack8(f, shift);
        ld_mod8(a.scale, a.mod_f32, rows.b * a.scale_sample + c, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += 1.f;
        if (a.weight) {
            ld_mod8(a.weight, 1, c, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= 1.f + w[e];
        }
        pack8(f, mul);
        if (a.y) ld_mod8(a.gate, a.mod_f32, rows.b * a.gate_sample + c, f);
        if (POST) {
            ld_mod8(a.post_weight, 1, c, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= 1.f + w[e];
        }
        pack8(f, gate);
    }
    int half = 0, s = 0;
    uint32_t phase = 0;
    const int64_t row0 = rows.b * a.tokens + rows.t0;
    T *rp = (T*)a.r + row0 * h + c, *zp = (T*)a.z + row0 * h + c;
    const f2 alpha = both(a.alpha);
    for (int i = 0; i < n; ++i) {
        const int64_t row = row0 + i;
        // a wait that gives up marks the error word; the block goes through its remaining rows without waiting
        umma::mbar_wait(umma::smem_u32(&bars[s]), phase, &abort_flag, status, 81);
        const uint8_t* st = ring_smem + s * stage_bytes + threadIdx.x * 8 * sizeof(T);
        f2 r[4];
        float v[1];
        {
            Raw8<T> x, y;
            x.zero();
            y.zero();
            if (in) x.ld(st);
            if (in && a.y) y.ld(st + row_bytes);
#pragma unroll
            for (int k = 0; k < 4; ++k) r[k] = pair_of(x, k);
            if (a.y) {
                f2 q = both(1.f);
                if (POST) {
                    f2 sq = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) sq = fma2(pair_of(y, k), pair_of(y, k), sq);
                    v[0] = sum2(sq);
                    block_sum<MAXT, 1>(v, area, half);
                    const float qs = rsqrt_f32(fmaf(v[0], inv_h, a.eps));
                    if (threadIdx.x == 0 && a.rstd) a.post_rstd[row] = qs;
                    q = both(qs);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) r[k] = fma2(gate[k], POST ? mul2(pair_of(y, k), q) : pair_of(y, k), mul2(alpha, r[k]));
            }
        }
        float mu = 0.f;
        f2 d[4];
        if (LAYER) {
            v[0] = sum2(add2(add2(r[0], r[1]), add2(r[2], r[3])));
            block_sum<MAXT, 1>(v, area, half);
            mu = v[0] * inv_h;
            const f2 m = both(-mu);
#pragma unroll
            for (int k = 0; k < 4; ++k) d[k] = add2(r[k], m);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) d[k] = r[k];
        }
        f2 sq = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) sq = fma2(d[k], d[k], sq);
        v[0] = in ? sum2(sq) : 0.f;
        block_sum<MAXT, 1>(v, area, half);  // every thread has read the stage
        if (threadIdx.x < inputs && i + stages < n) feed.fill(umma::smem_u32(&bars[s]), ring + s * stage_bytes, row_bytes, stage_bytes);
        const float rs = rsqrt_f32(fmaf(v[0], inv_h, a.eps));
        if (threadIdx.x == 0 && a.rstd) {
            a.rstd[row] = rs;
            if (LAYER) a.mean[row] = mu;
        }
        if (in) {
            if (a.r) st8(rp, r);
            const f2 rs2 = both(rs);
#pragma unroll
            for (int k = 0; k < 4; ++k) d[k] = fma2(mul2(d[k], rs2), mul[k], shift[k]);
            st8(zp, d);
            rp += h;
            zp += h;
        }
        if (++s == stages) { s = 0; phase ^= 1u; }
    }
    if (abort_flag)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the block ends
}

template <typename T, bool POST, bool LAYER, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) resnorm_bwd_ring_kernel(const Args a, const lq_residual_norm_grads g, int chunks, int64_t per,
                                                                      int stages, float* __restrict__ part, int* status) {
    __shared__ __align__(16) float area[2][2][kMaxWarps];
    __shared__ __align__(8) uint64_t bars[kMaxStages];
    __shared__ int abort_flag;
    const Rows rows(a.tokens, chunks, per);
    const int h = (int)a.h, c = threadIdx.x * 8;
    const bool in = c < h;
    const float inv_h = 1.f / (float)h;
    const int n = (int)max((int64_t)0, rows.t1 - rows.t0);
    const uint32_t row_bytes = (uint32_t)h * sizeof(T);
    // a stage holds x, then what there is of dz, dr, y
    const int i_dz = 1, i_dr = i_dz + (g.dz ? 1 : 0), i_y = i_dr + (g.dr ? 1 : 0), inputs = i_y + (a.y ? 1 : 0);
    const uint32_t at_dz = row_bytes, at_dr = i_dr * row_bytes, at_y = i_y * row_bytes, stage_bytes = inputs * row_bytes;
    const uint32_t ring = umma::smem_u32(ring_smem);
    Feed feed;
    if (threadIdx.x == 0) feed.of(a.x, rows.b * a.x_sample + rows.t0 * a.x_token, a.x_token, sizeof(T));
    else if (g.dz && threadIdx.x == i_dz) feed.of(g.dz, rows.b * g.dz_sample + rows.t0 * g.dz_token, g.dz_token, sizeof(T));
    else if (g.dr && threadIdx.x == i_dr) feed.of(g.dr, rows.b * g.dr_sample + rows.t0 * g.dr_token, g.dr_token, sizeof(T));
    else feed.of(a.y, rows.b * a.y_sample + rows.t0 * a.y_token, a.y_token, sizeof(T));
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) umma::mbar_init(umma::smem_u32(&bars[s]), 1);
        abort_flag = 0;
        umma::fence_barrier_init();
        umma::fence_proxy_async_smem();
    }
    if (threadIdx.x < 32) {
        __syncwarp();  // the barriers are there before any of the copying threads names one
        if (threadIdx.x < inputs)
            for (int s = 0; s < min(stages, n); ++s) feed.fill(umma::smem_u32(&bars[s]), ring + s * stage_bytes, row_bytes, stage_bytes);
    }
    clear_area(area);
    f2 gate[4] = {0, 0, 0, 0}, mul[4] = {0, 0, 0, 0}, S[4] = {0, 0, 0, 0}, D1[4] = {0, 0, 0, 0}, G[4] = {0, 0, 0, 0};
    if (in) {
        float f[8], w[8];
        ld_mod8(a.scale, a.mod_f32, rows.b * a.scale_sample + c, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += 1.f;
        if (a.weight) {
            ld_mod8(a.weight, 1, c, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= 1.f + w[e];
        }
        pack8(f, mul);
        if (a.y) ld_mod8(a.gate, a.mod_f32, rows.b * a.gate_sample + c, f);
        if (POST) {  // gate (1 + pw) is all that the row needs; dgate gets its (1 + pw) with the sums
            ld_mod8(a.post_weight, 1, c, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= 1.f + w[e];
        }
        if (a.y) pack8(f, gate);
    }
    int half = 0, s = 0;
    uint32_t phase = 0;
    const int64_t row0 = rows.b * a.tokens + rows.t0;
    T *dxp = (T*)g.dx + row0 * h + c, *dyp = (T*)g.dy + row0 * h + c;
    float rs = n > 0 ? a.rstd[row0] : 0.f, mu = n > 0 && LAYER ? a.mean[row0] : 0.f, q = n > 0 && POST ? a.post_rstd[row0] : 1.f;
    const f2 alpha = both(a.y ? a.alpha : 1.f);
    for (int i = 0; i < n; ++i) {
        const int64_t row = row0 + i;
        umma::mbar_wait(umma::smem_u32(&bars[s]), phase, &abort_flag, status, 82);
        const uint8_t* st = ring_smem + s * stage_bytes + threadIdx.x * 8 * sizeof(T);
        f2 rh[4], gz[4];
        Raw8<T> yr, dr;
        yr.zero();
        dr.zero();
        {
            Raw8<T> x, z;
            x.zero();
            z.zero();
            if (in) {
                x.ld(st);
                if (g.dz) z.ld(st + at_dz);
                if (g.dr) dr.ld(st + at_dr);
                if (a.y) yr.ld(st + at_y);
            }
            const f2 q2 = both(q), rs2 = both(rs), m = both(-mu);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                rh[k] = mul2(alpha, pair_of(x, k));
                if (a.y) rh[k] = fma2(gate[k], POST ? mul2(pair_of(yr, k), q2) : pair_of(yr, k), rh[k]);
                if (LAYER) rh[k] = add2(rh[k], m);
                rh[k] = mul2(rh[k], rs2);
                gz[k] = pair_of(z, k);
            }
        }
        f2 dot = 0, sum = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            S[k] = fma2(gz[k], rh[k], S[k]);
            D1[k] = add2(D1[k], gz[k]);
            gz[k] = mul2(gz[k], mul[k]);
            dot = fma2(gz[k], rh[k], dot);
            if (LAYER) sum = add2(sum, gz[k]);
        }
        float c0 = 0.f, c1;
        if (LAYER) {
            float v[2] = {sum2(dot), sum2(sum)};
            block_sum<MAXT, 2>(v, area, half);
            c1 = v[0] * inv_h, c0 = v[1] * inv_h;
        } else {
            float v[1] = {sum2(dot)};
            block_sum<MAXT, 1>(v, area, half);
            c1 = v[0] * inv_h;
        }
        // every thread has read the stage
        if (threadIdx.x < inputs && i + stages < n) feed.fill(umma::smem_u32(&bars[s]), ring + s * stage_bytes, row_bytes, stage_bytes);
        {
            const f2 m0 = both(-c0), m1 = both(-c1), rs2 = both(rs);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                f2 t = LAYER ? add2(gz[k], m0) : gz[k];
                rh[k] = fma2(rs2, fma2(rh[k], m1, t), pair_of(dr, k));  // D
            }
        }
        const f2 q2 = both(q);
        if (i + 1 < n) {  // the next row's statistics, behind the stores of this one
            rs = a.rstd[row + 1];
            if (LAYER) mu = a.mean[row + 1];
            if (POST) q = a.post_rstd[row + 1];
        }
        f2 p2 = 0;
        if (a.y) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f2 yh = POST ? mul2(pair_of(yr, k), q2) : pair_of(yr, k);
                G[k] = fma2(rh[k], yh, G[k]);
                gz[k] = mul2(gate[k], rh[k]);  // the gradient of yh
                if (POST) p2 = fma2(gz[k], yh, p2);
            }
        }
        if (g.dx && in) {
#pragma unroll
            for (int k = 0; k < 4; ++k) rh[k] = mul2(alpha, rh[k]);
            st8(dxp, rh);
        }
        dxp += h;
        if (a.y && g.dy) {
            if (POST) {
                float p[1] = {sum2(p2)};
                block_sum<MAXT, 1>(p, area, half);
                const f2 pm = both(-p[0] * inv_h);
#pragma unroll
                for (int k = 0; k < 4; ++k) gz[k] = mul2(q2, fma2(mul2(pair_of(yr, k), q2), pm, gz[k]));
            }
            if (in) st8(dyp, gz);
            dyp += h;
        }
        if (++s == stages) { s = 0; phase ^= 1u; }
    }
    if (part && in) {
        float* dst = part + (int64_t)blockIdx.x * 3 * h + c;
        st8(dst, S);
        st8(dst + h, D1);
        st8(dst + 2 * h, G);
    }
    if (abort_flag)
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
}

// ---- any rows -----------------------------------------------------------------------------------
// Single elements, for rows that do not all start on 16 bytes (an odd width, an odd offset) and for rows too wide
// for the ring: thread t owns the columns t, t + blockDim, ...  All of a row's loads are issued before the first is
// used, whatever columns the thread has (a place behind the row reads column 0 and counts as zero).  Up to 4096 columns
// (512 threads) the modulation stays in registers over the rows of a chunk and the next row is fetched into registers behind
// the current one's arithmetic; wider rows have no registers for either and take 1024 threads (4000 rows of 7777 bf16 columns:
// 145 us forward, 295 us backward; the backward with 512 threads 424 us), whose 64 registers spill 392-468 bytes a thread in the
// backward up to 8192 columns and 1372-1464 above (272-328 there in the forward).  Bound by instructions, two accesses and a dozen
// of arithmetic an element: 8000 rows of 4001 f32 columns 152 us forward and 166 us backward (51 % and 71 % of HBM),
// 24000 rows of 1155 bf16 columns 110 us and 153 us (31 % and 33 %; 1152 columns by the ring: 41 us and 69 us).
template <typename T, int VPT>
struct Raw {
    T v[VPT];
    __device__ __forceinline__ void ld(const T* p, int h) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            v[i] = p[c < h ? c : 0];
        }
    }
    __device__ __forceinline__ void get(int h, float (&f)[VPT]) const {
#pragma unroll
        for (int i = 0; i < VPT; ++i) f[i] = threadIdx.x + i * blockDim.x < h ? to_f(v[i]) : 0.f;
    }
};
template <typename T, int VPT>
__device__ __forceinline__ void ld_row(const T* p, int h, float (&f)[VPT]) {
    Raw<T, VPT> r;
    r.ld(p, h);
    r.get(h, f);
}
template <int VPT>
__device__ __forceinline__ void ld_mods(const void* p, int f32, int64_t at, int h, float (&f)[VPT]) {
    if (f32) ld_row<float, VPT>((const float*)p + at, h, f);
    else ld_row<__nv_bfloat16, VPT>((const __nv_bfloat16*)p + at, h, f);
}
template <typename T, int VPT>
__device__ __forceinline__ void st_row(T* p, int h, const float (&f)[VPT]) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        if (c < h) p[c] = from_f<T>(f[i]);
    }
}
// gate (1 + pw) and (1 + w)(1 + scale) of a sample, in this thread's columns.
template <int VPT>
__device__ __forceinline__ void ld_gate(const Args& a, int64_t b, int h, float (&f)[VPT]) {
    ld_mods<VPT>(a.gate, a.mod_f32, b * a.gate_sample, h, f);
    if (a.post_weight) {
        float pw[VPT];
        ld_row<float, VPT>(a.post_weight, h, pw);
#pragma unroll
        for (int i = 0; i < VPT; ++i) f[i] *= 1.f + pw[i];
    }
}
template <int VPT>
__device__ __forceinline__ void ld_mul(const Args& a, int64_t b, int h, float (&f)[VPT]) {
    ld_mods<VPT>(a.scale, a.mod_f32, b * a.scale_sample, h, f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) f[i] += 1.f;
    if (a.weight) {
        float w[VPT];
        ld_row<float, VPT>(a.weight, h, w);
#pragma unroll
        for (int i = 0; i < VPT; ++i) f[i] *= 1.f + w[i];
    }
}

template <typename T, int VPT, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 512 ? 2 : 1) resnorm_fwd_kernel(const Args a, int chunks, int64_t per) {
    constexpr bool KEEP = MAXT == 512;
    __shared__ __align__(16) float area[2][2][kMaxWarps];
    int half = 0;
    const Rows rows(a.tokens, chunks, per);
    const int64_t b = rows.b;
    const int h = (int)a.h;
    const float inv_h = 1.f / (float)h;
    clear_area(area);
    if (rows.t0 >= rows.t1) return;
    float gate[VPT], mul[VPT], shift[VPT];
    if (KEEP) {
        if (a.y) ld_gate<VPT>(a, b, h, gate);
        ld_mul<VPT>(a, b, h, mul);
        ld_mods<VPT>(a.shift, a.mod_f32, b * a.shift_sample, h, shift);
    }
    const T* xp = (const T*)a.x + b * a.x_sample + rows.t0 * a.x_token;
    const T* yp = (const T*)a.y + b * a.y_sample + rows.t0 * a.y_token;
    Raw<T, VPT> xr, yr;
    xr.ld(xp, h);
    if (a.y) yr.ld(yp, h);
    for (int64_t t = rows.t0; t < rows.t1; ++t) {
        const int64_t row = b * a.tokens + t;
        float r[VPT], y[VPT], v[1] = {0.f};
        xr.get(h, r);
        if (a.y) yr.get(h, y);
        if (KEEP && t + 1 < rows.t1) {
            xr.ld(xp += a.x_token, h);
            if (a.y) yr.ld(yp += a.y_token, h);
        }
        if (a.y) {
            if (!KEEP) ld_gate<VPT>(a, b, h, gate);
            if (a.post_weight) {
#pragma unroll
                for (int i = 0; i < VPT; ++i) v[0] = fmaf(y[i], y[i], v[0]);
                block_sum<MAXT, 1>(v, area, half);
                const float q = rsqrt_f32(fmaf(v[0], inv_h, a.eps));
                if (threadIdx.x == 0 && a.rstd) a.post_rstd[row] = q;
#pragma unroll
                for (int i = 0; i < VPT; ++i) y[i] *= q;
                v[0] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < VPT; ++i) r[i] = fmaf(gate[i], y[i], a.alpha * r[i]);
            if (a.r) st_row<T, VPT>((T*)a.r + row * h, h, r);
        }
        float mu = 0.f;
        if (a.layer) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) v[0] += r[i];
            block_sum<MAXT, 1>(v, area, half);
            mu = v[0] * inv_h;
            v[0] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (threadIdx.x + i * blockDim.x < h) v[0] = fmaf(r[i] - mu, r[i] - mu, v[0]);
        if (!KEEP) {
            ld_mul<VPT>(a, b, h, mul);
            ld_mods<VPT>(a.shift, a.mod_f32, b * a.shift_sample, h, shift);
        }
        block_sum<MAXT, 1>(v, area, half);
        const float s = rsqrt_f32(fmaf(v[0], inv_h, a.eps));
        if (threadIdx.x == 0 && a.rstd) {
            a.rstd[row] = s;
            if (a.layer) a.mean[row] = mu;
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) r[i] = fmaf((r[i] - mu) * s, mul[i], shift[i]);
        st_row<T, VPT>((T*)a.z + row * h, h, r);
        if (!KEEP && t + 1 < rows.t1) {
            xr.ld(xp += a.x_token, h);
            if (a.y) yr.ld(yp += a.y_token, h);
        }
    }
}

template <typename T, int VPT, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) resnorm_bwd_kernel(const Args a, const lq_residual_norm_grads g, int chunks, int64_t per,
                                                              float* __restrict__ part) {
    constexpr bool KEEP = MAXT == 512;
    __shared__ __align__(16) float area[2][2][kMaxWarps];
    int half = 0;
    const Rows rows(a.tokens, chunks, per);
    const int64_t b = rows.b;
    const int h = (int)a.h;
    const float inv_h = 1.f / (float)h;
    float S[VPT], D1[VPT], G[VPT], gate[VPT], mul[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) S[i] = D1[i] = G[i] = 0.f;
    clear_area(area);
    const T* xp = (const T*)a.x + b * a.x_sample + rows.t0 * a.x_token;
    const T* yp = (const T*)a.y + b * a.y_sample + rows.t0 * a.y_token;
    const T* zp = (const T*)g.dz + b * g.dz_sample + rows.t0 * g.dz_token;
    const T* rp = (const T*)g.dr + b * g.dr_sample + rows.t0 * g.dr_token;
    Raw<T, VPT> xr, yr, zr, rr;
    auto fetch = [&] {
        xr.ld(xp, h);
        if (g.dz) zr.ld(zp, h);
        if (a.y) yr.ld(yp, h);
        if (g.dr) rr.ld(rp, h);
        xp += a.x_token, yp += a.y_token, zp += g.dz_token, rp += g.dr_token;
    };
    if (rows.t0 < rows.t1) {
        if (KEEP) {
            if (a.y) ld_gate<VPT>(a, b, h, gate);
            ld_mul<VPT>(a, b, h, mul);
        }
        fetch();
    }
    for (int64_t t = rows.t0; t < rows.t1; ++t) {
        const int64_t row = b * a.tokens + t;
        float rh[VPT], gz[VPT], yh[VPT], d[VPT];
        const float s = a.rstd[row], mu = a.layer ? a.mean[row] : 0.f, q = a.post_weight ? a.post_rstd[row] : 1.f;
        xr.get(h, rh);
#pragma unroll
        for (int i = 0; i < VPT; ++i) gz[i] = yh[i] = d[i] = 0.f;
        if (g.dz) zr.get(h, gz);
        if (a.y) yr.get(h, yh);
        if (g.dr) rr.get(h, d);
        if (KEEP && t + 1 < rows.t1) fetch();
        if (!KEEP) {
            if (a.y) ld_gate<VPT>(a, b, h, gate);
            ld_mul<VPT>(a, b, h, mul);
        }
        if (a.y) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                if (a.post_weight) yh[i] *= q;
                rh[i] = fmaf(gate[i], yh[i], a.alpha * rh[i]);
            }
        }
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            rh[i] = (rh[i] - mu) * s;  // gz is zero behind the row
            S[i] = fmaf(gz[i], rh[i], S[i]);
            D1[i] += gz[i];
            gz[i] *= mul[i];
            v[0] = fmaf(gz[i], rh[i], v[0]);
            v[1] += gz[i];
        }
        block_sum<MAXT, 2>(v, area, half);
        const float c1 = v[0] * inv_h, c0 = a.layer ? v[1] * inv_h : 0.f;
        float p[1] = {0.f};
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            d[i] = fmaf(s, gz[i] - c0 - rh[i] * c1, d[i]);
            if (a.y) {
                G[i] = fmaf(d[i], yh[i], G[i]);
                gz[i] = gate[i] * d[i];
                p[0] = fmaf(gz[i], yh[i], p[0]);  // yh is zero behind the row
                d[i] *= a.alpha;
            }
        }
        if (g.dx) st_row<T, VPT>((T*)g.dx + row * h, h, d);
        if (a.y && g.dy) {
            if (a.post_weight) {
                block_sum<MAXT, 1>(p, area, half);
                const float pm = p[0] * inv_h;
#pragma unroll
                for (int i = 0; i < VPT; ++i) gz[i] = q * (gz[i] - yh[i] * pm);
            }
            st_row<T, VPT>((T*)g.dy + row * h, h, gz);
        }
        if (!KEEP && t + 1 < rows.t1) fetch();
    }
    if (!part) return;
    float* dst = part + (int64_t)blockIdx.x * 3 * h;
    st_row<float, VPT>(dst, h, S);
    st_row<float, VPT>(dst + h, h, D1);
    st_row<float, VPT>(dst + 2 * h, h, G);
}

__device__ __forceinline__ void st_mod(void* p, int f32, int64_t i, float v) {
    if (f32) ((float*)p)[i] = v;
    else ((__nv_bfloat16*)p)[i] = __float2bfloat16(v);
}

// Sums the partial rows in a fixed order.  Block = 32 columns x 16 ranges of chunks.  blockIdx.y < samples: the sums of
// that sample (dgate, dshift, dscale; of a single sample also the norm weights' gradients; into `totals`, when there is
// one); blockIdx.y == samples: the norm weights' gradients, over all samples and chunks.
__global__ void __launch_bounds__(512) resnorm_final_kernel(const Args a, const lq_residual_norm_grads g, int chunks,
                                                            const float* __restrict__ part, float* __restrict__ totals, int first) {
    __shared__ float sm[3][16][33];
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, h = (int)a.h;
    const int j = blockIdx.x * 32 + lane;
    const int64_t b = blockIdx.y + first;
    const bool weights = b == a.samples;
    float s[3] = {0.f, 0.f, 0.f};
    if (j < h) {
        if (!weights) {
#pragma unroll 4
            for (int c = grp; c < chunks; c += 16) {
                const float* p = part + (b * chunks + c) * 3 * h + j;
                s[0] += __ldg(p), s[1] += __ldg(p + h), s[2] += __ldg(p + 2 * h);
            }
        } else {
#pragma unroll 4
            for (int c = grp; c < (int)a.samples * chunks; c += 16) {
                const int bc = c / chunks;
                const float* p = part + (int64_t)c * 3 * h + j;
                s[0] = fmaf(__ldg(p), 1.f + mod_at(a.scale, a.mod_f32, bc * a.scale_sample + j), s[0]);
                if (a.y) s[2] = fmaf(__ldg(p + 2 * h), mod_at(a.gate, a.mod_f32, bc * a.gate_sample + j), s[2]);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) sm[k][grp][lane] = s[k];
    __syncthreads();
    if (grp >= 3 || j >= h) return;
    float v = 0.f;  // warp k adds up sum k
#pragma unroll
    for (int q = 0; q < 16; ++q) v += sm[grp][q][lane];
    if (weights) {
        if (grp == 0 && g.dweight) g.dweight[j] = v;
        if (grp == 2 && g.dpost_weight) g.dpost_weight[j] = v;
        return;
    }
    if (totals) totals[(b * 3 + grp) * h + j] = v;
    if (a.samples == 1) {
        if (grp == 0 && g.dweight) g.dweight[j] = v * (1.f + mod_at(a.scale, a.mod_f32, j));
        if (grp == 2 && g.dpost_weight) g.dpost_weight[j] = v * mod_at(a.gate, a.mod_f32, j);
    }
    if (grp == 0 && g.dscale) st_mod(g.dscale, a.mod_f32, b * h + j, v * (a.weight ? 1.f + a.weight[j] : 1.f));
    if (grp == 1 && g.dshift) st_mod(g.dshift, a.mod_f32, b * h + j, v);
    if (grp == 2 && g.dgate) st_mod(g.dgate, a.mod_f32, b * h + j, v * (a.post_weight ? 1.f + a.post_weight[j] : 1.f));
}

// ---- host ---------------------------------------------------------------------------------------

constexpr int64_t kMaxH = 16384;  // 1024 threads x 16 elements
static_assert(sizeof(float[2][2][kMaxWarps]) + sizeof(uint64_t[kMaxStages]) + 16 <= kRingStatic, "a ring block's own shared memory");

inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

bool vectors_ok(const Args& a, const lq_residual_norm_grads* g) {
    const int es = a.dtype == LQ_F32 ? 4 : 2, ms = a.mod_f32 ? 4 : 2;
    const int64_t v = 16 / es;
    bool ok = a.h % 8 == 0 && al16(a.x) && a.x_sample % v == 0 && a.x_token % v == 0;
    ok = ok && al16(a.shift) && al16(a.scale) && (a.shift_sample * ms) % 16 == 0 && (a.scale_sample * ms) % 16 == 0;
    ok = ok && al16(a.weight) && al16(a.post_weight) && al16(a.z) && al16(a.r);
    if (a.y)
        ok = ok && al16(a.y) && a.y_sample % v == 0 && a.y_token % v == 0 && al16(a.gate) && (a.gate_sample * ms) % 16 == 0;
    if (g) {
        ok = ok && al16(g->dx) && al16(g->dy);
        if (g->dz) ok = ok && al16(g->dz) && g->dz_sample % v == 0 && g->dz_token % v == 0;
        if (g->dr) ok = ok && al16(g->dr) && g->dr_sample % v == 0 && g->dr_token % v == 0;
    }
    return ok;
}

// Three partial rows a chunk, then three totals a sample.
size_t ws_bytes_of(int64_t samples, int64_t chunks, int64_t h) { return (size_t)samples * (chunks + 1) * 3 * h * sizeof(float); }

void check(const Args& a) {
    LQ_CHECK_ARG(a.dtype == LQ_F32 || a.dtype == LQ_BF16, "dtype must be LQ_F32 or LQ_BF16");
    LQ_CHECK_ARG(a.samples >= 0 && a.tokens >= 0, "samples and tokens must be >= 0");
    LQ_CHECK_ARG(a.h >= 1 && a.h <= kMaxH, "h must be in [1, 16384]");
    LQ_CHECK_ARG(a.samples < (int64_t)1 << 31 && a.tokens < (int64_t)1 << 31 && a.samples * a.tokens < (int64_t)1 << 31,
                 "samples * tokens must be below 2^31");
}

void check_pointers(const Args& a) {  // of a call with rows: an empty tensor has no address
    LQ_CHECK_ARG(a.x && a.shift && a.scale, "NULL argument");
    LQ_CHECK_ARG(!a.y || a.gate, "gate is needed with y");
    LQ_CHECK_ARG(!a.post_weight || a.y, "post_weight normalises y: y is NULL");
}

template <typename F>
int guarded_call(F&& f) {
    try {
        f();
        lq_set_last_error("");
        return LQ_OK;
    } catch (const LqError& e) {
        lq_set_last_error(e.what());
        return e.status;
    } catch (const std::exception& e) {
        lq_set_last_error(e.what());
        return LQ_ERR_INVALID;
    }
}

int current_device() {
    int dev = 0;
    LQ_CUDA(cudaGetDevice(&dev));
    return dev;
}

// Each kernel is allowed its largest ring once per device (the attribute is a driver call).
template <auto KERN, typename... A>
void launch_ring(int dev, unsigned grid, int threads, size_t smem, cudaStream_t st, A... args) {
    static std::atomic<uint64_t> allowed{0};
    const uint64_t bit = 1ull << (dev & 63);
    if (!(allowed.load() & bit)) {
        LQ_CUDA(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingBytes));
        allowed.fetch_or(bit);
    }
    KERN<<<grid, threads, smem, st>>>(args...);
}

#define LQ_RING_FWD(T, P, Y, ...)                                                                                          \
    do {                                                                                                                   \
        if (threads <= 64) launch_ring<resnorm_fwd_ring_kernel<T, P, Y, 64, 16>>(dev, grid, threads, smem, st, __VA_ARGS__);     \
        else if (threads <= 256) launch_ring<resnorm_fwd_ring_kernel<T, P, Y, 256, 4>>(dev, grid, threads, smem, st, __VA_ARGS__); \
        else if (threads <= 512) launch_ring<resnorm_fwd_ring_kernel<T, P, Y, 512, 2>>(dev, grid, threads, smem, st, __VA_ARGS__); \
        else if (threads <= 768) launch_ring<resnorm_fwd_ring_kernel<T, P, Y, 768, 1>>(dev, grid, threads, smem, st, __VA_ARGS__); \
        else launch_ring<resnorm_fwd_ring_kernel<T, P, Y, 1024, 1>>(dev, grid, threads, smem, st, __VA_ARGS__);                  \
    } while (0)
#define LQ_RING_BWD(T, P, Y, ...)                                                                                          \
    do {                                                                                                                   \
        if (threads <= 64) launch_ring<resnorm_bwd_ring_kernel<T, P, Y, 64, 12>>(dev, grid, threads, smem, st, __VA_ARGS__);     \
        else if (threads <= 256) launch_ring<resnorm_bwd_ring_kernel<T, P, Y, 256, 3>>(dev, grid, threads, smem, st, __VA_ARGS__); \
        else if (threads <= 384) launch_ring<resnorm_bwd_ring_kernel<T, P, Y, 384, 2>>(dev, grid, threads, smem, st, __VA_ARGS__); \
        else if (threads <= 512) launch_ring<resnorm_bwd_ring_kernel<T, P, Y, 512, 1>>(dev, grid, threads, smem, st, __VA_ARGS__); \
        else if (threads <= 768) launch_ring<resnorm_bwd_ring_kernel<T, P, Y, 768, 1>>(dev, grid, threads, smem, st, __VA_ARGS__); \
        else launch_ring<resnorm_bwd_ring_kernel<T, P, Y, 1024, 1>>(dev, grid, threads, smem, st, __VA_ARGS__);                  \
    } while (0)
#define LQ_RING(DIR, T, ...)                                          \
    do {                                                             \
        if (a.post_weight && a.layer) DIR(T, true, true, __VA_ARGS__); \
        else if (a.post_weight) DIR(T, true, false, __VA_ARGS__);      \
        else if (a.layer) DIR(T, false, true, __VA_ARGS__);            \
        else DIR(T, false, false, __VA_ARGS__);                        \
    } while (0)
#define LQ_SCALAR_T(KERN, T, ...)                                                              \
    do {                                                                                      \
        if (a.h <= 4096) KERN<T, 8, 512><<<grid, threads, 0, st>>>(__VA_ARGS__);               \
        else if (a.h <= 8192) KERN<T, 8, 1024><<<grid, threads, 0, st>>>(__VA_ARGS__);         \
        else KERN<T, 16, 1024><<<grid, threads, 0, st>>>(__VA_ARGS__);                         \
    } while (0)
#define LQ_SCALAR(KERN, ...)                                                                  \
    do {                                                                                      \
        const int threads = scalar_threads(a.h);                                              \
        if (a.dtype == LQ_F32) LQ_SCALAR_T(KERN, float, __VA_ARGS__);                          \
        else LQ_SCALAR_T(KERN, __nv_bfloat16, __VA_ARGS__);                                    \
    } while (0)

constexpr int64_t kRingMaxH = 8192;  // 1024 threads x 8 columns

void forward(const Args& a, int dev, cudaStream_t st) {
    const int inputs = a.y ? 2 : 1, stages = a.h <= kRingMaxH && vectors_ok(a, nullptr) ? stages_of(a.h, a.dtype == LQ_F32 ? 4 : 2, inputs, false) : 0;
    const int sms = lq_tc_sm_count(dev);
    const int chunks = chunks_of(a.samples, a.tokens, (int64_t)sms * (stages ? blocks_per_sm(a.h, false) : scalar_blocks_per_sm(a.h, false)), sms, false);
    const int64_t per = (a.tokens + chunks - 1) / chunks;
    LQ_CHECK_ARG(a.samples * chunks < (int64_t)1 << 31, "too many samples");
    const unsigned grid = (unsigned)(a.samples * chunks);
    LqProf prof(LQ_K_PREP, st);
    if (stages) {
        const int threads = threads_of(a.h);
        const size_t smem = (size_t)std::min<int64_t>(stages, per) * inputs * a.h * (a.dtype == LQ_F32 ? 4 : 2);
        int* status = lq_tc_status_word(dev);
        if (a.dtype == LQ_F32) LQ_RING(LQ_RING_FWD, float, a, chunks, per, stages, status);
        else LQ_RING(LQ_RING_FWD, __nv_bfloat16, a, chunks, per, stages, status);
    } else {
        LQ_SCALAR(resnorm_fwd_kernel, a, chunks, per);
    }
    LQ_CUDA(cudaGetLastError());
}

// Most chunks of the backward, whichever kernel the rows take: what the workspace is sized for.
int most_chunks(int64_t samples, int64_t tokens, int64_t h, int sms) {
    return std::max(chunks_of(samples, tokens, (int64_t)sms * blocks_per_sm(h, true), sms, true),
                    chunks_of(samples, tokens, (int64_t)sms * scalar_blocks_per_sm(h, true), sms, true));
}

// Returns the chunks that it used.
int backward(const Args& a, const lq_residual_norm_grads& g, float* part, int dev, cudaStream_t st) {
    const int inputs = 1 + (a.y ? 1 : 0) + (g.dz ? 1 : 0) + (g.dr ? 1 : 0);
    const int stages = a.h <= kRingMaxH && vectors_ok(a, &g) ? stages_of(a.h, a.dtype == LQ_F32 ? 4 : 2, inputs, true) : 0;
    const int sms = lq_tc_sm_count(dev);
    const int chunks = chunks_of(a.samples, a.tokens, (int64_t)sms * (stages ? blocks_per_sm(a.h, true) : scalar_blocks_per_sm(a.h, true)), sms, true);
    const int64_t per = (a.tokens + chunks - 1) / chunks;
    const unsigned grid = (unsigned)(a.samples * chunks);
    LqProf prof(LQ_K_PREP, st);
    if (stages) {
        const int threads = threads_of(a.h);
        const size_t smem = (size_t)std::min<int64_t>(stages, per) * inputs * a.h * (a.dtype == LQ_F32 ? 4 : 2);
        int* status = lq_tc_status_word(dev);
        if (a.dtype == LQ_F32) LQ_RING(LQ_RING_BWD, float, a, g, chunks, per, stages, part, status);
        else LQ_RING(LQ_RING_BWD, __nv_bfloat16, a, g, chunks, per, stages, part, status);
    } else {
        LQ_SCALAR(resnorm_bwd_kernel, a, g, chunks, per, part);
    }
    LQ_CUDA(cudaGetLastError());
    return chunks;
}

}  // namespace

extern "C" {

int lq_residual_norm_fwd(const lq_residual_norm_args* args, void* stream) {
    return guarded_call([&] {
        LQ_CHECK_ARG(args != nullptr, "NULL argument");
        const Args a = *args;
        check(a);
        if (a.samples * a.tokens == 0) return;
        check_pointers(a);
        LQ_CHECK_ARG(a.z != nullptr, "NULL argument");
        LQ_CHECK_ARG(!a.rstd || !a.layer || a.mean, "mean must be given with rstd for the layer norm");
        LQ_CHECK_ARG(!a.rstd || !a.post_weight || a.post_rstd, "post_rstd must be given with rstd and post_weight");
        forward(a, current_device(), (cudaStream_t)stream);
    });
}

size_t lq_residual_norm_workspace_bytes(int64_t samples, int64_t tokens, int64_t h) {
    if (samples < 1 || tokens < 1 || h < 1 || h > kMaxH) return 0;
    size_t n = 0;
    if (guarded_call([&] { n = ws_bytes_of(samples, most_chunks(samples, tokens, h, lq_tc_sm_count(current_device())), h); }) != LQ_OK) return 0;
    return n;
}

int lq_residual_norm_bwd(const lq_residual_norm_args* args, const lq_residual_norm_grads* grads, void* ws, size_t ws_bytes,
                         void* stream) {
    return guarded_call([&] {
        LQ_CHECK_ARG(args != nullptr && grads != nullptr, "NULL argument");
        const Args a = *args;
        const lq_residual_norm_grads g = *grads;
        check(a);
        cudaStream_t st = (cudaStream_t)stream;
        const bool sums = g.dshift || g.dscale || g.dgate || g.dweight || g.dpost_weight;
        if (a.samples * a.tokens == 0) {  // no rows: the sums are zero
            const size_t mods = (size_t)a.samples * a.h * (a.mod_f32 ? 4 : 2), ws_ = (size_t)a.h * 4;
            for (void* p : {g.dshift, g.dscale, g.dgate})
                if (p && mods) LQ_CUDA(cudaMemsetAsync(p, 0, mods, st));
            for (float* p : {g.dweight, g.dpost_weight})
                if (p) LQ_CUDA(cudaMemsetAsync(p, 0, ws_, st));
            return;
        }
        check_pointers(a);
        LQ_CHECK_ARG(a.y || (!g.dy && !g.dgate), "dy and dgate need y");
        LQ_CHECK_ARG(!g.dpost_weight || a.post_weight, "dpost_weight needs post_weight");
        LQ_CHECK_ARG(!g.dweight || a.weight, "dweight needs weight");
        LQ_CHECK_ARG(a.rstd && (!a.layer || a.mean) && (!a.post_weight || a.post_rstd), "the forward's statistics are needed");
        const int dev = current_device(), most = most_chunks(a.samples, a.tokens, a.h, lq_tc_sm_count(dev));
        LQ_CHECK_ARG(a.samples * most < (int64_t)1 << 31, "too many samples");
        if (sums && (!ws || ws_bytes < ws_bytes_of(a.samples, most, a.h)))
            throw LqError(LQ_ERR_WORKSPACE, "workspace too small for the residual-norm backward");
        LQ_CHECK_ARG(!sums || al16(ws), "the workspace must be 16-byte aligned");
        float* part = sums ? (float*)ws : nullptr;
        const int chunks = backward(a, g, part, dev, st);
        if (sums) {
            LqProf prof(LQ_K_REDUCE, st);
            const unsigned cols = (unsigned)((a.h + 31) / 32);
            const bool weights = a.samples > 1 && (g.dweight || g.dpost_weight);
            // the weights' sums over many partial rows would be one block's work per 32 columns: over the samples' totals instead
            float* totals = weights && a.samples * chunks > 64 ? part + (size_t)a.samples * chunks * 3 * a.h : nullptr;
            const int64_t places = a.samples + (weights && !totals ? 1 : 0);
            for (int64_t first = 0; first < places; first += 65535)  // the grid's second axis
                resnorm_final_kernel<<<dim3(cols, (unsigned)std::min<int64_t>(65535, places - first)), 512, 0, st>>>(a, g, chunks, part, totals, (int)first);
            if (totals) resnorm_final_kernel<<<dim3(cols, 1), 512, 0, st>>>(a, g, 1, totals, nullptr, (int)a.samples);
            LQ_CUDA(cudaGetLastError());
        }
    });
}

}  // extern "C"
