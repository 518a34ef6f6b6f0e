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
// byte more than reading r and keeps rh at f32 accuracy.
#include <algorithm>

#include <cuda_bf16.h>

#include "lq_internal.cuh"
#include "lq_prof.cuh"
#include "lq_tc.cuh"

namespace {

typedef lq_residual_norm_args Args;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// VEC elements of type T as f32, from an address aligned to the vector.  The token-shaped streams are read
// past L1 (each byte is used once), so that the modulation vectors stay in it.
template <typename T, int VEC>
struct Io;
template <typename T>
struct Io<T, 1> {
    static __device__ __forceinline__ void ld(const T* p, float (&f)[1]) { f[0] = to_f(*p); }
    static __device__ __forceinline__ void st(T* p, const float (&f)[1]) { *p = (T)f[0]; }
};
__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
template <>
struct Io<float, 4> {
    static __device__ __forceinline__ void ld(const float* p, float (&f)[4]) {
        const uint4 v = ld_stream(p);
        f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ void st(float* p, const float (&f)[4]) {
        *(float4*)p = make_float4(f[0], f[1], f[2], f[3]);
    }
};
template <>
struct Io<__nv_bfloat16, 8> {
    static __device__ __forceinline__ void ld(const __nv_bfloat16* p, float (&f)[8]) {
        const uint4 v = ld_stream(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ void st(__nv_bfloat16* p, const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *(const uint32_t*)&h;
        }
        *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// VEC values of a modulation vector (f32 or bf16 by the call) starting at element `i` of `p`.
template <int VEC>
__device__ __forceinline__ void ld_mod(const void* p, int f32, int64_t i, float (&f)[VEC]) {
    if (VEC == 1) {
        f[0] = f32 ? ((const float*)p)[i] : to_f(((const __nv_bfloat16*)p)[i]);
    } else if (f32) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const float4 v = *(const float4*)((const float*)p + i + e);
            f[e] = v.x, f[e + 1] = v.y, f[e + 2] = v.z, f[e + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const uint2 v = *(const uint2*)((const __nv_bfloat16*)p + i + e);
            f[e] = __uint_as_float(v.x << 16), f[e + 1] = __uint_as_float(v.x & 0xFFFF0000u);
            f[e + 2] = __uint_as_float(v.y << 16), f[e + 3] = __uint_as_float(v.y & 0xFFFF0000u);
        }
    }
}

// Sums of NV values over the threads of a block, in a fixed order; `buf` alternates between two areas,
// so that one barrier per reduction is enough (whoever writes an area again has passed the barrier of the
// reduction between).
constexpr int kMaxWarps = 16;
template <int NV>
__device__ __forceinline__ void block_sum(float (&v)[NV], float (*area)[kMaxWarps][2], int& buf) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1)
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < NV; ++k) area[buf][threadIdx.x >> 5][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float s = 0.f;
        for (int w = 0; w < warps; ++w) s += area[buf][w][k];
        v[k] = s;
    }
    buf ^= 1;
}

// One block per row; thread t owns the vectors t, t + blockDim, ... of the row and keeps r in registers
// between the statistics and the output.
template <typename T, int VEC, int VPT>
__global__ void __launch_bounds__(512) resnorm_fwd_kernel(const Args a) {
    __shared__ float area[2][kMaxWarps][2];
    int buf = 0;
    const int64_t row = blockIdx.x, b = row / a.tokens, t = row - b * a.tokens;
    const int h = (int)a.h, nvec = h / VEC;
    const float inv_h = 1.f / (float)h;
    const T* xr = (const T*)a.x + b * a.x_sample + t * a.x_token;
    float r[VPT][VEC];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[i][e] = 0.f;
        if (c < nvec) Io<T, VEC>::ld(xr + c * VEC, r[i]);
    }
    if (a.y) {
        const T* yr = (const T*)a.y + b * a.y_sample + t * a.y_token;
        float y[VPT][VEC];
        float q = 1.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[i][e] = 0.f;
            if (c < nvec) Io<T, VEC>::ld(yr + c * VEC, y[i]);
        }
        if (a.post_weight) {
            float v[1] = {0.f};
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[0] = fmaf(y[i][e], y[i][e], v[0]);
            block_sum<1>(v, area, buf);
            q = 1.f / sqrtf(v[0] * inv_h + a.eps);
            if (threadIdx.x == 0 && a.post_rstd) a.post_rstd[row] = q;
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c < nvec) {
                float g[VEC], pw[VEC];
                ld_mod<VEC>(a.gate, a.mod_f32, b * a.gate_sample + c * VEC, g);
                if (a.post_weight) ld_mod<VEC>(a.post_weight, 1, c * VEC, pw);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float u = a.post_weight ? y[i][e] * q * (1.f + pw[e]) : y[i][e];
                    r[i][e] = fmaf(g[e], u, a.alpha * r[i][e]);
                }
                if (a.r) Io<T, VEC>::st((T*)a.r + row * h + c * VEC, r[i]);
            }
        }
    }
    float mu = 0.f;
    if (a.layer) {
        float v[1] = {0.f};
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[0] += r[i][e];
        block_sum<1>(v, area, buf);
        mu = v[0] * inv_h;
    }
    float v[1] = {0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        if (threadIdx.x + i * blockDim.x < nvec)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[0] = fmaf(r[i][e] - mu, r[i][e] - mu, v[0]);
    block_sum<1>(v, area, buf);
    const float s = 1.f / sqrtf(v[0] * inv_h + a.eps);
    if (threadIdx.x == 0 && a.rstd) {
        a.rstd[row] = s;
        if (a.layer) a.mean[row] = mu;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        if (c < nvec) {
            float sh[VEC], sc[VEC], w[VEC];
            ld_mod<VEC>(a.shift, a.mod_f32, b * a.shift_sample + c * VEC, sh);
            ld_mod<VEC>(a.scale, a.mod_f32, b * a.scale_sample + c * VEC, sc);
            if (a.weight) ld_mod<VEC>(a.weight, 1, c * VEC, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float o = (r[i][e] - mu) * s;
                if (a.weight) o *= 1.f + w[e];
                sh[e] = fmaf(o, 1.f + sc[e], sh[e]);
            }
            Io<T, VEC>::st((T*)a.z + row * h + c * VEC, sh);
        }
    }
}

// One block per chunk of consecutive rows of one sample; thread t owns fixed columns, so that S, T and G
// stay in registers over the chunk and leave as one partial row each.
template <typename T, int VEC, int VPT>
__global__ void __launch_bounds__(512) resnorm_bwd_kernel(const Args a, const lq_residual_norm_grads g, int chunks,
                                                          int64_t rows_per_chunk, float* __restrict__ part) {
    __shared__ float area[2][kMaxWarps][2];
    int buf = 0;
    const int64_t b = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x - b * chunks);
    const int64_t t0 = chunk * rows_per_chunk, t1 = min(a.tokens, t0 + rows_per_chunk);
    const int h = (int)a.h, nvec = h / VEC;
    const float inv_h = 1.f / (float)h;
    float S[VPT][VEC], D1[VPT][VEC], G[VPT][VEC];
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) S[i][e] = D1[i][e] = G[i][e] = 0.f;

    for (int64_t t = t0; t < t1; ++t) {
        const int64_t row = b * a.tokens + t;
        const float s = a.rstd[row], mu = a.layer ? a.mean[row] : 0.f, q = a.post_weight ? a.post_rstd[row] : 1.f;
        float rh[VPT][VEC], gz[VPT][VEC], yh[VPT][VEC];
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
            for (int e = 0; e < VEC; ++e) rh[i][e] = gz[i][e] = yh[i][e] = 0.f;
            if (c >= nvec) continue;
            Io<T, VEC>::ld((const T*)a.x + b * a.x_sample + t * a.x_token + c * VEC, rh[i]);
            if (g.dz) Io<T, VEC>::ld((const T*)g.dz + b * g.dz_sample + t * g.dz_token + c * VEC, gz[i]);
            if (a.y) {
                float gt[VEC], pw[VEC];
                Io<T, VEC>::ld((const T*)a.y + b * a.y_sample + t * a.y_token + c * VEC, yh[i]);
                ld_mod<VEC>(a.gate, a.mod_f32, b * a.gate_sample + c * VEC, gt);
                if (a.post_weight) ld_mod<VEC>(a.post_weight, 1, c * VEC, pw);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    float u = yh[i][e];
                    if (a.post_weight) {
                        yh[i][e] *= q;
                        u = yh[i][e] * (1.f + pw[e]);
                    }
                    rh[i][e] = fmaf(gt[e], u, a.alpha * rh[i][e]);
                }
            }
            float sc[VEC], w[VEC];
            ld_mod<VEC>(a.scale, a.mod_f32, b * a.scale_sample + c * VEC, sc);
            if (a.weight) ld_mod<VEC>(a.weight, 1, c * VEC, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                rh[i][e] = (rh[i][e] - mu) * s;
                S[i][e] = fmaf(gz[i][e], rh[i][e], S[i][e]);
                D1[i][e] += gz[i][e];
                gz[i][e] *= 1.f + sc[e];
                if (a.weight) gz[i][e] *= 1.f + w[e];
                v[0] = fmaf(gz[i][e], rh[i][e], v[0]);
                v[1] += gz[i][e];
            }
        }
        block_sum<2>(v, area, buf);
        const float c1 = v[0] * inv_h, c0 = a.layer ? v[1] * inv_h : 0.f;
        float p[1] = {0.f};
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c >= nvec) continue;
            float d[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] = 0.f;
            if (g.dr) Io<T, VEC>::ld((const T*)g.dr + b * g.dr_sample + t * g.dr_token + c * VEC, d);
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] = fmaf(s, gz[i][e] - c0 - rh[i][e] * c1, d[e]);
            if (a.y) {
                float gt[VEC], pw[VEC];
                ld_mod<VEC>(a.gate, a.mod_f32, b * a.gate_sample + c * VEC, gt);
                if (a.post_weight) ld_mod<VEC>(a.post_weight, 1, c * VEC, pw);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    G[i][e] = fmaf(d[e], yh[i][e], G[i][e]);
                    gz[i][e] = gt[e] * d[e];  // du
                    if (a.post_weight) {
                        gz[i][e] *= 1.f + pw[e];
                        p[0] = fmaf(gz[i][e], yh[i][e], p[0]);
                    }
                    d[e] *= a.alpha;
                }
            }
            if (g.dx) Io<T, VEC>::st((T*)g.dx + row * h + c * VEC, d);
        }
        if (!a.y || !g.dy) continue;
        if (a.post_weight) block_sum<1>(p, area, buf);
        const float pm = p[0] * inv_h;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c >= nvec) continue;
            if (a.post_weight)
#pragma unroll
                for (int e = 0; e < VEC; ++e) gz[i][e] = q * (gz[i][e] - yh[i][e] * pm);
            Io<T, VEC>::st((T*)g.dy + row * h + c * VEC, gz[i]);
        }
    }
    if (!part) return;
    float* dst = part + (int64_t)blockIdx.x * 3 * h;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        if (c >= nvec) continue;
        Io<float, VEC == 1 ? 1 : 4> io;
#pragma unroll
        for (int e = 0; e < VEC; e += (VEC == 1 ? 1 : 4)) {
            typedef float Q[VEC == 1 ? 1 : 4];
            io.st(dst + c * VEC + e, *(const Q*)&S[i][e]);
            io.st(dst + h + c * VEC + e, *(const Q*)&D1[i][e]);
            io.st(dst + 2 * h + c * VEC + e, *(const Q*)&G[i][e]);
        }
    }
}

__device__ __forceinline__ void st_mod(void* p, int f32, int64_t i, float v) {
    if (f32) ((float*)p)[i] = v;
    else ((__nv_bfloat16*)p)[i] = __float2bfloat16(v);
}

// Sums the partial rows in a fixed order.  Block = 32 columns x 8 ranges of chunks; one sample per blockIdx.y,
// or (gridDim.y == 1) all samples one after the other when a norm weight's gradient sums over them too.
__global__ void __launch_bounds__(256) resnorm_final_kernel(const Args a, const lq_residual_norm_grads g, int chunks,
                                                            const float* __restrict__ part) {
    __shared__ float sm[3][8][33];
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, h = (int)a.h;
    const int j = blockIdx.x * 32 + lane;
    float dw = 0.f, dpw = 0.f;
    for (int64_t b = blockIdx.y; b < a.samples; b += gridDim.y) {
        float s[3] = {0.f, 0.f, 0.f};
        if (j < h)
            for (int c = grp; c < chunks; c += 8)
#pragma unroll
                for (int k = 0; k < 3; ++k) s[k] += part[((b * chunks + c) * 3 + k) * h + j];
        __syncthreads();  // the sums of the sample before have been read
#pragma unroll
        for (int k = 0; k < 3; ++k) sm[k][grp][lane] = s[k];
        __syncthreads();
        if (grp == 0 && j < h) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                s[k] = 0.f;
#pragma unroll
                for (int q = 0; q < 8; ++q) s[k] += sm[k][q][lane];
            }
            float sc[1], gt[1] = {0.f}, w = 0.f, pw = 0.f;
            ld_mod<1>(a.scale, a.mod_f32, b * a.scale_sample + j, sc);
            if (a.y) ld_mod<1>(a.gate, a.mod_f32, b * a.gate_sample + j, gt);
            if (a.weight) w = a.weight[j];
            if (a.post_weight) pw = a.post_weight[j];
            if (g.dscale) st_mod(g.dscale, a.mod_f32, b * h + j, s[0] * (1.f + w));
            if (g.dshift) st_mod(g.dshift, a.mod_f32, b * h + j, s[1]);
            if (g.dgate) st_mod(g.dgate, a.mod_f32, b * h + j, s[2] * (1.f + pw));
            dw = fmaf(s[0], 1.f + sc[0], dw);
            dpw = fmaf(s[2], gt[0], dpw);
        }
    }
    if (grp == 0 && j < h) {
        if (g.dweight) g.dweight[j] = dw;
        if (g.dpost_weight) g.dpost_weight[j] = dpw;
    }
}

// ---- host ---------------------------------------------------------------------------------------

constexpr int64_t kMaxH = 16384;  // 512 threads x 32 elements

struct Shape {
    int vec, ept, threads;  // elements per access, elements per thread, threads of a block
};

// 16-byte accesses need every row and vector to start on 16 bytes; otherwise single elements.  A thread holds
// 8 elements up to 4096 columns, then 16, then 32, in blocks of at most 512 threads (128 registers each).
Shape shape_of(int64_t h, int dtype, bool vectors) {
    Shape s;
    s.vec = vectors ? (dtype == LQ_F32 ? 4 : 8) : 1;
    s.ept = h <= 4096 ? 8 : (h <= 8192 ? 16 : 32);
    const int64_t per = (h / s.vec + s.ept / s.vec - 1) / (s.ept / s.vec);
    s.threads = (int)((per + 31) / 32 * 32);
    return s;
}

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

// Chunks of one sample: about as many blocks as fit the machine at 1024 threads an SM, each with at least one row.
int chunks_of(int64_t samples, int64_t tokens, int64_t h, int sms) {
    const int64_t threads = (h / 8 + 31) / 32 * 32;  // of the vector path up to 4096 columns; the rule only has to be fixed
    const int64_t blocks = (int64_t)sms * std::max<int64_t>(1, 1024 / std::min<int64_t>(512, std::max<int64_t>(32, threads)));
    return (int)std::max<int64_t>(1, std::min<int64_t>(tokens, (blocks + samples - 1) / samples));
}

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

int current_sms() {
    int dev = 0;
    LQ_CUDA(cudaGetDevice(&dev));
    return lq_tc_sm_count(dev);
}

template <typename T, int VEC, int EPT>
void launch_fwd(const Args& a, const Shape& s, cudaStream_t st) {
    resnorm_fwd_kernel<T, VEC, EPT / VEC><<<(unsigned)(a.samples * a.tokens), s.threads, 0, st>>>(a);
}
template <typename T, int VEC, int EPT>
void launch_bwd(const Args& a, const lq_residual_norm_grads& g, const Shape& s, int chunks, float* part, cudaStream_t st) {
    const int64_t per = (a.tokens + chunks - 1) / chunks;
    resnorm_bwd_kernel<T, VEC, EPT / VEC><<<(unsigned)(a.samples * chunks), s.threads, 0, st>>>(a, g, chunks, per, part);
}

#define LQ_RESNORM_EPT(F, T, V, ...)                                             \
    do {                                                                         \
        if (s.ept == 8) F<T, V, 8>(__VA_ARGS__);                                 \
        else if (s.ept == 16) F<T, V, 16>(__VA_ARGS__);                          \
        else F<T, V, 32>(__VA_ARGS__);                                           \
    } while (0)
#define LQ_RESNORM_DISPATCH(F, ...)                                              \
    do {                                                                         \
        if (a.dtype == LQ_F32 && s.vec == 4) LQ_RESNORM_EPT(F, float, 4, __VA_ARGS__);          \
        else if (a.dtype == LQ_F32) LQ_RESNORM_EPT(F, float, 1, __VA_ARGS__);                   \
        else if (s.vec == 8) LQ_RESNORM_EPT(F, __nv_bfloat16, 8, __VA_ARGS__);                  \
        else LQ_RESNORM_EPT(F, __nv_bfloat16, 1, __VA_ARGS__);                                  \
    } while (0)

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
        cudaStream_t st = (cudaStream_t)stream;
        const Shape s = shape_of(a.h, a.dtype, vectors_ok(a, nullptr));
        LqProf prof(LQ_K_PREP, st);
        LQ_RESNORM_DISPATCH(launch_fwd, a, s, st);
        LQ_CUDA(cudaGetLastError());
    });
}

size_t lq_residual_norm_workspace_bytes(int64_t samples, int64_t tokens, int64_t h) {
    if (samples < 1 || tokens < 1 || h < 1 || h > kMaxH) return 0;
    size_t n = 0;
    if (guarded_call([&] { n = (size_t)samples * chunks_of(samples, tokens, h, current_sms()) * 3 * h * sizeof(float); }) != LQ_OK)
        return 0;
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
        const int chunks = chunks_of(a.samples, a.tokens, a.h, current_sms());
        LQ_CHECK_ARG(a.samples * chunks < (int64_t)1 << 31, "too many samples");
        if (sums && (!ws || ws_bytes < (size_t)a.samples * chunks * 3 * a.h * sizeof(float)))
            throw LqError(LQ_ERR_WORKSPACE, "workspace too small for the residual-norm backward");
        LQ_CHECK_ARG(!sums || al16(ws), "the workspace must be 16-byte aligned");
        const Shape s = shape_of(a.h, a.dtype, vectors_ok(a, &g));
        float* part = sums ? (float*)ws : nullptr;
        {
            LqProf prof(LQ_K_PREP, st);
            LQ_RESNORM_DISPATCH(launch_bwd, a, g, s, chunks, part, st);
            LQ_CUDA(cudaGetLastError());
        }
        if (sums) {
            LqProf prof(LQ_K_REDUCE, st);
            const bool over_samples = g.dweight || g.dpost_weight;
            const dim3 grid((unsigned)((a.h + 31) / 32), over_samples ? 1u : (unsigned)std::min<int64_t>(a.samples, 65535));
            resnorm_final_kernel<<<grid, 256, 0, st>>>(a, g, chunks, part);
            LQ_CUDA(cudaGetLastError());
        }
    });
}

}  // extern "C"
