// The 2-norm of many gradient tensors taken as one vector, and clipping by it:
//
//   norm = grad_scale * sqrt(sum over all tensors and elements of g^2)
//   coef = min(1, max_norm / (norm + 1e-6)),   out = g * (grad_scale * coef)
//
// Squares and sums are f64: the square of an f32 is exact there and cannot overflow, so the norm is right
// over the whole f32 range and is finite exactly when every gradient is (the finite check of
// crates/loractl-core/src/diffusion_trainer.rs:1708-1725 comes with it).
//
// HBM-bound: one read of the gradients for the norm, a second read and a write for the clip.  The tensors
// are cut into chunks of 32 KB; a chunk belongs to one tensor and is read by one block with 16-byte loads,
// eight of them in flight per thread.  The list of tensors travels in the kernel's parameters, so a call
// copies nothing to the device and can be captured.  Every block leaves one f64 partial sum; the second launch
// adds them in a fixed order (each of its blocks for itself when it also scales), so there are no atomics and two
// runs are bit-identical.  The scaling launch walks the chunks backwards: what the first pass read last is
// still in the L2.
// 392 f32 tensors of 193 MB: 30.6 us for the sums (6.3 TB/s, 96 % of the measured copy rate) and 2.7 us for the norm;
// 126 tensors of both types, 70 MB, to outputs that start anywhere: 14.2 us and 25.6 us.
#include <algorithm>

#include <cuda_bf16.h>

#include "lq_internal.cuh"
#include "lq_prof.cuh"
#include "lq_tc.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kChunkBytes = 32768;
constexpr int kBlocksPerSm = 8;

// One launch's tensors; `first[i]` is the first chunk of tensor i within the launch.
template <int CAP>
struct List {
    const void* g[CAP];
    void* out[CAP];
    int64_t n[CAP];  // elements; negative for bf16
    int first[CAP + 1];
    int count;
};

template <int CAP>
__device__ __forceinline__ int tensor_of(const List<CAP>& l, int chunk) {
    int lo = 0, hi = l.count;  // first[lo] <= chunk < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (l.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ double sq(float v) {
    const double d = (double)v;
    return d * d;
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ double block_sum(double v, double* sm) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) v += sm[w];
    __syncthreads();
    return v;
}

// Single elements: the end of a tensor, or all of a chunk where source and output do not both start on 16 bytes.
// Sixteen are read before the first is used (source and output may share memory, so the compiler keeps the order that
// it is given).
constexpr int kBatch = 16;
template <typename T>
__device__ __forceinline__ double sq_elements(const T* src, int from, int n) {
    double s = 0.0;
    for (int k = from + threadIdx.x; k < n; k += kBatch * kThreads) {
        T v[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) v[e] = k + e * kThreads < n ? src[k + e * kThreads] : T(0.f);
#pragma unroll
        for (int e = 0; e < kBatch; ++e) s += sq((float)v[e]);
    }
    return s;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads) grad_sq_kernel(const __grid_constant__ List<CAP> l, double* __restrict__ part) {
    __shared__ double sm[kThreads / 32];
    const int chunks = l.first[l.count];
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int i = tensor_of(l, c);
        const bool bf = l.n[i] < 0;
        const int esz = bf ? 2 : 4;
        const int64_t e0 = (int64_t)(c - l.first[i]) * (kChunkBytes / esz);
        const int n = (int)min((int64_t)(kChunkBytes / esz), (bf ? -l.n[i] : l.n[i]) - e0);
        const char* base = (const char*)l.g[i] + e0 * esz;
        int done = 0;
        if (((uintptr_t)base & 15) == 0) {
            const int nv = n * esz / 16;
            const uint4* p = (const uint4*)base;
            constexpr int U = kChunkBytes / 16 / kThreads;
            uint4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = threadIdx.x + u * kThreads;
                v[u] = k < nv ? __ldg(p + k) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (bf) {
                    s[0] += sq(bf_lo(v[u].x)) + sq(bf_hi(v[u].x));
                    s[1] += sq(bf_lo(v[u].y)) + sq(bf_hi(v[u].y));
                    s[2] += sq(bf_lo(v[u].z)) + sq(bf_hi(v[u].z));
                    s[3] += sq(bf_lo(v[u].w)) + sq(bf_hi(v[u].w));
                } else {
                    s[0] += sq(__uint_as_float(v[u].x));
                    s[1] += sq(__uint_as_float(v[u].y));
                    s[2] += sq(__uint_as_float(v[u].z));
                    s[3] += sq(__uint_as_float(v[u].w));
                }
            }
            done = nv * (16 / esz);
        }
        s[0] += bf ? sq_elements((const __nv_bfloat16*)base, done, n) : sq_elements((const float*)base, done, n);
    }
    const double t = block_sum((s[0] + s[1]) + (s[2] + s[3]), sm);
    if (threadIdx.x == 0) part[blockIdx.x] = t;
}

struct Norm {
    const double* part;
    int parts;
    float grad_scale, max_norm;
    float* norm;
    float* coef;
    int* nonfinite;
};

// The sum of all partial sums, by every thread of the block.
__device__ __forceinline__ double total_of(const Norm& q, double* sm) {
    double s = 0.0;
    for (int k = threadIdx.x; k < q.parts; k += kThreads) s += q.part[k];
    return block_sum(s, sm);
}
// min(1, max_norm / (norm + 1e-6)) in f64; NaN stays NaN.
__device__ __forceinline__ double coef_of(const Norm& q, double norm) {
    const double c = (double)q.max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.0 : c;
}
__device__ __forceinline__ void publish(const Norm& q, double norm) {
    if (q.norm) *q.norm = (float)norm;
    if (q.coef) *q.coef = (float)coef_of(q, norm);
    if (q.nonfinite) *q.nonfinite = isfinite(norm) ? 0 : 1;
}

__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const Norm q) {
    __shared__ double sm[kThreads / 32];
    const double norm = fabs((double)q.grad_scale) * sqrt(total_of(q, sm));
    if (threadIdx.x == 0) publish(q, norm);
}

// The factor as m * p: p = 1 and m the factor rounded to f32, except where that would be subnormal (a norm
// above 2^126 max_norm): there m is in [0.5, 1], rounded up to 1 from just below, and p the power of two, so that m keeps all its bits.
struct Factor {
    float m, p;
    __device__ __forceinline__ float operator()(float v) const { return v * m * p; }
};
__device__ __forceinline__ Factor factor_of(double f) {
    if (!(fabs(f) < 1.1754943508222875e-38) || f == 0.0) return {(float)f, 1.f};
    int e;
    const double m = frexp(f, &e);
    return {(float)m, (float)ldexp(1.0, max(e, -149))};
}

__device__ __forceinline__ uint32_t scale2(uint32_t w, const Factor& f) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f(bf_lo(w)), f(bf_hi(w)));
    return *(const uint32_t*)&h;
}

template <typename T>
__device__ __forceinline__ void scale_elements(const T* src, T* dst, int from, int n, const Factor& f) {
    for (int k = from + threadIdx.x; k < n; k += kBatch * kThreads) {
        T v[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) v[e] = k + e * kThreads < n ? src[k + e * kThreads] : T(0.f);
#pragma unroll
        for (int e = 0; e < kBatch; ++e)
            if (k + e * kThreads < n) dst[k + e * kThreads] = T(f((float)v[e]));
    }
}
template <int CAP>
__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const __grid_constant__ List<CAP> l, const Norm q, int publishes) {
    __shared__ double sm[kThreads / 32];
    const double norm = fabs((double)q.grad_scale) * sqrt(total_of(q, sm));
    if (publishes && blockIdx.x == 0 && threadIdx.x == 0) publish(q, norm);
    const Factor f = factor_of((double)q.grad_scale * coef_of(q, norm));
    const int chunks = l.first[l.count];
    for (int c = chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
        const int i = tensor_of(l, c);
        if (f.m == 1.f && f.p == 1.f && l.out[i] == l.g[i]) continue;  // in place and nothing to scale: every value stays as it is
        const bool bf = l.n[i] < 0;
        const int esz = bf ? 2 : 4;
        const int64_t e0 = (int64_t)(c - l.first[i]) * (kChunkBytes / esz);
        const int n = (int)min((int64_t)(kChunkBytes / esz), (bf ? -l.n[i] : l.n[i]) - e0);
        const char* base = (const char*)l.g[i] + e0 * esz;
        char* dst = (char*)l.out[i] + e0 * esz;
        int done = 0;
        if ((((uintptr_t)base | (uintptr_t)dst) & 15) == 0) {
            const int nv = n * esz / 16;
            constexpr int U = kChunkBytes / 16 / kThreads;
            uint4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = threadIdx.x + u * kThreads;
                if (k < nv) v[u] = ((const uint4*)base)[k];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = threadIdx.x + u * kThreads;
                if (k >= nv) continue;
                if (bf) {
                    v[u] = make_uint4(scale2(v[u].x, f), scale2(v[u].y, f), scale2(v[u].z, f), scale2(v[u].w, f));
                } else {
                    v[u] = make_uint4(__float_as_uint(f(__uint_as_float(v[u].x))), __float_as_uint(f(__uint_as_float(v[u].y))),
                                      __float_as_uint(f(__uint_as_float(v[u].z))), __float_as_uint(f(__uint_as_float(v[u].w))));
                }
                ((uint4*)dst)[k] = v[u];
            }
            done = nv * (16 / esz);
        }
        if (bf) scale_elements((const __nv_bfloat16*)base, (__nv_bfloat16*)dst, done, n, f);
        else scale_elements((const float*)base, (float*)dst, done, n, f);
    }
}

// ---- host ---------------------------------------------------------------------------------------

struct Tensors {
    const void* const* grads;
    void* const* outs;  // NULL: norm only
    const int64_t* counts;
    const int32_t* dtypes;
    int n;
};

inline int64_t chunks_of(int64_t count, int dtype) {
    const int64_t per = kChunkBytes / (dtype == LQ_F32 ? 4 : 2);
    return (count + per - 1) / per;
}

// 128 tensors fit the classic 4 KB of parameters; longer lists take launches of 1024 (29 KB of the 32 KB that
// sm_70 and later accept), which the driver copies whole: with 512 (14 KB) a clip of 168 tensors takes 32 us instead of 34
// on the host, a norm of 392 one microsecond less.
constexpr int kSmall = 128, kMiddle = 512, kLarge = 1024;

// Calls f(list, grid) for every launch's worth of tensors, in order.
template <int CAP, typename F>
void for_lists(const Tensors& t, int sms, F&& f) {
    static_assert(sizeof(List<CAP>) <= 30 * 1024, "kernel parameters");
    List<CAP> l;
    l.count = 0;
    l.first[0] = 0;
    auto flush = [&] {
        if (l.first[l.count] > 0) f(l, (int)std::min<int64_t>(l.first[l.count], (int64_t)sms * kBlocksPerSm));
        l.count = 0;
    };
    for (int i = 0; i < t.n; ++i) {
        if (t.counts[i] == 0) continue;
        const int64_t c = chunks_of(t.counts[i], t.dtypes[i]);
        if (l.count == CAP || l.first[l.count] + c > INT32_MAX) flush();
        l.g[l.count] = t.grads[i];
        l.out[l.count] = t.outs ? t.outs[i] : nullptr;
        l.n[l.count] = t.dtypes[i] == LQ_F32 ? t.counts[i] : -t.counts[i];
        l.first[l.count + 1] = l.first[l.count] + (int)c;
        ++l.count;
    }
    flush();
}

int launches_bound(int n) { return n <= kSmall ? 1 : n / kLarge + 2; }

template <int CAP>
void run(const Tensors& t, Norm q, double* part, int sms, cudaStream_t st) {
    int parts = 0;
    for_lists<CAP>(t, sms, [&](const List<CAP>& l, int grid) {
        LqProf prof(LQ_K_REDUCE, st);
        grad_sq_kernel<CAP><<<grid, kThreads, 0, st>>>(l, part + parts);
        LQ_CUDA(cudaGetLastError());
        parts += grid;
    });
    q.part = part;
    q.parts = parts;
    bool published = false;
    if (t.outs)
        for_lists<CAP>(t, sms, [&](const List<CAP>& l, int grid) {
            LqProf prof(LQ_K_PREP, st);
            grad_scale_kernel<CAP><<<grid, kThreads, 0, st>>>(l, q, published ? 0 : 1);
            LQ_CUDA(cudaGetLastError());
            published = true;
        });
    if (!published) {
        LqProf prof(LQ_K_REDUCE, st);
        grad_norm_kernel<<<1, kThreads, 0, st>>>(q);
        LQ_CUDA(cudaGetLastError());
    }
}

int current_sms() {
    int dev = 0;
    LQ_CUDA(cudaGetDevice(&dev));
    return lq_tc_sm_count(dev);
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

}  // namespace

extern "C" {

size_t lq_grad_norm_workspace_bytes(int n_tensors) {
    if (n_tensors < 0) return 0;
    size_t n = 0;
    if (guarded_call([&] { n = (size_t)launches_bound(n_tensors) * current_sms() * kBlocksPerSm * sizeof(double); }) != LQ_OK)
        return 0;
    return n;
}

int lq_grad_norm(const void* const* grads, void* const* outs, const int64_t* counts, const int32_t* dtypes, int n_tensors,
                 float grad_scale, float max_norm, float* norm, float* coef, int* nonfinite, void* ws, size_t ws_bytes,
                 void* stream) {
    return guarded_call([&] {
        LQ_CHECK_ARG(n_tensors >= 0 && (n_tensors == 0 || (grads && counts && dtypes)), "NULL argument");
        LQ_CHECK_ARG(norm || coef || nonfinite || outs, "no output is asked for");
        LQ_CHECK_ARG(!(outs || coef) || max_norm >= 0.f, "max_norm must be >= 0");
        for (int i = 0; i < n_tensors; ++i) {
            LQ_CHECK_ARG(dtypes[i] == LQ_F32 || dtypes[i] == LQ_BF16, "dtype must be LQ_F32 or LQ_BF16");
            const int64_t mask = dtypes[i] == LQ_F32 ? 3 : 1;
            LQ_CHECK_ARG(counts[i] >= 0 && chunks_of(counts[i], dtypes[i]) <= INT32_MAX, "element count out of range");
            if (counts[i] == 0) continue;
            LQ_CHECK_ARG(grads[i] && (!outs || outs[i]), "NULL tensor");
            LQ_CHECK_ARG(((uintptr_t)grads[i] & mask) == 0 && (!outs || ((uintptr_t)outs[i] & mask) == 0),
                         "tensors must be aligned to their element");
        }
        const int sms = current_sms();
        LQ_CHECK_ARG(ws && ((uintptr_t)ws & 7) == 0, "an 8-byte aligned workspace is needed");
        if (ws_bytes < (size_t)launches_bound(n_tensors) * sms * kBlocksPerSm * sizeof(double))
            throw LqError(LQ_ERR_WORKSPACE, "workspace too small for the gradient norm");
        Tensors t{grads, outs, counts, dtypes, n_tensors};
        Norm q{nullptr, 0, grad_scale, max_norm, norm, coef, nonfinite};
        if (n_tensors <= kSmall) run<kSmall>(t, q, (double*)ws, sms, (cudaStream_t)stream);
        else if (n_tensors <= kMiddle) run<kMiddle>(t, q, (double*)ws, sms, (cudaStream_t)stream);
        else run<kLarge>(t, q, (double*)ws, sms, (cudaStream_t)stream);
    });
}

}  // extern "C"
