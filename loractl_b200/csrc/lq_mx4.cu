// Microscaled 4-bit floating point (MXFP4: e2m1 elements, one e8m0 scale per 32 along a row): quantisation,
// the product of two such tensors on the block-scaled tensor cores, and the backward through a frozen weight.
//
// A block of 32 values v has the scale 2^e, e = floor(log2(max |v|)) - 2 (2 is e2m1's largest exponent),
// clamped to [-127, 125], and the elements are v / 2^e rounded to nearest even among 0, .5, 1, 1.5, 2, 3, 4, 6 and
// saturated at 6.  Scaling by a power of two is exact, so an element is rounded once.  A block of zeros has e = -127;
// a block with an Inf or a NaN has the NaN scale (0xFF) and stands for 32 NaNs.
//
// Storage of [rows, k], k a multiple of 32:
//   codes   row-major, two elements a byte, the even one in the low nibble: what a TMA tile and the MMA read
//   scales  tiles of 128 rows x 4 scales (128 elements of k), 512 bytes each: row r, scale s at byte
//           (r % 32) * 16 + (r / 32) * 4 + s, which is 32 lanes x 4 columns of tensor memory;
//           tile (rt, kt) at (rt * k_tiles + kt) * 512 with k_tiles even (a k-block of the product is 256
//           elements = two tiles) and, above 128 rows, an even number of row tiles (its pair of SMs loads 256 rows).
//           Scales of padding are 0 (2^-127, never NaN: they meet zero codes).
//
// The product Y[n, m] = sum_k X[n, k] W[m, k] (+ bias) multiplies codes and scales where they lie: nothing is
// dequantised (tcgen05.mma kind::mxf4.block_scale, f32 accumulators).
#include <algorithm>
#include <mutex>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lq_internal.cuh"
#include "lq_prof.cuh"
#include "lq_stream.cuh"
#include "lq_tc.cuh"
#include "lq_umma.cuh"

namespace {

using namespace umma;

constexpr int kTile = 512;  // bytes of one scale tile

__host__ __device__ inline int64_t row_tiles(int64_t rows) { return rows <= 128 ? 1 : 2 * ((rows + 255) / 256); }
__host__ __device__ inline int64_t k_tiles(int64_t k) { return 2 * ((k + 255) / 256); }

// ---- quantise / dequantise ------------------------------------------------------------------------

// Eight f32 to eight e2m1 codes, element i in nibble i.
__device__ __forceinline__ uint32_t pack_e2m1(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
__device__ __forceinline__ void unpack_e2m1(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*(const __half2*)&h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ float scale_value(uint32_t byte) {
    const uint32_t bits = byte == 0 ? 0x00400000u : (byte == 255 ? 0x7FC00000u : byte << 23);
    return __uint_as_float(bits);
}

// Two products an instruction, each rounded as its scalar form is.
__device__ __forceinline__ void scale8(float (&f)[8], float s) {
    asm("{\n\t.reg .b64 s, p;\n\t"
        "mov.b64 s, {%8, %8};\n\t"
        "mov.b64 p, {%0, %1};\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {%0, %1}, p;\n\t"
        "mov.b64 p, {%2, %3};\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {%2, %3}, p;\n\t"
        "mov.b64 p, {%4, %5};\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {%4, %5}, p;\n\t"
        "mov.b64 p, {%6, %7};\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {%6, %7}, p;\n\t}"
        : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3]), "+f"(f[4]), "+f"(f[5]), "+f"(f[6]), "+f"(f[7])
        : "f"(s));
}

// Eight elements as they are stored, zeros where `in` is false; `vec`: they start on 16 bytes.
template <typename T>
struct In8 {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void ld(const T* p, bool in, bool vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (!in) return;
        if (vec) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldg((const uint4*)p + i);
        } else {
            T* e = (T*)v;
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[i];
        }
    }
    // The largest magnitude as f32 bits: an integer maximum, in which an Inf or a NaN stands above everything finite.
    __device__ __forceinline__ uint32_t top() const {
        if (sizeof(T) == 4) {
            const uint32_t m = 0x7FFFFFFFu;
            const uint4 a = v[0], b = v[sizeof(T) / 2 - 1];
            const uint32_t p = __vimax3_u32(a.x & m, a.y & m, a.z & m), q = __vimax3_u32(b.x & m, b.y & m, b.z & m);
            return __vimax3_u32(max(p, q), a.w & m, b.w & m);
        }
        const uint32_t m = 0x7FFF7FFFu;  // two bf16 magnitudes a word
        const uint32_t p = __vmaxu2(__vimax3_u16x2(v[0].x & m, v[0].y & m, v[0].z & m), v[0].w & m);
        return max(p & 0xFFFF0000u, p << 16);
    }
    __device__ __forceinline__ void scaled(float s, float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (sizeof(T) == 4) {
                    f[4 * i + j] = __uint_as_float(w[j]);
                } else {
                    f[2 * j] = __uint_as_float(w[j] << 16);
                    f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
                }
            }
        }
        scale8(f, s);
    }
};

// One warp per run of kRun pieces of 256 elements of a row: a lane holds 8 elements, 4 lanes a block, so that loads and
// code stores are whole lines; the run's loads are all in flight before the first is used.  The padding rows of the last
// scale tile are runs too and get zero scales.  Bound by instruction issue before HBM (1536 x 16384 bf16: 171
// instructions a piece 21 us, 75 % of the issue slots and 27 % of the HBM rate): hence the packed maxima and the runs
// within one row.
constexpr int kRun = 4;
template <typename T>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(const T* __restrict__ x, int64_t rows, int k, int64_t ld, int vec,
                                                           int64_t pad_rows, uint32_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales) {
    const int kb = (k + 255) / 256, runs = (kb + kRun - 1) / kRun;
    const int64_t items = pad_rows * runs;
    const int lane = threadIdx.x & 31;
    lqstream::pdl_launch_dependents();  // a product behind this launch may start fetching its weight
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += (int64_t)gridDim.x * 8) {
        const int64_t row = it / runs;
        const int b0 = (int)(it - row * runs) * kRun, col = b0 * 256 + lane * 8;
        const bool real = row < rows;
        const T* src = x + row * ld + col;
        In8<T> in[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) in[i].ld(src + i * 256, real && col + i * 256 < k, vec);
        uint32_t* dst = codes + ((row * k + col) >> 3);
        const int r = (int)(row & 127);
        uint8_t* sc = scales + ((row >> 7) * (2 * kb) + 2 * b0 + (lane >> 4)) * kTile + (r & 31) * 16 + (r >> 5) * 4;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            if (b0 + i >= kb) break;
            uint32_t top = in[i].top();
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the exponent field f stands for 2^(f - 127): e = f - 129, stored as e + 127; subnormals fall to the lowest
            const bool bad = top >= 0x7F800000u;
            const uint32_t e = max(top >> 23, 2u) - 2u, byte = bad ? 255u : e;
            float v[8];
            in[i].scaled(__uint_as_float((254u - e) << 23), v);
            const uint32_t w = bad ? 0u : pack_e2m1(v);
            if (real && col + i * 256 < k) dst[i * 32] = w;
            // the four scales of 128 elements as one word in the first lane of each half-warp
            uint32_t word = byte | __shfl_down_sync(0xffffffffu, byte, 4) << 8;
            word |= __shfl_down_sync(0xffffffffu, word, 8) << 16;
            if ((lane & 15) == 0) *(uint32_t*)(sc + i * 2 * kTile) = word;
        }
    }
}

// out[row, col .. col + 7] = code * scale, 8 elements a lane, a warp the same runs; exact in f32 and in bf16.
template <typename T>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             int64_t rows, int k, T* __restrict__ out) {
    const int kb = (k + 255) / 256, runs = (kb + kRun - 1) / kRun;
    const int64_t items = rows * runs;
    const int lane = threadIdx.x & 31;
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += (int64_t)gridDim.x * 8) {
        const int64_t row = it / runs;
        const int b0 = (int)(it - row * runs) * kRun, col = b0 * 256 + lane * 8;
        const int64_t at = row * k + col;
        const int r = (int)(row & 127);
        const uint8_t* sc = scales + ((row >> 7) * (2 * kb) + 2 * b0 + (lane >> 4)) * kTile + (r & 31) * 16 + (r >> 5) * 4 + ((lane >> 2) & 3);
        uint32_t w[kRun], byte[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const bool in = col + i * 256 < k;
            w[i] = in ? __ldg(codes + (at >> 3) + i * 32) : 0u;
            byte[i] = in ? __ldg(sc + i * 2 * kTile) : 0u;
        }
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            if (col + i * 256 >= k) break;
            const float s = scale_value(byte[i]);
            float v[8];
            unpack_e2m1(w[i], v);
            scale8(v, s);
            T* o = out + at + i * 256;
            if (sizeof(T) == 4) {
                ((float4*)o)[0] = make_float4(v[0], v[1], v[2], v[3]);
                ((float4*)o)[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                uint32_t q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
                    q[e] = *(const uint32_t*)&h;
                }
                *(uint4*)o = make_uint4(q[0], q[1], q[2], q[3]);
            }
        }
    }
}

// ---- the product ------------------------------------------------------------------------------------

// tcgen05.mma kind::mxf4, block scale of 32 elements: K = 64 per instruction, two scales per row.
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// Scales reach tensor memory through four warps of their own: a scale tile is 16 bytes for each of 32 lanes, which is
// one vector read and one four-column store per warp, and every lane quarter holds the same copy.  The tensor pipe's own
// copy (tcgen05.cp 32x128b.warpx4) needs no warps, but the products queue behind it: with six such copies per 256-element
// k-block the pair kernel ran at 4.6 PFLOP/s, without any at 6.2.
__device__ __forceinline__ void stage_scales(uint32_t taddr, const uint8_t* tile, int lane) {
    tmem_st_x4(taddr, *(const uint4*)(tile + lane * 16));
}
// Instruction descriptor of kind::mxf4: [4,6) which scale pair of B's column word, [7,10) and [10,12) e2m1 = 1,
// [17,23) N >> 3, [23] scales are e8m0, [24,29) M >> 4, [29,31) which scale pair of A's.
__host__ __device__ constexpr uint32_t idesc_mxf4(uint32_t M, uint32_t N, uint32_t pair) {
    return (2 * pair << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | (1u << 23) | ((M >> 4) << 24) | (2 * pair << 29);
}

struct ProductParams {
    const uint8_t* w_scales;
    const uint8_t* x_scales;
    int m, n, kb;             // d_out, tokens, k-blocks of 256
    int w_tiles, x_tiles;     // 128 weight rows; BN tokens, which is 128 (a whole scale tile) when there are several
    int splits;               // blocks of a tile: ranges of the reduction, one cluster
    int lora;                 // k-blocks of 64 bf16 after those (pairs only): s * H against B^T
    int early_w;              // the launch before this one is known not to write the weight (it quantises x)
    const float* bias;
    void* y;
    int y_f32;
    int* status;
};

constexpr int kThreads = 192;  // TMA warp, MMA warp, four warps that stage scales and then write the output

template <int BN>
struct CfgT {
    static constexpr uint32_t A_BYTES = 128 * 128, B_BYTES = BN * 128, S_BYTES = 2 * kTile;
    static constexpr uint32_t STAGE = A_BYTES + B_BYTES + 2 * S_BYTES;
    static constexpr int STAGES = (104 * 1024) / STAGE;  // two blocks to an SM
    static constexpr uint32_t TMEM = 256;
    // An MMA of few columns takes its latency, not its work, when the next one waits for its sum: the four MMAs
    // of a k-block then go to an accumulator each.
    static constexpr int ACCS = BN <= 32 ? 4 : 1;
    static constexpr uint32_t SCALE_COL = ACCS * BN;  // behind the accumulators: 16 columns per stage
    static_assert(SCALE_COL + 16 * STAGES <= TMEM, "tensor memory");
    static_assert(BN * 512 <= STAGES * STAGE, "the f32 tile takes the ring's place");
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + 1024 + 256;
};

__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld_x16(taddr, r); }
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_x32(taddr, r); }

__device__ __forceinline__ float4 ld_peer(uint32_t addr, uint32_t rank) {
    uint32_t at;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// Few tokens (or few weight rows): the weight is the 128-row operand and BN tokens are the columns, so that a
// narrow batch wastes no tensor rows.  The weight's bytes are the work, so every SM has to stream them: a tile's
// reduction is cut into `splits` ranges, one block each, and the blocks of a tile are a cluster that adds its f32
// tiles up through distributed shared memory, in rank order, each rank a share of the tokens.  (Partial tiles in HBM and
// a second launch took 5.8 us of 14.6 at 77 x 2592 -> 6151, where this takes 9.6.)  One token through 6144 -> 16384 takes
// 13.4 us from HBM (captured, eight weights in turn), 4.0 TB/s of weight, and 10.4 with the weight in the L2; the launch, its ramp and
// the loads alone take 11.3.  D's lane is a weight row, so a store of one
// token writes 32 consecutive outputs.
template <int BN>
__global__ void __launch_bounds__(kThreads, 2) mx4_stream_kernel(const __grid_constant__ CUtensorMap tmW,
                                                                 const __grid_constant__ CUtensorMap tmX, ProductParams p) {
    using C = CfgT<BN>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* smem_a = smem;
    uint8_t* smem_b = smem_a + (size_t)STAGES * C::A_BYTES;
    uint8_t* smem_s = smem_b + (size_t)STAGES * C::B_BYTES;  // per stage: W's two scale tiles, then X's
    uint64_t* bars = (uint64_t*)(smem_s + (size_t)STAGES * 2 * C::S_BYTES);
    uint64_t* full = bars;
    uint64_t* empty = bars + STAGES;
    uint64_t* scaled = bars + 2 * STAGES;  // the stage's scales are in tensor memory
    uint64_t* tfull = bars + 3 * STAGES;
    uint32_t* tmem_slot = (uint32_t*)(tfull + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // block = split of a tile; the grid is tiles x splits with the splits of a tile next to one another
    const int z = (int)blockIdx.x % p.splits, tile = (int)blockIdx.x / p.splits;
    const int wt = tile % p.w_tiles, xt = tile / p.w_tiles;
    const int k0 = (int)((long long)p.kb * z / p.splits), k1 = (int)((long long)p.kb * (z + 1) / p.splits);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
            mbar_init(smem_u32(&scaled[s]), 4);
        }
        mbar_init(smem_u32(tfull), 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&tmW);
        prefetch_tmap(&tmX);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), C::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            const int kt = 2 * p.kb;
            auto load_w = [&](int st, int kb) {
                const uint32_t bar = smem_u32(&full[st]);
                mbar_expect_tx(bar, C::STAGE);
                tma_load_2d(smem_u32(smem_a + (size_t)st * C::A_BYTES), &tmW, bar, kb * 128, wt * 128);
                bulk_load(smem_u32(smem_s + (size_t)st * 2 * C::S_BYTES), p.w_scales + ((int64_t)wt * kt + 2 * kb) * kTile, C::S_BYTES, bar);
            };
            // behind the quantisation of x, the weight's first stages are fetched while that runs; behind any other
            // launch (which may be the weight's own quantisation) nothing is read before it has ended
            if (!p.early_w) lqstream::pdl_wait();
            const int ahead = min(STAGES, k1 - k0);
            for (int i = 0; i < ahead; ++i) load_w(i, k0 + i);
            if (p.early_w) lqstream::pdl_wait();
            int s = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int kb = k0; kb < k1; ++kb) {
                if (kb - k0 >= ahead) {
                    if (!mbar_wait(smem_u32(&empty[s]), phase ^ 1u, abort_flag, p.status, 71)) { ok = false; break; }
                    load_w(s, kb);
                }
                const uint32_t bar = smem_u32(&full[s]);
                tma_load_2d(smem_u32(smem_b + (size_t)s * C::B_BYTES), &tmX, bar, kb * 128, xt * BN);
                bulk_load(smem_u32(smem_s + (size_t)s * 2 * C::S_BYTES + C::S_BYTES), p.x_scales + ((int64_t)xt * kt + 2 * kb) * kTile, C::S_BYTES, bar);
                if (++s == STAGES) { s = 0; phase ^= 1u; }
            }
            if (!ok)
                for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the block ends
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t d_hi = desc_hi(1024);
            int s = 0;
            uint32_t phase = 0;
            for (int kb = k0; kb < k1; ++kb) {
                if (!mbar_wait(smem_u32(&full[s]), phase, abort_flag, p.status, 73) ||
                    !mbar_wait(smem_u32(&scaled[s]), phase, abort_flag, p.status, 79)) break;
                tc_fence_after();
                const uint32_t sfa = tmem + C::SCALE_COL + (uint32_t)s * 16, sfb = sfa + 8;
                const uint32_t a_lo = desc_lo(smem_u32(smem_a + (size_t)s * C::A_BYTES), 16);
                const uint32_t b_lo = desc_lo(smem_u32(smem_b + (size_t)s * C::B_BYTES), 16);
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k)  // 64 elements = 32 bytes; scale pair k & 1 of tile k / 2
                    mma_mxf4(tmem + k % C::ACCS * BN, desc_join(a_lo + 2 * k, d_hi), desc_join(b_lo + 2 * k, d_hi),
                             idesc_mxf4(128, BN, k & 1), sfa + 4 * (k >> 1), sfb + 4 * (k >> 1), (kb > k0 || k >= C::ACCS) ? 1u : 0u);
                mma_commit(smem_u32(kb + 1 == k1 ? tfull : &empty[s]));
                if (++s == STAGES) { s = 0; phase ^= 1u; }
            }
        }
    } else {
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        int s = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = k0; kb < k1; ++kb) {
            // the stage was released before its copies began, so its columns are free too
            if (!mbar_wait(smem_u32(&full[s]), phase, abort_flag, p.status, 80)) { ok = false; break; }
            const uint8_t* sc = smem_s + (size_t)s * 2 * C::S_BYTES;
#pragma unroll
            for (int t = 0; t < 4; ++t) stage_scales(lanes + C::SCALE_COL + (uint32_t)(s * 16 + 4 * t), sc + t * kTile, lane);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&scaled[s]));
            if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
        if (ok && mbar_wait(smem_u32(tfull), 0, abort_flag, p.status, 74)) {
            tc_fence_after();
            const int r = (warp & 3) * 32 + lane, row = wt * 128 + r;
            const float bias = (p.splits == 1 && p.bias && row < p.m) ? p.bias[row] : 0.f;
            const uint32_t part = smem_u32(smem) + (uint32_t)r * 4;  // [token][128 rows]: the last product has read the ring
            constexpr int W = BN < 32 ? BN : 32;
#pragma unroll 1
            for (int c = 0; c < BN && xt * BN + c < p.n; c += W) {
                float f[W];
#pragma unroll
                for (int a = 0; a < C::ACCS; ++a) {
                    uint32_t v[W];
                    tmem_ld_cols(lanes + (uint32_t)(a * BN + c), v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < W; ++j) f[j] = a == 0 ? __uint_as_float(v[j]) : f[j] + __uint_as_float(v[j]);
                }
                if (p.splits > 1) {
#pragma unroll
                    for (int j = 0; j < W; ++j) asm volatile("st.shared.f32 [%0], %1;" ::"r"(part + (uint32_t)(c + j) * 512), "f"(f[j]) : "memory");
                } else if (row < p.m) {
                    const int toks = p.n - xt * BN - c;
                    const int64_t o = (int64_t)(xt * BN + c) * p.m + row;
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        if (j >= toks) break;
                        if (p.y_f32) ((float*)p.y)[o + (int64_t)j * p.m] = f[j] + bias;
                        else ((__nv_bfloat16*)p.y)[o + (int64_t)j * p.m] = __float2bfloat16(f[j] + bias);
                    }
                }
            }
        }
    }
    __syncwarp();  // the single-lane roles rejoin their warps before the aligned barriers
    if (p.splits > 1) {
        cluster_sync_all();
        const uint32_t part = smem_u32(smem);
        const int quads = min(BN, p.n - xt * BN) * 32;  // four weight rows of a token each; rank z's share is one run of them
        const int e1 = quads * (z + 1) / p.splits;
        const bool whole = p.m % 4 == 0 && ((uintptr_t)p.y & 15) == 0;
        for (int e = quads * z / p.splits + (int)threadIdx.x; e < e1; e += kThreads) {
            const int64_t row = wt * 128 + (e & 31) * 4, tok = xt * BN + (e >> 5), o = tok * p.m + row;
            float4 v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < p.splits) v[q] = ld_peer(part + (uint32_t)e * 16, (uint32_t)q);
            float f[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
            for (int q = 1; q < 8; ++q)
                if (q < p.splits) f[0] += v[q].x, f[1] += v[q].y, f[2] += v[q].z, f[3] += v[q].w;
            if (p.bias) {
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] += row + i < p.m ? p.bias[row + i] : 0.f;
            }
            if (whole && row < p.m && !p.y_f32) {  // rows of four start on 8 bytes
                const __nv_bfloat162 lo = __floats2bfloat162_rn(f[0], f[1]), hi = __floats2bfloat162_rn(f[2], f[3]);
                *(uint2*)((__nv_bfloat16*)p.y + o) = make_uint2(*(const uint32_t*)&lo, *(const uint32_t*)&hi);
            } else if (whole && row < p.m) {
                *(float4*)((float*)p.y + o) = make_float4(f[0], f[1], f[2], f[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (row + i >= p.m) break;
                    if (p.y_f32) ((float*)p.y)[o + i] = f[i];
                    else ((__nv_bfloat16*)p.y)[o + i] = __float2bfloat16(f[i]);
                }
            }
        }
        cluster_sync_all();  // the other ranks have read this block's tile
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM);
    }
}

// ---- many tokens: pairs of SMs ---------------------------------------------------------------------
// D tiles of 256 tokens x 256 outputs on a cluster of two CTAs (cta_group::2): each stages its own 128 token rows and
// HALF of the 256 weight rows, so an SM reads and writes 64 KB of shared memory per 16.8 MFLOP k-block instead of the 96 KB
// of a tile of its own; the scales of its rows and of all 256 columns go to its own tensor memory, into the columns of
// the stage they came with, so that a stage's release covers them.  The accumulator has one buffer (256 columns; two
// would leave no room for scales): the epilogue empties it into registers at once and converts and stores
// while the next tile's products run.  4096 x 6144 -> 16384: 167 us, 4.9 PFLOP/s (single CTAs with 128 x 128 tiles: 343 us);
// for seconds on end 4.3 PFLOP/s, at the card's power cap.  Its 128 registers a thread (448 threads) spill 44-56 bytes.  An adapter's product is one more k-block of bf16 for each 64 of
// rank (the ring's stages fit: 64 bf16 are 128 bytes a row too): 180 us with rank 16.
struct Cfg2 {
    static constexpr uint32_t A_BYTES = 128 * 128, B_BYTES = 128 * 128, SA_BYTES = 2 * kTile, SB_BYTES = 4 * kTile;
    static constexpr uint32_t STAGE = A_BYTES + B_BYTES + SA_BYTES + SB_BYTES;
    static constexpr int STAGES = 5;
    static constexpr uint32_t TMEM = 512, SCALE_COL = 256;
    static_assert(SCALE_COL + 24 * STAGES <= 512, "tensor memory");
    static constexpr uint32_t OUT = 8 * 2048;  // per epilogue warp: 32 rows x 32 bf16 (or 16 f32) columns
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + OUT + 1024 + 256;
};
constexpr int kThreads2 = 448;  // TMA warp, MMA warp, eight epilogue warps, four scale warps
constexpr int kGroupM = 8;      // token tiles per raster group

__device__ __forceinline__ void mma2_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tile2(const ProductParams& p, int item, int& xt, int& wt) {
    const int per = kGroupM * p.w_tiles, g = item / per, first = g * kGroupM;
    const int rows = min(kGroupM, p.x_tiles - first), r = item - g * per;
    xt = first + r % rows;
    wt = r / rows;
}

// LORA: an adapter's k-blocks follow (a variant of its own: the branches in every role cost the plain product 2-4 %).
template <bool TMA_OUT, bool LORA>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads2, 1)
mx4_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmXs,
                const __grid_constant__ CUtensorMap tmWs, const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmH,
                const __grid_constant__ CUtensorMap tmB, ProductParams p) {
    using C = Cfg2;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* smem_a = smem;
    uint8_t* smem_b = smem_a + (size_t)STAGES * C::A_BYTES;
    uint8_t* smem_sa = smem_b + (size_t)STAGES * C::B_BYTES;
    uint8_t* smem_sb = smem_sa + (size_t)STAGES * C::SA_BYTES;
    uint8_t* stage_out = smem_sb + (size_t)STAGES * C::SB_BYTES;
    uint64_t* bars = (uint64_t*)(stage_out + C::OUT);
    uint64_t* full = bars;            // leader's: the bytes of both CTAs' copies
    uint64_t* empty = bars + STAGES;  // in both, from the leader's multicast commit
    uint64_t* sfull = bars + 2 * STAGES;   // each CTA's own: its scale tiles have landed
    uint64_t* scaled = bars + 3 * STAGES;  // leader's: the scale warps of both CTAs have stored them
    uint64_t* tfull = bars + 4 * STAGES;
    uint64_t* tempty = tfull + 1;     // leader's: the epilogue warps of both CTAs
    uint32_t* tmem_slot = (uint32_t*)(tempty + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
            mbar_init(smem_u32(&sfull[s]), 1);
            mbar_init(smem_u32(&scaled[s]), 8);
        }
        mbar_init(smem_u32(tfull), 1);
        mbar_init(smem_u32(tempty), 16);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&tmX);
        prefetch_tmap(&tmW);
        prefetch_tmap(&tmXs);
        prefetch_tmap(&tmWs);
    }
    if (warp == 1) {
        tmem_alloc2(smem_u32(tmem_slot), C::TMEM);
        tmem_relinquish2();
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int items = p.x_tiles * p.w_tiles, cid = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
    const int blocks = LORA ? p.kb + p.lora : p.kb;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 0;
            bool ok = true;
            lqstream::pdl_wait();  // x is the output of the launch before
            for (int item = cid; ok && item < items; item += pairs) {
                int xt, wt;
                tile2(p, item, xt, wt);
                for (int kb = 0; kb < blocks; ++kb) {
                    if (!mbar_wait(smem_u32(&empty[s]), phase ^ 1u, abort_flag, p.status, 75)) { ok = false; break; }
                    const uint32_t bar = smem_u32(&full[s]), sbar = smem_u32(&sfull[s]);
                    const uint32_t sa = smem_u32(smem_a + (size_t)s * C::A_BYTES), sb = smem_u32(smem_b + (size_t)s * C::B_BYTES);
                    if (leader) mbar_expect_tx(bar, 2 * (C::A_BYTES + C::B_BYTES));
                    if (!LORA || kb < p.kb) {
                        tma_load_2d_pair(sa, &tmX, bar, kb * 128, xt * 256 + (int)rank * 128);
                        tma_load_2d_pair(sb, &tmW, bar, kb * 128, wt * 256 + (int)rank * 128);
                        mbar_expect_tx(sbar, C::SA_BYTES + C::SB_BYTES);
                        tma_load_2d(smem_u32(smem_sa + (size_t)s * C::SA_BYTES), &tmXs, sbar, kb * 256, xt * 2 + (int)rank);
                        tma_load_2d(smem_u32(smem_sb + (size_t)s * C::SB_BYTES), &tmWs, sbar, kb * 256, wt * 2);
                    } else {  // 64 columns of s * H and of B^T: rows of 128 bytes as well
                        tma_load_2d_pair(sa, &tmH, bar, (kb - p.kb) * 64, xt * 256 + (int)rank * 128);
                        tma_load_2d_pair(sb, &tmB, bar, (kb - p.kb) * 64, wt * 256 + (int)rank * 128);
                        mbar_arrive(sbar);
                    }
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                }
            }
            if (!ok)
                for (int i = 0; i < 64; ++i) __nanosleep(1000);
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            const uint32_t d_hi = desc_hi(1024);
            int s = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (int item = cid; ok && item < items; item += pairs) {
                if (!mbar_wait(smem_u32(tempty), acc_phase ^ 1u, abort_flag, p.status, 76)) { ok = false; break; }
                acc_phase ^= 1u;
                tc_fence_after();
                for (int kb = 0; kb < blocks; ++kb) {
                    if (!mbar_wait(smem_u32(&full[s]), phase, abort_flag, p.status, 77) ||
                        !mbar_wait(smem_u32(&scaled[s]), phase, abort_flag, p.status, 83)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t sfa = tmem + C::SCALE_COL + (uint32_t)s * 24, sfb = sfa + 8;
                    const uint32_t a_lo = desc_lo(smem_u32(smem_a + (size_t)s * C::A_BYTES), 16);
                    const uint32_t b_lo = desc_lo(smem_u32(smem_b + (size_t)s * C::B_BYTES), 16);
                    if (!LORA || kb < p.kb) {
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k)
                            mma2_mxf4(tmem, desc_join(a_lo + 2 * k, d_hi), desc_join(b_lo + 2 * k, d_hi), idesc_mxf4(256, 256, k & 1),
                                      sfa + 4 * (k >> 1), sfb + 8 * (k >> 1), (kb > 0 || k > 0) ? 1u : 0u);
                    } else {
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k)  // 16 bf16 an instruction: 32 bytes along the row, as 64 codes are
                            mma2_f16(tmem, desc_join(a_lo + 2 * k, d_hi), desc_join(b_lo + 2 * k, d_hi),
                                     make_idesc(1, 1, false, false, 256, 256), 1u);
                    }
                    mma2_commit_mc(smem_u32(&empty[s]), 3);
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                }
                if (!ok) break;
                mma2_commit_mc(smem_u32(tfull), 3);
            }
        }
    } else if (warp >= 10) {
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + C::SCALE_COL;
        int s = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int item = cid; ok && item < items; item += pairs) {
            for (int kb = 0; kb < blocks; ++kb) {
                if (!mbar_wait(smem_u32(&sfull[s]), phase, abort_flag, p.status, 84)) { ok = false; break; }
                const uint8_t *sa = smem_sa + (size_t)s * C::SA_BYTES, *sb = smem_sb + (size_t)s * C::SB_BYTES;
                const uint32_t sfa = lanes + (uint32_t)s * 24, sfb = sfa + 8;
                if (!LORA || kb < p.kb) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {  // tiles of 128 elements; B's rows 0-127 and 128-255
                        stage_scales(sfa + 4 * j, sa + j * kTile, lane);
                        stage_scales(sfb + 8 * j, sb + j * kTile, lane);
                        stage_scales(sfb + 8 * j + 4, sb + (2 + j) * kTile, lane);
                    }
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (leader) mbar_arrive(smem_u32(&scaled[s]));
                    else mbar_arrive_leader(smem_u32(&scaled[s]));
                }
                if (++s == STAGES) { s = 0; phase ^= 1u; }
            }
        }
    } else {
        const int quarter = warp & 3, chalf = (warp - 2) >> 2;
        uint8_t* mine = stage_out + (warp - 2) * 2048;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(chalf * 128);
        uint32_t acc_phase = 0;
        auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (leader) mbar_arrive(smem_u32(tempty));
                else mbar_arrive_leader(smem_u32(tempty));
            }
        };
        auto biased = [&](uint32_t v, int col) {
            return p.bias && col < p.m ? __uint_as_float(v) + __ldg(p.bias + col) : __uint_as_float(v);
        };
        for (int item = cid; item < items; item += pairs) {
            int xt, wt;
            tile2(p, item, xt, wt);
            if (!mbar_wait(smem_u32(tfull), acc_phase, abort_flag, p.status, 78)) break;
            acc_phase ^= 1u;
            tc_fence_after();
            const int row0 = xt * 256 + (int)rank * 128 + quarter * 32, col0 = wt * 256 + chalf * 128;
            if (TMA_OUT) {
                uint32_t w[4][16];  // 128 columns as bf16 pairs
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t r[2][32];
                    tmem_ld_x32(lanes + (uint32_t)(hf * 64), r[0]);
                    tmem_ld_x32(lanes + (uint32_t)(hf * 64 + 32), r[1]);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int col = col0 + hf * 64 + c * 32 + 2 * j;
                            const __nv_bfloat162 h = __floats2bfloat162_rn(biased(r[c][2 * j], col), biased(r[c][2 * j + 1], col + 1));
                            w[2 * hf + c][j] = *(const uint32_t*)&h;
                        }
                }
                release();
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (lane == 0) bulk_wait_read0();
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *(uint4*)(mine + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) =
                            make_uint4(w[c][4 * q], w[c][4 * q + 1], w[c][4 * q + 2], w[c][4 * q + 3]);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmY, smem_u32(mine), col0 + c * 32, row0);
                        bulk_commit();
                    }
                }
            } else {  // f32, or rows that do not start on 16 bytes: turned in shared memory, 16 columns at a time
#pragma unroll 1
                for (int c = 0; c < 128; c += 16) {
                    uint32_t r[16];
                    tmem_ld_x16(lanes + (uint32_t)c, r);
                    tmem_ld_wait();
                    if (c == 112) release();
                    float* t = (float*)mine;
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 16; ++j) t[lane * 16 + ((j + lane) & 15)] = biased(r[j], col0 + c + j);
                    __syncwarp();
                    const int j = lane & 15, cj = col0 + c + j;
#pragma unroll 4
                    for (int i = lane >> 4; i < 32; i += 2) {
                        const float v = t[i * 16 + ((j + i) & 15)];
                        if (row0 + i < p.n && cj < p.m) {
                            const int64_t o = (int64_t)(row0 + i) * p.m + cj;
                            if (p.y_f32) ((float*)p.y)[o] = v;
                            else ((__nv_bfloat16*)p.y)[o] = __float2bfloat16(v);
                        }
                    }
                }
            }
        }
        if (lane == 0) bulk_wait0();
    }
    __syncwarp();  // the single-lane roles rejoin their warps before the aligned barrier
    tc_fence_before();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc2(tmem, C::TMEM);
    }
}

// [n, m] bf16 with a row stride of `ld` elements, for the tensor maps' 16-byte rows.
__global__ void __launch_bounds__(256) pad_rows_kernel(const __nv_bfloat16* __restrict__ in, int64_t n, int64_t m, int64_t ld,
                                                       __nv_bfloat16* __restrict__ out) {
    const int64_t total = n * ld;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / ld, c = i - r * ld;
        out[i] = c < m ? in[r * m + c] : __float2bfloat16(0.f);
    }
}

// [n, m] f32 as three stacked bf16 matrices [3, n, ld] whose sum it is: each takes the eight leading bits of what the one
// before left, cut and not rounded, so nothing overflows and the third is exact too (down to bf16's last bit, 2^-133).  An Inf or a NaN goes to the first.
__global__ void __launch_bounds__(256) split3_kernel(const float* __restrict__ in, int64_t n, int64_t m, int64_t ld,
                                                     __nv_bfloat16* __restrict__ out) {
    const int64_t total = n * ld;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / ld, c = i - r * ld;
        const float v = c < m ? in[r * m + c] : 0.f;
        float rest = v;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            float part = __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
            if (k == 0 && isnan(v)) part = v;
            out[k * total + i] = __float2bfloat16(part);
            rest = isfinite(v) ? rest - part : 0.f;
        }
    }
}
// out = c[0] + (c[1] + c[2]) of the terms, each the sum of its ranges: [ranges, 3, n] f32 in, n4 = n / 4.
__global__ void __launch_bounds__(256) join3_kernel(const float4* __restrict__ c, int64_t n4, int ranges, float4* __restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n4; i += (int64_t)gridDim.x * blockDim.x) {
        float4 t[3] = {};
        for (int z = 0; z < ranges; ++z)
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                const float4 v = c[(3 * z + j) * n4 + i];
                t[j].x += v.x, t[j].y += v.y, t[j].z += v.z, t[j].w += v.w;
            }
        out[i] = make_float4(t[0].x + (t[1].x + t[2].x), t[0].y + (t[1].y + t[2].y), t[0].z + (t[1].z + t[2].z), t[0].w + (t[1].w + t[2].w));
    }
}

// ---- host ---------------------------------------------------------------------------------------

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
inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }
inline unsigned grid_of(int64_t items, int sms, int per_sm) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(items, (int64_t)sms * per_sm));
}

inline int64_t runs_of(int64_t k) { return ((k + 255) / 256 + kRun - 1) / kRun; }

void check_dims(int64_t rows, int64_t k) {
    LQ_CHECK_ARG(rows >= 0 && rows < (int64_t)1 << 31, "row count out of range");
    LQ_CHECK_ARG(k >= 32 && k % 32 == 0 && k <= (int64_t)1 << 30, "the block axis must be a positive multiple of 32");
}
void check_tensor(const void* codes, const void* scales) {
    LQ_CHECK_ARG(codes && scales, "NULL argument");
    LQ_CHECK_ARG(al16(codes) && al16(scales), "codes and scales must be 16-byte aligned");
}

int bn_of(int64_t n) { return n <= 16 ? 16 : (n <= 32 ? 32 : (n <= 64 ? 64 : 128)); }

// Ranges of the reduction (blocks of a cluster: 1, 2, 4 or 8): as many as two blocks an SM leave room for, each of at
// least two k-blocks.
int splits_of(int64_t tiles, int64_t kb, int sms) {
    int s = 1;
    while (s < 8 && tiles * s * 2 <= 2 * (int64_t)sms && kb >= 4 * s) s *= 2;
    return s;
}

// Pairs of SMs where their 256 x 256 tiles occupy two thirds of them; below, 128 x 128 tiles split along k spread
// wider.  At k = 6144 (pair | stream, us): 24 tiles 16.1 | 14.4, 48 tiles 16.4 | 16.1, 72 tiles 16.9 | 16.9, 128 tiles 28 | 35, 384 tiles 71 | 93.
bool use_pair(int64_t n, int64_t m) {
    constexpr int64_t kSms = 148;  // workspaces are sized by this rule too, without a device
    return n > 128 && m > 128 && ((n + 255) / 256) * ((m + 255) / 256) * 3 > kSms;
}

template <int BN>
void launch_stream(const ProductParams& p, const void* w_codes, const void* x_codes, int64_t k, cudaStream_t st) {
    using C = CfgT<BN>;
    const CUtensorMap tw = lq_tc_make_map_u8(w_codes, k / 2, p.m, k / 2, 128);
    const CUtensorMap tx = lq_tc_make_map_u8(x_codes, k / 2, p.n, k / 2, BN);
    LQ_CUDA(cudaFuncSetAttribute(mx4_stream_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
    const int64_t blocks = (int64_t)p.w_tiles * p.x_tiles * p.splits;
    LQ_CHECK_ARG(blocks < (int64_t)1 << 31, "too many tiles");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)p.splits, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = lqstream::pdl_enabled() ? 2 : 1;
    LqProf prof(LQ_K_GEMM_MAIN, st);
    LQ_CUDA(cudaLaunchKernelEx(&cfg, mx4_stream_kernel<BN>, tw, tx, p));
}

// Of a LoRA product that the pair kernel adds: s * H [n, ext] and B^T [m, ext] in bf16, zero beyond the rank.
struct LoraOperands {
    const __nv_bfloat16 *h, *bt;
    int ext;
};

// Pairs that can be resident at once, asked once per device.
int resident_pairs(int dev, int sms) {
    static std::mutex mu;
    static int known[64] = {};
    std::lock_guard<std::mutex> lk(mu);
    if (known[dev & 63] == 0) {
        LQ_CUDA(cudaFuncSetAttribute(mx4_pair_kernel<true, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg2::SMEM));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(sms & ~1);
        cfg.blockDim = dim3(kThreads2);
        cfg.dynamicSmemBytes = Cfg2::SMEM;
        int n = 0;
        LQ_CUDA(cudaOccupancyMaxActiveClusters(&n, mx4_pair_kernel<true, false>, &cfg));
        known[dev & 63] = std::max(1, std::min(n, sms / 2));
    }
    return known[dev & 63];
}

void launch_pair(ProductParams p, const void* w_codes, const void* x_codes, int64_t k, const LoraOperands* lora, int dev, int sms,
                 cudaStream_t st) {
    const CUtensorMap tx = lq_tc_make_map_u8(x_codes, k / 2, p.n, k / 2, 128);
    const CUtensorMap tw = lq_tc_make_map_u8(w_codes, k / 2, p.m, k / 2, 128);
    const CUtensorMap txs = lq_tc_make_map_u32(p.x_scales, k_tiles(k) * (kTile / 4), row_tiles(p.n), 256, 1);
    const CUtensorMap tws = lq_tc_make_map_u32(p.w_scales, k_tiles(k) * (kTile / 4), row_tiles(p.m), 256, 2);
    const int tma_store = !p.y_f32 && p.m % 8 == 0 && al16(p.y);
    const CUtensorMap th = lora ? lq_tc_make_map(lora->h, lora->ext, p.n, lora->ext, 128) : tx;
    const CUtensorMap tb = lora ? lq_tc_make_map(lora->bt, lora->ext, p.m, lora->ext, 128) : tx;
    p.lora = lora ? lora->ext / 64 : 0;
    LQ_CHECK_ARG(!lora || tma_store, "with an adapter the output is bf16 in rows of 16 bytes");
    const CUtensorMap ty = tma_store ? lq_tc_make_store_map(p.y, p.m, p.n, p.m) : tx;
    p.x_tiles = (p.n + 255) / 256;
    p.w_tiles = (p.m + 255) / 256;
    LQ_CHECK_ARG((int64_t)p.x_tiles * p.w_tiles < (int64_t)1 << 31, "too many tiles");
    const int pairs = std::min({resident_pairs(dev, sms), lq_tc_usable_sms(sms) / 2, p.x_tiles * p.w_tiles});
    auto kern = lora ? mx4_pair_kernel<true, true> : (tma_store ? mx4_pair_kernel<true, false> : mx4_pair_kernel<false, false>);
    LQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg2::SMEM));
    LqProf prof(LQ_K_GEMM_MAIN, st);
    lqstream::launch_pdl(kern, dim3(2 * pairs), dim3(kThreads2), Cfg2::SMEM, st, tx, tw, txs, tws, ty, th, tb, p);
    LQ_CUDA(cudaGetLastError());
}

size_t al256(size_t v) { return (v + 255) & ~(size_t)255; }

// The backward's workspace: the weight in bf16, dy's rows where they have to be copied (f32: three bf16 terms), and the
// product's partial sums (f32: the products of those terms).
struct DxSpace {
    int64_t ld;  // of the copied rows: the tensor maps want 16 bytes
    size_t rows, part, bytes;
};
DxSpace dx_space(int64_t n, int64_t m, int64_t k, int dtype) {
    DxSpace s;
    s.ld = (m + 7) / 8 * 8;
    s.rows = al256((size_t)m * k * 2);
    s.part = s.rows + (dtype == LQ_F32 ? al256((size_t)3 * n * s.ld * 2) : (s.ld != m ? al256((size_t)n * s.ld * 2) : 0));
    s.bytes = s.part + (dtype == LQ_F32 ? lq_tc_gemm_nn_part_bytes(3 * n, k, m, false) : lq_tc_gemm_nn_part_bytes(n, k, m, true));
    return s;
}

void quantize(const void* x, int dtype, int64_t rows, int64_t k, int64_t ld, void* codes, void* scales, int dev, cudaStream_t st) {
    const int64_t pad = row_tiles(rows) * 128;
    const unsigned grid = grid_of((pad * runs_of(k) + 7) / 8, lq_tc_sm_count(dev), 16);
    const int vec = al16(x) && (ld * (dtype == LQ_F32 ? 4 : 2)) % 16 == 0;
    LqProf prof(LQ_K_QUANT, st);
    if (dtype == LQ_F32)
        mx4_quantize_kernel<float><<<grid, 256, 0, st>>>((const float*)x, rows, (int)k, ld, vec, pad, (uint32_t*)codes, (uint8_t*)scales);
    else
        mx4_quantize_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>((const __nv_bfloat16*)x, rows, (int)k, ld, vec, pad, (uint32_t*)codes,
                                                                 (uint8_t*)scales);
    LQ_CUDA(cudaGetLastError());
}

void product(const void* x_codes, const void* x_scales, int64_t n, const void* w_codes, const void* w_scales, int64_t m, int64_t k,
             const float* bias, void* y, int y_dtype, bool early_w, int dev, cudaStream_t st, const LoraOperands* lora = nullptr) {
    const int sms = lq_tc_sm_count(dev), bn = bn_of(n);
    ProductParams p;
    p.w_scales = (const uint8_t*)w_scales;
    p.x_scales = (const uint8_t*)x_scales;
    p.m = (int)m;
    p.n = (int)n;
    p.kb = (int)((k + 255) / 256);
    p.w_tiles = (int)((m + 127) / 128);
    p.x_tiles = (int)((n + bn - 1) / bn);
    p.splits = splits_of((int64_t)p.w_tiles * p.x_tiles, p.kb, sms);
    p.lora = 0;
    p.early_w = early_w;
    p.bias = bias;
    p.y = y;
    p.y_f32 = y_dtype == LQ_F32;
    p.status = lq_tc_status_word(dev);
    if (use_pair(n, m)) launch_pair(p, w_codes, x_codes, k, lora, dev, sms, st);
    else if (bn == 16) launch_stream<16>(p, w_codes, x_codes, k, st);
    else if (bn == 32) launch_stream<32>(p, w_codes, x_codes, k, st);
    else if (bn == 64) launch_stream<64>(p, w_codes, x_codes, k, st);
    else launch_stream<128>(p, w_codes, x_codes, k, st);
}

// ---- with an adapter ------------------------------------------------------------------------------
// y = base + h . B for few tokens (or few outputs): base [n, m] the product in f32, h = s * H [n, ext] and B [r, m] in bf16, y
// rounded once, as the pair kernel's is.  A thread owns two columns of eight rows, base fetched ahead of the sums (240 blocks of
// 128 threads at 77 x 6144: 4.6 us; with 120 blocks of 256 and y last 6.9); launch and latency bound it.  The whole call, rank 16,
// takes 26.2 us as a graph, with a bf16 base that y rounded again 25.9.
constexpr int kDeltaRows = 8;
constexpr int kDeltaThreads = 128;
__global__ void __launch_bounds__(kDeltaThreads) mx4_add_delta_kernel(const float* __restrict__ base, __nv_bfloat16* __restrict__ y,
                                                            const __nv_bfloat16* __restrict__ h, const __nv_bfloat16* __restrict__ b,
                                                            int64_t n, int64_t m, int r, int ext) {
    extern __shared__ float hs[];  // [rank][row]
    const int64_t row0 = (int64_t)blockIdx.y * kDeltaRows, col = ((int64_t)blockIdx.x * kDeltaThreads + threadIdx.x) * 2;
    float2 acc[kDeltaRows] = {};  // fetched ahead of the sums
    if (col < m) {  // m is even
#pragma unroll
        for (int i = 0; i < kDeltaRows; ++i)
            if (row0 + i < n) acc[i] = *(const float2*)(base + (row0 + i) * m + col);
    }
    for (int i = threadIdx.x; i < r * kDeltaRows; i += kDeltaThreads) {
        const int row = i / r, j = i - row * r;
        hs[j * kDeltaRows + row] = row0 + row < n ? __bfloat162float(h[(row0 + row) * ext + j]) : 0.f;
    }
    __syncthreads();
    if (col >= m) return;
#pragma unroll 8
    for (int j = 0; j < r; ++j) {
        const float2 w = __bfloat1622float2(*(const __nv_bfloat162*)(b + j * m + col));
#pragma unroll
        for (int i = 0; i < kDeltaRows; ++i) {
            acc[i].x = fmaf(hs[j * kDeltaRows + i], w.x, acc[i].x);
            acc[i].y = fmaf(hs[j * kDeltaRows + i], w.y, acc[i].y);
        }
    }
#pragma unroll
    for (int i = 0; i < kDeltaRows; ++i)
        if (row0 + i < n) *(__nv_bfloat162*)(y + (row0 + i) * m + col) = __floats2bfloat162_rn(acc[i].x, acc[i].y);
}

// The forward's workspace: the quantised x, s * H, H where the caller does not keep it, the partial sums of H, and the product
// in f32 where the delta is added by a kernel of its own.
struct LoraSpace {
    size_t ext, h, part, base, bytes;
};
LoraSpace lora_space(int64_t n, int64_t m, int64_t k, int r) {
    LoraSpace s;
    s.ext = al256(lq_mx4_linear_workspace_bytes(n, k));
    s.h = s.ext + al256((size_t)n * lq_tc_ext_width(r) * 2);
    s.part = s.h + al256((size_t)n * r * 4);
    s.base = s.part + al256(lq_tc_lora_down_bytes(n, r));
    s.bytes = s.base + (use_pair(n, m) ? 0 : (size_t)n * m * 4);
    return s;
}
lq_weight lora_weight(const void* codes, const void* scales, int64_t m, int64_t k, int dev) {
    lq_weight w;
    w.device = dev;
    w.scheme = kSchemeMx4;
    w.M = m;
    w.K = k;
    w.packed = const_cast<void*>(codes);
    w.mx4_scales = scales;
    return w;
}
void check_lora(int64_t n, int64_t m, int64_t k, int r, const void* mirror) {
    check_dims(n, k);
    check_dims(m, k);
    LQ_CHECK_ARG(r >= 1 && r <= 256, "LoRA rank must be in [1, 256]");
    LQ_CHECK_ARG(m >= 8 && m % 8 == 0, "with an adapter d_out must be a positive multiple of 8");
    LQ_CHECK_ARG(mirror && ((uintptr_t)mirror & 255) == 0, "a 256-byte aligned mirror of the factors is needed");
}

}  // namespace

void lq_mx4_launch_dequant(const void* codes, const void* scales, int64_t rows, int64_t k, void* out, int out_dtype, cudaStream_t st) {
    const unsigned grid = grid_of((rows * runs_of(k) + 7) / 8, lq_tc_sm_count(current_device()), 16);
    LqProf prof(LQ_K_DEQUANT, st);
    if (out_dtype == LQ_F32)
        mx4_dequantize_kernel<float><<<grid, 256, 0, st>>>((const uint32_t*)codes, (const uint8_t*)scales, rows, (int)k, (float*)out);
    else
        mx4_dequantize_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>((const uint32_t*)codes, (const uint8_t*)scales, rows, (int)k,
                                                                   (__nv_bfloat16*)out);
    LQ_CUDA(cudaGetLastError());
}

extern "C" {

size_t lq_mx4_scale_bytes(int64_t rows, int64_t k) {
    if (rows < 1 || k < 32) return 0;
    return (size_t)row_tiles(rows) * k_tiles(k) * kTile;
}

int lq_mx4_quantize(const void* x, int dtype, int64_t rows, int64_t k, int64_t ld, void* codes, void* scales, void* stream) {
    return guarded_call([&] {
        LQ_CHECK_ARG(dtype == LQ_F32 || dtype == LQ_BF16, "dtype must be LQ_F32 or LQ_BF16");
        check_dims(rows, k);
        if (rows == 0) return;
        LQ_CHECK_ARG(x != nullptr, "NULL argument");
        check_tensor(codes, scales);
        LQ_CHECK_ARG(ld >= k || rows == 1, "rows overlap: the row stride is below their length");
        quantize(x, dtype, rows, k, ld, codes, scales, current_device(), (cudaStream_t)stream);
    });
}

int lq_mx4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t k, void* out, int out_dtype, void* stream) {
    return guarded_call([&] {
        LQ_CHECK_ARG(out_dtype == LQ_F32 || out_dtype == LQ_BF16, "dtype must be LQ_F32 or LQ_BF16");
        check_dims(rows, k);
        if (rows == 0) return;
        check_tensor(codes, scales);
        LQ_CHECK_ARG(out && al16(out), "the output must be 16-byte aligned");
        lq_mx4_launch_dequant(codes, scales, rows, k, out, out_dtype, (cudaStream_t)stream);
    });
}

int lq_mx4_matmul(const void* x_codes, const void* x_scales, int64_t n, const void* w_codes, const void* w_scales, int64_t m,
                  int64_t k, const float* bias, void* y, int y_dtype, void* stream) {
    return guarded_call([&] {
        LQ_CHECK_ARG(y_dtype == LQ_F32 || y_dtype == LQ_BF16, "dtype must be LQ_F32 or LQ_BF16");
        check_dims(n, k);
        check_dims(m, k);
        if (n == 0 || m == 0) return;
        check_tensor(x_codes, x_scales);
        check_tensor(w_codes, w_scales);
        LQ_CHECK_ARG(y != nullptr, "NULL argument");
        product(x_codes, x_scales, n, w_codes, w_scales, m, k, bias, y, y_dtype, false, current_device(), (cudaStream_t)stream);
    });
}

size_t lq_mx4_linear_workspace_bytes(int64_t n, int64_t k) {
    if (n < 1 || k < 32) return 0;
    return al256((size_t)n * k / 2) + lq_mx4_scale_bytes(n, k);
}

int lq_mx4_linear(const void* x, int dtype, int64_t n, int64_t ldx, const void* w_codes, const void* w_scales, int64_t m, int64_t k,
                  const float* bias, void* y, void* ws, size_t ws_bytes, void* stream) {
    return guarded_call([&] {
        LQ_CHECK_ARG(dtype == LQ_F32 || dtype == LQ_BF16, "dtype must be LQ_F32 or LQ_BF16");
        check_dims(n, k);
        check_dims(m, k);
        if (n == 0 || m == 0) return;
        check_tensor(w_codes, w_scales);
        LQ_CHECK_ARG(x && y, "NULL argument");
        LQ_CHECK_ARG(ldx >= k || n == 1, "rows overlap: the row stride is below their length");
        LQ_CHECK_ARG(ws && ((uintptr_t)ws & 255) == 0, "a 256-byte aligned workspace is needed");
        const int dev = current_device();
        const size_t cb = al256((size_t)n * k / 2);
        if (ws_bytes < lq_mx4_linear_workspace_bytes(n, k))
            throw LqError(LQ_ERR_WORKSPACE, "workspace too small for the microscaled linear");
        uint8_t* codes = (uint8_t*)ws;
        quantize(x, dtype, n, k, ldx, codes, codes + cb, dev, (cudaStream_t)stream);
        product(codes, codes + cb, n, w_codes, w_scales, m, k, bias, y, dtype, true, dev, (cudaStream_t)stream);
    });
}

size_t lq_mx4_matmul_dx_workspace_bytes(int64_t n, int64_t m, int64_t k, int dtype) {
    if (n < 1 || m < 1 || k < 32) return 0;
    return dx_space(n, m, k, dtype).bytes;
}

int lq_mx4_matmul_dx(const void* dy, int dtype, int64_t n, const void* w_codes, const void* w_scales, int64_t m, int64_t k, void* dx,
                     void* ws, size_t ws_bytes, void* stream) {
    return guarded_call([&] {
        LQ_CHECK_ARG(dtype == LQ_F32 || dtype == LQ_BF16, "dtype must be LQ_F32 or LQ_BF16");
        check_dims(n, k);
        check_dims(m, k);
        if (n == 0) return;
        LQ_CHECK_ARG(dx && al16(dx), "dx must be 16-byte aligned");
        cudaStream_t st = (cudaStream_t)stream;
        if (m == 0) {
            LQ_CUDA(cudaMemsetAsync(dx, 0, (size_t)n * k * (dtype == LQ_F32 ? 4 : 2), st));
            return;
        }
        LQ_CHECK_ARG(dy != nullptr, "NULL argument");
        check_tensor(w_codes, w_scales);
        LQ_CHECK_ARG(ws && ((uintptr_t)ws & 255) == 0, "a 256-byte aligned workspace is needed");
        if (ws_bytes < lq_mx4_matmul_dx_workspace_bytes(n, m, k, dtype))
            throw LqError(LQ_ERR_WORKSPACE, "workspace too small for the microscaled backward");
        lq_mx4_launch_dequant(w_codes, w_scales, m, k, ws, LQ_BF16, st);
        const DxSpace sp = dx_space(n, m, k, dtype);
        const int sms = lq_tc_sm_count(current_device());
        __nv_bfloat16* rows = (__nv_bfloat16*)((uint8_t*)ws + sp.rows);
        float* part = (float*)((uint8_t*)ws + sp.part);
        const size_t part_bytes = sp.bytes - sp.part;
        if (dtype == LQ_F32) {
            {
                LqProf prof(LQ_K_PREP, st);
                split3_kernel<<<grid_of((n * sp.ld + 255) / 256, sms, 16), 256, 0, st>>>((const float*)dy, n, m, sp.ld, rows);
                LQ_CUDA(cudaGetLastError());
            }
            const int ranges = lq_tc_gemm_nn(rows, sp.ld, ws, k, nullptr, part, part_bytes, 3 * n, k, m, st);
            LqProf prof(LQ_K_REDUCE, st);
            join3_kernel<<<grid_of((n * k / 4 + 255) / 256, sms, 16), 256, 0, st>>>((const float4*)part, n * k / 4, ranges, (float4*)dx);
            LQ_CUDA(cudaGetLastError());
            return;
        }
        const void* src = dy;
        if (sp.ld != m) {
            LqProf prof(LQ_K_PREP, st);
            pad_rows_kernel<<<grid_of((n * sp.ld + 255) / 256, sms, 16), 256, 0, st>>>((const __nv_bfloat16*)dy, n, m, sp.ld, rows);
            LQ_CUDA(cudaGetLastError());
            src = rows;
        } else {
            LQ_CHECK_ARG(al16(dy), "dy must be 16-byte aligned");
        }
        lq_tc_gemm_nn(src, sp.ld, ws, k, dx, part, part_bytes, n, k, m, st);
    });
}

size_t lq_mx4_lora_workspace_bytes(int64_t n, int64_t m, int64_t k, int rank, int backward) {
    if (n < 1 || m < 1 || k < 32 || rank < 1 || rank > 256) return 0;
    if (!backward) return lora_space(n, m, k, rank).bytes;
    const lq_weight w = lora_weight(nullptr, nullptr, m, k, 0);
    return lq_tc_workspace_bytes(&w, n, rank);
}

int lq_mx4_lora_fwd(const void* x, int64_t n, const void* w_codes, const void* w_scales, int64_t m, int64_t k, const float* bias,
                    const void* mirror, int rank, float scaling, void* y, float* h_out, void* ws, size_t ws_bytes, void* stream) {
    return guarded_call([&] {
        check_lora(n, m, k, rank, mirror);
        if (n == 0) return;
        check_tensor(w_codes, w_scales);
        LQ_CHECK_ARG(x && y && al16(x) && al16(y), "x and y must be 16-byte aligned");
        LQ_CHECK_ARG(ws && ((uintptr_t)ws & 255) == 0, "a 256-byte aligned workspace is needed");
        const LoraSpace sp = lora_space(n, m, k, rank);
        if (ws_bytes < sp.bytes) throw LqError(LQ_ERR_WORKSPACE, "workspace too small for the microscaled linear with an adapter");
        cudaStream_t st = (cudaStream_t)stream;
        const int dev = current_device(), sms = lq_tc_sm_count(dev), ext = lq_tc_ext_width(rank);
        const LqMirrorView mv = lq_tc_mirror_view(k, m, rank, mirror);
        uint8_t *codes = (uint8_t*)ws, *scales = codes + al256((size_t)n * k / 2);
        __nv_bfloat16* sh = (__nv_bfloat16*)(codes + sp.ext);
        lq_tc_lora_down(x, n, k, k, mv.At, rank, scaling, h_out ? h_out : (float*)(codes + sp.h), sh, codes + sp.part, sms, st);
        quantize(x, LQ_BF16, n, k, k, codes, scales, dev, st);
        if (use_pair(n, m)) {
            const LoraOperands lora{sh, mv.Bt, ext};
            product(codes, scales, n, w_codes, w_scales, m, k, bias, y, LQ_BF16, true, dev, st, &lora);
            return;
        }
        float* base = (float*)(codes + sp.base);
        product(codes, scales, n, w_codes, w_scales, m, k, bias, base, LQ_F32, true, dev, st);
        LqProf prof(LQ_K_REDUCE, st);
        const int64_t rows = (n + kDeltaRows - 1) / kDeltaRows;
        for (int64_t first = 0; first < rows; first += 65535) {
            const int64_t part = std::min<int64_t>(65535, rows - first), at = first * kDeltaRows;
            const dim3 grid((unsigned)((m + 2 * kDeltaThreads - 1) / (2 * kDeltaThreads)), (unsigned)part);
            mx4_add_delta_kernel<<<grid, kDeltaThreads, (size_t)rank * kDeltaRows * 4, st>>>(base + at * m, (__nv_bfloat16*)y + at * m,
                                                                                             sh + at * ext, mv.Bb, n - at, m, rank, ext);
            LQ_CUDA(cudaGetLastError());
        }
    });
}

int lq_mx4_lora_bwd(const void* dy, const void* x, const float* h, int64_t n, const void* w_codes, const void* w_scales, int64_t m,
                    int64_t k, const void* mirror, int rank, float scaling, void* dx, float* dA, float* dB, int accumulate, void* ws,
                    size_t ws_bytes, void* stream) {
    return guarded_call([&] {
        check_lora(n, m, k, rank, mirror);
        cudaStream_t st = (cudaStream_t)stream;
        if (n == 0) {  // sums over nothing
            if (dA && !accumulate) LQ_CUDA(cudaMemsetAsync(dA, 0, sizeof(float) * (size_t)k * rank, st));
            if (dB && !accumulate) LQ_CUDA(cudaMemsetAsync(dB, 0, sizeof(float) * (size_t)m * rank, st));
            return;
        }
        check_tensor(w_codes, w_scales);
        LQ_CHECK_ARG(dy && x && al16(dy) && al16(x) && al16(dx), "dy, x and dx must be 16-byte aligned");
        const lq_weight w = lora_weight(w_codes, w_scales, m, k, current_device());
        lq_tc_bwd(&w, dy, x, h, n, nullptr, nullptr, rank, scaling, dx, dA, dB, accumulate, ws, ws_bytes, st, mirror);
    });
}

}  // extern "C"
