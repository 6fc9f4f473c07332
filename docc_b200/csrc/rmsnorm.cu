// RMS norm with the residual's addition, and the same norm with an 8-bit output.
//
//   s = x + r,  S = round(s),  y = s * rsqrt(mean(s^2) + eps) * gamma,  Y = round(y)  or  Q = e4m3(y / scale_g)
//
// Bandwidth bound: x and r are read once, S and Y (or Q and its scales) written once. s stays in fp32 between the sum of
// squares and the output, so each output is rounded once. Rows of 8192 x 4096 bf16 with residual and 8-bit output: 236 MB, 45.6 us with
// fresh outputs per call (5.2 TB/s, 0.79 of the measured copy), 41.4 us replayed on the same ones; 8 rows of 1024: 2.1 us.
#include <cuda_fp8.h>

#include "common.cuh"
#include "device_math.cuh"
#include "ptx.cuh"

namespace docc_b200 {
namespace {

constexpr int64_t kRmsMaxCols = 32768;  // the row is staged in shared memory in fp32: 128 KB of 227
constexpr int kRmsGroup = 128, kRmsLoads = 4, kRmsWarpCols = 1024;
constexpr float kE4m3Max = 448.f;

// Maximum that keeps a NaN, so that a group holding one gets a NaN scale instead of a plausible one.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Of magnitudes: their bits are ordered as unsigned numbers, NaN above everything.
__device__ __forceinline__ float warp_max_nan(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); }
// What turns a group's values into codes: q = e4m3(y / scale), scale = max|y| / 448. The quotient is divided out only where it decides:
// y times the rounded reciprocal of the scale is off by 2^-23 of the value at most and the rounded quotient by 2^-24, so where both
// ends of +-2^-21 around that product have the same code, the quotient has it, too. Some 15 values in a million lie nearer to the middle
// between two codes. The second conversion costs 0.7 us of 41 at 8192 x 4096 and 0.6 of 10.6 at 1021 x 5003;
// a division per value cost 10 of 54.
// A scale that rounded to 0 gives codes of 0. One below fp32's smallest normal number may have no finite reciprocal: the ends 0 and NaN
// never agree. A scale of inf has the reciprocal 0, a NaN makes every code a NaN.
__device__ __noinline__ uint32_t quotient_codes(float a, float b, float scale) {  // rare, so a call: the row kernel's loops stay short
    return __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(a, scale), __fdiv_rn(b, scale)), __NV_SATFINITE, __NV_E4M3);
}
struct Quantiser {
    float low, high, scale;
    __device__ __forceinline__ explicit Quantiser(float top) {
        scale = __fdiv_rn(top, kE4m3Max);
        const float inv = scale == 0.f ? 0.f : __fdiv_rn(1.f, scale);
        const bool tiny = scale > 0.f && scale < 0x1p-126f;
        low = tiny ? 0.f : inv * (1.f - 0x1p-21f);
        high = tiny ? NAN : inv * (1.f + 0x1p-21f);
    }
    static __device__ __forceinline__ uint32_t codes(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }
    static __device__ __forceinline__ uint32_t codes(const float* y, float by) {  // of four, taken `by` times
        float2 f, g;
        asm("{\n.reg .b64 a, k;\nmov.b64 k, {%4, %4};\nmov.b64 a, {%2, %3};\nmul.rn.f32x2 a, a, k;\nmov.b64 {%0, %1}, a;\n}"
            : "=f"(f.x), "=f"(f.y) : "f"(y[0]), "f"(y[1]), "f"(by));
        asm("{\n.reg .b64 a, k;\nmov.b64 k, {%4, %4};\nmov.b64 a, {%2, %3};\nmul.rn.f32x2 a, a, k;\nmov.b64 {%0, %1}, a;\n}"
            : "=f"(g.x), "=f"(g.y) : "f"(y[2]), "f"(y[3]), "f"(by));
        return codes(f.x, f.y) | codes(g.x, g.y) << 16;
    }
    template <int N> __device__ __forceinline__ void all(const float (&y)[N], uint32_t (&c)[N / 4]) const {
        uint32_t differ = 0;
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            c[i] = codes(y + 4 * i, low);
            differ |= c[i] ^ codes(y + 4 * i, high);
        }
        if (differ) {
#pragma unroll
            for (int i = 0; i < N / 4; i++)
                c[i] = codes(__fdiv_rn(y[4 * i], scale), __fdiv_rn(y[4 * i + 1], scale)) |
                       codes(__fdiv_rn(y[4 * i + 2], scale), __fdiv_rn(y[4 * i + 3], scale)) << 16;
        }
    }
    __device__ __forceinline__ uint32_t two(float a, float b) const {
        const uint32_t c = codes(a * low, b * low);
        return c == codes(a * high, b * high) ? c : quotient_codes(a, b, scale);
    }
};

template <int N> __device__ __forceinline__ void store_codes(uint8_t* q, const float (&y)[N], const Quantiser& by) {
    uint32_t c[N / 4];
    by.all(y, c);
    if constexpr (N == 8) *reinterpret_cast<uint2*>(q) = make_uint2(c[0], c[1]);  // aligned: cols and the row's first code are multiples of N
    else *reinterpret_cast<uint32_t*>(q) = c[0];
}

struct RmsArgs {
    int64_t rows, cols, ldx, ldr;
    float eps;
    const float* gamma;
    int64_t group;  // 8-bit output: columns per scale
};

// Rows whose operands are aligned for 16-byte accesses: TPR threads to a row, which stays in registers (VPT packs each). Eight blocks of
// 128 threads to an SM (64 registers instead of 72) took the 8192 x 4096 case from 42.2 to 38.6 us, nine or ten spill.
template <typename T, bool Q8, int TPR, int VPT>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, TPR == 128 ? 8 : 1) rmsnorm_kernel(const T* X, const T* R, T* S, T* Y, uint8_t* Q, float* scales,
                                                                       RmsArgs a) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    constexpr int VEC = 16 / sizeof(T), BLOCK = TPR < 128 ? 128 : TPR, RPB = BLOCK / TPR, WPR = TPR / 32;
    constexpr int LANES = kRmsGroup / VEC;  // lanes that hold a group of columns: 16 or 32
    using P = Pack<T, VEC>;
    __shared__ float red[2][RPB][WPR];
    const int t = threadIdx.x % TPR, rib = threadIdx.x / TPR, wir = t / 32, lane = threadIdx.x & 31;
    const int packs = int(a.cols / VEC);
    const int64_t row = int64_t(blockIdx.x) * RPB + rib;
    const bool ok = row < a.rows;
    const P* x = reinterpret_cast<const P*>(X + row * a.ldx);
    const P* r = reinterpret_cast<const P*>(R + row * a.ldr);
    P px[VPT], pr[VPT];
#pragma unroll
    for (int i = 0; i < VPT; i++)
        if (ok && i * TPR + t < packs) px[i] = load_pack(x + i * TPR + t);
    if (R) {
#pragma unroll
        for (int i = 0; i < VPT; i++)
            if (ok && i * TPR + t < packs) pr[i] = load_pack(r + i * TPR + t);
    }
    float v[VPT][VEC];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int p = i * TPR + t;
        const bool in = ok && p < packs;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            v[i][e] = in ? to_float(px[i].v[e]) : 0.f;
            if (R && in) v[i][e] += to_float(pr[i].v[e]);
            ss = fmaf(v[i][e], v[i][e], ss);
        }
        if (S && in) {
            P ps;
#pragma unroll
            for (int e = 0; e < VEC; e++) ps.v[e] = from_float<T>(v[i][e]);
            store_pack(reinterpret_cast<P*>(S + row * a.cols) + p, ps);
        }
    }
    ss = warp_sum_f(ss);
    if constexpr (WPR > 1) {
        if (lane == 0) red[0][rib][wir] = ss;
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; w++) ss += red[0][rib][w];
    }
    const float rstd = rsqrtf(ss / float(a.cols) + a.eps);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int p = i * TPR + t;
        float g[VEC];
        if (a.gamma && p < packs) {
#pragma unroll
            for (int h = 0; h < VEC / 4; h++) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(a.gamma) + p * (VEC / 4) + h);
                g[4 * h] = f.x; g[4 * h + 1] = f.y; g[4 * h + 2] = f.z; g[4 * h + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) g[e] = 1.f;
        }
#pragma unroll
        for (int e = 0; e < VEC; e++) v[i][e] = v[i][e] * rstd * g[e];
        if constexpr (!Q8) {
            if (ok && p < packs) {
                P py;
#pragma unroll
                for (int e = 0; e < VEC; e++) py.v[e] = from_float<T>(v[i][e]);
                store_pack(reinterpret_cast<P*>(Y + row * a.cols) + p, py);
            }
        } else if (p < packs) {  // 0 * inf in a column that does not exist would be a NaN
#pragma unroll
            for (int e = 0; e < VEC; e++) top = max_nan(top, fabsf(v[i][e]));
        }
        if constexpr (Q8) {
            if (a.group < a.cols) {
                float m = top;
                top = 0.f;
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                const Quantiser by(m);
                if (ok && p < packs) {
                    store_codes<VEC>(Q + row * a.cols + int64_t(p) * VEC, v[i], by);
                    if (lane % LANES == 0) scales[row * ((a.cols + kRmsGroup - 1) / kRmsGroup) + p / LANES] = by.scale;
                }
            }
        }
    }
    if constexpr (Q8) {
        if (a.group >= a.cols) {
            top = warp_max_nan(top);
            if constexpr (WPR > 1) {
                if (lane == 0) red[1][rib][wir] = top;
                __syncthreads();
                top = red[1][rib][0];
#pragma unroll
                for (int w = 1; w < WPR; w++) top = max_nan(top, red[1][rib][w]);
            }
            const Quantiser by(top);
#pragma unroll
            for (int i = 0; i < VPT; i++) {
                const int p = i * TPR + t;
                if (ok && p < packs) store_codes<VEC>(Q + row * a.cols + int64_t(p) * VEC, v[i], by);
            }
            if (ok && t == 0) scales[row] = by.scale;
        }
    }
}

// Any width and alignment: one block per row, the row staged in shared memory, loops that stay loops. Bound by the instructions of
// these loops (one element per load, conversion and store, two more walks through shared memory), not by anything in the data: 1021 rows of
// 5003 with an 8-bit output take 10.6 us, 1.4 TB/s. The same in registers, unrolled over 20
// columns per thread, has half as many instructions and took 19.8 us: they no longer fit the instruction cache. On the 16-byte packs
// of the whole matrix, gamma moved into place by selects, it took 10.8.
// TPR threads to a row: a block, or a warp.
template <typename T, bool Q8, int TPR>
__global__ void __launch_bounds__(256) rmsnorm_row_kernel(const T* X, const T* R, T* S, T* Y, uint8_t* Q, float* scales, RmsArgs a) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    constexpr int RPB = 256 / TPR, WPR = TPR / 32;
    extern __shared__ float rows_s[];
    __shared__ float red[8];
    const int t = threadIdx.x % TPR, lane = t & 31, warp = t >> 5;
    const int cols = int(a.cols);
    float* row_s = rows_s + int(threadIdx.x / TPR) * cols;
    auto sync = [] {
        if constexpr (WPR > 1) __syncthreads();
        else __syncwarp();
    };
    for (int64_t row = int64_t(blockIdx.x) * RPB + threadIdx.x / TPR; row < a.rows; row += int64_t(gridDim.x) * RPB) {
        const T* x = X + row * a.ldx;
        const T* r = R ? R + row * a.ldr : nullptr;
        float ss = 0.f;
        for (int c0 = t; c0 < cols; c0 += TPR * kRmsLoads) {  // all loads of a round before the first use
            T vx[kRmsLoads], vr[kRmsLoads];
#pragma unroll
            for (int i = 0; i < kRmsLoads; i++)
                if (c0 + i * TPR < cols) vx[i] = x[c0 + i * TPR];
            if (r) {
#pragma unroll
                for (int i = 0; i < kRmsLoads; i++)
                    if (c0 + i * TPR < cols) vr[i] = r[c0 + i * TPR];
            }
#pragma unroll
            for (int i = 0; i < kRmsLoads; i++) {
                const int c = c0 + i * TPR;
                if (c >= cols) break;
                const float v = r ? to_float(vx[i]) + to_float(vr[i]) : to_float(vx[i]);
                row_s[c] = v;
                if (S) S[row * a.cols + c] = from_float<T>(v);
                ss = fmaf(v, v, ss);
            }
        }
        if constexpr (WPR > 1) ss = block_sum_f(ss, red);
        else ss = warp_sum_f(ss);
        const float rstd = rsqrtf(ss / float(cols) + a.eps);
        if constexpr (!Q8) {
            for (int c = t; c < cols; c += TPR) {
                const float y = row_s[c] * rstd;
                Y[row * a.cols + c] = from_float<T>(a.gamma ? y * a.gamma[c] : y);
            }
        } else if (a.group >= a.cols) {
            float m = 0.f;
            for (int c = t; c < cols; c += TPR) {
                const float y = a.gamma ? row_s[c] * rstd * a.gamma[c] : row_s[c] * rstd;
                row_s[c] = y;
                m = max_nan(m, fabsf(y));
            }
            m = warp_max_nan(m);
            if constexpr (WPR > 1) {
                __syncthreads();
                if (lane == 0) red[warp] = m;
                __syncthreads();
                m = red[0];
                for (int w = 1; w < WPR; w++) m = max_nan(m, red[w]);
            }
            const Quantiser by(m);
            for (int c = t; c < cols; c += 2 * TPR) {
                const bool second = c + TPR < cols;
                const uint32_t codes = by.two(row_s[c], second ? row_s[c + TPR] : 0.f);
                Q[row * a.cols + c] = uint8_t(codes);
                if (second) Q[row * a.cols + c + TPR] = uint8_t(codes >> 8);
            }
            if (t == 0) scales[row] = by.scale;
        } else {  // a group per warp in turn
            sync();
            const int64_t groups = (a.cols + a.group - 1) / a.group;
            for (int g = warp; g < groups; g += WPR) {
                const int c0 = int(g * a.group), c1 = int(c0 + a.group < a.cols ? c0 + a.group : a.cols);
                float y[kRmsGroup / 32], m = 0.f;
#pragma unroll
                for (int i = 0; i < kRmsGroup / 32; i++) {
                    const int c = c0 + lane + 32 * i;
                    y[i] = 0.f;
                    if (c < c1) y[i] = a.gamma ? row_s[c] * rstd * a.gamma[c] : row_s[c] * rstd;
                    m = max_nan(m, fabsf(y[i]));
                }
                const Quantiser by(warp_max_nan(m));
                uint32_t codes[1];
                by.all(y, codes);
#pragma unroll
                for (int i = 0; i < kRmsGroup / 32; i++) {
                    const int c = c0 + lane + 32 * i;
                    if (c < c1) Q[row * a.cols + c] = uint8_t(codes[0] >> (8 * i));
                }
                if (lane == 0) scales[row * groups + g] = by.scale;
            }
        }
        sync();  // row_s and red are reused by the next row
    }
}

template <typename T, bool Q8, int TPR, int VPT>
int launch_rms(Ctx* ctx, const RmsArgs& a, const void* X, const void* R, void* S, void* Y, void* Q, void* scales) {
    constexpr int BLOCK = TPR < 128 ? 128 : TPR;
    DOCC_CUDA_TRY(launch_pdl(rmsnorm_kernel<T, Q8, TPR, VPT>, dim3(unsigned(ceil_div(a.rows, BLOCK / TPR))), dim3(BLOCK), 0, ctx->stream,
                             static_cast<const T*>(X), static_cast<const T*>(R), static_cast<T*>(S), static_cast<T*>(Y),
                             static_cast<uint8_t*>(Q), static_cast<float*>(scales), a));
    return after_launch(ctx, "rmsnorm_kernel");
}

template <typename T, bool Q8, int TPR>
int launch_rms_row(Ctx* ctx, const RmsArgs& a, const void* X, const void* R, void* S, void* Y, void* Q, void* scales) {
    constexpr int RPB = 256 / TPR;
    const size_t smem = size_t(a.cols) * 4 * RPB;
    auto kernel = rmsnorm_row_kernel<T, Q8, TPR>;
    static std::atomic<unsigned> done{0};
    DOCC_TRY(set_smem(ctx, done, kernel, int((TPR == 32 ? kRmsWarpCols : kRmsMaxCols) * 4 * RPB)));
    const int64_t cap = int64_t(ctx->sm_count) * 8, blocks = ceil_div(a.rows, RPB);
    const int grid = int(blocks < cap ? blocks : cap);
    DOCC_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(256), smem, ctx->stream, static_cast<const T*>(X), static_cast<const T*>(R),
                             static_cast<T*>(S), static_cast<T*>(Y), static_cast<uint8_t*>(Q), static_cast<float*>(scales), a));
    return after_launch(ctx, "rmsnorm_row_kernel");
}

template <typename T, bool Q8>
int rms_device(Ctx* ctx, const RmsArgs& a, const void* X, const void* R, void* S, void* Y, void* Q, void* scales) {
    constexpr int VEC = 16 / sizeof(T);
    bool aligned = a.cols % VEC == 0 && a.ldx % VEC == 0 && (!R || a.ldr % VEC == 0) && a.rows < (int64_t(1) << 31);
    for (const void* p : {X, R, static_cast<const void*>(S), static_cast<const void*>(Y), static_cast<const void*>(Q),
                          static_cast<const void*>(a.gamma)})
        aligned = aligned && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    if (aligned) {
        const int64_t packs = a.cols / VEC;
        if (packs <= 32) return launch_rms<T, Q8, 32, 1>(ctx, a, X, R, S, Y, Q, scales);
        if (packs <= 128) return launch_rms<T, Q8, 32, 4>(ctx, a, X, R, S, Y, Q, scales);
        if (packs <= 512) return launch_rms<T, Q8, 128, 4>(ctx, a, X, R, S, Y, Q, scales);
        if (packs <= 1024) return launch_rms<T, Q8, 256, 4>(ctx, a, X, R, S, Y, Q, scales);
        if (packs <= 2048) return launch_rms<T, Q8, 512, 4>(ctx, a, X, R, S, Y, Q, scales);
        if (packs <= 4096) return launch_rms<T, Q8, 1024, 4>(ctx, a, X, R, S, Y, Q, scales);
    }
    // a warp per row where rows are short and enough to fill the SMs with warps: 9195 rows of 182 6.4 us against 22.0 with a block each,
    // 20000 of 801 35 against 75, but 300 of 501 4.7 against 2.7, and 5000 of 1501 without codes 24 against 15
    if (a.cols <= kRmsWarpCols && a.rows >= 8 * int64_t(ctx->sm_count)) return launch_rms_row<T, Q8, 32>(ctx, a, X, R, S, Y, Q, scales);
    return launch_rms_row<T, Q8, 256>(ctx, a, X, R, S, Y, Q, scales);
}

int rms_any(Ctx* ctx, int prec, const RmsArgs& a, const void* X, const void* R, void* S, void* Y, void* Q, void* scales) {
    const bool q8 = Q != nullptr;
    switch (prec) {
        case DOCC_B200_PREC_S:
            return q8 ? rms_device<float, true>(ctx, a, X, R, S, Y, Q, scales) : rms_device<float, false>(ctx, a, X, R, S, Y, Q, scales);
        case DOCC_B200_PREC_H:
            return q8 ? rms_device<__half, true>(ctx, a, X, R, S, Y, Q, scales) : rms_device<__half, false>(ctx, a, X, R, S, Y, Q, scales);
        default:
            return q8 ? rms_device<__nv_bfloat16, true>(ctx, a, X, R, S, Y, Q, scales)
                      : rms_device<__nv_bfloat16, false>(ctx, a, X, R, S, Y, Q, scales);
    }
}

int rms_checked(const char* what, int prec, const RmsArgs& a, const void* X, const void* R, void* S, void* Y, void* Q, void* scales,
                int flags) {
    DOCC_REQUIRE(prec == DOCC_B200_PREC_S || prec == DOCC_B200_PREC_B || prec == DOCC_B200_PREC_H,
                 "%s: precision %d not supported (use 's', 'b' or 'h')", what, prec);
    DOCC_REQUIRE(a.rows >= 0 && a.cols >= 0, "%s: negative extent", what);
    DOCC_REQUIRE(a.eps >= 0.f, "%s: eps must not be negative", what);
    Ctx* ctx;
    DOCC_TRY(get_ctx(&ctx));
    if (a.rows == 0 || a.cols == 0) {
        if (a.rows == 0 || a.group != 0 || !scales) return DOCC_B200_OK;
        // a scale per row: rows of nothing have scales of 0
        if (flags & DOCC_B200_FLAG_HOST_PTRS) memset(scales, 0, size_t(a.rows) * 4);
        else DOCC_CUDA_TRY(cudaMemsetAsync(scales, 0, size_t(a.rows) * 4, ctx->stream));
        return DOCC_B200_OK;
    }
    DOCC_REQUIRE(X && (Y || (Q && scales)), "%s: NULL data pointer", what);
    DOCC_REQUIRE(a.ldx >= a.cols && (!R || a.ldr >= a.cols), "%s: row stride below cols", what);
    if (a.cols > kRmsMaxCols) return set_error(DOCC_B200_ERR_UNSUPPORTED, "%s: cols %lld > %lld", what, (long long)a.cols, (long long)kRmsMaxCols);
    if (!(flags & DOCC_B200_FLAG_HOST_PTRS)) return rms_any(ctx, prec, a, X, R, S, Y, Q, scales);

    DOCC_REQUIRE(a.ldx == a.cols && (!R || a.ldr == a.cols), "%s: host pointers require contiguous rows", what);
    const size_t n = size_t(a.rows) * size_t(a.cols), es = prec_size(prec);
    const size_t n_scales = Q ? size_t(a.rows) * size_t(ceil_div(a.cols, a.group)) * 4 : 0;
    TempBuffers tmp;
    void *dX, *dR = nullptr, *dG = nullptr, *dS = nullptr, *dY = nullptr, *dQ = nullptr, *dScales = nullptr;
    RmsArgs d = a;
    DOCC_TRY(tmp.alloc(&dX, n * es));
    DOCC_CUDA_TRY(cudaMemcpyAsync(dX, X, n * es, cudaMemcpyHostToDevice, ctx->stream));
    if (R) {
        DOCC_TRY(tmp.alloc(&dR, n * es));
        DOCC_CUDA_TRY(cudaMemcpyAsync(dR, R, n * es, cudaMemcpyHostToDevice, ctx->stream));
    }
    if (a.gamma) {
        DOCC_TRY(tmp.alloc(&dG, size_t(a.cols) * 4));
        DOCC_CUDA_TRY(cudaMemcpyAsync(dG, a.gamma, size_t(a.cols) * 4, cudaMemcpyHostToDevice, ctx->stream));
        d.gamma = static_cast<const float*>(dG);
    }
    if (S) DOCC_TRY(tmp.alloc(&dS, n * es));
    if (Q) {
        DOCC_TRY(tmp.alloc(&dQ, n));
        DOCC_TRY(tmp.alloc(&dScales, n_scales));
    } else {
        DOCC_TRY(tmp.alloc(&dY, n * es));
    }
    DOCC_TRY(rms_any(ctx, prec, d, dX, dR, dS, dY, dQ, dScales));
    if (S) DOCC_CUDA_TRY(cudaMemcpyAsync(S, dS, n * es, cudaMemcpyDeviceToHost, ctx->stream));
    if (Q) {
        DOCC_CUDA_TRY(cudaMemcpyAsync(Q, dQ, n, cudaMemcpyDeviceToHost, ctx->stream));
        DOCC_CUDA_TRY(cudaMemcpyAsync(scales, dScales, n_scales, cudaMemcpyDeviceToHost, ctx->stream));
    } else {
        DOCC_CUDA_TRY(cudaMemcpyAsync(Y, dY, n * es, cudaMemcpyDeviceToHost, ctx->stream));
    }
    DOCC_CUDA_TRY(cudaStreamSynchronize(ctx->stream));
    return DOCC_B200_OK;
}

}  // namespace
}  // namespace docc_b200

using namespace docc_b200;

extern "C" int docc_b200_rmsnorm(int prec, int64_t rows, int64_t cols, const void* X, int64_t ldx, const void* residual, int64_t ldr,
                                 const void* gamma, double eps, void* S, void* Y, int flags) {
    const RmsArgs a{rows, cols, ldx, ldr, float(eps), static_cast<const float*>(gamma), cols};
    DOCC_REQUIRE(rows * cols == 0 || Y, "rmsnorm: NULL data pointer");
    return rms_checked("rmsnorm", prec, a, X, residual, S, Y, nullptr, nullptr, flags);
}

extern "C" int docc_b200_rmsnorm_q8(int prec, int64_t rows, int64_t cols, const void* X, int64_t ldx, const void* residual, int64_t ldr,
                                    const void* gamma, double eps, int64_t group, void* S, void* Q, void* scales, int flags) {
    DOCC_REQUIRE(group == 0 || group == kRmsGroup, "rmsnorm_q8: group %lld (use 0 for whole rows or %d)", (long long)group, kRmsGroup);
    const RmsArgs a{rows, cols, ldx, ldr, float(eps), static_cast<const float*>(gamma), group ? group : cols};
    DOCC_REQUIRE(rows * cols == 0 || (Q && scales), "rmsnorm_q8: NULL data pointer");
    return rms_checked("rmsnorm_q8", prec, a, X, residual, S, nullptr, Q, scales, flags);
}
