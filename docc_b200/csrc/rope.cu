// Rotary positions, alone and together with the write of a step's keys and values into a paged cache.
//
// Pair i < R/2 of a head turns by a = position * inv_freq[i]: (u, v) -> m (u cos a - v sin a, v cos a + u sin a). In fp32 the
// product is off by position * 2^-24 radians, a quarter of a turn at ten million and visible from a few thousand on, so the
// angle is formed in fp64 as a number of turns, reduced to [-1/2, 1/2] there, and only then handed to sincospif.
//
// Bandwidth bound: q, k and v are read once, q and the cache's places written once. 8192 tokens of 32 + 8 heads of 128 in fp16: 201 MB,
// 37.1 us with fresh outputs (5.4 TB/s, 0.83 of the measured copy); 16 tokens 2.05 us, a launch's time.
#include "common.cuh"
#include "device_math.cuh"
#include "ptx.cuh"

namespace docc_b200 {
namespace {

struct RopeArgs {
    int64_t tokens, D, rotary;
    int interleaved;
    float mscale, sign;  // sign -1: the transpose
    const int64_t* positions;
    const double* inv_freq;
    int64_t num_pages, page_size;
    const int64_t* slots;  // nullptr: no cache
    DeviceStatus* status;
};
struct RopeTensor {
    const void* in;
    void* out;
    int64_t in_t, in_h, out_t, out_h, out_s;  // strides of the input, and of the output (token or page, head, place)
    int heads;
};

// Blocks (x, y): block x takes tokens, block y a share of the token's units. A unit is VEC pairs, i.e. two runs of VEC elements:
// rotary / 2 apart in the half layout, next to each other otherwise and in the part that is only copied. A thread has up to UNITS units
// and asks for all of them before the token's cosines and sines are worked out, once per block, for all heads.
constexpr int kRopeThreads = 256;

// Elements 2i and 2i + 1 of a run as fp32, and back (rounded once).
template <typename T> __device__ __forceinline__ float2 get2(const T* x) { return make_float2(to_float(x[0]), to_float(x[1])); }
template <> __device__ __forceinline__ float2 get2<__half>(const __half* x) { return __half22float2(*reinterpret_cast<const __half2*>(x)); }
template <typename T> __device__ __forceinline__ void put2(T* x, float a, float b) {
    x[0] = from_float<T>(a);
    x[1] = from_float<T>(b);
}
template <> __device__ __forceinline__ void put2<__half>(__half* x, float a, float b) { *reinterpret_cast<__half2*>(x) = __floats2half2_rn(a, b); }
template <> __device__ __forceinline__ void put2<__nv_bfloat16>(__nv_bfloat16* x, float a, float b) {
    *reinterpret_cast<__nv_bfloat162*>(x) = __floats2bfloat162_rn(a, b);
}

// The VEC pairs of a unit, turned in place.
template <typename T, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void turn_unit(Pack<T, VEC>& x0, Pack<T, VEC>& x1, const float2* cs) {
    if constexpr (VEC == 1) {
        const float f0 = to_float(x0.v[0]), f1 = to_float(x1.v[0]);
        x0.v[0] = from_float<T>(f0 * cs[0].x - f1 * cs[0].y);
        x1.v[0] = from_float<T>(f1 * cs[0].x + f0 * cs[0].y);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float4 two = *reinterpret_cast<const float4*>(cs + i);  // pairs i and i + 1; i even, so 16-byte aligned
            if constexpr (INTERLEAVED) {
                T* a = i < VEC / 2 ? &x0.v[2 * i] : &x1.v[2 * i - VEC];
                T* b = i + 1 < VEC / 2 ? &x0.v[2 * i + 2] : &x1.v[2 * i + 2 - VEC];
                const float2 f = get2(a), g = get2(b);
                put2(a, f.x * two.x - f.y * two.y, f.y * two.x + f.x * two.y);
                put2(b, g.x * two.z - g.y * two.w, g.y * two.z + g.x * two.w);
            } else {
                const float2 f = get2(&x0.v[i]), g = get2(&x1.v[i]);
                put2(&x0.v[i], f.x * two.x - g.x * two.y, f.y * two.z - g.y * two.w);
                put2(&x1.v[i], g.x * two.x + f.x * two.y, g.y * two.z + f.y * two.w);
            }
        }
    }
}

template <typename T, int VEC, bool INTERLEAVED, int UNITS>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(RopeTensor q, RopeTensor k, RopeTensor v, RopeArgs a) {
    using P = Pack<T, VEC>;
    extern __shared__ __align__(16) float2 turn_s[];  // cosine and sine of each pair, times mscale
    __shared__ int64_t place_s[2];      // page (-1: nothing is written) and place of the token
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int half = int(a.rotary / 2), D = int(a.D), turned = half / VEC, threads = int(blockDim.x);
    const int per_head = turned + (D - int(a.rotary) + 2 * VEC - 1) / (2 * VEC);
    const int units = (q.heads + k.heads + v.heads) * per_head, pass = threads * UNITS;
    for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        bool ready = false;
        for (int base = int(blockIdx.y) * pass; base < units; base += pass * int(gridDim.y)) {
            P x0[UNITS], x1[UNITS];
            int which[UNITS], unit[UNITS], d0[UNITS], d1[UNITS];
            int64_t out_at[UNITS];
#pragma unroll
            for (int j = 0; j < UNITS; j++) {
                const int w = base + j * threads + int(threadIdx.x);
                which[j] = -1;
                if (w >= units) continue;
                int h = w / per_head;
                const int u = w - h * per_head;
                const bool is_q = h < q.heads, is_v = h >= q.heads + k.heads;
                which[j] = is_q ? 0 : is_v ? 2 : 1;
                h -= is_q ? 0 : is_v ? q.heads + k.heads : q.heads;
                unit[j] = u;
                if (u >= turned) {
                    d0[j] = int(a.rotary) + (u - turned) * 2 * VEC;
                    d1[j] = d0[j] + VEC;
                } else {
                    d0[j] = INTERLEAVED ? u * 2 * VEC : u * VEC;
                    d1[j] = INTERLEAVED ? d0[j] + VEC : d0[j] + half;
                }
                const T* in = static_cast<const T*>(is_q ? q.in : is_v ? v.in : k.in) +
                              t * (is_q ? q.in_t : is_v ? v.in_t : k.in_t) + h * (is_q ? q.in_h : is_v ? v.in_h : k.in_h);
                out_at[j] = h * (is_q ? q.out_h : is_v ? v.out_h : k.out_h);
                x0[j] = load_pack(reinterpret_cast<const P*>(in + d0[j]));
                if (VEC > 1 || d1[j] < D) x1[j] = load_pack(reinterpret_cast<const P*>(in + d1[j]));
            }
            if (!ready) {
                ready = true;
                for (int i = threadIdx.x; i < half; i += threads) {
                    const double turns = double(a.positions[t]) * (a.inv_freq[i] * 0.15915494309189533577);
                    float c, s;
                    sincospif(2.f * float(turns - rint(turns)), &s, &c);
                    turn_s[i] = make_float2(a.mscale * c, a.mscale * a.sign * s);
                }
                if (a.slots && int(threadIdx.x) == threads - 1) {
                    const int64_t slot = a.slots[t];
                    // a cache of 2^32 places or more takes the long division
                    const int64_t page = slot < 0 ? -1
                                         : ((slot | a.page_size) >> 32) == 0 ? int64_t(uint32_t(slot) / uint32_t(a.page_size))
                                                                             : slot / a.page_size;
                    if (page >= a.num_pages) report_bad_index(a.status, kIndexSlot);
                    place_s[0] = page < a.num_pages ? page : -1;
                    place_s[1] = slot - page * a.page_size;
                }
                __syncthreads();
            }
#pragma unroll
            for (int j = 0; j < UNITS; j++) {
                if (which[j] < 0) continue;
                T* out;
                if (which[j] == 0) {
                    out = static_cast<T*>(q.out) + t * q.out_t + out_at[j];
                } else {
                    if (place_s[0] < 0) continue;
                    const bool is_v = which[j] == 2;
                    out = static_cast<T*>(is_v ? v.out : k.out) + place_s[0] * (is_v ? v.out_t : k.out_t) +
                          place_s[1] * (is_v ? v.out_s : k.out_s) + out_at[j];
                }
                if (unit[j] < turned && which[j] != 2) turn_unit<T, VEC, INTERLEAVED>(x0[j], x1[j], turn_s + unit[j] * VEC);
                *reinterpret_cast<P*>(out + d0[j]) = x0[j];
                if (VEC > 1 || d1[j] < D) *reinterpret_cast<P*>(out + d1[j]) = x1[j];
            }
        }
        __syncthreads();  // turn_s and place_s are the next token's
    }
}

template <typename T, int VEC, int UNITS>
int launch_rope_units(Ctx* ctx, const RopeTensor& q, const RopeTensor& k, const RopeTensor& v, const RopeArgs& a, int64_t units, bool share) {
    int64_t threads = ceil_div(ceil_div(units, UNITS), 32) * 32;
    if (threads > kRopeThreads) threads = kRopeThreads;
    const int64_t y = share ? ceil_div(units, threads * UNITS) : 1;
    const int64_t cap = int64_t(1) << 20;  // tokens beyond it are taken in turn
    const size_t smem = size_t(a.rotary / 2) * sizeof(float2);
    DOCC_CUDA_TRY(launch_pdl(a.interleaved ? rope_kernel<T, VEC, true, UNITS> : rope_kernel<T, VEC, false, UNITS>,
                             dim3(unsigned(a.tokens < cap ? a.tokens : cap), unsigned(y)), dim3(unsigned(threads)), smem, ctx->stream, q, k, v, a));
    return after_launch(ctx, "rope_kernel");
}
template <typename T, int VEC>
int launch_rope(Ctx* ctx, const RopeTensor& q, const RopeTensor& k, const RopeTensor& v, const RopeArgs& a) {
    const int64_t per_head = a.rotary / 2 / VEC + ceil_div(a.D - a.rotary, 2 * VEC);
    const int64_t units = (int64_t(q.heads) + k.heads + v.heads) * per_head;
    // Few tokens: a unit per thread, and as many blocks per token as that takes (16 tokens of 384 units: 2.1 us, with three units per
    // thread 2.8). Many: a block per token and three units per thread, so that the angles are worked out once and 96 bytes per thread
    // are on their way meanwhile (8192 tokens: 34.7 us; with two units 39, with one 41).
    if (a.tokens * ceil_div(units, kRopeThreads) <= 2 * int64_t(ctx->sm_count)) return launch_rope_units<T, VEC, 1>(ctx, q, k, v, a, units, true);
    return launch_rope_units<T, VEC, 3>(ctx, q, k, v, a, units, false);
}

template <typename T>
int rope_typed(Ctx* ctx, const RopeTensor& q, const RopeTensor& k, const RopeTensor& v, const RopeArgs& a) {
    auto fits = [&](int vec) {
        bool ok = a.rotary / 2 % vec == 0 && (a.D - a.rotary) % (2 * vec) == 0;
        for (const RopeTensor* x : {&q, &k, &v}) {
            if (x->heads == 0) continue;
            for (const void* p : {x->in, static_cast<const void*>(x->out)}) ok = ok && reinterpret_cast<uintptr_t>(p) % (vec * sizeof(T)) == 0;
            for (int64_t s : {x->in_t, x->in_h, x->out_t, x->out_h, x->out_s}) ok = ok && s % vec == 0;
        }
        return ok;
    };
    constexpr int VEC = 16 / sizeof(T);
    if (fits(VEC)) return launch_rope<T, VEC>(ctx, q, k, v, a);
    if (fits(VEC / 2)) return launch_rope<T, VEC / 2>(ctx, q, k, v, a);
    return launch_rope<T, 1>(ctx, q, k, v, a);
}
int rope_device(Ctx* ctx, int prec, const RopeTensor& q, const RopeTensor& k, const RopeTensor& v, const RopeArgs& a) {
    if (prec == DOCC_B200_PREC_S) return rope_typed<float>(ctx, q, k, v, a);
    if (prec == DOCC_B200_PREC_H) return rope_typed<__half>(ctx, q, k, v, a);
    return rope_typed<__nv_bfloat16>(ctx, q, k, v, a);
}

int rope_check(const char* what, int prec, int64_t tokens, int64_t heads, int64_t D, int64_t rotary, const RopeArgs& a) {
    DOCC_REQUIRE(prec == DOCC_B200_PREC_S || prec == DOCC_B200_PREC_B || prec == DOCC_B200_PREC_H,
                 "%s: precision %d not supported (use 's', 'b' or 'h')", what, prec);
    DOCC_REQUIRE(tokens >= 0 && heads >= 0 && D >= 0, "%s: negative extent", what);
    DOCC_REQUIRE(heads <= 65536 && D <= 8192, "%s: more than 65536 heads or a head of more than 8192 elements", what);
    DOCC_REQUIRE(rotary >= 0 && rotary <= D && rotary % 2 == 0, "%s: rotary_dim %lld must be even and at most D = %lld", what,
                 (long long)rotary, (long long)D);
    DOCC_REQUIRE(tokens == 0 || rotary == 0 || (a.positions && a.inv_freq), "%s: NULL positions or inv_freq", what);
    return DOCC_B200_OK;
}

}  // namespace
}  // namespace docc_b200

using namespace docc_b200;

extern "C" int docc_b200_rope(int prec, int64_t tokens, int64_t heads, int64_t D, int64_t rotary_dim, int interleaved, int inverse,
                              const void* X, const int64_t* x_strides, const int64_t* positions, const double* inv_freq, float mscale,
                              void* Y, const int64_t* y_strides, int flags) {
    RopeArgs a{tokens, D, rotary_dim, interleaved ? 1 : 0, mscale, inverse ? -1.f : 1.f, positions, inv_freq, 0, 1, nullptr, nullptr};
    DOCC_TRY(rope_check("rope", prec, tokens, heads, D, rotary_dim, a));
    Ctx* ctx;
    DOCC_TRY(get_ctx(&ctx));
    if (tokens * heads * D == 0) return DOCC_B200_OK;
    DOCC_REQUIRE(X && Y, "rope: NULL data pointer");
    RopeTensor x{X, Y, heads * D, D, heads * D, D, 0, int(heads)};
    if (x_strides) { x.in_t = x_strides[0]; x.in_h = x_strides[1]; }
    if (y_strides) { x.out_t = y_strides[0]; x.out_h = y_strides[1]; }
    const RopeTensor none{nullptr, nullptr, 0, 0, 0, 0, 0, 0};
    if (!(flags & DOCC_B200_FLAG_HOST_PTRS)) return rope_device(ctx, prec, x, none, none, a);
    DOCC_REQUIRE(!x_strides && !y_strides, "rope: host pointers require contiguous [tokens, heads, D] tensors");
    const size_t bytes = size_t(tokens) * size_t(heads * D) * prec_size(prec), pb = size_t(tokens) * 8, fb = size_t(rotary_dim / 2) * 8;
    TempBuffers tmp;
    void *dX, *dP, *dF;
    DOCC_TRY(tmp.alloc(&dX, bytes));
    DOCC_TRY(tmp.alloc(&dP, pb));
    DOCC_TRY(tmp.alloc(&dF, fb));
    DOCC_CUDA_TRY(cudaMemcpyAsync(dX, X, bytes, cudaMemcpyHostToDevice, ctx->stream));
    if (rotary_dim) {
        DOCC_CUDA_TRY(cudaMemcpyAsync(dP, positions, pb, cudaMemcpyHostToDevice, ctx->stream));
        DOCC_CUDA_TRY(cudaMemcpyAsync(dF, inv_freq, fb, cudaMemcpyHostToDevice, ctx->stream));
    }
    x.in = dX;
    x.out = dX;  // in place: a thread reads its pair before it writes it
    a.positions = static_cast<const int64_t*>(dP);
    a.inv_freq = static_cast<const double*>(dF);
    DOCC_TRY(rope_device(ctx, prec, x, none, none, a));
    DOCC_CUDA_TRY(cudaMemcpyAsync(Y, dX, bytes, cudaMemcpyDeviceToHost, ctx->stream));
    DOCC_CUDA_TRY(cudaStreamSynchronize(ctx->stream));
    return DOCC_B200_OK;
}

extern "C" int docc_b200_rope_append(int prec, int64_t tokens, int64_t Hq, int64_t Hkv, int64_t D, int64_t rotary_dim, int interleaved,
                                     const void* Q, const int64_t* q_strides, const void* K, const int64_t* k_strides, const void* V,
                                     const int64_t* v_strides, const int64_t* positions, const double* inv_freq, float mscale, void* Qout,
                                     const int64_t* qo_strides, void* Kcache, const int64_t* kc_strides, void* Vcache,
                                     const int64_t* vc_strides, int64_t num_pages, int64_t page_size, const int64_t* slots, int flags) {
    RopeArgs a{tokens, D, rotary_dim, interleaved ? 1 : 0, mscale, 1.f, positions, inv_freq, num_pages, page_size, slots, nullptr};
    DOCC_REQUIRE(Hq >= 0 && Hkv >= 0, "rope_append: negative extent");
    DOCC_TRY(rope_check("rope_append", prec, tokens, Hq + 2 * Hkv, D, rotary_dim, a));
    DOCC_REQUIRE(num_pages >= 0 && page_size > 0, "rope_append: page_size must be positive and num_pages not negative");
    if (flags & DOCC_B200_FLAG_HOST_PTRS)
        return set_error(DOCC_B200_ERR_UNSUPPORTED, "rope_append: the cache lives on the device; host pointers are not taken");
    Ctx* ctx;
    DOCC_TRY(get_ctx(&ctx));
    if (tokens == 0 || D == 0 || Hq + Hkv == 0) return DOCC_B200_OK;
    DOCC_REQUIRE((Hq == 0 || (Q && Qout)) && (Hkv == 0 || (K && V && slots && (num_pages == 0 || (Kcache && Vcache)))),
                 "rope_append: NULL data pointer");
    a.status = ctx->status_dev;
    RopeTensor q{Q, Qout, Hq * D, D, Hq * D, D, 0, int(Hq)};
    RopeTensor k{K, Kcache, Hkv * D, D, Hkv * page_size * D, page_size * D, D, int(Hkv)};
    RopeTensor v{V, Vcache, Hkv * D, D, Hkv * page_size * D, page_size * D, D, int(Hkv)};
    if (q_strides) { q.in_t = q_strides[0]; q.in_h = q_strides[1]; }
    if (k_strides) { k.in_t = k_strides[0]; k.in_h = k_strides[1]; }
    if (v_strides) { v.in_t = v_strides[0]; v.in_h = v_strides[1]; }
    if (qo_strides) { q.out_t = qo_strides[0]; q.out_h = qo_strides[1]; }
    if (kc_strides) { k.out_t = kc_strides[0]; k.out_h = kc_strides[1]; k.out_s = kc_strides[2]; }
    if (vc_strides) { v.out_t = vc_strides[0]; v.out_h = vc_strides[1]; v.out_s = vc_strides[2]; }
    return rope_device(ctx, prec, q, k, v, a);
}
