// Rotary positions, alone and together with the write of a step's keys and values into a paged cache.
//
// Pair i < R/2 of a head turns by a = position * inv_freq[i]: (u, v) -> m (u cos a - v sin a, v cos a + u sin a). In fp32 the
// product is off by position * 2^-24 radians, a quarter of a turn at ten million and visible from a few thousand on, so the
// angle is formed in fp64 as a number of turns, reduced to [-1/2, 1/2] there, and only then handed to sincospif.
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

__device__ __forceinline__ void rope_angle(const RopeArgs& a, int64_t token, int i, float& c, float& s) {
    const double turns = double(a.positions[token]) * (a.inv_freq[i] * 0.15915494309189533577);
    float cs, sn;
    sincospif(2.f * float(turns - rint(turns)), &sn, &cs);
    c = a.mscale * cs;
    s = a.mscale * a.sign * sn;
}

// Any strides and sizes: a block per token, an element pair (or one copied element) per thread and step.
template <typename T>
__global__ void __launch_bounds__(256) rope_kernel(RopeTensor q, RopeTensor k, RopeTensor v, RopeArgs a) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int half = int(a.rotary / 2), D = int(a.D), units = half + (D - int(a.rotary));
    const int heads = q.heads + k.heads + v.heads;
    for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const int64_t slot = a.slots ? a.slots[t] : 0;
        const bool fits = !a.slots || (slot >= 0 && slot / a.page_size < a.num_pages);
        if (!fits && slot >= 0 && threadIdx.x == 0) report_bad_index(a.status, kIndexSlot);
        const int64_t page = a.slots ? slot / a.page_size : 0, place = a.slots ? slot % a.page_size : 0;
        for (int w = threadIdx.x; w < heads * units; w += 256) {
            int h = w / units;
            const int u = w % units;
            const RopeTensor* x = &q;
            if (h >= q.heads) { h -= q.heads; x = &k; if (h >= k.heads) { h -= k.heads; x = &v; } }
            const bool cached = x != &q;
            if (cached && !fits) continue;
            const T* in = static_cast<const T*>(x->in) + t * x->in_t + h * x->in_h;
            T* out = static_cast<T*>(x->out) + (cached ? page * x->out_t + place * x->out_s : t * x->out_t) + h * x->out_h;
            if (u >= half) {
                const int d = int(a.rotary) + u - half;
                out[d] = in[d];
                continue;
            }
            const int d0 = a.interleaved ? 2 * u : u, d1 = a.interleaved ? 2 * u + 1 : u + half;
            const T e0 = in[d0], e1 = in[d1];
            if (x == &v) {
                out[d0] = e0;
                out[d1] = e1;
                continue;
            }
            float c, s;
            rope_angle(a, t, u, c, s);
            const float x0 = to_float(e0), x1 = to_float(e1);
            out[d0] = from_float<T>(x0 * c - x1 * s);
            out[d1] = from_float<T>(x1 * c + x0 * s);
        }
    }
}

int rope_device(Ctx* ctx, int prec, const RopeTensor& q, const RopeTensor& k, const RopeTensor& v, const RopeArgs& a) {
    const int64_t cap = int64_t(ctx->sm_count) * 8;
    const dim3 grid(unsigned(a.tokens < cap ? a.tokens : cap));
    if (prec == DOCC_B200_PREC_S) DOCC_CUDA_TRY(launch_pdl(rope_kernel<float>, grid, dim3(256), 0, ctx->stream, q, k, v, a));
    else if (prec == DOCC_B200_PREC_H) DOCC_CUDA_TRY(launch_pdl(rope_kernel<__half>, grid, dim3(256), 0, ctx->stream, q, k, v, a));
    else DOCC_CUDA_TRY(launch_pdl(rope_kernel<__nv_bfloat16>, grid, dim3(256), 0, ctx->stream, q, k, v, a));
    return after_launch(ctx, "rope_kernel");
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
