// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale q.k_j (capped: c tanh(s_j / c)),  p = softmax(s),  o = sum p_j v_j,  lse = log sum exp(s_j)
//
// docc has no such node; beside the attention entry (contiguous K and V, every query at once) this is its form for serving.
#include "common.cuh"
#include "device_math.cuh"
#include "ptx.cuh"

namespace docc_b200 {
namespace {

struct PagedArgs {
    int B, Hq, Hkv, D, group;  // group = Hq / Hkv
    float scale, softcap;
    int64_t window;
    int64_t qs[2], os[2], ks[3], vs[3];  // element strides: (sequence, head), (page, head, place)
    int64_t num_pages, page_size, max_pages, table_stride;
    const int32_t* page_table;
    const int32_t* lengths;
    float* lse;
    DeviceStatus* status;
};

// Visible tokens [lo, n) of sequence b.
__device__ __forceinline__ void visible(const PagedArgs& a, int b, int64_t& lo, int64_t& n) {
    n = a.lengths[b];
    const int64_t most = a.max_pages * a.page_size;
    if (n < 0 || n > most) {
        report_bad_index(a.status, kIndexLength);
        n = n < 0 ? 0 : most;
    }
    lo = a.window > 0 && n > a.window ? n - a.window : 0;
}

// Any type, strides and size: a warp per (sequence, query head), the keys in order with the running maximum and sum.
template <typename T, int DPL>
__global__ void __launch_bounds__(128) paged_rows_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                         T* __restrict__ O, PagedArgs a) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t(blockIdx.x) * 128 + threadIdx.x) >> 5;
    if (row >= int64_t(a.B) * a.Hq) return;
    const int b = int(row / a.Hq), h = int(row % a.Hq), kvh = h / a.group;
    int64_t lo, n;
    visible(a, b, lo, n);
    const T* q = Q + b * a.qs[0] + h * a.qs[1];
    float qr[DPL], acc[DPL];
#pragma unroll
    for (int e = 0; e < DPL; e++) {
        const int d = lane + 32 * e;
        qr[e] = d < a.D ? to_float(q[d]) : 0.f;
        acc[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int64_t j = lo; j < n; j++) {
        const int64_t page = a.page_table[b * a.table_stride + j / a.page_size], place = j % a.page_size;
        if (page < 0 || page >= a.num_pages) {
            report_bad_index(a.status, kIndexPage);
            continue;
        }
        const T* kr = K + page * a.ks[0] + kvh * a.ks[1] + place * a.ks[2];
        const T* vr = V + page * a.vs[0] + kvh * a.vs[1] + place * a.vs[2];
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < DPL; e++) {
            const int d = lane + 32 * e;
            if (d < a.D) s = fmaf(qr[e], to_float(kr[d]), s);
        }
        s = warp_sum_f(s) * a.scale;
        if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
        const float m_new = fmaxf(m, s);
        const float ref = m_new == -INFINITY ? 0.f : m_new;  // scores of -inf only: exp(-inf - 0) = 0, not a NaN
        const float corr = expf(m - ref), p = expf(s - ref);
        l = l * corr + p;
#pragma unroll
        for (int e = 0; e < DPL; e++) {
            const int d = lane + 32 * e;
            if (d < a.D) acc[e] = fmaf(p, to_float(vr[d]), acc[e] * corr);
        }
        m = m_new;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* o = O + b * a.os[0] + h * a.os[1];
#pragma unroll
    for (int e = 0; e < DPL; e++) {
        const int d = lane + 32 * e;
        if (d < a.D) o[d] = from_float<T>(acc[e] * inv);
    }
    if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : m + logf(l);
}

template <typename T>
int paged_device(Ctx* ctx, const PagedArgs& a, const void* Q, const void* K, const void* V, void* O) {
    const dim3 grid(unsigned(ceil_div(int64_t(a.B) * a.Hq, 4)));
    auto kernel = a.D <= 64 ? paged_rows_kernel<T, 2> : a.D <= 128 ? paged_rows_kernel<T, 4> : paged_rows_kernel<T, 8>;
    DOCC_CUDA_TRY(launch_pdl(kernel, grid, dim3(128), 0, ctx->stream, static_cast<const T*>(Q), static_cast<const T*>(K),
                             static_cast<const T*>(V), static_cast<T*>(O), a));
    return after_launch(ctx, "paged_rows_kernel");
}

}  // namespace
}  // namespace docc_b200

using namespace docc_b200;

extern "C" int docc_b200_paged_attention_workspace(int prec, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, size_t* bytes) {
    DOCC_REQUIRE(bytes != nullptr, "paged_attention_workspace: bytes is NULL");
    DOCC_REQUIRE(prec_size(prec) != 0 && prec != DOCC_B200_PREC_D, "paged_attention_workspace: precision %d not supported (use 's', 'b' or 'h')", prec);
    DOCC_REQUIRE(B >= 0 && Hq >= 0 && Hkv >= 0 && D >= 0, "paged_attention_workspace: negative extent");
    *bytes = 0;
    return DOCC_B200_OK;
}

extern "C" int docc_b200_paged_attention(int prec, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, float scale, float softcap,
                                         int64_t window, const void* Q, const int64_t* q_strides, const void* Kcache,
                                         const int64_t* kc_strides, const void* Vcache, const int64_t* vc_strides, int64_t num_pages,
                                         int64_t page_size, const int32_t* page_table, int64_t max_pages, int64_t table_stride,
                                         const int32_t* lengths, void* O, const int64_t* o_strides, void* lse, void* workspace,
                                         size_t workspace_bytes, int flags) {
    DOCC_REQUIRE(prec == DOCC_B200_PREC_S || prec == DOCC_B200_PREC_B || prec == DOCC_B200_PREC_H,
                 "paged_attention: precision %d not supported (use 's', 'b' or 'h')", prec);
    DOCC_REQUIRE(B >= 0 && Hq >= 0 && Hkv >= 0 && D >= 0 && num_pages >= 0 && max_pages >= 0, "paged_attention: negative extent");
    DOCC_REQUIRE(page_size > 0, "paged_attention: page_size must be positive");
    DOCC_REQUIRE(softcap >= 0.f && window >= 0, "paged_attention: softcap and window must not be negative");
    if (flags & DOCC_B200_FLAG_HOST_PTRS)
        return set_error(DOCC_B200_ERR_UNSUPPORTED, "paged_attention: the cache lives on the device; host pointers are not taken");
    Ctx* ctx;
    DOCC_TRY(get_ctx(&ctx));
    if (B == 0 || Hq == 0 || D == 0) return DOCC_B200_OK;
    DOCC_REQUIRE(Hkv > 0 && Hq % Hkv == 0, "paged_attention: %lld query heads are not a multiple of %lld key-value heads", (long long)Hq,
                 (long long)Hkv);
    if (D > 256) return set_error(DOCC_B200_ERR_UNSUPPORTED, "paged_attention: head_dim %lld > 256", (long long)D);
    DOCC_REQUIRE(B <= 65535 && Hq <= 65535, "paged_attention: more than 65535 sequences or heads");
    DOCC_REQUIRE(Q && O && lengths && (max_pages == 0 || (page_table && (num_pages == 0 || (Kcache && Vcache)))),
                 "paged_attention: NULL data pointer");
    DOCC_REQUIRE(table_stride >= max_pages, "paged_attention: table_stride below max_pages");
    (void)workspace; (void)workspace_bytes;
    PagedArgs a;
    a.B = int(B); a.Hq = int(Hq); a.Hkv = int(Hkv); a.D = int(D); a.group = int(Hq / Hkv);
    a.scale = scale; a.softcap = softcap; a.window = window;
    a.qs[0] = q_strides ? q_strides[0] : Hq * D; a.qs[1] = q_strides ? q_strides[1] : D;
    a.os[0] = o_strides ? o_strides[0] : Hq * D; a.os[1] = o_strides ? o_strides[1] : D;
    const int64_t dense[3] = {Hkv * page_size * D, page_size * D, D};
    for (int i = 0; i < 3; i++) {
        a.ks[i] = kc_strides ? kc_strides[i] : dense[i];
        a.vs[i] = vc_strides ? vc_strides[i] : dense[i];
    }
    a.num_pages = num_pages; a.page_size = page_size; a.max_pages = max_pages; a.table_stride = table_stride;
    a.page_table = page_table; a.lengths = lengths; a.lse = static_cast<float*>(lse); a.status = ctx->status_dev;
    if (prec == DOCC_B200_PREC_S) return paged_device<float>(ctx, a, Q, Kcache, Vcache, O);
    if (prec == DOCC_B200_PREC_H) return paged_device<__half>(ctx, a, Q, Kcache, Vcache, O);
    return paged_device<__nv_bfloat16>(ctx, a, Q, Kcache, Vcache, O);
}
