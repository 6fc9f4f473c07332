// Log-probabilities of given tokens, with the row's entropy and its k largest logits.
//
//   z = scale x,  lse = m + log s0,  logp = z_id - lse,  H = log s0 - s1 / s0,
//   s0 = sum e^(z - m),  s1 = sum (z - m) e^(z - m)
#include "common.cuh"
#include "device_math.cuh"
#include "ptx.cuh"

namespace docc_b200 {
namespace {

constexpr int kMaxTop = 32;

// Order of the alternatives: larger logit first, then the lower index; a NaN is above everything. -0 and +0 are equal.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
    const float y = x + 0.f;  // -0 -> +0
    uint32_t u = __float_as_uint(y);
    u = y != y ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return (uint64_t(u) << 32) | uint32_t(~index);
}

struct LogpArgs {
    int64_t rows, vocab, ldx;
    float scale;
    const int64_t* ids;
    float* logp;
    float* entropy;
    int k;
    int64_t* top_ids;
    float* top_logp;
};

__device__ __forceinline__ float block_max_f(float v, float* smem) {
    v = warp_max_f(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = smem[0];
    for (int w = 1; w < int(blockDim.x >> 5); w++) r = fmaxf(r, smem[w]);
    return r;
}

// Block per row, the row read once for the sums and once more for every alternative.
template <typename T>
__global__ void __launch_bounds__(256) logprobs_kernel(const T* __restrict__ X, LogpArgs a) {
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    __shared__ float red[8];
    __shared__ unsigned long long best;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = X + row * a.ldx;
        float m = -INFINITY;
        for (int64_t c = threadIdx.x; c < a.vocab; c += 256) m = fmaxf(m, to_float(x[c]) * a.scale);
        m = block_max_f(m, red);
        float s0 = 0.f, s1 = 0.f;
        for (int64_t c = threadIdx.x; c < a.vocab; c += 256) {
            const float d = to_float(x[c]) * a.scale - m, e = expf(d);
            s0 += e;
            s1 += e == 0.f ? 0.f : d * e;
        }
        s0 = block_sum_f(s0, red);
        s1 = block_sum_f(s1, red);
        const float lse = m + logf(s0);
        if (threadIdx.x == 0) {
            if (a.logp) {
                const int64_t id = a.ids[row];
                a.logp[row] = id < 0 || id >= a.vocab ? NAN : to_float(x[id]) * a.scale - lse;
            }
            if (a.entropy) a.entropy[row] = logf(s0) - s1 / s0;
        }
        unsigned long long last = ~0ull;
        for (int i = 0; i < a.k; i++) {
            if (threadIdx.x == 0) best = 0;
            __syncthreads();
            unsigned long long mine = 0;
            for (int64_t c = threadIdx.x; c < a.vocab; c += 256) {
                const unsigned long long key = rank_key(to_float(x[c]), uint32_t(c));
                if ((key < last || i == 0) && key > mine) mine = key;
            }
            atomicMax(&best, mine);
            __syncthreads();
            last = best;
            if (threadIdx.x == 0) {
                const int64_t c = int64_t(uint32_t(~uint32_t(last)));
                a.top_ids[row * a.k + i] = c;
                a.top_logp[row * a.k + i] = to_float(x[c]) * a.scale - lse;
            }
            __syncthreads();
        }
    }
}

template <typename T>
int logprobs_device(Ctx* ctx, const void* X, const LogpArgs& a) {
    const int64_t cap = int64_t(ctx->sm_count) * 8;
    const dim3 grid(unsigned(a.rows < cap ? a.rows : cap));
    DOCC_CUDA_TRY(launch_pdl(logprobs_kernel<T>, grid, dim3(256), 0, ctx->stream, static_cast<const T*>(X), a));
    return after_launch(ctx, "logprobs_kernel");
}

int logprobs_any(Ctx* ctx, int prec, const void* X, const LogpArgs& a) {
    if (prec == DOCC_B200_PREC_S) return logprobs_device<float>(ctx, X, a);
    if (prec == DOCC_B200_PREC_H) return logprobs_device<__half>(ctx, X, a);
    return logprobs_device<__nv_bfloat16>(ctx, X, a);
}

}  // namespace
}  // namespace docc_b200

using namespace docc_b200;

extern "C" int docc_b200_token_logprobs(int prec, int64_t rows, int64_t vocab, const void* X, int64_t ldx, float scale,
                                        const int64_t* ids, void* logp, void* entropy, int64_t k, int64_t* top_ids, void* top_logp,
                                        int flags) {
    DOCC_REQUIRE(prec == DOCC_B200_PREC_S || prec == DOCC_B200_PREC_B || prec == DOCC_B200_PREC_H,
                 "token_logprobs: precision %d not supported (use 's', 'b' or 'h')", prec);
    DOCC_REQUIRE(rows >= 0 && vocab >= 0, "token_logprobs: negative extent");
    DOCC_REQUIRE(k >= 0 && k <= kMaxTop && k <= vocab, "token_logprobs: k = %lld must be in [0, %d] and at most the vocabulary",
                 (long long)k, kMaxTop);
    DOCC_REQUIRE(scale > 0.f && scale < INFINITY, "token_logprobs: scale must be positive and finite");
    Ctx* ctx;
    DOCC_TRY(get_ctx(&ctx));
    if (rows == 0) return DOCC_B200_OK;
    DOCC_REQUIRE(vocab > 0, "token_logprobs: empty vocabulary");
    DOCC_REQUIRE(vocab < (int64_t(1) << 31), "token_logprobs: vocabulary of 2^31 or more");
    DOCC_REQUIRE(ldx >= vocab, "token_logprobs: row stride below the vocabulary");
    DOCC_REQUIRE(X && (!logp || ids) && (k == 0 || (top_ids && top_logp)), "token_logprobs: NULL data pointer");
    LogpArgs a{rows, vocab, ldx, scale, ids, static_cast<float*>(logp), static_cast<float*>(entropy), int(k), top_ids,
               static_cast<float*>(top_logp)};
    if (!(flags & DOCC_B200_FLAG_HOST_PTRS)) return logprobs_any(ctx, prec, X, a);

    DOCC_REQUIRE(ldx == vocab, "token_logprobs: host pointers require contiguous rows");
    const size_t xb = size_t(rows) * size_t(vocab) * prec_size(prec), rb = size_t(rows), tb = rb * size_t(k);
    TempBuffers tmp;
    void *dX, *dI = nullptr, *dL = nullptr, *dE = nullptr, *dTi = nullptr, *dTl = nullptr;
    DOCC_TRY(tmp.alloc(&dX, xb));
    DOCC_CUDA_TRY(cudaMemcpyAsync(dX, X, xb, cudaMemcpyHostToDevice, ctx->stream));
    if (logp) {
        DOCC_TRY(tmp.alloc(&dI, rb * 8));
        DOCC_TRY(tmp.alloc(&dL, rb * 4));
        DOCC_CUDA_TRY(cudaMemcpyAsync(dI, ids, rb * 8, cudaMemcpyHostToDevice, ctx->stream));
    }
    if (entropy) DOCC_TRY(tmp.alloc(&dE, rb * 4));
    if (k) {
        DOCC_TRY(tmp.alloc(&dTi, tb * 8));
        DOCC_TRY(tmp.alloc(&dTl, tb * 4));
    }
    a.ids = static_cast<const int64_t*>(dI);
    a.logp = static_cast<float*>(dL);
    a.entropy = static_cast<float*>(dE);
    a.top_ids = static_cast<int64_t*>(dTi);
    a.top_logp = static_cast<float*>(dTl);
    DOCC_TRY(logprobs_any(ctx, prec, dX, a));
    if (logp) DOCC_CUDA_TRY(cudaMemcpyAsync(logp, dL, rb * 4, cudaMemcpyDeviceToHost, ctx->stream));
    if (entropy) DOCC_CUDA_TRY(cudaMemcpyAsync(entropy, dE, rb * 4, cudaMemcpyDeviceToHost, ctx->stream));
    if (k) {
        DOCC_CUDA_TRY(cudaMemcpyAsync(top_ids, dTi, tb * 8, cudaMemcpyDeviceToHost, ctx->stream));
        DOCC_CUDA_TRY(cudaMemcpyAsync(top_logp, dTl, tb * 4, cudaMemcpyDeviceToHost, ctx->stream));
    }
    DOCC_CUDA_TRY(cudaStreamSynchronize(ctx->stream));
    return DOCC_B200_OK;
}
