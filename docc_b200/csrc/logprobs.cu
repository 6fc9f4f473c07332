// Log-probabilities of given tokens, with the row's entropy and its k largest logits.
//
//   z = scale x,  lse = r + log s0,  logp = z_id - lse,  H = log s0 - s1 / s0,
//   s0 = sum e^(z - r),  s1 = sum (z - r) e^(z - r)         for any reference r
//
// Bound by reading the logits once. Sums are kept per thread in units of log 2 against a reference r that need not be the maximum:
// it is raised when a value lies 16 above it, so that in practice nothing is rescaled after a thread's first values.
//
// The alternatives cost no second pass. A thread keeps its largest logit and where it stood; the k-th largest of the threads' maxima
// is a lower bound T of the row's k-th largest, and only threads whose maximum reaches T can hold others: about k of 256. Their
// logits, k / 256 of the row, are read again (from L2), and what reaches T, few more than k values, is sorted.
//
// With fewer rows than fill the machine, a cluster of up to eight blocks takes a row; their sums and sorted lists meet in the first
// block's registers through distributed shared memory, in the order of the ranks.
#include "common.cuh"
#include "device_math.cuh"
#include "ptx.cuh"

namespace docc_b200 {
namespace {

constexpr int kMaxTop = 32;
constexpr int kBlock = 256, kLpWarps = kBlock / 32;
constexpr int kCandidates = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Order of the alternatives: larger logit first, then the lower index; a NaN is above everything. -0 and +0 are equal. No key is 0.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
    const float y = x + 0.f;  // -0 -> +0
    uint32_t u = __float_as_uint(y);
    u = y != y ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return (uint64_t(u) << 32) | uint32_t(~index);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t u = uint32_t(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~uint32_t(key); }

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

__device__ __forceinline__ float lp_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float lp_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float block_max_f(float v, float* smem) {
    v = warp_max_f(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = smem[0];
    for (int w = 1; w < kLpWarps; w++) r = fmaxf(r, smem[w]);
    return r;
}

// Rows that the one pass cannot take: a NaN or +inf among the logits, nothing but -inf, or a maximum whose product with log2 e leaves
// fp32's range (a row of the type's lowest value). The row is read once for the maximum, once for the sums and once per alternative.
template <typename T> __device__ __noinline__ void row_carefully(const T* x, const LogpArgs& a, int64_t row, float* red, unsigned long long* best) {
    float m = -INFINITY;
    for (int64_t c = threadIdx.x; c < a.vocab; c += kBlock) m = fmaxf(m, to_float(x[c]));
    m = block_max_f(m, red);
    float s0 = 0.f, s1 = 0.f;
    for (int64_t c = threadIdx.x; c < a.vocab; c += kBlock) {
        const float d = (to_float(x[c]) - m) * a.scale, e = expf(d);
        s0 += e;
        s1 += e == 0.f ? 0.f : d * e;
    }
    s0 = block_sum_f(s0, red);
    s1 = block_sum_f(s1, red);
    auto logp = [&](float v) { return (v - m) * a.scale - logf(s0); };
    if (threadIdx.x == 0) {
        if (a.logp) {
            const int64_t id = a.ids[row];
            a.logp[row] = id < 0 || id >= a.vocab ? NAN : logp(to_float(x[id]));
        }
        if (a.entropy) a.entropy[row] = logf(s0) - s1 / s0;
    }
    unsigned long long last = ~0ull;
    for (int i = 0; i < a.k; i++) {
        if (threadIdx.x == 0) *best = 0;
        __syncthreads();
        unsigned long long mine = 0;
        for (int64_t c = threadIdx.x; c < a.vocab; c += kBlock) {
            const unsigned long long key = rank_key(to_float(x[c]), uint32_t(c));
            if ((key < last || i == 0) && key > mine) mine = key;
        }
        atomicMax(best, mine);
        __syncthreads();
        last = *best;
        if (threadIdx.x == 0) {
            a.top_ids[row * a.k + i] = key_index(last);
            a.top_logp[row * a.k + i] = logp(to_float(x[key_index(last)]));
        }
        __syncthreads();
    }
}

// ---- sorting keys, one per lane, in descending order --------------------------------------------------------------------------
__device__ __forceinline__ uint64_t exchange(uint64_t v, int stride, bool larger) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, v, stride);
    return (v > o) == larger ? v : o;
}
__device__ __forceinline__ uint64_t sort32(uint64_t v, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) v = exchange(v, stride, ((lane & stride) == 0) == ((lane & size) == 0));
    return v;
}
// the 32 largest of two sorted lists
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
    uint64_t v = a > r ? a : r;
#pragma unroll
    for (int stride = 16; stride > 0; stride >>= 1) v = exchange(v, stride, (lane & stride) == 0);
    return v;
}
// Every warp holds a sorted list; list[0] receives the 32 largest of all of them. Ends with a barrier.
__device__ __forceinline__ uint64_t tournament(uint64_t mine, uint64_t (*list)[32], int lane, int warp) {
    list[warp][lane] = mine;
    __syncthreads();
#pragma unroll
    for (int half = kLpWarps / 2; half > 0; half >>= 1) {
        if (warp < half) {
            mine = merge32(mine, list[warp + half][lane], lane);
            list[warp][lane] = mine;
        }
        __syncthreads();
    }
    return list[0][lane];
}

// ---- the one pass ----------------------------------------------------------------------------------------------------------------
struct Sums {
    float ref, s0, s1;  // reference and sums in units of log 2
};
// Sums against the larger of two references; without values (s0 = 0) a reference counts as -inf.
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float ra = a.s0 == 0.f ? -INFINITY : a.ref, rb = b.s0 == 0.f ? -INFINITY : b.ref;
    Sums r;
    r.ref = fmaxf(ra, rb);
    if (r.ref == -INFINITY) return Sums{0.f, 0.f, 0.f};
    const float da = fmaxf(ra - r.ref, -200.f), db = fmaxf(rb - r.ref, -200.f);  // 2^-200 is 0: nothing is left of that side
    const float fa = lp_ex2(da), fb = lp_ex2(db);
    r.s0 = a.s0 * fa + b.s0 * fb;
    r.s1 = fmaf(a.s0, da, a.s1) * fa + fmaf(b.s0, db, b.s1) * fb;
    return r;
}
__device__ __forceinline__ Sums warp_join(Sums v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        // lanes o apart swap: the lower one's sums come first on both sides, so both get the same bits
        const Sums w{__shfl_xor_sync(0xffffffffu, v.ref, o), __shfl_xor_sync(0xffffffffu, v.s0, o), __shfl_xor_sync(0xffffffffu, v.s1, o)};
        v = (threadIdx.x & o) ? join(w, v) : join(v, w);
    }
    return v;
}

constexpr float kHeadroom = 16.f;

template <bool TOP> struct Scan {
    float c;               // scale log2 e
    float ref, limit;      // limit: the logit whose multiple by c lies kHeadroom above ref
    float s0, s1;
    float best;            // largest logit so far, and the first of the values it was found among
    int best_at;
    __device__ __forceinline__ explicit Scan(float c_) : c(c_), ref(0.f), limit(-INFINITY), s0(0.f), s1(0.f), best(-INFINITY), best_at(0) {}
    template <int N> __device__ __forceinline__ void take(const float (&x)[N], int at) {
        float top = x[0];
#pragma unroll
        for (int e = 1; e < N; e++) top = fmaxf(top, x[e]);
        if (top > limit) {
            // -inf, or a product beyond fp32: such values are left at 0 until a usable one comes (if none does, the row is taken carefully)
            const float r = top * c;
            const float next = r == -INFINITY ? 0.f : r;
            if (s0 != 0.f) {
                const float d = fmaxf(ref - next, -200.f), f = lp_ex2(d);
                s1 = fmaf(s0, d, s1) * f;
                s0 *= f;
            }
            ref = next;
            limit = r == -INFINITY ? -INFINITY : top + kHeadroom / c;
        }
        if (TOP && top > best) {
            best = top;
            best_at = at;
        }
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float d = lp_max_nan(fmaf(x[e], c, -ref), -200.f);  // finite, so that nothing times 0 is NaN; a NaN stays
            const float p = lp_ex2(d);
            s0 += p;
            s1 = fmaf(d, p, s1);
        }
    }
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kBlock) logprobs_kernel(const T* __restrict__ X, LogpArgs a, int ranks) {
    constexpr int VEC = 16 / sizeof(T), UNROLL = 4;
    using P = Pack<T, VEC>;
    __shared__ Sums sums_s[kLpWarps];
    __shared__ float red_s[kLpWarps];
    __shared__ unsigned long long best_s;
    __shared__ uint64_t list_s[kLpWarps][32];
    __shared__ uint64_t found_s[TOP ? kCandidates : 1];
    __shared__ int streams_s[TOP ? kBlock : 1];
    __shared__ int n_streams, n_found;
    __shared__ Sums block_s;  // read by the cluster's first block
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int rank = int(blockIdx.x % ranks);
    const float c = a.scale * kLog2e;
    for (int64_t row = blockIdx.x / ranks; row < a.rows; row += gridDim.x / ranks) {
        const T* x = X + row * a.ldx;
        const int vocab = int(a.vocab);
        // values before the first 16-byte boundary, whole packs, values behind the last
        int head = int((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T));
        if (head > vocab) head = vocab;
        const int packs = (vocab - head) / VEC, tail0 = head + packs * VEC;
        const int p0 = int(int64_t(packs) * rank / ranks), p1 = int(int64_t(packs) * (rank + 1) / ranks);
        const P* xp = reinterpret_cast<const P*>(x + head);

        Scan<TOP> scan(c);
        if (rank == 0 && t < head) {
            const float v[1] = {to_float(x[t])};
            scan.take(v, t);
        }
        int p = p0 + t;
        for (; p + (UNROLL - 1) * kBlock < p1; p += UNROLL * kBlock) {
            P pk[UNROLL];
#pragma unroll
            for (int i = 0; i < UNROLL; i++) pk[i] = load_pack(xp + p + i * kBlock);
#pragma unroll
            for (int i = 0; i < UNROLL; i++) {
                float v[VEC];
#pragma unroll
                for (int e = 0; e < VEC; e++) v[e] = to_float(pk[i].v[e]);
                scan.take(v, head + (p + i * kBlock) * VEC);
            }
        }
        for (; p < p1; p += kBlock) {
            const P pk = load_pack(xp + p);
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e++) v[e] = to_float(pk.v[e]);
            scan.take(v, head + p * VEC);
        }
        if (rank == ranks - 1 && t < vocab - tail0) {
            const float v[1] = {to_float(x[tail0 + t])};
            scan.take(v, tail0 + t);
        }

        const Sums mine = warp_join(Sums{scan.ref, scan.s0, scan.s1});
        if (lane == 0) sums_s[warp] = mine;
        uint64_t key = 0, list = 0;
        if constexpr (TOP) {
            if (scan.best > -INFINITY) {
                int at = scan.best_at;  // the first of up to VEC values is the one of lowest index that equals the maximum
                while (at + 1 < vocab && to_float(x[at]) != scan.best) at++;
                key = rank_key(scan.best, uint32_t(at));
            }
            list = tournament(sort32(key, lane), list_s, lane, warp);
        } else {
            __syncthreads();
        }
        Sums all = sums_s[0];
#pragma unroll
        for (int w = 1; w < kLpWarps; w++) all = join(all, sums_s[w]);

        if constexpr (TOP) {
            if (a.k > 1) {
                uint64_t bar = list_s[0][a.k - 1];  // 0 where fewer than k threads have a logit above -inf: everything is looked at
                while (true) {
                    if (t == 0) n_streams = n_found = 0;
                    __syncthreads();
                    if (key >= bar || bar == 0) streams_s[atomicAdd(&n_streams, 1)] = t;
                    __syncthreads();
                    auto offer = [&](float v, int at) {
                        const uint64_t k2 = rank_key(v, uint32_t(at));
                        if (k2 < bar) return;
                        const int place = atomicAdd(&n_found, 1);
                        if (place < kCandidates) found_s[place] = k2;
                    };
                    const int streams = n_streams, per = (p1 - p0 + kBlock - 1) / kBlock;
                    for (int i = t; i < streams * per; i += kBlock) {
                        const int q = p0 + streams_s[i % streams] + (i / streams) * kBlock;
                        if (q >= p1) continue;
                        const P pk = xp[q];
#pragma unroll
                        for (int e = 0; e < VEC; e++) offer(to_float(pk.v[e]), head + q * VEC + e);
                    }
                    if (rank == 0 && t < head) offer(to_float(x[t]), t);
                    if (rank == ranks - 1 && t < vocab - tail0) offer(to_float(x[tail0 + t]), tail0 + t);
                    __syncthreads();
                    const int found = n_found < kCandidates ? n_found : kCandidates;
                    uint64_t best = 0;
                    for (int i = warp * 32; i < found; i += kBlock) {
                        const uint64_t part = sort32(i + lane < found ? found_s[i + lane] : 0, lane);
                        best = i == warp * 32 ? part : merge32(best, part, lane);
                    }
                    const bool over = n_found > kCandidates;
                    list = tournament(best, list_s, lane, warp);
                    if (!over) break;
                    bar = list_s[0][a.k - 1];  // the k-th largest of those that found room: a higher bar, and fewer above it
                }
            }
        }
        if (ranks > 1) {
            if (t == 0) block_s = all;
            ptx::cluster_sync();
            if (rank == 0) {
                uint64_t other = 0;
                for (int r = 1; r < ranks; r++) {
                    const uint32_t from = ptx::map_to_cta(ptx::smem_u32(&block_s), uint32_t(r));
                    Sums s;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(s.ref) : "r"(from) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1+4];" : "=f"(s.s0) : "r"(from) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1+8];" : "=f"(s.s1) : "r"(from) : "memory");
                    all = join(all, s);
                }
                if constexpr (TOP) {
                    if (warp < ranks) {
                        const uint32_t from = ptx::map_to_cta(ptx::smem_u32(&list_s[0][lane]), uint32_t(warp));
                        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(other) : "r"(from) : "memory");
                    }
                }
                list = other;
            }
            ptx::cluster_sync();  // the other blocks' shared memory has been read
            if (rank != 0) continue;
            if constexpr (TOP) list = tournament(list, list_s, lane, warp);
        }

        if (!(fabsf(all.s0) < INFINITY) || all.s0 == 0.f || !(fabsf(all.ref) < INFINITY)) {
            __syncthreads();
            row_carefully(x, a, row, red_s, &best_s);
            __syncthreads();
            continue;
        }
        const float log_s0 = log2f(all.s0);
        auto logp = [&](float v) {
            const float r = (fmaf(v, c, -all.ref) - log_s0) * kLn2;
            // the multiple by log2 e may leave fp32's range where scale * x does not
            return r == -INFINITY && v > -INFINITY ? v * a.scale - (all.ref + log_s0) * kLn2 : r;
        };
        if (t == 0) {
            if (a.logp) {
                const int64_t id = a.ids[row];
                a.logp[row] = id < 0 || id >= a.vocab ? NAN : logp(to_float(x[id]));
            }
            if (a.entropy) a.entropy[row] = (log_s0 - all.s1 / all.s0) * kLn2;
        }
        if constexpr (TOP) {
            if (t < a.k) {  // k <= 32: one warp
                a.top_ids[row * a.k + t] = key_index(list);
                a.top_logp[row * a.k + t] = logp(key_value(list));
            }
        }
        __syncthreads();  // the shared arrays are reused by the next row
    }
}

template <typename T, bool TOP>
int launch_logprobs(Ctx* ctx, const void* X, const LogpArgs& a) {
    int ranks = 1;
    while (ranks < 8 && a.rows * ranks < int64_t(ctx->sm_count) * 2 && a.vocab / (2 * ranks) >= 2048) ranks *= 2;
    const int64_t cap = int64_t(1) << 20;  // rows beyond it are taken in turn
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned((a.rows < cap ? a.rows : cap) * ranks));
    cfg.blockDim = dim3(kBlock);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(ranks);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    DOCC_CUDA_TRY(cudaLaunchKernelEx(&cfg, logprobs_kernel<T, TOP>, static_cast<const T*>(X), a, ranks));
    return after_launch(ctx, "logprobs_kernel");
}
template <typename T>
int logprobs_device(Ctx* ctx, const void* X, const LogpArgs& a) {
    return a.k ? launch_logprobs<T, true>(ctx, X, a) : launch_logprobs<T, false>(ctx, X, a);
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
