// Log-probabilities of given tokens, with the row's entropy and its k largest logits.
//
//   z = scale x,  lse = r + log s0,  logp = z_id - lse,  H = log s0 - s1 / s0,
//   s0 = sum e^(z - r),  s1 = sum (z - r) e^(z - r)         for any reference r
//
// Bound by reading the logits once. Sums are kept per thread in units of log 2 against a reference r that need not be the maximum:
// it is raised when a value lies 16 above it, so that in practice nothing is rescaled after a thread's first values.
//
// The alternatives need no second pass over the row, but what they need begins when it has ended and takes as long again. A thread keeps
// its largest logit; T, a value that at least k threads' maxima reach, is a lower bound of the row's k-th largest, and only those threads
// can hold others: some thirty of 512 for k = 20. Their logits are read again (from L2), and what reaches T, few more than k values, is
// ranked by counting.
//
// 4096 rows of 50021 fp32 without alternatives: 820 MB, 138 us (5.9 TB/s, 0.91 of the measured copy); 256 rows of 128000 bf16 with
// twenty: 22.5 us, about 11 for the stream and the rest for what follows it, which nothing overlaps while all rows run at once; 4 rows
// of 32768: 5.9 us.
//
// With fewer rows than fill the machine, a cluster of up to eight blocks takes a row; the other blocks' sums and lists meet in the first
// block through distributed shared memory, in the order of the ranks.
#include "common.cuh"
#include "device_math.cuh"
#include "ptx.cuh"

namespace docc_b200 {
namespace {

constexpr int kMaxTop = 32;
constexpr int kCandidates = 1024, kRescan = 4;
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
    for (int w = 1; w < int(blockDim.x >> 5); w++) r = fmaxf(r, smem[w]);
    return r;
}

// Rows that the one pass cannot take: a NaN or +inf among the logits, nothing but -inf, or a maximum whose product with log2 e leaves
// fp32's range (a row of the type's lowest value). The row is read once for the maximum, once for the sums and once per alternative.
template <typename T> __device__ __noinline__ void row_carefully(const T* x, const LogpArgs& a, int64_t row, float* red, unsigned long long* best) {
    float m = -INFINITY;
    for (int64_t c = threadIdx.x; c < a.vocab; c += blockDim.x) m = fmaxf(m, to_float(x[c]));
    m = block_max_f(m, red);
    float s0 = 0.f, s1 = 0.f;
    for (int64_t c = threadIdx.x; c < a.vocab; c += blockDim.x) {
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
        for (int64_t c = threadIdx.x; c < a.vocab; c += blockDim.x) {
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

// ---- the one pass ----------------------------------------------------------------------------------------------------------------
struct Sums {
    float ref, s0, s1;  // reference and sums in units of log 2
};
// The sums of N lanes (a power of two, the same ones for every lane of a group) against the largest of their references. A side without
// values (s0 = 0) counts as -inf. The order of the additions is that of the lanes.
template <int N> __device__ __forceinline__ Sums join_lanes(const Sums& v) {
    const float own = v.s0 == 0.f ? -INFINITY : v.ref;
    float top = own;
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY) top = 0.f;
    const float d = fmaxf(own - top, -200.f), f = lp_ex2(d);  // 2^-200 is 0: nothing is left of that side
    Sums r{top, v.s0 * f, fmaf(v.s0, d, v.s1) * f};
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) {
        r.s0 += __shfl_xor_sync(0xffffffffu, r.s0, o);
        r.s1 += __shfl_xor_sync(0xffffffffu, r.s1, o);
    }
    return r;
}

constexpr float kHeadroom = 16.f;

// A 16-byte pack: its largest value, and its values raised to at least floor() so that no multiple of them is infinite and nothing
// times 0 becomes a NaN. 16-bit packs do both on pairs. A NaN is passed over by the first and kept by the second.
template <typename T> struct Packed;
template <> struct Packed<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ float floor() { return -1e30f; }
    static __device__ __forceinline__ float top(const uint4& w) {
        return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    }
    static __device__ __forceinline__ void values(const uint4& w, float (&x)[4]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = lp_max_nan(__uint_as_float(u[i]), floor());
    }
};
template <> struct Packed<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float floor() { return __uint_as_float(0xf1490000u); }  // -1e30
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float top(const uint4& w) {
        const uint32_t m = max2(max2(w.x, w.y), max2(w.z, w.w));
        return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
    static __device__ __forceinline__ void values(const uint4& w, float (&x)[8]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t r;
            asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u[i]), "r"(0xf149f149u));
            x[2 * i] = __uint_as_float(r << 16);
            x[2 * i + 1] = __uint_as_float(r & 0xffff0000u);
        }
    }
};
template <> struct Packed<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float floor() { return -65504.f; }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float top(const uint4& w) {
        const uint32_t m = max2(max2(w.x, w.y), max2(w.z, w.w));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ void values(const uint4& w, float (&x)[8]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t r;
            asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u[i]), "r"(0xfbfffbffu));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
};

// Where in a pack of N values the first one equal to v stands (N - 1 if none is).
template <typename T> __device__ __forceinline__ int first_of(const uint4& w, float v) {
    constexpr int N = 16 / sizeof(T);
    const T* x = reinterpret_cast<const T*>(&w);
    int at = N - 1;
#pragma unroll
    for (int e = N - 2; e >= 0; e--)
        if (to_float(x[e]) == v) at = e;
    return at;
}

struct Scan {
    float c;           // scale log2 e
    float ref, limit;  // limit: the logit whose multiple by c lies kHeadroom above ref
    float best;        // largest logit so far
    float2 s0, s1;     // sums of the even and the odd values
    __device__ __forceinline__ explicit Scan(float c_)
        : c(c_), ref(0.f), limit(-INFINITY), best(-INFINITY), s0(make_float2(0.f, 0.f)), s1(make_float2(0.f, 0.f)) {}
    __device__ __forceinline__ void rise(float top) {
        if (top > limit) {
            // -inf, or a product beyond fp32: such values count nothing until a usable one comes (if none does, the row is taken carefully)
            const float r = top * c;
            const float next = r == -INFINITY ? 0.f : r;
            const float d = fmaxf(ref - next, -200.f), f = lp_ex2(d);
            if (s0.x + s0.y != 0.f) {
                s1 = make_float2(fmaf(s0.x, d, s1.x) * f, fmaf(s0.y, d, s1.y) * f);
                s0 = make_float2(s0.x * f, s0.y * f);
            }
            ref = next;
            limit = r == -INFINITY ? -INFINITY : top + kHeadroom / c;
        }
        best = fmaxf(best, top);
    }
    __device__ __forceinline__ void one(float v, float floor) {
        rise(v);
        const float d = fmaf(lp_max_nan(v, floor), c, -ref), p = lp_ex2(d);
        s0.x += p;
        s1.x = fmaf(d, p, s1.x);
    }
    template <typename T> __device__ __forceinline__ void pack(const uint4& w) {
        rise(Packed<T>::top(w));
        float x[Packed<T>::N];
        Packed<T>::values(w, x);
#pragma unroll
        for (int e = 0; e < Packed<T>::N; e += 2) {  // packed pairs: one instruction for two products or sums
            float d0, d1;
            asm("{\n.reg .b64 a, b, k, r;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %4};\nmov.b64 k, {%5, %5};\nfma.rn.f32x2 r, a, b, k;\n"
                "mov.b64 {%0, %1}, r;\n}"
                : "=f"(d0), "=f"(d1)
                : "f"(x[e]), "f"(x[e + 1]), "f"(c), "f"(-ref));
            const float p0 = lp_ex2(d0), p1 = lp_ex2(d1);
            asm("{\n.reg .b64 a, b, r;\nmov.b64 a, {%0, %1};\nmov.b64 b, {%2, %3};\nadd.rn.f32x2 r, a, b;\nmov.b64 {%0, %1}, r;\n}"
                : "+f"(s0.x), "+f"(s0.y)
                : "f"(p0), "f"(p1));
            asm("{\n.reg .b64 a, b, k, r;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 k, {%0, %1};\nfma.rn.f32x2 r, a, b, k;\n"
                "mov.b64 {%0, %1}, r;\n}"
                : "+f"(s1.x), "+f"(s1.y)
                : "f"(d0), "f"(d1), "f"(p0), "f"(p1));
        }
    }
    __device__ __forceinline__ Sums sums() const { return Sums{ref, s0.x + s0.y, s1.x + s1.y}; }
};

__device__ __forceinline__ uint32_t ordered(float x) { return uint32_t(rank_key(x, 0) >> 32); }

// A value (as ordered bits) that at least k of the block's threads reach with theirs, near the k-th largest: a warp's j-th largest,
// j = ceil(k / active), of the r-th best warp, j r >= k. active: the warps whose every lane has values. `values_s` has room for one word
// per warp. 0 if there is none.
template <int WARPS> __device__ __forceinline__ uint32_t bound_of(uint32_t mine, int k, int active, uint32_t* values_s, int lane, int warp) {
    const int j = (k + active - 1) / active, r = (k + j - 1) / j;
    uint32_t rest = mine, nth = 0;
    for (int i = 0; i < j; i++) {
        nth = __reduce_max_sync(0xffffffffu, rest);
        if (lane == __ffs(__ballot_sync(0xffffffffu, rest == nth)) - 1) rest = 0;
    }
    if (lane == 0) values_s[warp] = nth;
    __syncthreads();
    const uint32_t v = lane < WARPS ? values_s[lane] : 0;
    int above = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
        const uint32_t o = __shfl_sync(0xffffffffu, v, w);
        above += o > v || (o == v && w < lane);
    }
    const unsigned hit = __ballot_sync(0xffffffffu, lane < WARPS && above == r - 1);
    return __shfl_sync(0xffffffffu, v, __ffs(hit) - 1);
}
// The k largest of n distinct keys, in order: a key's place is the number of keys above it, counted by a thread per key (a ballot of
// 32 comparisons per step has fewer instructions and takes twice as long: each step waits for the one before). Places past the last
// key hold 0.
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int n, int k, uint64_t* out) {
    if (int(threadIdx.x) < k && int(threadIdx.x) >= n) out[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const uint64_t mine = keys[i];
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) above += keys[j] > mine;
        if (above < k && mine != 0) out[above] = mine;
    }
}

template <typename T, bool TOP, int BLOCK>
__global__ void __launch_bounds__(BLOCK, 1024 / BLOCK) logprobs_kernel(const T* __restrict__ X, LogpArgs a, int log_ranks) {
    constexpr int VEC = 16 / sizeof(T), UNROLL = 4, WARPS = BLOCK / 32;
    __shared__ Sums sums_s[WARPS];
    __shared__ float red_s[WARPS];
    __shared__ uint32_t values_s[WARPS];
    __shared__ unsigned long long best_s;
    __shared__ uint64_t list_s[kMaxTop];
    __shared__ uint64_t found_s[TOP ? kCandidates : 1];
    __shared__ int streams_s[TOP ? BLOCK : 1];
    __shared__ int hits_s[TOP ? kCandidates : 1];
    __shared__ int n_streams, n_found, n_hits;
    __shared__ Sums block_s;  // read, like list_s, by the cluster's first block
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int ranks = 1 << log_ranks, rank = int(blockIdx.x) & (ranks - 1);
    const float c = a.scale * kLog2e;
    for (int64_t row = blockIdx.x >> log_ranks; row < a.rows; row += gridDim.x >> log_ranks) {
        const T* x = X + row * a.ldx;
        const int vocab = int(a.vocab);
        // values before the first 16-byte boundary, whole packs, values behind the last
        int head = int((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T));
        if (head > vocab) head = vocab;
        const int packs = (vocab - head) / VEC, tail0 = head + packs * VEC;
        const int share = (packs + ranks - 1) >> log_ranks, p0 = min(rank * share, packs), p1 = min(p0 + share, packs);
        const uint4* xp = reinterpret_cast<const uint4*>(x + head);

        // asked for now, used at the end
        const int64_t id = rank == 0 && t == 0 && a.logp ? a.ids[row] : -1;
        const float chosen = id >= 0 && id < a.vocab ? to_float(x[id]) : NAN;

        Scan scan(c);
        if (rank == 0 && t < head) scan.one(to_float(x[t]), Packed<T>::floor());
        int p = p0 + t;
        for (; p + (UNROLL - 1) * BLOCK < p1; p += UNROLL * BLOCK) {
            uint4 w[UNROLL];
#pragma unroll
            for (int i = 0; i < UNROLL; i++) w[i] = __ldcs(xp + p + i * BLOCK);
#pragma unroll
            for (int i = 0; i < UNROLL; i++) scan.template pack<T>(w[i]);
        }
        for (; p < p1; p += BLOCK) scan.template pack<T>(__ldcs(xp + p));
        if (rank == ranks - 1 && t < vocab - tail0) scan.one(to_float(x[tail0 + t]), Packed<T>::floor());

        const Sums mine = join_lanes<32>(scan.sums());
        if (lane == 0) sums_s[warp] = mine;
        uint32_t key = 0;
        uint64_t bar = 0;
        if constexpr (TOP) {
            if (t == 0) n_streams = n_found = n_hits = 0;
            if (scan.best > -INFINITY) key = ordered(scan.best);
            bar = uint64_t(bound_of<WARPS>(key, a.k, max(1, min(WARPS, (p1 - p0) / 32)), values_s, lane, warp)) << 32;  // 0: too few threads have a logit above -inf, all is looked at
        } else {
            __syncthreads();
        }
        Sums all = join_lanes<WARPS>(sums_s[lane % WARPS]);

        if constexpr (TOP) {
            key = max(key, ordered(-INFINITY));  // the bar may be a -inf: the threads that have nothing else hold those, too
            bool lift = bar == 0;
            while (true) {
                if (lift) {
                    // any k keys bound the k-th largest: the first k of the block's, which are the ones wanted where all but a few values
                    // are equal (a mask, a constant). 256 rows of 128000 bf16, three tokens unmasked: 37 us, 308 by the rounds alone
                    const int first = rank == 0 ? 0 : head + p0 * VEC, end = rank == ranks - 1 ? vocab : head + p1 * VEC;
                    if (end - first >= a.k) {
                        uint64_t least = lane < a.k ? rank_key(to_float(x[first + lane]), uint32_t(first + lane)) : ~uint64_t(0);
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) least = min(least, uint64_t(__shfl_xor_sync(0xffffffffu, (unsigned long long)least, o)));
                        bar = max(bar, least);
                    }
                }
                if (key >= uint32_t(bar >> 32)) streams_s[atomicAdd(&n_streams, 1)] = t;
                __syncthreads();
                // a warp per stream, a pack per lane; packs that hold something are queued
                const int streams = n_streams, per = (p1 - p0 + BLOCK - 1) / BLOCK;
                for (int j = lane; j < (per + 31) / 32 * 32; j += 32) {
                    for (int s0 = warp; s0 < streams; s0 += WARPS * kRescan) {
                        uint4 w[kRescan];
                        int q[kRescan];
#pragma unroll
                        for (int h = 0; h < kRescan; h++) {  // all of a round are asked for together
                            const int s = s0 + h * WARPS;
                            q[h] = s < streams ? p0 + streams_s[s] + j * BLOCK : p1;
                            if (q[h] < p1) w[h] = xp[q[h]];
                        }
#pragma unroll
                        for (int h = 0; h < kRescan; h++) {
                            if (q[h] >= p1) continue;
                            const float top = Packed<T>::top(w[h]);
                            const uint32_t value = ordered(top);
                            if (value < uint32_t(bar >> 32)) continue;
                            // of equal values only those up to the bar's index: what is queued holds a key that reaches the bar
                            if (value == uint32_t(bar >> 32) && rank_key(top, uint32_t(head + q[h] * VEC + first_of<T>(w[h], top))) < bar) continue;
                            const int place = atomicAdd(&n_hits, 1);
                            if (place < kCandidates) hits_s[place] = q[h];
                        }
                    }
                }
                __syncthreads();
                // of more packs than the queue holds, enough for a new bar
                const int hits = n_hits <= kCandidates ? n_hits : kCandidates / VEC, edges = (rank == 0 ? head : 0) + (rank == ranks - 1 ? vocab - tail0 : 0);
                for (int i = t; i < hits * VEC + edges; i += BLOCK) {
                    int at;
                    if (i < hits * VEC) at = head + hits_s[i / VEC] * VEC + i % VEC;
                    else at = i - hits * VEC < (rank == 0 ? head : 0) ? i - hits * VEC : tail0 + (i - hits * VEC - (rank == 0 ? head : 0));
                    const uint64_t k2 = rank_key(to_float(x[at]), uint32_t(at));
                    if (k2 >= bar) {
                        const int place = atomicAdd(&n_found, 1);
                        if (place < kCandidates) found_s[place] = k2;
                    }
                }
                __syncthreads();
                const int n = n_found, queued = n_hits;
                const bool room = n <= kCandidates && queued <= kCandidates;
                rank_keys(found_s, room ? n : min(n, kCandidates / 4), a.k, list_s);
                __syncthreads();
                if (room) break;
                // more than found room: those that were ranked are kCandidates / VEC distinct keys or more that reach the bar, and all but k
                // of them lie below their k-th largest, the next bar, so every round leaves some hundred fewer above it at least
                bar = list_s[a.k - 1];
                lift = true;
                if (t == 0) n_streams = n_found = n_hits = 0;
                __syncthreads();
            }
        }
        if (ranks > 1) {
            if (t == 0) block_s = all;
            ptx::cluster_sync();
            if (rank == 0) {
                Sums s{0.f, 0.f, 0.f};
                if (lane < ranks) {
                    const uint32_t from = ptx::map_to_cta(ptx::smem_u32(&block_s), uint32_t(lane));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(s.ref) : "r"(from) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1+4];" : "=f"(s.s0) : "r"(from) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1+8];" : "=f"(s.s1) : "r"(from) : "memory");
                }
                all = join_lanes<32>(s);
                if constexpr (TOP) {  // 32 lanes per rank: 8 ranks of up to 32 keys
                    if (warp < ranks && lane < a.k) {
                        const uint32_t from = ptx::map_to_cta(ptx::smem_u32(&list_s[lane]), uint32_t(warp));
                        uint64_t k2;
                        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(k2) : "r"(from) : "memory");
                        found_s[warp * a.k + lane] = k2;
                    }
                }
            }
            ptx::cluster_sync();  // the other blocks' shared memory has been read
            if (rank != 0) continue;
            if constexpr (TOP) {
                rank_keys(found_s, ranks * a.k, a.k, list_s);
                __syncthreads();
            }
        }

        // careful: no usable value, a NaN or +inf, or a maximum so near the floor that a value raised to it would count
        if (!(fabsf(all.s0) < INFINITY) || !(fabsf(all.s1) < INFINITY) || all.s0 == 0.f || !(all.ref - Packed<T>::floor() * c >= 200.f)) {
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
            if (a.logp) a.logp[row] = logp(chosen);  // of a NaN where there is no such token
            if (a.entropy) a.entropy[row] = (log_s0 - all.s1 / all.s0) * kLn2;
        }
        if constexpr (TOP) {
            if (t < a.k) {
                a.top_ids[row * a.k + t] = key_index(list_s[t]);
                a.top_logp[row * a.k + t] = logp(key_value(list_s[t]));
            }
        }
        __syncthreads();  // the shared arrays are reused by the next row
    }
}

template <typename T, bool TOP, int BLOCK>
int launch_logprobs(Ctx* ctx, const void* X, const LogpArgs& a) {
    // clusters only while every block has an SM of its own: at 256 rows two blocks per row took 29 us instead of 20, eight took 53
    int ranks = 1, log_ranks = 0;
    while (ranks < 8 && a.rows * ranks * 2 <= ctx->sm_count && a.vocab / (2 * ranks) >= 2048) {
        ranks *= 2;
        log_ranks++;
    }
    const int64_t cap = int64_t(1) << 20;  // rows beyond it are taken in turn
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned((a.rows < cap ? a.rows : cap) * ranks));
    cfg.blockDim = dim3(BLOCK);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(ranks);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    DOCC_CUDA_TRY(cudaLaunchKernelEx(&cfg, logprobs_kernel<T, TOP, BLOCK>, static_cast<const T*>(X), a, log_ranks));
    return after_launch(ctx, "logprobs_kernel");
}
template <typename T>
int logprobs_device(Ctx* ctx, const void* X, const LogpArgs& a) {
    // What follows the stream takes a block's time whatever the row's length, so short rows want small blocks, many to an SM, and long
    // ones large blocks. bf16, k = 20: 2000 rows of 32768 51 us with 128 threads, 54 with 256, 66 with 512; 600 of 128000 77, 60 and 52;
    // 64 of 20000, fewer than fill the SMs, 10.5, 8.8 and 8.4. k = 0: 1000 of 9000 5.9 with 128, 7.6 with 256; 600 of 60000 22.5 and 17.
    const bool is_short = a.vocab * int64_t(sizeof(T)) <= 64 * 1024, many = a.rows > 2 * int64_t(ctx->sm_count);
    if (is_short && many) return a.k ? launch_logprobs<T, true, 128>(ctx, X, a) : launch_logprobs<T, false, 128>(ctx, X, a);
    if (is_short || !a.k) return a.k ? launch_logprobs<T, true, 256>(ctx, X, a) : launch_logprobs<T, false, 256>(ctx, X, a);
    return launch_logprobs<T, true, 512>(ctx, X, a);
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
