// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale q.k_j (capped: c tanh(s_j / c)),  p = softmax(s),  o = sum p_j v_j,  lse = log sum exp(s_j)
//
// docc has no such node; beside the attention entry (contiguous K and V, every query at once) this is its form for serving.
//
// Bound by the bytes of the cache: every key and value is used by the group = Hq / Hkv query heads that share it and by nothing
// else, so it is read once, and the work is what keeps that stream full.
//   * The visible tokens of a (sequence, key-value head, tile of query heads) are a row of chunks. All rows' chunks form one line,
//     cut into as many equal runs as there are blocks: one long sequence, many short ones and any mixture load every SM alike. The
//     lengths are read on the device, so a captured graph follows them.
//   * A run that holds a whole row writes its output; rows that several runs share leave partial results (maximum, sum,
//     unnormalised output) in the scratch, which a second small kernel joins in the order of the runs: no atomics, and the same
//     result on every call.
//   * Inside a block every warp has its own keys of each chunk, its own ring of asynchronous copies and its own running maximum and
//     sum: nothing synchronises but the merge of the four warps at the end of a row.
//
// Measured (bf16 / fp16, heads of 128, fresh inputs per call): 64 ragged sequences up to 8192 tokens, 32 heads on 8, 609 MB: 116 us
// (5.2 TB/s, 0.80 of the measured copy); one of 131079 tokens, 16 heads on 2, capped scores, 134 MB: 37.2 us, of which the stream is 25,
// the first chunk's way through lengths, page table and keys 3, the join 8 with its launch; one of 1025: 10.0 us. In an early form the
// median block of the first case was done after 102 us and the slowest, with a run of short rows, after 142: hence kRowCost. More runs
// than resident blocks gained nothing (147, 155 and 166 us with 2, 4 and 8 times as many).
#include <type_traits>

#include "common.cuh"
#include "device_math.cuh"
#include "ptx.cuh"

namespace docc_b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRowCost = 1;
constexpr int64_t kMostTokens = (int64_t(1) << 31) - 4096;  // token numbers of a chunk past the end still fit in 32 bits
constexpr float kLog2e = 1.4426950408889634f;

struct PagedArgs {
    int B, Hq, Hkv, D, group, tiles, tile_rows;  // group = Hq / Hkv query heads share a key-value head, in `tiles` tiles of tile_rows
    int chunk;                                   // keys per chunk
    float scale, softcap;
    int64_t window;
    int64_t qs[2], os[2], ks[3], vs[3];  // element strides: (sequence, head), (page, head, place)
    int64_t num_pages, max_pages, table_stride;
    uint32_t page_size;
    const int32_t* page_table;
    const int32_t* lengths;
    float* lse;
    DeviceStatus* status;
    // scratch: two partial results per block (the row it finished for an earlier block, the row it began), and which rows are in
    // parts: an entry per row where there are fewer rows than blocks, else one per block for the row it began and did not finish
    int part_d;       // D rounded up to a multiple of 4
    float* part_o;    // [2 * blocks][tile_rows][part_d]
    float2* part_ml;  // [2 * blocks][tile_rows]: maximum of the scores, sum
    int4* split;      // {row or -1, its first block, its last block, 0}
    int by_row;
};

// Visible tokens [lo, n) of sequence b.
__device__ __forceinline__ void visible(const PagedArgs& a, int b, int& lo, int& n) {
    n = a.lengths[b];
    int64_t most = a.max_pages * int64_t(a.page_size);
    if (most > kMostTokens) most = kMostTokens;
    if (n < 0 || n > most) {
        report_bad_index(a.status, kIndexLength);
        n = n < 0 ? 0 : int(most);
    }
    lo = a.window > 0 && n > a.window ? n - int(a.window) : 0;
}
// An empty sequence has one chunk without visible keys, so that its output is written like any other.
__device__ __forceinline__ int chunks_of(const PagedArgs& a, int lo, int n) { return n > lo ? (n - lo + a.chunk - 1) / a.chunk : 1; }

// A place on the line of chunks: sequence-major, then key-value head, then tile of query heads, then chunk. Every row also counts
// kRowCost chunks in front of its first that hold nothing: they stand for the merge and the new queries, without which a run of
// many short rows takes far longer than a run of one long row.
struct Cursor {
    int b, kvh, tile, chunk, chunks, lo, n;
    int64_t left;  // what is left of the run on the line, this chunk included
    __device__ __forceinline__ void enter(const PagedArgs& a) {
        visible(a, b, lo, n);
        chunks = chunks_of(a, lo, n);
    }
    // to the run's next chunk; false if there is none
    __device__ __forceinline__ bool next(const PagedArgs& a) {
        if (--left <= 0) return false;
        if (++chunk < chunks) return true;
        left -= kRowCost;
        if (left <= 0) return false;
        chunk = 0;
        if (++tile < a.tiles) return true;
        tile = 0;
        if (++kvh < a.Hkv) return true;
        kvh = 0;
        b++;
        enter(a);
        return true;
    }
};

__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {  // both positive; 32 bits where they fit
    return ((a | b) >> 32) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

struct Run {
    int64_t begin, end, base, extra;  // the first `extra` runs are base + 1 long, the others base
    Cursor at;
    __device__ __forceinline__ int block_of(int64_t place) const {
        const int64_t longer = extra * (base + 1);
        return int(place < longer ? divide(place, base + 1) : extra + divide(place - longer, base));
    }
};

// The calling warp's run and its first chunk; false if the run holds none. Every warp works it out for itself, 32 sequences at a time.
__device__ __forceinline__ bool find_run(const PagedArgs& a, Run& r) {
    const int lane = threadIdx.x & 31;
    const int64_t rows = int64_t(a.Hkv) * a.tiles;
    auto length_of = [&](int b) -> int64_t {  // of a sequence's rows on the line
        if (b >= a.B) return 0;
        int lo, n;
        visible(a, b, lo, n);
        return (chunks_of(a, lo, n) + kRowCost) * rows;
    };
    const int64_t first = length_of(lane);
    int64_t total = first;
    for (int b = lane + 32; b < a.B; b += 32) total += length_of(b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    r.base = divide(total, gridDim.x);
    r.extra = total - r.base * gridDim.x;
    const int64_t c = blockIdx.x;
    r.begin = c * r.base + (c < r.extra ? c : r.extra);
    r.end = r.begin + r.base + (c < r.extra ? 1 : 0);
    if (r.begin == r.end) return false;
    int64_t before = 0;
    for (int base = 0; base < a.B; base += 32) {
        const int64_t mine = base == 0 ? first : length_of(base + lane);
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + upto > r.begin);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int64_t offset = r.begin - before - __shfl_sync(0xffffffffu, upto - mine, src);
            r.at.b = base + src;
            r.at.enter(a);
            const int length = r.at.chunks + kRowCost, row = int(divide(offset, length));
            const int place = int(offset - int64_t(row) * length);
            r.at.chunk = place < kRowCost ? 0 : place - kRowCost;
            r.at.left = r.end - r.begin - (place < kRowCost ? kRowCost - place : 0);
            r.at.kvh = row / a.tiles;
            r.at.tile = row - r.at.kvh * a.tiles;
            return r.at.left > 0;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;  // not reached: begin lies on the line
}
__device__ __forceinline__ int row_of(const PagedArgs& a, const Cursor& c) { return (c.b * a.Hkv + c.kvh) * a.tiles + c.tile; }

// The page entry of the calling lane's key (-1: not visible).
__device__ __forceinline__ int page_entry(const PagedArgs& a, const Cursor& c, int key) {
    if (key >= c.n) return -1;
    const int e = a.page_table[c.b * a.table_stride + uint32_t(key) / a.page_size];
    if (e < 0 || e >= a.num_pages) {
        report_bad_index(a.status, kIndexPage);
        return -1;
    }
    return e;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool keep) {
    const int bytes = keep ? 16 : 0;  // 0: the 16 bytes are filled with zeros and nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 2^((x - ref) log2 e): the difference is formed first, so that what is rounded by the product is as small as it. The hardware's
// exponential serves fp32 as well: 16 ragged sequences of 16 heads of 64 are 1.3e-7 from fp64 with it, the plain fp32 form 1.2e-7.
__device__ __forceinline__ float exp_from(float x, float ref) { return ex2((x - ref) * kLog2e); }

// Scaled and capped score.
__device__ __forceinline__ float score_of(const PagedArgs& a, float dot) {
    const float s = dot * a.scale;
    return a.softcap > 0.f ? a.softcap * tanhf(s / a.softcap) : s;
}
// The same for 16-bit keys without tanhf's two branches, which took half of the kernel's time: 1 - 2 / (e^2y + 1), off by 4 * 2^-24
// whatever y, and its series up to y^11, off by 2^-26 of the value, where y is below 0.35 and that would show.
__device__ __forceinline__ float capped_score(float dot, float per_cap, float cap) {
    const float y = dot * per_cap, z = y * y;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(ex2(y * (2.f * kLog2e)) + 1.f));
    float p = fmaf(z, -1382.f / 155925.f, 62.f / 2835.f);
    p = fmaf(z, p, -17.f / 315.f);
    p = fmaf(z, p, 2.f / 15.f);
    p = fmaf(z, p, -1.f / 3.f);
    p = fmaf(y * z, p, y);
    return cap * (fabsf(y) < 0.35f ? p : fmaf(-2.f, r, 1.f));
}

// The four warps' maxima and sums of one query head, and what each warp's output counts in the row's.
struct Merged {
    float top, sum, weight[kWarps];
    template <typename Rows> __device__ __forceinline__ Merged(const Rows& ml, int row) {
        top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; w++) top = fmaxf(top, ml[w][row].x);
        const float ref = top == -INFINITY ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            weight[w] = exp_from(ml[w][row].x, ref);
            sum = fmaf(weight[w], ml[w][row].y, sum);
        }
    }
    __device__ __forceinline__ float lse() const { return sum == 0.f ? -INFINITY : top + logf(sum); }
};

// ---- 16-bit inputs: tensor cores ---------------------------------------------------------------------------------------------
// A warp step is 16 keys. S = Q K^T and O += P V run as m16n8k16 products with the (up to 16) query heads of the tile as rows: one
// row tile is all the rows there are, and at 2 group flops per byte of cache the warp-level instruction has the rate several times
// over, while the 128-row accumulators of tcgen05 would be 8/128 full and pay the trip through tensor memory on every step.
// Q stays in registers, K comes as B fragments by ldmatrix, P goes from accumulator to A operand without leaving the registers.
// P enters the product as two 16-bit parts (p = hi + lo): a single bf16 would add an error as large as the output's own rounding.
// fp16 takes P times 2^15, which the output is divided by at the merge: both parts end at fp16's smallest step, 2^-24, and without the
// factor 8192 keys 18 below one that dominates, together a probability of 1e-4 each 1.5e-8, lost a fifth of their share. 1 becomes
// 32768, inside fp16's range, and what is lost is below 2^-40 of the largest probability. The sum needs no factor: it is fp32.
template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
// hi = the pair rounded to 16 bits towards zero, lo = what that left, rounded. Neither is negative, and lo is at least the type's
// smallest number (fp16: smallest step) where hi is not 0, so that an infinite value times the two gives twice that infinity: 0 inf
// or the difference of two infinities would be a NaN.
template <typename T> __device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    uint32_t least;
    if constexpr (std::is_same<T, __half>::value) {
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        lo = pack2<T>(x - f.x, y - f.y);
        asm("min.f16x2 %0, %1, %2;" : "=r"(least) : "r"(hi), "r"(0x00010001u));
        asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(least));
    } else {
        asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
        lo = pack2<T>(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
        asm("min.bf16x2 %0, %1, %2;" : "=r"(least) : "r"(hi), "r"(0x00800080u));
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(lo) : "r"(least));
    }
}

template <int DP> struct TcShape {
    static constexpr int kRow = DP * 2;                      // bytes of a key or value in shared memory
    static constexpr int kStage = 2 * 16 * kRow;             // 16 keys and 16 values of one warp
    static constexpr int kStages = DP <= 64 ? 5 : DP <= 96 ? 4 : 3;
    static constexpr int kBytes = kWarps * kStages * kStage + kWarps * 8 * DP * 4;
    // place of a pair of columns in a warp's eight merged rows: four rows at one column lie in different banks
    static __device__ __forceinline__ int merged(int warp, int row, int d) { return (warp * 8 + row) * DP + (d ^ ((row & 3) << 3)); }
    // 16-byte pieces of a row are permuted so that the eight rows an ldmatrix reads at one column lie in different banks
    static __device__ __forceinline__ uint32_t offset(int row, int piece) {
        const int turn = DP == 96 ? (row >> 1) & 3 : row & 7;
        return uint32_t(row * kRow + ((piece ^ turn) << 4));
    }
};

template <typename T> constexpr float kLift = std::is_same<T, __half>::value ? 0x1p15f : 1.f;

// HALVES: 1 where the tile has at most eight query heads (rows 8-15 of the fragments are padding), else 2.
template <typename T, int DP, int HALVES>
__global__ void __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) paged_tc_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                            T* __restrict__ O, PagedArgs a) {
    using Shape = TcShape<DP>;
    constexpr int S = Shape::kStages, PIECES = DP / 8, NT = DP / 8;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float2 ml_s[kWarps][16];
    __shared__ uint32_t mask_s[kWarps][S];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned char* ring = smem + warp * (S * Shape::kStage);
    const uint32_t ring_u = ptx::smem_u32(ring);
    float* merge = reinterpret_cast<float*>(smem + kWarps * S * Shape::kStage);
    const int pieces = a.D / 8;
    if (pieces < PIECES) {  // the padding of the head is never written again
        for (int i = lane; i < S * Shape::kStage / 16; i += 32) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();

    Run run;
    if (!find_run(a, run)) {
        if (threadIdx.x == 0 && !a.by_row) a.split[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
    }
    Cursor load = run.at, at = run.at;
    bool more = true;  // the load cursor stands on a chunk that has not been asked for

    const int key_lane = warp * 16 + (lane & 15);
    int key = load.lo + load.chunk * a.chunk + key_lane;
    int entry = page_entry(a, load, key);
    auto issue = [&](int stage) {  // copies of the load cursor's unit; `entry` and `key` are its own
        const bool ok = entry >= 0;
        const uint32_t mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
        if (lane == 0) mask_s[warp][stage] = mask;
        if (mask) {
            const uint32_t place = uint32_t(key) % a.page_size;
            const int64_t ko = ok ? entry * a.ks[0] + load.kvh * a.ks[1] + place * a.ks[2] : 0;
            const int64_t vo = ok ? entry * a.vs[0] + load.kvh * a.vs[1] + place * a.vs[2] : 0;
            const uint32_t dst = ring_u + stage * Shape::kStage;
#pragma unroll
            for (int i = 0; i < 16 * PIECES / 32; i++) {
                const int row = (i * 32 + lane) / PIECES, piece = (i * 32 + lane) % PIECES;
                const int64_t kr = __shfl_sync(0xffffffffu, ko, row), vr = __shfl_sync(0xffffffffu, vo, row);
                const bool keep = (mask >> row) & 1;
                if (piece < pieces) {
                    const uint32_t to = dst + Shape::offset(row, piece);
                    cp_async_16(to, K + kr + piece * 8, keep);
                    cp_async_16(to + 16 * Shape::kRow, V + vr + piece * 8, keep);
                }
            }
        }
        cp_async_commit();
    };
    auto advance = [&]() {  // the entry is fetched one step before its copies are issued
        more = load.next(a);
        if (more) {
            key = load.lo + load.chunk * a.chunk + key_lane;
            entry = page_entry(a, load, key);
        }
    };
#pragma unroll
    for (int s = 0; s < S - 1; s++) {
        if (more) {
            issue(s);
            advance();
        } else {
            cp_async_commit();
        }
    }

    const float per_cap = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
    uint32_t qf[DP / 16][4];
    float acc[NT][4], m[HALVES], l[HALVES];
    int first_chunk = -1, begun = -1, last = 0, stage = 0;
    do {
        if (first_chunk < 0) {  // a row begins
            first_chunk = at.chunk;
            const int r0 = at.tile * 16 + (lane >> 2);
            const T* q0 = Q + at.b * a.qs[0] + (int64_t(at.kvh) * a.group + r0) * a.qs[1];
            const T* q1 = q0 + 8 * a.qs[1];
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk++) {
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int d = kk * 16 + half * 8 + (lane & 3) * 2;
                    const bool in = d < a.D;
                    qf[kk][half * 2] = in && r0 < a.group ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
                    qf[kk][half * 2 + 1] = HALVES == 2 && in && r0 + 8 < a.group ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
                }
            }
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][e] = 0.f;
#pragma unroll
            for (int r = 0; r < HALVES; r++) {
                m[r] = -INFINITY;
                l[r] = 0.f;
            }
        }
        cp_async_wait<S - 2>();
        __syncwarp();  // every lane's copies of this step have landed, and every lane is done with the stage filled next
        if (more) {
            issue(stage == 0 ? S - 1 : stage - 1);
            advance();
        } else {
            cp_async_commit();
        }
        const uint32_t mask = mask_s[warp][stage];
        if (mask) {
            const uint32_t kb = ring_u + stage * Shape::kStage, vb = kb + 16 * Shape::kRow;
            float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk++) {
                uint32_t b[4];  // keys 0-7 and 8-15, dims 0-7 and 8-15 of this step
                ldmatrix_x4(b, kb + Shape::offset((lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
                mma16816<T>(s[0], qf[kk], b[0], b[1]);
                mma16816<T>(s[1], qf[kk], b[2], b[3]);
            }
            if (a.softcap > 0.f) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 2 * HALVES; e++) s[t][e] = capped_score(s[t][e], per_cap, a.softcap);
            } else {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 2 * HALVES; e++) s[t][e] *= a.scale;
            }
            if (mask != 0xffffu) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 2 * HALVES; e++)
                        if (!((mask >> (t * 8 + (lane & 3) * 2 + (e & 1))) & 1)) s[t][e] = -INFINITY;
            }
            float corr[HALVES], ref[HALVES];
            bool moved = false;
#pragma unroll
            for (int r = 0; r < HALVES; r++) {
                float x = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                const float mn = fmaxf(m[r], x);
                ref[r] = mn == -INFINITY ? 0.f : mn;  // only scores of -inf so far: e^(-inf - 0) = 0, not a NaN
                corr[r] = exp_from(m[r], ref[r]);
                moved = moved || m[r] != mn;
                m[r] = mn;
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int r = 0; r < HALVES; r++) {
                    l[r] *= corr[r];
#pragma unroll
                    for (int i = 0; i < NT; i++) {
                        acc[i][2 * r] *= corr[r];
                        acc[i][2 * r + 1] *= corr[r];
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (e >= 2 * HALVES) {
                        s[t][e] = 0.f;
                        continue;
                    }
                    s[t][e] = exp_from(s[t][e], ref[e >> 1]);
                    l[e >> 1] += s[t][e];
                }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                split2<T>(s[t][0] * kLift<T>, s[t][1] * kLift<T>, hi[2 * t], lo[2 * t]);
                split2<T>(s[t][2] * kLift<T>, s[t][3] * kLift<T>, hi[2 * t + 1], lo[2 * t + 1]);
            }
#pragma unroll
            for (int i = 0; i < NT / 2; i++) {
                uint32_t b[4];  // keys 0-7 and 8-15 of dims 16i..16i+7, then of the next eight
                ldmatrix_x4_trans(b, vb + Shape::offset(lane & 15, i * 2 + (lane >> 4)));
                mma16816<T>(acc[2 * i], hi, b[0], b[1]);
                mma16816<T>(acc[2 * i + 1], hi, b[2], b[3]);
                mma16816<T>(acc[2 * i], lo, b[0], b[1]);
                mma16816<T>(acc[2 * i + 1], lo, b[2], b[3]);
            }
        }
        const bool row_done = at.chunk + 1 == at.chunks;
        if (row_done || at.left == 1) {  // the row, or this block's part of it, is complete
#pragma unroll
            for (int r = 0; r < HALVES; r++) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
                if ((lane & 3) == 0) ml_s[warp][(lane >> 2) + 8 * r] = make_float2(m[r], l[r]);
            }
            const bool whole = first_chunk == 0 && row_done;
            const int64_t part = 2 * int64_t(blockIdx.x) + (first_chunk == 0 ? 1 : 0);
#pragma unroll
            for (int r = 0; r < HALVES; r++) {  // eight query heads at a time meet in shared memory
#pragma unroll
                for (int i = 0; i < NT; i++)
                    *reinterpret_cast<float2*>(merge + Shape::merged(warp, lane >> 2, i * 8 + (lane & 3) * 2)) =
                        make_float2(acc[i][2 * r] * (1.f / kLift<T>), acc[i][2 * r + 1] * (1.f / kLift<T>));
                __syncthreads();
                const int d = (threadIdx.x % (DP / 2)) * 2;
                for (int g = threadIdx.x / (DP / 2); g < 8; g += kThreads / (DP / 2)) {
                    const int in_group = at.tile * 16 + 8 * r + g;
                    if (in_group >= a.group || threadIdx.x >= kThreads / (DP / 2) * (DP / 2)) break;
                    const Merged all(ml_s, 8 * r + g);
                    float2 o = make_float2(0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < kWarps; w++) {
                        const float2 x = *reinterpret_cast<const float2*>(merge + Shape::merged(w, g, d));
                        o.x = fmaf(all.weight[w], x.x, o.x);
                        o.y = fmaf(all.weight[w], x.y, o.y);
                    }
                    const int64_t head = int64_t(at.kvh) * a.group + in_group;
                    if (whole) {
                        const float inv = all.sum == 0.f ? 0.f : 1.f / all.sum;
                        if (d < a.D) *reinterpret_cast<uint32_t*>(O + at.b * a.os[0] + head * a.os[1] + d) = pack2<T>(o.x * inv, o.y * inv);
                        if (a.lse && d == 0) a.lse[at.b * int64_t(a.Hq) + head] = all.lse();
                    } else {
                        if (d < a.D) *reinterpret_cast<float2*>(a.part_o + (part * a.tile_rows + 8 * r + g) * a.part_d + d) = o;
                        if (d == 0) a.part_ml[part * a.tile_rows + 8 * r + g] = make_float2(all.top, all.sum);
                    }
                }
                __syncthreads();  // the buffers are the next eight heads' or the next row's
            }
            if (first_chunk == 0) {
                if (!whole) {
                    begun = row_of(a, at);
                    last = run.block_of(run.end + (at.chunks - 2 - at.chunk));
                }
                if (a.by_row && threadIdx.x == 0) a.split[row_of(a, at)] = make_int4(begun, blockIdx.x, last, 0);
            }
            first_chunk = -1;
        }
        stage = stage + 1 == S ? 0 : stage + 1;
    } while (at.next(a));
    if (threadIdx.x == 0 && !a.by_row) a.split[blockIdx.x] = make_int4(begun, blockIdx.x, last, 0);
}

// ---- fp32, and whatever is not aligned for 16-byte copies: FMA units -------------------------------------------------------------
// A warp step is KS keys, 32 / KS lanes to a key for the scores and DP / 32 columns to a lane for the output; keys and values are
// staged as fp32. Up to GT query heads share the step. With one head per key-value head the stream bounds it (16 sequences of 16
// heads of 128: 63 us for a floor of 56; of 64: 22 for 15); with several, the query's and the values' trips through shared memory
// do, at 8 warps to an SM: 16 sequences with 4 heads to a key-value head of 128 take 55 us for a floor of 28, 16 to one of 80 60 for 9. Operands
// that are not aligned are loaded element by element, each load waiting where it is issued (16 heads of 64 off the boundary: 350 us, bf16 330).
template <int DP, int GT> struct SimtShape {
    static constexpr int kKeys = 1024 / DP;                      // 16, 8, 4
    static constexpr int kLanes = 32 / kKeys;                    // lanes per key
    static constexpr int kPieces = DP / 4;                       // 16-byte pieces of a row
    static constexpr int kStage = 2 * kKeys * DP * 4;            // 8 KB
    static constexpr int kStages = 3;
    // Query heads that are merged at a time: with all eight at DP = 128 the block had 117 KB and an SM room for one instead of two.
    static constexpr int kMerge = GT < 4 ? GT : 4;
    static constexpr int kBytes = kWarps * kStages * kStage + (kWarps * kMerge + GT) * DP * 4;  // the ring, the outputs, the queries
    static __device__ __forceinline__ int offset(int row, int piece) {  // in floats; eight lanes of a step read eight banks
        return row * DP + ((piece ^ ((row * kLanes) & 7)) << 2);
    }
};

template <typename T, int DP, int GT, bool ASYNC>
__global__ void __launch_bounds__(kThreads, 2) paged_simt_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                              T* __restrict__ O, PagedArgs a) {
    using Shape = SimtShape<DP, GT>;
    constexpr int S = Shape::kStages, KS = Shape::kKeys, LPK = Shape::kLanes, PIECES = Shape::kPieces, C = DP / 32;
    static_assert(!ASYNC || sizeof(T) == 4, "asynchronous copies keep the type");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float2 ml_s[kWarps][GT];
    __shared__ uint32_t mask_s[kWarps][S];
    __shared__ __align__(16) float p_s[kWarps][GT][KS];
    __shared__ float corr_s[kWarps][GT];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float* ring = reinterpret_cast<float*>(smem + warp * (S * Shape::kStage));
    float* merge = reinterpret_cast<float*>(smem + kWarps * S * Shape::kStage);
    float* q_s = merge + kWarps * Shape::kMerge * DP;
    if (a.D < DP) {
        for (int i = lane; i < S * Shape::kStage / 4; i += 32) ring[i] = 0.f;
        __syncwarp();
    }
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();

    Run run;
    if (!find_run(a, run)) {
        if (threadIdx.x == 0 && !a.by_row) a.split[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
    }
    Cursor load = run.at, at = run.at;
    bool more = true;  // the load cursor stands on a chunk that has not been asked for
    const int key_lane = warp * KS + (lane % KS);
    int key = load.lo + load.chunk * a.chunk + key_lane;
    int entry = page_entry(a, load, key);
    auto issue = [&](int stage) {
        const bool ok = entry >= 0;
        const uint32_t mask = __ballot_sync(0xffffffffu, ok) & ((1u << KS) - 1u);
        if (lane == 0) mask_s[warp][stage] = mask;
        if (mask) {
            const uint32_t place = uint32_t(key) % a.page_size;
            const int64_t ko = ok ? entry * a.ks[0] + load.kvh * a.ks[1] + place * a.ks[2] : 0;
            const int64_t vo = ok ? entry * a.vs[0] + load.kvh * a.vs[1] + place * a.vs[2] : 0;
            float* to = ring + stage * (Shape::kStage / 4);
            if constexpr (ASYNC) {
                const int pieces = a.D / 4;
#pragma unroll
                for (int i = 0; i < KS * PIECES / 32; i++) {
                    const int row = (i * 32 + lane) / PIECES, piece = (i * 32 + lane) % PIECES;
                    const int64_t kr = __shfl_sync(0xffffffffu, ko, row), vr = __shfl_sync(0xffffffffu, vo, row);
                    const bool keep = (mask >> row) & 1;
                    if (piece < pieces) {
                        const uint32_t dst = ptx::smem_u32(to + Shape::offset(row, piece));
                        cp_async_16(dst, K + kr + piece * 4, keep);
                        cp_async_16(dst + KS * DP * 4, V + vr + piece * 4, keep);
                    }
                }
            } else {
                for (int row = 0; row < KS; row++) {
                    const int64_t kr = __shfl_sync(0xffffffffu, ko, row), vr = __shfl_sync(0xffffffffu, vo, row);
                    const bool keep = (mask >> row) & 1;
                    for (int d = lane; d < a.D; d += 32) {
                        float* dst = to + Shape::offset(row, d >> 2) + (d & 3);
                        dst[0] = keep ? to_float(K[kr + d]) : 0.f;
                        dst[KS * DP] = keep ? to_float(V[vr + d]) : 0.f;
                    }
                }
            }
        }
        if constexpr (ASYNC) cp_async_commit();
    };
    auto advance = [&]() {
        more = load.next(a);
        if (more) {
            key = load.lo + load.chunk * a.chunk + key_lane;
            entry = page_entry(a, load, key);
        }
    };
#pragma unroll
    for (int s = 0; s < S - 1; s++) {
        if (more) {
            issue(s);
            advance();
        } else if constexpr (ASYNC) {
            cp_async_commit();
        }
    }

    // A lane's scores are those of GL query heads from `own` on, of one key; DUP lanes hold the same one.
    constexpr int GL = GT > LPK ? GT / LPK : 1, DUP = LPK > GT ? LPK / GT : 1;
    const int my_key = lane / LPK, sub = lane % LPK, own = sub / DUP * GL;
    float acc[GT][C], m[GL], l[GL];
    int first_chunk = -1, begun = -1, last = 0, stage = 0;
    do {
        if (first_chunk < 0) {
            first_chunk = at.chunk;
            // the merge that ended the row before was followed by a barrier: nobody reads q_s any more
            for (int i = threadIdx.x; i < GT * DP; i += kThreads) {
                const int g = i / DP, d = i % DP, in_group = at.tile * GT + g;
                q_s[i] = d < a.D && in_group < a.group
                             ? to_float(Q[at.b * a.qs[0] + (int64_t(at.kvh) * a.group + in_group) * a.qs[1] + d])
                             : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int g = 0; g < GT; g++)
#pragma unroll
                for (int c = 0; c < C; c++) acc[g][c] = 0.f;
#pragma unroll
            for (int i = 0; i < GL; i++) {
                m[i] = -INFINITY;
                l[i] = 0.f;
            }
        }
        if constexpr (ASYNC) cp_async_wait<S - 2>();
        __syncwarp();
        if (more) {
            issue(stage == 0 ? S - 1 : stage - 1);
            advance();
        } else if constexpr (ASYNC) {
            cp_async_commit();
        }
        const uint32_t mask = mask_s[warp][stage];
        if (mask) {
            const float* kb = ring + stage * (Shape::kStage / 4);
            const float* vb = kb + KS * DP;
            float s[GT];
#pragma unroll
            for (int g = 0; g < GT; g++) s[g] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int piece = i * LPK + sub;
                const float4 k4 = *reinterpret_cast<const float4*>(kb + Shape::offset(my_key, piece));
#pragma unroll
                for (int g = 0; g < GT; g++) {
                    const float4 q4 = *reinterpret_cast<const float4*>(q_s + g * DP + piece * 4);
                    s[g] = fmaf(k4.x, q4.x, fmaf(k4.y, q4.y, fmaf(k4.z, q4.z, fmaf(k4.w, q4.w, s[g]))));
                }
            }
            const bool seen = (mask >> my_key) & 1;
            // The lanes of a key add up their shares and divide the heads among themselves on the way: each step sends the half of the
            // heads that the other lane keeps. Cap, exponential and maximum are then taken once per key and head, not once per lane.
#pragma unroll
            for (int o = LPK / 2, n = GT; o > 0; o >>= 1) {
                if (n > 1) {
                    n >>= 1;
#pragma unroll
                    for (int i = 0; i < GT / 2; i++) {
                        if (i >= n) break;
                        const bool upper = sub & o;
                        const float give = upper ? s[i] : s[i + n], keep = upper ? s[i + n] : s[i];
                        s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                    }
                } else {
                    s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
                }
            }
            __syncwarp();  // p_s and corr_s of the step before have been read
            bool moved = false;
#pragma unroll
            for (int i = 0; i < GL; i++) {
                const float x = seen ? score_of(a, s[i]) : -INFINITY;
                float top = x;
#pragma unroll
                for (int o = LPK; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float mn = fmaxf(m[i], top), ref = mn == -INFINITY ? 0.f : mn;
                const float corr = exp_from(m[i], ref), p = exp_from(x, ref);
                moved = moved || m[i] != mn;
                m[i] = mn;
                l[i] = l[i] * corr + (sub % DUP == 0 ? p : 0.f);
                if (sub % DUP == 0) p_s[warp][own + i][my_key] = p;
                if (lane < LPK && sub % DUP == 0) corr_s[warp][own + i] = corr;
            }
            const bool any_moved = __any_sync(0xffffffffu, moved);
            __syncwarp();
            if (any_moved) {
#pragma unroll
                for (int g = 0; g < GT; g++) {
                    const float corr = corr_s[warp][g];
#pragma unroll
                    for (int c = 0; c < C; c++) acc[g][c] *= corr;
                }
            }
#pragma unroll
            for (int j4 = 0; j4 < KS / 4; j4++) {
                float v[4][C];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int row = j4 * 4 + j;
                    if constexpr (C == 2) {
                        const float2 f = *reinterpret_cast<const float2*>(vb + Shape::offset(row, lane >> 1) + (lane & 1) * 2);
                        v[j][0] = f.x; v[j][1] = f.y;
                    } else {
#pragma unroll
                        for (int h = 0; h < C / 4; h++) {
                            const float4 f = *reinterpret_cast<const float4*>(vb + Shape::offset(row, lane + 32 * h));
                            v[j][4 * h] = f.x; v[j][4 * h + 1] = f.y; v[j][4 * h + 2] = f.z; v[j][4 * h + 3] = f.w;
                        }
                    }
                }
#pragma unroll
                for (int g = 0; g < GT; g++) {
                    const float4 p4 = *reinterpret_cast<const float4*>(&p_s[warp][g][j4 * 4]);
#pragma unroll
                    for (int c = 0; c < C; c++)
                        acc[g][c] = fmaf(p4.x, v[0][c], fmaf(p4.y, v[1][c], fmaf(p4.z, v[2][c], fmaf(p4.w, v[3][c], acc[g][c]))));
                }
            }
        }
        const bool row_done = at.chunk + 1 == at.chunks;
        if (row_done || at.left == 1) {
            constexpr int M = Shape::kMerge;
            float* mine = merge + warp * (M * DP);
#pragma unroll
            for (int i = 0; i < GL; i++) {
#pragma unroll
                for (int o = LPK; o < 32; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
                if (lane < LPK && sub % DUP == 0) ml_s[warp][own + i] = make_float2(m[i], l[i]);
            }
            const bool whole = first_chunk == 0 && row_done;
            const int64_t part = 2 * int64_t(blockIdx.x) + (first_chunk == 0 ? 1 : 0);
#pragma unroll
            for (int g0 = 0; g0 < GT; g0 += M) {
#pragma unroll
                for (int g = 0; g < M; g++)
#pragma unroll
                    for (int c = 0; c < C; c++) mine[g * DP + (C == 2 ? lane * 2 + c : (c >> 2) * 128 + lane * 4 + (c & 3))] = acc[g0 + g][c];
                __syncthreads();
                for (int i = threadIdx.x; i < M * DP; i += kThreads) {
                    const int g = g0 + i / DP, d = i % DP, in_group = at.tile * GT + g;
                    if (in_group >= a.group) break;
                    const Merged all(ml_s, g);
                    float o = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; w++) o = fmaf(all.weight[w], merge[w * (M * DP) + i], o);
                    const int64_t head = int64_t(at.kvh) * a.group + in_group;
                    if (whole) {
                        if (d < a.D) O[at.b * a.os[0] + head * a.os[1] + d] = from_float<T>(all.sum == 0.f ? 0.f : o / all.sum);
                        if (a.lse && d == 0) a.lse[at.b * int64_t(a.Hq) + head] = all.lse();
                    } else {
                        if (d < a.D) a.part_o[(part * a.tile_rows + g) * a.part_d + d] = o;
                        if (d == 0) a.part_ml[part * a.tile_rows + g] = make_float2(all.top, all.sum);
                    }
                }
                __syncthreads();  // the buffers are the next heads' or the next row's
            }
            if (first_chunk == 0) {
                if (!whole) {
                    begun = row_of(a, at);
                    last = run.block_of(run.end + (at.chunks - 2 - at.chunk));
                }
                if (a.by_row && threadIdx.x == 0) a.split[row_of(a, at)] = make_int4(begun, blockIdx.x, last, 0);
            }
            first_chunk = -1;
        }
        stage = stage + 1 == S ? 0 : stage + 1;
    } while (at.next(a));
    if (threadIdx.x == 0 && !a.by_row) a.split[blockIdx.x] = make_int4(begun, blockIdx.x, last, 0);
}

// ---- join ----------------------------------------------------------------------------------------------------------------------
// Block (x, y, z): entry x of `split`, query head y of its tile, columns [z width, (z + 1) width). The row's parts lie in blocks first ..
// last: the first as the row begun, the others as the row finished for an earlier block. A part's columns are width / 4 lanes' (four
// each), the rest of the block's threads take other parts. The code is kept small: the kernel runs for a few microseconds, and
// unrolled eight-fold its instructions took longer to arrive than its data (17 against 11 against 7.4 us for 148 parts, caches cold).
constexpr int kJoinThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(T* __restrict__ O, PagedArgs a, int width) {
    __shared__ float4 sum_s[kJoinThreads / 32][32];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = int(blockIdx.y);
    const int4 entry = a.split[blockIdx.x];
    if (entry.x < 0) return;
    const int first = entry.y, parts = entry.z - first + 1;
    const int tile = entry.x % a.tiles, kvh = entry.x / a.tiles % a.Hkv, b = entry.x / a.tiles / a.Hkv;
    if (tile * a.tile_rows + r >= a.group) return;
    auto part = [&](int i) { return (2 * (first + i) + (i == 0 ? 1 : 0)) * a.tile_rows + r; };
    float top = -INFINITY, sum = 0.f;
#pragma unroll 2
    for (int i = lane; i < parts; i += 32) {
        const float2 ml = a.part_ml[part(i)];
        const float next = fmaxf(top, ml.x), ref = next == -INFINITY ? 0.f : next;
        sum = sum * exp_from(top, ref) + ml.y * exp_from(ml.x, ref);
        top = next;
    }
    const float all = warp_max_f(top), ref = all == -INFINITY ? 0.f : all;
    sum = warp_sum_f(sum * exp_from(top, ref));

    const int lanes = width / 4;  // to a part: 8, 16 or 32
    const int d = int(blockIdx.z) * width + (lane & (lanes - 1)) * 4;
    const float* columns = a.part_o + (d < a.part_d ? d : 0);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int i = int(threadIdx.x) / lanes; i < parts; i += int(blockDim.x) / lanes) {
        const float4 x = *reinterpret_cast<const float4*>(columns + int64_t(part(i)) * a.part_d);
        const float f = exp_from(a.part_ml[part(i)].x, ref);
        o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y); o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
    }
#pragma unroll 1
    for (int s = lanes; s < 32; s <<= 1) {
        o.x += __shfl_xor_sync(0xffffffffu, o.x, s); o.y += __shfl_xor_sync(0xffffffffu, o.y, s);
        o.z += __shfl_xor_sync(0xffffffffu, o.z, s); o.w += __shfl_xor_sync(0xffffffffu, o.w, s);
    }
    if (lane < lanes) sum_s[warp][lane] = o;
    __syncthreads();
    const int64_t head = int64_t(kvh) * a.group + tile * a.tile_rows + r;
    const int column = int(blockIdx.z) * width + int(threadIdx.x);
    if (int(threadIdx.x) < width && column < a.D) {
        float v = 0.f;
        for (int w = 0; w < int(blockDim.x >> 5); w++) v += reinterpret_cast<const float*>(sum_s[w])[threadIdx.x];
        O[b * a.os[0] + head * a.os[1] + column] = from_float<T>(sum == 0.f ? 0.f : v / sum);
    }
    if (a.lse && column == 0) a.lse[b * int64_t(a.Hq) + head] = sum == 0.f ? -INFINITY : all + logf(sum);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
constexpr int kTcRows = 16, kSimtRows = 8;

struct Scratch {
    size_t ml_at, o_at, bytes;
};
Scratch scratch_of(int blocks, int64_t group, int64_t D) {
    // the larger of the two kernels' tiles, so that the size does not depend on alignment
    const size_t rows = size_t(group < kTcRows ? group : kTcRows), parts = 2 * size_t(blocks);
    Scratch s;
    s.ml_at = (size_t(blocks) * sizeof(int4) + 255) / 256 * 256;
    s.o_at = s.ml_at + (parts * rows * sizeof(float2) + 255) / 256 * 256;
    s.bytes = s.o_at + parts * rows * size_t(ceil_div(D, 4) * 4) * 4;
    return s;
}
int blocks_of(Ctx* ctx, int64_t D) { return ctx->sm_count * (D <= 128 ? 2 : 1); }

template <typename T>
int launch_join(Ctx* ctx, const PagedArgs& a, int blocks, T* O) {
    const int entries = a.by_row ? int(int64_t(a.B) * a.Hkv * a.tiles) : blocks, heads = a.group < a.tile_rows ? a.group : a.tile_rows;
    // The fewer rows there are, the more parts each is in: 256 threads and narrow columns, hence up to 32 parts at a time, as long as
    // all blocks still run together; with many entries, most of which are gone after one load, 128 threads and whole rows.
    int width = 128, threads = 128;
    if (int64_t(entries) * heads <= int64_t(ctx->sm_count) * 4) {
        threads = kJoinThreads;
        while (width > 32 && int64_t(entries) * heads * ceil_div(a.D, width / 2) <= int64_t(ctx->sm_count) * 4) width /= 2;
    }
    const dim3 grid(unsigned(entries), unsigned(heads), unsigned(ceil_div(a.D, width)));
    DOCC_CUDA_TRY(launch_pdl(paged_join_kernel<T>, grid, dim3(unsigned(threads)), 0, ctx->stream, O, a, width));
    return after_launch(ctx, "paged_join_kernel");
}

template <typename T, int DP, int HALVES>
int launch_tc_rows(Ctx* ctx, PagedArgs& a, int blocks, const T* Q, const T* K, const T* V, T* O) {
    a.tile_rows = kTcRows;
    a.tiles = int(ceil_div(a.group, kTcRows));
    if (a.tiles == 1) a.tile_rows = a.group;  // the scratch holds no rows that do not exist
    a.chunk = kWarps * 16;
    a.by_row = int64_t(a.B) * a.Hkv * a.tiles <= blocks;
    auto kernel = paged_tc_kernel<T, DP, HALVES>;
    static std::atomic<unsigned> done{0};
    DOCC_TRY(set_smem(ctx, done, kernel, TcShape<DP>::kBytes));
    DOCC_CUDA_TRY(launch_pdl(kernel, dim3(unsigned(blocks)), dim3(kThreads), TcShape<DP>::kBytes, ctx->stream, Q, K, V, O, a));
    DOCC_TRY(after_launch(ctx, "paged_tc_kernel"));
    return launch_join<T>(ctx, a, blocks, O);
}

template <typename T, int DP>
int launch_tc(Ctx* ctx, PagedArgs& a, int blocks, const T* Q, const T* K, const T* V, T* O) {
    return a.group <= 8 ? launch_tc_rows<T, DP, 1>(ctx, a, blocks, Q, K, V, O) : launch_tc_rows<T, DP, 2>(ctx, a, blocks, Q, K, V, O);
}

template <typename T, int DP, int GT, bool ASYNC>
int launch_simt(Ctx* ctx, PagedArgs& a, int blocks, const T* Q, const T* K, const T* V, T* O) {
    a.tile_rows = GT;
    a.tiles = int(ceil_div(a.group, GT));
    if (a.tiles == 1) a.tile_rows = a.group;
    a.chunk = kWarps * SimtShape<DP, GT>::kKeys;
    a.by_row = int64_t(a.B) * a.Hkv * a.tiles <= blocks;
    auto kernel = paged_simt_kernel<T, DP, GT, ASYNC>;
    static std::atomic<unsigned> done{0};
    DOCC_TRY(set_smem(ctx, done, kernel, SimtShape<DP, GT>::kBytes));
    DOCC_CUDA_TRY(launch_pdl(kernel, dim3(unsigned(blocks)), dim3(kThreads), SimtShape<DP, GT>::kBytes, ctx->stream, Q, K, V, O, a));
    DOCC_TRY(after_launch(ctx, "paged_simt_kernel"));
    return launch_join<T>(ctx, a, blocks, O);
}
template <typename T, int DP, bool ASYNC>
int launch_simt_rows(Ctx* ctx, PagedArgs& a, int blocks, const T* Q, const T* K, const T* V, T* O) {
    if (a.group == 1) return launch_simt<T, DP, 1, ASYNC>(ctx, a, blocks, Q, K, V, O);
    if (a.group <= 4) return launch_simt<T, DP, 4, ASYNC>(ctx, a, blocks, Q, K, V, O);
    return launch_simt<T, DP, kSimtRows, ASYNC>(ctx, a, blocks, Q, K, V, O);
}
template <typename T, bool ASYNC>
int launch_simt_any(Ctx* ctx, PagedArgs& a, int blocks, const T* Q, const T* K, const T* V, T* O) {
    if (a.D <= 64) return launch_simt_rows<T, 64, ASYNC>(ctx, a, blocks, Q, K, V, O);
    if (a.D <= 128) return launch_simt_rows<T, 128, ASYNC>(ctx, a, blocks, Q, K, V, O);
    return launch_simt_rows<T, 256, ASYNC>(ctx, a, blocks, Q, K, V, O);
}

template <typename T>
int paged_device(Ctx* ctx, PagedArgs& a, int blocks, const void* Qv, const void* Kv, const void* Vv, void* Ov) {
    const T *Q = static_cast<const T*>(Qv), *K = static_cast<const T*>(Kv), *V = static_cast<const T*>(Vv);
    T* O = static_cast<T*>(Ov);
    constexpr int VEC = 16 / sizeof(T);
    bool aligned = a.D % VEC == 0;
    for (const void* p : {Qv, Kv, Vv, static_cast<const void*>(Ov)}) aligned = aligned && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int i = 0; i < 2; i++) aligned = aligned && a.qs[i] % VEC == 0 && a.os[i] % VEC == 0;
    for (int i = 0; i < 3; i++) aligned = aligned && a.ks[i] % VEC == 0 && a.vs[i] % VEC == 0;
    if constexpr (sizeof(T) == 2) {
        if (aligned) {
            if (a.D <= 64) return launch_tc<T, 64>(ctx, a, blocks, Q, K, V, O);
            if (a.D <= 96) return launch_tc<T, 96>(ctx, a, blocks, Q, K, V, O);
            if (a.D <= 128) return launch_tc<T, 128>(ctx, a, blocks, Q, K, V, O);
            return launch_tc<T, 256>(ctx, a, blocks, Q, K, V, O);
        }
    } else {
        if (aligned) return launch_simt_any<T, true>(ctx, a, blocks, Q, K, V, O);
    }
    return launch_simt_any<T, false>(ctx, a, blocks, Q, K, V, O);
}

}  // namespace
}  // namespace docc_b200

using namespace docc_b200;

extern "C" int docc_b200_paged_attention_workspace(int prec, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, size_t* bytes) {
    DOCC_REQUIRE(bytes != nullptr, "paged_attention_workspace: bytes is NULL");
    DOCC_REQUIRE(prec_size(prec) != 0 && prec != DOCC_B200_PREC_D, "paged_attention_workspace: precision %d not supported (use 's', 'b' or 'h')", prec);
    DOCC_REQUIRE(B >= 0 && Hq >= 0 && Hkv >= 0 && D >= 0, "paged_attention_workspace: negative extent");
    Ctx* ctx;
    DOCC_TRY(get_ctx(&ctx));
    *bytes = B == 0 || Hkv == 0 || D == 0 ? 0 : scratch_of(blocks_of(ctx, D), Hq / Hkv, D).bytes;
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
    DOCC_REQUIRE(softcap >= 0.f && softcap < INFINITY && window >= 0, "paged_attention: softcap must be finite, and neither it nor window negative");
    if (flags & DOCC_B200_FLAG_HOST_PTRS)
        return set_error(DOCC_B200_ERR_UNSUPPORTED, "paged_attention: the cache lives on the device; host pointers are not taken");
    Ctx* ctx;
    DOCC_TRY(get_ctx(&ctx));
    if (B == 0 || Hq == 0) return DOCC_B200_OK;
    if (D == 0) {
        DOCC_REQUIRE(!lse, "paged_attention: heads of no elements have no lse");
        return DOCC_B200_OK;
    }
    DOCC_REQUIRE(Hkv > 0 && Hq % Hkv == 0, "paged_attention: %lld query heads are not a multiple of %lld key-value heads", (long long)Hq,
                 (long long)Hkv);
    if (D > 256) return set_error(DOCC_B200_ERR_UNSUPPORTED, "paged_attention: head_dim %lld > 256", (long long)D);
    DOCC_REQUIRE(B <= 65535 && Hq <= 65535, "paged_attention: more than 65535 sequences or heads");
    DOCC_REQUIRE(B * Hq < (int64_t(1) << 31), "paged_attention: 2^31 or more rows");
    DOCC_REQUIRE(Q && O && lengths && (max_pages == 0 || (page_table && (num_pages == 0 || (Kcache && Vcache)))),
                 "paged_attention: NULL data pointer");
    DOCC_REQUIRE(table_stride >= max_pages, "paged_attention: table_stride below max_pages");
    DOCC_REQUIRE(page_size < (int64_t(1) << 31), "paged_attention: page_size of 2^31 or more");
    const int blocks = blocks_of(ctx, D);
    const Scratch scratch = scratch_of(blocks, Hq / Hkv, D);
    if (workspace) {
        DOCC_REQUIRE(workspace_bytes >= scratch.bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                     "paged_attention: the workspace needs %zu bytes on a 16-byte boundary", scratch.bytes);
    } else {
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        DOCC_CUDA_TRY(cudaStreamIsCapturing(ctx->stream, &capture));
        DOCC_REQUIRE(capture == cudaStreamCaptureStatusNone, "paged_attention: a captured call needs a workspace of its own");
        DOCC_TRY(get_workspace(ctx, 4, scratch.bytes, &workspace));
    }
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
    a.num_pages = num_pages; a.page_size = uint32_t(page_size); a.max_pages = max_pages; a.table_stride = table_stride;
    a.page_table = page_table; a.lengths = lengths; a.lse = static_cast<float*>(lse); a.status = ctx->status_dev;
    a.part_d = int(ceil_div(D, 4) * 4);
    a.split = static_cast<int4*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + scratch.ml_at);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + scratch.o_at);
    if (!Kcache) Kcache = Q;  // an empty cache: nothing of it is read, but copies of no bytes want an address
    if (!Vcache) Vcache = Q;
    if (prec == DOCC_B200_PREC_S) return paged_device<float>(ctx, a, blocks, Q, Kcache, Vcache, O);
    if (prec == DOCC_B200_PREC_H) return paged_device<__half>(ctx, a, blocks, Q, Kcache, Vcache, O);
    return paged_device<__nv_bfloat16>(ctx, a, blocks, Q, Kcache, Vcache, O);
}
