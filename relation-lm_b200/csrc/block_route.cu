// The choice of remote blocks for each query row by the router's block statistics: the TOP best blocks in descending order
// of their score, ties to the lowest block.
//
//     s_h(n) = (q_h . mean_h(n) + softplus(gamma_h) |q_h| . std_h(n)) / 4 + bias[h, bucket(t - end_n)]      (4 heads of 16)
//     s(n)   = log sum_h exp s_h(n),     end_n = (n + 1) BS - 1,     bucket(d) = floor(log2(max(d, 0) + 1))
//
// over the blocks that are complete at the row's position and, under the strict rule, end before its local window.
//
// The choice is the one that scores in 64 bits make.  All blocks are scored in 32 bits first, with a bound on the error
// from the sums of the magnitudes; what may belong to the TOP best by that bound (TOP or a few more) is scored again in
// 64 bits and ranked.  Near scores thus fall the same way in every form and whatever the order of a sum.
//
// Bytes bound long caches (256 bytes a block and row in 16 bits), latency the short ones.  Eight lanes share a block,
// 16 bytes of its mean and of its spread each, so a warp's load covers four whole rows of a statistic.  One row of 16 blocks
// 4.1 to 4.5 us, of 1024 blocks (over eight CTAs) 10.9; 256 rows of 1024 blocks 20 us from L2 (3.3 TB/s), 23.7 at unequal lengths
// from memory, a CTA a row.
#include "block_attention_mma.cuh"

namespace rlm {
namespace {

constexpr int kBrThreads = 256;
constexpr int kBrWarps = kBrThreads / 32;
constexpr int kBrMaxTop = 128;
constexpr int kBrWarpTop = 16;              // places that a warp alone chooses for
constexpr int kBtLeastRows = 8192;          // rows that the tiles of whole sequences take
constexpr int kBrMaxBuckets = 32;
constexpr int kBrBytesPerBlock = 40;        // of shared memory: 32-bit score, place in the list, the heads' 64-bit scores

constexpr int kBrMemory = kSmemDynamicLimit - 4096;
constexpr int kBrMaxParts = 8;              // CTAs that may share a row

struct RouteArgs {
    const void* query;
    const void* mean;
    const void* stdv;
    const void* gamma;
    const void* bias;
    Rows rows;
    int32_t* out_index;
    float* out_score;
    int32_t* status;
    int64_t q_stride;
    int n_blocks, block_size, buckets, window, top, strict;
    int parts, part_blocks;             // CTAs that share a row, blocks of each at most
    int query_dtype, param_dtype;
};

// Eight consecutive statistics.
template <typename T> __device__ __forceinline__ void load_stats(const T* p, float (&f)[8]) {
    load8(p, 0, sizeof(T) == 4 ? RLM_F32 : (std::is_same<T, __nv_bfloat16>::value ? RLM_BF16 : RLM_F16), f);
}

// A block's score in 64 bits.  exact_head: a head's by the two lanes that hold eight components each (both receive it).
template <typename T>
__device__ __forceinline__ double exact_head(const T* mean, const T* stdv, const float (&q)[8], double soft, double bias) {
    float m[8], s[8];
    load_stats(mean, m);
    load_stats(stdv, s);
    double near = 0.0, spread = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double qi = q[i];
        near = fma(qi, static_cast<double>(m[i]), near);
        spread = fma(fabs(qi), static_cast<double>(s[i]), spread);
    }
    near += __shfl_xor_sync(0xffffffffu, near, 1);
    spread += __shfl_xor_sync(0xffffffffu, spread, 1);
    return fma(soft, spread, near) * 0.25 + bias;
}

// The heads' logarithm of the sum of exponentials: an infinite head makes it infinite, a head that is NaN makes it NaN.
__device__ __forceinline__ double exact_term(double head, double top) { return top == INFINITY && head == head ? 0.0 : exp(head - top); }
__device__ __forceinline__ double exact_sum(double top, double part) { return top == INFINITY ? top + part : top + log(part); }
__device__ __forceinline__ double exact_join(double h0, double h1, double h2, double h3) {
    const double top = fmax(fmax(h0, h1), fmax(h2, h3));
    return exact_sum(top, (exact_term(h0, top) + exact_term(h1, top)) + (exact_term(h2, top) + exact_term(h3, top)));
}
// An integer that orders as the score does; NaN, like -inf, below all others (a zero's sign does not count).
__device__ __forceinline__ long long order_key(double x) {
    if (x != x) return static_cast<long long>(0x8000000000000000ull);
    const long long bits = __double_as_longlong(x + 0.0);
    return bits < 0 ? bits ^ 0x7fffffffffffffffll : bits;
}

__device__ __forceinline__ double soft_plus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }
__device__ __forceinline__ float fast_sqrt(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t load_pair(const void* p) { return __ldg(static_cast<const uint32_t*>(p)); }

// What a block's 32-bit score may be off by, twice: the error of a head's score is below 17 x 2^-24 of `size`, the sum of the
// magnitudes that it is made of (9 additions and the rounding of the products, 4 more operations, the shift by the largest),
// that of the exponentials' sum and its logarithm below 2^-19; twice as much is allowed for.
__device__ __forceinline__ float slack_of_size(float size) { return fmaf(size, 3.814697265625e-6f, 7.62939453125e-6f); }

// Squares below 2^-149 vanish from a norm, sixteen of them at most 2^-145: norms begin at a little more.  With that the bounds
// hold whatever the magnitudes, as long as the spreads' factor stays below kSteep; beyond it all blocks are scored in 64 bits.
constexpr float kLeastNorm = 1e-43f;
constexpr float kSteep = 1e10f;

// Eight consecutive statistics as they lie in memory.
template <typename T> struct RawStats;
template <> struct RawStats<float> {
    float4 lo, hi;
    __device__ __forceinline__ void load(const float* p) {
        lo = __ldg(reinterpret_cast<const float4*>(p));
        hi = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void widen(float (&f)[8]) const {
        f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w;
        f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
    }
};
template <typename T> struct RawStats {
    uint4 v;
    __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void widen(float (&f)[8]) const {
        load8(&v, 0, std::is_same<T, __nv_bfloat16>::value ? RLM_BF16 : RLM_F16, f);
    }
};

// kRowWarps warps work on a row: all eight of the CTA (few rows, long caches) or one (whole sequences).  With eight, a row's
// blocks may be divided over a cluster of CTAs: each finds its own TOP best, the first one ranks them all.
// kDeep: twice as many loads in flight and half as many CTAs an SM, for launches whose CTAs are few and long or hold too many
// scores to share an SM: 200 rows of 4096 blocks 85 us against 96, 256 rows of up to 1024 23.5 against 26.7, but 400 rows of 256
// 15.8 against 11.6.
template <typename T, int kRowWarps, bool kDeep>
__global__ void __launch_bounds__(kBrThreads, kDeep ? 2 : 4) block_route_kernel(const RouteArgs a) {
    constexpr int kRowsPerCta = kBrWarps / kRowWarps;
    constexpr int kRowThreads = 32 * kRowWarps;
    constexpr int kAhead = (sizeof(T) == 4 ? 2 : 4) * (kDeep ? 2 : 1);       // passes whose statistics are requested together
    extern __shared__ double row_memory[];               // per row: exact[NB][4] | approx[NB], list[NB]
    __shared__ float bias[4 * kBrMaxBuckets];
    __shared__ alignas(16) float lane_best[kBrThreads];
    __shared__ double soft_of[4];
    __shared__ int found_of[kRowsPerCta];
    __shared__ unsigned slack_of[kRowsPerCta];
    __shared__ float threshold_of[kRowsPerCta];
    __shared__ double best_value[kRowWarps == 1 ? 1 : kBrMaxTop];     // a cluster's CTA: its own best
    __shared__ int best_index[kRowWarps == 1 ? 1 : kBrMaxTop];

    const int own_row = threadIdx.x / kRowThreads, tid = threadIdx.x % kRowThreads;
    const int lane = threadIdx.x & 31, row_warp = tid >> 5;
    const int j = lane & 7, sub = lane >> 3, head = j >> 1;
    auto row_sync = [] { if (kRowWarps == 1) __syncwarp(); else __syncthreads(); };

    griddep_sync();
    const int parts = kRowWarps == 1 ? 1 : a.parts;
    const int row = kRowWarps == 1 ? blockIdx.x * kRowsPerCta + own_row : blockIdx.x / parts;
    const int rank_in_cluster = kRowWarps == 1 ? 0 : blockIdx.x - row * parts;
    const bool exists = row < a.rows.n_rows;
    // what does not depend on the row's position is requested before it is waited for
    static_assert(4 * kBrMaxBuckets <= kBrThreads - 4, "a thread a bias, four more for gamma");
    float parameter = 0.0f;
    if (static_cast<int>(threadIdx.x) < 4 * a.buckets) parameter = load_scalar(a.bias, threadIdx.x, a.param_dtype);
    if (threadIdx.x >= kBrThreads - 4) parameter = load_scalar(a.gamma, threadIdx.x - (kBrThreads - 4), a.param_dtype);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = exists ? load_scalar(a.query, row * a.q_stride + 8 * j + i, a.query_dtype) : 0.0f;
    int seq = 0, t = 0;
    const bool stands = exists && row_stands(a.rows, row, seq, t, a.status, tid == 0 && rank_in_cluster == 0);
    if (static_cast<int>(threadIdx.x) < 4 * a.buckets) bias[threadIdx.x] = parameter;
    if (threadIdx.x >= kBrThreads - 4) soft_of[threadIdx.x - (kBrThreads - 4)] = soft_plus(parameter);
    if (tid == 0) {
        found_of[own_row] = 0;
        slack_of[own_row] = 0;
        threshold_of[own_row] = kNegInf;
    }
    if (kRowWarps > 1 && parts > 1)
        for (int k = tid; k < a.top; k += kRowThreads) {
            best_value[k] = -INFINITY;
            best_index[k] = -1;
        }
    __syncthreads();
    if (!exists) return;                                 // whole warps, and with one row a CTA never
    if (rank_in_cluster == 0)
        for (int k = tid; k < a.top; k += kRowThreads) {
            a.out_index[static_cast<int64_t>(row) * a.top + k] = -1;
            a.out_score[static_cast<int64_t>(row) * a.top + k] = kNegInf;
        }
    if (!stands) return;                                 // all CTAs of a cluster alike
    const int start = max(t - a.window + 1, 0);
    int all_able = a.strict ? min(start / a.block_size, (t + 1) / a.block_size) : (t + 1) / a.block_size;
    all_able = min(all_able, a.n_blocks);
    if (all_able == 0) return;
    // this CTA's share of the blocks: [skip, skip + able)
    const int share = (all_able + parts - 1) / parts, skip = min(rank_in_cluster * share, all_able);
    const int able = min(share, all_able - skip);

    const double soft = soft_of[head];
    const float soft32 = static_cast<float>(soft);
    float norm = soft32 <= kSteep ? kLeastNorm : INFINITY;           // of the query's head, squared
#pragma unroll
    for (int i = 0; i < 8; ++i) norm = fmaf(q[i], q[i], norm);
    norm += __shfl_xor_sync(0xffffffffu, norm, 1);

    double* exact = row_memory + static_cast<size_t>(own_row) * (5 * a.part_blocks);
    float* approx = reinterpret_cast<float*>(exact + 4 * a.part_blocks);
    int* list = reinterpret_cast<int*>(approx + a.part_blocks);
    const T* means = static_cast<const T*>(a.mean) + (static_cast<int64_t>(seq) * a.n_blocks + skip) * 64 + 8 * j;
    const T* spreads = static_cast<const T*>(a.stdv) + (static_cast<int64_t>(seq) * a.n_blocks + skip) * 64 + 8 * j;

    auto bucket_of = [&](int n) {
        const int away = max(t - ((skip + n + 1) * a.block_size - 1), 0);
        return min(31 - __clz(away + 1), a.buckets - 1);
    };

    int found;
    const bool all = able <= 4 * kRowWarps;              // as few as one pass of exact scores takes: no choice before it
    if (all) {
        for (int n = tid; n < able; n += kRowThreads) list[n] = n;
        found = able;
        row_sync();
    } else {
        float most = 0.0f;
        for (int first = row_warp * 4; first < able; first += kAhead * 4 * kRowWarps) {
            RawStats<T> mean[kAhead], spreadv[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int n = min(first + u * 4 * kRowWarps + sub, able - 1);
                mean[u].load(means + static_cast<int64_t>(n) * 64);
                spreadv[u].load(spreads + static_cast<int64_t>(n) * 64);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int n = first + u * 4 * kRowWarps + sub;
                const bool live = n < able;
                float m[8], s[8];
                mean[u].widen(m);
                spreadv[u].widen(s);
                // magnitudes by Cauchy's inequality: |q . m| summed over magnitudes is at most |q| |m|
                float near = 0.0f, near_norm = kLeastNorm, spread = 0.0f, spread_norm = kLeastNorm;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    near = fmaf(q[i], m[i], near);
                    near_norm = fmaf(m[i], m[i], near_norm);
                    spread = fmaf(fabsf(q[i]), s[i], spread);
                    spread_norm = fmaf(s[i], s[i], spread_norm);
                }
                near += __shfl_xor_sync(0xffffffffu, near, 1);
                spread += __shfl_xor_sync(0xffffffffu, spread, 1);
                near_norm += __shfl_xor_sync(0xffffffffu, near_norm, 1);
                spread_norm += __shfl_xor_sync(0xffffffffu, spread_norm, 1);
                const float b = live ? bias[head * a.buckets + bucket_of(n)] : 0.0f;
                const float score = fmaf(soft32, spread, near) * 0.25f + b;
                const float size = 0.2501f * (fast_sqrt(norm * near_norm) + soft32 * fast_sqrt(norm * spread_norm)) +
                                   (fabsf(b) < 3.0e38f ? fabsf(b) : 0.0f);      // an infinite bias leaves no rounding error
                float top = fmaxf(score, __shfl_xor_sync(0xffffffffu, score, 2));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                float part = __expf(score - top);
                part += __shfl_xor_sync(0xffffffffu, part, 2);
                part += __shfl_xor_sync(0xffffffffu, part, 4);
                const float value = top + __logf(part);
                // what is not finite is told apart in 64 bits: NaN here stays in the choice
                const bool sound = fabsf(value) < 3.0e38f && size < 3.0e38f;
                const bool heads_sound = (__ballot_sync(0xffffffffu, sound) >> (lane & 24) & 255u) == 255u;
                if (live && heads_sound) most = fmaxf(most, size);
                if (live && j == 0) approx[n] = heads_sound ? value : __int_as_float(0x7fc00000);
            }
        }
        const unsigned widest = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
        if (lane == 0) atomicMax(&slack_of[own_row], widest);
        row_sync();
        const float slack = slack_of_size(__uint_as_float(slack_of[own_row]));
        // a threshold that TOP blocks reach: the TOP-th largest of the largest of 2 TOP or more groups of blocks
        if (a.top <= kRowThreads && a.top < able) {
            int groups = kRowThreads, of = 1;            // of consecutive threads share a group, every groups-th block
            while (of < 32 && groups >= 8 * a.top && groups > 32) {
                of <<= 1;
                groups >>= 1;
            }
            float best = kNegInf;
            for (int n = tid / of + (tid & (of - 1)) * groups; n < able; n += kRowThreads) best = fmaxf(best, approx[n]);
            for (int d = 1; d < of; d <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, d));
            float* bests = lane_best + own_row * kRowThreads;
            if ((tid & (of - 1)) == 0) bests[tid / of] = best;
            row_sync();
            if (tid < groups) {
                best = bests[tid];
                int before = 0;
                const float4* four = reinterpret_cast<const float4*>(bests);
#pragma unroll 8
                for (int i = 0; i < groups / 4; ++i) {
                    const float4 o = four[i];
                    before += (o.x > best || (o.x == best && 4 * i < tid)) + (o.y > best || (o.y == best && 4 * i + 1 < tid)) +
                              (o.z > best || (o.z == best && 4 * i + 2 < tid)) + (o.w > best || (o.w == best && 4 * i + 3 < tid));
                }
                if (before == a.top - 1) threshold_of[own_row] = best;
            }
            row_sync();
        }
        const float least = threshold_of[own_row] - slack;
        for (int n = tid; n < able; n += kRowThreads)
            if (!(approx[n] < least)) list[atomicAdd(&found_of[own_row], 1)] = n;
        row_sync();
        found = found_of[own_row];
    }

    // products by eight lanes a candidate, then exponentials and logarithms by a lane for each
    for (int base = row_warp * 4; base < found; base += 4 * kRowWarps) {
        const int c = base + sub;
        const int n = list[min(c, found - 1)];
        const double value = exact_head(means + static_cast<int64_t>(n) * 64, spreads + static_cast<int64_t>(n) * 64, q, soft,
                                        static_cast<double>(bias[head * a.buckets + bucket_of(n)]));
        if ((j & 1) == 0 && c < found) exact[4 * c + head] = value;
    }
    row_sync();
    for (int c = tid; c < found; c += kRowThreads) {
        double* heads = exact + 4 * c;
        const double value = exact_join(heads[0], heads[1], heads[2], heads[3]);
        heads[0] = value;
        reinterpret_cast<long long*>(heads)[1] = order_key(value);
    }
    row_sync();
    // a candidate's rank is the number of better ones, counted by eight lanes
    const long long* keys = reinterpret_cast<const long long*>(exact) + 1;
    for (int base = row_warp * 4; base < found; base += 4 * kRowWarps) {
        const int c = min(base + sub, found - 1), n = list[c];
        const long long mine = keys[4 * c];
        int rank = 0;
        for (int o = j; o < found; o += 8) {
            const long long other = keys[4 * o];
            rank += other > mine || (other == mine && list[o] < n);
        }
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        rank += __shfl_xor_sync(0xffffffffu, rank, 4);
        const double value = exact[4 * c];
        if (j != 0 || base + sub >= found || rank >= a.top || !(value > -INFINITY)) continue;
        if (kRowWarps > 1 && parts > 1) {
            best_value[rank] = value;
            best_index[rank] = skip + n;
        } else {
            a.out_index[static_cast<int64_t>(row) * a.top + rank] = n;
            a.out_score[static_cast<int64_t>(row) * a.top + rank] = static_cast<float>(value);
        }
    }
    if constexpr (kRowWarps > 1) {
        if (parts == 1) return;
        cluster_barrier();
        if (rank_in_cluster == 0) {
            // every CTA's list is sorted: a candidate's rank is its place in its own and what is better in the others'.  The
            // lists are brought here first (part_blocks is at least 4 TOP, so the scores' memory holds them)
            double* value_of = exact;
            int* index_of = reinterpret_cast<int*>(exact + parts * a.top);
            for (int c = tid; c < parts * a.top; c += kRowThreads) {
                const int from = c / a.top, k = c - from * a.top;
                value_of[c] = load_cluster_double(smem_u32(best_value + k), from);
                index_of[c] = load_cluster_int(smem_u32(best_index + k), from);
            }
            __syncthreads();
            for (int c = tid; c < parts * a.top; c += kRowThreads) {
                const int from = c / a.top, k = c - from * a.top;
                const double mine = value_of[c];
                if (!(mine > -INFINITY)) continue;
                int rank = k;
                for (int o = 0; o < parts; ++o) {
                    if (o == from) continue;
                    int low = 0, high = a.top;           // how many of list o come before: the lower part's ties do
                    while (low < high) {
                        const int mid = (low + high) >> 1;
                        const double other = value_of[o * a.top + mid];
                        if (other > mine || (other == mine && o < from)) low = mid + 1;
                        else high = mid;
                    }
                    rank += low;
                }
                if (rank >= a.top) continue;
                a.out_index[static_cast<int64_t>(row) * a.top + rank] = index_of[c];
                a.out_score[static_cast<int64_t>(row) * a.top + rank] = static_cast<float>(mine);
            }
        }
        cluster_barrier();                               // the lists stay until they have been read
    }
}

// Whole sequences with queries and statistics of one type.  A warp takes 16 consecutive positions: a head's products
// with eight blocks are one warp-level tensor instruction for the means and one for the spreads (a head is 16 wide), four
// scores a lane come out of sixteen instructions' worth of operands in place of 26 instructions a score.  Products of 16-bit
// values are exact, but how the tensor cores round their sums is not documented: 2^-17 of the magnitudes is allowed for each
// score, eight times the largest error that 16 truncated additions of 24 bits could make.  Single precision is cut to TF32
// for this (11 bits, 2^-9 of the magnitudes for two operands), which lets in a candidate or two more.
// Two warps share 16 positions: each scores every other eight blocks for all of them, then chooses for eight of them.  Their
// candidates are scored in 64 bits together: products by eight lanes a candidate, as in the kernel above and in its order,
// exponentials and logarithms by a lane for each.  8 x 4096 positions of 64 blocks: 41 us, of which set-up 8, scores 7, choice 8,
// 64-bit products 10, logarithms 7; a warp a row in the kernel above takes 90.
constexpr int kBtWarps = 4;
constexpr int kBtThreads = 32 * kBtWarps;
constexpr int kBtRows = 8 * kBtWarps;       // positions of a CTA
constexpr int kBtChunk = 64;                // blocks staged at a time
template <typename T> struct RouteTile {
    static constexpr int kRowBytes = 64 * sizeof(T) + 16;    // of a staged block: odd multiple of 16 bytes
    static constexpr int kStaged = 2 * kBtChunk * kRowBytes;
    static constexpr int kPieces = 64 * sizeof(T) / 16;
    static constexpr int kSteps = sizeof(T) == 4 ? 2 : 1;    // products of a head: 8 or 16 components at a time
    // twice what a score may be off by, of its magnitudes: 2 x 2^-17, or with operands cut to TF32 2 x 2^-9 and a little
    static constexpr float kSlack = sizeof(T) == 4 ? 0.0041f : 1.52587890625e-5f;
};

// Four heads' products of 16 rows and 8 blocks.
__device__ __forceinline__ void mma1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

inline int tile_candidates(int n_blocks) { return n_blocks < 64 ? 64 : (n_blocks + 31) / 32 * 32; }
inline int tile_stride(int n_blocks) { return (n_blocks + 7) / 8 * 8 + 4; }        // floats of a row of scores
// Bytes of a warp: scores of 8 of its rows, head scores and (row, block) of the candidates.
inline int tile_warp_bytes(int n_blocks) { return 8 * tile_stride(n_blocks) * 4 + tile_candidates(n_blocks) * 36; }

template <typename T>
__global__ void __launch_bounds__(kBtThreads, sizeof(T) == 4 ? 4 : 5) block_route_tile_kernel(const RouteArgs a, int stride, int room) {
    using R = RouteTile<T>;
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ float4 bias[kBrMaxBuckets];               // of the four heads
    __shared__ double soft_of[4];
    __shared__ float widest_of[4];                       // the largest finite bias; an infinite one leaves no rounding error
    __shared__ unsigned mean_norm[4], spread_norm[4];    // squared, of the sequence's blocks
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seq = blockIdx.y, t0 = blockIdx.x * kBtRows + 16 * (warp >> 1);        // of the two warps' 16 rows
    const int own = 8 * (warp & 1);                      // the first row that this warp chooses for
    griddep_sync();
    for (int i = threadIdx.x; i < a.buckets; i += kBtThreads)
        bias[i] = make_float4(load_scalar(a.bias, i, a.param_dtype), load_scalar(a.bias, a.buckets + i, a.param_dtype),
                              load_scalar(a.bias, 2 * a.buckets + i, a.param_dtype), load_scalar(a.bias, 3 * a.buckets + i, a.param_dtype));
    if (threadIdx.x < 4) {
        soft_of[threadIdx.x] = soft_plus(load_scalar(a.gamma, threadIdx.x, a.param_dtype));
        mean_norm[threadIdx.x] = spread_norm[threadIdx.x] = __float_as_uint(kLeastNorm);
        float widest = 0.0f;
        for (int k = 0; k < a.buckets; ++k) {
            const float b = fabsf(load_scalar(a.bias, threadIdx.x * a.buckets + k, a.param_dtype));
            if (b < 3.0e38f) widest = fmaxf(widest, b);
        }
        widest_of[threadIdx.x] = widest;
    }
    __syncthreads();
    const int length = a.rows.query_length;
    const int64_t first_row = static_cast<int64_t>(seq) * length;
    auto able_at = [&](int t) {
        const int start = max(t - a.window + 1, 0);
        const int n = a.strict ? min(start / a.block_size, (t + 1) / a.block_size) : (t + 1) / a.block_size;
        return min(n, a.n_blocks);
    };
    const int cta_able = able_at(min((static_cast<int>(blockIdx.x) + 1) * kBtRows, length) - 1);
    double* heads_of = reinterpret_cast<double*>(memory + R::kStaged) + warp * 4 * room;                      // [room][4]
    int* list = reinterpret_cast<int*>(memory + R::kStaged + kBtWarps * 32 * room) + warp * room;             // [room]
    float* scores = reinterpret_cast<float*>(memory + R::kStaged + kBtWarps * 36 * room) + (warp >> 1) * 16 * stride;      // [16][stride]
    for (int r = own; r < own + 8; ++r) {
        if (t0 + r >= length) break;
        const int64_t row = first_row + t0 + r;
        for (int k = lane; k < a.top; k += 32) {
            a.out_index[row * a.top + k] = -1;
            a.out_score[row * a.top + k] = kNegInf;
        }
    }

    // the queries as operands: rows lane / 4 and lane / 4 + 8 of the warp's 16, a head's components 2 (lane & 3) + {0, 1, 8, 9},
    // in single precision (lane & 3) + {0, 4, 8, 12}
    uint32_t q[4][R::kSteps][4];
    float norms[2][4];
    int t_of[2], able_of[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        t_of[i] = t0 + (lane >> 2) + 8 * i;
        const bool live = t_of[i] < length;
        able_of[i] = live ? able_at(t_of[i]) : 0;
        const T* row = static_cast<const T*>(a.query) + (first_row + (live ? t_of[i] : 0)) * a.q_stride;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            float n = kLeastNorm;
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float x = __ldg(row + 16 * h + 4 * k + (lane & 3));
                    q[h][k >> 1][2 * (k & 1) + i] = __float_as_uint(x);
                    n = fmaf(x, x, n);
                }
            } else {
                q[h][0][i] = load_pair(row + 16 * h + 2 * (lane & 3));
                q[h][0][2 + i] = load_pair(row + 16 * h + 8 + 2 * (lane & 3));
                const float2 x = unpack2<T>(q[h][0][i]), y = unpack2<T>(q[h][0][2 + i]);
                n += x.x * x.x + x.y * x.y + y.x * y.x + y.y * y.y;
            }
            n += __shfl_xor_sync(0xffffffffu, n, 1);
            n += __shfl_xor_sync(0xffffffffu, n, 2);
            norms[i][h] = n;
        }
    }
    const float soft[4] = {static_cast<float>(soft_of[0]), static_cast<float>(soft_of[1]), static_cast<float>(soft_of[2]), static_cast<float>(soft_of[3])};
    const T* means = static_cast<const T*>(a.mean) + static_cast<int64_t>(seq) * a.n_blocks * 64;
    const T* spreads = static_cast<const T*>(a.stdv) + static_cast<int64_t>(seq) * a.n_blocks * 64;
    const uint32_t staged = smem_u32(memory);
    for (int base = 0; base < cta_able; base += kBtChunk) {
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * kBtChunk * R::kPieces; i += kBtThreads) {
            const int which = i >= kBtChunk * R::kPieces, n = (i / R::kPieces) & (kBtChunk - 1), piece = i & (R::kPieces - 1);
            const bool live = base + n < cta_able;
            cp_async16_or_zero(staged + (which * kBtChunk + n) * R::kRowBytes + 16 * piece,
                               (which ? spreads : means) + static_cast<int64_t>(live ? base + n : 0) * 64 + 16 / sizeof(T) * piece, live);
        }
        cp_async_commit();
        cp_async_wait_all();
        __syncthreads();
        // the largest norms of the heads' means and spreads: a thread per (block, statistic); NaN is left out, its scores are
        // NaN as well
        if (threadIdx.x < 2 * kBtChunk) {
            const int which = threadIdx.x >= kBtChunk, n = threadIdx.x & (kBtChunk - 1);
            const unsigned char* row = memory + (which * kBtChunk + n) * R::kRowBytes;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float f[8];
                    load_stats(reinterpret_cast<const T*>(row) + 16 * h + 8 * c, f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum = fmaf(f[i], f[i], sum);
                }
                const unsigned key = sum == sum ? __float_as_uint(sum) : 0u;
                const unsigned most = __reduce_max_sync(0xffffffffu, key);
                if (lane == 0) atomicMax(which ? &spread_norm[h] : &mean_norm[h], most);
            }
        }
        const int chunk = min(kBtChunk, cta_able - base);
        for (int n0 = 8 * (warp & 1); n0 < chunk; n0 += 16) {
            float near[4][4], spread[4][4];
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) near[h][i] = spread[h][i] = 0.0f;
            if constexpr (sizeof(T) == 4) {
                const float* rows = reinterpret_cast<const float*>(memory + (n0 + (lane >> 2)) * R::kRowBytes) + (lane & 3);
                const float* spread_rows = rows + kBtChunk * R::kRowBytes / 4;
#pragma unroll
                for (int h = 0; h < 4; ++h)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t magnitude[4] = {q[h][k][0] & 0x7fffffffu, q[h][k][1] & 0x7fffffffu, q[h][k][2] & 0x7fffffffu, q[h][k][3] & 0x7fffffffu};
                        const int c = 16 * h + 8 * k;
                        mma1688(near[h], q[h][k], __float_as_uint(rows[c]), __float_as_uint(rows[c + 4]));
                        mma1688(spread[h], magnitude, __float_as_uint(spread_rows[c]), __float_as_uint(spread_rows[c + 4]));
                    }
            } else {
                // four 8 x 8 operands: blocks n0 .. n0 + 7, components 0-7, 8-15 (a head), 16-23, 24-31 (the next)
                const uint32_t at = staged + (n0 + (lane & 7)) * R::kRowBytes + 16 * (lane >> 3);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t m[4], s[4];
                    ldmatrix4(m, at + 64 * half);
                    ldmatrix4(s, at + 64 * half + kBtChunk * R::kRowBytes);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int h = 2 * half + x;
                        const uint32_t magnitude[4] = {q[h][0][0] & 0x7fff7fffu, q[h][0][1] & 0x7fff7fffu, q[h][0][2] & 0x7fff7fffu, q[h][0][3] & 0x7fff7fffu};
                        mma16816<T>(near[h], q[h][0], m[2 * x], m[2 * x + 1]);
                        mma16816<T>(spread[h], magnitude, s[2 * x], s[2 * x + 1]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = base + n0 + 2 * (lane & 3) + (i & 1), t = t_of[i >> 1];
                const int away = max(t - ((n + 1) * a.block_size - 1), 0);
                const float4 b = bias[min(31 - __clz(away + 1), a.buckets - 1)];
                const float s0 = fmaf(0.25f, fmaf(soft[0], spread[0][i], near[0][i]), b.x), s1 = fmaf(0.25f, fmaf(soft[1], spread[1][i], near[1][i]), b.y);
                const float s2 = fmaf(0.25f, fmaf(soft[2], spread[2][i], near[2][i]), b.z), s3 = fmaf(0.25f, fmaf(soft[3], spread[3][i], near[3][i]), b.w);
                const float top = fmaxf(fmaxf(s0, s1), fmaxf(s2, s3));
                const float value = top + __logf((__expf(s0 - top) + __expf(s1 - top)) + (__expf(s2 - top) + __expf(s3 - top)));
                if (n < able_of[i >> 1])
                    scores[((lane >> 2) + 8 * (i >> 1)) * stride + n] = fabsf(value) < 3.0e38f ? value : __int_as_float(0x7fc00000);
            }
        }
    }
    __syncthreads();
    // a row's slack: magnitudes by Cauchy's inequality from the norms; squares that overflow make everything a candidate
    bool wild = false;
#pragma unroll
    for (int h = 0; h < 4; ++h)
        wild = wild || !(__uint_as_float(mean_norm[h]) < 3.0e38f) || !(__uint_as_float(spread_norm[h]) < 3.0e38f) || !(soft[h] <= kSteep);
    float slack[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float size = 0.0f;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            wild = wild || !(norms[i][h] < 3.0e38f);
            size = fmaxf(size, 0.2501f * (sqrtf(norms[i][h]) * sqrtf(__uint_as_float(mean_norm[h])) +
                                          soft[h] * sqrtf(norms[i][h]) * sqrtf(__uint_as_float(spread_norm[h]))) + widest_of[h]);
        }
        slack[i] = wild ? -kNegInf : fmaf(size, R::kSlack, 7.62939453125e-6f);
    }

    // the candidates of as many rows as their list holds, scored in 64 bits and ranked
    int filled = 0;
    auto flush = [&] {
        __syncwarp();
        const int j = lane & 7, sub = lane >> 3, head = j >> 1;
#pragma unroll 2
        for (int c0 = 0; c0 < filled; c0 += 4) {
            const int c = min(c0 + sub, filled - 1), r = list[c] >> 24, n = list[c] & 0xffffff;
            float f[8];
            const T* query = static_cast<const T*>(a.query) + (first_row + t0 + r) * a.q_stride + 8 * j;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                if constexpr (sizeof(T) == 4) {
                    f[i] = __ldg(query + i);
                    f[i + 1] = __ldg(query + i + 1);
                } else {
                    const float2 x = unpack2<T>(load_pair(query + i));
                    f[i] = x.x;
                    f[i + 1] = x.y;
                }
            }
            const int away = max(t0 + r - ((n + 1) * a.block_size - 1), 0);
            const float b = reinterpret_cast<const float*>(&bias[min(31 - __clz(away + 1), a.buckets - 1)])[head];
            // one chunk of blocks is still staged
            const T* mean_row = cta_able <= kBtChunk ? reinterpret_cast<const T*>(memory + n * R::kRowBytes) : means + static_cast<int64_t>(n) * 64;
            const T* spread_row = cta_able <= kBtChunk ? reinterpret_cast<const T*>(memory + (kBtChunk + n) * R::kRowBytes)
                                                       : spreads + static_cast<int64_t>(n) * 64;
            const double value = exact_head(mean_row + 8 * j, spread_row + 8 * j, f, soft_of[head], static_cast<double>(b));
            if ((j & 1) == 0 && c0 + sub < filled) heads_of[4 * c + head] = value;
        }
        __syncwarp();
        for (int c = lane; c < filled; c += 32) {
            const double value = exact_join(heads_of[4 * c], heads_of[4 * c + 1], heads_of[4 * c + 2], heads_of[4 * c + 3]);
            heads_of[4 * c] = value;
            reinterpret_cast<long long*>(heads_of)[4 * c + 1] = order_key(value);
        }
        __syncwarp();
        for (int c = lane; c < filled; c += 32) {
            const double value = heads_of[4 * c];
            const int entry = list[c], r = entry >> 24, n = entry & 0xffffff;
            if (!(value > -INFINITY)) continue;
            const long long* keys = reinterpret_cast<const long long*>(heads_of) + 1;
            const long long mine = keys[4 * c];
            int rank = 0;                                // the candidates of a row lie together, in ascending order
            for (int o = c - 1; o >= 0 && list[o] >> 24 == r; --o) rank += keys[4 * o] >= mine;
            for (int o = c + 1; o < filled && list[o] >> 24 == r; ++o) rank += keys[4 * o] > mine;
            if (rank >= a.top) continue;
            const int64_t row = first_row + t0 + r;
            a.out_index[row * a.top + rank] = n;
            a.out_score[row * a.top + rank] = static_cast<float>(value);
        }
        __syncwarp();
        filled = 0;
    };
    // several rows at once, 8, 16 or 32 lanes each: twice as many as places, so that the TOP-th largest of the lanes' own largest
    // lets few others in
    const int lanes = 2 * a.top <= 8 ? 8 : 2 * a.top <= 16 ? 16 : 32;
    const int my_lane = lane & (lanes - 1), first_lane = lane & ~(lanes - 1);
    const unsigned my_lanes = (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1) << first_lane;
    for (int r0 = own; r0 < own + 8 && t0 + r0 < length; r0 += 32 / lanes) {
        const int r = r0 + lane / lanes;
        const int able = t0 + r < length ? able_at(t0 + r) : 0;
        const float* row = scores + r * stride;
        const float row_slack = __shfl_sync(0xffffffffu, (r0 & 8) ? slack[1] : slack[0], (r & 7) << 2);
        // eight scores a lane stay in registers; where there are more they are read again
        constexpr int kHeld = 8;
        const int most = __reduce_max_sync(0xffffffffu, able);
        const bool held = most <= kHeld * lanes;
        float value[kHeld];
        float best = kNegInf;
        if (held) {
#pragma unroll
            for (int k = 0; k < kHeld; ++k) {
                const int n = k * lanes + my_lane;
                value[k] = n < able ? row[n] : kNegInf;
                best = fmaxf(best, value[k]);
            }
        } else {
            for (int n = my_lane; n < able; n += lanes) best = fmaxf(best, row[n]);
        }
        float least = kNegInf;
        int before = 0;
        for (int d = 1; d < lanes; ++d) {
            const float other = __shfl_xor_sync(0xffffffffu, best, d);
            before += other > best || (other == best && (my_lane ^ d) < my_lane);
        }
        const unsigned which = __ballot_sync(0xffffffffu, before == a.top - 1) & my_lanes;
        const float reached = __shfl_sync(0xffffffffu, best, __ffs(which) - 1);
        if (a.top < able) least = reached - row_slack;
        auto candidate = [&](int n) { return n < able && !(row[n] < least); };
        int here = 0;
        unsigned held_votes = 0;                         // bit k: this lane's k-th score is a candidate
        if (held) {
#pragma unroll
            for (int k = 0; k < kHeld; ++k) {
                const bool take = k * lanes + my_lane < able && !(value[k] < least);
                here += __popc(__ballot_sync(0xffffffffu, take) & my_lanes);
                held_votes |= static_cast<unsigned>(take) << k;
            }
        } else {
            for (int n0 = 0; n0 < most; n0 += lanes) here += __popc(__ballot_sync(0xffffffffu, candidate(n0 + my_lane)) & my_lanes);
        }
        // the rows' places in the list, one after another; as many rows as it holds
        int from = 0, all = 0;
        for (int l = 0; l < 32; l += lanes) {
            const int other = __shfl_sync(0xffffffffu, here, l);
            if (l < first_lane) from += other;
            all += other;
        }
        if (filled + all > room && filled > 0) flush();
        const bool together = all <= room;
        for (int l = 0; l < 32; l += lanes) {            // one pass where the list holds them all, else a pass for each row
            const bool mine_now = together ? true : first_lane == l;
            int at = filled + (together ? from : 0);
            for (int n0 = 0, k = 0; n0 < most; n0 += lanes, ++k) {
                const int n = n0 + my_lane;
                const bool take = mine_now && (held ? (held_votes >> k & 1u) != 0u : candidate(n));
                const unsigned vote = __ballot_sync(0xffffffffu, take) & my_lanes;
                if (take) list[at + __popc(vote & ((1u << lane) - 1))] = r << 24 | n;
                at += __popc(vote);
            }
            if (together) {
                filled += all;
                break;
            }
            filled = __shfl_sync(0xffffffffu, here, l);
            flush();
        }
    }
    flush();
}

template <typename T>
int launch_route(RouteArgs& a, void* stream) {
    const int64_t rows = a.rows.n_rows;
    // A warp's lanes tell the candidates of up to 16 places apart (the TOP-th largest of 32 groups' largest); more places take
    // the 256 groups of a whole CTA.  Whole sequences of many rows go to the tiles, whose chain of steps is long (64 rows 12 us
    // against 4.5, 4096 rows of 64 blocks 31 against 21) but whose work is half (32768 rows 41 us against 90).
    const int mine = sizeof(T) == 4 ? RLM_F32 : std::is_same<T, __nv_bfloat16>::value ? RLM_BF16 : RLM_F16;
    const int tile_bytes = RouteTile<T>::kStaged + kBtWarps * tile_warp_bytes(a.n_blocks);
    const bool pairs = sizeof(T) == 4 || ((reinterpret_cast<uintptr_t>(a.query) & 3u) == 0 && a.q_stride % 2 == 0);
    if (!a.rows.position && !a.rows.row_position && rows > kBtLeastRows && a.top <= kBrWarpTop && a.query_dtype == mine && pairs &&
        tile_bytes <= kSmemDynamicLimit - 4096 && a.rows.n_seq <= 65535) {
        if (int rc = allow_large_smem(reinterpret_cast<const void*>(&block_route_tile_kernel<T>), kSmemDynamicLimit)) return rc;
        launch_kernel(block_route_tile_kernel<T>, dim3((a.rows.query_length + kBtRows - 1) / kBtRows, a.rows.n_seq), dim3(kBtThreads),
                      tile_bytes, stream, a, tile_stride(a.n_blocks), tile_candidates(a.n_blocks));
        count_launch();
        return check_launch("block_route_tile_kernel");
    }
    a.parts = 1;
    a.part_blocks = a.n_blocks;
    const int row_bytes = kBrBytesPerBlock * a.n_blocks;
    // A warp a row where there are many rows and few blocks: 1000 rows of 64 blocks 12 us against 16 with a CTA a row, of 128 blocks
    // 17.9 against 16.5; 3000 rows of 128 blocks 28 against 42, of 256 blocks 60 against 56; 400 rows of 8 blocks 6.4 against 4.9.
    if (rows > 512 && 16 * static_cast<int64_t>(a.n_blocks) <= rows && a.n_blocks <= 256 && a.top <= kBrWarpTop) {
        if (int rc = allow_large_smem(reinterpret_cast<const void*>(&block_route_kernel<T, 1, false>), kSmemDynamicLimit)) return rc;
        launch_kernel(block_route_kernel<T, 1, false>, dim3(static_cast<unsigned>((rows + kBrWarps - 1) / kBrWarps)), dim3(kBrThreads),
                      static_cast<size_t>(row_bytes) * kBrWarps, stream, a);
    } else {
        // a row's blocks over a cluster, while the rows leave SMs idle and every CTA keeps a few passes of work, or where
        // their scores would not fit one CTA's shared memory
        while (a.parts < kBrMaxParts && ((rows * a.parts * 2 <= 2 * sm_count() && a.n_blocks / (2 * a.parts) >= 128 &&
                                          a.n_blocks / (2 * a.parts) >= 4 * a.top) ||
                                         kBrBytesPerBlock * (a.n_blocks / a.parts + 1) > kBrMemory))
            a.parts *= 2;
        if (rows * a.parts > 0x7fffffff) {
            set_error("block_route: too many rows of so many blocks for one launch");
            return RLM_ERR_SHAPE;
        }
        a.part_blocks = (a.n_blocks + a.parts - 1) / a.parts;
        const int bytes = kBrBytesPerBlock * a.part_blocks;
        const bool deep = a.n_blocks >= 2048 || (a.part_blocks >= 512 && rows * a.parts <= 2 * sm_count());
        const auto kernel = deep ? block_route_kernel<T, kBrWarps, true> : block_route_kernel<T, kBrWarps, false>;
        if (int rc = allow_large_smem(reinterpret_cast<const void*>(kernel), kSmemDynamicLimit)) return rc;
        if (a.parts > 1)
            launch_kernel_cluster(kernel, dim3(static_cast<unsigned>(rows * a.parts)), dim3(kBrThreads), static_cast<unsigned>(a.parts),
                                  bytes, stream, a);
        else
            launch_kernel(kernel, dim3(static_cast<unsigned>(rows)), dim3(kBrThreads), bytes, stream, a);
    }
    count_launch();
    return check_launch("block_route_kernel");
}

}  // namespace
}  // namespace rlm

extern "C" int rlm_block_route(const void* router_query, int64_t query_row_stride, const void* block_mean, const void* block_std,
                               const void* gamma, const void* bias, const int64_t* position, const int32_t* row_batch,
                               const int32_t* row_position, int32_t* out_index, float* out_score, int n_rows, int n_seq,
                               int query_length, int n_blocks, int block_size, int buckets, int local_window, int top_blocks,
                               int strict_valid, int query_dtype, int stats_dtype, int param_dtype, int32_t* status, void* stream) {
    using namespace rlm;
    RouteArgs a{};
    a.rows = Rows{position, row_batch, row_position, n_rows, n_seq, query_length, 0x7fffffff};
    if (n_rows > 0 && (!router_query || !gamma || !bias || (top_blocks > 0 && (!out_index || !out_score)) ||
                       (n_blocks > 0 && (!block_mean || !block_std)))) {
        set_error("block_route: NULL argument");
        return RLM_ERR_NULL;
    }
    if (int rc = check_rows("block_route: row_batch and row_position come together",
                            "block_route: rows do not fit the sequences of the block statistics", a.rows))
        return rc;
    if (!valid_dtype(query_dtype) || !valid_dtype(stats_dtype) || !valid_dtype(param_dtype)) {
        set_error("block_route: unknown dtype");
        return RLM_ERR_DTYPE;
    }
    if (n_blocks < 0 || block_size < 1 || buckets < 1 || buckets > kBrMaxBuckets || local_window < 0 || top_blocks < 0 ||
        top_blocks > kBrMaxTop || static_cast<int64_t>(n_blocks + 1) * block_size > 0x7fffffff) {
        set_error("block_route: needs block_size >= 1, 1 to 32 buckets, local_window >= 0, 0 to 128 blocks a row");
        return RLM_ERR_SHAPE;
    }
    if (!aligned16(block_mean) || !aligned16(block_std)) {
        set_error("block_route: block statistics must be 16-byte aligned");
        return RLM_ERR_ALIGN;
    }
    if (static_cast<int64_t>(kBrBytesPerBlock) * (n_blocks / kBrMaxParts + 1) > kBrMemory) {
        set_error("block_route: too many blocks a sequence for the scores of a row in shared memory");
        return RLM_ERR_SMEM;
    }
    if (n_rows == 0 || top_blocks == 0) return RLM_OK;
    a.query = router_query;
    a.mean = block_mean;
    a.stdv = block_std;
    a.gamma = gamma;
    a.bias = bias;
    a.out_index = out_index;
    a.out_score = out_score;
    a.status = status;
    a.q_stride = query_row_stride;
    a.n_blocks = n_blocks;
    a.block_size = block_size;
    a.buckets = buckets;
    a.window = local_window;
    a.top = top_blocks;
    a.strict = strict_valid;
    a.query_dtype = query_dtype;
    a.param_dtype = param_dtype;
    if (stats_dtype == RLM_F32) return launch_route<float>(a, stream);
    if (stats_dtype == RLM_BF16) return launch_route<__nv_bfloat16>(a, stream);
    return launch_route<__half>(a, stream);
}
