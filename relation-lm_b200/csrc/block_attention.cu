// Attention of each query row over the blocks that a router chose for it and over its local window.
//
//     ls = max(0, t - L + 1),   keys = [ls, t]  and, for each distinct n >= 0 among the row's indices, [n BS, min((n + 1) BS, ls))
//     out = sum_k p_k v_k / sum_k p_k,   p_k = exp(scale q . k_k - m),   lse = m + log sum_k p_k
//
// A row that sees no key is zero, its lse -inf.
//
// block_attention_rows_kernel (16-bit types): the decode and per-row forms.  A CTA takes a row, a key head and up to 16 of
// its query heads, the height of the warp-level tensor instruction; its warps take 16 keys at a time, each through its own
// shared-memory ring (cp.async, whole rows, no barrier between warps) and with its own running maximum and sum.  Few rows:
// the keys are divided over a cluster of CTAs, joined through distributed shared memory, so that a row costs one launch
// and no workspace.  Bytes bound it: every key and value row is read once for its (up to 16) query heads.  64 rows of 1536 keys,
// 32 heads over 8 of width 128: 404 MB in 69 us, 89 % of the copy peak; one row of 128 keys: 4.7 us, the chain indices, keys,
// scores, join.
//
// block_attention_f32_kernel: the same division in single precision on the CUDA cores (the tensor cores would keep 11 of
// 24 bits): eight lanes share a key, four keys a warp pass.  77 rows of 228 keys, 12 heads of width 64: 16 us for 108 MB that come
// mostly from L2.
#include "block_attention_mma.cuh"

namespace rlm {
namespace {

constexpr int kBaWarps = 4;
constexpr int kBaThreads = 32 * kBaWarps;
constexpr int kBaMaxSplit = 8;

// What a CTA works on: CTAs of a cluster side by side, then the key heads of a row, whose cache rows lie side by side.
struct CtaPlace {
    int row, kv, tile, rank;
    bool first;                        // of the row's CTAs
    __device__ __forceinline__ explicit CtaPlace(const AttentionArgs& a) {
        const int tiles = a.kv_heads * a.head_tiles, of_row = tiles * a.splits;
        row = blockIdx.x / of_row;
        int rest = blockIdx.x - row * of_row;
        first = rest == 0;
        const int which = rest / a.splits;
        rank = rest - which * a.splits;
        kv = which / a.head_tiles;
        tile = which - kv * a.head_tiles;
    }
};

// The blocks of a row that hold keys before its window, each once: positions of their first rows.  By the first warp of a
// CTA; the count is returned to all threads through `count`, behind the caller's barrier.
// `first`: this lane's of the first 32 indices, loaded ahead.
__device__ __forceinline__ int first_index(const int32_t* index, int top) {
    const int lane = threadIdx.x & 31;
    return lane < top ? index[lane] : -1;
}
__device__ __forceinline__ void keep_blocks(const int32_t* index, int first, int top, int block_size, int start, int* kept, int* count) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int base = 0; base < top; base += 32) {
        const int i = base + lane;
        const int block = base == 0 ? first : i < top ? index[i] : -1;
        // a block counts at its first place in the list, and only if it begins before the window
        bool keep = block >= 0 && block < (start + block_size - 1) / block_size;
        for (int o = 0; o < base; ++o) keep = keep && index[o] != block;
        const unsigned same = __match_any_sync(0xffffffffu, block);
        keep = keep && lane == __ffs(same) - 1;
        const unsigned vote = __ballot_sync(0xffffffffu, keep);
        if (keep) kept[n + __popc(vote & ((1u << lane) - 1))] = block * block_size;
        n += __popc(vote);
    }
    if (lane == 0) *count = n;
}

// Joins the warps' partial results of a CTA and then the CTAs' of a cluster, and writes the row.  `parts`: per warp
// [kTile heads][D] sums, `part_m`, `part_l` [warps][16] maxima (of powers of two) and sums; `joined` [kTile][D], joined_m,
// joined_l [16] receive the CTA's.
template <typename T, int D, int kParts, int kTile>
__device__ __forceinline__ void join_and_write(const AttentionArgs& a, int row, int first_head, int n_heads, int rank,
                                               const float* parts, const float* part_m, const float* part_l, float* joined,
                                               float* joined_m, float* joined_l) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid < n_heads) {
        float m = kNegInf, l = 0.0f;
        for (int w = 0; w < kParts; ++w) m = fmaxf(m, part_m[w * 16 + tid]);
        for (int w = 0; w < kParts; ++w)
            if (part_l[w * 16 + tid] != 0.0f) l += part_l[w * 16 + tid] * power2(part_m[w * 16 + tid] - m);
        joined_m[tid] = m;
        joined_l[tid] = l;
    }
    __syncthreads();
    const bool alone = a.splits == 1;
    auto head_row = [&](int h) {
        return a.out + (static_cast<int64_t>(row) * a.heads + first_head + h) * (D * static_cast<int64_t>(sizeof(T)));
    };
    for (int i = tid; i < n_heads * D; i += blockDim.x) {
        const int h = i / D, c = i - h * D;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kParts; ++w)
            if (part_l[w * 16 + h] != 0.0f) sum += parts[(w * kTile + h) * D + c] * power2(part_m[w * 16 + h] - joined_m[h]);
        if (alone) store_value<T>(head_row(h), c, joined_l[h] == 0.0f ? 0.0f : sum / joined_l[h]);
        else joined[i] = sum;
    }
    if (alone) {
        if (tid < n_heads)
            a.lse[static_cast<int64_t>(row) * a.heads + first_head + tid] =
                joined_l[tid] == 0.0f ? kNegInf : (joined_m[tid] + log2f(joined_l[tid])) * kLn2;
        return;
    }
    cluster_barrier();
    const uint32_t joined_at = smem_u32(joined), m_at = smem_u32(joined_m), l_at = smem_u32(joined_l);
    for (int i = rank * blockDim.x + tid; i < n_heads * D; i += a.splits * blockDim.x) {
        const int h = i / D, c = i - h * D;
        float m[kBaMaxSplit], l[kBaMaxSplit], v[kBaMaxSplit];
        float most = kNegInf;
#pragma unroll
        for (int s = 0; s < kBaMaxSplit; ++s) {
            if (s >= a.splits) break;
            m[s] = load_cluster(m_at + 4 * h, s);
            l[s] = load_cluster(l_at + 4 * h, s);
            v[s] = load_cluster(joined_at + 4 * i, s);
            most = fmaxf(most, m[s]);
        }
        float sum = 0.0f, total = 0.0f;
#pragma unroll
        for (int s = 0; s < kBaMaxSplit; ++s) {
            if (s >= a.splits) break;
            if (l[s] != 0.0f) {
                const float w = power2(m[s] - most);
                sum += v[s] * w;
                total += l[s] * w;
            }
        }
        store_value<T>(head_row(h), c, total == 0.0f ? 0.0f : sum / total);
        if (c == 0)
            a.lse[static_cast<int64_t>(row) * a.heads + first_head + h] = total == 0.0f ? kNegInf : (most + log2f(total)) * kLn2;
    }
    cluster_barrier();                      // a CTA's shared memory stays until the others have read it
}

template <typename T, int D>
__device__ __forceinline__ void write_blank(const AttentionArgs& a, int row, int first_head, int n_heads, int rank) {
    if (rank != 0) return;
    for (int i = threadIdx.x; i < n_heads * D; i += blockDim.x)
        store_value<T>(a.out + (static_cast<int64_t>(row) * a.heads + first_head) * (D * static_cast<int64_t>(sizeof(T))), i, 0.0f);
    if (static_cast<int>(threadIdx.x) < n_heads) a.lse[static_cast<int64_t>(row) * a.heads + first_head + threadIdx.x] = kNegInf;
}

template <int D> struct RowsPlan {
    static constexpr int kStages = 3;        // four at width 64 leave room for fewer CTAs: 64 x 12 heads 38 us, three 33, two 44
    static constexpr int kRowBytes = 2 * D + 16;           // odd multiple of 16 bytes: ldmatrix without bank conflicts
    static constexpr int kStage = 2 * 16 * kRowBytes;      // 16 keys and 16 values
    static constexpr int kWarp = kStages * kStage;
    static constexpr int kQuery = 16 * kRowBytes;
    static constexpr int kParts = kBaWarps * 16 * D * 4;   // the warps' sums, then the CTA's, in the rings' place
    static_assert(kParts + 16 * D * 4 <= kBaWarps * kWarp, "the sums do not fit the rings");
    static constexpr int kTotal = kBaWarps * kWarp + kQuery;
};

template <typename T, int D>
__global__ void __launch_bounds__(kBaThreads) block_attention_rows_kernel(const AttentionArgs a) {
    using P = RowsPlan<D>;
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ int kept[kBaMaxTop];
    __shared__ int n_kept;
    __shared__ float part_m[kBaWarps * 16], part_l[kBaWarps * 16], joined_m[16], joined_l[16];

    const CtaPlace here(a);
    const int row = here.row, rank = here.rank, kv = here.kv, tile = here.tile;
    const int first_head = kv * a.group + 16 * tile;
    const int n_heads = min(16, a.group - 16 * tile);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_sync();

    // what does not depend on the row's position is requested before it is waited for
    unsigned char* query = memory + kBaWarps * P::kWarp;
    constexpr int kPieces = D / 8;                       // 16-byte pieces of a row
    for (int i = threadIdx.x; i < 16 * kPieces; i += kBaThreads) {
        const int h = i / kPieces, p = i - h * kPieces;
        const int from = min(h, n_heads - 1);            // rows of absent heads are zeros
        cp_async16_or_zero(smem_u32(query + h * P::kRowBytes + 16 * p), a.query + row * a.q_row + (first_head + from) * a.q_head + 16 * p, h < n_heads);
    }
    cp_async_commit();
    const int32_t* index = a.index + row * a.i_row + kv * a.i_head;
    const int first = first_index(index, a.top);
    int seq, t;
    if (!row_stands(a.rows, row, seq, t, a.status, threadIdx.x == 0 && here.first)) {
        write_blank<T, D>(a, row, first_head, n_heads, rank);
        cp_async_wait_all();
        return;                                          // all CTAs of the cluster return here, none waits for another
    }
    const int start = max(t - a.window + 1, 0);
    if (warp == 0) keep_blocks(index, first, a.top, a.block_size, start, kept, &n_kept);
    cp_async_wait_all();
    __syncthreads();

    // 16 keys at a time: first the kept blocks', each block from its own first row, then the window's
    const int per_block = (min(a.block_size, start) + 15) >> 4;      // a block's rows from the window on are the window's
    const int block_chunks = n_kept * per_block;
    const int chunks = block_chunks + ((t - start + 16) >> 4);
    const int step = kBaWarps * a.splits;
    const unsigned char* keys = a.key_cache + seq * a.k_seq + kv * a.k_head;
    const unsigned char* values = a.value_cache + seq * a.v_seq + kv * a.v_head;
    unsigned char* ring = memory + warp * P::kWarp;
    const uint32_t ring_at = smem_u32(ring);

    auto place = [&](int c, int& at, int& count) {
        if (c < block_chunks) {
            const int b = c / per_block, o = (c - b * per_block) << 4;
            at = kept[b] + o;
            count = min(min(a.block_size - o, 16), start - at);
        } else {
            at = start + ((c - block_chunks) << 4);
            count = min(16, t + 1 - at);
        }
    };
    auto request = [&](int c, int stage) {
        if (c < chunks) {
            int at, count;
            place(c, at, count);
            const uint32_t to = ring_at + stage * P::kStage;
#pragma unroll
            for (int i = 0; i < 16 * kPieces / 32; ++i) {
                const int item = i * 32 + lane, r = item / kPieces, p = item - r * kPieces;
                const bool live = r < count;
                const int64_t from = live ? at + r : t;  // a row that exists
                cp_async16_or_zero(to + r * P::kRowBytes + 16 * p, keys + from * a.k_row + 16 * p, live);
                cp_async16_or_zero(to + (16 + r) * P::kRowBytes + 16 * p, values + from * a.v_row + 16 * p, live);
            }
        }
        cp_async_commit();                               // an empty group past the end keeps the count
    };

    const int first_chunk = rank * kBaWarps + warp;
#pragma unroll
    for (int s = 0; s < P::kStages - 1; ++s) request(first_chunk + s * step, s);

    uint32_t q[D / 16][4];
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
        ldmatrix4(q[k], smem_u32(query + (lane & 15) * P::kRowBytes + 32 * k + 16 * (lane >> 4)));
    if (a.flip)
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) q[k][i] ^= a.flip;

    float acc[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
    float m[2] = {kNegInf, kNegInf}, l[2] = {0.0f, 0.0f};
    // ldmatrix: keys 0-7 and 8-15, each with both halves of a k step; values: keys 0-7 and 8-15 of two column groups
    const int key_row = (lane & 7) + ((lane >> 4) << 3), key_half = (lane >> 3) & 1;
    const int value_row = lane & 15, value_half = lane >> 4;

    int stage = 0;
    for (int c = first_chunk; c < chunks; c += step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(P::kStages - 2) : "memory");
        __syncwarp();
        const uint32_t at_key = ring_at + stage * P::kStage, at_value = at_key + 16 * P::kRowBytes;
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];
            ldmatrix4(b, at_key + key_row * P::kRowBytes + 32 * k + 16 * key_half);
            mma16816<T>(s[0], q[k], b[0], b[1]);
            mma16816<T>(s[1], q[k], b[2], b[3]);
        }
        int at, count;
        place(c, at, count);
        float top[2] = {kNegInf, kNegInf};
        if (count < 16)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (8 * n + 2 * (lane & 3) + (i & 1) >= count) s[n][i] = kNegInf;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) top[i >> 1] = fmaxf(top[i >> 1], s[n][i]);
        float grow[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
            const float next = fmaxf(m[i], top[i] * a.scale_log2);
            const float base = next == kNegInf ? 0.0f : next;       // nothing seen yet: every power below is zero
            grow[i] = power2(m[i] - base);
            m[i] = next;
            top[i] = base;
        }
        uint32_t p[4];
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[n][i] = power2(__fmul_rn(s[n][i], a.scale_log2) - top[i >> 1]);
                sum[i >> 1] += s[n][i];
            }
            p[2 * n] = pack_weights<T>(s[n][0], s[n][1]);
            p[2 * n + 1] = pack_weights<T>(s[n][2], s[n][3]);
        }
        l[0] = l[0] * grow[0] + sum[0];
        l[1] = l[1] * grow[1] + sum[1];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
            acc[n][0] *= grow[0];
            acc[n][1] *= grow[0];
            acc[n][2] *= grow[1];
            acc[n][3] *= grow[1];
        }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            uint32_t b[4];
            ldmatrix4_trans(b, at_value + value_row * P::kRowBytes + 32 * n + 16 * value_half);
            mma16816<T>(acc[2 * n], p, b[0], b[1]);
            mma16816<T>(acc[2 * n + 1], p, b[2], b[3]);
        }
        __syncwarp();                                    // every lane has read the stage that the next request overwrites
        int ahead = stage + P::kStages - 1;
        if (ahead >= P::kStages) ahead -= P::kStages;
        request(c + (P::kStages - 1) * step, ahead);
        if (++stage == P::kStages) stage = 0;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();                                        // the ring is free: the sums take its place

#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if ((lane & 3) == 0) {
            part_m[warp * 16 + (lane >> 2) + 8 * i] = m[i];
            part_l[warp * 16 + (lane >> 2) + 8 * i] = l[i];
        }
    }
    __syncthreads();                                     // the sums of a warp may reach into another warp's ring
    float* parts = reinterpret_cast<float*>(memory);
    constexpr float kDown = 1.0f / kWeightFactor<T>;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int h = (lane >> 2) + 8 * i;
            if (h < n_heads)
                *reinterpret_cast<float2*>(parts + (warp * 16 + h) * D + 8 * n + 2 * (lane & 3)) =
                    make_float2(acc[n][2 * i] * kDown, acc[n][2 * i + 1] * kDown);
        }
    join_and_write<T, D, kBaWarps, 16>(a, row, first_head, n_heads, rank, parts, part_m, part_l,
                                       reinterpret_cast<float*>(memory + P::kParts), joined_m, joined_l);
}

// ---------------------------------------------------------------------------- single precision

constexpr int kFpMaxHeads = 4;       // query heads a CTA at most
constexpr int kFpKeys = 4;           // keys of an eight-lane group at a time
constexpr int kFpChunk = 4 * kFpKeys;

// A CTA (4 warps) per row, key head and up to four query heads (one or two where no more share a key: the others' work would be
// thrown away).  At width 64 and one head 72 registers, seven CTAs an SM, are the fastest: 15.8 us for the 77 rows above, 17.6
// with eight, 20.2 unbounded; with four heads four CTAs (256 rows of 12 heads over 4: 47 us, 60 unbounded).  A lane keeps D / 8 components of the queries and of the
// sums, in pieces of four that lie 32 apart; a group of eight lanes keeps a maximum and a sum of its own, the four groups
// of a warp are joined at the end.
template <int D, int kFpHeads>
__global__ void __launch_bounds__(kBaThreads, D != 64 ? 1 : kFpHeads == 1 ? 7 : kFpHeads == 4 ? 4 : 1) block_attention_f32_kernel(const AttentionArgs a) {
    constexpr int kPieces = D / 32;
    __shared__ int kept[kBaMaxTop];
    __shared__ int n_kept;
    __shared__ float part_m[kBaWarps * 16], part_l[kBaWarps * 16], joined_m[16], joined_l[16];
    __shared__ alignas(16) float parts[kBaWarps * kFpHeads * D];      // written in pieces of 16 bytes
    __shared__ float joined[kFpHeads * D];
    const CtaPlace here(a);
    const int row = here.row, rank = here.rank, kv = here.kv, tile = here.tile;
    const int first_head = kv * a.group + kFpHeads * tile;
    const int n_heads = min(kFpHeads, a.group - kFpHeads * tile);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane >> 3, part = lane & 7;
    griddep_sync();
    float4 q[kFpHeads][kPieces];
#pragma unroll
    for (int h = 0; h < kFpHeads; ++h)
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
            q[h][p] = *reinterpret_cast<const float4*>(a.query + row * a.q_row + (first_head + min(h, n_heads - 1)) * a.q_head +
                                                       16 * (part + 8 * p));
    const int32_t* index = a.index + row * a.i_row + kv * a.i_head;
    const int first = first_index(index, a.top);
    int seq, t;
    if (!row_stands(a.rows, row, seq, t, a.status, threadIdx.x == 0 && here.first)) {
        write_blank<float, D>(a, row, first_head, n_heads, rank);
        return;
    }
    const int start = max(t - a.window + 1, 0);
    if (warp == 0) keep_blocks(index, first, a.top, a.block_size, start, kept, &n_kept);
    const float scale = a.flip ? -a.scale_log2 : a.scale_log2;
    __syncthreads();
    const int per_block = (min(a.block_size, start) + kFpChunk - 1) / kFpChunk;
    const int block_chunks = n_kept * per_block;
    const int chunks = block_chunks + (t - start + kFpChunk) / kFpChunk;
    const unsigned char* keys = a.key_cache + seq * a.k_seq + kv * a.k_head + 16 * part;
    const unsigned char* values = a.value_cache + seq * a.v_seq + kv * a.v_head + 16 * part;

    float4 acc[kFpHeads][kPieces];
    float m[kFpHeads], l[kFpHeads];
#pragma unroll
    for (int h = 0; h < kFpHeads; ++h) {
        m[h] = kNegInf;
        l[h] = 0.0f;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) acc[h][p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    for (int c = rank * kBaWarps + warp; c < chunks; c += kBaWarps * a.splits) {
        int at, count;
        if (c < block_chunks) {
            const int b = c / per_block, o = (c - b * per_block) * kFpChunk;
            at = kept[b] + o;
            count = min(min(a.block_size - o, kFpChunk), start - at);
        } else {
            at = start + (c - block_chunks) * kFpChunk;
            count = min(kFpChunk, t + 1 - at);
        }
        float s[kFpHeads][kFpKeys];
        float4 v[kFpKeys][kPieces];
#pragma unroll
        for (int u = 0; u < kFpKeys; ++u) {
            const int r = 4 * u + group;
            const bool live = r < count;
            float4 k[kPieces];
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
                const int64_t from = live ? at + r : t;
                k[p] = *reinterpret_cast<const float4*>(keys + from * a.k_row + 128 * p);
                v[u][p] = *reinterpret_cast<const float4*>(values + from * a.v_row + 128 * p);
                if (!live) v[u][p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int h = 0; h < kFpHeads; ++h) {
                float d = 0.0f;
#pragma unroll
                for (int p = 0; p < kPieces; ++p)
                    d = fmaf(q[h][p].x, k[p].x, fmaf(q[h][p].y, k[p].y, fmaf(q[h][p].z, k[p].z, fmaf(q[h][p].w, k[p].w, d))));
                d += __shfl_xor_sync(0xffffffffu, d, 1);
                d += __shfl_xor_sync(0xffffffffu, d, 2);
                d += __shfl_xor_sync(0xffffffffu, d, 4);
                s[h][u] = live ? d * scale : kNegInf;
            }
        }
#pragma unroll
        for (int h = 0; h < kFpHeads; ++h) {
            float next = m[h];
#pragma unroll
            for (int u = 0; u < kFpKeys; ++u) next = fmaxf(next, s[h][u]);
            const float base = next == kNegInf ? 0.0f : next;
            const float grow = power2(m[h] - base);
            m[h] = next;
            l[h] *= grow;
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
                acc[h][p].x *= grow;
                acc[h][p].y *= grow;
                acc[h][p].z *= grow;
                acc[h][p].w *= grow;
            }
#pragma unroll
            for (int u = 0; u < kFpKeys; ++u) {
                const float w = power2(s[h][u] - base);
                l[h] += w;
#pragma unroll
                for (int p = 0; p < kPieces; ++p) {
                    acc[h][p].x = fmaf(w, v[u][p].x, acc[h][p].x);
                    acc[h][p].y = fmaf(w, v[u][p].y, acc[h][p].y);
                    acc[h][p].z = fmaf(w, v[u][p].z, acc[h][p].z);
                    acc[h][p].w = fmaf(w, v[u][p].w, acc[h][p].w);
                }
            }
        }
    }
    // the four groups of the warp
#pragma unroll
    for (int h = 0; h < kFpHeads; ++h) {
        float next = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 8));
        next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, 16));
        const float grow = l[h] == 0.0f ? 0.0f : power2(m[h] - next);
        float sum = l[h] * grow;
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (lane == 0) {
            part_m[warp * 16 + h] = next;
            part_l[warp * 16 + h] = sum;
        }
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            float x[4] = {acc[h][p].x, acc[h][p].y, acc[h][p].z, acc[h][p].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = l[h] == 0.0f ? 0.0f : x[i] * grow;
                x[i] += __shfl_xor_sync(0xffffffffu, x[i], 8);
                x[i] += __shfl_xor_sync(0xffffffffu, x[i], 16);
            }
            if (group == 0)
                *reinterpret_cast<float4*>(parts + (warp * kFpHeads + h) * D + 4 * part + 32 * p) = make_float4(x[0], x[1], x[2], x[3]);
        }
    }
    join_and_write<float, D, kBaWarps, kFpHeads>(a, row, first_head, n_heads, rank, parts, part_m, part_l, joined, joined_m, joined_l);
}

template <typename Kernel>
int launch_rows(Kernel kernel, const char* name, const AttentionArgs& a, int smem, void* stream) {
    if (smem > 48 * 1024)
        if (int rc = allow_large_smem(reinterpret_cast<const void*>(kernel), kSmemDynamicLimit)) return rc;
    const dim3 grid(static_cast<unsigned>(a.rows.n_rows) * static_cast<unsigned>(a.splits * a.kv_heads * a.head_tiles));
    if (a.splits > 1) launch_kernel_cluster(kernel, grid, dim3(kBaThreads), static_cast<unsigned>(a.splits), smem, stream, a);
    else launch_kernel(kernel, grid, dim3(kBaThreads), smem, stream, a);
    count_launch();
    return check_launch(name);
}

template <int D>
int launch_width(AttentionArgs& a, int dtype, void* stream) {
    if (dtype == RLM_F32) {
        if (a.group == 1) return launch_rows(block_attention_f32_kernel<D, 1>, "block_attention_f32_kernel", a, 0, stream);
        if (a.group == 2) return launch_rows(block_attention_f32_kernel<D, 2>, "block_attention_f32_kernel", a, 0, stream);
        return launch_rows(block_attention_f32_kernel<D, 4>, "block_attention_f32_kernel", a, 0, stream);
    }
    if (dtype == RLM_BF16)
        return launch_rows(block_attention_rows_kernel<__nv_bfloat16, D>, "block_attention_rows_kernel", a, RowsPlan<D>::kTotal, stream);
    return launch_rows(block_attention_rows_kernel<__half, D>, "block_attention_rows_kernel", a, RowsPlan<D>::kTotal, stream);
}

}  // namespace
}  // namespace rlm

namespace rlm {
namespace {

// The sizes, strides and rule of a call; the checks that need no tensor are here, so that the workspace can be asked for
// before there is one.
int attention_args(AttentionArgs& a, const int64_t* position, const int32_t* row_batch, const int32_t* row_position,
                   const int64_t* strides, int n_rows, int n_seq, int max_t, int query_length, int heads, int kv_heads, int width,
                   int top_blocks, int block_size, int local_window, int dtype) {
    a.rows = Rows{position, row_batch, row_position, n_rows, n_seq, query_length, max_t};
    if (!strides) {
        set_error("block_attention: NULL argument");
        return RLM_ERR_NULL;
    }
    if (int rc = check_rows("block_attention: row_batch and row_position come together",
                            "block_attention: rows do not fit the sequences and positions of the caches", a.rows))
        return rc;
    if (!valid_dtype(dtype)) { set_error("block_attention: unknown dtype"); return RLM_ERR_DTYPE; }
    if (kv_heads < 1 || heads < 1 || heads % kv_heads != 0 || heads > 4096) {
        set_error("block_attention: the query heads (up to 4096) must be a multiple of the key heads");
        return RLM_ERR_SHAPE;
    }
    if (width != 32 && width != 64 && width != 96 && width != 128) {
        set_error("block_attention: head widths 32, 64, 96 and 128");
        return RLM_ERR_UNSUPPORTED;
    }
    if (top_blocks < 0 || top_blocks > kBaMaxTop || block_size < 1 || local_window < 0 ||
        static_cast<int64_t>(max_t) + block_size > 0x7fffffff) {
        set_error("block_attention: needs 0 to 128 blocks a row, block_size >= 1, local_window >= 0");
        return RLM_ERR_SHAPE;
    }
    const int e = dtype_size(dtype);
    int64_t* const to[8] = {&a.q_row, &a.q_head, &a.k_seq, &a.k_row, &a.k_head, &a.v_seq, &a.v_row, &a.v_head};
    const int extent[10] = {n_rows, heads, n_seq, max_t, kv_heads, n_seq, max_t, kv_heads, n_rows, kv_heads};
    auto step = [&](int i) { return extent[i] > 1 ? strides[i] : 0; };       // one of a kind has no step to the next
    for (int i = 0; i < 8; ++i) {
        *to[i] = step(i) * e;
        if (*to[i] % 16 != 0) {
            set_error("block_attention: queries and cache rows must lie on 16-byte boundaries");
            return RLM_ERR_ALIGN;
        }
    }
    a.i_row = step(8);
    a.i_head = step(9);
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.group = heads / kv_heads;
    a.top = top_blocks;
    a.block_size = block_size < max_t ? block_size : max_t;      // the first block is all that begins before a window
    a.window = local_window < max_t ? local_window : max_t;      // no row has more before it
    return RLM_OK;
}

}  // namespace
}  // namespace rlm

extern "C" int rlm_block_attention_workspace(const int64_t* strides, int n_rows, int n_seq, int max_t, int query_length, int heads,
                                             int kv_heads, int width, int top_blocks, int block_size, int local_window, int dtype,
                                             int64_t* bytes) {
    using namespace rlm;
    if (!bytes) { set_error("block_attention_workspace: NULL argument"); return RLM_ERR_NULL; }
    *bytes = 0;
    AttentionArgs a{};
    if (int rc = attention_args(a, nullptr, nullptr, nullptr, strides, n_rows, n_seq, max_t, query_length, heads, kv_heads, width,
                                top_blocks, block_size, local_window, dtype))
        return rc;
    if (n_rows > 0 && prefill_passes(a, width, dtype)) *bytes = prefill_workspace(a, width);
    return RLM_OK;
}

extern "C" int rlm_block_attention(const void* query, const void* key_cache, const void* value_cache, const int32_t* block_index,
                                   const int64_t* position, const int32_t* row_batch, const int32_t* row_position, void* out,
                                   float* lse, const int64_t* strides, int n_rows, int n_seq, int max_t, int query_length,
                                   int heads, int kv_heads, int width, int top_blocks, int block_size, int local_window,
                                   float scale, int dtype, void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
    using namespace rlm;
    AttentionArgs a{};
    if (n_rows > 0 && (!query || !key_cache || !value_cache || !out || !lse || (top_blocks > 0 && !block_index))) {
        set_error("block_attention: NULL argument");
        return RLM_ERR_NULL;
    }
    if (int rc = attention_args(a, position, row_batch, row_position, strides, n_rows, n_seq, max_t, query_length, heads, kv_heads,
                                width, top_blocks, block_size, local_window, dtype))
        return rc;
    if (n_rows == 0) return RLM_OK;
    if (!aligned16(query) || !aligned16(key_cache) || !aligned16(value_cache) || !aligned16(out)) {
        set_error("block_attention: queries and cache rows must lie on 16-byte boundaries");
        return RLM_ERR_ALIGN;
    }
    a.query = static_cast<const unsigned char*>(query);
    a.key_cache = static_cast<const unsigned char*>(key_cache);
    a.value_cache = static_cast<const unsigned char*>(value_cache);
    a.index = block_index;
    a.out = static_cast<unsigned char*>(out);
    a.lse = lse;
    a.status = status;
    a.scale_log2 = fabsf(scale) * kLog2e;
    if (a.scale_log2 == 0.0f) a.scale_log2 = 1e-37f;             // all weights are one, yet what is not seen stays at -inf
    a.flip = scale < 0.0f ? 0x80008000u : 0u;
    if (prefill_passes(a, width, dtype)) {
        const int64_t wanted = prefill_workspace(a, width);
        if (wanted > 0 && (!workspace || workspace_bytes < wanted || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)) {
            set_error("block_attention: whole sequences need the workspace that rlm_block_attention_workspace asks for, on a 256-byte boundary");
            return RLM_ERR_NULL;
        }
        return launch_prefill(a, width, dtype, static_cast<unsigned char*>(workspace), workspace_bytes, stream);
    }
    const int tile = dtype != RLM_F32 ? 16 : a.group <= 2 ? a.group : kFpMaxHeads;
    a.head_tiles = (a.group + tile - 1) / tile;
    // a row's keys over a cluster of CTAs, while the launch leaves SMs idle and every warp keeps a pass of 16 keys (beyond
    // that a cluster's joins cost more than the idle end of the launch: 512 CTAs of 1536 keys 69 us, as 1024 84)
    const int64_t ctas = static_cast<int64_t>(n_rows) * kv_heads * a.head_tiles;
    const int64_t passes = (static_cast<int64_t>(top_blocks) * ((a.block_size + 15) / 16) + (a.window + 15) / 16 + kBaWarps - 1) / kBaWarps;
    a.splits = 1;
    while (a.splits < kBaMaxSplit && ctas * a.splits * 2 <= 2 * sm_count() && passes >= 2 * a.splits) a.splits *= 2;
    if (ctas * a.splits > 0x7fffffff) {
        set_error("block_attention: too many rows or heads for one launch");
        return RLM_ERR_SHAPE;
    }
    switch (width) {
        case 32: return launch_width<32>(a, dtype, stream);
        case 64: return launch_width<64>(a, dtype, stream);
        case 96: return launch_width<96>(a, dtype, stream);
        default: return launch_width<128>(a, dtype, stream);
    }
}
