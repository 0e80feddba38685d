// Attention over router-chosen blocks for whole sequences (16-bit types), in three passes.
//
// Row by row every row would fetch its own blocks: 4 BS D bytes for each row, key head and block, from L2.  Here the pairs
// (row, block) are sorted by block instead, so that a block is fetched once for the 256 / group rows of a tile:
//
//   1. block_attention_sort_kernel: per segment of up to 4096 rows a counting sort of its pairs by block, and the list of
//      tiles: runs of up to 256 (row, query head) entries that share a block;
//   2. block_attention_tiles_kernel: per tile softmax(q K') V of the entries with the block, unnormalised (and times the factor
//      that fp16 weights carry), with the maximum and the sum, to the pair's place in the workspace (fp32);
//   3. block_attention_window_kernel: per 64 consecutive (row, query head) entries the attention over the local windows,
//      whose keys they share, joined with the pairs' partial results.
//
// An entry's arithmetic depends neither on its place in a tile nor on the entries beside it, nor thereby on the order of the
// sort: results are reproducible, those beside values that are not finite among them.
// The workspace is reused from segment to segment, which also keeps most of it in L2.
//
// The tiles of head widths 64 and 128 and blocks of up to 64 keys multiply on tcgen05; other widths and blocks, and the windows,
// whose keys differ from row to row, on the warp-level instruction, 16 entries a warp, operands in registers from the scores to
// the weighted sum.  What bounds the passes is the partial results' bytes, 8 D bytes an entry and block written and read, and
// the chain of steps of a tile.  8 x 4096 rows, 8 heads over 2 of width 64, four blocks of 64: 174 us, row by row 1471.  Each pass
// for itself under a profiler (its 185 are more than the 174 of the passes in a row): sort 11, tiles 89, windows 85.  In working
// copies the tiles without their stores took 69 us, the join alone 67 (268 MB of partial results, 4.0 TB/s), the windows alone 52,
// windows and join one after the other in a CTA 92.
#include "block_attention_mma.cuh"
#include "rlm_tcgen05.cuh"

namespace rlm {
namespace {

constexpr int kBpWarps = 4;
constexpr int kBpThreads = 32 * kBpWarps;
constexpr int kBpEntries = 16 * kBpWarps;       // entries at a time
constexpr int kBpTile = 4 * kBpEntries;         // entries of a tile that shares a block
constexpr int kBpWindowKeys = 32;                // keys of a window staged at a time
constexpr int kBpSegment = 4096;                // rows a segment at most
constexpr int kBpSortThreads = 1024;
constexpr int kBpHeldBlocks = 16;               // of a row, in registers
constexpr int kBpMaxBins = 16384;
constexpr int kBpRankBits = 7;                  // a pair: row of the segment and rank of the block, below kBaMaxTop
// Aimed at: few segments at a time would keep the partial results in L2, but the ends of the shorter launches cost more (48, 72,
// 100, 140 MB: 313, 240, 225, 212 us against 185 for the rows above); more than this gains nothing.
constexpr int64_t kBpWorkspace = int64_t{512} << 20;

struct Tile { int block, first, entries, pad; };         // entries of the pairs list from `first` / group on

// The workspace of a segment, in bytes from its start.  `sums`: an entry's row of D partial sums, of every 16 components the
// four that a lane of the tensor instruction's result holds side by side (2q, 2q + 1, 2q + 8, 2q + 9), so that it is written
// and read 16 bytes at a time.
struct SegmentPlan {
    int64_t sums, stats, pairs, kept, count, tiles, tile_count, total;
};

struct PrefillArgs {
    AttentionArgs a;
    unsigned char* workspace;
    SegmentPlan plan;
    int segment_rows, segments_per_seq, first_segment, choices, bins, max_tiles;
    Divisor by_group;
};

// Segment `s` of the launch: its sequence, its first position and its rows.
struct Segment { int seq, t0, rows; unsigned char* base; };
__device__ __forceinline__ Segment segment_of(const PrefillArgs& p, int s) {
    const int id = p.first_segment + s;
    Segment g;
    g.seq = id / p.segments_per_seq;
    g.t0 = (id - g.seq * p.segments_per_seq) * p.segment_rows;
    g.rows = min(p.segment_rows, p.a.rows.query_length - g.t0);
    g.base = p.workspace + s * p.plan.total;
    return g;
}

// The distinct blocks among a row's indices that begin before its window: a bit for each of up to kTop places.
template <int kTop>
__device__ __forceinline__ unsigned row_blocks(const int32_t* index, int top, int before, int (&block)[kTop > 0 ? kTop : 1]) {
#pragma unroll
    for (int i = 0; i < kTop; ++i) block[i] = i < top ? index[i] : -1;
    unsigned kept = 0;
#pragma unroll
    for (int i = 0; i < kTop; ++i) {
        bool keep = block[i] >= 0 && block[i] < before;
#pragma unroll
        for (int o = 0; o < i; ++o) keep = keep && block[o] != block[i];
        kept |= static_cast<unsigned>(keep) << i;
    }
    return kept;
}

// kTop: rows of up to so many blocks keep them in registers (a segment of more rows than threads reads them twice); 0: any number,
// by way of the workspace.  1024 rows of 16 blocks, 8 heads over 2: the three passes 41 us, 52 by way of the workspace.
template <int kTop>
__global__ void __launch_bounds__(kBpSortThreads) block_attention_sort_kernel(const PrefillArgs p) {
    extern __shared__ int bins[];               // [bins]: pairs of a block, then the place of its next pair
    __shared__ int warp_pairs[32], warp_tiles[32];
    griddep_sync();
    const AttentionArgs& a = p.a;
    const Segment g = segment_of(p, blockIdx.y);
    const int choice = blockIdx.x;
    int* kept = reinterpret_cast<int*>(g.base + p.plan.kept) + static_cast<int64_t>(choice) * p.segment_rows * a.top;
    int* count = reinterpret_cast<int*>(g.base + p.plan.count) + choice * p.segment_rows;
    int* pairs = reinterpret_cast<int*>(g.base + p.plan.pairs) + static_cast<int64_t>(choice) * p.segment_rows * a.top;
    Tile* tiles = reinterpret_cast<Tile*>(g.base + p.plan.tiles) + static_cast<int64_t>(choice) * p.max_tiles;
    for (int i = threadIdx.x; i < p.bins; i += kBpSortThreads) bins[i] = 0;
    __syncthreads();
    const int64_t first_row = static_cast<int64_t>(g.seq) * a.rows.query_length + g.t0;
    const int32_t* indices = a.index + first_row * a.i_row + choice * a.i_head;
    // blocks that begin before the window of row r
    auto blocks_before = [&](int r) { return (max(g.t0 + r - a.window + 1, 0) + a.block_size - 1) / a.block_size; };
    int block[kTop > 0 ? kTop : 1];
    unsigned mask = 0;
    for (int r = threadIdx.x; r < g.rows; r += kBpSortThreads) {
        const int32_t* index = indices + r * a.i_row;
        const int before = blocks_before(r);
        int n = 0;
        if constexpr (kTop > 0) {
            mask = row_blocks<kTop>(index, a.top, before, block);
#pragma unroll
            for (int i = 0; i < kTop; ++i)
                if (mask >> i & 1u) atomicAdd(&bins[block[i]], 1);
            n = __popc(mask);
        } else {
            for (int i = 0; i < a.top; ++i) {
                const int at = index[i];
                bool keep = at >= 0 && at < before;
                for (int o = 0; keep && o < i; ++o) keep = index[o] != at;
                if (keep) {
                    kept[r * a.top + n++] = at;
                    atomicAdd(&bins[at], 1);
                }
            }
        }
        count[r] = n;
    }
    __syncthreads();
    // exclusive sums over the blocks, of pairs and of tiles: a run of bins a thread, then the threads
    const int run = (p.bins + kBpSortThreads - 1) / kBpSortThreads;
    const int from = min(threadIdx.x * run, p.bins), to = min(from + run, p.bins);
    int my_pairs = 0, my_tiles = 0;
    for (int i = from; i < to; ++i) {
        my_pairs += bins[i];
        my_tiles += (bins[i] * a.group + kBpTile - 1) / kBpTile;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int pair_sum = my_pairs, tile_sum = my_tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, pair_sum, d), y = __shfl_up_sync(0xffffffffu, tile_sum, d);
        if (lane >= d) {
            pair_sum += x;
            tile_sum += y;
        }
    }
    if (lane == 31) {
        warp_pairs[warp] = pair_sum;
        warp_tiles[warp] = tile_sum;
    }
    __syncthreads();
    int pair = pair_sum - my_pairs, tile = tile_sum - my_tiles;
    for (int w = 0; w < warp; ++w) {
        pair += warp_pairs[w];
        tile += warp_tiles[w];
    }
    for (int i = from; i < to; ++i) {
        const int entries = bins[i] * a.group;
        for (int e = 0; e < entries; e += kBpTile) tiles[tile++] = Tile{i, pair * a.group + e, min(kBpTile, entries - e), 0};
        const int here = bins[i];
        bins[i] = pair;
        pair += here;
    }
    if (threadIdx.x == kBpSortThreads - 1) reinterpret_cast<int*>(g.base + p.plan.tile_count)[choice] = tile;
    __syncthreads();
    for (int r = threadIdx.x; r < g.rows; r += kBpSortThreads) {
        if constexpr (kTop > 0) {
            if (g.rows > kBpSortThreads) mask = row_blocks<kTop>(indices + r * a.i_row, a.top, blocks_before(r), block);
#pragma unroll
            for (int i = 0; i < kTop; ++i)
                if (mask >> i & 1u) pairs[atomicAdd(&bins[block[i]], 1)] = r << kBpRankBits | __popc(mask & ((1u << i) - 1));
        } else {
            const int n = count[r];
            for (int i = 0; i < n; ++i) pairs[atomicAdd(&bins[kept[r * a.top + i]], 1)] = r << kBpRankBits | i;
        }
    }
}

__device__ __forceinline__ float2 widen(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 widen(__half2 v) { return __half22float2(v); }

template <int D> struct TileShape {
    static constexpr int kRowBytes = 2 * D + 16;          // odd multiple of 16 bytes: ldmatrix without bank conflicts
    static constexpr int kPieces = D / 8;
};

// kKeys rows of a cache from position `at` on into shared memory, zeros beyond `count`.
template <int D, int kKeys>
__device__ __forceinline__ void request_rows(uint32_t to, const unsigned char* cache, int64_t row_stride, int at, int count) {
    using S = TileShape<D>;
    for (int i = threadIdx.x; i < kKeys * S::kPieces; i += kBpThreads) {
        const int r = i / S::kPieces, piece = i - r * S::kPieces;
        const bool live = r < count;
        cp_async16_or_zero(to + r * S::kRowBytes + 16 * piece, cache + (live ? at + r : 0) * row_stride + 16 * piece, live);
    }
}

// Whether this thread's share of kKeys staged rows (`of` threads take one each in turn) holds a value that is not finite:
// zero times it is NaN.
template <typename T, int D, int kKeys>
__device__ __forceinline__ bool staged_not_finite(const unsigned char* rows, int thread, int of) {
    using S = TileShape<D>;
    using Pair = std::conditional_t<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>;
    const uint32_t none = 0;
    const Pair zero = *reinterpret_cast<const Pair*>(&none);
    Pair sum = zero;
    for (int item = thread; item < kKeys * S::kPieces; item += of) {
        const int r = item / S::kPieces, piece = item - r * S::kPieces;
        const uint4 v = *reinterpret_cast<const uint4*>(rows + r * S::kRowBytes + 16 * piece);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = __hfma2(*reinterpret_cast<const Pair*>(&w[j]), zero, sum);
    }
    const float2 f = widen(sum);
    return f.x != 0.0f || f.y != 0.0f;                   // NaN is not equal to zero
}

// The running softmax of a warp's 16 entries: rows lane / 4 and lane / 4 + 8 of this lane.
template <int D> struct Running {
    float acc[D / 8][4];
    float m[2], l[2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
        m[0] = m[1] = kNegInf;
        l[0] = l[1] = 0.0f;
    }
};

// kKeys staged keys and values against a warp's 16 entries; an entry sees the keys [low, high) of them.  `careful`: some value
// is not finite and not every entry sees every key, so a weight of zero must not meet it: the weighted sums of this lane's
// entries that are `cut` are made on the CUDA cores, of the keys that they see.  In windows (kAscending) all entries are cut.
template <typename T, int D, int kKeys, bool kAscending>
__device__ __forceinline__ void take_keys(Running<D>& run, const uint32_t (&q)[D / 16][4], uint32_t keys, uint32_t values,
                                          const int (&low)[2], const int (&high)[2], float scale_log2, bool careful, const bool (&cut)[2],
                                          const unsigned char* value_rows) {
    using S = TileShape<D>;
    const int lane = threadIdx.x & 31;
    const int key_row = (lane & 7) + ((lane >> 4) << 3), key_half = (lane >> 3) & 1;
    const int value_row = lane & 15, value_half = lane >> 4;
    // the warp's entries ascend: the first sees the first keys, the last the last ones.  16 keys that none sees are passed by
    const int first_seen = kAscending ? __shfl_sync(0xffffffffu, low[0], 0) : 0;
    const int last_seen = kAscending ? __shfl_sync(0xffffffffu, high[1], 31) : kKeys;
    float s[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
    for (int n = 0; n < kKeys / 16; ++n)
        if (16 * n + 16 > first_seen && 16 * n < last_seen)
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];
            ldmatrix4(b, keys + (16 * n + key_row) * S::kRowBytes + 32 * k + 16 * key_half);
            mma16816<T>(s[2 * n], q[k], b[0], b[1]);
            mma16816<T>(s[2 * n + 1], q[k], b[2], b[3]);
        }
    float top[2] = {kNegInf, kNegInf};
    if (__any_sync(0xffffffffu, low[0] > 0 || low[1] > 0 || high[0] < kKeys || high[1] < kKeys))
#pragma unroll
        for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 8 * n + 2 * (lane & 3) + (i & 1);
                if (key < low[i >> 1] || key >= high[i >> 1]) s[n][i] = kNegInf;
            }
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i >> 1] = fmaxf(top[i >> 1], s[n][i]);
    float grow[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        const float next = fmaxf(run.m[i], top[i] * scale_log2);
        const float base = next == kNegInf ? 0.0f : next;           // nothing seen yet: every power below is zero
        grow[i] = power2(run.m[i] - base);
        run.m[i] = next;
        top[i] = base;
        run.l[i] *= grow[i];
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) run.acc[n][i] *= grow[i >> 1];
#pragma unroll
    for (int n = 0; n < kKeys / 16; ++n) {
        if (16 * n + 16 <= first_seen || 16 * n >= last_seen) continue;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float* x = s[2 * n + j];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = power2(__fmul_rn(x[i], scale_log2) - top[i >> 1]);
                run.l[i >> 1] += x[i];
            }
            w[2 * j] = pack_weights<T>(x[0], x[1]);
            w[2 * j + 1] = pack_weights<T>(x[2], x[3]);
        }
        if (careful) {
            if constexpr (!kAscending) {           // the other entries as ever: their sums do not hang on their neighbours
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    uint32_t b[4];
                    ldmatrix4_trans(b, values + (16 * n + value_row) * S::kRowBytes + 32 * d + 16 * value_half);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float* acc = run.acc[2 * d + j];
                        float sum[4] = {acc[0], acc[1], acc[2], acc[3]};
                        mma16816<T>(sum, w, b[2 * j], b[2 * j + 1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!cut[i >> 1]) acc[i] = sum[i];
                    }
                }
            }
#pragma unroll 1
            for (int k = 0; k < 16; ++k) {
                const int owner = (lane & ~3) | ((k & 7) >> 1), key = 16 * n + k;
                const uint32_t both[2] = {__shfl_sync(0xffffffffu, k < 8 ? w[0] : w[2], owner),
                                          __shfl_sync(0xffffffffu, k < 8 ? w[1] : w[3], owner)};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (!cut[i] || key < low[i] || key >= high[i]) continue;
                    const float2 pair = unpack2<T>(both[i]);
                    const float weight = (k & 1) ? pair.y : pair.x;
#pragma unroll
                    for (int d = 0; d < D / 8; ++d) {
                        const float2 v = unpack2<T>(*reinterpret_cast<const uint32_t*>(value_rows + key * S::kRowBytes + 16 * d + 4 * (lane & 3)));
                        run.acc[d][2 * i] = fmaf(weight, v.x, run.acc[d][2 * i]);
                        run.acc[d][2 * i + 1] = fmaf(weight, v.y, run.acc[d][2 * i + 1]);
                    }
                }
            }
            continue;
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            uint32_t b[4];
            ldmatrix4_trans(b, values + (16 * n + value_row) * S::kRowBytes + 32 * d + 16 * value_half);
            mma16816<T>(run.acc[2 * d], w, b[0], b[1]);
            mma16816<T>(run.acc[2 * d + 1], w, b[2], b[3]);
        }
    }
}

template <int D>
__device__ __forceinline__ void load_queries(uint32_t (&q)[D / 16][4], uint32_t staged, uint32_t flip) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
        ldmatrix4(q[k], staged + (lane & 15) * TileShape<D>::kRowBytes + 32 * k + 16 * (lane >> 4));
    if (flip)
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) q[k][i] ^= flip;
}

// A tile of up to 256 entries that share a block, against that block.  A block of up to kKeys keys is staged once; then
// each warp takes 16 entries at a time on its own, their queries requested while it works on the 16 before.
template <typename T, int D, int kKeys>
__global__ void __launch_bounds__(kBpThreads) block_attention_tiles_kernel(const PrefillArgs p) {
    using S = TileShape<D>;
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ int2 entries[kBpTile];              // pair and query head of each entry
    griddep_sync();
    const AttentionArgs& a = p.a;
    const Segment g = segment_of(p, blockIdx.z);
    const int kv = blockIdx.y, choice = p.choices == 1 ? 0 : kv;
    const Tile tile = reinterpret_cast<const Tile*>(g.base + p.plan.tiles)[static_cast<int64_t>(choice) * p.max_tiles + blockIdx.x];
    if (static_cast<int>(blockIdx.x) >= reinterpret_cast<const int*>(g.base + p.plan.tile_count)[choice]) return;
    const int* pairs = reinterpret_cast<const int*>(g.base + p.plan.pairs) + static_cast<int64_t>(choice) * p.segment_rows * a.top;
    const unsigned char* staged_values = memory + kKeys * S::kRowBytes;
    const uint32_t keys = smem_u32(memory), values = keys + kKeys * S::kRowBytes;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t staged_q = values + (kKeys + 32 * warp) * S::kRowBytes;          // two times 16 entries a warp

    const unsigned char* key_rows = a.key_cache + g.seq * a.k_seq + kv * a.k_head;
    const unsigned char* value_rows = a.value_cache + g.seq * a.v_seq + kv * a.v_head;
    const int at = tile.block * a.block_size;
    // rows of the block before the last window of the segment; no entry sees more
    const int cached = min(a.block_size, g.t0 + g.rows - a.window - at);
    request_rows<D, kKeys>(keys, key_rows, a.k_row, at, cached);
    request_rows<D, kKeys>(values, value_rows, a.v_row, at, cached);
    for (int e = threadIdx.x; e < tile.entries; e += kBpThreads) {
        const int pair = p.by_group.quotient(tile.first + e);
        entries[e] = make_int2(pairs[pair], tile.first + e - pair * a.group);
    }
    __syncthreads();
    const unsigned char* queries = a.query + (static_cast<int64_t>(g.seq) * a.rows.query_length + g.t0) * a.q_row + kv * a.group * a.q_head;
    auto request_queries = [&](int strip, int stage) {
        for (int i = lane; i < 16 * S::kPieces; i += 32) {
            const int e = i / S::kPieces, piece = i - e * S::kPieces;
            const bool live = 16 * strip + e < tile.entries;
            const int2 entry = live ? entries[16 * strip + e] : make_int2(0, 0);
            cp_async16_or_zero(staged_q + (16 * stage + e) * S::kRowBytes + 16 * piece,
                               queries + (entry.x >> kBpRankBits) * a.q_row + entry.y * a.q_head + 16 * piece, live);
        }
        cp_async_commit();
    };
    request_queries(warp, 0);
    const bool one_chunk = a.block_size <= kKeys;
    bool looked = false, finite = true;
    const int strips = (tile.entries + 15) >> 4, rounds = (strips + kBpWarps - 1) / kBpWarps;
    for (int j = 0; j < rounds; ++j) {
        const int strip = j * kBpWarps + warp;
        if (one_chunk && j > 0 && strip >= strips) break;
        cp_async_wait_all();
        if (j == 0) __syncthreads();               // the block has arrived
        else __syncwarp();
        int place[2], head_of[2], before[2];       // this lane's entries: pair, head, keys of the block before the row's window
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = 16 * strip + (lane >> 2) + 8 * i;
            const int2 entry = e < tile.entries ? entries[e] : make_int2(-1, 0);
            place[i] = entry.x;
            head_of[i] = entry.y;
            before[i] = entry.x < 0 ? cached : min(max(g.t0 + (entry.x >> kBpRankBits) - a.window + 1, 0) - at, cached);
        }
        uint32_t q[D / 16][4];
        load_queries<D>(q, staged_q + 16 * (j & 1) * S::kRowBytes, a.flip);
        request_queries(strip + kBpWarps, (j + 1) & 1);
        Running<D> run;
        run.clear();
        for (int o = 0; o < cached; o += kKeys) {
            if (!one_chunk && (o > 0 || j > 0)) {
                __syncthreads();
                request_rows<D, kKeys>(keys, key_rows, a.k_row, at + o, cached - o);
                request_rows<D, kKeys>(values, value_rows, a.v_row, at + o, cached - o);
                cp_async_commit();
                cp_async_wait_all();
                __syncthreads();
            }
            // where an entry sees less than the whole block, a value that is not finite must not meet a weight of zero
            const bool clipped = __any_sync(0xffffffffu, before[0] < cached || before[1] < cached);
            if (clipped && !(one_chunk && looked)) {
                finite = !__any_sync(0xffffffffu, staged_not_finite<T, D, kKeys>(staged_values, lane, 32));
                looked = true;
            }
            const int left = cached - o;
            const int low[2] = {0, 0}, high[2] = {min(before[0] - o, left), min(before[1] - o, left)};
            const bool cut[2] = {before[0] < cached, before[1] < cached};
            take_keys<T, D, kKeys, false>(run, q, keys, values, low, high, a.scale_log2, clipped && !finite, cut, staged_values);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            run.l[i] += __shfl_xor_sync(0xffffffffu, run.l[i], 1);
            run.l[i] += __shfl_xor_sync(0xffffffffu, run.l[i], 2);
            if (place[i] < 0) continue;
            const int row = place[i] >> kBpRankBits, rank = place[i] & ((1 << kBpRankBits) - 1);
            const int64_t entry = ((static_cast<int64_t>(row) * a.kv_heads + kv) * a.top + rank) * a.group + head_of[i];
            float* sums = reinterpret_cast<float*>(g.base + p.plan.sums) + entry * D + 4 * (lane & 3);
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
                *reinterpret_cast<float4*>(sums + 16 * n) = make_float4(run.acc[2 * n][2 * i], run.acc[2 * n][2 * i + 1],
                                                                        run.acc[2 * n + 1][2 * i], run.acc[2 * n + 1][2 * i + 1]);
            if ((lane & 3) == 0) reinterpret_cast<float2*>(g.base + p.plan.stats)[entry] = make_float2(run.m[i], run.l[i]);
        }
    }
    cp_async_wait_all();
}

// The same on the fifth-generation tensor cores, for head widths 64 and 128 and blocks of up to 64 keys: 128 entries at a
// time, a thread's row of scores in tensor memory.  Scores K-major times K-major; the weights go back to shared memory over
// the queries and multiply the values where they lie, MN-major (a block's rows are 64 components wide, eight keys 1024 bytes,
// 64-component halves of a wider head kKeys x 128 bytes apart).  The sums take the scores' columns.  Small CTAs, three to six
// an SM, hide one another's steps: 89 us for 1.05 million entries (140 with the warp-level instruction above, whose operands
// are read from shared memory again for every 16 entries).
__device__ __forceinline__ void tmem_ld_16x256b(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}

// Descriptor of values where they lie: rows of 128 bytes (64 components, MN-major), eight keys 1024 bytes apart, the next 64
// components `block` bytes further.
__device__ __forceinline__ uint64_t value_desc(uint32_t addr, uint32_t block) {
    return smem_desc_sw128(addr) - (uint64_t{1} << 16) + (static_cast<uint64_t>(block >> 4) << 16);
}
constexpr float kInfinity = __builtin_huge_valf();

constexpr int kTtRows = 128;
template <int D, int kKeys> struct TensorTile {
    static constexpr int kQueryBlock = kTtRows * 128;      // bytes of 64 components of the rows
    static constexpr int kKeyBlock = kKeys * 128;          // ... of the block's keys (values)
    static constexpr int kBlocks = D / 64;
    static constexpr int kQueries = kBlocks * kQueryBlock;
    static constexpr int kBytes = kQueries + 2 * kBlocks * kKeyBlock + 1024;
    static constexpr int kColumns = D > kKeys ? D : kKeys < 32 ? 32 : kKeys;
};

template <typename T, int D, int kKeys>
__global__ void __launch_bounds__(kTtRows, D == 64 ? 6 : 3) block_attention_tensor_tiles_kernel(const PrefillArgs p) {
    using S = TensorTile<D, kKeys>;
    constexpr int kPieces = D / 8;
    extern __shared__ __align__(1024) unsigned char raw_memory[];
    __shared__ int2 entries[kBpTile];              // pair and query head of each entry
    __shared__ __align__(8) unsigned long long bar_slot;
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    griddep_sync();
    const AttentionArgs& a = p.a;
    const Segment g = segment_of(p, blockIdx.z);
    const int kv = blockIdx.y, choice = p.choices == 1 ? 0 : kv;
    const Tile tile = reinterpret_cast<const Tile*>(g.base + p.plan.tiles)[static_cast<int64_t>(choice) * p.max_tiles + blockIdx.x];
    if (static_cast<int>(blockIdx.x) >= reinterpret_cast<const int*>(g.base + p.plan.tile_count)[choice]) return;
    const int* pairs = reinterpret_cast<const int*>(g.base + p.plan.pairs) + static_cast<int64_t>(choice) * p.segment_rows * a.top;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned char* memory = smem_align1024(raw_memory);
    unsigned char* staged_values = memory + S::kQueries + S::kBlocks * S::kKeyBlock;
    const uint32_t queries_at = smem_u32(memory), keys_at = queries_at + S::kQueries, values_at = keys_at + S::kBlocks * S::kKeyBlock;
    const uint32_t bar = smem_u32(&bar_slot);
    if (tid == 0) {
        mbar_init(bar, 1);
        fence_barrier_init();
        failed = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(S::kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const unsigned char* key_rows = a.key_cache + g.seq * a.k_seq + kv * a.k_head;
    const unsigned char* value_rows = a.value_cache + g.seq * a.v_seq + kv * a.v_head;
    const int at = tile.block * a.block_size, cached = min(a.block_size, a.rows.max_t - at);
#pragma unroll
    for (int i = tid; i < kKeys * kPieces; i += kTtRows) {
        const int r = i / kPieces, piece = i - r * kPieces;
        const bool live = r < cached;
        const int64_t from = live ? at + r : 0;
        cp_async16_or_zero(keys_at + swizzled(r, piece, S::kKeyBlock), key_rows + from * a.k_row + 16 * piece, live);
        cp_async16_or_zero(values_at + swizzled(r, piece, S::kKeyBlock), value_rows + from * a.v_row + 16 * piece, live);
    }
    for (int e = tid; e < kBpTile; e += kTtRows) {
        int2 entry = make_int2(-1, 0);
        if (e < tile.entries) {
            const int pair = p.by_group.quotient(tile.first + e);
            entry = make_int2(pairs[pair], tile.first + e - pair * a.group);
        }
        entries[e] = entry;
    }
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    const unsigned char* queries = a.query + (static_cast<int64_t>(g.seq) * a.rows.query_length + g.t0) * a.q_row + kv * a.group * a.q_head;
    constexpr uint32_t kFormat = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t kScores = (1u << 4) | (kFormat << 7) | (kFormat << 10) | (static_cast<uint32_t>(kKeys >> 3) << 17) | (8u << 24);
    constexpr uint32_t kSums = (1u << 4) | (kFormat << 7) | (kFormat << 10) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (8u << 24);
    uint32_t phase = 0;
    bool looked = false, finite = true;
    for (int first = 0; first < tile.entries; first += kTtRows) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int item = i * kTtRows + tid, e = item / kPieces, piece = item - e * kPieces;
            const int2 entry = entries[first + e];
            cp_async16_or_zero(queries_at + swizzled(e, piece, S::kQueryBlock),
                               queries + max(entry.x >> kBpRankBits, 0) * a.q_row + entry.y * a.q_head + 16 * piece, entry.x >= 0);
        }
        cp_async_commit();
        const int2 mine = entries[first + tid];
        const int before = mine.x < 0 ? cached : min(max(g.t0 + (mine.x >> kBpRankBits) - a.window + 1, 0) - at, cached);
        cp_async_wait_all();
        fence_proxy_async();
        const bool clipped = __syncthreads_or(before < cached);
        if (warp == 0) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const bool elected = elect_lane();
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                umma_f16_if(tmem, smem_desc_sw128(queries_at + (k >> 2) * S::kQueryBlock) + 2 * (k & 3),
                            smem_desc_sw128(keys_at + (k >> 2) * S::kKeyBlock) + 2 * (k & 3), kScores, k > 0, elected);
            umma_commit_if(bar, elected);
        }
        // where an entry sees less than the whole block, a value that is not finite must not meet a weight of zero
        if (clipped && !looked) {
            bool bad = false;
            for (int i = tid; i < kKeys * kPieces; i += kTtRows) {
                const uint4 v = *reinterpret_cast<const uint4*>(staged_values + i * 16);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 f = unpack2<T>(w[k]);
                    bad = bad || !(fabsf(f.x) < kInfinity && fabsf(f.y) < kInfinity);
                }
            }
            finite = !__syncthreads_or(bad);
            looked = true;
        }
        if (!mbar_wait(bar, phase)) failed = 1;
        phase ^= 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t my_rows = tmem + (static_cast<uint32_t>(32 * warp) << 16);
        // the scores twice from tensor memory, 16 or 32 at a time: their maximum, then the weights
        const bool some = __any_sync(0xffffffffu, before < kKeys);
        auto scores = [&](int c, float (&x)[16]) {
            uint32_t v[16];
            tmem_ld16(my_rows + 16 * c, v);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = __uint_as_float(v[k]);
            if (a.flip)
#pragma unroll
                for (int k = 0; k < 16; ++k) x[k] = -x[k];
            if (some)
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (16 * c + k >= before) x[k] = kNegInf;
        };
        float top = kNegInf;
#pragma unroll
        for (int c = 0; c < kKeys / 16; ++c) {
            float x[16];
            scores(c, x);
#pragma unroll
            for (int k = 0; k < 16; ++k) top = fmaxf(top, x[k]);
        }
        top *= a.scale_log2;
        const float base = top == kNegInf ? 0.0f : top;
        float2 sum2 = make_float2(0.0f, 0.0f);
        const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), base2 = make_float2(-base, -base);
#pragma unroll
        for (int c = 0; c < kKeys / 16; ++c) {
            float x[16];
            scores(c, x);
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
                const float2 y = __fadd2_rn(__fmul2_rn(make_float2(x[k], x[k + 1]), scale2), base2);
                x[k] = power2(y.x);
                x[k + 1] = power2(y.y);
            }
            float2 part[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) part[k] = __fadd2_rn(make_float2(x[4 * k], x[4 * k + 1]), make_float2(x[4 * k + 2], x[4 * k + 3]));
            sum2 = __fadd2_rn(sum2, __fadd2_rn(__fadd2_rn(part[0], part[1]), __fadd2_rn(part[2], part[3])));
            // in the queries' place: the first product is over
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<uint4*>(memory + swizzled(tid, 2 * c + h, S::kQueryBlock)) =
                    make_uint4(pack_weights<T>(x[8 * h], x[8 * h + 1]), pack_weights<T>(x[8 * h + 2], x[8 * h + 3]),
                               pack_weights<T>(x[8 * h + 4], x[8 * h + 5]), pack_weights<T>(x[8 * h + 6], x[8 * h + 7]));
        }
        if (mine.x >= 0) {
            const int row = mine.x >> kBpRankBits, rank = mine.x & ((1 << kBpRankBits) - 1);
            const int64_t entry = ((static_cast<int64_t>(row) * a.kv_heads + kv) * a.top + rank) * a.group + mine.y;
            reinterpret_cast<float2*>(g.base + p.plan.stats)[entry] = make_float2(top, sum2.x + sum2.y);
            if (!finite && before < cached) {
                // the weighted sum on the CUDA cores, of the keys that the entry sees, 16 components at a time: the entry's own
                // matter, so that its neighbours' sums do not hang on it; below, its place is passed by
                entries[first + tid].x = -1;
                float* sums = reinterpret_cast<float*>(g.base + p.plan.sums) + entry * D;
#pragma unroll 1
                for (int d = 0; d < D; d += 16) {
                    float acc[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
#pragma unroll 1
                    for (int k = 0; k < before; ++k) {
                        const float w = load_value<T>(memory + swizzled(tid, k >> 3, S::kQueryBlock) + 2 * (k & 7));
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint4 v = *reinterpret_cast<const uint4*>(staged_values + swizzled(k, (d >> 3) + i, S::kKeyBlock));
                            const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int n = 0; n < 4; ++n) {
                                const float2 f = unpack2<T>(word[n]);
                                acc[8 * i + 2 * n] = fmaf(w, f.x, acc[8 * i + 2 * n]);
                                acc[8 * i + 2 * n + 1] = fmaf(w, f.y, acc[8 * i + 2 * n + 1]);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4*>(sums + d + 4 * i) = make_float4(acc[2 * i], acc[2 * i + 1], acc[8 + 2 * i], acc[9 + 2 * i]);
                }
            }
        }
        fence_proxy_async();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();
        if (failed) break;
        if (warp == 0) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const bool elected = elect_lane();
#pragma unroll
            for (int k = 0; k < kKeys / 16; ++k)
                umma_f16_if(tmem, smem_desc_sw128(queries_at) + 2 * k, value_desc(values_at + 2048 * k, S::kKeyBlock), kSums, k > 0, elected);
            umma_commit_if(bar, elected);
        }
        if (!mbar_wait(bar, phase)) failed = 1;
        phase ^= 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float* to[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int2 other = entries[first + 32 * warp + 16 * half + (lane >> 2) + 8 * i];
                const int row = other.x >> kBpRankBits, rank = other.x & ((1 << kBpRankBits) - 1);
                const int64_t entry = ((static_cast<int64_t>(row) * a.kv_heads + kv) * a.top + rank) * a.group + other.y;
                to[i] = other.x < 0 ? nullptr : reinterpret_cast<float*>(g.base + p.plan.sums) + entry * D + 4 * (lane & 3);
            }
#pragma unroll
            for (int b = 0; b < D / 64; ++b) {
                uint32_t v[32];
                tmem_ld_16x256b(tmem + (static_cast<uint32_t>(32 * warp + 16 * half) << 16) + 64 * b, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (to[i])
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            *reinterpret_cast<uint4*>(to[i] + 64 * b + 16 * c) =
                                make_uint4(v[8 * c + 2 * i], v[8 * c + 2 * i + 1], v[8 * c + 4 + 2 * i], v[8 * c + 4 + 2 * i + 1]);
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();                           // the queries' place and the scores' columns are free
        if (failed) break;
    }
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns));
    }
    if (failed && tid == 0 && a.status) atomicOr(a.status, RLM_DEV_TIMEOUT);
}

// 64 consecutive (row, query head) entries of a segment and key head: their windows, whose keys they share, and the pairs'
// partial results, each requested ahead of a piece of the window and joined behind it.
template <typename T, int D>
__global__ void __launch_bounds__(kBpThreads, D <= 64 ? 4 : 2) block_attention_window_kernel(const PrefillArgs p) {
    using S = TileShape<D>;
    constexpr int kKeys = kBpWindowKeys;
    constexpr int kStage = 2 * kKeys * S::kRowBytes;
    extern __shared__ __align__(16) unsigned char memory[];
    griddep_sync();
    const AttentionArgs& a = p.a;
    const Segment g = segment_of(p, blockIdx.z);
    const int kv = blockIdx.y, choice = p.choices == 1 ? 0 : kv;
    const int first = blockIdx.x * kBpEntries, last = min(first + kBpEntries, g.rows * a.group) - 1;
    if (last < first) return;
    const int64_t first_row = static_cast<int64_t>(g.seq) * a.rows.query_length + g.t0;
    const uint32_t staged_q = smem_u32(memory), ring = staged_q + kBpEntries * S::kRowBytes;
    const unsigned char* key_rows = a.key_cache + g.seq * a.k_seq + kv * a.k_head;
    const unsigned char* value_rows = a.value_cache + g.seq * a.v_seq + kv * a.v_head;
    const int first_q = p.by_group.quotient(first), last_q = p.by_group.quotient(last);
    // keys [begin, end): the windows of the tile's rows
    const int begin = max(g.t0 + first_q - a.window + 1, 0), end = a.window > 0 ? g.t0 + last_q + 1 : begin;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int row_of[2], head_of[2], from[2], to[2], n[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int mine = first + 16 * warp + (lane >> 2) + 8 * i, entry = min(mine, last);
        row_of[i] = p.by_group.quotient(entry);
        head_of[i] = entry - row_of[i] * a.group;
        to[i] = g.t0 + row_of[i] + 1;
        from[i] = max(to[i] - a.window, 0);
        n[i] = a.top > 0 && mine <= last ? (reinterpret_cast<const int*>(g.base + p.plan.count) + choice * p.segment_rows)[row_of[i]] : 0;
    }
    for (int i = threadIdx.x; i < kBpEntries * S::kPieces; i += kBpThreads) {
        const int e = i / S::kPieces, piece = i - e * S::kPieces;
        const int entry = min(first + e, last);
        const int row = p.by_group.quotient(entry), head = entry - row * a.group;
        cp_async16_or_zero(staged_q + e * S::kRowBytes + 16 * piece,
                           a.query + (first_row + row) * a.q_row + (kv * a.group + head) * a.q_head + 16 * piece, first + e <= last);
    }
    cp_async_commit();
    auto request = [&](int at, int stage) {
        if (at < end) {
            request_rows<D, kKeys>(ring + stage * kStage, key_rows, a.k_row, at, end - at);
            request_rows<D, kKeys>(ring + stage * kStage + kKeys * S::kRowBytes, value_rows, a.v_row, at, end - at);
        }
        cp_async_commit();
    };
    request(begin, 0);

    Running<D> run;
    run.clear();
    const float* sums[2];
    const float2* stats[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t entry = ((static_cast<int64_t>(row_of[i]) * a.kv_heads + kv) * a.top) * a.group + head_of[i];
        stats[i] = reinterpret_cast<const float2*>(g.base + p.plan.stats) + entry;
        sums[i] = reinterpret_cast<const float*>(g.base + p.plan.sums) + entry * D + 4 * (lane & 3);
    }
    const int most = __reduce_max_sync(0xffffffffu, max(n[0], n[1]));
    const int chunks = (end - begin + kKeys - 1) / kKeys, rounds = max(chunks, most);
    uint32_t q[D / 16][4];
    int stage = 0;
    for (int round = 0; round < rounds; ++round) {
        // a pair's results are requested, then the window's next keys are worked on, then the results are joined
        float2 x[2];
        float4 v[2][D / 16];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = make_float2(kNegInf, 0.0f);
            if (round < n[i]) x[i] = __ldg(stats[i] + round * a.group);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                v[i][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (round < n[i]) v[i][c] = __ldg(reinterpret_cast<const float4*>(sums[i] + static_cast<int64_t>(round) * a.group * D + 16 * c));
            }
        }
        if (round < chunks) {
            const int at = begin + round * kKeys;
            request(at + kKeys, stage ^ 1);
            cp_async_wait_group1();
            __syncthreads();
            const unsigned char* staged_values = memory + kBpEntries * S::kRowBytes + stage * kStage + kKeys * S::kRowBytes;
            // keys that every row of the tile sees may hold anything
            const bool all = at >= g.t0 + last_q + 1 - a.window && at + kKeys <= g.t0 + first_q + 1;
            const bool careful = !all && __syncthreads_or(staged_not_finite<T, D, kKeys>(staged_values, threadIdx.x, kBpThreads));
            if (round == 0) load_queries<D>(q, staged_q + 16 * warp * S::kRowBytes, a.flip);
            const int low[2] = {from[0] - at, from[1] - at}, high[2] = {to[0] - at, to[1] - at};
            // a warp none of whose rows sees these keys passes
            if (__any_sync(0xffffffffu, high[1] > 0 && low[0] < kKeys))
                take_keys<T, D, kKeys, true>(run, q, ring + stage * kStage, ring + stage * kStage + kKeys * S::kRowBytes, low, high,
                                             a.scale_log2, careful, {true, true}, staged_values);
            __syncthreads();
            stage ^= 1;
        }
        if (round < most)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float next = fmaxf(run.m[i], x[i].x);
                const float base = next == kNegInf ? 0.0f : next;
                const float grow = power2(run.m[i] - base), w = power2(x[i].x - base);
                run.m[i] = next;
                // the other three lanes of a row hold their own part of the window's sum: here one of them counts
                run.l[i] = run.l[i] * grow + ((lane & 3) == 0 ? x[i].y * w : 0.0f);
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    run.acc[2 * c][2 * i] = fmaf(v[i][c].x, w, run.acc[2 * c][2 * i] * grow);
                    run.acc[2 * c][2 * i + 1] = fmaf(v[i][c].y, w, run.acc[2 * c][2 * i + 1] * grow);
                    run.acc[2 * c + 1][2 * i] = fmaf(v[i][c].z, w, run.acc[2 * c + 1][2 * i] * grow);
                    run.acc[2 * c + 1][2 * i + 1] = fmaf(v[i][c].w, w, run.acc[2 * c + 1][2 * i + 1] * grow);
                }
            }
    }
    cp_async_wait_all();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        run.l[i] += __shfl_xor_sync(0xffffffffu, run.l[i], 1);
        run.l[i] += __shfl_xor_sync(0xffffffffu, run.l[i], 2);
        if (first + 16 * warp + (lane >> 2) + 8 * i > last) continue;
        const int64_t to_row = (first_row + row_of[i]) * a.heads + kv * a.group + head_of[i];
        const float scale = run.l[i] == 0.0f ? 0.0f : 1.0f / (run.l[i] * kWeightFactor<T>);
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<uint32_t*>(a.out + (to_row * D + 8 * c + 2 * (lane & 3)) * 2) =
                pack2<T>(run.l[i] == 0.0f ? 0.0f : run.acc[c][2 * i] * scale, run.l[i] == 0.0f ? 0.0f : run.acc[c][2 * i + 1] * scale);
        if ((lane & 3) == 0) a.lse[to_row] = run.l[i] == 0.0f ? kNegInf : (run.m[i] + log2f(run.l[i])) * kLn2;
    }
}

int64_t up16(int64_t v) { return (v + 15) & ~int64_t{15}; }

// Rows a segment: as many as give a block some two tiles (a tile that is not full is time lost, a long segment's sort is
// one CTA's work), fewer where the partial results of so many would not fit the workspace.
int rows_a_segment(const AttentionArgs& a, int width) {
    const int64_t bins = (static_cast<int64_t>(a.rows.query_length) + a.block_size - 1) / a.block_size;
    int64_t rows = a.top > 0 ? 2 * kBpTile * bins / (static_cast<int64_t>(a.top) * a.group) : kBpSegment;
    if (rows < 512) rows = 512;
    if (rows > kBpSegment) rows = kBpSegment;
    const int64_t per_seq = (a.rows.query_length + rows - 1) / rows;              // equal parts of a sequence
    rows = (a.rows.query_length + per_seq - 1) / per_seq;
    const int64_t row_bytes = static_cast<int64_t>(a.top) * a.heads * (4 * width + 8);
    if (row_bytes > 0 && rows > kBpWorkspace / row_bytes) rows = kBpWorkspace / row_bytes;
    return static_cast<int>(rows);
}

PrefillArgs plan_of(const AttentionArgs& a, int width) {
    PrefillArgs p{};
    p.a = a;
    p.segment_rows = rows_a_segment(a, width);
    p.segments_per_seq = (a.rows.query_length + p.segment_rows - 1) / p.segment_rows;
    p.choices = a.i_head == 0 ? 1 : a.kv_heads;
    p.by_group = Divisor(static_cast<uint32_t>(a.group));
    p.bins = (a.rows.query_length + a.block_size - 1) / a.block_size;
    const int64_t rows = p.segment_rows, pairs = rows * a.top;
    p.max_tiles = static_cast<int>((pairs * a.group + kBpTile - 1) / kBpTile + p.bins);
    SegmentPlan& s = p.plan;
    int64_t at = 0;
    s.sums = at; at += up16(pairs * a.heads * width * 4);
    s.stats = at; at += up16(pairs * a.heads * 8);
    s.pairs = at; at += up16(pairs * p.choices * 4);
    s.kept = at; at += a.top > kBpHeldBlocks ? up16(pairs * p.choices * 4) : 0;
    s.count = at; at += up16(rows * p.choices * 4);
    s.tiles = at; at += static_cast<int64_t>(p.max_tiles) * p.choices * sizeof(Tile);
    s.tile_count = at; at += up16(p.choices * 4);
    s.total = (at + 255) & ~int64_t{255};
    return p;
}

template <typename T, int D, int kKeys>
int launch_tiles(const PrefillArgs& p, int segments, void* stream) {
    const dim3 grid(p.max_tiles, p.a.kv_heads, segments);
    if constexpr (D % 64 == 0) {
        if (p.a.block_size <= kKeys) {
            constexpr int smem = TensorTile<D, kKeys>::kBytes;
            if (int rc = allow_large_smem(reinterpret_cast<const void*>(&block_attention_tensor_tiles_kernel<T, D, kKeys>), kSmemDynamicLimit)) return rc;
            launch_kernel(block_attention_tensor_tiles_kernel<T, D, kKeys>, grid, dim3(kTtRows), smem, stream, p);
            count_launch();
            return check_launch("block_attention_tensor_tiles_kernel");
        }
    }
    if constexpr (D % 64 != 0 || kKeys == 64) {    // widths 64 and 128: only blocks of more keys than that come here
        constexpr int smem = (2 * kBpEntries + 2 * kKeys) * TileShape<D>::kRowBytes;
        if (smem > 48 * 1024)
            if (int rc = allow_large_smem(reinterpret_cast<const void*>(&block_attention_tiles_kernel<T, D, kKeys>), kSmemDynamicLimit)) return rc;
        launch_kernel(block_attention_tiles_kernel<T, D, kKeys>, grid, dim3(kBpThreads), smem, stream, p);
        count_launch();
    }
    return check_launch("block_attention_tiles_kernel");
}

template <typename T, int D>
int launch_passes(PrefillArgs& p, int64_t workspace_bytes, void* stream) {
    const int segments = p.segments_per_seq * p.a.rows.n_seq;
    const int64_t fit = p.a.top > 0 ? workspace_bytes / p.plan.total : segments;
    const int at_once = static_cast<int>(fit < segments ? (fit < 65535 ? fit : 65535) : (segments < 65535 ? segments : 65535));
    constexpr int window_smem = (kBpEntries + 4 * kBpWindowKeys) * TileShape<D>::kRowBytes;
    if (int rc = allow_large_smem(reinterpret_cast<const void*>(&block_attention_window_kernel<T, D>), kSmemDynamicLimit)) return rc;
    for (p.first_segment = 0; p.first_segment < segments; p.first_segment += at_once) {
        const int n = segments - p.first_segment < at_once ? segments - p.first_segment : at_once;
        if (p.a.top > 0) {
            const int smem = p.bins * 4;
            const auto sort = p.a.top <= 4 ? block_attention_sort_kernel<4> : p.a.top <= 8 ? block_attention_sort_kernel<8>
                              : p.a.top <= 16 ? block_attention_sort_kernel<16> : block_attention_sort_kernel<0>;
            if (smem > 48 * 1024)
                if (int rc = allow_large_smem(reinterpret_cast<const void*>(sort), kSmemDynamicLimit)) return rc;
            launch_kernel(sort, dim3(p.choices, n), dim3(kBpSortThreads), smem, stream, p);
            count_launch();
            if (int rc = check_launch("block_attention_sort_kernel")) return rc;
            int rc;
            if (p.a.block_size <= 16) rc = launch_tiles<T, D, 16>(p, n, stream);
            else if (p.a.block_size <= 32) rc = launch_tiles<T, D, 32>(p, n, stream);
            else rc = launch_tiles<T, D, 64>(p, n, stream);
            if (rc) return rc;
        }
        const int tiles = (p.segment_rows * p.a.group + kBpEntries - 1) / kBpEntries;
        launch_kernel(block_attention_window_kernel<T, D>, dim3(tiles, p.a.kv_heads, n), dim3(kBpThreads), window_smem, stream, p);
        count_launch();
        if (int rc = check_launch("block_attention_window_kernel")) return rc;
    }
    return RLM_OK;
}

template <typename T>
int launch_type(PrefillArgs& p, int width, int64_t workspace_bytes, void* stream) {
    switch (width) {
        case 32: return launch_passes<T, 32>(p, workspace_bytes, stream);
        case 64: return launch_passes<T, 64>(p, workspace_bytes, stream);
        case 96: return launch_passes<T, 96>(p, workspace_bytes, stream);
        default: return launch_passes<T, 128>(p, workspace_bytes, stream);
    }
}

}  // namespace

// The three passes cost some 20 us however short they are (the sort is one CTA's work, each pass waits for the one before):
// the per-row kernel is faster up to about a thousand (row, key head) tiles.  8 heads over 2, blocks of 64, four a row: 256
// rows 22 against 11 us, 1024 rows 23 against 34, 4096 rows 38 against 128; 24 over 8 of width 128: 256 rows 26 against 39.
bool prefill_passes(const AttentionArgs& a, int width, int dtype) {
    if (a.rows.position || a.rows.row_position || dtype == RLM_F32) return false;
    if (static_cast<int64_t>(a.rows.n_rows) * a.kv_heads * ((a.group + 15) / 16) <= 1024) return false;
    if ((a.rows.query_length + a.block_size - 1) / a.block_size > kBpMaxBins) return false;
    const int rows = rows_a_segment(a, width);           // few rows to a segment share few blocks
    return rows >= 256 || rows == a.rows.query_length;
}

int64_t prefill_workspace(const AttentionArgs& a, int width) {
    if (a.top == 0) return 0;
    const PrefillArgs p = plan_of(a, width);
    const int64_t segments = static_cast<int64_t>(p.segments_per_seq) * a.rows.n_seq;
    int64_t at_once = kBpWorkspace / p.plan.total;
    if (at_once < 1) at_once = 1;
    if (at_once > 65535) at_once = 65535;
    return p.plan.total * (at_once < segments ? at_once : segments);
}

int launch_prefill(const AttentionArgs& a, int width, int dtype, unsigned char* workspace, int64_t workspace_bytes, void* stream) {
    PrefillArgs p = plan_of(a, width);
    p.workspace = workspace;
    if (dtype == RLM_BF16) return launch_type<__nv_bfloat16>(p, width, workspace_bytes, stream);
    return launch_type<__half>(p, width, workspace_bytes, stream);
}

}  // namespace rlm
