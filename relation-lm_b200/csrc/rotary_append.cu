// Rotary positions on their way into the cache: queries and keys turned by their position, keys and values written into
// the cache rows of their positions, one launch.
//
//     angle(t, i) = t f_i,   (a, b) -> (a cos - b sin, b cos + a sin) magnitude,   i < R/2
//
// with (a, b) = (x_2i, x_2i+1) (interleaved) or (x_i, x_i+R/2); components R and up are copied.
//
// Every byte is read once and written once, so memory bounds it.  A CTA takes a few rows: it works out their cosines and
// sines once (all heads of a row share them) into shared memory, then walks the rows' 16-byte pieces.  The angle is a
// product in 64 bits, taken back to [-pi, pi] before it is rounded: in 32 bits a position of a million would be off by
// 0.03 rad.  8 x 4096 rows of 16 + 4 heads of 128 in 16 bits: 403 MB in 64.9 us, 95 % of the copy peak (72 with one piece a
// thread in flight, 76 with three, 78 with four, whose registers leave fewer threads); eight rows 2.4 us.
#include "block_attention.cuh"

namespace rlm {
namespace {

constexpr int kRaThreads = 256;
constexpr int kRaMaxRows = 32;

struct RotaryArgs {
    const unsigned char *query, *key, *value;
    unsigned char *query_out, *key_cache, *value_cache;
    const void* frequencies;
    Rows rows;
    int32_t* status;
    // strides in bytes
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    int64_t kc_seq, kc_row, kc_head, vc_seq, vc_row, vc_head;
    float magnitude;
    int heads, kv_heads, width, half;           // half: rotary / 2
    int frequency_is_double;
    int rows_per_cta;
    int turned_units, head_units;               // units of a head that turn, and all of them
    Divisor by_row, by_head;                    // units of a row, of a head
};

template <typename T> __device__ __forceinline__ float2 widen2(uint32_t v);
template <> __device__ __forceinline__ float2 widen2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 widen2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

template <typename T> __device__ __forceinline__ uint32_t narrow2(float a, float b);
template <> __device__ __forceinline__ uint32_t narrow2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t narrow2<__half>(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}

// The values of a 16-byte piece.
template <typename T> struct Piece {
    static constexpr int kCount = 16 / sizeof(T);
    float v[kCount];
    __device__ __forceinline__ explicit Piece(const uint4& raw) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
            } else {
                const float2 p = widen2<T>(w[i]);
                v[2 * i] = p.x;
                v[2 * i + 1] = p.y;
            }
        }
    }
    __device__ __forceinline__ uint4 raw() const {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
            else w[i] = narrow2<T>(v[2 * i], v[2 * i + 1]);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <typename T> __device__ __forceinline__ float load_one(const unsigned char* p);
template <> __device__ __forceinline__ float load_one<float>(const unsigned char* p) { return *reinterpret_cast<const float*>(p); }
template <> __device__ __forceinline__ float load_one<__nv_bfloat16>(const unsigned char* p) {
    return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
}
template <> __device__ __forceinline__ float load_one<__half>(const unsigned char* p) { return __half2float(*reinterpret_cast<const __half*>(p)); }
template <typename T> __device__ __forceinline__ void store_one(unsigned char* p, float v);
template <> __device__ __forceinline__ void store_one<float>(unsigned char* p, float v) { *reinterpret_cast<float*>(p) = v; }
template <> __device__ __forceinline__ void store_one<__nv_bfloat16>(unsigned char* p, float v) {
    *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ void store_one<__half>(unsigned char* p, float v) { *reinterpret_cast<__half*>(p) = __float2half_rn(v); }

// The work of a row in units: the heads of the query, of the key, of the value, head_units each.  With kWide a unit is a
// 16-byte piece, or the two pieces of a and b in the layout of halves; without, one pair or one copied component.
template <typename T, bool kInterleaved, bool kWide>
__global__ void __launch_bounds__(kRaThreads) rotary_append_kernel(const RotaryArgs a) {
    extern __shared__ float2 turn[];                     // [rows_per_cta][half]: cosine, sine
    __shared__ int seq_of[kRaMaxRows], at_of[kRaMaxRows];
    griddep_sync();
    const int first = blockIdx.x * a.rows_per_cta;
    const int n = min(a.rows_per_cta, a.rows.n_rows - first);
    if (static_cast<int>(threadIdx.x) < n) {
        int seq = 0, t = -1;
        if (!row_stands(a.rows, first + threadIdx.x, seq, t, a.status, blockIdx.y == 0)) t = -1;
        seq_of[threadIdx.x] = seq;
        at_of[threadIdx.x] = t;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * a.half; i += kRaThreads) {
        const int r = i / a.half, f = i - r * a.half;
        const int t = at_of[r];
        float2 cs = make_float2(0.0f, 0.0f);             // rows of padding turn into zeros
        if (t >= 0) {
            const double frequency = a.frequency_is_double ? static_cast<const double*>(a.frequencies)[f]
                                                           : static_cast<double>(static_cast<const float*>(a.frequencies)[f]);
            const double angle = static_cast<double>(t) * frequency;
            const double turns = rint(angle * 0.15915494309189535);
            // 2 pi as a sum of two doubles, so that the turns of a far position leave no error behind
            const double rest = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, angle));
            // sine and cosine of the angle rounded to 32 bits, then what the rounding left, to first order
            const float near = static_cast<float>(rest), left = static_cast<float>(rest - static_cast<double>(near));
            float s, c;
            sincosf(near, &s, &c);
            cs = make_float2(fmaf(-s, left, c) * a.magnitude, fmaf(c, left, s) * a.magnitude);
        }
        turn[i] = cs;
    }
    __syncthreads();
    constexpr int kVec = kWide ? 16 / static_cast<int>(sizeof(T)) : 1;
    constexpr int kAhead = kWide ? 2 : 1;                // units whose pieces are requested together
    const int units = n * static_cast<int>(a.by_row.d);
    const int half_bytes = a.half * static_cast<int>(sizeof(T));
    // where a unit's data lie: false for nothing to do (a row of padding leaves the caches alone)
    struct Unit {
        const unsigned char* src;
        unsigned char* dst;
        int row, unit;                                   // of the CTA's rows, of the head's units
        bool live, turns;
    };
    auto unit_of = [&](int u) {
        Unit x;
        x.live = u < units;
        if (!x.live) u = 0;
        x.row = a.by_row.quotient(u);
        const int in_row = u - x.row * static_cast<int>(a.by_row.d);
        const int head = a.by_head.quotient(in_row);
        x.unit = in_row - head * a.head_units;
        x.turns = x.unit < a.turned_units;
        const int t = at_of[x.row];
        const int64_t row = first + x.row, seq = seq_of[x.row];
        if (head < a.heads) {
            x.src = a.query + row * a.q_row + head * a.q_head;
            x.dst = a.query_out + (row * a.heads + head) * a.width * static_cast<int64_t>(sizeof(T));
        } else {
            x.live = x.live && t >= 0;
            const int g = head - a.heads, to = max(t, 0);
            if (g < a.kv_heads) {
                x.src = a.key + row * a.k_row + g * a.k_head;
                x.dst = a.key_cache + seq * a.kc_seq + to * a.kc_row + g * a.kc_head;
            } else {
                x.src = a.value + row * a.v_row + (g - a.kv_heads) * a.v_head;
                x.dst = a.value_cache + seq * a.vc_seq + to * a.vc_row + (g - a.kv_heads) * a.vc_head;
                x.turns = false;
            }
        }
        return x;
    };
    const int stride = gridDim.y * kRaThreads;
    for (int u0 = blockIdx.y * kRaThreads + threadIdx.x; u0 < units; u0 += kAhead * stride) {
        if constexpr (kWide) {
            Unit x[kAhead];
            uint4 lo[kAhead], hi[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                x[k] = unit_of(u0 + k * stride);
                // a piece of 8 or 4 consecutive components, or the pieces of a and of b in the layout of halves
                const bool two = !kInterleaved && x[k].unit < a.turned_units;
                const int column = kInterleaved || two ? x[k].unit * kVec : 2 * a.half + (x[k].unit - a.turned_units) * kVec;
                x[k].src += column * static_cast<int>(sizeof(T));
                x[k].dst += column * static_cast<int>(sizeof(T));
                lo[k] = hi[k] = make_uint4(0, 0, 0, 0);
                if (x[k].live && at_of[x[k].row] >= 0) { // rows of padding turn into zeros
                    lo[k] = *reinterpret_cast<const uint4*>(x[k].src);
                    if (two) hi[k] = *reinterpret_cast<const uint4*>(x[k].src + half_bytes);
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (!x[k].live) continue;
                if constexpr (kInterleaved) {
                    if (x[k].turns) {
                        Piece<T> p(lo[k]);
                        const float2* cs = turn + x[k].row * a.half + x[k].unit * (kVec / 2);
#pragma unroll
                        for (int i = 0; i < kVec / 2; ++i) {
                            const float2 w = cs[i];
                            const float y = p.v[2 * i], z = p.v[2 * i + 1];
                            p.v[2 * i] = y * w.x - z * w.y;
                            p.v[2 * i + 1] = z * w.x + y * w.y;
                        }
                        lo[k] = p.raw();
                    }
                } else if (x[k].turns) {
                    Piece<T> p(lo[k]), q(hi[k]);
                    const float2* cs = turn + x[k].row * a.half + x[k].unit * kVec;
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        const float2 w = cs[i];
                        const float y = p.v[i], z = q.v[i];
                        p.v[i] = y * w.x - z * w.y;
                        q.v[i] = z * w.x + y * w.y;
                    }
                    lo[k] = p.raw();
                    hi[k] = q.raw();
                }
                *reinterpret_cast<uint4*>(x[k].dst) = lo[k];
                if (!kInterleaved && x[k].unit < a.turned_units) *reinterpret_cast<uint4*>(x[k].dst + half_bytes) = hi[k];
            }
        } else {
            const Unit x = unit_of(u0);
            if (!x.live) continue;
            const bool blank = at_of[x.row] < 0;
            if (x.unit < a.turned_units) {
                const int ca = kInterleaved ? 2 * x.unit : x.unit, cb = kInterleaved ? 2 * x.unit + 1 : x.unit + a.half;
                float y = load_one<T>(x.src + ca * sizeof(T)), z = load_one<T>(x.src + cb * sizeof(T));
                if (x.turns) {
                    const float2 w = turn[x.row * a.half + x.unit];
                    const float p = y * w.x - z * w.y;
                    z = z * w.x + y * w.y;
                    y = p;
                }
                store_one<T>(x.dst + ca * sizeof(T), blank ? 0.0f : y);
                store_one<T>(x.dst + cb * sizeof(T), blank ? 0.0f : z);
            } else {
                const int c = 2 * a.half + x.unit - a.turned_units;
                store_one<T>(x.dst + c * sizeof(T), blank ? 0.0f : load_one<T>(x.src + c * sizeof(T)));
            }
        }
    }
}

template <typename T>
void launch_rotary(const RotaryArgs& a, bool interleaved, bool wide, dim3 grid, void* stream) {
    const size_t smem = static_cast<size_t>(a.rows_per_cta) * a.half * sizeof(float2);
    if (interleaved)
        launch_kernel(wide ? rotary_append_kernel<T, true, true> : rotary_append_kernel<T, true, false>, grid, dim3(kRaThreads), smem, stream, a);
    else
        launch_kernel(wide ? rotary_append_kernel<T, false, true> : rotary_append_kernel<T, false, false>, grid, dim3(kRaThreads), smem, stream, a);
}

}  // namespace
}  // namespace rlm

extern "C" int rlm_rotary_append(const void* query, const void* key, const void* value, void* query_out, void* key_cache,
                                 void* value_cache, const void* frequencies, const int64_t* position,
                                 const int32_t* row_batch, const int32_t* row_position, const int64_t* strides,
                                 float magnitude, int n_rows, int n_seq, int max_t, int query_length, int heads, int kv_heads,
                                 int width, int rotary, int interleaved, int dtype, int frequency_is_double,
                                 int32_t* status, void* stream) {
    using namespace rlm;
    RotaryArgs a{};
    a.rows = Rows{position, row_batch, row_position, n_rows, n_seq, query_length, max_t};
    if (!strides || (n_rows > 0 && (!query || !key || !value || !query_out || !key_cache || !value_cache || (rotary > 0 && !frequencies)))) {
        set_error("rotary_append: NULL argument");
        return RLM_ERR_NULL;
    }
    if (int rc = check_rows("rotary_append: row_batch and row_position come together",
                            "rotary_append: rows do not fit the sequences and positions of the caches", a.rows))
        return rc;
    if (!valid_dtype(dtype)) { set_error("rotary_append: unknown dtype"); return RLM_ERR_DTYPE; }
    if (heads < 1 || kv_heads < 1 || heads > 4096 || kv_heads > 4096 || width < 1 || width > 1024 || rotary < 0 ||
        rotary % 2 != 0 || rotary > width) {
        set_error("rotary_append: needs 1 to 4096 heads of width 1 to 1024 and an even rotary width within it");
        return RLM_ERR_SHAPE;
    }
    if (n_rows == 0) return RLM_OK;
    const int e = dtype_size(dtype);
    a.query = static_cast<const unsigned char*>(query);
    a.key = static_cast<const unsigned char*>(key);
    a.value = static_cast<const unsigned char*>(value);
    a.query_out = static_cast<unsigned char*>(query_out);
    a.key_cache = static_cast<unsigned char*>(key_cache);
    a.value_cache = static_cast<unsigned char*>(value_cache);
    a.frequencies = frequencies;
    a.status = status;
    int64_t* const to[12] = {&a.q_row, &a.q_head, &a.k_row, &a.k_head, &a.v_row, &a.v_head,
                             &a.kc_seq, &a.kc_row, &a.kc_head, &a.vc_seq, &a.vc_row, &a.vc_head};
    bool aligned = aligned16(query) && aligned16(key) && aligned16(value) && aligned16(query_out) && aligned16(key_cache) &&
                   aligned16(value_cache);
    const int extent[12] = {n_rows, heads, n_rows, kv_heads, n_rows, kv_heads, n_seq, max_t, kv_heads, n_seq, max_t, kv_heads};
    for (int i = 0; i < 12; ++i) {
        *to[i] = extent[i] > 1 ? strides[i] * e : 0;     // one of a kind has no step to the next
        aligned = aligned && *to[i] % 16 == 0;
    }
    a.magnitude = magnitude;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.width = width;
    a.half = rotary / 2;
    a.frequency_is_double = frequency_is_double;
    const int vec = 16 / e;
    const bool wide = aligned && width % vec == 0 && rotary % vec == 0 && (interleaved || a.half % vec == 0);
    if (wide) {
        a.turned_units = (interleaved ? rotary : a.half) / vec;
        a.head_units = a.turned_units + (width - rotary) / vec;
    } else {
        a.turned_units = a.half;
        a.head_units = a.half + width - rotary;
    }
    const int row_units = (heads + 2 * kv_heads) * a.head_units;
    // as many rows a CTA as give each thread about six units, while every SM has four CTAs (1237 rows of 8 + 2 heads of 64
    // 3.5 us, 4.7 while it has eight); one row over several CTAs
    // where the rows alone do not fill the SMs
    const int64_t sms = sm_count();
    int64_t per = (6 * kRaThreads + row_units - 1) / row_units;
    if (per > n_rows / (4 * sms)) per = n_rows / (4 * sms);
    if (per > kRaMaxRows) per = kRaMaxRows;
    while (per > 1 && per * a.half > 4096) --per;
    if (per < 1) per = 1;
    a.rows_per_cta = static_cast<int>(per);
    a.by_row = Divisor(static_cast<uint32_t>(row_units));
    a.by_head = Divisor(static_cast<uint32_t>(a.head_units));
    const int64_t ctas = (n_rows + per - 1) / per;
    int64_t split = (per * row_units + kRaThreads - 1) / kRaThreads;
    if (split > 2 * sms / ctas) split = 2 * sms / ctas;
    if (split < 1) split = 1;
    const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>(split));
    if (dtype == RLM_F32) launch_rotary<float>(a, interleaved != 0, wide, grid, stream);
    else if (dtype == RLM_BF16) launch_rotary<__nv_bfloat16>(a, interleaved != 0, wide, grid, stream);
    else launch_rotary<__half>(a, interleaved != 0, wide, grid, stream);
    count_launch();
    return check_launch("rotary_append_kernel");
}
