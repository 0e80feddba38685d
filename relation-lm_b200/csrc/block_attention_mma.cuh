// What the kernels of block_attention share: the arguments of a call, the warp-level tensor instruction and its operands,
// stores of one value.
#pragma once

#include <type_traits>

#include "block_attention.cuh"

namespace rlm {

constexpr int kBaMaxTop = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttentionArgs {
    const unsigned char *query, *key_cache, *value_cache;
    const int32_t* index;
    unsigned char* out;
    float* lse;
    Rows rows;
    int32_t* status;
    int64_t q_row, q_head, k_seq, k_row, k_head, v_seq, v_row, v_head;     // bytes
    int64_t i_row, i_head;                                                 // elements
    int heads, kv_heads, group, head_tiles, top, block_size, window;
    int splits;
    float scale_log2;                  // |scale| x log2(e): the softmax runs on powers of two
    uint32_t flip;                     // sign bits that turn a 16-bit query's components where the scale is negative
};

// Whole sequences in three passes (block_attention_prefill.cu); false where the per-row kernels serve.
bool prefill_passes(const AttentionArgs& a, int width, int dtype);
int64_t prefill_workspace(const AttentionArgs& a, int width);
int launch_prefill(const AttentionArgs& a, int width, int dtype, unsigned char* workspace, int64_t workspace_bytes, void* stream);

namespace {

// 2^x: two units in the last place, results below the smallest normal number are zero.
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}

// Softmax weights (powers of two of at most zero) as operands of the tensor cores are rounded to 16 bits: half a step, 2^-8 (bf16)
// or 2^-11 (fp16) of each weight, beside the same rounding of the result; twice the bits would take twice the products.
// In fp16 weights below 2^-14 would lose bits and those below 2^-25 vanish, however many or however large their values are,
// so there they are carried 2^15-fold: all bits down to 2^-29 of the largest, some down to 2^-39.  The sums take the factor out again.
template <typename T> constexpr float kWeightFactor = std::is_same<T, __half>::value ? 32768.0f : 1.0f;
template <typename T> __device__ __forceinline__ uint32_t pack_weights(float a, float b) {
    return pack2<T>(a * kWeightFactor<T>, b * kWeightFactor<T>);
}

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes, or zeros without a read where `live` is false.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool live) {
    const int bytes = live ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_cluster(uint32_t local, int rank) {
    uint32_t remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
    return v;
}
__device__ __forceinline__ int load_cluster_int(uint32_t local, int rank) { return __float_as_int(load_cluster(local, rank)); }
__device__ __forceinline__ double load_cluster_double(uint32_t local, int rank) {
    uint32_t remote;
    double v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(remote) : "memory");
    return v;
}

template <typename T> __device__ __forceinline__ float load_value(const void* p);
template <> __device__ __forceinline__ float load_value<__nv_bfloat16>(const void* p) { return __bfloat162float(*static_cast<const __nv_bfloat16*>(p)); }
template <> __device__ __forceinline__ float load_value<__half>(const void* p) { return __half2float(*static_cast<const __half*>(p)); }
template <typename T> __device__ __forceinline__ void store_value(unsigned char* row, int column, float v);
template <> __device__ __forceinline__ void store_value<float>(unsigned char* row, int column, float v) {
    reinterpret_cast<float*>(row)[column] = v;
}
template <> __device__ __forceinline__ void store_value<__nv_bfloat16>(unsigned char* row, int column, float v) {
    reinterpret_cast<__nv_bfloat16*>(row)[column] = __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ void store_value<__half>(unsigned char* row, int column, float v) {
    reinterpret_cast<__half*>(row)[column] = __float2half_rn(v);
}

}  // namespace
}  // namespace rlm
