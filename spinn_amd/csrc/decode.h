// decode.h - declarations and element types shared by the decoding-step operators
// (linear.hip, kv_attention.hip, kv_evict.hip, beam.hip).
#pragma once
#include "spinn_hip_internal.h"

namespace spinn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 16 bytes of a matrix operand per lane, a fragment of 16 rows or columns by kFrag<T> k:
// lane l holds row l%16, k = (16 / sizeof(T)) * (l/16) + 0.. . For 16-bit types that is
// one v_mfma_f32_16x16x32 operand; for fp32 element e of every lane feeds the e-th of four
// v_mfma_f32_16x16x4_f32 (k = l/16 there: the four take k in another order, the same
// for both operands). Accumulator element r of lane l is D[4*(l/16) + r][l%16].
template <class T>
constexpr int kFrag = 64 / (int)sizeof(T);

__device__ __forceinline__ void mfma_frag(f32x4 &c, u32x4 a, u32x4 b, float) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, (uint32_t)a[e]),
                                                 __builtin_bit_cast(float, (uint32_t)b[e]), c, 0, 0, 0);
}
__device__ __forceinline__ void mfma_frag(f32x4 &c, u32x4 a, u32x4 b, _Float16) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mfma_frag(f32x4 &c, u32x4 a, u32x4 b, __bf16) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The bits of an element, for copies and transposes.
template <class T>
struct Bits;
template <>
struct Bits<float> {
    typedef uint32_t type;
};
template <>
struct Bits<_Float16> {
    typedef uint16_t type;
};
template <>
struct Bits<__bf16> {
    typedef uint16_t type;
};

// 16 bytes at p, element by element: those from `left` on (elements to the row's end) are zero.
template <class T>
__device__ __forceinline__ u32x4 load_edge(const T *p, int left) {
    typedef typename Bits<T>::type B;
    constexpr int N = 16 / sizeof(T);
    u32x4 r = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < left) {
            const uint32_t b = (uint32_t) reinterpret_cast<const B *>(p)[i];
            if constexpr (N == 4) r[i] = b;
            else r[i / 2] |= b << (16 * (i % 2));
        }
    return r;
}

// N elements from d0 on of a row of `dim` >= N, zeros behind its end, from rows of any alignment: one load, which at the
// row's end starts early enough to stay inside, and a shift (17 sequences of 12724 to 28547 slots, 8 heads of 33,
// bf16: 266 us, element by element 756).
template <class T, int N>
__device__ __forceinline__ void load_loose(const T *row, int d0, int dim, uint32_t (&to)[N * sizeof(T) / 4]) {
    constexpr int W = N * sizeof(T) / 4;
    typedef uint32_t Words __attribute__((ext_vector_type(W)));
    typedef Words Loose __attribute__((aligned(sizeof(T))));
    const int at = min(d0, dim - N), skip = (d0 - at) * (int)sizeof(T) * 8; // bits of elements before d0
    const Words w = *reinterpret_cast<const Loose *>(row + at);
    if constexpr (W == 2) {
        const uint64_t v = __builtin_bit_cast(uint64_t, w);
        const uint64_t r = skip < 64 ? v >> skip : 0ull;
        to[0] = (uint32_t)r;
        to[1] = (uint32_t)(r >> 32);
    } else {
        static_assert(W == 4, "");
        const uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
        const int s = skip & 63;
        const uint64_t both = s ? lo >> s | hi << (64 - s) : lo, top = hi >> s;
        const uint64_t r0 = skip < 64 ? both : (skip < 128 ? top : 0ull), r1 = skip < 64 ? top : 0ull;
        to[0] = (uint32_t)r0;
        to[1] = (uint32_t)(r0 >> 32);
        to[2] = (uint32_t)r1;
        to[3] = (uint32_t)(r1 >> 32);
    }
}

// How rows are read.
enum Rows {
    kRuns,  // they are whole, aligned 16-byte runs
    kLoose, // of any length from 16 bytes on and any alignment: load_loose
    kShort, // shorter: load_edge
    kLaidOut // not where they are: as operand granules in the workspace (linear.hip)
};

inline int dtype_bytes(int dtype) {
    return dtype == ENNF_TYPE_FLOAT32 ? 4 : (dtype == ENNF_TYPE_FLOAT16 || dtype == ENNF_TYPE_BFLOAT16 ? 2 : 0);
}

// f(T()) for the element type of `dtype` (checked before).
template <class F>
int with_dtype(int dtype, F f) {
    switch (dtype) {
    case ENNF_TYPE_FLOAT32: return f(float());
    case ENNF_TYPE_FLOAT16: return f(_Float16());
    case ENNF_TYPE_BFLOAT16: return f(__bf16());
    default: return SPINN_HIP_EINVAL;
    }
}

// A launch has at most 2^32 threads; one of more wraps without an error and leaves the rest undone.
inline bool launch_fits(int64_t blocks, int64_t threads) { return blocks <= (int64_t)UINT32_MAX / threads; }

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
inline size_t round16(size_t v) { return (v + 15) & ~(size_t)15; }

// linear.hip
size_t linear_packed_bytes(const SpinnHipLinearDesc *d);
size_t linear_workspace_bytes(const SpinnHipLinearDesc *d);
int linear_pack(const SpinnHipLinearDesc *d, const void *w, void *packed, hipStream_t st);
int linear_run(const SpinnHipLinearDesc *d, const void *x, const void *packed, const void *bias, const void *res,
               void *y, void *ws, hipStream_t st);

// kv_attention.hip
int kv_append(const SpinnHipKvDesc *d, int64_t tokens, const int32_t *seq, const int32_t *slot, const int32_t *position,
              const void *k, int64_t k_stride, const void *v, int64_t v_stride, const int32_t *table, void *k_pages,
              void *v_pages, float *acc, int32_t *pos, int64_t acc_stride, hipStream_t st);
size_t kv_attention_workspace_bytes(const SpinnHipKvAttentionDesc *d);
int kv_attention(const SpinnHipKvAttentionDesc *d, const void *q, const void *k, const void *v, const int32_t *table,
                 const int32_t *lengths, const uint8_t *mask, const float *acc, float *acc_out, void *o, float *lse,
                 void *ws, hipStream_t st);

// kv_evict.hip
size_t kv_evict_workspace_bytes(const SpinnHipKvEvictDesc *d);
int kv_evict(const SpinnHipKvEvictDesc *d, const int32_t *table, const int32_t *lengths, const int32_t *next_pos,
             const float *acc, const int32_t *pos, float *acc_out, int32_t *pos_out, int32_t *lengths_out, void *k,
             void *v, void *ws, hipStream_t st);

// beam.hip
size_t beam_select_workspace_bytes(const SpinnHipBeamDesc *d);
int beam_select(const SpinnHipBeamDesc *d, const void *logits, const float *scores, const uint8_t *finished,
                float *out_scores, int32_t *out_parents, int32_t *out_tokens, void *ws, hipStream_t st);
int beam_reorder(const SpinnHipBeamState *states, int n, int batch, int beams, int k, const int32_t *parents,
                 hipStream_t st);

} // namespace spinn
