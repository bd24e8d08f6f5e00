// prompt_api.hip - the extern "C" entry points around a prompt: argument checks, then the kernels'
// launchers in kv_assign.hip, rope.hip, prompt_attention.hip and linear_i8.hip.
#include "decode.h"
#include <cmath>

namespace spinn {
namespace {

bool assign_ok(const SpinnHipKvAssignDesc *d) {
    if (!d || d->reserved != 0 || d->seqs < 0 || d->seqs > SPINN_HIP_ASSIGN_MAX_SEQS) return false;
    if (d->page_size <= 0 || d->n_pages <= 0 || d->max_pages <= 0 || d->max_tokens < 0 || d->max_tokens > (1 << 28)) return false;
    return d->n_pages <= (1 << 29) && (int64_t)d->max_pages * d->page_size <= (int64_t)INT32_MAX - 1024;
}

// What the table of frequencies depends on.
bool rope_table_ok(const SpinnHipRopeDesc *d) {
    if (!d || d->rot_dim < 2 || d->rot_dim > SPINN_HIP_ROPE_MAX_DIM || d->rot_dim % 2) return false;
    auto positive = [](float v) { return std::isfinite(v) && v > 0.f; };
    if (!positive(d->base) || !positive(d->factor)) return false;
    switch (d->scaling) {
    case SPINN_ROPE_PLAIN: return d->factor == 1.f;
    case SPINN_ROPE_LINEAR: return true;
    case SPINN_ROPE_BY_PARTS: return d->trained > 0 && std::isfinite(d->low) && std::isfinite(d->high) && d->low < d->high;
    default: return false;
    }
}

bool rope_ok(const SpinnHipRopeDesc *d) {
    if (!rope_table_ok(d) || !dtype_bytes(d->dtype) || d->heads <= 0 || d->head_dim < d->rot_dim) return false;
    if (d->head_dim > SPINN_HIP_ROPE_MAX_DIM || d->interleaved < 0 || d->interleaved > 1 || !std::isfinite(d->magnitude)) return false;
    if ((int64_t)d->heads * d->head_dim > (int64_t)1 << 30) return false;
    constexpr int64_t kFar = (int64_t)1 << 32;
    for (const int64_t s : {d->x_stride, d->y_stride, d->x_head_stride, d->y_head_stride})
        if (s < d->head_dim || s > kFar) return false;
    return true;
}

bool prompt_ok(const SpinnHipPromptAttentionDesc *d) {
    if (!d || !dtype_bytes(d->dtype) || d->reserved != 0 || d->seqs < 0 || d->heads <= 0 || d->kv_heads <= 0) return false;
    if (d->heads % d->kv_heads || d->head_dim <= 0 || d->head_dim > SPINN_HIP_KV_MAX_DIM) return false;
    if (d->causal < 0 || d->causal > 1 || d->q_rows < 0 || d->kv_rows < 0) return false;
    if (!(std::fabs(d->scale) <= 0x1p127f)) return false; // times log2 e it is still a number
    if (d->seqs > (1 << 24)) return false;
    // rows of (token, head) pairs and their tiles, and keys a tile behind the last, within 31 bits
    constexpr int64_t kMost = (int64_t)1 << 30;
    if ((int64_t)d->q_rows * d->heads > kMost || d->kv_rows > kMost) return false;
    const int64_t row = (int64_t)d->heads * d->head_dim, kv_row = (int64_t)d->kv_heads * d->head_dim;
    constexpr int64_t kFar = (int64_t)1 << 24; // a tile's rows lie within 32 bits of bytes
    return d->q_stride >= row && d->o_stride >= row && d->k_stride >= kv_row && d->v_stride >= kv_row && d->q_stride <= kFar &&
           d->o_stride <= kFar && d->k_stride <= kFar && d->v_stride <= kFar;
}

bool linear_i8_ok(const SpinnHipLinearI8Desc *d) {
    if (!d || d->m < 0 || d->n <= 0 || d->k <= 0 || d->k > SPINN_HIP_I8_MAX_K || !dtype_bytes(d->dtype)) return false;
    if (d->trans_w < 0 || d->trans_w > 1) return false;
    if (d->act != SPINN_LINEAR_NONE && d->act != SPINN_LINEAR_RELU && d->act != SPINN_LINEAR_SILU &&
        d->act != SPINN_LINEAR_GELU && d->act != SPINN_LINEAR_GELU_TANH)
        return false;
    // rows do not overlap; 0 = dense
    if ((d->ldx && d->ldx < (int64_t)round16(d->k)) || d->ldx % 16 || (d->ldres && d->ldres < d->n) || (d->ldy && d->ldy < d->n)) return false;
    constexpr int kMost = INT32_MAX - 1024;
    constexpr int64_t kFar = (int64_t)1 << 28;
    return d->m <= kMost && d->n <= kMost && d->ldx <= kFar && d->ldres <= kFar && d->ldy <= kFar;
}

// Descriptor with the dense strides filled in.
SpinnHipLinearI8Desc linear_i8_full(const SpinnHipLinearI8Desc *d) {
    SpinnHipLinearI8Desc f = *d;
    if (!f.ldx) f.ldx = (int64_t)round16(f.k);
    if (!f.ldres) f.ldres = f.n;
    if (!f.ldy) f.ldy = f.n;
    return f;
}

} // namespace
} // namespace spinn

using namespace spinn;

extern "C" {

int spinn_hip_kv_assign(const SpinnHipKvAssignDesc *d, const int32_t *new_tokens, const int32_t *lengths,
                        const int32_t *next_pos, const int32_t *held, const int32_t *free_count, int32_t *free_pages,
                        int32_t *page_table, int32_t *lengths_out, int32_t *next_out, int32_t *held_out,
                        int32_t *free_count_out, int32_t *starts, int32_t *served, int32_t *seq, int32_t *slot,
                        int32_t *position, void *stream) {
    if (!assign_ok(d)) return SPINN_HIP_EINVAL;
    if (d->seqs == 0) return SPINN_HIP_OK;
    if (!new_tokens || !lengths || !held || !free_count || !free_pages || !page_table || !lengths_out || !held_out ||
        !free_count_out || !starts || !served || (next_pos && !next_out))
        return SPINN_HIP_EINVAL;
    if (d->max_tokens > 0 && (!seq || !slot)) return SPINN_HIP_EINVAL;
    return kv_assign(d, new_tokens, lengths, next_pos, held, free_count, free_pages, page_table, lengths_out, next_out, held_out,
                     free_count_out, starts, served, seq, slot, position, (hipStream_t)stream);
}

size_t spinn_hip_rope_table_size(const SpinnHipRopeDesc *d) { return rope_table_ok(d) ? (size_t)d->rot_dim / 2 * 8 : 0; }

int spinn_hip_rope_table(const SpinnHipRopeDesc *d, void *table, void *stream) {
    if (!rope_table_ok(d) || !table || !aligned16(table)) return SPINN_HIP_EINVAL;
    return rope_table(d, table, (hipStream_t)stream);
}

int spinn_hip_rope(const SpinnHipRopeDesc *d, int64_t tokens, const int32_t *position, const void *table, const void *x,
                   void *y, void *stream) {
    if (!rope_ok(d) || tokens < 0 || tokens > (1 << 28)) return SPINN_HIP_EINVAL;
    if (tokens == 0) return SPINN_HIP_OK;
    if (!position || !table || !x || !y || !aligned16(table)) return SPINN_HIP_EINVAL;
    const size_t e = dtype_bytes(d->dtype);
    if (!multiple_of(x, e) || !multiple_of(y, e)) return SPINN_HIP_EINVAL;
    if (x == y && (d->x_stride != d->y_stride || d->x_head_stride != d->y_head_stride)) return SPINN_HIP_EINVAL;
    return rope_run(d, tokens, position, table, x, y, (hipStream_t)stream);
}

size_t spinn_hip_prompt_attention_workspace_size(const SpinnHipPromptAttentionDesc *d) {
    return prompt_ok(d) && d->seqs && d->q_rows ? prompt_attention_workspace_bytes(d) : 0;
}

int spinn_hip_prompt_attention(const SpinnHipPromptAttentionDesc *d, const void *q, const void *k, const void *v,
                               const int32_t *starts, const int32_t *kv_starts, void *o, float *lse, void *workspace,
                               size_t workspace_bytes, void *stream) {
    if (!prompt_ok(d)) return SPINN_HIP_EINVAL;
    if (!kv_starts && d->q_rows != d->kv_rows) return SPINN_HIP_EINVAL;
    if (d->seqs == 0 || d->q_rows == 0) return SPINN_HIP_OK;
    if (!q || !starts || !o || (d->kv_rows > 0 && (!k || !v)) || o == q || o == k || o == v) return SPINN_HIP_EINVAL;
    const size_t e = dtype_bytes(d->dtype);
    if (!multiple_of(q, e) || !multiple_of(k, e) || !multiple_of(v, e) || !multiple_of(o, e)) return SPINN_HIP_EINVAL;
    if (!workspace_ok(workspace, workspace_bytes, prompt_attention_workspace_bytes(d))) return SPINN_HIP_EWORKSPACE;
    return prompt_attention(d, q, k, v, starts, kv_starts, o, lse, workspace, (hipStream_t)stream);
}

int spinn_hip_quantize_rows(int32_t dtype, int64_t rows, int32_t k, const void *x, int64_t ldx, int8_t *xq, int64_t ldq,
                            float *scale, void *stream) {
    constexpr int64_t kFar = (int64_t)1 << 28;
    if (!dtype_bytes(dtype) || rows < 0 || rows > ((int64_t)1 << 31) || k <= 0 || k > INT32_MAX - 1024) return SPINN_HIP_EINVAL;
    if (ldx < k || ldq < k || ldq % 16 || ldx > kFar || ldq > kFar) return SPINN_HIP_EINVAL;
    if (rows == 0) return SPINN_HIP_OK;
    if (!x || !xq || !scale || !aligned16(xq) || !multiple_of(x, dtype_bytes(dtype))) return SPINN_HIP_EINVAL;
    return quantize_rows(dtype, rows, k, x, ldx, xq, ldq, scale, (hipStream_t)stream);
}

size_t spinn_hip_linear_i8_packed_size(const SpinnHipLinearI8Desc *d) { return linear_i8_ok(d) ? linear_i8_packed_bytes(d) : 0; }

size_t spinn_hip_linear_i8_workspace_size(const SpinnHipLinearI8Desc *d) {
    return linear_i8_ok(d) && d->m ? linear_i8_workspace_bytes(d) : 0;
}

int spinn_hip_linear_i8_pack_weights(const SpinnHipLinearI8Desc *d, const int8_t *w, void *packed_w, void *stream) {
    if (!linear_i8_ok(d) || !w || !packed_w || !aligned16(packed_w)) return SPINN_HIP_EINVAL;
    return linear_i8_pack(d, w, packed_w, (hipStream_t)stream);
}

int spinn_hip_linear_i8(const SpinnHipLinearI8Desc *d, const int8_t *x, const float *x_scale, const void *packed_w,
                        const float *w_scale, const void *bias, const void *residual, void *y, void *workspace,
                        size_t workspace_bytes, void *stream) {
    if (!linear_i8_ok(d)) return SPINN_HIP_EINVAL;
    if (d->m == 0) return SPINN_HIP_OK;
    if (!x || !x_scale || !packed_w || !w_scale || !y || y == (const void *)x) return SPINN_HIP_EINVAL;
    const SpinnHipLinearI8Desc f = linear_i8_full(d);
    const size_t e = dtype_bytes(f.dtype);
    if (!aligned16(x) || !aligned16(packed_w) || !multiple_of(x_scale, 4) || !multiple_of(w_scale, 4) || !multiple_of(bias, e) ||
        !multiple_of(residual, e) || !multiple_of(y, e))
        return SPINN_HIP_EINVAL;
    if (residual == y && f.ldres != f.ldy && f.m > 1) return SPINN_HIP_EINVAL;
    if (!workspace_ok(workspace, workspace_bytes, linear_i8_workspace_bytes(&f))) return SPINN_HIP_EWORKSPACE;
    return linear_i8_run(&f, x, x_scale, packed_w, w_scale, bias, residual, y, workspace, (hipStream_t)stream);
}

} // extern "C"
