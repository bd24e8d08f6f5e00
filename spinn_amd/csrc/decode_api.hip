// decode_api.hip - the extern "C" entry points of the decoding step: argument checks, then
// the kernels' launchers in linear.hip, kv_attention.hip, kv_evict.hip and beam.hip.
#include "decode.h"

namespace spinn {
namespace {

bool linear_ok(const SpinnHipLinearDesc *d) {
    if (!d || d->m < 0 || d->n <= 0 || d->k <= 0 || !dtype_bytes(d->dtype) || d->reserved != 0) return false;
    if (d->trans_w < 0 || d->trans_w > 1 || d->x_unaligned < 0 || d->x_unaligned > 1) return false;
    if (d->act != SPINN_LINEAR_NONE && d->act != SPINN_LINEAR_RELU && d->act != SPINN_LINEAR_SILU &&
        d->act != SPINN_LINEAR_GELU && d->act != SPINN_LINEAR_GELU_TANH)
        return false;
    // rows do not overlap; 0 = dense
    if ((d->ldx && d->ldx < d->k) || (d->ldres && d->ldres < d->n) || (d->ldy && d->ldy < d->n)) return false;
    // tile counts and padded sizes stay within 31 bits, byte offsets of x, residual and y within 62
    constexpr int kMost = INT32_MAX - 1024;
    constexpr int64_t kFar = (int64_t)1 << 28;
    return d->m <= kMost && d->n <= kMost && d->k <= kMost && d->ldx <= kFar && d->ldres <= kFar && d->ldy <= kFar;
}

// Descriptor with the dense strides filled in.
SpinnHipLinearDesc linear_full(const SpinnHipLinearDesc *d) {
    SpinnHipLinearDesc f = *d;
    if (!f.ldx) f.ldx = f.k;
    if (!f.ldres) f.ldres = f.n;
    if (!f.ldy) f.ldy = f.n;
    return f;
}

bool kv_ok(const SpinnHipKvDesc *d) {
    if (!d || !dtype_bytes(d->dtype) || d->reserved != 0) return false;
    if (d->seqs < 0 || d->kv_heads <= 0 || d->head_dim <= 0 || d->head_dim > SPINN_HIP_KV_MAX_DIM) return false;
    if (d->page_size <= 0 || d->n_pages <= 0 || d->max_pages <= 0) return false;
    if ((int64_t)d->max_pages * d->page_size > (int64_t)INT32_MAX - 1024) return false;
    if ((int64_t)d->seqs * d->kv_heads > (int64_t)INT32_MAX / 2) return false;
    // byte offsets within 62 bits
    constexpr int64_t kFar = (int64_t)1 << 45;
    if (d->page_stride < d->head_dim || d->head_stride < d->head_dim || d->slot_stride < d->head_dim) return false;
    return d->page_stride <= kFar / d->n_pages && d->head_stride <= kFar / d->kv_heads &&
           d->slot_stride <= kFar / d->page_size;
}

bool attention_ok(const SpinnHipKvAttentionDesc *d) {
    if (!d || !kv_ok(&d->kv) || d->heads <= 0 || d->heads % d->kv.kv_heads) return false;
    if (d->max_len < 0 || (int64_t)d->max_len > (int64_t)d->kv.max_pages * d->kv.page_size) return false;
    if (d->accumulate < 0 || d->accumulate > 1) return false;
    const int64_t row = (int64_t)d->heads * d->kv.head_dim;
    constexpr int64_t kFar = (int64_t)1 << 40;
    if (d->q_stride < row || d->o_stride < row || d->q_stride > kFar || d->o_stride > kFar) return false;
    if ((int64_t)d->kv.seqs * d->heads > (int64_t)INT32_MAX / 256) return false;
    if (d->accumulate && (d->acc_stride < d->max_len || d->acc_stride > kFar)) return false;
    return d->mask_stride >= 0 && d->mask_stride <= kFar;
}

bool evict_ok(const SpinnHipKvEvictDesc *d) {
    if (!d || !kv_ok(&d->kv) || d->budget < 0 || d->recent < 0 || d->sinks < 0 || d->max_len < 0) return false;
    if ((int64_t)d->max_len > (int64_t)d->kv.max_pages * d->kv.page_size) return false;
    constexpr int64_t kFar = (int64_t)1 << 40;
    return d->acc_stride >= d->max_len && d->acc_stride <= kFar;
}

bool beam_ok(const SpinnHipBeamDesc *d) {
    if (!d || !dtype_bytes(d->dtype) || d->batch < 0 || d->beams <= 0 || d->vocab <= 0 || d->k <= 0) return false;
    if (d->beams > SPINN_HIP_BEAM_MAX || d->k > SPINN_HIP_BEAM_MAX_K) return false;
    if ((int64_t)d->k > (int64_t)d->beams * d->vocab) return false;
    if (d->vocab > (1 << 28) || d->batch > (1 << 20)) return false;
    constexpr int64_t kFar = (int64_t)1 << 32;
    return d->logits_stride >= d->vocab && d->logits_stride <= kFar;
}

bool multiple_of(const void *p, size_t n) { return ((uintptr_t)p % n) == 0; }

bool workspace_ok(const void *ws, size_t bytes, size_t need) { return need == 0 || (ws && aligned16(ws) && bytes >= need); }

} // namespace
} // namespace spinn

using namespace spinn;

extern "C" {

size_t spinn_hip_linear_packed_size(const SpinnHipLinearDesc *d) { return linear_ok(d) ? linear_packed_bytes(d) : 0; }

size_t spinn_hip_linear_workspace_size(const SpinnHipLinearDesc *d) {
    if (!linear_ok(d) || d->m == 0) return 0;
    const SpinnHipLinearDesc f = linear_full(d);
    return linear_workspace_bytes(&f);
}

int spinn_hip_linear_pack_weights(const SpinnHipLinearDesc *d, const void *w, void *packed_w, void *stream) {
    if (!linear_ok(d) || !w || !packed_w) return SPINN_HIP_EINVAL;
    if (!aligned16(packed_w) || !multiple_of(w, dtype_bytes(d->dtype))) return SPINN_HIP_EINVAL;
    return linear_pack(d, w, packed_w, (hipStream_t)stream);
}

int spinn_hip_linear(const SpinnHipLinearDesc *d, const void *x, const void *packed_w, const void *bias,
                     const void *residual, void *y, void *workspace, size_t workspace_bytes, void *stream) {
    if (!linear_ok(d)) return SPINN_HIP_EINVAL;
    if (d->m == 0) return SPINN_HIP_OK;
    if (!x || !packed_w || !y || y == x) return SPINN_HIP_EINVAL;
    const SpinnHipLinearDesc f = linear_full(d);
    const size_t e = dtype_bytes(f.dtype);
    if (!multiple_of(x, f.x_unaligned ? e : 16) || !aligned16(packed_w) || !multiple_of(bias, e) ||
        !multiple_of(residual, e) || !multiple_of(y, e))
        return SPINN_HIP_EINVAL;
    if (residual == y && f.ldres != f.ldy && f.m > 1) return SPINN_HIP_EINVAL;
    if (!workspace_ok(workspace, workspace_bytes, linear_workspace_bytes(&f))) return SPINN_HIP_EWORKSPACE;
    return linear_run(&f, x, packed_w, bias, residual, y, workspace, (hipStream_t)stream);
}

int spinn_hip_kv_append(const SpinnHipKvDesc *d, int64_t tokens, const int32_t *seq, const int32_t *slot,
                        const int32_t *position, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                        const int32_t *page_table, void *k_pages, void *v_pages, float *acc, int32_t *pos,
                        int64_t acc_stride, void *stream) {
    if (!kv_ok(d) || tokens < 0 || tokens > (1 << 28)) return SPINN_HIP_EINVAL;
    const int64_t row = (int64_t)d->kv_heads * d->head_dim;
    constexpr int64_t kFar = (int64_t)1 << 32;
    if (row > (int64_t)1 << 30) return SPINN_HIP_EINVAL; // counted in 31 bits, a step of the workgroup behind its end too
    if (k_stride < row || v_stride < row || k_stride > kFar || v_stride > kFar) return SPINN_HIP_EINVAL;
    if (!seq && tokens > d->seqs) return SPINN_HIP_EINVAL;
    if ((acc || pos) && (acc_stride <= 0 || acc_stride > ((int64_t)1 << 40))) return SPINN_HIP_EINVAL;
    if (tokens == 0 || d->seqs == 0) return SPINN_HIP_OK;
    const size_t e = dtype_bytes(d->dtype);
    if (!slot || !k || !v || !page_table || !k_pages || !v_pages) return SPINN_HIP_EINVAL;
    if (!multiple_of(k, e) || !multiple_of(v, e) || !multiple_of(k_pages, e) || !multiple_of(v_pages, e))
        return SPINN_HIP_EINVAL;
    return kv_append(d, tokens, seq, slot, position, k, k_stride, v, v_stride, page_table, k_pages, v_pages, acc, pos,
                     acc_stride, (hipStream_t)stream);
}

size_t spinn_hip_kv_attention_workspace_size(const SpinnHipKvAttentionDesc *d) {
    return attention_ok(d) && d->kv.seqs ? kv_attention_workspace_bytes(d) : 0;
}

int spinn_hip_kv_attention(const SpinnHipKvAttentionDesc *d, const void *q, const void *k_pages, const void *v_pages,
                           const int32_t *page_table, const int32_t *lengths, const uint8_t *mask, const float *acc,
                           float *acc_out, void *o, float *lse, void *workspace, size_t workspace_bytes,
                           void *stream) {
    if (!attention_ok(d)) return SPINN_HIP_EINVAL;
    if (mask && d->mask_stride < d->max_len) return SPINN_HIP_EINVAL;
    if (d->kv.seqs == 0) return SPINN_HIP_OK;
    if (!q || !k_pages || !v_pages || !page_table || !lengths || !o) return SPINN_HIP_EINVAL;
    if (d->accumulate && (!acc || !acc_out)) return SPINN_HIP_EINVAL;
    const size_t e = dtype_bytes(d->kv.dtype);
    if (!multiple_of(q, e) || !multiple_of(k_pages, e) || !multiple_of(v_pages, e) || !multiple_of(o, e))
        return SPINN_HIP_EINVAL;
    if (!workspace_ok(workspace, workspace_bytes, kv_attention_workspace_bytes(d))) return SPINN_HIP_EWORKSPACE;
    return kv_attention(d, q, k_pages, v_pages, page_table, lengths, mask, acc, acc_out, o, lse, workspace,
                        (hipStream_t)stream);
}

size_t spinn_hip_kv_evict_workspace_size(const SpinnHipKvEvictDesc *d) {
    return evict_ok(d) && d->kv.seqs ? kv_evict_workspace_bytes(d) : 0;
}

int spinn_hip_kv_evict(const SpinnHipKvEvictDesc *d, const int32_t *page_table, const int32_t *lengths,
                       const int32_t *next_pos, const float *acc, const int32_t *pos, float *acc_out,
                       int32_t *pos_out, int32_t *lengths_out, void *k_pages, void *v_pages, void *workspace,
                       size_t workspace_bytes, void *stream) {
    if (!evict_ok(d)) return SPINN_HIP_EINVAL;
    if (d->kv.seqs == 0) return SPINN_HIP_OK;
    if (!page_table || !lengths || !next_pos || !acc || !pos || !acc_out || !pos_out || !lengths_out || !k_pages ||
        !v_pages)
        return SPINN_HIP_EINVAL;
    const size_t e = dtype_bytes(d->kv.dtype);
    if (!multiple_of(k_pages, e) || !multiple_of(v_pages, e)) return SPINN_HIP_EINVAL;
    if (!workspace_ok(workspace, workspace_bytes, kv_evict_workspace_bytes(d))) return SPINN_HIP_EWORKSPACE;
    return kv_evict(d, page_table, lengths, next_pos, acc, pos, acc_out, pos_out, lengths_out, k_pages, v_pages,
                    workspace, (hipStream_t)stream);
}

size_t spinn_hip_beam_select_workspace_size(const SpinnHipBeamDesc *d) {
    return beam_ok(d) && d->batch ? beam_select_workspace_bytes(d) : 0;
}

int spinn_hip_beam_select(const SpinnHipBeamDesc *d, const void *logits, const float *scores, const uint8_t *finished,
                          float *out_scores, int32_t *out_parents, int32_t *out_tokens, void *workspace,
                          size_t workspace_bytes, void *stream) {
    if (!beam_ok(d)) return SPINN_HIP_EINVAL;
    if (finished && (d->end_token < 0 || d->end_token >= d->vocab)) return SPINN_HIP_EINVAL;
    if (d->batch == 0) return SPINN_HIP_OK;
    if (!logits || !scores || !out_scores || !out_parents || !out_tokens) return SPINN_HIP_EINVAL;
    if (!multiple_of(logits, dtype_bytes(d->dtype))) return SPINN_HIP_EINVAL;
    if (!workspace_ok(workspace, workspace_bytes, beam_select_workspace_bytes(d))) return SPINN_HIP_EWORKSPACE;
    return beam_select(d, logits, scores, finished, out_scores, out_parents, out_tokens, workspace,
                       (hipStream_t)stream);
}

int spinn_hip_beam_reorder(const SpinnHipBeamState *states, int n_states, int32_t batch, int32_t beams, int32_t k,
                           const int32_t *parents, void *stream) {
    if (n_states < 0 || n_states > SPINN_HIP_MAX_BLOCKS || batch < 0 || beams <= 0 || k <= 0) return SPINN_HIP_EINVAL;
    if (n_states > 0 && !states) return SPINN_HIP_EINVAL;
    constexpr int64_t kRows = (int64_t)1 << 22; // rows of dst (one grid row each) and of src
    if ((int64_t)batch * k > kRows || (int64_t)batch * beams > kRows) return SPINN_HIP_EINVAL;
    constexpr int64_t kFar = (int64_t)1 << 38; // ends of tensors within 61 bits
    for (int i = 0; i < n_states; ++i) {
        const SpinnHipBeamState &s = states[i];
        if (s.row_bytes < 0 || s.src_stride < s.row_bytes || s.dst_stride < s.row_bytes) return SPINN_HIP_EINVAL;
        if (s.src_stride > kFar || s.dst_stride > kFar) return SPINN_HIP_EINVAL;
        if (s.row_bytes == 0 || batch == 0) continue;
        if (!s.src || !s.dst) return SPINN_HIP_EINVAL;
        // a destination over a source would be read after it was written
        const char *d0 = (const char *)s.dst, *d1 = d0 + ((int64_t)batch * k - 1) * s.dst_stride + s.row_bytes;
        for (int j = 0; j < n_states; ++j) {
            const char *s0 = (const char *)states[j].src;
            if (states[j].row_bytes <= 0 || !s0 || states[j].src_stride > kFar) continue;
            const char *s1 = s0 + ((int64_t)batch * beams - 1) * states[j].src_stride + states[j].row_bytes;
            if (d0 < s1 && s0 < d1) return SPINN_HIP_EINVAL;
        }
    }
    if (n_states == 0 || batch == 0) return SPINN_HIP_OK;
    if (!parents) return SPINN_HIP_EINVAL;
    return beam_reorder(states, n_states, batch, beams, k, parents, (hipStream_t)stream);
}

} // extern "C"
