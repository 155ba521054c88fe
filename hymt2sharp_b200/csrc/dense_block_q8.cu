// A prompt's step of a dense block with 8-bit weights launched by one call (host code only): norm to 8-bit rows, q/k/v projection, rotation and cache append,
// attention, 8-bit rows, output projection, norm with the addition, gate and up, 8-bit rows, down; each through its own entry point with the arguments that a
// caller would give it one by one.  Ten calls with their checks and the tensors in between cost the interpreter some 190 us a block, this one 25, and that
// is what a short prompt waits for.
#include "entries.cuh"

// One step of one block.  All sizes in elements; a row of `wide` 8-bit integers starts on 16 bytes.  Null pointers where the text says "or null".
struct Hymt2DenseBlockQ8 {
    float* residual;                                             // [T, hidden] float32
    const void *w_qkv, *w_o, *w_gate_up, *w_down;                // 8-bit rows
    const float *s_qkv, *s_o, *s_gate_up, *s_down;               // their scales
    const void *norm1_gain, *norm2_gain, *q_gain, *k_gain;       // the last two: or null
    const float* glu_bias;                                       // or null
    void *x8, *att8, *act8;                                      // 8-bit rows [T, hidden], [T, nh * d], [T, inner]
    float *x_scale, *att_scale, *act_scale;
    void *qkv, *q, *att, *added, *act;                           // bfloat16 [T, (nh + 2 nkv) * d], [T, nh * d] twice, [T, hidden], [T, inner]
    void *k_plane, *v_plane;                                     // one layer's planes
    const int *block_table, *token_seq, *token_pos, *slot_ids, *cu_seqlens, *kv_lens;
    const float* inv_freq;                                       // or null
    int* status;
    long cache_blocks, ld_qkv, ld_o, ld_gate_up, ld_down;        // blocks of the planes; the weight rows' distances
    int T, hidden, inner, nh, nkv, d, batch, max_new_tokens, table_stride, block_tokens, rope_dim, write_kv, window;
    int gain_dtype, norm1_dtype, norm2_dtype, glu_kind;
    float qk_eps, norm1_eps, norm2_eps, scale, glu_limit, glu_alpha;
};

HYMT2_API int hymt2_dense_block_q8_bytes() { return (int)sizeof(Hymt2DenseBlockQ8); }

// Ten kernels on `stream`.
HYMT2_API int hymt2_dense_block_q8(const Hymt2DenseBlockQ8* b, cudaStream_t stream) {
    HYMT2_REQUIRE(b, "dense_block_q8: no arguments");
    constexpr int STORE = 0, ADD = 1, GATED = 2;
    const int T = b->T, wide = b->nh * b->d, all = (b->nh + 2 * b->nkv) * b->d;
    const long ld_x = (b->hidden + 15) / 16 * 16, ld_att = (wide + 15) / 16 * 16, ld_act = (b->inner + 15) / 16 * 16;
    auto product = [&](void* out, int out_dtype, const void* a, const float* sa, const void* w, const float* sw, int n, int k, long lda, long ldw, int epilogue) {
        const bool gated = epilogue == GATED;
        return hymt2_gemm_q8_tc(out, out_dtype, a, sa, w, sw, T, n, k, lda, ldw, n, epilogue, 1, b->status, stream, gated ? b->glu_kind : (int)GLU_SILU,
                                gated ? b->glu_limit : 0.f, gated ? b->glu_alpha : 1.f, gated ? b->glu_bias : nullptr);
    };
    int rc = hymt2_rmsnorm_q8(b->x8, ld_x, b->x_scale, b->residual, HYMT2_F32, b->hidden, nullptr, HYMT2_F32, 0, nullptr, 0, b->norm1_gain, b->norm1_dtype, T,
                              b->hidden, b->norm1_eps, stream);
    if (!rc) rc = product(b->qkv, HYMT2_BF16, b->x8, b->x_scale, b->w_qkv, b->s_qkv, all, b->hidden, ld_x, b->ld_qkv, STORE);
    if (!rc) rc = hymt2_rope_kv(b->qkv, b->q, b->write_kv ? b->k_plane : nullptr, b->write_kv ? b->v_plane : nullptr, HYMT2_BF16, b->block_table,
                                b->table_stride, b->block_tokens, b->token_seq, b->token_pos, b->slot_ids, b->inv_freq, b->rope_dim, b->q_gain, b->k_gain,
                                b->gain_dtype, b->qk_eps, T, b->nh, b->nkv, b->d, b->write_kv, stream);
    if (!rc) rc = hymt2_attention_prefill_tc(b->att, b->q, b->k_plane, b->v_plane, b->cache_blocks, b->block_table, b->table_stride, b->block_tokens,
                                             b->cu_seqlens, b->slot_ids, b->kv_lens, b->batch, T, b->max_new_tokens, b->nh, b->nkv, b->d, b->scale,
                                             b->window, b->status, stream);
    if (!rc) rc = hymt2_quantize_q8(b->att8, ld_att, b->att_scale, b->att, HYMT2_BF16, wide, T, wide, stream);
    if (!rc) rc = product(b->added, HYMT2_BF16, b->att8, b->att_scale, b->w_o, b->s_o, b->hidden, wide, ld_att, b->ld_o, STORE);
    if (!rc) rc = hymt2_rmsnorm_q8(b->x8, ld_x, b->x_scale, b->residual, HYMT2_F32, b->hidden, b->added, HYMT2_BF16, b->hidden, b->residual, b->hidden,
                                   b->norm2_gain, b->norm2_dtype, T, b->hidden, b->norm2_eps, stream);
    if (!rc) rc = product(b->act, HYMT2_BF16, b->x8, b->x_scale, b->w_gate_up, b->s_gate_up, b->inner, b->hidden, ld_x, b->ld_gate_up, GATED);
    if (!rc) rc = hymt2_quantize_q8(b->act8, ld_act, b->act_scale, b->act, HYMT2_BF16, b->inner, T, b->inner, stream);
    if (!rc) rc = product(b->residual, HYMT2_F32, b->act8, b->act_scale, b->w_down, b->s_down, b->hidden, b->inner, ld_act, b->ld_down, ADD);
    return rc;
}
