// Backward of attention over packed sequences: how its passes are divided, their launches and the entry point (the kernels:
// seq_attention_bwd.h).
#include "seq_attention_bwd.h"

#include <algorithm>

void seq_bwd_two(const SeqBwdP& p, dim3 g, dim3 gk, hipStream_t st);                          // seq_attention_bwd_two.hip

// Row splits a key head, for all key heads together: enough for two workgroups a compute unit; three times that where causal, whose
// splits are empty to a half and uneven at the ends: long sequences gain up to a fifth, short ones lose 6 % at most.  None where the
// key tiles alone are that many.  Backward in us:
//   causal, at 512 / 1024 / 1536 / 2048: 6000 + 1999 + 193 tokens, 16 / 2 heads of 128, 711 / 669 / 621 / 627; 16384, 8 / 2 of 64,
//   1382 / 1104 / 1089 / 1046; 8192, 16 / 4 of 80, 1111 / 966 / 921 / 908; 2 x 2048, 16 / 4 of 128, 201 / 205 / 207 / 218; 8 x 512, the same heads,
//   95 / 91 / 91 / 93; 4096, 8 / 1 of 64, 130 / 131 / 131 / 137; fp32, 2 x 2048, 8 / 2 of 64, 495 / 518 / 523 / 538; 1000 + 700 + 300, 4 / 2 of 128, 196 / 197 / 197 / 197
//   full, at 256 / 512 / 768 / 1024: 8192, 16 / 2 of 128, 1830 / 1691 / 1708 / 1705; 2 x 2048, 16 / 4 of 128, 265 / 256 / 267 / 275; 4096, 8 / 1 of 64,
//   193 / 171 / 168 / 183; 700 + 3000 + 200, 8 / 2 of 64, 129 / 123 / 135 / 130; fp32, 2 x 2048, 8 / 2 of 64, 555 / 567 / 578 / 597
static int seq_bwd_slots(int tokens, int Hkv, int causal) {
    const int all = causal ? 1536 : 512, fill = all / Hkv < 1 ? 1 : all / Hkv;
    return tokens / 128 >= fill ? 0 : fill;
}
// Splits that there can be behind their tiles' first ones, sum_b tiles_b (splits_b - 1), a split having `least` rows or more: the
// slots, or fewer where the tokens do not allow that many - most where one sequence has them all.  None: no sequence is split, and
// nothing is joined.  (The partial sums of one utterance of 61 tokens, 2 heads of 192: none, where 1536 slots took 303 MB.)
static long seq_bwd_extra(int tokens, int G, int slots, int least) {
    return std::min((long)slots, ((long)tokens + 127) / 128 * (((long)tokens * G - 1) / least));
}

template <typename T, int DHP>
static void seq_bwd_launch(const SeqBwdP& p, hipStream_t st) {
    // the dQ pass divides its tiles as the forward does
    const int parts = seq_key_parts(p.tokens, p.B, p.G, p.Hkv, p.dh, sizeof(T) == 4, p.causal);
    const dim3 g((unsigned)(seq_units(p.tokens, p.B, p.G, 128 / parts) * p.Hkv));
    if constexpr (DHP <= (sizeof(T) == 4 ? 64 : 128)) {
        if (parts == 4) hipLaunchKernelGGL((seq_attn_dq_kernel<T, DHP, 4>), g, dim3(256), 0, st, p);
    }
    const dim3 gk((unsigned)((p.slots > 0 ? seq_split_units(p.tokens, p.B, 1, 128, p.extra) : seq_units(p.tokens, p.B, 1, 128)) * p.Hkv));
    const bool two = seq_two_parts(p.tokens, p.B, parts, sizeof(T) == 4);
    if (two) seq_bwd_two(p, g, gk, st);
    if constexpr (sizeof(T) == 2 || DHP <= 128) {
        if (parts == 2 && !two) hipLaunchKernelGGL((seq_attn_dq_kernel<T, DHP, 2>), g, dim3(256), 0, st, p);
    }
    if (parts == 1) hipLaunchKernelGGL((seq_attn_dq_kernel<T, DHP, 1>), g, dim3(256), 0, st, p);
    if (!two) hipLaunchKernelGGL((seq_attn_dkv_kernel<T, DHP, false>), gk, dim3(256), 0, st, p);
    if (p.slots > 0) hipLaunchKernelGGL((seq_dkv_join_kernel<T>), dim3((unsigned)(seq_units(p.tokens, p.B, 1, 128) * p.Hkv), 8), dim3(256), 0, st, p);
}
template <typename T>
static int seq_bwd_route(const SeqBwdP& p, hipStream_t st) {
    if (p.dh <= 64) seq_bwd_launch<T, 64>(p, st);
    else if (p.dh <= 128) seq_bwd_launch<T, 128>(p, st);
    else seq_bwd_launch<T, 192>(p, st);
    TTSMI_CHECK_LAUNCH("packed_attention_bwd");
    return TTSMI_OK;
}

static size_t seq_delta_bytes(int tokens, int H) { return (2 * (size_t)tokens * H * sizeof(float) + 255) / 256 * 256; }     // delta and lse2
extern "C" size_t ttsmi_packed_attention_bwd_ws_bytes(int B, int tokens, int H, int Hkv, int dh, int causal) {
    if (B < 0 || tokens <= 0 || H <= 0 || Hkv <= 0 || dh <= 0) return 0;
    const long extra = seq_bwd_extra(tokens, H / Hkv, seq_bwd_slots(tokens, Hkv, causal), std::min(SeqLeast<float>::ROWS, SeqLeast<__bf16>::ROWS));
    return seq_delta_bytes(tokens, H) + (extra ? (size_t)seq_split_units(tokens, B, 1, 128, extra) * Hkv * 2 * 128 * dh * sizeof(float) : 0);
}
extern "C" int ttsmi_packed_attention_bwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                                          const void* v, int64_t v_row, int64_t v_head, const void* out, int64_t o_row, int64_t o_head,
                                          const void* out_rest, const void* dout, int64_t d_row, int64_t d_head, const float* lse, const int32_t* starts,
                                          int B, int tokens, int H, int Hkv, int dh, float scale, int causal, void* dq, int64_t dq_row,
                                          int64_t dq_head, void* dk, int64_t dk_row, int64_t dk_head, void* dv, int64_t dv_row,
                                          int64_t dv_head, int zero_rest, void* ws, size_t ws_bytes, int dtype, ttsmi_stream_t stream) {
    SEQ_CHECK_COMMON("packed_attention_bwd");
    if (tokens == 0) return TTSMI_OK;
    TTSMI_CHECK_ARG(starts && lse, "packed_attention_bwd: null starts or lse");
    TTSMI_CHECK_ARG(seq_strides_ok(q, q_row, q_head, H / Hkv, dtype) && seq_strides_ok(k, k_row, k_head, 1, dtype) && seq_strides_ok(v, v_row, v_head, 1, dtype) &&
                        seq_strides_ok(out, o_row, o_head, 0, dtype) && seq_strides_ok(dout, d_row, d_head, H / Hkv, dtype) &&
                        seq_strides_ok(dq, dq_row, dq_head, 0, dtype) && seq_strides_ok(dk, dk_row, dk_head, 0, dtype) &&
                        seq_strides_ok(dv, dv_row, dv_head, 0, dtype), "packed_attention_bwd: a tensor is null or its rows or heads are not 16-byte aligned, or too far apart");
    TTSMI_CHECK_ARG(((uintptr_t)out_rest & 15) == 0, "packed_attention_bwd: out_rest is not 16-byte aligned");
    const size_t need = ttsmi_packed_attention_bwd_ws_bytes(B, tokens, H, Hkv, dh, causal);
    if (!ws || ws_bytes < need || ((uintptr_t)ws & 15)) {
        ttsmi_set_error("packed_attention_bwd: workspace of %zu bytes, %zu (16-byte aligned) needed", ws_bytes, need);
        return TTSMI_ERR_WORKSPACE;
    }
    SeqBwdP p = {};
    p.q = q; p.q_row = q_row; p.q_head = q_head; p.k = k; p.k_row = k_row; p.k_head = k_head; p.v = v; p.v_row = v_row; p.v_head = v_head;
    p.o = out; p.rest = dtype == TTSMI_BF16_IO ? out_rest : nullptr; p.o_row = o_row; p.o_head = o_head; p.d = dout; p.d_row = d_row; p.d_head = d_head;
    p.dq = dq; p.dq_row = dq_row; p.dq_head = dq_head; p.dk = dk; p.dk_row = dk_row; p.dk_head = dk_head; p.dv = dv; p.dv_row = dv_row; p.dv_head = dv_head;
    p.lse = lse; p.delta = (float*)ws; p.lse2 = (float*)ws + (size_t)tokens * H; p.starts = starts; p.B = B; p.tokens = tokens; p.Hkv = Hkv; p.G = H / Hkv; p.dh = dh;
    p.causal = causal != 0; p.zero_rest = zero_rest != 0; p.scale = scale; p.c1 = scale * SEQ_LOG2E;
    p.slots = seq_bwd_slots(tokens, Hkv, causal);
    p.extra = seq_bwd_extra(tokens, p.G, p.slots, dtype == TTSMI_F32 ? SeqLeast<float>::ROWS : SeqLeast<__bf16>::ROWS);
    if (p.extra == 0) p.slots = 0;
    p.part = (float*)((char*)ws + seq_delta_bytes(tokens, H));
    return dtype == TTSMI_F32 ? seq_bwd_route<float>(p, (hipStream_t)stream) : seq_bwd_route<__bf16>(p, (hipStream_t)stream);
}
