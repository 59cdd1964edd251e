// Attention over packed sequences (forward) and of new tokens over a paged key / value cache.
//
//   s_ij = scale q_i . k_j   (j at or before i where causal),  p = softmax_j(s),  o_i = sum_j p_ij v_j,  lse_i = log sum_j exp s_ij
//
// One pass over the keys with a running maximum and sum (fp32, log2 domain).  A workgroup of four waves owns 128 rows of one
// sequence and key head (seq_common.h: rows are (token, query head of the group) pairs), 32 rows a wave.  The wave forms the
// TRANSPOSED score tile S^T = K Q^T, so that a lane holds one row's scores for 16 keys: the softmax is in-lane plus one exchange
// of the two half-waves, and the accumulator registers, rounded, ARE the B operand of O^T += V^T P^T.
// Over a cache the keys can be split over workgroups (find_unit): each leaves its maximum, sum and unnormalised output, and a second
// launch joins them (paged_attention.hip).
#include "seq_common.h"

// CT: the cache's element type for PAGED (T, or uint8_t = e4m3)
template <typename T, typename CT, int DHP, bool PAGED>
__global__ __launch_bounds__(256, (DHP <= 128 && sizeof(T) == 2) ? 2 : 1) void seq_attn_fwd_kernel(SeqFwdP p) {
    using I = SeqImg<T, DHP>;
    using frag = typename SeqT<T>::frag;
    constexpr int KT = SeqT<T>::KT, NKB = KT / 32, NS = DHP / 16, NCB = DHP / 32, EPC = 16 / (int)sizeof(T);
    constexpr int ITEMS = KT * I::CH / 256;               // 16-byte chunks per thread and tile image
    __shared__ __attribute__((aligned(16))) unsigned char Ks[KT * I::ROWB], Vs[KT * I::ROWB];

    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % p.Hkv, unit = blockIdx.x / p.Hkv;       // bid % 8 = XCD: the tiles of a key head share few L2s
    SeqUnit un;
    if constexpr (PAGED) {
        if (p.slots > 0) un = find_unit(p.starts, p.lens, 1, p.B, p.tokens, p.G, 128, p.slots, KT, SEQ_TILE_LEAST, unit, false);
    }
    const bool splits = PAGED && p.slots > 0;
    const SeqTile st = splits ? un.t : find_tile(p.starts, p.B, p.tokens, p.G, 128, unit);
    if (st.seq < 0) {
        if (p.zero_rest) seq_zero_rest<T>((T*)p.o, p.o_row, p.o_head, p.starts, p.B, p.tokens, p.G, 128, hk * p.G, p.dh, st.tile);
        return;
    }
    const int tile = splits ? st.tile : st.ntile - 1 - st.tile;              // causal: the tiles with the most keys first
    const int rows = st.n * p.G;
    int len = st.n, off = 0;
    if (PAGED) {
        len = max(p.lens[st.seq], 0);
        off = len - st.n;                                 // position of the first new token
    }
    // this lane's row and the number of keys it sees
    const int r = tile * 128 + wave * 32 + l31;
    const bool rok = r < rows;
    const int tok = r / p.G, head = hk * p.G + r - tok * p.G;
    const int lim = !rok ? 0 : p.causal ? min(max(off + tok + 1, 0), len) : len;
    // the same for the workgroup's last row, and for this wave's: no key behind is fetched / multiplied
    const int last = min(tile * 128 + 127, rows - 1) / p.G;
    int kend = p.causal ? min(max(off + last + 1, 0), len) : len, kbeg = 0;
    const bool part = splits && un.nsplit > 1;
    if (part) {
        kbeg = min(un.split * un.per, kend);
        kend = min(kbeg + un.per, kend);
    }
    const int wrow = tile * 128 + wave * 32;
    const int wlast = min(wrow + 31, rows - 1) / p.G;
    const int wend = wrow >= rows ? 0 : min(kend, p.causal ? max(off + wlast + 1, 0) : len);
    const int wfull = wrow + 31 < rows ? (p.causal ? off + wrow / p.G + 1 : len) : 0;     // keys that every row of the wave sees

    frag qf[NS];
    {
        const T* qr = (const T*)p.q + (long)(st.s0 + tok) * p.q_row + (long)head * p.q_head;
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = seq_load8<T>(qr, 16 * s + 8 * hh, rok && 16 * s + 8 * hh < p.dh);
    }
    f32x16 o[NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[cb][i] = 0.f;
    float m = -INFINITY, l = 0.f;

    // ---- tile staging: global -> registers (a tile ahead) -> LDS; rows past the last key are zeros ----
    // PAGED: the page rows of a tile are looked up one tile earlier still, so that no load waits for another
    uint4 rk[ITEMS], rv[ITEMS];
    long at[PAGED ? ITEMS : 1];
    auto look = [&](int k0) {
        if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int key = k0 + (tid + 256 * i) / I::CH;
                at[i] = key < kend ? p.pg.row(st.seq, hk, key) : -1;
            }
        }
    };
    auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int id = tid + 256 * i, row = id / I::CH, ch = id - row * I::CH, key = k0 + row;
            rk[i] = rv[i] = make_uint4(0u, 0u, 0u, 0u);
            if constexpr (PAGED) {
                if (at[i] >= 0 && ch * EPC < p.dh) {
                    if constexpr (sizeof(CT) == 1) {
                        rk[i] = seq_dequant_chunk<T>((const uint8_t*)p.pg.k + at[i] * p.dh + ch * EPC, seq_scale_of(p.pg.ke[at[i]]));
                        rv[i] = seq_dequant_chunk<T>((const uint8_t*)p.pg.v + at[i] * p.dh + ch * EPC, seq_scale_of(p.pg.ve[at[i]]));
                    } else {
                        rk[i] = *reinterpret_cast<const uint4*>((const T*)p.pg.k + at[i] * p.dh + ch * EPC);
                        rv[i] = *reinterpret_cast<const uint4*>((const T*)p.pg.v + at[i] * p.dh + ch * EPC);
                    }
                }
            } else if (key < kend && ch * EPC < p.dh) {
                rk[i] = *reinterpret_cast<const uint4*>((const T*)p.k + (long)(st.s0 + key) * p.k_row + (long)hk * p.k_head + ch * EPC);
                rv[i] = *reinterpret_cast<const uint4*>((const T*)p.v + (long)(st.s0 + key) * p.v_row + (long)hk * p.v_head + ch * EPC);
            }
        }
    };
    auto stash = [&]() {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int id = tid + 256 * i, row = id / I::CH, ch = id - row * I::CH;
            *reinterpret_cast<uint4*>(Ks + I::at(row, ch)) = rk[i];
            *reinterpret_cast<uint4*>(Vs + I::at(row, ch)) = rv[i];
        }
    };

    if (kbeg < kend) {
        look(kbeg);
        fetch(kbeg);
        look(kbeg + KT);
    }
    for (int k0 = kbeg; k0 < kend; k0 += KT) {
        __syncthreads();
        stash();
        __syncthreads();
        if (k0 + KT < kend) {
            fetch(k0 + KT);
            look(k0 + 2 * KT);
        }
        if (k0 >= wend) continue;
        f32x16 s[NKB];
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
            for (int t = 0; t < NS; ++t) s[kb] = seq_mma(seq_frag<T, DHP>(Ks, kb * 32 + l31, t, hh), qf[t], s[kb]);
        }
        if (k0 + KT > wfull || k0 + KT > kend) {
            const int seen = min(lim, kend) - k0;
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (kb * 32 + seq_rowmap(i, hh) >= seen) s[kb][i] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
        mx = seq_half_max(mx) * p.c1;
        const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn;      // a row that has seen no key yet keeps p = 0
        const float a = __builtin_amdgcn_exp2f(m - ms);
        m = mn;
        float sum = 0.f;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kb][i] = __builtin_amdgcn_exp2f(s[kb][i] * p.c1 - ms);
                sum += s[kb][i];
            }
        l = l * a + sum;                                                     // (this half-wave's keys; joined at the end)
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[cb][i] *= a;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                frag pf;
                seq_to_frag(s[kb], t, pf);
#pragma unroll
                for (int cb = 0; cb < NCB; ++cb) o[cb] = seq_mma(seq_frag_t<T, DHP>(Vs, kb * 32, t, cb, lane), pf, o[cb]);
            }
    }
    l = seq_half_sum(l);
    if (!rok) return;
    const long slot = (long)hk * p.tokens * p.G + (long)st.s0 * p.G + r;
    if (part) {
        const long ps = ((un.first + un.split) * p.Hkv + hk) * 128 + wave * 32 + l31;
        if (hh == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * ps) = make_float2(m, l);
        if (l > 0.f || !(l == l)) {
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int c = cb * 32 + 8 * g + 4 * hh;
                    if (c < p.dh) *reinterpret_cast<float4*>(p.part_o + ps * p.dh + c) = make_float4(o[cb][4 * g], o[cb][4 * g + 1], o[cb][4 * g + 2], o[cb][4 * g + 3]);
                }
        }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (p.lse && hh == 0) p.lse[slot] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * SEQ_LN2;
    T* orow = (T*)p.o + (long)(st.s0 + tok) * p.o_row + (long)head * p.o_head;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = cb * 32 + 8 * g + 4 * hh;
            if (c >= p.dh) continue;
            if constexpr (sizeof(T) == 2) {
                bf16x4 h;
#pragma unroll
                for (int e = 0; e < 4; ++e) h[e] = (__bf16)(o[cb][4 * g + e] * inv);
                *reinterpret_cast<bf16x4*>(orow + c) = h;
            } else {
                *reinterpret_cast<float4*>(orow + c) = make_float4(o[cb][4 * g] * inv, o[cb][4 * g + 1] * inv, o[cb][4 * g + 2] * inv, o[cb][4 * g + 3] * inv);
            }
        }
}

// ---- launches -----------------------------------------------------------------------------------------

template <typename T, typename CT, bool PAGED>
static int seq_fwd_launch(const SeqFwdP& p, hipStream_t st) {
    const long units = p.slots > 0 ? seq_split_units(p.tokens, p.B, p.G, 128, p.slots) : seq_units(p.tokens, p.B, p.G, 128);
    const dim3 g((unsigned)(units * p.Hkv));
    if (p.dh <= 64) hipLaunchKernelGGL((seq_attn_fwd_kernel<T, CT, 64, PAGED>), g, dim3(256), 0, st, p);
    else if (p.dh <= 128) hipLaunchKernelGGL((seq_attn_fwd_kernel<T, CT, 128, PAGED>), g, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((seq_attn_fwd_kernel<T, CT, 192, PAGED>), g, dim3(256), 0, st, p);
    TTSMI_CHECK_LAUNCH("seq_attention");
    return TTSMI_OK;
}
// the tile form of the paged attention (paged_attention.hip)
int seq_paged_tiles(const SeqFwdP& p, int dtype, int cache_dtype, hipStream_t st) {
    if (dtype == TTSMI_F32)
        return cache_dtype == TTSMI_E4M3 ? seq_fwd_launch<float, uint8_t, true>(p, st) : seq_fwd_launch<float, float, true>(p, st);
    return cache_dtype == TTSMI_E4M3 ? seq_fwd_launch<__bf16, uint8_t, true>(p, st) : seq_fwd_launch<__bf16, __bf16, true>(p, st);
}

extern "C" int ttsmi_packed_attention_fwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                                          const void* v, int64_t v_row, int64_t v_head, const int32_t* starts, int B, int tokens,
                                          int H, int Hkv, int dh, float scale, int causal, void* out, int64_t o_row, int64_t o_head,
                                          float* lse, int zero_rest, int dtype, ttsmi_stream_t stream) {
    SEQ_CHECK_COMMON("packed_attention_fwd");
    if (tokens == 0) return TTSMI_OK;
    TTSMI_CHECK_ARG(starts, "packed_attention_fwd: null starts");
    TTSMI_CHECK_ARG(seq_strides_ok(q, q_row, q_head, dtype) && seq_strides_ok(k, k_row, k_head, dtype) && seq_strides_ok(v, v_row, v_head, dtype) &&
                        seq_strides_ok(out, o_row, o_head, dtype), "packed_attention_fwd: a tensor is null or its rows or heads are not 16-byte aligned");
    SeqFwdP p = {};
    p.q = q; p.q_row = q_row; p.q_head = q_head; p.k = k; p.k_row = k_row; p.k_head = k_head; p.v = v; p.v_row = v_row; p.v_head = v_head;
    p.o = out; p.zero_rest = zero_rest != 0; p.o_row = o_row; p.o_head = o_head; p.lse = lse; p.starts = starts;
    p.B = B; p.tokens = tokens; p.Hkv = Hkv; p.G = H / Hkv; p.dh = dh; p.causal = causal != 0; p.c1 = scale * SEQ_LOG2E;
    return dtype == TTSMI_F32 ? seq_fwd_launch<float, float, false>(p, (hipStream_t)stream) : seq_fwd_launch<__bf16, __bf16, false>(p, (hipStream_t)stream);
}
