// Backward of attention over packed sequences, in two passes that recompute the probabilities from lse (no [rows, keys] tensor,
// no atomics: every gradient element is summed by one workgroup in a fixed order).
//
//   delta_i = do_i . o_i     p_ij = exp(s_ij - lse_i)     ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i      dv_j = sum_i p_ij do_i      (i: every query head of the group)
//
// dQ:     as the forward - 128 rows a workgroup, 32 a wave, S^T and dP^T per key tile, dQ^T += K^T dS^T.  It also forms delta and
//         lse in log2 units, once, for the second pass.  delta is a small difference's other half where a row has a peak: from the
//         bf16 output alone its error is a third of dq's (2000 causal tokens, heads of 128, scores of deviation 1.6: dq off by
//         0.26 % instead of 0.24 %, of which 0.17 % is its own rounding), so the forward leaves what its rounding took (out_rest).
// dK, dV: 128 keys of one key head a workgroup, 32 a wave; the row tiles of every query head of the group pass through LDS, the
//         wave forms S and dP with a key per lane, so that P and dS are the B operands of dV^T += dO^T P and dK^T += Q^T dS.
//
// Bound like the forward (long batches: matrix pipes busy 52 %, LDS 26 - 33 %); the causal dK / dV pass leaves a quarter of the card idle
// at its ends.  The scores and dP are formed in both passes: seven products where five would do.
// Measured as in the forward, causal bf16, 6000 + 1999 + 193 tokens of 16 / 2 heads of 128: dQ 245 us (238), 1000 TFLOP/s of its three
// products, dK / dV 369 (353), 890 of its four, and 23 for the join of its row splits; 32 utterances of 202 .. 900, 4 heads of 64: 37 and
// 38 us; fp32, 8 utterances of 117 .. 700, 4 / 2 heads of 64: 32 (48 with two waves a row block), 38 and 6 us.
// fp32 heads of 129 .. 192 do not fit the registers: 258 of the dK / dV pass and 17 of dQ are spilled (756 bytes of scratch a lane in the
// former; of heads of 65 .. 128 it spills 10), whose reloads wait for the tile in flight behind them.  2048 causal tokens, 4 / 2 heads,
// forward / with the backward: 414 / 1346 us for heads of 192, 160 / 580 for heads of 128.
#pragma once
#include "seq_common.h"

struct SeqBwdP {
    const void* q; long q_row, q_head;
    const void* k; long k_row, k_head;
    const void* v; long v_row, v_head;
    const void* o; long o_row, o_head;
    const void* rest;                                     // [tokens][H][dh]: what the rounding of o to bf16 left, or null
    const void* d; long d_row, d_head;                    // gradient of the output
    void* dq; long dq_row, dq_head;
    void* dk; long dk_row, dk_head;
    void* dv; long dv_row, dv_head;
    const float* lse; float* lse2; float* delta;          // [Hkv][tokens G]; lse2: in log2 units
    const int* starts;
    int B, tokens, Hkv, G, dh, causal, zero_rest;
    float scale, c1;
    // row splits of the dK / dV pass (slots > 0): sums of unit u, key head hk at [(u Hkv + hk)][dK, dV][128 keys][dh], fp32.
    // extra: how many splits there can be behind their tiles' first ones, the slots or fewer (seq_bwd_extra)
    int slots; long extra; float* part;
};
// Rows of a split at least: eight tiles of work against the traffic of its partial sums; fp32 products are slower.  Backward in us:
//   bf16, at 256 / 512 / 1024 / 2048 rows: causal 8 x 512 tokens, 16 / 4 heads of 128, 106 / 92 / 94 / 118; 3 x 1024, 8 heads of 64,
//   53 / 55 / 57 / 56; 2048, 8 / 2 of 64, 66 / 59 / 64 / 85; 4096, 4 of 128, 169 / 168 / 160 / 173; full, 8 of 264 .. 900, 4 of 64, 56 / 57 / 60 / 60
//   fp32, at 96 / 192 / 384 / 768: causal 8 of 117 .. 700, 4 / 2 heads of 64, 111 / 104 / 123 / 176; 2048, 4 of 64, 177 / 164 / 154 / 194;
//   1000 + 500, 4 / 2 of 128, 208 / 193 / 241 / 343; full, 3 x 800, 8 of 64, 209 / 206 / 233 / 236; 1500, 4 / 1 of 64, 136 / 141 / 128 / 179
template <typename T> struct SeqLeast { static constexpr int ROWS = sizeof(T) == 2 ? 512 : 192; };

// four accumulator registers -> four consecutive elements of a gradient row
template <typename T>
__device__ __forceinline__ void seq_store4(T* dst, const f32x16& a, int g, float f) {
    if constexpr (sizeof(T) == 2) {
        bf16x4 h;
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = (__bf16)(a[4 * g + e] * f);
        *reinterpret_cast<bf16x4*>(dst) = h;
    } else {
        *reinterpret_cast<float4*>(dst) = make_float4(a[4 * g] * f, a[4 * g + 1] * f, a[4 * g + 2] * f, a[4 * g + 3] * f);
    }
}

// TWO: score gradients in two parts (seq_two_parts).
template <typename T, int DHP, int KS, bool TWO = false>
__global__ __launch_bounds__(256, (DHP <= 128 && sizeof(T) == 2) ? 2 : 1) void seq_attn_dq_kernel(SeqBwdP p) {
    using I = SeqImg<T, DHP>;
    using frag = typename SeqT<T>::frag;
    constexpr int KW = SeqKeys<T, DHP, KS>::KW, KT = KW * KS, NKB = KW / 32, NS = DHP / 16, NCB = DHP / 32, ROWS = 128 / KS;
    using D = SeqDma<T, DHP, KT>;
    constexpr int IMG = KT * I::ROWB, ITEMS = D::NI;
    __shared__ __attribute__((aligned(1024))) unsigned char sm[4 * IMG];             // two stages of a K and a V tile
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % p.Hkv, unit = blockIdx.x / p.Hkv;
    const SeqTile st = find_tile(p.starts, p.B, p.tokens, p.G, ROWS, unit, p.causal);
    if (st.seq < 0) {
        if (p.zero_rest) seq_zero_rest<T>((T*)p.dq, p.dq_row, p.dq_head, p.starts, p.B, p.tokens, p.G, ROWS, hk * p.G, p.dh, st.tile);
        return;
    }
    const int tile = st.ntile - 1 - st.tile, rows = st.n * p.G, len = st.n;
    constexpr int RW = 4 / KS;                                         // as in the forward
    const int kpart = wave / RW, wrow = tile * ROWS + wave % RW * 32;
    const int r = wrow + l31;
    const bool rok = r < rows;
    const int tok = r / p.G, head = hk * p.G + r - tok * p.G;
    const int lim = !rok ? 0 : p.causal ? min(tok + 1, len) : len;
    const int last = min(tile * ROWS + ROWS - 1, rows - 1) / p.G;
    const int kend = p.causal ? min(last + 1, len) : len;
    const int wend = wrow >= rows ? 0 : p.causal ? min(kend, min(wrow + 31, rows - 1) / p.G + 1) : kend;
    const int wfull = wrow + 31 < rows ? (p.causal ? wrow / p.G + 1 : len) : 0;
    const long slot = (long)hk * p.tokens * p.G + (long)st.s0 * p.G + r;

    frag qf[NS], df[NS];
    {
        const T* qr = (const T*)p.q + (long)(st.s0 + tok) * p.q_row + (long)head * p.q_head;
        const T* dr = (const T*)p.d + (long)(st.s0 + tok) * p.d_row + (long)head * p.d_head;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const bool ok = rok && 16 * s + 8 * hh < p.dh;
            qf[s] = seq_load8<T>(qr, 16 * s + 8 * hh, ok);
            df[s] = seq_load8<T>(dr, 16 * s + 8 * hh, ok);
        }
    }
    float lse2 = 0.f, delta = 0.f;
    if (rok) {                                                         // delta and lse2 of this row, left for the dK / dV pass too
        const T* orow = (const T*)p.o + (long)(st.s0 + tok) * p.o_row + (long)head * p.o_head;
        lse2 = p.lse[slot] * SEQ_LOG2E;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const frag f = seq_load8<T>(orow, 16 * s + 8 * hh, 16 * s + 8 * hh < p.dh);
            if (sizeof(T) == 2 && p.rest) {
                const frag x = seq_load8<T>((const T*)p.rest + ((long)(st.s0 + tok) * p.Hkv * p.G + head) * p.dh, 16 * s + 8 * hh, 16 * s + 8 * hh < p.dh);
#pragma unroll
                for (int e = 0; e < 8; ++e) delta += ((float)f[e] + (float)x[e]) * (float)df[s][e];
                continue;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) delta += (float)f[e] * (float)df[s][e];
        }
    }
    delta = seq_half_sum(delta);
    if (rok && hh == 0 && kpart == 0) {
        p.delta[slot] = delta;
        p.lse2[slot] = lse2;
    }
    f32x16 acc[NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[cb][i] = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) asm volatile("" : "+v"(qf[s]), "+v"(df[s]));
    asm volatile("" : "+v"(lse2), "+v"(delta));                        // everything loaded in front of the first DMA
    uint32_t ko[ITEMS], vo[ITEMS];
    const uint32_t krb = (uint32_t)(p.k_row * (long)sizeof(T)), vrb = (uint32_t)(p.v_row * (long)sizeof(T));
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        ko[i] = D::row(i, wave, lane) * krb + D::piece(i, wave, lane, p.dh);
        vo[i] = D::row(i, wave, lane) * vrb + D::piece(i, wave, lane, p.dh);
    }
    auto fetch = [&](int k0, int buf) {                                // a row past the last key repeats it (its score is masked)
        unsigned char* const img = sm + buf * 2 * IMG;
        const char* const kb = (const char*)p.k + ((long)(st.s0 + k0) * p.k_row + (long)hk * p.k_head) * (long)sizeof(T);
        const char* const vb = (const char*)p.v + ((long)(st.s0 + k0) * p.v_row + (long)hk * p.v_head) * (long)sizeof(T);
        const bool whole = k0 + KT <= kend;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t row = min(D::row(i, wave, lane), kend - 1 - k0), c = D::piece(i, wave, lane, p.dh);
            seq_dma16(kb, whole ? ko[i] : row * krb + c, seq_lds(img + (wave + 4 * i) * 1024));
            seq_dma16(vb, whole ? vo[i] : row * vrb + c, seq_lds(img + IMG + (wave + 4 * i) * 1024));
        }
    };
    fetch(0, 0);
    using A = SeqLane<T, DHP>;
    const uint32_t kbase = A::rows(sm, lane) + kpart * KW * I::ROWB, tbase = A::cols(sm, lane) + kpart * KW * I::ROWB;
    int buf = 0;
    for (int k0 = 0; k0 < kend; k0 += KT, buf ^= 1) {
        seq_dma_barrier();
        if (k0 + KT < kend) fetch(k0 + KT, buf ^ 1);
        const int kw = k0 + kpart * KW;                                // this wave's keys of the tile
        if (kw >= wend) continue;
        const uint32_t ka = kbase + buf * 2 * IMG, ta = tbase + buf * 2 * IMG;
        const bool edge = kw + KW > wfull;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
            if (kw + kb * 32 >= wend) break;
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
#pragma unroll
            for (int t = 0; t < NS; ++t) {
                s = seq_mma(A::row(ka, kb * 32, t), qf[t], s);
                dp = seq_mma(A::row(ka + IMG, kb * 32, t), df[t], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i] * p.c1 - lse2) * (dp[i] - delta);
            if (edge) {
                const int seen = seq_rare(lim - kw - kb * 32);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (seq_rowmap(i, hh) >= seen) s[i] = 0.f;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                frag f;
                seq_to_frag(s, t, f);
                if constexpr (TWO) {
                    frag fr;
                    seq_to_rest(s, t, f, fr);
#pragma unroll
                    for (int cb = 0; cb < NCB; ++cb) {
                        const frag kf = A::col(ta, kb * 32, t, cb);
                        acc[cb] = seq_mma(kf, fr, seq_mma(kf, f, acc[cb]));
                    }
                } else {
#pragma unroll
                    for (int cb = 0; cb < NCB; ++cb) acc[cb] = seq_mma(A::col(ta, kb * 32, t, cb), f, acc[cb]);
                }
            }
        }
    }
    if constexpr (KS > 1) {
        constexpr int PART = RW * 32 * (DHP + 4);
        float* mo = reinterpret_cast<float*>(sm) + (wave % RW * 32 + l31) * (DHP + 4) + 4 * hh;
        seq_dma_barrier();
        if (kpart > 0) {
            mo += (kpart - 1) * PART;
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
                for (int g = 0; g < 4; ++g) seq_store4<float>(mo + cb * 32 + 8 * g, acc[cb], g, 1.f);
        }
        __syncthreads();
        if (kpart > 0) return;
#pragma unroll
        for (int x = 1; x < KS; ++x, mo += PART)
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[cb][i] += mo[cb * 32 + 8 * (i >> 2) + (i & 3)];
    }
    if (!rok) return;
    T* dst = (T*)p.dq + (long)(st.s0 + tok) * p.dq_row + (long)head * p.dq_head;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (cb * 32 + 8 * g + 4 * hh < p.dh) seq_store4<T>(dst + cb * 32 + 8 * g + 4 * hh, acc[cb], g, p.scale);
}

// TWO: probabilities and score gradients in two parts (seq_two_parts); one wave a SIMD has the registers for it.
template <typename T, int DHP, bool TWO>
__global__ __launch_bounds__(256, (DHP <= 128 && sizeof(T) == 2 && !TWO) ? 2 : 1) void seq_attn_dkv_kernel(SeqBwdP p) {
    using I = SeqImg<T, DHP>;
    using frag = typename SeqT<T>::frag;
    constexpr int KT = SeqT<T>::KT, NKB = KT / 32, NS = DHP / 16, NCB = DHP / 32;
    using D = SeqDma<T, DHP, KT>;
    constexpr int IMG = KT * I::ROWB, ITEMS = D::NI, STAGE = 2 * IMG + 512;
    __shared__ __attribute__((aligned(1024))) unsigned char sm[2 * STAGE];           // two stages of a Q and a dO tile, lse2 and delta
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % p.Hkv, unit = blockIdx.x / p.Hkv;
    SeqUnit un;
    if (p.slots > 0) un = find_unit(p.starts, nullptr, p.G, 0x7fffffff, p.B, p.tokens, 1, 128, p.slots, KT, SeqLeast<T>::ROWS, unit, false);
    const SeqTile st = p.slots > 0 ? un.t : find_tile(p.starts, p.B, p.tokens, 1, 128, unit);   // causal: the first keys have the most rows
    if (st.seq < 0) {
        if (p.zero_rest) {
            seq_zero_rest<T>((T*)p.dk, p.dk_row, p.dk_head, p.starts, p.B, p.tokens, 1, 128, hk, p.dh, st.tile);
            seq_zero_rest<T>((T*)p.dv, p.dv_row, p.dv_head, p.starts, p.B, p.tokens, 1, 128, hk, p.dh, st.tile);
        }
        return;
    }
    const int key0 = st.tile * 128, key = key0 + wave * 32 + l31;
    const int first = p.causal ? key0 * p.G : 0;                                  // rows before see none of these keys
    int rows = st.n * p.G, r_begin = first / KT * KT;
    bool part = false;
    if (p.slots > 0 && un.nsplit > 1) {
        if ((un.split + 1) * (long)un.per <= first) return;                       // a split in front of the first row: nothing
        part = first / un.per < un.nsplit - 1;                                    // more than one split has rows
        r_begin = max(r_begin, un.split * un.per);
        rows = (int)min((long)rows, (un.split + 1) * (long)un.per);
    }
    const bool kok = key < st.n;
    const bool live = key0 + wave * 32 < st.n;
    frag kf[NS], vf[NS];
    {
        const T* kr = (const T*)p.k + (long)(st.s0 + key) * p.k_row + (long)hk * p.k_head;
        const T* vr = (const T*)p.v + (long)(st.s0 + key) * p.v_row + (long)hk * p.v_head;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const bool ok = kok && 16 * s + 8 * hh < p.dh;
            kf[s] = seq_load8<T>(kr, 16 * s + 8 * hh, ok);
            vf[s] = seq_load8<T>(vr, 16 * s + 8 * hh, ok);
        }
    }
    f32x16 dk[NCB], dv[NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) dk[cb][i] = dv[cb][i] = 0.f;
    const int wfirst = p.causal ? (key0 + wave * 32) * p.G : 0;
    const int wfull = p.causal ? (key0 + wave * 32 + 31) * p.G : 0;               // from here on rows see every key of the wave
    const long slot0 = (long)hk * p.tokens * p.G + (long)st.s0 * p.G;
#pragma unroll
    for (int s = 0; s < NS; ++s) asm volatile("" : "+v"(kf[s]), "+v"(vf[s]));        // loaded in front of the first DMA
    const float inv_g = 1.f / (float)p.G;
    // rows r0 .. r0 + KT into stage buf; a row past the last repeats it (masked).  Row r0 is head `rem` of token `tok`: the small
    // quotient (rem + row) / G is exact in fp32.  Where G divides the rows of an instruction, the items of a lane lie whole tokens
    // apart and share one offset.
    constexpr int RPI = 256 / I::CH;                                                 // image rows between a lane's items
    const bool even = 256 % I::CH == 0 && RPI % 16 == 0 && RPI % p.G == 0;          // (the permutation repeats after 16 rows)
    auto fetch = [&](int r0, int buf) {
        unsigned char* const img = sm + buf * STAGE;
        const int ln = seq_lane_here();
        const int tok = __builtin_amdgcn_readfirstlane(r0 / p.G), rem = r0 - tok * p.G;
        const uint32_t qrb = (uint32_t)(p.q_row * (long)sizeof(T)), qhb = (uint32_t)(p.q_head * (long)sizeof(T));
        const uint32_t drb = (uint32_t)(p.d_row * (long)sizeof(T)), dhb = (uint32_t)(p.d_head * (long)sizeof(T));
        const char* const qb = (const char*)p.q + ((long)(st.s0 + tok) * p.q_row + (long)hk * p.G * p.q_head) * (long)sizeof(T);
        const char* const db = (const char*)p.d + ((long)(st.s0 + tok) * p.d_row + (long)hk * p.G * p.d_head) * (long)sizeof(T);
        if (even && r0 + KT <= rows) {
            const int x = rem + D::row(0, wave, ln), t = (int)(((float)x + 0.5f) * inv_g), g = x - t * p.G;
            const uint32_t c = D::piece(0, wave, ln, p.dh), qo = t * qrb + g * qhb + c, dO = t * drb + g * dhb + c;
            const long qstep = (long)(RPI / p.G) * qrb, dstep = (long)(RPI / p.G) * drb;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                seq_dma16(qb + i * qstep, qo, seq_lds(img + (wave + 4 * i) * 1024));
                seq_dma16(db + i * dstep, dO, seq_lds(img + IMG + (wave + 4 * i) * 1024));
            }
        } else {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int x = rem + min(D::row(i, wave, ln), rows - 1 - r0), t = (int)(((float)x + 0.5f) * inv_g), g = x - t * p.G;
                const uint32_t c = D::piece(i, wave, ln, p.dh);
                seq_dma16(qb, t * qrb + g * qhb + c, seq_lds(img + (wave + 4 * i) * 1024));
                seq_dma16(db, t * drb + g * dhb + c, seq_lds(img + IMG + (wave + 4 * i) * 1024));
            }
        }
        const int x = min(r0 + (ln & (KT - 1)), rows - 1);
        if (wave == 0) seq_dma4(p.lse2 + slot0 + x, seq_lds(img + 2 * IMG));
        if (wave == 1) seq_dma4(p.delta + slot0 + x, seq_lds(img + 2 * IMG + 256));
    };
    r_begin = __builtin_amdgcn_readfirstlane(r_begin);
    rows = __builtin_amdgcn_readfirstlane(rows);
    fetch(r_begin, 0);
    using A = SeqLane<T, DHP>;
    const uint32_t rbase = A::rows(sm, lane), tbase = A::cols(sm, lane);
    int buf = 0;
    for (int r0 = r_begin; r0 < rows; r0 += KT, buf ^= 1) {
        seq_dma_barrier();
        if (r0 + KT < rows) fetch(r0 + KT, buf ^ 1);
        const uint32_t qa = rbase + buf * STAGE, ta = tbase + buf * STAGE;
        const float* const Ls = reinterpret_cast<const float*>(sm + buf * STAGE + 2 * IMG) + 4 * hh;
        if (!live || r0 + KT <= wfirst) continue;
        const bool edge = r0 < wfull || r0 + KT > rows;
#pragma unroll 1
        for (int kb = 0; kb < NKB; ++kb) {
            if (r0 + kb * 32 >= rows || r0 + kb * 32 + 32 <= wfirst) continue;
            const uint32_t qk = qa + kb * 32 * I::ROWB, tk = ta + kb * 32 * I::ROWB;
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
            // (operands two steps ahead of their products: with the registers that are left the compiler would read each
            // one just before its use, an LDS round trip per product)
            frag fq[2], fd[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                fq[t] = A::row(qk, 0, t);
                fd[t] = A::row(qk + IMG, 0, t);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < NS; ++t) {
                s = seq_mma(fq[t & 1], kf[t], s);
                dp = seq_mma(fd[t & 1], vf[t], dp);
                if (t + 2 < NS) {
                    fq[t & 1] = A::row(qk, 0, t + 2);
                    fd[t & 1] = A::row(qk + IMG, 0, t + 2);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 ls = *reinterpret_cast<const float4*>(Ls + kb * 32 + 8 * g);
                const float4 dl = *reinterpret_cast<const float4*>(Ls + 64 + kb * 32 + 8 * g);
                const float le[4] = {ls.x, ls.y, ls.z, ls.w}, de[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[4 * g + e] = __builtin_amdgcn_exp2f(s[4 * g + e] * p.c1 - le[e]);
                    dp[4 * g + e] = s[4 * g + e] * (dp[4 * g + e] - de[e]);
                }
            }
            if (edge) {
                const int ln = seq_lane_here(), base = r0 + kb * 32 + 4 * (ln >> 5);
                const int from = (p.causal ? (key0 + wave * 32 + (ln & 31)) * p.G : 0) - base, to = rows - base;      // rows >= the key's own see it
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = seq_rowmap(i, 0);
                    if (r < from || r >= to) s[i] = dp[i] = 0.f;
                }
            }
            frag pf[2], sf[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                seq_to_frag(s, t, pf[t]);
                seq_to_frag(dp, t, sf[t]);
            }
            if constexpr (TWO) {
                frag pr[2], sr[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    seq_to_rest(s, t, pf[t], pr[t]);
                    seq_to_rest(dp, t, sf[t], sr[t]);
                }
#pragma unroll
                for (int x = 0; x < 2 * NCB; ++x) {
                    const int t = x / NCB, cb = x % NCB;
                    const frag d = A::col(tk + IMG, 0, t, cb), q = A::col(tk, 0, t, cb);
                    dv[cb] = seq_mma(d, pr[t], seq_mma(d, pf[t], dv[cb]));
                    dk[cb] = seq_mma(q, sr[t], seq_mma(q, sf[t], dk[cb]));
                }
                continue;
            }
            fd[0] = A::col(tk + IMG, 0, 0, 0);
            fq[0] = A::col(tk, 0, 0, 0);
#pragma unroll
            for (int x = 0; x < 2 * NCB; ++x) {
                const int t = x / NCB, cb = x % NCB;
                if (x + 1 < 2 * NCB) {
                    fd[(x + 1) & 1] = A::col(tk + IMG, 0, (x + 1) / NCB, (x + 1) % NCB);
                    fq[(x + 1) & 1] = A::col(tk, 0, (x + 1) / NCB, (x + 1) % NCB);
                    __builtin_amdgcn_sched_barrier(0);
                }
                dv[cb] = seq_mma(fd[x & 1], pf[t], dv[cb]);
                dk[cb] = seq_mma(fq[x & 1], sf[t], dk[cb]);
            }
        }
    }
    if (!kok) return;
    if (part) {
        float* dst = p.part + (((un.first + (long)un.split * un.t.ntile) * p.Hkv + hk) * 2 * 128 + wave * 32 + l31) * p.dh;
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = cb * 32 + 8 * g + 4 * hh;
                if (c >= p.dh) continue;
                seq_store4<float>(dst + c, dk[cb], g, 1.f);
                seq_store4<float>(dst + 128 * p.dh + c, dv[cb], g, 1.f);
            }
        return;
    }
    T* dkr = (T*)p.dk + (long)(st.s0 + key) * p.dk_row + (long)hk * p.dk_head;
    T* dvr = (T*)p.dv + (long)(st.s0 + key) * p.dv_row + (long)hk * p.dv_head;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = cb * 32 + 8 * g + 4 * hh;
            if (c >= p.dh) continue;
            seq_store4<T>(dkr + c, dk[cb], g, p.scale);
            seq_store4<T>(dvr + c, dv[cb], g, 1.f);
        }
}

// the sums of a key tile's splits, in their order: 16 keys a workgroup (grid y), four elements a thread
template <typename T>
__global__ __launch_bounds__(256) void seq_dkv_join_kernel(SeqBwdP p) {
    const int hk = blockIdx.x % p.Hkv;
    const SeqUnit un = find_unit(p.starts, nullptr, p.G, 0x7fffffff, p.B, p.tokens, 1, 128, p.slots, SeqT<T>::KT, SeqLeast<T>::ROWS, blockIdx.x / p.Hkv, true);
    if (un.t.seq < 0) return;
    const int key0 = un.t.tile * 128, z0 = (p.causal ? key0 * p.G : 0) / un.per;
    if (un.nsplit - z0 < 2 || un.first + (long)(un.nsplit - 1) * un.t.ntile >= seq_split_units(p.tokens, p.B, 1, 128, p.extra)) return;   // (the latter: `starts` that overlap)
    const int per = p.dh / 4, keys = min(16, un.t.n - key0 - 16 * (int)blockIdx.y);
    const long step = 2L * 128 * p.dh * p.Hkv * un.t.ntile;
    for (int i = threadIdx.x; i < 2 * keys * per; i += 256) {
        const int which = i >= keys * per, j = i - which * keys * per, row = 16 * blockIdx.y + j / per, c = (j % per) * 4;
        const float* src = p.part + (((un.first + (long)z0 * un.t.ntile) * p.Hkv + hk) * 2 * 128 + which * 128 + row) * p.dh + c;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int z = z0; z < un.nsplit; ++z, src += step) {
            const float4 b = *reinterpret_cast<const float4*>(src);
            a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
        }
        const long tok = un.t.s0 + key0 + row;
        T* dst = which ? (T*)p.dv + tok * p.dv_row + (long)hk * p.dv_head + c : (T*)p.dk + tok * p.dk_row + (long)hk * p.dk_head + c;
        const float f = which ? 1.f : p.scale;
        dst[0] = (T)(a.x * f); dst[1] = (T)(a.y * f); dst[2] = (T)(a.z * f); dst[3] = (T)(a.w * f);
    }
}
