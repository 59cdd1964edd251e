// Attention over packed sequences (forward) and of new tokens over a paged key / value cache.
//
//   s_ij = scale q_i . k_j   (j at or before i where causal),  p = softmax_j(s),  o_i = sum_j p_ij v_j,  lse_i = log sum_j exp s_ij
//
// One pass over the keys with a running maximum and sum (fp32, log2 domain).  A workgroup of four waves owns 128 rows of one
// sequence and key head (seq_common.h: rows are (token, query head of the group) pairs), 32 rows a wave.  The wave forms the
// TRANSPOSED score tile S^T = K Q^T, so that a lane holds one row's scores for 16 keys: the softmax is in-lane plus one exchange
// of the two half-waves, and the accumulator registers, rounded, ARE the B operand of O^T += V^T P^T.
// Long prompts are bound by the matrix and the vector pipes together: the matrix pipes are busy half of the time, a wave's vector
// instructions (the softmax, 16 clocks an exponential) take as long as its products, and the two waves that the registers leave a
// SIMD overlap only in part.  LDS is busy a third of the time, without bank conflicts.  (Of 342 us a pass, taking away the reads of
// fragments saved 96, either product 80 .. 90, the loads 42, the exponentials 29.)  Batches of utterances are bound by balance - with all
// workgroups resident the slowest compute unit's three whole walks are the time -, the small fp32 batch by waits: 128 KB of LDS leave one
// wave a SIMD, and 60 of its 316 workgroups run in a second round.  One short utterance is a chain: starts, then Q, then K and V.
// Measured (average of 150 launches under the profiler, the least in brackets): prompts of 8192 + 3001 + 513 + 1 tokens, 16 / 8 heads of
// 128, causal, bf16: 329 us (309), 950 TFLOP/s (1010) where a large library product reaches 1330; 6000 + 1999 + 193 of 16 / 2 heads: 180 us
// (174), 910 TFLOP/s; 32 utterances of 202 .. 900, 4 heads of 64: 28 us; fp32, 8 utterances, 4 / 2 heads of 64: 26 us (38 with two waves a
// row block); 61 tokens of 2 heads of 192: 9 us.
// Where tiles are few, two or four waves share a row block and the keys (seq_key_parts).
// Over a cache the keys can be split over workgroups (find_unit): each leaves its maximum, sum and unnormalised output, and a second
// launch joins them (paged_attention.hip).
#include "seq_common.h"

// CT: the cache's element type for PAGED (T, or uint8_t = e4m3).  WIDE: pages of whole load instructions (the RPI rows that one
// brings), so that an instruction has one page and its address is a scalar base and a constant lane offset; without it every lane
// looks its rows up, forming 64-bit addresses of its own.
// TWO: probabilities in two parts (seq_two_parts).
template <typename T, typename CT, int DHP, bool PAGED, int KS = 1, bool WIDE = false, bool TWO = false>
__global__ __launch_bounds__(256, (DHP <= 128 && sizeof(T) == 2) ? 2 : 1) void seq_attn_fwd_kernel(SeqFwdP p) {
    using I = SeqImg<T, DHP>;
    using frag = typename SeqT<T>::frag;
    constexpr int KW = SeqKeys<T, DHP, KS>::KW, KT = KW * KS, NKB = KW / 32, NS = DHP / 16, NCB = DHP / 32;
    constexpr int ROWS = 128 / KS;
    using D = SeqDma<T, DHP, KT>;
    constexpr bool Q8 = PAGED && sizeof(CT) == 1;
    constexpr int IMG = KT * I::ROWB, ITEMS = D::NI;      // 16-byte pieces a lane and tile image
    __shared__ __attribute__((aligned(1024))) unsigned char sm[4 * IMG];         // two stages of a K and a V tile

    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % p.Hkv, unit = blockIdx.x / p.Hkv;       // bid % 8 = XCD: the tiles of a key head share few L2s
    SeqUnit un;
    if constexpr (PAGED) {
        if (p.slots > 0) un = find_unit(p.starts, p.lens, 1, p.most, p.B, p.tokens, p.G, 128, p.slots, KT, SEQ_TILE_LEAST, unit, false);
    }
    const bool splits = PAGED && p.slots > 0;
    const SeqTile st = splits ? un.t : find_tile(p.starts, p.B, p.tokens, p.G, ROWS, unit, !PAGED && p.causal);
    if (st.seq < 0) {
        if (p.zero_rest) seq_zero_rest<T>((T*)p.o, p.o_row, p.o_head, p.starts, p.B, p.tokens, p.G, ROWS, hk * p.G, p.dh, st.tile);
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
    constexpr int RW = 4 / KS;                            // row blocks of the workgroup; wave: row block wave % RW, part wave / RW
    const int kpart = wave / RW, wrow = tile * ROWS + wave % RW * 32;
    const int r = wrow + l31;
    const bool rok = r < rows;
    const int tok = r / p.G, head = hk * p.G + r - tok * p.G;
    const int lim = !rok ? 0 : p.causal ? min(max(off + tok + 1, 0), len) : len;
    // the same for the workgroup's last row, and for this wave's: no key behind is fetched / multiplied
    const int last = min(tile * ROWS + ROWS - 1, rows - 1) / p.G;
    int kend = p.causal ? min(max(off + last + 1, 0), len) : len, kbeg = 0;
    if (PAGED) kend = min(kend, p.most);
    const bool part = splits && un.nsplit > 1;
    if (part) {
        kbeg = min(un.split * un.per, kend);
        kend = min(kbeg + un.per, kend);
    }
    kbeg = __builtin_amdgcn_readfirstlane(kbeg);
    kend = __builtin_amdgcn_readfirstlane(kend);
    const int wlast = min(wrow + 31, rows - 1) / p.G;
    const int wend = wrow >= rows ? 0 : min(kend, p.causal ? max(off + wlast + 1, 0) : len);
    const int wfull = wrow + 31 < rows ? (p.causal ? off + wrow / p.G + 1 : len) : 0;     // keys that every row of the wave sees

    frag qf[NS];
    {
        const T* qr = (const T*)p.q + (long)(st.s0 + tok) * p.q_row + (long)head * p.q_head;
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = seq_load8<T>(qr, 16 * s + 8 * hh, rok && 16 * s + 8 * hh < p.dh);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) asm volatile("" : "+v"(qf[s]));          // waited for in front of the first DMA
    f32x16 o[NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[cb][i] = 0.f;
    float m = -INFINITY, l = 0.f;

    // ---- tile staging, two stages, one barrier a tile ----
    // Rows of this type: LDS-DMA; a row past the last key repeats it (its score is masked).  A paged tile's rows are looked up a
    // tile earlier, so that no load waits for another; rows of a page that is not there are cleared when they have landed.
    // e4m3 rows: through registers, converted on the way.
    uint32_t ko[ITEMS], vo[ITEMS];
    if constexpr (!PAGED) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            ko[i] = D::row(i, wave, lane) * (uint32_t)(p.k_row * (long)sizeof(T)) + D::piece(i, wave, lane, p.dh);
            vo[i] = D::row(i, wave, lane) * (uint32_t)(p.v_row * (long)sizeof(T)) + D::piece(i, wave, lane, p.dh);
        }
    }
    constexpr int RPI = 64 / I::CH;
    int pid[PAGED ? ITEMS : 1];                           // page numbers of the next tile's rows, as they come
    uint32_t gone = 0, gone_next = 0;                     // bit i: item i's row of the tile has no page
    uint2 wk[Q8 ? ITEMS : 1], wv[Q8 ? ITEMS : 1];
    uint32_t ek[Q8 ? ITEMS : 1], ev[Q8 ? ITEMS : 1];
    auto look = [&](int k0) {
        if constexpr (WIDE) {
            typedef __attribute__((address_space(4))) const int* scalar;                     // (a scalar load: uniform, and not written meanwhile)
            const scalar trow = (scalar)(p.pg.table + (long)st.seq * p.pg.table_width);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) pid[i] = trow[min(k0 + (wave + 4 * i) * RPI, kend - 1) >> p.pg.shift];
        } else if constexpr (PAGED) {
            const int* const trow = p.pg.table + (long)st.seq * p.pg.table_width;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int at = min(k0 + D::row(i, wave, lane), kend - 1) >> p.pg.shift;
                pid[i] = trow[at];
            }
        }
    };
    auto fetch = [&](int k0, int buf) {
        unsigned char* const img = sm + buf * 2 * IMG;
        long at[PAGED ? ITEMS : 1];                       // the lane's row of the pages; WIDE: the instruction's first row
        uint32_t in[WIDE ? ITEMS : 1];                    // WIDE: the lane's row behind it
        if constexpr (WIDE) {
            gone_next = 0;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int first = min(k0 + (wave + 4 * i) * RPI, kend - 1);
                const bool ok = (unsigned)pid[i] < (unsigned)p.pg.n_pages;
                if (!ok) gone_next |= 1u << i;
                at[i] = (((long)(ok ? pid[i] : 0) * p.pg.heads + hk) << p.pg.shift) + (first & ((1 << p.pg.shift) - 1));
                in[i] = min(lane / I::CH, kend - 1 - first);
            }
        } else if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) asm volatile("" : "+v"(pid[i]));                  // all of them, in front of the first load below
            gone_next = 0;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int key = min(k0 + D::row(i, wave, lane), kend - 1);
                const bool ok = (unsigned)pid[i] < (unsigned)p.pg.n_pages;
                if (!ok) gone_next |= 1u << i;
                at[i] = (((long)(ok ? pid[i] : 0) * p.pg.heads + hk) << p.pg.shift) + (key & ((1 << p.pg.shift) - 1));
            }
        }
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = (int)D::piece(i, wave, lane, p.dh) / (int)sizeof(T);
                wk[i] = wv[i] = make_uint2(0u, 0u);
                ek[i] = ev[i] = 127;
                if ((gone_next >> i) & 1) continue;
                const uint32_t off = (WIDE ? in[i] * (uint32_t)p.dh : 0) + c;
                const uint8_t* const a = (const uint8_t*)p.pg.k + at[i] * p.dh + off;
                const uint8_t* const b = (const uint8_t*)p.pg.v + at[i] * p.dh + off;
                if constexpr (sizeof(T) == 2) {
                    wk[i] = *reinterpret_cast<const uint2*>(a);
                    wv[i] = *reinterpret_cast<const uint2*>(b);
                } else {
                    wk[i].x = *reinterpret_cast<const uint32_t*>(a);
                    wv[i].x = *reinterpret_cast<const uint32_t*>(b);
                }
                ek[i] = p.pg.ke[at[i] + (WIDE ? in[i] : 0)];
                ev[i] = p.pg.ve[at[i] + (WIDE ? in[i] : 0)];
            }
        } else if constexpr (WIDE) {
            const uint32_t rb = (uint32_t)p.dh * (uint32_t)sizeof(T);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const uint32_t off = in[i] * rb + D::piece(i, wave, lane, p.dh);
                seq_dma16((const char*)p.pg.k + at[i] * rb, off, seq_lds(img + (wave + 4 * i) * 1024));
                seq_dma16((const char*)p.pg.v + at[i] * rb, off, seq_lds(img + IMG + (wave + 4 * i) * 1024));
            }
        } else if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const long src = at[i] * (p.dh * (long)sizeof(T)) + D::piece(i, wave, lane, p.dh);
                seq_dma16((const char*)p.pg.k + src, seq_lds(img + (wave + 4 * i) * 1024));
                seq_dma16((const char*)p.pg.v + src, seq_lds(img + IMG + (wave + 4 * i) * 1024));
            }
        } else {
            const char* const kb = (const char*)p.k + ((long)(st.s0 + k0) * p.k_row + (long)hk * p.k_head) * (long)sizeof(T);
            const char* const vb = (const char*)p.v + ((long)(st.s0 + k0) * p.v_row + (long)hk * p.v_head) * (long)sizeof(T);
            if (k0 + KT <= kend) {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    seq_dma16(kb, ko[i], seq_lds(img + (wave + 4 * i) * 1024));
                    seq_dma16(vb, vo[i], seq_lds(img + IMG + (wave + 4 * i) * 1024));
                }
            } else {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    const uint32_t row = min(D::row(i, wave, lane), kend - 1 - k0), c = D::piece(i, wave, lane, p.dh);
                    seq_dma16(kb, row * (uint32_t)(p.k_row * (long)sizeof(T)) + c, seq_lds(img + (wave + 4 * i) * 1024));
                    seq_dma16(vb, row * (uint32_t)(p.v_row * (long)sizeof(T)) + c, seq_lds(img + IMG + (wave + 4 * i) * 1024));
                }
            }
        }
    };
    auto land = [&](int buf) {                            // the wave's share of a tile is complete in LDS
        unsigned char* const img = sm + buf * 2 * IMG;
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                *reinterpret_cast<uint4*>(img + (wave + 4 * i) * 1024 + lane * 16) = seq_dequant_chunk<T>(wk[i], seq_scale_of(ek[i]));
                *reinterpret_cast<uint4*>(img + IMG + (wave + 4 * i) * 1024 + lane * 16) = seq_dequant_chunk<T>(wv[i], seq_scale_of(ev[i]));
            }
        } else if constexpr (PAGED) {
            gone = gone_next;
            if (__ballot(gone != 0)) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
                    if ((gone >> i) & 1)
                        *reinterpret_cast<uint4*>(img + (wave + 4 * i) * 1024 + lane * 16) = *reinterpret_cast<uint4*>(img + IMG + (wave + 4 * i) * 1024 + lane * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
        }
        seq_dma_barrier();
    };

    if (kbeg < kend) {
        look(kbeg);
        fetch(kbeg, 0);
        if (kbeg + KT < kend) look(kbeg + KT);
    }
    using A = SeqLane<T, DHP>;
    const uint32_t kbase = A::rows(sm, lane) + kpart * KW * I::ROWB, vbase = A::cols(sm + IMG, lane) + kpart * KW * I::ROWB;
    int buf = 0;
    for (int k0 = kbeg; k0 < kend; k0 += KT, buf ^= 1) {
        land(buf);
        if (k0 + KT < kend) {
            fetch(k0 + KT, buf ^ 1);
            look(k0 + 2 * KT);
        }
        const int kw = k0 + kpart * KW;                   // this wave's keys of the tile
        if (kw >= wend) continue;
        const uint32_t ka = kbase + buf * 2 * IMG, va = vbase + buf * 2 * IMG;
        f32x16 s[NKB];
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
            for (int t = 0; t < NS; ++t) s[kb] = seq_mma(A::row(ka, kb * 32, t), qf[t], s[kb]);
        }
        // The two waves of a SIMD are better off apart - one at its scores' product while the other is past it - so a wave that has its
        // scores goes first (8192 tokens, 16 / 8 heads of 128, causal: 306 -> 278 us; full, 2 x 4096: 287 -> 279).  The backward
        // passes do not gain by it.
        __builtin_amdgcn_s_setprio(1);
        if (kw + KW > wfull || kw + KW > kend) {
            const int seen = seq_rare(min(lim, kend) - kw);
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
        // The maximum follows with 8 binary digits of slack: until a score passes it by that much the probabilities are at most 2^8, no
        // less exact for it, and the output need not be scaled again (342 -> 332 us for prompts of 8192 + 3001 + 513 + 1 tokens).
        if (__ballot(mx > m + 8.f)) {
            const float mn = fmaxf(m, mx), a = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= a;
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[cb][i] *= a;
        }
        const float ms = m == -INFINITY ? 0.f : m;        // a row that has seen no key yet keeps p = 0
        float sum = 0.f;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kb][i] = __builtin_amdgcn_exp2f(s[kb][i] * p.c1 - ms);
                sum += s[kb][i];
            }
        l += sum;                                         // (this half-wave's keys; joined at the end)
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                frag pf;
                seq_to_frag(s[kb], t, pf);
                if constexpr (TWO) {
                    frag pr;
                    seq_to_rest(s[kb], t, pf, pr);
#pragma unroll
                    for (int cb = 0; cb < NCB; ++cb) {
                        const frag vf = A::col(va, kb * 32, t, cb);
                        o[cb] = seq_mma(vf, pr, seq_mma(vf, pf, o[cb]));
                    }
                } else {
#pragma unroll
                    for (int cb = 0; cb < NCB; ++cb) o[cb] = seq_mma(A::col(va, kb * 32, t, cb), pf, o[cb]);
                }
            }
        __builtin_amdgcn_s_setprio(0);
    }
    l = seq_half_sum(l);
    if constexpr (KS > 1) {                               // the parts of the keys: a row block's first wave takes over the others' sums
        constexpr int LDO = DHP + 4, PART = RW * 32 * (LDO + 2);
        float* mo = reinterpret_cast<float*>(sm) + (wave % RW * 32 + l31) * (LDO + 2);
        seq_dma_barrier();
        if (kpart > 0) {
            mo += (kpart - 1) * PART;
            if (hh == 0) *reinterpret_cast<float2*>(mo + LDO) = make_float2(m, l);
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float2*>(mo + cb * 32 + 8 * g + 4 * hh + 2 * e) = make_float2(o[cb][4 * g + 2 * e], o[cb][4 * g + 2 * e + 1]);
        }
        __syncthreads();
        if (kpart > 0) return;
#pragma unroll
        for (int x = 1; x < KS; ++x, mo += PART) {
            const float2 other = *reinterpret_cast<const float2*>(mo + LDO);
            const float mn = fmaxf(m, other.x), ms = mn == -INFINITY ? 0.f : mn;
            const float a = __builtin_amdgcn_exp2f(m - ms), b = __builtin_amdgcn_exp2f(other.x - ms);
            m = mn;
            l = l * a + other.y * b;
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[cb][i] = o[cb][i] * a + mo[cb * 32 + 8 * (i >> 2) + 4 * hh + (i & 3)] * b;
        }
    }
    if (!rok) return;
    const long slot = (long)hk * p.tokens * p.G + (long)st.s0 * p.G + r;
    if (part) {
        const long ps = ((un.first + (long)un.split * un.t.ntile) * p.Hkv + hk) * 128 + wave * 32 + l31;
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
                if (!PAGED && p.rest) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) h[e] = (__bf16)(o[cb][4 * g + e] * inv - (float)h[e]);
                    *reinterpret_cast<bf16x4*>((T*)p.rest + ((long)(st.s0 + tok) * p.Hkv * p.G + head) * p.dh + c) = h;
                }
            } else {
                *reinterpret_cast<float4*>(orow + c) = make_float4(o[cb][4 * g] * inv, o[cb][4 * g + 1] * inv, o[cb][4 * g + 2] * inv, o[cb][4 * g + 3] * inv);
            }
        }
}

// ---- launches -----------------------------------------------------------------------------------------

template <typename T, typename CT, int DHP, bool PAGED, int KS, bool WIDE = false, bool TWO = false>
static void seq_fwd_go(const SeqFwdP& p, long units, hipStream_t st) {
    hipLaunchKernelGGL((seq_attn_fwd_kernel<T, CT, DHP, PAGED, KS, WIDE, TWO>), dim3((unsigned)(units * p.Hkv)), dim3(256), 0, st, p);
}
template <typename T>
static int seq_packed_launch(const SeqFwdP& p, hipStream_t st) {
    const int parts = seq_key_parts(p.tokens, p.B, p.G, p.Hkv, p.dh, sizeof(T) == 4, p.causal);
    const long units = seq_units(p.tokens, p.B, p.G, 128 / parts);
    if constexpr (sizeof(T) == 2) {
        if (seq_two_parts(p.tokens, p.B, parts, false)) {
            if (p.dh <= 64) seq_fwd_go<T, T, 64, false, 2, false, true>(p, units, st);
            else if (p.dh <= 128) seq_fwd_go<T, T, 128, false, 2, false, true>(p, units, st);
            else seq_fwd_go<T, T, 192, false, 2, false, true>(p, units, st);
            ttsmi_note_kernel("seq_attn_fwd_kernel, keys in two");
            TTSMI_CHECK_LAUNCH("packed_attention_fwd");
            return TTSMI_OK;
        }
    }
    if (parts == 4) {
        if (p.dh <= 64) seq_fwd_go<T, T, 64, false, 4>(p, units, st);
        else if constexpr (sizeof(T) == 2) seq_fwd_go<T, T, 128, false, 4>(p, units, st);
    } else if (parts == 2) {
        if (p.dh <= 64) seq_fwd_go<T, T, 64, false, 2>(p, units, st);
        else if (p.dh <= 128) seq_fwd_go<T, T, 128, false, 2>(p, units, st);
        else if constexpr (sizeof(T) == 2) seq_fwd_go<T, T, 192, false, 2>(p, units, st);
    } else if (p.dh <= 64) seq_fwd_go<T, T, 64, false, 1>(p, units, st);
    else if (p.dh <= 128) seq_fwd_go<T, T, 128, false, 1>(p, units, st);
    else seq_fwd_go<T, T, 192, false, 1>(p, units, st);
    ttsmi_note_kernel(parts == 4 ? "seq_attn_fwd_kernel, keys in four" : parts == 2 ? "seq_attn_fwd_kernel, keys in two" : "seq_attn_fwd_kernel");
    TTSMI_CHECK_LAUNCH("packed_attention_fwd");
    return TTSMI_OK;
}
template <typename T, typename CT>
static int seq_paged_launch(const SeqFwdP& p, hipStream_t st) {
    const long units = p.slots > 0 ? seq_split_units(p.tokens, p.B, p.G, 128, p.slots) : seq_units(p.tokens, p.B, p.G, 128);
    // pages of 8 rows or more hold whole instructions of heads up to 128 (RPI 2 .. 8); an image row of 192 is no whole part of one
    const bool wide = p.pg.shift >= 3;
    if (p.dh <= 64 && wide) seq_fwd_go<T, CT, 64, true, 1, true>(p, units, st);
    else if (p.dh <= 64) seq_fwd_go<T, CT, 64, true, 1>(p, units, st);
    else if (p.dh <= 128 && wide) seq_fwd_go<T, CT, 128, true, 1, true>(p, units, st);
    else if (p.dh <= 128) seq_fwd_go<T, CT, 128, true, 1>(p, units, st);
    else seq_fwd_go<T, CT, 192, true, 1>(p, units, st);
    TTSMI_CHECK_LAUNCH("paged_attention");
    return TTSMI_OK;
}
// the tile form of the paged attention (paged_attention.hip)
int seq_paged_tiles(const SeqFwdP& p, int dtype, int cache_dtype, hipStream_t st) {
    if (dtype == TTSMI_F32)
        return cache_dtype == TTSMI_E4M3 ? seq_paged_launch<float, uint8_t>(p, st) : seq_paged_launch<float, float>(p, st);
    return cache_dtype == TTSMI_E4M3 ? seq_paged_launch<__bf16, uint8_t>(p, st) : seq_paged_launch<__bf16, __bf16>(p, st);
}

extern "C" int ttsmi_packed_attention_fwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                                          const void* v, int64_t v_row, int64_t v_head, const int32_t* starts, int B, int tokens,
                                          int H, int Hkv, int dh, float scale, int causal, void* out, int64_t o_row, int64_t o_head,
                                          float* lse, void* out_rest, int zero_rest, int dtype, ttsmi_stream_t stream) {
    SEQ_CHECK_COMMON("packed_attention_fwd");
    if (tokens == 0) return TTSMI_OK;
    TTSMI_CHECK_ARG(starts, "packed_attention_fwd: null starts");
    TTSMI_CHECK_ARG(seq_strides_ok(q, q_row, q_head, H / Hkv, dtype) && seq_strides_ok(k, k_row, k_head, 1, dtype) && seq_strides_ok(v, v_row, v_head, 1, dtype) &&
                        seq_strides_ok(out, o_row, o_head, 0, dtype), "packed_attention_fwd: a tensor is null or its rows or heads are not 16-byte aligned, or too far apart");
    TTSMI_CHECK_ARG(((uintptr_t)out_rest & 15) == 0, "packed_attention_fwd: out_rest is not 16-byte aligned");
    SeqFwdP p = {};
    p.q = q; p.q_row = q_row; p.q_head = q_head; p.k = k; p.k_row = k_row; p.k_head = k_head; p.v = v; p.v_row = v_row; p.v_head = v_head;
    p.o = out; p.rest = dtype == TTSMI_BF16_IO ? out_rest : nullptr; p.zero_rest = zero_rest != 0; p.o_row = o_row; p.o_head = o_head; p.lse = lse; p.starts = starts;
    p.B = B; p.tokens = tokens; p.Hkv = Hkv; p.G = H / Hkv; p.dh = dh; p.causal = causal != 0; p.c1 = scale * SEQ_LOG2E;
    return dtype == TTSMI_F32 ? seq_packed_launch<float>(p, (hipStream_t)stream) : seq_packed_launch<__bf16>(p, (hipStream_t)stream);
}
