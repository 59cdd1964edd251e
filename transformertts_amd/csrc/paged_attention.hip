// Attention of a few new tokens a sequence over the paged cache (a decoding step), the join of split keys, and the entry point.
//
// A decoding step is bound by the cache: every key and value is read once and meets G x (new tokens) rows.  So the workgroup's waves
// split the KEYS of one 32-row tile, not its rows: each wave owns every NW-th block of 32 keys, brings it in by itself
// (global -> LDS, 16 bytes a lane, no registers and no barrier in between), keeps its own running maximum, sum and output, and
// the waves are joined once at the end.  NBUF blocks a wave are in flight.
//
// The loads of a block are counted: every stage issues the same number of LDS-DMA instructions (K, V, the exponents of an e4m3
// cache, and the page numbers of the block that will take this stage's place NBUF blocks on), beyond the range with clamped
// addresses, so "stage j has landed" is one s_waitcnt and page numbers never stall the stream.
//
// e4m3 values stay bytes in LDS.  K fragments are converted with the row's scale (a lane is a key); V fragments come through the
// transposing 8-bit LDS read, and the value scales multiply the probabilities instead (both exact: powers of two).
//
// Measured (average of 150 launches under the profiler, the least in brackets): 32 single tokens over 262 .. 8192 keys, 16 / 4 heads of 128,
// bf16 pages of 16: 42 us (41), 5.5 TB/s, and 6.4 for the join; two over 131072 and 70001 keys, 32 / 8 heads, e4m3 pages of 64: 81 us (75),
// 5.1 TB/s, and 13.  The tile form, chunks of 512 + 384 + 97 + 1 tokens over 16384 .. 97 keys, 16 / 4 heads: 131 us (122), 730 TFLOP/s, and
// 15 for the join.
// Other types, a replayed call with its join, beside the time of its bytes at 6.5 TB/s or of its products: fp32, 32 single tokens over
// 100 .. 8192 keys, 16 / 4 heads of 128, 174 us (71: LDS holds two waves of two blocks a compute unit), of 64, 65 (36), 8 / 2 heads of 192,
// 259 (53: one such wave, and 88 registers spilled inside the counted loop, whose reloads wait for the blocks in flight); over e4m3 pages
// 98 (18), and of 192, which spills none, 83 (13).  The chunks above in fp32 1276 (624), over e4m3 pages 176 (72), fp32 over e4m3 1478 (624).
#include "seq_common.h"

template <int N> __device__ __forceinline__ void pg_wait() {
    static_assert(N >= 0 && N < 64, "the counter has six bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// 8 e4m3 bytes times a power of two
typedef __bf16 pg_bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void pg_cvt8(uint2 w, float scale, bf16x8& f) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = i ? w.y : w.x;
        const pg_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, scale, true);
        f[4 * i] = a[0]; f[4 * i + 1] = a[1]; f[4 * i + 2] = b[0]; f[4 * i + 3] = b[1];
    }
}
__device__ __forceinline__ void pg_cvt8(uint2 w, float scale, f32x8& f) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = i ? w.y : w.x;
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
        f[4 * i] = a[0] * scale; f[4 * i + 1] = a[1] * scale; f[4 * i + 2] = b[0] * scale; f[4 * i + 3] = b[1] * scale;
    }
}

// Waves a SIMD (WPS), waves a workgroup and stages: as much in flight as the 160 KB of a compute unit hold, at most 63 counted
// loads.  The bytes of an e4m3 block are half, so two waves a SIMD have room: one converts and multiplies while the other waits.
template <typename T, typename CT, int DHP> struct PgCfg {
    static constexpr int ROWB = DHP * (int)sizeof(CT), BLOCK = 2 * 32 * ROWB;          // bytes of a block's keys and values
    static constexpr int WPS = sizeof(CT) == 1 && sizeof(T) == 2 && DHP <= 128 ? 2 : 1;
    static constexpr int NW = BLOCK <= 16384 ? 2 : 1;
    static constexpr int FIT = 36864 / (WPS * BLOCK), NBUF = FIT > 4 ? 4 : FIT < 2 ? 2 : FIT;
    static constexpr int STAGES = NW * NBUF * BLOCK, JOIN = NW * 32 * (DHP + 4) * 4, MAIN = STAGES > JOIN ? STAGES : JOIN;
    static constexpr int SIDE = NW * NBUF * 256 * (sizeof(CT) == 1 ? 2 : 1), LDS = MAIN + SIDE + NW * 256 + 256;
    static constexpr int BY_LDS = 163840 / LDS, BY_WAVES = 4 * WPS / NW, RESIDENT = BY_LDS < BY_WAVES ? BY_LDS : BY_WAVES;   // workgroups a compute unit
};

// keys of a split and wave at least: two blocks (8 single tokens over 200 .. 1500 keys: 19 us; 22 with four)
#define PG_LEAST 64

// TWO: probabilities in two parts (pg_two_parts).
template <typename T, typename CT, int DHP, bool TWO>
__global__ __launch_bounds__((64 * PgCfg<T, CT, DHP>::NW), (PgCfg<T, CT, DHP>::WPS)) void paged_rows_kernel(SeqFwdP p) {
    using C = PgCfg<T, CT, DHP>;
    using frag = typename SeqT<T>::frag;
    constexpr bool Q8 = sizeof(CT) == 1;
    constexpr int NW = C::NW, NBUF = C::NBUF, ROWB = C::ROWB, CH = ROWB / 16;
    using I = SeqImg<CT, DHP>;
    using A = SeqLane<T, DHP>;
    constexpr int NI = 32 * CH / 64, PER = 2 * NI + 1 + (Q8 ? 1 : 0), NS = DHP / 16, NCB = DHP / 32;
    constexpr int MAIN = C::MAIN, SIDE = NW * NBUF * 256;
    __shared__ __attribute__((aligned(1024))) unsigned char sm[C::LDS];
    const int lane = threadIdx.x & 63, l31 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned char* const mine = sm + wave * NBUF * C::BLOCK;
    uint32_t* const ids = reinterpret_cast<uint32_t*>(sm + MAIN + wave * NBUF * 256);
    uint32_t* const exps = reinterpret_cast<uint32_t*>(sm + MAIN + SIDE + wave * NBUF * 256);
    float* const mls = reinterpret_cast<float*>(sm + MAIN + (Q8 ? 2 : 1) * SIDE);           // [NW][32][2]

    const int hk = blockIdx.x % p.Hkv;
    const SeqUnit un = find_unit(p.starts, p.lens, 1, p.most, p.B, p.tokens, p.G, 32, p.slots, 32 * NW, PG_LEAST * NW, blockIdx.x / p.Hkv, false);
    if (un.t.seq < 0) {
        if (p.zero_rest) seq_zero_rest<T>((T*)p.o, p.o_row, p.o_head, p.starts, p.B, p.tokens, p.G, 32, hk * p.G, p.dh, un.t.tile);
        return;
    }
    const int rows = un.t.n * p.G, r = un.t.tile * 32 + l31, len = un.len, off = len - un.t.n;
    const bool rok = r < rows;
    const int tok = r / p.G, head = hk * p.G + r - tok * p.G;
    const int lim = rok ? min(max(off + tok + 1, 0), len) : 0;
    const int last = min(un.t.tile * 32 + 31, rows - 1) / p.G;
    int kend = min(min(max(off + last + 1, 0), len), p.most);
    const int kbeg = min(un.split * un.per, kend);
    kend = min(kbeg + un.per, kend);
    const int full = off + un.t.tile * 32 / p.G + 1;                                        // keys that every row of the tile sees

    frag qf[NS];
    {
        const T* qr = (const T*)p.q + (long)(un.t.s0 + tok) * p.q_row + (long)head * p.q_head;
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = seq_load8<T>(qr, 16 * s + 8 * hh, rok && 16 * s + 8 * hh < p.dh);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) asm volatile("" : "+v"(qf[s]));      // waited for here: inside the loop that wait would drain the stream
    f32x16 o[NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[cb][i] = 0.f;
    float m = -INFINITY, l = 0.f;

    const int nblk = (kend - kbeg + 31) / 32, nb = nblk > wave ? (nblk - wave + NW - 1) / NW : 0;     // this wave's blocks
    if (nb > 0) {
        const int* trow = p.pg.table + (long)un.t.seq * p.pg.table_width;
        const int pmask = (1 << p.pg.shift) - 1, rowb = p.dh * (int)sizeof(CT);
        const uint32_t pageb = (uint32_t)rowb << p.pg.shift;
        auto key_of = [&](int x) { return min(kbeg + (x * NW + wave) * 32 + l31, kend - 1); };
        auto ask_ids = [&](int x, int st) { seq_dma4(trow + (key_of(x) >> p.pg.shift), seq_lds(ids + st * 64)); };
        uint32_t bad[NBUF];
        // block x into stage st: its page numbers have landed there
        auto request = [&](int x, int st) {
            const int key = key_of(x);
            const uint32_t id = ids[st * 64 + lane];
            const bool wrong = id >= (uint32_t)p.pg.n_pages;
            bad[st] = (uint32_t)__ballot(wrong);
            const uint32_t head_page = (wrong ? 0u : id) * (uint32_t)p.pg.heads + (uint32_t)hk;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                              // the stage's last readers are done
            unsigned char* const img = mine + st * C::BLOCK;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int id16 = i * 64 + lane, row = id16 / CH, phys = id16 - row * CH, ch = (phys ^ I::swz(row)) * 16;
                const int rkey = min(kbeg + (x * NW + wave) * 32 + row, kend - 1) & pmask;
                const uint64_t src = (uint64_t)(uint32_t)__shfl((int)head_page, row, 64) * pageb + (uint32_t)(rkey * rowb + (ch < rowb ? ch : 0));
                seq_dma16((const char*)p.pg.k + src, seq_lds(img + i * 1024));
                seq_dma16((const char*)p.pg.v + src, seq_lds(img + 32 * ROWB + i * 1024));
            }
            if constexpr (Q8) seq_dma1((hh ? p.pg.ve : p.pg.ke) + (((uint64_t)head_page << p.pg.shift) + (uint32_t)(key & pmask)), seq_lds(exps + st * 64));
            ask_ids(x + NBUF, st);
        };
#pragma unroll
        for (int st = 0; st < NBUF; ++st) ask_ids(st, st);
        pg_wait<0>();
#pragma unroll
        for (int st = 0; st < NBUF; ++st) request(st, st);

        auto block = [&](int x, int st) {
            unsigned char* const Ks = mine + st * C::BLOCK;
            unsigned char* const Vs = Ks + 32 * ROWB;
            const int k0 = kbeg + (x * NW + wave) * 32;
            if (bad[st]) {                                                                  // rows of pages that are not there: zeros
#pragma unroll
                for (int i = 0; i < 2 * NI; ++i) {
                    const int id16 = i * 64 + lane, row = (id16 / CH) & 31;
                    if ((bad[st] >> row) & 1) *reinterpret_cast<uint4*>(Ks + id16 * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                if (Q8 && ((bad[st] >> l31) & 1)) exps[st * 64 + lane] = 127;
            }
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.f;
            if constexpr (Q8) {
                const float ks = seq_scale_of(exps[st * 64 + l31]);
#pragma unroll
                for (int t = 0; t < NS; ++t) {
                    frag f;
                    pg_cvt8(*reinterpret_cast<const uint2*>(Ks + I::at(l31, t) + 8 * hh), ks, f);
                    s = seq_mma(f, qf[t], s);
                }
            } else {
#pragma unroll
                for (int t = 0; t < NS; ++t) s = seq_mma(A::row(A::rows(Ks, lane), 0, t), qf[t], s);
            }
            if (k0 + 32 > full || k0 + 32 > kend) {
                const int seen = seq_rare(min(lim, kend) - k0);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (seq_rowmap(i, hh) >= seen) s[i] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
            mx = seq_half_max(mx) * p.c1;
            if (__ballot(mx > m + 8.f)) {                                                   // 8 binary digits of slack, as in the tile kernels
                const float mn = fmaxf(m, mx), a = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
                m = mn;
                l *= a;
#pragma unroll
                for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[cb][i] *= a;
            }
            const float ms = m == -INFINITY ? 0.f : m;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = __builtin_amdgcn_exp2f(s[i] * p.c1 - ms);
                sum += s[i];
            }
            l += sum;
            if constexpr (Q8) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const uint4 e = *reinterpret_cast<const uint4*>(exps + st * 64 + 32 + 8 * g + 4 * hh);
                    s[4 * g] *= seq_scale_of(e.x); s[4 * g + 1] *= seq_scale_of(e.y); s[4 * g + 2] *= seq_scale_of(e.z); s[4 * g + 3] *= seq_scale_of(e.w);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                frag pf, pr;
                seq_to_frag(s, t, pf);
                if constexpr (TWO) seq_to_rest(s, t, pf, pr);
#pragma unroll
                for (int cb = 0; cb < NCB; ++cb) {
                    frag f;
                    if constexpr (Q8) {
                        typedef int pg_v2i __attribute__((ext_vector_type(2)));
                        typedef __attribute__((address_space(3))) pg_v2i* lds_ptr;
                        const int j = lane & 15, e = j >> 1, row = 16 * t + 8 * (e >> 2) + 4 * hh + (e & 3), ch = cb * 2 + ((lane >> 4) & 1);
                        const pg_v2i w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_ptr)(Vs + I::at(row, ch) + 8 * (j & 1)));
                        pg_cvt8(make_uint2((uint32_t)w[0], (uint32_t)w[1]), 1.f, f);
                    } else {
                        f = A::col(A::cols(Vs, lane), 0, t, cb);
                    }
                    o[cb] = seq_mma(f, pf, o[cb]);
                    if constexpr (TWO) o[cb] = seq_mma(f, pr, o[cb]);
                }
            }
        };
        for (int x = 0; x < nb; x += NBUF) {
#pragma unroll
            for (int st = 0; st < NBUF; ++st) {
                if (x + st < nb) {
                    pg_wait<(NBUF - 1) * PER>();
                    block(x + st, st);
                    request(x + st + NBUF, st);
                }
            }
        }
        pg_wait<0>();                                                                       // the clamped requests behind the end
    }
    // ---- join the waves ----
    l = seq_half_sum(l);
    if (hh == 0) *reinterpret_cast<float2*>(mls + (wave * 32 + l31) * 2) = make_float2(m, l);
    __syncthreads();
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, mls[(w * 32 + l31) * 2]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float2 v = *reinterpret_cast<const float2*>(mls + (w * 32 + l31) * 2);
        if (v.y != 0.f) L += v.y * __builtin_amdgcn_exp2f(v.x - M);
    }
    const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - M);
    constexpr int LDO = DHP + 4;
    float* const mo = reinterpret_cast<float*>(sm) + wave * 32 * LDO;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(mo + l31 * LDO + cb * 32 + 8 * g + 4 * hh) =
                l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[cb][4 * g] * f, o[cb][4 * g + 1] * f, o[cb][4 * g + 2] * f, o[cb][4 * g + 3] * f);
    float* const fin = mls + NW * 64;                                                       // [32][2]
    if (wave == 0 && hh == 0) *reinterpret_cast<float2*>(fin + 2 * l31) = make_float2(M, L);
    __syncthreads();
    const int per = p.dh / 4, live = min(32, rows - un.t.tile * 32);
    const long ubase = ((un.first + (long)un.split * un.t.ntile) * p.Hkv + hk) * 32;
    for (int i = threadIdx.x; i < live * per; i += 64 * NW) {
        const int row = i / per, c = (i - row * per) * 4;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm) + (w * 32 + row) * LDO + c);
            a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
        }
        const float2 ml = *reinterpret_cast<const float2*>(fin + 2 * row);
        if (un.nsplit > 1) {
            *reinterpret_cast<float4*>(p.part_o + (ubase + row) * p.dh + c) = a;
            if (c == 0) *reinterpret_cast<float2*>(p.part_ml + (ubase + row) * 2) = ml;
            continue;
        }
        const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
        const int rr = un.t.tile * 32 + row, t = rr / p.G;
        T* dst = (T*)p.o + (long)(un.t.s0 + t) * p.o_row + (long)(hk * p.G + rr - t * p.G) * p.o_head + c;
        if constexpr (sizeof(T) == 2) {
            bf16x4 h = {(__bf16)(a.x * inv), (__bf16)(a.y * inv), (__bf16)(a.z * inv), (__bf16)(a.w * inv)};
            *reinterpret_cast<bf16x4*>(dst) = h;
        } else {
            *reinterpret_cast<float4*>(dst) = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
        }
    }
}

// Joins: o = sum_z 2^(m_z - m) o_z / sum_z 2^(m_z - m) l_z over the splits z of a row.
//
// Few rows of many splits (the rows form): a wave a row (grid y: groups of four rows).  A wave is 64 / LPR groups of LPR lanes;
// group g takes the splits z = g (mod 64 / LPR), four elements a lane, and the groups are added.
struct PgJoinP { SeqFwdP f; int quantum, least; };
template <typename T, int LPR>
__global__ __launch_bounds__(256) void paged_join_kernel(PgJoinP j) {
    const SeqFwdP& p = j.f;
    constexpr int NG = 64 / LPR;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int hk = blockIdx.x % p.Hkv;
    const SeqUnit un = find_unit(p.starts, p.lens, 1, p.most, p.B, p.tokens, p.G, 32, p.slots, j.quantum, j.least, blockIdx.x / p.Hkv, true);
    if (un.t.seq < 0 || un.nsplit < 2) return;
    if (un.first + (long)(un.nsplit - 1) * un.t.ntile >= seq_split_units(p.tokens, p.B, p.G, 32, p.slots)) return;      // (`starts` that overlap)
    const int rows = un.t.n * p.G, live = min(32, rows - un.t.tile * 32);
    const int c = (lane % LPR) * 4, g = lane / LPR;
    for (int row = blockIdx.y * 4 + wave; row < live; row += 4 * gridDim.y) {
        float m = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const long step = 32L * p.Hkv * un.t.ntile, base = (un.first * p.Hkv + hk) * 32 + row;
        for (int z0 = 0; z0 < un.nsplit; z0 += 64) {
            float2 ml = make_float2(-INFINITY, 0.f);
            if (z0 + lane < un.nsplit) ml = *reinterpret_cast<const float2*>(p.part_ml + (base + (z0 + lane) * step) * 2);
            const float top = fmaxf(m, wave_max(ml.x)), a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
            const float w = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
            l = l * a + wave_sum(w * ml.y);
            m = top;
            acc.x *= a; acc.y *= a; acc.z *= a; acc.w *= a;
            const int n = min(64, un.nsplit - z0);
            // eight loads at a time, of every split: an empty one left its rows unwritten, its values are dropped, not its load
            for (int z = 0; z < n; z += 8 * NG) {
                float4 b[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    b[i] = *reinterpret_cast<const float4*>(p.part_o + (base + (z0 + min(z + i * NG + g, n - 1)) * step) * p.dh + (c < p.dh ? c : 0));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = z + i * NG + g;
                    const float wz = __shfl(w, at & 63, 64);
                    const bool live = at < n && wz != 0.f;
                    acc.x += live ? wz * b[i].x : 0.f; acc.y += live ? wz * b[i].y : 0.f;
                    acc.z += live ? wz * b[i].z : 0.f; acc.w += live ? wz * b[i].w : 0.f;
                }
            }
        }
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1) {
            acc.x += __shfl_xor(acc.x, o, 64); acc.y += __shfl_xor(acc.y, o, 64);
            acc.z += __shfl_xor(acc.z, o, 64); acc.w += __shfl_xor(acc.w, o, 64);
        }
        if (g != 0 || c >= p.dh) continue;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int rr = un.t.tile * 32 + row, t = rr / p.G;
        T* dst = (T*)p.o + (long)(un.t.s0 + t) * p.o_row + (long)(hk * p.G + rr - t * p.G) * p.o_head + c;
        dst[0] = (T)(acc.x * inv); dst[1] = (T)(acc.y * inv); dst[2] = (T)(acc.z * inv); dst[3] = (T)(acc.w * inv);
    }
}
// Many rows of few splits (the tile form): 16 rows a workgroup (grid y), four elements a thread, over the splits in their order,
// four of them in flight.
template <typename T>
__global__ __launch_bounds__(256) void paged_join_tiles_kernel(PgJoinP j) {
    const SeqFwdP& p = j.f;
    const int hk = blockIdx.x % p.Hkv;
    const SeqUnit un = find_unit(p.starts, p.lens, 1, p.most, p.B, p.tokens, p.G, 128, p.slots, j.quantum, j.least, blockIdx.x / p.Hkv, true);
    if (un.t.seq < 0 || un.nsplit < 2) return;
    if (un.first + (long)(un.nsplit - 1) * un.t.ntile >= seq_split_units(p.tokens, p.B, p.G, 128, p.slots)) return;      // (`starts` that overlap)
    const int r0 = un.t.tile * 128 + 16 * blockIdx.y, live = min(16, un.t.n * p.G - r0), per = p.dh / 4;
    const long step = 128L * p.Hkv * un.t.ntile;
    for (int i = threadIdx.x; i < live * per; i += 256) {
        const int row = i / per, c = (i - row * per) * 4;
        const long base = (un.first * p.Hkv + hk) * 128 + 16 * blockIdx.y + row;
        float m = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int z0 = 0; z0 < un.nsplit; z0 += 4) {
            float2 ml[4];
            float4 b[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const long at = base + min(z0 + z, un.nsplit - 1) * step;
                ml[z] = *reinterpret_cast<const float2*>(p.part_ml + 2 * at);
                b[z] = *reinterpret_cast<const float4*>(p.part_o + at * p.dh + c);
            }
            float top = m;
#pragma unroll
            for (int z = 0; z < 4; ++z) top = fmaxf(top, ml[z].x);
            const float ms = top == -INFINITY ? 0.f : top, a = __builtin_amdgcn_exp2f(m - ms);
            m = top;
            l *= a;
            acc.x *= a; acc.y *= a; acc.z *= a; acc.w *= a;
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                if (z0 + z >= un.nsplit || ml[z].y == 0.f) continue;      // (an empty split left its rows unwritten)
                const float w = __builtin_amdgcn_exp2f(ml[z].x - ms);
                l += w * ml[z].y;
                acc.x += w * b[z].x; acc.y += w * b[z].y; acc.z += w * b[z].z; acc.w += w * b[z].w;
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int rr = r0 + row, t = rr / p.G;
        T* dst = (T*)p.o + (long)(un.t.s0 + t) * p.o_row + (long)(hk * p.G + rr - t * p.G) * p.o_head + c;
        dst[0] = (T)(acc.x * inv); dst[1] = (T)(acc.y * inv); dst[2] = (T)(acc.z * inv); dst[3] = (T)(acc.w * inv);
    }
}
template <typename T>
static void pg_join_launch(const PgJoinP& j, bool rows_form, hipStream_t st) {
    const SeqFwdP& p = j.f;
    if (!rows_form) {
        hipLaunchKernelGGL((paged_join_tiles_kernel<T>), dim3((unsigned)(seq_units(p.tokens, p.B, p.G, 128) * p.Hkv), 8), dim3(256), 0, st, j);
        return;
    }
    const int groups = (int)((p.tokens * (long)p.G + 3) / 4);
    const dim3 g((unsigned)(seq_units(p.tokens, p.B, p.G, 32) * p.Hkv), (unsigned)(groups < 8 ? groups : 8));
    if (p.dh <= 64) hipLaunchKernelGGL((paged_join_kernel<T, 16>), g, dim3(256), 0, st, j);
    else if (p.dh <= 128) hipLaunchKernelGGL((paged_join_kernel<T, 32>), g, dim3(256), 0, st, j);
    else hipLaunchKernelGGL((paged_join_kernel<T, 64>), g, dim3(256), 0, st, j);
}

// ---- launches -----------------------------------------------------------------------------------------
// The rows form: rows of whole 16-byte pieces, and up to 16 of them a sequence on average in a bf16 cache (64 sequences of 512
// keys, 16 heads of 64: 58 us against the tile form's 34 with 8 rows, 71 against 32 with 32; 8 of 4096, 32 / 8 heads of 128: 37
// against 36 with 8, 41 against 37 with 32, 108 against 61 with 256; one row, 32 ragged ones, 8 heads of 64: 69 against 80), up to
// 64 elsewhere, where the tile form spends its time on converting and multiplying rows that are not there (e4m3, 64 sequences of
// 4096 keys, 32 / 8 heads of 128: 139 us against 164 with 32 rows, 148 against 175 with 64, 283 against 183 with 128; fp32, 32
// ragged ones, 4 heads of 64: 69 against 263 with one row).
static bool pg_rows_form(int B, int tokens, int G, int dh, int cache_dtype) {
    const int size = cache_dtype == TTSMI_F32 ? 4 : cache_dtype == TTSMI_E4M3 ? 1 : 2;
    return (long)tokens * G <= (size == 2 ? 16L : 64L) * B && dh * size % 16 == 0;
}
// Key splits a key head: together as many workgroups as the card holds at once; none where the tiles alone fill it.
template <typename T, typename CT>
static int pg_resident(int dh) {
    return 256 * (dh <= 64 ? PgCfg<T, CT, 64>::RESIDENT : dh <= 128 ? PgCfg<T, CT, 128>::RESIDENT : PgCfg<T, CT, 192>::RESIDENT);
}
static int pg_slots(int B, int tokens, int Hkv, int G, int dh, bool rows_form, int cache_dtype, int dtype) {
    // (the tile form, before its page lookups became scalars: 8192 keys and 512 new tokens of 32 / 8 heads of 128, 128 tiles: 93 us at
    // 512, 104 at 1024, 111 at 256, 178 unsplit - 83 at 512 since; 16 sequences of 2048 keys and 64 new tokens, 256 tiles: 56 us
    // unsplit, 66 at 512; [300, 200, 100] new over [400, 300, 20000] of 16 heads of 64: 45 us at 512, 53 at 1024, 369 unsplit)
    int all = dtype != TTSMI_F32 && dh <= 128 ? 512 : 256;
    if (rows_form) {
        if (dtype == TTSMI_F32) all = cache_dtype == TTSMI_E4M3 ? pg_resident<float, uint8_t>(dh) : pg_resident<float, float>(dh);
        else all = cache_dtype == TTSMI_E4M3 ? pg_resident<__bf16, uint8_t>(dh) : pg_resident<__bf16, __bf16>(dh);
    }
    const int fill = all / Hkv < 1 ? 1 : all / Hkv;
    return !rows_form && ((long)tokens * G / 128 + (B + 1) / 2) * Hkv >= all ? 0 : fill;
}
// Probabilities of bf16 queries as operands of two parts (seq_to_rest) where a sequence has one tile of rows on average: the kernel
// waits for memory, the second part costs 1 - 2 % (32 single tokens over 100 .. 8192 keys, 16 / 4 heads of 128, with the join: bf16
// 51.8 -> 52.5 us, e4m3 36.3 -> 36.9; 32 rows each of 64 sequences of 4096 e4m3 keys, 32 / 8 heads: 137 -> 140), and the error of one part, up to
// 1.6 times the output's own rounding in single tokens, is gone.  With two tiles it does not wait: 64 rows each, 155 -> 179 us.
static bool pg_two_parts(const SeqFwdP& p) { return (long)p.tokens * p.G <= 32L * p.B; }
template <typename T, typename CT>
static void pg_rows_launch(const SeqFwdP& p, PgJoinP& j, hipStream_t st) {
    const dim3 g((unsigned)(seq_split_units(p.tokens, p.B, p.G, 32, p.slots) * p.Hkv));
#define PG_GO(D)                                                                                                           \
    do {                                                                                                                   \
        constexpr int NW = PgCfg<T, CT, D>::NW;                                                                               \
        j.quantum = 32 * NW; j.least = PG_LEAST * NW;                                                                         \
        if constexpr (sizeof(T) == 2) {                                                                                    \
            if (pg_two_parts(p)) {                                                                                         \
                hipLaunchKernelGGL((paged_rows_kernel<T, CT, D, true>), g, dim3(64 * NW), 0, st, p);                       \
                break;                                                                                                     \
            }                                                                                                              \
        }                                                                                                                  \
        /* (over a bf16 cache this form has 16 rows a sequence at most, pg_rows_form: two parts always) */                 \
        if constexpr (sizeof(T) == 4 || sizeof(CT) == 1)                                                                   \
            hipLaunchKernelGGL((paged_rows_kernel<T, CT, D, false>), g, dim3(64 * NW), 0, st, p);                          \
    } while (0)
    if (p.dh <= 64) PG_GO(64);
    else if (p.dh <= 128) PG_GO(128);
    else PG_GO(192);
#undef PG_GO
}

extern "C" size_t ttsmi_paged_attention_ws_bytes(int B, int tokens, int H, int Hkv, int dh, int cache_dtype, int dtype) {
    if (B < 0 || tokens <= 0 || H <= 0 || Hkv <= 0 || dh <= 0) return 0;
    const int G = H / Hkv;
    const bool rows_form = pg_rows_form(B, tokens, G, dh, cache_dtype);
    const int slots = pg_slots(B, tokens, Hkv, G, dh, rows_form, cache_dtype, dtype), R = rows_form ? 32 : 128;
    return slots == 0 ? 0 : (size_t)seq_split_units(tokens, B, G, R, slots) * Hkv * R * (dh + 2) * sizeof(float);
}
extern "C" int ttsmi_paged_attention(const void* q, int64_t q_row, int64_t q_head, const void* k_pages, const void* v_pages,
                                     const uint8_t* k_exp, const uint8_t* v_exp, int cache_dtype, int n_pages, int page_size,
                                     const int32_t* table, int table_width, const int32_t* starts, const int32_t* lens, int B,
                                     int tokens, int H, int Hkv, int dh, float scale, void* out, int64_t o_row, int64_t o_head,
                                     int zero_rest, void* ws, size_t ws_bytes, int dtype, ttsmi_stream_t stream) {
    SEQ_CHECK_COMMON("paged_attention");
    TTSMI_CHECK_ARG(cache_dtype == dtype || cache_dtype == TTSMI_E4M3, "paged_attention: cache dtype %d with tensors of dtype %d", cache_dtype, dtype);
    SEQ_CHECK_PAGES("paged_attention");
    if (tokens == 0) return TTSMI_OK;
    SEQ_CHECK_CACHE("paged_attention");
    TTSMI_CHECK_ARG(seq_strides_ok(q, q_row, q_head, 0, dtype) && seq_strides_ok(out, o_row, o_head, 0, dtype),
                    "paged_attention: a tensor is null or its rows or heads are not 16-byte aligned");
    SeqFwdP p = {};
    p.q = q; p.q_row = q_row; p.q_head = q_head; p.o = out; p.o_row = o_row; p.o_head = o_head; p.starts = starts; p.lens = lens;
    p.pg.k = k_pages; p.pg.v = v_pages; p.pg.ke = k_exp; p.pg.ve = v_exp; p.pg.table = table; p.pg.table_width = table_width;
    p.pg.n_pages = n_pages; p.pg.shift = __builtin_ctz(page_size); p.pg.heads = Hkv; p.pg.dh = dh;
    p.B = B; p.tokens = tokens; p.Hkv = Hkv; p.G = H / Hkv; p.dh = dh; p.causal = 1; p.c1 = scale * SEQ_LOG2E; p.zero_rest = zero_rest != 0;
    const size_t need = ttsmi_paged_attention_ws_bytes(B, tokens, H, Hkv, dh, cache_dtype, dtype);
    if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) {
        ttsmi_set_error("paged_attention: workspace of %zu bytes, %zu (16-byte aligned) needed", ws_bytes, need);
        return TTSMI_ERR_WORKSPACE;
    }
    const bool rows_form = pg_rows_form(B, tokens, p.G, dh, cache_dtype);
    PgJoinP j = {};
    j.quantum = dtype == TTSMI_F32 ? 32 : 64; j.least = SEQ_TILE_LEAST;
    p.slots = pg_slots(B, tokens, Hkv, p.G, dh, rows_form, cache_dtype, dtype);
    if (p.slots > 0) {
        const int R = rows_form ? 32 : 128;
        p.part_o = (float*)ws;
        p.part_ml = (float*)ws + (size_t)seq_split_units(tokens, B, p.G, R, p.slots) * Hkv * R * dh;
    }
    const long held = (long)table_width << p.pg.shift;
    p.most = n_pages == 0 ? 0 : (int)(held < (1l << 30) ? held : 1l << 30);
    hipStream_t st = (hipStream_t)stream;
    if (rows_form) {
        if (dtype == TTSMI_F32) cache_dtype == TTSMI_E4M3 ? pg_rows_launch<float, uint8_t>(p, j, st) : pg_rows_launch<float, float>(p, j, st);
        else cache_dtype == TTSMI_E4M3 ? pg_rows_launch<__bf16, uint8_t>(p, j, st) : pg_rows_launch<__bf16, __bf16>(p, j, st);
    } else {
        const int rc = seq_paged_tiles(p, dtype, cache_dtype, st);
        if (rc != TTSMI_OK) return rc;
    }
    ttsmi_note_kernel(rows_form ? "paged_rows_kernel" : "seq_attn_fwd_kernel");
    if (p.slots > 0) {
        j.f = p;
        if (dtype == TTSMI_F32) pg_join_launch<float>(j, rows_form, st);
        else pg_join_launch<__bf16>(j, rows_form, st);
    }
    TTSMI_CHECK_LAUNCH("paged_attention");
    return TTSMI_OK;
}
