// Shared device code of the sequence operators (attention over packed sequences, the paged key / value cache and attention
// over it): element types, MFMA operand fragments, the row / tile maps of packed sequences and LDS tile images.
//
// Rows.  Sequence b owns the packed tokens [starts[b], starts[b + 1]).  The G = H / Hkv query heads of one key head share its
// keys and values, so they are worked on together: row r of sequence b and key head hk is token r / G, query head hk G + r % G.
// A tile is 128 (forward, dQ) such rows of ONE sequence.  Which tile a workgroup owns is found on the device from `starts`
// (find_tile): no host copy of the lengths, nothing to build ahead, so a call can be captured and replayed on other lengths.
#pragma once
#include "common.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

#define SEQ_LOG2E 1.4426950408889634f
#define SEQ_LN2 0.6931471805599453f

// ---- element types ------------------------------------------------------------------------------
// A fragment is 8 consecutive reduction indices of one operand row: lane l holds row l % 32, indices 8 (l / 32) .. + 7 of a
// 16-deep step.  bf16: one v_mfma_f32_32x32x16_bf16.  fp32: eight v_mfma_f32_32x32x2_f32, the i-th of which takes element i of
// both operands - index 8 (l / 32) + i on either side, so the same fragments serve, and the products are exact fp32.
template <typename T> struct SeqT;
template <> struct SeqT<__bf16> {
    typedef bf16x8 frag;
    static constexpr int KT = 64;            // keys (or query rows) of a staged tile
};
template <> struct SeqT<float> {
    typedef f32x8 frag;
    static constexpr int KT = 32;
};
__device__ __forceinline__ f32x16 seq_mma(const bf16x8& a, const bf16x8& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 seq_mma(const f32x8& a, const f32x8& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ int seq_rowmap(int r, int hh) { return (r & 3) + 8 * (r >> 2) + 4 * hh; }

// two accumulator halves (registers 8 t .. 8 t + 7) -> the B operand of reduction step t; for bf16 this is the ONE rounding of
// the probabilities / score gradients: they enter a product whose other operand is bf16 too, and are summed in fp32
__device__ __forceinline__ void seq_to_frag(const f32x16& p, int t, bf16x8& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (__bf16)p[8 * t + e];
}
__device__ __forceinline__ void seq_to_frag(const f32x16& p, int t, f32x8& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = p[8 * t + e];
}
// What that rounding took, as a second operand of the same product: together they are the fp32 value to 2^-16 (taken where
// seq_two_parts and, over a cache, pg_two_parts say).
__device__ __forceinline__ void seq_to_rest(const f32x16& p, int t, const bf16x8& f, bf16x8& g) {
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = (__bf16)(p[8 * t + e] - (float)f[e]);
}

// lanes l and l ^ 32 combined (both get the same bits); inline asm because the builtin's two results are folded into one
__device__ __forceinline__ float seq_half_max(float v) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\tv_max_f32 %0, %0, %1" : "+v"(a), "+v"(b));
    return a;
}
__device__ __forceinline__ float seq_half_sum(float v) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return a + b;
}

// inclusive prefix sum over the wave in eight vector instructions (row shifts, then the row totals carried up); lane 63 has the sum
__device__ __forceinline__ int seq_scan_add(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);              // row_shr:1, 2, 4, 8 within rows of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);              // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);              // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ int seq_wave_total(int v) { return __builtin_amdgcn_readlane(seq_scan_add(v), 63); }

// ---- which tile of which sequence ------------------------------------------------------------------
#define SEQ_NO_TILE 0x40000000
struct SeqTile {
    int seq, tile, ntile;         // seq < 0: this workgroup has none
    int s0, n;                    // first token and length of the sequence
};
// The sequences of 64 lanes in falling order of their lengths: with more workgroups than compute units the long ones start
// first and the short ones fill up behind them (a training step over 32 utterances of 202 .. 900 in any order, 4 heads of 64, 592
// tiles: 119 -> 102 us of kernels, 107 with out_rest; over 16 causal sequences of 20 .. 2000, 8 / 2 heads of 128: 358 -> 343, 16 heads of 64: 330 ->
// 307).  A lane's rank is the number of keys above its own - lengths, made distinct by the lane - and every lane sends its sequence
// to the lane of its rank.
__device__ __forceinline__ void seq_longest_first(int count, int& seq, int& s0, int& n) {
    const int lane = threadIdx.x & 63;
    const int key = lane < count ? (min(n, 0x1ffffff) << 6) | (63 - lane) : -1;
    int rank = lane < count ? 0 : lane;
    for (int j = 0; j < count; ++j) rank += lane < count && __builtin_amdgcn_readlane(key, j) > key ? 1 : 0;
    seq = __builtin_amdgcn_ds_permute(rank << 2, seq);
    s0 = __builtin_amdgcn_ds_permute(rank << 2, s0);
    n = __builtin_amdgcn_ds_permute(rank << 2, n);
}
// Tile `unit` of the sequences' tiles laid end to end; `tokens` rows of the packed tensors bound every length, so a `starts`
// that is not ascending or points outside gives wrong rows but no access out of range.  Every lane of the wave calls it; 64
// sequences are looked at at a time.
// `falling`: a tile's work grows with its place in the sequence (causal), and there is more than one round of workgroups: the tiles
// of 64 sequences in falling order of that place, all sequences mixed, so that the last ones to start are the smallest.  Level s is
// the tiles in place s - 1; N(s) = sum max(0, tiles - s + 1) of them lie at level s or above, and the level of a unit is found by
// halving.  (t.tile counts from the tile with the most work.)  Forward of 8 x 2048 tokens, 8 heads of 64: 70 -> 51 us; of 6000 + 1999 +
// 193, 16 / 2 heads of 128: 193 -> 175, the priority below among them.
__device__ __forceinline__ SeqTile find_tile(const int* starts, int B, int tokens, int G, int rows_per_tile, int unit, bool falling = false) {
    const int lane = threadIdx.x & 63;
    SeqTile t;
    t.seq = -1; t.tile = t.ntile = t.s0 = t.n = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        int b = b0 + lane, s0 = 0, n = 0;
        if (b < B) {
            s0 = min(max(starts[b], 0), tokens);
            n = min(max(starts[b + 1], s0), tokens) - s0;
        }
        if (B > 1 && gridDim.x > 256 && !falling) seq_longest_first(min(B - b0, 64), b, s0, n);
        const int tiles = (int)(((long)n * G + rows_per_tile - 1) / rows_per_tile);
        const int upto = seq_scan_add(tiles);
        if (falling && B > 1 && gridDim.x > 256 && unit < __builtin_amdgcn_readlane(upto, 63)) {
            int low = 1, high = __builtin_amdgcn_readlane(upto, 63) + 1, above = 0;             // N(low) > unit >= N(high) = above
            while (high - low > 1) {
                const int mid = low + (high - low) / 2, count = seq_wave_total(max(tiles - mid + 1, 0));
                if (count > unit) low = mid;
                else { high = mid; above = count; }
            }
            const uint64_t there = __ballot(tiles >= low);
            const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(there >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)there, 0));
            const uint64_t mine = __ballot(tiles >= low && before == unit - above);
            if (!mine) { t.tile = SEQ_NO_TILE; return t; }          // (`starts` that overlap: the count wrapped)
            const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(mine));
            t.seq = b0 + at;
            t.ntile = __builtin_amdgcn_readlane(tiles, at);
            t.tile = t.ntile - low;
            t.s0 = __builtin_amdgcn_readlane(s0, at);
            t.n = __builtin_amdgcn_readlane(n, at);
            return t;
        }
        const uint64_t hit = __ballot(upto > unit);
        if (hit) {
            const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
            t.seq = __builtin_amdgcn_readlane(b, at);
            t.ntile = __builtin_amdgcn_readlane(tiles, at);
            t.tile = unit - (__builtin_amdgcn_readlane(upto, at) - t.ntile);
            t.s0 = __builtin_amdgcn_readlane(s0, at);
            t.n = __builtin_amdgcn_readlane(n, at);
            if ((unsigned)t.tile >= (unsigned)t.ntile) { t.seq = -1; t.tile = SEQ_NO_TILE; }   // (`starts` that overlap: the count wrapped)
            return t;
        }
        unit -= __builtin_amdgcn_readlane(upto, 63);
    }
    t.tile = unit;                                                 // none: how many units past the last tile
    return t;
}
// Grid of tiles: at least the sum of the sequences' tiles, and at least one more unit for every tile of rows behind them.
static inline long seq_units(long tokens, int B, int G, int rows_per_tile) { return tokens * G / rows_per_tile + B + 1; }
// Zeros into the rows of no sequence - in front of the first and behind the last (tensors that the host mirror has just
// allocated): unit `past` of the grid past the last tile clears the past-th tile of them, for G heads from head0 on.
template <typename T>
__device__ __forceinline__ void seq_zero_rest(T* dst, long row, long head, const int* starts, int B, int tokens, int G, int rows_per_tile,
                                              int head0, int dh, int past) {
    const int front = min(max(starts[0], 0), tokens), end = min(max(starts[B], front), tokens), per = dh / 4;
    const long r0 = (long)past * rows_per_tile, rows = min((long)(front + tokens - end) * G - r0, (long)rows_per_tile);
    for (long i = threadIdx.x; i < rows * per; i += blockDim.x) {
        const long r = r0 + i / per, t = r / G;
        T* d = dst + (t < front ? t : end - front + t) * row + (head0 + r % G) * head + (i % per) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = (T)0.f;
    }
}

// ---- key splits: units of (sequence, row tile, key range) ---------------------------------------------
// With few row tiles the keys are split over workgroups.  One split length for the whole call, chosen on the device so that all
// splits together number about `slots` a key head: long sequences get many, short ones one, and no workgroup has more than
// one split's keys - the batch is even whatever its lengths.  Units of a sequence: the first split of all its tiles, then the second ...:
// workgroups that run together read the same range, through one L2.
struct SeqUnit {
    SeqTile t;
    int len;                      // cached length of the sequence, as `lens` has it
    int split, nsplit, per;       // key range [split per, (split + 1) per)
    long first;                   // unit number of the tile's first split; its next ones follow at steps of ntile
};
static inline __host__ __device__ long seq_split_units(long tokens, int B, int G, int R, long slots) { return tokens * G / R + B + 1 + slots; }
// Tiles: R rows of G a token.  Keys: lens, `most` of them at most, or `own` times the sequence's tokens where lens is null (the
// backward's splits of the rows that a key tile meets).  by_tile: `unit` counts tiles instead (the join).
__device__ __forceinline__ SeqUnit find_unit(const int* starts, const int* lens, int own, int most, int B, int tokens, int G, int R, int slots,
                                             int quantum, int least, int unit, bool by_tile) {
    const int lane = threadIdx.x & 63;
    float total = 0.f;
    int b = 0, s0 = 0, n = 0, len = 0, keys = 0, tiles = 0;
    auto look = [&](int b0) {
        b = b0 + lane;
        s0 = n = len = 0;
        if (b < B) {
            s0 = min(max(starts[b], 0), tokens);
            n = min(max(starts[b + 1], s0), tokens) - s0;
            len = lens ? max(lens[b], 0) : 0;
        }
        if (!lens) {
            if (B > 1) seq_longest_first(min(B - b0, 64), b, s0, n);
            len = n * own;
        }
        keys = min(len, most);
        tiles = (int)(((long)n * G + R - 1) / R);
    };
    for (int b0 = 0; b0 < B; b0 += 64) {
        look(b0);
        total += (float)tiles * (float)keys;
    }
    total = wave_sum_dpp(total) * (1.f + 0x1p-16f);                  // (never short of the true sum: the grid is sized by it)
    long per_l = max((long)(total / (float)slots) + 1, (long)least);
    per_l = min((per_l + quantum - 1) / quantum * quantum, 0x7fffff00l / quantum * quantum);
    int per = __builtin_amdgcn_readfirstlane((int)per_l);
    if (lens) {
        // Every sequence's last split is a partial one: lengthen the splits until the units really fit the slots (a few units more
        // would run alone in a second round), or the sequences' tiles alone are most of them.
        for (int it = 0; it < 8; ++it) {
            int units = 0, all = 0;
            for (int b0 = 0; b0 < B; b0 += 64) {
                if (B > 64) look(b0);
                units += tiles * max((int)(((long)keys + per - 1) / per), 1);
                all += tiles;
            }
            units = seq_wave_total(units);
            all = seq_wave_total(all);
            if (units <= max(slots, all + all / 2) || per >= 0x3fffff00) break;
            const int more = (int)min((long)per * (units - slots) / max(units, 1) / 2, 0x3fffff00l);
            per = __builtin_amdgcn_readfirstlane(per + max(more / quantum, 1) * quantum);
        }
    }
    SeqUnit u;
    u.t.seq = -1; u.t.tile = u.t.ntile = u.t.s0 = u.t.n = 0;
    u.len = u.split = 0; u.nsplit = 1; u.per = per; u.first = 0;
    long before = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        if (B > 64) look(b0);                                      // (the only 64 are still in registers)
        const int splits = max((int)(((long)keys + per - 1) / per), 1), units = tiles * splits, counted = by_tile ? tiles : units;
        const int upto = seq_scan_add(counted), all = by_tile ? seq_scan_add(units) : upto;
        const uint64_t hit = __ballot(upto > unit);
        if (hit) {
            const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
            const int rem = unit - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(counted, at));
            u.t.seq = __builtin_amdgcn_readlane(b, at);
            u.t.ntile = __builtin_amdgcn_readlane(tiles, at);
            u.t.s0 = __builtin_amdgcn_readlane(s0, at);
            u.t.n = __builtin_amdgcn_readlane(n, at);
            u.len = __builtin_amdgcn_readlane(len, at);
            u.nsplit = __builtin_amdgcn_readlane(splits, at);
            u.split = __builtin_amdgcn_readfirstlane(by_tile ? 0 : rem / u.t.ntile);
            u.t.tile = by_tile ? rem : rem - u.split * u.t.ntile;
            u.first = before + __builtin_amdgcn_readlane(all, at) - __builtin_amdgcn_readlane(units, at) + u.t.tile;
            if ((unsigned)u.t.tile >= (unsigned)u.t.ntile || u.split >= u.nsplit) { u.t.seq = -1; u.t.tile = SEQ_NO_TILE; }
            return u;
        }
        unit -= __builtin_amdgcn_readlane(upto, 63);
        before += __builtin_amdgcn_readlane(all, 63);
    }
    u.t.tile = unit;
    return u;
}

// ---- the paged cache ---------------------------------------------------------------------------------
// pages [n_pages][Hkv][2^shift][dh] of bf16, fp32 or e4m3 bytes; e4m3: exp [n_pages][Hkv][2^shift], the biased exponent of the
// row's power-of-two scale.  A page number outside [0, n_pages) reads as zeros and is never written.
struct SeqPages {
    const void* k; const void* v;
    const uint8_t* ke; const uint8_t* ve;
    const int* table; int table_width;
    int n_pages, shift, heads, dh;
    // element offset of row `key` of sequence b's head hk, -1 where there is no such page
    __device__ __forceinline__ long row(int b, int hk, int key) const {
        const int p = key >> shift;
        if (p >= table_width) return -1;
        const int page = table[(long)b * table_width + p];
        if ((unsigned)page >= (unsigned)n_pages) return -1;
        return (((long)page * heads + hk) << shift) + (key & ((1 << shift) - 1));
    }
};
// 2^(e - 127) of a stored exponent byte (0 and 255 are not written by the cache kernels)
__device__ __forceinline__ float seq_scale_of(uint32_t e) { return __builtin_bit_cast(float, e << 23); }

// ---- few tiles: the keys in parts --------------------------------------------------------------------
// With 128 rows a workgroup, 32 a wave, a small batch leaves most of the card idle and its time is one wave's walk over a whole
// sequence.  Then a workgroup takes 128 / KS rows and KS = 2 or 4 waves share a row block: each meets every KS-th run of KW keys, and
// their sums are joined through LDS at the end.  KW: keys of a wave's step; a stage of KS KW keys has to fit twice.
template <typename T, int DHP, int KS> struct SeqKeys {
    static constexpr int KW = KS == 4 || (KS == 2 && DHP > 128) ? 32 : SeqT<T>::KT;
};
// Parts where the workgroups - half a tile more than whole ones a sequence - are about one a compute unit, as far as LDS has room.
// A causal batch of long sequences is uneven enough for twice as many.  Forward and backward in us with the keys in 1 / 2 / 4:
//   8 heads of 64, bf16, causal: 1 x 512 tokens 50 / 44 / 41, 3 x 512 52 / 46 / 48, 1 x 2048 107 / 81 / 74, 20 x 102 38 / 41 / 51
//   16 / 4 heads of 128, bf16, causal: 1 x 512 79 / 71 / 67, 1 x 1024 110 / 94 / 104, 3 x 512 87 / 97 / 118, 1 x 2048 198 / 186 / 244, 10 x 102 57 / 72 / 90
//   4 heads of 128, bf16, full: 4 x 512 73 / 64 / 64, 8 x 512 77 / 73 / 93, 12 x 512 82 / 105 / 126, 3 x 2048 197 / 243 / 273
//   4 heads of 64, fp32, causal: 4 x 512 159 / 113 / 89, 6 x 512 185 / 137 / 139, 2 x 2048 576 / 387 / 320, 20 x 102 72 / 60 / 77, 40 x 102 92 / 92 / 118
static inline int seq_key_parts(long tokens, int B, int G, int Hkv, int dh, bool f32, int causal) {
    const long mean = tokens / (B > 0 ? B : 1);
    const bool uneven = causal && mean >= 1024;
    auto workgroups = [&](int parts) { return (tokens * G * parts / 128 + (B + 1) / 2) * Hkv; };
    if (dh <= (f32 ? 64 : 128) && mean >= 256 && workgroups(4) <= (uneven && dh <= 64 ? 528 : 320)) return 4;
    if (!(f32 && dh > 128) && workgroups(2) <= (uneven ? 528 : mean >= 256 ? 288 : 256)) return 2;
    return 1;
}

// Probabilities and score gradients of bf16 tensors as operands of two parts (seq_to_rest): batches of short sequences with few
// tiles.  Nothing averages the rounding of one part over a few keys - dq and dk of two keys were up to 2.1 times as far from the
// formula as their own rounding puts them, of 100 keys 1.5 times, and 1.0 with two parts - while the matrix pipes of a small launch
// have the time.  Forward and backward in us with one part / two: 61 tokens, 2 heads of 192, 38 / 37; 20 x 102, 8 heads of 64, 37 / 37;
// 10 x 102, 16 / 4 heads of 128, 56 / 57; longer ones pay more for less: 1 x 512, 8 heads of 64, 41 / 47, 1 x 2048, 16 / 4 of 128, 185 / 232.
static inline bool seq_two_parts(long tokens, int B, int parts, bool f32) { return !f32 && parts == 2 && tokens / (B > 0 ? B : 1) < 256; }

// ---- what a forward launch takes ----
// keys of a split, tile form: at least four tiles (200 new tokens over 2000 keys, 4 heads of 128: 24 us; 25 at 128, 28 at 512)
#define SEQ_TILE_LEAST 256
struct SeqFwdP {
    const void* q; long q_row, q_head;                    // element strides
    const void* k; long k_row, k_head;
    const void* v; long v_row, v_head;
    void* o; long o_row, o_head;
    float* lse;                                           // [Hkv][tokens G] natural log, or null
    void* rest;                                           // [tokens][H][dh]: what the rounding of o to bf16 left, or null
    const int* starts; const int* lens;                   // lens: paged only (tokens in the cache, the new ones among them)
    SeqPages pg;
    int B, tokens, Hkv, G, dh, causal, zero_rest;
    int most;                                             // positions that the table's pages hold (paged only)
    float c1;                                             // scale log2(e)
    // key splits (slots > 0): partial sums of unit u, key head hk at [(u Hkv + hk)][R rows][dh], their maximum and sum at [..][R][2]
    int slots; float* part_o; float* part_ml;
};


// ---- 16-byte chunks of an LDS tile image ----------------------------------------------------------
// A tile image is [rows][DHP] with the 16-byte chunks of a row permuted by an exclusive-or with swz(row), so that both ways of
// reading it touch all 64 banks once: a fragment read (one chunk of 16 consecutive rows at a time) needs swz to take 16 different
// bank places over 16 rows; a transposing read (4 chunks of 4 consecutive rows; of 8-bit elements 2 chunks of rows 0-3 and 8-11;
// of fp32 8 chunks of two rows 4 apart) needs the high bits of swz to differ between those rows.  With the plain row number in
// its place four rows of every transposing read met in the same 16 banks: 60 % of the LDS cycles of the bf16 kernels.
template <typename T, int DHP> struct SeqImg {
    static constexpr int CH = DHP * (int)sizeof(T) / 16;           // chunks per row
    static constexpr int ROWB = DHP * (int)sizeof(T);
    __device__ static __forceinline__ int swz(int row) {
        if constexpr (sizeof(T) == 4) return (row & 3) | ((row >> 1) & 4) | ((row << 1) & 8);            // row bits 0, 1, 3, 2
        else if constexpr (CH % 16 == 0) return ((row & 3) << 2) | ((row >> 2) & 3);                     // bits 2, 3, 0, 1
        else if constexpr (CH % 8 == 0) return ((row << 1) & 4) | ((row >> 2) & 2) | ((row >> 2) & 1);   // bits 2, 3, 1 (bit 0 is a half of the banks)
        else return ((row >> 2) & 2) | ((row >> 2) & 1);                                                 // bits 2, 3
    }
    __device__ static __forceinline__ int at(int row, int chunk) { return row * ROWB + ((chunk ^ swz(row)) << 4); }   // byte offset
};
typedef short seq_s16x4 __attribute__((ext_vector_type(4)));
typedef short seq_s16x8 __attribute__((ext_vector_type(8)));
// Fragment addresses.  The chunk number of a step is a constant, so a lane needs ONE base a tile - its row and first chunk,
// permuted - and flips the constant's low bits into it: (base ^ lo) + rest, the rest an instruction offset.  (Tables of the
// permuted addresses cost the dK / dV kernel its registers: reloading spilled ones waited for the tile in flight behind them.)
template <typename T, int DHP> struct SeqLane {
    using I = SeqImg<T, DHP>;
    using frag = typename SeqT<T>::frag;
    static constexpr int LOW = I::CH % 16 == 0 ? 15 : 7;
    typedef __attribute__((address_space(3))) const unsigned char* lds;
    // row operand: lane holds image row row0 + l31
    __device__ static __forceinline__ uint32_t rows(const unsigned char* img, int lane) {
        const int r = lane & 31, hh = lane >> 5;
        return (uint32_t)(size_t)(lds)img + r * I::ROWB + (((sizeof(T) == 2 ? hh : 2 * hh) ^ I::swz(r)) << 4);
    }
    __device__ static __forceinline__ frag row(uint32_t base, int row0, int step) {
        const int chunk = (sizeof(T) == 2 ? 2 : 4) * step, rest = row0 * I::ROWB + (chunk & ~LOW) * 16;
        const uint32_t a = base ^ ((chunk & LOW) << 4);
        if constexpr (sizeof(T) == 2) {
            return *(__attribute__((address_space(3))) const bf16x8*)(size_t)(a + rest);
        } else {
            typedef float f32x4 __attribute__((ext_vector_type(4)));
            const f32x4 x = *(__attribute__((address_space(3))) const f32x4*)(size_t)(a + rest);
            const f32x4 y = *(__attribute__((address_space(3))) const f32x4*)(size_t)((a ^ 16) + rest);
            f32x8 f = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            return f;
        }
    }
    // The transposed operand: lane holds column cb 32 + l31 of the image, reduction indices k0 + rowmap(8 t + e, hh), e < 8 - the
    // order in which accumulator registers become the other operand.  bf16: two transposing LDS reads (a 16-lane group fetches
    // [4 rows][16 columns] and lane c gets column c).  fp32: eight 4-byte reads, consecutive lanes on consecutive columns.
    __device__ static __forceinline__ uint32_t cols(const unsigned char* img, int lane) {
        const int hh = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            const int r = 4 * hh + ((lane & 15) >> 2);
            return (uint32_t)(size_t)(lds)img + r * I::ROWB + (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ I::swz(r)) << 4) + (lane & 1) * 8;
        } else {
            return (uint32_t)(size_t)(lds)img + 4 * hh * I::ROWB + ((((lane & 31) >> 2) ^ I::swz(4 * hh)) << 4) + (lane & 3) * 4;
        }
    }
    __device__ static __forceinline__ frag col(uint32_t base, int k0, int t, int cb) {
        if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) seq_s16x4* tr;
            const int chunk = 4 * cb, rest = (k0 + 16 * t) * I::ROWB + (chunk & ~LOW) * 16;
            const uint32_t a = base ^ ((chunk & LOW) << 4);
            const seq_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(size_t)(a + rest));
            const seq_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(size_t)((a ^ (I::swz(8) << 4)) + rest + 8 * I::ROWB));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            f32x8 f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = (e & 3) + 8 * (e >> 2), chunk = 8 * cb, rest = (k0 + 16 * t + r) * I::ROWB + (chunk & ~LOW) * 16;
                f[e] = *(__attribute__((address_space(3))) const float*)(size_t)((base ^ (((chunk & LOW) ^ I::swz(r)) << 4)) + rest);
            }
            return f;
        }
    }
};

// ---- LDS-DMA staging ---------------------------------------------------------------------------------
// global_load_lds_dwordx4: 64 lanes x 16 bytes to 1 KB of LDS behind a wave-uniform offset, no registers in between.  Inline asm
// because the compiler orders every LDS read behind a builtin DMA; the kernels wait themselves (vmcnt, then the barrier).
__device__ __forceinline__ void seq_dma16(const void* base, uint32_t off, unsigned lds) {          // uniform base + lane offset
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void seq_dma16(const void* src, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void seq_dma4(const void* src, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void seq_dma1(const void* src, unsigned lds) {                           // a byte a lane, stored as a dword
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ unsigned seq_lds(const void* p) { return (unsigned)(size_t)(__attribute__((address_space(3))) const void*)p; }
// the lane number, formed where it is used: what is derived from it does not stay in registers around a loop
__device__ __forceinline__ int seq_lane_here() {
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
    return l;
}
// a value used inside a rarely taken uniform branch: keeps it a branch (its selects would be done every time)
__device__ __forceinline__ int seq_rare(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
// this wave's loads have landed and its LDS reads are done, then everybody's
__device__ __forceinline__ void seq_dma_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// One wave's share of a tile image of ROWS rows: instructions wave, wave + 4, ... of 1 KB each; item i of lane l is image row
// row(i), and the 16-byte piece of the source row that belongs there (the swizzle is in the source address).  Pieces past
// dh repeat the row's first one: they meet zeros of the other operand, or end in columns that are not stored.
template <typename T, int DHP, int ROWS> struct SeqDma {
    using I = SeqImg<T, DHP>;
    static constexpr int NI = ROWS * I::CH / 256;                  // instructions a wave
    __device__ static __forceinline__ int row(int i, int wave, int lane) { return ((wave + 4 * i) * 64 + lane) / I::CH; }
    __device__ static __forceinline__ uint32_t piece(int i, int wave, int lane, int dh) {
        const int id = (wave + 4 * i) * 64 + lane, r = id / I::CH, c = ((id - r * I::CH) ^ I::swz(r)) * 16;
        return c < dh * (int)sizeof(T) ? c : 0;
    }
};

// a fragment straight from global memory: elements [c, c + 8) of a row, zeros past dh (dh is a multiple of 8)
template <typename T>
__device__ __forceinline__ typename SeqT<T>::frag seq_load8(const T* row, int c, bool ok) {
    typename SeqT<T>::frag f;
    if (ok) return *reinterpret_cast<const typename SeqT<T>::frag*>(row + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (T)0.f;
    return f;
}
// 16 bytes of tile row data in T from 16 / sizeof(T) e4m3 bytes: exact, the scale is a power of two
template <typename T>
__device__ __forceinline__ uint4 seq_dequant_chunk(uint2 w, float scale) {
    if constexpr (sizeof(T) == 2) {
        bf16x8 o;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t v = i ? w.y : w.x;
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
            o[4 * i] = (__bf16)(a[0] * scale); o[4 * i + 1] = (__bf16)(a[1] * scale);
            o[4 * i + 2] = (__bf16)(b[0] * scale); o[4 * i + 3] = (__bf16)(b[1] * scale);
        }
        return __builtin_bit_cast(uint4, o);
    } else {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, true);
        const float4 o = make_float4(a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale);
        return __builtin_bit_cast(uint4, o);
    }
}

// ---- argument checks of the entry points -----------------------------------------------------------
// What every tensor of [tokens, heads, dh] has to be: 16-byte aligned rows and heads, so that 16-byte accesses are whole; and
// where a kernel stages tiles of it, a tile (128 tokens and a partial one, `group` heads) within 32-bit offsets of its first row.
static inline bool seq_strides_ok(const void* ptr, int64_t row, int64_t head, int group, int dtype) {
    const int n = dtype == TTSMI_F32 ? 4 : 8;
    return ptr != nullptr && ((uintptr_t)ptr & 15) == 0 && row % n == 0 && head % n == 0 && row >= 0 && head >= 0 &&
           (group == 0 || (row < (1l << 25) && head < (1l << 32) && (130 * row + group * head) * (16 / n) < (1l << 32)));
}
#define SEQ_CHECK_COMMON(who)                                                                                               \
    TTSMI_CHECK_ARG(dtype == TTSMI_F32 || dtype == TTSMI_BF16_IO, who ": dtype %d (TTSMI_F32 or TTSMI_BF16_IO)", dtype);          \
    TTSMI_CHECK_ARG(B >= 0 && tokens >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0, who ": sequences %d, tokens %d, heads %d / %d", B, tokens, H, Hkv); \
    TTSMI_CHECK_ARG(dh > 0 && dh <= 192 && dh % 8 == 0, who ": head size %d (a multiple of 8 up to 192)", dh);             \
    TTSMI_CHECK_ARG(scale > 0.f && scale < INFINITY, who ": scale must be positive and finite");                          \
    TTSMI_CHECK_ARG((long)tokens * H + 512L * B * Hkv < (1L << 30), who ": tokens * heads too large");
#define SEQ_CHECK_PAGES(who)                                                                                                      \
    TTSMI_CHECK_ARG(n_pages >= 0 && page_size > 0 && page_size <= 1024 && (page_size & (page_size - 1)) == 0 && table_width >= 0 &&  \
                        (long)n_pages * Hkv < (1L << 31), who ": %d pages of %d rows (a power of two up to 1024)", n_pages, page_size)
#define SEQ_CHECK_CACHE(who)                                                                                                      \
    do {                                                                                                                          \
        TTSMI_CHECK_ARG(starts && (B == 0 || (lens && (table || table_width == 0))), who ": null starts, lens or table");         \
        TTSMI_CHECK_ARG(n_pages == 0 || (k_pages && v_pages && (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0),             \
                        who ": pages null or not 16-byte aligned");                                                               \
        TTSMI_CHECK_ARG(cache_dtype != TTSMI_E4M3 || n_pages == 0 || (k_exp && v_exp), who ": an e4m3 cache needs its exponents");  \
    } while (0)

int seq_paged_tiles(const SeqFwdP& p, int dtype, int cache_dtype, hipStream_t st);
