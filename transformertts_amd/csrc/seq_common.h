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

// ---- which tile of which sequence ------------------------------------------------------------------
struct SeqTile {
    int seq, tile, ntile;         // seq < 0: this workgroup has none
    int s0, n;                    // first token and length of the sequence
};
// Tile `unit` of the sequences' tiles laid end to end; `tokens` rows of the packed tensors bound every length, so a `starts`
// that is not ascending or points outside gives wrong rows but no access out of range.  Every lane of the wave calls it; 64
// sequences are looked at at a time.
__device__ __forceinline__ SeqTile find_tile(const int* starts, int B, int tokens, int G, int rows_per_tile, int unit) {
    const int lane = threadIdx.x & 63;
    SeqTile t;
    t.seq = -1; t.tile = t.ntile = t.s0 = t.n = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + lane;
        int s0 = 0, n = 0;
        if (b < B) {
            s0 = min(max(starts[b], 0), tokens);
            n = min(max(starts[b + 1], s0), tokens) - s0;
        }
        const int tiles = (int)(((long)n * G + rows_per_tile - 1) / rows_per_tile);
        int upto = tiles;                                          // inclusive prefix sum over the wave
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o, 64);
            if (lane >= o) upto += v;
        }
        const uint64_t hit = __ballot(upto > unit);
        if (hit) {
            const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
            t.seq = b0 + at;
            t.ntile = __builtin_amdgcn_readlane(tiles, at);
            t.tile = unit - (__builtin_amdgcn_readlane(upto, at) - t.ntile);
            t.s0 = __builtin_amdgcn_readlane(s0, at);
            t.n = __builtin_amdgcn_readlane(n, at);
            return t;
        }
        unit -= __builtin_amdgcn_readlane(upto, 63);
    }
    t.tile = unit;                                                 // none: how many units past the last tile
    return t;
}
// Grid of tiles: at least the sum of the sequences' tiles, and at least one more unit for every tile of rows behind them.
static inline long seq_units(long tokens, int B, int G, int rows_per_tile) { return tokens * G / rows_per_tile + B + 1; }
// Zeros into the rows behind the last sequence (tensors that the host mirror has just allocated): unit `past` of the grid past
// the last tile clears the past-th tile of them, for G heads from head0 on.
template <typename T>
__device__ __forceinline__ void seq_zero_rest(T* dst, long row, long head, const int* starts, int B, int tokens, int G, int rows_per_tile,
                                              int head0, int dh, int past) {
    const int end = min(max(starts[B], 0), tokens), per = dh / 4;
    const long r0 = (long)past * rows_per_tile, rows = min((long)(tokens - end) * G - r0, (long)rows_per_tile);
    for (long i = threadIdx.x; i < rows * per; i += blockDim.x) {
        const long r = r0 + i / per;
        T* d = dst + (end + r / G) * row + (head0 + r % G) * head + (i % per) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = (T)0.f;
    }
}

// ---- key splits: units of (sequence, row tile, key range) ---------------------------------------------
// With few row tiles the keys are split over workgroups.  One split length for the whole call, chosen on the device so that all
// splits together number about `slots` a key head: long sequences get many, short ones one, and no workgroup has more than
// one split's keys - the batch is even whatever its lengths.  Units of a sequence: its row tiles, each with its splits in turn.
struct SeqUnit {
    SeqTile t;
    int len;                      // keys of the sequence
    int split, nsplit, per;       // key range [split per, (split + 1) per)
    long first;                   // unit number of the tile's first split
};
static inline __host__ __device__ long seq_split_units(long tokens, int B, int G, int R, int slots) { return tokens * G / R + B + 1 + slots; }
// Tiles: R rows of G a token.  Keys: lens, or `own` times the sequence's tokens where lens is null (the backward's splits of the
// rows that a key tile meets).  by_tile: `unit` counts tiles instead (the join).
__device__ __forceinline__ SeqUnit find_unit(const int* starts, const int* lens, int own, int B, int tokens, int G, int R, int slots,
                                             int quantum, int least, int unit, bool by_tile) {
    const int lane = threadIdx.x & 63;
    long total = 0;
    int s0 = 0, n = 0, len = 0, tiles = 0;
    auto look = [&](int b) {
        s0 = n = len = 0;
        if (b < B) {
            s0 = min(max(starts[b], 0), tokens);
            n = min(max(starts[b + 1], s0), tokens) - s0;
            len = lens ? max(lens[b], 0) : n * own;
        }
        tiles = (int)(((long)n * G + R - 1) / R);
    };
    for (int b0 = 0; b0 < B; b0 += 64) {
        look(b0 + lane);
        total += (long)tiles * len;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
    const long even = (total + slots - 1) / slots;
    const int per = (int)min((max(even, (long)least) + quantum - 1) / quantum * quantum, (long)0x7fffff00);
    SeqUnit u;
    u.t.seq = -1; u.t.tile = u.t.ntile = u.t.s0 = u.t.n = 0;
    u.len = u.split = 0; u.nsplit = 1; u.per = per; u.first = 0;
    long before = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        if (B > 64) look(b0 + lane);                               // (the only 64 are still in registers)
        const int splits = max((len + per - 1) / per, 1), units = tiles * splits, counted = by_tile ? tiles : units;
        int upto = counted, all = units;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o, 64), w = __shfl_up(all, o, 64);
            if (lane >= o) { upto += v; all += w; }
        }
        const uint64_t hit = __ballot(upto > unit);
        if (hit) {
            const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
            const int rem = unit - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(counted, at));
            u.t.seq = b0 + at;
            u.t.ntile = __builtin_amdgcn_readlane(tiles, at);
            u.t.s0 = __builtin_amdgcn_readlane(s0, at);
            u.t.n = __builtin_amdgcn_readlane(n, at);
            u.len = __builtin_amdgcn_readlane(len, at);
            u.nsplit = __builtin_amdgcn_readlane(splits, at);
            u.t.tile = by_tile ? rem : rem / u.nsplit;
            u.split = by_tile ? 0 : rem - u.t.tile * u.nsplit;
            u.first = before + __builtin_amdgcn_readlane(all, at) - __builtin_amdgcn_readlane(units, at) + (long)u.t.tile * u.nsplit;
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

// ---- what a forward launch takes ----
#define SEQ_TILE_LEAST 256           // keys of a split, tile form: at least four tiles
struct SeqFwdP {
    const void* q; long q_row, q_head;                    // element strides
    const void* k; long k_row, k_head;
    const void* v; long v_row, v_head;
    void* o; long o_row, o_head;
    float* lse;                                           // [Hkv][tokens G] natural log, or null
    const int* starts; const int* lens;                   // lens: paged only (tokens in the cache, the new ones among them)
    SeqPages pg;
    int B, tokens, Hkv, G, dh, causal, zero_rest;
    float c1;                                             // scale log2(e)
    // key splits (slots > 0): partial sums of unit u, key head hk at [(u Hkv + hk)][R rows][dh], their maximum and sum at [..][R][2]
    int slots; float* part_o; float* part_ml;
};


// ---- 16-byte chunks of an LDS tile image ----------------------------------------------------------
// A tile image is [rows][DHP] with the 16-byte chunks of a row permuted by the row number, so that the 32 rows of a fragment
// read (same chunk, consecutive rows) and the 4 rows of a transposing read fall into different banks without padding.
template <typename T, int DHP> struct SeqImg {
    static constexpr int CH = DHP * (int)sizeof(T) / 16;           // chunks per row
    static constexpr int ROWB = DHP * (int)sizeof(T);
    static constexpr int MASK = CH % 16 == 0 ? 15 : 7;
    __device__ static __forceinline__ int at(int row, int chunk) { return row * ROWB + ((chunk ^ (row & MASK)) << 4); }   // byte offset
};
template <typename T, int DHP>
__device__ __forceinline__ typename SeqT<T>::frag seq_frag(const unsigned char* img, int row, int step, int hh) {
    using I = SeqImg<T, DHP>;
    if constexpr (sizeof(T) == 2) {
        return *reinterpret_cast<const bf16x8*>(img + I::at(row, 2 * step + hh));
    } else {
        const float4 a = *reinterpret_cast<const float4*>(img + I::at(row, 4 * step + 2 * hh));
        const float4 b = *reinterpret_cast<const float4*>(img + I::at(row, 4 * step + 2 * hh + 1));
        f32x8 f = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        return f;
    }
}
// The transposed operand: lane holds column cb 32 + l31 of the image, reduction indices k0 + rowmap(8 t + e, hh), e < 8 - the
// order in which accumulator registers become the other operand.  bf16: two transposing LDS reads (a 16-lane group fetches
// [4 rows][16 columns] and lane c gets column c).  fp32: eight 4-byte reads, consecutive lanes on consecutive columns.
typedef short seq_s16x4 __attribute__((ext_vector_type(4)));
typedef short seq_s16x8 __attribute__((ext_vector_type(8)));
template <typename T, int DHP>
__device__ __forceinline__ typename SeqT<T>::frag seq_frag_t(const unsigned char* img, int k0, int t, int cb, int lane) {
    using I = SeqImg<T, DHP>;
    if constexpr (sizeof(T) == 2) {
        typedef __attribute__((address_space(3))) seq_s16x4* lds_ptr;
        const int row = k0 + 16 * t + 4 * (lane >> 5) + ((lane & 15) >> 2);
        const int chunk = cb * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), sub = (lane & 1) * 8;
        const seq_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(img + I::at(row, chunk) + sub));
        const seq_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(img + I::at(row + 8, chunk) + sub));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
        const int c = cb * 32 + (lane & 31), hh = lane >> 5;
        f32x8 f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = *reinterpret_cast<const float*>(img + I::at(k0 + seq_rowmap(8 * t + e, hh), c >> 2) + (c & 3) * 4);
        return f;
    }
}
// a fragment straight from global memory: elements [c, c + 8) of a row, zeros past dh (dh is a multiple of 8)
template <typename T>
__device__ __forceinline__ typename SeqT<T>::frag seq_load8(const T* row, int c, bool ok) {
    typename SeqT<T>::frag f;
    if (ok) return *reinterpret_cast<const typename SeqT<T>::frag*>(row + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (T)0.f;
    return f;
}
// 16 bytes of tile row data in T from a cache of e4m3 bytes (16 / sizeof(T) elements): exact, the scale is a power of two
template <typename T>
__device__ __forceinline__ uint4 seq_dequant_chunk(const uint8_t* src, float scale) {
    if constexpr (sizeof(T) == 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(src);
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
        const uint32_t v = *reinterpret_cast<const uint32_t*>(src);
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
        const float4 o = make_float4(a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale);
        return __builtin_bit_cast(uint4, o);
    }
}

// ---- argument checks of the entry points -----------------------------------------------------------
// What every tensor of [tokens, heads, dh] has to be: 16-byte aligned rows and heads, so that 16-byte accesses are whole.
static inline bool seq_strides_ok(const void* ptr, int64_t row, int64_t head, int dtype) {
    const int n = dtype == TTSMI_F32 ? 4 : 8;
    return ptr != nullptr && ((uintptr_t)ptr & 15) == 0 && row % n == 0 && head % n == 0 && row >= 0 && head >= 0;
}
#define SEQ_CHECK_COMMON(who)                                                                                               \
    TTSMI_CHECK_ARG(dtype == TTSMI_F32 || dtype == TTSMI_BF16_IO, who ": dtype %d (TTSMI_F32 or TTSMI_BF16_IO)", dtype);          \
    TTSMI_CHECK_ARG(B >= 0 && tokens >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0, who ": sequences %d, tokens %d, heads %d / %d", B, tokens, H, Hkv); \
    TTSMI_CHECK_ARG(dh > 0 && dh <= 192 && dh % 8 == 0, who ": head size %d (a multiple of 8 up to 192)", dh);             \
    TTSMI_CHECK_ARG(scale > 0.f && scale < INFINITY, who ": scale must be positive and finite");                          \
    TTSMI_CHECK_ARG((long)tokens * H + 128L * B * Hkv < (1L << 31), who ": tokens * heads too large");
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
