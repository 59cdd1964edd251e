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
