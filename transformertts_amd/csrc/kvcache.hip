// The paged key / value cache: writing the keys and values of new tokens into their pages - as they are, or quantised to e4m3 -
// and reading sequences back in packed order.
//
// e4m3 rows.  Each row (token, key head) of K and of V has a power-of-two scale 2^(e - 127), the smallest that brings the row's
// largest finite magnitude to 448 at most, so that scaling is exact both ways and a value is off by the one rounding to e4m3
// (half a step: 2^-4 relative; below 2^-6 of the row's scale, 2^-10 of it absolute).  A row of zeros has scale 1.  NaN and
// infinity are stored as NaN: e4m3 has no infinity.
//
// Bound by memory: a wave owns a token, finds its sequence among `starts` (64 at a time) and moves the rows of all key heads, K
// and V, 8 elements a lane.  Measured: 12620 tokens of 8 heads of 128, bf16 into e4m3 pages 16.7 us and back 14.5 us, 155 MB in
// all or 5.0 TB/s, the rate of a copy; into bf16 pages and back, a replayed call each, 22 and 22 us (104 MB), fp32 38 and 37 (207 MB); 64
// single tokens into bf16 pages: 3.5 us, a launch.
#include "seq_common.h"

struct KvP {
    const void* k; long k_row, k_head;                    // [tokens, heads, dh]: the source of a write, the destination of a read
    const void* v; long v_row, v_head;
    SeqPages pg;
    const int* starts; const int* lens;
    int B, tokens, zero_rest;
};

// sequence and position of packed token `tok`: the tokens of sequence b are its last starts[b + 1] - starts[b] ones.  -1: none.
__device__ __forceinline__ int kv_find(const KvP& p, int tok, int lane, int& pos) {
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int b = b0 + lane, end = b < p.B ? p.starts[b + 1] : 0x7fffffff;
        const uint64_t hit = __ballot(b < p.B && end > tok);
        if (hit) {
            const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
            const int seq = b0 + at;
            if (p.starts[seq] > tok) return -1;
            pos = p.lens[seq] - (__builtin_amdgcn_readlane(end, at) - tok);
            return pos < 0 ? -1 : seq;
        }
    }
    return -1;
}

// LPR lanes of 8 elements move a row (dh <= 8 LPR)
template <typename T, typename CT, int LPR>
__global__ __launch_bounds__(256) void kv_write_kernel(KvP p) {
    const int lane = threadIdx.x & 63, tok = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tok >= p.tokens) return;
    int pos = 0;
    const int seq = kv_find(p, tok, lane, pos);
    if (seq < 0) return;
    const long at0 = p.pg.row(seq, 0, pos);
    if (at0 < 0) return;
    const int c = (lane % LPR) * 8;
    const bool in = c < p.pg.dh;
    for (int r = lane / LPR; r < 2 * p.pg.heads; r += 64 / LPR) {
        const int h = r >> 1;
        const bool is_v = r & 1;
        const long at = at0 + ((long)h << p.pg.shift);
        typedef typename SeqT<T>::frag frag;
        const T* src = is_v ? (const T*)p.v + (long)tok * p.v_row + (long)h * p.v_head : (const T*)p.k + (long)tok * p.k_row + (long)h * p.k_head;
        const frag f = seq_load8<T>(src, c, in);
        if constexpr (sizeof(CT) != 1) {
            if (in) *reinterpret_cast<frag*>((T*)(is_v ? p.pg.v : p.pg.k) + at * p.pg.dh + c) = f;
        } else {
            uint32_t top = 0;                              // magnitudes compare as their bits
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t a = __builtin_bit_cast(uint32_t, (float)f[e]) & 0x7fffffffu;
                top = max(top, a < 0x7f800000u ? a : 0u);
            }
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
            // top = 1.m 2^x <= 1.75 2^8 2^e: e = x - 8, one more where the fraction is above 1.75; biased, at least 1 (2^-126)
            int ex = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
            ex = top == 0 ? 127 : max(ex, 1);
            const float inv = __builtin_bit_cast(float, (uint32_t)(254 - ex) << 23);
            uint32_t w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = (float)f[4 * i + e] * inv;
                    if (!(__builtin_fabsf(x[e]) <= 448.f)) x[e] = __builtin_nanf("");
                }
                int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
                w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], v, true);
            }
            if (in) *reinterpret_cast<uint2*>((uint8_t*)(is_v ? p.pg.v : p.pg.k) + at * p.pg.dh + c) = make_uint2(w[0], w[1]);
            if (c == 0) const_cast<uint8_t*>(is_v ? p.pg.ve : p.pg.ke)[at] = (uint8_t)ex;
        }
    }
}

// T: the destination's type
template <typename T, typename CT, int LPR>
__global__ __launch_bounds__(256) void kv_read_kernel(KvP p) {
    const int lane = threadIdx.x & 63, tok = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tok >= p.tokens) return;
    int pos = 0;
    const int seq = kv_find(p, tok, lane, pos);
    // (a token that is in a sequence but before its first position - more rows asked for than are cached - reads zeros)
    if (seq < 0 && !p.zero_rest && (tok < p.starts[0] || tok >= p.starts[p.B])) return;
    const long at0 = seq < 0 ? -1 : p.pg.row(seq, 0, pos);
    const int c = (lane % LPR) * 8;
    if (c >= p.pg.dh) return;
    for (int r = lane / LPR; r < 2 * p.pg.heads; r += 64 / LPR) {
        const int h = r >> 1;
        const bool is_v = r & 1;
        const long at = at0 + ((long)h << p.pg.shift);
        typedef typename SeqT<T>::frag frag;
        frag f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (T)0.f;
        if (at0 >= 0) {
            if constexpr (sizeof(CT) == 1) {
                const uint2 w = *reinterpret_cast<const uint2*>((const uint8_t*)(is_v ? p.pg.v : p.pg.k) + at * p.pg.dh + c);
                const float s = seq_scale_of((is_v ? p.pg.ve : p.pg.ke)[at]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t v = i ? w.y : w.x;
                    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
                    f[4 * i] = (T)(a[0] * s); f[4 * i + 1] = (T)(a[1] * s);
                    f[4 * i + 2] = (T)(b[0] * s); f[4 * i + 3] = (T)(b[1] * s);
                }
            } else {
                typedef typename SeqT<CT>::frag cfrag;
                const cfrag w = *reinterpret_cast<const cfrag*>((const CT*)(is_v ? p.pg.v : p.pg.k) + at * p.pg.dh + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = (T)(float)w[e];
            }
        }
        T* dst = is_v ? (T*)p.v + (long)tok * p.v_row + (long)h * p.v_head : (T*)p.k + (long)tok * p.k_row + (long)h * p.k_head;
        *reinterpret_cast<frag*>(dst + c) = f;
    }
}

template <typename T, typename CT>
static int kv_launch(const KvP& p, bool write, hipStream_t st) {
    const dim3 g((unsigned)((p.tokens + 3) / 4));
#define KV_GO(LPR)                                                                                     \
    do {                                                                                               \
        if (write) hipLaunchKernelGGL((kv_write_kernel<T, CT, LPR>), g, dim3(256), 0, st, p);          \
        else hipLaunchKernelGGL((kv_read_kernel<T, CT, LPR>), g, dim3(256), 0, st, p);                 \
    } while (0)
    if (p.pg.dh <= 64) KV_GO(8);
    else if (p.pg.dh <= 128) KV_GO(16);
    else KV_GO(32);
#undef KV_GO
    TTSMI_CHECK_LAUNCH("kv_cache");
    return TTSMI_OK;
}

#define KV_CHECK(who)                                                                                                             \
    TTSMI_CHECK_ARG(dtype == TTSMI_F32 || dtype == TTSMI_BF16_IO, who ": dtype %d (TTSMI_F32 or TTSMI_BF16_IO)", dtype);                \
    TTSMI_CHECK_ARG(B >= 0 && tokens >= 0 && Hkv > 0, who ": sequences %d, tokens %d, key heads %d", B, tokens, Hkv);              \
    TTSMI_CHECK_ARG(dh > 0 && dh <= 192 && dh % 8 == 0, who ": head size %d (a multiple of 8 up to 192)", dh);                     \
    SEQ_CHECK_PAGES(who);                                                                                                         \
    if (tokens == 0) return TTSMI_OK;                                                                                             \
    SEQ_CHECK_CACHE(who);                                                                                                         \
    TTSMI_CHECK_ARG(seq_strides_ok(k, k_row, k_head, 0, dtype) && seq_strides_ok(v, v_row, v_head, 0, dtype),                         \
                    who ": a tensor is null or its rows or heads are not 16-byte aligned");                                      \
    KvP p = {};                                                                                                                   \
    p.k = k; p.k_row = k_row; p.k_head = k_head; p.v = v; p.v_row = v_row; p.v_head = v_head;                                      \
    p.pg.k = k_pages; p.pg.v = v_pages; p.pg.ke = k_exp; p.pg.ve = v_exp; p.pg.table = table; p.pg.table_width = table_width;      \
    p.pg.n_pages = n_pages; p.pg.shift = __builtin_ctz(page_size); p.pg.heads = Hkv; p.pg.dh = dh;                                 \
    p.starts = starts; p.lens = lens; p.B = B; p.tokens = tokens;

extern "C" int ttsmi_kv_cache_write(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                                    void* k_pages, void* v_pages, uint8_t* k_exp, uint8_t* v_exp, int cache_dtype, int n_pages,
                                    int page_size, const int32_t* table, int table_width, const int32_t* starts, const int32_t* lens,
                                    int B, int tokens, int Hkv, int dh, int dtype, ttsmi_stream_t stream) {
    TTSMI_CHECK_ARG(cache_dtype == dtype || cache_dtype == TTSMI_E4M3, "kv_cache_write: cache dtype %d with tensors of dtype %d", cache_dtype, dtype);
    KV_CHECK("kv_cache_write");
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TTSMI_F32) return cache_dtype == TTSMI_E4M3 ? kv_launch<float, uint8_t>(p, true, st) : kv_launch<float, float>(p, true, st);
    return cache_dtype == TTSMI_E4M3 ? kv_launch<__bf16, uint8_t>(p, true, st) : kv_launch<__bf16, __bf16>(p, true, st);
}
extern "C" int ttsmi_kv_cache_read(const void* k_pages, const void* v_pages, const uint8_t* k_exp, const uint8_t* v_exp, int cache_dtype,
                                   int n_pages, int page_size, const int32_t* table, int table_width, const int32_t* starts,
                                   const int32_t* lens, int B, int tokens, int Hkv, int dh, void* k, int64_t k_row, int64_t k_head,
                                   void* v, int64_t v_row, int64_t v_head, int zero_rest, int dtype, ttsmi_stream_t stream) {
    TTSMI_CHECK_ARG(cache_dtype == dtype || cache_dtype == TTSMI_E4M3, "kv_cache_read: cache dtype %d with tensors of dtype %d", cache_dtype, dtype);
    KV_CHECK("kv_cache_read");
    p.zero_rest = zero_rest != 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TTSMI_F32) return cache_dtype == TTSMI_E4M3 ? kv_launch<float, uint8_t>(p, false, st) : kv_launch<float, float>(p, false, st);
    return cache_dtype == TTSMI_E4M3 ? kv_launch<__bf16, uint8_t>(p, false, st) : kv_launch<__bf16, __bf16>(p, false, st);
}
