// Rotary positions: pair i of a head at position t is turned by the angle t w_i,
//     (a, b) -> (a c - b s, b c + a s),   c = scale cos(t w_i),  s = scale sin(t w_i);   the gradient turns back (s -> -s).
// Pairs are (2 i, 2 i + 1) (interleaved) or (i, i + rot / 2) (half) of the first `rot` elements; the rest passes through.
//
// Bound by memory: every element is read once and written once.  A wave owns a token: its lanes first form the rot / 2 angles
// (64-bit product and reduction to a turn, so positions of any size keep their angle, then sin / cos of the fraction in 32 bits),
// which pass through LDS, and then go over the token's query and key heads, 2 x 16 bytes a lane and step.  The run of a lane is
// the widest that every tensor's alignment and the head's division allow.  Measured: 16384 tokens of 32 / 8 heads of 128, bf16:
// 65 us, 5.1 TB/s, the rate of a copy on this card; 16 tokens of 4 / 4 heads of 64: 3.7 us, a launch.
#include "common.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct RotT {                       // one tensor [tokens, heads, dh]
    const void* x; long x_row, x_head;
    void* y; long y_row, y_head;
    int heads;
};
struct RotP {
    RotT t[2];
    const int* pos; const double* freq;
    int tokens, dh, rot;
    float scale, sign;
};
template <typename T, int N> struct RotVec { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct RotVec<T, 1> { typedef T type; };

// PV pairs per unit; a head has rot / (2 PV) turned units and (dh - rot) / (2 PV) copied ones.  ROT_MAX pairs at most.
#define ROT_MAX 256
template <typename T, int PV, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotP p) {
    __shared__ float2 cs[4][ROT_MAX];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long tok = (long)blockIdx.x * 4 + wave;
    const bool ok = tok < p.tokens;
    if (ok) {
        const double t = (double)p.pos[tok];
        for (int i = lane; i < p.rot / 2; i += 64) {
            double turn = t * p.freq[i] * 0.15915494309189535;             // 1 / (2 pi)
            turn -= rint(turn);
            float s, c;
            sincospif(2.f * (float)turn, &s, &c);
            cs[wave][i] = make_float2(c * p.scale, s * p.scale * p.sign);
        }
    }
    __syncthreads();
    if (!ok) return;
    typedef typename RotVec<T, PV>::type run;
    const int turned = p.rot / (2 * PV), per = p.dh / (2 * PV);
    const int step_h = 64 / per, step_u = 64 % per;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const RotT& r = p.t[which];
        const T* x = (const T*)r.x + tok * r.x_row;
        T* y = (T*)r.y + tok * r.y_row;
        int h = lane / per, u = lane - h * per;
        while (h < r.heads) {
            // up to four units in flight per lane
            run a[4], b[4];
            int hs[4], us[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                hs[j] = h; us[j] = u;
                if (h < r.heads) {
                    const int base = u < turned ? (INTER ? 2 * PV * u : PV * u) : p.rot + 2 * PV * (u - turned);
                    const int gap = !INTER && u < turned ? p.rot / 2 : PV;
                    const T* src = x + (long)h * r.x_head + base;
                    a[j] = *reinterpret_cast<const run*>(src);
                    b[j] = *reinterpret_cast<const run*>(src + gap);
                }
                u += step_u; h += step_h;
                if (u >= per) { u -= per; ++h; }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (hs[j] >= r.heads) continue;
                const int v = us[j];
                T ea[2 * PV], out[2 * PV];
                *reinterpret_cast<run*>(ea) = a[j];
                *reinterpret_cast<run*>(ea + PV) = b[j];
                if (v < turned) {
#pragma unroll
                    for (int i = 0; i < PV; ++i) {
                        const float2 w = cs[wave][PV * v + i];
                        const int ia = INTER ? 2 * i : i, ib = INTER ? 2 * i + 1 : PV + i;
                        const float fa = (float)ea[ia], fb = (float)ea[ib];
                        out[ia] = (T)(fa * w.x - fb * w.y);
                        out[ib] = (T)(fb * w.x + fa * w.y);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2 * PV; ++i) out[i] = ea[i];
                }
                const int base = v < turned ? (INTER ? 2 * PV * v : PV * v) : p.rot + 2 * PV * (v - turned);
                const int gap = !INTER && v < turned ? p.rot / 2 : PV;
                T* dst = y + (long)hs[j] * r.y_head + base;
                *reinterpret_cast<run*>(dst) = *reinterpret_cast<run*>(out);
                *reinterpret_cast<run*>(dst + gap) = *reinterpret_cast<run*>(out + PV);
            }
        }
    }
}

template <typename T, int PV>
static void rotary_launch(const RotP& p, int inter, hipStream_t st) {
    const dim3 g((unsigned)((p.tokens + 3) / 4));
    if (inter) hipLaunchKernelGGL((rotary_kernel<T, PV, true>), g, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((rotary_kernel<T, PV, false>), g, dim3(256), 0, st, p);
}
// widest run whose accesses are aligned for every tensor and that divides the turned half and the rest of a head
static int rotary_run(const RotP& p, int widest, int size) {
    for (int pv = widest; pv > 1; pv = pv > 2 ? 2 : 1) {
        bool ok = (p.rot / 2) % pv == 0 && (p.dh - p.rot) % (2 * pv) == 0;
        for (const RotT& t : p.t) {
            if (!t.heads) continue;
            ok = ok && (((uintptr_t)t.x | (uintptr_t)t.y) % (size_t)(pv * size)) == 0 && t.x_row % pv == 0 && t.x_head % pv == 0 && t.y_row % pv == 0 && t.y_head % pv == 0;
        }
        if (ok) return pv;
    }
    return 1;
}

extern "C" int ttsmi_rotary(const void* q, int64_t q_row, int64_t q_head, void* qo, int64_t qo_row, int64_t qo_head, int H, const void* k,
                            int64_t k_row, int64_t k_head, void* ko, int64_t ko_row, int64_t ko_head, int Hkv, const int32_t* positions,
                            const double* freqs, int tokens, int dh, int rot, int interleaved, float scale, int inverse, int dtype,
                            ttsmi_stream_t stream) {
    TTSMI_CHECK_ARG(dtype == TTSMI_F32 || dtype == TTSMI_BF16_IO, "rotary: dtype %d (TTSMI_F32 or TTSMI_BF16_IO)", dtype);
    TTSMI_CHECK_ARG(tokens >= 0 && H >= 0 && Hkv >= 0, "rotary: tokens %d, heads %d / %d", tokens, H, Hkv);
    TTSMI_CHECK_ARG(dh > 0 && dh % 2 == 0 && rot >= 0 && rot % 2 == 0 && rot <= dh && rot <= 2 * ROT_MAX,
                    "rotary: %d of a head of %d elements (even, up to %d turned)", rot, dh, 2 * ROT_MAX);
    if (tokens == 0 || H + Hkv == 0) return TTSMI_OK;
    TTSMI_CHECK_ARG(positions && (freqs || rot == 0), "rotary: null positions or frequencies");
    TTSMI_CHECK_ARG((H == 0 || (q && qo)) && (Hkv == 0 || (k && ko)), "rotary: null tensor");
    const int size = dtype == TTSMI_F32 ? 4 : 2;
    TTSMI_CHECK_ARG((((uintptr_t)q | (uintptr_t)qo | (uintptr_t)k | (uintptr_t)ko) & (size_t)(size - 1)) == 0, "rotary: tensors are not element-aligned");
    RotP p = {};
    p.t[0] = {q, (long)q_row, (long)q_head, qo, (long)qo_row, (long)qo_head, H};
    p.t[1] = {k, (long)k_row, (long)k_head, ko, (long)ko_row, (long)ko_head, Hkv};
    p.pos = positions; p.freq = freqs; p.tokens = tokens; p.dh = dh; p.rot = rot; p.scale = scale; p.sign = inverse ? -1.f : 1.f;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TTSMI_F32) {
        const int pv = rotary_run(p, 4, 4);
        if (pv == 4) rotary_launch<float, 4>(p, interleaved, st);
        else if (pv == 2) rotary_launch<float, 2>(p, interleaved, st);
        else rotary_launch<float, 1>(p, interleaved, st);
    } else {
        const int pv = rotary_run(p, 8, 2);
        if (pv == 8) rotary_launch<__bf16, 8>(p, interleaved, st);
        else if (pv == 2) rotary_launch<__bf16, 2>(p, interleaved, st);
        else rotary_launch<__bf16, 1>(p, interleaved, st);
    }
    TTSMI_CHECK_LAUNCH("rotary");
    return TTSMI_OK;
}
