// Rotary embedding by explicit positions: every token carries its position on each of up to 8 axes (time, height,
// width, ...), so documents with different grids can share one packed row of tokens.  The grid form (positions derived
// from one regular grid, fused with RMSNorm) is rmsnorm_rope_kernel of norm.hip; reference: rope_apply
// (omnivideo/modules/model.py:37-65), which loops over samples because their grids differ.
//
//   pair p of a head belongs to axis a(p) and turns by pos[t][a(p)] * freq[p] revolutions:
//   (x0, x1) -> (x0 c - x1 s, x0 s + x1 c),  pairs (2p, 2p + 1) or (p, p + D/2).
//
// The angle is a 64-bit product reduced to a quarter turn in 64 bits, then sine and cosine by their Taylor polynomials in
// 32 bits (|r| <= pi/4: truncation below 2e-9).  The roundings of the frequency and of the product move an angle by at most
// 2^-51 of the turns that it has made: below 2e-7 turns for every int32 position, and there is no table to outgrow; fp32
// positions go further, and lose all meaning from about 1e15 on.  The rotation itself is fp32: 2^-20 of |x0| + |x1| at most,
// then the rounding to x's type.
// HBM-bound (every element read and written once): a lane owns 8 (bf16, fp32 alike) values of a head, computes the
// turns of its pairs once per token and applies them to every head of the token that falls to it.  56640 tokens x 12 heads
// of 128, bf16: 65 us = 5.3 TB/s.
#include "common.h"

namespace {

struct Turn {
    float c, s;
};

__device__ __forceinline__ Turn turn_of(double rev, bool inverse) {
    const double f = rev - __builtin_rint(rev);              // [-1/2, 1/2] revolutions, exact
    const double q = __builtin_rint(4.0 * f);                // nearest quarter
    const float r = (float)((4.0 * f - q) * 1.5707963267948966);
    const float r2 = r * r;
    const float sn = r * fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), 1.f);
    const float cs = fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f),
                                   -0.5f), 1.f);
    const int k = (int)q & 3;                                // -2 and 2 are the same half turn
    Turn t;
    t.c = (k & 1) ? sn : cs;
    t.s = (k & 1) ? cs : sn;
    if (k == 1 || k == 2) t.c = -t.c;
    if (k >= 2) t.s = -t.s;
    if (!(rev == rev) || f != f) t.c = t.s = __builtin_nanf("");
    if (inverse) t.s = -t.s;
    return t;
}

__device__ __forceinline__ void load8(const bf16_t* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = bf2f(w[j] & 0xffff);
        v[2 * j + 1] = bf2f(w[j] >> 16);
    }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void store8(bf16_t* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

struct RopeArgs {
    long ldx, ldo;
    const double* freq;        // revolutions per unit of position, [D / 2]
    const int* axis;           // [D / 2]; < 0: the pair is passed through
    long tokens;
    int n_axes, heads, D, heads_per_pass, tokens_per_wave;
    int inverse;
};

// INTER: pairs (2p, 2p + 1): a lane holds 4 pairs = 8 consecutive values.  Otherwise pairs (p, p + D/2): 8 pairs, 8
// values of either half.  A head takes D / 8 (D / 16) lanes; the 64 / that slots of a wave are heads of one token, or,
// where a token has fewer heads, of several tokens.
template <typename T, typename P, bool INTER>
__global__ void __launch_bounds__(256) rope_positions_kernel(const T* x, T* out, const P* __restrict__ pos, RopeArgs a) {
    constexpr int PAIRS = INTER ? 4 : 8;
    const int lane = threadIdx.x & 63;
    const int lanes = a.D / (2 * PAIRS);                     // lanes per head
    const int slot = lane / lanes, c = lane - slot * lanes;
    const int tw = slot / a.heads_per_pass, h0 = slot - tw * a.heads_per_pass;
    const long t = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * a.tokens_per_wave + tw;
    if (tw >= a.tokens_per_wave || t >= a.tokens) return;
    Turn tn[PAIRS];
    bool on[PAIRS];
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
        const int p = c * PAIRS + j, ax = a.axis[p];
        on[j] = ax >= 0 && ax < a.n_axes;
        tn[j] = turn_of((double)pos[t * a.n_axes + (on[j] ? ax : 0)] * a.freq[p], a.inverse != 0);
    }
    const int half = a.D >> 1;
    for (int h = h0; h < a.heads; h += a.heads_per_pass) {
        const T* src = x + t * a.ldx + (long)h * a.D + c * 8;
        T* dst = out + t * a.ldo + (long)h * a.D + c * 8;
        float u[8];
        load8(src, u);
        if constexpr (INTER) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x0 = u[2 * j], x1 = u[2 * j + 1];
                u[2 * j] = on[j] ? x0 * tn[j].c - x1 * tn[j].s : x0;
                u[2 * j + 1] = on[j] ? x0 * tn[j].s + x1 * tn[j].c : x1;
            }
            store8(dst, u);
        } else {
            float w[8];
            load8(src + half, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x0 = u[j], x1 = w[j];
                u[j] = on[j] ? x0 * tn[j].c - x1 * tn[j].s : x0;
                w[j] = on[j] ? x0 * tn[j].s + x1 * tn[j].c : x1;
            }
            store8(dst, u);
            store8(dst + half, w);
        }
    }
}

}  // namespace

int ovd_impl_rope_positions(const void* x, int is_f32, long ldx, const void* pos, int pos_is_f32, int n_axes,
                            const double* freq, const int* axis, void* out, long ldo, long tokens, int heads, int D,
                            int interleaved, int inverse, hipStream_t st) {
    OVD_REQUIRE(D > 0 && D % 16 == 0 && D <= 512, "rope_positions: head_dim %d must be a multiple of 16, at most 512", D);
    OVD_REQUIRE(tokens >= 0 && heads > 0 && n_axes >= 1 && n_axes <= 8, "rope_positions: bad shape tokens=%ld heads=%d axes=%d",
                tokens, heads, n_axes);
    const int per16 = is_f32 ? 4 : 8;
    OVD_REQUIRE(ldx >= (long)heads * D && ldo >= (long)heads * D && ldx % per16 == 0 && ldo % per16 == 0 &&
                    reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
                "rope_positions: token rows must keep 16-byte alignment and hold %d heads of %d", heads, D);
    if (tokens == 0) return 0;
    RopeArgs a;
    a.ldx = ldx;
    a.ldo = ldo;
    a.freq = freq;
    a.axis = axis;
    a.tokens = tokens;
    a.n_axes = n_axes;
    a.heads = heads;
    a.D = D;
    a.inverse = inverse;
    const int slots = 64 / (D / (interleaved ? 8 : 16));
    a.heads_per_pass = heads < slots ? heads : slots;
    a.tokens_per_wave = slots / a.heads_per_pass;
    const long blocks = (tokens + 4L * a.tokens_per_wave - 1) / (4L * a.tokens_per_wave);
    OVD_REQUIRE(blocks < (1L << 24), "rope_positions: grid too large");
#define ROPE_LAUNCH(T, P, I)                                                                                \
    hipLaunchKernelGGL((rope_positions_kernel<T, P, I>), dim3((unsigned)blocks), dim3(256), 0, st, (const T*)x, \
                       (T*)out, (const P*)pos, a)
#define ROPE_TYPES(I)                                                                                       \
    do {                                                                                                    \
        if (is_f32 && pos_is_f32) ROPE_LAUNCH(float, float, I);                                             \
        else if (is_f32) ROPE_LAUNCH(float, int, I);                                                        \
        else if (pos_is_f32) ROPE_LAUNCH(bf16_t, float, I);                                                 \
        else ROPE_LAUNCH(bf16_t, int, I);                                                                   \
    } while (0)
    if (interleaved) ROPE_TYPES(true);
    else ROPE_TYPES(false);
#undef ROPE_TYPES
#undef ROPE_LAUNCH
    OVD_CHECK_LAUNCH("rope_positions");
    return 0;
}
