// MXFP4 (OCP microscaling, E2M1 elements, one E8M0 scale per 32 values of a row): quantisation of row matrices and
// the product of two of them, out = epilogue(A[M,K] * W[N,K]^T + bias[N]), on fp4 operands of v_mfma_scale_f32_16x16x128_f8f6f4
// (256 x 256 tiles) and v_mfma_scale_f32_32x32x64_f8f6f4 (fewer rows).  A reduced-precision form of the linear layers beside the e4m3 one of fp8.hip (the reference runs
// these layers in bf16: omnivideo/modules/model.py:125-154, :159-179, :218-258).
//
// Definition of the quantisation (a block is 32 consecutive k of one row):
//   scale byte s = max(floor(log2 max|x|) - 2 + 127, 0), value of the scale 2^(s - 127); 255 (NaN) if the block holds
//   an infinity or a NaN, 0 for a block of zeros;  code = E2M1(x / 2^(s - 127)), to nearest, ties to even, saturated
//   at 6.  Division by a power of two is exact, so a code depends on one rounding only.
//
// Operand layout ("tiles").  Row block rb = 32 rows, Kp = K rounded up to 256:
//   data  [ceil(M/32)][Kp/64][64 lanes][16 bytes]: lane l = 32 h + r holds the 32 codes (low nibble first) of row
//         32 rb + r, k = 64 kt + 32 h ..: one MFMA operand fragment is 1 KiB of consecutive memory, in lane order;
//   scale [ceil(M/32)][Kp/256][64 lanes][4 bytes]: lane l, byte j = the scale byte of that lane's block in the j-th
//         64-wide k-step of the group: one coalesced dword load feeds four MFMAs (op_sel picks the byte).
// k in [K, Kp) hold zeros with scale byte 0.  Rows past M are not written and never read as valid rows.
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(2))) float f32x2;

enum Epi { EPI_BF16 = 0, EPI_BF16_GELU = 1, EPI_F32 = 2, EPI_RESID = 3, EPI_MX_GELU = 4 };

constexpr int KG = 256;                 // k-group: four MFMA k-steps, one scale dword per lane
constexpr int FRAG = 1024;              // bytes of a 32-row x 64-k fragment
constexpr int GRP_DATA = 4 * FRAG;      // bytes of a 32-row x 256-k group
constexpr int GRP_SCALE = 256;          // bytes of its scales

// scale byte of a block from the bits of its largest magnitude
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;                   // biased exponent; 255: infinity or NaN
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// the scale as the conversion to codes takes it: a float of that exponent field (0: 2^-127).  255 is a NaN's; the codes of
// such a block do not matter
__device__ __forceinline__ float cvt_scale(uint32_t s) { return __uint_as_float(s << 23); }
// 2^(s - 127); s = 0 is the denormal 2^-127, s = 255 a NaN
__device__ __forceinline__ float scale_value(uint32_t s) {
    return __uint_as_float(s == 0u ? 0x00400000u : (s == 255u ? 0x7FC00000u : s << 23));
}

// eight floats divided by `scale` -> eight codes, k ascending from the low nibble
__device__ __forceinline__ uint32_t pack_fp4x8(const float* v, float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
    return w;
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// ------------------------------------------------------------------------------------------ quantise / dequantise
// One workgroup = one row block x one k-group, a wave 8 of its rows.  A load instruction covers 8 rows x 64 k (8 lanes of
// 8 values per row: whole 128-byte lines of bf16), a store instruction two runs of 8 rows x 16 bytes; the four lanes of an
// MX block exchange their largest magnitude.  HBM-bound: 2 (4) bytes read and 17/32 written per value: 40560 x 8960 bf16
// there and back 335 us = 5.5 TB/s (with a wave over all 32 rows of the block 366, and 550 x 8960 2.7 times as long).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<bf16_t>(const bf16_t* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = bf2f(w[j] & 0xffff);
        v[2 * j + 1] = bf2f(w[j] >> 16);
    }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

template <typename T>
__global__ void __launch_bounds__(256) mxfp4_quant_kernel(const T* __restrict__ x, long ldx, uint8_t* __restrict__ data,
                                                          uint8_t* __restrict__ scale, int M, int K, int groups) {
    const int lane = threadIdx.x & 63;
    const long wid = blockIdx.x;
    const long rb = wid / groups;
    const int kg = (int)(wid % groups);
    const int r8 = lane >> 3, c = lane & 7;               // row inside the 8-row group, 8-value chunk of the 64-k step
    uint8_t* dst = data + wid * GRP_DATA + (c >> 2) * 512 + (c & 3) * 4;
    uint32_t* sdst = reinterpret_cast<uint32_t*>(scale + wid * GRP_SCALE) + (c >> 2) * 32;
    const int r = (threadIdx.x >> 6) * 8 + r8;
    const long row = rb * 32 + r;
    if (row >= M) return;                                 // eight lanes of a row share it: the exchanges stay whole
    const T* src = x + row * ldx + (long)kg * KG + c * 8;
    float v[4][8];
    uint32_t sc = 0;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        if (kg * KG + ks * 64 + c * 8 < K) load8<T>(src + ks * 64, v[ks]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[ks][j] = 0.f;
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        uint32_t mx = 0;                              // magnitudes compare as their bit patterns (NaN above all)
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = umax(mx, __float_as_uint(v[ks][j]) & 0x7fffffffu);
        mx = umax(mx, __shfl_xor(mx, 1, 64));
        mx = umax(mx, __shfl_xor(mx, 2, 64));
        const uint32_t s = scale_byte(mx);
        *reinterpret_cast<uint32_t*>(dst + ks * FRAG + r * 16) = pack_fp4x8(v[ks], cvt_scale(s));
        sc |= s << (8 * ks);
    }
    if ((c & 3) == 0) sdst[r] = sc;
}

// the mapping above, the other way; a value is code * 2^(s - 127), exact in bf16 and fp32.  A store instruction writes whole
// 128-byte lines: 8 lanes hold 8 bf16 values of a row each, or 4 fp32 ones (8 as two stores: 40560 x 1536 77 us against 65)
template <typename T>
__global__ void __launch_bounds__(256) mxfp4_dequant_kernel(const uint8_t* __restrict__ data,
                                                            const uint8_t* __restrict__ scale, T* __restrict__ out,
                                                            long ldo, int M, int K, int groups) {
    const int lane = threadIdx.x & 63;
    const long wid = blockIdx.x;
    const long rb = wid / groups;
    const int kg = (int)(wid % groups);
    const int r = (threadIdx.x >> 6) * 8 + (lane >> 3), c = lane & 7;
    const long row = rb * 32 + r;
    if (row >= M) return;
    const uint8_t* src = data + wid * GRP_DATA + r * 16;
    const uint32_t* ssrc = reinterpret_cast<const uint32_t*>(scale + wid * GRP_SCALE) + r;
    T* dst = out + row * ldo + (long)kg * KG;
    if constexpr (sizeof(T) == 2) {
        const uint32_t sc = ssrc[(c >> 2) * 32];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(src + ks * FRAG + (c >> 2) * 512 + (c & 3) * 4);
            const float s = scale_value((sc >> (8 * ks)) & 255u);
            const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0) * s;
            const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1) * s;
            const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2) * s;
            const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3) * s;
            if (kg * KG + ks * 64 + c * 8 < K)
                *reinterpret_cast<uint4*>(dst + ks * 64 + c * 8) =
                    make_uint4(pack_bf2(p0[0], p0[1]), pack_bf2(p1[0], p1[1]), pack_bf2(p2[0], p2[1]), pack_bf2(p3[0], p3[1]));
        }
    } else {
        const uint32_t sc[2] = {ssrc[0], ssrc[32]};
#pragma unroll
        for (int i = 0; i < 8; ++i) {                     // MX block i of the group
            const uint32_t w = *reinterpret_cast<const uint16_t*>(src + (i >> 1) * FRAG + (i & 1) * 512 + c * 2);
            const float s = scale_value((sc[i & 1] >> (8 * (i >> 1))) & 255u);
            const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0) * s;
            const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1) * s;
            if (kg * KG + i * 32 < K)
                *reinterpret_cast<float4*>(dst + i * 32 + c * 4) = make_float4(p0[0], p0[1], p1[0], p1[1]);
        }
    }
}

// ------------------------------------------------------------------------------------------------------- product
struct Operand {
    const uint8_t* data;
    const uint8_t* scale;
    int rows;
};

struct Out {
    const bf16_t* bias;
    void* out;
    long ldo;
    const float* gate;
};

// bias of columns n .. n + 3 (n % 4 == 0; past N: some other columns', for outputs that are not stored)
__device__ __forceinline__ uint2 load_bias(const Out& o, int n, int N) {
    return o.bias ? *reinterpret_cast<const uint2*>(o.bias + min(n, N - 4)) : make_uint2(0, 0);
}
__device__ __forceinline__ void add_bias(float (&y)[4], const uint2& b) {
    y[0] += bf2f(b.x & 0xffff);
    y[1] += bf2f(b.x >> 16);
    y[2] += bf2f(b.y & 0xffff);
    y[3] += bf2f(b.y >> 16);
}

// four consecutive columns n .. n + 3 (n % 4 == 0, n < N) of row m, bias added; the pre-activation stays in fp32: the
// only rounding is that of the stored value
template <int EPI>
__device__ __forceinline__ void store4(const Out& o, long m, int n, float (&y)[4]) {
    if constexpr (EPI == EPI_BF16 || EPI == EPI_BF16_GELU) {
        if constexpr (EPI == EPI_BF16_GELU) {
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = gelu_tanh_f(y[j]);
        }
        *reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(o.out) + m * o.ldo + n) =
            make_uint2(pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]));
    } else {
        float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(o.out) + m * o.ldo + n);
        if constexpr (EPI == EPI_RESID) {
            float4 x = *p;
            const float4 g = o.gate ? *reinterpret_cast<const float4*>(o.gate + n) : make_float4(1.f, 1.f, 1.f, 1.f);
            *p = make_float4(fmaf(y[0], g.x, x.x), fmaf(y[1], g.y, x.y), fmaf(y[2], g.z, x.z), fmaf(y[3], g.w, x.w));
        } else {
            *p = make_float4(y[0], y[1], y[2], y[3]);
        }
    }
}

// EPI_MX_GELU: the 32 x 32 block of outputs that a wave holds in `acc` (register 4 g + j of lane l: row l & 31, column
// 8 g + 4 (l >> 5) + j) through bias and GELU and, still in fp32, into one MX block per row of the next product's operand:
// a row's 32 values lie in two lanes, so its largest magnitude is 15 maxima and one exchange, and each lane ends up with
// the whole 16 bytes of codes, stored here (o.out, N columns, out_groups k-groups a row block).  Returns the block's scale
// byte.  Columns past N are written as zeros: they are the padding of that operand.
__device__ __forceinline__ uint32_t store_mx(const Out& o, const f32x16& acc, const uint2 (&bias)[4], long rb, int nb, long m, int M,
                                         int N, int out_groups, int lane) {
    const int h = lane >> 5;
    float y[16];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float t[4] = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
        add_bias(t, bias[g]);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[4 * g + j] = t[j];
    }
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        y[i] = nb * 32 < N ? gelu_tanh_f(y[i]) : 0.f;
        mx = umax(mx, __float_as_uint(y[i]) & 0x7fffffffu);
    }
    const auto ex = __builtin_amdgcn_permlane32_swap(mx, mx, false, false);
    const uint32_t s = scale_byte(umax(ex[0], ex[1]));
    const uint32_t w[2] = {pack_fp4x8(y, cvt_scale(s)), pack_fp4x8(y + 8, cvt_scale(s))};      // 4 g + j ascending, 16 bits per g
    // word g of the block = columns 8 g .. 8 g + 7: 16 bits from the lower lane, 16 from the upper
    const auto e0 = __builtin_amdgcn_permlane32_swap(w[0], w[0], false, false);
    const auto e1 = __builtin_amdgcn_permlane32_swap(w[1], w[1], false, false);
    if (h == 0 && m < M) {
        uint8_t* data = reinterpret_cast<uint8_t*>(o.out) + ((rb * out_groups + (nb >> 3)) * 4 + ((nb >> 1) & 3)) * FRAG;
        *reinterpret_cast<uint4*>(data + ((nb & 1) * 32 + (lane & 31)) * 16) =
            make_uint4((e0[0] & 0xffffu) | (e0[1] << 16), (e0[0] >> 16) | (e0[1] & 0xffff0000u),
                       (e1[0] & 0xffffu) | (e1[1] << 16), (e1[0] >> 16) | (e1[1] & 0xffff0000u));
    }
    return s;
}
// The same for a wave that holds 16 rows x 32 columns of a block in two 16 x 16 pieces (register j of y0 / y1 of lane l: row
// l & 15, column 4 (l >> 4) + j / 16 + that): a row lies in four lanes, each of which ends up with four bytes of its codes
// and writes them to `row_codes`, the row's 16 bytes.
__device__ __forceinline__ uint32_t pack_mx16(const f32x4& y0, const f32x4& y1, const uint2 (&bias)[2], bool inside, char* row_codes,
                                              int lane) {
    float t0[4] = {y0[0], y0[1], y0[2], y0[3]}, t1[4] = {y1[0], y1[1], y1[2], y1[3]};
    add_bias(t0, bias[0]);
    add_bias(t1, bias[1]);
    float y[8];
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = inside ? gelu_tanh_f(i < 4 ? t0[i & 3] : t1[i & 3]) : 0.f;
        mx = umax(mx, __float_as_uint(y[i]) & 0x7fffffffu);
    }
    const auto e0 = __builtin_amdgcn_permlane16_swap(mx, mx, false, false);
    mx = umax(e0[0], e0[1]);
    const auto e1 = __builtin_amdgcn_permlane32_swap(mx, mx, false, false);
    const uint32_t s = scale_byte(umax(e1[0], e1[1]));
    // columns 4 q .. 4 q + 3 in the low half of lane quarter q's word, 16 columns on in the high half: even quarters take the
    // low halves of a pair, odd ones the high halves
    const uint32_t c = pack_fp4x8(y, cvt_scale(s));
    const auto ex = __builtin_amdgcn_permlane16_swap(c, c >> 16, false, false);
    const int q = lane >> 4;
    *reinterpret_cast<uint32_t*>(row_codes + (q & 1) * 8 + (q >> 1) * 4) = (ex[0] & 0xffffu) | (ex[1] << 16);
    return s;
}
// the scale buffer of an MXFP4 output (o.gate holds its address)
__device__ __forceinline__ uint8_t* mx_scales(const Out& o) { return reinterpret_cast<uint8_t*>(const_cast<float*>(o.gate)); }

// one 32-row x 256-k group of an operand in registers
struct Group {
    uint4 f[4];
    int s;
};

__device__ __forceinline__ Group load_group(const Operand& op, long rb, int kg, int groups, int lane) {
    Group g;
    if (rb * 32 + (lane & 31) < op.rows) {
        const uint4* p = reinterpret_cast<const uint4*>(op.data + (rb * groups + kg) * GRP_DATA) + lane;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) g.f[ks] = p[ks * 64];
        g.s = reinterpret_cast<const int*>(op.scale + (rb * groups + kg) * GRP_SCALE)[lane];
    } else {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) g.f[ks] = make_uint4(0, 0, 0, 0);
        g.s = 0;
    }
    return g;
}

__device__ __forceinline__ i32x8 frag8(const uint4& u) {
    return (i32x8){(int)u.x, (int)u.y, (int)u.z, (int)u.w, 0, 0, 0, 0};
}

// acc += W fragment x A fragment over a k-group; op_sel picks byte ks of the scale dwords
__device__ __forceinline__ void mfma_group(f32x16& acc, const Group& w, const Group& a) {
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag8(w.f[0]), frag8(a.f[0]), acc, 4, 4, 0, w.s, 0, a.s);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag8(w.f[1]), frag8(a.f[1]), acc, 4, 4, 1, w.s, 1, a.s);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag8(w.f[2]), frag8(a.f[2]), acc, 4, 4, 2, w.s, 2, a.s);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag8(w.f[3]), frag8(a.f[3]), acc, 4, 4, 3, w.s, 3, a.s);
}

// Not enough 256 x 256 tiles for the card: a workgroup of 8 waves owns MT x NT blocks of 32 x 32 outputs, its waves take
// the k-groups in turn, fragments straight from memory (they are in lane order there) one group ahead, and the eight
// partial sums meet in LDS in a fixed order.  Weight rows sit on the MFMA's M axis, so a lane ends with 4 consecutive
// columns of one row.  Bound by the trips to memory (4 to 5 a wave at K = 8960) and the traffic of L2: 550 x 1536 x 8960
// 12 us = 1.3 PFLOP/s (tiles in the order of the workgroups instead of runs per XCD: 15 us).
template <int MT, int NT, int EPI>
__global__ void __launch_bounds__(512) gemm_mxfp4_direct_kernel(Operand A, Operand W, Out o, int groups, unsigned tiles_m) {
    extern __shared__ float4 part[];          // [8 waves][MT * NT * 4 register quads][64 lanes]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // workgroups go to the XCDs in turn: XCD x takes the x-th run of tiles, column by column of the output
    const unsigned per = gridDim.x / 8, extra = gridDim.x % 8, xcd = blockIdx.x % 8;
    const unsigned tile = xcd * per + min(xcd, extra) + blockIdx.x / 8;
    const long rb0 = (long)(tile % tiles_m) * MT, nb0 = (long)(tile / tiles_m) * NT;
    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    Group a[MT], w[NT], an[MT], wn[NT];
    if (wave < groups) {
#pragma unroll
        for (int j = 0; j < NT; ++j) w[j] = load_group(W, nb0 + j, wave, groups, lane);
#pragma unroll
        for (int i = 0; i < MT; ++i) a[i] = load_group(A, rb0 + i, wave, groups, lane);
        for (int kg = wave; kg < groups; kg += 8) {
            const int nx = kg + 8 < groups ? kg + 8 : kg;          // the last step reads its own group again, unused
#pragma unroll
            for (int j = 0; j < NT; ++j) wn[j] = load_group(W, nb0 + j, nx, groups, lane);
#pragma unroll
            for (int i = 0; i < MT; ++i) an[i] = load_group(A, rb0 + i, nx, groups, lane);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) mfma_group(acc[i][j], w[j], a[i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) w[j] = wn[j];
#pragma unroll
            for (int i = 0; i < MT; ++i) a[i] = an[i];
        }
    }
    constexpr int Q = MT * NT * 4;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                part[(wave * Q + (i * NT + j) * 4 + g) * 64 + lane] =
                    make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
    __syncthreads();
    if constexpr (EPI == EPI_MX_GELU) {          // an MX block needs all 32 columns of a row: one wave per 32 x 32 block
        if (wave >= MT * NT) return;
        f32x16 t;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float4 p = part[(k * Q + wave * 4 + g) * 64 + lane];
                y.x += p.x;
                y.y += p.y;
                y.z += p.z;
                y.w += p.w;
            }
            t[4 * g] = y.x;
            t[4 * g + 1] = y.y;
            t[4 * g + 2] = y.z;
            t[4 * g + 3] = y.w;
        }
        const long rb = rb0 + wave / NT;
        uint2 bias[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) bias[g] = load_bias(o, (int)(nb0 + wave % NT) * 32 + 8 * g + 4 * (lane >> 5), W.rows);
        const int nb = (int)(nb0 + wave % NT), out_groups = (W.rows + KG - 1) / KG;
        const long m = rb * 32 + (lane & 31);
        const uint32_t sb = store_mx(o, t, bias, rb, nb, m, A.rows, W.rows, out_groups, lane);
        if (lane < 32 && m < A.rows)
            mx_scales(o)[(rb * out_groups + (nb >> 3)) * GRP_SCALE + ((nb & 1) * 32 + lane) * 4 + ((nb >> 1) & 3)] = (uint8_t)sb;
        return;
    }
    for (int q = wave; q < Q; q += 8) {
        float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float4 p = part[(k * Q + q) * 64 + lane];
            y[0] += p.x;
            y[1] += p.y;
            y[2] += p.z;
            y[3] += p.w;
        }
        const int g = q & 3, j = (q >> 2) % NT, i = (q >> 2) / NT;
        const long m = (rb0 + i) * 32 + (lane & 31);
        const int n = (int)(nb0 + j) * 32 + 8 * g + 4 * (lane >> 5);
        if constexpr (EPI != EPI_MX_GELU) {
            add_bias(y, load_bias(o, n, W.rows));
            if (m < A.rows && n < W.rows) store4<EPI>(o, m, n, y);
        }
    }
}

// A handful of rows (M <= FEW_ROWS) straight from bf16 / fp32: every workgroup quantises all of x into LDS (a few thousand
// values) under its first weight loads, so a token's layer is one launch.  A workgroup owns one block of 32 weight rows;
// its waves take the k-groups in turn and meet as above.  Bound by the weights: one row of 5120 x 5120 5.6 us (launch
// and one trip to memory 3, 13.9 MB of weights the rest, on the 160 CUs that have a block); as two launches 8.  LDS: codes [group][ks][h][FEW_ROWS][16], scales
// [group][h][FEW_ROWS][4], then the partial sums.
constexpr int FEW_ROWS = 8;
constexpr int FEW_GRP = 8 * FEW_ROWS * 16 + 2 * FEW_ROWS * 4;       // LDS bytes per k-group
constexpr int FEW_PART = 8 * 4 * 64 * 16;

template <typename T, int EPI>
__global__ void __launch_bounds__(512) linear_mxfp4_few_kernel(const T* __restrict__ x, long ldx, Operand W, Out o, int M, int K,
                                                               int groups) {
    extern __shared__ __attribute__((aligned(16))) char few_smem[];
    char* codes = few_smem;
    char* scales = few_smem + groups * (8 * FEW_ROWS * 16);
    float4* part = reinterpret_cast<float4*>(few_smem + (groups * FEW_GRP + 15) / 16 * 16);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 31, h = lane >> 5;
    Group w;
    if (wave < groups) w = load_group(W, blockIdx.x, wave, groups, lane);
    const int chunks = groups * 32;                       // 8-value chunks per row; a block's four sit in adjacent lanes
    for (int i = tid; i < M * chunks; i += 512) {
        const int m = i / chunks, c = i - m * chunks;
        float v[8];
        if (c * 8 < K) load8<T>(x + m * ldx + c * 8, v);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        uint32_t mx = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = umax(mx, __float_as_uint(v[j]) & 0x7fffffffu);
        mx = umax(mx, __shfl_xor(mx, 1, 64));
        mx = umax(mx, __shfl_xor(mx, 2, 64));
        const uint32_t s = scale_byte(mx);
        const int kg = c >> 5, ks = (c >> 3) & 3, hh = (c >> 2) & 1;
        *reinterpret_cast<uint32_t*>(codes + ((kg * 4 + ks) * 2 + hh) * (FEW_ROWS * 16) + m * 16 + (c & 3) * 4) =
            pack_fp4x8(v, cvt_scale(s));
        if ((c & 3) == 0) scales[((kg * 2 + hh) * FEW_ROWS + m) * 4 + ks] = (char)s;
    }
    __syncthreads();
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    for (int kg = wave; kg < groups; kg += 8) {
        Group a;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
            a.f[ks] = r < M ? *reinterpret_cast<const uint4*>(codes + ((kg * 4 + ks) * 2 + h) * (FEW_ROWS * 16) + r * 16)
                            : make_uint4(0, 0, 0, 0);
        a.s = r < M ? *reinterpret_cast<const int*>(scales + ((kg * 2 + h) * FEW_ROWS + r) * 4) : 0;
        const Group wn = load_group(W, blockIdx.x, kg + 8 < groups ? kg + 8 : kg, groups, lane);
        mfma_group(acc, w, a);
        w = wn;
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) part[(wave * 4 + g) * 64 + lane] = make_float4(acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]);
    __syncthreads();
    if (wave >= 4) return;
    float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float4 p = part[(k * 4 + wave) * 64 + lane];
        y[0] += p.x;
        y[1] += p.y;
        y[2] += p.z;
        y[3] += p.w;
    }
    const int n = blockIdx.x * 32 + 8 * wave + 4 * h;
    add_bias(y, load_bias(o, n, W.rows));
    if (r < M && n < W.rows) store4<EPI>(o, r, n, y);
}

// ------------------------------------------------------------------------------------------ product, many rows
// The four-phase schedule of gemm256.hip on 256 x 256 output tiles: K-tiles of one k-group (128 bytes of codes per row,
// 64 KiB for both operands), two LDS buffers, one 16 KiB half-tile staged per phase, DMA never drained inside the loop,
// the two wave groups one barrier apart.  A phase is 16 v_mfma_scale_f32_16x16x128_f8f6f4 on fp4 operands: the matrix time
// of the 4 e4m3 ones of fp8.hip's phase for twice the K, so LDS and DMA bytes per matrix cycle are the same.
// The tile layout makes every DMA instruction 1 KiB of consecutive memory and every fragment read four runs of 256 bytes of
// LDS: no swizzle.  Scales travel the same way, one 256-byte instruction per row block and K-tile (8 KiB of LDS for two
// buffers); they are issued with phase 4, so any four consecutive phases hold 10 DMA instructions of a wave.
// 32760 x 5120 x 13824: 0.99 ms = 4.7 PFLOP/s, bound by power: the matrix pipe is busy 61 % of cycles at the 1.6 to 1.9 GHz
// that the chip then holds, and operands of zeros take 785 us.  The instruction shape is a matter of power, too: a loop
// of products of Gaussian values alone holds 6.8 PFLOP/s as 32x32x64, 7.4 as 16x16x128 (fewer accumulators pass by per
// product), 7.55 where only one operand changes from one to the next; the whole product gains 2 to 4 %.
// 40560 x 8960 x 1536: 332 us bf16, 400 with GELU, 414 to 428 with the GELU quantised, 459 fp32, 722 with a residual: with six
// k-groups a tile the epilogue is a third of the time (its vector work and the stores).
// Not better: four waves of 128 x 128 outputs (4.3 PFLOP/s, a longer epilogue); 128 x 256 tiles in two workgroups per CU
// (long K 3.8 PFLOP/s; short K with GELU 406 us against 421 then); the closing barriers ahead of a phase's last products
// (2000 x 5120 x 5120 36.5 us against 34: the next reads wait behind them).
constexpr int TM = 256, TN = 256;
constexpr int PBUF = 2 * 8 * GRP_DATA;            // one buffer: A 8 row blocks x 4 KiB | W the same
constexpr int SBUF = 2 * 8 * GRP_SCALE;           // its scales
constexpr int BIG_LDS = 2 * PBUF + 2 * SBUF;

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// this wave's DMA sources: fragment `wave & 3` of two row blocks of either half, and the scales of row block `wave`
struct Feed {
    const uint8_t* data[4];      // instruction i of a tile: row block (i * 8 + wave) / 4, k-step wave & 3
    const uint8_t* scale;
};

template <int HALF>
__device__ __forceinline__ void stage_half(const Feed& f, long kg, char* part_wave) {
    __builtin_amdgcn_global_load_lds(f.data[2 * HALF] + kg * GRP_DATA, (lds_ptr)(part_wave + (2 * HALF) * 8192), 16, 0, 0);
    __builtin_amdgcn_global_load_lds(f.data[2 * HALF + 1] + kg * GRP_DATA, (lds_ptr)(part_wave + (2 * HALF + 1) * 8192), 16, 0, 0);
}
__device__ __forceinline__ void stage_scales(const Feed& fa, const Feed& fw, long kg, char* dst_wave) {
    __builtin_amdgcn_global_load_lds(fa.scale + kg * GRP_SCALE, (lds_ptr)dst_wave, 4, 0, 0);
    __builtin_amdgcn_global_load_lds(fw.scale + kg * GRP_SCALE, (lds_ptr)(dst_wave + 8 * GRP_SCALE), 4, 0, 0);
}

template <int N>
__device__ __forceinline__ void phase_open() {
    if (N == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (N == 2) asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
    if (N == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    if (N == 10) asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void phase_close() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
}

struct Frag4 {
    i32x4 f[2][2];               // a row block: its two halves of 16 rows, two k-steps of 128
};
__device__ __forceinline__ i32x8 frag8(const i32x4& u) { return (i32x8){u[0], u[1], u[2], u[3], 0, 0, 0, 0}; }
__device__ __forceinline__ Frag4 lds_frags(const char* p) {
    Frag4 r;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s) r.f[i][s] = *reinterpret_cast<const i32x4*>(p + s * 2 * FRAG + i * 256);
    return r;
}

// scales of N 16-row groups.  A lane's dword holds the bytes of k-blocks h, h + 2, h + 4, h + 6 (h = its quarter & 1): shifted by
// its quarter / 2 bytes, bytes 0 and 2 are those of its blocks in the two k-steps
template <int N>
__device__ __forceinline__ void read_scales(int (&s)[N], const char* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = *reinterpret_cast<const int*>(p + (i >> 1) * GRP_SCALE + (i & 1) * 64);
}
template <int N>
__device__ __forceinline__ void shift_scales(int (&s)[N], int shift) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = (unsigned)s[i] >> shift;
}

// 32 columns x 64 rows x 256 k.  From product to product only one operand changes: 2 % more than in plain order
#define MX_MFMA(J, I, S)                                                                                                     \
    c[J][I] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(frag8(w.f[J][S]), frag8(x[(I) >> 1].f[(I) & 1][S]), c[J][I], 4, 4, \
                                                               2 * (S), ws[J], 2 * (S), xs[I]);
#define MX_STEP(S)                                                                                                           \
    MX_MFMA(0, 0, S) MX_MFMA(1, 0, S) MX_MFMA(1, 1, S) MX_MFMA(0, 1, S)                                                      \
    MX_MFMA(0, 2, S) MX_MFMA(1, 2, S) MX_MFMA(1, 3, S) MX_MFMA(0, 3, S)
__device__ __forceinline__ void quadrant(f32x4 (&c)[2][4], const Frag4& w, const int (&ws)[2], const Frag4 (&x)[2], const int (&xs)[4]) {
    MX_STEP(0) MX_STEP(1)
}
#undef MX_STEP
#undef MX_MFMA

// TAIL 0: steady state, 1: next-to-last K-tile, 2: last
template <int TAIL>
__device__ __forceinline__ void k_tile(f32x4 (&acc)[2][2][2][4], char* smem, int buf, long kg1, long kg2, const Feed& fa, const Feed& fw,
                                       int a_rd, int w_rd, int sa_rd, int sw_rd, int wave, int shift) {
    const char* ca = smem + buf * PBUF + a_rd;
    const char* cw = smem + buf * PBUF + PBUF / 2 + w_rd;
    char* own = smem + buf * PBUF + wave * 1024;
    char* oth = smem + (buf ^ 1) * PBUF + wave * 1024;
    char* sbuf = smem + 2 * PBUF + buf * SBUF;
    Frag4 w0, w1, af[2];
    // phase 1
    w0 = lds_frags(cw);
    af[0] = lds_frags(ca);
    af[1] = lds_frags(ca + GRP_DATA);
    int xs[4], ws0[2], ws1[2];
    read_scales(xs, sbuf + sa_rd);
    read_scales(ws0, sbuf + 8 * GRP_SCALE + sw_rd);
    if (TAIL < 2) stage_half<1>(fw, kg1, oth + PBUF / 2);
    phase_open<TAIL == 2 ? 2 : 10>();
    shift_scales(xs, shift);
    shift_scales(ws0, shift);
    quadrant(acc[0][0], w0, ws0, af, xs);
    phase_close();
    // phase 2
    w1 = lds_frags(cw + 4 * GRP_DATA);
    read_scales(ws1, sbuf + 12 * GRP_SCALE + sw_rd);
    if (TAIL < 2) stage_half<1>(fa, kg1, oth);
    phase_open<TAIL == 2 ? 0 : 10>();
    shift_scales(ws1, shift);
    quadrant(acc[1][0], w1, ws1, af, xs);
    phase_close();
    // phase 3
    af[0] = lds_frags(ca + 4 * GRP_DATA);
    af[1] = lds_frags(ca + 5 * GRP_DATA);
    read_scales(xs, sbuf + 4 * GRP_SCALE + sa_rd);
    if (TAIL == 0) stage_half<0>(fw, kg2, own + PBUF / 2);
    phase_open<-1>();
    shift_scales(xs, shift);
    quadrant(acc[1][1], w1, ws1, af, xs);
    phase_close();
    // phase 4
    if (TAIL == 0) {
        stage_half<0>(fa, kg2, own);
        stage_scales(fa, fw, kg2, sbuf + wave * GRP_SCALE);
    }
    phase_open<TAIL == 0 ? 10 : TAIL == 1 ? 4 : -1>();
    quadrant(acc[0][1], w0, ws0, af, xs);
    if (TAIL != 0) {
        // a use in front of the closing barrier: the MFMAs of the last K-tiles would otherwise sink past it
#pragma unroll
        for (int i = 0; i < 16; ++i)
            asm volatile("" : "+v"(acc[i >> 3][(i >> 2) & 1][0][i & 3]), "+v"(acc[i >> 3][(i >> 2) & 1][1][i & 3]));
    }
    phase_close();
}

template <int EPI>
__device__ __forceinline__ void big_tile(const Operand& A, const Operand& W, const Out& o, int groups, int tiles_m, int tiles_n,
                                         int GM, int wide, int bid, char* smem) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));        // per-lane values are derived again for every tile instead of kept across the loop
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave >> 2, wc = wave & 3;
    const int per_group = GM * tiles_n;
    const int grp = bid / per_group, first_m = grp * GM;
    const int gsz = min(tiles_m - first_m, GM);
    const int tm = first_m + (bid % per_group) % gsz, tn = (bid % per_group) / gsz;
    const long row0 = (long)tm * TM;
    const int col0 = tn * TN;

    Feed fa, fw;
    {
        const int a_last = (A.rows - 1) >> 5, w_last = (W.rows - 1) >> 5;      // row blocks past the last repeat it
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int rb = (i * 8 + wave) >> 2, ks = wave & 3;
            const long ra = min(tm * 8 + rb, a_last), rw = min(tn * 8 + rb, w_last);
            fa.data[i] = A.data + ra * groups * GRP_DATA + ks * FRAG + lane * 16;
            fw.data[i] = W.data + rw * groups * GRP_DATA + ks * FRAG + lane * 16;
        }
        fa.scale = A.scale + (long)min(tm * 8 + wave, a_last) * groups * GRP_SCALE + lane * 4;
        fw.scale = W.scale + (long)min(tn * 8 + wave, w_last) * groups * GRP_SCALE + lane * 4;
    }
    // operand lanes of v_mfma_scale_f32_16x16x128: row l & 15, k-block quarter l >> 4 of a step of 128; in the layout, block
    // quarter q is half q & 1 of fragment q >> 1
    const int fr = lane & 15, quarter = lane >> 4;
    const int frag_at = (quarter >> 1) * FRAG + (quarter & 1) * 512 + fr * 16, scale_at = (quarter & 1) * 128 + fr * 4;
    const int a_rd = wr * 2 * GRP_DATA + frag_at, w_rd = wc * GRP_DATA + frag_at, shift = (quarter >> 1) * 8;
    const int sa_rd = wr * 2 * GRP_SCALE + scale_at, sw_rd = wc * GRP_SCALE + scale_at;
    uint2 bias[2][2];                    // loaded ahead of the DMA: no ordinary load waits behind it
    if (o.bias) {
#pragma unroll
        for (int nh = 0; nh < 2; ++nh)
#pragma unroll
            for (int g = 0; g < 2; ++g)
                bias[nh][g] = *reinterpret_cast<const uint2*>(o.bias + min(col0 + nh * 128 + wc * 32 + 16 * g + 4 * quarter, W.rows - 4));
    } else {
#pragma unroll
        for (int nh = 0; nh < 2; ++nh)
#pragma unroll
            for (int g = 0; g < 2; ++g) bias[nh][g] = make_uint2(0, 0);
    }
    f32x4 acc[2][2][2][4];               // [column half][row half][16 columns][16 rows]
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i >> 4][(i >> 3) & 1][(i >> 2) & 1][i & 3] = (f32x4){0.f, 0.f, 0.f, 0.f};
    char* const wd = smem + wave * 1024;
    char* const sd = smem + 2 * PBUF + wave * GRP_SCALE;
    stage_half<0>(fw, 0, wd + PBUF / 2);
    stage_half<0>(fa, 0, wd);
    stage_scales(fa, fw, 0, sd);
    stage_half<1>(fw, 0, wd + PBUF / 2);
    stage_half<1>(fa, 0, wd);
    stage_half<0>(fw, 1, wd + PBUF + PBUF / 2);
    stage_half<0>(fa, 1, wd + PBUF);
    stage_scales(fa, fw, 1, sd + SBUF);
    asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    if (wr == 1) __builtin_amdgcn_s_barrier();            // second half of the waves: one barrier behind
    int t = 0;
    for (; t + 2 < groups; ++t)
        k_tile<0>(acc, smem, t & 1, t + 1, t + 2, fa, fw, a_rd, w_rd, sa_rd, sw_rd, wave, shift);
    k_tile<1>(acc, smem, t & 1, t + 1, 0, fa, fw, a_rd, w_rd, sa_rd, sw_rd, wave, shift);
    ++t;
    k_tile<2>(acc, smem, t & 1, 0, 0, fa, fw, a_rd, w_rd, sa_rd, sw_rd, wave, shift);
    if (wr == 0) __builtin_amdgcn_s_barrier();            // balances the extra barrier above
    asm volatile("" ::: "memory");

    // acc[nh][mh][g][i] register j is out[m][n + j], m = row0 + mh * 128 + wr * 64 + i * 16 + (lane & 15),
    // n = col0 + nh * 128 + wc * 32 + 16 g + 4 (lane >> 4).  bf16 rows go through LDS (256 rows of 512 bytes, chunk c of row r
    // at c ^ (r & 15)) so that 32 lanes store one 512-byte row segment.
    constexpr bool NARROW = EPI == EPI_BF16 || EPI == EPI_BF16_GELU;
    if constexpr (EPI == EPI_MX_GELU) {          // a tile's 256 columns are one k-group of the next operand
        // codes and scale bytes meet in LDS, [row block][4 KiB] and [row block][lane][4] as in memory; a wave stores a row block
        const int out_groups = (W.rows + KG - 1) / KG;
        char* const scales = smem + 8 * GRP_DATA;
#pragma unroll
        for (int q = 0; q < 8; ++q)              // mh * 4 + i
#pragma unroll
            for (int nh = 0; nh < 2; ++nh) {
                const int rbl = (q >> 2) * 4 + wr * 2 + ((q >> 1) & 1), r = (wc & 1) * 32 + (q & 1) * 16 + fr, ks = nh * 2 + (wc >> 1);
                const uint32_t sb = pack_mx16(acc[nh][q >> 2][0][q & 3], acc[nh][q >> 2][1][q & 3], bias[nh],
                                              col0 + nh * 128 + wc * 32 < W.rows, smem + rbl * GRP_DATA + ks * FRAG + r * 16, lane);
                if (quarter == 0) scales[rbl * GRP_SCALE + r * 4 + ks] = (char)sb;
            }
        __syncthreads();
        const long rb = tm * 8 + wave;
        if (rb * 32 + (lane & 31) < A.rows) {
            u32x4* data = reinterpret_cast<u32x4*>(reinterpret_cast<uint8_t*>(o.out) + (rb * out_groups + tn) * GRP_DATA) + lane;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
                data[ks * 64] = *reinterpret_cast<const u32x4*>(smem + wave * GRP_DATA + ks * FRAG + lane * 16);
            reinterpret_cast<uint32_t*>(mx_scales(o) + (rb * out_groups + tn) * GRP_SCALE)[lane] =
                reinterpret_cast<const uint32_t*>(scales + wave * GRP_SCALE)[lane];
        }
    } else if (NARROW && wide) {
#pragma unroll
        for (int q = 0; q < 8; ++q)              // mh * 4 + i
#pragma unroll
            for (int nh = 0; nh < 2; ++nh)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const f32x4& v = acc[nh][q >> 2][g][q & 3];
                    float y[4] = {v[0], v[1], v[2], v[3]};
                    add_bias(y, bias[nh][g]);
                    if constexpr (EPI == EPI_BF16_GELU) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = gelu_tanh_f(y[j]);
                    }
                    const int rl = (q >> 2) * 128 + wr * 64 + (q & 3) * 16 + fr, c = nh * 16 + wc * 4 + g * 2 + (quarter >> 1);
                    *reinterpret_cast<uint2*>(smem + rl * 512 + ((c ^ fr) << 4) + (quarter & 1) * 8) =
                        make_uint2(pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]));
                }
        __syncthreads();
        const int rr = tid >> 5, cc = tid & 31;
        const int n = col0 + cc * 8;
        const char* img = smem + rr * 512 + ((cc ^ rr) << 4);                 // row r = 16 i + rr: r & 15 = rr
        bf16_t* ob = reinterpret_cast<bf16_t*>(o.out) + (row0 + rr) * o.ldo + n;
        const long step = 16 * o.ldo;
        if (row0 + TM <= A.rows && col0 + TN <= W.rows) {                     // uniform
#pragma unroll 8
            for (int i = 0; i < 16; ++i) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(img + i * 8192);
                __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(ob));
                ob += step;
            }
        } else {
            for (int i = 0; i < 16; ++i, ob += step) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(img + i * 8192);
                if (row0 + i * 16 + rr < A.rows) {
                    if (n + 8 <= W.rows)
                        __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(ob));
                    else if (n < W.rows)
                        *reinterpret_cast<uint2*>(ob) = make_uint2(v[0], v[1]);
                }
            }
        }
    } else if constexpr (!NARROW) {
        // fp32 rows through LDS in two halves of 128 rows of 1 KiB (chunk c of row r at c ^ (r & 15)): a wave reads and writes
        // whole rows of the tile (40560 x 8960 x 1536 with a residual 702 us, 64-byte pieces straight from the registers 826)
        const int n = col0 + lane * 4;
        const bool inside = n < W.rows;
        const float4 gate = EPI == EPI_RESID && o.gate && inside ? *reinterpret_cast<const float4*>(o.gate + n) : make_float4(1.f, 1.f, 1.f, 1.f);
#pragma unroll
        for (int mh = 0; mh < 2; ++mh) {
            if (mh) __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int nh = 0; nh < 2; ++nh)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const f32x4& v = acc[nh][mh][g][i];
                        float y[4] = {v[0], v[1], v[2], v[3]};
                        add_bias(y, bias[nh][g]);
                        const int rl = wr * 64 + i * 16 + fr, c = nh * 32 + wc * 8 + g * 4 + quarter;
                        *reinterpret_cast<f32x4*>(smem + rl * 1024 + ((c ^ fr) << 4)) = (f32x4){y[0], y[1], y[2], y[3]};
                    }
            __syncthreads();
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                f32x4 xs[8];
                const long m0 = row0 + mh * 128 + b * 64 + wave;               // rows m0, m0 + 8, ...
                float* ob = reinterpret_cast<float*>(o.out) + m0 * o.ldo + n;
                if constexpr (EPI == EPI_RESID) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (m0 + 8 * i < A.rows && inside) xs[i] = *reinterpret_cast<const f32x4*>(ob + 8 * i * o.ldo);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int rl = b * 64 + 8 * i + wave;
                    const f32x4 y = *reinterpret_cast<const f32x4*>(smem + rl * 1024 + ((lane ^ (rl & 15)) << 4));
                    if (m0 + 8 * i >= A.rows || !inside) continue;
                    if constexpr (EPI == EPI_RESID)
                        *reinterpret_cast<f32x4*>(ob + 8 * i * o.ldo) =
                            (f32x4){fmaf(y[0], gate.x, xs[i][0]), fmaf(y[1], gate.y, xs[i][1]), fmaf(y[2], gate.z, xs[i][2]),
                                    fmaf(y[3], gate.w, xs[i][3])};
                    else
                        *reinterpret_cast<f32x4*>(ob + 8 * i * o.ldo) = y;
                }
            }
        }
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const long m = row0 + (q >> 2) * 128 + wr * 64 + (q & 3) * 16 + fr;
#pragma unroll
            for (int nh = 0; nh < 2; ++nh)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int n = col0 + nh * 128 + wc * 32 + 16 * g + 4 * quarter;
                    const f32x4& v = acc[nh][q >> 2][g][q & 3];
                    float y[4] = {v[0], v[1], v[2], v[3]};
                    add_bias(y, bias[nh][g]);
                    if (m < A.rows && n < W.rows) store4<EPI>(o, m, n, y);
                }
        }
    }
}

// Persistent, one workgroup per CU; the workgroups of an XCD take the tiles of that XCD's chunk of the walk in turn
template <int EPI>
__global__ void __launch_bounds__(512, 2) gemm_mxfp4_big_kernel(Operand A, Operand W, Out o, int groups, int tiles_m, int tiles_n,
                                                                int GM, int wide) {
    extern __shared__ __attribute__((aligned(16))) char big_smem[];
    const int nwg = tiles_m * tiles_n;
    const int xcd = blockIdx.x & 7, q = nwg >> 3, r = nwg & 7;
    const int first = xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q;
    const int count = q + (xcd < r ? 1 : 0);
    const int per_xcd = (gridDim.x + 7) >> 3;
    // All tiles take equally long, so the workgroups of a launch store at the same time and then all compute.  Quarters of
    // them start 3.7 us apart, the ones with a tile fewer last: 40560 x 4608 x 1536 191 us without, 171 with, with GELU 232 and
    // 203, quantised 243 and 220; 4500 x 8960 x 1536 50 and 44.  With long K the stores are a small part and the delay is lost
    // (40560 x 1536 x 8960: 254 without, 261 with), and below two rounds it can cost a round (3000 x 8960 x 1536 quantised:
    // 39 without, 44 with)
    if (groups <= 20 && nwg >= 2 * (int)gridDim.x)
        for (int i = (int)(blockIdx.x >> 3) * 4 / per_xcd; i > 0; --i) __builtin_amdgcn_s_sleep(127);
    for (int t = blockIdx.x >> 3; t < count; t += per_xcd) {
        big_tile<EPI>(A, W, o, groups, tiles_m, tiles_n, GM, wide, first + t, big_smem);
        __syncthreads();          // the LDS buffers are staged again by the next tile
    }
}

}  // namespace

static long mx_groups(long K) { return (K + KG - 1) / KG; }

long ovd_impl_mxfp4_data_bytes(long rows, long K) { return (rows + 31) / 32 * mx_groups(K) * GRP_DATA; }
long ovd_impl_mxfp4_scale_bytes(long rows, long K) { return (rows + 31) / 32 * mx_groups(K) * GRP_SCALE; }

int ovd_impl_mxfp4_quant(const void* x, int x_is_f32, long ldx, uint8_t* data, uint8_t* scale, int M, int K, hipStream_t st) {
    OVD_REQUIRE(M >= 0 && K > 0 && K % 32 == 0, "mxfp4_quant: K=%d must be a positive multiple of 32 (M=%d)", K, M);
    OVD_REQUIRE(ldx >= K && ldx % (x_is_f32 ? 4 : 8) == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(data) % 16 == 0 && reinterpret_cast<uintptr_t>(scale) % 4 == 0,
                "mxfp4_quant: rows must keep 16-byte alignment (ldx=%ld)", ldx);
    if (M == 0) return 0;
    const int groups = (int)mx_groups(K);
    const long blocks = (long)ceil_div(M, 32) * groups;
    OVD_REQUIRE(blocks < (1L << 24), "mxfp4_quant: grid too large");
    const dim3 grid((unsigned)blocks), blk(256);
    if (x_is_f32)
        hipLaunchKernelGGL(mxfp4_quant_kernel<float>, grid, blk, 0, st, (const float*)x, ldx, data, scale, M, K, groups);
    else
        hipLaunchKernelGGL(mxfp4_quant_kernel<bf16_t>, grid, blk, 0, st, (const bf16_t*)x, ldx, data, scale, M, K, groups);
    OVD_CHECK_LAUNCH("mxfp4_quant");
    return 0;
}

int ovd_impl_mxfp4_dequant(const uint8_t* data, const uint8_t* scale, void* out, int out_is_f32, long ldo, int M, int K,
                           hipStream_t st) {
    OVD_REQUIRE(M >= 0 && K > 0 && K % 32 == 0, "mxfp4_dequant: K=%d must be a positive multiple of 32 (M=%d)", K, M);
    OVD_REQUIRE(ldo >= K && ldo % (out_is_f32 ? 4 : 8) == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(data) % 16 == 0 && reinterpret_cast<uintptr_t>(scale) % 4 == 0,
                "mxfp4_dequant: rows must keep 16-byte alignment (ldo=%ld)", ldo);
    if (M == 0) return 0;
    const int groups = (int)mx_groups(K);
    const long blocks = (long)ceil_div(M, 32) * groups;
    OVD_REQUIRE(blocks < (1L << 24), "mxfp4_dequant: grid too large");
    const dim3 grid((unsigned)blocks), blk(256);
    if (out_is_f32)
        hipLaunchKernelGGL(mxfp4_dequant_kernel<float>, grid, blk, 0, st, data, scale, (float*)out, ldo, M, K, groups);
    else
        hipLaunchKernelGGL(mxfp4_dequant_kernel<bf16_t>, grid, blk, 0, st, data, scale, (bf16_t*)out, ldo, M, K, groups);
    OVD_CHECK_LAUNCH("mxfp4_dequant");
    return 0;
}

// whether the M rows of x and of the output share memory (x += f(x) on a residual stream): a product that reads x while it
// writes its output must not run then
static bool rows_overlap(const void* x, long x_row_bytes, long x_last, const void* out, long out_row_bytes, long out_last, int M) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(out);
    return a < b + (M - 1) * out_row_bytes + out_last && b < a + (M - 1) * x_row_bytes + x_last;
}

static bool few_rows(int M, int K) { return M <= FEW_ROWS && mx_groups(K) * FEW_GRP + FEW_PART + 16 <= 160 * 1024; }

// bytes for the quantised x of ovd_impl_linear_mxfp4 (0: it needs none)
long ovd_impl_linear_mxfp4_workspace(int M, int K) {
    return few_rows(M, K) ? 0 : ovd_impl_mxfp4_data_bytes(M, K) + ovd_impl_mxfp4_scale_bytes(M, K);
}

int ovd_impl_gemm_mxfp4(const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*, const bf16_t*, void*, long,
                        const float*, int, int, int, int, int, hipStream_t);

// the output side of both products
static int check_out(int M, int N, int K, int epilogue, const void* out, long ldo, const void* bias, const void* gate,
                     const void* w_data, const void* w_scale) {
    OVD_REQUIRE(M >= 0 && N > 0 && N % 4 == 0 && K > 0 && K % 32 == 0,
                "gemm_mxfp4: M=%d N=%d K=%d not supported: N %% 4, K %% 32", M, N, K);
    OVD_REQUIRE(epilogue >= EPI_BF16 && epilogue <= EPI_MX_GELU, "gemm_mxfp4: unknown epilogue %d", epilogue);
    OVD_REQUIRE(reinterpret_cast<uintptr_t>(w_data) % 16 == 0 && reinterpret_cast<uintptr_t>(w_scale) % 4 == 0,
                "gemm_mxfp4: operands must be 16-byte aligned");
    if (epilogue == EPI_MX_GELU) {
        OVD_REQUIRE(N % 32 == 0 && gate != nullptr && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(gate) % 4 == 0 && reinterpret_cast<uintptr_t>(bias) % 8 == 0,
                    "gemm_mxfp4: an MXFP4 output needs N %% 32 == 0 (N=%d), codes and scales", N);
        return 0;
    }
    OVD_REQUIRE(gate == nullptr || epilogue == EPI_RESID, "gemm_mxfp4: a gate goes with the residual epilogue");
    OVD_REQUIRE(ldo >= N && ldo % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (epilogue <= EPI_BF16_GELU ? 8 : 16) == 0 &&
                    reinterpret_cast<uintptr_t>(bias) % 8 == 0 && reinterpret_cast<uintptr_t>(gate) % 16 == 0,
                "gemm_mxfp4: out rows, bias and gate must be aligned to 4 values (ldo=%ld)", ldo);
    return 0;
}

int ovd_impl_linear_mxfp4(const void* x, int x_is_f32, long ldx, const uint8_t* w_data, const uint8_t* w_scale,
                          const bf16_t* bias, void* out, long ldo, const float* gate, void* workspace, long workspace_bytes,
                          int M, int N, int K, int epilogue, hipStream_t st) {
    if (check_out(M, N, K, epilogue, out, ldo, bias, gate, w_data, w_scale)) return 1;
    if (M == 0) return 0;
    OVD_REQUIRE(epilogue != EPI_MX_GELU || !few_rows(M, K), "linear_mxfp4: an MXFP4 output takes a quantised x (ovd_gemm_mxfp4)");
    const int xb = x_is_f32 ? 4 : 2, ob = epilogue <= EPI_BF16_GELU ? 2 : 4;
    if (!few_rows(M, K) || rows_overlap(x, ldx * xb, (long)K * xb, out, ldo * ob, (long)N * ob, M)) {
        const long nd = ovd_impl_mxfp4_data_bytes(M, K), need = nd + ovd_impl_mxfp4_scale_bytes(M, K);
        OVD_REQUIRE(workspace != nullptr && workspace_bytes >= need,
                    "linear_mxfp4: %d rows of %d (or an output that shares memory with x) need %ld bytes of workspace, got %ld", M, K,
                    need, workspace_bytes);
        uint8_t* data = (uint8_t*)workspace;
        if (ovd_impl_mxfp4_quant(x, x_is_f32, ldx, data, data + nd, M, K, st)) return 1;
        return ovd_impl_gemm_mxfp4(data, data + nd, w_data, w_scale, bias, out, ldo, gate, M, N, K, epilogue, M, st);
    }
    OVD_REQUIRE(ldx >= K && ldx % (x_is_f32 ? 4 : 8) == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0,
                "linear_mxfp4: rows must keep 16-byte alignment (ldx=%ld)", ldx);
    const Operand W{w_data, w_scale, N};
    const Out o{bias, out, ldo, gate};
    const int groups = (int)mx_groups(K);
    const size_t lds = (groups * FEW_GRP + 15) / 16 * 16 + FEW_PART;
#define FEW(T, E)                                                                                                    \
    {                                                                                                                \
        static OvdLdsLimit lim;                                                                                      \
        if (!lim.ensure(reinterpret_cast<const void*>(&linear_mxfp4_few_kernel<T, E>), lds))                         \
            OVD_FAIL("linear_mxfp4: cannot reserve %zu bytes of LDS", lds);                                          \
        hipLaunchKernelGGL((linear_mxfp4_few_kernel<T, E>), dim3(ceil_div(N, 32)), dim3(512), lds, st, (const T*)x, ldx, W, o, \
                           M, K, groups);                                                                            \
    }
#define FEW_CASE(E) case E: if (x_is_f32) FEW(float, E) else FEW(bf16_t, E) break;
    switch (epilogue) { FEW_CASE(EPI_BF16) FEW_CASE(EPI_BF16_GELU) FEW_CASE(EPI_F32) FEW_CASE(EPI_RESID) }
#undef FEW_CASE
#undef FEW
    OVD_CHECK_LAUNCH("linear_mxfp4");
    return 0;
}

int ovd_impl_gemm_mxfp4(const uint8_t* a_data, const uint8_t* a_scale, const uint8_t* w_data, const uint8_t* w_scale,
                        const bf16_t* bias, void* out, long ldo, const float* gate, int M, int N, int K, int epilogue,
                        int order_rows, hipStream_t st) {
    if (check_out(M, N, K, epilogue, out, ldo, bias, gate, w_data, w_scale)) return 1;
    OVD_REQUIRE(order_rows >= 0, "gemm_mxfp4: order_rows=%d is negative", order_rows);
    OVD_REQUIRE(reinterpret_cast<uintptr_t>(a_data) % 16 == 0 && reinterpret_cast<uintptr_t>(a_scale) % 4 == 0,
                "gemm_mxfp4: operands must be 16-byte aligned");
    OVD_REQUIRE(epilogue != EPI_MX_GELU || (out != a_data && out != w_data), "gemm_mxfp4: the output matrix is one of the operands");
    if (M == 0) return 0;
    const Operand A{a_data, a_scale, M}, W{w_data, w_scale, N};
    const Out o{bias, out, ldo, gate};
    const int groups = (int)mx_groups(K);
#define DIRECT(MT, NT, E)                                                                                      \
    {                                                                                                          \
        const size_t lds = 8 * MT * NT * 4 * 64 * sizeof(float4);                                              \
        static OvdLdsLimit lim;                                                                                \
        if (!lim.ensure(reinterpret_cast<const void*>(&gemm_mxfp4_direct_kernel<MT, NT, E>), lds))             \
            OVD_FAIL("gemm_mxfp4: cannot reserve %zu bytes of LDS", lds);                                      \
        const long tm = ceil_div(M, 32 * MT), tn = ceil_div(E == EPI_MX_GELU ? ceil_div(N, KG) * KG : N, 32 * NT); \
        OVD_REQUIRE(tm * tn < (1L << 23), "gemm_mxfp4: grid too large");                                       \
        hipLaunchKernelGGL((gemm_mxfp4_direct_kernel<MT, NT, E>), dim3((unsigned)(tm * tn)), dim3(512),        \
                           lds, st, A, W, o, groups, (unsigned)tm);                                            \
    }
#define BIG(E)                                                                                                 \
    {                                                                                                          \
        static OvdLdsLimit lim;                                                                                \
        if (!lim.ensure(reinterpret_cast<const void*>(&gemm_mxfp4_big_kernel<E>), BIG_LDS))                    \
            OVD_FAIL("gemm_mxfp4: cannot reserve %d bytes of LDS", BIG_LDS);                                   \
        hipLaunchKernelGGL((gemm_mxfp4_big_kernel<E>), dim3(min(tiles_m * tiles_n, cus)), dim3(512), BIG_LDS, st, A, W, o, \
                           groups, tiles_m, tiles_n, 4, wide);                                                 \
    }
    const int tiles_m = ceil_div(M, TM), tiles_n = ceil_div(N, TN);
    const int cus = max(8, ovd_device_cus() / 8 * 8);
    OVD_REQUIRE((long)tiles_m * tiles_n < (1L << 30), "gemm_mxfp4: grid too large");
    // Which kernel, by the time that its rounds of workgroups take, in units of 0.19 us.  Measured over M 9 .. 2000 at
    // (N, K) of (1536, 1536), (8960, 1536), (1536, 8960), (5120, 5120), (13824, 5120), (5120, 13824), three operand sets in
    // turn: a round of 256 x 256 tiles 4.5 + 1.2 groups us, one of 64 x 64 tiles 3.1 + 0.19 groups (550 x 1536 x 8960:
    // 12 us against 47; 800 x 8960 x 1536: 31 against 15).  32 x 32 tiles, of which several share a CU, take 0.3 rounds of
    // 64 x 64 ones per tile and CU, and one such time to begin (64 x 1536 x 8960: 5.1 us against 10.2; 550: 15 against 12).
    const int outs = epilogue == EPI_MX_GELU ? ceil_div(N, KG) * KG : N;
    const auto t_small = [&](int rows) { return ceil_div((long)ceil_div(rows, 64) * ceil_div(outs, 64), cus) * (16L + groups); };
    const auto t_tiny = [&](int rows) { return 3 * ((long)ceil_div(rows, 32) * ceil_div(outs, 32) + cus) * (16L + groups) / (10L * cus); };
    // The 256 x 256 tiles add a row's products in another order than the other two, which share theirs: which of the two
    // orders goes by order_rows, so that a caller whose rows come in parts of any size gets the same bits for each
    const int as = order_rows > 0 ? order_rows : M;
    const long t_big = ceil_div((long)ceil_div(as, TM) * tiles_n, cus) * (23L + 6 * groups);
    const bool big = groups >= 2 && t_big < min(t_small(as), t_tiny(as));
    const int wide = (ldo % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0) ? 1 : 0;
#define GEMM_CASE(E) case E: if (big) BIG(E) else if (t_tiny(M) < t_small(M)) DIRECT(1, 1, E) else DIRECT(2, 2, E) break;
    switch (epilogue) { GEMM_CASE(EPI_BF16) GEMM_CASE(EPI_BF16_GELU) GEMM_CASE(EPI_F32) GEMM_CASE(EPI_RESID) GEMM_CASE(EPI_MX_GELU) }
#undef GEMM_CASE
#undef BIG
#undef DIRECT
    OVD_CHECK_LAUNCH("gemm_mxfp4");
    return 0;
}
