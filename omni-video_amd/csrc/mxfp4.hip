// MXFP4 (OCP microscaling, E2M1 elements, one E8M0 scale per 32 values of a row): quantisation of row matrices and
// the product of two of them, out = epilogue(A[M,K] * W[N,K]^T + bias[N]), on v_mfma_scale_f32_32x32x64_f8f6f4 with
// fp4 operands.  A reduced-precision form of the linear layers beside the e4m3 one of fp8.hip (the reference runs
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

enum Epi { EPI_BF16 = 0, EPI_BF16_GELU = 1, EPI_F32 = 2, EPI_RESID = 3 };

constexpr int KG = 256;                 // k-group: four MFMA k-steps, one scale dword per lane
constexpr int FRAG = 1024;              // bytes of a 32-row x 64-k fragment
constexpr int GRP_DATA = 4 * FRAG;      // bytes of a 32-row x 256-k group
constexpr int GRP_SCALE = 256;          // bytes of its scales

// scale byte of a block from the bits of its largest magnitude
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;                   // biased exponent; 255: infinity or NaN
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 2^(127 - s) as a float (s <= 252; 255 never reaches a finite value, its codes do not matter)
__device__ __forceinline__ float inv_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }
// 2^(s - 127); s = 0 is the denormal 2^-127, s = 255 a NaN
__device__ __forceinline__ float scale_value(uint32_t s) {
    return __uint_as_float(s == 0u ? 0x00400000u : (s == 255u ? 0x7FC00000u : s << 23));
}

// eight floats (already divided by their scale) -> eight codes, k ascending from the low nibble
__device__ __forceinline__ uint32_t pack_fp4x8(const float (&v)[8]) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.0f, 3);
    return w;
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// ------------------------------------------------------------------------------------------ quantise / dequantise
// One wave = one row block x one k-group.  A load instruction covers 8 rows x 64 k (8 lanes of 8 values per row: whole
// 128-byte lines of bf16), a store instruction two runs of 8 rows x 16 bytes; the four lanes of an MX block exchange
// their largest magnitude.  HBM-bound: 2 (4) bytes read and 17/32 written per value.
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
                                                          uint8_t* __restrict__ scale, int M, int K, int groups, long waves) {
    const int lane = threadIdx.x & 63;
    const long wid = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (wid >= waves) return;
    const long rb = wid / groups;
    const int kg = (int)(wid % groups);
    const int r8 = lane >> 3, c = lane & 7;               // row inside the 8-row group, 8-value chunk of the 64-k step
    uint8_t* dst = data + wid * GRP_DATA + (c >> 2) * 512 + (c & 3) * 4;
    uint32_t* sdst = reinterpret_cast<uint32_t*>(scale + wid * GRP_SCALE) + (c >> 2) * 32;
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
        const int r = rg * 8 + r8;
        const long row = rb * 32 + r;
        if (row >= M) break;
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
            const float inv = inv_scale(s);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[ks][j] *= inv;
            *reinterpret_cast<uint32_t*>(dst + ks * FRAG + r * 16) = pack_fp4x8(v[ks]);
            sc |= s << (8 * ks);
        }
        if ((c & 3) == 0) sdst[r] = sc;
    }
}

// the mapping above, the other way; a value is code * 2^(s - 127), exact in bf16 and fp32
template <typename T>
__global__ void __launch_bounds__(256) mxfp4_dequant_kernel(const uint8_t* __restrict__ data,
                                                            const uint8_t* __restrict__ scale, T* __restrict__ out,
                                                            long ldo, int M, int K, int groups, long waves) {
    const int lane = threadIdx.x & 63;
    const long wid = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (wid >= waves) return;
    const long rb = wid / groups;
    const int kg = (int)(wid % groups);
    const int r8 = lane >> 3, c = lane & 7;
    const uint8_t* src = data + wid * GRP_DATA + (c >> 2) * 512 + (c & 3) * 4;
    const uint32_t* ssrc = reinterpret_cast<const uint32_t*>(scale + wid * GRP_SCALE) + (c >> 2) * 32;
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
        const int r = rg * 8 + r8;
        const long row = rb * 32 + r;
        if (row >= M) break;
        const uint32_t sc = ssrc[r];
        T* dst = out + row * ldo + (long)kg * KG + c * 8;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(src + ks * FRAG + r * 16);
            const float s = scale_value((sc >> (8 * ks)) & 255u);
            const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0) * s;
            const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1) * s;
            const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2) * s;
            const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3) * s;
            if (kg * KG + ks * 64 + c * 8 >= K) continue;
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<uint4*>(dst + ks * 64) =
                    make_uint4(pack_bf2(p0[0], p0[1]), pack_bf2(p1[0], p1[1]), pack_bf2(p2[0], p2[1]), pack_bf2(p3[0], p3[1]));
            } else {
                reinterpret_cast<float4*>(dst + ks * 64)[0] = make_float4(p0[0], p0[1], p1[0], p1[1]);
                reinterpret_cast<float4*>(dst + ks * 64)[1] = make_float4(p2[0], p2[1], p3[0], p3[1]);
            }
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

// four consecutive columns n .. n + 3 (n % 4 == 0, n < N) of row m; the pre-activation stays in fp32: the only
// rounding is that of the stored value
template <int EPI>
__device__ __forceinline__ void store4(const Out& o, long m, int n, float (&y)[4]) {
    if (o.bias) {
        const uint2 b = *reinterpret_cast<const uint2*>(o.bias + n);
        y[0] += bf2f(b.x & 0xffff);
        y[1] += bf2f(b.x >> 16);
        y[2] += bf2f(b.y & 0xffff);
        y[3] += bf2f(b.y >> 16);
    }
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

// Few rows: a workgroup of 8 waves owns MT x NT blocks of 32 x 32 outputs, its waves take the k-groups in turn,
// fragments straight from memory (they are in lane order there) one group ahead, and the eight partial sums meet in
// LDS in a fixed order.  Weight rows sit on the MFMA's M axis, so a lane ends with 4 consecutive columns of one row.
template <int MT, int NT, int EPI>
__global__ void __launch_bounds__(512) gemm_mxfp4_direct_kernel(Operand A, Operand W, Out o, int groups) {
    extern __shared__ float4 part[];          // [8 waves][MT * NT * 4 register quads][64 lanes]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long rb0 = (long)blockIdx.y * MT, nb0 = (long)blockIdx.x * NT;
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
        if (m < A.rows && n < W.rows) store4<EPI>(o, m, n, y);
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
    const long waves = (long)ceil_div(M, 32) * groups;
    OVD_REQUIRE((waves + 3) / 4 < (1L << 31), "mxfp4_quant: grid too large");
    const dim3 grid((unsigned)((waves + 3) / 4)), blk(256);
    if (x_is_f32)
        hipLaunchKernelGGL(mxfp4_quant_kernel<float>, grid, blk, 0, st, (const float*)x, ldx, data, scale, M, K, groups, waves);
    else
        hipLaunchKernelGGL(mxfp4_quant_kernel<bf16_t>, grid, blk, 0, st, (const bf16_t*)x, ldx, data, scale, M, K, groups, waves);
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
    const long waves = (long)ceil_div(M, 32) * groups;
    OVD_REQUIRE((waves + 3) / 4 < (1L << 31), "mxfp4_dequant: grid too large");
    const dim3 grid((unsigned)((waves + 3) / 4)), blk(256);
    if (out_is_f32)
        hipLaunchKernelGGL(mxfp4_dequant_kernel<float>, grid, blk, 0, st, data, scale, (float*)out, ldo, M, K, groups, waves);
    else
        hipLaunchKernelGGL(mxfp4_dequant_kernel<bf16_t>, grid, blk, 0, st, data, scale, (bf16_t*)out, ldo, M, K, groups, waves);
    OVD_CHECK_LAUNCH("mxfp4_dequant");
    return 0;
}

int ovd_impl_gemm_mxfp4(const uint8_t* a_data, const uint8_t* a_scale, const uint8_t* w_data, const uint8_t* w_scale,
                        const bf16_t* bias, void* out, long ldo, const float* gate, int M, int N, int K, int epilogue,
                        hipStream_t st) {
    OVD_REQUIRE(M >= 0 && N > 0 && N % 4 == 0 && K > 0 && K % 32 == 0,
                "gemm_mxfp4: M=%d N=%d K=%d not supported: N %% 4, K %% 32", M, N, K);
    OVD_REQUIRE(epilogue >= EPI_BF16 && epilogue <= EPI_RESID, "gemm_mxfp4: unknown epilogue %d", epilogue);
    OVD_REQUIRE(gate == nullptr || epilogue == EPI_RESID, "gemm_mxfp4: a gate goes with the residual epilogue");
    OVD_REQUIRE(ldo >= N && ldo % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (epilogue <= EPI_BF16_GELU ? 8 : 16) == 0 &&
                    reinterpret_cast<uintptr_t>(bias) % 8 == 0 && reinterpret_cast<uintptr_t>(gate) % 16 == 0,
                "gemm_mxfp4: out rows, bias and gate must be aligned to 4 values (ldo=%ld)", ldo);
    OVD_REQUIRE(reinterpret_cast<uintptr_t>(a_data) % 16 == 0 && reinterpret_cast<uintptr_t>(w_data) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(a_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(w_scale) % 4 == 0,
                "gemm_mxfp4: operands must be 16-byte aligned");
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
        const int ty = ceil_div(M, 32 * MT);                                                                   \
        OVD_REQUIRE(ty <= 65535, "gemm_mxfp4: grid too large");                                                \
        hipLaunchKernelGGL((gemm_mxfp4_direct_kernel<MT, NT, E>), dim3(ceil_div(N, 32 * NT), ty), dim3(512),   \
                           lds, st, A, W, o, groups);                                                          \
    }
#define GEMM_CASE(E) case E: if (M <= 32) DIRECT(1, 1, E) else DIRECT(2, 2, E) break;
    switch (epilogue) { GEMM_CASE(EPI_BF16) GEMM_CASE(EPI_BF16_GELU) GEMM_CASE(EPI_F32) GEMM_CASE(EPI_RESID) }
#undef GEMM_CASE
#undef DIRECT
    OVD_CHECK_LAUNCH("gemm_mxfp4");
    return 0;
}
