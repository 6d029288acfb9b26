// Attention over packed documents, forward: bf16 operands, fp32 softmax and accumulation.  The probabilities are rounded to
// bf16 for the second product (a matrix instruction takes both operands so; their sum is that of the unrounded ones): 2^-9 of
// each, independently.  Outputs are 2.3e-3 off in relative L2, where fp32 probabilities and one rounding would leave 1.7e-3.
//
// Tokens of several documents (videos, images, prompts of different sizes) lie one after another in q [Tq, Nq, D] and
// k, v [Tk, Nkv, D]; document d owns query rows [cu_q[d], cu_q[d+1]) and key rows [cu_k[d], cu_k[d+1]).  Query i of a
// document sees its first
//     n(i) = Lk                                          (no causal mask)
//     n(i) = clamp(max(i + Lk - Lq + 1, prefix[d]), 0, Lk)   (causal, aligned at the end; a prefix that all may see)
// keys: document, causal and prefix masks are all ONE number per query row.  s = scale q.k, optionally capped,
// s -> cap tanh(s / cap); o = softmax(s) v, and 0 for a row that sees no key.  Query head h reads key head h / (Nq/Nkv).
// The equal-length, unmasked form is attn.hip; reference: the flash_attn_varlen_func call of
// omnivideo/modules/attention.py:96-130 (which packs a padded batch with cu_seqlens).
//
// Work split: the query rows of one document that share a key head, (token, head in group) pairs, are one list of
// Lq * group rows; a workgroup of NW waves takes 32 NW of them, 32 per wave, so a single token's group of heads fills a
// tile together and K / V are read once per group.  Which document a workgroup serves follows from cu_q on the device
// (a wave-wide scan), so lengths can change under a captured graph; the grid is the largest that the shapes allow.
// Few rows: the keys of long documents are split into parts and a second kernel joins them.
//
// S^T = K Q^T with the key on the MFMA row axis (v_mfma_f32_32x32x16_bf16): a lane holds 32 scores of ONE query, so row
// maxima and sums are in-lane plus one exchange, and P is already the B operand of O^T += V^T P^T.  V^T fragments come
// from the row-major V tile through ds_read_b64_tr_b16; K and V tiles of 64 keys stream HBM -> LDS by DMA with the
// bank swizzle applied to the source chunk.  Key rows past the document are clamped to its last row: what lies behind
// a document is never read, and a masked score is -inf whatever it was.
//
// What bounds it.  D = 128, long documents: the matrix pipe and the chip's power (20280, 1560, 14040 and 3600 tokens, 40
// heads: 10.7 ms = 1190 TFLOP/s; one document of 20280 as fast as attn.hip).  16x16x32 instructions instead of 32x32x16 would
// take 12 % less power a product, but twice as many of them and the two queries that a lane then serves cost issue slots: 3 %
// slower (one document), 5 to 20 % (short ones).  D = 64: vector instructions (197 a tile and
// wave beside 16 matrix ones: 970 TFLOP/s), the more so with a cap (two more transcendental instructions a score: 500).  Few
// tokens: bytes of K and V (8 tokens against 80750 keys, 8 key heads: 73 us with the join = 4.5 TB/s).  Prompts of
// some hundred tokens: the start and the last, partly filled round (8 of them, 16 heads of 64, a prefix: 44 us, 59 capped).
// The four-wave form with split keys spills about 70 registers at D = 128 and reloads some of them in every step (700 and 300
// queries against 700 and 9000 keys: 59 us before the join, 330 TFLOP/s); no other form spills.
#include "common.h"

namespace {

constexpr int BKV = 64;                       // keys per tile
constexpr float NEG_INF = -__builtin_inff();
constexpr float RESCALE_THR = 6.0f;

typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4_t;
typedef __attribute__((address_space(3))) bf16x4_t* lds_b4_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

// byte offset of 16-byte chunk c of row r of a K (V) tile: rows of 256 (D = 128) or 128 (D = 64) bytes, swizzled so that
// the b128 row reads of K and the transposed b64 reads of V spread over all banks
template <int D>
__device__ __forceinline__ int k_off(int r, int c) {
    return D == 128 ? r * 256 + ((c ^ (r & 15)) << 4) : r * 128 + ((c ^ ((r >> 1) & 7)) << 4);
}
template <int D>
__device__ __forceinline__ int v_off(int r, int c) {
    return D == 128 ? r * 256 + ((c ^ ((r & 3) << 2)) << 4) : r * 128 + ((c ^ (((r >> 1) & 1) << 2)) << 4);
}

__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

struct Args {
    const bf16_t *q, *k, *v;
    bf16_t* o;
    long q_ld, k_ld, v_ld, o_ld;              // elements between tokens
    const int *cu_q, *cu_k, *prefix;          // [docs + 1], [docs + 1], [docs] or null
    int total_q, total_k, docs, kv_heads, group, causal;
    float scale_log2;                         // softmax scale * log2(e)
    float cap_in, cap_out;                    // 2 scale log2(e) / cap, cap log2(e)  (capped form)
    float cap_x;                              // scale / cap
    int row_blocks, stripes;
    int chunk, max_splits;                    // split form: key tiles a work item should have, most parts of a document
    float* ws;                                // partial results of the parts
};

// rows [*q0, *q0 + *lq) and keys [*k0, *k0 + *lk) of document d; whatever cu_q / cu_k hold, inside the tensors
__device__ __forceinline__ void doc_range(const Args& a, int d, int& q0, int& lq, int& k0, int& lk) {
    q0 = min(max(a.cu_q[d], 0), a.total_q);
    lq = min(max(a.cu_q[d + 1], q0), a.total_q) - q0;
    k0 = min(max(a.cu_k[d], 0), a.total_k);
    lk = min(max(a.cu_k[d + 1], k0), a.total_k) - k0;
}

// parts into which the keys of a document of lk keys are split
__device__ __forceinline__ int parts_of(const Args& a, int lk) {
    const int nt = (lk + BKV - 1) / BKV;
    return min(max((nt + a.chunk - 1) / a.chunk, 1), a.max_splits);
}

// document, row block (of ROWS rows) and part of its keys of work item `blk`; false past the last one.  Up to SORTED
// documents are walked from the longest keys to the shortest, so that the last workgroups to start are short ones (packed
// prompts of 1 to 2100 tokens, 4 key heads, with eight-wave workgroups: 92 us in the order given, 77 sorted); more are taken in their order.
constexpr int SORTED = 32;

template <int ROWS, bool SPLIT>
__device__ __forceinline__ bool find_block(const Args& a, int blk, int lane, int& doc, int& rb, int& part, int& parts) {
    for (int d0 = 0; d0 < a.docs; d0 += 64) {
        const int d = d0 + lane;
        int n = 0, np = 1, keys = -1;
        if (d < a.docs) {
            int q0, lq, k0, lk;
            doc_range(a, d, q0, lq, k0, lk);
            keys = lk;
            n = (int)(((unsigned)(lq * a.group) + ROWS - 1) / ROWS);
            if (SPLIT) {
                np = parts_of(a, lk);
                n *= np;
            }
        }
        int before = 0, sum;                              // items of the documents that come before this lane's
        if (!SPLIT && a.docs <= SORTED) {
            sum = 1 << 30;                                // (one pass holds them all)
            for (int j = 0; j < a.docs; ++j) {
                const int nj = __builtin_amdgcn_readlane(n, j), kj = __builtin_amdgcn_readlane(keys, j);
                if (kj > keys || (kj == keys && j < lane)) before += nj;
            }
        } else {
            int incl = n;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const int up = __shfl_up(incl, s, 64);
                if (lane >= s) incl += up;
            }
            before = incl - n;
            sum = __shfl(incl, 63, 64);
        }
        const unsigned long long hit = __ballot(blk >= before && blk < before + n);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            doc = d0 + l;
            rb = blk - __shfl(before, l, 64);
            if (a.causal && !SPLIT) rb = __shfl(n, l, 64) - 1 - rb;          // the longest rows first
            part = 0;
            parts = 1;
            if (SPLIT) {
                parts = __shfl(np, l, 64);
                part = rb % parts;
                rb /= parts;
            }
            return true;
        }
        blk -= sum;
    }
    return false;
}

__device__ __forceinline__ int visible(const Args& a, int i, int lq, int lk, int prefix) {
    if (!a.causal) return lk;
    const int n = max(i + lk - lq + 1, prefix);
    return min(max(n, 0), lk);
}

// workspace: accumulators [max_splits][rows = total_q * Nq][D], then (maximum, sum) [max_splits][rows][2]
template <int D>
__device__ __forceinline__ float* ws_row(const Args& a, int part, long row) {
    const long rows = (long)a.total_q * a.kv_heads * a.group;
    return a.ws + (part * rows + row) * D;
}
template <int D>
__device__ __forceinline__ float* ws_stat(const Args& a, int part, long row) {
    const long rows = (long)a.total_q * a.kv_heads * a.group;
    return a.ws + a.max_splits * rows * D + (part * rows + row) * 2;
}

// 16 bytes a lane from `base + off` to 1 KiB of LDS.  As assembly because the compiler would wait for every DMA in flight ahead
// of the next transposed read of LDS, whatever either touches: half a step after their start (documents of 700 and 300 queries
// against 700 and 9000 keys 100 us against 70; 20280 and 14040 against 131 and 550 keys 109 against 101; one long document 0 to 1 %).
// The waits stand at the ends of the steps, before the barrier that precedes the reads.
// s_nop: m0 may be used one wait state after its write, an SGPR that a vector instruction wrote (the compiler spills to lanes
// of vector registers and does not see the load in here) five.
__device__ __forceinline__ void dma_1k(const char* base, unsigned off, char* dst) {
    const unsigned m0 = __builtin_amdgcn_readfirstlane((unsigned)reinterpret_cast<uintptr_t>((lds_ptr)dst));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m0), "v"(off), "s"(base) : "m0", "memory");
}
// the same twice, STEP bytes of LDS apart, with one such wait
template <int STEP>
__device__ __forceinline__ void dma_2k(const char* base, unsigned off0, unsigned off1, char* dst) {
    const unsigned m0 = __builtin_amdgcn_readfirstlane((unsigned)reinterpret_cast<uintptr_t>((lds_ptr)dst));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_add_u32 m0, m0, %4\n\ts_nop 0\n\t"
                 "global_load_lds_dwordx4 %2, %3" ::"s"(m0), "v"(off0), "v"(off1), "s"(base), "n"(STEP) : "m0", "scc", "memory");
}

// DMA of one operand: 64-row tiles HBM -> LDS.  A wave's instruction covers RPI rows; rows past the document's last key
// repeat it.  Tile bases advance in 64 bits, offsets inside a tile are 32 bits.
template <int D, int NW, bool IS_K>
struct Stream {
    static constexpr int CPR = D / 8, RPI = 64 / CPR, N = BKV / RPI / NW;
    const char* base;        // first key row of the document, this head
    long ld2;                // bytes between rows
    int lk;                  // keys of the document
    unsigned off[NW == 1 ? 1 : N];       // this lane's offsets in a whole tile
    __device__ __forceinline__ unsigned offset(int i, int lim, int wave, int lane) const {
        const int r = (i * NW + wave) * RPI + lane / CPR, c = lane % CPR;
        const int cs = IS_K ? (D == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7)) : (D == 128 ? c ^ ((r & 3) << 2) : c ^ (((r >> 1) & 1) << 2));
        return (unsigned)min(r, lim) * (unsigned)ld2 + (unsigned)cs * 16u;
    }
    __device__ __forceinline__ void init(const bf16_t* first, long ld, int keys, int wave, int lane) {
        base = reinterpret_cast<const char*>(first);
        ld2 = ld * 2;
        lk = keys;
        if constexpr (NW > 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) off[i] = offset(i, BKV, wave, lane);
        }
    }
    __device__ __forceinline__ void stage(int t, char* dst, int wave, int lane) const {
        const char* tb = base + (long)t * BKV * ld2;
        const int lim = lk - 1 - t * BKV;
        const bool whole = NW > 1 && lim >= BKV - 1;
        if constexpr (N == 1) {
            dma_1k(tb, whole ? off[0] : offset(0, lim, wave, lane), dst + wave * 1024);
        } else if (whole) {
#pragma unroll
            for (int i = 0; i < N; i += 2)
                dma_2k<NW * 1024>(tb, off[NW > 1 ? i : 0], off[NW > 1 ? i + 1 : 0], dst + (i * NW + wave) * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2)
                dma_2k<NW * 1024>(tb, offset(i, lim, wave, lane), offset(i + 1, lim, wave, lane), dst + (i * NW + wave) * 1024);
        }
    }
};

__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_fmaxf(__builtin_fmaxf(a, b), c); }

template <int D>
__device__ __forceinline__ bf16x8 read_v(const char* sv, int st, int db, int lane) {
    const int g = lane >> 4, i16 = lane & 15, qd = i16 >> 2, pp = i16 & 3;
    const int kr = 16 * st + 4 * (g >> 1) + qd;
    const int ch = db * 4 + 2 * (g & 1) + (pp >> 1);
    const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4_ptr)(sv + v_off<D>(kr, ch) + 8 * (pp & 1)));
    const bf16x4_t h4 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4_ptr)(sv + v_off<D>(kr + 8, ch) + 8 * (pp & 1)));
    const uint2 lo2 = __builtin_bit_cast(uint2, lo), hi2 = __builtin_bit_cast(uint2, h4);
    return __builtin_bit_cast(bf16x8, make_uint4(lo2.x, lo2.y, hi2.x, hi2.y));
}

// a capped score in units of log2, minus `minus`: cap log2(e) tanh(x), x = s scale / cap, tanh(x) = 1 - 2 / (1 + e^2x) (both
// ends saturate without overflow).  The difference cancels for small x: a score is off by up to 2^-21 of the cap, whatever
// the score.  That is 1.2e-4 at SMALL_CAP, next to nothing beside the bf16 rounding of the probabilities; above it (LARGE)
// scores below a quarter of the cap take the odd series instead, s (1 - x^2 / 3 + 2 x^4 / 15 - 17 x^6 / 315), cut off below
// 2^-21 of the score, and what is left of the form above is below 2^-18 of the score.  As its own instantiations, because
// the series costs what it does not bring to small caps (packed prompts 80 us against 62; causal, 20280 tokens, 12 heads 1759 against 1475).
constexpr float SMALL_CAP = 256.f;

template <bool LARGE>
__device__ __forceinline__ float capped(float s, const Args& a, float minus) {
    const float far = __builtin_fmaf(-2.f * a.cap_out, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * a.cap_in)), a.cap_out - minus);
    if (!LARGE) return far;
    const float x = s * a.cap_x, x2 = x * x;
    const float p = __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
    return __builtin_fabsf(x) < 0.25f ? __builtin_fmaf(s * a.scale_log2, p, -minus) : far;
}
template <bool LARGE>
__device__ __forceinline__ void cap_scores(f32x16& s, const Args& a) {
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = capped<LARGE>(s[j], a, 0.f);
}

__device__ __forceinline__ void mask_scores(f32x16& s0, f32x16& s1, int key0, int nvis, int hi) {
    const int left = nvis - key0 - 4 * hi;              // this lane's keys sit at (r & 3) + 8 (r >> 2) (+ 32)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int at = (r & 3) + 8 * (r >> 2);
        if (at >= left) s0[r] = NEG_INF;
        if (at + 32 >= left) s1[r] = NEG_INF;
    }
}

// ---- values that are infinite or NaN under a mask.  A hidden key's probability is 0, but 0 x inf in the matrix product
// is NaN in every row of the tile.  Tiles that are masked somewhere are therefore looked through (largest magnitude bits
// of the tile); a work item that met such a value is computed again, tile by tile, as the product over the finite
// values, then +-inf (NaN: both) wherever a key with a probability above 0 holds one, found by two products with 0 / 1
// matrices.
template <int D>
__device__ __forceinline__ bool tile_not_finite(const char* sv, int lane) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
    u16x2 mx = {0, 0};
#pragma unroll
    for (int i = 0; i < D * BKV * 2 / 1024; ++i) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(sv + i * 1024 + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = __builtin_elementwise_max(mx, __builtin_bit_cast(u16x2, w[j] & 0x7fff7fffu));
    }
    return __any(mx[0] >= 0x7f80 || mx[1] >= 0x7f80);
}

template <int D, int NW, bool CAP, bool LARGE>
__device__ __forceinline__ void careful_step(f32x16 (&o_acc)[D / 32], const bf16x8 (&qf)[D / 16], float& m_c, float& l_run,
                                             char* smem, const Stream<D, NW, true>& kst, const Stream<D, NW, false>& vst, int t,
                                             int nvis, const Args& a, int wave, int lane) {
    constexpr int TILE = BKV * D * 2;
    asm volatile("" : "+v"(lane));      // addresses are derived here again instead of kept in registers all along
    const int l31 = lane & 31, hi = lane >> 5;
    kst.stage(t, smem, wave, lane);
    vst.stage(t, smem + 2 * TILE, wave, lane);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const char* sv = smem + 2 * TILE;
    f32x16 s0, s1;
#pragma unroll
    for (int j = 0; j < 16; ++j) s0[j] = s1[j] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        const bf16x8 kf0 = *reinterpret_cast<const bf16x8*>(smem + k_off<D>(l31, 2 * ks + hi));
        const bf16x8 kf1 = *reinterpret_cast<const bf16x8*>(smem + k_off<D>(32 + l31, 2 * ks + hi));
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf0, qf[ks], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf1, qf[ks], s1, 0, 0, 0);
    }
    if (CAP) {
        cap_scores<LARGE>(s0, a);
        cap_scores<LARGE>(s1, a);
    }
    mask_scores(s0, s1, t * BKV, nvis, hi);
    const float sc = CAP ? 1.f : a.scale_log2;
    float mx = -3.0e38f;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = max3(mx, s0[r], s1[r]);
    const float m_new = __builtin_fmaxf(m_c, half_max(mx) * sc);
    const float alpha = __builtin_amdgcn_exp2f(m_c - m_new);
    m_c = m_new;
    float sum = 0.f;
    uint32_t pw[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const f32x16& c = i < 8 ? s0 : s1;
        const float pa = __builtin_amdgcn_exp2f(__builtin_fmaf(c[(i & 7) * 2], sc, -m_c));
        const float pb = __builtin_amdgcn_exp2f(__builtin_fmaf(c[(i & 7) * 2 + 1], sc, -m_c));
        sum += pa + pb;
        pw[i] = pack_bf2(pa, pb);
    }
    l_run = l_run * alpha + sum;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
        f32x16 pos, neg;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            pos[j] = neg[j] = 0.f;
            o_acc[db][j] *= alpha;
        }
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            const bf16x8 pf = __builtin_bit_cast(bf16x8, make_uint4(pw[4 * st], pw[4 * st + 1], pw[4 * st + 2], pw[4 * st + 3]));
            const bf16x8 v = read_v<D>(sv, st, db, lane);
            bf16x8 fin, vp, vn;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned u = (unsigned short)v[e];
                const bool bad = (u & 0x7f80u) == 0x7f80u, nan = bad && (u & 0x7fu);
                fin[e] = bad ? (short)0 : v[e];
                vp[e] = (nan || u == 0x7f80u) ? (short)0x3f80 : (short)0;
                vn[e] = (nan || u == 0xff80u) ? (short)0x3f80 : (short)0;
            }
            o_acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fin, pf, o_acc[db], 0, 0, 0);
            pos = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vp, pf, pos, 0, 0, 0);
            neg = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vn, pf, neg, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (pos[j] > 0.f) o_acc[db][j] += __builtin_inff();
            if (neg[j] > 0.f) o_acc[db][j] -= __builtin_inff();
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();          // every wave is done with the tiles
}

// Step t of a wave: the exponentials, sum and P V of tile t (scores c0 / c1, already computed) while the matrix pipe
// forms S^T of tile t + 1 in n0 / n1.  K of tile t + 2 and V of tile t + 1 are put in flight from inside.
// The running maximum m_c is raised only when a tile exceeds it by RESCALE_THR (log2 units): probabilities stay below
// 2^THR, which costs no relative precision, and most tiles skip the rescale of O.
// RAW (capped form): tile t's scores are not capped yet.  The cap is monotonic, so the running maximum needs it for one
// value of a row, and the rest pass through it between this step's products, on their way into the exponential (packed
// prompts with a cap 62 us; as a pass of its own between the two products 66 us).  Masked scores must not pass through it:
// such tiles are capped first, then masked.
template <int D, int NW, bool CAP, bool LARGE, bool HAS_NEXT, bool MASK_NEXT, bool RAW>
__device__ __forceinline__ void pipe_step(f32x16 (&o_acc)[D / 32], const bf16x8 (&qf)[D / 16], float& m_c, float& l_run,
                                          const f32x16& c0, const f32x16& c1, f32x16& n0, f32x16& n1, float& mx, bool& need,
                                          const char* sk_next, const char* sv_cur, const Stream<D, NW, true>& kst, char* k_dst,
                                          bool more_k, const Stream<D, NW, false>& vst, char* v_dst, bool more_v, int t,
                                          int nvis, bool masked_cur, bool& redo, const Args& a, int wave,
                                          int lane) {
    constexpr int DB = D / 32, KS = D / 16;
    const int l31 = lane & 31, hi = lane >> 5;
    if (need) {
        const float m_new = __builtin_fmaxf(m_c, mx);
        const float alpha = __builtin_amdgcn_exp2f(m_c - m_new);
        m_c = m_new;
        l_run *= alpha;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o_acc[i][j] *= alpha;
    }
    if (HAS_NEXT) {
#pragma unroll
        for (int j = 0; j < 16; ++j) n0[j] = n1[j] = 0.f;
    }
    const float sc = CAP ? 1.f : a.scale_log2;
    float rs0 = 0.f, rs1 = 0.f;
    uint32_t pw[16];
#define EXPONENT(x) (RAW ? capped<LARGE>(x, a, m_c) : CAP ? (x) - m_c : __builtin_fmaf(x, sc, -m_c))
#define SOFTMAX_PAIR(i)                                                                                    \
    do {                                                                                                   \
        const f32x16& c_ = (i) < 8 ? c0 : c1;                                                              \
        const int r_ = ((i) & 7) * 2;                                                                      \
        const float pa_ = __builtin_amdgcn_exp2f(EXPONENT(c_[r_]));                                        \
        const float pb_ = __builtin_amdgcn_exp2f(EXPONENT(c_[r_ + 1]));                                    \
        rs0 += pa_;                                                                                        \
        rs1 += pb_;                                                                                        \
        pw[i] = pack_bf2(pa_, pb_);                                                                        \
        asm volatile("" : "+v"(pw[i]), "+v"(rs0), "+v"(rs1));                                              \
    } while (0)
    bf16x8 kf[2][2], vf[2][DB];
    if (HAS_NEXT) {
        kf[0][0] = *reinterpret_cast<const bf16x8*>(sk_next + k_off<D>(l31, hi));
        kf[0][1] = *reinterpret_cast<const bf16x8*>(sk_next + k_off<D>(32 + l31, hi));
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        if (HAS_NEXT) {
            if (ks < KS - 1) {
                kf[(ks + 1) & 1][0] = *reinterpret_cast<const bf16x8*>(sk_next + k_off<D>(l31, 2 * ks + 2 + hi));
                kf[(ks + 1) & 1][1] = *reinterpret_cast<const bf16x8*>(sk_next + k_off<D>(32 + l31, 2 * ks + 2 + hi));
            }
            n0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks & 1][0], qf[ks], n0, 0, 0, 0);
            n1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks & 1][1], qf[ks], n1, 0, 0, 0);
        }
        if constexpr (D == 128) {
            SOFTMAX_PAIR(ks);
        } else {
            SOFTMAX_PAIR(2 * ks);
            SOFTMAX_PAIR(2 * ks + 1);
        }
        if (ks == 0 && more_k) kst.stage(t + 2, k_dst, wave, lane);
        if (ks == 1 && more_v) vst.stage(t + 1, v_dst, wave, lane);
        if (ks == KS - 1) {
#pragma unroll
            for (int db = 0; db < DB; ++db) vf[0][db] = read_v<D>(sv_cur, 0, db, lane);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if (HAS_NEXT && MASK_NEXT && CAP) {
        cap_scores<LARGE>(n0, a);
        cap_scores<LARGE>(n1, a);
    }
    if (HAS_NEXT && MASK_NEXT) mask_scores(n0, n1, (t + 1) * BKV, nvis, hi);
    float nmx = -3.0e38f;
    if ((MASK_NEXT || !HAS_NEXT) && masked_cur) redo |= tile_not_finite<D>(sv_cur, lane);
#pragma unroll
    for (int st = 0; st < 4; ++st) {
        if (st < 3) {
#pragma unroll
            for (int db = 0; db < DB; ++db) vf[(st + 1) & 1][db] = read_v<D>(sv_cur, st + 1, db, lane);
        }
        const bf16x8 pfrag =
            __builtin_bit_cast(bf16x8, make_uint4(pw[4 * st], pw[4 * st + 1], pw[4 * st + 2], pw[4 * st + 3]));
#pragma unroll
        for (int db = 0; db < DB; ++db)
            o_acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[st & 1][db], pfrag, o_acc[db], 0, 0, 0);
        if (st == 0) { SOFTMAX_PAIR(8); SOFTMAX_PAIR(9); SOFTMAX_PAIR(10); }
        if (st == 1) { SOFTMAX_PAIR(11); SOFTMAX_PAIR(12); SOFTMAX_PAIR(13); }
        if (st == 2) { SOFTMAX_PAIR(14); SOFTMAX_PAIR(15); }
        if (st >= 2 && HAS_NEXT) {
            const f32x16& n = st == 2 ? n0 : n1;
#pragma unroll
            for (int r = 0; r < 16; r += 2) nmx = max3(nmx, n[r], n[r + 1]);
            asm volatile("" : "+v"(nmx));
            if (st == 3) {
                mx = CAP ? (MASK_NEXT ? half_max(nmx) : capped<LARGE>(half_max(nmx), a, 0.f)) : half_max(nmx) * a.scale_log2;
                need = __any(mx > m_c + RESCALE_THR);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    l_run += rs0 + rs1;
#undef SOFTMAX_PAIR
#undef EXPONENT
}

// one work item: 32 NW rows of document `doc` under key head kvh, part `part` of `parts` of their keys
template <int D, int NW, bool CAP, bool LARGE, bool SPLIT>
__device__ __forceinline__ void attend(const Args& a, char* smem, int kvh, int doc, int rb, int part, int parts) {
    constexpr int ROWB = D * 2;                          // bytes per K / V row
    constexpr int TILE = BKV * ROWB;                     // bytes per tile; LDS: K[2] | V[2]
    constexpr int CPR = ROWB / 16;                       // chunks per row
    constexpr int RPI = 64 / CPR;                        // rows per DMA instruction of a wave
    constexpr int DB = D / 32, KS = D / 16;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    int q0, lq, k0, lk;
    doc_range(a, doc, q0, lq, k0, lk);
    const int prefix = a.prefix ? min(max(a.prefix[doc], 0), lk) : 0;
    const unsigned group = (unsigned)a.group;
    const int rows = lq * a.group;                       // below 2^31 (checked on the host)
    const int r_first = rb * (32 * NW) + wave * 32;
    const unsigned row = (unsigned)min(r_first + l31, rows - 1);       // rows past the last repeat it and are not stored
    const int tok = (int)(row / group), head = kvh * a.group + (int)(row % group);
    const int nvis = visible(a, tok, lq, lk, prefix);
    // visible counts grow with the row: the tile range follows from the workgroup's last row; a wave's own last row says
    // where its work ends, its first row which tiles need no mask
    const unsigned last_row = (unsigned)min(rb * (32 * NW) + 32 * NW - 1, rows - 1);
    const int kend = __builtin_amdgcn_readfirstlane(visible(a, (int)(last_row / group), lq, lk, prefix));
    const int wend = __builtin_amdgcn_readfirstlane(visible(a, (int)((unsigned)min(r_first + 31, rows - 1) / group), lq, lk, prefix));
    const int full = __builtin_amdgcn_readfirstlane(visible(a, (int)((unsigned)min(r_first, rows - 1) / group), lq, lk, prefix));
    const int nt = (kend + BKV - 1) / BKV;
    const int t0 = (int)((long)nt * part / parts), t1 = (int)((long)nt * (part + 1) / parts);
    const int tw = min(max((wend + BKV - 1) / BKV, t0), t1);     // this wave's tiles: [t0, tw)
    const int tf = min(max(full / BKV, t0), tw);                 // ... of which [t0, tf) are seen whole by all its rows

    bf16x8 qf[KS];
    {
        const bf16_t* qp = a.q + (long)(q0 + tok) * a.q_ld + (long)head * D + 8 * hi;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
    }
    Stream<D, NW, true> kst;
    Stream<D, NW, false> vst;
    kst.init(a.k + (long)k0 * a.k_ld + (long)kvh * D, a.k_ld, lk, wave, lane);
    vst.init(a.v + (long)k0 * a.v_ld + (long)kvh * D, a.v_ld, lk, wave, lane);
    f32x16 o_acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o_acc[i][j] = 0.f;
    // the running maximum starts at a finite number below every finite score: a row that has seen no key yet has
    // p = exp2(-inf - m) = 0 with no special case
    float m_c = -3.0e38f, l_run = 0.f;
    bool redo = false;
    if (t0 < t1) {
        kst.stage(t0, smem, wave, lane);
        vst.stage(t0, smem + 2 * TILE, wave, lane);
        if (t0 + 1 < t1) kst.stage(t0 + 1, smem + TILE, wave, lane);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        // Q has landed, too: said here, or the compiler waits for it (and every DMA with it) in the loop
#pragma unroll
        for (int i = 0; i < KS; ++i) asm volatile("" : "+v"(qf[i]));
        __syncthreads();
        f32x16 a0, a1, b0, b1;
        float mx = -3.0e38f;
        bool need = false;
        if (t0 < tw) {       // scores of the first tile
#pragma unroll
            for (int j = 0; j < 16; ++j) a0[j] = a1[j] = 0.f;
            const char* sk = smem;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const bf16x8 kf0 = *reinterpret_cast<const bf16x8*>(sk + k_off<D>(l31, 2 * ks + hi));
                const bf16x8 kf1 = *reinterpret_cast<const bf16x8*>(sk + k_off<D>(32 + l31, 2 * ks + hi));
                a0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf0, qf[ks], a0, 0, 0, 0);
                a1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf1, qf[ks], a1, 0, 0, 0);
            }
            if (t0 >= tf) {
                if (CAP) {
                    cap_scores<LARGE>(a0, a);
                    cap_scores<LARGE>(a1, a);
                }
                mask_scores(a0, a1, t0 * BKV, nvis, hi);
            }
            float nmx = -3.0e38f;
#pragma unroll
            for (int r = 0; r < 16; ++r) nmx = max3(nmx, a0[r], a1[r]);
            mx = CAP ? (t0 < tf ? capped<LARGE>(half_max(nmx), a, 0.f) : half_max(nmx)) : half_max(nmx) * a.scale_log2;
            need = __any(mx > m_c + RESCALE_THR);
        }
        __syncthreads();      // every wave is done with K(t0) before K(t0 + 2) overwrites it
        // step u handles tile t0 + u; buffers go by the parity of u.  LDS during it: K of the next tile, V of this one
#define PIPE_STEP(HAS_NEXT, MASK_NEXT, C0, C1, N0, N1, U)                                                           \
    do {                                                                                                            \
        const int u_ = (U), t_ = t0 + u_;                                                                           \
        pipe_step<D, NW, CAP, LARGE, HAS_NEXT, MASK_NEXT, CAP && HAS_NEXT && !MASK_NEXT>(                                  \
            o_acc, qf, m_c, l_run, C0, C1, N0, N1, mx, need,                                                        \
                                                   smem + ((u_ + 1) & 1) * TILE, smem + (2 + (u_ & 1)) * TILE, kst, \
                                                   smem + (u_ & 1) * TILE, t_ + 2 < t1, vst,                        \
                                                   smem + (2 + ((u_ + 1) & 1)) * TILE, t_ + 1 < t1, t_, nvis,       \
                                                   t_ >= tf, redo, a, wave, lane);                                  \
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                                                            \
        __syncthreads();                                                                                            \
    } while (0)
        int u = 0;
        for (; t0 + u + 2 < tf; u += 2) {     // next tile whole; two steps per turn: the score registers swap roles
            PIPE_STEP(true, false, a0, a1, b0, b1, u);
            PIPE_STEP(true, false, b0, b1, a0, a1, u + 1);
        }
        if (t0 + u + 1 < tf) {
            PIPE_STEP(true, false, a0, a1, b0, b1, u);
            a0 = b0;
            a1 = b1;
            ++u;
        }
        if (CAP && t0 < tf) {                 // the last whole tile
            cap_scores<LARGE>(a0, a);
            cap_scores<LARGE>(a1, a);
        }
        for (; t0 + u + 1 < tw; ++u) {
            PIPE_STEP(true, true, a0, a1, b0, b1, u);
            a0 = b0;
            a1 = b1;
        }
        if (t0 + u < tw) {
            PIPE_STEP(false, false, a0, a1, b0, b1, u);
            ++u;
        }
#undef PIPE_STEP
        for (; t0 + u < t1; ++u) {            // rows of other waves still see keys: keep their tiles coming
            if (t0 + u + 2 < t1) kst.stage(t0 + u + 2, smem + (u & 1) * TILE, wave, lane);
            if (t0 + u + 1 < t1) vst.stage(t0 + u + 1, smem + (2 + ((u + 1) & 1)) * TILE, wave, lane);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
    }
    // rows of the workgroup see different key counts: only then can a hidden value have been multiplied
    const int wfull = __builtin_amdgcn_readfirstlane(visible(a, (int)((unsigned)(rb * (32 * NW)) / group), lq, lk, prefix));
    if (t1 > wfull / BKV && t0 < t1) {
        int* flags = reinterpret_cast<int*>(smem);        // the tiles are free (last step's barrier)
        if (lane == 0) flags[wave] = redo;
        __syncthreads();
        int any = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) any |= flags[w];
        __syncthreads();
        if (__builtin_amdgcn_readfirstlane(any)) {
            m_c = -3.0e38f;
            l_run = 0.f;
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o_acc[i][j] = 0.f;
            for (int t = t0; t < t1; ++t)
                careful_step<D, NW, CAP, LARGE>(o_acc, qf, m_c, l_run, smem, kst, vst, t, nvis, a, wave, lane);
        }
    }
    l_run = half_sum(l_run);
    const bool live = r_first + l31 < rows;
    // register j of o_acc[db] is dimension 32 db + 8 (j >> 2) + 4 hi + (j & 3) of query row l31
    if (SPLIT && parts > 1) {
        if (!live) return;
        const long wrow = (long)(q0 + tok) * a.kv_heads * a.group + head;
        float* w = ws_row<D>(a, part, wrow) + 4 * hi;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4)
                *reinterpret_cast<float4*>(w + db * 32 + 8 * g4) =
                    make_float4(o_acc[db][4 * g4], o_acc[db][4 * g4 + 1], o_acc[db][4 * g4 + 2], o_acc[db][4 * g4 + 3]);
        if (hi == 0) *reinterpret_cast<float2*>(ws_stat<D>(a, part, wrow)) = make_float2(m_c, l_run);
        return;
    }
    const float inv = l_run > 0.f ? 1.f / l_run : (l_run == l_run ? 0.f : l_run);     // no key: 0; NaN stays NaN
    // the tiles are free (last step's barrier): 64 D bytes per wave for the output rows
    char* ep = smem + wave * (64 * D);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const uint2 w = make_uint2(pack_bf2(o_acc[db][4 * g4] * inv, o_acc[db][4 * g4 + 1] * inv),
                                       pack_bf2(o_acc[db][4 * g4 + 2] * inv, o_acc[db][4 * g4 + 3] * inv));
            *reinterpret_cast<uint2*>(ep + l31 * ROWB + (((db * 4 + g4) ^ (l31 & (CPR - 1))) << 4) + hi * 8) = w;
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
        const int r = i * RPI + lane / CPR, c = lane % CPR;
        const uint4 w = *reinterpret_cast<const uint4*>(ep + r * ROWB + ((c ^ (r & (CPR - 1))) << 4));
        const unsigned rr = (unsigned)(r_first + r);
        if (rr < (unsigned)rows)
            *reinterpret_cast<uint4*>(a.o + (long)(q0 + rr / group) * a.o_ld + (long)(kvh * group + rr % group) * D + c * 8) = w;
    }
}

// The grid holds `row_blocks` work items per key head: never fewer than the documents need, whatever their lengths
// (sum of ceil(rows / per) <= total / per + documents); the rest find nothing to do.  Workgroup ids go round-robin over
// the 8 XCDs, each with its own L2.  The row blocks of a key head form `stripes` = 8 / gcd(heads, 8) units, block b in
// unit b % stripes, and an XCD takes kv_heads * stripes / 8 consecutive units: a head's K / V stream is fetched into as
// few L2s as possible, and XCDs that share a head get the same mix of documents and (causal) lengths (contiguous ranges
// instead of stripes: 1040 against 1150 TFLOP/s with 12 heads over documents of 20280, 1560, 14040 and 3600 tokens).
template <int D, int NW, bool CAP, bool LARGE>
__global__ void __launch_bounds__(64 * NW, 2) attn_packed_kernel(Args a) {
#ifdef __HIP_DEVICE_COMPILE__     // the host pass has no use for the body (and refuses register constraints in shared parts of it)
    extern __shared__ __attribute__((aligned(16))) char smem[];   // (K | V)[2]
    const int id = blockIdx.x;
    const int per_unit = (a.row_blocks + a.stripes - 1) / a.stripes;
    const int unit = (id & 7) * (a.kv_heads * a.stripes >> 3) + (id >> 3) / per_unit;
    const int kvh = unit / a.stripes;
    const int blk = (id >> 3) % per_unit * a.stripes + unit % a.stripes;
    int doc, rb, part, parts;
    if (!find_block<32 * NW, false>(a, blk, threadIdx.x & 63, doc, rb, part, parts)) return;
    doc = __builtin_amdgcn_readfirstlane(doc);
    rb = __builtin_amdgcn_readfirstlane(rb);
    attend<D, NW, CAP, LARGE, false>(a, smem, kvh, doc, rb, 0, 1);
#endif
}

// Few query rows: the keys of a document are split into parts of about `chunk` tiles, all of one size per document, so
// that documents of very different lengths fill the chip evenly.  Workgroups go on with further items a grid away: the
// host sizes the grid by the lengths that it was told.  A document in one part is finished here, the others by the join.
template <int D, int NW, bool CAP, bool LARGE>
__global__ void __launch_bounds__(64 * NW, NW == 1 ? 1 : 2) attn_packed_split_kernel(Args a) {
#ifdef __HIP_DEVICE_COMPILE__
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int kvh = blockIdx.x % a.kv_heads;
    for (int blk = blockIdx.x / a.kv_heads;; blk += a.row_blocks) {
        int doc, rb, part, parts;
        if (!find_block<32 * NW, true>(a, blk, threadIdx.x & 63, doc, rb, part, parts)) return;
        doc = __builtin_amdgcn_readfirstlane(doc);
        rb = __builtin_amdgcn_readfirstlane(rb);
        part = __builtin_amdgcn_readfirstlane(part);
        parts = __builtin_amdgcn_readfirstlane(parts);
        attend<D, NW, CAP, LARGE, true>(a, smem, kvh, doc, rb, part, parts);
        __syncthreads();                      // the output staging of this item before the tiles of the next
    }
#endif
}

// out = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m) over the parts; one workgroup per (token, head), its waves take
// the parts in turn and meet in a fixed order
template <int D>
__global__ void __launch_bounds__(256) attn_packed_join_kernel(Args a) {
    __shared__ float2 acc[4][64];
    __shared__ float den[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int heads = a.kv_heads * a.group;
    const long row = blockIdx.x;
    const int tok = (int)(row / heads), head = (int)(row % heads);
    int parts = 1;
    for (int d0 = 0; d0 < a.docs; d0 += 64) {            // the token's document
        const int d = min(d0 + lane, a.docs - 1);
        int q0, lq, k0, lk;
        doc_range(a, d, q0, lq, k0, lk);
        const unsigned long long hit = __ballot(tok >= q0 && tok < q0 + lq);
        if (hit) {
            parts = parts_of(a, __shfl(lk, __builtin_ctzll(hit), 64));
            break;
        }
    }
    if (parts == 1) return;                              // finished already, or in no document
    float m = -3.0e38f;
    for (int s = lane; s < parts; s += 64) m = __builtin_fmaxf(m, ws_stat<D>(a, s, row)[0]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, o, 64));
    float l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll 4
    for (int s = wave; s < parts; s += 4) {
        const float2 st = *reinterpret_cast<const float2*>(ws_stat<D>(a, s, row));
        const float w = __builtin_amdgcn_exp2f(st.x - m);
        const float* p = ws_row<D>(a, s, row);
        l = fmaf(st.y, w, l);
        if constexpr (D == 128) {
            const float2 v = reinterpret_cast<const float2*>(p)[lane];
            o0 = fmaf(v.x, w, o0);
            o1 = fmaf(v.y, w, o1);
        } else {
            o0 = fmaf(p[lane], w, o0);
        }
    }
    acc[wave][lane] = make_float2(o0, o1);
    if (lane == 0) den[wave] = l;
    __syncthreads();
    if (wave != 0) return;
    l = (den[0] + den[1]) + (den[2] + den[3]);
    o0 = (acc[0][lane].x + acc[1][lane].x) + (acc[2][lane].x + acc[3][lane].x);
    o1 = (acc[0][lane].y + acc[1][lane].y) + (acc[2][lane].y + acc[3][lane].y);
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    bf16_t* dst = a.o + (long)tok * a.o_ld + (long)head * D;
    if constexpr (D == 128) reinterpret_cast<uint32_t*>(dst)[lane] = pack_bf2(o0 * inv, o1 * inv);
    else dst[lane] = f2bf(o0 * inv);
}

// How a call is launched, from what the host knows: totals, the number of documents and the caller's bounds on a
// document's lengths (hints: the kernels read the lengths themselves).
struct Plan {
    int waves;               // per workgroup: 32 query rows each
    bool split;              // the split kernel (a document's keys in up to max_splits parts of about `chunk` tiles)
    int row_blocks, chunk, max_splits;
};

// 8 waves (256 rows, one workgroup per CU) or 4 (128 rows, two that overlap each other's start and end)?  Eight read K and
// V half as often and are 7 % faster in full rounds, but a last round that is partly filled costs them a whole one.
//   short keys: four (60 documents of 257 tokens, 12 heads: 80 us against 98);
//   causal (lengths differ, longest first): four below three rounds of eight (packed prompts of 1 to 2100 tokens with a cap
//   68 us against 77, the cap being a pass of its own then; 6000 tokens, 12 heads 134 against 143; 20280 tokens, 12 heads:
//   1239 against 1188);
//   otherwise by rounds, a round of four-wave workgroups that run alone on their CUs counted as 0.6 (6000 tokens, 12
//   heads: 274 us against 297; three documents of 3000: 183 against 166; 20280: 2331 against 2151).
bool wide_workgroups(long rows, int docs, int kv_heads, int causal, long max_k, long cus) {
    const long w8 = (rows / 256 + (docs + 1) / 2) * kv_heads, w4 = (rows / 128 + (docs + 1) / 2) * kv_heads;
    if (max_k <= 1024) return false;
    if (causal) return w8 >= 3 * cus;
    const double rem = (double)(w4 % (2 * cus)) / cus;
    const double t4 = 1.07 * ((double)(w4 / (2 * cus)) + (rem == 0 ? 0. : rem <= 1. ? 0.6 : 1.));
    return (double)((w8 + cus - 1) / cus) < t4;
}

Plan plan_of(long total_q, long total_k, int docs, int kv_heads, int group, int D, long max_q, long max_k, int causal) {
    Plan p;
    const long cus = ovd_device_cus();
    max_q = max_q < 1 ? 1 : (max_q > total_q ? total_q : max_q);
    max_k = max_k < 1 ? 1 : (max_k > total_k ? (total_k < 1 ? 1 : total_k) : max_k);
    const long rows = max_q * group;
    p.waves = rows <= 32 ? 1 : (wide_workgroups(total_q * group, docs, kv_heads, causal, max_k, cus) ? 8 : 4);
    const long per = 32L * p.waves;
    p.row_blocks = (int)(total_q * group / per + docs);        // >= the sum of ceil(Lq group / per) over the documents
    p.split = p.waves == 1 || (p.waves == 4 && (long)p.row_blocks * kv_heads <= cus);
    p.chunk = 1 << 30;
    p.max_splits = 1;
    if (p.split) {
        // All parts have about the same number of tiles, `chunk`, and `slots` workgroups run at a time.  R rounds leave
        // R slots - (one partly filled part per row block) parts for the tiles; a workgroup's start costs about as much
        // as 4 tiles.  The number of rounds that this puts first (8 tokens against 1 to 32760 keys, 8 key heads: one
        // round of 23 tiles 70 us before the join, four rounds of 5 tiles 88 us).
        const long most = (max_k + BKV - 1) / BKV;
        long tiles = p.waves == 1 ? total_k / BKV + docs : most * p.row_blocks;
        if (tiles > most * p.row_blocks) tiles = most * p.row_blocks;
        const long slots = (D == 64 && p.waves == 1 ? 4 : 2) * cus, blocks = (long)p.row_blocks * kv_heads;
        long chunk = most, best = -1;
        for (long r = 1; r <= 8; ++r) {
            if (r * slots <= blocks) continue;
            long c = (tiles * kv_heads + (r * slots - blocks) - 1) / (r * slots - blocks);
            c = c < 4 ? 4 : (c > most ? most : c);
            const long cost = r * (c + 4);
            if (best < 0 || cost < best) {
                best = cost;
                chunk = c;
            }
        }
        if (chunk < 1) chunk = 1;
        p.chunk = (int)chunk;
        p.max_splits = (int)((most + chunk - 1) / chunk);
        if (p.max_splits > 256) p.max_splits = 256;
        p.row_blocks = (int)(tiles / chunk + p.row_blocks);     // work items, were every length at its bound
    }
    return p;
}

}  // namespace

long ovd_impl_attn_packed_workspace(long total_q, long total_k, int docs, int q_heads, int kv_heads, int D, long max_q,
                                    long max_k) {
    if (total_q <= 0 || docs <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads) return 0;
    int parts = 1;
    for (int causal = 0; causal < 2; ++causal) {
        const Plan p = plan_of(total_q, total_k, docs, kv_heads, q_heads / kv_heads, D, max_q, max_k, causal);
        if (p.max_splits > parts) parts = p.max_splits;
    }
    return parts > 1 ? (long)parts * total_q * q_heads * (D + 2) * (long)sizeof(float) : 0;
}

int ovd_impl_attn_packed(const bf16_t* q, const bf16_t* k, const bf16_t* v, bf16_t* out, long total_q, long total_k,
                         const int* cu_q, const int* cu_k, int docs, long max_q, long max_k, int q_heads, int kv_heads,
                         int D, long q_ld, long k_ld, long v_ld, long o_ld, int causal, const int* prefix,
                         float softmax_scale, float softcap, void* workspace, long workspace_bytes, hipStream_t st) {
    OVD_REQUIRE(D == 64 || D == 128, "attn_packed: head_dim %d not supported (64 or 128)", D);
    OVD_REQUIRE(total_q >= 0 && total_k >= 0 && total_q < (1L << 31) - 256 && total_k < (1L << 31) - 256 && docs > 0,
                "attn_packed: bad sizes Tq=%ld Tk=%ld documents=%d", total_q, total_k, docs);
    OVD_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0, "attn_packed: %d query heads over %d key heads",
                q_heads, kv_heads);
    OVD_REQUIRE(total_q * (q_heads / kv_heads) + 64L * docs < (1L << 31) - 1024, "attn_packed: too many query rows");
    OVD_REQUIRE(q_ld % 8 == 0 && k_ld % 8 == 0 && v_ld % 8 == 0 && o_ld % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(out) % 16 == 0,
                "attn_packed: token rows must keep 16-byte alignment");
    OVD_REQUIRE(q_ld >= (long)q_heads * D && o_ld >= (long)q_heads * D && k_ld >= (long)kv_heads * D && v_ld >= (long)kv_heads * D,
                "attn_packed: token stride shorter than the heads");
    OVD_REQUIRE(k_ld < (1L << 24) && v_ld < (1L << 24), "attn_packed: token stride too long");
    OVD_REQUIRE(softmax_scale > 0.f && softcap >= 0.f && softmax_scale < 1e30f && softcap < 1e30f,
                "attn_packed: softmax_scale must be positive, softcap positive or 0 (none)");
    OVD_REQUIRE(prefix == nullptr || causal, "attn_packed: a prefix goes with the causal mask");
    OVD_REQUIRE(max_q >= 0 && max_k >= 0, "attn_packed: negative length bound");
    if (total_q == 0) return 0;
    Args a;
    a.q = q; a.k = k; a.v = v; a.o = out;
    a.q_ld = q_ld; a.k_ld = k_ld; a.v_ld = v_ld; a.o_ld = o_ld;
    a.cu_q = cu_q; a.cu_k = cu_k; a.prefix = prefix;
    a.total_q = (int)total_q; a.total_k = (int)total_k; a.docs = docs;
    a.kv_heads = kv_heads; a.group = q_heads / kv_heads; a.causal = causal;
    a.scale_log2 = softmax_scale * 1.4426950408889634f;
    // finite, however small the cap: a score of zero has to stay one
    a.cap_in = softcap > 0.f ? fminf(2.f * a.scale_log2 / softcap, 3.0e38f) : 0.f;
    a.cap_out = softcap * 1.4426950408889634f;
    a.cap_x = softcap > 0.f ? softmax_scale / softcap : 0.f;
    const Plan p = plan_of(total_q, total_k, docs, kv_heads, a.group, D, max_q, max_k, causal);
    // no (or too small a) workspace: every document in one part
    const long part_bytes = total_q * q_heads * (D + 2) * (long)sizeof(float);
    const long room = workspace == nullptr ? 0 : workspace_bytes / part_bytes;
    a.max_splits = room < p.max_splits ? (room < 2 ? 1 : (int)room) : p.max_splits;
    a.chunk = p.chunk;
    a.row_blocks = p.row_blocks;
    a.ws = (float*)workspace;
    OVD_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "attn_packed: the workspace must be 16-byte aligned");
    a.stripes = kv_heads % 8 == 0 ? 1 : kv_heads % 4 == 0 ? 2 : kv_heads % 2 == 0 ? 4 : 8;
    const long per_unit = (p.row_blocks + a.stripes - 1) / a.stripes;
    const long grid = p.split ? (long)p.row_blocks * kv_heads : per_unit * a.stripes * kv_heads;
    // a launch holds fewer than 2^32 threads
    OVD_REQUIRE(grid * 64 * p.waves < (1L << 32) && (a.max_splits == 1 || total_q * q_heads < (1L << 24)),
                "attn_packed: grid too large");
    const size_t lds = 4 * BKV * D * 2;
#define PACKED(KERNEL, NW)                                                                                      \
    {                                                                                                           \
        static OvdLdsLimit lim;                                                                                 \
        if (!lim.ensure(reinterpret_cast<const void*>(&KERNEL), lds))                                           \
            OVD_FAIL("attn_packed: cannot reserve %zu bytes of LDS", lds);                                      \
        hipLaunchKernelGGL((KERNEL), dim3((unsigned)grid), dim3(64 * NW), lds, st, a);                          \
    }
#define PACKED_KIND(DD, CAP, LARGE)                                                                             \
    {                                                                                                           \
        if (p.waves == 8) PACKED(PK(attn_packed_kernel, DD, 8, CAP, LARGE), 8)                                  \
        else if (!p.split) PACKED(PK(attn_packed_kernel, DD, 4, CAP, LARGE), 4)                                 \
        else if (p.waves == 4) PACKED(PK(attn_packed_split_kernel, DD, 4, CAP, LARGE), 4)                       \
        else PACKED(PK(attn_packed_split_kernel, DD, 1, CAP, LARGE), 1)                                         \
    }
#define PACKED_CAP(DD)                                                                                          \
    {                                                                                                           \
        if (softcap > SMALL_CAP) PACKED_KIND(DD, true, true)                                                    \
        else if (softcap > 0.f) PACKED_KIND(DD, true, false)                                                    \
        else PACKED_KIND(DD, false, false)                                                                      \
    }
#define PK(K, DD, NW, CAP, LARGE) (K<DD, NW, CAP, LARGE>)
    if (D == 128) PACKED_CAP(128)
    else PACKED_CAP(64)
#undef PK
#undef PACKED_CAP
#undef PACKED_KIND
#undef PACKED
    OVD_CHECK_LAUNCH("attn_packed");
    if (p.split && a.max_splits > 1) {
        const dim3 jg((unsigned)(total_q * q_heads)), jb(256);
        if (D == 128) hipLaunchKernelGGL(attn_packed_join_kernel<128>, jg, jb, 0, st, a);
        else hipLaunchKernelGGL(attn_packed_join_kernel<64>, jg, jb, 0, st, a);
        OVD_CHECK_LAUNCH("attn_packed join");
    }
    return 0;
}
