// Attention over packed documents, forward: bf16 operands, fp32 softmax and accumulation.
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
// Few rows against long documents: n_splits workgroups share the keys of a tile and a second kernel joins them.
//
// S^T = K Q^T with the key on the MFMA row axis (v_mfma_f32_32x32x16_bf16): a lane holds 32 scores of ONE query, so row
// maxima and sums are in-lane plus one exchange, and P is already the B operand of O^T += V^T P^T.  V^T fragments come
// from the row-major V tile through ds_read_b64_tr_b16; K and V tiles of 64 keys stream HBM -> LDS by DMA with the
// bank swizzle applied to the source chunk.  Key rows past the document are clamped to its last row: what lies behind
// a document is never read, and a masked score is -inf whatever it was.
#include "common.h"

namespace {

constexpr int BKV = 64;                       // keys per tile
constexpr float NEG_INF = -__builtin_inff();

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
    int row_blocks, n_splits;
    float* ws;                                // partial results of the splits
};

// rows [*q0, *q0 + *lq) and keys [*k0, *k0 + *lk) of document d; whatever cu_q / cu_k hold, inside the tensors
__device__ __forceinline__ void doc_range(const Args& a, int d, int& q0, int& lq, int& k0, int& lk) {
    q0 = min(max(a.cu_q[d], 0), a.total_q);
    lq = min(max(a.cu_q[d + 1], q0), a.total_q) - q0;
    k0 = min(max(a.cu_k[d], 0), a.total_k);
    lk = min(max(a.cu_k[d + 1], k0), a.total_k) - k0;
}

// document and row block (of ROWS rows) of work item `blk`, and how many items follow it; false past the last one
template <int ROWS>
__device__ __forceinline__ bool find_block(const Args& a, int blk, int lane, int& doc, int& rb, int& left) {
    bool found = false;
    for (int d0 = 0; d0 < a.docs; d0 += 64) {
        const int d = d0 + lane;
        int n = 0;
        if (d < a.docs) {
            const int q0 = min(max(a.cu_q[d], 0), a.total_q);
            const int lq = min(max(a.cu_q[d + 1], q0), a.total_q) - q0;
            n = (int)(((long)lq * a.group + ROWS - 1) / ROWS);
        }
        int incl = n;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int up = __shfl_up(incl, s, 64);
            if (lane >= s) incl += up;
        }
        const int sum = __shfl(incl, 63, 64);
        if (found) {
            left += sum;
            continue;
        }
        const unsigned long long hit = __ballot(blk < incl);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            doc = d0 + l;
            rb = blk - __shfl(incl - n, l, 64);
            left = sum - blk - 1;
            found = true;
        }
        blk -= sum;
    }
    return found;
}

__device__ __forceinline__ int visible(const Args& a, int i, int lq, int lk, int prefix) {
    if (!a.causal) return lk;
    const int n = max(i + lk - lq + 1, prefix);
    return min(max(n, 0), lk);
}

// workspace: accumulators [n_splits][rows = total_q * Nq][D], then (maximum, sum) [n_splits][rows][2]
template <int D>
__device__ __forceinline__ float* ws_row(const Args& a, int split, long row) {
    const long rows = (long)a.total_q * a.kv_heads * a.group;
    return a.ws + (split * rows + row) * D;
}
template <int D>
__device__ __forceinline__ float* ws_stat(const Args& a, int split, long row) {
    const long rows = (long)a.total_q * a.kv_heads * a.group;
    return a.ws + a.n_splits * rows * D + (split * rows + row) * 2;
}

// one work item: 32 NW rows of document `doc` under key head kvh, keys of split `split`
template <int D, int NW, bool CAP>
__device__ __forceinline__ void attend(const Args& a, char* smem, int kvh, int split, int doc, int rb) {
    constexpr int ROWB = D * 2;                          // bytes per K / V row
    constexpr int TILE = BKV * ROWB;                     // bytes per tile
    constexpr int CPR = ROWB / 16;                       // chunks per row
    constexpr int RPI = 64 / CPR;                        // rows per DMA instruction of a wave
    constexpr int DB = D / 32, KS = D / 16;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    int q0, lq, k0, lk;
    doc_range(a, doc, q0, lq, k0, lk);
    const int prefix = a.prefix ? min(max(a.prefix[doc], 0), lk) : 0;
    const long rows = (long)lq * a.group;
    const long r_first = (long)rb * (32 * NW) + wave * 32;
    const long row = min(r_first + l31, rows - 1);       // rows past the last repeat it and are not stored
    const int tok = (int)(row / a.group), head = kvh * a.group + (int)(row % a.group);
    const int nvis = visible(a, tok, lq, lk, prefix);
    // visible counts grow with the row: the tile range follows from the workgroup's last row, the tiles that need no
    // mask from the wave's first
    const long last_row = min((long)(rb + 1) * (32 * NW), rows) - 1;
    const int kend = visible(a, (int)(last_row / a.group), lq, lk, prefix);
    const int full = visible(a, (int)(min(r_first, rows - 1) / a.group), lq, lk, prefix);
    const int nt = (kend + BKV - 1) / BKV;
    const int t0 = (int)((long)nt * split / a.n_splits), t1 = (int)((long)nt * (split + 1) / a.n_splits);

    bf16x8 qf[KS];
    {
        const bf16_t* qp = a.q + (long)(q0 + tok) * a.q_ld + (long)head * D + 8 * hi;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
    }
    const char* kb = reinterpret_cast<const char*>(a.k + (long)k0 * a.k_ld + (long)kvh * D);
    const char* vb = reinterpret_cast<const char*>(a.v + (long)k0 * a.v_ld + (long)kvh * D);
    auto stage = [&](int t, int buf) {
        char* dst = smem + buf * 2 * TILE;
#pragma unroll
        for (int i = 0; i < TILE / 1024 / NW; ++i) {
            const int r = (i * NW + wave) * RPI + lane / CPR, c = lane % CPR;
            const long key = min(t * BKV + r, lk - 1);
            const int ck = D == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
            const int cv = D == 128 ? c ^ ((r & 3) << 2) : c ^ (((r >> 1) & 1) << 2);
            __builtin_amdgcn_global_load_lds(kb + key * a.k_ld * 2 + ck * 16, (lds_ptr)(dst + (i * NW + wave) * 1024), 16, 0, 0);
            __builtin_amdgcn_global_load_lds(vb + key * a.v_ld * 2 + cv * 16, (lds_ptr)(dst + TILE + (i * NW + wave) * 1024), 16, 0, 0);
        }
    };
    f32x16 o_acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o_acc[i][j] = 0.f;
    float m_run = NEG_INF, l_run = 0.f;
    if (t0 < t1) stage(t0, 0);
    for (int t = t0; t < t1; ++t) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                      // tile t has landed everywhere, every wave is done with tile t - 1
        const int buf = (t - t0) & 1;
        if (t + 1 < t1) stage(t + 1, buf ^ 1);
        const char* sk = smem + buf * 2 * TILE;
        const char* sv = sk + TILE;
        f32x16 s0, s1;
#pragma unroll
        for (int j = 0; j < 16; ++j) s0[j] = s1[j] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16x8 kf0 = *reinterpret_cast<const bf16x8*>(sk + k_off<D>(l31, 2 * ks + hi));
            const bf16x8 kf1 = *reinterpret_cast<const bf16x8*>(sk + k_off<D>(32 + l31, 2 * ks + hi));
            s0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf0, qf[ks], s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf1, qf[ks], s1, 0, 0, 0);
        }
        // scores in units of log2: s * scale * log2(e), or cap log2(e) tanh(s scale / cap) with
        // tanh(x) = 1 - 2 / (1 + e^2x) (both ends saturate without overflow)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if constexpr (CAP) {
                s0[j] = a.cap_out - 2.f * a.cap_out * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s0[j] * a.cap_in));
                s1[j] = a.cap_out - 2.f * a.cap_out * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s1[j] * a.cap_in));
            } else {
                s0[j] *= a.scale_log2;
                s1[j] *= a.scale_log2;
            }
        }
        if ((t + 1) * BKV > full) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = t * BKV + (r & 3) + 8 * (r >> 2) + 4 * hi;
                if (key >= nvis) s0[r] = NEG_INF;
                if (key + 32 >= nvis) s1[r] = NEG_INF;
            }
        }
        float mx = s0[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = __builtin_fmaxf(mx, s0[r]);
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = __builtin_fmaxf(mx, s1[r]);
        const float m_new = __builtin_fmaxf(m_run, half_max(mx));
        const float m_ref = m_new == NEG_INF ? 0.f : m_new;       // no key seen yet: every p is exp2(-inf) = 0
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_ref);
        m_run = m_new;
        float sum = 0.f;
        uint32_t pw[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a0 = __builtin_amdgcn_exp2f(s0[2 * i] - m_ref), a1 = __builtin_amdgcn_exp2f(s0[2 * i + 1] - m_ref);
            const float b0 = __builtin_amdgcn_exp2f(s1[2 * i] - m_ref), b1 = __builtin_amdgcn_exp2f(s1[2 * i + 1] - m_ref);
            sum += (a0 + a1) + (b0 + b1);
            pw[i] = pack_bf2(a0, a1);
            pw[8 + i] = pack_bf2(b0, b1);
        }
        l_run = l_run * alpha + sum;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o_acc[i][j] *= alpha;
        const int g = lane >> 4, i16 = lane & 15, qd = i16 >> 2, pp = i16 & 3;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            const bf16x8 pf = __builtin_bit_cast(bf16x8, make_uint4(pw[4 * st], pw[4 * st + 1], pw[4 * st + 2], pw[4 * st + 3]));
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const int kr = 16 * st + 4 * (g >> 1) + qd;
                const int ch = db * 4 + 2 * (g & 1) + (pp >> 1);
                const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4_ptr)(sv + v_off<D>(kr, ch) + 8 * (pp & 1)));
                const bf16x4_t h4 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4_ptr)(sv + v_off<D>(kr + 8, ch) + 8 * (pp & 1)));
                const uint2 lo2 = __builtin_bit_cast(uint2, lo), hi2 = __builtin_bit_cast(uint2, h4);
                const bf16x8 vf = __builtin_bit_cast(bf16x8, make_uint4(lo2.x, lo2.y, hi2.x, hi2.y));
                o_acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf, o_acc[db], 0, 0, 0);
            }
        }
    }
    l_run = half_sum(l_run);
    const bool live = r_first + l31 < rows;
    // register j of o_acc[db] is dimension 32 db + 8 (j >> 2) + 4 hi + (j & 3) of query row l31
    if (a.n_splits > 1) {
        if (!live) return;
        const long wrow = (long)(q0 + tok) * a.kv_heads * a.group + head;
        float* w = ws_row<D>(a, split, wrow) + 4 * hi;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4)
                *reinterpret_cast<float4*>(w + db * 32 + 8 * g4) =
                    make_float4(o_acc[db][4 * g4], o_acc[db][4 * g4 + 1], o_acc[db][4 * g4 + 2], o_acc[db][4 * g4 + 3]);
        if (hi == 0) *reinterpret_cast<float2*>(ws_stat<D>(a, split, wrow)) = make_float2(m_run, l_run);
        return;
    }
    const float inv = l_run > 0.f ? 1.f / l_run : (l_run == l_run ? 0.f : l_run);     // no key: 0; NaN stays NaN
    __syncthreads();                          // the tiles are free: 64 D bytes per wave for the output rows
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
        const long rr = r_first + r;
        if (rr < rows)
            *reinterpret_cast<uint4*>(a.o + (q0 + rr / a.group) * a.o_ld + ((long)kvh * a.group + rr % a.group) * D + c * 8) = w;
    }
}

// The grid holds `row_blocks` work items per key head and split, enough for the lengths the host was told; should the
// documents be longer than that, a workgroup goes on with the items a grid further.
template <int D, int NW, bool CAP>
__global__ void __launch_bounds__(64 * NW) attn_packed_kernel(Args a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];   // (K | V)[2]
    const int split = blockIdx.x % a.n_splits, id = blockIdx.x / a.n_splits;
    const int kvh = id / a.row_blocks;
    for (int blk = id % a.row_blocks;; blk += a.row_blocks) {
        int doc, rb, left;
        if (!find_block<32 * NW>(a, blk, threadIdx.x & 63, doc, rb, left)) return;
        attend<D, NW, CAP>(a, smem, kvh, split, __builtin_amdgcn_readfirstlane(doc), __builtin_amdgcn_readfirstlane(rb));
        if (__builtin_amdgcn_readfirstlane(left) < a.row_blocks) return;
        __syncthreads();                      // the output staging of this item before the tiles of the next
    }
}

// out = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m) over the splits, in their order; one wave per (token, head), rows
// inside [cu_q[0], cu_q[docs]) only
template <int D>
__global__ void __launch_bounds__(256) attn_packed_join_kernel(Args a) {
    const int lane = threadIdx.x & 63;
    const int heads = a.kv_heads * a.group;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (long)a.total_q * heads) return;
    const int tok = (int)(row / heads), head = (int)(row % heads);
    if (tok < a.cu_q[0] || tok >= a.cu_q[a.docs]) return;
    float m = NEG_INF;
    for (int s = 0; s < a.n_splits; ++s) m = __builtin_fmaxf(m, ws_stat<D>(a, s, row)[0]);
    const float m_ref = m == NEG_INF ? 0.f : m;
    float l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int s = 0; s < a.n_splits; ++s) {
        const float2 st = *reinterpret_cast<const float2*>(ws_stat<D>(a, s, row));
        const float w = __builtin_amdgcn_exp2f(st.x - m_ref);
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
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    bf16_t* dst = a.o + (long)tok * a.o_ld + (long)head * D;
    if constexpr (D == 128) reinterpret_cast<uint32_t*>(dst)[lane] = pack_bf2(o0 * inv, o1 * inv);
    else dst[lane] = f2bf(o0 * inv);
}

// Rows per workgroup and key splits of a launch, from what the host knows: totals, the number of documents and the
// caller's bounds on a document's lengths (hints: they size the grid, the kernels read the lengths themselves).
struct Plan {
    int waves, row_blocks, splits;
};

Plan plan_of(long total_q, int docs, int kv_heads, int group, long max_q, long max_k) {
    Plan p;
    max_q = max_q < 1 ? 1 : (max_q > total_q ? total_q : max_q);
    const long rows = max_q * group;
    p.waves = rows <= 32 ? 1 : 4;
    const long per = 32L * p.waves;
    // sum over documents of ceil(Lq group / per) <= total / per + docs, and <= docs * ceil(max / per)
    long nb = total_q * group / per + docs;
    const long nb2 = docs * ((rows + per - 1) / per);
    p.row_blocks = (int)(nb < nb2 ? nb : nb2);
    p.splits = 1;
    const long wgs = (long)p.row_blocks * kv_heads;
    if (p.waves == 1 && wgs < 2L * ovd_device_cus()) {
        const long want = (2L * ovd_device_cus() + wgs - 1) / (wgs > 0 ? wgs : 1);
        const long most = (max_k + 4 * BKV - 1) / (4 * BKV);       // at least 4 tiles each
        p.splits = (int)(want < most ? want : most);
        if (p.splits > 64) p.splits = 64;
        if (p.splits < 1) p.splits = 1;
    }
    return p;
}

}  // namespace

long ovd_impl_attn_packed_workspace(long total_q, int docs, int q_heads, int kv_heads, int D, long max_q, long max_k) {
    if (total_q <= 0 || docs <= 0 || kv_heads <= 0 || q_heads % kv_heads) return 0;
    const Plan p = plan_of(total_q, docs, kv_heads, q_heads / kv_heads, max_q, max_k);
    return p.splits > 1 ? (long)p.splits * total_q * q_heads * (D + 2) * (long)sizeof(float) : 0;
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
    OVD_REQUIRE(total_q * (q_heads / kv_heads) / 32 + docs < (1L << 31) - 256, "attn_packed: too many query rows");
    OVD_REQUIRE(q_ld % 8 == 0 && k_ld % 8 == 0 && v_ld % 8 == 0 && o_ld % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(out) % 16 == 0,
                "attn_packed: token rows must keep 16-byte alignment");
    OVD_REQUIRE(q_ld >= (long)q_heads * D && o_ld >= (long)q_heads * D && k_ld >= (long)kv_heads * D && v_ld >= (long)kv_heads * D,
                "attn_packed: token stride shorter than the heads");
    OVD_REQUIRE(softmax_scale > 0.f && softcap >= 0.f && softmax_scale < 1e30f && softcap < 1e30f,
                "attn_packed: softmax_scale must be positive, softcap positive or 0 (none)");
    OVD_REQUIRE(prefix == nullptr || causal, "attn_packed: a prefix goes with the causal mask");
    OVD_REQUIRE(max_q >= 0 && max_k >= 0, "attn_packed: negative length bound");
    if (total_q == 0) return 0;
    if (max_k > total_k) max_k = total_k;       // the workspace was sized for the caller's bound: never more splits
    Args a;
    a.q = q; a.k = k; a.v = v; a.o = out;
    a.q_ld = q_ld; a.k_ld = k_ld; a.v_ld = v_ld; a.o_ld = o_ld;
    a.cu_q = cu_q; a.cu_k = cu_k; a.prefix = prefix;
    a.total_q = (int)total_q; a.total_k = (int)total_k; a.docs = docs;
    a.kv_heads = kv_heads; a.group = q_heads / kv_heads; a.causal = causal;
    a.scale_log2 = softmax_scale * 1.4426950408889634f;
    a.cap_in = softcap > 0.f ? 2.f * a.scale_log2 / softcap : 0.f;
    a.cap_out = softcap * 1.4426950408889634f;
    Plan p = plan_of(total_q, docs, kv_heads, a.group, max_q, max_k);
    if (p.splits > 1 && (workspace == nullptr ||
                         (long)p.splits * total_q * q_heads * (D + 2) * (long)sizeof(float) > workspace_bytes))
        p.splits = 1;
    a.row_blocks = p.row_blocks;
    a.n_splits = p.splits;
    a.ws = (float*)workspace;
    const long grid = (long)p.row_blocks * kv_heads * p.splits;
    OVD_REQUIRE(grid < (1L << 31), "attn_packed: grid too large");
    const size_t lds = 4 * BKV * D * 2;
#define PACKED(DD, NW, CAP)                                                                                     \
    {                                                                                                           \
        static OvdLdsLimit lim;                                                                                 \
        if (!lim.ensure(reinterpret_cast<const void*>(&attn_packed_kernel<DD, NW, CAP>), lds))                  \
            OVD_FAIL("attn_packed: cannot reserve %zu bytes of LDS", lds);                                      \
        hipLaunchKernelGGL((attn_packed_kernel<DD, NW, CAP>), dim3((unsigned)grid), dim3(64 * NW), lds, st, a); \
    }
#define PACKED_D(DD)                                                    \
    {                                                                   \
        if (p.waves == 1) {                                             \
            if (softcap > 0.f) PACKED(DD, 1, true) else PACKED(DD, 1, false) \
        } else {                                                        \
            if (softcap > 0.f) PACKED(DD, 4, true) else PACKED(DD, 4, false) \
        }                                                               \
    }
    if (D == 128) PACKED_D(128) else PACKED_D(64)
#undef PACKED_D
#undef PACKED
    OVD_CHECK_LAUNCH("attn_packed");
    if (p.splits > 1) {
        const long rows = total_q * q_heads;
        const dim3 jg((unsigned)((rows + 3) / 4)), jb(256);
        if (D == 128) hipLaunchKernelGGL(attn_packed_join_kernel<128>, jg, jb, 0, st, a);
        else hipLaunchKernelGGL(attn_packed_join_kernel<64>, jg, jb, 0, st, a);
        OVD_CHECK_LAUNCH("attn_packed join");
    }
    return 0;
}
