// paged_attn.hip -- causal attention of new tokens over a paged K/V cache.
//
//   out[i] = sum_{t <= pos(i)} w_t v_t / sum w_t,   w_t = 2^(s_t - m),
//   s_t = <q_i, k_t> scale log2(e),  m = max s_t    (online over key blocks)
//
// Products on the bf16 matrix cores without loss of fp32 precision: a number
// x of fp32 is the exact sum of three bf16 numbers (its mantissa's upper,
// middle and lower 8 bits, by truncation, so nothing overflows), a bf16 or
// 8-bit cached number is one bf16 number exactly.  A product of two fp32
// numbers takes the six of its nine partial products that reach 24 bits, one
// with a cached bf16 or 8-bit number three, all exact; sums are fp32.  An
// 8-bit key's scale multiplies its score, an 8-bit value's scale its weight.
//
// A head's queries: with G query heads to a cached head, rows r = token * G +
// (head in its group) of one cached head are computed together, so its keys
// and values are read once for all of them.
#include "common.h"
#include "../kernel_params.h"

#define PA_LOG2E 1.4426950408889634f
#define PA_NONE 0x7fffffff

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned pa_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned pa_u32x2 __attribute__((ext_vector_type(2)));

// The upper halves of two words, a's below b's: two floats truncated to bf16.
__device__ __forceinline__ unsigned pa_pack(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float pa_cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// Eight numbers as NT bf16 terms (NT 3: exact; NT 1: the numbers are bf16).
template <int NT>
__device__ __forceinline__ void pa_split(const float (&x)[8], pa_bf16x8 (&t)[NT]) {
    pa_u32x4 w[NT];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            w[n][i] = pa_pack(a, b);
            if (n + 1 < NT) {
                a -= pa_cut(a);
                b -= pa_cut(b);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++) t[n] = __builtin_bit_cast(pa_bf16x8, w[n]);
}

// acc += A B over the partial products that count: terms of A (NA) and B (3),
// smallest first.
template <int NA>
__device__ __forceinline__ f32x4 pa_mma(const pa_bf16x8 (&a)[NA], const pa_bf16x8 (&b)[3], f32x4 acc) {
#pragma unroll
    for (int d = 2; d >= 0; d--)
#pragma unroll
        for (int i = 0; i < NA; i++)
            if (d - i >= 0) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[d - i], acc, 0, 0, 0);
    return acc;
}

// N consecutive cached numbers of one row, as they lie in memory.
template <int TYPE, int N>
struct PaRun {
    static constexpr int BYTES = N * (TYPE == KV_F32 ? 4 : TYPE == KV_BF16 ? 2 : 1);
    static constexpr int NW = (BYTES + 3) / 4;
    unsigned w[NW];
    __device__ __forceinline__ void load(const void* pool, long long first) {
        const unsigned char* s = (const unsigned char*)pool + first * (BYTES / N);
        if constexpr (BYTES % 16 == 0) {
#pragma unroll
            for (int i = 0; i < NW / 4; i++) {
                const pa_u32x4 v = ((const pa_u32x4*)s)[i];
#pragma unroll
                for (int j = 0; j < 4; j++) w[4 * i + j] = v[j];
            }
        } else if constexpr (BYTES == 8) {
            const pa_u32x2 v = *(const pa_u32x2*)s;
            w[0] = v[0];
            w[1] = v[1];
        } else if constexpr (BYTES == 4) {
            w[0] = *(const unsigned*)s;
        } else if constexpr (BYTES == 2) {
            w[0] = *(const unsigned short*)s;
        } else {
            static_assert(BYTES == 1, "run");
            w[0] = *s;
        }
    }
    // number i as fp32 (8 bits: the integer)
    __device__ __forceinline__ float get(int i) const {
        if (TYPE == KV_F32) return __uint_as_float(w[i]);
        if (TYPE == KV_BF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        return (float)((int)(w[i / 4] << (24 - 8 * (i & 3))) >> 24);
    }
};

// ------------------------------------------------------------------ few rows
// 16 rows of one cached head over one split of its keys, four waves; wave w
// takes the key blocks (32 keys) w, w + 4, ...  of the split, straight from
// memory into the matrix operands (v_mfma_f32_16x16x32_bf16, lane l = 16 kq +
// i: A[i][8 kq + j], B[8 kq + j][i], result D[4 kq + r][i]); the order of the
// contraction is free as long as both operands keep to it, so each lane reads
// what lies together:
//   S^T = K Q^T: the lane's keys are row i of the block's two 16-key groups,
//     its numbers the HD / 4 from kq HD / 4 on;
//   O^T += V^T P^T: the result S^T[key 4 kq + r][row i] is already operand B of
//     keys {4 kq + r, 16 + 4 kq + r}; operand A is those eight keys' numbers i
//     HD / 16 + e, one product for each e.
// A row (query) is one lane column throughout, so its maximum and rescaling
// need two exchanges (lanes 16 and 32 away) and no broadcast.
template <int HD, int TYPE>
__device__ __forceinline__ void paged_attn_few(const PagedAttnParams& p) {
    constexpr int KD = HD / 4, VD = HD / 16, NS = (KD + 7) / 8;
    constexpr int NT = TYPE == KV_F32 ? 3 : 1;
    __shared__ __attribute__((aligned(16))) float wo[4][16][HD + 4];
    __shared__ float wm[4][16], wl[4][16];
    __shared__ int bad[HD];          // the first key whose number d is not finite, of blocks not all rows see whole
    const PagedKv& c = p.kv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, kq = lane >> 4;
    const int G = p.heads / c.kv_heads;
    const int tiles = (p.max_q * G + 15) >> 4;
    int x = blockIdx.x;
    const int tile = x % tiles;
    x /= tiles;
    const int h = x % c.kv_heads, seq = x / c.kv_heads;
    int q0 = c.q_start[seq], q1 = c.q_start[seq + 1];
    const int q1_said = q1;
    q0 = q0 < 0 ? 0 : q0;
    q1 = q1 > c.rows ? c.rows : q1;
    const int qn = q1 - q0 < p.max_q ? q1 - q0 : p.max_q;
    const int R = qn * G, r0 = tile * 16;
    if (r0 >= R) return;
    const int held = c.kv_len[seq];
    const int keys = held < 0 ? 0 : held > p.max_kv ? p.max_kv : held;
    const int nr = R - r0 < 16 ? R - r0 : 16;
    // keys that a row may see: [0, lim); first, the row's token
    const int tok = (r0 + (i < nr ? i : nr - 1)) / G, grp = (r0 + (i < nr ? i : nr - 1)) - tok * G;
    const int pos0 = held - (q1_said - q0);
    auto limit = [&](int t) {
        const int l = pos0 + t + 1;
        return l < 0 ? 0 : l > keys ? keys : l;
    };
    const int lim = limit(tok);
    const int lim_hi = limit((r0 + nr - 1) / G), lim_lo = limit(r0 / G);
    const int split = blockIdx.y;
    const int c0 = split * p.chunk;
    if (split > 0 && c0 >= lim_hi) return;
    const int c1 = c0 + p.chunk < lim_hi ? c0 + p.chunk : lim_hi;
    for (int d = threadIdx.x; d < HD; d += 256) bad[d] = PA_NONE;
    __syncthreads();

    // operand B of S^T: the row's numbers times scale log2(e)
    pa_bf16x8 qf[NS][3];
    {
        const float* qr = p.q + (long long)(q0 + tok) * p.ldq + (h * G + grp) * HD + kq * KD;
        const float f = p.scale * PA_LOG2E;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                f32x4 t = {0.f, 0.f, 0.f, 0.f};
                if (8 * s + j < KD) t = *(const f32x4*)(qr + 8 * s + j);
#pragma unroll
                for (int e = 0; e < 4; e++) v[j + e] = t[e] * f;
            }
            pa_split<3>(v, qf[s]);
        }
    }
    f32x4 o[VD];
#pragma unroll
    for (int e = 0; e < VD; e++) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    const int* table = c.pages + (long long)seq * c.max_pages;
    const int ps = 1 << c.page_shift;
    // the pool row of key k0's 16-key group (page sizes are multiples of 16),
    // -1 without a page
    auto group_row = [&](int k0) -> long long {
        int at = k0 >> c.page_shift;
        at = at < c.max_pages ? at : c.max_pages - 1;
        const int page = table[at];
        if (page < 0 || page >= c.num_pages) return -1;
        return (((long long)page * c.kv_heads + h) << c.page_shift) + (k0 & (ps - 1));
    };

    for (int b = c0 + 32 * wave; b < c1; b += 128) {
        long long g[2];
        bool ok[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            g[t] = group_row(b + 16 * t);
            ok[t] = g[t] >= 0;
            if (!ok[t]) g[t] = 0;
        }
        PaRun<TYPE, KD> kr[2];
        PaRun<TYPE, VD> vr[2][4];
        f32x4 ks[2], vs[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            kr[t].load(c.k, (g[t] + i) * HD + kq * KD);
            if (TYPE == KV_I8) ks[t] = *(const f32x4*)(c.ks + g[t] + 4 * kq);
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int r = 0; r < 4; r++) vr[t][r].load(c.v, (g[t] + 4 * kq + r) * HD + i * VD);
            if (TYPE == KV_I8) vs[t] = *(const f32x4*)(c.vs + g[t] + 4 * kq);
        }
        f32x4 s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = 0; n < NS; n++) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = 8 * n + j < KD ? kr[t].get(8 * n + j) : 0.f;
                pa_bf16x8 kf[NT];
                pa_split<NT>(v, kf);
                s[t] = pa_mma<NT>(kf, qf[n], s[t]);
            }
            if (TYPE == KV_I8) s[t] *= ks[t];
        }
        const bool whole = ok[0] && ok[1] && b + 32 <= lim_lo;
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (!ok[t] || b + 16 * t + 4 * kq + r >= lim) s[t][r] = -INFINITY;
        }
        float mx = fmaxf(m, fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                  fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))));
        mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
        mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE));
        const float ref = mx == -INFINITY ? 0.f : mx;     // a row that has seen no key yet keeps zeros
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = mx;
        float w[8], sum = 0.f;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float e = __builtin_amdgcn_exp2f(s[t][r] - ref);
                sum += e;
                w[4 * t + r] = TYPE == KV_I8 ? e * vs[t][r] : e;
            }
        l = l * alpha + sum;
        float v[VD][8];
#pragma unroll
        for (int e = 0; e < VD; e++)
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) v[e][4 * t + r] = vr[t][r].get(e);
        if (!whole) {
            // keys no row of the tile sees weigh nothing, whatever lies there;
            // a number that is not finite in a key that some rows see leaves
            // the product and is put into those rows' outputs at the end
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int key = b + 16 * t + 4 * kq + r;
                    const bool none = !ok[t] || key >= lim_hi;
                    const bool poor = TYPE == KV_I8 && !(__builtin_fabsf(vs[t][r]) < INFINITY);
                    if (none || poor) w[4 * t + r] = 0.f;
#pragma unroll
                    for (int e = 0; e < VD; e++) {
                        float& y = v[e][4 * t + r];
                        if (none) y = 0.f;
                        if (!(__builtin_fabsf(y) < INFINITY) || (poor && !none)) {
                            atomicMin(&bad[i * VD + e], key);
                            y = 0.f;
                        }
                    }
                }
        }
        pa_bf16x8 pf[3];
        pa_split<3>(w, pf);
#pragma unroll
        for (int e = 0; e < VD; e++) {
            pa_bf16x8 vf[NT];
            pa_split<NT>(v[e], vf);
            o[e] = pa_mma<NT>(vf, pf, o[e] * alpha);
        }
    }
    // the waves' parts, joined in wave order
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);
    if (kq == 0) {
        wm[wave][i] = m;
        wl[wave][i] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int e = 0; e < VD; e++) wo[wave][i][(4 * kq + r) * VD + e] = o[e][r];
    __syncthreads();
    const bool last = keys <= p.chunk;        // the sequence has one split: no other part to join
    for (int at = threadIdx.x; at < nr * (HD / 4); at += 256) {
        const int r = at / (HD / 4), d = 4 * (at % (HD / 4));
        const int t = (r0 + r) / G, head = h * G + (r0 + r) - t * G;
        float M = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
        const float ref = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float f = __builtin_amdgcn_exp2f(wm[k][r] - ref);
            L += f * wl[k][r];
            a += f * *(const f32x4*)&wo[k][r][d];
        }
        const int row_lim = limit(t);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (bad[d + e] < row_lim) a[e] = __uint_as_float(0x7fc00000u);
        const long long row = q0 + t;
        if (last) {
            if (row_lim > 0 && M != -INFINITY) a /= L;
            *(f32x4*)(p.out + row * p.ldo + head * HD + d) = a;
        } else {
            const long long slot = (row * p.heads + head) * p.splits + split;
            *(f32x4*)(p.part_o + slot * HD + d) = a;
            if (d == 0) {
                p.part_ml[2 * slot] = M;
                p.part_ml[2 * slot + 1] = L;
            }
        }
    }
}

// ------------------------------------------------------------------ join
// out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s over a row's splits, in
// their order; HD / 4 lanes a row.  Sequences of one split are finished already.
template <int HD>
__device__ __forceinline__ void paged_attn_join(const PagedAttnParams& p) {
    constexpr int LPR = HD / 4;
    __shared__ int qs[PAGED_MAX_SEQS + 1];
    const PagedKv& c = p.kv;
    const int per = 256 / LPR;
    const long long at = (long long)blockIdx.x * per + threadIdx.x / LPR;
    const int d = 4 * (threadIdx.x % LPR);
    paged_stage_starts(c, qs);
    if (at >= (long long)c.rows * p.heads) return;
    const int row = (int)(at / p.heads), head = (int)(at - (long long)row * p.heads);
    const int seq = paged_seq_of(qs, c.n, row);
    if (seq >= c.n || row - qs[seq] >= p.max_q) return;
    const int held = c.kv_len[seq];
    const int keys = held < 0 ? 0 : held > p.max_kv ? p.max_kv : held;
    if (keys <= p.chunk) return;
    int lim = held - (c.q_start[seq + 1] - row) + 1;
    lim = lim < 0 ? 0 : lim > keys ? keys : lim;
    const int ns = (lim + p.chunk - 1) / p.chunk;
    const long long slot = at * p.splits;
    float m = -INFINITY;
    for (int s = 0; s < ns; s++) m = fmaxf(m, p.part_ml[2 * (slot + s)]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < ns; s++) {
        const float f = __builtin_amdgcn_exp2f(p.part_ml[2 * (slot + s)] - ref);
        l += f * p.part_ml[2 * (slot + s) + 1];
        a += f * *(const f32x4*)(p.part_o + (slot + s) * HD + d);
    }
    if (m != -INFINITY) a /= l;
    *(f32x4*)(p.out + (long long)row * p.ldo + head * HD + d) = a;
}

#define PA_KERNELS(HD, NAME, TYPE)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) k_paged_attn_few_hd##HD##_##NAME(PagedAttnParams p) {     \
        paged_attn_few<HD, TYPE>(p);                                                                            \
    }
#define PA_TYPES(HD)                                                                                            \
    PA_KERNELS(HD, f32, KV_F32)                                                                                 \
    PA_KERNELS(HD, bf16, KV_BF16)                                                                               \
    PA_KERNELS(HD, i8, KV_I8)                                                                                   \
    extern "C" __global__ void __launch_bounds__(256) k_paged_attn_join_hd##HD(PagedAttnParams p) {             \
        paged_attn_join<HD>(p);                                                                                 \
    }
PA_TYPES(16)
PA_TYPES(32)
PA_TYPES(64)
PA_TYPES(128)
