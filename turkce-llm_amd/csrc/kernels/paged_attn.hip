// paged_attn.hip -- causal attention of new tokens over a paged K/V cache.
//
//   out[i] = sum_{t <= pos(i)} w_t v_t / sum w_t,   w_t = 2^(s_t - m),
//   s_t = <q_i, k_t> scale log2(e),  m = max s_t    (online over key blocks)
//
// Products keep fp32's precision on the 16-bit matrix cores.  Few rows (paged_attn_few),
// fp32 and bf16 caches: a number of fp32 is the exact sum of three bf16 numbers
// (its mantissa's upper, middle and lower 8 bits, by truncation, so nothing
// overflows), a bf16 number one; a product of two fp32 numbers takes the six of
// its nine partial products that reach 24 bits, one with a bf16 number three.
// 8-bit caches, and all caches in the many-rows kernel, where the products and
// not the memory bound: two f16 terms and exact powers of two, below.  Sums are
// fp32.  An 8-bit key's scale multiplies its score, an 8-bit value's its weight.
//
// A head's queries: with G query heads to a cached head, rows r = token * G +
// (head in its group) of one cached head are computed together, so its keys
// and values are read once for all of them.
#include "common.h"
#include "../kernel_params.h"

#define PA_LOG2E 1.4426950408889634f
#define PA_NONE 0x7fffffff

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 pa_f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned pa_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned pa_u32x2 __attribute__((ext_vector_type(2)));

#define PA_EXP_MIN 12      // rows below 2^-115 take the power of 2^-115 (their scale is then 2^126)
#define PA_W 10            // a row's weights go up to 2^10, and to 2^14 while its maximum grows (PA_GROW)
#define PA_UP 11           // a row's largest magnitude goes to about 2^11 ..
#define PA_ABOVE 3         // .. and may be up to 2^3 above that
#define PA_BELOW 6         // .. or 2^6 below; together below f16's 2^16
#define PA_FEW_W 13        // the few-rows kernel's weights (8 bits) go up to 2^14
#define PA_GROW 4.0f       // a row's maximum may grow by so much (weights to 2^PA_W 2^4) before its sums are rescaled

__device__ __forceinline__ float pa_pow2(int e) {       // 2^e, e kept in [-126, 127]
    e = e < -126 ? -126 : e > 127 ? 127 : e;
    return __uint_as_float((unsigned)(e + 127) << 23);
}

// q_start[i] within the rows (rows x heads is below 2^31, so is what follows from it).
__device__ __forceinline__ int pa_start(const PagedKv& c, int i) {
    const int v = c.q_start[i];
    return v < 0 ? 0 : v > c.rows ? c.rows : v;
}

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

// Eight 8-bit integers + 128 (offset binary) at bytes `at` of pairs of words
// as f16 numbers times 2^-9: a byte u alone is the f16 denormal 2^-24 u, and 2^15
// of it less 1/4 is (u - 128) 2^-9, all exact: one permutation and one packed
// multiply-add for two numbers.
__device__ __forceinline__ unsigned pa_two_ints(unsigned w0, unsigned w1, int b0, int b1) {
    const unsigned two = __builtin_amdgcn_perm(w1, w0, (unsigned)(b0 | 0x0c00 | (4 + b1) << 16 | 0x0c000000));
    const pa_f16x2 up = {(_Float16)32768.0f, (_Float16)32768.0f}, off = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_bit_cast(unsigned, __builtin_elementwise_fma(__builtin_bit_cast(pa_f16x2, two), up, off));
}

// Eight numbers times `up` as two f16 terms.
__device__ __forceinline__ void pa_split_f16(const float (&x)[8], float up, pa_f16x8 (&t)[2]) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float y = x[j] * up;
        t[0][j] = (_Float16)y;
        t[1][j] = (_Float16)(y - (float)t[0][j]);
    }
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
// Bound by the memory where the contexts are long: 32 single tokens over up to
// 8192, 8 bits, 32 heads on 8 of 128: 69 us with their join, 265 MB at 3.9 TB/s (three bf16
// terms for 8 bits too: 95; keys read a block ahead: no gain, the workgroups of
// a unit hide one another's loads); 64 over up to 1024, fp32, 6 heads of 64: 24 us
// and 5 of join, 110 MB.  By the latency of its two launches where they are
// short: one token over 1000 9.5 us.
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
    // A sequence's tiles next to one another; in a mixed batch, where most
    // sequences have one tile of the grid's four, all first tiles first (next to
    // one another those with work would be on every fourth place and so on few
    // of the units: one prompt of 1024 and 256 single tokens over 500, head_dim
    // 128, 340 us against 169).
    const int most = p.max_q * G < p.few_rows ? p.max_q * G : p.few_rows;
    const int tiles = (most + 15) >> 4, pairs = c.n * c.kv_heads;
    const int tile = p.few_apart ? blockIdx.x / pairs : blockIdx.x % tiles;
    const int pair = p.few_apart ? blockIdx.x % pairs : blockIdx.x / tiles;
    const int h = pair % c.kv_heads, seq = pair / c.kv_heads;
    const int q0 = pa_start(c, seq), q1 = pa_start(c, seq + 1);
    const int qn = q1 - q0 < 0 ? 0 : q1 - q0 < p.max_q ? q1 - q0 : p.max_q;
    const int R = qn * G, r0 = tile * 16;
    if (r0 >= R || R > p.few_rows) return;
    const int held = paged_held(c, seq), keys = held > p.max_kv ? p.max_kv : held;
    const int nr = R - r0 < 16 ? R - r0 : 16;
    // keys that a row may see: [0, lim); first, the row's token
    const int tok = (r0 + (i < nr ? i : nr - 1)) / G, grp = (r0 + (i < nr ? i : nr - 1)) - tok * G;
    const int pos0 = held - (q1 - q0);
    auto limit = [&](int t) {
        const int l = pos0 + t + 1;
        return l < 0 ? 0 : l > keys ? keys : l;
    };
    const int lim = limit(tok);
    const int lim_hi = limit((r0 + nr - 1) / G), lim_lo = limit(r0 / G);
    const int split = blockIdx.y;
    const int c0 = split * p.chunk_few;
    if (split > 0 && c0 >= lim_hi) return;
    const int c1 = c0 + p.chunk_few < lim_hi ? c0 + p.chunk_few : lim_hi;
    for (int d = threadIdx.x; d < HD; d += 256) bad[d] = PA_NONE;
    __syncthreads();

    // operand B of S^T: the row's numbers times scale log2(e); for 8 bits two
    // f16 terms, scaled by the row's own largest magnitude
    pa_bf16x8 qf[NS][3];
    pa_f16x8 qg[NS][2];
    float cq = 1.f;              // 8 bits: a product is so many times the operands' (NaN for a row not finite)
    if constexpr (TYPE == KV_I8) {
        const float* qr = p.q + (long long)(q0 + tok) * p.ldq + (h * G + grp) * HD + kq * KD;
        const float f = p.scale * PA_LOG2E;
        float v[NS][8];
        unsigned big = 0;
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                f32x4 t = {0.f, 0.f, 0.f, 0.f};
                if (8 * s + j < KD) t = *(const f32x4*)(qr + 8 * s + j);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[s][j + e] = t[e] * f;
                    big = max(big, __float_as_uint(v[s][j + e]) & 0x7fffffffu);
                }
            }
        big = max(big, (unsigned)__shfl_xor((int)big, 16, WAVE));
        big = max(big, (unsigned)__shfl_xor((int)big, 32, WAVE));
        const int e = max((int)(big >> 23), 20) - 127 - PA_UP;
        const bool poor = big >= 0x7f800000u;
#pragma unroll
        for (int s = 0; s < NS; s++) pa_split_f16(v[s], poor ? 0.f : pa_pow2(-e), qg[s]);
        cq = poor ? __uint_as_float(0x7fc00000u) : pa_pow2(e + 9);
    } else {
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
    float m = -INFINITY, l = 0.f, mo = -INFINITY;

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
            if constexpr (TYPE == KV_I8) {
#pragma unroll
                for (int n = 0; n < NS; n++) {
                    pa_u32x4 w = {0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (8 * n + 2 * j < KD) {
                            const unsigned y = kr[t].w[2 * n + j / 2] ^ 0x80808080u;
                            w[j] = pa_two_ints(y, y, 2 * (j & 1), 2 * (j & 1) + 1);
                        }
                    const pa_f16x8 kf = __builtin_bit_cast(pa_f16x8, w);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qg[n][1], s[t], 0, 0, 0);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qg[n][0], s[t], 0, 0, 0);
                }
                s[t] = s[t] * cq * ks[t];
            } else
#pragma unroll
            for (int n = 0; n < NS; n++) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = 8 * n + j < KD ? kr[t].get(8 * n + j) : 0.f;
                pa_bf16x8 kf[NT];
                pa_split<NT>(v, kf);
                s[t] = pa_mma<NT>(kf, qf[n], s[t]);
            }
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
        float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = mx;
        float w[8], sum = 0.f;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                w[4 * t + r] = __builtin_amdgcn_exp2f(s[t][r] - ref);
                sum += w[4 * t + r];
            }
        l = l * alpha + sum;
        if constexpr (TYPE == KV_I8) {
            // Weights times values' scales, v_s = mantissa 2^ev: against the
            // maximum mo of s + ev, as in the many-rows kernel, a key at a time.
            float mant[8], so[8], top = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int e = max((int)(__float_as_uint(vs[t][r]) >> 23 & 0xff), 1);
                    mant[4 * t + r] = vs[t][r] * pa_pow2(127 - e);
                    so[4 * t + r] = s[t][r] + (float)(e - 127);
                    top = fmaxf(top, so[4 * t + r]);
                }
            top = fmaxf(top, __shfl_xor(top, 16, WAVE));
            top = fmaxf(mo, fmaxf(top, __shfl_xor(top, 32, WAVE)));
            const float refo = top == -INFINITY ? 0.f : top;
            alpha = __builtin_amdgcn_exp2f(mo - refo);
            mo = top;
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = __builtin_amdgcn_exp2f(so[j] - refo + (float)PA_FEW_W) * mant[j];
        }
        float v[VD][8];
        if constexpr (TYPE != KV_I8)
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
                        if constexpr (TYPE == KV_I8) {
                            if (poor && !none) atomicMin(&bad[i * VD + e], key);
                        } else {
                            float& y = v[e][4 * t + r];
                            if (none) y = 0.f;
                            if (!(__builtin_fabsf(y) < INFINITY)) {
                                atomicMin(&bad[i * VD + e], key);
                                y = 0.f;
                            }
                        }
                    }
                }
        }
        if constexpr (TYPE == KV_I8) {
            pa_f16x8 pf[2];
            pa_split_f16(w, 1.0f, pf);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int n = 0; n < PaRun<TYPE, VD>::NW; n++) vr[t][r].w[n] ^= 0x80808080u;
#pragma unroll
            for (int e = 0; e < VD; e++) {
                pa_u32x4 two;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    two[j] = pa_two_ints(vr[j >> 1][2 * (j & 1)].w[e / 4], vr[j >> 1][2 * (j & 1) + 1].w[e / 4], e & 3, e & 3);
                const pa_f16x8 vf = __builtin_bit_cast(pa_f16x8, two);
                f32x4 y = o[e] * alpha;
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[1], y, 0, 0, 0);
                o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[0], y, 0, 0, 0);
            }
            continue;
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
    if (TYPE == KV_I8 && m != -INFINITY) {
        // to l's reference, in two steps: the power alone may leave fp32's range
        const float step = __builtin_amdgcn_exp2f(0.5f * (mo - (float)(PA_FEW_W - 9) - m));
#pragma unroll
        for (int e = 0; e < VD; e++) o[e] = o[e] * step * step;
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
    const bool last = keys <= p.chunk_few;        // the sequence has one split: no other part to join
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

// ------------------------------------------------------------------ many rows
// A workgroup takes 32 NW rows of one cached head over one split of its keys;
// every wave has 32 rows and all the keys, which pass through LDS in tiles of
// KB, double-buffered: while a tile is computed, the next is in LDS or on its
// way there and the one after it in flight from memory, one barrier a tile.
//
// Products on the f16 matrix cores (v_mfma_f32_32x32x16_f16): fp32 numbers as
// two f16 terms (22 bits and the sign of the second), products of three of
// their four partial products (the fourth is below 2^-22 of it, as fp32's own
// rounding is); bf16 and 8-bit numbers are one f16 number, two partial
// products.  Against three bf16 terms this halves the products for fp32 caches
// and saves a third for the others, and splitting a weight costs 1.5 VALU
// instructions for 5.5.  f16's range is met by powers of two that change
// nothing else:
//   a row of Q is scaled by its own largest magnitude;
//   keys are scaled by one power for a tile, values by another, which puts
//     their rows' largest magnitudes into [2^5, 2^15) (two terms are good to
//     22 bits of a number and to 2^-25: 30 bits of its row's largest at least);
//   with V' = 2^-ev V a second running maximum mo is kept, of s + ev: weights
//     2^(s + ev - mo + 10) are small against the largest contribution to the
//     row, not against the largest weight; their sum is taken back to m.  Both
//     maxima are followed only when a row outgrows its own by 2^4 (weights to
//     2^14), which saves most rescalings.
// The powers of a tile are those of the tile before it.  A tile whose rows do
// not fit them (the first one, or rows of very different magnitude next to one
// another) is taken again by classes of keys that fit one pair of powers,
// largest first, the others masked; the last pair stays.  Numbers that are not
// finite leave the products: the first such key of each column of V, and of
// K, is kept, and rows that see it get NaN at the end.
//
// S^T = K Q^T puts a row into a lane's column, as in attention.hip, and the
// exponentiated result is operand B of O^T += V^T P^T as it is: registers 8 u
// .. 8 u + 7 of lane half h are the keys 16 u + 8 a + 4 h + c (a < 2, c < 4).
// Bound by the matrix products and the exponentials' VALU work (38% and about
// half of the cycles) of the two waves that a SIMD's registers hold, which
// overlap in part: 2048 tokens over 16384 in bf16, 32 heads on 8 of 128: 1.1 ms, 465
// TF/s of the mathematics and 930 of f16 products (a large f16 product: 1149); 8 prompts of
// 1024, fp32, 6 heads of 64: 46 us and 4 of join, a unit's 8 tiles at 4.5 us and its
// start.  256 rows (eight waves of 32) share each staged tile: 128 rows in four
// waves, two workgroups a unit, staged everything twice and were slower.
// V^T is read from V's own rows by ds_read_b64_tr_b16: of 16 lanes, lanes 4 e ..
// 4 e + 3 address 16 numbers of row e, and lane j receives number j of rows 0 .. 3.
typedef unsigned short pa_u16x2 __attribute__((ext_vector_type(2)));
typedef short pa_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) pa_s16x4 pa_lds_s16x4;

// Maximum over the N lanes (a power of two up to 16) that share a row.
template <int N>
__device__ __forceinline__ unsigned pa_row_max(unsigned v) {
    if (N >= 2) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));    // lane ^ 1
    if (N >= 4) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));    // lane ^ 2
    if (N >= 8) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));   // 7 - lane of 8
    if (N >= 16) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));  // 15 - lane of 16
    return v;
}

__device__ __forceinline__ int pa_wave_max(int v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = max(v, __shfl_xor(v, o, WAVE));
    return v;
}

// Row tiles of a sequence in this kernel: none where the few-rows kernel takes it.
template <int NW>
__device__ __forceinline__ int pa_tiles_of(const PagedAttnParams& p, int seq) {
    const int q = pa_start(p.kv, seq + 1) - pa_start(p.kv, seq);
    const int R = (q < 0 ? 0 : q < p.max_q ? q : p.max_q) * (p.heads / p.kv.kv_heads);
    return R <= p.few_rows ? 0 : (R + 32 * NW - 1) / (32 * NW);
}

// One row tile of one sequence and head.
template <int HD, int TYPE, int NW, int KB>
__device__ __forceinline__ void paged_attn_tile(const PagedAttnParams& p, int h, int seq, int tile, int (&kbad)[64]) {
    constexpr int THREADS = 64 * NW, NT = TYPE == KV_F32 ? 2 : 1;
    constexpr int CPR = HD / 8, CH = KB * CPR, CK = (CH + THREADS - 1) / THREADS;   // 8-number chunks
    constexpr int NS = HD / 16, DB = (HD + 31) / 32, KT = KB / 32;
    static_assert(KB <= 64 && CH % 64 == 0 && (CH % THREADS == 0 || CH < THREADS), "chunks of whole waves");
    constexpr int KLD = HD * 2 + 16;            // bytes of a K row: 16 more keep eight rows' chunks on different banks
    constexpr int KTERM = KB * KLD, VTERM = KB * HD * 2, BUF = NT * (KTERM + VTERM);
    __shared__ __attribute__((aligned(16))) char tbuf[2 * BUF];   // two buffers of K terms, then V terms
    __shared__ __attribute__((aligned(16))) float ksc[TYPE == KV_I8 ? 2 : 1][KB], vsc[TYPE == KV_I8 ? 2 : 1][KB];
    __shared__ int misfit[2], lek[KB], lev[KB];
    __shared__ __attribute__((aligned(16))) int bad[HD];
    const PagedKv& c = p.kv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int G = p.heads / c.kv_heads;
    const int q0 = pa_start(c, seq), q1 = pa_start(c, seq + 1);
    const int qn = q1 - q0 < 0 ? 0 : q1 - q0 < p.max_q ? q1 - q0 : p.max_q;
    const int R = qn * G, r0 = tile * 32 * NW;
    if (r0 >= R || R <= p.few_rows) return;
    const int held = paged_held(c, seq), keys = held > p.max_kv ? p.max_kv : held;
    const int nr = R - r0 < 32 * NW ? R - r0 : 32 * NW;
    const int pos0 = held - (q1 - q0);
    auto limit = [&](int t) {
        const int l = pos0 + t + 1;
        return l < 0 ? 0 : l > keys ? keys : l;
    };
    const int lim_hi = limit((r0 + nr - 1) / G);
    const int split = blockIdx.y, c0 = split * p.chunk_tile;
    if (split > 0 && c0 >= lim_hi) return;
    const int c1 = c0 + p.chunk_tile < lim_hi ? c0 + p.chunk_tile : lim_hi;
    // this lane's row, and the keys that the wave's rows see
    const int w0 = r0 + 32 * wave, w1 = (w0 + 31 < R ? w0 + 31 : R - 1);
    const int row = w0 + (lane & 31) < R ? w0 + (lane & 31) : R - 1;
    const int tok = row / G, head = h * G + row - tok * G;
    const int lim = limit(tok);
    const bool busy = w0 < R;
    const int wave_lo = busy ? limit(w0 / G) : 0, wave_hi = busy ? limit(w1 / G) : 0;

    if (threadIdx.x < 2) misfit[threadIdx.x] = -1;
    if (threadIdx.x < 64) kbad[threadIdx.x] = PA_NONE;
    for (int d = threadIdx.x; d < HD; d += THREADS) bad[d] = PA_NONE;

    // operand B of S^T: the row's numbers times scale log2(e), two f16 terms
    pa_f16x8 qh[NS], ql[NS];
    int qe;                                  // the row's numbers are its f16 numbers times 2^qe
    bool qpoor;
    {
        const float* qr = p.q + (long long)(q0 + tok) * p.ldq + head * HD + 8 * half;
        const float f = p.scale * PA_LOG2E;
        f32x4 v[NS][2];
        unsigned m = 0;
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                v[s][j] = *(const f32x4*)(qr + 16 * s + 4 * j) * f;
#pragma unroll
                for (int e = 0; e < 4; e++) m = max(m, __float_as_uint(v[s][j][e]) & 0x7fffffffu);
            }
        m = max(m, (unsigned)__shfl_xor((int)m, 32, WAVE));
        qpoor = m >= 0x7f800000u;
        int e = (int)(m >> 23);
        e = e < 20 ? 20 : e;
        qe = e - 127 - PA_UP;
        const float up = qpoor ? 0.f : pa_pow2(-qe);
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = qpoor ? 0.f : v[s][j / 4][j % 4] * up;
                const _Float16 hi = (_Float16)y;
                qh[s][j] = hi;
                ql[s][j] = (_Float16)(y - (float)hi);
            }
    }
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.f;
    float m = -INFINITY, l = 0.f, mo = -INFINITY;   // maxima of s (l's reference) and of s + ev (o's)

    // ---- tiles: chunk i of a thread is numbers 8 cc .. + 7 of key ckey(i)
    const int* table = c.pages + (long long)seq * c.max_pages;
    const int cc = threadIdx.x % CPR;
    auto ckey = [&](int i) { return (int)(threadIdx.x + i * THREADS) / CPR; };
    const bool stages = CH >= THREADS || threadIdx.x < CH;
    auto page_of = [&](int key) {
        const int at = key >> c.page_shift;
        return table[at < c.max_pages ? at : c.max_pages - 1];
    };
    // the pool row of a key, or -1 where it is not held or not seen
    auto place_of = [&](int key, int page) -> long long {
        if (key >= c1 || page < 0 || page >= c.num_pages) return -1;
        return (((long long)page * c.kv_heads + h) << c.page_shift) + (key & ((1 << c.page_shift) - 1));
    };
    struct Raw {
        PaRun<TYPE, 8> k, v;
        float ks, vs;
        bool in;
    };
    auto load = [&](Raw& r, long long place) {
        r.in = place >= 0;
        const long long at = r.in ? place : 0;
        r.k.load(c.k, at * HD + 8 * cc);
        r.v.load(c.v, at * HD + 8 * cc);
        if (TYPE == KV_I8) {
            r.ks = c.ks[at];
            r.vs = c.vs[at];
        }
    };
    int EK = 128, EV = TYPE == KV_I8 ? 124 : 128;   // powers for rows with numbers up to 4 (scales up to 2^-2)
    // Eight numbers: the bits of their row's largest magnitude (fp32's, with
    // zeros below its exponent for bf16).  What is not finite becomes 0 and is
    // noted (K: the key, by lane; V: the key, by column).
    auto largest = [&](PaRun<TYPE, 8>& run, bool is_k, int key) -> unsigned {
        unsigned big = 0;
        if constexpr (TYPE == KV_F32) {
#pragma unroll
            for (int e = 0; e < 8; e++) big = max(big, run.w[e] & 0x7fffffffu);
        } else if constexpr (TYPE == KV_BF16) {
            pa_u16x2 two = __builtin_bit_cast(pa_u16x2, run.w[0] & 0x7fff7fffu);
#pragma unroll
            for (int e = 1; e < 4; e++)
                two = __builtin_elementwise_max(two, __builtin_bit_cast(pa_u16x2, run.w[e] & 0x7fff7fffu));
            const unsigned w = __builtin_bit_cast(unsigned, two);
            big = max(w & 0xffff0000u, w << 16);
        }
        if (TYPE != KV_I8 && big >= 0x7f800000u) {
            big = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const unsigned y = __float_as_uint(run.get(e)) & 0x7fffffffu;
                if (y >= 0x7f800000u) {
                    atomicMin(is_k ? &kbad[lane] : &bad[8 * cc + e], key);
                    if (TYPE == KV_F32) run.w[e] = 0;
                    if (TYPE == KV_BF16) run.w[e / 2] &= e & 1 ? 0xffffu : 0xffff0000u;
                } else {
                    big = max(big, y);
                }
            }
        }
        return pa_row_max<CPR>(big);
    };
    // a row of zeros in K fits any power; in V it has the least one, so that a
    // large weight on it does not stand before the others' contributions
    auto exponent = [](unsigned big) { return max((int)(big >> 23), PA_EXP_MIN); };
    // 8-bit scales: what is not finite as above
    auto scale_of = [&](float s, bool is_k, int key) -> float {
        if ((__float_as_uint(s) & 0x7fffffffu) < 0x7f800000u) return s;
#pragma unroll
        for (int e = 0; e < (is_k ? 1 : 8); e++) atomicMin(is_k ? &kbad[lane] : &bad[8 * cc + e], key);
        return 0.f;
    };
    // eight numbers times `up` as f16 terms into LDS, `gap` bytes apart
    auto terms = [&](const PaRun<TYPE, 8>& run, float up, char* to, int gap) {
        if constexpr (TYPE == KV_I8) {
            // byte u of an integer + 128 under 0x64: 1024 + u in f16; less 1152
            pa_u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const unsigned two = __builtin_amdgcn_perm(0x64646464u, run.w[i / 2] ^ 0x80808080u,
                                                           i & 1 ? 0x04030402u : 0x04010400u);
                const pa_f16x2 y = __builtin_bit_cast(pa_f16x2, two) - (pa_f16x2){(_Float16)1152.0f, (_Float16)1152.0f};
                w[i] = __builtin_bit_cast(unsigned, y);
            }
            *(pa_u32x4*)to = w;
        } else {
            pa_f16x8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                hi[e] = (_Float16)(run.get(e) * up);
                if (NT == 2) lo[e] = (_Float16)__builtin_fmaf(run.get(e), up, -(float)hi[e]);
            }
            *(pa_u32x4*)to = __builtin_bit_cast(pa_u32x4, hi);
            if (NT == 2) *(pa_u32x4*)(to + gap) = __builtin_bit_cast(pa_u32x4, lo);
        }
    };
    // one chunk into LDS under the current powers; whether its rows fit them
    auto stage = [&](Raw& r, bool in, int buf, int kk, int key) -> bool {
        if (!in) {
#pragma unroll
            for (int i = 0; i < PaRun<TYPE, 8>::NW; i++) r.k.w[i] = r.v.w[i] = 0;     // 8 bits: scales of 0 too
        }
        bool fits;
        float uk = 1.f, uv = 1.f;
        if (TYPE == KV_I8) {
            const float s = in ? scale_of(r.ks, true, key) : 0.f, t = in ? scale_of(r.vs, false, key) : 0.f;
            const int e = exponent(__float_as_uint(t) & 0x7fffffffu);
            fits = !in || (e <= EV && e >= EV - PA_BELOW);
            if (cc == 0) {
                ksc[buf][kk] = s;
                vsc[buf][kk] = t * pa_pow2(127 - EV);
            }
        } else {
            const unsigned bk = largest(r.k, true, key), bv = largest(r.v, false, key);
            const int a = exponent(bk), b = exponent(bv);
            fits = (bk == 0 || (a <= EK + PA_ABOVE && a >= EK - PA_BELOW)) &&
                   (!in || (b <= EV + PA_ABOVE && b >= EV - PA_BELOW));
            uk = pa_pow2(PA_UP + 127 - EK);
            uv = pa_pow2(PA_UP + 127 - EV);
        }
        // V rows of 128 bytes or more: odd rows have their 64-byte halves
        // exchanged, so that the transposing reads of four rows meet no bank twice
        const int swv = CPR >= 8 ? (kk & 1) << 2 : 0;
        char* at = tbuf + buf * BUF;
        terms(r.k, uk, at + kk * KLD + 16 * cc, KTERM);
        terms(r.v, uv, at + NT * KTERM + kk * HD * 2 + 16 * (cc ^ swv), VTERM);
        return fits;
    };
    // The keys of a tile that have a place and are seen by some row, from the
    // pages of its 16-key groups that lanes 0 .. KB / 16 - 1 hold.  (Read with
    // the vector loads: a scalar load in flight would make every wait for an
    // LDS read wait for it too.)
    auto live_keys = [&](int b, int page) -> unsigned long long {
        const unsigned groups = (unsigned)__ballot(page >= 0 && page < c.num_pages);
        unsigned long long live = 0;
#pragma unroll
        for (int g = 0; g < KB / 16; g++)
            if (groups >> g & 1) live |= 0xffffull << (16 * g);
        const int left = c1 - b;
        return left >= 64 ? live : live & ((1ull << (left > 0 ? left : 0)) - 1);
    };

    // ---- one tile of LDS into this wave's rows, 32 keys at a time: the score
    // products of the next 32 keys run beside the exponentials of these
    auto compute = [&](int buf, int b, unsigned long long live) {
        constexpr unsigned long long ALL = KB == 64 ? ~0ull : (1ull << (KB & 63)) - 1;
        const char* kt = tbuf + buf * BUF + (lane & 31) * KLD + 16 * half;
        const int i = lane & 15, p_ = CPR >= 8 ? (i >> 2) & 1 : 0;
        const int dims = (16 * ((lane >> 4) & 1) + 4 * (i & 3)) & (HD - 1);
        const char* vt = tbuf + buf * BUF + NT * KTERM + (4 * half + (i >> 2)) * HD * 2 + dims * 2;
        const float cu = pa_pow2(qe + (TYPE == KV_I8 ? 0 : EK - 127 - PA_UP));
        const float ev = (float)(EV - 127 - (TYPE == KV_I8 ? 0 : PA_UP));
        float minus = -1.0f;
        asm("" : "+s"(minus));      // kept a factor: v_fma_mix takes the f16 term as it is
        auto scores = [&](int t, f32x16& s) {
            constexpr int AHEAD = NS < 4 ? NS : HD == 128 ? 2 : 4;      // operands of so many products ahead
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = 0.f;
#pragma unroll
            for (int n0 = 0; n0 < NS; n0 += AHEAD) {
                pa_f16x8 kf[AHEAD][NT];
#pragma unroll
                for (int n = 0; n < AHEAD; n++)
#pragma unroll
                    for (int w = 0; w < NT; w++)
                        kf[n][w] = *(const pa_f16x8*)(kt + w * KTERM + 32 * t * KLD + 32 * (n0 + n));
#pragma unroll
                for (int n = 0; n < AHEAD; n++) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n][0], ql[n0 + n], s, 0, 0, 0);
                    if (NT == 2) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n][NT - 1], qh[n0 + n], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n][0], qh[n0 + n], s, 0, 0, 0);
                }
            }
        };
        f32x16 ss[KT];
        scores(0, ss[0]);
#pragma unroll
        for (int t = 0; t < KT; t++) {
            f32x16& s = ss[t];
            if (TYPE == KV_I8) {
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const f32x4 f = *(const f32x4*)&ksc[buf][32 * t + 8 * g + 4 * half];
#pragma unroll
                    for (int e = 0; e < 4; e++) s[4 * g + e] *= f[e];
                }
            }
            if (live != ALL || b + KB > wave_lo) {
                // bit kk: this lane's key 8 (e / 4) + e % 4 = kk is seen and held
                const int seen = lim - b - 4 * half - 32 * t;
                unsigned held_here = (unsigned)(live >> (32 * t)) >> (4 * half);
                held_here &= seen >= 32 ? ~0u : seen <= 0 ? 0u : (1u << seen) - 1;
                asm("" : "+v"(held_here));      // (the tests below stay in this branch)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (!(held_here >> (8 * (e >> 2) + (e & 3)) & 1)) s[e] = -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; e += 2) top = fmaxf(top, fmaxf(s[e], s[e + 1]));
            {
                const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * cu;
            }
            // The references m and mo follow the maxima only when one of the
            // wave's rows has outgrown its own (a row that has seen no key yet:
            // references of 0, and zeros).
            if (__ballot(top > m + PA_GROW || top + ev > mo + PA_GROW)) {
                const float m_new = fmaxf(m, top), mo_new = fmaxf(mo, top + ev);
                const float alpha = mo_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mo - mo_new);
                l *= m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
                m = m_new;
                mo = mo_new;
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int e = 0; e < 16; e++) o[d][e] *= alpha;
            }
            const float ref = m == -INFINITY ? 0.f : m, refo = mo == -INFINITY ? 0.f : mo;
            // a weight 2^(s - ref) is 2^gap of the same key's 2^(s + ev - refo + W)
            const float off = (float)PA_W + ev - refo, gap = -off - ref;
            float part = 1.0f;
            if (__ballot(gap > 60.0f)) {
                // values so much smaller than another key's that their weights
                // would leave fp32's range beside it: summed on their own
                part = 0.f;
#pragma unroll
                for (int e = 0; e < 16; e++) l += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], cu, -ref));
            }
            if (t + 1 < KT) scores(t + 1, ss[t + 1 < KT ? t + 1 : t]);
            pa_f16x8 ph[2], pl[2];
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 16; e++) {
                s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], cu, off));
                sum[e & 1] += s[e];
            }
            if (TYPE == KV_I8) {
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const f32x4 f = *(const f32x4*)&vsc[buf][32 * t + 8 * g + 4 * half];
#pragma unroll
                    for (int e = 0; e < 4; e++) s[4 * g + e] *= f[e];
                }
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const pa_f16x2 hi = __builtin_bit_cast(pa_f16x2, __builtin_amdgcn_cvt_pkrtz(s[8 * u + j], s[8 * u + j + 1]));
                    ph[u][j] = hi[0];
                    ph[u][j + 1] = hi[1];
                    pl[u][j] = (_Float16)__builtin_fmaf((float)hi[0], minus, s[8 * u + j]);
                    pl[u][j + 1] = (_Float16)__builtin_fmaf((float)hi[1], minus, s[8 * u + j + 1]);
                }
            l = __builtin_fmaf(sum[0] + sum[1], part * __builtin_amdgcn_exp2f(fminf(gap, 100.0f)), l);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int d0 = 0; d0 < DB; d0 += 2) {          // operands of two products ahead
                    pa_f16x8 vf[2][NT];
#pragma unroll
                    for (int d = d0; d < d0 + 2 && d < DB; d++)
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            pa_s16x4 a[2];
#pragma unroll
                            for (int rd = 0; rd < 2; rd++)
                                a[rd] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (pa_lds_s16x4*)(vt + n * VTERM + (32 * t + 16 * u + 8 * rd) * HD * 2 + 64 * (d ^ p_)));
                            vf[d - d0][n] =
                                __builtin_bit_cast(pa_f16x8, __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7));
                        }
#pragma unroll
                    for (int d = d0; d < d0 + 2 && d < DB; d++) {
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d - d0][0], pl[u], o[d], 0, 0, 0);
                        if (NT == 2) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d - d0][NT - 1], ph[u], o[d], 0, 0, 0);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d - d0][0], ph[u], o[d], 0, 0, 0);
                    }
                }
        }
    };

    // ---- the pipeline: tile it in LDS, it + 1 in registers, the pages of it + 2
    const int nt = (c1 - c0 + KB - 1) / KB;
    Raw raw[CK];
    int page[CK];
    auto fetch = [&](int it) {                 // tile it from its pages; the pages of tile it + 1
        const int b = c0 + it * KB;
#pragma unroll
        for (int i = 0; i < CK; i++) {
            load(raw[i], place_of(b + ckey(i), page[i]));
            page[i] = page_of(b + KB + ckey(i));
        }
    };
    auto put = [&](int it) {
        if (!stages) return;
        bool fits = true;
#pragma unroll
        for (int i = 0; i < CK; i++) fits &= stage(raw[i], raw[i].in, it & 1, ckey(i), c0 + it * KB + ckey(i));
        if (!fits) misfit[it & 1] = it;
    };
    if (stages) {
#pragma unroll
        for (int i = 0; i < CK; i++) page[i] = page_of(c0 + ckey(i));
    }
    int group_page = page_of(c0 + 16 * (lane & (KB / 16 - 1)));
    for (int it = -2; it < nt; it++) {
        const int b = c0 + it * KB, buf = it & 1;
        if (it >= 0) {
            const unsigned long long live = live_keys(b, group_page);
            group_page = page_of(b + KB + 16 * (lane & (KB / 16 - 1)));
            const bool classes = misfit[buf] == it;      // the same for every wave, and so are the turns below
            unsigned long long left = live;
            if (classes) {
                if (stages)
#pragma unroll 1
                    for (int i = 0; i < CK; i++) {
                        const int key = b + ckey(i);
                        Raw r;
                        load(r, place_of(key, page_of(key)));
                        int ek = 0, ev = PA_EXP_MIN;
                        if (r.in && TYPE == KV_I8) {
                            ev = exponent(__float_as_uint(scale_of(r.vs, false, key)) & 0x7fffffffu);
                        } else if (r.in) {
                            const unsigned bk = largest(r.k, true, key);
                            ek = bk ? exponent(bk) : 0;
                            ev = exponent(largest(r.v, false, key));
                        }
                        if (cc == 0) {
                            lek[ckey(i)] = ek;
                            lev[ckey(i)] = ev;
                        }
                    }
                __syncthreads();
            }
            do {
                unsigned long long set = left;
                if (classes) {
                    const int k = lane < KB ? lane : 0;
                    const bool in = lane < KB && (left >> k & 1);
                    const int ek = in ? lek[k] : 0, ev = in ? lev[k] : 0;
                    const int mk = pa_wave_max(ek);
                    const bool in_k = in && (ek == 0 || ek >= mk - PA_BELOW);
                    const int mv = pa_wave_max(in_k ? ev : 0);
                    set = __ballot(in_k && ev >= mv - PA_BELOW);
                    if (mk) EK = mk;
                    EV = mv;
                    if (stages)
#pragma unroll 1
                        for (int i = 0; i < CK; i++) {
                            const int key = b + ckey(i);
                            Raw r;
                            load(r, place_of(key, page_of(key)));
                            stage(r, r.in && (set >> ckey(i) & 1), buf, ckey(i), key);
                        }
                    __syncthreads();
                }
                if (b < wave_hi) compute(buf, b, set);
                left &= ~set;
                if (classes) __syncthreads();
            } while (left);
        }
        if (it + 1 >= 0 && it + 1 < nt) put(it + 1);
        if (stages && it + 2 < nt) fetch(it + 2);
        __syncthreads();
    }

    // ---- out, or this split's part
    l += __shfl_xor(l, 32, WAVE);
    int kfirst = kbad[lane];
#pragma unroll
    for (int f = 32; f >= 1; f >>= 1) kfirst = min(kfirst, __shfl_xor(kfirst, f, WAVE));
    if (w0 + (lane & 31) >= R) return;
    const float nan = __uint_as_float(0x7fc00000u);
    const bool poor = (qpoor && m != -INFINITY) || kfirst < lim;
    const bool last = keys <= p.chunk_tile;
    // o to l's reference (in two steps: the power alone may leave fp32's
    // range), and divided where this is the whole sum
    const float step = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(0.5f * (mo - (float)PA_W - m));
    const float inv = step * (last && m != -INFINITY ? 1.0f / l : 1.0f);
    const long long orow = q0 + tok, slot = (orow * p.heads + head) * p.splits + split;
    float* dst = last ? p.out + orow * p.ldo + head * HD : p.part_o + slot * HD;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int d0 = 32 * d + 8 * g + 4 * half;
            if (d0 < HD) {
                const int4 first = *(const int4*)&bad[d0];
                const int fe[4] = {first.x, first.y, first.z, first.w};
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = (poor | (fe[e] < lim)) ? nan : o[d][4 * g + e] * step * inv;
                *(f32x4*)(dst + d0) = v;
            }
        }
    if (!last && half == 0) {
        p.part_ml[2 * slot] = m;
        p.part_ml[2 * slot + 1] = l;
    }
}

// Where all sequences may be as long as the longest (or there is one) the grid
// holds max_q's tiles of each, the last rows, which see the most keys, first.
template <int HD, int TYPE, int NW, int KB>
__device__ __forceinline__ void paged_attn_tile_dense(const PagedAttnParams& p) {
    __shared__ int kbad[64];
    const int tiles = (p.max_q * (p.heads / p.kv.kv_heads) + 32 * NW - 1) / (32 * NW);
    const int x = blockIdx.x / p.kv.kv_heads;
    paged_attn_tile<HD, TYPE, NW, KB>(p, blockIdx.x % p.kv.kv_heads, x % p.kv.n, tiles - 1 - x / p.kv.n, kbad);
}

// In a mixed batch that would be mostly workgroups without work, each a compute
// unit's turn (a prompt of 2048 beside 64 single tokens 204 us, so 94).  There
// the grid holds the tiles that the call's rows make up with
// one sequence at its longest, and a workgroup finds its own among the sequences'
// counts, which its threads add up together; should there be more tiles, the
// workgroups take them in turns.
template <int HD, int TYPE, int NW, int KB>
__device__ __forceinline__ void paged_attn_tile_mixed(const PagedAttnParams& p) {
    const PagedKv& c = p.kv;
    __shared__ int few[64];
    const int h = blockIdx.x % c.kv_heads;
    int j = blockIdx.x / c.kv_heads, more;
    do {
        const int per = (c.n + 64 * NW - 1) / (64 * NW);
        const int s0 = threadIdx.x * per, s1 = s0 + per < c.n ? s0 + per : c.n;
        int own = 0;
        for (int s = s0; s < s1; s++) own += pa_tiles_of<NW>(p, s);
        int upto = own;                                // tiles up to this thread's last sequence
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o, WAVE);
            if ((int)(threadIdx.x & 63) >= o) upto += v;
        }
        if ((threadIdx.x & 63) == 63) few[threadIdx.x >> 6] = upto;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const int v = few[w];
            if (w < (int)(threadIdx.x >> 6)) upto += v;
            total += v;
        }
        if (j >= total) return;                        // the same for all threads
        if (j < upto && j >= upto - own) {
            int left = upto - j, s = s1 - 1, n = pa_tiles_of<NW>(p, s);
            while (left > n) {
                left -= n;
                n = pa_tiles_of<NW>(p, --s);
            }
            few[NW] = s;
            few[NW + 1] = left - 1;
        }
        __syncthreads();
        const int seq = __builtin_amdgcn_readfirstlane(few[NW]), tile = __builtin_amdgcn_readfirstlane(few[NW + 1]);
        j += gridDim.x / c.kv_heads;
        more = __builtin_amdgcn_readfirstlane(total) - j;
        __syncthreads();
        paged_attn_tile<HD, TYPE, NW, KB>(p, h, seq, tile, few);
        __syncthreads();
    } while (more > 0);
}

// ------------------------------------------------------------------ join
// out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s over a row's splits, in
// one order.  Sequences of one split are finished already.
#define PA_MAX_SPLITS 256

// Row `at / heads`, head `at % heads`: the splits that hold a key of the row, -1
// where there is nothing to join.
__device__ __forceinline__ int pa_row_splits(const PagedAttnParams& p, const int* qs, long long at) {
    const PagedKv& c = p.kv;
    if (at >= (long long)c.rows * p.heads) return -1;
    const int row = (int)(at / p.heads), seq = paged_seq_of(qs, c.n, row);
    if (seq >= c.n || row - qs[seq] >= p.max_q) return -1;
    const int held = paged_held(c, seq), keys = held > p.max_kv ? p.max_kv : held;
    const int qn = qs[seq + 1] - qs[seq] < p.max_q ? qs[seq + 1] - qs[seq] : p.max_q;
    const int chunk = qn * (p.heads / c.kv_heads) <= p.few_rows ? p.chunk_few : p.chunk_tile;
    if (keys <= chunk) return -1;
    int lim = held - (qs[seq + 1] - row) + 1;
    lim = lim < 0 ? 0 : lim > keys ? keys : lim;
    const int ns = (lim + chunk - 1) / chunk;
    return ns < p.splits ? ns : p.splits;
}

// A few splits: HD / 4 lanes a row, 256 / (HD / 4) rows a workgroup.
template <int HD>
__device__ __forceinline__ void paged_attn_join(const PagedAttnParams& p) {
    constexpr int LPR = HD / 4;
    __shared__ int qs[PAGED_MAX_SEQS + 1];
    const long long at = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int d = 4 * (threadIdx.x % LPR);
    paged_stage_starts(p.kv, qs);
    const int ns = pa_row_splits(p, qs, at);
    if (ns < 0) return;
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
    *(f32x4*)(p.out + at / p.heads * p.ldo + at % p.heads * HD + d) = a;
}

// Many splits: a wave a row.  Lane s takes the statistics of splits s, s + 64,
// ..; the weights go through LDS to 64 / (HD / 4) groups of lanes, which take
// the splits in turn, two loads in flight each, and are added at the end.
// Measured (one token over 8000 in 32 splits): 35 us with the form above, 14.
template <int HD>
__device__ __forceinline__ void paged_attn_join_long(const PagedAttnParams& p) {
    constexpr int LPR = HD / 4, NG = 64 / LPR;
    __shared__ int qs[PAGED_MAX_SEQS + 1];
    __shared__ float weight[4][PA_MAX_SPLITS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long at = (long long)blockIdx.x * 4 + wave;
    paged_stage_starts(p.kv, qs);
    const int ns = pa_row_splits(p, qs, at);
    if (ns < 0) return;
    const long long slot = at * p.splits;
    float ms[PA_MAX_SPLITS / 64], ls[PA_MAX_SPLITS / 64], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < PA_MAX_SPLITS / 64; i++) {
        const int s = lane + 64 * i;
        ms[i] = s < ns ? p.part_ml[2 * (slot + s)] : -INFINITY;
        ls[i] = s < ns ? p.part_ml[2 * (slot + s) + 1] : 0.f;
        m = fmaxf(m, ms[i]);
    }
    m = wave_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < PA_MAX_SPLITS / 64; i++) {
        const float f = __builtin_amdgcn_exp2f(ms[i] - ref);
        weight[wave][lane + 64 * i] = f;
        l += f * ls[i];
    }
    l = wave_sum(l);
    __builtin_amdgcn_wave_barrier();       // the weights are this wave's own
    const int g = lane / LPR, d = 4 * (lane % LPR);
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    for (int s = g; s < ns; s += 2 * NG) {
        const int s2 = s + NG < ns ? s + NG : s;
        const f32x4 x = *(const f32x4*)(p.part_o + (slot + s) * HD + d);
        const f32x4 y = *(const f32x4*)(p.part_o + (slot + s2) * HD + d);
        a += weight[wave][s] * x;
        if (s + NG < ns) b += weight[wave][s2] * y;
    }
    a += b;
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) a[e] += __shfl_xor(a[e], o, WAVE);
    if (m != -INFINITY) a /= l;
    if (g == 0) *(f32x4*)(p.out + at / p.heads * p.ldo + at % p.heads * HD + d) = a;
}

#define PA_KEYS(HD, TYPE) (HD == 128 && TYPE == KV_F32 ? 32 : 64)      // of a stage
#define PA_KERNELS(HD, NAME, TYPE)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) k_paged_attn_few_hd##HD##_##NAME(PagedAttnParams p) {     \
        paged_attn_few<HD, TYPE>(p);                                                                            \
    }                                                                                                           \
    extern "C" __global__ void __launch_bounds__(512, 2) k_paged_attn_tile_hd##HD##_##NAME(PagedAttnParams p) { \
        paged_attn_tile_dense<HD, TYPE, 8, PA_KEYS(HD, TYPE)>(p);                                               \
    }                                                                                                           \
    extern "C" __global__ void __launch_bounds__(512, 2) k_paged_attn_mixed_hd##HD##_##NAME(PagedAttnParams p) { \
        paged_attn_tile_mixed<HD, TYPE, 8, PA_KEYS(HD, TYPE)>(p);                                               \
    }
#define PA_TYPES(HD)                                                                                            \
    PA_KERNELS(HD, f32, KV_F32)                                                                                 \
    PA_KERNELS(HD, bf16, KV_BF16)                                                                               \
    PA_KERNELS(HD, i8, KV_I8)                                                                                   \
    extern "C" __global__ void __launch_bounds__(256) k_paged_attn_join_hd##HD(PagedAttnParams p) {             \
        paged_attn_join<HD>(p);                                                                                 \
    }                                                                                                           \
    extern "C" __global__ void __launch_bounds__(256) k_paged_attn_join_long_hd##HD(PagedAttnParams p) {        \
        paged_attn_join_long<HD>(p);                                                                            \
    }
PA_TYPES(16)
PA_TYPES(32)
PA_TYPES(64)
PA_TYPES(128)
