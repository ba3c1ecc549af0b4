// logits.hip -- rules on logits before a token is picked: penalties for
// repeated tokens, a bias list, a grammar's mask.
//
// One pass: a workgroup takes a slice of WIDTH tokens of one row.  It counts
// the row's tokens that fall into its slice in LDS (integer additions: the
// counts do not depend on their order), places the bias entries there, and
// then reads its slice of the logits once and writes it once.  The history is
// re-read by every slice of its row, from the L2.
// Bound by the memory where the rows are many: 256 rows of 131072 269 MB, 56 us,
// 4.8 TB/s (a copy: 4.9).  64 rows of 31769 with 1024 tokens of history 6.6 us, one
// row 4.8: the launch, and the history's dependent reads.
#include "common.h"
#include "../kernel_params.h"

// One token's rules.  seen: bit 0 set when the token is in the history, the
// rest its count from gen_start on.
__device__ __forceinline__ float rules_one(float x, unsigned seen, float rep, float freq, float pres, int bias_at,
                                           const float* bias) {
    if (seen & 1u) x = x > 0.0f ? x / rep : x * rep;
    if (seen >> 1) x = x - (freq * (float)(seen >> 1) + pres);
    if (bias_at >= 0) x += bias[bias_at];
    return x;
}

template <int WIDTH, bool VEC>
__device__ __forceinline__ void logits_rules(const RulesParams& p) {
    constexpr int THREADS = 256, NV = WIDTH / (4 * THREADS);
    __shared__ __attribute__((aligned(16))) unsigned seen[WIDTH];
    __shared__ __attribute__((aligned(16))) int bias_at[WIDTH];   // the last bias entry of each token, or -1
    const int t = threadIdx.x;
    const long long row = blockIdx.y;
    const int t0 = blockIdx.x * WIDTH;
    const int left = p.vocab - t0 < WIDTH ? p.vocab - t0 : WIDTH;
    const float* z = p.logits + row * p.ld + t0;
    float* o = p.out + row * p.ld_out + t0;
    const float* bias = p.bias + row * p.ld_bias;
    const unsigned* mask = p.mask ? p.mask + row * p.ld_mask : nullptr;

    // the slice's logits and mask words, in flight during the counting
    f32x4 x[NV];
    unsigned bits[NV];
    if (VEC) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = 4 * (t + i * THREADS);
            x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            bits[i] = 0xfu;
            if (at < left) {
                // a row ends at ld, a multiple of 4: the four numbers are in the row's own memory
                x[i] = *(const f32x4*)(z + at);
                if (mask) bits[i] = mask[(t0 + at) >> 5] >> (at & 31);
            }
        }
    }
    if (p.history || p.bias_ids) {
        // the first ids of the row, as far as its memory goes: in flight before
        // their number is known
        constexpr int AHEAD = 4;
        unsigned id[AHEAD], bid = 0;
        const unsigned* hist = p.history + row * p.ld_hist;
        const unsigned* ids = p.bias_ids + row * p.ld_bias;
        int len = 0, gen = 0, n = 0;
        if (p.history) {
#pragma unroll
            for (int a = 0; a < AHEAD; a++) id[a] = t + a * THREADS < p.ld_hist ? hist[t + a * THREADS] : 0;
            len = p.hist_len[row];
            len = len < 0 ? 0 : len > p.ld_hist ? (int)p.ld_hist : len;
            if (p.gen_start) gen = p.gen_start[row];
        }
        if (p.bias_ids) {
            if (t < p.ld_bias) bid = ids[t];
            n = p.n_bias[row];
            n = n < 0 ? 0 : n > p.ld_bias ? (int)p.ld_bias : n;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = 4 * (t + i * THREADS);
            *(uint4*)(seen + at) = make_uint4(0, 0, 0, 0);
            *(int4*)(bias_at + at) = make_int4(-1, -1, -1, -1);
        }
        __syncthreads();
        auto count = [&](unsigned k, int j) {
            k -= (unsigned)t0;
            if (k < (unsigned)left) {
                atomicOr(seen + k, 1u);
                if (j >= gen) atomicAdd(seen + k, 2u);
            }
        };
        if (p.history) {
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
                if (t + a * THREADS < len) count(id[a], t + a * THREADS);
            for (int j = t + AHEAD * THREADS; j < len; j += THREADS) count(hist[j], j);
        }
        auto place = [&](unsigned k, int j) {
            k -= (unsigned)t0;
            if (k < (unsigned)left) atomicMax(bias_at + k, j);
        };
        if (t < n) place(bid, t);
        for (int j = t + THREADS; j < n; j += THREADS) place(ids[j], j);
        __syncthreads();
    }
    const bool edit = p.history || p.bias_ids;
    const float rep = p.history && p.repetition ? p.repetition[row] : 1.0f;
    const float freq = p.history && p.frequency ? p.frequency[row] : 0.0f;
    const float pres = p.history && p.presence ? p.presence[row] : 0.0f;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = 4 * (t + i * THREADS);
            if (at >= left) continue;
            f32x4 y = x[i];
            if (edit) {
                const uint4 s = *(const uint4*)(seen + at);
                const int4 b = *(const int4*)(bias_at + at);
                y[0] = rules_one(y[0], s.x, rep, freq, pres, b.x, bias);
                y[1] = rules_one(y[1], s.y, rep, freq, pres, b.y, bias);
                y[2] = rules_one(y[2], s.z, rep, freq, pres, b.z, bias);
                y[3] = rules_one(y[3], s.w, rep, freq, pres, b.w, bias);
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (!(bits[i] >> e & 1u)) y[e] = -INFINITY;
            if (at + 4 <= left) {
                *(f32x4*)(o + at) = y;
            } else {
                for (int e = 0; at + e < left; e++) o[at + e] = y[e];
            }
        }
    } else {
        for (int at = t; at < left; at += THREADS) {
            float y = z[at];
            if (edit) y = rules_one(y, seen[at], rep, freq, pres, bias_at[at], bias);
            if (mask && !(mask[(t0 + at) >> 5] >> (at & 31) & 1u)) y = -INFINITY;
            o[at] = y;
        }
    }
}

#define RULES_KERNELS(WIDTH)                                                                                   \
    extern "C" __global__ void __launch_bounds__(256) k_logits_rules_##WIDTH(RulesParams p) {                  \
        logits_rules<WIDTH, true>(p);                                                                          \
    }                                                                                                          \
    extern "C" __global__ void __launch_bounds__(256) k_logits_rules_##WIDTH##_u(RulesParams p) {              \
        logits_rules<WIDTH, false>(p);                                                                         \
    }
RULES_KERNELS(1024)
RULES_KERNELS(4096)
