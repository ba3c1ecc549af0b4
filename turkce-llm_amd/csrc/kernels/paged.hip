// paged.hip -- a paged K/V cache: its places, and the kernels that write new
// tokens into it and read cached ones back.
//
// A cache is a pool of pages of [kv_heads][page_size][head_dim] numbers, k and
// v apart; token t of a sequence is row t % page_size of its page t /
// page_size.  Every (page, head) block is contiguous, so the attention of one
// head streams whole blocks, and consecutive new tokens of a head are written
// to consecutive rows.
#include "common.h"
#include "../kernel_params.h"

#define PAGED_MAX_SEQS 4096
#define PAGED_SCALE_MIN 0x1p-126f               // no quotient by zero or by a denormal
#define PAGED_SCALE_MAX (8454659.0f * 0x1p98f)  // the largest s with 127 s finite in fp32

enum { KV_F32 = 0, KV_BF16 = 1, KV_I8 = 2 };

typedef float pg_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 pg_bf16x2 __attribute__((ext_vector_type(2)));

// q_start into LDS (n + 1 entries, kept within [0, rows]), whole workgroup.
__device__ __forceinline__ void paged_stage_starts(const PagedKv& c, int* qs) {
    for (int i = threadIdx.x; i <= c.n; i += blockDim.x) {
        const int v = c.q_start[i];
        qs[i] = v < 0 ? 0 : v > c.rows ? c.rows : v;
    }
    __syncthreads();
}

// The sequence that holds `row`: the number of sequences that end at or before
// it; c.n for rows behind the last one.  (In [0, n] whatever qs holds.)
__device__ __forceinline__ int paged_seq_of(const int* qs, int n, int row) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (qs[mid + 1] <= row) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// The tokens sequence seq holds, within [0, 2^30], all that pages can hold: no
// position formed from it and from rows leaves 32 bits.
__device__ __forceinline__ int paged_held(const PagedKv& c, int seq) {
    const int v = c.kv_len[seq];
    return v < 0 ? 0 : v > 1 << 30 ? 1 << 30 : v;
}

// The pool row of (sequence, position, head), or -1 where the position has no
// page.  page_size <= 2^16 and kv_heads <= 2^10: the product is formed in 64 bits.
__device__ __forceinline__ long long paged_place(const PagedKv& c, int seq, int pos, int head) {
    if (pos < 0 || (pos >> c.page_shift) >= c.max_pages) return -1;
    const int page = c.pages[(long long)seq * c.max_pages + (pos >> c.page_shift)];
    if (page < 0 || page >= c.num_pages) return -1;
    return ((((long long)page * c.kv_heads + head) << c.page_shift) + (pos & ((1 << c.page_shift) - 1)));
}

// ------------------------------------------------------------------ append
// y0 = x0 cos - x1 sin, y1 = x0 sin + x1 cos.  The products of fp32 numbers are
// exact in 64 bits, so each result is the exact value rounded to 53 bits and
// then once to fp32: the same bits in any order of operations, which the 8-bit
// form needs (a last-bit difference next to a step's border is a whole step).
// The 64-bit arithmetic is hidden behind the memory.
__device__ __forceinline__ void paged_turn(float& x0, float& x1, double c, double s) {
    const double a = x0, b = x1;
    x0 = (float)(a * c - b * s);
    x1 = (float)(a * s + b * c);
}

// The angles of lane c4's numbers (columns 4 c4 .. + 3 of a head) at `pos`, in
// 64 bits: two pairs' in the interleaved layout, four in the half layout, whose
// columns i and i + rot / 2 share row i of the tables.
struct PagedAngles {
    double c[4], s[4];
    __device__ __forceinline__ void load(const KvAppendParams& p, int pos, int c4) {
#pragma unroll
        for (int e = 0; e < 4; e++) c[e] = s[e] = 0;
        if (!p.rot) return;
        const int far = p.rot >> 3;
        const long long t = (long long)pos * (p.rot >> 1) + (p.rot_half ? 4 * (c4 < far ? c4 : c4 - far) : 2 * c4);
        if (p.rot_half) {
            const f32x4 x = *(const f32x4*)(p.cos_t + t), y = *(const f32x4*)(p.sin_t + t);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                c[e] = x[e];
                s[e] = y[e];
            }
        } else {
            const pg_f32x2 x = *(const pg_f32x2*)(p.cos_t + t), y = *(const pg_f32x2*)(p.sin_t + t);
            c[0] = x[0]; c[1] = x[1];
            s[0] = y[0]; s[1] = y[1];
        }
    }
};

// Four numbers turned.  Half layout: a column's partner is rot / 2 away, in the
// lane rot / 8 away (rot % 8 == 0), fetched by a shuffle in which the whole wave
// takes part.
__device__ __forceinline__ f32x4 paged_rope(const KvAppendParams& p, f32x4 x, const PagedAngles& t, int c4, bool turn) {
    if (!p.rot_half) {
        float a = x[0], b = x[1], d = x[2], e = x[3];
        paged_turn(a, b, t.c[0], t.s[0]);
        paged_turn(d, e, t.c[1], t.s[1]);
        return turn ? f32x4{a, b, d, e} : x;
    }
    const int far = p.rot >> 3, lane = threadIdx.x & 63;
    const bool low = c4 < far, in = 4 * c4 < p.rot;
    const int from = !in ? lane : low ? lane + far : lane - far;
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = __shfl(x[e], from, WAVE);
    if (turn)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            // low columns: x cos - y sin; high ones: y sin + x cos
            const double xd = x[e], yd = y[e];
            x[e] = (float)(low ? xd * t.c[e] - yd * t.s[e] : yd * t.s[e] + xd * t.c[e]);
        }
    return x;
}

// x (4 numbers of a row of LPR lanes) to the cache row `place`.  8 bits: the
// row's largest magnitude as an integer maximum of the bit patterns (NaN above
// infinity above every number), s = amax / 127 and x / s as correctly rounded
// quotients, so that the stored integers are the definition's.
template <int HD, int TYPE>
__device__ __forceinline__ void paged_store(void* pool, float* scales, long long place, f32x4 x, int c4, bool ok) {
    constexpr int LPR = HD / 4;
    if (TYPE == KV_F32) {
        if (ok) *(f32x4*)((float*)pool + place * HD + 4 * c4) = x;
    } else if (TYPE == KV_BF16) {
        uint2 w;
        w.x = __builtin_bit_cast(unsigned, __builtin_convertvector((pg_f32x2{x[0], x[1]}), pg_bf16x2));
        w.y = __builtin_bit_cast(unsigned, __builtin_convertvector((pg_f32x2{x[2], x[3]}), pg_bf16x2));
        if (ok) *(uint2*)((unsigned short*)pool + place * HD + 4 * c4) = w;
    } else {
        unsigned m = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, WAVE));
        const bool finite = m < 0x7f800000u;
        const float s = finite ? fminf(fmaxf(__uint_as_float(m) / 127.0f, PAGED_SCALE_MIN), PAGED_SCALE_MAX)
                               : __uint_as_float(0x7fc00000u);
        unsigned w = 0;
        if (finite)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = (int)fminf(fmaxf(__builtin_rintf(x[e] / s), -127.0f), 127.0f);
                w |= ((unsigned)i & 0xffu) << (8 * e);
            }
        if (ok) {
            *(unsigned*)((unsigned char*)pool + place * HD + 4 * c4) = w;
            if (c4 == 0) scales[place] = s;
        }
    }
}

// U heads (blockIdx.y: of the query heads, then the key heads, then the value
// heads) of 256 / LPR consecutive rows per workgroup, LPR = HD / 4 lanes a row: a
// row's numbers of a head are read as one run, consecutive tokens of a sequence
// write consecutive cache rows, and a row's place and angles are found once for
// its U heads.  All U loads are in flight before the first use.
// Bound by the memory for prompts: 8 x 1024 tokens, 32 + 2 x 8 heads of 128, 8 bits, with
// their read back: 102 us, 441 MB at 4.3 TB/s (a copy: 4.9).  By the launch for
// single tokens: 64 of 6 + 2 x 6 heads of 64 3.7 us.
template <int HD, int TYPE, int U>
__device__ __forceinline__ void kv_append(const KvAppendParams& p) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR;
    __shared__ int qs[PAGED_MAX_SEQS + 1];
    const int c4 = threadIdx.x % LPR;
    const int row = blockIdx.x * RPB + threadIdx.x / LPR;
    const long long at_row = row < p.kv.rows ? row : 0;
    const int kh = p.kv.kv_heads, all = p.heads + 2 * kh;
    f32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int head = blockIdx.y * U + u < all ? blockIdx.y * U + u : all - 1;
        const float* src = head < p.heads ? p.q + at_row * p.ldq + head * HD
                           : head < p.heads + kh ? p.k + at_row * p.ldk + (head - p.heads) * HD
                                                 : p.v + at_row * p.ldv + (head - p.heads - kh) * HD;
        x[u] = *(const f32x4*)(src + 4 * c4);
    }
    paged_stage_starts(p.kv, qs);
    const int seq = row < p.kv.rows ? paged_seq_of(qs, p.kv.n, row) : p.kv.n;
    bool ok = seq < p.kv.n;
    int pos = 0;
    long long place = -1;
    if (ok) {
        pos = paged_held(p.kv, seq) - (qs[seq + 1] - row);
        ok = pos >= 0 && (p.rot == 0 || pos < p.max_pos);
        if (ok) place = paged_place(p.kv, seq, pos, 0);
        ok = ok && place >= 0;
    }
    const bool turn = ok && 4 * c4 < p.rot;
    PagedAngles angles;
    angles.load(p, turn ? pos : 0, turn ? c4 : 0);     // (the tables' first row stands in)
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int head = blockIdx.y * U + u;
        if (head >= all) continue;
        const f32x4 y = head < p.heads + kh && p.rot ? paged_rope(p, x[u], angles, c4, turn) : x[u];
        if (head < p.heads) {
            if (ok) *(f32x4*)(p.q_out + at_row * p.ldqo + head * HD + 4 * c4) = y;
        } else {
            const bool is_k = head < p.heads + kh;
            const int h = head - p.heads - (is_k ? 0 : kh);
            paged_store<HD, TYPE>(is_k ? p.kv.k : p.kv.v, is_k ? p.kv.ks : p.kv.vs,
                                  place + ((long long)h << p.kv.page_shift), y, c4, ok);
        }
    }
}

// ------------------------------------------------------------------ read
// The inverse, in the same order: blockIdx.y over the key heads, then the value
// heads.  Bound by the memory: 16 sequences in bf16 497 MB, 120 us, 4.1 TB/s.
template <int HD, int TYPE, int U>
__device__ __forceinline__ void kv_read(const KvReadParams& p) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR;
    __shared__ int qs[PAGED_MAX_SEQS + 1];
    const int c4 = threadIdx.x % LPR;
    const int row = blockIdx.x * RPB + threadIdx.x / LPR;
    const int kh = p.kv.kv_heads;
    paged_stage_starts(p.kv, qs);
    const int seq = row < p.kv.rows ? paged_seq_of(qs, p.kv.n, row) : p.kv.n;
    if (seq >= p.kv.n) return;
    const long long place = paged_place(p.kv, seq, paged_held(p.kv, seq) - (qs[seq + 1] - row), 0);
    f32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int head = blockIdx.y * U + u < 2 * kh ? blockIdx.y * U + u : 2 * kh - 1;
        const bool is_v = head >= kh;
        const void* pool = is_v ? p.kv.v : p.kv.k;
        // row 0 of the pool stands in for a missing place, and is not used
        const long long at = place < 0 ? 0 : place + ((long long)(is_v ? head - kh : head) << p.kv.page_shift);
        if (TYPE == KV_F32) {
            x[u] = *(const f32x4*)((const float*)pool + at * HD + 4 * c4);
        } else if (TYPE == KV_BF16) {
            const uint2 w = *(const uint2*)((const unsigned short*)pool + at * HD + 4 * c4);
            x[u] = f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                         __uint_as_float(w.y & 0xffff0000u)};
        } else {
            const int w = *(const int*)((const unsigned char*)pool + at * HD + 4 * c4);
            const float s = (is_v ? p.kv.vs : p.kv.ks)[at];
            x[u] = f32x4{(float)(w << 24 >> 24) * s, (float)(w << 16 >> 24) * s, (float)(w << 8 >> 24) * s,
                         (float)(w >> 24) * s};
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int head = blockIdx.y * U + u;
        if (head >= 2 * kh) continue;
        float* dst = head < kh ? p.k_out + (long long)row * p.ld + head * HD : p.v_out + (long long)row * p.ld + (head - kh) * HD;
        *(f32x4*)(dst + 4 * c4) = place < 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : x[u];
    }
}

#define PAGED_KERNELS(HD, NAME, TYPE)                                                                               \
    extern "C" __global__ void __launch_bounds__(256) k_kv_append_hd##HD##_##NAME(KvAppendParams p) {               \
        kv_append<HD, TYPE, 1>(p);                                                                                  \
    }                                                                                                               \
    extern "C" __global__ void __launch_bounds__(256) k_kv_append4_hd##HD##_##NAME(KvAppendParams p) {              \
        kv_append<HD, TYPE, 4>(p);                                                                                  \
    }                                                                                                               \
    extern "C" __global__ void __launch_bounds__(256) k_kv_read_hd##HD##_##NAME(KvReadParams p) {                   \
        kv_read<HD, TYPE, 1>(p);                                                                                    \
    }                                                                                                               \
    extern "C" __global__ void __launch_bounds__(256) k_kv_read4_hd##HD##_##NAME(KvReadParams p) {                  \
        kv_read<HD, TYPE, 4>(p);                                                                                    \
    }
#define PAGED_TYPES(HD)             \
    PAGED_KERNELS(HD, f32, KV_F32)  \
    PAGED_KERNELS(HD, bf16, KV_BF16) \
    PAGED_KERNELS(HD, i8, KV_I8)
PAGED_TYPES(16)
PAGED_TYPES(32)
PAGED_TYPES(64)
PAGED_TYPES(128)
