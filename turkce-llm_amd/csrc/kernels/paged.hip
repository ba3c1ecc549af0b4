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
__device__ __forceinline__ void paged_turn(float& x0, float& x1, float c, float s) {
    const double a = x0, b = x1, cd = c, sd = s;
    x0 = (float)(a * cd - b * sd);
    x1 = (float)(a * sd + b * cd);
}

// The four numbers of lane c4 (columns 4 c4 .. + 3 of its head) turned by the
// angles at `row` of the tables.  Half layout: a column's partner is rot / 2
// away, in the lane rot / 8 away (rot % 8 == 0), fetched by a shuffle in which
// the whole wave takes part.
__device__ __forceinline__ f32x4 paged_rope(const KvAppendParams& p, f32x4 x, int pos, int c4, bool turn) {
    if (!p.rot_half) {
        if (turn && 4 * c4 < p.rot) {
            const long long t = (long long)pos * (p.rot >> 1) + 2 * c4;
            const pg_f32x2 c = *(const pg_f32x2*)(p.cos_t + t), s = *(const pg_f32x2*)(p.sin_t + t);
            float a = x[0], b = x[1], d = x[2], e = x[3];
            paged_turn(a, b, c[0], s[0]);
            paged_turn(d, e, c[1], s[1]);
            x = f32x4{a, b, d, e};
        }
        return x;
    }
    const int far = p.rot >> 3, lane = threadIdx.x & 63;
    const bool low = c4 < far, in = 4 * c4 < p.rot;
    const int from = !in ? lane : low ? lane + far : lane - far;
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = __shfl(x[e], from, WAVE);
    if (turn && in) {
        const int i = 4 * (low ? c4 : c4 - far);
        const long long t = (long long)pos * (p.rot >> 1) + i;
        const f32x4 c = *(const f32x4*)(p.cos_t + t), s = *(const f32x4*)(p.sin_t + t);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float a = low ? x[e] : y[e], b = low ? y[e] : x[e];
            paged_turn(a, b, c[e], s[e]);
            x[e] = low ? a : b;
        }
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

// One head (blockIdx.y: the query heads, then the key heads, then the value
// heads) of U * 256 / LPR consecutive rows per workgroup, LPR = HD / 4 lanes a
// row: a row's numbers are read as one run, and consecutive tokens of a
// sequence write consecutive cache rows.  All U loads are in flight before the
// first use.
template <int HD, int TYPE, int U>
__device__ __forceinline__ void kv_append(const KvAppendParams& p) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR;
    __shared__ int qs[PAGED_MAX_SEQS + 1];
    const int c4 = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const int head = blockIdx.y;
    const int kh = p.kv.kv_heads;
    const int kind = head < p.heads ? 0 : head < p.heads + kh ? 1 : 2;
    const int h = kind == 0 ? head : kind == 1 ? head - p.heads : head - p.heads - kh;
    const float* src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const long long ld = kind == 0 ? p.ldq : kind == 1 ? p.ldk : p.ldv;
    const int row0 = blockIdx.x * (RPB * U) + sub;
    f32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * RPB;
        x[u] = *(const f32x4*)(src + (long long)(row < p.kv.rows ? row : 0) * ld + h * HD + 4 * c4);
    }
    paged_stage_starts(p.kv, qs);
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * RPB;
        const int seq = row < p.kv.rows ? paged_seq_of(qs, p.kv.n, row) : p.kv.n;
        bool ok = seq < p.kv.n;
        int pos = 0;
        long long place = -1;
        if (ok) {
            pos = p.kv.kv_len[seq] - (qs[seq + 1] - row);
            ok = pos >= 0 && (p.rot == 0 || pos < p.max_pos);
            if (ok) place = paged_place(p.kv, seq, pos, kind == 0 ? 0 : h);
            ok = ok && place >= 0;
        }
        const f32x4 y = kind < 2 && p.rot ? paged_rope(p, x[u], pos, c4, ok) : x[u];
        if (kind == 0) {
            if (ok) *(f32x4*)(p.q_out + (long long)row * p.ldqo + h * HD + 4 * c4) = y;
        } else {
            paged_store<HD, TYPE>(kind == 1 ? p.kv.k : p.kv.v, kind == 1 ? p.kv.ks : p.kv.vs, place, y, c4, ok);
        }
    }
}

// ------------------------------------------------------------------ read
// The inverse, in the same order: blockIdx.y the key heads, then the value
// heads.
template <int HD, int TYPE, int U>
__device__ __forceinline__ void kv_read(const KvReadParams& p) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR;
    __shared__ int qs[PAGED_MAX_SEQS + 1];
    const int c4 = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const bool is_v = (int)blockIdx.y >= p.kv.kv_heads;
    const int h = is_v ? blockIdx.y - p.kv.kv_heads : blockIdx.y;
    const void* pool = is_v ? p.kv.v : p.kv.k;
    const float* scales = is_v ? p.kv.vs : p.kv.ks;
    float* dst = is_v ? p.v_out : p.k_out;
    const int row0 = blockIdx.x * (RPB * U) + sub;
    paged_stage_starts(p.kv, qs);
    long long place[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * RPB;
        const int seq = row < p.kv.rows ? paged_seq_of(qs, p.kv.n, row) : p.kv.n;
        in[u] = seq < p.kv.n;
        place[u] = in[u] ? paged_place(p.kv, seq, p.kv.kv_len[seq] - (qs[seq + 1] - row), h) : -1;
    }
    f32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        // row 0 of the pool stands in for a missing place, and is not used
        const long long at = place[u] < 0 ? 0 : place[u];
        if (TYPE == KV_F32) {
            x[u] = *(const f32x4*)((const float*)pool + at * HD + 4 * c4);
        } else if (TYPE == KV_BF16) {
            const uint2 w = *(const uint2*)((const unsigned short*)pool + at * HD + 4 * c4);
            x[u] = f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                         __uint_as_float(w.y & 0xffff0000u)};
        } else {
            const int w = *(const int*)((const unsigned char*)pool + at * HD + 4 * c4);
            const float s = scales[at];
            x[u] = f32x4{(float)(w << 24 >> 24) * s, (float)(w << 16 >> 24) * s, (float)(w << 8 >> 24) * s,
                         (float)(w >> 24) * s};
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * RPB;
        if (in[u])
            *(f32x4*)(dst + (long long)row * p.ld + h * HD + 4 * c4) = place[u] < 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : x[u];
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
