// attn_tile.h -- the tile arithmetic shared by the attention over whole prompts (prompt.hip) and over the paged
// cache (paged.hip).
//
// Rows.  The query heads of one kv head read the same keys, so they share a tile: row r of a (sequence, kv head) is
// head r % G of token r / G.  A tile of rows starts at a multiple of its height, a sequence of n tokens has n G rows.
//
// Mathematics.  For a row with visible keys 0 .. lim the kernels fold the tokens in once, tile by tile:
//     s_j = q . k_j (f32 accumulation of exact bf16 products),  x_j = c s_j,  c = scale log2(e)
//     m' = max(m, max_j x_j),  l' = 2^(m - m') l + sum_j 2^(x_j - m'),  o' = 2^(m - m') o + sum_j 2^(x_j - m') v_j
// and end with o / l and the base-2 log-sum-exp m + log2 l.  m need not be the maximum, only near or above it: the weights
// are made with the m there is, and only where a lane's share of a tile's weights sums to more than 1024 (or the row has seen
// nothing yet) is the maximum looked for, m moved, o and l scaled and the weights made again.  Larger weights change neither the
// relative precision of f32 sums nor that of a bf16 weight, and most tiles cost no maximum and no scaling (3 % at 32 768 tokens).
// They cost range: over n keys l stays below 128 n (2048 a tile of 32 keys or more; 2 n of one tile), so o is finite for
// |v| < 2^120 / n.  m is rounded to f32, which moves a weight by 2^+-1 at most while |x| < 2^25.
// m, l, o are f32; the weights 2^(x - m) are rounded to bf16 once, for the second matrix product (relative error 2^-8 each at
// most, as the output's own rounding); l sums them unrounded.
//
// Lanes.  Both products are v_mfma_f32_32x32x16_bf16.  The first computes S^T = K Q^T: lane l holds column
// (row of q) l % 32 and, of 32 tokens, the 16 with (t >> 2) & 1 == l / 32.  So a row's maximum and sum are sums over a
// lane's own registers and one exchange with lane l ^ 32, and its weights are, as they lie, the right-hand operand of
// O^T = V^T P^T: the product's 16 inner indices may be any 16 tokens in any order as long as both operands agree, here
// inner index 8 (l / 32) + j is token 8 (j / 4) + 4 (l / 32) + j % 4.  V^T comes out of the row-major tile in LDS
// through ds_read_b64_tr_b16 (16 lanes read a 4 x 16 block and each gets a column of it).
//
// LDS.  Tile rows are 2 D bytes, 16-byte chunks.  Slot p of row r holds chunk p ^ key_swizzle(r) / p ^ value_swizzle(r): the 32
// rows that one K read touches then lie in all banks evenly, and so do the 4 rows x 64 bytes of a transposed V read.
// (The DMA into LDS writes lane after lane: the permutation is made on the global addresses.)
#pragma once
#include "common.h"

namespace mp {

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

#define MP_LDS __attribute__((address_space(3)))
#define MP_GLOBAL __attribute__((address_space(1)))

constexpr int TILE_TOKENS = 64;         // tokens staged at a time
constexpr float NEG_INF = -__builtin_inff();
constexpr float LAZY_SUM = 1024.f;       // see above

template <int D>
__device__ __forceinline__ int key_swizzle(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
template <int D>
__device__ __forceinline__ int value_swizzle(int row) { return D == 128 ? ((row & 3) << 2) : (((row >> 1) & 1) << 2); }

// max / sum with the lane 32 away; both get the result
__device__ __forceinline__ float halves_max(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    bf16x2 r;
    r[0] = (__bf16)a;
    r[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, r);
}

// 16 bytes of global memory per lane straight into LDS at `l` + 16 * lane (l wave-uniform)
__device__ __forceinline__ void dma16(const char* g, char* l) {
    __builtin_amdgcn_global_load_lds((const MP_GLOBAL void*)g, (MP_LDS void*)l, 16, 0, 0);
}
// every outstanding load and LDS write of this wave has landed, then the workgroup meets
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// What a wave keeps of its 32 rows.
template <int D>
struct RowState {
    bf16x8 q[D / 16];      // right-hand operand of S^T: row l % 32, dims 16 s + 8 (l / 32) ..
    f32x16 o[D / 32];      // O^T: dims 32 i + 8 (r / 4) + 4 (l / 32) + r % 4
    float m, l;            // running maximum (base 2) of both halves; this half's share of the sum
};

template <int D>
__device__ __forceinline__ void load_rows(RowState<D>& st, const uint16_t* q) {     // q: this lane's row
    const int h = lane_id() >> 5;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) st.q[s] = *reinterpret_cast<const bf16x8*>(q + 16 * s + 8 * h);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.o[i][r] = 0.f;
    st.m = NEG_INF;
    st.l = 0.f;
}

// This lane's left-hand operand of O^T: dims 32 i + l % 32, tokens 16 t + 8 (j / 4) + 4 (l / 32) + j % 4
template <int D>
__device__ __forceinline__ bf16x8 read_v(const char* vt, int i, int t) {
    const int l = lane_id(), r = (l & 15) >> 2;
    const int swz = D == 128 ? (i ^ r) : (i ^ (r >> 1));
    const char* p = vt + (4 * (l >> 5) + r) * (2 * D) + swz * 64 + ((l >> 4) & 1) * 32 + (l & 3) * 8 + t * 16 * (2 * D);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MP_LDS s16x4*)(p));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MP_LDS s16x4*)(p + 8 * (2 * D)));
    typedef __attribute__((ext_vector_type(8))) short s16x8;
    const s16x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, v);
}

// A masked tile may hold values that a row must not see, and 0 times an infinity is NaN.  Product with zeros first:
// finite values give 0, anything else NaN.  (Every row sees a tile without a mask: its values are multiplied as they are, and an
// infinity whose weight is 0 in f32 gives NaN there, as it does where a row that holds one is scaled by 0.)
template <int D, int SUB>
__device__ __forceinline__ bool tile_has_nonfinite(const char* vt) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    bf16x8 zero;
#pragma unroll
    for (int j = 0; j < 8; ++j) zero[j] = (__bf16)0.f;
#pragma unroll
    for (int t = 0; t < 2 * SUB; ++t)
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(read_v<D>(vt, i, t), zero, acc, 0, 0, 0);
    const float s = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    asm volatile("" ::: "memory");       // what follows reads the tile again: these 64 registers are not kept for it
    return __ballot(!(s == 0.f)) != 0;
}

// ... and where a masked tile does, its finite values alone go into the product (0 for the others) ...
// 0xffff in the halves of w that are not finite
__device__ __forceinline__ uint32_t nonfinite_halves(uint32_t w) {
    return ((((w & 0x7f807f80u) + 0x00800080u) >> 15) & 0x00010001u) * 0xffffu;
}
__device__ __forceinline__ bf16x8 finite_only(bf16x8 x) {
    u32x4 v = __builtin_bit_cast(u32x4, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] &= ~nonfinite_halves(v[j]);
    return __builtin_bit_cast(bf16x8, v);
}
// ... and the others are counted per row and dim over the tokens the row sees -- +inf, -inf and NaN as 1, 2^7 and 2^14 of
// one exact product, at most 64 of each -- and join as what a sum over them is.  Rare: one block at a time, few registers.
template <int D, int SUB>
__device__ __forceinline__ void add_nonfinite(f32x16 (&o)[D / 32], const char* vt, int lim) {
    const int h = lane_id() >> 5;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        f32x16 cnt;
#pragma unroll
        for (int r = 0; r < 16; ++r) cnt[r] = 0.f;
        asm volatile("" : "+v"(lim));        // (what depends on it is computed again, not kept in 16 registers)
#pragma unroll
        for (int t = 0; t < 2 * SUB; ++t) {
            __builtin_amdgcn_sched_barrier(0);
            const u32x4 v = __builtin_bit_cast(u32x4, read_v<D>(vt, i, t));
            u32x4 odd, see;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t nan = ((((v[j] & 0x007f007fu) + 0x007f007fu) >> 7) & 0x00010001u) * 0xffffu;   // given not finite
                const uint32_t neg = ((v[j] >> 15) & 0x00010001u) * 0xffffu;
                odd[j] = nonfinite_halves(v[j]) &
                         ((nan & 0x46804680u) | (~nan & ((neg & 0x43004300u) | (~neg & 0x3f803f80u))));
                const int tok = 16 * t + 8 * (j >> 1) + 4 * h + 2 * (j & 1);
                see[j] = ((uint32_t)((tok - lim - 1) >> 31) & 0x3f80u) | ((uint32_t)((tok - lim) >> 31) & 0x3f800000u);
            }
            cnt = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, odd), __builtin_bit_cast(bf16x8, see),
                                                          cnt, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int n = (int)cnt[r];
            const float pos = (n & 127) ? __builtin_inff() : 0.f, neg = (n >> 7 & 127) ? NEG_INF : 0.f;
            o[i][r] += n >> 14 ? __builtin_nanf("") : pos + neg;
        }
    }
}

// The steps of folding SUB * 32 tokens (K rows at kt, V rows at vt in LDS) into the wave's rows.
// s = K Q^T
template <int D, int SUB>
__device__ __forceinline__ void tile_scores(f32x16 (&s)[SUB], const RowState<D>& st, const char* kt) {
    const int l = lane_id(), h = l >> 5, row = l & 31;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const bf16x8 kf = *reinterpret_cast<const bf16x8*>(kt + (32 * u + row) * (2 * D) + (((2 * k + h) ^ key_swizzle<D>(row)) << 4));
            s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, st.q[k], s[u], 0, 0, 0);
        }
}
// only tokens <= lim (relative to the tile, per lane) are visible to the lane's row
template <int SUB>
__device__ __forceinline__ void mask_scores(f32x16 (&s)[SUB], int lim) {
    const int h = lane_id() >> 5;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (32 * u + 8 * (r >> 2) + 4 * h + (r & 3) > lim) s[u][r] = NEG_INF;
}
// m follows these scores
template <int D, int SUB>
__device__ __forceinline__ void move_maximum(RowState<D>& st, const f32x16 (&s)[SUB], float c) {
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
    const float m = fmaxf(st.m, halves_max(top) * c);
    const float f = m == NEG_INF ? 1.f : __builtin_amdgcn_exp2f(st.m - m);
    st.m = m;
    st.l *= f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.o[i][r] *= f;
}
// p = 2^(c s - m); returns their sum
template <int D, int SUB>
__device__ __forceinline__ float tile_weights(const RowState<D>& st, const f32x16 (&s)[SUB], float c, bf16x8 (&p)[2 * SUB]) {
    const float off = st.m == NEG_INF ? 0.f : st.m;      // nothing seen yet: every weight below is 2^-inf = 0
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], c, -off));
            sum += w;
            p[2 * u + (r >> 3)][r & 7] = (__bf16)w;
        }
    return sum;
}
// ... taken over, or made again from a maximum that follows
template <int D, int SUB>
__device__ __forceinline__ void settle_weights(RowState<D>& st, const f32x16 (&s)[SUB], float c, bf16x8 (&p)[2 * SUB], float sum) {
    if (__ballot(sum > LAZY_SUM || st.m == NEG_INF)) {
        move_maximum<D, SUB>(st, s, c);
        sum = tile_weights<D, SUB>(st, s, c, p);
    }
    st.l += sum;
}
// o += V^T p
template <int D, int SUB, bool MASK>
__device__ __forceinline__ void add_values(RowState<D>& st, const bf16x8 (&p)[2 * SUB], const char* vt, int lim) {
    const bool odd = MASK && tile_has_nonfinite<D, SUB>(vt);
#pragma unroll
    for (int t = 0; t < 2 * SUB; ++t) {
        if (MASK) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            bf16x8 v = read_v<D>(vt, i, t);
            if (MASK && odd) v = finite_only(v);
            st.o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p[t], st.o[i], 0, 0, 0);
        }
    }
    if (MASK && odd) add_nonfinite<D, SUB>(st.o, vt, lim);
}
// All of them.  `between` runs behind the first product.
template <int D, int SUB, bool MASK, class F>
__device__ __forceinline__ void fold_tile(RowState<D>& st, const char* kt, const char* vt, float c, int lim, F between) {
    f32x16 s[SUB];
    bf16x8 p[2 * SUB];
    tile_scores<D, SUB>(s, st, kt);
    between();
    if (MASK) mask_scores<SUB>(s, lim);
    const float sum = tile_weights<D, SUB>(st, s, c, p);
    settle_weights<D, SUB>(st, s, c, p, sum);
    add_values<D, SUB, MASK>(st, p, vt, lim);
}

template <int D, int SUB, bool MASK>
__device__ __forceinline__ void fold_tile(RowState<D>& st, const char* kt, const char* vt, float c, int lim) {
    fold_tile<D, SUB, MASK>(st, kt, vt, c, lim, [] {});
}

// Which sequence and which of its tiles a slot is.  Sequence b of rows cu[b] G .. cu[b + 1] G owns the slots from
// floor(cu[b] G / BM) + b on: at least as many as it has tiles, for every split of the rows, so the grid needs
// no list of tiles made beforehand -- floor(T G / BM) + B slots, at most B of them empty.  All lanes return the same.
struct TileOf {
    int seq;         // -1: no such sequence
    int start, n;    // its first row of q (token) and its tokens
    int row0;        // the tile's first row inside the sequence
};
template <int BM>
__device__ __forceinline__ TileOf find_tile(const int32_t* __restrict__ cu, int B, int T, int G, int slot) {
    auto first = [&](int i) { return (int)(((int64_t)min(max(cu[i], 0), T) * G) / BM) + i; };
    // the last sequence whose first slot is not behind this one: 64 candidates at a time, the whole wave looking (one load up to
    // 64 sequences, two up to 4096)
    int lo = -1, n = B;                              // it is lo or one of the n behind lo
    while (n > 0) {
        const int step = (n + WAVE - 1) / WAVE, i = lo + 1 + lane_id() * step;
        const int cnt = __popcll(__ballot(lane_id() * step < n && first(min(i, B - 1)) <= slot));
        const int hit = __builtin_amdgcn_readfirstlane(cnt);
        if (hit == 0) break;
        n = min(step, n - (hit - 1) * step) - 1;
        lo += 1 + (hit - 1) * step;
    }
    TileOf t;
    t.seq = -1;
    t.start = t.n = t.row0 = 0;
    const int b = lo;
    if (b < 0) return t;
    const int tile = slot - first(b);
    t.start = min(max(cu[b], 0), T);
    t.n = min(max(cu[b + 1], 0), T) - t.start;
    if (tile < 0 || t.n <= 0 || (int64_t)tile * BM >= (int64_t)t.n * G) return t;
    t.row0 = tile * BM;
    t.seq = b;
    return t;
}

// The same for at most 64 sequences, tile `at` of all in the order of their places in their sequences, last places first: under a
// causal mask a tile's work grows with its place, so workgroups begin with the longest whatever sequence it is of.  One lane a
// sequence; sum_b max(tiles_b - 1 - t, 0) tiles lie behind place t.  32 heads over 8, against one sequence after the other:
// 2 x 1000 tokens of head_dim 128 39 -> 34 us, of 64 24 -> 20; 8 x 1000 101 -> 97 and 58 -> 54; 50 to 4000 198 -> 194 and 119 -> 112;
// 8 heads over 1: 8 x 2000 97 -> 83.  It costs up to 5 % where the last workgroups were few before (2 x 2000 of 128: 83 -> 87).
template <int BM>
__device__ __forceinline__ TileOf find_tile_longest_first(const int32_t* __restrict__ cu, int B, int T, int G, int at) {
    const int l = lane_id(), i = min(l, B - 1);
    const int start = min(max(cu[i], 0), T), n = min(max(cu[i + 1], 0), T) - start;
    const int tiles = l < B && n > 0 ? (int)(((int64_t)n * G + BM - 1) / BM) : 0;
    auto behind = [&](int place) { return (int)wave_sum_u32((uint32_t)max(tiles - 1 - place, 0)); };
    TileOf t;
    t.seq = -1;
    t.start = t.n = t.row0 = 0;
    if (at < 0 || at >= behind(-1)) return t;
    int lo = 0, hi = (int)wave_max((float)tiles) - 1;      // the first place that at most `at` tiles lie behind (tiles <= 2^24: exact)
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (behind(mid) <= at) hi = mid;
        else lo = mid + 1;
    }
    const unsigned long long has = __ballot(tiles > lo);
    const int which = at - behind(lo);                               // among the sequences that have this place
    const unsigned long long hit = __ballot((has >> l & 1) && __popcll(has & ((1ull << l) - 1)) == which);
    if (hit == 0) return t;
    t.seq = __ffsll(hit) - 1;
    t.start = __builtin_amdgcn_readlane(start, t.seq);
    t.n = __builtin_amdgcn_readlane(n, t.seq);
    t.row0 = lo * BM;
    return t;
}

// 1 / l for a row's output.  A row that sees nothing is 0.  One that sees keys but whose weights are all 0 sees logits of -inf
// alone, and 0 / 0 is NaN: what the definition gives (its log-sum-exp is -inf as well).
__device__ __forceinline__ float inverse_sum(float l, bool sees) { return sees ? 1.f / l : 0.f; }

// Base-2 log-sum-exp of sum l over 2^m: -inf of nothing, +inf where a logit was (its weights are NaN, as inf - inf is).
__device__ __forceinline__ float log_sum(float m, float l) {
    return l == 0.f ? NEG_INF : m == __builtin_inff() ? m : m + __builtin_amdgcn_logf(l);
}

// The wave's rows as they leave: normalised, bf16, with the base-2 log-sum-exp; `sees`: there is a key that the row may see.
template <int D>
__device__ __forceinline__ void store_rows(const RowState<D>& st, uint16_t* out, float* lse, bool sees) {     // this lane's row
    const int h = lane_id() >> 5;
    const float l = halves_sum(st.l);
    const float inv = inverse_sum(l, sees);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            u32x2 w;
            w[0] = pack_bf16(st.o[i][4 * g] * inv, st.o[i][4 * g + 1] * inv);
            w[1] = pack_bf16(st.o[i][4 * g + 2] * inv, st.o[i][4 * g + 3] * inv);
            *reinterpret_cast<u32x2*>(out + 32 * i + 8 * g + 4 * h) = w;
        }
    if (lse != nullptr && h == 0) *lse = log_sum(st.m, l);
}

// Four waves that folded different keys into the same 32 rows: their sums joined.  Wave w leaves its 32 rows, f32, in its own
// 32 D * 4 bytes of LDS (`mine`; the waves' blocks lie `apart` 16-byte chunks from each other at `all`), chunk c of row r at place
// c ^ r, as a column's rows would all lie in one bank otherwise.  Then 8 threads a row: thread i gets chunks (i % 8) D / 32
// .. of row i / 8, scaled to the maximum m, and the row's sum of weights.  One barrier; all 256 threads call it.
template <int D>
__device__ __forceinline__ void join_waves(const RowState<D>& st, f32x4* mine, const f32x4* all, int apart, float2 (&ml)[4][32],
                                           float& m, float& total, f32x4 (&o)[D / 32]) {
    constexpr int NC = D / 4;                            // chunks of a row
    const int l = lane_id(), w = threadIdx.x >> 6;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // (the block held the wave's tile: its last reads come first)
    const float sum = halves_sum(st.l);
    if (l < 32) ml[w][l] = make_float2(st.m, sum);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            mine[(l & 31) * NC + ((8 * i + 2 * g + (l >> 5)) ^ (l & (NC - 1) & 31))] =
                f32x4{st.o[i][4 * g], st.o[i][4 * g + 1], st.o[i][4 * g + 2], st.o[i][4 * g + 3]};
    __syncthreads();
    const int r = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * (NC / 8);
    float2 x[4];
    m = NEG_INF;
    total = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        x[k] = ml[k][r];
        m = fmaxf(m, x[k].x);
    }
    const float off = m == NEG_INF ? 0.f : m;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float wt = __builtin_amdgcn_exp2f(x[k].x - off);
        total += wt * x[k].y;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            const f32x4 y = all[k * apart + r * NC + ((c0 + c) ^ (r & (NC - 1)))];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][e] += wt * y[e];
        }
    }
}
// ... and as they leave: this thread's chunks of its row
template <int D>
__device__ __forceinline__ void store_chunks(uint16_t* out, const f32x4 (&o)[D / 32], float total, bool sees) {
    const float inv = inverse_sum(total, sees);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        u32x2 b;
        b[0] = pack_bf16(o[c][0] * inv, o[c][1] * inv);
        b[1] = pack_bf16(o[c][2] * inv, o[c][3] * inv);
        *reinterpret_cast<u32x2*>(out + 4 * ((threadIdx.x & 7) * (D / 32) + c)) = b;
    }
}

}  // namespace mp
