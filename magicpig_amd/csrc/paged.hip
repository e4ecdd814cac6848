// paged.hip -- a paged key / value cache: rows written (bf16, or quantised to e4m3 as they are written) and read back,
// and the attention of each request's new tokens over its pages.
//
// Layout.  A page holds page_size tokens of every kv head; the page of one head is one block of rows, K and V of a token side
// by side: row ((page Hkv + head) page_size + slot) of [K | V], D elements each.  Position p of request b lies in page
// table[b][p / page_size], slot p % page_size (page_size is a power of two).
//
// Quantisation.  A K or V row x of D elements is stored as e4m3 codes c and one byte e + 127: e is the least integer with
// max |x_i| <= 448 * 2^e (448: the largest e4m3 number) and not below -126, c_i = e4m3(x_i 2^-e), round to nearest even.  A power of two costs a
// floating-point code no precision (it moves the exponents of all elements), makes both products exact, so that the code
// alone rounds (by 2^-4 relative, 2^-10 of 2^e below its normal range), and every stored value is a bf16 number again: the
// attention multiplies exactly what reading the cache returns.  An infinity or NaN is stored as NaN, and the row's maximum
// is that of its finite elements.
#include "attn_tile.h"

namespace mp {

// The rows a call works on, as append, read and attention describe them.
struct PagedRows {
    const int32_t *cu, *table, *kv_len;
    int B, T, P;                     // requests, rows of the packed tensors, table entries per request
    int shift, num_pages, Hkv;
    int* err;
};

// whether a request's table can hold this length
__device__ __forceinline__ int table_positions(const PagedRows& r) { return (int)min((int64_t)r.P << r.shift, (int64_t)0x7fffffff); }
__device__ __forceinline__ bool length_ok(const PagedRows& r, int want) {
    if (want >= 0 && want <= table_positions(r)) return true;
    atomicOr(r.err, 1);
    return false;
}
// a request's cache length for attention, which only reads: the nearest that its table can hold
__device__ __forceinline__ int cached(const PagedRows& r, int want) {
    return length_ok(r, want) ? want : want < 0 ? 0 : table_positions(r);
}
// page id -> a page that exists
__device__ __forceinline__ int page_ok(const PagedRows& r, int page) {
    if ((unsigned)page < (unsigned)r.num_pages) return page;
    atomicOr(r.err, 2);
    return -1;
}

// row of the cache that holds position `pos` (in page `page`, or page 0 if there is no such page) of a kv head
__device__ __forceinline__ uint32_t cache_row(const PagedRows& r, int page, int head, int pos) {
    const uint32_t pg = (uint32_t)max(page_ok(r, page), 0);
    return ((pg * (uint32_t)r.Hkv + (uint32_t)head) << r.shift) | (uint32_t)(pos & ((1 << r.shift) - 1));
}

// e4m3 pairs -> bf16 pairs times a power of two
__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi, float s) {
    u32x4 w;
    w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false));
    w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true));
    w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false));
    w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true));
    return w;
}

// bits of the largest magnitude over the D / 8 lanes that share a row (non-negative numbers order as their bits do)
template <int D>
__device__ __forceinline__ uint32_t row_lanes_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));      // lane ^ 1
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));      // lane ^ 2
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));     // the other quad of 8 lanes
    if (D == 128) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));   // the other 8 of 16
    return v;
}

struct CopyArgs {
    PagedRows r;
    const uint16_t *k, *v;                       // append: in
    int64_t k_st, k_sh, v_st, v_sh;
    uint16_t *ko, *vo;                           // read: out, contiguous
    char* pool;
    uint8_t* scale;
    int per_block;                               // tokens a workgroup copies
};

constexpr int COPY_TOKENS = 16;                  // at most
constexpr int COPY_SEQS = 255;                   // requests whose lengths a workgroup keeps in LDS
constexpr uint32_t NO_ROW = 0xffffffffu;

// Rows in (READ false) and out.  A workgroup takes `per_block` tokens, finds their places once, one thread a token, and then
// streams all their heads, 16 bytes of bf16 a lane and COPY_UNROLL of them in flight: a row is D / 8 neighbouring lanes, K and V
// of a (token, head) neighbouring rows.  Bound by memory: 4 D bytes in and 4 D (e4m3: 2 D + 2) out per token and kv head.
// The packed tensors are streamed past the caches, so that what stays in them is the pages, which are read next: 98 000
// tokens of 8 heads of 128 in (e4m3) and out again take 209 us (5.8 TB/s of rows; 265 us with cached accesses, 280 /
// 299 us with 16 / 32 tokens a workgroup instead of 8).
constexpr int COPY_UNROLL = 4;
template <int D, bool E4M3, bool READ>
__global__ __launch_bounds__(256) void paged_copy_kernel(const CopyArgs a) {
    constexpr int LANES = D / 8;
    __shared__ uint32_t place[COPY_TOKENS];
    __shared__ int s_cu[COPY_SEQS + 1], s_kv[COPY_SEQS];
    const PagedRows& r = a.r;
    const int t0 = blockIdx.x * a.per_block, tokens = min(a.per_block, r.T - t0);
    const bool small = r.B <= COPY_SEQS;
    if (small) {
        if ((int)threadIdx.x <= r.B) s_cu[threadIdx.x] = r.cu[threadIdx.x];
        if ((int)threadIdx.x < r.B) s_kv[threadIdx.x] = r.kv_len[threadIdx.x];
        __syncthreads();
    }
    if ((int)threadIdx.x < tokens) {
        const int tok = t0 + threadIdx.x;
        auto cu = [&](int i) { return small ? s_cu[i] : r.cu[i]; };
        int lo = 0, hi = r.B;                    // the first request that ends behind tok
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (cu(mid + 1) <= tok) lo = mid + 1;
            else hi = mid;
        }
        uint32_t at = NO_ROW;
        if (lo < r.B && cu(lo) <= tok) {
            // (the rows of a length that the table cannot hold have no place: any other would be another position's)
            const int len = small ? s_kv[lo] : r.kv_len[lo];
            const int pos = length_ok(r, len) ? len - min(cu(lo + 1), r.T) + tok : -1;
            if (pos >= 0) {
                const int page = page_ok(r, r.table[(int64_t)lo * r.P + (pos >> r.shift)]);
                if (page >= 0) at = (((uint32_t)page * (uint32_t)r.Hkv) << r.shift) | (uint32_t)(pos & ((1 << r.shift) - 1));
            }
        }
        place[threadIdx.x] = at;
    }
    __syncthreads();
    const int per_token = 2 * r.Hkv * LANES;     // 16-byte pieces
    const int step_t = 256 / per_token, step_c = 256 % per_token;
    int tl = (int)threadIdx.x / per_token, c = (int)threadIdx.x % per_token;
    while (__any(tl < tokens)) {
        const uint16_t* in[COPY_UNROLL];
        uint32_t row[COPY_UNROLL];
        int tc[COPY_UNROLL], cc[COPY_UNROLL];
        u32x4 x[COPY_UNROLL];
        uint32_t e[COPY_UNROLL];
#pragma unroll
        for (int u = 0; u < COPY_UNROLL; ++u) {
            tc[u] = tl;
            cc[u] = c;
            row[u] = NO_ROW;
            if (tl < tokens) {
                const uint32_t at = place[tl];
                if (at != NO_ROW) row[u] = at + ((uint32_t)(c / (2 * LANES)) << r.shift);
            }
            tl += step_t;
            c += step_c;
            if (c >= per_token) {
                c -= per_token;
                ++tl;
            }
        }
#pragma unroll
        for (int u = 0; u < COPY_UNROLL; ++u) {
            const int head = cc[u] / (2 * LANES), which = (cc[u] / LANES) & 1, p = cc[u] % LANES;
            if (row[u] == NO_ROW) continue;
            const uint64_t w = (uint64_t)row[u] * 2 + which;
            if (READ) {
                if (E4M3) {
                    const u32x2 y = *reinterpret_cast<const u32x2*>(a.pool + (w * LANES + p) * 8);
                    x[u][0] = y[0];
                    x[u][1] = y[1];
                    e[u] = a.scale[w];
                } else {
                    x[u] = *reinterpret_cast<const u32x4*>(a.pool + (w * LANES + p) * 16);
                }
            } else {
                const int64_t tok = t0 + tc[u];
                in[u] = which ? a.v + tok * a.v_st + head * a.v_sh : a.k + tok * a.k_st + head * a.k_sh;
                x[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(in[u] + 8 * p));
            }
        }
#pragma unroll
        for (int u = 0; u < COPY_UNROLL; ++u) {
            const int head = cc[u] / (2 * LANES), which = (cc[u] / LANES) & 1, p = cc[u] % LANES;
            if (row[u] == NO_ROW) continue;
            const uint64_t w = (uint64_t)row[u] * 2 + which;
            if (READ) {
                uint16_t* out = (which ? a.vo : a.ko) + ((int64_t)(t0 + tc[u]) * r.Hkv + head) * D + 8 * p;
                if (E4M3) x[u] = widen8(x[u][0], x[u][1], __uint_as_float(e[u] << 23));
                __builtin_nontemporal_store(x[u], reinterpret_cast<u32x4*>(out));
            } else if (!E4M3) {
                *reinterpret_cast<u32x4*>(a.pool + (w * LANES + p) * 16) = x[u];
            } else {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t l = x[u][i] & 0x7fffu, h = (x[u][i] >> 16) & 0x7fffu;
                    top = max(top, max(l < 0x7f80u ? l : 0u, h < 0x7f80u ? h : 0u));
                }
                top = row_lanes_max<D>(top);
                // exponent - 127 - 8, one more where the mantissa is above 1.75 = 448 / 2^8; as a biased exponent, at least 1
                const int ex = max((int)(top >> 7) - 8 + ((top & 127u) > 96u ? 1 : 0), 1);
                const float up = __uint_as_float((uint32_t)(254 - ex) << 23);
                u32x2 y;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    int word = __builtin_amdgcn_cvt_pk_fp8_f32(bf16_lo(x[u][2 * i]) * up, bf16_hi(x[u][2 * i]) * up, 0, false);
                    word = __builtin_amdgcn_cvt_pk_fp8_f32(bf16_lo(x[u][2 * i + 1]) * up, bf16_hi(x[u][2 * i + 1]) * up, word, true);
                    y[i] = (uint32_t)word;
                }
                *reinterpret_cast<u32x2*>(a.pool + (w * LANES + p) * 8) = y;
                if (p == 0) a.scale[w] = (uint8_t)ex;
            }
        }
    }
}

// ---------------------------------------------------------------- attention over the pages
// Work.  Request b has ceil(n_b G / BM) tiles of rows and ceil(kv_b / TOK) tiles of keys.  A workgroup gets one tile of rows
// of one kv head and one part of its keys.  What a part should be is found by every workgroup from the lengths on the device (so a
// captured graph follows them): the work over `units` workgroups a kv head, at least MIN_KEYS tokens.  Short requests are
// one part, long ones are cut evenly into parts of at most that, whatever the mix.  Parts of a row are joined by a second kernel.
struct PagedAttnArgs {
    PagedRows r;
    const uint16_t* q;
    int64_t q_st, q_sh;
    const char* pool;
    const uint8_t* scale;
    int H, G, units;                 // units: 0 = never cut the keys
    float c;
    uint16_t* out;
    float* lse;
    float* part_o;                   // [workgroup][BM][D], sums that are not normalised
    float2* part_ml;                 // [workgroup][BM], their maxima and sums of weights
    int2* part_of;                   // [T * H]: the row's place among the part_o of its first part, number of parts
    int grid;                        // workgroups
};

// Tokens of a part, at least: joining costs more than it spreads below.  One new token behind 2000 of one request takes 11.6 us
// with parts of 256 and 13.8 with 512; behind 8000 12.4, and 14.2 with 128.  With 128 rows a workgroup there are more rows
// to join: 512 new tokens of one request, 8 kv heads: 28.7 us in parts of 256, 18.7 in one.
template <int BM>
constexpr int MIN_KEYS = BM == 32 ? 256 : 512;

// From here on 256 rows a workgroup at head_dim 128, which read the keys from L2 half as often: 2048 new tokens of 32 heads over 8
// behind 67 584 2.12 ms against 2.30, 16 x 512 of 8 heads over 1 behind 2000 (e4m3) 81 us against 86.  (Where all keys are new and few
// heads share a chip, the shorter workgroups pack better: 8192 of 8 heads over 1, e4m3, 241 us against 232.)
constexpr int64_t WIDE_ROWS = 1 << 16;

struct PartOf {
    int seq;                         // -1: none
    int start, n, row0, kv;          // first row of q (token) and tokens of the request, first row of the tile, cached positions
    int part, parts;
};

// U: requests a lane looks at, side by side (their loads are in flight together, and one scan over the wave serves 64 U of them)
template <int BM, int TOK, int U>
__device__ __forceinline__ PartOf find_part_of(const PagedRows& r, int G, int units, int unit) {
    PartOf p;
    p.seq = -1;
    p.start = p.n = p.row0 = p.kv = p.part = p.parts = 0;
    auto first = [&](int i) { return min(max(r.cu[i], 0), r.T); };
    auto row_tiles = [&](int i) { return i < r.B ? (max(first(i + 1) - first(i), 0) * G + BM - 1) / BM : 0; };
    auto key_tiles = [&](int i) { return (int)(((int64_t)cached(r, r.kv_len[min(i, r.B - 1)]) + TOK - 1) / TOK); };
    float tiles = 0.f, work = 0.f;              // (products of large counts; the quotient need not be exact)
    for (int base = 0; base < r.B; base += U * WAVE)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + U * lane_id() + u;
            const float rt = (float)row_tiles(i);
            tiles += rt;
            work += rt * (float)key_tiles(i);
        }
    // half a part is lost to rounding up per tile of rows: aim so much lower that the parts still fit the chip at once
    const float aim = fmaxf((float)units - 0.5f * wave_sum(tiles), 0.5f * (float)units);
    const float per = fmaxf(__builtin_ceilf(wave_sum(work) / aim), (float)(MIN_KEYS<BM> / TOK)), inv = 1.f / per;
    int before = 0;
    for (int base = 0; base < r.B; base += U * WAVE) {
        int parts[U], units_of[U], sum = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + U * lane_id() + u, kt = key_tiles(i);
            // (what is less than half longer than the least part is not cut; every workgroup rounds alike)
            parts[u] = 2 * kt < 3 * (MIN_KEYS<BM> / TOK) ? 1 : max((int)__builtin_ceilf((float)kt * inv), 1);
            units_of[u] = row_tiles(i) * parts[u];
            sum += units_of[u];
        }
        const int upto = before + wave_incl_scan(sum);
        const unsigned long long past = __ballot(upto > unit);
        if (past) {
            const int k = __ffsll(past) - 1;
            int at = unit - (__builtin_amdgcn_readlane(upto, k) - __builtin_amdgcn_readlane(sum, k));
            p.seq = base + U * k;
            p.parts = __builtin_amdgcn_readlane(parts[0], k);
#pragma unroll
            for (int u = 0; u + 1 < U; ++u) {
                const int here = __builtin_amdgcn_readlane(units_of[u], k);
                if (p.seq == base + U * k + u && at >= here) {
                    at -= here;
                    ++p.seq;
                    p.parts = __builtin_amdgcn_readlane(parts[u + 1], k);
                }
            }
            p.seq = min(p.seq, r.B - 1);                                     // (offsets that are none could count past the end)
            p.start = first(p.seq);
            p.n = first(p.seq + 1) - p.start;
            p.kv = cached(r, r.kv_len[p.seq]);
            p.row0 = at / p.parts * BM;
            p.part = at % p.parts;
            if (p.row0 < 0 || (int64_t)p.row0 >= (int64_t)p.n * G) p.seq = -1;
            return p;
        }
        before = __builtin_amdgcn_readlane(upto, WAVE - 1);
    }
    return p;
}

template <int BM, int TOK>
__device__ __forceinline__ PartOf find_part(const PagedRows& r, int G, int units, int unit) {
    if (units > 0) return r.B <= WAVE ? find_part_of<BM, TOK, 1>(r, G, units, unit) : find_part_of<BM, TOK, 4>(r, G, units, unit);
    // one part a tile of rows: the slots of attn_tile.h, a request's longest first
    const TileOf t = find_tile<BM>(r.cu, r.B, r.T, G, (int)(gridDim.x / r.Hkv) - 1 - unit);
    return PartOf{t.seq, t.start, t.n, t.row0, t.seq < 0 ? 0 : cached(r, r.kv_len[t.seq]), 0, 1};
}

// Many rows: 128 or 256 of one (request, kv head) a workgroup, everything else as in prompt.hip.  An e4m3 tile passes through
// registers on its way to LDS: loaded while the tile before it is folded in, widened behind it (exact).
template <int D, bool E4M3, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_attention_kernel(const PagedAttnArgs a) {
    constexpr int THREADS = 64 * WAVES, BM = 32 * WAVES, CPR = D / 8, KB = TILE_TOKENS * 2 * D;
    constexpr int PER_ROW = E4M3 ? CPR / 2 : CPR;                     // 16-byte pieces of a cached row
    constexpr int PASSES = TILE_TOKENS * PER_ROW / THREADS;
    __shared__ __attribute__((aligned(1024))) char lds[2][2][KB];
    const int head = blockIdx.x % a.r.Hkv;
    const PartOf t = find_part<BM, TILE_TOKENS>(a.r, a.G, a.units, (int)(blockIdx.x / a.r.Hkv));
    if (t.seq < 0) return;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
    const int rows = t.n * a.G, old = t.kv - t.n;                     // old: positions in front of the new tokens
    const int lim_lo = old + t.row0 / a.G, lim_hi = old + min(t.row0 + BM - 1, rows - 1) / a.G;
    const int all = lim_hi < 0 ? 0 : lim_hi / TILE_TOKENS + 1;
    const int used = max(min(t.parts, all), 1);
    if (t.part >= used) return;
    const int begin = (int)((int64_t)all * t.part / used), end = (int)((int64_t)all * (t.part + 1) / used);

    const int wrow = t.row0 + 32 * w;
    const int row = min(wrow + (l & 31), rows - 1);
    const int tok = row / a.G, h = head * a.G + row % a.G, lim = old + tok;
    RowState<D> st;
    load_rows<D>(st, a.q + (int64_t)(t.start + tok) * a.q_st + (int64_t)h * a.q_sh);
    const int whole = min(lim_lo < 0 ? 0 : (lim_lo + 1) / TILE_TOKENS, end);
    const int wave_hi = old + min(wrow + 31, rows - 1) / a.G;
    const int seen = wrow < rows && wave_hi >= 0 ? min(wave_hi / TILE_TOKENS + 1, end) : 0;

    const int32_t* table = a.r.table + (int64_t)t.seq * a.r.P;
    // lane l looks up the cache row of token l of a tile (positions behind the last visible one: that one again, masked);
    // the lanes that load a row get it from there.  (A row number fits 32 bits: 2^32 rows are more than any HBM.)
    int page = 0;
    u32x4 kr[PASSES], vr[PASSES];
    uint32_t sr[PASSES];
    auto position = [&](int tile) { return min(tile * TILE_TOKENS + l, lim_hi); };
    auto fetch_pages = [&](int tile) { page = table[position(tile) >> a.r.shift]; };
    auto stage = [&](int tile) {
        const uint32_t row_of = cache_row(a.r, page, head, position(tile));
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int idx = i * THREADS + (int)threadIdx.x, r = idx / PER_ROW, p = idx % PER_ROW;
            const uint64_t at = (uint32_t)__builtin_amdgcn_ds_bpermute(r * 4, (int)row_of);
            if (E4M3) {
                const char* src = a.pool + at * (2 * D) + p * 16;
                kr[i] = *reinterpret_cast<const u32x4*>(src);
                vr[i] = *reinterpret_cast<const u32x4*>(src + D);
                sr[i] = *reinterpret_cast<const uint16_t*>(a.scale + at * 2);
            } else {
                const char* src = a.pool + at * (4 * D);
                char* dst = lds[tile & 1][0] + (i * THREADS + w * 64) * 16;
                dma16(src + ((p ^ key_swizzle<D>(r)) << 4), dst);
                dma16(src + 2 * D + ((p ^ value_swizzle<D>(r)) << 4), dst + KB);
            }
        }
    };
    auto widen = [&](int tile) {
        if (!E4M3) return;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int idx = i * THREADS + (int)threadIdx.x, r = idx / PER_ROW, p = idx % PER_ROW;
            char* kt = lds[tile & 1][0] + r * 2 * D;
            const float ks = __uint_as_float((sr[i] & 255u) << 23), vs = __uint_as_float((sr[i] >> 8) << 23);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                *reinterpret_cast<u32x4*>(kt + (((2 * p + e) ^ key_swizzle<D>(r)) << 4)) = widen8(kr[i][2 * e], kr[i][2 * e + 1], ks);
                *reinterpret_cast<u32x4*>(kt + KB + (((2 * p + e) ^ value_swizzle<D>(r)) << 4)) = widen8(vr[i][2 * e], vr[i][2 * e + 1], vs);
            }
        }
    };
    if (begin < end) {
        fetch_pages(begin);
        stage(begin);
        if (begin + 1 < end) fetch_pages(begin + 1);
        widen(begin);
    }
    int j = begin;
    auto ahead = [&] {
        if (j + 1 < end) {
            stage(j + 1);
            if (j + 2 < end) fetch_pages(j + 2);
        }
    };
    for (; j < whole; ++j) {
        tile_barrier();                                               // tile j is there, tile j - 1 no longer read
        // the next tile's loads: behind the first product in bf16 (2048 new tokens behind 67 584: 2.10 ms, 2.27 in front of it),
        // in front of it in e4m3, whose registers are wanted at the end (behind 32 000, 8 heads over 1: 284 us, 293 behind it)
        if (E4M3 || wrow >= rows) ahead();
        if (wrow < rows)
            fold_tile<D, 2, false>(st, lds[j & 1][0], lds[j & 1][1], a.c, 0, [&] { if (!E4M3) ahead(); });
        if (j + 1 < end) widen(j + 1);
    }
    for (; j < end; ++j) {
        tile_barrier();
        ahead();
        if (j < seen) fold_tile<D, 2, true>(st, lds[j & 1][0], lds[j & 1][1], a.c, lim - j * TILE_TOKENS);
        if (j + 1 < end) widen(j + 1);
    }

    if (wrow + (l & 31) >= rows) return;
    const int64_t orow = (int64_t)(t.start + tok) * a.H + h;
    // (a row that sees nothing, though others of its tile see more than one part, leaves with the first: nothing to join)
    const bool whole_row = used == 1 || (lim < 0 && t.part == 0);
    if (a.units > 0 && t.part == 0 && l < 32) a.part_of[orow] = make_int2((int)blockIdx.x * BM + 32 * w + l, whole_row ? 1 : used);
    if (whole_row) {
        store_rows<D>(st, a.out + orow * D, a.lse ? a.lse + orow : nullptr, lim >= 0);
        return;
    }
    const int64_t prow = (int64_t)blockIdx.x * BM + 32 * w + (l & 31);
    float* po = a.part_o + prow * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(po + 32 * i + 8 * g + 4 * (l >> 5)) =
                f32x4{st.o[i][4 * g], st.o[i][4 * g + 1], st.o[i][4 * g + 2], st.o[i][4 * g + 3]};
    const float sum = halves_sum(st.l);
    if (l < 32) a.part_ml[prow] = make_float2(st.m, sum);
}

// Few rows (a decode step, drafted tokens): one tile of 32 rows a workgroup, and the keys are what is shared out -- tiles
// of 32 tokens in turn over the four waves, each with its own running softmax over its own block of LDS (no barrier until
// the waves' results are joined at the end).  A tile passes through registers: its loads (16 KB a wave in bf16, 8 KB in
// e4m3, eight waves a CU) are in flight while the tile before it is folded in.
template <int D, bool E4M3>
__global__ __launch_bounds__(256, 2) void paged_step_kernel(const PagedAttnArgs a) {
    constexpr int BM = 32, TOK = 32, KB = TOK * 2 * D;
    constexpr int PER_ROW = E4M3 ? D / 16 : D / 8;
    constexpr int PASSES = TOK * PER_ROW / 64;
    __shared__ __attribute__((aligned(1024))) char lds[4][2 * KB];     // a wave's K and V tile; at the end its 32 rows of sums
    __shared__ float2 ml[4][BM];
    const int head = blockIdx.x % a.r.Hkv;
    const PartOf t = find_part<BM, TOK>(a.r, a.G, a.units, (int)(blockIdx.x / a.r.Hkv));
    if (t.seq < 0) return;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
    const int rows = t.n * a.G, old = t.kv - t.n;
    const int lim_lo = old + t.row0 / a.G, lim_hi = old + min(t.row0 + BM - 1, rows - 1) / a.G;
    const int all = lim_hi < 0 ? 0 : lim_hi / TOK + 1;
    const int used = max(min(t.parts, all), 1);
    if (t.part >= used) return;
    const int begin = (int)((int64_t)all * t.part / used), end = (int)((int64_t)all * (t.part + 1) / used);
    const int whole = min(lim_lo < 0 ? 0 : (lim_lo + 1) / TOK, end);

    RowState<D> st;
    const int row = min(t.row0 + (l & 31), rows - 1), tok = row / a.G, lim = old + tok;
    load_rows<D>(st, a.q + (int64_t)(t.start + tok) * a.q_st + (int64_t)(head * a.G + row % a.G) * a.q_sh);

    const int32_t* table = a.r.table + (int64_t)t.seq * a.r.P;
    char *kt = lds[w], *vt = lds[w] + KB;
    int page = 0;                        // as above; lane l: token l % 32
    u32x4 kr[PASSES], vr[PASSES];
    uint32_t sr[PASSES];
    auto position = [&](int tile) { return min(tile * TOK + (l & 31), lim_hi); };
    auto fetch_pages = [&](int tile) { page = table[position(tile) >> a.r.shift]; };
    auto load = [&](int tile) {
        const uint32_t at = cache_row(a.r, page, head, position(tile));
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = (i * 64 + l) / PER_ROW, p = (i * 64 + l) % PER_ROW;
            const uint64_t x = (uint32_t)__builtin_amdgcn_ds_bpermute(r * 4, (int)at);
            const char* src = a.pool + x * (E4M3 ? 2 * D : 4 * D) + p * 16;
            kr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src));
            vr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + (E4M3 ? D : 2 * D)));
            if (E4M3) sr[i] = *reinterpret_cast<const uint16_t*>(a.scale + x * 2);
        }
    };
    // (within a wave LDS works in order: what the lanes wrote is there for the reads behind it, and the tile's last reads are
    // in front of the next writes; the fences keep the compiler to that order)
    auto store = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = (i * 64 + l) / PER_ROW, p = (i * 64 + l) % PER_ROW;
            char *kd = kt + r * 2 * D, *vd = vt + r * 2 * D;
            if (!E4M3) {
                *reinterpret_cast<u32x4*>(kd + ((p ^ key_swizzle<D>(r)) << 4)) = kr[i];
                *reinterpret_cast<u32x4*>(vd + ((p ^ value_swizzle<D>(r)) << 4)) = vr[i];
            } else {
                const float ks = __uint_as_float((sr[i] & 255u) << 23), vs = __uint_as_float((sr[i] >> 8) << 23);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    *reinterpret_cast<u32x4*>(kd + (((2 * p + e) ^ key_swizzle<D>(r)) << 4)) = widen8(kr[i][2 * e], kr[i][2 * e + 1], ks);
                    *reinterpret_cast<u32x4*>(vd + (((2 * p + e) ^ value_swizzle<D>(r)) << 4)) = widen8(vr[i][2 * e], vr[i][2 * e + 1], vs);
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    int j = begin + w;
    if (j < end) {
        fetch_pages(j);
        load(j);
        if (j + 4 < end) fetch_pages(j + 4);
    }
    for (; j < whole; j += 4) {
        store();
        __builtin_amdgcn_sched_barrier(0);           // the next tile's loads take the registers just stored
        if (j + 4 < end) {
            load(j + 4);
            if (j + 8 < end) fetch_pages(j + 8);
        }
        fold_tile<D, 1, false>(st, kt, vt, a.c, 0);
    }
    if (j < end) {                       // 32 rows end in at most two tiles: one a wave
        store();
        fold_tile<D, 1, true>(st, kt, vt, a.c, lim - j * TOK);
    }

    float m, total;
    f32x4 o[D / 32];
    const int r = threadIdx.x >> 3, grow = t.row0 + r;
    join_waves<D>(st, reinterpret_cast<f32x4*>(lds[w]), reinterpret_cast<const f32x4*>(lds[0]), 2 * KB / 16, ml, m, total, o);
    if (grow >= rows) return;
    const int64_t orow = (int64_t)(t.start + grow / a.G) * a.H + head * a.G + grow % a.G;
    const int64_t prow = (int64_t)blockIdx.x * BM + r;
    if (used > 1) {                      // (32 rows and more than a tile of keys: each row sees some)
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
            *reinterpret_cast<f32x4*>(a.part_o + prow * D + 4 * ((threadIdx.x & 7) * (D / 32) + c)) = o[c];
    } else {
        store_chunks<D>(a.out + orow * D, o, total, old + grow / a.G >= 0);
    }
    if ((threadIdx.x & 7) != 0) return;
    if (a.units > 0 && t.part == 0) a.part_of[orow] = make_int2((int)blockIdx.x * BM + r, used);
    if (used > 1) a.part_ml[prow] = make_float2(m, total);
    else if (a.lse != nullptr) a.lse[orow] = log_sum(m, total);
}

// Parts of a row joined: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, in an order that does not depend on when they
// were ready.  WAVES waves a row take its parts in turn, four at a time, each with a running maximum of its own: nothing is
// waited for but the row's place, then the parts.
template <int D, int BM, int WAVES>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnArgs a) {
    constexpr int W = D / 64, ROWS = 4 / WAVES;
    __shared__ float so[4][D];
    __shared__ float2 sml[4];
    const int l = lane_id(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * ROWS + w / WAVES;
    const int tok = (int)(row / a.H), lo = a.r.cu[0], hi = a.r.cu[a.r.B];
    const int2 of = tok < a.r.T ? a.part_of[row] : make_int2(0, 0);
    // (part_of of a row outside the requests was never written, and offsets that are none could leave anything)
    const int64_t at = of.x, step = (int64_t)a.r.Hkv * BM;            // the parts of a row are neighbours among its head's workgroups
    const bool mine = tok >= lo && tok < hi && of.y > 1 && at >= 0 && at + (of.y - 1) * step < (int64_t)a.grid * BM;
    const int n = mine ? of.y : 0;
    if (WAVES == 4 && n == 0) return;
    float m = NEG_INF, sum = 0.f, o[W];
#pragma unroll
    for (int i = 0; i < W; ++i) o[i] = 0.f;
    for (int s0 = w % WAVES; s0 < n; s0 += 4 * WAVES) {
        float2 x[4];
        float y[4][W];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t part = at + min(s0 + u * WAVES, n - 1) * step;
            x[u] = a.part_ml[part];
#pragma unroll
            for (int i = 0; i < W; ++i) y[u][i] = a.part_o[part * D + l * W + i];
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (s0 + u * WAVES >= n) x[u] = make_float2(NEG_INF, 0.f);
            top = fmaxf(top, x[u].x);
        }
        const float off = top == NEG_INF ? 0.f : top, f = __builtin_amdgcn_exp2f(m - off);
        m = top;
        sum *= f;
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] *= f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float wt = __builtin_amdgcn_exp2f(x[u].x - off);
            sum += wt * x[u].y;
#pragma unroll
            for (int i = 0; i < W; ++i) o[i] += s0 + u * WAVES < n ? wt * y[u][i] : 0.f;
        }
    }
    if (WAVES == 4) {
#pragma unroll
        for (int i = 0; i < W; ++i) so[w][l * W + i] = o[i];
        if (l == 0) sml[w] = make_float2(m, sum);
        __syncthreads();
        if (w > 0) return;
        float2 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[k] = sml[k];
            m = fmaxf(m, x[k].x);
        }
        const float off = m == NEG_INF ? 0.f : m;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float wt = __builtin_amdgcn_exp2f(x[k].x - off);
            sum += wt * x[k].y;
#pragma unroll
            for (int i = 0; i < W; ++i) o[i] += wt * so[k][l * W + i];
        }
    }
    if (n == 0) return;
    const float inv = inverse_sum(sum, true);
    if (W == 2) *reinterpret_cast<uint32_t*>(a.out + row * D + 2 * l) = pack_bf16(o[0] * inv, o[W - 1] * inv);
    else a.out[row * D + l] = (uint16_t)(pack_bf16(o[0] * inv, 0.f) & 0xffffu);
    if (a.lse != nullptr && l == 0) a.lse[row] = log_sum(m, sum);
}

// What the kernels met since the last look: taken and cleared in one step, so that nothing that another stream reports meanwhile is lost.
__global__ void paged_take_flags_kernel(int* err) { err[1] = atomicExch(err, 0); }

// ---------------------------------------------------------------- host
hipError_t launch_paged_take_flags(int* err, hipStream_t st) {
    paged_take_flags_kernel<<<1, 1, 0, st>>>(err);
    return hipGetLastError();
}

// Tokens a workgroup copies: one pass of its threads at least, and from 2048 tokens on up to 8, as long as that leaves a CU
// eight workgroups (fewer lookups).
static int copy_tokens(int64_t T, int Hkv, int D) {
    const int64_t pass = 256 / (Hkv * D / 4), many = T / 2048 < 8 ? T / 2048 : 8, n = many > pass ? many : pass;
    return n < 1 ? 1 : n > COPY_TOKENS ? COPY_TOKENS : (int)n;
}

static PagedRows paged_rows(const int32_t* cu, int B, int T, const int32_t* table, int P, const int32_t* kv_len, int shift,
                            int num_pages, int Hkv, int* err) {
    return PagedRows{cu, table, kv_len, B, T, P, shift, num_pages, Hkv, err};
}

template <int D>
static void paged_copy(const CopyArgs& a, bool e4m3, bool read, hipStream_t st) {
    const dim3 grid((unsigned)((a.r.T + a.per_block - 1) / a.per_block));
    if (e4m3) {
        if (read) paged_copy_kernel<D, true, true><<<grid, 256, 0, st>>>(a);
        else paged_copy_kernel<D, true, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (read) paged_copy_kernel<D, false, true><<<grid, 256, 0, st>>>(a);
        else paged_copy_kernel<D, false, false><<<grid, 256, 0, st>>>(a);
    }
}

hipError_t launch_paged_append(const uint16_t* k, int64_t k_st, int64_t k_sh, const uint16_t* v, int64_t v_st, int64_t v_sh,
                               const int32_t* cu, int B, int T, const int32_t* table, int P, const int32_t* kv_len, int shift,
                               int num_pages, int Hkv, int D, bool e4m3, char* pool, uint8_t* scale, int* err, hipStream_t st) {
    const CopyArgs a{paged_rows(cu, B, T, table, P, kv_len, shift, num_pages, Hkv, err), k, v, k_st, k_sh, v_st, v_sh,
                     nullptr, nullptr, pool, scale, copy_tokens(T, Hkv, D)};
    if (D == 128) paged_copy<128>(a, e4m3, false, st);
    else paged_copy<64>(a, e4m3, false, st);
    return hipGetLastError();
}

hipError_t launch_paged_read(uint16_t* k, uint16_t* v, const int32_t* cu, int B, int T, const int32_t* table, int P,
                             const int32_t* kv_len, int shift, int num_pages, int Hkv, int D, bool e4m3, char* pool,
                             uint8_t* scale, int* err, hipStream_t st) {
    const CopyArgs a{paged_rows(cu, B, T, table, P, kv_len, shift, num_pages, Hkv, err), nullptr, nullptr, 0, 0, 0, 0,
                     k, v, pool, scale, copy_tokens(T, Hkv, D)};
    if (D == 128) paged_copy<128>(a, e4m3, true, st);
    else paged_copy<64>(a, e4m3, true, st);
    return hipGetLastError();
}

// How attention cuts a call's work, from what the host knows.
struct PagedPlan {
    int rows;            // of a workgroup: 32 (few rows a request), 128 or 256
    int units;           // workgroups a kv head that the keys are cut for, 0 = not cut
    int64_t grid;        // workgroups, at most
    int64_t bytes;       // workspace
};
PagedPlan paged_plan(int64_t T, int B, int H, int Hkv, int D, int64_t capacity, int cus) {
    const int64_t G = H / Hkv, live = T < B ? T : B;
    PagedPlan p;
    // Up to 32 rows a request and kv head on average, the keys are read once either way.  Beyond, every tile of 32 rows reads
    // them again, which costs less than the few, long workgroups of 128 rows as long as it is little in all: 16 new tokens of one
    // request, 32 heads over 8, behind 2000 tokens: 12.8 us against 19.8; behind 8000 (2^17 tokens x tiles) 21.4 against
    // 24.4; behind 32 000 50 against 42; 8 such requests behind 2000 (2^18) 31 against 26.  (The host knows the tables' size, not the lengths.)
    const bool step = T * G <= 32 * live || (T * G + 31) / 32 * Hkv <= (1 << 17) / capacity;
    p.rows = step ? 32 : D == 128 && T * H >= WIDE_ROWS ? 256 : 128;
    const int64_t tiles = T * G / p.rows + live, target = (p.rows == 256 ? 1 : 2) * (int64_t)cus;        // workgroups that fit the chip
    // rows alone that give every CU eight workgroups are not cut further; neither is what fits one part
    p.units = tiles * Hkv >= 4 * target || capacity <= (step ? MIN_KEYS<32> : MIN_KEYS<128>) ? 0 : (int)((target + Hkv - 1) / Hkv);
    p.grid = (p.units > 0 ? tiles + p.units + 1 : T * G / p.rows + B) * Hkv;
    p.bytes = p.units > 0 ? p.grid * p.rows * ((int64_t)D * 4 + 8) + T * H * 8 : 0;
    return p;
}

template <int D, bool E4M3>
static void paged_attention(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
    const int64_t rows = (int64_t)a.r.T * a.H;
    const dim3 grid((unsigned)p.grid), join((unsigned)((rows + 3) / 4));
    if (p.rows == 32) {
        paged_step_kernel<D, E4M3><<<grid, 256, 0, st>>>(a);
        if (p.units > 0) paged_join_kernel<D, 32, 4><<<dim3((unsigned)rows), 256, 0, st>>>(a);        // few rows, many parts
    } else if (p.rows == 256) {
        if constexpr (D == 128) {
            paged_attention_kernel<D, E4M3, 8><<<grid, 512, 0, st>>>(a);
            if (p.units > 0) paged_join_kernel<D, 256, 1><<<join, 256, 0, st>>>(a);
        }
    } else {
        paged_attention_kernel<D, E4M3, 4><<<grid, 256, 0, st>>>(a);
        if (p.units > 0) paged_join_kernel<D, 128, 1><<<join, 256, 0, st>>>(a);
    }
}

int64_t paged_attention_threads(int64_t T, int B, int H, int Hkv, int D, int64_t capacity, int cus) {
    const PagedPlan p = paged_plan(T, B, H, Hkv, D, capacity, cus);
    return p.grid * (p.rows == 256 ? 512 : 256);
}
int64_t paged_workspace_bytes(int64_t T, int B, int H, int Hkv, int D, int64_t capacity, int cus) {
    return paged_plan(T, B, H, Hkv, D, capacity, cus).bytes;
}

hipError_t launch_paged_attention(const uint16_t* q, int64_t q_st, int64_t q_sh, const int32_t* cu, int B, int T,
                                  const int32_t* table, int P, const int32_t* kv_len, int shift, int num_pages, int H,
                                  int Hkv, int D, bool e4m3, const char* pool, const uint8_t* scale, int* err, float c, int cus,
                                  uint16_t* out, float* lse, char* ws, hipStream_t st) {
    const PagedPlan p = paged_plan(T, B, H, Hkv, D, (int64_t)P << shift, cus);
    PagedAttnArgs a{paged_rows(cu, B, T, table, P, kv_len, shift, num_pages, Hkv, err), q, q_st, q_sh, pool, scale, H, H / Hkv,
                    p.units, c, out, lse, nullptr, nullptr, nullptr, (int)p.grid};
    if (p.units > 0) {
        const int64_t rows = p.grid * p.rows;
        a.part_o = reinterpret_cast<float*>(ws);
        a.part_ml = reinterpret_cast<float2*>(ws + rows * D * 4);
        a.part_of = reinterpret_cast<int2*>(ws + rows * (D * 4 + 8));
    }
    if (D == 128) {
        if (e4m3) paged_attention<128, true>(a, p, st);
        else paged_attention<128, false>(a, p, st);
    } else {
        if (e4m3) paged_attention<64, true>(a, p, st);
        else paged_attention<64, false>(a, p, st);
    }
    return hipGetLastError();
}

}  // namespace mp
