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

// cache length of request b, inside what its table can hold
__device__ __forceinline__ int cached(const PagedRows& r, int b) {
    const int want = r.kv_len[b], have = (int)min((int64_t)r.P << r.shift, (int64_t)0x7fffffff);
    if (want < 0 || want > have) {
        atomicOr(r.err, 1);
        return want < 0 ? 0 : have;
    }
    return want;
}
// page id -> a page that exists
__device__ __forceinline__ int page_ok(const PagedRows& r, int page) {
    if ((unsigned)page < (unsigned)r.num_pages) return page;
    atomicOr(r.err, 2);
    return -1;
}

// Row of the cache (in units of [K | V] rows) that holds packed row `tok` of kv head `head`, -1: none.
__device__ __forceinline__ int64_t cache_row(const PagedRows& r, int tok, int head) {
    int lo = 0, hi = r.B;            // the first sequence that ends behind tok
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (r.cu[mid + 1] <= tok) lo = mid + 1;
        else hi = mid;
    }
    if (lo >= r.B || r.cu[lo] > tok) return -1;
    const int pos = cached(r, lo) - min(r.cu[lo + 1], r.T) + tok;
    if (pos < 0) return -1;
    const int page = page_ok(r, r.table[(int64_t)lo * r.P + (pos >> r.shift)]);
    return page < 0 ? -1 : ((((int64_t)page * r.Hkv + head) << r.shift) | (pos & ((1 << r.shift) - 1)));
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
};

// One lane carries 8 elements (16 bytes of bf16); a row is D / 8 neighbouring lanes, K and V of a (token, head) neighbouring rows.
// Bound by memory: 4 D bytes in and 4 D (e4m3: 2 D + 2) out per token and kv head.
template <int D, bool E4M3, bool READ>
__global__ __launch_bounds__(256) void paged_copy_kernel(const CopyArgs a) {
    constexpr int LANES = D / 8;
    const int64_t idx = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int c = threadIdx.x % LANES, which = (int)(idx & 1);
    const int64_t th = idx >> 1;
    if (th >= (int64_t)a.r.T * a.r.Hkv) return;
    const int tok = (int)(th / a.r.Hkv), head = (int)(th % a.r.Hkv);
    const int64_t row = cache_row(a.r, tok, head);
    if (row < 0) return;
    if (READ) {
        uint16_t* out = (which ? a.vo : a.ko) + th * D + 8 * c;
        if (!E4M3) {
            *reinterpret_cast<u32x4*>(out) = *reinterpret_cast<const u32x4*>(a.pool + ((row * 2 + which) * LANES + c) * 16);
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2*>(a.pool + ((row * 2 + which) * LANES + c) * 8);
            const float s = __uint_as_float((uint32_t)a.scale[row * 2 + which] << 23);
            u32x4 o;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, false));
                o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, true));
            }
            *reinterpret_cast<u32x4*>(out) = o;
        }
        return;
    }
    const uint16_t* in = which ? a.v + tok * a.v_st + head * a.v_sh : a.k + tok * a.k_st + head * a.k_sh;
    const u32x4 x = *reinterpret_cast<const u32x4*>(in + 8 * c);
    if (!E4M3) {
        *reinterpret_cast<u32x4*>(a.pool + ((row * 2 + which) * LANES + c) * 16) = x;
        return;
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = x[i] & 0x7fffu, hi = (x[i] >> 16) & 0x7fffu;
        top = max(top, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
    }
    top = row_lanes_max<D>(top);
    // exponent - 127 - 8, one more where the mantissa is above 1.75 = 448 / 2^8; as a biased exponent, at least 1
    const int e = max((int)(top >> 7) - 8 + ((top & 127u) > 96u ? 1 : 0), 1);
    const float up = __uint_as_float((uint32_t)(254 - e) << 23);
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(bf16_lo(x[2 * i]) * up, bf16_hi(x[2 * i]) * up, 0, false);
        word = __builtin_amdgcn_cvt_pk_fp8_f32(bf16_lo(x[2 * i + 1]) * up, bf16_hi(x[2 * i + 1]) * up, word, true);
        w[i] = (uint32_t)word;
    }
    *reinterpret_cast<u32x2*>(a.pool + ((row * 2 + which) * LANES + c) * 8) = w;
    if (c == 0) a.scale[row * 2 + which] = (uint8_t)e;
}

// ---------------------------------------------------------------- attention over the pages
struct PagedAttnArgs {
    PagedRows r;
    const uint16_t* q;
    int64_t q_st, q_sh;
    const char* pool;
    const uint8_t* scale;
    int H, G, slots, S;              // S: parts the keys of a row tile may be cut into
    float c;
    uint16_t* out;
    float* lse;
    float* part_o;                   // [S][T * H][D], sums that are not normalised
    float2* part_ml;                 // [S][T * H], their maxima and sums of weights
    int* part_n;                     // [T * H], parts in use
};

constexpr int MIN_TILES = 4;         // a part is at least this many tiles: below, joining costs more than it spreads

// A workgroup owns 128 rows of one (request, kv head) and one part of its keys; everything else is as in prompt.hip.  An
// e4m3 tile passes through registers on its way to LDS: loaded while the tile before it is folded in, widened
// (v_cvt_scalef32_pk_bf16_fp8: exact) behind it.
template <int D, bool E4M3>
__global__ __launch_bounds__(256, 2) void paged_attention_kernel(const PagedAttnArgs a) {
    constexpr int BM = 128, CPR = D / 8, KB = TILE_TOKENS * 2 * D;
    constexpr int PER_ROW = E4M3 ? CPR / 2 : CPR;                     // 16-byte pieces of a cached row
    constexpr int PASSES = TILE_TOKENS * PER_ROW / 256;
    __shared__ __attribute__((aligned(1024))) char lds[2][2][KB];
    const int head = blockIdx.x % a.r.Hkv, split = (int)(blockIdx.x / a.r.Hkv) % a.S;
    const TileOf t = find_tile<BM>(a.r.cu, a.r.B, a.r.T, a.G, a.slots - 1 - (int)(blockIdx.x / a.r.Hkv) / a.S);
    if (t.seq < 0) return;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
    const int rows = t.n * a.G, old = cached(a.r, t.seq) - t.n;       // old: positions in front of the new tokens
    const int lim_lo = old + t.row0 / a.G, lim_hi = old + min(t.row0 + BM - 1, rows - 1) / a.G;
    const int all = lim_hi < 0 ? 0 : lim_hi / TILE_TOKENS + 1;
    const int per = max((all + a.S - 1) / a.S, MIN_TILES);
    const int used = max((all + per - 1) / per, 1);
    if (split >= used) return;
    const int begin = split * per, end = min(all, begin + per);

    const int wrow = t.row0 + 32 * w;
    const int row = min(wrow + (l & 31), rows - 1);
    const int tok = row / a.G, h = head * a.G + row % a.G, lim = old + tok;
    RowState<D> st;
    load_rows<D>(st, a.q + (int64_t)(t.start + tok) * a.q_st + (int64_t)h * a.q_sh);
    const int whole = min(lim_lo < 0 ? 0 : (lim_lo + 1) / TILE_TOKENS, end);
    const int wave_hi = old + min(wrow + 31, rows - 1) / a.G;
    const int seen = wrow < rows && wave_hi >= 0 ? min(wave_hi / TILE_TOKENS + 1, end) : 0;

    const int32_t* table = a.r.table + (int64_t)t.seq * a.r.P;
    const int slot_mask = (1 << a.r.shift) - 1;
    int page[PASSES];
    u32x4 kr[PASSES], vr[PASSES];
    uint32_t sr[PASSES];
    // positions behind the last visible one: that one again, masked
    auto position = [&](int tile, int i) { return min(tile * TILE_TOKENS + (i * 256 + (int)threadIdx.x) / PER_ROW, lim_hi); };
    auto fetch_pages = [&](int tile) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) page[i] = table[position(tile, i) >> a.r.shift];
    };
    auto stage = [&](int tile) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int idx = i * 256 + (int)threadIdx.x, r = idx / PER_ROW, p = idx % PER_ROW;
            const int pg = max(page_ok(a.r, page[i]), 0);
            const int64_t at = (((int64_t)pg * a.r.Hkv + head) << a.r.shift) | (position(tile, i) & slot_mask);
            if (E4M3) {
                const char* src = a.pool + at * (2 * D) + p * 16;
                kr[i] = *reinterpret_cast<const u32x4*>(src);
                vr[i] = *reinterpret_cast<const u32x4*>(src + D);
                sr[i] = *reinterpret_cast<const uint16_t*>(a.scale + at * 2);
            } else {
                const char* src = a.pool + at * (4 * D);
                char* dst = lds[tile & 1][0] + (i * 256 + w * 64) * 16;
                dma16(src + ((p ^ key_swizzle<D>(r)) << 4), dst);
                dma16(src + 2 * D + ((p ^ value_swizzle<D>(r)) << 4), dst + KB);
            }
        }
    };
    auto widen = [&](int tile) {
        if (!E4M3) return;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int idx = i * 256 + (int)threadIdx.x, r = idx / PER_ROW, p = idx % PER_ROW;
            char* kt = lds[tile & 1][0] + r * 2 * D;
            const float ks = __uint_as_float((sr[i] & 255u) << 23), vs = __uint_as_float((sr[i] >> 8) << 23);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                u32x4 kw, vw;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint32_t kc = kr[i][2 * e + x], vc = vr[i][2 * e + x];
                    kw[2 * x] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kc, ks, false));
                    kw[2 * x + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kc, ks, true));
                    vw[2 * x] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vc, vs, false));
                    vw[2 * x + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vc, vs, true));
                }
                *reinterpret_cast<u32x4*>(kt + (((2 * p + e) ^ key_swizzle<D>(r)) << 4)) = kw;
                *reinterpret_cast<u32x4*>(kt + KB + (((2 * p + e) ^ value_swizzle<D>(r)) << 4)) = vw;
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
    auto next = [&](auto fold) {
        tile_barrier();                                               // tile j is there, tile j - 1 no longer read
        if (j + 1 < end) {
            stage(j + 1);
            if (j + 2 < end) fetch_pages(j + 2);
        }
        fold(lds[j & 1][0], lds[j & 1][1]);
        if (j + 1 < end) widen(j + 1);
        ++j;
    };
    while (j < whole) next([&](const char* kt, const char* vt) { if (wrow < rows) fold_tile<D, 2, false>(st, kt, vt, a.c, 0); });
    while (j < end)
        next([&](const char* kt, const char* vt) { if (j < seen) fold_tile<D, 2, true>(st, kt, vt, a.c, lim - j * TILE_TOKENS); });

    if (wrow + (l & 31) >= rows) return;
    const int64_t orow = (int64_t)(t.start + tok) * a.H + h, R = (int64_t)a.r.T * a.H;
    if (split == 0 && a.S > 1 && l < 32) a.part_n[orow] = used;
    if (used == 1) {
        store_rows<D>(st, a.out + orow * D, a.lse ? a.lse + orow : nullptr);
        return;
    }
    float* po = a.part_o + (split * R + orow) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(po + 32 * i + 8 * g + 4 * (l >> 5)) =
                f32x4{st.o[i][4 * g], st.o[i][4 * g + 1], st.o[i][4 * g + 2], st.o[i][4 * g + 3]};
    const float sum = halves_sum(st.l);
    if (l < 32) a.part_ml[split * R + orow] = make_float2(st.m, sum);
}

// Parts of a row joined in their order: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, one wave a row.
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnArgs a) {
    const int64_t R = (int64_t)a.r.T * a.H, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= R) return;
    const int tok = (int)(row / a.H), l = lane_id();
    if (tok < a.r.cu[0] || tok >= a.r.cu[a.r.B]) return;              // (part_n of such a row was never written)
    const int n = min(a.part_n[row], a.S);
    if (n <= 1) return;
    float m = NEG_INF;
    for (int s = l; s < n; s += WAVE) m = fmaxf(m, a.part_ml[s * R + row].x);
    m = wave_max(m);
    const float off = m == NEG_INF ? 0.f : m;
    float sum = 0.f, o[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] = 0.f;
    for (int s0 = 0; s0 < n; s0 += WAVE) {
        const float2 ml = s0 + l < n ? a.part_ml[(s0 + l) * R + row] : make_float2(NEG_INF, 0.f);
        const float w = __builtin_amdgcn_exp2f(ml.x - off);
        sum += wave_sum(w * ml.y);
        const int k = min(n - s0, WAVE);
        for (int s = 0; s < k; ++s) {
            const float ws = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s));
            const float* po = a.part_o + ((s0 + s) * R + row) * D + l * (D / 64);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) o[i] += ws * po[i];
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (D == 128) *reinterpret_cast<uint32_t*>(a.out + row * D + 2 * l) = pack_bf16(o[0] * inv, o[D / 64 - 1] * inv);
    else a.out[row * D + l] = (uint16_t)(pack_bf16(o[0] * inv, 0.f) & 0xffffu);
    if (a.lse != nullptr && l == 0) a.lse[row] = log_sum(m, sum);
}

// ---------------------------------------------------------------- host
int64_t paged_copy_grid(int64_t T, int Hkv, int D) {
    const int rows = 256 / (D / 8);
    return (T * Hkv * 2 + rows - 1) / rows;
}

static PagedRows paged_rows(const int32_t* cu, int B, int T, const int32_t* table, int P, const int32_t* kv_len, int shift,
                            int num_pages, int Hkv, int* err) {
    return PagedRows{cu, table, kv_len, B, T, P, shift, num_pages, Hkv, err};
}

template <int D>
static void paged_copy(const CopyArgs& a, bool e4m3, bool read, hipStream_t st) {
    const dim3 grid((unsigned)paged_copy_grid(a.r.T, a.r.Hkv, D));
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
                     nullptr, nullptr, pool, scale};
    if (D == 128) paged_copy<128>(a, e4m3, false, st);
    else paged_copy<64>(a, e4m3, false, st);
    return hipGetLastError();
}

hipError_t launch_paged_read(uint16_t* k, uint16_t* v, const int32_t* cu, int B, int T, const int32_t* table, int P,
                             const int32_t* kv_len, int shift, int num_pages, int Hkv, int D, bool e4m3, char* pool,
                             uint8_t* scale, int* err, hipStream_t st) {
    const CopyArgs a{paged_rows(cu, B, T, table, P, kv_len, shift, num_pages, Hkv, err), nullptr, nullptr, 0, 0, 0, 0,
                     k, v, pool, scale};
    if (D == 128) paged_copy<128>(a, e4m3, true, st);
    else paged_copy<64>(a, e4m3, true, st);
    return hipGetLastError();
}

static int64_t paged_slots(int64_t T, int B, int G) { return T * G / 128 + B; }
int64_t paged_attention_grid(int64_t T, int B, int G, int Hkv, int S) { return paged_slots(T, B, G) * Hkv * S; }
int64_t paged_join_grid(int64_t T, int H) { return (T * H + 3) / 4; }

// Parts: enough that the row tiles fill the chip (two workgroups a CU), never finer than MIN_TILES tiles of the longest
// possible key list.
int paged_parts(int64_t T, int B, int G, int Hkv, int64_t capacity, int cus) {
    const int64_t tiles = (T * G / 128 + (T < B ? T : B)) * Hkv;
    const int64_t most = (capacity + MIN_TILES * TILE_TOKENS - 1) / (MIN_TILES * TILE_TOKENS);
    int64_t S = 2 * (int64_t)cus / (tiles > 0 ? tiles : 1);
    if (S > most) S = most;
    return S < 1 ? 1 : (int)S;
}
int64_t paged_workspace_bytes(int64_t T, int H, int D, int S) {
    return S > 1 ? S * T * H * ((int64_t)D * 4 + 8) + T * H * 4 : 0;
}

hipError_t launch_paged_attention(const uint16_t* q, int64_t q_st, int64_t q_sh, const int32_t* cu, int B, int T,
                                  const int32_t* table, int P, const int32_t* kv_len, int shift, int num_pages, int H,
                                  int Hkv, int D, bool e4m3, const char* pool, const uint8_t* scale, int* err, float c, int S,
                                  uint16_t* out, float* lse, char* ws, hipStream_t st) {
    const int G = H / Hkv;
    const int64_t R = (int64_t)T * H;
    PagedAttnArgs a{paged_rows(cu, B, T, table, P, kv_len, shift, num_pages, Hkv, err), q, q_st, q_sh, pool, scale, H, G,
                    (int)paged_slots(T, B, G), S, c, out, lse, nullptr, nullptr, nullptr};
    if (S > 1) {
        a.part_o = reinterpret_cast<float*>(ws);
        a.part_ml = reinterpret_cast<float2*>(ws + S * R * D * 4);
        a.part_n = reinterpret_cast<int*>(ws + S * R * (D * 4 + 8));
    }
    const dim3 grid((unsigned)paged_attention_grid(T, B, G, Hkv, S)), join((unsigned)paged_join_grid(T, H));
    if (D == 128) {
        if (e4m3) paged_attention_kernel<128, true><<<grid, 256, 0, st>>>(a);
        else paged_attention_kernel<128, false><<<grid, 256, 0, st>>>(a);
        if (S > 1) paged_join_kernel<128><<<join, 256, 0, st>>>(a);
    } else {
        if (e4m3) paged_attention_kernel<64, true><<<grid, 256, 0, st>>>(a);
        else paged_attention_kernel<64, false><<<grid, 256, 0, st>>>(a);
        if (S > 1) paged_join_kernel<64><<<join, 256, 0, st>>>(a);
    }
    return hipGetLastError();
}

}  // namespace mp
