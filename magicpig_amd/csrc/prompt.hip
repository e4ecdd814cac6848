// prompt.hip -- causal attention over whole prompts packed one behind the other, query heads in groups.
//
// A workgroup owns 128 or 256 rows (see attn_tile.h: a row is one query head of one token, the G heads of a kv head
// side by side) of one (sequence, kv head) and walks the sequence's keys in tiles of 64 tokens, two buffers in LDS:
// while tile j is folded in, the DMA engine fetches tile j + 1.  Its waves hold 32 rows each.
#include "attn_tile.h"

namespace mp {

struct PromptArgs {
    const uint16_t *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;     // strides of token and head, elements
    const int32_t* cu;
    int B, T, H, Hkv, G, slots;
    float c;
    uint16_t* out;
    float* lse;
};

// Rows of a workgroup at head_dim 128.  256 rows read every key tile from L2 half as often: 16 384 tokens of 8 heads over one
// kv head 511 us against 551, 32 768 tokens of 32 heads over 8 7.88 ms against 8.01.  They need 2^17 rows to give every CU two
// workgroups (8192 tokens of 8 heads: 205 us against 178), and long sequences, whose last workgroup is not a large part of the
// whole (8 sequences of 1000, 32 heads: 101 us against 97).  At head_dim 64 three workgroups of 128 rows fit a CU and one
// of 256 (8100 tokens, 32 heads: 182 us against 167).
constexpr int64_t WIDE_ROWS = 1 << 17, WIDE_TOKENS = 2048;

template <int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void prompt_attention_kernel(const PromptArgs a) {
    constexpr int THREADS = 64 * WAVES, BM = 32 * WAVES, CPR = D / 8, PASSES = TILE_TOKENS * CPR / THREADS, KB = TILE_TOKENS * 2 * D;
    __shared__ __attribute__((aligned(1024))) char lds[2][2][KB];      // [buffer][K, V]
    // heads fastest: with 8 kv heads the workgroups of one head meet in one XCD's L2; the longest first
    const int head = blockIdx.x % a.Hkv, at = (int)(blockIdx.x / a.Hkv);
    const TileOf t = a.B > 1 && a.B <= WAVE ? find_tile_longest_first<BM>(a.cu, a.B, a.T, a.G, at)
                                            : find_tile<BM>(a.cu, a.B, a.T, a.G, a.slots - 1 - at);
    if (t.seq < 0) return;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
    const int rows = t.n * a.G;

    const int wrow = t.row0 + 32 * w;                                   // the wave's first row
    const int row = min(wrow + (l & 31), rows - 1);
    const int tok = row / a.G, h = head * a.G + row % a.G;              // (row: the query's position in its sequence)
    RowState<D> st;
    load_rows<D>(st, a.q + (int64_t)(t.start + tok) * a.q_st + (int64_t)h * a.q_sh);

    const int tiles = min(t.row0 + BM - 1, rows - 1) / a.G / TILE_TOKENS + 1;
    const int whole = (t.row0 / a.G + 1) / TILE_TOKENS;                 // tiles that every row sees whole
    const int seen = wrow < rows ? min(wrow + 31, rows - 1) / a.G / TILE_TOKENS + 1 : 0;    // tiles that the wave's rows see any of

    const char* kb = reinterpret_cast<const char*>(a.k + (int64_t)t.start * a.k_st + (int64_t)head * a.k_sh);
    const char* vb = reinterpret_cast<const char*>(a.v + (int64_t)t.start * a.v_st + (int64_t)head * a.v_sh);
    const uint32_t kst = (uint32_t)a.k_st * 2, vst = (uint32_t)a.v_st * 2;
    auto stage = [&](int tile) {
        const char* kt = kb + (int64_t)tile * TILE_TOKENS * kst;
        const char* vt = vb + (int64_t)tile * TILE_TOKENS * vst;
        const int last = t.n - 1 - tile * TILE_TOKENS;                  // behind the end: the last token again, masked
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int idx = i * THREADS + (int)threadIdx.x, r = idx / CPR, p = idx % CPR;
            const uint32_t s = (uint32_t)min(r, last);
            dma16(kt + (s * kst + ((p ^ key_swizzle<D>(r)) << 4)), lds[tile & 1][0] + (i * THREADS + w * 64) * 16);
            dma16(vt + (s * vst + ((p ^ value_swizzle<D>(r)) << 4)), lds[tile & 1][1] + (i * THREADS + w * 64) * 16);
        }
    };
    stage(0);
    int j = 0;
    for (; j < whole; ++j) {
        tile_barrier();                                                 // tile j is there, tile j - 1 no longer read
        if (j + 1 < tiles) stage(j + 1);
        if (wrow < rows) fold_tile<D, 2, false>(st, lds[j & 1][0], lds[j & 1][1], a.c, 0);
    }
    for (; j < tiles; ++j) {
        tile_barrier();
        if (j + 1 < tiles) stage(j + 1);
        if (j < seen) fold_tile<D, 2, true>(st, lds[j & 1][0], lds[j & 1][1], a.c, tok - j * TILE_TOKENS);
    }
    if (wrow + (l & 31) >= rows) return;
    const int64_t orow = (int64_t)(t.start + tok) * a.H + h;
    store_rows<D>(st, a.out + orow * D, a.lse ? a.lse + orow : nullptr, true);      // (itself at least)
}

// Short prompts: too few workgroups of 128 rows to fill the chip, each walking its keys alone.  Here a workgroup owns 32 rows
// and its four waves take key tiles of 32 tokens in turn, each with its own running softmax over its own block of LDS
// (no barrier until the four are joined); a tile's loads are in flight through registers while the one before is folded in.
template <int D>
__global__ __launch_bounds__(256, 2) void prompt_short_kernel(const PromptArgs a) {
    constexpr int BM = 32, TOK = 32, KB = TOK * 2 * D, CPR = D / 8, PASSES = TOK * CPR / 64;
    __shared__ __attribute__((aligned(1024))) char lds[4][2 * KB];      // a wave's K and V tile; at the end its 32 rows of sums
    __shared__ float2 ml[4][BM];
    const int head = blockIdx.x % a.Hkv;
    const TileOf t = find_tile<BM>(a.cu, a.B, a.T, a.G, a.slots - 1 - (int)(blockIdx.x / a.Hkv));
    if (t.seq < 0) return;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
    const int rows = t.n * a.G;
    RowState<D> st;
    const int row = min(t.row0 + (l & 31), rows - 1), tok = row / a.G;
    load_rows<D>(st, a.q + (int64_t)(t.start + tok) * a.q_st + (int64_t)(head * a.G + row % a.G) * a.q_sh);
    const int tiles = min(t.row0 + BM - 1, rows - 1) / a.G / TOK + 1;
    const int whole = (t.row0 / a.G + 1) / TOK;

    const char* kb = reinterpret_cast<const char*>(a.k + (int64_t)t.start * a.k_st + (int64_t)head * a.k_sh);
    const char* vb = reinterpret_cast<const char*>(a.v + (int64_t)t.start * a.v_st + (int64_t)head * a.v_sh);
    const uint32_t kst = (uint32_t)a.k_st * 2, vst = (uint32_t)a.v_st * 2;
    char *kt = lds[w], *vt = lds[w] + KB;
    u32x4 kr[PASSES], vr[PASSES];
    auto load = [&](int tile) {
        const char* kf = kb + (int64_t)tile * TOK * kst;
        const char* vf = vb + (int64_t)tile * TOK * vst;
        const int last = t.n - 1 - tile * TOK;                          // behind the end: the last token again, masked
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const uint32_t r = (uint32_t)min((i * 64 + l) / CPR, last), p = (uint32_t)(i * 64 + l) % CPR;
            kr[i] = *reinterpret_cast<const u32x4*>(kf + (r * kst + p * 16));
            vr[i] = *reinterpret_cast<const u32x4*>(vf + (r * vst + p * 16));
        }
    };
    // (within a wave LDS works in order; the fences keep the compiler to that order)
    auto store = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = (i * 64 + l) / CPR, p = (i * 64 + l) % CPR;
            *reinterpret_cast<u32x4*>(kt + r * 2 * D + ((p ^ key_swizzle<D>(r)) << 4)) = kr[i];
            *reinterpret_cast<u32x4*>(vt + r * 2 * D + ((p ^ value_swizzle<D>(r)) << 4)) = vr[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    int j = w;
    if (j < tiles) load(j);
    for (; j < whole; j += 4) {
        store();
        __builtin_amdgcn_sched_barrier(0);           // the next tile's loads take the registers just stored
        if (j + 4 < tiles) load(j + 4);
        fold_tile<D, 1, false>(st, kt, vt, a.c, 0);
    }
    if (j < tiles) {                                 // 32 rows end in at most two tiles: one a wave
        store();
        fold_tile<D, 1, true>(st, kt, vt, a.c, tok - j * TOK);
    }

    float m, total;
    f32x4 o[D / 32];
    const int grow = t.row0 + (threadIdx.x >> 3);
    join_waves<D>(st, reinterpret_cast<f32x4*>(lds[w]), reinterpret_cast<const f32x4*>(lds[0]), 2 * KB / 16, ml, m, total, o);
    if (grow >= rows) return;
    const int64_t orow = (int64_t)(t.start + grow / a.G) * a.H + head * a.G + grow % a.G;
    store_chunks<D>(a.out + orow * D, o, total, true);
    if (a.lse != nullptr && (threadIdx.x & 7) == 0) a.lse[orow] = log_sum(m, total);
}

// The short kernel reads the keys once for 32 rows, but four waves share a row's keys.  It wins while its workgroups are at most
// two a CU (2^14 rows; 100 tokens of 32 heads over 8: 5.9 us against 8.6, 2048 tokens of 8 heads: 27 against 43), and up to twice
// as many rows where the sequences are long enough that the other kernel's last workgroups set the time (4096 tokens of 8
// heads: 67 us against 80; 16 x 300 tokens of 8 heads over 1: 22 against 18).  At head_dim 64 "long" starts earlier (768 tokens
// of 32 heads over 8: 10 us against 14).
static bool short_prompts(int64_t T, int B, int H, int D) {
    return T * H <= 1 << 14 || (T * H <= 1 << 15 && T >= (D == 64 ? 512 : 2048) * (int64_t)B);
}
// rows of a workgroup
static int prompt_rows(int64_t T, int B, int H, int D) {
    if (short_prompts(T, B, H, D)) return 32;
    return D == 128 && T * H >= WIDE_ROWS && T >= WIDE_TOKENS * B ? 256 : 128;
}
static int64_t prompt_slots(int64_t T, int B, int H, int Hkv, int D) { return T * (H / Hkv) / prompt_rows(T, B, H, D) + B; }
int64_t prompt_threads(int64_t T, int B, int H, int Hkv, int D) {
    return prompt_slots(T, B, H, Hkv, D) * Hkv * (prompt_rows(T, B, H, D) == 256 ? 512 : 256);
}

hipError_t launch_prompt_attention(const uint16_t* q, int64_t q_st, int64_t q_sh, const uint16_t* k, int64_t k_st,
                                   int64_t k_sh, const uint16_t* v, int64_t v_st, int64_t v_sh, const int32_t* cu, int B,
                                   int T, int H, int Hkv, int D, float c, uint16_t* out, float* lse, hipStream_t st) {
    const int slots = (int)prompt_slots(T, B, H, Hkv, D), rows = prompt_rows(T, B, H, D);
    const PromptArgs a{q, k, v, q_st, q_sh, k_st, k_sh, v_st, v_sh, cu, B, T, H, Hkv, H / Hkv, slots, c, out, lse};
    const dim3 grid((unsigned)((int64_t)slots * Hkv));
    if (rows == 32 && D == 128) prompt_short_kernel<128><<<grid, 256, 0, st>>>(a);
    else if (rows == 32) prompt_short_kernel<64><<<grid, 256, 0, st>>>(a);
    else if (rows == 256) prompt_attention_kernel<128, 8><<<grid, 512, 0, st>>>(a);
    else if (D == 128) prompt_attention_kernel<128, 4><<<grid, 256, 0, st>>>(a);
    else prompt_attention_kernel<64, 4><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace mp
