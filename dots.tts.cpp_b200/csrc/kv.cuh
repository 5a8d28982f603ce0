// The paged K/V cache: page layout, device metadata and the row codec shared by
// its kernels (kv_cache.cu: rows and pages; kv_attend.cu: attention).
//
// Pool: [page][layer][kv head] segments; a segment holds P token rows (16, 32, 64
// or 128) in blocks of 16 rows, each
//   K rows [16][RB] | V rows [16][RB] | K scales [16][SB] | V scales [16][SB]
// with RB = 2 D bytes (bf16) or D / 2 (int4), SB = 0 or D / 16 (one half per 32
// values).  So any run of whole blocks of a page is one contiguous copy.
//
// Row codec, int4: for every 32 consecutive values x (bf16) of a row
//   s = clamp(bf16(max|x| / 7), 2^-14, 9344),  c = clamp(rint(x / s), -7, 7),
// value = c s.  s has 8 significant bits and lies in half's normal range, c has
// 3, so s and every value are exact in half.  A group with a non-finite member
// gets s = NaN.  Nibbles hold c + 8.
//
// Order of the bytes inside a row, chosen for the fragments of the attention
// kernel's m16n8k16 products (a quad lane t = lane % 4, a row lane g = lane / 4):
//   int4 K: the word of dims 32 j + 8 t .. + 7 is word j of unit t (D / 8 bytes a
//           unit), so lane t takes its part of all groups j with one load;
//   int4 V: words in order; D = 128: 32-byte halves swapped in rows with bit 1 set;
//   bf16:   16-byte units (8 dims) XORed with a function of the row.
// The swaps make the loads of the attention kernel free of bank conflicts.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace dtts {

constexpr int kKvGroup = 32;
constexpr float kKvScaleMin = 6.103515625e-05f;   // 2^-14
constexpr float kKvScaleMax = 9344.f;             // 146 * 64: 8 bits, and 7 * 9344 < 65504

struct KvGeom {
    int L, H, D, P, lgP, i4;
    int RB, SB;                       // bytes of a row, of its scales
    long long seg, page_stride;       // bytes of a (page, layer, head) segment, of a page
    int n_pages, max_seqs, max_pages; // pool pages, table rows, pages of a table row
};

// Device metadata (ints): the current batch, then the page tables.
//   seq, start, cnt, len, pos [max_seqs] each: table row of batch entry b, its
//   first row among the batch's rows, its new tokens, its length with them, and
//   the position of its first new token; tables [max_seqs + 1][max_pages] (the
//   last row is the scratch table of a compaction).
struct KvMeta {
    const int *seq, *start, *cnt, *len, *pos, *table;
};

__host__ __device__ inline long long kv_seg_off(const KvGeom &g, int page, int layer, int head) {
    return (long long)page * g.page_stride + ((long long)layer * g.H + head) * g.seg;
}

// byte offset of row r and of its scales within a segment
__host__ __device__ inline int kv_row_off(const KvGeom &g, bool is_v, int r) {
    return (r >> 4) * 32 * (g.RB + g.SB) + (is_v ? 16 * g.RB : 0) + (r & 15) * g.RB;
}
__host__ __device__ inline int kv_scale_off(const KvGeom &g, bool is_v, int r) {
    return (r >> 4) * 32 * (g.RB + g.SB) + 32 * g.RB + (is_v ? 16 * g.SB : 0) + (r & 15) * g.SB;
}

// XOR of the 16-byte unit index inside row r (r: row within the page or tile)
__host__ __device__ constexpr int kv_swz_k(bool i4, int r) { return i4 ? 0 : (r & 1) << 2; }
__host__ __device__ constexpr int kv_swz_v(bool i4, int D, int r) {
    if (i4) return D == 128 ? ((r >> 1) & 1) << 1 : 0;
    return D == 128 ? (((r >> 1) & 1) | (((r >> 2) & 1) << 2)) : ((((r >> 1) & 1) << 1) | (((r >> 2) & 1) << 2));
}
// byte offset of the int4 word that holds dims 8 w .. 8 w + 7 of row r
__host__ __device__ constexpr int kv_word_k(int D, int w) { return (w & 3) * (D / 8) + (w >> 2) * 4; }
__host__ __device__ constexpr int kv_word_v(int D, int w, int r) {
    return (((w >> 2) ^ kv_swz_v(true, D, r)) << 4) + (w & 3) * 4;
}

// b with start[b] <= row < start[b] + cnt[b] among n entries (starts ascend; entries may be empty)
DTTS_DEV int kv_find_entry(const int *start, int n, int row) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {   // last b with start[b] <= row
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= row) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Whether the batch has rows or entries beyond those that a launch was sized for (a
// replayed graph meets the batch that is current then).
DTTS_DEV bool kv_batch_over(const KvGeom &g, const KvMeta &m, int n_seq, int rows) {
    const int beyond = n_seq < g.max_seqs ? m.cnt[n_seq] : 0;   // entries behind the batch hold no rows
    return m.start[n_seq - 1] + m.cnt[n_seq - 1] > rows || beyond > 0;
}

// Quantises 8 packed bf16 values (a quarter of a group whose four lanes are
// neighbours) to one word of nibbles; returns the group's scale through s16.  All
// lanes of the warp take part.
DTTS_DEV uint32_t kv_encode8(uint4 q, __half *s16) {
    const uint32_t e[4] = {q.x, q.y, q.z, q.w};
    // the largest |x|: magnitudes compare as integers, infinity and NaN above all others
    uint32_t top = __vmaxu2(__vmaxu2(e[0] & 0x7fff7fffu, e[1] & 0x7fff7fffu), __vmaxu2(e[2] & 0x7fff7fffu, e[3] & 0x7fff7fffu));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top = max(top & 0xffffu, top >> 16);
    const bool bad = top >= 0x7f80u;
    const float a = __uint_as_float(top << 16);
    // bf16(a / 7) from a product: a / 7 is never nearer than 1 / 14 of the last place (2^-11.8 relative) to a rounding
    // border (2 a 2^t - 14 k - 7 is odd for integers a 2^t and k), and the product is off by 2^-23
    float s = __bfloat162float(__float2bfloat16_rn(a * (1.0f / 7.0f)));
    s = fminf(fmaxf(s, kKvScaleMin), kKvScaleMax);
    *s16 = bad ? __ushort_as_half(0x7e00) : __float2half_rn(s);
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(e[i] << 16);
        x[2 * i + 1] = __uint_as_float(e[i] & 0xffff0000u);
    }
    // up to there |x / s| <= 7 (1 + 2^-8), which rounds to 7 at most
    if (a > 7.f * kKvScaleMax)
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = fminf(fmaxf(x[i], -7.f * kKvScaleMax), 7.f * kKvScaleMax);
    // c = rint(x / s) without a division a value.  x and s have 8 significant bits, so x / s lies on a rounding
    // border n + 1/2 exactly or at least 2^-9.2 away from it (numerator of the difference over 2 s).  x * (1 / s)
    // in one rounding to multiples of 2^-16 (an fma onto 192; 1 / s is good to 2^-23) is off by 2^-17 + 2^-20 at
    // most: on a border it comes out as the border, elsewhere on the right side of it.
    float rs;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rs) : "f"(s));
    uint32_t w = 0;
#pragma unroll
    for (int i = 7; i >= 0; i--) {
        // with the 192 this adds 1.5 * 2^23 + 8: rounds to the nearest even integer and leaves it, plus 8, in the low
        // bits, below 0x4b400000, which adds up to a constant over the word
        w = (w << 4) + __float_as_uint(fmaf(x[i], rs, 192.f) + 12582728.f);
    }
    constexpr uint32_t kAbove = (uint32_t)(0x4b400000ull * 0x11111111ull);
    return bad ? 0x88888888u : w - kAbove;
}

DTTS_DEV float kv_nibble(uint32_t w, int i) { return (float)((int)((w >> (4 * i)) & 15u) - 8); }

// dims 8 w .. 8 w + 7 of row r of a segment (r within the page): what is held, and as floats
struct KvRaw8 {
    uint4 q;      // 4-bit rows: the word in q.x
    __half s;
};
DTTS_DEV KvRaw8 kv_raw8(const KvGeom &g, const uint8_t *seg, bool is_v, int r, int w) {
    KvRaw8 a;
    if (g.i4) {
        a.q.x = *reinterpret_cast<const uint32_t *>(seg + kv_row_off(g, is_v, r) + (is_v ? kv_word_v(g.D, w, r) : kv_word_k(g.D, w)));
        a.s = *reinterpret_cast<const __half *>(seg + kv_scale_off(g, is_v, r) + (w >> 2) * 2);
    } else {
        const int u = w ^ (is_v ? kv_swz_v(false, g.D, r) : kv_swz_k(false, r));
        a.q = *reinterpret_cast<const uint4 *>(seg + kv_row_off(g, is_v, r) + u * 16);
    }
    return a;
}
DTTS_DEV void kv_values8(const KvGeom &g, const KvRaw8 &a, float (&x)[8]) {
    if (g.i4) {
        const float s = __half2float(a.s);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = kv_nibble(a.q.x, i) * s;
    } else {
        const uint32_t e[4] = {a.q.x, a.q.y, a.q.z, a.q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(e[i] << 16);
            x[2 * i + 1] = __uint_as_float(e[i] & 0xffff0000u);
        }
    }
}
DTTS_DEV void kv_load8(const KvGeom &g, const uint8_t *seg, bool is_v, int r, int w, float (&x)[8]) {
    kv_values8(g, kv_raw8(g, seg, is_v, r, w), x);
}

// Stores 8 bf16 values (packed in q) as dims 8 w .. of row r; all lanes of the
// warp call it, four neighbouring lanes hold one group; on: this lane stores.
DTTS_DEV void kv_store8(const KvGeom &g, uint8_t *seg, bool is_v, int r, int w, uint4 q, bool on) {
    if (g.i4) {
        __half s;
        const uint32_t c = kv_encode8(q, &s);
        if (!on) return;
        uint8_t *row = seg + kv_row_off(g, is_v, r);
        *reinterpret_cast<uint32_t *>(row + (is_v ? kv_word_v(g.D, w, r) : kv_word_k(g.D, w))) = c;
        if ((w & 3) == 0)
            *reinterpret_cast<__half *>(seg + kv_scale_off(g, is_v, r) + (w >> 2) * 2) = s;
    } else if (on) {
        const int u = w ^ (is_v ? kv_swz_v(false, g.D, r) : kv_swz_k(false, r));
        *reinterpret_cast<uint4 *>(seg + kv_row_off(g, is_v, r) + u * 16) = q;
    }
}

// ---------------------------------------------------------------- attention
struct KvAttendArgs {
    KvGeom g;
    KvMeta m;
    const uint8_t *pool;     // + the layer's offset
    const bf16 *q;
    bf16 *out;
    long long q_row, q_head, o_row, o_head;   // strides in elements
    int n_seq, G, total_rows;                 // batch entries, query heads per kv head, rows of q / out
    float scale_log2;                         // scale * log2(e)
    int window, sinks;
    int tiles_per_split;                      // key tiles a part of a long key range should hold
    short splits;                             // parts of a long key range: the workspace has room for 8937 at most
    short both;                               // the other kernel (few rows, many rows) is launched too
    // (shorts: with 8 bytes more of parameters a call took the host 0.3 us longer)
    float *ws;                                // partial results
    int *cnt;                                 // arrivals per split unit, zero between calls
    int *err;
};
// What sizes the launches of a cache's attention kernels.
struct KvShapes {
    int few_key_tile, few_warps;   // rows of a key tile; warps of a CTA, which take them in turn
    int few_ctas[2];               // resident CTAs per SM: up to 8, up to 16 query rows
    // microseconds a tile of a warp takes with 1, 2, 3 CTAs on an SM, divided by their number; what a launch of so
    // many takes beside (measured, see kv_attend_prepare)
    float few_tile_us[2][3], few_start_us[3];
};
constexpr int kKvManyKeyTile = 128;
// Sets the kernels' attributes on the current device.
cudaError_t kv_attend_prepare(const KvGeom &g, KvShapes *k);
// many: sequences of more than kKvFewRows rows, in rows_or_pairs pairs of row tiles
// (256 rows) at most; otherwise sequences of up to that many, rows_or_pairs at most
cudaError_t launch_kv_attend(const KvAttendArgs &a, bool many, int rows_or_pairs, cudaStream_t s);
// Rows (new tokens x query heads per kv head) that the few-row kernel takes.  At 12 rows (12 query heads over 2 of 128,
// two tokens) it measured 6.8 us where the many-row kernel takes 8.2 (one sequence of 100 bf16 rows), 24 where that takes 45
// (one of 16000), 51 and 60 (64 of 4000), 39 and 97 (the same in 4 bits), and lost nowhere by more than 0.2 us; at 16 rows
// (16 heads of 64) 4.6 and 7.3, 20 and 34, 167 and 359, 120 and 443.  From 17 rows on, its m16n8k16 columns would be three groups.
constexpr int kKvFewRows = 16;

}  // namespace dtts
