// Attention over the paged K/V cache (dtts_kv_attend).  For the new tokens i of
// every sequence of the current batch and every query head,
//   out_i = sum_j p_ij v_j,  p_ij = softmax_j(scale q_i . k_j)
// over the rows j <= i with window = 0, or j > i - window, or j < sinks.
#include "kv.cuh"

#include <cmath>
#include <type_traits>

namespace dtts {
bool pdl_enabled();
namespace {

DTTS_DEV bool kv_visible(int j, int i, int window, int sinks) {
    return j <= i && (window == 0 || j > i - window || j < sinks);   // nothing for i = -1
}

// The key tiles of KT rows that a range of queries can see: the tiles of the
// first `sinks` rows, then those from the first query's window on.
struct KeyTiles {
    int sink_tiles, win0, n;
    DTTS_DEV KeyTiles(int KT, int i0, int end, int window, int sinks) {
        const int lo = window ? max(0, i0 - window + 1) : 0;
        win0 = lo / KT;
        sink_tiles = min((min(sinks, lo) + KT - 1) / KT, win0);
        n = sink_tiles + (end + KT - 1) / KT - win0;
    }
    DTTS_DEV int tile(int v) const { return v < sink_tiles ? v : win0 + v - sink_tiles; }
};

// Where part s of n tiles in `parts` parts begins: parts differ by a tile at most.
DTTS_DEV int part_start(int n, int parts, int s) {
    const int q = n / parts;
    return s * q + min(s, n - parts * q);
}

// One query row against key tiles [v0, v1) by one warp in plain arithmetic: only
// visible rows are touched, so a non-finite value in a row that this query cannot
// see has no effect on it.  The fast kernels multiply such a row's V by zero and
// come here when that has left a NaN.  32 keys at a time: a lane scores one of
// them, then holds dims D / 32 lane .. of the sum over them.
template <int D>
__device__ __noinline__ void kv_row_plain(const KvAttendArgs &a, const int *trow, int head, const bf16 *q, int i, int KT,
                                          const KeyTiles &kt, int v0, int v1, float &m, float &l, float (&o)[D / 32]) {
    const int lane = threadIdx.x & 31;
    constexpr int C = D / 32;
    m = -INFINITY;
    l = 0.f;
    for (int c = 0; c < C; c++) o[c] = 0.f;
    for (int v = v0; v < v1; v++)
        for (int jj = 0; jj < KT; jj += 32) {
            const int j = kt.tile(v) * KT + jj + lane;
            const bool in = jj + lane < KT && kv_visible(j, i, a.window, a.sinks);   // KT may be 16
            const int page = in ? trow[j >> a.g.lgP] : -1;
            const bool on = (unsigned)page < (unsigned)a.g.n_pages;
            const uint8_t *seg = a.pool + kv_seg_off(a.g, on ? page : 0, 0, head);
            const int r = j & (a.g.P - 1);
            float s = 0.f;
            if (on) {
#pragma unroll 4
                for (int w = 0; w < D / 8; w++) {
                    float x[8];
                    kv_load8(a.g, seg, false, r, w, x);
#pragma unroll
                    for (int d = 0; d < 8; d++) s = fmaf(__bfloat162float(q[8 * w + d]), x[d], s);
                }
            }
            s = on ? s * a.scale_log2 : -INFINITY;
            const float mn = fmaxf(m, warp_max(s)), mu = mn == -INFINITY ? 0.f : mn;   // fmaxf drops a NaN; p keeps it
            const float corr = exp2f(m - mu), p = on ? exp2f(s - mu) : 0.f;
            l = l * corr + warp_sum(p);
            for (int c = 0; c < C; c++) o[c] *= corr;
            const unsigned live = __ballot_sync(0xffffffffu, on);
#pragma unroll 4
            for (int k = 0; k < 32; k++) {
                const float pk = __shfl_sync(0xffffffffu, p, k);
                const long long off = __shfl_sync(0xffffffffu, (long long)(seg - a.pool), k);
                const int rk = __shfl_sync(0xffffffffu, r, k);
                if (!((live >> k) & 1u)) continue;
                float x[8];
                kv_load8(a.g, a.pool + off, true, rk, lane * C / 8, x);
#pragma unroll
                for (int c = 0; c < C; c++) {
                    float xc = 0.f;   // x[lane * C % 8 + c], with a constant index
#pragma unroll
                    for (int d = c; d < 8; d += C) xc = lane * C % 8 + c == d ? x[d] : xc;
                    o[c] += pk * xc;
                }
            }
            m = mn;
        }
}

DTTS_DEV float merge_weight(float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); }

// Joins the parts of `rows` rows (row stride D + 2 floats: O, m, l; part stride
// `part` floats) and stores rows r -> out_of(r).  Parts are taken in order, so
// the result does not depend on which CTA arrived last.  Plain loads, which the fence
// behind the counter orders, eight parts in flight at a time (one after another, a part
// cost 0.28 us); eight dims a thread, so that 8 rows of 128 are one pass of 128 threads.
template <int D, int N, typename OutOf>
DTTS_DEV void kv_join_parts(const float *ws, long long part, int parts, int rows, OutOf out_of) {
    constexpr int kBatch = 8;   // parts in flight at a time
    for (int e = threadIdx.x; e < rows * (D / 8); e += N) {
        const int r = e / (D / 8), c = e % (D / 8);
        const float *w = ws + (long long)r * (D + 2);
        float top = -INFINITY;
        for (int s0 = 0; s0 < parts; s0 += kBatch) {
            float m[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; i++) m[i] = w[min(s0 + i, parts - 1) * part + D];
#pragma unroll
            for (int i = 0; i < kBatch; i++) top = fmaxf(top, m[i]);
        }
        float l = 0.f, o[8];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = 0.f;
        for (int s0 = 0; s0 < parts; s0 += kBatch) {
            float2 ml[kBatch], x[kBatch][4];
#pragma unroll
            for (int i = 0; i < kBatch; i++) {
                const float *p = w + min(s0 + i, parts - 1) * part;
                ml[i] = *reinterpret_cast<const float2 *>(p + D);
#pragma unroll
                for (int j = 0; j < 4; j++) x[i][j] = reinterpret_cast<const float2 *>(p + 8 * c)[j];
            }
#pragma unroll
            for (int i = 0; i < kBatch; i++)
                if (s0 + i < parts) {
                    const float f = merge_weight(ml[i].x, top);
                    l += f * ml[i].y;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        o[2 * j] += f * x[i][j].x;
                        o[2 * j + 1] += f * x[i][j].y;
                    }
                }
        }
        bf16 *dst = out_of(r);
        const float inv = 1.0f / l;   // l = 0: every score was -inf, and 0 * inf is the formula's NaN
        *reinterpret_cast<uint4 *>(dst + 8 * c) =
            make_uint4(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv),
                       pack_bf16x2(o[4] * inv, o[5] * inv), pack_bf16x2(o[6] * inv, o[7] * inv));
    }
}

// Counts the parts of a unit that have been written; true in the CTA that sees
// the last one, which resets the counter for the next call.
DTTS_DEV bool kv_last_part(int *cnt, int parts, int *flag) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const int old = atomicAdd(cnt, 1);
        *flag = old == parts - 1;
        if (old == parts - 1) *cnt = 0;
    }
    __syncthreads();
    const bool last = *flag;
    if (last) __threadfence();
    return last;
}

// ---------------------------------------------------------------- few rows
DTTS_DEV void mbar_expect_tx(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
DTTS_DEV uint32_t movmatrix_t(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <bool HALF>
DTTS_DEV void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// as mma16816<true>, the accumulators starting at c0, c1 (both rows)
DTTS_DEV void mma16816_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                            float c0, float c1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
DTTS_DEV uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
DTTS_DEV __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// (w & mask) | magic in one instruction; both constants stay in registers
DTTS_DEV uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(w), "r"(mask), "r"(magic));
    return y;
}
struct NibbleMasks {
    uint32_t lo, hi, magic;
    DTTS_DEV NibbleMasks() {
        // volatile: as constants they would be folded into two instructions a use
        asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(lo));
        asm volatile("mov.b32 %0, 0x00f000f0;" : "=r"(hi));
        asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
    }
};
// Nibbles (0, 4), (1, 5), (2, 6), (3, 7) of w as half pairs: OR with the bits of
// 1024 gives 1024 + n exactly (n in bits 0-3) or 1024 + 16 n (bits 4-7).
// unpack_raw: n - 8 in pairs 0 and 2, 1024 + 16 n in pairs 1 and 3;
// unpack_nibbles: n - 8 in all.
DTTS_DEV void unpack_raw(uint32_t w, const NibbleMasks &k, __half2 (&h)[4]) {
    const __half2 k1032 = __float2half2_rn(1032.f);
    const uint32_t x = w >> 8;
    h[0] = __hsub2(bits_h2(and_or(w, k.lo, k.magic)), k1032);
    h[1] = bits_h2(and_or(w, k.hi, k.magic));
    h[2] = __hsub2(bits_h2(and_or(x, k.lo, k.magic)), k1032);
    h[3] = bits_h2(and_or(x, k.hi, k.magic));
}
DTTS_DEV void unpack_nibbles(uint32_t w, const NibbleMasks &k, __half2 (&h)[4]) {
    const __half2 k72 = __float2half2_rn(-72.f), sixteenth = __float2half2_rn(0.0625f);
    unpack_raw(w, k, h);
    h[1] = __hfma2(h[1], sixteenth, k72);
    h[3] = __hfma2(h[3], sixteenth, k72);
}

// The largest exponent of the scaling of queries against 4-bit rows: 2^126 and 2^-126 are both normal.  It holds for
// rows below 2^-111; a bf16 number is a multiple of 2^-133, so their values become multiples of 2^-7, as halves exact.
constexpr int kMaxUp = 126;

// Row of a 16-row block that row k of a fragment stands for: adjacent k have rows
// of different parity, and {k = 0, 2, 4, 6}, {1, 3, 5, 7} all four residues mod 4.
__host__ __device__ constexpr int frag_row(int k) { return (k & 8) | ((k & 7) < 4 ? (k & 7) : (k & 7) ^ 1); }

template <int D, bool I4>
struct FewCfg {
    static constexpr int kWarps = 4, kThreads = kWarps * 32;
    static constexpr int KT = I4 ? 64 : D == 64 ? 32 : 16;     // keys a tile
    static constexpr int RB = I4 ? D / 2 : 2 * D, SB = I4 ? D / 16 : 0;
    static constexpr int kBlock = 32 * (RB + SB);              // 16 rows of K and V with their scales
    static constexpr int kStage = KT / 16 * kBlock;
    static constexpr int kStages = 2;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kMerge = kWarps * kKvFewRows * (D + 2) * 4;   // the warps' results, over the rings
    static constexpr int kSmem = (kRing > kMerge ? kRing : kMerge) + kWarps * kStages * 8 + 16;
};

// Attention of at most 8 NT rows (new tokens x query heads of one kv head) of one
// sequence.  Each warp takes every kWarps-th key tile of the CTA's part: bulk
// copies bring a tile's pages into the warp's own ring while earlier tiles are
// computed, so DRAM latency is covered without registers.  Products are m16n8k16
// with the keys (S^T = K Q^T) and then the dims (O^T = V^T P^T) as the 16-row
// side: a group of up to 8 query rows costs one column block, and K and V bytes
// become fragments in registers.  P^T comes from S^T by an in-register 8 x 8
// transpose.
// int4: K enters as its integers with the group's scale applied to the fp32
// partial sums.  Pairs 1 and 3 of a word enter as 64 + n (1024 + 16 n against q /
// 16), and the products' accumulators start at -72 sum of those q: the products
// are exact and a group's sums stay within 80 s sum |q|.  V enters as the exact half
// values c s; Q as half after an exact scaling by a power of two.  P is half (2^-11
// relative, against 2^-8 of the bf16 output); with bf16 rows P is split into two
// bf16 terms (2^-16).
// The running maximum m of a column is raised only when a score passes it by 2^8
// (P <= 2^8 is as exact as P <= 1), so most tiles need no exchange between lanes.
// Measured (12 query heads over 2 of 128): 32 sequences of 4097 .. 32768 4-bit rows 46.2 us, 3.7 TB/s of rows; the
// counters (53% of the issue slots, integer pipe 41% and its neighbour for fp32 and half 41% active, tensor pipe 21%,
// DRAM at half its rate) show no unit at its limit: three warps a scheduler do not cover the chains of instructions
// that turn words into products.  64 of 1000 .. 8191 bf16 rows 52.7 us, 5.7 TB/s, bound by DRAM; one of 48 rows 5.6 us, bound by
// latency.  4 warps of 64-key tiles and three CTAs an SM are best for long ranges: 8 warps of 32 keys and two CTAs
// measured 53.2 us for the first of these and 59.8 for the second, 12 of 64 and one 49.7 and 56.0, when these took
// 47.2 and 53.8.  Short ranges pay for it: 64 sequences of 65 .. 512 4-bit rows took 9.3 us against 8.3 with 8 warps of 32, 64 behind
// windows of 1024 16.1 against 13.5 with 12 of 64 and 15.4 with 8 of 32.  One shape serves all.
template <int D, bool I4, int NT>
__global__ void __launch_bounds__(FewCfg<D, I4>::kThreads, NT == 1 ? 3 : 1) kv_attend_few_kernel(const __grid_constant__ KvAttendArgs a) {
    using C = FewCfg<D, I4>;
    constexpr int KT = C::KT, NK = KT / 16, MI = D / 16, NG = D / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kSmem - 16 - C::kWarps * C::kStages * 8);
    int *flag = reinterpret_cast<int *>(smem + C::kSmem - 16);
    volatile int *abort_flag = flag + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kWarps * C::kStages; i++) mbar_init(bars + i, 1);
        *flag = 0;
        *abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();

    const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
    const int b = unit / a.g.H, head = unit % a.g.H;
    const int cnt = a.m.cnt[b], len = a.m.len[b], row0 = a.m.start[b], G = a.G;
    const int *trow = a.m.table + (long long)a.m.seq[b] * a.g.max_pages;
    const long long rows_ll = (long long)cnt * G;
    if (blockIdx.x == 0 && threadIdx.x == 0 && kv_batch_over(a.g, a.m, a.n_seq, a.total_rows)) atomicCAS(a.err, 0, DEVERR_BATCH);
    // none, or the other kernel's; or rows that a replayed graph was not captured for
    if (rows_ll < 1 || rows_ll > 8 * NT || (long long)row0 + cnt > a.total_rows) {
        if (rows_ll > 8 * NT && !(a.both && rows_ll > kKvFewRows) && threadIdx.x == 0) atomicCAS(a.err, 0, DEVERR_BATCH);
        return;
    }
    const int rows = (int)rows_ll;
    const int i0 = len - cnt;
    const KeyTiles kt(KT, i0, len, a.window, a.sinks);
    const int parts = min(a.splits, max(1, (kt.n + a.tiles_per_split - 1) / a.tiles_per_split));
    if (split >= parts) return;
    const int c0 = part_start(kt.n, parts, split), c1 = part_start(kt.n, parts, split + 1);

    uint8_t *ring = smem + warp * C::kStages * C::kStage;
    uint64_t *bar = bars + warp * C::kStages;
    const int P = a.g.P, chunk = min(P, KT);   // rows of a tile that are one copy
    const int n_mine = (c1 - c0 - warp + C::kWarps - 1) / C::kWarps;
    const uint8_t *head_pool = a.pool + kv_seg_off(a.g, 0, 0, head);
    auto tile_row = [&](int it) { return kt.tile(c0 + warp + it * C::kWarps) * KT; };
    // the page of the tile's first rows, loaded one issue ahead; -1: no tile, or freed
    auto page_of = [&](int it) { return it < n_mine ? trow[tile_row(it) >> a.g.lgP] : -1; };
    // a page that is not there: only a replayed graph can meet one that a query sees
    auto freed = [&](int j) {
        if (j + chunk > (a.window ? i0 - a.window + 1 : 0) || j < a.sinks) atomicCAS(a.err, 0, DEVERR_FREED);
    };
    // one lane requests the tile: a copy per page it touches
    auto issue = [&](int it, int stage, int page) {
        if (lane != 0) return;
        const int j0 = tile_row(it), rows_in = min(len - j0, KT);
        uint8_t *dst = ring + stage * C::kStage;
        if (chunk == KT) {
            const uint32_t bytes = (unsigned)page < (unsigned)a.g.n_pages ? ((rows_in + 15) >> 4) * C::kBlock : 0;
            mbar_arrive_expect_tx(bar + stage, bytes);
            if (bytes)
                bulk_load_1d(dst, head_pool + page * a.g.page_stride + ((j0 & (P - 1)) >> 4) * C::kBlock, bytes, bar + stage);
            else
                freed(j0);
            return;
        }
        for (int r = 0; r < rows_in; r += chunk) {   // whole pages
            if (r) page = trow[(j0 + r) >> a.g.lgP];
            if ((unsigned)page >= (unsigned)a.g.n_pages) {
                freed(j0 + r);
                continue;
            }
            // the phase completes with the arrival behind the last piece; the pieces only add bytes
            const uint32_t bytes = ((min(rows_in - r, chunk) + 15) >> 4) * C::kBlock;
            mbar_expect_tx(bar + stage, bytes);
            bulk_load_1d(dst + (r >> 4) * C::kBlock, head_pool + page * a.g.page_stride, bytes, bar + stage);
        }
        mbar_arrive(bar + stage);
    };
    {
        int pg[C::kStages];
#pragma unroll
        for (int s = 0; s < C::kStages; s++) pg[s] = page_of(s);
#pragma unroll
        for (int s = 0; s < C::kStages; s++)
            if (s < n_mine) issue(s, s, pg[s]);
    }
    int next_page = page_of(C::kStages);

    // Q^T fragments: lane (g, t) holds dims 32 j + 8 t .. + 7 of column g
    uint32_t qf[NT][2 * NG][2];
    float fac[NT][2];            // score factor of columns 2 t, 2 t + 1
    float off[NT][I4 ? NG : 1][2];   // where their partial sums start
    int qi[NT][2], qlo[NT][2];   // their query rows and the last row before their windows
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int col = nt * 8 + g;
        uint4 w[NG];
#pragma unroll
        for (int j = 0; j < NG; j++) {
            w[j] = make_uint4(0u, 0u, 0u, 0u);
            if (col < rows)
                w[j] = *reinterpret_cast<const uint4 *>(a.q + (long long)(row0 + col / G) * a.q_row +
                                                        (long long)(head * G + col % G) * a.q_head + 32 * j + 8 * t);
        }
        float f = a.scale_log2;
        if constexpr (I4) {
            // power of two that brings the largest |q| of the row to [2^14, 2^15)
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const uint32_t e[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                for (int i = 0; i < 4; i++) top = max(top, max(e[i] & 0x7fffu, (e[i] >> 16) & 0x7fffu));
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int ex = (int)(top >> 7);   // biased exponent; 0: zeros and subnormals, 255: inf or NaN
            const int sh = ex == 255 ? 0 : min(14 + 127 - ex, kMaxUp);
            const float up = __uint_as_float((uint32_t)(sh + 127) << 23);
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const uint32_t e[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
                float x[8];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[2 * i] = __uint_as_float(e[i] << 16) * up;
                    x[2 * i + 1] = __uint_as_float(e[i] & 0xffff0000u) * up;
                }
                // pairs 1 and 3 stand against 16 (64 + n): a sixteenth of q, rounded at 2^-24 for the smallest
                const __half2 q1 = __floats2half2_rn(x[1] * 0.0625f, x[5] * 0.0625f);
                const __half2 q3 = __floats2half2_rn(x[3] * 0.0625f, x[7] * 0.0625f);
                qf[nt][2 * j][0] = h2_bits(__floats2half2_rn(x[0], x[4]));
                qf[nt][2 * j][1] = h2_bits(q1);
                qf[nt][2 * j + 1][0] = h2_bits(__floats2half2_rn(x[2], x[6]));
                qf[nt][2 * j + 1][1] = h2_bits(q3);
                const float2 f1 = __half22float2(q1), f3 = __half22float2(q3);
                float sum = (f1.x + f1.y) + (f3.x + f3.y);
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum *= -16.f * 72.f;
                off[nt][j][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                off[nt][j][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
            }
            f *= __uint_as_float((uint32_t)(127 - sh) << 23);
        } else {
#pragma unroll
            for (int j = 0; j < NG; j++) {
                qf[nt][2 * j][0] = w[j].x;
                qf[nt][2 * j][1] = w[j].y;
                qf[nt][2 * j + 1][0] = w[j].z;
                qf[nt][2 * j + 1][1] = w[j].w;
            }
        }
        f = fmaxf(f, 1.17549435e-38f);   // -inf * f stays -inf
        // column g's factor; lanes need those of columns 2 t, 2 t + 1
        fac[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
        fac[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int col2 = nt * 8 + 2 * t + c;
            qi[nt][c] = col2 < rows ? i0 + col2 / G : -1;   // a column without a row sees nothing
            qlo[nt][c] = a.window ? qi[nt][c] - a.window : -1;
        }
    }
    const NibbleMasks nib;

    float o[MI][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[i][nt][c] = 0.f;
    }

    // one tile in shared memory; FULL: every row of it visible to every query row
    auto tile = [&](auto full_c, const uint8_t *sT, int j0) {
        constexpr bool FULL = decltype(full_c)::value;
        float s[NK][NT][4];
#pragma unroll
        for (int kb = 0; kb < NK; kb++) {
            const uint8_t *sK = sT + kb * C::kBlock;
            [[maybe_unused]] const __half *sKs = reinterpret_cast<const __half *>(sK + 32 * C::RB);
            const int ra = frag_row(g), rb = ra + 8;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 4; c++) s[kb][nt][c] = 0.f;
            if constexpr (I4) {
                uint32_t wa[NG], wb[NG];
                __half2 sa[NG / 2], sb[NG / 2];
                if constexpr (D == 128) {
                    *reinterpret_cast<uint4 *>(wa) = *reinterpret_cast<const uint4 *>(sK + ra * C::RB + 16 * t);
                    *reinterpret_cast<uint4 *>(wb) = *reinterpret_cast<const uint4 *>(sK + rb * C::RB + 16 * t);
                    *reinterpret_cast<uint2 *>(sa) = *reinterpret_cast<const uint2 *>(sKs + ra * NG);
                    *reinterpret_cast<uint2 *>(sb) = *reinterpret_cast<const uint2 *>(sKs + rb * NG);
                } else {
                    *reinterpret_cast<uint2 *>(wa) = *reinterpret_cast<const uint2 *>(sK + ra * C::RB + 8 * t);
                    *reinterpret_cast<uint2 *>(wb) = *reinterpret_cast<const uint2 *>(sK + rb * C::RB + 8 * t);
                    sa[0] = *reinterpret_cast<const __half2 *>(sKs + ra * NG);
                    sb[0] = *reinterpret_cast<const __half2 *>(sKs + rb * NG);
                }
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    __half2 ha[4], hb[4];
                    unpack_raw(wa[j], nib, ha);
                    unpack_raw(wb[j], nib, hb);
                    const float fa = j & 1 ? __high2float(sa[j / 2]) : __low2float(sa[j / 2]);
                    const float fb = j & 1 ? __high2float(sb[j / 2]) : __low2float(sb[j / 2]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float d[4];
                        mma16816_from(d, h2_bits(ha[0]), h2_bits(hb[0]), h2_bits(ha[1]), h2_bits(hb[1]), qf[nt][2 * j][0],
                                      qf[nt][2 * j][1], off[nt][j][0], off[nt][j][1]);
                        mma16816<true>(d, h2_bits(ha[2]), h2_bits(hb[2]), h2_bits(ha[3]), h2_bits(hb[3]),
                                       qf[nt][2 * j + 1][0], qf[nt][2 * j + 1][1]);
                        s[kb][nt][0] = fmaf(d[0], fa, s[kb][nt][0]);
                        s[kb][nt][1] = fmaf(d[1], fa, s[kb][nt][1]);
                        s[kb][nt][2] = fmaf(d[2], fb, s[kb][nt][2]);
                        s[kb][nt][3] = fmaf(d[3], fb, s[kb][nt][3]);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    const uint4 wa = *reinterpret_cast<const uint4 *>(sK + ra * C::RB + 16 * ((4 * j + t) ^ kv_swz_k(false, ra)));
                    const uint4 wb = *reinterpret_cast<const uint4 *>(sK + rb * C::RB + 16 * ((4 * j + t) ^ kv_swz_k(false, rb)));
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        mma16816<false>(s[kb][nt], wa.x, wb.x, wa.y, wb.y, qf[nt][2 * j][0], qf[nt][2 * j][1]);
                        mma16816<false>(s[kb][nt], wa.z, wb.z, wa.w, wb.w, qf[nt][2 * j + 1][0], qf[nt][2 * j + 1][1]);
                    }
                }
            }
            if constexpr (!FULL) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int j = j0 + kb * 16 + (c < 2 ? ra : rb);
                        const bool seen = (j <= qi[nt][c & 1]) & ((j > qlo[nt][c & 1]) | (j < a.sinks));
                        s[kb][nt][c] = seen ? s[kb][nt][c] : -INFINITY;
                    }
            }
        }
        // online softmax of the tile; l stays per lane until the end
        bool grow = false;
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float mx = -INFINITY;
#pragma unroll
                for (int kb = 0; kb < NK; kb++) mx = fmaxf(mx, fmaxf(s[kb][nt][c], s[kb][nt][c + 2]));
                top[nt][c] = mx * fac[nt][c];
                grow |= top[nt][c] > m[nt][c] + 8.f;   // m = -inf: any score
            }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float mx = fmaxf(m[nt][c], top[nt][c]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                    const float corr = mx == -INFINITY ? 1.f : ex2_hw(m[nt][c] - mx);
                    m[nt][c] = mx;
                    l[nt][c] *= corr;
#pragma unroll
                    for (int i = 0; i < MI; i++) {
                        o[i][nt][c] *= corr;
                        o[i][nt][c + 2] *= corr;
                    }
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const float mu = m[nt][c] == -INFINITY ? 0.f : m[nt][c];
#pragma unroll
                for (int kb = 0; kb < NK; kb++) {
                    s[kb][nt][c] = ex2_hw(fmaf(s[kb][nt][c], fac[nt][c], -mu));
                    s[kb][nt][c + 2] = ex2_hw(fmaf(s[kb][nt][c + 2], fac[nt][c], -mu));
                    l[nt][c] += s[kb][nt][c] + s[kb][nt][c + 2];
                }
            }
#pragma unroll
        for (int kb = 0; kb < NK; kb++) {
            // P^T fragments
            uint32_t ph[NT][2];
            [[maybe_unused]] uint32_t pl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float x = s[kb][nt][2 * c], y = s[kb][nt][2 * c + 1];
                    if constexpr (I4) {
                        ph[nt][c] = movmatrix_t(h2_bits(__floats2half2_rn(x, y)));
                    } else {
                        const uint32_t hi = pack_bf16x2(x, y);
                        ph[nt][c] = movmatrix_t(hi);
                        pl[nt][c] = movmatrix_t(pack_bf16x2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u)));
                    }
                }
            // the four keys of this lane's V^T columns 2 t, 2 t + 1, 2 t + 8, 2 t + 9
            int r[4];
#pragma unroll
            for (int c = 0; c < 4; c++) r[c] = frag_row(2 * t + (c & 1)) + (c >> 1) * 8;
            const uint8_t *sV = sT + kb * C::kBlock + 16 * C::RB;
            [[maybe_unused]] const __half *sVs = reinterpret_cast<const __half *>(sV + 16 * (C::RB + C::SB));
            // a row no query sees may hold anything: its V counts as zero
            bool dead[4] = {false, false, false, false};
            if constexpr (!FULL) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int j = j0 + kb * 16 + r[c];
                    dead[c] = (j >= len) | ((a.window != 0) & (j <= i0 - a.window) & (j >= a.sinks));
                }
            }
            if constexpr (I4) {
                __half2 sc[2];
                {
                    __half x[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        x[c] = sVs[r[c] * NG + (D == 128 ? g >> 1 : g >> 2)];
                        if (!FULL) x[c] = dead[c] ? __ushort_as_half(0) : x[c];
                    }
                    sc[0] = __halves2half2(x[0], x[1]);
                    sc[1] = __halves2half2(x[2], x[3]);
                }
                constexpr int W = D / 64;   // words (8 dims) a lane owns
                uint32_t w[4][W];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    if constexpr (D == 128)
                        *reinterpret_cast<uint2 *>(w[c]) =
                            *reinterpret_cast<const uint2 *>(sV + r[c] * C::RB + ((8 * g) ^ (kv_swz_v(true, D, r[c]) << 4)));
                    else
                        w[c][0] = *reinterpret_cast<const uint32_t *>(sV + r[c] * C::RB + 4 * g);
                }
#pragma unroll
                for (int x = 0; x < W; x++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {   // dims 4 hf .. 4 hf + 3 of the word
                        __half2 va[4], vb[4];
                        const uint32_t sel = hf ? 0x7632 : 0x5410;
                        unpack_nibbles(__byte_perm(w[0][x], w[1][x], sel), nib, va);
                        unpack_nibbles(__byte_perm(w[2][x], w[3][x], sel), nib, vb);
#pragma unroll
                        for (int n = 0; n < 4; n++) { va[n] = __hmul2(va[n], sc[0]); vb[n] = __hmul2(vb[n], sc[1]); }
#pragma unroll
                        for (int n = 0; n < 2; n++)
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
                                mma16816<true>(o[4 * x + 2 * hf + n][nt], h2_bits(va[2 * n]), h2_bits(va[2 * n + 1]),
                                               h2_bits(vb[2 * n]), h2_bits(vb[2 * n + 1]), ph[nt][0], ph[nt][1]);
                    }
            } else {
                constexpr int U = D / 64;   // 16-byte units (8 dims) a lane owns
#pragma unroll
                for (int x = 0; x < U; x++) {
                    uint32_t w[4][4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        *reinterpret_cast<uint4 *>(w[c]) =
                            *reinterpret_cast<const uint4 *>(sV + r[c] * C::RB + 16 * ((U * g + x) ^ kv_swz_v(false, D, r[c])));
#pragma unroll
                        for (int n = 0; n < 4; n++)
                            if (!FULL) w[c][n] = dead[c] ? 0u : w[c][n];
                    }
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const uint32_t a0 = __byte_perm(w[0][n], w[1][n], 0x5410), a1 = __byte_perm(w[0][n], w[1][n], 0x7632);
                        const uint32_t a2 = __byte_perm(w[2][n], w[3][n], 0x5410), a3 = __byte_perm(w[2][n], w[3][n], 0x7632);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            mma16816<false>(o[4 * x + n][nt], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
                            mma16816<false>(o[4 * x + n][nt], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
                        }
                    }
                }
            }
        }
    };
    for (int it = 0, stage = 0, ph = 0; it < n_mine; it++) {
        const int j0 = tile_row(it);
        if (!mbar_wait_warp(bar + stage, ph, abort_flag, a.err, DEVERR_TIMEOUT_PRODUCER)) break;
        const uint8_t *sT = ring + stage * C::kStage;
        if (j0 + KT - 1 <= i0 && (a.window == 0 || j0 > len - 1 - a.window || j0 + KT - 1 < a.sinks))
            tile(std::true_type{}, sT, j0);
        else
            tile(std::false_type{}, sT, j0);
        __syncwarp();   // every lane has read the stage
        if (it + C::kStages < n_mine) {
            issue(it + C::kStages, stage, next_page);
            next_page = page_of(it + C::kStages + 1);
        }
        if (++stage == C::kStages) { stage = 0; ph ^= 1; }
    }
    // a wait that ran out: let this warp's copies land before the rings are reused
    if (__any_sync(0xffffffffu, *abort_flag != 0)) {
        const unsigned long long t0 = globaltimer_ns();
        for (int s = 0; s < C::kStages && s < n_mine; s++) {
            const int last = (n_mine - 1 - s) / C::kStages;   // phases of this stage, if all were issued
            for (int ph = 0; ph <= last; ph++)
                while (!mbar_try_wait(bar + s, ph & 1) && globaltimer_ns() - t0 < kWaitLimitNs / 4) {}
        }
        __syncwarp();
    }

    // ---- join the warps: rows of D + 2 floats (O, m, l) a warp
    bool bad = false;
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 4; c++) bad |= o[i][nt][c] != o[i][nt][c] && qi[nt][c & 1] >= 0;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
    __syncthreads();   // all rings are free
    float *res = reinterpret_cast<float *>(smem);
    constexpr int RS = D + 2, WS = kKvFewRows * RS;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int col = nt * 8 + 2 * t + c;
            float *dst = res + warp * WS + col * RS;
#pragma unroll
            for (int i = 0; i < MI; i++)
                *reinterpret_cast<float2 *>(dst + (D / 8) * g + 2 * i) = make_float2(o[i][nt][c], o[i][nt][c + 2]);
            if (g == 0) {
                dst[D] = m[nt][c];
                dst[D + 1] = l[nt][c];
            }
        }
    if (__syncthreads_or(bad)) {
        // a NaN: recompute the part so that rows a query cannot see do not reach it
        for (int r = warp; r < rows; r += C::kWarps) {
            float mm, ll, oo[D / 32];
            kv_row_plain<D>(a, trow, head, a.q + (long long)(row0 + r / G) * a.q_row + (long long)(head * G + r % G) * a.q_head,
                            i0 + r / G, KT, kt, c0, c1, mm, ll, oo);
            for (int w = 0; w < C::kWarps; w++) {
                float *dst = res + w * WS + r * RS;
                for (int c = 0; c < D / 32; c++) dst[D / 32 * lane + c] = w ? 0.f : oo[c];
                if (lane == 0) { dst[D] = w ? -INFINITY : mm; dst[D + 1] = w ? 0.f : ll; }
            }
        }
        __syncthreads();
    }
    float *ws = a.ws + ((long long)unit * a.splits + split) * WS;
    for (int e = threadIdx.x; e < rows * (D / 8); e += C::kThreads) {
        const int r = e / (D / 8), c = e % (D / 8);
        float top = -INFINITY, ll = 0.f, x[8];
#pragma unroll
        for (int w = 0; w < C::kWarps; w++) top = fmaxf(top, res[w * WS + r * RS + D]);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = 0.f;
#pragma unroll
        for (int w = 0; w < C::kWarps; w++) {
            const float *src = res + w * WS + r * RS;
            const float f = merge_weight(src[D], top);
            ll += f * src[D + 1];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] += f * src[8 * c + i];
        }
        if (parts == 1) {
            const float inv = 1.0f / ll;   // ll = 0: every score was -inf, and 0 * inf is the formula's NaN
            *reinterpret_cast<uint4 *>(a.out + (long long)(row0 + r / G) * a.o_row + (long long)(head * G + r % G) * a.o_head +
                                       8 * c) =
                make_uint4(pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv),
                           pack_bf16x2(x[4] * inv, x[5] * inv), pack_bf16x2(x[6] * inv, x[7] * inv));
        } else {
            float *dst = ws + r * RS;
#pragma unroll
            for (int i = 0; i < 4; i++) reinterpret_cast<float2 *>(dst + 8 * c)[i] = make_float2(x[2 * i], x[2 * i + 1]);
            if (c == 0) { dst[D] = top; dst[D + 1] = ll; }
        }
    }
    if (parts == 1) return;
    if (kv_last_part(a.cnt + unit, parts, flag))
        kv_join_parts<D, C::kThreads>(a.ws + (long long)unit * a.splits * WS, WS, parts, rows, [&](int r) {
            return a.out + (long long)(row0 + r / G) * a.o_row + (long long)(head * G + r % G) * a.o_head;
        });
}

// ---------------------------------------------------------------- many rows
// tcgen05 pieces that only this kernel uses.  Its operand tiles are rows of 128 bytes in 64-element chunks with the
// 128-byte swizzle, 8-row groups 1024 bytes apart, so the upper word of every descriptor is the same (stride,
// version, layout: see sdesc_k128) and is put in beside each instruction; the lower one holds the address and,
// for the MN-major V tile, the distance of its chunks.  (A 64-bit descriptor kept across the kernel's loops came out
// of the compiler with its upper word lost.)
constexpr int kChunk = 128 * 128;   // 128 rows x 64 elements of 2 bytes
DTTS_DEV uint32_t desc_k(uint32_t saddr) { return ((saddr >> 4) & 0x3fffu) | (1u << 16); }
DTTS_DEV uint32_t desc_mn(uint32_t saddr) { return ((saddr >> 4) & 0x3fffu) | ((uint32_t)(kChunk >> 4) << 16); }
// D (tmem) (+)= A (smem) B^T (smem)
DTTS_DEV void tc_mma_ss(uint32_t d_tmem, uint32_t adesc, uint32_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, 0x40004040};\n\t"
        "mov.b64 b, {%2, 0x40004040};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(adesc), "r"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// D (tmem) (+)= A (tmem) B (smem, MN-major)
DTTS_DEV void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 b, {%2, 0x40004040};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_tmem), "r"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32 columns on their way to r; r may be used after tmem_ld_wait(r), which waits
// for all loads of the warp
DTTS_DEV void tmem_ld32_issue(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
DTTS_DEV void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29])
                 :
                 : "memory");
    asm volatile("" : "+r"(r[30]), "+r"(r[31])::"memory");   // an asm has 30 operands at most
}
DTTS_DEV void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
DTTS_DEV void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
DTTS_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// byte offset of 16-byte unit u (8 elements) of row r in a tile of 64-element chunks
DTTS_DEV int tile_unit(int r, int u) { return (u >> 3) * kChunk + r * 128 + (((u & 7) ^ (r & 7)) << 4); }

// 256 query rows of one (sequence, key head) pair
struct ManyUnit {
    bool on;
    int b, head, cnt, len, row0, base, rows, i0, i_last, parts;
    KeyTiles kt;
    DTTS_DEV ManyUnit(const KvAttendArgs &a, int bh, int pair)
        : b(bh / a.g.H), head(bh % a.g.H), cnt(a.m.cnt[b]), len(a.m.len[b]), row0(a.m.start[b]), base(pair * 256),
          rows((int)min(256ll, max(0ll, (long long)cnt * a.G - (long long)pair * 256))), i0(len - cnt),
          i_last(i0 + (base + rows - 1) / a.G),
          kt(kKvManyKeyTile, i0 + base / a.G, i_last + 1, a.window, a.sinks) {
        on = (long long)cnt * a.G > kKvFewRows && rows > 0 && (long long)row0 + cnt <= a.total_rows;
        parts = min(a.splits, max(1, (kt.n + a.tiles_per_split - 1) / a.tiles_per_split));
    }
};
// A part's result: O as [D / 4][256 rows][4], then m [256], l [256], so that a warp's rows are contiguous.
template <int D>
DTTS_DEV float *many_part(const KvAttendArgs &a, int unit, int split) {
    return a.ws + ((long long)unit * a.splits + split) * 256 * (D + 2);
}

// Joins the parts of a unit, a row a thread, 16 dims a block (blockIdx.y).  Bound by latency: 8.5 us alone, caches
// cold, for two chunks of 512 tokens in 3 parts.  A kernel of its own, since one CTA a unit that joins after its
// attention is too few: with whole-row loads of Q beside it, this took the two chunks from 79 to 44 us.
template <int D>
__global__ void __launch_bounds__(256) kv_join_many_kernel(const __grid_constant__ KvAttendArgs a, int pairs) {
    pdl_wait();
    pdl_trigger();
    const int unit = blockIdx.x, x0 = blockIdx.y * 16, r = threadIdx.x;
    const ManyUnit n(a, unit / pairs, unit % pairs);
    if (!n.on || n.parts == 1 || r >= n.rows) return;
    float top = -INFINITY;
#pragma unroll 4
    for (int s = 0; s < n.parts; s++) top = fmaxf(top, many_part<D>(a, unit, s)[256 * D + r]);
    float l = 0.f, o[16];
#pragma unroll
    for (int i = 0; i < 16; i++) o[i] = 0.f;
#pragma unroll 2
    for (int s = 0; s < n.parts; s++) {
        const float *p = many_part<D>(a, unit, s);
        const float f = merge_weight(p[256 * D + r], top);
        l += f * p[256 * (D + 1) + r];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 v = reinterpret_cast<const float4 *>(p)[(x0 / 4 + i) * 256 + r];
            o[4 * i] += f * v.x;
            o[4 * i + 1] += f * v.y;
            o[4 * i + 2] += f * v.z;
            o[4 * i + 3] += f * v.w;
        }
    }
    const float inv = 1.0f / l;   // l = 0: every score was -inf, and 0 * inf is the formula's NaN
    const int row = n.base + r;
    uint4 *dst = reinterpret_cast<uint4 *>(a.out + (long long)(n.row0 + row / a.G) * a.o_row +
                                           (long long)(n.head * a.G + row % a.G) * a.o_head + x0);
#pragma unroll
    for (int i = 0; i < 2; i++)
        dst[i] = make_uint4(pack_bf16x2(o[8 * i] * inv, o[8 * i + 1] * inv), pack_bf16x2(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                            pack_bf16x2(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack_bf16x2(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
}

// Where this CTA of the many-row kernel stands: its part, its (sequence, key head), its pair of row tiles
struct ManyPlace {
    int split, bh, pair;
    DTTS_DEV ManyPlace(const KvAttendArgs &a, int pairs, unsigned block) {
        const int u = block / a.splits;
        split = block % a.splits;
        bh = u % (a.n_seq * a.g.H);
        pair = pairs - 1 - u / (a.n_seq * a.g.H);   // longest key ranges first
    }
};

// Sets the error word where the unit has rows that a replayed graph was not captured for: its first CTA calls it.
DTTS_DEV void many_check_batch(const KvAttendArgs &a, int pairs, const ManyPlace &at, const ManyUnit &n) {
    if (at.split || at.pair) return;
    const long long all = (long long)n.cnt * a.G;
    if (all > 256ll * pairs || (all > 0 && all <= kKvFewRows && !a.both) ||
        (at.bh == 0 && kv_batch_over(a.g, a.m, a.n_seq, a.total_rows)))
        atomicCAS(a.err, 0, DEVERR_BATCH);
}

// That, and the error word where a row that the CTA's queries see stands on a page that is not there; a warp calls it.
// Works out its place again: kept live for it, the CTA's variables cost the kernel spilled registers (chunks 1% slower).
DTTS_DEV void many_check(const KvAttendArgs &a, int pairs) {
    constexpr int KT = kKvManyKeyTile;
    unsigned block;   // a blockIdx.x that is not known to be the one from the start
    asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(block));
    const ManyPlace at(a, pairs, block);
    const ManyUnit n(a, at.bh, at.pair);
    if ((threadIdx.x & 31) == 0) many_check_batch(a, pairs, at, n);
    const int *trow = a.m.table + (long long)a.m.seq[n.b] * a.g.max_pages;
    const int step = min(a.g.P, KT), first = n.i0 + n.base / a.G, lo = a.window ? first - a.window + 1 : 0;
    const int v0 = part_start(n.kt.n, n.parts, at.split), v1 = part_start(n.kt.n, n.parts, at.split + 1);
    for (int x = v0 * KT + (threadIdx.x & 31) * step; x < v1 * KT; x += 32 * step) {
        const int j = n.kt.tile(x / KT) * KT + x % KT;
        if (j <= n.i_last && (j + step > lo || j < a.sinks) && trow[j >> a.g.lgP] < 0) atomicCAS(a.err, 0, DEVERR_FREED);
    }
}

template <int D, bool I4>
struct ManyCfg {
    static constexpr int KT = kKvManyKeyTile, kTile = D / 64 * kChunk;   // one operand tile of 128 rows
    static constexpr int kProducerWarps = 6, kThreads = 512;   // beside 8 softmax and 2 issuing warps
    // registers a thread: 128 at launch (512 x 128 = 65536), then 256 x (176 + 80) = 65536
    static constexpr int kSoftmaxRegs = 176, kOtherRegs = 80;
    static constexpr int kSmem = 6 * kTile + 256 + 1024;      // Q x 2, K x 2, V x 2, barriers
    static constexpr int RB = I4 ? D / 2 : 2 * D, SB = I4 ? D / 16 : 0;
    static constexpr uint32_t kF16 = I4 ? 0u : (1u << 7) | (1u << 10);   // operand type: half or bf16
    __host__ __device__ static constexpr uint32_t idesc(int n) {
        return (1u << 4) | kF16 | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    }
};

// pairs (0, 4), (1, 5), (2, 6), (3, 7) of a word's values, as one 16-byte unit
DTTS_DEV uint4 dequant_unit(uint32_t w, const NibbleMasks &k, __half2 s) {
    __half2 h[4];
    unpack_nibbles(w, k, h);
    return make_uint4(h2_bits(__hmul2(h[0], s)), h2_bits(__hmul2(h[1], s)), h2_bits(__hmul2(h[2], s)),
                      h2_bits(__hmul2(h[3], s)));
}
// where dim i of 8 stands inside such a unit
__host__ __device__ constexpr int unit_dim(bool i4, int pos) { return i4 ? (pos >> 1) + (pos & 1) * 4 : pos; }

// two fp32 operations in one instruction
DTTS_DEV float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
DTTS_DEV float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// the lowest n bits, n clamped to 0 .. 32
DTTS_DEV uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// true in one lane of a converged warp
DTTS_DEV bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
    return p != 0;
}

// Waits like mbar_wait, asleep in the barrier for up to a microsecond a try, so that
// a waiting role leaves the issue slots to the working ones; five times as long, for
// a CTA may have to wait for TMEM until another one has recomputed rows.
DTTS_DEV bool kv_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int *err, int code) {
    const uint32_t addr = smem_u32(bar);
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    unsigned long long t0 = 0;
    while (true) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(ok)
            : "r"(addr), "r"(parity)
            : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
        const unsigned long long t = globaltimer_ns();
        if (t0 == 0) t0 = t;
        if (t - t0 > 5 * kWaitLimitNs) {
            if (err) atomicCAS(err, 0, code);
            *abort_flag = 1;
            return false;
        }
    }
}

// Attention of up to 256 rows (new token x query head of one kv head, two tiles of
// 128) of one sequence over a part of its keys, in blocks of 128 keys.
//   warps 0-3, 4-7: softmax of tile 0, 1, one row a thread, half a block (64 keys) at
//                   a time: S from TMEM, P back into the same columns, O rescaled
//                   when the row maximum has grown by more than 2^8 (so P <= 2^8 stays
//                   in half's range);
//   warps 8-13:     K and V rows from the pages into swizzled tiles (4-bit rows become
//                   exact halves on the way), 16 rows of K or V a job, two stages;
//   warps 14, 15:   S = Q K^T and O += P V of tile 0, 1 on tcgen05 (P from TMEM, V
//                   MN-major); while one warp waits, the other's products run.
// A tile has two score buffers of 64 columns: the scores of the next half are
// computed while the softmax of this one runs and P V of the one before, so no role
// waits for a round trip.  Bound by the chain of a half block (scores from TMEM,
// exponentials, P back) with two softmax warps a scheduler beside the unpacking ones: the
// tensor pipe is active 29% of the time, the unit of the exponentials 33%, half the
// issue slots are used.  The operands' shared memory reads would be next; they take
// longer than the products themselves (S: 128 x 64 x 16 a step reads 6 KB in 32 clocks).
// 4-bit rows: all operands half, Q after an exact power-of-two scaling of the row, P
// rounded by 2^-11.  bf16 rows: P is rounded to bf16 (2^-8 of the P-weighted mean
// of |v|, the size of the output's own rounding): a second term would cost half as
// much tensor time again.
// Measured: four prompts of 1501 .. 2047 tokens (12 query heads over 2 of 128, 4 bits) 75 us, 525 TFLOP/s; chunks of
// 512 tokens behind windows of 4096 (bf16) 44.7 us, 586 TFLOP/s.  A CTA per row-tile pair, longest first: resident CTAs
// that draw their pairs from a counter measured 81 and 45 us.
template <int D, bool I4>
__global__ void __launch_bounds__(512, 1) kv_attend_many_kernel(const __grid_constant__ KvAttendArgs a, int pairs) {
    using C = ManyCfg<D, I4>;
    constexpr int KT = C::KT, NU = D / 8;   // 16-byte units a row
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sQ = sm, *sK = sm + 2 * C::kTile, *sV = sm + 4 * C::kTile;
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + 6 * C::kTile);
    // s_full, p_full, pv_done: [tile][half]
    uint64_t *q_full = bars, *s_full = bars + 2, *p_full = bars + 6, *pv_done = bars + 10;
    uint64_t *k_full = bars + 14, *k_empty = bars + 16, *v_full = bars + 18, *v_empty = bars + 20, *drain = bars + 22;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 24);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();

    const ManyPlace at(a, pairs, blockIdx.x);
    const int split = at.split, bh = at.bh, pair = at.pair, unit = bh * pairs + pair;
    const ManyUnit mu(a, bh, pair);
    if (!mu.on || split >= mu.parts) {
        if (tid == 0) many_check_batch(a, pairs, at, mu);
        return;
    }
    const int head = mu.head, len = mu.len, row0 = mu.row0, G = a.G, base = mu.base, rows = mu.rows, parts = mu.parts;
    const int tiles = rows > 128 ? 2 : 1, i0 = mu.i0, i_last = mu.i_last;
    const KeyTiles &kt = mu.kt;
    const int *trow = a.m.table + (long long)a.m.seq[mu.b] * a.g.max_pages;
    const int c0 = part_start(kt.n, parts, split), c1 = part_start(kt.n, parts, split + 1), n = c1 - c0;
    // half blocks of 64 keys; the last one stays out where no row sees it
    const int halves = 2 * n - (kt.tile(c1 - 1) * KT + 64 > i_last ? 1 : 0);

    if (tid == 0) {
        for (int w = 0; w < 2; w++) {
            mbar_init(q_full + w, 128);
            for (int h = 0; h < 2; h++) {
                mbar_init(s_full + 2 * w + h, 1);
                mbar_init(p_full + 2 * w + h, 128);
                mbar_init(pv_done + 2 * w + h, 1);
            }
            mbar_init(k_full + w, 8);
            mbar_init(k_empty + w, tiles);
            mbar_init(v_full + w, 8);
            mbar_init(v_empty + w, tiles);
            mbar_init(drain + w, 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 15) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = *tmem_slot;   // S0 | S1 | O0 | O1
    // only now: the next kernel's CTAs may take TMEM before they wait for this grid
    pdl_trigger();

    // the same answer in all lanes of the warp
    auto wait_all = [&](uint64_t *bar, uint32_t parity, int code) {
        return __all_sync(0xffffffffu, kv_wait(bar, parity, abort_flag, a.err, code)) != 0;
    };
    // the register split stands in the branch that it is for: behind a join the smaller share would hold for both
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
        if (warp >= 14) {
            const int w = warp - 14;
            // The whole warp runs the loop, so that addresses and descriptors stay uniform; one elected lane issues.
            const bool lead = elect_one();
            constexpr uint32_t kTileD = C::kTile >> 4, kHalfD = (64 * 128) >> 4;   // descriptor units of 16 bytes
            const uint32_t qd = desc_k(smem_u32(sQ)) + w * kTileD, kd = desc_k(smem_u32(sK)), vd = desc_mn(smem_u32(sV));
            uint64_t *sf = s_full + 2 * w, *pf = p_full + 2 * w, *pd = pv_done + 2 * w;
            auto scores = [&](int i) {   // of half block i: Q K^T, 64 keys
                const uint32_t kw = kd + ((i >> 1) & 1) * kTileD + (i & 1) * kHalfD;
                const uint32_t d = tbase + w * 128 + (i & 1) * 64;
                if (lead) {
#pragma unroll
                    for (int x = 0; x < D / 16; x++) {
                        const uint32_t off = ((x >> 2) * kChunk + (x & 3) * 32) >> 4;
                        tc_mma_ss(d, qd + off, kw + off, C::idesc(64), x ? 1u : 0u);
                    }
                    tc_commit(sf + (i & 1));
                }
                __syncwarp();
            };
            if (w < tiles) {
                bool ok = wait_all(k_full, 0, DEVERR_TIMEOUT_MMA) && wait_all(q_full + w, 0, DEVERR_TIMEOUT_MMA);
                if (ok) {
                    tc_fence_after();
                    scores(0);
                }
                for (int i = 0; i < halves && ok; i++) {
                    const int k = i >> 1, h = i & 1;
                    if (i + 1 < halves) {
                        // the next half's scores take the columns that P of the half before this one is read from
                        if (h == 1) ok = wait_all(k_full + ((k + 1) & 1), ((k + 1) >> 1) & 1, DEVERR_TIMEOUT_MMA);
                        if (ok && i >= 1) ok = wait_all(pd + (h ^ 1), ((i - 1) >> 1) & 1, DEVERR_TIMEOUT_MMA);
                        if (!ok) break;
                        tc_fence_after();
                        scores(i + 1);
                    }
                    if (h == 0) {
                        if (lead) tc_commit(k_empty + (k & 1));   // both halves' scores are issued
                        __syncwarp();
                        ok = wait_all(v_full + (k & 1), (k >> 1) & 1, DEVERR_TIMEOUT_MMA);
                    }
                    ok = ok && wait_all(pf + h, k & 1, DEVERR_TIMEOUT_MMA);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t vw = vd + (k & 1) * kTileD + h * kHalfD;
                    const uint32_t d = tbase + 256 + w * 128, p = tbase + w * 128 + h * 64;
                    if (lead) {
#pragma unroll
                        for (int x = 0; x < 4; x++)
                            tc_mma_ts(d, p + 8 * x, vw + x * (2048 >> 4), C::idesc(D) | (1u << 16), i || x ? 1u : 0u);
                        tc_commit(pd + h);
                        if (h == 1) tc_commit(v_empty + (k & 1));
                    }
                    __syncwarp();
                }
            }
            // What only a replayed graph can meet, while the last softmax runs: pages that are not there, other rows
            // (in the loop of the unpacking warps this cost the prompts 2%).
            if (w == 1) many_check(a, pairs);
            // every product done before TMEM is given back (also after an abort)
            if (lead) tc_commit(drain + w);
            __syncwarp();
            const unsigned long long t0 = globaltimer_ns();
            while (!mbar_try_wait(drain + w, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {}
            __syncwarp();
        } else {
            // ---- pages -> tiles.  A job is 16 rows of K or V, one block of a page: jobs K0 .. K7, V0 .. V7
            // of key block 0, then of block 1, ...; producer warp pw takes jobs pw, pw + 6, ...  A job's page
            // number is loaded two jobs ahead, its rows one job ahead.
            const int P = a.g.P, lg = a.g.lgP, jobs = 16 * n;
            const uint8_t *head_pool = a.pool + kv_seg_off(a.g, 0, 0, head);
            auto row_of = [&](int job) { return kt.tile(c0 + (job >> 4)) * KT + (job & 7) * 16; };
            auto page_of = [&](int job) {   // -1: nothing to load
                if (job >= jobs) return -1;
                const int j = row_of(job);
                return j < len ? trow[j >> lg] : -1;
            };
            // the job's block of 16 rows and how many of them exist
            auto block_of = [&](int job, int page, int &live) -> const uint8_t * {
                const int j = row_of(job);
                live = (unsigned)page < (unsigned)a.g.n_pages ? len - j : 0;
                return head_pool + (live > 0 ? page : 0) * a.g.page_stride + ((j & (P - 1)) >> 4) * (32 * (C::RB + C::SB));
            };
            auto wait_empty = [&](int job) {
                const int k = job >> 4;
                return k < 2 || wait_all((job & 8 ? v_empty : k_empty) + (k & 1), ((k >> 1) - 1) & 1, DEVERR_TIMEOUT_PRODUCER);
            };
            auto announce = [&](int job) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive((job & 8 ? v_full : k_full) + ((job >> 4) & 1));
            };
            constexpr int kStep = C::kProducerWarps;
            int job = warp - 8;
            if constexpr (I4) {
                // A lane takes unit un = lane / 8 of rows lane % 8 and lane % 8 + 8: a quarter warp then stores eight
                // rows of one unit, which the tile's swizzle spreads over all banks.  K: the words of dims 32 j +
                // 8 un of all groups j; V: the dims of group un (D = 64: two groups a row, row by un / 2).
                const NibbleMasks nib;
                constexpr int kV = D / 64;   // V units a lane
                const int lr = lane & 7, un = lane >> 3, vr = D == 128 ? lr : lr + 8 * (un >> 1), vu = D == 128 ? un : un & 1;
                const uint32_t k_at = lr * C::RB + un * (D / 8), ks_at = 32 * C::RB + lr * C::SB;
                const uint32_t v_at = (16 + vr) * C::RB + 16 * (vu ^ kv_swz_v(true, D, vr));
                const uint32_t vs_at = 32 * C::RB + (16 + vr) * C::SB + 2 * vu;
                const uint32_t k_to = lr * 128 + ((un ^ lr) << 4);                                        // + j: see below
                const uint32_t v_to = (vu >> 1) * kChunk + vr * 128 + (((4 * (vu & 1)) ^ lr) << 4);       // vr % 8 = lr
                struct Raw {
                    uint4 w[2];
                    uint2 s[2];
                };
                auto load = [&](int jb, int page, Raw &raw) {
                    int live;
                    const uint8_t *blk = block_of(jb, page, live);
                    if (jb & 8) {
#pragma unroll
                        for (int x = 0; x < kV; x++) {
                            raw.w[x] = make_uint4(0u, 0u, 0u, 0u);
                            raw.s[x].x = 0u;
                            if (vr + 8 * x >= live) continue;
                            raw.w[x] = *reinterpret_cast<const uint4 *>(blk + v_at + 8 * x * C::RB);   // 8 rows on: the same swap
                            raw.s[x].x = *reinterpret_cast<const uint16_t *>(blk + vs_at + 8 * x * C::SB);
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            raw.w[x] = make_uint4(0u, 0u, 0u, 0u);
                            raw.s[x] = make_uint2(0u, 0u);
                            if (lr + 8 * x >= live) continue;
                            if constexpr (D == 128) {
                                raw.w[x] = *reinterpret_cast<const uint4 *>(blk + k_at + 8 * x * C::RB);
                                raw.s[x] = *reinterpret_cast<const uint2 *>(blk + ks_at + 8 * x * C::SB);
                            } else {
                                const uint2 y = *reinterpret_cast<const uint2 *>(blk + k_at + 8 * x * C::RB);
                                raw.w[x].x = y.x;
                                raw.w[x].y = y.y;
                                raw.s[x].x = *reinterpret_cast<const uint32_t *>(blk + ks_at + 8 * x * C::SB);
                            }
                        }
                    }
                };
                auto store = [&](int jb, const Raw &raw) {
                    uint8_t *dst = (jb & 8 ? sV : sK) + ((jb >> 4) & 1) * C::kTile + (jb & 7) * (16 * 128);
                    if (jb & 8) {
#pragma unroll
                        for (int x = 0; x < kV; x++) {
                            const uint32_t e[4] = {raw.w[x].x, raw.w[x].y, raw.w[x].z, raw.w[x].w};
                            const __half2 sc = bits_h2(__byte_perm(raw.s[x].x, 0u, 0x1010));
#pragma unroll
                            for (int q = 0; q < 4; q++)
                                *reinterpret_cast<uint4 *>(dst + x * 1024 + (v_to ^ (q << 4))) = dequant_unit(e[q], nib, sc);
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const uint32_t e[4] = {raw.w[x].x, raw.w[x].y, raw.w[x].z, raw.w[x].w};
#pragma unroll
                            for (int j = 0; j < D / 32; j++) {   // unit 4 j + un: chunk j / 2, place (4 (j % 2) + un) ^ row
                                const __half2 sc = bits_h2(__byte_perm((j >> 1) ? raw.s[x].y : raw.s[x].x, 0u, j & 1 ? 0x3232 : 0x1010));
                                *reinterpret_cast<uint4 *>(dst + (j >> 1) * kChunk + x * 1024 + (k_to ^ ((j & 1) << 6))) =
                                    dequant_unit(e[j], nib, sc);
                            }
                        }
                    }
                };
                Raw ra, rb;   // this job's rows and the next one's, in turn
                load(job, page_of(job), ra);
                int page = page_of(job + kStep);
                auto one = [&](Raw &cur, Raw &next) {
                    if (job + kStep < jobs) load(job + kStep, page, next);
                    page = page_of(job + 2 * kStep);
                    if (!wait_empty(job)) return false;
                    store(job, cur);
                    announce(job);
                    job += kStep;
                    return job < jobs;
                };
                while (one(ra, rb) && one(rb, ra)) {}
            } else {
                // a job is announced when the second one behind it has been requested
                int issued = 0, page = page_of(job);
                for (; job < jobs; job += kStep, issued++) {
                    int live;
                    const uint8_t *blk = block_of(job, page, live);
                    page = page_of(job + kStep);
                    if (!wait_empty(job)) break;
                    const int is_v = (job >> 3) & 1, r0 = (job & 7) * 16;
                    const uint32_t dst = smem_u32((is_v ? sV : sK) + ((job >> 4) & 1) * C::kTile);
#pragma unroll
                    for (int x = 0; x < 16 * NU / 32; x++) {
                        const int it = lane + 32 * x, r = it / NU, u = it % NU;
                        const int su = u ^ (is_v ? kv_swz_v(false, D, r) : kv_swz_k(false, r));
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + tile_unit(r0 + r, u)),
                                     "l"(blk + (is_v * 16 + r) * C::RB + su * 16), "r"(r < live ? 16 : 0)
                                     : "memory");
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (issued >= 2) {
                        asm volatile("cp.async.wait_group 2;" ::: "memory");
                        announce(job - 2 * kStep);
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                for (int i = min(issued, 2); i > 0; i--) announce(job - i * kStep);
            }
        }
    } else {
        // ---- softmax, a row a thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
        const int w = warp >> 2, r = tid & 127, rr = w * 128 + r;
        if (w < tiles) {
            const bool live = rr < rows;
            const int tok = (base + (live ? rr : 0)) / G, hg = (base + (live ? rr : 0)) % G, qi = live ? i0 + tok : -1;
            // Q: the warp loads its 32 rows two (D = 64: four) at a time, 16 bytes a lane; row offsets and scale
            // factors pass between the row's owner and the lanes that hold it
            constexpr int kRows = 32 / NU, kSteps = 32 / kRows, kBatch = 8;
            const long long q_off = (long long)(row0 + tok) * a.q_row + (long long)(head * G + hg) * a.q_head;
            const int wr = w * 128 + (warp & 3) * 32, lr = lane / NU, u = lane % NU;
            float c = a.scale_log2;
#pragma unroll 1
            for (int s0 = 0; s0 < kSteps; s0 += kBatch) {
                uint4 x[kBatch];
#pragma unroll
                for (int s = 0; s < kBatch; s++) {
                    const int row = (s0 + s) * kRows + lr;
                    const long long off = __shfl_sync(0xffffffffu, q_off, row);
                    x[s] = wr + row < rows ? *reinterpret_cast<const uint4 *>(a.q + off + 8 * u) : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int s = 0; s < kBatch; s++) {
                    if constexpr (I4) {
                        // as in the few-row kernel: the largest |q| of the row to [2^14, 2^15)
                        const uint32_t e[4] = {x[s].x, x[s].y, x[s].z, x[s].w};
                        uint32_t top = 0;
#pragma unroll
                        for (int y = 0; y < 4; y++) top = max(top, max(e[y] & 0x7fffu, (e[y] >> 16) & 0x7fffu));
#pragma unroll
                        for (int y = 1; y < NU; y <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, y));
                        const int ex = (int)(top >> 7), sh = ex == 255 ? 0 : min(14 + 127 - ex, kMaxUp);
                        const float up = __uint_as_float((uint32_t)(sh + 127) << 23);
                        float f[8];
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            f[2 * y] = __uint_as_float(e[y] << 16) * up;
                            f[2 * y + 1] = __uint_as_float(e[y] & 0xffff0000u) * up;
                        }
                        x[s] = make_uint4(h2_bits(__floats2half2_rn(f[0], f[4])), h2_bits(__floats2half2_rn(f[1], f[5])),
                                          h2_bits(__floats2half2_rn(f[2], f[6])), h2_bits(__floats2half2_rn(f[3], f[7])));
                        const int osh = __shfl_sync(0xffffffffu, sh, (lane % kRows) * NU);
                        if (lane / kRows == s0 + s) c *= __uint_as_float((uint32_t)(127 - osh) << 23);
                    }
                    *reinterpret_cast<uint4 *>(sQ + w * C::kTile + tile_unit((warp & 3) * 32 + (s0 + s) * kRows + lr, u)) = x[s];
                }
            }
            c = fmaxf(c, 1.17549435e-38f);   // -inf * c stays -inf
            fence_proxy_async_smem();
            mbar_arrive(q_full + w);
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t ts = tbase + w * 128 + lanes, to = tbase + 256 + w * 128 + lanes;
            const int q_min = i0 + (base + w * 128) / G, q_max = i0 + (base + min(rows, w * 128 + 128) - 1) / G;
            const int qlo = a.window ? qi - a.window : -1;   // the last row before the window
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int i = 0; i < halves; i++) {
                const int h = i & 1, j0 = kt.tile(c0 + (i >> 1)) * KT + 64 * h;
                const uint32_t ti = ts + 64 * h;
                ok = wait_all(s_full + 2 * w + h, (i >> 1) & 1, DEVERR_TIMEOUT_EPILOGUE);
                if (!ok) break;
                tc_fence_after();
                const bool all = j0 + 63 <= q_min && (a.window == 0 || j0 > q_max - a.window || j0 + 63 < a.sinks);
                // scores of columns 32 x .. 32 x + 31, -inf where this row does not see the key
                auto mask = [&](uint32_t (&s)[32], int x) {
                    if (all) return;
                    const uint32_t seen = low_bits(qi - j0 - 32 * x + 1) &
                                          (~low_bits(qlo - j0 - 32 * x + 1) | low_bits(a.sinks - j0 - 32 * x));
#pragma unroll
                    for (int y = 0; y < 32; y++) s[y] = (seen >> y) & 1u ? s[y] : 0xff800000u;
                };
                uint32_t s[2][32], p[2][16];
                tmem_ld32_issue(ti, s[0]);
                tmem_ld32_issue(ti + 32, s[1]);
                tmem_ld_wait(s[0]);
                tmem_ld_wait(s[1]);
                mask(s[0], 0);
                mask(s[1], 1);
                // Exponentials against the running maximum as it stands, the half's own maximum beside them;
                // where that passes it by 2^8 (m = -inf: any score) it is raised, and O and l with it, and the
                // exponentials are done again.
                float2 sum[2];
                while (true) {
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    const float mref = m == -INFINITY ? 0.f : m;
                    const float2 c2 = make_float2(c, c), mu2 = make_float2(-mref, -mref);
                    sum[0] = sum[1] = make_float2(0.f, 0.f);
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int y = 0; y < 16; y++) {
                            const float2 s2 = make_float2(__uint_as_float(s[x][2 * y]), __uint_as_float(s[x][2 * y + 1]));
                            const float2 e = fma2(s2, c2, mu2);
                            const float2 p2 = make_float2(ex2_hw(e.x), ex2_hw(e.y));
                            mx[y & 3] = fmaxf(mx[y & 3], fmaxf(s2.x, s2.y));
                            sum[y & 1] = add2(sum[y & 1], p2);
                            p[x][y] = I4 ? h2_bits(__float22half2_rn(p2)) : pack_bf16x2(p2.x, p2.y);
                        }
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
                    if (!__any_sync(0xffffffffu, top > m + 8.f)) break;
                    const float mn = fmaxf(m, top), corr = mn == -INFINITY ? 1.f : exp2f(m - mn);
                    if (i > 0) {
                        ok = wait_all(pv_done + 2 * w + (h ^ 1), ((i - 1) >> 1) & 1, DEVERR_TIMEOUT_EPILOGUE);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int x = 0; x < D; x += 16) {
                            float o[16];
                            uint32_t q[16];
                            tmem_ld16(to + x, o);
#pragma unroll
                            for (int y = 0; y < 16; y++) q[y] = __float_as_uint(o[y] * corr);
                            tmem_st16(to + x, q);
                        }
                    }
                    l *= corr;
                    m = mn;
                }
                if (!ok) break;
                tmem_st16(ti, p[0]);
                tmem_st16(ti + 16, p[1]);
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(p_full + 2 * w + h);
            }
            const int last = halves - 1;   // its product follows all others into O
            if (ok && wait_all(pv_done + 2 * w + (last & 1), (last >> 1) & 1, DEVERR_TIMEOUT_EPILOGUE)) {
                tc_fence_after();
                float *wp = many_part<D>(a, unit, split);
                uint8_t *sO = sQ + w * C::kTile;   // Q is dead: O's rows on their way to whole-row stores
                const float inv = 1.0f / l;   // l = 0: every score was -inf, and 0 * inf is the formula's NaN
                bool bad = false;
#pragma unroll 1
                for (int x = 0; x < D; x += 32) {
                    float o[32];
                    tmem_ld32(to + x, o);
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            v[unit_dim(I4, i)] = o[8 * y + i];
                            bad |= o[8 * y + i] != o[8 * y + i];
                        }
                        if (parts == 1) {
                            *reinterpret_cast<uint4 *>(sO + tile_unit(r, x / 8 + y)) =
                                make_uint4(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv),
                                           pack_bf16x2(v[4] * inv, v[5] * inv), pack_bf16x2(v[6] * inv, v[7] * inv));
                        } else {
                            float4 *dst = reinterpret_cast<float4 *>(wp) + (x / 4 + 2 * y) * 256 + rr;
                            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                            dst[256] = make_float4(v[4], v[5], v[6], v[7]);
                        }
                    }
                }
                if (parts > 1) {
                    wp[256 * D + rr] = m;
                    wp[256 * (D + 1) + rr] = l;
                }
                __syncwarp();
                // a NaN: recompute the row so that key rows it cannot see do not reach it, before anything is stored
                // over q, which out may be
                for (unsigned todo = __ballot_sync(0xffffffffu, bad && live); todo; todo &= todo - 1) {
                    const int x = __ffs(todo) - 1, xr = wr + x, xt = (base + xr) / G, xh = (base + xr) % G;
                    float mm, ll, oo[D / 32];
                    kv_row_plain<D>(a, trow, head, a.q + (long long)(row0 + xt) * a.q_row + (long long)(head * G + xh) * a.q_head,
                                    i0 + xt, KT, kt, c0, c1, mm, ll, oo);
                    for (int i = 0; i < D / 32; i++) {
                        const int d = D / 32 * lane + i;
                        if (parts == 1)
                            reinterpret_cast<bf16 *>(sO + tile_unit((warp & 3) * 32 + x, d >> 3))[d & 7] = __float2bfloat16_rn(oo[i] / ll);
                        else
                            wp[((d >> 2) * 256 + xr) * 4 + (d & 3)] = oo[i];
                    }
                    if (parts > 1 && lane == 0) {
                        wp[256 * D + xr] = mm;
                        wp[256 * (D + 1) + xr] = ll;
                    }
                    __syncwarp();
                }
                if (parts == 1) {
                    const long long o_off = (long long)(row0 + tok) * a.o_row + (long long)(head * G + hg) * a.o_head;
#pragma unroll 4
                    for (int s = 0; s < kSteps; s++) {
                        const int row = s * kRows + lr;
                        const long long off = __shfl_sync(0xffffffffu, o_off, row);
                        if (wr + row < rows)
                            *reinterpret_cast<uint4 *>(a.out + off + 8 * u) =
                                *reinterpret_cast<const uint4 *>(sO + tile_unit((warp & 3) * 32 + row, u));
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 15) {
        tc_fence_after();
        tmem_dealloc(tbase, 512);
    }
}

template <int D, bool I4>
cudaError_t launch_many(const KvAttendArgs &a, int pairs, cudaStream_t s) {
    const unsigned flags = pdl_enabled() ? kLaunchPdl : 0u, units = (unsigned)a.n_seq * a.g.H * pairs;
    cudaError_t e = launch_k(flags, kv_attend_many_kernel<D, I4>, dim3(units * a.splits), dim3(ManyCfg<D, I4>::kThreads),
                             ManyCfg<D, I4>::kSmem, s, a, pairs);
    if (e != cudaSuccess || a.splits == 1) return e;
    return launch_k(flags, kv_join_many_kernel<D>, dim3(units, D / 16), dim3(256), 0, s, a, pairs);
}

template <int D, bool I4, int NT>
cudaError_t prepare_few(int *ctas) {
    cudaError_t e = cudaFuncSetAttribute(kv_attend_few_kernel<D, I4, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         FewCfg<D, I4>::kSmem);
    if (e != cudaSuccess) return e;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(ctas, kv_attend_few_kernel<D, I4, NT>, FewCfg<D, I4>::kThreads,
                                                         FewCfg<D, I4>::kSmem);
}
template <int D, bool I4>
cudaError_t prepare(KvShapes *k) {
    k->few_key_tile = FewCfg<D, I4>::KT;
    k->few_warps = FewCfg<D, I4>::kWarps;
    // 64 sequences of 300 .. 32768 rows, 12 query heads over 2 of 128: 6.3 + 1.46 x, 8 + 1.45 x, 10 + 1.02 x us for x
    // tiles a warp, with 1, 2, 3 CTAs on an SM (4 bits; why a second CTA adds nothing is not known), 4 + 0.8 x, 0.72 x,
    // 0.68 x (bf16).  9 .. 16 query rows measured 2.2 x, 1.8 x against 4-bit rows.  Not measured: tiles of heads of 64, taken by
    // their size, and 9 .. 16 query rows against bf16 rows, taken like 8.
    constexpr float size = I4 ? D / 128.f : FewCfg<D, I4>::KT * D / 2048.f;
    const float one[3] = {I4 ? 1.46f : 0.8f, I4 ? 1.45f : 0.72f, I4 ? 1.02f : 0.68f}, start[3] = {0.f, I4 ? 1.5f : 0.5f, I4 ? 3.5f : 1.f};
    for (int c = 0; c < 3; c++) {
        k->few_tile_us[0][c] = one[c] * size;
        k->few_tile_us[1][c] = (I4 ? (c ? 1.8f : 2.2f) : one[c]) * size;
        k->few_start_us[c] = start[c];
    }
    cudaError_t e = prepare_few<D, I4, 1>(&k->few_ctas[0]);
    if (e == cudaSuccess) e = prepare_few<D, I4, 2>(&k->few_ctas[1]);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(kv_attend_many_kernel<D, I4>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                ManyCfg<D, I4>::kSmem);
}
template <int D, bool I4>
cudaError_t launch_few(const KvAttendArgs &a, int rows, cudaStream_t s) {
    const dim3 grid((unsigned)a.n_seq * a.g.H * a.splits);
    if (rows <= 8)
        return launch_k(pdl_enabled() ? kLaunchPdl : 0u, kv_attend_few_kernel<D, I4, 1>, grid, dim3(FewCfg<D, I4>::kThreads), FewCfg<D, I4>::kSmem, s, a);
    return launch_k(pdl_enabled() ? kLaunchPdl : 0u, kv_attend_few_kernel<D, I4, 2>, grid, dim3(FewCfg<D, I4>::kThreads), FewCfg<D, I4>::kSmem, s, a);
}

}  // namespace

cudaError_t kv_attend_prepare(const KvGeom &g, KvShapes *k) {
    if (g.i4) return g.D == 128 ? prepare<128, true>(k) : prepare<64, true>(k);
    return g.D == 128 ? prepare<128, false>(k) : prepare<64, false>(k);
}

cudaError_t launch_kv_attend(const KvAttendArgs &a, bool many, int rows_or_pairs, cudaStream_t s) {
    if (many) {
        if (a.g.i4) return a.g.D == 128 ? launch_many<128, true>(a, rows_or_pairs, s) : launch_many<64, true>(a, rows_or_pairs, s);
        return a.g.D == 128 ? launch_many<128, false>(a, rows_or_pairs, s) : launch_many<64, false>(a, rows_or_pairs, s);
    }
    if (a.g.i4) return a.g.D == 128 ? launch_few<128, true>(a, rows_or_pairs, s) : launch_few<64, true>(a, rows_or_pairs, s);
    return a.g.D == 128 ? launch_few<128, false>(a, rows_or_pairs, s) : launch_few<64, false>(a, rows_or_pairs, s);
}

}  // namespace dtts
