// Attention over the paged K/V cache (dtts_kv_attend).  For the new tokens i of
// every sequence of the current batch and every query head,
//   out_i = sum_j p_ij v_j,  p_ij = softmax_j(scale q_i . k_j)
// over the rows j <= i with window = 0, or j > i - window, or j < sinks.
#include "kv.cuh"

#include <cmath>

namespace dtts {
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

DTTS_DEV float kv_elem(const KvGeom &g, const uint8_t *seg, bool is_v, int r, int d) {
    if (g.i4) {
        const int w = d >> 3;
        const uint8_t *row = seg + (is_v ? g.P * g.RB : 0) + r * g.RB;
        const uint32_t q = *reinterpret_cast<const uint32_t *>(row + (is_v ? kv_word_v(g.D, w, r) : kv_word_k(g.D, w)));
        const float s = __half2float(*reinterpret_cast<const __half *>(
            seg + 2 * g.P * g.RB + (is_v ? g.P * g.SB : 0) + r * g.SB + (d >> 5) * 2));
        return kv_nibble(q, d & 7) * s;
    }
    const int u = (d >> 3) ^ (is_v ? kv_swz_v(false, g.D, r) : kv_swz_k(false, r));
    return __bfloat162float(*reinterpret_cast<const bf16 *>(seg + (is_v ? g.P * g.RB : 0) + r * g.RB + u * 16 + (d & 7) * 2));
}

// One query row against key tiles [v0, v1) by one warp in plain arithmetic: only
// visible rows are touched, so a non-finite value in a row that this query cannot
// see has no effect on it.  The fast kernels multiply such a row's V by zero and
// come here when that has left a NaN.  o[c]: dim lane + 32 c.
template <int D>
__device__ __noinline__ void kv_row_plain(const KvAttendArgs &a, const int *trow, int head, const bf16 *q, int i, int KT,
                                          const KeyTiles &kt, int v0, int v1, float &m, float &l, float (&o)[D / 32]) {
    const int lane = threadIdx.x & 31;
    m = -INFINITY;
    l = 0.f;
    for (int c = 0; c < D / 32; c++) o[c] = 0.f;
    for (int v = v0; v < v1; v++) {
        const int j0 = kt.tile(v) * KT;
        for (int jj = 0; jj < KT; jj++) {
            const int j = j0 + jj;
            if (!kv_visible(j, i, a.window, a.sinks)) continue;
            const int page = trow[j >> a.g.lgP];
            if (page < 0 || page >= a.g.n_pages) continue;
            const uint8_t *seg = a.pool + kv_seg_off(a.g, page, 0, head);
            const int r = j & (a.g.P - 1);
            float s = 0.f;
            for (int c = 0; c < D / 32; c++)
                s = fmaf(__bfloat162float(q[lane + 32 * c]), kv_elem(a.g, seg, false, r, lane + 32 * c), s);
            s = warp_sum(s) * a.scale_log2;
            const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
            const float corr = exp2f(m - mu), p = exp2f(s - mu);
            l = l * corr + p;
            for (int c = 0; c < D / 32; c++) o[c] = o[c] * corr + p * kv_elem(a.g, seg, true, r, lane + 32 * c);
            m = mn;
        }
    }
}

DTTS_DEV float merge_weight(float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); }

// Joins the parts of `rows` rows (row stride D + 2 floats: O, m, l; part stride
// `part` floats) and stores rows r -> out_of(r).  Parts are taken in order, so
// the result does not depend on which CTA arrived last.
template <int D, typename OutOf>
DTTS_DEV void kv_join_parts(const float *ws, long long part, int parts, int rows, OutOf out_of) {
    for (int e = threadIdx.x; e < rows * (D / 8); e += blockDim.x) {
        const int r = e / (D / 8), c = e % (D / 8);
        const float *w = ws + (long long)r * (D + 2);
        float top = -INFINITY;
        for (int s = 0; s < parts; s++) top = fmaxf(top, __ldcg(w + s * part + D));
        float l = 0.f, o[8];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = 0.f;
        for (int s = 0; s < parts; s++) {
            const float f = merge_weight(__ldcg(w + s * part + D), top);
            l += f * __ldcg(w + s * part + D + 1);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 x = __ldcg(reinterpret_cast<const float2 *>(w + s * part + 8 * c) + i);
                o[2 * i] += f * x.x;
                o[2 * i + 1] += f * x.y;
            }
        }
        bf16 *dst = out_of(r);
        if (!dst) continue;
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
DTTS_DEV uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
DTTS_DEV __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// Nibbles (0, 4), (1, 5), (2, 6), (3, 7) of w as half pairs c - 8: OR with the
// bits of 1024 gives 1024 + c exactly (c in bits 0-3) or 1024 + 16 c (bits 4-7).
DTTS_DEV void unpack_nibbles(uint32_t w, __half2 (&h)[4]) {
    const __half2 k1032 = __float2half2_rn(1032.f), k72 = __float2half2_rn(-72.f), sixteenth = __float2half2_rn(0.0625f);
    const uint32_t x = w >> 8;
    h[0] = __hsub2(bits_h2((w & 0x000f000fu) | 0x64006400u), k1032);
    h[1] = __hfma2(bits_h2((w & 0x00f000f0u) | 0x64006400u), sixteenth, k72);
    h[2] = __hsub2(bits_h2((x & 0x000f000fu) | 0x64006400u), k1032);
    h[3] = __hfma2(bits_h2((x & 0x00f000f0u) | 0x64006400u), sixteenth, k72);
}

// Row of a 16-row block that row k of a fragment stands for: adjacent k have rows
// of different parity, and {k = 0, 2, 4, 6}, {1, 3, 5, 7} all four residues mod 4.
__host__ __device__ constexpr int frag_row(int k) { return (k & 8) | ((k & 7) < 4 ? (k & 7) : (k & 7) ^ 1); }

template <int D, bool I4>
struct FewCfg {
    static constexpr int kWarps = 4, kThreads = kWarps * 32;
    static constexpr int KT = I4 ? 64 : (D == 64 ? 32 : 16);   // keys a tile
    static constexpr int RB = I4 ? D / 2 : 2 * D, SB = I4 ? D / 16 : 0;
    static constexpr int kStage = KT * 2 * (RB + SB);
    static constexpr int kStages = I4 ? (D == 128 ? 2 : 4) : 3;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kMerge = kWarps * kKvFewRows * (D + 2) * 4;   // the warps' results, over the rings
    static constexpr int kSmem = (kRing > kMerge ? kRing : kMerge) + kWarps * kStages * 8 + 16;
};

// Attention of at most 8 NT rows (new tokens x query heads of one kv head) of one
// sequence.  Each warp takes every fourth key tile of the CTA's part: bulk copies
// bring a tile's pages into the warp's own ring while earlier tiles are computed,
// so DRAM latency is covered without registers.  Products are m16n8k16 with the
// keys (S^T = K Q^T) and then the dims (O^T = V^T P^T) as the 16-row side: a
// group of up to 8 query rows costs one column block, and K and V bytes become
// fragments in registers.  P^T comes from S^T by an in-register 8 x 8 transpose.
// int4: K enters as the integers c with the group's scale applied to the fp32
// partial sums, V as the exact half values c s; Q as half after an exact scaling
// by a power of two.  P is half (2^-12 relative, against 2^-9 of the bf16
// output); with bf16 rows P is split into two bf16 terms (2^-17).
template <int D, bool I4, int NT>
__global__ void __launch_bounds__(128) kv_attend_few_kernel(const __grid_constant__ KvAttendArgs a) {
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
    const long long rows_ll = (long long)cnt * G;
    if (rows_ll < 1 || rows_ll > kKvFewRows) return;   // none, or the other kernel's
    const int rows = min((int)rows_ll, 8 * NT);
    if ((long long)row0 + cnt > a.total_rows) return;
    const int *trow = a.m.table + (long long)a.m.seq[b] * a.g.max_pages;
    const int i0 = len - cnt;
    const KeyTiles kt(KT, i0, len, a.window, a.sinks);
    const int parts = min(a.splits, max(1, (kt.n + a.tiles_per_split - 1) / a.tiles_per_split));
    if (split >= parts) return;
    const int c0 = (int)((long long)kt.n * split / parts), c1 = (int)((long long)kt.n * (split + 1) / parts);

    uint8_t *ring = smem + warp * C::kStages * C::kStage;
    uint64_t *bar = bars + warp * C::kStages;
    const int P = a.g.P, chunk = min(P, KT);
    // lane = 4 chunk + part copies one part (K, V, their scales) of one page's rows
    auto issue = [&](int v, int stage) {
        const int j0 = kt.tile(v) * KT;
        uint32_t bytes = 0, dst = 0;
        const uint8_t *src = nullptr;
        const int c = lane >> 2, part = lane & 3, j = j0 + c * chunk;
        if (c * chunk < KT && j < len && (I4 || part < 2)) {
            const int last = min(len, j + chunk) - 1;
            // a chunk that lies wholly between the sinks and the first query's window stays out
            const bool seen = a.window == 0 || last > i0 - a.window || j < a.sinks;
            const int page = trow[j >> a.g.lgP];
            if (seen && page >= 0 && page < a.g.n_pages) {
                const int n = (last - j + 16) & ~15;   // rows, whole 16-row blocks
                const int r = j & (P - 1), rb = part < 2 ? C::RB : C::SB;
                const long long off = (part < 2 ? (long long)part * P * C::RB
                                                : 2ll * P * C::RB + (long long)(part - 2) * P * C::SB) + (long long)r * rb;
                bytes = n * rb;
                src = a.pool + kv_seg_off(a.g, page, 0, head) + off;
                dst = (part < 2 ? part * KT * C::RB : 2 * KT * C::RB + (part - 2) * KT * C::SB) + c * chunk * rb;
            }
        }
        const uint32_t total = __reduce_add_sync(0xffffffffu, bytes);
        if (lane == 0) mbar_arrive_expect_tx(bar + stage, total);
        __syncwarp();
        if (bytes) bulk_load_1d(ring + stage * C::kStage + dst, src, bytes, bar + stage);
    };
    const int n_mine = (c1 - c0 - warp + C::kWarps - 1) / C::kWarps;
#pragma unroll
    for (int s = 0; s < C::kStages; s++)
        if (s < n_mine) issue(c0 + warp + s * C::kWarps, s);

    // Q^T fragments: lane (g, t) holds dims 32 j + 8 t .. + 7 of column g
    uint32_t qf[NT][2 * NG][2];
    float fac[NT][2];   // score factor of columns 2 t, 2 t + 1
    int qi[NT][2];      // their query rows
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
            const int sh = ex == 255 ? 0 : min(14 + 127 - ex, 127);
            const float up = __uint_as_float((uint32_t)(max(sh, -126) + 127) << 23);
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const uint32_t e[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
                float x[8];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[2 * i] = __uint_as_float(e[i] << 16) * up;
                    x[2 * i + 1] = __uint_as_float(e[i] & 0xffff0000u) * up;
                }
                qf[nt][2 * j][0] = h2_bits(__floats2half2_rn(x[0], x[4]));
                qf[nt][2 * j][1] = h2_bits(__floats2half2_rn(x[1], x[5]));
                qf[nt][2 * j + 1][0] = h2_bits(__floats2half2_rn(x[2], x[6]));
                qf[nt][2 * j + 1][1] = h2_bits(__floats2half2_rn(x[3], x[7]));
            }
            // column g's factor is 2^-sh scale; lanes need those of columns 2 t, 2 t + 1
            const float down = __uint_as_float((uint32_t)(127 - min(max(sh, -126), 126)) << 23) *
                               (sh == 127 ? 0.5f : 1.0f);
            f *= down;
        } else {
#pragma unroll
            for (int j = 0; j < NG; j++) {
                qf[nt][2 * j][0] = w[j].x;
                qf[nt][2 * j][1] = w[j].y;
                qf[nt][2 * j + 1][0] = w[j].z;
                qf[nt][2 * j + 1][1] = w[j].w;
            }
        }
        fac[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
        fac[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
        // a column without a row sees nothing
        qi[nt][0] = nt * 8 + 2 * t < rows ? i0 + (nt * 8 + 2 * t) / G : -1;
        qi[nt][1] = nt * 8 + 2 * t + 1 < rows ? i0 + (nt * 8 + 2 * t + 1) / G : -1;
    }

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

    for (int it = 0; it < n_mine; it++) {
        const int stage = it % C::kStages, v = c0 + warp + it * C::kWarps, j0 = kt.tile(v) * KT;
        if (!mbar_wait(bar + stage, (it / C::kStages) & 1, abort_flag, a.err, DEVERR_TIMEOUT_PRODUCER)) break;
        const uint8_t *sK = ring + stage * C::kStage, *sV = sK + KT * C::RB;
        const __half *sKs = reinterpret_cast<const __half *>(sK + 2 * KT * C::RB);
        const __half *sVs = sKs + KT * NG;
        // every row of the tile visible to every query row
        const bool full = j0 + KT - 1 <= i0 && (a.window == 0 || j0 > len - 1 - a.window || j0 + KT - 1 < a.sinks);
        float s[NK][NT][4];
#pragma unroll
        for (int kb = 0; kb < NK; kb++) {
            const int ra = kb * 16 + frag_row(g), rb = ra + 8;
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
                    unpack_nibbles(wa[j], ha);
                    unpack_nibbles(wb[j], hb);
                    const float fa = j & 1 ? __high2float(sa[j / 2]) : __low2float(sa[j / 2]);
                    const float fb = j & 1 ? __high2float(sb[j / 2]) : __low2float(sb[j / 2]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
                        mma16816<true>(d, h2_bits(ha[0]), h2_bits(hb[0]), h2_bits(ha[1]), h2_bits(hb[1]),
                                       qf[nt][2 * j][0], qf[nt][2 * j][1]);
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
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    s[kb][nt][c] *= fac[nt][c & 1];
                    if (!full && !kv_visible(j0 + (c < 2 ? ra : rb), qi[nt][c & 1], a.window, a.sinks))
                        s[kb][nt][c] = -INFINITY;
                }
        }
        // online softmax of the tile; l stays per lane until the end
        bool moved = false;
        float corr[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float mx = m[nt][c];
#pragma unroll
                for (int kb = 0; kb < NK; kb++) mx = fmaxf(mx, fmaxf(s[kb][nt][c], s[kb][nt][c + 2]));
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                const float mu = mx == -INFINITY ? 0.f : mx;
                corr[nt][c] = ex2_hw(m[nt][c] - mu);
                moved |= m[nt][c] != mx;
                m[nt][c] = mx;
                float sum = 0.f;
#pragma unroll
                for (int kb = 0; kb < NK; kb++) {
                    s[kb][nt][c] = ex2_hw(s[kb][nt][c] - mu);
                    s[kb][nt][c + 2] = ex2_hw(s[kb][nt][c + 2] - mu);
                    sum += s[kb][nt][c] + s[kb][nt][c + 2];
                }
                l[nt][c] = l[nt][c] * corr[nt][c] + sum;
            }
        if (__any_sync(0xffffffffu, moved))
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[i][nt][c] *= corr[nt][c & 1];
#pragma unroll
        for (int kb = 0; kb < NK; kb++) {
            // P^T fragments
            uint32_t ph[NT][2], pl[NT][2];
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
            for (int c = 0; c < 4; c++) r[c] = kb * 16 + frag_row(2 * t + (c & 1)) + (c >> 1) * 8;
            bool dead[4];   // a row no query sees may hold anything: its V counts as zero
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int j = j0 + r[c];
                dead[c] = !full && (j >= len || (a.window && j <= i0 - a.window && j >= a.sinks));
            }
            if constexpr (I4) {
                __half2 sc[2];
                {
                    __half x[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        x[c] = sVs[r[c] * NG + (D == 128 ? g >> 1 : g >> 2)];
                        if (dead[c]) x[c] = __ushort_as_half(0);
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
                        unpack_nibbles(__byte_perm(w[0][x], w[1][x], sel), va);
                        unpack_nibbles(__byte_perm(w[2][x], w[3][x], sel), vb);
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
                        if (dead[c]) w[c][0] = w[c][1] = w[c][2] = w[c][3] = 0u;
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
        __syncwarp();   // every lane has read the stage
        if (it + C::kStages < n_mine) issue(c0 + warp + (it + C::kStages) * C::kWarps, stage);
    }
    // a wait that ran out: let this warp's copies land before the rings are reused
    if (*abort_flag) {
        const unsigned long long t0 = globaltimer_ns();
        for (int s = 0; s < C::kStages && s < n_mine; s++) {
            const int last = (n_mine - 1 - s) / C::kStages;   // phases of this stage, if all were issued
            for (int ph = 0; ph <= last; ph++)
                while (!mbar_try_wait(bar + s, ph & 1) && globaltimer_ns() - t0 < kWaitLimitNs / 4) {}
        }
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
                for (int c = 0; c < D / 32; c++) dst[lane + 32 * c] = w ? 0.f : oo[c];
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
        kv_join_parts<D>(a.ws + (long long)unit * a.splits * WS, WS, parts, rows, [&](int r) {
            return a.out + (long long)(row0 + r / G) * a.o_row + (long long)(head * G + r % G) * a.o_head;
        });
}

// ---------------------------------------------------------------- many rows
// One warp a row, plain arithmetic.
template <int D>
__global__ void __launch_bounds__(128) kv_attend_rows_kernel(const __grid_constant__ KvAttendArgs a, int row_tiles) {
    pdl_wait();
    pdl_trigger();
    const int tile = blockIdx.x % row_tiles, unit = blockIdx.x / row_tiles;
    const int b = unit / a.g.H, head = unit % a.g.H;
    const int cnt = a.m.cnt[b], len = a.m.len[b], row0 = a.m.start[b], G = a.G;
    const long long rows = (long long)cnt * G;
    if (rows <= kKvFewRows || (long long)row0 + cnt > a.total_rows) return;
    const int *trow = a.m.table + (long long)a.m.seq[b] * a.g.max_pages;
    const KeyTiles kt(64, len - cnt, len, a.window, a.sinks);
    for (long long r = tile * 128ll + (threadIdx.x >> 5); r < min(rows, tile * 128ll + 128); r += 4) {
        const int tok = (int)(r / G), hg = (int)(r % G), lane = threadIdx.x & 31;
        float m, l, o[D / 32];
        kv_row_plain<D>(a, trow, head, a.q + (row0 + tok) * a.q_row + (head * G + hg) * a.q_head, len - cnt + tok, 64, kt, 0,
                        kt.n, m, l, o);
        for (int c = 0; c < D / 32; c++)
            a.out[(row0 + tok) * a.o_row + (head * G + hg) * a.o_head + lane + 32 * c] = __float2bfloat16_rn(o[c] / l);
    }
}

template <int D, bool I4, int NT>
cudaError_t prepare_few() {
    return cudaFuncSetAttribute(kv_attend_few_kernel<D, I4, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                FewCfg<D, I4>::kSmem);
}
template <int D, bool I4>
cudaError_t launch_few(const KvAttendArgs &a, int rows, cudaStream_t s) {
    const dim3 grid((unsigned)a.n_seq * a.g.H * a.splits);
    if (rows <= 8)
        return launch_k(kLaunchPdl, kv_attend_few_kernel<D, I4, 1>, grid, dim3(128), FewCfg<D, I4>::kSmem, s, a);
    return launch_k(kLaunchPdl, kv_attend_few_kernel<D, I4, 2>, grid, dim3(128), FewCfg<D, I4>::kSmem, s, a);
}

}  // namespace

// rows of a key tile of the few-row or the many-row kernel
int kv_key_tile(const KvGeom &g, bool many) {
    if (many) return 64;
    if (g.i4) return g.D == 128 ? FewCfg<128, true>::KT : FewCfg<64, true>::KT;
    return g.D == 128 ? FewCfg<128, false>::KT : FewCfg<64, false>::KT;
}

cudaError_t kv_attend_prepare() {
    cudaError_t e = cudaSuccess;
    if ((e = prepare_few<128, true, 1>()) || (e = prepare_few<128, true, 2>()) || (e = prepare_few<128, false, 1>()) ||
        (e = prepare_few<128, false, 2>()) || (e = prepare_few<64, true, 1>()) || (e = prepare_few<64, true, 2>()) ||
        (e = prepare_few<64, false, 1>()) || (e = prepare_few<64, false, 2>()))
        return e;
    return cudaSuccess;
}

// many: sequences of more than kKvFewRows rows, in rows_or_tiles row tiles of 128
// at most; otherwise sequences of up to that many, rows_or_tiles at most
cudaError_t launch_kv_attend(const KvAttendArgs &a, bool many, int rows_or_tiles, cudaStream_t s) {
    if (many) {
        const dim3 grid((unsigned)a.n_seq * a.g.H * rows_or_tiles);
        return a.g.D == 128 ? launch_k(kLaunchPdl, kv_attend_rows_kernel<128>, grid, dim3(128), 0, s, a, rows_or_tiles)
                            : launch_k(kLaunchPdl, kv_attend_rows_kernel<64>, grid, dim3(128), 0, s, a, rows_or_tiles);
    }
    if (a.g.i4) return a.g.D == 128 ? launch_few<128, true>(a, rows_or_tiles, s) : launch_few<64, true>(a, rows_or_tiles, s);
    return a.g.D == 128 ? launch_few<128, false>(a, rows_or_tiles, s) : launch_few<64, false>(a, rows_or_tiles, s);
}

}  // namespace dtts
