// The LLM decoder step of the autoregressive loop (Qwen2.5-1.5B as run by
// src/llm_manual.cpp): llm_kv_cache_init (:237) over a prompt and
// llm_kv_cache_step (:342), one new embedding per sequence, on sm_100a for a
// batch of sequences advancing together.
//
// Per layer: RMSNorm (eps 1e-6, gain) -> q|k|v projection with biases
// (tcgen05 GEMM, fp32 out) -> RoPE (half-split pairs, theta 1e6, angle
// pos * theta_d with theta_d advanced by repeated multiplication) on q and k,
// k and v appended to a bf16 cache -> grouped-query attention (12 query heads
// over 2 key/value heads of 128, causal) -> o_proj (+bias) into the fp32
// residual -> RMSNorm -> gate|up projection -> SiLU(gate) * up -> down_proj
// into the residual; then the final RMSNorm.  dtts_llm_extend runs the same
// layers over a paged cache (kv_host.h): sequences of different lengths, bf16 or
// 4-bit rows, an optional sliding window.
#include "kernels.cuh"
#include "kv_host.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <vector>

using namespace dtts;

namespace {

constexpr int kLH = 1536, kLF = 8960, kLNH = 12, kLNKV = 2, kLHD = 128, kLKV = kLNKV * kLHD;
constexpr int kLQKV = kLH + 2 * kLKV;   // 2048 columns: q | k | v

// ---------------------------------------------------------------- kernels
// RMSNorm of 1536-wide rows, one warp per row (manual_rms_norm,
// include/dit_manual.h:23-27): out = x / sqrt(mean(x^2) + 1e-6) * w.
template <bool OUT_BF16>
__global__ void __launch_bounds__(256) llm_rms_norm_kernel(const float *__restrict__ x, const float *__restrict__ w,
                                                           void *__restrict__ out, int M) {
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= M) return;
    const float4 *xr = reinterpret_cast<const float4 *>(x + (long long)row * kLH);
    float4 v[12];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 12; j++) {
        v[j] = xr[lane + 32 * j];
        ss += (v[j].x * v[j].x + v[j].y * v[j].y) + (v[j].z * v[j].z + v[j].w * v[j].w);
    }
    const float inv = 1.0f / sqrtf(warp_sum(ss) / (float)kLH + 1e-6f);
    const float4 *w4 = reinterpret_cast<const float4 *>(w);
#pragma unroll
    for (int j = 0; j < 12; j++) {
        const int c4 = lane + 32 * j;
        const float4 g = w ? __ldg(w4 + c4) : make_float4(1.f, 1.f, 1.f, 1.f);
        const float4 o = make_float4(v[j].x * inv * g.x, v[j].y * inv * g.y, v[j].z * inv * g.z, v[j].w * inv * g.w);
        if constexpr (OUT_BF16)
            reinterpret_cast<uint2 *>(out)[(long long)row * (kLH / 4) + c4] = make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
        else
            reinterpret_cast<float4 *>(out)[(long long)row * (kLH / 4) + c4] = o;
    }
}

// RoPE on q (12 heads) and k (2 heads) of token m = b * T + t at position
// pos0 + t, q to qout (fp32), k and v appended to the caches
// [b][kv head][cap][128] (bf16).  One block of 256 threads per token; work
// item i < 14 * 64 rotates pair (d, d + 64), d = i % 64, of q/k head i / 64,
// and the 256 v values follow.  pos_dev, if set, holds pos0 on the device
// (graph-captured steps); zero: each qkv value is cleared by the thread that
// read it (the next split-K reduce-add target).
__global__ void __launch_bounds__(256) llm_rope_cache_kernel(float *__restrict__ qkv, int T, int pos0,
                                                              const int *__restrict__ pos_dev,
                                                              const float2 *__restrict__ rope, float *__restrict__ qout,
                                                              bf16 *__restrict__ kc, bf16 *__restrict__ vc, int cap,
                                                              int zero) {
    pdl_wait();
    pdl_trigger();
    if (pos_dev) pos0 = *pos_dev;
    const int m = blockIdx.x, b = m / T, t = m % T, p = pos0 + t;
    float *row = qkv + (long long)m * kLQKV;
    constexpr int kRot = (kLNH + kLNKV) * 64;
    for (int i = threadIdx.x; i < kRot + kLKV; i += blockDim.x) {
        if (i < kRot) {
            const int hh = i >> 6, d = i & 63;
            const int c = hh * kLHD + d;   // q heads, then k heads (columns 1536..1791)
            const float2 cs = rope[(long long)p * 64 + d];
            const float x0 = row[c], x1 = row[c + 64];
            if (zero) row[c] = row[c + 64] = 0.f;
            const float y0 = x0 * cs.x - x1 * cs.y, y1 = x1 * cs.x + x0 * cs.y;
            if (hh < kLNH) {
                qout[(long long)m * kLH + c] = y0;
                qout[(long long)m * kLH + c + 64] = y1;
            } else {
                bf16 *dst = kc + (((long long)b * kLNKV + (hh - kLNH)) * cap + p) * kLHD;
                dst[d] = __float2bfloat16_rn(y0);
                dst[d + 64] = __float2bfloat16_rn(y1);
            }
        } else {
            const int j = i - kRot, hv = j >> 7, d = j & 127;
            const float x = row[kLH + kLKV + j];
            if (zero) row[kLH + kLKV + j] = 0.f;
            vc[(((long long)b * kLNKV + hv) * cap + p) * kLHD + d] = __float2bfloat16_rn(x);
        }
    }
}

// RoPE and cache rows for a batch over a paged cache: q to bf16 [M][1536], k and v
// (rounded to bf16, as the dense cache holds them) to the rows' pages.  One block
// of 160 threads per token: warp 0 rotates and stores the two k heads, warp 1
// stores v, warps 2-4 rotate q; a thread of a rotation has dims 8 u .. 8 u + 7 and
// 64 + 8 u .. of a head.  zero as above.
DTTS_DEV void llm_rope8(float *row, const float4 *cs4, int c, uint4 *lo, uint4 *hi, int zero) {
    float4 *a = reinterpret_cast<float4 *>(row + c), *b = reinterpret_cast<float4 *>(row + c + 64);
    const float4 x0 = a[0], x1 = a[1], y0 = b[0], y1 = b[1];
    if (zero) a[0] = a[1] = b[0] = b[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
    const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
    float p[8], q[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float4 cs = cs4[i];   // (cos, sin) of two dims
        p[2 * i] = x[2 * i] * cs.x - y[2 * i] * cs.y;
        q[2 * i] = y[2 * i] * cs.x + x[2 * i] * cs.y;
        p[2 * i + 1] = x[2 * i + 1] * cs.z - y[2 * i + 1] * cs.w;
        q[2 * i + 1] = y[2 * i + 1] * cs.z + x[2 * i + 1] * cs.w;
    }
    *lo = make_uint4(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7]));
    *hi = make_uint4(pack_bf16x2(q[0], q[1]), pack_bf16x2(q[2], q[3]), pack_bf16x2(q[4], q[5]), pack_bf16x2(q[6], q[7]));
}
__global__ void __launch_bounds__(160) llm_rope_pages_kernel(float *__restrict__ qkv, const __grid_constant__ KvGeom g,
                                                             const __grid_constant__ KvMeta m, uint8_t *__restrict__ pool,
                                                             int n_seq, const float2 *__restrict__ rope, int max_seq,
                                                             bf16 *__restrict__ qout, int zero) {
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = kv_find_entry(m.start, n_seq, row), off = row - m.start[b];
    const bool on = off < m.cnt[b];
    const int tok = m.len[b] - m.cnt[b] + off, pos = min(m.pos[b] + off, max_seq - 1);
    const int page = on ? m.table[(long long)m.seq[b] * g.max_pages + (tok >> g.lgP)] : -1;
    const bool held = page >= 0 && page < g.n_pages;
    float *x = qkv + (long long)row * kLQKV;
    const float4 *cs = reinterpret_cast<const float4 *>(rope + (long long)pos * 64 + 8 * (lane & 7));
    uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
    if (warp == 0) {
        const int head = (lane >> 3) & 1, u = lane & 7;
        if (lane < 16) llm_rope8(x, cs, kLH + head * kLHD + 8 * u, &lo, &hi, zero);
        uint8_t *seg = pool + kv_seg_off(g, held ? page : 0, 0, head);
        kv_store8(g, seg, false, tok & (g.P - 1), u, lo, held && lane < 16);
        kv_store8(g, seg, false, tok & (g.P - 1), 8 + u, hi, held && lane < 16);
    } else if (warp == 1) {
        const int head = lane >> 4, w = lane & 15;
        float4 *v = reinterpret_cast<float4 *>(x + kLH + kLKV + head * kLHD + 8 * w);
        const float4 a = v[0], c = v[1];
        if (zero) v[0] = v[1] = make_float4(0.f, 0.f, 0.f, 0.f);
        lo = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(c.x, c.y), pack_bf16x2(c.z, c.w));
        kv_store8(g, pool + kv_seg_off(g, held ? page : 0, 0, head), true, tok & (g.P - 1), w, lo, held);
    } else {
        const int head = (warp - 2) * 4 + (lane >> 3), c = head * kLHD + 8 * (lane & 7);
        llm_rope8(x, cs, c, &lo, &hi, zero);
        bf16 *q = qout + (long long)row * kLH + c;
        *reinterpret_cast<uint4 *>(q) = lo;
        *reinterpret_cast<uint4 *>(q + 64) = hi;
    }
}

// Grouped-query causal attention, one warp per (token m, query head): the
// lanes form two groups of 16 (g = lane / 16); lane c of group g owns dims
// 8c .. 8c+7 of key 2u + g, so each 16-byte load instruction reads two whole
// 256-byte K (or V) rows and a score needs a 4-step shuffle within the group.
// Keys 0 .. pos0 + t of the token's sequence, 16 per round; online softmax in
// fp32 (scores pre-scaled by log2(e) / sqrt(128), exp2); the two groups' P.V
// are merged at the end; the output row goes to ao (bf16, the o_proj input).
__global__ void __launch_bounds__(256, 2) llm_attn_kernel(const float *__restrict__ q, const bf16 *__restrict__ kc,
                                                       const bf16 *__restrict__ vc, int T, int pos0,
                                                       const int *__restrict__ pos_dev, int cap, int M,
                                                       bf16 *__restrict__ ao) {
    pdl_wait();
    pdl_trigger();
    if (pos_dev) pos0 = *pos_dev;
    const int wid = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (wid >= M * kLNH) return;
    const int m = wid / kLNH, h = wid % kLNH, b = m / T, t = m % T;
    const int kvh = h * kLNKV / kLNH;
    const int g = lane >> 4, c = lane & 15;
    const int n_keys = pos0 + t + 1;
    const float sc = 1.4426950408889634f / sqrtf((float)kLHD);
    float qv[8];
    {
        const float4 *q4 = reinterpret_cast<const float4 *>(q + (long long)m * kLH + h * kLHD + 8 * c);
        const float4 a = q4[0], bq = q4[1];
        qv[0] = a.x * sc; qv[1] = a.y * sc; qv[2] = a.z * sc; qv[3] = a.w * sc;
        qv[4] = bq.x * sc; qv[5] = bq.y * sc; qv[6] = bq.z * sc; qv[7] = bq.w * sc;
    }
    const bf16 *kb = kc + ((long long)b * kLNKV + kvh) * cap * kLHD + 8 * c;
    const bf16 *vb = vc + ((long long)b * kLNKV + kvh) * cap * kLHD + 8 * c;
    constexpr int U = 8;   // key pairs per round
    float mx = -INFINITY, l = 0.f, acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = 0.f;
    for (int j0 = 0; j0 < n_keys; j0 += 2 * U) {
        uint4 kr[U], vr[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = min(j0 + 2 * u + g, n_keys - 1);   // past the end: a valid row, masked below
            kr[u] = *reinterpret_cast<const uint4 *>(kb + (long long)j * kLHD);
            vr[u] = *reinterpret_cast<const uint4 *>(vb + (long long)j * kLHD);
        }
        float sv[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t w[4] = {kr[u].x, kr[u].y, kr[u].z, kr[u].w};
            float d = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // bf16 pair -> two floats by bit placement (exact)
                d = fmaf(qv[2 * i], __uint_as_float(w[i] << 16), d);
                d = fmaf(qv[2 * i + 1], __uint_as_float(w[i] & 0xFFFF0000u), d);
            }
            sv[u] = d;
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
#pragma unroll
            for (int u = 0; u < U; u++) sv[u] += __shfl_xor_sync(0xffffffffu, sv[u], o);
        float bm = mx;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (j0 + 2 * u + g >= n_keys) sv[u] = -INFINITY;
            bm = fmaxf(bm, sv[u]);
        }
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 16));
        const float corr = exp2f(mx - bm);
        l *= corr;
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] *= corr;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float p = exp2f(sv[u] - bm);
            l += p;
            const uint32_t w[4] = {vr[u].x, vr[u].y, vr[u].z, vr[u].w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                acc[2 * i] = fmaf(p, __uint_as_float(w[i] << 16), acc[2 * i]);
                acc[2 * i + 1] = fmaf(p, __uint_as_float(w[i] & 0xFFFF0000u), acc[2 * i + 1]);
            }
        }
        mx = bm;
    }
    // merge the two key groups (lanes c and c + 16)
    l += __shfl_xor_sync(0xffffffffu, l, 16);
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 16);
    if (g == 0) {
        const float inv = 1.0f / l;
        reinterpret_cast<uint4 *>(ao + (long long)m * kLH + h * kLHD)[c] =
            make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                       pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
    }
}

// out[m][j] = gate / (1 + e^-gate) * up with gu[m] = gate[8960] | up[8960]
// (src/llm_manual.cpp:333-334, :468), four columns per thread; zero: gu is
// cleared behind the read.
__global__ void llm_swiglu_kernel(float *__restrict__ gu, bf16 *__restrict__ out, long long n4, int zero) {
    pdl_wait();
    pdl_trigger();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n4) return;
    const long long m = i / (kLF / 4), j4 = i % (kLF / 4);
    float4 *g4 = reinterpret_cast<float4 *>(gu + m * 2 * kLF) + j4;
    float4 *u4 = reinterpret_cast<float4 *>(gu + m * 2 * kLF + kLF) + j4;
    const float4 g = *g4, u = *u4;
    if (zero) *g4 = *u4 = make_float4(0.f, 0.f, 0.f, 0.f);
    reinterpret_cast<uint2 *>(out)[i] =
        make_uint2(pack_bf16x2(g.x / (1.0f + expf(-g.x)) * u.x, g.y / (1.0f + expf(-g.y)) * u.y),
                   pack_bf16x2(g.z / (1.0f + expf(-g.z)) * u.z, g.w / (1.0f + expf(-g.w)) * u.w));
}

int up_f32(DeviceArena &a, const float *h, size_t n, float **out) {
    *out = nullptr;
    if (!h) return DTTS_OK;
    void *d = a.alloc(n * 4);
    DTTS_CHECK(d, DTTS_ERR_OOM, "cudaMalloc failed");
    DTTS_CUDA(cudaMemcpy(d, h, n * 4, cudaMemcpyHostToDevice));
    *out = (float *)d;
    return DTTS_OK;
}

// row-concatenation of parts (rows_i x cols fp32) uploaded as bf16
int up_bf16(DeviceArena &a, const std::vector<std::pair<const float *, size_t>> &parts, size_t cols, bf16 **out) {
    size_t rows = 0;
    for (auto &p : parts) rows += p.second;
    std::vector<uint16_t> tmp(rows * cols);
    size_t r0 = 0;
    for (auto &p : parts) {
        f32_to_bf16_host(p.first, tmp.data() + r0 * cols, p.second * cols);
        r0 += p.second;
    }
    void *d = a.alloc(tmp.size() * 2);
    DTTS_CHECK(d, DTTS_ERR_OOM, "cudaMalloc failed");
    DTTS_CUDA(cudaMemcpy(d, tmp.data(), tmp.size() * 2, cudaMemcpyHostToDevice));
    *out = (bf16 *)d;
    return DTTS_OK;
}

}  // namespace

struct dtts_llm {
    int device = 0, num_sms = 148, n_layers = 0, max_batch = 0, max_seq = 0;
    cudaStream_t own_stream = nullptr, stream = nullptr;
    DeviceArena wts, cache, ws;
    struct Layer {
        bf16 *wqkv = nullptr, *wo = nullptr, *wgu = nullptr, *wd = nullptr;
        float *bqkv = nullptr, *bo = nullptr, *an = nullptr, *fn = nullptr;
        CUtensorMap tqkv, to, tgu, td;             // 256-row boxes
        CUtensorMap tqkv_s, to_s, tgu_s, td_s;     // 128-row boxes (small batches)
    };
    std::vector<Layer> layers;
    float *final_norm = nullptr;
    bf16 *kc = nullptr, *vc = nullptr;   // [n_layers][max_batch][2][max_seq][128]
    float2 *rope = nullptr;              // [max_seq][64]
    int *d_len = nullptr;                // cache length on the device (graph-captured steps)
    int *d_err = nullptr;
    // step graphs, one per batch size; dropped when the workspace moves
    // (paged: also the cache, the window and the split of its attention; uid 0: the dense cache); the least recently
    // used first.  Of the paged ones, kPagedGraphs are kept.
    static constexpr int kPagedGraphs = 64;
    struct Graph {
        int B;
        long long uid;
        int window, sinks, splits;
        cudaGraphExec_t exec;
    };
    std::vector<Graph> graphs;
    void drop_graphs() {
        for (Graph &g : graphs) cudaGraphExecDestroy(g.exec);
        graphs.clear();
    }
    int cur_B = 0, cur_len = 0;
    long long cap_tok = 0;
    float *h = nullptr, *qkv = nullptr, *q = nullptr, *gu = nullptr;
    bf16 *act = nullptr, *ao = nullptr, *ffn = nullptr;
    CUtensorMap t_act, t_ao, t_ffn, t_h, t_qkv_r, t_gu_r;   // *_r: fp32 reduce-add targets

    ~dtts_llm() {
        drop_graphs();
        ws.free_all();
        cache.free_all();
        wts.free_all();
        if (own_stream) cudaStreamDestroy(own_stream);
    }

    int ensure(long long tok) {
        if (tok <= cap_tok) return DTTS_OK;
        DTTS_CUDA(cudaStreamSynchronize(stream));
        drop_graphs();
        ws.free_all();
        cap_tok = 0;   // until all of it is there
        const size_t T = (size_t)std::max<long long>(tok, 64);
        h = (float *)ws.alloc(T * kLH * 4);
        qkv = (float *)ws.alloc(T * kLQKV * 4);
        q = (float *)ws.alloc(T * kLH * 4);
        gu = (float *)ws.alloc(T * 2 * kLF * 4);
        act = (bf16 *)ws.alloc(T * kLH * 2);
        ao = (bf16 *)ws.alloc(T * kLH * 2);
        ffn = (bf16 *)ws.alloc(T * kLF * 2);
        if (!(h && qkv && q && gu && act && ao && ffn)) {
            ws.free_all();
            set_error("LLM workspace allocation failed (%lld tokens)", tok);
            return DTTS_ERR_OOM;
        }
        bool ok = make_tmap_bf16(&t_act, act, T, kLH, 128) && make_tmap_bf16(&t_ao, ao, T, kLH, 128) &&
                  make_tmap_bf16(&t_ffn, ffn, T, kLF, 128) && make_tmap_f32_resid(&t_h, h, T, kLH) &&
                  make_tmap_f32_resid(&t_qkv_r, qkv, T, kLQKV) && make_tmap_f32_resid(&t_gu_r, gu, T, 2 * kLF);
        DTTS_CHECK(ok, DTTS_ERR_CUDA, "tensor map (LLM workspace)");
        cap_tok = (long long)T;
        return DTTS_OK;
    }

    GemmOp op(const CUtensorMap &ta, const CUtensorMap &tb, int M, int N, int K, int epi, int bn) {
        GemmOp o;
        std::memset(&o, 0, sizeof(o));
        o.ta = ta; o.tb = tb; o.M = M; o.N = N; o.K = K; o.bn = bn; o.nw = 4; o.epi = epi;
        o.ep.err = d_err; o.ep.tok_per_row = 1; o.ep.ksplit = 1;
        o.pdl = 1;   // every GEMM follows another kernel
        return o;
    }

    // emb already in h ([B * T][1536]); runs every layer and the final norm into
    // `out`, then advances d_len; dev_pos: positions from d_len, not pos0
    // kv, plan: instead of the dense cache, the M rows of the paged cache's batch
    int enqueue(int B, int T, int pos0, bool dev_pos, float *out, dtts_kv *kv = nullptr,
                const KvAttendPlan *plan = nullptr) {
        const int *pd = dev_pos ? d_len : nullptr;
        const int M = kv ? kv->b_rows : B * T;
        const bool small = M <= 256;
        const int bn = small ? 128 : 256;
        const size_t layer_stride = (size_t)max_batch * kLNKV * max_seq * kLHD;
        // few rows: the QKV and gate|up GEMMs split K so that about 128 CTAs
        // stream the weights, partial sums reduce-added into fp32 rows that are
        // zeroed here once and then by their readers behind each read
        if (small) {
            DTTS_CUDA(cudaMemsetAsync(qkv, 0, (size_t)M * kLQKV * 4, stream));
            DTTS_CUDA(cudaMemsetAsync(gu, 0, (size_t)M * 2 * kLF * 4, stream));
        }
        // every kernel but the first starts programmatically behind the one before it
        const bool pdl = pdl_enabled();
        for (int l = 0; l < n_layers; l++) {
            const Layer &L = layers[l];
            launch_k(pdl && l > 0, llm_rms_norm_kernel<true>, dim3((M + 7) / 8), dim3(256), 0, stream,
                     (const float *)h, (const float *)L.an, (void *)act, M);
            if (small) {
                GemmOp o = op(t_act, L.tqkv_s, M, kLQKV, kLH, EPI_RESID, bn);
                o.tr = t_qkv_r; o.ep.bias = L.bqkv; o.ep.resid = qkv; o.ep.ldr = kLQKV; o.ep.ksplit = 8;
                DTTS_CUDA(launch_gemm(o, num_sms, stream));
            } else {
                GemmOp o = op(t_act, L.tqkv, M, kLQKV, kLH, EPI_F32, bn);
                o.ep.bias = L.bqkv; o.ep.out = qkv; o.ep.ldo = kLQKV;
                DTTS_CUDA(launch_gemm(o, num_sms, stream));
            }
            if (kv) {
                launch_k(pdl, llm_rope_pages_kernel, dim3(M), dim3(160), 0, stream, qkv, kv->g, kv->kv_meta(),
                         kv->pool + (long long)l * kv->g.H * kv->g.seg, (int)kv->b_seq.size(), (const float2 *)rope, max_seq,
                         (bf16 *)q, small ? 1 : 0);
                int st = kv->attend(*plan, l);
                if (st) return st;
            } else {
                launch_k(pdl, llm_rope_cache_kernel, dim3(M), dim3(256), 0, stream, qkv, T, pos0, pd, (const float2 *)rope,
                         q, kc + l * layer_stride, vc + l * layer_stride, max_seq, small ? 1 : 0);
                launch_k(pdl, llm_attn_kernel, dim3((M * kLNH + 7) / 8), dim3(256), 0, stream, (const float *)q,
                         (const bf16 *)(kc + l * layer_stride), (const bf16 *)(vc + l * layer_stride), T, pos0, pd,
                         max_seq, M, ao);
            }
            {
                GemmOp o = op(t_ao, small ? L.to_s : L.to, M, kLH, kLH, EPI_RESID, bn);
                o.tr = t_h; o.ep.bias = L.bo; o.ep.resid = h; o.ep.ldr = kLH;
                o.ep.ksplit = small ? 8 : 1;
                DTTS_CUDA(launch_gemm(o, num_sms, stream));
            }
            launch_k(pdl, llm_rms_norm_kernel<true>, dim3((M + 7) / 8), dim3(256), 0, stream, (const float *)h,
                     (const float *)L.fn, (void *)act, M);
            if (small) {
                GemmOp o = op(t_act, L.tgu_s, M, 2 * kLF, kLH, EPI_RESID, bn);
                o.tr = t_gu_r; o.ep.resid = gu; o.ep.ldr = 2 * kLF; o.ep.ksplit = 2;
                DTTS_CUDA(launch_gemm(o, num_sms, stream));
            } else {
                GemmOp o = op(t_act, L.tgu, M, 2 * kLF, kLH, EPI_F32, bn);
                o.ep.out = gu; o.ep.ldo = 2 * kLF;
                DTTS_CUDA(launch_gemm(o, num_sms, stream));
            }
            const long long nf4 = (long long)M * kLF / 4;
            launch_k(pdl, llm_swiglu_kernel, dim3((unsigned)((nf4 + 255) / 256)), dim3(256), 0, stream, gu, ffn, nf4,
                     small ? 1 : 0);
            {
                GemmOp o = op(t_ffn, small ? L.td_s : L.td, M, kLH, kLF, EPI_RESID, bn);
                o.tr = t_h; o.ep.resid = h; o.ep.ldr = kLH;
                o.ep.ksplit = small ? 10 : 1;
                // prefill: the 17.5 KB-per-token activations are read once from DRAM,
                // not once per N pass (M-block-major tiles)
                o.ep.mb_major = small ? 0 : 1;
                DTTS_CUDA(launch_gemm(o, num_sms, stream));
            }
        }
        launch_k(pdl, llm_rms_norm_kernel<false>, dim3((M + 7) / 8), dim3(256), 0, stream, (const float *)h,
                 (const float *)final_norm, (void *)out, M);
        if (!kv) launch_advance_len(d_len, T, stream, true);
        DTTS_CUDA(cudaGetLastError());
        return DTTS_OK;
    }

    int run(const float *emb, int B, int T, float *hidden, int mem) {
        DTTS_CHECK(emb && hidden, DTTS_ERR_ARG, "null argument");
        DTTS_CHECK(mem == DTTS_MEM_HOST || mem == DTTS_MEM_DEVICE, DTTS_ERR_ARG, "bad mem kind");
        DTTS_CHECK(cur_len + T <= max_seq, DTTS_ERR_ARG, "KV cache full (%d + %d > %d tokens)", cur_len, T, max_seq);
        DeviceGuard g(device);
        const long long M = (long long)B * T;
        int st = ensure(M + 1);
        if (st) return st;
        // the final norm writes into qkv's space (fp32, at least M x 1536), then out
        float *outd = qkv;
        DTTS_CUDA(cudaMemcpyAsync(h, emb, (size_t)M * kLH * 4,
                                  mem == DTTS_MEM_HOST ? cudaMemcpyHostToDevice : cudaMemcpyDeviceToDevice, stream));
        if (T == 1) {
            // decode step: one graph per batch size, positions from d_len
            cudaGraphExec_t exec = nullptr;
            for (Graph &g : graphs)
                if (g.B == B && g.uid == 0) exec = g.exec;
            if (!exec) {
                if ((st = capture(&exec, [&] { return enqueue(B, 1, 0, true, outd); }))) return st;
                graphs.push_back({B, 0, 0, 0, 0, exec});
            }
            DTTS_CUDA(cudaGraphLaunch(exec, stream));
        } else if ((st = enqueue(B, T, cur_len, false, outd))) {
            return st;
        }
        DTTS_CUDA(cudaMemcpyAsync(hidden, outd, (size_t)M * kLH * 4,
                                  mem == DTTS_MEM_HOST ? cudaMemcpyDeviceToHost : cudaMemcpyDeviceToDevice, stream));
        cur_len += T;
        return mem == DTTS_MEM_HOST ? finish() : DTTS_OK;
    }

    template <typename F>
    int capture(cudaGraphExec_t *exec, F body) {
        cudaGraph_t graph = nullptr;
        DTTS_CUDA(cudaStreamBeginCapture(stream, cudaStreamCaptureModeThreadLocal));
        int st = body();
        cudaError_t ce = cudaStreamEndCapture(stream, &graph);
        if (st) { if (graph) cudaGraphDestroy(graph); return st; }
        DTTS_CUDA(ce);
        ce = cudaGraphInstantiate(exec, graph, 0);
        cudaGraphDestroy(graph);
        DTTS_CUDA(ce);
        return DTTS_OK;
    }

    int finish() {
        int st = stream_wait(stream, 300.0);
        if (st) return st;
        int err = 0;
        DTTS_CUDA(cudaMemcpy(&err, d_err, 4, cudaMemcpyDeviceToHost));
        if (err) { cudaMemset(d_err, 0, 4); set_error("device wait limit reached (code %d)", err); return DTTS_ERR_TIMEOUT; }
        return DTTS_OK;
    }

    // The new tokens of a ragged batch over a paged cache.  A step (one token for
    // every sequence) is a graph: its kernels read lengths and tables on the device,
    // so one graph serves every step with the same batch size and split of the
    // attention (rounded down to 2^n or 3 * 2^n; a part holds at least 4 tiles).
    int extend(dtts_kv *kv, int n_seq, const int *seqs, const int *n_new, const float *emb, int window, int sinks,
               float *hidden, int mem) {
        long long M = 0;
        bool step = true;
        for (int b = 0; b < n_seq; b++) {
            DTTS_CHECK(kv->seqs[seqs[b]].pos + (long long)n_new[b] <= max_seq, DTTS_ERR_ARG,
                       "sequence %d would reach position %lld (limit %d)", seqs[b],
                       kv->seqs[seqs[b]].pos + (long long)n_new[b], max_seq);
            M += n_new[b];
            step = step && n_new[b] == 1;
        }
        DTTS_CHECK(M <= (1 << 24), DTTS_ERR_ARG, "%lld tokens in one call", M);
        DeviceGuard g(device);
        int st = kv->not_capturing("extend");   // the cache's stream; the engine's below
        if (st) return st;
        // the cache works on the engine's stream during the call; its own stream waits for what is enqueued here
        struct Streams {
            dtts_kv *kv;
            cudaStream_t back;
            ~Streams() { dtts_kv_set_stream(kv, back); }
        } streams{kv, kv->stream};
        if ((st = dtts_kv_set_stream(kv, stream)) || (st = kv->not_capturing("extend"))) return st;
        // what can be refused first: neither the workspace nor the cache changes for a request that does not fit
        long long pages = 0;
        if ((st = kv->check_window(n_seq, seqs, n_new, window, sinks))) return st;
        if ((st = kv->fits(n_seq, seqs, n_new, &pages))) return st;
        if ((st = ensure(M + 1))) return st;
        if ((st = kv->extend(n_seq, seqs, n_new))) return st;
        if (M == 0) return DTTS_OK;
        try {
            st = forward(kv, n_seq, emb, window, sinks, hidden, mem, step);
        } catch (const std::bad_alloc &) {
            kv->take_back();
            throw;
        }
        if (st) kv->take_back();
        return st;
    }

    // The decoder on the batch that kv->extend has just made.
    int forward(dtts_kv *kv, int n_seq, const float *emb, int window, int sinks, float *hidden, int mem, bool step) {
        int st;
        const long long M = kv->b_rows;
        dtts_kv_attend_args aa;
        std::memset(&aa, 0, sizeof(aa));
        aa.q = q; aa.q_row = kLH; aa.q_head = kLHD;
        aa.out = ao; aa.out_row = kLH; aa.out_head = kLHD;
        aa.n_heads = kLNH;
        aa.scale = 1.0f / sqrtf((float)kLHD);
        aa.window = window; aa.sinks = sinks;
        KvAttendPlan plan;
        if ((st = kv->plan_attend(aa, &plan))) return st;
        float *outd = qkv;
        DTTS_CUDA(cudaMemcpyAsync(h, emb, (size_t)M * kLH * 4,
                                  mem == DTTS_MEM_HOST ? cudaMemcpyHostToDevice : cudaMemcpyDeviceToDevice, stream));
        if (step) {
            KvAttendArgs &p = plan.args[0];
            int round = 1;   // 1, 2, 3, 4, 6, 8, 12, ...
            while (2 * round <= p.splits) round *= 2;
            if (round / 2 * 3 <= p.splits && round > 1) round = round / 2 * 3;
            const int splits = std::min(round, kv->max_splits(n_seq));
            cudaGraphExec_t exec = nullptr;
            const auto used = std::find_if(graphs.begin(), graphs.end(), [&](const Graph &g) {
                return g.B == n_seq && g.uid == kv->uid && g.window == window && g.sinks == sinks && g.splits == splits;
            });
            if (used != graphs.end()) {
                exec = used->exec;
                std::rotate(used, used + 1, graphs.end());
            } else {
                p.splits = (short)splits;
                p.tiles_per_split = 4;
                auto paged = [](const Graph &g) { return g.uid != 0; };
                if (std::count_if(graphs.begin(), graphs.end(), paged) >= kPagedGraphs) {
                    DTTS_CUDA(cudaStreamSynchronize(stream));   // it may be running
                    const auto oldest = std::find_if(graphs.begin(), graphs.end(), paged);
                    cudaGraphExecDestroy(oldest->exec);
                    graphs.erase(oldest);
                }
                graphs.reserve(graphs.size() + 1);
                if ((st = capture(&exec, [&] { return enqueue(n_seq, 1, 0, false, outd, kv, &plan); }))) return st;
                graphs.push_back({n_seq, kv->uid, window, sinks, splits, exec});
            }
            DTTS_CUDA(cudaGraphLaunch(exec, stream));
        } else if ((st = enqueue(n_seq, 0, 0, false, outd, kv, &plan))) {
            return st;
        }
        DTTS_CUDA(cudaMemcpyAsync(hidden, outd, (size_t)M * kLH * 4,
                                  mem == DTTS_MEM_HOST ? cudaMemcpyDeviceToHost : cudaMemcpyDeviceToDevice, stream));
        if (mem != DTTS_MEM_HOST) return DTTS_OK;
        if ((st = finish())) return st;
        return dtts_kv_sync(kv);
    }
};

extern "C" {

int dtts_llm_create(const dtts_llm_weights *w, int device, int max_batch, int max_seq, dtts_llm **out) {
    DTTS_CHECK(w && out, DTTS_ERR_ARG, "null argument");
    *out = nullptr;
    DTTS_CHECK(w->n_layers >= 1 && w->n_layers <= 64 && w->layers && w->final_norm, DTTS_ERR_ARG,
               "n_layers %d invalid or final norm missing", w->n_layers);
    DTTS_CHECK(max_batch >= 1 && max_seq >= 1 && max_seq <= 32768, DTTS_ERR_ARG, "bad capacity %d x %d", max_batch,
               max_seq);
    for (int l = 0; l < w->n_layers; l++) {
        const dtts_llm_layer_weights &L = w->layers[l];
        DTTS_CHECK(L.qw && L.kw && L.vw && L.ow && L.gw && L.uw && L.dw, DTTS_ERR_ARG, "missing weight in layer %d", l);
    }
    int nsm = 0, st = check_device(device, &nsm);
    if (st) return st;
    DeviceGuard g(device);
    std::unique_ptr<dtts_llm> e(new dtts_llm());
    e->device = device; e->num_sms = nsm; e->n_layers = w->n_layers; e->max_batch = max_batch; e->max_seq = max_seq;
    DTTS_CUDA(cudaStreamCreateWithFlags(&e->own_stream, cudaStreamNonBlocking));
    e->stream = e->own_stream;
    DTTS_CUDA(gemm_prepare_attributes());
    e->d_err = (int *)e->wts.alloc(4);
    DTTS_CHECK(e->d_err, DTTS_ERR_OOM, "cudaMalloc failed");
    DTTS_CUDA(cudaMemset(e->d_err, 0, 4));
    e->layers.resize(w->n_layers);
    std::vector<float> bqkv(kLQKV);
    for (int l = 0; l < w->n_layers; l++) {
        const dtts_llm_layer_weights &s = w->layers[l];
        dtts_llm::Layer &L = e->layers[l];
        if ((st = up_bf16(e->wts, {{s.qw, kLH}, {s.kw, kLKV}, {s.vw, kLKV}}, kLH, &L.wqkv))) return st;
        if ((st = up_bf16(e->wts, {{s.ow, kLH}}, kLH, &L.wo))) return st;
        if ((st = up_bf16(e->wts, {{s.gw, kLF}, {s.uw, kLF}}, kLH, &L.wgu))) return st;
        if ((st = up_bf16(e->wts, {{s.dw, kLH}}, kLF, &L.wd))) return st;
        std::fill(bqkv.begin(), bqkv.end(), 0.f);
        if (s.qb) std::memcpy(bqkv.data(), s.qb, kLH * 4);
        if (s.kb) std::memcpy(bqkv.data() + kLH, s.kb, kLKV * 4);
        if (s.vb) std::memcpy(bqkv.data() + kLH + kLKV, s.vb, kLKV * 4);
        if ((st = up_f32(e->wts, bqkv.data(), kLQKV, &L.bqkv))) return st;
        if ((st = up_f32(e->wts, s.ob, kLH, &L.bo))) return st;
        if ((st = up_f32(e->wts, s.an, kLH, &L.an))) return st;
        if ((st = up_f32(e->wts, s.fn, kLH, &L.fn))) return st;
        bool ok = make_tmap_bf16(&L.tqkv, L.wqkv, kLQKV, kLH, 256) && make_tmap_bf16(&L.to, L.wo, kLH, kLH, 256) &&
                  make_tmap_bf16(&L.tgu, L.wgu, 2 * kLF, kLH, 256) && make_tmap_bf16(&L.td, L.wd, kLH, kLF, 256) &&
                  make_tmap_bf16(&L.tqkv_s, L.wqkv, kLQKV, kLH, 128) && make_tmap_bf16(&L.to_s, L.wo, kLH, kLH, 128) &&
                  make_tmap_bf16(&L.tgu_s, L.wgu, 2 * kLF, kLH, 128) && make_tmap_bf16(&L.td_s, L.wd, kLH, kLF, 128);
        DTTS_CHECK(ok, DTTS_ERR_CUDA, "tensor map (LLM layer %d)", l);
    }
    if ((st = up_f32(e->wts, w->final_norm, kLH, &e->final_norm))) return st;
    const size_t cache_elems = (size_t)w->n_layers * max_batch * kLNKV * max_seq * kLHD;
    e->kc = (bf16 *)e->cache.alloc(cache_elems * 2);
    e->vc = (bf16 *)e->cache.alloc(cache_elems * 2);
    e->rope = (float2 *)e->cache.alloc((size_t)max_seq * 64 * sizeof(float2));
    e->d_len = (int *)e->cache.alloc(sizeof(int));
    DTTS_CHECK(e->kc && e->vc && e->rope && e->d_len, DTTS_ERR_OOM, "LLM KV cache allocation failed (%zu MB)", cache_elems * 4 >> 20);
    // (cos, sin)(pos * theta_d), theta_d = (1e6^(-2/128))^d by repeated
    // multiplication, as src/llm_manual.cpp:398-403 and :449-451 compute them
    std::vector<float2> rt((size_t)max_seq * 64);
    const float ts = powf(1000000.0f, -2.0f / (float)kLHD);
    for (int p = 0; p < max_seq; p++) {
        float theta = 1.0f;
        for (int d = 0; d < 64; d++) {
            rt[(size_t)p * 64 + d] = make_float2(cosf((float)p * theta), sinf((float)p * theta));
            theta *= ts;
        }
    }
    DTTS_CUDA(cudaMemcpy(e->rope, rt.data(), rt.size() * sizeof(float2), cudaMemcpyHostToDevice));
    *out = e.release();
    return DTTS_OK;
}

int dtts_llm_destroy(dtts_llm *e) {
    if (!e) return DTTS_OK;
    DeviceGuard g(e->device);
    cudaStreamSynchronize(e->stream);
    delete e;
    return DTTS_OK;
}

int dtts_llm_set_stream(dtts_llm *e, void *stream) {
    DTTS_CHECK(e, DTTS_ERR_ARG, "null engine");
    e->stream = stream ? static_cast<cudaStream_t>(stream) : e->own_stream;
    return DTTS_OK;
}

int dtts_llm_prefill(dtts_llm *e, const float *emb, int B, int n_tok, float *hidden, int mem) {
    DTTS_CHECK(e, DTTS_ERR_ARG, "null engine");
    DTTS_CHECK(B >= 1 && B <= e->max_batch && n_tok >= 1, DTTS_ERR_ARG, "bad prefill shape %d x %d", B, n_tok);
    DeviceGuard g(e->device);
    e->cur_B = B;
    e->cur_len = 0;
    DTTS_CUDA(cudaMemsetAsync(e->d_len, 0, sizeof(int), e->stream));
    return e->run(emb, B, n_tok, hidden, mem);
}

int dtts_llm_step(dtts_llm *e, const float *emb, int B, float *hidden, int mem) {
    DTTS_CHECK(e, DTTS_ERR_ARG, "null engine");
    DTTS_CHECK(B == e->cur_B && e->cur_len > 0, DTTS_ERR_ARG, "step needs a prefill of the same %d sequences", B);
    return e->run(emb, B, 1, hidden, mem);
}

int dtts_llm_kv_create(dtts_llm *e, int n_pages, int max_seqs, int page_tokens, int dtype, dtts_kv **out) {
    DTTS_CHECK(e && out, DTTS_ERR_ARG, "null argument");
    *out = nullptr;
    dtts_kv_config c;
    c.n_layers = e->n_layers;
    c.n_kv_heads = kLNKV;
    c.head_dim = kLHD;
    c.page_tokens = page_tokens;
    c.n_pages = n_pages;
    c.max_seqs = max_seqs;
    c.max_tokens = e->max_seq;
    c.dtype = dtype;
    return dtts_kv_create(&c, e->device, out);
}

int dtts_llm_extend(dtts_llm *e, dtts_kv *kv, int n_seq, const int *seqs, const int *n_new, const float *emb, int window,
                    int sinks, float *hidden, int mem) try {
    DTTS_CHECK(e && kv && seqs && n_new && emb && hidden, DTTS_ERR_ARG, "null argument");
    DTTS_CHECK(mem == DTTS_MEM_HOST || mem == DTTS_MEM_DEVICE, DTTS_ERR_ARG, "bad mem kind");
    DTTS_CHECK(kv->device == e->device && kv->g.L == e->n_layers && kv->g.H == kLNKV && kv->g.D == kLHD, DTTS_ERR_ARG,
               "the cache has %d layers of %d x %d on device %d, the engine needs %d of %d x %d on device %d", kv->g.L,
               kv->g.H, kv->g.D, kv->device, e->n_layers, kLNKV, kLHD, e->device);
    int st = kv->check_batch(n_seq, seqs, n_new);
    if (st) return st;
    return e->extend(kv, n_seq, seqs, n_new, emb, window, sinks, hidden, mem);
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return DTTS_ERR_OOM;
}

int dtts_llm_length(dtts_llm *e, int *tokens) {
    DTTS_CHECK(e && tokens, DTTS_ERR_ARG, "null argument");
    *tokens = e->cur_len;
    return DTTS_OK;
}

}  // extern "C"
