// The paged K/V cache (dtts_kv_*): page tables and reference counts on the host,
// rows in a pool of pages on the device.  A sequence is a list of pages; forks
// share pages and copy the last, partly filled one when they grow.  The kernels
// here store and read rows, copy the rows of a shared page, gather kept rows and
// apply metadata updates that travel in kernel parameters (no host buffer has to
// outlive a call).
#include "kv_host.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <type_traits>

using namespace dtts;

namespace dtts {
bool pdl_enabled();
}  // namespace dtts

namespace {

unsigned kv_pdl() { return pdl_enabled() ? kLaunchPdl : 0u; }

constexpr int kWsFloats = 9 * 1024 * 1024;     // 36 MB of partial results
static_assert(kWsFloats / (kKvFewRows * (64 + 2)) <= INT16_MAX, "KvAttendArgs::splits");
constexpr int kMaxUnits = 1 << 16;             // split units with an arrival counter

// ---------------------------------------------------------------- metadata
// Lists travel in kernel parameters.  A launch with 4 KB of parameters costs the host 4 us more than one with
// half a KB, so every list has a short form beside the long one.
template <int N>
struct Pokes {
    static constexpr int kMax = N;
    int n;
    int index[N], value[N];
};
template <int N>
__global__ void kv_poke_kernel(int *__restrict__ meta, const __grid_constant__ Pokes<N> p) {
    pdl_wait();
    pdl_trigger();
    for (int i = threadIdx.x; i < p.n; i += blockDim.x) meta[p.index[i]] = p.value[i];
}

// Kept rows as bits (bit i of word x: row 32 (first + x) + i), to their ascending list from dst[base] on; the
// updates p beside them.  A row costs a bit of parameters, so thousands of rows are one launch.
template <int N>
struct KeepBits {
    static constexpr int kMax = N;
    int n, first, base;
    uint32_t word[N];
};
template <int N>
__global__ void __launch_bounds__(1024) kv_keep_kernel(int *__restrict__ dst, const __grid_constant__ KeepBits<N> k,
                                                       int *__restrict__ meta, const __grid_constant__ Pokes<60> p) {
    static_assert(N <= 1024, "a thread a word");
    __shared__ int total[32];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x, lane = t & 31;
    for (int i = t; i < p.n; i += blockDim.x) meta[p.index[i]] = p.value[i];
    uint32_t w = t < k.n ? k.word[t] : 0u;
    int at = __popc(w);   // inclusive sum over the warp, then over the warps before
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, at, x);
        if (lane >= x) at += y;
    }
    if (lane == 31) total[t >> 5] = at;
    __syncthreads();
    at += k.base - __popc(w);
    for (int x = 0; x < t >> 5; x++) at += total[x];
    for (; w; w &= w - 1) dst[at++] = 32 * (k.first + t) + __ffs(w) - 1;
}

template <int N>
struct Forks {
    static constexpr int kMax = N;
    int n, src, pages;
    int dst[N];
};
// one block per new table row
template <int N>
__global__ void kv_fork_tables_kernel(int *__restrict__ table, int max_pages, const __grid_constant__ Forks<N> f) {
    pdl_wait();
    pdl_trigger();
    for (int i = threadIdx.x; i < f.pages; i += blockDim.x)
        table[(long long)f.dst[blockIdx.x] * max_pages + i] = table[(long long)f.src * max_pages + i];
}

// ---------------------------------------------------------------- rows
// the geometry with what the instance fixes as constants
template <bool I4, int D>
DTTS_DEV KvGeom fixed_geom(const KvGeom &g) {
    KvGeom c = g;
    c.i4 = I4;
    c.D = D;
    c.RB = I4 ? D / 2 : 2 * D;
    c.SB = I4 ? D / 16 : 0;
    return c;
}

// A lane handles 8 dims of K or of V; D / 4 lanes take one (row, head): K by the
// first half of them, V by the second.  The rows' places come from the batch; a
// warp takes kWriteItems times 128 / D of them, whose loads are all in flight
// before the first is encoded.  4 D bytes read and 2 (RB + SB) written a row and
// head.  26002 4-bit rows of 2 heads of 128: 11.1 us, 3.1 TB/s, bound by issuing the
// encoding; in bf16 11.2 us, 4.7 TB/s.
constexpr int kWriteItems = 4;
template <bool I4, int D>
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KvGeom geom, const __grid_constant__ KvMeta m,
                                                       uint8_t *__restrict__ pool, int n_seq, int rows,
                                                       const bf16 *__restrict__ k, const bf16 *__restrict__ v,
                                                       long long k_row, long long k_head, long long v_row,
                                                       long long v_head, int *__restrict__ err) {
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0 && kv_batch_over(geom, m, n_seq, rows)) atomicCAS(err, 0, DEVERR_BATCH);
    const KvGeom g = fixed_geom<I4, D>(geom);
    constexpr int lpr = D / 4, step = 32 / lpr;   // lanes a (row, head): 32 or 16; items a warp and turn
    const int lane = threadIdx.x & 31, l = lane % lpr, w = l % (lpr / 2);
    const bool is_v = l >= lpr / 2;
    const long long first = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * (kWriteItems * step) + lane / lpr;
    int row = (int)min(first / g.H, (long long)INT32_MAX), head = (int)(first % g.H);
    int b = 0, start = 0, end = -1, tok0 = 0;   // entry of the batch: its rows [start, end)
    const int *trow = m.table;
    const bf16 *src = (is_v ? v : k) + 8 * w;
    const long long src_row = is_v ? v_row : k_row, src_head = is_v ? v_head : k_head;
    uint4 q[kWriteItems];
    int page[kWriteItems], place[kWriteItems], hd[kWriteItems];   // place: row within the page
#pragma unroll
    for (int x = 0; x < kWriteItems; x++) {
        q[x] = make_uint4(0u, 0u, 0u, 0u);
        page[x] = -1;                           // nothing to store
        place[x] = 0;
        hd[x] = head;
        if (row < rows) {
            if (row >= end) {
                b = kv_find_entry(m.start, n_seq, row);
                start = m.start[b];
                end = start + m.cnt[b];
                tok0 = m.len[b] - m.cnt[b] - start;
                trow = m.table + (long long)m.seq[b] * g.max_pages;
            }
            const int tok = tok0 + row;
            place[x] = tok & (g.P - 1);
            if (row < end) page[x] = trow[tok >> g.lgP];
            q[x] = *reinterpret_cast<const uint4 *>(src + row * src_row + head * src_head);
        }
        for (head += step; head >= g.H; head -= g.H) row++;
    }
#pragma unroll
    for (int x = 0; x < kWriteItems; x++) {
        const bool on = (unsigned)page[x] < (unsigned)g.n_pages;
        kv_store8(g, pool + kv_seg_off(g, on ? page[x] : 0, 0, hd[x]), is_v, place[x], w, q[x], on);
    }
}

// 8 floats to 32-byte (wide) or 16-byte aligned memory: whole 32-byte sectors in one instruction where possible
DTTS_DEV void store8_f32(float *p, const float (&x)[8], bool wide) {
    if (wide) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
                     "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                     : "memory");
    } else {
        reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
}
template <int N>
struct Reads {
    static constexpr int kMax = N;
    int n, rows, n_layers;            // entries, rows a layer (of all entries of the call)
    int seq[N], first[N], start[N + 1];   // start: first output row, start[n]: end
};
// Rows [first, first + count) of the listed sequences, for n_layers layers, as
// [layer][row][head][D] fp32 or bf16.  Same lane split as the write.  Bound by
// memory: 28 layers of 2926 bf16 rows (2 heads of 128) 28.4 us, 5.9 TB/s; 26002 4-bit
// rows to fp32 10.4 us, 5.8 TB/s.
constexpr int kReadItems = 4;
template <bool I4, int D, bool F32, int N>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvGeom geom, const int *__restrict__ table,
                                                      const uint8_t *__restrict__ pool, const __grid_constant__ Reads<N> r,
                                                      void *__restrict__ k, void *__restrict__ v, int *__restrict__ err) {
    pdl_wait();
    pdl_trigger();
    const KvGeom g = fixed_geom<I4, D>(geom);
    constexpr int lpr = D / 4, step = 32 / lpr;
    const int lane = threadIdx.x & 31, l = lane % lpr, w = l % (lpr / 2), layer = blockIdx.y;
    const bool is_v = l >= lpr / 2;
    const long long item = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * (kReadItems * step) + lane / lpr;
    const int row_end = r.start[r.n];
    int row = (int)min(r.start[0] + item / g.H, (long long)row_end), head = (int)(item % g.H);
    int e = 0, end = -1, shift = 0;
    const int *trow = table;
    // rows, then their pages, then what is held, each for all items before the next depends on it
    int tok[kReadItems], page[kReadItems], hd[kReadItems];
    long long at[kReadItems];   // output element; -1: none
#pragma unroll
    for (int i = 0; i < kReadItems; i++) {
        at[i] = -1;
        tok[i] = 0;
        hd[i] = head;
        if (row < row_end) {
            if (row >= end) {
                e = kv_find_entry(r.start, r.n, row);
                end = r.start[e + 1];
                shift = r.first[e] - r.start[e];
                trow = table + (long long)r.seq[e] * g.max_pages;
            }
            tok[i] = row + shift;
            at[i] = (((long long)layer * r.rows + row) * g.H + head) * g.D + 8 * w;
        }
        page[i] = trow[tok[i] >> g.lgP];
        for (head += step; head >= g.H; head -= g.H) row++;
    }
    KvRaw8 raw[kReadItems];
#pragma unroll
    for (int i = 0; i < kReadItems; i++) {
        if ((unsigned)page[i] >= (unsigned)g.n_pages) {
            if (at[i] >= 0 && w == 0) atomicCAS(err, 0, DEVERR_FREED);
            page[i] = 0;
            at[i] = -1;
        }
        raw[i] = kv_raw8(g, pool + kv_seg_off(g, page[i], layer, hd[i]), is_v, tok[i] & (g.P - 1), w);
    }
    void *dst = is_v ? v : k;
    const bool wide = (reinterpret_cast<uintptr_t>(dst) & 31u) == 0;
#pragma unroll
    for (int i = 0; i < kReadItems; i++) {
        if (at[i] < 0) continue;
        float x[8];
        kv_values8(g, raw[i], x);
        if (F32)
            store8_f32(static_cast<float *>(dst) + at[i], x, wide);
        else if (I4)
            *reinterpret_cast<uint4 *>(static_cast<bf16 *>(dst) + at[i]) =
                make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
        else
            *reinterpret_cast<uint4 *>(static_cast<bf16 *>(dst) + at[i]) = raw[i].q;
    }
}

// The first `rows` rows of pages src to pages dst, all layers and heads: whole
// 16-row blocks, one contiguous run a segment.  The first block also applies the
// metadata updates p, which saves a growing fork a launch.  40 rows of a page for 16
// forks and 28 layers of 2 heads (4 bits): 3.9 us for 12.4 MB, bound by launch and latency.
template <int N>
struct Copies {
    static constexpr int kMax = N;
    int n;
    int src[N], dst[N], rows[N];
};
template <int N>
__global__ void __launch_bounds__(256) kv_copy_pages_kernel(const __grid_constant__ KvGeom g, uint8_t *__restrict__ pool,
                                                            const __grid_constant__ Copies<N> c, int *__restrict__ meta,
                                                            const __grid_constant__ Pokes<60> p) {
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = threadIdx.x; i < p.n; i += blockDim.x) meta[p.index[i]] = p.value[i];
    const int e = blockIdx.y, n = c.rows[e];
    const uint8_t *src = pool + (long long)c.src[e] * g.page_stride + (long long)blockIdx.x * g.seg;
    uint8_t *dst = pool + (long long)c.dst[e] * g.page_stride + (long long)blockIdx.x * g.seg;
    const int units = (n + 15) / 16 * 2 * (g.RB + g.SB);
    for (int i = threadIdx.x; i < units; i += blockDim.x)
        reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<const uint4 *>(src)[i];
}

// Rows keep[j] of table row src to rows j0 + j of table row dst (j < n), all
// layers and heads (blockIdx.y).  kLanes lanes move a row: a 16-byte unit of K or V
// each, or a row's K or V scales; units change their place within the row as the
// row's number does.  A warp has kGatherRows turns of rows in flight.  Bound by memory:
// 2926 of 6001 bf16 rows, 28 layers of 2 heads of 128: 23.5 us, 7.1 TB/s (what is
// written stays in L2 in part).
constexpr int kGatherRows = 4;
template <bool I4, int D>
__global__ void __launch_bounds__(256) kv_gather_kernel(const __grid_constant__ KvGeom geom, const int *__restrict__ table,
                                                        uint8_t *__restrict__ pool, const int *__restrict__ keep, int n,
                                                        int j0, int src, int dst) {
    pdl_wait();
    pdl_trigger();
    const KvGeom g = fixed_geom<I4, D>(geom);
    constexpr int kUnits = I4 ? D / 32 : D / 8;                  // of K, of V
    constexpr int kLanes = 2 * kUnits + (I4 ? 2 : 0) > 16 ? 32 : 16, kStep = 32 / kLanes;
    const int lane = threadIdx.x & 31, u = lane % kLanes;
    const bool unit = u < 2 * kUnits, mine = u < 2 * kUnits + (I4 ? 2 : 0);
    const bool is_v = unit ? u >= kUnits : u > 2 * kUnits;
    const int w = unit ? u - (is_v ? kUnits : 0) : 0;
    uint8_t *seg = pool + (long long)blockIdx.y * g.seg;   // (layer, head)
    const int *tsrc = table + (long long)src * g.max_pages, *tdst = table + (long long)dst * g.max_pages;
    const int j = (blockIdx.x * 8 + (threadIdx.x >> 5)) * (kGatherRows * kStep) + lane / kLanes;
    // row numbers, pages and values, each for all rows before the next depends on it
    int ra[kGatherRows], pa[kGatherRows], pb[kGatherRows];
#pragma unroll
    for (int i = 0; i < kGatherRows; i++) ra[i] = keep[min(j + i * kStep, n - 1)];
#pragma unroll
    for (int i = 0; i < kGatherRows; i++) {
        pa[i] = tsrc[ra[i] >> g.lgP];
        pb[i] = tdst[(j0 + min(j + i * kStep, n - 1)) >> g.lgP];
    }
    // where u's part of row r stands in a page
    auto place = [&](int r) {
        return unit ? kv_row_off(g, is_v, r) + (w ^ (is_v ? kv_swz_v(I4, D, r) : kv_swz_k(I4, r))) * 16 : kv_scale_off(g, is_v, r);
    };
    uint4 x[kGatherRows];
#pragma unroll
    for (int i = 0; i < kGatherRows; i++) {
        const uint8_t *at = seg + ((unsigned)pa[i] < (unsigned)g.n_pages ? pa[i] : 0) * g.page_stride + place(ra[i] & (g.P - 1));
        x[i] = make_uint4(0u, 0u, 0u, 0u);
        if (unit) x[i] = *reinterpret_cast<const uint4 *>(at);
        else if (mine && D == 128) *reinterpret_cast<uint2 *>(&x[i]) = *reinterpret_cast<const uint2 *>(at);
        else if (mine) x[i].x = *reinterpret_cast<const uint32_t *>(at);
    }
#pragma unroll
    for (int i = 0; i < kGatherRows; i++) {
        if (j + i * kStep >= n || (unsigned)pa[i] >= (unsigned)g.n_pages || (unsigned)pb[i] >= (unsigned)g.n_pages) continue;
        uint8_t *at = seg + pb[i] * g.page_stride + place((j0 + j + i * kStep) & (g.P - 1));
        if (unit) *reinterpret_cast<uint4 *>(at) = x[i];
        else if (mine && D == 128) *reinterpret_cast<uint2 *>(at) = make_uint2(x[i].x, x[i].y);
        else if (mine) *reinterpret_cast<uint32_t *>(at) = x[i].x;
    }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool seq_ok(const dtts_kv *kv, int s) { return s >= 0 && s < kv->g.max_seqs && kv->seqs[s].open; }

}  // namespace

dtts_kv::~dtts_kv() {
    mem.free_all();
    if (handoff) cudaEventDestroy(handoff);
    if (own_stream) cudaStreamDestroy(own_stream);
}

KvMeta dtts_kv::kv_meta() const {
    KvMeta m;
    m.seq = meta;
    m.start = meta + g.max_seqs;
    m.cnt = meta + 2 * g.max_seqs;
    m.len = meta + 3 * g.max_seqs;
    m.pos = meta + 4 * g.max_seqs;
    m.table = meta + 5 * g.max_seqs;
    return m;
}

// the next pending updates from i on, as many as fit
template <typename P>
void dtts_kv::take_pokes(P &p, size_t i) const {
    p.n = (int)std::min<size_t>(P::kMax, pokes.size() - i);
    for (int j = 0; j < p.n; j++) {
        p.index[j] = pokes[i + j];
        p.value[j] = meta_h[pokes[i + j]];   // an index listed twice gets its last value both times
    }
}

int dtts_kv::flush() {
    if (pokes.empty()) return DTTS_OK;
    // While the stream is capturing, a trim's marks may be pending (the calls that add pages send theirs): they stay so.
    // No call may reach the rows that they concern, and in a graph every replay would set them again, over the tables
    // of that time.
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    DTTS_CUDA(cudaStreamIsCapturing(stream, &cap));
    if (cap != cudaStreamCaptureStatusNone) return DTTS_OK;
    auto send = [&](auto &p, size_t i) -> int {
        constexpr int kMax = std::remove_reference_t<decltype(p)>::kMax;
        take_pokes(p, i);
        DTTS_CUDA(launch_k(kv_pdl(), kv_poke_kernel<kMax>, dim3(1), dim3(256), 0, stream, meta, p));
        return DTTS_OK;
    };
    Pokes<60> few;
    Pokes<500> many;
    for (size_t i = 0; i < pokes.size(); i += pokes.size() <= 60 ? 60 : 500) {
        int st = pokes.size() <= 60 ? send(few, i) : send(many, i);
        if (st) return st;
    }
    pokes.clear();
    return DTTS_OK;
}

void dtts_kv::drop_batch() {
    b_seq.clear();
    b_cnt.clear();
    b_len.clear();
    b_rows = 0;
}

int dtts_kv::not_capturing(const char *what) const {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    DTTS_CUDA(cudaStreamIsCapturing(stream, &st));
    DTTS_CHECK(st == cudaStreamCaptureStatusNone, DTTS_ERR_UNSUPPORTED,
               "%s changes the cache's tables and cannot be captured into a graph", what);
    return DTTS_OK;
}

int dtts_kv::fits(int n_seq, const int *sq, const int *n_new, long long *pages) {
    std::vector<int> listed(sq, sq + n_seq);
    std::sort(listed.begin(), listed.end());
    DTTS_CHECK(std::adjacent_find(listed.begin(), listed.end()) == listed.end(), DTTS_ERR_ARG,
               "a sequence is listed twice");
    long long need = 0, rows = 0;
    std::vector<int> lowered;   // shared tail pages counted as copied
    lowered.reserve(n_seq);
    for (int b = 0; b < n_seq; b++) {
        const Seq &s = seqs[sq[b]];
        const long long len = (long long)s.len + n_new[b];
        if (len > max_tokens || (long long)s.pos + n_new[b] > INT32_MAX) {
            for (int p : lowered) refs[p]++;
            set_error("sequence %d would hold %lld tokens (limit %lld)", sq[b], len, max_tokens);
            return DTTS_ERR_ARG;
        }
        rows += n_new[b];
        need += (len + g.P - 1) / g.P - (long long)s.pages.size();
        if (n_new[b] > 0 && (s.len & (g.P - 1)) && refs[s.pages.back()] > 1) {
            need++;
            refs[s.pages.back()]--;
            lowered.push_back(s.pages.back());
        }
    }
    for (int p : lowered) refs[p]++;
    DTTS_CHECK(rows <= INT32_MAX / 2, DTTS_ERR_ARG, "%lld new rows in one batch", rows);
    DTTS_CHECK(need <= (long long)free_pages.size(), DTTS_ERR_OOM, "%lld pages needed, %zu free", need,
               free_pages.size());
    *pages = need;
    return DTTS_OK;
}

void dtts_kv::take_back() {
    for (auto x = grown.rbegin(); x != grown.rend(); ++x) {
        Seq &s = seqs[x->seq];
        for (; (int)s.pages.size() > x->pages; s.pages.pop_back()) drop_page(s.pages.back());
        if (x->tail >= 0) {
            drop_page(s.pages.back());
            s.pages.back() = x->tail;
            refs[x->tail]++;
            poke(table_at(x->seq, x->pages - 1), x->tail);
        }
        s.len = x->len;
        s.pos = x->pos;
    }
    grown.clear();
    drop_batch();
}

// Grows the sequences and makes them the current batch.  Nothing changes unless
// everything fits and every launch succeeds.
int dtts_kv::extend(int n_seq, const int *sq, const int *n_new) {
    long long need = 0;
    int st = not_capturing("extend");
    if (st || (st = fits(n_seq, sq, n_new, &need))) return st;
    // room for all that is listed below first: from the first change on, nothing throws
    std::vector<Copy> copies;
    copies.reserve(n_seq);
    grown.clear();
    grown.reserve(n_seq);
    pokes.reserve(pokes.size() + (size_t)need + 5 * (size_t)g.max_seqs + 2 * (size_t)n_seq);   // also take_back's
    for (int b = 0; b < n_seq; b++) {
        Seq &s = seqs[sq[b]];
        const size_t pages = (size_t)((s.len + (long long)n_new[b] + g.P - 1) / g.P);
        if (pages > s.pages.capacity()) s.pages.reserve(std::max(pages, 2 * s.pages.size()));
    }
    b_seq.reserve(n_seq);
    b_cnt.reserve(n_seq);
    b_len.reserve(n_seq);
    b_seq.assign(sq, sq + n_seq);
    b_cnt.assign(n_new, n_new + n_seq);
    b_len.resize(n_seq);
    int start = 0;
    for (int b = 0; b < n_seq; b++) {
        Seq &s = seqs[sq[b]];
        Growth was = {sq[b], s.len, s.pos, (int)s.pages.size(), -1};
        if (n_new[b] > 0 && (s.len & (g.P - 1)) && refs[s.pages.back()] > 1) {
            const int from = s.pages.back(), to = take_page();
            refs[from]--;   // shared: never the last user here
            s.pages.back() = to;
            was.tail = from;
            poke(table_at(sq[b], (int)s.pages.size() - 1), to);
            copies.push_back({from, to, s.len & (g.P - 1)});
        }
        grown.push_back(was);
        const int pos = s.pos;
        s.len += n_new[b];
        s.pos += n_new[b];
        while ((long long)s.pages.size() * g.P < s.len) {
            s.pages.push_back(take_page());
            poke(table_at(sq[b], (int)s.pages.size() - 1), s.pages.back());
        }
        b_len[b] = s.len;
        poke(b, sq[b]);
        poke(g.max_seqs + b, start);
        poke(2 * g.max_seqs + b, n_new[b]);
        poke(3 * g.max_seqs + b, s.len);
        poke(4 * g.max_seqs + b, pos);
        start += n_new[b];
    }
    b_rows = start;
    last_entries = n_seq;
    // entries behind the batch hold no rows: row lookups of a graph captured for more entries stay in range, and
    // kv_batch_over tells by them that there are more entries than at a capture
    for (int b = n_seq; b < g.max_seqs; b++) {
        poke(g.max_seqs + b, start);
        poke(2 * g.max_seqs + b, 0);
    }
    if ((st = send_growth(copies))) take_back();
    return st;
}

// Enqueues the copies of shared last pages and the pending metadata updates.
int dtts_kv::send_growth(const std::vector<Copy> &copies) {
    int st = DTTS_OK;
    Pokes<60> own;   // sent with the first copies
    own.n = 0;
    if (!copies.empty() && pokes.size() <= 60) take_pokes(own, 0);
    auto send = [&](auto &c, size_t i) -> int {
        constexpr int kMax = std::remove_reference_t<decltype(c)>::kMax;
        c.n = (int)std::min<size_t>(kMax, copies.size() - i);
        for (int j = 0; j < c.n; j++) {
            c.src[j] = copies[i + j].src;
            c.dst[j] = copies[i + j].dst;
            c.rows[j] = copies[i + j].rows;
        }
        DTTS_CUDA(launch_k(kv_pdl(), kv_copy_pages_kernel<kMax>, dim3(g.L * g.H, c.n), dim3(256), 0, stream, g, pool, c, meta, own));
        return DTTS_OK;
    };
    Copies<40> few;
    Copies<240> many;
    for (size_t i = 0; i < copies.size(); i += copies.size() <= 40 ? 40 : 240)
        if ((st = copies.size() <= 40 ? send(few, i) : send(many, i))) return st;
    if (own.n) pokes.clear();
    return flush();
}

namespace {
// whether `cnt` queries from row i0 on see only rows that no trim has freed
bool reachable(const dtts_kv &kv, const dtts_kv::Seq &s, int i0, int cnt, int window, int sinks) {
    if (s.hole_lo >= s.hole_hi || cnt == 0) return true;
    const long long lo = window ? std::max(0ll, (long long)i0 - window + 1) : 0;
    return lo >= (long long)s.hole_hi * kv.g.P && std::min<long long>(sinks, lo) <= (long long)s.hole_lo * kv.g.P;
}
}  // namespace

int dtts_kv::check_window(int n_seq, const int *sq, const int *n_new, int window, int sinks) const {
    DTTS_CHECK(window >= 0 && sinks >= 0, DTTS_ERR_ARG, "window %d, sinks %d", window, sinks);
    for (int b = 0; b < n_seq; b++)
        if (!reachable(*this, seqs[sq[b]], seqs[sq[b]].len, n_new[b], window, sinks)) {
            set_error("the window reaches rows of sequence %d that a trim freed", sq[b]);
            return DTTS_ERR_ARG;
        }
    return DTTS_OK;
}

int dtts_kv::max_splits(int n_seq) const {
    const long long units = (long long)n_seq * g.H, slots = kWsFloats / ((long long)kKvFewRows * (g.D + 2));
    return units > kMaxUnits ? 1 : (int)std::max(1ll, slots / units);
}

int dtts_kv::plan_attend(const dtts_kv_attend_args &a, KvAttendPlan *plan) const {
    DTTS_CHECK(!b_seq.empty(), DTTS_ERR_ARG, "no current batch: call dtts_kv_extend first");
    DTTS_CHECK(a.n_heads >= 1 && a.n_heads % g.H == 0 && a.n_heads / g.H <= 128, DTTS_ERR_ARG,
               "%d query heads over %d key heads (a multiple, 128 to one at most)", a.n_heads, g.H);
    DTTS_CHECK(a.window >= 0 && a.sinks >= 0, DTTS_ERR_ARG, "window %d, sinks %d", a.window, a.sinks);
    DTTS_CHECK(a.scale > 0.f && a.scale <= 1e30f, DTTS_ERR_ARG, "scale %g", (double)a.scale);
    const int n_seq = (int)b_seq.size(), G = a.n_heads / g.H;
    for (int b = 0; b < n_seq; b++)
        if (!reachable(*this, seqs[b_seq[b]], b_len[b] - b_cnt[b], b_cnt[b], a.window, a.sinks)) {
            set_error("the window reaches rows of sequence %d that a trim freed", b_seq[b]);
            return DTTS_ERR_ARG;
        }
    plan->rows_or_pairs[0] = plan->rows_or_pairs[1] = 0;
    plan->args[0].both = plan->args[1].both = 0;
    if (b_rows == 0) return DTTS_OK;
    DTTS_CHECK(a.q && a.out, DTTS_ERR_ARG, "null argument");
    DTTS_CHECK(aligned16(a.q) && aligned16(a.out) && !((a.q_row | a.q_head | a.out_row | a.out_head) & 7), DTTS_ERR_ARG,
               "rows must start on 16-byte boundaries");
    KvAttendArgs p;
    p.g = g;
    p.m = kv_meta();
    p.pool = pool;
    p.q = (const bf16 *)a.q;
    p.out = (bf16 *)a.out;
    p.q_row = a.q_row; p.q_head = a.q_head; p.o_row = a.out_row; p.o_head = a.out_head;
    p.n_seq = n_seq; p.G = G; p.total_rows = b_rows;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    // what no sequence reaches, cut so that row numbers minus or plus them stay in 32 bits
    p.window = a.window >= max_tokens ? 0 : a.window;
    p.sinks = (int)std::min<long long>(a.sinks, max_tokens);
    p.ws = ws; p.cnt = cnt; p.err = d_err;
    std::vector<std::pair<int, int>> parts;
    // both kernels run where a batch mixes steps and prompts; each takes its own sequences
    for (int many = 0; many < 2; many++) {
        const int kt = many ? kKvManyKeyTile : shapes.few_key_tile;
        long long tiles = 0, max_tiles = 0;
        int max_rows = 0;
        parts.clear();   // (key tiles, row tiles) of this kernel's sequences
        int same[32] = {};   // sequences of so few key tiles are counted, not listed
        for (int b = 0; b < n_seq; b++) {
            const long long rows = (long long)b_cnt[b] * G;
            if (rows == 0 || (rows > kKvFewRows) != (many == 1)) continue;
            const long long lo = a.window ? std::max(0ll, (long long)b_len[b] - b_cnt[b] - a.window + 1) : 0;
            const long long nt = (b_len[b] + kt - 1) / kt - lo / kt + (std::min<long long>(a.sinks, lo) + kt - 1) / kt;
            const long long rt = many ? (rows + 255) / 256 : 1;
            tiles += nt * rt * g.H;
            max_tiles = std::max(max_tiles, nt);
            max_rows = (int)std::min<long long>(INT32_MAX / 2, std::max<long long>(max_rows, rows));
            if (nt < 32) same[nt] += (int)rt;
            else parts.emplace_back((int)nt, (int)rt);
        }
        for (int nt = 1; nt < 32; nt++)
            if (same[nt]) parts.emplace_back(nt, same[nt]);
        if (!max_rows) continue;
        const int rt = many ? (max_rows + 255) / 256 : 1;
        const long long units = (long long)n_seq * g.H * rt;
        DTTS_CHECK(units <= INT32_MAX, DTTS_ERR_ARG, "%lld row tiles in one batch", units);
        auto ctas = [&](long long per) {
            const int len = (int)per;
            long long n = 0;
            for (auto &x : parts) n += (long long)((x.first + len - 1) / len) * x.second;
            return n * g.H;
        };
        const long long slots = kWsFloats / (many ? 256ll : (long long)kKvFewRows) / (g.D + 2);
        const long long most = units > kMaxUnits ? 1 : std::max(1ll, slots / units);   // parts that the workspace has room for
        long long per = max_tiles;
        if (many) {
            // Parts of the key ranges: as short as they may be with all CTAs resident at once, or no split at all
            long long hi = per;
            per = std::min(hi, std::max(2ll, (tiles + num_sms - 1) / num_sms));
            while (per < hi) {
                const long long mid = (per + hi) / 2;
                if (ctas(mid) <= num_sms) hi = mid; else per = mid + 1;
            }
        } else {
            // The number of parts of the longest range with the least time for all: the tiles of the warps that share
            // an SM, and the join, 1.2 us and 0.16 more a part.  No split beats two halves for 64 sequences of 1000
            // 4-bit rows (12.0 against 14.7 us); as many parts as fit take 37 us for one of 16000 bf16 rows, this 15.
            const int wide = max_rows > 8, resident = std::min(3, std::max(1, shapes.few_ctas[wide]));
            float best = INFINITY;
            // whether parts of len tiles fit on the SMs at once; they are kept where they take the least time so far
            auto fits = [&](long long len) {
                const long long n = (max_tiles + len - 1) / len, c = (ctas(len) + num_sms - 1) / num_sms;
                if (n > 1 && c > resident) return false;
                const int at = (int)std::min<long long>(c, resident) - 1;
                const int w = shapes.few_warps;   // few tiles: the warp with one more counts
                const float turns = len < 8 * w ? (float)((len + w - 1) / w) : (float)len / w;
                const float us = turns * (float)c * shapes.few_tile_us[wide][at] +
                                 shapes.few_start_us[at] + (n > 1 ? 1.2f + 0.16f * (float)n : 0.f);
                if (us < best) {
                    best = us;
                    per = len;
                }
                return true;
            };
            long long hi = max_tiles, lo = 0;   // the shortest parts that fit, the longest that do not
            for (long long n = 1; n <= std::min(most, max_tiles) && !lo; n += 1 + n / 16) {
                const long long len = (max_tiles + n - 1) / n;
                if (fits(len)) hi = len; else lo = len;
            }
            while (lo && hi - lo > 1) {
                const long long mid = (lo + hi) / 2;
                if (fits(mid)) hi = mid; else lo = mid;
            }
        }
        const long long splits = std::max(1ll, std::min((max_tiles + per - 1) / per, most));
        p.splits = (short)splits;
        p.tiles_per_split = (int)per;
        plan->args[many] = p;
        plan->rows_or_pairs[many] = many ? rt : max_rows;
    }
    plan->args[0].both = plan->args[1].both = plan->rows_or_pairs[0] && plan->rows_or_pairs[1];
    return DTTS_OK;
}

int dtts_kv::attend(const KvAttendPlan &plan, int layer) {
    for (int many = 0; many < 2; many++) {
        if (!plan.rows_or_pairs[many]) continue;
        KvAttendArgs p = plan.args[many];
        p.pool += (long long)layer * g.H * g.seg;
        DTTS_CUDA(launch_kv_attend(p, many == 1, plan.rows_or_pairs[many], stream));
    }
    return DTTS_OK;
}

int dtts_kv::check_batch(int n_seq, const int *sq, const int *n_new) const {
    DTTS_CHECK(n_seq >= 1 && n_seq <= g.max_seqs, DTTS_ERR_ARG, "%d sequences (1..%d)", n_seq, g.max_seqs);
    for (int b = 0; b < n_seq; b++) {
        DTTS_CHECK(seq_ok(this, sq[b]), DTTS_ERR_ARG, "sequence %d is not open", sq[b]);
        DTTS_CHECK(n_new[b] >= 0, DTTS_ERR_ARG, "%d new tokens", n_new[b]);
    }
    return DTTS_OK;
}

extern "C" {

int dtts_kv_create(const dtts_kv_config *c, int device, dtts_kv **out) try {
    DTTS_CHECK(c && out, DTTS_ERR_ARG, "null argument");
    *out = nullptr;
    DTTS_CHECK(c->dtype == DTTS_DTYPE_BF16 || c->dtype == DTTS_DTYPE_INT4, DTTS_ERR_UNSUPPORTED, "dtype %d", c->dtype);
    DTTS_CHECK(c->head_dim == 64 || c->head_dim == 128, DTTS_ERR_UNSUPPORTED, "head_dim %d (64 or 128)", c->head_dim);
    DTTS_CHECK(c->page_tokens == 16 || c->page_tokens == 32 || c->page_tokens == 64 || c->page_tokens == 128,
               DTTS_ERR_UNSUPPORTED, "page_tokens %d (16, 32, 64 or 128)", c->page_tokens);
    DTTS_CHECK(c->n_layers >= 1 && c->n_layers <= 1024 && c->n_kv_heads >= 1 && c->n_kv_heads <= 256, DTTS_ERR_ARG,
               "bad geometry: %d layers, %d heads", c->n_layers, c->n_kv_heads);
    DTTS_CHECK((long long)c->n_layers * c->n_kv_heads <= 65535, DTTS_ERR_ARG, "%d layers of %d heads (65535 in all)",
               c->n_layers, c->n_kv_heads);
    DTTS_CHECK(c->n_pages >= 1 && c->max_seqs >= 1 && c->max_seqs <= 65535 && c->max_tokens >= 1 &&
                   c->max_tokens <= (1 << 24),
               DTTS_ERR_ARG, "bad capacity: %d pages, %d sequences of %d tokens", c->n_pages, c->max_seqs, c->max_tokens);
    const int P = c->page_tokens;
    const long long max_pages = ((long long)c->max_tokens + P - 1) / P;
    const long long ints = 5ll * c->max_seqs + (long long)(c->max_seqs + 1) * max_pages;
    DTTS_CHECK(ints <= INT32_MAX, DTTS_ERR_ARG, "page tables of %d sequences of %d tokens", c->max_seqs, c->max_tokens);
    int nsm = 0, st = check_device(device, &nsm);
    if (st) return st;
    DeviceGuard dg(device);
    std::unique_ptr<dtts_kv> kv(new dtts_kv());
    kv->device = device;
    kv->num_sms = nsm;
    static std::atomic<long long> uids{0};
    kv->uid = ++uids;
    kv->max_tokens = c->max_tokens;
    KvGeom &g = kv->g;
    g.L = c->n_layers; g.H = c->n_kv_heads; g.D = c->head_dim; g.P = P;
    g.lgP = P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : 7;
    g.i4 = c->dtype == DTTS_DTYPE_INT4;
    g.RB = g.i4 ? g.D / 2 : g.D * 2;
    g.SB = g.i4 ? g.D / kKvGroup * 2 : 0;
    g.seg = 2ll * P * (g.RB + g.SB);
    g.page_stride = g.seg * g.L * g.H;
    g.n_pages = c->n_pages; g.max_seqs = c->max_seqs; g.max_pages = (int)max_pages;
    DTTS_CUDA(cudaStreamCreateWithFlags(&kv->own_stream, cudaStreamNonBlocking));
    kv->stream = kv->own_stream;
    DTTS_CUDA(cudaEventCreateWithFlags(&kv->handoff, cudaEventDisableTiming));
    DTTS_CUDA(kv_attend_prepare(g, &kv->shapes));
    const size_t pool_bytes = (size_t)g.page_stride * g.n_pages;
    kv->pool = (uint8_t *)kv->mem.alloc(pool_bytes);
    kv->meta = (int *)kv->mem.alloc((size_t)ints * 4);
    kv->keep = (int *)kv->mem.alloc((size_t)c->max_tokens * 4);
    kv->cnt = (int *)kv->mem.alloc((size_t)kMaxUnits * 4);
    kv->d_err = (int *)kv->mem.alloc(4);
    kv->ws = (float *)kv->mem.alloc((size_t)kWsFloats * 4);
    if (!kv->pool || !kv->meta || !kv->keep || !kv->cnt || !kv->d_err || !kv->ws) {
        cudaGetLastError();   // a failed cudaMalloc must not surface in a later call
        set_error("K/V cache allocation failed (%zu MB of pages)", pool_bytes >> 20);
        return DTTS_ERR_OOM;
    }
    kv->meta_h.assign((size_t)ints, 0);
    DTTS_CUDA(cudaMemsetAsync(kv->pool, 0, pool_bytes, kv->stream));
    DTTS_CUDA(cudaMemsetAsync(kv->meta, 0, (size_t)ints * 4, kv->stream));
    DTTS_CUDA(cudaMemsetAsync(kv->cnt, 0, (size_t)kMaxUnits * 4, kv->stream));
    DTTS_CUDA(cudaMemsetAsync(kv->d_err, 0, 4, kv->stream));
    DTTS_CUDA(cudaStreamSynchronize(kv->stream));
    kv->seqs.resize(g.max_seqs);
    kv->refs.assign(g.n_pages, 0);
    for (int p = 0; p < g.n_pages; p++) kv->free_pages.push(p);
    *out = kv.release();
    return DTTS_OK;
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return DTTS_ERR_OOM;
}

int dtts_kv_destroy(dtts_kv *kv) {
    if (!kv) return DTTS_OK;
    DeviceGuard dg(kv->device);
    cudaDeviceSynchronize();   // its work may be on streams that no longer exist
    delete kv;
    return DTTS_OK;
}

int dtts_kv_set_stream(dtts_kv *kv, void *stream) {
    DTTS_CHECK(kv, DTTS_ERR_ARG, "null cache");
    cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : kv->own_stream;
    if (s == kv->stream) return DTTS_OK;
    DeviceGuard dg(kv->device);
    // work already enqueued on the old stream stays before what follows on the new one
    cudaStreamCaptureStatus a = cudaStreamCaptureStatusNone, b = cudaStreamCaptureStatusNone;
    DTTS_CUDA(cudaStreamIsCapturing(kv->stream, &a));
    DTTS_CUDA(cudaStreamIsCapturing(s, &b));
    if (a == cudaStreamCaptureStatusNone && b == cudaStreamCaptureStatusNone) {
        DTTS_CUDA(cudaEventRecord(kv->handoff, kv->stream));
        DTTS_CUDA(cudaStreamWaitEvent(s, kv->handoff, 0));
    }
    kv->stream = s;
    return DTTS_OK;
}

int dtts_kv_sync(dtts_kv *kv) {
    DTTS_CHECK(kv, DTTS_ERR_ARG, "null cache");
    DeviceGuard dg(kv->device);
    int st = stream_wait(kv->stream, 300.0);
    if (st) return st;
    int err = 0;
    DTTS_CUDA(cudaMemcpy(&err, kv->d_err, 4, cudaMemcpyDeviceToHost));
    if (err) {
        cudaMemset(kv->d_err, 0, 4);
        DTTS_CHECK(err != DEVERR_BATCH, DTTS_ERR_ARG,
                   "a replayed graph met a batch whose sequences have other numbers of new tokens than at its capture");
        DTTS_CHECK(err != DEVERR_FREED, DTTS_ERR_ARG, "a replayed graph reached rows that a trim had freed");
        set_error("device wait limit reached (code %d)", err);
        return DTTS_ERR_TIMEOUT;
    }
    return DTTS_OK;
}

int dtts_kv_open(dtts_kv *kv, int *seq) {
    DTTS_CHECK(kv && seq, DTTS_ERR_ARG, "null argument");
    for (int s = 0; s < kv->g.max_seqs; s++)
        if (!kv->seqs[s].open) {
            kv->seqs[s] = dtts_kv::Seq();
            kv->seqs[s].open = true;
            *seq = s;
            return DTTS_OK;
        }
    set_error("all %d sequences are open", kv->g.max_seqs);
    return DTTS_ERR_OOM;
}

int dtts_kv_close(dtts_kv *kv, int n, const int *seqs) try {
    DTTS_CHECK(kv && (n == 0 || seqs) && n >= 0, DTTS_ERR_ARG, "null argument");
    for (int i = 0; i < n; i++) DTTS_CHECK(seq_ok(kv, seqs[i]), DTTS_ERR_ARG, "sequence %d is not open", seqs[i]);
    std::vector<int> listed(seqs, seqs + n);
    std::sort(listed.begin(), listed.end());
    DTTS_CHECK(std::adjacent_find(listed.begin(), listed.end()) == listed.end(), DTTS_ERR_ARG,
               "a sequence is listed twice");
    for (int s : listed) {
        for (int p : kv->seqs[s].pages) kv->drop_page(p);
        kv->seqs[s] = dtts_kv::Seq();
    }
    for (int s : kv->b_seq)
        if (std::binary_search(listed.begin(), listed.end(), s)) { kv->drop_batch(); break; }
    return DTTS_OK;
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return DTTS_ERR_OOM;
}

int dtts_kv_fork(dtts_kv *kv, int src, int n, int *dst) try {
    DTTS_CHECK(kv && (n == 0 || dst) && n >= 0, DTTS_ERR_ARG, "null argument");
    DTTS_CHECK(seq_ok(kv, src), DTTS_ERR_ARG, "sequence %d is not open", src);
    DeviceGuard dg(kv->device);
    int st = kv->not_capturing("fork");
    if (st) return st;
    std::vector<int> to;
    for (int s = 0; s < kv->g.max_seqs && (int)to.size() < n; s++)
        if (!kv->seqs[s].open) to.push_back(s);
    DTTS_CHECK((int)to.size() == n, DTTS_ERR_OOM, "%d sequences wanted, %zu free", n, to.size());
    if ((st = kv->flush())) return st;   // the source's row on the device is current
    const int pages = (int)kv->seqs[src].pages.size();
    auto send = [&](auto &f, int i) -> int {
        constexpr int kMax = std::remove_reference_t<decltype(f)>::kMax;
        f.n = std::min(kMax, n - i);
        f.src = src;
        f.pages = pages;
        for (int j = 0; j < f.n; j++) f.dst[j] = to[i + j];
        DTTS_CUDA(launch_k(kv_pdl(), kv_fork_tables_kernel<kMax>, dim3(f.n), dim3(128), 0, kv->stream,
                           kv->meta + 5 * kv->g.max_seqs, kv->g.max_pages, f));
        return DTTS_OK;
    };
    Forks<60> few;
    Forks<900> many;
    for (int i = 0; i < n && pages; i += n <= 60 ? 60 : 900)
        if ((st = n <= 60 ? send(few, i) : send(many, i))) return st;
    for (int s : to) {
        kv->seqs[s] = kv->seqs[src];
        for (int p = 0; p < pages; p++) {
            kv->meta_h[kv->table_at(s, p)] = kv->meta_h[kv->table_at(src, p)];
            if (kv->seqs[s].pages[p] >= 0) kv->refs[kv->seqs[s].pages[p]]++;
        }
    }
    std::copy(to.begin(), to.end(), dst);
    return DTTS_OK;
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return DTTS_ERR_OOM;
}

int dtts_kv_truncate(dtts_kv *kv, int seq, int n_tokens) {
    DTTS_CHECK(kv, DTTS_ERR_ARG, "null cache");
    DTTS_CHECK(seq_ok(kv, seq), DTTS_ERR_ARG, "sequence %d is not open", seq);
    dtts_kv::Seq &s = kv->seqs[seq];
    DTTS_CHECK(n_tokens >= 0 && n_tokens <= s.len, DTTS_ERR_ARG, "sequence %d holds %d tokens, not %d", seq, s.len,
               n_tokens);
    const int keep = (n_tokens + kv->g.P - 1) / kv->g.P;
    DTTS_CHECK(keep == 0 || n_tokens == s.len || s.pages[keep - 1] >= 0, DTTS_ERR_ARG,
               "row %d of sequence %d was freed by a trim", n_tokens - 1, seq);
    if (n_tokens == s.len) return DTTS_OK;
    for (size_t p = keep; p < s.pages.size(); p++) kv->drop_page(s.pages[p]);
    s.pages.resize(keep);
    s.hole_hi = std::min(s.hole_hi, keep);
    if (s.hole_lo >= s.hole_hi) s.hole_lo = s.hole_hi = 0;
    s.pos -= s.len - n_tokens;
    s.len = n_tokens;
    for (int b : kv->b_seq)
        if (b == seq) { kv->drop_batch(); break; }
    return DTTS_OK;
}

int dtts_kv_trim(dtts_kv *kv, int seq, int window, int sinks) try {
    DTTS_CHECK(kv, DTTS_ERR_ARG, "null cache");
    DTTS_CHECK(seq_ok(kv, seq), DTTS_ERR_ARG, "sequence %d is not open", seq);
    DTTS_CHECK(window >= 1 && sinks >= 0, DTTS_ERR_ARG, "window %d, sinks %d", window, sinks);
    dtts_kv::Seq &s = kv->seqs[seq];
    const int P = kv->g.P;
    // the next token, at row len, sees rows > len - window and rows < sinks
    const long long lo = std::max(0ll, (long long)s.len - window + 1);
    const long long a = ((long long)sinks + P - 1) / P, b = std::min<long long>(lo / P, (long long)s.pages.size());
    if (a >= b) return DTTS_OK;
    bool any = false;
    for (long long p = a; p < b; p++)
        if (s.pages[p] >= 0) {
            kv->drop_page(s.pages[p]);
            s.pages[p] = -1;
            kv->poke(kv->table_at(seq, (int)p), -1);
            any = true;
        }
    if (!any) return DTTS_OK;
    if (s.hole_lo >= s.hole_hi) {
        s.hole_lo = (int)a;
        s.hole_hi = (int)b;
    } else {
        s.hole_lo = std::min(s.hole_lo, (int)a);
        s.hole_hi = std::max(s.hole_hi, (int)b);
    }
    for (int e : kv->b_seq)
        if (e == seq) { kv->drop_batch(); break; }
    return DTTS_OK;
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return DTTS_ERR_OOM;
}

int dtts_kv_compact(dtts_kv *kv, int seq, int n_keep, const int *keep) try {
    DTTS_CHECK(kv && (n_keep == 0 || keep) && n_keep >= 0, DTTS_ERR_ARG, "null argument");
    DTTS_CHECK(seq_ok(kv, seq), DTTS_ERR_ARG, "sequence %d is not open", seq);
    DeviceGuard dg(kv->device);
    int st = kv->not_capturing("compact");
    if (st) return st;
    dtts_kv::Seq &s = kv->seqs[seq];
    const KvGeom &g = kv->g;
    DTTS_CHECK(n_keep <= s.len, DTTS_ERR_ARG, "sequence %d holds %d rows, not %d", seq, s.len, n_keep);
    for (int j = 0; j < n_keep; j++) {
        DTTS_CHECK(keep[j] >= 0 && keep[j] < s.len && (j == 0 || keep[j] > keep[j - 1]), DTTS_ERR_ARG,
                   "kept rows must ascend within 0..%d (entry %d is %d)", s.len - 1, j, keep[j]);
        DTTS_CHECK(s.pages[keep[j] >> g.lgP] >= 0, DTTS_ERR_ARG, "row %d of sequence %d was freed by a trim", keep[j], seq);
    }
    // pages of the unchanged start stay; the rest goes to fresh pages
    int same = 0;
    while (same < n_keep && keep[same] == same) same++;
    const int stay = same == n_keep && n_keep == s.len ? (int)s.pages.size() : same >> g.lgP;
    const int total = (n_keep + g.P - 1) / g.P, fresh = std::max(0, total - stay);
    if (stay == (int)s.pages.size() && n_keep == s.len) return DTTS_OK;
    DTTS_CHECK(fresh <= (int)kv->free_pages.size(), DTTS_ERR_OOM, "%d pages needed, %zu free", fresh,
               kv->free_pages.size());
    // pages are about to change hands: without a current batch, a replayed graph (which is not allowed, but cannot be seen)
    // finds no rows any more that it could store on a page that the last batch had; extend, which also takes pages, makes
    // a batch of its own
    if (kv->b_seq.empty())
        for (int b = 0; b < kv->last_entries; b++) kv->poke(2 * g.max_seqs + b, 0);
    const int j0 = stay << g.lgP, n = n_keep - j0, scratch = g.max_seqs;
    std::vector<int> pages(s.pages.begin(), s.pages.begin() + stay);
    for (int p = stay; p < total; p++) {
        pages.push_back(kv->take_page());
        kv->poke(kv->table_at(scratch, p), pages.back());
    }
    Pokes<60> own;   // the new pages' entries travel with the first rows
    own.n = 0;
    const bool beside = n > 0 && kv->pokes.size() <= 60;
    if (beside)
        kv->take_pokes(own, 0);
    else if ((st = kv->flush()))
        return st;
    if (n > 0) {
        const int first = keep[j0] >> 5, words = (keep[n_keep - 1] >> 5) - first + 1;
        std::vector<uint32_t> bits((size_t)words, 0u);
        for (int j = j0; j < n_keep; j++) bits[(keep[j] >> 5) - first] |= 1u << (keep[j] & 31);
        int base = 0;
        auto send = [&](auto &k, int i) -> int {
            constexpr int kMax = std::remove_reference_t<decltype(k)>::kMax;
            k.n = std::min(kMax, words - i);
            k.first = first + i;
            k.base = base;
            for (int x = 0; x < k.n; x++) {
                k.word[x] = bits[i + x];
                base += __builtin_popcount(k.word[x]);
            }
            if (base == k.base) return DTTS_OK;   // none kept here; the first words hold a row
            DTTS_CUDA(launch_k(kv_pdl(), kv_keep_kernel<kMax>, dim3(1), dim3((k.n + 31) / 32 * 32), 0, kv->stream, kv->keep, k,
                               kv->meta, own));
            return DTTS_OK;
        };
        KeepBits<224> few;
        KeepBits<768> many;
        for (int i = 0; i < words; i += words <= 224 ? 224 : 768)
            if ((st = words <= 224 ? send(few, i) : send(many, i))) return st;
        if (beside) kv->pokes.clear();
        auto gather = [&](auto kernel, int rows_a_warp) {
            return launch_k(kv_pdl(), kernel, dim3((n + 8 * rows_a_warp - 1) / (8 * rows_a_warp), g.L * g.H), dim3(256), 0,
                            kv->stream, g, (const int *)(kv->meta + 5 * g.max_seqs), kv->pool, (const int *)kv->keep, n, j0,
                            seq, scratch);
        };
        DTTS_CUDA(g.i4 ? (g.D == 128 ? gather(kv_gather_kernel<true, 128>, 2 * kGatherRows)
                                     : gather(kv_gather_kernel<true, 64>, 2 * kGatherRows))
                       : (g.D == 128 ? gather(kv_gather_kernel<false, 128>, kGatherRows)
                                     : gather(kv_gather_kernel<false, 64>, 2 * kGatherRows)));
    }
    for (int p = 0; p < total; p++) kv->poke(kv->table_at(seq, p), pages[p]);
    if ((st = kv->flush())) return st;
    for (size_t p = stay; p < s.pages.size(); p++) kv->drop_page(s.pages[p]);
    s.pages.swap(pages);
    s.len = n_keep;
    s.hole_lo = s.hole_hi = 0;
    for (int b : kv->b_seq)
        if (b == seq) { kv->drop_batch(); break; }
    return DTTS_OK;
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return DTTS_ERR_OOM;
}

int dtts_kv_length(dtts_kv *kv, int seq, int *tokens, int *position) {
    DTTS_CHECK(kv, DTTS_ERR_ARG, "null cache");
    DTTS_CHECK(seq_ok(kv, seq), DTTS_ERR_ARG, "sequence %d is not open", seq);
    if (tokens) *tokens = kv->seqs[seq].len;
    if (position) *position = kv->seqs[seq].pos;
    return DTTS_OK;
}

int dtts_kv_free_pages(dtts_kv *kv, int *n) {
    DTTS_CHECK(kv && n, DTTS_ERR_ARG, "null argument");
    *n = (int)kv->free_pages.size();
    return DTTS_OK;
}

int dtts_kv_extend(dtts_kv *kv, int n_seq, const int *seqs, const int *n_new) try {
    DTTS_CHECK(kv && seqs && n_new, DTTS_ERR_ARG, "null argument");
    int st = kv->check_batch(n_seq, seqs, n_new);
    if (st) return st;
    DeviceGuard dg(kv->device);
    return kv->extend(n_seq, seqs, n_new);
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return DTTS_ERR_OOM;
}

int dtts_kv_write(dtts_kv *kv, int layer, const void *k, const void *v, long long k_row, long long k_head,
                  long long v_row, long long v_head) {
    DTTS_CHECK(kv, DTTS_ERR_ARG, "null cache");
    const KvGeom &g = kv->g;
    DTTS_CHECK(layer >= 0 && layer < g.L, DTTS_ERR_ARG, "layer %d of %d", layer, g.L);
    DTTS_CHECK(!kv->b_seq.empty(), DTTS_ERR_ARG, "no current batch: call dtts_kv_extend first");
    if (kv->b_rows == 0) return DTTS_OK;
    DTTS_CHECK(k && v, DTTS_ERR_ARG, "null argument");
    DTTS_CHECK(aligned16(k) && aligned16(v) && !((k_row | k_head | v_row | v_head) & 7), DTTS_ERR_ARG,
               "rows must start on 16-byte boundaries");
    DeviceGuard dg(kv->device);
    int st = kv->flush();
    if (st) return st;
    const int per_block = 256 / (g.D / 4) * kWriteItems;
    const long long items = (long long)kv->b_rows * g.H;
    DTTS_CHECK((items + per_block - 1) / per_block <= INT32_MAX, DTTS_ERR_ARG, "%d rows in one batch", kv->b_rows);
    auto write = [&](auto kernel) {
        return launch_k(kv_pdl(), kernel, dim3((unsigned)((items + per_block - 1) / per_block)), dim3(256), 0, kv->stream, g,
                        kv->kv_meta(), kv->pool + (long long)layer * g.H * g.seg, (int)kv->b_seq.size(), kv->b_rows,
                        (const bf16 *)k, (const bf16 *)v, k_row, k_head, v_row, v_head, kv->d_err);
    };
    DTTS_CUDA(g.i4 ? (g.D == 128 ? write(kv_write_kernel<true, 128>) : write(kv_write_kernel<true, 64>))
                   : (g.D == 128 ? write(kv_write_kernel<false, 128>) : write(kv_write_kernel<false, 64>)));
    return DTTS_OK;
}

int dtts_kv_read(dtts_kv *kv, int layer, int n_layers, int n, const int *seqs, const int *first, const int *count,
                 void *k, void *v, int dtype) try {
    DTTS_CHECK(kv && (n == 0 || (seqs && first && count)) && n >= 0, DTTS_ERR_ARG, "null argument");
    const KvGeom &g = kv->g;
    DTTS_CHECK(dtype == DTTS_DTYPE_F32 || dtype == DTTS_DTYPE_BF16, DTTS_ERR_UNSUPPORTED, "dtype %d", dtype);
    DTTS_CHECK(layer >= 0 && n_layers >= 1 && layer < g.L && n_layers <= g.L - layer, DTTS_ERR_ARG,
               "layers %d..%d of %d", layer, layer + n_layers - 1, g.L);
    long long rows = 0;
    for (int i = 0; i < n; i++) {
        DTTS_CHECK(seq_ok(kv, seqs[i]), DTTS_ERR_ARG, "sequence %d is not open", seqs[i]);
        const dtts_kv::Seq &s = kv->seqs[seqs[i]];
        DTTS_CHECK(first[i] >= 0 && count[i] >= 0 && (long long)first[i] + count[i] <= s.len, DTTS_ERR_ARG,
                   "rows %d..%lld of sequence %d, which holds %d", first[i], (long long)first[i] + count[i] - 1, seqs[i],
                   s.len);
        if (count[i] && s.hole_lo < s.hole_hi)
            for (int p = first[i] >> g.lgP; p <= (first[i] + count[i] - 1) >> g.lgP; p++)
                DTTS_CHECK(s.pages[p] >= 0, DTTS_ERR_ARG, "rows %d.. of sequence %d were freed by a trim", p * g.P, seqs[i]);
        rows += count[i];
    }
    if (rows == 0) return DTTS_OK;
    DTTS_CHECK(k && v && aligned16(k) && aligned16(v), DTTS_ERR_ARG, "outputs must be on 16-byte boundaries");
    DTTS_CHECK(rows <= INT32_MAX / 2, DTTS_ERR_ARG, "%lld rows in one call", rows);
    DeviceGuard dg(kv->device);
    int st = kv->flush();
    if (st) return st;
    const int per_block = 256 / (g.D / 4) * kReadItems;
    int start = 0;
    auto send = [&](auto &r, int i) -> int {
        constexpr int kMax = std::remove_reference_t<decltype(r)>::kMax;
        r.n = std::min(kMax, n - i);
        r.rows = (int)rows;
        r.n_layers = n_layers;
        for (int j = 0; j < r.n; j++) {
            r.seq[j] = seqs[i + j];
            r.first[j] = first[i + j];
            r.start[j] = start;
            start += count[i + j];
        }
        r.start[r.n] = start;
        const long long items = (long long)(start - r.start[0]) * g.H;
        if (!items) return DTTS_OK;
        const dim3 grid((unsigned)((items + per_block - 1) / per_block), n_layers);
        const uint8_t *pool = kv->pool + (long long)layer * g.H * g.seg;
        const int *table = kv->meta + 5 * g.max_seqs;
        auto read = [&](auto f32, auto b16) {
            return launch_k(kv_pdl(), dtype == DTTS_DTYPE_F32 ? f32 : b16, grid, dim3(256), 0, kv->stream, g, table, pool, r, k, v, kv->d_err);
        };
        DTTS_CUDA(g.i4 ? (g.D == 128 ? read(kv_read_kernel<true, 128, true, kMax>, kv_read_kernel<true, 128, false, kMax>)
                                     : read(kv_read_kernel<true, 64, true, kMax>, kv_read_kernel<true, 64, false, kMax>))
                       : (g.D == 128 ? read(kv_read_kernel<false, 128, true, kMax>, kv_read_kernel<false, 128, false, kMax>)
                                     : read(kv_read_kernel<false, 64, true, kMax>, kv_read_kernel<false, 64, false, kMax>)));
        return DTTS_OK;
    };
    Reads<40> few;
    Reads<320> many;
    for (int i = 0; i < n; i += n <= 40 ? 40 : 320)
        if ((st = n <= 40 ? send(few, i) : send(many, i))) return st;
    return DTTS_OK;
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return DTTS_ERR_OOM;
}

int dtts_kv_attend(dtts_kv *kv, int layer, const dtts_kv_attend_args *a) try {
    DTTS_CHECK(kv && a, DTTS_ERR_ARG, "null argument");
    DTTS_CHECK(layer >= 0 && layer < kv->g.L, DTTS_ERR_ARG, "layer %d of %d", layer, kv->g.L);
    KvAttendPlan p;
    int st = kv->plan_attend(*a, &p);
    if (st) return st;
    DeviceGuard dg(kv->device);
    if ((st = kv->flush())) return st;
    return kv->attend(p, layer);
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return DTTS_ERR_OOM;
}

}  // extern "C"
