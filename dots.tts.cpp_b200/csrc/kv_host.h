// The paged K/V cache object (dtts_kv): host-side page tables, the current
// batch and the device buffers; shared by its entry points (kv_cache.cu) and the
// LLM engine that runs on it (llm_engine.cu).
#pragma once
#include <queue>
#include <functional>
#include <vector>

#include "kv.cuh"
#include "runtime.h"

namespace dtts {
// Launches of one attention call on the current batch; the same for every layer.
struct KvAttendPlan {
    KvAttendArgs args[2];       // sequences of few rows, of many rows
    int rows_or_pairs[2];       // 0: no such sequence
};
}  // namespace dtts

struct dtts_kv {
    struct Seq {
        bool open = false;
        int len = 0, pos = 0;             // rows held; position of the next token
        int hole_lo = 0, hole_hi = 0;     // pages [hole_lo, hole_hi) were freed by a trim
        std::vector<int> pages;           // -1: freed
    };
    int device = 0, num_sms = 148;
    dtts::KvGeom g{};
    dtts::KvShapes shapes{};
    long long max_tokens = 0;
    cudaStream_t own_stream = nullptr, stream = nullptr;
    cudaEvent_t handoff = nullptr;
    dtts::DeviceArena mem;
    uint8_t *pool = nullptr;
    int *meta = nullptr, *keep = nullptr, *cnt = nullptr, *d_err = nullptr;
    float *ws = nullptr;
    std::vector<int> meta_h;              // what `meta` holds once the enqueued updates have run
    std::vector<int> pokes;               // indexes of meta_h whose values are not on the device yet
    std::vector<Seq> seqs;
    std::vector<int> refs;                // users of each page
    std::priority_queue<int, std::vector<int>, std::greater<int>> free_pages;   // lowest first
    // current batch
    std::vector<int> b_seq, b_cnt, b_len;
    int b_rows = 0;
    int last_entries = 0;                 // of the current or, where that has ended, the last batch
    long long uid = 0;                    // no two caches of a process share it

    ~dtts_kv();
    dtts::KvMeta kv_meta() const;
    int table_at(int seq, int page) const { return 5 * g.max_seqs + seq * g.max_pages + page; }
    void poke(int index, int value) {
        if (meta_h[index] == value) return;
        meta_h[index] = value;
        pokes.push_back(index);
    }
    template <typename P>
    void take_pokes(P &p, size_t i) const;
    int flush();                          // enqueues the pending metadata updates
    struct Copy {
        int src, dst, rows;               // pages, rows in use
    };
    int send_growth(const std::vector<Copy> &copies);
    int take_page() {
        const int p = free_pages.top();
        free_pages.pop();
        refs[p] = 1;
        return p;
    }
    void drop_page(int p) {
        if (p >= 0 && --refs[p] == 0) free_pages.push(p);
    }
    void drop_batch();
    int not_capturing(const char *what) const;
    int check_batch(int n_seq, const int *sq, const int *n_new) const;
    // What the last extend() changed of a sequence: its state before, and the shared last page that a copy replaced
    struct Growth {
        int seq, len, pos, pages, tail;   // tail: -1 where none was replaced
    };
    std::vector<Growth> grown;
    // Whether extend() would find everything it needs; *pages: how many it takes. Changes nothing.
    int fits(int n_seq, const int *sq, const int *n_new, long long *pages);
    int extend(int n_seq, const int *sq, const int *n_new);
    void take_back();                     // undoes the last extend(), before any other change; the batch ends
    // Whether attention of n_new[b] further tokens would reach rows that a trim freed.
    int check_window(int n_seq, const int *sq, const int *n_new, int window, int sinks) const;
    int max_splits(int n_seq) const;      // of the few-row kernel, for the workspace
    // Checks the arguments against the current batch and sizes the launches.
    int plan_attend(const dtts_kv_attend_args &a, dtts::KvAttendPlan *p) const;
    int attend(const dtts::KvAttendPlan &p, int layer);
};
