// The paged K/V cache object (dtts_kv): host-side page tables, the current
// batch and the device buffers; shared by its entry points (kv_cache.cu) and the
// LLM engine that runs on it (llm_engine.cu).
#pragma once
#include <queue>
#include <functional>
#include <vector>

#include "kv.cuh"
#include "runtime.h"

struct dtts_kv {
    struct Seq {
        bool open = false;
        int len = 0, pos = 0;             // rows held; position of the next token
        int hole_lo = 0, hole_hi = 0;     // pages [hole_lo, hole_hi) were freed by a trim
        std::vector<int> pages;           // -1: freed
    };
    int device = 0, num_sms = 148;
    dtts::KvGeom g{};
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
    long long b_id = 0;                   // changes with the batch and with anything that moves its rows

    ~dtts_kv();
    dtts::KvMeta kv_meta() const;
    int table_at(int seq, int page) const { return 5 * g.max_seqs + seq * g.max_pages + page; }
    void poke(int index, int value) {
        if (meta_h[index] == value) return;
        meta_h[index] = value;
        pokes.push_back(index);
    }
    int flush();                          // enqueues the pending metadata updates
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
    int extend(int n_seq, const int *sq, const int *n_new);
};
