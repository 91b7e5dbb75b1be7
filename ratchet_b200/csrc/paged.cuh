// Paged caches of many sequences (rcu_paged): what the kernels of paged_cache.cu, paged_attention.cu and paged_attention_tc.cu share.
#pragma once
#include "common.cuh"

namespace paged {

struct View {
    const void *keys, *values;              // [pages, G, R, D], [pages, G, R, E]
    const int *table, *starts, *lengths;
    float* mass;                            // [S, G, MP * R], nullable
    int S, MP, pages, G, R, shift, D, E;    // R = 1 << shift
    int T;                                  // tokens of the call
    int* status;
};

// A sequence's new tokens [start, start + n) and the L rows it has with them.  What lies outside its tensor is clamped, and reported once
// per call by report_bad: the other readers only have to be safe.
struct Seq {
    int start, n, L;
    __device__ __forceinline__ int old() const { return L - n; }        // row of the first new token (negative only for lengths that are reported)
};

#ifdef __CUDACC__
__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return max(lo, min(v, hi)); }

__device__ __forceinline__ Seq seq_of(const View& p, int s) {
    Seq q;
    q.start = clamp_int(p.starts[s], 0, p.T);
    q.n = clamp_int(p.starts[s + 1], q.start, p.T) - q.start;
    q.L = clamp_int(p.lengths[s], 0, p.MP << p.shift);
    return q;
}
__device__ __forceinline__ bool seq_bad(const View& p, int s) {
    const int a = p.starts[s], b = p.starts[s + 1], L = p.lengths[s];
    return a < 0 || b < a || b > p.T || L < b - a || L > (p.MP << p.shift);
}
__device__ __forceinline__ void report_bad(int* status) { atomicOr(status, RCU_DEVFLAG_BOUNDS); }

// The sequence that token t belongs to, -1 for a token of none; all lanes of a warp ask for the same token.  32 starts are looked at per step.
__device__ __forceinline__ int seq_of_token(const View& p, int t) {
    int lo = 0, hi = p.S;                   // the last s with starts[s] <= t lies in [lo, hi], if there is one
    while (hi > lo) {
        const int step = (hi - lo + 31) / 32, at = lo + ((int)(threadIdx.x & 31) + 1) * step;
        const int k = __popc(__ballot_sync(0xffffffffu, at <= hi && p.starts[min(at, hi)] <= t));
        hi = min(hi, lo + (k + 1) * step - 1);
        lo += k * step;
    }
    return lo < p.S && p.starts[lo] <= t && t < p.starts[lo + 1] ? lo : -1;
}

// Page that holds row r of sequence s; an id outside the pool is reported and becomes page 0.
__device__ __forceinline__ int page_of(const View& p, int s, int r) {
    const int id = p.table[(size_t)s * p.MP + (r >> p.shift)];
    if ((unsigned)id < (unsigned)p.pages) return id;
    report_bad(p.status);
    return 0;
}
// first element of row r (of its page) of kv head g, rows of `width` elements
__device__ __forceinline__ size_t row_at(const View& p, int page, int g, int r, int width) {
    return (((size_t)page * p.G + g) * p.R + (r & (p.R - 1))) * (size_t)width;
}
#endif

// rcu_paged as the kernels take it; checks what every call needs.  tokens: of the call; starts: whether they are read
rcu_status view(rcu_device* dev, const char* op, const rcu_paged* c, uint64_t tokens, bool starts, View* out);

// Device memory of a call: the caller's, or the pool's for the length of the call (never while the stream is being captured, since a
// replay would find the block with other owners).
struct Scratch {
    Scratch(const Scratch&) = delete;
    Scratch& operator=(const Scratch&) = delete;
    rcu_device* dev;
    void* ptr = nullptr;
    bool pooled = false;
    explicit Scratch(rcu_device* d) : dev(d) {}
    ~Scratch() {
        if (pooled) rcu_free(dev, ptr);          // the pool reuses blocks in stream order
    }
    rcu_status take(const char* op, const rcu_tensor* given, uint64_t bytes);
};

}  // namespace paged
