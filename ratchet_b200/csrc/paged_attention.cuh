// What the kernels of attention over paged caches share (paged_attention.cu, paged_attention_tc.cu): arguments, which rows a token sees, how
// the work is cut, and the form of partial results.
#pragma once
#include "paged.cuh"

namespace paged {

constexpr float kLog2e = 1.4426950408889634f;

struct AttendArgs {
    View p;
    const void* q;             // [T, H, D]
    void* out;                 // [T, H * E]
    const float* sink;         // [H], nullable
    float* lse;                // [T, H] in units of log 2; where mass is kept
    int H, window, first;
    float c;                   // scale log2 e
};

#ifdef __CUDACC__
// rows that the token at row r sees: [0, head) and [low, r + 1)
__device__ __forceinline__ void visible(int window, int first, int r, int& head, int& low) {
    low = window > 0 && r >= window ? r - window + 1 : 0;
    head = min(first, low);
}
#endif

// ------------------------------------------------------------------------------------------------ how the work is cut
// An item is up to `tokens` consecutive new tokens of one sequence, with all heads of a group, over the tiles of kTileK rows that any of them
// sees; an item exists once per kv head.  All items' tiles in a row, kv head by kv head, are cut into equal runs, one per CTA: a CTA takes
// the end of one item, some whole ones and the beginning of another, whatever the lengths are.  Items that one CTA covers are finished by it,
// the others' parts are joined by merge_kernel.  plan_kernel works this out on the device, where the lengths are.
constexpr int kTileK = 128;

struct Item {
    int s, token, count, row;  // sequence; its first token of the item (in rows: first row of queries), how many; row of the first one
};
struct Plan {
    int items;                 // upper bound: T / tokens + S
    int tokens;                // of an item
    int ctas, least;           // CTAs at most; tiles that a CTA takes at least
    int extra;                 // see Walk
    int stride;                // rows of a part in scratch
    // scratch
    int* head;                 // [0] length of a kv head, [1] CTAs at work
    int* prefix;               // [items + 1]: where each item of a kv head begins
    Item* item;                // [items]
    float2* ml;                // [2 * ctas, stride]: a part's maximum and sum, per row
    float4* o;                 // [2 * ctas, E / 4, stride]: its weighted sum of values
};

#ifdef __CUDACC__
// Tiles that tokens at rows r0 .. r1 see: the first `head` ones, then lo, lo + 1, ..
struct Span {
    int head, lo, count;
    __device__ __forceinline__ int tile(int n) const { return n < head ? n : lo + n - head; }
};
__device__ __forceinline__ Span span_of(int window, int first, int r0, int r1) {
    Span sp;
    const int hi = r1 / kTileK + 1, low0 = window > 0 ? max(0, r0 - window + 1) : 0, low1 = window > 0 ? max(0, r1 - window + 1) : 0;
    sp.lo = low0 / kTileK;
    sp.head = (min(first, low1) + kTileK - 1) / kTileK;
    if (sp.head >= sp.lo) sp.head = sp.lo = 0;
    sp.count = r1 < 0 ? 0 : sp.head + hi - sp.lo;
    return sp;
}

// A call's items and where they begin, into pl.head, pl.prefix and pl.item, by a CTA of THREADS threads.  One thread per item; `starts` (nullable) has room
// for the sequences' starts in shared memory, where looking for an item's sequence takes no time.
template <int THREADS>
__device__ __forceinline__ void plan_items_block(const View& p, const Plan& pl, int window, int first, int group, int* starts) {
    __shared__ int warps[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (starts) {
        for (int s = tid; s < p.S; s += THREADS) starts[s] = clamp_int(p.starts[s], 0, p.T);
        __syncthreads();
    }
    int before = 0;
#pragma unroll 1
    for (int base = 0; base < pl.items; base += THREADS) {
        const int i = base + tid;
        Item it{-1, 0, 0, 0};
        int w = 0;
        if (i < pl.items) {
            // sequence s has the items from starts[s] group / tokens + s on
            auto begins = [&](int s) { return (int)((long long)(starts ? starts[s] : clamp_int(p.starts[s], 0, p.T)) * group / pl.tokens) + s; };
            int lo = 0, hi = p.S - 1;
#pragma unroll 1
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (begins(mid) <= i) lo = mid;
                else hi = mid - 1;
            }
            const Seq q = seq_of(p, lo);
            const long long at = (long long)(i - begins(lo)) * pl.tokens;
            if (at >= 0 && at < (long long)q.n * group) {
                it = Item{lo, (int)at, (int)min((long long)pl.tokens, (long long)q.n * group - at), q.old() + (int)at / group};
                w = span_of(window, first, it.row, min(q.old() + ((int)at + it.count - 1) / group, q.L - 1)).count;
                w += w > 0 ? pl.extra : 0;
            }
            pl.item[i] = it;
        }
        int upto = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) warps[warp] = upto;
        __syncthreads();
        int add = before, all = 0;
#pragma unroll 4
        for (int j = 0; j < THREADS / 32; ++j) {
            if (j < warp) add += warps[j];
            all += warps[j];
        }
        if (i < pl.items) pl.prefix[i] = add + upto - w;
        before += all;
        __syncthreads();
    }
    if (tid == 0) {
        pl.prefix[pl.items] = before;
        pl.head[0] = before;
        const long long total = (long long)before * p.G;
        pl.head[1] = (int)max(1ll, min((long long)pl.ctas, (total + pl.least - 1) / pl.least));
    }
    __syncthreads();
}

// The tiles that CTA b of C takes of `total`
__device__ __forceinline__ int first_tile(long long total, int b, int C) { return (int)(total * b / C); }

// The item at place y of a kv head's row, by whole warps: 32 places are looked at per step
__device__ __forceinline__ int item_at(const Plan& pl, int items, int y) {
    int lo = 0, hi = items - 1;                  // the last item that begins there or before
#pragma unroll 1
    while (hi > lo) {
        const int step = (hi - lo + 31) / 32, at = lo + ((int)(threadIdx.x & 31) + 1) * step;
        const int k = __popc(__ballot_sync(0xffffffffu, at <= hi && pl.prefix[min(at, hi)] <= y));
        hi = min(hi, lo + (k + 1) * step - 1);
        lo += k * step;
    }
    return lo;
}

// A CTA's walk over its run: item by item.  An item's place in the row of all is as long as its tiles and `extra` more, which stand for what beginning
// and ending it costs: nothing is done in these.
struct Walk {
    const Plan& pl;
    int items, W, at, end;     // items, length of a kv head; run
    int g, i;                  // kv head and item at `at`
    Item it;
    int n0, n1, whole;         // tiles [n0, n1) of the item, not empty; whether these are all of them
    __device__ __forceinline__ Walk(const Plan& plan, int b, int G, int count) : pl(plan), items(count) {
        W = plan.head[0];
        const int C = plan.head[1];
        const long long total = (long long)W * G;
        at = b < C ? first_tile(total, b, C) : 0;
        end = b < C ? first_tile(total, b + 1, C) : 0;
        if (at >= end) return;
        find();
        if (n0 >= n1) next();
    }
    // the item at place `at`, and what of it lies before `end`
    __device__ __forceinline__ void find() {
        g = at / W;
        i = item_at(pl, items, at - g * W);
        load();
    }
    __device__ __forceinline__ void load() {
        it = pl.item[i];
        const int p0 = g * W + pl.prefix[i] + pl.extra, p1 = g * W + pl.prefix[i + 1];
        n0 = max(0, at - p0);
        n1 = min(end, p1) - p0;
        whole = n0 == 0 && p0 + n1 == p1;
    }
    __device__ __forceinline__ bool more() const { return at < end; }
    // a CTA has one part that goes on with an item at most, and one that begins an item and does not end it
    __device__ __forceinline__ int slot(int b) const { return 2 * b + (n0 == 0); }
    __device__ __forceinline__ void next() {
        do {
            at = g * W + pl.prefix[i + 1];
            if (at >= end) return;
            if (at >= (g + 1) * W) {
                ++g;
                i = -1;
            }
            do ++i;
            while (pl.prefix[i + 1] == pl.prefix[i]);       // ends: at < end <= W G, so a later item has a place
            load();
        } while (n0 >= n1);
    }
};

// The parts that have to be joined at the boundary between CTAs b and b + 1: `count` of them, the first in slot 2 b + 1, the others in slots
// 2 (b + 1), 2 (b + 2), ..; none where the boundary cuts no item's tiles, or an earlier one has cut the same item
struct Join {
    int count;
    int g;
    Item it;
    __device__ __forceinline__ Join(const Plan& pl, int b, int G, int items) : count(0) {
        const int W = pl.head[0], C = pl.head[1];
        if (b + 1 >= C) return;
        const long long total = (long long)W * G;
        const int before = first_tile(total, b, C), cut = first_tile(total, b + 1, C);
        if (cut >= total) return;
        g = cut / W;
        const int i = item_at(pl, items, cut - g * W), p0 = g * W + pl.prefix[i] + pl.extra, p1 = g * W + pl.prefix[i + 1];
        if (cut <= p0 || before > p0) return;
        it = pl.item[i];
        count = (int)min((long long)C, ((long long)p1 * C + total - 1) / total) - b;          // CTAs from b on that begin before p1
    }
    __device__ __forceinline__ int slot(int b, int k) const { return k == 0 ? 2 * b + 1 : 2 * (b + k); }
};
#endif

// Any type, width and alignment (paged_attention.cu); f16 and bf16 up to 128 features on the tensor cores (paged_attention_tc.cu)
bool attend_tc_takes(const rcu_device* dev, const View& p, int H, int dt);
// few rows per sequence, and f32 (paged_attention_rows.cu): sums the weights where mass is kept
bool attend_rows_takes(const rcu_device* dev, const View& p, int H, int dt);
uint64_t attend_rows_scratch(const rcu_device* dev, const View& p, int H, int dt);
rcu_status attend_rows(rcu_device* dev, const AttendArgs& a, int dt, void* scratch);
// launches plan_kernel: items of `plan.tokens` tokens, or of that many rows of queries where `group` of them make a token
rcu_status plan_items(rcu_device* dev, const View& p, const Plan& plan, int window, int first, int group);
uint64_t attend_tc_scratch(const rcu_device* dev, const View& p, int H);
rcu_status attend_tc(rcu_device* dev, const AttendArgs& a, int dt, void* scratch);
// the weights that every row receives, added to its mass; after the attention, whose lse it reads (paged_mass_tc.cu)
uint64_t mass_tc_scratch(const rcu_device* dev, const View& p, int H);
rcu_status mass_tc(rcu_device* dev, const AttendArgs& a, int dt, void* scratch);

}  // namespace paged
