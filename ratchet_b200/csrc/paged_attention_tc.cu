// Attention of new tokens over paged caches on the 5th-generation tensor cores (tcgen05): f16 and bf16, heads of up to 128 features.
//
// A tile of queries is 128 / group tokens with all query heads of a kv head, so that keys and values are read once for the group.  CTA = two
// such tiles that take turns: while the softmax warps of one work, the tensor core runs the other's products.
//   warp 0              brings the queries, then keys and values of 128 rows in turns into a ring, page by page (a box per page or part of one;
//                       rows of no page stay as they are in shared memory);
//   warp 1              per tile n and query tile w: O_w += P_w V of tile n - 1, with P_w read from tensor memory, then S_w = Q_w K^T of tile n,
//                       which takes P_w's place;
//   warps 4-7, 8-11     softmax of query tile 0 / 1, a query per thread: scores from tensor
//                       memory, mask, running maximum, weights back over the scores, half a tile of rows at a time: the scores of one half are there
//                       while the weights of the other are worked out.  The maximum that weights are taken against only moves when a score exceeds
//                       it by more than 2^8, so that O_w is rescaled rarely.
// An item of one query tile (generation) gives it to both groups, which take the tiles of rows in turns and join their sums at the end.
// Weights enter the second product in the operands' type, which the matrix instructions want: each is off by half a step of itself at most, the output by half a
// step of sum p |v| (paged_tc.cuh has how f16 weights keep out of the type's small numbers).  Their sum, the maximum and O are f32.
// What is masked must not reach the sum even where it is not finite, and 0 times infinity is NaN.  Rows behind the sequence's last one are zeroed in
// shared memory.  In a tile that some of the queries see in part, an infinity or NaN among the values sends the query tile to attend_rows, which
// reads only what each query sees.
// Every wait is bounded; one that gives up raises RCU_DEVFLAG_TIMEOUT and ends all others of the CTA.
// Bound by the softmax warps' chains (two of them a scheduler): 4096 tokens into an empty cache, 32 heads over 8 of 128 features, bf16: 196 us (700 TFLOP/s; 189 in passes
// right behind one another; tensor pipe 40 %, exponentials 30 %, issue slots 44 %); 777 tokens over 20000 rows, 80 features, f16: 288 us.  Two threads a query had taken
// 229 us for 184 and 365 for 283: what they have to tell each other costs more than the shorter chains gain.  A whole warp keeping step with the issuing lane 291 for 283.
#include <cuda.h>

#include "paged_attention.cuh"
#include "paged_rows.cuh"
#include "paged_tc.cuh"

namespace paged {
namespace {

constexpr int kThreadsP = 384, kMostStages = 8;
// A group's notes that a segment has values which are not finite, by the segment's number.  A warp that has passed segment i's meeting may note something
// of segment i + 1 before a slower one has read what was noted of i, hence not one.  Note i is cleared behind the meeting of i + 1, to which every
// warp of the group comes with i read; it is next written in segment i + kNotes, and with two notes a warp of that segment could write before a slower
// one, just past the meeting of i + 1, clears.  With three the meeting of i + 2 lies between.
constexpr int kNotes = 3;

__global__ void __launch_bounds__(1024) plan_kernel(const __grid_constant__ View p, const __grid_constant__ Plan pl, int window, int first, int group) {
    rcu_kernel_entry();
    __shared__ int starts[2048];
    for (int s = threadIdx.x; s < p.S; s += 1024)
        if (seq_bad(p, s)) report_bad(p.status);
    plan_items_block<1024>(p, pl, window, first, group, p.S <= 2048 ? starts : nullptr);
}

struct TcArgs {
    AttendArgs a;
    Plan pl;
    int group, tq;             // query heads of a kv head; tokens of a query tile
    int stages, nb, eb, stage_bytes;
};

// Which tiles of an item's span (by their place in it) some query at rows t0 .. t1 sees
struct Sight {
    int head, a, b;
    __device__ __forceinline__ bool operator()(int n) const { return n < head || (n >= a && n < b); }
};
__device__ __forceinline__ Sight sight_of(int window, int first, const Span& sp, int t0, int t1) {
    Sight v{0, 0, 0};
    if (t1 < t0 || t1 < 0) return v;
    const int low = window > 0 ? max(0, t0 - window + 1) : 0;
    v.head = window > 0 ? (sp.head > 0 ? sp.head : (min(first, t1 + 1) + kTileK - 1) / kTileK) : 0;
    v.a = max(low / kTileK - sp.lo, 0) + sp.head;
    v.b = t1 / kTileK + 1 - sp.lo + sp.head;
    return v;
}

// A CTA's share of an item, as one warp works it out for the others
struct alignas(16) Segment {
    Item it;
    int g, n0, n1, slot;
    int whole, more, L, two;             // more 0: the run has ended; two: the item has a second query tile
    Span sp;
    Sight see[2];
    int pad[3];
    // An item of two query tiles: group w has tile w.  Of one: both groups have it, the tiles of rows in turns.
    __device__ __forceinline__ bool has(int w, int n) const { return see[w](n) && (two || ((n - n0) & 1) == w); }
};
constexpr int kSegments = 4;

// A query tile whose values are not all finite, row by row
template <class T>
__device__ __noinline__ void redo_rows(const TcArgs& x, const Segment& seg, int w, int quarter) {
    const int tile0 = seg.two ? w * x.tq : 0;
#pragma unroll 1
    for (int i = 0; i < 32; ++i) {
        const int r = quarter * 32 + i, t = tile0 + r / x.group, h = seg.g * x.group + r % x.group;
        if (r >= x.tq * x.group || t >= seg.it.count) continue;
        RowPart part;
        attend_row<T>(x.a, seg.it.s, seg.g, seg.it.token + t, h, seg.it.row + t, seg.sp, seg.n0, seg.n1, part);
        if (seg.whole) finish_row<T>(x.a, seg.it.token + t, h, part);
        else store_part(x.pl, x.a.p.E, seg.slot, (seg.two ? w : 0) * kTileQ + r, part);
    }
}

template <class T>
__global__ void __launch_bounds__(kThreadsP, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                const __grid_constant__ TcArgs x) {
    extern __shared__ unsigned char smem_dyn[];
    const AttendArgs& a = x.a;
    const View& p = a.p;
    unsigned char* qs = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    unsigned char* ring = qs + 2 * x.nb * kBlock;
    // [query tile][half of a tile of rows]
    __shared__ __align__(8) uint64_t q_full, q_empty, full[kMostStages], empty[kMostStages], s_full[2][2], p_full[2][2], pv_done[2], o_full[2], met[2], joined, taken, drained,
        seg_full[kSegments], seg_empty[kSegments];
    __shared__ Segment segments[kSegments];
    __shared__ float2 other[kTileQ];                  // maximum and sum that the second group hands to the first
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag, poison[2][kNotes];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 1);
        mbar_init(&joined, 8);
        mbar_init(&taken, 4);
        mbar_init(&drained, 1);
#pragma unroll 1
        for (int i = 0; i < x.stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
#pragma unroll 1
        for (int i = 0; i < kSegments; ++i) {
            mbar_init(&seg_full[i], 1);
            mbar_init(&seg_empty[i], 10);
        }
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i][0], 1);
            mbar_init(&s_full[i][1], 1);
            mbar_init(&p_full[i][0], 4);
            mbar_init(&p_full[i][1], 4);
            mbar_init(&pv_done[i], 1);
            mbar_init(&o_full[i], 1);
            mbar_init(&met[i], 4);
            for (int k = 0; k < kNotes; ++k) poison[i][k] = 0;
        }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    rcu_kernel_entry_wait_only();        // nothing before this touches global memory
    const uint32_t tmem = tmem_slot;       // S_w (then P_w) at 128 w, O_w at 256 + 128 w

    auto wait = [&](uint64_t* bar, int phase) { return wait_warp(bar, phase, &abort_flag, p.status); };
    // The i-th segment; false where the run has ended, or a wait gave up (ok)
    auto take = [&](int i, bool& ok) -> const Segment& {
        ok = wait(&seg_full[i % kSegments], i / kSegments);
        return segments[i % kSegments];
    };
    auto release = [&](int i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[i % kSegments]);
    };

    if (warp == 2) {
        Walk wk(x.pl, blockIdx.x, p.G, x.pl.items);
        bool ok = true;
#pragma unroll 1
        for (int i = 0; ok; ++i) {
            ok = wait(&seg_empty[i % kSegments], (i / kSegments) ^ 1);
            if (!ok) break;
            const bool more = wk.more();
            Segment& seg = segments[i % kSegments];
            if (lane == 0) {
                seg.more = more;
                if (more) {
                    const Span sp = span_of(a.window, a.first, wk.it.row, wk.it.row + wk.it.count - 1);
                    const bool two = wk.it.count > x.tq;
                    seg.it = wk.it;
                    seg.it.token += clamp_int(p.starts[wk.it.s], 0, p.T);
                    seg.g = wk.g;
                    seg.n0 = wk.n0;
                    seg.n1 = wk.n1;
                    seg.slot = wk.slot(blockIdx.x);
                    seg.whole = wk.whole;
                    seg.L = clamp_int(p.lengths[wk.it.s], 0, p.MP << p.shift);
                    seg.two = two;
                    seg.sp = sp;
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const int t0 = wk.it.row + (two ? w * x.tq : 0);
                        seg.see[w] = sight_of(a.window, a.first, sp, t0, min(t0 + x.tq, wk.it.row + wk.it.count) - 1);
                    }
                }
                mbar_arrive(&seg_full[i % kSegments]);
            }
            __syncwarp();
            if (!more) break;
            wk.next();
        }
    } else if (warp == 0) {
        const int rows_box = min(p.R, kTileK), boxes = kTileK / rows_box;
        const bool mine_k = lane < boxes * x.nb, mine_v = lane < boxes * x.eb;
        const int box = lane % boxes, col = lane / boxes;
        int fills = 0, i = 0;
        RingAt at{x.stages, 0, 0};
        bool ok = true;
#pragma unroll 1
        for (;; ++i) {
            const Segment& seg = take(i, ok);
            if (!ok || !seg.more) break;
            ok = wait(&q_empty, i ^ 1);
            if (!ok) break;
            if (lane == 0) {
                const int tiles = seg.two ? 2 : 1;
                mbar_expect_tx(&q_full, tiles * x.nb * x.group * x.tq * 128);
#pragma unroll 1
                for (int w = 0; w < tiles * x.nb; ++w)
                    tma_load_4d(qs + w * kBlock, &qmap, w % x.nb * 64, 0, seg.g, seg.it.token + w / x.nb * x.tq, &q_full);
            }
            __syncwarp();
            PageIds ids;
            const int L = seg.L, have = min(p.MP, (L + p.R - 1) >> p.shift), s_id = seg.it.s, g = seg.g, n1 = seg.n1;
            const Span sp = seg.sp;
#pragma unroll 1
            for (int n = seg.n0; n < n1 && ok; ++n) {
                const int j0 = sp.tile(n) * kTileK, i0 = j0 >> p.shift, row0 = j0 & (p.R - 1);
                const bool in = j0 + box * rows_box < L;               // boxes behind the last row are left out
                const int page = ids.of(p, s_id, i0, i0 + box, i0 + boxes - 1, have);
                const int pages = min(boxes, (L - j0 + rows_box - 1) / rows_box);
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv) {
                    ok = wait(&empty[at.s], at.phase ^ 1);
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&full[at.s], pages * (kv ? x.eb : x.nb) * rows_box * 128);
                    __syncwarp();
                    if ((kv ? mine_v : mine_k) && in)
                        tma_load_4d(ring + (size_t)at.s * x.stage_bytes + col * kBlock + box * rows_box * 128, kv ? &vmap : &kmap, col * 64, row0, g, page, &full[at.s]);
                    at.go(1);
                    ++fills;
                }
            }
            if (!ok) break;
            release(i);
        }
        if (!ok) {          // given up: let the copies in flight land before the memory is somebody else's
#pragma unroll 1
            for (int k = max(0, fills - x.stages); k < fills; ++k) land(&full[k % x.stages], k / x.stages);
            land(&q_full, i);
        }
    } else if (warp == 1) {
        // one lane: what it does between two products, tensor memory waits for
        if (elect_one()) {
            constexpr bool bf16 = !std::is_same<T, __half>::value;
            const uint32_t idesc_s = umma_idesc_f16(kTileQ, kTileK / 2, bf16);
            const uint32_t idesc_o = umma_idesc_f16(kTileQ, (p.E + 15) & ~15, bf16) | (1u << 16);     // V is stored with its columns contiguous
            const int ksteps = (p.D + 15) / 16, stage16 = x.stage_bytes >> 4;
            const uint64_t qd = umma_desc_sw128(qs), kd = umma_desc_sw128(ring), vd = umma_desc_sw128_mn(ring, kBlock);
            auto wait1 = [&](uint64_t* bar, int phase) { return gemvq8::mbar_try_wait(bar, phase & 1) || wait_on(bar, phase & 1, &abort_flag, p.status); };
            bool ok = true;
            int weights0 = 0, weights1 = 0;                // hand-overs of P_w so far
            RingAt kat{x.stages, 0, 0}, vat{x.stages, 1, 0};
#pragma unroll 1
            for (int i = 0;; ++i) {
                ok = wait1(&seg_full[i % kSegments], i / kSegments);
                const Segment seg = segments[i % kSegments];
                if (!ok || !seg.more) break;
                mbar_arrive(&seg_empty[i % kSegments]);
                bool any0 = false, any1 = false, v0 = false, v1 = false;
                ok = wait1(&q_full, i);
                // Half a tile of rows at a time, two halves in flight: while the weights of one are worked out, the scores of the other are there.
                // At place n the products with V of tile n - 1, and the scores of tile n, half by half, in the same columns.
#pragma unroll 1
                for (int n = seg.n0; n <= seg.n1 && ok; ++n) {
                    const bool first = n == seg.n0, last = n == seg.n1;
                    const uint64_t kb = kd + (uint64_t)(kat.s * stage16), vb = vd + (uint64_t)(vat.s * stage16);
                    const bool s0 = !last && seg.has(0, n), s1 = !last && seg.has(1, n);
                    auto scores = [&](auto w, int half) {
                        tc_fence_after();
                        const uint64_t qa = qd + (uint64_t)((seg.two ? w() : 0) * x.nb * (kBlock >> 4)), ka = kb + 512 * half;
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (k < ksteps)
                                umma_f16(tmem + 128 * w + 64 * half, qa + (k >> 2) * (kBlock >> 4) + 2 * (k & 3), ka + (k >> 2) * (kBlock >> 4) + 2 * (k & 3), idesc_s, k > 0 ? 1u : 0u);
                        umma_commit(&s_full[w][half]);
                    };
                    auto values = [&](auto w, int half, int weights, bool more) {
                        ok = wait1(&p_full[w][half], weights);
                        if (!ok) return;
                        tc_fence_after();
#pragma unroll
                        for (int k = 0; k < 4; ++k)      // 16 rows are two 1024-byte groups of V, eight columns of P
                            umma_f16_ta(tmem + 256 + 128 * w, tmem + 128 * w + 64 * half + 8 * k, vb + 512 * half + 128 * k, idesc_o, k > 0 || more ? 1u : 0u);
                        umma_commit(&pv_done[w]);
                    };
                    using W0 = std::integral_constant<int, 0>;
                    using W1 = std::integral_constant<int, 1>;
                    if (!last) ok = wait1(&full[kat.s], kat.phase);
                    if (!ok) break;
                    // in turns, the two groups' tiles are different ones: the scores of one need not wait for the weights of the other
                    if (!seg.two) {
#pragma unroll 1
                        for (int half = 0; half < 2; ++half) {
                            if (s0) scores(W0{}, half);
                            if (s1) scores(W1{}, half);
                        }
                    }
                    if (!first) ok = wait1(&full[vat.s], vat.phase);
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        if (ok && v0) values(W0{}, half, weights0, any0 || half);
                        if (ok && seg.two && s0) scores(W0{}, half);
                        if (ok && v1) values(W1{}, half, weights1, any1 || half);
                        if (ok && seg.two && s1) scores(W1{}, half);
                    }
                    if (!ok) break;
                    weights0 += v0;
                    weights1 += v1;
                    any0 |= v0;
                    any1 |= v1;
                    v0 = s0;
                    v1 = s1;
                    if (!last) umma_commit(&empty[kat.s]);
                    if (n == seg.n1 - 1) umma_commit(&q_empty);
                    if (!first) umma_commit(&empty[vat.s]);
                    if (last && any0) umma_commit(&o_full[0]);
                    if (last && any1) umma_commit(&o_full[1]);
                    if (!last) kat.go(2);
                    if (!first) vat.go(2);
                }
                if (!ok) break;
            }
            if (!ok) {            // given up: let the products in flight end before tensor memory is freed
                umma_commit(&drained);
#pragma unroll 1
                for (int k = 0; k < 16; ++k) land(&drained, 0);
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int w = warp < 8 ? 0 : 1, quarter = warp & 3;
        const int r = quarter * 32 + lane;                                   // row of the query tile
        const int own = r / x.group, head = r - own * x.group;               // token of the tile, query head of the group
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16, ts = tmem + 128 * w + lanes, to = tmem + 256 + 128 * w + lanes;
        const int ocols = (p.E + 31) & ~31;
        uint4* turn = reinterpret_cast<uint4*>(ring + (size_t)x.stages * x.stage_bytes) + (warp - 4) * 128;      // 32 rows of 64 bytes, the warp's own
        int tiles = 0, products = 0, outs = 0, meets = 0, joins = 0;      // tiles and halves of them so far
        RingAt vat{x.stages, 1, 0};
        bool ok = true;
        // places of the output that this lane writes once rows are turned around: token of the tile, elements from its first row on
        int turn_token[4], turn_at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int u = quarter * 32 + 8 * k + (lane >> 2);
            turn_token[k] = u < x.tq * x.group ? u / x.group : 1 << 20;
            turn_at[k] = (u / x.group * a.H + u % x.group) * p.E + 8 * (lane & 3);
        }
#pragma unroll 1
        for (int i = 0;; ++i) {
            const Segment& seg = take(i, ok);
            if (!ok || !seg.more) break;
            const int note = i % kNotes;
            const bool two = seg.two;
            const Item it = seg.it;
            const Sight see = seg.see[w];            // copies: what is in shared memory is read again behind every wait
            const Span sp = seg.sp;
            const int tile0 = two ? w * x.tq : 0, token = tile0 + own, L = seg.L, n0 = seg.n0, n1 = seg.n1;
            const bool valid = r < x.tq * x.group && token < it.count;
            const int row = it.row + token;
            const bool live = __any_sync(0xffffffffu, valid);               // warps without a query only keep step
            // rows of the tile's and of the warp's first and last query
            const int t0 = it.row + tile0, t1 = min(t0 + x.tq, it.row + it.count) - 1;
            const int w0 = __reduce_min_sync(0xffffffffu, valid ? row : 0x7fffffff), w1 = __reduce_max_sync(0xffffffffu, valid ? row : -1);
            float m = valid ? -INFINITY : INFINITY, l = 0.f;                // a row of no query never moves the maximum
            bool any = false;
#pragma unroll 1
            for (int n = n0; n < n1; ++n, vat.go(2)) {
                if (!see(n) || (!two && ((n - n0) & 1) != w)) continue;
                const int j0 = sp.tile(n) * kTileK;
                // a tile that is not whole to all queries: rows behind the last one become zero, values that are not finite are noted
                if (j0 + kTileK - 1 > t0 || (a.window > 0 && j0 <= t1 - a.window && j0 + kTileK > a.first)) {
                    ok = wait(&full[vat.s], vat.phase);
                    if (!ok) break;
                    unsigned char* v = ring + (size_t)vat.s * x.stage_bytes + r * 128;
                    const bool behind = j0 + r >= L;
                    uint32_t bad = 0;
#pragma unroll 4
                    for (int c = 0; c < 8 * x.eb; ++c) {
                        uint4* at = reinterpret_cast<uint4*>(v + (c >> 3) * kBlock + (((c ^ lane) & 7) << 4));
                        const uint4 u = *at;
                        if (behind) *at = make_uint4(0, 0, 0, 0);
                        else bad |= not_finite<T>(u.x) | not_finite<T>(u.y) | not_finite<T>(u.z) | not_finite<T>(u.w);
                    }
                    if (bad) poison[w][note] = 1;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    ok = wait(&s_full[w][half], tiles);
                    if (!ok) break;
                    tc_fence_after();
                    if (live) {
                        const int j1 = j0 + 64 * half;
                        float s[64];
                        tmem_ld_32x64(ts + 64 * half, s);
                        if (j1 + 63 > w0 || (a.window > 0 && j1 <= w1 - a.window && j1 + 64 > a.first)) {
                            asm volatile("" ::: "memory");          // a branch, not 64 predicated selections in every tile
                            const int hi = row - j1, lo = a.window > 0 ? hi - a.window : -1, head_end = a.first - j1;
#pragma unroll
                            for (int j = 0; j < 64; ++j)
                                if (j > hi || (j <= lo && j >= head_end)) s[j] = -INFINITY;
                        }
                        float top4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                        for (int j = 4; j < 60; j += 8)
#pragma unroll
                            for (int e = 0; e < 4; ++e) top4[e] = max3(top4[e], s[j + e], s[j + 4 + e]);
                        const float top = max3(max3(top4[0], top4[1], top4[2]), max3(top4[3], s[60], s[61]), fmaxf(s[62], s[63])) * a.c - Above<T>::value;      // c > 0
                        const bool move = top > m + 8.f || (m == -INFINITY && top > -INFINITY);
                        const float next = move ? top : m;
                        const float corr = move ? ex2(m - next) : 1.f;                    // 0 while no key has been seen
                        m = next;
                        const float z = m == -INFINITY ? 0.f : -m;
                        // O may be rescaled behind the last product with V; the one before that was ahead of these scores
                        if (any && __any_sync(0xffffffffu, move)) {
                            ok = wait(&pv_done[w], products - 1);
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < ocols; c += 32) {
                                float o[32];
                                tmem_ld_32x32(to + c, o);
#pragma unroll
                                for (int j = 0; j < 32; ++j) o[j] *= corr;
                                tmem_st_32x32(to + c, reinterpret_cast<const uint32_t*>(o));
                            }
                        }
                        const float2 c2 = make_float2(a.c, a.c), z2 = make_float2(z, z);
                        float2 l4[4] = {make_float2(l * corr, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                        uint32_t pw[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float2 t = fma2(make_float2(s[2 * j], s[2 * j + 1]), c2, z2);
                            // every fourth pair on the FMA pipe, which takes that off the exponential unit
                            const float2 u = (j & 3) == 3 ? ex2_fma(t) : make_float2(ex2(t.x), ex2(t.y));
                            l4[j & 3] = add2(l4[j & 3], u);
                            pw[j] = pack2<T>(u.x, u.y);
                        }
                        tmem_st_32x32(ts + 64 * half, pw);
                        const float2 lb = add2(add2(l4[0], l4[1]), add2(l4[2], l4[3]));
                        l = lb.x + lb.y;
                    }
                    any = true;
                    ++products;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[w][half]);
                }
                if (!ok) break;
                ++tiles;
            }
            if (!ok) break;
            if (any) {
                ok = wait(&o_full[w], outs++);
                if (!ok) break;
                tc_fence_after();
            } else if (valid) {
                m = -INFINITY;
            }
            // all of the tile's warps, or of both groups where these join their sums
            if (!two && w == 1) other[r] = make_float2(m, l);
            tc_fence_before();
            uint64_t* bar = two ? &met[w] : &joined;
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
            ok = wait(bar, two ? meets++ : joins);
            if (!ok) break;
            tc_fence_after();
            if (lane == 0) poison[w][note == 0 ? kNotes - 1 : note - 1] = 0;          // what the segment before noted: all have read it (kNotes)
            if (!two && w == 1) {
                ok = wait(&taken, joins++);
                if (!ok) break;
                release(i);
                continue;
            }
            float scale0 = 1.f, scale1 = 0.f;                         // of this group's O and, where it joins the two, of the other's
            bool both = false;                                        // whether the other group has had a tile
            if (!two) {
                const float2 ml = other[r];
                const float t = fmaxf(m, ml.x);
                if (t > -INFINITY) {
                    scale0 = ex2(m - t);
                    scale1 = ex2(ml.x - t);
                }
                l = l * scale0 + ml.y * scale1;
                m = t;
#pragma unroll 1
                for (int n = seg.n0 + 1; n < n1 && !both; n += 2) both = seg.see[0](n);
            }
            // the second group, which goes on behind `taken` alone, writes no note of its own before this one has been read
            if (poison[w][note] || (!two && poison[1][note])) {
                if (live) redo_rows<T>(x, seg, w, quarter);
            } else if (live) {
                const int h = seg.g * x.group + head, part_row = (two ? w : 0) * kTileQ + r;
                float inv = scale0;
                if (seg.whole) {
                    float f = 1.f;
                    if (a.sink && valid) {          // against the larger one: the maximum may be minus infinity
                        const float sk = a.sink[h] * kLog2e, top = fmaxf(m, sk);
                        f = ex2(m - top);
                        l = l * f + ex2(sk - top);
                        m = top;
                    }
                    f = valid && row >= 0 ? f / l : 0.f;
                    inv *= f;
                    scale1 *= f;
                    if (a.lse && valid) a.lse[(size_t)(it.token + token) * a.H + h] = m + log2f(l);
                } else if (valid) {
                    x.pl.ml[(size_t)seg.slot * x.pl.stride + part_row] = make_float2(m, l);
                }
                T* out = (T*)a.out + ((size_t)(it.token + tile0) * a.H + seg.g * x.group) * p.E;
                float4* parts = x.pl.o + (size_t)seg.slot * (p.E / 4) * x.pl.stride + part_row;
#pragma unroll 1
                for (int c = 0; c < ocols && (any || both); c += 32) {
                    float o[32];
                    if (any) {
                        tmem_ld_32x32(to + c, o);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] *= inv;
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = 0.f;
                    }
                    if (both) {
                        float e[32];
                        tmem_ld_32x32(to + 128 + c, e);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = fmaf(e[j], scale1, o[j]);
                    }
                    if (seg.whole) {
                        // turned around in shared memory, so that four lanes write 64 bytes of a row
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            turn[lane * 4 + (j ^ ((lane >> 1) & 3))] = make_uint4(pack2<T>(o[8 * j], o[8 * j + 1]), pack2<T>(o[8 * j + 2], o[8 * j + 3]), pack2<T>(o[8 * j + 4], o[8 * j + 5]),
                                                                                  pack2<T>(o[8 * j + 6], o[8 * j + 7]));
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int from = 8 * k + (lane >> 2);
                            const uint4 v = turn[from * 4 + ((lane & 3) ^ ((from >> 1) & 3))];
                            if (tile0 + turn_token[k] < it.count && c + 8 * (lane & 3) < p.E) *reinterpret_cast<uint4*>(out + turn_at[k] + c) = v;
                        }
                        __syncwarp();
                    } else if (valid) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            if (c + j < p.E) parts[(size_t)((c + j) / 4) * x.pl.stride] = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    }
                }
            }
            if (!two) {                  // the second group may go on
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&taken);
                ++joins;
            }
            release(i);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
}

// Joins the parts of items that several CTAs had, in their order.  Block b has the item that the boundary between CTAs b and b + 1 cuts, unless an earlier boundary cuts it too.
template <class T>
__global__ void __launch_bounds__(256) merge_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ Plan pl, int group, int tq) {
    rcu_kernel_entry();
    const View& p = a.p;
    const int b = blockIdx.x;
    const Join jn(pl, b, p.G, pl.items);
    if (jn.count == 0) return;
    const int rows = jn.it.count * group, quads = p.E / 4, first_token = clamp_int(p.starts[jn.it.s], 0, p.T) + jn.it.token;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < rows * quads; i += gridDim.y * 256) {
        const int u = i % rows, c = i / rows, token = u / group, h = jn.g * group + u % group;
        const int r = token / tq * kTileQ + u - token / tq * tq * group;
        float m = -INFINITY;
        for (int k = 0; k < jn.count; ++k) m = fmaxf(m, pl.ml[(size_t)jn.slot(b, k) * pl.stride + r].x);
        const float sk = a.sink ? a.sink[h] * kLog2e : -INFINITY, top = fmaxf(m, sk);
        float l = a.sink ? ex2(sk - top) : 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < jn.count; ++k) {
            const float2 ml = pl.ml[(size_t)jn.slot(b, k) * pl.stride + r];
            if (ml.x == -INFINITY && ml.y == 0.f) continue;          // a part that sees nothing has no sum
            const float w = ex2(ml.x - top);
            const float4 v = pl.o[((size_t)jn.slot(b, k) * quads + c) * pl.stride + r];
            l = fmaf(ml.y, w, l);
            o.x = fmaf(v.x, w, o.x);
            o.y = fmaf(v.y, w, o.y);
            o.z = fmaf(v.z, w, o.z);
            o.w = fmaf(v.w, w, o.w);
        }
        const float inv = 1.f / l;
        const size_t at = (size_t)(first_token + token) * a.H + h;
        uint2 v;
        v.x = pack2<T>(o.x * inv, o.y * inv);
        v.y = pack2<T>(o.z * inv, o.w * inv);
        *reinterpret_cast<uint2*>((T*)a.out + at * p.E + 4 * c) = v;
        if (a.lse && c == 0) a.lse[at] = top + log2f(l);
    }
}

// The cut of a call, and its scratch behind `mem` (nullable: sizes only); returns the bytes
uint64_t plan_of(const rcu_device* dev, const View& p, int H, char* mem, Plan* out) {
    const int group = H / p.G, tq = kTileQ / group;
    Plan pl{};
    pl.tokens = 2 * tq;
    pl.items = p.T / pl.tokens + p.S;
    pl.ctas = dev->sm_count;
    pl.least = 2;
    // a CTA's work on an item of two query tiles begins and ends for as long as two tiles take; with one it is less, and in generation tiles are dearer
    pl.extra = 2;
    pl.stride = p.T <= tq ? (p.T * group + 7) & ~7 : 2 * kTileQ;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        char* ptr = mem + at;
        at += align256(bytes);
        return ptr;
    };
    pl.head = (int*)take(8);
    pl.prefix = (int*)take(4ull * (pl.items + 1));
    pl.item = (Item*)take(sizeof(Item) * (uint64_t)pl.items);
    pl.ml = (float2*)take(8ull * 2 * pl.ctas * pl.stride);
    pl.o = (float4*)take(4ull * 2 * pl.ctas * pl.stride * p.E);
    if (out) *out = pl;
    return at;
}

template <class T> rcu_status launch(rcu_device* dev, const AttendArgs& a, int dt, void* scratch) {
    const View& p = a.p;
    TcArgs x{a, {}, a.H / p.G, kTileQ / (a.H / p.G), 0, (p.D + 63) / 64, (p.E + 63) / 64, 0};
    plan_of(dev, p, a.H, (char*)scratch, &x.pl);
    x.stage_bytes = (x.nb > x.eb ? x.nb : x.eb) * kBlock;
    constexpr int kTurn = 8 * 2048;
    const int room = dev->smem_optin - 3 * 1024 - kTurn - 2 * x.nb * kBlock;          // 1 KB to align, 2 KB of static shared memory
    x.stages = room / x.stage_bytes < kMostStages ? room / x.stage_bytes : kMostStages;
    const size_t smem = 1024 + (size_t)2 * x.nb * kBlock + (size_t)x.stages * x.stage_bytes + kTurn;
    CUtensorMap qm, km, vm;
    if (!map_queries(&qm, dt, p, a.q, x.group, x.tq) || !map_pages(&km, dt, p, p.keys, p.D) || !map_pages(&vm, dt, p, p.values, p.E))
        return rcu_fail(dev, RCU_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled failed (%d tokens, %d heads, %d pages)", p.T, a.H, p.pages);
    const rcu_status planned = plan_items(dev, p, x.pl, a.window, a.first, 1);
    if (planned != RCU_OK) return planned;
    void (*kern)(CUtensorMap, CUtensorMap, CUtensorMap, TcArgs) = paged_tc_kernel<T>;
    RCU_CUDA(dev, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    RCU_CUDA(dev, rcu_launch(dev, kern, x.pl.ctas, kThreadsP, smem, qm, km, vm, x));
    RCU_LAUNCH_CHECK(dev);
    if (x.pl.ctas > 1) {
        // a part has 256 rows at most: four blocks an item; with few rows one
        const int work = x.pl.stride * p.E / 4, split = work >= 4096 ? 8 : work >= 1024 ? 2 : 1;
        rcu_launch(dev, merge_kernel<T>, dim3(x.pl.ctas - 1, split), 256, 0, a, x.pl, x.group, x.tq);
        RCU_LAUNCH_CHECK(dev);
    }
    return RCU_OK;
}

}  // namespace

rcu_status plan_items(rcu_device* dev, const View& p, const Plan& plan, int window, int first, int group) {
    rcu_launch(dev, plan_kernel, 1, 1024, 0, p, plan, window, first, group);
    RCU_LAUNCH_CHECK(dev);
    return RCU_OK;
}

bool attend_tc_takes(const rcu_device* dev, const View& p, int H, int dt) {
    const int group = H / p.G;
    if (dt == RCU_F32 || p.D > 128 || p.E > 128 || group > kTileQ || dev->smem_optin < 227 * 1024) return false;
    // 32-bit tile numbers: all kv heads' tiles over the longest rows that the table allows
    return (uint64_t)(p.T / (kTileQ / group) + p.S) * (((uint64_t)p.MP << p.shift) / kTileK + 3) * p.G < (1ull << 31);
}

uint64_t attend_tc_scratch(const rcu_device* dev, const View& p, int H) { return plan_of(dev, p, H, nullptr, nullptr); }

rcu_status attend_tc(rcu_device* dev, const AttendArgs& a, int dt, void* scratch) {
    return dt == RCU_BF16 ? launch<__nv_bfloat16>(dev, a, dt, scratch) : launch<__half>(dev, a, dt, scratch);
}

}  // namespace paged
