// Attention of new tokens over paged caches on the 5th-generation tensor cores (tcgen05): f16 and bf16, heads of up to 128 features.
//
// A tile of queries is 128 / group tokens with all query heads of a kv head, so that keys and values are read once for the group.  CTA = two
// such tiles that take turns: while the softmax warps of one work, the tensor core runs the other's products.
//   warp 0              brings the queries, then keys and values of 128 rows in turns into a ring, page by page (a box per page or part of one;
//                       rows of no page stay as they are in shared memory);
//   warp 1              per tile n and query tile w: O_w += P_w V of tile n - 1, with P_w read from tensor memory, then S_w = Q_w K^T of tile n,
//                       which takes P_w's place;
//   warps 2-5, 6-9      softmax of tile 0 / 1, a query per thread: scores from tensor memory, mask, running maximum, weights back over the scores.
//                       The maximum that weights are taken against only moves when a score exceeds it by more than 2^8, so that O_w is rescaled rarely.
// Weights enter the second product in the operands' type: half a step of theirs moves the sum by as much as the rounding of the output does.  Their
// sum, the maximum and O are f32.
// What is masked must not reach the sum even where it is not finite, and 0 times infinity is NaN.  Rows behind the sequence's last one are zeroed in
// shared memory.  In a tile that some of the queries see in part, an infinity or NaN among the values sends the query tile to attend_rows, which
// reads only what each query sees.
// Every wait is bounded; one that gives up raises RCU_DEVFLAG_TIMEOUT and ends all others of the CTA.
#include <cuda.h>

#include "paged_attention.cuh"
#include "paged_rows.cuh"
#include "paged_tc.cuh"

namespace paged {
namespace {

constexpr int kThreadsP = 320, kMostStages = 8;

template <class T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// whether one of the two 16-bit values is an infinity or NaN
template <class T> __device__ __forceinline__ uint32_t not_finite(uint32_t x);
template <> __device__ __forceinline__ uint32_t not_finite<__half>(uint32_t x) { return __vcmpgeu2(x & 0x7fff7fffu, 0x7c007c00u); }
template <> __device__ __forceinline__ uint32_t not_finite<__nv_bfloat16>(uint32_t x) { return __vcmpgeu2(x & 0x7fff7fffu, 0x7f807f80u); }

// One thread per item: its tokens and tiles; then the sums before each.  One CTA.
__global__ void __launch_bounds__(1024) plan_kernel(const View p, const Plan pl, int window, int first) {
    rcu_kernel_entry();
    __shared__ int warps[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int s = tid; s < p.S; s += 1024)
        if (seq_bad(p, s)) report_bad(p.status);
    int before = 0;
    for (int base = 0; base < pl.items; base += 1024) {
        const int i = base + tid;
        Item it{-1, 0, 0, 0};
        int w = 0;
        if (i < pl.items) {
            // sequence s has the items from starts[s] / tokens + s on
            int lo = 0, hi = p.S - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (clamp_int(p.starts[mid], 0, p.T) / pl.tokens + mid <= i) lo = mid;
                else hi = mid - 1;
            }
            const Seq q = seq_of(p, lo);
            const int at = (i - q.start / pl.tokens - lo) * pl.tokens;
            if (at >= 0 && at < q.n) {
                it = Item{lo, q.start + at, min(pl.tokens, q.n - at), q.old() + at};
                w = span_of(window, first, it.row, min(it.row + it.count, q.L) - 1).count;
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
        for (int j = 0; j < 32; ++j) {
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
}

struct TcArgs {
    AttendArgs a;
    Plan pl;
    int group, tq;             // query heads of a kv head; tokens of a query tile
    int stages, nb, eb, stage_bytes;
};

template <class T>
__global__ void __launch_bounds__(kThreadsP, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const TcArgs x) {
    extern __shared__ unsigned char smem_dyn[];
    const AttendArgs& a = x.a;
    const View& p = a.p;
    unsigned char* qs = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    unsigned char* ring = qs + 2 * x.nb * kBlock;
    __shared__ __align__(8) uint64_t q_full, q_empty, full[kMostStages], empty[kMostStages], s_full[2], p_full[2], o_full[2], met[2], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag, poison[2];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 1);
        mbar_init(&drained, 1);
        for (int i = 0; i < x.stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
            mbar_init(&met[i], 4);
            poison[i] = 0;
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

    // whether query tile w of an item sees any of the rows j0 .. j0 + 127; the item's tokens are at rows row .. row + count - 1
    auto sees = [&](const Item& it, int w, int j0) {
        const int r0 = it.row + w * x.tq, r1 = min(r0 + x.tq, it.row + it.count) - 1;
        return r0 <= r1 && j0 <= r1 && (a.window == 0 || j0 + kTileK - 1 > r0 - a.window || j0 < a.first);
    };
    auto spans = [&](const Item& it) { return span_of(a.window, a.first, it.row, it.row + it.count - 1); };

    if (warp == 0) {
        const int rows_box = min(p.R, kTileK), boxes = kTileK / rows_box;
        const bool mine_k = lane < boxes * x.nb, mine_v = lane < boxes * x.eb;
        const int box = lane % boxes, col = lane / boxes;
        int fills = 0, seg = 0;
        bool ok = true;
        for (Walk wk(x.pl, blockIdx.x, p.G); wk.more() && ok; wk.next(), ++seg) {
            const Span sp = spans(wk.it);
            const int L = clamp_int(p.lengths[wk.it.s], 0, p.MP << p.shift);
            const bool second = wk.it.count > x.tq;
            if (seg > 0) ok = __all_sync(0xffffffffu, mbar_wait(&q_empty, (seg - 1) & 1, &abort_flag, p.status));
            if (!ok) break;
            if (lane == 0) {
                const int tiles = second ? 2 : 1;
                mbar_expect_tx(&q_full, tiles * x.nb * x.group * x.tq * 128);
                for (int w = 0; w < tiles; ++w)
                    for (int b = 0; b < x.nb; ++b) tma_load_4d(qs + (w * x.nb + b) * kBlock, &qmap, b * 64, 0, wk.g, wk.it.token + w * x.tq, &q_full);
            }
            __syncwarp();
            auto page_at = [&](int n) {          // of this lane's box; -1 behind the last row
                const int j = sp.tile(n) * kTileK + box * rows_box;
                return j < L ? page_of(p, wk.it.s, j) : -1;
            };
            int page = page_at(wk.n0);
            for (int n = wk.n0; n < wk.n1 && ok; ++n) {
                const int j0 = sp.tile(n) * kTileK, at = j0 & (p.R - 1);
                const int next = n + 1 < wk.n1 ? page_at(n + 1) : -1;
                const int pages = __popc(__ballot_sync(0xffffffffu, lane < boxes && page >= 0));
#pragma unroll
                for (int kv = 0; kv < 2; ++kv, ++fills) {
                    const int s = fills % x.stages;
                    if (fills >= x.stages) ok = ok && __all_sync(0xffffffffu, mbar_wait(&empty[s], (fills / x.stages - 1) & 1, &abort_flag, p.status));
                    if (!ok) break;
                    const int blocks = kv ? x.eb : x.nb;
                    if (lane == 0) mbar_expect_tx(&full[s], pages * blocks * rows_box * 128);
                    __syncwarp();
                    if ((kv ? mine_v : mine_k) && page >= 0)
                        tma_load_4d(ring + (size_t)s * x.stage_bytes + col * kBlock + box * rows_box * 128, kv ? &vmap : &kmap, col * 64, at, wk.g, page, &full[s]);
                }
                page = next;
            }
        }
        if (!ok) {          // given up: let the copies in flight land before the memory is somebody else's
            for (int i = max(0, fills - x.stages); i < fills; ++i)
                for (int k = 0; k < (1 << 16) && !gemvq8::mbar_test_wait(&full[i % x.stages], (i / x.stages) & 1); ++k) {}
            for (int k = 0; k < (1 << 16) && !gemvq8::mbar_test_wait(&q_full, seg & 1); ++k) {}
        }
    } else if (warp == 1) {
        // the whole warp keeps step, one elected lane issues
        constexpr bool bf16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
        const uint32_t idesc_s = umma_idesc_f16(kTileQ, kTileK, bf16);
        const uint32_t idesc_o = umma_idesc_f16(kTileQ, (p.E + 15) & ~15, bf16) | (1u << 16);     // V is stored with its columns contiguous
        const int ksteps = (p.D + 15) / 16;
        const uint64_t qd = umma_desc_sw128(qs), kd = umma_desc_sw128(ring), vd = umma_desc_sw128_mn(ring, kBlock);
        const bool leader = elect_one();
        auto wait = [&](uint64_t* bar, int phase) { return (bool)__all_sync(0xffffffffu, mbar_wait_spin(bar, phase & 1, &abort_flag, p.status)); };
        bool ok = true;
        int seg = 0, base = 0, weights[2] = {0, 0};          // base: fills before this run; weights: hand-overs of P_w so far
        for (Walk wk(x.pl, blockIdx.x, p.G); wk.more() && ok; wk.next(), ++seg) {
            const Span sp = spans(wk.it);
            const int count = wk.n1 - wk.n0;
            bool any[2] = {false, false};
            ok = wait(&q_full, seg);
            for (int m = 0; m <= count && ok; ++m) {
                const int kf = base + 2 * m, vf = base + 2 * m - 1;          // fills of K of this tile, V of the one before
                const int j0 = m < count ? sp.tile(wk.n0 + m) * kTileK : 0, i0 = m > 0 ? sp.tile(wk.n0 + m - 1) * kTileK : 0;
                if (m < count) ok = wait(&full[kf % x.stages], kf / x.stages);
                if (ok && m > 0) ok = wait(&full[vf % x.stages], vf / x.stages);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (ok && m > 0 && sees(wk.it, w, i0)) {
                        ok = wait(&p_full[w], weights[w]++);
                        tc_fence_after();
                        if (ok && leader) {
                            const uint64_t bd = vd + (uint64_t)((vf % x.stages) * (x.stage_bytes >> 4));
#pragma unroll
                            for (int k = 0; k < kTileK / 16; ++k)      // 16 rows are two 1024-byte groups of V, eight columns of P
                                umma_f16_ta(tmem + 256 + 128 * w, tmem + 128 * w + 8 * k, bd + 128 * k, idesc_o, k > 0 || any[w] ? 1u : 0u);
                        }
                        any[w] = true;
                        __syncwarp();
                    }
                    if (ok && m < count && sees(wk.it, w, j0)) {
                        tc_fence_after();
                        if (leader) {
                            const uint64_t ad = qd + (uint64_t)(w * x.nb * (kBlock >> 4)), bd = kd + (uint64_t)((kf % x.stages) * (x.stage_bytes >> 4));
                            for (int k = 0; k < ksteps; ++k) {
                                const uint64_t off = (k >> 2) * (kBlock >> 4) + 2 * (k & 3);
                                umma_f16(tmem + 128 * w, ad + off, bd + off, idesc_s, k > 0 ? 1u : 0u);
                            }
                            umma_commit(&s_full[w]);
                        }
                        __syncwarp();
                    }
                }
                if (!ok) break;
                if (leader) {
                    if (m < count) umma_commit(&empty[kf % x.stages]);
                    if (m == count - 1) umma_commit(&q_empty);
                    if (m > 0) umma_commit(&empty[vf % x.stages]);
                    if (m == count) {
                        if (any[0]) umma_commit(&o_full[0]);
                        if (any[1]) umma_commit(&o_full[1]);
                    }
                }
                __syncwarp();
            }
            base += 2 * count;
        }
        if (!ok && leader) {            // given up: let the products in flight end before tensor memory is freed
            umma_commit(&drained);
            for (int i = 0; i < (1 << 20) && !gemvq8::mbar_test_wait(&drained, 0); ++i) {}
        }
        __syncwarp();
    } else {
        const int w = warp < 6 ? 0 : 1, quarter = warp & 3;
        const int r = quarter * 32 + lane;                                   // row of the query tile
        const int token = w * x.tq + r / x.group, head = r % x.group;        // token of the item, query head of the group
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16, ts = tmem + 128 * w + lanes, to = tmem + 256 + 128 * w + lanes;
        const int ocols = (p.E + 31) & ~31;
        int base = 0, scores = 0, outs = 0, meets = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, int phase) { return (bool)__all_sync(0xffffffffu, mbar_wait_spin(bar, phase & 1, &abort_flag, p.status)); };
        auto meet = [&]() {              // the tile's four warps; bounded like every wait
            __syncwarp();
            if (lane == 0) mbar_arrive(&met[w]);
            return wait(&met[w], meets++);
        };
        for (Walk wk(x.pl, blockIdx.x, p.G); wk.more() && ok; wk.next()) {
            const Span sp = spans(wk.it);
            const int L = clamp_int(p.lengths[wk.it.s], 0, p.MP << p.shift);
            const bool valid = r < x.tq * x.group && token < wk.it.count;
            const int row = wk.it.row + token;
            const bool live = __any_sync(0xffffffffu, valid);               // warps without a query only keep step
            // rows of the tile's and of the warp's first and last query
            const int t0 = wk.it.row + w * x.tq, t1 = min(t0 + x.tq, wk.it.row + wk.it.count) - 1;
            const int w0 = __reduce_min_sync(0xffffffffu, valid ? row : 0x7fffffff), w1 = __reduce_max_sync(0xffffffffu, valid ? row : -1);
            float m = valid ? -INFINITY : INFINITY, l = 0.f;                // a row of no query never moves the maximum
            bool any = false;
            for (int n = wk.n0; n < wk.n1 && ok; ++n) {
                const int j0 = sp.tile(n) * kTileK, vf = base + 2 * (n - wk.n0) + 1;
                if (!sees(wk.it, w, j0)) continue;
                // a tile that is not whole to all queries: rows behind the last one become zero, values that are not finite are noted
                const bool part = j0 + kTileK - 1 > t0 || (a.window > 0 && j0 <= t1 - a.window && j0 + kTileK > a.first);
                if (part) {
                    ok = wait(&full[vf % x.stages], vf / x.stages);
                    if (!ok) break;
                    unsigned char* v = ring + (size_t)(vf % x.stages) * x.stage_bytes + r * 128;
                    const bool behind = j0 + r >= L;
                    uint32_t bad = 0;
                    for (int b = 0; b < x.eb; ++b)
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            uint4* at = reinterpret_cast<uint4*>(v + b * kBlock + ((c ^ (lane & 7)) << 4));
                            if (behind) *at = make_uint4(0, 0, 0, 0);
                            else {
                                const uint4 u = *at;
                                bad |= not_finite<T>(u.x) | not_finite<T>(u.y) | not_finite<T>(u.z) | not_finite<T>(u.w);
                            }
                        }
                    if (bad) poison[w] = 1;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                ok = wait(&s_full[w], scores++);
                if (!ok) break;
                tc_fence_after();
                if (live) {
                    float s[128];
                    tmem_ld_32x64(ts, s);
                    tmem_ld_32x64(ts + 64, s + 64);
                    if (j0 + kTileK - 1 > w0 || (a.window > 0 && j0 <= w1 - a.window && j0 + kTileK > a.first)) {
                        const int hi = row - j0, lo = a.window > 0 ? hi - a.window : -1, head_end = a.first - j0;
#pragma unroll
                        for (int j = 0; j < 128; ++j)
                            if (j > hi || (j <= lo && j >= head_end)) s[j] = -INFINITY;
                    }
                    float top4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int j = 4; j < 128; ++j) top4[j & 3] = fmaxf(top4[j & 3], s[j]);
                    const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * a.c;      // c > 0
                    const bool move = top > m + 8.f || (m == -INFINITY && top > -INFINITY);
                    const float next = move ? top : m;
                    const float corr = move ? ex2(m - next) : 1.f;                    // 0 while no key has been seen
                    m = next;
                    const float z = m == -INFINITY ? 0.f : -m;
                    float l4[4] = {l * corr, 0.f, 0.f, 0.f};
                    uint32_t pw[64];
#pragma unroll
                    for (int j = 0; j < 64; ++j) {
                        const float u = ex2(fmaf(s[2 * j], a.c, z)), v = ex2(fmaf(s[2 * j + 1], a.c, z));
                        l4[j & 3] += u + v;
                        pw[j] = pack2<T>(u, v);
                    }
                    l = (l4[0] + l4[1]) + (l4[2] + l4[3]);
                    // the scores came behind the tile before's product with V: O may be rescaled
                    if (any && __any_sync(0xffffffffu, move)) {
                        for (int c = 0; c < ocols; c += 32) {
                            float o[32];
                            tmem_ld_32x32(to + c, o);
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] *= corr;
                            tmem_st_32x32(to + c, reinterpret_cast<const uint32_t*>(o));
                        }
                    }
                    tmem_st_32x64(ts, pw);
                }
                any = true;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[w]);
            }
            if (!ok) break;
            base += 2 * (wk.n1 - wk.n0);
            if (any) {
                ok = wait(&o_full[w], outs++);
                if (!ok) break;
                tc_fence_after();
            }
            const int slot = wk.slot(blockIdx.x), part_row = w * kTileQ + r;
            const int h = wk.g * x.group + head;
            const size_t q_at = (size_t)(wk.it.token + token) * a.H + h;
            ok = meet();
            if (!ok) break;
            if (poison[w]) {
                if (live)
                    for (int i = 0; i < 32; ++i) {
                        const int ri = quarter * 32 + i, ti = w * x.tq + ri / x.group;
                        if (ri >= x.tq * x.group || ti >= wk.it.count) continue;
                        RowPart part;
                        attend_row<T>(a, wk.it.s, wk.g, wk.it.token + ti, wk.g * x.group + ri % x.group, wk.it.row + ti, sp, wk.n0, wk.n1, part);
                        if (wk.whole) finish_row<T>(a, wk.it.token + ti, wk.g * x.group + ri % x.group, part);
                        else store_part(x.pl, p.E, slot, w * kTileQ + ri, part);
                    }
                ok = meet();
                if (!ok) break;
                poison[w] = 0;
                ok = meet();
            } else if (live) {
                float inv = 1.f;
                if (wk.whole) {
                    if (a.sink && valid) l += ex2(a.sink[h] * kLog2e - m);
                    inv = valid && any && row >= 0 ? 1.f / l : 0.f;
                    if (a.lse && valid) a.lse[q_at] = m + log2f(l);
                } else if (valid) {
                    x.pl.ml[(size_t)slot * x.pl.stride + part_row] = make_float2(any ? m : -INFINITY, l);
                }
                if (any) {
                    T* out = (T*)a.out + q_at * p.E;
                    float4* parts = x.pl.o + (size_t)slot * (p.E / 4) * x.pl.stride + part_row;
                    for (int c = 0; c < ocols; c += 32) {
                        float o[32];
                        tmem_ld_32x32(to + c, o);
                        if (!valid) continue;
                        if (wk.whole) {
#pragma unroll
                            for (int j = 0; j < 32; j += 8)
                                if (c + j < p.E) {          // E is a multiple of 8
                                    uint4 v;
                                    v.x = pack2<T>(o[j] * inv, o[j + 1] * inv);
                                    v.y = pack2<T>(o[j + 2] * inv, o[j + 3] * inv);
                                    v.z = pack2<T>(o[j + 4] * inv, o[j + 5] * inv);
                                    v.w = pack2<T>(o[j + 6] * inv, o[j + 7] * inv);
                                    *reinterpret_cast<uint4*>(out + c + j) = v;
                                }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; j += 4)
                                if (c + j < p.E) parts[(size_t)((c + j) / 4) * x.pl.stride] = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                        }
                    }
                }
            }
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
__global__ void __launch_bounds__(256) merge_kernel(const AttendArgs a, const Plan pl, int group, int tq) {
    rcu_kernel_entry();
    const View& p = a.p;
    const int W = pl.head[0], C = pl.head[1], b = blockIdx.x;
    if (b + 1 >= C) return;
    const long long total = (long long)W * p.G;
    const int begin = first_tile(total, b, C), cut = first_tile(total, b + 1, C);
    Walk wk(pl, b + 1, p.G);             // the item at the boundary
    const int start = wk.g * W + pl.prefix[wk.i], stop = wk.g * W + pl.prefix[wk.i + 1];
    if (start == cut || start < begin) return;
    int parts = 1;                       // CTAs b .. b + parts - 1
    while (b + parts < C && first_tile(total, b + parts, C) < stop) ++parts;
    const int first_slot = 2 * b + (start != begin);
    auto slot = [&](int i) { return i == 0 ? first_slot : 2 * (b + i); };
    const int rows = wk.it.count * group, quads = p.E / 4;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < rows * quads; i += gridDim.y * 256) {
        const int u = i % rows, c = i / rows, token = u / group, h = wk.g * group + u % group;
        const int r = token / tq * kTileQ + u - token / tq * tq * group;
        float m = -INFINITY;
        for (int k = 0; k < parts; ++k) m = fmaxf(m, pl.ml[(size_t)slot(k) * pl.stride + r].x);
        const float sk = a.sink ? a.sink[h] * kLog2e : -INFINITY, top = fmaxf(m, sk);
        float l = a.sink ? ex2(sk - top) : 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < parts; ++k) {
            const float2 ml = pl.ml[(size_t)slot(k) * pl.stride + r];
            if (ml.x == -INFINITY && ml.y == 0.f) continue;          // a part that sees nothing has no sum
            const float w = ex2(ml.x - top);
            const float4 v = pl.o[((size_t)slot(k) * quads + c) * pl.stride + r];
            l = fmaf(ml.y, w, l);
            o.x = fmaf(v.x, w, o.x);
            o.y = fmaf(v.y, w, o.y);
            o.z = fmaf(v.z, w, o.z);
            o.w = fmaf(v.w, w, o.w);
        }
        const float inv = 1.f / l;
        const size_t at = (size_t)(wk.it.token + token) * a.H + h;
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
    pl.rows = tq * group;
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
    const int room = dev->smem_optin - 2048 - 2 * x.nb * kBlock;          // 1 KB to align, 1 KB of static shared memory
    x.stages = room / x.stage_bytes < kMostStages ? room / x.stage_bytes : kMostStages;
    const size_t smem = 1024 + (size_t)2 * x.nb * kBlock + (size_t)x.stages * x.stage_bytes;
    CUtensorMap qm, km, vm;
    if (!map_queries(&qm, dt, p, a.q, x.group, x.tq) || !map_pages(&km, dt, p, p.keys, p.D) || !map_pages(&vm, dt, p, p.values, p.E))
        return rcu_fail(dev, RCU_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled failed (%d tokens, %d heads, %d pages)", p.T, a.H, p.pages);
    rcu_launch(dev, plan_kernel, 1, 1024, 0, p, x.pl, a.window, a.first);
    RCU_LAUNCH_CHECK(dev);
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

bool attend_tc_takes(const rcu_device* dev, const AttendArgs& a, int dt) {
    const View& p = a.p;
    if (dt == RCU_F32 || p.D > 128 || p.E > 128 || a.H / p.G > kTileQ || !(a.c > 0.f) || !(a.c < INFINITY)) return false;
    // 32-bit tile numbers: all kv heads' tiles over the longest rows that the table allows
    if ((uint64_t)(p.T / (kTileQ / (a.H / p.G)) + p.S) * (((uint64_t)p.MP << p.shift) / kTileK + 1) * p.G >= (1ull << 31)) return false;
    return ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0 && dev->smem_optin >= 227 * 1024;
}

uint64_t attend_tc_scratch(const rcu_device* dev, const View& p, int H) { return plan_of(dev, p, H, nullptr, nullptr); }

rcu_status attend_tc(rcu_device* dev, const AttendArgs& a, int dt, void* scratch) {
    return dt == RCU_BF16 ? launch<__nv_bfloat16>(dev, a, dt, scratch) : launch<__half>(dev, a, dt, scratch);
}

}  // namespace paged
