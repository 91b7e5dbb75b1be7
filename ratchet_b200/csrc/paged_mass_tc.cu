// The attention weight that every cached row receives (rcu_paged_attention where mass is kept), f16 and bf16 up to 128 features:
//
//   mass[j] += sum over the group's heads and the new tokens that see j of 2^(c q.k_j - lse(q))
//
// with the lse that the attention has left.  The scores are worked out again, the other way round: S^T = K Q^T has a row of the cache per lane of tensor
// memory, so a thread adds up its own row's weights in a register, in the same order in every call, and nothing is exchanged between
// lanes.  A tile of 128 rows stays in shared memory while the query tiles that see it pass by (paged_attention.cuh's cut, with rows and
// queries in each other's place).
//   warp 0            a tile of rows per item, two of them in turns; query tiles and their lse into a ring;
//   warp 1            S^T of every query tile, four buffers of tensor memory;
//   warps 2-5, 6-9    every other query tile each: exponentials and sums, which are joined at the end of the item.
// Bound by the exponentials and what is issued around them: 128 x 128 of them take 1024 cycles of an SM, the product half of that.  777 tokens over 20000 rows,
// 32 heads over 8, 80 features: 193 us (exponential pipe 52 %, issue slots 49 %, tensor pipe 21 %).
// Every wait is bounded; one that gives up raises RCU_DEVFLAG_TIMEOUT and ends all others of the CTA.
#include "paged_tc.cuh"

namespace paged {
namespace {

constexpr int kThreadsM = 320, kStagesQ = 4, kStagesL = 8;       // query tiles in shared memory; their lse, which are read for longer

// Query tiles j of sequence q (tq tokens each) that see any of the rows j0 .. j0 + 127: [lo, hi)
__device__ __forceinline__ void seen_by(const Seq& q, int window, int first, int tq, int j0, int& lo, int& hi) {
    const int tiles = (q.n + tq - 1) / tq;
    lo = j0 > q.old() ? (j0 - q.old()) / tq : 0;
    hi = tiles;
    if (window > 0 && j0 >= first) {
        const int last = j0 + kTileK - 1 + window - 1 - q.old();         // the last token whose window reaches the tile
        hi = last < 0 ? 0 : min(tiles, last / tq + 1);
    }
    lo = min(lo, hi);
}

// Items are tiles of rows: Item{sequence, tile, its first query tile, -}.  First the sequences' tiles before each (base), then as plan_kernel.
__global__ void __launch_bounds__(1024) mass_plan_kernel(const View p, const Plan pl, int* base, int window, int first, int tq) {
    rcu_kernel_entry();
    __shared__ int warps[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int before = 0;
    auto scan = [&](int w, int& at) {          // exclusive sum over the CTA, on top of `before`, which moves on
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
        at = add + upto - w;
        before += all;
        __syncthreads();
    };
    for (int b = 0; b < p.S; b += 1024) {
        int w = 0, at;
        if (b + tid < p.S) {
            const Seq q = seq_of(p, b + tid);
            w = q.n > 0 ? (q.L + kTileK - 1) / kTileK : 0;
        }
        scan(w, at);
        if (b + tid < p.S) base[b + tid] = at;
    }
    const int items = min(before, pl.items);
    __syncthreads();                          // base is read by others
    before = 0;
    for (int b = 0; b < items; b += 1024) {
        const int i = b + tid;
        int w = 0, at;
        if (i < items) {
            int lo = 0, hi = p.S - 1;            // the last sequence with base <= i
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (base[mid] <= i) lo = mid;
                else hi = mid - 1;
            }
            int j0, j1;
            seen_by(seq_of(p, lo), window, first, tq, (i - base[lo]) * kTileK, j0, j1);
            pl.item[i] = Item{lo, i - base[lo], j0, 0};
            w = j1 - j0;
        }
        scan(w, at);
        if (i < items) pl.prefix[i] = at;
    }
    if (tid == 0) {
        pl.prefix[items] = before;
        pl.head[0] = before;
        const long long total = (long long)before * p.G;
        pl.head[1] = (int)max(1ll, min((long long)pl.ctas, (total + pl.least - 1) / pl.least));
        pl.head[2] = items;
    }
}

struct MassArgs {
    AttendArgs a;
    Plan pl;
    int group, tq, nb;
};

template <class T>
__global__ void __launch_bounds__(kThreadsM, 1) mass_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ MassArgs x) {
    extern __shared__ unsigned char smem_dyn[];
    const AttendArgs& a = x.a;
    const View& p = a.p;
    const int tile_bytes = x.nb * kBlock;
    unsigned char* ks = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    unsigned char* ring = ks + 2 * tile_bytes;
    __shared__ __align__(16) float lse[kStagesL][kTileQ];             // -lse of a tile's queries, -infinity where there is none
    __shared__ float sums[2][kTileK];
    __shared__ __align__(8) uint64_t k_full[2], k_empty[2], q_full[kStagesQ], q_empty[kStagesQ], l_full[kStagesL], l_empty[kStagesL], s_full[4], s_empty[4], handed[2], taken[2], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&drained, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&handed[i], 4);
            mbar_init(&taken[i], 4);
        }
        for (int i = 0; i < kStagesQ; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < kStagesL; ++i) {
            mbar_init(&l_full[i], 32);
            mbar_init(&l_empty[i], 4);           // of the group that has the tile
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], 4);
        }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // rows of a query tile that no box fills
    const int filled = x.tq * x.group;
    for (int i = threadIdx.x; i < kStagesQ * x.nb * (kTileQ - filled) * 8; i += kThreadsM) {
        const int block = i / ((kTileQ - filled) * 8), at = i % ((kTileQ - filled) * 8);
        reinterpret_cast<uint4*>(ring + (size_t)block * kBlock + filled * 128)[at] = make_uint4(0, 0, 0, 0);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    rcu_kernel_entry_wait_only();        // nothing before this touches global memory
    const uint32_t tmem = tmem_slot;
    const int items = x.pl.head[2];
    auto wait = [&](uint64_t* bar, int phase) { return wait_warp(bar, phase, &abort_flag, p.status); };

    if (warp == 0) {
        const int rows_box = min(p.R, kTileK), boxes = kTileK / rows_box, box = lane % boxes, col = lane / boxes;
        // this lane's four queries of a tile: token and head
        int token[4], head[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = lane + 32 * i;
            token[i] = u < filled ? u / x.group : 1 << 30;
            head[i] = u % x.group;
        }
        int item = 0, fills = 0;
        RingAt at{kStagesQ, 0, 0}, lat{kStagesL, 0, 0};
        bool ok = true;
#pragma unroll 1
        for (Walk wk(x.pl, blockIdx.x, p.G, items); wk.more() && ok; wk.next(), ++item) {
            const Seq q = seq_of(p, wk.it.s);
            const int j0 = wk.it.token * kTileK, b = item & 1;
            const int page = j0 + box * rows_box < q.L ? page_of(p, wk.it.s, j0 + box * rows_box) : -1;
            const int pages = __popc(__ballot_sync(0xffffffffu, lane < boxes && page >= 0));
            ok = wait(&k_empty[b], (item / 2) ^ 1);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(&k_full[b], pages * x.nb * rows_box * 128);
            __syncwarp();
            if (lane < boxes * x.nb && page >= 0) tma_load_4d(ks + b * tile_bytes + col * kBlock + box * rows_box * 128, &kmap, col * 64, j0 & (p.R - 1), wk.g, page, &k_full[b]);
            // the lse of a tile's queries is asked for while the tile before goes its way
            auto ask = [&](int n, float (&v)[4]) {
                const int t0 = (wk.it.count + n) * x.tq;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = token[i] < q.n - t0;
                    v[i] = in ? a.lse[(size_t)(q.start + t0 + token[i]) * a.H + wk.g * x.group + head[i]] : INFINITY;
                }
            };
            float v[4];
            ask(wk.n0, v);
#pragma unroll 1
            for (int n = wk.n0; n < wk.n1; ++n, ++fills) {
                const int t0 = (wk.it.count + n) * x.tq;
                float next[4] = {0.f, 0.f, 0.f, 0.f};
                if (n + 1 < wk.n1) ask(n + 1, next);
                ok = wait(&q_empty[at.s], at.phase ^ 1);
                if (!ok) break;
                if (lane == 0) {
                    mbar_expect_tx(&q_full[at.s], x.nb * filled * 128);
#pragma unroll 1
                    for (int c = 0; c < x.nb; ++c) tma_load_4d(ring + (size_t)at.s * tile_bytes + c * kBlock, &qmap, c * 64, 0, wk.g, q.start + t0, &q_full[at.s]);
                }
                __syncwarp();
                ok = wait(&l_empty[lat.s], lat.phase ^ 1);
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    lse[lat.s][lane + 32 * i] = -v[i];
                    v[i] = next[i];
                }
                mbar_arrive(&l_full[lat.s]);
                lat.go(1);
                __syncwarp();
                at.go(1);
            }
        }
        if (!ok) {          // given up: let the copies in flight land before the memory is somebody else's
#pragma unroll 1
            for (int i = max(0, fills - kStagesQ); i <= fills; ++i) land(&q_full[i % kStagesQ], i / kStagesQ);
#pragma unroll 1
            for (int i = max(0, item - 1); i <= item; ++i) land(&k_full[i & 1], i / 2);
        }
    } else if (warp == 1) {
        // one lane: what it does between two products, tensor memory waits for.  Every lane walks, one goes on.
        const bool leader = elect_one();
        constexpr bool bf16 = !std::is_same<T, __half>::value;
        const uint32_t idesc = umma_idesc_f16(kTileK, kTileQ, bf16);
        const int ksteps = (p.D + 15) / 16, tile16 = tile_bytes >> 4;
        const uint64_t kd = umma_desc_sw128(ks), qd = umma_desc_sw128(ring);
        auto wait1 = [&](uint64_t* bar, int phase) { return gemvq8::mbar_try_wait(bar, phase & 1) || wait_on(bar, phase & 1, &abort_flag, p.status); };
        bool ok = true;
        int item = 0, done = 0;                    // done: query tiles so far
        RingAt at{kStagesQ, 0, 0};
#pragma unroll 1
        for (Walk wk(x.pl, blockIdx.x, p.G, items); wk.more() && ok; wk.next(), ++item) {
            const int b = item & 1;
            if (leader) {
                ok = wait1(&k_full[b], item / 2);
#pragma unroll 1
                for (int n = wk.n0; n < wk.n1 && ok; ++n) {
                    const int t = done & 3;
                    ok = wait1(&q_full[at.s], at.phase) && wait1(&s_empty[t], (done / 4) ^ 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t ad = kd + (uint64_t)(b * tile16), bd = qd + (uint64_t)(at.s * tile16);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k < ksteps) umma_f16(tmem + 128 * t, ad + (k >> 2) * (kBlock >> 4) + 2 * (k & 3), bd + (k >> 2) * (kBlock >> 4) + 2 * (k & 3), idesc, k > 0 ? 1u : 0u);
                    umma_commit(&s_full[t]);
                    umma_commit(&q_empty[at.s]);
                    if (n == wk.n1 - 1) umma_commit(&k_empty[b]);
                    ++done;
                    at.go(1);
                }
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok && leader) {            // given up: let the products in flight end before tensor memory is freed
            umma_commit(&drained);
#pragma unroll 1
            for (int k = 0; k < 16; ++k) land(&drained, 0);
        }
        __syncwarp();
    } else {
        const int w = warp < 6 ? 0 : 1, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        bool ok = true;
        int item = 0, at = 0;
        for (Walk wk(x.pl, blockIdx.x, p.G, items); wk.more() && ok; wk.next(), ++item) {
            const Seq q = seq_of(p, wk.it.s);
            const int j0 = wk.it.token * kTileK, j = j0 + r;
            float sum = 0.f;
            for (int n = wk.n0; n < wk.n1 && ok; ++n, ++at) {
                if ((at & 1) != w) continue;
                const int s = at % kStagesL, t = at & 3;
                ok = wait(&l_full[s], at / kStagesL) && wait(&s_full[t], at / 4);
                if (!ok) break;
                tc_fence_after();
                const int t0 = (wk.it.count + n) * x.tq, r0 = q.old() + t0, r1 = r0 + x.tq - 1;
                // every query sees every row of the tile
                const bool whole = t0 + x.tq <= q.n && j0 + kTileK - 1 <= r0 && (a.window == 0 || j0 > r1 - a.window || j0 + kTileK <= a.first);
                // the queries that see row j are a run of the tile's columns: those from its own token on, as far as the window reaches
                const int from = clamp_int(j - r0, 0, x.tq) * x.group;
                const int last = a.window > 0 && j >= a.first ? clamp_int(j + a.window - r0, 0, x.tq) : x.tq, upto = min(last, q.n - t0) * x.group;
                float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    float z[64];
                    tmem_ld_32x64(tmem + 128 * t + 64 * half + lanes, z);
                    const float4* ls = reinterpret_cast<const float4*>(&lse[s][64 * half]);
                    const float2 c2 = make_float2(a.c, a.c);
                    auto weights = [&](auto masked) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            const float4 v = ls[c];
                            float2 x[2] = {fma2(make_float2(z[4 * c], z[4 * c + 1]), c2, make_float2(v.x, v.y)), fma2(make_float2(z[4 * c + 2], z[4 * c + 3]), c2, make_float2(v.z, v.w))};
                            // behind lse: a query that has none (NaN, or minus infinity for all it sees) must not reach the rows that it does not see
                            auto seen = [&](int i) { return 4 * c + i >= from - 64 * half && 4 * c + i < upto - 64 * half; };
                            if (masked())
#pragma unroll
                                for (int i = 0; i < 2; ++i) x[i] = make_float2(seen(2 * i) ? x[i].x : -INFINITY, seen(2 * i + 1) ? x[i].y : -INFINITY);
                            add[0] = add2(add[0], make_float2(ex2(x[0].x), ex2(x[0].y)));
                            // every fourth pair on the FMA pipe, which takes that off the exponential unit
                            add[1] = add2(add[1], c & 1 ? ex2_fma(x[1]) : make_float2(ex2(x[1].x), ex2(x[1].y)));
                        }
                    };
                    if (whole) weights(std::false_type{});          // a branch, not 64 selections in every tile
                    else weights(std::true_type{});
                }
                tc_fence_before();
                const float2 both = add2(add[0], add[1]);
                sum += both.x + both.y;
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&s_empty[t]);
                    mbar_arrive(&l_empty[s]);
                }
            }
            if (!ok) break;
            // the second group's sums to the first: two places in turns
            const int b = item & 1;
            if (w == 1) {
                if (item >= 2) ok = wait(&taken[b], item / 2 - 1);
                if (!ok) break;
                sums[b][r] = sum;
                __syncwarp();
                if (lane == 0) mbar_arrive(&handed[b]);
            } else {
                ok = wait(&handed[b], item / 2);
                if (!ok) break;
                sum += sums[b][r];
                __syncwarp();
                if (lane == 0) mbar_arrive(&taken[b]);
                if (!wk.whole) reinterpret_cast<float*>(x.pl.ml)[wk.slot(blockIdx.x) * kTileK + r] = sum;
                else if (j < q.L) p.mass[((size_t)wk.it.s * p.G + wk.g) * ((size_t)p.MP << p.shift) + j] += sum;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
}

// Adds the parts of tiles that several CTAs had, in their order (as merge_kernel).
__global__ void __launch_bounds__(kTileK) mass_merge_kernel(const __grid_constant__ View p, const __grid_constant__ Plan pl) {
    rcu_kernel_entry();
    const int b = blockIdx.x;
    const Join jn(pl, b, p.G, pl.head[2]);
    if (jn.count == 0) return;
    const float* parts = reinterpret_cast<const float*>(pl.ml);
    const int r = threadIdx.x, j = jn.it.token * kTileK + r, L = clamp_int(p.lengths[jn.it.s], 0, p.MP << p.shift);
    float sum = 0.f;
    for (int k = 0; k < jn.count; ++k) sum += parts[jn.slot(b, k) * kTileK + r];
    if (j < L) p.mass[((size_t)jn.it.s * p.G + jn.g) * ((size_t)p.MP << p.shift) + j] += sum;
}

uint64_t mass_plan_of(const rcu_device* dev, const View& p, char* mem, Plan* out, int** base) {
    Plan pl{};
    pl.items = p.S * (((p.MP << p.shift) + kTileK - 1) / kTileK);
    pl.ctas = dev->sm_count;
    pl.least = 4;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        char* ptr = mem + at;
        at += align256(bytes);
        return ptr;
    };
    pl.head = (int*)take(12);
    pl.prefix = (int*)take(4ull * (pl.items + 1));
    pl.item = (Item*)take(sizeof(Item) * (uint64_t)pl.items);
    pl.ml = (float2*)take(4ull * 2 * pl.ctas * kTileK);
    int* b = (int*)take(4ull * p.S);
    if (out) *out = pl;
    if (base) *base = b;
    return at;
}

template <class T> rcu_status launch_mass(rcu_device* dev, const AttendArgs& a, int dt, void* scratch) {
    const View& p = a.p;
    MassArgs x{a, {}, a.H / p.G, kTileQ / (a.H / p.G), (p.D + 63) / 64};
    int* base;
    mass_plan_of(dev, p, (char*)scratch, &x.pl, &base);
    CUtensorMap qm, km;
    if (!map_queries(&qm, dt, p, a.q, x.group, x.tq) || !map_pages(&km, dt, p, p.keys, p.D))
        return rcu_fail(dev, RCU_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled failed (%d tokens, %d heads, %d pages)", p.T, a.H, p.pages);
    rcu_launch(dev, mass_plan_kernel, 1, 1024, 0, p, x.pl, base, a.window, a.first, x.tq);
    RCU_LAUNCH_CHECK(dev);
    const size_t smem = 1024 + (size_t)(2 + kStagesQ) * x.nb * kBlock;
    void (*kern)(CUtensorMap, CUtensorMap, MassArgs) = mass_tc_kernel<T>;
    RCU_CUDA(dev, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    RCU_CUDA(dev, rcu_launch(dev, kern, x.pl.ctas, kThreadsM, smem, qm, km, x));
    RCU_LAUNCH_CHECK(dev);
    if (x.pl.ctas > 1) {
        rcu_launch(dev, mass_merge_kernel, x.pl.ctas - 1, kTileK, 0, p, x.pl);
        RCU_LAUNCH_CHECK(dev);
    }
    return RCU_OK;
}

}  // namespace

uint64_t mass_tc_scratch(const rcu_device* dev, const View& p, int) { return mass_plan_of(dev, p, nullptr, nullptr, nullptr); }

rcu_status mass_tc(rcu_device* dev, const AttendArgs& a, int dt, void* scratch) {
    return dt == RCU_BF16 ? launch_mass<__nv_bfloat16>(dev, a, dt, scratch) : launch_mass<__half>(dev, a, dt, scratch);
}

}  // namespace paged
