// Attention of few new tokens over paged caches: generation in f16 and bf16, and f32 of any length.  Heads of up to 128 features.
//
// An item is up to 16 (f32: 8) rows of queries - tokens with the heads of a group, one after the other - and a warp takes slices of 16 cached rows,
// which lie in one page, by itself: it asks for them by TMA into a ring of its own, three slices deep (f32: one to three, launch_rows), works out scores, weights and
// sums in registers, and meets the other warps only at the end of the item's part, where their maxima and sums are joined.  Nothing in between waits for
// another warp, so what bounds it is the memory: 64 bytes a row and feature pair are in flight on every SM all the time.
//   f16, bf16   both products by mma.sync m16n8k16: 16 rows do not fill a tile of the 5th-generation tensor cores, whose turn-around through tensor
//               memory took 2500 cycles for 128 rows here (tensor memory, softmax of one warp, tensor memory again) against 1300 that the memory needs;
//   f32         FMA: a lane has a cached row and four queries for the scores, four features of the values and all queries for the sum; bound by the chain of a
//               slice in a warp (1600 instructions with eight queries, two warps a scheduler, 45 % of the issue slots).
// 64 sequences of 100 to 8000 rows, 32 heads over 8, 128 features: bf16 191 us of 164 that the memory needs (5.6 TB/s), f16 the same; f32 402 us (5.3 TB/s).
// One token of one sequence of 1000 rows, 32 heads of 96 features: 15.3 us, of which the attention 11: items, then a chain of three slices, then the joins.
// Weights are rounded to the operands' type for the second product and taken against the maximum less 7 in f16, as in paged_attention_tc.cu; values that are masked and not
// finite are kept out the same way.  Every wait is bounded; a warp whose wait gave up goes through the motions, so that the CTA's barriers are met.
#include "paged_rows.cuh"
#include "paged_tc.cuh"

namespace paged {
namespace {

constexpr int kSlice = 16, W = 8, kPlanned = 256;          // rows of a slice; warps of a CTA; items that every CTA works out for itself

template <class T> struct Form {
    static constexpr int kRows = 16, kCols = 64;          // columns of 128 bytes
};
template <> struct Form<float> {
    static constexpr int kRows = 8, kCols = 32;
};

struct RowsArgs {
    AttendArgs a;
    Plan pl;
    int group, nb, eb;         // query heads of a kv head; 128-byte blocks of a key and of a value
    int plans;                 // the kernel works the items out itself (kPlanned at most), and leaves them for the next one
    float* scores;             // [T * H, MP * R]: scores in units of log 2, where mass is kept
};

template <class T> __device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// byte offset of 16-byte piece `c` of row r in a slice of 128-byte blocks, 128-byte swizzle
__device__ __forceinline__ uint32_t piece(int r, int c) { return (uint32_t)((c >> 3) * (kSlice * 128) + r * 128 + (((c ^ r) & 7) << 4)); }
__device__ __forceinline__ void ldsm4(uint32_t (&v)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&v)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
}
template <class T> __device__ __forceinline__ bool finite16(uint4 u) { return (not_finite<T>(u.x) | not_finite<T>(u.y) | not_finite<T>(u.z) | not_finite<T>(u.w)) == 0; }
template <> __device__ __forceinline__ bool finite16<float>(uint4 u) {
    auto bad = [](uint32_t x) { return (x & 0x7f800000u) == 0x7f800000u; };
    return !(bad(u.x) || bad(u.y) || bad(u.z) || bad(u.w));
}

// What one warp has of an item's rows.  16-bit types: lane holds rows lane / 4 and lane / 4 + 8, features 8 t + 2 (lane % 4) and the next.
template <class T> struct Part {
    uint32_t q[8][4];
    float o[16][4], m[2], l[2];

    __device__ __forceinline__ void begin(const RowsArgs& x, const T* q0, const T* q1) {      // the lane's two rows, nullable
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = 16 * k + 8 * (e >> 1) + 2 * (lane & 3);
                const T* row = e & 1 ? q1 : q0;
                q[k][e] = row && col < x.a.p.D ? *reinterpret_cast<const uint32_t*>(row + col) : 0u;
            }
#pragma unroll
        for (int t = 0; t < 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][e] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }
    // scores z of the slice's keys 8 t + 2 (lane % 4) + e: z[t][e] row lane / 4, z[t][2 + e] row lane / 4 + 8
    __device__ __forceinline__ void step(const RowsArgs& x, uint32_t ks, uint32_t vs, bool masked, int j, int pos0, int pos1, float* to0, float* to1) {
        const int lane = threadIdx.x & 31;
        const AttendArgs& a = x.a;
        float z[2][4] = {};
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (16 * k < a.p.D) {
                uint32_t b[4];
                ldsm4(b, ks + piece((lane & 7) + ((lane >> 4) & 1) * 8, 2 * k + ((lane >> 3) & 1)));
                mma16<T>(z[0], q[k], b[0], b[1]);
                mma16<T>(z[1], q[k], b[2], b[3]);
            }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                z[t][e] *= a.c;
                if (masked) {
                    const int r = e < 2 ? pos0 : pos1, at = j + 8 * t + 2 * (lane & 3) + (e & 1);
                    if (at > r || (a.window > 0 && at <= r - a.window && at >= a.first)) z[t][e] = -INFINITY;
                }
            }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (to0) *reinterpret_cast<float2*>(to0 + j + 8 * t + 2 * (lane & 3)) = make_float2(z[t][0], z[t][1]);
            if (to1) *reinterpret_cast<float2*>(to1 + j + 8 * t + 2 * (lane & 3)) = make_float2(z[t][2], z[t][3]);
        }
        float corr[2];
        bool moved = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float top = fmaxf(fmaxf(z[0][2 * h], z[0][2 * h + 1]), fmaxf(z[1][2 * h], z[1][2 * h + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) - Above<T>::value;
            // the maximum only moves when a score exceeds it by more than 2^8
            const bool move = top > m[h] + 8.f || (m[h] == -INFINITY && top > -INFINITY);
            corr[h] = move ? ex2(m[h] - top) : 1.f;
            if (move) m[h] = top;
            moved |= move;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int t = 0; t < 16; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t][e] *= corr[e >> 1];
        }
        uint32_t w[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float base = m[h] == -INFINITY ? 0.f : m[h];
            float u[4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) u[2 * t + e] = ex2(z[t][2 * h + e] - base);
            l[h] = l[h] * corr[h] + ((u[0] + u[1]) + (u[2] + u[3]));
            w[h] = pack2<T>(u[0], u[1]);
            w[2 + h] = pack2<T>(u[2], u[3]);
        }
#pragma unroll
        for (int t = 0; t < 8; ++t)
            if (16 * t < a.p.E) {
                uint32_t b[4];
                ldsm4_t(b, vs + piece((lane & 7) + ((lane >> 3) & 1) * 8, 2 * t + (lane >> 4)));
                mma16<T>(o[2 * t], w, b[0], b[1]);
                mma16<T>(o[2 * t + 1], w, b[2], b[3]);
            }
    }
    // maxima and sums of the warp's rows; its sum of values as [rows][E]
    __device__ __forceinline__ void end(float2* ml, float* sums, int E) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if ((lane & 3) == 0) ml[(lane >> 2) + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
            for (int t = 0; t < 16; ++t)
                if (8 * t < E) *reinterpret_cast<float2*>(sums + ((lane >> 2) + 8 * h) * E + 8 * t + 2 * (lane & 3)) = make_float2(o[t][2 * h], o[t][2 * h + 1]);
        }
    }
};

// f32: for the scores lane has cached row lane % 16 of the slice and queries 4 (lane / 16) .. + 3, for the sum features 4 lane .. + 3 of all queries.
// With FEW, up to four queries: a cached row's two lanes have half of its features each, and the same four queries: 64 sequences of 32 heads over 8,
// 128 features 488 -> 403 us, 64 features 351 -> 309; items of eight rows pay 2.8 % for the longer kernel (64 heads over 8: 486 -> 500).
template <> struct Part<float> {
    float4 o[8];
    float m[4], l[4];

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int r = 0; r < 8; ++r) o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
    }
    // pos: rows of the lane's queries' tokens (-1: none); qs: the item's queries [8][128]; own: [16][8] weights and [8] factors of the warp's own
    template <bool FEW>
    __device__ __forceinline__ void step(const RowsArgs& x, const unsigned char* ks, const unsigned char* vs, bool masked, int j, const int (&pos)[4], float* const (&to)[4],
                                         const float* qs, float* own) {
        const AttendArgs& a = x.a;
        const int lane = threadIdx.x & 31, key = lane & 15, rg = lane >> 4;
        float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 16
        for (int i = 0; i < a.p.D / (FEW ? 8 : 4); ++i) {
            const int c = FEW ? 2 * i + rg : i;
            const float4 k = *reinterpret_cast<const float4*>(ks + piece(key, c));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 q = *reinterpret_cast<const float4*>(qs + (FEW ? r : 4 * rg + r) * 128 + 4 * c);
                z[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, z[r]))));
            }
        }
        bool moved = false;
        float corr[4], u[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (FEW) z[r] += __shfl_xor_sync(0xffffffffu, z[r], 16);
            z[r] *= a.c;
            const int at = j + key;
            if (masked && (at > pos[r] || (a.window > 0 && at <= pos[r] - a.window && at >= a.first))) z[r] = -INFINITY;
            if (to[r]) to[r][at] = z[r];
            float top = z[r];
#pragma unroll
            for (int s = 1; s < 16; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
            const float next = fmaxf(m[r], top), base = next == -INFINITY ? 0.f : next;
            corr[r] = exp2f(m[r] - base);
            moved |= next > m[r];
            m[r] = next;
            u[r] = exp2f(z[r] - base);
            l[r] = l[r] * corr[r] + u[r];
        }
        *reinterpret_cast<float4*>(own + key * 8 + 4 * rg) = make_float4(u[0], u[1], u[2], u[3]);
        const bool scale = __any_sync(0xffffffffu, moved);
        if (scale && key == 0) *reinterpret_cast<float4*>(own + 128 + 4 * rg) = make_float4(corr[0], corr[1], corr[2], corr[3]);
        __syncwarp();
        if (scale) {
            const float4 c0 = *reinterpret_cast<const float4*>(own + 128), c1 = *reinterpret_cast<const float4*>(own + 132);
            const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
            for (int r = 0; r < (FEW ? 4 : 8); ++r) o[r] = make_float4(o[r].x * c[r], o[r].y * c[r], o[r].z * c[r], o[r].w * c[r]);
        }
        if (4 * lane < a.p.E) {
#pragma unroll
            for (int k = 0; k < kSlice; ++k) {
                const float4 v = *reinterpret_cast<const float4*>(vs + piece(k, lane));
                const float4 p0 = *reinterpret_cast<const float4*>(own + k * 8), p1 = *reinterpret_cast<const float4*>(own + k * 8 + 4);
                const float w[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
#pragma unroll
                for (int r = 0; r < (FEW ? 4 : 8); ++r) o[r] = make_float4(fmaf(w[r], v.x, o[r].x), fmaf(w[r], v.y, o[r].y), fmaf(w[r], v.z, o[r].z), fmaf(w[r], v.w, o[r].w));
            }
        }
        __syncwarp();
    }
    __device__ __forceinline__ void end(float2* ml, float* sums, int E) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int s = 1; s < 16; s <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], s);
            if ((lane & 15) == 0) ml[4 * (lane >> 4) + r] = make_float2(m[r], l[r]);
        }
        if (4 * lane < E)
#pragma unroll
            for (int r = 0; r < 8; ++r) *reinterpret_cast<float4*>(sums + r * E + 4 * lane) = o[r];
    }
};

template <class T, int kRing>
__global__ void __launch_bounds__(W * 32, 1)
rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ RowsArgs x) {
    constexpr int BQ = Form<T>::kRows, C = Form<T>::kCols;
    constexpr bool f32 = sizeof(T) == 4;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) uint64_t full[W][kRing];
    __shared__ __align__(16) float qs[f32 ? BQ * 128 : 4], own[f32 ? W : 1][136];
    __shared__ float2 ml[W][BQ];
    __shared__ volatile int abort_flag, poison[2];          // a note per item's part, in turns
    const AttendArgs& a = x.a;
    const View& p = a.p;
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kbytes = x.nb * kSlice * 128, slot_bytes = kbytes + x.eb * kSlice * 128;
    unsigned char* ring = base + (size_t)warp * kRing * slot_bytes;
    if (threadIdx.x == 0) {
        for (int i = 0; i < W * kRing; ++i) mbar_init(&full[0][i], 1);
        abort_flag = 0;
        poison[0] = poison[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    rcu_kernel_entry_wait_only();          // nothing before this touches global memory
    // Few items (one per thread) are worked out by every CTA for itself: with a kernel of one CTA in front, one token of one sequence takes 18.1 us for 15.4,
    // 64 sequences 190.2 for 187.0.  Beyond that the steps of a CTA's plan are as long for each of them as for the one.
    __shared__ int starts[kPlanned], prefix[kPlanned + 1], head[2];
    __shared__ Item items[kPlanned];
    Plan pl = x.pl;
    if (x.plans) {
        pl.head = head;
        pl.prefix = prefix;
        pl.item = items;
        plan_items_block<W * 32>(p, pl, a.window, a.first, x.group, starts);
        if (blockIdx.x == 0) {
            for (int s = threadIdx.x; s < p.S; s += W * 32)
                if (seq_bad(p, s)) report_bad(p.status);
            for (int i = threadIdx.x; i <= pl.items; i += W * 32) {
                x.pl.prefix[i] = prefix[i];
                if (i < pl.items) x.pl.item[i] = items[i];
                if (i < 2) x.pl.head[i] = head[i];
            }
        }
    }
    bool ok = true;
    int asked = 0, had = 0, turn = 0;      // slices so far; parity of the part
#pragma unroll 1
    for (Walk wk(pl, blockIdx.x, p.G, pl.items); wk.more(); wk.next(), turn ^= 1) {
        // rows f0 .. f0 + count - 1 of the sequence's queries: token f / group, head f % group
        const Seq sq = seq_of(p, wk.it.s);
        const int f0 = wk.it.token, count = wk.it.count, g = wk.g, s = wk.it.s;
        const int r0 = wk.it.row, r1 = sq.old() + (f0 + count - 1) / x.group, L = sq.L;
        const Span sp = span_of(a.window, a.first, r0, r1);
        const int end = min(L, r1 + 1), slices = (wk.n1 - wk.n0) * (kTileK / kSlice / W);
        auto slice_at = [&](int i) { return sp.tile(wk.n0 + i / (kTileK / kSlice / W)) * kTileK + (i % (kTileK / kSlice / W) * W + warp) * kSlice; };
        PageIds ids;
        const int have = min(p.MP, (L + p.R - 1) >> p.shift);
        auto ask = [&](int i) {
            const int j = slice_at(i);
            if (j >= end || !ok) return;
            const int at = j >> p.shift, page = ids.of(p, s, at, at, at, have), st = asked % kRing;
            if (lane == 0) {
                unsigned char* to = ring + st * slot_bytes;
                mbar_expect_tx(&full[warp][st], slot_bytes);
                for (int b = 0; b < x.nb; ++b) tma_load_4d(to + b * kSlice * 128, &kmap, b * C, j & (p.R - 1), g, page, &full[warp][st]);
                for (int b = 0; b < x.eb; ++b) tma_load_4d(to + kbytes + b * kSlice * 128, &vmap, b * C, j & (p.R - 1), g, page, &full[warp][st]);
            }
            ++asked;
        };
#pragma unroll 1
        for (int i = 0; i < kRing - 1 && i < slices; ++i) ask(i);

        Part<T> part;
        const size_t H = a.H;
        auto query = [&](int u) { return ((size_t)(sq.start + (f0 + u) / x.group) * H + (size_t)g * x.group + (f0 + u) % x.group); };      // place of the item's row u
        auto row_of = [&](int u) { return sq.old() + (f0 + u) / x.group; };
        const size_t room = (size_t)p.MP << p.shift;
        int pos[4];
        float* to[4] = {nullptr, nullptr, nullptr, nullptr};
        if constexpr (f32) {
            for (int i = threadIdx.x; i < BQ * 32; i += W * 32) {
                const int u = i >> 5, c = i & 31;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (u < count && 4 * c < p.D) v = *reinterpret_cast<const float4*>((const float*)a.q + query(u) * p.D + 4 * c);
                *reinterpret_cast<float4*>(qs + u * 128 + 4 * c) = v;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int u = (count > 4 ? 4 * (lane >> 4) : 0) + r;
                pos[r] = u < count ? row_of(u) : -1;
                if (x.scores && u < count && (count > 4 || lane < 16)) to[r] = x.scores + query(u) * room;
            }
            part.begin();
            __syncthreads();
        } else {
            const int u0 = lane >> 2, u1 = u0 + 8;
            pos[0] = u0 < count ? row_of(u0) : -1;
            pos[1] = u1 < count ? row_of(u1) : -1;
            if (x.scores && u0 < count) to[0] = x.scores + query(u0) * room;
            if (x.scores && u1 < count) to[1] = x.scores + query(u1) * room;
            part.begin(x, u0 < count ? (const T*)a.q + query(u0) * p.D : nullptr, u1 < count ? (const T*)a.q + query(u1) * p.D : nullptr);
        }
#pragma unroll 1
        for (int i = 0; i < slices; ++i) {
            if (i + kRing - 1 < slices) ask(i + kRing - 1);
            const int j = slice_at(i);
            if (j >= end) continue;
            const int st = had % kRing;
            if (ok) {
                ok = wait_warp(&full[warp][st], had / kRing, &abort_flag, p.status);
                if (!ok)                   // given up: let the copies in flight land before the memory is somebody else's
                    for (int k = had; k < asked; ++k) land(&full[warp][k % kRing], k / kRing);
            }
            ++had;
            if (!ok) continue;
            unsigned char *ks = ring + st * slot_bytes, *vs = ks + kbytes;
            // a slice that is not whole to all queries: rows behind the last one become zero, values that are not finite are noted
            const bool masked = j + kSlice - 1 > r0 || count < BQ || (a.window > 0 && j <= r1 - a.window && j + kSlice > a.first);
            if (j + kSlice - 1 > r0 || (a.window > 0 && j <= r1 - a.window && j + kSlice > a.first)) {
                bool bad = false;
                for (int c = lane; c < kSlice * 8 * x.eb; c += 32) {
                    uint4* at = reinterpret_cast<uint4*>(vs + c * 16);
                    if (j + (c >> 3) % kSlice >= L) *at = make_uint4(0, 0, 0, 0);
                    else bad |= !finite16<T>(*at);
                }
                if (bad) poison[turn] = 1;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            if constexpr (f32) {
                if (count > 4) part.template step<false>(x, ks, vs, masked, j, pos, to, qs, own[warp]);
                else part.template step<true>(x, ks, vs, masked, j, pos, to, qs, own[warp]);
            } else part.step(x, smem_u32(ks), smem_u32(vs), masked, j, pos[0], pos[1], to[0], to[1]);
            __syncwarp();
        }
        // the warps' maxima and sums
        __syncthreads();
        float* sums = reinterpret_cast<float*>(base);
        part.end(ml[warp], sums + (size_t)warp * BQ * p.E, p.E);
        __syncthreads();
        const int slot = wk.slot(blockIdx.x);
        if (threadIdx.x == 0) poison[turn ^ 1] = 0;
        if (poison[turn]) {
            for (int u = warp; u < count; u += W) {
                const int t = sq.start + (f0 + u) / x.group, h = g * x.group + (f0 + u) % x.group;
                RowPart row;
                attend_row<T>(a, s, g, t, h, row_of(u), sp, wk.n0, wk.n1, row);
                if (wk.whole) finish_row<T>(a, t, h, row);
                else store_part(x.pl, p.E, slot, u, row);
            }
        } else {
            const int quads = p.E / 4;
            for (int i = threadIdx.x; i < count * quads; i += W * 32) {
                const int u = i / quads, c = i - u * quads;
                float m = -INFINITY, l = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) m = fmaxf(m, ml[w][u].x);
                const size_t q = query(u);
                const float sk = wk.whole && a.sink ? a.sink[q % H] * kLog2e : -INFINITY, top = fmaxf(m, sk);
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float2 v = ml[w][u];
                    const float f = v.x == -INFINITY && v.y == 0.f ? 0.f : ex2(v.x - top);          // a warp that saw nothing has no sum
                    const float4 e = *reinterpret_cast<const float4*>(sums + ((size_t)w * BQ + u) * p.E + 4 * c);
                    l = fmaf(v.y, f, l);
                    o = make_float4(fmaf(e.x, f, o.x), fmaf(e.y, f, o.y), fmaf(e.z, f, o.z), fmaf(e.w, f, o.w));
                }
                if (wk.whole) {
                    if (a.sink) l += ex2(sk - top);
                    const float inv = 1.f / l;
                    T* out = (T*)a.out + q * p.E + 4 * c;
                    if constexpr (f32) *reinterpret_cast<float4*>(out) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
                    else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
                    if (a.lse && c == 0) a.lse[q] = top + log2f(l);
                } else {
                    x.pl.o[((size_t)slot * quads + c) * x.pl.stride + u] = o;
                    if (c == 0) x.pl.ml[(size_t)slot * x.pl.stride + u] = make_float2(m, l);
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");          // the sums lie where the next slices go
        __syncthreads();
    }
}

// As merge_kernel of paged_attention_tc.cu, for items of rows: the parts' factors first, in shared memory, then their sums
template <class T>
__global__ void __launch_bounds__(256) rows_merge_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ Plan pl, int group) {
    constexpr int BQ = Form<T>::kRows;
    rcu_kernel_entry();
    extern __shared__ float factor[];          // [parts][BQ]
    __shared__ float total[BQ];
    const View& p = a.p;
    const int b = blockIdx.x;
    const Join jn(pl, b, p.G, pl.items);
    if (jn.count == 0) return;
    const int start = clamp_int(p.starts[jn.it.s], 0, p.T), quads = p.E / 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int u = warp; u < jn.it.count; u += 8) {
        const int f = jn.it.token + u, h = jn.g * group + f % group;
        float m = a.sink ? a.sink[h] * kLog2e : -INFINITY;
        const float sk = m;
        for (int k = lane; k < jn.count; k += 32) m = fmaxf(m, pl.ml[(size_t)jn.slot(b, k) * pl.stride + u].x);
        m = warp_max(m);
        float l = 0.f;
        for (int k = lane; k < jn.count; k += 32) {
            const float2 ml = pl.ml[(size_t)jn.slot(b, k) * pl.stride + u];
            const float w = ml.x == -INFINITY && ml.y == 0.f ? 0.f : ex2(ml.x - m);          // a part that sees nothing has no sum
            factor[k * BQ + u] = w;
            l = fmaf(ml.y, w, l);
        }
        l = warp_sum(l) + (a.sink ? ex2(sk - m) : 0.f);
        if (lane == 0) {
            total[u] = 1.f / l;
            if (a.lse) a.lse[(size_t)(start + f / group) * a.H + h] = m + log2f(l);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < jn.it.count * quads; i += 256) {
        const int u = i % jn.it.count, c = i / jn.it.count, f = jn.it.token + u, h = jn.g * group + f % group;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int k = 0; k < jn.count; ++k) {
            const float4 v = pl.o[((size_t)jn.slot(b, k) * quads + c) * pl.stride + u];
            const float w = factor[k * BQ + u];
            o = make_float4(fmaf(v.x, w, o.x), fmaf(v.y, w, o.y), fmaf(v.z, w, o.z), fmaf(v.w, w, o.w));
        }
        const float inv = total[u];
        T* out = (T*)a.out + ((size_t)(start + f / group) * a.H + h) * p.E + 4 * c;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
    }
}

// The weights that a row receives, from the scores that rows_kernel has left: a thread per row, tokens and heads in their order.
__global__ void __launch_bounds__(256) scores_mass_kernel(const __grid_constant__ AttendArgs a, const float* __restrict__ scores, int group) {
    rcu_kernel_entry();
    const View& p = a.p;
    const int s = blockIdx.y / p.G, g = blockIdx.y % p.G;
    const Seq q = seq_of(p, s);
    const size_t room = (size_t)p.MP << p.shift;
    for (int j = blockIdx.x * 1024 + threadIdx.x; j < min(q.L, (int)blockIdx.x * 1024 + 1024); j += 256) {
        float sum = 0.f;
        for (int t = 0; t < q.n; ++t) {
            const int r = q.old() + t;
            if (j > r || (a.window > 0 && j <= r - a.window && j >= a.first)) continue;
            const size_t at = (size_t)(q.start + t) * a.H + g * group;
#pragma unroll 4
            for (int h = 0; h < group; ++h) sum += ex2(__ldcs(scores + (at + h) * room + j) - a.lse[at + h]);
        }
        if (q.n > 0) p.mass[((size_t)s * p.G + g) * room + j] += sum;
    }
}

uint64_t rows_plan_of(const rcu_device* dev, const View& p, int H, int dt, char* mem, Plan* out, float** scores) {
    const int group = H / p.G, bq = dt == RCU_F32 ? Form<float>::kRows : Form<__half>::kRows;
    Plan pl{};
    pl.tokens = bq;
    pl.items = (int)((uint64_t)p.T * group / bq) + p.S;
    pl.ctas = dev->sm_count;
    pl.least = 1;
    pl.extra = 1;
    pl.stride = bq;
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
    float* z = (float*)mem;
    if (p.mass) z = (float*)take(4ull * p.T * H * ((uint64_t)p.MP << p.shift));
    if (out) *out = pl;
    if (scores) *scores = z;
    return at;
}

template <class T> rcu_status launch_rows(rcu_device* dev, const AttendArgs& a, int dt, void* scratch) {
    const View& p = a.p;
    constexpr int C = Form<T>::kCols;
    RowsArgs x{a, {}, a.H / p.G, (p.D + C - 1) / C, (p.E + C - 1) / C, 0, nullptr};
    rows_plan_of(dev, p, a.H, dt, (char*)scratch, &x.pl, &x.scores);
    if (!p.mass) x.scores = nullptr;
    CUtensorMap km, vm;
    if (!map_slices(&km, dt, p, p.keys, p.D, kSlice) || !map_slices(&vm, dt, p, p.values, p.E, kSlice))
        return rcu_fail(dev, RCU_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled failed (%d tokens, %d heads, %d pages)", p.T, a.H, p.pages);
    x.plans = x.pl.items <= kPlanned && p.S <= kPlanned;
    if (!x.plans) {
        const rcu_status st = plan_items(dev, p, x.pl, a.window, a.first, x.group);
        if (st != RCU_OK) return st;
    }
    // Rings three slices deep, which always fit in 16 bits; in f32 as deep as shared memory allows.  Eight warps with a ring of one or two slices are faster than
    // four with three: 64 sequences of up to 8000 rows, 128 features 542 us against 744, 96 features 431 against 651.
    const size_t slots = (size_t)W * (x.nb + x.eb) * kSlice * 128, sums = (size_t)W * Form<T>::kRows * p.E * 4;
    const int ring = 3 * slots <= 192 * 1024 ? 3 : 2 * slots <= 192 * 1024 ? 2 : 1;
    const size_t smem = 1024 + (ring * slots > sums ? ring * slots : sums);
    constexpr bool f32 = sizeof(T) == 4;
    void (*kern)(CUtensorMap, CUtensorMap, RowsArgs) = ring == 3 ? rows_kernel<T, 3> : ring == 2 ? rows_kernel<T, f32 ? 2 : 3> : rows_kernel<T, f32 ? 1 : 3>;
    RCU_CUDA(dev, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    RCU_CUDA(dev, rcu_launch(dev, kern, x.pl.ctas, W * 32, smem, km, vm, x));
    RCU_LAUNCH_CHECK(dev);
    if (x.pl.ctas > 1) {
        rcu_launch(dev, rows_merge_kernel<T>, x.pl.ctas - 1, 256, (size_t)x.pl.ctas * Form<T>::kRows * 4, a, x.pl, x.group);
        RCU_LAUNCH_CHECK(dev);
    }
    if (p.mass) {
        rcu_launch(dev, scores_mass_kernel, dim3((unsigned)((((uint64_t)p.MP << p.shift) + 1023) / 1024), p.S * p.G), 256, 0, a, x.scores, x.group);
        RCU_LAUNCH_CHECK(dev);
    }
    return RCU_OK;
}

}  // namespace

bool attend_rows_takes(const rcu_device* dev, const View& p, int H, int dt) {
    if (p.D > 128 || p.E > 128 || dev->smem_optin < 227 * 1024) return false;
    const int group = H / p.G;
    // 16-bit: as long as the sequences bring 16 rows or less on average.  One call has one kernel: which sequence brings how many is known on the device alone.
    // This kernel against the tensor cores', 64 sequences of up to 8000 rows, 8 kv heads: 8 rows 189 us / 213, 16 rows 201 / 228, 32 rows 380 / 225;
    // up to 500 rows long: 16 rows 53 / 66, 32 rows 84 / 55; one sequence of 131000: 16 rows 105 / 120, 32 rows 182 / 120; one of 1000 rows: 16 rows 18.0 / 22.0,
    // 32 rows 18.5 / 21.3 (the only place on the far side where this one leads).
    // All of these have sequences that bring the same; what the average hides is dear: one chunk of 769 tokens behind 16000 rows among 255 single tokens behind 500, four
    // heads a group, takes 2640 us here, where the chunk by itself takes 251 and the others 154 (65 tokens behind 131000 rows, eight heads: 2734 and 418).
    if (dt != RCU_F32 && (uint64_t)p.T * group > 16ull * p.S) return false;
    if (((uint64_t)p.T * group / 8 + p.S) * (((uint64_t)p.MP << p.shift) / kTileK + 2) * p.G >= (1ull << 31)) return false;
    // The scores: half a GB, by the table's width, since the host knows no lengths.  f32 beyond it has the plain kernels alone: 64 sequences of 500 rows, 32 heads over 8,
    // 64 features, in tables of 65536 rows 107 us, of 131072 rows 1431.
    return !p.mass || (uint64_t)p.T * H * ((uint64_t)p.MP << p.shift) <= (1ull << 27);
}

uint64_t attend_rows_scratch(const rcu_device* dev, const View& p, int H, int dt) { return rows_plan_of(dev, p, H, dt, nullptr, nullptr, nullptr); }

rcu_status attend_rows(rcu_device* dev, const AttendArgs& a, int dt, void* scratch) {
    return dt == RCU_F32 ? launch_rows<float>(dev, a, dt, scratch) : dt == RCU_F16 ? launch_rows<__half>(dev, a, dt, scratch) : launch_rows<__nv_bfloat16>(dev, a, dt, scratch);
}

}  // namespace paged
