// What writes and shrinks a paged cache: rows of new tokens into their pages (rcu_paged_append), and the eviction of rows that received
// little attention (rcu_paged_evict).
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace paged {

rcu_status view(rcu_device* dev, const char* op, const rcu_paged* c, uint64_t tokens, bool starts, View* out) {
    RCU_REQUIRE(dev, c && t_valid(&c->keys) && t_valid(&c->values) && t_valid(&c->table) && t_valid(&c->lengths) && (!starts || t_valid(&c->starts)),
                "%s: invalid tensor descriptor", op);
    const rcu_tensor &k = c->keys, &v = c->values;
    RCU_REQUIRE(dev, k.rank == 4 && v.rank == 4 && k.dt == v.dt && dt_is_float(k.dt) && k.shape[0] == v.shape[0] && k.shape[1] == v.shape[1] && k.shape[2] == v.shape[2],
                "%s: keys and values are float [pages, kv_heads, page_rows, features] of one dtype", op);
    const uint64_t P = k.shape[0], G = k.shape[1], R = k.shape[2], D = k.shape[3], E = v.shape[3];
    RCU_REQUIRE(dev, P >= 1 && P < (1ull << 31) && G >= 1 && G <= 65535, "%s: %llu pages of %llu kv heads", op, (unsigned long long)P, (unsigned long long)G);
    RCU_REQUIRE(dev, R >= 16 && R <= 1024 && (R & (R - 1)) == 0, "%s: pages of %llu rows (a power of two, 16 to 1024)", op, (unsigned long long)R);
    if (D < 8 || D % 8 || D > 256 || E < 8 || E % 8 || E > 256)
        return rcu_fail(dev, RCU_ERR_UNSUPPORTED, "%s: heads of %llu and %llu features (multiples of 8, at most 256)", op, (unsigned long long)D, (unsigned long long)E);
    RCU_REQUIRE(dev, ((reinterpret_cast<uintptr_t>(k.data) | reinterpret_cast<uintptr_t>(v.data)) & 15) == 0, "%s: pages start on 16 bytes", op);
    RCU_REQUIRE(dev, c->table.dt == RCU_I32 && c->table.rank == 2 && c->lengths.dt == RCU_I32, "%s: the table is i32 [sequences, max_pages], lengths are i32", op);
    const uint64_t S = c->table.shape[0], MP = c->table.shape[1];
    RCU_REQUIRE(dev, S >= 1 && S <= (1u << 20) && MP >= 1 && MP * R <= (1ull << 29), "%s: %llu sequences of up to %llu pages", op, (unsigned long long)S, (unsigned long long)MP);
    RCU_REQUIRE(dev, t_numel(&c->lengths) == S, "%s: one length per sequence", op);
    if (starts) RCU_REQUIRE(dev, c->starts.dt == RCU_I32 && t_numel(&c->starts) == S + 1, "%s: starts are i32 [sequences + 1]", op);
    RCU_REQUIRE(dev, tokens <= (1ull << 29), "%s: %llu tokens", op, (unsigned long long)tokens);
    const bool mass = c->mass.data != nullptr;
    if (mass)
        RCU_REQUIRE(dev, c->mass.dt == RCU_F32 && c->mass.rank == 3 && c->mass.shape[0] == S && c->mass.shape[1] == G && c->mass.shape[2] == MP * R,
                    "%s: mass is f32 [sequences, kv_heads, max_pages * page_rows]", op);
    int shift = 4;
    while ((1u << shift) < R) ++shift;
    *out = View{k.data, v.data, (const int*)c->table.data, starts ? (const int*)c->starts.data : nullptr, (const int*)c->lengths.data,
                mass ? (float*)c->mass.data : nullptr, (int)S, (int)MP, (int)P, (int)G, (int)R, shift, (int)D, (int)E, (int)tokens, dev->d_status};
    return RCU_OK;
}

rcu_status Scratch::take(const char* op, const rcu_tensor* given, uint64_t bytes) {
    if (bytes == 0) return RCU_OK;
    if (given) {
        RCU_REQUIRE(dev, t_valid(given) && rcu_dtype_nbytes(given->dt, t_numel(given)) >= bytes && (reinterpret_cast<uintptr_t>(given->data) & 255) == 0,
                    "%s: the scratch needs %llu bytes on a 256-byte boundary", op, (unsigned long long)bytes);
        ptr = given->data;
        return RCU_OK;
    }
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    RCU_CUDA(dev, cudaStreamIsCapturing(dev->stream, &capture));
    RCU_REQUIRE(dev, capture == cudaStreamCaptureStatusNone, "%s: a captured call takes its scratch from the caller", op);
    const rcu_status st = rcu_alloc(dev, bytes, &ptr);
    pooled = st == RCU_OK;
    return st;
}

}  // namespace paged

namespace {

using namespace paged;

// ------------------------------------------------------------------------------------------------ append
// A CTA per token: its sequence, then its row's units of keys and of values.  Reads and writes 2 G (D + E) elements per token, bound by
// memory for prompts (8 heads of 128, bf16, seven prompts of up to 1700 tokens: 14.2 us, 5.0 TB/s) and by the launch for single tokens (96 of them 3.9 us).
template <class Unit>
__global__ void __launch_bounds__(128) append_kernel(const View p, const Unit* __restrict__ k, long long k_pitch, const Unit* __restrict__ v, long long v_pitch,
                                                     int du, int eu, int* lengths_out) {
    rcu_kernel_entry();
    const int t = blockIdx.x;
    if (t == 0) {
        for (int s = threadIdx.x; s < p.S; s += 128) {
            if (seq_bad(p, s)) report_bad(p.status);
            if (lengths_out) lengths_out[s] = p.lengths[s];
        }
        if (p.T == 0) return;
    }
    // the row's first units are on their way while its place is found
    const Unit *ks = k + t * k_pitch, *vs = v + t * v_pitch;
    constexpr int kAhead = 2;
    const int kn = p.G * du, vn = p.G * eu;
    Unit kb[kAhead], vb[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
        const int i = threadIdx.x + 128 * j;
        if (i < kn) kb[j] = ks[i];
        if (i < vn) vb[j] = vs[i];
    }
    const int s = seq_of_token(p, t);
    if (s < 0) return;
    const Seq q = seq_of(p, s);
    const int r = q.old() + t - q.start;
    if (r < 0 || r >= p.MP << p.shift) return;         // a reported length
    const int page = page_of(p, s, r), at = r & (p.R - 1);
    Unit* kd = const_cast<Unit*>(reinterpret_cast<const Unit*>(p.keys)) + ((size_t)page * p.G * p.R + at) * du;
    Unit* vd = const_cast<Unit*>(reinterpret_cast<const Unit*>(p.values)) + ((size_t)page * p.G * p.R + at) * eu;
    auto put = [&](Unit* to, int i, int units, const Unit& value) { to[(size_t)(i / units) * p.R * units + i % units] = value; };
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
        const int i = threadIdx.x + 128 * j;
        if (i < kn) put(kd, i, du, kb[j]);
        if (i < vn) put(vd, i, eu, vb[j]);
    }
#pragma unroll 4
    for (int i = threadIdx.x + 128 * kAhead; i < kn; i += 128) put(kd, i, du, ks[i]);
#pragma unroll 4
    for (int i = threadIdx.x + 128 * kAhead; i < vn; i += 128) put(vd, i, eu, vs[i]);
    if (p.mass)
        for (int g = threadIdx.x; g < p.G; g += 128) p.mass[((size_t)s * p.G + g) * ((size_t)p.MP << p.shift) + r] = 0.f;
}

template <class Unit>
void launch_append(rcu_device* dev, const View& p, const void* k, uint64_t k_pitch, const void* v, uint64_t v_pitch, size_t e, int* lengths_out) {
    const size_t n = sizeof(Unit) / e;                 // elements of a unit
    rcu_launch(dev, append_kernel<Unit>, (unsigned)max(1, p.T), 128, 0, p, (const Unit*)k, (long long)(k_pitch / n), (const Unit*)v, (long long)(v_pitch / n),
               (int)(p.D / n), (int)(p.E / n), lengths_out);
}

// ------------------------------------------------------------------------------------------------ eviction
// A cluster of CTAs per (sequence, kv head).
//   1. The K = keep - first - recent largest of the masses between: a radix select over the four bytes of an order-preserving code.  Every CTA
//      counts the digits of its run of rows, whose codes it keeps in shared memory (with the masses read again in each pass the selection of 4096 of 16000
//      rows took 85 us), the counts are added up over distributed shared memory.
//   2. Places: a row stays when its code is above the threshold or is one of the first `need` that equal it; runs of rows are numbered in
//      order, so the list of what stays is ascending and the same in every call.
//   3. In place: rows in order of their new places, as many per round as the cluster's registers hold: read, wait for the cluster, write.  A row's new
//      place is never behind its old one, so what a round writes has been read in it or before.  Into other arrays: a kernel behind this one, in
//      which nobody waits (in rounds the copy of 4096 rows of 16 sequences by 8 heads took 130 us, 4.1 TB/s).
// Bound by memory: the masses, then 2 keep (D + E) elements.  4096 of up to 16000 rows, 16 sequences, 8 heads, bf16, 128 features: 132 us, of which the selection 40 (four
// passes with a barrier of the cluster each), the copy 92 at 6.0 TB/s; 1000 of 2048 rows of one sequence 18.6 us.  In place, where the copy goes in rounds: 220 us for 132.
// 64 registers a thread keep four CTAs on an SM and spill 40 bytes.
constexpr int kEvictThreads = 256, kEvictUnits = 8, kEvictCluster = 8, kEvictCodes = 6144;

struct EvictArgs {
    View src, dst;
    int* lengths_out;
    unsigned* list;            // [S * G, middle]
    int keep, first, recent, ordered, in_place;       // in_place: the page arrays are the same
    int ku, vu;                // 16-byte units of a key and of a value
};

// larger masses have larger codes; NaN has the least, both zeros have one
__device__ __forceinline__ unsigned code_of(float m) {
    if (m != m) return 0u;
    const unsigned b = __float_as_uint(m == 0.f ? 0.f : m);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(kEvictThreads, 4) evict_kernel(const EvictArgs a) {
    rcu_kernel_entry();
    __shared__ unsigned hist[2][256], codes[kEvictCodes];          // codes of the first rows of the CTA's run; the others are made again each time
    __shared__ int total[256], warp_gt[16], warp_eq[16], counts[2], pick[2];
    __shared__ long long from[2][kEvictThreads], to[2][kEvictThreads];          // places of a round's rows, in turns
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int pair = blockIdx.x / C, s = pair / a.src.G, g = pair % a.src.G;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const View &p = a.src, &o = a.dst;
    const int given = p.lengths[s], L = clamp_int(given, 0, p.MP << p.shift);
    const int n = min(min(L, a.keep), o.MP << o.shift);
    const bool whole = L <= a.keep;
    if (rank == 0 && g == 0 && tid == 0) {
        if (given != L || n < min(L, a.keep)) report_bad(p.status);
        a.lengths_out[s] = n;
    }
    const float* mass = p.mass + ((size_t)s * p.G + g) * ((size_t)p.MP << p.shift);
    float* mass_to = o.mass + ((size_t)s * o.G + g) * ((size_t)o.MP << o.shift);
    const int middle = a.keep - a.first - a.recent;
    unsigned* list = a.list + (size_t)pair * middle;

    if (!whole && middle > 0) {
        const int lo = a.first, M = L - a.recent - lo;
        const int b0 = lo + (int)((long long)M * rank / C), b1 = lo + (int)((long long)M * (rank + 1) / C);
#pragma unroll 4
        for (int i = tid; i < min(b1 - b0, kEvictCodes); i += kEvictThreads) codes[i] = code_of(mass[b0 + i]);
        auto code_at = [&](int i) { return i - b0 < kEvictCodes ? codes[i - b0] : code_of(mass[i]); };
        unsigned prefix = 0;
        int left = middle;
        for (int d = 0; d < 4; ++d) {
            const int shift = 24 - 8 * d;
            unsigned* h = hist[d & 1];
            if (tid < 256) h[tid] = 0;
            __syncthreads();
            for (int i = b0 + tid; i < b0 + (b1 - b0 + 31) / 32 * 32; i += kEvictThreads) {       // whole warps
                const unsigned c = i < b1 ? code_at(i) : 0u;
                const bool in = i < b1 && (d == 0 || c >> (shift + 8) == prefix);
                const unsigned digit = in ? c >> shift & 255u : 256u;
                const unsigned same = __match_any_sync(0xffffffffu, digit);
                if (in && lane == __ffs(same) - 1) atomicAdd(&h[digit], __popc(same));
            }
            cluster.sync();
            if (tid < 256) {
                int sum = 0;
#pragma unroll
                for (int r = 0; r < kEvictCluster; ++r)            // all asked for at once: one after the other they took most of the selection's time
                    if (r < C) sum += (int)cluster.map_shared_rank(h, r)[tid];
                total[tid] = sum;
            }
            __syncthreads();
            if (warp == 0) {               // the digit of the left-th largest: lane l has digits 255 - 8 l .. 248 - 8 l
                int mine = 0;
                for (int j = 0; j < 8; ++j) mine += total[255 - 8 * lane - j];
                int upto = mine;
                for (int w = 1; w < 32; w <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, w);
                    if (lane >= w) upto += v;
                }
                int above = upto - mine;
                if (above < left && left <= upto) {
                    int digit = 255 - 8 * lane;
                    while (above + total[digit] < left) above += total[digit--];
                    pick[0] = digit;
                    pick[1] = above;
                }
            }
            __syncthreads();
            prefix = prefix << 8 | (unsigned)pick[0];
            left -= pick[1];
        }
        // `left` rows of code `prefix` stay, and every one above it
        auto flags = [&](int i, bool& gt, bool& eq) {
            const unsigned c = i < b1 ? code_at(i) : 0u;
            gt = i < b1 && c > prefix;
            eq = i < b1 && c == prefix;
        };
        if (tid < 2) counts[tid] = 0;
        __syncthreads();
        int gts = 0, eqs = 0;
        for (int i = b0 + tid; i < b1; i += kEvictThreads) {
            bool gt, eq;
            flags(i, gt, eq);
            gts += gt;
            eqs += eq;
        }
        gts = __reduce_add_sync(0xffffffffu, gts);
        eqs = __reduce_add_sync(0xffffffffu, eqs);
        if (lane == 0) {
            atomicAdd(&counts[0], gts);
            atomicAdd(&counts[1], eqs);
        }
        cluster.sync();
        int gt0 = 0, eq0 = 0;               // rows above / at the threshold before this place
#pragma unroll
        for (int r = 0; r < kEvictCluster; ++r)
            if (r < rank) {
                const int* c = cluster.map_shared_rank(counts, r);
                gt0 += c[0];
                eq0 += c[1];
            }
        for (int base = b0; base < b1; base += kEvictThreads) {
            bool gt, eq;
            flags(base + tid, gt, eq);
            const unsigned gm = __ballot_sync(0xffffffffu, gt), em = __ballot_sync(0xffffffffu, eq), below = (1u << lane) - 1;
            if (lane == 0) {
                warp_gt[warp] = __popc(gm);
                warp_eq[warp] = __popc(em);
            }
            __syncthreads();
            int gb = gt0 + __popc(gm & below), eb = eq0 + __popc(em & below);
#pragma unroll
            for (int w = 0; w < kEvictThreads / 32; ++w) {
                const int x = warp_gt[w], y = warp_eq[w];
                if (w < warp) {
                    gb += x;
                    eb += y;
                }
                gt0 += x;
                eq0 += y;
            }
            if (gt || (eq && eb < left)) list[gb + min(eb, left)] = (unsigned)(base + tid);
            __syncthreads();
        }
    }
    cluster.sync();                          // the list is complete, and nobody reads a mass or a neighbour's counts any more
    if (!a.ordered) return;                  // the rows go by move_kernel

    const int per_row = a.ku + a.vu, rows_cta = min(kEvictThreads, kEvictThreads * kEvictUnits / per_row);
    const uint4 *ks = (const uint4*)p.keys, *vs = (const uint4*)p.values;
    uint4 *kd = (uint4*)const_cast<void*>(o.keys), *vd = (uint4*)const_cast<void*>(o.values);
    // the rows of the round from `base` on; returns the mass of this thread's row
    auto find = [&](int base, int b) {
        const int d = base + rank * rows_cta + tid;
        if (tid >= rows_cta || d >= n) return 0.f;
        const int r = whole || d < a.first ? d : d >= a.keep - a.recent ? L - a.keep + d : (int)__ldcg(list + (d - a.first));
        from[b][tid] = (long long)((size_t)page_of(p, s, r) * p.G + g) * p.R + (r & (p.R - 1));
        to[b][tid] = (long long)((size_t)page_of(o, s, d) * o.G + g) * o.R + (d & (o.R - 1));
        return mass[r];
    };
    float m = find(0, 0);
    __syncthreads();
    for (int base = 0, b = 0; base < n; base += rows_cta * C, b ^= 1) {
        const int d0 = base + rank * rows_cta, rows = clamp_int(n - d0, 0, rows_cta);
        uint4 buf[kEvictUnits];
#pragma unroll
        for (int j = 0; j < kEvictUnits; ++j) {
            const int i = tid + j * kEvictThreads, row = i / per_row, u = i - row * per_row;
            if (row < rows && !(a.in_place && from[b][row] == to[b][row])) buf[j] = u < a.ku ? __ldcs(ks + from[b][row] * a.ku + u) : __ldcs(vs + from[b][row] * a.vu + (u - a.ku));
        }
        const float sum = m;
        if (a.ordered) cluster.sync();
        // where the next round's rows lie is found while this one's are on their way (what it reads lies behind what this round writes)
        m = find(base + rows_cta * C, b ^ 1);
#pragma unroll
        for (int j = 0; j < kEvictUnits; ++j) {
            const int i = tid + j * kEvictThreads, row = i / per_row, u = i - row * per_row;
            if (row < rows && !(a.in_place && from[b][row] == to[b][row])) {
                if (u < a.ku) kd[to[b][row] * a.ku + u] = buf[j];
                else vd[to[b][row] * a.vu + (u - a.ku)] = buf[j];
            }
        }
        if (tid < rows) mass_to[d0 + tid] = sum;
        __syncthreads();
    }
}

// The rows that stay into arrays that nobody reads: a warp takes kMoveRows of them, all asked for before the first is stored.
constexpr int kMoveRows = 4;
__global__ void __launch_bounds__(256) move_kernel(const __grid_constant__ EvictArgs a) {
    rcu_kernel_entry();
    const View &p = a.src, &o = a.dst;
    const int pair = blockIdx.y, s = pair / p.G, g = pair % p.G, lane = threadIdx.x & 31;
    const int L = clamp_int(p.lengths[s], 0, p.MP << p.shift), n = min(min(L, a.keep), o.MP << o.shift);
    const int d0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kMoveRows;
    if (d0 >= n) return;
    const float* mass = p.mass + ((size_t)s * p.G + g) * ((size_t)p.MP << p.shift);
    float* mass_to = o.mass + ((size_t)s * o.G + g) * ((size_t)o.MP << o.shift);
    const unsigned* list = a.list + (size_t)pair * (a.keep - a.first - a.recent);
    // lane i < kMoveRows finds row d0 + i
    long long from = 0, to = 0;
    if (lane < kMoveRows && d0 + lane < n) {
        const int d = d0 + lane, r = L <= a.keep || d < a.first ? d : d >= a.keep - a.recent ? L - a.keep + d : (int)list[d - a.first];
        from = (long long)((size_t)page_of(p, s, r) * p.G + g) * p.R + (r & (p.R - 1));
        to = (long long)((size_t)page_of(o, s, d) * o.G + g) * o.R + (d & (o.R - 1));
        mass_to[d] = mass[r];
    }
    const uint4 *ks = (const uint4*)p.keys, *vs = (const uint4*)p.values;
    uint4 *kd = (uint4*)const_cast<void*>(o.keys), *vd = (uint4*)const_cast<void*>(o.values);
    for (int u = lane; u < (a.ku + a.vu + 31) / 32 * 32; u += 32) {
        uint4 buf[kMoveRows];
        const bool in = u < a.ku + a.vu, key = u < a.ku;
#pragma unroll
        for (int i = 0; i < kMoveRows; ++i) {
            const long long f = __shfl_sync(0xffffffffu, from, i);
            if (in && d0 + i < n) buf[i] = key ? __ldcs(ks + f * a.ku + u) : __ldcs(vs + f * a.vu + (u - a.ku));
        }
#pragma unroll
        for (int i = 0; i < kMoveRows; ++i) {
            const long long t = __shfl_sync(0xffffffffu, to, i);
            if (in && d0 + i < n) {
                if (key) kd[t * a.ku + u] = buf[i];
                else vd[t * a.vu + (u - a.ku)] = buf[i];
            }
        }
    }
}

bool overlap(const void* a, uint64_t an, const void* b, uint64_t bn) {
    const char *x = (const char*)a, *y = (const char*)b;
    return x < y + bn && y < x + an;
}

}  // namespace

// rcu_paged_append that also leaves the lengths in lengths_out (nullable), for who has to come after it (graph.cu)
rcu_status rcu_paged_append_to(rcu_device* dev, const rcu_tensor* k, uint32_t k_col, const rcu_tensor* v, uint32_t v_col, const rcu_paged* cache, int* lengths_out) {
    RCU_REQUIRE(dev, t_valid(k) && t_valid(v) && k->rank == 2 && v->rank == 2 && k->shape[0] == v->shape[0], "paged_append: rows k and v of the same tokens");
    View p;
    const rcu_status st = view(dev, "paged_append", cache, k->shape[0], true, &p);
    if (st != RCU_OK) return st;
    RCU_REQUIRE(dev, k->dt == cache->keys.dt && v->dt == cache->keys.dt, "paged_append: rows of the pages' dtype");
    RCU_REQUIRE(dev, (uint64_t)k_col + (uint64_t)p.G * p.D <= k->shape[1] && (uint64_t)v_col + (uint64_t)p.G * p.E <= v->shape[1], "paged_append: the heads lie outside the rows");
    DevGuard guard(dev->ordinal);
    const size_t e = dt_esize(k->dt);
    const char *kp = (const char*)k->data + k_col * e, *vp = (const char*)v->data + v_col * e;
    const bool wide = ((reinterpret_cast<uintptr_t>(kp) | reinterpret_cast<uintptr_t>(vp) | k->shape[1] * e | v->shape[1] * e) & 15) == 0;
    if (wide) launch_append<uint4>(dev, p, kp, k->shape[1], vp, v->shape[1], e, lengths_out);
    else if (e == 4) launch_append<uint32_t>(dev, p, kp, k->shape[1], vp, v->shape[1], e, lengths_out);
    else launch_append<uint16_t>(dev, p, kp, k->shape[1], vp, v->shape[1], e, lengths_out);
    RCU_LAUNCH_CHECK(dev);
    return RCU_OK;
}

extern "C" {

rcu_status rcu_paged_append(rcu_device* dev, const rcu_tensor* k, uint32_t k_col, const rcu_tensor* v, uint32_t v_col, const rcu_paged* cache) {
    return dev ? rcu_paged_append_to(dev, k, k_col, v, v_col, cache, nullptr) : RCU_ERR_INVALID_ARG;
}

uint64_t rcu_paged_evict_scratch(rcu_device* dev, const rcu_paged* cache, uint32_t keep) {
    View p;
    if (!dev || view(dev, "paged_evict", cache, 0, false, &p) != RCU_OK) return 0;
    const uint64_t rows = (uint64_t)p.MP << p.shift;         // a sequence that is cut has more rows than it keeps
    return align256((uint64_t)p.S * p.G * (keep < rows ? keep : 0) * sizeof(unsigned));
}

rcu_status rcu_paged_evict(rcu_device* dev, const rcu_paged* cache, const rcu_paged* into, uint32_t keep, uint32_t first, uint32_t recent,
                           const rcu_tensor* scratch) {
    if (!dev) return RCU_ERR_INVALID_ARG;
    EvictArgs a{};
    rcu_status st = view(dev, "paged_evict", cache, 0, false, &a.src);
    if (st == RCU_OK) st = view(dev, "paged_evict", into, 0, false, &a.dst);
    if (st != RCU_OK) return st;
    const View &p = a.src, &o = a.dst;
    RCU_REQUIRE(dev, p.S == o.S && p.G == o.G && p.R == o.R && p.D == o.D && p.E == o.E && cache->keys.dt == into->keys.dt, "paged_evict: both caches have the same sequences, heads, pages and dtype");
    RCU_REQUIRE(dev, p.mass && o.mass, "paged_evict: needs the mass of both caches");
    const uint64_t rows = (uint64_t)p.MP << p.shift, room = (uint64_t)o.MP << o.shift;
    RCU_REQUIRE(dev, keep >= 1 && keep <= (1u << 30) && (uint64_t)first + recent <= keep, "paged_evict: %u first and %u recent rows of %u to keep", first, recent, keep);
    RCU_REQUIRE(dev, (keep < rows ? keep : rows) <= room, "paged_evict: the new tables hold %llu rows of %u to keep", (unsigned long long)room, keep);
    const size_t e = dt_esize(cache->keys.dt);
    RCU_REQUIRE(dev, !overlap(cache->lengths.data, 4ull * p.S, into->lengths.data, 4ull * p.S), "paged_evict: the new lengths lie over the old ones");
    RCU_REQUIRE(dev, p.mass == o.mass ? rows == room : !overlap(p.mass, 4ull * p.S * p.G * rows, o.mass, 4ull * o.S * o.G * room), "paged_evict: the masses overlap, but are not the same");
    auto meet = [&](const rcu_tensor& x, const rcu_tensor& y) { return overlap(x.data, t_numel(&x) * e, y.data, t_numel(&y) * e); };
    const bool ks = meet(cache->keys, into->keys), vs = meet(cache->values, into->values);
    RCU_REQUIRE(dev, (!ks || p.keys == o.keys) && (!vs || p.values == o.values) && !meet(cache->keys, into->values) && !meet(cache->values, into->keys),
                "paged_evict: the page arrays overlap, but are not the same");
    a.lengths_out = (int*)into->lengths.data;
    a.keep = (int)keep;
    a.first = (int)first;
    a.recent = (int)recent;
    a.ordered = ks || vs || p.mass == o.mass;
    a.in_place = ks && vs;
    a.ku = (int)(p.D * e / 16);
    a.vu = (int)(p.E * e / 16);
    DevGuard guard(dev->ordinal);
    Scratch list(dev);
    st = list.take("paged_evict", scratch, rcu_paged_evict_scratch(dev, cache, keep));
    if (st != RCU_OK) return st;
    a.list = (unsigned*)list.ptr;
    // clusters as large as four CTAs an SM allow, which is what fits: 16 sequences of up to 16000 rows by 8 heads 132 us (two 153, eight 140), of up to 5000 rows
    // 38.6 (41.9, 49.8); few sequences have clusters of eight in any case
    constexpr long long kPerSm = 4;
    const int pairs = p.S * p.G;
    int cluster = kEvictCluster;
    while (cluster > 1 && (long long)pairs * cluster > kPerSm * dev->sm_count) cluster /= 2;
    RCU_REQUIRE(dev, (long long)pairs * cluster <= 0x7fffffffll && (a.ordered || pairs <= 65535), "paged_evict: %d sequences of %d heads", p.S, p.G);
    const cudaError_t err = rcu_launch_cluster(dev, evict_kernel, (unsigned)(pairs * cluster), kEvictThreads, 0, cluster, a);
    if (err != cudaSuccess) return rcu_fail(dev, RCU_ERR_CUDA, "paged_evict: %s", cudaGetErrorString(err));
    RCU_LAUNCH_CHECK(dev);
    if (!a.ordered) {
        const uint64_t most = keep < rows ? keep : rows;
        rcu_launch(dev, move_kernel, dim3((unsigned)((most + 8 * kMoveRows - 1) / (8 * kMoveRows)), pairs), 256, 0, a);
        RCU_LAUNCH_CHECK(dev);
    }
    return RCU_OK;
}

}  // extern "C"
