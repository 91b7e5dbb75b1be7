// Attention of new tokens over paged caches (rcu_paged_attention): the call's checks, and the kernels that take any type, width and alignment.
//
//   o = sum_j p_j v_j,  p_j = 2^(c q.k_j - lse),  c = scale log2 e,  lse = log2 (sum_j 2^(c q.k_j) + 2^(sink log2 e))
//
// over the rows j that the token at row r sees: j <= r, and with a window j > r - window or j < first.
#include "paged_attention.cuh"
#include "paged_rows.cuh"

namespace {

using namespace paged;

// A warp per token and head, for what the other two kernels do not take; a lane reads keys element by element.  64 sequences of 4000 rows, 32 heads over 8 of 192
// features, bf16: 14.8 ms (of 128 features, on the other path, 0.19); a prompt of 1024 tokens 17.0 ms (0.05).
template <class T>
__global__ void __launch_bounds__(128) attend_kernel(const AttendArgs a) {
    rcu_kernel_entry();
    const View& p = a.p;
    if (blockIdx.x == 0)
        for (int s = threadIdx.x; s < p.S; s += 128)
            if (seq_bad(p, s)) report_bad(p.status);
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, t = (int)(item / a.H), h = (int)(item % a.H);
    if (t >= p.T) return;
    const int s = seq_of_token(p, t);
    if (s < 0) return;
    const Seq sq = seq_of(p, s);
    const int r = min(sq.old() + t - sq.start, sq.L - 1);
    RowPart part;
    const Span sp = span_of(a.window, a.first, r, r);
    attend_row<T>(a, s, h / (a.H / p.G), t, h, r, sp, 0, sp.count, part);
    finish_row<T>(a, t, h, part);
}

// A warp per 32 rows of a sequence and kv head, a lane for each row: the weights that its tokens and heads give, in their order.
template <class T>
__global__ void __launch_bounds__(128) mass_kernel(const AttendArgs a) {
    rcu_kernel_entry();
    const View& p = a.p;
    const int rows = p.MP << p.shift, lane = threadIdx.x & 31, per = a.H / p.G;
    const int g = blockIdx.y % p.G, s = blockIdx.y / p.G;
    const Seq sq = seq_of(p, s);
    const int j = (blockIdx.x * 4 + (threadIdx.x >> 5)) * 32 + lane;
    if (j >= sq.L) return;
    const T* k = (const T*)p.keys + row_at(p, page_of(p, s, j), g, j, p.D);
    float sum = 0.f;
    for (int i = 0; i < sq.n; ++i) {
        const int r = sq.old() + i;
        int head, low;
        visible(a.window, a.first, r, head, low);
        if (j > r || (j >= head && j < low)) continue;
        for (int h = g * per; h < (g + 1) * per; ++h) {
            const size_t at = (size_t)(sq.start + i) * a.H + h;
            const T* q = (const T*)a.q + at * p.D;
            float z = 0.f;
            for (int d = 0; d < p.D; ++d) z = fmaf(to_f32<T>(q[d]), to_f32<T>(k[d]), z);
            sum += exp2f(z * a.c - a.lse[at]);
        }
    }
    p.mass[((size_t)s * p.G + g) * rows + j] += sum;
}

template <class T> rcu_status attend(rcu_device* dev, const AttendArgs& a, int dt, void* scratch) {
    const View& p = a.p;
    // both paths take a scale above zero, and queries and output that start on 16 bytes
    const bool plain = !(a.c > 0.f) || !(a.c < INFINITY) || ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15) != 0;
    if (!plain && attend_rows_takes(dev, p, a.H, dt)) return attend_rows(dev, a, dt, scratch);
    if (!plain && attend_tc_takes(dev, p, a.H, dt)) {
        // the two run one after the other: they share the scratch
        const rcu_status st = attend_tc(dev, a, dt, scratch);
        return st != RCU_OK || !p.mass ? st : mass_tc(dev, a, dt, scratch);
    }
    const long long items = (long long)p.T * a.H;
    rcu_launch(dev, attend_kernel<T>, (unsigned)((items + 3) / 4), 128, 0, a);
    RCU_LAUNCH_CHECK(dev);
    if (p.mass) {
        rcu_launch(dev, mass_kernel<T>, dim3((unsigned)(((p.MP << p.shift) + 127) / 128), p.S * p.G), 128, 0, a);
        RCU_LAUNCH_CHECK(dev);
    }
    return RCU_OK;
}

// lse of every query where mass is kept, and behind it what the tensor-core path takes (whether a call goes there is decided by more than the sizes)
uint64_t lse_bytes(const View& p, uint64_t H) { return p.mass ? align256((uint64_t)p.T * H * 4) : 0; }
uint64_t scratch_bytes(const rcu_device* dev, const View& p, uint64_t H, int dt) {
    if (attend_rows_takes(dev, p, (int)H, dt)) return lse_bytes(p, H) + attend_rows_scratch(dev, p, (int)H, dt);
    if (!attend_tc_takes(dev, p, (int)H, dt)) return lse_bytes(p, H);
    const uint64_t attend = attend_tc_scratch(dev, p, (int)H), mass = p.mass ? mass_tc_scratch(dev, p, (int)H) : 0;
    return lse_bytes(p, H) + (attend > mass ? attend : mass);
}

}  // namespace

extern "C" {

uint64_t rcu_paged_attention_scratch(rcu_device* dev, const rcu_tensor* q, const rcu_paged* cache) {
    View p;
    if (!dev || !t_valid(q) || q->rank != 3 || view(dev, "paged_attention", cache, q->shape[0], true, &p) != RCU_OK) return 0;
    const uint64_t H = q->shape[1];
    return H >= (uint64_t)p.G && H % p.G == 0 && H <= 65535 ? scratch_bytes(dev, p, H, q->dt) : 0;
}

rcu_status rcu_paged_attention(rcu_device* dev, const rcu_tensor* q, const rcu_paged* cache, const rcu_tensor* sink, uint32_t window, uint32_t first,
                               float scale, const rcu_tensor* scratch, rcu_tensor* dst) {
    if (!dev) return RCU_ERR_INVALID_ARG;
    RCU_REQUIRE(dev, t_valid(q) && (!sink || t_valid(sink)) && t_valid(dst) && q->rank == 3, "paged_attention: q is [tokens, heads, dim]");
    AttendArgs a{};
    rcu_status st = view(dev, "paged_attention", cache, q->shape[0], true, &a.p);
    if (st != RCU_OK) return st;
    const View& p = a.p;
    const uint64_t T = q->shape[0], H = q->shape[1];
    RCU_REQUIRE(dev, q->dt == cache->keys.dt && dst->dt == q->dt && q->shape[2] == (uint64_t)p.D, "paged_attention: queries and output of the pages' dtype and width");
    RCU_REQUIRE(dev, H >= 1 && H % p.G == 0 && H <= 65535, "paged_attention: %llu query heads over %d kv heads", (unsigned long long)H, p.G);
    RCU_REQUIRE(dev, !sink || (sink->dt == RCU_F32 && t_numel(sink) == H), "paged_attention: one f32 sink per query head");
    RCU_REQUIRE(dev, t_numel(dst) == T * H * p.E, "paged_attention: dst holds %llu elements, expected %llu", (unsigned long long)t_numel(dst), (unsigned long long)(T * H * p.E));
    RCU_REQUIRE(dev, T * H < (1ull << 31) && (!p.mass || (uint64_t)p.S * p.G <= 65535), "paged_attention: %llu tokens of %llu heads, %d sequences", (unsigned long long)T,
                (unsigned long long)H, p.S);
    const size_t e = dt_esize(q->dt);
    const char *qb = (const char*)q->data, *ob = (const char*)dst->data;
    RCU_REQUIRE(dev, ob >= qb + T * H * p.D * e || qb >= ob + T * H * p.E * e, "paged_attention: the output overlaps the queries");
    if (T == 0) return RCU_OK;
    a.q = q->data;
    a.out = dst->data;
    a.sink = sink ? (const float*)sink->data : nullptr;
    a.H = (int)H;
    // a window as long as a sequence's room is none; sums of rows and windows stay below 2^31
    a.window = window >= (uint64_t)p.MP << p.shift ? 0 : (int)window;
    a.first = first > (1u << 29) ? 1 << 29 : (int)first;
    a.c = scale * kLog2e;
    DevGuard guard(dev->ordinal);
    Scratch mem(dev);
    st = mem.take("paged_attention", scratch, scratch_bytes(dev, p, H, q->dt));
    if (st != RCU_OK) return st;
    a.lse = p.mass ? (float*)mem.ptr : nullptr;
    void* rest = (char*)mem.ptr + lse_bytes(p, H);
    return q->dt == RCU_F32 ? attend<float>(dev, a, q->dt, rest) : q->dt == RCU_F16 ? attend<__half>(dev, a, q->dt, rest) : attend<__nv_bfloat16>(dev, a, q->dt, rest);
}

}  // extern "C"
