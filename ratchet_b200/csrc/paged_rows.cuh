// Attention of one query over the rows that it sees and no others, by a warp: any type, width, alignment and value.
#pragma once
#include "paged_attention.cuh"

namespace paged {

// What a warp has of one query: the maximum score (units of log 2), the sum of weights, and every 32nd feature from `lane` on of the weighted values
struct RowPart {
    float m, l, o[8];
};

// Rows [j0, j1) of a sequence for one query: 32 keys a step, a lane for each; then a lane for every 32nd feature of the values.
template <class T>
__device__ void attend_run(const AttendArgs& a, int s, int g, const T* q, int j0, int j1, RowPart& part) {
    const View& p = a.p;
    const int lane = threadIdx.x & 31;
    const T *keys = (const T*)p.keys, *values = (const T*)p.values;
    for (int j = j0; j < j1; j += 32) {
        const int r = j + lane;
        float z = -INFINITY;
        int page = 0;
        if (r < j1) {
            page = page_of(p, s, r);
            const T* k = keys + row_at(p, page, g, r, p.D);
            float sum = 0.f;
            for (int d = 0; d < p.D; ++d) sum = fmaf(to_f32<T>(q[d]), to_f32<T>(k[d]), sum);
            z = sum * a.c;
        }
        const float next = fmaxf(part.m, warp_max(z)), base = next == -INFINITY ? 0.f : next;
        const float corr = exp2f(part.m - base), w = r < j1 ? exp2f(z - base) : 0.f;
        part.l = part.l * corr + warp_sum(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) part.o[i] *= corr;
        part.m = next;
        for (int u = 0; u < min(32, j1 - j); ++u) {
            const float pw = __shfl_sync(0xffffffffu, w, u);
            const T* v = values + row_at(p, __shfl_sync(0xffffffffu, page, u), g, j + u, p.E);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane + 32 * i < p.E) part.o[i] = fmaf(pw, to_f32<T>(v[lane + 32 * i]), part.o[i]);
        }
    }
}

// The query of token t, head h, at row r, over what it sees of the tiles [n0, n1) of a span
template <class T>
__device__ __noinline__ void attend_row(const AttendArgs& a, int s, int g, int t, int h, int r, Span sp, int n0, int n1, RowPart& part) {
    part.m = -INFINITY;
    part.l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) part.o[i] = 0.f;
    if (r < 0) return;
    const T* q = (const T*)a.q + ((size_t)t * a.H + h) * a.p.D;
    const int L = clamp_int(a.p.lengths[s], 0, a.p.MP << a.p.shift);
    int head, low;
    visible(a.window, a.first, r, head, low);
    for (int n = n0; n < n1; ++n) {
        const int j0 = sp.tile(n) * kTileK, j1 = min(j0 + kTileK, min(r + 1, L));
        attend_run<T>(a, s, g, q, j0, min(j1, head), part);
        attend_run<T>(a, s, g, q, max(j0, max(low, head)), j1, part);
    }
}

// A query whose rows one warp has had: sink, output, and lse where it is wanted
template <class T> __device__ void finish_row(const AttendArgs& a, int t, int h, const RowPart& part) {
    const int lane = threadIdx.x & 31;
    const size_t at = (size_t)t * a.H + h;
    float m = part.m, l = part.l, corr = 1.f;
    if (a.sink) {
        const float sk = a.sink[h] * kLog2e, top = fmaxf(m, sk);
        corr = exp2f(m - top);
        l = l * corr + exp2f(sk - top);
        m = top;
    }
    const float inv = 1.f / l;
    T* out = (T*)a.out + at * a.p.E;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < a.p.E) out[lane + 32 * i] = from_f32<T>(part.o[i] * corr * inv);
    if (a.lse && lane == 0) a.lse[at] = m + log2f(l);
}

__device__ __forceinline__ void store_part(const Plan& pl, int E, int slot, int row, const RowPart& part) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) pl.ml[(size_t)slot * pl.stride + row] = make_float2(part.m, part.l);
    float* o = reinterpret_cast<float*>(pl.o);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = lane + 32 * i;
        if (c < E) o[(((size_t)slot * (E / 4) + c / 4) * pl.stride + row) * 4 + (c & 3)] = part.o[i];
    }
}

}  // namespace paged
