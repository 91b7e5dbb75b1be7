// Rotation of head features by positions that are given per token, on up to four axes (rcu_rotary_axes): what a batch of sequences at
// different places needs, and models of images and video, whose pairs turn by time, row or column.
//
//   (u, v) <- m (u cos a - v sin a, v cos a + u sin a),  a = position[axis of the pair][token] * frequency[pair]
//
// Bound by memory: every row is read and written once.  A CTA takes a few tokens: it works out their angles once, in shared memory, and then
// turns all their heads, sixteen bytes of a row per thread and step.  The angle is a product of doubles, brought into [-pi, pi] by doubles
// (so positions of any size keep their low bits), and only there goes on in f32, which costs a tenth of a double's sine: its rounding moves the angle by 2^-23
// (1.2e-7) at most, and sincosf's results are off by two units in the last place at most (1.2e-7 again).  The table's two floats leave 2^-48 of the angle open.
// 8192 tokens, 16 heads of 128, three axes, f16: 20.5 us (3.3 TB/s), 17 where the passes before have left the rows in L2; 32 tokens 5.1 us.
#include "lm_math.cuh"

namespace {

struct AxesArgs {
    const float* freqs;
    const int* positions;      // [axes, T]
    int ends[4];               // pairs that go by axis 0, 0..1, 0..2, 0..3
    long long T;
    long long pitch;           // of x's rows
    int H, D, first, pairs, halves;
    float magnitude;
};

__device__ __forceinline__ float2 turn_of(const AxesArgs& a, long long t, int i) {
    const int axis = (i >= a.ends[0]) + (i >= a.ends[1]) + (i >= a.ends[2]);
    const double angle = (double)a.positions[axis * a.T + t] * ((double)a.freqs[i] + (double)a.freqs[a.pairs + i]);
    const double turns = rint(angle * 0.15915494309189535);
    // 2 pi as two doubles
    const double r = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, angle));
    float s, c;
    sincosf((float)r, &s, &c);
    return make_float2(c * a.magnitude, s * a.magnitude);
}

// V elements of 16 bytes (VEC), or one by one; `tokens` tokens per CTA
template <class T, bool VEC>
__global__ void __launch_bounds__(256) rotary_axes_kernel(const AxesArgs a, const T* x, T* out, int tokens, int ahead) {
    rcu_kernel_entry();
    extern __shared__ float2 cs[];
    const long long t0 = (long long)blockIdx.x * tokens;
    const int n = (int)min((long long)tokens, a.T - t0);
    if (VEC && ahead) {                      // the rows are on their way while the angles are worked out
        const int lines = (int)(((long long)a.H * a.D * (int)sizeof(T) + 127) / 128);
        for (int i = threadIdx.x; i < n * lines; i += 256)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(x + (t0 + i / lines) * a.pitch + (long long)(i % lines) * (128 / (int)sizeof(T))));
    }
    for (int i = threadIdx.x; i < n * a.pairs; i += 256) cs[i] = turn_of(a, t0 + i / a.pairs, i % a.pairs);
    __syncthreads();
    const int lo = a.first, hi = a.first + 2 * a.pairs;
    if constexpr (VEC) {
        constexpr int V = 16 / (int)sizeof(T);
        struct alignas(16) Vec { T v[V]; };
        // a thread has one place of a row, in every token or every few, one after the other: dst may be x itself, so no token is read ahead of the one before
        const int places = a.H * (a.halves ? a.pairs / V + (a.D - 2 * a.pairs) / V : a.D / V), abreast = max(1, 256 / places);
        const int first_place = places < 256 ? (int)threadIdx.x % places : (int)threadIdx.x, first_token = places < 256 ? (int)threadIdx.x / places : 0;
        if (first_token >= abreast) return;
        if (a.halves) {
            // units of V pairs: V features of the first half and V of the second; then what is not turned
            const int units = a.pairs / V, rest = (a.D - 2 * a.pairs) / V, per = units + rest;
            for (int j = first_place; j < places; j += 256) {
                const int h = j / per, u = j - h * per;
                int d = u < units ? lo + u * V : (u - units) * V;
                if (u >= units && d >= lo) d += 2 * a.pairs;
                const int e = u < units ? d + a.pairs : d;
                const T* xr = x + t0 * a.pitch + (size_t)h * a.D;
                T* o = out + (t0 * a.H + h) * (size_t)a.D;
#pragma unroll 4
                for (int t = first_token; t < n; t += abreast) {
                    Vec p = *reinterpret_cast<const Vec*>(xr + t * a.pitch + d), q = *reinterpret_cast<const Vec*>(xr + t * a.pitch + e);
                    if (u < units) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const float2 w = cs[t * a.pairs + u * V + i];
                            const float f = to_f32<T>(p.v[i]), g = to_f32<T>(q.v[i]);
                            p.v[i] = from_f32<T>(f * w.x - g * w.y);
                            q.v[i] = from_f32<T>(g * w.x + f * w.y);
                        }
                        *reinterpret_cast<Vec*>(o + (size_t)t * a.H * a.D + e) = q;
                    }
                    *reinterpret_cast<Vec*>(o + (size_t)t * a.H * a.D + d) = p;
                }
            }
        } else {
            const int per = a.D / V;
            for (int j = first_place; j < places; j += 256) {
                const int h = j / per, d = (j - h * per) * V;
                const T* xr = x + t0 * a.pitch + (size_t)h * a.D + d;
                T* o = out + (t0 * a.H + h) * (size_t)a.D + d;
                const bool turned = d >= lo && d < hi;
#pragma unroll 4
                for (int t = first_token; t < n; t += abreast) {
                    Vec p = *reinterpret_cast<const Vec*>(xr + t * a.pitch);
                    if (turned) {
#pragma unroll
                        for (int e = 0; e < V; e += 2) {
                            const float2 w = cs[t * a.pairs + (d - lo + e) / 2];
                            const float f = to_f32<T>(p.v[e]), g = to_f32<T>(p.v[e + 1]);
                            p.v[e] = from_f32<T>(f * w.x - g * w.y);
                            p.v[e + 1] = from_f32<T>(g * w.x + f * w.y);
                        }
                    }
                    *reinterpret_cast<Vec*>(o + (size_t)t * a.H * a.D) = p;
                }
            }
        }
    } else {
        const int rest = a.D - 2 * a.pairs, per = a.pairs + rest;
        for (int j = threadIdx.x; j < n * a.H * per; j += 256) {
            const int t = j / (a.H * per), h = j / per % a.H, u = j % per;
            const T* xr = x + (t0 + t) * a.pitch + (size_t)h * a.D;
            T* o = out + ((t0 + t) * a.H + h) * (size_t)a.D;
            if (u >= a.pairs) {
                int d = u - a.pairs;
                if (d >= lo) d += 2 * a.pairs;
                o[d] = xr[d];
                continue;
            }
            const int d = lo + (a.halves ? u : 2 * u), e = d + (a.halves ? a.pairs : 1);
            const float2 w = cs[t * a.pairs + u];
            const float f = to_f32<T>(xr[d]), g = to_f32<T>(xr[e]);
            o[d] = from_f32<T>(f * w.x - g * w.y);
            o[e] = from_f32<T>(g * w.x + f * w.y);
        }
    }
}

template <class T> void launch_axes(rcu_device* dev, const AxesArgs& a, const void* x, void* out) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool vec = a.D % V == 0 && a.first % V == 0 && (a.halves ? a.pairs : 2 * a.pairs) % V == 0 && a.pitch % V == 0 &&
                     ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    // enough work for a CTA's threads, as long as every SM gets some and the angles take 16 KB at most
    int tokens = 1;
    while (tokens < 8 && (long long)tokens * a.H * a.D < 8 * 256 * V && a.T / (2 * tokens) >= 2 * dev->sm_count && 2 * tokens * a.pairs <= 2048) tokens *= 2;
    const unsigned grid = (unsigned)((a.T + tokens - 1) / tokens);
    const size_t smem = (size_t)tokens * a.pairs * sizeof(float2);
    // Rows are asked for ahead of the angles where x and dst together are larger than L2, so that x comes from memory: 8192 tokens, 32 heads of 128 in f32 50.4 -> 43.4 us;
    // with half the heads in f16, which stay in L2 from one such pass to the next, the requests cost 16.4 -> 17.2.  Where other work has put smaller rows out of L2,
    // nobody asks ahead, and the latter case takes 20.5
    const int ahead = 2 * a.T * a.H * a.D * (long long)sizeof(T) > (126ll << 20);
    if (vec) rcu_launch(dev, rotary_axes_kernel<T, true>, grid, 256, smem, a, (const T*)x, (T*)out, tokens, ahead);
    else rcu_launch(dev, rotary_axes_kernel<T, false>, grid, 256, smem, a, (const T*)x, (T*)out, tokens, ahead);
}

}  // namespace

extern "C" {

rcu_status rcu_rotary_axes(rcu_device* dev, const rcu_tensor* x, uint32_t x_col, uint32_t first, const rcu_tensor* freqs, float magnitude,
                           const rcu_tensor* positions, const uint32_t* sections, int halves, rcu_tensor* dst) {
    if (!dev) return RCU_ERR_INVALID_ARG;
    RCU_REQUIRE(dev, t_valid(x) && t_valid(freqs) && t_valid(positions) && sections && t_valid(dst), "rotary_axes: invalid tensor descriptor");
    RCU_REQUIRE(dev, x->rank == 2 && dst->rank == 3 && x->dt == dst->dt && dt_is_float(x->dt) && dst->shape[0] == x->shape[0],
                "rotary_axes: float rows x [tokens, width] and dst [tokens, heads, dim] of one dtype");
    RCU_REQUIRE(dev, freqs->dt == RCU_F32 && freqs->rank == 2 && freqs->shape[0] == 2, "rotary_axes: the frequency table is f32 [2, pairs]");
    const uint64_t T = x->shape[0], W = x->shape[1], H = dst->shape[1], D = dst->shape[2], pairs = freqs->shape[1];
    RCU_REQUIRE(dev, positions->dt == RCU_I32 && positions->rank == 2 && positions->shape[0] >= 1 && positions->shape[0] <= 4 && positions->shape[1] == T,
                "rotary_axes: positions are i32 [axes, tokens] of one to four axes");
    RCU_REQUIRE(dev, H <= (1u << 20) && D <= (1u << 20) && H * D <= W && x_col <= W - H * D && W <= (1ull << 31), "rotary_axes: the heads lie outside the rows");
    RCU_REQUIRE(dev, pairs <= 2048 && (uint64_t)first + 2 * pairs <= D && T < (1ull << 31) / 4, "rotary_axes: the rotated features lie outside the head");
    AxesArgs a{(const float*)freqs->data, (const int*)positions->data, {}, (long long)T, (long long)W, (int)H, (int)D, (int)first, (int)pairs, halves != 0, magnitude};
    uint64_t sum = 0;
    for (int i = 0; i < 4; ++i) {
        if ((uint64_t)i < positions->shape[0]) sum += sections[i];
        a.ends[i] = (int)(sum < pairs ? sum : pairs);
    }
    RCU_REQUIRE(dev, sum == pairs, "rotary_axes: the sections hold %llu of %llu pairs", (unsigned long long)sum, (unsigned long long)pairs);
    const size_t e = dt_esize(x->dt);
    const char *xb = (const char*)x->data, *xe = xb + T * W * e, *ob = (const char*)dst->data, *oe = ob + T * H * D * e;
    RCU_REQUIRE(dev, ob >= xe || oe <= xb || (ob == xb && W == H * D), "rotary_axes: dst overlaps rows of x that hold more than the heads");
    if (T == 0 || H * D == 0) return RCU_OK;
    // a wider index than an int holds is left out rather than wrapped: eight tokens' units per CTA
    RCU_REQUIRE(dev, 8 * H * D < (1ull << 31), "rotary_axes: rows of %llu features", (unsigned long long)(H * D));
    DevGuard g(dev->ordinal);
    const void* xp = xb + (size_t)x_col * e;
    if (x->dt == RCU_F32) launch_axes<float>(dev, a, xp, dst->data);
    else if (x->dt == RCU_F16) launch_axes<__half>(dev, a, xp, dst->data);
    else launch_axes<__nv_bfloat16>(dev, a, xp, dst->data);
    RCU_LAUNCH_CHECK(dev);
    return RCU_OK;
}

}  // extern "C"
