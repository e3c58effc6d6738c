// Group norm of tensors with their channels last, with the shortcut and the activation that follow it, and its gradients.
//
//   xhat = (x - mean) r,  r = 1 / sqrt(var + epsilon), mean and var over a sample's places and the channels of a group
//   z = xhat scale + offset + residual,  y = act(z)
//   dz = dy act'(z),  doffset = sum of dz, dscale = sum of dz xhat (over samples and places),  dresidual = dz
//   dx = r (dz scale - S1 / m - xhat S2 / m),  S1 and S2: the group's sums of dz scale and dz scale xhat, m its number of values
//
// Bound by memory: x (and the residual) in, y out; x, dy (and the residual) in, dx (and dresidual) out.  A sum over the group stands between the
// two, so a span of channels, one or several whole groups of a sample, stays in the shared memory of a block or of a cluster of blocks in the
// meantime (norm_forward_kernel, norm_backward_kernel), and the tensors cross the memory's bus once.  The blocks of a cluster read one
// another's sums from shared memory.  Where a span is larger than what a cluster holds, the tensors are read twice, by the kernels with
// the sums and by those that use them, the second ones from the end on, where the first have just been.
//
// Threads: values are taken 16 bytes at a time, neighbouring threads neighbouring ones.  The number of threads that take part is such
// that a thread's channels repeat with every step, so that it keeps their mean, factor, offset and sums in registers; that holds for lines that
// start anywhere, too (20 channels of fp16: 5 vectors hold two lines), as a whole tensor has no gaps.  A vector that sticks out of what a block
// has, at its start or its end, is moved value by value.
//
// Sums are fp32.  Those of the variance are never of squares that nearly cancel: a thread adds the squares of a few values less their own mean, and
// means and squares are joined pair by pair (Chan, Golub and LeVeque).  Every sum has a fixed order.
// Between the two passes of the gradients dz stays fp32.  Nothing is rounded to fewer bits but the outputs.
#include <atomic>
#include <type_traits>
#include <vector>

#include "axc_gemm.h"
#include "axc_mma.cuh"
#include "axc_norm_plan.h"

namespace axc {
namespace {

struct NormArgs {
    const void *x, *residual, *scale, *offset, *dy;
    void *y, *dx, *dresidual;
    int scale_type, offset_type, activation;
    float epsilon;
    long long samples, places, channels;
    int groups, each;                          // channels of a group: each
    float2 *statistics;                        // [samples][groups] {mean, r}
    int span, spans, blocks, active;           // channels of a block's span, spans of a sample, blocks that share one
    long long shares;
    float2 *part;                              // [samples][shares][channels] sums of a share of the places
    float2 *sums;                              // [samples][channels] {sum of dz, sum of dz xhat}
    float2 *group_sums;                        // [samples][groups] {S1 r / m, S2 r r / m}
    void *dscale, *doffset;
    __host__ __device__ long long values() const { return samples * places * channels; }
};

template <int BYTES> struct Bits;
template <> struct Bits<2> { typedef unsigned short type; };
template <> struct Bits<4> { typedef unsigned type; };
template <> struct Bits<16> { typedef uint4 type; };
template <typename T, int V>
union Pack {
    typename Bits<V * sizeof(T)>::type w;
    T t[V];
    __device__ Pack() {}
};

// Values before a block's first one back to a multiple of 16 bytes.  (Pieces of lines start on one.)
template <typename T, int V>
__device__ __forceinline__ int shift_of(const NormArgs &P, long long sample, long long place0)
{
    return V == 1 || P.span < P.channels ? 0 : int((sample * P.places + place0) * P.channels & (V - 1));
}

template <typename T, int V>
__device__ __forceinline__ void load(const T *sample, const Walk<V> &w, int j, Pack<T, V> &v, [[maybe_unused]] const T *base, [[maybe_unused]] long long count)
{
    const T *from = sample + w.at + j * w.step;
    if (w.whole(j)) {
        if (AXC_VALUES_OK(from, V, base, count, 501u)) v.w = *reinterpret_cast<const typename Bits<V * sizeof(T)>::type *>(from);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v.t[i] = w.has(j, i) && AXC_VALUES_OK(from + i, 1, base, count, 502u) ? from[i] : narrow<T>(0.0f);
    }
}
template <typename T, int V>
__device__ __forceinline__ void store(T *sample, const Walk<V> &w, int j, const float (&x)[V], [[maybe_unused]] T *base, [[maybe_unused]] long long count)
{
    T *to = sample + w.at + j * w.step;
    Pack<T, V> v;
#pragma unroll
    for (int i = 0; i < V; ++i) v.t[i] = narrow<T>(x[i]);
    if (w.whole(j)) {
        if (AXC_VALUES_OK(to, V, base, count, 503u)) *reinterpret_cast<typename Bits<V * sizeof(T)>::type *>(to) = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (w.has(j, i) && AXC_VALUES_OK(to + i, 1, base, count, 504u)) to[i] = v.t[i];
    }
}

template <int V, bool EXACT>
__device__ __forceinline__ void activate_all(float (&z)[V], int act)
{
    if (act == kActNone) return;
    if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = activate(z[i], kActRelu, EXACT);
    } else if (act == kActGelu) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = activate(z[i], kActGelu, EXACT);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = activate(z[i], kActSilu, EXACT);
    }
}
// d *= act'(z)
template <int V, bool EXACT>
__device__ __forceinline__ void slopes(float (&d)[V], const float (&z)[V], int act)
{
    if (act == kActNone) return;
    if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] *= slope_of<kActRelu, EXACT>(z[i]);
    } else if (act == kActGelu) {
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] *= slope_of<kActGelu, EXACT>(z[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] *= slope_of<kActSilu, EXACT>(z[i]);
    }
}

// Mean and sum of squared distances from it, for each of a thread's channels
template <int V>
struct Moments {
    float n = 0.0f, mean[V], square[V];        // n: whole vectors so far
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N][V])
    {
        const float sum = n + N, w = __fdividef(float(N), sum), w2 = n * w;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float m = v[0][i], q = 0.0f;
#pragma unroll
            for (int k = 1; k < N; ++k) m += v[k][i];
            m *= 1.0f / N;
#pragma unroll
            for (int k = 0; k < N; ++k) q = fmaf(v[k][i] - m, v[k][i] - m, q);
            if (n == 0.0f) {
                mean[i] = m;
                square[i] = q;
            } else {
                const float d = m - mean[i];
                mean[i] = fmaf(d, w, mean[i]);
                square[i] = fmaf(d * d, w2, square[i] + q);
            }
        }
        n = sum;
    }
    // one value of channel i, which has had `k` so far
    __device__ __forceinline__ void add_one(int i, float v, float k)
    {
        if (k == 0.0f) {
            mean[i] = v;
            square[i] = 0.0f;
        } else {
            const float d = v - mean[i];
            mean[i] += __fdividef(d, k + 1.0f);
            square[i] = fmaf(d, v - mean[i], square[i]);
        }
    }
};

// x's moments, `chunk` vectors on their way at a time; keep(j, vector) sees every vector
template <typename T, int V, typename Keep>
__device__ __forceinline__ void take_moments(const T *sample, const Walk<V> &w, Moments<V> &mo, const T *base, long long count, Keep keep)
{
    constexpr int N = V == 1 ? 8 : 4;
    const int first = w.count > 0 && !w.whole(0) ? 1 : 0, end = w.count > first && !w.whole(w.count - 1) ? w.count - 1 : w.count;
    int j = first;
    for (; j + N <= end; j += N) {
        Pack<T, V> v[N];
        float f[N][V];
#pragma unroll
        for (int k = 0; k < N; ++k) load(sample, w, j + k, v[k], base, count);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            keep(j + k, v[k]);
#pragma unroll
            for (int i = 0; i < V; ++i) f[k][i] = widen(v[k].t[i]);
        }
        mo.add(f);
    }
    if (j < end) {
        Pack<T, V> v[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (j + k < end) load(sample, w, j + k, v[k], base, count);
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (j + k < end) {
                float f[1][V];
                keep(j + k, v[k]);
#pragma unroll
                for (int i = 0; i < V; ++i) f[0][i] = widen(v[k].t[i]);
                mo.add(f);
            }
    }
    if (V > 1 && (first > 0 || end < w.count)) {
        float had[V];
#pragma unroll
        for (int i = 0; i < V; ++i) had[i] = mo.n;
        for (int side = 0; side < 2; ++side) {
            if (side == 0 ? first == 0 : end == w.count) continue;
            const int at = side == 0 ? 0 : end;
            Pack<T, V> v;
            load(sample, w, at, v, base, count);
            keep(at, v);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (w.has(at, i)) {
                    mo.add_one(i, widen(v.t[i]), had[i]);
                    had[i] += 1.0f;
                }
        }
    }
}

// ---- sums over the threads of a block ------------------------------------------------------------------------------------------
// Lanes that share one of `items` sums: a power of two
__device__ __forceinline__ int lanes_for(int items)
{
    int q = 32;
    while (q > 1 && q * items > int(blockDim.x)) q >>= 1;
    return q;
}
__device__ __forceinline__ float over_lanes(float x, int q)
{
    for (int o = q >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// {mean, squared distances} of `items` neighbouring sets of `each` channels, from the threads' entries: give(item, mean, square) in one thread
template <typename Give>
__device__ __forceinline__ void join_moments(const float2 *entries, const Entries &E, int items, int each, float values, Give give)
{
    const int q = lanes_for(items), lane = threadIdx.x & (q - 1), step = int(blockDim.x) / q;
    for (int first = 0; first < items; first += step) {
        const int item = first + int(threadIdx.x) / q;
        const bool mine = item < items;
        float sum = 0.0f;
        if (mine) {
            for (int d = 0; d < each; ++d)
                for (int k = lane; k < E.copies; k += q) {
                    const int e = E.entry(item * each + d, k);
                    const float n = E.values(e);
                    if (n > 0.0f) sum = fmaf(n, entries[e].x, sum);
                }
        }
        const float mean = __fdiv_rn(over_lanes(sum, q), values);
        float square = 0.0f;
        if (mine) {
            for (int d = 0; d < each; ++d)
                for (int k = lane; k < E.copies; k += q) {
                    const int e = E.entry(item * each + d, k);
                    const float n = E.values(e);
                    if (n > 0.0f) {
                        const float off = entries[e].x - mean;
                        square += fmaf(n * off, off, entries[e].y);
                    }
                }
        }
        square = over_lanes(square, q);
        if (mine && lane == 0) give(item, mean, square);
    }
}

// Sums of pairs, for every channel of the span
template <typename Give>
__device__ __forceinline__ void join_sums(const float2 *entries, const Entries &E, Give give)
{
    const int q = lanes_for(E.span), lane = threadIdx.x & (q - 1), step = int(blockDim.x) / q;
    for (int first = 0; first < E.span; first += step) {
        const int l = first + int(threadIdx.x) / q;
        float a = 0.0f, b = 0.0f;
        if (l < E.span)
            for (int k = lane; k < E.copies; k += q) {
                const float2 f = entries[E.entry(l, k)];
                a += f.x;
                b += f.y;
            }
        a = over_lanes(a, q);
        b = over_lanes(b, q);
        if (l < E.span && lane == 0) give(l, a, b);
    }
}

// A pair from the same place in the shared memory of the cluster's block `rank`
__device__ __forceinline__ float2 of_block(const float2 *at, int rank)
{
    float2 f;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(mma::in_cta(mma::smem_address(at), unsigned(rank))));
    return f;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Where a resident block is
struct Place {
    long long sample, place0;
    int rank, span, channel0, places;
    __device__ __forceinline__ explicit Place(const NormArgs &P)
    {
        rank = P.blocks > 1 ? int(mma::cluster_rank()) : 0;
        const unsigned unit = blockIdx.x / unsigned(P.blocks);
        sample = unit / unsigned(P.spans);
        span = int(unit - unsigned(sample) * unsigned(P.spans));
        channel0 = span * P.span;
        place0 = P.places * rank / P.blocks;
        places = int(P.places * (rank + 1) / P.blocks - place0);
    }
};

// What a thread needs of its channels
template <int V>
struct Channels {
    float mean[V], factor[V], offset[V];
    // channel(i), group's {mean, r}(channel)
    template <typename Channel, typename Stats>
    __device__ __forceinline__ void fill(const NormArgs &P, Channel channel, Stats stats)
    {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = channel(i);
            const float2 s = stats(c);
            mean[i] = s.x;
            factor[i] = s.y * (P.scale && AXC_GLOBAL_OK(c, P.channels, 505u) ? load_as_float(P.scale, c, P.scale_type) : 1.0f);
            offset[i] = P.offset && AXC_GLOBAL_OK(c, P.channels, 506u) ? load_as_float(P.offset, c, P.offset_type) : 0.0f;
        }
    }
    __device__ __forceinline__ float z(int i, float x) const { return fmaf(x - mean[i], factor[i], offset[i]); }
};

// y of one vector
template <typename T, int V>
__device__ __forceinline__ void finish(const NormArgs &P, const Channels<V> &ch, const Walk<V> &w, int j, const Pack<T, V> &x, long long sample0)
{
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = ch.z(i, widen(x.t[i]));
    if (P.residual) {
        Pack<T, V> r;
        load(static_cast<const T *>(P.residual) + sample0, w, j, r, static_cast<const T *>(P.residual), P.values());
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] += widen(r.t[i]);
    }
    activate_all<V, sizeof(T) == 4>(z, P.activation);
    store(static_cast<T *>(P.y) + sample0, w, j, z, static_cast<T *>(P.y), P.values());
}

// dz of one vector, and x less its mean
template <typename T, int V>
__device__ __forceinline__ void slope_at(const NormArgs &P, const Channels<V> &ch, const Pack<T, V> &x, const Pack<T, V> &dy, const Pack<T, V> &residual, float (&dz)[V],
                                         float (&off)[V])
{
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        off[i] = widen(x.t[i]) - ch.mean[i];
        z[i] = fmaf(off[i], ch.factor[i], ch.offset[i]);
        dz[i] = widen(dy.t[i]);
    }
    if (P.residual && P.activation != kActNone) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] += widen(residual.t[i]);
    }
    slopes<V, sizeof(T) == 4>(dz, z, P.activation);
}

// ---- resident spans -------------------------------------------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 3) norm_forward_kernel(const NormArgs P)
{
    after_previous();
    extern __shared__ __align__(16) char raw[];
    const Place at(P);
    const int shift = shift_of<T, V>(P, at.sample, at.place0);
    const Walk<V> w(threadIdx.x, P.active, shift, at.places, P.span, P.channels, at.place0, at.channel0);
    const int steps = (int((P.places + P.blocks - 1) / P.blocks) * P.span + V - 1 + P.active * V - 1) / (P.active * V), groups = P.span / P.each;
    typedef typename Bits<V * sizeof(T)>::type Word;
    Word *kept = reinterpret_cast<Word *>(raw);
    float2 *entries = reinterpret_cast<float2 *>(raw + norm_up16(size_t(steps) * P.active * V * sizeof(T)));
    float2 *mine = entries + P.active * V, *result = mine + groups;
    const long long sample0 = at.sample * P.places * P.channels;
    const T *x = static_cast<const T *>(P.x);
    Moments<V> mo;
    take_moments(x + sample0, w, mo, x, P.values(), [&](int j, const Pack<T, V> &v) { kept[j * P.active + int(threadIdx.x)] = v.w; });
    if (int(threadIdx.x) < P.active) {
#pragma unroll
        for (int i = 0; i < V; ++i) entries[threadIdx.x * V + i] = make_float2(mo.mean[i], mo.square[i]);
    }
    __syncthreads();
    const Entries E(P.active, V, P.span, shift, w.total);
    join_moments(entries, E, groups, P.each, float(at.places) * float(P.each), [&](int g, float mean, float square) { mine[g] = make_float2(mean, square); });
    __syncwarp();
    if (P.blocks > 1) mma::cluster_sync();
    else __syncthreads();
    const float all = float(P.places) * float(P.each);
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
        float2 f = mine[g];
        if (P.blocks > 1) {
            float sum = 0.0f, square = 0.0f;
            for (int r = 0; r < P.blocks; ++r) {
                const float n = float(P.places * (r + 1) / P.blocks - P.places * r / P.blocks) * float(P.each);
                sum = fmaf(n, of_block(mine + g, r).x, sum);
            }
            const float mean = __fdiv_rn(sum, all);
            for (int r = 0; r < P.blocks; ++r) {
                const float n = float(P.places * (r + 1) / P.blocks - P.places * r / P.blocks) * float(P.each);
                const float2 other = of_block(mine + g, r);
                square += fmaf(n * (other.x - mean), other.x - mean, other.y);
            }
            f = make_float2(mean, square);
        }
        f.y = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(f.y, all) + P.epsilon));
        result[g] = f;
        const long long to = at.sample * P.groups + at.span * groups + g;
        if (at.rank == 0 && P.statistics && AXC_GLOBAL_OK(to, P.samples * P.groups, 507u)) P.statistics[to] = f;
    }
    __syncthreads();
    if (P.blocks > 1) cluster_arrive();
    Channels<V> ch;
    ch.fill(P, [&](int i) { return at.channel0 + local_channel<V>(w, P.span, i); }, [&](int c) { return result[(c - at.channel0) / P.each]; });
    constexpr int N = 4;
    for (int j = 0; j < w.count; j += N) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (j + k < w.count) {
                Pack<T, V> v;
                v.w = kept[(j + k) * P.active + int(threadIdx.x)];
                finish<T, V>(P, ch, w, j + k, v, sample0);
            }
    }
    __syncwarp();
    if (P.blocks > 1) cluster_wait();          // what others read of this block's shared memory
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 3) norm_backward_kernel(const NormArgs P)
{
    after_previous();
    extern __shared__ __align__(16) char raw[];
    const Place at(P);
    const int shift = shift_of<T, V>(P, at.sample, at.place0);
    const Walk<V> w(threadIdx.x, P.active, shift, at.places, P.span, P.channels, at.place0, at.channel0);
    const int steps = (int((P.places + P.blocks - 1) / P.blocks) * P.span + V - 1 + P.active * V - 1) / (P.active * V), groups = P.span / P.each;
    typedef typename Bits<V * sizeof(T)>::type Word;
    constexpr int kQuads = V >= 4 ? V / 4 : 1;
    typedef typename Bits<V >= 4 ? 16 : 4>::type Quad;                         // four values of dz, or one
    const int slots = steps * P.active;
    Quad *kept_dz = reinterpret_cast<Quad *>(raw);
    Word *kept = reinterpret_cast<Word *>(raw + norm_up16(size_t(slots) * V * 4));
    float2 *entries = reinterpret_cast<float2 *>(raw + norm_up16(size_t(slots) * V * 4) + norm_up16(size_t(slots) * V * sizeof(T)));
    float2 *channels = entries + P.active * V, *mine = channels + P.span, *result = mine + groups;
    const long long sample0 = at.sample * P.places * P.channels, values = P.values();
    const T *x = static_cast<const T *>(P.x), *dy = static_cast<const T *>(P.dy), *residual = static_cast<const T *>(P.residual);
    auto stats = [&](int c) {
        const long long from = at.sample * P.groups + c / P.each;
        return AXC_GLOBAL_OK(from, P.samples * P.groups, 508u) ? P.statistics[from] : make_float2(0.0f, 0.0f);
    };
    Channels<V> ch;
    ch.fill(P, [&](int i) { return at.channel0 + local_channel<V>(w, P.span, i); }, stats);
    float sum[V], sum_off[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = sum_off[i] = 0.0f;
    const bool with = P.residual && P.activation != kActNone;
    constexpr int N = 2;
    for (int j = 0; j < w.count; j += N) {
        Pack<T, V> vx[N], vd[N], vr[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (j + k < w.count) {
                load(x + sample0, w, j + k, vx[k], x, values);
                load(dy + sample0, w, j + k, vd[k], dy, values);
                if (with) load(residual + sample0, w, j + k, vr[k], residual, values);
            }
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (j + k < w.count) {
                float dz[V], off[V];
                slope_at<T, V>(P, ch, vx[k], vd[k], vr[k], dz, off);
                if (!w.whole(j + k)) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (!w.has(j + k, i)) dz[i] = off[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sum[i] += dz[i];
                    sum_off[i] = fmaf(dz[i], off[i], sum_off[i]);
                }
                const int slot = (j + k) * P.active + int(threadIdx.x);
                kept[slot] = vx[k].w;
#pragma unroll
                for (int q = 0; q < kQuads; ++q) {
                    if constexpr (V >= 4)
                        kept_dz[q * slots + slot] = make_uint4(__float_as_uint(dz[4 * q]), __float_as_uint(dz[4 * q + 1]), __float_as_uint(dz[4 * q + 2]),
                                                               __float_as_uint(dz[4 * q + 3]));
                    else kept_dz[slot] = __float_as_uint(dz[0]);
                }
                if (P.dresidual) store(static_cast<T *>(P.dresidual) + sample0, w, j + k, dz, static_cast<T *>(P.dresidual), values);
            }
    }
    if (int(threadIdx.x) < P.active) {
#pragma unroll
        for (int i = 0; i < V; ++i) entries[threadIdx.x * V + i] = make_float2(sum[i], sum_off[i]);
    }
    __syncthreads();
    const Entries E(P.active, V, P.span, shift, w.total);
    join_sums(entries, E, [&](int l, float a, float b) { channels[l] = make_float2(a, b * stats(at.channel0 + l).y); });
    __syncthreads();
    {
        const int q = lanes_for(groups), lane = threadIdx.x & (q - 1), step = int(blockDim.x) / q;
        for (int first = 0; first < groups; first += step) {
            const int g = first + int(threadIdx.x) / q;
            float a = 0.0f, b = 0.0f;
            if (g < groups)
                for (int d = lane; d < P.each; d += q) {
                    const int c = at.channel0 + g * P.each + d;
                    const float scale = P.scale && AXC_GLOBAL_OK(c, P.channels, 509u) ? load_as_float(P.scale, c, P.scale_type) : 1.0f;
                    const float2 f = channels[g * P.each + d];
                    a = fmaf(scale, f.x, a);
                    b = fmaf(scale, f.y, b);
                }
            a = over_lanes(a, q);
            b = over_lanes(b, q);
            if (g < groups && lane == 0) mine[g] = make_float2(a, b);
        }
    }
    __syncwarp();
    if (P.blocks > 1) mma::cluster_sync();
    else __syncthreads();
    const float all = float(P.places) * float(P.each);
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
        float2 f = mine[g];
        if (P.blocks > 1) {
            f = make_float2(0.0f, 0.0f);
            for (int r = 0; r < P.blocks; ++r) {
                const float2 other = of_block(mine + g, r);
                f.x += other.x;
                f.y += other.y;
            }
        }
        const float r = stats(at.channel0 + g * P.each).y;
        result[g] = make_float2(__fdiv_rn(f.x, all) * r, __fdiv_rn(f.y, all) * r * r);
    }
    // the sums of single channels, shared out among the cluster's blocks
    for (int l = at.rank + int(threadIdx.x) * P.blocks; l < P.span; l += int(blockDim.x) * P.blocks) {
        float2 f = channels[l];
        if (P.blocks > 1) {
            f = make_float2(0.0f, 0.0f);
            for (int r = 0; r < P.blocks; ++r) {
                const float2 other = of_block(channels + l, r);
                f.x += other.x;
                f.y += other.y;
            }
        }
        const long long to = at.sample * P.channels + at.channel0 + l;
        if (P.sums && AXC_GLOBAL_OK(to, P.samples * P.channels, 510u)) P.sums[to] = f;
    }
    __syncthreads();
    if (P.blocks > 1) cluster_arrive();
    if (P.dx) {
        float first[V], second[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 f = result[local_channel<V>(w, P.span, i) / P.each];
            first[i] = f.x;
            second[i] = f.y;
        }
#pragma unroll 2
        for (int j = 0; j < w.count; ++j) {
            const int slot = j * P.active + int(threadIdx.x);
            Pack<T, V> v;
            v.w = kept[slot];
            float dx[V];
#pragma unroll
            for (int q = 0; q < kQuads; ++q) {
                if constexpr (V >= 4) {
                    const uint4 d = kept_dz[q * slots + slot];
                    dx[4 * q] = __uint_as_float(d.x);
                    dx[4 * q + 1] = __uint_as_float(d.y);
                    dx[4 * q + 2] = __uint_as_float(d.z);
                    dx[4 * q + 3] = __uint_as_float(d.w);
                } else dx[0] = __uint_as_float(kept_dz[slot]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) dx[i] = fmaf(-second[i], widen(v.t[i]) - ch.mean[i], fmaf(dx[i], ch.factor[i], -first[i]));
            store(static_cast<T *>(P.dx) + sample0, w, j, dx, static_cast<T *>(P.dx), values);
        }
    }
    __syncwarp();
    if (P.blocks > 1) cluster_wait();
}

// ---- tensors that are read twice -------------------------------------------------------------------------------------------------
// Block -> sample, share of the places, columns
struct Share {
    long long sample, share, place0;
    int channel0, span, places, active;
    template <int V>
    static __device__ __forceinline__ Share of(const NormArgs &P, long long block, std::integral_constant<int, V>)
    {
        Share s;
        const long long columns = P.spans;
        s.channel0 = int(block % columns) * P.span;
        block /= columns;
        s.share = block % P.shares;
        s.sample = block / P.shares;
        s.span = int(P.channels - s.channel0 < P.span ? P.channels - s.channel0 : P.span);
        s.place0 = P.places * s.share / P.shares;
        s.places = int(P.places * (s.share + 1) / P.shares - s.place0);
        // as norm_active has it; a narrower last span has a divisor of its own
        s.active = s.span == P.span ? P.active : int(blockDim.x) / (s.span / V) * (s.span / V);
        return s;
    }
};

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads) norm_moments_kernel(const NormArgs P)
{
    after_previous();
    __shared__ float2 entries[kNormThreads * V];
    const Share at = Share::of(P, blockIdx.x, std::integral_constant<int, V>());
    const int shift = shift_of<T, V>(P, at.sample, at.place0);
    const Walk<V> w(threadIdx.x, at.active, shift, at.places, at.span, P.channels, at.place0, at.channel0);
    const T *x = static_cast<const T *>(P.x);
    Moments<V> mo;
    take_moments(x + at.sample * P.places * P.channels, w, mo, x, P.values(), [](int, const Pack<T, V> &) {});
    if (int(threadIdx.x) < at.active) {
#pragma unroll
        for (int i = 0; i < V; ++i) entries[threadIdx.x * V + i] = make_float2(mo.mean[i], mo.square[i]);
    }
    __syncthreads();
    const Entries E(at.active, V, at.span, shift, w.total);
    const long long to = (at.sample * P.shares + at.share) * P.channels + at.channel0;
    join_moments(entries, E, at.span, 1, float(at.places), [&](int l, float mean, float square) {
        if (AXC_GLOBAL_OK(to + l, P.samples * P.shares * P.channels, 511u)) P.part[to + l] = make_float2(mean, square);
    });
}

__device__ __forceinline__ float over_block(float x, float *room)
{
    x = over_lanes(x, 32);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = x;
    __syncthreads();
    float sum = 0.0f;
    for (int i = 0; i < int(blockDim.x) / 32; ++i) sum += room[i];
    return sum;
}

// A block joins the shares of one sample's group
__global__ void __launch_bounds__(kNormThreads) norm_join_kernel(const NormArgs P)
{
    after_previous();
    __shared__ float room[kNormThreads / 32];
    const long long sample = blockIdx.x / P.groups;
    const int group = int(blockIdx.x - sample * P.groups);
    const float2 *part = P.part + sample * P.shares * P.channels + group * P.each;
    const long long entries = P.shares * P.each;
    const float all = float(P.places) * float(P.each);
    auto values = [&](long long s) { return float(P.places * (s + 1) / P.shares - P.places * s / P.shares); };
    [[maybe_unused]] const long long room_for = P.shares * P.channels - group * P.each;
    float sum = 0.0f, square = 0.0f;
    for (long long e = threadIdx.x; e < entries; e += kNormThreads) {
        const long long s = e / P.each, from = s * P.channels + (e - s * P.each);
        if (AXC_GLOBAL_OK(from, room_for, 512u)) sum = fmaf(values(s), part[from].x, sum);
    }
    const float mean = __fdiv_rn(over_block(sum, room), all);
    for (long long e = threadIdx.x; e < entries; e += kNormThreads) {
        const long long s = e / P.each, from = s * P.channels + (e - s * P.each);
        if (!AXC_GLOBAL_OK(from, room_for, 513u)) continue;
        const float2 f = part[from];
        square += fmaf(values(s) * (f.x - mean), f.x - mean, f.y);
    }
    square = over_block(square, room);
    if (threadIdx.x == 0) P.statistics[blockIdx.x] = make_float2(mean, __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(square, all) + P.epsilon)));
}

template <int V>
__device__ __forceinline__ void fill_channels(const NormArgs &P, const Share &at, const Walk<V> &w, Channels<V> &ch)
{
    ch.fill(P, [&](int i) { return at.channel0 + local_channel<V>(w, at.span, i); },
            [&](int c) {
                const long long from = at.sample * P.groups + c / P.each;
                return AXC_GLOBAL_OK(from, P.samples * P.groups, 514u) ? P.statistics[from] : make_float2(0.0f, 0.0f);
            });
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 3) norm_apply_kernel(const NormArgs P)
{
    after_previous();
    const Share at = Share::of(P, (long long)gridDim.x - 1 - blockIdx.x, std::integral_constant<int, V>());
    const Walk<V> w(threadIdx.x, at.active, shift_of<T, V>(P, at.sample, at.place0), at.places, at.span, P.channels, at.place0, at.channel0);
    if (w.count == 0) return;
    Channels<V> ch;
    fill_channels<V>(P, at, w, ch);
    const long long sample0 = at.sample * P.places * P.channels;
    const T *x = static_cast<const T *>(P.x);
    constexpr int N = 4;
    for (int j = 0; j < w.count; j += N) {
        Pack<T, V> v[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (j + k < w.count) load(x + sample0, w, j + k, v[k], x, P.values());
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (j + k < w.count) finish<T, V>(P, ch, w, j + k, v[k], sample0);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 3) norm_sums_kernel(const NormArgs P)
{
    after_previous();
    __shared__ float2 entries[kNormThreads * V];
    const Share at = Share::of(P, blockIdx.x, std::integral_constant<int, V>());
    const int shift = shift_of<T, V>(P, at.sample, at.place0);
    const Walk<V> w(threadIdx.x, at.active, shift, at.places, at.span, P.channels, at.place0, at.channel0);
    float sum[V], sum_off[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = sum_off[i] = 0.0f;
    if (w.count > 0) {
        Channels<V> ch;
        fill_channels<V>(P, at, w, ch);
        const long long sample0 = at.sample * P.places * P.channels, values = P.values();
        const T *x = static_cast<const T *>(P.x), *dy = static_cast<const T *>(P.dy), *residual = static_cast<const T *>(P.residual);
        const bool with = P.residual && P.activation != kActNone;
        constexpr int N = 2;
        for (int j = 0; j < w.count; j += N) {
            Pack<T, V> vx[N], vd[N], vr[N];
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (j + k < w.count) {
                    load(x + sample0, w, j + k, vx[k], x, values);
                    load(dy + sample0, w, j + k, vd[k], dy, values);
                    if (with) load(residual + sample0, w, j + k, vr[k], residual, values);
                }
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (j + k < w.count) {
                    float dz[V], off[V];
                    slope_at<T, V>(P, ch, vx[k], vd[k], vr[k], dz, off);
                    if (!w.whole(j + k)) {
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            if (!w.has(j + k, i)) dz[i] = off[i] = 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        sum[i] += dz[i];
                        sum_off[i] = fmaf(dz[i], off[i], sum_off[i]);
                    }
                    if (P.dresidual) store(static_cast<T *>(P.dresidual) + sample0, w, j + k, dz, static_cast<T *>(P.dresidual), values);
                }
        }
    }
    if (int(threadIdx.x) < at.active) {
#pragma unroll
        for (int i = 0; i < V; ++i) entries[threadIdx.x * V + i] = make_float2(sum[i], sum_off[i]);
    }
    __syncthreads();
    const Entries E(at.active, V, at.span, shift, w.total);
    const long long to = (at.sample * P.shares + at.share) * P.channels + at.channel0;
    join_sums(entries, E, [&](int l, float a, float b) {
        if (AXC_GLOBAL_OK(to + l, P.samples * P.shares * P.channels, 515u)) P.part[to + l] = make_float2(a, b);
    });
}

// A block joins the shares of one sample's group: a warp has a channel, its lanes have shares
__global__ void __launch_bounds__(kNormThreads) norm_join_sums_kernel(const NormArgs P)
{
    after_previous();
    __shared__ float room[kNormThreads / 32];
    const long long sample = blockIdx.x / P.groups;
    const int group = int(blockIdx.x - sample * P.groups), lane = threadIdx.x & 31;
    const float r = P.statistics[blockIdx.x].y;
    float first = 0.0f, second = 0.0f;
    for (int d = threadIdx.x >> 5; d < P.each; d += kNormThreads / 32) {
        const int c = group * P.each + d;
        float a = 0.0f, b = 0.0f;
        for (long long s = lane; s < P.shares; s += 32) {
            const long long from = (sample * P.shares + s) * P.channels + c;
            if (!AXC_GLOBAL_OK(from, P.samples * P.shares * P.channels, 516u)) continue;
            a += P.part[from].x;
            b += P.part[from].y;
        }
        a = over_lanes(a, 32);
        b = over_lanes(b, 32) * r;
        if (lane == 0) {
            if (P.sums) P.sums[sample * P.channels + c] = make_float2(a, b);
            const float scale = P.scale ? load_as_float(P.scale, c, P.scale_type) : 1.0f;
            first = fmaf(scale, a, first);
            second = fmaf(scale, b, second);
        }
    }
    const float all = float(P.places) * float(P.each);
    first = over_block(first, room);
    second = over_block(second, room);
    if (threadIdx.x == 0) P.group_sums[blockIdx.x] = make_float2(__fdiv_rn(first, all) * r, __fdiv_rn(second, all) * r * r);
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 3) norm_gradient_kernel(const NormArgs P)
{
    after_previous();
    const Share at = Share::of(P, (long long)gridDim.x - 1 - blockIdx.x, std::integral_constant<int, V>());
    const Walk<V> w(threadIdx.x, at.active, shift_of<T, V>(P, at.sample, at.place0), at.places, at.span, P.channels, at.place0, at.channel0);
    if (w.count == 0) return;
    Channels<V> ch;
    fill_channels<V>(P, at, w, ch);
    float first[V], second[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const long long from = at.sample * P.groups + (at.channel0 + local_channel<V>(w, at.span, i)) / P.each;
        const float2 f = AXC_GLOBAL_OK(from, P.samples * P.groups, 517u) ? P.group_sums[from] : make_float2(0.0f, 0.0f);
        first[i] = f.x;
        second[i] = f.y;
    }
    const long long sample0 = at.sample * P.places * P.channels, values = P.values();
    const T *x = static_cast<const T *>(P.x), *dy = static_cast<const T *>(P.dy), *residual = static_cast<const T *>(P.residual);
    const bool with = P.residual && P.activation != kActNone;
    constexpr int N = 2;
    for (int j = 0; j < w.count; j += N) {
        Pack<T, V> vx[N], vd[N], vr[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (j + k < w.count) {
                load(x + sample0, w, j + k, vx[k], x, values);
                load(dy + sample0, w, j + k, vd[k], dy, values);
                if (with) load(residual + sample0, w, j + k, vr[k], residual, values);
            }
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (j + k < w.count) {
                float dz[V], off[V];
                slope_at<T, V>(P, ch, vx[k], vd[k], vr[k], dz, off);
#pragma unroll
                for (int i = 0; i < V; ++i) dz[i] = fmaf(-second[i], off[i], fmaf(dz[i], ch.factor[i], -first[i]));
                store(static_cast<T *>(P.dx) + sample0, w, j + k, dz, static_cast<T *>(P.dx), values);
            }
    }
}

// The channels' sums over the samples: 32 channels a block, its warps share the samples
__global__ void __launch_bounds__(1024) norm_parameters_kernel(const NormArgs P)
{
    after_previous();
    __shared__ float2 room[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long c = (long long)blockIdx.x * 32 + lane;
    float2 f = make_float2(0.0f, 0.0f);
    if (c < P.channels)
        for (long long n = warp; n < P.samples; n += 32) {
            if (!AXC_GLOBAL_OK(n * P.channels + c, P.samples * P.channels, 518u)) continue;
            const float2 more = P.sums[n * P.channels + c];
            f.x += more.x;
            f.y += more.y;
        }
    room[warp][lane] = f;
    __syncthreads();
    if (warp > 0 || c >= P.channels) return;
    for (int i = 1; i < 32; ++i) {
        f.x += room[i][lane].x;
        f.y += room[i][lane].y;
    }
    if (P.doffset) store_from_float(P.doffset, c, P.offset_type, f.x);
    if (P.dscale) store_from_float(P.dscale, c, P.scale_type, f.y);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
template <typename Kernel>
int allow_smem(Kernel kernel, std::atomic<unsigned long long> &ready)
{
    int device = 0;
    AXC_CUDA(cudaGetDevice(&device));
    const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
    if (!(ready.load(std::memory_order_acquire) & bit) || !bit) {
        AXC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kNormSmem)));
        ready.fetch_or(bit, std::memory_order_release);
    }
    return AXC_OK;
}

template <typename T, int V>
int forward(NormArgs P, const NormPlan &plan, Queue &q)
{
    if (plan.resident) {
        static std::atomic<unsigned long long> ready{0};
        const int rc = allow_smem(norm_forward_kernel<T, V>, ready);
        if (rc) return rc;
        return launch(q, norm_forward_kernel<T, V>, dim3(unsigned(P.samples * P.spans * P.blocks)), unsigned(plan.threads), plan.smem, unsigned(plan.blocks), P);
    }
    const dim3 grid(unsigned(P.samples * P.shares * P.spans));
    int rc = launch(q, norm_moments_kernel<T, V>, grid, kNormThreads, 0, 1, P);
    if (!rc) rc = launch(q, norm_join_kernel, dim3(unsigned(P.samples * P.groups)), kNormThreads, 0, 1, P);
    if (!rc) rc = launch(q, norm_apply_kernel<T, V>, grid, kNormThreads, 0, 1, P);
    return rc;
}

template <typename T, int V>
int backward(NormArgs P, const NormPlan &plan, Queue &q)
{
    int rc;
    if (plan.resident) {
        static std::atomic<unsigned long long> ready{0};
        rc = allow_smem(norm_backward_kernel<T, V>, ready);
        if (!rc) rc = launch(q, norm_backward_kernel<T, V>, dim3(unsigned(P.samples * P.spans * P.blocks)), unsigned(plan.threads), plan.smem, unsigned(plan.blocks), P);
    } else {
        const dim3 grid(unsigned(P.samples * P.shares * P.spans));
        rc = launch(q, norm_sums_kernel<T, V>, grid, kNormThreads, 0, 1, P);
        if (!rc) rc = launch(q, norm_join_sums_kernel, dim3(unsigned(P.samples * P.groups)), kNormThreads, 0, 1, P);
        if (!rc && P.dx) rc = launch(q, norm_gradient_kernel<T, V>, grid, kNormThreads, 0, 1, P);
    }
    return rc;
}

constexpr long long kMostBlocks = 0x7fffffffll;

int sm_count(int device, int *sms)
{
    if (device < 0) return AXC_INVALID_ARGUMENT;
    AXC_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
    return AXC_OK;
}

int check_desc(const axc_norm_desc *d)
{
    if (!d || d->samples < 0 || d->places < 0 || d->channels < 1 || d->groups < 1 || d->channels % d->groups) return AXC_INVALID_ARGUMENT;
    if (d->type < kFloat32 || d->type > kFloat16 || d->scale_type < kFloat32 || d->scale_type > kFloat16 || d->offset_type < kFloat32 || d->offset_type > kFloat16)
        return AXC_INVALID_ARGUMENT;
    if (d->activation < kActNone || d->activation > kActSilu || !(d->epsilon >= 0.0f) || !(d->epsilon <= FLT_MAX)) return AXC_INVALID_ARGUMENT;
    // sizes whose product leaves 2^60, or a line that 31 bits cannot count
    if (d->channels > (1ll << 30) || d->samples > (1ll << 31) || d->places > (1ll << 40)) return AXC_INVALID_ARGUMENT;
    if (double(d->samples) * double(d->places) * double(d->channels) > double(1ll << 60)) return AXC_INVALID_ARGUMENT;
    if (double(d->samples) * double(d->groups) > double(kMostBlocks)) return AXC_INVALID_ARGUMENT;
    return AXC_OK;
}

NormShape shape_of(const axc_norm_desc &d, bool aligned) { return {d.samples, d.places, d.channels, d.groups, d.type == kFloat32 ? 4 : 2, aligned}; }

// The plan of a call.  Searching for one takes some 20 us of the host's time, so plans are remembered: they are functions of the shape alone.
NormPlan plan_of(const NormShape &s, bool backward, bool residual, int sms)
{
    struct Known {
        NormShape shape;
        int key;
        NormPlan plan;
    };
    thread_local std::vector<Known> known(512);
    const int key = 1 + (backward ? 1 : 0) + (residual ? 2 : 0) + (s.aligned ? 4 : 0) + 8 * sms;
    unsigned long long hash = (unsigned long long)s.samples;
    for (const long long v : {s.places, s.channels, s.groups, (long long)(key * 8 + s.size)}) hash = (hash ^ (unsigned long long)v) * 0x9E3779B97F4A7C15ull, hash ^= hash >> 29;
    Known &k = known[hash % known.size()];
    if (k.key != key || k.shape.samples != s.samples || k.shape.places != s.places || k.shape.channels != s.channels || k.shape.groups != s.groups || k.shape.size != s.size)
        k = {s, key, backward ? norm_plan(s, s.size + 4, s.size * (residual ? 5 : 3), 1, sms) : norm_plan(s, s.size, s.size * (residual ? 3 : 2), 0, sms)};
    return k.plan;
}

NormArgs args_of(const axc_norm_desc &d, const NormPlan &plan)
{
    NormArgs P = {};
    P.scale_type = d.scale_type;
    P.offset_type = d.offset_type;
    P.activation = d.activation;
    P.epsilon = d.epsilon;
    P.samples = d.samples;
    P.places = d.places;
    P.channels = d.channels;
    P.groups = int(d.groups);
    P.each = int(d.channels / d.groups);
    P.span = plan.span;
    P.spans = int((d.channels + plan.span - 1) / plan.span);
    P.blocks = plan.blocks;
    P.active = norm_active(plan.threads, plan.span, plan.vec);
    P.shares = plan.shares;
    return P;
}

bool too_many(const NormArgs &P, const NormPlan &plan)
{
    return double(P.samples) * double(P.spans) * double(plan.resident ? P.blocks : P.shares) > double(kMostBlocks);
}

size_t workspace_of(const NormShape &s, const NormPlan &plan, bool backward)
{
    return norm_part_bytes(s, plan) + (backward ? norm_sums_bytes(s) + norm_group_bytes(s) : 0);
}

template <typename... P>
bool on_16(P... p) { return aligned_to(16, p...); }

template <typename Call>
int on_device(int device, Call call)
{
    int prev = 0;
    AXC_CUDA(cudaGetDevice(&prev));
    if (prev != device) AXC_CUDA(cudaSetDevice(device));
    int rc = call();
    const cudaError_t e = cudaGetLastError();
    if (!rc && e != cudaSuccess) rc = cuda_failed(e);
    if (prev != device) cudaSetDevice(prev);
    return rc;
}

}  // namespace

AXC_DEFINE_BOUNDS_READER(bounds_record_norm)

}  // namespace axc

extern "C" int axc_group_norm_workspace_bytes(const axc_norm_desc *desc, int device, size_t *forward, size_t *backward)
{
    using namespace axc;
    int rc = check_desc(desc), sms = 0;
    if (rc) return rc;
    rc = sm_count(device, &sms);
    if (rc) return rc;
    // for tensors at any address
    if (forward) *forward = 0;
    if (backward) *backward = 0;
    for (int i = 0; i < 4; ++i) {
        const NormShape s = shape_of(*desc, i & 1);
        const size_t f = workspace_of(s, plan_of(s, false, i & 2, sms), false), b = workspace_of(s, plan_of(s, true, i & 2, sms), true);
        if (forward && f > *forward) *forward = f;
        if (backward && b > *backward) *backward = b;
    }
    return AXC_OK;
}

extern "C" int axc_group_norm_forward(const axc_norm_desc *desc, const void *x, const void *scale, const void *offset, const void *residual, void *y, float *statistics,
                                      void *workspace, size_t workspace_bytes, int device, void *stream)
{
    using namespace axc;
    int rc = check_desc(desc), sms = 0;
    if (rc) return rc;
    const axc_norm_desc &d = *desc;
    if (d.samples == 0 || d.places == 0) return AXC_OK;
    if (!x || !y || !statistics) return AXC_INVALID_ARGUMENT;
    if (!aligned_to(type_size(d.type), x, residual, y) || !aligned_to(type_size(d.scale_type), scale) || !aligned_to(type_size(d.offset_type), offset) ||
        !aligned_to(8, statistics))
        return AXC_INVALID_ARGUMENT;
    rc = sm_count(device, &sms);
    if (rc) return rc;
    const NormShape s = shape_of(d, on_16(x, residual, y));
    const NormPlan plan = plan_of(s, false, residual != nullptr, sms);
    NormArgs P = args_of(d, plan);
    if (too_many(P, plan)) return AXC_INVALID_ARGUMENT;
    const size_t need = workspace_of(s, plan, false);
    if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < need)) return AXC_INTERNAL;
    P.x = x;
    P.scale = scale;
    P.offset = offset;
    P.residual = residual;
    P.y = y;
    P.statistics = reinterpret_cast<float2 *>(statistics);
    P.part = static_cast<float2 *>(workspace);
    Queue q = {cudaStream_t(stream)};
    return on_device(device, [&] {
        if (d.type == kFloat32) return plan.vec > 1 ? forward<float, 4>(P, plan, q) : forward<float, 1>(P, plan, q);
        if (d.type == kBfloat16) return plan.vec > 1 ? forward<__nv_bfloat16, 8>(P, plan, q) : forward<__nv_bfloat16, 1>(P, plan, q);
        return plan.vec > 1 ? forward<__half, 8>(P, plan, q) : forward<__half, 1>(P, plan, q);
    });
}

extern "C" int axc_group_norm_backward(const axc_norm_desc *desc, const void *dy, const void *x, const float *statistics, const void *scale, const void *offset,
                                       const void *residual, void *dx, void *dscale, void *doffset, void *dresidual, void *workspace, size_t workspace_bytes, int device,
                                       void *stream)
{
    using namespace axc;
    int rc = check_desc(desc), sms = 0;
    if (rc) return rc;
    const axc_norm_desc &d = *desc;
    const bool some = d.samples > 0 && d.places > 0;
    if (some && (!dy || !x || !statistics)) return AXC_INVALID_ARGUMENT;
    if (!some && !dscale && !doffset) return AXC_OK;
    if (!dx && !dscale && !doffset && !dresidual) return AXC_OK;
    if (!aligned_to(type_size(d.type), dy, x, residual, dx, dresidual) || !aligned_to(type_size(d.scale_type), scale, dscale) ||
        !aligned_to(type_size(d.offset_type), offset, doffset) || !aligned_to(8, statistics))
        return AXC_INVALID_ARGUMENT;
    rc = sm_count(device, &sms);
    if (rc) return rc;
    const NormShape s = shape_of(d, on_16(dy, x, residual, dx, dresidual));
    const NormPlan plan = plan_of(s, true, residual != nullptr, sms);
    NormArgs P = args_of(d, plan);
    if (too_many(P, plan)) return AXC_INVALID_ARGUMENT;
    if (some && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < workspace_of(s, plan, true))) return AXC_INTERNAL;
    P.dy = dy;
    P.x = x;
    P.statistics = reinterpret_cast<float2 *>(const_cast<float *>(statistics));
    P.scale = scale;
    P.offset = offset;
    P.residual = residual;
    P.dx = dx;
    P.dscale = dscale;
    P.doffset = doffset;
    P.dresidual = dresidual;
    char *ws = static_cast<char *>(workspace);
    P.part = reinterpret_cast<float2 *>(ws);
    P.sums = dscale || doffset ? reinterpret_cast<float2 *>(ws + norm_part_bytes(s, plan)) : nullptr;
    P.group_sums = reinterpret_cast<float2 *>(ws + norm_part_bytes(s, plan) + norm_sums_bytes(s));
    if (!some) P.samples = 0;
    Queue q = {cudaStream_t(stream)};
    return on_device(device, [&] {
        int rc = AXC_OK;
        if (some) {
            if (d.type == kFloat32) rc = plan.vec > 1 ? backward<float, 4>(P, plan, q) : backward<float, 1>(P, plan, q);
            else if (d.type == kBfloat16) rc = plan.vec > 1 ? backward<__nv_bfloat16, 8>(P, plan, q) : backward<__nv_bfloat16, 1>(P, plan, q);
            else rc = plan.vec > 1 ? backward<__half, 8>(P, plan, q) : backward<__half, 1>(P, plan, q);
        }
        if (!rc && (dscale || doffset)) rc = launch(q, norm_parameters_kernel, dim3(unsigned((P.channels + 31) / 32)), 1024, 0, 1, P);
        return rc;
    });
}
