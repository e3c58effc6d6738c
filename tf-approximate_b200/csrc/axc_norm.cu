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
// has, at its start or its end, is moved value by value.  Where the order of the channels repeats after more vectors than a block has threads (channels / gcd(channels,
// values of a vector) > 256: 777 channels of fp16), or a tensor does not start on 16 bytes, all values are moved one by one: 64 x 56 x 56 x 777 fp16, silu, takes 931 us forward and
// 1740 backward, with 776 channels 240 and 389.
//
// Sums are fp32.  Those of the variance are never of squares that nearly cancel: a thread adds the squares of up to 32 values less the first of them,
// and means and squared distances are joined by their means (Chan, Golub and LeVeque).  Every sum has a fixed order.
// Roundings to 16 bits: the outputs alone.  dx is a difference: where dz is nearly the same all over a group, as behind a mean over the places, next to
// nothing of it is left, and a dz rounded to bf16 on the way makes dx off by 43 % (dy = 1, silu, an offset of 6).  So a resident block holds dz in fp32, in
// the places of dy and of the residual together, and without a residual keeps dy and computes the slope again: fp32 places of its own would take half
// as much shared memory again, which is what bounds how many loads are on their way (256 x 56 x 56 x 256 bf16, silu: 499 us, the slope again 428, a rounded dz 376).
//
// Measured (256 x 56 x 56 x 256 bf16, groups of 8, shortcut, silu; us, bytes at memory's rate in brackets): forward 274 to 286 (188), backward 565 to 571
// (314), the latter bound by instructions and by the time between a block's phases; without the shortcut 203 (126) and 428 (188).  The first two with the tensors
// read twice: 307 and 638.
// 2 x 512 x 512 x 128 bf16, which no cluster holds: 88 (41) and 134 (61).
#include <type_traits>

#include "axc_gemm.h"
#include "axc_mma.cuh"
#include "axc_norm_plan.h"
#include "axc_two.cuh"

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
    Span span, last;                           // of a block; the last one of a line may be narrower where the tensors are read twice
    int spans, blocks;                         // spans of a line, blocks that share one
    long long per;                             // places of a block; the last one has the rest
    int steps, span_groups;                    // resident: steps that the threads take, groups of a span
    bool whole_vectors;                        // a thread's channels are neighbours, and of one group
    Span vectors;                              // then: the span's vectors in place of its channels
    Divider by_group;                          // channels of a group
    int entries, lanes;                        // norm_entries, norm_lanes
    bool single;                               // resident, one sample: no launch for the parameters' gradients
    long long shares;
    float2 *part;                              // [samples][shares][channels] sums of a share of the places
    float2 *sums;                              // [samples][channels] {sum of dz, sum of dz xhat}; may be NULL
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
    return V == 1 || P.span.channels < P.channels ? 0 : int((sample * P.places + place0) * P.channels & (V - 1));
}

// Pairs that hold V values; a single one has nothing beside it
template <int V> constexpr int kPairs = (V + 1) / 2;

template <typename T, int V>
__device__ __forceinline__ void widen_pairs(const Pack<T, V> &v, Two (&x)[kPairs<V>])
{
    if constexpr (V == 1) x[0] = Two(widen(v.t[0]), 0.0f);
    else {
        const unsigned w[4] = {v.w.x, v.w.y, v.w.z, v.w.w};
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            if constexpr (sizeof(T) == 4) x[i] = Two(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
            else if constexpr (std::is_same<T, __nv_bfloat16>::value) x[i] = Two(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            else {
                const float2 f = __half22float2(reinterpret_cast<const __half2 &>(w[i]));
                x[i] = Two(f.x, f.y);
            }
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> narrow_pairs(const Two (&x)[kPairs<V>])
{
    Pack<T, V> v;
    if constexpr (V == 1) v.t[0] = narrow<T>(x[0].both().x);
    else {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 f = x[i].both();
            if constexpr (sizeof(T) == 4) {
                w[2 * i] = __float_as_uint(f.x);
                w[2 * i + 1] = __float_as_uint(f.y);
            } else w[i] = pack2(f.x, f.y, std::is_same<T, __nv_bfloat16>::value);
        }
        v.w = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
}
__device__ __forceinline__ void set_lane(Two &x, int lane, float v)
{
    const float2 f = x.both();
    x = lane ? Two(f.x, v) : Two(v, f.y);
}

// The j-th vector of a tensor, at `from`: whole, or value by value where some are outside of the block's.  base, count: all there is.
template <bool WHOLE, typename T, int V>
__device__ __forceinline__ void load(const T *from, const Walk<V> &w, int j, Pack<T, V> &v, [[maybe_unused]] const T *base, [[maybe_unused]] long long count)
{
    if (WHOLE) {
        if (AXC_VALUES_OK(from, V, base, count, 501u)) v.w = *reinterpret_cast<const typename Bits<V * sizeof(T)>::type *>(from);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v.t[i] = w.has(j, i) && AXC_VALUES_OK(from + i, 1, base, count, 502u) ? from[i] : narrow<T>(0.0f);
    }
}
template <bool WHOLE, typename T, int V>
__device__ __forceinline__ void store(T *to, const Walk<V> &w, int j, const Two (&x)[kPairs<V>], [[maybe_unused]] T *base, [[maybe_unused]] long long count)
{
    const Pack<T, V> v = narrow_pairs<T, V>(x);
    if (WHOLE) {
        if (AXC_VALUES_OK(to, V, base, count, 503u)) *reinterpret_cast<typename Bits<V * sizeof(T)>::type *>(to) = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (w.has(j, i) && AXC_VALUES_OK(to + i, 1, base, count, 504u)) to[i] = v.t[i];
    }
}

// body(whole, how many, the first) for all vectors of a thread, N whole ones at a time as long as there are so many
template <int V, typename N, typename Body>
__device__ __forceinline__ void batches(const Walk<V> &w, N n, Body body)
{
    const std::integral_constant<int, 1> one;
    int j = w.first;
    for (; j + N::value <= w.end; j += N::value) body(std::true_type(), n, j);
    for (; j < w.end; ++j) body(std::true_type(), one, j);
    if constexpr (V > 1) {
        if (w.first > 0) body(std::false_type(), one, 0);
        if (w.end < w.count) body(std::false_type(), one, w.end);
    }
}

// All vectors of a thread into its own places of shared memory, `stride` apart, asynchronously where there is a copy of that size: nothing waits
// for one before the next is on its way, and what a thread has copied it alone reads, after wait_copies().
template <typename T, int V, typename Word>
__device__ __forceinline__ void fetch(const T *sample, const Walk<V> &w, Word *to, int stride, const T *base, long long count)
{
    constexpr int kBytes = V * sizeof(T);
    if constexpr (kBytes >= 4) {
        const T *from = sample + w.at + w.first * w.step;
        unsigned place = mma::smem_address(to) + unsigned(w.first * stride) * unsigned(sizeof(Word));
#pragma unroll 4
        for (int j = w.first; j < w.end; ++j) {
            if (AXC_VALUES_OK(from, V, base, count, 519u)) {
                if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(place), "l"(from) : "memory");
                else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(place), "l"(from) : "memory");
            }
            from += w.step;
            place += unsigned(stride) * unsigned(sizeof(Word));
        }
        if constexpr (V > 1) {
            for (int side = 0; side < 2; ++side) {
                if (side == 0 ? w.first == 0 : w.end == w.count) continue;
                const int j = side == 0 ? 0 : w.end;
                Pack<T, V> v;
                load<false>(sample + w.at + j * w.step, w, j, v, base, count);
                to[j * stride] = v.w;
            }
        }
    } else {
        constexpr int N = 8;
        for (int j = 0; j < w.count; j += N) {
            Pack<T, V> v[N];
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (j + k < w.count) load<true>(sample + w.at + (j + k) * w.step, w, j + k, v[k], base, count);
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (j + k < w.count) to[(j + k) * stride] = v[k].w;
        }
    }
}
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <int H, bool EXACT>
__device__ __forceinline__ void activate_pairs(Two (&z)[H], int act)
{
    if (act == kActNone) return;
    if (act == kActSilu) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if constexpr (EXACT) {
                const float2 f = z[i].both();
                z[i] = Two(activate(f.x, kActSilu, true), activate(f.y, kActSilu, true));
            } else z[i] = mul2(z[i], sigmoid2(z[i]));
        }
    } else if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const float2 f = z[i].both();
            z[i] = Two(activate(f.x, kActRelu, EXACT), activate(f.y, kActRelu, EXACT));
        }
    } else {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if constexpr (EXACT) {
                const float2 f = z[i].both();
                z[i] = Two(activate(f.x, kActGelu, true), activate(f.y, kActGelu, true));
            } else {
                Two bell;
                z[i] = mul2(z[i], normal_below2(z[i], bell));
            }
        }
    }
}
// d *= act'(z)
template <int ACT, bool EXACT>
__device__ __forceinline__ Two slope2(Two z)
{
    const float2 f = z.both();
    return Two(slope_of<ACT, EXACT>(f.x), slope_of<ACT, EXACT>(f.y));
}
template <int H, bool EXACT>
__device__ __forceinline__ void slopes(Two (&d)[H], const Two (&z)[H], int act)
{
    if (act == kActSilu) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if constexpr (EXACT) d[i] = mul2(d[i], slope2<kActSilu, true>(z[i]));
            else {
                const Two s = sigmoid2(z[i]);
                d[i] = mul2(d[i], mul2(s, fma2(z[i], fma2(s, Two(-1.0f), Two(1.0f)), Two(1.0f))));
            }
        }
    } else if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < H; ++i) d[i] = mul2(d[i], slope2<kActRelu, EXACT>(z[i]));
    } else {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if constexpr (EXACT) d[i] = mul2(d[i], slope2<kActGelu, true>(z[i]));
            else {
                Two bell;
                const Two below = normal_below2(z[i], bell);
                d[i] = mul2(d[i], fma2(mul2(z[i], bell), Two(0.39894228f), below));
            }
        }
    }
}

// Mean and sum of squared distances from it, for each of a thread's channels.  Values are counted from the first of a run of up to kRun, so the
// sum of their squares is at most as many times that of the distances from the mean as the run has values, whatever they are: the difference
// loses no more than that.  Runs are joined by their means.
constexpr int kRun = 32;
template <int V>
struct Moments {
    static constexpr int H = kPairs<V>;
    float n = 0.0f;                            // whole vectors in the runs that are over
    Two mean[H], square[H];
    Two pivot[H], sum[H], squares[H];          // of this run
    template <typename T>
    __device__ __forceinline__ void open(const Pack<T, V> &v)
    {
        widen_pairs<T, V>(v, pivot);
#pragma unroll
        for (int i = 0; i < H; ++i) {
            pivot[i] = mul2(pivot[i], Two(-1.0f));
            sum[i] = squares[i] = Two(0.0f);
        }
    }
    template <typename T>
    __device__ __forceinline__ void add(const Pack<T, V> &v)
    {
        Two x[H];
        widen_pairs<T, V>(v, x);
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const Two d = add2(x[i], pivot[i]);
            sum[i] = add2(sum[i], d);
            squares[i] = fma2(d, d, squares[i]);
        }
    }
    // `k`: values of the run
    __device__ __forceinline__ void close(float k)
    {
        const float all = n + k, w = __fdividef(k, all);
        const Two share(__fdividef(1.0f, k)), minus(-1.0f), w1(w), w2(n * w);
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const Two m = mul2(sum[i], share), q = fma2(mul2(m, minus), sum[i], squares[i]), at = fma2(pivot[i], minus, m);
            if (n == 0.0f) {
                mean[i] = at;
                square[i] = q;
            } else {
                const Two d = fma2(mean[i], minus, at);
                mean[i] = fma2(d, w1, mean[i]);
                square[i] = fma2(mul2(d, d), w2, add2(square[i], q));
            }
        }
        n = all;
    }
    // one value of channel i, which has had `k` so far
    __device__ __forceinline__ void add_one(int i, float v, float k)
    {
        const float2 m2 = mean[i / 2].both(), s2 = square[i / 2].both();
        float m = i & 1 ? m2.y : m2.x, s = i & 1 ? s2.y : s2.x;
        if (k == 0.0f) {
            m = v;
            s = 0.0f;
        } else {
            const float d = v - m;
            m += __fdividef(d, k + 1.0f);
            s = fmaf(d, v - m, s);
        }
        set_lane(mean[i / 2], i & 1, m);
        set_lane(square[i / 2], i & 1, s);
    }
    __device__ __forceinline__ float2 of(int i) const
    {
        const float2 m = mean[i / 2].both(), s = square[i / 2].both();
        return i & 1 ? make_float2(m.y, fmaxf(s.y, 0.0f)) : make_float2(m.x, fmaxf(s.x, 0.0f));
    }
};

// The moments of a thread's vectors; get(j, vector, whether it is whole) has the j-th, N of them at a time
template <int N, typename T, int V, typename Get>
__device__ __forceinline__ void take_moments(const Walk<V> &w, Moments<V> &mo, Get get)
{
    for (int j0 = w.first; j0 < w.end; j0 += kRun) {
        const int end = min(j0 + kRun, w.end);
        int j = j0;
        for (; j + N <= end; j += N) {
            Pack<T, V> v[N];
#pragma unroll
            for (int k = 0; k < N; ++k) get(j + k, v[k], std::true_type());
            if (j == j0) mo.open(v[0]);
#pragma unroll
            for (int k = 0; k < N; ++k) mo.add(v[k]);
        }
        for (; j < end; ++j) {
            Pack<T, V> v;
            get(j, v, std::true_type());
            if (j == j0) mo.open(v);
            mo.add(v);
        }
        mo.close(float(end - j0));
    }
    if constexpr (V > 1) {
        if (w.first > 0 || w.end < w.count) {
            float had[V];
#pragma unroll
            for (int i = 0; i < V; ++i) had[i] = mo.n;
            for (int side = 0; side < 2; ++side) {
                if (side == 0 ? w.first == 0 : w.end == w.count) continue;
                const int at = side == 0 ? 0 : w.end;
                Pack<T, V> v;
                get(at, v, std::false_type());
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (w.has(at, i)) {
                        mo.add_one(i, widen(v.t[i]), had[i]);
                        had[i] += 1.0f;
                    }
            }
        }
    }
}

// ---- sums over the threads of a block ------------------------------------------------------------------------------------------
// Lanes that share one of `items` sums, as a power of two: all 32, or what the block's threads allow
__device__ __forceinline__ int lanes_for(int items)
{
    const int each = int(blockDim.x) >= 32 * items ? 5 : 31 - __clz(max(1, int(float(blockDim.x) / float(items))));
    return each;
}
__device__ __forceinline__ float over_lanes(float x, int log2)
{
#pragma unroll
    for (int o = 4; o >= 0; --o)
        if (o < log2) x += __shfl_xor_sync(0xffffffffu, x, 1 << o);
    return x;
}

// A thread's sums into their places
template <int V, typename Get>
__device__ __forceinline__ void give_entries(float2 *entries, const Span &s, Get get)
{
    int e = int(threadIdx.x) * V, copy = int(s.by_channels.of(unsigned(e))), left = s.channels - (e - copy * s.channels);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        entries[e + copy] = get(i);
        ++e;
        if (--left == 0) ++copy, left = s.channels;
    }
}

// {mean, squared distances} of `items` neighbouring sets of `each` channels, from the threads' entries, `of_entry` values each for every one that the
// entry counts: give(item, mean, square) in one thread
template <typename Give>
__device__ __forceinline__ void join_moments(const float2 *entries, const Entries &E, const Divider &by_copies, int items, int each, float values, float of_entry, Give give)
{
    const int log2 = lanes_for(items), q = 1 << log2, lane = threadIdx.x & (q - 1), step = int(blockDim.x) >> log2, all = each * E.copies;
    const float share = __fdividef(1.0f, values);
    for (int first = 0; first < items; first += step) {
        const int item = first + (int(threadIdx.x) >> log2), end = item < items ? all : 0;
        // f(values of it, the entry)
        auto each_entry = [&](auto f) {
            for (int i = lane; i < end; i += q) {
                const int d = int(by_copies.of(unsigned(i))), k = i - d * E.copies, e = E.first_entry(item * each + d) + k * E.span;
                const float n = of_entry * E.values(e);
                if (n > 0.0f) f(n, entries[E.place(e, k)]);
            }
        };
        float sum = 0.0f, square = 0.0f;
        each_entry([&](float n, float2 f) { sum = fmaf(n, f.x, sum); });
        const float mean = over_lanes(sum, log2) * share;
        each_entry([&](float n, float2 f) { square += fmaf(n * (f.x - mean), f.x - mean, f.y); });
        square = over_lanes(square, log2);
        if (item < items && lane == 0) give(item, mean, square);
    }
}

// Sums of pairs, for every channel of the span
template <typename Give>
__device__ __forceinline__ void join_sums(const float2 *entries, const Entries &E, Give give)
{
    const int log2 = lanes_for(E.span), q = 1 << log2, lane = threadIdx.x & (q - 1), step = int(blockDim.x) >> log2;
    for (int first = 0; first < E.span; first += step) {
        const int l = first + (int(threadIdx.x) >> log2);
        float a = 0.0f, b = 0.0f;
        if (l < E.span) {
            const float2 *from = entries + E.first_entry(l);
            for (int k = lane; k < E.copies; k += q) {
                const float2 f = from[k * (E.span + 1)];
                a += f.x;
                b += f.y;
            }
        }
        a = over_lanes(a, log2);
        b = over_lanes(b, log2);
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

// The same for all blocks of the cluster, all of them on their way at once; what lies behind the last block is this block's own, not used
__device__ __forceinline__ void of_all(const float2 *at, int blocks, float2 (&f)[kNormCluster])
{
#pragma unroll
    for (int r = 0; r < kNormCluster; ++r) f[r] = of_block(at, r < blocks ? r : 0);
}
__device__ __forceinline__ float2 sum_of_all(const float2 *at, int blocks)
{
    float2 f[kNormCluster], sum = make_float2(0.0f, 0.0f);
    of_all(at, blocks, f);
#pragma unroll
    for (int r = 0; r < kNormCluster; ++r)
        if (r < blocks) {
            sum.x += f[r].x;
            sum.y += f[r].y;
        }
    return sum;
}

// Where a resident block is
struct Place {
    long long sample, sample0;
    int rank, span, channel0, place0, places;
    __device__ __forceinline__ explicit Place(const NormArgs &P)
    {
        unsigned unit = blockIdx.x, n;
        rank = 0;
        if (P.blocks > 1) {
            rank = int(mma::cluster_rank());
            asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(unit));
        }
        n = P.spans > 1 ? unit / unsigned(P.spans) : unit;
        sample = n;
        sample0 = sample * P.places * P.channels;
        span = int(unit - n * unsigned(P.spans));
        channel0 = span * P.span.channels;
        place0 = rank * int(P.per);
        places = min(int(P.per), int(P.places) - place0);
    }
};

// A parameter at V channels, `none` where there is none; in_line: the channels are neighbours
template <int V>
__device__ __forceinline__ void load_parameters(const void *from, int type, const int (&c)[V], bool in_line, [[maybe_unused]] long long count, float none, float (&out)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = none;
    if (!from) return;
    if (type == kFloat32 && in_line) {
        const float *at = static_cast<const float *>(from) + c[0];
        if (!AXC_VALUES_OK(at, V, static_cast<const float *>(from), count, 505u)) return;
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = at[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (AXC_GLOBAL_OK(c[i], count, 506u)) out[i] = load_as_float(from, c[i], type);
    }
}

// What a thread needs of its channels
template <int V>
struct Channels {
    static constexpr int H = kPairs<V>;
    Two less[H], factor[H], offset[H];         // less: the mean with its sign turned
    // stats(group of the span): {mean, r}; in_line: the channels are neighbours, and of one group
    template <typename Stats>
    __device__ __forceinline__ void fill(const NormArgs &P, int channel0, const int (&local)[V], const int (&group)[V], bool in_line, Stats stats)
    {
        int c[V];
        float a[V], b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = channel0 + local[i];
        load_parameters<V>(P.scale, P.scale_type, c, in_line, P.channels, 1.0f, a);
        load_parameters<V>(P.offset, P.offset_type, c, in_line, P.channels, 0.0f, b);
        const float2 s0 = stats(group[0]);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const int k = V > 1 ? i + 1 : i;
            const float2 s = in_line ? s0 : stats(group[i]), t = in_line ? s0 : stats(group[k]);
            less[i / 2] = Two(-s.x, -t.x);
            factor[i / 2] = Two(a[i] * s.y, a[k] * t.y);
            offset[i / 2] = Two(b[i], b[k]);
        }
    }
};

// y of one vector
template <typename T, int V>
__device__ __forceinline__ void output_of(const NormArgs &P, const Channels<V> &ch, const Pack<T, V> &x, const Pack<T, V> &residual, Two (&z)[kPairs<V>])
{
    constexpr int H = kPairs<V>;
    widen_pairs<T, V>(x, z);
#pragma unroll
    for (int i = 0; i < H; ++i) z[i] = fma2(add2(z[i], ch.less[i]), ch.factor[i], ch.offset[i]);
    if (P.residual) {
        Two r[H];
        widen_pairs<T, V>(residual, r);
#pragma unroll
        for (int i = 0; i < H; ++i) z[i] = add2(z[i], r[i]);
    }
    activate_pairs<H, sizeof(T) == 4>(z, P.activation);
}

// dz of one vector, and x less its mean
template <typename T, int V>
__device__ __forceinline__ void slope_at(const NormArgs &P, const Channels<V> &ch, const Pack<T, V> &x, const Pack<T, V> &dy, const Pack<T, V> &residual,
                                         Two (&dz)[kPairs<V>], Two (&off)[kPairs<V>])
{
    constexpr int H = kPairs<V>;
    widen_pairs<T, V>(x, off);
    widen_pairs<T, V>(dy, dz);
#pragma unroll
    for (int i = 0; i < H; ++i) off[i] = add2(off[i], ch.less[i]);
    if (P.activation == kActNone) return;
    Two z[H];
#pragma unroll
    for (int i = 0; i < H; ++i) z[i] = fma2(off[i], ch.factor[i], ch.offset[i]);
    if (P.residual) {
        Two r[H];
        widen_pairs<T, V>(residual, r);
#pragma unroll
        for (int i = 0; i < H; ++i) z[i] = add2(z[i], r[i]);
    }
    slopes<H, sizeof(T) == 4>(dz, z, P.activation);
}
// Sums of dz and of dz (x - mean); values outside of a block's are left out (their x and dy are zeros, which is not enough)
template <int V>
struct Sums {
    static constexpr int H = kPairs<V>;
    Two dz[H], off[H];
    // of more than a run of values, which are added up by themselves first, so that no chain of additions is longer than one
    __device__ __forceinline__ void take(Sums &run)
    {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            dz[i] = add2(dz[i], run.dz[i]);
            off[i] = add2(off[i], run.off[i]);
            run.dz[i] = run.off[i] = Two(0.0f);
        }
    }
    __device__ __forceinline__ Sums()
    {
#pragma unroll
        for (int i = 0; i < H; ++i) dz[i] = off[i] = Two(0.0f);
    }
    template <bool WHOLE>
    __device__ __forceinline__ void add(const Walk<V> &w, int j, Two (&d)[H], const Two (&o)[H])
    {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if (!WHOLE) {
                const float2 f = d[i].both();
                d[i] = Two(w.has(j, 2 * i) ? f.x : 0.0f, w.has(j, 2 * i + 1) ? f.y : 0.0f);
            }
            dz[i] = add2(dz[i], d[i]);
            off[i] = fma2(d[i], o[i], off[i]);
        }
    }
    // of all lanes of the warp whose number is this one's modulo `period`
    __device__ __forceinline__ void over_lanes(int period)
    {
        for (int o = 16; o >= period; o >>= 1) {
#pragma unroll
            for (int i = 0; i < H; ++i) {
                Two a, b;
                a.v = __shfl_xor_sync(0xffffffffu, dz[i].v, o);
                b.v = __shfl_xor_sync(0xffffffffu, off[i].v, o);
                dz[i] = add2(dz[i], a);
                off[i] = add2(off[i], b);
            }
        }
    }
    __device__ __forceinline__ float2 of(int i) const
    {
        const float2 a = dz[i / 2].both(), b = off[i / 2].both();
        return i & 1 ? make_float2(a.y, b.y) : make_float2(a.x, b.x);
    }
};
// fp32 values of one vector in the places of two 16-bit ones
template <int V, typename Word>
__device__ __forceinline__ void split_pairs(const Two (&x)[kPairs<V>], Word &a, Word &b)
{
    if constexpr (V == 1) {
        const unsigned w = __float_as_uint(x[0].both().x);
        a = Word(w & 0xffffu);
        b = Word(w >> 16);
    } else {
        static_assert(V == 8, "16 bytes are four of them");
        const float2 f[4] = {x[0].both(), x[1].both(), x[2].both(), x[3].both()};
        a = make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
        b = make_uint4(__float_as_uint(f[2].x), __float_as_uint(f[2].y), __float_as_uint(f[3].x), __float_as_uint(f[3].y));
    }
}
template <int V, typename Word>
__device__ __forceinline__ void join_pairs(const Word &a, const Word &b, Two (&x)[kPairs<V>])
{
    if constexpr (V == 1) x[0] = Two(__uint_as_float(unsigned(a) | unsigned(b) << 16), 0.0f);
    else {
        x[0] = Two(__uint_as_float(a.x), __uint_as_float(a.y));
        x[1] = Two(__uint_as_float(a.z), __uint_as_float(a.w));
        x[2] = Two(__uint_as_float(b.x), __uint_as_float(b.y));
        x[3] = Two(__uint_as_float(b.z), __uint_as_float(b.w));
    }
}
// dx = dz factor - first - (x - mean) second
template <int V>
struct Gradient {
    static constexpr int H = kPairs<V>;
    Two first[H], second[H];                   // both with their signs turned
    template <typename Stats>
    __device__ __forceinline__ void fill(const int (&group)[V], bool in_line, Stats stats)
    {
        const float2 s0 = stats(group[0]);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 s = in_line ? s0 : stats(group[i]), t = in_line ? s0 : stats(group[V > 1 ? i + 1 : i]);
            first[i / 2] = Two(-s.x, -t.x);
            second[i / 2] = Two(-s.y, -t.y);
        }
    }
    __device__ __forceinline__ void of(const Channels<V> &ch, const Two (&off)[H], Two (&d)[H]) const
    {
#pragma unroll
        for (int i = 0; i < H; ++i) d[i] = fma2(second[i], off[i], fma2(d[i], ch.factor[i], first[i]));
    }
};

// ---- resident spans -------------------------------------------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 3) norm_forward_kernel(const NormArgs P)
{
    after_previous();
    extern __shared__ __align__(16) char raw[];
    const Place at(P);
    const int shift = shift_of<T, V>(P, at.sample, at.place0), thread = threadIdx.x, groups = P.span_groups, stride = P.span.active;
    const Walk<V> w(thread, P.span, shift, at.places, P.channels, at.place0, at.channel0);
    typedef typename Bits<V * sizeof(T)>::type Word;
    const size_t room = norm_up16(size_t(P.steps) * P.span.active * V * sizeof(T));
    Word *kept = reinterpret_cast<Word *>(raw) + thread;
    float2 *entries = reinterpret_cast<float2 *>(raw + room);
    float2 *mine = entries + P.entries, *result = mine + groups;
    const T *x = static_cast<const T *>(P.x), *residual = static_cast<const T *>(P.residual);
    fetch<T, V>(x + at.sample0, w, kept, stride, x, P.values());
    wait_copies();
    Moments<V> mo;
    take_moments<2, T, V>(w, mo, [&](int j, Pack<T, V> &v, auto) { v.w = kept[j * stride]; });
    const float all = float(P.places) * float(P.each), part = float(at.places) * float(P.each);
    if (P.whole_vectors) {
        // a thread's channels are all of one group: one entry for them
        if (thread < P.span.active) {
            float mean = 0.0f, square = 0.0f;
            if (w.count > 0) {
#pragma unroll
                for (int i = 0; i < V; ++i) mean += mo.of(i).x;
                mean *= 1.0f / V;
#pragma unroll
                for (int i = 0; i < V; ++i) square += fmaf(mo.n * (mo.of(i).x - mean), mo.of(i).x - mean, mo.of(i).y);
            }
            give_entries<1>(entries, P.vectors, [&](int) { return make_float2(mean, square); });
        }
        __syncthreads();
        const Entries E(P.vectors, 0, at.places * P.vectors.channels);
        join_moments(entries, E, P.vectors.by_copies, groups, P.each / V, part, float(V), [&](int g, float mean, float square) { mine[g] = make_float2(mean, square); });
    } else {
        if (thread < P.span.active) give_entries<V>(entries, P.span, [&](int i) { return mo.of(i); });
        __syncthreads();
        const Entries E(P.span, shift, w.total);
        join_moments(entries, E, P.span.by_copies, groups, P.each, part, 1.0f, [&](int g, float mean, float square) { mine[g] = make_float2(mean, square); });
    }
    __syncwarp();
    if (P.blocks > 1) mma::cluster_sync();
    else __syncthreads();
    for (int g = thread; g < groups; g += blockDim.x) {
        float2 f = mine[g];
        if (P.blocks > 1) {
            float2 other[kNormCluster];
            of_all(mine + g, P.blocks, other);
            const float n = float(int(P.per)) * float(P.each), last = float(int(P.places) - int(P.per) * (P.blocks - 1)) * float(P.each);
            float sum = 0.0f, square = 0.0f;
#pragma unroll
            for (int r = 0; r < kNormCluster; ++r)
                if (r < P.blocks) sum = fmaf(r + 1 < P.blocks ? n : last, other[r].x, sum);
            const float mean = __fdiv_rn(sum, all);
#pragma unroll
            for (int r = 0; r < kNormCluster; ++r)
                if (r < P.blocks) square += fmaf((r + 1 < P.blocks ? n : last) * (other[r].x - mean), other[r].x - mean, other[r].y);
            f = make_float2(mean, square);
        }
        f.y = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(f.y, all) + P.epsilon));
        result[g] = f;
        const long long to = at.sample * P.groups + at.span * groups + g;
        if (at.rank == 0 && AXC_GLOBAL_OK(to, P.samples * P.groups, 507u)) P.statistics[to] = f;
    }
    __syncthreads();
    if (P.blocks > 1) cluster_arrive();
    int local[V], group[V];
    local_channels<V>(w, P.span, P.by_group, local, group);
    Channels<V> ch;
    ch.fill(P, at.channel0, local, group, P.whole_vectors, [&](int g) { return result[g]; });
    T *y = static_cast<T *>(P.y);
    batches<V>(w, std::integral_constant<int, 4>(), [&](auto whole, auto n, int j) {
        constexpr int N = decltype(n)::value;
        const long long from = at.sample0 + w.at + j * w.step;
        Pack<T, V> r[N];
        if (P.residual) {
#pragma unroll
            for (int k = 0; k < N; ++k) load<decltype(whole)::value>(residual + from + k * w.step, w, j + k, r[k], residual, P.values());
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            Pack<T, V> v;
            v.w = kept[(j + k) * stride];
            Two z[kPairs<V>];
            output_of<T, V>(P, ch, v, r[k], z);
            store<decltype(whole)::value>(y + from + k * w.step, w, j + k, z, y, P.values());
        }
    });
    __syncwarp();
    if (P.blocks > 1) cluster_wait();          // what others read of this block's shared memory
}

// AGAIN: the slope is computed a second time for dx (an activation, 16-bit types, no residual)
template <typename T, int V, bool AGAIN>
__global__ void __launch_bounds__(kNormThreads, 2) norm_backward_kernel(const NormArgs P)
{
    after_previous();
    extern __shared__ __align__(16) char raw[];
    const Place at(P);
    const int shift = shift_of<T, V>(P, at.sample, at.place0), thread = threadIdx.x, groups = P.span_groups, stride = P.span.active;
    const Walk<V> w(thread, P.span, shift, at.places, P.channels, at.place0, at.channel0);
    typedef typename Bits<V * sizeof(T)>::type Word;
    const bool with = !AGAIN && P.residual && P.activation != kActNone;
    const size_t room = norm_up16(size_t(P.steps) * P.span.active * V * sizeof(T));
    Word *kept = reinterpret_cast<Word *>(raw) + thread, *kept_dz = reinterpret_cast<Word *>(raw + room) + thread;      // dy's, first
    Word *kept_residual = reinterpret_cast<Word *>(raw + 2 * room) + thread;
    float2 *entries = reinterpret_cast<float2 *>(raw + (with ? 3 : 2) * room);
    float2 *channels = entries + P.entries, *mine = channels + P.span.channels, *result = mine + groups;
    const long long values = P.values();
    const T *x = static_cast<const T *>(P.x), *dy = static_cast<const T *>(P.dy), *residual = static_cast<const T *>(P.residual);
    fetch<T, V>(x + at.sample0, w, kept, stride, x, values);
    fetch<T, V>(dy + at.sample0, w, kept_dz, stride, dy, values);
    if (with) fetch<T, V>(residual + at.sample0, w, kept_residual, stride, residual, values);
    const float2 *statistics = P.statistics + at.sample * P.groups + at.span * groups;
    [[maybe_unused]] const long long in_statistics = P.samples * P.groups - (at.sample * P.groups + at.span * groups);
    auto stats = [&](int g) { return AXC_GLOBAL_OK(g, in_statistics, 508u) ? statistics[g] : make_float2(0.0f, 0.0f); };
    int local[V], group[V];
    local_channels<V>(w, P.span, P.by_group, local, group);
    Channels<V> ch;
    ch.fill(P, at.channel0, local, group, P.whole_vectors, stats);
    Sums<V> sums;
    T *dresidual = static_cast<T *>(P.dresidual);
    wait_copies();
    batches<V>(w, std::integral_constant<int, 2>(), [&](auto whole, auto n, int j) {
        constexpr int N = decltype(n)::value;
        const long long from = at.sample0 + w.at + j * w.step;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            Pack<T, V> vx, vd, vr;
            vx.w = kept[(j + k) * stride];
            vd.w = kept_dz[(j + k) * stride];
            if (with) vr.w = kept_residual[(j + k) * stride];
            Two dz[kPairs<V>], off[kPairs<V>];
            slope_at<T, V>(P, ch, vx, vd, vr, dz, off);
            sums.template add<decltype(whole)::value>(w, j + k, dz, off);
            if constexpr (sizeof(T) == 4) {
                if (P.activation != kActNone) kept_dz[(j + k) * stride] = narrow_pairs<T, V>(dz).w;
            } else if (with) split_pairs<V>(dz, kept_dz[(j + k) * stride], kept_residual[(j + k) * stride]);
            if (dresidual) store<decltype(whole)::value>(dresidual + from + k * w.step, w, j + k, dz, dresidual, values);
        }
    });
    Entries E(P.span, shift, w.total);
    if (P.lanes) {
        // (every thread takes part, and no line starts inside 16 bytes)
        sums.over_lanes(P.lanes);
        E.copies = int(blockDim.x) / 32;
        if ((thread & 31) < P.lanes) {
            float2 *to = entries + (thread >> 5) * (P.span.channels + 1) + (thread & 31) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) to[i] = sums.of(i);
        }
    } else if (thread < P.span.active) give_entries<V>(entries, P.span, [&](int i) { return sums.of(i); });
    __syncthreads();
    join_sums(entries, E, [&](int l, float a, float b) { channels[l] = make_float2(a, b); });
    __syncthreads();
    {
        const int log2 = lanes_for(groups), q = 1 << log2, lane = thread & (q - 1), step = int(blockDim.x) >> log2;
        for (int first = 0; first < groups; first += step) {
            const int g = first + (thread >> log2);
            float a = 0.0f, b = 0.0f;
            if (g < groups)
                for (int d = lane; d < P.each; d += q) {
                    const int l = g * P.each + d, c = at.channel0 + l;
                    const float scale = P.scale && AXC_GLOBAL_OK(c, P.channels, 509u) ? load_as_float(P.scale, c, P.scale_type) : 1.0f;
                    const float2 f = channels[l];
                    a = fmaf(scale, f.x, a);
                    b = fmaf(scale, f.y, b);
                }
            a = over_lanes(a, log2);
            b = over_lanes(b, log2);
            if (g < groups && lane == 0) mine[g] = make_float2(a, b);
        }
    }
    __syncwarp();
    if (P.blocks > 1) mma::cluster_sync();
    else __syncthreads();
    const float share = __fdiv_rn(1.0f, float(P.places) * float(P.each));
    for (int g = thread; g < groups; g += blockDim.x) {
        const float2 f = P.blocks > 1 ? sum_of_all(mine + g, P.blocks) : mine[g];
        const float r = stats(g).y;
        // the sums are of dz and of dz (x - mean): r makes xhat of that
        result[g] = make_float2(f.x * share * r, f.y * share * r * r * r);
    }
    // the sums of single channels, shared out among the cluster's blocks; those of a single sample are the parameters' gradients
    if (P.sums || P.single) {
        for (int l = at.rank + thread * P.blocks; l < P.span.channels; l += int(blockDim.x) * P.blocks) {
            const float2 f = P.blocks > 1 ? sum_of_all(channels + l, P.blocks) : channels[l];
            const long long to = at.sample * P.channels + at.channel0 + l;
            if (!AXC_GLOBAL_OK(to, P.samples * P.channels, 510u)) continue;
            const float by_scale = f.y * stats(int(P.by_group.of(unsigned(l)))).y;
            if (P.sums) P.sums[to] = make_float2(f.x, by_scale);
            else {
                if (P.doffset) store_from_float(P.doffset, to, P.offset_type, f.x);
                if (P.dscale) store_from_float(P.dscale, to, P.scale_type, by_scale);
            }
        }
    }
    __syncthreads();
    if (P.blocks > 1) cluster_arrive();
    if (P.dx) {
        T *dx = static_cast<T *>(P.dx);
        Gradient<V> gradient;
        gradient.fill(group, P.whole_vectors, [&](int g) { return result[g]; });
        batches<V>(w, std::integral_constant<int, 2>(), [&](auto whole, auto n, int j) {
            constexpr int N = decltype(n)::value;
            const long long from = at.sample0 + w.at + j * w.step;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                Pack<T, V> v, vd;
                v.w = kept[(j + k) * stride];
                vd.w = kept_dz[(j + k) * stride];
                Two d[kPairs<V>], off[kPairs<V>];
                if constexpr (AGAIN) slope_at<T, V>(P, ch, v, vd, vd, d, off);
                else {
                    if constexpr (sizeof(T) == 4) widen_pairs<T, V>(vd, d);
                    else if (with) join_pairs<V>(vd.w, kept_residual[(j + k) * stride], d);
                    else widen_pairs<T, V>(vd, d);
                    widen_pairs<T, V>(v, off);
#pragma unroll
                    for (int i = 0; i < kPairs<V>; ++i) off[i] = add2(off[i], ch.less[i]);
                }
                gradient.of(ch, off, d);
                store<decltype(whole)::value>(dx + from + k * w.step, w, j + k, d, dx, values);
            }
        });
    }
    __syncwarp();
    if (P.blocks > 1) cluster_wait();
}

// ---- tensors that are read twice -------------------------------------------------------------------------------------------------
// Block -> sample, share of the places, columns
struct Share {
    long long sample, place0;
    int share, channel0, places;
    bool last;                                 // of a line's spans
    __device__ __forceinline__ Share(const NormArgs &P, unsigned block)
    {
        unsigned rest = P.spans > 1 ? block / unsigned(P.spans) : block;
        const int span = int(block - rest * unsigned(P.spans));
        const unsigned n = rest / unsigned(P.shares);
        sample = n;
        share = int(rest - n * unsigned(P.shares));
        channel0 = span * P.span.channels;
        last = span + 1 == P.spans;
        place0 = share * P.per;
        places = int(min(P.per, P.places - place0));
    }
    __device__ __forceinline__ const Span &span(const NormArgs &P) const { return last ? P.last : P.span; }
};

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 3) norm_moments_kernel(const NormArgs P)
{
    after_previous();
    __shared__ float2 entries[2 * kNormThreads * V];
    const Share at(P, blockIdx.x);
    const Span &span = at.span(P);
    const int shift = shift_of<T, V>(P, at.sample, at.place0);
    const Walk<V> w(threadIdx.x, span, shift, at.places, P.channels, at.place0, at.channel0);
    const T *x = static_cast<const T *>(P.x);
    Moments<V> mo;
    const T *sample = x + at.sample * P.places * P.channels;
    take_moments<V == 1 ? 8 : 4, T, V>(w, mo, [&](int j, Pack<T, V> &v, auto whole) { load<decltype(whole)::value>(sample + w.at + j * w.step, w, j, v, x, P.values()); });
    if (int(threadIdx.x) < span.active) give_entries<V>(entries, span, [&](int i) { return mo.of(i); });
    __syncthreads();
    const Entries E(span, shift, w.total);
    const long long to = (at.sample * P.shares + at.share) * P.channels + at.channel0;
    join_moments(entries, E, span.by_copies, span.channels, 1, float(at.places), 1.0f, [&](int l, float mean, float square) {
        if (AXC_GLOBAL_OK(to + l, P.samples * P.shares * P.channels, 511u)) P.part[to + l] = make_float2(mean, square);
    });
}

__device__ __forceinline__ float over_block(float x, float *room)
{
    x = over_lanes(x, 5);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = x;
    __syncthreads();
    float sum = 0.0f;
    for (int i = 0; i < int(blockDim.x) / 32; ++i) sum += room[i];
    return sum;
}

// f(channel of the group, share) for all that are a thread's: neighbouring lanes have neighbouring channels, as many as a warp holds, the other lanes and the
// warps other shares
template <typename Each>
__device__ __forceinline__ void over_shares(const NormArgs &P, Each f)
{
    const int log2 = P.each >= 32 ? 5 : 32 - __clz(max(P.each, 2) - 1), width = 1 << log2, lane = threadIdx.x & 31;
    const long long first = (long long)(threadIdx.x >> 5) * (32 >> log2) + (lane >> log2), step = (kNormThreads / 32) * (32 >> log2);
    for (int d = lane & (width - 1); d < P.each; d += width)
#pragma unroll 8
        for (long long s = first; s < P.shares; s += step) f(d, s);
}

// A block joins the shares of one sample's group
__global__ void __launch_bounds__(kNormThreads) norm_join_kernel(const NormArgs P)
{
    after_previous();
    __shared__ float room[kNormThreads / 32];
    const unsigned sample = blockIdx.x / unsigned(P.groups);
    const int group = int(blockIdx.x - sample * unsigned(P.groups));
    const float2 *part = P.part + sample * P.shares * P.channels + (long long)group * P.each;
    const float all = float(P.places) * float(P.each);
    const float of_share = float(P.per), of_last = float(P.places - P.per * (P.shares - 1));
    [[maybe_unused]] const long long room_for = P.shares * P.channels - (long long)group * P.each;
    float sum = 0.0f, square = 0.0f;
    over_shares(P, [&](int d, long long s) {
        if (AXC_GLOBAL_OK(s * P.channels + d, room_for, 512u)) sum = fmaf(s + 1 < P.shares ? of_share : of_last, part[s * P.channels + d].x, sum);
    });
    const float mean = __fdiv_rn(over_block(sum, room), all);
    over_shares(P, [&](int d, long long s) {
        if (!AXC_GLOBAL_OK(s * P.channels + d, room_for, 513u)) return;
        const float2 f = part[s * P.channels + d];
        square += fmaf((s + 1 < P.shares ? of_share : of_last) * (f.x - mean), f.x - mean, f.y);
    });
    square = over_block(square, room);
    if (threadIdx.x == 0) P.statistics[blockIdx.x] = make_float2(mean, __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(square, all) + P.epsilon)));
}

// body(whole, one, j, vectors of the tensors) for all vectors of a thread, from tensors at p[0] .. p[n - 1] (from the sample's start).  Where there
// is an asynchronous copy of that size, the next D - 1 of them are on their way: a thread has D places in `ring` for each tensor, which it alone uses.
// Else one after the other.
constexpr int ring_bytes(int depth, int tensors) { return depth * tensors * kNormThreads * 16; }
template <int D, int NT, typename T, int V, typename Body>
__device__ __forceinline__ void stream(const Walk<V> &w, const T *const (&p)[NT], int n, char *ring, [[maybe_unused]] const T *const (&base)[NT], [[maybe_unused]] long long count,
                                       Body body)
{
    if constexpr (V * sizeof(T) == 16) {
        const unsigned place = mma::smem_address(ring) + threadIdx.x * 16u;
        auto at = [&](int slot, int t) { return unsigned((slot * NT + t) * kNormThreads * 16); };
        long long ahead = w.at + w.first * w.step;
        int slot_in = 0, slot = 0;
        auto issue = [&](int j) {
            if (j < w.end) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    if (t < n && AXC_VALUES_OK(p[t] + ahead, V, base[t], count, 520u))
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(place + at(slot_in, t)), "l"(p[t] + ahead) : "memory");
                ahead += w.step;
                if (++slot_in == D) slot_in = 0;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int d = 0; d < D - 1; ++d) issue(w.first + d);
        for (int j = w.first; j < w.end; ++j) {
            issue(j + D - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
            Pack<T, V> v[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (t < n) v[t].w = *reinterpret_cast<const uint4 *>(ring + threadIdx.x * 16u + at(slot, t));
            if (++slot == D) slot = 0;
            body(std::true_type(), j, v);
        }
        wait_copies();
    } else {
        for (int j = w.first; j < w.end; ++j) {
            Pack<T, V> v[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (t < n) load<true>(p[t] + w.at + j * w.step, w, j, v[t], base[t], count);
            body(std::true_type(), j, v);
        }
    }
    if constexpr (V > 1) {
        for (int side = 0; side < 2; ++side) {
            if (side == 0 ? w.first == 0 : w.end == w.count) continue;
            const int j = side == 0 ? 0 : w.end;
            Pack<T, V> v[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (t < n) load<false>(p[t] + w.at + j * w.step, w, j, v[t], base[t], count);
            body(std::false_type(), j, v);
        }
    }
}

template <int V>
__device__ __forceinline__ void fill_channels(const NormArgs &P, const Share &at, const Walk<V> &w, Channels<V> &ch, int (&group)[V])
{
    // (a span that starts inside a group counts its channels from there)
    int local[V];
    local_channels<V>(w, at.span(P), at.span(P).by_channels, local, group);
#pragma unroll
    for (int i = 0; i < V; ++i) group[i] = (at.channel0 + local[i]) / P.each;
    const float2 *statistics = P.statistics + at.sample * P.groups;
    ch.fill(P, at.channel0, local, group, false, [&](int g) { return AXC_GLOBAL_OK(g, P.groups, 514u) ? statistics[g] : make_float2(0.0f, 0.0f); });
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 3) norm_apply_kernel(const NormArgs P)
{
    after_previous();
    extern __shared__ __align__(16) char ring[];
    const Share at(P, gridDim.x - 1 - blockIdx.x);
    const Span &span = at.span(P);
    const Walk<V> w(threadIdx.x, span, shift_of<T, V>(P, at.sample, at.place0), at.places, P.channels, at.place0, at.channel0);
    if (w.count == 0) return;
    Channels<V> ch;
    int group[V];
    fill_channels<V>(P, at, w, ch, group);
    const long long sample0 = at.sample * P.places * P.channels;
    const T *x = static_cast<const T *>(P.x), *residual = static_cast<const T *>(P.residual);
    T *y = static_cast<T *>(P.y);
    const T *const base[2] = {x, residual}, *const p[2] = {x + sample0, P.residual ? residual + sample0 : nullptr};
    stream<6>(w, p, P.residual ? 2 : 1, ring, base, P.values(), [&](auto whole, int j, const Pack<T, V> (&v)[2]) {
        Two z[kPairs<V>];
        output_of<T, V>(P, ch, v[0], v[1], z);
        store<decltype(whole)::value>(y + sample0 + w.at + j * w.step, w, j, z, y, P.values());
    });
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 2) norm_sums_kernel(const NormArgs P)
{
    after_previous();
    extern __shared__ __align__(16) char ring[];
    float2 *entries = reinterpret_cast<float2 *>(ring);        // once all has come through
    const Share at(P, blockIdx.x);
    const Span &span = at.span(P);
    const int shift = shift_of<T, V>(P, at.sample, at.place0);
    const Walk<V> w(threadIdx.x, span, shift, at.places, P.channels, at.place0, at.channel0);
    Sums<V> sums, run;
    if (w.count > 0) {
        Channels<V> ch;
        int group[V];
        fill_channels<V>(P, at, w, ch, group);
        const long long sample0 = at.sample * P.places * P.channels, values = P.values();
        const T *x = static_cast<const T *>(P.x), *dy = static_cast<const T *>(P.dy), *residual = static_cast<const T *>(P.residual);
        T *dresidual = static_cast<T *>(P.dresidual);
        const bool with = P.residual && P.activation != kActNone;
        const T *const base[3] = {x, dy, residual}, *const p[3] = {x + sample0, dy + sample0, with ? residual + sample0 : nullptr};
        stream<4>(w, p, with ? 3 : 2, ring, base, values, [&](auto whole, int j, const Pack<T, V> (&v)[3]) {
            Two dz[kPairs<V>], off[kPairs<V>];
            slope_at<T, V>(P, ch, v[0], v[1], v[2], dz, off);
            run.template add<decltype(whole)::value>(w, j, dz, off);
            if (dresidual) store<decltype(whole)::value>(dresidual + sample0 + w.at + j * w.step, w, j, dz, dresidual, values);
            if (((j - w.first) & (kRun - 1)) == kRun - 1) sums.take(run);
        });
        sums.take(run);
    }
    __syncthreads();
    if (int(threadIdx.x) < span.active) give_entries<V>(entries, span, [&](int i) { return sums.of(i); });
    __syncthreads();
    const Entries E(span, shift, w.total);
    const long long to = (at.sample * P.shares + at.share) * P.channels + at.channel0;
    join_sums(entries, E, [&](int l, float a, float b) {
        if (AXC_GLOBAL_OK(to + l, P.samples * P.shares * P.channels, 515u)) P.part[to + l] = make_float2(a, b);
    });
}

// A block joins the shares of one sample's group, for up to 32 channels at a time
__global__ void __launch_bounds__(kNormThreads) norm_join_sums_kernel(const NormArgs P)
{
    after_previous();
    __shared__ float2 room[kNormThreads / 32][32];
    __shared__ float sums[kNormThreads / 32];
    const unsigned sample = blockIdx.x / unsigned(P.groups);
    const int group = int(blockIdx.x - sample * unsigned(P.groups)), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float r = P.statistics[blockIdx.x].y;
    const int log2 = P.each >= 32 ? 5 : 32 - __clz(max(P.each, 2) - 1), width = 1 << log2;
    float first = 0.0f, second = 0.0f;
    for (int d0 = 0; d0 < P.each; d0 += width) {
        const int d = d0 + (lane & (width - 1));
        const long long c = (long long)group * P.each + d;
        float2 f = make_float2(0.0f, 0.0f);
        if (d < P.each) {
            const long long step = (kNormThreads / 32) * (32 >> log2);
#pragma unroll 8
            for (long long s = (long long)warp * (32 >> log2) + (lane >> log2); s < P.shares; s += step) {
                const long long from = (sample * P.shares + s) * P.channels + c;
                if (!AXC_GLOBAL_OK(from, P.samples * P.shares * P.channels, 516u)) continue;
                const float2 more = P.part[from];
                f.x += more.x;
                f.y += more.y;
            }
        }
        for (int o = 16; o >= width; o >>= 1) {
            f.x += __shfl_xor_sync(0xffffffffu, f.x, o);
            f.y += __shfl_xor_sync(0xffffffffu, f.y, o);
        }
        __syncthreads();
        room[warp][lane] = f;
        __syncthreads();
        if (warp == 0 && lane < width && d < P.each) {
            for (int i = 1; i < kNormThreads / 32; ++i) {
                f.x += room[i][lane].x;
                f.y += room[i][lane].y;
            }
            f.y *= r;
            if (P.sums) P.sums[sample * P.channels + c] = f;
            const float scale = P.scale ? load_as_float(P.scale, c, P.scale_type) : 1.0f;
            first = fmaf(scale, f.x, first);
            second = fmaf(scale, f.y, second);
        }
    }
    const float all = float(P.places) * float(P.each);
    first = over_block(first, sums);
    second = over_block(second, sums);
    if (threadIdx.x == 0) P.group_sums[blockIdx.x] = make_float2(__fdiv_rn(first, all) * r, __fdiv_rn(second, all) * r * r);
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads, 2) norm_gradient_kernel(const NormArgs P)
{
    after_previous();
    extern __shared__ __align__(16) char ring[];
    const Share at(P, gridDim.x - 1 - blockIdx.x);
    const Span &span = at.span(P);
    const Walk<V> w(threadIdx.x, span, shift_of<T, V>(P, at.sample, at.place0), at.places, P.channels, at.place0, at.channel0);
    if (w.count == 0) return;
    Channels<V> ch;
    int group[V];
    fill_channels<V>(P, at, w, ch, group);
    Gradient<V> gradient;
    gradient.fill(group, false, [&](int g) { return AXC_GLOBAL_OK(g, P.groups, 517u) ? P.group_sums[at.sample * P.groups + g] : make_float2(0.0f, 0.0f); });
    const long long sample0 = at.sample * P.places * P.channels, values = P.values();
    const T *x = static_cast<const T *>(P.x), *dy = static_cast<const T *>(P.dy), *residual = static_cast<const T *>(P.residual);
    T *dx = static_cast<T *>(P.dx);
    const bool with = P.residual && P.activation != kActNone;
    const T *const base[3] = {x, dy, residual}, *const p[3] = {x + sample0, dy + sample0, with ? residual + sample0 : nullptr};
    stream<4>(w, p, with ? 3 : 2, ring, base, values, [&](auto whole, int j, const Pack<T, V> (&v)[3]) {
        Two dz[kPairs<V>], off[kPairs<V>];
        slope_at<T, V>(P, ch, v[0], v[1], v[2], dz, off);
        gradient.of(ch, off, dz);
        store<decltype(whole)::value>(dx + sample0 + w.at + j * w.step, w, j, dz, dx, values);
    });
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
template <typename T, int V>
int forward(NormArgs P, const NormPlan &plan, Queue &q)
{
    if (plan.resident) {
        static std::atomic<unsigned long long> ready{0};
        const int rc = allow_smem(norm_forward_kernel<T, V>, kNormSmem, ready);
        if (rc) return rc;
        return launch(q, norm_forward_kernel<T, V>, dim3(unsigned(P.samples * P.spans * P.blocks)), unsigned(plan.threads), plan.smem, unsigned(plan.blocks), P);
    }
    const dim3 grid(unsigned(P.samples * P.shares * P.spans));
    int rc = launch(q, norm_moments_kernel<T, V>, grid, kNormThreads, 0, 1, P);
    if (!rc) rc = launch(q, norm_join_kernel, dim3(unsigned(P.samples * P.groups)), kNormThreads, 0, 1, P);
    if (!rc) rc = launch(q, norm_apply_kernel<T, V>, grid, kNormThreads, ring_bytes(6, 2), 1, P);
    return rc;
}

template <typename T, int V>
int backward(NormArgs P, const NormPlan &plan, Queue &q)
{
    int rc;
    if (plan.resident) {
        auto run = [&](auto kernel, std::atomic<unsigned long long> &ready) {
            const int rc = allow_smem(kernel, kNormSmem, ready);
            return rc ? rc : launch(q, kernel, dim3(unsigned(P.samples * P.spans * P.blocks)), unsigned(plan.threads), plan.smem, unsigned(plan.blocks), P);
        };
        static std::atomic<unsigned long long> ready[2];
        if (sizeof(T) == 2 && P.activation != kActNone && !P.residual) rc = run(norm_backward_kernel<T, V, sizeof(T) == 2>, ready[1]);
        else rc = run(norm_backward_kernel<T, V, false>, ready[0]);
    } else {
        const dim3 grid(unsigned(P.samples * P.shares * P.spans));
        static_assert(ring_bytes(4, 3) >= int(sizeof(float2)) * 2 * kNormThreads * V, "the entries fit where the tensors came through");
        rc = launch(q, norm_sums_kernel<T, V>, grid, kNormThreads, ring_bytes(4, 3), 1, P);
        if (!rc) rc = launch(q, norm_join_sums_kernel, dim3(unsigned(P.samples * P.groups)), kNormThreads, 0, 1, P);
        if (!rc && P.dx) rc = launch(q, norm_gradient_kernel<T, V>, grid, kNormThreads, ring_bytes(4, 3), 1, P);
    }
    return rc;
}

constexpr long long kMostBlocks = 0x7fffffffll;

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

// The plan of a call; `residual`: whether its values take part.  Searching for one takes 1 to 8 us of the host's time, so plans are remembered: they are functions of the shape alone.
// (Shapes whose hashes collide, and every new thread, search again.)
NormPlan plan_of(const NormShape &s, bool backward, bool residual, int sms)
{
    struct Known {
        NormShape shape;
        int key;
        NormPlan plan;
    };
    constexpr unsigned kKnown = 256;
    thread_local Known known[kKnown];          // zeros at first: no call has the key 0
    const int key = 1 + (backward ? 1 : 0) + (residual ? 2 : 0) + (s.aligned ? 4 : 0) + 8 * sms;
    unsigned long long hash = (unsigned long long)s.samples;
    for (const long long v : {s.places, s.channels, s.groups, (long long)(key * 8 + s.size)}) hash = (hash ^ (unsigned long long)v) * 0x9E3779B97F4A7C15ull, hash ^= hash >> 29;
    Known &k = known[hash % kKnown];
    if (k.key != key || k.shape.samples != s.samples || k.shape.places != s.places || k.shape.channels != s.channels || k.shape.groups != s.groups || k.shape.size != s.size)
        k = {s, key, backward ? norm_plan(s, (residual ? 3 : 2) * s.size, s.size * (residual ? 5 : 3), true, sms)
                              : norm_plan(s, s.size, s.size * (residual ? 3 : 2), false, sms)};
    return k.plan;
}

NormArgs args_of(const axc_norm_desc &d, const NormPlan &plan, bool backward)
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
    P.by_group = divider(unsigned(P.each));
    P.spans = int((d.channels + plan.span - 1) / plan.span);
    P.span = span_of(plan.span, norm_active(plan.threads, plan.span, plan.vec), plan.vec);
    const int rest = int(d.channels - (long long)(P.spans - 1) * plan.span);
    P.last = span_of(rest, norm_active(plan.threads, rest, plan.vec), plan.vec);
    P.blocks = plan.blocks;
    const long long parts = plan.resident ? plan.blocks : plan.shares;
    P.per = (d.places + parts - 1) / parts;
    if (plan.resident) {
        P.steps = int(norm_steps(P.per, plan.span, plan.vec, P.span.active));
        P.span_groups = plan.span / P.each;
        P.whole_vectors = plan.vec > 1 && P.each % plan.vec == 0;
        P.entries = int(norm_entries(plan.span, plan.vec, plan.threads, P.span.active, P.each, backward));
        P.lanes = norm_lanes(plan.span, plan.vec, plan.threads);
        if (P.whole_vectors) P.vectors = span_of(plan.span / plan.vec, P.span.active, 1);
    }
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
    NormArgs P = args_of(d, plan, false);
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
    const NormPlan plan = plan_of(s, true, residual && d.activation != kActNone, sms);
    NormArgs P = args_of(d, plan, true);
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
    P.single = plan.resident && d.samples == 1 && (dscale || doffset);
    P.sums = (dscale || doffset) && !P.single ? reinterpret_cast<float2 *>(ws + norm_part_bytes(s, plan)) : nullptr;
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
        if (!rc && (dscale || doffset) && !(some && P.single)) rc = launch(q, norm_parameters_kernel, dim3(unsigned((P.channels + 31) / 32)), 1024, 0, 1, P);
        return rc;
    });
}
