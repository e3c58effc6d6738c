// One step of AdamW (decoupled weight decay) over many tensors in one launch, with moments in fp32 or in 8 bits.
//
//   m = m + (1 - beta1) (g - m)          v = v + (1 - beta2) (g^2 - v)              g = grad_scale * gradient
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// all in fp32; a 16-bit parameter is rounded once, when it is written.  The moments of all tensors lie in one buffer, each
// tensor's at a multiple of 256 values.  In 8 bits a block of 256 values has e4m3 codes and one fp32 scale (the block's largest
// magnitude is code 448): m itself, and the ROOT of v.  The step divides by that root, so its relative error there is the code's
// (1/16 at most), and its range within a block, 2^17.8, is that of the first moment: held as v, the codes would reach gradients
// down to 1/470 of the block's largest only.  A root above zero keeps the smallest code, or a first moment that still has a code
// would be divided by eps.  The step itself uses the moments before they are rounded.
// The reciprocals and roots are the approximations to 2^-22: their error is below a hundredth of an ulp of a fp32 parameter for steps up
// to a hundredth of its size, and the exact ones would make the 8-bit kernel bound by arithmetic.
//
// Bound by memory: 28 bytes per fp32 value with fp32 moments, 16.06 with 8-bit ones (two scales of 256 values read and written), 10.06 for a 16-bit
// value with those.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <float.h>

#include <type_traits>

#include "axc_internal.h"

namespace axc {
namespace {

constexpr int kBlock = AXC_ADAMW_BLOCK;        // values that share a scale: a warp's work at a time, 8 per lane
constexpr int kWarps = 8;

struct AdamwEntry {
    void *param;
    const void *grad;
    long long count;
    unsigned first;                            // first block of 256 values
    float decay, step_size;                    // 1 - lr * weight decay; lr / (1 - beta1^t)
    unsigned pad;
};
static_assert(sizeof(AdamwEntry) == 40, "table entries are packed");

// Kernel parameters carry the table: no copy, no buffer that a later call could overwrite.  4 KiB of them cost nothing to launch;
// the large form holds what 32 KiB of parameters can.
template <int CAP>
struct AdamwTable {
    int count;                                 // tensors
    unsigned base, blocks;                     // blocks of this launch: [base, base + blocks)
    float c1, c2, inv_root, eps, grad_scale;   // 1 - beta1, 1 - beta2, 1 / sqrt(1 - beta2^t)
    void *m, *v;
    float *m_scale, *v_scale;
    AdamwEntry entry[CAP];
    unsigned state_blocks;                     // of the moments of all tensors
};
constexpr int kSmallTable = 96, kLargeTable = 800;

__device__ __forceinline__ float reciprocal(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// also of a value below the normal ones, and inf of inf: a gradient whose square leaves fp32's range still steps as the formula has it (2^29 bf16 values
// with 8-bit moments: 1235 us, 1195 with the root that takes values below the normal ones for 0)
__device__ __forceinline__ float square_root(float x)
{
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two fp32 values that one instruction computes with
struct Two {
    unsigned long long v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
    __device__ __forceinline__ float2 both() const
    {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ Two fma2(Two a, Two b, Two c)
{
    Two d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
__device__ __forceinline__ Two add2(Two a, Two b)
{
    Two d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b)
{
    Two d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

template <int BYTES> struct Word;
template <> struct Word<4> { typedef unsigned type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<16> { typedef uint4 type; };

// V values as they lie in memory
template <typename T, int V>
union Packed {
    typename Word<V * sizeof(T)>::type w;
    T t[V];
    __device__ Packed() {}
};
// (`left`: how many there are from `at` on)
template <typename T, int V>
__device__ __forceinline__ void load_values(const T *at, bool vec, long long left, Packed<T, V> &x)
{
    if (vec && AXC_GLOBAL_OK(V - 1, left, 481u)) x.w = __ldcs(reinterpret_cast<const typename Word<V * sizeof(T)>::type *>(at));
    else {
#pragma unroll
        for (int i = 0; i < V; ++i) x.t[i] = i < left ? at[i] : T(0);
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_values(T *at, bool vec, long long left, const float (&x)[V])
{
    Packed<T, V> u;
#pragma unroll
    for (int i = 0; i < V; ++i) u.t[i] = from_float<T>(x[i]);
    if (vec && AXC_GLOBAL_OK(V - 1, left, 482u)) __stcs(reinterpret_cast<typename Word<V * sizeof(T)>::type *>(at), u.w);
    else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < left) at[i] = u.t[i];
    }
}
// codes 2 i and 2 i + 1, times `scale`
template <int V>
__device__ __forceinline__ Two decode(const Packed<uint8_t, V> &codes, int i, Two scale)
{
    const __nv_fp8x2_storage_t two = __nv_fp8x2_storage_t(codes.t[2 * i] | codes.t[2 * i + 1] << 8);
    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
    return mul2(Two(f.x, f.y), scale);
}
template <int V>
__device__ __forceinline__ void store_codes(uint8_t *at, long long left, const float (&x)[V])
{
    if (!AXC_GLOBAL_OK(V - 1, left, 483u)) return;
    union { typename Word<V>::type w; __nv_fp8x2_storage_t c[V / 2]; } u;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) u.c[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i], x[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    __stcs(reinterpret_cast<typename Word<V>::type *>(at), u.w);
}
// At most 2 kNear where a quotient is within kNear units in the last place of the middle between two codes: e4m3 has 3 bits of fraction,
// the middle has the next one and no more.  (Below the normal codes, 3.5e-5 of the block's largest value, the middles are others: there a
// quotient that close to one, 1 in a million, may get the other code.)
constexpr unsigned kNear = 8;
__device__ __forceinline__ unsigned edge(float q) { return (__float_as_uint(q) + (kNear - 0x80000u)) & 0xfffffu; }

__device__ __forceinline__ float warp_max(float x)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// What a lane has of a block of 256 values: V neighbours, N times
template <typename T, int BITS>
struct Part {
    // 16-bit parameters with 8-bit moments: 8 neighbours (16-byte and 8-byte accesses), all else 4 neighbours twice
    static constexpr int V = sizeof(T) == 2 && BITS == 8 ? 8 : 4, N = kBlock / 32 / V;
    typedef typename std::conditional<BITS == 32, float, uint8_t>::type State;
    Packed<T, V> p[N], g[N];
    Packed<State, V> m[N], v[N];
    float m_scale = 0.0f, v_scale = 0.0f, decay, step_size;
    T *param;
    const T *grad;
    long long left;                            // values of the tensor from the block's first on; 0: a tensor without a gradient
    bool vec;

    // values of the moments from block b on
    template <int CAP>
    static __device__ __forceinline__ long long in_state(const AdamwTable<CAP> &tab, unsigned b) { return ((long long)tab.state_blocks - b) * kBlock; }

    template <int CAP>
    __device__ __forceinline__ void load(const AdamwTable<CAP> &tab, int at, unsigned b, int lane)
    {
        const AdamwEntry &e = tab.entry[at];
        const long long first = (long long)(b - e.first) * kBlock;
        left = AXC_GLOBAL_OK(at, tab.count, 486u) ? e.count - first : 0;
        param = static_cast<T *>(e.param) + first;
        grad = static_cast<const T *>(e.grad) + first;
        decay = e.decay;
        step_size = e.step_size;
        vec = left >= kBlock && ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad)) & (V * sizeof(T) - 1)) == 0;
        if (left <= 0) return;
        const State *ms = static_cast<const State *>(tab.m) + size_t(b) * kBlock, *vs = static_cast<const State *>(tab.v) + size_t(b) * kBlock;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = (n * 32 + lane) * V;
            load_values<T, V>(grad + i, vec, left - i, g[n]);
            load_values<T, V>(param + i, vec, left - i, p[n]);
            load_values<State, V>(ms + i, true, in_state(tab, b) - i, m[n]);
            load_values<State, V>(vs + i, true, in_state(tab, b) - i, v[n]);
        }
        if constexpr (BITS == 8) {
            if (AXC_GLOBAL_OK(b, tab.state_blocks, 485u)) {
                m_scale = tab.m_scale[b];
                v_scale = tab.v_scale[b];
            }
        }
    }

    // The moments of values i and i + 1, each operation rounded by itself
    template <int CAP>
    __device__ __forceinline__ void moments(const AdamwTable<CAP> &tab, int n, int i, Two &m1, Two &v1) const
    {
        const Two minus(-1.0f), gi = mul2(Two(to_float(g[n].t[i]), to_float(g[n].t[i + 1])), Two(tab.grad_scale));
        Two m0, v0, v0_finite;
        if constexpr (BITS == 32) {
            m0 = Two(m[n].t[i], m[n].t[i + 1]);
            v0 = Two(v[n].t[i], v[n].t[i + 1]);
            v0_finite = Two(fminf(v[n].t[i], FLT_MAX), fminf(v[n].t[i + 1], FLT_MAX));          // what is infinite stays so
        } else {
            m0 = decode<V>(m[n], i / 2, Two(m_scale));
            v0 = decode<V>(v[n], i / 2, Two(v_scale));
            v0_finite = v0 = mul2(v0, v0);
        }
        m1 = add2(m0, mul2(Two(tab.c1), fma2(m0, minus, gi)));
        v1 = add2(v0, mul2(Two(tab.c2), fma2(v0_finite, minus, mul2(gi, gi))));
    }

    template <int CAP>
    __device__ __forceinline__ void step(const AdamwTable<CAP> &tab, unsigned b, int lane)
    {
        if (left <= 0) return;
        State *ms = static_cast<State *>(tab.m) + size_t(b) * kBlock, *vs = static_cast<State *>(tab.v) + size_t(b) * kBlock;
        float first[N][V], second[N][V], m_top = 0.0f, v_top = 0.0f;
        const Two inv_root(tab.inv_root), eps(tab.eps), keep(decay), move(-step_size);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float x[V];
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                Two m1, v1;
                moments(tab, n, i, m1, v1);
                const float2 vf = v1.both();
                const Two root(square_root(vf.x), square_root(vf.y));
                const float2 den = fma2(root, inv_root, eps).both();
                const Two p1 = fma2(mul2(m1, move), Two(reciprocal(den.x), reciprocal(den.y)), mul2(Two(to_float(p[n].t[i]), to_float(p[n].t[i + 1])), keep));
                const float2 xf = p1.both(), mf = m1.both(), rf = root.both();
                x[i] = xf.x;
                x[i + 1] = xf.y;
                first[n][i] = mf.x;
                first[n][i + 1] = mf.y;
                second[n][i] = BITS == 32 ? vf.x : rf.x;
                second[n][i + 1] = BITS == 32 ? vf.y : rf.y;
                if (BITS == 8) {
                    m_top = fmaxf(m_top, fmaxf(fabsf(mf.x), fabsf(mf.y)));
                    v_top = fmaxf(v_top, fmaxf(vf.x, vf.y));
                }
            }
            const int i = (n * 32 + lane) * V;
            store_values<T, V>(param + i, vec, left - i, x);
        }
        if constexpr (BITS == 32) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int i = (n * 32 + lane) * V;
                store_values<float, V>(ms + i, true, in_state(tab, b) - i, first[n]);
                store_values<float, V>(vs + i, true, in_state(tab, b) - i, second[n]);
            }
        } else {
            // a scale below the smallest normal number has no reciprocal: the block's moments are then zeros
            float m_new = warp_max(m_top) * (1.0f / 448.0f), r_new = __fsqrt_rn(warp_max(v_top)) * (1.0f / 448.0f);
            if (m_new < 1.17549435e-38f) m_new = 0.0f;
            if (r_new < 1.17549435e-38f) r_new = 0.0f;
            const float mi = m_new > 0.0f ? __fdividef(1.0f, m_new) : 0.0f, ri = r_new > 0.0f ? __fdividef(1.0f, r_new) : 0.0f;
            unsigned near_edge = 0xffffffffu;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const float2 f = mul2(Two(first[n][i], first[n][i + 1]), Two(mi)).both(), r = mul2(Two(second[n][i], second[n][i + 1]), Two(ri)).both();
                    near_edge = min(min(near_edge, edge(f.x)), min(edge(f.y), min(edge(r.x), edge(r.y))));
                    first[n][i] = f.x;
                    first[n][i + 1] = f.y;
                    second[n][i] = r.x > 0.0f ? fmaxf(r.x, 0.001953125f) : r.x;
                    second[n][i + 1] = r.y > 0.0f ? fmaxf(r.y, 0.001953125f) : r.y;
                }
            // The quotients are a few units in the last place off.  Where that could take one over the edge between two codes, the lane's are
            // computed again, rounded at every step: the codes are those of the formula to the bit, as its definition has them.
            // (What that takes is read again rather than kept in registers.)
            if (near_edge <= 2 * kNear) {
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int at = (n * 32 + lane) * V;
                    load_values<T, V>(grad + at, vec, left - at, g[n]);
                    load_values<State, V>(ms + at, true, in_state(tab, b) - at, m[n]);
                    load_values<State, V>(vs + at, true, in_state(tab, b) - at, v[n]);
                }
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        Two m1, v1;
                        moments(tab, n, i, m1, v1);
                        const float2 mf = m1.both(), vf = v1.both();
                        first[n][i] = m_new > 0.0f ? __fdiv_rn(mf.x, m_new) : 0.0f;
                        first[n][i + 1] = m_new > 0.0f ? __fdiv_rn(mf.y, m_new) : 0.0f;
                        const float rx = r_new > 0.0f ? __fdiv_rn(__fsqrt_rn(vf.x), r_new) : 0.0f, ry = r_new > 0.0f ? __fdiv_rn(__fsqrt_rn(vf.y), r_new) : 0.0f;
                        second[n][i] = rx > 0.0f ? fmaxf(rx, 0.001953125f) : rx;
                        second[n][i + 1] = ry > 0.0f ? fmaxf(ry, 0.001953125f) : ry;
                    }
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int i = (n * 32 + lane) * V;
                store_codes<V>(ms + i, in_state(tab, b) - i, first[n]);
                store_codes<V>(vs + i, in_state(tab, b) - i, second[n]);
            }
            if (lane == 0 && AXC_GLOBAL_OK(b, tab.state_blocks, 484u)) {
                tab.m_scale[b] = m_new;
                tab.v_scale[b] = r_new;
            }
        }
    }
};

// A warp takes one block of 256 values and a CTA eight.  Warps that walk over several blocks, with or without the next one's loads on
// their way, took up to twice as long (bf16 with 8-bit moments, 2^27 values: 276 us so, 339 to 541 us otherwise): new CTAs keep more
// loads in flight.  The registers are held to what lets 40 warps be there with 8-bit moments.
template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(kWarps * 32, BITS == 32 ? 1 : 5) adamw_kernel(const __grid_constant__ AdamwTable<CAP> tab)
{
    const unsigned b = tab.base + blockIdx.x * kWarps + (threadIdx.x >> 5), end = tab.base + tab.blocks;
    if (b >= end) return;
    int at = 0, hi = tab.count;                 // the last tensor that starts at b or before
    while (hi - at > 1) {
        const int mid = (at + hi) >> 1;
        if (tab.entry[mid].first <= b) at = mid;
        else hi = mid;
    }
    Part<T, BITS> part;
    part.load(tab, at, b, threadIdx.x & 31);
    part.step(tab, b, threadIdx.x & 31);
}

template <typename T, int BITS, int CAP>
void launch_adamw(const AdamwTable<CAP> &tab, cudaStream_t stream)
{
    const unsigned grid = (tab.blocks + kWarps - 1) / kWarps;
    adamw_kernel<T, BITS, CAP><<<grid, kWarps * 32, 0, stream>>>(tab);
    count_launch();
}

template <int CAP>
void launch_adamw(const AdamwTable<CAP> &tab, int type, int bits, cudaStream_t stream)
{
    if (type == AXC_TYPE_FLOAT32) bits == 32 ? launch_adamw<float, 32>(tab, stream) : launch_adamw<float, 8>(tab, stream);
    else if (type == AXC_TYPE_BFLOAT16) bits == 32 ? launch_adamw<__nv_bfloat16, 32>(tab, stream) : launch_adamw<__nv_bfloat16, 8>(tab, stream);
    else bits == 32 ? launch_adamw<__half, 32>(tab, stream) : launch_adamw<__half, 8>(tab, stream);
}

// The tensors in as many launches as their tables need.
template <int CAP>
void run_adamw(const axc_adamw_desc &d, const axc_adamw_tensor *tensors, int32_t count, int64_t blocks, cudaStream_t stream)
{
    const double root = sqrt(1.0 - pow(d.beta2, double(d.step))), first_left = 1.0 - pow(d.beta1, double(d.step));
    long long block = 0;
    AdamwTable<CAP> tab;
    for (int32_t at = 0; at < count;) {
        tab.c1 = float(1.0 - d.beta1);
        tab.c2 = float(1.0 - d.beta2);
        tab.inv_root = float(1.0 / root);
        tab.eps = float(d.eps);
        tab.grad_scale = d.grad_scale;
        tab.m = d.exp_avg;
        tab.v = d.exp_avg_sq;
        tab.m_scale = d.exp_avg_scale;
        tab.v_scale = d.exp_avg_sq_scale;
        tab.base = tab.blocks = 0;
        tab.state_blocks = unsigned(blocks);
        tab.count = 0;
        for (; at < count && tab.count < CAP; ++at) {
            const long long first = block;
            block += (tensors[at].count + kBlock - 1) / kBlock;
            if (tensors[at].count == 0 || !tensors[at].grad) continue;
            if (tab.count == 0) tab.base = unsigned(first);
            tab.blocks = unsigned(block) - tab.base;
            AdamwEntry &e = tab.entry[tab.count++];
            e.param = tensors[at].param;
            e.grad = tensors[at].grad;
            e.count = tensors[at].count;
            e.first = unsigned(first);
            e.decay = float(1.0 - tensors[at].lr * tensors[at].weight_decay);
            e.step_size = float(tensors[at].lr / first_left);
            e.pad = 0;
        }
        if (tab.count > 0) launch_adamw<CAP>(tab, d.type, d.state_bits, stream);
    }
}

}  // namespace

AXC_DEFINE_BOUNDS_READER(bounds_record_adamw)

}  // namespace axc

extern "C" int axc_adamw_state_blocks(const int64_t *counts, int32_t tensors, int64_t *blocks)
{
    if (!blocks || tensors < 0 || (tensors > 0 && !counts)) return AXC_INVALID_ARGUMENT;
    int64_t sum = 0;
    for (int32_t i = 0; i < tensors; ++i) {
        if (counts[i] < 0) return AXC_INVALID_ARGUMENT;
        sum += counts[i] / AXC_ADAMW_BLOCK + (counts[i] % AXC_ADAMW_BLOCK != 0);
    }
    if (sum > 0x7fffffffll) return AXC_INVALID_ARGUMENT;
    *blocks = sum;
    return AXC_OK;
}

extern "C" int axc_adamw_step(const axc_adamw_desc *desc, const axc_adamw_tensor *tensors, int32_t count, int device, void *stream)
{
    using namespace axc;
    if (!desc || count < 0 || (count > 0 && !tensors)) return AXC_INVALID_ARGUMENT;
    const axc_adamw_desc &d = *desc;
    if (d.type < AXC_TYPE_FLOAT32 || d.type > AXC_TYPE_FLOAT16 || (d.state_bits != 32 && d.state_bits != 8) || d.step < 1) return AXC_INVALID_ARGUMENT;
    if (!(d.beta1 >= 0.0 && d.beta1 < 1.0) || !(d.beta2 >= 0.0 && d.beta2 < 1.0) || !(d.eps >= 0.0)) return AXC_INVALID_ARGUMENT;
    const uintptr_t size = d.type == AXC_TYPE_FLOAT32 ? 4 : 2;
    int64_t blocks = 0;
    for (int32_t i = 0; i < count; ++i) {
        const axc_adamw_tensor &t = tensors[i];
        if (t.count < 0 || (t.count > 0 && !t.param)) return AXC_INVALID_ARGUMENT;
        if ((reinterpret_cast<uintptr_t>(t.param) | reinterpret_cast<uintptr_t>(t.grad)) % size) return AXC_INVALID_ARGUMENT;
        blocks += t.count / kBlock + (t.count % kBlock != 0);
    }
    if (blocks > 0x7fffffffll) return AXC_INVALID_ARGUMENT;
    if (blocks == 0) return AXC_OK;
    if (!d.exp_avg || !d.exp_avg_sq || ((reinterpret_cast<uintptr_t>(d.exp_avg) | reinterpret_cast<uintptr_t>(d.exp_avg_sq)) & 15u)) return AXC_INVALID_ARGUMENT;
    if (d.state_bits == 8 && (!d.exp_avg_scale || !d.exp_avg_sq_scale)) return AXC_INVALID_ARGUMENT;
    DeviceInfo di;
    int rc = device_info(device, &di);
    if (rc) return rc;
    int prev = 0;
    AXC_CUDA(cudaGetDevice(&prev));
    if (prev != device) AXC_CUDA(cudaSetDevice(device));
    if (count <= kSmallTable) run_adamw<kSmallTable>(d, tensors, count, blocks, cudaStream_t(stream));
    else run_adamw<kLargeTable>(d, tensors, count, blocks, cudaStream_t(stream));
    const cudaError_t e = cudaGetLastError();
    if (prev != device) cudaSetDevice(prev);
    return e == cudaSuccess ? AXC_OK : cuda_failed(e);
}
