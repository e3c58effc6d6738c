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
// The square root and the quotient are the 2^-22 approximations: their error is below a hundredth of an ulp of a fp32 parameter for
// steps up to a hundredth of its size, and the exact ones would make the 8-bit kernel bound by arithmetic.
//
// Bound by memory: 28 bytes per fp32 value with fp32 moments, 16.03 with 8-bit ones, 10.03 for a 16-bit value with those.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

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
    int count, per_cta;                        // tensors; blocks per CTA
    unsigned base, blocks;                     // blocks of this launch: [base, base + blocks)
    float c1, c2, inv_root, eps, grad_scale;   // 1 - beta1, 1 - beta2, 1 / sqrt(1 - beta2^t)
    void *m, *v;
    float *m_scale, *v_scale;
    AdamwEntry entry[CAP];
};
constexpr int kSmallTable = 96, kLargeTable = 800;

__device__ __forceinline__ float approx_sqrt(float x)
{
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
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

// V values at `at`, as one load or store where `vec`, else those below `left`
template <typename T, int V>
__device__ __forceinline__ void load_values(const T *at, bool vec, long long left, float (&x)[V])
{
    typedef typename Word<V * sizeof(T)>::type word;
    if (vec) {
        union { word w; T t[V]; } u;
        u.w = __ldcs(reinterpret_cast<const word *>(at));
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = to_float(u.t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = i < left ? to_float(at[i]) : 0.0f;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_values(T *at, bool vec, long long left, const float (&x)[V])
{
    typedef typename Word<V * sizeof(T)>::type word;
    if (vec) {
        union { word w; T t[V]; } u;
#pragma unroll
        for (int i = 0; i < V; ++i) u.t[i] = from_float<T>(x[i]);
        __stcs(reinterpret_cast<word *>(at), u.w);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < left) at[i] = from_float<T>(x[i]);
    }
}
template <int V>
__device__ __forceinline__ void load_codes(const uint8_t *at, float scale, float (&x)[V])
{
    union { typename Word<V>::type w; __nv_fp8x2_storage_t c[V / 2]; } u;
    u.w = __ldcs(reinterpret_cast<const typename Word<V>::type *>(at));
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(u.c[i], __NV_E4M3)));
        x[2 * i] = f.x * scale;
        x[2 * i + 1] = f.y * scale;
    }
}
template <int V>
__device__ __forceinline__ void store_codes(uint8_t *at, const float (&x)[V])
{
    union { typename Word<V>::type w; __nv_fp8x2_storage_t c[V / 2]; } u;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) u.c[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i], x[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    __stcs(reinterpret_cast<typename Word<V>::type *>(at), u.w);
}
__device__ __forceinline__ float warp_max(float x)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// A warp takes 256 values at a time: 16-bit parameters with 8-bit moments 8 neighbours per lane (16-byte and 8-byte accesses), all
// else 4 neighbours twice.
template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(kWarps * 32) adamw_kernel(const __grid_constant__ AdamwTable<CAP> tab)
{
    constexpr int V = sizeof(T) == 2 && BITS == 8 ? 8 : 4, N = kBlock / 32 / V;
    const int lane = threadIdx.x & 31;
    unsigned b = tab.base + blockIdx.x * unsigned(tab.per_cta) + (threadIdx.x >> 5);
    const unsigned end = min(tab.base + blockIdx.x * unsigned(tab.per_cta) + unsigned(tab.per_cta), tab.base + tab.blocks);
    int lo = 0, hi = tab.count;                 // the last tensor that starts at b or before
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.entry[mid].first <= b) lo = mid;
        else hi = mid;
    }
    for (; b < end; b += kWarps) {
        while (lo + 1 < tab.count && tab.entry[lo + 1].first <= b) ++lo;
        const AdamwEntry &e = tab.entry[lo];
        const long long at = (long long)(b - e.first) * kBlock, left = e.count - at;
        if (left <= 0) continue;               // blocks of a tensor without a gradient
        T *param = static_cast<T *>(e.param) + at;
        const T *grad = static_cast<const T *>(e.grad) + at;
        const bool vec = left >= kBlock && ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad)) & (V * sizeof(T) - 1)) == 0;
        const size_t state = size_t(b) * kBlock;
        float p[N][V], g[N][V], m[N][V], v[N][V];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = (n * 32 + lane) * V;
            load_values<T, V>(grad + i, vec, left - i, g[n]);
            load_values<T, V>(param + i, vec, left - i, p[n]);
            if constexpr (BITS == 32) {
                load_values<float, V>(static_cast<const float *>(tab.m) + state + i, true, 0, m[n]);
                load_values<float, V>(static_cast<const float *>(tab.v) + state + i, true, 0, v[n]);
            } else {
                load_codes<V>(static_cast<const uint8_t *>(tab.m) + state + i, tab.m_scale[b], m[n]);
                load_codes<V>(static_cast<const uint8_t *>(tab.v) + state + i, tab.v_scale[b], v[n]);
            }
        }
        float m_top = 0.0f, r_top = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float gi = g[n][i] * tab.grad_scale;
                const float old = BITS == 32 ? v[n][i] : v[n][i] * v[n][i];
                m[n][i] = fmaf(tab.c1, gi - m[n][i], m[n][i]);
                const float second = fmaf(tab.c2, fmaf(gi, gi, -old), old);
                const float root = approx_sqrt(second);
                p[n][i] = p[n][i] * e.decay - e.step_size * __fdividef(m[n][i], fmaf(root, tab.inv_root, tab.eps));
                v[n][i] = BITS == 32 ? second : root;
                m_top = fmaxf(m_top, fabsf(m[n][i]));
                r_top = fmaxf(r_top, root);
            }
            const int i = (n * 32 + lane) * V;
            store_values<T, V>(param + i, vec, left - i, p[n]);
        }
        if constexpr (BITS == 8) {
            // a scale below the smallest normal number has no reciprocal: the block's moments are then zeros
            float ms = warp_max(m_top) * (1.0f / 448.0f), rs = warp_max(r_top) * (1.0f / 448.0f);
            if (ms < 1.17549435e-38f) ms = 0.0f;
            if (rs < 1.17549435e-38f) rs = 0.0f;
            const float mi = ms > 0.0f ? __fdividef(1.0f, ms) : 0.0f, ri = rs > 0.0f ? __fdividef(1.0f, rs) : 0.0f;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    m[n][i] *= mi;
                    const float r = v[n][i] * ri;
                    v[n][i] = r > 0.0f ? fmaxf(r, 0.001953125f) : r;
                }
            if (lane == 0) {
                tab.m_scale[b] = ms;
                tab.v_scale[b] = rs;
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const size_t i = state + (n * 32 + lane) * V;
            if constexpr (BITS == 32) {
                store_values<float, V>(static_cast<float *>(tab.m) + i, true, 0, m[n]);
                store_values<float, V>(static_cast<float *>(tab.v) + i, true, 0, v[n]);
            } else {
                store_codes<V>(static_cast<uint8_t *>(tab.m) + i, m[n]);
                store_codes<V>(static_cast<uint8_t *>(tab.v) + i, v[n]);
            }
        }
    }
}

template <typename T, int BITS, int CAP>
void launch_adamw(AdamwTable<CAP> &tab, const DeviceInfo &di, cudaStream_t stream)
{
    // four blocks per warp where that leaves every SM several CTAs, else one
    tab.per_cta = tab.blocks >= unsigned(di.sm_count) * kWarps * 4 * 8 ? kWarps * 4 : kWarps;
    const unsigned grid = (tab.blocks + unsigned(tab.per_cta) - 1) / unsigned(tab.per_cta);
    adamw_kernel<T, BITS, CAP><<<grid, kWarps * 32, 0, stream>>>(tab);
    count_launch();
}

template <int CAP>
void launch_adamw(AdamwTable<CAP> &tab, int type, int bits, const DeviceInfo &di, cudaStream_t stream)
{
    if (type == AXC_TYPE_FLOAT32) bits == 32 ? launch_adamw<float, 32>(tab, di, stream) : launch_adamw<float, 8>(tab, di, stream);
    else if (type == AXC_TYPE_BFLOAT16) bits == 32 ? launch_adamw<__nv_bfloat16, 32>(tab, di, stream) : launch_adamw<__nv_bfloat16, 8>(tab, di, stream);
    else bits == 32 ? launch_adamw<__half, 32>(tab, di, stream) : launch_adamw<__half, 8>(tab, di, stream);
}

// The tensors in as many launches as their tables need.
template <int CAP>
void run_adamw(const axc_adamw_desc &d, const axc_adamw_tensor *tensors, int32_t count, const DeviceInfo &di, cudaStream_t stream)
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
        if (tab.count > 0) launch_adamw<CAP>(tab, d.type, d.state_bits, di, stream);
    }
}

}  // namespace
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
    if (count <= kSmallTable) run_adamw<kSmallTable>(d, tensors, count, di, cudaStream_t(stream));
    else run_adamw<kLargeTable>(d, tensors, count, di, cudaStream_t(stream));
    const cudaError_t e = cudaGetLastError();
    if (prev != device) cudaSetDevice(prev);
    return e == cudaSuccess ? AXC_OK : cuda_failed(e);
}
