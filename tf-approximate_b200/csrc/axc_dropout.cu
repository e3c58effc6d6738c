// Dropout whose mask is never stored: it is computed where it is needed, in the forward and in the backward pass, from a counter.
//
//   y[i] = (bits[i] >= share ? x[i] * factor : 0) + residual[i],  share = round(rate 2^16),  factor = 2^16 / (2^16 - share)
//
// bits[i]: 16 of the 128 that Philox 4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) makes of
// the counter {i / 8, offset} under the key `seed`.  Eight values share a counter: 20 wide multiplications and 20 three-way xors for eight values are
// less than the time that memory takes for them, with four values a counter (32 bits each) they would be as much.  16 bits hold a rate to 2^-17, and
// the factor is that of the rate as it is held, so that the mean stays what it was.
//
// Bound by memory: one tensor read (two with a residual), one written.  Products are fp32, rounded once.
#include "axc_gemm.h"

namespace axc {
namespace {

struct DropoutArgs {
    const void *x, *residual;
    void *y;
    long long count;
    unsigned share;                            // of 2^16 that are dropped
    float factor;
    unsigned key[2], offset[2];
    const long long *offset_device;
};

constexpr int kValues = 8;                     // of a counter
constexpr int kDropoutThreads = 256;

__device__ __forceinline__ uint4 philox(uint4 c, unsigned k0, unsigned k1)
{
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long p = (unsigned long long)c.x * 0xD2511F53u, q = (unsigned long long)c.z * 0xCD9E8D57u;
        c = make_uint4(unsigned(q >> 32) ^ c.y ^ k0, unsigned(q), unsigned(p >> 32) ^ c.w ^ k1, unsigned(p));
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}

template <typename T>
union Eight {
    uint4 w[kValues * sizeof(T) / 16];
    T t[kValues];
    __device__ Eight() {}
};
template <typename T, bool VEC>
__device__ __forceinline__ void load_eight(const T *from, long long left, Eight<T> &v)
{
    if (VEC && AXC_GLOBAL_OK(kValues - 1, left, 521u)) {
#pragma unroll
        for (int i = 0; i < int(kValues * sizeof(T) / 16); ++i) v.w[i] = reinterpret_cast<const uint4 *>(from)[i];
    } else {
#pragma unroll
        for (int i = 0; i < kValues; ++i) v.t[i] = i < left ? from[i] : narrow<T>(0.0f);
    }
}

// N counters a thread, kDropoutThreads apart
template <typename T, bool VEC, int N>
__global__ void __launch_bounds__(kDropoutThreads) dropout_kernel(const DropoutArgs P)
{
    after_previous();
    const T *x = static_cast<const T *>(P.x), *residual = static_cast<const T *>(P.residual);
    T *y = static_cast<T *>(P.y);
    const long long first = (long long)blockIdx.x * (kDropoutThreads * N) + threadIdx.x;
    unsigned offset0 = P.offset[0], offset1 = P.offset[1];
    if (P.offset_device) {
        const unsigned long long o = (unsigned long long)*P.offset_device;
        offset0 = unsigned(o);
        offset1 = unsigned(o >> 32);
    }
    Eight<T> v[N], r[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const long long at = (first + n * kDropoutThreads) * kValues, left = P.count - at;
        if (left <= 0) break;
        if (left >= kValues) {
            load_eight<T, VEC>(x + at, left, v[n]);
            if (residual) load_eight<T, VEC>(residual + at, left, r[n]);
        } else {
            load_eight<T, false>(x + at, left, v[n]);
            if (residual) load_eight<T, false>(residual + at, left, r[n]);
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const long long counter = first + n * kDropoutThreads, at = counter * kValues, left = P.count - at;
        if (left <= 0) break;
        const uint4 words = philox(make_uint4(unsigned(counter), unsigned(counter >> 32), offset0, offset1), P.key[0], P.key[1]);
        const unsigned word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            const unsigned bits = i & 1 ? word[i / 2] >> 16 : word[i / 2] & 0xffffu;
            float f = bits >= P.share ? widen(v[n].t[i]) * P.factor : 0.0f;
            if (residual) f += widen(r[n].t[i]);
            v[n].t[i] = narrow<T>(f);
        }
        if (VEC && left >= kValues) {
#pragma unroll
            for (int i = 0; i < int(kValues * sizeof(T) / 16); ++i) reinterpret_cast<uint4 *>(y + at)[i] = v[n].w[i];
        } else {
#pragma unroll
            for (int i = 0; i < kValues; ++i)
                if (i < left) y[at + i] = v[n].t[i];
        }
    }
}

template <typename T>
int run_dropout(const DropoutArgs &P, bool vec, Queue &q)
{
    constexpr int N = 2;
    const long long counters = (P.count + kValues - 1) / kValues, blocks = (counters + kDropoutThreads * N - 1) / (kDropoutThreads * N);
    if (blocks > 0x7fffffffll) return AXC_INVALID_ARGUMENT;
    return launch(q, vec ? dropout_kernel<T, true, N> : dropout_kernel<T, false, N>, dim3(unsigned(blocks)), kDropoutThreads, 0, 1, P);
}

}  // namespace

AXC_DEFINE_BOUNDS_READER(bounds_record_dropout)

}  // namespace axc

extern "C" int axc_dropout(const axc_dropout_desc *desc, const void *x, const void *residual, void *y, const int64_t *offset_device, int device, void *stream)
{
    using namespace axc;
    if (!desc || desc->count < 0 || desc->type < kFloat32 || desc->type > kFloat16 || !(desc->rate >= 0.0 && desc->rate <= 1.0) || device < 0) return AXC_INVALID_ARGUMENT;
    const axc_dropout_desc &d = *desc;
    if (d.count == 0) return AXC_OK;
    if (!x || !y || !aligned_to(type_size(d.type), x, residual, y) || !aligned_to(8, offset_device)) return AXC_INVALID_ARGUMENT;
    DropoutArgs P = {};
    P.x = x;
    P.residual = residual;
    P.y = y;
    P.count = d.count;
    P.share = unsigned(d.rate * 65536.0 + 0.5);
    P.factor = P.share < 65536u ? float(65536.0 / double(65536u - P.share)) : 0.0f;
    P.key[0] = unsigned(d.seed);
    P.key[1] = unsigned(d.seed >> 32);
    P.offset[0] = unsigned(d.offset);
    P.offset[1] = unsigned(d.offset >> 32);
    P.offset_device = reinterpret_cast<const long long *>(offset_device);
    int prev = 0;
    AXC_CUDA(cudaGetDevice(&prev));
    if (prev != device) AXC_CUDA(cudaSetDevice(device));
    Queue q = {cudaStream_t(stream)};
    const bool vec = aligned_to(16, x, residual, y);
    int rc = d.type == kFloat32 ? run_dropout<float>(P, vec, q) : d.type == kBfloat16 ? run_dropout<__nv_bfloat16>(P, vec, q) : run_dropout<__half>(P, vec, q);
    const cudaError_t e = cudaGetLastError();
    if (!rc && e != cudaSuccess) rc = cuda_failed(e);
    if (prev != device) cudaSetDevice(prev);
    return rc;
}
