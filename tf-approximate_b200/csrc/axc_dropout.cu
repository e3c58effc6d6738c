// Dropout whose mask is never stored: it is computed where it is needed, in the forward and in the backward pass, from a counter.
//
//   y[i] = (bits[i] >= share ? x[i] * factor : 0) + residual[i],  share = round(rate 2^16),  factor = 2^16 / (2^16 - share)
//
// bits[i]: 16 of the 128 that Philox 4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) makes of
// the counter {i / 8, offset} under the key `seed`.  Eight values share a counter: its 20 wide multiplications and 20 three-way xors take about as long
// as memory takes for eight 16-bit values in and out; with 32 bits a value they would take twice that.  16 bits hold a rate to 2^-17, and the factor is
// that of the rate as it is held, so that the mean stays what it was.
//
// Bound by memory: one tensor read (two with a residual), one written; for 16-bit types without a residual by the generator.  Products are fp32, rounded
// once.  802 816 x 256 bf16: 170 us (82 % of it the generator and what is made of its words; memory alone 126), with a residual 195 (188); 401 408 x 256 fp32:
// 123 us (126).  One, two and four counters a thread: 177, 170, 162 us; for 7.8 million values 10.1, 9.3, 10.6.
#include <type_traits>

#include "axc_gemm.h"

namespace axc {
namespace {

constexpr int kRounds = 10;

struct DropoutArgs {
    const void *x, *residual;
    void *y;
    long long count;
    unsigned least;                            // a value whose 16 bits, as the high ones of a word, are below it is dropped
    bool nothing;                              // all are
    float factor;
    unsigned key[kRounds][2], offset[2];       // the keys of all rounds
    const long long *offset_device;
};

constexpr int kValues = 8;                     // of a counter
constexpr int kDropoutThreads = 256;

__device__ __forceinline__ uint4 philox(uint4 c, const unsigned (&key)[kRounds][2])
{
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const unsigned long long p = (unsigned long long)c.x * 0xD2511F53u, q = (unsigned long long)c.z * 0xCD9E8D57u;
        c = make_uint4(unsigned(q >> 32) ^ c.y ^ key[r][0], unsigned(q), unsigned(p >> 32) ^ c.w ^ key[r][1], unsigned(p));
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
        for (int i = 0; i < int(kValues * sizeof(T) / 16); ++i) v.w[i] = __ldcs(reinterpret_cast<const uint4 *>(from) + i);
    } else {
#pragma unroll
        for (int i = 0; i < kValues; ++i) v.t[i] = i < left ? from[i] : narrow<T>(0.0f);
    }
}
// values 2 i and 2 i + 1
template <typename T>
__device__ __forceinline__ Two pair_of(const Eight<T> &v, int i)
{
    if constexpr (sizeof(T) == 4) return Two(v.t[2 * i], v.t[2 * i + 1]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const unsigned w = reinterpret_cast<const unsigned *>(v.w)[i];
        return Two(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else {
        const float2 f = __half22float2(reinterpret_cast<const __half2 *>(v.w)[i]);
        return Two(f.x, f.y);
    }
}

// N counters a thread, kDropoutThreads apart
template <typename T, bool VEC, int N>
__global__ void __launch_bounds__(kDropoutThreads) dropout_kernel(const __grid_constant__ DropoutArgs P)
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
        const uint4 words = philox(make_uint4(unsigned(counter), unsigned(counter >> 32), offset0, offset1), P.key);
        const unsigned word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
        for (int i = 0; i < kValues / 2; ++i) {
            float2 f = mul2(pair_of(v[n], i), Two(P.factor)).both();
            f.x = word[i] << 16 >= P.least && !P.nothing ? f.x : 0.0f;
            f.y = word[i] >= P.least && !P.nothing ? f.y : 0.0f;
            if (residual) f = add2(Two(f.x, f.y), pair_of(r[n], i)).both();
            if constexpr (sizeof(T) == 4) {
                v[n].t[2 * i] = f.x;
                v[n].t[2 * i + 1] = f.y;
            } else reinterpret_cast<unsigned *>(v[n].w)[i] = pack2(f.x, f.y, std::is_same<T, __nv_bfloat16>::value);
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
    const unsigned share = unsigned(d.rate * 65536.0 + 0.5);
    P.nothing = share >= 65536u;
    P.least = share << 16;
    P.factor = P.nothing ? 0.0f : float(65536.0 / double(65536u - share));
    for (unsigned r = 0; r < kRounds; ++r) {
        P.key[r][0] = unsigned(d.seed) + r * 0x9E3779B9u;
        P.key[r][1] = unsigned(d.seed >> 32) + r * 0xBB67AE85u;
    }
    P.offset[0] = unsigned(d.offset);
    P.offset[1] = unsigned(d.offset >> 32);
    P.offset_device = reinterpret_cast<const long long *>(offset_device);
    Queue q = {cudaStream_t(stream)};
    const bool vec = aligned_to(16, x, residual, y);
    return on_device(device, [&] {
        return d.type == kFloat32 ? run_dropout<float>(P, vec, q) : d.type == kBfloat16 ? run_dropout<__nv_bfloat16>(P, vec, q) : run_dropout<__half>(P, vec, q);
    });
}
