// Matrix products on the tensor cores, shared by the dense layer and the dense cross entropy.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include "axc_internal.h"
#include "axc_pieces.h"

namespace axc {

enum { kFloat32 = AXC_TYPE_FLOAT32, kBfloat16 = AXC_TYPE_BFLOAT16, kFloat16 = AXC_TYPE_FLOAT16 };
// The launches of a call.  Every kernel after the first may start while the one before it ends: it waits for that one, whole and
// visible, before it touches memory (after_previous), so that only its set-up overlaps.
struct Queue {
    cudaStream_t stream;
    bool first = true;
};
template <typename... Params, typename... Args>
inline int launch(Queue &q, void (*kernel)(Params...), dim3 grid, unsigned threads, unsigned smem, unsigned cluster, Args &&...args)
{
    cudaLaunchAttribute attr[2] = {};
    unsigned n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (!q.first) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    q.first = false;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = q.stream;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    AXC_CUDA(cudaLaunchKernelEx(&cfg, kernel, Params(args)...));
    count_launch();
    return AXC_OK;
}
// First in every kernel that `launch` starts: the next kernel may come, the one before is over.
__device__ __forceinline__ void after_previous()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

inline size_t type_size(int type) { return type == kFloat32 ? 4 : 2; }
// Whether every address is a multiple of `size`: what a kernel cannot load or store elsewhere (NULL is)
template <typename... P>
inline bool aligned_to(size_t size, P... p)
{
    return ((uintptr_t(0) | ... | reinterpret_cast<uintptr_t>(p)) % size) == 0;
}

template <typename T> __device__ __forceinline__ float widen(T x);
template <> __device__ __forceinline__ float widen<float>(float x) { return x; }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float widen<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ float narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

// element i of an array of `type`
__device__ __forceinline__ float load_as_float(const void *p, long long i, int type)
{
    if (type == kFloat32) return *(static_cast<const float *>(p) + i);
    if (type == kBfloat16) return __bfloat162float(*(static_cast<const __nv_bfloat16 *>(p) + i));
    return __half2float(*(static_cast<const __half *>(p) + i));
}
__device__ __forceinline__ void store_from_float(void *p, long long i, int type, float x)
{
    if (type == kFloat32) static_cast<float *>(p)[i] = x;
    else if (type == kBfloat16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
    else static_cast<__half *>(p)[i] = __float2half_rn(x);
}
// two values of a 16-bit type, the first in the low half
__device__ __forceinline__ unsigned pack2(float a, float b, bool bf16)
{
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return reinterpret_cast<const unsigned &>(h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return reinterpret_cast<const unsigned &>(h);
}

__device__ __forceinline__ float reciprocal(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// exp(x) of a softmax, x <= 0: exact for fp32 operands; the other one is off by some |x| 2^-23 of itself
__device__ __forceinline__ float exponential(float x, bool exact) { return exact ? expf(x) : __expf(x); }

// Phi(z), the normal distribution below z, and bell = exp(-z^2 / 2), which it is made of.  The smaller side, erfc(|z| / sqrt 2) / 2, is bell times a
// polynomial in t = 1 / (1 + p |z| / sqrt 2), as Hastings has it, with coefficients of its own: the least largest RELATIVE error for |z| up to 13 (an
// exchange over 20 000 points), so that GELU's tail, which is that side times z, is as good as the rest; 1 + erf has lost it.
//   exact    fp32 results: p = 0.375, nine terms, 1.1e-8, six units of 2^-24 with its operations' rounding; expf, whose argument's rounding is z^2 units
//   else     16-bit results: p = 0.435, six terms, 3.7e-6, and an exponential good to 2^-20 of itself
__device__ __forceinline__ float normal_below(float z, float &bell, bool exact)
{
    const float a = fabsf(z);
    float poly;
    if (exact) {
        const float t = reciprocal(fmaf(0.265165031f, a, 1.0f));
        bell = expf(-0.5f * a * a);
        poly = fmaf(t, 0.0308483057f, -0.144037679f);
        poly = fmaf(t, poly, 0.21694687f);
        poly = fmaf(t, poly, -0.115538195f);
        poly = fmaf(t, poly, 0.137422055f);
        poly = fmaf(t, poly, 0.0605194829f);
        poly = fmaf(t, poly, 0.102715209f);
        poly = fmaf(t, poly, 0.105316751f);
        poly = t * fmaf(t, poly, 0.105807208f);
    } else {
        const float t = reciprocal(fmaf(0.30759144f, a, 1.0f));
        bell = __expf(-0.5f * a * a);
        poly = fmaf(t, -0.0758679435f, 0.191902518f);
        poly = fmaf(t, poly, 0.00506413169f);
        poly = fmaf(t, poly, 0.137423128f);
        poly = fmaf(t, poly, 0.118498363f);
        poly = t * fmaf(t, poly, 0.122977965f);
    }
    const float side = poly * bell;
    return z < 0.0f ? side : 1.0f - side;
}
// 1 / (1 + exp(-z))
__device__ __forceinline__ float sigmoid(float z, bool exact) { return reciprocal(1.0f + (exact ? expf(-z) : __expf(-z))); }

// The three bf16 terms of x and of y, x in the low half: the value rounded, the rest rounded again, and what is left then, which bf16
// holds exactly.  A value beyond bf16's range has its largest finite term first.  An infinity is (1, 0, inf) with its sign: of the six products of terms
// that are summed, the third one is in that with the other operand's first term alone, so that inf meets no term that is zero because
// the value needs no more of them; its own first term stands for it where the other operand is infinite, too.  NaN likewise.
__device__ __forceinline__ void split_terms(float x, float y, unsigned (&term)[3])
{
    constexpr float kLargest = 3.38953139e38f;                 // of bf16
    const bool fx = fabsf(x) <= FLT_MAX, fy = fabsf(y) <= FLT_MAX;
    float rx = fx ? x : copysignf(1.0f, x), ry = fy ? y : copysignf(1.0f, y);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const float hx = p == 0 ? fminf(fmaxf(rx, -kLargest), kLargest) : p == 2 && !fx ? x : rx;
        const float hy = p == 0 ? fminf(fmaxf(ry, -kLargest), kLargest) : p == 2 && !fy ? y : ry;
        const __nv_bfloat162 h = __floats2bfloat162_rn(hx, hy);
        term[p] = reinterpret_cast<const unsigned &>(h);
        const float2 back = __bfloat1622float2(h);
        rx -= back.x;
        ry -= back.y;
    }
}

// A matrix of `rows` x `k` as the tensor cores read it: 16-bit values (bf16, or fp16), either k or the rows contiguous, 16-byte
// aligned lines.  fp32 matrices are three such planes whose sum is the value to the bit (see split_terms).
struct Operand {
    const void *data;
    long long line;             // values from one line to the next
    long long plane;            // values from one plane to the next
    bool rows_contiguous;
};

enum { kActNone = AXC_ACTIVATION_NONE, kActRelu = AXC_ACTIVATION_RELU, kActGelu = AXC_ACTIVATION_GELU, kActSilu = AXC_ACTIVATION_SILU };

// What becomes of a sum: out = act(alpha * sum + bias[column] + addend), columns of the output.
struct Finish {
    float alpha;
    const float *alpha_dev;     // NULL, or a factor in device memory
    const void *bias;
    int bias_type;
    const void *addend;
    int addend_type;
    long long addend_line;
    int activation;
    void *out;
    int out_type;
    long long out_line;
    void *pre;                  // NULL, or where the activation's argument goes (out_type, out_line)
    long long lines, columns;   // of the output; set by the products
    __host__ __device__ long long out_values() const { return (lines - 1) * out_line + columns; }
    __host__ __device__ long long addend_values() const { return (lines - 1) * addend_line + columns; }
};
inline Finish sized(Finish f, long long lines, long long columns)
{
    f.lines = lines;
    f.columns = columns;
    return f;
}

// `exact`: for fp32 results
__device__ __forceinline__ float activate(float z, int act, bool exact)
{
    if (act == kActRelu) return max_keep_nan(z, 0.0f);
    float bell;
    if (act == kActGelu) return z * normal_below(z, bell, exact);
    if (act == kActSilu) return z * sigmoid(z, exact);
    return z;
}

// One value of an output: line, column
__device__ __forceinline__ void finish_value(const Finish &f, float z, long long line, long long column)
{
    if (f.bias && AXC_GLOBAL_OK(column, f.columns, 421u)) z += load_as_float(f.bias, column, f.bias_type);
    if (f.addend && AXC_GLOBAL_OK(line * f.addend_line + column, f.addend_values(), 422u)) z += load_as_float(f.addend, line * f.addend_line + column, f.addend_type);
    const long long at = line * f.out_line + column;
    if (!AXC_GLOBAL_OK(at, f.out_values(), 423u)) return;
    if (f.pre) store_from_float(f.pre, at, f.out_type, z);
    store_from_float(f.out, at, f.out_type, activate(z, f.activation, f.out_type == kFloat32));
}

// What the cross entropy makes of a tile of logits; see axc_entropy.cu.
struct EntropyArgs {
    const void *bias;
    int bias_type;
    const long long *labels;
    void *keep;                 // exponentials relative to their segment's largest logit, or (gradient) the logits' gradient
    long long line, plane;
    int keep_fp32;              // exponentials as fp32 instead of fp16
    float2 *stats;              // [rows][segments] {largest logit, sum of exponentials relative to it}
    int segments;
    float *label_logit;
    const float2 *softmax;      // gradient only: a row's largest logit, and 1 / its sum of exponentials relative to that
    const float *row_scale;     // gradient only: 0 for rows without a label, else the scale of the stored gradient
    int column0;                // gradient only: first class of this piece
};

struct Gemm {
    long long m, n, k;          // out[m, n] = sum over k of a[m, k] b[n, k]
    Operand a, b;
    int planes;                 // 1, or 3 for fp32 operands
    bool bf16;
    Finish fin;
};

// Scratch for the partial sums of a product whose k is split; 0 where it is not.
size_t gemm_scratch(long long m, long long n, long long k, int planes, const DeviceInfo &di);
// `first`: of the products of a call; it clears the status word.
int gemm(const Gemm &g, void *scratch, unsigned *status, bool first, const DeviceInfo &di, Queue &q);
// The sums alone, as `count` parts that are to be added in order: part i of out[r, c] at data[i * stride + r * line + c].
struct Parts {
    const float *data;
    long long line, stride;
    int count;
};
int finish_parts(const Parts &parts, long long lines, long long columns, const Finish &f, const DeviceInfo &di, Queue &q);
size_t gemm_parts_scratch(long long m, long long n, long long k, int planes, const DeviceInfo &di);
int gemm_parts(const Gemm &g, void *scratch, Parts *parts, unsigned *status, bool first, const DeviceInfo &di, Queue &q);
// Tiles of logits, never split; `gradient`: the second pass of the piecewise form.
int gemm_entropy(const Gemm &g, const EntropyArgs &e, bool gradient, unsigned *status, bool first, const DeviceInfo &di, Queue &q);

// Gradient of an activation and the sums of its columns, in one pass over dy [rows, columns]:
//   dz = dy * act'(kept);  to `same` (dy's type and layout) and / or to the 16-bit planes of an operand, where given;
//   sums[column] = scale * sum of dz, as bias_type, where given.
// `kept`: the activation's argument, for relu its value; NULL without an activation.
struct Slope {
    const void *dy, *kept;
    int type;
    long long rows, columns, dy_line;
    int activation;
    void *same;
    uint16_t *planes;
    long long line, plane;
    int dy_planes;              // 1, or 3: dy is bf16 and the sum of three planes `plane` apart
    bool padded;                // dy's lines have values that do not matter up to a multiple of 16 bytes
    void *sums;
    int sums_type;
    float scale;
    const float *scale_dev;
    // values of dy, and of a tensor or operand that has a line for every row
    __host__ __device__ long long dy_values() const { return (rows - 1) * dy_line + (padded ? dy_line : columns) + (dy_planes - 1) * plane; }
    __host__ __device__ long long tensor_values() const { return rows * columns; }
    __host__ __device__ long long operand_values() const { return rows * line; }
};
// `room`: bytes of the scratch, slope_scratch(rows, columns) at least; less is refused.
int slope(const Slope &s, void *scratch, size_t room, Queue &q);

// ---- operands -----------------------------------------------------------------------------------------------------------
// A matrix in the caller's memory: element (r, c) at data[r * row_stride + c * column_stride]
struct Matrix {
    const void *data;
    long long rows, columns, row_stride, column_stride;
    int type;
};
// Whether the tensor cores can read it where it is (16-bit, one unit stride, lines of a multiple of 16 bytes, aligned).
bool readable_in_place(const Matrix &x);
size_t operand_bytes(const Matrix &x);          // scratch that operand() fills, 0 where it reads in place
// Two matrices as operands whose rows are theirs; copies and splits into the scratch as needed, in one launch.
int make_operands(const Matrix &x, void *x_scratch, Operand *ox, const Matrix &y, void *y_scratch, Operand *oy, const DeviceInfo &di, Queue &q);
inline Operand transposed(Operand o)
{
    o.rows_contiguous = !o.rows_contiguous;
    return o;
}

}  // namespace axc
