// The exact dense layer: y = act(x kernel + bias + residual), and its gradients.  The products are those of axc_gemm.cu; here are
// the pass over the output's gradient between them, and the entry points.
#include "axc_gemm.h"

namespace axc {
namespace {

// ------------------------------------------------------------------------------------------------
// dz = dy act'(kept), column sums on the way.  A block takes 32 groups of V neighbouring columns and a share of the rows, four times 8
// rows at a time; the sums of its 8 rows are added in shared memory, those of the blocks by a second kernel, in a fixed order.  Bound
// by reading dy and kept and writing dz once.
// ------------------------------------------------------------------------------------------------
constexpr int kShares = 64;                    // blocks that share the rows, at most
constexpr int kRows = 4;                       // of a thread, whose loads are in flight together

template <int ACT, bool EXACT>
__device__ __forceinline__ float slope_of(float kept)
{
    if (ACT == kActRelu) return kept > 0.0f ? 1.0f : (kept != kept ? kept : 0.0f);
    if (ACT == kActGelu) return 0.5f * (1.0f + (EXACT ? erff(kept * 0.70710678f) : erf_16bit(kept * 0.70710678f))) + kept * __expf(-0.5f * kept * kept) * 0.39894228f;
    const float s = __fdividef(1.0f, 1.0f + __expf(-kept));
    return s * (1.0f + kept * (1.0f - s));
}

template <typename T>
union Group {                                  // 16 bytes of values
    static constexpr int V = 16 / sizeof(T);
    uint4 w;
    T t[V];
    __device__ Group() {}
};

template <typename T>
__device__ __forceinline__ void load_group(const T *at, bool vec, long long left, Group<T> &g)
{
    if (vec) g.w = __ldcs(reinterpret_cast<const uint4 *>(at));
    else {
#pragma unroll
        for (int i = 0; i < Group<T>::V; ++i) g.t[i] = i < left ? at[i] : narrow<T>(0.0f);
    }
}

// What is loaded stays packed until it is needed: 8 loads of a thread in flight and three blocks on an SM.
template <typename T, int ACT>
__global__ void __launch_bounds__(256, 3) slope_kernel(const Slope S, float *part, bool vec)
{
    constexpr int V = Group<T>::V;
    __shared__ float sums[8][32 * V];
    const int group = threadIdx.x & 31, r0 = threadIdx.x >> 5;
    const long long c = ((long long)blockIdx.x * 32 + group) * V, left = S.columns - c;
    const long long begin = S.rows * blockIdx.y / gridDim.y, end = S.rows * (blockIdx.y + 1) / gridDim.y;
    const bool full = vec && (left >= V || S.padded);
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    if (left > 0) {
        for (long long first = begin + r0; first < end; first += 8 * kRows) {
            Group<T> dy[kRows], kept[ACT != kActNone ? kRows : 1];
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                const long long r = first + 8 * q < end ? first + 8 * q : first;
                load_group(static_cast<const T *>(S.dy) + r * S.dy_line + c, full, left, dy[q]);
                if constexpr (ACT != kActNone) load_group(static_cast<const T *>(S.kept) + r * S.columns + c, full, left, kept[q]);
            }
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                const long long r = first + 8 * q;
                if (r >= end) continue;
                float d[V];
#pragma unroll
                for (int i = 0; i < V; ++i) d[i] = widen(dy[q].t[i]);
                for (int p = 1; p < S.dy_planes; ++p) {
                    Group<T> more;
                    load_group(static_cast<const T *>(S.dy) + p * S.plane + r * S.dy_line + c, full, left, more);
#pragma unroll
                    for (int i = 0; i < V; ++i) d[i] += widen(more.t[i]);
                }
                if constexpr (ACT != kActNone) {
#pragma unroll
                    for (int i = 0; i < V; ++i) d[i] *= slope_of<ACT, sizeof(T) == 4>(widen(kept[q].t[i]));
                }
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += d[i];
                if (S.same || (S.planes && sizeof(T) == 2)) {
                    Group<T> u;
#pragma unroll
                    for (int i = 0; i < V; ++i) u.t[i] = narrow<T>(i < left ? d[i] : 0.0f);
                    if (S.same) {
                        T *to = static_cast<T *>(S.same) + r * S.columns + c;
                        if (full) *reinterpret_cast<uint4 *>(to) = u.w;
                        else {
#pragma unroll
                            for (int i = 0; i < V; ++i)
                                if (i < left) to[i] = u.t[i];
                        }
                    }
                    // lines of a multiple of 8 values, zeros behind the last column
                    if (S.planes && sizeof(T) == 2) *reinterpret_cast<uint4 *>(S.planes + r * S.line + c) = u.w;
                }
                if (S.planes && sizeof(T) == 4) {
                    uint16_t *to = S.planes + r * S.line + c;
                    for (int p = 0; p < 3; ++p) {
                        union { uint2 w; uint16_t h[4]; } u;
#pragma unroll
                        for (int i = 0; i < 4; ++i) u.h[i] = split_term(i < left ? d[i] : 0.0f, d[i]);
                        *reinterpret_cast<uint2 *>(to + p * S.plane) = u.w;
                    }
                }
            }
        }
    }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < V; ++i) sums[r0][group * V + i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V; i += 256) {
        float s = sums[0][i];
#pragma unroll
        for (int k = 1; k < 8; ++k) s += sums[k][i];
        const long long column = (long long)blockIdx.x * 32 * V + i;
        if (column < S.columns) part[(long long)blockIdx.y * S.columns + column] = s;
    }
}

__global__ void __launch_bounds__(256) slope_sums_kernel(const float *__restrict__ part, long long columns, int shares, float scale, const float *scale_dev,
                                                         void *sums, int type)
{
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    if (c >= columns) return;
    float s = 0.0f;
    for (int k = 0; k < shares; ++k) s += part[k * columns + c];
    store_from_float(sums, c, type, s * scale * (scale_dev ? *scale_dev : 1.0f));
}

int shares_of(long long rows, long long columns)
{
    // about eight blocks for every SM, of at least one round of rows each
    long long shares = (rows + 8 * kRows - 1) / (8 * kRows);
    const long long across = columns / 256 + 1, most = 1184 / across + 1;
    if (shares > most) shares = most;
    if (shares > kShares) shares = kShares;
    return int(shares < 1 ? 1 : shares);
}

template <typename T>
void launch_slope(const Slope &s, float *part, int shares, bool vec, cudaStream_t stream)
{
    const dim3 grid(unsigned((s.columns + 32 * Group<T>::V - 1) / (32 * Group<T>::V)), unsigned(shares));
    if (!s.kept) slope_kernel<T, kActNone><<<grid, 256, 0, stream>>>(s, part, vec);
    else if (s.activation == kActRelu) slope_kernel<T, kActRelu><<<grid, 256, 0, stream>>>(s, part, vec);
    else if (s.activation == kActGelu) slope_kernel<T, kActGelu><<<grid, 256, 0, stream>>>(s, part, vec);
    else slope_kernel<T, kActSilu><<<grid, 256, 0, stream>>>(s, part, vec);
    count_launch();
}

}  // namespace

size_t slope_scratch(long long rows, long long columns) { return size_t(shares_of(rows, columns)) * size_t(columns) * 4; }

int slope(const Slope &s, void *scratch, const DeviceInfo &di, cudaStream_t stream)
{
    (void)di;
    if (s.columns == 0 || (s.rows == 0 && !s.sums)) return AXC_OK;
    const int shares = shares_of(s.rows, s.columns);
    float *part = s.sums ? static_cast<float *>(scratch) : nullptr;
    const uintptr_t all = reinterpret_cast<uintptr_t>(s.dy) | reinterpret_cast<uintptr_t>(s.kept) | reinterpret_cast<uintptr_t>(s.same);
    const long long size = s.type == kFloat32 ? 4 : 2;
    const bool vec = (all & 15u) == 0 && s.dy_line * size % 16 == 0 && ((!s.kept && !s.same) || s.columns * size % 16 == 0) && s.plane * size % 16 == 0;
    if (s.type == kFloat32) launch_slope<float>(s, part, shares, vec, stream);
    else if (s.type == kBfloat16) launch_slope<__nv_bfloat16>(s, part, shares, vec, stream);
    else launch_slope<__half>(s, part, shares, vec, stream);
    if (s.sums) {
        slope_sums_kernel<<<unsigned((s.columns + 255) / 256), 256, 0, stream>>>(part, s.columns, shares, s.scale, s.scale_dev, s.sums, s.sums_type);
        count_launch();
    }
    return AXC_OK;
}

namespace {

bool valid_type(int t) { return t >= kFloat32 && t <= kFloat16; }

int check_desc(const axc_dense_desc *d)
{
    if (!d || !valid_type(d->type) || !valid_type(d->bias_type) || d->activation < kActNone || d->activation > kActSilu) return AXC_INVALID_ARGUMENT;
    if (d->rows < 0 || d->inputs < 0 || d->units < 0 || d->rows > 0x7fffff00ll || d->inputs > 0x7fffff00ll || d->units > 0x7fffff00ll) return AXC_INVALID_ARGUMENT;
    if (d->x_row_stride < 0 || d->x_column_stride < 0 || d->kernel_row_stride < 0 || d->kernel_column_stride < 0 || d->residual_row_stride < 0)
        return AXC_INVALID_ARGUMENT;
    return AXC_OK;
}

Matrix x_of(const axc_dense_desc &d, const void *x) { return {x, d.rows, d.inputs, d.x_row_stride, d.x_column_stride, d.type}; }
// rows: units
Matrix kernel_of(const axc_dense_desc &d, const void *k) { return {k, d.units, d.inputs, d.kernel_column_stride, d.kernel_row_stride, d.type}; }
Matrix dy_of(const axc_dense_desc &d, const void *dy) { return {dy, d.rows, d.units, d.units, 1, d.type}; }

// Where the parts of a call's workspace lie.
struct Parts {
    size_t x, kernel, dz, part, scratch, total;
};
size_t up(size_t n) { return (n + 255) / 256 * 256; }
size_t largest(size_t a, size_t b) { return a > b ? a : b; }

// Addresses that no tensor has stand for unknown ones: sized for a copy of every operand.
const void *const kUnknown = reinterpret_cast<const void *>(uintptr_t(2));

Parts parts_of(const axc_dense_desc &d, bool backward, const void *x, const void *kernel, const DeviceInfo &di)
{
    const int planes = d.type == kFloat32 ? 3 : 1;
    Parts p;
    p.x = 256;
    p.kernel = p.x + up(operand_bytes(x_of(d, x)));
    p.dz = p.kernel + up(operand_bytes(kernel_of(d, kernel)));
    p.part = p.dz + (backward ? up(size_t(d.rows) * size_t((d.units + 7) / 8 * 8) * 2 * planes) : 0);
    p.scratch = p.part + (backward ? up(slope_scratch(d.rows, d.units)) : 0);
    size_t most = 0;
    if (!backward) most = gemm_scratch(d.rows, d.units, d.inputs, planes, di);
    else most = largest(gemm_scratch(d.rows, d.inputs, d.units, planes, di),
                        d.kernel_gradient_transposed ? gemm_scratch(d.units, d.inputs, d.rows, planes, di) : gemm_scratch(d.inputs, d.units, d.rows, planes, di));
    p.total = p.scratch + up(most);
    return p;
}

int enter(int device, DeviceInfo *di, int *prev)
{
    const int rc = device_info(device, di);
    if (rc) return rc;
    AXC_CUDA(cudaGetDevice(prev));
    if (*prev != device) AXC_CUDA(cudaSetDevice(device));
    return AXC_OK;
}
int leave(int rc, int device, int prev)
{
    const cudaError_t e = cudaGetLastError();
    if (prev != device) cudaSetDevice(prev);
    return rc != AXC_OK ? rc : e == cudaSuccess ? AXC_OK : cuda_failed(e);
}

int forward(const axc_dense_desc &d, const void *x, const void *kernel, const void *bias, const void *residual, void *y, void *pre, char *ws,
            const DeviceInfo &di, cudaStream_t stream)
{
    const Parts parts = parts_of(d, false, x, kernel, di);
    Gemm g = {};
    g.m = d.rows;
    g.n = d.units;
    g.k = d.inputs;
    g.planes = d.type == kFloat32 ? 3 : 1;
    g.bf16 = d.type != kFloat16;
    int rc = AXC_OK;
    if (d.inputs > 0) {
        rc = make_operand(x_of(d, x), ws + parts.x, &g.a, di, stream);
        if (rc == AXC_OK) rc = make_operand(kernel_of(d, kernel), ws + parts.kernel, &g.b, di, stream);
        if (rc) return rc;
    }
    g.fin.alpha = 1.0f;
    g.fin.bias = bias;
    g.fin.bias_type = d.bias_type;
    g.fin.addend = residual;
    g.fin.addend_type = d.type;
    g.fin.addend_line = d.residual_row_stride;
    g.fin.activation = d.activation;
    g.fin.out = y;
    g.fin.out_type = d.type;
    g.fin.out_line = d.units;
    g.fin.pre = pre;
    return gemm(g, ws + parts.scratch, reinterpret_cast<unsigned *>(ws), true, di, stream);
}

int backward(const axc_dense_desc &d, const void *dy, const void *x, const void *kernel, const void *kept, void *dx, void *dkernel, void *dbias,
             void *dresidual, char *ws, const DeviceInfo &di, cudaStream_t stream)
{
    const Parts parts = parts_of(d, true, x, kernel, di);
    const int planes = d.type == kFloat32 ? 3 : 1;
    const long long line = (d.units + 7) / 8 * 8;
    unsigned *status = reinterpret_cast<unsigned *>(ws);
    // the operand dz: dy itself, or what the pass over it writes
    const bool act = d.activation != kActNone, product = dx || dkernel;
    const bool direct = !act && readable_in_place(dy_of(d, dy));
    Operand dz = {dy, d.units, 0, false};
    Slope s = {};
    s.dy = dy;
    s.kept = act ? kept : nullptr;
    s.type = d.type;
    s.rows = d.rows;
    s.columns = s.dy_line = d.units;
    s.activation = d.activation;
    s.same = dresidual;
    s.dy_planes = 1;
    if (product && !direct) {
        const bool in_place = dresidual && readable_in_place(dy_of(d, dresidual));
        if (in_place) dz.data = dresidual;
        else {
            s.planes = reinterpret_cast<uint16_t *>(ws + parts.dz);
            s.line = line;
            s.plane = line * d.rows;
            dz = {s.planes, line, s.plane, false};
        }
    }
    s.sums = dbias;
    s.sums_type = d.bias_type;
    s.scale = 1.0f;
    int rc = AXC_OK;
    if (s.same || s.planes || s.sums) rc = slope(s, ws + parts.part, di, stream);
    if (rc) return rc;
    bool first = true;
    Operand operand = {};
    if (dx) {
        if (d.units > 0) rc = make_operand(kernel_of(d, kernel), ws + parts.kernel, &operand, di, stream);
        if (rc) return rc;
        Gemm g = {};
        g.m = d.rows;
        g.n = d.inputs;
        g.k = d.units;
        g.planes = planes;
        g.bf16 = d.type != kFloat16;
        g.a = dz;
        g.b = transposed(operand);
        g.fin.alpha = 1.0f;
        g.fin.out = dx;
        g.fin.out_type = d.type;
        g.fin.out_line = d.inputs;
        rc = gemm(g, ws + parts.scratch, status, first, di, stream);
        if (rc) return rc;
        first = false;
    }
    if (dkernel) {
        if (d.rows > 0) rc = make_operand(x_of(d, x), ws + parts.x, &operand, di, stream);
        if (rc) return rc;
        Gemm g = {};
        g.k = d.rows;
        g.planes = planes;
        g.bf16 = d.type != kFloat16;
        g.fin.alpha = 1.0f;
        g.fin.out = dkernel;
        g.fin.out_type = d.type;
        if (d.kernel_gradient_transposed) {
            g.m = d.units;
            g.n = d.inputs;
            g.a = transposed(dz);
            g.b = transposed(operand);
        } else {
            g.m = d.inputs;
            g.n = d.units;
            g.a = transposed(operand);
            g.b = transposed(dz);
        }
        g.fin.out_line = g.n;
        rc = gemm(g, ws + parts.scratch, status, first, di, stream);
        if (rc) return rc;
        first = false;
    }
    if (first) AXC_CUDA(cudaMemsetAsync(status, 0, sizeof(unsigned), stream));
    return AXC_OK;
}

}  // namespace
}  // namespace axc

extern "C" int axc_dense_workspace_bytes(const axc_dense_desc *desc, const void *x, const void *kernel, int device, size_t *forward, size_t *backward)
{
    using namespace axc;
    int rc = check_desc(desc);
    if (rc) return rc;
    DeviceInfo di;
    rc = device_info(device, &di);
    if (rc) return rc;
    if (!x) x = kUnknown;
    if (!kernel) kernel = kUnknown;
    if (forward) *forward = parts_of(*desc, false, x, kernel, di).total;
    if (backward) *backward = parts_of(*desc, true, x, kernel, di).total;
    return AXC_OK;
}

extern "C" int axc_dense_forward(const axc_dense_desc *desc, const void *x, const void *kernel, const void *bias, const void *residual, void *y, void *pre,
                                 void *workspace, size_t workspace_bytes, int device, void *stream)
{
    using namespace axc;
    int rc = check_desc(desc);
    if (rc) return rc;
    const axc_dense_desc &d = *desc;
    if (d.rows == 0 || d.units == 0) return AXC_OK;
    if (!y || (d.inputs > 0 && (!x || !kernel))) return AXC_INVALID_ARGUMENT;
    DeviceInfo di;
    rc = device_info(device, &di);
    if (rc) return rc;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < parts_of(d, false, x, kernel, di).total) return AXC_INTERNAL;
    int prev = 0;
    rc = enter(device, &di, &prev);
    if (rc) return rc;
    return leave(forward(d, x, kernel, bias, residual, y, pre, static_cast<char *>(workspace), di, cudaStream_t(stream)), device, prev);
}

extern "C" int axc_dense_backward(const axc_dense_desc *desc, const void *dy, const void *x, const void *kernel, const void *kept, void *dx, void *dkernel,
                                  void *dbias, void *dresidual, void *workspace, size_t workspace_bytes, int device, void *stream)
{
    using namespace axc;
    int rc = check_desc(desc);
    if (rc) return rc;
    const axc_dense_desc &d = *desc;
    const bool some = d.rows > 0 && d.units > 0;
    if (some && (!dy || (d.activation != kActNone && !kept))) return AXC_INVALID_ARGUMENT;
    if (d.inputs > 0 && some && ((dx && !kernel) || (dkernel && !x))) return AXC_INVALID_ARGUMENT;
    if (d.rows == 0 && d.units == 0) return AXC_OK;
    DeviceInfo di;
    rc = device_info(device, &di);
    if (rc) return rc;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < parts_of(d, true, x, kernel, di).total) return AXC_INTERNAL;
    int prev = 0;
    rc = enter(device, &di, &prev);
    if (rc) return rc;
    return leave(backward(d, dy, x, kernel, kept, dx, dkernel, dbias, dresidual, static_cast<char *>(workspace), di, cudaStream_t(stream)), device, prev);
}

extern "C" int axc_matrix_status(const void *workspace, int32_t *status, int device, void *stream)
{
    using namespace axc;
    if (!workspace || !status) return AXC_INVALID_ARGUMENT;
    int prev = 0;
    AXC_CUDA(cudaGetDevice(&prev));
    if (prev != device) AXC_CUDA(cudaSetDevice(device));
    cudaError_t e = cudaMemcpyAsync(status, workspace, sizeof(*status), cudaMemcpyDeviceToHost, cudaStream_t(stream));
    if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStream_t(stream));
    if (prev != device) cudaSetDevice(prev);
    return e == cudaSuccess ? AXC_OK : cuda_failed(e);
}
