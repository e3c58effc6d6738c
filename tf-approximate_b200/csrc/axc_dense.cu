// The exact dense layer: y = act(x kernel + bias + residual), and its gradients.  The products are those of axc_gemm.cu; here are
// the pass over the output's gradient between them, and the entry points.
#include "axc_rows.h"

namespace axc {
namespace {

// ------------------------------------------------------------------------------------------------
// dz = dy act'(kept), column sums on the way.  A block takes 32 groups of V columns (16 bytes) and a share of the rows; a thread has
// the V columns of a group, 2 to 8 rows in flight, packed until they are needed.  Lines that do not start on 16 bytes are read value by
// value, the V values of a thread 32 apart, so that neighbouring lanes still read neighbouring ones.  The sums of the block's 8 rows are
// added in shared memory, those of the blocks by a second kernel, in a fixed order.  Bound by reading dy and kept and writing dz once.
// Nothing is read or written behind the last column (packed groups: S.padded or columns that are whole groups): the operand's tensor maps end
// there, so what its lines have up to a multiple of 8 values does not matter.
// Roundings, for 16-bit operands: dz is rounded once to their type, as the products' operand and as dresidual (the bias's sum takes it before that), and
// `kept`, at which the slope is taken, was rounded to it in the forward pass.  fp32 values in their place would be two bytes a value more for each
// (8192 x 16384: 268 MB, 41 us at the copy rate for every time that they are written or read) and two terms an operand, which is twice the products.
// They make bf16 GELU's results off by 0.0024 in all, where the rounding of the results alone makes 0.0017; a linear layer has none of it.  fp32
// has neither.
// ------------------------------------------------------------------------------------------------
template <int ACT, bool EXACT>
__device__ __forceinline__ float slope_of(float kept)
{
    if (ACT == kActRelu) return kept > 0.0f ? 1.0f : (kept != kept ? kept : 0.0f);
    if (ACT == kActGelu) {
        float bell;
        const float below = normal_below(kept, bell, EXACT);
        return fmaf(kept * bell, 0.39894228f, below);
    }
    const float s = sigmoid(kept, EXACT);
    return s * fmaf(kept, 1.0f - s, 1.0f);
}

template <typename T>
union Group {                                  // 16 bytes of values
    static constexpr int V = 16 / sizeof(T);
    uint4 w;
    T t[V];
    __device__ Group() {}
};

// V columns of a row: neighbours at `at`, or 32 apart, those below `left`.  base, count: all there is (debug flavour).
template <bool VEC, typename T>
__device__ __forceinline__ void load_group(const T *at, long long left, Group<T> &g, const T *base, long long count)
{
    if (VEC) {
        if (AXC_VALUES_OK(at, Group<T>::V, base, count, 401u)) g.w = __ldcs(reinterpret_cast<const uint4 *>(at));
        else g.w = make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
        for (int i = 0; i < Group<T>::V; ++i) g.t[i] = 32 * i < left && AXC_VALUES_OK(at + 32 * i, 1, base, count, 402u) ? at[32 * i] : narrow<T>(0.0f);
    }
}
// The same way out
template <bool VEC, typename T>
__device__ __forceinline__ void store_group(T *at, long long left, const Group<T> &g, const T *base, long long count)
{
    if (VEC) {
        if (AXC_VALUES_OK(at, Group<T>::V, base, count, 403u)) *reinterpret_cast<uint4 *>(at) = g.w;
    } else {
#pragma unroll
        for (int i = 0; i < Group<T>::V; ++i)
            if (32 * i < left && AXC_VALUES_OK(at + 32 * i, 1, base, count, 404u)) at[32 * i] = g.t[i];
    }
}

template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256, 3) slope_kernel(const Slope S, float *part, long long part_values)
{
    after_previous();
    constexpr int V = Group<T>::V, kRows = (ACT == kActNone ? 8 : 4) / (VEC ? 1 : 2), kApart = VEC ? 1 : 32;
    __shared__ float sums[8][32 * V];
    const int group = threadIdx.x & 31, r0 = threadIdx.x >> 5, first_column = VEC ? group * V : group;
    const long long c = (long long)blockIdx.x * 32 * V + first_column, left = S.columns - c;
    const long long begin = S.rows * blockIdx.y / gridDim.y, end = S.rows * (blockIdx.y + 1) / gridDim.y;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    if (left > 0) {
        const T *dy = static_cast<const T *>(S.dy) + (begin + r0) * S.dy_line + c, *kept = static_cast<const T *>(S.kept) + (begin + r0) * S.columns + c;
        for (long long r = begin + r0; r < end; r += 8 * kRows, dy += 8 * kRows * S.dy_line, kept += 8 * kRows * S.columns) {
            Group<T> g[kRows], k[ACT != kActNone ? kRows : 1];
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                const int step = r + 8 * q < end ? 8 * q : 0;      // behind the last row: the first one again, not used
                load_group<VEC>(dy + step * S.dy_line, left, g[q], static_cast<const T *>(S.dy), S.dy_values());
                if constexpr (ACT != kActNone) load_group<VEC>(kept + step * S.columns, left, k[q], static_cast<const T *>(S.kept), S.tensor_values());
            }
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                const long long row = r + 8 * q;
                if (row >= end) continue;
                float d[V];
#pragma unroll
                for (int i = 0; i < V; ++i) d[i] = widen(g[q].t[i]);
                for (int p = 1; p < S.dy_planes; ++p) {
                    Group<T> more;
                    load_group<VEC>(dy + 8 * q * S.dy_line + p * S.plane, left, more, static_cast<const T *>(S.dy), S.dy_values());
#pragma unroll
                    for (int i = 0; i < V; ++i) d[i] += widen(more.t[i]);
                }
                if constexpr (ACT != kActNone) {
#pragma unroll
                    for (int i = 0; i < V; ++i) d[i] *= slope_of<ACT, sizeof(T) == 4>(widen(k[q].t[i]));
                }
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += d[i];
                if (S.same || (S.planes && sizeof(T) == 2)) {
                    Group<T> u;
#pragma unroll
                    for (int i = 0; i < V; ++i) u.t[i] = narrow<T>(d[i]);
                    T *same = static_cast<T *>(S.same), *operand = reinterpret_cast<T *>(S.planes);
                    if (S.same) store_group<VEC>(same + row * S.columns + c, left, u, same, S.tensor_values());
                    if (S.planes && sizeof(T) == 2) store_group<VEC>(operand + row * S.line + c, left, u, operand, S.operand_values());
                }
                if (S.planes && sizeof(T) == 4) {
                    uint16_t *to = S.planes + row * S.line + c;
                    unsigned t[2][3];
                    split_terms(d[0], d[1], t[0]);
                    split_terms(d[2], d[3], t[1]);
#pragma unroll
                    for (int p = 0; p < 3; ++p, to += S.plane) {
                        union { uint2 w; uint16_t h[4]; } u;
                        u.w = make_uint2(t[0][p], t[1][p]);
                        if (VEC) {
                            if (AXC_VALUES_OK(to, 4, S.planes, 3 * S.operand_values(), 405u)) *reinterpret_cast<uint2 *>(to) = u.w;
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (32 * i < left && AXC_VALUES_OK(to + 32 * i, 1, S.planes, 3 * S.operand_values(), 406u)) to[32 * i] = u.h[i];
                        }
                    }
                }
            }
        }
    }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < V; ++i) sums[r0][first_column + kApart * i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V; i += 256) {
        float s = sums[0][i];
#pragma unroll
        for (int k = 1; k < 8; ++k) s += sums[k][i];
        const long long column = (long long)blockIdx.x * 32 * V + i;
        const long long at = (long long)blockIdx.y * S.columns + column;
        if (column < S.columns && AXC_GLOBAL_OK(at, part_values, 407u)) part[at] = s;
    }
}

__global__ void __launch_bounds__(256) slope_sums_kernel(const float *part, long long part_values, long long columns, int shares, float scale,
                                                         const float *scale_dev, void *sums, int type)
{
    after_previous();
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    if (c >= columns) return;
    float s = 0.0f;
    for (int k = 0; k < shares; ++k)
        if (AXC_GLOBAL_OK(k * columns + c, part_values, 408u)) s += part[k * columns + c];
    store_from_float(sums, c, type, s * scale * (scale_dev ? *scale_dev : 1.0f));
}

template <typename T, bool VEC>
int launch_slope(const Slope &s, float *part, long long part_values, int shares, Queue &q)
{
    const dim3 grid(unsigned((s.columns + 32 * Group<T>::V - 1) / (32 * Group<T>::V)), unsigned(shares));
    return launch(q, !s.kept ? slope_kernel<T, kActNone, VEC> : s.activation == kActRelu ? slope_kernel<T, kActRelu, VEC>
                     : s.activation == kActGelu ? slope_kernel<T, kActGelu, VEC> : slope_kernel<T, kActSilu, VEC>, grid, 256, 0, 1, s, part, part_values);
}

}  // namespace

AXC_DEFINE_BOUNDS_READER(bounds_record_dense)

int slope(const Slope &s, void *scratch, size_t room, Queue &q)
{
    if (s.columns == 0 || (s.rows == 0 && !s.sums)) return AXC_OK;
    if (s.sums && room < slope_scratch(s.rows, s.columns)) return AXC_INTERNAL;
    const int shares = column_shares(s.rows, s.columns);
    float *part = s.sums ? static_cast<float *>(scratch) : nullptr;
    const long long values = (long long)(room / sizeof(float));
    // whole groups of 16 bytes, in every line of every tensor
    const uintptr_t all = reinterpret_cast<uintptr_t>(s.dy) | reinterpret_cast<uintptr_t>(s.kept) | reinterpret_cast<uintptr_t>(s.same);
    const long long size = s.type == kFloat32 ? 4 : 2;
    const bool vec = (all & 15u) == 0 && s.dy_line * size % 16 == 0 && (s.padded || s.columns * size % 16 == 0) && s.plane * size % 16 == 0;
    int rc;
    if (s.type == kFloat32) rc = vec ? launch_slope<float, true>(s, part, values, shares, q) : launch_slope<float, false>(s, part, values, shares, q);
    else if (s.type == kBfloat16) rc = vec ? launch_slope<__nv_bfloat16, true>(s, part, values, shares, q) : launch_slope<__nv_bfloat16, false>(s, part, values, shares, q);
    else rc = vec ? launch_slope<__half, true>(s, part, values, shares, q) : launch_slope<__half, false>(s, part, values, shares, q);
    if (rc || !s.sums) return rc;
    return launch(q, slope_sums_kernel, dim3(unsigned((s.columns + 255) / 256)), 256, 0, 1, part, values, s.columns, shares, s.scale, s.scale_dev, s.sums, s.sums_type);
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
struct Room {
    size_t x, kernel, dz, part, scratch, total;
};
size_t up(size_t n) { return (n + 255) / 256 * 256; }
size_t largest(size_t a, size_t b) { return a > b ? a : b; }

// Addresses that no tensor has stand for unknown ones: sized for a copy of every operand.
const void *const kUnknown = reinterpret_cast<const void *>(uintptr_t(2));

Room room_of(const axc_dense_desc &d, bool backward, const void *x, const void *kernel, const DeviceInfo &di)
{
    const int planes = d.type == kFloat32 ? 3 : 1;
    Room p;
    if (!backward && few_rows(x_of(d, x), kernel_of(d, kernel))) {
        p.x = p.kernel = p.dz = p.part = p.scratch = 256;
        p.total = p.scratch + up(few_rows_scratch(x_of(d, x), kernel_of(d, kernel), di));
        return p;
    }
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

// A call without outputs: no more than its status.  Without a workspace there is nothing to do, not even a device to look for.
int nothing(void *workspace, size_t bytes, int device, void *stream)
{
    if (!workspace || bytes < sizeof(unsigned)) return AXC_OK;
    DeviceInfo di;
    int prev = 0;
    const int rc = enter(device, &di, &prev);
    if (rc) return rc;
    const cudaError_t e = cudaMemsetAsync(workspace, 0, sizeof(unsigned), cudaStream_t(stream));
    return leave(e == cudaSuccess ? AXC_OK : cuda_failed(e), device, prev);
}

int forward(const axc_dense_desc &d, const void *x, const void *kernel, const void *bias, const void *residual, void *y, void *pre, char *ws,
            const DeviceInfo &di, Queue &q)
{
    const Room parts = room_of(d, false, x, kernel, di);
    Gemm g = {};
    g.m = d.rows;
    g.n = d.units;
    g.k = d.inputs;
    g.planes = d.type == kFloat32 ? 3 : 1;
    g.bf16 = d.type != kFloat16;
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
    if (few_rows(x_of(d, x), kernel_of(d, kernel)))
        return few_rows_product(x_of(d, x), kernel_of(d, kernel), g.fin, ws + parts.scratch, reinterpret_cast<unsigned *>(ws), di, q);
    if (d.inputs > 0) {
        const int rc = make_operands(x_of(d, x), ws + parts.x, &g.a, kernel_of(d, kernel), ws + parts.kernel, &g.b, di, q);
        if (rc) return rc;
    }
    return gemm(g, ws + parts.scratch, reinterpret_cast<unsigned *>(ws), true, di, q);
}

int backward(const axc_dense_desc &d, const void *dy, const void *x, const void *kernel, const void *kept, void *dx, void *dkernel, void *dbias,
             void *dresidual, char *ws, const DeviceInfo &di, Queue &q)
{
    const Room parts = room_of(d, true, x, kernel, di);
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
    if (s.same || s.planes || s.sums) rc = slope(s, ws + parts.part, parts.scratch - parts.part, q);
    if (rc) return rc;
    bool first = true;
    Operand ox = {}, ok = {};
    const Matrix none = {};
    rc = make_operands(dkernel ? x_of(d, x) : none, ws + parts.x, &ox, dx ? kernel_of(d, kernel) : none, ws + parts.kernel, &ok, di, q);
    if (rc) return rc;
    if (dx) {
        Gemm g = {};
        g.m = d.rows;
        g.n = d.inputs;
        g.k = d.units;
        g.planes = planes;
        g.bf16 = d.type != kFloat16;
        g.a = dz;
        g.b = transposed(ok);
        g.fin.alpha = 1.0f;
        g.fin.out = dx;
        g.fin.out_type = d.type;
        g.fin.out_line = d.inputs;
        rc = gemm(g, ws + parts.scratch, status, first, di, q);
        if (rc) return rc;
        first = false;
    }
    if (dkernel) {
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
            g.b = transposed(ox);
        } else {
            g.m = d.inputs;
            g.n = d.units;
            g.a = transposed(ox);
            g.b = transposed(dz);
        }
        g.fin.out_line = g.n;
        rc = gemm(g, ws + parts.scratch, status, first, di, q);
        if (rc) return rc;
        first = false;
    }
    if (first) AXC_CUDA(cudaMemsetAsync(status, 0, sizeof(unsigned), q.stream));
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
    if (forward) *forward = room_of(*desc, false, x, kernel, di).total;
    if (backward) *backward = room_of(*desc, true, x, kernel, di).total;
    return AXC_OK;
}

extern "C" int axc_dense_forward(const axc_dense_desc *desc, const void *x, const void *kernel, const void *bias, const void *residual, void *y, void *pre,
                                 void *workspace, size_t workspace_bytes, int device, void *stream)
{
    using namespace axc;
    int rc = check_desc(desc);
    if (rc) return rc;
    const axc_dense_desc &d = *desc;
    if (d.rows == 0 || d.units == 0) return nothing(workspace, workspace_bytes, device, stream);
    if (!y || (d.inputs > 0 && (!x || !kernel))) return AXC_INVALID_ARGUMENT;
    if (!aligned_to(type_size(d.type), x, kernel, residual, y, pre) || !aligned_to(type_size(d.bias_type), bias)) return AXC_INVALID_ARGUMENT;
    DeviceInfo di;
    rc = device_info(device, &di);
    if (rc) return rc;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < room_of(d, false, x, kernel, di).total) return AXC_INTERNAL;
    int prev = 0;
    rc = enter(device, &di, &prev);
    if (rc) return rc;
    Queue q = {cudaStream_t(stream)};
    return leave(forward(d, x, kernel, bias, residual, y, pre, static_cast<char *>(workspace), di, q), device, prev);
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
    if (!aligned_to(type_size(d.type), dy, x, kernel, kept, dx, dkernel, dresidual) || !aligned_to(type_size(d.bias_type), dbias)) return AXC_INVALID_ARGUMENT;
    if (d.rows == 0 && d.units == 0) return nothing(workspace, workspace_bytes, device, stream);
    DeviceInfo di;
    rc = device_info(device, &di);
    if (rc) return rc;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < room_of(d, true, x, kernel, di).total) return AXC_INTERNAL;
    int prev = 0;
    rc = enter(device, &di, &prev);
    if (rc) return rc;
    Queue q = {cudaStream_t(stream)};
    return leave(backward(d, dy, x, kernel, kept, dx, dkernel, dbias, dresidual, static_cast<char *>(workspace), di, q), device, prev);
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
