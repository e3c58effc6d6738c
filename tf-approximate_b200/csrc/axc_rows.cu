// The dense layer's forward product for a few rows, as a model answers them one by one: bound by reading the kernel once, in the type
// and order that it has.  No tensor cores: up to 8 products for every value read stay below what the fp32 pipes do meanwhile.
//   inputs contiguous  a warp has 1 or 4 units and walks along their inputs, 16 bytes a lane; the rows of x come through L1
//   units contiguous   (fp32) a lane has 16 bytes of neighbouring units, the warps and the blocks of a column share the inputs, and their
//                      sums are added in a fixed order (shared memory, then the second kernel of split products)
// 16-bit kernels with more than two rows, or with units contiguous, are as quick or quicker on the tensor cores.  us for 4096 inputs x
// 16384 units, and 2048 x 1000:
//   bf16, inputs contiguous   1 row 24.1, 2 rows 34, 4 rows 43 (tensor cores 34 to 37; reading it once: 20.5); 4.1, 4.6, 6.7 (9.3)
//   fp32, inputs contiguous   44 to 112 for 1 to 8 rows (tensor cores 215; 41.0); 5.1 to 10.9 (17.7)
//   fp32, units contiguous    67 to 112 (226; 41.0); 10.1 to 11.8 (18.1)
#include "axc_rows.h"

namespace axc {
namespace {

template <typename T, int N> union Values {
    uint4 w[(N * sizeof(T) + 15) / 16];
    T t[N];
    __device__ Values() {}
};

// R rows of x (those behind the last are the last one again), U units per warp; VEC: everything starts on 16 bytes
template <typename T, int R, int U, bool VEC>
__global__ void __launch_bounds__(256) rows_dot_kernel(const RowsArgs A)
{
    after_previous();
    if (blockIdx.x == 0 && threadIdx.x == 0) *A.status = 0u;
    constexpr int V = VEC ? 16 / int(sizeof(T)) : 1;
    const int lane = threadIdx.x & 31;
    const long long u0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * U;
    if (u0 >= A.units) return;
    const T *x = static_cast<const T *>(A.x), *w[U];
    [[maybe_unused]] const long long x_values = (A.rows - 1) * A.x_line + A.inputs, kernel_values = (A.units - 1) * A.kernel_line + A.inputs;
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = static_cast<const T *>(A.kernel) + (u0 + u < A.units ? u0 + u : A.units - 1) * A.kernel_line;
    float sum[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) sum[u][r] = 0.0f;
    constexpr int kBatch = U >= 4 ? 2 : 4;                      // loads of a unit in flight
    for (long long k0 = (long long)lane * V; k0 < A.inputs; k0 += 32 * V * kBatch) {
        Values<T, V> b[kBatch][U];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long k = k0 + 32 * V * i;
                if (k < A.inputs) {
                    if (!AXC_VALUES_OK(w[u] + k, V, static_cast<const T *>(A.kernel), kernel_values, 441u)) continue;
                    if constexpr (VEC) b[i][u].w[0] = __ldcs(reinterpret_cast<const uint4 *>(w[u] + k));
                    else b[i][u].t[0] = w[u][k];
                }
            }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const long long k = k0 + 32 * V * i;
            if (k >= A.inputs) break;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                Values<T, V> a;
                const T *from = x + (r < A.rows ? r : A.rows - 1) * A.x_line + k;
                if (!AXC_VALUES_OK(from, V, x, x_values, 442u)) continue;
                if constexpr (VEC) a.w[0] = *reinterpret_cast<const uint4 *>(from);
                else a.t[0] = *from;
#pragma unroll
                for (int j = 0; j < V; ++j)
#pragma unroll
                    for (int u = 0; u < U; ++u) sum[u][r] = fmaf(widen(a.t[j]), widen(b[i][u].t[j]), sum[u][r]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum[u][r] += __shfl_xor_sync(0xffffffffu, sum[u][r], o);
            if (lane == u * R + r && r < A.rows && u0 + u < A.units) finish_value(A.fin, sum[u][r], r, u0 + u);
        }
}

// Blocks: x over the columns, y over shares of the inputs.  A warp takes every eighth of its block's inputs, 32 of x's values by lane.
template <int R, bool VEC>
__global__ void __launch_bounds__(256) rows_sum_kernel(const RowsArgs A, float *part, long long part_line, long long part_stride)
{
    after_previous();
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *A.status = 0u;
    typedef float T;
    constexpr int V = 4;
    __shared__ float sums[8][32 * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long c = ((long long)blockIdx.x * 32 + lane) * V;
    const long long begin = A.inputs * blockIdx.y / gridDim.y, end = A.inputs * (blockIdx.y + 1) / gridDim.y;
    const T *x = static_cast<const T *>(A.x), *kernel = static_cast<const T *>(A.kernel);
    [[maybe_unused]] const long long x_values = (A.rows - 1) * A.x_line + A.inputs, kernel_values = (A.inputs - 1) * A.kernel_line + A.units;
    float sum[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) sum[r][j] = 0.0f;
    for (long long k0 = begin + warp * 32; k0 < end; k0 += 256) {
        float mine[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const long long at = (r < A.rows ? r : A.rows - 1) * A.x_line + k0 + lane;
            mine[r] = k0 + lane < end && AXC_GLOBAL_OK(at, x_values, 443u) ? widen(x[at]) : 0.0f;
        }
#pragma unroll
        for (int i0 = 0; i0 < 32; i0 += 8) {
            Values<T, V> b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const long long k = k0 + i0 + i;
#pragma unroll
                for (int j = 0; j < V; ++j) b[i].t[j] = narrow<T>(0.0f);
                if (k < end) {
                    const T *from = kernel + k * A.kernel_line + c;
                    if (VEC && c + V <= A.units && AXC_VALUES_OK(from, V, kernel, kernel_values, 444u)) b[i].w[0] = __ldcs(reinterpret_cast<const uint4 *>(from));
                    else {
#pragma unroll
                        for (int j = 0; j < V; ++j)
                            if (c + j < A.units && AXC_VALUES_OK(from + j, 1, kernel, kernel_values, 445u)) b[i].t[j] = from[j];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float a = __shfl_sync(0xffffffffu, mine[r], i0 + i);
#pragma unroll
                    for (int j = 0; j < V; ++j) sum[r][j] = fmaf(a, k0 + i0 + i < end ? widen(b[i].t[j]) : 0.0f, sum[r][j]);
                }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= A.rows) break;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) sums[warp][lane * V + j] = sum[r][j];
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * V; i += 256) {
            float s = sums[0][i];
#pragma unroll
            for (int k = 1; k < 8; ++k) s += sums[k][i];
            const long long column = (long long)blockIdx.x * 32 * V + i;
            if (column < A.units) {
                if (gridDim.y > 1) {
                    const long long at = blockIdx.y * part_stride + r * part_line + column;
                    if (AXC_GLOBAL_OK(at, gridDim.y * part_stride, 446u)) part[at] = s;
                } else finish_value(A.fin, s, r, column);
            }
        }
    }
}

template <typename T, int R>
int launch_dot(const RowsArgs &A, bool vec, const DeviceInfo &di, Queue &q)
{
    // one unit a warp until that makes eight warps for every SM four times over
    const bool four = R <= 4 && A.units >= (long long)di.sm_count * 8 * 4 * 2;
    const unsigned grid = unsigned((A.units + (four ? 31 : 7)) / (four ? 32 : 8));
    if constexpr (R <= 4) {
        if (four) return launch(q, vec ? rows_dot_kernel<T, R, 4, true> : rows_dot_kernel<T, R, 4, false>, dim3(grid), 256, 0, 1, A);
    }
    return launch(q, vec ? rows_dot_kernel<T, R, 1, true> : rows_dot_kernel<T, R, 1, false>, dim3(grid), 256, 0, 1, A);
}

template <typename T>
int launch_dots(const RowsArgs &A, bool vec, const DeviceInfo &di, Queue &q)
{
    if (A.rows == 1) return launch_dot<T, 1>(A, vec, di, q);
    if (A.rows == 2) return launch_dot<T, 2>(A, vec, di, q);
    if constexpr (sizeof(T) == 4) return A.rows <= 4 ? launch_dot<T, 4>(A, vec, di, q) : launch_dot<T, 8>(A, vec, di, q);
    return AXC_INTERNAL;
}

constexpr int kColumns = 128;                  // of a block of rows_sum_kernel

int launch_sums(const RowsArgs &A, bool vec, int shares, float *scratch, const DeviceInfo &di, Queue &q)
{
    const dim3 grid(unsigned((A.units + kColumns - 1) / kColumns), unsigned(shares));
    const long long line = (A.units + 3) / 4 * 4, stride = line * A.rows;
    int rc;
    if (A.rows == 1) rc = launch(q, vec ? rows_sum_kernel<1, true> : rows_sum_kernel<1, false>, grid, 256, 0, 1, A, scratch, line, stride);
    else if (A.rows == 2) rc = launch(q, vec ? rows_sum_kernel<2, true> : rows_sum_kernel<2, false>, grid, 256, 0, 1, A, scratch, line, stride);
    else if (A.rows <= 4) rc = launch(q, vec ? rows_sum_kernel<4, true> : rows_sum_kernel<4, false>, grid, 256, 0, 1, A, scratch, line, stride);
    else rc = launch(q, vec ? rows_sum_kernel<8, true> : rows_sum_kernel<8, false>, grid, 256, 0, 1, A, scratch, line, stride);
    if (rc || shares == 1) return rc;
    const Parts parts = {scratch, line, stride, shares};
    return finish_parts(parts, A.rows, A.units, A.fin, di, q);
}

bool inputs_contiguous(const Matrix &kernel) { return kernel.column_stride == 1 || kernel.columns == 1; }

int shares_of(const Matrix &x, const Matrix &kernel, const DeviceInfo &di)
{
    if (inputs_contiguous(kernel)) return 1;
    // enough blocks for every SM four times, of at least 256 inputs
    const long long across = (kernel.rows + kColumns - 1) / kColumns, want = ((long long)di.sm_count * 4 + across - 1) / across;
    const long long most = x.columns / 256 > 0 ? x.columns / 256 : 1;
    const long long shares = want < most ? want : most;
    return int(shares < 32 ? shares : 32);
}

}  // namespace

AXC_DEFINE_BOUNDS_READER(bounds_record_rows)

bool few_rows(const Matrix &x, const Matrix &kernel)
{
    if (x.rows == 0 || x.columns == 0 || (x.column_stride != 1 && x.columns > 1)) return false;
    if (x.type != kFloat32) return x.rows <= 2 && inputs_contiguous(kernel);
    return x.rows <= 8 && (inputs_contiguous(kernel) || kernel.row_stride == 1 || kernel.rows == 1);
}

size_t few_rows_scratch(const Matrix &x, const Matrix &kernel, const DeviceInfo &di)
{
    const int shares = shares_of(x, kernel, di);
    return shares > 1 ? size_t(shares) * size_t(x.rows) * size_t((kernel.rows + 3) / 4 * 4) * 4 : 0;
}

int few_rows_product(const Matrix &x, const Matrix &kernel, const Finish &f, void *scratch, unsigned *status, const DeviceInfo &di, Queue &q)
{
    const bool dot = inputs_contiguous(kernel);
    RowsArgs A = {x.data, kernel.data, int(x.rows), x.columns, kernel.rows, x.row_stride, dot ? kernel.row_stride : kernel.column_stride,
                  sized(f, x.rows, kernel.rows), status};
    const long long size = (long long)type_size(x.type);
    const uintptr_t all = reinterpret_cast<uintptr_t>(kernel.data) | uintptr_t(A.kernel_line * size) | (dot ? reinterpret_cast<uintptr_t>(x.data) | uintptr_t(A.x_line * size) : 0);
    const bool vec = all % 16 == 0 && (!dot || x.columns * size % 16 == 0);
    if (!dot) return launch_sums(A, vec, shares_of(x, kernel, di), static_cast<float *>(scratch), di, q);
    if (x.type == kFloat32) return launch_dots<float>(A, vec, di, q);
    return x.type == kBfloat16 ? launch_dots<__nv_bfloat16>(A, vec, di, q) : launch_dots<__half>(A, vec, di, q);
}

}  // namespace axc
