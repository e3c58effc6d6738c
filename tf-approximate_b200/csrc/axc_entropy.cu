// Softmax cross entropy of a dense classifier with its gradients:
//   l = x kernel + bias,  loss_t = log sum_v exp(l_tv) - l_t,label,  dl = w (softmax(l) - onehot),  dx = dl kernel^T,  dkernel = x^T dl
// The logits never reach memory.  One pass of matrix tiles over the classes (axc_gemm.cu) leaves, for every row and segment of 64
// classes, the largest logit and the sum of exponentials relative to it.  A pass over the rows joins them to the row's
// largest logit and sum (never to their one number log sum_v exp(l_tv): it is rounded to a part of the logits' size, which may be all
// that there is of a small loss or gradient).  Then one of two forms gives the gradient of the logits, 16-bit values that are rounded once:
//   kept     the exponentials, relative to their segment's largest logit, were kept in scratch, and the pass over the rows turns them
//            into the gradient: 6 T D V operations, 2 bytes of scratch per logit (bf16; 6 for fp16, 10 for fp32)
//   pieces   the logits of a piece of the classes are computed again, with the row's largest logit and sum at hand, and become the gradient
//            in the tile's last step: 8 T D V operations, scratch for one piece
// Where the logits are few (2^20, of at most 8192 classes) their product is split over CTAs like any other, and the pass over the rows
// adds the parts up in shared memory and does all the rest: 128 CTAs instead of 32 for 256 x 2048 x 1000, 14.2 to 8.3 us.
// Roundings, for 16-bit operands; fp32 ones have none (fp32 exponentials, the gradient as three bf16 terms):
//   exponentials kept for bf16 are fp16: 2 bytes a logit written and read instead of 4 (the pass over 2 GiB of them is 721 us of 11 to 13 ms for 8192 x
//                  2048 x 131072).  To 2^-12 of themselves down to 2^-14 of their segment's largest, to 2^-25 of that one below: a class below 2^-25 of
//                  the largest of its segment of 64 gets no gradient, where its segment's largest one is rounded by 2^-9 of itself.  Kept for fp16: fp32
//   gradient       dl is rounded once to bf16 (2^-9), or to fp16 (2^-12) times 2^14, so that its smallest normal value is 3.7e-9 (the products' factor takes
//                  the 2^14 out), before both products and the bias's sum: the matrix units multiply 16-bit values at full rate, a second term would
//                  double the products.  dx and dkernel are then off by 0.0019 instead of the 0.0017 that their own rounding to bf16 makes
//   __expf         16-bit operands' exponentials are good to 2^-19 for |x| up to 20, which the two above hide
#include "axc_gemm.h"

namespace axc {
namespace {

constexpr int kSegment = 64;
constexpr float kHalfScale = 16384.0f;

constexpr int kFewClasses = 8192;              // their logits fit into a block's shared memory
constexpr long long kFewLogits = 1ll << 20;

struct RowArgs {
    long long rows, classes;
    const long long *labels;
    long long ignore;
    const float2 *stats;
    int segments;
    float *label_logit;
    float2 *softmax;                           // see EntropyArgs
    float *row_scale, *row_loss;
    float stored;                              // scale of the stored gradient
    // kept form
    void *keep;
    long long line;
    uint16_t *gradient;                        // planes of [rows][line]; may be `keep`
    long long plane;
    // few logits
    Parts parts;
    const void *bias;
    int bias_type, planes, bf16;
    // the call's result
    unsigned *done;                            // rows that are done
    int mean;
    float grad_factor;
    float *loss, *alpha;
};

__device__ __forceinline__ float block_max(float v, float *shared)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = shared[0];
    for (int i = 1; i < int(blockDim.x >> 5); ++i) r = fmaxf(r, shared[i]);
    return r;
}
__device__ __forceinline__ float block_sum(float v, float *shared)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = 0.0f;
    for (int i = 0; i < int(blockDim.x >> 5); ++i) r += shared[i];
    return r;
}

// The last block to come here adds the rows' losses up, in an order that does not depend on which block that is, and leaves the loss
// and the factor of the gradients.  Compensated: a sum may run over a million rows.
__device__ __forceinline__ void add_losses(const RowArgs &A, float *shared)
{
    __shared__ bool last;
    if (threadIdx.x == 0) {
        __threadfence();                       // this thread wrote the row's loss
        last = atomicAdd(A.done, 1u) == gridDim.x - 1;
        __threadfence();
    }
    __syncthreads();
    if (!last) return;
    float sum = 0.0f, count = 0.0f, low = 0.0f;
    for (long long i = threadIdx.x; i < A.rows; i += 256) {
        if (A.labels[i] == A.ignore) continue;
        const float y = __ldcg(A.row_loss + i) - low, t = sum + y;
        low = isfinite(t) ? (t - sum) - y : 0.0f;
        sum = t;
        count += 1.0f;
    }
    sum = block_sum(sum, shared);
    count = block_sum(count, shared);
    if (threadIdx.x == 0) {
        const float share = A.mean ? (count > 0.0f ? 1.0f / count : 0.0f) : 1.0f;
        *A.loss = sum * share;
        *A.alpha = A.grad_factor * share;
    }
}

// One block per row: its largest logit, sum and loss; FORM 0: no more, 1: fp16 exponentials in place to bf16 gradients, 2: fp32 to fp16,
// 3: fp32 to three bf16 planes.  Bound by reading and writing the exponentials once.
template <int FORM>
__global__ void __launch_bounds__(256) row_kernel(const RowArgs A)
{
    after_previous();
    __shared__ float shared[8];
    const long long row = blockIdx.x;
    const float2 *stats = A.stats + row * A.segments;
    float top = -INFINITY;
    for (int i = threadIdx.x; i < A.segments; i += 256)
        if (AXC_GLOBAL_OK(row * A.segments + i, A.rows * A.segments, 461u)) top = fmaxf(top, stats[i].x);
    top = block_max(top, shared);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int i = threadIdx.x; i < A.segments; i += 256) {
        const float2 s = stats[i];
        sum += s.x == -INFINITY ? s.y : s.y * exponential(s.x - base, FORM == 3 || (FORM == 0 && A.planes == 3));
    }
    sum = block_sum(sum, shared);
    const long long label = A.labels[row];
    const bool counts = label != A.ignore, known = label >= 0 && label < A.classes;
    // a label outside the classes shows in the loss and in every gradient
    const float scale = !counts ? 0.0f : known ? A.stored : NAN;
    if (threadIdx.x == 0) {
        // the largest logit comes off the label's first: the logits' size does not decide what is left of a small loss
        A.row_loss[row] = !counts ? 0.0f : known ? logf(sum) - (A.label_logit[row] - base) : NAN;
        if (FORM == 0 && A.softmax) {
            A.softmax[row] = make_float2(base, 1.0f / sum);
            A.row_scale[row] = scale;
        }
    }
    const int groups = FORM == 0 ? 0 : int(A.line / 8);
    for (int i = threadIdx.x; i < groups; i += 256) {
        const int c = i * 8;
        if (!AXC_GLOBAL_OK(c / kSegment, A.segments, 462u) || !AXC_GLOBAL_OK(row * A.line + c + 7, A.rows * A.line, 463u)) continue;
        const float first = stats[c / kSegment].x;
        float factor = scale / sum;
        if (first != -INFINITY) factor *= exponential(first - base, FORM == 3);
        if (!counts) factor = 0.0f;
        float v[8];
        if (FORM == 1) {
            const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(A.keep) + row * A.line + c);
            const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 t = __half22float2(reinterpret_cast<const __half2 &>(u[j]));
                v[2 * j] = t.x;
                v[2 * j + 1] = t.y;
            }
        } else {
            const float4 *from = reinterpret_cast<const float4 *>(static_cast<const float *>(A.keep) + row * A.line + c);
            const float4 w0 = from[0], w1 = from[1];
            v[0] = w0.x; v[1] = w0.y; v[2] = w0.z; v[3] = w0.w;
            v[4] = w1.x; v[5] = w1.y; v[6] = w1.z; v[7] = w1.w;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = counts ? v[j] * factor : 0.0f;               // a row without a label stays out, whatever its logits are
            if (c + j == label && counts) v[j] -= scale;
        }
        uint16_t *to = A.gradient + row * A.line + c;
        for (int p = 0; p < (FORM == 3 ? 3 : 1); ++p, to += A.plane) {
            unsigned u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] = pack2(v[2 * j], v[2 * j + 1], FORM != 2);
                if (FORM == 3) {
                    const float2 t = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162 &>(u[j]));
                    v[2 * j] -= t.x;
                    v[2 * j + 1] -= t.y;
                }
            }
            if (AXC_VALUES_OK(to, 8, A.gradient, A.rows * A.line + (FORM == 3 ? 2 : 0) * A.plane, 464u)) *reinterpret_cast<uint4 *>(to) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
    add_losses(A, shared);
}

// The same for few logits, from the parts of their sums.
template <bool EXACT>
__global__ void __launch_bounds__(256) few_kernel(const RowArgs A)
{
    after_previous();
    __shared__ float logits[kFewClasses], shared[8];
    const long long row = blockIdx.x;
    const int classes = int(A.classes);
    float top = -INFINITY;
    bool nan = false;
    for (int c = threadIdx.x; c < classes; c += 256) {
        const float *at = A.parts.data + row * A.parts.line + c;
        if (!AXC_GLOBAL_OK(c, kFewClasses, 465u) || !AXC_VALUES_OK(at + (A.parts.count - 1) * A.parts.stride, 1, A.parts.data, A.parts.count * A.parts.stride, 466u)) continue;
        float l = at[0];
        for (int i = 1; i < A.parts.count; ++i) l += at[i * A.parts.stride];
        if (A.bias) l += load_as_float(A.bias, c, A.bias_type);
        logits[c] = l;
        nan |= l != l;
        top = fmaxf(top, l);
    }
    top = block_max(top, shared);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = nan ? NAN : 0.0f;
    for (int c = threadIdx.x; c < classes; c += 256) sum += exponential(logits[c] - base, EXACT);
    sum = block_sum(sum, shared);
    const long long label = A.labels[row];
    const bool counts = label != A.ignore, known = label >= 0 && label < A.classes;
    const float scale = !counts ? 0.0f : known ? A.stored : NAN, factor = scale / sum;
    if (threadIdx.x == 0) A.row_loss[row] = !counts ? 0.0f : known ? logf(sum) - (logits[label] - base) : NAN;
    for (int c = A.gradient ? int(threadIdx.x) * 8 : int(A.line); c < A.line; c += 2048) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = counts && c + j < classes ? exponential(logits[c + j < classes ? c + j : 0] - base, EXACT) * factor : 0.0f;
            if (c + j == label && counts) v[j] -= scale;
        }
        uint16_t *to = A.gradient + row * A.line + c;
        for (int p = 0; p < A.planes; ++p, to += A.plane) {
            unsigned u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] = pack2(v[2 * j], v[2 * j + 1], A.bf16);
                if (A.planes == 3) {
                    const float2 t = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162 &>(u[j]));
                    v[2 * j] -= t.x;
                    v[2 * j + 1] -= t.y;
                }
            }
            if (AXC_VALUES_OK(to, 8, A.gradient, A.rows * A.line + (A.planes - 1) * A.plane, 467u)) *reinterpret_cast<uint4 *>(to) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
    add_losses(A, shared);
}

// Gradients times the factor that comes from above in a backward pass, a fp32 number in device memory, each value rounded once.  Up to kScaleParts
// tensors a launch; a block has kScaleBytes of one of them.  Bound by reading and writing them once (2^28 bf16 values: 160 us, 6.7
// TB/s; torch's product with a number on the device 560, with a rounded factor).
constexpr int kScaleParts = 4, kScaleBytes = 256 * 16 * 4;
struct ScaleArgs {
    axc_scale_tensor part[kScaleParts];
    unsigned first[kScaleParts];               // blocks
    int parts;
    const float *factor;
};
template <typename T>
__device__ __forceinline__ void scale_block(const axc_scale_tensor &t, long long begin, float factor)
{
    constexpr int V = 16 / int(sizeof(T)), kValues = kScaleBytes / int(sizeof(T));
    const T *x = static_cast<const T *>(t.x) + begin;
    T *out = static_cast<T *>(t.out) + begin;
    const long long left = t.count - begin;
    const bool vec = ((reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.out)) & 15u) == 0;
    union Group { uint4 w; T t[V]; __device__ Group() {} };
    if (vec && left >= kValues) {
        Group g[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = (i * 256 + int(threadIdx.x)) * V;
            if (AXC_GLOBAL_OK(at + V - 1, left, 468u)) g[i].w = __ldcs(reinterpret_cast<const uint4 *>(x + at));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = (i * 256 + int(threadIdx.x)) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) g[i].t[j] = narrow<T>(widen(g[i].t[j]) * factor);
            if (AXC_GLOBAL_OK(at + V - 1, left, 469u)) __stcs(reinterpret_cast<uint4 *>(out + at), g[i].w);
        }
    } else {
        for (int i = threadIdx.x; i < kValues && i < left; i += 256) out[i] = narrow<T>(widen(x[i]) * factor);
    }
}
__global__ void __launch_bounds__(256) scale_kernel(const ScaleArgs A)
{
    int p = 0;
    while (p + 1 < A.parts && blockIdx.x >= A.first[p + 1]) ++p;
    const axc_scale_tensor &t = A.part[p];
    const float factor = *A.factor;
    const long long block = blockIdx.x - A.first[p];
    if (t.type == kFloat32) scale_block<float>(t, block * (kScaleBytes / 4), factor);
    else if (t.type == kBfloat16) scale_block<__nv_bfloat16>(t, block * (kScaleBytes / 2), factor);
    else scale_block<__half>(t, block * (kScaleBytes / 2), factor);
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }
size_t largest(size_t a, size_t b) { return a > b ? a : b; }

const void *const kUnknown = reinterpret_cast<const void *>(uintptr_t(2));

Matrix x_of(const axc_entropy_desc &d, const void *x) { return {x, d.rows, d.inputs, d.x_row_stride, d.x_column_stride, d.type}; }
Matrix kernel_of(const axc_entropy_desc &d, const void *k) { return {k, d.classes, d.inputs, d.kernel_column_stride, d.kernel_row_stride, d.type}; }

// How a call runs: the exponentials kept, or so many classes at a time; and where the parts of its workspace lie.
struct Layout {
    bool gradients, kept, few;
    long long piece, line;                     // classes at a time, and values from row to row of what is stored for them
    int segments;
    size_t x, kernel, stats, rows, keep, gradient, dx, part, scratch, total;
};

Layout layout_of(const axc_entropy_desc &d, bool gradients, const void *x, const void *kernel, const DeviceInfo &di)
{
    Layout l = {};
    const int planes = d.type == kFloat32 ? 3 : 1;
    const long long whole = (d.classes + kSegment - 1) / kSegment * kSegment;
    const size_t keep_bytes = d.type == kBfloat16 ? 2 : 4, gradient_bytes = d.type == kFloat32 ? 6 : d.type == kFloat16 ? 2 : 0;
    l.gradients = gradients;
    l.segments = int(whole / kSegment);
    const size_t limit = d.scratch_limit > 0 ? size_t(d.scratch_limit) : size_t(AXC_ENTROPY_SCRATCH);
    // a limit below what few logits take asks for pieces
    l.few = d.classes <= kFewClasses && d.rows * d.classes <= kFewLogits && (d.scratch_limit == 0 || d.scratch_limit >= kFewLogits * 64);
    l.kept = gradients && !l.few && size_t(d.rows) * size_t(whole) * (keep_bytes + gradient_bytes) <= limit;
    l.piece = whole;
    if (gradients && !l.kept && !l.few) l.piece = classes_of_piece(d.rows, whole, planes, limit);
    l.line = l.piece < whole ? l.piece : whole;
    l.x = 256;
    l.kernel = l.x + up(operand_bytes(x_of(d, x)));
    l.stats = l.kernel + up(operand_bytes(kernel_of(d, kernel)));
    l.rows = l.stats + up(size_t(d.rows) * l.segments * 8);
    l.keep = l.rows + 5 * up(size_t(d.rows) * 4) + 256;
    l.gradient = l.keep + (l.kept ? up(size_t(d.rows) * l.line * keep_bytes) : 0);
    if (gradients && l.kept && d.type == kBfloat16) l.gradient = l.keep;
    l.dx = l.keep;
    if (gradients) l.dx = (l.kept && d.type == kBfloat16 ? l.keep + up(size_t(d.rows) * l.line * 2) : l.gradient + up(size_t(d.rows) * l.line * 2 * planes));
    const bool pieces = gradients && !l.kept && !l.few;
    l.part = l.dx + (pieces ? up(size_t(d.rows) * size_t((d.inputs + 3) / 4 * 4) * 4) : 0);
    l.scratch = l.part + (gradients ? up(slope_scratch_of_pieces(d.rows, d.classes, pieces ? l.piece : d.classes)) : 0);
    size_t most = 0;
    if (gradients) {
        const PieceSizes sizes = piece_sizes(d.classes, pieces ? l.piece : d.classes);
        for (const long long n : sizes.n) {
            most = largest(most, gemm_scratch(d.rows, d.inputs, n, planes, di));
            most = largest(most, d.kernel_gradient_transposed ? gemm_scratch(n, d.inputs, d.rows, planes, di) : gemm_scratch(d.inputs, n, d.rows, planes, di));
        }
    }
    if (l.few) most = largest(most, gemm_parts_scratch(d.rows, d.classes, d.inputs, planes, di));
    l.total = l.scratch + up(most);
    return l;
}

int check_desc(const axc_entropy_desc *d)
{
    if (!d || d->type < kFloat32 || d->type > kFloat16 || d->bias_type < kFloat32 || d->bias_type > kFloat16) return AXC_INVALID_ARGUMENT;
    if (d->rows < 0 || d->inputs < 1 || d->classes < 1 || d->rows > 0x7fffff00ll || d->inputs > 0x7fffff00ll || d->classes > 0x7fffff00ll) return AXC_INVALID_ARGUMENT;
    if (d->x_row_stride < 0 || d->x_column_stride < 0 || d->kernel_row_stride < 0 || d->kernel_column_stride < 0) return AXC_INVALID_ARGUMENT;
    if (d->reduction != AXC_REDUCE_MEAN && d->reduction != AXC_REDUCE_SUM) return AXC_INVALID_ARGUMENT;
    return AXC_OK;
}

int entropy(const axc_entropy_desc &d, const Layout &l, const void *x, const void *kernel, const void *bias, const long long *labels, float *loss, float *row_loss,
            void *dx, void *dkernel, void *dbias, char *ws, const DeviceInfo &di, Queue &q)
{
    const int planes = d.type == kFloat32 ? 3 : 1;
    const float stored = d.type == kFloat16 ? kHalfScale : 1.0f;
    unsigned *status = reinterpret_cast<unsigned *>(ws);
    const size_t per_row = up(size_t(d.rows) * 4);
    float2 *softmax = reinterpret_cast<float2 *>(ws + l.rows);
    float *label_logit = reinterpret_cast<float *>(ws + l.rows + 2 * per_row), *row_scale = reinterpret_cast<float *>(ws + l.rows + 3 * per_row);
    float *alpha = reinterpret_cast<float *>(ws + l.rows + 5 * per_row);
    if (!row_loss) row_loss = reinterpret_cast<float *>(ws + l.rows + 4 * per_row);
    Gemm g = {};
    g.planes = planes;
    g.bf16 = d.type != kFloat16;
    Operand ox = {}, ok = {};
    int rc = AXC_OK;
    if (d.rows > 0) {
        rc = make_operands(x_of(d, x), ws + l.x, &ox, kernel_of(d, kernel), ws + l.kernel, &ok, di, q);
        if (rc) return rc;
        g.m = d.rows;
        g.n = d.classes;
        g.k = d.inputs;
        g.a = ox;
        g.b = ok;
        EntropyArgs e = {};
        e.bias = bias;
        e.bias_type = d.bias_type;
        e.labels = labels;
        e.keep = l.kept ? ws + l.keep : nullptr;
        e.line = l.line;
        e.keep_fp32 = d.type != kBfloat16;
        e.stats = reinterpret_cast<float2 *>(ws + l.stats);
        e.segments = l.segments;
        e.label_logit = label_logit;
        RowArgs r = {};
        rc = l.few ? gemm_parts(g, ws + l.scratch, &r.parts, status, true, di, q) : gemm_entropy(g, e, false, status, true, di, q);
        if (rc) return rc;
        r.rows = d.rows;
        r.classes = d.classes;
        r.labels = labels;
        r.ignore = d.ignore_index;
        r.stats = e.stats;
        r.segments = l.segments;
        r.label_logit = label_logit;
        r.softmax = l.gradients ? softmax : nullptr;
        r.row_scale = row_scale;
        r.row_loss = row_loss;
        r.stored = stored;
        r.keep = e.keep;
        r.line = l.line;
        r.gradient = l.gradients ? reinterpret_cast<uint16_t *>(ws + l.gradient) : nullptr;
        r.bias = bias;
        r.bias_type = d.bias_type;
        r.planes = planes;
        r.bf16 = g.bf16;
        r.plane = l.line * d.rows;
        const unsigned grid = unsigned(d.rows);
        r.done = status + 1;
        r.mean = d.reduction == AXC_REDUCE_MEAN;
        r.grad_factor = d.grad_scale / stored;
        r.loss = loss;
        r.alpha = alpha;
        rc = launch(q, l.few ? (planes == 3 ? few_kernel<true> : few_kernel<false>) : !l.kept ? row_kernel<0> : d.type == kBfloat16 ? row_kernel<1> : d.type == kFloat16 ? row_kernel<2> : row_kernel<3>, dim3(grid), 256, 0, 1, r);
        if (rc) return rc;
    } else {                                   // a sum over nothing
        AXC_CUDA(cudaMemsetAsync(status, 0, sizeof(unsigned), q.stream));
        AXC_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), q.stream));
        AXC_CUDA(cudaMemsetAsync(alpha, 0, sizeof(float), q.stream));
    }
    if (!l.gradients) return AXC_OK;
    const size_t size = type_size(d.type);
    float *dx_sum = reinterpret_cast<float *>(ws + l.dx);
    const long long dx_line = (d.inputs + 3) / 4 * 4;
    const bool pieces = !l.kept && !l.few;
    for (long long c0 = 0; c0 < d.classes; c0 += pieces ? l.piece : d.classes) {
        const long long n = !pieces ? d.classes : d.classes - c0 < l.piece ? d.classes - c0 : l.piece;
        Operand part = ok;                     // the kernel's rows from class c0 on
        part.data = static_cast<const uint16_t *>(ok.data) + (ok.rows_contiguous ? c0 : c0 * ok.line);
        if (pieces && d.rows > 0) {
            Gemm again = g;
            again.n = n;
            again.b = part;
            EntropyArgs e = {};
            e.bias = bias;
            e.bias_type = d.bias_type;
            e.labels = labels;
            e.keep = ws + l.gradient;
            e.line = l.line;
            e.plane = l.line * d.rows;
            e.softmax = softmax;
            e.row_scale = row_scale;
            e.column0 = int(c0);
            rc = gemm_entropy(again, e, true, status, false, di, q);
            if (rc) return rc;
        }
        const Operand dl = {ws + l.gradient, l.line, l.line * d.rows, false};
        Gemm p = {};
        p.planes = planes;
        p.bf16 = g.bf16;
        p.fin.alpha = 1.0f;
        p.fin.alpha_dev = alpha;
        if (dx) {
            const bool last = c0 + n >= d.classes;
            p.m = d.rows;
            p.n = d.inputs;
            p.k = n;
            p.a = dl;
            p.b = transposed(part);
            p.fin.addend = c0 > 0 ? dx_sum : nullptr;
            p.fin.addend_type = kFloat32;
            p.fin.addend_line = dx_line;
            p.fin.out = last ? dx : dx_sum;
            p.fin.out_type = last ? d.type : kFloat32;
            p.fin.out_line = last ? d.inputs : dx_line;
            rc = gemm(p, ws + l.scratch, status, false, di, q);
            if (rc) return rc;
            p.fin.addend = nullptr;
        }
        if (dkernel) {
            p.k = d.rows;
            p.fin.out_type = d.type;
            if (d.kernel_gradient_transposed) {
                p.m = n;
                p.n = d.inputs;
                p.a = transposed(dl);
                p.b = transposed(ox);
                p.fin.out = static_cast<char *>(dkernel) + size_t(c0) * size_t(d.inputs) * size;
                p.fin.out_line = d.inputs;
            } else {
                p.m = d.inputs;
                p.n = n;
                p.a = transposed(ox);
                p.b = transposed(dl);
                p.fin.out = static_cast<char *>(dkernel) + size_t(c0) * size;
                p.fin.out_line = d.classes;
            }
            rc = gemm(p, ws + l.scratch, status, false, di, q);
            if (rc) return rc;
        }
        if (dbias) {
            Slope s = {};
            s.dy = ws + l.gradient;
            s.type = d.type == kFloat16 ? kFloat16 : kBfloat16;
            s.dy_planes = planes;
            s.padded = true;
            s.plane = l.line * d.rows;
            s.rows = d.rows;
            s.columns = n;
            s.dy_line = l.line;
            s.sums = static_cast<char *>(dbias) + size_t(c0) * type_size(d.bias_type);
            s.sums_type = d.bias_type;
            s.scale = 1.0f;
            s.scale_dev = alpha;
            rc = slope(s, ws + l.part, l.scratch - l.part, q);
            if (rc) return rc;
        }
    }
    return AXC_OK;
}

}  // namespace

AXC_DEFINE_BOUNDS_READER(bounds_record_entropy)

}  // namespace axc

extern "C" int axc_entropy_workspace_bytes(const axc_entropy_desc *desc, const void *x, const void *kernel, int device, size_t *loss_only, size_t *gradients)
{
    using namespace axc;
    int rc = check_desc(desc);
    if (rc) return rc;
    DeviceInfo di;
    rc = device_info(device, &di);
    if (rc) return rc;
    if (!x) x = kUnknown;
    if (!kernel) kernel = kUnknown;
    if (loss_only) *loss_only = layout_of(*desc, false, x, kernel, di).total;
    if (gradients) *gradients = layout_of(*desc, true, x, kernel, di).total;
    return AXC_OK;
}

extern "C" int axc_entropy(const axc_entropy_desc *desc, const void *x, const void *kernel, const void *bias, const int64_t *labels, float *loss, float *row_loss,
                           void *dx, void *dkernel, void *dbias, void *workspace, size_t workspace_bytes, int device, void *stream)
{
    using namespace axc;
    int rc = check_desc(desc);
    if (rc) return rc;
    const axc_entropy_desc &d = *desc;
    if (!loss || !kernel || (d.rows > 0 && (!x || !labels))) return AXC_INVALID_ARGUMENT;
    if (!aligned_to(type_size(d.type), x, kernel, dx, dkernel) || !aligned_to(type_size(d.bias_type), bias, dbias) || !aligned_to(sizeof(float), loss, row_loss) ||
        !aligned_to(sizeof(int64_t), labels))
        return AXC_INVALID_ARGUMENT;
    DeviceInfo di;
    rc = device_info(device, &di);
    if (rc) return rc;
    const bool gradients = dx || dkernel || dbias;
    const Layout l = layout_of(d, gradients, x ? x : kUnknown, kernel, di);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < l.total) return AXC_INTERNAL;
    int prev = 0;
    AXC_CUDA(cudaGetDevice(&prev));
    if (prev != device) AXC_CUDA(cudaSetDevice(device));
    Queue q = {cudaStream_t(stream)};
    rc = entropy(d, l, x, kernel, bias, reinterpret_cast<const long long *>(labels), loss, row_loss, dx, dkernel, dbias, static_cast<char *>(workspace), di, q);
    const cudaError_t e = cudaGetLastError();
    if (prev != device) cudaSetDevice(prev);
    return rc != AXC_OK ? rc : e == cudaSuccess ? AXC_OK : cuda_failed(e);
}

extern "C" int axc_scale(const axc_scale_tensor *tensors, int32_t count, const float *factor, int device, void *stream)
{
    using namespace axc;
    if (count < 0 || (count > 0 && !tensors) || !factor || !aligned_to(sizeof(float), factor)) return AXC_INVALID_ARGUMENT;
    long long values = 0;
    for (int32_t i = 0; i < count; ++i) {
        const axc_scale_tensor &t = tensors[i];
        if (t.type < kFloat32 || t.type > kFloat16 || t.count < 0 || t.count > (1ll << 42) || (t.count > 0 && (!t.x || !t.out))) return AXC_INVALID_ARGUMENT;
        if (!aligned_to(type_size(t.type), t.x, t.out)) return AXC_INVALID_ARGUMENT;
        values += t.count;
    }
    if (values == 0) return AXC_OK;
    int prev = 0;
    AXC_CUDA(cudaGetDevice(&prev));
    if (prev != device) AXC_CUDA(cudaSetDevice(device));
    for (int32_t at = 0; at < count;) {
        ScaleArgs A = {};
        A.factor = factor;
        long long blocks = 0;
        for (; at < count && A.parts < kScaleParts; ++at) {
            const long long each = kScaleBytes / (long long)type_size(tensors[at].type), more = (tensors[at].count + each - 1) / each;
            if (more == 0) continue;
            if (blocks + more > 0x7fffffffll) break;           // (one tensor's fit: 2^42 values of 4 bytes are 2^30 blocks)
            A.part[A.parts] = tensors[at];
            A.first[A.parts++] = unsigned(blocks);
            blocks += more;
        }
        if (A.parts == 0) break;
        scale_kernel<<<unsigned(blocks), 256, 0, cudaStream_t(stream)>>>(A);
        count_launch();
    }
    const cudaError_t e = cudaGetLastError();
    if (prev != device) cudaSetDevice(prev);
    return e == cudaSuccess ? AXC_OK : cuda_failed(e);
}
