// The dense layer in 8-bit floating point: y = act(x kernel^T + bias + residual), operands in e4m3 with an fp32 scale for each block of 128 inputs.
//
//   y[r, u] = act( sum over blocks b of sx[r, b] sw[u / 128, b] * (sum over k in b of qx[r, k] qw[u, k]) + bias[u] + residual[r, u] )
//
// The kernel is quantised once (axc_quantize_blocks, 128 x 128 values to a scale); rows are quantised in the call, each block of 128 by itself.  A
// scale is the least power of two with which the block's largest value is a code (448 at most): dividing by it is exact, so that the codes are
// the definition's to the bit, and as codes are floating point, too, it costs no more than the codes below 2^-9 of the largest.
//
//   many rows     tcgen05 matrix instructions on 8-bit operands, 128 k a stage, which is a block: its sums are taken out of tensor memory, times the two
//                 scales, and added in registers, while the next block's are made in the other half of the tensor memory.  The ring of stages is that
//                 of the 16-bit products (axc_gemm.cu).  Bound by taking the sums out: a stage of a tile of 64, 128, 256 columns takes 740, 990, 1430
//                 clocks, its matrix instructions alone 390 to 512, and with sums taken out every eighth block only 977 (at the clocks that the power limit
//                 then leaves); four buffers of 128 columns instead of two of 256 change nothing, so it is the tensor memory's reading, not the waits.
//                 8192 x 4096 x 16384, bf16: 665 to 700 us without an activation (1650 to 1570 TFLOP/s; the same product in 16 bits 680), with gelu 757 to 867, by the
//                 values and the card: the power limit is what differs.
//   up to 8 rows  bound by reading the kernel once.  Four warps share 16 units and have every fourth block of 128 inputs each; a lane reads 16 bytes of two
//                 units at a time, two blocks on their way, and multiplies them, as they are, by mma with the rows as its columns: with plain
//                 multiply-adds 8 rows would cost eight times what one does.  The order of k within a block is the lanes' own, the same for both operands.
//                 1 row of 4096 x 16384: 15.6 us, 8 rows 16.3, 2.5 of it the rows' quantisation (reading the codes once: 10.2); with codes turned into fp16
//                 first 22.8 and 33.5.  Lines that do not start on 16 bytes are read a byte at a time: 1 and 8 rows of 4094 x 16384 take 69 us, 19 with lines
//                 of 4096 bytes.
// Sums within a block are the matrix pipes', over blocks fp32 with rounding; y is rounded once.
#include <cuda_fp8.h>

#include "axc_gemm.h"
#include "axc_lines.cuh"
#include "axc_mma.cuh"
#include "axc_two.cuh"

namespace axc {
namespace {

constexpr int kBlock = AXC_SCALE_BLOCK;        // inputs (and units of the kernel) that share a scale
constexpr int kFewRows = 8;

// ---- quantisation ---------------------------------------------------------------------------------------------------------------
// The scale of a block whose largest magnitude is `top`, and its reciprocal; NaN for a block that has an infinity or a NaN
__device__ __forceinline__ float scale_of(float top, float &inverse)
{
    const unsigned bits = __float_as_uint(top);
    if (bits >= 0x7f800000u) {
        inverse = 0.0f;
        return __uint_as_float(0x7fc00000u);
    }
    // 448 = 1.75 * 2^8
    int power = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    power = max(power, -126);
    inverse = __uint_as_float(unsigned(127 - power) << 23);
    return __uint_as_float(unsigned(127 + power) << 23);
}
// The product of two scales: fp32's largest value where it would leave that range, so that a sum of zeros stays one; NaN stays NaN
__device__ __forceinline__ float scales_product(float a, float b)
{
    const float s = a * b;
    return s > FLT_MAX ? FLT_MAX : s < -FLT_MAX ? -FLT_MAX : s;
}
// (two values' codes, the first in the low byte)
__device__ __forceinline__ unsigned codes_of(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }
// of a block without a scale: any code will do
__device__ __forceinline__ float times(float x, float inverse) { return inverse == 0.0f ? 0.0f : x * inverse; }

struct QuantArgs {
    const void *x;
    long long rows, inputs, row_stride;
    uint8_t *codes;
    long long line;                            // bytes from a row's codes to the next one's; zeros behind the inputs up to it
    float *scales;
    long long scale_row, scale_block;          // scale of (row, block) at row * scale_row + block * scale_block
    unsigned *status;                          // NULL, or cleared
};

// 16 lanes have a row's block, 8 neighbours each
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs A)
{
    after_previous();
    if (A.status && blockIdx.x == 0 && threadIdx.x == 0) A.status[0] = A.status[1] = 0u;
    const long long blocks = (A.inputs + kBlock - 1) / kBlock, total = A.rows * blocks;
    const int lane = threadIdx.x & 15;
    for (long long first = (long long)blockIdx.x * 16; first < total; first += (long long)gridDim.x * 16) {
        const long long item = first + (threadIdx.x >> 4), at = item < total ? item : total - 1, row = at / blocks, block = at - row * blocks;
        const long long k = block * kBlock + lane * 8;
        const T *from = static_cast<const T *>(A.x) + row * A.row_stride + k;
        float v[8];
        [[maybe_unused]] const long long values = (A.rows - 1) * A.row_stride + A.inputs;
        if (VEC && k + 8 <= A.inputs) {
            if (!AXC_VALUES_OK(from, 8, static_cast<const T *>(A.x), values, 601u)) continue;
            union {
                uint4 w[8 * sizeof(T) / 16];
                T t[8];
            } u;
#pragma unroll
            for (int i = 0; i < int(8 * sizeof(T) / 16); ++i) u.w[i] = reinterpret_cast<const uint4 *>(from)[i];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = widen(u.t[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < A.inputs && AXC_VALUES_OK(from + i, 1, static_cast<const T *>(A.x), values, 602u) ? widen(from[i]) : 0.0f;
        }
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max_keep_nan(top, fabsf(v[i]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max_keep_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        float inverse;
        const float scale = scale_of(top, inverse);
        if (item >= total) continue;
        uint8_t *to = A.codes + row * A.line + k;
        const uint2 c = make_uint2(codes_of(times(v[0], inverse), times(v[1], inverse)) | codes_of(times(v[2], inverse), times(v[3], inverse)) << 16,
                                   codes_of(times(v[4], inverse), times(v[5], inverse)) | codes_of(times(v[6], inverse), times(v[7], inverse)) << 16);
        const long long room = A.line - k;     // of the row's line
        if (room >= 8 && (reinterpret_cast<uintptr_t>(to) & 7u) == 0) {
            if (AXC_GLOBAL_OK(row * A.line + k + 7, A.rows * A.line, 603u)) *reinterpret_cast<uint2 *>(to) = c;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < room && AXC_GLOBAL_OK(row * A.line + k + i, A.rows * A.line, 604u)) to[i] = uint8_t((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
        }
        const long long place = row * A.scale_row + block * A.scale_block;
        if (lane == 0 && AXC_GLOBAL_OK(place, A.rows * blocks, 605u)) A.scales[place] = scale;
    }
}

// A block of threads has a block of 128 x 128 values: a thread 8 neighbours of every sixteenth row.  It reads them twice, one by one: a kernel is quantised once.
// 16384 x 4096: bf16 108 us (31 at memory's rate), fp32 160 (51).
template <typename T>
__global__ void __launch_bounds__(256) quantize_squares_kernel(const QuantArgs A)
{
    after_previous();
    __shared__ float tops[8];
    const long long blocks = (A.inputs + kBlock - 1) / kBlock;
    const long long row0 = (long long)(blockIdx.x / blocks) * kBlock, block = blockIdx.x % blocks, k = block * kBlock + (threadIdx.x & 15) * 8;
    [[maybe_unused]] const long long values = (A.rows - 1) * A.row_stride + A.inputs;
    const T *x = static_cast<const T *>(A.x);
    float top = 0.0f;
    for (int r = threadIdx.x >> 4; r < kBlock && row0 + r < A.rows; r += 16) {
        const T *from = x + (row0 + r) * A.row_stride + k;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < A.inputs && AXC_VALUES_OK(from + i, 1, x, values, 606u)) top = max_keep_nan(top, fabsf(widen(from[i])));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_keep_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max_keep_nan(top, tops[i]);
    float inverse;
    const float scale = scale_of(top, inverse);
    for (int r = threadIdx.x >> 4; r < kBlock && row0 + r < A.rows; r += 16) {
        const T *from = x + (row0 + r) * A.row_stride + k;
        uint8_t *to = A.codes + (row0 + r) * A.line + k;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < A.inputs && AXC_VALUES_OK(from + i, 1, x, values, 607u) && AXC_GLOBAL_OK((row0 + r) * A.line + k + i, A.rows * A.line, 608u))
                to[i] = uint8_t(codes_of(times(widen(from[i]), inverse), 0.0f));
    }
    if (threadIdx.x == 0) A.scales[blockIdx.x] = scale;
}

// Codes into lines of a multiple of 16 bytes, zeros behind them
__global__ void __launch_bounds__(256) lay_out_codes_kernel(const uint8_t *src, long long rows, long long inputs, long long stride, uint8_t *dst, long long line)
{
    after_previous();
    const long long groups = line / 16, total = rows * groups;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = i / groups, k = (i - row * groups) * 16;
        const uint8_t *from = src + row * stride + k;
        unsigned w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (k + j < inputs && AXC_VALUES_OK(from + j, 1, src, (rows - 1) * stride + inputs, 609u)) w[j / 4] |= unsigned(from[j]) << (8 * (j & 3));
        if (AXC_GLOBAL_OK(row * line + k + 15, rows * line, 610u)) *reinterpret_cast<uint4 *>(dst + row * line + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ---- many rows ------------------------------------------------------------------------------------------------------------------
// Warps: 0 loads and holds the tensor memory, 1 multiplies, 4 to 19 take the sums out.  Those hold 64 sums a thread beside what is on its way, so the
// first warpgroup leaves them its registers: 640 threads are launched with 96 each, 128 * 32 + 512 * 112 is as many.
constexpr int kThreads = 640, kFewRegisters = 32, kManyRegisters = 112, kTakers = 16;
constexpr unsigned kHeader = 1024, kSmem = 227 * 1024;
constexpr int kMaxStages = 12, kUnits = 4;     // 16-byte units of a row that a warp turns over at a time

#ifdef AXC_BOUNDS_CHECK
__device__ int g_wait_polls = mma::kWaitPolls;
#define AXC_DENSE8_POLLS (*(volatile int *)&g_wait_polls)
#else
#define AXC_DENSE8_POLLS mma::kWaitPolls
#endif

struct Gemm8Args {
    CUtensorMap map_a, map_b;
    int m, n;
    int tiles_m, tiles_n, splits, blocks;      // blocks: of the inputs, a stage each
    int stages;
    unsigned b_bytes, shape;
    const float *a_scales, *b_scales;          // [blocks][m], [ceil(n / 128)][blocks]
    Finish fin;
    float *part;
    long long part_line, part_stride;
    unsigned *status;
};
constexpr unsigned kABytes = 128 * kBlock;     // of a stage, per CTA

struct Header8 {
    uint64_t full[kMaxStages], empty[kMaxStages], sums_full[2], sums_empty[2];
    unsigned tmem;
};

template <int CG>
__device__ __forceinline__ void multiply8(unsigned d, uint64_t a, uint64_t b, unsigned shape, bool add)
{
    if constexpr (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"(unsigned(add)) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"(unsigned(add)) : "memory");
}

// As barrier_wait and barrier_arrive_cluster of axc_mma.cuh, for barriers that hand over nothing but tensor memory and what bulk copies bring, which the
// matrix pipes' own fences order: without a scope that reaches the other CTA's generic memory.  With it each cost about a thousand clocks, once
// for every block of inputs.
__device__ __forceinline__ bool wait_here(unsigned bar, unsigned parity, int polls)
{
    for (int it = 0; it < polls; ++it) {
        unsigned done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (__all_sync(0xffffffffu, done != 0)) return true;
    }
    return false;
}
__device__ __forceinline__ void arrive_at(unsigned bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

// groups of 8 rows of tiles, so that the tiles in flight share lines of both operands
__device__ __forceinline__ void place_of(const Gemm8Args &P, int tile, int &tm, int &tn)
{
    const int per = 8 * P.tiles_n, group = tile / per, first = group * 8, rows = min(8, P.tiles_m - first);
    tm = first + (tile - group * per) % rows;
    tn = (tile - group * per) / rows;
}

// As gemm_kernel, with a block of the inputs to a stage and the scales where the sums are taken out
template <int CG, int BN, bool PARTIAL>
__global__ void __launch_bounds__(kThreads, 1) gemm8_kernel(const __grid_constant__ Gemm8Args P)
{
    constexpr int TM = 128 * CG;
    constexpr unsigned kColumns = BN < 32 ? 32 : BN;
    constexpr int kBuffers = 2;
    extern __shared__ char raw[];
    const unsigned base = (mma::smem_address(raw) + 1023u) & ~1023u;
    Header8 *head = reinterpret_cast<Header8 *>(raw + (base - mma::smem_address(raw)));
    const unsigned lines = base + kHeader, ring = lines + unsigned(kTakers * kUnits) * 512u, stage_bytes = kABytes + P.b_bytes;
    const unsigned full = mma::smem_address(head->full), empty = mma::smem_address(head->empty);
    const unsigned sums_full = mma::smem_address(head->sums_full), sums_empty = mma::smem_address(head->sums_empty);
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const unsigned rank = CG == 2 ? mma::cluster_rank() : 0u;
    const int worker = int(blockIdx.x) / CG, workers = int(gridDim.x) / CG;
    const int units = P.tiles_m * P.tiles_n * P.splits;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int i = 0; i < P.stages; ++i) {
            mma::barrier_init(full + 8 * i, 1);
            mma::barrier_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < kBuffers; ++i) {
            mma::barrier_init(sums_full + 8 * i, 1);
            mma::barrier_init(sums_empty + 8 * i, kTakers * CG);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mma::prefetch_map(&P.map_a);
        mma::prefetch_map(&P.map_b);
    }
    if (warp == 0) mma::tmem_alloc<CG>(mma::smem_address(&head->tmem), kColumns * kBuffers);
    mma::fence_before();
    if (CG == 2) mma::cluster_sync();
    else __syncthreads();
    mma::fence_after();
    const unsigned tmem = head->tmem;
    asm volatile("griddepcontrol.wait;" ::: "memory");          // the codes of the rows come from the kernel before
    bool ok = true;
    const int polls = AXC_DENSE8_POLLS;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
        if (warp == 0) {
            const bool leader = mma::elect();
            const unsigned signal = CG == 2 ? mma::in_cta(full, 0) : full;
            int s = 0;
            unsigned phase = 1;
            for (int u = worker; u < units && ok; u += workers) {
                int tm, tn;
                place_of(P, u / P.splits, tm, tn);
                const int split = u % P.splits;
                const int k0 = int((long long)P.blocks * split / P.splits), k1 = int((long long)P.blocks * (split + 1) / P.splits);
                const int row_a = tm * TM + int(rank) * 128, row_b = tn * BN + int(rank) * (BN / CG);
                for (int k = k0; k < k1; ++k) {
                    if (!(ok = wait_here(empty + 8 * s, phase, polls))) break;
                    if (leader) {
                        if (CG == 1 || rank == 0) mma::barrier_expect(full + 8 * s, stage_bytes * CG);
                        const unsigned at = ring + unsigned(s) * stage_bytes;
                        // (a stage that is not loaded runs the waits out)
                        if (AXC_SHARED_OK(at, 1024u, ring, ring + unsigned(P.stages) * stage_bytes, 611u)) {
                            mma::load_box<CG>(at, &P.map_a, signal + 8 * s, k * kBlock, row_a, 0);
                            mma::load_box<CG>(at + kABytes, &P.map_b, signal + 8 * s, k * kBlock, row_b, 0);
                        }
                    }
                    __syncwarp();
                    if (++s == P.stages) s = 0, phase ^= 1u;
                }
            }
        } else if (warp == 1 && rank == 0) {
            const bool leader = mma::elect();
            int s = 0, buffer = 0;
            unsigned phase = 0, sums_phase = 1;
            for (int u = worker; u < units && ok; u += workers) {
                const int split = u % P.splits;
                const int k0 = int((long long)P.blocks * split / P.splits), k1 = int((long long)P.blocks * (split + 1) / P.splits);
                for (int k = k0; k < k1; ++k) {
                    if (!(ok = wait_here(sums_empty + 8 * buffer, sums_phase, polls))) break;
                    if (!(ok = wait_here(full + 8 * s, phase, polls))) break;
                    mma::fence_after();
                    const unsigned at = (ring + unsigned(s) * stage_bytes) >> 4, d = tmem + unsigned(buffer) * kColumns;
                    if (leader) {
                        // 32 inputs an instruction: 32 bytes of each line
    #pragma unroll
                        for (int j = 0; j < kBlock / 32; ++j)
                            multiply8<CG>(d, mma::operand(at + 2 * j, 0), mma::operand(at + (kABytes >> 4) + 2 * j, 0), P.shape, j > 0);
                        mma::commit<CG>(empty + 8 * s);
                        mma::commit<CG>(sums_full + 8 * buffer);
                    }
                    __syncwarp();
                    if (++s == P.stages) s = 0, phase ^= 1u;
                    if (++buffer == kBuffers) buffer = 0, sums_phase ^= 1u;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
        // four warps take a part of the columns, which has one scale of the kernel at a time
        constexpr int kParts = BN >= 128 ? 4 : BN >= 64 ? 2 : 1, kMine = BN / kParts, W = kMine < 32 ? 16 : 32, kChunks = kMine / W;
        const int part = (warp - 4) >> 2, quarter = warp & 3;
        int buffer = 0;
        unsigned phase = 0;
        for (int u = worker; u < units && ok; u += workers) {
            int tm, tn;
            place_of(P, u / P.splits, tm, tn);
            const int split = u % P.splits;
            const int row0 = tm * TM + int(rank) * 128 + quarter * 32, n0 = tn * BN + part * kMine;
            const int k0 = int((long long)P.blocks * split / P.splits), k1 = int((long long)P.blocks * (split + 1) / P.splits);
            const Lines L = {lines + unsigned(warp - 4) * kUnits * 512u, lane, min(32, P.m - row0)};
            const int row = min(row0 + lane, P.m - 1), square = min(n0, P.n - 1) / kBlock;
            const float *sa = P.a_scales + row, *sb = P.b_scales + (long long)square * P.blocks;
            const unsigned mine = tmem + unsigned(part * kMine) + (unsigned(quarter * 32) << 16);
            Two sum[kMine / 2];
#pragma unroll
            for (int i = 0; i < kMine / 2; ++i) sum[i] = Two(0.0f);
            // two blocks' scales are on their way ahead of the sums that they belong to
            auto a_scale = [&](int k) { return AXC_GLOBAL_OK((long long)k * P.m + row, (long long)P.blocks * P.m, 612u) ? __ldg(sa + (long long)k * P.m) : 0.0f; };
            float a0 = a_scale(k0), b0 = __ldg(sb + k0), a1 = a_scale(min(k0 + 1, k1 - 1)), b1 = __ldg(sb + min(k0 + 1, k1 - 1));
            for (int k = k0; k < k1; ++k) {
                const float a2 = a_scale(min(k + 2, k1 - 1)), b2 = __ldg(sb + min(k + 2, k1 - 1));
                if (!(ok = wait_here(sums_full + 8 * buffer, phase, polls))) break;
                mma::fence_after();
                __syncwarp();
                auto release = [&] {
                    mma::fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_at(mma::in_cta(sums_empty + 8 * buffer, 0));
                };
                if (part < kParts) {
                    const Two both(scales_product(a0, b0));
                    const unsigned at = mine + unsigned(buffer) * kColumns;
                    unsigned x[W];
                    mma::load_columns(at, x);
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
                        mma::load_wait(x);
                        // the matrix instructions may write here again as soon as all has been read
                        if (c + 1 == kChunks) release();
#pragma unroll
                        for (int i = 0; i < W; i += 2)
                            sum[(c * W + i) / 2] = fma2(Two(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), both, sum[(c * W + i) / 2]);
                        if (c + 1 < kChunks) mma::load_columns(at + (c + 1) * W, x);
                    }
                } else release();
                if (++buffer == kBuffers) buffer = 0, phase ^= 1u;
                a0 = a1, b0 = b1, a1 = a2, b1 = b2;
            }
            if (!ok) break;
            if (part < kParts) {
#pragma unroll
                for (int c = 0; c < kMine; c += W) {
                    unsigned x[W];
#pragma unroll
                    for (int i = 0; i < W; i += 2) {
                        const float2 f = sum[(c + i) / 2].both();
                        x[i] = __float_as_uint(f.x);
                        x[i + 1] = __float_as_uint(f.y);
                    }
                    if constexpr (PARTIAL) store_part<W, kUnits>(P.part, P.part_line, P.part_stride, P.splits, P.n, L, x, row0, n0 + c, split);
                    else finish_row<W, kUnits, true>(P.fin, P.n, L, x, row0, n0 + c, 1.0f);
                }
            }
        }
    }
    if (!ok) {
        // A wait ran out: no further copy is started; those in flight end within microseconds, this waits for milliseconds.
        atomicMax(P.status, 3u);
        for (int i = 0; i < 64; ++i) __nanosleep(200000);
    }
    __syncwarp();
    mma::fence_before();
    if (CG == 2) mma::cluster_sync();
    else __syncthreads();
    if (warp == 0) {
        mma::fence_after();
        mma::tmem_free<CG>(tmem, kColumns * kBuffers);
    }
}

// ---- up to 8 rows -----------------------------------------------------------------------------------------------------------------
struct Few8Args {
    int rows;
    long long inputs, units;
    const uint8_t *codes;                      // of the rows, [rows][blocks * 128]
    const float *a_scales;                     // [blocks][rows]
    const uint8_t *kernel;
    long long kernel_stride;
    const float *b_scales;
    Finish fin;
};
constexpr int kFewWarps = 4, kFewUnits = 16;

// D += A B^T for 16 units, 8 rows and 32 inputs
__device__ __forceinline__ void mma_16832(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A block has 16 units; its warps have every kFewWarps-th block of inputs each, and add up in shared memory what they have.
template <bool VEC>
__global__ void __launch_bounds__(kFewWarps * 32, VEC ? 7 : 4) few8_kernel(const Few8Args A)
{
    __shared__ float sums[kFewWarps][kFewUnits][kFewRows + 1];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int blocks = int((A.inputs + kBlock - 1) / kBlock);
    const long long unit0 = (long long)blockIdx.x * kFewUnits;
    // the lane's two units, the last one again behind the last; its row, the last one again (its sums are not used)
    const long long u0 = unit0 + g < A.units ? unit0 + g : A.units - 1, u1 = unit0 + g + 8 < A.units ? unit0 + g + 8 : A.units - 1;
    const int row = min(g, A.rows - 1), column = 2 * t, row0 = min(column, A.rows - 1), row1 = min(column + 1, A.rows - 1);
    const uint8_t *w0 = A.kernel + u0 * A.kernel_stride + t * 16, *w1 = A.kernel + u1 * A.kernel_stride + t * 16;
    const uint8_t *x = A.codes + (long long)row * blocks * kBlock + t * 16;
    [[maybe_unused]] const long long kernel_bytes = (A.units - 1) * A.kernel_stride + A.inputs, code_bytes = (long long)A.rows * blocks * kBlock;
    auto read = [&](const uint8_t *from, long long k) {
        if (VEC && k + 16 <= A.inputs) return AXC_VALUES_OK(from, 16, A.kernel, kernel_bytes, 613u) ? __ldcs(reinterpret_cast<const uint4 *>(from)) : make_uint4(0u, 0u, 0u, 0u);
        unsigned w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (k + i < A.inputs && AXC_VALUES_OK(from + i, 1, A.kernel, kernel_bytes, 614u)) w[i / 4] |= unsigned(from[i]) << (8 * (i & 3));
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    // a block of 128 inputs of the lane's units, 64 at a time
    auto read_block = [&](int b, uint4 (&a)[2][2]) {
        if (b >= blocks) return;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const long long k = (long long)b * kBlock + c * 64;
            a[c][0] = read(w0 + k, k + t * 16);
            a[c][1] = read(w1 + k, k + t * 16);
        }
    };
    // Two blocks' codes are on their way from here on.  (They do not come from the kernel before, which quantises the rows, and that one has started
    // when all before it was over.)
    uint4 a[2][2][2];
    read_block(warp, a[0]);
    read_block(warp + kFewWarps, a[1]);
    const float *b_scales = A.b_scales + unit0 / kBlock * blocks;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add_block = [&](int b, uint4 (&a)[2][2]) {
        const float sb = __ldg(b_scales + b);
        const bool there = AXC_GLOBAL_OK((long long)b * A.rows + row1, (long long)blocks * A.rows, 616u);
        const float s0 = there ? A.a_scales[b * A.rows + row0] : 0.0f, s1 = there ? A.a_scales[b * A.rows + row1] : 0.0f;
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint8_t *from = x + b * kBlock + c * 64;
            const uint4 r = AXC_VALUES_OK(from, 16, A.codes, code_bytes, 615u) ? *reinterpret_cast<const uint4 *>(from) : make_uint4(0u, 0u, 0u, 0u);
            mma_16832(d, a[c][0].x, a[c][1].x, a[c][0].y, a[c][1].y, r.x, r.y);
            mma_16832(d, a[c][0].z, a[c][1].z, a[c][0].w, a[c][1].w, r.z, r.w);
        }
        const float t0 = scales_product(s0, sb), t1 = scales_product(s1, sb);
        sum[0] = fmaf(d[0], t0, sum[0]);
        sum[1] = fmaf(d[1], t1, sum[1]);
        sum[2] = fmaf(d[2], t0, sum[2]);
        sum[3] = fmaf(d[3], t1, sum[3]);
    };
    for (int b = warp; b < blocks; b += 2 * kFewWarps) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (b + i * kFewWarps < blocks) {
                add_block(b + i * kFewWarps, a[i]);
                read_block(b + (i + 2) * kFewWarps, a[i]);
            }
    }
    sums[warp][g][column] = sum[0];
    sums[warp][g][column + 1] = sum[1];
    sums[warp][g + 8][column] = sum[2];
    sums[warp][g + 8][column + 1] = sum[3];
    __syncthreads();
    if (threadIdx.x < kFewUnits * kFewRows) {
        const int unit = threadIdx.x & (kFewUnits - 1), line = threadIdx.x / kFewUnits;
        if (line < A.rows && unit0 + unit < A.units) {
            float z = sums[0][unit][line];
#pragma unroll
            for (int i = 1; i < kFewWarps; ++i) z += sums[i][unit][line];
            finish_value(A.fin, z, line, unit0 + unit);
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
size_t up(size_t bytes) { return (bytes + 255) / 256 * 256; }

// The calls that take the kernel for few rows
bool few_rows8(const axc_dense8_desc &d) { return d.rows <= kFewRows; }
// Codes that TMA reads where they are
bool in_place(const axc_dense8_desc &d, const void *kernel) { return (reinterpret_cast<uintptr_t>(kernel) & 15u) == 0 && d.kernel_row_stride % 16 == 0 && d.kernel_row_stride >= d.inputs; }

// The cheapest tiles and splits by an estimate in clocks, as choose_plan's, with what was measured here: taking a block's sums out bounds a stage, 400 clocks
// and 4.2 for each column of a tile, and what follows the sums is not hidden by the next tile's.  Of all tiles and splits of 11 products, from 20 x 4096 x 300 to
// 3000 x 2000 x 9000, the one chosen was the fastest or within 4 % of it for eight, 8 to 12 % slower for three.
Plan choose_plan8(long long m, long long n, long long blocks, int sms)
{
    Plan best = {1, 128, 1};
    double least = 1e300;
    const double memory = (double(m) + double(n)) * double(blocks) * kBlock / 3400;
    for (int c = 0; c < 6; ++c) {
        static const int kCg[6] = {2, 1, 1, 1, 1, 1}, kBn[6] = {256, 256, 128, 64, 32, 16};
        const int cg = kCg[c], bn = kBn[c];
        const double bytes = (double(m < 128 ? m : 128) + bn / cg) * kBlock;
        const long long tiles = ceil_div(m, 128 * cg) * ceil_div(n, bn), workers = sms / cg;
        for (int splits = 1; splits <= 16; splits *= 2) {
            if (splits > 1 && blocks / splits < 2) break;
            const long long units = tiles * splits;
            const double copies = bytes / 114 * double(units < workers ? units : workers) / double(workers), taking = 400 + 4.2 * bn, stage = taking > copies ? taking : copies;
            double clocks = double(ceil_div(units, workers)) * (double(ceil_div(blocks, splits)) * stage + 2500 + 12 * bn);
            if (clocks < memory) clocks = memory;
            clocks += 4500;
            if (splits > 1) clocks += 7600 + double(m) * double(n) * splits * 8 / 7400;
            if (clocks < least) {
                least = clocks;
                best = {cg, bn, splits};
            }
        }
    }
    return best;
}

struct Room8 {
    size_t codes, scales, kernel, part, total;
};
Room8 room_of(const axc_dense8_desc &d, const void *kernel, int sms)
{
    Room8 r = {256, 256, 256, 256, 256};       // the status word comes first
    const long long blocks = ceil_div(d.inputs, kBlock);
    r.scales = r.codes + up(size_t(d.rows) * size_t(blocks) * kBlock);
    r.total = r.part = r.kernel = r.scales + up(size_t(d.rows) * size_t(blocks) * 4);
    if (few_rows8(d)) return r;
    r.part = r.kernel + (in_place(d, kernel) ? 0 : up(size_t(d.units) * size_t(ceil_div(d.inputs, 16)) * 16));
    const Plan plan = choose_plan8(d.rows, d.units, blocks, sms);
    r.total = r.part + (plan.splits > 1 ? up(size_t(plan.splits) * size_t(d.rows) * size_t(ceil_div(d.units, 4)) * 16) : 0);
    return r;
}

bool make_map8(const void *data, long long rows, long long inputs, long long line, unsigned box, CUtensorMap *map)
{
    PFN_cuTensorMapEncodeTiled_v12000 encode = encoder();
    if (!encode) return false;
    const cuuint64_t dims[3] = {cuuint64_t(inputs), cuuint64_t(rows), 1}, strides[2] = {cuuint64_t(line), cuuint64_t(line)};
    const cuuint32_t boxes[3] = {unsigned(kBlock), box, 1}, unit[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(data), dims, strides, boxes, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int CG, int BN, bool PARTIAL>
int launch_gemm8(Gemm8Args &P, int sms, Queue &q)
{
    const unsigned stage = kABytes + P.b_bytes, lines = kTakers * kUnits * 512;
    P.stages = int((kSmem - kHeader - 1024 - lines) / stage);
    if (P.stages > kMaxStages) P.stages = kMaxStages;
    static std::atomic<unsigned long long> ready{0};
    const int rc = allow_smem(gemm8_kernel<CG, BN, PARTIAL>, kSmem, ready);
    if (rc) return rc;
    const long long units = (long long)P.tiles_m * P.tiles_n * P.splits, workers = sms / CG;
    return launch(q, gemm8_kernel<CG, BN, PARTIAL>, dim3(unsigned((units < workers ? units : workers) * CG)), kThreads,
                  kHeader + 1024 + lines + unsigned(P.stages) * stage, CG, P);
}
template <bool PARTIAL>
int launch_tiles8(Gemm8Args &P, const Plan &plan, int sms, Queue &q)
{
    if (plan.bn == 256) return plan.cg == 2 ? launch_gemm8<2, 256, PARTIAL>(P, sms, q) : launch_gemm8<1, 256, PARTIAL>(P, sms, q);
    if (plan.bn == 128) return launch_gemm8<1, 128, PARTIAL>(P, sms, q);
    if (plan.bn == 64) return launch_gemm8<1, 64, PARTIAL>(P, sms, q);
    if (plan.bn == 32) return launch_gemm8<1, 32, PARTIAL>(P, sms, q);
    return launch_gemm8<1, 16, PARTIAL>(P, sms, q);
}

template <typename T>
int launch_quantize(const QuantArgs &A, bool vec, int sms, Queue &q)
{
    const long long items = A.rows * ceil_div(A.inputs, kBlock), want = ceil_div(items, 16), most = (long long)sms * 16;
    return launch(q, vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, dim3(unsigned(want < most ? want : most)), 256, 0, 1, A);
}
int quantize_rows(const QuantArgs &A, int type, int sms, Queue &q)
{
    const bool vec = (reinterpret_cast<uintptr_t>(A.x) & 15u) == 0 && A.row_stride * (long long)type_size(type) % 16 == 0;
    if (type == kFloat32) return launch_quantize<float>(A, vec, sms, q);
    return type == kBfloat16 ? launch_quantize<__nv_bfloat16>(A, vec, sms, q) : launch_quantize<__half>(A, vec, sms, q);
}
int quantize_squares(const QuantArgs &A, int type, Queue &q)
{
    const dim3 grid(unsigned(ceil_div(A.rows, kBlock) * ceil_div(A.inputs, kBlock)));
    if (type == kFloat32) return launch(q, quantize_squares_kernel<float>, grid, 256, 0, 1, A);
    return type == kBfloat16 ? launch(q, quantize_squares_kernel<__nv_bfloat16>, grid, 256, 0, 1, A) : launch(q, quantize_squares_kernel<__half>, grid, 256, 0, 1, A);
}

Finish finish_of(const axc_dense8_desc &d, const void *bias, const void *residual, void *y)
{
    Finish f = {};
    f.alpha = 1.0f;
    f.bias = bias;
    f.bias_type = d.bias_type;
    f.addend = residual;
    f.addend_type = d.type;
    f.addend_line = d.residual_row_stride;
    f.activation = d.activation;
    f.out = y;
    f.out_type = d.type;
    f.out_line = d.units;
    return f;
}

int forward(const axc_dense8_desc &d, const void *x, const uint8_t *kernel, const float *kernel_scales, const void *bias, const void *residual, void *y, char *ws, int sms,
            Queue &q)
{
    unsigned *status = reinterpret_cast<unsigned *>(ws);
    const Finish fin = sized(finish_of(d, bias, residual, y), d.rows, d.units);
    const Room8 room = room_of(d, kernel, sms);
    const long long blocks = ceil_div(d.inputs, kBlock);
    QuantArgs A = {};
    A.x = x;
    A.rows = d.rows;
    A.inputs = d.inputs;
    A.row_stride = d.x_row_stride;
    A.codes = reinterpret_cast<uint8_t *>(ws + room.codes);
    A.line = blocks * kBlock;
    A.scales = reinterpret_cast<float *>(ws + room.scales);
    A.scale_row = 1;
    A.scale_block = d.rows;
    A.status = status;
    int rc = quantize_rows(A, d.type, sms, q);
    if (rc) return rc;
    if (few_rows8(d)) {
        const Few8Args F = {int(d.rows), d.inputs, d.units, A.codes, A.scales, kernel, d.kernel_row_stride, kernel_scales, fin};
        const dim3 grid(unsigned(ceil_div(d.units, kFewUnits)));
        return launch(q, in_place(d, kernel) ? few8_kernel<true> : few8_kernel<false>, grid, kFewWarps * 32, 0, 1, F);
    }
    const void *codes = kernel;
    long long line = d.kernel_row_stride;
    if (!in_place(d, kernel)) {
        line = ceil_div(d.inputs, 16) * 16;
        codes = ws + room.kernel;
        const long long work = ceil_div(d.units * (line / 16), 256), most = (long long)sms * 16;
        rc = launch(q, lay_out_codes_kernel, dim3(unsigned(work < most ? work : most)), 256, 0, 1, kernel, (long long)d.units, (long long)d.inputs, (long long)d.kernel_row_stride,
                    reinterpret_cast<uint8_t *>(ws + room.kernel), line);
        if (rc) return rc;
    }
    const Plan plan = choose_plan8(d.rows, d.units, blocks, sms);
    Gemm8Args P = {};
    P.m = int(d.rows);
    P.n = int(d.units);
    P.tiles_m = int(ceil_div(d.rows, 128 * plan.cg));
    P.tiles_n = int(ceil_div(d.units, plan.bn));
    P.splits = plan.splits;
    P.blocks = int(blocks);
    P.b_bytes = unsigned(plan.bn / plan.cg) * kBlock;
    // e4m3 both, fp32 sums, k contiguous
    P.shape = (1u << 4) | (unsigned(plan.bn >> 3) << 17) | (unsigned(128 * plan.cg >> 4) << 24);
    P.a_scales = A.scales;
    P.b_scales = kernel_scales;
    P.fin = fin;
    P.status = status;
    if ((long long)P.tiles_m * P.tiles_n * P.splits > 0x7fffffffll) return AXC_INVALID_ARGUMENT;
    if (!make_map8(A.codes, d.rows, d.inputs, A.line, 128, &P.map_a) || !make_map8(codes, d.units, d.inputs, line, unsigned(plan.bn / plan.cg), &P.map_b)) return AXC_INTERNAL;
    if (plan.splits == 1) return launch_tiles8<false>(P, plan, sms, q);
    P.part = reinterpret_cast<float *>(ws + room.part);
    P.part_line = ceil_div(d.units, 4) * 4;
    P.part_stride = P.part_line * d.rows;
    rc = launch_tiles8<true>(P, plan, sms, q);
    if (rc) return rc;
    DeviceInfo di = {};
    di.sm_count = sms;
    return finish_parts(Parts{P.part, P.part_line, P.part_stride, plan.splits}, d.rows, d.units, fin, di, q);
}

int check_desc(const axc_dense8_desc *d)
{
    if (!d || d->rows < 0 || d->inputs < 1 || d->units < 0 || d->rows > 0x7fffff00ll || d->inputs > 0x7fffff00ll || d->units > 0x7fffff00ll) return AXC_INVALID_ARGUMENT;
    if (d->type < kFloat32 || d->type > kFloat16 || d->bias_type < kFloat32 || d->bias_type > kFloat16) return AXC_INVALID_ARGUMENT;
    if (d->activation < kActNone || d->activation > kActSilu || d->x_row_stride < 0 || d->kernel_row_stride < 0 || d->residual_row_stride < 0) return AXC_INVALID_ARGUMENT;
    return AXC_OK;
}

}  // namespace

AXC_DEFINE_BOUNDS_READER(bounds_record_dense8)

#ifdef AXC_BOUNDS_CHECK
int set_dense8_wait_polls(int polls)
{
    const int value = polls < 0 ? mma::kWaitPolls : polls;
    AXC_CUDA(cudaMemcpyToSymbol(g_wait_polls, &value, sizeof(value)));
    return AXC_OK;
}
#endif

}  // namespace axc

extern "C" int axc_quantize_blocks(const void *x, int64_t rows, int64_t inputs, int64_t row_stride, int32_t type, int32_t block_rows, uint8_t *codes, float *scales, int device,
                                   void *stream)
{
    using namespace axc;
    if (rows < 0 || inputs < 0 || row_stride < 0 || type < kFloat32 || type > kFloat16 || (block_rows != 1 && block_rows != kBlock)) return AXC_INVALID_ARGUMENT;
    if (rows == 0 || inputs == 0) return AXC_OK;
    if (!x || !codes || !scales || !aligned_to(type_size(type), x) || !aligned_to(4, scales)) return AXC_INVALID_ARGUMENT;
    if (double(ceil_div(rows, block_rows)) * double(ceil_div(inputs, kBlock)) > double(0x7fffffffll)) return AXC_INVALID_ARGUMENT;
    int sms = 0;
    const int rc = sm_count(device, &sms);
    if (rc) return rc;
    const long long blocks = ceil_div(inputs, kBlock);
    const QuantArgs A = {x, rows, inputs, row_stride, codes, inputs, scales, blocks, 1, nullptr};
    Queue q = {cudaStream_t(stream)};
    return on_device(device, [&] { return block_rows == 1 ? quantize_rows(A, type, sms, q) : quantize_squares(A, type, q); });
}

extern "C" int axc_dense8_workspace_bytes(const axc_dense8_desc *desc, const void *kernel, int device, size_t *bytes)
{
    using namespace axc;
    int rc = check_desc(desc), sms = 0;
    if (rc) return rc;
    if (!bytes) return AXC_INVALID_ARGUMENT;
    rc = sm_count(device, &sms);
    if (rc) return rc;
    *bytes = desc->rows == 0 || desc->units == 0 ? 256 : room_of(*desc, kernel ? kernel : reinterpret_cast<const void *>(uintptr_t(1)), sms).total;
    return AXC_OK;
}

extern "C" int axc_dense8_forward(const axc_dense8_desc *desc, const void *x, const void *kernel, const float *kernel_scales, const void *bias, const void *residual, void *y,
                                  void *workspace, size_t workspace_bytes, int device, void *stream)
{
    using namespace axc;
    int rc = check_desc(desc), sms = 0;
    if (rc) return rc;
    const axc_dense8_desc &d = *desc;
    if (d.rows == 0 || d.units == 0) return AXC_OK;
    if (!x || !kernel || !kernel_scales || !y) return AXC_INVALID_ARGUMENT;
    if (!aligned_to(type_size(d.type), x, residual, y) || !aligned_to(type_size(d.bias_type), bias) || !aligned_to(4, kernel_scales)) return AXC_INVALID_ARGUMENT;
    rc = sm_count(device, &sms);
    if (rc) return rc;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < room_of(d, kernel, sms).total) return AXC_INTERNAL;
    Queue q = {cudaStream_t(stream)};
    return on_device(device, [&] {
        return forward(d, x, static_cast<const uint8_t *>(kernel), kernel_scales, bias, residual, y, static_cast<char *>(workspace), sms, q);
    });
}
