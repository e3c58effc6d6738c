// Matrix products on the 5th-generation tensor cores: out[m, n] = sum over k of a[m, k] b[n, k], either operand with k or with its
// rows contiguous, so that a layer's forward product and both of its gradients read their operands where they lie.
//
// A CTA (or a pair of CTAs on two SMs that share one tile) is persistent and walks over tiles.  One thread keeps a ring of stages
// of 64 k full with tiled bulk copies (128-byte swizzle), one thread issues the matrix instructions, whose sums stay in tensor
// memory, and eight warps take finished sums out while the next tile's are being made in the other half of the tensor memory.
//   pairs, 256 x 256 tiles    each SM loads 128 rows of a and half of b: 64 bytes of shared memory written and as many read per
//                             clock, half of what a lone SM needs for 128 x 256
//   lone CTAs, 128 x N tiles  for products with too few tiles to fill the GPU
//
// fp32 operands are split exactly into three bf16 terms, x = x0 + x1 + x2, each 2^-8 of the one before; six of the nine products
// of terms are summed (x2 y0, x1 y1, x0 y2, x1 y0, x0 y1, x0 y0), the three left out are below 2^-24 of x y.  Infinities are split so that
// their products are those of the values (split_terms).
//
// Sums are fp32.  The tensor cores cut a sum off at 24 bits at every step of 16 k (measured: 2e-8 of it on average, always towards
// zero), which 16-bit results do not show.  For fp32 the sums of every 64 k, the small products first, are taken out and added in
// registers, with rounding: an error of 1e-7 instead of 2e-5 at k = 16384; the eight warps do that while the next 64 k run.  So are the
// sums of 256 k (512 where k is over 1536) for 16-bit operands whose result a ReLU cuts: the sign of a sum near zero decides about a whole
// gradient there.  Of 4.25 million sums of 1030 products about one had another sign than the exact sum; with runs of 512 one in four such
// products has one, with 256 one in sixteen.  That costs 10 % (1531 x 1032 x 2776: 18.9 to 20.8 us; 4096 x 4096 x 4096 in runs of 512: 97 to
// 107, of 256: 129).  Longer sums would want the shorter runs as much; they have the longer ones for their price alone, 10 instead
// of 33 %.  (128 sums a thread spill in the tiles of 256 columns: 88 to 92 bytes written and 860 to 908 read, 344 and 256 in the split form.)
//
// Products whose tiles are too few have k split over CTAs; the partial sums are added in a fixed order by a second
// kernel, which also applies what follows the product.
#include <atomic>

#include "axc_gemm.h"
#include "axc_lines.cuh"
#include "axc_mma.cuh"

namespace axc {
namespace {

constexpr int kStageK = 64;                    // k of a stage: 128 bytes, a swizzled line
constexpr int kThreads = 320;                  // warps: 0 loads and holds the tensor memory, 1 multiplies, 2 to 9 take the sums out
constexpr unsigned kHeader = 1024;             // barriers and such, before the stages
constexpr unsigned kSmem = 227 * 1024;
constexpr int kMaxStages = 12;
constexpr int kSegment = 64;                   // columns whose exponentials share a largest logit

// Polls after which a wait gives up.  The debug flavour reads them from device memory, so that a test can make the waits run out.
#ifdef AXC_BOUNDS_CHECK
__device__ int g_wait_polls = mma::kWaitPolls;
#define AXC_MATRIX_POLLS (*(volatile int *)&g_wait_polls)
#else
#define AXC_MATRIX_POLLS mma::kWaitPolls
#endif

enum { kStore = 0, kPartial = 1, kEntropy = 2, kGradient = 3 };

struct GemmArgs {
    CUtensorMap map_a, map_b;
    int m, n;
    int tiles_m, tiles_n, splits, k_steps;     // k_steps: stages of the whole k
    int planes, stages;
    unsigned a_bytes, b_bytes;                 // of one plane of a stage, per CTA
    unsigned a_box_rows, b_box_rows;           // a box has that many rows (k contiguous), or 64 (rows contiguous)
    bool a_rows, b_rows;
    unsigned shape;
    Finish fin;
    EntropyArgs ent;
    float *part;                               // [split][line][part_line]
    long long part_line, part_stride;
    unsigned *status;
    bool first;                                // of a call: clears the status
    int run;                                   // CLOSE, 16-bit operands: stages between two takings out
};

struct Header {                                // in shared memory
    uint64_t full[kMaxStages], empty[kMaxStages], sums_full[2], sums_empty[2];
    unsigned tmem;
};

// One segment of 64 logits of a row: the exponentials relative to the largest, their sum, and the label's logit on the way.
// A segment of -inf has the exponentials 0 (relative to 0, not to itself); one with a NaN has nothing else.  `label`: the row's.
template <int N, bool EXACT>
__device__ __forceinline__ void entropy_segment(const GemmArgs &P, const Lines &L, unsigned (&x)[64], int row0, int n0, long long label)
{
    const EntropyArgs &e = P.ent;
    if (n0 >= P.n) return;
    const int row = row0 + L.lane;
    float v[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(x[i]);
    if (e.bias || n0 + 64 > P.n) {             // classes that are not there count as -inf
        const ColumnValues<64> bias(e.bias, e.bias_type, n0, P.n, L.lane);
#pragma unroll
        for (int i = 0; i < 64; ++i) {
            const float b = bias.column(i);
            v[i] = n0 + i < P.n ? v[i] + b : -INFINITY;
        }
    }
    float top4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int i = 4; i < 64; ++i) top4[i & 3] = max_keep_nan(top4[i & 3], v[i]);
    const float top = max_keep_nan(max_keep_nan(top4[0], top4[1]), max_keep_nan(top4[2], top4[3]));
    label -= n0;
    if (row < P.m && label >= 0 && label < kSegment && n0 + label < P.n && AXC_GLOBAL_OK(row, P.m, 438u)) {
        float mine = -INFINITY;
#pragma unroll
        for (int i = 0; i < 64; ++i) mine = fmaxf(mine, i == int(label) ? v[i] : -INFINITY);
        e.label_logit[row] = mine;
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float sum4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 64; ++i) {
        v[i] = exponential(v[i] - base, EXACT);
        sum4[i & 3] += v[i];
    }
    if (row < P.m && AXC_GLOBAL_OK((long long)row * e.segments + n0 / kSegment, (long long)P.m * e.segments, 439u))
        e.stats[(long long)row * e.segments + n0 / kSegment] = make_float2(top, (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
    if (e.keep) store_row<64, N>(L, v, e.keep, e.keep_fp32 ? kFloat32 : kFloat16, e.line, row0, n0, int(e.line), P.m * e.line);
}

// W logits of a row and what the loss's gradient is there: row_scale * (exp(logit - largest) / sum - [label])
template <int W, int N, bool EXACT>
__device__ __forceinline__ void gradient_columns(const GemmArgs &P, const Lines &L, unsigned (&x)[W], int row0, int n0)
{
    const EntropyArgs &e = P.ent;
    if (n0 >= e.line) return;
    const int row = row0 + L.lane < P.m ? row0 + L.lane : P.m - 1;
    const float2 softmax = e.softmax[row];
    const float scale = e.row_scale[row];
    const long long label = e.labels[row] - e.column0 - n0;
    float v[W];
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = __uint_as_float(x[i]);
    if (e.bias || n0 + W > P.n) {
        const ColumnValues<W> bias(e.bias ? static_cast<const char *>(e.bias) + (long long)e.column0 * (e.bias_type == kFloat32 ? 4 : 2) : nullptr, e.bias_type, n0,
                                   P.n, L.lane);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float b = bias.column(i);
            v[i] = n0 + i < P.n ? v[i] + b : -INFINITY;
        }
    }
    // a row without a label stays out, whatever its logits are
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = scale != 0.0f ? scale * (exponential(v[i] - softmax.x, EXACT) * softmax.y - (label == i ? 1.0f : 0.0f)) : 0.0f;
    uint16_t *keep = static_cast<uint16_t *>(e.keep);
    const int type = (P.shape >> 7 & 1) ? kBfloat16 : kFloat16;
    for (int plane = 0; plane < P.planes; ++plane) {
        store_row<W, N>(L, v, keep, type, e.line, row0, n0, int(e.line), P.m * e.line);
        if (P.planes == 3) {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] -= __bfloat162float(__float2bfloat16_rn(v[i]));
        }
        keep += e.plane;
    }
}

// tile index -> place: groups of 8 rows of tiles, so that the tiles in flight share lines of both operands
__device__ __forceinline__ void place_of(const GemmArgs &P, int tile, int &tm, int &tn)
{
    const int per = 8 * P.tiles_n, group = tile / per, first = group * 8, rows = min(8, P.tiles_m - first);
    tm = first + (tile - group * per) % rows;
    tn = (tile - group * per) / rows;
}

// CG: CTAs per tile.  BN: columns of a tile.  MODE: what becomes of the sums.  PLANES: terms of an operand.  CLOSE: sums are taken out and
// added in registers on the way.
template <int CG, int BN, int MODE, int PLANES, bool CLOSE>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ GemmArgs P)
{
    constexpr int TM = 128 * CG;
    constexpr unsigned kColumns = BN < 32 ? 32 : BN;           // tensor memory of one tile's sums
    constexpr int kBuffers = 2, kUnits = PLANES == 3 ? 2 : 8;
    const int run = PLANES == 3 ? 1 : P.run;                   // stages between two takings out, a power of two
    extern __shared__ char raw[];
    const unsigned base = (mma::smem_address(raw) + 1023u) & ~1023u;
    Header *head = reinterpret_cast<Header *>(raw + (base - mma::smem_address(raw)));
    const unsigned lines = base + kHeader, ring = lines + 8u * kUnits * 512u, stage_bytes = unsigned(PLANES) * (P.a_bytes + P.b_bytes);
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
            mma::barrier_init(sums_empty + 8 * i, 8 * CG);
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
    asm volatile("griddepcontrol.wait;" ::: "memory");          // operands may come from the kernel before
    // a wait runs out after a second, not before this; the word behind the status counts what a later kernel has done
    if (P.first && blockIdx.x == 0 && threadIdx.x == 0) P.status[0] = P.status[1] = 0u;
    bool ok = true;
    const int polls = AXC_MATRIX_POLLS;

    // The loading and the multiplying warp run as a whole and one of their threads acts, so that what it hands over is computed once for
    // the warp: with a branch around the loop the 4 matrix instructions of a stage took 660 clocks instead of 512, the issuing thread's own.
    if (warp == 0) {
        const bool leader = mma::elect();
        const unsigned signal = CG == 2 ? mma::in_cta(full, 0) : full;
        int s = 0;
        unsigned phase = 1;
        for (int u = worker; u < units && ok; u += workers) {
            int tm, tn;
            place_of(P, u / P.splits, tm, tn);
            const int split = u % P.splits;
            const int k0 = int((long long)P.k_steps * split / P.splits), k1 = int((long long)P.k_steps * (split + 1) / P.splits);
            const int row_a = tm * TM + int(rank) * 128, row_b = tn * BN + int(rank) * (BN / CG);
            for (int k = k0; k < k1; ++k) {
                if (!(ok = mma::barrier_wait(empty + 8 * s, phase, polls))) break;
                if (leader) {
                    if (CG == 1 || rank == 0) mma::barrier_expect(full + 8 * s, stage_bytes * CG);
                    unsigned at = ring + unsigned(s) * stage_bytes;
                    // (a stage that is not loaded runs the waits out)
                    for (int p = 0; p < PLANES && AXC_SHARED_OK(at, 1024u, ring, ring + unsigned(P.stages) * stage_bytes, 440u); ++p) {
                        if (P.a_rows) {
                            for (int r = 0; r < 128; r += 64) mma::load_box<CG>(at + unsigned(r) * 128u, &P.map_a, signal + 8 * s, row_a + r, k * kStageK, p);
                        } else mma::load_box<CG>(at, &P.map_a, signal + 8 * s, k * kStageK, row_a, p);
                        at += P.a_bytes;
                        if (P.b_rows) {
                            for (int r = 0; r < BN / CG; r += 64) mma::load_box<CG>(at + unsigned(r) * 128u, &P.map_b, signal + 8 * s, row_b + r, k * kStageK, p);
                        } else mma::load_box<CG>(at, &P.map_b, signal + 8 * s, k * kStageK, row_b, p);
                        at += P.b_bytes;
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
        // the products of the three terms, smallest first: the terms of a and of b
        const unsigned of_a = PLANES == 3 ? 0x001012u : 0u, of_b = PLANES == 3 ? 0x010210u : 0u;
        constexpr int kProducts = PLANES == 3 ? 6 : 1;
        const unsigned chunk_a = P.a_rows ? 8192u : 0u, chunk_b = P.b_rows ? 8192u : 0u;
        const unsigned step_a = (P.a_rows ? 2048u : 32u) >> 4, step_b = (P.b_rows ? 2048u : 32u) >> 4;
        for (int u = worker; u < units && ok; u += workers) {
            const int split = u % P.splits;
            const int k0 = int((long long)P.k_steps * split / P.splits), k1 = int((long long)P.k_steps * (split + 1) / P.splits);
            unsigned d = 0;
            for (int k = k0; k < k1; ++k) {
                const bool opens = CLOSE ? ((k - k0) & (run - 1)) == 0 : k == k0, closes = k + 1 == k1 || (CLOSE && ((k - k0) & (run - 1)) == run - 1);
                if (opens) {
                    if (!(ok = mma::barrier_wait(sums_empty + 8 * buffer, sums_phase, polls))) break;
                    d = tmem + unsigned(buffer) * kColumns;
                }
                if (!(ok = mma::barrier_wait(full + 8 * s, phase, polls))) break;
                mma::fence_after();
                const unsigned at = (ring + unsigned(s) * stage_bytes) >> 4, plane = (P.a_bytes + P.b_bytes) >> 4;
                if (leader) {
#pragma unroll
                    for (int q = 0; q < kProducts; ++q) {
                        const unsigned a = at + (of_a >> (4 * q) & 15u) * plane, b = at + (of_b >> (4 * q) & 15u) * plane + (P.a_bytes >> 4);
#pragma unroll
                        for (int j = 0; j < kStageK / 16; ++j)
                            mma::multiply<CG>(d, mma::operand(a + j * step_a, chunk_a), mma::operand(b + j * step_b, chunk_b), P.shape,
                                              !opens || q > 0 || j > 0);
                    }
                    mma::commit<CG>(empty + 8 * s);
                    if (closes) mma::commit<CG>(sums_full + 8 * buffer);
                }
                __syncwarp();
                if (++s == P.stages) s = 0, phase ^= 1u;
                if (closes) {
                    if (++buffer == kBuffers) buffer = 0, sums_phase ^= 1u;
                }
            }
        }
    } else if (warp >= 2) {
        // warps 2 to 5 take the first half of the columns, 6 to 9 the second; a warp reaches the 32 lanes of its place in four
        constexpr int kHalves = BN >= 128 ? 2 : 1;
        const int half = (warp - 2) >> 2, quarter = warp & 3;
        const float alpha = MODE == kStore ? P.fin.alpha * (P.fin.alpha_dev ? *P.fin.alpha_dev : 1.0f) : 1.0f;
        int buffer = 0;
        unsigned phase = 0;
        constexpr int kMine = BN / kHalves, W = kMine < 32 ? 16 : kMine < 64 || (CLOSE && MODE != kEntropy) ? 32 : 64;
        for (int u = worker; u < units && ok; u += workers) {
            int tm, tn;
            place_of(P, u / P.splits, tm, tn);
            const int split = u % P.splits;
            const int row0 = tm * TM + int(rank) * 128 + quarter * 32, n0 = tn * BN + half * kMine;
            const Lines L = {lines + unsigned(warp - 2) * kUnits * 512u, lane, min(32, P.m - row0)};
            const int of_lane = row0 + lane < P.m ? row0 + lane : P.m - 1;
            const long long label = MODE == kEntropy ? P.ent.labels[of_lane] : 0;
            auto take = [&](unsigned (&x)[W], int c) {
                if constexpr (MODE == kStore) finish_row<W, kUnits>(P.fin, P.n, L, x, row0, n0 + c, alpha);
                else if constexpr (MODE == kPartial) store_part<W, kUnits>(P.part, P.part_line, P.part_stride, P.splits, P.n, L, x, row0, n0 + c, split);
                else if constexpr (MODE == kGradient) gradient_columns<W, kUnits, PLANES == 3>(P, L, x, row0, n0 + c);
                else entropy_segment<kUnits, PLANES == 3>(P, L, x, row0, n0 + c, label);
            };
            const unsigned mine = tmem + unsigned(half * kMine) + (unsigned(quarter * 32) << 16);
            if constexpr (CLOSE) {
                const int k0 = int((long long)P.k_steps * split / P.splits), k1 = int((long long)P.k_steps * (split + 1) / P.splits);
                unsigned sum[kMine / W][W];
#pragma unroll
                for (int c = 0; c < kMine / W; ++c)
#pragma unroll
                    for (int i = 0; i < W; ++i) sum[c][i] = 0u;
                for (int k = k0; k < k1; k += run) {
                    if (!(ok = mma::barrier_wait(sums_full + 8 * buffer, phase, polls))) break;
                    mma::fence_after();
                    __syncwarp();
                    if (half < kHalves) {
#pragma unroll
                        for (int c = 0; c < kMine; c += (W < 32 ? W : 32)) {
                            unsigned x[W < 32 ? W : 32];
                            mma::load_columns(mine + unsigned(buffer) * kColumns + c, x);
                            mma::load_wait(x);
#pragma unroll
                            for (int i = 0; i < (W < 32 ? W : 32); ++i)
                                sum[c / W][c % W + i] = __float_as_uint(__uint_as_float(sum[c / W][c % W + i]) + __uint_as_float(x[i]));
                        }
                    }
                    mma::fence_before();
                    __syncwarp();
                    if (lane == 0) mma::barrier_arrive_cluster(mma::in_cta(sums_empty + 8 * buffer, 0));
                    if (++buffer == kBuffers) buffer = 0, phase ^= 1u;
                }
                if (!ok) break;
                if (half < kHalves) {
#pragma unroll
                    for (int c = 0; c < kMine / W; ++c) take(sum[c], c * W);
                }
            } else {
                if (!(ok = mma::barrier_wait(sums_full + 8 * buffer, phase, polls))) break;
                mma::fence_after();
                __syncwarp();
                if (half < kHalves) {
                    const unsigned at = mine + unsigned(buffer) * kColumns;
#pragma unroll 1
                    for (int c = 0; c < kMine; c += W) {
                        unsigned x[W];
                        mma::load_columns(at + c, x);
                        mma::load_wait(x);
                        take(x, c);
                    }
                }
                mma::fence_before();
                __syncwarp();
                if (lane == 0) mma::barrier_arrive_cluster(mma::in_cta(sums_empty + 8 * buffer, 0));
                if (++buffer == kBuffers) buffer = 0, phase ^= 1u;
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

// The partial sums of a split product, added in the order of the splits, and what follows the product
__global__ void __launch_bounds__(256) finish_kernel(const float *part, long long stride, long long part_line, int splits, int lines,
                                                     int columns, const Finish f)
{
    after_previous();
    const int quads = (columns + 3) / 4;
    const long long total = (long long)lines * quads;
    const float alpha = f.alpha * (f.alpha_dev ? *f.alpha_dev : 1.0f);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long line = i / quads;
        const int c = int(i - line * quads) * 4;
        const float *at = part + line * part_line + c;
        if (!AXC_VALUES_OK(at + (splits > 0 ? splits - 1 : 0) * stride, splits > 0 ? 4 : 0, part, splits * stride, 426u)) continue;
        float4 s = splits > 0 ? *reinterpret_cast<const float4 *>(at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int k = 1; k < splits; ++k) {
            const float4 t = *reinterpret_cast<const float4 *>(at + k * stride);
            s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
        }
        const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (c + j < columns) {
                finish_value(f, alpha * v[j], line, c + j);
            }
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
}  // namespace

PFN_cuTensorMapEncodeTiled_v12000 encoder()
{
    static PFN_cuTensorMapEncodeTiled_v12000 fn = []() -> PFN_cuTensorMapEncodeTiled_v12000 {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

namespace {

// Boxes of 64 k x `box` rows (k contiguous), or 64 rows x 64 k; what lies outside the matrix arrives as zeros.
bool make_map(const Operand &o, long long rows, long long k, int planes, bool bf16, unsigned box, CUtensorMap *map)
{
    PFN_cuTensorMapEncodeTiled_v12000 encode = encoder();
    if (!encode) return false;
    const cuuint64_t inner = cuuint64_t(o.rows_contiguous ? rows : k), outer = cuuint64_t(o.rows_contiguous ? k : rows);
    const cuuint64_t dims[3] = {inner, outer, cuuint64_t(planes)};
    const cuuint64_t line = cuuint64_t(o.line) * 2, strides[2] = {line, planes > 1 ? cuuint64_t(o.plane) * 2 : line};
    const cuuint32_t boxes[3] = {64, o.rows_contiguous ? 64u : box, 1}, unit[3] = {1, 1, 1};
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(o.data), dims, strides,
                  boxes, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// The cheapest of the tiles and splits by an estimate in clocks.  A stage takes what its matrix instructions take (2 for each column of
// a tile, 390 at least) or what its bytes take (114 a clock and SM when all SMs have tiles, in proportion when few have), whichever is
// more; a wave of tiles 3400 more until its sums are out, the product another 4500 for its first bytes and its last tile; a split one 7600
// for the second kernel and its partial sums' way to L2 and back.  Fitted to all tiles and splits measured for 34 products, in bf16 from
// 4 x 2048 x 1000 to 8192 x 8192 x 2048 and 2047 x 50001 x 1024, in fp32 from 64 x 300 x 64 to 2000 x 2000 x 2000: the one chosen so was
// the fastest or within 2 % of it for 30, 3 to 12 % slower for three (3000 x 3000 x 700: 27.6 us instead of 24.6) and 29 % for 4 x 4096 x
// 16384 (37 instead of 28.7: so few rows of a are the same few lines of memory for every CTA).
Plan choose_plan(long long m, long long n, long long k, int planes, bool may_split, int sms)
{
    Plan best = {1, 128, 1};
    double least = 1e300;
    const long long steps = ceil_div(k > 0 ? k : 1, kStageK);
    const double memory = (double(m) + double(n)) * double(k) * 2 * planes / 3400;         // the operands, once, at memory's rate
    for (int c = 0; c < 6; ++c) {
        static const int kCg[6] = {2, 1, 1, 1, 1, 1}, kBn[6] = {256, 256, 128, 64, 32, 16};
        const int cg = kCg[c], bn = planes == 3 && cg == 2 ? 128 : kBn[c];
        if (!may_split && bn < 64) continue;                    // logits: segments of 64 columns
        if (planes == 3 && bn == 256) continue;                 // its sums do not fit into registers
        const double products = (planes == 3 ? 6 : 1) * (bn > 195 ? 2.0 * bn : 390.0), bytes = planes * (double(m < 128 ? m : 128) + bn / cg) * 128;
        const long long tiles = ceil_div(m, 128 * cg) * ceil_div(n, bn), workers = sms / cg;
        for (int splits = 1; splits <= (may_split ? 16 : 1); splits *= 2) {
            if (splits > 1 && steps / splits < 2) break;
            const long long units = tiles * splits;
            const double copies = bytes / 114 * double(units < workers ? units : workers) / double(workers), stage = products > copies ? products : copies;
            double clocks = double(ceil_div(units, workers)) * (double(ceil_div(steps, splits)) * stage + 3400);
            if (clocks < memory) clocks = memory;
            clocks += 4500 + 8 * bn;
            if (splits > 1) clocks += 7600 + double(m) * n * splits * 8 / 7400;
            if (clocks < least) {
                least = clocks;
                best = {cg, bn, splits};
            }
        }
    }
    return best;
}

template <int CG, int BN, int MODE, int PLANES, bool CLOSE>
int launch_gemm(GemmArgs &P, long long units, const DeviceInfo &di, Queue &q)
{
    const unsigned stage = unsigned(PLANES) * (P.a_bytes + P.b_bytes);
    const unsigned lines = PLANES == 3 ? 8 * 1024 : 8 * 4096;
    P.stages = int((kSmem - kHeader - 1024 - lines) / stage);
    if (P.stages > kMaxStages) P.stages = kMaxStages;
    const unsigned smem = kHeader + 1024 + lines + unsigned(P.stages) * stage;
    static std::atomic<unsigned long long> ready{0};           // devices on which the kernel may have all shared memory
    int device = 0;
    AXC_CUDA(cudaGetDevice(&device));
    const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
    if (!(ready.load(std::memory_order_acquire) & bit) || !bit) {
        AXC_CUDA(cudaFuncSetAttribute(gemm_kernel<CG, BN, MODE, PLANES, CLOSE>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmem)));
        ready.fetch_or(bit, std::memory_order_release);
    }
    const long long workers = di.sm_count / CG;
    return launch(q, gemm_kernel<CG, BN, MODE, PLANES, CLOSE>, dim3(unsigned((units < workers ? units : workers) * CG)), kThreads, smem, CG, P);
}

template <int MODE, int PLANES, bool CLOSE>
int launch_tiles(GemmArgs &P, const Plan &plan, long long units, const DeviceInfo &di, Queue &q)
{
    if constexpr (PLANES == 1) {
        if (plan.bn == 256) return plan.cg == 2 ? launch_gemm<2, 256, MODE, 1, CLOSE>(P, units, di, q) : launch_gemm<1, 256, MODE, 1, CLOSE>(P, units, di, q);
    } else {
        if (plan.cg == 2) return launch_gemm<2, 128, MODE, 3, true>(P, units, di, q);
    }
    if (plan.bn == 128) return launch_gemm<1, 128, MODE, PLANES, CLOSE>(P, units, di, q);
    if (plan.bn == 64) return launch_gemm<1, 64, MODE, PLANES, CLOSE>(P, units, di, q);
    if constexpr (MODE == kStore || MODE == kPartial) {
        if (plan.bn == 32) return launch_gemm<1, 32, MODE, PLANES, CLOSE>(P, units, di, q);
        return launch_gemm<1, 16, MODE, PLANES, CLOSE>(P, units, di, q);
    }
    return AXC_INTERNAL;
}

template <int MODE>
int launch_plan(GemmArgs &P, const Plan &plan, long long units, const DeviceInfo &di, Queue &q)
{
    if (P.planes == 3) return launch_tiles<MODE, 3, true>(P, plan, units, di, q);
    if constexpr (MODE == kStore || MODE == kPartial) {
        if (P.fin.activation == kActRelu) return launch_tiles<MODE, 1, true>(P, plan, units, di, q);
    }
    return launch_tiles<MODE, 1, false>(P, plan, units, di, q);
}

int fill_args(const Gemm &g, const Plan &plan, unsigned *status, bool first, GemmArgs *P)
{
    const Operand &a = g.a, &b = g.b;
    if (g.m > 0x7fffff00ll || g.n > 0x7fffff00ll || g.k > 0x7fffff00ll) return AXC_INVALID_ARGUMENT;
    const unsigned b_rows_per_cta = unsigned(plan.bn / plan.cg);
    P->m = int(g.m);
    P->n = int(g.n);
    P->tiles_m = int(ceil_div(g.m, 128 * plan.cg));
    P->tiles_n = int(ceil_div(g.n, plan.bn));
    P->splits = plan.splits;
    P->k_steps = int(ceil_div(g.k, kStageK));
    P->planes = g.planes;
    P->a_rows = a.rows_contiguous;
    P->b_rows = b.rows_contiguous;
    P->a_bytes = 128 * 128;
    P->b_bytes = (b.rows_contiguous && b_rows_per_cta < 64 ? 64u : b_rows_per_cta) * 128u;
    P->shape = mma::instruction_shape(128 * plan.cg, plan.bn, g.bf16, a.rows_contiguous, b.rows_contiguous);
    P->fin = sized(g.fin, g.m, g.n);
    P->status = status;
    P->first = first;
    P->run = P->k_steps <= 24 ? 4 : 8;
    if (!make_map(a, g.m, g.k, g.planes, g.bf16, 128, &P->map_a) || !make_map(b, g.n, g.k, g.planes, g.bf16, b_rows_per_cta, &P->map_b))
        return AXC_INTERNAL;
    return AXC_OK;
}

}  // namespace

#ifdef AXC_BOUNDS_CHECK
int set_matrix_wait_polls(int polls)
{
    const int value = polls < 0 ? mma::kWaitPolls : polls;
    AXC_CUDA(cudaMemcpyToSymbol(g_wait_polls, &value, sizeof(value)));
    return AXC_OK;
}
#endif

int finish_parts(const Parts &parts, long long lines, long long columns, const Finish &f, const DeviceInfo &di, Queue &q)
{
    const long long work = ceil_div(lines * ceil_div(columns, 4), 256), most = (long long)di.sm_count * 8;
    return launch(q, finish_kernel, dim3(unsigned(work < most ? work : most)), 256, 0, 1, parts.data, parts.stride, parts.line, parts.count, int(lines),
                  int(columns), sized(f, lines, columns));
}

AXC_DEFINE_BOUNDS_READER(bounds_record_gemm)

size_t gemm_scratch(long long m, long long n, long long k, int planes, const DeviceInfo &di)
{
    if (m == 0 || n == 0 || k == 0) return 0;
    const Plan plan = choose_plan(m, n, k, planes, true, di.sm_count);
    return plan.splits > 1 ? size_t(plan.splits) * size_t(m) * size_t((n + 3) / 4 * 4) * 4 : 0;
}

size_t gemm_parts_scratch(long long m, long long n, long long k, int planes, const DeviceInfo &di)
{
    const Plan plan = choose_plan(m, n, k, planes, true, di.sm_count);
    return size_t(plan.splits) * size_t(m) * size_t((n + 3) / 4 * 4) * 4;
}

int gemm_parts(const Gemm &g, void *scratch, Parts *parts, unsigned *status, bool first, const DeviceInfo &di, Queue &q)
{
    const Plan plan = choose_plan(g.m, g.n, g.k, g.planes, true, di.sm_count);
    GemmArgs P = {};
    const int rc = fill_args(g, plan, status, first, &P);
    if (rc) return rc;
    P.part = static_cast<float *>(scratch);
    P.part_line = (g.n + 3) / 4 * 4;
    P.part_stride = P.part_line * g.m;
    *parts = {P.part, P.part_line, P.part_stride, plan.splits};
    return launch_plan<kPartial>(P, plan, (long long)P.tiles_m * P.tiles_n * plan.splits, di, q);
}

int gemm(const Gemm &g, void *scratch, unsigned *status, bool first, const DeviceInfo &di, Queue &q)
{
    if (g.m == 0 || g.n == 0 || g.k == 0) {                     // nothing, or sums of nothing: no kernel that would clear the status
        if (first) AXC_CUDA(cudaMemsetAsync(status, 0, sizeof(unsigned), q.stream));
        return g.m == 0 || g.n == 0 ? AXC_OK : finish_parts(Parts{}, g.m, g.n, g.fin, di, q);
    }
    const Plan plan = choose_plan(g.m, g.n, g.k, g.planes, true, di.sm_count);
    if (plan.splits > 1) {
        Parts parts;
        const int rc = gemm_parts(g, scratch, &parts, status, first, di, q);
        return rc ? rc : finish_parts(parts, g.m, g.n, g.fin, di, q);
    }
    GemmArgs P = {};
    const int rc = fill_args(g, plan, status, first, &P);
    if (rc) return rc;
    const long long units = (long long)P.tiles_m * P.tiles_n;
    if (units > 0x7fffffffll) return AXC_INVALID_ARGUMENT;
    return launch_plan<kStore>(P, plan, units, di, q);
}

int gemm_entropy(const Gemm &g, const EntropyArgs &e, bool gradient, unsigned *status, bool first, const DeviceInfo &di, Queue &q)
{
    if (g.m == 0 || g.n == 0) return AXC_OK;
    const Plan plan = choose_plan(g.m, g.n, g.k, g.planes, false, di.sm_count);
    GemmArgs P = {};
    int rc = fill_args(g, plan, status, first, &P);
    if (rc) return rc;
    const long long units = (long long)P.tiles_m * P.tiles_n;
    if (units > 0x7fffffffll) return AXC_INVALID_ARGUMENT;
    P.ent = e;
    return gradient ? launch_plan<kGradient>(P, plan, units, di, q) : launch_plan<kEntropy>(P, plan, units, di, q);
}

// ---- operands -----------------------------------------------------------------------------------------------------------
namespace {

// What lay_out_kernel copies: `outer` lines of `inner` values
struct Layout {
    const void *src;
    uint16_t *dst;
    long long outer, inner, outer_stride, inner_stride, line, plane;
    bool split;
};

// Copies one matrix or two into lines of a multiple of 8 values, 16-bit types as they are, fp32 as three bf16 planes: the value rounded
// to bf16, the rest rounded again, and what is left then, which bf16 holds exactly.  The first `blocks` blocks have the first matrix.
__global__ void __launch_bounds__(256) lay_out_kernel(const Layout one, const Layout two, int blocks)
{
    after_previous();
    const bool second = int(blockIdx.x) >= blocks;
    const Layout &m = second ? two : one;
    const long long groups = m.line / 8, total = m.outer * groups, stride = (long long)(second ? gridDim.x - blocks : blocks) * 256;
    for (long long i = (long long)(blockIdx.x - (second ? blocks : 0)) * 256 + threadIdx.x; i < total; i += stride) {
        const long long o = i / groups, c = (i - o * groups) * 8;
        uint16_t *to = m.dst + o * m.line + c;
        const long long from = o * m.outer_stride + c * m.inner_stride;
        [[maybe_unused]] const long long values = (m.outer - 1) * m.outer_stride + (m.inner - 1) * m.inner_stride + 1;
        if (!AXC_GLOBAL_OK(from + ((c + 8 < m.inner ? c + 8 : m.inner) - 1 - c) * m.inner_stride, values, 424u) ||
            !AXC_GLOBAL_OK(o * m.line + c + 7 + (m.split ? 2 : 0) * m.plane, m.outer * m.line * (m.split ? 3 : 1), 425u))
            continue;
        if (m.split) {
            const float *src = static_cast<const float *>(m.src) + from;
            float x[8];
            if (m.inner_stride == 1 && c + 8 <= m.inner && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
                const float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + 4);
                x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
                x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = c + j < m.inner ? src[j * m.inner_stride] : 0.0f;
            }
            unsigned t[4][3];
#pragma unroll
            for (int j = 0; j < 4; ++j) split_terms(x[2 * j], x[2 * j + 1], t[j]);
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4 *>(to + p * m.plane) = make_uint4(t[0][p], t[1][p], t[2][p], t[3][p]);
        } else {
            const uint16_t *src = static_cast<const uint16_t *>(m.src) + from;
            union { uint16_t h[8]; uint4 w; } out;
#pragma unroll
            for (int j = 0; j < 8; ++j) out.h[j] = c + j < m.inner ? src[j * m.inner_stride] : uint16_t(0);
            *reinterpret_cast<uint4 *>(to) = out.w;
        }
    }
}

// rows or columns contiguous: which of the two is the inner dimension of the copy
bool columns_inner(const Matrix &x) { return x.column_stride == 1 || x.columns == 1 || x.row_stride != 1; }

}  // namespace

bool readable_in_place(const Matrix &x)
{
    if (x.type == kFloat32 || (reinterpret_cast<uintptr_t>(x.data) & 15u)) return false;
    const bool by_columns = x.column_stride == 1 && x.row_stride % 8 == 0 && x.row_stride >= x.columns;
    const bool by_rows = x.row_stride == 1 && x.column_stride % 8 == 0 && x.column_stride >= x.rows;
    return by_columns || by_rows;
}

size_t operand_bytes(const Matrix &x)
{
    if (x.rows == 0 || x.columns == 0 || readable_in_place(x)) return 0;
    const bool in = columns_inner(x);
    const size_t inner = size_t(in ? x.columns : x.rows), outer = size_t(in ? x.rows : x.columns);
    return (outer * ((inner + 7) / 8 * 8) * 2 * (x.type == kFloat32 ? 3 : 1) + 255) / 256 * 256;
}

namespace {

// The operand, and in `copy` how it gets there (outer = 0: it is read in place)
Operand plan_operand(const Matrix &x, void *scratch, Layout *copy)
{
    *copy = {};
    if (x.rows == 0 || x.columns == 0) return {nullptr, 8, 0, false};
    if (readable_in_place(x)) {
        const bool by_columns = x.column_stride == 1 && x.row_stride % 8 == 0 && x.row_stride >= x.columns;
        return {x.data, by_columns ? x.row_stride : x.column_stride, 0, !by_columns};
    }
    const bool in = columns_inner(x);
    copy->src = x.data;
    copy->dst = static_cast<uint16_t *>(scratch);
    copy->inner = in ? x.columns : x.rows;
    copy->outer = in ? x.rows : x.columns;
    copy->outer_stride = in ? x.row_stride : x.column_stride;
    copy->inner_stride = in ? x.column_stride : x.row_stride;
    copy->line = (copy->inner + 7) / 8 * 8;
    copy->plane = copy->outer * copy->line;
    copy->split = x.type == kFloat32;
    return {scratch, copy->line, copy->plane, !in};
}

}  // namespace

int make_operands(const Matrix &x, void *x_scratch, Operand *ox, const Matrix &y, void *y_scratch, Operand *oy, const DeviceInfo &di, Queue &q)
{
    Layout one, two;
    *ox = plan_operand(x, x_scratch, &one);
    *oy = plan_operand(y, y_scratch, &two);
    const long long most = (long long)di.sm_count * 16;
    long long a = ceil_div(one.outer * (one.line / 8), 256), b = ceil_div(two.outer * (two.line / 8), 256);
    if (a + b == 0) return AXC_OK;
    if (a > most) a = most;
    if (b > most) b = most;
    return launch(q, lay_out_kernel, dim3(unsigned(a + b)), 256, 0, 1, one, two, int(a));
}

}  // namespace axc
