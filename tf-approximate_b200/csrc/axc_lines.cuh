// A tile's way from a warp's registers to memory, and what follows a product on it.
#pragma once
#include "axc_gemm.h"

namespace axc {

// ---- lines of 32 rows between a warp's registers and memory --------------------------------------------------------------
// A lane has a row of the sums, memory wants neighbouring lanes to have neighbouring values: 16 bytes stored by every lane to its own
// row took 11 300 clocks for a tile of 128 x 256, three times what 512 k of the matrix instructions take.  So the warp turns the
// rows over in shared memory, 16-byte units exchanged by row so that neither side has bank conflicts, and moves N units of a row
// (128 bytes, or 32 where the stages leave no more room) at a time.
struct Lines {
    unsigned stage;                            // the warp's shared memory
    int lane, rows;                            // rows of the 32 that exist
};
// What the lines are a part of (debug flavour)
struct Whole {
    const char *base;
    long long bytes;
};

template <int N>
__device__ __forceinline__ unsigned unit_at(unsigned stage, int row, int unit) { return stage + unsigned(row * N + (unit ^ (row & (N - 1)))) * 16u; }

// Lines that do not start on 16 bytes: value by value, neighbouring lanes neighbouring ones, several on their way at a time.
template <int N, typename Pointer, typename Move>
__device__ __forceinline__ void single_values(const Lines &L, Pointer lines, long long line, int left, int size, const Whole &all, Move move)
{
    const int in_row = N * 16 / size;          // a power of two, 8 to 64
#pragma unroll 8
    for (int i = 0; i < in_row; ++i) {
        const int at = i * 32 + L.lane, r = at / in_row, b = (at & (in_row - 1)) * size;
        if (r < L.rows && b < left && AXC_VALUES_OK(lines + r * line + b, size, all.base, all.bytes, 431u) &&
            AXC_SHARED_OK(unit_at<N>(L.stage, r, b >> 4) + unsigned(b & 15), unsigned(size), L.stage, L.stage + N * 512u, 432u))
            move(unit_at<N>(L.stage, r, b >> 4) + unsigned(b & 15), lines + r * line + b, size);
    }
}

// `bytes`: how many of a row exist; aligned: all rows start on 16 bytes
template <int M, int N>
__device__ __forceinline__ void store_lines(const Lines &L, const uint4 (&q)[M], char *out, long long line, int bytes, int size, bool aligned, const Whole &all)
{
#pragma unroll
    for (int part = 0; part < M; part += N) {
        __syncwarp();
#pragma unroll
        for (int u = 0; u < N; ++u) {
            if (!AXC_SHARED_OK(unit_at<N>(L.stage, L.lane, u), 16u, L.stage, L.stage + N * 512u, 433u)) continue;
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(unit_at<N>(L.stage, L.lane, u)), "r"(q[part + u].x), "r"(q[part + u].y),
                         "r"(q[part + u].z), "r"(q[part + u].w) : "memory");
        }
        __syncwarp();
        char *to = out + part * 16;
        const int left = bytes - part * 16;
        if (aligned && left >= N * 16) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = (i * 32 + L.lane) / N, u = L.lane % N;
                uint4 w;
                asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(unit_at<N>(L.stage, r, u)));
                if (r < L.rows && AXC_VALUES_OK(to + r * line + u * 16, 16, all.base, all.bytes, 434u)) *reinterpret_cast<uint4 *>(to + r * line + u * 16) = w;
            }
        } else {
            single_values<N>(L, to, line, left, size, all, [](unsigned from, char *at, int size) {
                if (size == 2) {
                    unsigned short h;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(from));
                    *reinterpret_cast<unsigned short *>(at) = h;
                } else {
                    unsigned w;
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(from));
                    *reinterpret_cast<unsigned *>(at) = w;
                }
            });
        }
    }
}

// The other way: M units of the lane's row, zeros where there is nothing.
template <int M, int N, bool BATCH = false>
__device__ __forceinline__ void load_lines(const Lines &L, uint4 (&q)[M], const char *in, long long line, int bytes, int size, bool aligned, const Whole &all)
{
#pragma unroll
    for (int part = 0; part < M; part += N) {
        __syncwarp();
        const char *from = in + part * 16;
        const int left = bytes - part * 16;
        if (BATCH && aligned && left >= N * 16) {
            uint4 w[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = (i * 32 + L.lane) / N, u = L.lane % N;
                w[i] = make_uint4(0u, 0u, 0u, 0u);
                if (r < L.rows && AXC_VALUES_OK(from + r * line + u * 16, 16, all.base, all.bytes, 435u)) w[i] = *reinterpret_cast<const uint4 *>(from + r * line + u * 16);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = (i * 32 + L.lane) / N, u = L.lane % N;
                if (!AXC_SHARED_OK(unit_at<N>(L.stage, r, u), 16u, L.stage, L.stage + N * 512u, 436u)) continue;
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(unit_at<N>(L.stage, r, u)), "r"(w[i].x), "r"(w[i].y), "r"(w[i].z), "r"(w[i].w) : "memory");
            }
        } else if (BATCH) {
            constexpr int kBatch = 8;
            const int in_row = N * 16 / size;
            for (int first = 0; first < in_row; first += kBatch) {
                unsigned w[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int at = (first + i) * 32 + L.lane, r = at / in_row, b = (at & (in_row - 1)) * size;
                    const char *place = from + r * line + b;
                    w[i] = 0u;
                    if (r < L.rows && b < left && AXC_VALUES_OK(place, size, all.base, all.bytes, 431u))
                        w[i] = size == 2 ? *reinterpret_cast<const unsigned short *>(place) : *reinterpret_cast<const unsigned *>(place);
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int at = (first + i) * 32 + L.lane, r = at / in_row, b = (at & (in_row - 1)) * size;
                    const unsigned to = unit_at<N>(L.stage, r, b >> 4) + unsigned(b & 15);
                    if (!AXC_SHARED_OK(to, unsigned(size), L.stage, L.stage + N * 512u, 432u)) continue;
                    if (size == 2) asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"((unsigned short)w[i]) : "memory");
                    else asm volatile("st.shared.u32 [%0], %1;" ::"r"(to), "r"(w[i]) : "memory");
                }
            }
        } else if (aligned && left >= N * 16) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = (i * 32 + L.lane) / N, u = L.lane % N;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (r < L.rows && AXC_VALUES_OK(from + r * line + u * 16, 16, all.base, all.bytes, 435u)) w = *reinterpret_cast<const uint4 *>(from + r * line + u * 16);
                if (!AXC_SHARED_OK(unit_at<N>(L.stage, r, u), 16u, L.stage, L.stage + N * 512u, 436u)) continue;
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(unit_at<N>(L.stage, r, u)), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
            }
        } else {
            single_values<N>(L, from, line, left, size, all, [](unsigned to, const char *at, int size) {
                if (size == 2) asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(*reinterpret_cast<const unsigned short *>(at)) : "memory");
                else asm volatile("st.shared.u32 [%0], %1;" ::"r"(to), "r"(*reinterpret_cast<const unsigned *>(at)) : "memory");
            });
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < N; ++u)
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(q[part + u].x), "=r"(q[part + u].y), "=r"(q[part + u].z), "=r"(q[part + u].w)
                         : "r"(unit_at<N>(L.stage, L.lane, u)));
    }
}

__device__ __forceinline__ bool lines_aligned(const void *base, long long line_bytes) { return ((reinterpret_cast<uintptr_t>(base) | uintptr_t(line_bytes)) & 15u) == 0; }

// W fp32 values of every lane's row, as `type`; columns n0 .. of n; values: all that there are from `base` on
template <int W, int N>
__device__ __forceinline__ void store_row(const Lines &L, const float (&v)[W], void *base, int type, long long line, int row0, int n0, int n, long long values)
{
    const int size = type == kFloat32 ? 4 : 2, left = n - n0;
    char *out = static_cast<char *>(base) + (row0 * line + n0) * size;
    const bool aligned = lines_aligned(base, line * size);
    const int bytes = (left < W ? left : W) * size;
    const Whole all = {static_cast<const char *>(base), values * size};
    if (type == kFloat32) {
        uint4 q[W / 4];
#pragma unroll
        for (int i = 0; i < W / 4; ++i)
            q[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
        store_lines<W / 4, (W / 4 < N ? W / 4 : N)>(L, q, out, line * 4, bytes, 4, aligned, all);
    } else {
        const bool bf16 = type == kBfloat16;
        uint4 q[W / 8];
#pragma unroll
        for (int i = 0; i < W / 8; ++i)
            q[i] = make_uint4(pack2(v[8 * i], v[8 * i + 1], bf16), pack2(v[8 * i + 2], v[8 * i + 3], bf16), pack2(v[8 * i + 4], v[8 * i + 5], bf16),
                              pack2(v[8 * i + 6], v[8 * i + 7], bf16));
        store_lines<W / 8, (W / 8 < N ? W / 8 : N)>(L, q, out, line * 2, bytes, 2, aligned, all);
    }
}

// bias[n0 + i] of W columns, W / 32 in each lane; column() hands one to all lanes
template <int W>
struct ColumnValues {
    float mine[W < 32 ? 1 : W / 32];
    __device__ __forceinline__ ColumnValues(const void *values, int type, int n0, int n, int lane)
    {
#pragma unroll
        for (int i = 0; i < (W < 32 ? 1 : W / 32); ++i) {
            const int c = n0 + 32 * i + lane;
            mine[i] = values && c < n && AXC_GLOBAL_OK(c, n, 437u) ? load_as_float(values, c, type) : 0.0f;
        }
    }
    __device__ __forceinline__ float column(int i) const { return __shfl_sync(0xffffffffu, mine[i / 32], i & 31); }
};

// One row of W sums (columns n0 ..), W a multiple of 16; all lanes of the warp, whether their row exists or not.  PAIRS: activations of 16-bit
// results two at a time, and the addend's values loaded before the first of them is put down (each took the memory's latency else: 12 of 30 us for
// 1531 x 2777 fp16 values that start anywhere).
template <int W, int N, bool PAIRS = false>
__device__ __forceinline__ void finish_row(const Finish &f, int n, const Lines &L, unsigned (&x)[W], int row0, int n0, float alpha)
{
    if (n0 >= n) return;
    const bool exact = f.out_type == kFloat32;
    float v[W];
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = alpha * __uint_as_float(x[i]);
    if (f.bias) {
        const ColumnValues<W> bias(f.bias, f.bias_type, n0, n, L.lane);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] += bias.column(i);
    }
    if (f.addend) {
        const int size = f.addend_type == kFloat32 ? 4 : 2, left = n - n0, bytes = (left < W ? left : W) * size;
        const char *in = static_cast<const char *>(f.addend) + ((long long)row0 * f.addend_line + n0) * size;
        const bool aligned = lines_aligned(f.addend, f.addend_line * size);
        const Whole all = {static_cast<const char *>(f.addend), f.addend_values() * size};
        if (size == 4) {
            uint4 q[W / 4];
            load_lines<W / 4, (W / 4 < N ? W / 4 : N), PAIRS>(L, q, in, f.addend_line * 4, bytes, 4, aligned, all);
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                v[4 * i] += __uint_as_float(q[i].x);
                v[4 * i + 1] += __uint_as_float(q[i].y);
                v[4 * i + 2] += __uint_as_float(q[i].z);
                v[4 * i + 3] += __uint_as_float(q[i].w);
            }
        } else {
            uint4 q[W / 8];
            load_lines<W / 8, (W / 8 < N ? W / 8 : N), PAIRS>(L, q, in, f.addend_line * 2, bytes, 2, aligned, all);
#pragma unroll
            for (int i = 0; i < W / 8; ++i) {
                const unsigned u[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 t = f.addend_type == kBfloat16 ? __bfloat1622float2(reinterpret_cast<const __nv_bfloat162 &>(u[j]))
                                                                : __half22float2(reinterpret_cast<const __half2 &>(u[j]));
                    v[8 * i + 2 * j] += t.x;
                    v[8 * i + 2 * j + 1] += t.y;
                }
            }
        }
    }
    if (f.pre) store_row<W, N>(L, v, f.pre, f.out_type, f.out_line, row0, n0, n, f.out_values());
    if (PAIRS && !exact && f.activation >= kActGelu) {
#pragma unroll
        for (int i = 0; i < W; i += 2) {
            const Two z(v[i], v[i + 1]);
            Two bell;
            const float2 y = mul2(z, f.activation == kActGelu ? normal_below2(z, bell) : sigmoid2(z)).both();
            v[i] = y.x;
            v[i + 1] = y.y;
        }
    } else if (f.activation == kActRelu) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = activate(v[i], kActRelu, exact);
    } else if (f.activation == kActGelu) {
        if (exact) {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = activate(v[i], kActGelu, true);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = activate(v[i], kActGelu, false);
        }
    } else if (f.activation == kActSilu) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = exact ? activate(v[i], kActSilu, true) : activate(v[i], kActSilu, false);
    }
    store_row<W, N>(L, v, f.out, f.out_type, f.out_line, row0, n0, n, f.out_values());
}

// Partial sums in the order of the output's lines
template <int W, int N>
__device__ __forceinline__ void store_part(float *parts, long long part_line, long long part_stride, int splits, int n, const Lines &L, unsigned (&x)[W], int row0, int n0,
                                           int split)
{
    if (n0 >= n) return;
    float *part = parts + (long long)split * part_stride;
    float v[W];
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = __uint_as_float(x[i]);
    store_row<W, N>(L, v, part, kFloat32, part_line, row0, n0, n, (splits - split) * part_stride);
}

}  // namespace axc
