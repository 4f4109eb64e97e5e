// Layer norm over the last dimension, forward and backward.
//
//   m = mean x,  r = 1 / sqrt(mean (x - m)^2 + eps),  xh = (x - m) r,  y = xh w + b
//   g = dy w,    dx = r (g - mean g - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Both directions are bound by memory: forward moves x and y once, backward x, dy and dx.  A row is held in the
// registers of a group of lanes -- 1 .. 64 lanes of a wave, or a whole block -- so that the variance is taken around the
// mean without reading the row again.  The mean of n values s away from zero is off by up to n 2^-24 s, as much as the
// deviations themselves where a row lies far out: what is left of it is summed over the deviations and taken off
// them, here and again in the backward pass, whose mean has been rounded to a float32 (one more sum across lanes: 7.0 -> 7.6 us
// forward for 120000 rows of 24 float32, 42 -> 44 us backward for 32768 of 1024 bfloat16, others within the noise).
//
// The backward pass adds dy xh and dy of all rows of a group in registers (a lane keeps its columns from row to row);
// the groups of a block are added through LDS, the blocks by a second kernel, each in a fixed order: no atomics, the
// same bits from call to call.  Rows of more vectors than a block holds in registers -- 2048, of 16 bytes where the row's
// length and alignment allow and else of less, down to one value -- are read four times, which the cache serves, and
// their weight gradients are summed by columns.
//
// Measured: 32768 rows of 1024 bfloat16 23 us forward (134 MB, 5.8 TB/s: some of it stays in the last cache) and 43 + 4 us
// backward (201 MB, 4.7 TB/s, and the join); 120000 rows of 24 float32 7.6 us (23 MB); 2048 rows of 900 float32 5.5 us
// forward, 13.5 + 3.9 us backward: 512 blocks of one row a wave, whose sums are 3.7 MB written and read again beside the 22 MB.
// Rows too long for registers: 2048 of 8191 bfloat16 47 us forward and 63 backward, of 8192 (in registers) 16 and 48.

#include "sequence_device.h"

namespace vad {
namespace {
using namespace sq;

constexpr int kThreads = 256;

template <typename T, int VE>
struct Vec {
    typedef T type __attribute__((ext_vector_type(VE)));
};
template <typename T>
struct Vec<T, 1> {
    typedef T type;
};

template <typename T, int VE>
using Raw = typename Vec<T, VE>::type;

template <typename T, int VE>
__device__ __forceinline__ void unpack(Raw<T, VE> x, float (&v)[VE]) {
    T e[VE];
    __builtin_memcpy(e, &x, sizeof(x));
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = (float)e[i];
}
template <typename T, int VE>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VE]) {
    T e[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) e[i] = (T)v[i];
    typename Vec<T, VE>::type x;
    __builtin_memcpy(&x, e, sizeof(x));
    *reinterpret_cast<typename Vec<T, VE>::type*>(p) = x;
}

// Weights are float32 or of x's type.  VE of them from column c on, `absent` where there are none: whole words where the
// pointer allows (columns come in multiples of VE).
template <typename T>
struct Params {
    const void* w;
    const void* b;
    bool f32;
    __device__ __forceinline__ float at(const void* p, int c) const {
        return f32 ? static_cast<const float*>(p)[c] : (float)static_cast<const T*>(p)[c];
    }
    template <int VE>
    __device__ __forceinline__ void load(const void* p, int c, int cols, float absent, float (&v)[VE]) const {
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] = absent;
        if (!p || c >= cols) return;
        if (f32) {
            const float* q = static_cast<const float*>(p) + c;
            if (VE % 4 == 0) {
#pragma unroll
                for (int i = 0; i < VE; i += 4) {
                    const u32x4 r = *reinterpret_cast<const u32x4_any*>(q + i);
                    __builtin_memcpy(v + i, &r, 16);
                }
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i) v[i] = q[i];
            }
        } else {
            const T* q = static_cast<const T*>(p) + c;
            if (sizeof(T) == 2 && VE % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 4 == 0) {
                const u32x4 r = *reinterpret_cast<const u32x4_any*>(q);
                T e[VE];
                __builtin_memcpy(e, &r, 16);
#pragma unroll
                for (int i = 0; i < VE; ++i) v[i] = (float)e[i];
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i) v[i] = (float)q[i];
            }
        }
    }
};

__device__ __forceinline__ float group_sum(float v, int lanes, float* scratch) {
    if (lanes <= 64) return lanes_sum(v, lanes);
    // a whole block: the same order for every thread
    v = lanes_sum(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) v += scratch[i];
    return v;
}

struct Rows {
    int64_t rows, x_stride;
    int cols, lanes;      // lanes: threads that share a row (a power of two up to 64, or kThreads)
    float eps;
};

template <typename T, int VE, int NV>
__global__ __launch_bounds__(kThreads) void layer_norm_kernel(const T* __restrict__ x, Rows a, Params<T> pr, T* __restrict__ y,
                                                              float* __restrict__ stats) {
    __shared__ float scratch[kThreads / 64];
    const int l = threadIdx.x & (a.lanes - 1);
    const int per_block = kThreads / a.lanes;
    const int64_t step = (int64_t)gridDim.x * per_block;
    float w[NV][VE], b[NV][VE];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        pr.load(pr.w, (l + n * a.lanes) * VE, a.cols, 1.0f, w[n]);
        pr.load(pr.b, (l + n * a.lanes) * VE, a.cols, 0.0f, b[n]);
    }
    Raw<T, VE> ahead[NV];                      // the next row is on its way while this one is worked on
    const auto fetch = [&](int64_t base) {
        const int64_t row = base + threadIdx.x / a.lanes;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (l + n * a.lanes) * VE;
            if (row < a.rows && c < a.cols) ahead[n] = *reinterpret_cast<const Raw<T, VE>*>(x + row * a.x_stride + c);
        }
    };
#pragma unroll
    for (int n = 0; n < NV; ++n) ahead[n] = Raw<T, VE>{};
    fetch((int64_t)blockIdx.x * per_block);
    const float inv = 1.0f / (float)a.cols;
    // every group of a block makes the same number of turns: a whole-block group meets barriers
    for (int64_t base = (int64_t)blockIdx.x * per_block; base < a.rows; base += step) {
        const int64_t row = base + threadIdx.x / a.lanes;
        const bool live = row < a.rows;
        float v[NV][VE];
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NV; ++n) unpack<T, VE>(ahead[n], v[n]);
        fetch(base + step);
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < VE; ++e) sum += v[n][e];
        const float mean = group_sum(sum, a.lanes, scratch) / (float)a.cols;
        float left = 0.0f, sq = 0.0f;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if ((l + n * a.lanes) * VE < a.cols) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    v[n][e] -= mean;
                    left += v[n][e];
                }
            }
        }
        left = group_sum(left, a.lanes, scratch) * inv;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if ((l + n * a.lanes) * VE < a.cols) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    v[n][e] -= left;
                    sq = fmaf(v[n][e], v[n][e], sq);
                }
            }
        }
        const float rstd = 1.0f / sqrtf(group_sum(sq, a.lanes, scratch) / (float)a.cols + a.eps);
        if (!live) continue;
        if (stats && l == 0) {
            stats[2 * row] = mean + left;
            stats[2 * row + 1] = rstd;
        }
        T* yr = y + row * a.cols;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (l + n * a.lanes) * VE;
            if (c < a.cols) {
#pragma unroll
                for (int e = 0; e < VE; ++e) v[n][e] = fmaf(v[n][e] * rstd, w[n][e], b[n][e]);
                store_vec<T, VE>(yr + c, v[n]);
            }
        }
    }
}

// dx of every row, and per block the sums over its rows of dy xh (part[block][0][c]) and of dy (part[block][1][c]).
template <typename T, int VE, int NV>
__global__ __launch_bounds__(kThreads) void layer_norm_grad_kernel(const T* __restrict__ x, const T* __restrict__ dy, Rows a,
                                                                   int64_t dy_stride, Params<T> pr, const float* __restrict__ stats,
                                                                   T* __restrict__ dx, float* __restrict__ part) {
    __shared__ float scratch[kThreads / 64];
    extern __shared__ float sums[];            // 2 * cols floats, where several groups share a block
    const int l = threadIdx.x & (a.lanes - 1);
    const int per_block = kThreads / a.lanes;
    const int64_t step = (int64_t)gridDim.x * per_block;
    float dw[NV][VE], db[NV][VE], w[NV][VE];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        pr.load(pr.w, (l + n * a.lanes) * VE, a.cols, 1.0f, w[n]);
#pragma unroll
        for (int e = 0; e < VE; ++e) dw[n][e] = db[n][e] = 0.0f;
    }
    Raw<T, VE> ahead_x[NV], ahead_g[NV];
    const auto fetch = [&](int64_t base) {
        const int64_t row = base + threadIdx.x / a.lanes;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (l + n * a.lanes) * VE;
            if (row < a.rows && c < a.cols) {
                ahead_x[n] = *reinterpret_cast<const Raw<T, VE>*>(x + row * a.x_stride + c);
                ahead_g[n] = *reinterpret_cast<const Raw<T, VE>*>(dy + row * dy_stride + c);
            }
        }
    };
#pragma unroll
    for (int n = 0; n < NV; ++n) ahead_x[n] = ahead_g[n] = Raw<T, VE>{};
    fetch((int64_t)blockIdx.x * per_block);
    const float inv = 1.0f / (float)a.cols;
    for (int64_t base = (int64_t)blockIdx.x * per_block; base < a.rows; base += step) {
        const int64_t row = base + threadIdx.x / a.lanes;
        const bool live = row < a.rows;
        const float mean = live ? stats[2 * row] : 0.0f, rstd = live ? stats[2 * row + 1] : 0.0f;
        float v[NV][VE], g[NV][VE];
        float left = 0.0f, s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            unpack<T, VE>(ahead_x[n], v[n]);
            unpack<T, VE>(ahead_g[n], g[n]);
        }
        fetch(base + step);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (live && (l + n * a.lanes) * VE < a.cols) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    v[n][e] -= mean;
                    left += v[n][e];
                }
            }
        }
        left = group_sum(left, a.lanes, scratch) * inv;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (live && (l + n * a.lanes) * VE < a.cols) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    v[n][e] = (v[n][e] - left) * rstd;
                    dw[n][e] = fmaf(g[n][e], v[n][e], dw[n][e]);
                    db[n][e] += g[n][e];
                    g[n][e] *= w[n][e];
                    s1 += g[n][e];
                    s2 = fmaf(g[n][e], v[n][e], s2);
                }
            }
        }
        s1 = group_sum(s1, a.lanes, scratch) * inv;
        s2 = group_sum(s2, a.lanes, scratch) * inv;
        if (!live || !dx) continue;
        // Of two columns g - mean g is a multiple of xh, and eps / (var + eps) of it is left: formed as that, not as a difference.
        const bool pair = a.cols == 2;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (l + n * a.lanes) * VE;
            if (c < a.cols) {
#pragma unroll
                for (int e = 0; e < VE; ++e) g[n][e] = rstd * (pair ? (g[n][e] - s1) * (a.eps * rstd * rstd) : g[n][e] - s1 - v[n][e] * s2);
                store_vec<T, VE>(dx + row * a.cols + c, g[n]);
            }
        }
    }
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * 2 * a.cols;
    if (a.lanes == kThreads) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const int c = (l + n * a.lanes) * VE + e;
                if (c < a.cols) {
                    out[c] = dw[n][e];
                    out[a.cols + c] = db[n][e];
                }
            }
        return;
    }
    // groups within a wave hold the same columns at the same l: add them by shuffles, then the waves in turn through LDS
    for (int o = a.lanes; o < 64; o <<= 1)
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                dw[n][e] += __shfl_xor(dw[n][e], o);
                db[n][e] += __shfl_xor(db[n][e], o);
            }
    const int wave = threadIdx.x >> 6;
    for (int turn = 0; turn < kThreads / 64; ++turn) {
        if (wave == turn && (threadIdx.x & 63) < a.lanes) {
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const int c = (l + n * a.lanes) * VE + e;
                    if (c < a.cols) {
                        sums[c] = (turn ? sums[c] : 0.0f) + dw[n][e];
                        sums[a.cols + c] = (turn ? sums[a.cols + c] : 0.0f) + db[n][e];
                    }
                }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * a.cols; c += kThreads) out[c] = sums[c];
}

// What is left of a row's mean behind `mean`, by a whole block.
template <typename T>
__device__ __forceinline__ float mean_left(const T* x, float mean, int cols, float* scratch) {
    float sum = 0.0f;
    for (int c = threadIdx.x; c < cols; c += kThreads) sum += (float)x[c] - mean;
    return group_sum(sum, kThreads, scratch) / (float)cols;
}

// Rows of more vectors than a block holds in registers: four passes over the row.
template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_long_kernel(const T* __restrict__ x, Rows a, Params<T> pr, T* __restrict__ y,
                                                                   float* __restrict__ stats) {
    __shared__ float scratch[kThreads / 64];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* xr = x + row * a.x_stride;
        float sum = 0.0f, sq = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) sum += (float)xr[c];
        const float mean = group_sum(sum, kThreads, scratch) / (float)a.cols, left = mean_left(xr, mean, a.cols, scratch);
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const float d = (float)xr[c] - mean - left;
            sq = fmaf(d, d, sq);
        }
        const float rstd = 1.0f / sqrtf(group_sum(sq, kThreads, scratch) / (float)a.cols + a.eps);
        if (stats && threadIdx.x == 0) {
            stats[2 * row] = mean + left;
            stats[2 * row + 1] = rstd;
        }
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            y[row * a.cols + c] = (T)fmaf(((float)xr[c] - mean - left) * rstd, pr.w ? pr.at(pr.w, c) : 1.0f, pr.b ? pr.at(pr.b, c) : 0.0f);
        }
    }
}

// left[row] for the weights' gradients of long rows.
template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_left_kernel(const T* __restrict__ x, Rows a, const float* __restrict__ stats,
                                                                   float* __restrict__ left) {
    __shared__ float scratch[kThreads / 64];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float m = mean_left(x + row * a.x_stride, stats[2 * row], a.cols, scratch);
        if (threadIdx.x == 0) left[row] = m;
    }
}

// left: that of every row where it is known, else null.
template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_grad_long_kernel(const T* __restrict__ x, const T* __restrict__ dy, Rows a,
                                                                        int64_t dy_stride, Params<T> pr, const float* __restrict__ stats,
                                                                        const float* __restrict__ left, T* __restrict__ dx) {
    __shared__ float scratch[kThreads / 64];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* xr = x + row * a.x_stride;
        const T* gr = dy + row * dy_stride;
        const float mean = stats[2 * row], rstd = stats[2 * row + 1], rest = left ? left[row] : mean_left(xr, mean, a.cols, scratch);
        float s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const float g = (float)gr[c] * (pr.w ? pr.at(pr.w, c) : 1.0f);
            s1 += g;
            s2 = fmaf(g, ((float)xr[c] - mean - rest) * rstd, s2);
        }
        s1 = group_sum(s1, kThreads, scratch) / (float)a.cols;
        s2 = group_sum(s2, kThreads, scratch) / (float)a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const float g = (float)gr[c] * (pr.w ? pr.at(pr.w, c) : 1.0f);
            dx[row * a.cols + c] = (T)(rstd * (g - s1 - ((float)xr[c] - mean - rest) * rstd * s2));
        }
    }
}

// Weight gradients of long rows: a thread owns a column, a block (x, y) 256 columns and every gridDim.y-th row.
template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_columns_kernel(const T* __restrict__ x, const T* __restrict__ dy, Rows a,
                                                                      int64_t dy_stride, const float* __restrict__ stats,
                                                                      const float* __restrict__ left, float* __restrict__ part) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.cols) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = (float)dy[row * dy_stride + c];
        dw = fmaf(g, ((float)x[row * a.x_stride + c] - stats[2 * row] - left[row]) * stats[2 * row + 1], dw);
        db += g;
    }
    float* out = part + (int64_t)blockIdx.y * 2 * a.cols;
    out[c] = dw;
    out[a.cols + c] = db;
}

// Adds the blocks' sums: a block owns 16 columns of one of the two gradients, 16 threads a column in strides.
template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_join_kernel(const float* __restrict__ part, int parts, int cols, bool f32,
                                                                   void* __restrict__ dw, void* __restrict__ db) {
    __shared__ float s[16][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4, which = blockIdx.y;
    float v = 0.0f;
    if (c < cols)
#pragma unroll 8
        for (int p = r; p < parts; p += 16) v += part[((int64_t)p * 2 + which) * cols + c];
    s[r][threadIdx.x & 15] = v;
    __syncthreads();
    if (r == 0 && c < cols) {
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) v += s[i][threadIdx.x];
        void* o = which ? db : dw;
        if (!o) return;
        if (f32)
            static_cast<float*>(o)[c] = v;
        else
            static_cast<T*>(o)[c] = (T)v;
    }
}

constexpr int kMaxVecs = 8;
constexpr int kMaxParts = 512;

// How a row is spread: vectors of `ve` elements (the widest up to 16 bytes that divides the row and its alignment), `nv`
// of them per lane, `lanes` lanes; nv == 0: too long for registers.
struct Shape {
    int ve, nv, lanes;
};
Shape row_shape(int cols, int elem, uintptr_t align) {
    Shape s;
    s.ve = 16 / elem;
    while (s.ve > 1 && (cols % s.ve || align % (s.ve * elem))) s.ve >>= 1;
    const int vecs = (cols + s.ve - 1) / s.ve;
    s.lanes = 1;
    while (s.lanes < 64 && s.lanes < vecs) s.lanes <<= 1;
    if (vecs > 64 * 4) s.lanes = kThreads;
    s.nv = 1;
    while (s.nv < kMaxVecs && s.nv * s.lanes < vecs) s.nv <<= 1;
    if (s.nv * s.lanes < vecs) s.nv = 0;
    return s;
}

int64_t row_blocks(int64_t rows, int lanes, int64_t most) {
    const int64_t per = kThreads / lanes, n = (rows + per - 1) / per;
    return n < 1 ? 1 : (n < most ? n : most);
}

int grad_parts(int64_t rows, const Shape& s) { return (int)row_blocks(rows, s.nv ? s.lanes : kThreads, s.nv ? kMaxParts : 64); }

#define VAD_LN_NV(KERNEL, T, VE, ...)                                                                        \
    do {                                                                                                     \
        if (sh.nv == 1) hipLaunchKernelGGL((KERNEL<T, VE, 1>), __VA_ARGS__);                                 \
        else if (sh.nv == 2) hipLaunchKernelGGL((KERNEL<T, VE, 2>), __VA_ARGS__);                            \
        else if (sh.nv == 4) hipLaunchKernelGGL((KERNEL<T, VE, 4>), __VA_ARGS__);                            \
        else hipLaunchKernelGGL((KERNEL<T, VE, 8>), __VA_ARGS__);                                            \
    } while (0)
#define VAD_LN_LAUNCH(KERNEL, T, ...)                                                                        \
    do {                                                                                                     \
        if (sh.ve == 1) VAD_LN_NV(KERNEL, T, 1, __VA_ARGS__);                                                \
        else if (sh.ve == 2) VAD_LN_NV(KERNEL, T, 2, __VA_ARGS__);                                           \
        else if (sh.ve == 4) VAD_LN_NV(KERNEL, T, 4, __VA_ARGS__);                                           \
        else VAD_LN_NV(KERNEL, T, (16 / (int)sizeof(T)), __VA_ARGS__);                                       \
    } while (0)

template <typename T>
int run_forward(const void* x, int64_t rows, int64_t cols, int64_t x_stride, const void* w, const void* b, int w_f32, float eps,
                void* y, float* stats, hipStream_t st) {
    const Shape sh = row_shape((int)cols, sizeof(T),
                               reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | (uintptr_t)(x_stride * sizeof(T)));
    Rows a = {rows, x_stride, (int)cols, sh.lanes, eps};
    Params<T> pr = {w, b, w_f32 != 0};
    const T* xp = static_cast<const T*>(x);
    T* yp = static_cast<T*>(y);
    if (sh.nv) {
        const dim3 grid((unsigned)row_blocks(rows, sh.lanes, 256 * 8));
        VAD_LN_LAUNCH(layer_norm_kernel, T, grid, dim3(kThreads), 0, st, xp, a, pr, yp, stats);
    } else {
        hipLaunchKernelGGL((layer_norm_long_kernel<T>), dim3((unsigned)row_blocks(rows, kThreads, 256 * 8)), dim3(kThreads), 0, st,
                           xp, a, pr, yp, stats);
    }
    VAD_HIP_CHECK(hipGetLastError());
    return VAD_OK;
}

template <typename T>
int run_backward(const void* x, const void* dy, int64_t rows, int64_t cols, int64_t x_stride, int64_t dy_stride, const void* w,
                 int w_f32, float eps, const float* stats, void* dx, void* dw, void* db, float* part, hipStream_t st) {
    const Shape sh = row_shape((int)cols, sizeof(T),
                               reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx) |
                                   (uintptr_t)(x_stride * sizeof(T)) | (uintptr_t)(dy_stride * sizeof(T)));
    Rows a = {rows, x_stride, (int)cols, sh.lanes, eps};
    Params<T> pr = {w, nullptr, w_f32 != 0};
    const T* xp = static_cast<const T*>(x);
    const T* gp = static_cast<const T*>(dy);
    T* dxp = static_cast<T*>(dx);
    const bool sums = dw || db;
    const int parts = rows ? grad_parts(rows, sh) : 0;      // no rows: the joining kernel writes zeros
    if (rows == 0) {
    } else if (sh.nv) {
        // at most 64 lanes * 4 vectors * 8 elements = 2048 columns share a block: 16 KB of sums
        const size_t lds = sums && sh.lanes < kThreads ? 2 * (size_t)cols * sizeof(float) : 0;
        VAD_LN_LAUNCH(layer_norm_grad_kernel, T, dim3((unsigned)parts), dim3(kThreads), lds, st, xp, gp, a, dy_stride, pr, stats, dxp,
                      sums ? part : nullptr);
    } else {
        const dim3 grid((unsigned)row_blocks(rows, kThreads, 256 * 8));
        float* left = sums ? part + (int64_t)parts * 2 * cols : nullptr;
        if (sums) hipLaunchKernelGGL((layer_norm_left_kernel<T>), grid, dim3(kThreads), 0, st, xp, a, stats, left);
        if (dx) hipLaunchKernelGGL((layer_norm_grad_long_kernel<T>), grid, dim3(kThreads), 0, st, xp, gp, a, dy_stride, pr, stats, left, dxp);
        if (sums)
            hipLaunchKernelGGL((layer_norm_columns_kernel<T>), dim3((unsigned)((cols + kThreads - 1) / kThreads), (unsigned)parts),
                               dim3(kThreads), 0, st, xp, gp, a, dy_stride, stats, left, part);
    }
    VAD_HIP_CHECK(hipGetLastError());
    if (sums) {
        hipLaunchKernelGGL((layer_norm_join_kernel<T>), dim3((unsigned)((cols + 15) / 16), 2), dim3(kThreads), 0, st, part, parts,
                           (int)cols, w_f32 != 0, dw, db);
        VAD_HIP_CHECK(hipGetLastError());
    }
    return VAD_OK;
}

}  // namespace
}  // namespace vad

extern "C" size_t vad_layer_norm_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    // rows of more than 2048 values may be too long for registers: what is left of their means as well, a float a row
    const size_t left = cols > vad::kMaxVecs * vad::kThreads ? (size_t)rows : 0;
    return ((size_t)(rows < vad::kMaxParts ? rows : vad::kMaxParts) * 2 * (size_t)cols + left) * sizeof(float);
}

extern "C" int vad_layer_norm_forward(const void* x_dev, int64_t rows, int64_t cols, int64_t x_stride, const void* weight_dev,
                                      const void* bias_dev, int dtype, int weight_dtype, float eps, void* y_dev, float* stats_dev,
                                      void* stream) {
    using namespace vad;
    VAD_REQUIRE(dtype == VAD_DTYPE_F32 || dtype == VAD_DTYPE_BF16, "dtype must be VAD_DTYPE_F32 or VAD_DTYPE_BF16, got %d", dtype);
    VAD_REQUIRE(weight_dtype == VAD_DTYPE_F32 || weight_dtype == dtype, "weight_dtype must be VAD_DTYPE_F32 or dtype");
    VAD_REQUIRE(rows >= 0 && cols >= 1 && cols <= (1 << 28) && x_stride >= 0, "rows %lld, cols %lld or x_stride %lld out of range",
                (long long)rows, (long long)cols, (long long)x_stride);
    VAD_REQUIRE(eps >= 0.0f && eps < INFINITY, "eps must be finite and not negative");
    if (rows == 0) return VAD_OK;
    VAD_REQUIRE(x_dev && y_dev, "null pointer argument");
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == VAD_DTYPE_F32
               ? run_forward<float>(x_dev, rows, cols, x_stride, weight_dev, bias_dev, weight_dtype == VAD_DTYPE_F32, eps, y_dev,
                                    stats_dev, st)
               : run_forward<__bf16>(x_dev, rows, cols, x_stride, weight_dev, bias_dev, weight_dtype == VAD_DTYPE_F32, eps, y_dev,
                                     stats_dev, st);
}

extern "C" int vad_layer_norm_backward(const void* x_dev, const void* dy_dev, int64_t rows, int64_t cols, int64_t x_stride,
                                       int64_t dy_stride, const void* weight_dev, int dtype, int weight_dtype, float eps,
                                       const float* stats_dev, void* dx_dev, void* dweight_dev, void* dbias_dev,
                                       void* workspace_dev, size_t workspace_bytes, void* stream) {
    using namespace vad;
    VAD_REQUIRE(dtype == VAD_DTYPE_F32 || dtype == VAD_DTYPE_BF16, "dtype must be VAD_DTYPE_F32 or VAD_DTYPE_BF16, got %d", dtype);
    VAD_REQUIRE(weight_dtype == VAD_DTYPE_F32 || weight_dtype == dtype, "weight_dtype must be VAD_DTYPE_F32 or dtype");
    VAD_REQUIRE(rows >= 0 && cols >= 1 && cols <= (1 << 28) && x_stride >= 0 && dy_stride >= 0,
                "rows %lld, cols %lld, x_stride %lld or dy_stride %lld out of range", (long long)rows, (long long)cols,
                (long long)x_stride, (long long)dy_stride);
    VAD_REQUIRE(eps >= 0.0f && eps < INFINITY, "eps must be finite and not negative");
    VAD_REQUIRE(rows == 0 || (x_dev && dy_dev && stats_dev), "null pointer argument");
    VAD_REQUIRE((!dweight_dev && !dbias_dev) || workspace_bytes >= vad_layer_norm_workspace_bytes(rows, cols),
                "workspace of %zu bytes is too small", workspace_bytes);
    VAD_REQUIRE((!dweight_dev && !dbias_dev) || rows == 0 || workspace_dev, "null workspace");
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* part = static_cast<float*>(workspace_dev);
    if (rows == 0 && !dweight_dev && !dbias_dev) return VAD_OK;
    return dtype == VAD_DTYPE_F32
               ? run_backward<float>(x_dev, dy_dev, rows, cols, x_stride, dy_stride, weight_dev, weight_dtype == VAD_DTYPE_F32,
                                     eps, stats_dev, dx_dev, dweight_dev, dbias_dev, part, st)
               : run_backward<__bf16>(x_dev, dy_dev, rows, cols, x_stride, dy_stride, weight_dev, weight_dtype == VAD_DTYPE_F32,
                                      eps, stats_dev, dx_dev, dweight_dev, dbias_dev, part, st);
}
