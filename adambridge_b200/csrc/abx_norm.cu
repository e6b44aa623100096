// abx_norm.cu -- layer norm and RMS norm over the last axis, forward and backward (libabx).
//
// Rows of N values, in fp32 whatever the tensors' type, rounded once on the way out:
//   mu = mean x (RMS norm: 0),  r = 1 / sqrt(mean (x - mu)^2 + eps),  h = (x - mu) r,  y = h w + b
//   a = dy w,  dx = r (a - mean a - h mean(a h))  (RMS norm: without mean a),  dw = sum_rows dy h,  db = sum_rows dy
//
// A row stays in registers between its load and its store: the forward pass reads x once and writes y once, the
// backward pass reads x and dy once and writes dx once.  The variance is taken about the mean (a second sum over the
// registers), so no large squares cancel.  A row is owned by part of a warp, a warp or a CTA, by its length; HBM bounds
// all of them.
//
// The weights' gradients are sums over rows: a CTA of the backward kernel goes through many rows and keeps its columns'
// sums in registers, writes them once to a workspace, and a second small launch adds the CTAs' sums in a fixed order.
// No atomics: the same input gives the same bits.  Rows too long for that (the sums would not fit in registers) take
// dx row by row and the sums in a pass of their own over x and dy.
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "../../include/abx.h"
#include "abx_device.cuh"

#define ABX_API extern "C" __attribute__((visibility("default")))

namespace abx {
int set_error(const char* what, cudaError_t e);   // abx_kernels.cu
extern std::atomic<uint64_t> g_launches;
}  // namespace abx

namespace {

using abx::f2u;
using abx::u2f;

struct bf16 { uint16_t bits; };

struct Args {
    const void* x;
    const void* dy;
    const void* w;      // may be null: 1
    const void* b;      // may be null: 0
    void* y;            // forward: y; backward: dx (may be null)
    float* mean;        // forward: may be null
    float* rstd;
    float* partial;     // backward: sums of dy h, then of dy: [2][parts][cols] (null: not wanted)
    int64_t rows, cols;
    int64_t x_stride, dy_stride;   // elements between rows
    int32_t w_bf16;
    int32_t w_vec;      // w and b allow vector loads
    int32_t has_db;
    float eps;
};

// ---- 16 bytes of a row -------------------------------------------------------------------------

template <typename T> struct Vec;
template <> struct Vec<bf16> { static constexpr int V = 8; };
template <> struct Vec<float> { static constexpr int V = 4; };

struct Raw { uint32_t w[4]; };

template <typename T>
__device__ __forceinline__ void unpack(const Raw& r, float (&x)[Vec<T>::V])
{
    if constexpr (Vec<T>::V == 8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[2 * j] = u2f(r.w[j] << 16); x[2 * j + 1] = u2f(r.w[j] & 0xffff0000U); }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = u2f(r.w[j]);
    }
}

template <typename T>
__device__ __forceinline__ Raw pack(const float (&x)[Vec<T>::V])
{
    Raw r;
    if constexpr (Vec<T>::V == 8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r.w[j] = abx::pack_bf16_rne(x[2 * j], x[2 * j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) r.w[j] = f2u(x[j]);
    }
    return r;
}

// Vector i of a thread covers the columns column<VEC>(i, k), k < V: neighbours where rows allow vector access, else
// LANES apart, so that a warp's scalar accesses are neighbours instead.
template <bool VEC, int LANES, int V>
__device__ __forceinline__ int64_t column(int lane, int i, int k)
{
    return VEC ? ((int64_t)i * LANES + lane) * V + k : ((int64_t)i * V + k) * LANES + lane;
}

template <typename T, bool VEC, int LANES>
__device__ __forceinline__ Raw load(const T* row, int64_t cols, int lane, int i)
{
    constexpr int V = Vec<T>::V;
    Raw r = {{0U, 0U, 0U, 0U}};
    if constexpr (VEC) {
        const int64_t c = column<VEC, LANES, V>(lane, i, 0);
        if (c < cols) {
            const uint4 q = *reinterpret_cast<const uint4*>(row + c);
            r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int64_t c = column<VEC, LANES, V>(lane, i, k);
            if (c < cols) {
                if constexpr (V == 8) r.w[k >> 1] |= (uint32_t)row[c].bits << (16 * (k & 1));
                else r.w[k] = f2u(row[c]);
            }
        }
    }
    return r;
}

template <typename T, bool VEC, int LANES>
__device__ __forceinline__ void store(T* row, int64_t cols, int lane, int i, const float (&x)[Vec<T>::V])
{
    constexpr int V = Vec<T>::V;
    const Raw r = pack<T>(x);
    if constexpr (VEC) {
        const int64_t c = column<VEC, LANES, V>(lane, i, 0);
        if (c < cols) *reinterpret_cast<uint4*>(row + c) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int64_t c = column<VEC, LANES, V>(lane, i, k);
            if (c < cols) {
                if constexpr (V == 8) row[c].bits = (uint16_t)(r.w[k >> 1] >> (16 * (k & 1)));
                else row[c] = x[k];
            }
        }
    }
}

// V values of a weight vector of either type (`fill` where there is none)
template <bool VEC, int LANES, int V>
__device__ __forceinline__ void load_w(const void* w, const Args& a, int lane, int i, float fill, float (&x)[V])
{
    const int64_t c0 = column<VEC, LANES, V>(lane, i, 0);
    if (w == nullptr) {
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = fill;
    } else if (VEC && a.w_vec && c0 < a.cols) {
        if (a.w_bf16) {
            const uint16_t* p = static_cast<const uint16_t*>(w) + c0;
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                const uint2 q = reinterpret_cast<const uint2*>(p)[h];
                x[4 * h] = u2f(q.x << 16); x[4 * h + 1] = u2f(q.x & 0xffff0000U);
                x[4 * h + 2] = u2f(q.y << 16); x[4 * h + 3] = u2f(q.y & 0xffff0000U);
            }
        } else {
            const float* p = static_cast<const float*>(w) + c0;
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                const float4 q = reinterpret_cast<const float4*>(p)[h];
                x[4 * h] = q.x; x[4 * h + 1] = q.y; x[4 * h + 2] = q.z; x[4 * h + 3] = q.w;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int64_t c = column<VEC, LANES, V>(lane, i, k);
            x[k] = 0.0f;
            if (c < a.cols)
                x[k] = a.w_bf16 ? u2f((uint32_t)static_cast<const uint16_t*>(w)[c] << 16) : static_cast<const float*>(w)[c];
        }
    }
}

// ---- sums over the threads that own a row -----------------------------------------------------------

// K sums at once, each over LANES threads; every thread gets them.  `buf` alternates between two halves, so one
// barrier per call is enough (a thread is at most one call ahead of another).
template <int LANES, int K>
__device__ __forceinline__ void row_sum(float (&s)[K], float* buf, int& half)
{
#pragma unroll
    for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] += __shfl_xor_sync(0xffffffffU, s[k], o);
    if constexpr (LANES > 32) {
        constexpr int kW = LANES / 32;
        float* const b = buf + half * (2 * kW);
        half ^= 1;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) b[k * kW + (threadIdx.x >> 5)] = s[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            s[k] = (threadIdx.x & 31) < kW ? b[k * kW + (threadIdx.x & 31)] : 0.0f;
#pragma unroll
            for (int o = (kW < 32 ? kW : 32) / 2; o > 0; o >>= 1) s[k] += __shfl_xor_sync(0xffffffffU, s[k], o);
            if constexpr (kW < 32) s[k] = __shfl_sync(0xffffffffU, s[k], 0);
        }
    }
}

template <int LANES> __host__ __device__ constexpr int threads_of() { return LANES > 32 ? LANES : 256; }

// ---- forward -----------------------------------------------------------------------------------------

template <typename T, bool RMS, bool VEC, int LANES, int NV>
__global__ void __launch_bounds__(threads_of<LANES>()) forward_kernel(const __grid_constant__ Args a)
{
    constexpr int V = Vec<T>::V, kRows = threads_of<LANES>() / LANES;
    __shared__ float buf[LANES > 32 ? 4 * (LANES / 32) : 1];
    int half = 0;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.0f / (float)a.cols;
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < a.rows; row0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = row0 + group;
        const bool live = row < a.rows;          // a group without a row still takes part in the shuffles
        const T* const x = static_cast<const T*>(a.x) + (live ? row : row0) * a.x_stride;
        Raw raw[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = load<T, VEC, LANES>(x, a.cols, lane, i);
        float mean = 0.0f;
        if constexpr (!RMS) {
            float s[1] = {0.0f};
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float v[V];
                unpack<T>(raw[i], v);
#pragma unroll
                for (int k = 0; k < V; ++k) s[0] += v[k];
            }
            row_sum<LANES, 1>(s, buf, half);
            mean = s[0] * inv;
        }
        float q[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float v[V];
            unpack<T>(raw[i], v);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = RMS || column<VEC, LANES, V>(lane, i, k) < a.cols ? v[k] - mean : 0.0f;
                q[0] = __fmaf_rn(d, d, q[0]);
            }
        }
        row_sum<LANES, 1>(q, buf, half);
        const float rstd = __frcp_rn(__fsqrt_rn(__fmaf_rn(q[0], inv, a.eps)));
        if (!live) continue;
        T* const y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float v[V], w[V], b[V];
            unpack<T>(raw[i], v);
            load_w<VEC, LANES, V>(a.w, a, lane, i, 1.0f, w);
            if constexpr (RMS) {
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = (v[k] * rstd) * w[k];
            } else {
                load_w<VEC, LANES, V>(a.b, a, lane, i, 0.0f, b);
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = __fmaf_rn((v[k] - mean) * rstd, w[k], b[k]);
            }
            store<T, VEC, LANES>(y, a.cols, lane, i, v);
        }
        if (lane == 0) {
            if (!RMS && a.mean != nullptr) a.mean[row] = mean;
            if (a.rstd != nullptr) a.rstd[row] = rstd;
        }
    }
}

// Rows longer than a CTA's registers: three passes over the row, the later ones from the caches.
constexpr int kLong = 1024;

template <typename T, bool RMS, bool VEC>
__global__ void __launch_bounds__(kLong) forward_long(const __grid_constant__ Args a)
{
    constexpr int V = Vec<T>::V;
    __shared__ float buf[4 * (kLong / 32)];
    int half = 0;
    const int lane = threadIdx.x;
    const float inv = 1.0f / (float)a.cols;
    const int steps = (int)((a.cols + (int64_t)kLong * V - 1) / ((int64_t)kLong * V));
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(a.x) + row * a.x_stride;
        float mean = 0.0f;
        if constexpr (!RMS) {
            float s[1] = {0.0f};
            for (int i = 0; i < steps; ++i) {
                float v[V];
                unpack<T>(load<T, VEC, kLong>(x, a.cols, lane, i), v);
#pragma unroll
                for (int k = 0; k < V; ++k) s[0] += v[k];
            }
            row_sum<kLong, 1>(s, buf, half);
            mean = s[0] * inv;
        }
        float q[1] = {0.0f};
        for (int i = 0; i < steps; ++i) {
            float v[V];
            unpack<T>(load<T, VEC, kLong>(x, a.cols, lane, i), v);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = RMS || column<VEC, kLong, V>(lane, i, k) < a.cols ? v[k] - mean : 0.0f;
                q[0] = __fmaf_rn(d, d, q[0]);
            }
        }
        row_sum<kLong, 1>(q, buf, half);
        const float rstd = __frcp_rn(__fsqrt_rn(__fmaf_rn(q[0], inv, a.eps)));
        T* const y = static_cast<T*>(a.y) + row * a.cols;
        for (int i = 0; i < steps; ++i) {
            float v[V], w[V], b[V];
            unpack<T>(load<T, VEC, kLong>(x, a.cols, lane, i), v);
            load_w<VEC, kLong, V>(a.w, a, lane, i, 1.0f, w);
            load_w<VEC, kLong, V>(a.b, a, lane, i, 0.0f, b);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = __fmaf_rn((v[k] - mean) * rstd, w[k], b[k]);
            store<T, VEC, kLong>(y, a.cols, lane, i, v);
        }
        if (lane == 0) {
            if (!RMS && a.mean != nullptr) a.mean[row] = mean;
            if (a.rstd != nullptr) a.rstd[row] = rstd;
        }
    }
}

// ---- backward ----------------------------------------------------------------------------------------

// dx of every row, and this CTA's part of dw and db over its rows.
template <typename T, bool RMS, bool VEC, int LANES, int NV>
__global__ void __launch_bounds__(threads_of<LANES>()) backward_kernel(const __grid_constant__ Args a)
{
    constexpr int V = Vec<T>::V, kThreads = threads_of<LANES>(), kRows = kThreads / LANES;
    constexpr int kSums = RMS ? 1 : 2;
    __shared__ float buf[LANES > 32 ? 4 * (LANES / 32) : (kThreads / 32) * LANES * NV * V];
    int half = 0;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.0f / (float)a.cols;
    float dw[NV][V], db[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0.0f;
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < a.rows; row0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = row0 + group;
        const bool live = row < a.rows;
        const T* const x = static_cast<const T*>(a.x) + (live ? row : row0) * a.x_stride;
        const T* const dy = static_cast<const T*>(a.dy) + (live ? row : row0) * a.dy_stride;
        Raw rx[NV], rd[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            rx[i] = load<T, VEC, LANES>(x, a.cols, lane, i);
            rd[i] = load<T, VEC, LANES>(dy, a.cols, lane, i);
        }
        const float mean = RMS ? 0.0f : a.mean[live ? row : row0];
        const float rstd = a.rstd[live ? row : row0];
        float s[kSums];
#pragma unroll
        for (int k = 0; k < kSums; ++k) s[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float v[V], d[V], w[V];
            unpack<T>(rx[i], v);
            unpack<T>(rd[i], d);
            load_w<VEC, LANES, V>(a.w, a, lane, i, 1.0f, w);
#pragma unroll
            for (int k = 0; k < V; ++k) {   // beyond the row's end d is 0
                const float h = (v[k] - mean) * rstd, t = d[k] * w[k];
                s[0] = __fmaf_rn(t, h, s[0]);
                if constexpr (!RMS) s[1] += t;
                if (live) {
                    dw[i][k] = __fmaf_rn(d[k], h, dw[i][k]);
                    if constexpr (!RMS) db[i][k] += d[k];
                }
            }
        }
        row_sum<LANES, kSums>(s, buf, half);
        if (!live || a.y == nullptr) continue;
        const float c2 = s[0] * inv, c1 = RMS ? 0.0f : s[kSums - 1] * inv;
        T* const dx = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float v[V], d[V], w[V];
            unpack<T>(rx[i], v);
            unpack<T>(rd[i], d);
            load_w<VEC, LANES, V>(a.w, a, lane, i, 1.0f, w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float h = (v[k] - mean) * rstd;
                float t = d[k] * w[k];
                if constexpr (!RMS) t -= c1;
                v[k] = __fmaf_rn(-h, c2, t) * rstd;
            }
            store<T, VEC, LANES>(dx, a.cols, lane, i, v);
        }
    }
    if (a.partial == nullptr) return;
    float* const out = a.partial + (int64_t)blockIdx.x * a.cols;
    const int64_t second = (int64_t)gridDim.x * a.cols;
#pragma unroll
    for (int which = 0; which < kSums; ++which) {
        if (which == 1 && !a.has_db) break;
        if constexpr (LANES > 32) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const int64_t c = column<VEC, LANES, V>(lane, i, k);
                    if (c < a.cols) out[which * second + c] = which ? db[i][k] : dw[i][k];
                }
        } else {
            // the groups of a warp by shuffles, then the warps through shared memory, in order
            constexpr int kCols = LANES * NV * V;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    float t = which ? db[i][k] : dw[i][k];
#pragma unroll
                    for (int o = LANES; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffU, t, o);
                    if ((threadIdx.x & 31) < LANES)
                        buf[(threadIdx.x >> 5) * kCols + (int)column<VEC, LANES, V>(lane, i, k)] = t;
                }
            __syncthreads();
            for (int c = threadIdx.x; c < kCols && c < a.cols; c += kThreads) {
                float t = 0.0f;
#pragma unroll
                for (int j = 0; j < kThreads / 32; ++j) t += buf[j * kCols + c];
                out[which * second + c] = t;
            }
        }
    }
}

// dx of long rows.
template <typename T, bool RMS, bool VEC>
__global__ void __launch_bounds__(kLong) backward_long(const __grid_constant__ Args a)
{
    constexpr int V = Vec<T>::V;
    constexpr int kSums = RMS ? 1 : 2;
    __shared__ float buf[4 * (kLong / 32)];
    int half = 0;
    const int lane = threadIdx.x;
    const float inv = 1.0f / (float)a.cols;
    const int steps = (int)((a.cols + (int64_t)kLong * V - 1) / ((int64_t)kLong * V));
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* const dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
        const float mean = RMS ? 0.0f : a.mean[row], rstd = a.rstd[row];
        float s[kSums];
#pragma unroll
        for (int k = 0; k < kSums; ++k) s[k] = 0.0f;
        for (int i = 0; i < steps; ++i) {
            float v[V], d[V], w[V];
            unpack<T>(load<T, VEC, kLong>(x, a.cols, lane, i), v);
            unpack<T>(load<T, VEC, kLong>(dy, a.cols, lane, i), d);
            load_w<VEC, kLong, V>(a.w, a, lane, i, 1.0f, w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float t = d[k] * w[k];
                s[0] = __fmaf_rn(t, (v[k] - mean) * rstd, s[0]);
                if constexpr (!RMS) s[1] += t;
            }
        }
        row_sum<kLong, kSums>(s, buf, half);
        const float c2 = s[0] * inv, c1 = RMS ? 0.0f : s[kSums - 1] * inv;
        T* const dx = static_cast<T*>(a.y) + row * a.cols;
        for (int i = 0; i < steps; ++i) {
            float v[V], d[V], w[V];
            unpack<T>(load<T, VEC, kLong>(x, a.cols, lane, i), v);
            unpack<T>(load<T, VEC, kLong>(dy, a.cols, lane, i), d);
            load_w<VEC, kLong, V>(a.w, a, lane, i, 1.0f, w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float h = (v[k] - mean) * rstd;
                v[k] = __fmaf_rn(-h, c2, d[k] * w[k] - c1) * rstd;
            }
            store<T, VEC, kLong>(dx, a.cols, lane, i, v);
        }
    }
}

// The sums of long rows: a CTA takes 32 threads' columns (blockIdx.x) of a run of rows (blockIdx.y), 8 rows at a time.
constexpr int kSumRows = 8;

template <typename T, bool RMS, bool VEC>
__global__ void __launch_bounds__(32 * kSumRows) sums_long(const __grid_constant__ Args a)
{
    constexpr int V = Vec<T>::V, kCols = 32 * V;
    __shared__ float buf[kSumRows * kCols];
    const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c0 = (int64_t)blockIdx.x * kCols, left = a.cols - c0;
    const int64_t first = a.rows * blockIdx.y / gridDim.y, last = a.rows * (blockIdx.y + 1) / gridDim.y;
    float dw[V], db[V];
#pragma unroll
    for (int k = 0; k < V; ++k) dw[k] = db[k] = 0.0f;
    for (int64_t row = first + ty; row < last; row += kSumRows) {
        float v[V], d[V];
        unpack<T>(load<T, VEC, 32>(static_cast<const T*>(a.x) + row * a.x_stride + c0, left, lane, 0), v);
        unpack<T>(load<T, VEC, 32>(static_cast<const T*>(a.dy) + row * a.dy_stride + c0, left, lane, 0), d);
        const float mean = RMS ? 0.0f : a.mean[row], rstd = a.rstd[row];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            dw[k] = __fmaf_rn(d[k], (v[k] - mean) * rstd, dw[k]);
            db[k] += d[k];
        }
    }
    float* const out = a.partial + (int64_t)blockIdx.y * a.cols + c0;
    const int64_t second = (int64_t)gridDim.y * a.cols;
#pragma unroll
    for (int which = 0; which < (RMS ? 1 : 2); ++which) {
        if (which == 1 && !a.has_db) break;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V; ++k) buf[ty * kCols + (int)column<VEC, 32, V>(lane, 0, k)] = which ? db[k] : dw[k];
        __syncthreads();
        for (int c = threadIdx.x; c < kCols && c < left; c += 32 * kSumRows) {
            float t = 0.0f;
#pragma unroll
            for (int j = 0; j < kSumRows; ++j) t += buf[j * kCols + c];
            out[which * second + c] = t;
        }
    }
}

// dw (blockIdx.y 0) and db (1) from the parts: 32 columns per CTA, 8 threads per column, in a fixed order.
struct FinishArgs {
    const float* partial;
    void* out[2];
    int64_t cols;
    int32_t parts;
    int32_t bf16_out;
};

__global__ void __launch_bounds__(256) finish_sums(const __grid_constant__ FinishArgs a)
{
    __shared__ float buf[8][33];
    const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    void* const out = blockIdx.y ? a.out[1] : a.out[0];
    const float* p = a.partial + (int64_t)blockIdx.y * a.parts * a.cols;
    float t = 0.0f;
    if (c < a.cols)
        for (int i = ty; i < a.parts; i += 8) t += p[(int64_t)i * a.cols + c];
    buf[ty][lane] = t;
    __syncthreads();
    if (ty == 0 && c < a.cols) {
#pragma unroll
        for (int j = 1; j < 8; ++j) t += buf[j][lane];
        if (a.bf16_out) static_cast<uint16_t*>(out)[c] = (uint16_t)abx::pack_bf16_rne(t, 0.0f);
        else static_cast<float*>(out)[c] = t;
    }
}

// ---- host side ---------------------------------------------------------------------------------------

bool off(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }
int size_of(int32_t dtype) { return dtype == ABX_DT_BF16 ? 2 : 4; }

int check(const abx_norm* n)
{
    if (!n || n->rows < 0 || n->cols < 1 || !(n->eps >= 0.0f)) return ABX_E_ARG;
    if (n->dtype != ABX_DT_F32 && n->dtype != ABX_DT_BF16) return ABX_E_G_DTYPE;
    if ((n->w || n->b) && n->w_dtype != ABX_DT_F32 && n->w_dtype != ABX_DT_BF16) return ABX_E_P_DTYPE;
    if (n->rms && n->b) return ABX_E_ARG;
    if (n->rows > 0 && !n->x) return ABX_E_NULL_PTR;
    if (off(n->x, size_of(n->dtype)) || off(n->w, size_of(n->w_dtype)) || off(n->b, size_of(n->w_dtype))) return ABX_E_ALIGN;
    return ABX_OK;
}

int sm_count(int* sms)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
    return e == cudaSuccess ? ABX_OK : abx::set_error("launch geometry", e);
}

int launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return abx::set_error(what, e);
    abx::g_launches.fetch_add(1, std::memory_order_relaxed);
    return ABX_OK;
}

Args args_of(const abx_norm& n)
{
    Args a;
    std::memset(&a, 0, sizeof a);
    a.x = n.x; a.w = n.w; a.b = n.b;
    a.rows = n.rows; a.cols = n.cols; a.x_stride = n.x_stride;
    a.w_bf16 = n.w_dtype == ABX_DT_BF16;
    a.w_vec = !off(n.w, 16) && !off(n.b, 16);
    a.eps = n.eps;
    return a;
}

// Whether rows can be accessed in 16-byte vectors.
bool vectors(const abx_norm& n, const void* second, int64_t second_stride, const void* out)
{
    const int v = 16 / size_of(n.dtype);
    return n.cols % v == 0 && n.x_stride % v == 0 && second_stride % v == 0 && !off(n.x, 16) && !off(second, 16) && !off(out, 16);
}

// The shape of the row kernels: vectors per row to threads per row and vectors per thread.
//   up to 128 vectors (1024 bf16 values): part of a warp or a warp, no barrier;  up to `most`: a CTA, two or four
//   vectors per thread;  above: the long form.
template <typename F>
int by_width(int64_t nvec, int64_t most, F&& f)
{
    using std::integral_constant;
#define ABX_ROW(L, N) return f(integral_constant<int, L>{}, integral_constant<int, N>{})
    if (nvec <= 8) ABX_ROW(8, 1);
    if (nvec <= 16) ABX_ROW(16, 1);
    if (nvec <= 32) ABX_ROW(32, 1);
    if (nvec <= 64) ABX_ROW(32, 2);
    if (nvec <= 128) ABX_ROW(32, 4);
    if (nvec <= 256) ABX_ROW(128, 2);
    if (nvec <= 512) ABX_ROW(256, 2);
    if (nvec <= 1024 && most >= 1024) ABX_ROW(512, 2);
    return f(integral_constant<int, 0>{}, integral_constant<int, 0>{});
#undef ABX_ROW
}

template <typename F>
int by_flags(const abx_norm& n, bool vec, F&& f)
{
    using T = std::true_type;
    using N = std::false_type;
    if (n.dtype == ABX_DT_BF16) {
        if (n.rms) return vec ? f(bf16{}, T{}, T{}) : f(bf16{}, T{}, N{});
        return vec ? f(bf16{}, N{}, T{}) : f(bf16{}, N{}, N{});
    }
    if (n.rms) return vec ? f(0.0f, T{}, T{}) : f(0.0f, T{}, N{});
    return vec ? f(0.0f, N{}, T{}) : f(0.0f, N{}, N{});
}

constexpr int64_t kMostVectors = 1024;   // per row in the register kernels
constexpr int kMaxGrid = 1 << 30;

// CTAs of the backward pass (each has a part of the sums): two per SM, or fewer when there are few rows -- a part is
// written and read again, 8 bytes per column, so it should cover some rows.
int backward_parts(const abx_norm& n, int sms)
{
    const int64_t v = 16 / size_of(n.dtype), nvec = (n.cols + v - 1) / v;
    if (nvec > kMostVectors) {   // sums_long: row runs so that all column tiles together fill the SMs
        const int64_t tiles = (nvec + 31) / 32, want = (8 * sms + tiles - 1) / tiles, most = (n.rows + 31) / 32;
        const int64_t p = want < most ? want : most;
        return (int)(p > 0 ? p : 1);
    }
    const int64_t rows = nvec <= 8 ? 32 : nvec <= 16 ? 16 : nvec <= 128 ? 8 : 1;   // per CTA at a time
    const int64_t need = (n.rows + rows - 1) / rows;
    const int64_t most = (nvec <= 256 ? 4 : 2) * (int64_t)sms;
    return (int)(need < most ? (need > 0 ? need : 1) : most);
}

}  // namespace

ABX_API int abx_norm_size(void) { return (int)sizeof(abx_norm); }

ABX_API int abx_norm_forward(void* stream, const abx_norm* norm, void* y, float* mean, float* rstd)
{
    if (int rc = check(norm)) return rc;
    const abx_norm& n = *norm;
    if (n.rows == 0) return ABX_OK;
    if (!y) return ABX_E_NULL_PTR;
    if (off(y, size_of(n.dtype)) || off(mean, 4) || off(rstd, 4)) return ABX_E_ALIGN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Args a = args_of(n);
    a.y = y; a.mean = mean; a.rstd = rstd;
    return by_flags(n, vectors(n, nullptr, 0, y), [&](auto t, auto rms, auto vec) {
        using T = decltype(t);
        constexpr bool kRms = decltype(rms)::value, kVec = decltype(vec)::value;
        const int64_t nvec = (n.cols + Vec<T>::V - 1) / Vec<T>::V;
        return by_width(nvec, kMostVectors, [&](auto lanes, auto nv) {
            constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value;
            if constexpr (L == 0) {
                const int grid = (int)(n.rows < kMaxGrid ? n.rows : kMaxGrid);
                forward_long<T, kRms, kVec><<<grid, kLong, 0, st>>>(a);
            } else {
                constexpr int rows = threads_of<L>() / L;
                const int64_t need = (n.rows + rows - 1) / rows;
                const int grid = (int)(need < kMaxGrid ? need : kMaxGrid);
                forward_kernel<T, kRms, kVec, L, NV><<<grid, threads_of<L>(), 0, st>>>(a);
            }
            return launched("norm forward launch");
        });
    });
}

ABX_API size_t abx_norm_backward_workspace_bytes(const abx_norm* norm)
{
    int sms = 0;
    if (check(norm) || sm_count(&sms)) return 0;
    return (size_t)backward_parts(*norm, sms) * (size_t)norm->cols * 4 * (norm->rms ? 1 : 2);
}

ABX_API int abx_norm_backward(void* stream, const abx_norm* norm, const void* dy, int64_t dy_stride, const float* mean,
                              const float* rstd, void* dx, void* dw, void* db, void* workspace, size_t workspace_bytes)
{
    if (int rc = check(norm)) return rc;
    const abx_norm& n = *norm;
    const bool sums = dw || db;
    if (n.rms && db) return ABX_E_ARG;
    if (n.rows > 0 && (!dy || !rstd || (!n.rms && !mean))) return ABX_E_NULL_PTR;
    if (sums && n.w_dtype != ABX_DT_F32 && n.w_dtype != ABX_DT_BF16) return ABX_E_P_DTYPE;
    if (off(dy, size_of(n.dtype)) || off(dx, size_of(n.dtype)) || off(mean, 4) || off(rstd, 4)) return ABX_E_ALIGN;
    if (sums && (off(dw, size_of(n.w_dtype)) || off(db, size_of(n.w_dtype)) || off(workspace, 16))) return ABX_E_ALIGN;
    if (!dx && !sums) return ABX_OK;
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    const int parts = backward_parts(n, sms);
    if (sums && (!workspace || workspace_bytes < (size_t)parts * (size_t)n.cols * 4 * (n.rms ? 1 : 2))) return ABX_E_OOM;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Args a = args_of(n);
    a.dy = dy; a.dy_stride = dy_stride;
    a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    a.y = dx;
    a.partial = sums ? static_cast<float*>(workspace) : nullptr;
    a.has_db = db != nullptr;
    int rc = by_flags(n, vectors(n, dy, dy_stride, dx), [&](auto t, auto rms, auto vec) {
        using T = decltype(t);
        constexpr bool kRms = decltype(rms)::value, kVec = decltype(vec)::value;
        const int64_t nvec = (n.cols + Vec<T>::V - 1) / Vec<T>::V;
        return by_width(nvec, kMostVectors, [&](auto lanes, auto nv) {
            constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value;
            if constexpr (L == 0) {
                if (dx && n.rows > 0) {
                    const int grid = (int)(n.rows < kMaxGrid ? n.rows : kMaxGrid);
                    backward_long<T, kRms, kVec><<<grid, kLong, 0, st>>>(a);
                    if (int e = launched("norm backward launch")) return e;
                }
                if (!sums) return (int)ABX_OK;
                const int64_t tiles = (nvec + 31) / 32;
                if (tiles > kMaxGrid) return (int)ABX_E_ARG;
                sums_long<T, kRms, kVec><<<dim3((unsigned)tiles, (unsigned)parts), 32 * kSumRows, 0, st>>>(a);
                return launched("norm sums launch");
            } else {
                backward_kernel<T, kRms, kVec, L, NV><<<parts, threads_of<L>(), 0, st>>>(a);
                return launched("norm backward launch");
            }
        });
    });
    if (rc || !sums) return rc;
    FinishArgs f;
    f.partial = a.partial;
    f.out[0] = dw ? dw : db;
    f.out[1] = db;
    f.cols = n.cols;
    f.parts = parts;
    f.bf16_out = n.w_dtype == ABX_DT_BF16;
    if (!dw) f.partial += (int64_t)parts * n.cols;      // db alone
    finish_sums<<<dim3((unsigned)((n.cols + 31) / 32), dw && db ? 2 : 1), 256, 0, st>>>(f);
    return launched("norm finish launch");
}
