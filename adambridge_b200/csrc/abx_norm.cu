// abx_norm.cu -- layer norm and RMS norm over the last axis, forward and backward (libabx).
//
// Rows of N values, in fp32 whatever the tensors' type, rounded once on the way out:
//   mu = mean x (RMS norm: 0),  r = 1 / sqrt(mean (x - mu)^2 + eps),  h = (x - mu) r,  y = h w + b
//   a = dy w,  dx = r (a - mean a - h mean(a h))  (RMS norm: without mean a),  dw = sum_rows dy h,  db = sum_rows dy
//
// A row stays in registers between its load and its store: the forward pass reads x once and writes y once, the
// backward pass reads x and dy once (long rows a second time from shared memory) and writes dx once.  The variance is taken
// about the mean (a second sum over the registers), so no large squares cancel.  A row is owned by part of a warp, a warp or
// a CTA, by its length.  HBM bounds rows that start on 16 bytes (layer norm of 32768 x 8192 bf16 values: 174 us forward,
// 283 backward, 0.94 and 0.87 of the copy bandwidth); instructions those whose values are accessed one by one (8000 x 4097
// bf16 values: 31 per value forward and 37 backward, against 16 and 19, at the same 0.5 to 0.6 issued per cycle).
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
    int32_t kept;       // rows that a long kernel keeps in shared memory
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
__device__ __forceinline__ void load_w(const void* w, const Args& a, int64_t cols, int lane, int i, float fill, float (&x)[V])
{
    const int64_t c0 = column<VEC, LANES, V>(lane, i, 0);
    if (w == nullptr) {
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = fill;
    } else if (VEC && a.w_vec && c0 < cols) {
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
            if (c < cols)
                x[k] = a.w_bf16 ? u2f((uint32_t)static_cast<const uint16_t*>(w)[c] << 16) : static_cast<const float*>(w)[c];
        }
    }
}

// V weights of type W as they are stored, held by a thread for all of its rows.
template <typename W, int V>
struct Weights {
    uint32_t raw[V * (int)sizeof(W) / 4];

    // `fill` where there are none; 0 beyond the row
    template <bool VEC, int LANES>
    __device__ __forceinline__ void load(const void* w, const Args& a, int64_t cols, int lane, int i, float fill)
    {
        float x[V];
        load_w<VEC, LANES, V>(w, a, cols, lane, i, fill, x);
#pragma unroll
        for (int k = 0; k < V * (int)sizeof(W) / 4; ++k) {
            if constexpr (sizeof(W) == 4) raw[k] = f2u(x[k]);
            else raw[k] = abx::pack_bf16_rne(x[2 * k], x[2 * k + 1]);   // exact: the values are bf16
        }
    }
    __device__ __forceinline__ abx::f2x pair(int j) const
    {
        if constexpr (sizeof(W) == 4) return abx::pk2(u2f(raw[2 * j]), u2f(raw[2 * j + 1]));
        else return abx::pk2(u2f(raw[j] << 16), u2f(raw[j] & 0xffff0000U));
    }
};

// ---- sums over the threads that own a row -----------------------------------------------------------

// Floats of shared memory that row_sum wants: two halves of two sums per warp of the row.
template <int LANES> __host__ __device__ constexpr int sum_floats() { return LANES > 32 ? 4 * (LANES / 32) : 1; }

// K sums at once, each over the LANES threads of a row; every thread gets them.  `buf` alternates between two halves, so
// one barrier per call is enough (a thread is at most one call ahead of another).
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
        const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) b[k * kW + warp] = s[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            s[k] = lane < kW ? b[k * kW + lane] : 0.0f;
#pragma unroll
            for (int o = kW > 16 ? 16 : kW > 8 ? 8 : kW > 4 ? 4 : kW > 2 ? 2 : 1; o > 0; o >>= 1)
                s[k] += __shfl_xor_sync(0xffffffffU, s[k], o);
            if constexpr (kW < 32) s[k] = __shfl_sync(0xffffffffU, s[k], 0);
        }
    }
}

template <int LANES> __host__ __device__ constexpr int threads_of() { return LANES > 32 ? LANES : 256; }

// ---- pairs: two values per FP32 instruction ------------------------------------------------------------

using abx::f2x;
using abx::fma2;
using abx::mul2;
using abx::pk2;
using abx::up2;

__device__ __forceinline__ f2x both(float x) { return pk2(x, x); }

__device__ __forceinline__ f2x add2(f2x a, f2x b)
{
    f2x d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <int V>
__device__ __forceinline__ void pairs(const float (&x)[V], f2x (&p)[V / 2])
{
#pragma unroll
    for (int j = 0; j < V / 2; ++j) p[j] = pk2(x[2 * j], x[2 * j + 1]);
}

template <int V>
__device__ __forceinline__ void singles(const f2x (&p)[V / 2], float (&x)[V])
{
#pragma unroll
    for (int j = 0; j < V / 2; ++j) up2(p[j], x[2 * j], x[2 * j + 1]);
}

__device__ __forceinline__ float sum_of(f2x x)
{
    float a, b;
    up2(x, a, b);
    return a + b;
}

// ---- rows under way ------------------------------------------------------------------------------------
// A thread copies its own vectors of the rows to come into shared memory and reads them back itself: no registers for
// what is under way, and nothing to synchronize.  Vector j of stage s lies at ((s * PER + j) * threads + thread) * 16.

__device__ __forceinline__ void copy_async(void* to, const void* from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)),
                 "l"(__cvta_generic_to_global(from)) : "memory");
}

template <int AHEAD>
__device__ __forceinline__ void copies_but(void) { asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory"); }

__device__ __forceinline__ Raw stored(const uint8_t* p)
{
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    return Raw{{q.x, q.y, q.z, q.w}};
}

// Where rows do not allow that, a thread loads the values of its next row into registers while it computes one (8000 x 4097
// in bf16: 67 instead of 113 us forward, on 512 threads); forward not where a row is a warp's or less and other warps hide
// the wait (300000 x 37 in fp32: 20 instead of 25 us).
template <typename T, int LANES, int NV>
struct Ahead {
    static constexpr int V = Vec<T>::V;
    uint32_t e[NV][V];

    __device__ __forceinline__ void load(const T* row, int64_t cols, int lane)
    {
        const T* const p = row + lane;
        const int left = (int)cols - lane;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                e[i][k] = 0U;
                if ((i * V + k) * LANES < left) {
                    if constexpr (V == 8) e[i][k] = p[(i * V + k) * LANES].bits;
                    else e[i][k] = f2u(p[(i * V + k) * LANES]);
                }
            }
    }
    __device__ __forceinline__ void values(int i, float (&x)[V]) const
    {
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = u2f(V == 8 ? e[i][k] << 16 : e[i][k]);
    }
};

template <typename T, int LANES>
__device__ __forceinline__ void start_copy(uint8_t* to, const T* row, int64_t cols, int lane, int i)
{
    const int64_t c = column<true, LANES, Vec<T>::V>(lane, i, 0);
    if (c < cols) copy_async(to, row + c);
}

// Stages of 16 bytes x `vectors` per thread that fit in `bytes`, between 2 and 4.
constexpr int stages_in(int bytes, int vectors, int threads)
{
    const int s = bytes / (16 * vectors * threads);
    return s < 2 ? 2 : s > 4 ? 4 : s;
}

// ---- forward -----------------------------------------------------------------------------------------

// A row of 4096 bf16 values: three stages for layer norm (90 us for 32768 rows; two: 95), two for RMS norm (92; three or
// four: 98, its shorter kernel runs further ahead and spreads over more of the DRAM's pages).
template <bool RMS, bool VEC, int LANES, int NV>
struct ForwardRing {
    static constexpr int kThreads = threads_of<LANES>();
    static constexpr int kStages = VEC ? stages_in(RMS ? 16384 : 24576, NV, kThreads) : 1;
    static constexpr int kBytes = VEC ? kStages * NV * kThreads * 16 : 0;
};

template <typename T, typename W, bool RMS, bool VEC, int LANES, int NV>
__global__ void __launch_bounds__(threads_of<LANES>()) forward_kernel(const __grid_constant__ Args a)
{
    using R = ForwardRing<RMS, VEC, LANES, NV>;
    constexpr int V = Vec<T>::V, kRows = threads_of<LANES>() / LANES;
    __shared__ float buf[sum_floats<LANES>()];
    extern __shared__ __align__(16) uint8_t ring[];
    int half = 0;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.0f / (float)a.cols;
    const int64_t stride = (int64_t)gridDim.x * kRows, first = (int64_t)blockIdx.x * kRows, cols = a.cols;
    uint8_t* const mine = ring + threadIdx.x * 16;
    const auto row_at = [&](int64_t row0) {   // a group without a row takes part with the first group's
        return static_cast<const T*>(a.x) + (row0 + group < a.rows ? row0 + group : row0) * a.x_stride;
    };
    const auto prefetch = [&](int64_t row0, int stage) {
        if constexpr (VEC) {
            if (row0 < a.rows) {
                const T* const x = row_at(row0);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    start_copy<T, LANES>(mine + (stage * NV + i) * (R::kThreads * 16), x, cols, lane, i);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    };
    bool valid[NV];   // vectors within the row (where VEC, a vector is either wholly in it or not at all)
    Weights<W, V> w[NV], b[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        valid[i] = column<VEC, LANES, V>(lane, i, 0) < cols;
        w[i].template load<VEC, LANES>(a.w, a, cols, lane, i, 1.0f);
        if constexpr (!RMS) b[i].template load<VEC, LANES>(a.b, a, cols, lane, i, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < R::kStages - 1; ++i) prefetch(first + i * stride, i);
    int stage = 0;
    constexpr bool kEarly = !VEC && LANES * NV > 32;
    Ahead<T, LANES, NV> ahead;
    if constexpr (kEarly) if (first < a.rows) ahead.load(row_at(first), cols, lane);
    for (int64_t row0 = first; row0 < a.rows; row0 += stride) {
        prefetch(row0 + (R::kStages - 1) * stride, stage == 0 ? R::kStages - 1 : stage - 1);
        f2x v[NV][V / 2];
        if constexpr (VEC) copies_but<R::kStages - 1>();
        else if constexpr (!kEarly) ahead.load(row_at(row0), cols, lane);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float x[V];
            if constexpr (VEC) {
                Raw raw = {{0U, 0U, 0U, 0U}};
                if (valid[i]) raw = stored(mine + (stage * NV + i) * (R::kThreads * 16));
                unpack<T>(raw, x);
            } else {
                ahead.values(i, x);
            }
            pairs<V>(x, v[i]);
        }
        if constexpr (kEarly) if (row0 + stride < a.rows) ahead.load(row_at(row0 + stride), cols, lane);
        stage = stage + 1 == R::kStages ? 0 : stage + 1;
        float mean = 0.0f;
        if constexpr (!RMS) {
            f2x t = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V / 2; ++j) t = add2(t, v[i][j]);
            float s[1] = {sum_of(t)};
            row_sum<LANES, 1>(s, buf, half);
            mean = s[0] * inv;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const f2x less = both(valid[i] ? -mean : 0.0f);   // what lies beyond the row stays 0
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    v[i][j] = add2(v[i][j], less);
                    if constexpr (!VEC) {
                        float p, q;
                        up2(v[i][j], p, q);
                        v[i][j] = pk2(column<VEC, LANES, V>(lane, i, 2 * j) < cols ? p : 0.0f,
                                      column<VEC, LANES, V>(lane, i, 2 * j + 1) < cols ? q : 0.0f);
                    }
                }
            }
        }
        f2x t = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V / 2; ++j) t = fma2(v[i][j], v[i][j], t);
        float q[1] = {sum_of(t)};
        row_sum<LANES, 1>(q, buf, half);
        const float rstd = __frcp_rn(__fsqrt_rn(__fmaf_rn(q[0], inv, a.eps)));
        const int64_t row = row0 + group;
        if (row >= a.rows) continue;
        T* const y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float x[V];
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                const f2x h = mul2(v[i][j], both(rstd));
                if constexpr (RMS) v[i][j] = mul2(h, w[i].pair(j));
                else v[i][j] = fma2(h, w[i].pair(j), b[i].pair(j));
            }
            singles<V>(v[i], x);
            store<T, VEC, LANES>(y, cols, lane, i, x);
        }
        if (lane == 0) {
            if (!RMS && a.mean != nullptr) a.mean[row] = mean;
            if (a.rstd != nullptr) a.rstd[row] = rstd;
        }
    }
}

// Rows longer than a CTA's registers (and backward, long rows that are few): three passes over the row, which is kept in
// shared memory where it fits and rows allow vector access (each thread copies and reads its own vectors), and read again
// from the caches where not.
constexpr int kLong = 512;

// A thread's vector i of the row, of `count` rows of one image each (x, or x and dy).
template <typename T, bool VEC>
struct LongRow {
    const Args& a;
    uint8_t* const ring;
    const int count;

    __device__ __forceinline__ uint8_t* slot(int stage, int image, int i) const
    {
        return ring + ((int64_t)(stage * count + image) * a.cols * (int64_t)sizeof(T) + ((int64_t)i * kLong + threadIdx.x) * 16);
    }
    __device__ __forceinline__ void prefetch(const T* row, int stage, int image, int steps) const
    {
        for (int i = 0; i < steps; ++i)
            if (((int64_t)i * kLong + threadIdx.x) * Vec<T>::V < a.cols)
                copy_async(slot(stage, image, i), row + ((int64_t)i * kLong + threadIdx.x) * Vec<T>::V);
    }
    __device__ __forceinline__ Raw get(const T* row, int stage, int image, int i) const
    {
        if constexpr (VEC) {
            if (a.kept) {
                if (((int64_t)i * kLong + threadIdx.x) * Vec<T>::V < a.cols) return stored(slot(stage, image, i));
                return Raw{{0U, 0U, 0U, 0U}};
            }
        }
        return load<T, VEC, kLong>(row, a.cols, threadIdx.x, i);
    }
};

template <typename T, bool RMS, bool VEC>
__global__ void __launch_bounds__(kLong) forward_long(const __grid_constant__ Args a)
{
    constexpr int V = Vec<T>::V;
    __shared__ float buf[sum_floats<kLong>()];
    extern __shared__ __align__(16) uint8_t ring[];
    int half = 0, stage = 0;
    const int lane = threadIdx.x;
    const float inv = 1.0f / (float)a.cols;
    const int steps = (int)((a.cols + (int64_t)kLong * V - 1) / ((int64_t)kLong * V));
    const LongRow<T, VEC> rows{a, ring, 1};
    const auto prefetch = [&](int64_t row, int to) {
        if constexpr (VEC) {
            if (a.kept && row < a.rows) rows.prefetch(static_cast<const T*>(a.x) + row * a.x_stride, to, 0, steps);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    };
    if (a.kept == 2) prefetch(blockIdx.x, 0);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(a.x) + row * a.x_stride;
        if constexpr (VEC) {
            if (a.kept == 2) {
                prefetch(row + gridDim.x, stage ^ 1);
                copies_but<1>();
            } else {
                prefetch(row, 0);
                copies_but<0>();
            }
        }
        float mean = 0.0f;
        if constexpr (!RMS) {
            float s[1] = {0.0f};
            for (int i = 0; i < steps; ++i) {
                float v[V];
                unpack<T>(rows.get(x, stage, 0, i), v);
#pragma unroll
                for (int k = 0; k < V; ++k) s[0] += v[k];
            }
            row_sum<kLong, 1>(s, buf, half);
            mean = s[0] * inv;
        }
        float q[1] = {0.0f};
        for (int i = 0; i < steps; ++i) {
            float v[V];
            unpack<T>(rows.get(x, stage, 0, i), v);
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
            unpack<T>(rows.get(x, stage, 0, i), v);
            load_w<VEC, kLong, V>(a.w, a, a.cols, lane, i, 1.0f, w);
            load_w<VEC, kLong, V>(a.b, a, a.cols, lane, i, 0.0f, b);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = __fmaf_rn((v[k] - mean) * rstd, w[k], b[k]);
            store<T, VEC, kLong>(y, a.cols, lane, i, v);
        }
        if (lane == 0) {
            if (!RMS && a.mean != nullptr) a.mean[row] = mean;
            if (a.rstd != nullptr) a.rstd[row] = rstd;
        }
        if (a.kept == 2) stage ^= 1;
    }
}

// ---- backward ----------------------------------------------------------------------------------------

template <bool VEC, int LANES, int NV>
struct BackwardRing {
    static constexpr int kThreads = threads_of<LANES>();
    static constexpr int kStages = VEC ? stages_in(65536, 2 * NV, kThreads) : 1;
    static constexpr int kBytes = VEC ? kStages * 2 * NV * kThreads * 16 : 0;
};

// With three vectors or more per thread the sums leave no registers for a row: it is read from shared memory twice.
template <bool VEC, int LANES, int NV>
__host__ __device__ constexpr bool twice() { return VEC && LANES > 32 && NV > 2; }

// Resident CTAs of the backward kernel per SM: 1024 threads of one vector, 512 of two; 768 of one where values are accessed
// one by one and a row ahead takes registers.
template <bool VEC, int LANES, int NV>
__host__ __device__ constexpr int backward_ctas()
{
    const int c = twice<VEC, LANES, NV>() ? 512 / threads_of<LANES>()
                : VEC ? 1024 / (threads_of<LANES>() * (NV > 2 ? 4 : NV)) : (NV == 1 ? 768 : 512) / threads_of<LANES>();
    return c < 1 ? 1 : c;
}

// Whether h = (0 - mean) rstd, of the zeros that stand beyond a row's end, is not finite: rows of large equal values.  The
// branch costs 1 to 3% of a backward pass over short rows accessed value by value (210526 x 19 in bf16: 21.5 against 20.6
// us), elsewhere nothing that can be measured.
__device__ __forceinline__ bool overflows(float mean, float rstd) { return !(fabsf(mean * rstd) <= 3.402823466e38f); }

// dx of every row, and this CTA's part of dw and db over its rows.
template <typename T, typename W, bool RMS, bool VEC, int LANES, int NV>
__global__ void __launch_bounds__(threads_of<LANES>(), backward_ctas<VEC, LANES, NV>()) backward_kernel(const __grid_constant__ Args a)
{
    using R = BackwardRing<VEC, LANES, NV>;
    constexpr int V = Vec<T>::V, kThreads = threads_of<LANES>(), kRows = kThreads / LANES;
    constexpr int kSums = RMS ? 1 : 2;
    __shared__ float buf[sum_floats<LANES>()];
    extern __shared__ __align__(16) uint8_t ring[];   // the rows under way; at the end, the warps' sums
    int half = 0;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.0f / (float)a.cols;
    const int64_t stride = (int64_t)gridDim.x * kRows, first = (int64_t)blockIdx.x * kRows, cols = a.cols;
    uint8_t* const mine = ring + threadIdx.x * 16;
    const auto row_of = [&](int64_t row0) { return row0 + group < a.rows ? row0 + group : row0; };
    const auto prefetch = [&](int64_t row0, int stage) {
        if constexpr (VEC) {
            if (row0 < a.rows) {
                const T* const x = static_cast<const T*>(a.x) + row_of(row0) * a.x_stride;
                const T* const dy = static_cast<const T*>(a.dy) + row_of(row0) * a.dy_stride;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    start_copy<T, LANES>(mine + (stage * 2 * NV + i) * (kThreads * 16), x, cols, lane, i);
                    start_copy<T, LANES>(mine + (stage * 2 * NV + NV + i) * (kThreads * 16), dy, cols, lane, i);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    };
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // finish_sums may come up
    f2x dw[NV][V / 2], db[NV][V / 2];
    bool valid[NV];
    Weights<W, V> w[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        valid[i] = column<VEC, LANES, V>(lane, i, 0) < cols;
        w[i].template load<VEC, LANES>(a.w, a, cols, lane, i, 1.0f);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) dw[i][j] = db[i][j] = 0;
    }
#pragma unroll
    for (int i = 0; i < R::kStages - 1; ++i) prefetch(first + i * stride, i);
    int stage = 0;
    float next_mean = 0.0f, next_rstd = 0.0f;   // a row ahead
    const auto statistics = [&](int64_t row0) {
        if (row0 < a.rows) {
            if constexpr (!RMS) next_mean = a.mean[row_of(row0)];
            next_rstd = a.rstd[row_of(row0)];
        }
    };
    statistics(first);
    Ahead<T, LANES, NV> next_x, next_dy;
    const auto look_ahead = [&](int64_t row0) {
        if (row0 >= a.rows) return;
        next_x.load(static_cast<const T*>(a.x) + row_of(row0) * a.x_stride, cols, lane);
        next_dy.load(static_cast<const T*>(a.dy) + row_of(row0) * a.dy_stride, cols, lane);
    };
    constexpr bool kEarly = !VEC && NV < 3;   // three vectors have no registers for it
    if constexpr (kEarly) look_ahead(first);
    for (int64_t row0 = first; row0 < a.rows; row0 += stride) {
        prefetch(row0 + (R::kStages - 1) * stride, stage == 0 ? R::kStages - 1 : stage - 1);
        const int64_t row = row_of(row0);
        const bool live = row0 + group < a.rows;
        const float mean = next_mean, rstd = next_rstd;
        statistics(row0 + stride);
        if constexpr (VEC) copies_but<R::kStages - 1>();
        else if constexpr (!kEarly) look_ahead(row0);
        if constexpr (twice<VEC, LANES, NV>()) {
            uint8_t* const here = mine + stage * (2 * NV * kThreads * 16);
            const auto read = [&](int i, f2x (&h)[V / 2], f2x (&d)[V / 2]) {
                float x[V];
                unpack<T>(stored(here + i * (kThreads * 16)), x);
                pairs<V>(x, h);
                unpack<T>(stored(here + (NV + i) * (kThreads * 16)), x);
                pairs<V>(x, d);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    if constexpr (!RMS) h[j] = add2(h[j], both(-mean));
                    h[j] = mul2(h[j], both(rstd));
                }
            };
            f2x s0 = 0, s1 = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!valid[i]) continue;
                f2x h[V / 2], d[V / 2];
                read(i, h, d);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const f2x g = mul2(d[j], w[i].pair(j));
                    s0 = fma2(g, h[j], s0);
                    if constexpr (!RMS) s1 = add2(s1, g);
                }
            }
            float s[kSums];
            s[0] = sum_of(s0);
            if constexpr (!RMS) s[1] = sum_of(s1);
            row_sum<LANES, kSums>(s, buf, half);
            const float c2 = s[0] * inv, c1 = RMS ? 0.0f : s[kSums - 1] * inv;
            T* const dx = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!valid[i]) continue;
                f2x h[V / 2], d[V / 2];
                read(i, h, d);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    dw[i][j] = fma2(d[j], h[j], dw[i][j]);
                    if constexpr (!RMS) db[i][j] = add2(db[i][j], d[j]);
                    d[j] = mul2(d[j], w[i].pair(j));
                    if constexpr (!RMS) d[j] = add2(d[j], both(-c1));
                    d[j] = mul2(fma2(h[j], both(-c2), d[j]), both(rstd));
                }
                float x[V];
                singles<V>(d, x);
                if (a.y != nullptr) store<T, VEC, LANES>(dx, cols, lane, i, x);
            }
            stage = stage + 1 == R::kStages ? 0 : stage + 1;
            continue;
        }
        f2x h[NV][V / 2], g[NV][V / 2];   // the normalized values and dy w
        f2x s0 = 0, s1 = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float x[V], y[V];
            f2x d[V / 2];
            if constexpr (VEC) {
                Raw rx = {{0U, 0U, 0U, 0U}}, rd = rx;
                if (valid[i]) {
                    rx = stored(mine + (stage * 2 * NV + i) * (kThreads * 16));
                    rd = stored(mine + (stage * 2 * NV + NV + i) * (kThreads * 16));
                }
                unpack<T>(rx, y);
                unpack<T>(rd, x);
            } else {
                next_x.values(i, y);
                next_dy.values(i, x);
            }
            pairs<V>(y, h[i]);
            if (!live) {   // a group without a row adds nothing
#pragma unroll
                for (int k = 0; k < V; ++k) x[k] = 0.0f;
            }
            pairs<V>(x, d);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {   // beyond the row's end d is 0
                if constexpr (!RMS) h[i][j] = add2(h[i][j], both(-mean));
                h[i][j] = mul2(h[i][j], both(rstd));
                g[i][j] = mul2(d[j], w[i].pair(j));
                s0 = fma2(g[i][j], h[i][j], s0);
                dw[i][j] = fma2(d[j], h[i][j], dw[i][j]);
                if constexpr (!RMS) {
                    s1 = add2(s1, g[i][j]);
                    db[i][j] = add2(db[i][j], d[j]);
                }
            }
        }
        if constexpr (kEarly && NV == 1) look_ahead(row0 + stride);   // two vectors have no registers for it yet
        if constexpr (!RMS) {
            if (__builtin_expect(overflows(mean, rstd), 0)) {   // beyond the row's end g h is 0 times infinity
                int left = (int)cols - lane * (VEC ? V : 1);
                asm volatile("" : "+r"(left));   // compared here, not held for this in registers all along
                s0 = 0;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) {
                        float p, q;
                        up2(mul2(g[i][j], h[i][j]), p, q);
                        s0 = add2(s0, pk2(left > (int)column<VEC, LANES, V>(0, i, 2 * j) ? p : 0.0f,
                                          left > (int)column<VEC, LANES, V>(0, i, 2 * j + 1) ? q : 0.0f));
                    }
            }
        }
        if constexpr (kEarly && NV > 1) look_ahead(row0 + stride);
        stage = stage + 1 == R::kStages ? 0 : stage + 1;
        float s[kSums];
        s[0] = sum_of(s0);
        if constexpr (!RMS) s[1] = sum_of(s1);
        row_sum<LANES, kSums>(s, buf, half);
        if (!live || a.y == nullptr) continue;
        const float c2 = s[0] * inv, c1 = RMS ? 0.0f : s[kSums - 1] * inv;
        T* const dx = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                if constexpr (!RMS) g[i][j] = add2(g[i][j], both(-c1));
                g[i][j] = mul2(fma2(h[i][j], both(-c2), g[i][j]), both(rstd));
            }
            float x[V];
            singles<V>(g[i], x);
            store<T, VEC, LANES>(dx, cols, lane, i, x);
        }
    }
    if (a.partial == nullptr) return;
    float* const out = a.partial + (int64_t)blockIdx.x * cols;
    const int64_t second = (int64_t)gridDim.x * cols;
#pragma unroll
    for (int which = 0; which < kSums; ++which) {
        if (which == 1 && !a.has_db) break;
        float sums[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i) singles<V>(which ? db[i] : dw[i], sums[i]);
        if constexpr (LANES > 32 && VEC) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float4* const to = reinterpret_cast<float4*>(out + which * second + column<VEC, LANES, V>(lane, i, 0));
#pragma unroll
                for (int k = 0; k < V / 4; ++k)
                    if (valid[i]) to[k] = make_float4(sums[i][4 * k], sums[i][4 * k + 1], sums[i][4 * k + 2], sums[i][4 * k + 3]);
            }
        } else if constexpr (LANES > 32) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const int64_t c = column<VEC, LANES, V>(lane, i, k);
                    if (c < cols) out[which * second + c] = sums[i][k];
                }
        } else {
            // the groups of a warp by shuffles, then the warps through shared memory, in order
            constexpr int kCols = LANES * NV * V;
            float* const mem = reinterpret_cast<float*>(ring);
            __syncthreads();   // every thread is through with its rows, or with the first sums
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    float t = sums[i][k];
#pragma unroll
                    for (int o = LANES; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffU, t, o);
                    if ((threadIdx.x & 31) < LANES)
                        mem[(threadIdx.x >> 5) * kCols + (int)column<VEC, LANES, V>(lane, i, k)] = t;
                }
            __syncthreads();
            for (int c = threadIdx.x; c < kCols && c < cols; c += kThreads) {
                float t = 0.0f;
#pragma unroll
                for (int j = 0; j < kThreads / 32; ++j) t += mem[j * kCols + c];
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
    __shared__ float buf[sum_floats<kLong>()];
    extern __shared__ __align__(16) uint8_t ring[];
    int half = 0, stage = 0;
    const int lane = threadIdx.x;
    const float inv = 1.0f / (float)a.cols;
    const int steps = (int)((a.cols + (int64_t)kLong * V - 1) / ((int64_t)kLong * V));
    const LongRow<T, VEC> rows{a, ring, 2};
    const auto prefetch = [&](int64_t row, int to) {
        if constexpr (VEC) {
            if (a.kept && row < a.rows) {
                rows.prefetch(static_cast<const T*>(a.x) + row * a.x_stride, to, 0, steps);
                rows.prefetch(static_cast<const T*>(a.dy) + row * a.dy_stride, to, 1, steps);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    };
    if (a.kept == 2) prefetch(blockIdx.x, 0);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* const dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
        const float mean = RMS ? 0.0f : a.mean[row], rstd = a.rstd[row];
        if constexpr (VEC) {
            if (a.kept == 2) {
                prefetch(row + gridDim.x, stage ^ 1);
                copies_but<1>();
            } else {
                prefetch(row, 0);
                copies_but<0>();
            }
        }
        const bool far = !RMS && overflows(mean, rstd);   // see there
        float s[kSums];
#pragma unroll
        for (int k = 0; k < kSums; ++k) s[k] = 0.0f;
        for (int i = 0; i < steps; ++i) {
            float v[V], d[V], w[V];
            unpack<T>(rows.get(x, stage, 0, i), v);
            unpack<T>(rows.get(dy, stage, 1, i), d);
            load_w<VEC, kLong, V>(a.w, a, a.cols, lane, i, 1.0f, w);
            if constexpr (!RMS) {
                if (__builtin_expect(far, 0)) {
#pragma unroll
                    for (int k = 0; k < V; ++k) if (column<VEC, kLong, V>(lane, i, k) >= a.cols) v[k] = mean;
                }
            }
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
            unpack<T>(rows.get(x, stage, 0, i), v);
            unpack<T>(rows.get(dy, stage, 1, i), d);
            load_w<VEC, kLong, V>(a.w, a, a.cols, lane, i, 1.0f, w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float h = (v[k] - mean) * rstd;
                v[k] = __fmaf_rn(-h, c2, d[k] * w[k] - c1) * rstd;
            }
            store<T, VEC, kLong>(dx, a.cols, lane, i, v);
        }
        if (a.kept == 2) stage ^= 1;
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
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // finish_sums may come up
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

// dw (blockIdx.y 0) and db (1) from the parts: 32 columns per CTA, 32 threads per column, in a fixed order.
struct FinishArgs {
    const float* partial;
    void* out[2];
    int64_t cols;
    int32_t parts;
    int32_t bf16_out;
};

__global__ void __launch_bounds__(1024) finish_sums(const __grid_constant__ FinishArgs a)
{
    __shared__ float buf[32][33];
    const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    const float* p = a.partial + (int64_t)blockIdx.y * a.parts * a.cols;
    float t = 0.0f;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // for the parts
    if (c < a.cols)
#pragma unroll 8
        for (int i = ty; i < a.parts; i += 32) t += p[(int64_t)i * a.cols + c];
    buf[ty][lane] = t;
    __syncthreads();
    t = buf[lane][ty];   // the parts of column ty
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffU, t, o);
    const int64_t col = (int64_t)blockIdx.x * 32 + ty;
    if (lane == 0 && col < a.cols) {
        void* const out = blockIdx.y ? a.out[1] : a.out[0];
        if (a.bf16_out) static_cast<uint16_t*>(out)[col] = (uint16_t)abx::pack_bf16_rne(t, 0.0f);
        else static_cast<float*>(out)[col] = t;
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

// CTAs of a kernel that are resident on the current device.  Asked for once per device where its shared memory is always
// the same (a query is about as long as a launch): KERNEL's launches share the answer.
template <auto KERNEL>
int resident(int threads, size_t bytes, bool same, int* out)
{
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];
    int dev = 0, sms = 0, per = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const bool keep = same && e == cudaSuccess && dev < kDevices;
    if (keep && (*out = known[dev].load(std::memory_order_relaxed)) > 0) return ABX_OK;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, (const void*)KERNEL, threads, bytes);
    if (e != cudaSuccess) return abx::set_error("launch geometry", e);
    *out = sms * (per > 0 ? per : 1);
    if (keep) known[dev].store(*out, std::memory_order_relaxed);
    return ABX_OK;
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

// The shape of the row kernels, by the vectors of a row: threads per row, vectors per thread.
//
// Two vectors per thread (a row of 4096 bf16 values: 256 threads) beat one (layer norm of 16384 x 4096: 48 against 63 us
// forward, 73 against 93 backward), narrow rows forward too (RMS norm of 262144 x 128: 19.8 against 21.6 us); backward these,
// as fast with one, keep their registers.  A row of 5120 to 6144 bf16 values takes three, where two would need 512 threads
// and one CTA per SM (RMS norm of 32768 x 5120: 154 against 191 us backward).  Of 8192 it takes four forward (32768 rows:
// 174 against 191 us; fp32 rows are as fast with two), but not backward, where the sums leave no registers for that (343
// against 289 us).  Longer rows take up to five vectors of 512 threads, one CTA per SM; they beat the long kernels, which
// go through a row's memory again (5000 x 20000 bf16 values: 92 against 145 us forward, 162 against 240 backward).
// Where values are accessed one by one, instructions count, and so do threads without a value: finer steps (8000 x 4097 in
// bf16: 51 and 70 us against 67 and 95 with 512 threads; 100000 x 301: 39 and 58 against 44 and 57 with room for 64
// vectors, 54 and 81 with one vector per thread).
// (Sharing a long row among a cluster of CTAs was slower still: a cluster barrier per sum and row, 59 us instead of 12.6 for
// 515 x 20000 forward.)
template <int V, bool VEC, bool BACKWARD, typename F>
int by_width(int64_t nvec, F&& f)
{
    using std::integral_constant;
#define ABX_ROW(L, N) return f(integral_constant<int, L>{}, integral_constant<int, N>{})
    if (nvec <= 8) ABX_ROW(8, 1);
    if constexpr (VEC && !BACKWARD) {
        if (nvec <= 16) ABX_ROW(8, 2);
        if (nvec <= 32) ABX_ROW(16, 2);
    } else {
        if (nvec <= 16) ABX_ROW(16, 1);
        if (nvec <= 32) ABX_ROW(32, 1);
    }
    if constexpr (VEC) {
        if (nvec <= 64) ABX_ROW(32, 2);
        if (nvec <= 128) ABX_ROW(32, 4);
        if (nvec <= 256) ABX_ROW(128, 2);
        if (nvec <= 512) ABX_ROW(256, 2);
        if constexpr (!BACKWARD && V == 8) {
            if (nvec <= 768) ABX_ROW(256, 3);
            if (nvec <= 1024) ABX_ROW(256, 4);
        }
        if constexpr (BACKWARD) {
            if (nvec <= 768) ABX_ROW(256, 3);
        }
        if (nvec <= 1024) ABX_ROW(512, 2);
        if (nvec <= 1536) ABX_ROW(512, 3);
        if constexpr (BACKWARD) {
            if (nvec <= 2048) ABX_ROW(512, 4);
            if (nvec <= 2560) ABX_ROW(512, 5);
        }
    } else if constexpr (!BACKWARD) {
        if (nvec <= 48) ABX_ROW(16, 3);
        if (nvec <= 64) ABX_ROW(32, 2);
        if (nvec <= 96) ABX_ROW(32, 3);
        if (nvec <= 128) ABX_ROW(64, 2);
        if (nvec <= 192) ABX_ROW(64, 3);
        if (nvec <= 256) ABX_ROW(128, 2);
        if (nvec <= 384) ABX_ROW(128, 3);
        if (nvec <= 512) ABX_ROW(256, 2);
        if (nvec <= 768) ABX_ROW(256, 3);
        if (nvec <= 1024) ABX_ROW(512, 2);
        if (nvec <= 1536) ABX_ROW(512, 3);
    } else {
        if (nvec <= 64) ABX_ROW(32, 2);
        if (nvec <= 128) ABX_ROW(64, 2);
        if (nvec <= 192) ABX_ROW(96, 2);
        if (nvec <= 256) ABX_ROW(128, 2);
        if (nvec <= 384) ABX_ROW(192, 2);
        if (nvec <= 512) ABX_ROW(256, 2);
        if (nvec <= 768) ABX_ROW(384, 2);
        if (nvec <= 1024) ABX_ROW(512, 2);
        if (nvec <= 1536) ABX_ROW(512, 3);
    }
    if constexpr (!BACKWARD) {
        if (nvec <= 2048) ABX_ROW(512, 4);
        if (nvec <= 2560) ABX_ROW(512, 5);
    }
    return f(integral_constant<int, 0>{}, integral_constant<int, 0>{});
#undef ABX_ROW
}

template <typename F>
int by_flags(const abx_norm& n, bool vec, F&& f)
{
    using Y = std::true_type;
    using N = std::false_type;
    const auto flags = [&](auto t, auto w) {
        if (n.rms) return vec ? f(t, w, Y{}, Y{}) : f(t, w, Y{}, N{});
        return vec ? f(t, w, N{}, Y{}) : f(t, w, N{}, N{});
    };
    if (n.dtype == ABX_DT_BF16) return n.w_dtype == ABX_DT_BF16 ? flags(bf16{}, bf16{}) : flags(bf16{}, 0.0f);
    return n.w_dtype == ABX_DT_BF16 ? flags(0.0f, bf16{}) : flags(0.0f, 0.0f);
}

constexpr int kMaxGrid = 1 << 30;

// The vectors that the backward kernel's shape goes by.  Long rows in vectors take the long kernels where they are few: a
// CTA's sums, 8 bytes per column written and read again, are then more than what the second pass reads, 2 values per row and
// column (300 x 12288 bf16 values 18.5 against 19.2 us, 1000 41 against 29).
int64_t backward_vectors(const abx_norm& n, int sms, bool vec)
{
    const int64_t es = size_of(n.dtype), nvec = (n.cols * es + 15) / 16;
    return vec && nvec > 1024 && n.rows * es < (int64_t)8 * sms ? INT64_MAX : nvec;
}

// Parts of the sums: a CTA of the backward kernel each, as many as are resident, or fewer when there are few
// rows (a part is written and read again, so it should cover some).  Long rows: row runs of sums_long, so that all column
// tiles together fill the SMs.
template <bool VEC>
int backward_parts(const abx_norm& n, int sms)
{
    const int64_t v = 16 / size_of(n.dtype), nvec = (n.cols + v - 1) / v;
    return by_width<8, VEC, true>(backward_vectors(n, sms, VEC), [&](auto lanes, auto nv) {
        constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value;
        if constexpr (L == 0) {
            const int64_t tiles = (nvec + 31) / 32, want = (8 * sms + tiles - 1) / tiles, most = (n.rows + 31) / 32;
            const int64_t p = want < most ? want : most;
            return (int)(p > 0 ? p : 1);
        } else {
            constexpr int64_t rows = threads_of<L>() / L;
            const int64_t need = (n.rows + rows - 1) / rows, all = backward_ctas<VEC, L, NV>() * (int64_t)sms;
            return (int)(need < all ? (need > 0 ? need : 1) : all);
        }
    });
}

constexpr int kMostKept = 220 * 1024;   // bytes of rows that a long kernel keeps in shared memory, at most

// A launch with `bytes` of dynamic shared memory, for this kernel always the same or not; `most` CTAs, or as many as are
// resident.
template <auto KERNEL>
int launch_rows(int64_t most, bool all_resident, int threads, size_t bytes, bool same, const Args& a, cudaStream_t st,
                const char* what)
{
    if (bytes > 40960) {   // with the kernels' static shared memory that may exceed what needs no asking
        // always the same for a kernel: a smaller limit would fail a larger row that another thread is about to launch
        const cudaError_t e = cudaFuncSetAttribute((const void*)KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   same ? (int)bytes : kMostKept);
        if (e != cudaSuccess) return abx::set_error(what, e);
    }
    if (all_resident) {
        int ctas = 0;
        if (int rc = resident<KERNEL>(threads, bytes, same, &ctas)) return rc;
        if (ctas < most) most = ctas;
    }
    KERNEL<<<(unsigned)most, threads, bytes, st>>>(a);
    return launched(what);
}

// Rows of `bytes` that a long kernel keeps in shared memory: two (the next one under way) where two CTAs then still share
// an SM's 227 KB, one as far as it fits; 0: the row is read again instead.
int rows_kept(int64_t bytes)
{
    constexpr int64_t kHalf = 110 * 1024;
    return 2 * bytes <= kHalf ? 2 : bytes <= kMostKept ? 1 : 0;
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
    return by_flags(n, vectors(n, nullptr, 0, y), [&](auto t, auto weight, auto rms, auto vec) {
        using T = decltype(t);
        using W = decltype(weight);
        constexpr bool kRms = decltype(rms)::value, kVec = decltype(vec)::value;
        const int64_t nvec = (n.cols + Vec<T>::V - 1) / Vec<T>::V;
        return by_width<Vec<T>::V, kVec, false>(nvec, [&](auto lanes, auto nv) {
            constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value;
            if constexpr (L == 0) {
                const int64_t bytes = n.cols * (int64_t)sizeof(T);
                a.kept = kVec ? rows_kept(bytes) : 0;
                return launch_rows<forward_long<T, kRms, kVec>>(n.rows, true, kLong, (size_t)(a.kept * bytes), false, a, st,
                                   "norm forward launch");
            } else {
                constexpr int rows = threads_of<L>() / L;
                return launch_rows<forward_kernel<T, W, kRms, kVec, L, NV>>((n.rows + rows - 1) / rows, true, threads_of<L>(),
                                   ForwardRing<kRms, kVec, L, NV>::kBytes, true, a, st, "norm forward launch");
            }
        });
    });
}

ABX_API size_t abx_norm_backward_workspace_bytes(const abx_norm* norm)
{
    int sms = 0;
    if (check(norm) || sm_count(&sms)) return 0;
    // whether the vector kernels run depends on dy and dx too: enough for either
    const int a = backward_parts<true>(*norm, sms), b = backward_parts<false>(*norm, sms);
    return (size_t)(a > b ? a : b) * (size_t)norm->cols * 4 * (norm->rms ? 1 : 2);
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
    const bool vec_rows = vectors(n, dy, dy_stride, dx);
    const int parts = vec_rows ? backward_parts<true>(n, sms) : backward_parts<false>(n, sms);
    if (sums && (!workspace || workspace_bytes < (size_t)parts * (size_t)n.cols * 4 * (n.rms ? 1 : 2))) return ABX_E_OOM;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Args a = args_of(n);
    a.dy = dy; a.dy_stride = dy_stride;
    a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    a.y = dx;
    a.partial = sums ? static_cast<float*>(workspace) : nullptr;
    a.has_db = db != nullptr;
    int rc = by_flags(n, vec_rows, [&](auto t, auto weight, auto rms, auto vec) {
        using T = decltype(t);
        using W = decltype(weight);
        constexpr bool kRms = decltype(rms)::value, kVec = decltype(vec)::value;
        const int64_t nvec = (n.cols + Vec<T>::V - 1) / Vec<T>::V;
        return by_width<Vec<T>::V, kVec, true>(backward_vectors(n, sms, kVec), [&](auto lanes, auto nv) {
            constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value;
            if constexpr (L == 0) {
                if (dx && n.rows > 0) {
                    const int64_t bytes = 2 * n.cols * (int64_t)sizeof(T);
                    a.kept = kVec ? rows_kept(bytes) : 0;
                    if (int e = launch_rows<backward_long<T, kRms, kVec>>(n.rows, true, kLong, (size_t)(a.kept * bytes), false, a, st,
                                            "norm backward launch"))
                        return e;
                }
                if (!sums) return (int)ABX_OK;
                const int64_t tiles = (nvec + 31) / 32;
                if (tiles > kMaxGrid) return (int)ABX_E_ARG;
                sums_long<T, kRms, kVec><<<dim3((unsigned)tiles, (unsigned)parts), 32 * kSumRows, 0, st>>>(a);
                return launched("norm sums launch");
            } else {
                using R = BackwardRing<kVec, L, NV>;
                // the rows under way, or at the end the warps' sums
                constexpr int sums_bytes = L > 32 ? 0 : threads_of<L>() / 32 * L * NV * Vec<T>::V * 4;
                constexpr int bytes = R::kBytes > sums_bytes ? R::kBytes : sums_bytes;
                return launch_rows<backward_kernel<T, W, kRms, kVec, L, NV>>(parts, false, threads_of<L>(), bytes, true, a, st,
                                   "norm backward launch");
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
    // Brought up while the parts are being computed, it waits for them on the device: 25.6 against 26.8 us for the backward
    // pass of 4096 x 4096.
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t shape = {};
    shape.gridDim = dim3((unsigned)((n.cols + 31) / 32), dw && db ? 2 : 1);
    shape.blockDim = dim3(1024);
    shape.stream = st;
    shape.attrs = &early;
    shape.numAttrs = 1;
    if (const cudaError_t e = cudaLaunchKernelEx(&shape, finish_sums, f); e != cudaSuccess)
        return abx::set_error("norm finish launch", e);
    return launched("norm finish launch");
}
