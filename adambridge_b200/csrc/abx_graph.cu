// abx_graph.cu -- AdamW over many tensors whose step lives on the device (libabx).
//
// The update kernels of abx_kernels.cu take the step count, the learning rate and the rounding seed from the
// host with every call; a CUDA graph that captured one would repeat that step for ever.  Here they are read on
// the device: step counts are device integers, the learning rate may be one, and the gradient scale (a clip
// coefficient) and the decision to skip the step are device scalars.  So a captured training step replays.
//
// Per element, fp32, each operation rounded once (nothing is fused, so an elementwise restatement has the same bits):
//   g = g * scale;  p = p * decay;  m = b1 m + (1-b1) g;  v = b2 v + ((1-b2) g) g
//   p = p - a * (m / (sqrt(v) c + eps)),   a = lr / (1 - b1^t),  c = 1 / sqrt(1 - b2^t)
//
// 8-bit moments are blocks of 256 values with an fp32 scale each: m = q s (q in -127..127, s = max|m| / 127) and
// v = (q s)^2 (q in 0..255, s = max sqrt(v) / 255; the root is the one that the update takes anyway).  A code is
// the nearest, or one of the two neighbours at random so that the expected value is m or v itself: for v, between
// (q s)^2 and ((q + 1) s)^2, the upper one with probability (x - q)(x + q) / (2 q + 1), x = sqrt(v) / s.  Without
// that an average that moves by less than half a code per step would never move.  A positive v never gets code 0,
// or the next update could divide a moment by eps alone.  A block with a moment that is not finite is stored as NaN.
//
// One launch for up to 384 tensors, which streams everything once: 16.1 bytes per parameter with 8-bit moments and
// bf16 weights.  A warp works the coefficients out again whenever its tensor changes (fp64, from the tensor's step
// count); the last CTA to finish advances the step counts, when every other has read them.
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

constexpr int kBlock = ABX_I8_BLOCK;      // values per scale: 8 per lane of a warp
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = kWarps * kBlock;    // elements of one tensor that a CTA takes at a time
constexpr int kMany = 384;                // tensors per launch: the parameter block stays under 32764 bytes
constexpr int kFew = 24;                  // ... of the variant for few tensors (a smaller block to pass)

constexpr int64_t kMaxTiles = int64_t(1) << 30;   // of a launch: a tile index plus the grid fits 32 bits

static_assert(kBlock == 256, "a lane owns 8 consecutive values of its warp's block");

struct Item {
    void* w;
    const void* g;
    float* master;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    int64_t* step;
    int64_t n;
    int32_t tile_begin;   // first tile in the launch's tile space
    uint32_t index_vec;   // index << 1 | (w and g start on 16-byte boundaries)
};

template <int N>
struct Args {
    double lr, b1d, b2d, weight_decay;
    const void* lr_ptr;
    const float* g_scale;
    const float* skip;
    const float* norm;
    uint32_t* ticket;     // CTAs that have finished; 0 between launches
    int32_t lr_f64;
    int32_t count;
    int32_t tiles;
    uint32_t seed;
    float b1, omb1, b2, omb2, eps;
    Item t[N];
};

static_assert(sizeof(Args<kMany>) <= 32764, "kernel parameter space");

// ---- the coefficients of one step --------------------------------------------------------------

struct StepCoef {
    float decay, step_size, inv_sqrt_bc2;
    uint32_t stream;
};

// b^t by squaring: at most 2 log2(t) roundings of 2^-53, far below the fp32 coefficients' own
__device__ __forceinline__ double power(double b, int64_t t)
{
    double r = 1.0;
    for (; t > 0; t >>= 1) {
        if (t & 1) r *= b;
        b *= b;
    }
    return r;
}

// Called by whole warps: even lanes raise beta1, odd lanes beta2.
template <int N>
__device__ __forceinline__ StepCoef step_coef(const Args<N>& a, const Item& t)
{
    const int64_t step = *t.step + 1;
    double lr = a.lr;
    if (a.lr_ptr != nullptr) {
        if (a.lr_f64) lr = *static_cast<const double*>(a.lr_ptr);
        else lr = *static_cast<const float*>(a.lr_ptr);
    }
    const double bc = 1.0 - power((threadIdx.x & 1) ? a.b2d : a.b1d, step);
    const double bc1 = __shfl_sync(0xffffffffU, bc, 0), bc2 = __shfl_sync(0xffffffffU, bc, 1);
    StepCoef c;
    c.decay = (float)(1.0 - lr * a.weight_decay);
    c.step_size = (float)(lr / bc1);
    c.inv_sqrt_bc2 = (float)(1.0 / sqrt(bc2));
    c.stream = abx::hash32(abx::hash32(abx::hash32(a.seed) ^ (t.index_vec >> 1)) ^ (uint32_t)step);
    return c;
}

// ---- eight values of a lane --------------------------------------------------------------------

__device__ __forceinline__ void load8(const float* p, float (&x)[8])
{
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

__device__ __forceinline__ void store8(float* p, const float (&x)[8])
{
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// cnt valid values at p (0 beyond them); one vector where they are all there and aligned
__device__ __forceinline__ void load8(const float* p, int cnt, bool vec, float (&x)[8])
{
    if (vec && cnt == 8) {
        load8(p, x);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = k < cnt ? p[k] : 0.0f;
    }
}

__device__ __forceinline__ void load8(const uint16_t* p, int cnt, bool vec, float (&x)[8])
{
    if (vec && cnt == 8) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[2 * j] = u2f(w[j] << 16); x[2 * j + 1] = u2f(w[j] & 0xffff0000U); }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = k < cnt ? u2f((uint32_t)p[k] << 16) : 0.0f;
    }
}

__device__ __forceinline__ void store8(float* p, int cnt, bool vec, const float (&x)[8])
{
    if (vec && cnt == 8) {
        store8(p, x);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) if (k < cnt) p[k] = x[k];
    }
}

__device__ __forceinline__ void store8(uint16_t* p, int cnt, bool vec, const float (&x)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = abx::pack_bf16_rne(x[2 * j], x[2 * j + 1]);
    if (vec && cnt == 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) if (k < cnt) p[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
    }
}

// ---- the 8-bit block format ----------------------------------------------------------------------

// Bytes become floats by way of the significand of 2^23 + byte: one byte permute and one exact subtraction each.
__device__ __forceinline__ void decode_m(uint2 codes, float s, float (&x)[8])
{
    const uint32_t w[2] = {codes.x ^ 0x80808080U, codes.y ^ 0x80808080U};   // code + 128
#pragma unroll
    for (int k = 0; k < 8; ++k)
        x[k] = __fmul_rn(u2f(__byte_perm(w[k >> 2], 0x4b000000U, 0x7440 + (k & 3))) - (8388608.0f + 128.0f), s);
}

__device__ __forceinline__ void decode_v(uint2 codes, float s, float (&x)[8])
{
    const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float r = __fmul_rn(u2f(__byte_perm(w[k >> 2], 0x4b000000U, 0x7440 + (k & 3))) - 8388608.0f, s);
        x[k] = __fmul_rn(r, r);
    }
}

// The block's largest magnitude; a NaN's bits are above every number's, so it is a NaN if any value is.
__device__ __forceinline__ float block_max(const float (&x)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, f2u(x[k]) & 0x7fffffffU);
    return u2f(__reduce_max_sync(0xffffffffU, m));
}

// The factor from values to codes and the stored scale.  `below` is the float next below the largest code: value
// * (below / top) then never rounds above that code.  A block under 2^-100 is stored as zeros: below / top would
// overflow.  top not finite: the stored scale is NaN.
__device__ __forceinline__ float block_scale(float top, float below, float inverse, float& scale)
{
    const bool some = !(top <= 0x1p-100f);
    scale = some ? __fmul_rn(top, inverse) : 0.0f;
    if (!(top <= 3.402823466e38f)) scale = u2f(0x7fffffffU);
    return some ? __fdiv_rn(below, top) : 0.0f;
}

constexpr float kBelow127 = 126.99999237060546875f, kBelow255 = 254.9999847412109375f;
constexpr float kWhole = 12582912.0f;   // 1.5 * 2^23: a sum with it has the addend, rounded, in its low bits

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <bool SR>
__device__ __forceinline__ uint2 encode_m(const float (&m)[8], float f, const uint32_t (&r)[8])
{
    uint32_t q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float x = __fmul_rn(m[k], f);
        if (SR) {   // floor(x + u), u = the low 16 bits / 2^16
            const float u = __fmul_rn(u2f(0x4b000000U | (r[k] & 0xffffU)) - 8388608.0f, 0x1p-16f);
            q[k] = f2u(__fadd_rd(__fadd_rn(x, u), kWhole));
        } else {
            q[k] = f2u(__fadd_rn(x, kWhole));
        }
    }
    return make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
}

template <bool SR>
__device__ __forceinline__ uint2 encode_v(const float (&root)[8], float f, const uint32_t (&r)[8])
{
    uint32_t c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float x = __fmul_rn(root[k], f);
        if (SR) {
            const float z = __fadd_rd(x, kWhole);
            const float q = z - kWhole;
            const float u = __fmul_rn(u2f(__byte_perm(r[k], 0x4b000000U, 0x7632)) - 8388608.0f, 0x1p-16f);
            const bool up = __fmul_rn(x - q, x + q) > __fmul_rn(u, q + q + 1.0f);
            c[k] = (f2u(z) & 0xffU) + (up ? 1U : 0U);
        } else {
            c[k] = f2u(__fadd_rn(x, kWhole)) & 0xffU;
        }
        c[k] = root[k] > 0.0f ? max(c[k], 1U) : c[k];
    }
    return make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
}

// ---- the step ------------------------------------------------------------------------------------

template <int N>
__device__ __forceinline__ int find_item(const Args<N>& a, int tile)
{
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.t[mid].tile_begin <= tile) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// W: the weights' and gradients' type (float, or uint16_t for bf16 bits with an fp32 master).
template <bool I8, bool SR, typename W, int N>
__global__ void __launch_bounds__(kThreads) step_kernel(const __grid_constant__ Args<N> a)
{
    constexpr bool kMaster = sizeof(W) == 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // skip is a flag as loss scalers write it; a norm that is not finite says the same of the gradients
    if (a.skip != nullptr && !(*a.skip == 0.0f)) return;
    if (a.norm != nullptr && !(fabsf(*a.norm) <= 3.402823466e38f)) return;
    const float scale = a.g_scale != nullptr ? *a.g_scale : 1.0f;
    StepCoef c;
    int current = -1;
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        const int it = find_item(a, tile);
        const Item& t = a.t[it];
        if (it != current) {
            c = step_coef(a, t);
            current = it;
        }
        const bool vec = t.index_vec & 1;
        const int64_t b0 = (int64_t)(tile - t.tile_begin) * kTile + warp * kBlock;
        if (b0 >= t.n) continue;
        const int64_t i0 = b0 + lane * 8;
        const int64_t left = t.n - i0;
        const int cnt = left >= 8 ? 8 : (left > 0 ? (int)left : 0);

        float g[8], p[8], m[8], v[8], root[8];
        load8(static_cast<const W*>(t.g) + i0, cnt, vec, g);
        if constexpr (kMaster) load8(t.master + i0, p);
        else load8(static_cast<const float*>(t.w) + i0, cnt, vec, p);
        if constexpr (I8) {
            const uint2 mc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.m) + i0);
            const uint2 vc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.v) + i0);
            decode_m(mc, t.m_scale[b0 / kBlock], m);
            decode_v(vc, t.v_scale[b0 / kBlock], v);
        } else {
            load8(static_cast<const float*>(t.m) + i0, m);
            load8(static_cast<const float*>(t.v) + i0, v);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float gk = __fmul_rn(g[k], scale);
            m[k] = __fadd_rn(__fmul_rn(m[k], a.b1), __fmul_rn(gk, a.omb1));
            v[k] = __fadd_rn(__fmul_rn(v[k], a.b2), __fmul_rn(__fmul_rn(gk, a.omb2), gk));
            root[k] = __fsqrt_rn(v[k]);
            const float d = __fadd_rn(__fmul_rn(root[k], c.inv_sqrt_bc2), a.eps);
            p[k] = __fsub_rn(__fmul_rn(p[k], c.decay), __fmul_rn(__fdiv_rn(m[k], d), c.step_size));
        }
        if (cnt < 8) {   // beyond the tensor's end the state stays zero
#pragma unroll
            for (int k = 0; k < 8; ++k) if (k >= cnt) p[k] = m[k] = root[k] = 0.0f;
        }
        if constexpr (kMaster) store8(t.master + i0, p);
        store8(static_cast<W*>(t.w) + i0, cnt, vec, p);
        if constexpr (I8) {
            uint32_t r[8];
            if constexpr (SR) {
                uint32_t r0[4], r1[4];
                abx::hash4((uint32_t)i0, c.stream, r0);
                abx::hash4((uint32_t)i0 + 4, c.stream, r1);
#pragma unroll
                for (int k = 0; k < 4; ++k) { r[k] = r0[k]; r[4 + k] = r1[k]; }
            }
            float sm, sv;
            const float fm = block_scale(block_max(m), kBelow127, 1.0f / 127.0f, sm);
            const float fv = block_scale(block_max(root), kBelow255, 1.0f / 255.0f, sv);
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(t.m) + i0) = encode_m<SR>(m, fm, r);
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(t.v) + i0) = encode_v<SR>(root, fv, r);
            if (lane == 0) {
                t.m_scale[b0 / kBlock] = sm;
                t.v_scale[b0 / kBlock] = sv;
            }
        } else {
            store8(static_cast<float*>(t.m) + i0, m);
            store8(static_cast<float*>(t.v) + i0, v);
        }
    }
    __shared__ bool last;
    __syncthreads();                      // this CTA has read its step counts
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(a.ticket, 1U) == gridDim.x - 1;
    }
    __syncthreads();
    if (last) {
        for (int i = threadIdx.x; i < a.count; i += kThreads) *a.t[i].step += 1;
        if (threadIdx.x == 0) *a.ticket = 0;
    }
}

// ---- 8-bit moments to and from fp32 ----------------------------------------------------------------

struct I8Args {
    void* codes;
    float* scales;
    float* values;
    int64_t n;
    int64_t blocks;
};

template <bool V>
__global__ void __launch_bounds__(kThreads) i8_decode(const I8Args a)
{
    const int lane = threadIdx.x & 31;
    const bool vec = (reinterpret_cast<uintptr_t>(a.values) & 15) == 0;
    for (int64_t b = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); b < a.blocks; b += (int64_t)gridDim.x * kWarps) {
        const int64_t i0 = b * kBlock + lane * 8, left = a.n - i0;
        if (left <= 0) continue;
        const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.codes) + i0);
        float x[8];
        if constexpr (V) decode_v(c, a.scales[b], x);
        else decode_m(c, a.scales[b], x);
        store8(a.values + i0, left < 8 ? (int)left : 8, vec, x);
    }
}

// Nearest codes.  A negative second moment counts as 0.
template <bool V>
__global__ void __launch_bounds__(kThreads) i8_encode(const I8Args a)
{
    const int lane = threadIdx.x & 31;
    const bool vec = (reinterpret_cast<uintptr_t>(a.values) & 15) == 0;
    for (int64_t b = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); b < a.blocks; b += (int64_t)gridDim.x * kWarps) {
        const int64_t i0 = b * kBlock + lane * 8, left = a.n - i0;
        float x[8];
        load8(a.values + i0, left >= 8 ? 8 : (left > 0 ? (int)left : 0), vec, x);
        if constexpr (V) {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = __fsqrt_rn(x[k] < 0.0f ? 0.0f : x[k]);
        }
        uint32_t none[8] = {};
        float s;
        uint2 c;
        if constexpr (V) c = encode_v<false>(x, block_scale(block_max(x), kBelow255, 1.0f / 255.0f, s), none);
        else c = encode_m<false>(x, block_scale(block_max(x), kBelow127, 1.0f / 127.0f, s), none);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.codes) + i0) = c;
        if (lane == 0) a.scales[b] = s;
    }
}

// ---- host side ---------------------------------------------------------------------------------------

bool off(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

int check(const abx_graph_tensor& t, const abx_graph_step& h)
{
    if (t.n < 0 || t.n > kTile * kMaxTiles || t.index >= 0x80000000U) return ABX_E_ARG;
    if (t.dtype != ABX_DT_F32 && t.dtype != ABX_DT_BF16) return ABX_E_G_DTYPE;
    if (t.n == 0) return ABX_OK;
    if (!t.w || !t.g || !t.m || !t.v || !t.step) return ABX_E_NULL_PTR;
    if (t.dtype == ABX_DT_BF16 && !t.master) return ABX_E_NULL_PTR;
    if (h.moments == ABX_DT_I8 && (!t.m_scale || !t.v_scale)) return ABX_E_SCALE_NULL;
    const uintptr_t es = t.dtype == ABX_DT_BF16 ? 2 : 4;
    if (off(t.w, es) || off(t.g, es) || off(t.step, 8)) return ABX_E_ALIGN;
    if (off(t.m, 16) || off(t.v, 16) || (t.dtype == ABX_DT_BF16 && off(t.master, 16))) return ABX_E_ALIGN;
    if (h.moments == ABX_DT_I8 && (off(t.m_scale, 4) || off(t.v_scale, 4))) return ABX_E_ALIGN;
    return ABX_OK;
}

int resident_ctas(const void* kernel, int* out)
{
    int dev = 0, sms = 0, per = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kThreads, 0);
    if (e != cudaSuccess) return abx::set_error("launch geometry", e);
    *out = sms * (per > 0 ? per : 1);
    return ABX_OK;
}

template <bool I8, bool SR, typename W, int N>
int launch_step(const Args<N>& a, int32_t max_ctas, cudaStream_t st)
{
    int grid = 0;
    if (int rc = resident_ctas((const void*)step_kernel<I8, SR, W, N>, &grid)) return rc;
    if (grid > a.tiles) grid = a.tiles;
    if (max_ctas > 0 && grid > max_ctas) grid = max_ctas;
    step_kernel<I8, SR, W, N><<<grid, kThreads, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return abx::set_error("step_kernel launch", e);
    abx::g_launches.fetch_add(1, std::memory_order_relaxed);
    return ABX_OK;
}

// One launch for `count` tensors (indices `order`) of one dtype.
template <int N>
int run_batch(const abx_graph_tensor* t, const int32_t* order, int32_t count, int64_t tiles, const abx_graph_step& h,
              uint32_t* ticket, int32_t max_ctas, cudaStream_t st)
{
    static thread_local Args<N> a;   // kept off the stack
    a.lr = h.lr; a.b1d = h.beta1; a.b2d = h.beta2; a.weight_decay = h.weight_decay;
    a.lr_ptr = h.lr_ptr; a.lr_f64 = h.lr_f64;
    a.g_scale = h.g_scale; a.skip = h.skip; a.norm = h.norm; a.ticket = ticket;
    a.count = count; a.tiles = (int32_t)tiles; a.seed = h.seed;
    a.b1 = (float)h.beta1; a.omb1 = (float)(1.0 - h.beta1);
    a.b2 = (float)h.beta2; a.omb2 = (float)(1.0 - h.beta2);
    a.eps = (float)h.eps;
    int64_t next = 0;
    for (int32_t j = 0; j < count; ++j) {
        const abx_graph_tensor& s = t[order[j]];
        const uint32_t vec = !off(s.w, 16) && !off(s.g, 16);
        a.t[j] = Item{s.w, s.g, s.master, s.m, s.v, s.m_scale, s.v_scale, s.step, s.n, (int32_t)next, s.index << 1 | vec};
        next += (s.n + kTile - 1) / kTile;
    }
    const bool wide = t[order[0]].dtype == ABX_DT_F32;
    if (h.moments == ABX_DT_F32)
        return wide ? launch_step<false, false, float, N>(a, max_ctas, st) : launch_step<false, false, uint16_t, N>(a, max_ctas, st);
    if (h.stochastic)
        return wide ? launch_step<true, true, float, N>(a, max_ctas, st) : launch_step<true, true, uint16_t, N>(a, max_ctas, st);
    return wide ? launch_step<true, false, float, N>(a, max_ctas, st) : launch_step<true, false, uint16_t, N>(a, max_ctas, st);
}

int i8_check(const void* codes, const float* scales, const float* values, int64_t n, int32_t role)
{
    if (n < 0 || (role != 0 && role != 1)) return ABX_E_ARG;
    if (n == 0) return ABX_OK;
    if (!codes || !values) return ABX_E_NULL_PTR;
    if (!scales) return ABX_E_SCALE_NULL;
    if (off(codes, 8) || off(scales, 4) || off(values, 4)) return ABX_E_ALIGN;
    return ABX_OK;
}

template <void (*KM)(const I8Args), void (*KV)(const I8Args)>
int i8_run(void* stream, void* codes, float* scales, float* values, int64_t n, int32_t role, const char* what)
{
    if (int rc = i8_check(codes, scales, values, n, role)) return rc;
    if (n == 0) return ABX_OK;
    const I8Args a{codes, scales, values, n, (n + kBlock - 1) / kBlock};
    int grid = 0;
    if (int rc = resident_ctas(role ? (const void*)KV : (const void*)KM, &grid)) return rc;
    const int64_t need = (a.blocks + kWarps - 1) / kWarps;
    if (need < grid) grid = (int)need;
    if (role) KV<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    else KM<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return abx::set_error(what, e);
    abx::g_launches.fetch_add(1, std::memory_order_relaxed);
    return ABX_OK;
}

}  // namespace

ABX_API int abx_graph_tensor_size(void) { return (int)sizeof(abx_graph_tensor); }
ABX_API int abx_graph_step_size(void) { return (int)sizeof(abx_graph_step); }

ABX_API int abx_graph_adamw(void* stream, const abx_graph_tensor* tensors, int32_t n, const abx_graph_step* step,
                            uint32_t* ticket, int32_t max_ctas)
{
    if (n < 0 || !step || max_ctas < 0 || (n > 0 && (!tensors || !ticket))) return ABX_E_ARG;
    const abx_graph_step& h = *step;
    if (h.moments != ABX_DT_F32 && h.moments != ABX_DT_I8) return ABX_E_MV_DTYPE;
    if (!(h.beta1 >= 0.0 && h.beta1 < 1.0 && h.beta2 >= 0.0 && h.beta2 < 1.0)) return ABX_E_ARG;
    if (off(h.g_scale, 4) || off(h.skip, 4) || off(h.norm, 4) || off(h.lr_ptr, h.lr_f64 ? 8 : 4)) return ABX_E_ALIGN;
    if (off(ticket, 4)) return ABX_E_ALIGN;
    for (int32_t i = 0; i < n; ++i)
        if (int rc = check(tensors[i], h)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // batches of one dtype, at most kMany tensors and kMaxTiles tiles each
    int32_t order[kMany];
    for (const int32_t dtype : {ABX_DT_F32, ABX_DT_BF16}) {
        int32_t i = 0;
        while (i < n) {
            int32_t count = 0;
            int64_t tiles = 0;
            for (; i < n && count < kMany; ++i) {
                if (tensors[i].dtype != dtype || tensors[i].n == 0) continue;
                const int64_t more = (tensors[i].n + kTile - 1) / kTile;
                if (tiles + more > kMaxTiles) break;
                order[count++] = i;
                tiles += more;
            }
            if (count == 0) break;   // only other dtypes and empty tensors were left
            const int rc = count <= kFew ? run_batch<kFew>(tensors, order, count, tiles, h, ticket, max_ctas, st)
                                         : run_batch<kMany>(tensors, order, count, tiles, h, ticket, max_ctas, st);
            if (rc) return rc;
        }
    }
    return ABX_OK;
}

ABX_API int abx_i8_decode(void* stream, const void* codes, const float* scales, float* values, int64_t n, int32_t role)
{
    return i8_run<i8_decode<false>, i8_decode<true>>(stream, const_cast<void*>(codes), const_cast<float*>(scales), values,
                                                     n, role, "i8_decode launch");
}

ABX_API int abx_i8_encode(void* stream, const float* values, void* codes, float* scales, int64_t n, int32_t role)
{
    return i8_run<i8_encode<false>, i8_encode<true>>(stream, codes, scales, const_cast<float*>(values), n, role,
                                                     "i8_encode launch");
}
